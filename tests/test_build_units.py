"""Which units _build.py compiles anew, with a compiler that only writes down how it was called."""
import os
import shutil
from importlib import util

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "z-ant_b200", "_build.py")
NVCC = """#!/bin/sh
echo "$*" >> "$CALLS"
while [ $# -gt 0 ]; do
    case "$1" in -o) out="$2"; shift;; -MF) dep="$2"; shift;; *.cu) unit="$1";; esac
    shift
done
echo object > "$out"
[ -z "$dep" ] || printf '%s: %s\\n' "$out" "$unit" > "$dep"
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A package of two units, whose sources are an hour old."""
    package = tmp_path / "package"
    (package / "csrc").mkdir(parents=True)
    (tmp_path / "include").mkdir()
    (tmp_path / "bin").mkdir()
    for name in ("package/csrc/lib.cu", "package/csrc/decode_ops.cu", "include/zant_b200.h"):
        (tmp_path / name).write_text("\n")
        shift(tmp_path / name, -3600)
    shutil.copy(SOURCE, package / "_build.py")
    shift(package / "_build.py", -3600)
    nvcc = tmp_path / "bin" / "nvcc"
    nvcc.write_text(NVCC)
    nvcc.chmod(0o755)
    monkeypatch.setenv("PATH", f"{tmp_path / 'bin'}{os.pathsep}{os.environ['PATH']}")
    monkeypatch.setenv("CALLS", str(tmp_path / "calls"))

    def build():
        """The commands of a build by a process of its own."""
        calls = tmp_path / "calls"
        calls.write_text("")
        spec = util.spec_from_file_location("built", package / "_build.py")
        module = util.module_from_spec(spec)
        spec.loader.exec_module(module)
        module.build()
        return calls.read_text().splitlines()
    return tmp_path, build


def shift(path, seconds):
    t = os.path.getmtime(path) + seconds
    os.utime(path, (t, t))


def compiled(calls):
    return sorted(c.split()[-1].rsplit("/", 1)[1] for c in calls if " -c " in c)


def age(tmp_path):
    """Everything there is becomes a minute older."""
    for root, _, files in os.walk(tmp_path):
        for f in files:
            shift(os.path.join(root, f), -60)


def test_what_a_change_compiles(tree):
    tmp_path, build = tree
    first = build()
    assert compiled(first) == ["decode_ops.cu", "lib.cu"] and len(first) == 3
    assert build() == []
    age(tmp_path)
    (tmp_path / "package/csrc/decode_ops.cu").write_text("// changed\n")
    again = build()
    assert compiled(again) == ["decode_ops.cu"] and len(again) == 2


@pytest.mark.parametrize("edit", [True, False])
def test_other_flags_compile_all_units(tree, edit):
    tmp_path, build = tree
    build()
    age(tmp_path)
    script = tmp_path / "package/_build.py"
    script.write_text(script.read_text().replace('"-O3"', '"-O2"'))
    if edit:
        (tmp_path / "package/csrc/decode_ops.cu").write_text("// changed\n")
    calls = build()
    assert compiled(calls) == ["decode_ops.cu", "lib.cu"] and len(calls) == 3
    assert all("-O2" in c and "-O3" not in c for c in calls)
