"""Compiles libzant_b200.so in-tree with nvcc for sm_100a (cross-compiles without a GPU)."""
import os
import shutil
import subprocess

_HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(_HERE, "csrc")
OUT = os.path.join(_HERE, "libzant_b200.so")
OBJECTS = os.path.join(_HERE, "build")
UNITS = ["lib.cu", "decode_ops.cu"]      # compiled side by side; the first takes minutes

NVCC_FLAGS = [
    "-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
    "-fmad=false",            # fp32 reference arithmetic: multiply and add are never fused
    "-Xcompiler", "-fPIC",
]


def _newest_source():
    newest = os.path.getmtime(os.path.abspath(__file__))       # the flags are in here
    for root, _dirs, files in os.walk(CSRC):
        for f in files:
            newest = max(newest, os.path.getmtime(os.path.join(root, f)))
    newest = max(newest, os.path.getmtime(os.path.join(_HERE, "..", "include", "zant_b200.h")))
    return newest


def _stale(target, depfile):
    """`target` is missing or older than a file that went into it (`depfile`, as nvcc wrote it), or than this one, which has the flags."""
    if not os.path.exists(target) or not os.path.exists(depfile):
        return True
    with open(depfile) as f:
        parts = f.read().replace("\\\n", " ").split(":", 1)[1].split() + [os.path.abspath(__file__)]
    made = os.path.getmtime(target)
    return any(not os.path.exists(p) or os.path.getmtime(p) > made for p in parts)


def _check(proc, out):
    if proc.returncode != 0:
        raise RuntimeError("nvcc failed:\n" + out)


def build(force=False, verbose=False):
    if not force and os.path.exists(OUT) and os.path.getmtime(OUT) >= _newest_source():
        return OUT
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    os.makedirs(OBJECTS, exist_ok=True)
    objects, running = [], []
    for unit in UNITS:
        stem = os.path.join(OBJECTS, unit[:-3])
        obj, dep = stem + ".o", stem + ".d"
        objects.append(obj)
        if force or _stale(obj, dep):
            cmd = [nvcc] + NVCC_FLAGS + (["-Xptxas", "-v"] if verbose else []) + ["-MMD", "-MF", dep, "-c", "-o", obj, os.path.join(CSRC, unit)]
            running.append(subprocess.Popen(cmd, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
    done = [(p, p.communicate()[0]) for p in running]
    for p, out in done:
        _check(p, out)
        if verbose:
            print(out)
    p = subprocess.run([nvcc] + NVCC_FLAGS + ["-shared", "-o", OUT] + objects, stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    _check(p, p.stdout)
    return OUT


if __name__ == "__main__":
    print(build(force=True, verbose=True))
