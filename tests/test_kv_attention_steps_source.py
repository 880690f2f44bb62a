"""KvSteps and KvPromptSteps as the sources have them, compiled for the CPU with overflow of int as an error, against the same arithmetic in Python's integers (test_kv_attention_steps); windows and sinks up to the
end of int32."""
import os
import random
import re
import shutil
import subprocess

import pytest

from test_kv_attention_steps import prompt_steps, steps_of

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "z-ant_b200", "csrc")
MAIN = r"""
#include <algorithm>
#include <cstdio>
#define __device__
#define __forceinline__ inline
using std::max;
using std::min;
%s
int main() {
    int low, high, window, sinks, tile_low, tile_high;
    while (std::scanf("%%d %%d %%d %%d %%d %%d", &low, &high, &window, &sinks, &tile_low, &tile_high) == 6) {
        for (int S : {16, 32, 128}) { const KvSteps s(low, high, window, sinks, S); std::printf("%%d %%d %%d ", s.sink, s.first, s.total); }
        const KvPromptSteps p(KvSteps(low, high, window, sinks, 128), tile_low, tile_high, window, sinks);
        std::printf("%%d %%d %%d %%d %%d\n", p.sink, p.from, p.to, p.whole_from, p.whole_to);
    }
}
"""


def struct(file, name):
    return re.search(r"^struct %s \{.*?^\};" % name, open(os.path.join(CSRC, file)).read(), re.M | re.S).group(0)


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no C++ compiler")
    at = tmp_path_factory.mktemp("steps")
    (at / "steps.cpp").write_text(MAIN % (struct("kv_attention.cuh", "KvSteps") + "\n" + struct("kv_prompt.cuh", "KvPromptSteps")))
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover", "-o", str(at / "steps"), str(at / "steps.cpp")], check=True)
    return str(at / "steps")


def test_the_sources_arithmetic_fits_32_bits(program):
    rng = random.Random(2)
    ends = [0, 0, 1, 5, 64, 128, 129, 300, 1000] + [2 ** 31 - n for n in (1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300)]
    cases = []
    for _ in range(20000):
        first, group, rows, row0 = rng.choice([rng.randint(-300, 3000), rng.randint(0, 2 ** 31 - 2 ** 17)]), rng.choice([1, 2, 5, 8]), rng.randint(1, 256), rng.randint(0, 3) * 256
        tiles = [(max(first + row0 // group, -1), max(first + (row0 + min(rows, 128) - 1) // group, -1)),
                 (max(first + (row0 + 128) // group, -1), -1 if rows <= 128 else max(first + (row0 + rows - 1) // group, -1))]
        window, sinks = rng.choice(ends), rng.choice(ends)
        for tile in tiles:
            cases.append((tiles[0][0], max(tiles[0][1], tiles[1][1]), window, sinks) + tile)
    run = subprocess.run([program], input="\n".join(" ".join(map(str, c)) for c in cases), capture_output=True, text=True)
    got = [tuple(map(int, line.split())) for line in run.stdout.splitlines()]
    assert run.returncode == 0, (run.stderr, cases[len(got)])
    for c, numbers in zip(cases, got, strict=True):
        want = sum((steps_of(*c[:4], size) for size in (16, 32, 128)), ()) + prompt_steps(steps_of(*c[:4], 128), *c[4:], *c[2:4])
        assert numbers == want, c
