"""The division of the prompt kernel's work (csrc/attention/kv4_tiles.cuh), compiled for the host: the tiles before each row block against a count one by one,
also where they pass 32 bits."""
import os
import random
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "unimonomoe_b200", "csrc", "attention")
MAIN = r"""
#include <algorithm>
#include <cstdio>
using std::max;
using std::min;
#define __device__
#define __forceinline__ inline
#define __noinline__
#include "kv4_tiles.cuh"
int main() {
  mono::kv4::Item it;
  int rb;
  while (std::scanf("%d %d %d %d %d %d", &it.place0, &it.n, &it.len, &it.tb, &it.window, &rb) == 6)
    std::printf("%lld\n", static_cast<long long>(mono::kv4::tiles_before(it, rb)));
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    d = tmp_path_factory.mktemp("tiles")
    (d / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=signed-integer-overflow", "-fno-sanitize-recover=all", "-I", CSRC, str(d / "main.cpp"), "-o",
                    str(d / "tiles")], check=True)
    return str(d / "tiles")


def count(place0, n, length, tb, window, rb):
    i = np.arange(rb, dtype=np.int64)
    begin = np.maximum(place0 + i * tb + 1 - window, 0) if window else np.zeros_like(i)
    seen = np.minimum(length, np.maximum(place0 + np.minimum((i + 1) * tb, n), 0))
    return int(np.maximum(1, (seen + 127) // 128 - begin // 128).sum()) + 2 * rb


def ask(program, cases):
    text = "".join(" ".join(map(str, c)) + "\n" for c in cases)
    r = subprocess.run([program], input=text, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    return [int(x) for x in r.stdout.split()]


def test_small_and_ordinary_requests(program):
    rng, cases = random.Random(1), []
    for _ in range(4000):
        tb, n = rng.choice([1, 2, 3, 5, 8, 16, 21, 32, 64, 128, 256]), int(2 ** rng.uniform(0, 13))
        length = max(0, n + rng.choice([0, 1, 127, 128, -n // 2, -n, rng.randrange(9000)]))
        cases.append((length - n, n, length, tb, rng.choice([0, 0, 1, 90, 128, rng.randrange(1, 9000)]), rng.randrange(-(-n // tb) + 1)))
    assert ask(program, cases) == [count(*c) for c in cases]


def test_requests_whose_tiles_pass_32_bits(program):
    cases = [(0, 800_000, 800_000, 1, 0, 800_000), (0, 4_000_000, 4_000_000, 2, 0, 2_000_000), (2 ** 30, 3_000_000, 2 ** 30 + 3_000_000, 1, 0, 2_999_999),
             (0, 12_000_000, 12_000_000, 2, 5_000_000, 6_000_000), (0x7FFF0000 - 900_000, 900_000, 0x7FFF0000, 1, 0x7FFE0000, 900_000),
             (77, 5_500_000, 5_500_077, 1, 129, 5_499_999)]
    got = ask(program, cases)
    assert got == [count(*c) for c in cases] and max(got) > 2 ** 40 and min(got[:5]) > 2 ** 31
