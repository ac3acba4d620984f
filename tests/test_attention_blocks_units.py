"""What a launch of attention of blocks of rows counts in 32 bits (include/mi355_kernels/attention_blocks_units.h), without a device."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    exe = tmp_path_factory.mktemp("units") / "attention_blocks_units"
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(ROOT, "include"),
                           "-o", str(exe), os.path.join(ROOT, "tests", "cpp", "attention_blocks_units.cc")])

    def many(cases):
        out = subprocess.run([str(exe)], input="".join("%d %d %d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True).stdout
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]

    return many


def test_threads_of_a_launch_fit_32_bits(ask):
    rng = random.Random(1)
    cases = []
    for _ in range(30000):
        sequences, group, kv = (int(2 ** rng.uniform(0, p)) for p in (31, 20, 20))
        ragged = rng.random() < 0.5
        tokens = min(int(2 ** rng.uniform(0, 31)), 2 ** 31 - 1) if ragged else sequences * int(2 ** rng.uniform(0, 12))
        cases.append((tokens, group, kv, sequences, int(ragged)))
    counted = 0
    for case, (fits, units) in zip(cases, ask(cases)):
        tokens, group, kv, sequences, ragged = case
        assert units * 256 < 2 ** 32, case
        if fits:
            counted += 1
            assert tokens * group <= 2 ** 30, case
    assert 1000 < counted < len(cases)


def test_ends(ask):
    most = 2 ** 24 - 1
    assert ask([(0, 4, 8, 0, 0), (0, 4, 8, 0, 1)]) == [(1, 0), (1, 0)]
    # many sequences of one block a head take several launches, of a ragged batch as many as one launch holds
    assert ask([(2 ** 26, 1, 8, 2 ** 26, 0)]) == [(1, most // 8 * 8)]
    assert ask([(4, 1, 1, most, 1), (4, 1, 1, most + 1, 1)]) == [(1, most), (0, 0)]
    # one sequence of more blocks than a launch has
    assert ask([(2 ** 20, 2 ** 10, 1, 1, 0), (2 ** 20, 2 ** 10, 2, 1, 0), (2 ** 20, 2 ** 11, 1, 1, 0)]) == [(1, 2 ** 23), (0, 0), (0, 0)]
