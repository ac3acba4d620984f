"""What a launch of paged attention counts in 32 bits (include/mi355_kernels/paged_units.h), without a device."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    exe = tmp_path_factory.mktemp("units") / "paged_units"
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", str(exe),
                           os.path.join(ROOT, "tests", "cpp", "paged_units.cc")])

    def many(cases):
        out = subprocess.run([str(exe)], input="".join("%d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True).stdout
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]

    return many


def _refused(kv, rows, keys):  # the limit the C ABI and the graph's operator have
    return kv * (rows // 16 + 1) * (keys // 128 + 2) > (2 ** 31 - 1) // 4


def test_units_fit_an_int(ask):
    """At every number of keys up to two thousand, and far ones: one head a sequence, many, the most that are not refused."""
    cases = []
    for keys in list(range(1, 2100)) + [1 << p for p in range(12, 31)] + [(1 << 30) - 1, 12345678]:
        for rows in (1, 8, 15, 16, 17, 32, 71, 1000):
            most = ((2 ** 31 - 1) // 4) // ((rows // 16 + 1) * (keys // 128 + 2))
            cases += [(kv, rows, keys) for kv in {1, 8, 128, most // 2, most // 3, most - 1, most} if kv >= 1]
    rng = random.Random(1)
    cases += [(int(2 ** rng.uniform(0, 29)), int(2 ** rng.uniform(0, 20)), int(2 ** rng.uniform(0, 30))) for _ in range(20000)]
    cases = [c for c in cases if c[0] * c[1] <= 1 << 29]  # (others are refused before)
    for case, (refused, at_once, units) in zip(cases, ask(cases)):
        assert refused == _refused(*case), case
        if not refused:
            assert at_once >= 1 and units < 2 ** 31 - 4096, (case, at_once, units)


def test_a_million_sequences_of_many_short_heads(ask):
    """128 heads of 8 over tables of 512 keys: 16 units of one wavefront each a head."""
    (refused, at_once, units), = ask([(128, 1, 512)])
    assert not refused and at_once < 1 << 20 and units <= (2 ** 31 - 1) // 2


def test_batches_that_were_one_launch_are(ask):
    for case in ((8, 4, 4096), (8, 8, 131072), (4, 40, 4096), (8, 4, 100), (32, 1, 1 << 17)):
        assert ask([case])[0][1] >= 128, case
