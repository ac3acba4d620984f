"""What a launch of attention of few rows within a window counts in 32 bits (include/mi355_kernels/paged_units.h), without a device: the units are those of
the keys that are seen, of which a long table has many more."""
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ask(tmp_path_factory):
    exe = tmp_path_factory.mktemp("units") / "masked_units"
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), "-o", str(exe),
                           os.path.join(ROOT, "tests", "cpp", "masked_units.cc")])

    def many(cases):
        out = subprocess.run([str(exe)], input="".join("%d %d %d %d %d %d\n" % c for c in cases), capture_output=True, text=True, check=True).stdout
        return [tuple(int(x) for x in line.split()) for line in out.splitlines()]

    return many


def test_units_fit_an_int(ask):
    cases = [(kv, 1, 1, keys, window, sinks) for kv in (1, 8, 64, 1000) for keys in (512, 513, 600, 767, 768, 5000, 1 << 30)
             for window, sinks in ((512, 0), (508, 4), (500, 13), (1, 0), (2000, 4), (0, 0))]
    rng = random.Random(1)
    for _ in range(20000):
        group, tokens = rng.choice([(1, 1), (4, 1), (16, 1), (1, 16), (4, 4), (3, 5)])
        keys, window, sinks = (int(2 ** rng.uniform(0, p)) for p in (30, 12, 10))
        cases.append((int(2 ** rng.uniform(0, 20)), group, tokens, keys, window, sinks))
    cases = [c for c in cases if c[0] * (c[1] * c[2] // 16 + 1) * (c[3] // 128 + 2) <= (2 ** 31 - 1) // 4]  # (others go to blocks of rows)
    assert len(cases) > 10000
    for case, (at_once, units) in zip(cases, ask(cases)):
        assert at_once >= 1 and units < 2 ** 31 - 4096, (case, at_once, units)
