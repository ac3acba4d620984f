"""Batches in several launches (csrc/backend/slices.h), up to the largest that an int counts."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_part_follows_the_one_before(tmp_path):
    exe = tmp_path / "launch_slices"
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-Wall", "-Werror", "-I", os.path.join(ROOT, "attention_superoptimizer_amd", "csrc", "backend"),
                           "-o", str(exe), os.path.join(ROOT, "tests", "cpp", "launch_slices.cc")])
    cases = [(0, 5), (1, 5), (5, 5), (6, 5), (65535, 65535), (65536, 65535), (2 ** 31 - 1, 65535), (2 ** 31 - 1, 2 ** 31 - 1),
             (2 ** 31 - 1, 2 ** 30), (2 ** 31 - 65535, 65535), (2 ** 31 - 1, 4096)]
    out = subprocess.run([str(exe)], input="".join("%d %d\n" % c for c in cases), capture_output=True, text=True, check=True).stdout
    for (total, most), line in zip(cases, out.splitlines()):
        assert [int(x) for x in line.split()] == [0, -(-total // most), total], (total, most)
