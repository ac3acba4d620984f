"""mirage::search in C++ on graphs with operators that have no fingerprint: refused before anything is computed."""
import os
import signal
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "attention_superoptimizer_amd")


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    exe = tmp_path_factory.mktemp("guard") / "fingerprint_guard"
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I", os.path.join(ROOT, "include"), "-I", "/opt/rocm/include",
                           "-o", str(exe), os.path.join(ROOT, "tests", "cpp", "fingerprint_guard.cc"), "-L" + PKG, "-lmirage_runtime",
                           "-lmi355_backend", "-Wl,-rpath," + PKG])
    return exe


def _call(exe, what):
    return subprocess.run([str(exe), what], env=dict(os.environ, MIRAGE_HOST_ONLY="1"), capture_output=True, text=True)


@pytest.mark.parametrize("what", ["graph", "candidate", "reference", "outputs"])
def test_graphs_without_a_fingerprint_are_refused(exe, what):
    r = _call(exe, what)
    assert r.returncode == -signal.SIGABRT and "kn_rotary_op has no fingerprint" in r.stderr, r.stderr


def test_others_are_not(exe):
    r = _call(exe, "plain")  # (goes as far as it does without a device, or runs)
    assert "has no fingerprint" not in r.stderr
    r = _call(exe, "ask")
    assert r.returncode == 0 and r.stdout == "1 0\n"
