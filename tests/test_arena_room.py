"""An arena that is full to the byte: where large tensors begin (at a line of the caches) takes nothing of its size."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MB = 1 << 20

PRELUDE = """
from attention_superoptimizer_amd import _native as N, graph as G
G.set_smem_budget(1 << 20)
g = G.KNGraph()
left = lambda: N.runtime().mirage_arena_total() - N.runtime().mirage_arena_offset()
small = g.new_input((8,))
"""


def _run(text, size):
    r = subprocess.run([sys.executable, "-c", PRELUDE + text], cwd=ROOT, capture_output=True, text=True,
                       env=dict(os.environ, MIRAGE_HOST_ONLY="1", MIRAGE_ARENA_BYTES=str(size)))
    return r


INPUTS = """
a, b = g.new_input((1 << 10, 1 << 9)), g.new_input((1 << 10, 1 << 9))
assert left() == 0 and a.device_ptr(False) % 256 == 0 and b.device_ptr(False) % 256 == 0
g.pop_operator()
assert left() == 2 << 20
"""
TWO_RESULTS = """
x, y = g.new_input((1 << 10, 1 << 9)), g.new_input((1 << 10, 1 << 9))
plan = dict(grid_dim=[16, 1, 1], forloop_range=1, input_map=[[0, -1, -1], [0, -1, -1]], forloop_dim=[-1, -1], output_map=[0, -1, -1],
            ops=[("tb_exp_op", [(0, 0)]), ("tb_exp_op", [(1, 0)])])
out = g.customized([x, y], plan)
assert len(out) == 2 and left() == 0
"""
ROTARY = """
x, p, w = g.new_input((1 << 10, 8, 64)), g.new_input((1 << 10,), G.DT_INT32), g.new_input((2, 32), G.DT_DOUBLE)
try:
    g.rotary(x, p, w)
    print("taken", left())
except G.InfeasibleOperator:
    print("refused")
"""


@pytest.mark.parametrize("text,size", [(INPUTS, 32 + 4 * MB), (TWO_RESULTS, 32 + 8 * MB)])
def test_what_fits_to_the_byte_is_built(text, size):
    r = _run(text, size)
    assert r.returncode == 0, r.stderr


def test_an_operator_of_a_decoding_step_fits_to_the_byte(capfd):
    size = 32 + 2 * MB + (4096 + 2048) + (512 + 128) + 2 * MB
    assert _run(ROTARY, size).stdout == "taken 0\n"
    assert _run(ROTARY, size - 16).stdout == "refused\n"


def test_one_byte_less_does_not_fit():
    r = _run(INPUTS, 32 + 4 * MB - 16)
    assert r.returncode != 0
