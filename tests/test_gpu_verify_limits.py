"""Numbers of drafts that no int of the kernel counts are refused by the C ABI, as the graph's operator refuses them."""
import numpy as np
import pytest

from attention_superoptimizer_amd import graph as G
from decoding_reference import put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("drafts,code", [(2 ** 30, -4), (2 ** 31 - 64, -4), (2 ** 31 - 2, -4), (2 ** 31 - 1, -3)])
def test_too_many_drafts(rt, abi, drafts, code):
    g = G.KNGraph()
    try:
        at = put(g, np.zeros(64, np.float32)).device_ptr(False)
        for draft in (None, at):
            assert abi.mi355_verify_drafts(at, draft, at, at, at, at, 1, drafts, 1, 930) == code
    finally:
        g.close()
