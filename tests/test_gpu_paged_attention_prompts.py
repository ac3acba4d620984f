"""paged_attention of whole prompts and of chunks behind a cache: hundreds of new tokens, many blocks of rows a head."""
import numpy as np
import pytest

from decoding_reference import attention, check
from test_gpu_paged_attention import _case, _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lengths,new,kv_heads,group,head,window,kind", [
    ([600], 600, 1, 3, 64, 0, "fp16"),       # a prompt
    ([257, 300], 257, 2, 1, 128, 0, "bf16"),
    ([900, 310], 300, 1, 2, 96, 0, "fp16"),  # a chunk behind a cache
    ([1500], 200, 1, 4, 128, 130, "bf16"),   # with a window that most of its rows have left
    ([90, 0, 400], 400, 1, 1, 256, 0, "fp16"),  # fewer keys than new tokens: the first rows see none
])
def test_prompts(rt, lengths, new, kv_heads, group, head, window, kind):
    x = _case(new + head, lengths, new, kv_heads, group, head, 16, kind)
    scale = float(np.float32(head ** -0.5))
    want, bound = attention(*x, scale, window, kind)
    check(_run(*x, kind, scale, window), want, bound)
    for b, length in enumerate(lengths):
        if length < new:
            assert (want[b, :new - length] == 0).all()
