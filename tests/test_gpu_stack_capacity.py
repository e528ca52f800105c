"""A Stack whose context is no whole number of pages: what it holds, and that the step after the last token says so."""
import numpy as np
import pytest

import decode_ref as R
from test_gpu_attention import check
from test_gpu_stack_context import SMALL, bits
from viper_amd.stack import Stack

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("window", [0, 20])
def test_capacity_is_the_context_in_whole_pages(window):
    s = Stack(torch, **SMALL, context=100, page_size=32, window=window, sinks=2)
    assert s.context == 100 and s.capacity == 128
    s.seq_len.fill_(99)
    for n in range(100, 131):
        s.step_fused()
        torch.cuda.synchronize()
        assert s.seq_len.item() == n
        assert torch.isfinite(s.attn.float()).all() if n <= 128 else torch.isnan(s.attn.float()).all(), n
        if n in (101, 128):
            g = s.kv[3]
            c = R.Cache(False, 4, 32, 2, 64)
            c.k, c.v = bits(g.k).ravel(), bits(g.v).ravel()
            o, bound = R.attention(c, np.arange(4)[None, :], [n], 1, None, bits(s.q), 8, 64 ** -0.5, window, 2)
            check(bits(s.attn), o, bound, [n], 1, None, n)
