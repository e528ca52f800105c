"""attention_paged where lengths, scores or values are far from ordinary: results, and what they cost."""
import numpy as np
import pytest

import decode_ref as R
import viper_amd as va
from test_gpu_attention import check, setup, workspace
from test_gpu_kv_cache import SENT, back, dev, gpu_cache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def took_us(call, n=4):
    """The fastest of n calls, GPU time."""
    call()
    best = float("inf")
    for _ in range(n):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        b.synchronize()
        best = min(best, 1000 * a.elapsed_time(b))
    return best


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("ws", [True, False])
def test_lengths_past_the_table_walk_no_more_than_the_table(i8, ws):
    """First tokens and a window of a length that no table holds: the rows are NaN, and no tile past the table is walked."""
    D, page, kvh, heads, rows = 128, 64, 4, 20, 2
    c, table, offs, total, q, _ = setup(D, i8, page, kvh, heads, [600], rows, seed=33)
    g = gpu_cache(c)
    most = 2 ** 31 - 1
    for n in (most, most - 40, 10 ** 9, table.shape[1] * page + rows):
        batch = va.KVBatch(dev(table), dev(np.array([n], np.int32)), rows)
        w = workspace(g, batch, heads) if ws else None
        Q, out = dev(q), dev(np.full((rows, heads * D), SENT))
        for window, sinks in ((1, most), (1, most - 40), (40, 10 ** 9), (most, most), (1, 100)):
            print(f"length {n} window {window} sinks {sinks}", flush=True)
            assert took_us(lambda: va.attention_paged(g, batch, Q, out, window=window, sinks=sinks, workspace=w), 2) < 2000
            assert np.all(np.isnan(R.bf16_val(back(out))))
