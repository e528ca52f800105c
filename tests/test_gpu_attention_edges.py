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


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("ws", [True, False])
def test_a_poisoned_token_costs_no_second_pass(i8, ws):
    """A row that sees a key that is not a number is NaN whatever the rest holds: nothing is read again for it."""
    D, kvh, heads = 128, 4, 20
    n = 65536 if ws else 8192
    c, table, offs, total, q, batch = setup(D, i8, 256, kvh, heads, [n], 1, seed=30)
    g = gpu_cache(c)
    Q, out = dev(q), dev(np.full((total, heads * D), SENT))
    w = workspace(g, batch, heads) if ws else None

    def call():
        assert va.attention_paged(g, batch, Q, out, workspace=w).ok()

    clean = took_us(call)
    assert np.all(np.isfinite(R.bf16_val(back(out))))
    j = n - 700
    pg, at = int(table[0, j // 256]), j % 256
    for h in range(kvh):
        if i8:
            g.k_scales[c.scale_at(pg, at, h)] = float("nan")
        else:
            g.k[torch.from_numpy(c.places(pg, at, h, True)).cuda()] = 0x7FC0
    poisoned = took_us(call)
    assert np.all(np.isnan(R.bf16_val(back(out))))
    print(f"i8={i8} ws={ws}: clean {clean:.1f} us, poisoned {poisoned:.1f} us", flush=True)
    assert poisoned < 3 * clean + 100
    q[:, 5] = 0x7F80  # and a query that is not finite
    Q.copy_(dev(q))
    assert took_us(call) < 3 * clean + 100


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("ws", [True, False])
def test_an_infinite_value_costs_one_more_pass(i8, ws):
    """Rows that see an infinite value are computed again, each by one workgroup; rows that see a missing page are not."""
    D, kvh, heads = 128, 4, 20
    n = 65536 if ws else 8192
    c, table, offs, total, q, batch = setup(D, i8, 256, kvh, heads, [n], 1, seed=34)
    j = n - 700
    pg, at = int(table[0, j // 256]), j % 256
    for h in range(kvh):
        if i8:
            c.vs[c.scale_at(pg, at, h)] = np.inf
            c.v[c.places(pg, at, h, False)] = 3
        else:
            c.v[c.places(pg, at, h, False)] = 0x7F80
    g = gpu_cache(c)
    Q, out = dev(q), dev(np.full((total, heads * D), SENT))
    w = workspace(g, batch, heads) if ws else None

    def call(b=batch):
        assert va.attention_paged(g, b, Q, out, workspace=w).ok()

    us = took_us(call)
    assert np.all(np.isinf(R.bf16_val(back(out))))
    table[0, 1] = -1
    missing = va.KVBatch(dev(table), dev(np.array([n], np.int32)), 1)
    us_missing = took_us(lambda: call(missing))
    assert np.all(np.isnan(R.bf16_val(back(out))))
    print(f"i8={i8} ws={ws}: infinite value {us:.0f} us, missing page {us_missing:.0f} us", flush=True)
    assert us < (8000 if ws else 2500) and us_missing < 500


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("ws", [True, False])
def test_values_whose_sum_leaves_32_bits(i8, ws):
    """A weighted mean of finite values is finite, also where the sum of the values is not."""
    D, page, kvh, heads, lens, rows = 64, 32, 2, 4, [700, 33, 5], 3
    c, table, offs, total, q, batch = setup(D, i8, page, kvh, heads, lens, rows, seed=31, std=0.3)
    if i8:
        c.vs[:] = np.float32(2.6e36)  # codes up to 127: 3.3e38
        c.v[:] = np.abs(c.v)
    else:
        c.v[:] = R.bf16_bits(np.float32(3e38) * (1 + 0.1 * np.random.default_rng(32).uniform(-1, 1, len(c.v))).astype(np.float32))
    g = gpu_cache(c)
    out = dev(np.full((total, heads * D), SENT))
    assert va.attention_paged(g, batch, dev(q), out, workspace=workspace(g, batch, heads) if ws else None).ok()
    o, bound = R.attention(c, table, lens, rows, offs, q, heads, D ** -0.5)
    assert all(np.isfinite(x).all() for x in o.values())
    check(back(out), o, bound, lens, rows, offs)
