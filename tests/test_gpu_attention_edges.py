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


def apart(D, i8, kvh, heads, lens, rows, seed, **kw):
    """A setup whose table is wide enough that parts are joined by a launch of their own (80000 bytes of sums and more)."""
    c, table, offs, total, q, _ = setup(D, i8, 64, kvh, heads, lens, rows, seed=seed, **kw)
    wide = np.full((len(lens), 600), -1, np.int32)
    wide[:, :table.shape[1]] = table
    batch = va.KVBatch(dev(wide), dev(np.array(lens, np.int32)), rows)
    return c, wide, offs, total, q, batch


def assert_apart(batch, cache, D, kvh, heads, rows):
    g = heads // kvh * rows
    qt = -(-g // 16)
    assert qt <= 2  # (one group of rows)
    splits = (va.attention_workspace_bytes(cache, batch, heads) - 8192) // (batch.batch * kvh * qt * 16 * (D + 2) * 4)
    assert splits * g * D * 4 >= 80000


SHAPES = [(128, 4, 20, 3), (64, 2, 16, 4), (256, 1, 5, 3)]


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("D,kvh,heads,rows", SHAPES)
@pytest.mark.parametrize("value", [0x7F80, 0xFF80, 0x7FC0])
def test_join_of_values_that_are_not_finite(i8, D, kvh, heads, rows, value):
    """The newest row's own token holds it: the rows before do not see it; with a window that leaves an early one behind."""
    n = 3000
    for window, sinks, hit in ((0, 0, n - 1), (700, 5, n - 1), (700, 0, n - 701)):  # the last: behind the newest row's window
        c, table, offs, total, q, batch = apart(D, i8, kvh, heads, [n], rows, 60)
        pg, at = table[0, hit // 64], hit % 64
        for h in range(kvh):
            if i8:
                c.vs[c.scale_at(pg, at, h)] = R.bf16_val(np.uint16(value))
                c.v[c.places(pg, at, h, False)] = np.int8(3)
            else:
                c.v[c.places(pg, at, h, False)[::7]] = value
        g = gpu_cache(c)
        assert_apart(batch, g, D, kvh, heads, rows)
        out = dev(np.full((total, heads * D), SENT))
        assert va.attention_paged(g, batch, dev(q), out, window=window, sinks=sinks, workspace=workspace(g, batch, heads)).ok()
        o, bound = R.attention(c, table, [n], rows, offs, q, heads, D ** -0.5, window, sinks)
        finite = [bool(np.all(np.isfinite(o[r]))) for r in range(rows)]
        assert finite == ([True] * (rows - 1) + [False] if hit == n - 1 else [False] * (rows - 1) + [True])
        check(back(out), o, bound, [n], rows, offs, (window, hit))


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("D,kvh,heads,rows", SHAPES)
def test_join_of_missing_pages_and_keys_that_are_not_numbers(i8, D, kvh, heads, rows):
    """A page that only the newest row sees, one that every row sees, a NaN key of the newest token, a length past the table."""
    n = 45 * 64 + 1  # the newest token begins a page, the rows before it see the whole pages up to there
    c, table, offs, total, q, _ = apart(D, i8, kvh, heads, [n], rows, 61)
    o, bound = R.attention(c, table, [n], rows, offs, q, heads, D ** -0.5)

    def run(tb, length=n, cache=c):
        g = gpu_cache(cache)
        b = va.KVBatch(dev(tb), dev(np.array([length], np.int32)), rows)
        assert_apart(b, g, D, kvh, heads, rows)
        out = dev(np.full((total, heads * D), SENT))
        assert va.attention_paged(g, b, dev(q), out, workspace=workspace(g, b, heads)).ok()
        return back(out)

    def older_rows_only(got):
        y = R.bf16_val(got)
        assert np.all(np.isnan(y[rows - 1]))
        for r in range(rows - 1):
            assert np.all(np.abs(y[r].reshape(heads, D) - o[r]) <= bound[r]), r

    bad = table.copy()
    bad[0, 45] = c.pages  # the newest token's page
    older_rows_only(run(bad))
    bad[0, 45], bad[0, 20] = table[0, 45], -1
    assert np.all(np.isnan(R.bf16_val(run(bad))))
    for h in range(kvh):
        if i8:
            c.ks[c.scale_at(table[0, 45], 0, h)] = np.nan
        else:
            c.k[c.places(table[0, 45], 0, h, True)[9]] = 0x7FC0
    older_rows_only(run(table))
    cap = table.shape[1] * 64
    full = np.zeros_like(table)  # (every page is there: page 0 again and again)
    y = R.bf16_val(run(full, cap + 1))
    assert np.all(np.isnan(y[rows - 1])) and np.all(np.isfinite(y[:rows - 1]))


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("D,kvh,heads,rows", SHAPES)
def test_join_of_values_whose_sum_leaves_32_bits(i8, D, kvh, heads, rows):
    n = 1500
    c, table, offs, total, q, batch = apart(D, i8, kvh, heads, [n], rows, 62, std=0.3)
    if i8:
        c.vs[:] = np.float32(2.6e36)
        c.v[:] = np.abs(c.v)
    else:
        c.v[:] = R.bf16_bits(np.float32(3e38) * (1 + 0.1 * np.random.default_rng(63).uniform(-1, 1, len(c.v))).astype(np.float32))
    g = gpu_cache(c)
    assert_apart(batch, g, D, kvh, heads, rows)
    out = dev(np.full((total, heads * D), SENT))
    assert va.attention_paged(g, batch, dev(q), out, workspace=workspace(g, batch, heads)).ok()
    o, bound = R.attention(c, table, [n], rows, offs, q, heads, D ** -0.5)
    check(back(out), o, bound, [n], rows, offs)
