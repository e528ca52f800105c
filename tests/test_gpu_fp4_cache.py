"""The 4-bit cache: kv_append and kv_read against the plain 64-bit implementation, attention_paged over it with the derived bound of
decode_ref.attention, a decode step's stack on it."""
import numpy as np
import pytest

import decode_ref as R
import fp4_ref as F
import viper_amd as va
from test_gpu_attention import check, workspace
from test_gpu_kv_cache import SENT, back, dev, step_of, table_for

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

APPEND = [  # D, page, kvh, heads, lens, counts (None: uniform rows), rows
    (128, 64, 4, 20, [1], None, 1),
    (128, 64, 4, 20, [1000, 31, 32, 33], None, 1),
    (64, 32, 1, 3, [70, 5], None, 5),
    (64, 32, 8, 8, [129, 40, 17], [16, 3, 1], 16),
    (256, 128, 2, 2, [300, 128, 127], [7, 0, 9], 9),
    (256, 256, 3, 12, [513, 258], [300, 258], 300),
    (128, 256, 8, 48, [700], None, 700),
    (128, 64, 2, 2, [3, 0, 64], None, 4),          # rows at negative positions
    (128, 64, 5, 10, [100003], None, 3),           # a far position
    (128, 64, 2, 4, [8, 16, 24, 15], None, 8),     # octets that begin and end with the rows
]


@pytest.mark.parametrize("D,page,kvh,heads,lens,counts,rows", APPEND)
@pytest.mark.parametrize("theta", [None, 10000.0])
def test_append_and_read(D, page, kvh, heads, lens, counts, rows, theta):
    rng = np.random.default_rng(D * 7 + rows)
    print(f"append fp4 D={D} page={page} rows={rows} lens={lens} theta={theta}", flush=True)
    table, pages = table_for(rng, lens, page)
    c = F.Cache4(pages, page, kvh, D, rng)
    offs = None if counts is None else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    total = len(lens) * rows if counts is None else int(offs[-1])
    wide = (heads + 2 * kvh) * D + 24  # rows of one projection, some columns behind them
    x = R.bf16_bits(rng.standard_normal((total, wide)) * np.exp(rng.uniform(-3, 3, (total, 1))))
    x[total // 2, heads * D:(heads + 1) * D] = 0  # a row of zeros
    g = F.gpu_cache(c, va, dev)
    X = dev(x)
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows, None if offs is None else dev(offs))
    q, k, v = X[:, :heads * D], X[:, heads * D:(heads + kvh) * D], X[:, (heads + kvh) * D:(heads + 2 * kvh) * D]
    qo = dev(np.full((total, heads * D + 8), SENT))
    st = va.kv_append(g, batch, k, v) if theta is None else va.kv_append(g, batch, k, v, q=q, q_out=qo[:, :heads * D], rope_theta=theta)
    assert st.ok(), st
    ko, vo = (dev(np.full((total, kvh, D), SENT)) for _ in range(2))
    assert va.kv_read(g, batch, ko, vo).ok()
    torch.cuda.synchronize()

    n = F.Cache4(pages, page, kvh, D)  # what is held now
    n.k, n.v, n.ks, n.vs = (back(t).ravel() for t in (g.k, g.v, g.k_scales, g.v_scales))
    qo, ko, vo = back(qo), back(ko), back(vo)
    elements = 32 * D * (pages * kvh * page // 32)
    kept = {"k": np.ones(elements, bool), "v": np.ones(elements, bool), "ks": np.ones(len(c.ks), bool), "vs": np.ones(len(c.vs), bool)}
    d = np.arange(D)
    for b, r, p in R.row_map(lens, rows, offs):
        if p < 0:
            assert np.all(qo[r] == SENT) and np.all(ko[r] == SENT) and np.all(vo[r] == SENT)
            continue
        row = lambda lo, m: R.bf16_val(x[r, lo:lo + m * D]).astype(np.float64).reshape(m, D)
        qr, kr, vr = row(0, heads), row(heads * D, kvh), row((heads + kvh) * D, kvh)
        if theta is not None:
            qr, kr = R.rotate(qr, p, theta), R.rotate(kr, p, theta)
            # (64 bits through 32 to bf16, as test_gpu_kv_cache derives it)
            assert np.all(np.abs(R.bf16_val(qo[r, :heads * D]).reshape(heads, D) - qr) <= step_of(qr) * (0.5 + 2.0 ** -16) + 1e-9)
            assert np.all(qo[r, heads * D:] == SENT)
        kr = R.bf16_val(R.bf16_bits(kr.astype(np.float32))).astype(np.float64)
        kh, kb = F.quantize_k(kr)
        pg, at = int(table[b, p // page]), p % page
        for h in range(kvh):
            vh, s = F.quantize_v(vr[h])
            t, tile = c.at(pg, at, h)
            for name, e in (("k", tile * 32 * D + F.k_nibble(t, d, D)), ("v", tile * 32 * D + F.v_nibble(t, d)),
                            ("ks", tile * D + F.exp_byte(t, np.arange(D // 32), D)), ("vs", tile * 32 + t)):
                kept[name][e] = False
            np.testing.assert_array_equal(n.ks[tile * D + F.exp_byte(t, np.arange(D // 32), D)], kb[h])
            assert n.vs[tile * 32 + t] == s
            np.testing.assert_array_equal(n.held(pg, at, h, True), kh[h])
            np.testing.assert_array_equal(F.value(n.code(n.v, tile * 32 * D + F.v_nibble(t, d))), vh)
            np.testing.assert_array_equal(R.bf16_val(ko[r, h]), kh[h])
            np.testing.assert_array_equal(R.bf16_val(vo[r, h]), R.bf16_val(R.bf16_bits(vh.astype(np.float32) * s)))
    e = np.arange(elements)
    for name in ("k", "v"):  # nothing else was written
        np.testing.assert_array_equal(n.code(getattr(n, name), e)[kept[name]], c.code(getattr(c, name), e)[kept[name]])
    for name in ("ks", "vs"):
        np.testing.assert_array_equal(getattr(n, name)[kept[name]], getattr(c, name)[kept[name]])


def test_every_mantissa_of_a_value_under_every_mantissa_of_a_row_s_largest():
    """All 128 mantissas of the largest value times all values down to 2^-6 of it, at three exponents: codes, scales, exponents.
    (Quotients depend on the exponents' difference alone, and values under 2^-6 are under a tenth of the least step.)"""
    D, page = 128, 256
    amax = 1 + np.arange(128) / 128
    x = np.concatenate([amax * 2.0 ** -e for e in range(7)] + [np.zeros(1)])
    rows = []
    for a in amax:
        v = np.concatenate([x[x < a], -x[x < a]])
        v = np.concatenate([v, np.zeros(-len(v) % (D - 1))]).reshape(-1, D - 1)
        rows.append(np.concatenate([np.full((len(v), 1), a), v], 1))
    rows = np.concatenate(rows)
    print(len(rows), "rows", flush=True)
    for e in (0, -20, 100):
        y = rows * 2.0 ** e
        bits = R.bf16_bits(y.astype(np.float32))
        np.testing.assert_array_equal(R.bf16_val(bits), y)
        n = len(y)
        pages = -(-n // page)
        g = va.KVCache.empty(va.KVType.FP4, pages, page, 1, D)
        table = dev(np.arange(pages, dtype=np.int32)[None, :])
        batch = va.KVBatch(table, dev(np.array([n], np.int32)), n)
        assert va.kv_append(g, batch, dev(bits), dev(bits)).ok()
        ko, vo = (dev(np.zeros((n, 1, D), np.uint16)) for _ in range(2))
        assert va.kv_read(g, batch, ko, vo).ok()
        np.testing.assert_array_equal(R.bf16_val(back(ko))[:, 0], F.quantize_k(y)[0])
        s = np.maximum(np.abs(y).max(1).astype(np.float32) / np.float32(6), np.float32(1e-8))
        held = F.nearest(y.astype(np.float32) / s[:, None]).astype(np.float32) * s[:, None]
        np.testing.assert_array_equal(R.bf16_val(back(vo))[:, 0], R.bf16_val(R.bf16_bits(held)))


def test_blocks_and_rows_that_are_not_finite_and_ends_of_the_range():
    D, page = 128, 32
    c = F.Cache4(2, page, 1, D)
    g = F.gpu_cache(c, va, dev)
    x = np.zeros((6, D), np.float32)
    x[0, 40], x[1, 3], x[2, 100] = np.nan, np.inf, -np.inf
    x[3], x[4, :64], x[5] = 3.3e38, 1e-38, -1e-6
    x[0, 0] = x[1, 127] = 2.0
    bits = R.bf16_bits(x)
    batch = va.KVBatch(dev(np.array([[1, 0]], np.int32)), dev(np.array([37], np.int32)), 6)
    assert va.kv_append(g, batch, dev(bits), dev(bits)).ok()
    ko, vo = (dev(np.zeros((6, 1, D), np.uint16)) for _ in range(2))
    assert va.kv_read(g, batch, ko, vo).ok()
    val = R.bf16_val(bits).astype(np.float64)
    kh, _ = F.quantize_k(val)
    np.testing.assert_array_equal(R.bf16_val(back(ko))[:, 0], kh)
    for r in range(6):
        vh, s = F.quantize_v(val[r])
        np.testing.assert_array_equal(R.bf16_val(back(vo)[r, 0]), R.bf16_val(R.bf16_bits(vh.astype(np.float32) * s)))


def test_tokens_written_by_steps_and_by_two_sequences_of_a_page():
    """Single tokens one call after the other, and a shared page of which two sequences of one call write different octets."""
    D, page, rng = 64, 32, np.random.default_rng(2)
    c = F.Cache4(1, page, 2, D, rng)
    g = F.gpu_cache(c, va, dev)
    x = R.bf16_bits(rng.standard_normal((32, 2 * D)))
    table = dev(np.zeros((2, 1), np.int32))
    assert va.kv_append(g, va.KVBatch(table, dev(np.array([3, 20], np.int32)), 2), dev(x[[1, 2, 18, 19]]), dev(x[[1, 2, 18, 19]])).ok()
    steps = (0, 3, 6, 7, 8, 31)
    for t in steps:
        one = va.KVBatch(table[:1].contiguous(), dev(np.array([t + 1], np.int32)), 1)
        assert va.kv_append(g, one, dev(x[t:t + 1]), dev(x[t:t + 1])).ok()
    n = F.Cache4(1, page, 2, D)
    n.k, n.v, n.ks, n.vs = (back(t).ravel() for t in (g.k, g.v, g.k_scales, g.v_scales))
    for t in range(32):
        for h in range(2):
            for is_k in (True, False):
                if t not in steps and t not in (1, 2, 18, 19):
                    want = c.held(0, t, h, is_k)
                else:
                    y = R.bf16_val(x[t, h * D:(h + 1) * D]).astype(np.float64)
                    want = F.quantize_k(y)[0] if is_k else F.quantize_v(y)[0] * np.float64(F.quantize_v(y)[1])
                np.testing.assert_array_equal(n.held(0, t, h, is_k), want, err_msg=f"token {t} head {h} {is_k}")


ATTN = [  # D, page, kvh, heads, lens, rows, counts, window, sinks
    (128, 64, 4, 20, [1], 1, None, 0, 0),
    (128, 64, 4, 20, [31, 32, 33, 63, 64, 65, 127, 129], 1, None, 0, 0),
    (64, 32, 1, 1, [2, 1, 300], 1, None, 0, 0),
    (256, 128, 2, 6, [500, 17], 1, None, 0, 0),
    (64, 256, 3, 12, [257, 90], 1, None, 0, 0),
    (256, 32, 2, 2, [1000], 1, None, 0, 0),
    (128, 64, 4, 20, [16, 40, 333], 16, None, 0, 0),        # 80 rows to a key head
    (128, 64, 1, 8, [16, 200], 16, None, 0, 0),             # 128 rows
    (256, 64, 1, 5, [70], 13, None, 0, 0),
    (64, 32, 2, 14, [100, 9, 64], 7, [7, 1, 5], 0, 0),      # 49 rows: a group of 4 operands
    (128, 64, 8, 48, [90, 5, 64, 33], 5, [5, 0, 2, 3], 0, 0),
    (128, 32, 2, 2, [4, 2], 4, None, 0, 0),                 # rows at negative positions
    (128, 64, 4, 20, [700, 40, 3], 3, None, 1, 0),          # a window of one token
    (128, 32, 4, 20, [900, 41], 4, None, 65, 4),            # and first tokens
    (64, 64, 1, 64, [333], 3, None, 2 ** 31 - 1, 2 ** 31 - 1),
    (128, 256, 4, 8, [9000, 4097], 1, None, 0, 0),          # many parts
    (128, 128, 1, 4, [20000], 2, None, 0, 0),
    (256, 64, 2, 8, [12000], 2, None, 5000, 64),
]


@pytest.mark.parametrize("case", ATTN)
@pytest.mark.parametrize("ws", [True, False])
def test_attention(case, ws):
    D, page, kvh, heads, lens, rows, counts, window, sinks = case
    print(f"attention fp4 {case} ws={ws}", flush=True)
    rng = np.random.default_rng(0)
    table, pages = table_for(rng, lens, page)
    c = F.Cache4(pages, page, kvh, D, rng)
    offs = None if counts is None else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    total = len(lens) * rows if counts is None else int(offs[-1])
    q = R.bf16_bits(1.5 * rng.standard_normal((total, heads * D)))
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows, None if offs is None else dev(offs))
    # stale places behind the sequences: NaN exponents and scales
    for b, n in enumerate(lens):
        for j in range(n, len(table[b]) * page):
            pg = int(table[b, j // page])
            if pg < 0:
                continue
            for h in range(kvh):
                t, tile = c.at(pg, j % page, h)
                c.ks[tile * D + F.exp_byte(t, np.arange(D // 32), D)] = 255
                c.vs[tile * 32 + t] = np.nan
    g = F.gpu_cache(c, va, dev)
    out = dev(np.full((total + 2, heads * D), SENT))  # rows behind the last sequence
    w = workspace(g, batch, heads) if ws else None
    for _ in range(2):  # the workspace serves the next call
        assert va.attention_paged(g, batch, dev(q), out[:total], window=window, sinks=sinks, workspace=w).ok()
    o, bound = R.attention(c, table, lens, rows, offs, q, heads, D ** -0.5, window, sinks)
    got = back(out)
    check(got, o, bound, lens, rows, offs, case)
    assert np.all(got[total:] == SENT)


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("ws", [True, False])
def test_tokens_that_are_not_finite(rows, ws):
    """A NaN key makes the rows that see it NaN, an infinite value those rows; earlier rows of the same tile are untouched."""
    D, page, kvh, heads, n = 128, 64, 2, 6, 1500
    rng = np.random.default_rng(4)
    for what in ("key", "value"):
        table, pages = table_for(rng, [n], page)
        c = F.Cache4(pages, page, kvh, D, rng)
        pg = int(table[0, (n - 2) // page])
        t, tile = c.at(pg, (n - 2) % page, 1)  # seen by the last two rows
        if what == "key":
            c.ks[tile * D + F.exp_byte(t, 2, D)] = 255
        else:
            c.vs[tile * 32 + t] = np.nan
        g = F.gpu_cache(c, va, dev)
        q = R.bf16_bits(rng.standard_normal((rows, heads * D)))
        batch = va.KVBatch(dev(table), dev(np.array([n], np.int32)), rows)
        out = dev(np.zeros((rows, heads * D), np.uint16))
        assert va.attention_paged(g, batch, dev(q), out, workspace=workspace(g, batch, heads) if ws else None).ok()
        y = R.bf16_val(back(out)).reshape(rows, heads, D)
        o, bound = R.attention(c, table, [n], rows, None, q, heads, D ** -0.5)
        for r in range(rows):
            sees = n - rows + r >= n - 2
            assert np.isnan(y[r, 3:]).all() == sees and not np.isnan(y[r, :3]).any()
            fine = ~np.isnan(y[r])
            assert np.all(np.abs(y[r] - o[r])[fine] <= bound[r][fine])


def test_a_stack_on_a_4_bit_cache():
    from test_gpu_stack_context import SMALL, bits
    from viper_amd.stack import Stack
    s = Stack(torch, **SMALL, context=100, kv_type=va.KVType.FP4, page_size=32, window=40, sinks=3)
    seen, plain = [], s.attend

    def attend(l):
        plain(l)
        seen.append((l, bits(s.q), bits(s.attn)))

    s.attend = attend
    for _ in range(70):
        del seen[:]
        s.step_fused()
    torch.cuda.synchronize()
    for l, q, out in seen:
        c, g = F.Cache4(4, 32, 2, 64), s.kv[l]
        c.k, c.v, c.ks, c.vs = (back(t).ravel() for t in (g.k, g.v, g.k_scales, g.v_scales))
        o, bound = R.attention(c, np.arange(4)[None, :], [70], 1, None, q, 8, 64 ** -0.5, 40, 3)
        check(out, o, bound, [70], 1, None, l)
    assert torch.isfinite(s.logits.float()).all()


@pytest.mark.parametrize("D,kvh,heads", [(64, 1, 3), (128, 4, 20), (256, 2, 6)])
@pytest.mark.parametrize("at", range(8))
def test_one_row_at_every_place_of_an_octet(D, kvh, heads, at):
    """Rows alone in their octet of tokens: at each place their angles are in LDS by themselves (nothing else is written there)."""
    test_append_and_read(D, 64, kvh, heads, [8 * i + at + 1 for i in range(0, 120, 3)], None, 1, 10000.0)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_exponents_of_an_empty_cache_are_tiles(D):
    """k_scales [num_pages, kv_heads, tile, head_dim]: a row's bytes lie in its tile where the header says, and nowhere else."""
    page, kvh, t = 64, 2, 45
    g = va.KVCache.empty(va.KVType.FP4, 3, page, kvh, D)
    assert tuple(g.k_scales.shape) == (3, kvh, 2, D) and bool((g.k_scales == 2).all())
    x = np.zeros((1, kvh, D), np.float32)
    x[0, 1] = 2.0 ** (np.arange(D) // 32 * 3)
    row = dev(R.bf16_bits(x))
    assert va.kv_append(g, va.KVBatch(dev(np.array([[2]], np.int32)), dev(np.array([t + 1], np.int32))), row, row).ok()
    want = np.full((3, kvh, 2, D), 2, np.uint8)
    want[2, 1, t // 32, F.exp_byte(t % 32, np.arange(D // 32), D)] = F.quantize_k(x[0, 1].astype(np.float64))[1]
    np.testing.assert_array_equal(back(g.k_scales), want)
