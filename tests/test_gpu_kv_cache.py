"""kv_append and kv_read against the plain 64-bit implementation: rotation, tile order, int8 codes and scales, what is skipped."""
import numpy as np
import pytest

import decode_ref as R
import viper_amd as va

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SENT = np.uint16(0x4D4D)  # a bf16 value that no row has


def dev(a):
    a = np.ascontiguousarray(a)
    return torch.from_numpy(a.view(np.int16) if a.dtype == np.uint16 else a).to("cuda")


def back(t):
    a = t.cpu().numpy()
    return a.view(np.uint16) if a.dtype == np.int16 else a


def gpu_cache(c):
    return va.KVCache(va.KVType.INT8 if c.i8 else va.KVType.BF16, dev(c.k), dev(c.v), c.page, c.kvh, c.D,
                      dev(c.ks) if c.i8 else None, dev(c.vs) if c.i8 else None)


def step_of(x):
    """bf16 step at |x|: the distance to the next value (float64)."""
    with np.errstate(divide="ignore"):
        return 2.0 ** (np.floor(np.log2(np.maximum(np.abs(x), 1e-30))) - 7)


def table_for(rng, lens, page, spare=2):
    W = max(1, max(-(-int(n) // page) for n in lens))
    pages = sum(-(-int(n) // page) for n in lens) + spare
    ids = rng.permutation(pages)
    t = np.full((len(lens), W), -1, np.int32)
    at = 0
    for b, n in enumerate(lens):
        k = -(-int(n) // page)
        t[b, :k] = ids[at:at + k]
        at += k
    return t, pages


CASES = [  # D, i8, page, kvh, heads, lens, counts (None: uniform rows), rows
    (128, False, 64, 4, 20, [1], None, 1),
    (128, True, 64, 4, 20, [1000, 31, 32, 33], None, 1),
    (64, False, 32, 1, 3, [70, 5], None, 5),
    (64, True, 32, 8, 8, [129, 40, 17], [16, 3, 1], 16),
    (256, False, 128, 2, 2, [300, 128, 127], [7, 0, 9], 9),
    (256, True, 256, 3, 12, [513, 258], [300, 258], 300),
    (128, False, 256, 8, 48, [700], None, 700),
    (128, False, 64, 2, 2, [3, 0, 64], None, 4),          # rows at negative positions
    (128, True, 64, 5, 10, [100003], None, 3),            # a far position
]


@pytest.mark.parametrize("D,i8,page,kvh,heads,lens,counts,rows", CASES)
@pytest.mark.parametrize("theta", [None, 10000.0])
def test_append_and_read(D, i8, page, kvh, heads, lens, counts, rows, theta):
    rng = np.random.default_rng(D * 7 + rows)
    print(f"append D={D} i8={i8} page={page} rows={rows} theta={theta}", flush=True)
    table, pages = table_for(rng, lens, page)
    c = R.Cache(i8, pages, page, kvh, D, rng)
    offs = None if counts is None else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    total = len(lens) * rows if counts is None else int(offs[-1])
    wide = (heads + 2 * kvh) * D + 24  # rows of one projection, some columns behind them
    x = R.bf16_bits(rng.standard_normal((total, wide)) * np.exp(rng.uniform(-3, 3, (total, 1))))
    x[total // 2, heads * D:(heads + 1) * D] = 0  # a row of zeros
    g = gpu_cache(c)
    X = dev(x)
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows, None if offs is None else dev(offs))
    q, k, v = X[:, :heads * D], X[:, heads * D:(heads + kvh) * D], X[:, (heads + kvh) * D:(heads + 2 * kvh) * D]
    qo = dev(np.full((total, heads * D + 8), SENT))
    st = va.kv_append(g, batch, k, v) if theta is None else va.kv_append(g, batch, k, v, q=q, q_out=qo[:, :heads * D], rope_theta=theta)
    assert st.ok(), st
    ko, vo = (dev(np.full((total, kvh, D), SENT)) for _ in range(2))
    assert va.kv_read(g, batch, ko, vo).ok()
    torch.cuda.synchronize()

    got = {n: back(getattr(g, n)) for n in ("k", "v")}
    gks, gvs = (back(g.k_scales), back(g.v_scales)) if i8 else (None, None)
    qo, ko, vo = back(qo), back(ko), back(vo)
    want = {"k": c.k.copy(), "v": c.v.copy()}
    untouched = {"k": np.ones(len(c.k), bool), "v": np.ones(len(c.v), bool)}
    turned = 0
    for b, r, p in R.row_map(lens, rows, offs):
        if p < 0:
            assert np.all(qo[r] == SENT) and np.all(ko[r] == SENT) and np.all(vo[r] == SENT)
            continue
        row = lambda lo, n: R.bf16_val(x[r, lo:lo + n * D]).astype(np.float64).reshape(n, D)
        qr, kr, vr = row(0, heads), row(heads * D, kvh), row((heads + kvh) * D, kvh)
        if theta is not None:
            qr, kr = R.rotate(qr, p, theta), R.rotate(kr, p, theta)
            # the 64-bit value goes through 32 bits to bf16: 2^-24 |x| and half a step, where |x| <= 2^8 steps, so
            # at most step * (1/2 + 2^-16); what the angles lose (1e-9 here) is far below
            d = np.abs(R.bf16_val(qo[r, :heads * D]).reshape(heads, D) - qr)
            assert np.all(d <= step_of(qr) * (0.5 + 2.0 ** -16) + 1e-9)
            assert np.all(qo[r, heads * D:] == SENT)
            turned += 1
        pg, at = int(table[b, p // page]), p % page
        for h in range(kvh):
            for name, val, is_k, sc, out in (("k", kr[h], True, gks, ko), ("v", vr[h], False, gvs, vo)):
                e = c.places(pg, at, h, is_k)
                untouched[name][e] = False
                stored = got[name][e]
                if i8:
                    # the bf16 row that is quantized: the kernel's own rounding of the rotated value
                    bits = R.bf16_bits(val.astype(np.float32))
                    codes, s = R.quantize_row(R.bf16_val(bits))
                    assert sc.ravel()[c.scale_at(pg, at, h)] == s
                    np.testing.assert_array_equal(stored, codes)
                    np.testing.assert_array_equal(out[r, h], R.bf16_bits(codes.astype(np.float32) * s))
                else:
                    np.testing.assert_array_equal(stored, R.bf16_bits(val.astype(np.float32)))
                    np.testing.assert_array_equal(out[r, h], stored)
    for name in ("k", "v"):  # nothing else was written
        np.testing.assert_array_equal(got[name][untouched[name]], want[name][untouched[name]])
    assert theta is None or turned > 0


def test_rotation_in_place_and_far_positions():
    """q rotated into itself; positions up to 2^31 - 1, where 32-bit angles would be meaningless."""
    rng = np.random.default_rng(5)
    D, heads, theta = 128, 2, 500000.0
    lens = np.array([2 ** 31 - 1, 10 ** 6 + 1, 131073], np.int32)  # far past the table: nothing is stored
    c = R.Cache(False, 2, 64, 1, D)
    g = gpu_cache(c)
    x = R.bf16_bits(rng.standard_normal((3, heads * D)))
    kv = dev(R.bf16_bits(rng.standard_normal((3, D))))
    q = dev(x)
    batch = va.KVBatch(dev(np.zeros((3, 2), np.int32)), dev(lens), 1)
    assert va.kv_append(g, batch, kv, kv, q=q, q_out=q, rope_theta=theta).ok()
    got = R.bf16_val(back(q)).reshape(3, heads, D)
    for r in range(3):
        want = R.rotate(R.bf16_val(x[r]).astype(np.float64).reshape(heads, D), int(lens[r]) - 1, theta)
        # angles of 2^31 in 64 bits: off by 2^31 2^-53 and as much again from theta's power
        assert np.all(np.abs(got[r] - want) <= step_of(want) * 0.5 + 8 * 2.0 ** -20)
    assert not np.any(back(g.k)) and not np.any(back(g.v))


def test_bad_pages_store_nothing_and_read_zero():
    rng = np.random.default_rng(6)
    D, kvh, page = 64, 2, 32
    table = np.array([[0, 7, 2], [-1, 3, 2 ** 31 - 1]], np.int32)  # 4 pages in the pool
    lens = np.array([200, 96], np.int32)                            # the first is longer than its table
    for i8 in (False, True):
        c = R.Cache(i8, 4, page, kvh, D, rng)
        g = gpu_cache(c)
        batch = va.KVBatch(dev(table), dev(lens), 200, dev(np.array([0, 200, 296], np.int32)))
        k, v = (dev(R.bf16_bits(rng.standard_normal((296, kvh * D)))) for _ in range(2))
        assert va.kv_append(g, batch, k, v).ok()
        ko, vo = (dev(np.full((296, kvh, D), SENT)) for _ in range(2))
        assert va.kv_read(g, batch, ko, vo).ok()
        good = [p // 32 in (0, 2) for p in range(200)] + [p // 32 == 1 for p in range(96)]
        for out, src in ((back(ko), back(k)), (back(vo), back(v))):
            assert not np.any(out[~np.array(good)])
            if not i8:  # page 2 is named twice by the table: the same token of two positions is not
                np.testing.assert_array_equal(out[np.array(good)], src.reshape(296, kvh, D)[np.array(good)])
        # page 1 is nobody's
        for pool, before in ((back(g.k), c.k), (back(g.v), c.v)):
            n = kvh * page * D
            np.testing.assert_array_equal(pool[n:2 * n], before[n:2 * n])


def test_offsets_that_do_not_fit_leave_everything_alone():
    c = R.Cache(False, 4, 32, 1, 64)
    x = dev(R.bf16_bits(np.ones((6, 64), np.float32)))
    for offs in ([0, 7], [-1, 3], [4, 2], [0, 5]):
        g = gpu_cache(c)
        batch = va.KVBatch(dev(np.array([[0, 1]], np.int32)), dev(np.array([40], np.int32)), 4, dev(np.array(offs, np.int32)))
        assert va.kv_append(g, batch, x, x).ok()
        ko, vo = (dev(np.full((6, 1, 64), SENT)) for _ in range(2))
        assert va.kv_read(g, batch, ko, vo).ok()
        assert not np.any(back(g.k)) and not np.any(back(g.v)) and np.all(back(ko) == SENT) and np.all(back(vo) == SENT)


def test_int8_rows_that_are_not_finite_read_back_as_nan():
    rng = np.random.default_rng(8)
    D = 128
    x = R.bf16_bits(rng.standard_normal((3, D)))
    x[0, 5], x[1, 127] = 0x7FC0, 0x7F80
    c = R.Cache(True, 1, 32, 1, D)
    g = gpu_cache(c)
    batch = va.KVBatch(dev(np.zeros((1, 1), np.int32)), dev(np.array([3], np.int32)), 3)
    assert va.kv_append(g, batch, dev(x), dev(x)).ok()
    ko, vo = (dev(np.zeros((3, 1, D), np.uint16)) for _ in range(2))
    assert va.kv_read(g, batch, ko, vo).ok()
    for out in (R.bf16_val(back(ko)), R.bf16_val(back(vo))):
        assert np.all(np.isnan(out[:2])) and np.all(np.isfinite(out[2]))


def test_large_pool_offsets_past_32_bits():
    """Pages whose bytes lie past 2^32 (and elements past 2^31) in each pool."""
    D, kvh, page = 128, 8, 256
    pages = 10000  # 512 KiB each: 5.2 GB a pool
    g = va.KVCache.empty(va.KVType.BF16, pages, page, kvh, D)
    rng = np.random.default_rng(9)
    table = np.array([[pages - 1, 8191, 8192, 3]], np.int32)
    n = 4 * page
    k, v = (R.bf16_bits(rng.standard_normal((n, kvh * D))) for _ in range(2))
    batch = va.KVBatch(dev(table), dev(np.array([n], np.int32)), n)
    assert va.kv_append(g, batch, dev(k), dev(v)).ok()
    ko, vo = (torch.zeros((n, kvh, D), dtype=torch.int16, device="cuda") for _ in range(2))
    assert va.kv_read(g, batch, ko, vo).ok()
    np.testing.assert_array_equal(back(ko).reshape(n, -1), k)
    np.testing.assert_array_equal(back(vo).reshape(n, -1), v)
    q = R.bf16_bits(rng.standard_normal((1, kvh * D)))
    out = dev(np.zeros((1, kvh * D), np.uint16))
    one = va.KVBatch(dev(table), dev(np.array([n], np.int32)), 1)
    assert va.attention_paged(g, one, dev(q), out).ok()
    small = R.Cache(False, 4, page, kvh, D)
    elems = kvh * page * D
    kc, vc = g.k.view(torch.int16).view(pages, -1), g.v.view(torch.int16).view(pages, -1)
    for i, pg in enumerate(table[0]):
        small.k[i * elems:(i + 1) * elems] = back(kc[int(pg)])
        small.v[i * elems:(i + 1) * elems] = back(vc[int(pg)])
    o, bound = R.attention(small, np.arange(4)[None, :], [n], 1, None, q, kvh, D ** -0.5)
    assert np.all(np.abs(R.bf16_val(back(out)).reshape(kvh, D) - o[0]) <= bound[0])
