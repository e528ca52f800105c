"""kv_page_bounds, select_pages and attention_selected against the plain implementations of pages_ref, alone and as a decode step uses
them together."""
import numpy as np
import pytest

import decode_ref as R
import fp4_ref as F
import pages_ref as P
import viper_amd as va
from test_gpu_attention import check
from test_gpu_kv_cache import SENT, back, dev, table_for

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

KINDS = ("bf16", "int8", "fp4")


def ws_of(n):
    return torch.zeros((max(16, n),), dtype=torch.uint8, device="cuda")


def offsets(counts):
    return None if counts is None else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)


def setup(kind, D, page, kvh, lens, rows, counts, seed=0):
    rng = np.random.default_rng(seed)
    table, pages = table_for(rng, [max(n, 0) for n in lens], page)
    c = F.make_cache(kind, pages, page, kvh, D, rng)
    offs = offsets(counts)
    total = len(lens) * rows if counts is None else int(offs[-1])
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows, None if offs is None else dev(offs), total)
    return rng, c, table, offs, total, batch, F.gpu_cache(c, va, dev)


BOUNDS = [  # D, page, kvh, lens, rows, counts
    (128, 64, 4, [1], 1, None),
    (128, 64, 4, [64, 65, 63, 31, 32, 33], 1, None),
    (64, 32, 3, [100, 7, 0], 5, [5, 3, 0]),
    (256, 256, 2, [700, 257], 300, None),
    (128, 128, 1, [1000, 4], 1000, [990, 4]),
    (64, 256, 5, [3, 500], 4, None),           # rows at negative positions
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,page,kvh,lens,rows,counts", BOUNDS)
def test_bounds(kind, D, page, kvh, lens, rows, counts):
    print("bounds", kind, D, page, kvh, lens, rows, counts, flush=True)
    rng, c, table, offs, total, batch, g = setup(kind, D, page, kvh, lens, rows, counts)
    before = R.bf16_bits(rng.standard_normal((c.pages, kvh, 2, D)))
    out = dev(before)
    assert va.kv_page_bounds(g, batch, out).ok()
    want = R.bf16_val(before).astype(np.float64)
    P.bounds(c, table, lens, rows, offs, want)
    np.testing.assert_array_equal(R.bf16_val(back(out)), want)


def test_bounds_of_keys_that_are_not_finite():
    D, page = 128, 32
    rng = np.random.default_rng(1)
    c = R.Cache(False, 2, page, 1, D, rng)
    for t, d, v in ((3, 7, np.nan), (4, 8, np.inf), (5, 9, -np.inf), (6, 10, -np.nan), (31, 11, np.nan), (7, 12, 0.0), (8, 12, -0.0)):
        c.k[c.places(1, t, 0, True)[d]] = R.bf16_bits(np.array([v], np.float32))[0]
    c.k[c.places(1, 6, 0, True)[10]] = 0xFFFF
    g = F.gpu_cache(c, va, dev)
    out = dev(np.zeros((2, 1, 2, D), np.uint16))
    assert va.kv_page_bounds(g, va.KVBatch(dev(np.array([[1]], np.int32)), dev(np.array([20], np.int32)), 20), out).ok()
    want = np.zeros((2, 1, 2, D))
    P.bounds(c, [[1]], [20], 20, None, want)
    np.testing.assert_array_equal(R.bf16_val(back(out)), want)
    assert np.isnan(want[1, 0, :, 7]).all() and want[1, 0, 1, 8] == np.inf and np.isfinite(want[1, 0, :, 11]).all()


def test_bounds_past_the_table_and_of_missing_pages():
    D, page = 64, 32
    c = R.Cache(True, 3, page, 2, D, np.random.default_rng(1))
    g = F.gpu_cache(c, va, dev)
    table, lens = np.array([[2, 7, -5], [0, 1, 2]], np.int32), [96, 2 ** 31 - 1]
    out = dev(np.full((3, 2, 2, D), SENT))
    offs = np.array([0, 96, 99], np.int32)
    assert va.kv_page_bounds(g, va.KVBatch(dev(table), dev(np.array(lens, np.int32)), 96, dev(offs), 99), out).ok()
    want = np.broadcast_to(R.bf16_val(SENT).astype(np.float64), (3, 2, 2, D)).copy()
    P.bounds(c, table, [96], 96, None, want)
    np.testing.assert_array_equal(R.bf16_val(back(out)), want)
    # offsets that do not fit leave all as it was
    bad = va.KVBatch(dev(table), dev(np.array([50, 50], np.int32)), 2, dev(np.array([1, 5, 2], np.int32)), 2)
    assert va.kv_page_bounds(g, bad, out).ok()
    np.testing.assert_array_equal(R.bf16_val(back(out)), want)


SELECT = [  # D, page, kvh, heads, lens, rows, counts, first, last, count
    (128, 64, 4, 20, [1], 1, None, 1, 1, 4),
    (128, 64, 4, 20, [5000, 640, 641, 63, 64, 65], 1, None, 1, 2, 8),
    (64, 32, 2, 2, [1000, 33, 0], 3, [3, 1, 0], 0, 1, 5),
    (64, 32, 1, 8, [3000, 2], 4, None, 4, 5, 9),                  # nothing but the first and last; a row at a negative position
    (256, 32, 1, 64, [900], 16, None, 1, 1, 17),                  # queries in several turns
    (256, 256, 2, 6, [20000, 4097], 2, None, 2, 1, 7),
    (128, 32, 8, 48, [2000, 1500, 31], 5, [5, 2, 4], 1, 1, 40),
    (128, 32, 1, 1, [4096 * 32 + 5], 1, None, 1, 1, 1000),        # more pages than a workgroup holds
    (64, 32, 2, 4, [100000, 290001], 2, None, 3, 2, 2900),        # and many of them listed
    (128, 64, 2, 4, [1000], 1, None, 1, 1, 200),                  # more entries than pages
]


@pytest.mark.parametrize("D,page,kvh,heads,lens,rows,counts,first,last,count", SELECT)
def test_select(D, page, kvh, heads, lens, rows, counts, first, last, count):
    print("select", D, page, kvh, heads, lens, rows, counts, first, last, count, flush=True)
    rng = np.random.default_rng(3)
    table, pages = table_for(rng, lens, page)
    offs = offsets(counts)
    total = len(lens) * rows if counts is None else int(offs[-1])
    pool = torch.zeros((pages, kvh, page // 32, 16 * D), dtype=torch.uint8, device="cuda")
    g = va.KVCache(va.KVType.FP4, pool, pool.clone(), page, kvh, D, torch.zeros((pages, kvh, page, D // 32), dtype=torch.uint8, device="cuda"),
                   torch.zeros((pages, kvh, page), device="cuda"))
    near = rng.standard_normal((pages, kvh, 1, D)) + np.array([-1.0, 1.0])[:, None] * rng.uniform(0.2, 1.5, (pages, kvh, 1, D))
    near = R.bf16_bits(near)
    if pages > 8:  # pages alike: of equal scores the first
        near[pages // 2:pages // 2 + 3] = near[3]
        near[5::7] = near[5]
    q = R.bf16_bits(rng.standard_normal((total, heads * D)))
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows, None if offs is None else dev(offs), total)
    sel = dev(np.full((total + 1, kvh, count), 77, np.int32))
    ws = torch.full((va.select_workspace_bytes(g, batch, heads, count),), 0xab, dtype=torch.uint8, device="cuda")
    for _ in range(2):
        assert va.select_pages(g, batch, dev(q), dev(near), sel[:total], first=first, last=last, workspace=ws).ok()
    got, G = back(sel), heads // kvh
    f = R.bf16_val(near).astype(np.float64)
    for b, r, p in R.row_map(lens, rows, offs):
        x = R.bf16_val(q[r]).astype(np.float64).reshape(kvh, G, D)
        for h in range(kvh):
            want = P.select(x[h], f[:, h], table[b], pages, page, p, first, last, count)
            assert got[r, h].tolist() == want, (b, r, p, h)
    assert np.all(got[total:] == 77)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("alike", [2, 9, 60, 300])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -110, 2.0 ** 100])
def test_select_near_the_border(D, alike, scale):
    """Pages at the border whose scores differ by a part in 2^20 and less, or not at all, amid others far from it."""
    page, kvh, heads, pages = 32, 2, 6, 700
    rng = np.random.default_rng(alike + D)
    table = rng.permutation(pages).astype(np.int32)[None, :]
    near = np.sort(rng.standard_normal((pages, kvh, 2, D)), 2)
    order = rng.permutation(pages)
    near[order[:100]] += 1.5                                        # in
    like = order[100:100 + alike]
    near[like] = near[like[0]] + np.array([0.5, 0.7])[:, None]      # at the border
    q = rng.standard_normal((3, heads, D))
    q[:, :, 5] = 2.0 ** -14
    near[like, :, 1, 5] += rng.integers(0, 4, (alike, kvh)) * 2.0 ** -7
    q, near = R.bf16_bits(q.reshape(3, heads * D)), R.bf16_bits(near * scale)
    g = va.KVCache.empty(va.KVType.BF16, pages, page, kvh, D)
    n = pages * page - 7
    batch = va.KVBatch(dev(table), dev(np.array([n], np.int32)), 3)
    f = R.bf16_val(near).astype(np.float64)
    for count in (101, 102 + alike // 2, 101 + alike, 400):
        sel = dev(np.zeros((3, kvh, count), np.int32))
        ws = ws_of(va.select_workspace_bytes(g, batch, heads, count))
        for _ in range(2):
            assert va.select_pages(g, batch, dev(q), dev(near), sel, first=0, last=1, workspace=ws).ok()
        got = back(sel)
        for r in range(3):
            x = R.bf16_val(q[r]).astype(np.float64).reshape(kvh, heads // kvh, D)
            for h in range(kvh):
                assert got[r, h].tolist() == P.select(x[h], f[:, h], table[0], pages, page, n - 3 + r, 0, 1, count), (count, r, h)


def test_select_among_missing_pages_and_scores_that_are_not_finite():
    D, page, kvh, pages, n = 64, 32, 1, 40, 30
    rng = np.random.default_rng(5)
    table = rng.permutation(pages)[:n].astype(np.int32)[None, :]
    table[0, [0, 4, 9, 28]] = [-1, -7, pages, 2 ** 31 - 1]
    near = np.sort(rng.standard_normal((pages, kvh, 2, D)), 2)
    near[table[0, 7], 0, 1, 3] = np.inf
    near[table[0, 8], 0, :, 9] = np.nan
    near[table[0, 11], 0] = -np.inf      # q_d < 0 with -inf: +inf; mixed signs: NaN
    near = R.bf16_bits(near)
    g = va.KVCache.empty(va.KVType.BF16, pages, page, kvh, D)
    q = R.bf16_bits(rng.standard_normal((2, 3 * D)))
    q[1] = 0                              # all scores are 0, or NaN
    for lens in ([n * page], [n * page + 1000], [5]):  # the second past the table
        batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), 2)
        for first, last, count in ((0, 1, 6), (2, 3, 6), (1, 1, 29), (1, 1, 64)):
            sel = dev(np.zeros((2, kvh, count), np.int32))
            ws = ws_of(va.select_workspace_bytes(g, batch, 3, count))
            assert va.select_pages(g, batch, dev(q), dev(near), sel, first=first, last=last, workspace=ws).ok()
            got = back(sel)
            for r in range(2):
                want = P.select(R.bf16_val(q[r]).astype(np.float64).reshape(3, D), R.bf16_val(near).astype(np.float64)[:, 0], table[0], pages,
                                page, lens[0] - 2 + r, first, last, count)
                assert got[r, 0].tolist() == want, (lens, first, last, count, r)


ATTN = [  # D, page, kvh, heads, lens, rows, counts, count
    (128, 64, 4, 20, [1], 1, None, 3),
    (128, 64, 4, 20, [3000, 640, 63, 64, 65], 1, None, 8),
    (64, 32, 1, 1, [2, 700], 3, None, 5),
    (256, 128, 2, 6, [2000, 17], 2, None, 4),
    (64, 256, 3, 12, [2570, 900], 1, None, 6),
    (128, 64, 1, 64, [700], 3, None, 7),                 # 64 heads to a key head
    (256, 64, 1, 33, [700], 2, None, 7),                 # two groups of them
    (128, 32, 8, 48, [900, 5, 640, 33], 5, [5, 0, 2, 3], 9),
    (128, 32, 2, 2, [4, 2, 100], 4, None, 3),            # rows at negative positions
    (128, 256, 2, 10, [30000], 1, None, 64),             # many parts
    (64, 32, 2, 2, [20000], 16, None, 300),
]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case", ATTN)
def test_attention_selected(kind, case):
    D, page, kvh, heads, lens, rows, counts, count = case
    print("attention over lists", kind, case, flush=True)
    rng, c, table, offs, total, batch, g = setup(kind, D, page, kvh, lens, rows, counts)
    q = R.bf16_bits(1.5 * rng.standard_normal((total, heads * D)))
    lists = np.full((total, kvh, count), -1, np.int32)
    for i, (b, r, p) in enumerate(R.row_map(lens, rows, offs)):
        n = max(p, 0) // page + 1
        for h in range(kvh):
            k = min(count, n)
            pick = rng.permutation(n)[:k]
            pick[rng.integers(k)] = n - 1 if n - 1 not in pick else pick[0]  # (mostly distinct; twice counts twice)
            lists[r, h, rng.permutation(count)[:k]] = pick                 # in any order, none between them
            if i % 3 == 1:
                lists[r, h, lists[r, h] == -1] = n + 3                     # past the row's page: none
    o, bound = P.attention(c, table, lens, rows, offs, q, heads, D ** -0.5, lists)
    n = va.attention_selected_workspace_bytes(g, batch, heads, count)
    for w in (ws_of(n), None):
        out = dev(np.full((total + 2, heads * D), SENT))
        for _ in range(2):
            assert va.attention_selected(g, batch, dev(q), dev(lists), out[:total], workspace=w).ok()
        got = back(out)
        check(got, o, bound, lens, rows, offs, case)
        assert np.all(got[total:] == SENT)


@pytest.mark.parametrize("kind", KINDS)
def test_lists_that_are_empty_pages_that_are_missing_and_entries_out_of_range(kind):
    D, page, kvh, heads, lens = 128, 64, 2, 6, [500, 64 * 40 + 9, 300]
    rng, c, table, offs, total, batch, g = setup(kind, D, page, kvh, lens, 1, None)
    q = R.bf16_bits(rng.standard_normal((3, heads * D)))
    table[2, 1] = -1
    table[0, 3] = c.pages
    short = va.KVBatch(dev(table), dev(np.array([500, 64 * 60, 300], np.int32)), 1)  # the second is past its table
    count = 33
    for entries in ([], [-1, -2 ** 31], [2 ** 31 - 1, 2 ** 26, 8], [0, 2, -5], [1, 0], [3], [2 ** 31 - 1] * 30 + [0, 1, 2]):
        lists = np.full((3, kvh, count), -1, np.int32)
        lists[:, :, :len(entries)] = entries
        lists[:, 1] = lists[:, 1, ::-1]
        for bt, ln in ((va.KVBatch(dev(table), dev(np.array(lens, np.int32)), 1), lens), (short, [500, 64 * 60, 300])):
            o, bound = P.attention(c, table, ln, 1, None, q, heads, 0.07, lists)
            n = va.attention_selected_workspace_bytes(g, bt, heads, count)
            for w in (ws_of(n), None):
                out = dev(np.full((3, heads * D), SENT))
                assert va.attention_selected(g, bt, dev(q), dev(lists), out, scale=0.07, workspace=w).ok()
                check(back(out), o, bound, ln, 1, None, (entries, ln))


@pytest.mark.parametrize("ws", [True, False])
def test_values_that_are_not_finite_reach_only_rows_that_list_them(ws):
    """Infinite and NaN values and keys in a bf16 cache: rows whose list lacks their page, or that come before them, are untouched."""
    D, page, kvh, heads, n = 128, 64, 1, 3, 64 * 9 + 40
    rng = np.random.default_rng(8)
    table, pages = table_for(rng, [n], page)
    c = R.Cache(False, pages, page, kvh, D, rng)
    put = lambda j, d, v, k: (c.k if k else c.v).__setitem__(c.places(int(table[0, j // page]), j % page, 0, k)[d], R.bf16_bits(np.float32([v]))[0])
    put(64 * 4 + 5, 3, np.inf, False)
    put(64 * 5 + 6, 4, np.nan, False)
    put(64 * 6 + 7, 5, np.nan, True)
    put(n - 2, 6, -np.inf, False)       # seen by the last two rows
    put(64 * 7, 7, 3e38, False), put(64 * 7 + 1, 7, 3e38, False)
    put(n + 2, 8, np.nan, False), put(n + 2, 8, np.nan, True)  # behind the sequence
    g = F.gpu_cache(c, va, dev)
    batch = va.KVBatch(dev(table), dev(np.array([n], np.int32)), 4)
    q = R.bf16_bits(rng.standard_normal((4, heads * D)))
    for entries in ([0, 1, 2, 3], [4, 0, 1], [0, 5], [6, 2], [0, 9], [7, 8], [0, 1, 2, 3, 4, 5, 6, 7, 8, 9]):
        lists = np.full((4, 1, 12), -1, np.int32)
        lists[:, 0, 12 - len(entries):] = entries
        o, bound = P.attention(c, table, [n], 4, None, q, heads, D ** -0.5, lists)
        w = ws_of(va.attention_selected_workspace_bytes(g, batch, heads, 12)) if ws else None
        out = dev(np.full((4, heads * D), SENT))
        assert va.attention_selected(g, batch, dev(q), dev(lists), out, workspace=w).ok()
        check(back(out), o, bound, [n], 4, None, entries)


@pytest.mark.parametrize("kind", KINDS)
def test_all_pages_listed_is_attention_paged(kind):
    D, page, kvh, heads, lens, rows = 128, 64, 2, 10, [1500, 70], 3
    rng, c, table, offs, total, batch, g = setup(kind, D, page, kvh, lens, rows, None)
    q = dev(R.bf16_bits(rng.standard_normal((total, heads * D))))
    bounds = torch.zeros((c.pages, kvh, 2, D), dtype=torch.int16, device="cuda")
    sel = torch.zeros((total, kvh, 24), dtype=torch.int32, device="cuda")
    a, b = (dev(np.zeros((total, heads * D), np.uint16)) for _ in range(2))
    assert va.kv_page_bounds(g, batch, bounds).ok()
    assert va.select_pages(g, batch, q, bounds, sel, workspace=ws_of(va.select_workspace_bytes(g, batch, heads, 24))).ok()
    assert va.attention_selected(g, batch, q, sel, a).ok() and va.attention_paged(g, batch, q, b).ok()
    va_, vb = R.bf16_val(back(a)).astype(np.float64), R.bf16_val(back(b)).astype(np.float64)
    # two roundings of the same value and two sums of it, each as far from it as the other bound says
    _, bound = R.attention(c, table, lens, rows, None, back(q), heads, D ** -0.5)
    for b_, r, p in R.row_map(lens, rows, None):
        assert np.all(np.abs(va_[r] - vb[r]).reshape(heads, D) <= 2 * bound[r])
    for r in range(total):
        n = (lens[r // rows] - rows + r % rows) // page + 1
        assert sel[r, 0].tolist() == list(range(n)) + [-1] * (24 - n)


@pytest.mark.parametrize("kind", KINDS)
def test_a_decode_step_captured_and_replayed(kind):
    """append, bounds, selection and attention of one growing sequence in a graph: every replay equals the eager calls on a cache of
    their own, while eager work on the same workspaces' shapes runs between the replays."""
    D, page, kvh, heads, count, n0 = 64, 32, 2, 8, 4, 250
    rng = np.random.default_rng(9)
    tokens = dev(R.bf16_bits(rng.standard_normal((n0 + 40, (heads + 2 * kvh) * D))))

    class Side:
        def __init__(self):
            self.g = va.KVCache.empty(va.KVType[kind.upper()], 12, page, kvh, D)
            self.table = torch.arange(11, -1, -1, dtype=torch.int32, device="cuda").view(1, 12).contiguous()
            self.len = torch.zeros((1,), dtype=torch.int32, device="cuda")
            self.one = va.KVBatch(self.table, self.len)
            self.row = torch.zeros((1, tokens.shape[1]), dtype=torch.int16, device="cuda")
            self.bounds = torch.zeros((12, kvh, 2, D), dtype=torch.int16, device="cuda")
            self.sel = torch.zeros((1, kvh, count), dtype=torch.int32, device="cuda")
            self.out = torch.zeros((1, heads * D), dtype=torch.int16, device="cuda")
            self.ws = [ws_of(va.select_workspace_bytes(self.g, self.one, heads, count)),
                       ws_of(va.attention_selected_workspace_bytes(self.g, self.one, heads, count))]
            # the prompt
            self.len.fill_(n0)
            rows = tokens[:n0]
            first = va.KVBatch(self.table, self.len, n0)
            kv = rows[:, heads * D:(heads + kvh) * D], rows[:, (heads + kvh) * D:]
            assert va.kv_append(self.g, first, *kv).ok() and va.kv_page_bounds(self.g, first, self.bounds).ok()

        def step(self):
            self.len.add_(1)
            q, k, v = self.row[:, :heads * D], self.row[:, heads * D:(heads + kvh) * D], self.row[:, (heads + kvh) * D:]
            for st in (va.kv_append(self.g, self.one, k, v, q=q, q_out=q, rope_theta=1e4),
                       va.kv_page_bounds(self.g, self.one, self.bounds),
                       va.select_pages(self.g, self.one, q, self.bounds, self.sel, workspace=self.ws[0]),
                       va.attention_selected(self.g, self.one, q, self.sel, self.out, workspace=self.ws[1])):
                assert st.ok(), st

    a, b = Side(), Side()
    a.row.copy_(tokens[n0:n0 + 1]), b.row.copy_(tokens[n0:n0 + 1])
    a.step(), b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for i in range(1, 36):
        for s in (a, b):
            s.row.copy_(tokens[n0 + i:n0 + i + 1])
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert a.len.item() == b.len.item() == n0 + 1 + i
        assert torch.equal(a.sel, b.sel) and torch.equal(a.out, b.out) and torch.equal(a.bounds, b.bounds)
        assert a.sel[0, 0, 0].item() == 0 and (n0 + i) // page in a.sel[0, 1].tolist()
    # the eager result against the plain one, over what the cache holds
    c = F.Cache4(12, page, kvh, D) if kind == "fp4" else R.Cache(kind == "int8", 12, page, kvh, D)
    c.k, c.v = (back(t if kind != "bf16" else t.view(torch.int16)).ravel() for t in (b.g.k, b.g.v))
    if kind != "bf16":
        c.ks, c.vs = back(b.g.k_scales).ravel(), back(b.g.v_scales).ravel()
    table, n = back(b.table), b.len.item()
    near = np.zeros((12, kvh, 2, D))
    P.bounds(c, table, [n], n, None, near)
    np.testing.assert_array_equal(R.bf16_val(back(b.bounds)), near)
    q = back(b.row)[:, :heads * D]
    x = R.bf16_val(q[0]).astype(np.float64).reshape(kvh, heads // kvh, D)
    lists = [[P.select(x[h], near[:, h], table[0], 12, page, n - 1, 1, 1, count) for h in range(kvh)]]
    assert b.sel.tolist() == lists
    o, bound = P.attention(c, table, [n], 1, None, q, heads, D ** -0.5, lists)
    check(back(b.out), o, bound, [n], 1, None)


def test_arguments():
    g = va.KVCache.empty(va.KVType.FP4, 4, 64, 2, 128)
    batch = va.KVBatch(torch.zeros((2, 2), dtype=torch.int32, device="cuda"), torch.ones((2,), dtype=torch.int32, device="cuda"))
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")
    q, near, sel, out, ws = bf(2, 8 * 128), bf(4, 2, 2, 128), torch.zeros((2, 2, 4), dtype=torch.int32, device="cuda"), bf(2, 8 * 128), ws_of(1 << 16)
    pick = lambda q=q, near=near, sel=sel, **kw: va.select_pages(g, batch, q, near, sel, **{**dict(workspace=ws), **kw})
    look = lambda q=q, sel=sel, out=out, **kw: va.attention_selected(g, batch, q, sel, out, **kw)
    assert pick().ok() and look().ok() and va.kv_page_bounds(g, batch, near).ok()
    mism, inval = va.StatusCode.SHAPE_MISMATCH, va.StatusCode.INVALID_ARGUMENT
    for st in (pick(sel=sel[:1]), pick(sel=sel.transpose(1, 2)), pick(sel=sel[..., :0]), pick(sel=sel.view(-1)), pick(near=bf(4, 2, 128, 2)),
               pick(q=bf(2, 100)), pick(q=bf(3, 1024)), look(sel=sel[:, :1]), look(sel=sel.view(2, -1)), look(q=bf(2, 100), out=bf(2, 100)),
               look(out=bf(1, 1024)), va.kv_page_bounds(g, batch, bf(4, 2, 128, 2)), va.kv_page_bounds(g, batch, bf(3, 2, 2, 128))):
        assert st.code == mism, st
    for st in (pick(first=1 << 32), pick(last=(1 << 32) + 1), pick(first=4), pick(last=0), pick(workspace=None), pick(workspace=ws[:16]),
               look(out=q), look(scale=float("nan"))):
        assert st.code == inval, st
    for f in (lambda: pick(sel=sel.float()), lambda: pick(near=near.half()), lambda: pick(sel=sel.cpu()), lambda: look(sel=sel.long()),
              lambda: va.kv_page_bounds(g, batch, near.float()), lambda: pick(sel=torch.zeros((2, 4, 2), dtype=torch.int32, device="cuda").transpose(1, 2))):
        with pytest.raises(ValueError):
            f()
    # ragged batches whose number of rows the row tensors tell
    some = va.KVBatch(batch.block_table, batch.seq_lens, 3, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"))
    assert va.kv_page_bounds(g, some, near).ok()
    assert va.select_pages(g, some, q, near, sel, workspace=ws_of(va.select_workspace_bytes(g, some, 8, 4))).ok()


@pytest.mark.parametrize("given", [False, True])
def test_bounds_where_rows_begin_past_the_first(given):
    """Row tensors with rows before the first sequence's: the rows count as kv_append takes them, whether the batch says how many
    the tensors hold or not."""
    D, page, kvh, lens, offs = 64, 32, 2, [40, 7], np.array([5, 6, 8], np.int32)
    rng = np.random.default_rng(2)
    table, pages = table_for(rng, lens, page)
    c = F.make_cache("int8", pages, page, kvh, D, rng)
    g = F.gpu_cache(c, va, dev)
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), 2, dev(offs), 8 if given else None)
    rows = dev(R.bf16_bits(rng.standard_normal((8, kvh * D))))
    assert va.kv_append(g, batch, rows, rows).ok()
    c.k, c.ks = back(g.k).ravel(), back(g.k_scales).ravel()
    out = dev(np.full((pages, kvh, 2, D), SENT))
    assert va.kv_page_bounds(g, batch, out).ok()
    want = np.broadcast_to(R.bf16_val(SENT).astype(np.float64), (pages, kvh, 2, D)).copy()
    P.bounds(c, table, lens, 2, offs, want)
    np.testing.assert_array_equal(R.bf16_val(back(out)), want)
    assert np.any(want != R.bf16_val(SENT))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("page", [32, 128])
@pytest.mark.parametrize("kind", ["int8", "fp4"])
def test_bounds_of_scales_that_are_not_finite(kind, page, D):
    """A block of keys that is not finite (FP4: exponent 255) makes its 32 dimensions' bounds NaN, a scale of NaN or an infinity
    (int8) what kv_read makes of it; places past the sequence hold anything."""
    n, kvh = 2 * page + 21, 2
    rng = np.random.default_rng(D + page)
    c = F.make_cache(kind, 4, page, kvh, D, rng)
    table = np.array([[2, 0, 3]], np.int32)
    for t, head, block in ((5, 0, 0), (page + 3, 1, D // 32 - 1), (page + 9, 0, 1), (2 * page + 20, 1, 0)):
        tile = (int(table[0, t // page]) * kvh + head) * (page // 32) + t % page // 32
        if kind == "fp4":
            c.ks[tile * D + F.exp_byte(t % 32, block, D)] = 255
        else:
            c.ks[tile * 32 + t % 32] = np.nan if block == 0 else np.inf
    past = 2 * page + 21
    tile = (3 * kvh + 0) * (page // 32) + past % page // 32
    if kind == "fp4":
        c.ks[tile * D + F.exp_byte(past % 32, np.arange(D // 32), D)] = 255
    else:
        c.ks[tile * 32 + past % 32] = np.nan
    g = F.gpu_cache(c, va, dev)
    out = dev(np.full((4, kvh, 2, D), SENT))
    assert va.kv_page_bounds(g, va.KVBatch(dev(table), dev(np.array([n], np.int32)), n), out).ok()
    want = np.broadcast_to(R.bf16_val(SENT).astype(np.float64), (4, kvh, 2, D)).copy()
    with np.errstate(all="ignore"):
        P.bounds(c, table, [n], n, None, want)
    np.testing.assert_array_equal(R.bf16_val(back(out)), want)
    assert np.isnan(want[2, 0]).any() and np.isnan(want[3, 1]).any() and np.isfinite(want[3, 0]).all()
    if kind == "fp4":
        assert np.isnan(want[2, 0, :, :32]).all() and np.isfinite(want[2, 0, :, 32:]).all()
