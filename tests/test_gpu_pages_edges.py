"""The ends of the ranges of the 4-bit cache and of attention over selected pages: many sequences of unequal lengths, pools past 4 GiB, other
streams, several batches through one workspace, large vocabularies of pages."""
import numpy as np
import pytest

import decode_ref as R
import fp4_ref as F
import pages_ref as P
import viper_amd as va
from test_gpu_attention import check, workspace
from test_gpu_kv_cache import SENT, back, dev, table_for
from test_gpu_page_select import offsets, ws_of

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("B", [2, 3, 33, 64, 65])
@pytest.mark.parametrize("counts", [False, True])
def test_many_sequences_of_unequal_lengths(B, counts):
    """Parts are shared out by lengths up to 64 sequences; empty sequences and ones without rows among them, one much longer."""
    D, page, kvh, heads, rows = 64, 32, 2, 4, 3
    rng = np.random.default_rng(B)
    lens = rng.integers(rows, 400, B)
    lens[B // 2] = 6000
    lens[0] = 0 if B > 3 else lens[0]
    lens[-1] = rows
    n = rng.integers(0, rows + 1, B) if counts else None
    table, pages = table_for(rng, lens, page)
    c = F.Cache4(pages, page, kvh, D, rng)
    g, offs = F.gpu_cache(c, va, dev), offsets(n)
    total = B * rows if offs is None else int(offs[-1])
    q = R.bf16_bits(1.5 * rng.standard_normal((total, heads * D)))
    batch = va.KVBatch(dev(table), dev(lens.astype(np.int32)), rows, None if offs is None else dev(offs), total)
    w = workspace(g, batch, heads)
    o, bound = R.attention(c, table, lens, rows, offs, q, heads, D ** -0.5)
    for ws in (w, w, None):
        out = dev(np.full((total + 1, heads * D), SENT))
        assert va.attention_paged(g, batch, dev(q), out[:total], workspace=ws).ok()
        check(back(out), o, bound, lens, rows, offs, B)
        assert np.all(back(out)[total:] == SENT)


def test_lengths_change_under_one_plan():
    """The same batch at other lengths (a captured call's replays): longer, past the table, negative, empty."""
    D, page, kvh, heads, B = 128, 64, 1, 8, 5
    rng = np.random.default_rng(3)
    table, pages = table_for(rng, [1280] * B, page)
    c = F.Cache4(pages, page, kvh, D, rng)
    g = F.gpu_cache(c, va, dev)
    q = R.bf16_bits(rng.standard_normal((B, heads * D)))
    lens = torch.zeros((B,), dtype=torch.int32, device="cuda")
    batch, out = va.KVBatch(dev(table), lens), dev(np.zeros((B, heads * D), np.uint16))
    w, gq = workspace(g, batch, heads), dev(q)
    assert va.attention_paged(g, batch, gq, out, workspace=w).ok()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert va.attention_paged(g, batch, gq, out, workspace=w).ok()
    for now in ([1280] * B, [1, 1280, 3, 2000, 700], [0, 0, 1, 0, 0], [-5, 64, 65, 2 ** 31 - 1, 1280], [33] * B):
        lens.copy_(dev(np.array(now, np.int32)))
        graph.replay()
        torch.cuda.synchronize()
        fits = [n if n <= 1280 else 0 for n in now]
        o, bound = R.attention(c, table, fits, 1, None, q, heads, D ** -0.5)
        got = back(out).copy()
        for b, n in enumerate(now):
            if n > 1280:  # past the table
                assert np.isnan(R.bf16_val(got[b])).all()
                got[b] = 0
        check(got, o, bound, fits, 1, None, now)


@pytest.mark.parametrize("kind", ["fp4", "bf16"])
def test_pools_past_4_gib(kind):
    """Pages at the far end of pools of 5 GiB: stored, read back, bounded, listed and looked at."""
    D, page, kvh, heads = 128, 256, 8, 16
    token = kvh * (D // 2 if kind == "fp4" else 2 * D)
    pages = (5 << 30) // (page * token)
    g = va.KVCache.empty(va.KVType[kind.upper()], pages, page, kvh, D)
    rng = np.random.default_rng(1)
    table, n = np.array([[pages - 1, 3, pages - 2, pages // 2 + 1]], np.int32), 900
    x = R.bf16_bits(rng.standard_normal((n, kvh * D)))
    batch = va.KVBatch(dev(table), dev(np.array([n], np.int32)), n)
    assert va.kv_append(g, batch, dev(x), dev(x[::-1].copy())).ok()
    ko, vo = (dev(np.zeros((n, kvh, D), np.uint16)) for _ in range(2))
    assert va.kv_read(g, batch, ko, vo).ok()
    k, v = (R.bf16_val(back(t)).astype(np.float64) for t in (ko, vo))
    want = R.bf16_val(x).astype(np.float64).reshape(n, kvh, D)
    np.testing.assert_array_equal(k, F.quantize_k(want)[0] if kind == "fp4" else want)
    if kind == "bf16":
        np.testing.assert_array_equal(v, want[::-1])
    near = torch.zeros((pages, kvh, 2, D), dtype=torch.int16, device="cuda")
    assert va.kv_page_bounds(g, batch, near).ok()
    for c, pg in enumerate(table[0]):
        got = R.bf16_val(back(near[int(pg)])).astype(np.float64)
        part = k[c * page:(c + 1) * page]
        np.testing.assert_array_equal(got[:, 0], part.min(0))
        np.testing.assert_array_equal(got[:, 1], part.max(0))
    one = va.KVBatch(batch.block_table, batch.seq_lens)
    q = R.bf16_bits(rng.standard_normal((1, heads * D)))
    sel = torch.zeros((1, kvh, 3), dtype=torch.int32, device="cuda")
    assert va.select_pages(g, one, dev(q), near, sel, first=0, workspace=ws_of(va.select_workspace_bytes(g, one, heads, 3))).ok()
    out, whole = (dev(np.zeros((1, heads * D), np.uint16)) for _ in range(2))
    assert va.attention_selected(g, one, dev(q), sel, out, workspace=ws_of(va.attention_selected_workspace_bytes(g, one, heads, 3))).ok()
    assert va.attention_paged(g, one, dev(q), whole, workspace=workspace(g, one, heads)).ok()
    f = R.bf16_val(back(near)[table[0]]).astype(np.float64)
    x = R.bf16_val(q[0]).astype(np.float64).reshape(kvh, 2, D)
    for h in range(kvh):
        want = P.select(x[h], f[:, h], range(4), 4, page, n - 1, 0, 1, 3)
        assert sel[0, h].tolist() == want
        for got, j in ((out, np.concatenate([np.arange(c * page, min(n, (c + 1) * page)) for c in want])), (whole, np.arange(n))):
            kk, vv = k[j, h], v[j, h]
            s = D ** -0.5 * (x[h] @ kk.T)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            # (decode_ref.attention's bound; FP4 values are read back as bf16 here: half a step more of each)
            size = (D ** -0.5 * (np.abs(x[h]) @ np.abs(kk).T)).max()
            e = 2 * D * 2.0 ** -24 * size + 8 * 2.0 ** -23 * np.abs(s).max() + 2.0 ** -15 + len(j) * 2.0 ** -28 + 2.0 ** -8
            y = R.bf16_val(back(got)).reshape(kvh, 2, D)[h]
            assert np.all(np.abs(y - w @ vv) <= 2.0 ** -8 * np.abs(w @ vv) + e * (w @ np.abs(vv)))


def test_other_streams():
    """The whole chain on a side stream, by argument and as the current one, beside the same chain on the default stream."""
    D, page, kvh, heads, n, count = 128, 64, 2, 10, 2000, 6
    rng = np.random.default_rng(4)
    table, pages = table_for(rng, [n], page)
    rows = dev(R.bf16_bits(rng.standard_normal((n, kvh * D))))
    q = dev(R.bf16_bits(rng.standard_normal((1, heads * D))))

    def chain(stream):
        g = va.KVCache.empty(va.KVType.FP4, pages, page, kvh, D)
        lens = dev(np.array([n], np.int32))
        fill, one = va.KVBatch(dev(table), lens, n), va.KVBatch(dev(table), lens)
        near = torch.zeros((pages, kvh, 2, D), dtype=torch.int16, device="cuda")
        sel = torch.zeros((1, kvh, count), dtype=torch.int32, device="cuda")
        out = dev(np.zeros((1, heads * D), np.uint16))
        ws = [ws_of(va.select_workspace_bytes(g, one, heads, count)), ws_of(va.attention_selected_workspace_bytes(g, one, heads, count))]
        torch.cuda.synchronize()
        for st in (va.kv_append(g, fill, rows, rows, stream=stream), va.kv_page_bounds(g, fill, near, stream=stream),
                   va.select_pages(g, one, q, near, sel, workspace=ws[0], stream=stream),
                   va.attention_selected(g, one, q, sel, out, workspace=ws[1], stream=stream)):
            assert st.ok(), st
        return g, near, sel, out, ws

    side = torch.cuda.Stream()
    runs = [chain(None), chain(side), chain(side.cuda_stream)]
    with torch.cuda.stream(side):
        runs.append(chain(None))
    torch.cuda.synchronize()
    for r in runs[1:]:
        for a, b in zip(r[1:4], runs[0][1:4]):
            assert torch.equal(a, b)


def test_one_workspace_serves_shapes_in_turn():
    """attention_paged and attention_selected of several shapes and cache types through one workspace, each twice."""
    rng = np.random.default_rng(6)
    calls = []
    for kind, D, page, kvh, heads, lens, rows, count in (("fp4", 128, 64, 2, 10, [3000, 100, 900], 1, 20), ("bf16", 64, 32, 1, 4, [900], 2, 9),
                                                         ("int8", 256, 128, 2, 6, [700, 4000], 1, 5), ("fp4", 64, 256, 4, 4, [5000], 16, 3)):
        table, pages = table_for(rng, lens, page)
        c = F.make_cache(kind, pages, page, kvh, D, rng)
        g = F.gpu_cache(c, va, dev)
        total = len(lens) * rows
        batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows)
        q = R.bf16_bits(rng.standard_normal((total, heads * D)))
        lists = np.stack([[rng.permutation(p // page + 1)[:count].tolist() + [-1] * (count - min(count, p // page + 1)) for _ in range(kvh)]
                          for _, _, p in R.row_map(lens, rows, None)]).astype(np.int32)
        calls.append((g, batch, q, lists, heads, lens, rows, R.attention(c, table, lens, rows, None, q, heads, D ** -0.5),
                      P.attention(c, table, lens, rows, None, q, heads, D ** -0.5, lists)))
    w = ws_of(max(max(va.attention_workspace_bytes(g, b, h), va.attention_selected_workspace_bytes(g, b, h, l.shape[2]))
                  for g, b, _, l, h, *_ in calls))
    for _ in range(2):
        for g, batch, q, lists, heads, lens, rows, whole, listed in calls:
            for want, run in ((whole, lambda o: va.attention_paged(g, batch, dev(q), o, workspace=w)),
                              (listed, lambda o: va.attention_selected(g, batch, dev(q), dev(lists), o, workspace=w))):
                out = dev(np.zeros(q.shape, np.uint16))
                assert run(out).ok()
                check(back(out), *want, lens, rows, None)


@pytest.mark.parametrize("n", [511, 512, 513, 1025, 2048, 2049, 4096, 4097, 9000])
def test_as_many_pages_as_a_workgroup_holds_and_one_more(n):
    """Tables of every variant of the selection's workgroup: distinct and equal scores, among few and many wanted."""
    D, page, kvh, heads = 64, 32, 1, 2
    rng = np.random.default_rng(n)
    table = rng.permutation(n).astype(np.int32)[None, :]
    near = R.bf16_bits(np.sort(rng.standard_normal((n, kvh, 2, D)), 2))
    near[rng.permutation(n)[:n // 3]] = near[0]
    g = va.KVCache(va.KVType.FP4, *(torch.zeros((n, kvh, 1, 16 * D), dtype=torch.uint8, device="cuda") for _ in range(2)), page, kvh, D,
                   torch.zeros((n, kvh, page, 2), dtype=torch.uint8, device="cuda"), torch.zeros((n, kvh, page), device="cuda"))
    f = R.bf16_val(near).astype(np.float64)[:, 0]
    for length in (n * page, n * page - 40):
        batch = va.KVBatch(dev(table), dev(np.array([length], np.int32)), 2)
        q = R.bf16_bits(rng.standard_normal((2, heads * D)))
        for count in (5, n // 3, n // 2 + 7, n - 1):
            sel = dev(np.zeros((2, kvh, count), np.int32))
            ws = ws_of(va.select_workspace_bytes(g, batch, heads, count))
            assert va.select_pages(g, batch, dev(q), dev(near), sel, first=1, last=2, workspace=ws).ok()
            for r in range(2):
                x = R.bf16_val(q[r]).astype(np.float64).reshape(heads, D)
                assert back(sel)[r, 0].tolist() == P.select(x, f, table[0], n, page, length - 2 + r, 1, 2, count), (length, count, r)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 5, 8, 9, 16, 17, 32, 33, 40, 64])
def test_every_head_of_a_key_head_counts(D, G):
    """Rows of up to 64 heads to a key head (queries of several turns of 16, padded or not): each head alone decides about pages of its own."""
    page, kvh, n, rows = 32, 2, 70, [16, 0, 5, 1]
    rng = np.random.default_rng(D + G)
    lens = [n * page - 3, 40, 33 * page, 17 * page + 1]
    table = np.stack([rng.permutation(n) for _ in lens]).astype(np.int32)
    near = np.sort(rng.standard_normal((n, kvh, 2, D)), 2)
    q = 0.05 * rng.standard_normal((sum(rows), kvh, G, D))
    for i in range(sum(rows)):  # the head that looks along the page's own dimension
        h = i % G
        q[i, :, h, (7 * h) % D] = 4.0
        q[i, 1, (h + G // 2) % G, (11 * h + 3) % D] = -3.0
    near, q = R.bf16_bits(near), R.bf16_bits(q.reshape(sum(rows), kvh * G * D))
    offs = offsets(rows)
    g = va.KVCache.empty(va.KVType.BF16, n, page, kvh, D)
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), 16, dev(offs), sum(rows))
    f = R.bf16_val(near).astype(np.float64)
    count = 12
    sel = dev(np.zeros((sum(rows), kvh, count), np.int32))
    ws = ws_of(va.select_workspace_bytes(g, batch, kvh * G, count))
    assert va.select_pages(g, batch, dev(q), dev(near), sel, first=1, last=2, workspace=ws).ok()
    got = back(sel)
    for b, r, p in R.row_map(lens, 16, offs):
        x = R.bf16_val(q[r]).astype(np.float64).reshape(kvh, G, D)
        for h in range(kvh):
            assert got[r, h].tolist() == P.select(x[h], f[:, h], table[b], n, page, p, 1, 2, count), (b, r, p, h)


def busy(stream, a, b):
    """Copies of 600 GB in all (over a tenth of a second) on a stream, which the host is well ahead of."""
    with torch.cuda.stream(stream):
        for _ in range(300):
            a.copy_(b)


@pytest.mark.parametrize("how", ["argument", "number", "current"])
@pytest.mark.parametrize("kind", ["fp4", "bf16"])
def test_each_call_waits_for_the_work_before_it_on_its_stream(kind, how):
    """Inputs change on a side stream behind a delay, then the call: a launch of it on any other stream (the second of the selection,
    and of attentions that join apart, among them) would still see the former inputs, or what the former call left of them."""
    D, page, kvh, heads, n, count = 128, 64, 2, 10, 20000, 64
    rng = np.random.default_rng(7)
    table, pages = table_for(rng, [n], page)
    lens = dev(np.array([n], np.int32))
    fill, one = va.KVBatch(dev(table), lens, 300), va.KVBatch(dev(table), lens)
    caches = [F.gpu_cache(F.make_cache(kind, pages, page, kvh, D, rng), va, dev) for _ in range(2)]
    g = F.gpu_cache(F.make_cache(kind, pages, page, kvh, D, rng), va, dev)
    pools = [t for t in ("k", "v", "k_scales", "v_scales") if getattr(g, t) is not None]
    rows = [dev(R.bf16_bits(rng.standard_normal((300, kvh * D)))) for _ in range(2)]
    qs = [dev(R.bf16_bits(rng.standard_normal((1, heads * D)))) for _ in range(2)]
    near = dev(R.bf16_bits(np.sort(rng.standard_normal((pages, kvh, 2, D)), 2)))
    lists = [torch.stack([torch.randperm(n // page, device="cuda")[:count] for _ in range(kvh)])[None].to(torch.int32) for _ in range(2)]
    row, q, sel = rows[0].clone(), qs[0].clone(), lists[0].clone()
    box = lambda *s, dt=torch.int16: torch.zeros(s, dtype=dt, device="cuda")
    bounds, chosen, out, whole, ko, vo = (box(pages, kvh, 2, D), box(1, kvh, count, dt=torch.int32), box(1, heads * D), box(1, heads * D),
                                          box(300, kvh, D), box(300, kvh, D))
    ws = [ws_of(va.select_workspace_bytes(g, one, heads, count)), ws_of(va.attention_selected_workspace_bytes(g, one, heads, count)),
          workspace(g, one, heads)]
    content = [[getattr(c, t) for t in pools] for c in caches]
    held = [getattr(g, t) for t in pools]
    steps = [  # name, inputs, what they hold before and after, outputs, call
        ("append", [row], [[x] for x in rows], held, lambda st: va.kv_append(g, fill, row, row, stream=st)),
        ("read", held, content, [ko, vo], lambda st: va.kv_read(g, fill, ko, vo, stream=st)),
        ("bounds", held, content, [bounds], lambda st: va.kv_page_bounds(g, fill, bounds, stream=st)),
        ("select", [q], [[x] for x in qs], [chosen], lambda st: va.select_pages(g, one, q, near, chosen, workspace=ws[0], stream=st)),
        ("lists", [sel], [[x] for x in lists], [out], lambda st: va.attention_selected(g, one, q, sel, out, workspace=ws[1], stream=st)),
        ("queries", [q], [[x] for x in qs], [out], lambda st: va.attention_selected(g, one, q, sel, out, workspace=ws[1], stream=st)),
        ("whole", [q], [[x] for x in qs], [whole], lambda st: va.attention_paged(g, one, q, whole, workspace=ws[2], stream=st))]
    side = torch.cuda.Stream()
    given = {"argument": side, "number": side.cuda_stream, "current": None}[how]
    big = [torch.zeros(1 << 30, dtype=torch.uint8, device="cuda") for _ in range(2)]
    for name, inputs, (old, new), outputs, call in steps:
        print("stream", kind, how, name, flush=True)

        def now(values):
            for t, x in zip(inputs, values):
                t.copy_(x)

        start = [t.clone() for t in outputs]
        now(new)
        assert call(None).ok()
        want = [t.clone() for t in outputs]
        for t, x in zip(outputs, start):
            t.copy_(x)
        now(old)
        assert call(None).ok()
        assert not all(torch.equal(t, x) for t, x in zip(outputs, want))
        torch.cuda.synchronize()
        busy(side, *big)
        with torch.cuda.stream(side):
            now(new)
            if how == "current":
                assert call(None).ok()
        if how != "current":
            assert call(given).ok()
        assert not side.query()  # (the delay still runs: nothing before the call has)
        with torch.cuda.stream(side):
            got = [t.clone() for t in outputs]
        side.synchronize()
        for t, x in zip(got, want):
            assert torch.equal(t.view(torch.uint8), x.view(torch.uint8)), name


def test_chains_on_several_streams_at_once():
    """Four chains, each of tensors of its own, all queued before the first is waited for, on the default stream and three others."""
    D, page, kvh, heads, n, count = 128, 64, 2, 10, 9000, 40
    rng = np.random.default_rng(8)
    table, pages = table_for(rng, [n], page)
    lens = dev(np.array([n], np.int32))
    fill, one = va.KVBatch(dev(table), lens, n), va.KVBatch(dev(table), lens)
    rows = [dev(R.bf16_bits(rng.standard_normal((n, kvh * D)))) for _ in range(4)]
    qs = [dev(R.bf16_bits(rng.standard_normal((1, heads * D)))) for _ in range(4)]

    def tensors():
        g = va.KVCache.empty(va.KVType.FP4, pages, page, kvh, D)
        return (g, torch.zeros((pages, kvh, 2, D), dtype=torch.int16, device="cuda"),
                torch.zeros((1, kvh, count), dtype=torch.int32, device="cuda"), dev(np.zeros((1, heads * D), np.uint16)),
                ws_of(va.select_workspace_bytes(g, one, heads, count)), ws_of(va.attention_selected_workspace_bytes(g, one, heads, count)))

    def calls(i, t, stream):
        g, near, sel, out, w0, w1 = t
        return (lambda: va.kv_append(g, fill, rows[i], rows[i], stream=stream), lambda: va.kv_page_bounds(g, fill, near, stream=stream),
                lambda: va.select_pages(g, one, qs[i], near, sel, workspace=w0, stream=stream),
                lambda: va.attention_selected(g, one, qs[i], sel, out, workspace=w1, stream=stream))

    want = []
    for i in range(4):  # one after the other
        t = tensors()
        for call in calls(i, t, None):
            assert call().ok()
        torch.cuda.synchronize()
        want.append([x.clone() for x in t[1:4]])
    streams = [None] + [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        runs = [tensors() for _ in range(4)]
        chains = [calls(i, t, s) for i, (t, s) in enumerate(zip(runs, streams))]
        torch.cuda.synchronize()
        for step in zip(*chains):
            for call in step:
                assert call().ok()
        torch.cuda.synchronize()
        for t, w in zip(runs, want):
            for a, b in zip(t[1:4], w):
                assert torch.equal(a, b)
