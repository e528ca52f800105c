"""attention_paged against the plain 64-bit implementation, with its derived bound (decode_ref.attention)."""
import numpy as np
import pytest

import decode_ref as R
import viper_amd as va
from test_gpu_kv_cache import SENT, back, dev, gpu_cache, table_for

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def workspace(cache, batch, heads, fill=0):
    return torch.zeros((max(16, va.attention_workspace_bytes(cache, batch, heads)),), dtype=torch.uint8, device="cuda")


def check(got, o, bound, lens, rows, offs, what=""):
    """got: bf16 bits [rows, heads * D]."""
    for b, r, p in R.row_map(lens, rows, offs):
        y = R.bf16_val(got[r]).astype(np.float64).reshape(o[r].shape)
        nan = np.isnan(o[r])
        assert np.array_equal(np.isnan(y), nan), (what, b, r, p)
        fin = np.isfinite(o[r])
        assert np.array_equal(y[~fin & ~nan], o[r][~fin & ~nan]), (what, b, r, p)
        off = np.abs(y[fin] - o[r][fin])
        assert np.all(off <= bound[r][fin]), (what, b, r, p, off.max(), (off / bound[r][fin]).max())


def setup(D, i8, page, kvh, heads, lens, rows, counts=None, seed=0, q_std=1.5, std=1.0):
    rng = np.random.default_rng(seed)
    table, pages = table_for(rng, lens, page)
    c = R.Cache(i8, pages, page, kvh, D, rng, std)
    offs = None if counts is None else np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    total = len(lens) * rows if counts is None else int(offs[-1])
    q = R.bf16_bits(q_std * rng.standard_normal((total, heads * D)))
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows, None if offs is None else dev(offs))
    return c, table, offs, total, q, batch


CASES = [  # D, i8, page, kvh, heads, lens, rows, counts, window, sinks
    (128, False, 64, 4, 20, [1], 1, None, 0, 0),
    (128, False, 64, 4, 20, [31, 32, 33, 63, 64, 65, 127, 129], 1, None, 0, 0),
    (64, False, 32, 1, 1, [2, 1, 300], 1, None, 0, 0),
    (256, False, 128, 2, 6, [500, 17], 1, None, 0, 0),
    (128, True, 64, 4, 20, [1, 32, 33, 700], 1, None, 0, 0),
    (64, True, 256, 3, 12, [257, 90], 1, None, 0, 0),
    (256, True, 32, 2, 2, [1000], 1, None, 0, 0),
    (128, False, 64, 4, 20, [16, 40, 333], 16, None, 0, 0),        # 80 rows to a key head
    (128, True, 64, 1, 8, [16, 200], 16, None, 0, 0),              # 128 rows
    (256, False, 64, 1, 5, [70], 13, None, 0, 0),
    (64, False, 32, 2, 14, [100, 9, 64], 7, [7, 1, 5], 0, 0),      # 49 rows: a group of 4 operands
    (128, False, 64, 8, 48, [90, 5, 64, 33], 5, [5, 0, 2, 3], 0, 0),
    (128, False, 32, 2, 2, [4, 2], 4, None, 0, 0),                 # rows at negative positions
    (128, False, 64, 4, 20, [700, 40, 3], 1, None, 100, 0),        # windows
    (128, False, 64, 4, 20, [700, 40, 3], 3, None, 1, 0),          # a window of one token
    (128, False, 32, 4, 20, [900, 41], 4, None, 65, 4),            # and first tokens
    (128, True, 64, 2, 10, [900, 64, 700], 16, None, 32, 33),
    (64, False, 64, 1, 3, [500], 2, None, 450, 100),               # first tokens that meet the window
    (64, False, 64, 1, 3, [500], 2, None, 1000, 7),                # a window longer than the sequence
    (64, True, 64, 1, 64, [333], 3, None, 2 ** 31 - 1, 2 ** 31 - 1),
    (128, False, 256, 4, 8, [9000, 4097], 1, None, 0, 0),          # many parts
    (128, True, 128, 1, 4, [20000], 2, None, 0, 0),
    (128, False, 64, 2, 8, [30000], 2, None, 5000, 64),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("ws", [True, False])
def test_attention(case, ws):
    D, i8, page, kvh, heads, lens, rows, counts, window, sinks = case
    print(f"attention {case} ws={ws}", flush=True)
    c, table, offs, total, q, batch = setup(D, i8, page, kvh, heads, lens, rows, counts)
    g = gpu_cache(c)
    out = dev(np.full((total + 2, heads * D), SENT))  # rows behind the last sequence
    w = workspace(g, batch, heads) if ws else None
    for _ in range(2):  # the workspace serves the next call
        assert va.attention_paged(g, batch, dev(q), out[:total], window=window, sinks=sinks, workspace=w).ok()
    o, bound = R.attention(c, table, lens, rows, offs, q, heads, D ** -0.5, window, sinks)
    got = back(out)
    check(got, o, bound, lens, rows, offs, case)
    assert np.all(got[total:] == SENT)
    if w is not None:
        assert not np.any(back(w)[:8192])  # its counters are zero again


def test_rows_behind_the_last_sequence_and_offsets_that_do_not_fit():
    c, table, _, _, q, _ = setup(128, False, 64, 2, 4, [90, 50], 3, [3, 2])
    g = gpu_cache(c)
    q = np.concatenate([q, q])[:8]
    for offs, kept in (([0, 3, 5], [5, 6, 7]), ([2, 5, 5], [0, 1, 5, 6, 7]), ([0, 4, 5], [0, 1, 2, 3, 5, 6, 7]),
                       ([0, 3, 9], [3, 4, 5, 6, 7]), ([-1, 2, 5], [0, 1, 5, 6, 7])):
        batch = va.KVBatch(dev(table), dev(np.array([90, 50], np.int32)), 3, dev(np.array(offs, np.int32)))
        out = dev(np.full((8, 4 * 128), SENT))
        assert va.attention_paged(g, batch, dev(q), out, workspace=workspace(g, batch, 4)).ok()
        got = back(out)
        written = [r for r in range(8) if not np.all(got[r] == SENT)]
        assert written == [r for r in range(8) if r not in kept], (offs, written)


@pytest.mark.parametrize("i8", [False, True])
def test_what_no_row_sees_never_counts(i8):
    """Places past the length, pages behind the window and table entries behind it hold NaN, infinities or no page at all."""
    D, page, kvh, heads = 128, 64, 2, 8
    lens, rows, window, sinks = [1000, 70], 3, 100, 5
    c, table, offs, total, q, _ = setup(D, i8, page, kvh, heads, lens, rows)
    o, bound = R.attention(c, table, lens, rows, offs, q, heads, D ** -0.5, window, sinks)
    rng = np.random.default_rng(1)
    bad = np.array([0x7FC0, 0x7F80, 0xFF80, 0x7F7F], np.uint16)
    for b, n in enumerate(lens):
        first = n - rows - window + 1
        for col in range(-(-n // page)):
            for at in range(page):
                j = col * page + at
                if j >= n or sinks <= j < first:
                    for h in range(kvh):
                        if i8:
                            c.ks[c.scale_at(table[b, col], at, h)] = np.nan
                            c.vs[c.scale_at(table[b, col], at, h)] = np.inf
                        else:
                            c.k[c.places(table[b, col], at, h, True)] = rng.choice(bad, D)
                            c.v[c.places(table[b, col], at, h, False)] = rng.choice(bad, D)
            if col * page >= sinks and (col + 1) * page <= first:
                table[b, col] = rng.choice([-1, 10 ** 9])
    g = gpu_cache(c)
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows)
    out = dev(np.full((total, heads * D), SENT))
    assert va.attention_paged(g, batch, dev(q), out, window=window, sinks=sinks, workspace=workspace(g, batch, heads)).ok()
    check(back(out), o, bound, lens, rows, offs)


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("ws", [True, False])
@pytest.mark.parametrize("value", [0x7F80, 0xFF80, 0x7FC0])
def test_values_that_are_not_finite_reach_only_rows_that_see_them(i8, ws, value):
    """The newest rows' own tokens hold infinities or NaN: earlier rows of the draft do not see them, later ones do; a window
    lets the later rows forget an early one."""
    D, page, kvh, heads, lens, rows = 64, 32, 1, 3, [600, 45], 6
    # rows at 594..599 and 39..44: three of six finite in each sequence, but none of the first where 557 and 597 are both hit
    for window, hit, finite in ((0, [(0, 597), (1, 42)], 6), (40, [(0, 597), (1, 42), (0, 557)], 3), (40, [(0, 557), (1, 42)], 6)):
        c, table, offs, total, q, batch = setup(D, i8, page, kvh, heads, lens, rows, seed=3)
        for b, j in hit:
            pg, at = table[b, j // page], j % page
            if i8:
                c.vs[c.scale_at(pg, at, 0)] = R.bf16_val(np.uint16(value))
                c.v[c.places(pg, at, 0, False)] = np.int8(3)
            else:
                c.v[c.places(pg, at, 0, False)[5]] = value
        g = gpu_cache(c)
        out = dev(np.full((total, heads * D), SENT))
        assert va.attention_paged(g, batch, dev(q), out, window=window, workspace=workspace(g, batch, heads) if ws else None).ok()
        o, bound = R.attention(c, table, lens, rows, offs, q, heads, D ** -0.5, window, 0)
        assert sum(bool(np.all(np.isfinite(x))) for x in o.values()) == finite
        check(back(out), o, bound, lens, rows, offs, (window, value))


def test_keys_that_are_not_finite():
    """NaN keys make the rows that see them NaN; keys of -inf weigh nothing; a row of nothing but such keys is 0 / 0."""
    D, page, lens, rows = 64, 32, [40, 2], 2
    c, table, offs, total, q, batch = setup(D, False, page, 1, 1, lens, rows, seed=4)
    q[:] = R.bf16_bits(np.abs(R.bf16_val(q)) + 0.01)
    c.k[c.places(table[0, 1], 39 % 32, 0, True)[3]] = 0x7FC0           # seen by the last row only
    c.k[c.places(table[0, 0], 7, 0, True)[1]] = 0xFF80                  # -inf: no weight
    for j in (0, 1):
        c.k[c.places(table[1, 0], j, 0, True)[9]] = 0xFF80
    g = gpu_cache(c)
    out = dev(np.full((total, D), SENT))
    assert va.attention_paged(g, batch, dev(q), out).ok()
    o, bound = R.attention(c, table, lens, rows, offs, q, 1, D ** -0.5)
    assert np.isfinite(o[0]).all() and np.isnan(o[1]).all() and np.isnan(o[2]).all() and np.isnan(o[3]).all()
    bound[0] = 2.0 ** -8 * np.abs(o[0]) + 2.0 ** -10  # (the -inf key's product size is infinite: a plain bound, |v| < 4 and w e < 2^-13)
    check(back(out), o, bound, lens, rows, offs)


@pytest.mark.parametrize("ws", [True, False])
def test_missing_pages_and_lengths_past_the_table(ws):
    D, page, kvh, heads, rows = 64, 32, 1, 2, 4
    lens = [600, 34, 100]
    c, table, offs, total, q, _ = setup(D, False, page, kvh, heads, lens, rows)
    want, bound = R.attention(c, table, lens, rows, offs, q, heads, D ** -0.5)
    table[0, 7] = c.pages                    # every row of the first sequence sees it
    table[1, 1] = -5                         # tokens 32, 33: the last two rows see it, the first two do not
    g = gpu_cache(c)
    batch = va.KVBatch(dev(table), dev(np.array(lens, np.int32)), rows)
    out = dev(np.full((total, heads * D), SENT))
    assert va.attention_paged(g, batch, dev(q), out, workspace=workspace(g, batch, heads) if ws else None).ok()
    y = R.bf16_val(back(out))
    assert np.all(np.isnan(y[:4])) and np.all(np.isnan(y[6:8]))
    for r in (4, 5, 8, 9, 10, 11):
        assert np.all(np.abs(y[r].reshape(heads, D) - want[r]) <= bound[r])
    cap = table.shape[1] * page
    for n in (cap + 2, cap + 100, 2 ** 31 - 1):   # the first: its first two rows are inside
        b1 = va.KVBatch(dev(np.where(table < 0, 0, np.minimum(table, c.pages - 1))[:1].copy()), dev(np.array([n], np.int32)), rows)
        out = dev(np.full((rows, heads * D), SENT))
        assert va.attention_paged(g, b1, dev(q[:rows]), out, workspace=workspace(g, b1, heads) if ws else None).ok()
        y = R.bf16_val(back(out))
        inside = [r for r in range(rows) if n - rows + r < cap]
        assert [r for r in range(rows) if np.all(np.isfinite(y[r]))] == inside
        assert all(np.all(np.isnan(y[r])) for r in range(rows) if r not in inside)


def test_peaked_and_flat_scores():
    """Scores of +-80 (weights that leave 32 bits) and equal ones."""
    for std, q_std in ((4.0, 8.0), (0.0, 1.0)):
        c, table, offs, total, q, batch = setup(128, False, 64, 2, 4, [3000], 2, q_std=q_std, std=std)
        if std == 0.0:
            c.v[:] = R.bf16_bits(np.random.default_rng(2).standard_normal(len(c.v)))
        g = gpu_cache(c)
        out = dev(np.full((total, 4 * 128), SENT))
        assert va.attention_paged(g, batch, dev(q), out, workspace=workspace(g, batch, 4)).ok()
        o, bound = R.attention(c, table, [3000], 2, offs, q, 4, 128 ** -0.5)
        check(back(out), o, bound, [3000], 2, offs)


def test_columns_of_wider_rows_and_scale():
    D, kvh, heads, lens, rows = 128, 4, 20, [77, 300], 3
    c, table, offs, total, q, batch = setup(D, False, 64, kvh, heads, lens, rows)
    g = gpu_cache(c)
    wide = np.full((total, heads * D + 1024), SENT)
    wide[:, 256:256 + heads * D] = q
    W, O = dev(wide), dev(np.full((total, heads * D + 64), SENT))
    assert va.attention_paged(g, batch, W[:, 256:256 + heads * D], O[:, 32:32 + heads * D], scale=0.03).ok()
    o, bound = R.attention(c, table, lens, rows, offs, q, heads, float(np.float32(0.03)))
    got = back(O)
    check(got[:, 32:32 + heads * D], o, bound, lens, rows, offs)
    assert np.all(got[:, :32] == SENT) and np.all(got[:, 32 + heads * D:] == SENT)
    three = va.attention_paged(g, batch, dev(q).view(total, heads, D), O[:, :heads * D].unflatten(1, (heads, D)), scale=0.03)
    assert three.ok()
    check(back(O)[:, :heads * D], o, bound, lens, rows, offs)


def test_one_workspace_for_calls_of_every_shape():
    w = torch.zeros((64 << 20,), dtype=torch.uint8, device="cuda")
    for i, (D, i8, kvh, heads, lens, rows) in enumerate([(128, False, 4, 20, [9000], 1), (64, True, 1, 8, [5000, 70], 16),
                                                         (256, False, 2, 4, [3000], 2), (128, False, 8, 8, [600] * 9, 1),
                                                         (128, False, 4, 20, [9000], 1)]):
        c, table, offs, total, q, batch = setup(D, i8, 64, kvh, heads, lens, rows, seed=i)
        g = gpu_cache(c)
        out = dev(np.full((total, heads * D), SENT))
        assert va.attention_paged(g, batch, dev(q), out, workspace=w).ok()
        o, bound = R.attention(c, table, lens, rows, offs, q, heads, D ** -0.5)
        check(back(out), o, bound, lens, rows, offs, i)


def test_same_inputs_same_bits():
    c, table, offs, total, q, batch = setup(128, False, 64, 4, 20, [20000], 1)
    g = gpu_cache(c)
    Q, w = dev(q), workspace(g, batch, 20)
    outs = []
    for _ in range(8):
        out = dev(np.full((1, 20 * 128), SENT))
        assert va.attention_paged(g, batch, Q, out, workspace=w).ok()
        outs.append(back(out))
    assert all(np.array_equal(outs[0], o) for o in outs[1:])


def test_streams_and_graphs():
    """Another stream than the current one; a captured append + attention replayed while sequences grow, two graphs on one
    workspace, eager calls between the replays."""
    D, page, kvh, heads, B = 128, 64, 4, 20, 3
    rng = np.random.default_rng(12)
    cap = [4000, 900, 130]
    table, pages = table_for(rng, cap, page)
    c = R.Cache(False, pages, page, kvh, D, rng)
    g = gpu_cache(c)
    lens = torch.tensor([3990, 880, 62], dtype=torch.int32, device="cuda")
    batch = va.KVBatch(dev(table), lens, 1)
    qkv = torch.zeros((B, (heads + 2 * kvh) * D), dtype=torch.bfloat16, device="cuda")
    q, k, v = qkv[:, :heads * D], qkv[:, heads * D:(heads + kvh) * D], qkv[:, (heads + kvh) * D:]
    out, qr = (torch.zeros((B, heads * D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    w = workspace(g, batch, heads)

    def step():
        lens.add_(1)
        assert va.kv_append(g, batch, k, v, q=q, q_out=qr, rope_theta=10000.0).ok()
        assert va.attention_paged(g, batch, qr, out, workspace=w).ok()

    def read():
        lens.sub_(0)
        assert va.attention_paged(g, batch, qr, out, window=50, sinks=3, workspace=w).ok()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        read()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for f in (step, read):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f()
        graphs.append(gr)
    eager = torch.zeros_like(out)
    for i in range(4):
        qkv.copy_(torch.from_numpy(rng.standard_normal(tuple(qkv.shape)).astype(np.float32)).to("cuda"))
        n0 = lens.tolist()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert lens.tolist() == [n + 1 for n in n0]
        first = out.clone()
        # the plain result from what the cache holds now
        c.k, c.v = back(g.k.view(torch.int16)).ravel(), back(g.v.view(torch.int16)).ravel()
        bits = back(qr.view(torch.int16))
        n = lens.tolist()
        o, bound = R.attention(c, table, n, 1, None, bits, heads, D ** -0.5)
        check(back(first.view(torch.int16)), o, bound, n, 1, None, i)
        for b in range(B):  # the newest token is the rotated k
            pg, at = table[b, (n[b] - 1) // page], (n[b] - 1) % page
            want = R.rotate(k[b].view(kvh, D)[1].float().cpu().numpy().astype(np.float64), n[b] - 1, 10000.0)
            np.testing.assert_array_equal(c.k[c.places(pg, at, 1, True)], R.bf16_bits(want.astype(np.float32)))
        graphs[1].replay()
        torch.cuda.synchronize()
        o, bound = R.attention(c, table, n, 1, None, bits, heads, D ** -0.5, 50, 3)
        check(back(out.view(torch.int16)), o, bound, n, 1, None, i)
        assert va.attention_paged(g, batch, qr, eager, workspace=w, stream=side).ok()
        side.synchronize()
        assert torch.equal(eager.view(torch.int16), first.view(torch.int16))


@pytest.mark.parametrize("i8", [False, True])
def test_a_prompt_in_chunks_then_tokens(i8):
    """The operators together: a prompt appended 16 rows at a time, then single tokens; every row's attention against the
    plain result over what the cache holds, and over unquantized rows for the bf16 cache."""
    D, page, kvh, heads, theta = 64, 32, 2, 6, 10000.0
    rng = np.random.default_rng(21)
    total = 75
    x = R.bf16_bits(rng.standard_normal((total, (heads + 2 * kvh) * D)))
    table, pages = table_for(rng, [total], page)
    c = R.Cache(i8, pages, page, kvh, D)
    g = gpu_cache(c)
    X = dev(x)
    at = 0
    for n in [16, 16, 16, 16, 3] + [1] * 8:
        rows = X[at:at + n]
        at += n
        batch = va.KVBatch(dev(table), dev(np.array([at], np.int32)), n)
        q = rows[:, :heads * D].clone()
        assert va.kv_append(g, batch, rows[:, heads * D:(heads + kvh) * D], rows[:, (heads + kvh) * D:], q=q, q_out=q,
                            rope_theta=theta).ok()
        out = dev(np.full((n, heads * D), SENT))
        assert va.attention_paged(g, batch, q, out, workspace=workspace(g, batch, heads)).ok()
        c.k, c.v = back(g.k).ravel(), back(g.v).ravel()
        if i8:
            c.ks, c.vs = back(g.k_scales).ravel(), back(g.v_scales).ravel()
        o, bound = R.attention(c, table, [at], n, None, back(q), heads, D ** -0.5)
        check(back(out), o, bound, [at], n, None, at)
    assert at == total
    if not i8:
        for j in (0, 31, 32, 74):
            want = R.rotate(R.bf16_val(x[j, heads * D:(heads + 1) * D]).astype(np.float64), j, theta)
            np.testing.assert_array_equal(R.bf16_bits(want.astype(np.float32)), R.bf16_bits(c.rows(table[0], np.array([j]), 0, True)[0]))


@pytest.mark.parametrize("i8", [False, True])
@pytest.mark.parametrize("D,gqa", [(64, 1), (64, 2), (64, 3), (64, 4), (128, 1), (128, 2), (128, 3), (128, 4), (256, 1), (256, 2),
                                   (128, 9), (256, 5)])
def test_every_kernel_over_short_and_wide_tables(i8, D, gqa):
    """16 rows of gqa heads: gqa groups of 16, so each number of operands; tables of few columns and of many (what decides the
    waves of a workgroup and the parts), a length in each range of parts, one that no workgroup splits."""
    page, rows = 64, 16
    lens = [700, 16, 4500 if D == 64 else 1500]
    c, table, offs, total, q, _ = setup(D, i8, page, 1, gqa, lens, rows, seed=D + gqa)
    g = gpu_cache(c)
    o, bound = R.attention(c, table, lens, rows, offs, q, gqa, D ** -0.5)
    for W in (table.shape[1], 300):
        wide = np.full((3, W), -1, np.int32)
        wide[:, :table.shape[1]] = table
        batch = va.KVBatch(dev(wide), dev(np.array(lens, np.int32)), rows)
        one = va.KVBatch(dev(wide[2:]), dev(np.array(lens[2:], np.int32)), rows)
        for b, r0, n in ((batch, 0, total), (one, 2 * rows, rows)):
            for w in (None, workspace(g, b, gqa)):
                out = dev(np.full((n, gqa * D), SENT))
                assert va.attention_paged(g, b, dev(q[r0:r0 + n]), out, workspace=w).ok()
                full = np.full((total, gqa * D), SENT)
                full[r0:r0 + n] = back(out)
                if n == total:
                    check(full, o, bound, lens, rows, offs, (W, w is None))
                else:
                    for r in range(r0, total):
                        off = np.abs(R.bf16_val(full[r]).reshape(gqa, D) - o[r])
                        assert np.all(off <= bound[r]), (W, w is None, r)


def test_a_batch_that_fills_the_gpu_by_itself():
    """More sequences than the workspace has counters for: nothing is split, no workspace is wanted."""
    lens = [1 + (i * 37) % 90 for i in range(1100)]
    c, table, offs, total, q, batch = setup(64, False, 32, 2, 2, lens, 1)
    g = gpu_cache(c)
    assert va.attention_workspace_bytes(g, batch, 2) == 0
    out = dev(np.full((total, 2 * 64), SENT))
    assert va.attention_paged(g, batch, dev(q), out).ok()
    o, bound = R.attention(c, table, lens, 1, offs, q, 2, 64 ** -0.5)
    check(back(out), o, bound, lens, 1, offs)


def test_sequences_that_share_pages():
    """Two sequences with one prefix: the same pages in both rows of the table."""
    c, table, offs, total, q, _ = setup(128, False, 64, 2, 8, [300, 300], 2)
    table[1, :3] = table[0, :3]
    g = gpu_cache(c)
    batch = va.KVBatch(dev(table), dev(np.array([300, 250], np.int32)), 2)
    out = dev(np.full((total, 8 * 128), SENT))
    assert va.attention_paged(g, batch, dev(q), out, workspace=workspace(g, batch, 8)).ok()
    o, bound = R.attention(c, table, [300, 250], 2, offs, q, 8, 128 ** -0.5)
    check(back(out), o, bound, [300, 250], 2, offs)


def test_python_refusals_and_empty_calls():
    c, table, offs, total, q, batch = setup(128, False, 64, 2, 4, [90, 50], 1)
    g = gpu_cache(c)
    Q, out = dev(q), dev(np.full((2, 4 * 128), SENT))
    S = va.StatusCode
    assert va.attention_paged(g, batch, Q[:1], out[:1]).code == S.SHAPE_MISMATCH
    assert va.attention_paged(g, batch, Q, out[:1]).code == S.SHAPE_MISMATCH
    assert va.attention_paged(g, batch, dev(q[:, :200].copy()), out[:, :200]).code == S.SHAPE_MISMATCH
    assert va.attention_paged(g, batch, Q, out, scale=0.0).code == S.INVALID_ARGUMENT
    assert va.attention_paged(g, batch, dev(q[:, :384].copy()), dev(q[:, :384].copy())).code == S.INVALID_ARGUMENT  # 3 heads on 2
    assert va.kv_append(g, batch, Q[:, :256], Q[:, 256:], q=Q, q_out=Q).code == S.INVALID_ARGUMENT          # no rotation
    assert va.kv_append(g, batch, Q[:, :256], Q[:, 256:], q=Q, rope_theta=1e4).code == S.SHAPE_MISMATCH
    for bad in (Q.cpu(), Q.float(), Q.t().contiguous().t()):
        with pytest.raises(ValueError):
            va.attention_paged(g, batch, bad, out)
    with pytest.raises(AttributeError):
        batch.seq_lens = dev(np.array([1, 2], np.int32))
    with pytest.raises(AttributeError):
        g.k = g.v
    assert np.all(back(out) == SENT)
    none = va.KVBatch(dev(table), dev(np.zeros(2, np.int32)), 1, dev(np.zeros(3, np.int32)))
    z = torch.empty((0, 4 * 128), dtype=torch.int16, device="cuda")
    kv = torch.empty((0, 256), dtype=torch.int16, device="cuda")
    assert va.attention_paged(g, none, z, z).ok() and va.kv_append(g, none, kv, kv).ok() and va.kv_read(g, none, kv, kv).ok()
