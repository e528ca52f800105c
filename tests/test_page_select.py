"""What the calls for selected pages refuse before any launch, and their workspaces (no GPU)."""
import numpy as np
import pytest

import decode_ref as R
import fp4_ref as F
import pages_ref as P
import viper_amd as va
from test_decode_refusals import BAD_BATCH, BAD_CACHE, FAKE, INVALID, OK, batch, cache, ref

torch = pytest.importorskip("torch")
BIG = 1 << 40  # another place than FAKE


def calls(c, b, **kw):
    L = va.lib()
    a = dict(q=FAKE, qs=2560, heads=20, bounds=2 * BIG, first=1, last=2, sel=3 * BIG, count=16, ws=BIG, nws=1 << 30, scale=0.1, out=4 * BIG,
             os=2560)
    a.update(kw)
    return [
        L.viper_hip_kv_page_bounds(ref(c), ref(b), a["bounds"], None),
        L.viper_hip_select_pages(ref(c), ref(b), a["q"], a["qs"], a["heads"], a["bounds"], a["first"], a["last"], a["sel"], a["count"],
                                 a["ws"], a["nws"], None),
        L.viper_hip_attention_selected(ref(c), ref(b), a["q"], a["qs"], a["heads"], a["scale"], a["sel"], a["count"], a["out"], a["os"],
                                       a["ws"], a["nws"], None)]


def sizes(c, b, heads=20, count=16):
    L = va.lib()
    return [f(ref(c), ref(b), heads, count) for f in (L.viper_hip_select_pages_workspace_bytes, L.viper_hip_attention_selected_workspace_bytes)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_bad_cache(bad):
    assert calls(cache(**bad), batch()) == [INVALID] * 3 and sizes(cache(**bad), batch()) == [0, 0]


@pytest.mark.parametrize("bad", BAD_BATCH)
def test_bad_batch(bad):
    assert calls(cache(), batch(**bad)) == [INVALID] * 3 and sizes(cache(), batch(**bad)) == [0, 0]


def test_null_descriptions_and_no_rows():
    assert calls(None, batch()) == [INVALID] * 3 and calls(cache(), None) == [INVALID] * 3
    assert calls(cache(), batch(total_rows=0, row_offsets=FAKE)) == [OK] * 3


@pytest.mark.parametrize("bad", [dict(bounds=None), dict(bounds=2 * BIG + 8), dict(bounds=FAKE)])
def test_bounds_refusals(bad):
    assert calls(cache(), batch(), **bad)[0] == INVALID  # (FAKE: the cache's keys)


def test_bounds_over_scales_are_refused():
    assert calls(cache(kv_type=1, k_scales=2 * BIG + 16, v_scales=FAKE), batch())[0] == INVALID
    assert calls(cache(kv_type=4, k_scales=2 * BIG + 16, v_scales=FAKE), batch())[0] == INVALID


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=FAKE + 2), dict(qs=2552), dict(qs=2564), dict(heads=0), dict(heads=18), dict(heads=-4),
                                 dict(heads=4 * 65, qs=4 * 65 * 128), dict(bounds=None), dict(bounds=2 * BIG + 2), dict(first=-1), dict(last=0),
                                 dict(last=-1), dict(first=15), dict(first=2 ** 31 - 1, last=2 ** 31 - 1), dict(count=0), dict(count=-1),
                                 dict(count=1 << 25), dict(sel=None), dict(sel=3 * BIG + 2), dict(ws=None), dict(ws=BIG + 4), dict(nws=16),
                                 dict(sel=BIG), dict(sel=FAKE), dict(sel=2 * BIG), dict(ws=FAKE), dict(ws=2 * BIG), dict(qs=1 << 48), dict(qs=1 << 62)])
def test_select_refusals(bad):
    assert calls(cache(), batch(), **bad)[1] == INVALID


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=FAKE + 2), dict(qs=2552), dict(heads=0), dict(heads=18), dict(out=None), dict(out=FAKE),
                                 dict(out=4 * BIG + 8), dict(os=100), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(count=0), dict(count=1 << 25), dict(sel=None), dict(sel=3 * BIG + 1), dict(ws=BIG + 8), dict(nws=16),
                                 dict(sel=4 * BIG), dict(sel=4 * BIG + 5000), dict(sel=4 * BIG - 8)])
def test_attention_refusals(bad):
    # (two rows of 256 listed pages: a call that is split)
    assert calls(cache(), batch(), **{"count": 256, **bad})[2] == INVALID


def test_rows_are_a_verify_steps():
    b = batch(max_rows=17, total_rows=34)
    assert calls(cache(), b)[1:] == [INVALID] * 2 and sizes(cache(), b) == [0, 0]


def test_largest_selection():
    c, b = cache(page_size=32, kv_heads=1024, num_pages=1), batch(batch=1, total_rows=1, table_width=1 << 20)
    assert calls(c, b, heads=1024, qs=1024 * 128, os=1024 * 128, nws=1 << 40)[1] == INVALID  # 2^24 workgroups


def test_workspaces():
    assert sizes(cache(), batch())[0] == 2 * 4 * (4 + 1) * 4  # a score of each row, key head and page, and how far 16 may be off
    c, one, many = cache(), batch(batch=1, total_rows=1), batch(batch=4096, total_rows=4096)
    assert sizes(c, one, count=1)[1] == 0 and sizes(c, one, count=512)[1] > 8192 and sizes(c, many, count=512)[1] == 0


def test_tensors():
    pool = torch.zeros((8, 4, 2, 32 * 128), dtype=torch.bfloat16)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(ValueError):
        va.KVCache(va.KVType.BF16, pool, pool, 64, 4, 128)  # (host memory: no cache to call with)
    assert P.select(np.ones((1, 2)), np.zeros((9, 2, 2)), [3, -1, 5, 6, 8, 7], 9, 32, 191, 1, 1, 4) == [0, 2, 3, 5]
    assert i32(1).dtype == torch.int32


@pytest.mark.parametrize("kind", [0, 1, 4])
def test_bounds_over_any_part_of_the_cache_are_refused(kind):
    """Keys, values and the scales of either: their first and last bytes, and none that lie right beside."""
    token = 8 * 4 * 64  # pages, key heads, tokens of a page
    size = dict(k=token * {0: 256, 1: 128, 4: 64}[kind])
    size["v"] = size["k"]
    if kind:
        size["k_scales"], size["v_scales"] = token * 4, token * 4  # (FP4: 4 exponents of a byte)
    bounds = 8 * 4 * 2 * 128 * 2
    none = batch(total_rows=0, row_offsets=FAKE)  # (refused all the same, and no launch)
    for name, n in size.items():
        place = {x: (16 + i) * BIG for i, x in enumerate(size)}
        for at, want in ((0, INVALID), (n - 16, INVALID), (16 - bounds, INVALID), (n, OK), (-bounds, OK)):
            c = cache(kv_type=kind, **{**place, name: 2 * BIG - at})
            assert calls(c, none, bounds=2 * BIG)[0] == want, (name, at)


@pytest.mark.parametrize("bad,says", [(dict(select=4), "context"), (dict(context=64, select=4, sinks=3), "sinks"),
                                      (dict(context=64, select=4, window=9), "window"), (dict(context=64, select=2), "keep"),
                                      (dict(context=64, select=-1), "keep"), (dict(context=64, select=4, keep_last=0), "keep"),
                                      (dict(context=64, select=4, keep_first=-1), "keep")])
def test_a_stack_refuses_a_selection_that_it_could_not_follow(bad, says):
    from viper_amd.stack import Stack
    with pytest.raises(ValueError, match=says):  # (before it lays anything out)
        Stack(torch, hidden=512, inter=1024, n_heads=8, n_kv_heads=2, head_dim=64, layers=1, passes=1, vocab=64, **bad)


@pytest.mark.parametrize("kind", ["bf16", "int8", "fp4"])
def test_scores_bound_the_keys_of_their_pages(kind):
    """A page's score, unrounded, against q . k of each of its keys as attention takes them: at least that for bf16 and FP4; int8
    keys are bounded after a rounding to bf16 (half a step, 2^-8 of the value), and some do lie above."""
    D, page, pages = 64, 32, 40
    rng = np.random.default_rng(9)
    c = F.make_cache(kind, pages, page, 1, D, rng)
    near = np.zeros((pages, 1, 2, D))
    table = [np.arange(pages)]
    P.bounds(c, table, [pages * page], pages * page, None, near)
    k = c.rows(table[0], np.arange(pages * page), 0, True).reshape(pages, page, D)
    q = R.bf16_val(R.bf16_bits(rng.standard_normal((500, D)))).astype(np.float64)
    q = np.concatenate([q, np.sign(k[:, 0]), np.sign(k[:, 1])])  # (along a key's own signs: nearest to the bound)
    over = -np.inf
    for p in range(pages):
        score = np.maximum(q * near[p, 0, 0], q * near[p, 0, 1]).sum(1)
        dot, size = q @ k[p].T, np.abs(q) @ np.abs(k[p]).T
        slack = 2.0 ** -8 * size if kind == "int8" else 0.0
        assert np.all(dot <= score[:, None] + slack + D * 2.0 ** -52 * size)  # (sums in 64 bits)
        one = q * k[p, 0]  # of a page that holds one key alone
        r = R.bf16_val(R.bf16_bits(k[p, 0].astype(np.float32))).astype(np.float64)
        over = max(over, (one.sum(1) - (q * r).sum(1)).max())
    assert (over > 1e-6) == (kind == "int8")
