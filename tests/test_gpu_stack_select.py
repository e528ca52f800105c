"""The decode step over selected pages (Stack with select): every slot's list and attention against the plain implementations over
what its cache and bounds hold, a captured step against the eager one, and a list of all pages against the whole attention."""
import numpy as np
import pytest

import decode_ref as R
import fp4_ref as F
import pages_ref as P
import viper_amd as va
from test_gpu_attention import check
from test_gpu_kv_cache import back
from test_gpu_stack_context import SMALL, bits
from viper_amd.stack import Stack

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
PAGES = 10


def held(kind, g):
    c = F.Cache4(PAGES, 32, 2, 64) if kind == "fp4" else R.Cache(kind == "int8", PAGES, 32, 2, 64)
    c.k, c.v = (back(t if kind != "bf16" else t.view(torch.int16)).ravel() for t in (g.k, g.v))
    if kind != "bf16":
        c.ks, c.vs = back(g.k_scales).ravel(), back(g.v_scales).ravel()
    return c


@pytest.mark.parametrize("kind", ["bf16", "int8", "fp4"])
@pytest.mark.parametrize("fused", [True, False])
def test_slots_attend_over_selected_pages(kind, fused):
    s = Stack(torch, **SMALL, context=PAGES * 32, kv_type=va.KVType[kind.upper()], page_size=32, select=4, keep_first=1, keep_last=1)
    seen, plain = [], s.attend

    def attend(l):
        plain(l)
        seen.append((l, bits(s.q), s.selected.cpu().numpy(), bits(s.attn)))

    s.attend = attend
    for _ in range(300):
        del seen[:]
        s._step(fused)
    torch.cuda.synchronize()
    table, n = np.arange(PAGES)[None, :], 300
    for l, q, lists, out in seen:
        c = held(kind, s.kv[l])
        near = np.zeros((PAGES, 2, 2, 64))
        P.bounds(c, table, [n], n, None, near)
        np.testing.assert_array_equal(R.bf16_val(back(s.bounds[l].view(torch.int16))), near)
        x = R.bf16_val(q[0]).astype(np.float64).reshape(2, 4, 64)
        assert lists[0].tolist() == [P.select(x[h], near[:, h], table[0], PAGES, 32, n - 1, 1, 1, 4) for h in range(2)]
        o, bound = P.attention(c, table, [n], 1, None, q, 8, 64 ** -0.5, lists)
        check(out, o, bound, [n], 1, None, l)
    assert torch.isfinite(s.logits.float()).all()


def test_captured_step_follows_the_sequence():
    a, b = (Stack(torch, **SMALL, context=128, page_size=32, kv_type=va.KVType.FP4, select=3, keep_last=1) for _ in range(2))
    a.step_fused(), b.step_fused()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step_fused()
    for n in range(100):
        graph.replay()
        b.step_fused()
        if n % 20 == 0 or n > 92:
            torch.cuda.synchronize()
            assert a.seq_len.item() == b.seq_len.item() == n + 2
            np.testing.assert_array_equal(bits(a.logits), bits(b.logits))
            assert torch.equal(a.selected, b.selected) and a.token.item() == b.token.item()


def test_all_pages_listed_is_the_whole_context():
    a = Stack(torch, **SMALL, context=96, page_size=32, select=3, keep_last=1)
    b = Stack(torch, **SMALL, context=96, page_size=32)
    for _ in range(90):
        a.step_fused(), b.step_fused()
    # the first slot's caches hold the same rows (its attention is the same sum in another order)
    assert torch.equal(a.kv[0].k, b.kv[0].k) and torch.equal(a.kv[0].v, b.kv[0].v)


def test_a_window_excludes_a_selection():
    with pytest.raises(ValueError, match="window"):
        Stack(torch, **SMALL, context=64, page_size=32, window=10, select=2)


@pytest.mark.parametrize("kind", ["bf16", "int8", "fp4"])
def test_attention_over_all_pages_listed_is_the_whole_contexts(kind):
    """Slot 0 of a stack whose lists hold every page and of one without lists (its inputs are the same at each step): the lists,
    and both attentions within the derived bound of one plain result."""
    kw = dict(context=96, page_size=32, kv_type=va.KVType[kind.upper()])
    a, b = Stack(torch, **SMALL, **kw, select=3, keep_last=1), Stack(torch, **SMALL, **kw)
    seen = {}
    for name, s in (("listed", a), ("whole", b)):
        def attend(l, name=name, s=s, plain=s.attend):
            plain(l)
            if l == 0:
                seen[name] = bits(s.q), bits(s.attn)
        s.attend = attend
    for n in range(1, 97):
        a.step_fused(), b.step_fused()
        held_pages = -(-n // 32)
        assert a.selected.cpu().numpy()[0].tolist() == [list(range(held_pages)) + [-1] * (3 - held_pages)] * 2
        if n not in (1, 2, 31, 32, 33, 64, 65, 95, 96):
            continue
        np.testing.assert_array_equal(seen["listed"][0], seen["whole"][0])
        c = F.Cache4(3, 32, 2, 64) if kind == "fp4" else R.Cache(kind == "int8", 3, 32, 2, 64)
        g = a.kv[0]
        c.k, c.v = (back(t if kind != "bf16" else t.view(torch.int16)).ravel() for t in (g.k, g.v))
        if kind != "bf16":
            c.ks, c.vs = back(g.k_scales).ravel(), back(g.v_scales).ravel()
        o, bound = R.attention(c, np.arange(3)[None, :], [n], 1, None, seen["whole"][0], 8, 64 ** -0.5)
        assert np.abs(o[0]).max() > 0
        for name in seen:
            check(seen[name][1], o, bound, [n], 1, None, (name, n))
