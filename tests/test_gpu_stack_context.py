"""The decode step with its attention (Stack with a context): every slot's attention against the plain 64-bit implementation
over what its cache holds, both launch sequences, a captured step that is replayed, and a draft verified from its logits."""
import numpy as np
import pytest

import decode_ref as R
import viper_amd as va
from test_gpu_attention import check
from test_gpu_kv_cache import back
from viper_amd.stack import Stack

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

SMALL = dict(hidden=512, inter=1024, n_heads=8, n_kv_heads=2, head_dim=64, layers=2, passes=2, vocab=4096)


def bits(t):
    return back(t.contiguous().view(torch.int16))


@pytest.mark.parametrize("kv_type", [va.KVType.BF16, va.KVType.INT8])
@pytest.mark.parametrize("fused", [True, False])
def test_slots_attend_over_their_caches(kv_type, fused):
    s = Stack(torch, **SMALL, context=100, kv_type=kv_type, page_size=32, window=40, sinks=3)
    seen = []
    plain = s.attend

    def attend(l):
        plain(l)
        seen.append((l, bits(s.q), bits(s.attn)))

    s.attend = attend
    for step in range(70):
        del seen[:]
        s._step(fused)
    torch.cuda.synchronize()
    assert s.seq_len.item() == 70 and [l for l, _, _ in seen] == [0, 1, 2, 3]
    i8 = kv_type == va.KVType.INT8
    for l, q, out in seen:
        c = R.Cache(i8, 4, 32, 2, 64)
        g = s.kv[l]
        c.k, c.v = (back(t if i8 else t.view(torch.int16)).ravel() for t in (g.k, g.v))
        if i8:
            c.ks, c.vs = back(g.k_scales).ravel(), back(g.v_scales).ravel()
        o, bound = R.attention(c, np.arange(4)[None, :], [70], 1, None, q, 8, 64 ** -0.5, 40, 3)
        check(out, o, bound, [70], 1, None, l)
    assert torch.isfinite(s.logits.float()).all()


def test_captured_step_follows_the_sequence():
    a, b = (Stack(torch, **SMALL, context=64, page_size=32) for _ in range(2))
    a.step_fused()  # (first use outside the capture)
    b.step_fused()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step_fused()
    for n in range(5):
        graph.replay()
        b.step_fused()
        torch.cuda.synchronize()
        assert a.seq_len.item() == b.seq_len.item() == n + 2
        np.testing.assert_array_equal(bits(a.logits), bits(b.logits))
        assert a.token.item() == b.token.item()
    # past its context the step says so
    for _ in range(64):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.isnan(a.attn.float()).all()


def test_without_a_context_nothing_changes():
    s = Stack(torch, **SMALL)
    before = bits(s.attn)
    s.step_fused()
    torch.cuda.synchronize()
    np.testing.assert_array_equal(bits(s.attn), before)
    assert not hasattr(s, "kv")


def test_a_draft_is_verified_by_the_step_s_logits():
    """Tokens drafted greedily from one step's logits and verified against them: all accepted by the greedy rule."""
    s = Stack(torch, **SMALL, context=64, page_size=32)
    rows = []
    for _ in range(4):
        s.step_fused()
        rows.append((s.logits.clone(), s.token.clone()))
    V = s.V
    target = torch.cat([r[0] for r in rows]).view(1, 4, V)
    tokens = torch.cat([r[1] for r in rows])
    out = torch.zeros((1, 4), dtype=torch.int32, device="cuda")
    acc = torch.zeros((1,), dtype=torch.int32, device="cuda")
    ws = torch.zeros((va.verify_workspace_bytes(1, 4, V),), dtype=torch.uint8, device="cuda")
    u = torch.full((1, 4), 0.5, device="cuda")
    for T, n in ((0.0, 3), (1.0, None)):
        t = torch.full((1,), T, device="cuda")
        assert va.verify_draft(target, tokens[:3].contiguous().view(1, 3), u, out, acc, temperature=t, workspace=ws).ok()
        torch.cuda.synchronize()
        f = R.bf16_val(bits(target)).astype(np.float64)
        wo, wa, _ = R.verify(f, None, tokens[:3].cpu().numpy()[None], None, u.cpu().numpy(), [T])
        assert out.tolist() == wo and acc.tolist() == wa
        assert n is None or (acc.item() == n and out.tolist() == [tokens.tolist()])
