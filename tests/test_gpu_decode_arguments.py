"""What the Python calls of the cache, attention and verification refuse on the GPU, and that a refused call writes nothing."""
import numpy as np
import pytest

import viper_amd as va
from test_gpu_attention import setup
from test_gpu_kv_cache import SENT, back, dev, gpu_cache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def verify_args(B=2, R=3, V=104):
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt, device="cuda")
    return dict(target_logits=z(B, R, V, dt=torch.bfloat16), draft_tokens=z(B, R - 1), uniforms=z(B, R, dt=torch.float32),
                out_tokens=z(B, R) - 7, out_accepted=z(B) - 7, draft_logits=z(B, R - 1, V, dt=torch.bfloat16), draft_lens=z(B),
                temperature=z(B, dt=torch.float32), accept_probs=z(B, R - 1, dt=torch.float32),
                workspace=z(va.verify_workspace_bytes(B, R, V), dt=torch.uint8))


@pytest.mark.parametrize("name", ["target_logits", "draft_logits", "draft_tokens", "uniforms", "out_tokens", "out_accepted",
                                  "draft_lens", "temperature", "accept_probs"])
def test_verify_refuses_elements_of_another_type(name):
    ok = verify_args()
    other = {torch.bfloat16: torch.float16, torch.float32: torch.int32, torch.int32: torch.float32}[ok[name].dtype]
    with pytest.raises(ValueError, match="elements"):
        va.verify_draft(**{**ok, name: ok[name].to(other)})
    assert torch.all(ok["out_tokens"] == -7) and torch.all(ok["out_accepted"] == -7)
    assert va.verify_draft(**ok).ok()


def test_rows_of_another_type():
    c, table, offs, total, q, batch = setup(128, False, 64, 2, 4, [90, 50], 1)
    g = gpu_cache(c)
    out = dev(np.full((2, 512), SENT))
    half = lambda n: torch.zeros((2, n), dtype=torch.float16, device="cuda")
    good = lambda n: torch.zeros((2, n), dtype=torch.bfloat16, device="cuda")
    for call in (lambda: va.attention_paged(g, batch, half(512), out), lambda: va.attention_paged(g, batch, good(512), half(512)),
                 lambda: va.kv_append(g, batch, half(256), good(256)), lambda: va.kv_append(g, batch, good(256), half(256)),
                 lambda: va.kv_append(g, batch, good(256), good(256), q=half(512), q_out=half(512), rope_theta=1e4),
                 lambda: va.kv_read(g, batch, half(256), good(256)), lambda: va.kv_read(g, batch, good(256), half(256))):
        with pytest.raises(ValueError, match="bf16 elements"):
            call()
    assert np.all(back(out) == SENT) and np.array_equal(back(g.k), c.k) and np.array_equal(back(g.v), c.v)


def test_rows_of_another_shape():
    """Rows by head instead of by token, and tensors that are no rows."""
    c, table, offs, total, q, batch = setup(128, False, 64, 4, 4, [90, 50], 1)
    g = gpu_cache(c)
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")
    out = z(2, 512)
    for bad in (z(4, 2, 128), z(2, 128, 4), z(4, 256)):
        assert va.kv_read(g, batch, bad, z(2, 4, 128)).code == va.StatusCode.SHAPE_MISMATCH
        assert va.kv_read(g, batch, z(2, 4, 128), bad).code == va.StatusCode.SHAPE_MISMATCH
    for fine in (z(2, 4, 128), z(2, 512), z(1024), z(1, 1024)):
        assert va.kv_read(g, batch, fine, z(2, 4, 128)).ok()
    for call in (lambda: va.attention_paged(g, batch, z(1024), out), lambda: va.attention_paged(g, batch, out, z(1024)),
                 lambda: va.kv_append(g, batch, z(1024), out), lambda: va.kv_append(g, batch, out, out, q=z(1024), q_out=out, rope_theta=1e4)):
        with pytest.raises(ValueError, match="rows"):
            call()


def test_a_window_that_leaves_32_bits():
    """A window of 2^32 tokens hides nothing: it is refused rather than taken for one of 0 or of a few tokens."""
    c, table, offs, total, q, batch = setup(128, False, 64, 2, 4, [90, 50], 1)
    g = gpu_cache(c)
    out = dev(np.full((2, 512), SENT))
    for kw in (dict(window=1 << 32), dict(window=(1 << 32) + 5), dict(window=1 << 31), dict(window=5, sinks=1 << 32), dict(window=-1),
               dict(window=3, sinks=-1)):
        assert va.attention_paged(g, batch, dev(q), out, **kw).code == va.StatusCode.INVALID_ARGUMENT
    assert np.all(back(out) == SENT)
    assert va.attention_workspace_bytes(g, batch, (1 << 32) + 4) == 0
    assert va.attention_paged(g, batch, dev(q), out, window=2 ** 31 - 1, sinks=2 ** 31 - 1).ok()


def test_overlapping_rows_are_refused_and_no_others():
    """Rows of q and of the output anywhere in one buffer, against a look at every element."""
    rng = np.random.default_rng(50)
    c, table, offs, total, q, _ = setup(64, False, 32, 1, 1, [40] * 6, 1)
    g = gpu_cache(c)
    buf = torch.zeros((6000,), dtype=torch.bfloat16, device="cuda")
    seen = {True: 0, False: 0}
    for _ in range(300):
        n = int(rng.integers(1, 7))
        batch = va.KVBatch(dev(table[:n].copy()), dev(np.full(n, 40, np.int32)), 1)
        strides = [64 + 8 * int(rng.integers(0, 12)) for _ in range(2)]
        if rng.random() < 0.5:
            strides[1] = strides[0]
        at = [8 * int(rng.integers(0, 200)) for _ in range(2)]
        rows = [{a + i * s + e for i in range(n) for e in range(64)} for a, s in zip(at, strides)]
        Q, out = (buf.as_strided((n, 64), (s, 1), a) for a, s in zip(at, strides))
        meet = bool(rows[0] & rows[1])
        st = va.attention_paged(g, batch, Q, out)
        assert st.code == (va.StatusCode.INVALID_ARGUMENT if meet else va.StatusCode.OK), (n, at, strides)
        seen[meet] += 1
        same = at[0] == at[1] and (strides[0] == strides[1] or n == 1)
        kv = torch.zeros((n, 64), dtype=torch.bfloat16, device="cuda")
        st = va.kv_append(g, batch, kv, kv, q=Q, q_out=out, rope_theta=1e4)
        assert st.code == (va.StatusCode.INVALID_ARGUMENT if meet and not same else va.StatusCode.OK), (n, at, strides)
        assert va.kv_append(g, batch, kv, kv, q=Q, q_out=Q, rope_theta=1e4).ok()
        assert va.kv_append(g, batch, Q, Q, q=kv, q_out=out, rope_theta=1e4).ok() != meet, (n, at, strides)
    assert min(seen.values()) > 40


def test_verify_takes_neighbours_in_one_buffer():
    """Everything but the logits side by side in one buffer, with nothing between: nothing overlaps."""
    a = verify_args(B=3, R=4, V=100)
    assert va.verify_draft(**a).ok()
    names = ["draft_tokens", "out_tokens", "draft_lens", "out_accepted", "uniforms", "accept_probs", "temperature"]
    buf = torch.zeros((sum(a[n].numel() for n in names),), dtype=torch.int32, device="cuda")
    at, views = 0, {}
    for n in names:
        views[n] = buf[at:at + a[n].numel()].view(a[n].dtype).view(a[n].shape)
        at += a[n].numel()
    assert va.verify_draft(**{**a, **views}).ok()
    for n in ("out_tokens", "out_accepted", "accept_probs"):
        assert views[n].tolist() == a[n].tolist()
    assert a["out_accepted"].tolist() == [0] * 3 and a["out_tokens"].tolist() == [[0, -1, -1, -1]] * 3
    for x, y in (("out_tokens", "uniforms"), ("accept_probs", "uniforms"), ("out_accepted", "draft_lens")):
        over = views[y].view(torch.int32).flatten()
        if over.numel() == a[x].numel():
            assert va.verify_draft(**{**a, **views, x: over.view(a[x].dtype)}).code == va.StatusCode.INVALID_ARGUMENT
