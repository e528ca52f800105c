"""verify_draft against the plain 64-bit implementation: tokens and counts equal, acceptance probabilities to a 32-bit step."""
import numpy as np
import pytest

import decode_ref as R
import viper_amd as va
from test_gpu_kv_cache import back, dev

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def run(target, draft, tokens, lens, uniforms, temperature, ws=None, stream=None, probs=True):
    """numpy bf16 bits and arrays -> (out_tokens, accepted, accept_probs)"""
    B, Rr, V = target.shape
    out = torch.full((B, Rr), -7, dtype=torch.int32, device="cuda")
    acc = torch.full((B,), -7, dtype=torch.int32, device="cuda")
    pr = torch.full((B, Rr - 1), -7.0, dtype=torch.float32, device="cuda") if probs else None
    ws = torch.zeros((va.verify_workspace_bytes(B, Rr, V),), dtype=torch.uint8, device="cuda") if ws is None else ws
    opt = lambda a: None if a is None else dev(a)
    args = [dev(target), opt(tokens), dev(uniforms)]
    kw = dict(draft_logits=opt(draft), draft_lens=opt(lens), temperature=opt(temperature))
    torch.cuda.synchronize()
    st = va.verify_draft(args[0], args[1], args[2], out, acc, accept_probs=pr, workspace=ws, stream=stream, **kw)
    assert st.ok(), st
    torch.cuda.synchronize()
    assert not np.any(back(ws)[:4096 * 4])  # its counters are zero again
    return out.cpu().numpy(), acc.cpu().numpy(), None if pr is None else pr.cpu().numpy()


def check(target, draft, tokens, lens, uniforms, temperature, **kw):
    out, acc, pr = run(target, draft, tokens, lens, uniforms, temperature, **kw)
    f = lambda x: None if x is None else R.bf16_val(x).astype(np.float64)
    wo, wa, wp = R.verify(f(target), f(draft), tokens, lens, uniforms, temperature)
    np.testing.assert_array_equal(acc, wa)
    np.testing.assert_array_equal(out, wo)
    if pr is not None:
        # 64-bit values rounded once to 32 bits: half a step, 2^-24
        np.testing.assert_allclose(pr, np.array(wp).reshape(pr.shape), rtol=2.0 ** -24 * 1.001, atol=1e-38)
    return out, acc


def inputs(rng, B, Rr, V, point=False, noise=0.7, std=2.5):
    t = std * rng.standard_normal((B, Rr, V))
    d = t[:, :Rr - 1] + noise * rng.standard_normal((B, Rr - 1, V))
    g = -np.log(-np.log(rng.uniform(1e-12, 1, d.shape)))
    tokens = np.argmax(d + g, -1).astype(np.int32) if Rr > 1 else None
    u = rng.uniform(0, 1, (B, Rr)).astype(np.float32)
    u = np.minimum(u, np.float32(1 - 2.0 ** -24))
    return R.bf16_bits(t), None if point or Rr == 1 else R.bf16_bits(d), tokens, u


@pytest.mark.parametrize("V", [1, 2, 7, 8, 500, 4095, 4096, 4097, 4104, 32000, 50257, 166144])
@pytest.mark.parametrize("B,Rr", [(1, 1), (3, 2), (2, 16), (9, 5)])
@pytest.mark.parametrize("point", [False, True])
def test_verify(V, B, Rr, point):
    if V > 5000 and B * Rr > 16 and (B, Rr) != (2, 16):
        B = 3
    print(f"verify V={V} B={B} R={Rr} point={point}", flush=True)
    rng = np.random.default_rng(V * 31 + B * 5 + Rr + point)
    t, d, tokens, u = inputs(rng, B, Rr, V, point)
    temp = rng.uniform(0.3, 1.6, B).astype(np.float32)
    lens = rng.integers(0, Rr, B).astype(np.int32)
    check(t, d, tokens, None, u, None)
    check(t, d, tokens, lens, u, temp)
    check(t, d, tokens, lens, u, np.where(np.arange(B) % 2, temp, 0).astype(np.float32), probs=Rr > 1)


def test_large_vocabulary():
    """More chunks of 4096 logits than a workgroup has threads."""
    rng = np.random.default_rng(77)
    V = 4096 * 300 + 5
    for point in (False, True):
        t, d, tokens, u = inputs(rng, 2, 2, V, point, std=0.5)
        for x in (0.0, 0.25, 0.5, 0.999999):
            u[:, -1] = x
            check(t, d, tokens, None, u, None)


def test_every_border_of_a_small_distribution():
    """Uniforms on and beside each border of the cumulated weights (exact binary fractions)."""
    t = R.bf16_bits(np.log2(np.array([0.25, 0.0, 0.5, 0.125, 0.125]) + 1e-300) * 1.0)[None, None]
    t[0, 0, 1] = 0xFF80
    temp = np.array([1.0 / np.log(2)], np.float32)  # weights 2^l up to a rounding of the temperature
    for u, want in ((0.0, 0), (0.2499, 0), (0.2501, 2), (0.7499, 2), (0.7501, 3), (0.8749, 3), (0.8751, 4), (1 - 2.0 ** -24, 4)):
        out, acc, _ = run(t, None, None, None, np.array([[u]], np.float32), temp, probs=False)
        assert out.tolist() == [[want]] and acc.tolist() == [0]


def test_equal_distributions_accept_everything():
    rng = np.random.default_rng(3)
    t, _, tokens, u = inputs(rng, 4, 6, 5000)
    u[:, :-1] = np.float32(1 - 2.0 ** -24)
    out, acc = check(t, t[:, :5].copy(), tokens, None, u, None)
    assert acc.tolist() == [5] * 4


def test_rows_that_are_not_plain_numbers():
    rng = np.random.default_rng(4)
    V = 9000
    t, d, tokens, u = inputs(rng, 8, 3, V)
    t[0] = 0x7FC0                                            # NaN alone: token 0
    t[1] = 0xFF80                                            # -inf alone
    t[2, :, :] = 0xFF80
    t[2, :, 8191] = R.bf16_bits(np.float32([-3e38]))[0]      # one finite value
    t[3, :, 100] = t[3, :, 5000] = t[3, :, 8999] = 0x7F80    # infinite ones share
    t[4, :, ::2] = 0x7FC0                                    # NaN among numbers
    t[5, :, :8000] = 0xFF80                                  # whole chunks ruled out
    d[6] = 0xFF80
    d[7] = 0x7FC0
    tokens[3] = [5000, 100]
    tokens[6] = [0, 1]
    for _ in range(4):
        u = np.minimum(rng.uniform(0, 1, u.shape).astype(np.float32), np.float32(1 - 2.0 ** -24))
        check(t, d, tokens, None, u, None)
        check(t, None, tokens, None, u, np.full(8, 0.5, np.float32))
        check(t, d, tokens, None, u, np.zeros(8, np.float32))


def test_arguments_on_the_device_that_do_not_fit():
    rng = np.random.default_rng(5)
    t, d, tokens, u = inputs(rng, 6, 4, 700)
    temp = np.array([-1.0, np.nan, np.inf, 1.0, 1.0, 0.5], np.float32)
    lens = np.array([3, 3, 3, 4, -1, 2], np.int32)
    out, acc = check(t, d, tokens, lens, u, temp)
    assert acc[:5].tolist() == [-1] * 5 and np.all(out[:5] == -1) and acc[5] >= 0
    tokens[:, 0] = [-1, 700, 2 ** 31 - 1, -2 ** 31, 0, 699]
    out, acc = check(t, d, tokens, None, u, None)
    assert acc[:4].tolist() == [0] * 4
    check(t, None, tokens, None, u, None)


def test_uniforms_of_zero_and_next_to_one():
    rng = np.random.default_rng(6)
    for std in (0.0, 3.0):
        t, d, tokens, u = inputs(rng, 5, 4, 4097, std=std)
        for x in (0.0, 1 - 2.0 ** -24):
            u[:] = x
            check(t, d, tokens, None, u, None)
            check(t, None, tokens, None, u, None)


def test_greedy_is_the_greedy_pick():
    """Temperature 0 gives, row by row, what sampling_greedy picks."""
    rng = np.random.default_rng(7)
    B, V = 5, 166144
    t, _, _, _ = inputs(rng, B, 1, V)
    t[1, 0, 70000] = t[1, 0, 9] = R.bf16_bits(np.float32([50.0]))[0]
    out, acc, _ = run(t, None, None, None, np.full((B, 1), 0.7, np.float32), np.zeros(B, np.float32), probs=False)
    pick = torch.zeros((B,), dtype=torch.int32, device="cuda")
    assert va.sampling_greedy(dev(t.reshape(B, V)), pick).ok()
    assert out[:, 0].tolist() == pick.tolist() and out[1, 0] == 9


def test_misaligned_rows():
    """An odd vocabulary and logits that start 2 bytes into a buffer."""
    rng = np.random.default_rng(8)
    t, d, tokens, u = inputs(rng, 2, 3, 5001)
    flat = dev(np.concatenate([np.zeros(1, np.uint16), t.ravel()]))[1:].view(2, 3, 5001)
    out = torch.zeros((2, 3), dtype=torch.int32, device="cuda")
    acc = torch.zeros((2,), dtype=torch.int32, device="cuda")
    ws = torch.zeros((va.verify_workspace_bytes(2, 3, 5001),), dtype=torch.uint8, device="cuda")
    assert va.verify_draft(flat, dev(tokens), dev(u), out, acc, draft_logits=dev(d), workspace=ws).ok()
    wo, wa, _ = R.verify(R.bf16_val(t).astype(np.float64), R.bf16_val(d).astype(np.float64), tokens, None, u, None)
    assert out.tolist() == wo and acc.tolist() == wa


def test_one_workspace_streams_and_graphs():
    rng = np.random.default_rng(9)
    ws = torch.zeros((va.verify_workspace_bytes(8, 16, 166144),), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    for B, Rr, V in ((8, 4, 40000), (2, 16, 500), (1, 1, 166144), (8, 4, 40000)):
        t, d, tokens, u = inputs(rng, B, Rr, V)
        check(t, d, tokens, None, u, None, ws=ws, stream=side, probs=Rr > 1)
    t, d, tokens, u = inputs(rng, 4, 5, 32000)
    T, Dr, tk, U = dev(t), dev(d), dev(tokens), dev(u)
    out = torch.zeros((4, 5), dtype=torch.int32, device="cuda")
    acc = torch.zeros((4,), dtype=torch.int32, device="cuda")

    def call():
        assert va.verify_draft(T, tk, U, out, acc, draft_logits=Dr, workspace=ws).ok()

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for i in range(4):
        t, d, tokens, u = inputs(rng, 4, 5, 32000)
        for dst, src in ((T, t), (Dr, d), (tk, tokens), (U, u)):
            dst.copy_(dev(src))
        graph.replay()
        torch.cuda.synchronize()
        wo, wa, _ = R.verify(R.bf16_val(t).astype(np.float64), R.bf16_val(d).astype(np.float64), tokens, None, u, None)
        assert out.tolist() == wo and acc.tolist() == wa
        call()
        torch.cuda.synchronize()
        assert out.tolist() == wo


def test_python_refusals():
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt, device="cuda")
    t = z(2, 3, 100, dt=torch.bfloat16)
    ok = dict(target_logits=t, draft_tokens=z(2, 2), uniforms=z(2, 3, dt=torch.float32), out_tokens=z(2, 3), out_accepted=z(2),
              workspace=z(va.verify_workspace_bytes(2, 3, 100), dt=torch.uint8))
    assert va.verify_draft(**ok).ok()
    for bad in (dict(draft_tokens=z(2, 3)), dict(uniforms=z(2, 2, dt=torch.float32)), dict(out_tokens=z(6, 3)),
                dict(draft_logits=t), dict(draft_lens=z(3)), dict(temperature=z(1, dt=torch.float32)), dict(target_logits=t[0])):
        assert va.verify_draft(**{**ok, **bad}).code == va.StatusCode.SHAPE_MISMATCH
    assert va.verify_draft(**{**ok, "workspace": None}).code == va.StatusCode.INVALID_ARGUMENT
    assert va.verify_draft(**{**ok, "draft_tokens": None}).code == va.StatusCode.INVALID_ARGUMENT
    for bad in (dict(target_logits=t.transpose(0, 1)), dict(uniforms=z(2, 3, dt=torch.float64)), dict(draft_tokens=z(2, 2, dt=torch.int64))):
        with pytest.raises(ValueError):
            va.verify_draft(**{**ok, **bad}) if "target_logits" not in bad else va.verify_draft(
                **{**ok, **bad, "draft_tokens": z(3, 1), "uniforms": z(3, 2, dt=torch.float32), "out_tokens": z(3, 2), "out_accepted": z(3)})


def test_many_odd_rows():
    """Rows of no whole octets, enough of them for the larger chunks."""
    rng = np.random.default_rng(10)
    for point in (False, True):
        t, d, tokens, u = inputs(rng, 8, 16, 50257, point)
        check(t, d, tokens, None, u, np.full(8, 0.8, np.float32))
        check(t, d, tokens, rng.integers(0, 16, 8).astype(np.int32), u, None)


def test_two_calls_at_once():
    """Two streams, a workspace each."""
    rng = np.random.default_rng(11)
    cases = []
    for _ in range(2):
        t, d, tokens, u = inputs(rng, 4, 8, 40000)
        out = torch.zeros((4, 8), dtype=torch.int32, device="cuda")
        acc = torch.zeros((4,), dtype=torch.int32, device="cuda")
        ws = torch.zeros((va.verify_workspace_bytes(4, 8, 40000),), dtype=torch.uint8, device="cuda")
        cases.append((t, d, tokens, u, out, acc, ws, dev(t), dev(d), dev(tokens), dev(u), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for t, d, tokens, u, out, acc, ws, T, D, K, U, st in cases:
            assert va.verify_draft(T, K, U, out, acc, draft_logits=D, workspace=ws, stream=st).ok()
    torch.cuda.synchronize()
    for t, d, tokens, u, out, acc, *_ in cases:
        wo, wa, _ = R.verify(R.bf16_val(t).astype(np.float64), R.bf16_val(d).astype(np.float64), tokens, None, u, None)
        assert out.tolist() == wo and acc.tolist() == wa
