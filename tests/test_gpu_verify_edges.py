"""verify_draft at the ends of the temperatures' range, against the plain 64-bit implementation."""
import numpy as np
import pytest

import decode_ref as R
from test_gpu_verify import check, inputs, run

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FLT_MAX = float(np.finfo(np.float32).max)


@pytest.mark.parametrize("T", [1e30, 1e34, 1e36, 1e38, FLT_MAX])
@pytest.mark.parametrize("point", [False, True])
def test_logits_ruled_out_stay_out_at_any_temperature(T, point):
    """-inf weighs nothing and an infinite largest logit leaves nothing to finite ones, however flat the rest is."""
    rng = np.random.default_rng(20)
    V = 9000
    t, d, tokens, _ = inputs(rng, 6, 3, V, point)
    t[0, :, 1:] = 0xFF80                                     # one token is allowed
    t[1, :, ::2] = 0xFF80
    t[2, :, [17, 8200]] = 0x7F80                             # two infinite ones share
    t[3, :, 4000] = 0x7F80
    t[3, :, ::3] = 0xFF80
    t[4, :, 5] = R.bf16_bits(np.float32([3.38e38]))[0]       # the largest finite values
    t[4, :, 6] = R.bf16_bits(np.float32([-3.38e38]))[0]
    if d is not None:
        d[1, :, 1::2] = 0xFF80
        d[5, :, 100] = 0x7F80
    tokens[1] = 4                                            # a ruled-out token was drafted
    tokens[2] = 17
    temp = np.full(6, T, np.float32)
    for x in (0.0, 0.3, 0.62, 0.9, 1 - 2.0 ** -24):
        u = np.minimum(rng.uniform(0, 1, (6, 3)).astype(np.float32), np.float32(1 - 2.0 ** -24))
        u[:, -1] = x
        out, _ = check(t, d, tokens, None, u, temp)
        for b, row in enumerate(out):
            for i, tok in enumerate(row):
                assert tok < 0 or t[b, i, tok] != 0xFF80, (T, b, i, tok)


def test_small_logits_at_small_temperatures():
    """Logits below the normal range keep their differences, and zeros of either sign are one value."""
    T = np.float32(1e-36)
    t = R.bf16_bits(np.float32([0.0, -0.0]))[None, None].copy()
    for x, want in ((0.499, 0), (0.501, 1)):
        out, _, _ = run(t, None, None, None, np.array([[x]], np.float32), np.array([T]), probs=False)
        assert out.tolist() == [[want]], (x, want)
    rng = np.random.default_rng(21)
    for scale in (1e-35, 1e-36, 3e-38, 1e-39):
        t, d, tokens, u = inputs(rng, 4, 4, 3001)
        t, d = (R.bf16_bits((R.bf16_val(x) * np.float32(scale)).astype(np.float32)) for x in (t, d))
        for _ in range(3):
            u = np.minimum(rng.uniform(0, 1, u.shape).astype(np.float32), np.float32(1 - 2.0 ** -24))
            check(t, d, tokens, None, u, np.full(4, T, np.float32))
            check(t, None, tokens, None, u, np.full(4, T, np.float32))


def test_the_smallest_temperatures_take_ordinary_logits():
    rng = np.random.default_rng(22)
    t, d, tokens, u = inputs(rng, 4, 4, 3001)
    for T in (1e-20, 1e-30, 1e-38, 1.5e-45):
        check(t, d, tokens, None, u, np.full(4, T, np.float32))
        check(t, None, tokens, None, u, np.full(4, T, np.float32))
