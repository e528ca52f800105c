"""Arguments of the cache, attention and verification calls that are refused before any launch (no GPU)."""
import pytest

import viper_amd as va

torch = pytest.importorskip("torch")


def test_verify_draft_refuses_host_tensors():
    """Tensors that are all on the host agree on their device, and their addresses mean nothing on the GPU."""
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt)
    with pytest.raises(ValueError, match="GPU"):
        va.verify_draft(z(2, 3, 100, dt=torch.bfloat16), z(2, 2), z(2, 3, dt=torch.float32), z(2, 3), z(2),
                        workspace=z(va.verify_workspace_bytes(2, 3, 100), dt=torch.uint8))


FAKE = 0x10000  # never dereferenced: every call below fails validation first


def test_a_bound_of_rows_that_leaves_31_bits_is_no_small_grid():
    """max_rows = 2^31 - 1: the tiles of a sequence's rows are counted in 64 bits, and a grid too large is refused."""
    from viper_amd.decode import _CBatch, _CCache
    import ctypes as C
    most = 2 ** 31 - 1
    for D, kvh in ((128, 8), (64, 1), (256, 2)):
        c = _CCache(0, kvh, D, 64, 8, FAKE, FAKE, None, None)
        for batch in (4, 65535):
            b = _CBatch(batch, most, most, 4, FAKE, FAKE, FAKE)
            assert va.lib().viper_hip_kv_read(C.addressof(c), C.addressof(b), FAKE, FAKE, None) == 2
            assert va.lib().viper_hip_kv_append(C.addressof(c), C.addressof(b), FAKE, FAKE, kvh * D, None, 0, 0, None, 0, 0.0,
                                                None) == 2


def test_pools_and_arrays_of_another_type():
    """Elements of the same size that are read as something else are refused before the device is looked at."""
    pool = lambda dt: torch.zeros((2, 4, 2, 32 * 128), dtype=dt)
    scales = torch.zeros((2, 4, 64))
    for kv, bad in ((va.KVType.BF16, torch.float16), (va.KVType.BF16, torch.int8), (va.KVType.BF16, torch.float32),
                    (va.KVType.INT8, torch.bool), (va.KVType.INT8, torch.bfloat16)):
        sc = (scales, scales) if kv == va.KVType.INT8 else (None, None)
        with pytest.raises(ValueError, match="elements"):
            va.KVCache(kv, pool(bad), pool(bad), 64, 4, 128, *sc)
    with pytest.raises(ValueError, match="fp32 elements"):
        va.KVCache(va.KVType.INT8, pool(torch.int8), pool(torch.int8), 64, 4, 128, scales.int(), scales.int())
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    for args in ((i32(1, 2).float(), i32(1)), (i32(1, 2), i32(1).float()), (i32(1, 2), i32(1), 1, i32(2).float())):
        with pytest.raises(ValueError, match="int32"):
            va.KVBatch(*args)


def test_verify_draft_refuses_another_order_of_axes():
    """Tensors that hold as many elements, laid out [R, B] for [B, R]; flat ones and axes of one are taken."""
    z = lambda *s, dt=torch.int32: torch.zeros(s, dtype=dt)
    f32, bf = torch.float32, torch.bfloat16
    B, R, V = 4, 3, 104
    ok = dict(target_logits=z(B, R, V, dt=bf), draft_tokens=z(B, R - 1), uniforms=z(B, R, dt=f32), out_tokens=z(B, R),
              out_accepted=z(B), draft_logits=z(B, R - 1, V, dt=bf), draft_lens=z(B), temperature=z(B, dt=f32),
              accept_probs=z(B, R - 1, dt=f32))
    for bad in (dict(draft_tokens=z(R - 1, B)), dict(uniforms=z(R, B, dt=f32)), dict(out_tokens=z(R, B)),
                dict(draft_logits=z(R - 1, B, V, dt=bf)), dict(draft_logits=z(B, V, R - 1, dt=bf)),
                dict(accept_probs=z(R - 1, B, dt=f32)), dict(out_accepted=z(2, 2)), dict(draft_lens=z(5)), dict(uniforms=z(2, 6, dt=f32))):
        assert va.verify_draft(**{**ok, **bad}).code == va.StatusCode.SHAPE_MISMATCH, bad.keys()
    for fine in ({}, dict(draft_tokens=z(B * (R - 1))), dict(uniforms=z(B, 1, R, dt=f32)), dict(out_accepted=z(B, 1))):
        with pytest.raises(ValueError, match="GPU"):  # (host tensors: what comes after the shapes)
            va.verify_draft(**{**ok, **fine})


def test_scales_of_another_order_of_axes():
    pool, scales = torch.zeros((2, 4, 2, 32 * 128), dtype=torch.int8), torch.zeros((2, 64, 4))
    with pytest.raises(ValueError, match="one scale"):
        va.KVCache(va.KVType.INT8, pool, pool, 64, 4, 128, scales, scales)


def test_numbers_that_leave_32_bits():
    """2^32 + n is not n, and an unknown type is not bf16."""
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    for kw in (dict(max_rows=(1 << 32) + 1), dict(max_rows=1 << 31), dict(max_rows=4, row_offsets=i32(2), total_rows=(1 << 32) + 4)):
        with pytest.raises(ValueError, match="32-bit"):
            va.KVBatch(i32(1, 2), i32(1), **kw)
    pool = torch.zeros((2, 4, 2, 32 * 128), dtype=torch.bfloat16)
    for kv in (1 << 32, 2, -1):
        with pytest.raises(ValueError, match="KVType"):
            va.KVCache(kv, pool, pool, 64, 4, 128)


def test_rows_that_overlap_are_refused():
    from viper_amd.decode import _CBatch, _CCache
    import ctypes as C
    L, c = va.lib(), _CCache(0, 4, 128, 64, 8, FAKE, FAKE, None, None)

    def attn(q, qs, o, os, n=8):
        b = _CBatch(n, 1, n, 4, FAKE, FAKE, None)
        return L.viper_hip_attention_paged(C.addressof(c), C.addressof(b), q, qs, 8, 0.1, 0, 0, o, os, None, 0, None)

    def append(k, v, ks, q, qs, o, os, n=8):
        b = _CBatch(n, 1, n, 4, FAKE, FAKE, None)
        return L.viper_hip_kv_append(C.addressof(c), C.addressof(b), k, v, ks, q, qs, 8, o, os, 1e4, None)

    W, F = 1024, 1 << 30  # 8 heads of 128
    for q, qs, o, os in ((F, W, F, W), (F, W, F + 2 * W, W), (F + 2 * W, W, F, W), (F, W, F + 16, W), (F, 2 * W, F + 2 * W - 16, 2 * W),
                         (F, 2 * W, F - 2 * W + 16, 2 * W), (F, W, F + 2 * 7 * W, W), (F, 2 * W, F + 2 * 7 * W, W),
                         (F, W, F + 2 * W, 2 * W), (F, 2 * W, F + 2 * 3 * W + 16, 3 * W), (F, 1 << 40, F + 2 * (1 << 40), 1 << 40)):
        assert attn(q, qs, o, os) == 2, (q - F, qs, o - F, os)
    assert attn(F, W, F + 2 * W - 16, W, 1) == 2
    K = F << 2
    for k, v, ks, q, qs, o, os in ((K, K, 512, F, W, F + 16, W), (K, K, 512, F, W, F, W + 8), (K, K, 512, F, W, F + 2 * W, W),
                                   (K, K, 512, F, W, K, W), (K, 3 * K, 512, F, W, 3 * K + 7 * 1024, W),
                                   (F + 2 * W - 1024, K, 2048, F, 2048, F, 2048)):
        assert append(k, v, ks, q, qs, o, os) == 2, (k, v, ks, q - F, qs, o - F, os)
    for d in (0, 16, 2 * 512 * 7):
        b = _CBatch(8, 1, 8, 4, FAKE, FAKE, None)
        assert L.viper_hip_kv_read(C.addressof(c), C.addressof(b), F, F + d, None) == 2
        assert L.viper_hip_kv_read(C.addressof(c), C.addressof(b), F + d, F, None) == 2


def test_verify_outputs_that_overlap_are_refused():
    import ctypes as C
    L, M = va.lib(), 1 << 20
    B, R, V = 4, 5, 1000
    ws = va.verify_workspace_bytes(B, R, V)
    ok = dict(target=10 * M, draft=20 * M, tokens=30 * M, lens=31 * M, u=32 * M, t=33 * M, out=34 * M, acc=35 * M, probs=36 * M, ws=40 * M)
    size = dict(target=B * R * V * 2, draft=B * (R - 1) * V * 2, tokens=B * (R - 1) * 4, lens=B * 4, u=B * R * 4, t=B * 4, out=B * R * 4,
                acc=B * 4, probs=B * (R - 1) * 4, ws=ws)
    for x in ("out", "acc", "probs", "ws"):
        for y in ok:
            if x == y:
                continue
            for at in (ok[y], ok[y] + size[y] // 32 * 16, ok[y] + size[y] - 16):
                a = {**ok, x: at}
                assert L.viper_hip_verify_draft(a["target"], a["draft"], a["tokens"], a["lens"], a["u"], a["t"], B, R, V, a["out"], a["acc"],
                                                a["probs"], a["ws"], ws, None) == 2, (x, y, at)


def test_workspace_is_sized_for_the_cache_s_device(monkeypatch):
    """The plan counts the CUs of the device that the call runs on, not of the current one."""
    import ctypes as C
    from types import SimpleNamespace
    from viper_amd import decode
    from viper_amd.decode import _CBatch, _CCache
    c, b = _CCache(0, 4, 128, 64, 8, FAKE, FAKE, None, None), _CBatch(1, 1, 1, 512, FAKE, FAKE, None)
    seen, now = [], [0]

    class Device:
        def __init__(self, n):
            self.n = n

        def __enter__(self):
            now.append(self.n)

        def __exit__(self, *e):
            now.pop()

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[-1])
    monkeypatch.setattr(decode, "lib", lambda: SimpleNamespace(
        viper_hip_attention_workspace_bytes=lambda *a: seen.append(now[-1]) or va.lib().viper_hip_attention_workspace_bytes(*a)))
    for dev in (1, 0):
        n = va.attention_workspace_bytes(SimpleNamespace(_ref=C.addressof(c), _dev=dev), SimpleNamespace(_ref=C.addressof(b)), 20)
        assert n > 8192
    assert seen == [1, 0] and now == [0]
