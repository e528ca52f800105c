"""What the cache, attention and verification entry points refuse before any launch, the workspace sizes, and that the plain
64-bit implementation's tile order is a permutation (no GPU)."""
import ctypes as C

import numpy as np
import pytest

import decode_ref as R
import viper_amd as va
from viper_amd.decode import _CBatch, _CCache

FAKE = 0x10000  # never dereferenced: every call below fails validation first, or has no rows
OK, INVALID = 0, 2


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("i8", [False, True])
def test_tile_order_is_a_permutation(D, i8):
    t, d = np.meshgrid(np.arange(32), np.arange(D), indexing="ij")
    for place in (R.k_place, R.v_place):
        assert sorted(place(t, d, i8).ravel().tolist()) == list(range(32 * D))
    # octets of a K row and 8 tokens of a V dim are contiguous
    assert np.all(np.diff(R.k_place(t[:, :8], d[:, :8], i8), axis=1) == 1)
    assert np.all(np.diff(R.v_place(t[:8], d[:8], i8), axis=0) == 1)


def cache(**kw):
    a = dict(kv_type=0, kv_heads=4, head_dim=128, page_size=64, num_pages=8, k=FAKE, v=FAKE, k_scales=None, v_scales=None)
    a.update(kw)
    return _CCache(*a.values())


def batch(**kw):
    a = dict(batch=2, max_rows=1, total_rows=2, table_width=4, block_table=FAKE, seq_lens=FAKE, row_offsets=None)
    a.update(kw)
    return _CBatch(*a.values())


def ref(s):
    return None if s is None else C.addressof(s)


BAD_CACHE = [dict(kv_type=2), dict(kv_type=-1), dict(head_dim=96), dict(head_dim=0), dict(page_size=16), dict(page_size=48),
             dict(page_size=512), dict(kv_heads=0), dict(kv_heads=1025), dict(num_pages=0), dict(k=None), dict(v=None),
             dict(k=FAKE + 8), dict(v=FAKE + 2), dict(k_scales=FAKE, v_scales=FAKE), dict(kv_type=1),
             dict(kv_type=1, k_scales=FAKE), dict(kv_type=1, k_scales=FAKE, v_scales=FAKE + 4)]
BAD_BATCH = [dict(batch=0), dict(batch=65536, total_rows=65536), dict(max_rows=0), dict(total_rows=-1), dict(table_width=0),
             dict(table_width=1 << 26), dict(block_table=None), dict(seq_lens=None), dict(seq_lens=FAKE + 2),
             dict(row_offsets=FAKE + 1), dict(total_rows=3), dict(total_rows=1)]


def calls(c, b, **kw):
    """The status of every entry point over a cache."""
    L = va.lib()
    a = dict(stride=512, q=FAKE, qs=2560, heads=20, theta=1e4, scale=0.1, window=0, sinks=0, out=2 * FAKE, os=2560, ws=None, nws=0)
    a.update(kw)
    return [
        L.viper_hip_kv_append(ref(c), ref(b), FAKE, FAKE, a["stride"], a["q"], a["qs"], a["heads"], a["out"], a["os"], a["theta"],
                              None),
        L.viper_hip_kv_read(ref(c), ref(b), FAKE, FAKE, None),
        L.viper_hip_attention_paged(ref(c), ref(b), a["q"], a["qs"], a["heads"], a["scale"], a["window"], a["sinks"], a["out"],
                                    a["os"], a["ws"], a["nws"], None)]


@pytest.mark.parametrize("bad", BAD_CACHE)
def test_bad_cache(bad):
    assert calls(cache(**bad), batch()) == [INVALID] * 3
    assert va.lib().viper_hip_attention_workspace_bytes(ref(cache(**bad)), ref(batch()), 20) == 0


@pytest.mark.parametrize("bad", BAD_BATCH)
def test_bad_batch(bad):
    assert calls(cache(), batch(**bad)) == [INVALID] * 3


def test_null_descriptions():
    assert calls(None, batch()) == [INVALID] * 3 and calls(cache(), None) == [INVALID] * 3


def test_no_rows_is_no_launch():
    assert calls(cache(), batch(total_rows=0, row_offsets=FAKE)) == [OK] * 3


@pytest.mark.parametrize("bad", [dict(stride=508), dict(stride=504), dict(qs=2552), dict(qs=2564), dict(heads=0), dict(q=FAKE + 2),
                                 dict(out=None), dict(out=FAKE + 8), dict(os=100), dict(theta=-1.0), dict(theta=float("nan")),
                                 dict(theta=0.5), dict(theta=float("inf")), dict(theta=0.0), dict(q=None)])
def test_append_refusals(bad):
    assert calls(cache(), batch(), **bad)[0] == INVALID


@pytest.mark.parametrize("bad", [dict(q=None), dict(q=FAKE + 2), dict(qs=2552), dict(qs=2564), dict(heads=0), dict(heads=18),
                                 dict(heads=-4), dict(heads=4 * 65, qs=4 * 65 * 128, os=4 * 65 * 128), dict(out=None),
                                 dict(out=FAKE + 8), dict(os=100), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                 dict(scale=float("inf")), dict(window=-1), dict(sinks=-1), dict(ws=FAKE, nws=16),
                                 dict(ws=FAKE + 8, nws=1 << 30)])
def test_attention_refusals(bad):
    assert calls(cache(), batch(), **bad)[2] == INVALID


def test_attention_in_place_is_refused():
    assert calls(cache(), batch(), q=FAKE, out=FAKE)[2] == INVALID


def test_attention_rows_are_a_verify_steps():
    b = batch(max_rows=17, total_rows=34)
    assert calls(cache(), b)[2] == INVALID
    assert va.lib().viper_hip_attention_workspace_bytes(ref(cache()), ref(b), 20) == 0


def test_attention_workspace_grows_with_the_length_only_where_it_is_split():
    f = lambda c, b, h: va.lib().viper_hip_attention_workspace_bytes(ref(c), ref(b), h)
    assert f(cache(), batch(batch=1, total_rows=1, table_width=1), 20) == 0          # one part
    long = f(cache(), batch(batch=1, total_rows=1, table_width=2048), 20)
    assert long > 8192 and long % 4 == 0
    assert f(cache(), batch(batch=4096, total_rows=4096, table_width=2048), 20) == 0  # the batch fills the GPU


def verify_call(**kw):
    a = dict(target=FAKE, draft=FAKE, tokens=FAKE, lens=None, u=FAKE, t=None, B=2, R=4, V=1000, out=FAKE, acc=FAKE, probs=None,
             ws=FAKE, nws=1 << 20)
    a.update(kw)
    return va.lib().viper_hip_verify_draft(*a.values(), None)


@pytest.mark.parametrize("bad", [dict(target=None), dict(u=None), dict(out=None), dict(acc=None), dict(tokens=None), dict(B=0),
                                 dict(B=4097), dict(R=0), dict(R=17), dict(V=0), dict(V=1 << 26), dict(ws=None), dict(nws=100),
                                 dict(ws=FAKE + 8), dict(target=FAKE + 1), dict(draft=FAKE + 1), dict(tokens=FAKE + 2),
                                 dict(lens=FAKE + 2), dict(u=FAKE + 2), dict(t=FAKE + 2), dict(out=FAKE + 2), dict(acc=FAKE + 2),
                                 dict(probs=FAKE + 2), dict(B=4096, R=16, V=(1 << 26) - 1, nws=1 << 60),
                                 dict(B=4096, R=1, V=4096 * 1024 + 1, nws=1 << 60)])
def test_verify_refusals(bad):
    assert verify_call(**bad) == INVALID


def test_verify_workspace_bytes():
    assert va.verify_workspace_bytes(0, 4, 1000) == va.verify_workspace_bytes(2, 17, 1000) == 0
    small, large = va.verify_workspace_bytes(1, 1, 10), va.verify_workspace_bytes(8, 16, 166144)
    assert 0 < small < large < 1 << 20


def test_python_refuses_host_tensors():
    import torch
    pool = torch.zeros((2, 4, 2, 32 * 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        va.KVCache(va.KVType.BF16, pool, pool, 64, 4, 128)
    with pytest.raises(ValueError, match="whole pages"):
        va.KVCache(va.KVType.BF16, pool[:, :3], pool[:, :3], 64, 4, 128)
    with pytest.raises(ValueError, match="int32"):
        va.KVBatch(torch.zeros((1, 2), dtype=torch.int64), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="batch"):
        va.KVBatch(torch.zeros((1, 2), dtype=torch.int32), torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="GPU"):
        va.KVBatch(torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


def test_plain_verify_small_cases():
    """The plain implementation against sums done by hand."""
    t = np.log(np.array([[[0.5, 0.25, 0.25], [0.1, 0.2, 0.7]]]))
    d = np.log(np.array([[[0.25, 0.5, 0.25]]]))
    # token 1: p = 0.25, q = 0.5: accepted below 0.5
    assert R.verify(t, d, [[1]], None, [[0.49, 0.05]], None)[:2] == ([[1, 0]], [1])
    assert R.verify(t, d, [[1]], None, [[0.49, 0.5]], None)[:2] == ([[1, 2]], [1])
    # rejected: max(p - q, 0) = (0.25, 0, 0)
    out, acc, pr = R.verify(t, d, [[1]], None, [[0.51, 0.99]], None)
    assert (out, acc) == ([[0, -1]], [0]) and abs(pr[0][0] - 0.5) < 1e-12
    # a certain drafter: accepted below p, else the rest of p
    assert R.verify(t, None, [[0]], None, [[0.51, 0.49]], None)[:2] == ([[1, -1]], [0])
    assert R.verify(t, None, [[0]], None, [[0.51, 0.51]], None)[:2] == ([[2, -1]], [0])
    assert R.verify(t, None, [[0]], [0], [[0.0, 0.6]], None)[:2] == ([[1, -1]], [0])
    assert R.verify(t, d, [[1]], None, [[0.0, 0.0]], [0.0])[:2] == ([[0, -1]], [0])
