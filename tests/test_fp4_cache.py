"""The 4-bit cache without a GPU: the tile orders are permutations, the reference's rounding, the cache's arguments."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import decode_ref as R
import fp4_ref as F
import viper_amd as va
from test_decode_refusals import FAKE, INVALID, OK, batch, cache, calls, ref

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("D", [64, 128, 256])
def test_tile_orders_are_permutations(D):
    t, d = np.meshgrid(np.arange(32), np.arange(D), indexing="ij")
    for e in (F.k_nibble(t, d, D), F.v_nibble(t, d)):
        assert sorted(e.ravel().tolist()) == list(range(32 * D))
    t, c = np.meshgrid(np.arange(32), np.arange(D // 32), indexing="ij")
    assert sorted(F.exp_byte(t, c, D).ravel().tolist()) == list(range(D))
    # 8 dims of a key and 8 tokens of a value are a word
    d = np.arange(D)
    assert np.all(np.diff(F.k_nibble(5, d, D).reshape(-1, 8)) == 1) and np.all(F.k_nibble(5, d[::8], D) % 8 == 0)
    assert np.all(np.diff(F.v_nibble(np.arange(32).reshape(4, 8), 70 % D)) == 1)


def test_rounding_of_the_reference():
    y = np.array([0, 0.25, 0.26, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 5.01, 7, -0.75, -5.0])
    assert F.nearest(y).tolist() == [0, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6, -1, -4]
    for amax, e in ((7.0, 0), (7.03125, 1), (3.5, -1), (6.0, 0), (0.0, -125), (3e38, 125), (1e-45, -125)):
        held, b = F.quantize_k(np.r_[amax, np.zeros(31)])
        assert b[0] == e + 127, (amax, b)


def fp4(**kw):
    return cache(**{**dict(kv_type=4, k_scales=FAKE, v_scales=FAKE), **kw})


def test_an_fp4_cache_is_a_cache():
    assert calls(fp4(), batch(total_rows=0, row_offsets=FAKE)) == [OK] * 3
    c, b = fp4(), batch(batch=1, total_rows=1, table_width=2048)
    assert va.lib().viper_hip_attention_workspace_bytes(ref(c), ref(b), 20) > 0


@pytest.mark.parametrize("bad", [dict(k_scales=None), dict(v_scales=None), dict(k_scales=FAKE + 8), dict(v_scales=FAKE + 4), dict(k=FAKE + 8),
                                 dict(head_dim=96), dict(kv_type=3), dict(kv_type=5)])
def test_bad_fp4_caches(bad):
    assert calls(fp4(**bad), batch()) == [INVALID] * 3


def test_tensors_of_an_fp4_cache():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    f32 = lambda *s: torch.zeros(s, dtype=torch.float32)
    pool, ks, vs = u8(3, 4, 2, 16 * 128), u8(3, 4, 64, 4), f32(3, 4, 64)
    make = lambda k=pool, v=pool, a=ks, b=vs: va.KVCache(va.KVType.FP4, k, v, 64, 4, 128, a, b)
    for kw in (dict(k=pool.float(), v=pool.float()), dict(a=ks.float()), dict(b=vs.to(torch.uint8)), dict(a=vs), dict(a=ks[..., :3].contiguous()),
               dict(a=u8(3, 64, 4, 4)), dict(b=f32(3, 4, 32)), dict(a=None), dict(k=pool[:2], v=pool), dict(k=pool[:, :3], v=pool[:, :3])):
        with pytest.raises(ValueError):
            make(**kw)
    with pytest.raises(ValueError, match="GPU|device|CUDA"):  # all fits, but for where it is
        make()


@pytest.mark.parametrize("compiler,flags", [("gcc", ["-std=c99", "-x", "c"]), ("g++", ["-std=c++17", "-x", "c++"])])
def test_scales_in_c(compiler, flags):
    """The scales of a cache description are read as floats in C and C++ (int8), and exponents go in by their address (FP4)."""
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    source = """#include "viper_qlinear.h"
        float first(const viper_kv_cache* c) { const float* s = c->k_scales; return s[0] + c->k_scales[1] + c->v_scales[1]; }
        void scales(viper_kv_cache* c, float* k, float* v) { c->k_scales = k; c->v_scales = v; }
        void exponents(viper_kv_cache* c, unsigned char* k) { c->kv_type = VIPER_KV_FP4; c->k_scales = (float*)k; }"""
    p = subprocess.run([compiler, *flags, "-Wall", "-Wextra", "-pedantic", "-Werror", "-fsyntax-only", "-I", include, "-"], input=source,
                       capture_output=True, text=True)
    assert p.returncode == 0, p.stderr


@pytest.mark.parametrize("D,page", [(64, 32), (128, 64), (256, 256)])
def test_exponents_have_the_shape_of_their_tiles(D, page):
    """Tiles of head_dim bytes, whose order within is the header's; the same bytes by rows, and no other shape."""
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)
    pool, vs = u8(3, 4, page // 32, 16 * D), torch.zeros((3, 4, page), dtype=torch.float32)
    make = lambda ks: va.KVCache(va.KVType.FP4, pool, pool, page, 4, D, ks, vs)
    for ks in (u8(3, 4, page // 32, D), u8(3, 4, page, D // 32), u8(12 * page * D // 32)):
        with pytest.raises(ValueError, match="GPU|device|CUDA"):  # all fits, but for where it is
            make(ks)
    for ks in (u8(3, 4, D, page // 32 + 1), u8(4, 3, page // 32, D), u8(3, 2, 2 * page // 32, D), u8(3, 4, page // 32, D // 2)):
        with pytest.raises(ValueError, match="exponent"):
            make(ks)
