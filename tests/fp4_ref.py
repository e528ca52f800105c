"""Plain 64-bit implementations (numpy, CPU) of the 4-bit cache, written from the header's definitions, for the tests of
viper_amd.decode: a cache with the interface of decode_ref.Cache, so that decode_ref.attention runs over it."""
import numpy as np

import decode_ref as R

MAG = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def value(code):
    code = np.asarray(code).astype(int)
    return np.where(code >= 8, -MAG[code & 7], MAG[code & 7])


def nearest(y):
    """Magnitude of the nearest value to |y| with y's sign, the even code of two; over 6: 6."""
    d = np.abs(np.abs(np.asarray(y, np.float64))[..., None] - MAG)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    pick = np.where(even.any(-1, keepdims=True), even, near)
    return np.copysign((pick * MAG).max(-1), y)


def k_nibble(t, d, D):
    """Element number of (token, dim) in a tile of 32 * D; element e is the low (even) or high half of byte e / 2."""
    s, m = t // 4 % 2, 4 * (t // 8) + t % 4
    if D == 64:
        return 32 * (16 * (d // 16) + m) + 16 * s + d % 16
    return 2048 * (2 * (d // 128) + s) + 32 * (16 * (d // 32 % 4) + m) + d % 32


def v_nibble(t, d):
    return 2048 * (d // 64) + 32 * (16 * (t // 8) + d % 16) + 8 * (d // 16 % 4) + t % 8


def exp_byte(t, c, D):
    """Byte of block c of token t in a tile's D powers of two."""
    s, m = t // 4 % 2, 4 * (t // 8) + t % 4
    return 2 * (16 * c + m) + s if D == 64 else (16 * (c % 4) + m) * (D // 64) + 2 * (c // 4) + s


def quantize_k(x):
    """float64 [..., D] of bf16 values -> (values held [..., D], exponent bytes [..., D / 32])"""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    fine = np.isfinite(b).all(-1)
    amax = np.where(np.isfinite(b), np.abs(b), 0).max(-1)
    e = np.searchsorted(7.0 * 2.0 ** np.arange(-125, 126), amax).clip(0, 250) - 125
    p = 2.0 ** e[..., None].astype(np.float64)
    with np.errstate(all="ignore"):
        held = np.where(fine[..., None], nearest(np.where(np.isfinite(b), b, 0) / p) * p, np.nan)
    return held.reshape(x.shape), np.where(fine, e + 127, 255).astype(np.uint8)


def quantize_v(x):
    """float64 [D] of bf16 values -> (codes' values [D], fp32 scale); a value that is not finite: scale NaN."""
    x = np.asarray(x, np.float64)
    if not np.isfinite(x).all():
        return np.zeros_like(x), np.float32(np.nan)
    s = max(np.float32(np.float32(np.abs(x).max()) / np.float32(6)), np.float32(1e-8))
    return nearest(x.astype(np.float32) / s), s


class Cache4:
    """Pools as flat byte arrays, exponents of keys, scales of values."""
    i8 = False

    def __init__(self, pages, page, kvh, D, rng=None):
        self.pages, self.page, self.kvh, self.D = pages, page, kvh, D
        n = pages * kvh * page
        draw = (lambda lo, hi, n: rng.integers(lo, hi, n).astype(np.uint8)) if rng is not None else (lambda lo, hi, n: np.zeros(n, np.uint8))
        self.k, self.v = draw(0, 256, n * D // 2), draw(0, 256, n * D // 2)
        self.ks = draw(124, 128, n * (D // 32))
        self.vs = (rng.uniform(0.1, 0.5, n) if rng is not None else np.zeros(n)).astype(np.float32)

    def at(self, pg, j, head):
        """(token of its tile, tile of the pool)"""
        return j % 32, (pg * self.kvh + head) * (self.page // 32) + j // 32

    def code(self, pool, e):
        return (pool[e // 2] >> (e % 2 * 4).astype(np.uint8)) & 15

    def held(self, pg, j, head, is_k):
        """Token `j` (0..page-1) of page pg, arrays allowed, float64 [..., D]."""
        t, tile = self.at(np.asarray(pg)[..., None], np.asarray(j)[..., None], head)
        d = np.arange(self.D)
        pool = self.k if is_k else self.v
        x = value(self.code(pool, tile * 32 * self.D + (k_nibble(t, d, self.D) if is_k else v_nibble(t, d))))
        if is_k:
            b = self.ks[tile * self.D + exp_byte(t, d // 32, self.D)].astype(np.float64)
            with np.errstate(all="ignore"):
                return np.where(b == 255, np.nan, x * 2.0 ** (b - 127))
        return x * self.vs[tile * 32 + t].astype(np.float64)

    def rows(self, table_row, j, head, is_k):
        return self.held(np.asarray(table_row)[j // self.page], j % self.page, head, is_k)


def gpu_cache(c, va, dev):
    """The cache on the GPU, from any of the reference caches."""
    if isinstance(c, Cache4):
        shape = (c.pages, c.kvh, c.page)
        return va.KVCache(va.KVType.FP4, dev(c.k), dev(c.v), c.page, c.kvh, c.D, dev(c.ks).view(*shape, c.D // 32), dev(c.vs).view(shape))
    return va.KVCache(va.KVType.INT8 if c.i8 else va.KVType.BF16, dev(c.k), dev(c.v), c.page, c.kvh, c.D,
                      dev(c.ks) if c.i8 else None, dev(c.vs) if c.i8 else None)


def make_cache(kind, pages, page, kvh, D, rng, std=1.0):
    return Cache4(pages, page, kvh, D, rng) if kind == "fp4" else R.Cache(kind == "int8", pages, page, kvh, D, rng, std)
