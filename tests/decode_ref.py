"""Plain 64-bit implementations (numpy, CPU) of the paged cache, its attention and the verification of drafted tokens,
written from their definitions, for the tests of viper_amd.decode."""
import math

import numpy as np


def bf16_bits(x):
    """fp32 values -> bf16 bit patterns, round to nearest even (finite, infinite and NaN)."""
    u = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where((u & 0x7FFFFFFF) > 0x7F800000, np.uint16(0x7FC0), r)


def bf16_val(b):
    return (np.asarray(b, dtype=np.uint16).astype(np.uint32) << 16).view(np.float32)


def k_place(t, d, i8):
    s, m, g = t // 4 % 2, 4 * (t // 8) + t % 4, d // 8 % 4
    if i8:
        return 1024 * (2 * (d // 64) + s) + 16 * (16 * g + m) + 8 * (d // 32 % 2) + d % 8
    return 512 * (2 * (d // 32) + s) + 8 * (16 * g + m) + d % 8


def v_place(t, d, i8):
    if i8:
        return 1024 * (d // 32) + 16 * (16 * (t // 8) + d % 16) + 8 * (d // 16 % 2) + t % 8
    return 512 * (d // 16) + 8 * (16 * (t // 8) + d % 16) + t % 8


class Cache:
    """Pools as flat arrays: bf16 bits (uint16) or int8 codes with fp32 scales."""

    def __init__(self, i8, pages, page, kvh, D, rng=None, std=1.0):
        self.i8, self.pages, self.page, self.kvh, self.D = i8, pages, page, kvh, D
        n = pages * kvh * page * D
        self.ks = self.vs = None
        if i8:
            draw = lambda: rng.integers(-127, 128, n).astype(np.int8) if rng is not None else np.zeros(n, np.int8)
            self.k, self.v = draw(), draw()
            sc = lambda: (rng.uniform(0.004, 0.03, pages * kvh * page) if rng is not None
                          else np.zeros(pages * kvh * page)).astype(np.float32)
            self.ks, self.vs = sc(), sc()
        else:
            draw = lambda: bf16_bits(std * rng.standard_normal(n, dtype=np.float32)) if rng is not None else np.zeros(n, np.uint16)
            self.k, self.v = draw(), draw()

    def places(self, pg, at, head, is_k):
        """Element numbers of the row of token `at` (0..page-1) on page pg."""
        d = np.arange(self.D)
        block = (pg * self.kvh + head) * (self.page // 32) + at // 32
        return block * 32 * self.D + (k_place if is_k else v_place)(at % 32, d, self.i8)

    def scale_at(self, pg, at, head):
        return (pg * self.kvh + head) * self.page + at

    def rows(self, table_row, j, head, is_k):
        """Tokens j of a sequence as float64 [len(j), D]."""
        pool, sc = (self.k, self.ks) if is_k else (self.v, self.vs)
        pg, at = np.asarray(table_row)[j // self.page], j % self.page
        d = np.arange(self.D)[None, :]
        block = (pg * self.kvh + head) * (self.page // 32) + at // 32
        e = pool[(block * 32 * self.D)[:, None] + (k_place if is_k else v_place)((at % 32)[:, None], d, self.i8)]
        if self.i8:
            return e.astype(np.float64) * sc[(pg * self.kvh + head) * self.page + at].astype(np.float64)[:, None]
        return bf16_val(e).astype(np.float64)


def row_map(lens, max_rows, offs):
    """[(sequence, row number, position)] of every row of a call."""
    out = []
    for b, n in enumerate(lens):
        r0, r1 = (b * max_rows, (b + 1) * max_rows) if offs is None else (offs[b], offs[b + 1])
        out += [(b, r, int(n) - (r1 - r0) + i) for i, r in enumerate(range(r0, r1))]
    return out


def sees(p, window, sinks):
    j = np.arange(p + 1)
    return j if not window else j[(j > p - window) | (j < sinks)]


def attention(cache, table, lens, max_rows, offs, q, heads, scale, window=0, sinks=0):
    """(o, bound): float64 [rows, heads, D] by row number (dict), and how far a kernel may be off.

    The bound, per output value: half a step of its rounding to bf16, 2^-8 |o|, and sum_j w_j |v_j| times the relative error of
    weights.  A score is a sum of D products in 32 bits: off by at most D 2^-24 scale sum |q k| =: e, so its weight by 2 e
    (numerator and denominator); the exponential, the scale and the argument's reduction add a few 2^-23 times the largest
    |score|; the weights are given to the product in 16 bits (2^-16); sums over L tokens run in lanes and parts, at most L / 32
    additions after each other (L 2^-28)."""
    D, G = cache.D, heads // cache.kvh
    out, bound = {}, {}
    for b, r, p in row_map(lens, max_rows, offs):
        o, bd = np.zeros((heads, D)), np.zeros((heads, D))
        if p >= 0:
            j = sees(p, window, sinks)
            for h in range(cache.kvh):
                k, v = cache.rows(table[b], j, h, True), cache.rows(table[b], j, h, False)
                for x in range(h * G, (h + 1) * G):
                    qq = bf16_val(q[r, x * D:(x + 1) * D]).astype(np.float64)
                    with np.errstate(all="ignore"):
                        s = scale * (k @ qq)
                        w = np.exp(s - np.max(s))
                        w /= w.sum()
                        o[x] = w @ v
                        size = scale * (np.abs(k) @ np.abs(qq))
                        e = 2 * D * 2.0 ** -24 * size.max() + 8 * 2.0 ** -23 * np.abs(s).max() + 2.0 ** -15 + len(j) * 2.0 ** -28
                        bd[x] = 2.0 ** -8 * np.abs(o[x]) + e * (w @ np.abs(v)) + 1e-38
        out[r], bound[r] = o, bd
    return out, bound


def rotate(x, p, theta):
    """x float64 [..., D] at position p."""
    D = x.shape[-1]
    a = p * theta ** (-np.arange(0, D, 2) / D)
    lo, hi = x[..., :D // 2], x[..., D // 2:]
    return np.concatenate([lo * np.cos(a) - hi * np.sin(a), hi * np.cos(a) + lo * np.sin(a)], -1)


def quantize_row(x):
    """bf16 values (float32 [D]) -> codes, scale."""
    s = np.float32(max(np.float32(np.abs(x).max()) / np.float32(127.0), np.float32(1e-8)))
    return np.rint(x.astype(np.float32) / s).astype(np.int8), s


def weights(logits, T):
    """p of one row, float64: NaN weighs nothing, nothing above -inf is token 0, infinite logits share, T = 0 is the first largest."""
    l = np.asarray(logits, dtype=np.float64)
    l = np.where(np.isnan(l), -np.inf, l)
    M = l.max()
    w = np.zeros(len(l))
    if M == -np.inf:
        w[0] = 1.0
        return w
    if T == 0:
        w[int(np.argmax(l))] = 1.0
        return w
    with np.errstate(all="ignore"):
        w = np.where(l == M, 1.0, np.exp((l - M) / T))
    return w / w.sum()


def verify(target, draft, tokens, lens, uniforms, temperature):
    """Lists (out_tokens rows, accepted, accept_probs rows) from float arrays; draft None: certain drafter."""
    B, R, V = target.shape
    outs, counts, probs = [], [], []
    for b in range(B):
        T = 1.0 if temperature is None else float(temperature[b])
        n = R - 1 if lens is None else int(lens[b])
        if not (T >= 0 and math.isfinite(T)) or not 0 <= n < R:
            outs.append([-1] * R)
            counts.append(-1)
            probs.append([0.0] * (R - 1))
            continue
        pr = [0.0] * (R - 1)
        r, stop = 0, False
        for i in range(n):
            d = int(tokens[b][i])
            p, q = 0.0, 1.0
            if 0 <= d < V:
                p = weights(target[b, i], T)[d]
                q = 1.0 if draft is None else weights(draft[b, i], T)[d]
            with np.errstate(all="ignore"):
                pr[i] = min(1.0, p / q if q > 0 else np.inf) if p > 0 else 0.0
            if not stop and float(uniforms[b][i]) * q < p:
                r += 1
            else:
                stop = True
        w = weights(target[b, r], T)
        if r < n:
            if draft is not None:
                q = weights(draft[b, r], T)
            else:
                q = np.zeros(V)
                if 0 <= int(tokens[b][r]) < V:
                    q[int(tokens[b][r])] = 1.0
            left = np.maximum(w - q, 0.0)
            if left.sum() > 0:
                w = left
        c = np.cumsum(w)
        over = np.nonzero((c > max(0.0, float(uniforms[b][R - 1])) * c[-1]) & (w > 0))[0]
        t = int(over[0]) if len(over) else int(np.nonzero(w)[0][-1])
        outs.append([int(x) for x in tokens[b][:r]] + [t] + [-1] * (R - 1 - r) if R > 1 else [t])
        counts.append(r)
        probs.append(pr)
    return outs, counts, probs
