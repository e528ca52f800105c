"""Plain 64-bit implementations (numpy, CPU) of page bounds, page selection and attention over lists of pages, from the header's
definitions, for caches of decode_ref and fp4_ref."""
import math

import numpy as np

import decode_ref as R


def keys(cache, pg, at, head):
    """bf16 values of the keys at places `at` of page pg as kv_read gives them back, float64 [len(at), D]."""
    at = np.asarray(at)
    if hasattr(cache, "held"):
        return cache.held(np.full(len(at), pg), at, head, True)
    k = cache.rows(np.full(1, pg), at, head, True)  # (a table of that page alone)
    return R.bf16_val(R.bf16_bits(k.astype(np.float32))).astype(np.float64)


def touched(lens, rows, offs, page):
    """(sequence, page number, tokens held there) of every page with a new row."""
    out = []
    for b, n in enumerate(lens):
        new = rows if offs is None else offs[b + 1] - offs[b]
        if new == 0 or n <= 0:
            continue
        for c in range(max(0, n - new) // page, -(-n // page)):
            out.append((b, c, min(page, n - c * page)))
    return out


def bounds(cache, table, lens, rows, offs, out):
    """out float64 [pages, kvh, 2, D], changed in place."""
    for b, c, n in touched(lens, rows, offs, cache.page):
        pg = int(table[b][c]) if c < len(table[b]) else -1
        if not 0 <= pg < cache.pages:
            continue
        for h in range(cache.kvh):
            k = keys(cache, pg, np.arange(n), h)
            bad = np.isnan(k).any(0)
            out[pg, h, 0], out[pg, h, 1] = np.where(bad, np.nan, k.min(0)), np.where(bad, np.nan, k.max(0))


def select(q, near, table_row, pages, page, p, first, last, count):
    """The list of one row and key head: q float64 [G, D], near float64 [pages, 2, D] of the head."""
    n = 0 if p < 0 else min(p // page + 1, len(table_row))
    score = {}
    for c in range(n):
        pg = int(table_row[c])
        if 0 <= pg < pages:
            with np.errstate(all="ignore"):
                lo, hi = q * near[pg, 0], q * near[pg, 1]
                s = np.float32(np.max([math.fsum(x) if np.isfinite(x).all() else x.sum() for x in np.maximum(lo, hi)]))
            score[c] = math.inf if np.isnan(s) else float(s)
    keep = [c for c in range(n) if c < first or c >= n - last]
    ranked = sorted((c for c in score if c not in keep), key=lambda c: (-score[c], c))
    keep = sorted(keep + ranked[:count - len(keep)])
    return keep + [-1] * (count - len(keep))


def attention(cache, table, lens, max_rows, offs, q, heads, scale, lists):
    """(o, bound) as decode_ref.attention over the tokens of the listed pages; lists int [rows][kvh][count]."""
    D, G, page = cache.D, heads // cache.kvh, cache.page
    out, bound = {}, {}
    for b, r, p in R.row_map(lens, max_rows, offs):
        o, bd = np.zeros((heads, D)), np.zeros((heads, D))
        for h in range(cache.kvh if p >= 0 else 0):
            pages = [int(c) for c in lists[r][h] if 0 <= c <= p // page]
            if not pages:
                continue
            if p >= len(table[b]) * page or any(not 0 <= table[b][c] < cache.pages for c in pages):
                o[h * G:(h + 1) * G] = np.nan
                continue
            j = np.concatenate([np.arange(c * page, min((c + 1) * page, p + 1)) for c in pages])
            k, v = cache.rows(table[b], j, h, True), cache.rows(table[b], j, h, False)
            for x in range(h * G, (h + 1) * G):
                qq = R.bf16_val(q[r, x * D:(x + 1) * D]).astype(np.float64)
                with np.errstate(all="ignore"):
                    s = scale * (k @ qq)
                    w = np.exp(s - np.max(s))
                    w /= w.sum()
                    o[x] = w @ v
                    size = scale * (np.abs(k) @ np.abs(qq))
                    # (the terms of decode_ref.attention's bound)
                    e = 2 * D * 2.0 ** -24 * size.max() + 8 * 2.0 ** -23 * np.abs(s).max() + 2.0 ** -15 + len(j) * 2.0 ** -28
                    bd[x] = 2.0 ** -8 * np.abs(o[x]) + e * (w @ np.abs(v)) + 1e-38
        out[r], bound[r] = o, bd
    return out, bound
