"""Long contexts in little memory: plain forms, calls and cases of the 4-bit key/value cache and of attention over selected pages.

Kinds of work (`op`), each what a serving program does at a step:
  store   kv_append into a 4-bit cache (keys rotated, then in blocks of 32 dimensions with a power of two each; values with one fp32
          scale per token and head), and kv_read of the same rows
  attn    attention_paged over a 4-bit cache
  bounds  kv_page_bounds: the least and largest key values of every page that the new rows lie on
  select  select_pages: for each new row and key head the pages whose bounds promise the largest scores, with the first and the last ones
  pages   attention_selected: the new rows over the pages of such a list

Codes of 4 bits are e2m1: a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  A tile of 32 tokens is kept in the order in which matrix
instructions take it (`_k_rows`, `_v_rows`).
"""
import math

import torch

own = False

DEV = "cuda"
BF16, INT8, FP4 = 0, 1, 4
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    base = dict(heads=20, kv_heads=4, head_dim=128, page=64, kv=FP4, ragged=False)
    return [
        # the smallest work: one sequence's new token stored and read back
        dict(base, name="store_decode", op="store", batch=1, rows=1, max_len=1000, min_len=1000, theta=10000.0),
        # the prompts of a batch, of uneven lengths
        dict(base, name="store_prompts", op="store", batch=12, rows=1500, ragged=True, max_len=2100, min_len=1500, theta=1e6),
        # one token of a short conversation: latency alone
        dict(base, name="attn_short", op="attn", batch=1, rows=1, max_len=611, min_len=611),
        # one token of one very long document
        dict(base, name="attn_long", op="attn", batch=1, rows=1, max_len=131072, min_len=131072, page=256),
        # a serving batch, lengths spread
        dict(base, name="attn_batch", op="attn", batch=32, rows=1, max_len=16384, min_len=700),
        # drafts verified, ragged, with smaller heads, more of them to a key head, odd lengths
        dict(base, name="attn_verify", op="attn", heads=48, kv_heads=8, head_dim=64, page=32, batch=4, rows=7, ragged=True,
             max_len=9001, min_len=2003),
        # a serving batch's step: the page of each new token again
        dict(base, name="bounds_decode", op="bounds", kv=BF16, batch=16, rows=1, max_len=4000, min_len=100),
        # long prompts just stored in 8 bits: all of their pages
        dict(base, name="bounds_prompts", op="bounds", kv=INT8, batch=3, rows=20000, ragged=True, max_len=20011, min_len=20000, page=32),
        # one token of a very long document: 64 of 2048 pages
        dict(base, name="select_decode", op="select", batch=1, rows=1, max_len=131072, min_len=131072, count=64, first=1, last=2),
        # a batch's drafts over long contexts, smaller pages
        dict(base, name="select_batch", op="select", batch=16, rows=4, ragged=True, max_len=65003, min_len=9000, page=32, count=128,
             first=2, last=4),
        # 64 pages of that document, 16 bits
        dict(base, name="pages_decode", op="pages", kv=BF16, batch=1, rows=1, max_len=131072, min_len=131072, count=64, first=1, last=2),
        # and those of the batch's drafts, 4 bits
        dict(base, name="pages_batch", op="pages", batch=16, rows=4, ragged=True, max_len=65003, min_len=9000, page=32, count=128,
             first=2, last=4),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("store", "attn", "attn", "attn", "bounds", "select", "select", "pages", "pages", "pages"))
    kvh = rng.choice((1, 2, 4, 4, 8))
    c = dict(op=op, kv_heads=kvh, heads=kvh * rng.choice((1, 2, 4, 5, 6, 8)), head_dim=rng.choice((64, 128, 128, 128, 256)),
             page=rng.choice((32, 64, 128, 256)), ragged=rng.random() < 0.5)
    c["kv"] = FP4 if op in ("store", "attn") else rng.choice((BF16, INT8, FP4, FP4))
    row = kvh * c["head_dim"]
    if op in ("store", "bounds"):
        c["batch"] = _log(rng, 1, 64)
        c["rows"] = min(rng.choice((1, 1, 2, 5, 16, 100, 1000, 9000)), max(1, 10000 * 512 // (c["batch"] * max(row, c["heads"] * c["head_dim"] // 5))))
        c["max_len"] = c["rows"] + _log(rng, 1, 3000)
        c["min_len"] = max(c["rows"], c["max_len"] // 3)
        if op == "store":
            c["theta"] = rng.choice((10000.0, 500000.0, 1e6))
        return c
    c["rows"] = rng.choice((1, 1, 1, 2, 3, 4, 5, 8, 13, 16))
    if op == "attn":
        c["batch"] = _log(rng, 1, 48)
        most = min(131072, int(1.3e8 / (c["batch"] * row * max(1, c["rows"] // 4))))  # as many tokens as the serving batch holds
        c["max_len"] = max(c["rows"], _log(rng, 17, max(18, most)))
        c["min_len"] = max(c["rows"], c["max_len"] // rng.choice((1, 2, 9)))
        return c
    c["batch"] = _log(rng, 1, 24)
    c["first"], c["last"] = rng.choice((0, 1, 2, 4)), rng.choice((1, 2, 5))
    c["count"] = c["first"] + c["last"] + _log(rng, 1, 160)
    # as much as the largest listed ones: the lists' tokens, the bounds of the sequences
    while c["batch"] * c["rows"] * c["count"] * c["page"] * row > 40 * 128 * 32 * 512 and c["batch"] * c["rows"] > 1:
        c["batch"], c["rows"] = max(1, c["batch"] // 2), max(1, c["rows"] - 1)
    if c["count"] * c["page"] > 16384:
        c["count"] = 16384 // c["page"]
    most = min(131072, int(c["page"] * 16e6 / (c["batch"] * c["rows"] * row)))
    c["max_len"] = max(c["rows"], _log(rng, 100, max(101, most)))
    if op == "select":  # of more pages than are listed
        c["max_len"] = max(c["max_len"], c["page"] * (c["first"] + c["last"] + 3) + 1)
        c["count"] = min(c["count"], max(c["first"] + c["last"] + 1, c["max_len"] // c["page"] * 2 // 3))
    c["min_len"] = max(c["rows"], c["max_len"] // rng.choice((1, 2, 5)))
    return c


# ----------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _ints(g, lo, hi, shape, dtype=torch.int32):
    return torch.randint(lo, hi + 1, shape, dtype=dtype, device=DEV, generator=g)


def _counts(case):
    """The rows of every sequence of a ragged batch, by the case alone (outputs of one case have one shape)."""
    B, R = case["batch"], case["rows"]
    return [1 + (b * 7919 + 13) % R for b in range(B - 1)] + [R]


def _total(case):
    return sum(_counts(case)) if case["ragged"] else case["batch"] * case["rows"]


def prepare(case, seed):
    g = _gen(seed)
    op, B, R, H, KVH, D, page, kv = (case[k] for k in ("op", "batch", "rows", "heads", "kv_heads", "head_dim", "page", "kv"))
    lens = _ints(g, case["min_len"], case["max_len"], (B,))
    lens[0] = case["max_len"]
    T, offsets = _total(case), None
    if case["ragged"]:
        offsets = torch.tensor([0] + _counts(case), device=DEV).cumsum(0).to(torch.int32)
    # pages dealt out in random order
    W = -(-case["max_len"] // page)
    held = torch.arange(W, device=DEV)[None, :] * page < lens[:, None]
    P, n = B * W + 3, int(held.sum())
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    table[held] = torch.randperm(P, device=DEV, generator=g)[:n].to(torch.int32)
    s = dict(op=op, kv=kv, page=page, rows=R, kv_heads=KVH, head_dim=D, heads=H, table=table, lens=lens, offsets=offsets,
             theta=case.get("theta"), first=case.get("first"), last=case.get("last"), ks=None, vs=None)
    tiles = (P, KVH, page // 32)
    fill = op in ("attn", "bounds", "pages")  # (a selection reads no keys, a store writes its own)
    for name in ("k", "v"):
        if kv == BF16:
            s[name] = torch.randn((*tiles, 32 * D), device=DEV, generator=g, dtype=torch.bfloat16) if fill else \
                torch.zeros((*tiles, 32 * D), device=DEV, dtype=torch.bfloat16)
        elif kv == INT8:
            s[name] = torch.randint(-127, 128, (*tiles, 32 * D), dtype=torch.int8, device=DEV, generator=g) if fill else \
                torch.zeros((*tiles, 32 * D), device=DEV, dtype=torch.int8)
            s[name + "s"] = 0.005 + 0.02 * torch.rand((P, KVH, page), device=DEV, generator=g)
        else:
            s[name] = torch.randint(0, 256, (*tiles, 16 * D), dtype=torch.uint8, device=DEV, generator=g) if fill else \
                torch.zeros((*tiles, 16 * D), device=DEV, dtype=torch.uint8)
    if kv == FP4:  # blocks of keys are largest at 1 to 7, rows of values at 0.6 to 3
        s["ks"] = _ints(g, 125, 127, (P, KVH, page, D // 32), torch.uint8)
        s["vs"] = 0.1 + 0.4 * torch.rand((P, KVH, page), device=DEV, generator=g)
    bf = torch.bfloat16
    if op == "store":  # the rows of one projection: q, k and v side by side; some channels of the keys are larger
        qkv = torch.randn((T, (H + 2 * KVH) * D), device=DEV, generator=g)
        qkv[:, H * D:(H + KVH) * D] *= torch.exp(0.8 * torch.randn((1, KVH * D), device=DEV, generator=g))
        qkv = qkv.to(bf)
        s["q"], s["new_k"], s["new_v"] = qkv[:, :H * D], qkv[:, H * D:(H + KVH) * D], qkv[:, (H + KVH) * D:]
        s["q_out"] = torch.empty((T, H * D), dtype=bf, device=DEV)
        s["k_out"], s["v_out"] = (torch.empty((T, KVH, D), dtype=bf, device=DEV) for _ in range(2))
        return s
    if op != "bounds":
        s["q"] = (1.5 * torch.randn((T, H * D), device=DEV, generator=g)).to(bf)
    if op in ("bounds", "select"):
        mid = torch.randn((P, KVH, 1, D), device=DEV, generator=g)
        reach = 0.5 + 2.0 * torch.rand((P, KVH, 1, D), device=DEV, generator=g)
        s["bounds"] = torch.cat((mid - reach, mid + reach), 2).to(bf)
    if op == "select":
        s["selected"] = torch.empty((T, KVH, case["count"]), dtype=torch.int32, device=DEV)
    if op == "pages":  # a list as select_pages leaves it: the first pages, the last ones, others between them
        n = (_rows(s, T)[1] // page + 1)[:, None, None]
        idx = torch.arange(W, device=DEV)
        key = torch.rand((T, KVH, W), device=DEV, generator=g)
        key = torch.where((idx < case["first"]) | (idx >= n - case["last"]), 2.0, key).masked_fill(idx >= n, -1.0)
        count = min(case["count"], W)
        best = key.topk(count, -1)
        best = torch.where(best.values < 0, W, best.indices).sort(-1).values
        s["selected"] = torch.full((T, KVH, case["count"]), -1, dtype=torch.int32, device=DEV)
        s["selected"][..., :count] = torch.where(best < W, best, -1)
    if op in ("attn", "pages"):
        s["out"] = torch.zeros((T, H * D), dtype=bf, device=DEV)
    return s


# ----------------------------------------------------------------- plain forms


def _rows(s, total):
    """Of every row: its sequence, its position."""
    r = torch.arange(total, device=DEV)
    if s["offsets"] is None:
        seq = r // s["rows"]
        return seq, s["lens"].long()[seq] - s["rows"] + r % s["rows"]
    off = s["offsets"].long()
    seq = torch.searchsorted(off, r, right=True) - 1
    return seq, s["lens"].long()[seq] - (off[seq + 1] - r)


def _values(codes):
    """uint8 [..., n] of two codes each -> fp32 [..., 2 n]"""
    lut = torch.tensor(VALUES + tuple(-x for x in VALUES), device=DEV)
    return torch.stack((lut[(codes & 15).long()], lut[(codes >> 4).long()]), -1).flatten(-2)


def _k_rows(s, pages):
    """Keys of pages [n] as they are held, fp32 [n, page, KVH, D]."""
    D, kv, KVH = s["head_dim"], s["kv"], s["kv_heads"]
    x, n = s["k"][pages], len(pages)
    T = x.shape[2]
    if kv == BF16:  # chunk (kb, s), lane 16 g + 4 a + i, element j: token 8a + 4s + i, dim 32 kb + 8 g + j
        return x.view(n, KVH, T, D // 32, 2, 4, 4, 4, 8).permute(0, 2, 6, 4, 7, 1, 3, 5, 8).reshape(n, 32 * T, KVH, D).float()
    if kv == INT8:  # chunk (kb pair, s), lane, half, element
        x = x.view(n, KVH, T, D // 64, 2, 4, 4, 4, 2, 8).permute(0, 2, 6, 4, 7, 1, 3, 8, 5, 9).reshape(n, 32 * T, KVH, D).float()
        return x * s["ks"][pages].transpose(1, 2)[..., None]
    e = s["ks"][pages].view(n, KVH, T, D)
    if D == 64:  # lane 16 g + 4 a + i, s, 16 dims from 16 g; exponents block, a, i, s
        x = _values(x.view(n, KVH, T, 4, 4, 4, 2, 8)).permute(0, 2, 4, 6, 5, 1, 3, 7)
        e = e.view(n, KVH, T, 2, 4, 4, 2).permute(0, 2, 4, 6, 5, 1, 3)
    else:  # chunk (quad, s), lane, 32 dims from 128 quad + 32 g; exponents g, a, i, quad, s
        x = _values(x.view(n, KVH, T, D // 128, 2, 4, 4, 4, 16)).permute(0, 2, 6, 4, 7, 1, 3, 5, 8)
        e = e.view(n, KVH, T, 4, 4, 4, D // 128, 2).permute(0, 2, 4, 7, 5, 1, 6, 3)
    return (x.reshape(n, 32 * T, KVH, D // 32, 32) * torch.exp2(e.reshape(n, 32 * T, KVH, D // 32, 1).float() - 127.0)).flatten(-2)


def _v_rows(s, pages):
    """Values of pages [n], fp32 [n, page, KVH, D]."""
    D, kv, KVH = s["head_dim"], s["kv"], s["kv_heads"]
    x, n = s["v"][pages], len(pages)
    T = x.shape[2]
    if kv == BF16:  # chunk db, lane 16 g + m, element j: token 8g + j, dim 16 db + m
        return x.view(n, KVH, T, D // 16, 4, 16, 8).permute(0, 2, 4, 6, 1, 3, 5).reshape(n, 32 * T, KVH, D).float()
    if kv == INT8:  # chunk db pair, lane, half, element
        x = x.view(n, KVH, T, D // 32, 4, 16, 2, 8).permute(0, 2, 4, 7, 1, 3, 6, 5).reshape(n, 32 * T, KVH, D).float()
    else:  # chunk db quad, lane, word, token: dim 64 dq + 16 word + m
        x = _values(x.view(n, KVH, T, D // 64, 4, 16, 4, 4)).permute(0, 2, 4, 7, 1, 3, 6, 5).reshape(n, 32 * T, KVH, D)
    return x * s["vs"][pages].transpose(1, 2)[..., None]


def _rotate(x, pos, theta):
    """x [T, heads, D] bf16 -> bf16, in 64 bits."""
    D = x.shape[-1]
    freq = torch.pow(torch.tensor(theta, dtype=torch.float64, device=DEV), -torch.arange(D // 2, dtype=torch.float64, device=DEV) * (2.0 / D))
    a = (pos.double()[:, None] * freq)[:, None, :]
    lo, hi = x[..., :D // 2].double(), x[..., D // 2:].double()
    c, n = torch.cos(a), torch.sin(a)
    return torch.cat((lo * c - hi * n, hi * c + lo * n), -1).float().bfloat16()


def _codes(y):
    """The nearest code of fp32 values, ties to the even one; 7 and the sign's bit 8."""
    a = y.abs()
    c = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    return (c + 8 * (y < 0)).to(torch.uint8)


def _plain_store(s):
    T, H, KVH, D, page = s["q"].shape[0], s["heads"], s["kv_heads"], s["head_dim"], s["page"]
    seq, pos = _rows(s, T)
    pg, tile, t = s["table"].long()[seq, pos // page], pos % page // 32, pos % 32
    q = _rotate(s["q"].reshape(T, H, D), pos, s["theta"]).view(T, H * D)
    k = _rotate(s["new_k"].reshape(T, KVH, D), pos, s["theta"]).float().view(T, KVH, D // 32, 32)
    v = s["new_v"].reshape(T, KVH, D).float()
    # keys: the least power of two that leaves a block's largest value at 7 or under
    f, ex = torch.frexp(k.abs().amax(-1))
    e = torch.where(f > 0, (ex - 3 + (f > 0.875)).clamp(-125, 125), -125)
    k = _codes(torch.ldexp(k, -e[..., None])).view(T, KVH, D)
    vs = (v.abs().amax(-1).double() / 6.0).float().clamp_min(1e-8)
    v = _codes((v.double() / vs[..., None].double()).float())
    # keys: two dims to a byte, a row's bytes and exponents in their places
    k = (k[..., 0::2] + 16 * k[..., 1::2])
    a, sub, i = t // 8, t // 4 % 2, t % 4
    exps = s["ks"].view(*s["k"].shape[:3], D)
    e = (e + 127).to(torch.uint8)
    if D == 64:
        s["k"].view(*s["k"].shape[:3], 4, 4, 4, 2, 8).permute(0, 2, 4, 6, 5, 1, 3, 7)[pg, tile, a, sub, i] = k.view(T, KVH, 4, 8)
        exps.view(*exps.shape[:3], 2, 4, 4, 2).permute(0, 2, 4, 6, 5, 1, 3)[pg, tile, a, sub, i] = e
    else:
        s["k"].view(*s["k"].shape[:3], D // 128, 2, 4, 4, 4, 16).permute(0, 2, 6, 4, 7, 1, 3, 5, 8)[pg, tile, a, sub, i] = \
            k.view(T, KVH, D // 128, 4, 16)
        exps.view(*exps.shape[:3], 4, 4, 4, D // 128, 2).permute(0, 2, 4, 7, 5, 1, 6, 3)[pg, tile, a, sub, i] = e.view(T, KVH, D // 128, 4)
    # values: two tokens to a byte, so one half after the other
    place = s["v"].view(*s["v"].shape[:3], D // 64, 4, 16, 4, 4).permute(0, 2, 4, 7, 1, 3, 6, 5)  # [P, tile, g, byte, KVH, quad, word, m]
    new = v.view(T, KVH, D // 64, 4, 16)
    even = (pos % 2 == 0).nonzero()[:, 0]
    odd = (pos % 2 == 1).nonzero()[:, 0]
    at = (pg[even], tile[even], t[even] // 8, t[even] % 8 // 2)
    place[at] = (place[at] & 0xf0) + new[even]
    at = (pg[odd], tile[odd], t[odd] // 8, t[odd] % 8 // 2)
    place[at] = (place[at] & 0x0f) + 16 * new[odd]
    s["vs"][pg, :, pos % page] = vs
    # and back
    pages, where = torch.unique(pg, return_inverse=True)
    return (q, _k_rows(s, pages)[where, pos % page].bfloat16(), _v_rows(s, pages)[where, pos % page].bfloat16())


def _attend(q, k, v, see, G, D):
    """q [B, R, KVH, G, D], k and v [B, L, KVH, D] fp32, see [B, R, L] -> [B, R, KVH, G, D]"""
    B, R, KVH = q.shape[:3]
    L = k.shape[1]
    qq = q.permute(0, 2, 1, 3, 4).reshape(B, KVH, R * G, D)
    scores = torch.matmul(qq, k.permute(0, 2, 3, 1).contiguous()).view(B, KVH, R, G, L) * (D ** -0.5)
    scores = scores.masked_fill(~see[:, None, :, None, :], -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(w.view(B, KVH, R * G, L), v.permute(0, 2, 1, 3).contiguous())
    return o.view(B, KVH, R, G, D).permute(0, 2, 1, 3, 4)


def _spread(s, T):
    """The rows as [B, R]: (seq, slot, q [B, R, KVH, G, D], position or -1 [B, R])."""
    H, KVH, D, B, R = s["heads"], s["kv_heads"], s["head_dim"], s["table"].shape[0], s["rows"]
    seq, pos = _rows(s, T)
    slot = torch.arange(T, device=DEV) - (s["offsets"].long()[seq] if s["offsets"] is not None else seq * R)
    q = torch.zeros((B, R, H, D), device=DEV)
    q[seq, slot] = s["q"].view(T, H, D).float()
    at = torch.full((B, R), -1, dtype=torch.long, device=DEV)
    at[seq, slot] = pos
    return seq, slot, q.view(B, R, KVH, H // KVH, D), at


def _plain_attn(s):
    T, H, KVH, D, B = s["q"].shape[0], s["heads"], s["kv_heads"], s["head_dim"], s["table"].shape[0]
    seq, slot, q, at = _spread(s, T)
    pages = s["table"].clamp_min(0).long().reshape(-1)
    k, v = (x(s, pages).view(B, -1, KVH, D) for x in (_k_rows, _v_rows))
    see = torch.arange(k.shape[1], device=DEV) <= at[..., None]
    return _attend(q, k, v, see, H // KVH, D).reshape(B, -1, H * D)[seq, slot].bfloat16()


def _plain_bounds(s):
    B, W = s["table"].shape
    n = s["offsets"].diff().long() if s["offsets"] is not None else torch.full((B,), s["rows"], device=DEV)
    col = torch.arange(W, device=DEV)[None, :]
    lens = s["lens"].long()[:, None]
    b, c = ((col * s["page"] < lens) & (col >= torch.div(lens - n[:, None], s["page"], rounding_mode="floor"))).nonzero().T
    pages = s["table"].long()[b, c]
    k = _k_rows(s, pages).bfloat16().float()
    past = (c[:, None] * s["page"] + torch.arange(s["page"], device=DEV) >= lens[b])[..., None, None]
    s["bounds"][pages, :, 0] = k.masked_fill(past, math.inf).amin(1).bfloat16()
    s["bounds"][pages, :, 1] = k.masked_fill(past, -math.inf).amax(1).bfloat16()
    return s["bounds"]


def _plain_select(s):
    T, KVH, count, (B, W) = s["q"].shape[0], s["kv_heads"], s["selected"].shape[2], s["table"].shape
    seq, slot, q, at = _spread(s, T)
    D, R, G = s["head_dim"], s["rows"], s["heads"] // KVH
    # in 64 bits: a page at the border is in or out
    near = s["bounds"][s["table"].clamp_min(0).long()].double().permute(0, 2, 3, 4, 1).contiguous()  # [B, KVH, 2, D, W]
    qq = q.double().permute(0, 2, 1, 3, 4).reshape(B, KVH, R * G, D)
    score = torch.matmul(qq.clamp_min(0.0), near[:, :, 1].contiguous()) + torch.matmul(qq.clamp_max(0.0), near[:, :, 0].contiguous())
    score = score.view(B, KVH, R, G, W).amax(3).permute(0, 2, 1, 3)[seq, slot].float()  # [T, KVH, W]
    col = torch.arange(W, device=DEV)
    n = (at[seq, slot] // s["page"] + 1)[:, None, None]
    always = ((col < s["first"]) | (col >= n - s["last"])) & (col < n)
    may = (s["table"] >= 0)[seq][:, None, :] & ~always & (col < n)
    order = torch.where(may, score, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, col.expand_as(order).contiguous())
    chosen = always | (may & (rank < count - always.sum(-1, keepdim=True)))
    out = torch.where(chosen, col, W).sort(-1).values
    if W < count:
        out = torch.cat((out, out.new_full((T, KVH, count - W), W)), -1)
    return torch.where(out < W, out, -1)[..., :count].int()


def _plain_pages(s):
    T, KVH, D, page, H = s["q"].shape[0], s["kv_heads"], s["head_dim"], s["page"], s["heads"]
    seq, pos = _rows(s, T)
    count = s["selected"].shape[2]
    lists = s["selected"].clamp_min(0).long()
    pages, where = torch.unique(s["table"].clamp_min(0).long()[seq[:, None, None], lists], return_inverse=True)  # [T, KVH, count]
    head = torch.arange(KVH, device=DEV)[None, :, None]
    j = (lists[..., None] * page + torch.arange(page, device=DEV)).view(T, KVH, count * page)
    see = (j <= pos[:, None, None]) & (s["selected"] >= 0).repeat_interleave(page, -1)
    k, v = (x(s, pages).transpose(1, 2).contiguous()[where, head].view(T * KVH, count * page, 1, D) for x in (_k_rows, _v_rows))
    q = s["q"].view(T * KVH, 1, 1, H // KVH, D).float()
    return _attend(q, k, v, see.view(T * KVH, 1, -1), H // KVH, D).reshape(T, H * D).bfloat16()


# ----------------------------------------------------------------- a pass


def run(state):
    s = state
    if not own:
        return {"store": _plain_store, "attn": _plain_attn, "bounds": _plain_bounds, "select": _plain_select,
                "pages": _plain_pages}[s["op"]](s)
    import viper_amd as va
    if "cache" not in s:  # a program's own descriptions and workspace, made once
        s["cache"] = va.KVCache(va.KVType(s["kv"]), s["k"], s["v"], s["page"], s["kv_heads"], s["head_dim"], s["ks"], s["vs"])
        s["batch"] = va.KVBatch(s["table"], s["lens"], s["rows"], s["offsets"])
        need = 0
        if s["op"] == "attn":
            need = va.attention_workspace_bytes(s["cache"], s["batch"], s["heads"])
        elif s["op"] == "select":
            need = va.select_workspace_bytes(s["cache"], s["batch"], s["heads"], s["selected"].shape[2])
        elif s["op"] == "pages":
            need = va.attention_selected_workspace_bytes(s["cache"], s["batch"], s["heads"], s["selected"].shape[2])
        s["ws"] = torch.zeros((need,), dtype=torch.uint8, device=DEV)
    cache, batch = s["cache"], s["batch"]
    if s["op"] == "store":
        st = va.kv_append(cache, batch, s["new_k"], s["new_v"], q=s["q"], q_out=s["q_out"], rope_theta=s["theta"])
        if st.ok():
            st = va.kv_read(cache, batch, s["k_out"], s["v_out"])
        out = (s["q_out"], s["k_out"], s["v_out"])
    elif s["op"] == "attn":
        st = va.attention_paged(cache, batch, s["q"], s["out"], workspace=s["ws"])
        out = s["out"]
    elif s["op"] == "bounds":
        st = va.kv_page_bounds(cache, batch, s["bounds"])
        out = s["bounds"]
    elif s["op"] == "select":
        st = va.select_pages(cache, batch, s["q"], s["bounds"], s["selected"], first=s["first"], last=s["last"], workspace=s["ws"])
        out = s["selected"]
    else:
        st = va.attention_selected(cache, batch, s["q"], s["selected"], s["out"], workspace=s["ws"])
        out = s["out"]
    if not st.ok():
        raise RuntimeError(st.message)
    return out


# ----------------------------------------------------------------- what a pass cannot do without


def work(case):
    B, R, H, KVH, D, page, kv = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "head_dim", "page", "kv"))
    T = _total(case)
    keys = {BF16: 2 * D, INT8: D + 4, FP4: D // 2 + D // 32}[kv]  # a token's and head's K, and V, as they are held
    values = {BF16: 2 * D, INT8: D + 4, FP4: D // 2 + 4}[kv]
    mean = (case["min_len"] + case["max_len"]) / 2
    if case["op"] == "store":
        return dict(bytes=int(T * (4 * H * D + 8 * KVH * D + 2 * KVH * (keys + values))), flops=int(T * 3 * (H + KVH) * D))
    if case["op"] == "attn":
        return dict(bytes=int(B * mean * KVH * (keys + values) + 4 * T * H * D), flops=int(4 * T * H * D * mean))
    if case["op"] == "bounds":
        tokens = T if R > page else B * page // 2
        return dict(bytes=int(tokens * KVH * keys + max(B, tokens // page) * KVH * 4 * D), flops=int(2 * tokens * KVH * D))
    if case["op"] == "select":
        pages = mean / page
        return dict(bytes=int(B * pages * KVH * 4 * D + T * (2 * H * D + 4 * KVH * case["count"])), flops=int(4 * T * H * D * pages))
    tokens = min(mean, case["count"] * page)
    return dict(bytes=int(T * KVH * (tokens * (keys + values) + 4 * case["count"]) + 4 * T * H * D), flops=int(4 * T * H * D * tokens))


# ----------------------------------------------------------------- from the definitions, in 64 bits


def _code_value(c):
    """Of codes 0 .. 15, from the format's bits: a sign, two of exponent, one of fraction."""
    c = c.long()
    ex, f = c // 2 % 4, (c % 2).double()
    mag = torch.where(ex == 0, 0.5 * f, (1 + 0.5 * f) * torch.exp2((ex - 1).double()))
    return torch.where(c >= 8, -mag, mag)


def _nearest(y):
    """The nearest of the format's values to y in 64 bits, the even code of two."""
    vals = torch.tensor(VALUES, dtype=torch.float64, device=DEV)
    d = (y.abs()[..., None] - vals).abs()
    near = d == d.amin(-1, keepdim=True)
    even = near & (torch.arange(8, device=DEV) % 2 == 0)
    pick = torch.where(even.any(-1, keepdim=True), even, near)
    return torch.copysign((pick * vals).amax(-1), y)


def _token(s, b, j, h, is_k):
    """Tokens j of sequence b for key head h, [len(j), D] in 64 bits, by each value's place in the pool."""
    D, KVH, page, kv = s["head_dim"], s["kv_heads"], s["page"], s["kv"]
    pg = s["table"][b].long()[torch.div(j, page, rounding_mode="floor")]
    t = (j % 32)[:, None]
    d = torch.arange(D, device=DEV)[None, :]
    block = ((pg * KVH + h) * (page // 32) + j % page // 32)[:, None]
    sub, m = t // 4 % 2, t // 8 * 4 + t % 4
    if is_k and kv == BF16:
        place = (d // 32 * 2 + sub) * 512 + (d // 8 % 4 * 16 + m) * 8 + d % 8
    elif is_k and kv == INT8:
        place = (d // 64 * 2 + sub) * 1024 + (d // 8 % 4 * 16 + m) * 16 + d // 32 % 2 * 8 + d % 8
    elif is_k and D == 64:
        place = 2 * ((d // 16 * 16 + m) * 16 + sub * 8) + d % 16
    elif is_k:
        place = 2 * ((d // 128 * 2 + sub) * 1024 + (d // 32 % 4 * 16 + m) * 16) + d % 32
    elif kv == BF16:
        place = d // 16 * 512 + (t // 8 * 16 + d % 16) * 8 + t % 8
    elif kv == INT8:
        place = d // 32 * 1024 + (t // 8 * 16 + d % 16) * 16 + d // 16 % 2 * 8 + t % 8
    else:
        place = 2 * (d // 64 * 1024 + (t // 8 * 16 + d % 16) * 16 + d // 16 % 4 * 4) + t % 8
    place = block * (32 * D) + place
    pool = s["k" if is_k else "v"].reshape(-1)
    if kv == BF16:
        return pool[place].double()
    if kv == INT8:
        return pool[place].double() * s["ks" if is_k else "vs"].reshape(-1)[block * 32 + t].double()
    x = _code_value((pool[place // 2] >> (place % 2 * 4).to(torch.uint8)) & 15)
    if not is_k:
        return x * s["vs"].reshape(-1)[block * 32 + t].double()
    bk = d // 32
    if D == 64:
        at = (bk * 16 + m) * 2 + sub
    else:
        at = ((bk % 4 * 16 + m) * (D // 128) + bk // 4) * 2 + sub
    return x * torch.exp2(s["ks"].reshape(-1)[block * D + at].double() - 127)


def _turned(x, pos, theta):
    D = x.shape[-1]
    a = torch.outer(pos.double(), torch.exp(torch.arange(0, D, 2, device=DEV, dtype=torch.float64) * (-math.log(theta) / D)))
    z = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * torch.polar(torch.ones_like(a), a)[:, None]
    return torch.cat((z.real, z.imag), -1)


def _exact_store(s, pos):
    T, H, KVH, D = len(pos), s["heads"], s["kv_heads"], s["head_dim"]
    q = _turned(s["q"].reshape(T, H, D), pos, s["theta"]).reshape(T, H * D)
    k = _turned(s["new_k"].reshape(T, KVH, D), pos, s["theta"]).float().bfloat16().double().view(T, KVH, D // 32, 32)
    most = 7.0 * torch.exp2(torch.arange(-125, 126, dtype=torch.float64, device=DEV))
    e = torch.searchsorted(most, k.abs().amax(-1)).clamp_max(250).double() - 125
    k = _nearest(k / torch.exp2(e)[..., None]) * torch.exp2(e)[..., None]
    v = s["new_v"].reshape(T, KVH, D).double()
    step = (v.abs().amax(-1, keepdim=True) / 6).float().clamp_min(1e-8).double()
    return q, k.reshape(T, KVH, D), _nearest((v / step).float().double()) * step


def exact(case, seed):
    s = prepare(case, seed)
    B, R, H, KVH, D, page = s["table"].shape[0], s["rows"], s["heads"], s["kv_heads"], s["head_dim"], s["page"]
    G = H // KVH
    lens = s["lens"].tolist()
    off = s["offsets"].tolist() if s["offsets"] is not None else [b * R for b in range(B + 1)]
    pos = torch.cat([torch.arange(lens[b] - (off[b + 1] - off[b]), lens[b], device=DEV) for b in range(B)])
    if s["op"] == "store":
        return _exact_store(s, pos)
    if s["op"] == "bounds":
        out = s["bounds"].double()
        table = s["table"].tolist()
        if off[-1] * KVH > 300000:  # (a page at a time)
            return None
        for b in range(B):
            for c in range((lens[b] - (off[b + 1] - off[b])) // page, -(-lens[b] // page)):
                j = torch.arange(c * page, min(lens[b], (c + 1) * page), device=DEV)
                for h in range(KVH):
                    k = _token(s, b, j, h, True)
                    out[table[b][c], h, 0], out[table[b][c], h, 1] = k.min(0).values, k.max(0).values
        return out
    if s["op"] == "select":
        lists = []
        for b in range(B):
            near = s["bounds"].double()[s["table"][b].clamp_min(0).long()]  # [W, KVH, 2, D]
            for r in range(off[b], off[b + 1]):
                p = int(pos[r])
                n = p // page + 1
                for h in range(KVH):
                    q = s["q"][r].double().view(H, D)[h * G:(h + 1) * G]
                    score = torch.maximum(q[:, None] * near[None, :n, h, 0], q[:, None] * near[None, :n, h, 1]).sum(-1).amax(0).float()
                    keep = {x for x in range(n) if x < s["first"] or x >= n - s["last"]}
                    ranked = sorted((x for x in range(n) if x not in keep), key=lambda x, v=score.tolist(): (-v[x], x))
                    keep |= set(ranked[:s["selected"].shape[2] - len(keep)])
                    lists.append(sorted(keep) + [-1] * (s["selected"].shape[2] - len(keep)))
        return torch.tensor(lists, dtype=torch.int32).view(off[-1], KVH, -1)
    if s["op"] == "attn" and sum(lens) * KVH * D > 1 << 31:
        return None
    out = torch.empty((off[-1], H, D), dtype=torch.float64, device=DEV)
    for b in range(B):
        for h in range(KVH):
            if s["op"] == "attn":
                j = torch.arange(lens[b], device=DEV)
                k, v = (_token(s, b, j, h, is_k) for is_k in (True, False))
            for r in range(off[b], off[b + 1]):
                p = int(pos[r])
                if s["op"] == "pages":
                    pages = s["selected"][r, h]
                    j = (pages[pages >= 0].long()[:, None] * page + torch.arange(page, device=DEV)).reshape(-1)
                    k, v = (_token(s, b, j[j <= p], h, is_k) for is_k in (True, False))
                n = p + 1 if s["op"] == "attn" else len(k)
                q = s["q"][r].double().view(H, D)[h * G:(h + 1) * G]
                out[r, h * G:(h + 1) * G] = torch.softmax((q @ k[:n].T) / math.sqrt(D), -1) @ v[:n]
    return out.view(off[-1], H * D)
