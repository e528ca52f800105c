"""The decode step's operators over a paged key/value cache, and the verification of drafted tokens: plain forms, calls and cases.

Kinds of work (`op`), each one call of a serving program:
  append  kv_append: rotate the new rows' q and k, store k and v in the cache's pages
  read    kv_read: rows of the cache back as bf16 (a prefix that moves to another cache, a check of what is stored)
  attn    attention_paged: the newest 1..16 rows of every sequence over its pages
  verify  verify_draft: accept or reject drafted tokens, sample the token that follows

The cache keeps tiles of 32 tokens in the order in which matrix instructions take them (`_k_view`, `_v_view`), in bf16 or in int8
with one fp32 scale per token and head.
"""
import math

import torch

own = False

DEV = "cuda"
BF16, INT8 = 0, 1


def listed():
    base = dict(heads=20, kv_heads=4, head_dim=128, page=64, kv=BF16, window=0, sinks=0)
    return [
        # the smallest work: one sequence's new token stored, its query rotated
        dict(base, name="append_decode", op="append", batch=1, rows=1, ragged=False, max_len=1000, min_len=1000, theta=10000.0),
        # a batch's verify rows into an 8-bit cache, and read back
        dict(base, name="append_verify_int8", op="append", kv=INT8, batch=64, rows=16, ragged=True, max_len=9000, min_len=40,
             theta=1e6),
        # a long prefix handed to another cache
        dict(base, name="read_prefix", op="read", batch=1, rows=16384, ragged=False, max_len=16384, min_len=16384),
        # several prefixes of an 8-bit cache with smaller heads, lengths that are no whole pages
        dict(base, name="read_ragged_int8", op="read", kv=INT8, heads=8, kv_heads=8, head_dim=64, page=32, batch=8, rows=3000,
             ragged=True, max_len=5000, min_len=3000),
        # one token of a short conversation: latency alone
        dict(base, name="decode_short", op="attn", batch=1, rows=1, ragged=False, max_len=611, min_len=611),
        # one token at an ordinary context
        dict(base, name="decode_4k", op="attn", batch=1, rows=1, ragged=False, max_len=4096, min_len=4096),
        # one token of one very long document
        dict(base, name="decode_long", op="attn", batch=1, rows=1, ragged=False, max_len=131072, min_len=131072, page=256),
        # a serving batch on the 8-bit cache, lengths spread
        dict(base, name="batch_int8", op="attn", kv=INT8, batch=32, rows=1, ragged=False, max_len=16384, min_len=700),
        # a full draft verified: 16 rows a sequence, few sequences
        dict(base, name="verify_rows", op="attn", batch=2, rows=16, ragged=False, max_len=8000, min_len=4100),
        # a window with the first tokens kept, long sequences, more query heads to each key head, ragged drafts
        dict(base, name="window_sinks", op="attn", heads=48, kv_heads=8, batch=16, rows=5, ragged=True, max_len=60000,
             min_len=3000, window=4096, sinks=64),
        # a short draft of a deterministic drafter, a small vocabulary
        dict(name="draft_point", op="verify", batch=1, rows=5, vocab=32000, point=True, ragged=False),
        # full drafts of a batch with the drafter's own probabilities
        dict(name="draft_batch", op="verify", batch=8, rows=16, vocab=166144, point=False, ragged=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "read", "attn", "attn", "attn", "attn", "verify", "verify"))
    if op == "verify":
        c = dict(op=op, batch=_log(rng, 1, 16), rows=rng.randint(2, 16), vocab=_log(rng, 500, 166144),
                 point=rng.random() < 0.4, ragged=rng.random() < 0.5)
        while c["batch"] * c["rows"] * c["vocab"] > 8 * 16 * 166144:
            c["batch"] = max(1, c["batch"] // 2)
            c["rows"] = min(c["rows"], 15)
        return c
    kvh = rng.choice((1, 2, 4, 4, 8))
    c = dict(op=op, kv=rng.choice((BF16, BF16, INT8)), kv_heads=kvh, heads=kvh * rng.choice((1, 2, 4, 5, 6, 8)),
             head_dim=rng.choice((64, 128, 128, 128, 256)), page=rng.choice((32, 64, 128, 256)), window=0, sinks=0,
             ragged=rng.random() < 0.5)
    if op == "attn":
        c["rows"] = rng.choice((1, 1, 1, 2, 3, 4, 5, 8, 13, 16))
        c["batch"] = _log(rng, 1, 48)
        if rng.random() < 0.35:
            c.update(window=_log(rng, 16, 8192), sinks=rng.choice((0, 1, 4, 37, 128)))
        most = min(131072, int(2.6e8 / (c["batch"] * kvh * c["head_dim"] * 4)))  # K and V of a bf16 batch in 260 MB
        c["max_len"] = max(c["rows"], _log(rng, 17, max(18, most)))
        c["min_len"] = max(c["rows"], c["max_len"] // rng.choice((1, 2, 9)))
    elif op == "append":
        c["batch"] = _log(rng, 1, 64)
        c["rows"] = rng.choice((1, 1, 2, 4, 7, 16, 100))
        c["max_len"] = c["rows"] + _log(rng, 1, 2000)
        c["min_len"] = max(c["rows"], c["max_len"] // 3)
        c["theta"] = rng.choice((10000.0, 500000.0, 1e6))
    else:
        c["batch"] = _log(rng, 1, 16)
        c["rows"] = _log(rng, 1, 16384 // c["batch"])
        c["max_len"] = c["rows"] + _log(rng, 1, 500)
        c["min_len"] = c["rows"]
    return c


# ----------------------------------------------------------------- the cache's order


def _k_view(pool, kv, D):
    """[P, KVH, tiles, 32 * D] as [P, tiles, a, s, i, KVH, ...]: token 8a + 4s + i of its tile, the row's D values last in order."""
    P, H, T, _ = pool.shape
    if kv == BF16:  # chunk (kb, s), lane 16 g + 4 a + i, element j: dim 32 kb + 8 g + j
        return pool.view(P, H, T, D // 32, 2, 4, 4, 4, 8).permute(0, 2, 6, 4, 7, 1, 3, 5, 8)
    # chunk (kb pair, s), lane, half, element: dim 64 kp + 32 half + 8 g + j
    return pool.view(P, H, T, D // 64, 2, 4, 4, 4, 2, 8).permute(0, 2, 6, 4, 7, 1, 3, 8, 5, 9)


def _v_view(pool, kv, D):
    """[P, KVH, tiles, 32 * D] as [P, tiles, g, j, KVH, ...]: token 8g + j of its tile, the row's D values last in order."""
    P, H, T, _ = pool.shape
    if kv == BF16:  # chunk db, lane 16 g + m, element j: dim 16 db + m
        return pool.view(P, H, T, D // 16, 4, 16, 8).permute(0, 2, 4, 6, 1, 3, 5)
    # chunk db pair, lane, half, element: dim 32 dp + 16 half + m
    return pool.view(P, H, T, D // 32, 4, 16, 2, 8).permute(0, 2, 4, 7, 1, 3, 6, 5)


def _gather(s, D):
    """K and V of every sequence in fp32, [B, L, KVH, D] over all of its table's pages (pages that it lacks: page 0)."""
    table = s["table"].clamp_min(0).long()
    B, W = table.shape

    def held(pool, view, scales):
        x = view(pool[table.reshape(-1)], s["kv"], D).reshape(B, W * s["page"], pool.shape[1], D).float()
        return x if s["kv"] == BF16 else x * scales[table.reshape(-1)].transpose(1, 2).reshape(B, W * s["page"], pool.shape[1], 1)
    return held(s["k"], _k_view, s["ks"]), held(s["v"], _v_view, s["vs"])


# ----------------------------------------------------------------- inputs


def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), dtype=torch.int32, device=DEV, generator=g)


def _counts(case):
    """The rows of every sequence of a ragged batch, by the case alone (outputs of one case have one shape)."""
    B, R = case["batch"], case["rows"]
    return [1 + (b * 7919 + 13) % R for b in range(B - 1)] + [R]


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "verify":
        B, R, V = case["batch"], case["rows"], case["vocab"]
        # logits as a head gives them, the drafter's near the target's; some entries ruled out
        t = 2.5 * torch.randn((B, R, V), device=DEV, generator=g)
        d = t[:, :-1] + 0.7 * torch.randn((B, R - 1, V), device=DEV, generator=g)
        t[:, :, 3] = -math.inf
        temp = 0.6 + 0.6 * torch.rand((B,), device=DEV, generator=g)
        u = torch.rand((B, R - 1, V), device=DEV, generator=g).clamp_min_(1e-9)
        x = d / temp[:, None, None] if not case["point"] else 3.0 * d
        tokens = (x - torch.log(-torch.log(u))).argmax(-1).to(torch.int32)
        lens = _ints(g, 0 if R > 2 else 1, R - 1, B) if case["ragged"] else None
        return dict(op="verify", target=t.bfloat16(), draft=None if case["point"] else d.bfloat16(), tokens=tokens, lens=lens,
                    uniforms=torch.rand((B, R), device=DEV, generator=g), temperature=temp)
    B, R, H, KVH, D, page, kv = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "head_dim", "page", "kv"))
    lens = _ints(g, case["min_len"], case["max_len"], B)
    lens[0] = case["max_len"]
    offsets, total = None, B * R
    if case["ragged"]:
        n = _counts(case)
        offsets = torch.tensor([0] + n, device=DEV).cumsum(0).to(torch.int32)
        total = sum(n)
    # pages dealt out in random order; with a window those it has left behind are given back
    W = -(-case["max_len"] // page)
    col = torch.arange(W, device=DEV)[None, :]
    first = col * page
    held = first < lens[:, None]
    if case["window"]:
        held &= (first < case["sinks"]) | (first + page > (lens - R - case["window"])[:, None])
    P = int(held.sum()) + 3
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    table[held] = torch.randperm(P, device=DEV, generator=g)[:P - 3].to(torch.int32)
    s = dict(op=case["op"], kv=kv, page=page, rows=R, kv_heads=KVH, head_dim=D, heads=H, table=table, lens=lens, offsets=offsets,
             window=case["window"], sinks=case["sinks"], theta=case.get("theta"))
    shape = (P, KVH, page // 32, 32 * D)
    for name in ("k", "v"):
        if kv == BF16:
            s[name] = torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16)
            s[name + "s"] = None
        else:
            s[name] = torch.randint(-127, 128, shape, dtype=torch.int8, device=DEV, generator=g)
            s[name + "s"] = 0.005 + 0.02 * torch.rand((P, KVH, page), device=DEV, generator=g)
    bf = torch.bfloat16
    if case["op"] == "read":
        s["k_out"], s["v_out"] = (torch.empty((total, KVH, D), dtype=bf, device=DEV) for _ in range(2))
        return s
    if case["op"] == "append":  # the rows of one projection: q, k and v side by side
        qkv = torch.randn((total, (H + 2 * KVH) * D), device=DEV, generator=g).to(bf)
        s["q"], s["new_k"], s["new_v"] = qkv[:, :H * D], qkv[:, H * D:(H + KVH) * D], qkv[:, (H + KVH) * D:]
        s["q_out"] = torch.empty((total, H * D), dtype=bf, device=DEV)
        s["k_out"], s["v_out"] = (torch.empty((total, KVH, D), dtype=bf, device=DEV) for _ in range(2))
        return s
    s["q"] = (1.5 * torch.randn((total, H * D), device=DEV, generator=g)).to(bf)
    s["out"] = torch.zeros((total, H * D), dtype=bf, device=DEV)
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


def _rotate(x, pos, theta):
    """x [T, heads, D] bf16 -> bf16, in 64 bits."""
    D = x.shape[-1]
    freq = torch.pow(torch.tensor(theta, dtype=torch.float64, device=DEV), -torch.arange(D // 2, dtype=torch.float64, device=DEV) * (2.0 / D))
    a = (pos.double()[:, None] * freq)[:, None, :]
    lo, hi = x[..., :D // 2].double(), x[..., D // 2:].double()
    c, n = torch.cos(a), torch.sin(a)
    return torch.cat((lo * c - hi * n, hi * c + lo * n), -1).float().bfloat16()


def _at(s, total):
    seq, pos = _rows(s, total)
    return s["table"].long()[seq, pos // s["page"]], pos % s["page"], pos


def _plain_append(s):
    T, H, KVH, D = s["q"].shape[0], s["heads"], s["kv_heads"], s["head_dim"]
    pg, at, pos = _at(s, T)
    q = _rotate(s["q"].reshape(T, H, D), pos, s["theta"]).view(T, H * D)
    k = _rotate(s["new_k"].reshape(T, KVH, D), pos, s["theta"])
    v = s["new_v"].reshape(T, KVH, D)
    if s["kv"] == INT8:
        kf, vf = k.float(), v.float()
        ks, vs = ((x.abs().amax(-1) / 127.0).clamp_min(1e-8) for x in (kf, vf))
        s["ks"][pg, :, at], s["vs"][pg, :, at] = ks, vs
        k, v = (torch.round(x / y[..., None]).to(torch.int8) for x, y in ((kf, ks), (vf, vs)))
    t = at % 32
    kd = (KVH, D // 32, 4, 8) if s["kv"] == BF16 else (KVH, D // 64, 2, 4, 8)
    vd = (KVH, D // 16, 16) if s["kv"] == BF16 else (KVH, D // 32, 2, 16)
    _k_view(s["k"], s["kv"], D)[pg, at // 32, t // 8, t // 4 % 2, t % 4] = k.view(T, *kd)
    _v_view(s["v"], s["kv"], D)[pg, at // 32, t // 8, t % 8] = v.view(T, *vd)
    return (q, s["k"], s["v"]) if s["kv"] == BF16 else (q, *_plain_read(s))


def _plain_read(s):
    T, KVH, D = s["k_out"].shape[0], s["kv_heads"], s["head_dim"]
    pg, at, _ = _at(s, T)
    t = at % 32
    k = _k_view(s["k"], s["kv"], D)[pg, at // 32, t // 8, t // 4 % 2, t % 4].reshape(T, KVH, D)
    v = _v_view(s["v"], s["kv"], D)[pg, at // 32, t // 8, t % 8].reshape(T, KVH, D)
    if s["kv"] == INT8:
        k = (k.float() * s["ks"][pg, :, at][..., None]).bfloat16()
        v = (v.float() * s["vs"][pg, :, at][..., None]).bfloat16()
    return k, v


def _plain_attn(s):
    T, H, KVH, D = s["q"].shape[0], s["heads"], s["kv_heads"], s["head_dim"]
    G, B, R = H // KVH, s["table"].shape[0], s["rows"]
    seq, pos = _rows(s, T)
    k, v = _gather(s, D)
    L = k.shape[1]
    slot = torch.arange(T, device=DEV) - (s["offsets"].long()[seq] if s["offsets"] is not None else seq * R)
    q = torch.zeros((B, R, H, D), device=DEV)
    q[seq, slot] = s["q"].view(T, H, D).float()
    at = torch.full((B, R), -1, dtype=torch.long, device=DEV)
    at[seq, slot] = pos
    q = q.view(B, R, KVH, G, D).permute(0, 2, 1, 3, 4).reshape(B, KVH, R * G, D)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).view(B, KVH, R, G, L) * (D ** -0.5)
    j = torch.arange(L, device=DEV)
    see = j <= at[..., None]
    if s["window"]:
        see = see & ((j > at[..., None] - s["window"]) | (j < s["sinks"]))
    scores = scores.masked_fill(~see[:, None, :, None, :], -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True).clamp_min(-1e30))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(w.view(B, KVH, R * G, L), v.permute(0, 2, 1, 3).contiguous())
    o = o.view(B, KVH, R, G, D).permute(0, 2, 1, 3, 4).reshape(B, R, H * D)
    return o[seq, slot].bfloat16()


def _softmax64(x, temperature):
    """Over the last axis in 64 bits (values next to a border decide tokens)."""
    x = x.double()
    e = torch.exp((x - x.amax(-1, keepdim=True)) / temperature.double()[:, None, None])
    return e / e.sum(-1, keepdim=True)


def _plain_verify(s):
    B, R, V = s["target"].shape
    p = _softmax64(s["target"], s["temperature"])
    d = s["tokens"].long()
    n = s["lens"].long() if s["lens"] is not None else torch.full((B,), R - 1, dtype=torch.long, device=DEV)
    if s["draft"] is not None:
        q = _softmax64(s["draft"], s["temperature"])
    else:
        q = torch.zeros((B, R - 1, V), dtype=torch.float64, device=DEV).scatter_(2, d[..., None], 1.0)
    i = torch.arange(R - 1, device=DEV)[None, :]
    pd, qd = p[:, :-1].gather(2, d[..., None])[..., 0], q.gather(2, d[..., None])[..., 0]
    u = s["uniforms"].double()
    drafted = i < n[:, None]
    accepted = ((u[:, :-1] * qd < pd) & drafted).long().cumprod(-1).sum(-1)
    ratio = torch.where(drafted & (pd > 0), (pd / qd).clamp_max(1.0), 0.0).float()
    b = torch.arange(B, device=DEV)
    p_r = p[b, accepted]
    q_r = torch.where((accepted < n)[:, None], q[b, accepted.clamp_max(R - 2)], 0.0)
    w = (p_r - q_r).clamp_min(0.0)
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, p_r)
    c = w.cumsum(-1)
    token = (c > u[:, -1:] * c[:, -1:]).long().argmax(-1)
    cols = torch.arange(R, device=DEV)[None, :]
    padded = torch.cat((d, d.new_zeros((B, 1))), 1)
    out = torch.where(cols < accepted[:, None], padded, torch.where(cols == accepted[:, None], token[:, None], -1))
    return out.int(), accepted.int(), ratio


def run(state):
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attn": _plain_attn, "verify": _plain_verify}[state["op"]](state)
    import viper_amd as va
    s = state
    if s["op"] == "verify":
        if "out" not in s:  # a program's own buffers, allocated once
            B, R, V = s["target"].shape
            s["out"] = (torch.empty((B, R), dtype=torch.int32, device=DEV), torch.empty((B,), dtype=torch.int32, device=DEV),
                        torch.empty((B, R - 1), dtype=torch.float32, device=DEV))
            s["ws"] = torch.zeros((va.verify_workspace_bytes(B, R, V),), dtype=torch.uint8, device=DEV)
        out, accepted, ratio = s["out"]
        st = va.verify_draft(s["target"], s["tokens"], s["uniforms"], out, accepted, draft_logits=s["draft"], draft_lens=s["lens"],
                             temperature=s["temperature"], accept_probs=ratio, workspace=s["ws"])
        if not st.ok():
            raise RuntimeError(st.message)
        return s["out"]
    if "cache" not in s:
        s["cache"] = va.KVCache(va.KVType(s["kv"]), s["k"], s["v"], s["page"], s["kv_heads"], s["head_dim"], s["ks"], s["vs"])
        s["batch"] = va.KVBatch(s["table"], s["lens"], s["rows"], s["offsets"])
        if s["op"] == "attn":
            s["ws"] = torch.zeros((va.attention_workspace_bytes(s["cache"], s["batch"], s["heads"]),), dtype=torch.uint8, device=DEV)
    cache, batch = s["cache"], s["batch"]
    if s["op"] == "attn":
        st = va.attention_paged(cache, batch, s["q"], s["out"], window=s["window"], sinks=s["sinks"], workspace=s["ws"])
        out = s["out"]
    elif s["op"] == "read":
        st = va.kv_read(cache, batch, s["k_out"], s["v_out"])
        out = (s["k_out"], s["v_out"])
    else:
        st = va.kv_append(cache, batch, s["new_k"], s["new_v"], q=s["q"], q_out=s["q_out"], rope_theta=s["theta"])
        out = (s["q_out"], s["k"], s["v"])
        if st.ok() and s["kv"] == INT8:
            st = va.kv_read(cache, batch, s["k_out"], s["v_out"])
            out = (s["q_out"], s["k_out"], s["v_out"])
    if not st.ok():
        raise RuntimeError(st.message)
    return out


# ----------------------------------------------------------------- what a pass cannot do without


def work(case):
    if case["op"] == "verify":
        B, R, V = case["batch"], case["rows"], case["vocab"]
        drafted = (R - 1) / 2 if case["ragged"] else R - 1
        logits = B * V * (drafted + 1 + (0 if case["point"] else drafted))
        return dict(bytes=int(2 * logits + B * R * 16), flops=int(8 * logits))
    B, R, H, KVH, D = (case[k] for k in ("batch", "rows", "heads", "kv_heads", "head_dim"))
    rows = sum(_counts(case)) if case["ragged"] else B * R
    token = KVH * (4 * D if case["kv"] == BF16 else 2 * D + 8)  # a token's K and V as they are held
    if case["op"] == "append":
        back = KVH * 4 * D + token if case["kv"] == INT8 else 0
        return dict(bytes=int(rows * (4 * H * D + 4 * KVH * D + token + back)), flops=int(rows * 3 * (H + KVH) * D))
    if case["op"] == "read":
        return dict(bytes=int(rows * (token + 4 * KVH * D)), flops=int(rows * 2 * KVH * D))
    length = (case["min_len"] + case["max_len"]) / 2
    if case["window"]:
        length = min(length, case["window"] + R + case["sinks"])
    return dict(bytes=int(B * length * token + rows * 4 * H * D), flops=int(4 * rows * H * D * length))


# ----------------------------------------------------------------- from the definitions, in 64 bits


def _token(s, pool, b, j, is_k):
    """The values of tokens j of sequence b, [len(j), KVH, D] in 64 bits, by each element's place in the pool."""
    D, KVH, page = s["head_dim"], s["kv_heads"], s["page"]
    pg = s["table"][b].long()[torch.div(j, page, rounding_mode="floor")]
    t = j % 32
    d = torch.arange(D, device=DEV)
    lane16 = d // 8 % 4 * 16 if is_k else t // 8 * 16
    if is_k:
        lane = lane16[None, :] + (t // 8 * 4 + t % 4)[:, None]
        if s["kv"] == BF16:
            place = ((d // 32 * 2)[None, :] + (t // 4 % 2)[:, None]) * 512 + lane * 8 + (d % 8)[None, :]
        else:
            place = ((d // 64 * 2)[None, :] + (t // 4 % 2)[:, None]) * 1024 + lane * 16 + (d // 32 % 2 * 8 + d % 8)[None, :]
    else:
        lane = lane16[:, None] + (d % 16)[None, :]
        if s["kv"] == BF16:
            place = (d // 16 * 512)[None, :] + lane * 8 + (t % 8)[:, None]
        else:
            place = (d // 32 * 1024 + d // 16 % 2 * 8)[None, :] + lane * 16 + (t % 8)[:, None]
    head = torch.arange(KVH, device=DEV)
    block = (pg[:, None] * KVH + head[None, :]) * (page // 32) + (j % page // 32)[:, None]
    return (block * 32 * D)[..., None] + place[:, None, :], pg, block


def _turned(x, pos, theta):
    D = x.shape[-1]
    a = torch.outer(pos.double(), torch.exp(torch.arange(0, D, 2, device=DEV, dtype=torch.float64) * (-math.log(theta) / D)))
    z = torch.complex(x[..., :D // 2].double(), x[..., D // 2:].double()) * torch.polar(torch.ones_like(a), a)[:, None]
    return torch.cat((z.real, z.imag), -1)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "verify":
        B, R, V = s["target"].shape
        tokens, counts, ratios = [], [], []
        for b in range(B):
            n = int(s["lens"][b]) if s["lens"] is not None else R - 1
            T = float(s["temperature"][b].double())
            out, ratio, i = [], [0.0] * (R - 1), 0
            us = s["uniforms"][b].double().tolist()
            drafted = s["tokens"][b].tolist()

            def chances(x):
                return torch.softmax(x.double() / T, -1)

            def q_of(i):
                if s["draft"] is not None:
                    return chances(s["draft"][b, i])
                one = torch.zeros((V,), dtype=torch.float64, device=DEV)
                one[drafted[i]] = 1.0
                return one
            for k in range(n):
                pd, qd = float(chances(s["target"][b, k])[drafted[k]]), float(q_of(k)[drafted[k]])
                ratio[k] = min(1.0, pd / qd) if pd > 0 else 0.0
            while i < n and us[i] * float(q_of(i)[drafted[i]]) < float(chances(s["target"][b, i])[drafted[i]]):
                out.append(drafted[i])
                i += 1
            w = chances(s["target"][b, i])
            if i < n:
                left = torch.relu(w - q_of(i))
                w = left if float(left.sum()) > 0 else w
            c = torch.cumsum(w, 0)
            out.append(int((c > us[-1] * c[-1]).nonzero()[0]))
            tokens.append(out + [-1] * (R - len(out)))
            counts.append(i)
            ratios.append(ratio)
        return (torch.tensor(tokens, dtype=torch.int32), torch.tensor(counts, dtype=torch.int32),
                torch.tensor(ratios, dtype=torch.float64))
    B, R, H, KVH, D = s["table"].shape[0], s["rows"], s["heads"], s["kv_heads"], s["head_dim"]
    lens = s["lens"].tolist()
    off = s["offsets"].tolist() if s["offsets"] is not None else [b * R for b in range(B + 1)]
    if s["op"] == "append":
        pos = torch.cat([torch.arange(lens[b] - (off[b + 1] - off[b]), lens[b], device=DEV) for b in range(B)])
        T = off[-1]
        q = _turned(s["q"].reshape(T, H, D), pos, s["theta"]).reshape(T, H * D)
        k, v = _turned(s["new_k"].reshape(T, KVH, D), pos, s["theta"]), s["new_v"].reshape(T, KVH, D).double()
        if s["kv"] == INT8:
            held = []
            for x in (k.float().bfloat16().double(), v):
                step = (x.abs().amax(-1, keepdim=True).float() / 127.0).clamp_min(1e-8)
                held.append(torch.round((x.float() / step).double()) * step.double())
            return (q, *held)
        pools = [s["k"].double().reshape(-1), s["v"].double().reshape(-1)]
        for b in range(B):
            rows = slice(off[b], off[b + 1])
            for pool, x, is_k in zip(pools, (k, v), (True, False)):
                pool[_token(s, pool, b, pos[rows], is_k)[0]] = x[rows]
        return (q, *(p.view(s["k"].shape) for p in pools))
    if s["op"] == "attn" and sum(lens) * KVH * D > 1 << 31:
        return None
    outs = []
    for b in range(B):
        n = off[b + 1] - off[b]
        if s["op"] == "read":
            j = torch.arange(lens[b] - n, lens[b], device=DEV)
        else:
            j = torch.arange(lens[b], device=DEV)
            if s["window"]:
                j = j[(j < s["sinks"]) | (j > lens[b] - n - s["window"])]
        held = []
        for name, is_k in (("k", True), ("v", False)):
            place, pg, block = _token(s, s[name], b, j, is_k)
            x = s[name].reshape(-1)[place].double()
            if s["kv"] == INT8:
                x *= s[name + "s"].reshape(-1)[block * 32 + (j % 32)[:, None]][..., None].double()
            held.append(x)
        k, v = held
        if s["op"] == "read":
            outs.append(held)
            continue
        q = s["q"][off[b]:off[b + 1]].double().view(n, KVH, H // KVH, D)
        o = torch.empty((n, H, D), dtype=torch.float64, device=DEV)
        for r in range(n):
            p = lens[b] - n + r
            see = j <= p
            if s["window"]:
                see &= (j < s["sinks"]) | (j > p - s["window"])
            for h in range(KVH):
                w = torch.softmax((q[r, h] @ k[see, h].T) / math.sqrt(D), -1)
                o[r, h * (H // KVH):(h + 1) * (H // KVH)] = w @ v[see, h]
        outs.append(o.view(n, H * D))
    if s["op"] == "read":
        return tuple(torch.cat(x) for x in zip(*outs))
    return torch.cat(outs)
