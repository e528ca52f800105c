"""The attention side of a decode / verify step, and the verification of drafted tokens (include/viper_qlinear.h).

A ``KVCache`` describes the pages of one layer's keys and values, a ``KVBatch`` the rows of one call: build each once
and pass it to every call (the arrays that a batch points to are read on the device at each launch, so they may be
updated in place between calls, also under a captured graph).  Calls return a ``Status`` as ``linear`` does; tensors that
no call could take raise ``ValueError``.

    cache = KVCache.empty(KVType.BF16, num_pages=512, page_size=64, kv_heads=4, head_dim=128)
    batch = KVBatch(block_table, seq_lens)                   # one new token each; seq_lens counts it
    ws = torch.zeros(attention_workspace_bytes(cache, batch, heads), dtype=torch.uint8, device="cuda")
    kv_append(cache, batch, k, v, q=q, q_out=q, rope_theta=1e6)
    attention_paged(cache, batch, q, out, workspace=ws)
"""
from __future__ import annotations

import ctypes as C
import enum
import math
from dataclasses import dataclass, field
from typing import Any, Optional

from .qlinear import Status, StatusCode, _status, lib, ptr


class KVType(enum.IntEnum):
    BF16 = 0
    INT8 = 1


class _CCache(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("kv_type", "kv_heads", "head_dim", "page_size", "num_pages")] + \
               [(n, C.c_void_p) for n in ("k", "v", "k_scales", "v_scales")]


class _CBatch(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("batch", "max_rows", "total_rows", "table_width")] + \
               [(n, C.c_void_p) for n in ("block_table", "seq_lens", "row_offsets")]


@dataclass
class KVCache:
    """Pages of keys and values of one layer: ``k`` and ``v`` bf16 or int8 tensors of num_pages * kv_heads * page_size *
    head_dim elements (their order within a page: include/viper_qlinear.h), ``k_scales`` and ``v_scales`` fp32
    [num_pages, kv_heads, page_size] for int8."""
    kv_type: KVType
    k: Any
    v: Any
    page_size: int
    kv_heads: int
    head_dim: int
    k_scales: Any = None
    v_scales: Any = None
    num_pages: int = field(init=False, default=0)

    def __post_init__(self):
        size = 1 if int(self.kv_type) == KVType.INT8 else 2
        page = self.kv_heads * self.page_size * self.head_dim
        if page <= 0 or self.k.numel() != self.v.numel() or self.k.numel() % page:
            raise ValueError("KVCache: k and v hold whole pages of kv_heads * page_size * head_dim elements")
        self.num_pages = self.k.numel() // page
        if (self.k_scales is None) != (self.v_scales is None):
            raise ValueError("KVCache: k_scales and v_scales go together")
        if self.k_scales is not None and not (self.k_scales.numel() == self.v_scales.numel() ==
                                              self.num_pages * self.kv_heads * self.page_size):
            raise ValueError("KVCache: one scale for each token and head")
        _one_device(self.k, self.v, self.k_scales, self.v_scales)
        self._c = _CCache(int(self.kv_type), self.kv_heads, self.head_dim, self.page_size, self.num_pages, ptr(self.k, size),
                          ptr(self.v, size), ptr(self.k_scales, 4), ptr(self.v_scales, 4))
        self._ref = C.addressof(self._c)
        self.device = self.k.device

    @classmethod
    def empty(cls, kv_type, num_pages, page_size, kv_heads, head_dim, device="cuda"):
        """A cache of zeroed pages."""
        import torch
        i8 = int(kv_type) == KVType.INT8
        shape = (num_pages, kv_heads, page_size // 32, 32 * head_dim)
        pool = lambda: torch.zeros(shape, dtype=torch.int8 if i8 else torch.bfloat16, device=device)
        scales = lambda: torch.zeros((num_pages, kv_heads, page_size), dtype=torch.float32, device=device) if i8 else None
        return cls(KVType(kv_type), pool(), pool(), page_size, kv_heads, head_dim, scales(), scales())


@dataclass
class KVBatch:
    """The rows of a call: ``block_table`` int32 [batch, table_width], ``seq_lens`` int32 [batch] (tokens held, the call's
    rows among them), and either ``max_rows`` rows for every sequence, or with ``row_offsets`` int32 [batch + 1] the rows
    row_offsets[b]..row_offsets[b + 1] - 1 (at most max_rows) of ``total_rows`` (default: what the row tensors hold)."""
    block_table: Any
    seq_lens: Any
    max_rows: int = 1
    row_offsets: Any = None
    total_rows: Optional[int] = None

    def __post_init__(self):
        if self.block_table.dim() != 2 or self.seq_lens.numel() != self.block_table.shape[0]:
            raise ValueError("KVBatch: block_table is [batch, table_width], seq_lens [batch]")
        self.batch = self.block_table.shape[0]
        if self.row_offsets is not None and self.row_offsets.numel() != self.batch + 1:
            raise ValueError("KVBatch: row_offsets is [batch + 1]")
        if self.row_offsets is None:
            if self.total_rows not in (None, self.batch * self.max_rows):
                raise ValueError("KVBatch: without row_offsets every sequence has max_rows rows")
            self.total_rows = self.batch * self.max_rows
        for t in (self.block_table, self.seq_lens, self.row_offsets):
            if t is not None and (t.is_floating_point() or t.element_size() != 4):
                raise ValueError("KVBatch: int32 arrays")
        _one_device(self.block_table, self.seq_lens, self.row_offsets)
        self._c = _CBatch(self.batch, self.max_rows, self.total_rows or 0, self.block_table.shape[1], ptr(self.block_table, 4),
                          ptr(self.seq_lens, 4), ptr(self.row_offsets, 4))
        self._ref = C.addressof(self._c)
        self.device = self.seq_lens.device

    def _rows(self, n):
        """The C view for row tensors of n rows; None where they do not fit."""
        if self.total_rows is not None:
            return self._ref if n == self.total_rows else None
        self._c.total_rows = n
        return self._ref


def _one_device(*tensors):
    d = [t.device for t in tensors if t is not None]
    if any(x != d[0] for x in d):
        raise ValueError("viper_amd: tensors on more than one device")


def _row_view(t, width):
    """(address, row stride in elements, rows) of a bf16 tensor of rows of `width` values: [rows, width] or [rows, heads,
    head_dim], each row dense, rows any multiple of 8 elements apart (columns of a wider matrix)."""
    if not t.is_cuda:
        raise ValueError("viper_amd: tensor arguments must be GPU tensors")
    if t.element_size() != 2:
        raise ValueError(f"viper_amd: expected 2-byte elements, got {t.dtype}")
    s = t.stride()
    if t.dim() < 2 or t.shape[-1] * (t.shape[1] if t.dim() == 3 else 1) != width or t.dim() > 3 or s[-1] != 1 or \
            (t.dim() == 3 and t.shape[1] > 1 and s[1] != t.shape[2]):
        raise ValueError(f"viper_amd: expected rows of {width} dense values, got {tuple(t.shape)} strides {s}")
    rows = t.shape[0]
    return t.data_ptr(), s[0] if rows > 1 else max(width, s[0] if s[0] % 8 == 0 else width), rows


def _call(fn, what, device, stream, *args) -> Status:
    """The launch on the tensors' device, on `stream` or that device's current one."""
    import torch
    if stream is None or not isinstance(stream, int):
        if stream is not None and stream.device != device:
            return Status(StatusCode.INVALID_ARGUMENT, f"{what}: the stream is on another device")
        if device.index != torch.cuda.current_device():
            with torch.cuda.device(device):
                st = torch.cuda.current_stream() if stream is None else stream
                return _status(fn(*args, st.cuda_stream), what)
        stream = (torch.cuda.current_stream() if stream is None else stream).cuda_stream
    return _status(fn(*args, stream), what)


def _mismatch(what, text) -> Status:
    return Status(StatusCode.SHAPE_MISMATCH, f"{what}: {text}")


def kv_append(cache: KVCache, batch: KVBatch, k, v, q=None, q_out=None, rope_theta: Optional[float] = None,
              stream=None) -> Status:
    """Stores rows k and v ([rows, kv_heads * head_dim], or [rows, kv_heads, head_dim]) in the cache.  With rope_theta, k is
    rotated by its position first and q ([rows, heads * head_dim]) into q_out (may be q)."""
    what = "viper_hip_kv_append"
    if (q is None) != (q_out is None):
        return _mismatch(what, "q and q_out go together")
    width = cache.kv_heads * cache.head_dim
    kp, ks, rows = _row_view(k, width)
    vp, vs, vrows = _row_view(v, width)
    if rows != vrows or (rows > 1 and ks != vs):
        return _mismatch(what, "k and v are laid out alike")
    ref = batch._rows(rows)
    if ref is None:
        return _mismatch(what, "the rows do not match the batch")
    qp = qs = op = os = heads = 0
    if q is not None:
        if rope_theta is None:
            return Status(StatusCode.INVALID_ARGUMENT, f"{what}: q is taken for its rotation")
        qw = q.shape[-1] * (q.shape[1] if q.dim() == 3 else 1)
        heads = qw // cache.head_dim
        qp, qs, qrows = _row_view(q, heads * cache.head_dim)
        op, os, orows = _row_view(q_out, heads * cache.head_dim)
        if qrows != rows or orows != rows:
            return _mismatch(what, "q rows != k rows")
    _one_device(cache, batch, k, v, q, q_out)
    return _call(lib().viper_hip_kv_append, what, cache.device, stream, cache._ref, batch._ref, kp, vp, ks, qp or None, qs, heads,
                 op or None, os, float(rope_theta or 0.0))


def kv_read(cache: KVCache, batch: KVBatch, k_out, v_out, stream=None) -> Status:
    """The batch's rows back from the cache: k_out and v_out bf16 [rows, kv_heads, head_dim]."""
    what = "viper_hip_kv_read"
    width = cache.kv_heads * cache.head_dim
    if k_out.numel() != v_out.numel() or k_out.numel() % width or batch._rows(k_out.numel() // width) is None:
        return _mismatch(what, "the rows do not match the batch")
    _one_device(cache, batch, k_out, v_out)
    return _call(lib().viper_hip_kv_read, what, cache.device, stream, cache._ref, batch._ref, ptr(k_out, 2), ptr(v_out, 2))


def attention_workspace_bytes(cache: KVCache, batch: KVBatch, heads: int) -> int:
    """Bytes of workspace (zero before its first use) that lets attention_paged split the cache's length over workgroups;
    0 where the batch alone fills the GPU."""
    return int(lib().viper_hip_attention_workspace_bytes(cache._ref, batch._ref, heads))


def attention_paged(cache: KVCache, batch: KVBatch, q, out, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
                    workspace=None, stream=None) -> Status:
    """out = attention of the rows q ([rows, heads * head_dim], heads a multiple of the cache's) over their sequences' pages:
    causal; with window > 0 the newest `window` tokens and the first `sinks`.  scale defaults to head_dim ** -0.5."""
    what = "viper_hip_attention_paged"
    heads = q.shape[-1] * (q.shape[1] if q.dim() == 3 else 1) // cache.head_dim
    qp, qs, rows = _row_view(q, heads * cache.head_dim)
    op, os, orows = _row_view(out, heads * cache.head_dim)
    if orows != rows or batch._rows(rows) is None:
        return _mismatch(what, "the rows do not match the batch")
    _one_device(cache, batch, q, out, workspace)
    ws, nws = (None, 0) if workspace is None or workspace.numel() == 0 else \
        (ptr(workspace), workspace.numel() * workspace.element_size())
    return _call(lib().viper_hip_attention_paged, what, cache.device, stream, cache._ref, batch._ref, qp, qs, heads,
                 1.0 / math.sqrt(cache.head_dim) if scale is None else float(scale), window, sinks, op, os, ws, nws)


def verify_workspace_bytes(B: int, R: int, V: int) -> int:
    return int(lib().viper_hip_verify_workspace_bytes(B, R, V))


def verify_draft(target_logits, draft_tokens, uniforms, out_tokens, out_accepted, draft_logits=None, draft_lens=None,
                 temperature=None, accept_probs=None, workspace=None, stream=None) -> Status:
    """Accepts or rejects drafted tokens (int32 [B, R - 1]) by the target's logits (bf16 [B, R, V]) and uniforms (fp32 [B, R])
    and draws the token that follows: out_tokens int32 [B, R] (accepted, next, then -1), out_accepted int32 [B].
    draft_logits bf16 [B, R - 1, V] (None: a deterministic drafter), draft_lens int32 [B], temperature fp32 [B] (None: 1, 0:
    greedy), accept_probs fp32 [B, R - 1].  workspace: verify_workspace_bytes(B, R, V) bytes, zero before its first use."""
    what = "viper_hip_verify_draft"
    if target_logits.dim() != 3:
        return _mismatch(what, "target_logits is [B, R, V]")
    B, R, V = target_logits.shape
    for t, n, name in ((draft_tokens, B * (R - 1), "draft_tokens"), (uniforms, B * R, "uniforms"), (out_tokens, B * R, "out_tokens"),
                       (out_accepted, B, "out_accepted"), (draft_logits, B * (R - 1) * V, "draft_logits"),
                       (draft_lens, B, "draft_lens"), (temperature, B, "temperature"), (accept_probs, B * (R - 1), "accept_probs")):
        if t is not None and t.numel() != n:
            return _mismatch(what, f"{name} does not match target_logits")
    _one_device(target_logits, draft_tokens, uniforms, out_tokens, out_accepted, draft_logits, draft_lens, temperature,
                accept_probs, workspace)
    opt = lambda t, size: None if t is None or t.numel() == 0 else ptr(t, size)
    nws = 0 if workspace is None else workspace.numel() * workspace.element_size()
    return _call(lib().viper_hip_verify_draft, what, target_logits.device, stream, ptr(target_logits, 2), opt(draft_logits, 2),
                 opt(draft_tokens, 4), opt(draft_lens, 4), ptr(uniforms, 4), opt(temperature, 4), B, R, V, ptr(out_tokens, 4),
                 ptr(out_accepted, 4), opt(accept_probs, 4), ptr(workspace), nws)
