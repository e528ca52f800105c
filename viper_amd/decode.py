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

import torch

from .qlinear import Status, StatusCode, _status, lib, ptr


class KVType(enum.IntEnum):
    BF16 = 0
    INT8 = 1


class _Fixed:
    """What a call reads is taken from the fields once, so they are not replaced afterwards (tensors change in place)."""

    def __setattr__(self, name, value):
        if "_ref" in self.__dict__ and name in self.__dataclass_fields__:
            raise AttributeError(f"{type(self).__name__}.{name} is fixed: write into the tensor, or build another")
        object.__setattr__(self, name, value)


class _CCache(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("kv_type", "kv_heads", "head_dim", "page_size", "num_pages")] + \
               [(n, C.c_void_p) for n in ("k", "v", "k_scales", "v_scales")]


class _CBatch(C.Structure):
    _fields_ = [(n, C.c_int32) for n in ("batch", "max_rows", "total_rows", "table_width")] + \
               [(n, C.c_void_p) for n in ("block_table", "seq_lens", "row_offsets")]


@dataclass
class KVCache(_Fixed):
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
        i8 = KVType(self.kv_type) == KVType.INT8
        for t in (self.k, self.v):
            _typed(t, _INT8 if i8 else _BF16)
        for t in (self.k_scales, self.v_scales):
            _typed(t, _FP32)
        size = 1 if i8 else 2
        page = self.kv_heads * self.page_size * self.head_dim
        if page <= 0 or self.k.numel() != self.v.numel() or self.k.numel() % page:
            raise ValueError("KVCache: k and v hold whole pages of kv_heads * page_size * head_dim elements")
        self.num_pages = self.k.numel() // page
        if (self.k_scales is None) != (self.v_scales is None):
            raise ValueError("KVCache: k_scales and v_scales go together")
        if self.k_scales is not None and not all(_laid(t, (self.num_pages, self.kv_heads, self.page_size))
                                                 for t in (self.k_scales, self.v_scales)):
            raise ValueError("KVCache: one scale for each token and head, [num_pages, kv_heads, page_size]")
        _one_device(self.k, self.v, self.k_scales, self.v_scales)
        self._c = _CCache(int(self.kv_type), self.kv_heads, self.head_dim, self.page_size, self.num_pages, ptr(self.k, size),
                          ptr(self.v, size), ptr(self.k_scales, 4), ptr(self.v_scales, 4))
        self._dev = self.k.get_device()
        self._width = self.kv_heads * self.head_dim
        self._scale = 1.0 / math.sqrt(self.head_dim)
        self._ref = C.addressof(self._c)

    @classmethod
    def empty(cls, kv_type, num_pages, page_size, kv_heads, head_dim, device="cuda"):
        """A cache of zeroed pages."""
        i8 = int(kv_type) == KVType.INT8
        shape = (num_pages, kv_heads, page_size // 32, 32 * head_dim)
        pool = lambda: torch.zeros(shape, dtype=torch.int8 if i8 else torch.bfloat16, device=device)
        scales = lambda: torch.zeros((num_pages, kv_heads, page_size), dtype=torch.float32, device=device) if i8 else None
        return cls(KVType(kv_type), pool(), pool(), page_size, kv_heads, head_dim, scales(), scales())


@dataclass
class KVBatch(_Fixed):
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
        if not (_int32(self.max_rows) and _int32(self.total_rows or 0)):
            raise ValueError("KVBatch: max_rows and total_rows are 32-bit")
        for t in (self.block_table, self.seq_lens, self.row_offsets):
            _typed(t, _INT32)
        _one_device(self.block_table, self.seq_lens, self.row_offsets)
        self._views = {}  # C views by the number of rows
        self._dev = self.seq_lens.get_device()
        self._ref = self._view(self.total_rows or 0)

    def _rows(self, n, dev):
        """The C view for row tensors of n rows; None where they do not fit."""
        if dev != self._dev:
            raise ValueError("viper_amd: tensors on more than one device")
        if self.total_rows is not None:
            return self._ref if n == self.total_rows else None
        v = self._views.get(n)
        return C.addressof(v) if v is not None else self._view(n)

    def _view(self, n):
        v = _CBatch(self.batch, self.max_rows, n, self.block_table.shape[1], ptr(self.block_table, 4), ptr(self.seq_lens, 4),
                    ptr(self.row_offsets, 4))
        return C.addressof(self._views.setdefault(n, v))


# What the elements of each kind of argument may be (bf16 values also as their bit patterns): another type of the same size
# would be read as it
_BF16 = (torch.bfloat16, torch.int16, torch.uint16)
_INT8 = (torch.int8, torch.uint8)
_FP32 = (torch.float32,)
_INT32 = (torch.int32, torch.uint32)


def _typed(t, types):
    if t is not None and t.dtype not in types:
        raise _untyped(t, types)


def _untyped(t, types):
    name = {_BF16: "bf16", _INT8: "int8", _FP32: "fp32", _INT32: "int32"}[types]
    return ValueError(f"viper_amd: expected {name} elements, got {t.dtype}")


def _laid(t, shape):
    """Whether t has this shape, but for axes of one, or is flat with as many elements."""
    a, b = ([n for n in x if n != 1] for x in (t.shape, shape))
    return t.numel() == math.prod(shape) and (a == b or len(a) < 2)


def _int32(n):
    """Whether n reaches the library as it is (ctypes drops the bits that do not fit)."""
    return -1 << 31 <= n < 1 << 31


def _one_device(*tensors):
    d = [t.device for t in tensors if t is not None]
    if any(x != d[0] for x in d):
        raise ValueError("viper_amd: tensors on more than one device")


def _row_view(t, width, dev):
    """(address, row stride in elements, rows) of a bf16 tensor of rows of `width` values on device number dev: [rows, width]
    or [rows, heads, head_dim], each row dense, rows any multiple of 8 elements apart (columns of a wider matrix)."""
    if t.dtype not in _BF16:
        raise _untyped(t, _BF16)
    if t.get_device() != dev:
        raise ValueError("viper_amd: tensor arguments must be GPU tensors, all on one device")
    shape, s = t.shape, t.stride()
    if len(s) == 2:
        fine = shape[1] == width and s[1] == 1
    else:
        fine = len(s) == 3 and shape[1] * shape[2] == width and s[2] == 1 and (shape[1] == 1 or s[1] == shape[2])
    if not fine:
        raise ValueError(f"viper_amd: expected rows of {width} dense values, got {tuple(shape)} strides {s}")
    rows, stride = shape[0], s[0]
    if rows == 1 and (stride < width or stride % 8):
        stride = width
    return t.data_ptr(), stride, rows


def _row_width(t):
    if t.dim() < 2:
        raise ValueError(f"viper_amd: expected rows, got a tensor of shape {tuple(t.shape)}")
    return t.shape[-1] if t.dim() == 2 else t.shape[-1] * t.shape[1]


def _flat(t, types, dev):
    """Address of a dense tensor of elements of one of `types` (None: any) on device number dev."""
    if t is None:
        return None
    if types is not None and t.dtype not in types:
        raise _untyped(t, types)
    if t.get_device() != dev:
        raise ValueError("viper_amd: tensor arguments must be GPU tensors, all on one device")
    if not t.is_contiguous():
        raise ValueError("viper_amd: tensor arguments must be contiguous")
    return t.data_ptr()


def _call(fn, what, dev, stream, *args) -> Status:
    """The launch on device number dev, on `stream` or that device's current one."""
    if stream is not None and not isinstance(stream, int):
        if stream.device.index != dev:
            return Status(StatusCode.INVALID_ARGUMENT, f"{what}: the stream is on another device")
        stream = stream.cuda_stream
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            rc = fn(*args, torch.cuda.current_stream().cuda_stream if stream is None else stream)
    else:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(dev) if stream is None else stream)
    return _OK if rc == 0 else _status(rc, what)


_OK = Status()


def _mismatch(what, text) -> Status:
    return Status(StatusCode.SHAPE_MISMATCH, f"{what}: {text}")


def kv_append(cache: KVCache, batch: KVBatch, k, v, q=None, q_out=None, rope_theta: Optional[float] = None,
              stream=None) -> Status:
    """Stores rows k and v ([rows, kv_heads * head_dim], or [rows, kv_heads, head_dim]) in the cache.  With rope_theta, k is
    rotated by its position first and q ([rows, heads * head_dim]) into q_out (may be q)."""
    what = "viper_hip_kv_append"
    if (q is None) != (q_out is None):
        return _mismatch(what, "q and q_out go together")
    dev, D = cache._dev, cache.head_dim
    kp, ks, rows = _row_view(k, cache._width, dev)
    vp, vs, vrows = _row_view(v, cache._width, dev)
    if rows != vrows or (rows > 1 and ks != vs):
        return _mismatch(what, "k and v are laid out alike")
    ref = batch._rows(rows, dev)
    if ref is None:
        return _mismatch(what, "the rows do not match the batch")
    if rows == 0:
        return _OK
    qp = op = None
    qs = os = heads = 0
    if q is not None:
        if rope_theta is None:
            return Status(StatusCode.INVALID_ARGUMENT, f"{what}: q is taken for its rotation")
        width = _row_width(q)
        heads = width // D
        if heads * D != width:
            return _mismatch(what, "q rows are not whole heads")
        qp, qs, qrows = _row_view(q, width, dev)
        op, os, orows = _row_view(q_out, width, dev)
        if qrows != rows or orows != rows:
            return _mismatch(what, "q rows != k rows")
    return _call(lib().viper_hip_kv_append, what, dev, stream, cache._ref, ref, kp, vp, ks, qp, qs, heads, op, os,
                 rope_theta or 0.0)


def kv_read(cache: KVCache, batch: KVBatch, k_out, v_out, stream=None) -> Status:
    """The batch's rows back from the cache: k_out and v_out bf16 [rows, kv_heads, head_dim]."""
    what = "viper_hip_kv_read"
    dev, n = cache._dev, k_out.numel()
    ref = batch._rows(n // cache._width, dev)
    if v_out.numel() != n or n % cache._width or ref is None:
        return _mismatch(what, "the rows do not match the batch")
    rows = n // cache._width
    for t in (k_out, v_out):
        if t.shape != (rows, cache.kv_heads, cache.head_dim) and t.shape != (rows, cache._width) and \
                not _laid(t, (rows, cache.kv_heads, cache.head_dim)) and not _laid(t, (rows, cache._width)):
            return _mismatch(what, f"rows of shape {tuple(t.shape)} are not [rows, kv_heads, head_dim]")
    if n == 0:
        return _OK
    return _call(lib().viper_hip_kv_read, what, dev, stream, cache._ref, ref, _flat(k_out, _BF16, dev), _flat(v_out, _BF16, dev))


def attention_workspace_bytes(cache: KVCache, batch: KVBatch, heads: int) -> int:
    """Bytes of workspace (zero before its first use) that lets attention_paged split the cache's length over workgroups;
    0 where the batch alone fills the GPU."""
    if not _int32(heads):
        return 0
    if cache._dev != torch.cuda.current_device():  # (the plan counts a device's CUs)
        with torch.cuda.device(cache._dev):
            return int(lib().viper_hip_attention_workspace_bytes(cache._ref, batch._ref, heads))
    return int(lib().viper_hip_attention_workspace_bytes(cache._ref, batch._ref, heads))


def attention_paged(cache: KVCache, batch: KVBatch, q, out, scale: Optional[float] = None, window: int = 0, sinks: int = 0,
                    workspace=None, stream=None) -> Status:
    """out = attention of the rows q ([rows, heads * head_dim], heads a multiple of the cache's) over their sequences' pages:
    causal; with window > 0 the newest `window` tokens and the first `sinks`.  scale defaults to head_dim ** -0.5."""
    what = "viper_hip_attention_paged"
    dev, width = cache._dev, _row_width(q)
    heads = width // cache.head_dim
    if heads * cache.head_dim != width:
        return _mismatch(what, "q rows are not whole heads")
    qp, qs, rows = _row_view(q, width, dev)
    op, os, orows = _row_view(out, width, dev)
    if not (_int32(window) and _int32(sinks)):
        return Status(StatusCode.INVALID_ARGUMENT, f"{what}: window and sinks are 32-bit")
    ref = batch._rows(rows, dev)
    if orows != rows or ref is None:
        return _mismatch(what, "the rows do not match the batch")
    if rows == 0:
        return _OK
    ws, nws = None, 0
    if workspace is not None:
        nws = workspace.numel() * workspace.element_size()
        if nws:
            ws = _flat(workspace, None, dev)
    return _call(lib().viper_hip_attention_paged, what, dev, stream, cache._ref, ref, qp, qs, heads,
                 cache._scale if scale is None else scale, window, sinks, op, os, ws, nws)


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
    dev, n = target_logits.get_device(), B * (R - 1)
    each, every, drafted = (B,), (B, R), (B, R - 1)
    for t, shape in ((uniforms, every), (out_tokens, every), (out_accepted, each), (draft_tokens, drafted),
                     (draft_logits, (B, R - 1, V)), (draft_lens, each), (temperature, each), (accept_probs, drafted)):
        if t is not None and t.shape != shape and not _laid(t, shape):
            return _mismatch(what, f"a tensor of shape {tuple(t.shape)} does not match target_logits, {shape} is wanted")
    if dev < 0:
        raise ValueError("viper_amd: tensor arguments must be GPU tensors, all on one device")
    if n == 0:  # nothing drafted: empty tensors have no address
        draft_tokens = draft_logits = accept_probs = None
    nws = 0 if workspace is None else workspace.numel() * workspace.element_size()
    f = _flat
    return _call(lib().viper_hip_verify_draft, what, dev, stream, f(target_logits, _BF16, dev), f(draft_logits, _BF16, dev),
                 f(draft_tokens, _INT32, dev), f(draft_lens, _INT32, dev), f(uniforms, _FP32, dev), f(temperature, _FP32, dev),
                 B, R, V, f(out_tokens, _INT32, dev), f(out_accepted, _INT32, dev), f(accept_probs, _FP32, dev),
                 f(workspace, None, dev), nws)
