"""The paged KV cache of 8-bit codes and the attention over it (``ktmoe_kv_append_dev``, ``ktmoe_kv_read_dev``,
``ktmoe_attention_dev`` of ``include/ktmoe.h``, which states the arithmetic).

Device buffers are torch tensors (memory only; every value comes from libktmoe.so's kernels). Calls are ordered on
torch's current stream unless ``stream`` gives another (a raw CUDA stream handle; 0: the context's own stream), and are
not synchronised. AttentionHalf and MoeStack run on the context's stream by default, which does not wait for torch's nor
torch's for it: give ``stream=0`` to the calls on a cache that go with them, or synchronise in between. What only the
device can find wrong in a batch (a page outside the pool, lengths that do not fit) is raised by the next
``Context.sync`` that waits for the call: ``sync(stream)`` for one on another stream. A scale is two int64 words, {mant,
shift}: one pair, or one pair a row.
"""

from __future__ import annotations

import ctypes
from typing import Optional

import numpy as np

from ._native import KtmoeKvBatch, KtmoeKvCache, KtmoeRope, check, lib

__all__ = ["KvCache", "KvBatch", "Rope", "rope_table"]

STREAM_LEGACY = 1  # cudaStreamLegacy: torch's default stream, whose handle 0 means the context's own stream here


def rope_table(theta: float, rot_dim: int, positions: int) -> np.ndarray:
    """Rotation table int32 [positions][rot_dim / 2][2] (ktmoe_rope_table): cosine and sine times 2^30."""
    if rot_dim < 2 or rot_dim % 2 or positions < 1:
        raise ValueError("rope_table: rot_dim is even and at least 2, positions at least 1")
    out = np.empty((positions, rot_dim // 2, 2), dtype=np.int32)
    check(lib().ktmoe_rope_table(float(theta), rot_dim, positions, out.ctypes.data_as(ctypes.POINTER(ctypes.c_int32))))
    return out


_torch = None  # torch and what the calls below take from it, imported with the first class that needs it
_raw_stream = None


def _load_torch():
    global _torch, _raw_stream
    if _torch is None:
        import torch

        # the current stream's handle without building a Stream object, where torch offers it
        _raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
            lambda device: torch.cuda.current_stream(device).cuda_stream)
        _torch = torch
    return _torch


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _tensor(t, name: str, dtype: str, dims: int) -> None:
    torch = _load_torch()
    _need(isinstance(t, torch.Tensor) and t.dtype is getattr(torch, dtype), f"{name}: a torch tensor of {dtype}")
    _need(t.dim() == dims, f"{name}: {dims} dimensions")
    _need(t.is_contiguous(), f"{name}: contiguous")


def _matrix(t, name: str, dtype, rows: int, width: int) -> int:
    """Check a [rows or more][width] matrix whose rows are contiguous; returns its row stride. (These checks run before
    every launch, so they touch each property of a tensor once and build no message unless one fails.)"""
    if not isinstance(t, _torch.Tensor) or t.dtype is not dtype:
        raise ValueError(f"{name}: a torch tensor of {dtype}")
    shape = t.shape
    if len(shape) != 2 or shape[0] < rows or shape[1] != width:
        raise ValueError(f"{name}: at least {rows} rows of {width}")
    ld, step = t.stride()
    if step != 1 and width != 1:
        raise ValueError(f"{name}: the elements of a row lie side by side")
    if shape[0] <= 1:
        return width  # one row has no stride of its own (torch reports any)
    if ld < width:
        raise ValueError(f"{name}: rows that do not overlap")
    return ld


class Rope:
    """Rotary positions: a device table (int32 [positions][rot_dim / 2][2], see :func:`rope_table`) and the pairing:
    (i, i + rot_dim / 2), or (2i, 2i + 1) when ``interleaved``."""

    def __init__(self, table, interleaved: bool = False):
        _tensor(table, "rotation table", "int32", 3)
        _need(table.shape[0] >= 1 and table.shape[1] >= 1 and table.shape[2] == 2,
              "rotation table: [positions][rot_dim / 2][2]")
        self.table, self.interleaved = table, bool(interleaved)
        self.device_index = table.get_device()
        self._c = KtmoeRope(table.data_ptr(), table.shape[0], 2 * table.shape[1], 1 if interleaved else 0)


class KvBatch:
    """The new tokens of a batch of sequences: device int32 tensors ``q_begin`` [n + 1] (ascending row offsets),
    ``kv_len`` [n] (lengths with the new tokens), ``page_table`` [n][max_pages], and the number of ``rows`` that the
    calls' buffers hold. The tensors are read when the kernels run, so their contents may change between calls."""

    def __init__(self, q_begin, kv_len, page_table, rows: int):
        _tensor(q_begin, "q_begin", "int32", 1)
        _tensor(kv_len, "kv_len", "int32", 1)
        _tensor(page_table, "page_table", "int32", 2)
        n = kv_len.shape[0]
        _need(q_begin.shape[0] == n + 1 and page_table.shape[0] == n, "q_begin has one entry more than kv_len, page_table as many rows")
        _need(0 <= int(rows) <= 1 << 30, "rows: from 0 to 2^30")
        _need(q_begin.device == kv_len.device == page_table.device, "the batch's tensors lie on one device")
        self.device_index = kv_len.get_device()
        self.q_begin, self.kv_len, self.page_table, self.rows = q_begin, kv_len, page_table, int(rows)
        self._c = KtmoeKvBatch(n, page_table.shape[1], q_begin.data_ptr(), kv_len.data_ptr(), page_table.data_ptr(),
                               self.rows)


class KvCache:
    """Pages of cached keys and values on a context's device: int8 codes [n_pages][n_kv_heads][page_tokens][head_dim]
    and bfloat16 scales [n_pages][n_kv_heads][page_tokens], allocated here or given as ``pools = (k, v, k_scale,
    v_scale)``. Which page belongs to whom is the caller's business (:class:`KvBatch`)."""

    def __init__(self, ctx, n_pages: int, page_tokens: int, n_kv_heads: int, head_dim: int, pools=None):
        _need(page_tokens in (16, 32, 64, 128), "page_tokens: 16, 32, 64 or 128")
        _need(16 <= head_dim <= 256 and head_dim % 16 == 0, "head_dim: a multiple of 16 from 16 to 256")
        _need(1 <= n_kv_heads <= 1024 and n_pages >= 1, "n_kv_heads from 1 to 1024, n_pages at least 1")
        self.ctx = ctx
        self.n_pages, self.page_tokens, self.n_kv_heads, self.head_dim = n_pages, page_tokens, n_kv_heads, head_dim
        shape = (n_pages, n_kv_heads, page_tokens)
        torch = _load_torch()
        if pools is None:
            dev = torch.device("cuda", ctx.device)
            pools = [torch.zeros(*shape, head_dim, dtype=torch.int8, device=dev) for _ in range(2)]
            pools += [torch.zeros(shape, dtype=torch.bfloat16, device=dev) for _ in range(2)]
            # cleared before anything can write them: the context's stream does not wait for torch's
            if not torch.cuda.is_current_stream_capturing():
                torch.cuda.current_stream(dev).synchronize()
        self.k, self.v, self.k_scale, self.v_scale = pools
        for t, name in ((self.k, "k pool"), (self.v, "v pool")):
            _tensor(t, name, "int8", 4)
            _need(tuple(t.shape) == (*shape, head_dim), f"{name}: [n_pages][n_kv_heads][page_tokens][head_dim]")
        for t, name in ((self.k_scale, "k scales"), (self.v_scale, "v scales")):
            _tensor(t, name, "bfloat16", 3)
            _need(tuple(t.shape) == shape, f"{name}: [n_pages][n_kv_heads][page_tokens]")
        self.device_index = self.k.get_device()
        if any(t.get_device() != self.device_index for t in (self.v, self.k_scale, self.v_scale)):
            raise ValueError("the pools lie on one device")
        L = lib()
        self._append, self._read, self._attend = L.ktmoe_kv_append_dev, L.ktmoe_kv_read_dev, L.ktmoe_attention_dev
        self._c = KtmoeKvCache(self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(),
                               n_pages, page_tokens, n_kv_heads, head_dim)

    def _prepare(self, batch: KvBatch, rope: Optional[Rope], stream: Optional[int], *tensors):
        """Every tensor on the context's device; the stream to launch on."""
        device = self.ctx.device
        for t in tensors:
            if t.get_device() != device:
                raise ValueError(f"every tensor lies on the context's device (cuda:{device})")
        if batch.device_index != device or self.device_index != device or (rope and rope.device_index != device):
            raise ValueError(f"every tensor lies on the context's device (cuda:{device})")
        if stream is None:
            return _raw_stream(device) or STREAM_LEGACY
        return stream or None

    def _scale(self, scale, rows: int) -> int:
        """0: one scale for all rows, 1: one a row."""
        if not isinstance(scale, _torch.Tensor) or scale.dtype is not _torch.int64 or not scale.is_contiguous():
            raise ValueError("scale: a contiguous torch tensor of int64")
        shape = scale.shape
        if len(shape) == 2 and shape[1] == 2 and shape[0] >= rows:
            return 1
        if shape == (2,) or shape == (1, 2):
            return 0
        raise ValueError("scale: [2], or [rows][2] with a scale for each row")

    def append(self, batch: KvBatch, k, v, scale, rope: Optional[Rope] = None, v_scale=None,
               stream: Optional[int] = None) -> None:
        """Write the batch's new keys and values (int32 codes [rows][n_kv_heads * head_dim], row strides allowed) at
        ``scale`` (the values at ``v_scale`` when given) into their pages, the keys rotated by ``rope``."""
        width, rows, int32 = self.n_kv_heads * self.head_dim, batch.rows, _torch.int32
        ld_k = _matrix(k, "k", int32, rows, width)
        ld_v = _matrix(v, "v", int32, rows, width)
        stride = self._scale(scale, rows)
        if v_scale is None:
            at = self._prepare(batch, rope, stream, k, v, scale)
        else:
            _need(self._scale(v_scale, rows) == stride, "scale and v_scale: both one for all rows or both one a row")
            at = self._prepare(batch, rope, stream, k, v, scale, v_scale)
        status = self._append(self.ctx.handle, self._c, batch._c, k.data_ptr(), ld_k, v.data_ptr(), ld_v,
                              scale.data_ptr(), None if v_scale is None else v_scale.data_ptr(), stride,
                              rope._c if rope else None, at)
        if status:
            self.ctx.check(status)

    def read(self, batch: KvBatch, k, v, stream: Optional[int] = None) -> None:
        """Read the batch's rows back as values (float32 [rows][n_kv_heads * head_dim]) into ``k`` and ``v``."""
        width, rows, float32 = self.n_kv_heads * self.head_dim, batch.rows, _torch.float32
        ld_k = _matrix(k, "k", float32, rows, width)
        ld_v = _matrix(v, "v", float32, rows, width)
        at = self._prepare(batch, None, stream, k, v)
        status = self._read(self.ctx.handle, self._c, batch._c, k.data_ptr(), ld_k, v.data_ptr(), ld_v, at)
        if status:
            self.ctx.check(status)

    def attention(self, batch: KvBatch, q, scale, out, out_scale, n_heads: int, rope: Optional[Rope] = None,
                  softmax_scale: Optional[float] = None, window: int = 0, sinks: int = 0,
                  stream: Optional[int] = None) -> None:
        """Attention of the batch's new tokens (``q``: int32 codes [rows][n_heads * head_dim] at ``scale``) over the
        cache, which already holds their keys and values, into ``out`` (int32 [rows][n_heads * head_dim]) at
        ``out_scale`` (int64 [rows][n_kv_heads][2]). ``softmax_scale`` defaults to head_dim ** -0.5; ``window`` > 0
        keeps the last ``window`` positions and the first ``sinks``."""
        if n_heads < 1 or n_heads % self.n_kv_heads != 0 or not (0 <= window < 1 << 31 and 0 <= sinks < 1 << 31):
            raise ValueError("n_heads: a multiple of n_kv_heads; window and sinks: from 0 to 2^31 - 1")
        width, rows, int32 = n_heads * self.head_dim, batch.rows, _torch.int32
        ld_q = _matrix(q, "q", int32, rows, width)
        ld_o = _matrix(out, "out", int32, rows, width)
        stride = self._scale(scale, rows)
        shape = out_scale.shape
        if (out_scale.dtype is not _torch.int64 or len(shape) != 3 or shape[0] < rows or shape[1] != self.n_kv_heads
                or shape[2] != 2 or not out_scale.is_contiguous()):
            raise ValueError("out_scale: a contiguous torch tensor of int64, [rows][n_kv_heads][2]")
        at = self._prepare(batch, rope, stream, q, out, scale, out_scale)
        status = self._attend(self.ctx.handle, self._c, batch._c, q.data_ptr(), ld_q, scale.data_ptr(), stride,
                              rope._c if rope else None, n_heads,
                              self.head_dim ** -0.5 if softmax_scale is None else float(softmax_scale), window, sinks,
                              out.data_ptr(), ld_o, out_scale.data_ptr(), at)
        if status:
            self.ctx.check(status)
