"""A decoder layer's attention over a paged key/value cache: vw_rope_append, vw_prompt_attention, vw_decode_attention.

Mirrors what voxwerk's ``DecoderStack.ForwardSegments`` (src/Voxwerk/Talker/DecoderStack.cs:144-228) does between the
projections, over its ``KvCache`` (:21), for a batch of sequences whose keys and values lie in pages of one cache:

    cache = KvCache.empty(n_pages, 16, n_kv_heads, head_dim)      # or KvCache(k, v) over tensors of your own
    rope = RopeTable.build(max_positions, head_dim, base=1e6)
    batch = KvBatch(page_table, kv_lens, q_offsets)
    rope_append(device, q, k, v, cache, batch, rope, q_out, q_norm=wq, k_norm=wk)
    prompt_attention(device, q_out, cache, batch, out)            # rows of several tokens per sequence
    decode_attention(device, q_out, cache, batch, out, prefix=KvPrefix(...))    # one row per sequence

``KvCache``, ``KvBatch``, ``KvPrefix`` and ``RopeTable`` hold references to CUDA tensors; they are built once and keep
describing the same tensors as their contents change from step to step.  ``stream`` is a cudaStream_t (an int, as
``torch.cuda.Stream.cuda_stream``; 0 is torch's default stream): given, a call is enqueued on it, behind what the caller
put there.  None runs on torch's current stream, waits for it, and raises what the kernels reported.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from ._lib import VW_BF16, VW_F32, VwAttnRows, VwKvBatch, VwKvCache, VwKvPrefix, VwRopeRows, check, lib
from .sampler import DEFAULT_STREAM, Device


_BF16, _F32 = torch.bfloat16, torch.float32


def _need(ok: bool, message: str) -> None:
    if not ok:
        raise ValueError(message)


def _cuda(t, dtype: str, dims: int, what: str):
    if not getattr(t, "is_cuda", False):
        raise TypeError(f"{what} must be a CUDA tensor")
    if t.dtype is not getattr(torch, dtype):
        raise TypeError(f"{what} must be {dtype}, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{what} must have {dims} dimensions")
    return t


def _same_gpu(gpu: int, index: int, what: str) -> None:
    if index != gpu:
        raise ValueError(f"{what} is on cuda:{index}, the device handle on cuda:{gpu}")


def _one_gpu(first, *others) -> int:
    for t in others:
        _need(t.get_device() == first.get_device(), "the tensors must be on one GPU")
    return first.get_device()


def _call(function, device: Device, stream: Optional[int], *args) -> None:
    handle = device.handle
    if stream is not None:
        check(function(handle, *args, stream or DEFAULT_STREAM), handle)
        return
    if torch.cuda.is_current_stream_capturing():
        raise ValueError("a call that is captured takes the capturing stream")
    stream = torch.cuda.current_stream(device.device).cuda_stream or DEFAULT_STREAM
    check(function(handle, *args, stream), handle)
    check(lib.vw_synchronize(handle, stream), handle)


def _no_gpu() -> int:
    return -1


def _rows(gpu: int, t, dtype, shape, what: str):
    """Pointer, row and head stride of a [rows, heads, dim] tensor; a dimension of size one has no stride of its own."""
    index = getattr(t, "get_device", _no_gpu)()
    if index != gpu:
        if not getattr(t, "is_cuda", False):
            raise TypeError(f"{what} must be a CUDA tensor")
        _same_gpu(gpu, index, what)
    if t.dtype is not dtype:
        raise TypeError(f"{what} must be {str(dtype)[6:]}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{what} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    row, head, one = t.stride()
    rows, heads, dim = shape
    if one != 1 and dim != 1:
        raise ValueError(f"{what}: the last dimension must be contiguous")
    if heads == 1:
        head = (dim + 7) // 8 * 8
    if rows == 1:
        row = heads * head
    return t.data_ptr(), row, head


class KvCache:
    """Keys and values [n_pages, page_size, n_kv_heads, head_dim] bfloat16 (equal strides, last dimension contiguous).
    page_size is a power of two from 16 to 256; a [n_pages, n_kv_heads, page_size, head_dim] layout is passed as its
    transpose(1, 2)."""

    def __init__(self, k, v):
        _cuda(k, "bfloat16", 4, "k")
        _cuda(v, "bfloat16", 4, "v")
        _need(k.shape == v.shape and k.stride() == v.stride(), "k and v must have the same shape and strides")
        _need(k.stride(3) == 1, "k and v: the last dimension must be contiguous")
        self.k, self.v = k, v
        self._gpu = _one_gpu(k, v)
        pages, size, heads, dim = k.shape
        self.n_kv_heads, self.head_dim = heads, dim
        page, token, head, _ = k.stride()
        head = dim if heads == 1 else head
        self.c = VwKvCache(k.data_ptr(), v.data_ptr(), page if pages > 1 else size * max(token, size * heads * dim),
                           token, head, pages, size, heads, dim)
        self._ref = ctypes.byref(self.c)

    @staticmethod
    def empty(n_pages: int, page_size: int, n_kv_heads: int, head_dim: int, device="cuda") -> "KvCache":
        shape = (n_pages, page_size, n_kv_heads, head_dim)
        return KvCache(*(torch.empty(shape, dtype=torch.bfloat16, device=device) for _ in range(2)))


class KvBatch:
    """The sequences of a call: page_table [n_seqs, max_pages] int32, kv_lens [n_seqs] int32 (keys each sequence holds,
    the call's rows included) and q_offsets [n_seqs + 1] int32 (its rows; None: one row per sequence)."""

    def __init__(self, page_table, kv_lens, q_offsets=None):
        _cuda(page_table, "int32", 2, "page_table")
        _cuda(kv_lens, "int32", 1, "kv_lens")
        n = page_table.shape[0]
        _need(page_table.shape[1] <= 1 or page_table.stride(1) == 1, "page_table rows must be contiguous")
        _need(kv_lens.shape[0] == n and kv_lens.is_contiguous(), "kv_lens must be a contiguous [n_seqs]")
        if q_offsets is not None:
            _cuda(q_offsets, "int32", 1, "q_offsets")
            _need(q_offsets.shape[0] == n + 1 and q_offsets.is_contiguous(), "q_offsets must be a contiguous [n_seqs + 1]")
        self.page_table, self.kv_lens, self.q_offsets, self.n_seqs = page_table, kv_lens, q_offsets, n
        self._gpu = _one_gpu(page_table, kv_lens, *([] if q_offsets is None else [q_offsets]))
        self._c = (page_table.data_ptr(), page_table.stride(0) if n > 1 else page_table.shape[1], page_table.shape[1], n,
                   kv_lens.data_ptr(), None if q_offsets is None else q_offsets.data_ptr())
        self._last = None, None

    def _rows(self, n: int):   # a struct once made does not change: threads with a handle each may share a batch
        rows, ref = self._last
        if rows != n:
            ref = ctypes.byref(VwKvBatch(*self._c, n))
            self._last = n, ref
        return ref


class KvPrefix:
    """Prefixes that groups of sequences share: page_table [n_groups, max_pages] int32, lens [n_groups] int32,
    group_offsets [n_groups + 1] int32 (sequences group_offsets[g] .. group_offsets[g + 1) see prefix g)."""

    def __init__(self, page_table, lens, group_offsets):
        _cuda(page_table, "int32", 2, "page_table")
        _cuda(lens, "int32", 1, "lens")
        _cuda(group_offsets, "int32", 1, "group_offsets")
        n = page_table.shape[0]
        _need(page_table.shape[1] <= 1 or page_table.stride(1) == 1, "page_table rows must be contiguous")
        _need(lens.shape[0] == n and lens.is_contiguous(), "lens must be a contiguous [n_groups]")
        _need(group_offsets.shape[0] == n + 1 and group_offsets.is_contiguous(),
              "group_offsets must be a contiguous [n_groups + 1]")
        self.page_table, self.lens, self.group_offsets = page_table, lens, group_offsets
        self._gpu = _one_gpu(page_table, lens, group_offsets)
        self.c = VwKvPrefix(page_table.data_ptr(), page_table.stride(0) if n > 1 else page_table.shape[1],
                            page_table.shape[1], n, lens.data_ptr(), group_offsets.data_ptr())
        self._ref = ctypes.byref(self.c)


class RopeTable:
    """Cosines and sines [n_positions, rotary_dim / 2] float32 of each position's angles; `interleaved` pairs dims
    (2 i, 2 i + 1) instead of (i, i + rotary_dim / 2)."""

    def __init__(self, cos, sin, interleaved: bool = False):
        _cuda(cos, "float32", 2, "cos")
        _cuda(sin, "float32", 2, "sin")
        _need(cos.shape == sin.shape and cos.is_contiguous() and sin.is_contiguous(),
              "cos and sin must be contiguous and of one shape")
        self.cos, self.sin, self.interleaved = cos, sin, bool(interleaved)
        self._gpu = _one_gpu(cos, sin)
        self.rotary_dim = 2 * int(cos.shape[1])
        self._c = (int(cos.shape[0]), cos.data_ptr(), sin.data_ptr(), self.rotary_dim, int(self.interleaved))

    @staticmethod
    def angles(n_positions: int, rotary_dim: int, base: float = 10000.0, linear: float = 1.0,
               yarn: Optional[float] = None, trained_positions: int = 0, beta_fast: float = 32.0, beta_slow: float = 1.0):
        """(angles [n_positions, rotary_dim / 2] float64, amplitude).  `linear` divides every position; `yarn` is the
        factor of YaRN (Peng et al. 2023): frequencies that turn fewer than beta_slow times over `trained_positions`
        are divided by it, those that turn more than beta_fast times are kept, the ones between are blended, and the
        amplitude is 0.1 ln(yarn) + 1."""
        if rotary_dim < 2 or rotary_dim % 2:
            raise ValueError("rotary_dim must be a positive even number")
        half = rotary_dim // 2
        freq = base ** (-torch.arange(half, dtype=torch.float64) / half)
        amplitude = 1.0
        if yarn is not None:
            if yarn < 1 or trained_positions < 1:
                raise ValueError("yarn >= 1 and trained_positions are required")
            turns = trained_positions * freq / (2 * math.pi)
            keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0, 1)
            freq = freq * keep + freq / yarn * (1 - keep)
            amplitude = 0.1 * math.log(yarn) + 1.0
        return torch.arange(n_positions, dtype=torch.float64)[:, None] / linear * freq, amplitude

    @staticmethod
    def build(n_positions: int, rotary_dim: int, base: float = 10000.0, interleaved: bool = False, device="cuda",
              **scaling) -> "RopeTable":
        """The table of `angles(...)`, computed in 64 bits and rounded once."""
        angles, amplitude = RopeTable.angles(n_positions, rotary_dim, base, **scaling)
        return RopeTable((angles.cos() * amplitude).float().to(device), (angles.sin() * amplitude).float().to(device),
                         interleaved)


_NO_ROPE = (0, None, None, 0, 0)


def _held_elsewhere(gpu: int, *held) -> None:
    for h in held:
        if h is not None:
            _same_gpu(gpu, h._gpu, type(h).__name__)


def _norm(gpu: int, w, dim: int, what: str) -> int:
    _cuda(w, "float32", 1, what)
    _same_gpu(gpu, w.get_device(), what)
    _need(w.shape[0] == dim and w.is_contiguous(), f"{what} must be a contiguous [head_dim]")
    return w.data_ptr()


def rope_append(device: Device, q, k, v, cache: KvCache, batch: KvBatch, rope: Optional[RopeTable], q_out, q_norm=None,
                k_norm=None, eps: float = 1e-6, positions=None, stream: Optional[int] = None) -> None:
    """vw_rope_append: q [n, n_q_heads, D], k and v [n, n_kv_heads, D] (float32 or bfloat16, views of one projection
    allowed) are normalised per head (weights q_norm / k_norm [D] float32; None: not), turned to their positions (int32
    [n], rows of the table; None: each key's index) and rounded to bfloat16; q goes to q_out, k and v into the cache.
    rope None: nothing turns."""
    gpu = device.device
    if cache._gpu != gpu or batch._gpu != gpu or (rope is not None and rope._gpu != gpu):
        _held_elsewhere(gpu, cache, batch, rope)
    dtype, shape = q.dtype, q.shape
    if dtype is not _BF16 and dtype is not _F32:
        raise TypeError(f"q, k and v must be float32 or bfloat16, got {dtype}")
    n, heads, dim = shape if len(shape) == 3 else (0, 0, -1)
    _need(dim == cache.head_dim, "q must be [n, Hq, D] of the cache's D")
    kv = (n, cache.n_kv_heads, dim)
    q_ptr, q_row, q_head = _rows(gpu, q, dtype, shape, "q")
    k_ptr, k_row, k_head = _rows(gpu, k, dtype, kv, "k")
    v_ptr, v_row, v_head = _rows(gpu, v, dtype, kv, "v")
    out_ptr, out_row, out_head = _rows(gpu, q_out, _BF16, shape, "q_out")
    at = None
    if positions is not None:
        _cuda(positions, "int32", 1, "positions")
        _same_gpu(gpu, positions.get_device(), "positions")
        _need(positions.shape[0] == n and positions.is_contiguous(), "positions must be a contiguous [n]")
        at = positions.data_ptr()
    n_positions, cos, sin, rotary, interleaved = _NO_ROPE if rope is None else rope._c
    rows = VwRopeRows(q_ptr, k_ptr, v_ptr, q_row, q_head, k_row, k_head, v_row, v_head,
                      VW_F32 if dtype is _F32 else VW_BF16, heads,
                      None if q_norm is None else _norm(gpu, q_norm, dim, "q_norm"),
                      None if k_norm is None else _norm(gpu, k_norm, dim, "k_norm"), eps, n_positions, cos, sin, at, rotary,
                      interleaved, out_ptr, out_row, out_head)
    _call(lib.vw_rope_append, device, stream, cache._ref, batch._rows(n), ctypes.byref(rows))


def _attn_rows(gpu: int, q, out, lse, cache: KvCache, scale: Optional[float]):
    shape = q.shape
    n, heads, dim = shape if len(shape) == 3 else (0, 0, -1)
    _need(dim == cache.head_dim, "q must be [n, Hq, D] of the cache's D")
    q_ptr, q_row, q_head = _rows(gpu, q, _BF16, shape, "q")
    out_ptr, out_row, out_head = _rows(gpu, out, _BF16, shape, "out")
    lse_ptr = None
    if lse is not None:
        _cuda(lse, "float32", 2, "lse")
        _same_gpu(gpu, lse.get_device(), "lse")
        _need(lse.shape == (n, heads) and lse.is_contiguous(), "lse must be a contiguous [n, Hq]")
        lse_ptr = lse.data_ptr()
    return n, VwAttnRows(q_ptr, q_row, q_head, heads, dim ** -0.5 if scale is None else scale, out_ptr, out_row, out_head,
                         lse_ptr)


def prompt_attention(device: Device, q, cache: KvCache, batch: KvBatch, out, scale: Optional[float] = None, lse=None,
                     stream: Optional[int] = None) -> None:
    """vw_prompt_attention: causal attention of packed sequences over their keys in the cache.  q and out
    [n, n_q_heads, D] bfloat16 (batch.q_offsets gives each sequence's rows, its last keys), scale 1/sqrt(D) unless
    given, lse optionally [n, n_q_heads] float32.  Rows that see no key get 0 and -inf."""
    gpu = device.device
    if cache._gpu != gpu or batch._gpu != gpu:
        _held_elsewhere(gpu, cache, batch)
    n, rows = _attn_rows(gpu, q, out, lse, cache, scale)
    _call(lib.vw_prompt_attention, device, stream, cache._ref, batch._rows(n), ctypes.byref(rows))


def decode_attention(device: Device, q, cache: KvCache, batch: KvBatch, out, prefix: Optional[KvPrefix] = None,
                     scale: Optional[float] = None, lse=None, stream: Optional[int] = None) -> None:
    """vw_decode_attention: one row per sequence (row s is sequence s; batch.q_offsets is ignored) over all of its keys
    and, with `prefix`, those its group shares, which are read once for the group.  Tensors as in prompt_attention."""
    gpu = device.device
    if cache._gpu != gpu or batch._gpu != gpu or (prefix is not None and prefix._gpu != gpu):
        _held_elsewhere(gpu, cache, batch, prefix)
    n, rows = _attn_rows(gpu, q, out, lse, cache, scale)
    _call(lib.vw_decode_attention, device, stream, cache._ref, batch._rows(n), None if prefix is None else prefix._ref,
          ctypes.byref(rows))
