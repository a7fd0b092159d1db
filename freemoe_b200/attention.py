"""The attention side of a decoder layer over the C ABI: RMS norm with the
residual's addition, rotary positions with the write into a paged K/V cache,
and attention of new tokens over that cache.

Like :mod:`freemoe_b200.hotpath` these are thin calls through
``libfreemoe_b200.so`` on torch tensors; outputs and workspaces are allocated
on the stream of the call.  A cache is a tensor ``[pages, kv_heads, page_size,
head_dim]`` with any strides but the last (token-major pages are its
``permute(0, 2, 1, 3)`` view).
"""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch._C import _cuda_getCurrentRawStream as _raw_stream
from torch._C import _cuda_getDevice as _current_device

from ._lib import (ROPE_BANDS, ROPE_BASE, ROPE_LINEAR, ROPE_PLAIN, ROPE_RAMP, X_BF16, X_E4M3, X_F16, X_F32, FmError,
                   PagedAttentionArgs, RmsNormArgs, RopeAppendArgs, RopeScaling, check, load, packed_entry, packer)

FP8_GROUP = 128
_DTYPES = {torch.float32: X_F32, torch.bfloat16: X_BF16, torch.float16: X_F16}
_NO_DTYPE = -1  # refused by the C entry
_ROPE_KINDS = {"plain": ROPE_PLAIN, "linear": ROPE_LINEAR, "base": ROPE_BASE, "ramp": ROPE_RAMP, "bands": ROPE_BANDS}
INVALID_ARGUMENT, SHAPE_MISMATCH = 26, 8

# A decoding step makes these calls for every layer with a few microseconds of GPU work
# each, so the wrappers test what the C entry cannot see in one expression, pack the
# arguments into bytes, and leave types, strides and alignment to the C entry's checks.
_pack_norm = packer(RmsNormArgs).pack
_pack_rope = packer(RopeAppendArgs).pack
_pack_attention = packer(PagedAttentionArgs).pack


class _Entries:
    """The C entries taking packed arguments, bound at their first use."""

    def __getattr__(self, name: str):
        argtypes = {"norm": ("fmcuda_add_rms_norm", C.c_void_p), "rope": ("fmcuda_rope_append", C.c_void_p),
                    "attention_bytes": ("fmcuda_paged_attention_workspace_bytes", C.c_void_p),
                    "attention": ("fmcuda_paged_attention", C.c_void_p, C.c_uint64, C.c_void_p)}[name]
        fn = packed_entry(*argtypes)
        setattr(self, name, fn)
        return fn


_entries = _Entries()


def _refuse(message: str, code: int = SHAPE_MISMATCH):
    raise FmError(code, message)


def _elsewhere():
    _refuse(f"a tensor is not on the current device, cuda:{torch.cuda.current_device()}", INVALID_ARGUMENT)


def _norm(x, weight, residual, epsilon, y, y_dtype, scales):
    device = x.get_device()
    if device != _current_device() or weight.get_device() != device or (
            residual is not None and residual.get_device() != device):
        _elsewhere()
    tokens, dim = x.shape
    if weight.shape != (dim,) or (residual is not None and residual.shape != x.shape):
        _refuse("norm takes [tokens, d_model], a weight of d_model and a residual like x")
    xs, ys = x.stride(), y.stride()
    dense = (xs[1] == 1 or dim == 1) and (weight.stride(0) == 1 or dim == 1)
    h, rs, r_at, h_at, r_dtype = None, 0, 0, 0, 0
    if residual is not None:
        # h like the residual in memory too: the C entry takes one stride for both
        rs = residual.stride()
        h = torch.empty_strided(residual.shape, rs, dtype=residual.dtype, device=residual.device)
        dense = dense and (rs[1] == 1 or dim == 1)
        rs, r_at, h_at, r_dtype = rs[0], residual.data_ptr(), h.data_ptr(), _DTYPES.get(residual.dtype, _NO_DTYPE)
    if not dense:
        _refuse("norm inputs must be contiguous in their rows")
    rc = _entries.norm(
        _pack_norm(x.data_ptr(), r_at, weight.data_ptr(), y.data_ptr(), h_at, 0 if scales is None else scales.data_ptr(),
                   xs[0], rs, ys[0], _DTYPES.get(x.dtype, _NO_DTYPE), r_dtype, _DTYPES.get(weight.dtype, _NO_DTYPE),
                   y_dtype, tokens, dim, epsilon), _raw_stream(device))
    if rc:
        check(rc)
    return h


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
                 epsilon: float = 1e-5, out_dtype: torch.dtype | None = None, stream=None):
    """``h = x + residual``, ``y = h * weight / sqrt(mean(h^2) + epsilon)``.

    ``x`` is [tokens, d_model]; returns ``(y, h)``, ``h`` in the residual's type
    and None without one."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return add_rms_norm(x, weight, residual=residual, epsilon=epsilon, out_dtype=out_dtype)
    if x.dim() != 2:
        _refuse("norm takes [tokens, d_model]")
    y = torch.empty_like(x, dtype=out_dtype, memory_format=torch.contiguous_format)
    return y, _norm(x, weight, residual, epsilon, y, _DTYPES.get(y.dtype, _NO_DTYPE), None)


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
                     epsilon: float = 1e-5, stream=None):
    """The norm with an 8-bit output: ``(codes, scales, h)``, codes
    ``float8_e4m3fn`` [tokens, d_model] and one f32 scale for each 128 values
    of a row: ``y ~ codes * scales``."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return add_rms_norm_fp8(x, weight, residual=residual, epsilon=epsilon)
    if x.dim() != 2:
        _refuse("norm takes [tokens, d_model]")
    codes = torch.empty_like(x, dtype=torch.float8_e4m3fn, memory_format=torch.contiguous_format)
    scales = x.new_empty((x.shape[0], -(-x.shape[1] // FP8_GROUP)), dtype=torch.float32)
    return codes, scales, _norm(x, weight, residual, epsilon, codes, X_E4M3, scales)


def rope_frequencies(rot_dim: int, base: float = 10000.0, *, kind: str = "plain", factor: float = 1.0,
                     trained_context: float = 0.0, fast: float = 0.0, slow: float = 0.0, device="cuda"):
    """Rotary frequencies, scaled for contexts longer than the trained one:
    ``(inv_freq [rot_dim / 2] f32, attention_factor)`` (``fmcuda_rope_frequencies``).

    ``kind``: "plain", "linear", "base", "ramp" or "bands"."""
    if kind not in _ROPE_KINDS:
        _refuse(f"unknown rotary scaling {kind!r}", INVALID_ARGUMENT)
    if rot_dim < 0:
        _refuse("rotary width must be even, 2 to 1024")
    scaling = RopeScaling(_ROPE_KINDS[kind], factor, trained_context, fast, slow)
    host = (C.c_float * max(1, rot_dim // 2))()
    attention_factor = C.c_float(1.0)
    check(load().fmcuda_rope_frequencies(rot_dim, base, C.byref(scaling), host, C.byref(attention_factor)))
    return torch.tensor(list(host), dtype=torch.float32).to(device), attention_factor.value


def rope_append(q: torch.Tensor, k: torch.Tensor | None, v: torch.Tensor | None, positions: torch.Tensor,
                inv_freq: torch.Tensor, k_cache: torch.Tensor | None, v_cache: torch.Tensor | None,
                slots: torch.Tensor | None, *, interleaved: bool = False, attention_factor: float = 1.0,
                out_dtype: torch.dtype | None = None, stream=None) -> torch.Tensor:
    """Rotates ``q`` [tokens, heads, head_dim] and ``k`` [tokens, kv_heads,
    head_dim] by their positions, writes ``k`` and ``v`` into the caches' pages at
    ``slots`` (int64: page * page_size + row; negative: nowhere) and returns the
    rotated q in the caches' type (``out_dtype`` without caches).

    ``positions`` int32 [tokens]; ``inv_freq`` f32, one per rotated pair."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return rope_append(q, k, v, positions, inv_freq, k_cache, v_cache, slots, interleaved=interleaved,
                               attention_factor=attention_factor, out_dtype=out_dtype)
    if q.dim() != 3:
        _refuse("q is [tokens, heads, head_dim]")
    device = q.get_device()
    if device != _current_device() or positions.get_device() != device or inv_freq.get_device() != device:
        _elsewhere()
    tokens, heads, dim = q.shape
    qs = q.stride()
    if (positions.shape != (tokens,) or positions.dtype != torch.int32 or not positions.is_contiguous() or
            inv_freq.dim() != 1 or inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous()):
        _refuse("positions are int32 [tokens], inv_freq is float32 [rot_dim / 2]")
    dense = qs[2] == 1 or dim == 1
    if k is not None or v is not None or k_cache is not None or v_cache is not None or slots is not None:
        if k is None or v is None or k_cache is None or v_cache is None or slots is None:
            _refuse("k, v, their caches and slots come together", INVALID_ARGUMENT)
        if (k.get_device() != device or v.get_device() != device or k_cache.get_device() != device or
                v_cache.get_device() != device or slots.get_device() != device):
            _elsewhere()
        shape = k.shape
        kv_heads = shape[1] if len(shape) == 3 else -1
        if shape != (tokens, kv_heads, dim) or v.shape != shape:
            _refuse("k and v are [tokens, kv_heads, head_dim]")
        cache, ks, vs, cs = k_cache.shape, k.stride(), v.stride(), k_cache.stride()
        if (len(cache) != 4 or v_cache.shape != cache or v_cache.stride() != cs or cache[1] != kv_heads or
                cache[3] != dim):
            _refuse("caches are [pages, kv_heads, page_size, head_dim], of one layout")
        if slots.shape != (tokens,) or slots.dtype != torch.int64 or not slots.is_contiguous():
            _refuse("slots are int64 [tokens]")
        kind = k_cache.dtype
        if k.dtype != q.dtype or v.dtype != q.dtype or v_cache.dtype != kind or out_dtype not in (None, kind):
            _refuse("q, k and v have one type, the output and the caches have one", INVALID_ARGUMENT)
        dense = dense and (dim == 1 or ks[2] == vs[2] == cs[3] == 1)
        at = (k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), slots.data_ptr())
        strides = (ks[0], ks[1], vs[0], vs[1])
        pages, page_size, cs = cache[0], cache[2], cs[:3]
    else:
        kind = q.dtype if out_dtype is None else out_dtype
        at, strides, kv_heads, pages, page_size, cs = (0,) * 5, (0,) * 4, 0, 0, 0, (0, 0, 0)
    if not dense:
        _refuse("q, k, v and caches must be contiguous in their heads")
    out = torch.empty_like(q, dtype=kind, memory_format=torch.contiguous_format)
    rc = _entries.rope(
        _pack_rope(q.data_ptr(), at[0], at[1], out.data_ptr(), at[2], at[3], positions.data_ptr(), at[4],
                   inv_freq.data_ptr(), qs[0], qs[1], *strides, heads * dim, dim, *cs, _DTYPES.get(q.dtype, _NO_DTYPE),
                   _DTYPES.get(kind, _NO_DTYPE), tokens, heads, kv_heads, dim, 2 * inv_freq.shape[0],
                   1 if interleaved else 0, attention_factor, pages, page_size), _raw_stream(device))
    if rc:
        check(rc)
    return out


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                    q_start: torch.Tensor, kv_len: torch.Tensor, *, max_q_len: int, max_kv_len: int,
                    scale: float | None = None, causal: bool = True, window: int = 0, return_lse: bool = False,
                    workspace: torch.Tensor | None = None, stream=None):
    """Attention of the new tokens ``q`` [tokens, heads, head_dim] over the
    pages of their sequences (``fmcuda_paged_attention``).

    Sequence b has the rows ``q_start[b]:q_start[b + 1]`` and ``kv_len[b]`` keys
    (its new tokens' own among them), key i on page ``page_table[b, i //
    page_size]``; all three are int32 on the device.  ``max_q_len`` and
    ``max_kv_len`` bound the lengths.  ``workspace``: device bytes to use instead
    of allocating (256-byte aligned, not shared with a call that overlaps).
    Returns the output, and with ``return_lse`` the f32 [tokens, heads] log-sum-exp."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return paged_attention(q, k_cache, v_cache, page_table, q_start, kv_len, max_q_len=max_q_len,
                                   max_kv_len=max_kv_len, scale=scale, causal=causal, window=window,
                                   return_lse=return_lse, workspace=workspace)
    if q.dim() != 3 or k_cache.dim() != 4:
        _refuse("q is [tokens, heads, head_dim], caches are [pages, kv_heads, page_size, head_dim]")
    device = q.get_device()
    if (device != _current_device() or k_cache.get_device() != device or v_cache.get_device() != device or
            page_table.get_device() != device or q_start.get_device() != device or kv_len.get_device() != device or
            (workspace is not None and workspace.get_device() != device)):
        _elsewhere()
    tokens, heads, dim = q.shape
    cache, table = k_cache.shape, page_table.shape
    pages, kv_heads, page_size, cache_dim = cache
    qs, cs, ts = q.stride(), k_cache.stride(), page_table.stride()
    if v_cache.shape != cache or v_cache.stride() != cs or cache_dim != dim:
        _refuse("caches are [pages, kv_heads, page_size, head_dim], of one layout")
    kind = q.dtype
    if k_cache.dtype != kind or v_cache.dtype != kind:
        _refuse("q and the caches have one type", INVALID_ARGUMENT)
    seqs = kv_len.shape[0] if kv_len.dim() == 1 else -1
    if len(table) != 2 or table[0] != seqs or q_start.shape != (seqs + 1,):
        _refuse("page_table is [seqs, pages], q_start [seqs + 1], kv_len [seqs]")
    if (page_table.dtype != torch.int32 or q_start.dtype != torch.int32 or kv_len.dtype != torch.int32 or
            not q_start.is_contiguous() or not kv_len.is_contiguous()):
        _refuse("page_table, q_start and kv_len are int32", INVALID_ARGUMENT)
    if max_q_len < 0 or max_kv_len < 0 or window < 0:
        _refuse("lengths must not be negative", INVALID_ARGUMENT)
    if table[1] * page_size < max_kv_len:
        _refuse("page table is shorter than max_kv_len")
    if qs[2] != 1 or cs[3] != 1 or (ts[1] != 1 and table[1] > 1):
        _refuse("q, caches and page_table must be contiguous in their last dimension")
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if return_lse else None
    args = _pack_attention(
        q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0,
        page_table.data_ptr(), q_start.data_ptr(), kv_len.data_ptr(), qs[0], qs[1], heads * dim, dim, cs[0], cs[1], cs[2],
        ts[0], _DTYPES.get(kind, _NO_DTYPE), seqs, tokens, heads, kv_heads, dim, pages, page_size,
        min(max_q_len, tokens), max_kv_len, 1 if causal else 0, window, 1.0 / math.sqrt(dim) if scale is None else scale)
    if workspace is None:
        need = C.c_uint64()
        rc = _entries.attention_bytes(args, C.addressof(need))
        if rc:
            check(rc)
        size = need.value
        at = (workspace := q.new_empty(size, dtype=torch.uint8)).data_ptr() if size else 0
    else:
        at, size = workspace.data_ptr(), workspace.numel() * workspace.element_size()
    rc = _entries.attention(args, at, size, _raw_stream(device))
    if rc:
        check(rc)
    return (out, lse) if return_lse else out
