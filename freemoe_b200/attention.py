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

import contextlib
import ctypes as C
import math

import torch

from ._lib import (ROPE_BANDS, ROPE_BASE, ROPE_LINEAR, ROPE_PLAIN, ROPE_RAMP, X_BF16, X_E4M3, X_F16, X_F32, FmError,
                   PagedAttentionArgs, RmsNormArgs, RopeAppendArgs, RopeScaling, check, load)

FP8_GROUP = 128
_DTYPES = {torch.float32: X_F32, torch.bfloat16: X_BF16, torch.float16: X_F16}
_ROPE_KINDS = {"plain": ROPE_PLAIN, "linear": ROPE_LINEAR, "base": ROPE_BASE, "ramp": ROPE_RAMP, "bands": ROPE_BANDS}
INVALID_ARGUMENT, SHAPE_MISMATCH = 26, 8


def _dtype(t: torch.dtype) -> int:
    code = _DTYPES.get(t)
    if code is None:
        raise FmError(INVALID_ARGUMENT, f"{t} is not float32, bfloat16 or float16")
    return code


def _need(ok: bool, message: str, code: int = SHAPE_MISMATCH) -> None:
    if not ok:
        raise FmError(code, message)


def _on_device(*tensors) -> None:
    """Device memory of the current device, rows contiguous."""
    device = torch.cuda.current_device()
    for t in tensors:
        if t is not None and (not t.is_cuda or t.device.index != device):
            raise FmError(INVALID_ARGUMENT, f"tensor on {t.device}: the current device is cuda:{device}")


def _dense(what: str, *tensors) -> None:
    """The innermost dimension is contiguous."""
    for t in tensors:
        if t is not None and t.stride(-1) != 1 and t.shape[-1] != 1:
            raise FmError(SHAPE_MISMATCH, f"{what} must be contiguous in its last dimension")


def _stream(stream):
    """The stream's handle, and a context in which torch allocates on it."""
    if stream is None:
        return torch.cuda.current_stream().cuda_stream, contextlib.nullcontext()
    return stream.cuda_stream, torch.cuda.stream(stream)


def _norm(x, weight, residual, epsilon, y, scales, stream):
    _need(x.dim() == 2 and weight.dim() == 1 and weight.shape[0] == x.shape[1],
          "norm takes [tokens, d_model] and a weight of d_model")
    _need(residual is None or residual.shape == x.shape, "residual and x differ in shape")
    _on_device(x, weight, residual)
    _dense("norm input", x, weight, residual)
    h = None
    if residual is not None:
        h = torch.empty_strided(residual.shape, residual.stride(), dtype=residual.dtype, device=x.device)
    a = RmsNormArgs(x.data_ptr(), None if residual is None else residual.data_ptr(), weight.data_ptr(), y.data_ptr(),
                    None if h is None else h.data_ptr(), None if scales is None else scales.data_ptr(),
                    x.stride(0), 0 if residual is None else residual.stride(0), y.stride(0), _dtype(x.dtype),
                    0 if residual is None else _dtype(residual.dtype), _dtype(weight.dtype),
                    X_E4M3 if scales is not None else _dtype(y.dtype), x.shape[0], x.shape[1], epsilon)
    check(load().fmcuda_add_rms_norm(C.byref(a), stream))
    return h


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
                 epsilon: float = 1e-5, out_dtype: torch.dtype | None = None, stream=None):
    """``h = x + residual``, ``y = h * weight / sqrt(mean(h^2) + epsilon)``.

    ``x`` is [tokens, d_model]; returns ``(y, h)``, ``h`` in the residual's type
    and None without one."""
    handle, on_stream = _stream(stream)
    with on_stream:
        y = torch.empty(x.shape, dtype=x.dtype if out_dtype is None else out_dtype, device=x.device)
        return y, _norm(x, weight, residual, epsilon, y, None, handle)


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
                     epsilon: float = 1e-5, stream=None):
    """The norm with an 8-bit output: ``(codes, scales, h)``, codes
    ``float8_e4m3fn`` [tokens, d_model] and one f32 scale for each 128 values
    of a row: ``y ~ codes * scales``."""
    handle, on_stream = _stream(stream)
    _need(x.dim() == 2, "norm takes [tokens, d_model]")
    with on_stream:
        codes = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
        scales = torch.empty((x.shape[0], -(-x.shape[1] // FP8_GROUP)), dtype=torch.float32, device=x.device)
        return codes, scales, _norm(x, weight, residual, epsilon, codes, scales, handle)


def rope_frequencies(rot_dim: int, base: float = 10000.0, *, kind: str = "plain", factor: float = 1.0,
                     trained_context: float = 0.0, fast: float = 0.0, slow: float = 0.0, device="cuda"):
    """Rotary frequencies, scaled for contexts longer than the trained one:
    ``(inv_freq [rot_dim / 2] f32, attention_factor)`` (``fmcuda_rope_frequencies``).

    ``kind``: "plain", "linear", "base", "ramp" or "bands"."""
    if kind not in _ROPE_KINDS:
        raise FmError(INVALID_ARGUMENT, f"unknown rotary scaling {kind!r}")
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
    handle, on_stream = _stream(stream)
    _need(q.dim() == 3, "q is [tokens, heads, head_dim]")
    tokens, heads, dim = q.shape
    _need(positions.shape == (tokens,) and positions.dtype == torch.int32 and positions.is_contiguous(),
          "positions are int32 [tokens]")
    _need(inv_freq.dim() == 1 and inv_freq.dtype == torch.float32 and inv_freq.is_contiguous(),
          "inv_freq is float32 [rot_dim / 2]")
    _on_device(q, k, v, positions, inv_freq, k_cache, v_cache, slots)
    _dense("q, k, v and caches", q, k, v, k_cache, v_cache)
    cached = (k, v, k_cache, v_cache, slots)
    if any(t is not None for t in cached):
        _need(all(t is not None for t in cached), "k, v, their caches and slots come together", INVALID_ARGUMENT)
        _need(k.dim() == 3 and k.shape == v.shape and k.shape[0] == tokens and k.shape[2] == dim,
              "k and v are [tokens, kv_heads, head_dim]")
        kv_heads = k.shape[1]
        _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride() and
              k_cache.shape[1] == kv_heads and k_cache.shape[3] == dim,
              "caches are [pages, kv_heads, page_size, head_dim], of one layout")
        _need(k.dtype == q.dtype and v.dtype == q.dtype, "q, k and v have one type", INVALID_ARGUMENT)
        _need(k_cache.dtype == v_cache.dtype and out_dtype in (None, k_cache.dtype),
              "the output and the caches have one type", INVALID_ARGUMENT)
        _need(slots.shape == (tokens,) and slots.dtype == torch.int64 and slots.is_contiguous(),
              "slots are int64 [tokens]")
        out_dtype = k_cache.dtype
        cache = (k_cache.stride(0), k_cache.stride(1), k_cache.stride(2))
        pages, page_size = k_cache.shape[0], k_cache.shape[2]
        strides = (k.stride(0), k.stride(1), v.stride(0), v.stride(1))
    else:
        kv_heads, pages, page_size, cache, strides = 0, 0, 0, (0, 0, 0), (0, 0, 0, 0)
    with on_stream:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype if out_dtype is None else out_dtype, device=q.device)
    at = [None if t is None else t.data_ptr() for t in (k, v, k_cache, v_cache, slots)]
    a = RopeAppendArgs(q.data_ptr(), at[0], at[1], out.data_ptr(), at[2], at[3], positions.data_ptr(), at[4],
                       inv_freq.data_ptr(), q.stride(0), q.stride(1), *strides, out.stride(0), out.stride(1), *cache,
                       _dtype(q.dtype), _dtype(out.dtype), tokens, heads, kv_heads, dim, 2 * inv_freq.shape[0],
                       1 if interleaved else 0, attention_factor, pages, page_size)
    check(load().fmcuda_rope_append(C.byref(a), handle))
    return out


def paged_attention_workspace_bytes(args: PagedAttentionArgs) -> int:
    v = C.c_uint64(0)
    check(load().fmcuda_paged_attention_workspace_bytes(C.byref(args), C.byref(v)))
    return v.value


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
    handle, on_stream = _stream(stream)
    _need(q.dim() == 3, "q is [tokens, heads, head_dim]")
    tokens, heads, dim = q.shape
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride() and
          k_cache.shape[3] == dim, "caches are [pages, kv_heads, page_size, head_dim], of one layout")
    _need(q.dtype == k_cache.dtype == v_cache.dtype, "q and the caches have one type", INVALID_ARGUMENT)
    seqs = kv_len.shape[0]
    _need(page_table.dim() == 2 and page_table.shape[0] == seqs and q_start.shape == (seqs + 1,) and kv_len.dim() == 1,
          "page_table is [seqs, pages], q_start [seqs + 1], kv_len [seqs]")
    _need(page_table.dtype == q_start.dtype == kv_len.dtype == torch.int32 and q_start.is_contiguous() and
          kv_len.is_contiguous(), "page_table, q_start and kv_len are int32", INVALID_ARGUMENT)
    _need(page_table.shape[1] * k_cache.shape[2] >= max_kv_len, "page table is shorter than max_kv_len")
    _need(max_q_len >= 0 and max_kv_len >= 0 and window >= 0, "lengths must not be negative", INVALID_ARGUMENT)
    _on_device(q, k_cache, v_cache, page_table, q_start, kv_len, workspace)
    _dense("q, caches and page_table", q, k_cache, v_cache, page_table)
    with on_stream:
        out = torch.empty((tokens, heads, dim), dtype=q.dtype, device=q.device)
        lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
        a = PagedAttentionArgs(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
                               None if lse is None else lse.data_ptr(), page_table.data_ptr(), q_start.data_ptr(),
                               kv_len.data_ptr(), q.stride(0), q.stride(1), out.stride(0), out.stride(1),
                               k_cache.stride(0), k_cache.stride(1), k_cache.stride(2), page_table.stride(0),
                               _dtype(q.dtype), seqs, tokens, heads, k_cache.shape[1], dim, k_cache.shape[0],
                               k_cache.shape[2], min(max_q_len, tokens), max_kv_len, 1 if causal else 0, window,
                               1.0 / math.sqrt(dim) if scale is None else scale)
        if workspace is None:
            workspace = torch.empty(paged_attention_workspace_bytes(a), dtype=torch.uint8, device=q.device)
        check(load().fmcuda_paged_attention(C.byref(a), workspace.data_ptr(),
                                            workspace.numel() * workspace.element_size(), handle))
    return (out, lse) if return_lse else out
