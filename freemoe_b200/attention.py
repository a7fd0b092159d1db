"""The attention side of a decoder layer over the C ABI: RMS norm with the
residual's addition, rotary positions with the write into a paged K/V cache,
and attention of new tokens over that cache.

Like :mod:`freemoe_b200.hotpath` these are thin calls through
``libfreemoe_b200.so`` on torch tensors; outputs and workspaces are allocated
on the stream of the call (``stream``, or torch's current one).  The calls are
short, so their tensors are taken apart in C++ (``csrc/torch_calls.cpp``) and not
through ctypes.  A cache is a tensor ``[pages, kv_heads, page_size, head_dim]``
with any strides but the last (token-major pages are its ``permute(0, 2, 1, 3)``
view).
"""
from __future__ import annotations

import ctypes as C
import importlib.util

import torch

from ._lib import (ROPE_BANDS, ROPE_BASE, ROPE_LINEAR, ROPE_PLAIN, ROPE_RAMP, FmError, RopeScaling, check, load)
from .build import torch_calls_path

FP8_GROUP = 128
_ROPE_KINDS = {"plain": ROPE_PLAIN, "linear": ROPE_LINEAR, "base": ROPE_BASE, "ramp": ROPE_RAMP, "bands": ROPE_BANDS}
INVALID_ARGUMENT, SHAPE_MISMATCH = 26, 8


class _Calls:
    """The entry points for torch tensors, loaded and given the library's addresses at
    their first use; a missing build is an error, there is no fallback."""

    def __getattr__(self, name: str):
        path = torch_calls_path()
        if not path.exists():
            raise FmError(24, f"{path} is missing: build it with `python freemoe_b200/build.py`")
        spec = importlib.util.spec_from_file_location("_torch_calls", path)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        lib = load()
        module.bind(FmError, *(C.cast(getattr(lib, f), C.c_void_p).value for f in (
            "fmcuda_last_error", "fmcuda_add_rms_norm", "fmcuda_rope_append", "fmcuda_paged_attention_workspace_bytes",
            "fmcuda_paged_attention")))
        for f in ("add_rms_norm", "add_rms_norm_fp8", "rope_append", "paged_attention"):
            setattr(self, f, getattr(module, f))
        return getattr(self, name)


_calls = _Calls()


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
                 epsilon: float = 1e-5, out_dtype: torch.dtype | None = None, stream=None):
    """``h = x + residual``, ``y = h * weight / sqrt(mean(h^2) + epsilon)``
    (``fmcuda_add_rms_norm``).

    ``x`` is [tokens, d_model]; returns ``(y, h)``, ``h`` in the residual's type
    and None without one."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return _calls.add_rms_norm(x, weight, residual, epsilon, out_dtype)
    return _calls.add_rms_norm(x, weight, residual, epsilon, out_dtype)


def add_rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, *, residual: torch.Tensor | None = None,
                     epsilon: float = 1e-5, stream=None):
    """The norm with an 8-bit output: ``(codes, scales, h)``, codes
    ``float8_e4m3fn`` [tokens, d_model] and one f32 scale for each 128 values
    of a row: ``y ~ codes * scales``."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return _calls.add_rms_norm_fp8(x, weight, residual, epsilon)
    return _calls.add_rms_norm_fp8(x, weight, residual, epsilon)


def rope_frequencies(rot_dim: int, base: float = 10000.0, *, kind: str = "plain", factor: float = 1.0,
                     trained_context: float = 0.0, fast: float = 0.0, slow: float = 0.0, device="cuda"):
    """Rotary frequencies, scaled for contexts longer than the trained one:
    ``(inv_freq [rot_dim / 2] f32, attention_factor)`` (``fmcuda_rope_frequencies``).

    ``kind``: "plain", "linear", "base", "ramp" or "bands"."""
    if kind not in _ROPE_KINDS:
        raise FmError(INVALID_ARGUMENT, f"unknown rotary scaling {kind!r}")
    if rot_dim < 0:
        raise FmError(SHAPE_MISMATCH, "rotary width must be even, 2 to 1024")
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
    rotated q in the caches' type (``out_dtype`` without caches)
    (``fmcuda_rope_append``).

    ``positions`` int32 [tokens]; ``inv_freq`` f32, one per rotated pair."""
    if stream is not None:
        with torch.cuda.stream(stream):
            return _calls.rope_append(q, k, v, positions, inv_freq, k_cache, v_cache, slots, interleaved,
                                      attention_factor, out_dtype)
    return _calls.rope_append(q, k, v, positions, inv_freq, k_cache, v_cache, slots, interleaved, attention_factor,
                              out_dtype)


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
    out, lse = _calls.paged_attention(q, k_cache, v_cache, page_table, q_start, kv_len, max_q_len, max_kv_len, scale,
                                      causal, window, return_lse, workspace)
    return (out, lse) if return_lse else out
