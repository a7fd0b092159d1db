"""The outputs of the calls for torch tensors are torch's own: dispatch modes and the profiler see
them allocated, deterministic algorithms find fresh memory filled, inference mode makes inference
tensors of them."""
from __future__ import annotations

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def tensor(*shape, dtype=BF16, seed=0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda").to(dtype)


def calls():
    """Each call, and the tensors that it allocates."""
    from freemoe_b200 import attention, hotpath

    x, r, w = tensor(5, 256), tensor(5, 256, seed=1), torch.ones(256, device="cuda")
    q, k, v = tensor(5, 4, 64), tensor(5, 2, 64, seed=1), tensor(5, 2, 64, seed=2)
    caches = [torch.zeros(2, 2, 8, 64, dtype=BF16, device="cuda") for _ in range(2)]
    at = torch.arange(5, dtype=torch.int32, device="cuda")
    slots, freq = at.long(), torch.ones(32, device="cuda")
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    lens = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 5], [9])]
    logits = tensor(5, 1000, dtype=F32)
    return {
        "norm": (lambda: attention.add_rms_norm(x, w, residual=r), 2),
        "norm to 8 bits": (lambda: attention.add_rms_norm_fp8(x, w, residual=r), 3),
        "norms": (lambda: attention.norm_add_norm(x, w, r, w), 2),
        "norms to 8 bits": (lambda: attention.norm_add_norm_fp8(x, w, r, w), 3),
        "rotation": (lambda: attention.rope_append(q, k, v, at, freq, *caches, slots), 1),
        "attention": (lambda: attention.paged_attention(q, *caches, table, *lens, max_q_len=5, max_kv_len=9,
                                                        return_lse=True), 2),
        "probabilities": (lambda: hotpath.token_logprobs(logits, at, top=3), 4),
    }


NAMES = ["norm", "norm to 8 bits", "norms", "norms to 8 bits", "rotation", "attention", "probabilities"]


def tensors(result):
    return [t for t in (result if isinstance(result, tuple) else (result,)) if t is not None]


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.made = 0

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.made += func.overloadpacket in (torch.ops.aten.empty, torch.ops.aten.empty_strided)
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("name", NAMES)
def test_a_dispatch_mode_sees_them(cuda, name):
    call, made = calls()[name]
    want = tensors(call())
    with Seen() as seen:
        got = tensors(call())
    assert seen.made == made
    for a, b in zip(want, got):
        assert a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a.float(), b.float())


@pytest.mark.parametrize("name", NAMES)
def test_the_profiler_sees_them(cuda, name):
    call, made = calls()[name]
    call()
    with torch.autograd.profiler.profile() as seen:
        call()
    assert sum(e.count for e in seen.key_averages() if e.key in ("aten::empty", "aten::empty_strided")) == made


@pytest.mark.parametrize("name", NAMES)
def test_inference_mode(cuda, name):
    call, _ = calls()[name]
    assert not any(t.is_inference() or t.requires_grad for t in tensors(call()))
    with torch.inference_mode():
        assert all(t.is_inference() for t in tensors(call()))


def test_deterministic_algorithms_fill_fresh_memory(cuda):
    """Rows behind the last sequence, which attention does not write, are not what lay there."""
    from freemoe_b200 import attention

    q, caches = tensor(70, 4, 64), [tensor(2, 2, 8, 64, seed=i) for i in (1, 2)]
    table = torch.tensor([[0, 1]], dtype=torch.int32, device="cuda")
    lens = [torch.tensor(t, dtype=torch.int32, device="cuda") for t in ([0, 5], [9])]

    def call():
        return attention.paged_attention(q, *caches, table, *lens, max_q_len=5, max_kv_len=9, return_lse=True)

    for left in (1.0, 2.0):
        used = [torch.full((n,), left, dtype=t, device="cuda") for n, t in ((70 * 256, BF16), (280, F32)) for _ in range(8)]
        del used  # what the next outputs may lie on
        want = call()
    torch.use_deterministic_algorithms(True)
    try:
        for left in (1.0, 2.0):
            used = [torch.full((n,), left, dtype=t, device="cuda") for n, t in ((70 * 256, BF16), (280, F32)) for _ in range(8)]
            del used
            out, lse = call()
            assert out[5:].isnan().all() and lse[5:].isnan().all()
            assert torch.equal(out[:5], want[0][:5]) and torch.equal(lse[:5], want[1][:5])
    finally:
        torch.use_deterministic_algorithms(False)


@pytest.mark.parametrize("name", NAMES)
def test_calls_with_deterministic_algorithms(cuda, name):
    call, _ = calls()[name]
    want = tensors(call())
    torch.use_deterministic_algorithms(True)
    try:
        got = tensors(call())
    finally:
        torch.use_deterministic_algorithms(False)
    for a, b in zip(want, got):
        assert a.stride() == b.stride() and torch.equal(a.float(), b.float())
