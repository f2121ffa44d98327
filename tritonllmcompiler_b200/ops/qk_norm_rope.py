"""Per-head RMS norms of queries and keys with a rotation by positions of several axes, in one
pass, with a backward pass.

The reference's ``rmsnorm_rope`` (python/triton_llm/ops/rmsnorm_rope.py:51-75) norms and rotates
one tensor by one position per row and is forward only. ``qk_norm_rope`` takes the queries and the
keys of a packed batch (views of one projection's output, each with its own weight), any position
per token, and up to four position axes (time, height, width of image and video tokens), each
owning a section of the rotary pairs. ``qk_norm_rope_backward`` gives the gradients of both inputs
and both weights; ``qk_norm_rope_train`` wraps the two in a ``torch.autograd.Function``. These are
extensions: the package root and ``ops`` keep the reference's four exports.

Unlike ``rmsnorm_rope`` the normed value is not rounded before the rotation, and the cos/sin
tables are fp32 with one column per rotary pair.
"""
from __future__ import annotations

import ctypes
import functools

import torch

from tritonllmcompiler_b200 import _lib


def _ok(t: torch.Tensor) -> bool:
    s = t.stride()
    return s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and t.data_ptr() % 16 == 0


@functools.lru_cache(maxsize=64)
def _axis_words(sections: tuple, interleaved: bool, half: int):
    """The axis of each rotary pair, 2 bits each, as the library takes them."""
    assert 1 <= len(sections) <= 4 and all(n >= 0 for n in sections) and sum(sections) == half, \
        f"sections {sections} do not add up to {half} rotary pairs of at most 4 axes"
    if interleaved:
        axes = [0] * half
        for a, n in list(enumerate(sections))[1:]:
            for i in range(a, min(len(sections) * n, half), len(sections)):
                axes[i] = a
    else:
        axes = [a for a, n in enumerate(sections) for _ in range(n)]
    words = (ctypes.c_uint32 * 4)()
    for i, a in enumerate(axes):
        words[i // 16] |= a << (2 * (i % 16))
    return words


def _arguments(q, k, q_weight, k_weight, cos, sin, positions, sections, interleaved):
    """Checks shared by both directions; the tensors as the library takes them."""
    assert q.is_cuda and q.dim() == 3 and k.dim() == 3 and k.shape[0] == q.shape[0]
    t, _, d = q.shape
    assert d in (16, 32, 64, 128) and k.shape[2] == d
    assert q.dtype in _lib.DTYPE_CODES and k.dtype == q.dtype
    assert q_weight.shape == (d,) and k_weight.shape == (d,)
    assert q_weight.dtype == q.dtype and k_weight.dtype == q.dtype
    assert cos.dim() == 2 and cos.shape[1] == d // 2 and sin.shape == cos.shape
    assert cos.dtype == torch.float32 and sin.dtype == torch.float32
    if positions.dim() == 1:
        positions = positions.unsqueeze(0)
    assert positions.dim() == 2 and positions.shape[1] == t
    sections = (d // 2,) if sections is None else tuple(sections)
    assert positions.shape[0] == len(sections), "one row of positions per section"
    for x in (k, q_weight, k_weight, cos, sin, positions):
        assert x.device == q.device
    words = _axis_words(sections, bool(interleaved), d // 2)
    if positions.dtype != torch.int32 or positions.stride(1) != 1:
        positions = positions.to(torch.int32).contiguous()
    q, k = (x if _ok(x) else x.contiguous() for x in (q, k))
    vec = lambda x, m: x.stride(-1) == 1 and x.stride(0) % m == 0 and x.data_ptr() % 16 == 0  # noqa: E731
    cos, sin = (x if vec(x, 4) else x.contiguous() for x in (cos, sin))
    q_weight, k_weight = (x if vec(x, 1) else x.contiguous().clone() for x in (q_weight, k_weight))
    return q, k, q_weight, k_weight, cos, sin, positions, words


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
                 sections: tuple | None = None, interleaved: bool = False,
                 eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor]:
    """RMS norm over D of every head of q [T, Hq, D] and k [T, Hkv, D], times q_weight / k_weight
    [D], then the rotate-half rotation: rotary pair i of token t (elements i and i + D / 2) turns
    by row positions[a, t], column i of cos / sin ([P, D / 2] fp32), a being the pair's axis.

    positions: [T], or [axes, T] with one row per entry of sections (rotary pairs per axis, adding
    up to D / 2; one axis by default). interleaved=False gives the axes consecutive sections;
    interleaved=True gives axis a > 0 the pairs a, a + axes, a + 2 axes, ..., as many as its section
    says while the pairs last, and the first axis all others. A position outside the table uses row 0 and is flagged
    (``_lib.debug_status()`` returns 0x200). Returns new contiguous tensors."""
    q, k, wq, wk, cos, sin, pos, words = _arguments(q, k, q_weight, k_weight, cos, sin, positions,
                                                    sections, interleaved)
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ko = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    with _lib.on_device(q):
        _lib.check(_lib.load().tllm_qk_norm_rope(
            q.data_ptr(), k.data_ptr(), wq.data_ptr(), wk.data_ptr(), cos.data_ptr(),
            sin.data_ptr(), pos.data_ptr(), qo.data_ptr(), ko.data_ptr(), q.shape[0], q.shape[1],
            k.shape[1], q.shape[2], cos.shape[0], cos.stride(0), sin.stride(0), pos.shape[0],
            pos.stride(0), words, _lib.strides(q, 2), _lib.strides(k, 2), _lib.strides(qo, 2),
            _lib.strides(ko, 2), eps, _lib.DTYPE_CODES[q.dtype], _lib.stream_of(q)))
    return qo, ko


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor,
                          k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                          cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
                          sections: tuple | None = None, interleaved: bool = False,
                          eps: float = 1e-6):
    """(dq, dk, dq_weight, dk_weight) of ``qk_norm_rope`` at its inputs, given the gradients of
    its two outputs. The norms are recomputed from q and k; the weights' gradients are summed in
    fp32 in a fixed order, so equal inputs give equal bits."""
    assert dq_out.shape == q.shape and dk_out.shape == k.shape
    assert dq_out.dtype == q.dtype and dk_out.dtype == q.dtype
    assert dq_out.device == q.device and dk_out.device == q.device
    q, k, wq, wk, cos, sin, pos, words = _arguments(q, k, q_weight, k_weight, cos, sin, positions,
                                                    sections, interleaved)
    dqo, dko = (x if _ok(x) else x.contiguous() for x in (dq_out, dk_out))
    t, hq, d = q.shape
    hkv = k.shape[1]
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk = torch.empty(k.shape, dtype=k.dtype, device=k.device)
    dw = torch.empty((2, d), dtype=q.dtype, device=q.device)
    lib = _lib.load()
    with _lib.on_device(q):
        ws_bytes = lib.tllm_qk_norm_rope_bwd_workspace_size(t, hq, hkv, d)
        ws = torch.empty(max(ws_bytes, 16), dtype=torch.uint8, device=q.device)
        _lib.check(lib.tllm_qk_norm_rope_bwd(
            dqo.data_ptr(), dko.data_ptr(), q.data_ptr(), k.data_ptr(), wq.data_ptr(),
            wk.data_ptr(), cos.data_ptr(), sin.data_ptr(), pos.data_ptr(), dq.data_ptr(),
            dk.data_ptr(), dw.data_ptr(), dw.data_ptr() + d * dw.element_size(), ws.data_ptr(),
            ws_bytes, t, hq, hkv, d, cos.shape[0], cos.stride(0), sin.stride(0), pos.shape[0],
            pos.stride(0), words, _lib.strides(dqo, 2), _lib.strides(dko, 2), _lib.strides(q, 2),
            _lib.strides(k, 2), _lib.strides(dq, 2), _lib.strides(dk, 2), eps,
            _lib.DTYPE_CODES[q.dtype], _lib.stream_of(q)))
    return dq, dk, dw[0], dw[1]


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, sections, interleaved, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.how = dict(sections=sections, interleaved=interleaved, eps=eps)
        return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, **ctx.how)

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        grads = qk_norm_rope_backward(dq_out, dk_out, *ctx.saved_tensors, **ctx.how)
        return (*grads, None, None, None, None, None, None)


def qk_norm_rope_train(q, k, q_weight, k_weight, cos, sin, positions, *, sections=None,
                       interleaved=False, eps: float = 1e-6):
    """``qk_norm_rope`` with a backward pass (torch autograd) for q, k and the two weights."""
    return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, sections, interleaved,
                             eps)
