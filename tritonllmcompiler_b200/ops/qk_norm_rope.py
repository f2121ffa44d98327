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
from torch.autograd.function import once_differentiable

from tritonllmcompiler_b200 import _lib


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


def _rows_ok(stride: tuple) -> bool:
    return stride[2] == 1 and stride[0] % 8 == 0 and stride[1] % 8 == 0


def _table_ok(stride: tuple) -> bool:
    return stride[1] == 1 and stride[0] % 4 == 0


@functools.lru_cache(maxsize=256)
def _checked(q, sq, k, sk, wq, swq, wk, swk, cos, scos, sin, ssin, pos, spos, dtypes, sections, interleaved,
             *grads):
    """Checks a set of shapes, strides and types, once (a call's checks took longer than the kernel at
    one decode step). Returns what the library takes of them, or None where something has to be
    copied first."""
    assert len(q) == 3 and len(k) == 3 and k[0] == q[0]
    t, _, d = q
    assert d in (16, 32, 64, 128) and k[2] == d
    dtype, k_dtype, wq_dtype, wk_dtype, cos_dtype, sin_dtype, pos_dtype = dtypes[:7]
    assert dtype in _lib.DTYPE_CODES and k_dtype == dtype
    assert wq == (d,) and wk == (d,) and wq_dtype == dtype and wk_dtype == dtype
    assert len(cos) == 2 and cos[1] == d // 2 and sin == cos
    assert cos_dtype == torch.float32 and sin_dtype == torch.float32
    axes = 1 if len(pos) == 1 else pos[0]
    assert len(pos) in (1, 2) and pos[-1] == t and pos_dtype in _lib.INTEGERS
    sections = (d // 2,) if sections is None else sections
    assert axes == len(sections), "one row of positions per section"
    words = _axis_words(sections, interleaved, d // 2)
    if grads:
        assert grads[0] == q and grads[2] == k and dtypes[7] == dtype and dtypes[8] == dtype
    ready = all(_rows_ok(x) for x in (sq, sk, *grads[1::2])) and swq == (1,) and swk == (1,)
    ready = ready and _table_ok(scos) and _table_ok(ssin) and pos_dtype == torch.int32 and spos[-1] == 1
    if not ready:
        return None
    table = (cos[0], scos[0], ssin[0], axes, spos[0] if len(pos) == 2 else t, words)
    return (t, q[1], k[1], d), table, [_lib.int64s(*s[:2]) for s in (*grads[1::2], sq, sk)], \
        [_lib.int64s(x[1] * d, d) for x in (q, k)], _lib.DTYPE_CODES[dtype]


def _arguments(tensors, sections, interleaved):
    """(tensors as the library takes them, what _checked gives): q, k, weights, cos, sin, positions and,
    for the backward pass, the gradients of the two outputs."""
    q, k, wq, wk, cos, sin, pos = tensors[:7]
    if sections is not None and type(sections) is not tuple:
        sections = tuple(sections)
    device = q.get_device()
    assert device >= 0 and all([x.get_device() == device for x in tensors])
    address = q.data_ptr() | k.data_ptr() | wq.data_ptr() | wk.data_ptr() | cos.data_ptr() | sin.data_ptr()
    more = ()
    if len(tensors) > 7:
        dqo, dko = tensors[7:]
        address |= dqo.data_ptr() | dko.data_ptr()
        more = (dqo.shape, dqo.stride(), dko.shape, dko.stride())
    known = _checked(q.shape, q.stride(), k.shape, k.stride(), wq.shape, wq.stride(), wk.shape,
                     wk.stride(), cos.shape, cos.stride(), sin.shape, sin.stride(), pos.shape,
                     pos.stride(), tuple([x.dtype for x in tensors]), sections, bool(interleaved), *more)
    if known is None or address % 16:
        return _arguments(_readable(tensors), sections, interleaved)
    return tensors, known, device


def _readable(tensors):
    """The tensors with those that the library cannot read where they are copied."""
    def fix(i, x):
        s = x.stride()
        if i == 6:
            x = _lib.int32(x)
            return x if x.stride()[-1] == 1 else x.clone(memory_format=torch.contiguous_format)
        ok = s == (1,) if i in (2, 3) else _table_ok(s) if i in (4, 5) else _rows_ok(s)
        return x if ok and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)

    return tuple([fix(i, x) for i, x in enumerate(tensors)])


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
    says while the pairs last, and the first axis all others. A position outside the table uses
    row 0 and is flagged (``_lib.debug_status()`` returns 0x200). Returns new contiguous tensors."""
    (q, k, wq, wk, cos, sin, pos), (sizes, table, strides, out_strides, code), device = _arguments(
        (q, k, q_weight, k_weight, cos, sin, positions), sections, interleaved)
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    _lib.launch(device, _lib.load().tllm_qk_norm_rope, q.data_ptr(), k.data_ptr(), wq.data_ptr(),
                wk.data_ptr(), cos.data_ptr(), sin.data_ptr(), pos.data_ptr(), qo.data_ptr(),
                ko.data_ptr(), *sizes, *table, *strides, *out_strides, eps, code)
    return qo, ko


def qk_norm_rope_backward(dq_out: torch.Tensor, dk_out: torch.Tensor, q: torch.Tensor,
                          k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                          cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, *,
                          sections: tuple | None = None, interleaved: bool = False,
                          eps: float = 1e-6):
    """(dq, dk, dq_weight, dk_weight) of ``qk_norm_rope`` at its inputs, given the gradients of
    its two outputs. The norms are recomputed from q and k; the weights' gradients are summed in
    fp32 in a fixed order, so equal inputs give equal bits."""
    (q, k, wq, wk, cos, sin, pos, dqo, dko), (sizes, table, strides, out_strides, code), device = _arguments(
        (q, k, q_weight, k_weight, cos, sin, positions, dq_out, dk_out), sections, interleaved)
    dq = torch.empty_like(q, memory_format=torch.contiguous_format)
    dk = torch.empty_like(k, memory_format=torch.contiguous_format)
    dwq, dwk = torch.empty_like(wq), torch.empty_like(wk)
    lib = _lib.load()
    ws_bytes = lib.tllm_qk_norm_rope_bwd_workspace_size(*sizes)
    ws = cos.new_empty((ws_bytes // 4 + 4,))
    _lib.launch(device, lib.tllm_qk_norm_rope_bwd, dqo.data_ptr(), dko.data_ptr(), q.data_ptr(),
                k.data_ptr(), wq.data_ptr(), wk.data_ptr(), cos.data_ptr(), sin.data_ptr(),
                pos.data_ptr(), dq.data_ptr(), dk.data_ptr(), dwq.data_ptr(), dwk.data_ptr(),
                ws.data_ptr(), ws_bytes, *sizes, *table, *strides, *out_strides, eps, code)
    return dq, dk, dwq, dwk


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, cos, sin, positions, sections, interleaved, eps):
        ctx.save_for_backward(q, k, q_weight, k_weight, cos, sin, positions)
        ctx.how = dict(sections=sections, interleaved=interleaved, eps=eps)
        return qk_norm_rope(q, k, q_weight, k_weight, cos, sin, positions, **ctx.how)

    @staticmethod
    @once_differentiable  # a second derivative is an error, not left out of a sum
    def backward(ctx, dq_out, dk_out):
        grads = qk_norm_rope_backward(dq_out, dk_out, *ctx.saved_tensors, **ctx.how)
        return (*grads, None, None, None, None, None, None)


def qk_norm_rope_train(q, k, q_weight, k_weight, cos, sin, positions, *, sections=None,
                       interleaved=False, eps: float = 1e-6):
    """``qk_norm_rope`` with a backward pass (torch autograd, once) for q, k and the two weights."""
    return _QkNormRope.apply(q, k, q_weight, k_weight, cos, sin, positions, sections, interleaved,
                             eps)
