"""Normed and rotated queries and keys, and their gradients, against 64 bits.

Bounds, per element, with u the unit roundoff of the dtype (2^-11 fp16, 2^-8 bf16): the outputs are
fp32 arithmetic rounded once, so u |z| (half an ulp, doubled for results near a power of two), and
for the fp32 part 2^-18 of the sizes of the added terms: about 2^6 roundings of 2^-24 (sums of up to
128 squares in chains of at most 16, rsqrt within 2 ulp, four products). The weights' gradients add
up to 2^12 rows a lane at most: 2^-12 of the sizes is the sure bound of such a chain; the test's
chains are under 2^7 long, so 2^-16. fp16 results below 2^-14 have absolute steps of 2^-24.
"""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from tritonllmcompiler_b200 import _lib
from tritonllmcompiler_b200.ops.qk_norm_rope import (qk_norm_rope, qk_norm_rope_backward,
                                                     qk_norm_rope_train)

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _case(seed, T, hq, hkv, D, sections, dtype, rows=97, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    qkv = (torch.randn(T, hq + 2 * hkv, D, generator=g) * scale).to(dtype).cuda()
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2)]
    ang = torch.randn(rows, D // 2, generator=g) * 3
    pos = torch.randint(0, rows, (len(sections), T), generator=g, dtype=torch.int32)
    return (qkv[:, :hq], qkv[:, hq:hq + hkv], *w, ang.cos().cuda(), ang.sin().cuda(), pos.cuda())


def _np(t):
    return t.double().cpu().numpy()


def _bounded(got, want, size, dtype, share=2.0 ** -18):
    err = np.abs(_np(got) - want)
    assert np.isfinite(_np(got)).all()
    assert (err <= U[dtype] * np.abs(want) + share * size + 2.0 ** -25).all(), err.max()


CASES = [
    (1, 1, 1, 16, (8,), False, torch.float16),
    (1, 32, 8, 128, (16, 24, 24), False, torch.bfloat16),
    (5, 3, 1, 64, (8, 12, 12), False, torch.float16),  # a section ends inside a lane's 8 pairs
    (37, 9, 3, 64, (12, 10, 10), True, torch.bfloat16),
    (21, 3, 3, 64, (8, 12, 12), True, torch.float16),  # the pairs end before the sections do
    (130, 4, 4, 32, (4, 4, 4, 4), True, torch.float16),
    (63, 8, 8, 128, (64,), False, torch.float16),
    (17, 6, 2, 128, (1, 62, 1), False, torch.float16),
    (2000, 8, 4, 64, (0, 32), False, torch.bfloat16),  # an axis without pairs; several heads a lane
    (700, 16, 8, 128, (24, 20, 20), True, torch.float16),
]


@pytest.mark.parametrize("T,hq,hkv,D,sections,mix,dtype", CASES)
def test_forward(cuda_device, T, hq, hkv, D, sections, mix, dtype):
    q, k, wq, wk, cos, sin, pos = _case(T + D, T, hq, hkv, D, sections, dtype)
    outs = qk_norm_rope(q, k, wq, wk, cos, sin, pos, sections=sections, interleaved=mix)
    for x, w, z in ((q, wq, outs[0]), (k, wk, outs[1])):
        assert z.is_contiguous() and z.dtype == dtype
        args = (_np(x), _np(w), _np(cos), _np(sin), pos.cpu().numpy(), sections, mix)
        y = np.abs(O.norm_rope(args[0], args[1], np.ones_like(args[2]), np.zeros_like(args[3]), *args[4:]))
        size = y + np.roll(y, D // 2, -1)
        _bounded(z, O.norm_rope(*args), size, dtype)
    assert _lib.debug_status() == 0


@pytest.mark.parametrize("T,hq,hkv,D,sections,mix,dtype", CASES)
def test_backward(cuda_device, T, hq, hkv, D, sections, mix, dtype):
    q, k, wq, wk, cos, sin, pos = _case(T + D + 1, T, hq, hkv, D, sections, dtype)
    g = torch.Generator().manual_seed(T)
    dq, dk = (torch.randn(x.shape, generator=g).to(dtype).cuda() for x in (q, k))
    how = dict(sections=sections, interleaved=mix)
    got = qk_norm_rope_backward(dq, dk, q, k, wq, wk, cos, sin, pos, **how)
    again = qk_norm_rope_backward(dq, dk, q, k, wq, wk, cos, sin, pos, **how)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for x, w, dz, dx, dw in ((q, wq, dq, got[0], got[2]), (k, wk, dk, got[1], got[3])):
        want = O.norm_rope_grad(_np(dz), _np(x), _np(w), _np(cos), _np(sin), pos.cpu().numpy(), sections, mix)
        _bounded(dx, want[0], want[2], dtype)
        _bounded(dw, want[1], want[3], dtype, 2.0 ** -16)
    assert _lib.debug_status() == 0


def test_autograd(cuda_device):
    q, k, wq, wk, cos, sin, pos = _case(9, 33, 4, 2, 64, (32,), torch.bfloat16)
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, wq, wk)]
    qo, ko = qk_norm_rope_train(*leaves, cos, sin, pos[0])
    (qo.float().sum() + 2 * ko.float().sum()).backward()  # gradients that are expanded scalars
    ones = lambda t, v: torch.full_like(t, v)  # noqa: E731
    want = qk_norm_rope_backward(ones(qo, 1), ones(ko, 2), q, k, wq, wk, cos, sin, pos)
    assert all(torch.equal(a.grad, b) for a, b in zip(leaves, want))


def test_odd_strides_and_alignment(cuda_device):
    q, k, wq, wk, cos, sin, pos = _case(4, 20, 4, 2, 64, (16, 16), torch.float16)
    ref = qk_norm_rope(q, k, wq, wk, cos, sin, pos, sections=(16, 16))
    wide = torch.zeros(20, 4, 65, dtype=q.dtype, device="cuda")
    wide[..., 1:] = q
    cw = torch.zeros(cos.shape[0], 33, device="cuda")
    cw[:, 1:] = cos
    w2 = torch.zeros(65, dtype=q.dtype, device="cuda")
    w2[1:] = wq
    got = qk_norm_rope(wide[..., 1:], k.transpose(0, 1).contiguous().transpose(0, 1), w2[1:], wk, cw[:, 1:],
                       sin, pos.long().T.contiguous().T, sections=(16, 16))
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])


def test_values_at_the_edges(cuda_device):
    """Zero rows give zeros (and zero gradients through x r), a NaN stays in its row, and large
    values do not overflow the fp32 sums."""
    q, k, wq, wk, cos, sin, pos = _case(5, 6, 2, 1, 128, (64,), torch.bfloat16)
    q = q.contiguous()
    q[0] = 0
    q[1, 0, 5] = float("nan")
    q[2] = 1e18
    qo, _ = qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    assert (qo[0] == 0).all() and qo[1, 0].isnan().all()
    assert qo[1, 1].isfinite().all() and qo[2:].isfinite().all()


def test_positions_outside_the_table_are_flagged(cuda_device):
    q, k, wq, wk, cos, sin, pos = _case(6, 8, 2, 1, 64, (32,), torch.float16)
    bad = pos.clone()
    bad[0, 3], bad[0, 5] = 97, -1
    got = qk_norm_rope(q, k, wq, wk, cos, sin, bad)
    torch.cuda.synchronize()
    assert _lib.debug_status() == 0x200
    pos[0, 3] = pos[0, 5] = 0
    assert torch.equal(got[0], qk_norm_rope(q, k, wq, wk, cos, sin, pos)[0])
    assert _lib.debug_status() == 0


@pytest.mark.parametrize("T,hq,hkv", [(0, 4, 2), (3, 0, 2), (3, 4, 0)])
def test_empty(cuda_device, T, hq, hkv):
    q, k, wq, wk, cos, sin, pos = _case(7, T, hq, hkv, 64, (32,), torch.float16)
    qo, ko = qk_norm_rope(q, k, wq, wk, cos, sin, pos)
    assert qo.shape == q.shape and ko.shape == k.shape
    grads = qk_norm_rope_backward(qo, ko, q, k, wq, wk, cos, sin, pos)
    for x, dw in ((q, grads[2]), (k, grads[3])):
        if x.numel() == 0:
            assert (dw == 0).all()


def test_refused_arguments(cuda_device):
    q, k, wq, wk, cos, sin, pos = _case(8, 4, 2, 1, 64, (32,), torch.float16)
    for bad in (dict(q=q.float()), dict(k=k[:2]), dict(wq=wq[:32]), dict(wq=wq.float()), dict(cos=cos.half()),
                dict(cos=cos[:, :16]), dict(pos=pos[:, :2]), dict(pos=pos.cpu())):
        a = dict(dict(q=q, k=k, wq=wq, wk=wk, cos=cos, sin=sin, pos=pos), **bad)
        with pytest.raises(AssertionError):
            qk_norm_rope(*a.values())
    for sections, mix in (((16, 17), False), ((8,) * 5, False), ((33, -1), True)):
        with pytest.raises(AssertionError):
            qk_norm_rope(q, k, wq, wk, cos, sin, pos.expand(len(sections), -1), sections=sections, interleaved=mix)


# Enough rows that a lane group takes 8, 4 and 2 heads (the last group of a block is not full in one).
@pytest.mark.parametrize("T,hq,hkv,D,sections,mix,dtype", [
    (1901, 32, 8, 128, (16, 24, 24), False, torch.bfloat16),
    (2503, 12, 4, 128, (64,), False, torch.float16),
    (5003, 6, 2, 64, (12, 10, 10), True, torch.bfloat16),
])
def test_many_rows(cuda_device, T, hq, hkv, D, sections, mix, dtype):
    test_forward(cuda_device, T, hq, hkv, D, sections, mix, dtype)
    test_backward(cuda_device, T, hq, hkv, D, sections, mix, dtype)
