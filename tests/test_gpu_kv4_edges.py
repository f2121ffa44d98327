"""Edges of the serving step over the 4-bit paged cache. Bounds of the attention are those of
test_gpu_paged_kv4.py unless a test derives its own."""
import pytest
import torch

from oracle import kv4_oracle as O
from tests.test_gpu_paged_kv4 import _case, _check
from tritonllmcompiler_b200.ops.paged_kv4 import (new_kv4_cache, paged_attention_kv4,
                                                  paged_kv4_append, paged_kv4_gather)

pytestmark = pytest.mark.gpu
F, BF = torch.float16, torch.bfloat16


def _newest(case, bs, k=None, v=None):
    """Replaces the newest token of the first sequence in the case's cache and values."""
    _, cache, table, ctx, _, ks, vs = case
    last = int(ctx[0]) - 1
    if k is not None:
        ks[last] = k
    if v is not None:
        vs[last] = v
    slot = (table[0, last // bs] * bs + last % bs).view(1).cuda()
    paged_kv4_append(ks[last:last + 1].cuda(), vs[last:last + 1].cuda(), cache, slot, block_size=bs)


def _attend(case, new, bs, **how):
    q, cache, table, ctx, cu, _, _ = case
    return paged_attention_kv4(q.cuda(), cache, table.cuda(), ctx.cuda(), cu.cuda(), max(new), block_size=bs, **how)


@pytest.mark.parametrize("new", [[1, 1], [7, 1], [60, 1]])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("D", [64, 128])
def test_fp16_values_that_round_past_the_largest(cuda_device, D, which, new):
    """Groups from -60000 to 65504: a scale rounded to the nearest would put their largest code at 65520,
    which is no fp16 number. Rows that see the newest token get what it stands for, and the others what they
    had (bit for bit from the kernel for many rows; the one for few scales its weights by the tile's
    largest scale, seen or not)."""
    lens = [90, 33]
    case = _case(20, lens, new, 2, 4, D, 16, F)
    scale = 2.0 ** -20 if which == "k" else None
    before = _attend(case, new, 16, sm_scale=scale)
    wide = torch.linspace(-60000, 65504, 32).to(F).repeat(2, D // 32)
    _newest(case, 16, **{which: wide})
    got = _check(case, lens, new, 16, F, scale=scale, norm=False)
    assert got.isfinite().all()
    if 4 * max(new) > 32:
        assert torch.equal(got[:new[0] - 1], before[:new[0] - 1])


@pytest.mark.parametrize("D", [64, 128])
def test_a_foreign_scale_stays_with_its_token(cuda_device, D):
    """A V scale that no append writes (finite, but its largest code is past fp16): NaN in that group of the
    rows that see the token, the others bit for bit as before."""
    lens, new, G = [90, 33], [60, 1], 4
    case = _case(26, lens, new, 1, G, D, 16, F)
    before = _attend(case, new, 16)
    t, W = 89 % 16, D // 32
    at = 18 * D + 2 * (t * W + 1)
    scale = torch.tensor([8368.0], dtype=F).view(torch.uint8)
    zero = torch.tensor([-30000.0], dtype=F).view(torch.uint8)
    page = int(case[2][0, 89 // 16])
    case[1][page, 0, 0, at:at + 2] = scale.cuda()
    case[1][page, 0, 0, 19 * D + 2 * (16 + t):19 * D + 2 * (16 + t) + 2] = zero.cuda()
    got = _attend(case, new, 16)
    assert torch.equal(got[:59], before[:59]) and torch.equal(got[60:], before[60:])
    assert got[59, :, 32:64].isnan().all()
    rest = torch.cat([got[59, :, :32], got[59, :, 64:]], -1), torch.cat([before[59, :, :32], before[59, :, 64:]], -1)
    assert torch.equal(*rest)


def test_fp16_groups_stay_in_fp16(cuda_device):
    """Whatever an fp16 group holds, its codes stand for fp16 numbers, within a step of the values."""
    g = torch.Generator().manual_seed(6)
    ends = torch.cat([65504 - 32.0 * torch.randint(0, 4, (400, 1), generator=g),
                      -65504 + 131008 * torch.rand(400, 1, generator=g)], 1)
    x = ends[:, 1:] + (ends[:, :1] - ends[:, 1:]) * torch.rand(400, 64, generator=g)
    x[:, [0, 40]], x[:, [1, 41]] = ends[:, :1], ends[:, 1:]
    x = x.to(F).view(400, 1, 64)
    cache = new_kv4_cache(25, 1, 16, 64)
    slots = torch.arange(400, dtype=torch.int32).cuda()
    paged_kv4_append(x.cuda(), -x.cuda(), cache, slots, block_size=16)
    step = (ends[:, 0] - ends[:, 1]).abs().view(400, 1, 1) / 15
    for got, want in zip(paged_kv4_gather(cache, slots, block_size=16), (x, -x)):
        codes, s, z = O.quantise(want.float().numpy())
        assert torch.equal(got.cpu(), torch.from_numpy(O.dequantise(codes, s, z)[0]).to(F))
        # half a step, 15 steps of the scale's rounding (2^-10 at most), and fp16's
        err = (got.cpu().double() - want.double()).abs()
        assert (err <= step * (0.5 + 15 * 2.0 ** -10) + 2.0 ** -11 * want.double().abs()).all()
