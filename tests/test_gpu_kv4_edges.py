"""Edges of the serving step over the 4-bit paged cache. Bounds of the attention are those of
test_gpu_paged_kv4.py unless a test derives its own."""
import math

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from tests.test_gpu_paged_kv4 import U, _case, _check, _np
from tritonllmcompiler_b200 import _lib
from tritonllmcompiler_b200.ops.paged_kv4 import (new_kv4_cache, paged_attention_kv4,
                                                  paged_kv4_append, paged_kv4_gather)
from tritonllmcompiler_b200.ops.paged_plan import paged_plan
from tritonllmcompiler_b200.ops.qk_norm_rope import qk_norm_rope

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


@pytest.mark.parametrize("new", [1, 5, 60])
@pytest.mark.parametrize("length", [64, 65, 96, 128, 129])
@pytest.mark.parametrize("lo,hi", [(-70000, -70000), (-70000, 0), (70000, 70000)])
def test_zeros_beyond_fp16(cuda_device, lo, hi, length, new):
    """A V group with finite scale whose zero is no fp16 number gives no numbers to the rows that see its
    token, wherever in a tile the context ends, and nothing to the others."""
    case = _case(21, [length], [new], 1, 4, 128, 16, BF)
    before = _attend(case, [new], 16)
    v = torch.randn(1, 128, generator=torch.Generator().manual_seed(2))
    v[0, 32:64] = torch.linspace(lo, hi, 32)
    _newest(case, 16, v=v.to(BF))
    got = _attend(case, [new], 16)
    assert torch.equal(got[:-1], before[:-1])
    assert not got[-1, :, 32:64].isfinite().any()
    assert got[-1, :, :32].isfinite().all() and got[-1, :, 64:].isfinite().all()


@pytest.mark.parametrize("scale,zero", [(float("inf"), 1.0), (float("nan"), 1.0), (1.0, float("nan")), (8000.0, 60000.0)])
@pytest.mark.parametrize("D,new", [(64, [1, 3]), (128, [6, 3]), (128, [2, 1])])
def test_any_group_without_numbers_is_hidden(cuda_device, D, new, scale, zero):
    """Scales and zeros of any kind in the newest token and in the next slot, which is no key: the
    first reach the row that sees them, the others no row, whatever the weights are."""
    lens, G, W = [90, 33], 4, D // 32
    case = _case(27, lens, new, 1, G, D, 16, F)
    before = _attend(case, new, 16)
    for b in (0, 1):
        page = int(case[2][b, lens[b] // 16])
        t = lens[b] % 16
        for token in ((t - 1, t) if b == 0 else (t,)):
            for value, at in ((scale, 18 * D + 2 * (token * W)), (zero, 19 * D + 2 * token)):
                case[1][page, 0, 0, at:at + 2] = torch.tensor([value], dtype=F).view(torch.uint8).cuda()
    got = _attend(case, new, 16)
    last = new[0] - 1
    assert torch.equal(got[:last], before[:last]) and torch.equal(got[new[0]:], before[new[0]:])
    assert not got[last, :, :32].isfinite().any() and got[last, :, 32:].isfinite().all()


def test_groups_beyond_fp16_are_no_numbers(cuda_device):
    """Groups with a value that fp16 has no room for read back as NaN, whole, also where their scale and zero
    would be finite; groups that end at its largest bf16 number do not."""
    x = torch.randn(7, 1, 64, generator=torch.Generator().manual_seed(1))
    x[0, 0, :32] = torch.linspace(60000, 200000, 32)
    x[1, 0, :32] = torch.linspace(50000, 100000, 32)
    x[2, 0, :32] = torch.linspace(-70000, 100, 32)
    x[3, 0, :32] = -1e5
    x[4, 0, 5] = float("inf")
    x[5, 0, 5] = float("nan")
    x[6, 0, :32] = torch.linspace(-60000, 65280, 32)
    x = x.to(BF)
    cache = new_kv4_cache(1, 1, 16, 64)
    slots = torch.arange(7, dtype=torch.int32).cuda()
    paged_kv4_append(x.cuda(), -x.cuda(), cache, slots, block_size=16)
    for got, want in zip(paged_kv4_gather(cache, slots, block_size=16, dtype=BF), (x, -x)):
        assert got[:6, 0, :32].isnan().all() and got[:6, 0, 32:].isfinite().all() and got[6].isfinite().all()
        values = torch.from_numpy(O.dequantise(*O.quantise(want.float().numpy()))[0]).to(BF)
        assert torch.equal(got.cpu().nan_to_num(7.0), values.nan_to_num(7.0))


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("length", [64, 65])
@pytest.mark.parametrize("which", ["k", "v"])
def test_attention_over_groups_beyond_fp16(cuda_device, which, length, new):
    """The same NaN from both attention kernels, at any length of the context."""
    case = _case(28, [length], [new], 1, 4, 64, 16, BF)
    before = _attend(case, [new], 16)
    wide = torch.randn(1, 64, generator=torch.Generator().manual_seed(2))
    wide[0, 32:] = torch.linspace(50000, 100000, 32)
    _newest(case, 16, **{which: wide.to(BF)})
    got = _attend(case, [new], 16)
    assert torch.equal(got[:-1], before[:-1])
    assert got[-1].isnan().all() if which == "k" else got[-1, :, 32:].isnan().all() and got[-1, :, :32].isfinite().all()


@pytest.mark.parametrize("new,most", [([5, 1, 9], 4), ([40, 300, 2], 50), ([3, 2, 1], 0), ([1, 70, 1], 1)])
def test_more_new_tokens_than_promised(cuda_device, new, most):
    """Flagged; the first max_new tokens of each sequence are what they are, the others NaN (not what the
    output's memory had), whichever kernel max_new selects."""
    lens = [60, 400, 33]
    case = _case(22, lens, new, 2, 4, 64, 16, F)
    q, cache, table, ctx, cu, _, _ = case
    whole = _check(case, lens, new, 16, F)
    torch.full_like(whole, 7.0)  # in the memory that the output gets
    got = paged_attention_kv4(q.cuda(), cache, table.cuda(), ctx.cuda(), cu.cuda(), most, block_size=16)
    torch.cuda.synchronize()
    assert _lib.debug_status() == 0x200
    for b, n in enumerate(new):
        r, m = int(cu[b]), min(n, most)
        # two kernels or two divisions of the keys: each within its bound, some 2^-9 of values of size 4
        assert ((got[r:r + m].float() - whole[r:r + m].float()).abs() <= 2.0 ** -7).all()
        assert got[r + m:r + n].isnan().all()


@pytest.mark.parametrize("new", [[2, 1], [60, 9]])
def test_rows_before_the_first_sequence_are_zero(cuda_device, new):
    """Some sequences of a larger packed batch: the rows of the others are cleared."""
    lens = [90, 33]
    q, cache, table, ctx, cu, _, _ = _case(23, lens, new, 1, 4, 128, 16, BF)
    ref = paged_attention_kv4(q.cuda(), cache, table.cuda(), ctx.cuda(), cu.cuda(), max(new), block_size=16)
    more = torch.cat([torch.full((21, 4, 128), 3.0, dtype=BF), q, torch.full((5, 4, 128), 3.0, dtype=BF)]).cuda()
    torch.full_like(more, 7.0)
    got = paged_attention_kv4(more, cache, table.cuda(), ctx.cuda(), cu.cuda() + 21, max(new), block_size=16)
    assert (got[:21] == 0).all() and torch.equal(got[21:-5], ref) and (got[-5:] == 0).all()
    one = paged_attention_kv4(q.cuda(), cache, table.cuda()[1:], ctx.cuda()[1:], cu.cuda()[1:], new[1], block_size=16)
    assert (one[:new[0]] == 0).all() and ((one[new[0]:].float() - ref[new[0]:].float()).abs() <= 2.0 ** -5).all()
    assert _lib.debug_status() == 0


def _scores_bounded(q, k, scale, dtype):
    """Decode over tokens whose K are the rows of k [n, D] (read back from the cache) and V one 1 each,
    so that the outputs are the weights, against 64 bits.

    Scores may be off by E = 2^-20 of the sizes of their terms, |q| (code s + |z|): the sums of q are held in
    22 bits, and up to 140 products are added in fp32 or by MMAs that cut off below 2^-23. Each weight changes by
    a factor within 1 +- 2 E, is rounded to 11 bits, or its product with the scale is (2^-10), and the
    output once."""
    n, D = k.shape
    H = q.shape[0]
    cache = new_kv4_cache(1, 1, 16, D)
    v = torch.zeros(n, 1, D, dtype=dtype)
    for t in range(n):
        v[t, 0, 32 * (t % (D // 32)):32 * (t % (D // 32)) + 32] = 1  # token t: group t
    slots = torch.arange(n, dtype=torch.int32).cuda()
    paged_kv4_append(k[:, None].cuda(), v.cuda(), cache, slots, block_size=16)
    codes, s, z = O.quantise(k.float().numpy())
    values, size = O.dequantise(codes, s, z)
    table, ctx = torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    cu = torch.tensor([0, 1], dtype=torch.int32).cuda()
    for h in range(0, H, 8):
        part = q[h:h + 8]
        got = _np(paged_attention_kv4(part[None].cuda(), cache, table, ctx, cu, 1, block_size=16, sm_scale=scale))[0]
        x = values @ _np(part).T * scale  # [n, heads]
        p = np.exp(x - x.max(0))
        p /= p.sum(0)
        E = 2.0 ** -20 * scale * (size @ np.abs(_np(part)).T).max(0)
        for t in range(n):
            bound = (U[dtype] + 2.0 ** -10 + 2 * E) * p[t] + 2.0 ** -24
            assert (np.abs(got[:, 32 * t] - p[t]) <= bound).all(), (t, got[:, 32 * t], p[t], bound)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [F, BF])
def test_scores_of_offset_keys(cuda_device, dtype, D):
    """Keys far from 0, of opposite sign, under queries whose channels nearly cancel: what is left of a
    group's sum is a fraction of the unit of the largest element."""
    rng = np.random.default_rng(3)
    q = torch.zeros(64, D, dtype=torch.float64)
    q[:, 2], q[:, 3] = 2.5, -2.5
    q[:, 4::32] = torch.from_numpy(rng.uniform(0.1, 0.45, (64, 1)) / 2 ** 11)  # (2^12 is 2 to 4 here)
    k = torch.full((2, D), 500.0)
    k[1] = -500
    _scores_bounded(q.to(dtype), k.to(dtype), 1.0, dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [F, BF])
def test_scores_of_random_keys_with_offsets(cuda_device, dtype, D):
    g = torch.Generator().manual_seed(4)
    q = torch.randn(64, D, generator=g)
    k = torch.randn(2, D, generator=g) + 50 * torch.randn(1, D // 32, generator=g).repeat_interleave(32, 1)
    _scores_bounded(q.to(dtype), k.to(dtype), D ** -0.5, dtype)


@pytest.mark.parametrize("dtype", [F, BF])
@pytest.mark.parametrize("log2", [12.0, 16.5, 20.6, -20.6])
@pytest.mark.parametrize("new", [1, 5, 256])
def test_many_keys_of_small_weight(cuda_device, new, log2, dtype):
    """One key of weight 1 and value 0 (first, or with log2 < 0 last of all), thousands of weight 2^-|log2| and
    value 1: what the rows get is the small weights' sum. Bound as in test_gpu_paged_kv4.py, with the score of
    the one key, |log2| ln 2, as the size of all terms. A run of a worker holds some 40 tiles here where there
    are many rows."""
    n, D, Hkv, G, bs, B = 5000, 64, 8, 4, 64, 2
    blocks = -(-n // bs)
    one = 0 if log2 > 0 else n - new
    k, v = torch.zeros(n, Hkv, D, dtype=dtype), torch.ones(n, Hkv, D, dtype=dtype)
    k[one], v[one] = 1, 0
    cache = new_kv4_cache(blocks, Hkv, bs, D)
    paged_kv4_append(k.cuda(), v.cuda(), cache, torch.arange(n, dtype=torch.int32).cuda(), block_size=bs)
    table = torch.arange(blocks, dtype=torch.int32).expand(B, -1).cuda()
    cu = torch.arange(0, B * new + 1, new, dtype=torch.int32).cuda()
    q = torch.ones(B * new, Hkv * G, D, dtype=dtype, device="cuda")
    size = abs(log2) * math.log(2)
    got = _np(paged_attention_kv4(q, cache, table, torch.full((B,), n, dtype=torch.int32).cuda(), cu, new, block_size=bs,
                                  sm_scale=size / D))
    small = (n - new + np.arange(new)) * 2.0 ** -abs(log2)  # visible keys but one
    want = np.tile(small / (1 + small), B)[:, None, None]
    E = size * (2.0 ** -12 + 2.0 ** -21)
    assert (np.abs(got - want) <= (U[dtype] + 2.0 ** -10 + 2.0 ** -20 + 2 * E) * want + 2.0 ** -24).all(), \
        np.abs(got / want - 1).max()
    assert _lib.debug_status() == 0


@pytest.mark.parametrize("bad", [torch.float32, torch.float16, torch.float64, torch.bool])
def test_only_integers_are_indexes(cuda_device, bad):
    case = _case(24, [20], [2], 1, 2, 64, 16, F)
    q, cache, table, ctx, cu, k, v = (t.cuda() for t in case)
    slots = torch.arange(20).cuda()
    calls = [lambda: paged_kv4_append(k, v, cache, slots.to(bad), block_size=16),
             lambda: paged_kv4_gather(cache, slots.to(bad), block_size=16)]
    for i in range(3):
        a = [table, ctx, cu]
        a[i] = a[i].to(bad)
        calls.append(lambda a=a: paged_attention_kv4(q, cache, *a, 2, block_size=16))
    for i in range(4):
        a = [ctx, ctx, ctx, ctx]
        a[i] = a[i].to(bad)
        calls.append(lambda a=a: paged_plan(table, *a[:3], block_size=16, max_tokens=4, free_start=a[3]))
    w, cs = torch.ones(64, dtype=F, device="cuda"), torch.ones(32, 32, device="cuda")
    calls.append(lambda: qk_norm_rope(k, k, w, w, cs, cs, slots.to(bad)))
    before = cache.clone(), table.clone()
    for call in calls:
        with pytest.raises(AssertionError):
            call()
    assert torch.equal(cache, before[0]) and torch.equal(table, before[1])


@pytest.mark.parametrize("dtype", [torch.int64, torch.int16, torch.uint8])
def test_integers_of_other_sizes(cuda_device, dtype):
    case = _case(24, [20, 90], [2, 1], 1, 2, 64, 16, F)
    q, cache, table, ctx, cu, k, v = (t.cuda() for t in case)
    ref = paged_attention_kv4(q, cache, table, ctx, cu, 2, block_size=16)
    got = paged_attention_kv4(q, cache, table.to(dtype), ctx.to(dtype), cu.to(dtype), 2, block_size=16)
    assert torch.equal(got, ref)
    slots = torch.arange(20, device="cuda")
    for a, b in zip(paged_kv4_gather(cache, slots.to(dtype), block_size=16), paged_kv4_gather(cache, slots, block_size=16)):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    w, cs = torch.ones(64, dtype=F, device="cuda"), torch.rand(128, 32, device="cuda")
    at = torch.arange(110, device="cuda")
    for a, b in zip(qk_norm_rope(k, k, w, w, cs, cs, at.to(dtype)), qk_norm_rope(k, k, w, w, cs, cs, at.int())):
        assert torch.equal(a, b)
    assert _lib.debug_status() == 0


def test_integers_past_32_bits_do_not_wrap(cuda_device):
    """Slots, blocks and positions of 2^32 and more are outside everything, not inside after wrapping; lengths are
    as long as the table."""
    case = _case(25, [20], [2], 1, 2, 64, 16, F)
    q, cache, table, ctx, cu, k, v = (t.cuda() for t in case)
    before = cache.clone()
    bad = torch.tensor([2 ** 32, 2 ** 32 + 5, -2 ** 32, -2 ** 33 + 1, 2 ** 31], device="cuda")
    paged_kv4_append(k[:5], v[:5], cache, bad, block_size=16)
    torch.cuda.synchronize()
    assert torch.equal(cache, before) and _lib.debug_status() == 0x200
    gk, gv = paged_kv4_gather(cache, bad, block_size=16)
    torch.cuda.synchronize()
    assert (gk == 0).all() and (gv == 0).all() and _lib.debug_status() == 0x200
    attend = lambda t, c: paged_attention_kv4(q, cache, t, c, cu, 2, block_size=16)  # noqa: E731
    attend(table.long() + 2 ** 32, ctx)
    torch.cuda.synchronize()
    assert _lib.debug_status() == 0x200
    full = torch.full_like(ctx, 32)
    assert torch.equal(attend(table, ctx.long() + 2 ** 32).nan_to_num(7.0), attend(table, full).nan_to_num(7.0))
    assert _lib.debug_status() == 0
    plan = paged_plan(table.clone(), ctx.long() + 2 ** 32, ctx // ctx, table[0], block_size=16, max_tokens=1)
    assert plan.slots.tolist() == [-1] and plan.new_lens.tolist() == [2 ** 31 - 1] and plan.taken.tolist() == [0]
    w, cs = torch.ones(64, dtype=F, device="cuda"), torch.rand(32, 32, device="cuda")
    at = torch.arange(20, device="cuda")
    got = qk_norm_rope(k, k, w, w, cs, cs, at + 2 ** 32)
    torch.cuda.synchronize()
    assert _lib.debug_status() == 0x200
    assert torch.equal(got[0], qk_norm_rope(k, k, w, w, cs, cs, at * 0)[0])


def test_slots_past_32_bits(cuda_device):
    """Blocks whose slots int32 has no number for: the plan gives one slot for all of them, and nothing is
    written there (here a pool of 2^31 slots over the memory of one block)."""
    table = torch.full((1, 2), 2 ** 27 + 3, dtype=torch.int32, device="cuda")
    n = lambda v: torch.tensor([v], dtype=torch.int32, device="cuda")  # noqa: E731
    plan = paged_plan(table, n(5), n(3), n(0), block_size=16, max_tokens=3)
    assert plan.slots.tolist() == [2 ** 31 - 1] * 3
    one = torch.zeros(1, 1, 1, 1280, dtype=torch.uint8, device="cuda")
    cache = one.expand(2 ** 27, 1, 1, 1280)
    k = torch.randn(3, 1, 64, dtype=F, device="cuda")
    paged_kv4_append(k, k, cache, plan.slots, block_size=16)
    torch.cuda.synchronize()
    assert (one == 0).all() and _lib.debug_status() == 0x200
    paged_kv4_append(k, k, cache, plan.slots - 1, block_size=16)
    torch.cuda.synchronize()
    assert not (one == 0).all() and _lib.debug_status() == 0
