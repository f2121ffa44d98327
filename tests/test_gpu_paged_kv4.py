"""The 4-bit paged cache: what is read back equals the definition bit for bit, and attention over
it holds to 64 bits.

Bounds of the attention, per element. The kernels round each weight, or its product with a scale,
to 11 bits before the products with the codes (2^-10 of A, the weighted sum of the sizes of the
values' two terms: one rounding each for the weight and the product), the scores are off by at
most E (see the oracle), which changes every weight by a factor within 1 +- 2 E, and the output is
rounded once (u |o|, u = 2^-11 fp16, 2^-8 bf16). With 2^-20 A for sums in fp32 that is
u |o| + (2^-10 + 2^-20 + 2 E) A + 2^-24. Over a whole output these are random: a 2-norm of 2 u.
"""
import math

import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from tritonllmcompiler_b200 import _lib
from tritonllmcompiler_b200.ops.paged_kv4 import (new_kv4_cache, paged_attention_kv4,
                                                  paged_kv4_append, paged_kv4_gather)

pytestmark = pytest.mark.gpu
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def _np(t):
    return t.double().cpu().numpy()


def _values(x, dtype):
    """What the cache gives back for x, rounded to dtype as the library rounds it."""
    v, _ = O.dequantise(*O.quantise(x.float().cpu().numpy()))
    return torch.from_numpy(v).float().to(dtype)


def _slots(T, bs, blocks, seed):
    """Slots of T tokens in blocks of the pool in random order."""
    perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed))
    i = torch.arange(T)
    return (perm[i // bs] * bs + i % bs).int()


@pytest.mark.parametrize("T,H,D,bs,dtype", [(1, 1, 64, 16, torch.float16), (16, 2, 128, 16, torch.bfloat16),
                                             (33, 3, 128, 32, torch.float16), (129, 8, 64, 64, torch.bfloat16),
                                             (1000, 2, 128, 64, torch.float16)])
def test_append_and_gather(cuda_device, T, H, D, bs, dtype):
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randn(T, H, D, generator=g) * (1 + 5 * torch.rand(H, D, generator=g)) for _ in range(2))
    k, v = k.to(dtype), v.to(dtype)
    blocks = -(-T // bs) + 2
    slots = _slots(T, bs, blocks, T)
    cache = new_kv4_cache(blocks, H, bs, D)
    cache.fill_(0xA5)
    before = cache.clone()
    order = torch.randperm(T, generator=g)  # tokens of a piece arrive in any order
    paged_kv4_append(k[order].cuda(), v[order].cuda(), cache, slots[order].cuda(), block_size=bs)
    gk, gv = paged_kv4_gather(cache, slots.cuda(), block_size=bs, dtype=dtype)
    assert torch.equal(gk.cpu(), _values(k, dtype)) and torch.equal(gv.cpu(), _values(v, dtype))
    # nothing else was touched: the free slots read back as before
    free = torch.tensor(sorted(set(range(blocks * bs)) - set(slots.tolist())), dtype=torch.int32).cuda()
    for a, b in zip(paged_kv4_gather(cache, free, block_size=bs), paged_kv4_gather(before, free, block_size=bs)):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))
    assert _lib.debug_status() == 0


def test_append_special_groups(cuda_device):
    """Constant groups, ranges too small for fp16, negatives, NaN and infinities."""
    x = torch.randn(8, 1, 64, generator=torch.Generator().manual_seed(1))
    x[0] = 3.25
    x[1] = 0
    x[2] = -1 + 1e-9 * x[2]
    x[3] = 1e-7 * x[3]
    x[4] = -50000 + x[4]
    x[5, 0, 3] = math.nan
    x[6, 0, 40] = math.inf
    x[7, 0, 1] = 1e9
    k = x.bfloat16()
    cache = new_kv4_cache(1, 1, 16, 64)
    slots = torch.arange(8, dtype=torch.int32).cuda()
    paged_kv4_append(k.cuda(), (-k).cuda(), cache, slots, block_size=16)
    gk, gv = (t.cpu() for t in paged_kv4_gather(cache, slots, block_size=16, dtype=torch.bfloat16))
    assert torch.equal(gk[:5], _values(k[:5], torch.bfloat16)) and torch.equal(gv[:5], _values(-k[:5], torch.bfloat16))
    for t, hit in ((5, 0), (6, 1), (7, 0)):  # the other group of the row is whole
        for got, src in ((gk, k), (gv, -k)):
            a, b = got[t, 0].view(2, 32), _values(src[t], torch.bfloat16)[0].view(2, 32)
            assert torch.equal(a[1 - hit], b[1 - hit]) and not a[hit].isfinite().any()


def test_append_skips(cuda_device):
    k = torch.randn(4, 2, 128, dtype=torch.float16, device="cuda")
    cache = new_kv4_cache(2, 2, 16, 128)
    slots = torch.tensor([-1, 5, 32, -7], dtype=torch.int32, device="cuda")
    paged_kv4_append(k, k, cache, slots, block_size=16)
    torch.cuda.synchronize()
    assert _lib.debug_status() == 0x200
    gk, gv = paged_kv4_gather(cache, slots, block_size=16)
    torch.cuda.synchronize()
    assert _lib.debug_status() == 0x200
    assert (gk[[0, 2, 3]] == 0).all() and (gv[[0, 2, 3]] == 0).all()
    assert torch.equal(gk[1].cpu(), _values(k[1], torch.float16))
    rest = [i for i in range(32) if i != 5]
    gk, _ = paged_kv4_gather(cache, torch.tensor(rest, device="cuda"), block_size=16)
    assert (gk == 0).all()
    e = torch.empty(0, 2, 128, dtype=torch.float16, device="cuda")
    paged_kv4_append(e, e, cache, slots[:0], block_size=16)
    assert paged_kv4_gather(cache, slots[:0], block_size=16)[0].shape == (0, 2, 128)
    assert _lib.debug_status() == 0


def test_append_strided(cuda_device):
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(20, 8, 128, generator=g).half().cuda()
    whole = torch.zeros(3, 2, 2, 2, 2560, dtype=torch.uint8, device="cuda")  # two layers side by side
    cache = whole[:, :, 1].transpose(0, 1).contiguous().transpose(0, 1)
    slots = _slots(20, 32, 3, 4).cuda()
    odd = torch.zeros(20, 2, 129, dtype=torch.float16, device="cuda")
    odd[..., 1:] = qkv[:, 6:]
    paged_kv4_append(qkv[:, 4:6], odd[..., 1:], cache, slots, block_size=32)
    gk, gv = paged_kv4_gather(cache, slots.long(), block_size=32)
    assert torch.equal(gk.cpu(), _values(qkv[:, 4:6], torch.float16))
    assert torch.equal(gv.cpu(), _values(qkv[:, 6:], torch.float16))


# ------------------------------------------------------------------------------ attention
def _case(seed, lens, new, hkv, G, D, bs, dtype, spread=1.0, extra=2):
    """A filled cache, block tables, packed queries, and the values in the cache."""
    g = torch.Generator().manual_seed(seed)
    nb = [-(-n // bs) for n in lens]
    blocks = sum(nb) + extra
    perm = torch.randperm(blocks, generator=g).int()
    table = torch.full((len(lens), max(max(nb), 1)), blocks + 5, dtype=torch.int32)  # bad where unused
    at = 0
    k, v, slots = [], [], []
    for b, n in enumerate(lens):
        table[b, :nb[b]] = perm[at:at + nb[b]]
        at += nb[b]
        i = torch.arange(n)
        slots.append(table[b, i // bs] * bs + i % bs)
        k.append(torch.randn(n, hkv, D, generator=g) * (1 + 3 * (torch.rand(hkv, D, generator=g) < 0.1)))
        v.append(torch.randn(n, hkv, D, generator=g) * spread)
    k, v = torch.cat(k).to(dtype), torch.cat(v).to(dtype)
    cache = new_kv4_cache(blocks, hkv, bs, D)
    cache.fill_(0xFF)  # unwritten slots: every scale and zero a NaN
    slots = torch.cat(slots).int()
    paged_kv4_append(k.cuda(), v.cuda(), cache, slots.cuda(), block_size=bs)
    q = torch.randn(sum(new), hkv * G, D, generator=g).to(dtype)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32)
    return q, cache, table, torch.tensor(lens, dtype=torch.int32), cu, k, v


def _check(case, lens, new, bs, dtype, causal=True, scale=None, rows=None, norm=True):
    q, cache, table, ctx, cu, k, v = case
    got = paged_attention_kv4(q.cuda(), cache, table.cuda(), ctx.cuda(), cu.cuda(), max(new), block_size=bs,
                              causal=causal, sm_scale=scale)
    assert got.shape == q.shape and got.dtype == dtype
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, at = _np(got), 0
    sq = [0.0, 0.0]
    for b, n in enumerate(lens):
        r = slice(int(cu[b]), int(cu[b + 1]))
        kb, vb = k[at:at + n], v[at:at + n]
        at += n
        if new[b] == 0:
            continue
        kv, ks = O.dequantise(*O.quantise(kb.float().numpy()))
        vv, vs = O.dequantise(*O.quantise(vb.float().numpy()))
        qb = _np(q[r])
        o, A, E = O.attention(qb, kv, vv, ks, vs, scale=scale, causal=causal, n_new=new[b])
        assert np.array_equal(np.isnan(out[r]), np.isnan(o)), b
        err = np.nan_to_num(np.abs(out[r] - o))
        bound = U[dtype] * np.nan_to_num(np.abs(o)) + (2.0 ** -10 + 2.0 ** -20 + 2 * E) * A + 2.0 ** -24
        assert (err <= bound).all(), (b, err.max(), (err / bound).max())
        sq[0] += (err ** 2).sum()
        sq[1] += np.nansum(o ** 2)
    if norm:
        assert math.sqrt(sq[0]) <= 2 * U[dtype] * math.sqrt(sq[1])
    assert _lib.debug_status() == 0
    return got


F, BF = torch.float16, torch.bfloat16
ATTN = [
    # lens, new, hkv, G, D, bs, dtype
    ([1], [1], 1, 1, 64, 16, F),
    ([33], [1], 2, 4, 64, 16, F),
    ([15, 16, 17], [1, 1, 1], 2, 4, 128, 16, BF),
    ([31, 32, 33, 64, 65], [1, 1, 1, 1, 1], 3, 8, 128, 32, F),
    ([127, 128, 129, 500], [1, 0, 1, 1], 1, 5, 128, 64, BF),
    ([700, 3, 2049], [2, 3, 4], 2, 2, 64, 32, F),
    ([700, 5, 1300], [4, 5, 1], 2, 4, 128, 16, F),
    ([64, 200], [16, 16], 1, 1, 128, 16, BF),
    ([1025, 90], [7, 3], 1, 16, 64, 64, BF),
    ([40, 300], [40, 17], 2, 4, 128, 16, F),
    ([140, 77, 260], [129, 1, 64], 1, 3, 64, 32, BF),
    ([400, 257, 16], [200, 257, 0], 2, 2, 128, 64, F),
    ([333], [333], 1, 1, 64, 16, BF),
    ([6000], [1], 1, 8, 128, 16, F),
    ([9000, 10], [2, 2], 1, 1, 64, 64, F),
]


@pytest.mark.parametrize("lens,new,hkv,G,D,bs,dtype", ATTN)
def test_attention(cuda_device, lens, new, hkv, G, D, bs, dtype):
    case = _case(sum(lens) + G, lens, new, hkv, G, D, bs, dtype)
    _check(case, lens, new, bs, dtype)


# Many short requests: runs of the line start and end everywhere in their row tiles, before the first key too.
@pytest.mark.parametrize("B,longest,most,hkv,G,D,dtype", [
    (250, 200, 1, 4, 4, 64, F), (300, 400, 4, 2, 4, 128, BF), (100, 500, 40, 2, 4, 128, BF), (61, 150, 150, 3, 2, 64, F)])
def test_many_requests(cuda_device, B, longest, most, hkv, G, D, dtype):
    rng = np.random.default_rng(B)
    new = [int(n) for n in rng.integers(0, most + 1, B)]
    lens = [int(rng.integers(n, longest + 1)) for n in new]
    _check(_case(B, lens, new, hkv, G, D, 16, dtype), lens, new, 16, dtype)


@pytest.mark.parametrize("lens,new,G,D", [([50, 130, 5], [3, 20, 5], 4, 128), ([300, 40], [150, 2], 2, 64)])
def test_attention_not_causal(cuda_device, lens, new, G, D):
    _check(_case(5, lens, new, 2, G, D, 16, F), lens, new, 16, F, causal=False)


@pytest.mark.parametrize("new", [[6, 3], [150, 30]])
def test_rows_without_keys(cuda_device, new):
    """More new tokens than the context counts: the first see nothing and give NaN, and a sequence
    without a context gives only NaN."""
    lens = [4, 0]
    _check(_case(6, lens, new, 2, 2, 64, 16, F), lens, new, 16, F)


@pytest.mark.parametrize("new", [[1, 1], [9, 140]])
def test_rows_past_the_batch_are_zero(cuda_device, new):
    lens = [70, 160]
    q, cache, table, ctx, cu, k, v = _case(7, lens, new, 1, 4, 128, 16, BF)
    ref = paged_attention_kv4(q.cuda(), cache, table.cuda(), ctx.cuda(), cu.cuda(), max(new), block_size=16)
    more = torch.cat([q, torch.full((37, 4, 128), float("nan"), dtype=BF)])
    got = paged_attention_kv4(more.cuda(), cache, table.cuda(), ctx.cuda(), cu.cuda(), max(new), block_size=16)
    assert torch.equal(got[:q.shape[0]], ref) and (got[q.shape[0]:] == 0).all()
    none = paged_attention_kv4(q.cuda(), cache, table.cuda()[:0], ctx.cuda()[:0], cu.cuda()[:1] * 0, 1, block_size=16)
    assert (none == 0).all()


@pytest.mark.parametrize("lens,new", [([90, 33], [4, 1]), ([97, 33], [1, 1]), ([90, 33], [40, 1])])
def test_nan_keys_behind_the_mask(cuda_device, lens, new):
    """A NaN or an infinity in the newest token reaches the rows that see it (also where it is alone
    in its tile) and no others."""
    G, last = 4, lens[0] - 1
    q, cache, table, ctx, cu, k, v = _case(8, lens, new, 1, G, 128, 16, F)
    args = (table.cuda(), ctx.cuda(), cu.cuda(), max(new))
    ref = paged_attention_kv4(q.cuda(), cache, *args, block_size=16)
    slot = (table[0, last // 16] * 16 + last % 16).view(1).cuda()
    bad = torch.full((1, 1, 128), float("nan"), dtype=F, device="cuda")
    bad[0, 0, 64:] = float("inf")
    paged_kv4_append(bad, bad, cache, slot, block_size=16)
    got = paged_attention_kv4(q.cuda(), cache, *args, block_size=16)
    n = new[0]
    assert torch.equal(got[:n - 1], ref[:n - 1]) and torch.equal(got[n:], ref[n:])
    assert got[n - 1].isnan().all()


@pytest.mark.parametrize("new", [[2, 1], [50, 1]])
def test_special_queries(cuda_device, new):
    """A zero query averages the values; a NaN query gives NaN in its own rows alone; queries of
    very large and very small size keep their scores."""
    lens = [60, 20]
    q, cache, table, ctx, cu, k, v = _case(9, lens, new, 1, 4, 64, 16, BF)
    q[0, 0] = 0
    q[0, 1, 7] = float("nan")
    q[1, 0] *= 2.0 ** 60
    q[1, 1] *= 2.0 ** -60
    got = paged_attention_kv4(q.cuda(), cache, table.cuda(), ctx.cuda(), cu.cuda(), max(new), block_size=16)
    vv, vs = O.dequantise(*O.quantise(v[:60].float().numpy()))
    m = 60 - new[0] + 1
    for row, h, n in ((0, 0, m), (1, 1, m + 1)):
        want, A = vv[:n, 0].mean(0), vs[:n, 0].mean(0)
        assert (np.abs(_np(got[row, h]) - want) <= U[BF] * np.abs(want) + 2.0 ** -9 * A).all()
    kv, _ = O.dequantise(*O.quantise(k[:60].float().numpy()))
    top = int((kv[:m + 1, 0] @ _np(q[1, 0])).argmax())  # all the weight on one key
    assert (np.abs(_np(got[1, 0]) - vv[top, 0]) <= 2 * U[BF] * np.abs(vv[top, 0]) + 2.0 ** -10 * vs[top, 0]).all()
    assert got[0, 1].isnan().all() and not got[0, [0, 2, 3]].isnan().any() and not got[1:].isnan().any()


@pytest.mark.parametrize("spread", [2.0 ** -12, 2.0 ** 9])
@pytest.mark.parametrize("new", [[1, 3], [70, 1]])
def test_small_and_large_values(cuda_device, spread, new):
    """V far from 1: the weights' products with the scales keep their bits. (At 2^-12 the zeros
    and scales are near fp16's smallest normals, which the oracle's quantisation has too.)"""
    lens = [300, 700]
    _check(_case(10, lens, new, 1, 4, 128, 16, BF, spread=spread), lens, new, 16, BF)


def test_values_of_growing_size(cuda_device):
    """The scales of V grow by 2^16 along the context."""
    lens, new, D = [1500], [2], 128
    q, cache, table, ctx, cu, k, v = _case(11, lens, new, 1, 4, D, 16, BF)
    v = (v.float() * torch.logspace(-2, 2.8, 1500, dtype=torch.float64).float()[:, None, None]).to(BF)
    i = torch.arange(1500)
    slots = (table[0, i // 16] * 16 + i % 16).cuda()
    paged_kv4_append(k.cuda(), v.cuda(), cache, slots, block_size=16)
    _check((q, cache, table, ctx, cu, k, v), lens, new, 16, BF)


def test_scores_of_large_size(cuda_device):
    """One key takes all the weight, late in a long context and early in it."""
    lens, new = [2000, 2000], [1, 1]
    case = _case(12, lens, new, 1, 4, 64, 32, F)
    q, cache, table, ctx, cu, k, v = case
    for b, at in ((0, 1990), (1, 3)):
        k[2000 * b + at] = 6 * torch.sign(q[b, 0].float()).to(F)
        slot = (table[b, at // 32] * 32 + at % 32).view(1).cuda()
        paged_kv4_append(k[2000 * b + at:][:1].cuda(), v[2000 * b + at:][:1].cuda(), cache, slot, block_size=32)
    _check(case, lens, new, 32, F, scale=1.0, norm=False)


def test_bad_blocks_are_flagged(cuda_device):
    for new in ([1], [40]):
        q, cache, table, ctx, cu, k, v = _case(13, [100], new, 2, 4, 64, 16, F)
        table[0, 2] = 10 ** 6
        paged_attention_kv4(q.cuda(), cache, table.cuda(), ctx.cuda(), cu.cuda(), new[0], block_size=16)
        torch.cuda.synchronize()
        assert _lib.debug_status() == 0x200
    assert _lib.debug_status() == 0


def test_strided_queries_tables_and_another_stream(cuda_device):
    lens, new = [200, 50, 90], [1, 2, 1]
    q, cache, table, ctx, cu, k, v = _case(14, lens, new, 2, 4, 128, 16, F)
    ref = _check((q, cache, table, ctx, cu, k, v), lens, new, 16, F)
    qkv = torch.zeros(q.shape[0], 14, 129, dtype=F, device="cuda")
    qkv[:, :8, 1:] = q.cuda()
    wide = torch.zeros(3, 2 * table.shape[1], dtype=torch.int32, device="cuda")
    wide[:, ::2] = table.cuda()
    wide = wide[:, ::2]
    layers = torch.zeros(cache.shape[0], 3, *cache.shape[1:], dtype=torch.uint8, device="cuda")
    layers[:, 1] = cache
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = paged_attention_kv4(qkv[:, :8, 1:], layers[:, 1], wide, ctx.cuda().long(), cu.cuda().long(), 2,
                                  block_size=16)
    s.synchronize()
    assert torch.equal(got, ref)


def test_graph_replay(cuda_device):
    """The call captures into a CUDA graph and follows its inputs' contents, lengths included."""
    lens, new = [100, 300], [1, 1]
    q, cache, table, ctx, cu, k, v = _case(15, lens, new, 1, 4, 64, 16, F)
    dq, dt, dc, du = q.cuda(), table.cuda(), ctx.cuda(), cu.cuda()
    call = lambda: paged_attention_kv4(dq, cache, dt, dc, du, 1, block_size=16)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    dc.copy_(torch.tensor([60, 299], dtype=torch.int32))
    dq.mul_(0.5)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, call())


def test_a_cache_past_32_bits(cuda_device):
    """Byte offsets beyond 2^32: the last blocks of a 5 GB cache."""
    blocks = (5 << 30) // (2 * 4 * 2560)
    cache = torch.zeros((blocks, 2, 4, 2560), dtype=torch.uint8, device="cuda")
    g = torch.Generator().manual_seed(1)
    lens, bs = [150], 64
    table = torch.tensor([[blocks - 1, 1, blocks - 7]], dtype=torch.int32)
    i = torch.arange(150)
    slots = (table[0, i // bs].long() * bs + i % bs).int()
    k, v = (torch.randn(150, 2, 128, generator=g).half() for _ in range(2))
    paged_kv4_append(k.cuda(), v.cuda(), cache, slots.cuda(), block_size=bs)
    gk, _ = paged_kv4_gather(cache, slots.cuda(), block_size=bs)
    assert torch.equal(gk.cpu(), _values(k, F))
    for n in (1, 60):
        q = torch.randn(n, 8, 128, generator=g).half()
        cu = torch.tensor([0, n], dtype=torch.int32)
        _check((q, cache, table, torch.tensor(lens, dtype=torch.int32), cu, k, v), lens, [n], bs, F)


def test_refused_arguments(cuda_device):
    q, cache, table, ctx, cu, k, v = (t.cuda() for t in _case(16, [20], [2], 1, 2, 64, 16, F))
    good = dict(q=q, cache=cache, table=table, ctx=ctx, cu=cu, max_new=2)
    for bad in (dict(q=q.float()), dict(q=q[..., :32]), dict(cache=cache.float()), dict(cache=cache[..., :1000]),
                dict(ctx=ctx.cpu()), dict(cu=cu[:1]), dict(cache=new_kv4_cache(4, 1, 16, 128)[..., ::2])):
        with pytest.raises(AssertionError):
            paged_attention_kv4(*dict(good, **bad).values(), block_size=16)
    with pytest.raises(AssertionError):
        paged_attention_kv4(*good.values(), block_size=32)
    three = torch.zeros(2, 3, 64, dtype=F, device="cuda")
    with pytest.raises(AssertionError):
        paged_attention_kv4(*dict(good, q=three, cache=new_kv4_cache(4, 2, 16, 64)).values(), block_size=16)
    with pytest.raises(AssertionError):
        paged_kv4_append(k, v[:1], cache, ctx, block_size=16)
    with pytest.raises(AssertionError):
        paged_kv4_append(k.float(), v.float(), cache, torch.zeros(20, device="cuda"), block_size=16)
    with pytest.raises(AssertionError):
        paged_kv4_gather(cache, ctx, block_size=16, dtype=torch.float32)
    with pytest.raises(AssertionError):
        new_kv4_cache(1, 1, 16, 96)
