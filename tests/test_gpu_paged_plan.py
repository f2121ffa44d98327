"""Block tables and slot maps against the sequential restatement: whole numbers, equal."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from tritonllmcompiler_b200.ops.paged_plan import paged_plan

pytestmark = pytest.mark.gpu


def _check(lens, new, bs, width, n_free, max_tokens=None, seed=0, strided=False):
    rng = np.random.RandomState(seed)
    lens, new = np.array(lens, np.int32), np.array(new, np.int32)
    pool = rng.permutation(400000).astype(np.int32)
    free, pool = pool[:n_free], pool[n_free:]
    table = np.full((len(lens), width), -7, np.int32)
    at = 0
    for b, n in enumerate(lens):
        have = min(width, -(-max(0, int(n)) // bs))
        table[b, :have] = pool[at:at + have]
        at += have
    total = int(np.maximum(new, 0).sum()) if max_tokens is None else max_tokens
    want = O.paged_plan(table, lens, new, free, block_size=bs, max_tokens=total)
    if strided:
        big = torch.zeros(len(lens), 2 * width, dtype=torch.int32).cuda()
        dev = big[:, ::2]
        dev.copy_(torch.from_numpy(table))
    else:
        dev = torch.from_numpy(table).cuda()
    got = paged_plan(dev, torch.from_numpy(lens).cuda(), torch.from_numpy(new).cuda(),
                     torch.from_numpy(free).cuda(), block_size=bs, max_tokens=total)
    for name, w in zip(("slots", "positions", "cu_seqlens", "new_lens"), want):
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), w, err_msg=name)
    assert int(got.taken) == want[4]
    np.testing.assert_array_equal(dev.cpu().numpy(), want[5])


@pytest.mark.parametrize("lens,new,bs,width", [
    ([0], [1], 16, 1),
    ([15, 16, 17, 0, 31], [1, 1, 1, 1, 1], 16, 4),
    ([5, 0, 64, 33], [0, 0, 0, 0], 32, 3),
    ([0, 100, 3], [97, 64, 130], 64, 4),
    ([7, 2, 9], [5, 6, 30], 5, 9),  # a block size that is no power of two
    ([-3, 4], [2, -1], 16, 2),  # negative lengths count as none
])
def test_small(cuda_device, lens, new, bs, width):
    _check(lens, new, bs, width, n_free=40)


def test_refusals(cuda_device):
    # the third does not fit its row, the fourth the free list, the fifth takes no block, and
    # the last finds nothing left.
    _check([16, 0, 60, 10, 20, 16], [20, 16, 9, 60, 3, 1], 16, 4, n_free=4)
    _check([16, 0], [1, 1], 16, 4, n_free=0)
    _check([0, 0, 0], [10, 10, 10], 16, 4, n_free=9, max_tokens=25)  # the packed batch is full
    _check([0, 3], [10, 2], 16, 4, n_free=9, max_tokens=40)  # rows past the last token


@pytest.mark.parametrize("B,seed", [(1, 1), (31, 2), (257, 3), (1000, 4), (12000, 5)])
def test_many(cuda_device, B, seed):
    rng = np.random.RandomState(seed)
    lens, new = rng.randint(0, 300, B), rng.randint(0, 40 if B < 5000 else 3, B)
    _check(lens, new, 16, 22, n_free=min(90000, 3 * B + 5), seed=seed, strided=B == 257)
    _check(lens, new, 16, 22, n_free=max(1, B // 2), seed=seed)


def test_nothing(cuda_device):
    e = torch.empty(0, dtype=torch.int32).cuda()
    p = paged_plan(torch.empty(0, 4, dtype=torch.int32).cuda(), e, e, e, block_size=16, max_tokens=3)
    assert p.slots.tolist() == [-1] * 3 and p.positions.tolist() == [0] * 3
    assert p.cu_seqlens.tolist() == [0] and p.new_lens.numel() == 0 and p.taken.tolist() == [0]


def test_wide_types_and_another_stream(cuda_device):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        table = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
        i = lambda *v: torch.tensor(v, device="cuda")  # noqa: E731  (int64)
        p = paged_plan(table, i(0, 16), i(3, 1), i(9, 8, 7), block_size=16, max_tokens=4)
        assert p.slots.tolist() == [144, 145, 146, 128]
    s.synchronize()


def test_refused_arguments(cuda_device):
    t = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    v = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(AssertionError):
        paged_plan(t.long(), v, v, v, block_size=16, max_tokens=1)
    with pytest.raises(AssertionError):
        paged_plan(t, v[:1], v, v, block_size=16, max_tokens=1)
    with pytest.raises(AssertionError):
        paged_plan(t, v, v.cpu(), v, block_size=16, max_tokens=1)
    with pytest.raises(AssertionError):
        paged_plan(t, v, v, v, block_size=0, max_tokens=1)
    big = torch.zeros(16385, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="at most 16384"):
        paged_plan(big.view(-1, 1), big, big, v, block_size=16, max_tokens=1)
