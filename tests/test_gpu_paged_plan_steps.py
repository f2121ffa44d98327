"""Steps that follow one another over one free list: no block goes to two requests."""
import numpy as np
import pytest
import torch

from oracle import kv4_oracle as O
from tritonllmcompiler_b200.ops.paged_plan import paged_plan

pytestmark = pytest.mark.gpu


def _cuda(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("start", [0, 1, 7, 20, 21, 1000, -3])
def test_the_list_from_an_entry(cuda_device, start):
    """As a list without the entries before it; past its end nothing is left."""
    rng = np.random.RandomState(1)
    free = rng.permutation(500)[:20]
    lens, new = [16, 0, 60, 10, 33], [20, 16, 9, 60, 0]
    table = np.arange(1000, 1030).reshape(5, 6)
    want = O.paged_plan(table, lens, new, free[max(start, 0):], block_size=16, max_tokens=120)
    dev = _cuda(table)
    got = paged_plan(dev, _cuda(lens), _cuda(new), _cuda(free), block_size=16, max_tokens=120, free_start=_cuda([start]))
    for name, w in zip(("slots", "positions", "cu_seqlens", "new_lens"), want):
        np.testing.assert_array_equal(getattr(got, name).cpu().numpy(), w, err_msg=name)
    assert int(got.taken) == want[4]
    np.testing.assert_array_equal(dev.cpu().numpy(), want[5])


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_no_block_twice(cuda_device, dtype):
    """A loop that reads nothing back, until the list is empty: every block has one owner, requests that
    find none keep their lengths, and the others go on."""
    rng = np.random.RandomState(2)
    B, F, bs = 9, 40, 16
    free = rng.permutation(F)
    table, lens = _cuda(np.full((B, 16), -1)), _cuda(np.zeros(B))
    taken = torch.zeros(1, dtype=dtype, device="cuda")
    steps = []
    for _ in range(30):
        new = _cuda(rng.randint(0, 9, B))
        plan = paged_plan(table, lens, new, _cuda(free), block_size=bs, max_tokens=9 * B, free_start=taken)
        taken += plan.taken
        steps.append((lens, new, plan))
        lens = plan.new_lens
    owned = [b for row, n in zip(table.tolist(), lens.tolist()) for b in row[:-(-n // bs)]]
    assert len(set(owned)) == len(owned) == int(taken) and set(owned) <= set(free.tolist())
    refused = [(plan.new_lens != old + new).sum().item() for old, new, plan in steps]
    assert refused[0] == 0 and refused[-1] > 0 and int(taken) > F - B
    # a slot is written once
    slots = [s for _, _, plan in steps for s in plan.slots.tolist() if s >= 0]
    assert len(set(slots)) == len(slots) == int(lens.sum())


def test_refused_arguments(cuda_device):
    table, one = _cuda([[0]]), _cuda([1])
    for bad in (_cuda([0, 0]), one.cpu()):
        with pytest.raises(AssertionError):
            paged_plan(table, one, one, one, block_size=16, max_tokens=1, free_start=bad)
