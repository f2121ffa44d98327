"""examples/kv4_serving.py with pools that run low."""
import pytest
import torch

from tests.test_gpu_kv4_serving import serving  # noqa: F401  (the module, as a fixture)
from tritonllmcompiler_b200 import _lib

pytestmark = pytest.mark.gpu
PROMPTS = [[(i * 31 + b) % 256 for i in range(n)] for b, n in enumerate((40, 30, 3))]


def test_a_pool_that_just_holds(cuda_device, serving):  # noqa: F811
    """8 blocks for 51, 41 and 14 tokens, the last entry of the list in use: the same tokens' logits as
    from a large pool (to the fp16 rounding of the layers: the keys may be split at other places)."""
    model = serving.Decoder(dtype=torch.float16, seed=5)
    tokens, want = serving.generate(model, PROMPTS, 12, blocks=32, max_blocks=8)
    again, got = serving.generate(model, PROMPTS, 12, blocks=8, max_blocks=8)
    assert torch.equal(tokens, again) and ((got - want).norm() / want.norm()).item() < 0.02
    assert _lib.debug_status() == 0


@pytest.mark.parametrize("blocks", [3, 6, 7])
def test_a_pool_that_runs_out(cuda_device, serving, blocks):  # noqa: F811
    """Requests that find no block are reported; the others' logits are those of a large pool."""
    model = serving.Decoder(dtype=torch.float16, seed=5)
    tokens, want = serving.generate(model, PROMPTS, 12, blocks=32, max_blocks=8)
    with pytest.raises(RuntimeError, match="cannot hold requests"):
        serving.generate(model, PROMPTS, 12, blocks=blocks, max_blocks=8)
    server = serving.Server(model, 3, blocks=blocks, max_blocks=8)
    flat, n = torch.tensor(sum(PROMPTS, []), device="cuda"), [len(p) for p in PROMPTS]
    for step in range(12):
        logits = server.step(flat, torch.tensor(n, dtype=torch.int32, device="cuda"), max(n))
        for b in range(3):
            if server.refused[b]:
                assert logits[b].isnan().all()
            else:
                assert ((logits[b] - want[b, step]).norm() / want[b, step].norm()).item() < 0.02
        flat, n = tokens[:, step], [1, 1, 1]
    assert server.refused.any() and (blocks == 3 or not server.refused.all())


def test_idle_requests_have_no_logits(cuda_device, serving):  # noqa: F811
    server = serving.Server(serving.Decoder(dtype=torch.float16, seed=5), 3, blocks=8, max_blocks=8)
    logits = server.step(torch.tensor([5, 6], device="cuda"), torch.tensor([0, 2, 0], dtype=torch.int32, device="cuda"), 2)
    assert logits[[0, 2]].isnan().all() and logits[1].isfinite().all()
