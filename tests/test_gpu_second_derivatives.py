"""The training forms give first derivatives: a second one is refused, not left out of a sum."""
import pytest
import torch

from tritonllmcompiler_b200.ops.flash_backward import flash_attention_train
from tritonllmcompiler_b200.ops.qk_norm_rope import qk_norm_rope_train

pytestmark = pytest.mark.gpu


def _refused(outputs, leaf):
    loss = sum(o.float().square().sum() for o in outputs)
    grad, = torch.autograd.grad(loss, leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        (loss + grad.float().square().sum()).backward()


def test_qk_norm_rope(cuda_device):
    q, k = (torch.randn(4, h, 64, dtype=torch.float16, device="cuda", requires_grad=True) for h in (2, 1))
    w = torch.ones(64, dtype=torch.float16, device="cuda", requires_grad=True)
    cos, sin = torch.ones(8, 32, device="cuda"), torch.zeros(8, 32, device="cuda")
    at = torch.arange(4, dtype=torch.int32, device="cuda")
    for leaf in (q, k, w):
        _refused(qk_norm_rope_train(q, k, w, w, cos, sin, at), leaf)


def test_flash_attention(cuda_device):
    q, k, v = (torch.randn(1, 2, 128, 64, dtype=torch.float16, device="cuda", requires_grad=True) for _ in range(3))
    for leaf in (q, k, v):
        _refused([flash_attention_train(q, k, v, causal=True)], leaf)
