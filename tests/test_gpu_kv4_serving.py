"""The serving step as a whole: examples/kv4_serving.py against the same decoder in fp32 torch with
the cache's values kept in full, and against itself with the prompts fed in pieces."""
import importlib.util
import os

import pytest
import torch

from oracle import kv4_oracle as O
from tritonllmcompiler_b200 import _lib

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def serving():
    spec = importlib.util.spec_from_file_location("kv4_serving", os.path.join(ROOT, "examples", "kv4_serving.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def _plain(S, model, tokens):
    """Logits after every token of one request, in fp32, K and V through 4 bits."""
    x = model.embed[torch.tensor(tokens, device="cuda")].float()
    t, hq, hkv, d = x.shape[0], model.heads, model.kv_heads, model.head_dim
    norm = lambda v: v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    four = lambda v: torch.from_numpy(O.dequantise(*O.quantise(v.cpu().numpy()))[0]).float().cuda()  # noqa: E731
    cos, sin = model.cos[:t, None], model.sin[:t, None]

    def turn(v):
        a, b = norm(v).chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)

    for layer in model.layers:
        w = {k: v.float() for k, v in layer.items()}
        q, k, v = (norm(x) @ w["qkv"]).view(t, -1, d).split([hq, hkv, hkv], 1)
        q, k, v = turn(q), four(turn(k)), four(v)
        k, v = (z.repeat_interleave(hq // hkv, 1) for z in (k, v))
        s = torch.einsum("qhd,khd->hqk", q, k) * d ** -0.5
        s = s.masked_fill(torch.ones(t, t, device="cuda").triu(1).bool(), float("-inf")).softmax(-1)
        x = x + torch.einsum("hqk,khd->qhd", s, v).reshape(t, -1) @ w["out"]
        y = norm(x)
        x = x + (torch.nn.functional.silu(y @ w["w1"]) * (y @ w["w3"])) @ w["down"]
    return norm(x) @ model.embed.float().T


@pytest.mark.parametrize("dtype,bound", [(torch.float16, 0.05), (torch.bfloat16, 0.1)])
def test_generation_follows_the_plain_decoder(cuda_device, serving, dtype, bound):
    """Logits of prompts and generated tokens. fp16 or bf16 activations between the layers move some
    K and V values across the 1/15 steps of their groups: the logits differ by a few per cent of
    their size (a wrong position, page or mask moves them by all of it)."""
    model = serving.Decoder(dtype=dtype, seed=3)
    prompts = [[5, 9, 250], list(range(40, 90)), [7], [(i * 37) % 256 for i in range(130)]]
    tokens, logits = serving.generate(model, prompts, 6, blocks=64, max_blocks=16)
    assert _lib.debug_status() == 0
    for b, p in enumerate(prompts):
        want = _plain(serving, model, p + tokens[b].tolist())[len(p) - 1:len(p) + 5]
        assert ((logits[b] - want).norm() / want.norm()).item() < bound


def test_prompts_in_pieces(cuda_device, serving):
    """The same requests with their prompts fed a few tokens at a time: the same slots, nearly the
    same logits (different kernels, the same rounding points)."""
    model = serving.Decoder(dtype=torch.float16, seed=4)
    prompts = [[(i * 31 + b) % 256 for i in range(n)] for b, n in enumerate((70, 3, 33))]
    _, whole = serving.generate(model, prompts, 1, blocks=32, max_blocks=8)
    server = serving.Server(model, 3, blocks=32, max_blocks=8)
    fed = [0, 0, 0]
    while any(f < len(p) for f, p in zip(fed, prompts)):
        n = [min(9, len(p) - f) for f, p in zip(fed, prompts)]
        flat = torch.tensor([t for f, k, p in zip(fed, n, prompts) for t in p[f:f + k]], device="cuda")
        out = server.step(flat, torch.tensor(n, dtype=torch.int32, device="cuda"), 9)
        for b, k in enumerate(n):
            fed[b] += k
            if k and fed[b] == len(prompts[b]):
                assert ((out[b] - whole[b, 0]).norm() / whole[b, 0].norm()).item() < 0.05
    assert server.lens.tolist() == [70, 3, 33] and _lib.debug_status() == 0
