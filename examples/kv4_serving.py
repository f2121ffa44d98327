"""A small decoder served from a 4-bit paged cache, with the operators a serving step is made of.

Random weights, greedy tokens. Every step takes a packed batch of new tokens (whole prompts first,
one token per request after that) through, per layer: RMS norm and projection, ``qk_norm_rope``,
``paged_kv4_append``, ``paged_attention_kv4``, the output projection and ``swiglu``. ``paged_plan``
extends the block tables and gives slots, positions and offsets without reading anything back.

    python examples/kv4_serving.py --requests 16 --new 32
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tritonllmcompiler_b200 import swiglu  # noqa: E402
from tritonllmcompiler_b200.ops.paged_kv4 import (new_kv4_cache, paged_attention_kv4,  # noqa: E402
                                                  paged_kv4_append)
from tritonllmcompiler_b200.ops.paged_plan import paged_plan  # noqa: E402
from tritonllmcompiler_b200.ops.qk_norm_rope import qk_norm_rope  # noqa: E402


class Decoder:
    """Weights of a decoder of `layers` layers, on the GPU."""

    def __init__(self, *, vocab=256, width=512, layers=2, heads=8, kv_heads=2, head_dim=64, hidden=1024,
                 positions=4096, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rand = lambda *s: (torch.randn(s, generator=g, device="cuda") * s[0] ** -0.5).to(dtype)  # noqa: E731
        self.heads, self.kv_heads, self.head_dim, self.dtype = heads, kv_heads, head_dim, dtype
        self.embed = (rand(vocab, width).float() * vocab ** 0.5).to(dtype)
        one = lambda: torch.ones(head_dim, dtype=dtype, device="cuda")  # noqa: E731
        self.layers = [dict(qkv=rand(width, (heads + 2 * kv_heads) * head_dim), q_norm=one(), k_norm=one(),
                            out=rand(heads * head_dim, width), w1=rand(width, hidden), w3=rand(width, hidden),
                            down=rand(hidden, width)) for _ in range(layers)]
        inv = 10000.0 ** (-torch.arange(0, head_dim, 2, device="cuda") / head_dim)
        angle = torch.arange(positions, device="cuda")[:, None] * inv
        self.cos, self.sin = angle.cos(), angle.sin()


def _norm(x: torch.Tensor) -> torch.Tensor:
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6)).to(x.dtype)


class Server:
    """Requests over one pool of blocks: block tables, lengths, and a 4-bit cache per layer."""

    def __init__(self, model: Decoder, requests: int, *, blocks=512, max_blocks=64, block_size=16):
        self.model, self.block_size = model, block_size
        self.caches = [new_kv4_cache(blocks, model.kv_heads, block_size, model.head_dim) for _ in model.layers]
        self.tables = torch.zeros((requests, max_blocks), dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(blocks, device="cuda").int()
        self.taken = torch.zeros(1, dtype=torch.int32, device="cuda")  # entries of free that are in use
        # Requests that the pool or their table could not hold at some step: their logits are NaN from there on.
        self.refused = torch.zeros(requests, dtype=torch.bool, device="cuda")

    def step(self, tokens: torch.Tensor, n_new: torch.Tensor, most: int) -> torch.Tensor:
        """Runs the packed new tokens, n_new[b] of request b (at most `most`); returns the logits after
        each request's last one, NaN for a request without new tokens or refused."""
        m, bs = self.model, self.block_size
        plan = paged_plan(self.tables, self.lens, n_new, self.free, block_size=bs, max_tokens=tokens.shape[0],
                          free_start=self.taken)
        self.taken += plan.taken
        self.refused |= plan.new_lens != self.lens + n_new
        self.lens = plan.new_lens.clone()
        x = m.embed[tokens]
        t, hq, hkv = tokens.shape[0], m.heads, m.kv_heads
        for layer, cache in zip(m.layers, self.caches):
            qkv = (_norm(x) @ layer["qkv"]).view(t, hq + 2 * hkv, m.head_dim)
            q, k = qk_norm_rope(qkv[:, :hq], qkv[:, hq:hq + hkv], layer["q_norm"], layer["k_norm"], m.cos, m.sin,
                                plan.positions)
            paged_kv4_append(k, qkv[:, hq + hkv:], cache, plan.slots, block_size=bs)
            o = paged_attention_kv4(q, cache, self.tables, self.lens, plan.cu_seqlens, most, block_size=bs)
            x = x + o.view(t, -1) @ layer["out"]
            x = x + swiglu(_norm(x), layer["w1"], layer["w3"]) @ layer["down"]
        last = plan.cu_seqlens[1:].long() - 1
        logits = _norm(x[last]).float() @ m.embed.float().T
        return logits.masked_fill((self.refused | (n_new <= 0))[:, None], float("nan"))


def generate(model: Decoder, prompts: list[list[int]], new: int, **how) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens [requests, new], the logits they were taken from): prompts of any lengths in one step,
    then a token per request and step. Raises where the pool or a table is too small for that (seen at the
    end: nothing is read back between the steps)."""
    server = Server(model, len(prompts), **how)
    tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
    n_new = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
    most, out, logits = max(map(len, prompts)), [], []
    one = torch.ones_like(n_new)
    for _ in range(new):
        logits.append(server.step(tokens, n_new, most))
        tokens, n_new, most = logits[-1].argmax(-1), one, 1
        out.append(tokens)
    if server.refused.any():
        raise RuntimeError(f"the cache cannot hold requests {server.refused.nonzero().flatten().tolist()}")
    return torch.stack(out, 1), torch.stack(logits, 1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=16)
    ap.add_argument("--new", type=int, default=32)
    a = ap.parse_args()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 256, (int(torch.randint(1, 400, (1,), generator=g)),), generator=g).tolist()
               for _ in range(a.requests)]
    model = Decoder()
    how = dict(blocks=32 * a.requests, max_blocks=32)
    generate(model, prompts, 2, **how)
    torch.cuda.synchronize()
    t = time.perf_counter()
    tokens, _ = generate(model, prompts, a.new, **how)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    print(f"{a.requests} requests, {sum(map(len, prompts))} prompt tokens, {tokens.numel()} new tokens in {t * 1e3:.1f} ms")
    print("first request:", tokens[0].tolist())


if __name__ == "__main__":
    main()
