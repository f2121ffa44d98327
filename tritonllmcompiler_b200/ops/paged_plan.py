"""Block tables and slot maps of a paged cache, built on the GPU from request lengths.

The reference decodes from block tables that its caller fills on the host
(python/triton_llm/ops/paged_attention.py:92-128). A serving step has to extend them before
every model call: new blocks for the requests whose tokens do not fit their last block, the slot
of every new token, its position and the packed batch's cumulative lengths. ``paged_plan`` does
all of it in one launch without reading anything back. It is an extension: the package root and
``ops`` keep the reference's four exports, and it is imported from this module.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from tritonllmcompiler_b200 import _lib


class PagedPlan(NamedTuple):
    """What one step needs (int32, on the device)."""

    slots: torch.Tensor  # [max_tokens]: block * block_size + offset of each packed new token, or -1
    positions: torch.Tensor  # [max_tokens]: position of each new token in its sequence
    cu_seqlens: torch.Tensor  # [B + 1]: packed row where each sequence's new tokens start
    new_lens: torch.Tensor  # [B]: length of each sequence after the step
    taken: torch.Tensor  # [1]: how many entries of free_blocks the step took, from free_start on


def paged_plan(block_tables: torch.Tensor, seq_lens: torch.Tensor, n_new: torch.Tensor,
               free_blocks: torch.Tensor, *, block_size: int, max_tokens: int,
               free_start: torch.Tensor | None = None) -> PagedPlan:
    """Plans one step: n_new[b] new tokens for sequence b, which has seq_lens[b] tokens in the
    cache and their blocks in block_tables[b].

    block_tables [B, max_blocks] (int32) gets the new blocks, in place, taken from free_blocks in the
    order of the sequences, from entry free_start[0] on ([1], on the device; the first entry without it).
    A loop of steps over one list keeps that count and adds plan.taken to it after each step; the
    same entries given twice are the same blocks given to two requests. max_tokens is the length of the packed batch
    (at least the sum of n_new; rows past that sum get slot -1 and position 0). A sequence that
    its table row, the free list or max_tokens cannot hold is refused whole: its slots are -1,
    its new length is the old one and its table row stays. Negative lengths count as 0."""
    assert block_tables.dim() == 2 and block_tables.dtype == torch.int32
    device = block_tables.get_device()
    b, max_blocks = block_tables.shape
    assert device >= 0 and seq_lens.shape == (b,) and n_new.shape == (b,) and free_blocks.dim() == 1
    assert seq_lens.get_device() == device and n_new.get_device() == device
    assert free_blocks.get_device() == device and block_size >= 1 and max_tokens >= 0
    assert free_start is None or (free_start.numel() == 1 and free_start.get_device() == device)
    max_tokens = int(max_tokens)
    sl, nn, fb = (t if t.dtype == torch.int32 and t.is_contiguous() else _lib.int32(t).contiguous()
                  for t in (seq_lens, n_new, free_blocks))
    out = block_tables.new_empty((2 * max_tokens + 2 * b + 2,))
    at = out.data_ptr()
    fs = None if free_start is None else _lib.int32(free_start)
    _lib.launch(device, _lib.load().tllm_paged_plan_from, block_tables.data_ptr(), sl.data_ptr(),
                nn.data_ptr(), fb.data_ptr(), None if fs is None else fs.data_ptr(), at, at + 4 * max_tokens, at + 8 * max_tokens,
                at + 4 * (2 * max_tokens + b + 1), at + 4 * (2 * max_tokens + 2 * b + 1), b,
                max_blocks, fb.shape[0], max_tokens, block_size, _lib.strides(block_tables))
    return PagedPlan(*out.split_with_sizes((max_tokens, max_tokens, b + 1, b, 1)))
