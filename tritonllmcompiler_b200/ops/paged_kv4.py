"""A paged KV cache held in 4 bits: writing it, reading rows back, and attention over it.

The reference's cache (python/triton_llm/ops/paged_attention.py:92-128) holds fp16 or bf16. Here
each group of 32 channels of a token and head is 16 levels between its minimum and maximum, with
an fp16 scale and zero: 1.25 * D bytes per token and KV head for K and V together instead of 4 * D,
so decode, which is bound by reading the cache, reads less than a third. Tokens are addressed by
slot (block * block_size + offset) when written, as ``paged_plan`` gives them, and by block table
when attended to. These are extensions: the package root and ``ops`` keep the reference's four
exports, and they are imported from this module.
"""
from __future__ import annotations

import functools

import torch

from tritonllmcompiler_b200 import _lib

GROUP = 32  # channels that share a scale and a zero


def new_kv4_cache(num_blocks: int, num_kv_heads: int, block_size: int, head_dim: int, *,
                  device: torch.device | str = "cuda") -> torch.Tensor:
    """An empty cache: uint8 [num_blocks, num_kv_heads, block_size / 16, 20 * head_dim], K and V
    of 16 tokens of one head per innermost row. Head dims 64 and 128, block sizes 16, 32, 64."""
    assert head_dim in (64, 128) and block_size in (16, 32, 64)
    return torch.zeros((num_blocks, num_kv_heads, block_size // 16, 20 * head_dim),
                       dtype=torch.uint8, device=device)


@functools.lru_cache(maxsize=256)
def _cache_sizes(shape: tuple, stride: tuple, dtype: torch.dtype, block_size: int):
    """(num_blocks, num_kv_heads, head_dim, strides for the library) of a cache made by
    ``new_kv4_cache``, or a slice of a larger one that keeps its two innermost dimensions together."""
    assert len(shape) == 4 and dtype == torch.uint8
    n, h, pieces, row = shape
    assert block_size in (16, 32, 64) and pieces == block_size // 16
    assert row in (1280, 2560), "head dim must be 64 or 128"
    assert stride[3] == 1 and (stride[2] == row or pieces == 1) and stride[0] % 16 == 0 and stride[1] % 16 == 0, \
        "cache rows must be contiguous and 16-byte aligned"
    return n, h, row // 20, _lib.int64s(*stride[:2])


def _check_cache(cache: torch.Tensor, block_size: int):
    assert cache.get_device() >= 0 and cache.data_ptr() % 16 == 0
    return _cache_sizes(cache.shape, cache.stride(), cache.dtype, block_size)


@functools.lru_cache(maxsize=256)
def _row_strides(stride: tuple):
    """The strides of [T, H, D] rows for the library, or None where it cannot read them."""
    if stride[2] != 1 or stride[0] % 8 or stride[1] % 8:
        return None
    return _lib.int64s(*stride[:2])


def _rows(t: torch.Tensor):
    """(the rows as the library reads them, their strides)."""
    s = _row_strides(t.stride())
    if s is None or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        s = _row_strides(t.stride())
    return t, s


def _int32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int32 and t.is_contiguous() else _lib.int32(t).contiguous()


def paged_kv4_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor,
                     *, block_size: int) -> None:
    """Quantises k[t] and v[t] ([T, Hkv, D], fp16 or bf16) into slot slots[t] of the cache, in
    place, for every t with slots[t] >= 0. A slot past the pool is skipped and flagged
    (``_lib.debug_status()`` returns 0x200). A group of 32 channels that holds a NaN, an infinity or a
    value beyond fp16's range reads back as NaN, and so do its channels in the attention of rows that
    see the token."""
    n, h, d, sc = _check_cache(cache, block_size)
    t = k.shape[0]
    assert k.shape == (t, h, d) and v.shape == k.shape and slots.shape == (t,)
    assert k.dtype in _lib.DTYPE_CODES and v.dtype == k.dtype
    device = cache.get_device()
    assert k.get_device() == device and v.get_device() == device and slots.get_device() == device
    if t == 0:
        return
    k, sk = _rows(k)
    v, sv = _rows(v)
    sl = _int32(slots)
    _lib.launch(device, _lib.load().tllm_paged_kv4_append, k.data_ptr(), v.data_ptr(),
                cache.data_ptr(), sl.data_ptr(), t, h, d, block_size, n, sk, sv, sc,
                _lib.DTYPE_CODES[k.dtype])


def paged_kv4_gather(cache: torch.Tensor, slots: torch.Tensor, *, block_size: int,
                     dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows ([T, Hkv, D] each, of the given dtype) that slots [T] hold; zeros where
    slots[t] < 0 or past the pool (the latter flagged)."""
    n, h, d, sc = _check_cache(cache, block_size)
    device = cache.get_device()
    assert dtype in _lib.DTYPE_CODES and slots.dim() == 1 and slots.get_device() == device
    t = slots.shape[0]
    k = cache.new_empty((t, h, d), dtype=dtype)
    v = torch.empty_like(k)
    sl = _int32(slots)
    so = _row_strides((h * d, d, 1))
    _lib.launch(device, _lib.load().tllm_paged_kv4_gather, cache.data_ptr(), sl.data_ptr(),
                k.data_ptr(), v.data_ptr(), t, h, d, block_size, n, so, so, sc,
                _lib.DTYPE_CODES[dtype])
    return k, v


def paged_attention_kv4(q: torch.Tensor, cache: torch.Tensor, block_tables: torch.Tensor,
                        context_lens: torch.Tensor, cu_seqlens: torch.Tensor, max_new: int, *,
                        block_size: int, sm_scale: float | None = None,
                        causal: bool = True) -> torch.Tensor:
    """Attention of packed new tokens over the 4-bit paged cache.

    q: [T, Hq, D] with Hq % Hkv == 0 (query head h reads KV head h // (Hq // Hkv)); sequence b's
    new tokens are rows cu_seqlens[b] .. cu_seqlens[b + 1] ([B + 1]), at most max_new of them, and
    are already in the cache: context_lens[b] counts them. New token s sits at position
    context_lens[b] - n_b + s; with causal it sees keys up to its own position. Decode is one row
    per sequence; prefill chunks, speculative tokens and idle sequences may be mixed in one call.
    Returns a new [T, Hq, D] tensor: NaN in rows that see no key, as in ``paged_attention``, and
    zeros in rows before cu_seqlens[0] or past cu_seqlens[B]. A sequence with more than max_new tokens
    is flagged (``_lib.debug_status()`` returns 0x200); its tokens past the first max_new give NaN."""
    n, hkv, d, sc = _check_cache(cache, block_size)
    assert q.dim() == 3 and q.shape[2] == d and q.dtype in _lib.DTYPE_CODES
    t, hq, _ = q.shape
    assert hkv >= 1 and hq % hkv == 0
    assert block_tables.dim() == 2 and context_lens.dim() == 1 and cu_seqlens.dim() == 1
    b, max_blocks = block_tables.shape
    assert context_lens.shape[0] == b and cu_seqlens.shape[0] == b + 1
    device = cache.get_device()
    assert q.get_device() == device and block_tables.get_device() == device
    assert context_lens.get_device() == device and cu_seqlens.get_device() == device
    if sm_scale is None:
        sm_scale = d ** -0.5
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if t == 0 or hq == 0:
        return out
    q, sq = _rows(q)
    bt = _lib.int32(block_tables)
    cl, cu = _int32(context_lens), _int32(cu_seqlens)
    max_new = min(int(max_new), t)
    lib = _lib.load()
    ws_bytes = lib.tllm_paged_kv4_attn_workspace_size(b, t, hq, hkv, max_new, d, block_size, max_blocks)
    ws = cache.new_empty((ws_bytes,))
    _lib.launch(device, lib.tllm_paged_kv4_attn, q.data_ptr(), cache.data_ptr(), bt.data_ptr(),
                cl.data_ptr(), cu.data_ptr(), out.data_ptr(), ws.data_ptr(), ws_bytes, b, t, hq,
                hkv, max_new, d, block_size, max_blocks, n, sq, sc, _lib.strides(bt),
                _row_strides((hq * d, d, 1)), float(sm_scale), int(bool(causal)),
                _lib.DTYPE_CODES[q.dtype])
    return out
