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


def _check_cache(cache: torch.Tensor, block_size: int) -> tuple[int, int, int]:
    """(num_blocks, num_kv_heads, head_dim) of a cache made by ``new_kv4_cache`` (or a slice of a
    larger one that keeps its two innermost dimensions together)."""
    assert cache.is_cuda and cache.dim() == 4 and cache.dtype == torch.uint8
    n, h, pieces, row = cache.shape
    assert block_size in (16, 32, 64) and pieces == block_size // 16
    assert row in (1280, 2560), "head dim must be 64 or 128"
    s = cache.stride()
    assert s[3] == 1 and (s[2] == row or pieces == 1) and s[0] % 16 == 0 and s[1] % 16 == 0 \
        and cache.data_ptr() % 16 == 0, "cache rows must be contiguous and 16-byte aligned"
    return n, h, row // 20


def _rows_ok(t: torch.Tensor) -> bool:
    s = t.stride()
    return s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and t.data_ptr() % 16 == 0


def _int32(t: torch.Tensor) -> torch.Tensor:
    return t if t.dtype == torch.int32 and t.is_contiguous() else t.to(torch.int32).contiguous()


def paged_kv4_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, slots: torch.Tensor,
                     *, block_size: int) -> None:
    """Quantises k[t] and v[t] ([T, Hkv, D], fp16 or bf16) into slot slots[t] of the cache, in
    place, for every t with slots[t] >= 0. A slot past the pool is skipped and flagged
    (``_lib.debug_status()`` returns 0x200). Groups that hold a NaN, an infinity or values beyond
    fp16's range do not read back as numbers."""
    n, h, d = _check_cache(cache, block_size)
    assert k.is_cuda and k.dim() == 3 and v.shape == k.shape and tuple(k.shape[1:]) == (h, d)
    assert k.dtype in _lib.DTYPE_CODES and v.dtype == k.dtype
    t = k.shape[0]
    assert slots.shape == (t,)
    assert k.device == cache.device and v.device == cache.device and slots.device == cache.device
    if t == 0:
        return
    kk, vv = (x if _rows_ok(x) else x.contiguous() for x in (k, v))
    sl = _int32(slots)
    with _lib.on_device(cache):
        _lib.check(_lib.load().tllm_paged_kv4_append(
            kk.data_ptr(), vv.data_ptr(), cache.data_ptr(), sl.data_ptr(), t, h, d, block_size, n,
            _lib.strides(kk, 2), _lib.strides(vv, 2), _lib.strides(cache, 2),
            _lib.DTYPE_CODES[k.dtype], _lib.stream_of(cache)))


def paged_kv4_gather(cache: torch.Tensor, slots: torch.Tensor, *, block_size: int,
                     dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows ([T, Hkv, D] each, of the given dtype) that slots [T] hold; zeros where
    slots[t] < 0 or past the pool (the latter flagged)."""
    n, h, d = _check_cache(cache, block_size)
    assert dtype in _lib.DTYPE_CODES and slots.dim() == 1 and slots.device == cache.device
    t = slots.shape[0]
    k = torch.empty((t, h, d), dtype=dtype, device=cache.device)
    v = torch.empty((t, h, d), dtype=dtype, device=cache.device)
    sl = _int32(slots)
    with _lib.on_device(cache):
        _lib.check(_lib.load().tllm_paged_kv4_gather(
            cache.data_ptr(), sl.data_ptr(), k.data_ptr(), v.data_ptr(), t, h, d, block_size, n,
            _lib.strides(k, 2), _lib.strides(v, 2), _lib.strides(cache, 2),
            _lib.DTYPE_CODES[dtype], _lib.stream_of(cache)))
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
    zeros in rows past cu_seqlens[B]."""
    n, hkv, d = _check_cache(cache, block_size)
    assert q.is_cuda and q.dim() == 3 and q.shape[2] == d and q.dtype in _lib.DTYPE_CODES
    t, hq, _ = q.shape
    assert hkv >= 1 and hq % hkv == 0
    assert block_tables.dim() == 2 and context_lens.dim() == 1 and cu_seqlens.dim() == 1
    b = block_tables.shape[0]
    assert context_lens.shape[0] == b and cu_seqlens.shape[0] == b + 1
    assert q.device == cache.device and block_tables.device == cache.device
    assert context_lens.device == cache.device and cu_seqlens.device == cache.device
    if sm_scale is None:
        sm_scale = d ** -0.5
    out = torch.empty((t, hq, d), device=q.device, dtype=q.dtype)
    if t == 0 or hq == 0:
        return out
    qq = q if _rows_ok(q) else q.contiguous()
    bt = block_tables if block_tables.dtype == torch.int32 else block_tables.to(torch.int32)
    cl, cu = _int32(context_lens), _int32(cu_seqlens)
    max_new = min(int(max_new), t)
    lib = _lib.load()
    with _lib.on_device(q):
        ws_bytes = lib.tllm_paged_kv4_attn_workspace_size(b, t, hq, hkv, max_new, d, block_size,
                                                          bt.shape[1])
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device) if ws_bytes else None
        _lib.check(lib.tllm_paged_kv4_attn(
            qq.data_ptr(), cache.data_ptr(), bt.data_ptr(), cl.data_ptr(), cu.data_ptr(),
            out.data_ptr(), None if ws is None else ws.data_ptr(), ws_bytes, b, t, hq, hkv,
            max_new, d, block_size, bt.shape[1], n, _lib.strides(qq, 2), _lib.strides(cache, 2),
            _lib.strides(bt), _lib.strides(out, 2), float(sm_scale), int(bool(causal)),
            _lib.DTYPE_CODES[q.dtype], _lib.stream_of(q)))
    return out
