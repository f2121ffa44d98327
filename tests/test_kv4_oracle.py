"""The oracle of the serving-step operators, pinned on the CPU: against the existing oracles where
they overlap, against differences, and by hand where neither says anything. And the C entries'
refusals, which come before any CUDA call."""
import ctypes

import numpy as np
import pytest

from oracle import kv4_oracle as O
from oracle import ops_oracle
from tritonllmcompiler_b200 import _lib
from tritonllmcompiler_b200.ops import qk_norm_rope as Q


def test_norm_rope_is_rmsnorm_rope_with_one_axis():
    """Where the normed value is not rounded the two definitions meet."""
    rng = np.random.RandomState(0)
    x, w = rng.randn(1, 7, 3, 16).astype(np.float32), (1 + rng.rand(16)).astype(np.float32)
    a = rng.randn(7, 8).astype(np.float32)
    full = np.concatenate([a, a], -1)
    want = ops_oracle.rmsnorm_rope(x, w, np.cos(full), np.sin(full), dtype="fp32")
    got = O.norm_rope(x[0], w, np.cos(a), np.sin(a), np.arange(7)[None], (8,))
    assert np.abs(got - want[0]).max() < 1e-5


def test_axes_of_pairs():
    assert O.axis_of_pair((2, 1, 3), False).tolist() == [0, 0, 1, 2, 2, 2]
    assert O.axis_of_pair((4, 1, 1), True).tolist() == [0, 1, 2, 0, 0, 0]
    assert O.axis_of_pair((0, 3, 3), True).tolist() == [0, 1, 2, 0, 1, 2]
    for sections, mix in (((2, 1, 3), False), ((4, 2, 2), True), ((1, 3, 4), True), ((2, 2, 2, 2), True), ((8,), True)):
        words = Q._axis_words(sections, mix, sum(sections))
        got = [(words[i // 16] >> (2 * (i % 16))) & 3 for i in range(sum(sections))]
        assert got == O.axis_of_pair(sections, mix).tolist()


def test_norm_rope_gradient_against_differences():
    """Central differences in 64 bits: the step's error is third derivatives times 1e-10, the
    cancellation's 1e-16 / 1e-5."""
    rng = np.random.RandomState(3)
    T, H, D, sec = 2, 2, 16, (3, 5)
    x, dz = rng.randn(T, H, D), rng.randn(T, H, D)
    w, ang = 1 + 0.2 * rng.randn(D), rng.randn(11, 8)
    pos = rng.randint(0, 11, (2, T))
    f = lambda x, w: (O.norm_rope(x, w, np.cos(ang), np.sin(ang), pos, sec) * dz).sum()  # noqa: E731
    dx, dw, _, _ = O.norm_rope_grad(dz, x, w, np.cos(ang), np.sin(ang), pos, sec)
    e = 1e-5
    for at, grad, of in ((x, dx, lambda d: f(x + d, w) - f(x - d, w)), (w, dw, lambda d: f(x, w + d) - f(x, w - d))):
        for i in np.ndindex(at.shape):
            d = np.zeros_like(at)
            d[i] = e
            assert abs(of(d) / (2 * e) - grad[i]) < 1e-7


def test_quantise_by_hand():
    x = np.zeros((1, 32), np.float32)
    x[0, :4] = [-1.5, 0.0, 3.0, 6.0]  # range 7.5: steps of 0.5 from -1.5
    codes, s, z = O.quantise(x)
    assert s.item() == 0.5 and z.item() == -1.5
    assert codes[0, 0, :5].tolist() == [0, 3, 9, 15, 3]
    v, size = O.dequantise(codes, s, z)
    assert v[0, :4].tolist() == [-1.5, 0.0, 3.0, 6.0] and size[0, 0] == 1.5
    codes, s, z = O.quantise(np.full((1, 32), 2.25, np.float32))
    assert (codes == 0).all() and O.dequantise(codes, s, z)[0].tolist() == [[2.25] * 32]


def test_attention_is_the_flash_oracle_on_the_values():
    rng = np.random.RandomState(5)
    q, k, v = rng.randn(6, 4, 16), rng.randn(6, 2, 16), rng.randn(6, 2, 16)
    o, _, _ = O.attention(q, k, v, np.abs(k), np.abs(v), scale=0.25, causal=True, n_new=6)
    for h in range(4):
        args = [np.float32(x[None, None]) for x in (q[:, h], k[:, h // 2], v[:, h // 2])]
        want = ops_oracle.flash_attention(*args, causal=True, sm_scale=0.25, dtype="fp32")
        assert np.abs(o[:, h] - want[0, 0]).max() < 1e-5


def test_plan_by_hand():
    table = [[4, -1, -1], [-1, -1, -1]]
    slots, pos, cu, lens, taken, table = O.paged_plan(table, [3, 0], [2, 5], [9, 8, 7, 6], block_size=4, max_tokens=8)
    assert slots.tolist() == [19, 36, 32, 33, 34, 35, 28, -1] and pos.tolist() == [3, 4, 0, 1, 2, 3, 4, 0]
    assert cu.tolist() == [0, 2, 7] and lens.tolist() == [5, 5] and taken == 3
    assert table.tolist() == [[4, 9, -1], [8, 7, -1]]


def _arr(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_entries_validate_before_any_launch():
    lib = _lib.load()
    said = lambda rc, text: rc != 0 and text in lib.tllm_last_error()  # noqa: E731
    s2, words = _arr(64, 64), (ctypes.c_uint32 * 4)()
    plan = lambda B=1, n=4, bs=16, sbt=_arr(4, 1), out=16: lib.tllm_paged_plan(  # noqa: E731
        16, 16, 16, 16, 16, 16, out, 16, out, B, 4, n, 8, bs, sbt, None)
    assert said(plan(B=-1), b"negative") and said(plan(bs=0), b"block_size 0") and said(plan(B=16385), b"16384")
    assert said(plan(sbt=None), b"null stride") and said(plan(out=None), b"null output")
    rope = lambda D=64, axes=1, w=words, sq=s2, dtype=0, rows=8, p=16, scos=32: lib.tllm_qk_norm_rope(  # noqa: E731
        p, 16, 16, 16, 16, 16, 16, 16, 16, 1, 1, 1, D, rows, scos, 32, axes, 1, w, sq, s2, s2, s2, 1e-6, dtype, None)
    assert said(rope(D=48), b"head dim 48") and said(rope(axes=5), b"5 position axes") and said(rope(dtype=2), b"dtype 2")
    two = (ctypes.c_uint32 * 4)(2, 0, 0, 0)
    assert said(rope(w=two, axes=2), b"rotary pair 0") and said(rope(sq=_arr(65, 64)), b"multiples of 8")
    assert said(rope(rows=0), b"empty cos/sin") and said(rope(p=8), b"16-byte aligned") and said(rope(p=None), b"null tensor")
    assert said(rope(scos=33), b"cos/sin rows")
    grad = lib.tllm_qk_norm_rope_bwd(16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, 16, None, 0, 1, 1, 1, 64, 8, 32, 32, 1, 1,
                                     words, s2, s2, s2, s2, s2, s2, 1e-6, 0, None)
    assert grad == 3 and b"workspace" in lib.tllm_last_error()
    append = lambda D=64, bs=16, sk=s2, sc=_arr(1280, 1280), c=16, dtype=0: lib.tllm_paged_kv4_append(  # noqa: E731
        16, 16, c, 16, 1, 1, D, bs, 4, sk, s2, sc, dtype, None)
    assert said(append(D=32), b"head dim 32") and said(append(bs=8), b"block_size 8") and said(append(sk=_arr(4, 64)), b"multiples")
    assert said(append(sc=_arr(1288, 8)), b"cache strides") and said(append(c=None), b"null tensor") and said(append(dtype=7), b"dtype 7")
    attn = lambda Hq=2, Hkv=1, D=64, bs=16, ws=0, T=1, sq=s2, q=16: lib.tllm_paged_kv4_attn(  # noqa: E731
        q, 16, 16, 16, 16, 16, None, ws, 1, T, Hq, Hkv, 1, D, bs, 4, 4, sq, _arr(1280, 1280), _arr(4, 1), s2, 0.1, 1, 0, None)
    assert said(attn(Hq=3, Hkv=2), b"do not group") and said(attn(D=96), b"head dim 96") and said(attn(bs=128), b"block_size 128")
    assert said(attn(T=-1), b"negative") and said(attn(sq=_arr(60, 64)), b"multiples of 8") and said(attn(q=None), b"null tensor")
    assert attn() == 3 and b"workspace" in lib.tllm_last_error()
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.check(3)


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.tllm_qk_norm_rope_bwd_workspace_size(0, 4, 2, 64) == 0
    assert lib.tllm_qk_norm_rope_bwd_workspace_size(100, 4, 2, 64) % (64 * 4) == 0
    size = lib.tllm_paged_kv4_attn_workspace_size
    assert size(1, 0, 8, 2, 1, 64, 16, 4) == 0 and size(1, 1, 8, 3, 1, 64, 16, 4) == 0
    one, many, rows = size(1, 1, 8, 2, 1, 64, 16, 4), size(64, 64, 8, 2, 1, 64, 16, 512), size(8, 4096, 8, 2, 512, 64, 16, 512)
    assert 0 < one < many and rows > 0
    # bounded by the GPU, not by the lengths
    assert size(64, 64, 8, 2, 1, 64, 16, 1 << 16) == many
