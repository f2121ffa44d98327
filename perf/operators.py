"""The serving-step operators over the 4-bit paged cache, and the normed, rotated queries and
keys in front of attention: cases, inputs, the plain torch form of each, and the same results in
64 bits. ``own`` selects the plain form (False) or this package's operators (True).

Kinds of cases:

* ``plan``: block tables and slot maps from request lengths (``paged_plan``).
* ``rope`` / ``rope_grad``: RMS norm of every query and key head and rotation by positions of
  several axes, forward and backward (``qk_norm_rope``, ``qk_norm_rope_backward``).
* ``append``: quantising new K/V rows into the 4-bit paged cache, and reading them back
  (``paged_kv4_append``, ``paged_kv4_gather``).
* ``attn``: attention of new tokens over that cache (``paged_attention_kv4``).

Cache layout, per physical block and KV head, in pieces of 16 tokens of 20 * D bytes: K codes
(8 D), K scales [token][group] and zeros [token][group] (fp16, D bytes each), V codes (8 D), V
scales [token][group], V zeros [group][token]. A group is 32 channels. Within a token's K codes,
32-bit word 4 * (D / 32) is indexed [lane 4][word w], holding channels 32 w + 8 lane + j, channel
j at bits 4 (j / 2) + 16 (j % 2). V codes are stored by pairs of tokens: 8 chunks of D / 8 bytes,
chunk n ^ swz(pair) holding, for each of the two tokens, 16 bits per group g with channels
32 g + 4 n + j at bits 4 j; swz is 2 (pair % 4) at D 128 and 4 (pair / 2 % 2) at D 64.
"""
import math
import random

import torch

own = False

GROUP = 32
PIECE = 16  # tokens per piece of the cache
EPS = 1e-6
THETA = 10000.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# --------------------------------------------------------------------------- cases
def listed():
    return [
        # One decode step's bookkeeping for 64 running requests: latency only.
        dict(name="plan_decode", kind="plan", B=64, ctx_lo=512, ctx_hi=8192, new_lo=1, new_hi=1, bs=16, lens=3),
        # A mixed batch: prompts, chunks and idle requests, some 64 K new tokens.
        dict(name="plan_mixed", kind="plan", B=509, ctx_lo=0, ctx_hi=8192, new_lo=0, new_hi=256, bs=32, lens=5),
        # One decode step's queries and keys: 64 tokens, grouped heads, three position axes.
        dict(name="rope_decode", kind="rope", T=64, Hq=32, Hkv=8, D=128, axes=3, mix=False, dtype="fp16"),
        # A prefill of 16 K tokens of text and image patches.
        dict(name="rope_prefill", kind="rope", T=16384, Hq=32, Hkv=8, D=128, axes=3, mix=False, dtype="bf16"),
        # A training step's backward pass, two sequences of 4096.
        dict(name="rope_grad", kind="rope_grad", T=8192, Hq=32, Hkv=8, D=128, axes=1, mix=False, dtype="bf16"),
        # The same with an odd token count, odd head counts and interleaved axes.
        dict(name="rope_grad_odd", kind="rope_grad", T=1021, Hq=9, Hkv=3, D=64, axes=3, mix=True, dtype="fp16"),
        # The new token of each of 64 running requests.
        dict(name="append_decode", kind="append", T=64, Hkv=8, D=128, bs=16, dtype="fp16"),
        # A prefill chunk of an odd number of tokens.
        dict(name="append_prefill", kind="append", T=16001, Hkv=8, D=128, bs=64, dtype="bf16"),
        # The smallest call: one request, a 33-token context.
        dict(name="attn_one", kind="attn", B=1, ctx_lo=33, ctx_hi=33, new_lo=1, new_hi=1, Hkv=2, G=4, D=64, bs=16,
             dtype="fp16", lens=0),
        # Decode of 64 requests with contexts U[512, 8192] and grouped heads.
        dict(name="attn_decode", kind="attn", B=64, ctx_lo=512, ctx_hi=8192, new_lo=1, new_hi=1, Hkv=8, G=4, D=128, bs=16,
             dtype="fp16", lens=3),
        # Four long contexts, up to four speculative tokens each, 64 query heads over 8.
        dict(name="attn_long", kind="attn", B=4, ctx_lo=65536, ctx_hi=131072, new_lo=1, new_hi=4, Hkv=8, G=8, D=128, bs=64,
             dtype="bf16", lens=7),
        # A mixed batch with prefill chunks of up to 512 tokens over contexts of up to 4096.
        dict(name="attn_chunk", kind="attn", B=8, ctx_lo=1024, ctx_hi=4096, new_lo=1, new_hi=512, Hkv=8, G=4, D=128, bs=16,
             dtype="bf16", lens=9),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["plan", "rope", "rope_grad", "append", "attn", "attn"])
    dtype = rng.choice(["fp16", "bf16"])
    D = rng.choice([64, 128])
    bs = rng.choice([16, 32, 64])
    if kind == "plan":
        hi = _log_int(rng, 16, 8192)
        return dict(kind=kind, B=_log_int(rng, 1, 500), ctx_lo=rng.randint(0, hi // 2), ctx_hi=hi, new_lo=rng.randint(0, 1),
                    new_hi=_log_int(rng, 1, 256), bs=bs, lens=rng.randint(0, 10 ** 6))
    if kind in ("rope", "rope_grad"):
        hkv = rng.choice([1, 2, 3, 5, 8])
        return dict(kind=kind, T=_log_int(rng, 1, 16384 if kind == "rope" else 8192), Hq=hkv * rng.choice([1, 2, 3, 4]), Hkv=hkv,
                    D=D, axes=rng.choice([1, 2, 3, 4]), mix=rng.random() < 0.5, dtype=dtype)
    if kind == "append":
        return dict(kind=kind, T=_log_int(rng, 1, 16000), Hkv=rng.choice([1, 2, 3, 8]), D=D, bs=bs, dtype=dtype)
    if rng.random() < 0.5:  # decode, a few tokens for each request
        hi = _log_int(rng, 16, 32768)
        most = max(1, min(64, 524288 // hi))
        new = rng.choice([1, 1, 2, 4])
        return dict(kind=kind, B=_log_int(rng, 1, most), ctx_lo=rng.randint(1, hi), ctx_hi=hi, new_lo=1, new_hi=new,
                    Hkv=rng.choice([1, 2, 3, 8]), G=rng.choice([1, 2, 3, 4, 8]), D=D, bs=bs, dtype=dtype,
                    lens=rng.randint(0, 10 ** 6))
    hi = _log_int(rng, 64, 4096)  # chunks of prompts
    return dict(kind=kind, B=rng.randint(1, 8), ctx_lo=rng.randint(1, hi), ctx_hi=hi, new_lo=rng.randint(0, 1),
                new_hi=_log_int(rng, 5, min(hi, 512)), Hkv=rng.choice([1, 2, 3, 8]), G=rng.choice([1, 2, 4]), D=D, bs=bs,
                dtype=dtype, lens=rng.randint(0, 10 ** 6))


def _lengths(case):
    """(context lengths before the step, new tokens) of a plan case; (context lengths with the
    new tokens, new tokens) of an attn case. Fixed by the case."""
    r = random.Random(case["lens"])
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["B"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])]
    new[0] = max(new[0], 1)
    if case["kind"] == "attn":
        ctx = [max(c, n) for c, n in zip(ctx, new)]
    return ctx, new


def _sections(case):
    """Rotary pairs per axis: the first axis gets what the others leave."""
    half, a = case["D"] // 2, case["axes"]
    rest = [3 * half // 8 if a == 3 else half // a] * (a - 1)
    return tuple([half - sum(rest)] + rest)


def _axis_of_pair(case):
    """The position axis of each rotary pair: consecutive sections, or (mix) axis a at pairs
    a, a + axes, ... for as many pairs as it has, and the first axis elsewhere."""
    sec = _sections(case)
    if not case["mix"]:
        return [a for a, n in enumerate(sec) for _ in range(n)]
    out = [0] * (case["D"] // 2)
    for a in range(1, len(sec)):
        for i in range(a, min(len(sec) * sec[a], len(out)), len(sec)):
            out[i] = a
    return out


# --------------------------------------------------------------------------- the cache's layout
def _quantise(x):
    """x [..., D] fp32 -> codes uint8 [..., D], scales and zeros fp16 [..., D / 32]."""
    g = x.unflatten(-1, (x.shape[-1] // GROUP, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) * (1 / 15)).half()
    z = lo.half()
    sf = s.float()
    inv = torch.where(sf > 0, 1.0 / sf, torch.zeros_like(sf))
    c = ((g - z.float().unsqueeze(-1)) * inv.unsqueeze(-1)).round_().clamp_(0, 15).to(torch.uint8)
    return c.flatten(-2), s, z


def _swizzle(D, device):
    """[pair 8][chunk 8] -> the n that the chunk holds."""
    pr = torch.arange(8, device=device)
    x = 2 * (pr % 4) if D == 128 else 4 * (pr // 2 % 2)
    return torch.arange(8, device=device)[None, :] ^ x[:, None]


def _pack(kc, ks, kz, vc, vs, vz):
    """Codes [N, 16, D], scales and zeros [N, 16, D / 32] of K and V -> pieces [N, 20 D] uint8."""
    n, _, D = kc.shape
    w = D // GROUP
    k = kc.view(n, 16, w, 4, 2, 2, 2)  # token, word, lane, half of the bits, nibble, parity
    kb = (k[:, :, :, :, :, 0] | k[:, :, :, :, :, 1] << 4).permute(0, 1, 3, 2, 5, 4).reshape(n, 8 * D)
    v = vc.view(n, 8, 2, w, 8, 2, 2)  # pair, token, group, n, byte, nibble
    vb = (v[..., 0] | v[..., 1] << 4).permute(0, 1, 4, 2, 3, 5).reshape(n, 8, 8, D // 8)
    at = _swizzle(D, kc.device)
    vb = vb[:, torch.arange(8, device=kc.device)[:, None], at].reshape(n, 8 * D)
    u8 = lambda t: t.contiguous().view(n, -1).view(torch.uint8)  # noqa: E731
    return torch.cat([kb, u8(ks), u8(kz), vb, u8(vs), u8(vz.transpose(1, 2))], 1)


def _unpack(p, D):
    """Pieces [N, 20 D] uint8 -> the K and V values [N, 16, D] that they stand for, fp32."""
    n, w = p.shape[0], D // GROUP
    f16 = lambda i: p[:, i:i + D].contiguous().view(torch.float16).float()  # noqa: E731

    def value(codes, s, z):
        return (codes.view(n, 16, w, GROUP).float() * s.unsqueeze(-1) + z.unsqueeze(-1)).view(n, 16, D)

    kb = p[:, :8 * D].reshape(n, 16, 4, w, 2, 2).permute(0, 1, 3, 2, 5, 4)  # token, word, lane, half, parity
    kc = torch.stack([kb & 15, kb >> 4], 5).reshape(n, 16, D)
    k = value(kc, f16(8 * D).view(n, 16, w), f16(9 * D).view(n, 16, w))
    vb = p[:, 10 * D:18 * D].reshape(n, 8, 8, D // 8)
    vb = vb[:, torch.arange(8, device=p.device)[:, None], _swizzle(D, p.device)]
    vb = vb.view(n, 8, 8, 2, w, 2).permute(0, 1, 3, 4, 2, 5)  # pair, token, group, n, byte
    vc = torch.stack([vb & 15, vb >> 4], 6).reshape(n, 16, D)
    v = value(vc, f16(18 * D).view(n, 16, w), f16(19 * D).view(n, w, 16).transpose(1, 2))
    return k, v


# --------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 11)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _angles(rows, D):
    inv = THETA ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    randn = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    if kind == "plan":
        ctx, new = _lengths(case)
        bs = case["bs"]
        width = -(-(case["ctx_hi"] + case["new_hi"]) // bs)
        have = [-(-c // bs) for c in ctx]
        need = [-(-(c + n) // bs) - h for c, n, h in zip(ctx, new, have)]
        pool = torch.randperm(sum(have) + sum(need) + 7, generator=g, device="cuda").int()
        table = torch.full((case["B"], width), -1, dtype=torch.int32, device="cuda")
        used = torch.arange(width, device="cuda")[None, :] < _ints(have)[:, None]
        table[used] = pool[:sum(have)]
        return dict(case=case, table=table, seq_lens=_ints(ctx), n_new=_ints(new), free=pool[sum(have):].clone(), total=sum(new))
    dtype, D = DTYPES[case["dtype"]], case["D"]
    if kind in ("rope", "rope_grad"):
        T, hq, hkv = case["T"], case["Hq"], case["Hkv"]
        rows = 8192
        cos, sin = _angles(rows, D)
        # q and k are parts of one projection's output, as a model has them.
        qkv = randn(T, hq + 2 * hkv, D).to(dtype)
        pos = torch.randint(0, rows, (case["axes"], T), generator=g, device="cuda", dtype=torch.int32)
        st = dict(case=case, q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], wq=(1 + 0.1 * randn(D)).to(dtype), wk=(1 + 0.1 * randn(D)).to(dtype),
                  cos=cos, sin=sin, pos=pos, sections=_sections(case), axis=torch.tensor(_axis_of_pair(case), device="cuda"))
        if kind == "rope_grad":
            st["dq"], st["dk"] = randn(T, hq, D).to(dtype), randn(T, hkv, D).to(dtype)
        return st
    hkv, bs = case["Hkv"], case["bs"]
    gain = 1 + 3 * (torch.rand(hkv, D, generator=g, device="cuda") < 0.05)  # a few strong channels of K
    if kind == "append":
        T = case["T"]
        blocks = -(-T // bs) + 5
        at = torch.arange(T, device="cuda")
        slots = (torch.randperm(blocks, generator=g, device="cuda")[at // bs] * bs + at % bs).int()
        cache = torch.randint(0, 256, (blocks, hkv, bs // PIECE, 20 * D), generator=g, device="cuda", dtype=torch.uint8)
        return dict(case=case, k=(randn(T, hkv, D) * gain).to(dtype), v=randn(T, hkv, D).to(dtype), slots=slots, cache=cache)
    ctx, new = _lengths(case)
    have = [-(-c // bs) for c in ctx]
    blocks, width = sum(have) + 3, max(have)
    table = torch.zeros((case["B"], width), dtype=torch.int32, device="cuda")
    used = torch.arange(width, device="cuda")[None, :] < _ints(have)[:, None]
    table[used] = torch.randperm(blocks, generator=g, device="cuda").int()[:sum(have)]
    shape = (blocks, hkv, bs, D)
    k = _quantise(randn(*shape) * gain[:, None])
    v = _quantise(randn(*shape))
    pieces = lambda t: t.reshape(-1, PIECE, t.shape[-1])  # noqa: E731
    cache = _pack(*map(pieces, k), *map(pieces, v)).view(blocks, hkv, bs // PIECE, 20 * D)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = randn(cu[-1], hkv * case["G"], D).to(dtype)
    return dict(case=case, q=q, cache=cache, table=table, ctx=_ints(ctx), cu=_ints(cu), most=max(new))


# --------------------------------------------------------------------------- plain forms
def _plan_plain(st):
    table, L, n, free, bs = st["table"], st["seq_lens"].long(), st["n_new"].long(), st["free"], st["case"]["bs"]
    have, want = (L + bs - 1) // bs, (L + n + bs - 1) // bs
    fits = want <= table.shape[1]
    need = torch.where(fits, want - have, 0)
    end = need.cumsum(0)
    off = end - need
    ok = fits & ((need == 0) | (end <= free.shape[0]))
    cu = torch.cat([n.new_zeros(1), n.cumsum(0)])
    i = torch.arange(st["total"], device=table.device)
    b = torch.searchsorted(cu, i, right=True) - 1
    pos = L[b] + i - cu[b]
    j = pos // bs
    fresh = j >= have[b]
    at = (off[b] + j - have[b]).clamp(0, max(free.shape[0] - 1, 0))
    block = torch.where(fresh, free[at], table[b, j.clamp(max=table.shape[1] - 1)]).long()
    slots = torch.where(ok[b], block * bs + pos % bs, -1)
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    new = (col >= have[:, None]) & (col < want[:, None]) & ok[:, None]
    at = (off[:, None] + col - have[:, None]).clamp(0, max(free.shape[0] - 1, 0))
    table.copy_(torch.where(new, free[at], table))
    return [slots.int(), pos.int(), cu.int(), torch.where(ok, L + n, L).int(), torch.where(ok, need, 0).sum().int().view(1), table]


def _cos_sin(st):
    row = st["pos"].long()[st["axis"]].T  # [T, D / 2]
    i = torch.arange(row.shape[1], device=row.device)
    return st["cos"][row, i][:, None], st["sin"][row, i][:, None]


def _rope_plain(st, x, w):
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    c, s = _cos_sin(st)
    a, b = y.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _rope_grad_plain(st, dz, x, w):
    x, dz = x.float(), dz.float()
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    c, s = _cos_sin(st)
    a, b = dz.chunk(2, -1)
    dy = torch.cat([a * c + b * s, b * c - a * s], -1)
    g = dy * w.float()
    dx = r * (g - x * (r * r * (g * x).mean(-1, keepdim=True)))
    return dx.to(st["q"].dtype), (dy * x * r).sum((0, 1)).to(w.dtype)


def _append_plain(st):
    case, cache = st["case"], st["cache"]
    D, hkv, bs = case["D"], case["Hkv"], case["bs"]
    slot = st["slots"].long()
    block, piece, tok = slot // bs, slot % bs // PIECE, slot % PIECE
    w, T = D // GROUP, slot.shape[0]
    kc, ks, kz = _quantise(st["k"].float())
    vc, vs, vz = _quantise(st["v"].float())
    k = kc.view(T, hkv, w, 4, 2, 2, 2)
    kb = (k[..., 0, :] | k[..., 1, :] << 4).permute(0, 1, 3, 2, 5, 4).reshape(T, hkv, D // 2)
    v = vc.view(T, hkv, w, 8, 2, 2)
    vb = (v[..., 0] | v[..., 1] << 4).permute(0, 1, 3, 2, 4).reshape(T, hkv, 8, D // 16)
    h = torch.arange(hkv, device=slot.device)[None, :, None]
    at = lambda t: t[:, None, None]  # noqa: E731
    span = lambda n: torch.arange(n, device=slot.device)[None, None]  # noqa: E731
    u8 = lambda t: t.contiguous().view(torch.uint8)  # noqa: E731

    def put(where, what):
        cache[at(block), h, at(piece), where] = what

    put(at(tok) * (D // 2) + span(D // 2), kb)
    put(8 * D + at(tok) * 2 * w + span(2 * w), u8(ks))
    put(9 * D + at(tok) * 2 * w + span(2 * w), u8(kz))
    chunk = torch.arange(8, device=slot.device)[None] ^ (2 * (tok // 2 % 4) if D == 128 else 4 * (tok // 4 % 2))[:, None]
    where = (tok // 2 * D + tok % 2 * (D // 16))[:, None, None] + chunk[:, :, None] * (D // 8) + span(D // 16)
    put(10 * D + where.reshape(T, 1, D // 2), vb.reshape(T, hkv, D // 2))
    put(18 * D + at(tok) * 2 * w + span(2 * w), u8(vs))
    put(19 * D + (span(w)[..., None] * 32 + tok[:, None, None, None] * 2 + span(2)[:, :, None]).reshape(T, 1, 2 * w), u8(vz))
    value = lambda c, s, z: (c.unflatten(-1, (w, GROUP)).float() * s.float().unsqueeze(-1) + z.float().unsqueeze(-1)).flatten(-2)  # noqa: E731
    return [value(kc, ks, kz).to(st["k"].dtype), value(vc, vs, vz).to(st["v"].dtype)]


def _attn_plain(st):
    case, q = st["case"], st["q"]
    D, hkv, G, bs, B = case["D"], case["Hkv"], case["G"], case["bs"], case["B"]
    table, ctx, cu, most = st["table"].long(), st["ctx"].long(), st["cu"].long(), st["most"]
    width = table.shape[1]
    k, v = _unpack(st["cache"][table].reshape(-1, 20 * D), D)  # [B, width, Hkv, bs / 16] pieces
    rows = lambda t: t.view(B, width, hkv, bs, D).transpose(1, 2).reshape(B, hkv, width * bs, D)  # noqa: E731
    k, v = rows(k), rows(v)
    i = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(cu, i, right=True) - 1
    s = i - cu[b]
    qp = q.new_zeros((B, most, hkv * G, D), dtype=torch.float32)
    qp[b, s] = q.float()
    qp = qp.view(B, most, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * most, D)
    sc = (qp @ k.transpose(-1, -2)).mul_(D ** -0.5).view(B, hkv, G, most, -1)
    del k
    pos = (ctx - (cu[1:] - cu[:-1]))[:, None] + torch.arange(most, device=q.device)  # [B, most]
    hide = torch.arange(width * bs, device=q.device)[None, None] > pos[:, :, None]
    sc.masked_fill_(hide[:, None, None], float("-inf"))
    sc.sub_(sc.amax(-1, keepdim=True)).exp_()
    total = sc.sum(-1, keepdim=True)
    v = torch.where((torch.arange(width * bs, device=q.device)[None] < ctx[:, None])[:, None, :, None], v, 0.0)
    o = (sc.view(B, hkv, G * most, -1) @ v).view(B, hkv, G, most, D) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B, most, hkv * G, D)[b, s].to(q.dtype)


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        if kind == "plan":
            return _plan_plain(state)
        if kind == "rope":
            return [_rope_plain(state, state[x], state["w" + x]).to(state[x].dtype) for x in ("q", "k")]
        if kind == "rope_grad":
            (dq, dwq), (dk, dwk) = (_rope_grad_plain(state, state["d" + x], state[x], state["w" + x]) for x in ("q", "k"))
            return [dq, dk, dwq, dwk]
        return _append_plain(state) if kind == "append" else [_attn_plain(state)]
    if kind == "plan":
        from tritonllmcompiler_b200.ops.paged_plan import paged_plan

        p = paged_plan(state["table"], state["seq_lens"], state["n_new"], state["free"], block_size=case["bs"],
                       max_tokens=state["total"])
        return [p.slots, p.positions, p.cu_seqlens, p.new_lens, p.taken, state["table"]]
    if kind in ("rope", "rope_grad"):
        from tritonllmcompiler_b200.ops.qk_norm_rope import qk_norm_rope, qk_norm_rope_backward

        args = (state["q"], state["k"], state["wq"], state["wk"], state["cos"], state["sin"], state["pos"])
        how = dict(sections=state["sections"], interleaved=case["mix"], eps=EPS)
        if kind == "rope":
            return list(qk_norm_rope(*args, **how))
        return list(qk_norm_rope_backward(state["dq"], state["dk"], *args, **how))
    from tritonllmcompiler_b200.ops.paged_kv4 import paged_attention_kv4, paged_kv4_append, paged_kv4_gather

    if kind == "append":
        paged_kv4_append(state["k"], state["v"], state["cache"], state["slots"], block_size=case["bs"])
        return list(paged_kv4_gather(state["cache"], state["slots"], block_size=case["bs"], dtype=state["k"].dtype))
    return [paged_attention_kv4(state["q"], state["cache"], state["table"], state["ctx"], state["cu"], state["most"],
                                block_size=case["bs"])]


# --------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "plan":
        ctx, new = _lengths(case)
        bs, T = case["bs"], sum(new)
        fresh = sum(-(-(c + n) // bs) - -(-c // bs) for c, n in zip(ctx, new))
        # lengths in and out, cumulative counts, a table entry for each open block, new blocks in and out, slots, positions
        return {"bytes": 4 * (4 * case["B"] + 2 + case["B"] + 2 * fresh + 2 * T), "flops": 0}
    D = case["D"]
    if kind in ("rope", "rope_grad"):
        T, heads = case["T"], case["Hq"] + case["Hkv"]
        small = 4 * case["axes"] * T + 4 * D * min(T, 8192) + 4 * D  # positions, cos and sin rows, weights
        n = T * heads * D
        return {"bytes": (2 if kind == "rope" else 3) * 2 * n + small, "flops": (10 if kind == "rope" else 20) * n}
    if kind == "append":
        n = 2 * case["T"] * case["Hkv"] * D  # K and V elements: read, written and read in 4 bits, written as values
        return {"bytes": 2 * n + 2 * n * 5 // 8 + 2 * n + 8 * case["T"], "flops": 10 * n}
    ctx, new = _lengths(case)
    hq = case["Hkv"] * case["G"]
    pairs = sum(n * c - n * (n - 1) // 2 for c, n in zip(ctx, new))
    cache = sum(c for c, n in zip(ctx, new) if n) * case["Hkv"] * D * 5 // 4
    table = 4 * sum(-(-c // case["bs"]) for c in ctx)
    return {"bytes": cache + 2 * 2 * sum(new) * hq * D + table + 8 * case["B"] + 4, "flops": 4 * hq * D * pairs}


# --------------------------------------------------------------------------- the same in 64 bits
def _exact_value(x):
    """The values of x [..., D] after 4 bits, in 64 bits (scales and zeros are held in fp16)."""
    g = x.double().reshape(*x.shape[:-1], -1, GROUP)
    lo = g.min(-1, keepdim=True).values
    s = ((g.max(-1, keepdim=True).values - lo) / 15).to(torch.float16).double()
    z = lo.to(torch.float16).double()
    c = torch.where(s > 0, (g - z) / s, torch.zeros_like(g)).round().clamp(0, 15)
    return (c * s + z).reshape(x.shape)


def _exact_rows(cache, blocks, h, D):
    """K and V of head h in `blocks` [n], token by token, in 64 bits: by the place of each code."""
    p = cache[blocks, h].reshape(-1, 20 * D)
    dev, w = p.device, D // GROUP
    t = torch.arange(PIECE, device=dev)[:, None]
    d = torch.arange(D, device=dev)[None]
    j, lane = d % 8, d // 8 % 4
    bit = 4 * (j // 2) + 16 * (j % 2)
    kat = t * (D // 2) + 4 * (lane * w + d // 32) + bit // 8
    n, jv = d % 32 // 4, d % 4
    pair = t // 2
    chunk = n ^ (2 * (pair % 4) if D == 128 else 4 * (pair // 2 % 2))
    vat = 10 * D + pair * D + chunk * (D // 8) + t % 2 * (D // 16) + 2 * (d // 32) + jv // 2
    half = lambda at: p[:, at:at + D].contiguous().view(torch.float16).double()  # noqa: E731
    grp = (d // 32).expand(PIECE, D)
    tok = t.expand(PIECE, D)
    k = ((p[:, kat] >> (bit % 8 + 0 * t).to(torch.uint8)) & 15).double()
    k = k * half(8 * D)[:, tok * w + grp] + half(9 * D)[:, tok * w + grp]
    v = ((p[:, vat] >> (4 * (jv % 2) + 0 * t).to(torch.uint8)) & 15).double()
    v = v * half(18 * D)[:, tok * w + grp] + half(19 * D)[:, grp * PIECE + tok]
    return k.reshape(-1, D), v.reshape(-1, D)


def exact(case, seed):
    kind = case["kind"]
    if kind == "plan":
        return None
    st = prepare(case, seed)
    if kind == "append":
        return [_exact_value(st["k"]), _exact_value(st["v"])]
    if kind in ("rope", "rope_grad"):
        half = case["D"] // 2
        axis = torch.tensor(_axis_of_pair(case), device="cuda")
        row = st["pos"].long().index_select(0, axis).transpose(0, 1).unsqueeze(1)  # [T, 1, D / 2]
        turn = torch.complex(st["cos"].double(), st["sin"].double())
        turn = torch.stack([turn[row[:, 0, i], i] for i in range(half)], -1).unsqueeze(1)
        back, weights = [], []
        for x, w in (("q", "wq"), ("k", "wk")):
            u, wt = st[x].double(), st[w].double()
            norm = (u.pow(2).sum(-1, keepdim=True) / case["D"] + EPS).sqrt()
            if kind == "rope":
                y = u / norm * wt
                z = torch.complex(y[..., :half], y[..., half:]) * turn
                back.append(torch.cat([z.real, z.imag], -1))
                continue
            dz = st["d" + x].double()
            dy = torch.complex(dz[..., :half], dz[..., half:]) * turn.conj()
            dy = torch.cat([dy.real, dy.imag], -1)
            hat = u / norm
            weights.append((dy * hat).sum(0).sum(0))
            e = dy * wt
            back.append((e - hat * (e * hat).mean(-1, keepdim=True)) / norm)
        return back + weights
    ctx, new = _lengths(case)
    D, G = case["D"], case["G"]
    out = torch.empty(st["q"].shape, dtype=torch.float64, device="cuda")
    row = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        if n == 0:
            continue
        blocks = st["table"][b, :-(-c // case["bs"])].long()
        for h in range(case["Hkv"]):
            k, v = (x[:c] for x in _exact_rows(st["cache"], blocks, h, D))
            q = st["q"][row:row + n, h * G:(h + 1) * G].double()
            x = torch.einsum("sgd,td->sgt", q, k) / math.sqrt(D)
            seen = torch.arange(c, device="cuda")[None] <= (c - n + torch.arange(n, device="cuda"))[:, None]
            p = torch.softmax(x.masked_fill(~seen[:, None], -math.inf), -1)
            out[row:row + n, h * G:(h + 1) * G] = torch.einsum("sgt,td->sgd", p, v)
        row += n
    return [out]
