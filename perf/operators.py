"""Measured cases of the quantised decode operators: linears with 4-bit weights, the append to an
8-bit KV cache, and attention over that cache.

``run`` with ``own`` false computes each operator in a plain form (elementary torch operations
in fp32); with ``own`` true it makes the calls a user of neokernel_b200 makes.

The operators:

* ``w4``: ``y[m, n] = sum_k x[m, k] (q[n, k] - z[n, k // g]) s[n, k // g]``, x bf16 [M, K], q
  4-bit codes [N, K] packed two to a byte (even k in the low half), s bf16 or fp16, z 4-bit zero
  points (8 where there are none); the sum rounded once to bf16.
* ``append``: the rows ``[q heads | k heads | v heads]`` of T new tokens per sequence; q and k
  heads get RMSNorm and RoPE with the decode step's bf16 cast points, k and v are stored as e4m3
  codes times a power of two held for each (sequence, kv head, block of tokens). A block's scale is the
  smallest power of two ``s >= 2^-64`` with ``amax <= 448 s`` over its new tokens, and at least its
  former scale where it holds earlier tokens, whose codes are rounded anew when the scale rises.
* ``attention``: T new query tokens per sequence over that cache; token t of sequence b sees
  slots 0..position[b] + t of it, and a sequence with a negative position is idle (zeros).
"""

import math

import torch

own = False

HEAD_DIM = 128
EPS = 1e-6


def listed():
    return [
        # one token through the smallest decode linear of the 0.6B shape: all latency
        {"name": "w4_m1_o_proj", "op": "w4", "M": 1, "K": 2048, "N": 1024, "group": 128,
         "zeros": False, "scale": "bf16"},
        # one token through the widest layer linear of the 8B shape: a weight stream
        {"name": "w4_m1_gate_up", "op": "w4", "M": 1, "K": 4096, "N": 24576, "group": 128,
         "zeros": False, "scale": "bf16"},
        # a full decode batch through the 8B QKV linear
        {"name": "w4_m16_qkv", "op": "w4", "M": 16, "K": 4096, "N": 6144, "group": 64,
         "zeros": False, "scale": "bf16"},
        # half a batch through the 8B down projection: long K, small groups with zero points
        {"name": "w4_m8_down", "op": "w4", "M": 8, "K": 12288, "N": 4096, "group": 32,
         "zeros": True, "scale": "fp16"},
        # sizes that fit no tile: an odd K whose last group is short, an odd N
        {"name": "w4_m5_odd", "op": "w4", "M": 5, "K": 2477, "N": 1003, "group": 64,
         "zeros": True, "scale": "bf16"},
        # a draft of 64 tokens verified at once through the 8B gate_up
        {"name": "w4_m64_gate_up", "op": "w4", "M": 64, "K": 4096, "N": 24576, "group": 128,
         "zeros": True, "scale": "bf16"},
        # one sequence's next token into the cache of one layer
        {"name": "append_b1", "op": "append", "B": 1, "T": 1, "heads": 32, "kv_heads": 8,
         "S": 1024, "block": 64, "layout": "bhsd"},
        # drafts of 16 tokens for 16 sequences, crossing block ends, 32B head counts
        {"name": "append_b16_t16", "op": "append", "B": 16, "T": 16, "heads": 64, "kv_heads": 8,
         "S": 1024, "block": 32, "layout": "bshd"},
        # one sequence at the decode benchmark's cache length
        {"name": "attn_b1_1k", "op": "attention", "B": 1, "T": 1, "heads": 32, "kv_heads": 8,
         "S": 1024, "block": 64, "layout": "bhsd", "ragged": False},
        # a served batch: lengths from zero (an idle slot) to 8192
        {"name": "attn_b16_8k_ragged", "op": "attention", "B": 16, "T": 1, "heads": 32,
         "kv_heads": 8, "S": 8192, "block": 64, "layout": "bhsd", "ragged": True},
        # short drafts being verified over caches of odd lengths, tokens-major layout
        {"name": "attn_b5_t4_odd", "op": "attention", "B": 5, "T": 4, "heads": 64, "kv_heads": 8,
         "S": 2999, "block": 16, "layout": "bshd", "ragged": True},
        # two long documents
        {"name": "attn_b2_128k", "op": "attention", "B": 2, "T": 1, "heads": 64, "kv_heads": 8,
         "S": 131072, "block": 128, "layout": "bhsd", "ragged": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["w4", "w4", "append", "attention", "attention"])
    if op == "w4":
        c = {"op": op, "M": _log(rng, 1, 64), "K": _log(rng, 256, 25600), "N": _log(rng, 256, 32768),
             "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
             "scale": rng.choice(["bf16", "fp16"])}
        c["N"] = max(1, min(c["N"], 4096 * 24576 // c["K"]))
        if rng.random() < 0.6:  # most models' widths are whole groups
            c["K"], c["N"] = max(128, c["K"] // 128 * 128), max(16, c["N"] // 16 * 16)
        return c
    heads, kv_heads = rng.choice([(16, 8), (32, 8), (64, 8), (8, 8), (8, 2), (4, 1), (28, 4), (5, 1)])
    c = {"op": op, "B": _log(rng, 1, 32), "T": rng.choice([1, 1, 1, 2, 3, 5, 8, 16]),
         "heads": heads, "kv_heads": kv_heads, "block": rng.choice([16, 32, 64, 128]),
         "layout": rng.choice(["bhsd", "bshd"])}
    if op == "append":
        c["S"] = _log(rng, 32, 2048)
        return c
    c["S"] = min(_log(rng, 16, 131072), 2 * 8 * 131072 // (c["B"] * kv_heads))
    c["T"] = min(c["T"], 8)
    c["ragged"] = rng.random() < 0.6
    return c


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _codes(gen, *shape):
    """e4m3 codes as a cache holds them: each block's largest value near the top of the range."""
    t = torch.empty(shape, device="cuda", dtype=torch.uint8)
    for part in t.view(-1).split(1 << 26):  # bounded fp32 scratch
        part.copy_(_randn(gen, part.numel()).mul_(80.0).clamp_(-448.0, 448.0)
                   .to(torch.float8_e4m3fn).view(torch.uint8))
    return t


def _scales(gen, lo, hi, *shape):
    return torch.exp2(torch.randint(lo, hi, shape, generator=gen, device="cuda").float())


def _cache(case, gen, lo, hi):
    B, H, S = case["B"], case["kv_heads"], case["S"]
    st = {}
    for n in ("k", "v"):
        if case["layout"] == "bhsd":
            st[n] = _codes(gen, B, H, S, HEAD_DIM)
        else:  # tokens-major storage seen as [B, H, S, 128]
            st[n] = _codes(gen, B, S, H, HEAD_DIM).transpose(1, 2)
        st[n + "_scale"] = _scales(gen, lo, hi, B, H, -(-S // case["block"]))
    if own:
        from neokernel_b200 import decode_ops
        st["cache"] = decode_ops.Q8Cache(st["k"].view(torch.float8_e4m3fn),
                                         st["v"].view(torch.float8_e4m3fn), st["k_scale"],
                                         st["v_scale"], case["block"])
    return st


def _positions(case, gen):
    """Slot of the first new token of each sequence; totals do not depend on the seed."""
    B, room = case["B"], case["S"] - case["T"]
    if not case["ragged"]:
        return torch.full((B,), room, device="cuda", dtype=torch.int64)
    p = torch.tensor([room * (b + 1) // B for b in range(B)], device="cuda")
    if B >= 4:
        p[0] = -1  # an idle slot of the batch
    return p[torch.randperm(B, generator=gen, device="cuda")].contiguous()


def prepare(case, seed):
    gen = _gen(seed)
    st = {"case": case}
    if case["op"] == "w4":
        M, K, N, g = case["M"], case["K"], case["N"], case["group"]
        groups = -(-K // g)
        st["x"] = _randn(gen, M, K).to(torch.bfloat16)
        q = torch.randint(0, 256, (N, -(-K // 2)), generator=gen, device="cuda", dtype=torch.uint8)
        if K % 2:
            q[:, -1] &= 15
        # weights of standard deviation near 0.02, as the framework's own
        s = (0.002 + 0.004 * torch.rand(N, groups, generator=gen, device="cuda"))
        st["q"] = q
        st["s"] = s.to(torch.bfloat16 if case["scale"] == "bf16" else torch.float16)
        st["z"] = (torch.randint(4, 12, (N, groups), generator=gen, device="cuda",
                                 dtype=torch.uint8) if case["zeros"] else None)
        st["out"] = torch.empty(M, N, device="cuda", dtype=torch.bfloat16)
        if own:
            import neokernel_b200 as nk
            st["w"] = nk.W4Weight.pack(q, st["s"], st["z"], K=K, group=g)
        return st
    B, T, H, Hkv = case["B"], case["T"], case["heads"], case["kv_heads"]
    st["case"] = case
    if case["op"] == "append":
        S = case["S"]
        st.update(_cache(case, gen, -9, -5))
        st["qkv"] = _randn(gen, B * T, (H + 2 * Hkv) * HEAD_DIM).to(torch.bfloat16)
        for n in ("qn", "kn"):
            st[n] = (0.5 + torch.rand(HEAD_DIM, generator=gen, device="cuda")).to(torch.bfloat16)
        inv = 1.0 / (1e6 ** (torch.arange(0, HEAD_DIM, 2, device="cuda").double() / HEAD_DIM))
        ang = torch.outer(torch.arange(S, device="cuda").double(), inv)
        ang = torch.cat((ang, ang), dim=-1)
        st["cos"], st["sin"] = ang.cos().to(torch.bfloat16), ang.sin().to(torch.bfloat16)
        st["pos"] = torch.randint(0, S - T + 1, (B,), generator=gen, device="cuda")
        st["q_out"] = torch.empty(B * T, H * HEAD_DIM, device="cuda", dtype=torch.bfloat16)
        return st
    st.update(_cache(case, gen, -8, -4))
    st["q"] = _randn(gen, B * T, H * HEAD_DIM).to(torch.bfloat16)
    st["pos"] = _positions(case, gen)
    st["out"] = torch.empty_like(st["q"])
    if own:
        from neokernel_b200 import decode_ops
        st["ws"] = decode_ops.attention_q8_workspace(st["cache"], H, T)
    return st


# ------------------------------------------------------------------------------------------
# plain forms
# ------------------------------------------------------------------------------------------
def _unpack(q, K):
    return torch.stack((q & 15, q >> 4), dim=-1).flatten(1)[:, :K]


def _plain_w4(st):
    c = st["case"]
    K, g = c["K"], c["group"]
    w = _unpack(st["q"], K).float()
    group = torch.arange(K, device=w.device) // g
    w = w - (8.0 if st["z"] is None else st["z"].float()[:, group])
    w = w * st["s"].float()[:, group]
    return torch.mm(st["x"].float(), w.t()).to(torch.bfloat16)


def _pow2_scale(amax):
    """Smallest power of two s >= 2^-64 with amax <= 448 s (0 for 0): 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    s = torch.exp2((e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-64).double()).float()
    return torch.where(amax > 0, s, torch.zeros_like(s))


def _norm_rope(x, gain, cos, sin):
    """x [B, T, h, 128] fp64 of bf16 values -> RMSNorm and RoPE, each step rounded to bf16.

    In 64 bits between the roundings, as a value next to a bf16 border moves its e4m3 code."""
    r = lambda v: v.to(torch.bfloat16).double()  # noqa: E731
    x = r(r(x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)) * gain)
    half = HEAD_DIM // 2
    rot = torch.cat((-x[..., half:], x[..., :half]), dim=-1)
    return r(r(x * cos) + r(rot * sin))


def _plain_append(st):
    c = st["case"]
    B, T, H, Hkv, S, block = (c[n] for n in ("B", "T", "heads", "kv_heads", "S", "block"))
    pos = st["pos"]
    rows = st["qkv"].view(B, T, H + 2 * Hkv, HEAD_DIM).double()
    at = pos[:, None] + torch.arange(T, device=pos.device)  # [B, T] slots of the new tokens
    cos = st["cos"][at].double()[:, :, None]
    sin = st["sin"][at].double()[:, :, None]
    st["q_out"].copy_(_norm_rope(rows[:, :, :H], st["qn"].double(), cos, sin).view(B * T, -1))
    new = {"k": _norm_rope(rows[:, :, H:H + Hkv], st["kn"].double(), cos, sin),
           "v": rows[:, :, H + Hkv:]}
    # the window of whole blocks that the new tokens touch
    nb = (T + block - 2) // block + 1
    first = pos // block
    slot = first[:, None] * block + torch.arange(nb * block, device=pos.device)  # [B, W]
    blk = first[:, None] + torch.arange(nb, device=pos.device)
    there = slot < S
    earlier = (slot < pos[:, None])[:, None, :, None]
    fresh = ((slot >= pos[:, None]) & (slot < pos[:, None] + T))[:, None, :, None]
    tok = (slot - pos[:, None]).clamp(0, T - 1)
    slot_in, blk_in = slot.clamp(max=S - 1), blk.clamp(max=st["k_scale"].shape[2] - 1)
    b, h = torch.arange(B, device=pos.device), torch.arange(Hkv, device=pos.device)
    bb, hh = b[:, None, None], h[None, :, None]
    for n in ("k", "v"):
        codes, scale = st[n], st[n + "_scale"]
        old = codes[bb, hh, slot_in[:, None]]                                   # [B, Hkv, W, 128]
        s_old = scale[bb, hh, blk_in[:, None]]                                  # [B, Hkv, nb]
        x = new[n][bb, tok[:, None], hh].float()                                # [B, Hkv, W, 128]
        amax = torch.where(fresh, x.abs(), torch.zeros_like(x)).view(B, Hkv, nb, -1).amax(-1)
        kept = torch.where((pos % block > 0)[:, None, None]
                           & (torch.arange(nb, device=pos.device) == 0), s_old,
                           torch.zeros_like(s_old))
        s_new = torch.maximum(kept, _pow2_scale(amax))
        wide = lambda s: s.repeat_interleave(block, dim=2)[..., None]  # noqa: E731
        div = torch.where(wide(s_new) > 0, wide(s_new), torch.ones_like(wide(s_new)))
        was = old.view(torch.float8_e4m3fn).float() * (wide(s_old) / div)
        want = torch.where(earlier, was, x / div)
        want = want.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
        want = torch.where(earlier | fresh, want, old)
        bi, wi = torch.nonzero(there, as_tuple=True)
        codes[bi, :, slot[bi, wi]] = want.transpose(1, 2)[bi, wi]
        touched = blk * block < pos[:, None] + T
        bi, ji = torch.nonzero(touched, as_tuple=True)
        scale[bi, :, blk[bi, ji]] = s_new.transpose(1, 2)[bi, ji]
    return _append_out(st)


def _append_out(st):
    return {"q": st["q_out"], "k": st["k"].view(torch.float8_e4m3fn),
            "v": st["v"].view(torch.float8_e4m3fn), "k_scale": st["k_scale"],
            "v_scale": st["v_scale"]}


def _dequant(codes, scale, block):
    s = scale.repeat_interleave(block, dim=2)[:, :, :codes.shape[2], None]
    return codes.view(torch.float8_e4m3fn).float() * s


def _plain_attention(st):
    c = st["case"]
    B, T, H, Hkv, S, block = (c[n] for n in ("B", "T", "heads", "kv_heads", "S", "block"))
    G = H // Hkv
    q = st["q"].view(B, T, Hkv, G, HEAD_DIM).float().permute(0, 2, 1, 3, 4).reshape(
        B, Hkv, T * G, HEAD_DIM)
    scores = torch.matmul(q, _dequant(st["k"], st["k_scale"], block).transpose(-1, -2))
    scores = scores * (1.0 / math.sqrt(HEAD_DIM))
    last = st["pos"][:, None] + torch.arange(T, device=q.device)               # [B, T]
    last = torch.where(st["pos"][:, None] < 0, torch.full_like(last, -1), last)
    seen = torch.arange(S, device=q.device) <= last.repeat_interleave(G, dim=1)[:, None, :, None]
    scores = torch.where(seen, scores, torch.full_like(scores, float("-inf")))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top.isinf(), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, _dequant(st["v"], st["v_scale"], block))
    out = out / torch.where(total > 0, total, torch.ones_like(total))
    out = out.view(B, Hkv, T, G, HEAD_DIM).permute(0, 2, 1, 3, 4).reshape(B * T, -1)
    return out.to(torch.bfloat16)


def run(state):
    c = state["case"]
    if own:
        from neokernel_b200 import decode_ops as ops
        import neokernel_b200 as nk
        if c["op"] == "w4":
            return nk.mm_w4(state["x"], state["w"], out=state["out"])
        if c["op"] == "append":
            ops.qk_norm_rope_cache_q8(state["qkv"], state["qn"], state["kn"], state["cos"],
                                      state["sin"], state["pos"], state["q_out"], state["cache"],
                                      c["heads"], EPS)
            return _append_out(state)
        return ops.attention_decode_q8(state["q"], state["cache"], state["pos"], state["out"],
                                       state["ws"], c["heads"])
    if c["op"] == "w4":
        return _plain_w4(state)
    if c["op"] == "append":
        return _plain_append(state)
    return _plain_attention(state)


# ------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------
def _round_e4m3(x):
    """Nearest e4m3 value, ties to even: 3 mantissa bits, least exponent -6."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "w4":
        x, q, s = st["x"].double(), st["q"], st["s"].double()
        K, g = case["K"], case["group"]
        y = torch.zeros(case["M"], case["N"], device="cuda", dtype=torch.float64)
        low, high = (q & 15).double(), (q >> 4).double()
        for j in range(s.shape[1]):  # one group at a time
            k0, k1 = j * g, min(K, j * g + g)
            z = 8.0 if st["z"] is None else st["z"][:, j:j + 1].double()
            n = (k1 - k0 + 1) // 2
            part = x[:, k0:k1:2] @ (low[:, k0 // 2:k0 // 2 + n] - z).t()
            part = part + x[:, k0 + 1:k1:2] @ (high[:, k0 // 2:k0 // 2 + (k1 - k0) // 2] - z).t()
            y += part * s[:, j]
        return y
    B, T, H, Hkv, S, block = (case[n] for n in ("B", "T", "heads", "kv_heads", "S", "block"))
    pos = st["pos"].tolist()
    if case["op"] == "attention":
        out = torch.zeros(B, T, H, HEAD_DIM, device="cuda", dtype=torch.float64)
        q = st["q"].view(B, T, H, HEAD_DIM).double()
        for b in range(B):
            if pos[b] < 0:
                continue
            for h in range(Hkv):
                n = pos[b] + T
                of = torch.arange(n, device="cuda") // block
                k, v = (st[m][b, h, :n].contiguous().view(torch.float8_e4m3fn).double()
                        * st[m + "_scale"][b, h].double()[of][:, None] for m in ("k", "v"))
                heads = slice(h * (H // Hkv), (h + 1) * (H // Hkv))
                for t in range(T):
                    m = pos[b] + t + 1
                    w = torch.softmax(q[b, t, heads] @ k[:m].t() / math.sqrt(HEAD_DIM), dim=-1)
                    out[b, t, heads] = w @ v[:m]
        return out.view(B * T, -1)
    # append: the stored values, sequence by sequence, head by head
    rows = st["qkv"].view(B, T, H + 2 * Hkv, HEAD_DIM).double()
    bf = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    at = (st["pos"][:, None] + torch.arange(T, device="cuda")).view(B, T, 1)
    cos, sin = (st[n].double()[at] for n in ("cos", "sin"))

    def rotated(x, gain):
        n = bf(bf(x / torch.sqrt(x.square().sum(-1, keepdim=True) / HEAD_DIM + EPS)) * gain.double())
        lo, hi = n.chunk(2, dim=-1)
        c0, c1 = cos.chunk(2, dim=-1)
        s0, s1 = sin.chunk(2, dim=-1)
        return torch.cat((bf(bf(lo * c0) - bf(hi * s0)), bf(bf(hi * c1) + bf(lo * s1))), dim=-1)

    res = {"q": rotated(rows[:, :, :H], st["qn"]).view(B * T, -1)}
    new = {"k": rotated(rows[:, :, H:H + Hkv], st["kn"]), "v": rows[:, :, H + Hkv:]}
    for n in ("k", "v"):
        vals = st[n].contiguous().view(torch.float8_e4m3fn).double()
        scale = st[n + "_scale"].double()
        for b in range(B):
            for j in range(pos[b] // block, (pos[b] + T - 1) // block + 1):
                lo, hi = max(pos[b], j * block), min(pos[b] + T, (j + 1) * block)
                x = new[n][b, lo - pos[b]:hi - pos[b]].transpose(0, 1)       # [Hkv, n, 128]
                need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448.0)).clamp(min=-64))
                kept = lo > j * block
                s = torch.maximum(need, scale[b, :, j]) if kept else need
                if kept:
                    before = slice(j * block, lo)
                    ratio = (scale[b, :, j] / s)[:, None, None]
                    vals[b, :, before] = _round_e4m3(vals[b, :, before] * ratio)
                vals[b, :, lo:hi] = _round_e4m3(x / s[:, None, None])
                scale[b, :, j] = s
        res[n], res[n + "_scale"] = vals, scale
    return res


def work(case):
    if case["op"] == "w4":
        M, K, N = case["M"], case["K"], case["N"]
        groups = -(-K // case["group"])
        b = N * -(-K // 2) + N * groups * (3 if case["zeros"] else 2) + 2 * M * K + 2 * M * N
        return {"bytes": b, "flops": 2 * M * N * K}
    B, T, H, Hkv, S = (case[n] for n in ("B", "T", "heads", "kv_heads", "S"))
    if case["op"] == "append":
        # the rows, the tables' rows, q out, the new codes and their scales (codes of earlier
        # tokens move only when a scale rises, and are left out)
        b = B * T * (2 * (2 * H + 2 * Hkv) * HEAD_DIM + 2 * 2 * HEAD_DIM + 2 * Hkv * HEAD_DIM)
        return {"bytes": b + 2 * B * Hkv * 4, "flops": 10 * B * T * (H + Hkv) * HEAD_DIM}
    if case["ragged"]:
        pos = [(S - T) * (b + 1) // B for b in range(B)][1 if B >= 4 else 0:]
    else:
        pos = [S - T] * B
    slots = sum(p + T for p in pos)
    blocks = sum(-(-(p + T) // case["block"]) for p in pos)
    b = Hkv * (slots * 2 * HEAD_DIM + blocks * 2 * 4) + 2 * 2 * B * T * H * HEAD_DIM
    return {"bytes": b, "flops": 4 * H * HEAD_DIM * sum(T * p + T * (T + 1) // 2 for p in pos)}
