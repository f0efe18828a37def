"""The 8-bit KV cache (neokernel_b200.decode_ops: Q8Cache, qk_norm_rope_cache_q8,
attention_decode_q8) against plain implementations in 64 bits."""

import math

import pytest
import torch

import neokernel_b200 as nk
from neokernel_b200 import _lib, decode_ops as ops, qwen3

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rand(*shape, std=1.0, seed=0):
    return (torch.randn(shape, generator=gen(seed), device=DEV) * std).to(torch.bfloat16)


def filled_cache(B, H, S, block, layout="bhsd", seed=0, lo=-9, hi=-4):
    c = ops.Q8Cache.empty(B, H, S, DEV, block=block, layout=layout)
    for n, t in ((0, c.k), (1, c.v)):
        x = torch.randn(t.shape, generator=gen(seed + n), device=DEV).mul_(80).clamp_(-448, 448)
        t.view(torch.uint8).copy_(x.to(torch.float8_e4m3fn).view(torch.uint8))
    for n, t in ((2, c.k_scale), (3, c.v_scale)):
        t.copy_(torch.exp2(torch.randint(lo, hi, t.shape, generator=gen(seed + n), device=DEV).float()))
    return c


def poison(cache, first_free):
    """Codes of NaN and scales of NaN from slot first_free[b] on (scales: of whole free blocks)."""
    for b, n in enumerate(first_free):
        for t in (cache.k, cache.v):
            t.view(torch.uint8)[b, :, n:] = 0x7f
        for t in (cache.k_scale, cache.v_scale):
            t[b, :, -(-n // cache.block):] = float("nan")


# ---------------------------------------------------------------------------- attention
def attention_ref(q, cache, pos, heads, scale=None):
    """(out, tolerance) in 64 bits. Errors: a score's fp32 sum of 128 exact products in 8 matrix
    instructions, at most 128 + 8 additions and 4 products each off by 2^-23 of sum |q k|; an
    exponential off by the score's error times ln 2 plus 2^-21 (exp2f and the argument's
    rounding at magnitudes to 2^7: 2^-17); a probability rounded to f16 (2^-11); fp32 sums over the
    slots, at most len additions of 2^-23; the bf16 rounding of the result."""
    B, T, Hkv = cache.batch, q.shape[0] // cache.batch, cache.kv_heads
    G = heads // Hkv
    scale = 1 / math.sqrt(128) if scale is None else scale
    out = torch.zeros(B, T, heads, 128, device=DEV, dtype=torch.float64)
    tol = torch.zeros_like(out)
    qd = q.view(B, T, heads, 128).double()
    for b in range(B):
        p0 = pos[b]
        if p0 < 0 or p0 > cache.capacity - T:
            continue
        n = p0 + T
        k, v = (t[b, :, :n].double() * s[b].double().repeat_interleave(cache.block, 1)[:, :n, None]
                for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        for h in range(Hkv):
            hs = slice(h * G, h * G + G)
            x = torch.einsum("tgd,sd->tgs", qd[b, :, hs], k[h]) * scale
            seen = torch.arange(n, device=DEV)[None, None] <= (p0 + torch.arange(T, device=DEV))[:, None, None]
            w = torch.softmax(x.masked_fill(~seen, float("-inf")), dim=-1)
            o = w @ v[h]
            mag = torch.einsum("tgd,sd->tgs", qd[b, :, hs].abs(), k[h].abs()) * scale
            err = 140 * 2.0 ** -23 * (mag * seen).amax(-1, keepdim=True) + 2.0 ** -17
            rel = 2 * err + 2.0 ** -11 + (n + 64) * 2.0 ** -23
            out[b, :, hs] = o
            tol[b, :, hs] = torch.finfo(torch.bfloat16).eps / 2 * o.abs() + rel * (w @ v[h].abs())
    return out.view(B * T, -1), tol.view(B * T, -1)


def run_attention(q, cache, pos, heads, scale=None, out=None):
    T = q.shape[0] // cache.batch
    ws = ops.attention_q8_workspace(cache, heads, T)
    ws.fill_(0xff)
    out = torch.full_like(q, float("nan")) if out is None else out
    position = torch.tensor(pos, device=DEV)
    assert ops.attention_decode_q8(q, cache, position, out, ws, heads, scale) is out
    again = torch.full_like(q, float("nan"))  # with the workspace as the first call left it
    ops.attention_decode_q8(q, cache, position, again, ws, heads, scale)
    assert torch.equal(out.view(torch.int16), again.view(torch.int16))
    return out


def check_attention(q, cache, pos, heads, scale=None):
    full = pos if len(pos) == cache.batch else pos * cache.batch
    out = run_attention(q, cache, pos, heads, scale)
    ref, tol = attention_ref(q, cache, full, heads, scale)
    # a NaN among the codes (values past 448 become one) makes the formula's row NaN too
    bad = ~(((out.double() - ref).abs() <= tol) | (out.isnan() & ref.isnan()))
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst "
                           f"{((out.double() - ref).abs() / tol.clamp_min(1e-30)).max().item()} tol")
    return out


@pytest.mark.parametrize("heads,kv", [(32, 8), (64, 8), (8, 8), (4, 1), (5, 1), (28, 4), (16, 1)])
@pytest.mark.parametrize("T", (1, 2, 5, 16))
def test_attention_heads_and_tokens(heads, kv, T):
    S = 300
    cache = filled_cache(3, kv, S, 64, seed=heads + T)
    pos = [0, 131, S - T]
    poison(cache, [p + T for p in pos])
    check_attention(rand(3 * T, heads * 128, seed=T), cache, pos, heads)


@pytest.mark.parametrize("block", (16, 32, 64, 128))
@pytest.mark.parametrize("layout", ("bhsd", "bshd"))
@pytest.mark.parametrize("S", (1, 16, 17, 63, 64, 65, 129, 1000))
def test_attention_lengths(block, layout, S):
    cache = filled_cache(2, 2, S, block, layout, seed=S)
    for pos in sorted({0, S // 2, max(0, S - 2), S - 1}):
        poison(cache, [pos + 1, S])
        check_attention(rand(2, 8 * 128, seed=pos), cache, [pos, S - 1], 8)
        cache = filled_cache(2, 2, S, block, layout, seed=S)


@pytest.mark.parametrize("B,S", [(1, 8192), (40, 700), (7, 5000)])
def test_attention_ragged_batches(B, S):
    """Lengths from nothing to everything; an idle sequence's rows come out zero."""
    cache = filled_cache(B, 8, S, 64, seed=B)
    pos = [(S - 1) * (b + 1) // B for b in range(B)]
    if B > 2:
        pos[1] = -1
        pos[B // 2] = 0
    poison(cache, [p + 1 if p >= 0 else 0 for p in pos])
    out = check_attention(rand(B, 32 * 128, seed=B), cache, pos, 32)
    if B > 2:
        assert (out[1] == 0).all()
    assert nk.device_error() == 0


@pytest.mark.parametrize("B", (1, 5, 6, 7, 12, 13, 24, 25))
@pytest.mark.parametrize("T,heads", [(1, 32), (3, 32), (4, 64)])
def test_attention_short_and_long_capacities(B, T, heads):
    """The same slots at the start of a short cache and of a long one: the launch depends on the
    capacity and on how many (sequence, kv head) pairs there are."""
    long = filled_cache(B, 8, 4608, 64, seed=B)
    for S in (192, 1024):
        short = ops.Q8Cache(long.k[:, :, :S], long.v[:, :, :S],
                            long.k_scale[:, :, :S // 64].clone(), long.v_scale[:, :, :S // 64].clone(), 64)
        pos = [(S - T) * (b + 1) // B for b in range(B)]
        if B > 5:
            pos[2], pos[4] = -1, 0
        q = rand(B * T, heads * 128, seed=S + T)
        for cache in (short, long):
            check_attention(q, cache, pos, heads)


def test_attention_shared_position_and_scale():
    cache = filled_cache(4, 8, 512, 32, seed=3)
    q = rand(4, 32 * 128, seed=4)
    shared = check_attention(q, cache, [300], 32, scale=0.3)
    each = run_attention(q, cache, [300] * 4, 32, scale=0.3)
    assert torch.equal(shared, each)


def test_attention_all_idle_and_out_of_range():
    cache = filled_cache(3, 2, 64, 16)
    poison(cache, [0, 0, 0])
    q = rand(3, 4 * 128)
    assert (run_attention(q, cache, [-1, -5, -2 ** 62], 4) == 0).all()
    assert nk.device_error() == 0
    assert (run_attention(q, cache, [64, -1, 2 ** 62], 4) == 0).all()
    assert nk.device_error() == _lib.NK_ERR_RANGE
    assert nk.device_error() == 0


def test_attention_value_scales_far_apart():
    """Blocks whose values differ by 2^90, with a peaked softmax on either end."""
    cache = filled_cache(1, 1, 256, 16, seed=5)
    cache.v_scale[0, 0] = torch.exp2(torch.linspace(-60, 30, 16, device=DEV).round())
    for target in (3, 250):
        q = (cache.k[0, 0, target].float() * 0.05).to(torch.bfloat16).view(1, 128)
        cache.k_scale.fill_(2.0 ** -3)
        check_attention(q, cache, [255], 1)


def test_attention_zero_scales_and_flat_scores():
    cache = filled_cache(2, 2, 200, 32, seed=6)
    cache.k_scale.zero_()          # every score 0: a mean of the values
    cache.v_scale[1].zero_()       # and values of 0
    out = check_attention(rand(2, 4 * 128, seed=2), cache, [199, 150], 4)
    assert (out[1] == 0).all()


@pytest.mark.parametrize("where", ("k", "v", "q"))
def test_attention_nan_is_not_lost(where):
    cache = filled_cache(2, 2, 400, 64, seed=7)
    q = rand(2, 4 * 128, seed=3)
    clean = run_attention(q, cache, [399, 399], 4)
    if where == "q":
        q[1, 5] = float("nan")
    else:
        getattr(cache, where).view(torch.uint8)[1, 0, 100:164, 7 if where == "v" else slice(None)] = 0x7f
    out = run_attention(q, cache, [399, 399], 4)
    assert torch.equal(out[0], clean[0])
    row, before = out[1].view(4, 128), clean[1].view(4, 128)
    if where == "q":
        assert row[0].isnan().all() and torch.equal(row[1:], before[1:])
    elif where == "k":
        assert row[:2].isnan().all() and torch.equal(row[2:], before[2:])
    else:
        assert row[:2, 7].isnan().all() and torch.equal(row[2:], before[2:])
        assert torch.equal(row[:2, :7], before[:2, :7])


@pytest.mark.parametrize("T,heads,kv", [(4, 4, 2), (16, 4, 2), (5, 8, 1), (2, 16, 1)])
@pytest.mark.parametrize("pos", (0, 13, 250))
def test_attention_nan_in_later_tokens_stays_there(T, heads, kv, pos):
    """A draft token whose value or key is not finite: the rows before it do not see it."""
    cache = filled_cache(1, kv, 300, 64, seed=11)
    q = rand(T, heads * 128, seed=12)
    clean = run_attention(q, cache, [pos], heads).view(T, heads, 128)
    v = cache.v.view(torch.uint8)
    v[0, 0, pos + T - 1, 7] = 0x7f
    v[0, 0, pos + T // 2, 40:100] = 0xff
    out = run_attention(q, cache, [pos], heads).view(T, heads, 128)
    want = clean.clone()
    G = heads // kv
    want[T - 1:, :G, 7] = float("nan")
    want[T // 2:, :G, 40:100] = float("nan")
    same = (out == want) | (out.isnan() & want.isnan())
    assert same.all()
    cache.k.view(torch.uint8)[0, 0, pos + T - 1, 3] = 0x7f
    out = run_attention(q, cache, [pos], heads).view(T, heads, 128)
    want[T - 1:, :G] = float("nan")
    assert ((out == want) | (out.isnan() & want.isnan())).all()


def test_attention_queries_next_to_the_largest():
    """Scores of 0 whatever the query's size: the mean of the values."""
    cache = filled_cache(1, 1, 128, 64, seed=8)
    cache.k_scale.zero_()
    q = torch.full((1, 128), torch.finfo(torch.bfloat16).max, dtype=torch.bfloat16, device=DEV)
    check_attention(q, cache, [127], 1)
    cache.k_scale.fill_(2.0 ** -64)
    check_attention(q * 2.0 ** -66, cache, [127], 1)


def test_attention_large_and_tiny_queries():
    cache = filled_cache(1, 1, 128, 64, seed=8)
    for std in (1e-30, 1e-4, 30.0):
        check_attention(rand(1, 2 * 128, std=std, seed=9), cache, [127], 2)


def test_attention_past_32_bit_offsets():
    """A cache of 4.5 GB of keys: the last sequence's codes start past 2^32."""
    B, H, S = 9, 8, 1 << 19
    k = torch.zeros(B, H, S, 128, dtype=torch.uint8, device=DEV)
    v = torch.zeros_like(k)
    s = torch.full((B, H, S // 128), 2.0 ** -6, device=DEV)
    for t in (k, v):
        x = torch.randn(H, 2000, 128, generator=gen(1), device=DEV).mul_(80)
        t[-1, :, :2000] = x.to(torch.float8_e4m3fn).view(torch.uint8)
    cache = ops.Q8Cache(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), s, s.clone(), 128)
    pos = [-1] * (B - 1) + [1999]
    check_attention(rand(B, 8 * 128, seed=1), cache, pos, 8)


def test_attention_same_bits_and_captured():
    cache = filled_cache(6, 8, 3000, 64, seed=10)
    q = rand(6, 32 * 128, seed=11)
    pos = [5, 2999, 1000, -1, 64, 2000]
    a, b = run_attention(q, cache, pos, 32), run_attention(q, cache, pos, 32)
    assert torch.equal(a, b)
    # captured at one set of lengths, replayed at others; two graphs with a workspace each
    position = torch.zeros(6, dtype=torch.int64, device=DEV)
    graphs, outs = [], []
    for _ in range(2):
        ws, out = ops.attention_q8_workspace(cache, 32), torch.empty_like(q)
        g = torch.cuda.CUDAGraph()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            ops.attention_decode_q8(q, cache, position, out, ws, 32)
        graphs.append((g, ws, s))
        outs.append(out)
    position.copy_(torch.tensor(pos, device=DEV))
    torch.cuda.synchronize()
    for g, _, s in graphs:
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], a) and torch.equal(outs[1], a)


# ---------------------------------------------------------------------------- append
def e4m3(x):
    """Nearest e4m3 value of fp64 x, ties to even."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return torch.round(x / step) * step


def scale_of(amax):
    if amax == 0:
        return 0.0
    return 2.0 ** max(-64, math.ceil(math.log2(amax / 448.0)))


def rows_ref(x, gain, cos, sin):
    """RMSNorm + RoPE with the step's bf16 cast points, in 64 bits between them; x [..., 128]."""
    r = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    n = r(r(x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)) * gain.double())
    rot = torch.cat((-n[..., 64:], n[..., :64]), dim=-1)
    return r(r(n * cos) + r(rot * sin))


def tables(S):
    return qwen3.rope_tables(qwen3.Qwen3Dims(1024, 1024, 8, 8, 128, 1, 64), S, DEV)


def append(cache, qkv, heads, pos, cos, sin, qn, kn):
    q_out = torch.full((qkv.shape[0], heads * 128), 3.0, dtype=torch.bfloat16, device=DEV)
    assert ops.qk_norm_rope_cache_q8(qkv, qn, kn, cos, sin, torch.tensor(pos, device=DEV), q_out,
                                     cache, heads, EPS) is q_out
    return q_out


def check_append(cache, qkv, heads, pos, T):
    """Scales and value codes exactly; queries and key codes as the cast points leave them, save
    that a value whose fp32 norm falls on the other side of a bf16 rounding border (2^-24 errors
    on steps of 2^-8: one in thousands) moves by one bf16 step (2^-7), and its code by one
    e4m3 step (2^-3 of it)."""
    B, H, S, block = cache.batch, cache.kv_heads, cache.capacity, cache.block
    cos, sin = tables(S)
    qn, kn = (torch.rand(128, generator=gen(i), device=DEV) + 0.5 for i in (50, 51))
    qn, kn = qn.to(torch.bfloat16), kn.to(torch.bfloat16)
    before = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]
    q_out = append(cache, qkv, heads, pos, cos, sin, qn, kn)
    rows = qkv.view(B, T, heads + 2 * H, 128).double()
    for b in range(B):
        p = pos[b if len(pos) > 1 else 0]
        if p < 0 or p > S - T:
            assert (q_out[b * T:b * T + T] == 3.0).all()
            for t, t0 in zip((cache.k, cache.v), before):
                assert torch.equal(t[b].view(torch.uint8), t0[b].view(torch.uint8))
            for t, t0 in zip((cache.k_scale, cache.v_scale), before[2:]):
                assert torch.equal(t[b], t0[b], )
            continue
        c, s = (t[p:p + T].double()[:, None] for t in (cos, sin))
        want_q = rows_ref(rows[b, :, :heads], qn, c, s).view(T, -1)
        got_q = q_out[b * T:b * T + T].double()
        assert ((got_q - want_q).abs() <= 2.0 ** -7 * want_q.abs() + 2.0 ** -7 * 4).all()
        assert (got_q == want_q).double().mean() > 0.99
        new = (rows_ref(rows[b, :, heads:heads + H], kn, c, s), rows[b, :, heads + H:])
        for i, (code, scale) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
            code0, scale0 = before[i][b], before[2 + i][b]
            want, want_s = code0.double(), scale0.clone()
            for j in range(p // block, (p + T - 1) // block + 1):
                lo, hi = max(p, j * block), min(p + T, j * block + block)
                for h in range(H):
                    x = new[i][lo - p:hi - p, h]
                    fin = x[x.isfinite()]
                    sc = scale_of(fin.abs().max().item() if fin.numel() else 0.0)
                    if lo > j * block:
                        sc = max(sc, scale0[h, j].item())
                        old = code0[h, j * block:lo].double()
                        want[h, j * block:lo] = e4m3(old * (scale0[h, j].item() / sc)) if sc else old
                    want_s[h, j] = sc
                    q8 = e4m3(x / sc) if sc else torch.zeros_like(x)
                    want[h, lo:hi] = torch.where(x.isfinite(), q8, torch.full_like(x, float("nan")))
            assert torch.equal(scale[b], want_s)
            got = code[b].double()
            same = (got == want) | (got.isnan() & want.isnan())
            if i == 1:
                assert same.all()
            else:
                near = (got - want).abs() <= 2.0 ** -3 * want.abs() + 2.0 ** -9
                assert (same | near).all() and same.double().mean() > 0.99


@pytest.mark.parametrize("block", (16, 32, 64, 128))
@pytest.mark.parametrize("layout", ("bhsd", "bshd"))
@pytest.mark.parametrize("T", (1, 3, 16))
def test_append(block, layout, T):
    S = 200
    for seed, pos in enumerate(([0, 1, 15, 16], [63, 64, 100, S - T], [127 - T, 128 - T, -1, 31])):
        cache = filled_cache(4, 2, S, block, layout, seed=seed)
        qkv = rand(4 * T, 8 * 128, seed=10 + seed)
        check_append(cache, qkv, 4, pos, T)
    assert nk.device_error() == 0


@pytest.mark.parametrize("heads,kv", [(32, 8), (64, 8), (8, 8), (5, 1), (3, 3)])
def test_append_heads(heads, kv):
    cache = filled_cache(2, kv, 64, 16, seed=kv)
    check_append(cache, rand(2 * 2, (heads + 2 * kv) * 128, seed=heads), heads, [30], 2)


def test_append_rises_and_stays():
    """A block's scale rises with a larger token (earlier codes are rounded anew) and does not
    fall with smaller ones; the first token of a block ignores what the block held before."""
    cache = filled_cache(1, 1, 64, 16, seed=1, lo=20, hi=21)
    for p, std in ((16, 1e-3), (17, 1.0), (18, 1e-4), (19, 3e4), (20, 0.0), (32, 0.0), (33, 1e-20)):
        check_append(cache, rand(1, 3 * 128, std=std, seed=p), 1, [p], 1)


def test_append_extremes():
    """Zeros, the largest bf16 values, values below the least scale, and values that are not
    finite (stored as NaN, the block's scale from the others)."""
    qkv = rand(4, 3 * 128, seed=2)
    qkv[0, 256:] = 0.0
    qkv[1, 256:300] = torch.finfo(torch.bfloat16).max
    qkv[2, 256:] = 2.0 ** -100
    qkv[3, 256] = float("inf")
    qkv[3, 257] = float("nan")
    for p in (0, 5):
        check_append(filled_cache(1, 1, 32, 16, seed=4), qkv, 1, [p], 4)
        check_append(filled_cache(4, 1, 32, 16, seed=5), qkv, 1, [p], 1)


def test_append_out_of_range_and_strided_rows():
    cache = filled_cache(3, 2, 40, 16, seed=6)
    wide = rand(3, 8 * 128 + 12, seed=7)
    check_append(cache, wide[:, 4:4 + 8 * 128].contiguous(), 4, [40, 39, -7], 1)
    assert nk.device_error() == _lib.NK_ERR_RANGE
    a, b = filled_cache(3, 2, 40, 16, seed=6), filled_cache(3, 2, 40, 16, seed=6)
    cos, sin = tables(40)
    qn = kn = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    qa = append(a, wide[:, 4:4 + 8 * 128], 4, [3, 4, 5], cos, sin, qn, kn)
    qb = append(b, wide[:, 4:4 + 8 * 128].contiguous(), 4, [3, 4, 5], cos, sin, qn, kn)
    assert torch.equal(qa, qb)
    assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))


def test_append_then_attend():
    """Tokens appended one by one, in drafts and all at once, then attended: the attention of
    what the cache stands for, close to that of the unrounded keys and values."""
    B, heads, kv, S = 2, 8, 2, 96
    cos, sin = tables(S)
    qn = kn = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    qkv = rand(B * 48, (heads + 2 * kv) * 128, seed=8).view(B, 48, -1)
    for T in (1, 4, 16):
        cache = ops.Q8Cache.empty(B, kv, S, DEV, block=16)
        poison(cache, [0, 0])
        for p in range(0, 48, T):
            x = qkv[:, p:p + T].reshape(B * T, -1)
            q = append(cache, x, heads, [p, p], cos, sin, qn, kn)
            out = check_attention(q, cache, [p, p], heads)
        k, v = cache.dequantize()
        want = qkv.view(B, 48, heads + 2 * kv, 128)[:, :, heads + kv:].transpose(1, 2).float()
        # a code is off by half a step (2^-4) of the value or of the least normal code, and by a
        # whole one more where the block's scale rose later
        tol = 2.0 ** -3 * want.abs() + 2.0 ** -8 * cache.v_scale[:, :, :3].repeat_interleave(16, 2)[..., None]
        assert ((v[:, :, :48] - want).abs() <= tol).all()
        assert out.isfinite().all()


def test_refusals():
    cache = filled_cache(2, 2, 64, 16)
    q = rand(2, 4 * 128)
    out = torch.empty_like(q)
    ws = ops.attention_q8_workspace(cache, 4)
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    ok = dict(q=q, cache=cache, position=pos, out=out, ws=ws, heads=4)
    for bad in (dict(heads=3), dict(heads=34), dict(q=q.float()), dict(q=q[:1]), dict(out=out[:1]),
                dict(q=q.cpu()), dict(position=pos.int()), dict(position=pos.cpu()),
                dict(position=torch.zeros(3, dtype=torch.int64, device=DEV)),
                dict(ws=ws[:16]), dict(ws=ws.cpu()),
                dict(q=rand(34, 512), out=rand(34, 512)),
                dict(q=rand(2, 1024)[:, ::2], out=out)):
        with pytest.raises(ValueError):
            ops.attention_decode_q8(**(ok | bad))
    with pytest.raises(ValueError):
        ops.attention_q8_workspace(cache, 3)
    cos, sin = tables(64)
    gain = torch.ones(128, dtype=torch.bfloat16, device=DEV)
    ok = dict(qkv=rand(2, 8 * 128), q_norm=gain, k_norm=gain, cos=cos, sin=sin, position=pos,
              q_out=out, cache=cache, heads=4, eps=EPS)
    for bad in (dict(heads=5), dict(qkv=rand(2, 7 * 128)), dict(qkv=rand(4, 8 * 128)),
                dict(cos=cos[:63]), dict(sin=sin.float()), dict(q_norm=gain[:64]),
                dict(q_out=out.float()), dict(position=pos[:0]), dict(qkv=rand(2, 8 * 128).cpu())):
        with pytest.raises(ValueError):
            ops.qk_norm_rope_cache_q8(**(ok | bad))
    k, s = cache.k, cache.k_scale
    for args in ((k, cache.v, s, s[:, :, :1], 16), (k, cache.v[:1], s, s, 16),
                 (k.view(torch.uint8), cache.v, s, s, 16), (k, cache.v, s.double(), s, 16),
                 (k[:, :1].expand(2, 2, 64, 128), cache.v[:, :1].expand(2, 2, 64, 128), s, s, 16),
                 (k, cache.v, s, s, 32)):
        with pytest.raises(ValueError):
            ops.Q8Cache(*args)


def test_cache_refuses_shared_arrays():
    c = ops.Q8Cache.empty(1, 2, 64, DEV)
    with pytest.raises(ValueError, match="share"):
        ops.Q8Cache(c.k, c.k, c.k_scale, c.v_scale, 64)
    with pytest.raises(ValueError, match="share"):
        ops.Q8Cache(c.k, c.v, c.k_scale, c.k_scale, 64)
    both = torch.zeros(1, 2, 64, 2, 128, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    ops.Q8Cache(both[..., 0, :], both[..., 1, :], c.k_scale, c.v_scale, 64)  # side by side


@pytest.mark.parametrize("S", (1024, 6000))  # a cluster per pair; the partition and its join
def test_attention_on_two_streams_at_once(S):
    caches = [filled_cache(3, 8, S, 64, seed=n) for n in (1, 2)]
    qs = [rand(3, 32 * 128, seed=n) for n in (3, 4)]
    pos = torch.tensor([S - 1, -1, S // 3], device=DEV)
    want = [run_attention(q, c, pos.tolist(), 32) for q, c in zip(qs, caches)]
    outs = [[torch.full_like(q, float("nan")) for _ in range(20)] for q in qs]
    ws = [ops.attention_q8_workspace(c, 32) for c in caches]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    for i in range(20):
        for n, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                ops.attention_decode_q8(qs[n], caches[n], pos, outs[n][i], ws[n], 32)
    torch.cuda.synchronize()
    for n in range(2):
        for out in outs[n]:
            assert torch.equal(out.view(torch.int16), want[n].view(torch.int16))


@pytest.mark.parametrize("S", (200, 1024, 6000))  # a cluster per pair; the partition and its join
@pytest.mark.parametrize("T,heads", [(1, 4), (3, 16)])
@pytest.mark.parametrize("power", (24, 45, 80))
def test_attention_beside_a_large_scale_that_nothing_uses(S, T, heads, power):
    """Blocks of zero codes whose value scale is 2^power times the others' (a large value that was
    appended and overwritten leaves one behind) take nothing away from the rest.

    Beside attention_ref's errors: what f16 loses of a probability below its normal range is
    2^-33 of the row's largest, and the largest weighs 1 at most."""
    H = 2
    cache = filled_cache(2, H, S, 16, seed=S + power, lo=-8, hi=-4)
    n = S // 16
    for j in {0, 1, 2, 3, 5, n // 3, n // 2, n - 3, n - 1} | set(range(n // 2 + 8, n, 7)):
        cache.v.view(torch.uint8)[:, :, 16 * j:16 * j + 16] = 0
        cache.v_scale[:, :, j] = 2.0 ** (power - 6)
    pos = [S - T, S // 2]
    q = rand(2 * T, heads * 128, std=0.2, seed=power)
    out = run_attention(q, cache, pos, heads)
    ref, tol = attention_ref(q, cache, pos, heads)
    v = cache.dequantize()[1].double().abs()
    total = torch.stack([v[b, :, :p + T].sum(1) for b, p in enumerate(pos)])
    tol = tol.view(2, T, heads, 128) + 2.0 ** -33 * total.repeat_interleave(heads // H, 1)[:, None]
    off = (out.double() - ref).abs().view_as(tol)
    assert (off <= tol).all(), (off / tol).max().item()


@pytest.mark.parametrize("power", (70, 100, 118))
@pytest.mark.parametrize("tiny", (0, 80, 92))
def test_attention_keys_next_to_the_largest(power, tiny):
    """Keys of up to 2^126 against ordinary and tiny queries: scores of up to 2^55 past the others pick
    out one slot, and no product on the way is larger than the score (nor lost where it is not).

    Key codes are powers of two of one sign and each slot has one of its own, so that scores are
    exact and no two are alike; queries are powers of two."""
    S = 96
    cache = filled_cache(1, 1, S, 32, seed=power)
    k = torch.zeros(S, 128, device=DEV)
    for j in range(S):
        k[j, j] = 1.0 + (j % 8) / 8
    cache.k.view(torch.uint8)[0, 0] = k.to(torch.float8_e4m3fn).view(torch.uint8)
    cache.k_scale.fill_(2.0 ** power)
    q = torch.zeros(2, 128, dtype=torch.bfloat16, device=DEV)
    q[0] = 2.0 ** -tiny
    q[1] = -2.0 ** -tiny
    q[0, 71], q[1, 40] = 2.0 ** (1 - tiny), -2.0 ** (-1 - tiny)
    out = run_attention(q.view(1, 256), cache, [S - 1], 2)
    if power - tiny > 12:  # the runner-up is at least 2^(power - tiny) / 8 / sqrt(128) behind
        want = cache.dequantize()[1][0, 0][[71, 40]]
        assert torch.equal(out.view(2, 128).float(), want)
    else:
        check_attention(q.view(1, 256), cache, [S - 1], 2)


@pytest.mark.parametrize("B", (1, 16, 65))
def test_attention_all_idle_in_a_long_cache(B):
    """No sequence has a unit of work, in the form of two launches."""
    cache = filled_cache(B, 8, 8192 // (1 + B // 16), 64, seed=B)
    poison(cache, [0] * B)
    q = rand(2 * B, 16 * 128, seed=B)
    assert (run_attention(q, cache, [-1 - b for b in range(B)], 16) == 0).all()
    assert nk.device_error() == 0


def test_cache_refuses_arrays_that_overlap_at_an_offset():
    f8 = torch.float8_e4m3fn
    c = ops.Q8Cache.empty(2, 2, 64, DEV)
    n = c.k.numel()
    flat = torch.zeros(2 * n, dtype=torch.uint8, device=DEV)

    def codes(start):
        return flat[start:start + n].view(2, 2, 64, 128).view(f8)

    ops.Q8Cache(codes(0), codes(n), c.k_scale, c.v_scale, 64)
    for start in (16, 128, 64 * 128, n - 16):
        for k, v in ((0, start), (start, 0)):
            with pytest.raises(ValueError, match="k and v must not share"):
                ops.Q8Cache(codes(k), codes(v), c.k_scale, c.v_scale, 64)
    # rows of 256 bytes: the values between the keys' rows, or half over them
    pair = torch.zeros(2, 2, 64, 2, 128, dtype=torch.uint8, device=DEV)
    k = pair[..., 0, :].view(f8)
    for at, fine in ((128, True), (64, False), (192, False), (256, False)):
        v = pair.view(-1)[at:].as_strided((2, 2, 64, 128), k.stride()).view(f8) if at <= 128 else \
            torch.zeros(pair.numel() + 512, dtype=torch.uint8, device=DEV)
        if at > 128:
            v, k2 = (v[o:].as_strided((2, 2, 64, 128), k.stride()).view(f8) for o in (at, 0))
        else:
            k2 = k
        if fine:
            ops.Q8Cache(k2, v, c.k_scale, c.v_scale, 64)
        else:
            with pytest.raises(ValueError, match="k and v must not share"):
                ops.Q8Cache(k2, v, c.k_scale, c.v_scale, 64)
    s = torch.zeros(8, device=DEV)
    ops.Q8Cache(c.k, c.v, s[:4].view(2, 2, 1), s[4:].view(2, 2, 1), 64)
    with pytest.raises(ValueError, match="k_scale and v_scale must not share"):
        ops.Q8Cache(c.k, c.v, s[:4].view(2, 2, 1), s[3:7].view(2, 2, 1), 64)
    inside = flat[n - 16:n].view(torch.float32).view(2, 2, 1)
    with pytest.raises(ValueError, match="codes and scales must not share"):
        ops.Q8Cache(codes(0), codes(n), inside, c.v_scale, 64)
    with pytest.raises(ValueError, match="codes and scales must not share"):
        ops.Q8Cache(codes(0), codes(n), c.k_scale, inside, 64)


@pytest.mark.parametrize("B,T,heads,kv,block", [(16, 16, 32, 8, 32), (64, 4, 24, 8, 16), (200, 1, 28, 4, 64)])
@pytest.mark.parametrize("std", (1.0, 1e-3))
def test_append_rounds_as_64_bits_do(B, T, heads, kv, block, std):
    """Queries and key codes equal those of a norm in 64 bits, every one of them.

    The kernel's normalised value is x times 1 / rms as a pair of floats, with the product's own error
    added: within some 2^-46 of the exact one before it is rounded to fp32, as the 64-bit value is on its
    way to bf16. The two fp32 values differ where the exact one lies within 2^-46 of the middle between two
    of them, 2^-21 of all (some 1 of the 10^6 here), and bf16 shows that for one in 2^16 of those. A norm
    in fp32 (errors of 2^-24 and more) moves one value in 10^4 or so across a bf16 border."""
    S = 128
    cache = ops.Q8Cache.empty(B, kv, S, DEV, block=block)
    qkv = rand(B * T, (heads + 2 * kv) * 128, std=std, seed=B)
    cos, sin = tables(S)
    qn, kn = (torch.rand(128, generator=gen(i), device=DEV).add(0.5).to(torch.bfloat16) for i in (60, 61))
    pos = [(7 * b) % (S // block) * block for b in range(B)]  # the first slots of a block
    q_out = append(cache, qkv, heads, pos, cos, sin, qn, kn)
    rows = qkv.view(B, T, heads + 2 * kv, 128).double()
    at = torch.tensor(pos, device=DEV)[:, None] + torch.arange(T, device=DEV)
    c, s = cos[at].double()[:, :, None], sin[at].double()[:, :, None]
    assert torch.equal(q_out.view(B, T, heads, 128).double(), rows_ref(rows[:, :, :heads], qn, c, s))
    keys = rows_ref(rows[:, :, heads:heads + kv], kn, c, s)
    amax = keys.abs().amax(dim=(1, 3))  # of the new tokens, all of one block
    scale = torch.exp2(torch.ceil(torch.log2(amax / 448.0)).clamp(min=-64))
    b = torch.arange(B, device=DEV)
    assert torch.equal(cache.k_scale[b, :, torch.tensor(pos, device=DEV) // block].double(), scale)
    got = cache.k[b[:, None], :, at].double()  # [B, T, kv, 128]
    assert torch.equal(got, e4m3(keys / scale[:, None, :, None]))


def test_each_refusal_is_its_own():
    """Every bad argument beside three good ones, and the message that names it."""
    c = filled_cache(2, 2, 64, 16)
    k, v, ks, vs = c.k, c.v, c.k_scale, c.v_scale
    ops.Q8Cache(k, v, ks, vs, 16)

    def refused(match, **bad):
        with pytest.raises(ValueError, match=match):
            ops.Q8Cache(**(dict(k=k, v=v, k_scale=ks, v_scale=vs, block=16) | bad))

    refused("float8_e4m3fn", k=k.view(torch.uint8))
    refused("float8_e4m3fn", v=v.view(torch.uint8))
    refused("float8_e4m3fn", k=k[..., :64])
    refused("float8_e4m3fn", k=k[0])
    refused("float8_e4m3fn", v=torch.zeros_like(v.view(torch.uint8), device="cpu").view(v.dtype))
    refused("same shape", v=v[:1])
    refused("same shape", v=torch.zeros(2, 64, 2, 128, dtype=torch.uint8, device=DEV).transpose(1, 2).view(v.dtype))
    refused("block must be", block=24)
    refused("scales must be", block=32)
    refused("scales must be", k_scale=ks[:, :, :1])
    refused("scales must be", v_scale=vs.double())
    refused("scales must be", v_scale=vs.cpu())
    refused("scales must be", k_scale=ks.transpose(0, 1))
    refused("layout", k=k[:, :1].expand(2, 2, 64, 128), v=v[:, :1].expand(2, 2, 64, 128))
    refused("layout", k=k[:1].expand(2, 2, 64, 128), v=v[:1].expand(2, 2, 64, 128))
    wide = torch.zeros(2, 2, 2, 64, 136, dtype=torch.uint8, device=DEV).view(k.dtype)
    refused("layout", k=wide[0, ..., :128], v=wide[1, ..., :128])  # strides of 136
    wide = torch.zeros(2, 2, 2, 64, 144, dtype=torch.uint8, device=DEV).view(k.dtype)
    ops.Q8Cache(wide[0, ..., :128], wide[1, ..., :128], ks, vs, 16)
    refused("layout", k=wide[0, ..., 8:136], v=wide[1, ..., 8:136])  # addresses of 8
    refused("batch 1", k=k[:0], v=v[:0], k_scale=ks[:0], v_scale=vs[:0])


def test_largest_batch():
    B, S, T = ops.Q8_MAX_BATCH, 90, 2
    cache = filled_cache(B, 1, S, 32, seed=20)
    pos = [(37 * b) % (S - T + 1) if b % 5 else -1 for b in range(B)]
    check_append(cache, rand(B * T, 4 * 128, seed=21), 2, pos, T)
    out = check_attention(rand(B * T, 2 * 128, seed=22), cache, pos, 2)
    assert (out.view(B, -1)[::5] == 0).all()
    with pytest.raises(ValueError, match="batch 1"):
        ops.Q8Cache.empty(B + 1, 1, 16, DEV)
    assert nk.device_error() == 0


def test_largest_head_counts_and_drafts():
    heads, kv, T = 4096, 256, 16
    cache = filled_cache(1, kv, 40, 16, seed=23)
    check_append(cache, rand(T, (heads + 2 * kv) * 128, seed=24), heads, [13], T)
    check_attention(rand(T, heads * 128, seed=25), cache, [13], heads)
    with pytest.raises(ValueError):
        ops.attention_q8_workspace(filled_cache(1, 257, 16, 16), 257 * 16)
