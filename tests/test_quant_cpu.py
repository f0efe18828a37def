"""4-bit weights and the 8-bit cache without a GPU: storage layout against its description in
include/nk_quant.h, and what the entry points refuse before any launch."""

import ctypes

import pytest
import torch

import neokernel_b200 as nk
from neokernel_b200 import _lib, decode_ops as ops


def random_w4(N, K, group, zeros, dtype=torch.bfloat16, seed=0):
    g = torch.Generator().manual_seed(seed)
    G = -(-K // group)
    q = torch.randint(0, 256, (N, -(-K // 2)), generator=g, dtype=torch.uint8)
    s = torch.rand(N, G, generator=g).to(dtype)
    z = torch.randint(0, 16, (N, G), generator=g, dtype=torch.uint8) if zeros else None
    return q, s, z


@pytest.mark.parametrize("N,K,group,zeros", [(1, 1, 32, True), (16, 128, 128, False),
                                             (17, 129, 64, True), (40, 300, 32, True),
                                             (33, 257, 128, True)])
def test_storage_layout(N, K, group, zeros):
    q, s, z = random_w4(N, K, group, zeros)
    w = nk.W4Weight.pack(q, s, z, K=K, group=group)
    L = _lib.load()
    assert w.codes.nbytes == L.nk_w4_code_bytes(N, K)
    assert w.scales.nbytes == L.nk_w4_scale_bytes(N, K, group)
    if zeros:
        assert w.zeros.nbytes == L.nk_w4_zero_bytes(N, K, group)
    NB, KB, GP = -(-N // 128), -(-K // 128), -(-K // 128) * 128 // group
    words = w.codes.view(torch.int32).view(NB, KB, 4, 128, 4)
    scales, zp = w.scales.view(NB, GP, 128), w.zeros.view(NB, GP, 128) if zeros else None
    for n in range(NB * 128):
        i, r = n // 128, n % 128
        for k in range(0, KB * 128, 7):
            b, piece, j, e = k // 128, k % 128 // 32, k % 32 // 8, k % 8
            word = int(words[i, b, piece, r, j]) & 0xffffffff
            code = word >> (4 * (e // 2) + 16 * (e % 2)) & 15
            if n < N and k < K:
                assert code == int(q[n, k // 2]) >> 4 * (k % 2) & 15
                assert scales[i, k // group, r] == s[n, k // group]
                if zeros:
                    assert zp[i, k // group, r] == z[n, k // group]
            else:
                assert code == 0
                if n >= N or k // group >= s.shape[1]:
                    assert scales[i, k // group, r] == 0


@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("N,K,group", [(5, 77, 32), (48, 384, 128)])
def test_dequantize_is_the_formula(N, K, group, zeros):
    q, s, z = random_w4(N, K, group, zeros, torch.float16)
    w = nk.W4Weight.pack(q, s, z, K=K, group=group)
    codes = torch.stack((q & 15, q >> 4), dim=-1).reshape(N, -1)[:, :K].float()
    at = torch.arange(K) // group
    want = (codes - (z.float()[:, at] if zeros else 8.0)) * s.float()[:, at]
    assert torch.equal(w.dequantize(), want)
    assert w.shape == (K, N)


def test_quantize_of_zeros_and_exact_codes():
    w = nk.W4Weight.quantize(torch.zeros(3, 64), 32)
    assert torch.equal(w.dequantize(), torch.zeros(3, 64))
    exact = torch.randint(-7, 8, (4, 128)).float()
    exact[:, 0] = 7.0
    assert torch.equal(nk.W4Weight.quantize(exact * 0.5, 128).dequantize(), exact * 0.5)


def test_pack_refuses():
    q, s, z = random_w4(8, 64, 32, True)
    ok = dict(q=q, scales=s, zeros=z, K=64, group=32)
    for bad in (dict(group=16), dict(group=48), dict(q=q.int()), dict(q=q[0]), dict(K=66),
                dict(scales=s.float()), dict(scales=s[:, :1]), dict(zeros=z.int()),
                dict(zeros=z[:4]), dict(zeros=torch.full_like(z, 16)), dict(K=0)):
        with pytest.raises(ValueError):
            nk.W4Weight.pack(**(ok | bad))
    with pytest.raises(ValueError):
        nk.W4Weight.quantize(torch.zeros(3, 64), 16)
    with pytest.raises(ValueError):
        nk.W4Weight.quantize(torch.zeros(3, 64, dtype=torch.int32))
    w = nk.W4Weight.pack(**ok)  # on the CPU: a linear needs it on the GPU
    with pytest.raises(ValueError):
        nk.mm_w4(torch.zeros(1, 64, dtype=torch.bfloat16), w,
                 out=torch.zeros(1, 8, dtype=torch.bfloat16))


def test_w4_sizes_out_of_range():
    L = _lib.load()
    assert L.nk_w4_code_bytes(0, 128) == 0 and L.nk_w4_code_bytes(16, 0) == 0
    assert L.nk_w4_scale_bytes(16, 128, 16) == 0 and L.nk_w4_scale_bytes(16, 128, 0) == 0
    assert L.nk_w4_code_bytes((1 << 24) + 1, 128) == 0


def test_gemm_w4_abi_refusals():
    L = _lib.load()
    p = 1 << 20  # aligned and never read: every call is refused
    ok = dict(x=p, ldx=256, codes=p, scales=p, zeros=None, y=p, ldy=64, M=1, N=64, K=256, group=128,
              st=0)

    def call(**kw):
        v = ok | kw
        w = _lib.NkW4Weight(v["codes"], v["scales"], v["zeros"], v["N"], v["K"], v["group"], v["st"])
        return L.nk_gemm_w4(v["x"], v["ldx"], ctypes.addressof(w), v["y"], v["ldy"], v["M"], None)

    assert L.nk_gemm_w4(p, 256, None, p, 64, 1, None) == _lib.NK_ERR_ARG
    for kw in (dict(x=None), dict(codes=None), dict(scales=None), dict(y=None), dict(st=2),
               dict(st=-1)):
        assert call(**kw) == _lib.NK_ERR_ARG, kw
    for kw in (dict(M=0), dict(M=-1), dict(M=(1 << 20) + 1), dict(N=0), dict(K=0), dict(group=16),
               dict(group=0), dict(ldx=255), dict(ldy=63), dict(N=(1 << 24) + 1)):
        assert call(**kw) == _lib.NK_ERR_SHAPE, kw
    for kw in (dict(codes=p + 8), dict(scales=p + 2), dict(zeros=p + 4), dict(x=p + 1),
               dict(y=p + 1)):
        assert call(**kw) == _lib.NK_ERR_ALIGN, kw


CACHE = dict(k=1 << 20, v=1 << 20, ks=1 << 20, vs=1 << 20, batch=2, hkv=8, d=128, cap=64, block=16,
             reserved=0, cb=8 * 64 * 128, ch=64 * 128, cs=128)
BAD_SHAPES = (dict(batch=0), dict(batch=1025), dict(tokens=0), dict(tokens=17), dict(hq=0),
              dict(hkv=0), dict(hq=33), dict(hq=136), dict(d=64), dict(cap=0),
              dict(cap=(1 << 30) + 1), dict(tokens=16, cap=15), dict(block=8), dict(block=48),
              dict(block=256), dict(cs=112))
BAD_ALIGNMENT = (dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 4), dict(ks=(1 << 20) + 2),
                 dict(vs=(1 << 20) + 1), dict(pos=(1 << 20) + 4), dict(cs=136),
                 dict(ch=64 * 128 + 8), dict(cb=8 * 64 * 128 + 4))


def test_append_q8_abi_refusals():
    L = _lib.load()
    p = 1 << 20
    ok = dict(qkv=p, ld=48 * 128, qn=p, kn=p, cos=p, sin=p, pos=p, per=1, q=p, tokens=1, hq=32)

    def call(**kw):
        v = ok | kw
        c = _lib.NkQ8Cache(*(kw.get(n, x) for n, x in CACHE.items()))
        return L.nk_qk_norm_rope_cache_q8(
            v["qkv"], v["ld"], v["qn"], v["kn"], v["cos"], v["sin"], v["pos"], v["per"], v["q"],
            kw.get("cache", ctypes.addressof(c)), v["tokens"], v["hq"], 1e-6, None)

    for n in ("qkv", "qn", "kn", "cos", "sin", "pos", "q", "k", "v", "ks", "vs", "cache"):
        assert call(**{n: None}) == _lib.NK_ERR_ARG, n
    for kw in BAD_SHAPES + (dict(ld=48 * 128 - 4),):
        assert call(**kw) == _lib.NK_ERR_SHAPE, kw
    for kw in BAD_ALIGNMENT + (dict(qkv=p + 4), dict(q=p + 2), dict(ld=48 * 128 + 2),
                               dict(cos=p + 2)):
        assert call(**kw) == _lib.NK_ERR_ALIGN, kw


def test_attention_q8_abi_refusals():
    L = _lib.load()
    p = 1 << 20
    need = L.nk_attention_q8_ws_bytes(1, 32, 8)
    assert need > 0
    ok = dict(q=p, pos=p, per=0, out=p, tokens=1, hq=32, ws=p, n=need)

    def call(**kw):
        v = ok | kw
        c = _lib.NkQ8Cache(*(kw.get(n, x) for n, x in CACHE.items()))
        return L.nk_attention_decode_q8(v["q"], kw.get("cache", ctypes.addressof(c)), v["pos"],
                                        v["per"], v["out"], v["tokens"], v["hq"], 0.1, v["ws"],
                                        v["n"], None)

    for n in ("q", "k", "v", "ks", "vs", "pos", "out", "cache"):
        assert call(**{n: None}) == _lib.NK_ERR_ARG, n
    for kw in BAD_SHAPES + (dict(cap=1 << 30, batch=1024),):
        assert call(**kw) == _lib.NK_ERR_SHAPE, kw
    for kw in (dict(ws=None), dict(n=need - 1), dict(tokens=16)):
        assert call(**kw) == _lib.NK_ERR_WORKSPACE, kw
    for kw in BAD_ALIGNMENT + (dict(q=p + 4), dict(out=p + 2), dict(ws=p + 8)):
        assert call(**kw) == _lib.NK_ERR_ALIGN, kw


def test_attention_q8_workspace_sizes():
    L = _lib.load()
    assert L.nk_attention_q8_ws_bytes(0, 32, 8) == 0
    assert L.nk_attention_q8_ws_bytes(17, 32, 8) == 0
    assert L.nk_attention_q8_ws_bytes(1, 33, 8) == 0
    assert L.nk_attention_q8_ws_bytes(1, 136, 8) == 0
    sizes = [L.nk_attention_q8_ws_bytes(t, 64, 8) for t in range(1, 17)]
    assert sizes == sorted(sizes)  # a workspace for T tokens serves fewer


def test_q8_cache_refuses_cpu_tensors_and_bad_blocks():
    k = torch.zeros(1, 2, 64, 128, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s = torch.zeros(1, 2, 1)
    with pytest.raises(ValueError):
        ops.Q8Cache(k, k.clone(), s, s.clone(), 64)
    with pytest.raises(ValueError):
        ops.Q8Cache.empty(1, 2, 64, "cpu", block=24)
    with pytest.raises(ValueError):
        ops.Q8Cache.empty(1, 2, 64, "cpu", layout="sbhd")


def test_quantize_refuses_what_has_no_scale():
    for bad in (float("nan"), float("inf")):
        w = torch.ones(4, 64)
        w[2, 5] = bad
        for zeros in (False, True):
            with pytest.raises(ValueError, match="finite"):
                nk.W4Weight.quantize(w, 32, zeros=zeros)
    w = torch.full((2, 32), 1e6)  # 1e6 / 7 is past fp16
    with pytest.raises(ValueError, match="finite"):
        nk.W4Weight.quantize(w, 32, scale_dtype=torch.float16)
    assert torch.isfinite(nk.W4Weight.quantize(w, 32).dequantize()).all()


def test_withhold_w4_request_rejects_a_bad_cta():
    L = _lib.load()
    assert L.nk_test_withhold_w4(-2) == _lib.NK_ERR_ARG
    assert L.nk_test_withhold_w4(-1) == 0


def test_rows_of_two_arrays_meet_or_not():
    """The search that Q8Cache refuses overlapping arrays by, against all sums."""
    g = torch.Generator().manual_seed(7)

    def some(lo, hi):
        return int(torch.randint(lo, hi, (1,), generator=g))

    met = 0
    for _ in range(3000):
        dims, extent = [], 4
        for _ in range(some(0, 4)):  # each stride past what is below it, as a cache's are
            stride, count = extent + some(0, 9), some(2, 5)
            dims.insert(0, (stride, count))
            extent = stride * count
        both = [(st, 2 * n - 1) for st, n in dims]
        for d in (dims, both):
            sums = [0]
            for st, n in d:
                sums = [x + i * st for x in sums for i in range(n)]
            lo = some(-20, 2 * extent + 20)
            hi = lo + some(1, 30)
            want = any(lo < x < hi for x in sums)
            assert ops._meets(d, lo, hi) == want, (d, lo, hi)
            met += want
    assert 1000 < met < 5000
