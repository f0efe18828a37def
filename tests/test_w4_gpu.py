"""Linears with 4-bit weights (neokernel_b200.mm_w4) against the formula in 64 bits.

Tolerance, derived: codes minus zero points and bf16 activations multiply exactly, so errors are
those of the fp32 sums and of the one bf16 rounding. A sum over K runs through K / 16 matrix
instructions of 16 products, then one multiply-add per group and at most 64 additions of
partials; taking every one of those additions (16 inside an instruction) as off by 2^-23 of the
sum of magnitudes so far, |y - ref| <= eps_bf16 / 2 |ref| + (K + K / 32 + 64) 2^-23 sum |x w|.
"""

import time

import pytest
import torch

import neokernel_b200 as nk
from neokernel_b200 import _lib, synthetic

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(N, K, group, zeros, scale_dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    G = -(-K // group)
    q = torch.randint(0, 256, (N, -(-K // 2)), generator=g, device=DEV, dtype=torch.uint8)
    s = (torch.rand(N, G, generator=g, device=DEV) * 0.01 - 0.002).to(scale_dtype)
    z = (torch.randint(0, 16, (N, G), generator=g, device=DEV, dtype=torch.uint8)
         if zeros else None)
    codes = torch.stack((q & 15, q >> 4), dim=-1).reshape(N, -1)[:, :K].double()
    at = torch.arange(K, device=DEV) // group
    w = (codes - (z.double()[:, at] if zeros else 8.0)) * s.double()[:, at]
    return nk.W4Weight.pack(q, s, z, K=K, group=group), w


def check(y, x, w):
    ref = x.double() @ w.t()
    K = x.shape[1]
    tol = (torch.finfo(torch.bfloat16).eps / 2 * ref.abs()
           + (K + K / 32 + 64) * 2.0 ** -23 * (x.double().abs() @ w.abs().t()))
    bad = (y.double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(y.double() - ref).abs().max()}"


@pytest.mark.parametrize("M", (1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 130))
@pytest.mark.parametrize("group,zeros,scale", [(32, True, torch.float16), (64, False, torch.bfloat16),
                                               (128, True, torch.bfloat16)])
def test_tokens(M, group, zeros, scale):
    W, w = make(400, 1152, group, zeros, scale, seed=M)
    x = synthetic.activation(M, 1152, seed=M, device=DEV)
    y = torch.full((M, 400), float("nan"), dtype=torch.bfloat16, device=DEV)
    assert nk.mm_w4(x, W, out=y) is y
    check(y, x, w)


@pytest.mark.parametrize("N,K", [(1, 1), (1, 128), (15, 127), (16, 129), (17, 31), (33, 4097),
                                 (1003, 2477), (5000, 96), (128, 12288), (24576, 256)])
@pytest.mark.parametrize("M", (1, 5, 40))
@pytest.mark.parametrize("group,zeros", [(32, False), (64, True), (128, False), (128, True)])
def test_sizes(N, K, M, group, zeros):
    W, w = make(N, K, group, zeros, torch.bfloat16, seed=N + K)
    x = synthetic.activation(M, K, seed=K, device=DEV)
    y = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
    nk.mm_w4(x, W, out=y)
    check(y, x, w)


@pytest.mark.parametrize("M", (1, 4, 20))
def test_strided_rows_and_guard(M):
    """Rows of a wider x at an odd offset (no 16-byte pieces), rows of a wider y; what surrounds
    the output stays as it was."""
    W, w = make(200, 320, 64, True, torch.bfloat16)
    for off, ld in ((0, 328), (1, 331), (3, 400)):
        wide = synthetic.activation(M, ld + 8, seed=off, device=DEV)
        x = wide[:, off:off + 320]
        big = torch.full((M + 2, 260), 7.0, dtype=torch.bfloat16, device=DEV)
        y = big[1:M + 1, 30:230]
        nk.mm_w4(x, W, out=y)
        check(y, x, w)
        big[1:M + 1, 30:230] = 7.0
        assert (big == 7.0).all()


def test_same_bits_again_and_in_a_graph():
    W, _ = make(6144, 4096, 128, False, torch.bfloat16)
    x = synthetic.activation(4, 4096, seed=1, device=DEV)
    ys = [torch.empty(4, 6144, dtype=torch.bfloat16, device=DEV) for _ in range(3)]
    nk.mm_w4(x, W, out=ys[0])
    nk.mm_w4(x, W, out=ys[1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        nk.mm_w4(x, W, out=ys[2])
    x.mul_(2.0)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(ys[0], ys[1])
    assert torch.equal(ys[2], ys[0] * 2.0)


def test_two_streams_at_once():
    W, w = make(4096, 4096, 64, True, torch.bfloat16)
    x = [synthetic.activation(m, 4096, seed=m, device=DEV) for m in (3, 12)]
    y = [torch.empty(t.shape[0], 4096, dtype=torch.bfloat16, device=DEV) for t in x]
    streams = [torch.cuda.Stream() for _ in x]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            nk.mm_w4(x[i], W, out=y[i], stream=s)
    torch.cuda.synchronize()
    for i in range(2):
        check(y[i], x[i], w)


def test_non_finite_values_stay_in_their_token():
    W, w = make(300, 640, 128, False, torch.bfloat16)
    x = synthetic.activation(6, 640, seed=3, device=DEV)
    y0, y1 = (torch.empty(6, 300, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    nk.mm_w4(x, W, out=y0)
    x[2, 17] = float("nan")
    x[4, 600] = float("inf")
    nk.mm_w4(x, W, out=y1)
    for m in (0, 1, 3, 5):
        assert torch.equal(y0[m], y1[m])
    assert y1[2].isnan().all()
    assert not y1[4].isfinite().any()


@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("zeros", (False, True))
def test_quantize_runs_as_a_linear(group, zeros):
    """quantize: each weight within half a code step (plus the scale's own rounding) of the
    original, and the linear computes with what dequantize says."""
    N, K = 272, 512
    full = synthetic.weight(N, K, seed=5, device=DEV).float() + (0.01 if zeros else 0.0)
    W = nk.W4Weight.quantize(full, group, zeros=zeros)
    got = W.dequantize()
    v = full.view(N, K // group, group)
    span = (v.amax(-1).clamp(min=0) - v.amin(-1).clamp(max=0)) / 15 if zeros else v.abs().amax(-1) / 7
    # half a step, and a whole one more where a zero point or a rounded scale clips the end
    assert ((got - full).abs().view_as(v) <= 1.52 * span[..., None]).all()
    assert ((got - full).abs().view_as(v) <= 0.51 * span[..., None]).float().mean() > 0.9
    x = synthetic.activation(9, K, seed=6, device=DEV)
    y = torch.empty(9, N, dtype=torch.bfloat16, device=DEV)
    nk.mm_w4(x, W, out=y)
    check(y, x, got.double())


def test_zero_tokens():
    W, _ = make(64, 128, 128, False, torch.bfloat16)
    y = torch.empty(0, 64, dtype=torch.bfloat16, device=DEV)
    assert nk.mm_w4(torch.empty(0, 128, dtype=torch.bfloat16, device=DEV), W, out=y) is y


def test_refusals():
    W, _ = make(64, 128, 128, False, torch.bfloat16)
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=DEV)
    y = torch.zeros(2, 64, dtype=torch.bfloat16, device=DEV)
    for bad in (dict(a=x.float()), dict(a=x[0]), dict(a=x[:, :64]), dict(a=x.cpu()),
                dict(a=torch.zeros(128, 2, dtype=torch.bfloat16, device=DEV).t()),
                dict(a=x[:1].expand(2, 128)),
                dict(out=y.float()), dict(out=y[:1]), dict(out=y.cpu()), dict(w=x),
                dict(out=torch.zeros(64, 2, dtype=torch.bfloat16, device=DEV).t())):
        args = dict(a=x, w=W, out=y) | bad
        with pytest.raises(ValueError):
            nk.mm_w4(args["a"], args["w"], out=args["out"])


# (M, N, K, group, CTAs of a tile): one CTA a tile; a cluster of eight, of three (two or three steps each) and
# of two; each way in which the sums leave tensor memory
@pytest.mark.parametrize("M,N,K,group,S", [(1, 24576, 512, 128, 1), (4, 4096, 4096, 64, 8),
                                           (16, 4096, 896, 32, 3), (40, 12288, 1024, 32, 2)])
def test_a_wait_that_runs_out_writes_nothing_of_its_tile(M, N, K, group, S):
    """The CTA's waits expire (nothing faults or hangs), no CTA of its cluster stores sums that lack
    its part, the error is reported, and the next call is right."""
    L = _lib.load()
    W, w = make(N, K, group, True, torch.bfloat16)
    x = synthetic.activation(M, K, seed=M, device=DEV)
    clean = torch.empty(M, N, dtype=torch.bfloat16, device=DEV)
    nk.mm_w4(x, W, out=clean)
    check(clean, x, w)
    for tile, rank in ((1, 0), (2, S - 1)):
        y = torch.full((M, N), 7.0, dtype=torch.bfloat16, device=DEV)
        assert L.nk_test_withhold_w4(tile * S + rank) == 0
        t0 = time.perf_counter()
        nk.mm_w4(x, W, out=y)
        torch.cuda.synchronize()
        waited = time.perf_counter() - t0
        assert nk.device_error() == _lib.NK_ERR_TIMEOUT
        assert 1.0 <= waited <= 30.0, waited
        rows = slice(128 * tile, 128 * tile + 128)
        assert (y[:, rows] == 7.0).all(), "a tile without one of its parts was written"
        y[:, rows] = clean[:, rows]
        assert torch.equal(y, clean)
        nk.mm_w4(x, W, out=y.fill_(7.0))  # the request was consumed
        assert torch.equal(y, clean)
        assert nk.device_error() == 0


def test_withhold_request_is_validated():
    L = _lib.load()
    assert L.nk_test_withhold_w4(-2) == _lib.NK_ERR_ARG
    assert L.nk_test_withhold_w4(5) == 0
    assert L.nk_test_withhold_w4(-1) == 0  # cleared
    W, w = make(256, 256, 128, False, torch.bfloat16)
    x = synthetic.activation(2, 256, seed=1, device=DEV)
    y = torch.empty(2, 256, dtype=torch.bfloat16, device=DEV)
    nk.mm_w4(x, W, out=y)
    check(y, x, w)
    assert nk.device_error() == 0


@pytest.mark.parametrize("M,N,K", [(70000, 130, 200), (1 << 20, 3, 16)])
def test_many_tokens(M, N, K):
    W, w = make(N, K, 32, True, torch.bfloat16)
    x = synthetic.activation(M, K, seed=1, device=DEV)
    y = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=DEV)
    nk.mm_w4(x, W, out=y)
    check(y, x, w)
    if M == 1 << 20:
        with pytest.raises(ValueError):
            nk.mm_w4(torch.cat((x, x[:1])), W, out=torch.cat((y, y[:1])))
