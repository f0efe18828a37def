// Linears with 4-bit weights and group scales (nk_gemm_w4, include/nk_quant.h).
//
//   y[m, n] = bf16( sum_groups s[n, G] * ( sum_{k in G} (q[n, k] - z[n, G]) x[m, k] ) )
//
// The inner sum's operands are exact in bf16 (q - z is an integer in -15..15), so the tensor
// cores add exact products in fp32 and the group's scale multiplies that fp32 sum: nothing is
// rounded before the one rounding of y.
//
// What bounds it: at decode batches the weight bytes (half a byte each) over HBM. Per SM that
// stream brings about 46 weights a clock, so widening them must cost little: a code becomes a
// bf16 by OR-ing it under the exponent of 128 (0x4300 | q = 128 + q) and subtracting 128 + z, two
// codes per instruction, in the registers of the lane that loaded them, and goes straight into
// mma.sync m16n8k16 with the weights as the 16-row operand and eight tokens as its columns (a
// shared-memory operand would cost four times the weight bytes again in stores). The weights'
// storage is that operand's register layout, so a warp's loads are whole 512-byte rows.
//
// A CTA is eight warps: RW row tiles of 16 weight rows by KW = 8 / RW interleaved K steps (128
// wide). Activations of the CTA's K range go through shared memory in chunks, in operand order.
// CTAs of a cluster share a row tile and split K; partials are added in a fixed order, through
// shared memory within a CTA and distributed shared memory across the cluster, so there is no
// workspace and no order that changes between runs.
#include "nk_common.cuh"
#include "../../include/nk_quant.h"

namespace nk {

constexpr int kW4Threads = 256;
constexpr int kW4Warps = 8;
constexpr int kW4MaxCluster = 8;

struct W4Args {
    const __nv_bfloat16* x; int64_t ldx;
    const uint4* codes;
    const uint32_t* scales;       // pairs of rows (r, r + 8)
    const uint16_t* zeros;        // pairs of rows, or nullptr
    __nv_bfloat16* y; int64_t ldy;
    int M, N, K;
    int KB, NB;                   // K steps of 128, row tiles of 16
    int rw;                       // row tiles per CTA (1, 2, 4 or 8)
    int chunk;                    // K steps staged together
    int nbuf;                     // staging buffers (1 when one chunk holds the CTA's range)
    int fp16_scales;
    int wide_x;                   // x rows may be read in 16-byte pieces
};

__device__ __forceinline__ void mma_w4(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                       uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// (word >> 4p) & 0x000f000f under bf16's 128: two codes as bf16 128 + q, minus 128 + z.
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int p, __nv_bfloat162 base) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xEA;" : "=r"(r) : "r"(word >> (4 * p)));
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&r), base);
    return *reinterpret_cast<const uint32_t*>(&v);
}

__device__ __forceinline__ float w4_scale(uint32_t bits16, int fp16_scales) {
    if (fp16_scales) return __half2float(__ushort_as_half((unsigned short)bits16));
    return __uint_as_float(bits16 << 16);
}

__device__ __forceinline__ uint32_t ld_nc_u32(const void* p) {
    uint32_t v;
    asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ld_nc_u16(const void* p) {
    uint16_t v;
    asm volatile("ld.global.nc.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// 16 bytes of x to shared memory, the first `bytes` of them (0, 2, .. 16) from memory, the rest 0.
__device__ __forceinline__ void w4_stage16(uint32_t dst, const __nv_bfloat16* src, int bytes,
                                           bool wide) {
    if (wide) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
                     "r"(bytes) : "memory");
    } else {
        uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (2 * i < bytes)
                v[i >> 1] |= (uint32_t)__bfloat16_as_ushort(src[i]) << (16 * (i & 1));
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v[0]), "r"(v[1]),
                     "r"(v[2]), "r"(v[3]) : "memory");
    }
}

// One K step (128 wide) of one 16-row tile in registers: two 16-byte code pieces (rows g and
// g + 8) and the NG = 128 / group scale and zero-point pairs.
template <int NG, bool ZP>
struct W4Step {
    uint4 w0, w1;
    uint32_t sc[NG];
    uint32_t zp[ZP ? NG : 1];
};

// NT: token tiles of eight; NG: groups per K step; ZP: zero points given; D: K steps in flight per
// warp.
template <int NT, int NG, bool ZP, int D>
__global__ void __launch_bounds__(kW4Threads, 2) w4_kernel(const W4Args a) {
    extern __shared__ __align__(128) uint8_t w4_smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int rw = a.rw, kw = kW4Warps / rw;
    const int rt = warp % rw, kp = warp / rw;
    const int S = (int)cluster_size(), rank = (int)cluster_rank();
    const int row_block = blockIdx.x / S;           // the cluster's rows
    const int tile = row_block * rw + rt;           // 16-row tile of this warp
    const int m0 = blockIdx.y * (8 * NT);
    const int mcount = min(8 * NT, a.M - m0);
    const int k_begin = (int)((int64_t)rank * a.KB / S);
    const int k_end = (int)((int64_t)(rank + 1) * a.KB / S);
    const bool live = tile < a.NB;

    auto load = [&](int st, W4Step<NG, ZP>& r) {
        if (!live || st >= k_end) return;
        const uint4* c = a.codes + ((int64_t)tile * a.KB + st) * 64 + lane;
        r.w0 = ld_stream_v4(c);
        r.w1 = ld_stream_v4(c + 32);
        const int64_t s0 = ((int64_t)tile * a.KB + st) * NG * 8 + g;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            r.sc[i] = ld_nc_u32(a.scales + s0 + i * 8);
            if (ZP) r.zp[i] = ld_nc_u16(a.zeros + s0 + i * 8);
        }
    };

    W4Step<NG, ZP> q[D];
    // the weights do not depend on the previous launch: their first loads go out before the wait
#pragma unroll
    for (int d = 0; d < D; ++d) load(k_begin + kp + d * kw, q[d]);
    if (threadIdx.x == 0) griddep_launch_dependents();
    griddep_wait();

    const uint32_t s0 = static_cast<uint32_t>(__cvta_generic_to_shared(w4_smem));
    const int buf_bytes = a.chunk * NT * 2048;
    auto stage = [&](int c0, int buf) {  // K steps [c0, c0 + chunk) of every token
        const int steps = min(a.chunk, k_end - c0);
        const int pieces = steps * 16;
        const uint32_t base = s0 + buf * buf_bytes;
        for (int i = threadIdx.x; i < pieces * 8 * NT; i += kW4Threads) {
            const int m = i / pieces, c = i - m * pieces;  // token, 8-wide piece of the chunk
            const int k = c0 * 128 + c * 8;
            const int n = m < mcount ? min(max(a.K - k, 0), 8) : 0;
            const uint32_t dst = base + ((c >> 2) * NT + (m >> 3)) * 512 + ((m & 7) * 4 + (c & 3)) * 16;
            const __nv_bfloat16* src = n > 0 ? a.x + (int64_t)(m0 + m) * a.ldx + k : a.x;
            w4_stage16(dst, src, 2 * n, a.wide_x != 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;

    auto compute = [&](const W4Step<NG, ZP>& r, uint32_t xs) {  // xs: the step's operand pieces
        constexpr int WPG = 4 / NG;  // words per group
        const uint32_t w0[4] = {r.w0.x, r.w0.y, r.w0.z, r.w0.w};
        const uint32_t w1[4] = {r.w1.x, r.w1.y, r.w1.z, r.w1.w};
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            __nv_bfloat162 z0, z1;
            if (ZP) {
                z0 = __bfloat162bfloat162(__ushort_as_bfloat16(0x4300u | (r.zp[i] & 0xffu)));
                z1 = __bfloat162bfloat162(__ushort_as_bfloat16(0x4300u | (r.zp[i] >> 8)));
            } else {
                z0 = z1 = __bfloat162bfloat162(__ushort_as_bfloat16(0x4308u));
            }
            float part[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n) part[n][0] = part[n][1] = part[n][2] = part[n][3] = 0.f;
#pragma unroll
            for (int jj = 0; jj < WPG; ++jj) {
                const int j = i * WPG + jj;
                uint32_t f0[4], f1[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    f0[p] = w4_pair(w0[j], p, z0);
                    f1[p] = w4_pair(w1[j], p, z1);
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t b0, b1, b2, b3;
                    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(b0), "=r"(b1), "=r"(b2), "=r"(b3)
                                 : "r"(xs + (j * NT + n) * 512 + lane * 16));
                    mma_w4(part[n], f0[0], f1[0], f0[1], f1[1], b0, b1);
                    mma_w4(part[n], f0[2], f1[2], f0[3], f1[3], b2, b3);
                }
            }
            const float sa = w4_scale(r.sc[i] & 0xffffu, a.fp16_scales);
            const float sb = w4_scale(r.sc[i] >> 16, a.fp16_scales);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                acc[n][0] = fmaf(sa, part[n][0], acc[n][0]);
                acc[n][1] = fmaf(sa, part[n][1], acc[n][1]);
                acc[n][2] = fmaf(sb, part[n][2], acc[n][2]);
                acc[n][3] = fmaf(sb, part[n][3], acc[n][3]);
            }
        }
    };

    // chunk = kw * D * m steps, so every warp takes D * m steps of a whole chunk and slot d of its
    // queue is always step kp + (..D + d) * kw of it
    stage(k_begin, 0);
    int buf = 0;
    for (int c0 = k_begin; c0 < k_end; c0 += a.chunk) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the chunk is staged; everyone is done with the other buffer
        if (c0 + a.chunk < k_end) stage(c0 + a.chunk, buf ^ 1);
        const int c1 = min(c0 + a.chunk, k_end);
        const uint32_t xb = s0 + buf * buf_bytes;
        for (int st = c0 + kp; st < c1; st += kw * D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const int s = st + d * kw;
                if (s < c1) {
                    if (live) compute(q[d], xb + (s - c0) * (NT * 2048));
                    load(s + kw * D, q[d]);
                }
            }
        }
        buf ^= 1;
    }

    // partial tiles [kp][token][row] in shared memory, over the staging buffers
    __syncthreads();
    float* red = reinterpret_cast<float*>(w4_smem);
    const int rows = 16 * rw, elems = rows * 8 * NT;
    {
        float* p = red + kp * elems + rt * 16;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            p[(8 * n + 2 * t) * rows + g] = acc[n][0];
            p[(8 * n + 2 * t + 1) * rows + g] = acc[n][1];
            p[(8 * n + 2 * t) * rows + g + 8] = acc[n][2];
            p[(8 * n + 2 * t + 1) * rows + g + 8] = acc[n][3];
        }
    }
    __syncthreads();
    const int n0 = row_block * rows;
    const int count = rows * mcount;
    if (S == 1) {
        for (int e = threadIdx.x; e < count; e += kW4Threads) {
            float v = red[e];
            for (int p = 1; p < kw; ++p) v += red[p * elems + e];
            const int m = e / rows, r = e - m * rows;
            if (n0 + r < a.N) a.y[(int64_t)(m0 + m) * a.ldy + n0 + r] = __float2bfloat16_rn(v);
        }
        return;
    }
    if (kw > 1) {  // this CTA's sum into slice 0
        for (int e = threadIdx.x; e < count; e += kW4Threads) {
            float v = red[e];
            for (int p = 1; p < kw; ++p) v += red[p * elems + e];
            red[e] = v;
        }
    }
    cluster_arrive();
    cluster_wait();
    const int per = (count + S - 1) / S;
    const uint32_t r0 = s0;
    for (int e = rank * per + threadIdx.x; e < min(count, (rank + 1) * per); e += kW4Threads) {
        float part[kW4MaxCluster];
#pragma unroll
        for (int s = 0; s < kW4MaxCluster; ++s)
            if (s < S) part[s] = ld_cluster_f32(r0 + 4 * e, s);
        float v = part[0];
#pragma unroll
        for (int s = 1; s < kW4MaxCluster; ++s)
            if (s < S) v += part[s];
        const int m = e / rows, r = e - m * rows;
        if (n0 + r < a.N) a.y[(int64_t)(m0 + m) * a.ldy + n0 + r] = __float2bfloat16_rn(v);
    }
    cluster_arrive();  // no CTA leaves while another may still read its shared memory
    cluster_wait();
}

struct W4Plan {
    int nt, rw, S, chunk, nbuf, smem;
};

template <int NT, int D>
static W4Plan w4_plan(int M, int NB, int KB) {
    W4Plan p;
    p.nt = NT;
    p.rw = NT == 1 ? 2 : (NT == 2 ? 4 : 8);
    const int kw = kW4Warps / p.rw;
    const int tiles = ((NB + p.rw - 1) / p.rw) * ((M + 8 * NT - 1) / (8 * NT));
    p.S = 1;
    while (p.S < kW4MaxCluster && tiles * p.S < 2 * kNumSMs && KB >= 2 * p.S * kw) p.S *= 2;
    const int range = (KB + p.S - 1) / p.S;  // most K steps of one CTA
    const int unit = kw * D;
    int m = (32 * 1024) / (unit * NT * 2048);
    if (m < 1) m = 1;
    if (m > (range + unit - 1) / unit) m = (range + unit - 1) / unit;
    p.chunk = unit * m;
    p.nbuf = range > p.chunk ? 2 : 1;
    const int stage = p.nbuf * p.chunk * NT * 2048;
    const int red = kW4Warps * 16 * 8 * NT * 4;
    p.smem = stage > red ? stage : red;
    return p;
}

template <int NT, int NG, bool ZP, int D>
static int w4_launch(const W4Args& base, cudaStream_t s) {
    const W4Plan p = w4_plan<NT, D>(base.M, base.NB, base.KB);
    W4Args a = base;
    a.rw = p.rw;
    a.chunk = p.chunk;
    a.nbuf = p.nbuf;
    auto kernel = w4_kernel<NT, NG, ZP, D>;
    static bool ready[64] = {};  // shared-memory limit raised, per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return NK_ERR_CUDA;
    if (dev < 0 || dev >= 64) return NK_ERR_DEVICE;
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024) !=
            cudaSuccess)
            return NK_ERR_CUDA;
        ready[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.S * ((a.NB + p.rw - 1) / p.rw), (a.M + 8 * NT - 1) / (8 * NT));
    cfg.blockDim = dim3(kW4Threads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.S;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? NK_OK : NK_ERR_CUDA;
}

template <int NT, int D>
static int w4_dispatch(const W4Args& a, int group, cudaStream_t s) {
    const bool zp = a.zeros != nullptr;
    switch (group) {
        case 32: return zp ? w4_launch<NT, 4, true, D>(a, s) : w4_launch<NT, 4, false, D>(a, s);
        case 64: return zp ? w4_launch<NT, 2, true, D>(a, s) : w4_launch<NT, 2, false, D>(a, s);
        default: return zp ? w4_launch<NT, 1, true, D>(a, s) : w4_launch<NT, 1, false, D>(a, s);
    }
}

static bool w4_shape_ok(int N, int K) {
    return N >= 1 && K >= 1 && N <= (1 << 24) && K <= (1 << 24);
}
static bool w4_group_ok(int group) { return group == 32 || group == 64 || group == 128; }

}  // namespace nk

extern "C" size_t nk_w4_code_bytes(int N, int K) {
    if (!nk::w4_shape_ok(N, K)) return 0;
    return (size_t)((N + 15) / 16) * (size_t)((K + 127) / 128) * 1024;
}

extern "C" size_t nk_w4_scale_bytes(int N, int K, int group) {
    if (!nk::w4_shape_ok(N, K) || !nk::w4_group_ok(group)) return 0;
    return (size_t)((N + 15) / 16) * (size_t)((K + 127) / 128) * (128 / group) * 32;
}

extern "C" size_t nk_w4_zero_bytes(int N, int K, int group) {
    return nk_w4_scale_bytes(N, K, group) / 2;
}

extern "C" int nk_gemm_w4(const void* x, int64_t ldx, const void* codes, const void* scales,
                          const void* zeros, void* y, int64_t ldy, int M, int N, int K, int group,
                          int scale_type, nk_stream_t stream) {
    using namespace nk;
    if (!x || !codes || !scales || !y) return NK_ERR_ARG;
    if (scale_type != NK_W4_SCALE_BF16 && scale_type != NK_W4_SCALE_FP16) return NK_ERR_ARG;
    if (!w4_shape_ok(N, K) || !w4_group_ok(group) || M < 1 || M > (1 << 20) || ldx < K || ldy < N)
        return NK_ERR_SHAPE;
    if (((uintptr_t)codes & 15u) || ((uintptr_t)scales & 15u) || ((uintptr_t)zeros & 1u) ||
        ((uintptr_t)x & 1u) || ((uintptr_t)y & 1u))
        return NK_ERR_ALIGN;
    W4Args a{};
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ldx = ldx;
    a.codes = static_cast<const uint4*>(codes);
    a.scales = static_cast<const uint32_t*>(scales);
    a.zeros = static_cast<const uint16_t*>(zeros);
    a.y = static_cast<__nv_bfloat16*>(y);
    a.ldy = ldy;
    a.M = M;
    a.N = N;
    a.K = K;
    a.KB = (K + 127) / 128;
    a.NB = (N + 15) / 16;
    a.fp16_scales = scale_type == NK_W4_SCALE_FP16;
    a.wide_x = ((uintptr_t)x & 15u) == 0 && ldx % 8 == 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (M <= 8) return w4_dispatch<1, 4>(a, group, s);
    if (M <= 16) return w4_dispatch<2, 4>(a, group, s);
    if (M <= 32) return w4_dispatch<4, 2>(a, group, s);
    return w4_dispatch<8, 2>(a, group, s);
}
