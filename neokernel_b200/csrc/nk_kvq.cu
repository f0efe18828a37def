// KV cache in 8 bits (include/nk_quant.h): the append that fills it and the attention that reads
// it. Codes are e4m3, with one power-of-two scale per (sequence, kv head, block of tokens).
#include <cuda_fp16.h>

#include "nk_common.cuh"
#include "../../include/nk_quant.h"

namespace nk {

constexpr int kQ8MinScaleExp = -64;
constexpr int kQ8MaxCapacity = 1 << 30;  // slot arithmetic on the host stays within 32 bits

// First new slot of sequence b, or -1 where nothing is to be done for it (idle, or out of range).
__device__ __forceinline__ int64_t q8_position(const int64_t* position, int per_sequence, int b,
                                               int tokens, int capacity) {
    const int64_t p = position[per_sequence ? b : 0];
    return p < 0 || p > (int64_t)capacity - tokens ? -1 : p;
}

// ---------------------------------------------------------------------------------------
// Append. RMSNorm + RoPE as qk_norm_rope_cache_kernel rounds them, a warp per 128-element head
// row (lane l owns elements 4l .. 4l + 3; its RoPE partner is lane l ^ 16).
//
// A CTA of eight warps takes either query rows (one or four a warp, their loads in flight
// together), or one (sequence, kv head, touched block): it holds the block's new rows in registers
// (at most 16 tokens, two a warp), finds their largest magnitudes, fixes the block's two scales, rounds
// earlier tokens' codes anew where a scale rose, and stores. Each block belongs to one CTA, so nothing
// is shared between CTAs. The launch and two dependent round trips to memory bound it at one token (2.8
// us, 0.75 where every sequence is idle; 16 sequences 3.2), issue slots at 16 sequences of 16 tokens and
// 64 heads (7.5 us for 10 MB, 1.3 TB/s). Where a scale rises, a warp takes one earlier row after the
// other, each a load, a conversion and a store: 6.5 us where a full block of 64 is rounded anew, 9.5
// for one of 128, against 3.2 measured the same way where none rises.
// ---------------------------------------------------------------------------------------
struct Q8AppendArgs {
    const __nv_bfloat16* qkv; int64_t ld;
    const __nv_bfloat16 *qn, *kn, *cos_t, *sin_t;
    const int64_t* position; int per_sequence;
    __nv_bfloat16* q_out;
    uint8_t *k, *v;
    float *ks, *vs;
    int batch, tokens, hq, hkv, capacity, block, blocks;
    int64_t cb, ch, cs;
    float eps;
    int q_ctas;                  // CTAs of query rows per sequence
};

struct Row4 { float v[4]; };

__device__ __forceinline__ Row4 load_row4(const __nv_bfloat16* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    return Row4{{bf16lo(u.x), bf16hi(u.x), bf16lo(u.y), bf16hi(u.y)}};
}

// Two floats rounded to a bf16 pair in one instruction (the low half first).
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ Row4 bf16_row(const Row4& r) {  // rounded to bf16 and back
    const uint32_t a = bf16_pair(r.v[0], r.v[1]), b = bf16_pair(r.v[2], r.v[3]);
    return Row4{{bf16lo(a), bf16hi(a), bf16lo(b), bf16hi(b)}};
}

// bf16 cast points of the decode step: the normalised value, its product with the gain, each
// RoPE product, and their sum. The result's values are bf16 values.
__device__ __forceinline__ Row4 q8_norm_rope(Row4 x, const __nv_bfloat16* gain,
                                             const __nv_bfloat16* cos_r,
                                             const __nv_bfloat16* sin_r, int lane, float eps) {
    // The mean square and the normalised value in more than 32 bits (1 / rms as a pair of floats):
    // an fp32 error there carries a value next to a bf16 border to the other side (one in some ten
    // thousand), and with it an e4m3 code by a whole step. 128 elements a row: it costs 0.3 us of
    // 2.9 at one token.
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) ss = fma((double)x.v[i], (double)x.v[i], ss);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
    const double inv = rsqrt(ss * (1.0 / kHeadDim) + (double)eps);
    const float ih = (float)inv, il = (float)(inv - (double)ih);
    const Row4 w = load_row4(gain + 4 * lane), c = load_row4(cos_r + 4 * lane),
               s = load_row4(sin_r + 4 * lane);
    Row4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = x.v[i] * ih;
        y.v[i] = p + fmaf(x.v[i], il, fmaf(x.v[i], ih, -p));
    }
    y = bf16_row(y);
#pragma unroll
    for (int i = 0; i < 4; ++i) y.v[i] *= w.v[i];
    y = bf16_row(y);
    Row4 a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float o = __shfl_xor_sync(0xffffffffu, y.v[i], 16);
        a.v[i] = y.v[i] * c.v[i];
        b.v[i] = (lane < 16 ? -o : o) * s.v[i];
    }
    a = bf16_row(a);
    b = bf16_row(b);
#pragma unroll
    for (int i = 0; i < 4; ++i) a.v[i] += b.v[i];
    return bf16_row(a);
}

// Smallest power of two s >= 2^-64 with amax <= 448 s (0 for 0). 448 = 1.75 * 2^8.
__device__ __forceinline__ float q8_scale(float amax) {
    if (amax == 0.f) return 0.f;
    const uint32_t u = __float_as_uint(amax);
    int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = max(e, kQ8MinScaleExp);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}

__device__ __forceinline__ uint32_t q8_codes(const Row4& r, float inv) {  // r * inv; NaN if not finite
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)  // (the conversion saturates infinities)
        f[i] = fabsf(r.v[i]) <= 3.4028235e38f ? r.v[i] * inv : __uint_as_float(0x7fc00000u);
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(f[1]), "f"(f[0]));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(f[3]), "f"(f[2]));
    return (uint32_t)lo | (uint32_t)hi << 16;
}

__device__ __forceinline__ float2 q8_decode2(uint32_t codes16) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((unsigned short)codes16));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

__device__ __forceinline__ uint32_t q8_requant(uint32_t codes, float ratio) {
    const float2 a = q8_decode2(codes & 0xffffu), b = q8_decode2(codes >> 16);
    const Row4 r{{a.x, a.y, b.x, b.y}};
    return q8_codes(r, ratio);
}

__device__ __forceinline__ float finite_max(const Row4& r, float m) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float x = fabsf(r.v[i]);
        if (x <= 3.4028235e38f) m = fmaxf(m, x);
    }
    return m;
}

constexpr int kQ8Warps = 8;

// QR: query rows per warp.
template <int QR>
__global__ void __launch_bounds__(32 * kQ8Warps) q8_append_kernel(const Q8AppendArgs a) {
    __shared__ float s_max[2][kQ8Warps];
    if (threadIdx.x == 0) griddep_launch_dependents();
    griddep_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.y;
    const int64_t raw = a.position[a.per_sequence ? b : 0];
    const int64_t pos = q8_position(a.position, a.per_sequence, b, a.tokens, a.capacity);
    if (pos < 0) {
        if (raw >= 0 && blockIdx.x == 0 && threadIdx.x == 0) atomicExch(&g_error, NK_ERR_RANGE);
        return;
    }
    const int T = a.tokens;
    if ((int)blockIdx.x < a.q_ctas) {  // query rows
        const int row0 = (blockIdx.x * kQ8Warps + warp) * QR, rows = T * a.hq;
        const __nv_bfloat16* base = a.qkv + (int64_t)b * T * a.ld + 4 * lane;
        __nv_bfloat16* out = a.q_out + ((int64_t)b * rows) * kHeadDim + 4 * lane;
        Row4 x[QR];
        int t[QR];
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const int row = min(row0 + i, rows - 1);
            t[i] = row / a.hq;
            x[i] = load_row4(base + t[i] * a.ld + (row - t[i] * a.hq) * kHeadDim);
        }
#pragma unroll
        for (int i = 0; i < QR; ++i) {
            const Row4 y = q8_norm_rope(x[i], a.qn, a.cos_t + (pos + t[i]) * kHeadDim,
                                        a.sin_t + (pos + t[i]) * kHeadDim, lane, a.eps);
            if (row0 + i < rows)
                *reinterpret_cast<uint2*>(out + (int64_t)(row0 + i) * kHeadDim) =
                    make_uint2(bf16_pair(y.v[0], y.v[1]), bf16_pair(y.v[2], y.v[3]));
        }
        return;
    }
    const int u = blockIdx.x - a.q_ctas;
    const int h = u % a.hkv;
    const int64_t blk = pos / a.block + u / a.hkv;
    const int64_t s0 = blk * a.block;                            // the block's first slot
    const int64_t lo = pos > s0 ? pos : s0;                      // its new slots [lo, hi)
    const int64_t hi = min(pos + T, s0 + a.block);
    if (lo >= hi) return;
    const int n = (int)(hi - lo);
    const bool earlier = lo > s0;
    const int64_t si = ((int64_t)b * a.hkv + h) * a.blocks + blk;
    const float k_old = earlier ? a.ks[si] : 0.f, v_old = earlier ? a.vs[si] : 0.f;
    Row4 kr[2], vr[2];
    float km = 0.f, vm = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = warp + i * kQ8Warps;
        if (j < n) {
            const int64_t slot = lo + j;
            const __nv_bfloat16* src = a.qkv + ((int64_t)b * T + (slot - pos)) * a.ld + 4 * lane;
            kr[i] = q8_norm_rope(load_row4(src + (int64_t)(a.hq + h) * kHeadDim), a.kn,
                                 a.cos_t + slot * kHeadDim, a.sin_t + slot * kHeadDim, lane, a.eps);
            vr[i] = load_row4(src + (int64_t)(a.hq + a.hkv + h) * kHeadDim);
            km = finite_max(kr[i], km);
            vm = finite_max(vr[i], vm);
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        km = fmaxf(km, __shfl_xor_sync(0xffffffffu, km, off));
        vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, off));
    }
    if (lane == 0) {
        s_max[0][warp] = km;
        s_max[1][warp] = vm;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kQ8Warps; ++w) {
        km = fmaxf(km, s_max[0][w]);
        vm = fmaxf(vm, s_max[1][w]);
    }
    const float k_new = fmaxf(k_old, q8_scale(km)), v_new = fmaxf(v_old, q8_scale(vm));
    // scales are powers of two in [2^-64, 2^120], or 0 (every value 0): the reciprocals are exact
    const float k_inv = k_new > 0.f ? 1.f / k_new : 0.f, v_inv = v_new > 0.f ? 1.f / v_new : 0.f;
    const int64_t base = (int64_t)b * a.cb + (int64_t)h * a.ch + 4 * lane;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = warp + i * kQ8Warps;
        if (j < n) {
            const int64_t at = base + (lo + j) * a.cs;
            *reinterpret_cast<uint32_t*>(a.k + at) = q8_codes(kr[i], k_inv);
            *reinterpret_cast<uint32_t*>(a.v + at) = q8_codes(vr[i], v_inv);
        }
    }
    if (threadIdx.x == 0) {
        a.ks[si] = k_new;
        a.vs[si] = v_new;
    }
    const bool k_rose = earlier && k_new != k_old, v_rose = earlier && v_new != v_old;
    if (k_rose || v_rose) {
        const float kq = k_old * k_inv, vq = v_old * v_inv;
        for (int64_t slot = s0 + warp; slot < lo; slot += kQ8Warps) {
            const int64_t at = base + slot * a.cs;
            if (k_rose) {
                uint32_t* p = reinterpret_cast<uint32_t*>(a.k + at);
                *p = q8_requant(*p, kq);
            }
            if (v_rose) {
                uint32_t* p = reinterpret_cast<uint32_t*>(a.v + at);
                *p = q8_requant(*p, vq);
            }
        }
    }
}

// ---------------------------------------------------------------------------------------
// Attention of T new tokens over the 8-bit cache.
//
// Bound by the cache's bytes over HBM (a token of one kv head is 256 bytes), so every byte is read
// once and must be requested early: the work is the list of 64-slot units of all (sequence, kv
// head) pairs, and CTA c of the launch takes the contiguous units [U c / G, U (c + 1) / G), so
// ragged batches leave every CTA the same number of bytes. Each of a CTA's four warps streams its
// own 16 slots of every unit through a private ring of asynchronous copies, with no barrier
// between warps until a pair ends.
//
// Per 16 slots (lane = 4 g + t): S^T = K Q^T by mma.m16n8k16 in f16 with the slots as rows and
// up to 8 query rows (token, head of the group) per column tile. e4m3 values are exact in f16;
// a query row is made exact there by a power of two that the score multiplies back. Softmax in fp32 with
// running maxima. O^T += V^T P^T: V^T comes from transposed 8x8 loads of byte pairs, P^T from
// transposing the probabilities' registers (movmatrix).
//
// The value scale differs between blocks, so it cannot be taken out of the sum. A warp holds O in a
// unit 2^U next to the scales it meets: the matrix instruction takes p = 2^(x - m) times
// c = 2^14 s_v / 2^U, and where a block's scale leaves [2^(U-6), 2^(U+1)) the unit moves to it and O is
// multiplied by the power of two between them. So what a probability loses in f16 goes by the
// probability alone, whatever scales (of blocks whose codes may all be 0) stand beside its own: 11
// bits down to 2^-22 of the row's largest (2^-14 in f16, c at least 2^8), absolutely 2^-33 of the
// largest below that. The unit stays within 2^64 of the largest scale seen (O must not overflow in
// fp32: 2^15 2^9 a term and up to 2^30 terms). l = sum 2^(x - m) stays in fp32, and out = (O / l) 2^(U - 14).
//
// Short caches take the same walk in another frame: a cluster of CTAs per pair, joined through
// distributed shared memory in one launch (the rule and its figures are in nk_attention_decode_q8).
//
// A pair covered by one CTA is written directly; otherwise its CTAs write (m, U, l, O) of their
// part, and a second launch adds the parts in order of their slots, its rows spread over the
// GPU; it works out where its parts lie before it waits for the first (20.5 -> 18.8 us at five
// sequences of 3000 with 32 query rows). (Measured: the last CTA of a pair adding the parts in the first launch instead takes
// 11.2 us where the two launches took 8.5, at one sequence of 1024 slots, and 60 where they took
// 30 at five of 3000 with 32 query rows: one CTA walks through all rows of the pair.)
//
// Measured, 8 kv heads (us, all launches; in brackets the cache's bytes at 6456 GB/s): two
// sequences of 128k slots 85.3 [83.2], 6.3 TB/s; 16 ragged ones of up to 8192 slots 31.4 [22.0]; one
// of 1024 slots (a cluster per pair) 5.1 [0.3]; five of up to 2999, four tokens x 64 heads, 18.3
// [2.8]. Long caches stream at the copy rate; the fixed part (first bytes, join, two launches) is
// some 4 to 6 us; many query rows are bound by the conversions and the matrix instructions (issue
// slots 45% busy at 12 warps an SM).
// ---------------------------------------------------------------------------------------
constexpr int kQ8Unit = 64;                 // slots per unit, 16 per warp
constexpr int kQ8AttnThreads = 128;
constexpr int kQ8Stages = 2;                // units in flight per warp (with four, an SM has no room for
                                            // the next launch's CTAs: 2 x 128k slots 86 -> 101 us)
constexpr int kQ8WarpStage = 2 * 16 * 128;  // K and V rows of 16 slots
constexpr int kQ8Ring = kQ8Stages * 4 * kQ8WarpStage;         // 32 KB
constexpr int kQ8OPitch = kHeadDim + 4;      // floats; spreads a warp's rows over the banks
__host__ __device__ constexpr int q8_o_bytes(int nt) { return 4 * 8 * nt * kQ8OPitch * 4; }
// the ring (or, once it is idle, the warps' sums), then each stage's two scales
__host__ __device__ constexpr int q8_scale_off(int nt) {
    return kQ8Ring > q8_o_bytes(nt) ? kQ8Ring : q8_o_bytes(nt);
}
__host__ __device__ constexpr int q8_attn_smem(int nt) { return q8_scale_off(nt) + 4 * kQ8Stages * 8; }
constexpr int kQ8MaxGrid = 148 * 4;
constexpr int kQ8PartFloats = kHeadDim + 4; // O, then m, U, l
constexpr int kQ8Shift = 14;                // c of a scale in the unit's own binade is in [2^14, 2^15)
constexpr int kQ8UnitBelow = 6;             // binades below the unit that a scale may lie in
constexpr int kQ8UnitRange = 64;            // and the unit below the largest scale seen
constexpr int kQ8LeastUnit = -100;          // also where a warp begins; the append's scales are 2^-64 or more
constexpr int kQ8MergeWarps = 8;
constexpr int kQ8MaxCluster = 8;

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}

struct Q8AttnArgs {
    const __nv_bfloat16* q;
    const uint8_t *k, *v;
    const float *ks, *vs;
    const int64_t* position; int per_sequence;
    __nv_bfloat16* out;
    float* part;                 // [grid][2][rows][kQ8PartFloats]
    int batch, tokens, hq, hkv, G, g_mul, capacity, lg_block, blocks;
    int rows, row_blocks;        // query rows of a CTA (8 NT), row blocks of a pair's T * G rows
    int grid;                    // CTAs of the first launch
    int lg_wpr;                  // merge: log2 of the warps that share a row
    int lg_cluster;              // short-cache form: log2 of the cluster's CTAs
    int64_t cb, ch, cs;
    float scale_log2;            // softmax scale times log2(e)
};

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t movm_t(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// Four e4m3 codes as two f16 pairs (codes 0, 1 and 2, 3).
__device__ __forceinline__ void e4m3x4_f16(uint32_t v, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t"
        "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(v));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 2^x by the special-function unit (relative error 2^-22, far below the 2^-11 of the f16
// probabilities; results below 2^-126 are 0).
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^k, 0 for k < -126.
__device__ __forceinline__ float q8_pow2(int k) {
    return __uint_as_float((uint32_t)(max(k, -127) + 127) << 23);
}
// Factor of a part with running maximum m where all parts have maximum M. A part that saw nothing
// (m = -inf) has sums of 0, or NaN if what it saw was NaN: 1 keeps both.
__device__ __forceinline__ float q8_weight(float m, float M) {
    return m == -INFINITY ? 1.f : ex2(m - M);
}

// Units of sequence b, of one (kv head, row block).
__device__ __forceinline__ int q8_seq_units(const Q8AttnArgs& a, int b) {
    const int64_t p = q8_position(a.position, a.per_sequence, b, a.tokens, a.capacity);
    return p < 0 ? 0 : ((int)p + a.tokens + kQ8Unit - 1) / kQ8Unit;
}

// The partition of U units over G <= U CTAs, q = U / G or one more each, and its inverse.
struct Q8Split {
    uint32_t q, r;
    __device__ Q8Split(uint32_t U, uint32_t G) : q(U / G), r(U - U / G * G) {}
    __device__ uint32_t begin(uint32_t c) const { return c * q + min(c, r); }
    __device__ uint32_t cta_of(uint32_t u) const {
        const uint32_t t = r * (q + 1);
        return u < t ? u / (q + 1) : r + (u - t) / q;
    }
};

// CL: the short-cache form. A cluster of 2, 4 or 8 CTAs shares one pair's units and joins through
// distributed shared memory: no partition over pairs, no partial sums in memory, no second launch.
template <int NT, bool CL>
__global__ void __launch_bounds__(kQ8AttnThreads, 3)
q8_attn_kernel(const Q8AttnArgs a) {
    extern __shared__ __align__(1024) uint8_t q8_smem[];
    __shared__ int s_end[CL ? 1 : NK_Q8_MAX_BATCH];     // running sum of the sequences' units
    __shared__ float s_stat[4][8 * NT][4];
    __shared__ uint2 s_q[NT > 1 ? NT * 8 * 32 : 1];     // Q^T operand, shared by the warps
    __shared__ float s_down[8 * NT];                    // and its rows' powers of two
    // in this order: the joining launch reads the positions ahead of its wait for this one, and so
    // must not start before what wrote them has finished
    griddep_wait();
    if (threadIdx.x == 0) griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const uint32_t per_b = a.hkv * a.row_blocks;        // pairs per sequence
    const int total_rows = a.tokens * a.G;
    uint32_t u = 0, u_end = 0, G = 0, U = 0;
    if (!CL && warp == 0) {  // 128 sequences at a time, their positions read together
        int base = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 128) {
            int x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = b0 + 32 * i + lane;
                x[i] = b < a.batch ? q8_seq_units(a, b) : 0;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int b = b0 + 32 * i + lane;
                if (b0 + 32 * i >= a.batch) break;
#pragma unroll
                for (int off = 1; off < 32; off <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, x[i], off);
                    if (lane >= off) x[i] += y;
                }
                x[i] += base;
                if (b < a.batch) s_end[b] = x[i];
                base = __shfl_sync(0xffffffffu, x[i], 31);
            }
        }
    } else if (blockIdx.x == 0 && warp == 1) {
        for (int b = lane; b < a.batch; b += 32)
            if (a.position[a.per_sequence ? b : 0] > (int64_t)a.capacity - a.tokens)
                atomicExch(&g_error, NK_ERR_RANGE);
    }
    if (!CL) {
        __syncthreads();
        U = s_end[a.batch - 1] * per_b;
        G = min((uint32_t)a.grid, U);                   // no CTA of the partition is empty
    }
    // rows of idle sequences are zero
    for (int b = blockIdx.x; b < a.batch; b += gridDim.x)
        if (CL ? q8_seq_units(a, b) == 0 : s_end[b] == (b > 0 ? s_end[b - 1] : 0)) {
            const int vecs = a.tokens * a.hq * (kHeadDim / 4);
            uint2* o = reinterpret_cast<uint2*>(a.out + (int64_t)b * a.tokens * a.hq * kHeadDim);
            for (int i = threadIdx.x; i < vecs; i += kQ8AttnThreads) o[i] = make_uint2(0u, 0u);
        }
    if (!CL) {
        if (blockIdx.x >= G) return;
        const Q8Split split(U, G);
        u = split.begin(blockIdx.x);
        u_end = split.begin(blockIdx.x + 1);
    }
    const uint32_t smem0 = static_cast<uint32_t>(__cvta_generic_to_shared(q8_smem));
    const uint32_t ring = smem0 + warp * (kQ8Stages * kQ8WarpStage);
    const uint32_t s_scale = smem0 + q8_scale_off(NT) + warp * (kQ8Stages * 8);

    do {
        // the pair of unit u: sequence b, kv head h, row block rb; its units [p0, p0 + n), of which
        // this CTA takes [c0, c1)
        int b, c0, c1;
        uint32_t n, pr, p0 = 0;
        if (CL) {
            const uint32_t pair = blockIdx.x >> a.lg_cluster;
            const uint32_t rank = blockIdx.x - (pair << a.lg_cluster);
            b = pair / per_b;
            pr = pair - b * per_b;
            n = q8_seq_units(a, b);
            if (n == 0) return;  // (the whole cluster)
            c0 = n * rank >> a.lg_cluster;
            c1 = n * (rank + 1) >> a.lg_cluster;
        } else {
            int lo = 0, hi = a.batch - 1;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (s_end[mid] * per_b > u) hi = mid; else lo = mid + 1;
            }
            b = lo;
            const int first = b > 0 ? s_end[b - 1] : 0;
            const uint32_t before = first * per_b;
            n = s_end[b] - first;
            pr = (u - before) / n;
            p0 = before + pr * n;
            c0 = u - p0;
            c1 = min(u_end, p0 + n) - p0;
        }
        const int h = pr / a.row_blocks, rb = pr - h * a.row_blocks;
        const int pos = (int)a.position[a.per_sequence ? b : 0];
        const int len = pos + a.tokens;

        // 16 slots of a unit: eight 16-byte pieces a row, piece c at c ^ (row & 7); this lane
        // copies piece lane % 8 of rows lane / 8 + 0, 4, 8, 12
        int slot = c0 * kQ8Unit + warp * 16 + (lane >> 3);
        const int64_t pair = (int64_t)b * a.cb + (int64_t)h * a.ch;
        const uint8_t* kp = a.k + pair + (int64_t)slot * a.cs + (lane & 7) * 16;
        const uint8_t* vp = a.v + pair + (int64_t)slot * a.cs + (lane & 7) * 16;
        const float* sp = (lane & 1 ? a.vs : a.ks) + ((int64_t)b * a.hkv + h) * a.blocks;
        const uint32_t d0 = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);
        const uint32_t d1 = d0 ^ (4 << 4);  // rows 4 on: (row & 7) has bit 2 set
        const int64_t row4 = 4 * a.cs, next = kQ8Unit * a.cs;
        int fill = c0;
        auto issue = [&]() {
            if (fill < c1) {
                const uint32_t st = fill & (kQ8Stages - 1);
                const uint32_t dst = ring + st * kQ8WarpStage;
                const int s0 = fill * kQ8Unit + warp * 16;
                if (s0 + 16 <= len) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t d = dst + (i & 1 ? d1 : d0) + i * 512;
                        cp_async<16>(d, kp + i * row4, true);
                        cp_async<16>(d + 16 * 128, vp + i * row4, true);
                    }
                } else {  // the sequence ends in this tile: what is past it reads as zero
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const bool ok = slot + 4 * i < len;
                        const uint32_t d = dst + (i & 1 ? d1 : d0) + i * 512;
                        cp_async<16>(d, ok ? kp + i * row4 : a.k, ok);
                        cp_async<16>(d + 16 * 128, ok ? vp + i * row4 : a.v, ok);
                    }
                }
                if (lane < 2 && s0 < len)
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                                     s_scale + st * 8 + lane * 4), "l"(sp + (s0 >> a.lg_block))
                                 : "memory");
                slot += kQ8Unit;
                kp += next;
                vp += next;
                ++fill;
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < kQ8Stages - 1; ++i) issue();

        // Q^T operand: column g of tile nt is query row 8 nt + g; dims 16 s + 4 t .. + 3 of step s.
        // With several tiles the warps take turns and share them through shared memory.
        uint2 qf[NT > 1 ? 1 : 8];
        float qs[NT][2];     // 2^-shift of rows 8 nt + 2t, + 1, times the softmax scale
        int last[NT][2];     // last slot those rows see, relative to pos (-1: no such row)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (NT > 1 && warp % NT != nt) continue;
            const int r = rb * a.rows + 8 * nt + g;
            const bool ok = r < total_rows;
            const int tok = ok ? r * a.g_mul >> 16 : 0, hh = ok ? r - tok * a.G : 0;
            const __nv_bfloat16* src =
                a.q + (((int64_t)b * a.tokens + tok) * a.hq + (int64_t)h * a.G + hh) * kHeadDim + 4 * t;
            uint2 w[8];
#pragma unroll
            for (int s = 0; s < 8; ++s)
                w[s] = ok ? *reinterpret_cast<const uint2*>(src + 16 * s) : make_uint2(0u, 0u);
            float m = 0.f;
#pragma unroll
            for (int s = 0; s < 8; ++s)
                m = fmaxf(m, fmaxf(fmaxf(fabsf(bf16lo(w[s].x)), fabsf(bf16hi(w[s].x))),
                                   fmaxf(fabsf(bf16lo(w[s].y)), fabsf(bf16hi(w[s].y)))));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            // largest magnitude to [2^12, 2^13): a bf16 value keeps its 8 bits down to 2^-29 of it
            int e = (int)(__float_as_uint(m) >> 23) - 127 - 12;
            e = min(max(e, -100), 115);
            const float up = __uint_as_float((uint32_t)(127 - e) << 23);
            const float down = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const uint2 f = make_uint2(pack_f16x2(bf16lo(w[s].x) * up, bf16hi(w[s].x) * up),
                                           pack_f16x2(bf16lo(w[s].y) * up, bf16hi(w[s].y) * up));
                if (NT == 1) qf[NT == 1 ? s : 0] = f;
                else s_q[(nt * 8 + s) * 32 + lane] = f;
            }
            if (NT == 1) {
                qs[0][0] = __shfl_sync(0xffffffffu, down, 8 * t);
                qs[0][1] = __shfl_sync(0xffffffffu, down, 8 * t + 4);
            } else if (t == 0) {
                s_down[8 * nt + g] = down;
            }
        }
        if (NT > 1) __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                qs[nt][i] = (NT == 1 ? qs[nt][i] : s_down[8 * nt + 2 * t + i]) * a.scale_log2;
                const int rr = rb * a.rows + 8 * nt + 2 * t + i;
                last[nt][i] = rr < total_rows ? rr * a.g_mul >> 16 : -1;
            }

        // m: running maximum of x; ref: what the exponents subtract (0 while nothing was seen)
        float m[NT][2], ref[NT][2], l[NT][2], o[8][NT][4];
        int unit = kQ8LeastUnit, unit_max = kQ8LeastUnit;  // U, and the largest scale's exponent so far
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            ref[nt][0] = ref[nt][1] = l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[d][nt][0] = o[d][nt][1] = o[d][nt][2] = o[d][nt][3] = 0.f;
        }

        // ldmatrix rows: matrix mi = lane / 8 = (slots half mi & 1, piece + (mi >> 1)), row lane % 8
        const uint32_t mrow = ((lane >> 3) & 1) * 8 + (lane & 7), mpiece = lane >> 4;
        const uint32_t mbase = ring + mrow * 128, mx7 = mrow & 7;
#pragma unroll 1
        for (int c = c0; c < c1; ++c) {
            issue();
            asm volatile("cp.async.wait_group %0;" ::"n"(kQ8Stages - 1) : "memory");
            __syncwarp();
            const uint32_t stage = c & (kQ8Stages - 1), st = mbase + stage * kQ8WarpStage;
            const int j0 = c * kQ8Unit + warp * 16;     // the warp's first slot of the unit
            if (j0 < len) {
                float k_scale, v_scale;
                asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];" : "=f"(k_scale), "=f"(v_scale)
                             : "r"(s_scale + stage * 8) : "memory");
                // the unit that this block asks for (one of scale 0 leaves it), ahead of the scores
                const int ve = max((int)(__float_as_uint(v_scale) >> 23 & 0xff) - 127, kQ8LeastUnit);
                const bool moves = v_scale != 0.f && (uint32_t)(unit - ve) > (uint32_t)kQ8UnitBelow;
                if (moves) unit_max = max(unit_max, ve);
                const int next_unit = moves ? max(ve, unit_max - kQ8UnitRange) : unit;
                const float moved = q8_pow2(unit - next_unit);
                const float up = v_scale * q8_pow2(kQ8Shift - next_unit);  // c
                unit = next_unit;
                float s[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
                for (int p = 0; p < 8; p += 2) {
                    uint32_t r[4];
                    ldsm_x4(st + (((p + mpiece) ^ mx7) << 4), r);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t a0, a1, a2, a3;
                        e4m3x4_f16(r[2 * k], a0, a2);
                        e4m3x4_f16(r[2 * k + 1], a1, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const uint2 f = NT == 1 ? qf[NT == 1 ? p + k : 0]
                                                    : s_q[(nt * 8 + p + k) * 32 + lane];
                            mma_f16(s[nt], a0, a1, a2, a3, f.x, f.y);
                        }
                    }
                }
                // scores of slots j0 + g and j0 + 8 + g against rows 2t, 2t + 1
                const bool all_seen = j0 + 15 <= pos;
                const bool big = k_scale > 0x1p64f;  // (s is below 2^30, qs 2^-103 or more)
                bool grown = moves;
                float mx[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)  // neither order's first product passes fp32 unless the score does
                        s[nt][e] = big ? s[nt][e] * qs[nt][e & 1] * k_scale : s[nt][e] * k_scale * qs[nt][e & 1];
                    if (!all_seen) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (j0 - pos + g + (e >> 1) * 8 > last[nt][e & 1]) s[nt][e] = -INFINITY;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float y = fmaxf(s[nt][e], s[nt][e + 2]);
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
                        y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
                        mx[nt][e] = y;
                        grown |= y > m[nt][e];
                    }
                }
                if (__any_sync(0xffffffffu, grown)) {  // a new maximum or unit: rescale the sums
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float al[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float mn = fmaxf(m[nt][e], mx[nt][e]);
                            ref[nt][e] = mn == -INFINITY ? 0.f : mn;
                            const float w = ex2(m[nt][e] - ref[nt][e]);
                            l[nt][e] *= w;
                            al[e] = w * moved;
                            m[nt][e] = mn;
                        }
#pragma unroll
                        for (int d = 0; d < 8; ++d) {
                            o[d][nt][0] *= al[0];
                            o[d][nt][1] *= al[1];
                            o[d][nt][2] *= al[0];
                            o[d][nt][3] *= al[1];
                        }
                    }
                }
                uint32_t pf[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float f[2][2];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float p0 = ex2(s[nt][e] - ref[nt][e]), p1 = ex2(s[nt][e + 2] - ref[nt][e]);
                        l[nt][e] += p0 + p1;
                        f[0][e] = p0 * up;
                        f[1][e] = p1 * up;
                    }
                    pf[nt][0] = movm_t(pack_f16x2(f[0][0], f[0][1]));
                    pf[nt][1] = movm_t(pack_f16x2(f[1][0], f[1][1]));
                }
                // A NaN among new tokens' values must not reach the rows before it (0 * NaN): it is
                // made 0 here and given to the sums of the rows that see it. Byte i of `first`: first
                // slot of the tile with one in element 4 lane + i, 0xff for none.
                if (!all_seen && a.tokens > 1) {
                    const uint32_t v0 = ring + stage * kQ8WarpStage + 16 * 128 + (lane & 3) * 4;
                    uint32_t first = 0xffffffffu;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const uint32_t at = v0 + j * 128 + (((lane >> 2) ^ (j & 7)) << 4);
                        uint32_t w;
                        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(at) : "memory");
                        const uint32_t bad = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
                        if (bad) {
                            const uint32_t bytes = (bad >> 7) * 0xffu;
                            const uint32_t open = ((first >> 7) & 0x01010101u) * 0xffu & bytes;
                            first = (first & ~open) | (j * 0x01010101u & open);
                            asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(w & ~bytes) : "memory");
                        }
                    }
                    if (__any_sync(0xffffffffu, first != 0xffffffffu)) {
#pragma unroll
                        for (int d = 0; d < 8; ++d) {
                            const uint32_t w = __shfl_sync(0xffffffffu, first, 4 * d + (g >> 1)) >> (16 * (g & 1));
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const int j = (w >> (8 * k)) & 0xff;
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int i = 0; i < 2; ++i)
                                        if (j < 16 && j0 + j - pos <= last[nt][i])
                                            o[d][nt][i + 2 * k] = __uint_as_float(0x7fc00000u);
                            }
                        }
                    }
                    __syncwarp();
                }
                // V^T: rows of tile d are dims 16 d + 2 g (first eight) and 16 d + 2 g + 1
#pragma unroll
                for (int p = 0; p < 8; p += 2) {
                    uint32_t r[4];
                    ldsm_x4_t(st + 16 * 128 + (((p + mpiece) ^ mx7) << 4), r);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t a0, a1, a2, a3;
                        e4m3x4_f16(__byte_perm(r[2 * k], 0u, 0x3120), a0, a1);
                        e4m3x4_f16(__byte_perm(r[2 * k + 1], 0u, 0x3120), a2, a3);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            mma_f16(o[p + k][nt], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
                    }
                }
            }
            __syncwarp();  // the stage may be refilled
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");

        // sums over the slots of a warp, then over the four warps
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float x = l[nt][i];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0)
                    *reinterpret_cast<float4*>(s_stat[warp][8 * nt + 2 * t + i]) =
                        make_float4(m[nt][i], (float)unit, x, 0.f);
            }
        __syncthreads();  // statistics are there; every warp is done with its ring
        float* s_o = reinterpret_cast<float*>(q8_smem);  // [warp][row][128]
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int d = 0; d < 8; ++d)
                    *reinterpret_cast<float2*>(s_o + (warp * 8 * NT + 8 * nt + 2 * t + i) * kQ8OPitch +
                                               16 * d + 2 * g) =
                        make_float2(o[d][nt][i], o[d][nt][i + 2]);
        __syncthreads();
        const bool whole = c0 == 0 && c1 == (int)n;
        // the CTA's first segment can only start inside a pair (slot 0), and only its last can end
        // inside one that it starts (slot 1)
        float* part = a.part + ((int64_t)blockIdx.x * 2 + (c0 > 0 ? 0 : 1)) * a.rows * kQ8PartFloats;
        const int rows = min(8 * NT, total_rows - rb * a.rows);
        for (int r = warp; r < rows; r += 4) {
            float4 st[4];
            float M = -INFINITY, Y = kQ8LeastUnit;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                st[w] = *reinterpret_cast<const float4*>(s_stat[w][r]);
                M = fmaxf(M, st[w].x);
                Y = fmaxf(Y, st[w].y);
            }
            float L = 0.f;
            float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float p = q8_weight(st[w].x, M), f = p * ex2(st[w].y - Y);
                L += st[w].z * p;
                const float4 x = *reinterpret_cast<const float4*>(
                    s_o + (w * 8 * NT + r) * kQ8OPitch + 4 * lane);
                A.x = fmaf(x.x, f, A.x);
                A.y = fmaf(x.y, f, A.y);
                A.z = fmaf(x.z, f, A.z);
                A.w = fmaf(x.w, f, A.w);
            }
            if (CL) {  // over warp 0's sums and statistics of this row, which are used up
                __syncwarp();
                *reinterpret_cast<float4*>(s_o + r * kQ8OPitch + 4 * lane) = A;
                if (lane == 0) *reinterpret_cast<float4*>(s_stat[0][r]) = make_float4(M, Y, L, 0.f);
            } else if (whole) {
                const int rr = rb * a.rows + r, tok = rr * a.g_mul >> 16, hh = rr - tok * a.G;
                const float f = ex2(Y - kQ8Shift) / L;
                *reinterpret_cast<uint2*>(
                    a.out + (((int64_t)b * a.tokens + tok) * a.hq + (int64_t)h * a.G + hh) * kHeadDim +
                    4 * lane) = make_uint2(bf16_pair(A.x * f, A.y * f), bf16_pair(A.z * f, A.w * f));
            } else {
                float* p = part + r * kQ8PartFloats;
                *reinterpret_cast<float4*>(p + 4 * lane) = A;
                if (lane == 0) *reinterpret_cast<float4*>(p + kHeadDim) = make_float4(M, Y, L, 0.f);
            }
        }
        if (CL) {  // rows shared out among the cluster's warps, the CTAs' parts in order of their slots
            cluster_arrive();
            cluster_wait();
            const int C = 1 << a.lg_cluster;
            for (int r = (blockIdx.x & (C - 1)) * 4 + warp; r < rows; r += 4 * C) {
                const uint32_t oa = smem0 + (r * kQ8OPitch + 4 * lane) * 4;
                const uint32_t sa = static_cast<uint32_t>(__cvta_generic_to_shared(s_stat[0][r]));
                float4 x[kQ8MaxCluster], st[kQ8MaxCluster];
#pragma unroll
                for (int k = 0; k < kQ8MaxCluster; ++k) {
                    st[k] = k < C ? ld_cluster_f4(sa, k) : make_float4(-INFINITY, kQ8LeastUnit, 0.f, 0.f);
                    x[k] = k < C ? ld_cluster_f4(oa, k) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                float M = -INFINITY, Y = kQ8LeastUnit, L = 0.f;
                float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int k = 0; k < kQ8MaxCluster; ++k) {
                    M = fmaxf(M, st[k].x);
                    Y = fmaxf(Y, st[k].y);
                }
#pragma unroll
                for (int k = 0; k < kQ8MaxCluster; ++k) {
                    const float p = q8_weight(st[k].x, M), f = p * ex2(st[k].y - Y);
                    L += st[k].z * p;
                    A.x = fmaf(x[k].x, f, A.x);
                    A.y = fmaf(x[k].y, f, A.y);
                    A.z = fmaf(x[k].z, f, A.z);
                    A.w = fmaf(x[k].w, f, A.w);
                }
                const int rr = rb * a.rows + r, tok = rr * a.g_mul >> 16, hh = rr - tok * a.G;
                const float f = ex2(Y - kQ8Shift) / L;
                *reinterpret_cast<uint2*>(
                    a.out + (((int64_t)b * a.tokens + tok) * a.hq + (int64_t)h * a.G + hh) * kHeadDim +
                    4 * lane) = make_uint2(bf16_pair(A.x * f, A.y * f), bf16_pair(A.z * f, A.w * f));
            }
            cluster_arrive();  // no CTA leaves while another may still read its shared memory
            cluster_wait();
            return;
        }
        __syncthreads();  // the ring and the statistics may be written again
        u = p0 + c1;
    } while (u < u_end);
}

// 2^lg_wpr warps per query row: adds the parts of a pair that several CTAs share (each warp its
// share of the parts in order of their slots, then the warps in order). Lane l holds elements 4l .. 4l + 3 of the row.
__global__ void __launch_bounds__(32 * kQ8MergeWarps) q8_merge_kernel(const Q8AttnArgs a) {
    __shared__ float4 s_a[kQ8MergeWarps][32], s_st[kQ8MergeWarps];
    if (threadIdx.x == 0) griddep_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int wpr = 1 << a.lg_wpr, sub = warp & (wpr - 1);
    const int b = blockIdx.y;
    const int row = blockIdx.x * (kQ8MergeWarps >> a.lg_wpr) + (warp >> a.lg_wpr);  // t * hq + head
    // units of the sequences before b, of b and of all
    uint32_t before = 0, all = 0;
#pragma unroll 4
    for (int i = lane; i < a.batch; i += 32) {
        const uint32_t x = q8_seq_units(a, i);
        all += x;
        before += i < b ? x : 0;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    const uint32_t n = q8_seq_units(a, b);
    const bool live = n > 0 && row < a.tokens * a.hq;  // (an idle sequence has no units to look up)
    const int tok = row / a.hq, head = row - tok * a.hq;
    const int h = head / a.G, rr = tok * a.G + head - h * a.G;
    const int rb = rr / a.rows, r = rr - rb * a.rows;
    const uint32_t per_b = a.hkv * a.row_blocks;
    uint2* out = reinterpret_cast<uint2*>(
        a.out + (((int64_t)b * a.tokens + tok) * a.hq + head) * kHeadDim + 4 * lane);
    const uint32_t U = all * per_b;
    const Q8Split split(U, max(min((uint32_t)a.grid, U), 1u));
    const uint32_t p0 = before * per_b + (h * a.row_blocks + rb) * n;
    const int cf = live ? split.cta_of(p0) : 0, cl = live ? split.cta_of(p0 + n - 1) : 0;
    const bool shared_pair = cf != cl;  // (else that CTA wrote the row, or there is no row)
    const int parts = cl - cf + 1;
    const int i0 = sub * parts >> a.lg_wpr, i1 = (sub + 1) * parts >> a.lg_wpr;
    griddep_wait();  // all of the above is on hand when the first launch ends
    if (n == 0) return;  // idle: the first launch wrote the zeros
    float M = -INFINITY, Y = kQ8LeastUnit, L = 0.f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    if (shared_pair) {
        for (int i = i0; i < i1; i += 4) {  // four parts' loads together
            float4 x[4], st[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int c = cf + min(i + k, i1 - 1);
                // the first CTA's part starts the pair (slot 1), the others' do not
                const float* p = a.part + (((int64_t)c * 2 + (c == cf ? 1 : 0)) * a.rows + r) * kQ8PartFloats;
                st[k] = *reinterpret_cast<const float4*>(p + kHeadDim);
                x[k] = *reinterpret_cast<const float4*>(p + 4 * lane);
            }
            float Mn = M, Yn = Y;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                Mn = fmaxf(Mn, st[k].x);
                Yn = fmaxf(Yn, st[k].y);
            }
            const float la = q8_weight(M, Mn), fa = la * ex2(Y - Yn);
            L *= la;
            A.x *= fa; A.y *= fa; A.z *= fa; A.w *= fa;
            M = Mn;
            Y = Yn;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (i + k >= i1) break;
                const float p = q8_weight(st[k].x, M), f = p * ex2(st[k].y - Y);
                L += st[k].z * p;
                A.x = fmaf(x[k].x, f, A.x);
                A.y = fmaf(x[k].y, f, A.y);
                A.z = fmaf(x[k].z, f, A.z);
                A.w = fmaf(x[k].w, f, A.w);
            }
        }
    }
    if (wpr > 1) {  // the row's warps, in order
        s_a[warp][lane] = A;
        if (lane == 0) s_st[warp] = make_float4(M, Y, L, 0.f);
        __syncthreads();
        if (sub != 0) return;
        for (int w = 0; w < wpr; ++w) {
            M = fmaxf(M, s_st[warp + w].x);
            Y = fmaxf(Y, s_st[warp + w].y);
        }
        L = 0.f;
        A = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < wpr; ++w) {
            const float4 st = s_st[warp + w], x = s_a[warp + w][lane];
            const float p = q8_weight(st.x, M), f = p * ex2(st.y - Y);
            L += st.z * p;
            A.x = fmaf(x.x, f, A.x);
            A.y = fmaf(x.y, f, A.y);
            A.z = fmaf(x.z, f, A.z);
            A.w = fmaf(x.w, f, A.w);
        }
    }
    if (!shared_pair) return;
    const float f = ex2(Y - kQ8Shift) / L;
    *out = make_uint2(bf16_pair(A.x * f, A.y * f), bf16_pair(A.z * f, A.w * f));
}

static bool q8_heads_ok(int tokens, int hq, int hkv) {
    return tokens >= 1 && tokens <= NK_Q8_MAX_TOKENS && hkv >= 1 && hq >= 1 && hq % hkv == 0 &&
           hq / hkv <= 16 && hq <= 4096;
}
static bool q8_block_ok(int block) {
    return block == 16 || block == 32 || block == 64 || block == 128;
}
// Query rows of one CTA: one or two column tiles of eight. More rows take several CTAs, which read
// the cache again (from L2) and widen it again. Four tiles a CTA leave two CTAs an SM: measured (us, two
// tiles / four) 22.7 / 33.1 at 32 rows (five sequences of 2999 slots), 199 / 179 at 64 rows and 392 /
// 342 at 128 (16 of 8192), 25.1 / 20.3 at 128 (two of 2048). So two serve drafts of up to 32 rows a kv
// head, and lose 10 to 19% at 64 and more, where what costs is the widening either way.
static int q8_rows(int rows) { return rows <= 8 ? 8 : 16; }

// The short-cache form: one launch of a cluster per pair.
template <int NT>
static int q8_launch_cluster(const Q8AttnArgs& a, cudaStream_t s) {
    auto kernel = q8_attn_kernel<NT, true>;
    static bool ready[64] = {};  // per device: the kernel's shared-memory limit is raised
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return NK_ERR_CUDA;
    if (dev < 0 || dev >= 64) return NK_ERR_DEVICE;
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 q8_attn_smem(NT)) != cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 (int)cudaSharedmemCarveoutMaxShared) != cudaSuccess)
            return NK_ERR_CUDA;
        ready[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.batch * a.hkv * a.row_blocks) << a.lg_cluster);
    cfg.blockDim = dim3(kQ8AttnThreads);
    cfg.dynamicSmemBytes = q8_attn_smem(NT);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 1 << a.lg_cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, a) == cudaSuccess ? NK_OK : NK_ERR_CUDA;
}

template <int NT>
static int q8_launch_attn(Q8AttnArgs a, cudaStream_t s) {
    static int slots[64] = {};  // CTAs resident at once, per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return NK_ERR_CUDA;
    if (dev < 0 || dev >= 64) return NK_ERR_DEVICE;
    if (slots[dev] == 0) {
        int sms = 0, per_sm = 0;
        if (cudaFuncSetAttribute(q8_attn_kernel<NT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 q8_attn_smem(NT)) != cudaSuccess ||
            cudaFuncSetAttribute(q8_attn_kernel<NT, false>, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 (int)cudaSharedmemCarveoutMaxShared) != cudaSuccess ||
            cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, q8_attn_kernel<NT, false>,
                                                          kQ8AttnThreads, q8_attn_smem(NT)) !=
                cudaSuccess ||
            per_sm < 1)
            return NK_ERR_CUDA;
        slots[dev] = min(sms * per_sm, kQ8MaxGrid);
    }
    const int64_t pairs = (int64_t)a.batch * a.hkv * a.row_blocks;
    const int64_t most = (int64_t)((a.capacity + kQ8Unit - 1) / kQ8Unit) * pairs;
    a.grid = (int)min((int64_t)slots[dev], most);
    const int rc = launch_pdl_smem(q8_attn_kernel<NT, false>, dim3(a.grid), dim3(kQ8AttnThreads),
                                   (size_t)q8_attn_smem(NT), s, a);
    if (rc != NK_OK) return rc;
    // about grid / pairs parts to a row: up to eight warps share them, at least two each
    a.lg_wpr = 0;
    while (a.lg_wpr < 3 && (int64_t)a.grid > pairs * (4 << a.lg_wpr)) ++a.lg_wpr;
    const int per_cta = kQ8MergeWarps >> a.lg_wpr;
    return launch_pdl_smem(q8_merge_kernel, dim3((a.tokens * a.hq + per_cta - 1) / per_cta, a.batch),
                           dim3(32 * kQ8MergeWarps), 0, s, a);
}

static bool q8_cache_ok(const nk_q8_cache* c, int tokens, int q_heads) {
    return c->head_dim == kHeadDim && c->batch >= 1 && c->batch <= NK_Q8_MAX_BATCH &&
           q8_heads_ok(tokens, q_heads, c->kv_heads) && c->capacity >= 1 &&
           c->capacity <= kQ8MaxCapacity && tokens <= c->capacity && q8_block_ok(c->block) &&
           c->seq_stride >= c->head_dim;
}
static bool q8_cache_aligned(const nk_q8_cache* c) {
    return !((((uintptr_t)c->k_codes | (uintptr_t)c->v_codes) & 15u) ||
             (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3u) || c->batch_stride % 16 ||
             c->head_stride % 16 || c->seq_stride % 16);
}

}  // namespace nk

extern "C" int nk_qk_norm_rope_cache_q8(const void* qkv, int64_t ld_qkv, const void* q_norm,
                                        const void* k_norm, const void* cos_table,
                                        const void* sin_table, const int64_t* position,
                                        int per_sequence, void* q_out, const nk_q8_cache* c,
                                        int tokens, int q_heads, float eps, nk_stream_t stream) {
    using namespace nk;
    if (!qkv || !q_norm || !k_norm || !cos_table || !sin_table || !position || !q_out || !c ||
        !c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale)
        return NK_ERR_ARG;
    if (!q8_cache_ok(c, tokens, q_heads) ||
        ld_qkv < (int64_t)(q_heads + 2 * c->kv_heads) * kHeadDim)
        return NK_ERR_SHAPE;
    if ((((uintptr_t)qkv | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)cos_table |
          (uintptr_t)sin_table | (uintptr_t)position | (uintptr_t)q_out) & 7u) ||
        ld_qkv % 4 || !q8_cache_aligned(c))
        return NK_ERR_ALIGN;
    Q8AppendArgs a{};
    a.qkv = static_cast<const __nv_bfloat16*>(qkv);
    a.ld = ld_qkv;
    a.qn = static_cast<const __nv_bfloat16*>(q_norm);
    a.kn = static_cast<const __nv_bfloat16*>(k_norm);
    a.cos_t = static_cast<const __nv_bfloat16*>(cos_table);
    a.sin_t = static_cast<const __nv_bfloat16*>(sin_table);
    a.position = position;
    a.per_sequence = per_sequence != 0;
    a.q_out = static_cast<__nv_bfloat16*>(q_out);
    a.k = static_cast<uint8_t*>(c->k_codes);
    a.v = static_cast<uint8_t*>(c->v_codes);
    a.ks = c->k_scale;
    a.vs = c->v_scale;
    a.batch = c->batch;
    a.tokens = tokens;
    a.hq = q_heads;
    a.hkv = c->kv_heads;
    a.capacity = c->capacity;
    a.block = c->block;
    a.blocks = (c->capacity + c->block - 1) / c->block;
    a.cb = c->batch_stride;
    a.ch = c->head_stride;
    a.cs = c->seq_stride;
    a.eps = eps;
    const int touched = (tokens + c->block - 2) / c->block + 1;  // blocks that T tokens can touch
    // One query row per warp while that is at most five CTAs per SM, four rows beyond: measured
    // (one a warp / four) 4.2 / 5.1 us at 4096 query rows, 6.3 / 6.0 at 8192, 8.6 / 7.5 at 16384.
    const bool many = (int64_t)c->batch * tokens * q_heads > 5ll * kNumSMs * kQ8Warps;
    const int per_cta = kQ8Warps * (many ? 4 : 1);
    a.q_ctas = (tokens * q_heads + per_cta - 1) / per_cta;
    const dim3 grid(a.q_ctas + c->kv_heads * touched, c->batch), block(32 * kQ8Warps);
    return many ? launch_pdl_smem(q8_append_kernel<4>, grid, block, 0, (cudaStream_t)stream, a)
                : launch_pdl_smem(q8_append_kernel<1>, grid, block, 0, (cudaStream_t)stream, a);
}

extern "C" size_t nk_attention_q8_ws_bytes(int tokens, int q_heads, int kv_heads) {
    using namespace nk;
    if (!q8_heads_ok(tokens, q_heads, kv_heads)) return 0;
    return (size_t)kQ8MaxGrid * 2 * q8_rows(tokens * (q_heads / kv_heads)) * kQ8PartFloats *
           sizeof(float);
}

extern "C" int nk_attention_decode_q8(const void* q, const nk_q8_cache* c,
                                      const int64_t* position, int per_sequence, void* out,
                                      int tokens, int q_heads, float scale, void* ws,
                                      size_t ws_bytes, nk_stream_t stream) {
    using namespace nk;
    if (!q || !c || !c->k_codes || !c->v_codes || !c->k_scale || !c->v_scale || !position || !out)
        return NK_ERR_ARG;
    if (!q8_cache_ok(c, tokens, q_heads)) return NK_ERR_SHAPE;
    Q8AttnArgs a{};
    a.G = q_heads / c->kv_heads;
    a.rows = q8_rows(tokens * a.G);
    a.row_blocks = (tokens * a.G + a.rows - 1) / a.rows;
    // units of the whole launch are counted in 32 bits
    if ((int64_t)((c->capacity + kQ8Unit - 1) / kQ8Unit) * c->batch * c->kv_heads * a.row_blocks >
        (1 << 30))
        return NK_ERR_SHAPE;
    if (!ws || ws_bytes < nk_attention_q8_ws_bytes(tokens, q_heads, c->kv_heads))
        return NK_ERR_WORKSPACE;
    if ((((uintptr_t)q | (uintptr_t)position | (uintptr_t)out) & 7u) || ((uintptr_t)ws & 15u) ||
        !q8_cache_aligned(c))
        return NK_ERR_ALIGN;
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.k = static_cast<const uint8_t*>(c->k_codes);
    a.v = static_cast<const uint8_t*>(c->v_codes);
    a.ks = c->k_scale;
    a.vs = c->v_scale;
    a.position = position;
    a.per_sequence = per_sequence != 0;
    a.out = static_cast<__nv_bfloat16*>(out);
    a.part = static_cast<float*>(ws);
    a.batch = c->batch;
    a.tokens = tokens;
    a.hq = q_heads;
    a.hkv = c->kv_heads;
    a.capacity = c->capacity;
    a.lg_block = __builtin_ctz(c->block);
    a.g_mul = (65536 + a.G - 1) / a.G;  // r / G for the at most 256 rows of a pair
    a.blocks = (c->capacity + c->block - 1) / c->block;
    a.cb = c->batch_stride;
    a.ch = c->head_stride;
    a.cs = c->seq_stride;
    a.scale_log2 = scale * 1.4426950408889634f;
    cudaStream_t s = (cudaStream_t)stream;
    // The short-cache form with the largest cluster that leaves every CTA resident (384 of them, in
    // clusters, at three CTAs an SM), if a CTA then has at most 512 slots to walk. Measured (us, one
    // launch / two): 8 pairs 5.1 / 6.1 at 1024 slots, 9.3 / 9.7 at 4096, 11.6 / 11.5 at 6000; 64 pairs
    // (clusters of 4) 8.5 / 11.3 at 1024, 12.3 / 13.8 at 2048, 18.8 / 18.2 at 4096; 128 pairs (of 2)
    // 8.4 / 11.2 at 512, 12.1 / 13.5 at 1024, 18.8 / 18.4 at 2048; past one wave, 64 pairs in
    // clusters of 8, 16.0 / 13.8 at 2048.
    const int64_t pairs = (int64_t)a.batch * a.hkv * a.row_blocks;
    for (int lg = 3; lg > 0 && !a.lg_cluster; --lg)
        if (pairs << lg <= 384) a.lg_cluster = lg;
    const bool cluster = a.lg_cluster && a.capacity <= 512 << a.lg_cluster;
    if (a.rows == 8) return cluster ? q8_launch_cluster<1>(a, s) : q8_launch_attn<1>(a, s);
    return cluster ? q8_launch_cluster<2>(a, s) : q8_launch_attn<2>(a, s);
}
