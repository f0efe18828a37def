// Linears with 4-bit weights and group scales (nk_gemm_w4, include/nk_quant.h).
//
//   y[m, n] = bf16( sum_groups s[n, G] * ( sum_{k in G} (q[n, k] - z[n, G]) x[m, k] ) )
//
// The inner sum's operands are exact in bf16 (q - z is an integer in -15..15), so the tensor
// cores add exact products in fp32 and the group's scale multiplies that fp32 sum: nothing is
// rounded before the one rounding of y.
//
// What bounds it: at decode batches the weight bytes (half a byte each) over HBM, some 46 weights
// a clock and SM, each of which has to be widened. A 16-bit word 0x00vv is the bf16 number vv *
// 2^-133 (the format's subnormals and first binade are one straight line), so masking a word of
// codes leaves pairs q * 2^-133 or 16 q * 2^-133, and one fma.bf16x2 with 2^127 or 2^123 and -z
// 2^-6 makes them (q - z) 2^-6, exactly: nine instructions per eight codes. Shared memory could not
// take the widened weights (four times the stream again), tensor memory can: the weights are the
// MMA's A operand there (128 rows = 128 lanes), the tokens its B operand in shared memory.
//
// Measured in CUDA graphs (us; in brackets the weight bytes' time at 6456 GB/s, the copy rate):
//   N 24576, K 4096   M=1 16.1 [8.0], M=64 24.9 [8.3]     group 128
//   N 6144, K 4096    M=16 8.0 [2.1]                      group 64
//   N 4096, K 12288   M=8 11.6 [4.7]                      group 32 with zero points
//   N 1024, K 2048    M=1 3.4 [0.2]: the launch and one pass through the pipeline
// Per step of 128 x 128 the eight MMAs take some 256 cycles (each reads 4 KB of A from tensor
// memory at 128 bytes a cycle), and a step of a CTA 450 to 500, with its barriers. So what bounds
// the wide shapes is the time per step on the SMs that hold two CTAs while others hold one (192
// row tiles on 148 SMs), the narrow ones the fixed parts (some 3 us: launch, first bytes, the
// cluster's sum). Against this library's bf16 linear (30.8 us at N 24576, K 4096, M=1) it is ahead up
// to 64 tokens (24.3 against 36.6 at group 128, 31.5 at 64) but for groups of 32 (45.4 at 64 tokens), and
// behind from some 128 on, as the weights are widened again for every 64: at M=128, 37.5, 48.9 and 70.8
// us (groups 128, 64, 32) against 41.8; at 256, 70, 91 and 130 against 67.5. On mma.sync, with the weights widened in registers, the same cases took 14.2
// (M=1), 75 (M=64), 12 and 19 us.
//
// A CTA takes 128 weight rows and a range of K steps (128 wide). Its warps:
//   0      lane 0 streams codes, scales and zero points of each step (one contiguous 8 KB piece
//          and two small ones) through a ring of bulk copies
//   1      lane 0 issues the MMAs: 8 per step, the accumulator started anew for each group
//   2      lane 0 brings each step's activations into shared memory (TMA, 128-byte swizzled); rows
//          that TMA cannot take are copied by warps 2 and 3
//   fold   (4 warps, 8 for 64 tokens) take each group's sums out of tensor memory, multiply by the
//          row's scale and add, in fp32 registers (one thread = one weight row)
//   widen  (8 warps, 4 for 64 tokens) turn a step's codes into the A operand (one thread = one row)
// Two CTAs share an SM. Where there are few rows, CTAs of a cluster share them and split K; their
// fp32 sums are added in rank order through distributed shared memory, after tensor memory is
// given back (so no CTA that holds some ever waits for another). No workspace, and no order of
// additions that changes between runs.
//
// Every mbarrier wait is bounded: on expiry the thread records NK_ERR_TIMEOUT in the device error
// word, its role ends, and the CTA drains its copies and MMAs (bounded), stores nothing, frees
// its tensor memory and exits. In a cluster no CTA stores anything of the tile then: its sum lacks a part.
#include <atomic>

#include "nk_common.cuh"
#include "../../include/nk_quant.h"

namespace nk {

constexpr int kW4Threads = 512;
constexpr int kW4MaxCluster = 8;
constexpr int kW4Rows = 128;
constexpr int kW4StepBytes = kW4Rows * 64;  // codes of one step

struct W4Args {
    const __nv_bfloat16* x; int64_t ldx;
    const uint8_t* codes;
    const uint8_t* scales;
    const uint8_t* zeros;
    __nv_bfloat16* y; int64_t ldy;
    int M, N, K;
    int KB;                       // K steps of 128
    int wide_x;                   // x rows are 16-byte aligned: TMA reads them
    int withhold;                 // failure-detection tests only (nk_test_withhold_w4), else -1
};

// CTA that the next launch's last step is withheld in; consumed by that launch.
static std::atomic<int> g_withhold_w4{-1};

template <int NT, int NG>
struct W4Smem {
    static constexpr int kScale = NG * kW4Rows * 2, kZero = NG * kW4Rows;
    static constexpr int kW = kW4StepBytes + kScale + kZero;  // one step of weights
    static constexpr int kX = NT * 256;                       // one step of activations: two boxes
    static constexpr int kXStages = NT == 16 ? 12 : (NT == 32 ? 6 : 4);
    static constexpr int kBudget = 112 * 1024;                // two CTAs per SM
    static constexpr int kFit = (kBudget - 2048 - kXStages * kX) / kW;
    static constexpr int kWStages = kFit > 8 ? 8 : kFit;
    static constexpr int kAccs = NT == 16 ? 8 : (NT == 32 ? 4 : 2);  // accumulators in tensor memory
    static constexpr int kTmemA = 2 * 64;                     // two A buffers of 64 columns
    static constexpr int kTmemCols = 256;
    // Where the accumulators hold two steps' groups, the fold warps take a step's groups together,
    // and their release of it is one of the arrivals that a later step's MMAs wait for; else they
    // take each group as it is summed, and the MMAs wait for each accumulator.
    static constexpr bool kStepRelease = kAccs >= 2 * NG;
    static constexpr int kLag = kAccs / NG;                   // steps from a release to its reuse
    static constexpr int kGroupBars = kAccs > 4 ? kAccs : 4;  // group barriers (see the kernel)
    static constexpr int kWOff = kXStages * kX;
    static constexpr int kBarOff = kWOff + kWStages * kW;
    static constexpr int kBars = 2 * kWStages + 2 * kXStages + kGroupBars + kAccs + 1;
    static constexpr int kMiscOff = kBarOff + kBars * 8;
    static constexpr int kAlloc = kMiscOff + 16 + 1024;       // slack to align the base to 1 KB
    static constexpr int kFoldHalves = NT <= 32 ? 1 : 2;      // fold warps per lane quarter
    static constexpr int kWidenSets = NT <= 32 ? 2 : 1;       // sets of four widening warps
    static_assert(kTmemA + kAccs * NT <= kTmemCols, "tensor memory");
    static_assert(kAccs <= kGroupBars && NG - 1 <= kGroupBars, "group barriers");
    static_assert(NT * kW4Rows * 4 <= kWOff, "the sums must fit over the activations");
    static_assert(4 + 4 * kFoldHalves + 4 * kWidenSets == kW4Threads / 32, "roles");
    static_assert(kW % 128 == 0 && kX % 1024 == 0 && kWStages >= 4, "ring layout");
};

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
__device__ __forceinline__ void st_cluster_u32(uint32_t saddr, uint32_t rank, uint32_t v) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t saddr, uint32_t rank) {
    uint32_t a;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a) : "memory");
    return v;
}

// Bulk copy into this CTA's shared memory, lines marked to leave L2 first (weights are read once).
__device__ __forceinline__ void bulk_load_hint(uint32_t dst, const void* src, uint32_t bytes,
                                               uint32_t bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
                 " [%0], [%1], %2, [%3], %4;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)),
                 "r"(bytes), "r"(bar), "l"(policy) : "memory");
}

// D[128 rows, N tokens] (+)= A[128 rows, 16] in tensor memory x B in shared memory.
__device__ __forceinline__ void tc_mma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc,
                                          uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 lanes x 8 consecutive columns of tensor memory -> 8 registers per thread, there after
// tcgen05.wait::ld; loaded() keeps uses of them behind that wait.
__device__ __forceinline__ void tmem_ld8_async(uint32_t taddr, float (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]),
                   "=f"(v[6]), "=f"(v[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void loaded(float (&v)[8]) {
    asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]),
                      "+f"(v[6]), "+f"(v[7])::"memory");
}

// 16 registers per thread -> 32 lanes x 16 consecutive 32-bit columns of tensor memory.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
        " {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
        "r"(r[15])
        : "memory");
}

// Wait for the phase with the given parity, for two seconds at most (then false, error recorded).
__device__ __forceinline__ bool w4_wait(uint32_t bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_ns();
    do {
#pragma unroll 1
        for (int i = 0; i < 64; ++i)
            if (mbar_try_wait(bar, parity)) return true;
    } while (global_ns() - t0 < 2000000000ull);
    atomicExch(&g_error, NK_ERR_TIMEOUT);
    return false;
}

__device__ __forceinline__ bool elect_one() {  // true in one lane of the converged warp
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(p));
    return p != 0;
}

// Codes at bits 0..3 (HI = 0) or 4..7 (HI = 1) of the word's halves as bf16 pairs
// (q - z) 2^-6; zc: -z 2^-6 in both halves.
template <int HI>
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, uint32_t zc) {
    uint32_t r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;"
        : "=r"(r)
        : "r"(word & (HI ? 0x00f000f0u : 0x000f000fu)), "r"(HI ? 0x7d007d00u : 0x7f007f00u), "r"(zc));
    return r;
}

__device__ __forceinline__ uint32_t w4_zero(uint32_t z) {  // -z 2^-6 as a bf16 pair
    return __byte_perm(__float_as_uint((float)z * -0x1p-6f), 0u, 0x3232);
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
    return r;
}

// 16 bytes of x to shared memory, the first `bytes` of them (0, 2, .. 16) from memory, the rest 0.
__device__ __forceinline__ void w4_stage16(uint32_t dst, const __nv_bfloat16* src, int bytes) {
    uint32_t v[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (2 * i < bytes) v[i >> 1] |= (uint32_t)__bfloat16_as_ushort(src[i]) << (16 * (i & 1));
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]) : "memory");
}

// NT: token tile (16, 32 or 64); NG: groups per K step; ZP: zero points given; FP16: scales are
// fp16, else bf16.
template <int NT, int NG, bool ZP, bool FP16>
__global__ void __launch_bounds__(kW4Threads, 2)
w4_kernel(const __grid_constant__ CUtensorMap tmap_x, const W4Args a) {
    using L = W4Smem<NT, NG>;
    constexpr int WS = L::kWStages, XS = L::kXStages, DB = L::kAccs;
    constexpr int FH = L::kFoldHalves, SETS = L::kWidenSets;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);

    // (the shuffles tell the compiler that a value is the same in every lane)
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int S = (int)cluster_size(), rank = (int)cluster_rank();
    const int tile = blockIdx.x / S;
    const int m0 = blockIdx.y * NT;
    const int mcount = min(NT, a.M - m0);
    const int k_begin = (int)((int64_t)rank * a.KB / S);
    const int n = (int)((int64_t)(rank + 1) * a.KB / S) - k_begin;  // steps, at least one
    const int loads = n - (a.withhold == (int)(blockIdx.y * gridDim.x + blockIdx.x));

    const uint32_t bar_full = base + L::kBarOff;         // weights of a step have landed
    const uint32_t bar_empty = bar_full + WS * 8;        // ... and are used up
    const uint32_t bar_ready = bar_empty + WS * 8;       // a step's operands (and accumulators) are ready
    const uint32_t bar_done = bar_ready + XS * 8;        // a step's MMAs have finished
    const uint32_t bar_group = bar_done + XS * 8;        // a group that is not its step's last is summed
    const uint32_t bar_free = bar_group + L::kGroupBars * 8;  // an accumulator may be overwritten
    const uint32_t bar_drain = bar_free + DB * 8;
    volatile uint32_t* misc = reinterpret_cast<volatile uint32_t*>(gbase + L::kMiscOff);
    volatile uint32_t* abort_flag = misc + 1;

    // Weights do not depend on the previous launch: the first steps' are on their way before tensor
    // memory is allocated and before the wait for that launch.
    const uint64_t policy = l2_evict_first_policy();
    auto load_step = [&](int i, int st) {
        const int64_t at = (int64_t)tile * a.KB + k_begin + i;
        const uint32_t dst = base + L::kWOff + st * L::kW, bar = bar_full + 8 * st;
        mbar_expect_tx(bar, kW4StepBytes + L::kScale + (ZP ? L::kZero : 0));
        bulk_load_hint(dst, a.codes + at * kW4StepBytes, kW4StepBytes, bar, policy);
        bulk_load_hint(dst + kW4StepBytes, a.scales + at * L::kScale, L::kScale, bar, policy);
        if (ZP)
            bulk_load_hint(dst + kW4StepBytes + L::kScale, a.zeros + at * L::kZero, L::kZero, bar,
                           policy);
    };
    if (warp == 0) {
        for (int i = lane; i < L::kBars; i += 32) {
            int count = 1;
            if (i >= WS && i < 2 * WS) count = 4 + 4 * FH;
            else if (i >= 2 * WS && i < 2 * WS + XS) count = 2 + 4 + (L::kStepRelease ? 4 * FH : 0);
            else if (i >= 2 * WS + 2 * XS + L::kGroupBars && i < L::kBars - 1) count = 4 * FH;
            mbar_init(bar_full + 8 * i, count);
        }
        if (lane == 0) *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0)
            for (int i = 0; i < min(loads, WS); ++i) load_step(i, i);
        __syncwarp();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32((const void*)misc)),
                     "r"((uint32_t)L::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, misc[0], 0);
    if (threadIdx.x == 0) griddep_launch_dependents();

    constexpr int kFold0 = 4, kWiden0 = 4 + 4 * FH;
    // A group's barrier completes once per round of the index that names it, and no second time
    // before the fold warps have seen the first: by accumulator where a round of the DB
    // accumulators is whole steps, else by the group's place in its step (the MMAs are never a
    // step of groups ahead of the fold warps there).
    constexpr bool kByAcc = DB >= NG;
    // A step's barriers come round after XS steps; the MMAs are never that far ahead.
    static_assert(XS >= DB && XS >= L::kLag && XS >= 3, "step barriers");
    if (warp == 0) {
        if (lane == 0) {
            int st = 0, ph = 0;
#pragma unroll 1
            for (int i = WS; i < loads; ++i) {
                if (!w4_wait(bar_empty + 8 * st, ph)) {
                    *abort_flag = 1u;
                    break;
                }
                load_step(i, st);
                if (++st == WS) {
                    st = 0;
                    ph ^= 1;
                }
            }
        }
    } else if (warp == 1) {
        // the whole warp walks the loop, so that descriptors stay in uniform registers
        constexpr uint32_t idesc = tc_idesc(kW4Rows, NT);
        const bool leader = elect_one();
        bool ok = true;
        int xs = 0, xph = 0, db = 0, dph = 1;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            ok = w4_wait(bar_ready + 8 * xs, xph);
            if (!ok) break;
            const uint64_t bdesc = sw128_desc(base + xs * L::kX);
            const uint32_t ta = tmem + (i & 1) * 64;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                if (!L::kStepRelease) {
                    ok = w4_wait(bar_free + 8 * db, dph);  // passes at once for the first DB groups
                    if (!ok) break;
                }
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int k = 0; k < 8 / NG; ++k) {
                        const int kk = j * (8 / NG) + k;
                        tc_mma_ts(tmem + L::kTmemA + db * NT, ta + kk * 8,
                                  bdesc + (((kk >> 2) * (NT * 128) + 32 * (kk & 3)) >> 4), idesc,
                                  k > 0);
                    }
                    if (j == NG - 1) tc_commit(bar_done + 8 * xs);
                    else if (!L::kStepRelease) tc_commit(bar_group + 8 * (kByAcc ? db : j));
                }
                __syncwarp();
                if (++db == DB) {
                    db = 0;
                    dph ^= 1;
                }
            }
            if (!ok) break;
            if (++xs == XS) {
                xs = 0;
                xph ^= 1;
            }
        }
        if (!ok) {
            *abort_flag = 1u;
            if (leader) tc_commit(bar_drain);
            __syncwarp();
            w4_wait(bar_drain, 0);
        }
    } else if (warp < kFold0 && a.wide_x) {
        if (warp == 2 && lane == 0) {
            griddep_wait();  // x is the previous launch's
            int xs = 0, ph = 1;
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                if (!w4_wait(bar_done + 8 * xs, ph)) {  // passes at once for the first XS steps
                    *abort_flag = 1u;
                    break;
                }
                const uint32_t bar = bar_ready + 8 * xs, dst = base + xs * L::kX;
                mbar_expect_tx(bar, L::kX);
                mbar_arrive(bar);  // (two arrivals, as the copying warps make)
                tma_load_2d(dst, &tmap_x, bar, (k_begin + i) * 128, m0);
                tma_load_2d(dst + NT * 128, &tmap_x, bar, (k_begin + i) * 128 + 64, m0);
                if (++xs == XS) {
                    xs = 0;
                    ph ^= 1;
                }
            }
        }
    } else if (warp < kFold0) {
        griddep_wait();
        // 64 threads: piece c (8 wide) of tokens r, r + 4, ..
        const int tid = threadIdx.x - 64, c = tid & 15, r = tid >> 4;
        const __nv_bfloat16* src = a.x + (int64_t)(m0 + r) * a.ldx + k_begin * 128 + c * 8;
        const uint32_t dst = base + (c >> 3) * (NT * 128) + r * 128;
        const uint32_t sw0 = ((c & 7) ^ r) << 4, sw1 = ((c & 7) ^ (r + 4)) << 4;
        const int64_t row4 = 4 * a.ldx;
        const int left = a.K - k_begin * 128 - c * 8;  // elements from the first step's piece on
        auto issue = [&](int i, int xs) {
            const int bytes = 2 * min(max(left - i * 128, 0), 8);
            const __nv_bfloat16* p = bytes > 0 ? src + i * 128 : a.x;
            const int64_t next = bytes > 0 ? row4 : 0;
            uint32_t d = dst + xs * L::kX;
            // columns of tokens past mcount stay as they are: they only reach sums never stored
#pragma unroll 1
            for (int m = r; m < mcount; m += 4, p += next, d += 512)
                w4_stage16(d + ((m & 4) ? sw1 : sw0), p, bytes);
        };
        bool ok = true;
        int xs = 0, ph = 1;
#pragma unroll 1
        for (int i = 0; i < n; ++i) {
            ok = __all_sync(0xffffffffu, w4_wait(bar_done + 8 * xs, ph));
            if (!ok) break;
            issue(i, xs);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_ready + 8 * xs);
            if (++xs == XS) {
                xs = 0;
                ph ^= 1;
            }
        }
        if (!ok) *abort_flag = 1u;
    } else if (warp < kWiden0) {
        const int quarter = warp & 3, half = (warp - kFold0) >> 2;
        const int row = quarter * 32 + lane;
        constexpr int COLS = NT / FH;
        const uint32_t taddr = tmem + L::kTmemA + ((uint32_t)(quarter * 32) << 16) + half * COLS;
        float acc[COLS];
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[c] = 0.f;
        bool ok = true;
        int st = 0, wph = 0, xs = 0, xph = 0, db = 0, dph = 0, later = L::kLag % XS;
        if (L::kStepRelease && lane == 0)  // the first steps find every accumulator free
            for (int i = 0; i < L::kLag; ++i) mbar_arrive(bar_ready + 8 * i);
#pragma unroll 1
        for (int i = 0; i < n && ok; ++i) {
            ok = __all_sync(0xffffffffu, w4_wait(bar_full + 8 * st, wph));
            if (!ok) break;
            const uint8_t* sc = gbase + L::kWOff + st * L::kW + kW4StepBytes + row * 2;
            float s[NG];
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const uint16_t bits = *reinterpret_cast<const uint16_t*>(sc + j * kW4Rows * 2);
                s[j] = FP16 ? __half2float(__ushort_as_half(bits))
                            : __uint_as_float((uint32_t)bits << 16);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_empty + 8 * st);
            if (++st == WS) {
                st = 0;
                wph ^= 1;
            }
            if constexpr (L::kStepRelease) {
                // the step's groups together: one wait and one round trip to tensor memory per eight
                // tokens, none for columns past the last token
                ok = __all_sync(0xffffffffu, w4_wait(bar_done + 8 * xs, xph));
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < COLS; c += 8) {
                    if (half * COLS + c >= mcount) break;
                    float v[NG][8];
#pragma unroll
                    for (int j = 0; j < NG; ++j) tmem_ld8_async(taddr + (db + j) * NT + c, v[j]);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < NG; ++j) {
                        loaded(v[j]);
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[c + e] = fmaf(s[j], v[j][e], acc[c + e]);
                    }
                }
                tc_fence_before();
                if ((db += NG) == DB) db = 0;
            } else {
#pragma unroll
                for (int j = 0; j < NG; ++j) {
                    ok = __all_sync(0xffffffffu,
                                    j == NG - 1 ? w4_wait(bar_done + 8 * xs, xph)
                                                : w4_wait(bar_group + 8 * (kByAcc ? db : j),
                                                          kByAcc ? dph : i & 1));
                    if (!ok) break;
                    tc_fence_after();
                    // (eight tokens a trip for the 64-token tile, whose registers are full, 16 for 32:
                    // measured 45.5 against 46.7 us, and 33.1 against 29.4; N 24576, K 4096, group 32)
                    if constexpr (FH == 2) {
#pragma unroll
                        for (int c = 0; c < COLS; c += 8) {
                            if (half * COLS + c >= mcount) break;
                            float v[8];
                            tmem_ld8_async(taddr + db * NT + c, v);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                            loaded(v);
#pragma unroll
                            for (int e = 0; e < 8; ++e) acc[c + e] = fmaf(s[j], v[e], acc[c + e]);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < COLS; c += 16) {
                            float v[16];
                            tmem_ld16(taddr + db * NT + c, v);
#pragma unroll
                            for (int e = 0; e < 16; ++e) acc[c + e] = fmaf(s[j], v[e], acc[c + e]);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar_free + 8 * db);
                    if (++db == DB) {
                        db = 0;
                        dph ^= 1;
                    }
                }
            }
            if (L::kStepRelease) {
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_ready + 8 * later);
                if (++later == XS) later = 0;
            }
            if (++xs == XS) {
                xs = 0;
                xph ^= 1;
            }
        }
        if (!ok) *abort_flag = 1u;
        // Every MMA has finished (the last group's sums are read), so the activations' ring may hold
        // the sums: [token][row], out of the codes' unit 2^-6.
        if (ok) {
            float* red = reinterpret_cast<float*>(gbase) + half * COLS * kW4Rows + row;
#pragma unroll
            for (int c = 0; c < COLS; ++c) red[c * kW4Rows] = acc[c] * 64.f;
        }
    } else {
        const int quarter = warp & 3, set = (warp - kWiden0) >> 2;
        const int row = quarter * 32 + lane;
        bool ok = true;
        int st = set, wph = 0, xs = XS - 2 + set, xph = 1;  // xs, xph: of step i - 2
        int ready = set;
        uint4 u[4];         // the step's codes of this row, and its groups' zero points: fetched
        uint32_t zc[NG];    // before the step before it is handed over
        auto fetch = [&]() {
            ok = __all_sync(0xffffffffu, w4_wait(bar_full + 8 * st, wph));
            if (!ok) return;
            const uint32_t w = L::kWOff + st * L::kW;
#pragma unroll
            for (int c = 0; c < 4; ++c) u[c] = lds128(base + w + c * 2048 + row * 16);
#pragma unroll
            for (int j = 0; j < NG; ++j)
                zc[j] = ZP ? w4_zero(gbase[w + kW4StepBytes + L::kScale + j * kW4Rows + row])
                           : 0xbe00be00u;
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_empty + 8 * st);
            if ((st += SETS) >= WS) {
                st -= WS;
                wph ^= 1;
            }
        };
        if (set < n) fetch();
#pragma unroll 1
        for (int i = set; i < n && ok; i += SETS) {
            // the MMAs of step i - 2 have read this buffer (passes at once for the first two)
            ok = __all_sync(0xffffffffu, w4_wait(bar_done + 8 * xs, xph));
            if (!ok) break;
            tc_fence_after();
            const uint32_t ta = tmem + ((uint32_t)(quarter * 32) << 16) + (i & 1) * 64;
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // 32 K elements: one group or part of one
                const uint32_t z = zc[c * NG / 4];
                const uint32_t word[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
                uint32_t r[16];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    r[4 * k] = w4_pair<0>(word[k], z);
                    r[4 * k + 1] = w4_pair<1>(word[k], z);
                    r[4 * k + 2] = w4_pair<0>(word[k] >> 8, z);
                    r[4 * k + 3] = w4_pair<1>(word[k] >> 8, z);
                }
                tmem_st16(ta + c * 16, r);
            }
            if (i + SETS < n) fetch();
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_ready + 8 * ready);
            if ((ready += SETS) >= XS) ready -= XS;
            if ((xs += SETS) >= XS) {
                xs -= XS;
                xph ^= 1;
            }
        }
        if (!ok) *abort_flag = 1u;
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_flag && threadIdx.x == 0) {  // copies in flight must land before the CTA goes: they
        const uint64_t t0 = global_ns();    // take microseconds, and get a millisecond
        while (global_ns() - t0 < 1000000ull) __nanosleep(1000);
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"((uint32_t)L::kTmemCols)
                     : "memory");
    }
    griddep_wait();  // outputs may still be read by the previous launch
    const float* red = reinterpret_cast<const float*>(gbase);
    const int count = mcount * kW4Rows, n0 = tile * kW4Rows;
    if (S == 1) {
        const bool good = *abort_flag == 0u;
        for (int e = threadIdx.x; e < count; e += kW4Threads) {
            const int m = e / kW4Rows, r = e % kW4Rows;
            if (good && n0 + r < a.N)
                a.y[(int64_t)(m0 + m) * a.ldy + n0 + r] = __float2bfloat16_rn(red[e]);
        }
        return;
    }
    // each CTA of the cluster adds its share of the elements, in rank order; one whose waits expired
    // has told the others
    if (*abort_flag && threadIdx.x < S) st_cluster_u32(base + L::kMiscOff + 4, threadIdx.x, 1u);
    cluster_arrive();
    cluster_wait();
    const bool good = *abort_flag == 0u;
    const int per = (count + S - 1) / S;
    for (int e = rank * per + threadIdx.x; e < min(count, (rank + 1) * per); e += kW4Threads) {
        float part[kW4MaxCluster];
#pragma unroll
        for (int s = 0; s < kW4MaxCluster; ++s)
            if (s < S) part[s] = ld_cluster_f32(base + 4 * e, s);
        float v = part[0];
#pragma unroll
        for (int s = 1; s < kW4MaxCluster; ++s)
            if (s < S) v += part[s];
        const int m = e / kW4Rows, r = e % kW4Rows;
        if (good && n0 + r < a.N)
            a.y[(int64_t)(m0 + m) * a.ldy + n0 + r] = __float2bfloat16_rn(v);
    }
    cluster_arrive();  // no CTA leaves while another may still read its shared memory
    cluster_wait();
}

template <int NT, int NG, bool ZP, bool FP16>
static int w4_launch(const W4Args& a, cudaStream_t s) {
    using L = W4Smem<NT, NG>;
    auto kernel = w4_kernel<NT, NG, ZP, FP16>;
    static bool ready[64] = {};  // per device: the kernel's shared-memory limit is raised
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return NK_ERR_CUDA;
    if (dev < 0 || dev >= 64) return NK_ERR_DEVICE;
    if (!ready[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlloc) !=
                cudaSuccess ||
            cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                 (int)cudaSharedmemCarveoutMaxShared) != cudaSuccess)
            return NK_ERR_CUDA;
        ready[dev] = true;
    }
    const int tiles = (a.N + kW4Rows - 1) / kW4Rows, mt = (a.M + NT - 1) / NT;
    // K is split while the CTAs still fit the GPU at once (clusters of up to eight pack into its
    // GPCs up to some 256 CTAs, two an SM; more wait for a second wave) and keep two steps each.
    // Measured: 48 tiles, S = 4 / 5 / 6 / 8 (288 and 384 CTAs): 7.9 / 8.1 / 12.6 / 11.6 us; 32 tiles,
    // S = 5 / 7 / 8: 16.1 / 13.6 / 12.7; 192 tiles, S = 1 / 2 / 3: 16.5 / 18.4 / 23.7.
    int S = (int)min((int64_t)kW4MaxCluster, (int64_t)256 / ((int64_t)tiles * mt));
    S = max(1, min(S, a.KB / 2));
    CUtensorMap mx{};
    if (a.wide_x && (get_encoder() != NK_OK || make_map(&mx, a.x, a.M, a.K, a.ldx, NT) != NK_OK))
        return NK_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * S, mt);
    cfg.blockDim = dim3(kW4Threads);
    cfg.dynamicSmemBytes = L::kAlloc;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = S;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = S > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, mx, a) == cudaSuccess ? NK_OK : NK_ERR_CUDA;
}

template <int NT, int NG>
static int w4_types(const W4Args& a, bool fp16, cudaStream_t s) {
    if (a.zeros)
        return fp16 ? w4_launch<NT, NG, true, true>(a, s) : w4_launch<NT, NG, true, false>(a, s);
    return fp16 ? w4_launch<NT, NG, false, true>(a, s) : w4_launch<NT, NG, false, false>(a, s);
}

template <int NT>
static int w4_dispatch(const W4Args& a, int group, bool fp16, cudaStream_t s) {
    switch (group) {
        case 32: return w4_types<NT, 4>(a, fp16, s);
        case 64: return w4_types<NT, 2>(a, fp16, s);
        default: return w4_types<NT, 1>(a, fp16, s);
    }
}

static bool w4_shape_ok(int N, int K) {
    return N >= 1 && K >= 1 && N <= (1 << 24) && K <= (1 << 24);
}
static bool w4_group_ok(int group) { return group == 32 || group == 64 || group == 128; }

}  // namespace nk

extern "C" size_t nk_w4_code_bytes(int N, int K) {
    if (!nk::w4_shape_ok(N, K)) return 0;
    return (size_t)((N + 127) / 128) * (size_t)((K + 127) / 128) * nk::kW4StepBytes;
}

extern "C" size_t nk_w4_scale_bytes(int N, int K, int group) {
    if (!nk::w4_shape_ok(N, K) || !nk::w4_group_ok(group)) return 0;
    return (size_t)((N + 127) / 128) * (size_t)((K + 127) / 128) * (128 / group) * 256;
}

extern "C" size_t nk_w4_zero_bytes(int N, int K, int group) {
    return nk_w4_scale_bytes(N, K, group) / 2;
}

extern "C" int nk_gemm_w4(const void* x, int64_t ldx, const nk_w4_weight* w, void* y, int64_t ldy,
                          int M, nk_stream_t stream) {
    using namespace nk;
    if (!x || !w || !w->codes || !w->scales || !y) return NK_ERR_ARG;
    const int N = w->N, K = w->K, group = w->group;
    if (w->scale_type != NK_W4_SCALE_BF16 && w->scale_type != NK_W4_SCALE_FP16) return NK_ERR_ARG;
    if (!w4_shape_ok(N, K) || !w4_group_ok(group) || M < 1 || M > (1 << 20) || ldx < K || ldy < N)
        return NK_ERR_SHAPE;
    if ((((uintptr_t)w->codes | (uintptr_t)w->scales | (uintptr_t)w->zeros) & 15u) ||
        (((uintptr_t)x | (uintptr_t)y) & 1u))
        return NK_ERR_ALIGN;
    W4Args a{};
    a.x = static_cast<const __nv_bfloat16*>(x);
    a.ldx = M == 1 ? (K + 7) / 8 * 8 : ldx;  // (one row: any stride)
    a.codes = static_cast<const uint8_t*>(w->codes);
    a.scales = static_cast<const uint8_t*>(w->scales);
    a.zeros = static_cast<const uint8_t*>(w->zeros);
    a.y = static_cast<__nv_bfloat16*>(y);
    a.ldy = ldy;
    a.M = M;
    a.N = N;
    a.K = K;
    a.KB = (K + 127) / 128;
    a.wide_x = ((uintptr_t)x & 15u) == 0 && a.ldx % 8 == 0;
    a.withhold = g_withhold_w4.exchange(-1);
    const bool fp16 = w->scale_type == NK_W4_SCALE_FP16;
    cudaStream_t s = (cudaStream_t)stream;
    // the narrowest token tile that holds M (a wider one costs MMA columns, fold registers and ring
    // stages: N 24576, K 4096 takes 16.1 us with 16 columns, 18.8 with 32, 24.8 with 64); beyond 64 tokens the
    // weights are read once per 64
    if (M <= 16) return w4_dispatch<16>(a, group, fp16, s);
    if (M <= 32) return w4_dispatch<32>(a, group, fp16, s);
    return w4_dispatch<64>(a, group, fp16, s);
}

extern "C" int nk_test_withhold_w4(int cta) {
    if (cta < -1) return NK_ERR_ARG;
    nk::g_withhold_w4.store(cta);
    return NK_OK;
}
