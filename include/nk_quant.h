/*
 * nk_quant.h — the quantised decode step of libnkgemm.so (sm_100a): linears with 4-bit weights,
 * and a KV cache held in 8 bits with the append that fills it and the attention that reads it.
 * They stand beside nk_gemm_bf16 (nk_gemm.h), nk_qk_norm_rope_cache_bf16 and
 * nk_attention_decode_bf16 (nk_decode.h), read a quarter and half of their bytes, and share
 * their conventions: device pointers, a cudaStream_t, 0 or NK_ERR_* returned before anything is
 * launched, no allocation, no host synchronisation, capture-safe, programmatic dependent launch.
 * The reference engine is bf16 throughout and has no counterpart of these.
 */
#ifndef NK_QUANT_H
#define NK_QUANT_H

#include "nk_gemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- 4-bit weights with group scales ------------------------------------------------------
 *
 *   y[m, n] = bf16_rne( sum_k x[m, k] * (q[n, k] - z[n, k / group]) * s[n, k / group] )
 *
 * q: 4-bit codes 0..15, s: bf16 or fp16 scales, z: zero points 0..15 (8 when there are none);
 * differences and products exact, sums in fp32, one rounding at the end.
 *
 * Storage, laid out once when the weights are loaded (KB = ceil(K / 128), NB = ceil(N / 128);
 * codes, scales and zero points past K or N are 0):
 *   codes:  [NB][KB][4][128] 16-byte pieces. Piece (i, b, c, r) holds row n = 128 i + r; its 32-bit
 *           word j (0..3) holds k = 128 b + 32 c + 8 j + 0..7: element 2 p in bits [4p, 4p + 4) and
 *           element 2 p + 1 in bits [16 + 4p, 20 + 4p), p = 0..3. A step of 128 rows by 128 K is 8 KB
 *           in one piece, and masking (word >> 4p) with 0x000f000f gives a pair of neighbours in
 *           the halves of a register.
 *   scales: [NB][KB][128 / group][128] 16-bit, row 128 i + r last.
 *   zeros:  the same order, bytes (NULL: every zero point is 8).
 */
#define NK_W4_SCALE_BF16 0
#define NK_W4_SCALE_FP16 1

/* A weight in this storage. codes, scales and zeros (or NULL) 16-byte aligned. */
typedef struct nk_w4_weight {
    const void* codes;
    const void* scales;
    const void* zeros;
    int32_t N, K;
    int32_t group;       /* 32, 64 or 128                       */
    int32_t scale_type;  /* NK_W4_SCALE_*                       */
} nk_w4_weight;

/* Bytes of the three arrays above (0 for arguments out of range: N, K >= 1, group 32, 64 or
 * 128). */
NK_API size_t nk_w4_code_bytes(int N, int K);
NK_API size_t nk_w4_scale_bytes(int N, int K, int group);
NK_API size_t nk_w4_zero_bytes(int N, int K, int group);

/* x: [M, K] bf16, row stride ldx >= K (elements); y: [M, N] bf16, row stride ldy >= N; both 2-byte
 * aligned (x 16-byte aligned with ldx % 8 == 0 is read by TMA, others by a slower copy); y not in x's
 * memory. Any M from 1 to 2^20; the weights are read and widened once per 64 rows of x, so past some
 * 128 rows (64 with groups of 32) nk_gemm_bf16 is the faster linear. No workspace. The weights must have been written before the launch that precedes this one on the
 * stream (they are read ahead of it); weights made at load time always are. */
NK_API int nk_gemm_w4(const void* x, int64_t ldx, const nk_w4_weight* w, void* y, int64_t ldy,
                      int M, nk_stream_t stream);

/* Failure-detection tests only: CTA `cta` of the next nk_gemm_w4 launch (tiles of 128 rows first, a
 * tile's CTAs side by side) never requests its last step's weights, so its waits for them expire (about 2 s).
 * The tile's outputs are not written, whichever of its CTAs they fall to, the launch returns, and
 * nk_device_error then reports NK_ERR_TIMEOUT. Consumed by that launch; -1 withholds nothing. */
NK_API int nk_test_withhold_w4(int cta);

/* ---- KV cache in 8 bits -------------------------------------------------------------------
 *
 * Keys and values are e4m3 codes (1 byte, finite range +-448) times a scale held for each
 * (sequence, kv head, block of `block` token slots), in fp32 [batch][kv_heads][ceil(capacity /
 * block)]. block is 16, 32, 64 or 128. Code arrays have unit stride along the 128 head elements
 * and any batch, head and token strides that are multiples of 16 (bytes); no two sequences,
 * heads, tokens or arrays share memory. capacity <= 2^30.
 *
 * `position` is a device int64 array: entry b (or entry 0 for every sequence when
 * per_sequence == 0) is the slot of sequence b's first new token; `tokens` (1..16) new tokens take
 * slots position .. position + tokens - 1. A negative position marks an idle sequence.
 * A position with position + tokens > capacity is treated as idle and sets the device error
 * word to NK_ERR_RANGE (nk_device_error).
 */
#define NK_Q8_MAX_TOKENS 16
#define NK_Q8_MAX_BATCH 1024

typedef struct nk_q8_cache {
    void* k_codes;         /* 16-byte aligned                             */
    void* v_codes;
    float* k_scale;
    float* v_scale;
    int32_t batch;         /* 1..1024                                     */
    int32_t kv_heads;
    int32_t head_dim;      /* 128                                         */
    int32_t capacity;      /* token slots, up to 2^30                     */
    int32_t block;         /* 16, 32, 64 or 128                           */
    int32_t reserved;
    int64_t batch_stride;  /* bytes, multiples of 16                      */
    int64_t head_stride;
    int64_t seq_stride;
} nk_q8_cache;

/* Per-head RMSNorm and RoPE of the new tokens' query and key heads with the cast points of
 * nk_qk_norm_rope_cache_bf16; queries to q_out, keys and values appended to the cache. For each
 * block that the new tokens touch, with amax their largest finite magnitude
 * in it: scale = max(former scale if the block holds earlier tokens, smallest power of two
 * s >= 2^-64 with amax <= 448 s, 0 for amax = 0). When the scale rises, the earlier tokens' codes c
 * become e4m3_rne(c * former / new); new codes are e4m3_rne(value / scale), NaN for a value
 * that is not finite. Slots past the new tokens, and everything of an idle sequence (its q_out
 * rows included), are left as they are.
 *   qkv: [batch * tokens, (q_heads + 2 kv_heads) * 128] bf16, row stride ld_qkv, row b * tokens + t
 *   q_out: [batch * tokens, q_heads * 128] bf16, not in qkv's memory
 *   q_norm, k_norm: [128]; cos, sin: [capacity, 128]
 * bf16 pointers 8-byte aligned and ld_qkv a multiple of 4. */
NK_API int nk_qk_norm_rope_cache_q8(const void* qkv, int64_t ld_qkv, const void* q_norm,
                                    const void* k_norm, const void* cos_table,
                                    const void* sin_table, const int64_t* position,
                                    int per_sequence, void* q_out, const nk_q8_cache* cache,
                                    int tokens, int q_heads, float eps, nk_stream_t stream);

/* Workspace bytes of nk_attention_decode_q8, whatever the batch and capacity (0: out of range).
 * It needs no initialisation. One workspace serves any sequence of ordered calls with up to as
 * many tokens; calls that may overlap on the GPU (streams, graphs) need one each. */
NK_API size_t nk_attention_q8_ws_bytes(int tokens, int q_heads, int kv_heads);

/* Grouped attention of the new tokens over the cache: query row (b, t, h) sees slots
 * 0 .. position + t of kv head h / (q_heads / kv_heads); rows of idle sequences are zero. Scores,
 * softmax and sums in fp32, the result rounded once to bf16. The matrix instructions take f16 on the way:
 *   probabilities rounded to 11 bits down to 2^-22 of the row's largest, to 2^-33 of it below that
 *   (blocks whose value scale is less than 2^-64 of the largest one lose more);
 *   a query row as it is, save that elements below 2^-29 of its largest (of 2^-88, where that is
 *   more) keep fewer bits, and may keep none below 2^-37 of it.
 * q, out: [batch * tokens, q_heads * 128] bf16, 8-byte aligned. q_heads / kv_heads between 1 and 16;
 * ws 16-byte aligned. */
NK_API int nk_attention_decode_q8(const void* q, const nk_q8_cache* cache,
                                  const int64_t* position, int per_sequence, void* out, int tokens,
                                  int q_heads, float scale, void* ws, size_t ws_bytes,
                                  nk_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* NK_QUANT_H */
