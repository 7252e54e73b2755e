/*
 * attn_decode.cu -- attention of one new token per sequence over the KV cache.
 * sm_100a, HBM-bound.
 *
 *   s_j = scale q . k_j,   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
 *
 * Every live row of K and V is read once for all the query heads of its cache
 * head: 4 G flops an element (G query heads to a cache head), 14 flops a byte
 * for the 7B heads in FP16, 28 in FP8 -- too many for the FP32 pipes beside the
 * conversions, few for the tensor cores. So both products run on mma.m16n8k16
 * with the KEYS (or the head's dims) as the 16 rows and the query heads as the 8
 * columns, S^T = K Q^T and O^T = V^T P^T: 7 of 8 columns carry work, where heads
 * as rows would waste nine of sixteen. (tcgen05 wants 64 rows and its operands
 * in shared memory behind barriers; at the rate HBM delivers, mma.sync is idle
 * nine tenths of the time.)
 *
 * No data crosses lanes through shared memory. A contraction may take its terms
 * in any order, so each lane's share of a fragment is chosen to be what 16-byte
 * loads of one row bring: of K, row `lane / 4` (and + 8) of the group, 16 bytes
 * at 16 (lane % 4) of each 64; of V, rows 2t, 2t+1, 2t+8, 2t+9 (t = lane % 4),
 * 16 bytes at 16 (lane / 4) of each 128, the pairs of rows interleaved by byte
 * permutes. A lane copies its own bytes with cp.async into its own 16-byte
 * column of the warp's ring and reads them back itself: waiting for its own
 * copies is all the synchronisation there is, warps never wait for one another,
 * and three stages of 8 KB a warp are in flight without holding registers.
 *
 * Work: the 64-position blocks of all (sequence, cache head) items in one line,
 * cut into as many equal parts as there are CTAs (two an SM). The cut depends on
 * the lengths alone, which every CTA sums up on the device. The CTA's four warps
 * take a quarter of each block. An item that a CTA holds whole is finished by
 * it; of one that is cut, each CTA leaves its part (running maximum, sum, output)
 * in scratch and a second small kernel joins them in CTA order.
 *
 * Precision: scores, maximum, sums and outputs in FP32. A weight e^(s - m) goes
 * to the tensor cores as a pair of FP16 values, rounded-down head plus rest, times 2^15: one
 * FP16 value alone would add an error as large as the output's own rounding.
 * Both are kept positive, so that an infinity in V stays one. For the rotated
 * formats the levels times a common factor become FP16 values within 9e-5 of
 * themselves (alpha below, found by trying factors in [1, 2); 1.6e-4 for the
 * 1.5-bit code words), the RMS of a key multiplies its score, the RMS of V the
 * weight, relative to a power of two that follows the largest RMS.
 */
#include "fp8_kv.cuh"
#include "tq_kv.cuh"
#include "vvb_launch.h"

#include <atomic>
#include <type_traits>

namespace vvb {

extern std::atomic<uint64_t> g_launches;

constexpr int kAttnPageShift = 6;
constexpr int kAttnWarps = 4;                   /* a quarter of a 64-position block each */
#ifndef VVB_ATTN_WAVES
#define VVB_ATTN_WAVES 1
#endif
constexpr int kAttnParts = VVB_ATTN_WAVES * 3 * 148;      /* parts the work is cut into, at most */
constexpr int kAttnJoinCtas = 2 * 148;
constexpr int kAttnItemCost = 1;                /* what beginning and ending an item costs, in blocks */
constexpr int kAttnJoinThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kWeightLog2 = 12.0f;            /* a weight of 1 is kept as 2^12 ... */
constexpr float kWeightTop = 15.0f;             /* ... and the maximum follows the scores once one passes 2^15 */
constexpr float kNoMax = -3e38f;

struct AttnArgs {
    const __half* q;
    __half* out;
    float* lse;                /* may be null */
    const uint8_t* k_store;
    const uint8_t* v_store;
    const __half* k_meta;      /* TurboQuant */
    const __half* v_meta;
    const int* block_table;    /* null: contiguous */
    const int* lens;
    int2* desc;                /* [kAttnParts] item that ends in this CTA and began in an earlier one, that CTA; or -1 */
    float2* part_ml;           /* [2 kAttnParts][heads of an item] maximum, sum */
    float4* part_o;            /* [2 kAttnParts][tiles][32] output, in the lanes' layout */
    int n_seqs, n_q, n_kv, n_slots, table_stride, len_add;
    int group, head_blocks;    /* query heads to a cache head, items a cache head is cut into */
    float scale2;              /* scale * log2(e) */
};

/* ---------------------------------------------------------------- formats */

/* What a lane copies of a group of 16 keys: KN units of KU bytes of each of its two K rows,
 * VN units of VU bytes of each of its four V rows. */
template <int FMT, int HD> struct AttnFmt {
    static constexpr int VEC = FMT == KV_RAW ? 2 * HD : HD;      /* bytes of a stored vector */
    static constexpr int KU = 16, KN = VEC / 64;
    static constexpr int VU = VEC >= 128 ? 16 : 8, VN = VEC >= 128 ? VEC / 128 : 1;
    static constexpr int META = 0, LUT = 0;
};
template <int HD> struct AttnFmt<KV_TQ4, HD> {
    static constexpr int VEC = 64, KU = 16, KN = 1, VU = 8, VN = 1, META = 4, LUT = 256;      /* two codes -> two levels */
};
template <int HD> struct AttnFmt<KV_TQ3, HD> {
    static constexpr int VEC = 48, KU = 4, KN = 3, VU = 4, VN = 2, META = 4, LUT = 64;
};
template <int HD> struct AttnFmt<KV_TQ2, HD> {
    static constexpr int VEC = 32, KU = 8, KN = 1, VU = 4, VN = 1, META = 4, LUT = 16;
};
template <int HD> struct AttnFmt<KV_TQ1_5, HD> {
    static constexpr int VEC = 24, KU = 4, KN = 2, VU = 4, VN = 2, META = 4, LUT = 8 + 128;   /* code -> pair; two keys' codes -> two pairs */
};

/* Factor that brings all the levels of a code book near FP16 values. */
template <int FMT> __host__ __device__ constexpr float attn_alpha() {
    return FMT == KV_TQ4 ? 1.2162726f : FMT == KV_TQ3 ? 1.4423765f : FMT == KV_TQ2 ? 1.8130219f : FMT == KV_TQ1_5 ? 1.0849942f : 1.0f;
}

template <int FMT, int HD, int NT> struct AttnShape {
    using F = AttnFmt<FMT, HD>;
    static constexpr int K_BYTES = 2 * F::KU * F::KN, V_BYTES = 4 * F::VU * F::VN;
    static constexpr int LANE_BYTES = K_BYTES + V_BYTES + 4 * F::META;                        /* of a stage */
    static constexpr int CTAS = HD == 256 || NT == 2 ? 2 : 3;                                 /* an SM's, by registers and shared memory */
    static constexpr int STAGES = LANE_BYTES >= 256 ? 2 : kv_is_tq(FMT) ? 3 : 4;
    static constexpr int RING = 32 * LANE_BYTES * STAGES;                                     /* a warp's */
    static constexpr int TILES = HD / 16;                                                     /* 16-dim tiles of the output */
    static constexpr int MINE = NT * TILES / kAttnWarps;                                      /* of them a warp finishes, ... */
    static constexpr int PER_ROUND = 1, ROUNDS = MINE / PER_ROUND;                            /* ... so many in one round of the exchange */
    static constexpr int XCHG = kAttnWarps * (kAttnWarps - 1) * PER_ROUND * 32 * 16;
    static constexpr int LUT = F::LUT * 128;
    static constexpr int SMEM = LUT + kAttnWarps * RING + XCHG;       /* in this order */
};

/* ---------------------------------------------------------------- instructions */

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
/* BYTES of a row into shared memory at dst + AT; `some`: only n of them are read, the rest become zeros. */
template <int BYTES, int AT> __device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0 + %2], [%1], 16;" ::"r"(dst), "l"(src), "n"(AT) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0 + %3], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES), "n"(AT) : "memory");
}
template <int BYTES, int AT> __device__ __forceinline__ void cp_async_some(uint32_t dst, const void* src, int n) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0 + %3], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(AT) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0 + %4], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n), "n"(AT) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack2_rz(float a, float b) {       /* two halves, rounded toward zero; low half = a */
    uint32_t r;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ uint32_t hmax2_bits(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
/* Two outputs, and the log-sum-exp, from a head's sums (maximum and sum are those of weights times 2^12).
 * A sum of zero: no keys, or none with a score above -inf. */
__device__ __forceinline__ uint32_t attn_out(float a, float b, float sum) {
    const float r = 1.0f / sum;
    return sum == 0.0f ? 0u : pack2(a * r, b * r);
}
__device__ __forceinline__ float attn_lse(float top, float sum) {
    return sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}
/* Transpose of an 8 x 8 matrix of halves held as fragments. */
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <int FMT> __device__ __forceinline__ uint32_t fp8_pair(uint32_t two) {               /* two bytes -> two halves */
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, FMT == KV_E4M3 ? __NV_E4M3 : __NV_E5M2);
    return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(a));
    return r;
}
template <int UNIT, int AT> __device__ __forceinline__ void lds_unit(uint32_t a, uint32_t* w) {
    if constexpr (UNIT == 16)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a), "n"(AT));
    else if constexpr (UNIT == 8)
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2 + %3];" : "=r"(w[0]), "=r"(w[1]) : "r"(a), "n"(AT));
    else
        asm volatile("ld.shared.b32 %0, [%1 + %2];" : "=r"(w[0]) : "r"(a), "n"(AT));
}

extern __shared__ __align__(16) uint8_t attn_smem[];           /* the code table first: its address is then a constant */
/* Entry c / 128 of the code table, this lane's copy (c a multiple of 128 below the table's size). */
__device__ __forceinline__ uint32_t attn_lut(uint32_t c, uint32_t mask, uint32_t lane4, int from = 0) {
    return *reinterpret_cast<const uint32_t*>(attn_smem + from + ((c & mask) | lane4));
}

/* ---------------------------------------------------------------- code books */

__constant__ float c_lev4[16] = {tq_lev4(0), tq_lev4(1), tq_lev4(2), tq_lev4(3), tq_lev4(4), tq_lev4(5), tq_lev4(6), tq_lev4(7),
                                 tq_lev4(8), tq_lev4(9), tq_lev4(10), tq_lev4(11), tq_lev4(12), tq_lev4(13), tq_lev4(14), tq_lev4(15)};
__constant__ float c_lev3[8] = {tq_lev3(0), tq_lev3(1), tq_lev3(2), tq_lev3(3), tq_lev3(4), tq_lev3(5), tq_lev3(6), tq_lev3(7)};
__constant__ float c_lev2[4] = {tq_lev2(0), tq_lev2(1), tq_lev2(2), tq_lev2(3)};
__constant__ float c_vq15[16] = {tq_vq15(0), tq_vq15(1), tq_vq15(2), tq_vq15(3), tq_vq15(4), tq_vq15(5), tq_vq15(6), tq_vq15(7),
                                 tq_vq15(8), tq_vq15(9), tq_vq15(10), tq_vq15(11), tq_vq15(12), tq_vq15(13), tq_vq15(14), tq_vq15(15)};

/* Entry e of the table, one copy for each lane (a lane reads its own bank, whatever its codes are). */
template <int FMT> __device__ __forceinline__ uint32_t attn_lut_entry(int e) {
    constexpr float A = attn_alpha<FMT>();
    if constexpr (FMT == KV_TQ4) return pack2(c_lev4[e & 15] * A, c_lev4[e >> 4] * A);
    else if constexpr (FMT == KV_TQ3) return pack2(c_lev3[e & 7] * A, c_lev3[e >> 3] * A);
    else if constexpr (FMT == KV_TQ2) return pack2(c_lev2[e & 3] * A, c_lev2[e >> 2] * A);
    else {
        if (e < 8) return pack2(c_vq15[2 * e] * A, c_vq15[2 * e + 1] * A);
        const int c = (e - 8) & 63, i = (e - 8) >> 6;                     /* first, then second values of keys A, B */
        return pack2(c_vq15[2 * (c & 7) + i] * A, c_vq15[2 * (c >> 3) + i] * A);
    }
}

/* ---------------------------------------------------------------- fragments */

/* First dim of the 8 that words 4n .. 4n+3 of a lane's K row (as halves) hold. */
template <int FMT> __device__ __forceinline__ int attn_k_dim(int n, int t) {
    return FMT == KV_RAW ? 32 * n + 8 * t : kv_is_tq(FMT) ? 32 * t + 8 * n : 64 * (n >> 1) + 16 * t + 8 * (n & 1);
}
/* Dim of value 2 j (2 j + 1 follows) of a lane's V row. */
template <int FMT, int HD> __device__ __forceinline__ int attn_v_dim(int j, int g) {
    if (FMT == KV_RAW) return 64 * (j >> 2) + 8 * g + 2 * (j & 3);
    if (HD == 64) return 8 * g + 2 * j;
    return 128 * (j >> 3) + 16 * g + 2 * (j & 7);
}

/* A lane's K row as halves: word i holds dims attn_k_dim(i / 4) + 2 (i % 4), + 1. */
template <int FMT, int HD>
__device__ __forceinline__ void attn_k_words(const uint32_t* raw, uint32_t (&w)[HD / 8], uint32_t lane4) {
    if constexpr (FMT == KV_RAW) {
#pragma unroll
        for (int i = 0; i < HD / 8; i++) w[i] = raw[i];
    } else if constexpr (!kv_is_tq(FMT)) {
#pragma unroll
        for (int i = 0; i < HD / 16; i++) {
            w[2 * i] = fp8_pair<FMT>(raw[i] & 0xffffu);
            w[2 * i + 1] = fp8_pair<FMT>(raw[i] >> 16);
        }
    } else {
        constexpr int NB = FMT == KV_TQ4 ? 8 : FMT == KV_TQ3 ? 6 : FMT == KV_TQ2 ? 4 : 3;     /* bits of two dims */
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int bit = NB * i, at = bit & 31;
            uint32_t c;                                /* the code pair times 128 */
            if (at + NB > 32) c = (__funnelshift_r(raw[bit >> 5], raw[(bit >> 5) + 1], at) << 7);
            else c = at >= 7 ? raw[bit >> 5] >> (at - 7) : raw[bit >> 5] << (7 - at);
            w[i] = attn_lut(c, ((1u << NB) - 1u) << 7, lane4);
        }
    }
}

/* Two keys' V rows: x[e] = (key A, key B) at the lane's value e. */
template <int FMT, int HD>
__device__ __forceinline__ void attn_v_pairs(const uint32_t* a, const uint32_t* b, uint32_t (&x)[HD / 8], uint32_t lane4) {
    if constexpr (FMT == KV_RAW) {
#pragma unroll
        for (int i = 0; i < HD / 16; i++) {
            x[2 * i] = __byte_perm(a[i], b[i], 0x5410);
            x[2 * i + 1] = __byte_perm(a[i], b[i], 0x7632);
        }
    } else if constexpr (!kv_is_tq(FMT)) {
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            const uint32_t lo = __byte_perm(a[i], b[i], 0x5140), hi = __byte_perm(a[i], b[i], 0x7362);
            x[4 * i] = fp8_pair<FMT>(lo & 0xffffu);
            x[4 * i + 1] = fp8_pair<FMT>(lo >> 16);
            x[4 * i + 2] = fp8_pair<FMT>(hi & 0xffffu);
            x[4 * i + 3] = fp8_pair<FMT>(hi >> 16);
        }
    } else if constexpr (FMT == KV_TQ4) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t even = (a[i] & 0x0f0f0f0fu) | ((b[i] & 0x0f0f0f0fu) << 4);         /* dims 0, 2, 4, 6 of the eight */
            const uint32_t odd = ((a[i] >> 4) & 0x0f0f0f0fu) | (b[i] & 0xf0f0f0f0u);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int s = 8 * k - 7;
                x[8 * i + 2 * k] = attn_lut(s > 0 ? even >> s : even << -s, 0x7f80u, lane4);
                x[8 * i + 2 * k + 1] = attn_lut(s > 0 ? odd >> s : odd << -s, 0x7f80u, lane4);
            }
        }
    } else {
        constexpr int W = FMT == KV_TQ2 ? 2 : 3;       /* bits of a code */
        constexpr int N = FMT == KV_TQ1_5 ? 8 : 16;    /* codes of a lane's row; word 1 holds what word 0 does not */
#pragma unroll
        for (int e = 0; e < N; e++) {
            const int bit = W * e;
            const uint32_t ca = (bit + W <= 32 ? a[0] >> bit : bit >= 32 ? a[1] >> (bit - 32) : __funnelshift_r(a[0], a[1], bit)) & ((1u << W) - 1u);
            const uint32_t cb = (bit + W <= 32 ? b[0] >> bit : bit >= 32 ? b[1] >> (bit - 32) : __funnelshift_r(b[0], b[1], bit)) & ((1u << W) - 1u);
            const uint32_t c = (ca | (cb << W)) << 7;
            if constexpr (FMT == KV_TQ1_5) {
                x[2 * e] = attn_lut(c, ~0u, lane4, 8 * 128);
                x[2 * e + 1] = attn_lut(c, ~0u, lane4, (8 + 64) * 128);
            } else {
                x[e] = attn_lut(c, ~0u, lane4);
            }
        }
    }
}

/* Where in a vector a lane's K and V bytes begin, unit n. */
template <int FMT, int HD> __device__ __forceinline__ int attn_k_byte(int n, int t) {
    if (FMT == KV_TQ3) return 12 * t + 4 * n;
    if (FMT == KV_TQ2) return 8 * t;
    if (FMT == KV_TQ1_5) return ((6 * t) & ~3) + 4 * n;
    return 64 * n + 16 * t;                            /* TQ4: n = 0 */
}
template <int FMT, int HD> __device__ __forceinline__ int attn_v_byte(int n, int g) {
    if (FMT == KV_TQ3) return ((6 * g) & ~3) + 4 * n;
    if (FMT == KV_TQ2) return 4 * g;
    if (FMT == KV_TQ1_5) return ((3 * g) & ~3) + (g < 7 ? 4 * n : 0);      /* the last lane's three bytes lie in one word */
    return AttnFmt<FMT, HD>::VU == 16 ? 128 * n + 16 * g : 8 * g;
}
/* The odd start of a lane's bits in those words. */
template <int FMT> __device__ __forceinline__ int attn_k_shift(int t) { return FMT == KV_TQ1_5 ? 8 * (6 * t - ((6 * t) & ~3)) : 0; }
template <int FMT> __device__ __forceinline__ int attn_v_shift(int g) {
    if (FMT == KV_TQ3) return 8 * ((6 * g) & 3);
    if (FMT == KV_TQ1_5) return 8 * ((3 * g) & 3);
    return 0;
}

/* ---------------------------------------------------------------- work */

/* Number of keys of sequence b. */
__device__ __forceinline__ int attn_keys(const AttnArgs& A, int b) {
    const long long cap = A.block_table != nullptr ? (long long)A.table_stride << kAttnPageShift : (long long)A.table_stride;
    const long long n = (long long)__ldg(A.lens + b) + A.len_add;
    return (int)min(min(max(n, 0ll), cap), 0x7fffffc0ll);
}
__device__ __forceinline__ int attn_blocks(int n) { return (n + 63) >> kAttnPageShift; }
__device__ __forceinline__ int attn_places(int n) { return n > 0 ? attn_blocks(n) + kAttnItemCost : 0; }
/* f(0), f(1) .. f(N - 1) with the number as a type. */
template <int N> struct AttnUnits {
    template <typename Fn> static __device__ __forceinline__ void each(Fn&& f) {
        AttnUnits<N - 1>::each(f);
        f(std::integral_constant<int, N - 1>());
    }
};
template <> struct AttnUnits<0> {
    template <typename Fn> static __device__ __forceinline__ void each(Fn&&) {}
};

/* A place in the line of blocks: block blk of nb of item h (cache head x head block) of sequence b. */
struct AttnAt {
    int b, h, hk, blk, nb, n, n_next;                  /* cache head hk; n keys here, n_next in sequence b + 1 */
    __device__ __forceinline__ void set(const AttnArgs& A, int seq, int item, int block) {
        b = seq;
        h = item;
        hk = h / A.head_blocks;
        blk = block;
        n = attn_keys(A, b);
        nb = attn_blocks(n);
        n_next = b + 1 < A.n_seqs ? attn_keys(A, b + 1) : 0;
    }
    __device__ __forceinline__ bool last() const { return blk + 1 >= nb; }                    /* of the item */
    __device__ __forceinline__ void next_item(const AttnArgs& A, int items) {
        blk = 0;
        if (++h < items) {
            hk = h / A.head_blocks;
            return;
        }
        h = hk = 0;
        do {
            b++;
            n = n_next;
            n_next = b + 1 < A.n_seqs ? attn_keys(A, b + 1) : 0;
        } while (n == 0 && b < A.n_seqs);
        nb = attn_blocks(n);
    }
};

template <int FMT, int HD, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps, AttnShape<FMT, HD, NT>::CTAS) attn_decode_kernel(const __grid_constant__ AttnArgs A) {
    using F = AttnFmt<FMT, HD>;
    using S = AttnShape<FMT, HD, NT>;
    constexpr bool TQ = kv_is_tq(FMT);
    constexpr int TILES = S::TILES, MINE = S::MINE;    /* tiles of the output, those a warp finishes */
    __shared__ float m_s[kAttnWarps][8 * NT], l_s[kAttnWarps][8 * NT], f_s[kAttnWarps];
    __shared__ long long scan_s[kAttnWarps + 1];
    __shared__ int find_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t smem0 = (uint32_t)__cvta_generic_to_shared(attn_smem);
    const uint32_t ring = smem0 + S::LUT + warp * S::RING;
    const uint32_t xchg = smem0 + S::LUT + kAttnWarps * S::RING + 16 * lane;
    const uint32_t lane4 = 4 * lane;                   /* this lane's copy of the table */

    if constexpr (F::LUT > 0) {
        for (int e = warp; e < F::LUT; e += kAttnWarps) *reinterpret_cast<uint32_t*>(attn_smem + 128 * e + lane4) = attn_lut_entry<FMT>(e);
    }
    pdl_wait();
    pdl_trigger();

    /* This CTA's part of the line: sum the sequences' blocks, then find where the part begins. Each
     * item counts kAttnItemCost places more than it has blocks, ahead of its first block. */
    const int items = A.n_kv * A.head_blocks;
    const int per = (A.n_seqs + 32 * kAttnWarps - 1) / (32 * kAttnWarps);
    const int s0 = min(tid * per, A.n_seqs), s1 = min(s0 + per, A.n_seqs);
    long long mine = 0;
    for (int b = s0; b < s1; b++) mine += attn_places(attn_keys(A, b));
    long long upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) scan_s[warp] = upto;
    __syncthreads();
    long long total = 0, before = upto - mine;
#pragma unroll
    for (int w = 0; w < kAttnWarps; w++) {
        if (w < warp) before += scan_s[w];
        total += scan_s[w];
    }
    total *= items;
    const int parts = (int)min((long long)gridDim.x, total / (1 + kAttnItemCost));
    const int part = blockIdx.x;
    const long long u0 = part < parts ? total * part / parts : 0, u1 = part < parts ? total * (part + 1) / parts : 0;
    if (u0 < u1 && mine > 0 && u0 >= before * items && u0 < (before + mine) * items) {
        long long at = before;                         /* one thread finds itself here */
        for (int b = s0; b < s1; b++) {
            const int np = attn_places(attn_keys(A, b));
            if (u0 < (at + np) * items) {
                find_s = b;
                scan_s[kAttnWarps] = u0 - at * items;
                break;
            }
            at += np;
        }
    }
    /* rows without keys */
    for (int b = part; b < A.n_seqs; b += gridDim.x) {
        if (attn_keys(A, b) > 0) continue;
        uint32_t* o = reinterpret_cast<uint32_t*>(A.out + (size_t)b * A.n_q * HD);
        for (int i = tid; i < A.n_q * HD / 2; i += 32 * kAttnWarps) o[i] = 0;
        if (A.lse != nullptr)
            for (int i = tid; i < A.n_q; i += 32 * kAttnWarps) A.lse[(size_t)b * A.n_q + i] = -INFINITY;
    }
    __syncthreads();

    AttnAt to, at;                                     /* what is copied next, what is computed next */
    int places = (int)(u1 - u0), skipped = 0;          /* of the line that are left to this CTA */
    if (places > 0) {
        const long long in = scan_s[kAttnWarps];
        const int b = find_s, np = attn_places(attn_keys(A, b)), item = (int)(in / np);
        const int off = (int)(in - (long long)item * np);
        to.set(A, b, item, max(off - kAttnItemCost, 0));
        skipped = max(kAttnItemCost - off, 0);         /* the places ahead of the item's first block */
        places -= skipped;
    }
    if (places <= 0) {
        if (tid == 0) A.desc[part] = make_int2(-1, 0);
        return;
    }
    at = to;
    bool began = at.blk == 0;                          /* this CTA holds the beginning of the item */
    /* the item that ends here and began in an earlier CTA; which one it began in follows from the cut */
    if (tid == 0) {
        int2 d = make_int2(-1, 0);
        if (!began && places >= at.nb - at.blk) {
            const long long first = u0 + skipped - at.blk;       /* place of the item's first block */
            int p = (int)(first * parts / total);
            while (total * p / parts > first) p--;
            while (total * (p + 1) / parts <= first) p++;
            d = make_int2(at.b * items + at.h, p);
        }
        A.desc[part] = d;
    }

    /* What is copied next. A lane's K rows are g, g + 8 of the warp's 16, its V rows 2t, 2t + 1, 2t + 8,
     * 2t + 9; the pointers are those of its bytes in row 0 of the cache. */
    const uint32_t row_bytes = (uint32_t)A.n_kv * F::VEC;
    const uint8_t *klane, *vlane;
    int row_to;                                        /* cache row of the block's first position, -1: none; read one step ahead */
    auto aim_item = [&]() {
        klane = A.k_store + (size_t)g * row_bytes + to.hk * F::VEC + attn_k_byte<FMT, HD>(0, t);
        vlane = A.v_store + (size_t)(2 * t) * row_bytes + to.hk * F::VEC + attn_v_byte<FMT, HD>(0, g);
    };
    auto aim = [&]() {
        if (A.block_table != nullptr) {
            const int page = __ldg(A.block_table + (size_t)to.b * A.table_stride + to.blk);
            row_to = (unsigned)page <= (unsigned)(A.n_slots - 1) >> kAttnPageShift ? page << kAttnPageShift : -1;
        } else {
            const long long row = (long long)to.b * A.table_stride + ((long long)to.blk << kAttnPageShift);
            row_to = row < A.n_slots ? (int)row : -1;
        }
    };
    aim_item();
    aim();
    int to_places = places;                            /* places from `to` on */
    const bool odd_end = TQ && (((size_t)A.n_slots * A.n_kv) & 1) != 0;      /* the last RMS value stands alone in its word */
    auto issue = [&](int stage) -> int {               /* returns how many of the warp's 16 rows hold keys */
        int live = 0;
        if (to_places > 0) {
            const uint32_t base = ring + stage * (32 * S::LANE_BYTES);
            const uint32_t kd = base + lane * F::KU, vd = base + 32 * S::K_BYTES + lane * F::VU;
            const uint32_t md = base + 32 * (S::K_BYTES + S::V_BYTES) + lane4;
            const int row0 = row_to + 16 * warp;
            live = row_to < 0 ? 0 : min(min(to.n - (to.blk << kAttnPageShift) - 16 * warp, A.n_slots - row0), 16);
            if (live == 16 && !(TQ && odd_end && row0 + 16 >= A.n_slots)) {
                const uint8_t* kp = klane + (size_t)(uint32_t)row0 * row_bytes;
                const uint8_t* vp = vlane + (size_t)(uint32_t)row0 * row_bytes;
                AttnUnits<F::KN>::each([&](auto n) {
                    constexpr int N = decltype(n)::value;
                    const int off = attn_k_byte<FMT, HD>(N, t) - attn_k_byte<FMT, HD>(0, t);
                    cp_async<F::KU, N * 32 * F::KU>(kd, kp + off);
                    cp_async<F::KU, (F::KN + N) * 32 * F::KU>(kd, kp + 8 * (size_t)row_bytes + off);
                });
                AttnUnits<F::VN>::each([&](auto n) {
                    constexpr int N = decltype(n)::value;
                    const int off = attn_v_byte<FMT, HD>(N, g) - attn_v_byte<FMT, HD>(0, g);
                    cp_async<F::VU, N * 32 * F::VU>(vd, vp + off);
                    cp_async<F::VU, (F::VN + N) * 32 * F::VU>(vd, vp + row_bytes + off);
                    cp_async<F::VU, (2 * F::VN + N) * 32 * F::VU>(vd, vp + 8 * (size_t)row_bytes + off);
                    cp_async<F::VU, (3 * F::VN + N) * 32 * F::VU>(vd, vp + 9 * (size_t)row_bytes + off);
                });
                if constexpr (TQ) {
                    /* the RMS values of rows g, g + 8: the 32-bit words that hold them */
                    const size_t at = (((size_t)(uint32_t)(row0 + g) * A.n_kv + to.hk) * 2) & ~(size_t)3;
                    const uint8_t* mk = reinterpret_cast<const uint8_t*>(A.k_meta) + at;
                    const uint8_t* mv = reinterpret_cast<const uint8_t*>(A.v_meta) + at;
                    cp_async<4, 0>(md, mk);
                    cp_async<4, 128>(md, mk + 16 * (size_t)A.n_kv);
                    cp_async<4, 256>(md, mv);
                    cp_async<4, 384>(md, mv + 16 * (size_t)A.n_kv);
                }
            } else if (live > 0) {
                /* rows behind the last key are filled with zeros, nothing of them is read */
                const size_t first = (size_t)(uint32_t)row0 * row_bytes;
                AttnUnits<F::KN>::each([&](auto n) {
                    constexpr int N = decltype(n)::value;
                    const int off = attn_k_byte<FMT, HD>(N, t) - attn_k_byte<FMT, HD>(0, t);
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const bool ok = g + 8 * r < live;
                        const uint8_t* p = ok ? klane + first + 8 * r * (size_t)row_bytes + off : A.k_store;
                        if (r == 0) cp_async_some<F::KU, N * 32 * F::KU>(kd, p, ok ? F::KU : 0);
                        else cp_async_some<F::KU, (F::KN + N) * 32 * F::KU>(kd, p, ok ? F::KU : 0);
                    }
                });
                AttnUnits<4 * F::VN>::each([&](auto n) {
                    constexpr int N = decltype(n)::value % F::VN, R = decltype(n)::value / F::VN, KEY = (R & 1) + 8 * (R >> 1);
                    const int off = attn_v_byte<FMT, HD>(N, g) - attn_v_byte<FMT, HD>(0, g);
                    const bool ok = 2 * t + KEY < live;
                    cp_async_some<F::VU, decltype(n)::value * 32 * F::VU>(vd, ok ? vlane + first + KEY * (size_t)row_bytes + off : A.v_store, ok ? F::VU : 0);
                });
                if constexpr (TQ) {
                    const size_t end = (size_t)A.n_slots * A.n_kv * 2;         /* bytes of an array */
                    AttnUnits<4>::each([&](auto n) {
                        constexpr int R = decltype(n)::value;
                        const bool ok = g + 8 * (R & 1) < live;
                        const size_t at = ok ? (((size_t)(uint32_t)(row0 + g + 8 * (R & 1)) * A.n_kv + to.hk) * 2) & ~(size_t)3 : 0;
                        const uint8_t* p = reinterpret_cast<const uint8_t*>(R < 2 ? A.k_meta : A.v_meta) + at;
                        cp_async_some<4, R * 128>(md, p, !ok ? 0 : at + 4 > end ? 2 : 4);
                    });
                }
            }
            live = max(live, 0);
            to_places--;
            if (!to.last()) {
                to.blk++;
                if (to_places > 0) aim();
            } else {
                to_places -= kAttnItemCost;
                if (to_places > 0) {
                    to.next_item(A, items);
                    aim_item();
                    aim();
                }
            }
        }
        cp_commit();
        return live;
    };
    int live_q[S::STAGES];                             /* of the stages in flight, oldest first */
#pragma unroll
    for (int s = 0; s < S::STAGES - 1; s++) live_q[s] = issue(s);

    uint32_t q[NT][HD / 8];
    auto load_q = [&](const AttnAt& x) {
        const int h0 = (x.h - x.hk * A.head_blocks) * 8 * NT, heads = A.group - h0;      /* of this block: at most 8 NT */
        const __half* src = A.q + ((size_t)x.b * A.n_q + (size_t)x.hk * A.group + h0) * HD;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int n = 0; n < HD / 32; n++) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (8 * nt + g < heads)
                    v = *reinterpret_cast<const uint4*>(src + (size_t)(8 * nt + g) * HD + attn_k_dim<FMT>(n, t));
                q[nt][4 * n] = v.x; q[nt][4 * n + 1] = v.y; q[nt][4 * n + 2] = v.z; q[nt][4 * n + 3] = v.w;
            }
    };
    float o[NT][TILES][4], m[NT][2], l[NT][2], vref;   /* m: the maximum less kWeightLog2 */
    auto begin_item = [&]() {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int j = 0; j < TILES; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) o[nt][j][c] = 0.0f;
            m[nt][0] = m[nt][1] = kNoMax;
            l[nt][0] = l[nt][1] = 0.0f;
        }
        vref = TQ ? 5.9604645e-8f : 1.0f;              /* the smallest RMS there is: 2^-24 */
    };
    load_q(at);
    begin_item();

    int stage = 0;
    for (;;) {
        cp_wait<S::STAGES - 2>();
        live_q[S::STAGES - 1] = issue(stage == 0 ? S::STAGES - 1 : stage - 1);     /* into the slot that the previous step emptied */
        const int live = live_q[0];
#pragma unroll
        for (int s = 0; s + 1 < S::STAGES; s++) live_q[s] = live_q[s + 1];
        const uint32_t base = ring + stage * (32 * S::LANE_BYTES);
        const uint32_t kd = base + lane * F::KU, vd = base + 32 * S::K_BYTES + lane * F::VU;
        if (++stage == S::STAGES) stage = 0;
        float sk[2] = {1.0f, 1.0f}, sv[2] = {1.0f, 1.0f};
        float s[NT][4];
        if (live > 0) {                                /* uniform over the warp */
            uint32_t klo[HD / 8], khi[HD / 8];
            {
                uint32_t raw[2][F::KN * F::KU / 4 + 1];
                AttnUnits<F::KN>::each([&](auto n) {
                    constexpr int N = decltype(n)::value;
                    lds_unit<F::KU, N * 32 * F::KU>(kd, &raw[0][N * (F::KU / 4)]);
                    lds_unit<F::KU, (F::KN + N) * 32 * F::KU>(kd, &raw[1][N * (F::KU / 4)]);
                });
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    if constexpr (FMT == KV_TQ1_5) {
                        const int sh = attn_k_shift<FMT>(t);
                        raw[r][0] = __funnelshift_r(raw[r][0], raw[r][1], sh);
                        raw[r][1] >>= sh;
                    }
                }
                attn_k_words<FMT, HD>(raw[0], klo, lane4);
                attn_k_words<FMT, HD>(raw[1], khi, lane4);
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float s0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks += 2) {
                    mma16816(s0, klo[2 * ks], khi[2 * ks], klo[2 * ks + 1], khi[2 * ks + 1], q[nt][2 * ks], q[nt][2 * ks + 1]);
                    mma16816(s1, klo[2 * ks + 2], khi[2 * ks + 2], klo[2 * ks + 3], khi[2 * ks + 3], q[nt][2 * ks + 2], q[nt][2 * ks + 3]);
                }
#pragma unroll
                for (int c = 0; c < 4; c++) s[nt][c] = s0[c] + s1[c];
            }
        }
        /* the next item's Q is on its way while this one is finished */
        const bool item_done = at.last();
        places--;
        const bool more = item_done ? places > kAttnItemCost : places > 0;
        AttnAt nx = at;
        if (!item_done) {
            nx.blk++;
        } else if (more) {
            nx.next_item(A, items);
            load_q(nx);
        }
        if (live > 0) {
            if constexpr (TQ) {
                const uint32_t mb = base + 32 * (S::K_BYTES + S::V_BYTES) + lane4;
                /* which half of the word: the parity of the value's index (64 blk + 16 warp + 8 are even) */
                const int bk = A.block_table != nullptr ? 0 : (int)(((long long)at.b * A.table_stride) & 1);
                const int shift = (((bk + g) * A.n_kv + at.hk) & 1) * 16;
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    sk[r] = __half2float(__ushort_as_half((unsigned short)(lds32(mb + 128 * r) >> shift)));
                    sv[r] = __half2float(__ushort_as_half((unsigned short)(lds32(mb + 128 * (2 + r)) >> shift)));
                }
            }
            /* scores in base 2; rows behind the last key have none */
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++) s[nt][c] *= TQ ? A.scale2 * (sk[c >> 1] * (1.0f / attn_alpha<FMT>())) : A.scale2;
            if (live < 16) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++)
                        if (g + 8 * (c >> 1) >= live) s[nt][c] = -INFINITY;
            }
            bool up = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++) up |= s[nt][c] > m[nt][c & 1] + kWeightTop;
            if constexpr (TQ) up |= fmaxf(sv[0], sv[1]) > vref;
            if (__any_sync(0xffffffffu, up)) {
                /* a new maximum (or a larger RMS of V): rescale what there is */
                float rv = 1.0f;
                if constexpr (TQ) {
                    float x = fmaxf(sv[0], sv[1]);
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    if (x > vref) {                    /* the next power of two above it */
                        const float nref = x < INFINITY ? __uint_as_float((__float_as_uint(x) & 0x7f800000u) + 0x00800000u) : vref;
                        rv = vref / nref;
                        vref = nref;
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float x = fmaxf(s[nt][c], s[nt][c + 2]);
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                        x = fmaxf(x - kWeightLog2, m[nt][c]);
                        const float a = ex2(m[nt][c] - x);
                        m[nt][c] = x;
                        l[nt][c] *= a;
#pragma unroll
                        for (int j = 0; j < TILES; j++) {
                            o[nt][j][c] *= a * rv;
                            o[nt][j][c + 2] *= a * rv;
                        }
                    }
            }
            /* weights: FP32 sums, FP16 pairs for the product */
            uint32_t bh[NT][2], bl[NT][2];
            const float inv = 1.0f / vref;             /* (a power of two) */
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    float w[2];
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        w[c] = ex2(s[nt][2 * r + c] - m[nt][c]);
                        l[nt][c] += w[c];
                        if constexpr (TQ) w[c] *= sv[r] * inv;
                    }
                    const uint32_t hi = pack2_rz(w[0], w[1]);
                    const float2 h = unpack2(hi);
                    const uint32_t lo = hmax2_bits(pack2(w[0] - h.x, w[1] - h.y), 0x00010001u);      /* at least 2^-24 */
                    bh[nt][r] = movmatrix(hi);
                    bl[nt][r] = movmatrix(lo);
                }
            {
                uint32_t xa[HD / 8], xc[HD / 8];       /* keys (2t, 2t+1), (2t+8, 2t+9) */
                {
                    uint32_t raw[4][F::VN * F::VU / 4];
                    AttnUnits<4 * F::VN>::each([&](auto n) {
                        constexpr int N = decltype(n)::value;
                        lds_unit<F::VU, N * 32 * F::VU>(vd, &raw[N / F::VN][N % F::VN * (F::VU / 4)]);
                    });
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if constexpr (FMT == KV_TQ3 || FMT == KV_TQ1_5) {
                            const int sh = attn_v_shift<FMT>(g);
                            raw[r][0] = __funnelshift_r(raw[r][0], raw[r][1], sh);
                            raw[r][1] >>= sh;
                        }
                    }
                    attn_v_pairs<FMT, HD>(raw[0], raw[1], xa, lane4);
                    attn_v_pairs<FMT, HD>(raw[2], raw[3], xc, lane4);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < TILES; j++) {
                        mma16816(o[nt][j], xa[2 * j], xa[2 * j + 1], xc[2 * j], xc[2 * j + 1], bh[nt][0], bh[nt][1]);
                        mma16816(o[nt][j], xa[2 * j], xa[2 * j + 1], xc[2 * j], xc[2 * j + 1], bl[nt][0], bl[nt][1]);
                    }
            }
        }
        if (!item_done && more) {
            at = nx;
            continue;
        }
        /* the item (or the part) ends: join the four warps; warp d finishes tiles d * MINE .. + MINE - 1 */
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 4);
                l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 8);
                l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 16);
            }
        const int h0 = (at.h - at.hk * A.head_blocks) * 8 * NT, heads = A.group - h0;
        const size_t head0 = (size_t)at.b * A.n_q + (size_t)at.hk * A.group + h0;
        const bool whole = began && item_done;
        const int slot = 2 * part + (began ? 1 : 0);               /* an item that began here is this CTA's last */
        float top[NT][2], sum[NT][2], f[NT][kAttnWarps][2];
#pragma unroll
        for (int round = 0; round < S::ROUNDS; round++) {
            __syncthreads();                           /* what the exchange held has been read */
            if (round == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    if (g == 0) {
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            m_s[warp][8 * nt + 2 * t + c] = m[nt][c];
                            l_s[warp][8 * nt + 2 * t + c] = l[nt][c];
                        }
                    }
                if (lane == 0) f_s[warp] = vref;
            }
#pragma unroll
            for (int x = 0; x < NT * TILES; x++) {
                const int d = x / MINE, k = (warp - d - 1) & (kAttnWarps - 1);
                if ((x % MINE) / S::PER_ROUND != round) continue;
                if (d != warp) {
                    const float(&v)[4] = o[x / TILES][x % TILES];
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(xchg + ((d * (kAttnWarps - 1) + k) * S::PER_ROUND + x % S::PER_ROUND) * 512),
                                 "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
                }
            }
            __syncthreads();
            if (round == 0) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int h = 8 * nt + 2 * t + c;
                        top[nt][c] = m_s[0][h];
#pragma unroll
                        for (int w = 1; w < kAttnWarps; w++) top[nt][c] = fmaxf(top[nt][c], m_s[w][h]);
                        sum[nt][c] = 0.0f;
#pragma unroll
                        for (int w = 0; w < kAttnWarps; w++) {
                            f[nt][w][c] = ex2(m_s[w][h] - top[nt][c]);
                            sum[nt][c] += f[nt][w][c] * l_s[w][h];
                            f[nt][w][c] *= f_s[w] * (1.0f / attn_alpha<FMT>());
                        }
                        if (warp == 0 && g == 0) {
                            if (!whole) A.part_ml[(size_t)slot * (8 * NT) + h] = make_float2(top[nt][c], sum[nt][c]);
                            else if (A.lse != nullptr && h < heads) A.lse[head0 + h] = attn_lse(top[nt][c], sum[nt][c]);
                        }
                    }
            }
#pragma unroll
            for (int x = 0; x < NT * TILES; x++) {
                if ((x % MINE) / S::PER_ROUND != round || x / MINE != warp) continue;
                const int nt = x / TILES, j = x % TILES;
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kAttnWarps; w++) { /* in warp order, whoever adds */
                    float v[4];
                    if (w == warp) {
#pragma unroll
                        for (int c = 0; c < 4; c++) v[c] = o[nt][j][c];
                    } else {
                        const int k = (w - warp - 1) & (kAttnWarps - 1);
                        asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                                     : "r"(xchg + ((warp * (kAttnWarps - 1) + k) * S::PER_ROUND + x % S::PER_ROUND) * 512));
                    }
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[c] = fmaf(v[c], f[nt][w][c & 1], acc[c]);
                }
                if (whole) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int h = 8 * nt + 2 * t + c;
                        if (h < heads)
                            *reinterpret_cast<uint32_t*>(A.out + (head0 + h) * HD + attn_v_dim<FMT, HD>(j, g)) =
                                attn_out(acc[c], acc[c + 2], sum[nt][c]);
                    }
                } else {
                    A.part_o[((size_t)slot * (NT * TILES) + x) * 32 + lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                }
            }
        }
        if (!more) break;
        places -= kAttnItemCost;
        at = nx;
        began = true;
        begin_item();
    }
    cp_wait<0>();
}

/* One CTA per part: the item that ends in the part and began in part `first` has its pieces in slots
 * 2 first + 1, 2 (first + 1), 2 (first + 2) .. 2 part. Warp w takes tile w % TILES of the output and
 * every (32 / TILES)-th piece. */
template <int FMT, int HD, int NT>
__global__ void __launch_bounds__(kAttnJoinThreads) attn_join_kernel(const __grid_constant__ AttnArgs A) {
    constexpr int TILES = HD / 16, LANES = kAttnJoinThreads / 32 / TILES;
    __shared__ float top_s[8], sum_s[8];
    __shared__ float4 acc_s[kAttnJoinThreads / 32][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int nt = blockIdx.y;
    pdl_wait();
    pdl_trigger();
    for (int part = blockIdx.x; part < kAttnParts; part += gridDim.x) {
    const int2 d = A.desc[part];
    if (d.x < 0) continue;
    const int first = d.y, pieces = part - first + 1;
    auto slot_of = [&](int p) { return p == 0 ? 2 * first + 1 : 2 * (first + p); };
    if (warp < 8) {                                    /* head `warp` of the item */
        float top = kNoMax;
        for (int p = lane; p < pieces; p += 32) top = fmaxf(top, A.part_ml[(size_t)slot_of(p) * (8 * NT) + 8 * nt + warp].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        float sum = 0.0f;
        for (int p = lane; p < pieces; p += 32) {
            const float2 ml = A.part_ml[(size_t)slot_of(p) * (8 * NT) + 8 * nt + warp];
            sum += ml.y * ex2(ml.x - top);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) { top_s[warp] = top; sum_s[warp] = sum; }
    }
    __syncthreads();
    const int j = warp % TILES, sub = warp / TILES;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float top0 = top_s[2 * t], top1 = top_s[2 * t + 1];
#pragma unroll 4
    for (int p = sub; p < pieces; p += LANES) {
        const size_t slot = slot_of(p);
        const float4 v = A.part_o[(slot * (NT * TILES) + nt * TILES + j) * 32 + lane];
        const float f0 = ex2(A.part_ml[slot * (8 * NT) + 8 * nt + 2 * t].x - top0);
        const float f1 = ex2(A.part_ml[slot * (8 * NT) + 8 * nt + 2 * t + 1].x - top1);
        acc.x = fmaf(v.x, f0, acc.x);
        acc.y = fmaf(v.y, f1, acc.y);
        acc.z = fmaf(v.z, f0, acc.z);
        acc.w = fmaf(v.w, f1, acc.w);
    }
    acc_s[warp][lane] = acc;
    __syncthreads();
    const int items = A.n_kv * A.head_blocks;
    const int b = d.x / items, item = d.x - b * items, hk = item / A.head_blocks, hb = item - hk * A.head_blocks;
    const int heads = A.group - hb * 8 * NT;
    const size_t head0 = (size_t)b * A.n_q + (size_t)hk * A.group + hb * 8 * NT;
    if (sub == 0) {
        for (int k = 1; k < LANES; k++) {
            const float4 v = acc_s[warp + k * TILES][lane];
            acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
        }
        const float a[4] = {acc.x, acc.y, acc.z, acc.w};
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int h = 8 * nt + 2 * t + c;
            if (h >= heads) continue;
            *reinterpret_cast<uint32_t*>(A.out + (head0 + h) * HD + attn_v_dim<FMT, HD>(j, g)) = attn_out(a[c], a[c + 2], sum_s[2 * t + c]);
        }
    }
    if (A.lse != nullptr && tid < 8 && 8 * nt + tid < heads)
        A.lse[head0 + 8 * nt + tid] = attn_lse(top_s[tid], sum_s[tid]);
    __syncthreads();
    }
}

/* Column tiles of 8 query heads an item holds: two where the group has more than eight heads
 * (head_dim 256: one, for the registers), the rest in further items of the same cache head. */
static int attn_col_tiles(int group, int head_dim) { return group > 8 && head_dim <= 128 ? 2 : 1; }

struct AttnScratch { size_t ml, o, bytes; };
static AttnScratch attn_scratch(int group, int head_dim) {
    const size_t heads = 8 * (size_t)attn_col_tiles(group, head_dim);
    AttnScratch s;
    s.ml = kAttnParts * sizeof(int2);                                   /* 16-byte multiples */
    s.o = s.ml + 2 * kAttnParts * heads * sizeof(float2);
    s.bytes = s.o + 2 * kAttnParts * heads * head_dim * sizeof(float);
    return s;
}

template <int FMT, int HD, int NT>
static cudaError_t launch_attn(const AttnArgs& A, cudaStream_t s) {
    constexpr int SMEM = AttnShape<FMT, HD, NT>::SMEM;
    cudaError_t e = cudaFuncSetAttribute((const void*)attn_decode_kernel<FMT, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    e = launch_pdl(attn_decode_kernel<FMT, HD, NT>, dim3(kAttnParts), dim3(32 * kAttnWarps), (size_t)SMEM, s, A);
    if (e != cudaSuccess) return e;
    e = launch_pdl(attn_join_kernel<FMT, HD, NT>, dim3(kAttnJoinCtas, NT), dim3(kAttnJoinThreads), 0, s, A);
    if (e == cudaSuccess) g_launches.fetch_add(2, std::memory_order_relaxed);
    return e;
}
template <int FMT>
static cudaError_t launch_attn(const AttnArgs& A, int head_dim, int nt, cudaStream_t s) {
    if constexpr (!kv_is_tq(FMT)) {
        if (head_dim == 64) return nt == 2 ? launch_attn<FMT, 64, 2>(A, s) : launch_attn<FMT, 64, 1>(A, s);
        if (head_dim == 256) return launch_attn<FMT, 256, 1>(A, s);
    }
    if (head_dim == 128) return nt == 2 ? launch_attn<FMT, 128, 2>(A, s) : launch_attn<FMT, 128, 1>(A, s);
    return cudaErrorNotSupported;
}

}  // namespace vvb

using namespace vvb;

extern "C" size_t vvbk_attn_decode_scratch(int n_seqs, int n_q_heads, int n_kv_heads, int head_dim) {
    (void)n_seqs;
    return attn_scratch(n_q_heads / n_kv_heads, head_dim).bytes;
}

extern "C" int vvbk_attn_decode(const void* q, void* out, float* lse, const void* k_store, const void* v_store,
                                const void* k_meta, const void* v_meta, const int* block_table, const int* lens,
                                void* scratch, int n_seqs, int n_q_heads, int n_kv_heads, int head_dim, int n_slots,
                                int table_stride, int len_add, int kv_format, float scale, void* stream) {
    const int group = n_q_heads / n_kv_heads, nt = attn_col_tiles(group, head_dim);
    const AttnScratch sc = attn_scratch(group, head_dim);
    uint8_t* const base = (uint8_t*)scratch;
    const AttnArgs A = {(const __half*)q, (__half*)out, lse, (const uint8_t*)k_store, (const uint8_t*)v_store,
                        (const __half*)k_meta, (const __half*)v_meta, block_table, lens,
                        (int2*)base, (float2*)(base + sc.ml), (float4*)(base + sc.o),
                        n_seqs, n_q_heads, n_kv_heads, n_slots, table_stride, len_add,
                        group, (group + 8 * nt - 1) / (8 * nt), scale * kLog2e};
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
    switch (kv_format) {
        case KV_RAW: e = launch_attn<KV_RAW>(A, head_dim, nt, s); break;
        case KV_E4M3: e = launch_attn<KV_E4M3>(A, head_dim, nt, s); break;
        case KV_E5M2: e = launch_attn<KV_E5M2>(A, head_dim, nt, s); break;
        case KV_TQ4: e = launch_attn<KV_TQ4>(A, head_dim, nt, s); break;
        case KV_TQ3: e = launch_attn<KV_TQ3>(A, head_dim, nt, s); break;
        case KV_TQ2: e = launch_attn<KV_TQ2>(A, head_dim, nt, s); break;
        case KV_TQ1_5: e = launch_attn<KV_TQ1_5>(A, head_dim, nt, s); break;
        default: return (int)cudaErrorNotSupported;
    }
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}
