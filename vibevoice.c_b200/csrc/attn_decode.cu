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

namespace vvb {

extern std::atomic<uint64_t> g_launches;

constexpr int kAttnPageShift = 6;
constexpr int kAttnWarps = 4;                   /* a quarter of a 64-position block each */
constexpr int kAttnCtas = 2 * 148;              /* parts the work is cut into */
constexpr int kAttnJoinThreads = 1024;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kWeightScale = 32768.0f;        /* weights are at most 1 */
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
    int2* desc;                /* [kAttnCtas] item that ends in this CTA and began in an earlier one, that CTA; or -1 */
    float2* part_ml;           /* [2 kAttnCtas][heads of an item] maximum, sum */
    float4* part_o;            /* [2 kAttnCtas][tiles][32] output, in the lanes' layout */
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
    static constexpr int LANE_BYTES = K_BYTES + V_BYTES + 4 * F::META + 4;                    /* of a stage; the last word: live rows */
    static constexpr int STAGES = FMT == KV_RAW ? (HD == 256 ? 2 : 3) : 4;
    static constexpr int RING = 32 * LANE_BYTES * STAGES;                                     /* a warp's */
    static constexpr int TILES = HD / 16;                                                     /* 16-dim tiles of the output */
    static constexpr int XCHG = kAttnWarps * (kAttnWarps - 1) * (NT * TILES / kAttnWarps) * 32 * 16;
    static constexpr int LUT = F::LUT * 128;
    static constexpr int SMEM = LUT + kAttnWarps * RING + XCHG;       /* in this order */
};

/* ---------------------------------------------------------------- instructions */

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool live) {
    const int n = live ? BYTES : 0;                    /* 0: the destination is filled with zeros, nothing is read */
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_some(uint32_t dst, const void* src, int n) {         /* n of 4 bytes */
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
template <int UNIT> __device__ __forceinline__ void lds_unit(uint32_t a, uint32_t* w) {
    if constexpr (UNIT == 16) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
    else if constexpr (UNIT == 8) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
    else w[0] = lds32(a);
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
    if (FMT == KV_TQ1_5) return min(((3 * g) & ~3) + 4 * n, 20);      /* the last lane's three bytes lie in one word */
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

/* A place in the line of blocks: block blk of item h (cache head x head block) of sequence b. */
struct AttnAt {
    int b, h, blk, n, n_next;                          /* n keys here, n_next in sequence b + 1 */
    __device__ __forceinline__ void set(const AttnArgs& A, int seq) {
        b = seq;
        n = attn_keys(A, b);
        n_next = b + 1 < A.n_seqs ? attn_keys(A, b + 1) : 0;
    }
    __device__ __forceinline__ bool last() const { return blk + 1 >= attn_blocks(n); }        /* of the item */
    __device__ __forceinline__ void step(const AttnArgs& A, int items) {
        if (!last()) { blk++; return; }
        blk = 0;
        if (++h < items) return;
        h = 0;
        do {
            b++;
            n = n_next;
            n_next = b + 1 < A.n_seqs ? attn_keys(A, b + 1) : 0;
        } while (n == 0 && b < A.n_seqs);
    }
};

template <int FMT, int HD, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps, 2) attn_decode_kernel(const __grid_constant__ AttnArgs A) {
    using F = AttnFmt<FMT, HD>;
    using S = AttnShape<FMT, HD, NT>;
    constexpr bool TQ = kv_is_tq(FMT);
    constexpr int TILES = S::TILES, MINE = NT * TILES / kAttnWarps;    /* tiles of the output, those a warp finishes */
    __shared__ float m_s[kAttnWarps][8 * NT], l_s[kAttnWarps][8 * NT], f_s[kAttnWarps];
    __shared__ long long scan_s[kAttnWarps + 1];
    __shared__ int find_s[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t smem0 = (uint32_t)__cvta_generic_to_shared(attn_smem);
    const uint32_t ring = smem0 + S::LUT + warp * S::RING;
    const uint32_t xchg = smem0 + S::LUT + kAttnWarps * S::RING;
    const uint32_t lane4 = 4 * lane;                   /* this lane's copy of the table */

    if constexpr (F::LUT > 0) {
        for (int e = warp; e < F::LUT; e += kAttnWarps) *reinterpret_cast<uint32_t*>(attn_smem + 128 * e + lane4) = attn_lut_entry<FMT>(e);
    }
    pdl_wait();
    pdl_trigger();

    /* This CTA's part of the line: sum the sequences' blocks, then find where the part begins. */
    const int items = A.n_kv * A.head_blocks;
    const int per = (A.n_seqs + 32 * kAttnWarps - 1) / (32 * kAttnWarps);
    const int s0 = min(tid * per, A.n_seqs), s1 = min(s0 + per, A.n_seqs);
    long long mine = 0;
    for (int b = s0; b < s1; b++) mine += attn_blocks(attn_keys(A, b));
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
    const int parts = (int)min((long long)gridDim.x, total);
    const int part = blockIdx.x;
    const long long u0 = part < parts ? total * part / parts : 0, u1 = part < parts ? total * (part + 1) / parts : 0;
    if (u0 < u1 && mine > 0 && u0 >= before * items && u0 < (before + mine) * items) {
        long long at = before;                         /* one thread finds itself here */
        for (int b = s0; b < s1; b++) {
            const int nb = attn_blocks(attn_keys(A, b));
            if (u0 < (at + nb) * items) {
                find_s[0] = b;
                scan_s[kAttnWarps] = u0 - at * items;
                break;
            }
            at += nb;
        }
    }
    /* rows without keys */
    for (int b = part; b < A.n_seqs; b += gridDim.x) {
        if (attn_keys(A, b) > 0) continue;
        uint32_t* o = reinterpret_cast<uint32_t*>(A.out + (size_t)b * A.n_q * HD);
        for (int i = tid; i < A.n_q * HD / 2; i += 32 * kAttnWarps) o[i] = 0;
        if (A.lse != nullptr)
            for (int i = tid; i < A.n_q; i += 32 * kAttnWarps) A.lse[(size_t)b * A.n_q + i] = __int_as_float(0xff800000);
    }
    __syncthreads();
    if (tid == 0 && (u0 >= u1)) A.desc[part] = make_int2(-1, 0);
    if (u0 >= u1) return;

    AttnAt to, at;                                     /* what is copied next, what is computed next */
    to.set(A, find_s[0]);
    {
        const long long in = scan_s[kAttnWarps];
        const int nb = attn_blocks(to.n);
        to.h = (int)(in / nb);
        to.blk = (int)(in - (long long)to.h * nb);
    }
    at = to;
    bool began = at.blk == 0;                          /* this CTA holds the beginning of the item */
    /* the item that ends here and began in an earlier CTA; which one it began in follows from the cut */
    if (tid == 0) {
        int2 d = make_int2(-1, 0);
        const int nb = attn_blocks(at.n);
        if (!began && u1 - u0 >= nb - at.blk) {
            const long long first = u0 - at.blk;       /* the part that holds block `first` of the line */
            int p = (int)(first * parts / total);
            while (total * p / parts > first) p--;
            while (total * (p + 1) / parts <= first) p++;
            d = make_int2(at.b * items + at.h, p);
        }
        A.desc[part] = d;
    }

    const int steps = (int)(u1 - u0);
    auto page_row = [&](const AttnAt& x) -> long long {            /* cache row of the block's first position */
        if (A.block_table != nullptr)
            return (long long)__ldg(A.block_table + (size_t)x.b * A.table_stride + x.blk) << kAttnPageShift;
        return (long long)x.b * A.table_stride + ((long long)x.blk << kAttnPageShift);
    };
    long long row_to = page_row(to);                   /* read one step ahead of its use */
    int issued = 0;
    auto issue = [&](int stage) {
        if (issued < steps) {
            const long long row0 = row_to + 16 * warp;
            const long long left = min((long long)(to.n - (to.blk << kAttnPageShift) - 16 * warp), (long long)A.n_slots - row0);
            const int live = row_to < 0 ? 0 : (int)max(min(left, 16ll), 0ll);
            const int hk = to.h / A.head_blocks;
            const uint32_t base = ring + stage * (32 * S::LANE_BYTES);
            const size_t vec0 = (size_t)(live > 0 ? row0 : 0) * A.n_kv + hk;
            const uint8_t* kp = A.k_store + vec0 * F::VEC;
            const uint8_t* vp = A.v_store + vec0 * F::VEC;
            const size_t row_bytes = (size_t)A.n_kv * F::VEC;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const int key = g + 8 * r;
                const uint8_t* p = kp + (key < live ? key * row_bytes : 0);
#pragma unroll
                for (int n = 0; n < F::KN; n++)
                    cp_async<F::KU>(base + (r * F::KN + n) * (32 * F::KU) + lane * F::KU, p + attn_k_byte<FMT, HD>(n, t), key < live);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int key = 2 * t + (r & 1) + 8 * (r >> 1);
                const uint8_t* p = vp + (key < live ? key * row_bytes : 0);
#pragma unroll
                for (int n = 0; n < F::VN; n++)
                    cp_async<F::VU>(base + 32 * S::K_BYTES + (r * F::VN + n) * (32 * F::VU) + lane * F::VU, p + attn_v_byte<FMT, HD>(n, g), key < live);
            }
            if constexpr (TQ) {
                /* the RMS values of K rows g, g + 8, then of V's: the 32-bit word that holds each; the
                 * array's last value may stand alone in its word */
                const size_t last = (size_t)A.n_slots * A.n_kv - 1;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int key = g + 8 * (r & 1);
                    const size_t i = vec0 + (key < live ? (size_t)key * A.n_kv : 0);
                    const __half* m = (r < 2 ? A.k_meta : A.v_meta) + (i & ~(size_t)1);
                    cp_async_some(base + 32 * (S::K_BYTES + S::V_BYTES) + r * 128 + lane * 4, m, key >= live ? 0 : (i & ~(size_t)1) == last ? 2 : 4);
                }
            }
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(base + 32 * (S::LANE_BYTES - 4) + 4 * lane), "r"(live) : "memory");
            issued++;
            if (issued < steps) {
                to.step(A, items);
                row_to = page_row(to);
            }
        }
        cp_commit();
    };
#pragma unroll
    for (int s = 0; s < S::STAGES - 1; s++) issue(s);

    uint32_t q[NT][HD / 8];
    float o[NT][TILES][4], m[NT][2], l[NT][2], vref = 0.0f;
    auto begin_item = [&]() {
        const int hk = at.h / A.head_blocks, hb = at.h - hk * A.head_blocks;
        const int h0 = hb * 8 * NT, heads = A.group - h0;          /* heads of this block: at most 8 NT */
        const __half* src = A.q + ((size_t)at.b * A.n_q + (size_t)hk * A.group + h0) * HD;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
#pragma unroll
            for (int n = 0; n < HD / 32; n++) {
                uint4 x = make_uint4(0, 0, 0, 0);
                if (8 * nt + g < heads)
                    x = *reinterpret_cast<const uint4*>(src + (size_t)(8 * nt + g) * HD + attn_k_dim<FMT>(n, t));
                q[nt][4 * n] = x.x; q[nt][4 * n + 1] = x.y; q[nt][4 * n + 2] = x.z; q[nt][4 * n + 3] = x.w;
            }
#pragma unroll
            for (int j = 0; j < TILES; j++)
#pragma unroll
                for (int c = 0; c < 4; c++) o[nt][j][c] = 0.0f;
            m[nt][0] = m[nt][1] = kNoMax;
            l[nt][0] = l[nt][1] = 0.0f;
        }
        vref = TQ ? 5.9604645e-8f : 1.0f;              /* the smallest RMS there is: 2^-24 */
    };
    begin_item();

    int stage = 0;
    for (int i = 0; i < steps; i++) {
        cp_wait<S::STAGES - 2>();
        issue(stage == 0 ? S::STAGES - 1 : stage - 1);             /* into the slot that the previous step emptied */
        const uint32_t base = ring + stage * (32 * S::LANE_BYTES);
        const int live = (int)lds32(base + 32 * (S::LANE_BYTES - 4) + 4 * lane);
        if (live > 0) {                                /* uniform over the warp */
            float sk[2] = {1.0f, 1.0f}, sv[2] = {1.0f, 1.0f};
            float s[NT][4];
            {
                uint32_t klo[HD / 8], khi[HD / 8];
                {
                    uint32_t raw[2][F::KN * F::KU / 4 + 1];
#pragma unroll
                    for (int r = 0; r < 2; r++) {
#pragma unroll
                        for (int n = 0; n < F::KN; n++)
                            lds_unit<F::KU>(base + (r * F::KN + n) * (32 * F::KU) + lane * F::KU, &raw[r][n * (F::KU / 4)]);
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
            if constexpr (TQ) {
                const uint32_t mb = base + 32 * (S::K_BYTES + S::V_BYTES) + 4 * lane;
                /* which half of the word: the parity of the value's index */
                const int hk = at.h / A.head_blocks;
                const int bk = A.block_table != nullptr ? 0 : (int)(((long long)at.b * A.table_stride) & 1);      /* 64 blk + 16 warp are even */
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const int odd = ((bk + g + 8 * r) * A.n_kv + hk) & 1;
                    const uint32_t wk = lds32(mb + 128 * r), wv = lds32(mb + 128 * (2 + r));
                    sk[r] = __half2float(__ushort_as_half((unsigned short)(odd ? wk >> 16 : wk)));
                    sv[r] = __half2float(__ushort_as_half((unsigned short)(odd ? wv >> 16 : wv)));
                }
            }
            /* scores in base 2; rows behind the last key have none */
            bool up = false;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    const float f = TQ ? A.scale2 * (sk[c >> 1] * (1.0f / attn_alpha<FMT>())) : A.scale2;
                    s[nt][c] = g + 8 * (c >> 1) < live ? s[nt][c] * f : -INFINITY;
                    up |= s[nt][c] > m[nt][c & 1];
                }
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
                        x = fmaxf(x, m[nt][c]);
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
            const float inv = TQ ? kWeightScale / vref : kWeightScale;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    float hi[2], lo[2];
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const float p = ex2(s[nt][2 * r + c] - m[nt][c]);
                        l[nt][c] += p;
                        const float w = TQ ? p * (sv[r] * inv) : p * kWeightScale;
                        hi[c] = __half2float(__float2half_rz(w));
                        lo[c] = w > 0.0f ? fmaxf(w - hi[c], 5.9604645e-8f) : w - hi[c];
                    }
                    bh[nt][r] = movmatrix(pack2(hi[0], hi[1]));
                    bl[nt][r] = movmatrix(pack2(lo[0], lo[1]));
                }
            {
                uint32_t xa[HD / 8], xc[HD / 8];       /* keys (2t, 2t+1), (2t+8, 2t+9) */
                {
                    uint32_t raw[4][F::VN * F::VU / 4];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
#pragma unroll
                        for (int n = 0; n < F::VN; n++)
                            lds_unit<F::VU>(base + 32 * S::K_BYTES + (r * F::VN + n) * (32 * F::VU) + lane * F::VU, &raw[r][n * (F::VU / 4)]);
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
        if (++stage == S::STAGES) stage = 0;

        const bool item_done = at.last();
        if (item_done || i + 1 == steps) {
            /* join the four warps: warp d finishes tiles d * MINE .. + MINE - 1 */
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 4);
                    l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 8);
                    l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], 16);
                }
            __syncthreads();                           /* the previous item's exchange has been read */
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
#pragma unroll
            for (int x = 0; x < NT * TILES; x++) {
                const int d = x / MINE, k = (warp - d - 1) & (kAttnWarps - 1);
                if (d != warp) {
                    const float(&v)[4] = o[x / TILES][x % TILES];
                    asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(xchg + (((d * (kAttnWarps - 1) + k) * MINE + x % MINE) * 32 + lane) * 16),
                                 "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]) : "memory");
                }
            }
            __syncthreads();
            const int hk = at.h / A.head_blocks, hb = at.h - hk * A.head_blocks;
            const int heads = A.group - hb * 8 * NT;
            const size_t head0 = (size_t)at.b * A.n_q + (size_t)hk * A.group + hb * 8 * NT;
            const bool whole = began && item_done;
            const int slot = 2 * part + (began ? 1 : 0);           /* an item that began here is this CTA's last */
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float top[2], sum[2], f[kAttnWarps][2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int h = 8 * nt + 2 * t + c;
                    top[c] = m_s[0][h];
#pragma unroll
                    for (int w = 1; w < kAttnWarps; w++) top[c] = fmaxf(top[c], m_s[w][h]);
                    sum[c] = 0.0f;
#pragma unroll
                    for (int w = 0; w < kAttnWarps; w++) {
                        f[w][c] = ex2(m_s[w][h] - top[c]);
                        sum[c] += f[w][c] * l_s[w][h];
                        f[w][c] *= f_s[w] * (1.0f / (kWeightScale * attn_alpha<FMT>()));
                    }
                }
#pragma unroll
                for (int x = 0; x < NT * TILES; x++) {
                    if (x / TILES != nt || x / MINE != warp) continue;
                    const int j = x % TILES;
                    float acc[4];
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[c] = 0.0f;
#pragma unroll
                    for (int w = 0; w < kAttnWarps; w++) {         /* in warp order, whoever adds */
                        float v[4];
                        if (w == warp) {
#pragma unroll
                            for (int c = 0; c < 4; c++) v[c] = o[nt][j][c];
                        } else {
                            const int k = (w - warp - 1) & (kAttnWarps - 1);
                            asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                                         : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                                         : "r"(xchg + (((warp * (kAttnWarps - 1) + k) * MINE + x % MINE) * 32 + lane) * 16));
                        }
#pragma unroll
                        for (int c = 0; c < 4; c++) acc[c] = fmaf(v[c], f[w][c & 1], acc[c]);
                    }
                    if (whole) {
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            const int h = 8 * nt + 2 * t + c;
                            if (h < heads) {
                                const float r = sum[c] == 0.0f ? 0.0f : 1.0f / sum[c];
                                *reinterpret_cast<uint32_t*>(A.out + (head0 + h) * HD + attn_v_dim<FMT, HD>(j, g)) =
                                    pack2(sum[c] == 0.0f ? 0.0f : acc[c] * r, sum[c] == 0.0f ? 0.0f : acc[c + 2] * r);
                            }
                        }
                    } else {
                        A.part_o[((size_t)slot * (NT * TILES) + x) * 32 + lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                    }
                }
                if (warp == 0 && g == 0) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int h = 8 * nt + 2 * t + c;
                        if (!whole) A.part_ml[(size_t)slot * (8 * NT) + h] = make_float2(top[c], sum[c]);
                        else if (A.lse != nullptr && h < heads)
                            A.lse[head0 + h] = sum[c] == 0.0f ? -INFINITY : (top[c] + log2f(sum[c])) * kLn2;
                    }
                }
            }
            if (i + 1 < steps) {
                at.step(A, items);
                began = true;
                begin_item();
            }
        } else {
            at.step(A, items);
        }
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
    const int part = blockIdx.x, nt = blockIdx.y;
    pdl_wait();
    pdl_trigger();
    const int2 d = A.desc[part];
    if (d.x < 0) return;
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
            const float sum = sum_s[2 * t + c], r = sum == 0.0f ? 0.0f : 1.0f / sum;
            *reinterpret_cast<uint32_t*>(A.out + (head0 + h) * HD + attn_v_dim<FMT, HD>(j, g)) =
                pack2(sum == 0.0f ? 0.0f : a[c] * r, sum == 0.0f ? 0.0f : a[c + 2] * r);
        }
    }
    if (A.lse != nullptr && tid < 8 && 8 * nt + tid < heads)
        A.lse[head0 + 8 * nt + tid] = sum_s[tid] == 0.0f ? -INFINITY : (top_s[tid] + log2f(sum_s[tid])) * kLn2;
}

/* Column tiles of 8 query heads an item holds: two where the group has more than eight heads
 * (head_dim 256: one, for the registers), the rest in further items of the same cache head. */
static int attn_col_tiles(int group, int head_dim) { return group > 8 && head_dim <= 128 ? 2 : 1; }

struct AttnScratch { size_t ml, o, bytes; };
static AttnScratch attn_scratch(int group, int head_dim) {
    const size_t heads = 8 * (size_t)attn_col_tiles(group, head_dim);
    AttnScratch s;
    s.ml = kAttnCtas * sizeof(int2);                                   /* 16-byte multiples */
    s.o = s.ml + 2 * kAttnCtas * heads * sizeof(float2);
    s.bytes = s.o + 2 * kAttnCtas * heads * head_dim * sizeof(float);
    return s;
}

template <int FMT, int HD, int NT>
static cudaError_t launch_attn(const AttnArgs& A, cudaStream_t s) {
    constexpr int SMEM = AttnShape<FMT, HD, NT>::SMEM;
    cudaError_t e = cudaFuncSetAttribute((const void*)attn_decode_kernel<FMT, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    e = launch_pdl(attn_decode_kernel<FMT, HD, NT>, dim3(kAttnCtas), dim3(32 * kAttnWarps), (size_t)SMEM, s, A);
    if (e != cudaSuccess) return e;
    e = launch_pdl(attn_join_kernel<FMT, HD, NT>, dim3(kAttnCtas, NT), dim3(kAttnJoinThreads), 0, s, A);
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
