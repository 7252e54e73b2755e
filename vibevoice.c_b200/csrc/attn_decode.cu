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
 * as rows would waste nine of sixteen. (tcgen05 wants 64 rows at least, both
 * operands of a product at hand behind barriers, and the weights back through
 * shared memory; at the rate HBM delivers, the tensor pipe of this kernel is
 * busy 14 % of the time in FP16, 28 % in FP8.)
 *
 * A warp takes 16 keys of one cache head at a time (two or four such groups a
 * step where rows are short). It copies their rows with cp.async into a ring of
 * its own, whole rows by neighbouring lanes: a request to L2 is then a whole
 * 128-byte line. (With each lane copying just the 16-byte pieces that its own
 * fragments need, which takes no data across lanes at all, requests are half
 * lines, and 64 x 4096 FP16 took 122.8 us, compute or no compute, instead of
 * 91.5.) The 16-byte pieces of a row lie permuted by bits of its number, so that
 * ldmatrix reads eight rows from eight banks; V through its transposing form,
 * which makes it the product's operand as it is. Between warps there is no
 * synchronisation until an item (a sequence's cache head) ends.
 *
 * FP8: e4m3 by cvt, two to an instruction; e5m2 is the upper half of an FP16
 * value and needs one byte permute. TurboQuant: two codes index a table in
 * shared memory of two FP16 levels, a copy for each lane, so that 32 lanes never
 * meet in a bank. 16 keys of the 4-bit format are 417 instructions a warp, all told,
 * 71 of them reads of shared memory (smsp__inst_executed over the groups of 48
 * sequences; FP16 328, E4M3 272): it is bound by its instructions and the latencies
 * between them, issue slots 52 % busy, three warps a scheduler (tried: entries 128
 * bytes apart, three CTAs of four warps with a table each: 61.6 us for 48 sequences
 * of 4100 - 8200; 256 apart, where one byte permute forms the address, and twelve
 * warps over one table: 58.9; fourteen and sixteen warps of fewer registers: 69, 84).
 *
 * Work: the blocks of 64 (128, 256, 384) positions of all items in one line, cut
 * into equal parts, one for each CTA that fits the GPU at once. The cut depends
 * on the lengths alone, which every warp sums up on the device, so the same
 * inputs give the same bits. (A line of less than 2^22 places is cut in 32-bit
 * numbers without a long division ahead of the first load: 0.45 us a call.) The
 * CTA's warps share each block. An item that a CTA holds whole is finished by it,
 * the warps' outputs exchanged in the ring's stage read last; of one that is cut,
 * each CTA leaves its part (running maximum, sum, output) in scratch and a second
 * kernel joins them. attn_whole says when items stay whole instead and the second
 * kernel is saved: by the room in the block tables, not by the lengths.
 *
 * Measured, replayed from a graph (28 heads over 4, 128 wide; GB/s of K and V):
 * 64 x 4096 FP16 87.9 us (86.2 .. 88.7 by box) = 6.11 TB/s, 0.93 of the device's
 * copy rate; 96 sequences of 1 .. 16384 58.1 us, 0.83; 48 of 4100 .. 8200 in E4M3
 * 55.0 us, 0.83; the same in 4 bits 60.6 us, 0.39, in 3 bits 83.7, 2 bits 62.6, 1.5
 * bits 71.8; 1 x 14449 FP16 12.4 us, latency: the first loads behind lens and
 * table, three steps, and the join. With tables of little more room than the
 * sequence, whole items in one kernel: 1 x 300 6.1, 1 x 64 3.6; with tables of 512
 * pages, cut: 7.2, 5.9. Bytes in flight: one stage of 8 KB for each of 12 warps an
 * SM beside the one being read; two stages are slower (64 x 4096 89.4 us where one
 * was 86.0), and so are two CTAs an SM (88.3).
 * A cluster of eight CTAs for an item, joined through distributed shared memory
 * in one launch, costs more than the second kernel (1 x 300, cut: 8.4 us, 7.1).
 *
 * Precision: scores, maximum, sums and outputs in FP32. A weight e^(s - m), times
 * 2^12, goes to the tensor cores as a pair of FP16 values, the one rounded toward
 * zero and the rest: one FP16 value alone would add an error as large as the
 * output's own rounding; below 2^-37 of the largest a weight is nothing. An infinity
 * in V meets two positive factors where its weight is 2^-20 of the largest or more
 * (weight_rest); under less it can make the sum a NaN, which is then looked up
 * (attn_infinite). The maximum follows the scores only beyond a factor of 2^3 (8 %
 * of the steps instead of 41 % for normal scores over 600 keys): 2^15 is the
 * largest weight then. For the rotated formats the levels times a common factor
 * become FP16 values within 9e-5 of themselves (attn_alpha, found by trying factors
 * in [1, 2); 1.6e-4 for the 1.5-bit code words), since the product takes FP16: it
 * costs 2.8e-4 of the output where its own rounding is 2.1e-4. The RMS of a key
 * multiplies its score, the RMS of V the weight, relative to a power of two that
 * follows the largest RMS.
 */
#include "fp8_kv.cuh"
#include "tq_kv.cuh"
#include "vvb_launch.h"

#include <atomic>

namespace vvb {

extern std::atomic<uint64_t> g_launches;

constexpr int kAttnPageShift = 6;
constexpr int kAttnSms = 148, kAttnParts = 3 * kAttnSms;      /* parts the work is cut into, at most */
constexpr int kAttnFewItems = 37;               /* so many items, in eight tiles each, are one wave of the joining kernel */
constexpr int kAttnJoinParts = 4, kAttnJoinChunk = 4;
constexpr int kAttnNarrow = 1 << 22;
constexpr int kAttnItemCost = 1;                /* what beginning and ending an item costs, in blocks */
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kWeightLog2 = 12.0f;            /* a weight of 1 is kept as 2^12 ... */
constexpr float kWeightTop = 15.0f;             /* ... and the maximum follows the scores once one passes 2^15 */
constexpr float kNoMax = -3e38f;
constexpr unsigned short kAttnMark = 0x7fff;    /* an output to look up (attn_infinite) */

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
    int2* desc;                /* cut items, see attn_join_kernel; -1: none. By item where there are few, else by part */
    float2* part_ml;           /* [2 kAttnParts][heads of an item] maximum, sum */
    float4* part_o;            /* [2 kAttnParts][tiles][32] output, in the lanes' layout */
    int n_seqs, n_q, n_kv, n_slots, table_stride, len_add;
    int group, head_blocks;    /* query heads to a cache head, items a cache head is cut into */
    int parts;                 /* CTAs of the launch */
    int by_item, whole_items, one_each;
    int narrow;                /* the line has fewer than kAttnNarrow places */
    float scale2;              /* scale * log2(e) */
};

/* ---------------------------------------------------------------- formats */

/* Rows of a group of 16 keys in shared memory: VEC bytes each, copied in units of UNIT. Where a row is 2, 4
 * or more 16-byte pieces the fragments are read with ldmatrix and the pieces are permuted for it (attn_place);
 * rows of 48 and 24 bytes lie as they are in the cache and are read in 32-bit words. */
template <int FMT, int HD> struct AttnFmt {
    static constexpr int VEC = kv_is_tq(FMT) ? tq_bytes_per_vec(FMT) : FMT == KV_RAW ? 2 * HD : HD;
    static constexpr bool MAT = FMT != KV_TQ3 && FMT != KV_TQ1_5;
    static constexpr int UNIT = FMT == KV_TQ1_5 ? 8 : 16;
    static constexpr int KG = VEC >= 256 ? 1 : VEC >= 64 ? 2 : 4;                     /* groups a warp takes in a step; the warps' groups are a block */
    static constexpr int W = FMT == KV_TQ4 ? 12 : 4;             /* warps of a CTA; the 4-bit code table is for many */
    static constexpr int KEYS = 16 * KG, BLOCK = W * KEYS;
    static constexpr int PER_ROW = VEC / UNIT, UNITS = KEYS * PER_ROW, COPIES = (UNITS + 31) / 32;    /* of a step, copies a lane makes */
    /* dims of a word that ldmatrix brings: of K a lane's 4 bytes, of V the 2 bytes of one key */
    static constexpr int K_DIMS = FMT == KV_RAW ? 2 : FMT == KV_TQ4 ? 8 : FMT == KV_TQ2 ? 16 : 4;
    /* entries of the code table: two codes -> two levels; 1.5 bits: code -> pair, then two keys' codes -> two pairs */
    static constexpr int LUT_STEP = FMT == KV_TQ4 ? 256 : 128;   /* bytes from entry to entry: 32 lanes' copies, and room */
    static constexpr int LUT = FMT == KV_TQ4 ? 256 : FMT == KV_TQ3 ? 64 : FMT == KV_TQ2 ? 16 : FMT == KV_TQ1_5 ? 8 + 128 : 0;
};

/* Factor that brings all the levels of a code book near FP16 values. */
template <int FMT> __host__ __device__ constexpr float attn_alpha() {
    return FMT == KV_TQ4 ? 1.2162726f : FMT == KV_TQ3 ? 1.4423765f : FMT == KV_TQ2 ? 1.8130219f : FMT == KV_TQ1_5 ? 1.0849942f : 1.0f;
}

template <int FMT, int HD, int NT> struct AttnShape {
    using F = AttnFmt<FMT, HD>;
    static constexpr int GROUP = 16 * F::VEC, ROWS = F::KG * GROUP;                           /* bytes of a group's K, or V; of a step's */
    static constexpr int USED = 2 * ROWS + (kv_is_tq(FMT) ? 8 * F::KEYS : 0);                 /* then the words that hold the rows' RMS values */
    static constexpr int OUT = NT * HD * 32;                                                  /* a warp's output, left in the stage it has read last */
    static constexpr int STAGE = USED > OUT ? USED : OUT;
    static constexpr int LUT = F::LUT * F::LUT_STEP;
    /* CTAs that an SM has registers for, and those that it has shared memory for too: the work is cut into a part for
     * each that is resident at once, and one more would be a wave of its own. Three stages of short rows, where as many
     * CTAs have room for them. (One CTA of 256-wide FP16 heads, two of 16 heads in 1.5 bits and three of 3 bits in two
     * stages, against one more that waited for room: 48 sequences of 4100 .. 8200 106.7 -> 100.5, 76.3 -> 52.9 and
     * 106.4 -> 85.2 us; 3 bits in three stages, two CTAs: 93.4.) */
    static constexpr int OF_SM = 228 << 10, OF_CTA = 1 << 10;                                 /* shared memory; what the system takes of it */
    static constexpr int STATIC = (F::W * (16 * NT + 1) * 4 + 4 + 127) / 128 * 128;           /* the kernel's own arrays */
    static constexpr int BY_REGS = F::W == 12 ? 1 : HD == 256 || NT == 2 ? 2 : 3;
    static constexpr int STAGES = FMT == KV_TQ4 || F::VEC * F::KG >= 256 || BY_REGS * (LUT + F::W * 3 * STAGE + STATIC + OF_CTA) > OF_SM ? 2 : 3;
    static constexpr int RING = STAGE * STAGES;                                               /* a warp's */
    static constexpr int TILES = HD / 16;                                                     /* 16-dim tiles of the output */
    static constexpr int MINE = (NT * TILES + F::W - 1) / F::W;                               /* of them a warp finishes */
    static constexpr int SMEM = LUT + F::W * RING;                                            /* in this order */
    static constexpr int BY_SMEM = OF_SM / (SMEM + STATIC + OF_CTA), CTAS = BY_REGS < BY_SMEM ? BY_REGS : BY_SMEM;
    static_assert(CTAS > 0, "a CTA fits an SM");
};

/* ---------------------------------------------------------------- instructions */

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
/* BYTES of global memory to shared memory at dst + AT; `some`: only n of them are read, the rest become zeros. */
template <int BYTES> __device__ __forceinline__ void cp_async(uint32_t dst, int at, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + at), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst + at), "l"(src), "n"(BYTES) : "memory");
}
template <int BYTES> __device__ __forceinline__ void cp_async_some(uint32_t dst, int at, const void* src, int n) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + at), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst + at), "l"(src), "n"(BYTES), "r"(n) : "memory");
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
/* The rest of two weights whose heads are `hi`: at least 2^-24 where the head is 2^-8 or more, so that an infinity in V
 * meets two positive factors; where the head is less than that, 2^-20 of the largest weight, the rest stays as it is,
 * since so much for each of many keys would add up (hi 2^-16 is 0 below 2^-9), and attn_infinite has the last word. */
__device__ __forceinline__ uint32_t weight_rest(uint32_t hi, uint32_t rest) {
    const __half2 s = __half2(__ushort_as_half(0x0100), __ushort_as_half(0x0100)), least = __half2(__ushort_as_half(1), __ushort_as_half(1));
    const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&rest), __hmin2(__hmul2(*reinterpret_cast<const __half2*>(&hi), s), least));
    return *reinterpret_cast<const uint32_t*>(&r);
}
/* Two outputs, and the log-sum-exp, from a head's sums (maximum and sum are those of weights times 2^12).
 * A sum of zero: no keys, or none with a score above -inf. A sum that is NaN: outputs 0x7e00; any other NaN is what
 * the conversion makes of it, kAttnMark, and `odd` says that there may be one. */
__device__ __forceinline__ uint32_t attn_out(float a, float b, float sum, bool& odd) {
    const float r = 1.0f / sum;
    a *= r;
    b *= r;
    if (a != a || b != b) odd = true;
    return sum == 0.0f ? 0u : sum != sum ? 0x7e007e00u : pack2(a, b);
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
/* Four FP8 values -> (0, 1) and (2, 3) as halves, or (SWAP) (0, 2) and (1, 3). An E5M2 byte is the upper half of
 * its FP16 value, so a byte permute is the whole conversion. */
template <int FMT, bool SWAP> __device__ __forceinline__ void fp8_halves(uint32_t w, uint32_t& a, uint32_t& b) {
    if constexpr (FMT == KV_E5M2) {
        a = __byte_perm(w, 0, SWAP ? 0x2404 : 0x1404);
        b = __byte_perm(w, 0, SWAP ? 0x3414 : 0x3424);
    } else {
        if (SWAP) w = __byte_perm(w, 0, 0x3120);
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
            : "=r"(a), "=r"(b) : "r"(w));
    }
}
__device__ __forceinline__ uint32_t lds32(uint32_t a, int at = 0) {
    uint32_t r;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r) : "r"(a + at));
    return r;
}
/* Four 8 x 8 matrices of 16-bit values; lane l gives the address of row l % 8 of matrix l / 8. */
__device__ __forceinline__ void ldmatrix4(uint32_t a, int at, uint32_t (&w)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a + at));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t a, int at, uint32_t (&w)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a + at));
}

extern __shared__ __align__(128) uint8_t attn_smem[];           /* the code table first: its address is then a constant */
/* Entry c / 128 of the code table, this lane's copy (c a multiple of 128 below the table's size). */
__device__ __forceinline__ uint32_t attn_lut(uint32_t c, uint32_t mask, uint32_t lane4, int from = 0) {
    return *reinterpret_cast<const uint32_t*>(attn_smem + from + ((c & mask) | lane4));
}

/* The same for byte k of w, entries 256 bytes apart: one byte permute puts the byte above the lane's offset. */
__device__ __forceinline__ uint32_t attn_lut_byte(uint32_t w, int k, uint32_t lane4) {
    return *reinterpret_cast<const uint32_t*>(attn_smem + __byte_perm(w, lane4, 0x7704 + (k << 4)));
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

/* Place of 16-byte piece c of row `row`: the eight rows an ldmatrix reads at one c lie in eight different
 * 16-byte banks. The permutation is an exclusive or of the piece's low bits with bits of the row. */
template <int VEC> __host__ __device__ constexpr int attn_place(int row, int c) {
    return VEC >= 128 ? row * VEC + ((c ^ (row & 7)) << 4)
         : VEC == 64 ? row * 64 + ((c ^ ((row >> 1) & 3)) << 4)
                     : row * VEC + ((c ^ ((row >> 2) & 1)) << 4);
}
/* The same for piece 2p + c, given a lane's address for piece c (the shared memory is 128-byte aligned). */
template <int VEC> __device__ __forceinline__ uint32_t attn_pair(uint32_t a, int p) { return a ^ (32u * (p & (VEC >= 128 ? 3 : 1))); }
__host__ __device__ constexpr int attn_pair_at(int p) { return 128 * (p >> 2); }

/* Dim of half 0 of word i of a lane's K row (half 1 is the next dim). */
template <int FMT> __device__ __forceinline__ int attn_k_dim(int i, int t) {
    constexpr int D = AttnFmt<FMT, 128>::K_DIMS;
    return AttnFmt<FMT, 128>::MAT ? (i / (D / 2)) * 4 * D + t * D + 2 * (i % (D / 2)) : 32 * t + 2 * i;
}
/* Dim of value e of a lane's V rows. */
template <int FMT> __device__ __forceinline__ int attn_v_dim(int e, int g) {
    constexpr int D = AttnFmt<FMT, 128>::K_DIMS / 2;
    return AttnFmt<FMT, 128>::MAT ? (e / D) * 8 * D + g * D + e % D : 16 * g + e;
}

/* Two dims' codes at bit `bit` of words w -> two halves. */
template <int FMT> __device__ __forceinline__ uint32_t attn_decode2(const uint32_t* w, int bit, uint32_t lane4) {
    constexpr int NB = FMT == KV_TQ3 ? 6 : FMT == KV_TQ2 ? 4 : 3;
    const int at = bit & 31;
    uint32_t c;                                        /* the codes times 128 */
    if (at + NB > 32) c = __funnelshift_r(w[bit >> 5], w[(bit >> 5) + 1], at) << 7;
    else c = at >= 7 ? w[bit >> 5] >> (at - 7) : w[bit >> 5] << (7 - at);
    return attn_lut(c, ((1u << NB) - 1u) << 7, lane4);
}

/* K of a group as fragments: words of row g (lo) and row g + 8 (hi). `a`: the lane's address in the group's K. */
template <int FMT, int HD>
__device__ __forceinline__ void attn_load_k(uint32_t a, int t, uint32_t (&lo)[HD / 8], uint32_t (&hi)[HD / 8], uint32_t lane4) {
    using F = AttnFmt<FMT, HD>;
    if constexpr (F::MAT) {
        constexpr int W = F::K_DIMS / 2;               /* halves' words of a word */
#pragma unroll
        for (int p = 0; p < F::PER_ROW / 2; p++) {     /* matrices: rows 0-7 and 8-15 of piece 2p, of piece 2p + 1 */
            uint32_t w[4];
            ldmatrix4(attn_pair<F::VEC>(a, p), attn_pair_at(p), w);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int i = (2 * p + k) * W;
                if constexpr (FMT == KV_RAW) {
                    lo[i] = w[2 * k];
                    hi[i] = w[2 * k + 1];
                } else if constexpr (!kv_is_tq(FMT)) {
                    fp8_halves<FMT, false>(w[2 * k], lo[i], lo[i + 1]);
                    fp8_halves<FMT, false>(w[2 * k + 1], hi[i], hi[i + 1]);
                } else {
#pragma unroll
                    for (int x = 0; x < W; x++) {
                        lo[i + x] = FMT == KV_TQ4 ? attn_lut_byte(w[2 * k], x, lane4) : attn_decode2<FMT>(&w[2 * k], 32 / W * x, lane4);
                        hi[i + x] = FMT == KV_TQ4 ? attn_lut_byte(w[2 * k + 1], x, lane4) : attn_decode2<FMT>(&w[2 * k + 1], 32 / W * x, lane4);
                    }
                }
            }
        }
    } else {
        constexpr int N = FMT == KV_TQ3 ? 3 : 2, NB = FMT == KV_TQ3 ? 6 : 3;
        uint32_t w[2][N + 1];
#pragma unroll
        for (int r = 0; r < 2; r++) {
#pragma unroll
            for (int n = 0; n < N; n++) w[r][n] = lds32(a, 8 * r * F::VEC + 4 * n);
            if constexpr (FMT == KV_TQ1_5) {           /* the lane's 6 bytes begin in the middle of a word for odd t */
                const int sh = (t & 1) * 16;
                w[r][0] = __funnelshift_r(w[r][0], w[r][1], sh);
                w[r][1] >>= sh;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            lo[i] = attn_decode2<FMT>(w[0], NB * i, lane4);
            hi[i] = attn_decode2<FMT>(w[1], NB * i, lane4);
        }
    }
}
/* V of a group: xa[e] = keys (2t, 2t + 1), xc[e] = keys (2t + 8, 2t + 9) at the lane's value e. */
template <int FMT, int HD>
__device__ __forceinline__ void attn_load_v(uint32_t a, int g, uint32_t (&xa)[HD / 8], uint32_t (&xc)[HD / 8], uint32_t lane4) {
    using F = AttnFmt<FMT, HD>;
    if constexpr (F::MAT) {
#pragma unroll
        for (int p = 0; p < F::PER_ROW / 2; p++) {
            uint32_t w[4];                             /* as K's, transposed: a word is (key 2t, key 2t + 1) */
            ldmatrix4_trans(attn_pair<F::VEC>(a, p), attn_pair_at(p), w);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t(&x)[HD / 8] = (FMT == KV_RAW ? k >> 1 : k & 1) ? xc : xa;
                const int c = 2 * p + (FMT == KV_RAW ? k & 1 : k >> 1);
                if constexpr (FMT == KV_RAW) {
                    x[c] = w[k];
                } else if constexpr (!kv_is_tq(FMT)) {
                    fp8_halves<FMT, true>(w[k], x[2 * c], x[2 * c + 1]);
                } else if constexpr (FMT == KV_TQ4) {
                    /* A's dims 0, 1 and 2, 3 of the four, B's: pairs by dim, then interleaved */
                    const uint32_t a0 = attn_lut_byte(w[k], 0, lane4), a1 = attn_lut_byte(w[k], 1, lane4);
                    const uint32_t b0 = attn_lut_byte(w[k], 2, lane4), b1 = attn_lut_byte(w[k], 3, lane4);
                    x[4 * c] = __byte_perm(a0, b0, 0x5410);
                    x[4 * c + 1] = __byte_perm(a0, b0, 0x7632);
                    x[4 * c + 2] = __byte_perm(a1, b1, 0x5410);
                    x[4 * c + 3] = __byte_perm(a1, b1, 0x7632);
                } else {
                    uint32_t even = w[k] & 0x33333333u, odd = (w[k] >> 2) & 0x33333333u;      /* every other code, A's in the low half */
                    even |= even >> 14;                /* fields of 4 bits: A0 B0, A2 B2, .. */
                    odd |= odd >> 14;
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        x[8 * c + 2 * y] = attn_lut(4 * y >= 7 ? even >> (4 * y - 7) : even << (7 - 4 * y), 0x780u, lane4);
                        x[8 * c + 2 * y + 1] = attn_lut(4 * y >= 7 ? odd >> (4 * y - 7) : odd << (7 - 4 * y), 0x780u, lane4);
                    }
                }
            }
        }
    } else {
        constexpr int W = 3, N = FMT == KV_TQ1_5 ? 8 : 16;      /* codes of a lane's 24 or 48 bits of a row */
        uint32_t w[4][2];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int sh = 8 * (((FMT == KV_TQ3 ? 6 : 3) * g) & 3);
            const uint32_t w0 = lds32(a, ((r & 1) + 8 * (r >> 1)) * F::VEC), w1 = lds32(a, ((r & 1) + 8 * (r >> 1)) * F::VEC + 4);
            w[r][0] = __funnelshift_r(w0, w1, sh);
            w[r][1] = w1 >> sh;
        }
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            uint32_t(&x)[HD / 8] = r ? xc : xa;
#pragma unroll
            for (int e = 0; e < N; e++) {
                const int bit = W * e;
                uint32_t c[2];
#pragma unroll
                for (int k = 0; k < 2; k++)
                    c[k] = (bit + W <= 32 ? w[r + k][0] >> bit : bit >= 32 ? w[r + k][1] >> (bit - 32) : __funnelshift_r(w[r + k][0], w[r + k][1], bit)) & 7u;
                const uint32_t both = (c[0] | (c[1] << W)) << 7;
                if constexpr (FMT == KV_TQ1_5) {
                    x[2 * e] = attn_lut(both, ~0u, lane4, 8 * 128);
                    x[2 * e + 1] = attn_lut(both, ~0u, lane4, (8 + 64) * 128);
                } else {
                    x[e] = attn_lut(both, ~0u, lane4);
                }
            }
        }
    }
}
/* A lane's address in a group's K, and in its V, relative to their beginning. */
template <int FMT, int HD> __device__ __forceinline__ uint32_t attn_k_at(int lane) {
    using F = AttnFmt<FMT, HD>;
    if (F::MAT) return attn_place<F::VEC>((lane & 7) + (lane & 8), lane >> 4);
    return (lane >> 2) * F::VEC + (FMT == KV_TQ3 ? 12 * (lane & 3) : (6 * (lane & 3)) & ~3);
}
template <int FMT, int HD> __device__ __forceinline__ uint32_t attn_v_at(int lane) {
    using F = AttnFmt<FMT, HD>;
    if (FMT == KV_RAW) return attn_place<F::VEC>((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);      /* order of the product's operand */
    if (F::MAT) return attn_place<F::VEC>((lane & 7) + (lane & 8), lane >> 4);
    return 2 * (lane & 3) * F::VEC + (((FMT == KV_TQ3 ? 6 : 3) * (lane >> 2)) & ~3);
}

/* A lane's values 2 j and 2 j + 1 of a head's output. */
template <int FMT> __device__ __forceinline__ void attn_store(__half* out, int j, int g, uint32_t two) {
    if constexpr (FMT == KV_RAW) {
        const __half2 h = *reinterpret_cast<const __half2*>(&two);
        out[attn_v_dim<FMT>(2 * j, g)] = __low2half(h);
        out[attn_v_dim<FMT>(2 * j + 1, g)] = __high2half(h);
    } else {
        *reinterpret_cast<uint32_t*>(out + attn_v_dim<FMT>(2 * j, g)) = two;
    }
}

/* ---------------------------------------------------------------- work */

/* Number of keys of sequence b: no more than its table, or its stretch of the contiguous cache, has places for. */
__device__ __forceinline__ int attn_keys(const AttnArgs& A, int b) {
    const long long cap = A.block_table != nullptr ? (long long)A.table_stride << kAttnPageShift
                                                   : min((long long)A.table_stride, (long long)A.n_slots - (long long)b * A.table_stride);
    const long long n = (long long)__ldg(A.lens + b) + A.len_add;
    return (int)max(min(min(n, cap), 0x7fffff00ll), 0ll);
}
template <int BLOCK> __device__ __forceinline__ int attn_blocks(int n) { return (int)(((unsigned)n + (BLOCK - 1)) / BLOCK); }
template <int BLOCK> __device__ __forceinline__ int attn_places(int n) { return n > 0 ? attn_blocks<BLOCK>(n) + kAttnItemCost : 0; }
/* A place in the line of blocks: block blk of nb of item h (cache head x head block) of sequence b. */
template <int BLOCK> struct AttnAt {
    int b, h, hk, blk, nb, n, n_next;                  /* cache head hk; n keys here, n_next in sequence b + 1 */
    __device__ __forceinline__ void set(const AttnArgs& A, int seq, int item, int block) {
        b = seq;
        h = item;
        hk = A.head_blocks == 1 ? h : h / A.head_blocks;
        blk = block;
        n = attn_keys(A, b);
        nb = attn_blocks<BLOCK>(n);
        n_next = b + 1 < A.n_seqs ? attn_keys(A, b + 1) : 0;
    }
    __device__ __forceinline__ bool last() const { return blk + 1 >= nb; }                    /* of the item */
    __device__ __forceinline__ void next_item(const AttnArgs& A, int items) {
        blk = 0;
        if (++h < items) {
            hk = A.head_blocks == 1 ? h : h / A.head_blocks;
            return;
        }
        h = hk = 0;
        do {
            b++;
            n = n_next;
            n_next = b + 1 < A.n_seqs ? attn_keys(A, b + 1) : 0;
        } while (n == 0 && b < A.n_seqs);
        nb = attn_blocks<BLOCK>(n);
    }
};

/* The sign of the stored value at `dim` of a row of V that holds codes (none of the levels is 0). */
template <int FMT> __device__ __forceinline__ bool attn_code_negative(const uint8_t* row, int dim) {
    constexpr int NB = FMT == KV_TQ4 ? 4 : FMT == KV_TQ2 ? 2 : 3;
    const int bit = NB * (FMT == KV_TQ1_5 ? dim >> 1 : dim);
    unsigned w = row[bit >> 3];
    if ((bit & 7) + NB > 8) w |= (unsigned)row[(bit >> 3) + 1] << 8;
    const unsigned c = (w >> (bit & 7)) & ((1u << NB) - 1u);
    return FMT == KV_TQ1_5 ? c_vq15[2 * c + (dim & 1)] < 0.0f : c < (1u << (NB - 1));
}
/* Outputs that attn_out has marked, of `heads` heads of cache head hk of sequence b, at sixteen dims; by a warp, once
 * they are all written. What such a NaN stands for are infinities in V: they have their sign in the result under any
 * weight of a finite score, but are NaN where the weight, or a half of it, is 0 in FP16 or in FP32. So V is looked
 * through at those dims, a key a lane. That happens to infinite values only, and takes what reading V of sixteen
 * dims by one warp does: 64 x 4096 255 us with infinities in one dim, 637 in all, 1 x 14449 320. (Infinities of both signs and NaNs give NaN. V of a key whose score is -inf counts as any.) */
template <int FMT, int HD, typename Dim>
__device__ __forceinline__ void attn_infinite(const AttnArgs& A, int b, int hk, __half* out, int heads, Dim dim_of, int lane) {
    constexpr int VEC = AttnFmt<FMT, HD>::VEC;
    const int mine = dim_of(lane & 15);
    bool marked = false;
    for (int h = lane >> 4; h < heads; h += 2) marked |= __half_as_ushort(out[h * HD + mine]) == kAttnMark;
    if (!__any_sync(0xffffffffu, marked)) return;
    const int n = attn_keys(A, b);
    unsigned pos = 0, neg = 0, nan = 0;                /* a bit a dim */
#pragma unroll 1
    for (int j = lane; j < n; j += 32) {
        long long row = (long long)b * A.table_stride + j;
        if (A.block_table != nullptr) {
            const int page = __ldg(A.block_table + (size_t)b * A.table_stride + (j >> kAttnPageShift));
            if ((unsigned)page > (unsigned)(A.n_slots - 1) >> kAttnPageShift) continue;
            row = ((long long)page << kAttnPageShift) + (j & 63);
        }
        if (row >= A.n_slots) continue;
        const size_t at = (size_t)row * A.n_kv + hk;
        if constexpr (kv_is_tq(FMT)) {
            const float rms = __half2float(A.v_meta[at]);
            if (rms != rms) nan = 0xffffu;
            if (rms == INFINITY)
                for (int k = 0; k < 16; k++) (attn_code_negative<FMT>(A.v_store + at * VEC, dim_of(k)) ? neg : pos) |= 1u << k;
        } else {
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const float v = FMT == KV_RAW ? __half2float(reinterpret_cast<const __half*>(A.v_store)[at * HD + dim_of(k)])
                                              : __half2float(__ushort_as_half((unsigned short)(A.v_store[at * VEC + dim_of(k)] << 8)));
                nan |= (v != v ? 1u : 0u) << k;
                pos |= (v == INFINITY ? 1u : 0u) << k;
                neg |= (v == -INFINITY ? 1u : 0u) << k;
            }
        }
    }
    pos = __reduce_or_sync(0xffffffffu, pos);
    neg = __reduce_or_sync(0xffffffffu, neg);
    nan = __reduce_or_sync(0xffffffffu, nan) | ~(pos ^ neg);
    const unsigned bit = 1u << (lane & 15);
    if (nan & bit) return;
    for (int h = lane >> 4; h < heads; h += 2)
        if (__half_as_ushort(out[h * HD + mine]) == kAttnMark) out[h * HD + mine] = __ushort_as_half(pos & bit ? 0x7c00 : 0xfc00);
}
/* All outputs of items first .. last (whole ones, by their places in the line), by warps `warp` of `warps`. */
template <int FMT, int HD> __device__ __noinline__ void attn_look_up(const AttnArgs& A, int first, int last, int heads_of, int warp, int warps) {
    const int items = A.n_kv * A.head_blocks;
    for (int i = first; i <= last; i++) {
        const int b = i / items, h = i - b * items, hk = h / A.head_blocks, h0 = (h - hk * A.head_blocks) * heads_of;
        if (attn_keys(A, b) == 0) continue;            /* zeros, perhaps another CTA's, and perhaps not written yet */
        __half* const out = A.out + ((size_t)b * A.n_q + (size_t)hk * A.group + h0) * HD;
        for (int d0 = 16 * warp; d0 < HD; d0 += 16 * warps)
            attn_infinite<FMT, HD>(A, b, hk, out, min(heads_of, A.group - h0), [d0](int k) { return d0 + k; }, threadIdx.x & 31);
    }
}

/* floor(a / b) for 0 <= a < kAttnNarrow, 0 < b <= kAttnNarrow. Both are exact as floats and the quotient is off by
 * 2 units in the last place, 2^-22 of less than 2^22: its floor is one off at most. */
__device__ __forceinline__ int attn_div(int a, int b) {
    int q = (int)__fdividef((float)a, (float)b);
    q -= q * b > a;
    q += (q + 1) * b <= a;
    return q;
}
__device__ __forceinline__ long long attn_div(long long a, long long b) { return a / b; }

template <int FMT, int HD, int NT, bool SOLO>
__global__ void __launch_bounds__(32 * AttnFmt<FMT, HD>::W, AttnShape<FMT, HD, NT>::CTAS) attn_decode_kernel(const __grid_constant__ AttnArgs A) {
    using F = AttnFmt<FMT, HD>;
    using S = AttnShape<FMT, HD, NT>;
    constexpr bool TQ = kv_is_tq(FMT);
    constexpr int W = F::W, TILES = S::TILES, MINE = S::MINE;    /* tiles of the output, those a warp finishes */
    constexpr int BLOCK = SOLO ? F::KEYS : F::BLOCK;   /* a warp alone takes a block by itself */
    __shared__ float m_s[W][8 * NT], l_s[W][8 * NT], f_s[W];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int warp_key = SOLO ? 0 : F::KEYS * warp;    /* of the block: the warp's first */
    const uint32_t smem0 = (uint32_t)__cvta_generic_to_shared(attn_smem);
    const uint32_t ring = smem0 + S::LUT + warp * S::RING;
    const uint32_t lane4 = 4 * lane;                   /* this lane's copy of the table */

    if constexpr (F::LUT > 0) {
        for (int e = warp; e < F::LUT; e += W) *reinterpret_cast<uint32_t*>(attn_smem + F::LUT_STEP * e + lane4) = attn_lut_entry<FMT>(e);
        if (SOLO) __syncthreads();
    }
    pdl_wait();

    /* This CTA's (SOLO: warp's) part of the line: sum the sequences' blocks, then find where the part begins. Each
     * item counts kAttnItemCost places more than it has blocks, ahead of its first block. Every warp does it for
     * itself, a lane for every 32nd of the sequences. */
    const int items = A.n_kv * A.head_blocks;
    const bool whole_items = SOLO || A.whole_items;    /* an item belongs to the part in which it begins */
    const int part = SOLO ? blockIdx.x * W + warp : blockIdx.x;
    AttnAt<BLOCK> to, at;                              /* what is copied next, what is computed next */
    int places = 0, skipped = 0;                       /* of the line that are left to this part; ahead of its first block */
    long long u0 = 0, largest = 1;                     /* the part's first place, and how many a part has */
    if (A.one_each) {                                  /* fewer items than CTAs, whole: item number `part` */
        const int b = part / items;
        if (b < A.n_seqs) {
            to.set(A, b, part - b * items, 0);
            places = to.nb;
        }
    } else {
        auto find = [&](auto zero) {                   /* in 32-bit numbers where they do: it is 0.8 us before the first load */
            using T = decltype(zero);
            const int per = (A.n_seqs + 31) / 32, s0 = min(lane * per, A.n_seqs), s1 = min(s0 + per, A.n_seqs);
            T mine = 0;
#pragma unroll 4
            for (int b = s0; b < s1; b++) mine += attn_places<BLOCK>(attn_keys(A, b));
            T upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const T x = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += x;
            }
            const T total = __shfl_sync(0xffffffffu, upto, 31) * items, before = (upto - mine) * items;
            if (total == 0) return;
            /* as few parts as make the largest no larger: 908 places on 444 CTAs are 303 parts of three, not 444 of two or three */
            const T most = SOLO ? gridDim.x * W : gridDim.x;
            const T each = max(attn_div(total + most - 1, most), (T)(1 + kAttnItemCost));
            const T first = min((T)part * each, total), end = min(first + each, total);
            u0 = first;
            largest = each;
            places = (int)(end - first);
            if (places <= 0) return;
            const int who = __ffs(__ballot_sync(0xffffffffu, first >= before && first < before + mine * items)) - 1;
            int b = 0;
            T in = 0;                                  /* place in sequence b's stretch of the line */
            if (lane == who) {
                in = first - before;
                for (b = s0; b < s1; b++) {
                    const T stretch = (T)attn_places<BLOCK>(attn_keys(A, b)) * items;
                    if (in < stretch) break;
                    in -= stretch;
                }
            }
            b = __shfl_sync(0xffffffffu, b, who);
            in = __shfl_sync(0xffffffffu, in, who);
            const int np = attn_places<BLOCK>(attn_keys(A, b));
            const int item = (int)attn_div(in, (T)np), off = (int)(in - (T)item * np);
            to.set(A, b, item, max(off - kAttnItemCost, 0));
            skipped = max(kAttnItemCost - off, 0);     /* the places ahead of the item's first block */
            if (whole_items && off > 0) {              /* begun in an earlier part */
                skipped = np - off + kAttnItemCost;
                if (places > np - off) to.next_item(A, items);
            }
            places -= skipped;
            if (whole_items) places = places + kAttnItemCost > 0 ? max(places, 1) : 0;
        };
        if (A.narrow) find(0);
        else find(0ll);
    }
    /* rows without keys */
    for (int b = blockIdx.x; b < A.n_seqs; b += gridDim.x) {
        if (attn_keys(A, b) > 0) continue;
        uint32_t* o = reinterpret_cast<uint32_t*>(A.out + (size_t)b * A.n_q * HD);
        for (int i = tid; i < A.n_q * HD / 2; i += 32 * W) o[i] = 0;
        if (A.lse != nullptr)
            for (int i = tid; i < A.n_q; i += 32 * W) A.lse[(size_t)b * A.n_q + i] = -INFINITY;
        if (A.by_item && tid < items) A.desc[b * items + tid] = make_int2(-1, 0);
    }
    if (places <= 0) {
        if (!whole_items && tid == 0 && !A.by_item) A.desc[part] = make_int2(-1, 0);
        return;
    }
    at = to;
    bool began = at.blk == 0;                          /* this part holds the beginning of the item */
    [[maybe_unused]] __shared__ int first_s[SOLO ? W : 1];       /* the first item that is whole here, for the look-up at the end */
    if (SOLO ? lane == 0 : tid == 0) first_s[SOLO ? warp : 0] = at.b * items + at.h + (began ? 0 : 1);
    bool odd = false;

    /* What is copied next: units lane, lane + 32, .. of the group's rows. The pointers are those of the first
     * of them in row 0 of the cache. */
    const uint32_t row_bytes = (uint32_t)A.n_kv * F::VEC;
    const uint8_t *klane, *vlane;
    int row_to;                                        /* cache row of the warp's first key, -1: none; read one step ahead */
    const uint32_t lane_off = (lane / F::PER_ROW) * row_bytes + (lane % F::PER_ROW) * F::UNIT;
    auto copy_off = [&](int i) -> size_t {             /* of copy i beyond the lane's first */
        if constexpr (32 % F::PER_ROW == 0) return (size_t)(i * (32 / F::PER_ROW)) * row_bytes;
        else return (size_t)((32 * i + lane) / F::PER_ROW) * row_bytes + (32 * i + lane) % F::PER_ROW * F::UNIT - lane_off;
    };
    auto copy_row = [&](int i) -> int { return 32 % F::PER_ROW == 0 ? i * (32 / F::PER_ROW) + lane / F::PER_ROW : (32 * i + lane) / F::PER_ROW; };
    /* where unit 32 i + lane goes: an exclusive or of the lane's first place with bits of i, or the same order */
    const uint32_t lane_dst = F::MAT ? attn_place<F::VEC>(lane / F::PER_ROW, lane % F::PER_ROW) : lane * F::UNIT;
    auto copy_dst = [](uint32_t d, int i) -> uint32_t {
        constexpr int R = 32 / F::PER_ROW;             /* rows of a copy */
        return F::MAT && F::VEC >= 128 ? d ^ (16u * ((i * R) & 7)) : d;
    };
    auto aim_item = [&]() {
        klane = A.k_store + to.hk * F::VEC + lane_off;
        vlane = A.v_store + to.hk * F::VEC + lane_off;
    };
    auto aim = [&]() {                                 /* this warp's rows of block to.blk: never across a page */
        const int at = to.blk * BLOCK + warp_key;
        row_to = -1;
        if (at < to.n) {
            if (A.block_table != nullptr) {
                const int page = __ldg(A.block_table + (size_t)to.b * A.table_stride + (at >> kAttnPageShift));
                if ((unsigned)page <= (unsigned)(A.n_slots - 1) >> kAttnPageShift) row_to = (page << kAttnPageShift) + (at & 63);
            } else {
                const long long row = (long long)to.b * A.table_stride + at;
                if (row < A.n_slots) row_to = (int)row;
            }
        }
    };
    aim_item();
    aim();
    int to_places = places;                            /* places from `to` on */
    bool to_more = true;                               /* something is left to copy */
    const bool odd_end = TQ && (((size_t)A.n_slots * A.n_kv) & 1) != 0;      /* the last RMS value stands alone in its word */
    auto issue = [&](int stage) -> int {               /* returns how many of the warp's 16 rows hold keys */
        int live = 0;
        if (to_more) {
            const uint32_t base = ring + stage * S::STAGE, kd = base + lane_dst, md = base + 2 * S::ROWS + lane4;
            const int row0 = row_to;
            live = row_to < 0 ? 0 : min(min(to.n - to.blk * BLOCK - warp_key, A.n_slots - row0), F::KEYS);
            if (live == F::KEYS && !(TQ && odd_end && row0 + F::KEYS >= A.n_slots)) {
                const uint8_t* kp = klane + (size_t)(uint32_t)row0 * row_bytes;
                const uint8_t* vp = vlane + (size_t)(uint32_t)row0 * row_bytes;
#pragma unroll
                for (int i = 0; i < F::COPIES; i++) {
                    if (F::UNITS % 32 != 0 && 32 * i + lane >= F::UNITS) continue;
                    cp_async<F::UNIT>(copy_dst(kd, i), 32 * F::UNIT * i, kp + copy_off(i));
                    cp_async<F::UNIT>(copy_dst(kd, i), S::ROWS + 32 * F::UNIT * i, vp + copy_off(i));
                }
                if constexpr (TQ) {
                    /* the RMS values: for each row the 32-bit word that holds it, K's rows, then V's */
#pragma unroll
                    for (int i = 0; i < F::KG; i++) {
                        const int w = 32 * i + lane;
                        const size_t at = (((size_t)(uint32_t)(row0 + w % F::KEYS) * A.n_kv + to.hk) * 2) & ~(size_t)3;
                        cp_async<4>(md, 128 * i, reinterpret_cast<const uint8_t*>(w < F::KEYS ? A.k_meta : A.v_meta) + at);
                    }
                }
            } else if (live > 0) {
                /* rows behind the last key are filled with zeros, nothing of them is read */
                const size_t first = (size_t)(uint32_t)row0 * row_bytes;
#pragma unroll
                for (int i = 0; i < F::COPIES; i++) {
                    if (F::UNITS % 32 != 0 && 32 * i + lane >= F::UNITS) continue;
                    const bool ok = copy_row(i) < live;
                    const size_t off = ok ? first + copy_off(i) : 0;
                    cp_async_some<F::UNIT>(copy_dst(kd, i), 32 * F::UNIT * i, ok ? klane + off : A.k_store, ok ? F::UNIT : 0);
                    cp_async_some<F::UNIT>(copy_dst(kd, i), S::ROWS + 32 * F::UNIT * i, ok ? vlane + off : A.v_store, ok ? F::UNIT : 0);
                }
                if constexpr (TQ) {
                    const size_t end = (size_t)A.n_slots * A.n_kv * 2;         /* bytes of an array */
#pragma unroll
                    for (int i = 0; i < F::KG; i++) {
                        const int w = 32 * i + lane, row = w % F::KEYS;
                        const bool ok = row < live;
                        const size_t at = ok ? (((size_t)(uint32_t)(row0 + row) * A.n_kv + to.hk) * 2) & ~(size_t)3 : 0;
                        cp_async_some<4>(md, 128 * i, reinterpret_cast<const uint8_t*>(w < F::KEYS ? A.k_meta : A.v_meta) + at, !ok ? 0 : at + 4 > end ? 2 : 4);
                    }
                }
            }
            live = max(live, 0);
            to_places--;
            const bool ends = to.last();
            to_more = whole_items ? !ends || to_places > 0 : to_places > (ends ? kAttnItemCost : 0);
            if (to_more) {
                if (ends) {
                    to_places -= kAttnItemCost;
                    to.next_item(A, items);
                    aim_item();
                } else {
                    to.blk++;
                }
                aim();
            }
        }
        cp_commit();
        return live;
    };
    int live_q[S::STAGES];                             /* of the stages in flight, oldest first */
#pragma unroll
    for (int s = 0; s < S::STAGES - 1; s++) live_q[s] = issue(s);

    uint32_t q[NT][HD / 8];
    auto load_q = [&](const AttnAt<BLOCK>& x) {
        const int h0 = (x.h - x.hk * A.head_blocks) * 8 * NT, heads = A.group - h0;      /* of this block: at most 8 NT */
        const __half* src = A.q + ((size_t)x.b * A.n_q + (size_t)x.hk * A.group + h0) * HD;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < HD / 8; i++)
                q[nt][i] = 8 * nt + g < heads ? *reinterpret_cast<const uint32_t*>(src + (size_t)(8 * nt + g) * HD + attn_k_dim<FMT>(i, t)) : 0u;
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
    /* the item that ends here and began in an earlier part; which one it began in follows from the cut */
    if (!whole_items && tid == 0) {
        int2 d = make_int2(-1, 0);
        if (!began && places >= at.nb - at.blk) {
            const long long first = u0 + skipped - at.blk;       /* place of the item's first block */
            const int p = (int)(A.narrow ? (unsigned)first / (unsigned)largest : first / largest);
            d = make_int2(A.by_item ? part : at.b * items + at.h, p);
        }
        if (!A.by_item) A.desc[part] = d;
        else if (d.x >= 0) A.desc[at.b * items + at.h] = d;
    }

    if (F::LUT > 0 && !SOLO) __syncthreads();          /* the code table */
    const uint32_t k_at = attn_k_at<FMT, HD>(lane), v_at = attn_v_at<FMT, HD>(lane);
    int stage = 0;
    for (;;) {
        /* Waiting first keeps one stage less in flight, which is enough, and better: 64 x 4096 86.0 us, 89.4 when the
         * copies are issued ahead of the wait. */
        cp_wait<S::STAGES - 2>();
        __syncwarp();                                  /* every lane's copies are there, and all have read the slot before */
        live_q[S::STAGES - 1] = issue(stage == 0 ? S::STAGES - 1 : stage - 1);     /* into the slot that the previous step emptied */
        const int live = live_q[0];
#pragma unroll
        for (int s = 0; s + 1 < S::STAGES; s++) live_q[s] = live_q[s + 1];
        const uint32_t base = ring + stage * S::STAGE;
        if (++stage == S::STAGES) stage = 0;
        float s[F::KG][NT][4];
        if (live > 0) {                                /* uniform over the warp */
#pragma unroll
            for (int gi = 0; gi < F::KG; gi++) {
                uint32_t klo[HD / 8], khi[HD / 8];
                attn_load_k<FMT, HD>(base + gi * S::GROUP + k_at, t, klo, khi, lane4);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float s0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int ks = 0; ks < HD / 16; ks += 2) {
                        mma16816(s0, klo[2 * ks], khi[2 * ks], klo[2 * ks + 1], khi[2 * ks + 1], q[nt][2 * ks], q[nt][2 * ks + 1]);
                        mma16816(s1, klo[2 * ks + 2], khi[2 * ks + 2], klo[2 * ks + 3], khi[2 * ks + 3], q[nt][2 * ks + 2], q[nt][2 * ks + 3]);
                    }
#pragma unroll
                    for (int c = 0; c < 4; c++) s[gi][nt][c] = s0[c] + s1[c];
                }
            }
        }
        /* the next item's Q is on its way while this one is finished */
        const bool item_done = at.last();
        places--;
        const bool more = whole_items ? !item_done || places > 0 : places > (item_done ? kAttnItemCost : 0);
        AttnAt<BLOCK> nx = at;
        if (!item_done) {
            nx.blk++;
        } else if (more) {
            nx.next_item(A, items);
            load_q(nx);
        }
        if (live > 0) {
            float sv[F::KG][2], sv_top = 0.0f;
            if constexpr (TQ) {
                const uint32_t mb = base + 2 * S::ROWS + 4 * g;
                /* which half of the word: the parity of the value's index (a warp's first position is even, and so is 8) */
                const int bk = A.block_table != nullptr ? 0 : (int)(((long long)at.b * A.table_stride) & 1);
                const int shift = (((bk + g) * A.n_kv + at.hk) & 1) * 16;
#pragma unroll
                for (int gi = 0; gi < F::KG; gi++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const float sk = __half2float(__ushort_as_half((unsigned short)(lds32(mb, 64 * gi + 32 * r) >> shift)));
                        const float f = A.scale2 * (sk * (1.0f / attn_alpha<FMT>()));
                        sv[gi][r] = __half2float(__ushort_as_half((unsigned short)(lds32(mb, 64 * F::KG + 64 * gi + 32 * r) >> shift)));
                        sv_top = fmaxf(sv_top, sv[gi][r]);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int c = 0; c < 2; c++) s[gi][nt][2 * r + c] *= f;
                    }
            } else {
#pragma unroll
                for (int gi = 0; gi < F::KG; gi++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int c = 0; c < 4; c++) s[gi][nt][c] *= A.scale2;
            }
            /* scores in base 2; rows behind the last key have none */
            if (live < F::KEYS) {
#pragma unroll
                for (int gi = 0; gi < F::KG; gi++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int c = 0; c < 4; c++)
                            if (16 * gi + g + 8 * (c >> 1) >= live) s[gi][nt][c] = -INFINITY;
            }
            bool up = TQ && sv_top > vref;
#pragma unroll
            for (int gi = 0; gi < F::KG; gi++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) up |= s[gi][nt][c] > m[nt][c & 1] + kWeightTop;
            if (__any_sync(0xffffffffu, up)) {
                /* a new maximum (or a larger RMS of V): rescale what there is */
                float rv = 1.0f;
                if constexpr (TQ) {
                    float x = sv_top;
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    if (x > vref) {                    /* the next power of two above it, or above all finite ones */
                        const float nref = x < INFINITY ? __uint_as_float((__float_as_uint(x) & 0x7f800000u) + 0x00800000u) : 65536.0f;
                        rv = vref / nref;
                        vref = nref;
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float x = fmaxf(s[0][nt][c], s[0][nt][c + 2]);
#pragma unroll
                        for (int gi = 1; gi < F::KG; gi++) x = fmaxf(x, fmaxf(s[gi][nt][c], s[gi][nt][c + 2]));
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
            const float inv = 1.0f / vref;             /* (a power of two) */
#pragma unroll
            for (int gi = 0; gi < F::KG; gi++) {
                /* weights: FP32 sums, FP16 pairs for the product */
                uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        float w[2];
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            w[c] = ex2(s[gi][nt][2 * r + c] - m[nt][c]);
                            l[nt][c] += w[c];
                            if constexpr (TQ) w[c] *= sv[gi][r] * inv;
                        }
                        const uint32_t hi = pack2_rz(w[0], w[1]);
                        const float2 h = unpack2(hi);
                        const uint32_t lo = weight_rest(hi, pack2(w[0] - h.x, w[1] - h.y));
                        bh[nt][r] = movmatrix(hi);
                        bl[nt][r] = movmatrix(lo);
                    }
                uint32_t xa[HD / 8], xc[HD / 8];
                attn_load_v<FMT, HD>(base + S::ROWS + gi * S::GROUP + v_at, g, xa, xc, lane4);
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
        /* the item (or the part) ends: join the warps; warp d finishes tiles d * MINE .. + MINE - 1 */
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
        const bool whole = SOLO || (began && item_done);
        const int slot = 2 * part + (began ? 1 : 0);               /* an item that began here is this CTA's last */
        if (!whole_items && A.by_item && whole && tid == 0) A.desc[at.b * items + at.h] = make_int2(-1, 0);
        if constexpr (SOLO) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const int h = 8 * nt + 2 * t + c;
                    if (h >= heads) continue;
                    const float f = vref * (1.0f / attn_alpha<FMT>());
#pragma unroll
                    for (int j = 0; j < TILES; j++)
                        attn_store<FMT>(A.out + (head0 + h) * HD, j, g, attn_out(o[nt][j][c] * f, o[nt][j][c + 2] * f, l[nt][c], odd));
                    if (A.lse != nullptr && g == 0) A.lse[head0 + h] = attn_lse(m[nt][c], l[nt][c]);
                }
        } else {
        /* each warp leaves its output in the stage that it has read last, which nothing is copied into before the
         * next step */
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            if (g == 0) {
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    m_s[warp][8 * nt + 2 * t + c] = m[nt][c];
                    l_s[warp][8 * nt + 2 * t + c] = l[nt][c];
                }
            }
#pragma unroll
            for (int j = 0; j < TILES; j++)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(base + 16 * lane + (nt * TILES + j) * 512),
                             "f"(o[nt][j][0]), "f"(o[nt][j][1]), "f"(o[nt][j][2]), "f"(o[nt][j][3]) : "memory");
        }
        if (lane == 0) f_s[warp] = vref;
        __syncthreads();
        if (warp * MINE < NT * TILES) {
            const int nt = warp * MINE / TILES;        /* a warp's tiles are of one column tile */
            float top[2], sum[2], f[W][2];
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const int h = 8 * nt + 2 * t + c;
                top[c] = m_s[0][h];
#pragma unroll
                for (int w = 1; w < W; w++) top[c] = fmaxf(top[c], m_s[w][h]);
                sum[c] = 0.0f;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    f[w][c] = ex2(m_s[w][h] - top[c]);
                    sum[c] += f[w][c] * l_s[w][h];
                    f[w][c] *= f_s[w] * (1.0f / attn_alpha<FMT>());
                }
                if (warp * MINE % TILES == 0 && g == 0) {
                    if (!whole) A.part_ml[(size_t)slot * (8 * NT) + h] = make_float2(top[c], sum[c]);
                    else if (A.lse != nullptr && h < heads) A.lse[head0 + h] = attn_lse(top[c], sum[c]);
                }
            }
            const uint32_t from = base - warp * S::RING + 16 * lane + warp * MINE * 512;
#pragma unroll
            for (int k = 0; k < MINE; k++) {
                const int x = warp * MINE + k, j = x % TILES;
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < W; w++) {          /* in warp order, whoever adds */
                    float v[4];
                    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(from + w * S::RING + k * 512));
#pragma unroll
                    for (int c = 0; c < 4; c++) acc[c] = fmaf(v[c], f[w][c & 1], acc[c]);
                }
                if (whole) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const int h = 8 * nt + 2 * t + c;
                        if (h < heads) attn_store<FMT>(A.out + (head0 + h) * HD, j, g, attn_out(acc[c], acc[c + 2], sum[c], odd));
                    }
                } else {
                    A.part_o[((size_t)slot * (NT * TILES) + x) * 32 + lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                }
            }
        }
        __syncthreads();                               /* all has been read */
        }
        if (!more) break;
        places -= kAttnItemCost;
        at = nx;
        began = true;
        begin_item();
    }
    cp_wait<0>();
    if constexpr (FMT != KV_E4M3) {                    /* (it has no infinities) */
        if (SOLO ? __any_sync(0xffffffffu, odd) : __syncthreads_or(odd)) {
            const int last = at.b * items + at.h - (SOLO || at.last() ? 0 : 1);
            if (SOLO) __syncwarp();                    /* (all outputs are written; a barrier does it for the CTA) */
            attn_look_up<FMT, HD>(A, first_s[SOLO ? warp : 0], last, 8 * NT, SOLO ? 0 : warp, SOLO ? 1 : W);
        }
    }
}

/* Joins the pieces of items that are cut: an item that ends in part `last` and began in part `first` has them in
 * slots 2 first + 1, 2 (first + 1), 2 (first + 2) .. 2 last. CTA (x, y) takes tile y of the output, of item x where
 * there are few items (desc[item] = last, first), else of the items that end in parts 4 x .. 4 x + 3 (desc[last] =
 * item, first). An item of up to four pieces is one warp's work, all its loads in flight at once; of a longer one
 * each warp takes every WARPS-th piece and their results meet in shared memory. The order of every sum follows from
 * the number of pieces alone. */
struct AttnState {                                     /* a lane's: maximum and sum of heads 2t, 2t + 1, four outputs */
    float m[2], l[2], o[4];
    __device__ __forceinline__ void add(const float4& ml, const float4& v) {
        const float m1[2] = {ml.x, ml.z}, l1[2] = {ml.y, ml.w}, v1[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const float top = fmaxf(m[c], m1[c]), a = ex2(m[c] - top), b = ex2(m1[c] - top);
            m[c] = top;
            l[c] = l[c] * a + l1[c] * b;
            o[c] = o[c] * a + v1[c] * b;
            o[c + 2] = o[c + 2] * a + v1[c + 2] * b;
        }
    }
};
template <int FMT, int HD, int NT, int WARPS>
/* (24 warps an SM: the look-up of infinities must not take registers from what hides the loads' latency) */
__global__ void __launch_bounds__(32 * WARPS, 24 / WARPS) attn_join_kernel(const __grid_constant__ AttnArgs A) {
    constexpr int TILES = HD / 16;
    __shared__ float4 ml_s[WARPS][32], o_s[WARPS][32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int x = blockIdx.y, nt = x / TILES, j = x % TILES;
    pdl_wait();
    const int per = A.by_item ? 1 : kAttnJoinParts, mine = blockIdx.x * per + lane;
    int2 d = make_int2(-1, 0);
    if (lane < per && (A.by_item || mine < A.parts)) d = A.desc[mine];
    /* (a scratch that another call has written to in between must not lead outside of it) */
    const int limit = A.by_item ? A.parts : A.n_seqs * A.n_kv * A.head_blocks;
    unsigned todo = __ballot_sync(0xffffffffu, (unsigned)d.x < (unsigned)limit && (unsigned)d.y <= (unsigned)(A.by_item ? d.x : mine));
    for (int n = 0; todo != 0; todo &= todo - 1) {
        const int i = __ffs(todo) - 1, which = blockIdx.x * per + i;
        const int dx = __shfl_sync(0xffffffffu, d.x, i), first = __shfl_sync(0xffffffffu, d.y, i);
        const int item = A.by_item ? which : dx, pieces = (A.by_item ? dx : which) - first + 1;
        const bool all = pieces > kAttnJoinChunk;
        if (!all && (n++ % WARPS) != warp) continue;
        AttnState s = {{kNoMax, kNoMax}, {0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        const int step = all ? WARPS : 1;
        for (int p0 = all ? warp : 0; p0 < pieces; p0 += kAttnJoinChunk * step) {
            float4 ml[kAttnJoinChunk], v[kAttnJoinChunk];
#pragma unroll
            for (int k = 0; k < kAttnJoinChunk; k++) {
                const int p = p0 + k * step;
                if (p < pieces) {
                    const size_t slot = p == 0 ? 2 * first + 1 : 2 * (first + p);
                    ml[k] = *reinterpret_cast<const float4*>(A.part_ml + slot * (8 * NT) + 8 * nt + 2 * t);
                    v[k] = A.part_o[(slot * (NT * TILES) + x) * 32 + lane];
                }
            }
#pragma unroll
            for (int k = 0; k < kAttnJoinChunk; k++)
                if (p0 + k * step < pieces) s.add(ml[k], v[k]);
        }
        if (all) {
            __syncthreads();                           /* the previous long item has been read */
            ml_s[warp][lane] = make_float4(s.m[0], s.l[0], s.m[1], s.l[1]);
            o_s[warp][lane] = make_float4(s.o[0], s.o[1], s.o[2], s.o[3]);
            __syncthreads();
            if (warp != 0) continue;
            for (int w = 1; w < WARPS; w++) s.add(ml_s[w][lane], o_s[w][lane]);
        }
        const int items = A.n_kv * A.head_blocks;
        const int b = item / items, it = item - b * items, hk = it / A.head_blocks, hb = it - hk * A.head_blocks;
        const int heads = A.group - hb * 8 * NT;
        const size_t head0 = (size_t)b * A.n_q + (size_t)hk * A.group + hb * 8 * NT;
        bool odd = false;
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int h = 8 * nt + 2 * t + c;
            if (h >= heads) continue;
            attn_store<FMT>(A.out + (head0 + h) * HD, j, g, attn_out(s.o[c], s.o[c + 2], s.l[c], odd));
            if (A.lse != nullptr && j == 0 && g == 0) A.lse[head0 + h] = attn_lse(s.m[c], s.l[c]);
        }
        if constexpr (FMT != KV_E4M3) {
            if (!__any_sync(0xffffffffu, odd)) continue;
            __syncwarp();                              /* the tile's outputs are all written by this warp */
            attn_infinite<FMT, HD>(A, b, hk, A.out + (head0 + 8 * nt) * HD, min(8, heads - 8 * nt),
                                   [j](int k) { return attn_v_dim<FMT>(2 * j + (k & 1), k >> 1); }, lane);
        }
    }
}

/* Column tiles of 8 query heads an item holds: two where the group has more than eight heads (one for 256-wide heads,
 * by registers, and for the 4-bit format, by shared memory), the rest in further items of the same cache head. */
static int attn_col_tiles(int group, int head_dim, int fmt) { return group > 8 && head_dim <= 128 && fmt != KV_TQ4 ? 2 : 1; }

/* Whether items stay whole, which saves the joining kernel: 2, each a warp's; 1, each a CTA's; 0, they are cut. By
 * the blocks that a table has room for, since the lengths are known on the device alone: wide tables are cut however
 * short their sequences are. A warp each pays where there are items for the `warps` of the launch, for longer ones
 * the more there are; a CTA each where that takes less than the second kernel's 3 us more, or where there are items
 * enough to even out. A block of a rotated format takes longer. The limits are by the mean time over sequences as long as
 * the table has room for, by the logarithm from one position to that, and both for every table down to a third (a
 * server's table has room to grow). Measured, us, cut / CTA / warp, every sequence as long as the table and that mean;
 * 28 heads over 4 of 128, 1776 warps; at the last size that stays whole and the next:
 *   items  blocks  FP16                                     blocks  4 bits
 *   4      8       7.5 / 8.2            7.4 / 6.5           4       12.4 / 13.7          12.4 / 11.5
 *   4      10      7.6 / 9.5            7.5 / 7.3           5       12.6 / 15.8          12.4 / 12.5
 *   64     10      10.4 / 9.9           9.1 / 7.6           5       16.1 / 15.9          14.3 / 12.7
 *   64     12      10.6 / 11.2          9.2 / 8.0           6       18.6 / 18.1          14.6 / 13.6
 *   128    14      17.7 / 17.1          11.0 / 9.4          7       26.3 / 20.8          16.8 / 15.8
 *   128    16      19.5 / 19.2          11.6 / 10.6         8       28.4 / 22.9          17.5 / 16.7
 *   384    16      40.7 / 34.1          19.1 / 15.5         8       66.5 / 65.7          35.0 / 36.1
 *   384    18      44.4 / 37.3          19.8 / 16.3         10      76.7 / 78.8          37.9 / 40.2
 *   640    2       15.5 / 11.8 / 11.0   12.5 / 10.2 / 8.8   2       42.7 / 40.9 / 40.8   31.7 / 29.8 / 27.3
 *   640    3       20.5 / 18.0 / 18.2   13.6 / 11.2 / 10.5  3       55.1 / 52.7 / 57.8   34.8 / 32.9 / 33.9
 *   1200   3       30.5 / 26.2 / 25.2   18.8 / 16.4 / 14.0  3       89.0 / 89.6 / 73.6   56.3 / 54.5 / 43.0
 *   1200   4       36.1 / 31.1 / 30.9   22.7 / 19.8 / 18.6  4       105 / 107 / 95.2     65.2 / 64.4 / 61.0
 *   1776   5       52.8 / 50.6 / 49.1   30.4 / 27.9 / 25.1  4       143 / 141 / 98.9     87.6 / 85.4 / 67.5
 *   1776   6       61.2 / 58.8 / 57.0   32.2 / 29.8 / 27.4
 * One limit serves all of FP16 and FP8, one all of the rotated formats: FP8 and the narrow codes are cut better at
 * the CTA's limits (4 x 8 E4M3 7.9 / 10.0, the mean 7.7 / 7.7; 4 x 4 2 bits 11.4 / 13.6 and 11.4 / 11.1), FP16 would
 * stay whole a little longer. 3, 2 and 1.5 bits take a warp each from more items on (2 bits, 640 x 2: 28.4 / 25.5 /
 * 29.4). Over 1667 points (1 .. 24 blocks, 4 .. 4000 items, ten forms, 16 heads to a cache head and heads of 64 and
 * 256 among them) the way taken has a mean 1.007 times the best one's. */
static int attn_whole(long long items, long long blocks, long long warps, int fmt) {
    const bool tq = kv_is_tq(fmt), narrow = tq && fmt != KV_TQ4;
    int solo = items >= 3 * warps ? (tq ? 5 : 8) : items >= warps ? 5 : 2 * items >= warps ? 3 : 3 * items >= warps ? 2 : 0;
    if (narrow && 3 * items < 2 * warps) solo = 0;
    if (blocks <= solo) return 2;
    const int most = items < 48 ? 8 : items < 96 ? 10 : items < 192 ? 14 : 16;
    return blocks <= (tq ? most / 2 : most) ? 1 : 0;
}

struct AttnScratch { size_t ml, o, bytes; };
static AttnScratch attn_scratch(int group, int head_dim) {
    const size_t heads = group > 8 && head_dim <= 128 ? 16 : 8;          /* of an item, whatever the format */
    AttnScratch s;
    s.ml = kAttnParts * sizeof(int2);                                   /* 16-byte multiples */
    s.o = s.ml + 2 * kAttnParts * heads * sizeof(float2);
    s.bytes = s.o + 2 * kAttnParts * heads * head_dim * sizeof(float);
    return s;
}

template <int FMT, int HD, int NT>
static cudaError_t launch_attn(AttnArgs A, long long capacity, cudaStream_t s) {
    constexpr int SMEM = AttnShape<FMT, HD, NT>::SMEM, parts = AttnShape<FMT, HD, NT>::CTAS * kAttnSms;
    static_assert(parts <= kAttnParts, "the scratch holds kAttnParts parts");
    A.parts = parts;
    const long long items = (long long)A.n_seqs * A.n_kv * A.head_blocks;
    A.whole_items = attn_whole(items, (capacity + AttnFmt<FMT, HD>::BLOCK - 1) / AttnFmt<FMT, HD>::BLOCK, parts * AttnFmt<FMT, HD>::W, FMT);
    A.one_each = A.whole_items == 1 && items <= parts;
    const int ctas = A.one_each ? (int)items : parts;
    const bool solo = A.whole_items == 2;
    cudaError_t e = cudaFuncSetAttribute(solo ? (const void*)attn_decode_kernel<FMT, HD, NT, true> : (const void*)attn_decode_kernel<FMT, HD, NT, false>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return e;
    /* Even parts want evenly filled SMs. A CTA that is placed while the kernel before still holds some of them
     * starts where there is room, and its part ends late (64 x 4096: 107 us instead of 86, behind a kernel of 888
     * small CTAs), so this is an ordinary launch unless there are few items: then the launch itself is what counts. */
    const dim3 block(32 * AttnFmt<FMT, HD>::W);
    if (solo) {
        e = launch_pdl(attn_decode_kernel<FMT, HD, NT, true>, dim3(ctas), block, (size_t)SMEM, s, A);
    } else if (A.by_item || A.whole_items) {
        e = launch_pdl(attn_decode_kernel<FMT, HD, NT, false>, dim3(ctas), block, (size_t)SMEM, s, A);
    } else {
        attn_decode_kernel<FMT, HD, NT, false><<<dim3(ctas), block, (size_t)SMEM, s>>>(A);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) return e;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    if (A.whole_items) return e;
    constexpr int TILES = NT * (HD / 16);
    if (A.by_item) e = launch_pdl(attn_join_kernel<FMT, HD, NT, 8>, dim3(A.n_seqs * A.n_kv * A.head_blocks, TILES), dim3(256), 0, s, A);
    else e = launch_pdl(attn_join_kernel<FMT, HD, NT, 4>, dim3((parts + kAttnJoinParts - 1) / kAttnJoinParts, TILES), dim3(128), 0, s, A);
    if (e == cudaSuccess) g_launches.fetch_add(1, std::memory_order_relaxed);
    return e;
}
template <int FMT>
static cudaError_t launch_attn(const AttnArgs& A, int head_dim, int nt, long long capacity, cudaStream_t s) {
    if constexpr (!kv_is_tq(FMT)) {
        if (head_dim == 64) return nt == 2 ? launch_attn<FMT, 64, 2>(A, capacity, s) : launch_attn<FMT, 64, 1>(A, capacity, s);
        if (head_dim == 256) return launch_attn<FMT, 256, 1>(A, capacity, s);
    }
    if (head_dim == 128) {
        if constexpr (FMT != KV_TQ4) {
            if (nt == 2) return launch_attn<FMT, 128, 2>(A, capacity, s);
        }
        return launch_attn<FMT, 128, 1>(A, capacity, s);
    }
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
    const int group = n_q_heads / n_kv_heads, nt = attn_col_tiles(group, head_dim, kv_format);
    const AttnScratch sc = attn_scratch(group, head_dim);
    uint8_t* const base = (uint8_t*)scratch;
    const int head_blocks = (group + 8 * nt - 1) / (8 * nt);
    const long long items = (long long)n_seqs * n_kv_heads * head_blocks;
    const long long capacity = block_table != nullptr ? (long long)table_stride << kAttnPageShift : (long long)table_stride;
    const AttnArgs A = {(const __half*)q, (__half*)out, lse, (const uint8_t*)k_store, (const uint8_t*)v_store,
                        (const __half*)k_meta, (const __half*)v_meta, block_table, lens,
                        (int2*)base, (float2*)(base + sc.ml), (float4*)(base + sc.o),
                        n_seqs, n_q_heads, n_kv_heads, n_slots, table_stride, len_add,
                        group, head_blocks, 0, items <= kAttnFewItems, 0, 0, items * (capacity / 16 + 2) < kAttnNarrow / 2, scale * kLog2e};
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
    switch (kv_format) {
        case KV_RAW: e = launch_attn<KV_RAW>(A, head_dim, nt, capacity, s); break;
        case KV_E4M3: e = launch_attn<KV_E4M3>(A, head_dim, nt, capacity, s); break;
        case KV_E5M2: e = launch_attn<KV_E5M2>(A, head_dim, nt, capacity, s); break;
        case KV_TQ4: e = launch_attn<KV_TQ4>(A, head_dim, nt, capacity, s); break;
        case KV_TQ3: e = launch_attn<KV_TQ3>(A, head_dim, nt, capacity, s); break;
        case KV_TQ2: e = launch_attn<KV_TQ2>(A, head_dim, nt, capacity, s); break;
        case KV_TQ1_5: e = launch_attn<KV_TQ1_5>(A, head_dim, nt, capacity, s); break;
        default: return (int)cudaErrorNotSupported;
    }
    return (int)(e != cudaSuccess ? e : cudaGetLastError());
}
