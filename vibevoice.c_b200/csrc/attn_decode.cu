/*
 * attn_decode.cu -- attention of one new token per sequence over the KV cache.
 *
 * One CTA per (sequence, query head): its four warps take the keys in turn, each
 * lane holding head_dim / 32 consecutive values of q and of the running output.
 * One pass with the running maximum and sum of the softmax; the warps' states
 * are joined through shared memory.
 */
#include "fp8_kv.cuh"
#include "tq_kv.cuh"
#include "vvb_launch.h"

#include <atomic>

namespace vvb {

extern std::atomic<uint64_t> g_launches;

constexpr int kAttnPageShift = 6;

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
    int n_seqs, n_q, n_kv, n_slots, table_stride, len_add;
    float scale;
};

/* Number of keys of sequence b. */
__device__ __forceinline__ int attn_keys(const AttnArgs& A, int b) {
    const long long cap = A.block_table != nullptr ? (long long)A.table_stride << kAttnPageShift : (long long)A.table_stride;
    const long long n = (long long)A.lens[b] + A.len_add;
    return (int)min(max(n, 0ll), cap);
}

/* Cache row of key j of sequence b, -1 when it lies outside the cache. */
__device__ __forceinline__ int attn_row(const AttnArgs& A, int b, int j) {
    long long row;
    if (A.block_table != nullptr)
        row = ((long long)__ldg(A.block_table + (size_t)b * A.table_stride + (j >> kAttnPageShift)) << kAttnPageShift) + (j & 63);
    else
        row = (long long)b * A.table_stride + j;
    return row >= 0 && row < A.n_slots ? (int)row : -1;
}

template <int FMT, int HD> __host__ __device__ constexpr int attn_vec_bytes() {
    return kv_is_tq(FMT) ? tq_bytes_per_vec(FMT) : FMT == KV_RAW ? 2 * HD : HD;
}

/* Values d0 .. d0 + HD/32 - 1 of a stored vector, d0 = lane * HD/32. */
template <int FMT, int HD>
__device__ __forceinline__ void attn_load(const uint8_t* vec, float sigma, int lane, float (&x)[HD / 32]) {
    constexpr int N = HD / 32;
    if constexpr (FMT == KV_RAW) {
        const __half* p = reinterpret_cast<const __half*>(vec) + lane * N;
#pragma unroll
        for (int i = 0; i < N; i++) x[i] = __half2float(p[i]);
    } else if constexpr (FMT == KV_E4M3 || FMT == KV_E5M2) {
#pragma unroll
        for (int i = 0; i < N; i++)
            x[i] = __half2float(__half(__nv_cvt_fp8_to_halfraw(vec[lane * N + i], FMT == KV_E4M3 ? __NV_E4M3 : __NV_E5M2)));
    } else {
        constexpr int NB = TqBits<FMT>::N;
        const int bit = NB * lane;
        uint32_t w = vec[bit >> 3];
        if ((bit & 7) + NB > 8) w |= (uint32_t)vec[(bit >> 3) + 1] << 8;
        w = (w >> (bit & 7)) & ((1u << NB) - 1u);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float lev = 0.0f;
            if constexpr (FMT == KV_TQ1_5) {
                const uint32_t c = (w >> (3 * (i >> 1))) & 7u;
#pragma unroll
                for (int j = 0; j < 8; j++) lev = (c == (uint32_t)j) ? tq_vq15(2 * j + (i & 1)) : lev;
            } else {
                constexpr int W = NB / 4;
                const uint32_t c = (w >> (W * i)) & ((1u << W) - 1u);
#pragma unroll
                for (int j = 0; j < (1 << W); j++)
                    lev = (c == (uint32_t)j) ? (FMT == KV_TQ4 ? tq_lev4(j) : FMT == KV_TQ3 ? tq_lev3(j & 7) : tq_lev2(j & 3)) : lev;
            }
            x[i] = lev * sigma;
        }
    }
}

template <int FMT, int HD>
__global__ void __launch_bounds__(128) attn_decode_kernel(const __grid_constant__ AttnArgs A) {
    constexpr int N = HD / 32, BYTES = attn_vec_bytes<FMT, HD>();
    __shared__ float part[4][HD];
    __shared__ float mw[4];
    __shared__ double lw[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.y, h = blockIdx.x, hk = h / (A.n_q / A.n_kv);
    pdl_wait();
    pdl_trigger();
    const int n = attn_keys(A, b);
    const float scale2 = A.scale * 1.4426950408889634f;       /* scores in units of ln 2 */
    float q[N], o[N], m = -3e38f;
    double l = 0.0;             /* a long tail of tiny weights beside a large one */
    const size_t qoff = ((size_t)b * A.n_q + h) * HD + lane * N;
#pragma unroll
    for (int i = 0; i < N; i++) { q[i] = __half2float(A.q[qoff + i]); o[i] = 0.0f; }
    for (int j = warp; j < n; j += 4) {
        const int row = attn_row(A, b, j);
        if (row < 0) continue;
        const size_t vec = (size_t)row * A.n_kv + hk;
        float x[N], s = 0.0f;
        attn_load<FMT, HD>(A.k_store + vec * BYTES, kv_is_tq(FMT) ? __half2float(A.k_meta[vec]) : 1.0f, lane, x);
#pragma unroll
        for (int i = 0; i < N; i++) s = fmaf(q[i], x[i], s);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        s *= scale2;
        if (s > m) {
            const float a = exp2f(m - s);
            l *= a;
#pragma unroll
            for (int i = 0; i < N; i++) o[i] *= a;
            m = s;
        }
        const float p = exp2f(s - m);
        l += p;
        attn_load<FMT, HD>(A.v_store + vec * BYTES, kv_is_tq(FMT) ? __half2float(A.v_meta[vec]) : 1.0f, lane, x);
#pragma unroll
        for (int i = 0; i < N; i++) o[i] = fmaf(p, x[i], o[i]);
    }
#pragma unroll
    for (int i = 0; i < N; i++) part[warp][lane * N + i] = o[i];
    if (lane == 0) { mw[warp] = m; lw[warp] = l; }
    __syncthreads();
    const float top = fmaxf(fmaxf(mw[0], mw[1]), fmaxf(mw[2], mw[3]));
    double sum64 = 0.0;
    float f[4];
#pragma unroll
    for (int w = 0; w < 4; w++) { f[w] = exp2f(mw[w] - top); sum64 += lw[w] * f[w]; }
    const float sum = (float)sum64;
    /* no keys, or all of them outside the cache: zeros, -inf (m is then still the start value) */
    const bool none = top == -3e38f && sum == 0.0f;
    for (int d = threadIdx.x; d < HD; d += 128) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) v = fmaf(part[w][d], f[w], v);
        A.out[((size_t)b * A.n_q + h) * HD + d] = __float2half_rn(none ? 0.0f : v / sum);
    }
    if (A.lse != nullptr && threadIdx.x == 0)
        A.lse[(size_t)b * A.n_q + h] = none ? __int_as_float(0xff800000) : (top + log2f(sum)) * 0.6931471805599453f;
}

template <int FMT>
static cudaError_t launch_attn(const AttnArgs& A, int head_dim, cudaStream_t s) {
    const dim3 grid((unsigned)A.n_q, (unsigned)A.n_seqs), block(128);
    if constexpr (!kv_is_tq(FMT)) {
        if (head_dim == 64) return launch_pdl(attn_decode_kernel<FMT, 64>, grid, block, 0, s, A);
        if (head_dim == 256) return launch_pdl(attn_decode_kernel<FMT, 256>, grid, block, 0, s, A);
    }
    if (head_dim == 128) return launch_pdl(attn_decode_kernel<FMT, 128>, grid, block, 0, s, A);
    return cudaErrorNotSupported;
}

}  // namespace vvb

using namespace vvb;

extern "C" size_t vvbk_attn_decode_scratch(int n_seqs, int n_q_heads, int n_kv_heads, int head_dim) { return 16; }

extern "C" int vvbk_attn_decode(const void* q, void* out, float* lse, const void* k_store, const void* v_store,
                                const void* k_meta, const void* v_meta, const int* block_table, const int* lens,
                                void* scratch, int n_seqs, int n_q_heads, int n_kv_heads, int head_dim, int n_slots,
                                int table_stride, int len_add, int kv_format, float scale, void* stream) {
    const AttnArgs A = {(const __half*)q, (__half*)out, lse, (const uint8_t*)k_store, (const uint8_t*)v_store,
                        (const __half*)k_meta, (const __half*)v_meta, block_table, lens,
                        n_seqs, n_q_heads, n_kv_heads, n_slots, table_stride, len_add, scale};
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
    switch (kv_format) {
        case KV_RAW: e = launch_attn<KV_RAW>(A, head_dim, s); break;
        case KV_E4M3: e = launch_attn<KV_E4M3>(A, head_dim, s); break;
        case KV_E5M2: e = launch_attn<KV_E5M2>(A, head_dim, s); break;
        case KV_TQ4: e = launch_attn<KV_TQ4>(A, head_dim, s); break;
        case KV_TQ3: e = launch_attn<KV_TQ3>(A, head_dim, s); break;
        case KV_TQ2: e = launch_attn<KV_TQ2>(A, head_dim, s); break;
        case KV_TQ1_5: e = launch_attn<KV_TQ1_5>(A, head_dim, s); break;
        default: return (int)cudaErrorNotSupported;
    }
    if (e != cudaSuccess) return (int)e;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return (int)cudaGetLastError();
}
