/*
 * kv_plan.cu -- one serving step's bookkeeping over the paged KV cache, on the
 * device: block tables, slot map and positions from request lengths. sm_100a,
 * latency-bound.
 *
 * For sequence b with L = lens[b] cached positions and n = new_tokens[b]:
 *   have   = ceil(L / 64) pages, need = ceil((L + n) / 64) - have more,
 *   rows   = [row_start[b], row_start[b + 1]), row_start the exclusive sum of max(n, 0).
 * n < 0 gives the sequence's pages back. Pages come from a stack of free page
 * numbers: released pages are pushed in sequence order, then page number j of
 * the call (j from the exclusive sum of `need`) is the j-th from the top. So the
 * three sums are all that couples the sequences; a sequence whose inclusive sum
 * passes the stack's height is refused, which leaves the sums of those before
 * it as they are: no second pass and no order that depends on timing.
 *
 * Shape: one CTA, or one cluster of 8 or 16 for long row lists. Every CTA works
 * out the sums by itself (8 bytes a sequence, from L2) and keeps them in shared
 * memory, 20 bytes a sequence; from there everything is flat: released pages,
 * new pages and rows are each split over all threads, which find their sequence
 * by a binary search in the sums (a loop over its pages by the thread that owns
 * a sequence took 31 us where this takes 11, at 2000 sequences of up to 256
 * pages and 131072 rows). One cluster barrier: the released pages are on the
 * stack, and lens and the stack's height are read, before pages are taken from
 * it and those are overwritten. Rows do not wait for the tables: a row's page is
 * either in the table from before or at a known place of the stack.
 */
#include "vvb_device.cuh"
#include "vvb_launch.h"

#include <atomic>

namespace vvb {

extern std::atomic<uint64_t> g_launches;

constexpr int kPlanPageShift = 6;
constexpr int kPlanMaxSeqs = 8192;
constexpr size_t plan_smem_bytes(int n_seqs) { return (5 * (size_t)n_seqs + 3) * sizeof(int); }      /* 160 KB at most */

struct PlanArgs {
    const int* new_tokens;
    const int* lens;
    int* lens_out;
    int* block_table;
    int* free_pages;
    const int* free_count;
    int* free_count_out;
    int* row_start;
    int* slot_map;
    int* positions;
    int* status;               /* may be null */
    int n_seqs, table_stride, n_pages, max_rows;
};

/* Sums stop at INT_MAX instead of wrapping (min(a + b, INT_MAX) is associative for a, b >= 0). */
__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) { return min(a + b, 0x7fffffffu); }

/* Exclusive sums over the CTA of two values a thread; every thread also gets the totals. */
__device__ __forceinline__ void block_scan2(unsigned a, unsigned b, unsigned* ws, unsigned& ea, unsigned& eb, unsigned& ta,
                                            unsigned& tb) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarps = blockDim.x >> 5;
    unsigned sa = a, sb = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned xa = __shfl_up_sync(0xffffffffu, sa, o), xb = __shfl_up_sync(0xffffffffu, sb, o);
        if (lane >= o) { sa = sat_add(sa, xa); sb = sat_add(sb, xb); }
    }
    if (lane == 31) { ws[warp] = sa; ws[32 + warp] = sb; }
    __syncthreads();
    unsigned wa = lane < nwarps ? ws[lane] : 0u, wb = lane < nwarps ? ws[32 + lane] : 0u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned xa = __shfl_up_sync(0xffffffffu, wa, o), xb = __shfl_up_sync(0xffffffffu, wb, o);
        if (lane >= o) { wa = sat_add(wa, xa); wb = sat_add(wb, xb); }
    }
    ta = __shfl_sync(0xffffffffu, wa, 31);
    tb = __shfl_sync(0xffffffffu, wb, 31);
    const unsigned ba = warp ? __shfl_sync(0xffffffffu, wa, warp - 1) : 0u;
    const unsigned bb = warp ? __shfl_sync(0xffffffffu, wb, warp - 1) : 0u;
    const unsigned la = __shfl_up_sync(0xffffffffu, sa, 1), lb = __shfl_up_sync(0xffffffffu, sb, 1);
    ea = sat_add(ba, lane ? la : 0u);
    eb = sat_add(bb, lane ? lb : 0u);
    __syncthreads();                                   /* ws is used again */
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

/* Largest i in [0, n) with a[i] <= x, for ascending a and a[0] <= x < a[n]: among equal entries the last, so that
 * entry's part is not empty. */
__device__ __forceinline__ int plan_find(const unsigned* a, int n, unsigned x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

template <bool CLUSTER>
__global__ void __launch_bounds__(1024, 1) kv_plan_kernel(const __grid_constant__ PlanArgs A) {
    extern __shared__ unsigned plan_smem[];
    const int n = A.n_seqs;
    unsigned* const start_s = plan_smem;                       /* [n + 1] first row of each sequence */
    unsigned* const push_s = plan_smem + n + 1;                /* [n + 1] its first released page */
    unsigned* const take_s = plan_smem + 2 * (n + 1);          /* [n + 1] its first new page */
    int* const new_s = reinterpret_cast<int*>(plan_smem + 3 * (n + 1));      /* [n] new tokens */
    int* const base_s = new_s + n;                             /* [n] cached positions; then -1 when refused or released */
    __shared__ unsigned ws[64];
    __shared__ unsigned taken_s;
    const int t = threadIdx.x, nt = blockDim.x;
    const int rank = CLUSTER ? (int)blockIdx.x : 0, ranks = CLUSTER ? (int)gridDim.x : 1;   /* the grid is one cluster */
    if (t == 0) taken_s = 0;
    pdl_wait();
    pdl_trigger();

    const unsigned cap = (unsigned)A.table_stride << kPlanPageShift;         /* < 2^31 */
    auto pages_of = [&](int len) { return min(((unsigned)len + 63u) >> kPlanPageShift, (unsigned)A.table_stride); };
    auto full = [&](int add, int len) { return add >= 0 && ((unsigned)len > cap || (unsigned)add > cap - (unsigned)len); };
    /* lens and the height may be overwritten below (lens_out, free_count_out), so they are not read-only data */
    const unsigned held = (unsigned)min(max(__ldcg(A.free_count), 0), A.n_pages);
    const int per = (n + nt - 1) / nt;
    const int b0 = min(t * per, n), b1 = min(b0 + per, n);
    /* rows and released pages */
    unsigned rows = 0, rel = 0;
    for (int b = b0; b < b1; b++) {
        const int add = __ldg(A.new_tokens + b), len = max(__ldcg(A.lens + b), 0);
        new_s[b] = add;
        base_s[b] = len;
        rows = sat_add(rows, (unsigned)max(add, 0));
        rel = sat_add(rel, add < 0 ? pages_of(len) : 0u);
    }
    unsigned row, push, rows_total, rel_total;
    block_scan2(rows, rel, ws, row, push, rows_total, rel_total);
    /* pages asked for, by the sequences that have a table and rows for them */
    unsigned want = 0;
    for (int b = b0; b < b1; b++) {
        const int add = new_s[b], len = base_s[b];
        start_s[b] = row;
        push_s[b] = push;
        row = sat_add(row, (unsigned)max(add, 0));
        push = sat_add(push, add < 0 ? pages_of(len) : 0u);
        if (add > 0 && row <= (unsigned)A.max_rows && !full(add, len))
            want = sat_add(want, (((unsigned)len + (unsigned)add + 63u) >> kPlanPageShift) - pages_of(len));
    }
    unsigned upto, unused0, want_total, unused1;
    block_scan2(want, 0u, ws, upto, unused0, want_total, unused1);
    const unsigned avail = min(sat_add(held, rel_total), (unsigned)A.n_pages);
    row = b0 < b1 ? start_s[b0] : 0u;
    for (int b = b0; b < b1; b++) {
        const int add = new_s[b], len = base_s[b];
        row = sat_add(row, (unsigned)max(add, 0));
        const bool no_table = full(add, len), no_rows = add > 0 && !no_table && row > (unsigned)A.max_rows;
        const unsigned ask = add > 0 && !no_table && !no_rows ? (((unsigned)len + (unsigned)add + 63u) >> kPlanPageShift) - pages_of(len) : 0u;
        take_s[b] = upto;
        upto = sat_add(upto, ask);
        const bool no_pages = ask > 0 && upto > avail;
        const bool ok = !(no_table || no_rows || no_pages || add < 0);
        if (ok && ask > 0) atomicMax(&taken_s, upto);
        base_s[b] = ok ? len : -1;
        if (rank == 0) {
            A.row_start[b] = (int)start_s[b];
            if (A.status != nullptr) A.status[b] = no_table ? 2 : no_rows ? 3 : no_pages ? 1 : 0;
        }
    }
    if (t == 0) {
        start_s[n] = rows_total;
        push_s[n] = rel_total;
        take_s[n] = want_total;
        if (rank == 0) A.row_start[n] = (int)rows_total;
    }
    __syncthreads();
    const unsigned taken = taken_s;                            /* pages 0 .. taken - 1 of the call are given out */
    const int first = rank * nt + t, step = ranks * nt;

    /* released pages onto the stack */
    for (unsigned i = first; i < rel_total && held + i < (unsigned)A.n_pages; i += step) {
        const int b = plan_find(push_s, n, i);
        A.free_pages[held + i] = A.block_table[(size_t)b * A.table_stride + (i - push_s[b])];
    }
    __syncthreads();
    if (CLUSTER) cluster_barrier();      /* all CTAs have read lens and the height; the released pages are on the stack */

    if (rank == 0) {
        for (int b = t; b < n; b += nt) {
            const int add = new_s[b];
            if (add < 0) A.lens_out[b] = 0;
            else if (base_s[b] >= 0) A.lens_out[b] = base_s[b] + add;
            else if (A.lens_out != A.lens) A.lens_out[b] = A.lens[b];
        }
        if (t == 0) *A.free_count_out = (int)(avail - taken);
    }
    /* new pages into the tables, page j from the j-th place below the stack's top */
    for (unsigned j = first; j < taken; j += step) {
        const int b = plan_find(take_s, n, j);
        if (base_s[b] >= 0) A.block_table[(size_t)b * A.table_stride + pages_of(base_s[b]) + (j - take_s[b])] = __ldcg(A.free_pages + (avail - 1u - j));
    }
    /* rows: four consecutive ones a thread, each with a page look-up of its own, all in flight at once: a look-up
     * only where a page or a sequence begins costs its latency once a row, since some lane of a warp is always there */
    constexpr int kRun = 4;
    const bool vec = ((reinterpret_cast<uintptr_t>(A.slot_map) | reinterpret_cast<uintptr_t>(A.positions)) & 15u) == 0;
    const unsigned max_rows = (unsigned)A.max_rows;
    for (unsigned long long run0 = (unsigned long long)kRun * first; run0 < max_rows; run0 += (unsigned long long)kRun * step) {
        const unsigned r0 = (unsigned)run0;
        int b = r0 < rows_total ? plan_find(start_s, n, r0) : 0;
        int slot[kRun], pos[kRun];
#pragma unroll
        for (int j = 0; j < kRun; j++) {
            const unsigned r = r0 + j;
            slot[j] = pos[j] = -1;
            if (r >= rows_total || r >= max_rows) continue;
            while (start_s[b + 1] <= r) b++;
            const int from = base_s[b];
            if (from < 0) continue;
            const unsigned p = (unsigned)from + (r - start_s[b]), blk = p >> kPlanPageShift, had = pages_of(from);
            pos[j] = (int)p;
            slot[j] = __ldcg(blk < had ? A.block_table + (size_t)b * A.table_stride + blk : A.free_pages + (avail - 1u - take_s[b] - (blk - had)));
        }
#pragma unroll
        for (int j = 0; j < kRun; j++)
            if (pos[j] >= 0)               /* (what is no page of the pool would wrap to one from 2^26 on) */
                slot[j] = (unsigned)slot[j] < (unsigned)A.n_pages ? (int)(((unsigned)slot[j] << kPlanPageShift) + ((unsigned)pos[j] & 63u)) : -1;
#pragma unroll
        for (int j = 0; j < kRun; j += 4) {
            if (vec && r0 + j + 4 <= max_rows) {
                *reinterpret_cast<int4*>(A.slot_map + r0 + j) = make_int4(slot[j], slot[j + 1], slot[j + 2], slot[j + 3]);
                *reinterpret_cast<int4*>(A.positions + r0 + j) = make_int4(pos[j], pos[j + 1], pos[j + 2], pos[j + 3]);
            } else {
                for (int k = j; k < j + 4; k++)
                    if (r0 + k < max_rows) {
                        A.slot_map[r0 + k] = slot[k];
                        A.positions[r0 + k] = pos[k];
                    }
            }
        }
    }
}

/* Whether the current device has room for a cluster of 16 such CTAs, which a part of a GPU need not have; asked once a
 * device. The attributes are the same in every call, so threads may come at the same time. */
static bool plan_wide_clusters() {
    static std::atomic<signed char> known[64];             /* 0: not asked; 1: no; 2: yes */
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
    const signed char k = known[dev].load(std::memory_order_relaxed);
    if (k != 0) return k == 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = plan_smem_bytes(kPlanMaxSeqs);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = 16;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    int fit = 0;
    const void* f = (const void*)kv_plan_kernel<true>;
    bool ok = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plan_smem_bytes(kPlanMaxSeqs)) == cudaSuccess &&
              cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
              cudaOccupancyMaxActiveClusters(&fit, kv_plan_kernel<true>, &cfg) == cudaSuccess && fit > 0;
    if (!ok) cudaGetLastError();                           /* eight will do */
    known[dev].store(ok ? 2 : 1, std::memory_order_relaxed);
    return ok;
}

}  // namespace vvb

using namespace vvb;

extern "C" int vvbk_kv_plan(const int* new_tokens, const int* lens, int* lens_out, int* block_table, int* free_pages,
                            const int* free_count, int* free_count_out, int* row_start, int* slot_map, int* positions,
                            int* status, int n_seqs, int table_stride, int n_pages, int max_rows, void* stream) {
    const PlanArgs A = {new_tokens, lens, lens_out, block_table, free_pages, free_count, free_count_out, row_start,
                        slot_map, positions, status, n_seqs, table_stride, n_pages, max_rows};
    /* Rows are what takes time beyond the first few thousand, 1024 threads a CTA; 16 CTAs (the most a cluster can have,
     * by opt-in) from where that shows and the GPU has room: 131072 rows of 2000 sequences 14.6 us with 8, 11.1 with 16. */
    const int ctas = max_rows <= 4096 ? 1 : max_rows > 32768 && plan_wide_clusters() ? 16 : 8;
    const bool cluster = ctas > 1;
    const size_t smem = plan_smem_bytes(n_seqs);
    void (*kernel)(const PlanArgs) = cluster ? kv_plan_kernel<true> : kv_plan_kernel<false>;
    if (smem > 48 * 1024) {
        /* the most that any call asks for: the attribute is the function's, and another thread may be about to launch */
        const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plan_smem_bytes(kPlanMaxSeqs));
        if (e != cudaSuccess) return (int)e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    /* few rows of few sequences: fewer threads, whose barriers are quicker */
    const int threads = max_rows / 4 > n_seqs ? max_rows / 4 : n_seqs;
    cfg.blockDim = dim3(cluster || threads > 512 ? 1024u : threads > 128 ? 512u : 128u);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = ctas;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, A);
    if (e != cudaSuccess) return (int)e;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return (int)cudaGetLastError();
}
