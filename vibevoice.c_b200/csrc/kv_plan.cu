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
 * Shape: one CTA, or one cluster of eight for long row lists. Every CTA works
 * out the sums by itself (8 bytes a sequence, from L2) and keeps each
 * sequence's first row and first position in shared memory; CTA 0 writes what
 * is per sequence; the rows are split over the CTAs, each thread four
 * consecutive rows (16-byte stores) after one binary search. Two cluster
 * barriers order the releases before the pages taken, and the tables before the
 * rows that look pages up in them.
 */
#include "vvb_device.cuh"
#include "vvb_launch.h"

#include <atomic>

namespace vvb {

extern std::atomic<uint64_t> g_launches;

constexpr int kPlanPageShift = 6;
constexpr int kPlanCluster = 8;

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

struct PlanSeq {
    unsigned add, have, released, want;     /* rows, pages held, pages given back, pages asked for */
    bool full;
    __device__ __forceinline__ PlanSeq(const PlanArgs& A, int b) {
        const int n = A.new_tokens[b];
        const unsigned len = (unsigned)max(A.lens[b], 0);
        add = (unsigned)max(n, 0);
        const unsigned cap = (unsigned)A.table_stride << kPlanPageShift;         /* < 2^31 */
        have = min((len + 63u) >> kPlanPageShift, (unsigned)A.table_stride);
        released = n < 0 ? have : 0u;
        full = n >= 0 && (len > cap || add > cap - len);
        want = (n < 0 || full) ? 0u : ((len + add + 63u) >> kPlanPageShift) - have;
    }
};

template <bool CLUSTER>
__global__ void __launch_bounds__(1024, 1) kv_plan_kernel(const __grid_constant__ PlanArgs A) {
    extern __shared__ int plan_smem[];
    int* const start_s = plan_smem;                     /* [n_seqs + 1] first row of each sequence */
    int* const base_s = plan_smem + A.n_seqs + 1;       /* [n_seqs] its first new position, -1 when refused or released */
    __shared__ unsigned ws[64];
    __shared__ unsigned taken_s;
    const int t = threadIdx.x, nt = blockDim.x;
    const int rank = CLUSTER ? (int)blockIdx.x : 0, ranks = CLUSTER ? (int)gridDim.x : 1;   /* the grid is one cluster */
    if (t == 0) taken_s = 0;
    pdl_wait();
    pdl_trigger();

    const int per = (A.n_seqs + nt - 1) / nt;
    const int b0 = min(t * per, A.n_seqs), b1 = min(b0 + per, A.n_seqs);
    /* rows and released pages */
    unsigned rows = 0, rel = 0;
    for (int b = b0; b < b1; b++) {
        const PlanSeq s(A, b);
        rows = sat_add(rows, s.add);
        rel = sat_add(rel, s.released);
    }
    unsigned row0, rel0, rows_total, rel_total;
    block_scan2(rows, rel, ws, row0, rel0, rows_total, rel_total);
    /* pages asked for, by the sequences whose rows fit */
    unsigned want = 0, row = row0;
    for (int b = b0; b < b1; b++) {
        const PlanSeq s(A, b);
        row = sat_add(row, s.add);
        if (row <= (unsigned)A.max_rows) want = sat_add(want, s.want);   /* (no rows: nothing wanted either) */
    }
    unsigned want0, unused0, want_total, unused1;
    block_scan2(want, 0u, ws, want0, unused0, want_total, unused1);

    const unsigned held = (unsigned)min(max(*A.free_count, 0), A.n_pages);
    const unsigned avail = min(sat_add(held, rel_total), (unsigned)A.n_pages);
    /* what is per sequence: kept in shared memory by every CTA, written by the first */
    unsigned push = rel0, upto = want0;
    row = row0;
    for (int b = b0; b < b1; b++) {
        const PlanSeq s(A, b);
        const unsigned end = sat_add(row, s.add);
        const bool no_rows = s.add > 0 && !s.full && end > (unsigned)A.max_rows;
        const unsigned ask = no_rows ? 0u : s.want;
        const unsigned total = sat_add(upto, ask);
        const bool no_pages = ask > 0 && total > avail;
        const bool ends = A.new_tokens[b] < 0;
        const bool ok = !(s.full || no_rows || no_pages || ends);
        const int len = max(A.lens[b], 0);
        start_s[b] = (int)row;
        base_s[b] = ok ? len : -1;
        if (ok && ask > 0) atomicMax(&taken_s, total);
        if (rank == 0) {
            A.row_start[b] = (int)row;
            if (A.status != nullptr) A.status[b] = s.full ? 2 : no_rows ? 3 : no_pages ? 1 : 0;
            const int* mine = A.block_table + (size_t)b * A.table_stride;
            for (unsigned k = 0; k < s.released; k++) {
                const unsigned at = held + push + k;
                if (at < (unsigned)A.n_pages) A.free_pages[at] = mine[k];
            }
        }
        push = sat_add(push, s.released);
        upto = total;
        row = end;
    }
    if (t == 0) start_s[A.n_seqs] = (int)rows_total;
    if (rank == 0 && t == 0) A.row_start[A.n_seqs] = (int)rows_total;
    __syncthreads();
    if (CLUSTER) cluster_barrier();      /* all CTAs have read lens; the released pages are on the stack */

    if (rank == 0) {
        upto = want0;
        for (int b = b0; b < b1; b++) {
            const PlanSeq s(A, b);                       /* this thread has not yet overwritten these */
            const unsigned ask = (!s.full && sat_add((unsigned)start_s[b], s.add) > (unsigned)A.max_rows) ? 0u : s.want;
            if (base_s[b] >= 0) {
                int* mine = A.block_table + (size_t)b * A.table_stride + s.have;
                for (unsigned k = 0; k < ask; k++) mine[k] = __ldcg(A.free_pages + (avail - 1u - upto - k));
            }
            upto = sat_add(upto, ask);
            A.lens_out[b] = A.new_tokens[b] < 0 ? 0 : base_s[b] >= 0 ? base_s[b] + (int)s.add : A.lens[b];
        }
        if (t == 0) *A.free_count_out = (int)(avail - taken_s);
    }
    __syncthreads();
    if (CLUSTER) cluster_barrier();      /* the tables are written */

    /* rows: four consecutive ones a thread */
    const bool vec = ((reinterpret_cast<uintptr_t>(A.slot_map) | reinterpret_cast<uintptr_t>(A.positions)) & 15u) == 0;
    for (long long r0 = 4ll * (rank * nt + t); r0 < A.max_rows; r0 += 4ll * ranks * nt) {
        int slot[4], pos[4];
        int b = 0;
        if (r0 < (long long)rows_total) {               /* the last sequence that starts at or before r0 and is not empty there */
            int lo = 0, hi = A.n_seqs;                   /* start_s[lo] <= r0 < start_s[hi] */
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start_s[mid] <= (int)r0) lo = mid; else hi = mid;
            }
            b = lo;
        }
        int page_of = -1, page = 0, seen = -1;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const long long r = r0 + j;
            slot[j] = pos[j] = -1;
            if (r >= A.max_rows || r >= (long long)rows_total) continue;
            while (start_s[b + 1] <= (int)r) b++;
            const int first = base_s[b];
            if (first < 0) continue;
            const int p = first + (int)r - start_s[b];
            const int blk = p >> kPlanPageShift;
            if (blk != page_of || b != seen) {
                page = __ldcg(A.block_table + (size_t)b * A.table_stride + blk);
                page_of = blk;
                seen = b;
            }
            pos[j] = p;
            slot[j] = (page << kPlanPageShift) + (p & 63);
        }
        if (vec && r0 + 4 <= A.max_rows) {
            *reinterpret_cast<int4*>(A.slot_map + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4*>(A.positions + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
            for (int j = 0; j < 4 && r0 + j < A.max_rows; j++) {
                A.slot_map[r0 + j] = slot[j];
                A.positions[r0 + j] = pos[j];
            }
        }
    }
}

}  // namespace vvb

using namespace vvb;

extern "C" int vvbk_kv_plan(const int* new_tokens, const int* lens, int* lens_out, int* block_table, int* free_pages,
                            const int* free_count, int* free_count_out, int* row_start, int* slot_map, int* positions,
                            int* status, int n_seqs, int table_stride, int n_pages, int max_rows, void* stream) {
    const PlanArgs A = {new_tokens, lens, lens_out, block_table, free_pages, free_count, free_count_out, row_start,
                        slot_map, positions, status, n_seqs, table_stride, n_pages, max_rows};
    const bool cluster = max_rows > 4096;
    const size_t smem = (2 * (size_t)n_seqs + 1) * sizeof(int);       /* n_seqs <= 8192: 64 KB */
    void (*kernel)(const PlanArgs) = cluster ? kv_plan_kernel<true> : kv_plan_kernel<false>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster ? kPlanCluster : 1);
    cfg.blockDim = dim3(1024);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = kPlanCluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, A);
    if (e != cudaSuccess) return (int)e;
    g_launches.fetch_add(1, std::memory_order_relaxed);
    return (int)cudaGetLastError();
}
