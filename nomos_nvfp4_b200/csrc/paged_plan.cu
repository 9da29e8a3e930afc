// Block tables and slot maps of a serving step, from request lengths (sm_100a).  Integer work only:
//   end_b   = sum of max(n_new, 0) up to and including request b              (rows of the step)
//   need_b  = pages request b lacks for len_b + n_b keys, 0 where it cannot be served
//   upto_b  = sum of need up to and including b: granted while upto_b fits the free pages (finished requests' included)
// A few thousand requests are three prefix sums; what costs is the latency of one launch and the 12 bytes written per row.
// So every CTA works the sums out for itself in shared memory (no global scratch, no second launch) and the CTAs share the
// rows.  Where an output is an input's array (held_out = held, free_count_out = free_count: one step after another), the
// CTAs are one thread-block cluster that meets once between the last read of the inputs and the first write.
#include <cooperative_groups.h>

#include <algorithm>
#include <atomic>

#include "common.cuh"
#include "launch.h"

namespace nomos {

constexpr int PLAN_PAGE = 128;           // keys per page
constexpr int PLAN_THREADS = 1024;

struct PlanParams {
    const int *seq_lens, *n_new, *held;
    int *free_pages;
    const int *free_count;
    int *block_table, *held_out, *free_count_out, *granted, *row_start, *slot_map, *row_seq, *row_pos;
    int batch, max_pages, n_pages, max_rows;
    int vec;                             // the three row arrays start on 16-byte boundaries
    int in_place;                        // an output lies over an input: the grid is one cluster
};

struct Sums { long long rows, need, rel; };

__device__ __forceinline__ Sums warp_scan(Sums v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, v.rows, o), b = __shfl_up_sync(0xffffffffu, v.need, o), c = __shfl_up_sync(0xffffffffu, v.rel, o);
        if (lane >= o) { v.rows += a; v.need += b; v.rel += c; }
    }
    return v;
}

// Inclusive prefix sums over the block, of which the first `busy` warps have any; tot = the block's sums.  `scratch`: 32 entries.
__device__ __forceinline__ Sums block_scan(Sums v, Sums *scratch, Sums &tot, int busy) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nwarp = blockDim.x >> 5;
    if (warp < busy) v = warp_scan(v, lane);                          // (the others hold zeros)
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    if (warp == 0) {
        Sums w = lane < nwarp ? scratch[lane] : Sums{0, 0, 0};
        w = warp_scan(w, lane);
        __syncwarp();
        scratch[lane] = w;
    }
    __syncthreads();
    if (warp > 0) { v.rows += scratch[warp - 1].rows; v.need += scratch[warp - 1].need; v.rel += scratch[warp - 1].rel; }
    tot = scratch[31];
    return v;
}

// First index i with v[i] > x, v ascending, x < v[n - 1].
__device__ __forceinline__ int first_above(const int *v, int n, int x) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] > x) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

__global__ void __launch_bounds__(PLAN_THREADS) paged_plan_kernel(const __grid_constant__ PlanParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ int plan_sm[];
    const int B = p.batch;
    int *s_end = plan_sm;                // rows up to and including the request, at most max_rows
    int *s_len = s_end + B;              // keys cached so far
    int *s_held = s_len + B;             // pages held; -1 - pages: not served in this step
    int *s_upto = s_held + B;            // pages needed up to and including the request
    int *s_rel = s_upto + B;             // pages released up to and including the request
    __shared__ Sums scratch[32];
    __shared__ int s_taken;

    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (threadIdx.x == 0) s_taken = 0;
    const int F = max(0, min(p.free_count[0], p.n_pages));
    const int per = (B + blockDim.x - 1) / blockDim.x, b0 = threadIdx.x * per, b1 = min(B, b0 + per);
    const int busy = ((B + per - 1) / per + 31) / 32;

    // Rows, pages needed and pages released, in one scan.  Whether a request's rows end behind max_rows is not known yet: those
    // that do are a tail of the requests, so what they would need is in no other request's sum.
    Sums own{0, 0, 0};
    for (int b = b0; b < b1; ++b) {
        const int n = p.n_new[b], len = max(p.seq_lens[b], 0), held = max(0, min(p.held[b], p.max_pages));
        const long long keys = (long long)len + n;
        const bool fits = n > 0 && keys <= (long long)p.max_pages * PLAN_PAGE;
        const int need = fits ? max(0, (int)((keys + PLAN_PAGE - 1) / PLAN_PAGE) - held) : 0;
        s_end[b] = n;
        s_len[b] = len;
        s_held[b] = fits ? held : -1 - held;
        s_upto[b] = need;
        own.rows += max(n, 0);
        own.need += need;
        own.rel += n < 0 ? held : 0;
    }
    Sums tot;
    const Sums upto = block_scan(own, scratch, tot, busy);
    const int total_rows = (int)min(tot.rows, (long long)p.max_rows);
    const int R = (int)min(tot.rel, (long long)p.n_pages);
    const long long avail = (long long)F + R;
    // each request's own place in the sums (saturated: a sum beyond the pool is never granted)
    long long end = upto.rows - own.rows, need_upto = upto.need - own.need, rel = upto.rel - own.rel;
    int taken = 0;
    for (int b = b0; b < b1; ++b) {
        const int n = s_end[b], need = s_upto[b], h = s_held[b];
        end += max(n, 0);
        need_upto += need;
        if (n < 0) rel += -1 - h;
        if (h >= 0) {
            if (end > p.max_rows || (need > 0 && need_upto > avail)) s_held[b] = -1 - h;
            else if (need > 0) taken = (int)need_upto;                // it only grows: what is granted is a prefix
        }
        s_end[b] = (int)min(end, (long long)p.max_rows);
        s_upto[b] = (int)min(need_upto, 0x7fffffffll);
        s_rel[b] = (int)min(rel, 0x7fffffffll);
    }
    if (taken > 0) atomicMax(&s_taken, taken);
    // everything that may be overwritten in place has been read: the CTAs may write from here on
    if (p.in_place && gridDim.x > 1) cluster.sync();
    else __syncthreads();
    const int T = s_taken;

    // page at index i of the stack of free pages, the finished requests' pages on top of it
    auto released = [&](int e) {
        const int b = first_above(s_rel, B, e);
        const int before = b > 0 ? s_rel[b - 1] : 0;
        return p.block_table[(size_t)b * p.max_pages + (e - before)];
    };
    auto stack = [&](int i) { return i < F ? p.free_pages[i] : released(i - F); };
    auto need_before = [&](int b) { return b > 0 ? s_upto[b - 1] : 0; };
    const int top = (int)avail - 1;
    auto page_of = [&](int b, int j) {
        const int held = s_held[b];
        return j < held ? p.block_table[(size_t)b * p.max_pages + j] : stack(top - need_before(b) - (j - held));
    };
    const int tid = blockIdx.x * blockDim.x + threadIdx.x, nthreads = gridDim.x * blockDim.x;

    // rows: four consecutive ones per thread, one search for the four
    for (long long r0 = 4ll * tid; r0 < p.max_rows; r0 += 4ll * nthreads) {
        int slot[4] = {-1, -1, -1, -1}, seq[4] = {-1, -1, -1, -1}, pos[4] = {-1, -1, -1, -1};
        if (r0 < total_rows) {
            int b = first_above(s_end, B, (int)r0);
            const int first = b > 0 ? s_end[b - 1] : 0, at0 = s_len[b] + ((int)r0 - first);
            if (r0 + 4 <= s_end[b] && at0 % PLAN_PAGE + 4 <= PLAN_PAGE) {     // one request, one page
                if (s_held[b] >= 0) {
                    const int s0 = (int)((unsigned)page_of(b, at0 / PLAN_PAGE) * PLAN_PAGE + (unsigned)(at0 % PLAN_PAGE));
#pragma unroll
                    for (int k = 0; k < 4; ++k) { slot[k] = s0 + k; seq[k] = b; pos[k] = at0 + k; }
                }
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = (int)r0 + k;
                    if (r >= total_rows) break;
                    while (s_end[b] <= r) ++b;
                    if (s_held[b] < 0) continue;
                    const int at = s_len[b] + (r - (b > 0 ? s_end[b - 1] : 0));
                    slot[k] = (int)((unsigned)page_of(b, at / PLAN_PAGE) * PLAN_PAGE + (unsigned)(at % PLAN_PAGE));
                    seq[k] = b;
                    pos[k] = at;
                }
            }
        }
        if (p.vec && r0 + 4 <= p.max_rows) {
            *reinterpret_cast<int4 *>(p.slot_map + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
            *reinterpret_cast<int4 *>(p.row_seq + r0) = make_int4(seq[0], seq[1], seq[2], seq[3]);
            *reinterpret_cast<int4 *>(p.row_pos + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (r0 + k < p.max_rows) {
                    p.slot_map[r0 + k] = slot[k];
                    p.row_seq[r0 + k] = seq[k];
                    p.row_pos[r0 + k] = pos[k];
                }
        }
    }
    // the new pages' table entries, and the released pages back onto the stack.  (No CTA reads a table entry or a stack
    // entry that another one writes: new entries lie behind the held ones, pushes at or above F.)
    // (the first CTA has the requests' own numbers to write: these start at the last one and in the middle)
    for (int e = nthreads - 1 - tid; e < T; e += nthreads) {
        const int b = first_above(s_upto, B, e), i = e - need_before(b);
        p.block_table[(size_t)b * p.max_pages + s_held[b] + i] = stack(top - e);
    }
    for (int e = tid >= nthreads / 2 ? tid - nthreads / 2 : tid + (nthreads + 1) / 2; e < R; e += nthreads)
        if (F + e < p.n_pages) p.free_pages[F + e] = released(e);
    if (blockIdx.x == 0) {
        for (int b = threadIdx.x; b < B; b += blockDim.x) {
            const int h = s_held[b], n_b = s_end[b] - (b > 0 ? s_end[b - 1] : 0);
            const int need = s_upto[b] - need_before(b), rel_b = s_rel[b] - (b > 0 ? s_rel[b - 1] : 0);
            p.granted[b] = h >= 0 ? n_b : 0;
            p.held_out[b] = h >= 0 ? h + need : -1 - h - rel_b;     // a finished request releases what it held
            p.row_start[b + 1] = s_end[b];
        }
        if (threadIdx.x == 0) {
            p.row_start[0] = 0;
            p.free_count_out[0] = (int)min(avail - T, (long long)p.n_pages);
        }
    }
}

int launch_paged_plan(cudaStream_t st, const int *seq_lens, const int *n_new, const int *held, int *free_pages, const int *free_count,
                      int *block_table, int *held_out, int *free_count_out, int *granted, int *row_start, int *slot_map, int *row_seq,
                      int *row_pos, int batch, int max_pages, int n_pages, int max_rows) {
    PlanParams p{seq_lens, n_new, held, free_pages, free_count, block_table, held_out, free_count_out, granted, row_start, slot_map,
                 row_seq, row_pos, batch, max_pages, n_pages, max_rows, 0, 0};
    p.vec = ((reinterpret_cast<uintptr_t>(slot_map) | reinterpret_cast<uintptr_t>(row_seq) | reinterpret_cast<uintptr_t>(row_pos)) & 15) == 0;
    const size_t smem = (size_t)batch * 5 * sizeof(int);
    // (48 KB without the attribute, the kernel's own static arrays included)
    cudaError_t e = smem > 40 * 1024 ? cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PLAN_MAX_BATCH * 5 * (int)sizeof(int)) : cudaSuccess;
    if (e != cudaSuccess) { set_error("nomos_kv_paged_plan: shared memory: %s", cudaGetErrorString(e)); return NOMOS_ECUDA; }
    const auto over = [](const void *x, long nx, const void *y, long ny) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(x), b = reinterpret_cast<uintptr_t>(y);
        return a < b + 4 * (uintptr_t)ny && b < a + 4 * (uintptr_t)nx;
    };
    const struct { const void *x; long n; } ins[4] = {{seq_lens, batch}, {n_new, batch}, {held, batch}, {free_count, 1}},
                                            outs[7] = {{held_out, batch}, {free_count_out, 1}, {granted, batch}, {row_start, batch + 1l},
                                                       {slot_map, max_rows}, {row_seq, max_rows}, {row_pos, max_rows}};
    for (const auto &o : outs)
        for (const auto &in : ins) p.in_place |= over(o.x, o.n, in.x, in.n) ? 1 : 0;
    // One CTA while its threads cover the rows in one round.  Else CTAs of half the threads, enough to cover them in one round,
    // at most one per SM; in place a cluster of sixteen, of eight where the driver does not allow that.  261120 rows of 1024
    // requests: 7.4 us with 128 CTAs of 512 threads (8.9 with 64 of 1024, 9.1 with 148 of 256), 21.3 in a cluster of sixteen.
    int ctas = max_rows <= 4 * PLAN_THREADS ? 1 : p.in_place ? 16 : std::min(148, (max_rows + 2 * PLAN_THREADS - 1) / (2 * PLAN_THREADS));
    static std::atomic<uint64_t> large_clusters{0};                   // devices on which the attribute is set
    if (p.in_place && ctas == 16 && !(large_clusters.load(std::memory_order_relaxed) & device_bit())) {
        if (cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
            large_clusters.fetch_or(device_bit(), std::memory_order_relaxed);
        } else {
            cudaGetLastError();
            ctas = 8;
        }
    }
    const int most = std::max(batch, (max_rows + 3) / 4);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.in_place ? ctas : 1; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(ctas > 1 ? PLAN_THREADS / 2 : std::min(PLAN_THREADS, (most + 31) / 32 * 32));
    cfg.dynamicSmemBytes = smem; cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = p.in_place && ctas > 1 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, paged_plan_kernel, p);
    if (e != cudaSuccess && p.in_place && ctas == 16) {
        cudaGetLastError();
        cfg.gridDim = dim3(8);
        attr[1].val.clusterDim.x = 8;
        e = cudaLaunchKernelEx(&cfg, paged_plan_kernel, p);
    }
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { set_error("nomos_kv_paged_plan: %s", cudaGetErrorString(e)); return NOMOS_ECUDA; }
    return NOMOS_OK;
}

}  // namespace nomos
