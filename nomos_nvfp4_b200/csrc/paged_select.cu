// Page selection of the sparse paged attention (sm_100a, head_dim 128): which pages of its sequence a query row reads.
// One unit = (query row, KV head).  With the query quantised per head to int8 (row codec, elements that are not finite
// count 0), q^, scale s, and a page's bounds hi8, lo8, scale t (paged_rows.cu):
//   bound(page, head) = fl(fl(t * sum_d (max(q^_d, 0) hi8_d + min(q^_d, 0) lo8_d)) * s)
//   score(page) = max over the group's heads, NaN -> largest finite value, clamped to finite values
// The sum is one of whole numbers below 2^24 on the int8 tensor cores, exact in any order, so the selection is reproducible
// to the bit.  Taken are the first `sink` pages, the last `local` ones and the best of the others (ties: lower page first),
// `top` in all, listed in ascending order: of the pages listed only the last, the row's own, is partial.
// Bytes: 260 per page and KV head, against 33 792 for the page itself.  A unit is spread over a cluster (more CTAs read
// the bounds at once than there are units); its scores meet in the first CTA's shared memory, which selects.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "kv_rows.cuh"
#include "launch.h"

namespace nomos {

constexpr int SEL_PAGE = 128, SEL_HD = 128;
constexpr int SEL_THREADS = 256, SEL_WARPS = SEL_THREADS / 32;
constexpr float SEL_FLT_MAX = 3.402823466e38f;

struct SelectParams {
    const uint8_t *q;                    // [rows][nh][128]
    const int8_t *kb_pool;               // [n_pages][nkv][hi, lo][128]
    const float *kbs_pool;               // [n_pages][nkv]
    const int *block_table, *row_seq, *row_pos;
    int *lists, *lens;                   // [rows][nkv][top] pages of the pool; [rows][nkv] keys to attend (0: row skipped)
    int *sel;                            // optional [rows][nkv][top] page numbers within the sequence, -1 beyond
    int q_bf16, batch, nh, nkv, kvg, n_pages, max_pages, max_len, top, sink, local;
};

// Scores as unsigned numbers that order like them.
__device__ __forceinline__ uint32_t score_key(float s) {
    s = s != s ? SEL_FLT_MAX : fminf(fmaxf(s, -SEL_FLT_MAX), SEL_FLT_MAX);
    const uint32_t u = __float_as_uint(__fadd_rn(s, 0.0f));          // -0 -> +0
    return (u >> 31) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(SEL_THREADS) paged_select_kernel(const __grid_constant__ SelectParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) uint32_t keys[];                 // first CTA: a key per page
    __shared__ __align__(16) int8_t qs[8][2 * SEL_HD];               // per head: max(q^, 0), then min(q^, 0)
    __shared__ float qscale[8];
    __shared__ uint2 s_count[2][SEL_WARPS];
    const int rank = blockIdx.x, C = gridDim.x, h = blockIdx.y, row = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const size_t unit = (size_t)row * p.nkv + h;
    const int b = p.row_seq[row], pos = p.row_pos[row];
    // (the same in every CTA of the cluster: it leaves as a whole)
    if (b < 0 || b >= p.batch || pos < 0 || pos >= p.max_len) {
        if (rank == 0 && threadIdx.x == 0) p.lens[unit] = 0;
        return;
    }
    const int n = pos / SEL_PAGE + 1;    // pages of the row; max_len <= 128 * max_pages
    const int *table = p.block_table + (size_t)b * p.max_pages;
    int *list = p.lists + unit * p.top;
    int *sel = p.sel ? p.sel + unit * p.top : nullptr;
    if (rank == 0 && threadIdx.x == 0) p.lens[unit] = (min(n, p.top) - 1) * SEL_PAGE + pos % SEL_PAGE + 1;
    if (n <= p.top) {                    // all of them
        if (rank == 0)
            for (int i = threadIdx.x; i < p.top; i += SEL_THREADS) {
                if (i < n) list[i] = table[i];
                if (sel) sel[i] = i < n ? i : -1;
            }
        return;
    }
    // ---- the group's queries, one warp per head
    if (warp < 8) {
        float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (warp < p.kvg) {
            const size_t at = ((size_t)row * p.nh + h * p.kvg + warp) * SEL_HD + lane;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float v = p.q_bf16 ? __uint_as_float((uint32_t)reinterpret_cast<const uint16_t *>(p.q)[at + 32 * k] << 16)
                                         : reinterpret_cast<const float *>(p.q)[at + 32 * k];
                x[k] = fabsf(v) <= SEL_FLT_MAX ? v : 0.0f;
            }
        }
        const float amax = warp_absmax(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
        float scale = __fdiv_rn(amax, 127.0f);
        if (scale == 0.0f) scale = 1.0f;
        const float inv = __fdiv_rn(1.0f, scale);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = round_away_clamp(__fmul_rn(x[k], inv), 127);
            qs[warp][lane + 32 * k] = (int8_t)max(c, 0);
            qs[warp][SEL_HD + lane + 32 * k] = (int8_t)min(c, 0);
        }
        if (lane == 0) qscale[warp] = scale;
    }
    cluster.sync();                      // and every CTA of the cluster is running: its shared memory may be written
    // ---- scores: 16 pages per warp and step.  The 256 codes of a page meet the 256 of the query in any order, as long as
    // both use the same one: lane (g, t) takes bytes [64 j + 16 t, + 16) of page g (and g + 8) with one wide load each and
    // feeds its words to the operand positions of two instructions; the query's words go the same way.
    {
        const int g = lane >> 2, t = lane & 3;
        uint4 qf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[j] = *reinterpret_cast<const uint4 *>(&qs[g][64 * j + 16 * t]);
        const bool c0_ok = 2 * t < p.kvg, c1_ok = 2 * t + 1 < p.kvg;
        const float s0 = qscale[2 * t], s1 = qscale[2 * t + 1];
        uint32_t *out = cluster.map_shared_rank(keys, 0);
        const int steps = (n + 15) / 16;
        for (int s = rank * SEL_WARPS + warp; s < steps; s += C * SEL_WARPS) {
            uint4 d[2][4];
            float t_page[2];
            bool ok[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int i = 16 * s + g + 8 * k;
                const int page = i < n ? table[i] : -1;
                ok[k] = page >= 0 && page < p.n_pages;
                const size_t u = (size_t)(ok[k] ? page : 0) * p.nkv + h;
                const uint4 *src = reinterpret_cast<const uint4 *>(p.kb_pool + u * 2 * SEL_HD) + t;
#pragma unroll
                for (int j = 0; j < 4; ++j) d[k][j] = src[4 * j];
                t_page[k] = p.kbs_pool[u];
            }
            int acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t a0[4] = {d[0][j].x, d[1][j].x, d[0][j].y, d[1][j].y};
                mma_s8s8(acc, a0, qf[j].x, qf[j].y);
                const uint32_t a1[4] = {d[0][j].z, d[1][j].z, d[0][j].w, d[1][j].w};
                mma_s8s8(acc, a1, qf[j].z, qf[j].w);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                // keys order like scores: the maximum over the heads is taken of the keys
                uint32_t key = 0;
                if (c0_ok) key = score_key(__fmul_rn(__fmul_rn((float)acc[2 * k], t_page[k]), s0));
                if (c1_ok) key = max(key, score_key(__fmul_rn(__fmul_rn((float)acc[2 * k + 1], t_page[k]), s1)));
                key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
                key = max(key, __shfl_xor_sync(0xffffffffu, key, 2));
                const int i = 16 * s + g + 8 * k;
                if (t == 0 && i < n) {
                    if (!ok[k]) key = 0;                              // no such page in the pool: last of all
                    if (i < p.sink || i >= n - p.local) key = 0xffffffffu;
                    out[i] = key;
                }
            }
        }
    }
    cluster.sync();
    if (rank != 0) return;
    // ---- the top-th largest key: two bits per round, from the top; counts of three candidates at once
    const int span = ((n + SEL_WARPS - 1) / SEL_WARPS + 31) / 32 * 32;   // keys of a warp, neighbouring
    const int w0 = warp * span, w1 = min(n, w0 + span);
    uint32_t thr = 0;
#pragma unroll 1
    for (int bit = 30, it = 0; bit >= 0; bit -= 2, ++it) {
        const uint32_t t1 = thr | (1u << bit), t2 = thr | (2u << bit), t3 = thr | (3u << bit);
        uint32_t c12 = 0, c3 = 0;
        for (int i = w0 + lane; i < w1; i += 32) {
            const uint32_t k = keys[i];
            c12 += (k >= t1 ? 1u : 0u) + (k >= t2 ? 0x10000u : 0u);
            c3 += k >= t3;
        }
        c12 = __reduce_add_sync(0xffffffffu, c12);
        c3 = __reduce_add_sync(0xffffffffu, c3);
        if (lane == 0) s_count[it & 1][warp] = make_uint2(c12, c3);
        __syncthreads();
        uint32_t n1 = 0, n2 = 0, n3 = 0;
#pragma unroll
        for (int k = 0; k < SEL_WARPS; ++k) {
            const uint2 c = s_count[it & 1][k];
            n1 += c.x & 0xffffu; n2 += c.x >> 16; n3 += c.y;
        }
        thr = n3 >= (uint32_t)p.top ? t3 : n2 >= (uint32_t)p.top ? t2 : n1 >= (uint32_t)p.top ? t1 : thr;
    }
    // ---- everything above it, and as many equal to it, from the front, as are still wanted
    uint32_t above = 0, equal = 0;
    for (int i = w0 + lane; i < w1; i += 32) {
        const uint32_t k = keys[i];
        above += k > thr;
        equal += k == thr;
    }
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) s_count[0][warp] = make_uint2(above, equal);
    __syncthreads();
    int above_all = 0, a0 = 0, e0 = 0;   // of all warps; of the warps before this one
#pragma unroll
    for (int k = 0; k < SEL_WARPS; ++k) {
        const uint2 c = s_count[0][k];
        above_all += (int)c.x;
        a0 += k < warp ? (int)c.x : 0;
        e0 += k < warp ? (int)c.y : 0;
    }
    const int equal_wanted = p.top - above_all;
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t k = i < w1 ? keys[i] : 0u;
        const bool gt = i < w1 && k > thr, eq = i < w1 && k == thr;
        const unsigned mg = __ballot_sync(0xffffffffu, gt), me = __ballot_sync(0xffffffffu, eq);
        const unsigned below = (1u << lane) - 1;
        const int ga = a0 + __popc(mg & below), ea = e0 + __popc(me & below);
        if (gt || (eq && ea < equal_wanted)) {
            const int at = ga + min(ea, equal_wanted);
            list[at] = table[i];
            if (sel) sel[at] = i;
        }
        a0 += __popc(mg);
        e0 += __popc(me);
    }
}

int launch_paged_select(cudaStream_t st, const PagedSelect &s) {
    const int pages = (s.max_len + SEL_PAGE - 1) / SEL_PAGE;
    const size_t smem = pages > s.top ? (size_t)pages * 4 : 0;
    cudaError_t e = smem > 40 * 1024 ? cudaFuncSetAttribute(paged_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SELECT_MAX_PAGES * 4) : cudaSuccess;
    if (e != cudaSuccess) { set_error("nomos_attn_paged_sparse_i8: shared memory: %s", cudaGetErrorString(e)); return NOMOS_ECUDA; }
    SelectParams p{static_cast<const uint8_t *>(s.q), static_cast<const int8_t *>(s.kb_pool), static_cast<const float *>(s.kbs_pool),
                   s.block_table, s.row_seq, s.row_pos, s.lists, s.lens, s.sel, s.q_bf16, s.batch, s.nh, s.nkv, s.kvg, s.n_pages,
                   s.max_pages, s.max_len, s.top, s.sink, s.local};
    // CTAs per unit: enough to fill the GPU twice over, at most the portable cluster size, none without a step of pages per warp
    const long units = (long)s.rows * s.nkv;
    int ctas = 8;
    while (ctas > 1 && (ctas * units > 4 * 148 || ctas * SEL_WARPS * 16 > pages)) ctas /= 2;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, s.nkv, s.rows); cfg.blockDim = dim3(SEL_THREADS); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, paged_select_kernel, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { set_error("nomos_attn_paged_sparse_i8: page selection: %s", cudaGetErrorString(e)); return NOMOS_ECUDA; }
    return NOMOS_OK;
}

}  // namespace nomos
