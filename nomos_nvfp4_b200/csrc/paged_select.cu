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
// Bound by latency: 4.7 us for 4 units of 64 pages, 10.8 us for 384 units of 256 (25 MB of bounds), 10 us for 8 units of 4096, of
// which scores 2, key range and rounds 3, the lists 2; launches back to back, the rest dependent loads and the cluster's barriers.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "kv_rows.cuh"
#include "launch.h"

namespace nomos {

constexpr int SEL_PAGE = 128, SEL_HD = 128;
constexpr int SEL_WARPS = 16;            // most warps of a CTA
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

// Bounds of 16 pages, as one lane holds them: 64 bytes of page g and of page g + 8 of the step, and their scales.
struct PageStep {
    uint4 d[2][4];
    float t_page[2];
    bool ok[2];
};

__global__ void __launch_bounds__(SEL_WARPS * 32, 1) paged_select_kernel(const __grid_constant__ SelectParams p) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    extern __shared__ __align__(16) uint32_t keys[];                 // first CTA: a key per page
    __shared__ __align__(16) int8_t qs[8][2 * SEL_HD + 16];          // per head: max(q^, 0), then min(q^, 0) (rows 16 bytes apart in the banks)
    __shared__ float qscale[8];
    __shared__ uint2 s_count[2][SEL_WARPS];
    __shared__ uint32_t s_range[2][SEL_WARPS];
    const int rank = blockIdx.x, C = gridDim.x, h = blockIdx.y, row = blockIdx.z;
    const int nthreads = blockDim.x, nwarps = nthreads >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
            for (int i = threadIdx.x; i < p.top; i += nthreads) {
                if (i < n) list[i] = table[i];
                if (sel) sel[i] = i < n ? i : -1;
            }
        return;
    }
    // every CTA of the cluster is running before anyone writes to the first one's shared memory; asked for here, waited for there
    if (C > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    // ---- bounds of the first step's pages: on their way while the query is prepared.  The 256 codes of a page meet the 256 of
    // the query in any order, as long as both use the same one: lane (g, t) takes bytes [64 j + 16 t, + 16) of page g (and
    // g + 8) with one wide load each and feeds its words to the operand positions of two instructions; the query's words go
    // the same way.
    const int g = lane >> 2, t = lane & 3;
    const int steps = (n + 15) / 16, stride = C * nwarps;
    auto load_step = [&](int s, PageStep &x) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int i = 16 * s + g + 8 * k;
            const int page = i < n ? table[i] : -1;
            x.ok[k] = page >= 0 && page < p.n_pages;
            const size_t u = (size_t)(x.ok[k] ? page : 0) * p.nkv + h;
            const uint4 *src = reinterpret_cast<const uint4 *>(p.kb_pool + u * 2 * SEL_HD) + t;
#pragma unroll
            for (int j = 0; j < 4; ++j) x.d[k][j] = src[4 * j];
            x.t_page[k] = p.kbs_pool[u];
        }
    };
    float xq[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const size_t at = ((size_t)row * p.nh + h * p.kvg + min(warp + nwarps * i, p.kvg - 1)) * SEL_HD + lane;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            xq[i][k] = p.q_bf16 ? __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const uint16_t *>(p.q) + at + 32 * k) << 16)
                                : __ldcg(reinterpret_cast<const float *>(p.q) + at + 32 * k);
    }
    PageStep cur;
    int s = rank * nwarps + warp;
    if (s < steps) load_step(s, cur);
    // ---- the group's queries, a warp per head
    for (int i2 = 0; i2 < 2; ++i2) {
        const int j = warp + nwarps * i2;
        if (j >= 8) break;
        float x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[k] = i2 ? xq[1][k] : xq[0][k];
            x[k] = fabsf(x[k]) <= SEL_FLT_MAX ? x[k] : 0.0f;
        }
        const float amax = warp_absmax(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))));
        float scale = __fdiv_rn(amax, 127.0f);
        if (scale == 0.0f) scale = 1.0f;
        const float inv = __fdiv_rn(1.0f, scale);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int c = round_away_clamp(__fmul_rn(x[k], inv), 127);
            qs[j][lane + 32 * k] = (int8_t)max(c, 0);
            qs[j][SEL_HD + lane + 32 * k] = (int8_t)min(c, 0);
        }
        if (lane == 0) qscale[j] = scale;
    }
    __syncthreads();
    if (C > 1) asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
    // ---- scores: 16 pages per warp and step, the next step's bounds requested before this one's are used
    {
        uint4 qf[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[j] = *reinterpret_cast<const uint4 *>(&qs[g][64 * j + 16 * t]);
        const bool c0_ok = 2 * t < p.kvg, c1_ok = 2 * t + 1 < p.kvg;
        const float s0 = qscale[2 * t], s1 = qscale[2 * t + 1];
        uint32_t *out = C > 1 ? cluster.map_shared_rank(keys, 0) : keys;
        while (s < steps) {
            const int s_next = s + stride;
            PageStep next;
            if (s_next < steps) load_step(s_next, next);
            int acc[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t a0[4] = {cur.d[0][j].x, cur.d[1][j].x, cur.d[0][j].y, cur.d[1][j].y};
                mma_s8s8(acc, a0, qf[j].x, qf[j].y);
                const uint32_t a1[4] = {cur.d[0][j].z, cur.d[1][j].z, cur.d[0][j].w, cur.d[1][j].w};
                mma_s8s8(acc, a1, qf[j].z, qf[j].w);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                // keys order like scores: the maximum over the heads is taken of the keys
                uint32_t key = 0;
                if (c0_ok) key = score_key(__fmul_rn(__fmul_rn((float)acc[2 * k], cur.t_page[k]), s0));
                if (c1_ok) key = max(key, score_key(__fmul_rn(__fmul_rn((float)acc[2 * k + 1], cur.t_page[k]), s1)));
                key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
                key = max(key, __shfl_xor_sync(0xffffffffu, key, 2));
                const int i = 16 * s + g + 8 * k;
                if (t == 0 && i < n) {
                    if (!cur.ok[k]) key = 0;                          // no such page in the pool: last of all
                    if (i < p.sink || i >= n - p.local) key = 0xffffffffu;
                    out[i] = key;
                }
            }
            s = s_next;
            cur = next;
        }
    }
    if (C > 1) {
        cluster.sync();
        if (rank != 0) return;
    } else {
        __syncthreads();
    }
    // ---- the top-th largest key, two bits per round from the highest one in which the keys differ; counts of three candidates
    // at once.  A warp owns neighbouring keys, the first 8 of each lane in registers.  Ends as soon as exactly `top` keys
    // reach the candidate: a dozen bits tell most sets of pages apart.
    constexpr int KR = 8;
    const int span = ((n + nwarps - 1) / nwarps + 31) / 32 * 32;
    const int w0 = warp * span, w1 = min(n, w0 + span);
    uint32_t kreg[KR];
    uint32_t lo = 0xffffffffu, hi = 0;   // range of the keys that are not forced
#pragma unroll
    for (int j = 0; j < KR; ++j) {
        const int i = w0 + 32 * j + lane;
        kreg[j] = i < w1 ? keys[i] : 0u;
        if (i < w1 && kreg[j] != 0xffffffffu) { lo = min(lo, kreg[j]); hi = max(hi, kreg[j]); }
    }
    for (int i = w0 + 32 * KR + lane; i < w1; i += 32)
        if (keys[i] != 0xffffffffu) { lo = min(lo, keys[i]); hi = max(hi, keys[i]); }
    lo = __reduce_min_sync(0xffffffffu, lo);
    hi = __reduce_max_sync(0xffffffffu, hi);
    if (lane == 0) { s_range[0][warp] = lo; s_range[1][warp] = hi; }
    __syncthreads();
    lo = __reduce_min_sync(0xffffffffu, lane < nwarps ? s_range[0][lane] : 0xffffffffu);
    hi = __reduce_max_sync(0xffffffffu, lane < nwarps ? s_range[1][lane] : 0u);
    // all keys that are not forced agree above `bit`; the forced ones (fewer than top, or all that is wanted) lie above them
    const int bits = lo < hi ? 32 - __clz(lo ^ hi) : 0;
    uint32_t thr = bits == 32 ? 0u : (hi >> bits) << bits;
    const uint32_t want = (uint32_t)p.top;
    if (p.sink + p.local == p.top) thr = 0xffffffffu;                 // only the forced ones
    else {
#pragma unroll 1
        for (int bit = (bits + 1) / 2 * 2 - 2, it = 0; bit >= 0; bit -= 2, ++it) {
            const uint32_t t1 = thr | (1u << bit), t2 = thr | (2u << bit), t3 = thr | (3u << bit);
            uint32_t c12 = 0, c3 = 0;
            auto count = [&](uint32_t k) {
                c12 += (k >= t1 ? 1u : 0u) + (k >= t2 ? 0x10000u : 0u);
                c3 += k >= t3 ? 1u : 0u;
            };
#pragma unroll
            for (int j = 0; j < KR; ++j)
                if (32 * j < span) count(kreg[j]);                    // (the fill, 0, reaches no candidate)
            for (int i = w0 + 32 * KR + lane; i < w1; i += 32) count(keys[i]);
            c12 = __reduce_add_sync(0xffffffffu, c12);
            c3 = __reduce_add_sync(0xffffffffu, c3);
            if (lane == 0) s_count[it & 1][warp] = make_uint2(c12, c3);
            __syncthreads();
            uint2 c = lane < nwarps ? s_count[it & 1][lane] : make_uint2(0, 0);
            const uint32_t n1 = __reduce_add_sync(0xffffffffu, c.x & 0xffffu), n2 = __reduce_add_sync(0xffffffffu, c.x >> 16),
                           n3 = __reduce_add_sync(0xffffffffu, c.y);
            uint32_t reach = 0;
            if (n3 >= want) { thr = t3; reach = n3; }
            else if (n2 >= want) { thr = t2; reach = n2; }
            else if (n1 >= want) { thr = t1; reach = n1; }
            if (reach == want) break;
        }
    }
    __syncthreads();                     // s_count is written again
    // ---- everything above it, and as many equal to it, from the front, as are still wanted
    uint32_t above = 0, equal = 0;
    auto tally = [&](uint32_t k) { above += k > thr; equal += k == thr; };
#pragma unroll
    for (int j = 0; j < KR; ++j)
        if (w0 + 32 * j + lane < w1) tally(kreg[j]);
    for (int i = w0 + 32 * KR + lane; i < w1; i += 32) tally(keys[i]);
    above = __reduce_add_sync(0xffffffffu, above);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) s_count[0][warp] = make_uint2(above, equal);
    __syncthreads();
    const uint2 of_warp = lane < nwarps ? s_count[0][lane] : make_uint2(0, 0);
    const int above_all = (int)__reduce_add_sync(0xffffffffu, of_warp.x);
    // of the warps before this one
    int a0 = (int)__reduce_add_sync(0xffffffffu, lane < warp ? of_warp.x : 0u), e0 = (int)__reduce_add_sync(0xffffffffu, lane < warp ? of_warp.y : 0u);
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
    // CTAs per unit: enough to fill the GPU, at most the portable cluster size, none without a step of 16 pages per warp
    const long units = (long)s.rows * s.nkv;
    const int steps = (pages + 15) / 16;
    int ctas = 8;
    while (ctas > 1 && (ctas * units > 2 * 148 || ctas * SEL_WARPS > steps)) ctas /= 2;
    // warps of a CTA: one step each, at least four (the selection's and the query's work); fewer where there are more units than
    // the SMs hold at sixteen warps
    int warps = 4;
    while (warps < SEL_WARPS && warps * ctas < steps && 2 * warps * ctas * units <= 148 * SEL_WARPS) warps *= 2;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, s.nkv, s.rows); cfg.blockDim = dim3(warps * 32); cfg.dynamicSmemBytes = smem; cfg.stream = st;
    cfg.attrs = attr; cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, paged_select_kernel, p);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { set_error("nomos_attn_paged_sparse_i8: page selection: %s", cudaGetErrorString(e)); return NOMOS_ECUDA; }
    return NOMOS_OK;
}

}  // namespace nomos
