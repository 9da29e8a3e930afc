// Rows of a step into paged int8 caches by slot map, and the page bounds that page selection reads (sm_100a, head_dim 128).
// Row codec: that of kv_rows.cuh, bit for bit.  Page bounds, per page and KV head: with v = fl(code * row scale) over the
// page's 128 rows, hi[d] = max v, lo[d] = min v, a = max_d max(|hi|, |lo|), t = a / 127 (0 -> 1), stored as int8
// min(127, ceil(hi / t)) and max(-127, floor(lo / t)): rounded outwards, so that  sum_d max(q hi, q lo) * t  is at least
// q . k of every key of the page.  A page with a row scale that is not finite gets t = +inf and codes 0.
// Both are streams: a row is read once and written once, a completed page's K codes are read back once, mostly out of L2.
// 8168 rows x 16 heads: fp32 rows 26 us (6.4 TB/s, close to the copy rate), bf16 rows 22 us (4.6 TB/s, bound by instruction issue); the bounds
// of their 1024 pages and heads 10 us alone (17 MB; latency and the ALU pipe), 6 beside the V rows.
#include <math_constants.h>

#include <algorithm>

#include "common.cuh"
#include "kv_rows.cuh"
#include "launch.h"

namespace nomos {

constexpr int PR_PAGE = 128, PR_HD = 128;

struct PagedRowsArgs {
    const void *src_k, *src_v;
    int8_t *k_pool, *v_pool;
    float *ks_pool, *vs_pool;
    const int *slot_map;
    int n_rows, nkv, l_kvd, head_bits;
    unsigned n_slots;                    // n_pages * 128 < 2^31: slots outside [0, n_slots) are skipped
};

constexpr int PR_WARPS = 8;              // warps per block: sixteen halves

// Four codes trunc(x * inv +- 0.5) as bytes.  With a finite reciprocal of the row's scale |x * inv| <= 127 (1 + 2^-21), so the
// clamp of the codec (round_away_clamp) has nothing to do.  The conversion packs two at a time.
__device__ __forceinline__ uint32_t pack_codes(const float *x, float inv) {
    int q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float t = __fmul_rn(x[e], inv);
        q[e] = __float2int_rz(__fadd_rn(t, __uint_as_float((__float_as_uint(t) & 0x80000000u) | 0x3f000000u)));
    }
    uint32_t hi, w;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(q[3]), "r"(q[2]));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w) : "r"(q[1]), "r"(q[0]), "r"(hi));
    return w;
}

__device__ __forceinline__ float load_cg(const float *p) { return __ldcg(p); }
__device__ __forceinline__ float load_cg(const __nv_bfloat16 *p) {
    return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short *>(p)) << 16);
}

// Half a warp per row of one (K or V, KV head): lane l holds elements 8l .. 8l + 7, one or two wide loads and one 8-byte store of
// codes.  The half warp takes rows r0, r0 + rows_step, ... (STEPS of them, loaded before the first use).
// VEC: rows start on a boundary of eight elements; otherwise the same elements one by one.
// Everything is read through L2 (ld.global.cg): nothing is read twice.
template <typename SrcT, bool VEC, int STEPS>
__device__ __forceinline__ void append_rows(const PagedRowsArgs &a, int kv, int h, int r0, int rows_step) {
    // wide fp32 loads: lane l holds elements 4l .. 4l + 3 of each half of the row, so that a load takes whole sectors
    constexpr bool HALVES = VEC && sizeof(SrcT) == 4;
    const int l = threadIdx.x & 15;
    const SrcT *base = static_cast<const SrcT *>(kv ? a.src_v : a.src_k) + min(h, a.nkv - 1) * PR_HD + (HALVES ? 4 : 8) * l;
    float x[STEPS][8];
    unsigned slot[STEPS];                // outside the pool: skipped
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int r = min(r0 + s * rows_step, a.n_rows - 1);
        slot[s] = (unsigned)__ldcg(a.slot_map + r);
        const SrcT *src = base + (size_t)r * a.l_kvd;
        if constexpr (VEC && sizeof(SrcT) == 4) {
            const float4 u = __ldcg(reinterpret_cast<const float4 *>(src)), v = __ldcg(reinterpret_cast<const float4 *>(src + PR_HD / 2));
            x[s][0] = u.x; x[s][1] = u.y; x[s][2] = u.z; x[s][3] = u.w;
            x[s][4] = v.x; x[s][5] = v.y; x[s][6] = v.z; x[s][7] = v.w;
        } else if constexpr (VEC) {
            const uint4 u = __ldcg(reinterpret_cast<const uint4 *>(src));
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) { x[s][2 * k] = __uint_as_float(w[k] << 16); x[s][2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u); }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) x[s][k] = load_cg(src + k);
        }
    }
    // Row maxima; lane l of a half keeps that of its step l % STEPS, so that the two divisions are done once for all steps.
    float mine = 0.0f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(x[s][k]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (l % STEPS == s) mine = m;
    }
    float scale = __fdiv_rn(mine, 127.0f);
    if (scale == 0.0f) scale = 1.0f;
    const float my_inv = __frcp_rn(scale);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const float sc = __shfl_sync(0xffffffffu, scale, s, 16), inv = __shfl_sync(0xffffffffu, my_inv, s, 16);
        if (slot[s] >= a.n_slots || h >= a.nkv || r0 + s * rows_step >= a.n_rows) continue;   // the same in all lanes of the half
        uint32_t codes[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) codes[k] = pack_codes(&x[s][4 * k], inv);
        if (!(inv <= 3.402823466e38f)) {                              // a scale below 2^-128: the products may be infinite
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                codes[k] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) codes[k] |= ((uint32_t)round_away_clamp(__fmul_rn(x[s][4 * k + e], inv), 127) & 0xffu) << (8 * e);
            }
        }
        const size_t row = ((size_t)(slot[s] / PR_PAGE) * a.nkv + h) * PR_PAGE + (size_t)(slot[s] % PR_PAGE);
        int8_t *dst = (kv ? a.v_pool : a.k_pool) + row * PR_HD;
        if constexpr (HALVES) {
            reinterpret_cast<uint32_t *>(dst)[l] = codes[0];
            reinterpret_cast<uint32_t *>(dst + PR_HD / 2)[l] = codes[1];
        } else {
            reinterpret_cast<uint2 *>(dst)[l] = make_uint2(codes[0], codes[1]);
        }
        if (l == 0) (kv ? a.vs_pool : a.ks_pool)[row] = sc;
    }
}

// The sixteen half warps of a block take the heads of one row (nkv <= 8: of several rows, 2^head_bits half warps each; nkv > 16:
// sixteen heads per blockIdx.z), so that no index needs a division, and STEPS such sets of rows.
template <typename SrcT, bool VEC, int STEPS>
__global__ void __launch_bounds__(PR_WARPS * 32) append_slots_i8_kernel(const __grid_constant__ PagedRowsArgs a) {
    const int hw = threadIdx.x >> 4;
    const int rows_step = (2 * PR_WARPS) >> a.head_bits;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    append_rows<SrcT, VEC, STEPS>(a, blockIdx.y, 2 * PR_WARPS * blockIdx.z + (hw & ((1 << a.head_bits) - 1)),
                                  blockIdx.x * (rows_step * STEPS) + (hw >> a.head_bits), rows_step);
}

constexpr int PB_THREADS = 256;
static_assert(PB_THREADS == PR_WARPS * 32, "the append of a head's rows works its pages' bounds out with the same block");
struct BoundsScratch {
    __align__(16) float red[PB_THREADS / 32][2][PR_HD];
    float amax[PB_THREADS / 32];
    int bad;
};

// Bounds of one page and head by a block of 256 threads: warp = 16 rows, lane = four channels, whose largest and smallest
// values stay in registers; every load of the page is in flight at once.
__device__ __forceinline__ void page_bounds(const int8_t *k_pool, const float *ks_pool, int8_t *kb_pool, float *kbs_pool, size_t unit,
                                            BoundsScratch &sm) {
    constexpr int RPW = PR_PAGE / (PB_THREADS / 32);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t *kp = reinterpret_cast<const uint32_t *>(k_pool + unit * PR_PAGE * PR_HD) + warp * RPW * 32 + lane;
    uint32_t raw[RPW];
#pragma unroll
    for (int i = 0; i < RPW; ++i) raw[i] = __ldcg(kp + 32 * i);
    const float sc = __ldcg(ks_pool + unit * PR_PAGE + warp * RPW + (lane & (RPW - 1)));
    const bool bad = !(fabsf(sc) <= 3.402823466e38f);
    float hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) { hi[e] = -CUDART_INF_F; lo[e] = CUDART_INF_F; }
    // two rows at a time: the largest and the smallest of three are one instruction each
#pragma unroll
    for (int i = 0; i < RPW; i += 2) {
        const float s0 = __shfl_sync(0xffffffffu, sc, i), s1 = __shfl_sync(0xffffffffu, sc, i + 1);
        const uint32_t u0 = raw[i] ^ 0x80808080u, u1 = raw[i + 1] ^ 0x80808080u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            // code + 128 as the low byte of the float 2^23 + code + 128: no conversion instruction (a quarter of the rate)
            const float v0 = __fmul_rn(__uint_as_float(prmt(u0, 0x4b000000u, 0x7440u | e)) - 8388736.0f, s0);
            const float v1 = __fmul_rn(__uint_as_float(prmt(u1, 0x4b000000u, 0x7440u | e)) - 8388736.0f, s1);
            hi[e] = fmaxf(hi[e], fmaxf(v0, v1));
            lo[e] = fminf(lo[e], fminf(v0, v1));
        }
    }
    __syncthreads();                     // the scratch may still be read for the block's previous page
    if (tid == 0) { sm.bad = 0; }
    reinterpret_cast<float4 *>(sm.red[warp][0])[lane] = make_float4(hi[0], hi[1], hi[2], hi[3]);
    reinterpret_cast<float4 *>(sm.red[warp][1])[lane] = make_float4(lo[0], lo[1], lo[2], lo[3]);
    __syncthreads();
    if (bad) sm.bad = 1;
    const int side = tid >> 7, d = tid & 127;                         // threads 0..127: hi, 128..255: lo
    float b = sm.red[0][side][d];
#pragma unroll
    for (int k = 1; k < PB_THREADS / 32; ++k) b = side ? fminf(b, sm.red[k][side][d]) : fmaxf(b, sm.red[k][side][d]);
    const float wa = warp_absmax(b);
    if (lane == 0) sm.amax[warp] = wa;
    __syncthreads();
    float amax = sm.amax[0];
#pragma unroll
    for (int k = 1; k < PB_THREADS / 32; ++k) amax = fmaxf(amax, sm.amax[k]);
    const bool finite = !sm.bad && amax <= 3.402823466e38f;
    float t = __fdiv_rn(amax, 127.0f);
    if (t == 0.0f) t = 1.0f;
    const float q = __fdiv_rn(b, t);
    const int code = !finite ? 0 : side ? max(-127, __float2int_rd(q)) : min(127, __float2int_ru(q));
    kb_pool[unit * 2 * PR_HD + tid] = (int8_t)code;
    if (tid == 0) kbs_pool[unit] = finite ? t : CUDART_INF_F;
}

// A decode step's rows (at most OWN_ROWS), and the bounds of the pages they complete, in one launch: a block takes every row of a
// head, so all that a completed page holds of this call was written by the block itself.  64 rows x 16 heads: 3.0 us, 3.6 as two
// launches (and 2 us more of host time); 200 rows 7.0 against 5.0.
constexpr int OWN_ROWS = 128;
template <typename SrcT, bool VEC>
__global__ void __launch_bounds__(PR_WARPS * 32) append_head_i8_kernel(const __grid_constant__ PagedRowsArgs a, int8_t *kb_pool, float *kbs_pool) {
    __shared__ BoundsScratch sm;
    __shared__ int s_pages[OWN_ROWS], s_n;
    const int h = blockIdx.x, kv = blockIdx.y;
    if (threadIdx.x == 0) s_n = 0;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int slot = (int)threadIdx.x < a.n_rows ? a.slot_map[threadIdx.x] : -1;
#pragma unroll 1
    for (int r0 = 0; r0 < a.n_rows; r0 += 4 * PR_WARPS) append_rows<SrcT, VEC, 2>(a, kv, h, r0 + (threadIdx.x >> 4), 2 * PR_WARPS);
    if (kv) return;
    __syncthreads();                     // the block's codes and scales are in
    if (slot >= 0 && (unsigned)slot < a.n_slots && slot % PR_PAGE == PR_PAGE - 1) s_pages[atomicAdd(&s_n, 1)] = slot / PR_PAGE;
    __syncthreads();
    const int n = s_n;
    for (int k = 0; k < n; ++k) page_bounds(a.k_pool, a.ks_pool, kb_pool, kbs_pool, (size_t)s_pages[k] * a.nkv + h, sm);
}

// Longer appends: the K rows in a grid of their own (append_slots_i8_kernel), then this grid, whose first `bound_blocks` blocks each
// look through 128 slots and work out the bounds of one head of the pages that end there (one, in a prompt); the others are V rows.
// So the bounds, bound by latency, share the SMs with a stream of rows instead of running after it.  Every block waits for the K grid:
// the bounds blocks read its rows, and for the V rows nothing else promises that what the calls before wrote (sources, slots) is
// visible.  8168 rows x 16 heads: bf16 28.3 us, fp32 33.0 (bounds blocks in the middle of the V rows 0.9 and 0.6 more; all rows in one
// grid, then the bounds, 31.1 and 34.1; V rows and slots read without the wait, 26.8 and 30.6).
struct BoundsArgs {
    int8_t *kb_pool;
    float *kbs_pool;
    int bound_blocks, row_blocks;        // row_blocks: blocks of one blockIdx.z of the row kernels
};
template <typename SrcT, bool VEC, int STEPS>
__global__ void __launch_bounds__(PR_WARPS * 32) append_v_bounds_i8_kernel(const __grid_constant__ PagedRowsArgs a, const __grid_constant__ BoundsArgs bd) {
    __shared__ BoundsScratch sm;
    __shared__ int s_pages[PR_PAGE], s_n;
    int block = blockIdx.x;
    if (threadIdx.x == 0) s_n = 0;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (block >= bd.bound_blocks) {
        block -= bd.bound_blocks;
        const int z = block / bd.row_blocks, x = block - z * bd.row_blocks, hw = threadIdx.x >> 4;
        const int rows_step = (2 * PR_WARPS) >> a.head_bits;
        append_rows<SrcT, VEC, STEPS>(a, 1, 2 * PR_WARPS * z + (hw & ((1 << a.head_bits) - 1)), x * (rows_step * STEPS) + (hw >> a.head_bits), rows_step);
        return;
    }
    const int span = block / a.nkv, h = block - span * a.nkv;
    __syncthreads();
    const int r = span * PR_PAGE + (int)threadIdx.x;
    if ((int)threadIdx.x < PR_PAGE && r < a.n_rows) {
        const unsigned slot = (unsigned)__ldcg(a.slot_map + r);
        if (slot < a.n_slots && slot % PR_PAGE == PR_PAGE - 1) s_pages[atomicAdd(&s_n, 1)] = (int)(slot / PR_PAGE);   // any order: pages are independent
    }
    __syncthreads();
    const int n = s_n;
    for (int k = 0; k < n; ++k) page_bounds(a.k_pool, a.ks_pool, bd.kb_pool, bd.kbs_pool, (size_t)s_pages[k] * a.nkv + h, sm);
}

// Bounds of listed pages, a block per page and head.
struct PageListArgs {
    const int8_t *k_pool;
    const float *ks_pool;
    int8_t *kb_pool;
    float *kbs_pool;
    const int *pages;
    int nkv, n_pages;
};
__global__ void __launch_bounds__(PB_THREADS) page_bounds_kernel(const __grid_constant__ PageListArgs a) {
    __shared__ BoundsScratch sm;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int page = a.pages[blockIdx.x];
    if (page < 0 || page >= a.n_pages) return;
    page_bounds(a.k_pool, a.ks_pool, a.kb_pool, a.kbs_pool, (size_t)page * a.nkv + blockIdx.y, sm);
}

template <typename... P, typename... A>
static int launch_rows(const char *who, cudaStream_t st, dim3 grid, void (*kernel)(P...), const A &...args) {
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(PR_WARPS * 32); cfg.stream = st;
    cfg.attrs = pdl; cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { set_error("%s: %s", who, cudaGetErrorString(e)); return NOMOS_ECUDA; }
    return NOMOS_OK;
}

int launch_page_bounds(cudaStream_t st, const void *k_pool, const void *ks_pool, void *kb_pool, void *kbs_pool, const int *pages, int n,
                       int nkv, int n_pages) {
    const PageListArgs a{static_cast<const int8_t *>(k_pool), static_cast<const float *>(ks_pool), static_cast<int8_t *>(kb_pool),
                         static_cast<float *>(kbs_pool), pages, nkv, n_pages};
    return launch_rows("nomos_kv_paged_page_bounds_i8", st, dim3(n, nkv), page_bounds_kernel, a);
}

template <typename SrcT, bool VEC>
static int launch_append(cudaStream_t st, const PagedRowsArgs &a, int8_t *kb_pool, float *kbs_pool) {
    const char *who = "nomos_kv_paged_append_rows_i8";
    if (kb_pool != nullptr && a.n_rows <= OWN_ROWS) return launch_rows(who, st, dim3(a.nkv, 2), append_head_i8_kernel<SrcT, VEC>, a, kb_pool, kbs_pool);
    // two sets of rows per block once one each would fill the GPU's warps several times over
    const bool many = (long)a.n_rows * a.nkv > 2 * 148 * 64;
    const int per_block = ((2 * PR_WARPS) >> a.head_bits) * (many ? 2 : 1);
    const int row_blocks = (int)(((long)a.n_rows + per_block - 1) / per_block), z = (a.nkv + 2 * PR_WARPS - 1) / (2 * PR_WARPS);
    int rc = launch_rows(who, st, dim3(row_blocks, kb_pool ? 1 : 2, z), many ? append_slots_i8_kernel<SrcT, VEC, 2> : append_slots_i8_kernel<SrcT, VEC, 1>, a);
    if (rc != NOMOS_OK || kb_pool == nullptr) return rc;
    const BoundsArgs bd{kb_pool, kbs_pool, (a.n_rows + PR_PAGE - 1) / PR_PAGE * a.nkv, row_blocks};
    return launch_rows(who, st, dim3(row_blocks * z + bd.bound_blocks),
                       many ? append_v_bounds_i8_kernel<SrcT, VEC, 2> : append_v_bounds_i8_kernel<SrcT, VEC, 1>, a, bd);
}

int launch_append_slots_i8(cudaStream_t st, const void *src_k, const void *src_v, void *k_pool, void *v_pool, void *ks_pool, void *vs_pool,
                           void *kb_pool, void *kbs_pool, const int *slot_map, int n_rows, int nkv, int l_kvd, int n_pages, int src_bf16) {
    PagedRowsArgs a{src_k, src_v, static_cast<int8_t *>(k_pool), static_cast<int8_t *>(v_pool), static_cast<float *>(ks_pool),
                    static_cast<float *>(vs_pool), slot_map, n_rows, nkv, l_kvd, 0, (unsigned)n_pages * PR_PAGE};
    while (a.head_bits < 4 && (1 << a.head_bits) < nkv) ++a.head_bits;
    const bool vec = l_kvd % 8 == 0 && ((reinterpret_cast<uintptr_t>(src_k) | reinterpret_cast<uintptr_t>(src_v)) & 15) == 0;
    int8_t *kb = static_cast<int8_t *>(kb_pool);
    float *kbs = static_cast<float *>(kbs_pool);
    if (src_bf16) return vec ? launch_append<__nv_bfloat16, true>(st, a, kb, kbs) : launch_append<__nv_bfloat16, false>(st, a, kb, kbs);
    return vec ? launch_append<float, true>(st, a, kb, kbs) : launch_append<float, false>(st, a, kb, kbs);
}

}  // namespace nomos
