// Rows of a step into paged int8 caches by slot map, and the page bounds that page selection reads (sm_100a, head_dim 128).
// Row codec: that of kv_rows.cuh, bit for bit.  Page bounds, per page and KV head: with v = fl(code * row scale) over the
// page's 128 rows, hi[d] = max v, lo[d] = min v, a = max_d max(|hi|, |lo|), t = a / 127 (0 -> 1), stored as int8
// min(127, ceil(hi / t)) and max(-127, floor(lo / t)): rounded outwards, so that  sum_d max(q hi, q lo) * t  is at least
// q . k of every key of the page.  A page with a row scale that is not finite gets t = +inf and codes 0.
// Both are streams: a row is read once and written once, a completed page's K codes are read back once, mostly out of L2.
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
    int n_rows, nkv, l_kvd;
    long n_slots;                        // n_pages * 128: slots outside [0, n_slots) are skipped
};

constexpr int PR_WARPS = 8;              // rows per block

// A warp per (row, K or V, KV head); lane l holds elements 4l .. 4l + 3: one wide load, one 4-byte store of codes.
// VEC: rows start on a boundary of four elements; otherwise the same elements one by one.
template <typename SrcT, bool VEC>
__global__ void __launch_bounds__(PR_WARPS * 32) append_slots_i8_kernel(const __grid_constant__ PagedRowsArgs a) {
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const long w = (long)blockIdx.x * PR_WARPS + (threadIdx.x >> 5);
    if (w >= 2l * a.n_rows * a.nkv) return;
    const int lane = threadIdx.x & 31;
    const long t = w >> 1;
    const int kv = (int)(w & 1), h = (int)(t % a.nkv);
    const long r = t / a.nkv;
    const SrcT *src = static_cast<const SrcT *>(kv ? a.src_v : a.src_k) + (size_t)r * a.l_kvd + (size_t)h * PR_HD + 4 * lane;
    float x[4];
    if constexpr (VEC && sizeof(SrcT) == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(src);
        x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
    } else if constexpr (VEC) {
        const uint2 v = *reinterpret_cast<const uint2 *>(src);
        x[0] = __uint_as_float(v.x << 16); x[1] = __uint_as_float(v.x & 0xffff0000u);
        x[2] = __uint_as_float(v.y << 16); x[3] = __uint_as_float(v.y & 0xffff0000u);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = load_as_f32(src + k);
    }
    const long slot = a.slot_map[r];
    if (slot < 0 || slot >= a.n_slots) return;
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = fmaxf(m, fabsf(x[k]));
    m = warp_absmax(m);
    float scale = __fdiv_rn(m, 127.0f);
    if (scale == 0.0f) scale = 1.0f;
    const float inv = __fdiv_rn(1.0f, scale);
    uint32_t codes = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) codes |= ((uint32_t)round_away_clamp(__fmul_rn(x[k], inv), 127) & 0xffu) << (8 * k);
    const size_t row = ((size_t)(slot / PR_PAGE) * a.nkv + h) * PR_PAGE + (size_t)(slot % PR_PAGE);
    reinterpret_cast<uint32_t *>((kv ? a.v_pool : a.k_pool) + row * PR_HD)[lane] = codes;
    if (lane == 0) (kv ? a.vs_pool : a.ks_pool)[row] = scale;
}

constexpr int PB_THREADS = 256;

// Bounds of one page and head by a block of 256 threads: thread = 16 channels of rows (tid / 8), + 32, + 64, + 96.
__device__ __forceinline__ void page_bounds(const int8_t *k_pool, const float *ks_pool, int8_t *kb_pool, float *kbs_pool, size_t unit,
                                            float (*red)[2][PR_HD], float *s_amax, int *s_bad) {
    const int tid = threadIdx.x, row0 = tid >> 3, c0 = (tid & 7) * 16, warp = tid >> 5, lane = tid & 31;
    const uint4 *kp = reinterpret_cast<const uint4 *>(k_pool + unit * PR_PAGE * PR_HD);
    const float *sp = ks_pool + unit * PR_PAGE;
    uint4 raw[4];
    float sc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        raw[i] = __ldcg(kp + (size_t)(row0 + 32 * i) * 8 + (tid & 7));
        sc[i] = __ldcg(sp + row0 + 32 * i);
    }
    bool bad = false;
    float hi[16], lo[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) { hi[e] = -CUDART_INF_F; lo[e] = CUDART_INF_F; }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bad |= !(fabsf(sc[i]) <= 3.402823466e38f);
        const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float v = __fmul_rn((float)(int8_t)(w[e >> 2] >> (8 * (e & 3))), sc[i]);
            hi[e] = fmaxf(hi[e], v);
            lo[e] = fminf(lo[e], v);
        }
    }
    // rows of the warp (lanes 8 apart hold the same channels), then of the eight warps
#pragma unroll
    for (int o = 8; o < 32; o <<= 1)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            hi[e] = fmaxf(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], o));
            lo[e] = fminf(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], o));
        }
    __syncthreads();                     // the scratch may still be read for the block's previous page
    if (tid == 0) { *s_bad = 0; }
    if (lane < 8)
#pragma unroll
        for (int e = 0; e < 16; ++e) { red[warp][0][c0 + e] = hi[e]; red[warp][1][c0 + e] = lo[e]; }
    __syncthreads();
    if (bad) *s_bad = 1;
    const int side = tid >> 7, d = tid & 127;                         // threads 0..127: hi, 128..255: lo
    float b = red[0][side][d];
#pragma unroll
    for (int k = 1; k < PB_THREADS / 32; ++k) b = side ? fminf(b, red[k][side][d]) : fmaxf(b, red[k][side][d]);
    const float wa = warp_absmax(b);
    if (lane == 0) s_amax[warp] = wa;
    __syncthreads();
    float amax = s_amax[0];
#pragma unroll
    for (int k = 1; k < PB_THREADS / 32; ++k) amax = fmaxf(amax, s_amax[k]);
    const bool finite = !*s_bad && amax <= 3.402823466e38f;
    float t = __fdiv_rn(amax, 127.0f);
    if (t == 0.0f) t = 1.0f;
    const float q = __fdiv_rn(b, t);
    const int code = !finite ? 0 : side ? max(-127, __float2int_rd(q)) : min(127, __float2int_ru(q));
    kb_pool[unit * 2 * PR_HD + tid] = (int8_t)code;
    if (tid == 0) kbs_pool[unit] = finite ? t : CUDART_INF_F;
}

struct PageBoundsArgs {
    const int8_t *k_pool;
    const float *ks_pool;
    int8_t *kb_pool;
    float *kbs_pool;
    const int *list;                     // slots (a page is taken where its last row was written) or page ids
    int n, nkv, span;                    // entries, and how many of them a block looks at
    long n_pages;
    int slots;
};

// grid (entry spans, KV heads): a block finds the pages of its span and works them out one after the other.
__global__ void __launch_bounds__(PB_THREADS) page_bounds_kernel(const __grid_constant__ PageBoundsArgs a) {
    __shared__ float red[PB_THREADS / 32][2][PR_HD];
    __shared__ float s_amax[PB_THREADS / 32];
    __shared__ int s_bad;
    __shared__ int s_pages[PB_THREADS], s_n;
    if (threadIdx.x == 0) s_n = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int i = blockIdx.x * a.span + threadIdx.x;
    if ((int)threadIdx.x < a.span && i < a.n) {
        const int v = a.list[i];
        const bool last = !a.slots || (v >= 0 && v % PR_PAGE == PR_PAGE - 1);
        const int page = a.slots ? v / PR_PAGE : v;
        if (last && page >= 0 && page < a.n_pages) s_pages[atomicAdd(&s_n, 1)] = page;   // any order: pages are independent
    }
    __syncthreads();
    const int n = s_n;
    for (int k = 0; k < n; ++k)
        page_bounds(a.k_pool, a.ks_pool, a.kb_pool, a.kbs_pool, (size_t)s_pages[k] * a.nkv + blockIdx.y, red, s_amax, &s_bad);
}

static int launch_bounds(cudaStream_t st, const PageBoundsArgs &in, const char *who) {
    PageBoundsArgs a = in;
    // In a decode step few rows end a page, in a prompt every 128th does: spans short enough that a block rarely finds more
    // than one, long enough that the blocks that find none are few.
    a.span = a.slots ? 64 : 1;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((a.n + a.span - 1) / a.span, a.nkv); cfg.blockDim = dim3(PB_THREADS); cfg.stream = st;
    cfg.attrs = pdl; cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, page_bounds_kernel, a);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { set_error("%s: %s", who, cudaGetErrorString(e)); return NOMOS_ECUDA; }
    return NOMOS_OK;
}

int launch_page_bounds(cudaStream_t st, const void *k_pool, const void *ks_pool, void *kb_pool, void *kbs_pool, const int *pages, int n,
                       int nkv, int n_pages) {
    return launch_bounds(st, PageBoundsArgs{static_cast<const int8_t *>(k_pool), static_cast<const float *>(ks_pool), static_cast<int8_t *>(kb_pool),
                                            static_cast<float *>(kbs_pool), pages, n, nkv, 1, n_pages, 0}, "nomos_kv_paged_page_bounds_i8");
}

int launch_append_slots_i8(cudaStream_t st, const void *src_k, const void *src_v, void *k_pool, void *v_pool, void *ks_pool, void *vs_pool,
                           void *kb_pool, void *kbs_pool, const int *slot_map, int n_rows, int nkv, int l_kvd, int n_pages, int src_bf16) {
    const char *who = "nomos_kv_paged_append_rows_i8";
    PagedRowsArgs a{src_k, src_v, static_cast<int8_t *>(k_pool), static_cast<int8_t *>(v_pool), static_cast<float *>(ks_pool),
                    static_cast<float *>(vs_pool), slot_map, n_rows, nkv, l_kvd, (long)n_pages * PR_PAGE};
    const int unit = src_bf16 ? 8 : 16;  // four elements
    const bool vec = l_kvd % 4 == 0 && ((reinterpret_cast<uintptr_t>(src_k) | reinterpret_cast<uintptr_t>(src_v)) & (unit - 1)) == 0;
    cudaLaunchAttribute pdl[1];
    pdl[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((2l * n_rows * nkv + PR_WARPS - 1) / PR_WARPS)); cfg.blockDim = dim3(PR_WARPS * 32); cfg.stream = st;
    cfg.attrs = pdl; cfg.numAttrs = 1;
    cudaError_t e = src_bf16 ? cudaLaunchKernelEx(&cfg, vec ? append_slots_i8_kernel<__nv_bfloat16, true> : append_slots_i8_kernel<__nv_bfloat16, false>, a)
                             : cudaLaunchKernelEx(&cfg, vec ? append_slots_i8_kernel<float, true> : append_slots_i8_kernel<float, false>, a);
    if (e == cudaSuccess) e = cudaGetLastError();
    if (e != cudaSuccess) { set_error("%s: %s", who, cudaGetErrorString(e)); return NOMOS_ECUDA; }
    if (kb_pool == nullptr) return NOMOS_OK;
    return launch_bounds(st, PageBoundsArgs{a.k_pool, a.ks_pool, static_cast<int8_t *>(kb_pool), static_cast<float *>(kbs_pool), slot_map, n_rows,
                                            nkv, 0, n_pages, 1}, who);
}

}  // namespace nomos
