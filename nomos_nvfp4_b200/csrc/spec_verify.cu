// Speculative verification: drafted tokens against the target's probabilities, from given random numbers (sm_100a).
//   draft i of sequence b is accepted iff u_i * q_i(x_i) < p_i(x_i)          (64-bit products of 32-bit values: exact)
//   the first one that is not, a, is replaced by a draw from w = max(p_a - q_a, 0); if all n are accepted a token is drawn
//   from w = p_n.  The draw: whole weights W_i = rint(w_i * 2^50), T = floor(u * sum W), the first i with W_0 + .. + W_i > T.
// Sums of whole numbers do not depend on their order, so the split over threads and CTAs cannot change a token; a weight
// below 2^-51 counts as nothing (the sum of a row of 2^18 of them would be 2^-33).
// What it must read: one target row per sequence, and one drafter row where a draft was rejected.  The rows are streamed
// once by the CTAs of a cluster; the stretch of the one warp that holds T is read a second time, out of L2.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "launch.h"

namespace nomos {

constexpr int SV_THREADS = 512, SV_WARPS = SV_THREADS / 32;

struct SpecVerifyArgs {
    const float *p, *q;                  // [batch][max_draft + 1][p_stride], [batch][max_draft][q_stride] or nullptr
    const int *tokens, *n_draft;
    const float *u_accept, *u_sample;
    const int *lens;
    int *lens_out, *n_accepted, *out_tokens;
    int batch, max_draft, vocab;
    long p_stride, q_stride;
};

// W of a weight d = p - q in 64 bits.  6 + d lies in [4, 8), whose doubles are 2^-50 apart: the addition rounds d to whole
// units and the difference of the bit patterns is their number.  (The conversion instruction to 64-bit integers is slower.)
__device__ __forceinline__ unsigned long long whole_weight(double d) {
    const long long u = __double_as_longlong(__dadd_rn(fmin(d, 1.0), 6.0)) - __double_as_longlong(6.0);
    return d > 0.0 ? (unsigned long long)u : 0ull;                   // NaN counts as nothing
}

// One row's weights: target row, drafter row (nullptr: none), and the index whose drafter probability is 1 (a drafter that
// gives tokens only; -1: none).
struct RowWeights {
    const float *p, *q;
    int one;
    __device__ __forceinline__ unsigned long long at(int i) const { return of(p[i], q ? q[i] : 0.0f, i); }
    __device__ __forceinline__ unsigned long long of(float pv, float qv, int i) const {
        return whole_weight((double)pv - (i == one ? 1.0 : (double)qv));
    }
};

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sum over [i0, i1) by one warp; float4 loads where both rows allow them.
__device__ __forceinline__ unsigned long long warp_range(const RowWeights &w, int i0, int i1, bool vec, int lane) {
    unsigned long long s = 0;
    if (vec) {                           // i0 is a multiple of 4
        int i = i0 + 4 * lane;
#pragma unroll 4
        for (; i + 3 < i1; i += 128) {
            const float4 pv = *reinterpret_cast<const float4 *>(w.p + i);
            const float4 qv = w.q ? *reinterpret_cast<const float4 *>(w.q + i) : make_float4(0.f, 0.f, 0.f, 0.f);
            s += w.of(pv.x, qv.x, i) + w.of(pv.y, qv.y, i + 1) + w.of(pv.z, qv.z, i + 2) + w.of(pv.w, qv.w, i + 3);
        }
        for (; i < i1; ++i) s += w.at(i);                             // the one lane whose four elements the end cuts
    } else {
#pragma unroll 4
        for (int i = i0 + lane; i < i1; i += 32) s += w.at(i);
    }
    return warp_sum(s);
}

__global__ void __launch_bounds__(SV_THREADS) spec_verify_kernel(const __grid_constant__ SpecVerifyArgs a) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ unsigned long long s_warp[2][SV_WARPS], s_total[2], s_scan[SV_WARPS];
    __shared__ int s_accepted;
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int b = blockIdx.y, rank = blockIdx.x, C = gridDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n = min(a.n_draft ? a.n_draft[b] : a.max_draft, a.max_draft);
    if (n < 0) return;                   // an idle entry of a padded batch; the whole cluster leaves
    // ---- how many drafts stand: every CTA of the cluster finds out for itself
    if (warp == 0) {
        int acc = n;
        for (int i0 = 0; i0 < n; i0 += 32) {
            const int i = i0 + lane;
            bool ok = true;
            if (i < n) {
                const int x = a.tokens[(size_t)b * a.max_draft + i];
                const double u = a.u_accept[(size_t)b * a.max_draft + i];
                ok = x >= 0 && x < a.vocab;                           // not a token: rejected
                if (ok) {
                    const double px = a.p[((size_t)b * (a.max_draft + 1) + i) * a.p_stride + x];
                    const double qx = a.q ? (double)a.q[((size_t)b * a.max_draft + i) * a.q_stride + x] : 1.0;
                    ok = __dmul_rn(u, qx) < px;
                }
            }
            const unsigned no = __ballot_sync(0xffffffffu, !ok);
            if (no) { acc = i0 + __ffs(no) - 1; break; }
        }
        if (lane == 0) s_accepted = acc;
    }
    __syncthreads();
    const int acc = s_accepted;
    RowWeights w;
    w.p = a.p + ((size_t)b * (a.max_draft + 1) + acc) * a.p_stride;
    w.q = acc < n && a.q ? a.q + ((size_t)b * a.max_draft + acc) * a.q_stride : nullptr;
    w.one = acc < n && !a.q ? a.tokens[(size_t)b * a.max_draft + acc] : -1;
    const bool vec = ((reinterpret_cast<uintptr_t>(w.p) | reinterpret_cast<uintptr_t>(w.q)) & 15) == 0;
    // stretch of this warp: [i0, i1) of the vocabulary, in multiples of four
    const int per = (int)((((long)a.vocab + (long)C * SV_WARPS - 1) / ((long)C * SV_WARPS) + 3) / 4 * 4);
    const long unit = (long)rank * SV_WARPS + warp;
    const int i0 = (int)min(unit * per, (long)a.vocab), i1 = (int)min(unit * per + per, (long)a.vocab);

#pragma unroll 1
    for (int round = 0; round < 2; ++round) {
        const unsigned long long mine = warp_range(w, i0, i1, vec, lane);
        if (lane == 0) s_warp[round][warp] = mine;
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned long long t = 0;
            for (int k = 0; k < SV_WARPS; ++k) t += s_warp[round][k];
            s_total[round] = t;
        }
        cluster.sync();
        unsigned long long total = 0, before = 0;
        for (int k = 0; k < C; ++k) {
            const unsigned long long t = *cluster.map_shared_rank(&s_total[round], k);
            before += k < rank ? t : 0;
            total += t;
        }
        if (total == 0 && round == 0 && (w.q || w.one >= 0)) {
            // the drafter covers the target everywhere (u outside [0, 1) only): the target's own row decides
            w.q = nullptr; w.one = -1;
            continue;
        }
        if (total > 0) {
            const long long t0 = (long long)floor(__dmul_rn((double)a.u_sample[b], (double)total));
            const unsigned long long T = (unsigned long long)max(0ll, min(t0, (long long)total - 1));
            if (T >= before && T < before + s_total[round]) {         // uniform over the CTA
                unsigned long long base = before;
                int k = 0;
                while (k < SV_WARPS - 1 && T >= base + s_warp[round][k]) base += s_warp[round][k++];
                // the k-th warp's stretch again, by the whole CTA: `each` neighbouring elements per thread
                const long u0 = ((long)rank * SV_WARPS + k) * per;
                const int j0 = (int)min(u0, (long)a.vocab), j1 = (int)min(u0 + per, (long)a.vocab);
                const int each = (j1 - j0 + SV_THREADS - 1) / SV_THREADS;
                const int e0 = min(j1, j0 + (int)threadIdx.x * each), e1 = min(j1, e0 + each);
                unsigned long long s = 0;
                for (int i = e0; i < e1; ++i) s += w.at(i);
                unsigned long long incl = s;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                if (lane == 31) s_scan[warp] = incl;
                __syncthreads();
                for (int k2 = 0; k2 < warp; ++k2) base += s_scan[k2];
                const unsigned long long lo = base + incl - s;
                if (T >= lo && T < lo + s) {                          // one thread of the cluster
                    unsigned long long c = lo;
                    int token = e0;
                    for (; token < e1 - 1; ++token) {
                        c += w.at(token);
                        if (c > T) break;
                    }
                    a.out_tokens[(size_t)b * (a.max_draft + 1) + acc] = token;
                }
            }
        } else if (rank == 0 && threadIdx.x == 0) {
            a.out_tokens[(size_t)b * (a.max_draft + 1) + acc] = -1;   // nothing to draw from
        }
        break;
    }
    if (rank == 0) {
        for (int i = threadIdx.x; i <= a.max_draft; i += SV_THREADS)
            if (i != acc) a.out_tokens[(size_t)b * (a.max_draft + 1) + i] = i < acc ? a.tokens[(size_t)b * a.max_draft + i] : -1;
        if (threadIdx.x == 0) {
            a.n_accepted[b] = acc;
            if (a.lens) a.lens_out[b] = a.lens[b] + acc + 1;
        }
    }
    cluster.sync();                      // the totals stay where the peers read them
}

int launch_spec_verify(cudaStream_t st, const float *p, const float *q, const int *tokens, const int *n_draft, const float *u_accept,
                       const float *u_sample, const int *lens, int *lens_out, int *n_accepted, int *out_tokens, int batch, int max_draft,
                       int vocab, long p_stride, long q_stride) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    // as many CTAs per sequence as fill the GPU about twice over, at most the portable cluster size
    int ctas = 8;
    while (ctas > 1 && (long)ctas * std::min(batch, 65535) > 2 * 148 * 2) ctas /= 2;
    while (ctas > 1 && vocab < ctas * SV_THREADS * 4) ctas /= 2;
    attr[1].val.clusterDim.x = ctas;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(SV_THREADS); cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 2;
    for (int b0 = 0; b0 < batch; b0 += 65535) {                       // the grid's y dimension
        const int nb = std::min(65535, batch - b0);
        SpecVerifyArgs a{p + (size_t)b0 * (max_draft + 1) * p_stride, q ? q + (size_t)b0 * max_draft * q_stride : nullptr,
                         tokens + (size_t)b0 * max_draft, n_draft ? n_draft + b0 : nullptr, u_accept + (size_t)b0 * max_draft, u_sample + b0,
                         lens ? lens + b0 : nullptr, lens_out ? lens_out + b0 : nullptr, n_accepted + b0, out_tokens + (size_t)b0 * (max_draft + 1),
                         nb, max_draft, vocab, p_stride, q_stride};
        cfg.gridDim = dim3(ctas, nb);
        cudaError_t e = cudaLaunchKernelEx(&cfg, spec_verify_kernel, a);
        if (e == cudaSuccess) e = cudaGetLastError();
        if (e != cudaSuccess) { set_error("nomos_attn_spec_verify: %s", cudaGetErrorString(e)); return NOMOS_ECUDA; }
    }
    return NOMOS_OK;
}

}  // namespace nomos
