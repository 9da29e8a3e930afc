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
#include <atomic>

#include "common.cuh"
#include "launch.h"

namespace nomos {

// 48 warps per SM, each with two 16-byte loads per lane and row in flight: 96 sequences x 262144 tokens take 33.7 us (two rows
// each: 6.0 TB/s); 54.9 with half the warps and twice the loads each, 36.4 with as many warps in CTAs of 256 threads.
constexpr int SV_THREADS = 512, SV_WARPS = SV_THREADS / 32, SV_CTAS_PER_SM = 3;
constexpr int SV_UNROLL = 2;

struct SpecVerifyArgs {
    const float *p, *q;                  // [batch][max_draft + 1][p_stride], [batch][max_draft][q_stride] or nullptr
    const int *tokens, *n_draft;
    const float *u_accept, *u_sample;
    const int *lens, *granted;           // granted: rows the step placed for the sequence, or nullptr
    int *lens_out, *n_accepted, *out_tokens;
    int batch, max_draft, vocab;
    long p_stride, q_stride;
};

// Adds the whole weight of max(p - q, 0) to a sum.  6 + (p - q) lies in [4, 8), whose doubles are 2^-50 apart: the addition
// rounds to whole units, and the bit pattern less that of 6.0 (whose low word is zero) is their number.  (A conversion to a
// 64-bit integer is slower.)  p above 1 counts as 1, and only then is compared: q may be above 1 as well, and a negative difference
// would wrap.  A NaN stays one through the minimum and compares false: it weighs nothing.
__device__ __forceinline__ void add_weight(unsigned long long &sum, float p, float q) {
    float pc;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(pc) : "f"(p), "f"(1.0f));
    const long long u = __double_as_longlong(__dadd_rn(__dsub_rn((double)pc, (double)q), 6.0));
    if (pc > q) sum += (unsigned long long)(u - 0x4018000000000000ll);
}

// One row's weights: target row, drafter row (nullptr: none), and the index whose drafter probability is 1 (a drafter that
// gives tokens only; -1: none).
struct RowWeights {
    const float *p, *q;
    int one;
    __device__ __forceinline__ unsigned long long at(int i) const {
        unsigned long long w = 0;
        add_weight(w, p[i], q ? q[i] : i == one ? 1.0f : 0.0f);
        return w;
    }
};

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Inclusive prefix sums over a warp.
__device__ __forceinline__ unsigned long long warp_prefix(unsigned long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Sum over [i0, i1) by one warp, where p + i0 is a 16-byte boundary: batches of 256 elements, every load of a batch in flight
// before the first weight.  Q: 0 no drafter row, 1 drafter row on the same boundary, 2 drafter row anywhere.
template <int Q>
__device__ __forceinline__ unsigned long long warp_range(const RowWeights &w, int i0, int i1, int lane) {
    constexpr int U = SV_UNROLL;
    unsigned long long s = 0;
    for (int i = i0 + 4 * lane; i < i1; i += 128 * U) {
        float4 pv[U], qv[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int j = i + 128 * k;
            pv[k] = qv[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (j + 4 <= i1) {
                pv[k] = __ldcs(reinterpret_cast<const float4 *>(w.p + j));
                if constexpr (Q == 1) qv[k] = __ldcs(reinterpret_cast<const float4 *>(w.q + j));
                if constexpr (Q == 2) qv[k] = make_float4(w.q[j], w.q[j + 1], w.q[j + 2], w.q[j + 3]);
            } else if (j < i1) {                                      // the one lane whose four elements the end cuts
                pv[k].x = w.p[j];
                if (j + 1 < i1) pv[k].y = w.p[j + 1];
                if (j + 2 < i1) pv[k].z = w.p[j + 2];
                if constexpr (Q != 0) {
                    qv[k].x = w.q[j];
                    if (j + 1 < i1) qv[k].y = w.q[j + 1];
                    if (j + 2 < i1) qv[k].z = w.q[j + 2];
                }
            }
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if constexpr (Q == 0) {
                const int d = w.one - (i + 128 * k);                  // (a drafted token's own place: its probability counts 1)
                if ((unsigned)d < 4u) {
                    qv[k].x = d == 0 ? 1.0f : 0.0f; qv[k].y = d == 1 ? 1.0f : 0.0f;
                    qv[k].z = d == 2 ? 1.0f : 0.0f; qv[k].w = d == 3 ? 1.0f : 0.0f;
                }
            }
            add_weight(s, pv[k].x, qv[k].x); add_weight(s, pv[k].y, qv[k].y);
            add_weight(s, pv[k].z, qv[k].z); add_weight(s, pv[k].w, qv[k].w);
        }
    }
    return warp_sum(s);
}

__global__ void __launch_bounds__(SV_THREADS, SV_CTAS_PER_SM) spec_verify_kernel(const __grid_constant__ SpecVerifyArgs a) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ unsigned long long s_warp[2][SV_WARPS], s_total[2], s_scan[SV_WARPS];
    __shared__ int s_accepted;
    __shared__ float s_u;                // (every register counts here: forty per thread, so that three CTAs share an SM)
    asm volatile("griddepcontrol.wait;\n" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int b = blockIdx.y, rank = blockIdx.x, C = gridDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // Drafts to look at (a draft whose row was not placed is none), and the rows that stay whatever becomes of them.
    const auto counts = [&](int &other) {
        const int k = min(a.n_draft ? a.n_draft[b] : a.max_draft, a.max_draft), rows = a.granted ? a.granted[b] : k + 1;
        const int m = rows > 0 ? min(k, rows - 1) : -1;
        other = rows - max(m, 0);
        return m;
    };
    int other;
    const int n = counts(other);
    if (threadIdx.x == SV_THREADS - 1) s_u = a.u_sample[b];
    if (n < 0) {                         // idle, or without pages: nothing of it is read or written; the whole cluster leaves
        if (a.granted && other > 0 && a.lens && rank == 0 && threadIdx.x == 0) a.lens_out[b] = a.lens[b] + other;   // part of a prompt
        return;
    }
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
    // stretch of this warp: [i0, i1) of the vocabulary, cut where the target row crosses 16-byte boundaries (`lead` elements
    // precede the first one; they belong to the first warp)
    const int lead = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(w.p) & 15)) & 15) / 4);
    const int per = ((a.vocab + C * SV_WARPS - 1) / (C * SV_WARPS) + 3) / 4 * 4;                 // (vocab <= 2^30: 32 bits hold it all)
    const auto cut = [&](int unit) { return unit == 0 ? 0 : min(unit * per + lead, a.vocab); };
    const int unit = rank * SV_WARPS + warp;
    const int i0 = cut(unit), i1 = unit == C * SV_WARPS - 1 ? a.vocab : cut(unit + 1);

#pragma unroll 1
    for (int round = 0; round < 2; ++round) {
        unsigned long long mine = 0;
        const int v0 = unit == 0 ? lead : i0;
        if (!w.q) mine = warp_range<0>(w, v0, i1, lane);
        else if (((reinterpret_cast<uintptr_t>(w.q + v0)) & 15) == 0) mine = warp_range<1>(w, v0, i1, lane);
        else mine = warp_range<2>(w, v0, i1, lane);
        if (unit == 0)
            for (int i = 0; i < lead; ++i) mine += w.at(i);
        if (lane == 0) s_warp[round][warp] = mine;
        __syncthreads();
        if (warp == 0) {
            const unsigned long long t = warp_sum(lane < SV_WARPS ? s_warp[round][lane] : 0);
            if (lane == 0) s_total[round] = t;
        }
        cluster.sync();
        // every warp fetches the CTAs' totals, a lane each: one trip through the cluster's shared memory
        const unsigned long long upto = warp_prefix(lane < C ? *cluster.map_shared_rank(&s_total[round], lane) : 0, lane);
        const unsigned long long total = __shfl_sync(0xffffffffu, upto, 31);
        const unsigned long long after = __shfl_sync(0xffffffffu, upto, rank), before = after - s_total[round];
        if (total == 0 && round == 0 && (w.q || w.one >= 0)) {
            // nothing is left of the target's row: the drafter covers it everywhere (equal rows and a drafted token of probability 0
            // in both, or one that is none), by less than 2^-51 at most, or u was outside [0, 1).  The target's own row decides
            w.q = nullptr; w.one = -1;
            continue;
        }
        if (total > 0) {
            const long long t0 = (long long)floor(__dmul_rn((double)s_u, (double)total));
            const unsigned long long T = (unsigned long long)max(0ll, min(t0, (long long)total - 1));
            if (T >= before && T < after) {                           // uniform over the CTA
                // the warp whose stretch holds T
                const unsigned long long mine_w = lane < SV_WARPS ? s_warp[round][lane] : 0, w_upto = before + warp_prefix(mine_w, lane);
                const int k = min(SV_WARPS - 1, __popc(__ballot_sync(0xffffffffu, lane < SV_WARPS && T >= w_upto)));
                unsigned long long base = __shfl_sync(0xffffffffu, w_upto - mine_w, k);
                // the k-th warp's stretch again, by the whole CTA: `each` neighbouring elements per thread
                const int u0 = rank * SV_WARPS + k;
                const int j0 = cut(u0), j1 = u0 == C * SV_WARPS - 1 ? a.vocab : cut(u0 + 1);
                const int each = (j1 - j0 + SV_THREADS - 1) / SV_THREADS;
                const int e0 = min(j1, j0 + (int)threadIdx.x * each), e1 = min(j1, e0 + each);
                unsigned long long s = 0;
                for (int i = e0; i < e1; ++i) s += w.at(i);
                const unsigned long long incl = warp_prefix(s, lane);
                if (lane == 31) s_scan[warp] = incl;
                __syncthreads();
                base += warp_sum(lane < warp ? s_scan[lane] : 0);
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
            if (a.lens) {                // (asked for again rather than kept in a register over the streams; before n_accepted, which
                counts(other);           // may lie over n_draft)
                a.lens_out[b] = a.lens[b] + other + acc;
            }
            a.n_accepted[b] = acc;
        }
    }
    cluster.sync();                      // the totals stay where the peers read them
}

int launch_spec_verify(cudaStream_t st, const float *p, const float *q, const int *tokens, const int *n_draft, const float *u_accept,
                       const float *u_sample, const int *lens, const int *granted, int *lens_out, int *n_accepted, int *out_tokens, int batch,
                       int max_draft, int vocab, long p_stride, long q_stride) {
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
    // As many CTAs per sequence as are resident at once, at most sixteen (eight where the driver does not allow that), and none
    // without a load per lane for each of its warps (sixteen: a whole batch; 16 sequences of 50001 tokens 7.0 us with 8, 8.7 with 16;
    // one of 32000 5.6 with 4, 5.2 with 8).  One sequence of 262144 tokens: 24.0 / 13.6 / 9.0 / 7.3 us with 2 / 4 /
    // 8 / 16; 96 sequences of 32000: 10.2 with 4, 10.5 with 2.
    int ctas = 16;
    while (ctas > 1 && ((long)ctas * std::min(batch, 65535) > 148 * SV_CTAS_PER_SM || vocab < ctas * SV_WARPS * 128 * (ctas > 8 ? SV_UNROLL : 1))) ctas /= 2;
    static std::atomic<uint64_t> large_clusters{0};                   // devices on which the attribute is set
    if (ctas == 16 && !(large_clusters.load(std::memory_order_relaxed) & device_bit())) {
        if (cudaFuncSetAttribute(spec_verify_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
            large_clusters.fetch_or(device_bit(), std::memory_order_relaxed);
        } else {
            cudaGetLastError();
            ctas = 8;
        }
    }
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(SV_THREADS); cfg.stream = st; cfg.attrs = attr; cfg.numAttrs = 2;
    for (int b0 = 0; b0 < batch; b0 += 65535) {                       // the grid's y dimension
        const int nb = std::min(65535, batch - b0);
        SpecVerifyArgs a{p + (size_t)b0 * (max_draft + 1) * p_stride, q ? q + (size_t)b0 * max_draft * q_stride : nullptr,
                         tokens + (size_t)b0 * max_draft, n_draft ? n_draft + b0 : nullptr, u_accept + (size_t)b0 * max_draft, u_sample + b0,
                         lens ? lens + b0 : nullptr, granted ? granted + b0 : nullptr, lens_out ? lens_out + b0 : nullptr, n_accepted + b0,
                         out_tokens + (size_t)b0 * (max_draft + 1), nb, max_draft, vocab, p_stride, q_stride};
        attr[1].val.clusterDim.x = ctas;
        cfg.gridDim = dim3(ctas, nb);
        cudaError_t e = cudaLaunchKernelEx(&cfg, spec_verify_kernel, a);
        if (e != cudaSuccess && ctas == 16) {                         // no sixteen SMs of one group to be had
            cudaGetLastError();
            ctas = 8;
            attr[1].val.clusterDim.x = ctas;
            cfg.gridDim = dim3(ctas, nb);
            e = cudaLaunchKernelEx(&cfg, spec_verify_kernel, a);
        }
        if (e == cudaSuccess) e = cudaGetLastError();
        if (e != cudaSuccess) { set_error("nomos_attn_spec_verify: %s", cudaGetErrorString(e)); return NOMOS_ECUDA; }
    }
    return NOMOS_OK;
}

}  // namespace nomos
