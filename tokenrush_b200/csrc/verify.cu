// Verification of drafted tokens by sampling (the batch's counterpart of the greedy commit in append.cu).
//
// Draft i (token x_i) stands while u_i q_i(x_i) < p_i(x_i).  The first draft that falls leaves the row p_i, q_i from
// whose residual max(p - q, 0) the new token is drawn; when all stand it is drawn from the row behind the last draft.
// The draw is the lowest index whose running sum exceeds u_k times the row's total, so the weights need no
// normalisation; products and sums are held in 64 bits (the two products compared are then exact, and a running sum of 2^18
// fp32 weights keeps its place next to a border).
//
// Bound by HBM: one row of p (and of q) per sequence.  One cluster of CTAs per sequence: each CTA sums its part of the
// row warp by warp, the warps' totals go to every CTA of the cluster through distributed shared memory, and the CTA
// whose warp's part holds the border goes over that part (now in L2) once more, in eight pieces and then one of them step by step.  No
// workspace, one launch.
#include <cooperative_groups.h>

#include "common.cuh"

namespace trb {

constexpr int SV_THREADS = 256, SV_WARPS = SV_THREADS / 32, SV_MAX_CLUSTER = 16, SV_MAX_K = 64;

struct SpecVerifyParams {
    const void *p, *q;
    long long pss, prs, qss, qrs;
    const long long *drafts;
    const float *u;
    const int *n_drafts;
    long long *tokens, *n_accepted;
    void *lens;
    int lens_width, k, vocab;
    int vec;                     // every row starts on a 16-byte boundary
};

template <typename T> __device__ __forceinline__ float sv_to_float(T x);
template <> __device__ __forceinline__ float sv_to_float<float>(float x) { return x; }
template <> __device__ __forceinline__ float sv_to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float sv_to_float<__half>(__half x) { return __half2float(x); }

// a probability as given; what is not positive and finite counts as zero
__device__ __forceinline__ float sv_clean(float x) { return x > 0.f && x <= 3.402823466e38f ? x : 0.f; }

// The weights of a row: max(p - q, 0), or p where there is nothing to take away, or p without the one certain draft.
template <typename T> struct SvRow {
    const T *p, *q;              // q nullptr: none
    long long without;           // index whose weight is zero (-1: none)
    __device__ __forceinline__ double at(int i, float pv, float qv) const {
        if (i == without) return 0.0;
        const double w = (double)sv_clean(pv) - (double)sv_clean(qv);
        return w > 0.0 ? w : 0.0;
    }
};

// One warp over elements [lo, hi) of a row in order; f(index of the lane's first element, its weights) for every step of
// 32 * PER elements.  With VEC a lane has 16 consecutive bytes, else PER single elements 32 apart.
template <typename T, bool VEC> struct SvStep {
    static constexpr int PER = VEC ? 16 / (int)sizeof(T) : 4;
    static constexpr int SPAN = 32 * PER;
};
template <typename T, bool VEC>
__device__ __forceinline__ void sv_load(const SvRow<T> &r, int base, int hi, int lane, double (&w)[SvStep<T, VEC>::PER]) {
    constexpr int PER = SvStep<T, VEC>::PER;
    T pv[PER], qv[PER];
    if constexpr (VEC) {
        const int i = base + lane * PER;
        const bool whole = i + PER <= hi;
        if (whole) {
            *reinterpret_cast<uint4 *>(pv) = *reinterpret_cast<const uint4 *>(r.p + i);
            if (r.q) *reinterpret_cast<uint4 *>(qv) = *reinterpret_cast<const uint4 *>(r.q + i);
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e)
                if (i + e < hi) { pv[e] = r.p[i + e]; if (r.q) qv[e] = r.q[i + e]; }
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) w[e] = i + e < hi ? r.at(i + e, sv_to_float(pv[e]), r.q ? sv_to_float(qv[e]) : 0.f) : 0.0;
    } else {
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int i = base + e * 32 + lane;
            if (i < hi) { pv[e] = r.p[i]; if (r.q) qv[e] = r.q[i]; }
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int i = base + e * 32 + lane;
            w[e] = i < hi ? r.at(i, sv_to_float(pv[e]), r.q ? sv_to_float(qv[e]) : 0.f) : 0.0;
        }
    }
}
__device__ __forceinline__ double sv_warp_sum(double x) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

// This lane's share of the weights in [lo, hi).  Whole steps, four at a time: p' = max(p, 0) and q' = min(max(q, 0), p') clear
// negative values and NaN, and p' - q' is the weight, exact enough in 64 bits; an infinity (which counts as zero) shows in the largest value seen, and
// the steps are then done again one by one.  So are the ones that hold the index without weight.
template <typename T, bool VEC>
__device__ __forceinline__ double sv_sum(const SvRow<T> &r, int lo, int hi, int lane) {
    constexpr int PER = SvStep<T, VEC>::PER, SPAN = SvStep<T, VEC>::SPAN, UNR = sizeof(T) == 2 && VEC ? 2 : 4;
    double s0 = 0.0, s1 = 0.0;
    int base = lo;
    while (base < hi) {
        if (base + UNR * SPAN <= hi && !(r.without >= base && r.without < base + UNR * SPAN)) {
            T pv[UNR][PER], qv[UNR][PER];
#pragma unroll
            for (int x = 0; x < UNR; ++x) {
                if constexpr (VEC) {
                    *reinterpret_cast<uint4 *>(pv[x]) = *reinterpret_cast<const uint4 *>(r.p + base + x * SPAN + lane * PER);
                    if (r.q) *reinterpret_cast<uint4 *>(qv[x]) = *reinterpret_cast<const uint4 *>(r.q + base + x * SPAN + lane * PER);
                } else {
#pragma unroll
                    for (int e = 0; e < PER; ++e) {
                        pv[x][e] = r.p[base + x * SPAN + e * 32 + lane];
                        if (r.q) qv[x][e] = r.q[base + x * SPAN + e * 32 + lane];
                    }
                }
            }
            double a0 = 0.0, a1 = 0.0;
            float top = 0.f;
#pragma unroll
            for (int x = 0; x < UNR; ++x)
#pragma unroll
                for (int e = 0; e < PER; e += 2) {
                    const float p0 = fmaxf(sv_to_float(pv[x][e]), 0.f), p1 = fmaxf(sv_to_float(pv[x][e + 1]), 0.f);
                    double w0 = (double)p0, w1 = (double)p1;
                    top = fmaxf(top, fmaxf(p0, p1));
                    if (r.q) {
                        const float q0 = fmaxf(sv_to_float(qv[x][e]), 0.f), q1 = fmaxf(sv_to_float(qv[x][e + 1]), 0.f);
                        top = fmaxf(top, fmaxf(q0, q1));
                        w0 -= (double)fminf(q0, p0);
                        w1 -= (double)fminf(q1, p1);
                    }
                    a0 += w0;
                    a1 += w1;
                }
            if (!__any_sync(0xffffffffu, !(top <= 3.402823466e38f))) {
                s0 += a0;
                s1 += a1;
                base += UNR * SPAN;
                continue;
            }
        }
        const int end = min(hi, base + UNR * SPAN);
        for (; base < end; base += SPAN) {
            double w[PER];
            sv_load<T, VEC>(r, base, hi, lane, w);
#pragma unroll
            for (int e = 0; e < PER; ++e) s0 += w[e];
        }
    }
    return s0 + s1;
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(SV_THREADS, 3) spec_verify_kernel(const SpecVerifyParams a) {
    namespace cg = cooperative_groups;
    constexpr int PER = SvStep<T, VEC>::PER, SPAN = SvStep<T, VEC>::SPAN;
    __shared__ double sm_tot[2][SV_MAX_CLUSTER * SV_WARPS];             // totals of every warp of the cluster, in row order
    __shared__ double sm_piece[SV_WARPS];
    __shared__ int sm_n;
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int b = blockIdx.x / ranks, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    cluster.barrier_arrive();                                           // (remote shared memory may be written once every CTA has started)
    pdl_wait();
    pdl_launch_dependents();
    int nd = a.n_drafts ? a.n_drafts[b] : a.k;
    const bool used = nd >= 0;
    nd = nd > a.k ? a.k : nd;
    const T *p0 = (const T *)a.p + b * a.pss, *q0 = a.q ? (const T *)a.q + b * a.qss : nullptr;
    const long long *drafts = a.drafts + (long long)b * a.k;
    const float *u = a.u + (long long)b * (a.k + 1);

    // ---- the first draft that falls (every CTA of the cluster finds it itself)
    if (warp == 0) {
        int n = nd < 0 ? 0 : nd;
        for (int i0 = 0; i0 < nd; i0 += 32) {
            const int i = i0 + lane;
            bool falls = false;
            if (i < nd) {
                const long long x = drafts[i];
                falls = true;
                if (x >= 0 && x < a.vocab) {
                    const float pv = sv_clean(sv_to_float(p0[i * a.prs + x]));
                    const float qv = q0 ? sv_clean(sv_to_float(q0[i * a.qrs + x])) : 1.f;
                    falls = !((double)u[i] * (double)qv < (double)pv);
                }
            }
            const unsigned int f = __ballot_sync(0xffffffffu, falls);
            if (f) { n = i0 + __ffs(f) - 1; break; }
        }
        if (lane == 0) sm_n = n;
    }
    __syncthreads();
    const int n = sm_n;
    const bool fell = used && n < nd;

    // ---- sums: warp w of rank r has the (r * SV_WARPS + w)-th of ranks * SV_WARPS equal parts, in whole steps
    const int parts = ranks * SV_WARPS, part = rank * SV_WARPS + warp;
    const int steps = (a.vocab + SPAN - 1) / SPAN;
    const int lo = (int)((long long)part * steps / parts) * SPAN, hi = min(a.vocab, (int)((long long)(part + 1) * steps / parts) * SPAN);
    SvRow<T> row;
    row.p = p0 + n * a.prs;
    row.q = fell && q0 ? q0 + n * a.qrs : nullptr;
    row.without = fell && !q0 ? drafts[n] : -1;
    double total = 0.0, tot[SV_MAX_CLUSTER / 4], inc = 0.0;             // this lane's run of parts, and the sum before it
    const int run_len = (parts + 31) / 32;                              // parts per lane
    cluster.barrier_wait();
    if (used) {
        for (int round = 0; round < 2; ++round) {                       // a second one only where the residual has no mass
            const double s = sv_warp_sum(sv_sum<T, VEC>(row, lo, hi, lane));
            if (lane < ranks) *cluster.map_shared_rank(&sm_tot[round][part], lane) = s;
            cluster.sync();
            double own = 0.0;
#pragma unroll
            for (int e = 0; e < SV_MAX_CLUSTER / 4; ++e) {
                tot[e] = e < run_len && lane * run_len + e < parts ? sm_tot[round][lane * run_len + e] : 0.0;
                own += tot[e];
            }
            inc = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { const double v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
            total = __shfl_sync(0xffffffffu, inc, 31);
            inc -= own;                                                 // now the sum before this lane's parts
            if (total > 0.0 || !fell) break;
            row.q = nullptr;
            row.without = -1;
        }
    }
    // ---- the border
    long long token = -1;
    bool mine = false;                                                  // this warp holds the answer
    if (used && total > 0.0) {
        const double border = (double)u[a.k] * total;
        int hit = -1, some = -1;                                        // the part that passes the border; the last part with mass
        double hit_start = 0.0, some_start = 0.0;
#pragma unroll
        for (int e = 0; e < SV_MAX_CLUSTER / 4; ++e) {
            if (tot[e] > 0.0) {
                some = lane * run_len + e;
                some_start = inc;
                if (hit < 0 && inc + tot[e] > border) { hit = some; hit_start = inc; }
            }
            inc += tot[e];
        }
        const unsigned int hits = __ballot_sync(0xffffffffu, hit >= 0), with_mass = __ballot_sync(0xffffffffu, some >= 0);
        const int src = hits ? __ffs(hits) - 1 : 31 - __clz(with_mass); // none passes it: a number of 1 or more, or not a number
        const int at = __shfl_sync(0xffffffffu, hits ? hit : some, src);
        const double start = __shfl_sync(0xffffffffu, hits ? hit_start : some_start, src);
        // the CTA that holds the part goes over it once more, first in eight pieces
        if (at / SV_WARPS != rank) return;
        const int a_lo = (int)((long long)at * steps / parts), a_n = (int)((long long)(at + 1) * steps / parts) - a_lo;
        const int b_lo = (a_lo + warp * a_n / SV_WARPS) * SPAN, b_hi = min(a.vocab, (a_lo + (warp + 1) * a_n / SV_WARPS) * SPAN);
        const double s = sv_warp_sum(sv_sum<T, VEC>(row, b_lo, b_hi, lane));
        if (lane == 0) sm_piece[warp] = s;
        __syncthreads();
        double before = start, run = start;
        int owner = -1, last_owner = 0;
#pragma unroll
        for (int x = 0; x < SV_WARPS; ++x) {
            const double v = sm_piece[x];
            if (v > 0.0) {
                if (owner < 0 && before + v > border) { owner = x; run = before; }
                if (owner < 0) { last_owner = x; some_start = before; }
            }
            before += v;
        }
        if (owner < 0) { owner = last_owner; run = some_start; }        // (sums in another order: the border lies behind the last piece with mass)
        mine = owner == warp;
        if (mine) {
            int found = -1, last = -1;
            for (int base = b_lo; base < b_hi && found < 0; base += SPAN) {
                double w[PER];
                sv_load<T, VEC>(row, base, b_hi, lane, w);
                // running sums in index order: VEC lanes hold consecutive elements, else every 32 are a turn
                constexpr int TURNS = VEC ? 1 : PER, EACH = VEC ? PER : 1;
#pragma unroll
                for (int turn = 0; turn < TURNS; ++turn) {
                    double mine_sum = 0.0;
#pragma unroll
                    for (int e = 0; e < EACH; ++e) mine_sum += w[turn * EACH + e];
                    double inc = mine_sum;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) { const double v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
                    double c = run + (inc - mine_sum);
                    int hit = -1, with = -1;
#pragma unroll
                    for (int e = 0; e < EACH; ++e) {
                        const double v = w[turn * EACH + e];
                        c += v;
                        if (v > 0.0) {
                            const int idx = VEC ? base + lane * PER + e : base + turn * 32 + lane;
                            with = idx;
                            if (hit < 0 && c > border) hit = idx;
                        }
                    }
                    run += __shfl_sync(0xffffffffu, inc, 31);
                    const unsigned int f = __ballot_sync(0xffffffffu, hit >= 0);
                    if (f && found < 0) found = __shfl_sync(0xffffffffu, hit, __ffs(f) - 1);
                    const unsigned int m = __ballot_sync(0xffffffffu, with >= 0);
                    if (m) last = __shfl_sync(0xffffffffu, with, 31 - __clz(m));
                }
            }
            token = found >= 0 ? found : last;
        }
    } else {
        mine = part == 0;
    }
    if (mine) {
        const int count = used ? n : 0;
        for (int i = lane; i <= a.k; i += 32) a.tokens[(long long)b * (a.k + 1) + i] = used && i < count ? drafts[i] : used && i == count ? token : -1;
        if (lane == 0) {
            a.n_accepted[b] = count;
            if (a.lens && used) {
                if (a.lens_width == 4) { int *d = (int *)a.lens + b; if (*d >= 0) *d += count + 1; }
                else { long long *d = (long long *)a.lens + b; if (*d >= 0) *d += count + 1; }
            }
        }
    }
}

template <typename T>
static cudaError_t launch_verify(const SpecVerifyParams &p, int n_seqs, int ranks, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)n_seqs * ranks); cfg.blockDim = dim3(SV_THREADS); cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    if (ranks > 8) {                                                    // beyond the portable cluster size
        static bool attr_set[64] = {};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e == cudaSuccess && !attr_set[dev & 63]) {
            e = cudaFuncSetAttribute(spec_verify_kernel<T, true>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(spec_verify_kernel<T, false>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
            attr_set[dev & 63] = e == cudaSuccess;
        }
        if (e != cudaSuccess) return e;
    }
    note_launch();
    return p.vec ? cudaLaunchKernelEx(&cfg, spec_verify_kernel<T, true>, p) : cudaLaunchKernelEx(&cfg, spec_verify_kernel<T, false>, p);
}

}  // namespace trb

using namespace trb;

extern "C" int trb_spec_verify(const trb_spec_verify_args_t *a, trb_stream_t stream) {
    if (!a || !a->probs || (!a->drafts && a->k > 0) || !a->u || !a->tokens || !a->n_accepted || a->n_seqs < 1 || a->k < 0 || a->vocab < 1) return TRB_E_ARG;
    if (a->dtype != TRB_DT_F32 && a->dtype != TRB_DT_BF16 && a->dtype != TRB_DT_F16) return TRB_E_ARG;
    if (a->lens && a->lens_width != 4 && a->lens_width != 8) return TRB_E_ARG;
    if (a->k > SV_MAX_K || a->vocab > (1 << 30) || a->n_seqs > (1 << 24)) return TRB_E_UNSUPPORTED;
    const int size = a->dtype == TRB_DT_F32 ? 4 : 2;
    if (((uintptr_t)a->probs | (uintptr_t)a->draft_probs) & (size - 1)) return TRB_E_ALIGN;
    if ((((uintptr_t)a->drafts | (uintptr_t)a->tokens | (uintptr_t)a->n_accepted) & 7) || (((uintptr_t)a->u | (uintptr_t)a->n_drafts) & 3)) return TRB_E_ALIGN;
    if (a->lens && ((uintptr_t)a->lens & (a->lens_width - 1))) return TRB_E_ALIGN;
    SpecVerifyParams p;
    p.p = a->probs; p.q = a->draft_probs;
    p.pss = a->probs_seq_stride; p.prs = a->probs_row_stride; p.qss = a->draft_seq_stride; p.qrs = a->draft_row_stride;
    p.drafts = (const long long *)a->drafts; p.u = a->u; p.n_drafts = a->n_drafts;
    p.tokens = (long long *)a->tokens; p.n_accepted = (long long *)a->n_accepted;
    p.lens = a->lens; p.lens_width = a->lens_width; p.k = a->k; p.vocab = a->vocab;
    const int64_t strides = a->probs_seq_stride | a->probs_row_stride | (a->draft_probs ? a->draft_seq_stride | a->draft_row_stride : 0);
    p.vec = (((uintptr_t)a->probs | (uintptr_t)a->draft_probs) & 15) == 0 && (strides * size) % 16 == 0;
    // As many CTAs per row as let all rows run in one wave of three per SM, while a warp's part has half a step of 512 bytes.  (192 rows of
    // 250000: 2 CTAs each; with 8, 3.5 waves paid the chain draft -> row -> sums -> border one after another.)  Clusters of 16, the largest, only
    // while they leave SMs free: 24 of them do not fit the GPCs at once (24 rows of 16000: 11.0 us, with 8 CTAs 6.9).
    const int steps = (a->vocab + 4096 / size - 1) / (4096 / size), most = (long long)a->n_seqs * 16 <= sm_count() ? 16 : 8;
    int ranks = std::max(1, std::min(std::min(3 * sm_count() / a->n_seqs, most), 2 * steps));
    if (ranks > 8 && ranks < 16) ranks = 8;                               // (beyond 8 only 16: the size the device is asked for)
    cudaStream_t st = (cudaStream_t)stream;
    pdl_forget(st);
    if (a->dtype == TRB_DT_F32) TRB_CUDA_CHECK(launch_verify<float>(p, a->n_seqs, ranks, st));
    else if (a->dtype == TRB_DT_BF16) TRB_CUDA_CHECK(launch_verify<__nv_bfloat16>(p, a->n_seqs, ranks, st));
    else TRB_CUDA_CHECK(launch_verify<__half>(p, a->n_seqs, ranks, st));
    return TRB_OK;
}
