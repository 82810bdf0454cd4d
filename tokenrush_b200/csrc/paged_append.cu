// Append of a step's K / V rows to a paged cache, with the heads' RMSNorm and the rotation of q and k on the way.
//
//   x' = x * rsqrt(mean x^2 + eps) * (1 + w)            (optional)
//   (a, b) -> (a cos - b sin, b cos + a sin) * amplitude     on pairs of the first rotary_dim dims, angle = position * inv_freq
//   q -> bf16;  k, v -> bf16 or (code = e4m3(x / s), s = max(amax, 1e-6) / 448)
//
// Bound by HBM bytes (every q, k, v element read once, written once), by latency for a handful of tokens.
// A CTA owns 32 (token, head) rows of one token at a time, eight warps with four rows each: the four rows of a
// warp are requested before anything else, and while they are on their way the CTA's threads compute the token's cos and
// sin into shared memory, once for all heads (computed per row they would cost more issue slots than the rows' own
// work).  The angle is reduced to a fraction of a turn in 64 bits: at position 2e6 an fp32 product is already off by 0.1 rad.
#include "paged.cuh"

namespace trb {

constexpr int PA_THREADS = 256, PA_RPW = 4, PA_ROWS = PA_THREADS / 32 * PA_RPW;

struct PagedAppendParams {
    PagedView c;
    BatchView b;
    const __nv_bfloat16 *q, *k, *v;
    __nv_bfloat16 *q_out;
    long long qrs, qhs, krs, khs, vrs, vhs;
    const __nv_bfloat16 *qw, *kw;
    const double *inv_freq;
    const int *cu;
    int n_rows, rows_per_seq, hq, rd, interleaved;
    float eps, amplitude;
    Cursor base;
};

template <int D>
__global__ void __launch_bounds__(PA_THREADS) paged_append_kernel(const PagedAppendParams p) {
    constexpr int EPT = D / 32;
    __shared__ float2 sm_cs[D / 2];
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = (p.q ? p.hq : 0) + 2 * p.c.hkv;                    // rows of a token: q heads, k heads, v heads
    const int row0 = blockIdx.y * PA_ROWS + warp * PA_RPW;
    pdl_wait();
    pdl_launch_dependents();

    __nv_bfloat16 raw[PA_RPW][EPT];
#pragma unroll
    for (int r = 0; r < PA_RPW; ++r) {
        int h = row0 + r;
        if (h < heads) {
            const __nv_bfloat16 *src;
            if (p.q && h < p.hq) src = p.q + t * p.qrs + h * p.qhs;
            else {
                h -= p.q ? p.hq : 0;
                src = h < p.c.hkv ? p.k + t * p.krs + h * p.khs : p.v + t * p.vrs + (h - p.c.hkv) * p.vhs;
            }
            if (EPT == 8) *reinterpret_cast<uint4 *>(raw[r]) = *reinterpret_cast<const uint4 *>(src + lane * EPT);
            else *reinterpret_cast<uint2 *>(raw[r]) = *reinterpret_cast<const uint2 *>(src + lane * EPT);
        }
    }
    // the token's sequence: cu is ascending, so it is the number of sequences that end at or before t
    int seq, i;
    if (p.cu) {
        int n = 0;
        for (int s0 = 0; s0 < p.b.n_seqs; s0 += PA_THREADS) {
            const int s = s0 + threadIdx.x;
            n += __syncthreads_count(s < p.b.n_seqs && p.cu[s + 1] <= t);
        }
        seq = n < p.b.n_seqs ? n : -1;
        i = seq >= 0 ? t - p.cu[seq] : 0;
    } else {
        seq = t / p.rows_per_seq;
        i = t - seq * p.rows_per_seq;
        if (seq >= p.b.n_seqs) seq = -1;
    }
    const long long len = seq >= 0 && i >= 0 ? load_len(p.b, seq) : -1;
    const bool live = len >= 0;
    const long long own = len + i;
    if (p.rd > 0 && live) {
        const long long pos = load_cursor(p.base) + own;
        for (int x = threadIdx.x; x < p.rd / 2; x += PA_THREADS) {
            const double turns = (double)pos * (p.inv_freq[x] * 0.15915494309189533577);      // 1 / (2 pi)
            float sn, cs;
            sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
            sm_cs[x] = make_float2(cs * p.amplitude, sn * p.amplitude);
        }
    }
    int page = -1;                                                       // of the pool, -1: no row is written
    if (live) {
        const long long slot = own >> p.c.page_shift;
        if (slot < p.b.table_pages) page = p.b.table[seq * p.b.table_stride + slot];
        if (page < 0 || page >= p.c.num_pages) {
            if (threadIdx.x == 0 && blockIdx.y == 0) raise_status(TRB_ST_CURSOR_RANGE);
            page = -1;
        }
    }
    const int in_page = (int)(own & ((1LL << p.c.page_shift) - 1));
    __syncthreads();

#pragma unroll
    for (int r = 0; r < PA_RPW; ++r) {
        int h = row0 + r;
        if (h >= heads) break;
        const bool is_q = p.q && h < p.hq;
        if (!is_q) h -= p.q ? p.hq : 0;
        const bool is_v = !is_q && h >= p.c.hkv;
        if (is_v) h -= p.c.hkv;
        float f[EPT];
#pragma unroll
        for (int e = 0; e < EPT; ++e) f[e] = __bfloat162float(raw[r][e]);
        if (!is_v) {
            const __nv_bfloat16 *w = is_q ? p.qw : p.kw;
            if (w) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < EPT; ++e) ss = fmaf(f[e], f[e], ss);
                const float inv = __frsqrt_rn(warp_sum(ss) * (1.0f / D) + p.eps);
                __nv_bfloat16 wb[EPT];
                if (EPT == 8) *reinterpret_cast<uint4 *>(wb) = *reinterpret_cast<const uint4 *>(w + lane * EPT);
                else *reinterpret_cast<uint2 *>(wb) = *reinterpret_cast<const uint2 *>(w + lane * EPT);
#pragma unroll
                for (int e = 0; e < EPT; ++e) f[e] = f[e] * inv * (1.0f + __bfloat162float(wb[e]));
            }
            if (p.rd > 0 && live) {
                if (p.interleaved) {
#pragma unroll
                    for (int e = 0; e < EPT; e += 2) {
                        const int dim = lane * EPT + e;
                        if (dim < p.rd) {
                            const float2 cs = sm_cs[dim >> 1];
                            const float a = f[e], b = f[e + 1];
                            f[e] = a * cs.x - b * cs.y;
                            f[e + 1] = b * cs.x + a * cs.y;
                        }
                    }
                } else {
                    // half is a multiple of EPT, so the partner of (lane, e) is (lane +- half / EPT, e)
                    const int half = p.rd / 2, hl = half / EPT;
                    const bool first = lane < hl;
                    const int partner = (first ? lane + hl : lane - hl) & 31;
#pragma unroll
                    for (int e = 0; e < EPT; ++e) {
                        const float o = __shfl_sync(0xffffffffu, f[e], partner);
                        const int dim = lane * EPT + e;
                        if (dim < p.rd) {
                            const float2 cs = sm_cs[first ? dim : dim - half];
                            f[e] = first ? f[e] * cs.x - o * cs.y : f[e] * cs.x + o * cs.y;
                        }
                    }
                }
            }
        }
        if (is_q || !p.c.ks) {
            __nv_bfloat16 ob[EPT];
#pragma unroll
            for (int e = 0; e < EPT; ++e) ob[e] = __float2bfloat16_rn(is_q && !live ? 0.f : f[e]);
            __nv_bfloat16 *dst = nullptr;
            if (is_q) dst = p.q_out + ((long long)t * p.hq + h) * D;
            else if (page >= 0) dst = (__nv_bfloat16 *)(is_v ? p.c.v : p.c.k) + ((((long long)page * p.c.hkv + h) << p.c.page_shift) + in_page) * D;
            if (dst) {
                if (EPT == 8) *reinterpret_cast<uint4 *>(dst + lane * EPT) = *reinterpret_cast<const uint4 *>(ob);
                else *reinterpret_cast<uint2 *>(dst + lane * EPT) = *reinterpret_cast<const uint2 *>(ob);
            }
        } else if (page >= 0) {
            const long long row = (((long long)page * p.c.hkv + h) << p.c.page_shift) + in_page;
            float amax = 0.f;
#pragma unroll
            for (int e = 0; e < EPT; ++e) amax = fmaxf(amax, fabsf(f[e]));
            amax = warp_max(amax);
            const float sc = __fdiv_rn(fmaxf(amax, 1e-6f), 448.0f);
            uint32_t w[EPT / 4];
#pragma unroll
            for (int x = 0; x < EPT / 4; ++x) {
                w[x] = 0;
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    w[x] |= (uint32_t)__nv_cvt_float_to_fp8(__fdiv_rn(f[x * 4 + b], sc), __NV_SATFINITE, __NV_E4M3) << (8 * b);
            }
            uint8_t *dst = (is_v ? p.c.v : p.c.k) + row * D + lane * EPT;
            if (EPT == 8) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t *>(dst) = w[0];
            if (lane == 0) (is_v ? p.c.vs : p.c.ks)[row] = sc;
        }
    }
}

}  // namespace trb

using namespace trb;

extern "C" int trb_paged_append(const trb_paged_t *pool, const trb_batch_t *batch, const trb_paged_append_args_t *a, trb_stream_t stream) {
    PagedAppendParams p;
    int rc = make_paged_view(pool, &p.c);
    if (rc || (rc = make_batch_view(batch, &p.b))) return rc;
    if (!a || !a->k || !a->v || a->n_rows < 0 || (rc = check_cursor(&a->base))) return rc ? rc : TRB_E_ARG;
    if (a->q && (!a->q_out || a->hq < 1)) return TRB_E_ARG;
    if (!a->cu && (a->rows_per_seq < 1 || (long long)a->rows_per_seq * batch->n_seqs != a->n_rows)) return TRB_E_ARG;
    if (a->rotary_dim < 0 || a->rotary_dim > pool->d || (a->rotary_dim & 1)) return TRB_E_UNSUPPORTED;
    if (a->rotary_dim > 0 && !a->inv_freq) return TRB_E_ARG;
    if (a->rotary_dim > 0 && !a->interleaved && a->rotary_dim % (2 * (pool->d / 32))) return TRB_E_UNSUPPORTED;
    const uintptr_t ptrs = (uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out | (uintptr_t)a->q_norm_w | (uintptr_t)a->k_norm_w;
    const int64_t strides = (a->q ? a->q_row_stride | a->q_head_stride : 0) | a->k_row_stride | a->k_head_stride | a->v_row_stride | a->v_head_stride;
    if ((ptrs & 15) || (strides & 7) || ((uintptr_t)a->cu & 3) || ((uintptr_t)a->inv_freq & 7)) return TRB_E_ALIGN;
    if (a->n_rows == 0) return TRB_OK;
    p.q = (const __nv_bfloat16 *)a->q; p.k = (const __nv_bfloat16 *)a->k; p.v = (const __nv_bfloat16 *)a->v; p.q_out = (__nv_bfloat16 *)a->q_out;
    p.qrs = a->q_row_stride; p.qhs = a->q_head_stride; p.krs = a->k_row_stride; p.khs = a->k_head_stride; p.vrs = a->v_row_stride; p.vhs = a->v_head_stride;
    p.qw = (const __nv_bfloat16 *)a->q_norm_w; p.kw = (const __nv_bfloat16 *)a->k_norm_w; p.inv_freq = a->inv_freq; p.cu = a->cu;
    p.n_rows = a->n_rows; p.rows_per_seq = a->rows_per_seq; p.hq = a->hq; p.rd = a->rotary_dim; p.interleaved = a->interleaved != 0;
    p.eps = a->eps; p.amplitude = a->amplitude; p.base = make_cursor(&a->base);
    const int heads = (a->q ? a->hq : 0) + 2 * p.c.hkv;
    cudaStream_t st = (cudaStream_t)stream;
    pdl_forget(st);
    TRB_CUDA_CHECK(launch_kernel(pool->d == 256 ? paged_append_kernel<256> : paged_append_kernel<128>,
                                 dim3(a->n_rows, (heads + PA_ROWS - 1) / PA_ROWS), dim3(PA_THREADS), 0, st, true, p));
    return TRB_OK;
}
