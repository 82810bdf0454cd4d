// Append of a step's K / V rows to a paged cache, with the heads' RMSNorm and the rotation of q and k on the way.
//
//   x' = x * rsqrt(mean x^2 + eps) * (1 + w)            (optional)
//   (a, b) -> (a cos - b sin, b cos + a sin) * amplitude     on pairs of the first rotary_dim dims, angle = position * inv_freq
//   q -> bf16;  k, v -> bf16 or (code = e4m3(x / s), s = max(amax, 1e-6) / 448)
//
// Bound by HBM bytes (every q, k, v element read once, written once) once the work per row is small, by latency for a handful of tokens.
// Norm gain and rotation of a token are folded into two factors per dim, out = inv_rms (x A + partner(x) B), which a CTA computes once
// per token in shared memory for all heads; a row then costs a warp one 16-byte load per lane, the sum of squares, one exchange with the
// partner lanes (of bf16 pairs, before they are unpacked) and two packed multiply-adds per dim pair.  Issue slots are what the kernel
// is short of next to HBM, so nothing is computed per row that a token or a head shares.
// Many tokens: four per CTA and four heads per warp, the four tokens' rows of the next head requested while this head's are finished;
// the chain sequence -> length -> page is then walked once for four tokens.  Few tokens: one, and one head per warp.
// The angle is reduced to a fraction of a turn in 64 bits: at position 2e6 an fp32 product is already off by 0.1 rad.
#include "paged.cuh"

namespace trb {

constexpr int PA_THREADS = 256, PA_WARPS = PA_THREADS / 32;

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

// RN(x / b) for y = RN(1 / b): q = x y is within an ulp, its residual is exact in one fma, and q + r y rounds correctly (Markstein, IBM
// J. Res. Dev. 34, 1990).  Here b >= 2e-9 and |x / b| <= 448.00003; a residual that underflows belongs to a quotient far below e4m3's smallest code.
__device__ __forceinline__ float div_by(float x, float b, float y) {
    const float q = x * y;
    return fmaf(fmaf(-q, b, x), y, q);
}

template <int N> __device__ __forceinline__ void load_bf16(const __nv_bfloat16 *src, uint32_t (&w)[N / 2]) {
    if constexpr (N == 8) { const uint4 v = *reinterpret_cast<const uint4 *>(src); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else { const uint2 v = *reinterpret_cast<const uint2 *>(src); w[0] = v.x; w[1] = v.y; }
}
__device__ __forceinline__ float2 unpack_bf16x2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

template <int D, int TPC, int RPW>
__global__ void __launch_bounds__(PA_THREADS, 3) paged_append_kernel(const PagedAppendParams p) {
    constexpr int EPT = D / 32, W = EPT / 2, F4 = EPT / 4;
    __shared__ float4 sm_a[TPC][2][F4][32], sm_b[TPC][2][F4][32];        // factors of token, kind (q, k), piece of four dims, lane
    __shared__ long long sm_own[TPC];                                    // own row, -1: the token writes no cache row
    __shared__ int sm_page[TPC];
    const int t0 = blockIdx.x * TPC, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int hq = p.q ? p.hq : 0, heads = hq + 2 * p.c.hkv;             // rows of a token: q heads, k heads, v heads
    const int h0 = (blockIdx.y * PA_WARPS + warp) * RPW;
    pdl_wait();
    pdl_launch_dependents();

    uint32_t raw[TPC][W];
    auto request = [&](int h) {                                          // head h of the CTA's tokens
        const __nv_bfloat16 *src;
        long long step;
        if (h < hq) { src = p.q + h * p.qhs; step = p.qrs; }
        else if (h < hq + p.c.hkv) { src = p.k + (h - hq) * p.khs; step = p.krs; }
        else { src = p.v + (h - hq - p.c.hkv) * p.vhs; step = p.vrs; }
        src += t0 * step + lane * EPT;
#pragma unroll
        for (int tk = 0; tk < TPC; ++tk)
            if (h < heads && t0 + tk < p.n_rows) load_bf16<EPT>(src + tk * step, raw[tk]);
    };
    request(h0);

    // ---- the tokens' sequences, own rows and pages
    int n_before[TPC];
    if (p.cu) {                                                          // cu is ascending: the sequence of t is the number that end at or before it
#pragma unroll
        for (int tk = 0; tk < TPC; ++tk) n_before[tk] = 0;
        for (int s0 = 0; s0 < p.b.n_seqs; s0 += PA_THREADS) {
            const int s = s0 + threadIdx.x;
            const int end = s < p.b.n_seqs ? p.cu[s + 1] : 0x7fffffff;
#pragma unroll
            for (int tk = 0; tk < TPC; ++tk) n_before[tk] += __syncthreads_count(end <= t0 + tk);
        }
    }
    if (threadIdx.x < TPC) {
        const int t = t0 + threadIdx.x;
        int seq, i = 0;
        if (p.cu) {
            seq = 0;
#pragma unroll
            for (int tk = 0; tk < TPC; ++tk) seq = tk == (int)threadIdx.x ? n_before[tk] : seq;
            if (seq < p.b.n_seqs) i = t - p.cu[seq];
        } else {
            seq = t / p.rows_per_seq;
            i = t - seq * p.rows_per_seq;
        }
        const long long len = t < p.n_rows && seq < p.b.n_seqs && i >= 0 ? load_len(p.b, seq) : -1;
        const long long own = len < 0 ? -1 : len + i, slot = own >> p.c.page_shift;
        int page = -1;
        if (own >= 0) {
            if (slot < p.b.table_pages) page = p.b.table[seq * p.b.table_stride + slot];
            if (page < 0 || page >= p.c.num_pages) {
                if (blockIdx.y == 0) raise_status(TRB_ST_CURSOR_RANGE);
                page = -1;
            }
        }
        sm_own[threadIdx.x] = own;
        sm_page[threadIdx.x] = page;
    }
    const int half = p.rd / 2;
    __syncthreads();
    // ---- the factors, a pair of dims (d, e) at a time: out_d = x_d g_d c - x_e g_e s, out_e = x_e g_e c + x_d g_d s
    for (int x = threadIdx.x; x < TPC * (D / 2); x += PA_THREADS) {
        const int tk = x / (D / 2), pair = x % (D / 2);
        float sn = 0.f, cs = 1.f;
        int d = 2 * pair, e = d + 1;
        if (pair < half) {
            const double pos = (double)(load_cursor(p.base) + sm_own[tk]);
            const double turns = pos * (p.inv_freq[pair] * 0.15915494309189533577);                  // 1 / (2 pi)
            sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
            cs *= p.amplitude;
            sn *= p.amplitude;
            if (!p.interleaved) { d = pair; e = pair + half; }
        }
        const int at_d = d / EPT, at_e = e / EPT;                        // lane; then piece and place in it
        const int f_d = d % EPT / 4, f_e = e % EPT / 4;
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            const __nv_bfloat16 *w = kind ? p.kw : p.qw;
            const float gd = w ? 1.f + __bfloat162float(w[d]) : 1.f, ge = w ? 1.f + __bfloat162float(w[e]) : 1.f;
            reinterpret_cast<float *>(&sm_a[tk][kind][f_d][at_d])[d & 3] = gd * cs;
            reinterpret_cast<float *>(&sm_b[tk][kind][f_d][at_d])[d & 3] = -ge * sn;
            reinterpret_cast<float *>(&sm_a[tk][kind][f_e][at_e])[e & 3] = ge * cs;
            reinterpret_cast<float *>(&sm_b[tk][kind][f_e][at_e])[e & 3] = gd * sn;
        }
    }
    __syncthreads();

    // the lane that holds the partners of this one's dims (half layout: rd is a multiple of 2 EPT, so it is one lane for all of them)
    const int hl = half / EPT;
    const int partner = (lane < hl ? lane + hl : lane - hl) & 31;
#pragma unroll 1
    for (int r = 0; r < RPW; ++r) {
        const int h_all = h0 + r;
        if (h_all >= heads) break;
        uint32_t now[TPC][W];
#pragma unroll
        for (int tk = 0; tk < TPC; ++tk)
#pragma unroll
            for (int e = 0; e < W; ++e) now[tk][e] = raw[tk][e];
        if (r + 1 < RPW) request(h_all + 1);
        const bool is_q = h_all < hq, is_v = h_all >= hq + p.c.hkv;
        const int h = is_q ? h_all : is_v ? h_all - hq - p.c.hkv : h_all - hq;
        const bool norm = (is_q ? p.qw : p.kw) != nullptr;
#pragma unroll
        for (int tk = 0; tk < TPC; ++tk) {
            const int t = t0 + tk;
            if (t >= p.n_rows) break;
            const int page = sm_page[tk];
            float2 f[W];
#pragma unroll
            for (int e = 0; e < W; ++e) f[e] = unpack_bf16x2(now[tk][e]);
            if (!is_v) {
                float inv = 1.f;
                if (norm) {
                    float2 ss = __fmul2_rn(f[0], f[0]);
#pragma unroll
                    for (int e = 1; e < W; ++e) ss = __ffma2_rn(f[e], f[e], ss);
                    inv = rsqrtf(fmaf(warp_sum(ss.x + ss.y), 1.0f / D, p.eps));
                }
                uint32_t o[W];
                if (p.interleaved) {
#pragma unroll
                    for (int e = 0; e < W; ++e) o[e] = lane * EPT + 2 * e < p.rd ? prmt(now[tk][e], 0, 0x1032) : 0u;
                } else {
#pragma unroll
                    for (int e = 0; e < W; ++e) {
                        o[e] = __shfl_sync(0xffffffffu, now[tk][e], partner);
                        o[e] = lane * EPT < p.rd ? o[e] : 0u;            // (another dim times zero would still carry an infinity)
                    }
                }
                const float2 inv2 = make_float2(inv, inv);
#pragma unroll
                for (int x = 0; x < F4; ++x) {
                    const float4 fa = sm_a[tk][is_q ? 0 : 1][x][lane], fb = sm_b[tk][is_q ? 0 : 1][x][lane];
                    f[2 * x] = __fmul2_rn(__ffma2_rn(f[2 * x], make_float2(fa.x, fa.y), __fmul2_rn(unpack_bf16x2(o[2 * x]), make_float2(fb.x, fb.y))), inv2);
                    f[2 * x + 1] = __fmul2_rn(__ffma2_rn(f[2 * x + 1], make_float2(fa.z, fa.w), __fmul2_rn(unpack_bf16x2(o[2 * x + 1]), make_float2(fb.z, fb.w))), inv2);
                }
            }
            if (is_q || !p.c.ks) {
                const bool zero = is_q && sm_own[tk] < 0;
                uint32_t ob[W];
#pragma unroll
                for (int e = 0; e < W; ++e) ob[e] = zero ? 0u : pack_bf16x2(f[e].x, f[e].y);
                __nv_bfloat16 *dst = nullptr;
                if (is_q) dst = p.q_out + ((long long)t * p.hq + h) * D;
                else if (page >= 0) {
                    const int in_page = (int)(sm_own[tk] & ((1LL << p.c.page_shift) - 1));
                    dst = (__nv_bfloat16 *)(is_v ? p.c.v : p.c.k) + ((((long long)page * p.c.hkv + h) << p.c.page_shift) + in_page) * D;
                }
                if (dst) {
                    if constexpr (EPT == 8) *reinterpret_cast<uint4 *>(dst + lane * EPT) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
                    else *reinterpret_cast<uint2 *>(dst + lane * EPT) = make_uint2(ob[0], ob[1]);
                }
            } else if (page >= 0) {
                const int in_page = (int)(sm_own[tk] & ((1LL << p.c.page_shift) - 1));
                const long long row = (((long long)page * p.c.hkv + h) << p.c.page_shift) + in_page;
                float amax = 0.f;
#pragma unroll
                for (int e = 0; e < W; ++e) amax = fmaxf(amax, fmaxf(fabsf(f[e].x), fabsf(f[e].y)));
                amax = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(amax)));       // not negative: ordered as their bits
                const float sc = __fdiv_rn(fmaxf(amax, 1e-6f), 448.0f), rcp = __frcp_rn(sc);
                uint32_t w[F4];
#pragma unroll
                for (int x = 0; x < F4; ++x) {
                    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(div_by(f[2 * x].x, sc, rcp), div_by(f[2 * x].y, sc, rcp)), __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(div_by(f[2 * x + 1].x, sc, rcp), div_by(f[2 * x + 1].y, sc, rcp)), __NV_SATFINITE, __NV_E4M3);
                    w[x] = lo | hi << 16;
                }
                uint8_t *dst = (is_v ? p.c.v : p.c.k) + row * D + lane * EPT;
                if constexpr (EPT == 8) *reinterpret_cast<uint2 *>(dst) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t *>(dst) = w[0];
                if (lane == 0) (is_v ? p.c.vs : p.c.ks)[row] = sc;
            }
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
    // four tokens per CTA and four heads per warp once that still gives every SM several CTAs
    const bool many = (long long)(a->n_rows / 4) * ((heads + 31) / 32) >= 4LL * sm_count();
    const int tpc = many ? 4 : 1, rows = PA_WARPS * (many ? 4 : 1);
    cudaStream_t st = (cudaStream_t)stream;
    pdl_forget(st);
    TRB_CUDA_CHECK(launch_kernel(pool->d == 256 ? (many ? paged_append_kernel<256, 4, 4> : paged_append_kernel<256, 1, 1>)
                                                : (many ? paged_append_kernel<128, 4, 4> : paged_append_kernel<128, 1, 1>),
                                 dim3((a->n_rows + tpc - 1) / tpc, (heads + rows - 1) / rows), dim3(PA_THREADS), 0, st, true, p));
    return TRB_OK;
}
