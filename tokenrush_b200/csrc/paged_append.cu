// Append of a step's K / V rows to a paged cache, with the heads' RMSNorm and the rotation of q and k on the way.
//
//   x' = x * rsqrt(mean x^2 + eps) * (1 + w)            (optional)
//   (a, b) -> (a cos - b sin, b cos + a sin) * amplitude     on pairs of the first rotary_dim dims, angle = position * inv_freq
//   q -> bf16;  k, v -> bf16 or (code = e4m3(x / s), s = max(amax, 1e-6) / 448)
//
// Bound by HBM bytes (every q, k, v element read once, written once) once the work per row is small, by latency for a handful of tokens.
// Norm gain and rotation of a token are folded into two factors per dim, out = inv_rms (x A + partner(x) B), which a CTA computes once
// per token in shared memory for all heads.  Issue slots are what the kernel is short of next to HBM (a warp per row took 175
// instructions a row and 66 us for 7472 tokens of 24 + 4 + 4 heads, 36 us at copy rate), so a row is held by D / 16 lanes, two
// 16-byte chunks each, half a row apart: one stream of instructions serves 2 (256 dims) or 4 rows, sums take fewer exchanges, the upper half
// of a row needs no partner when at most half the head is rotated, and a fully rotated head finds its partners in the same lane.
// Before its first row a CTA walks a chain of latencies (sequence -> length -> page, angles, factors), so many small ones are resident: two tokens
// and four warps each, eight CTAs per SM (with four tokens and eight warps, three per SM, 7472 tokens took 59 us, now 50).  Few tokens: one per CTA, one
// round of heads.
// The angle is reduced to a fraction of a turn in 64 bits: at position 2e6 an fp32 product is already off by 0.1 rad.
#include "paged.cuh"

namespace trb {

constexpr int PA_THREADS = 128, PA_WARPS = PA_THREADS / 32;

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

__device__ __forceinline__ float2 unpack_bf16x2(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

template <int D, int TPC, int R>
__global__ void __launch_bounds__(PA_THREADS, 8) paged_append_kernel(const PagedAppendParams p) {
    constexpr int LPR = D / 16, RPI = 32 / LPR;                          // lanes of a row, rows (heads) of a warp
    __shared__ float4 sm_a[2 * TPC + 1][4][LPR], sm_b[2 * TPC + 1][4][LPR];    // factors of (token, q or k) and of v; piece of four dims (chunk 0: 0, 1; chunk 1: 2, 3); lane
    __shared__ long long sm_own[TPC];                                    // own row, -1: the token writes no cache row
    __shared__ int sm_page[TPC];
    const int t0 = blockIdx.x * TPC, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LPR;
    const int hq = p.q ? p.hq : 0, heads = hq + 2 * p.c.hkv;             // rows of a token: q heads, k heads, v heads
    const int h0 = (blockIdx.y * PA_WARPS + warp) * R * RPI + lane / LPR;
    pdl_wait();
    pdl_launch_dependents();

    uint4 raw[TPC][2];
    auto request = [&](int h) {                                          // head h of the CTA's tokens (beyond the last: the last, not stored)
        h = min(h, heads - 1);
        const bool of_q = h < hq, of_k = h < hq + p.c.hkv;
        const __nv_bfloat16 *src = of_q ? p.q + h * p.qhs : of_k ? p.k + (h - hq) * p.khs : p.v + (h - hq - p.c.hkv) * p.vhs;
        const long long step = of_q ? p.qrs : of_k ? p.krs : p.vrs;
        src += t0 * step + l * 8;
#pragma unroll
        for (int tk = 0; tk < TPC; ++tk) {
#pragma unroll
            for (int c = 0; c < 2; ++c) raw[tk][c] = *reinterpret_cast<const uint4 *>(src + c * (D / 2));
            if (t0 + tk + 1 < p.n_rows) src += step;
        }
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
    // ---- the factors, a pair of dims (d, e) per thread and token, its gains loaded once: out_d = x_d g_d c - x_e g_e s, out_e = x_e g_e c + x_d g_d s
    constexpr int PAIRS = D / 2, GROUPS = PA_THREADS / PAIRS;
    static_assert(PA_THREADS % PAIRS == 0, "a thread per pair");
    const int half = p.rd / 2, pair = threadIdx.x % PAIRS;
    const bool turn = pair < half;
    const int d = turn && !p.interleaved ? pair : 2 * pair, e = turn && !p.interleaved ? pair + half : d + 1;
    float gain[2][2];                                                    // q, k; d, e
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
        const __nv_bfloat16 *w = kind ? p.kw : p.qw;
        gain[kind][0] = w ? 1.f + __bfloat162float(w[d]) : 1.f;
        gain[kind][1] = w ? 1.f + __bfloat162float(w[e]) : 1.f;
    }
    const double freq = turn ? p.inv_freq[pair] * 0.15915494309189533577 : 0.0;        // 1 / (2 pi)
    const long long base = p.rd > 0 ? load_cursor(p.base) : 0;
    auto put = [&](int at, int dim, float fa, float fb) {                // chunk dim / (D / 2) of lane dim % (D / 2) / 8
        const int in = dim % (D / 2), piece = dim / (D / 2) * 2 + in % 8 / 4;
        reinterpret_cast<float *>(&sm_a[at][piece][in / 8])[dim & 3] = fa;
        reinterpret_cast<float *>(&sm_b[at][piece][in / 8])[dim & 3] = fb;
    };
    if (threadIdx.x < PAIRS) {                                           // -0: x * 1 + 0 * -0 is x, a negative zero too
        put(2 * TPC, d, 1.f, -0.f);
        put(2 * TPC, e, 1.f, -0.f);
    }
    __syncthreads();
    for (int tk = threadIdx.x / PAIRS; tk < TPC; tk += GROUPS) {
        float sn = -0.f, cs = 1.f;
        if (turn) {
            const double turns = (double)(base + sm_own[tk]) * freq;
            sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
            cs *= p.amplitude;
            sn *= p.amplitude;
        }
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
            put(2 * tk + kind, d, gain[kind][0] * cs, turn ? -gain[kind][1] * sn : -0.f);
            put(2 * tk + kind, e, gain[kind][1] * cs, turn ? gain[kind][0] * sn : -0.f);
        }
    }
    __syncthreads();

    // Where a chunk's partners are (half layout): chunk number x = c * LPR + l, partner x + hl or x - hl.  rd is a multiple of 16, so a chunk is
    // rotated as a whole.
    const int half8 = p.rd / 16, rot8 = 2 * half8;                       // chunks of half the rotation, of all of it
    const int hl = half8;
    const bool same_set = rot8 <= LPR, in_lane = hl == LPR;
#pragma unroll 1
    for (int r = 0; r < R; ++r) {
        const int h_all = h0 + r * RPI;
        if (h_all - lane / LPR >= heads) break;                          // (the same for the whole warp)
        if (r > 0) request(h_all);
        const bool ok = h_all < heads, is_q = h_all < hq, is_v = h_all >= hq + p.c.hkv;
        const int h = is_q ? h_all : is_v ? h_all - hq - p.c.hkv : h_all - hq, kind = is_q ? 0 : is_v ? 2 : 1;
        const bool norm = !is_v && (is_q ? p.qw : p.kw) != nullptr;
        const bool any_norm = __any_sync(0xffffffffu, norm), any_rot = p.rd > 0 && __any_sync(0xffffffffu, !is_v);
        const bool codes = !is_q && p.c.ks != nullptr, any_codes = __any_sync(0xffffffffu, codes && ok);
#pragma unroll
        for (int tk = 0; tk < TPC; ++tk) {
            const int t = t0 + tk;
            if (t >= p.n_rows) break;
            const uint32_t x[8] = {raw[tk][0].x, raw[tk][0].y, raw[tk][0].z, raw[tk][0].w, raw[tk][1].x, raw[tk][1].y, raw[tk][1].z, raw[tk][1].w};
            float2 f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = unpack_bf16x2(x[e]);
            float inv = 1.f;
            if (any_norm) {
                float2 ss = __fmul2_rn(f[0], f[0]);
#pragma unroll
                for (int e = 1; e < 8; ++e) ss = __ffma2_rn(f[e], f[e], ss);
                float s = ss.x + ss.y;
#pragma unroll
                for (int o = LPR / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                inv = norm ? rsqrtf(fmaf(s, 1.0f / D, p.eps)) : 1.f;
            }
            // partners of the two chunks; zero where a dim has none (its factor is zero too, but zero times an infinity is not)
            uint32_t o[8];
            bool lower = any_rot, upper = any_rot && !(same_set && !p.interleaved);
            if (p.interleaved) upper = any_rot && p.rd > D / 2;
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = 0u;
            if (any_rot) {
                if (p.interleaved) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int dim = (e >> 2) * (D / 2) + l * 8 + (e & 3) * 2;
                        o[e] = !is_v && dim < p.rd ? prmt(x[e], 0, 0x1032) : 0u;
                    }
                } else if (in_lane) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) o[e] = is_v ? 0u : x[e ^ 4];
                } else if (same_set) {
                    const int from = (lane & ~(LPR - 1)) + ((l < hl ? l + hl : l - hl) & (LPR - 1));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[e] = __shfl_sync(0xffffffffu, x[e], from);
                        o[e] = !is_v && l < rot8 ? o[e] : 0u;
                    }
                } else {                                                 // between half the head and all of it: a chunk's partner may be in either set
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int at = c * LPR + l, to = at < hl ? at + hl : at - hl;
                        const int from = (lane & ~(LPR - 1)) + (to & (LPR - 1));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t a = __shfl_sync(0xffffffffu, x[e], from), b = __shfl_sync(0xffffffffu, x[4 + e], from);
                            o[c * 4 + e] = is_v || at >= rot8 ? 0u : to < LPR ? a : b;
                        }
                    }
                }
            }
            const float2 inv2 = make_float2(inv, inv);
            const int table = kind == 2 ? 2 * TPC : 2 * tk + kind;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const float4 fa = sm_a[table][y][l];
                float2 u = make_float2(-0.f, -0.f), v = u;
                if (y < 2 ? lower : upper) {
                    const float4 fb = sm_b[table][y][l];
                    u = __fmul2_rn(unpack_bf16x2(o[2 * y]), make_float2(fb.x, fb.y));
                    v = __fmul2_rn(unpack_bf16x2(o[2 * y + 1]), make_float2(fb.z, fb.w));
                }
                f[2 * y] = __fmul2_rn(__ffma2_rn(f[2 * y], make_float2(fa.x, fa.y), u), inv2);
                f[2 * y + 1] = __fmul2_rn(__ffma2_rn(f[2 * y + 1], make_float2(fa.z, fa.w), v), inv2);
            }
            const long long own = sm_own[tk];
            const int page = sm_page[tk];
            const long long row = (((long long)page * p.c.hkv + h) << p.c.page_shift) + (int)(own & ((1LL << p.c.page_shift) - 1));
            if (ok && !codes && (is_q || page >= 0)) {
                __nv_bfloat16 *dst = (is_q ? p.q_out + ((long long)t * p.hq + h) * D : (__nv_bfloat16 *)(is_v ? p.c.v : p.c.k) + row * D) + l * 8;
                const bool zero = is_q && own < 0;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t ob[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) ob[e] = zero ? 0u : pack_bf16x2(f[c * 4 + e].x, f[c * 4 + e].y);
                    *reinterpret_cast<uint4 *>(dst + c * (D / 2)) = make_uint4(ob[0], ob[1], ob[2], ob[3]);
                }
            }
            if (any_codes) {
                float amax = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fmaxf(fabsf(f[e].x), fabsf(f[e].y)));
#pragma unroll
                for (int s = LPR / 2; s > 0; s >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, s));
                if (codes && ok && page >= 0) {
                    const float sc = __fdiv_rn(fmaxf(amax, 1e-6f), 448.0f), rcp = __frcp_rn(sc);
                    uint8_t *dst = (is_v ? p.c.v : p.c.k) + row * D + l * 8;
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        uint32_t w[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float2 a = f[c * 4 + 2 * e], b = f[c * 4 + 2 * e + 1];
                            const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(div_by(a.x, sc, rcp), div_by(a.y, sc, rcp)), __NV_SATFINITE, __NV_E4M3);
                            const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(div_by(b.x, sc, rcp), div_by(b.y, sc, rcp)), __NV_SATFINITE, __NV_E4M3);
                            w[e] = lo | hi << 16;
                        }
                        *reinterpret_cast<uint2 *>(dst + c * (D / 2)) = make_uint2(w[0], w[1]);
                    }
                    if (l == 0) (is_v ? p.c.vs : p.c.ks)[row] = sc;
                }
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
    if (a->rotary_dim > 0 && !a->interleaved && a->rotary_dim % 16) return TRB_E_UNSUPPORTED;
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
    // two tokens per CTA and four rounds of heads per warp once that still gives every SM its eight CTAs
    const int rpi = 512 / pool->d;                                        // heads of a warp at a time
    const int wide = 4 * PA_WARPS * rpi;
    const bool many = (long long)(a->n_rows / 2) * ((heads + wide - 1) / wide) >= 8LL * sm_count();
    const int tpc = many ? 2 : 1, rows = many ? wide : PA_WARPS * rpi;
    cudaStream_t st = (cudaStream_t)stream;
    pdl_forget(st);
    TRB_CUDA_CHECK(launch_kernel(pool->d == 256 ? (many ? paged_append_kernel<256, 2, 4> : paged_append_kernel<256, 1, 1>)
                                                : (many ? paged_append_kernel<128, 2, 4> : paged_append_kernel<128, 1, 1>),
                                 dim3((a->n_rows + tpc - 1) / tpc, (heads + rows - 1) / rows), dim3(PA_THREADS), 0, st, true, p));
    return TRB_OK;
}
