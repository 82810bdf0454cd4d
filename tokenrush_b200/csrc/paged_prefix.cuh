// The shared prefix of a batch, read once for all its query rows, on the 5th-generation tensor cores.
//
// All query rows of a kv head (n_seqs * m tokens * hq / hkv heads) see every prefix row, so they form one dense product:
// blocks of 128 query rows against the prefix, cut along the keys into `splits` pieces so that the CTAs fill the SMs; a piece
// leaves a (max, sum, acc) partial per query row that paged_merge_kernel joins with the pieces of the sequence's own rows.
// With one block of rows the kernel is bound by HBM even though the block may be mostly padding (a 128-key e4m3 tile is 64 KB,
// 1.5 us of an SM's share of HBM, and its MMAs take 1.1 us); with more it is bound by the tensor side.
//
// The tile loop is that of the prefill kernel (prefill.cu): S = Q K^T into two alternating tensor-memory buffers, softmax,
// P written over the scores it came from and taken from there as the A operand of O += P V.  The softmax pass of a tile is
// bound by dependency latency, so four warpgroups share it (thread = one query row and a quarter of the keys).  e4m3 codes feed kind::f8f6f4 MMAs unconverted, with q and P as hi + lo terms; bf16 pools
// feed kind::f16.  Different here: tiles are put together from pages (one TMA box per page and 128-byte column), there is no
// causal edge, and the rows of the last tile behind the prefix are cleared in shared memory before P V, because pages may hold
// anything there.
#pragma once
#include "paged.cuh"
#include "tc.cuh"
#include "tmap.h"

namespace trb {

struct PrefixParams {
    PagedView c;
    const __nv_bfloat16 *q;
    int n_seqs, m, hq, g;
    float scale_log2;
    const int *table;
    int pages;
    Cursor len;
    int splits, blocks;                // pieces of the key axis, blocks of 128 query rows
    float *part_ml;                    // [splits][hkv][rows][2]
    float *part_acc;                   // [splits][hkv][rows][D]
};

constexpr int PX_BM = 128, PX_WG = 4, PX_SOFTMAX = PX_WG * 128, PX_WARPS = PX_SOFTMAX / 32, PX_THREADS = PX_SOFTMAX + 64;

template <int D_, bool FP8_> struct PrefixCfg {
    static constexpr int D = D_;
    static constexpr bool FP8 = FP8_;
    static constexpr int BN = FP8 || D == 128 ? 128 : 64;              // keys per tile: S, P, O and Q share 512 tensor-memory columns
    static constexpr int ROWB = D * (FP8 ? 1 : 2), SEGS = ROWB / 128, TILE = BN * ROWB;
    static constexpr int STAGES = FP8 ? (D == 256 ? 2 : 4) : 3;
    static constexpr int SLOTS = STAGES + 1;                           // tables of per-key factors in use at once
    static constexpr int Q_BYTES = PX_BM * D;                          // one e4m3 copy of the query block
    static constexpr int OFF_KV = FP8 ? 2 * Q_BYTES : 0;
    static constexpr int OFF_SC = OFF_KV + STAGES * 2 * TILE;          // [SLOTS][2][BN] floats: scales as they lie in the pool
    static constexpr int OFF_FAC = OFF_SC + (FP8 ? SLOTS * 2 * BN * 4 : 0);   // [SLOTS][3][BN] floats: factors of a tile's keys
    static constexpr int OFF_MX = OFF_FAC + (FP8 ? SLOTS * 3 * BN * 4 : 0);   // [2][PX_WG][128] floats: row maxima of the four quarters
    static constexpr int OFF_BAR = OFF_MX + 2 * PX_WG * PX_BM * 4;
    static constexpr int SMEM = OFF_BAR + 256 + 1024;
    // Weights are staged as 2^(t - reference + LIFT), and a row's reference follows the largest score of a tile lazily.  bf16 weights keep 8 bits at any
    // size: the reference moves only when a score passes it by more than SLACK (a correction of O waits for the PV before it: 128 readers of
    // 65536 rows 265 -> 245 us).  e4m3 weights as hi + lo keep 8 bits down to 2^-10 of the reference and are off by up to 2^-18 of it below, so a
    // tail far under the largest weight would be lost whatever its mass: the reference also comes down, to within DROP bits of every
    // tile's own largest score.  What the small weights of a tile lose is then at most 128 * 2^-18 * 2^DROP = 2^-9 of its largest, however many keys there
    // are (one sink and 65535 keys 18.5 bits below, a piece over all of them: off by 23 % -> 0.4 %; 64 readers of 8192 rows 40.4 -> 40.6 us, 128 of 65536
    // rows 230 -> 239, 512 query rows of 32/8 x 128 heads 934 -> 1021).
    // It stops DEPTH bits under the row's largest score, where a tile is worth nothing and O (<= keys * 448 * 2^(LIFT + DEPTH)) still fits fp32.
    static constexpr float LIFT = FP8 ? 8.f : 0.f, SLACK = 8.f, DROP = 2.f, DEPTH = 40.f;
    static constexpr int TM_S = 0, TM_O = 256, TM_Q = FP8 ? 0 : (D == 256 ? 128 : 384);
    static_assert(SMEM <= 227 * 1024, "shared memory budget");
    static_assert(STAGES * 2 * TILE >= PX_BM * D * 4, "the output block is turned in the ring");
};

template <typename C>
__global__ void __launch_bounds__(PX_THREADS, 1)
paged_prefix_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PrefixParams p) {
    constexpr int D = C::D, BN = C::BN, KPT = BN / PX_WG, SEGS = C::SEGS, TILE = C::TILE, STAGES = C::STAGES, SLOTS = C::SLOTS;
    constexpr bool FP8 = C::FP8;
    extern __shared__ uint8_t px_smem_raw[];
    uint8_t *smem = px_smem_raw + ((1024u - (smem_u32(px_smem_raw) & 1023u)) & 1023u);
    float *sm_sc = reinterpret_cast<float *>(smem + C::OFF_SC);
    float *sm_fac = reinterpret_cast<float *>(smem + C::OFF_FAC);
    float *sm_mx = reinterpret_cast<float *>(smem + C::OFF_MX);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
    // K and V tiles have barriers of their own: a K tile is refilled as soon as its product has run
    uint64_t *k_full = bars, *v_full = k_full + STAGES, *k_free = v_full + STAGES, *v_free = k_free + STAGES;
    uint64_t *s_full = v_free + STAGES, *p_full = s_full + 2, *o_done = p_full + 2, *o_last = o_done + 1, *q_ready = o_last + 1, *mma_out = q_ready + 1, *v_clean = mma_out + 1, *fac_full = v_clean + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(fac_full + SLOTS);
    static_assert((4 * C::STAGES + 9 + C::SLOTS) * 8 + 4 <= 256, "barriers");

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = blockIdx.x % p.splits, blk = blockIdx.x / p.splits % p.blocks, j = blockIdx.x / p.splits / p.blocks;
    const int rows_seq = p.g * p.m, rows_all = p.n_seqs * rows_seq;    // query rows of a kv head
    const int q0 = blk * PX_BM;
    const int rows_here = min(PX_BM, rows_all - q0);
    // where the block's query rows lie (-1: no row); needs no memory, so it is done before the wait for the launches before this one
    long long *sm_off = reinterpret_cast<long long *>(sm_mx);          // [128]; read by all before the first tile's maxima are written here
    if (threadIdx.x < PX_BM) {
        const int rr = q0 + threadIdx.x, seq = rr / rows_seq, r = rr - seq * rows_seq, i = r / p.g;
        sm_off[threadIdx.x] = (int)threadIdx.x < rows_here ? (((long long)seq * p.m + i) * p.hq + j * p.g + r - i * p.g) * D : -1;
    }

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(&k_full[s], FP8 ? 33u : 1u); mbar_init(&v_full[s], 1u);      // e4m3: 32 lanes' scales come with the K tile
            mbar_init(&k_free[s], 1u); mbar_init(&v_free[s], 1u);
        }
        // P has a barrier per buffer: the softmax warps may finish tile i + 1 while the MMA warp still waits for V of tile i, and a second
        // phase of one barrier would hide the first from its parity
        for (int b = 0; b < 2; ++b) { mbar_init(&s_full[b], 1u); mbar_init(&p_full[b], PX_WARPS); }
        for (int b = 0; b < SLOTS; ++b) mbar_init(&fac_full[b], 1u);
        mbar_init(o_done, 1u); mbar_init(o_last, 1u); mbar_init(q_ready, PX_WARPS); mbar_init(mma_out, 1u); mbar_init(v_clean, 1u);
        mbar_fence_init();
        tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v);
    }
    if (warp == 0) { tmem_alloc(tmem_slot, 512); tmem_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_wait();
    pdl_launch_dependents();

    const int n_prefix = paged_prefix_rows(p.len, p.pages, p.c.page_shift, blockIdx.x == 0 && threadIdx.x == 0);
    const int all_tiles = (n_prefix + BN - 1) / BN;
    const int t0 = (int)((long long)split * all_tiles / p.splits), n_tiles = (int)((long long)(split + 1) * all_tiles / p.splits) - t0;
    const int left_last = n_prefix - (t0 + n_tiles - 1) * BN;           // keys of this piece's last tile (>= BN: it is whole)

    if (warp == PX_WARPS) {
        // ================================ TMA producer ================================
        // lane x holds the page of the x-th 16 keys of the tile; it is requested a tile ahead
        const int page_mask = (1 << p.c.page_shift) - 1;
        const int box = min(1 << p.c.page_shift, BN), per_tile = BN / box;
        auto page_at = [&](int tile) -> int {
            const int row = (t0 + tile) * BN + lane * 16;
            if (tile >= n_tiles || lane >= BN / 16 || row >= n_prefix) return -1;
            return p.table[row >> p.c.page_shift];
        };
        auto build_factors = [&](int t) -> bool {
            if (!mbar_wait_warp(&k_full[t % STAGES], (t / STAGES) & 1)) return false;      // the tile's scales have landed
            float *fn = sm_fac + (t % SLOTS) * 3 * BN;
            const float *sc = sm_sc + (t % SLOTS) * 2 * BN;
#pragma unroll
            for (int hh = 0; hh < BN / 32; ++hh) {
                const int k = lane + 32 * hh;
                const float ks = sc[k], vs = sc[BN + k];
                fn[k] = ks * p.scale_log2;
                fn[BN + k] = vs > 0.f ? __log2f(vs) : -INFINITY;
                fn[2 * BN + k] = vs > 0.f ? __fdividef(1.f, vs) : 0.f;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&fac_full[t % SLOTS]);
            return true;
        };
        int next = page_at(0), k_sent = 0, v_sent = 0;
        for (int i = 0; i < n_tiles; ++i) {
            const int s = i % STAGES, row0 = (t0 + i) * BN;
            int page = next;
            next = page_at(i + 1);
            const bool exists = lane < BN / 16 && row0 + lane * 16 < n_prefix;
            if (exists && (page < 0 || page >= p.c.num_pages)) { raise_status(TRB_ST_CURSOR_RANGE); page = -1; }
            const int boxes = min(per_tile, (n_prefix - row0 + box - 1) / box);     // boxes with live rows: the others are not loaded
            uint8_t *kt = smem + C::OFF_KV + s * 2 * TILE, *vt = kt + TILE;
            const uint32_t par = ((i / STAGES) & 1) ^ 1;
            // box b, column block sg of this tile: its page is that of the box's first 16 keys; a page outside the pool reads zeros.
            // The stage is free once the product with its last tile has run
            auto load = [&](uint8_t *dst, const CUtensorMap *map, uint64_t *bar, uint64_t *free) -> bool {
                if (i >= STAGES && !mbar_wait_warp(free, par)) return false;
                if (lane == 0) mbar_arrive_expect_tx(bar, boxes * box * C::ROWB);
                __syncwarp();
                for (int x0 = 0; x0 < per_tile * SEGS; x0 += 32) {
                    const int x = x0 + lane, b = min(x / SEGS, per_tile - 1), sg = x % SEGS;
                    const int pg = __shfl_sync(0xffffffffu, page, b * box / 16);
                    if (x < per_tile * SEGS && b < boxes)
                        tma_load_4d(dst + sg * (BN * 128) + b * box * 128, map, bar, 0, sg, (row0 + b * box) & page_mask, pg < 0 ? -1 : pg * p.c.hkv + j);
                }
                __syncwarp();
                return true;
            };
            if (!load(kt, &tm_k, &k_full[s], &k_free[s])) break;
            ++k_sent;
            if constexpr (FP8) {
                float *sc = sm_sc + (i % SLOTS) * 2 * BN;
#pragma unroll
                for (int hh = 0; hh < BN / 32; ++hh) {
                    const int k = lane + 32 * hh, pg = __shfl_sync(0xffffffffu, page, k / 16);
                    const bool ok = row0 + k < n_prefix && pg >= 0;                // the scales of the others are zero: weight zero
                    const long long off = ok ? ((((long long)pg * p.c.hkv + j) << p.c.page_shift) + ((row0 + k) & page_mask)) : 0;
                    cp_async_4(&sc[k], p.c.ks + off, ok ? 4u : 0u);
                    cp_async_4(&sc[BN + k], p.c.vs + off, ok ? 4u : 0u);
                }
                cp_async_mbar_arrive_noinc(&k_full[s]);
                if (i >= 1 && !build_factors(i - 1)) break;
            }
            if (!load(vt, &tm_v, &v_full[s], &v_free[s])) break;
            ++v_sent;
        }
        if constexpr (FP8) { if (n_tiles > 0) build_factors(n_tiles - 1); }
        if (n_tiles > 0 && v_sent == n_tiles && left_last < BN) {                  // V rows behind the prefix: 0 * NaN must not reach O
            const int s = (n_tiles - 1) % STAGES;
            uint8_t *v_tile = smem + C::OFF_KV + s * 2 * TILE + TILE;
            if (mbar_wait_warp(&v_full[s], ((n_tiles - 1) / STAGES) & 1)) {
                for (int x = lane; x < (BN - left_last) * SEGS * 8; x += 32) {
                    const int row = left_last + x / (SEGS * 8), sg = x / 8 % SEGS;
                    *reinterpret_cast<uint4 *>(v_tile + sg * (BN * 128) + row * 128 + (x & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_clean);
            }
        }
        // no copy is on its way when the CTA leaves, also after a wait that ran out
        for (int t = max(0, k_sent - STAGES); t < k_sent; ++t) mbar_drain(&k_full[t % STAGES], (t / STAGES) & 1);
        for (int t = max(0, v_sent - STAGES); t < v_sent; ++t) mbar_drain(&v_full[t % STAGES], (t / STAGES) & 1);
        __syncwarp();
    } else if (warp == PX_WARPS + 1) {
        // ================================ MMA issuer: one thread ==================================
        // QK(0), QK(1), PV(0), QK(2), PV(1), ..: the pipe runs in order of issue, so QK(i + 2) overwrites the buffer that holds
        // P(i) only after PV(i) has read it
        if (lane != 0) return;                                                     // (the block's last barrier counts the threads that are left)
        if (n_tiles > 0) {
            const uint32_t q_tm = tmem + C::TM_Q;
            const uint32_t q_hi = smem_u32(smem), q_lo = q_hi + C::Q_BYTES;
            constexpr uint32_t IDESC_QK = FP8 ? umma_idesc_f8(PX_BM, BN, false, false) : umma_idesc_bf16(PX_BM, BN, false, false);
            constexpr uint32_t IDESC_PV = FP8 ? umma_idesc_f8(PX_BM, D, false, true) : umma_idesc_bf16(PX_BM, D, false, true);
            auto issue_qk = [&](int i) -> bool {
                const int s = i % STAGES, b = i & 1;
                const uint32_t kt = smem_u32(smem + C::OFF_KV + s * 2 * TILE);
                if (!mbar_wait(&k_full[s], (i / STAGES) & 1)) return false;
                tc_fence_after();
                if constexpr (FP8) {
#pragma unroll
                    for (int term = 0; term < 2; ++term)
#pragma unroll
                        for (int sg = 0; sg < SEGS; ++sg)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                tc_mma_f8(tmem + C::TM_S + b * BN, umma_desc((term ? q_lo : q_hi) + sg * (PX_BM * 128) + k * 32, 16, 1024),
                                          umma_desc(kt + sg * (BN * 128) + k * 32, 16, 1024), IDESC_QK, (term | sg | k) ? 1u : 0u);
                } else {
#pragma unroll
                    for (int sg = 0; sg < SEGS; ++sg)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            tc_mma_bf16_ts(tmem + C::TM_S + b * BN, q_tm + (sg * 4 + k) * 8, umma_desc(kt + sg * (BN * 128) + k * 32, 16, 1024), IDESC_QK,
                                           (sg | k) ? 1u : 0u);
                }
                tc_commit(&k_free[s]);
                tc_commit(&s_full[b]);
                return true;
            };
            bool ok = mbar_wait(q_ready, 0) && issue_qk(0);
            for (int i = 0; i < n_tiles && ok; ++i) {
                const int s = i % STAGES;
                const uint32_t vt = smem_u32(smem + C::OFF_KV + s * 2 * TILE + TILE), p_tm = tmem + C::TM_S + (i & 1) * BN;
                if (i + 1 < n_tiles && !(ok = issue_qk(i + 1))) break;
                if (!(ok = mbar_wait(&v_full[s], (i / STAGES) & 1))) break;
                if (i == n_tiles - 1 && left_last < BN && !(ok = mbar_wait(v_clean, 0))) break;
                if (!(ok = mbar_wait(&p_full[i & 1], (i >> 1) & 1))) break;        // P staged, O corrected
                tc_fence_after();
                if constexpr (FP8) {
#pragma unroll
                    for (int term = 0; term < 2; ++term)
#pragma unroll
                        for (int k = 0; k < BN / 32; ++k)
                            tc_mma_f8_ts(tmem + C::TM_O, p_tm + term * (BN / 4) + k * 8, umma_desc(vt + k * (32 * 128), BN * 128, 1024), IDESC_PV,
                                         (i | term | k) ? 1u : 0u);
                } else {
#pragma unroll
                    for (int k = 0; k < BN / 16; ++k)
                        tc_mma_bf16_ts(tmem + C::TM_O, p_tm + k * 8, umma_desc(vt + k * (16 * 128), BN * 128, 1024), IDESC_PV, (i | k) ? 1u : 0u);
                }
                tc_commit(&v_free[s]);
                tc_commit(i == n_tiles - 1 ? o_last : o_done);
            }
            // no product is under way when the tensor memory is given back, also after a wait that ran out
            tc_commit(mma_out);
            mbar_drain(mma_out, 0);
        }
    } else {
        // ============ softmax / correction / epilogue: thread = (row, quarter of the keys and of the output columns) ============
        const int row = (warp & 3) * 32 + lane, part = warp >> 2;                  // query row = TMEM lane
        const bool row_ok = row < rows_here, warp_ok = (warp & 3) * 32 < rows_here;
        const uint32_t lane_addr = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        float qinv = 1.f;
        if (n_tiles > 0) {
            if constexpr (!FP8) {
                // two dims per column, this thread's quarter of the row; rows past the last are zero
                const uint4 *qp = reinterpret_cast<const uint4 *>(p.q + (row_ok ? sm_off[row] : 0) + part * (D / PX_WG));
                uint32_t w[D / PX_WG / 2];
#pragma unroll
                for (int c = 0; c < D / PX_WG / 8; ++c) {
                    const uint4 raw = row_ok ? qp[c] : make_uint4(0u, 0u, 0u, 0u);
                    w[c * 4 + 0] = raw.x; w[c * 4 + 1] = raw.y; w[c * 4 + 2] = raw.z; w[c * 4 + 3] = raw.w;
                }
                if constexpr (D == 256) tmem_st32_raw(lane_addr + C::TM_Q + part * 32, w);
                else tmem_st16_raw(lane_addr + C::TM_Q + part * 16, w);
                tmem_st_wait();
            } else {
                // hi + lo e4m3 copies with a power-of-two factor for the row.  A warp takes 8 rows, D / 8 lanes with 16 bytes each per row,
                // all requested at once: read by the thread that owns the row, the block took most of 20 us
                float *sm_qinv = sm_mx + 2 * PX_BM;                                // behind the offsets
                constexpr int LPR = D / 8, RPL = 32 / LPR, LOADS = PX_BM / PX_WARPS / RPL;
                uint4 raw[LOADS];
#pragma unroll
                for (int x = 0; x < LOADS; ++x) {
                    const long long off = sm_off[warp * (PX_BM / PX_WARPS) + x * RPL + lane / LPR];
                    raw[x] = off >= 0 ? *reinterpret_cast<const uint4 *>(p.q + off + lane % LPR * 8) : make_uint4(0u, 0u, 0u, 0u);
                }
#pragma unroll
                for (int x = 0; x < LOADS; ++x) {
                    const int wr = warp * (PX_BM / PX_WARPS) + x * RPL + lane / LPR;
                    const __nv_bfloat162 *b2 = reinterpret_cast<const __nv_bfloat162 *>(&raw[x]);
                    float f[8], amax = 0.f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 v = __bfloat1622float2(b2[e]);
                        f[2 * e] = v.x; f[2 * e + 1] = v.y;
                        amax = fmaxf(amax, fmaxf(fabsf(v.x), fabsf(v.y)));
                    }
#pragma unroll
                    for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
                    int e = (int)((__float_as_uint(amax) >> 23) & 0xffu) - 127;
                    if (amax == 0.f || e < -90) e = 7;
                    if (e > 90) e = 90;
                    const float sc = __uint_as_float((uint32_t)(127 + 7 - e) << 23);
                    if (lane % LPR == 0) sm_qinv[wr] = __uint_as_float((uint32_t)(127 - 7 + e) << 23);
                    uint32_t hw[2], lw[2];
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const float y[4] = {f[4 * w] * sc, f[4 * w + 1] * sc, f[4 * w + 2] * sc, f[4 * w + 3] * sc};
                        pf_split4(y, hw[w], lw[w]);
                    }
                    const int byte = lane % LPR * 8;
                    const uint32_t off = (byte >> 7) * (PX_BM * 128) + sw128(wr, byte & 127);
                    *reinterpret_cast<uint2 *>(smem + off) = make_uint2(hw[0], hw[1]);
                    *reinterpret_cast<uint2 *>(smem + C::Q_BYTES + off) = make_uint2(lw[0], lw[1]);
                }
                fence_async_smem();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
            if constexpr (FP8) {
                named_barrier(1, PX_SOFTMAX);
                qinv = sm_mx[2 * PX_BM + row];
                named_barrier(1, PX_SOFTMAX);                                      // (read by all before a tile's maxima are written over it)
            }
        }

        float m_run = -INFINITY, m_top = -INFINITY, l_run = 0.f;                   // reference and largest score of the row; l_run: this thread's quarter of the keys
        bool ok = true;
        for (int i = 0; i < n_tiles; ++i) {
            const int b = i & 1;
            const float *fac = sm_fac + (i % SLOTS) * 3 * BN + part * KPT;
            float *mxbuf = sm_mx + b * PX_WG * PX_BM;
            ok = ok && mbar_wait(&s_full[b], (i >> 1) & 1);
            if constexpr (FP8) ok = ok && mbar_wait(&fac_full[i % SLOTS], (i / SLOTS) & 1);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            // a warp without query rows, or one whose wait ran out, only takes part in the barriers
            if (warp_ok && ok) {
                float sv[KPT];
                if constexpr (KPT == 32) tmem_ld32(lane_addr + C::TM_S + b * BN + part * KPT, sv);
                else tmem_ld16(lane_addr + C::TM_S + b * BN + part * KPT, sv);
                if constexpr (!FP8) {
                    const float2 sl2 = make_float2(p.scale_log2, p.scale_log2);
#pragma unroll
                    for (int c = 0; c < KPT / 2; ++c) {
                        const float2 a = __fmul2_rn(make_float2(sv[2 * c], sv[2 * c + 1]), sl2);
                        sv[2 * c] = a.x; sv[2 * c + 1] = a.y;
                    }
                } else {
                    const float2 qinv2 = make_float2(qinv, qinv);
#pragma unroll
                    for (int c4 = 0; c4 < KPT / 4; ++c4) {
                        const float4 fa = *reinterpret_cast<const float4 *>(fac + c4 * 4);
                        const float4 fb = *reinterpret_cast<const float4 *>(fac + BN + c4 * 4);
                        const float2 a = __ffma2_rn(__fmul2_rn(make_float2(sv[c4 * 4 + 0], sv[c4 * 4 + 1]), make_float2(fa.x, fa.y)), qinv2, make_float2(fb.x, fb.y));
                        const float2 c = __ffma2_rn(__fmul2_rn(make_float2(sv[c4 * 4 + 2], sv[c4 * 4 + 3]), make_float2(fa.z, fa.w)), qinv2, make_float2(fb.z, fb.w));
                        sv[c4 * 4 + 0] = a.x; sv[c4 * 4 + 1] = a.y; sv[c4 * 4 + 2] = c.x; sv[c4 * 4 + 3] = c.y;
                    }
                }
                if (i == n_tiles - 1 && left_last < BN) {
#pragma unroll
                    for (int c = 0; c < KPT; ++c)
                        if (part * KPT + c >= left_last) sv[c] = -INFINITY;
                }
                float mt4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int c = 0; c < KPT / 2; ++c) mt4[c & 3] = pf_max3(mt4[c & 3], sv[2 * c], sv[2 * c + 1]);
                mxbuf[part * PX_BM + row] = fmaxf(fmaxf(mt4[0], mt4[1]), fmaxf(mt4[2], mt4[3]));
                named_barrier(1, PX_SOFTMAX);
                const float top = fmaxf(pf_max3(-INFINITY, mxbuf[row], mxbuf[PX_BM + row]), fmaxf(mxbuf[2 * PX_BM + row], mxbuf[3 * PX_BM + row]));
                float m_new, alpha;
                if constexpr (!FP8) {
                    m_new = top > m_run + C::SLACK ? top : m_run;
                    alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
                } else {                                                           // whole references: the factors of their moves are exact
                    m_top = fmaxf(m_top, top);
                    m_new = top > m_run || top < m_run - C::DROP ? fmaxf(ceilf(top), ceilf(m_top) - C::DEPTH) : m_run;
                    const float by = m_run - m_new;                                // <= DEPTH
                    alpha = m_new == m_run ? 1.f : by > -127.f ? __uint_as_float((uint32_t)((int)by + 127) << 23) : 0.f;
                }
                const float m_off = (m_new == -INFINITY ? 0.f : m_new) - C::LIFT;
                // O is corrected only in warps where a row's reference moved (S of this tile exists, so PV(i - 2) has completed: the
                // parity cannot be mistaken)
                if (__any_sync(0xffffffffu, alpha != 1.f) && i > 0) {
                    ok = mbar_wait_warp(o_done, (i - 1) & 1);
                    if (ok) {
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < D / PX_WG / 32; ++c) {
                            float ov[32];
                            tmem_ld32(lane_addr + C::TM_O + part * (D / PX_WG) + c * 32, ov);
#pragma unroll
                            for (int e = 0; e < 32; ++e) ov[e] *= alpha;
                            tmem_st32(lane_addr + C::TM_O + part * (D / PX_WG) + c * 32, ov);
                        }
                    }
                }
                const uint32_t p_tm = lane_addr + C::TM_S + b * BN;                // (all of S was read before the barrier above)
                float lsum = 0.f;
                if constexpr (!FP8) {
                    uint32_t w[KPT / 2];
#pragma unroll
                    for (int e = 0; e < KPT / 2; ++e) {
                        w[e] = pack_bf16x2(fast_exp2(sv[e * 2] - m_off), fast_exp2(sv[e * 2 + 1] - m_off));
                        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w[e]));   // the sum takes the weights as they multiply V
                        lsum += f.x + f.y;
                    }
                    if constexpr (KPT == 32) tmem_st16_raw(p_tm + part * 16, w);
                    else tmem_st8_raw(p_tm + part * 8, w);
                } else {
                    const float2 nm2 = make_float2(-m_off, -m_off);
                    float2 lsa = make_float2(0.f, 0.f), lsb = make_float2(0.f, 0.f);
                    uint32_t hw8[8], lw8[8];
#pragma unroll
                    for (int w = 0; w < 8; ++w) {
                        const int k0 = w * 4;
                        const float4 fr = *reinterpret_cast<const float4 *>(fac + 2 * BN + k0);
                        const float2 d01 = __fadd2_rn(make_float2(sv[k0 + 0], sv[k0 + 1]), nm2);
                        const float2 d23 = __fadd2_rn(make_float2(sv[k0 + 2], sv[k0 + 3]), nm2);
                        const float2 p01 = make_float2(fast_exp2(d01.x), fast_exp2(d01.y));
                        const float2 p23 = make_float2(fast_exp2(d23.x), fast_exp2(d23.y));
                        lsa = __ffma2_rn(p01, make_float2(fr.x, fr.y), lsa);
                        lsb = __ffma2_rn(p23, make_float2(fr.z, fr.w), lsb);
                        uint32_t h01, l01, h23, l23;
                        pf_split2_h(p01.x, p01.y, h01, l01);
                        pf_split2_h(p23.x, p23.y, h23, l23);
                        hw8[w] = h01 | (h23 << 16);
                        lw8[w] = l01 | (l23 << 16);
                    }
                    tmem_st8_raw(p_tm + part * 8, hw8);
                    tmem_st8_raw(p_tm + BN / 4 + part * 8, lw8);
                    lsum = (lsa.x + lsa.y) + (lsb.x + lsb.y);
                }
                l_run = fmaf(l_run, alpha, lsum);
                m_run = m_new;
                tmem_st_wait();
                tc_fence_before();
            } else {
                named_barrier(1, PX_SOFTMAX);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[b]);
        }
        // ---- the piece's partial.  The last PV has a barrier of its own: a warp that skipped corrections does not know how many phases
        // of o_done have passed, so no parity of it would name the last one
        if (ok && n_tiles > 0) ok = mbar_wait(o_last, 0);
        ok = __all_sync(0xffffffffu, ok);
        tc_fence_after();
        // O goes through the ring (every tile has been consumed), so that it leaves in whole rows: 16-byte pieces, swizzled by row
        float4 *sm_o = reinterpret_cast<float4 *>(smem + C::OFF_KV);
        float *sm_l = sm_mx + (n_tiles & 1) * PX_WG * PX_BM;                       // (the other buffer may still be read)
        sm_l[part * PX_BM + row] = l_run;
        if (n_tiles > 0 && warp_ok) {
#pragma unroll 1
            for (int c = 0; c < D / PX_WG / 32; ++c) {
                float ov[32];
                tmem_ld32(lane_addr + C::TM_O + part * (D / PX_WG) + c * 32, ov);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int piece = part * (D / PX_WG / 4) + c * 8 + e;
                    sm_o[row * (D / 4) + (piece ^ (row & 7))] = make_float4(ov[e * 4], ov[e * 4 + 1], ov[e * 4 + 2], ov[e * 4 + 3]);
                }
            }
        }
        named_barrier(1, PX_SOFTMAX);
        const long long at = ((long long)split * p.c.hkv + j) * rows_all + q0;
        if (row_ok && part == 0)
            *reinterpret_cast<float2 *>(p.part_ml + (at + row) * 2) =
                make_float2(m_run - C::LIFT, (sm_l[row] + sm_l[PX_BM + row]) + (sm_l[2 * PX_BM + row] + sm_l[3 * PX_BM + row]));
        if (n_tiles > 0) {
            float4 *dst = reinterpret_cast<float4 *>(p.part_acc + at * D);
#pragma unroll 4
            for (int x = warp * 32 + lane; x < rows_here * (D / 4); x += PX_SOFTMAX) {
                const int orow = x / (D / 4), piece = x % (D / 4);
                dst[x] = sm_o[orow * (D / 4) + (piece ^ (orow & 7))];
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 0) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

}  // namespace trb
