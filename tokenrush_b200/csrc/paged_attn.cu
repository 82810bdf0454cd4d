// Attention of a batch of sequences over a shared prefix and each sequence's own pages.
//
//   o = sum_x exp(s_x - m) v_x / sum_x exp(s_x - m),   s_x = scale q . k_x,   x over the prefix rows and the own rows <= lens[b] + i
//
// paged_scan_kernel reads cache rows for the few query rows of one sequence (G = hq / hkv heads x m tokens per kv
// head) and is bound by HBM: the work is cut along one line of key tiles that runs through all sequences, every CTA
// takes an equal piece of it whatever the lengths are, and a piece that covers part of a sequence leaves a (max, sum,
// acc) partial that paged_merge_kernel joins.  The lengths are device integers: every CTA finds its piece itself.
//
// Inside a CTA four warps work on key tiles of their own, with a private ring of stages filled by TMA: no barrier is
// passed while tiles stream.  A tile is 16 keys, so it lies in one page: a copy per 128-byte column, swizzled, and 64 bytes of scales.
// The products run with the keys (resp. the head dims) as the 16-row operand of mma.m16n8k16 and the
// query rows as the 8 columns, as in the contiguous decode kernel:
//   S^T[16 keys x 8] = K Q^T,   O^T[dims x 8] += V^T P^T.
// The order of dims inside a contraction is free, so a lane reads 16-byte chunks of a row instead of fragments, and the
// chunk's order is carried by how Q is laid out and O is read back.  e4m3 codes become f16 in registers; the K scale
// multiplies the score, the V scale moves into the exponent, so codes are never scaled.
//
// While tiles stream, three CTAs of four warps keep HBM full (a warp's 8 KB step takes 1.8 us).  What remains is what a sequence costs apart from
// its tiles: finding its page, its query rows, the join of the warps.  The line therefore counts PS_TURN steps for the
// start of every sequence, and the next sequence's first tiles and query rows are requested before the join of this one.
#include "paged.cuh"
#include "paged_prefix.cuh"
#include "tmap.h"

namespace trb {

constexpr int PS_WARPS = 4, PS_THREADS = PS_WARPS * 32;
constexpr int PS_TURN = 10;             // steps that a change of sequence costs a CTA (3: 65.4 us, 6: 64.1, 10: 63.2, 20: 63.8 for the 64 chats)

struct PagedAttnParams {
    PagedView c;
    BatchView b;
    const __nv_bfloat16 *q;
    __nv_bfloat16 *out;
    const __nv_bfloat16 *gate;
    long long gate_rs, gate_hs;
    int m, hq, g;                      // g = hq / hkv
    float scale_log2;
    const int *prefix_table;
    int prefix_pages;                  // rows of the prefix that the scan itself reads come from here (0: none)
    Cursor prefix_len;
    int after_prefix;                  // launched behind paged_prefix_kernel, which reads the prefix
    int splits;                        // its pieces (0: none)
    const float *px_ml, *px_acc;       // [splits][hkv][n_seqs * m * g][2] and [..][D]
    int ctas;                          // CTAs per (kv head, row group)
    int groups;                        // groups of 8 * NS query rows
    int *plan;                         // [n_seqs][2]: first and last CTA with keys of the sequence
    float *part_ml;                    // [hkv * groups][ctas + n_seqs][8 NS][2]
    float *part_acc;                   // [hkv * groups][ctas + n_seqs][8 NS][D]
};

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}

template <int D_, bool FP8_, int NS_> struct ScanCfg {
    static constexpr int D = D_, NS = NS_, SUB = D_ == 128 && FP8_ ? 2 : 1;     // 16-key tiles per pipeline step: 8 KB of K and V, 16 KB for 256-dim bf16
    static constexpr bool FP8 = FP8_;
    static constexpr int ROWB = D * (FP8 ? 1 : 2), CPR = ROWB / 16, SEGS = ROWB / 128;   // bytes, 16-byte chunks and 128-byte columns of a row
    static constexpr int TILE = 16 * ROWB, STAGE = SUB * 2 * TILE;
    static constexpr int STAGES = NS == 1 && STAGE == 8192 ? 2 : 3;
    static constexpr int CTAS = STAGE > 8192 ? 1 : NS == 1 ? 3 : 2;    // per SM, by shared memory and registers
    static constexpr int RING = STAGES * STAGE;                        // per warp
    static constexpr int KJ = CPR / 4, VC = CPR / 8;                   // chunks per lane of a K row, of a V row
    static constexpr int KS = D / 16;                                  // MMA steps of a QK product = row tiles of a PV product
    static constexpr int RED = (NS * 8 * D * 4 + STAGE - 1) / STAGE;   // stages that a warp's accumulators take when they are exchanged
    static constexpr int OFF_SC = PS_WARPS * RING;                     // [warps][stages][SUB][K, V][16] floats
    static constexpr int OFF_Q = OFF_SC + (FP8 ? PS_WARPS * STAGES * SUB * 128 : 0);      // [NS][KS][32] uint2
    static constexpr int OFF_QINV = OFF_Q + (NS > 1 ? NS * KS * 256 : 0);      // [warps or slices][8] floats
    static constexpr int OFF_ML = OFF_QINV + PS_WARPS * 32;            // [warps][8 NS][2] floats
    static constexpr int OFF_BAR = OFF_ML + PS_WARPS * NS * 64;        // [warps][4] mbarriers
    static constexpr int OFF_CNT = OFF_BAR + PS_WARPS * 32;            // [PG_MAX_SEQS + 1] ints, then 8 for the scan
    static constexpr int SMEM = OFF_CNT + (PG_MAX_SEQS + 16) * 4 + 1024;      // + slack to align the base
    static_assert(RED < STAGES && NS <= PS_WARPS && STAGES <= 4, "the exchange leaves a stage for the next sequence");
    static_assert(CTAS * (SMEM + 1024) <= 228 * 1024, "shared memory of an SM");
};

// Untiled copy global -> shared (both addresses and the size multiples of 16 bytes) that completes on the mbarrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

template <typename C>
__global__ void __launch_bounds__(PS_THREADS, C::CTAS)
paged_scan_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const PagedAttnParams p) {
    constexpr int D = C::D, NS = C::NS, SUB = C::SUB, KS = C::KS, KJ = C::KJ, VC = C::VC, CPR = C::CPR;
    constexpr int SEGS = C::SEGS, STAGES = C::STAGES;
    constexpr bool FP8 = C::FP8;
    extern __shared__ uint8_t ps_smem_raw[];
    uint8_t *ps_smem = ps_smem_raw + ((1024u - (smem_u32(ps_smem_raw) & 1023u)) & 1023u);
    float *sm_qinv = reinterpret_cast<float *>(ps_smem + C::OFF_QINV);
    float *sm_ml = reinterpret_cast<float *>(ps_smem + C::OFF_ML);
    int *sm_cnt = reinterpret_cast<int *>(ps_smem + C::OFF_CNT);
    uint2 *sm_q = reinterpret_cast<uint2 *>(ps_smem + C::OFF_Q);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int j = blockIdx.y % p.c.hkv, grp = blockIdx.y / p.c.hkv, hg = blockIdx.y;
    const int rows = p.g * p.m, r0 = grp * 8 * NS;
    const uint32_t ring = smem_u32(ps_smem + warp * C::RING), scales = smem_u32(ps_smem + C::OFF_SC) + warp * STAGES * SUB * 128;
    uint64_t *full = reinterpret_cast<uint64_t *>(ps_smem + C::OFF_BAR) + warp * 4;      // one per stage
    uint32_t phases = 0, armed = 0;                                    // bit s: parity of stage s's next completion; of the one after its last load
    bool ok = true;                                                    // no wait of this warp has run out
    if (lane == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1u);
        mbar_fence_init();
        if (warp == 0) { tma_prefetch_desc(&tm_k); tma_prefetch_desc(&tm_v); }
    }
    __syncwarp();
    // behind the prefix kernel this one starts when that has passed its own wait: everything before both is complete, and what
    // the two write is apart.  It then waits at its end, so that its completion says the same of the prefix kernel.
    if (!p.after_prefix) pdl_wait();
    pdl_launch_dependents();

    // ---- the line of pipeline steps: sequence b has places sm_cnt[b] .. sm_cnt[b + 1] - 1 of it, PS_TURN for its start and then its steps
    const bool report = blockIdx.x == 0 && blockIdx.y == 0;
    const int n_prefix = paged_prefix_rows(p.prefix_len, p.prefix_pages, p.c.page_shift, report && threadIdx.x == 0);
    const int prefix_tiles = (n_prefix + 15) >> 4;
    const int per = (p.b.n_seqs + PS_THREADS - 1) / PS_THREADS;
    {
        const int b0 = threadIdx.x * per;
        int sum = 0;
        for (int b = b0; b < b0 + per && b < p.b.n_seqs; ++b) {
            const int own = paged_own_rows(p.b, b, p.m, p.c.page_shift, report);
            int steps = own < 0 ? 0 : (prefix_tiles + ((own + 15) >> 4) + SUB - 1) / SUB;
            steps += steps > 0 ? PS_TURN : 0;
            sm_cnt[b] = sum;
            sum += steps;
        }
        int inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += v; }
        int *wsum = sm_cnt + PG_MAX_SEQS + 1;
        if (lane == 31) wsum[warp] = inc;
        __syncthreads();
        int before = inc - sum;
        for (int w = 0; w < warp; ++w) before += wsum[w];
        for (int b = b0; b < b0 + per && b < p.b.n_seqs; ++b) sm_cnt[b] += before;
        if (threadIdx.x == PS_THREADS - 1) sm_cnt[p.b.n_seqs] = before + sum;
        __syncthreads();
    }
    const int total = sm_cnt[p.b.n_seqs];
    // a CTA gets about a step for each of its warps at least
    const int active = max(1, min(p.ctas, total / PS_WARPS));
    if (report) {
        for (int b = threadIdx.x; b < p.b.n_seqs; b += PS_THREADS) {
            const int lo = sm_cnt[b], hi = sm_cnt[b + 1];
            p.plan[2 * b] = hi > lo ? (int)((((long long)lo + PS_TURN + 1) * active - 1) / total) : 0;    // the CTA that has the first step
            p.plan[2 * b + 1] = hi > lo ? (int)(((long long)hi * active - 1) / total) : -1;               // ... and the last
        }
    }
    if ((int)blockIdx.x >= active || total == 0) { pdl_wait(); return; }
    const int lo = (int)((long long)blockIdx.x * total / active), hi = (int)(((long long)blockIdx.x + 1) * total / active);
    if (lo >= hi) { pdl_wait(); return; }
    int seq;
    {
        int a = 0, z = p.b.n_seqs;                                      // last sequence that starts at or before lo
        while (z - a > 1) { const int mid = (a + z) >> 1; if (sm_cnt[mid] <= lo) a = mid; else z = mid; }
        seq = a;
        while (sm_cnt[seq + 1] <= lo) ++seq;                            // (skips slots without steps that start at lo)
    }

    // ---- pipeline of a warp over the steps s0 + warp, s0 + warp + 4, .. of the current sequence
    int s0, s1, own, steps, pages[SUB];
    long long len;
    const int *own_table;
    auto page_of = [&](int tile) -> int {                              // pool page of a tile, -1: none
        const int x = tile - prefix_tiles;
        int pg = -1;
        if (x < 0) pg = p.prefix_table[(tile * 16) >> p.c.page_shift];
        else if (x * 16 < own) pg = own_table[(x * 16) >> p.c.page_shift];
        else return -1;
        if (pg < 0 || pg >= p.c.num_pages) { if (lane == 0) raise_status(TRB_ST_CURSOR_RANGE); pg = -1; }
        return pg;
    };
    auto fetch_pages = [&](int k) {
#pragma unroll
        for (int sb = 0; sb < SUB; ++sb) pages[sb] = k < steps ? page_of((s0 + warp + k * PS_WARPS) * SUB + sb) : -1;
    };
    // A step's copies, one per lane: K and V columns, K and V scales of each of its tiles.  A tile behind the sequence's last row, or of a
    // page outside the pool, reads zeros (a coordinate outside the tensor).
    auto load_step = [&](int step, int stage, const int (&pg)[SUB]) {
        constexpr int OPS = 2 * SEGS + (FP8 ? 2 : 0);
        const int sb = SUB == 1 ? 0 : lane / OPS, op = lane - sb * OPS;
        const int page = SUB == 1 || sb == 0 ? pg[0] : pg[SUB - 1];
        const int x = step * SUB + sb - prefix_tiles, in_page = ((x < 0 ? x + prefix_tiles : x) * 16) & ((1 << p.c.page_shift) - 1);
        if (lane == 0) {
            int scaled = 0;
#pragma unroll
            for (int y = 0; y < SUB; ++y) scaled += pg[y] >= 0 ? 128 : 0;
            mbar_arrive_expect_tx(&full[stage], C::STAGE + (FP8 ? scaled : 0));
        }
        __syncwarp();
        if (lane < SUB * OPS) {
            const bool of_v = op < 2 * SEGS ? op >= SEGS : op > 2 * SEGS;
            if (op < 2 * SEGS) {
                const int sg = of_v ? op - SEGS : op;
                tma_load_4d(ps_smem + warp * C::RING + stage * C::STAGE + (sb * 2 + (of_v ? 1 : 0)) * C::TILE + sg * 2048, of_v ? &tm_v : &tm_k, &full[stage],
                            0, sg, in_page, page < 0 ? -1 : page * p.c.hkv + j);
            } else if (page >= 0) {
                const long long row = (((long long)page * p.c.hkv + j) << p.c.page_shift) + in_page;
                bulk_load(scales + (stage * SUB + sb) * 128 + (of_v ? 64 : 0), (of_v ? p.c.vs : p.c.ks) + row, 64u, &full[stage]);
            }
        }
    };
    // step k of a sequence goes to stage (k + RED) mod STAGES: the first RED stages hold the accumulators that the warps
    // exchange at the end of the sequence before, while the first steps of this one are already on their way
    constexpr int RED = C::RED, EARLY = STAGES - RED;
    auto request = [&](int k) {
        int now[SUB];
#pragma unroll
        for (int sb = 0; sb < SUB; ++sb) now[sb] = pages[sb];
        fetch_pages(k + 1);
        if (k < steps && ok) {
            load_step(s0 + warp + k * PS_WARPS, (k + RED) % STAGES, now);
            armed ^= 1u << (k + RED) % STAGES;
        }
    };
    // ---- the query rows as MMA fragments: step (jj, w) of lane (g, t) holds dims of chunk 8 (jj / 2) + 2 t + jj % 2 (so that the eight lanes
    // of a shared-memory phase, two rows by four t, meet eight different places of the swizzle).  e4m3: f16 with a power-of-two
    // factor for each row (a bf16 value may lie outside f16's range); bf16: as they are.
    constexpr int DPC = FP8 ? 16 : 8;                                  // dims of a chunk
    uint2 qf[KS];
    const int q_slice = NS == 1 ? 0 : warp, q_row = r0 + q_slice * 8 + g;      // one slice: every warp for itself; else a slice per warp
    const bool q_ok = q_slice < NS && q_row < rows;
    const long long q_at = ((long long)(q_ok ? q_row / p.g : 0) * p.hq + j * p.g + (q_ok ? q_row % p.g : 0)) * D;
    auto begin = [&]() {                                               // sequence seq: its piece, its query rows and the first EARLY steps
        const int first = sm_cnt[seq] + PS_TURN;
        s0 = max(lo, first) - first;
        s1 = min(hi, sm_cnt[seq + 1]) - first;
        if (NS == 1 || warp < NS) {
            const __nv_bfloat16 *src = p.q + (long long)seq * p.m * p.hq * D + q_at;
#pragma unroll
            for (int jj = 0; jj < KJ; ++jj)
#pragma unroll
                for (int x = 0; x < DPC / 8; ++x) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(src + (8 * (jj >> 1) + 2 * t + (jj & 1)) * DPC + x * 8);
                    qf[jj * (DPC / 4) + 2 * x] = make_uint2(v.x, v.y);
                    qf[jj * (DPC / 4) + 2 * x + 1] = make_uint2(v.z, v.w);
                }
        }
        len = load_len(p.b, seq);
        own = (int)(min(len, ((long long)p.b.table_pages << p.c.page_shift) - p.m) + p.m);
        own_table = p.b.table + seq * p.b.table_stride;
        steps = ok && s1 - s0 > warp ? (s1 - s0 - warp + PS_WARPS - 1) / PS_WARPS : 0;
        fetch_pages(0);
#pragma unroll
        for (int k = 0; k < (EARLY < STAGES - 1 ? EARLY : STAGES - 1); ++k) request(k);
    };
    if (lo >= sm_cnt[seq + 1] || hi <= sm_cnt[seq] + PS_TURN) {         // (the piece ends in the start of its only sequence)
        pdl_wait();
        return;
    }
    begin();
    while (true) {
        const int now = seq;
#pragma unroll
        for (int k = EARLY; k < STAGES - 1; ++k) request(k);

        if (NS == 1 || warp < NS) {
#pragma unroll
            for (int x = 0; x < KS; ++x) qf[x] = q_ok ? qf[x] : make_uint2(0u, 0u);
            float q_inv = 1.f;
            if constexpr (FP8) {
                float amax = 0.f;
#pragma unroll
                for (int x = 0; x < KS; ++x) {
                    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&qf[x].x));
                    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&qf[x].y));
                    amax = fmaxf(amax, fmaxf(fmaxf(fabsf(a.x), fabsf(a.y)), fmaxf(fabsf(b.x), fabsf(b.y))));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                int e = (int)((__float_as_uint(amax) >> 23) & 0xffu) - 127;
                e = amax == 0.f ? 0 : max(-90, min(90, e));
                const float mult = __uint_as_float((uint32_t)(127 - e) << 23);
                q_inv = __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
                for (int x = 0; x < KS; ++x) {
                    const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&qf[x].x));
                    const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&qf[x].y));
                    qf[x] = make_uint2(pack_f16x2(a.x * mult, a.y * mult), pack_f16x2(b.x * mult, b.y * mult));
                }
            }
            if (t == 0) sm_qinv[warp * 8 + g] = q_inv;
            if constexpr (NS > 1) {                                    // through shared memory
#pragma unroll
                for (int x = 0; x < KS; ++x) sm_q[(warp * KS + x) * 32 + lane] = qf[x];
            }
        }
        if constexpr (NS > 1) __syncthreads();
        else __syncwarp();
        // this thread's query rows are columns 2t, 2t + 1 of each slice
        float qinv[NS * 2], ref[NS * 2], l[NS * 2], acc[NS][KS][4];
        int last[NS * 2];                                              // own rows below this are visible
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int r = r0 + s * 8 + 2 * t + e;
                qinv[s * 2 + e] = FP8 ? sm_qinv[(NS == 1 ? warp : s) * 8 + 2 * t + e] * p.scale_log2 : p.scale_log2;
                last[s * 2 + e] = (int)min((long long)own, len + 1 + (r < rows ? r / p.g : p.m));
                ref[s * 2 + e] = -INFINITY;
                l[s * 2 + e] = 0.f;
            }
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int a = 0; a < KS; ++a)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[s][a][e] = 0.f;

        for (int k = 0; k < steps; ++k) {
            request(k + STAGES - 1);
            const int stage = (k + RED) % STAGES, step = s0 + warp + k * PS_WARPS;
            ok = mbar_wait_warp(&full[stage], (phases >> stage) & 1u);
            if (!ok) steps = 0;                                        // (the output is undefined, but nothing hangs)
            phases ^= (uint32_t)ok << stage;
            const uint32_t base = ring + stage * C::STAGE;
#pragma unroll
            for (int sb = 0; sb < SUB; ++sb) {                         // V rows behind the last one: a weight of zero times NaN must not reach O
                const int x = step * SUB + sb - prefix_tiles, left = x < 0 ? n_prefix - (x + prefix_tiles) * 16 : own - x * 16;
                if (left < 16) {
                    const int from = max(left, 0);
                    for (int y = lane; y < (16 - from) * CPR; y += 32)
                        *reinterpret_cast<uint4 *>(ps_smem + warp * C::RING + stage * C::STAGE + (sb * 2 + 1) * C::TILE + (y & 7) * 16 +
                                                   (y >> 3) % SEGS * 2048 + (from + (y >> 3) / SEGS) * 128) = make_uint4(0u, 0u, 0u, 0u);
                    fence_async_smem();
                    __syncwarp();
                }
            }

            // S^T: two chains of MMAs per tile
            float sc[SUB][NS][4];
#pragma unroll
            for (int sb = 0; sb < SUB; ++sb) {
                float s2[NS][2][4];
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s2[s][0][e] = s2[s][1][e] = 0.f;
                const uint32_t kb = base + sb * 2 * C::TILE + g * 128;
#pragma unroll
                for (int jj = 0; jj < KJ; ++jj) {
                    const uint32_t ch = (jj >> 1) * 2048 + (((2 * t + (jj & 1)) ^ g) << 4);       // (rows g and g + 8 are swizzled alike)
                    const uint4 x = ld_shared_v4(kb + ch), y = ld_shared_v4(kb + 8 * 128 + ch);
                    const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
                    if constexpr (FP8) {
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const uint32_t a[4] = {e4m3x2_to_f16x2((uint16_t)xw[w]), e4m3x2_to_f16x2((uint16_t)yw[w]),
                                                   e4m3x2_to_f16x2((uint16_t)(xw[w] >> 16)), e4m3x2_to_f16x2((uint16_t)(yw[w] >> 16))};
#pragma unroll
                            for (int s = 0; s < NS; ++s) {
                                const uint2 b = NS == 1 ? qf[jj * 4 + w] : sm_q[(s * KS + jj * 4 + w) * 32 + lane];
                                mma_f16(s2[s][w & 1], a, b.x, b.y);
                            }
                        }
                    } else {
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const uint32_t a[4] = {xw[2 * w], yw[2 * w], xw[2 * w + 1], yw[2 * w + 1]};
#pragma unroll
                            for (int s = 0; s < NS; ++s) {
                                const uint2 b = NS == 1 ? qf[jj * 2 + w] : sm_q[(s * KS + jj * 2 + w) * 32 + lane];
                                mma_bf16(s2[s][w], a, b.x, b.y);
                            }
                        }
                    }
                }
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sc[sb][s][e] = s2[s][0][e] + s2[s][1][e];
            }
            // scores in log2 units (+ log2 of the V scale), masked; element e: key g + 8 (e >> 1), column 2t + (e & 1)
            float vinv[SUB][2];
            bool raise = false;
#pragma unroll
            for (int sb = 0; sb < SUB; ++sb) {
                float kf[2] = {1.f, 1.f}, vl[2] = {0.f, 0.f};
                if constexpr (FP8) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float kk, vv;
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(kk) : "r"(scales + (stage * SUB + sb) * 128 + (g + 8 * h) * 4));
                        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(vv) : "r"(scales + (stage * SUB + sb) * 128 + 64 + (g + 8 * h) * 4));
                        kf[h] = kk;
                        vl[h] = __log2f(vv);
                        vinv[sb][h] = __fdividef(1.f, vv);
                    }
                }
                const int tile = step * SUB + sb, x = tile - prefix_tiles;
                const int row = x < 0 ? tile * 16 : x * 16;
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc[sb][s][e] = FP8 ? fmaf(sc[sb][s][e] * kf[e >> 1], qinv[s * 2 + (e & 1)], vl[e >> 1]) : sc[sb][s][e] * qinv[s * 2 + (e & 1)];
                if (row + 16 > (x < 0 ? (long long)n_prefix : len + 1)) {      // a key of the tile is hidden from some row
#pragma unroll
                    for (int s = 0; s < NS; ++s)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int limit = x < 0 ? n_prefix : last[s * 2 + (e & 1)];
                            if (row + g + 8 * (e >> 1) >= limit) sc[sb][s][e] = -INFINITY;
                        }
                }
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int e = 0; e < 4; ++e) raise |= sc[sb][s][e] > ref[s * 2 + (e & 1)] + 8.f;
            }
            // the reference of a row follows its maximum lazily: weights up to 2^8 fit f16, so it moves only when a score
            // passes it by more
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int sb = 0; sb < SUB; ++sb) mx = fmaxf(mx, fmaxf(sc[sb][s][e], sc[sb][s][e + 2]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        mx = fmaxf(mx, ref[s * 2 + e]);
                        const float alpha = mx == -INFINITY ? 1.f : fast_exp2(ref[s * 2 + e] - mx);
                        ref[s * 2 + e] = mx;
                        l[s * 2 + e] *= alpha;
#pragma unroll
                        for (int a = 0; a < KS; ++a) { acc[s][a][e] *= alpha; acc[s][a][e + 2] *= alpha; }
                    }
            }
            // weights and O^T += V^T P^T
#pragma unroll
            for (int sb = 0; sb < SUB; ++sb) {
                uint32_t pb[NS][2];
#pragma unroll
                for (int s = 0; s < NS; ++s) {
                    float w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float m0 = ref[s * 2 + (e & 1)];
                        w[e] = fast_exp2(sc[sb][s][e] - (m0 == -INFINITY ? 0.f : m0));
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t pk;
                        if constexpr (FP8) {
                            pk = pack_f16x2(w[2 * h], w[2 * h + 1]);      // 11 bits down to 2^-14 of the reference, off by 2^-25 of it below
#pragma unroll
                            for (int e = 0; e < 2; ++e) l[s * 2 + e] += w[2 * h + e] > 0.f ? w[2 * h + e] * vinv[sb][h] : w[2 * h + e] * 0.f;
                        } else {
                            // bf16 like the V they multiply (one MMA takes one type, f16 cannot hold V): 8 bits at any size.  The sum takes them as they are then
                            pk = pack_bf16x2(w[2 * h], w[2 * h + 1]);
                            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&pk));
                            l[s * 2] += f.x;
                            l[s * 2 + 1] += f.y;
                        }
                        pb[s][h] = movmatrix_trans(pk);
                    }
                }
                const uint32_t vb = base + sb * 2 * C::TILE + C::TILE + 2 * t * 128;
#pragma unroll
                for (int c = 0; c < VC; ++c) {
                    // keys 2t, 2t + 1, 2t + 8, 2t + 9
                    const uint32_t c0 = c * 2048 + ((g ^ (2 * t)) << 4), c1 = c * 2048 + ((g ^ (2 * t + 1)) << 4);
                    const uint4 v[4] = {ld_shared_v4(vb + c0), ld_shared_v4(vb + 128 + c1), ld_shared_v4(vb + 8 * 128 + c0), ld_shared_v4(vb + 9 * 128 + c1)};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const uint32_t k0 = w == 0 ? v[0].x : w == 1 ? v[0].y : w == 2 ? v[0].z : v[0].w;
                        const uint32_t k1 = w == 0 ? v[1].x : w == 1 ? v[1].y : w == 2 ? v[1].z : v[1].w;
                        const uint32_t k2 = w == 0 ? v[2].x : w == 1 ? v[2].y : w == 2 ? v[2].z : v[2].w;
                        const uint32_t k3 = w == 0 ? v[3].x : w == 1 ? v[3].y : w == 2 ? v[3].z : v[3].w;
                        if constexpr (FP8) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const uint32_t x01 = prmt(k0, k1, h ? 0x7362 : 0x5140), x23 = prmt(k2, k3, h ? 0x7362 : 0x5140);
                                const uint32_t a[4] = {e4m3x2_to_f16x2((uint16_t)x01), e4m3x2_to_f16x2((uint16_t)(x01 >> 16)),
                                                       e4m3x2_to_f16x2((uint16_t)x23), e4m3x2_to_f16x2((uint16_t)(x23 >> 16))};
#pragma unroll
                                for (int s = 0; s < NS; ++s) mma_f16(acc[s][c * 8 + w * 2 + h], a, pb[s][0], pb[s][1]);
                            }
                        } else {
                            const uint32_t a[4] = {prmt(k0, k1, 0x5410), prmt(k0, k1, 0x7632), prmt(k2, k3, 0x5410), prmt(k2, k3, 0x7632)};
#pragma unroll
                            for (int s = 0; s < NS; ++s) mma_bf16(acc[s][c * 4 + w], a, pb[s][0], pb[s][1]);
                        }
                    }
                }
            }
            __syncwarp();                                              // the stage may be refilled
        }
        if (!ok) {                                                     // no copy may land in the exchange below, or after the CTA has left
            for (int s = 0; s < STAGES; ++s)
                if ((armed ^ phases) >> s & 1u) mbar_drain(&full[s], (phases >> s) & 1u);
            armed = phases;
        }
        // every step of this sequence has been consumed: on to the next one that has some in this CTA's piece
        do ++seq; while (seq < p.b.n_seqs && sm_cnt[seq + 1] <= sm_cnt[seq]);
        const bool more = seq < p.b.n_seqs && sm_cnt[seq] + PS_TURN < hi;
        if (more) begin();

        // ---- join the four warps through their rings and write the piece's partial
#pragma unroll
        for (int x = 0; x < NS * 2; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 4);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 8);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 16);
            if (g == 0) {
                float *ml = sm_ml + (warp * 8 * NS + (x >> 1) * 8 + 2 * t + (x & 1)) * 2;
                ml[0] = ref[x];
                ml[1] = l[x];
            }
        }
        // a lane's accumulators as 16-byte pieces of consecutive dims: [slice][column parity][chunk c][piece f]
        constexpr int PIECES = (FP8 ? 16 : 8) / 4, QUADS = 2 * VC * PIECES;
        float4 *red = reinterpret_cast<float4 *>(ps_smem + warp * C::RING);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int c = 0; c < VC; ++c)
#pragma unroll
                    for (int f = 0; f < PIECES; ++f) {
                        const int a = c * 2 * PIECES + f * 2;          // two row tiles hold four consecutive dims
                        red[(s * QUADS + (e * VC + c) * PIECES + f) * 32 + lane] = make_float4(acc[s][a][e], acc[s][a][e + 2], acc[s][a + 1][e], acc[s][a + 1][e + 2]);
                    }
        __syncthreads();
        const long long slot = (long long)hg * (p.ctas + p.b.n_seqs) + blockIdx.x + now;
        for (int x = warp; x < NS * QUADS; x += PS_WARPS) {
            const int s = x / QUADS, e = (x / (VC * PIECES)) & 1, c = (x / PIECES) % VC, f = x % PIECES;
            const int col = s * 8 + 2 * t + e;
            float m4[PS_WARPS], mx = -INFINITY;
#pragma unroll
            for (int w = 0; w < PS_WARPS; ++w) { m4[w] = sm_ml[(w * 8 * NS + col) * 2]; mx = fmaxf(mx, m4[w]); }
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
            float lt = 0.f;
#pragma unroll
            for (int w = 0; w < PS_WARPS; ++w) {
                const float al = m4[w] == -INFINITY ? 0.f : fast_exp2(m4[w] - mx);
                const float4 v = reinterpret_cast<const float4 *>(ps_smem + w * C::RING)[x * 32 + lane];
                o.x = fmaf(v.x, al, o.x); o.y = fmaf(v.y, al, o.y); o.z = fmaf(v.z, al, o.z); o.w = fmaf(v.w, al, o.w);
                lt = fmaf(sm_ml[(w * 8 * NS + col) * 2 + 1], al, lt);
            }
            if (r0 + col < rows) {
                const int dim = (g + 8 * c) * (FP8 ? 16 : 8) + f * 4;
                *reinterpret_cast<float4 *>(p.part_acc + (slot * 8 * NS + col) * D + dim) = o;
                if (c == 0 && f == 0 && g == 0) *reinterpret_cast<float2 *>(p.part_ml + (slot * 8 * NS + col) * 2) = make_float2(mx, lt);
            }
        }
        if (!more) break;
        fence_async_smem();                                            // (the exchange area is refilled by TMA)
        __syncthreads();
    }
    pdl_wait();
}

// Joins the partials of a query row: plan[1] - plan[0] + 1 pieces of the scan, then those of the prefix.  WPR warps share a
// row; each of them finds the weights exp2(m - max) of all pieces, 32 at a time, one per lane, and adds up every
// WPR-th piece with four of them requested at once.  A few KB per row, from L2: bound by the latency of plan -> (m, l) -> acc.
template <int D, int WPR>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttnParams p, const int ns) {
    constexpr int EPT = D / 32, RPC = 8 / WPR;
    __shared__ float sm_o[WPR > 1 ? 8 * D : 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WPR;
    const long long row = (long long)blockIdx.x * RPC + warp / WPR;        // (sequence, token, head)
    const bool row_ok = row < (long long)p.b.n_seqs * p.m * p.hq;
    pdl_wait();
    pdl_launch_dependents();
    const int h = (int)(row % p.hq), i = (int)(row / p.hq % p.m), seq = row_ok ? (int)(row / p.hq / p.m) : 0;
    const int j = h / p.g, r = i * p.g + h % p.g, grp = r / (8 * ns), col = r % (8 * ns);
    const int c0 = p.plan[2 * seq], n_scan = p.plan[2 * seq + 1] - c0 + 1;
    const int n = !row_ok || load_len(p.b, seq) < 0 ? 0 : n_scan + p.splits;
    const long long slot0 = ((long long)(grp * p.c.hkv + j) * (p.ctas + p.b.n_seqs) + seq + c0) * 8 * ns + col;
    const long long px0 = ((long long)j * p.b.n_seqs + seq) * p.g * p.m + r, px_step = (long long)p.c.hkv * p.b.n_seqs * p.g * p.m;
    float mx = -INFINITY, l = 0.f, o[EPT];
#pragma unroll
    for (int e = 0; e < EPT; ++e) o[e] = 0.f;
    for (int base = 0; base < n; base += 32) {
        const int x = base + lane;
        float2 ml = make_float2(-INFINITY, 0.f);
        const float *acc = nullptr;
        if (x < n_scan) {
            const long long at = slot0 + (long long)x * 8 * ns;
            ml = *reinterpret_cast<const float2 *>(p.part_ml + at * 2);
            acc = p.part_acc + at * D;
        } else if (x < n) {
            const long long at = px0 + (x - n_scan) * px_step;
            ml = *reinterpret_cast<const float2 *>(p.px_ml + at * 2);
            acc = p.px_acc + at * D;
        }
        const float m_new = fmaxf(mx, warp_max(ml.x));
        const float w = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - m_new);
        const float alpha = mx == -INFINITY ? 0.f : fast_exp2(mx - m_new);
        l = l * alpha + warp_sum(ml.y * w);
#pragma unroll
        for (int e = 0; e < EPT; ++e) o[e] *= alpha;
        mx = m_new;
        if (ml.y == 0.f) acc = nullptr;                                    // a piece without keys: its acc is not written
        const int here = min(32, n - base);
        for (int x0 = sub; x0 < here; x0 += 4 * WPR) {
            float4 v[4][EPT / 4];
            float wx[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int from = x0 + y * WPR;
                const unsigned long long a = __shfl_sync(0xffffffffu, (unsigned long long)acc, from & 31);
                wx[y] = __shfl_sync(0xffffffffu, w, from & 31);
                const bool ok = from < here && a != 0;
                const float4 *src = reinterpret_cast<const float4 *>(a) + lane * (EPT / 4);
#pragma unroll
                for (int e = 0; e < EPT / 4; ++e) v[y][e] = ok ? src[e] : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int e = 0; e < EPT / 4; ++e) {
                    const float wy = x0 + y * WPR < here ? wx[y] : 0.f;
                    o[e * 4] = fmaf(v[y][e].x, wy, o[e * 4]); o[e * 4 + 1] = fmaf(v[y][e].y, wy, o[e * 4 + 1]);
                    o[e * 4 + 2] = fmaf(v[y][e].z, wy, o[e * 4 + 2]); o[e * 4 + 3] = fmaf(v[y][e].w, wy, o[e * 4 + 3]);
                }
        }
    }
    if constexpr (WPR > 1) {                                               // the row's warps, in order
#pragma unroll
        for (int e = 0; e < EPT; ++e) sm_o[warp * D + e * 32 + lane] = o[e];
        __syncthreads();
        if (sub != 0) return;
#pragma unroll
        for (int y = 1; y < WPR; ++y)
#pragma unroll
            for (int e = 0; e < EPT; ++e) o[e] += sm_o[(warp + y) * D + e * 32 + lane];
    }
    if (!row_ok) return;
    const float inv = l == 0.f ? 0.f : __fdiv_rn(1.f, l);                 // a row that sees no key is zero
    __nv_bfloat16 ob[EPT];
#pragma unroll
    for (int e = 0; e < EPT; ++e) ob[e] = __float2bfloat16_rn(o[e] * inv);
    if (p.gate) {
        const __nv_bfloat16 *gp = p.gate + ((long long)seq * p.m + i) * p.gate_rs + h * p.gate_hs + lane * EPT;
#pragma unroll
        for (int e = 0; e < EPT; ++e) {
            const __nv_bfloat16 sg = __float2bfloat16_rn(__fdiv_rn(1.f, 1.f + __expf(-__bfloat162float(gp[e]))));
            ob[e] = __float2bfloat16_rn(__bfloat162float(ob[e]) * __bfloat162float(sg));
        }
    }
    __nv_bfloat16 *dst = p.out + row * D + lane * EPT;
    if (EPT == 8) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(ob);
    else *reinterpret_cast<uint2 *>(dst) = *reinterpret_cast<const uint2 *>(ob);
}

// Bytes that the scans of all sequences would read of the prefix from which on it is read once, by a kernel of its own.  Its rows are those of
// prefix_len where the host knows it; a length on the device counts as a full table (the launches are chosen before it can be read).  That kernel costs 8
// to 12 us before it pays.  Measured with / without it (us; own rows 100 - 300): 24/4 heads x 256 e4m3, 8 sequences over 4096 rows (68 MB)
// 23.4 / 20.6, 16 over 4096 (136 MB) 25.5 / 29.3, 32 over 16384 43 / 137; bf16 4 over 4096 (67 MB) 17.6 / 17.1, 8 over 4096 (134 MB) 19.5 / 25.2;
// 32/8 x 128 e4m3, 8 over 4096 (69 MB) 19.8 / 20.7; 16/16 x 128 bf16, 8 over 1024 (67 MB) 16.0 / 16.1; 32 over 256 (33 MB) 24.7 / 17.8.
constexpr long long PREFIX_BYTES = 72LL << 20;
static std::atomic<long long> g_prefix_bytes{PREFIX_BYTES};

// How a call is cut: query-row slices per CTA, row groups, CTAs per (kv head, group), pieces of the prefix and blocks of 128 query
// rows of its kernel (0: the scan reads the prefix itself), and where the partials lie.
struct PagedAttnPlan {
    int ns, groups, ctas, splits, blocks;
    size_t off_ml, off_acc, off_px_ml, off_px_acc, bytes;
};
static PagedAttnPlan paged_attn_plan(int d, bool fp8, int hkv, int hq, int n_seqs, int m, long long prefix_rows) {
    PagedAttnPlan o;
    const int rows = hq / hkv * m;
    o.ns = rows <= 8 ? 1 : 2;
    o.groups = (rows + 8 * o.ns - 1) / (8 * o.ns);
    const int per_sm = o.ns == 1 ? (d == 256 ? (fp8 ? ScanCfg<256, true, 1>::CTAS : ScanCfg<256, false, 1>::CTAS)
                                             : (fp8 ? ScanCfg<128, true, 1>::CTAS : ScanCfg<128, false, 1>::CTAS))
                                 : (d == 256 ? (fp8 ? ScanCfg<256, true, 2>::CTAS : ScanCfg<256, false, 2>::CTAS)
                                             : (fp8 ? ScanCfg<128, true, 2>::CTAS : ScanCfg<128, false, 2>::CTAS));
    o.ctas = std::max(1, sm_count() * per_sm / (hkv * o.groups));
    o.splits = o.blocks = 0;
    const double scanned = (double)n_seqs * o.groups * prefix_rows * hkv * (fp8 ? 2 * d + 8 : 4 * d);
    if (prefix_rows > 0 && n_seqs > 1 && scanned >= (double)g_prefix_bytes) {
        const int tile = fp8 || d == 128 ? 128 : 64;
        const long long tiles = (prefix_rows + tile - 1) / tile;
        o.blocks = (int)(((long long)n_seqs * rows + 127) / 128);
        const int units = o.blocks * hkv;
        // one wave of CTAs, and at least two tiles for each
        o.splits = (int)std::max(1LL, std::min((long long)sm_count() / units, tiles / 2));
    }
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    const size_t slots = (size_t)hkv * o.groups * (o.ctas + n_seqs) * 8 * o.ns, px = (size_t)o.splits * hkv * n_seqs * rows;
    o.off_ml = up((size_t)n_seqs * 8);
    o.off_acc = up(o.off_ml + slots * 8);
    o.off_px_ml = up(o.off_acc + slots * d * 4);
    o.off_px_acc = up(o.off_px_ml + px * 8);
    o.bytes = up(o.off_px_acc + px * d * 4);
    return o;
}

template <typename C>
static int launch_prefix(const PagedAttnParams &p, const PagedAttnPlan &plan, cudaStream_t st) {
    static bool attr_set[64] = {};
    int dev = 0, rc;
    TRB_CUDA_CHECK(cudaGetDevice(&dev));
    if (!attr_set[dev & 63]) {
        TRB_CUDA_CHECK(cudaFuncSetAttribute(paged_prefix_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        attr_set[dev & 63] = true;
    }
    PrefixParams x;
    x.c = p.c; x.q = p.q; x.n_seqs = p.b.n_seqs; x.m = p.m; x.hq = p.hq; x.g = p.g; x.scale_log2 = p.scale_log2;
    x.table = p.prefix_table; x.pages = p.prefix_pages; x.len = p.prefix_len;
    x.splits = plan.splits; x.blocks = plan.blocks; x.part_ml = const_cast<float *>(p.px_ml); x.part_acc = const_cast<float *>(p.px_acc);
    // the pool as [num_pages * hkv][page_size] rows; a box is a page, or a tile of a larger page
    CUtensorMap mk, mv;
    const int page = 1 << p.c.page_shift, box = std::min(page, (int)C::BN);
    if ((rc = get_row_tile_map(p.c.k, page, (int)(p.c.num_pages * p.c.hkv), C::ROWB, box, &mk))) return rc;
    if ((rc = get_row_tile_map(p.c.v, page, (int)(p.c.num_pages * p.c.hkv), C::ROWB, box, &mv))) return rc;
    TRB_CUDA_CHECK(launch_kernel(paged_prefix_kernel<C>, dim3((unsigned)plan.splits * plan.blocks * p.c.hkv), dim3(PX_THREADS), C::SMEM, st, true, mk, mv, x));
    return TRB_OK;
}

template <typename C>
static int launch_scan(const PagedAttnParams &p, cudaStream_t st) {
    static bool attr_set[64] = {};
    int dev = 0, rc;
    TRB_CUDA_CHECK(cudaGetDevice(&dev));
    if (!attr_set[dev & 63]) {
        TRB_CUDA_CHECK(cudaFuncSetAttribute(paged_scan_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
        attr_set[dev & 63] = true;
    }
    CUtensorMap mk, mv;
    if ((rc = get_row_tile_map(p.c.k, 1 << p.c.page_shift, (int)(p.c.num_pages * p.c.hkv), C::ROWB, 16, &mk))) return rc;
    if ((rc = get_row_tile_map(p.c.v, 1 << p.c.page_shift, (int)(p.c.num_pages * p.c.hkv), C::ROWB, 16, &mv))) return rc;
    TRB_CUDA_CHECK(launch_kernel(paged_scan_kernel<C>, dim3(p.ctas, p.c.hkv * p.groups), dim3(PS_THREADS), C::SMEM, st, true, mk, mv, p));
    return TRB_OK;
}

}  // namespace trb

using namespace trb;

static int check_paged_geometry(const trb_paged_t *pool, int n_seqs, int m, int hq, int prefix_pages) {
    if (n_seqs < 1 || m < 1 || hq < 1 || prefix_pages < 0 || hq % pool->hkv) return TRB_E_ARG;
    if (n_seqs > PG_MAX_SEQS || (long long)(hq / pool->hkv) * m > 128) return TRB_E_UNSUPPORTED;
    return TRB_OK;
}

extern "C" int trb_set_paged_prefix_bytes(int64_t min_bytes) {
    g_prefix_bytes.store(min_bytes < 0 ? PREFIX_BYTES : min_bytes);
    return TRB_OK;
}

extern "C" size_t trb_attn_paged_workspace_bytes(const trb_paged_t *pool, int32_t n_seqs, int32_t m, int32_t hq, int32_t prefix_pages) {
    PagedView v;
    if (make_paged_view(pool, &v) || check_paged_geometry(pool, n_seqs, m, hq, prefix_pages)) return 0;
    return paged_attn_plan(pool->d, v.ks != nullptr, pool->hkv, hq, n_seqs, m, (long long)prefix_pages << v.page_shift).bytes;
}

extern "C" int trb_attn_paged(const trb_paged_t *pool, const trb_batch_t *batch, const trb_attn_paged_args_t *a, trb_stream_t stream) {
    PagedAttnParams p;
    int rc = make_paged_view(pool, &p.c);
    if (rc || (rc = make_batch_view(batch, &p.b))) return rc;
    if (!a || !a->q || !a->out || !a->workspace || (a->prefix_pages > 0 && !a->prefix_table)) return TRB_E_ARG;
    if ((rc = check_paged_geometry(pool, batch->n_seqs, a->m, a->hq, a->prefix_pages))) return rc;
    if (a->prefix_pages > 0 && (rc = check_cursor(&a->prefix_len))) return rc;
    // rows are counted in 32 bits, with room for a step of tiles behind the last one
    if (((long long)a->prefix_pages + batch->table_pages) << p.c.page_shift > 0x7fffff00LL) return TRB_E_UNSUPPORTED;
    if (((((long long)a->prefix_pages + batch->table_pages) << p.c.page_shift) / 16 + 2 + PS_TURN) * batch->n_seqs > 0x7fffffffLL) return TRB_E_UNSUPPORTED;
    if ((((uintptr_t)a->q | (uintptr_t)a->out) & 15) || ((uintptr_t)a->workspace & 255) || ((uintptr_t)a->prefix_table & 3) || ((uintptr_t)a->gate & 1)) return TRB_E_ALIGN;
    const bool fp8 = p.c.ks != nullptr;
    long long prefix_rows = (long long)a->prefix_pages << p.c.page_shift;
    if (a->prefix_pages > 0 && !a->prefix_len.dev) prefix_rows = std::max(0LL, std::min(prefix_rows, (long long)a->prefix_len.host));
    const PagedAttnPlan plan = paged_attn_plan(pool->d, fp8, pool->hkv, a->hq, batch->n_seqs, a->m, prefix_rows);
    if (a->workspace_bytes < plan.bytes) return TRB_E_CAPACITY;
    p.q = (const __nv_bfloat16 *)a->q; p.out = (__nv_bfloat16 *)a->out; p.gate = (const __nv_bfloat16 *)a->gate;
    p.gate_rs = a->gate_row_stride; p.gate_hs = a->gate_head_stride;
    p.m = a->m; p.hq = a->hq; p.g = a->hq / pool->hkv; p.scale_log2 = a->scale * 1.4426950408889634f;
    p.prefix_table = a->prefix_table; p.prefix_pages = a->prefix_pages; p.prefix_len = make_cursor(&a->prefix_len);
    p.ctas = plan.ctas; p.groups = plan.groups;
    uint8_t *ws = (uint8_t *)a->workspace;
    p.plan = (int *)ws; p.part_ml = (float *)(ws + plan.off_ml); p.part_acc = (float *)(ws + plan.off_acc);
    p.px_ml = (const float *)(ws + plan.off_px_ml); p.px_acc = (const float *)(ws + plan.off_px_acc);
    p.splits = plan.splits; p.after_prefix = plan.splits > 0;
    cudaStream_t st = (cudaStream_t)stream;
    pdl_forget(st);
    if (plan.splits > 0) {
        rc = pool->d == 256 ? (fp8 ? launch_prefix<PrefixCfg<256, true>>(p, plan, st) : launch_prefix<PrefixCfg<256, false>>(p, plan, st))
                            : (fp8 ? launch_prefix<PrefixCfg<128, true>>(p, plan, st) : launch_prefix<PrefixCfg<128, false>>(p, plan, st));
        if (rc) return rc;
        p.prefix_pages = 0;                                               // the scan has the own rows alone
    }
    if (plan.ns == 1) rc = pool->d == 256 ? (fp8 ? launch_scan<ScanCfg<256, true, 1>>(p, st) : launch_scan<ScanCfg<256, false, 1>>(p, st))
                                          : (fp8 ? launch_scan<ScanCfg<128, true, 1>>(p, st) : launch_scan<ScanCfg<128, false, 1>>(p, st));
    else rc = pool->d == 256 ? (fp8 ? launch_scan<ScanCfg<256, true, 2>>(p, st) : launch_scan<ScanCfg<256, false, 2>>(p, st))
                             : (fp8 ? launch_scan<ScanCfg<128, true, 2>>(p, st) : launch_scan<ScanCfg<128, false, 2>>(p, st));
    if (rc) return rc;
    // as many warps per row as the SMs hold at once
    const long long out_rows = (long long)batch->n_seqs * a->m * a->hq, most = 24LL * sm_count() / out_rows;
    const int wpr = most >= 8 ? 8 : most >= 4 ? 4 : most >= 2 ? 2 : 1;
    const bool wide = pool->d == 256;
    auto *merge = wpr == 8 ? (wide ? paged_merge_kernel<256, 8> : paged_merge_kernel<128, 8>) : wpr == 4 ? (wide ? paged_merge_kernel<256, 4> : paged_merge_kernel<128, 4>)
                  : wpr == 2 ? (wide ? paged_merge_kernel<256, 2> : paged_merge_kernel<128, 2>) : (wide ? paged_merge_kernel<256, 1> : paged_merge_kernel<128, 1>);
    TRB_CUDA_CHECK(launch_kernel(merge, dim3((unsigned)((out_rows * wpr + 7) / 8)), dim3(256), 0, st, true, p, plan.ns));
    return TRB_OK;
}
