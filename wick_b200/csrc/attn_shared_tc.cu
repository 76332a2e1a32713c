// The shared keys of groups of sequences on the 5th-generation tensor cores (tcgen05), bfloat16, head sizes 64 and 128: a record
// (maximum, sum of weights, weighted sum of values) for every run of units of a tile of 128 rows (attn_shared.cuh).
//
// A tile's rows are query heads of one key head times the group's tokens, whatever sequences they belong to: all of them see all
// shared keys, so there is no mask anywhere.  A block of keys is a page.  There are two streams, each with its own sums and two places for
// scores in tensor memory (4 x 64 columns, and twice the head size) and four softmax warps, so that one stream's softmax runs beside the
// other's products, and a stream's softmax of one block beside the scores of its next:
//   * a group of more than 128 rows: two tiles of rows, a stream each, that share every tile of keys and values;
//   * the last tile of an odd number: even blocks of keys go to one stream, odd ones to the other, joined when the run ends.
// Roles:
//   * a producer warp fetches the query rows of a run and its key and value tiles through a ring (TMA, 128-byte swizzle, first to leave the
//     L2 cache: each is read once for 256 rows, and the records, which are read again, stay there; 24 sequences behind 31,000 positions 60.7
//     and 55.6 us);
//   * an issuing lane alternates between the streams: O += P V of one, then the scores S = Q K^T of its block after the next (P lies over
//     the scores it came from, as bfloat16 pairs).  It waits by itself, without votes, and arrives once a block for both of its tiles:
//     with a whole warp's votes and an arrival for each tile and product a turn took 1,400 clocks, of which 580 were its instructions;
//   * a softmax thread owns a row.  O and the sum are scaled by a maximum that follows the true one lazily: O is rescaled only when a
//     block's maximum exceeds it by more than 8 (in units of log2 e).  Warps whose rows are all beyond the group's tokens compute nothing.
//     Weights enter the second product rounded to bfloat16, as its operand has to be; their sum, in 32 bits, is of the unrounded ones but for
//     each block's largest, whose rounding would else show: it is not 1 where the maximum lags.  (64 behind 8,192, error against 64 bits:
//     0.00215 of unrounded ones, 0.00209 so, 0.00209 of rounded ones, whose sum took 4 % longer behind 31,000 positions, this 1 %.)
// REHEARSE: a run has few blocks, and a block's code is met for the first time while all SMs fill their rings: instructions then
// come through the same queues as 24 MB of keys and values, and the first block's softmax took 4,300 clocks.  So the softmax warps go through
// their code once while there is nothing to do yet.  (The issuing lane does not: it changed nothing.)
// What bounds it: the start of a run (10 to 15 thousand clocks until four turns are through, of which the kernel before hides 4), then the
// tensor pipe, 830 clocks a turn of 12 products (64 keys of a stream; the softmax beside it 550; scores of 64 columns cost as much as of
// 128, but with 128 there is room for one place each, and a stream then stands still between its softmax and its next scores: 1,100).  64
// sequences behind 8,192 positions, 32 heads over 8 of 128, on 83 SMs: 24.8 us; 24 behind 31,000, 64 over 8, on 128 SMs: 46 us.
// (Measured and left: an issuing warp for either stream, 1 to 2 % of long runs and as much slower short ones.)
// Every wait is bounded and reports through the status word (code 7).
#include "tc_attention.cuh"
#include "attn_shared.cuh"

#ifndef WICK_HD
#error "compile with -DWICK_HD=<head_dim>"
#endif

namespace wick {
namespace shared_prefix {

namespace tc {

constexpr bool SUPPORTED = WICK_HD == 64 || WICK_HD == 128;
constexpr int HD = SUPPORTED ? WICK_HD : 64;           // other head sizes: never launched
constexpr int BQ = TC_ROWS, BK = kPage;
constexpr int PANELS = HD / 64;                        // 64-column panels of a head row
constexpr int Q_PANEL = BQ * 128, KV_PANEL = BK * 128; // bytes: rows of 128
constexpr int Q_BYTES = PANELS * Q_PANEL, KV_BYTES = PANELS * KV_PANEL;        // a tile of queries, of keys or of values
constexpr int NSLOT = 5;                               // pairs of a value and a key tile in flight
constexpr int AHEAD = 4;                               // turns that the scores are ahead of the products (two a stream)
constexpr int THREADS = 320;                           // warp 0: TMA, warp 1: MMA + tensor memory, warps 2-5 and 6-9: softmax
constexpr uint32_t TMEM_COLS = 512;                    // S of both streams | O of both
constexpr uint32_t COL_S = 0, COL_O = 4 * BK;          // S: two of either stream
constexpr int REC = BQ * (HD + 2);

struct Smem {
    float ml[2][2][BQ];                                // the streams' maxima and sums
    uint64_t q_full, q_empty, full[NSLOT], empty[NSLOT], s_full[2][2], p_full[2][2], before_last[2], o_full[2], o_empty[2], join, joined;
    uint32_t tmem_slot;
    int abort_flag;
};
constexpr int SMEM_BYTES = 2 * Q_BYTES + NSLOT * 2 * KV_BYTES + (int)sizeof(Smem);
static_assert(SMEM_BYTES <= 227 * 1024, "a block's shared memory");

__global__ void __launch_bounds__(THREADS, 1)
attn_shared_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap kv_map, const Groups G, int64_t kv_pages, float scale,
                      int* plan, float* records, int* status) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* q_s = smem_raw;
    uint8_t* kv_s = q_s + 2 * Q_BYTES;
    Smem& sh = *reinterpret_cast<Smem*>(kv_s + NSLOT * 2 * KV_BYTES);
    volatile int* abort_flag = &sh.abort_flag;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        sh.abort_flag = 0;
        mbar_init(&sh.q_full, 1), mbar_init(&sh.q_empty, 1);
        for (int i = 0; i < NSLOT; ++i) mbar_init(&sh.full[i], 1), mbar_init(&sh.empty[i], 1);
        // (every waiter below sees every phase of the barrier it waits on, so that a parity is never ambiguous)
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.o_full[i], 1), mbar_init(&sh.o_empty[i], 4), mbar_init(&sh.before_last[i], 1);
            for (int b = 0; b < 2; ++b) mbar_init(&sh.s_full[i][b], 1), mbar_init(&sh.p_full[i][b], 4);
        }
        mbar_init(&sh.join, 8), mbar_init(&sh.joined, 8);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0 && lane < 2) {
        const CUtensorMap* map = lane == 0 ? &q_map : &kv_map;
        asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_slot)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // (The description lies ready before the step's kernels start; the plan is written behind the wait.)
    Runs runs(G, gridDim.x);                           // (every warp knows them on its own)
    Segment seg;
    // The producer's lanes hold a page number of each of two runs of 32, read ahead.
    auto pages = [&](int run) {
        const int j = seg.from + run * 32 + lane;
        int page = j < seg.to ? G.page_table[(int64_t)seg.cut.seq * G.table_width + j] : 0;
        if (page < 0 || page >= kv_pages) {
            atomicCAS(status, 0, 10);
            page = 0;
        }
        return page;
    };
    int even = 0, odd = 0;
    if (warp == 0 && blockIdx.x < runs.all) seg = runs.segment(blockIdx.x), even = pages(0), odd = pages(1);
    pdl_wait();
    pdl_trigger();                                     // (behind the wait: the next kernel reads what this one reads without a wait of its own)
    if (blockIdx.x == 0 && warp == 2) Runs(G, gridDim.x).write(plan, status);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_slot;
    const bool aligned = (smem_u32(smem_raw) & 1023) == 0;   // (always: the block's dynamic shared memory is all there is)
    if (!aligned && threadIdx.x == 0) atomicCAS(status, 0, 7);
    int k = 0;                                         // runs so far
    bool ok = aligned;

    if (warp == 0) {
        // ---------------- producer ----------------
        const bool one = elect_one();
        int slot = 0, turn = 0;                        // of the ring
        const uint64_t policy = read_once_policy();
#pragma unroll 1
        for (int at = blockIdx.x; ok && at < runs.all; at += gridDim.x, ++k) {
            if (k > 0) seg = runs.segment(at), even = pages(0), odd = pages(1);
            const int n = seg.to - seg.from;
            const bool split = seg.tiles == 1;
            if (k > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.q_empty, (k - 1) & 1, abort_flag, status, 7));
            if (!ok) break;
            if (one) {
                mbar_expect_tx(&sh.q_full, seg.tiles * PANELS * G.rows * 128);
                for (int i = 0; i < seg.tiles; ++i)
                    for (int pn = 0; pn < PANELS; ++pn)
                        tma_load_3d(&q_map, &sh.q_full, q_s + i * Q_BYTES + pn * Q_PANEL, pn * 64, seg.column * G.gs,
                                    seg.cut.tok0 + (seg.tile + i) * (G.rows / G.gs));
            }
            // A slot: the values of block i beside the keys of the block that the issuing warp scores in the same turn.
            const int ahead = split ? AHEAD : AHEAD / 2;
#pragma unroll 1
            for (int i = -ahead; i < n; ++i) {
                if (turn > 0) ok = __all_sync(0xffffffffu, mbar_wait(&sh.empty[slot], (turn - 1) & 1, abort_flag, status, 7));
                if (!ok) break;
                const int j = i + ahead, v = max(i, 0);
                const int k_page = __shfl_sync(0xffffffffu, j >> 5 & 1 ? odd : even, j & 31), v_page = __shfl_sync(0xffffffffu, v >> 5 & 1 ? odd : even, v & 31);
                if (i >= 32 && (i & 31) == 0) {        // (keys and values have left the run before)
                    if (i >> 5 & 1) even = pages((i >> 5) + 1);
                    else odd = pages((i >> 5) + 1);
                }
                if (one) {
                    mbar_expect_tx(&sh.full[slot], ((i >= 0) + (j < n)) * KV_BYTES);
#pragma unroll 1
                    for (int is_v = 0; is_v < 2; ++is_v) {
                        if (is_v ? i < 0 : j >= n) continue;
                        const int y = (((is_v ? v_page : k_page) * 2 + is_v) * G.kv_heads + seg.column / G.per_kv) * kPage;
                        for (int pn = 0; pn < PANELS; ++pn)
                            tma_load_2d(&kv_map, &sh.full[slot], kv_s + (2 * slot + is_v) * KV_BYTES + pn * KV_PANEL, pn * 64, y, policy);
                    }
                }
                if (++slot == NSLOT) slot = 0, ++turn;
                __syncwarp();
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer ----------------
        // (One lane by itself, without a vote or a shuffle: what it does between its instructions bounds the kernel.)
        const uint32_t idesc_s = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BK >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
        const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
        const uint32_t q_lo0 = desc_lo(smem_u32(q_s), 16), k_lo0 = desc_lo(smem_u32(kv_s), 16), v_lo0 = desc_lo(smem_u32(kv_s) + KV_BYTES, KV_PANEL);
        const bool one = elect_one();
        int slot = 0, round = 0;                       // of the ring
        int scores[2] = {0, 0}, steps[2] = {0, 0}, uses[2] = {0, 0};           // scores, products and runs of each stream so far
#pragma unroll 1
        for (int at = blockIdx.x; ok && at < runs.all; at += gridDim.x, ++k) {
            seg = runs.segment(at);
            const int n = seg.to - seg.from;
            const bool split = seg.tiles == 1;
            const int N = split ? n : 2 * n;           // turns
            // turn i: stream i & 1's product of one block, then its scores of the block after the next.
            auto turn = [&](int i, auto stream) {
                constexpr int s = (int)stream;
                if (split || s == 0) {
                    if (!mbar_wait(&sh.full[slot], round & 1, abort_flag, status, 7)) return false;
                }
                if (i >= 0) {
                    const int at_s = steps[s] & 1;
                    // (the sums of the stream's run before have been read)
                    if (i < 2 && uses[s] > 0 && !mbar_wait(&sh.o_empty[s], (uses[s] - 1) & 1, abort_flag, status, 7)) return false;
                    if (!mbar_wait(&sh.p_full[s][at_s], (steps[s] >> 1) & 1, abort_flag, status, 7)) return false;
                    tc_fence_after();
                    const uint32_t vp = v_lo0 + slot * (2 * KV_BYTES >> 4), pp = tmem + COL_S + (2 * s + at_s) * BK, d = tmem + COL_O + s * HD;
                    mma_ts(d, pp, vp, idesc_o, i >= 2);
                    static_for<1, BK / 16>([&](auto ks) { mma_ts(d, pp + (int)ks * 8, vp + (int)ks * (2048 >> 4), idesc_o, 1); });
                    ++steps[s];
                    if (i + 2 >= N) tc_commit(&sh.o_full[s]), ++uses[s];
                    else if (i + 4 >= N) tc_commit(&sh.before_last[s]);
                }
                if (i + AHEAD < N) {
                    const int at_s = scores[s] & 1;
                    if (i < 0) tc_fence_after();
                    const uint32_t k_lo = k_lo0 + slot * (2 * KV_BYTES >> 4), q_lo = q_lo0 + (split ? 0 : s * (Q_BYTES >> 4));
                    const uint32_t d = tmem + COL_S + (2 * s + at_s) * BK;
                    static_for<0, HD / 16>([&](auto ks) {
                        constexpr uint32_t in = ((int)ks & 3) * 32, pn = (int)ks >> 2;
                        mma_ss<((int)ks > 0)>(d, q_lo + ((pn * Q_PANEL + in) >> 4), k_lo + ((pn * KV_PANEL + in) >> 4), idesc_s);
                    });
                    tc_commit(&sh.s_full[s][at_s]);
                    ++scores[s];
                    if (i + AHEAD == N - 1) tc_commit(&sh.q_empty);            // (the run's last scores)
                }
                if (split || s == 1) {
                    tc_commit(&sh.empty[slot]);        // (behind the last reader of both tiles)
                    if (++slot == NSLOT) slot = 0, ++round;
                }
                return true;
            };
            if (one) {
                ok = mbar_wait(&sh.q_full, k & 1, abort_flag, status, 7);
#pragma unroll 1
                for (int i = -AHEAD; ok && i < N; i += 2) {
                    ok = turn(i, std::integral_constant<int, 0>{});
                    if (ok && i + 1 < N) ok = turn(i + 1, std::integral_constant<int, 1>{});
                }
            }
            ok = __any_sync(0xffffffffu, one && ok);
        }
    } else {
        // ---------------- softmax: a row per thread ----------------
        // (a warp reads the 32 lanes of tensor memory given by its index modulo 4)
        const int quad = warp & 3, s = (warp - 2) >> 2;
        const int r = quad * 32 + lane;
        const float sl2 = scale * 1.4426950408889634f;
        const uint32_t lane_base = tmem + ((uint32_t)(quad * 32) << 16);
        const uint32_t o_addr = lane_base + COL_O + s * HD;
        int step = 0, lasts = 0, uses0 = 0, uses1 = 0, joins = 0;  // this stream's blocks, its runs of two blocks or more, both streams' runs, joins so far
#pragma unroll 1
        for (int at = blockIdx.x; ok && at < runs.all; at += gridDim.x, ++k) {
            seg = runs.segment(at);
            const int n = seg.to - seg.from;
            const bool split = seg.tiles == 1;
            const int tile = seg.tile + (split ? 0 : s), n_rows = min(G.rows, seg.cut.n_tok * G.gs - tile * G.rows);
            const bool store = r < n_rows, busy = quad * 32 < n_rows;
            const int dj = split ? 2 : 1;
            float m = -INFINITY, l = 0.f;              // what O and the sum are scaled by (it follows the maximum lazily), the sum
#pragma unroll 1
            for (int j = (split ? s : 0) - (k == 0 ? dj : 0); j < n; j += dj) {
                const bool rehearsed = j < 0, first = j < dj;      // (a block before the first: see REHEARSE)
                const int at_s = step & 1;
                const uint32_t s_addr = lane_base + COL_S + (2 * s + at_s) * BK;
                if (!rehearsed) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.s_full[s][at_s], (step >> 1) & 1, abort_flag, status, 7));
                    if (!ok) break;
                    ++step;
                }
                tc_fence_after();
                auto hand_over = [&]() {
                    if (rehearsed) return;
                    tc_st_wait();
                    tc_fence_before();                 // P and the rescaled O before it multiplies and accumulates
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.p_full[s][at_s]);
                };
                if (!first && !rehearsed && j + dj >= n) {             // (no scores come behind the last block's: its rescaling waits here)
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.before_last[s], lasts & 1, abort_flag, status, 7));
                    if (!ok) break;
                    ++lasts;
                }
                if (!busy) {
                    hand_over();
                    continue;
                }
                float y[BK];
                tc_ld32_nowait(s_addr, reinterpret_cast<uint32_t*>(y));
                tc_ld32_nowait(s_addr + 32, reinterpret_cast<uint32_t*>(y + 32));
                tc_ld_wait();
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < BK; i += 8) {
                    mx4[0] = max3(mx4[0], y[i], y[i + 1]);
                    mx4[1] = max3(mx4[1], y[i + 2], y[i + 3]);
                    mx4[2] = max3(mx4[2], y[i + 4], y[i + 5]);
                    mx4[3] = max3(mx4[3], y[i + 6], y[i + 7]);
                }
                const float most = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])), mx = most * sl2;
                const bool grow = mx > m + 8.0f;
                float alpha = 1.0f;
                if (grow) {
                    alpha = ex2(m - mx);               // 0 for the first block
                    m = mx;
                }
                const float neg_m = m == -INFINITY ? 0.f : -m;
                if (!first && __any_sync(0xffffffffu, grow)) {
                    // Rare.  O must hold the product of the block before, which the next block's scores come behind.
                    if (j + dj < n) ok = __all_sync(0xffffffffu, mbar_wait(&sh.s_full[s][at_s ^ 1], (step >> 1) & 1, abort_flag, status, 7));
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        tc_ld16(o_addr + c, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] *= alpha;
                        tc_st16(o_addr + c, reinterpret_cast<uint32_t*>(o));
                    }
                }
                float2 sum2[4] = {{0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}, {0.f, 0.f}};
                const float2 sl2_2 = make_float2(sl2, sl2), neg_m2 = make_float2(neg_m, neg_m);
#pragma unroll
                for (int c = 0; c < BK; c += 32) {
                    uint32_t packed[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 e = fma2(make_float2(y[c + i], y[c + i + 1]), sl2_2, neg_m2);
                        const float2 p = make_float2(ex2(e.x), ex2(e.y));
                        sum2[(i >> 1) & 3] = add2(sum2[(i >> 1) & 3], p);
                        const __nv_bfloat162 h = __floats2bfloat162_rn(p.x, p.y);      // key 2k in the low half, key 2k + 1 in the high half
                        packed[i >> 1] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    if (!rehearsed) tc_st16(s_addr + c / 2, packed);
                }
                hand_over();
                const float big = ex2(fmaf(most, sl2, neg_m));         // (the block's largest weight, the same bits as above)
                l = l * alpha + (__bfloat162float(__float2bfloat16_rn(big)) - big);
                l += (((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y)) + ((sum2[2].x + sum2[2].y) + (sum2[3].x + sum2[3].y)));
                if (rehearsed) m = -INFINITY, l = 0.f;
            }
            if (!ok) break;
            // The record: [HD / 4][128] groups of four sums, [128] pairs of maximum and sum.
            float* rec = records + (int64_t)(seg.record * G.pair + tile - seg.tile) * REC;
            auto put = [&](int c, const float* v) {    // 32 numbers of the row from column c on
                if (store) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(rec + ((c + i) / 4 * BQ + r) * 4) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            };
            if (!split || n == 1) {
                // the row is the stream's own (of one block: the even stream's)
                if (!split || s == 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_full[s], (s == 0 ? uses0 : uses1) & 1, abort_flag, status, 7));
                    if (!ok) break;
                    tc_fence_after();
                    if (busy) {
                        if (store) *reinterpret_cast<float2*>(rec + BQ * HD + 2 * r) = make_float2(m, l);
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            float v[32];
                            tc_ld32_nowait(o_addr + c, reinterpret_cast<uint32_t*>(v));
                            tc_ld_wait();
                            put(c, v);
                            __syncwarp();
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.o_empty[s]);    // (read before the next run's product writes)
                }
                ++uses0, uses1 += split ? 0 : 1;
                continue;
            }
            // both streams hold a part of every row: each stream's warps make half of the columns
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_full[0], uses0 & 1, abort_flag, status, 7) && mbar_wait(&sh.o_full[1], uses1 & 1, abort_flag, status, 7));
            if (!ok) break;
            ++uses0, ++uses1;
            sh.ml[s][0][r] = m;
            sh.ml[s][1][r] = l;
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.join);
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.join, joins & 1, abort_flag, status, 7));
            if (!ok) break;
            tc_fence_after();
            if (busy) {
                const float m0 = sh.ml[0][0][r], m1 = sh.ml[1][0][r], mm = fmaxf(m0, m1);
                const float f0 = m0 == -INFINITY ? 0.f : ex2(m0 - mm), f1 = m1 == -INFINITY ? 0.f : ex2(m1 - mm);
                if (store && s == 0) *reinterpret_cast<float2*>(rec + BQ * HD + 2 * r) = make_float2(mm, sh.ml[0][1][r] * f0 + sh.ml[1][1][r] * f1);
                constexpr int HALF = HD / 2;
#pragma unroll 1
                for (int c = s * HALF; c < (s + 1) * HALF; c += 32) {
                    float v[32], w[32];
                    tc_ld32_nowait(lane_base + COL_O + c, reinterpret_cast<uint32_t*>(v));
                    tc_ld32_nowait(lane_base + COL_O + HD + c, reinterpret_cast<uint32_t*>(w));
                    tc_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = fmaf(w[i], f1, v[i] * f0);
                    put(c, v);
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.joined);    // (both streams' warps have read both sums)
            ok = __all_sync(0xffffffffu, mbar_wait(&sh.joined, joins & 1, abort_flag, status, 7));
            if (!ok) break;
            ++joins;
            if (lane == 0) mbar_arrive(&sh.o_empty[s]);
        }
    }

    tc_fence_before();
    __syncthreads();
    if (sh.abort_flag) {
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) __nanosleep(1000);   // copies in flight land before the block leaves
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS));
    }
}

}  // namespace tc

int launch_tc(const void* q, int n_tokens, const void* kv, int64_t kv_pages, const Groups& G, int blocks, float scale, int* plan, float* records, int* status,
              cudaStream_t s) {
    using namespace tc;
    WICK_REQUIRE(kv_pages * 2 * G.kv_heads * kPage <= INT32_MAX, "attention (shared prefix): a cache of %lld pages is beyond the copies' coordinates", (long long)kv_pages);
    CUtensorMap q_map, kv_map;
    if (int e = make_heads_map(&q_map, q, n_tokens, G.heads, HD, G.gs, G.rows / G.gs)) return e;
    if (int e = make_bf16_map(&kv_map, kv, kv_pages * 2 * G.kv_heads * kPage, HD, BK, "attention (shared prefix)")) return e;
    static bool raised = false;
    if (!raised) {
        WICK_CUDA(cudaFuncSetAttribute(attn_shared_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
        raised = true;
    }
    WICK_CUDA(launch(attn_shared_tc_kernel, dim3(blocks), dim3(THREADS), (size_t)SMEM_BYTES, s, q_map, kv_map, G, kv_pages, scale, plan, records, status));
    return check_launch("attn_shared_tc");
}

}  // namespace shared_prefix
}  // namespace wick
