// Attention over a 4-bit cache on the 5th-generation tensor cores: bfloat16, head size 128 (attn_kv4.cu has the mathematics and how the work is cut).
//
// A group of four warps computes a node of a (sequence, key head, tile of up to 32 rows), 128 positions (two pages) at a time:
//   scores  S^T [128 positions x rows] = K Q^T:  the keys' values go from registers into tensor memory as the first operand, the queries lie in shared memory;
//   weights: a thread has one position's scores; P goes to shared memory as bfloat16 numbers;
//   O^T [128 channels x rows] += V^T P:  the values go from registers into shared memory (128-byte swizzle) as the first operand, read with channels along its
//            rows; the accumulator stays in tensor memory over the node.
// One lane issues the products, one lane the copies: a tile's codes are fetched in halves, the next tile's keys as soon as this one's have been read, its values
// when this one's have.  The scores' products run beside the making of the values, the second products beside the making of the next keys.
// Weights are relative to a maximum that follows the true one lazily (it moves when a score exceeds it by more than 8 in units of log2 e), so that the
// positions' common maximum has to be found, across 128 threads, only in a node's first tile and where scores rise.  They enter the product, and their sum, as
// bfloat16 numbers, so that the rounding of the largest cancels.
//
// Why: with mma.sync a page of 128 channels costs 64 products of 8 clocks that run beside nothing else (measured: 14 shifts and AND-ORs, 8 multiply-adds and 2
// products take 50 clocks, without the products 28), 2,600 clocks a page and scheduler where the codes alone are 1,300.  And the
// codes are opened once for 32 rows here, for 8 or 16 there.
#include "attn_kv4.cuh"
#include "tc_attention.cuh"

namespace wick {
namespace kv4 {

#if WICK_HD == 128
namespace tc {

constexpr int GROUP_THREADS = 128;
constexpr int POSITIONS = 2 * kPage;
constexpr int V_PANEL = POSITIONS * 128, V_BYTES = 2 * V_PANEL;  // 64 channels x 128 positions, rows of 128 bytes
constexpr int COL_S = 64, COL_O = 96, GROUP_COLS = 128;  // columns of tensor memory: 64 of the keys' values as pairs, S^T, O^T

template <int NR> constexpr int N = NR <= 16 ? 16 : 32;          // of the products (a multiple of 16)

struct Tile {                                                    // what a group is to compute next
    int b, kvh, row0, place, nodes;                              // nodes: of the sequence that the row tile sees
    int page, pages;                                             // of the sequence: the first, and how many (1 or 2)
    int first, start, len, new_tokens;                           // of the sequence
    int begins, ends, none;                                      // the node's first tile, its last; nothing is left
};
template <int NR> struct Shared {                                // a group's
    uint8_t codes[2 * TILE];
    uint8_t v[V_BYTES];
    uint8_t q[N<NR> * 256];
    uint8_t p[N<NR> * 256];
    float top[4][NR], sum[4][NR], neg_m[NR], alpha[NR], node_m[NR], node_l[NR];
    int limit[NR];
    uint32_t odd[4];                                             // rows that see a value that is no number, per 32 channels
    Tile tile[2];
    uint64_t full_k, full_v, scores, sums;
};
template <int NR> constexpr int shared_bytes() { return ((int)sizeof(Shared<NR>) + 1023) / 1024 * 1024; }

__device__ __forceinline__ void group_sync(int id) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ bool group_any(int id, bool mine) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %1, 0;\n\tbarrier.cta.red.or.pred p, %2, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(any) : "r"((uint32_t)mine), "r"(id) : "memory");
    return any != 0;
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 16 lanes x 64 columns: lane (r, j) gives columns 8 n + 2 j, + 1 of rows r (v[4 n], v[4 n + 1]) and r + 8 (v[4 n + 2], v[4 n + 3]).
__device__ __forceinline__ void tc_st_16x256b_x8(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.16x256b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
          "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tc_ld8(uint32_t taddr, float* v) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
}
__device__ __forceinline__ void tc_st8(uint32_t taddr, const float* v) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
// D (tensor memory) (+)= A (shared memory) * B (shared memory), either with a layout of its own.
__device__ __forceinline__ void mma_ss2(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, int acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "mov.b64 da, {%1, %2};\n\t"
        "mov.b64 db, {%3, %4};\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
        : "memory");
}
// Numbers as integers of the same order.
__device__ __forceinline__ int order_of(float x) {
    const int i = __float_as_int(x);
    return i ^ ((i >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float number_of(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7FFFFFFF)); }

// The group's items: nodes of row tiles.
struct Item {
    Tile t;                                                      // (page: the next to be fetched)
    int end;
};

// CLUSTERS: a block has one group and one node, and the nodes of a (sequence, key head, row tile) are a cluster, whose blocks join them out of each other's
// shared memory.  Otherwise blocks stay, one an SM, with an equal run of all items of the step, which their groups take one by one; nodes leave records.
template <int NR, int GROUPS, bool CLUSTERS>
__global__ void __launch_bounds__(GROUPS * GROUP_THREADS, CLUSTERS ? 2 : 1) attn_kv4_tc_kernel(const Args a) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ int cum[CLUSTERS ? 1 : MAX_SEQS + 1], lens[CLUSTERS ? 1 : MAX_SEQS], firsts[CLUSTERS ? 1 : MAX_SEQS + 1];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag, taken;
    constexpr int NN = N<NR>;
    constexpr uint32_t TMEM_COLS = GROUPS == 1 ? 128 : (GROUPS == 2 ? 256 : 512);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = warp >> 2, quad = warp & 3, tid = threadIdx.x & 127, id = 1 + group;
    Shared<NR>& sh = *reinterpret_cast<Shared<NR>*>(smem_raw + group * shared_bytes<NR>());
    if (threadIdx.x == 0) abort_flag = 0;
    if (tid == 0) {
        mbar_init(&sh.full_k, 1);
        mbar_init(&sh.full_v, 1);
        mbar_init(&sh.scores, 1);
        mbar_init(&sh.sums, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    auto tiles_of = [&](const Seq& s) { return (s.new_tokens * a.group + NR - 1) / NR; };
    // An item from a sequence and its number there (nodes innermost, then row tiles, heads); false where the row tile sees none of the node's pages.
    auto make = [&](Item& it, int b, const Seq& s, int local) {
        const int all = nodes_of(s.pages, a.n_kv), per = LEAVES * leaf_pages(s.pages, a.n_kv), tiles = tiles_of(s), n_rows = s.new_tokens * a.group;
        it.t.place = local % all;
        const int rest = local / all;
        it.t.row0 = rest % tiles * NR;
        it.t.kvh = rest / tiles;
        it.t.b = b;
        it.t.first = s.first;
        it.t.start = s.start;
        it.t.len = s.len;
        it.t.new_tokens = s.new_tokens;
        const int seen = (s.start + (min(it.t.row0 + NR, n_rows) - 1) / a.group) / kPage + 1;
        it.t.nodes = CLUSTERS ? (seen + per - 1) / per : all;
        it.t.page = it.t.place * per;
        it.end = min(seen, it.t.page + per);
        it.t.begins = 1;
        return it.t.page < seen;
    };
    Item cn, nn;                                                 // (warp 1 of a group: the item whose pages are being fetched, and the next one)
    cn.t.b = nn.t.b = -1;
    int stop = 0;
    if (CLUSTERS) {
        unsigned at = blockIdx.x;
        const int node = (int)(at % (unsigned)a.nodes);
        at /= (unsigned)a.nodes;
        const int tile = (int)(at % (unsigned)a.tiles);
        at /= (unsigned)a.tiles;
        const int kvh = (int)(at % (unsigned)a.n_kv), b = (int)(at / (unsigned)a.n_kv);
        const Seq s = sequence(a, b);
        if (s.new_tokens > 0 && tile < tiles_of(s) && fits(a, s) && node < nodes_of(s.pages, a.n_kv)) {
            const int all = nodes_of(s.pages, a.n_kv);
            if (!make(cn, b, s, node + all * (tile + tiles_of(s) * kvh))) cn.t.b = -1;
        }
    } else {
        for (int b = threadIdx.x; b < a.n_seqs; b += GROUPS * GROUP_THREADS) {
            const Seq s = sequence(a, b);
            lens[b] = s.len;
            firsts[b] = s.first;
            if (b == a.n_seqs - 1) firsts[b + 1] = s.first + s.new_tokens;
            cum[b + 1] = s.new_tokens > 0 && fits(a, s) ? nodes_of(s.pages, a.n_kv) * tiles_of(s) * a.n_kv : 0;
        }
        __syncthreads();
        if (warp == 1) {
            int before = 0;
#pragma unroll 1
            for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
                const int b = s0 + lane, mine = b < a.n_seqs ? cum[b + 1] : 0;
                int upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                if (b < a.n_seqs) cum[b + 1] = before + upto;
                before += __shfl_sync(0xffffffffu, upto, 31);
            }
            if (lane == 0) {
                cum[0] = 0;
                taken = (int)((int64_t)blockIdx.x * before / gridDim.x);
            }
        }
        __syncthreads();
        stop = (int)((int64_t)(blockIdx.x + 1) * cum[a.n_seqs] / gridDim.x);
    }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();                                               // (tensor memory is this block's: a block of the next kernel cannot take it first)
    const uint32_t tmem = tmem_slot + group * GROUP_COLS;
    const uint32_t lanes = (uint32_t)(quad * 32) << 16;          // this warp's part of tensor memory

    const Tile whole = cn.t;                                     // (CLUSTERS: the block's node)
    // ---- fetching (warp 1) ----
    int ids = 0, next_ids = 0, held = 0, id0 = 0, id1 = 0;       // page ids of up to 32 pages of either item, and of the tile whose keys were fetched last
    auto page_ids = [&](const Item& it) {
        return it.t.page + lane < it.end ? checked_page(a, a.page_table[(int64_t)it.t.b * a.table_width + it.t.page + lane]) : 0;
    };
    auto take = [&](Item& it) {
        it.t.b = -1;
        while (!CLUSTERS) {
            int u = 0;
            if (lane == 0) u = atomicAdd(&taken, 1);
            u = __shfl_sync(0xffffffffu, u, 0);
            if (u >= stop) return;
            int lo = 0, hi = a.n_seqs - 1;                       // the last sequence with cum[b] <= u
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (cum[mid] <= u) lo = mid;
                else hi = mid - 1;
            }
            Seq s;
            s.first = firsts[lo];
            s.new_tokens = firsts[lo + 1] - s.first;
            s.len = lens[lo];
            s.start = s.len - s.new_tokens;
            s.pages = (s.len + kPage - 1) / kPage;
            if (make(it, lo, s, u - cum[lo])) return;
            it.t.b = -1;
        }
    };
    auto fetch = [&](uint64_t* bar, int half, int n, int kvh) {  // keys or values of the n pages id0, id1: their codes and their scales
        if (lane == 0) {
            mbar_expect_tx(bar, n * (TILE / 2));
            for (int i = 0; i < n; ++i) {
                const uint8_t* src = a.kv + ((int64_t)(i ? id1 : id0) * a.n_kv + kvh) * TILE;
                uint8_t* dst = sh.codes + i * TILE;
                bulk_load(dst + half * value_codes(D), src + half * value_codes(D), 32 * D, bar);
                bulk_load(dst + key_scales(D) + half * 8 * D, src + key_scales(D) + half * 8 * D, 8 * D, bar);
            }
        }
    };
    // The next tile's description into place `at`, and its keys on their way.
    auto next_keys = [&](int at) {
        Tile& t = sh.tile[at];
        if (cn.t.b < 0) {
            if (lane == 0) {
                t.none = 1;
                mbar_arrive(&sh.full_k);
            }
            return;
        }
        const int n = min(2, cn.end - cn.t.page);
        id0 = __shfl_sync(0xffffffffu, ids, held);
        id1 = __shfl_sync(0xffffffffu, ids, (held + 1) & 31);
        if (lane == 0) {
            t = cn.t;
            t.pages = n;
            t.ends = cn.t.page + n >= cn.end;
            t.none = 0;
        }
        __syncwarp();
        fetch(&sh.full_k, 0, n, cn.t.kvh);
        cn.t.begins = 0;
        cn.t.page += n;
        held += 2;
        if (cn.t.page >= cn.end) {
            cn = nn;
            ids = next_ids;
            held = 0;
            take(nn);
            if (nn.t.b >= 0) next_ids = page_ids(nn);
        } else if (held == 32) {
            held = 0;
            ids = page_ids(cn);
        }
    };
    if (quad == 1) {
        if (!CLUSTERS) take(cn);
        if (cn.t.b >= 0) {
            ids = page_ids(cn);
            take(nn);
            if (nn.t.b >= 0) next_ids = page_ids(nn);
        }
        const int n = min(2, cn.end - cn.t.page), kvh = cn.t.kvh, any = cn.t.b;
        next_keys(0);
        if (any >= 0) fetch(&sh.full_v, 1, n, kvh);
    }

    const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(NN >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
    const uint32_t idesc_s = idesc, idesc_o = idesc | (1u << 15) | (1u << 16);
    const uint32_t q_lo = desc_lo(smem_u32(sh.q), 16), v_lo = desc_lo(smem_u32(sh.v), V_PANEL), p_lo = desc_lo(smem_u32(sh.p), 128);
    constexpr uint32_t P_HI = (2048u >> 4) | (1u << 14);         // rows of 8: 2,048 bytes apart; no swizzle
    const int r = lane >> 2, j = lane & 3;
    float part[NR];                                              // this position's share of the rows' sums
    bool bad = false;
    uint32_t sums = 0;                                           // second products so far
#pragma unroll 1
    for (uint32_t it = 0;; ++it) {
        bad = __any_sync(0xffffffffu, bad || !mbar_wait(&sh.full_k, it & 1, &abort_flag, a.status, 16));
        const Tile& t = sh.tile[it & 1];
        const bool over = bad || t.none;
        const int first_pos = t.page * kPage, pos = first_pos + tid;
        const bool begins = t.begins != 0, masked = first_pos + POSITIONS - 1 > t.start, several = t.new_tokens > 1;
        if (!over && begins) {
            // the rows' queries, in the order that the keys' channels come in; zeros behind the last
            const int n_rows = t.new_tokens * a.group;
#pragma unroll 1
            for (int i = tid; i < NR * 8; i += GROUP_THREADS) {
                const int row = i >> 3, w = (i >> 1) & 3, jp = i & 1, at = t.row0 + row;
                uint4 x = make_uint4(0, 0, 0, 0), y = x;
                if (at < n_rows) {
                    const int tok = at / a.group;
                    const uint4* src = reinterpret_cast<const uint4*>(
                        (const bf16*)a.q + ((int64_t)(t.first + tok) * a.n_heads + t.kvh * a.group + at - tok * a.group) * D + 64 * jp + 8 * w);
                    x = src[0];
                    y = src[4];                                  // (32 channels on)
                    x.x ^= a.flip, x.y ^= a.flip, x.z ^= a.flip, x.w ^= a.flip;
                    y.x ^= a.flip, y.y ^= a.flip, y.z ^= a.flip, y.w ^= a.flip;
                }
                const uint4 even = make_uint4(low_halves(x.x, x.z), high_halves(x.x, x.z), low_halves(y.x, y.z), high_halves(y.x, y.z));
                const uint4 odd = make_uint4(low_halves(x.y, x.w), high_halves(x.y, x.w), low_halves(y.y, y.w), high_halves(y.y, y.w));
                const int c0 = 4 * w + jp, c1 = c0 + 2;
                *reinterpret_cast<uint4*>(sh.q + (c0 >> 3) * (NN * 128) + row * 128 + (((c0 & 7) ^ (row & 7)) << 4)) = even;
                *reinterpret_cast<uint4*>(sh.q + (c1 >> 3) * (NN * 128) + row * 128 + (((c1 & 7) ^ (row & 7)) << 4)) = odd;
            }
            if (tid < NR) sh.limit[tid] = t.start + min(t.row0 + tid, n_rows - 1) / a.group;
            if (tid < 4) sh.odd[tid] = 0;
            proxy_fence();
#pragma unroll
            for (int i = 0; i < NR; ++i) part[i] = 0.f;
        }
        // ---- keys: lane (r, j) makes quarter j of positions r, r + 8, ... of its warp's 32 ----
        if (!over) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t out[32];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int row = quad * 32 + h * 16 + u * 8 + r;
                const uint8_t* page = sh.codes + (row >> 6) * TILE;
                const uint4 x = *reinterpret_cast<const uint4*>(page + (row & 63) * (D / 2) + j * 16);
                const uint32_t sc = *reinterpret_cast<const uint32_t*>(page + key_scales(D) + (row & 63) * (D / 8) + j * 4);
                const uint32_t a2 = low_halves(sc, sc), b2 = high_halves(sc, sc), w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t v[4];
                    key_word(w[i], a2, b2, v);
                    out[8 * i + 2 * u] = v[0];
                    out[8 * i + 2 * u + 1] = v[1];
                    out[8 * i + 4 + 2 * u] = v[2];
                    out[8 * i + 4 + 2 * u + 1] = v[3];
                }
            }
            tc_st_16x256b_x8(tmem + lanes + ((uint32_t)(h * 16) << 16), out);
        }
        tc_st_wait();
        tc_fence_before();
        }
        if (group_any(id, over)) break;                          // (nothing is left, or a wait gave up: all of the group leave together)
        if (quad == 0) {
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    mma_ts(tmem + COL_S, tmem + ks * 8, q_lo + (((ks >> 2) * (NN * 128) + (ks & 3) * 32) >> 4), idesc_s, ks > 0);
                tc_commit(&sh.scores);
            }
            __syncwarp();
        }
        const int n_pages = t.pages, kvh = t.kvh;
        const bool ends = t.ends != 0;
        if (quad == 1) next_keys((it + 1) & 1);
        // ---- values: a thread makes one position's; the tile before must have been multiplied ----
        if (sums > 0) bad |= !mbar_wait(&sh.sums, (sums - 1) & 1, &abort_flag, a.status, 16);
        bad |= !mbar_wait(&sh.full_v, it & 1, &abort_flag, a.status, 16);
        {
            const int row = tid & 63;
            const uint8_t* page = sh.codes + (tid >> 6) * TILE;
            const bool beyond = pos >= t.len || (tid >> 6) >= n_pages;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int piece = (i + (tid >> 1)) & 3, group32 = piece ^ (2 * value_turn<D>(row));      // 16 bytes as they lie there; the 32 channels that they are
                const uint4 x = *reinterpret_cast<const uint4*>(page + value_codes(D) + row * (D / 2) + piece * 16);
                uint32_t sc = *reinterpret_cast<const uint32_t*>(page + value_scales(D) + row * (D / 8) + group32 * 4);
                if (masked) {                                    // (behind the sequence's end anything may lie)
                    if (beyond) sc = 0;
                    else if (several && no_number(sc)) {
                        // it shows in the rows that see its position, and in no others (a weight of 0 would not hide it in the product)
                        uint32_t rows = 0;
                        for (int k = 0; k < NR; ++k) rows |= (uint32_t)(sh.limit[k] >= pos) << k;
                        atomicOr(&sh.odd[group32], rows);
                        sc = 0;
                    }
                }
                const uint32_t a2 = low_halves(sc, sc), b2 = high_halves(sc, sc), w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t lo = __byte_perm(w[k], w[k], 0x1100), hi = __byte_perm(w[k], w[k], 0x3322);
                    const uint4 v = make_uint4(two_values(lo, a2, b2), two_values(lo >> 4, a2, b2), two_values(hi, a2, b2), two_values(hi >> 4, a2, b2));
                    const int c = 4 * group32 + k;               // the channels 8 c .. 8 c + 7 in the order 0 2 1 3 4 6 5 7
                    *reinterpret_cast<uint4*>(sh.v + (c >> 3) * V_PANEL + tid * 128 + (((c & 7) ^ (tid & 7)) << 4)) = v;
                }
            }
        }
        // ---- weights ----
        bad |= !mbar_wait(&sh.scores, it & 1, &abort_flag, a.status, 16);
        tc_fence_after();
        float s[NR];
#pragma unroll
        for (int k = 0; k < NR; k += 8) tc_ld8(tmem + lanes + COL_S + k, s + k);
        tc_ld_wait();
        const bool beyond = masked && (pos >= t.len || (tid >> 6) >= n_pages);
        if (masked) {
#pragma unroll
            for (int k = 0; k < NR; ++k)
                if (beyond || pos > sh.limit[k]) s[k] = -INFINITY;
        }
        bool rises = begins;
        if (!begins) {
            float most = -INFINITY;
#pragma unroll
            for (int k = 0; k < NR; ++k) most = fmaxf(most, s[k] == -INFINITY ? -INFINITY : fmaf(s[k], a.scale2, sh.neg_m[k]));
            rises = group_any(id, most > 8.0f);
        }
        if (rises) {
            // the rows' largest scores over the 128 positions
#pragma unroll
            for (int k = 0; k < NR; ++k) {
                const float top = number_of(__reduce_max_sync(0xffffffffu, order_of(s[k] == -INFINITY || s[k] != s[k] ? -INFINITY : s[k] * a.scale2)));
                if (lane == 0) sh.top[quad][k] = top;
            }
            group_sync(id);
            if (tid < NR) {
                const float top = fmaxf(fmaxf(sh.top[0][tid], sh.top[1][tid]), fmaxf(sh.top[2][tid], sh.top[3][tid]));
                const float was = begins ? -INFINITY : sh.node_m[tid], m = fmaxf(was, top);
                sh.node_m[tid] = m;
                sh.neg_m[tid] = m == -INFINITY ? 0.f : -m;
                sh.alpha[tid] = weight(was, m);
            }
            group_sync(id);
            if (!begins) {
                // (the second products so far have ended: they were waited for above)
                float o[8];
#pragma unroll
                for (int k = 0; k < NR; k += 8) {
                    tc_ld8(tmem + lanes + COL_O + k, o);
                    tc_ld_wait();
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        o[e] *= sh.alpha[k + e];
                        part[k + e] *= sh.alpha[k + e];
                    }
                    tc_st8(tmem + lanes + COL_O + k, o);
                }
                tc_st_wait();
            }
        }
#pragma unroll
        for (int k = 0; k < NR; k += 8) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float x = s[k + e], y = s[k + e + 1];
                const float px = x == -INFINITY ? 0.f : ex2(fmaf(x, a.scale2, sh.neg_m[k + e]));
                const float py = y == -INFINITY ? 0.f : ex2(fmaf(y, a.scale2, sh.neg_m[k + e + 1]));
                w[e / 2] = pack_bf16(px, py);
                part[k + e] += __uint_as_float(w[e / 2] << 16);
                part[k + e + 1] += __uint_as_float(w[e / 2] & 0xFFFF0000u);
            }
            *reinterpret_cast<uint4*>(sh.p + (k >> 3) * 2048 + tid * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        proxy_fence();                                           // V and P before the products read them
        tc_fence_before();
        group_sync(id);
        if (quad == 0) {
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < POSITIONS / 16; ++ks)
                    mma_ss2(tmem + COL_O, v_lo + ks * (2048 >> 4), DESC_HI, p_lo + ks * (256 >> 4), P_HI, idesc_o, !begins || ks > 0);
                tc_commit(&sh.sums);
            }
            __syncwarp();
        }
        ++sums;
        if (quad == 1) {
            const Tile& nx = sh.tile[(it + 1) & 1];
            if (!nx.none) fetch(&sh.full_v, 1, nx.pages, nx.kvh);
        }
        if (!ends) continue;
        // ---- the node's end: a thread has one channel of all rows ----
#pragma unroll
        for (int k = 0; k < NR; k += 8) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = part[k + e];
            const float sum = warp_sums(v);
            if ((lane & 3) == 0) sh.sum[quad][k + (lane >> 2)] = sum;
        }
        bad |= !mbar_wait(&sh.sums, (sums - 1) & 1, &abort_flag, a.status, 16);
        tc_fence_after();
        float o[NR];
#pragma unroll
        for (int k = 0; k < NR; k += 8) tc_ld8(tmem + lanes + COL_O + k, o + k);
        tc_ld_wait();
        group_sync(id);
        const int ch = (tid & ~3) | (tid & 1) << 1 | (tid >> 1 & 1);
        const uint32_t odd = sh.odd[tid >> 5];
        const bool alone = t.nodes == 1;
        const int n_rows = t.new_tokens * a.group;
#pragma unroll
        for (int k = 0; k < NR; ++k) {
            const int row = t.row0 + k;
            if (row >= n_rows) break;
            const int tok = row / a.group;
            const int64_t flat = (int64_t)(t.first + tok) * a.n_heads + kvh * a.group + row - tok * a.group;
            const float l = (sh.sum[0][k] + sh.sum[1][k]) + (sh.sum[2][k] + sh.sum[3][k]);
            const float x = odd >> k & 1 ? __int_as_float(0x7FFFFFFF) : o[k];
            if (alone) {
                ((bf16*)a.out)[flat * D + ch] = __float2bfloat16_rn(result(x, l));
            } else if (CLUSTERS) {
                reinterpret_cast<float*>(sh.v)[k * D + ch] = x;
                if (tid == 0) sh.node_l[k] = l;
            } else {
                a.rec[(flat * a.nodes + t.place) * D + ch] = x;
                if (tid == 0) *reinterpret_cast<float2*>(a.rec + a.rec_rows * a.nodes * D + (flat * a.nodes + t.place) * 2) = make_float2(sh.node_m[k], l);
            }
        }
        tc_fence_before();
        group_sync(id);                                          // (what was read here is written again for the next node)
        tc_fence_after();
    }
    if constexpr (CLUSTERS) {
        // The nodes meet: the rows are shared out among the blocks, and joined out of all blocks' shared memory, in the nodes' order.
        if (whole.b >= 0 && whole.nodes > 1) {
            cluster_sync();
            const int n_rows = whole.new_tokens * a.group;
#pragma unroll 1
            for (int k = whole.place; k < NR && whole.row0 + k < n_rows; k += whole.nodes) {
                Fold f;
                f.m = -INFINITY;
                f.l = 0.f;
                float o = 0.f;
#pragma unroll 4
                for (int p = 0; p < whole.nodes; ++p) {
                    f.step(ld_cluster(in_block(smem_u32(&sh.node_m[k]), p)), ld_cluster(in_block(smem_u32(&sh.node_l[k]), p)));
                    o = f.of(o, ld_cluster(in_block(smem_u32(sh.v) + (uint32_t)(k * D + tid) * 4, p)));
                }
                const int row = whole.row0 + k, tok = row / a.group;
                ((bf16*)a.out)[((int64_t)(whole.first + tok) * a.n_heads + whole.kvh * a.group + row - tok * a.group) * D + tid] = __float2bfloat16_rn(result(o, f.l));
            }
            cluster_sync();                                      // (nobody leaves while others read)
        }
    }
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) __nanosleep(1000);   // copies in flight land before the block leaves
        __syncthreads();
    }
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_slot), "r"(TMEM_COLS));
    }
}

template <int NR> int launch(const Args& a, bool clusters, int64_t blocks, cudaStream_t s) {
    constexpr int GROUPS = 3;
    auto kernel = clusters ? attn_kv4_tc_kernel<NR, 1, true> : attn_kv4_tc_kernel<NR, GROUPS, false>;
    const int smem = (clusters ? 1 : GROUPS) * shared_bytes<NR>();
    static bool raised[2] = {false, false};
    if (!raised[clusters]) {
        WICK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        raised[clusters] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((clusters ? 1 : GROUPS) * GROUP_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = clusters ? a.nodes : 1;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 2 : 1;
    WICK_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
    return check_launch("attention_kv4 (tcgen05)");
}

}  // namespace tc

int launch_tc(const Args& a, int rows, bool clusters, int64_t blocks, cudaStream_t s) {
    return rows == 8 ? tc::launch<8>(a, clusters, blocks, s) : rows == 16 ? tc::launch<16>(a, clusters, blocks, s) : rows == 24 ? tc::launch<24>(a, clusters, blocks, s)
                                                                                                                        : tc::launch<32>(a, clusters, blocks, s);
}
#else
int launch_tc(const Args&, int, bool, int64_t, cudaStream_t) { return fail("attention_kv4: the tcgen05 kernel takes heads of 128"); }
#endif

}  // namespace kv4
}  // namespace wick
