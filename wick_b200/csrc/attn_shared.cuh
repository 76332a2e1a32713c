// Attention of a step's new tokens where groups of sequences share their first pages: what the kernels agree on.
//
// With L_g the positions of group g's shared pages, a row (a token's query head) at position p is
//   y = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q . k_j,  j = 0 .. p
// and the sum splits at L_g: keys below it are the same for all rows of the group, and are read once for as many rows as a tile
// holds; the rest are the sequence's own.  Each part is kept as (m, l, o) = (maximum, sum of weights, weighted sum of values), all
// in float32, and parts are joined by M = max m_i, l = sum l_i 2^(m_i - M), o likewise (scores in units of log2 e).
//
// A tile's rows see the shared keys in blocks of G.block pages; a tile (or, where a block of threads takes two, a pair of neighbouring
// tiles) with all its blocks is an ITEM, a tile and block a UNIT of work.  The units of all items, one behind the other, are dealt to
// the thread blocks in equal contiguous runs, so that no last round is half empty, whatever the groups' sizes; where a run ends inside an
// item the item has a further record.  Who has which unit follows from the description alone, so the kernel that joins finds the
// records by arithmetic, in a fixed order.
#pragma once

#include "common.cuh"

namespace wick {
namespace shared_prefix {

constexpr int MAX_GROUPS = 1024;

// The step's description and how the shared part is cut.
struct Groups {
    const int *cu_groups, *pages, *group_of;       // sequences of group g: cu_groups[g] .. ; its shared pages; the group of a sequence
    const int *cu_seqlens, *start, *page_table;
    int n, n_seqs, table_width, max_pages;
    int single;                                    // every sequence brings one token: token i is sequence i's
    int heads, kv_heads;
    int rows;                                      // of a tile
    int gs, per_kv, columns;                       // heads of a tile; tiles of heads to a key head, in all
    int block, pair;                               // pages of a block of keys; tiles of an item, at most
};
__device__ __forceinline__ int pages_of(const Groups& G, int g) { return max(0, min(min(G.pages[g], G.max_pages), G.table_width)); }

// Something whose tiles see the same keys: a group and its shared pages, or a sequence and its own.
struct Cut {
    int pages, tok0, n_tok, tiles, blocks;
    int seq, first, end;                           // the row of the page table, its first column, the end of the positions
};
// How such things are dealt: tiles of an item at most, columns, and the cut of number i of n.
struct SharedParts {
    static constexpr bool OWN = false;
    const Groups G;
    __device__ __forceinline__ int n() const { return G.n; }
    __device__ __forceinline__ int pair() const { return G.pair; }
    __device__ __forceinline__ int columns() const { return G.columns; }
    __device__ __forceinline__ Cut operator()(int g) const {
        Cut c;
        c.pages = pages_of(G, g);
        const int a = max(0, min(G.cu_groups[g], G.n_seqs)), b = max(a, min(G.cu_groups[g + 1], G.n_seqs));
        c.seq = a, c.first = 0;
        c.tok0 = G.single ? a : G.cu_seqlens[a];
        c.n_tok = (G.single ? b : G.cu_seqlens[b]) - c.tok0;
        c.tiles = c.pages > 0 ? (c.n_tok * G.gs + G.rows - 1) / G.rows : 0;
        c.blocks = (c.pages + G.block - 1) / G.block;
        c.end = c.pages * kPage;
        return c;
    }
};
// The own keys of a sequence that does not fit its group or its page table: none.
struct OwnParts {
    static constexpr bool OWN = true;
    const Groups G;
    int rows;                                      // of a tile
    __device__ __forceinline__ int n() const { return G.n_seqs; }
    __device__ __forceinline__ int pair() const { return 1; }
    __device__ __forceinline__ int columns() const { return G.kv_heads; }
    __device__ __forceinline__ bool fits(int b, const Cut& c) const {
        return G.group_of[b] >= 0 && G.group_of[b] < G.n && G.start[b] >= c.first * kPage && (c.end + kPage - 1) / kPage <= G.table_width;
    }
    __device__ __forceinline__ Cut operator()(int b) const {
        Cut c;
        const int g = G.group_of[b];
        c.seq = b;
        c.tok0 = G.single ? b : G.cu_seqlens[b];
        c.n_tok = G.single ? 1 : G.cu_seqlens[b + 1] - c.tok0;
        c.first = g >= 0 && g < G.n ? pages_of(G, g) : 0;
        c.end = G.start[b] + c.n_tok;
        c.blocks = c.pages = c.n_tok > 0 && fits(b, c) ? (c.end + kPage - 1) / kPage - c.first : 0;
        c.tiles = c.pages > 0 ? (c.n_tok * (G.heads / G.kv_heads) + rows - 1) / rows : 0;
        return c;
    }
};
// By a warp: the sequences that do not fit are reported, and their rows are made zero.
template <typename T> __device__ __forceinline__ void clear_unfit(const OwnParts& parts, T* out, int row_numbers, int* status) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < parts.n(); b0 += 32) {
        Cut c = Cut{0, 0, 0, 0, 0, 0, 0, 0};
        if (b0 + lane < parts.n()) c = parts(b0 + lane);
        unsigned bad = __ballot_sync(0xffffffffu, c.n_tok > 0 && c.pages == 0);
        if (bad && lane == 0) atomicCAS(status, 0, 11);
        for (; bad; bad &= bad - 1) {
            const int l = __ffs(bad) - 1;
            const int64_t at = (int64_t)__shfl_sync(0xffffffffu, c.tok0, l) * row_numbers, n = (int64_t)__shfl_sync(0xffffffffu, c.n_tok, l) * row_numbers;
            for (int64_t i = lane; i < n; i += 32) st(out + at + i, 0.f);
        }
    }
}
// Item i of a thing is pair i / columns of tiles: how many they are, and the units of the thing before it.
__device__ __forceinline__ int items_of(const Cut& c, int pair, int columns) { return (c.tiles + pair - 1) / pair * columns; }
__device__ __forceinline__ int width_of(const Cut& c, int pair, int k) { return min(pair, c.tiles - k * pair); }
__device__ __forceinline__ int units_before(const Cut& c, int pair, int columns, int k, int column) {
    return (k * pair * columns + column * width_of(c, pair, k)) * c.blocks;
}

// The units dealt: thread block c of S takes those from run_start(c) to run_start(c + 1), U / S of them or one more, and `pair` at least.
struct Deal {
    int U, S, per, more;                           // more: thread blocks that have one more than per
    __device__ __forceinline__ Deal(int units, int blocks, int pair) : U(units) {
        S = max(1, min(blocks, U / pair));
        per = U / S, more = U - per * S;
    }
    __device__ __forceinline__ int run_start(int c) const { return c * per + min(c, more); }
    __device__ __forceinline__ int block_of(int u) const { return u < more * (per + 1) ? u / (per + 1) : more + (u - more * (per + 1)) / per; }
};

// A run's part of one item: `tiles` tiles from `tile` on, blocks of keys from .. to.
struct Segment {
    Cut cut;
    int tile, tiles, column;
    int from, to;
    int record;                                    // its number among all segments that there can be
    int item0;                                     // the item's first unit
};

// A warp's way through its thread block's run.  A lane knows one thing of 32.
template <typename Parts> struct Walk {
    const Parts parts;
    Deal deal;
    int u, end;                                    // where it is in its run, the run's end
    int g0, units, items;                          // first of the things known; units and items before it
    Cut mine;
    int upto_units, upto_items;                    // ... and up to this lane's

    __device__ __forceinline__ void know(int first) {
        g0 = first;
        const int g = g0 + (int)(threadIdx.x & 31);
        mine = Cut{0, 0, 0, 0, 0, 0, 0, 0};
        if (g < parts.n()) mine = parts(g);
        int x = mine.tiles * parts.columns() * mine.blocks, y = items_of(mine, parts.pair(), parts.columns());
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int tx = __shfl_up_sync(0xffffffffu, x, o), ty = __shfl_up_sync(0xffffffffu, y, o);
            if ((int)(threadIdx.x & 31) >= o) x += tx, y += ty;
        }
        upto_units = units + x, upto_items = items + y;
    }
    __device__ __forceinline__ void next() {       // what was known becomes what lies before
        units = __shfl_sync(0xffffffffu, upto_units, 31), items = __shfl_sync(0xffffffffu, upto_items, 31);
        know(g0 + 32);
    }
    // plan: where the thread blocks' number and the units and items before each thing are written down, or null.
    __device__ __forceinline__ Walk(const Parts& p, int blocks, int* plan) : parts(p), deal(0, 1, 1), units(0), items(0) {
        const int lane = threadIdx.x & 31;
        know(0);
        for (;;) {
            const int g = g0 + lane;
            if (plan && g < parts.n()) plan[2 + g] = upto_units, plan[3 + parts.n() + g] = upto_items;
            if (g0 + 32 >= parts.n()) break;
            next();
        }
        deal = Deal(__shfl_sync(0xffffffffu, upto_units, 31), blocks, parts.pair());
        if (plan && lane == 0) plan[0] = deal.S, plan[1] = 0, plan[2 + parts.n()] = 0;
        const bool in = deal.U > 0 && (int)blockIdx.x < deal.S;
        u = in ? deal.run_start(blockIdx.x) : 0;
        end = in ? deal.run_start(blockIdx.x + 1) : 0;
        if (parts.n() > 32) units = items = 0, know(0);
    }
    // The next part of the run; false: there is none.
    __device__ __forceinline__ bool segment(Segment& s) {
        while (u < end) {
            while (u >= __shfl_sync(0xffffffffu, upto_units, 31)) next();
            const int l = __ffs(__ballot_sync(0xffffffffu, u < upto_units)) - 1, pair = parts.pair(), columns = parts.columns();
            Cut& c = s.cut;
            c.pages = __shfl_sync(0xffffffffu, mine.pages, l), c.tok0 = __shfl_sync(0xffffffffu, mine.tok0, l);
            c.n_tok = __shfl_sync(0xffffffffu, mine.n_tok, l), c.tiles = __shfl_sync(0xffffffffu, mine.tiles, l);
            c.blocks = __shfl_sync(0xffffffffu, mine.blocks, l), c.seq = __shfl_sync(0xffffffffu, mine.seq, l);
            c.first = __shfl_sync(0xffffffffu, mine.first, l), c.end = __shfl_sync(0xffffffffu, mine.end, l);
            const int base = __shfl_sync(0xffffffffu, upto_units - mine.tiles * columns * mine.blocks, l), local = u - base;
            const int k = local / (pair * columns * c.blocks), w = width_of(c, pair, k), before = units_before(c, pair, columns, k, 0);
            s.column = (local - before) / (w * c.blocks);
            const int off = local - before - s.column * w * c.blocks, left = min(w * c.blocks - off, end - u);
            s.tile = k * pair, s.tiles = w, s.item0 = u - off;
            // (a block of two tiles is done by whoever has the second one's unit)
            s.from = off / w, s.to = (off + left) / w;
            // (items and thread blocks rise together along the runs: no two segments share the sum)
            s.record = __shfl_sync(0xffffffffu, upto_items - items_of(mine, pair, columns), l) + k * columns + s.column + (int)blockIdx.x;
            u += left;
            if (s.from < s.to) return true;
        }
        return false;
    }
};

// A record: [HD / 4][rows] groups of four sums, then [rows] pairs of maximum and sum.  Records of a kind of parts, and the plan of the Walk
// that dealt them (null: there are none):
struct Records {
    const int* plan;
    const float* at;
    int rows;                                      // that a record has room for
};

// 2^(a - b) for maxima that may be -inf (nothing seen): then the weight is 0.
__device__ __forceinline__ float weight(float a, float b) { return a == -INFINITY ? 0.f : exp2f(a - b); }

constexpr float LOG2E = 1.4426950408889634f;

// The forms for bfloat16 at head sizes 64 and 128: the shared part on tcgen05 (attn_shared_tc.cu; tiles of up to TC_ROWS rows, two an item,
// blocks of two pages), and the own keys streamed through shared memory (attn_shared_own.cu).
constexpr int TC_ROWS = 128, OWN_ROWS = 16, OWN_WARPS = 6;   // (warps an SM at head size 128, twice as many at 64)
bool fast_supported();
int launch_tc(const void* q, int n_tokens, const void* kv, int64_t kv_pages, const Groups& G, int blocks, float scale, int* plan, float* records, int* status,
              cudaStream_t s);
int launch_own(const void* q, const void* kv, int64_t kv_pages, void* out, const Groups& G, bool after_shared, int blocks, float scale, int* plan,
               float* records, int* status, cudaStream_t s);

}  // namespace shared_prefix
}  // namespace wick
