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
    const int *cu_seqlens, *start, *positions, *page_table;
    int n, n_seqs, table_width, max_pages;
    int heads, kv_heads;
    int rows;                                      // of a tile
    int gs, per_kv, columns;                       // heads of a tile; tiles of heads to a key head, in all
    int block, pair;                               // pages of a block of keys; tiles of an item, at most
};

// One group as it is cut.
struct Cut {
    int pages, tok0, n_tok, tiles, blocks;
    __device__ __forceinline__ int items(const Groups& G) const { return (tiles + G.pair - 1) / G.pair * G.columns; }
    __device__ __forceinline__ int units(const Groups& G) const { return tiles * G.columns * blocks; }
    // Item i of the group is pair i / columns of tiles: how many they are, and the units of the group before it.
    __device__ __forceinline__ int width(const Groups& G, int pair) const { return min(G.pair, tiles - pair * G.pair); }
    __device__ __forceinline__ int before(const Groups& G, int pair, int column) const { return (pair * G.pair * G.columns + column * width(G, pair)) * blocks; }
};
__device__ __forceinline__ int pages_of(const Groups& G, int g) { return max(0, min(min(G.pages[g], G.max_pages), G.table_width)); }
__device__ __forceinline__ int first_token(const Groups& G, int g) { return G.cu_seqlens[max(0, min(G.cu_groups[g], G.n_seqs))]; }
__device__ __forceinline__ Cut cut_of(const Groups& G, int g) {
    Cut c;
    c.pages = pages_of(G, g);
    c.tok0 = first_token(G, g);
    c.n_tok = first_token(G, g + 1) - c.tok0;
    c.tiles = c.pages > 0 ? (c.n_tok * G.gs + G.rows - 1) / G.rows : 0;
    c.blocks = (c.pages + G.block - 1) / G.block;
    return c;
}

// Thread block c of S takes the units c U / S .. (c + 1) U / S; the block of unit u.  A run has G.pair units at least.
__device__ __forceinline__ int run_start(int c, int U, int S) { return (int)((int64_t)c * U / S); }
__device__ __forceinline__ int block_of(int u, int U, int S) { return (int)(((int64_t)S * (u + 1) - 1) / U); }

// A run's part of one item: `tiles` tiles from `tile` on, blocks of keys from .. to.
struct Segment {
    int g, pages, tok0, n_tok, tile, tiles, column, record;
    int from, to;
};

// A warp's way through its thread block's run.  A lane knows one group of 32.
struct Walk {
    const Groups& G;
    int U, S, cta, u, end;                         // units of all groups; thread blocks that take part; this one, where it is in its run, the run's end
    int g0, units, items;                          // first group of those known; units and items of the groups before it
    Cut mine;
    int upto_units, upto_items;                    // ... and up to this lane's group

    __device__ __forceinline__ void know(int first) {
        g0 = first;
        const int g = g0 + (int)(threadIdx.x & 31);
        mine = Cut{0, 0, 0, 0, 0};
        if (g < G.n) mine = cut_of(G, g);
        int x = mine.units(G), y = mine.items(G);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int tx = __shfl_up_sync(0xffffffffu, x, o), ty = __shfl_up_sync(0xffffffffu, y, o);
            if ((int)(threadIdx.x & 31) >= o) x += tx, y += ty;
        }
        upto_units = units + x, upto_items = items + y;
    }
    // The groups known before become those before the first known.
    __device__ __forceinline__ void next() {
        units = __shfl_sync(0xffffffffu, upto_units, 31), items = __shfl_sync(0xffffffffu, upto_items, 31);
        know(g0 + 32);
    }
    // plan: where the thread blocks' number and the units and items before each group are written down, or null.
    __device__ __forceinline__ Walk(const Groups& groups, int blocks, int* plan) : G(groups), units(0), items(0) {
        know(0);
        for (;;) {
            const int g = g0 + (int)(threadIdx.x & 31);
            if (plan && g < G.n) plan[2 + g] = upto_units, plan[3 + G.n + g] = upto_items;
            if (g0 + 32 >= G.n) break;
            next();
        }
        U = __shfl_sync(0xffffffffu, upto_units, 31);
        S = max(1, min(blocks, U / G.pair));
        if (plan && (threadIdx.x & 31) == 0) plan[0] = S, plan[1] = 0, plan[2 + G.n] = 0;
        cta = blockIdx.x;
        u = U > 0 && cta < S ? run_start(cta, U, S) : 0;
        end = U > 0 && cta < S ? run_start(cta + 1, U, S) : 0;
        if (G.n > 32) units = items = 0, know(0);
    }
    // The next part of the run; false: there is none.
    __device__ __forceinline__ bool segment(Segment& s) {
        while (u < end) {
            while (u >= __shfl_sync(0xffffffffu, upto_units, 31)) next();
            const int l = __ffs(__ballot_sync(0xffffffffu, u < upto_units)) - 1;
            Cut c;
            c.pages = __shfl_sync(0xffffffffu, mine.pages, l), c.tok0 = __shfl_sync(0xffffffffu, mine.tok0, l);
            c.n_tok = __shfl_sync(0xffffffffu, mine.n_tok, l), c.tiles = __shfl_sync(0xffffffffu, mine.tiles, l);
            c.blocks = __shfl_sync(0xffffffffu, mine.blocks, l);
            const int local = u - __shfl_sync(0xffffffffu, upto_units - mine.units(G), l), pair = local / (G.pair * G.columns * c.blocks);
            const int w = c.width(G, pair), column = (local - c.before(G, pair, 0)) / (w * c.blocks), off = local - c.before(G, pair, column);
            const int left = min(w * c.blocks - off, end - u);
            s.g = g0 + l, s.pages = c.pages, s.tok0 = c.tok0, s.n_tok = c.n_tok;
            s.tile = pair * G.pair, s.tiles = w, s.column = column;
            // (a block of two tiles is done by whoever has the second one's unit)
            s.from = off / w, s.to = (off + left) / w;
            // (items and thread blocks rise together along the runs: no two segments share the sum)
            s.record = (__shfl_sync(0xffffffffu, upto_items - mine.items(G), l) + pair * G.columns + column + cta) * G.pair;
            u += left;
            if (s.from < s.to) return true;
        }
        return false;
    }
};

// The tcgen05 form of the shared part (attn_shared_tc.cu): bfloat16, tiles of up to TC_ROWS rows, two an item, blocks of two pages.
constexpr int TC_ROWS = 128;
bool tc_supported();
int launch_tc(const void* q, int n_tokens, const void* kv, int64_t kv_pages, const Groups& G, int blocks, float scale, int* plan, float* records, int* status,
              cudaStream_t s);

}  // namespace shared_prefix
}  // namespace wick
