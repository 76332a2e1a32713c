// Attention of a step's new tokens where groups of sequences share their first pages: what the kernels agree on.
//
// With L_g the positions of group g's shared pages, a row (a token's query head) at position p is
//   y = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q . k_j,  j = 0 .. p
// and the sum splits at L_g: keys below it are the same for all rows of the group, and are read once for as many rows as a tile
// holds; the rest are the sequence's own.  Each part is kept as (m, l, o) = (maximum, sum of weights, weighted sum of values), all
// in float32, and parts are joined by M = max m_i, l = sum l_i 2^(m_i - M), o likewise (scores in units of log2 e).
//
// The shared part is cut into UNITS (a run of pages for one tile of rows and one key head) that are dealt to the blocks of the
// grid in equal contiguous runs, so that the last round of blocks is never half empty, whatever the groups' sizes; where a
// run ends inside a tile's units the tile has a further record.  Who has which unit follows from the description alone, so
// the kernel that joins finds the records by arithmetic, in a fixed order.
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
    int unit_pages;
};

// A block's copy of the plan: units and items (a tile's units together) of the groups before each one.
struct Cum {
    int units[MAX_GROUPS + 1], items[MAX_GROUPS + 1];
};

__device__ __forceinline__ int pages_of(const Groups& G, int g) { return max(0, min(min(G.pages[g], G.max_pages), G.table_width)); }
__device__ __forceinline__ int first_token(const Groups& G, int g) { return G.cu_seqlens[max(0, min(G.cu_groups[g], G.n_seqs))]; }
__device__ __forceinline__ int units_per_item(const Groups& G, int pages) { return (pages + G.unit_pages - 1) / G.unit_pages; }

// By one warp.
__device__ __forceinline__ void make_plan(const Groups& G, int* units, int* items) {
    const int lane = threadIdx.x & 31;
    int bu = 0, bi = 0;
    if (lane == 0) units[0] = 0, items[0] = 0;
    for (int g0 = 0; g0 < G.n; g0 += 32) {
        const int g = g0 + lane;
        int u = 0, i = 0;
        if (g < G.n) {
            const int pages = pages_of(G, g);
            if (pages > 0) {
                i = ((first_token(G, g + 1) - first_token(G, g)) * G.gs + G.rows - 1) / G.rows * G.columns;
                u = i * units_per_item(G, pages);
            }
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int tu = __shfl_up_sync(0xffffffffu, u, o), ti = __shfl_up_sync(0xffffffffu, i, o);
            if (lane >= o) u += tu, i += ti;
        }
        if (g < G.n) units[g + 1] = bu + u, items[g + 1] = bi + i;
        bu += __shfl_sync(0xffffffffu, u, 31), bi += __shfl_sync(0xffffffffu, i, 31);
    }
    __syncwarp();
}

// Block c of S takes the units c U / S .. (c + 1) U / S; the block of unit u.
__device__ __forceinline__ int run_start(int c, int U, int S) { return (int)((int64_t)c * U / S); }
__device__ __forceinline__ int block_of(int u, int U, int S) { return (int)(((int64_t)S * (u + 1) - 1) / U); }
// (the fewest units that a further block is worth)
__device__ __forceinline__ int blocks_used(int U, int blocks, int least) { return max(1, min(blocks, U / least)); }

// A run of units of one item.
struct Segment {
    int g, pages, tile, column, record;
    int from, to;                                  // units of the item
};
// The segment that begins at unit u of a run that ends at `end`; g: a group at or before the unit's.
__device__ __forceinline__ Segment segment_at(const Groups& G, const int* units, const int* items, int g, int u, int end, int block) {
    Segment s;
    while (u >= units[g + 1]) ++g;
    s.g = g;
    s.pages = pages_of(G, g);
    const int per = units_per_item(G, s.pages), local = u - units[g], item = local / per;
    s.from = local - item * per;
    s.to = min(per, s.from + end - u);
    s.tile = item / G.columns;
    s.column = item - s.tile * G.columns;
    s.record = items[g] + item + block;            // (item and block rise together along the runs: no two segments share the sum)
    return s;
}

// The tcgen05 form of the shared part (attn_shared_tc.cu): bfloat16, tiles of TC_ROWS rows, units of two pages.
constexpr int TC_ROWS = 128;
bool tc_supported();
int launch_tc(const void* q, int n_tokens, const void* kv, int64_t kv_pages, const Groups& G, int blocks, float scale, int* plan, float* records, int* status,
              cudaStream_t s);

}  // namespace shared_prefix
}  // namespace wick
