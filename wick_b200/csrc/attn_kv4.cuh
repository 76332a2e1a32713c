// What the kernels of attention over a 4-bit cache share (attn_kv4.cu, attn_kv4_tc.cu): their arguments, how the work is cut, the fold of partial results.
#pragma once

#include "kv4.cuh"
#include "sm100.cuh"

#ifndef WICK_HD
#error "compile with -DWICK_HD=<head_dim>"
#endif

namespace wick {
namespace kv4 {

constexpr int D = WICK_HD;
static_assert(D % 64 == 0 && D >= 64 && D <= 256, "head sizes of 64, 128, 192 and 256");
typedef __nv_bfloat16 bf16;

constexpr int LEAVES = 8;                                        // of a node; warps of a block
constexpr int THREADS = LEAVES * 32;
constexpr int TILE = head_bytes(D);                              // a page of one key head
constexpr int NW = D / 32;                                       // words of a key that a lane reads (its quarter of the row)
constexpr int NV = D / 64;                                       // words of a value that a lane reads (its eighth)
constexpr int MAX_STAGES = D <= 128 ? 2 : 1;                      // of a warp's ring (eight rings of two larger tiles are more than an SM has)
constexpr int STAY_WARPS = D == 64 ? 16 : (D == 128 ? 12 : 8);   // of a block that stays (as many as registers allow)
constexpr int CLUSTER = 8;                                       // nodes that a cluster joins at most
constexpr int MAX_SEQS = 1024;                                   // of the form whose blocks stay
constexpr int MT = D / 16;                                       // tiles of 16 channels

// Nodes of the longest sequences: enough that one sequence alone gives nearly every SM a block (8 key heads: 16), no more (each costs a record).
__host__ __device__ inline int most_nodes(int n_kv) {
    const int n = 128 / n_kv;
    return n < 4 ? 4 : (n > 64 ? 64 : n);
}
__host__ __device__ inline int leaf_pages(int n_pages, int n_kv) {
    const int most = LEAVES * most_nodes(n_kv);
    return n_pages <= most ? 1 : (n_pages + most - 1) / most;
}
__host__ __device__ inline int nodes_of(int n_pages, int n_kv) {
    const int n = LEAVES * leaf_pages(n_pages, n_kv);
    return (n_pages + n - 1) / n;
}

struct Args {
    const void* q;                                               // [n_tokens, n_heads, d]
    void* out;
    const uint8_t* kv;
    int64_t kv_pages;
    const int* cu_seqlens;
    const int* start;
    const int* page_table;
    int table_width, n_seqs, n_heads, n_kv, group;
    float scale2;                                                // |scale| log2 e
    uint32_t flip;                                               // sign bits of two bfloat16 numbers if the scale is negative (the queries then change sign), else 0
    int n_tokens, max_q, pages;                                  // the most new tokens of a sequence, and the most pages that there are places for
    float* rec;                                                  // records: accumulators [row, node, d], then maximum and sum [row, node, 2]; a row is a (token, head)
    int64_t rec_rows;
    int nodes;                                                   // places for nodes in a row's records
    int tiles;                                                   // row tiles of a (sequence, key head) that the grid has
    int stages;                                                  // of a warp's ring
    int* status;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^(a - b) for maxima that may be -inf (nothing seen yet): then the weight is 0.
__device__ __forceinline__ float weight(float a, float b) { return a == -INFINITY ? 0.f : ex2(a - b); }
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same with nothing to add to.
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// An 8 x 8 matrix of 16-bit elements, a row per four lanes: the transposed one in the same layout.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ bool no_number(uint32_t scale) { return (scale & 0x7F80u) == 0x7F80u || (scale & 0x7F800000u) == 0x7F800000u; }
// The position (of 8) in row i of the instruction's position side.
__device__ __forceinline__ int position_of(int i) { return i ^ ((i >> 1) & 1); }

// A sequence's place in the step, as far as its rows see it.
struct Seq {
    int first, new_tokens, start, len, pages;                    // flat number of its first new token; ...; pages that fit its table
};
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
    Seq s;
    s.first = a.cu_seqlens[b];
    s.new_tokens = a.cu_seqlens[b + 1] - s.first;
    s.start = a.start[b];
    s.len = s.start + s.new_tokens;
    s.pages = (s.len + kPage - 1) / kPage;
    return s;
}
// Whether a sequence fits the step, its page table and the records' places (else it is left out, and said).
__device__ __forceinline__ bool fits(const Args& a, const Seq& s) {
    const bool ok = s.start >= 0 && s.first >= 0 && s.first + s.new_tokens <= a.n_tokens && s.new_tokens <= a.max_q && s.pages <= a.table_width && s.pages <= a.pages;
    if (!ok) atomicCAS(a.status, 0, 15);
    return ok;
}
// A page id, within the cache (else reported, and page 0).
__device__ __forceinline__ int checked_page(const Args& a, int id) {
    if (id < 0 || id >= a.kv_pages) {
        atomicCAS(a.status, 0, 15);
        return 0;
    }
    return id;
}
__device__ __forceinline__ void start_copy(const Args& a, int page, int kvh, uint8_t* dst, uint64_t* bar) {
    mbar_expect_tx(bar, TILE);
    bulk_load(dst, a.kv + ((int64_t)page * a.n_kv + kvh) * TILE, TILE, bar);
}

// The fold of a leaf (or a node) p into what came before, the same operations wherever it is done:
//   M' = max(M, m_p);  l = l 2^(M - M') + l_p 2^(m_p - M');  o likewise.
struct Fold {
    float m, l, was, now;
    __device__ __forceinline__ void step(float mp, float lp) {
        const float t = fmaxf(m, mp);
        was = weight(m, t);
        now = weight(mp, t);
        l = of(l, lp);
        m = t;
    }
    __device__ __forceinline__ float of(float o, float op) const { return __fmaf_rn(op, now, __fmul_rn(o, was)); }
};
__device__ __forceinline__ float result(float o, float l) { return __fmul_rn(o, __fdiv_rn(1.0f, l)); }

// Row i of a tile's unit n (rows 8 n ..): where its token's head lies in the step, or -1.
__device__ __forceinline__ int64_t flat_row(const Args& a, const Seq& s, int kvh, int row) {
    if (row >= s.new_tokens * a.group) return -1;
    const int tok = row / a.group;
    return (int64_t)(s.first + tok) * a.n_heads + kvh * a.group + (row - tok * a.group);
}
// A lane's four numbers of tile i (channels r d / 8 + 2 i and + 1 of rows 2 j and 2 j + 1): the result, or a node's record.
__device__ __forceinline__ void write_result(const Args& a, int64_t flat, int ch, float x, float y, float l) {
    *reinterpret_cast<uint32_t*>((bf16*)a.out + flat * D + ch) = pack_bf16(result(x, l), result(y, l));
}
__device__ __forceinline__ void write_record(const Args& a, int64_t flat, int node, int ch, float x, float y) {
    *reinterpret_cast<float2*>(a.rec + (flat * a.nodes + node) * D + ch) = make_float2(x, y);
}
__device__ __forceinline__ void write_weights(const Args& a, int64_t flat, int node, float m, float l) {
    *reinterpret_cast<float2*>(a.rec + a.rec_rows * a.nodes * D + (flat * a.nodes + node) * 2) = make_float2(m, l);
}

__device__ __forceinline__ uint32_t in_block(uint32_t smem, int rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem), "r"(rank));
    return at;
}
__device__ __forceinline__ float ld_cluster(uint32_t at) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Which kernels a call of these sizes launches, and what they need.
enum Form { AUTO = 0, PLAIN = 1, RECORDS = 2, CLUSTERS = 3, STAY = 4, STAY_LEAVES = 5, TC = 6, TC_CLUSTERS = 7 };
// The tcgen05 kernel (attn_kv4_tc.cu).  rows: of a tile (8, 16, 24 or 32).
int launch_tc(const Args& a, int rows, bool clusters, int64_t blocks, cudaStream_t s);
struct Plan {
    bool possible;
    int form, nt, rows, tiles, nodes, stages, kernels;
    int64_t scratch, blocks;
};
}  // namespace kv4
}  // namespace wick
