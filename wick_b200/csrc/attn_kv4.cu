// Causal attention over a cache that holds keys and values in 4 bits (kv4.cuh), for any number of new tokens a sequence.
//
//   out[i, h] = sum_t p_t v_t,  p = softmax over t <= position(i) of scale q[i, h] . k_t,  k_t and v_t the bfloat16 values that the codes stand for.
//
// How the work is cut.  The rows of a (sequence, key head) are its new tokens times the query heads of the key head; they come in tiles of 8, 16 or
// 24.  The sequence's pages are cut by its OWN length and the number of key heads alone: into leaves of as many pages (leaf_pages) and nodes of eight
// leaves.  A leaf is computed by one warp, page by page, into a running maximum, sum and accumulator; a node's leaves are folded in order, a row's nodes
// likewise.  While all sequences have up to eight rows, which warp computes what changes no bit, and a sequence's result does not depend on the batch
// it is in; with more rows tile, form and cut follow the whole step.  Three forms for bfloat16 (plan() has the rule):
//   * a block per node, a warp per leaf: the leaves meet in shared memory.  A sequence's nodes, where they are up to CLUSTER, are a cluster whose blocks
//     read each other's results and write the outcome; more leave records (accumulator, maximum, sum) that a second, small kernel joins.  Few nodes:
//     as many warps as there are leaves work on a sequence;
//   * blocks that stay, one per SM, with an equal run of all nodes of the step each, which their warps take one by one: a warp folds a node's leaves in
//     registers (with more than eight rows a node is one leaf), and its next page is on its way while it computes one.  Many nodes; records as above.
// A sequence with one node is written directly.
//
// The kernel on the tensor cores.  Keys and values stand on the 16-row side of mma.sync (16 positions, or 16 channels), the rows on the 8-column side, so
// that the eight rows of most head layouts fill it.  A page of one key head (80 d bytes) comes in one bulk copy.  Values are made from codes in registers, in
// the layout that the instruction wants: what a lane reads of a key are d / 4 neighbouring channels of a position (the queries are permuted to match),
// and of a value d / 8 neighbouring channels of four positions.  Rows 0, 1, ... 7 of the instruction's position side are
// the positions 0, 1, 3, 2, 4, 5, 7, 6 of eight, so that either reading touches every bank of the shared memory once.
//
// The float32 form (and the plain twin of the other): CUDA cores, the same leaves' values, everything in 32 bits.
#include "kv4.cuh"
#include "packed.cuh"
#include "tc_attention.cuh"

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
constexpr int CLUSTER = 8;                                       // nodes that a cluster joins at most
constexpr int MAX_SEQS = 1024;                                   // of the form whose blocks stay
constexpr int MT = D / 16;                                       // tiles of 16 channels
// What records may take.  A step with more than eight rows a sequence and key head whose records would take more is cut into fewer pieces: its row tiles alone are work
// enough then (2,000 tokens behind 62,000, 16 heads of 256 over one: 2,000 tiles, and records of 4.1 GB as cut by the length alone).  With up to eight rows
// the cut is the length's, and a node's records are a twentieth of the bytes of its pages at most (a leaf's, on the CUDA cores, two fifths).
constexpr int64_t RECORD_BYTES = 256 << 20;

// A leaf is one page while one sequence alone so gives every SM up to two blocks (8 key heads: 37 nodes, 296 pages).  Longer sequences have nodes for one block
// an SM (18) of long leaves, whose next page is on its way.  us, 32 heads over 8 of 128: 8 sequences of up to 12,000 positions, 24 nodes / 12 of twice the
// leaves 40 / 49, one of 12,000 12.8 / 11.8; one of up to 32,000, 32 nodes of 2 pages a leaf / 16 of 4: 22 / 17; two of up to 131,000, 64 heads, 37 / 18: 80 / 72.
// (148 and 296, one and two blocks for each SM of a B200, stand here as numbers: the cut, and with it a sequence's bits, does not follow the device.)
__host__ __device__ inline int most_nodes(int n_kv, int blocks) { return max(4, min(128, blocks / n_kv)); }
__host__ __device__ inline int leaf_pages(int n_pages, int n_kv) {
    const int most = LEAVES * most_nodes(n_kv, 148);
    return n_pages <= LEAVES * most_nodes(n_kv, 296) ? 1 : (n_pages + most - 1) / most;
}
__host__ __device__ inline int nodes_of(int n_pages, int n_kv) {
    const int n = LEAVES * leaf_pages(n_pages, n_kv);
    return (n_pages + n - 1) / n;
}
// The most that a sequence of up to n_pages has (a longer one can have fewer).
inline int most_leaves(int n_pages, int n_kv) { return min(n_pages, LEAVES * most_nodes(n_kv, 296)); }

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
    int whole;                                                   // sequences are not cut: a row tile is one node
    int most;                                                    // leaves of a sequence at most (RECORD_BYTES); 0: as its length says
    int* status;
};
__device__ __forceinline__ int leaf_pages(const Args& a, int n_pages) {
    if (a.whole) return n_pages;
    const int lp = leaf_pages(n_pages, a.n_kv);
    return a.most == 0 ? lp : max(lp, (n_pages + a.most - 1) / a.most);
}
__device__ __forceinline__ int nodes_of(const Args& a, int n_pages) {
    if (a.whole) return 1;
    const int n = LEAVES * leaf_pages(a, n_pages);
    return (n_pages + n - 1) / n;
}

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
// Whether a sequence fits the step, its page table and the records' places (else it is left out, and said).  (Sums of two numbers that may be anything
// are 64 bits wide: a start near 2^31 would else make a length below 0, which passes every bound.)
__device__ __forceinline__ bool fits(const Args& a, const Seq& s) {
    const bool ok = s.start >= 0 && s.first >= 0 && s.new_tokens >= 0 && (int64_t)s.first + s.new_tokens <= a.n_tokens && s.new_tokens <= a.max_q &&
                    (int64_t)s.start + s.new_tokens <= (int64_t)min(a.table_width, a.pages) * kPage;
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
// The same for the neighbours 2 j, 2 j + 1 of a lane's rows, two numbers an instruction.
__device__ __forceinline__ void fold_pair(const Fold (&f)[2], float& o0, float& o1, float p0, float p1) {
    const float2 r = fma2(make_float2(p0, p1), make_float2(f[0].now, f[1].now), mul2(make_float2(o0, o1), make_float2(f[0].was, f[1].was)));
    o0 = r.x;
    o1 = r.y;
}
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
enum Form { AUTO = 0, PLAIN = 1, RECORDS = 2, CLUSTERS = 3, STAY = 4 };
struct Plan {
    bool possible;
    int form, nt, tiles, nodes, stages, whole, most, kernels;
    int64_t scratch, blocks;
};

// ---- one page on the tensor cores -------------------------------------------------------
template <int NT> struct Sum {                                   // of a leaf or a node: lane (r, j) = (lane / 4, lane % 4) holds rows 2 j, 2 j + 1 of every eight,
    float o[MT][NT][4];                                          //   channels r d / 8 + 2 m (o[m][.][0], [1]) and + 1 ([2], [3])
    float m[NT][2], l[NT][2];                                    //   (l: the lane's share until finish_leaf)
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int i = 0; i < MT; ++i) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.f;
        }
    }
};

template <int NT> struct Rows {
    uint32_t q[2 * NW][NT][2];                                   // the second operand of the scores, channels in the order of the keys' codes
    int limit[NT][2];                                            // the last position that rows 2 j, 2 j + 1 see
};

// Rows row0 .. of a (sequence, key head): row i is head i % group of new token i / group.  A lane has its quarter of rows r, 8 + r ..; first as they are in
// memory (fetch_rows), then in the order of the keys' codes (order_rows, in place).
template <int NT>
__device__ __forceinline__ void fetch_rows(const Args& a, const Seq& s, int kvh, int row0, Rows<NT>& w) {
    const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int row = row0 + 8 * n + r, tok = row / a.group, g = row - tok * a.group;
        const uint4* src = reinterpret_cast<const uint4*>((const bf16*)a.q + ((int64_t)(s.first + tok) * a.n_heads + kvh * a.group + g) * D + 8 * j * NW);
        const bool there = row < s.new_tokens * a.group;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const uint4 x = there ? src[i] : make_uint4(0, 0, 0, 0);
            w.q[2 * i][n][0] = x.x;
            w.q[2 * i][n][1] = x.y;
            w.q[2 * i + 1][n][0] = x.z;
            w.q[2 * i + 1][n][1] = x.w;
        }
    }
}
template <int NT>
__device__ __forceinline__ void order_rows(const Args& a, Rows<NT>& w) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const uint32_t x = w.q[2 * i][n][0] ^ a.flip, y = w.q[2 * i][n][1] ^ a.flip, z = w.q[2 * i + 1][n][0] ^ a.flip, v = w.q[2 * i + 1][n][1] ^ a.flip;
            w.q[2 * i][n][0] = low_halves(x, z);
            w.q[2 * i][n][1] = high_halves(x, z);
            w.q[2 * i + 1][n][0] = low_halves(y, v);
            w.q[2 * i + 1][n][1] = high_halves(y, v);
        }
}
template <int NT>
__device__ __forceinline__ void load_rows(const Args& a, const Seq& s, int kvh, int row0, Rows<NT>& w) {
    const int j = threadIdx.x & 3, n_rows = s.new_tokens * a.group;
    fetch_rows<NT>(a, s, kvh, row0, w);
    order_rows<NT>(a, w);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) w.limit[n][c] = s.start + min(row0 + 8 * n + 2 * j + c, n_rows - 1) / a.group;
}

template <int N> __device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 x = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const uint2 x = reinterpret_cast<const uint2*>(p)[i];
            w[2 * i] = x.x; w[2 * i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
    }
}

// One page (in shared memory) into a leaf.  MASK: some of its positions are not seen by some row; first: the position of the page's first row, len: the
// sequence's length; several: rows of several tokens.  FRESH: the leaf's first page (nothing is in the sum, its members have no value yet).  between: what is to be done when the keys have been read and before
// the values are.
template <int NT, bool MASK, bool FRESH, typename Between>
__device__ __forceinline__ void page_step(const uint8_t* tile, const Rows<NT>& w, float scale2, int first, int len, bool several, Sum<NT>& sum, Between between) {
    const int lane = threadIdx.x & 31, r = lane >> 2, j = lane & 3;
    const int tr = position_of(r), ta = position_of(2 * j), tb = position_of(2 * j + 1);
    float s[4][NT][4];
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
        uint32_t k[2][NW];
        const uint8_t* sc[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int t = mt * 16 + 8 * u + tr;
            load_words<NW>(tile + t * (D / 2) + j * (D / 8), k[u]);
            sc[u] = tile + key_scales(D) + t * (D / 8);
        }
        uint32_t a2[2], b2[2];
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            if (i % (D == 192 ? 2 : 4) == 0) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t x = *reinterpret_cast<const uint32_t*>(sc[u] + ((j * NW + i) >> 2) * 4);
                    a2[u] = low_halves(x, x);
                    b2[u] = high_halves(x, x);
                }
            }
            uint32_t v0[4], v1[4];
            key_word(k[0][i], a2[0], b2[0], v0);
            key_word(k[1][i], a2[1], b2[1], v1);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (i == 0) mma16816_first(s[mt][n], v0[0], v1[0], v0[1], v1[1], w.q[2 * i][n][0], w.q[2 * i][n][1]);
                else mma16816(s[mt][n], v0[0], v1[0], v0[1], v1[1], w.q[2 * i][n][0], w.q[2 * i][n][1]);
                mma16816(s[mt][n], v0[2], v1[2], v0[3], v1[3], w.q[2 * i + 1][n][0], w.q[2 * i + 1][n][1]);
            }
        }
    }
    between();
    // the running maximum in units of log2 e, weights
    uint32_t p[4][NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        if (MASK) {
#pragma unroll
            for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (first + mt * 16 + 8 * (e >> 1) + tr > w.limit[n][e & 1]) s[mt][n][e] = -INFINITY;
        }
        float was[2], ref[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float top = max3(max3(s[0][n][c], s[0][n][c + 2], s[1][n][c]), max3(s[1][n][c + 2], s[2][n][c], s[2][n][c + 2]), fmaxf(s[3][n][c], s[3][n][c + 2]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float mine = top == -INFINITY ? top : top * scale2, m = FRESH ? mine : fmaxf(sum.m[n][c], mine);
            was[c] = FRESH ? 0.f : weight(sum.m[n][c], m);
            ref[c] = m == -INFINITY ? 0.f : -m;                  // (nothing seen: weights 0; a score that is no number still shows)
            sum.m[n][c] = m;
        }
        float2 l = make_float2(0.f, 0.f);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int h = 0; h < 4; h += 2) {
                const float2 x = fma2(make_float2(s[mt][n][h], s[mt][n][h + 1]), make_float2(scale2, scale2), make_float2(ref[0], ref[1]));
                // (a scale of 0 and a position that is not seen would else give a number that is none)
                const float2 y = make_float2(MASK && s[mt][n][h] == -INFINITY ? 0.f : ex2(x.x), MASK && s[mt][n][h + 1] == -INFINITY ? 0.f : ex2(x.y));
                s[mt][n][h] = y.x;
                s[mt][n][h + 1] = y.y;
                l = add2(l, y);
            }
        sum.l[n][0] = FRESH ? l.x : sum.l[n][0] * was[0] + l.x;
        sum.l[n][1] = FRESH ? l.y : sum.l[n][1] * was[1] + l.y;
        if (!FRESH && __any_sync(0xffffffffu, was[0] != 1.f || was[1] != 1.f)) {
            const float2 f = make_float2(was[0], was[1]);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int h = 0; h < 4; h += 2) {
                    const float2 x = mul2(make_float2(sum.o[i][n][h], sum.o[i][n][h + 1]), f);
                    sum.o[i][n][h] = x.x;
                    sum.o[i][n][h + 1] = x.y;
                }
        }
        // The weights enter the second product as bfloat16 numbers (the sum above has them unrounded: at most 2^-9 each, as in the other kernels).
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) {
            p[mt][n][0] = transpose8x8(pack_bf16(s[mt][n][0], s[mt][n][1]));
            p[mt][n][1] = transpose8x8(pack_bf16(s[mt][n][2], s[mt][n][3]));
        }
    }
#pragma unroll
    for (int mt = 0; mt < 4; ++mt) {
        uint32_t v[4][NV];                                       // positions ta, tb of the first eight, of the second
        const uint8_t* sc[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = mt * 16 + 8 * (u >> 1) + (u & 1 ? tb : ta);
            load_words<NV>(tile + value_codes(D) + t * (D / 2) + value_byte<D>(t, r * (D / 16)), v[u]);
            sc[u] = tile + value_scales(D) + t * (D / 8);
        }
        uint32_t a2[2], b2[2];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i == 0 || D == 192) {
                uint32_t x[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    x[u] = *reinterpret_cast<const uint32_t*>(sc[u] + ((r * NV + i) >> 2) * 4);
                    if (MASK) {                                  // (behind the sequence's end: anything may lie there; a value that is no number: see below)
                        const int t = first + mt * 16 + 8 * (u >> 1) + (u & 1 ? tb : ta);
                        if (t >= len || (several && no_number(x[u]))) x[u] = 0;
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    a2[u] = low_halves(x[2 * u], x[2 * u + 1]);
                    b2[u] = high_halves(x[2 * u], x[2 * u + 1]);
                }
            }
            uint32_t e[4][2], o[4][2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                value_pair<0>(v[2 * u][i], v[2 * u + 1][i], a2[u], b2[u], e[0][u], o[0][u]);
                value_pair<1>(v[2 * u][i], v[2 * u + 1][i], a2[u], b2[u], e[1][u], o[1][u]);
                value_pair<2>(v[2 * u][i], v[2 * u + 1][i], a2[u], b2[u], e[2][u], o[2][u]);
                value_pair<3>(v[2 * u][i], v[2 * u + 1][i], a2[u], b2[u], e[3][u], o[3][u]);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    if (FRESH && mt == 0) mma16816_first(sum.o[4 * i + k][n], e[k][0], o[k][0], e[k][1], o[k][1], p[mt][n][0], p[mt][n][1]);
                    else mma16816(sum.o[4 * i + k][n], e[k][0], o[k][0], e[k][1], o[k][1], p[mt][n][0], p[mt][n][1]);
                }
        }
    }
    if (MASK && several) {
        // A value that is no number shows in the rows that see its position, and in no others (a weight of 0 would not hide it in the product).
        const uint32_t* all = reinterpret_cast<const uint32_t*>(tile + value_scales(D));
        bool any = false;
        for (int i = lane; i < kPage * NW; i += 32) any |= first + i / NW < len && no_number(all[i]);
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll 1
            for (int t = 0; t < kPage && first + t < len; ++t)
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (no_number(all[t * NW + ((r * NV + i) >> 2)]))
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int c = 0; c < 2; ++c)
                                if (first + t <= w.limit[n][c])
#pragma unroll
                                    for (int k = 0; k < 4; ++k) sum.o[4 * i + k][n][c] = sum.o[4 * i + k][n][c + 2] = __int_as_float(0x7FFFFFFF);
        }
    }
}

struct Nothing {
    __device__ __forceinline__ void operator()() const {}
};
// (single: leaves of one page.  Other leaves take their first page as any other, so that the warps of a block run the same code.)
template <int NT, typename Between = Nothing>
__device__ __forceinline__ void leaf_page(const Args& a, const uint8_t* tile, const Rows<NT>& w, const Seq& s, int page, bool fresh, bool single, Sum<NT>& sum,
                                          Between between = Nothing()) {
    const int first = page * kPage;
    const bool mask = first + kPage - 1 > s.start;
    if (fresh && (mask || !single)) sum.clear();
    if (mask) page_step<NT, true, false>(tile, w, a.scale2, first, s.len, s.new_tokens > 1, sum, between);
    else if (single) page_step<NT, false, true>(tile, w, a.scale2, first, s.len, false, sum, between);
    else page_step<NT, false, false>(tile, w, a.scale2, first, s.len, false, sum, between);
}

// A leaf's sum over its positions: every lane gets its rows'.
template <int NT> __device__ __forceinline__ void finish_leaf(Sum<NT>& sum) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) sum.l[n][c] += __shfl_xor_sync(0xffffffffu, sum.l[n][c], o);
}

// ---- a block per node ---------------------------------------------------------------------
constexpr int leaves_smem(int nt, int stages, bool clusters) { return LEAVES * stages * TILE + (clusters ? nt * 8 * D * 4 : 0); }

// The grid: nodes innermost, then tiles, heads, sequences.  CLUSTERS: a sequence's nodes are a cluster.
// What bounds it: with few nodes the way of one page through the warp (table, copy, scores, values, fold, join), 7 us with the launch; with many as above.
// 8 sequences of up to 4,000 positions, 32 heads over 8 of 128: 17 us.
template <int NT, bool CLUSTERS>
__global__ void __launch_bounds__(THREADS, NT == 1 && D <= 128 ? 2 : 1) leaves_kernel(const Args a) {
    extern __shared__ __align__(128) uint8_t ring_all[];
    __shared__ uint64_t full[LEAVES][2];
    __shared__ float stat_m[LEAVES][8 * NT], stat_l[LEAVES][8 * NT];
    __shared__ float node_m[8 * NT], node_l[8 * NT];
    __shared__ int abort_flag;
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, j = lane & 3;
    unsigned at = blockIdx.x;
    const int node = (int)(at % (unsigned)a.nodes);
    at /= (unsigned)a.nodes;
    const int tile = (int)(at % (unsigned)a.tiles);
    at /= (unsigned)a.tiles;
    const int kvh = (int)(at % (unsigned)a.n_kv), b = (int)(at / (unsigned)a.n_kv);
    const Seq s = sequence(a, b);
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int w = 0; w < LEAVES; ++w) {
            mbar_init(&full[w][0], 1);
            mbar_init(&full[w][1], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const int n_rows = s.new_tokens * a.group, row0 = tile * 8 * NT;
    const int last = (min(row0 + 8 * NT, n_rows) - 1) / a.group;
    const int seen = (s.start + last) / kPage + 1;               // pages that any row of the tile sees
    const int lp = a.whole ? (seen + LEAVES - 1) / LEAVES : leaf_pages(a, s.pages);
    const int first_page = node * LEAVES * lp;
    pdl_wait();
    if (row0 >= n_rows || !fits(a, s)) return;                   // (so do all blocks of its cluster)
    if (first_page >= seen) return;                              // (a cluster does not wait for blocks that have left)
    const int n_nodes = CLUSTERS ? (seen + LEAVES * lp - 1) / (LEAVES * lp) : nodes_of(a, s.pages);
    const int p0 = first_page + warp * lp, count = max(0, min(seen, p0 + lp) - p0);
    uint8_t* ring = ring_all + (size_t)warp * a.stages * TILE;
    int ids = 0;
    auto issue = [&](int k) {                                    // (in order; the lanes hold 32 page ids at a time)
        if ((k & 31) == 0 && k + lane < count) ids = checked_page(a, a.page_table[(int64_t)b * a.table_width + p0 + k + lane]);
        const int id = __shfl_sync(0xffffffffu, ids, k & 31);
        if (lane == 0) start_copy(a, id, kvh, ring + (k % a.stages) * TILE, &full[warp][k % a.stages]);
    };
    for (int k = 0; k < min(a.stages, count); ++k) issue(k);
    Sum<NT> sum;
    if (count == 0) sum.clear();
    if (count > 0) {
        Rows<NT> w;
        load_rows<NT>(a, s, kvh, row0, w);
#pragma unroll 1
        for (int k = 0; k < count; ++k) {
            // (all lanes leave together: those whose wait runs out as those that saw the copy arrive in the same instant)
            if (!__all_sync(0xffffffffu, mbar_wait(&full[warp][k % a.stages], (k / a.stages) & 1, &abort_flag, a.status, 16))) {
                // (what is on its way has to arrive before this block's shared memory is somebody else's; again with a limit)
                for (int i = k; i < min(count, k + a.stages); ++i) {
                    int mine = 0;
                    mbar_wait(&full[warp][i % a.stages], (i / a.stages) & 1, &mine, a.status, 16);
                }
                break;
            }
            leaf_page<NT>(a, ring + (k % a.stages) * TILE, w, s, p0 + k, k == 0, lp == 1, sum);
            __syncwarp();
            if (k + a.stages < count) issue(k + a.stages);
        }
        finish_leaf<NT>(sum);
    }
    // The leaves meet: registers as they are, behind one another, in each warp's own part of the ring.
    if (r == 0) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                stat_m[warp][8 * n + 2 * j + c] = sum.m[n][c];
                stat_l[warp][8 * n + 2 * j + c] = sum.l[n][c];
            }
    }
    if (count > 0) {
        float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) mine[((i * NT + n) * 4 + e) * 32 + lane] = sum.o[i][n][e];
    }
    __syncthreads();
    const int leaves = min(LEAVES, (seen - first_page + lp - 1) / lp);
    float* rec = reinterpret_cast<float*>(ring_all + LEAVES * a.stages * TILE);
#pragma unroll 1
    for (int u = warp; u < MT * NT; u += LEAVES) {
        const int i = u / NT, n = u % NT;
        // Lane (p, j) has the fold's step of leaf p for rows 2 j, 2 j + 1: the maxima so far by a scan over the leaves.
        float was[2], now[2], m[2], l[2] = {0.f, 0.f}, lp_[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float mine = r < leaves ? stat_m[r][8 * n + 2 * j + c] : -INFINITY;
            lp_[c] = r < leaves ? stat_l[r][8 * n + 2 * j + c] : 0.f;
            float upto = mine;
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                const float t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto = fmaxf(upto, t);
            }
            float before = __shfl_up_sync(0xffffffffu, upto, 4);
            if (r == 0) before = -INFINITY;
            was[c] = weight(before, upto);
            now[c] = weight(mine, upto);
            m[c] = __shfl_sync(0xffffffffu, upto, 28 + j);
        }
        float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int p = 0; p < leaves; ++p) {
            const float* theirs = reinterpret_cast<const float*>(ring_all + (size_t)p * a.stages * TILE) + u * 4 * 32 + lane;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                Fold f;
                f.was = __shfl_sync(0xffffffffu, was[c], 4 * p + j);
                f.now = __shfl_sync(0xffffffffu, now[c], 4 * p + j);
                l[c] = f.of(l[c], __shfl_sync(0xffffffffu, lp_[c], 4 * p + j));
                o[c] = f.of(o[c], theirs[c * 32]);
                o[c + 2] = f.of(o[c + 2], theirs[(c + 2) * 32]);
            }
        }
        if (CLUSTERS && n_nodes > 1) {
#pragma unroll
            for (int e = 0; e < 4; ++e) rec[(u * 4 + e) * 32 + lane] = o[e];
            if (i == 0 && r == 0) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    node_m[8 * n + 2 * j + c] = m[c];
                    node_l[8 * n + 2 * j + c] = l[c];
                }
            }
            continue;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int64_t flat = flat_row(a, s, kvh, row0 + 8 * n + 2 * j + c);
            if (flat < 0) continue;
            const int ch = r * (D / 8) + 2 * i;
            if (n_nodes == 1) {
                write_result(a, flat, ch, o[c], o[c + 2], l[c]);
            } else {
                write_record(a, flat, node, ch, o[c], o[c + 2]);
                if (i == 0 && r == 0) write_weights(a, flat, node, m[c], l[c]);
            }
        }
    }
    if constexpr (CLUSTERS) {
        if (n_nodes == 1) return;                                // (all blocks of the cluster know)
        // The nodes meet: the tiles of 16 channels are shared out among the blocks' warps, and joined out of all blocks' shared memory, in the nodes' order.
        cluster_sync();
#pragma unroll 1
        for (int u = warp * n_nodes + node; u < MT * NT; u += LEAVES * n_nodes) {
            const int i = u / NT, n = u % NT;
            Fold f[2];
            float o[4] = {0.f, 0.f, 0.f, 0.f};
            f[0].m = f[1].m = -INFINITY;
            f[0].l = f[1].l = 0.f;
#pragma unroll 4
            for (int p = 0; p < n_nodes; ++p) {
                const uint32_t theirs = in_block(smem_u32(rec + u * 4 * 32 + lane), p);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    f[c].step(ld_cluster(in_block(smem_u32(&node_m[8 * n + 2 * j + c]), p)), ld_cluster(in_block(smem_u32(&node_l[8 * n + 2 * j + c]), p)));
                    o[c] = f[c].of(o[c], ld_cluster(theirs + c * 128));
                    o[c + 2] = f[c].of(o[c + 2], ld_cluster(theirs + (c + 2) * 128));
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int64_t flat = flat_row(a, s, kvh, row0 + 8 * n + 2 * j + c);
                if (flat >= 0) write_result(a, flat, r * (D / 8) + 2 * i, o[c], o[c + 2], f[c].l);
            }
        }
        cluster_sync();                                          // (nobody leaves while others read)
    }
}

// ---- blocks that stay ------------------------------------------------------------------------
// A block has a run of the step's items (a node of a row tile of a key head of a sequence each) with an equal part of the pages, or of the items while each has
// a warp, and its warps take the next one whenever they are done with one.  64 sequences of 6,000 to 12,000 positions, 16 heads of 128, nodes of 8 to 24
// pages: equal parts of the nodes 605 us, of the pages 382; 16 of 2,000 to 4,000: 38, 51 (some blocks have more nodes than warps).
// A warp's tile is filled again while it is read: the next page's keys as soon as the scores are there, its values when the page is done.
// One unit of rows (NT 1): a node's leaves are folded in registers.  More: there is no room for a second accumulator, and a node is one leaf.
// What bounds it: the instructions that make values of codes (654 of a page's 1,331, half as fast as the others) and the matrix instructions beside them, which
// mostly add up: a scheduler is active for 2,600 clocks a page, with two warps as with three (whose waits for one another are a part of it).  64 sequences of 4,000
// to 8,191 positions, 32 heads over 8 of 128 (504 MB of pages): 130 us, 59 % of the copy's rate; at 133, 8 warps a block took 140, 16 (which spill) 149.
struct Item {
    int b, kvh, row0, place, lp;                                 // place: the node's number in the sequence; none left: b < 0
    int page, end;                                               // of the sequence, as far as the row tile sees
    int alone;                                                   // the sequence has one node
};
// An item's pages, about (nodes of a long sequence have more than those of a short one), and one for what goes with it.
__device__ __forceinline__ int item_work(const Args& a, int n_pages) {
    const int nodes = max(1, nodes_of(a, n_pages));
    return (n_pages + nodes - 1) / nodes + 1;
}
template <int NT> constexpr int stay_warps() { return NT > 1 || D > 128 ? 8 : (D == 64 ? 16 : 12); }      // (as many as registers allow)

template <int NT>
__global__ void __launch_bounds__(stay_warps<NT>() * 32, 1) stay_kernel(const Args a) {
    constexpr int WARPS = stay_warps<NT>();
    extern __shared__ __align__(128) uint8_t ring_all[];
    __shared__ uint64_t full[WARPS][2];                          // keys, values
    __shared__ int cum[MAX_SEQS + 1], lens[MAX_SEQS], firsts[MAX_SEQS + 1];  // items before a sequence; its length (with new tokens) and the first of these
    __shared__ int64_t work[MAX_SEQS + 1];                       // pages, about, before a sequence
    __shared__ int abort_flag, taken, end_of_run;
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, j = lane & 3;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int w = 0; w < WARPS; ++w) {
            mbar_init(&full[w][0], 1);
            mbar_init(&full[w][1], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    for (int b = threadIdx.x; b < a.n_seqs; b += WARPS * 32) {
        const Seq s = sequence(a, b);
        cum[b + 1] = s.new_tokens > 0 && fits(a, s) ? nodes_of(a, s.pages) * ((s.new_tokens * a.group + 8 * NT - 1) / (8 * NT)) * a.n_kv : 0;
        work[b + 1] = (int64_t)cum[b + 1] * item_work(a, s.pages);
        lens[b] = s.len;
        firsts[b] = s.first;
        if (b == a.n_seqs - 1) firsts[b + 1] = s.first + s.new_tokens;
    }
    __syncthreads();
    if (warp == 0) {
        int before = 0;
        int64_t work_before = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
            const int b = s0 + lane;
            int upto = b < a.n_seqs ? cum[b + 1] : 0;
            int64_t work_upto = b < a.n_seqs ? work[b + 1] : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int t = __shfl_up_sync(0xffffffffu, upto, o);
                const int64_t u = __shfl_up_sync(0xffffffffu, work_upto, o);
                if (lane >= o) {
                    upto += t;
                    work_upto += u;
                }
            }
            if (b < a.n_seqs) {
                cum[b + 1] = before + upto;
                work[b + 1] = work_before + work_upto;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
            work_before += __shfl_sync(0xffffffffu, work_upto, 31);
        }
        if (lane == 0) {
            cum[0] = 0;
            work[0] = 0;
        }
        __syncwarp();
        if (lane < 2) {                                          // the first item of this block's run, and of the next one's
            const int64_t block = blockIdx.x + lane;
            int first = (int)(block * before / gridDim.x);       // (a warp for every item: equal numbers)
            if (before > WARPS * (int)gridDim.x && block < gridDim.x) {
                const int64_t at = (int64_t)((double)work_before * block / gridDim.x);
                int lo = 0, hi = a.n_seqs - 1;                   // the last sequence with work[b] <= at
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (work[mid] <= at) lo = mid;
                    else hi = mid - 1;
                }
                const int one = item_work(a, (lens[lo] + kPage - 1) / kPage);
                first = cum[lo] + (int)min((at - work[lo] + one - 1) / one, (int64_t)(cum[lo + 1] - cum[lo]));
            }
            *(lane == 0 ? &taken : &end_of_run) = first;
        }
    }
    __syncthreads();
    const int stop = end_of_run;
    pdl_wait();
    uint8_t* tile = ring_all + (size_t)warp * TILE;

    auto place_of = [&](int b) {
        Seq s;
        s.first = firsts[b];
        s.new_tokens = firsts[b + 1] - s.first;
        s.len = lens[b];
        s.start = s.len - s.new_tokens;
        s.pages = (s.len + kPage - 1) / kPage;
        return s;
    };
    auto take = [&](Item& n, int& ids) {
        while (true) {
            int u = 0;
            if (lane == 0) u = atomicAdd(&taken, 1);
            u = __shfl_sync(0xffffffffu, u, 0);
            n.b = -1;
            if (u >= stop) break;
            int lo = 0, hi = a.n_seqs - 1;                       // the last sequence with cum[b] <= u
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (cum[mid] <= u) lo = mid;
                else hi = mid - 1;
            }
            n.b = lo;
            const Seq s = place_of(lo);
            const int local = u - cum[lo], n_rows = s.new_tokens * a.group, tiles = (n_rows + 8 * NT - 1) / (8 * NT), nodes = nodes_of(a, s.pages);
            n.lp = leaf_pages(a, s.pages);
            n.place = local % nodes;
            n.row0 = NT == 1 && tiles == 1 ? 0 : local / nodes % tiles * 8 * NT;
            n.kvh = local / (nodes * tiles);
            n.alone = nodes == 1;
            const int seen = (s.start + (min(n.row0 + 8 * NT, n_rows) - 1) / a.group) / kPage + 1;
            n.page = n.place * LEAVES * n.lp;
            n.end = min(seen, n.page + LEAVES * n.lp);
            if (n.page >= seen) continue;                        // (the tile's rows see none of it)
            ids = n.page + lane < n.end ? checked_page(a, a.page_table[(int64_t)lo * a.table_width + n.page + lane]) : 0;
            break;
        }
    };
    auto start_half = [&](int id, int kvh, int half) {           // keys or values of a page: their codes and their scales
        if (lane == 0) {
            const uint8_t* src = a.kv + ((int64_t)id * a.n_kv + kvh) * TILE;
            mbar_expect_tx(&full[warp][half], TILE / 2);
            bulk_load(tile + half * value_codes(D), src + half * value_codes(D), 32 * D, &full[warp][half]);
            bulk_load(tile + key_scales(D) + half * 8 * D, src + key_scales(D) + half * 8 * D, 8 * D, &full[warp][half]);
        }
    };
    Item cn, nn;                                                 // the item that is computed, and the next one
    int ids = 0, next_ids = 0, parity = 0;
    take(cn, ids);
    if (cn.b < 0) return;
    {
        const int id = __shfl_sync(0xffffffffu, ids, 0);
        start_half(id, cn.kvh, 0);
        start_half(id, cn.kvh, 1);
    }
    Rows<NT> w;
    fetch_rows<NT>(a, place_of(cn.b), cn.kvh, cn.row0, w);
#pragma unroll 1
    while (true) {
        const Seq s = place_of(cn.b);
        order_rows<NT>(a, w);
        const int n_rows = s.new_tokens * a.group;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) w.limit[n][c] = s.start + min(cn.row0 + 8 * n + 2 * j + c, n_rows - 1) / a.group;
        take(nn, next_ids);
        Fold f[2];
        float o[NT == 1 ? MT : 1][4];
        Sum<NT> sum;
        if (NT == 1) {
            f[0].m = f[1].m = -INFINITY;
            f[0].l = f[1].l = 0.f;
#pragma unroll
            for (int i = 0; i < (NT == 1 ? MT : 1); ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        }
        int held = 0;                                            // of the 32 ids that the lanes have
#pragma unroll 1
        for (int page = cn.page; page < cn.end;) {
            const int leaf_end = NT == 1 ? min(cn.end, page + cn.lp) : cn.end;
            bool fresh = true;
#pragma unroll 1
            for (; page < leaf_end; ++page) {
                int next_id = -1, next_kvh = cn.kvh;
                bool ok = mbar_wait(&full[warp][0], parity, &abort_flag, a.status, 16);
                const bool keys = ok;                            // (of lane 0, which starts the copies)
                leaf_page<NT>(a, tile, w, s, page, fresh, NT == 1 && cn.lp == 1, sum, [&]() {
                    if (page + 1 < cn.end) {
                        if (++held == 32) {
                            held = 0;
                            ids = page + 1 + lane < cn.end ? checked_page(a, a.page_table[(int64_t)cn.b * a.table_width + page + 1 + lane]) : 0;
                        }
                        next_id = __shfl_sync(0xffffffffu, ids, held);
                    } else if (nn.b >= 0) {
                        next_id = __shfl_sync(0xffffffffu, next_ids, 0);
                        next_kvh = nn.kvh;
                    }
                    __syncwarp();
                    if (next_id >= 0 && keys) start_half(next_id, next_kvh, 0);
                    // (the queries are not needed any more behind a node's last scores: the next item's are asked for)
                    if (NT == 1 && page + 1 == cn.end && nn.b >= 0) fetch_rows<NT>(a, place_of(nn.b), nn.kvh, nn.row0, w);
                    // (all lanes leave together: a wait may run out for one as the copy arrives for another)
                    ok = __all_sync(0xffffffffu, mbar_wait(&full[warp][1], parity, &abort_flag, a.status, 16) && ok);
                });
                if (!ok) {                                       // (what is on its way has to arrive before this shared memory is somebody else's)
                    int mine = 0;
                    if (lane == 0) mbar_wait(&full[warp][0], next_id >= 0 && keys ? parity ^ 1 : parity, &mine, a.status, 16);
                    mine = 0;
                    if (lane == 0) mbar_wait(&full[warp][1], parity, &mine, a.status, 16);
                    return;
                }
                fresh = false;
                parity ^= 1;
                __syncwarp();
                if (next_id >= 0) start_half(next_id, next_kvh, 1);
            }
            finish_leaf<NT>(sum);
            if constexpr (NT == 1) {
#pragma unroll
                for (int c = 0; c < 2; ++c) f[c].step(sum.m[0][c], sum.l[0][c]);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    fold_pair(f, o[i][0], o[i][1], sum.o[i][0][0], sum.o[i][0][1]);
                    fold_pair(f, o[i][2], o[i][3], sum.o[i][0][2], sum.o[i][0][3]);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int64_t flat = flat_row(a, s, cn.kvh, cn.row0 + 8 * n + 2 * j + c);
                if (flat < 0) continue;
                const float l = NT == 1 ? f[c].l : sum.l[n][c];
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const float x = NT == 1 ? o[NT == 1 ? i : 0][c] : sum.o[i][n][c], y = NT == 1 ? o[NT == 1 ? i : 0][c + 2] : sum.o[i][n][c + 2];
                    if (cn.alone) write_result(a, flat, r * (D / 8) + 2 * i, x, y, l);
                    else write_record(a, flat, cn.place, r * (D / 8) + 2 * i, x, y);
                }
                if (!cn.alone && r == 0) write_weights(a, flat, cn.place, NT == 1 ? f[c].m : sum.m[n][c], l);
            }
        if (nn.b < 0) return;
        if (NT > 1) fetch_rows<NT>(a, place_of(nn.b), nn.kvh, nn.row0, w);
        cn = nn;
        ids = next_ids;
    }
}

// ---- joining the nodes ----------------------------------------------------------------------
// A warp per row (a token's head): its records folded in order.  BY_LEAF: records of leaves, folded to nodes first.  Sequences with one node (leaf) have
// been written already.
template <typename T, bool BY_LEAF>
__global__ void __launch_bounds__(128) join_kernel(const Args a, const int* __restrict__ seq_of_token, int n_tokens) {
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int tok = (int)min(row / a.n_heads, (int64_t)n_tokens - 1), b = seq_of_token[tok];
    const Seq s = sequence(a, min(max(b, 0), a.n_seqs - 1));
    pdl_wait();
    if (row >= (int64_t)n_tokens * a.n_heads || b < 0 || b >= a.n_seqs) return;
    if (tok < s.first || tok >= s.first + s.new_tokens) return;  // (a token that fills the step up)
    if (!fits(a, s)) return;
    const int seen = (s.start + tok - s.first) / kPage + 1, per = (BY_LEAF ? 1 : LEAVES) * leaf_pages(a, s.pages), n = (seen + per - 1) / per;
    if (s.pages <= per) return;
    const float* o_rec = fresh(a.rec) + row * a.nodes * D;
    const float* m_rec = fresh(a.rec) + a.rec_rows * a.nodes * D + row * a.nodes * 2;
    Fold f, g;
    g.m = f.m = -INFINITY;
    g.l = f.l = 0.f;
    float2 o[D / 64], x[D / 64];
#pragma unroll
    for (int e = 0; e < D / 64; ++e) x[e] = o[e] = make_float2(0.f, 0.f);
    auto fold = [](Fold& t, float2 (&into)[D / 64], float m, float l, const float2 (&y)[D / 64]) {
        t.step(m, l);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
            into[e].x = t.of(into[e].x, y[e].x);
            into[e].y = t.of(into[e].y, y[e].y);
        }
    };
#pragma unroll 1
    for (int p0 = 0; p0 < n; p0 += LEAVES) {                     // (a node's leaves, or eight nodes: asked for together)
        float2 ml[LEAVES], y[LEAVES][D / 64];
#pragma unroll
        for (int p = 0; p < LEAVES; ++p) {
            if (p0 + p < n) {
                ml[p] = *reinterpret_cast<const float2*>(m_rec + 2 * (p0 + p));
#pragma unroll
                for (int e = 0; e < D / 64; ++e) y[p][e] = *reinterpret_cast<const float2*>(o_rec + (int64_t)(p0 + p) * D + 64 * e + 2 * lane);
            }
        }
#pragma unroll
        for (int p = 0; p < LEAVES; ++p)
            if (p0 + p < n) fold(BY_LEAF ? g : f, BY_LEAF ? x : o, ml[p].x, ml[p].y, y[p]);
        if (BY_LEAF) {
            fold(f, o, g.m, g.l, x);
            g.m = -INFINITY;
            g.l = 0.f;
#pragma unroll
            for (int e = 0; e < D / 64; ++e) x[e] = make_float2(0.f, 0.f);
        }
    }
    T* dst = (T*)a.out + row * D;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
        st(dst + 64 * e + 2 * lane, result(o[e].x, f.l));
        st(dst + 64 * e + 2 * lane + 1, result(o[e].y, f.l));
    }
}

// ---- CUDA cores --------------------------------------------------------------------------------
// A block of eight warps per (leaf, tile of eight rows, key head, sequence): page by page the scores (four lanes a position, a quarter of the channels each, the
// queries in shared memory), the rows' weights (a warp a row), the weighted values (a thread two channels, the positions shared out among D / 2
// threads' worth of groups).  Everything in 32 bits; a leaf leaves a record.  What bounds it: three barriers a page, and
// codes that are asked for when they are needed.  6 float32 sequences of up to 1,000 positions, 16 heads over 2 of 128: a block of four warps per
// node 49 us, this 13.
constexpr int PR = 8;                                            // rows of a tile
constexpr int Q_PAD = D / 4 + 4;                                 // a quarter of a query, so that quarters lie in different banks
constexpr int V_GROUPS = 256 / (D / 2);                          // groups of positions (192: two, and 64 threads without)

template <typename T>
__global__ void __launch_bounds__(256) plain_kernel(const Args a) {
    __shared__ __align__(16) float qs[PR][4][Q_PAD];
    __shared__ __align__(16) float ps[kPage][PR];                // scores, then weights
    __shared__ float so[V_GROUPS][PR][D];
    __shared__ float sm[PR], sl[PR], sa[PR];
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned at = blockIdx.x;
    const int leaf = (int)(at % (unsigned)a.nodes);
    at /= (unsigned)a.nodes;
    const int tile = (int)(at % (unsigned)a.tiles);
    at /= (unsigned)a.tiles;
    const int kvh = (int)(at % (unsigned)a.n_kv), b = (int)(at / (unsigned)a.n_kv);
    const Seq s = sequence(a, b);
    const int n_rows = s.new_tokens * a.group, row0 = tile * PR;
    const int lp = leaf_pages(a, s.pages), last = (min(row0 + PR, n_rows) - 1) / a.group;
    const int seen = (s.start + last) / kPage + 1, first_page = leaf * lp;
    pdl_wait();
    if (row0 >= n_rows || !fits(a, s) || first_page >= seen) return;
    for (int i = threadIdx.x; i < PR * D; i += 256) {
        const int row = row0 + i / D, tok = row / a.group, ch = i % D;
        qs[i / D][ch / (D / 4)][ch % (D / 4)] =
            row < n_rows ? ld((const T*)a.q + ((int64_t)(s.first + tok) * a.n_heads + kvh * a.group + (row - tok * a.group)) * D + ch) : 0.f;
    }
    if (threadIdx.x < PR) {
        sm[threadIdx.x] = -INFINITY;
        sl[threadIdx.x] = 0.f;
    }
    const float scale2 = a.flip ? -a.scale2 : a.scale2;
    const int pair = threadIdx.x % (D / 2), part = threadIdx.x / (D / 2);
    float o[PR][2];
#pragma unroll
    for (int u = 0; u < PR; ++u) o[u][0] = o[u][1] = 0.f;
    const int stop = min(seen, first_page + lp);
#pragma unroll 1
    for (int page = first_page; page < stop; ++page) {
        const int id = checked_page(a, a.page_table[(int64_t)b * a.table_width + page]), first = page * kPage;
        const uint8_t* head = a.kv + ((int64_t)id * a.n_kv + kvh) * TILE;
        const int rows = min(kPage, s.len - first);
        __syncthreads();                                         // (queries are there; the weights of the page before have been used)
        {
            const int t = warp * 8 + (lane >> 2), j = lane & 3;
            uint32_t w[NW], x = 0;
            load_words<NW>(head + t * (D / 2) + j * (D / 8), w);
            float sc[PR];
#pragma unroll
            for (int u = 0; u < PR; ++u) sc[u] = 0.f;
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                if (i % (D == 192 ? 2 : 4) == 0) x = *reinterpret_cast<const uint32_t*>(head + key_scales(D) + (t * (D / GROUP) + ((j * NW + i) >> 2)) * 4);
                uint32_t v[4];
                key_word(w[i], low_halves(x, x), high_halves(x, x), v);
                float k[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    k[e] = __uint_as_float(v[e] << 16);
                    k[e + 4] = __uint_as_float(v[e] & 0xFFFF0000u);
                }
#pragma unroll
                for (int u = 0; u < PR; ++u) {
                    const float4 x0 = *reinterpret_cast<const float4*>(&qs[u][j][8 * i]), x1 = *reinterpret_cast<const float4*>(&qs[u][j][8 * i + 4]);
                    sc[u] += x0.x * k[0] + x0.y * k[1] + x0.z * k[2] + x0.w * k[3] + x1.x * k[4] + x1.y * k[5] + x1.z * k[6] + x1.w * k[7];
                }
            }
#pragma unroll
            for (int u = 0; u < PR; ++u) {
                sc[u] += __shfl_xor_sync(0xffffffffu, sc[u], 1);
                sc[u] += __shfl_xor_sync(0xffffffffu, sc[u], 2);
            }
            if (j == 0) {
#pragma unroll
                for (int u = 0; u < PR; ++u)
                    ps[t][u] = first + t > s.start + min(row0 + u, n_rows - 1) / a.group ? -INFINITY : sc[u] * scale2;
            }
        }
        __syncthreads();
        {
            const int u = warp;                                  // (eight warps, eight rows)
            const float x = ps[lane][u], y = ps[lane + 32][u];
            const float m0 = sm[u], m = fmaxf(m0, warp_max(fmaxf(x, y))), ref = m == -INFINITY ? 0.f : m;
            const float e0 = exp2f(x - ref), e1 = exp2f(y - ref), sum = warp_sum(e0 + e1), was = m0 == -INFINITY ? 0.f : exp2f(m0 - m);
            ps[lane][u] = e0;
            ps[lane + 32][u] = e1;
            __syncwarp();
            if (lane == 0) {
                sm[u] = m;
                sl[u] = sl[u] * was + sum;
                sa[u] = was;
            }
        }
        __syncthreads();
        if (part < V_GROUPS) {
#pragma unroll
            for (int u = 0; u < PR; ++u) {
                o[u][0] *= sa[u];
                o[u][1] *= sa[u];
            }
            const bool all = first + kPage - 1 <= s.start;       // every row sees every position
            // A position's two values, and their part in the rows that see it (a value that is no number does not show in the others).
            auto add = [&](int t, bool check) {
                const uint32_t x = *reinterpret_cast<const uint32_t*>(head + value_scales(D) + (t * (D / GROUP) + pair / 16) * 4);
                const uint32_t byte = head[value_codes(D) + t * (D / 2) + value_byte<D>(t, pair)];
                uint32_t even, odd;
                value_pair<0>(byte, byte, low_halves(x, x), high_halves(x, x), even, odd);
                const float v0 = __uint_as_float(even << 16), v1 = __uint_as_float(odd << 16);
                const float4 p0 = *reinterpret_cast<const float4*>(&ps[t][0]), p1 = *reinterpret_cast<const float4*>(&ps[t][4]);
                const float p[PR] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
#pragma unroll
                for (int u = 0; u < PR; ++u) {
                    if (check && first + t > s.start + min(row0 + u, n_rows - 1) / a.group) continue;
                    o[u][0] += p[u] * v0;
                    o[u][1] += p[u] * v1;
                }
            };
            if (all) {
#pragma unroll 8
                for (int t = part; t < kPage; t += V_GROUPS) add(t, false);
            } else {
#pragma unroll 1
                for (int t = part; t < rows; t += V_GROUPS) add(t, true);
            }
        }
    }
    if (part < V_GROUPS) {
#pragma unroll
        for (int u = 0; u < PR; ++u) *reinterpret_cast<float2*>(&so[part][u][2 * pair]) = make_float2(o[u][0], o[u][1]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < PR * D; i += 256) {
        const int u = i / D, ch = i % D;
        const int64_t flat = flat_row(a, s, kvh, row0 + u);
        if (flat < 0) continue;
        float x = so[0][u][ch];
#pragma unroll
        for (int p = 1; p < V_GROUPS; ++p) x += so[p][u][ch];
        if (s.pages <= lp) {
            st((T*)a.out + flat * D + ch, result(x, sl[u]));
        } else {
            const int64_t rec = flat * a.nodes + leaf;
            a.rec[rec * D + ch] = x;
            if (ch == 0) *reinterpret_cast<float2*>(a.rec + a.rec_rows * a.nodes * D + rec * 2) = make_float2(sm[u], sl[u]);
        }
    }
}

static Plan plan(int n_tokens, int n_seqs, int n_heads, int n_kv, int max_q, int kv_bound, bool f32, int form) {
    Plan p = {};
    const int pages = (kv_bound + kPage - 1) / kPage;
    const int64_t rows = (int64_t)max_q * (n_heads / n_kv), sm = sm_count();
    p.form = f32 && form == AUTO ? PLAIN : form;
    p.nt = p.form == PLAIN || rows <= 8 ? 1 : (rows <= 16 || D > 128 ? 2 : 3);
    p.tiles = (int)((rows + 8 * p.nt - 1) / (8 * p.nt));
    // Prompts have enough row tiles without cuts, and would need records beyond measure (a row and node: 4 d bytes); two tiles a warp that stays, four blocks an SM.
    p.whole = rows > 8 && (int64_t)n_seqs * n_kv * p.tiles >= (p.form == PLAIN ? 4 : 2 * LEAVES) * sm;
    const int leaves = p.whole ? 1 : most_leaves(pages, n_kv);
    p.nodes = p.form == PLAIN ? leaves : (leaves + LEAVES - 1) / LEAVES;      // (places for records)
    const int64_t places = RECORD_BYTES / (4 * (int64_t)max(n_tokens, 1) * n_heads * (D + 2));
    if (rows > 8 && p.nodes > places) {
        p.whole = places <= 1;
        p.nodes = (int)max(places, (int64_t)1);
        p.most = p.whole ? 0 : p.nodes * (p.form == PLAIN ? 1 : LEAVES);
    }
    // Measured at 1 to 64 sequences of up to 300 to 131,000 positions, heads of 64 to 256, 2 to 16 key heads.  Blocks that stay want many nodes: a warp's first
    // one takes 15 us.  us a block per node / blocks that stay, heads of 128, up to eight rows: 512 nodes (one a sequence, 300 positions) 15 / 16, 512 (two a sequence,
    // 1,000) 20 / 24, 576 (18, 9,000) 21 / 25, 1,024 (one) 29 / 21, (two) 34 / 30, (eight) 30 / 30, 2,048 (eight) 53 / 39; 16 rows: 64 nodes 9 / 17, 768 43 / 33;
    // heads of 64, 42 rows: 512 24 / 23.
    // Clusters want to run all at once: 256 blocks 11.7 in records / 10.8, 512 19.3 / 20.4; heads of 256 (a block an SM) 64 11.7 / 10.8, 128 12.2 / 15.4.
    const int64_t nodes = (int64_t)n_seqs * n_kv * (p.whole ? 1 : min(p.nodes, nodes_of(pages, n_kv))) * p.tiles;
    const bool can_stay = n_seqs <= MAX_SEQS;
    if (p.form == AUTO)
        p.form = can_stay && nodes >= (p.nt > 1 ? 4 : 6) * sm ? STAY : (p.nodes <= CLUSTER && nodes <= (D <= 128 ? 2 * sm : sm / 2) ? CLUSTERS : RECORDS);
    p.possible = p.form >= PLAIN && p.form <= STAY && !(f32 && p.form != PLAIN) && !(p.form == STAY && !can_stay) && !(p.form == CLUSTERS && p.nodes > CLUSTER);
    p.stages = p.whole || p.most > 0 || leaf_pages(pages, n_kv) > 1 || p.nt == 3 ? MAX_STAGES : 1;
    p.blocks = p.form == STAY ? sm : (int64_t)n_seqs * n_kv * p.tiles * p.nodes;
    const bool records = p.nodes > 1 && p.form != CLUSTERS;
    p.scratch = records ? (int64_t)n_tokens * n_heads * p.nodes * (D + 2) : 0;
    p.kernels = records ? 2 : 1;
    return p;
}

// Dynamic shared memory beyond what a kernel has without asking (of the current device: each is asked once).
static int allow(void (*kernel)(Args), int bytes) {
    static void (*asked[64][16])(Args) = {};                      // (two host threads may both ask: it does no harm)
    int dev = 0;
    WICK_CUDA(cudaGetDevice(&dev));
    void (**mine)(Args) = dev >= 0 && dev < 64 ? asked[dev] : nullptr;
    for (int i = 0; mine && i < 16; ++i) {
        if (mine[i] == kernel) return 0;
        if (mine[i] == nullptr) {
            WICK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
            mine[i] = kernel;
            return 0;
        }
    }
    WICK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return 0;
}

template <typename T>
static int attention(const void* q, int n_tokens, const void* kv, int64_t kv_pages, void* out, const int* cu_seqlens, int n_seqs, const int* start,
                     const int* seq_of_token, const int* page_table, int table_width, int n_heads, int n_kv, int max_q, int kv_bound, float scale,
                     float* scratch, int64_t scratch_size, int form, int* status, void* stream) {
    WICK_REQUIRE(n_tokens >= 0 && n_seqs > 0 && n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && table_width > 0 && max_q >= 0 && kv_bound >= 0,
                 "attention_kv4: bad sizes");
    WICK_REQUIRE((((uintptr_t)q | (uintptr_t)kv | (uintptr_t)out | (uintptr_t)scratch) & 15) == 0, "attention_kv4: arrays must begin on multiples of 16 bytes");
    if (n_tokens == 0) return 0;
    // (a page outside the cache is read as page 0)
    WICK_REQUIRE(kv_pages > 0, "attention_kv4: %d tokens, and a cache without pages", n_tokens);
    WICK_REQUIRE(max_q > 0 && kv_bound > 0, "attention_kv4: %d tokens, but up to %d a sequence and %d positions", n_tokens, max_q, kv_bound);
    const Plan p = plan(n_tokens, n_seqs, n_heads, n_kv, max_q, kv_bound, sizeof(T) == 4, form);
    WICK_REQUIRE(p.possible, "attention_kv4: the kernel asked for (%d) does not take these sizes", form);
    WICK_REQUIRE(scratch_size >= p.scratch, "attention_kv4: scratch of %lld floats, %lld needed", (long long)scratch_size, (long long)p.scratch);
    WICK_REQUIRE(p.blocks < (1ll << 31), "attention_kv4: %lld blocks are beyond the grid's limit", (long long)p.blocks);
    Args a;
    a.q = q;
    a.out = out;
    a.kv = (const uint8_t*)kv;
    a.kv_pages = kv_pages;
    a.cu_seqlens = cu_seqlens;
    a.start = start;
    a.page_table = page_table;
    a.table_width = table_width;
    a.n_seqs = n_seqs;
    a.n_tokens = n_tokens;
    a.max_q = max_q;
    a.pages = (kv_bound + kPage - 1) / kPage;
    a.n_heads = n_heads;
    a.n_kv = n_kv;
    a.group = n_heads / n_kv;
    a.scale2 = fabsf(scale) * 1.44269504088896340736f;
    a.flip = scale < 0.f ? 0x80008000u : 0u;
    a.rec = scratch;
    a.rec_rows = (int64_t)n_tokens * n_heads;
    a.nodes = p.nodes;
    a.tiles = p.tiles;
    a.stages = p.stages;
    a.whole = p.whole;
    a.most = p.most;
    a.status = status;
    const cudaStream_t st = (cudaStream_t)stream;
    const dim3 grid((unsigned)p.blocks);
    if (p.form == PLAIN) {
        WICK_CUDA(launch(plain_kernel<T>, grid, dim3(256), 0, st, a));
    } else if (p.form == STAY) {
        void (*kernel)(Args) = p.nt == 1 ? stay_kernel<1> : (p.nt == 2 ? stay_kernel<2> : stay_kernel<D <= 128 ? 3 : 2>);
        const int warps = p.nt == 1 ? stay_warps<1>() : stay_warps<2>();
        if (int rc = allow(kernel, warps * TILE)) return rc;
        WICK_CUDA(launch(kernel, grid, dim3(warps * 32), warps * TILE, st, a));
    } else {
        const bool clusters = p.form == CLUSTERS && p.nodes > 1;
        void (*kernel)(Args) = p.nt == 1 ? (clusters ? leaves_kernel<1, true> : leaves_kernel<1, false>) : p.nt == 2 ? (clusters ? leaves_kernel<2, true> : leaves_kernel<2, false>) : (clusters ? leaves_kernel<D <= 128 ? 3 : 2, true> : leaves_kernel<D <= 128 ? 3 : 2, false>);
        if (int rc = allow(kernel, leaves_smem(p.nt, MAX_STAGES, true))) return rc;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = leaves_smem(p.nt, p.stages, clusters);
        cfg.stream = st;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = clusters ? p.nodes : 1;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        WICK_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
    }
    if (int rc = check_launch("attention_kv4")) return rc;
    if (p.kernels == 2) {
        WICK_CUDA(launch(p.form == PLAIN ? join_kernel<T, true> : join_kernel<T, false>, dim3((unsigned)(((int64_t)n_tokens * n_heads + 3) / 4)), dim3(128), 0, st, a, seq_of_token, n_tokens));
        return check_launch("attention_kv4 (join)");
    }
    return 0;
}

}  // namespace kv4
}  // namespace wick

using namespace wick;
typedef __nv_bfloat16 bf16;

// float32 words of scratch of a call of these sizes, and the kernels that it launches.  form: 0 as the sizes say, or one of Form where it is possible.
WICK_API long long wick_attn_kv4_scratch(int n_tokens, int n_seqs, int n_heads, int n_kv, int max_q, int kv_bound, int f32, int form, int* kernels) {
    if (n_seqs < 1 || n_heads < 1 || n_kv < 1 || n_heads % n_kv || max_q < 0 || kv_bound < 0) {
        fail("attention_kv4: bad sizes");
        return -1;
    }
    const kv4::Plan p = kv4::plan(n_tokens, n_seqs, n_heads, n_kv, max_q, kv_bound, f32 != 0, form);
    if (!p.possible) {
        fail("attention_kv4: the kernel asked for (%d) does not take these sizes", form);
        return -1;
    }
    *kernels = p.kernels;
    return (long long)p.scratch;
}

#define WICK_KV4_ATTENTION(NAME, T)                                                                                                                  \
    WICK_API int NAME(const void* q, int n_tokens, const void* kv, int64_t kv_pages, void* out, const int* cu_seqlens, int n_seqs, const int* start, \
                      const int* seq_of_token, const int* page_table, int table_width, int n_heads, int n_kv, int max_q, int kv_bound, float scale,  \
                      float* scratch, int64_t scratch_size, int form, int* status, void* stream) {                                                  \
        return kv4::attention<T>(q, n_tokens, kv, kv_pages, out, cu_seqlens, n_seqs, start, seq_of_token, page_table, table_width, n_heads, n_kv,    \
                                 max_q, kv_bound, scale, scratch, scratch_size, form, status, stream);                                              \
    }                                                                                                                                                \
    WICK_PACKED(NAME)
WICK_KV4_ATTENTION(wick_attn_kv4_bf16, bf16)
WICK_KV4_ATTENTION(wick_attn_kv4_f32, float)
