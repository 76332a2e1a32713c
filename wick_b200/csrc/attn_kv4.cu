// Causal attention over a cache that holds keys and values in 4 bits (kv4.cuh), for any number of new tokens a sequence.
//
//   out[i, h] = sum_t p_t v_t,  p = softmax over t <= position(i) of scale q[i, h] . k_t,  k_t and v_t the bfloat16 values that the codes stand for.
//
// How the work is cut.  The rows of a (sequence, key head) are its new tokens times the query heads of the key head; they come in tiles of eight or
// sixteen.  The sequence's pages are cut by its OWN length and the number of key heads alone: into leaves of as many pages (one, for up to 8 most_nodes
// pages) and nodes of eight leaves.  A leaf is computed by one warp, page by page, into a running maximum, sum and accumulator; a node's leaves
// are folded in order, a row's nodes likewise.  Which warp computes what changes no bit, so that a sequence's result does not depend on the batch it is
// in.  Three forms for bfloat16 (Plan has the rule):
//   * a block per node, a warp per leaf: the leaves meet in shared memory.  A sequence's nodes, where they are up to CLUSTER, are a cluster whose blocks
//     read each other's results and write the outcome; more leave records (accumulator, maximum, sum) that a second, small kernel joins.  Few nodes:
//     as many warps as there are leaves work on a sequence;
//   * blocks that stay, one per SM, with an equal run of all nodes (or leaves) of the step each, which their warps take one by one: a warp folds a node's
//     leaves in registers, and its next page is on its way while it computes one.  Many nodes of one row tile each (decode steps); records as above.
// A sequence with one node is written directly.
//
// The kernel on the tensor cores.  Keys and values stand on the 16-row side of mma.sync (16 positions, or 16 channels), the rows on the 8-column side, so
// that the eight rows of most head layouts fill it.  A page of one key head (80 d bytes) comes in one bulk copy.  Values are made from codes in registers, in
// the layout that the instruction wants: what a lane reads of a key are d / 4 neighbouring channels of a position (the queries are permuted to match),
// and of a value d / 8 neighbouring channels of four positions.  Rows 0, 1, ... 7 of the instruction's position side are
// the positions 0, 1, 3, 2, 4, 5, 7, 6 of eight, so that either reading touches every bank of the shared memory once.
//
// The float32 form (and the plain twin of the other): CUDA cores, the same leaves' values, everything in 32 bits.
#include "attn_kv4.cuh"
#include "packed.cuh"

namespace wick {
namespace kv4 {

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
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (MASK && first + mt * 16 + 8 * (e >> 1) + tr > w.limit[n][e & 1]) s[mt][n][e] = -INFINITY;
                top[e & 1] = fmaxf(top[e & 1], s[mt][n][e]);
            }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
            const float mine = top[c] == -INFINITY ? top[c] : top[c] * scale2, m = FRESH ? mine : fmaxf(sum.m[n][c], mine);
            const float was = FRESH ? 0.f : weight(sum.m[n][c], m);
            const float ref = m == -INFINITY ? 0.f : m;          // (nothing seen: weights 0; a score that is no number still shows)
            sum.m[n][c] = m;
            float l = 0.f;
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float& x = s[mt][n][c + 2 * h];
                    const float y = ex2(fmaf(x, scale2, -ref));
                    x = MASK && x == -INFINITY ? 0.f : y;        // (a scale of 0 and nothing else makes a difference)
                    l += x;
                }
            }
            sum.l[n][c] = FRESH ? l : sum.l[n][c] * was + l;
            if (!FRESH) {
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    sum.o[i][n][c] *= was;
                    sum.o[i][n][c + 2] *= was;
                }
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
template <int NT, typename Between = Nothing>
__device__ __forceinline__ void leaf_page(const Args& a, const uint8_t* tile, const Rows<NT>& w, const Seq& s, int page, bool fresh, Sum<NT>& sum,
                                          Between between = Nothing()) {
    const int first = page * kPage;
    if (first + kPage - 1 > s.start) {
        if (fresh) sum.clear();
        page_step<NT, true, false>(tile, w, a.scale2, first, s.len, s.new_tokens > 1, sum, between);
    } else if (fresh) {
        page_step<NT, false, true>(tile, w, a.scale2, first, s.len, false, sum, between);
    } else {
        page_step<NT, false, false>(tile, w, a.scale2, first, s.len, false, sum, between);
    }
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
    const int lp = leaf_pages(s.pages, a.n_kv), last = (min(row0 + 8 * NT, n_rows) - 1) / a.group;
    const int seen = (s.start + last) / kPage + 1;               // pages that any row of the tile sees
    const int first_page = node * LEAVES * lp;
    pdl_wait();
    if (row0 >= n_rows || !fits(a, s)) return;                   // (so do all blocks of its cluster)
    if (first_page >= seen) return;                              // (a cluster does not wait for blocks that have left)
    const int n_nodes = CLUSTERS ? (seen + LEAVES * lp - 1) / (LEAVES * lp) : nodes_of(s.pages, a.n_kv);
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
            if (!mbar_wait(&full[warp][k % a.stages], (k / a.stages) & 1, &abort_flag, a.status, 16)) {
                // (what is on its way has to arrive before this block's shared memory is somebody else's; again with a limit)
                for (int i = k; i < min(count, k + a.stages); ++i) {
                    int mine = 0;
                    mbar_wait(&full[warp][i % a.stages], (i / a.stages) & 1, &mine, a.status, 16);
                }
                break;
            }
            leaf_page<NT>(a, ring + (k % a.stages) * TILE, w, s, p0 + k, k == 0, sum);
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
// One row tile a sequence and key head (one new token, up to eight heads).  A block has an equal run of the step's nodes (BY_LEAF: of its leaves), and its
// warps take the next one whenever they are done with one.  A warp's tile is filled again while it is read: the next page's keys as soon as the scores are
// there, its values when the page is done.
struct Item {
    int b, kvh, place, nodes, lp;                                // place: the node's number in the sequence (BY_LEAF: the leaf's); none left: b < 0
    int page, end;                                               // of the sequence
};

template <bool BY_LEAF>
__global__ void __launch_bounds__(STAY_WARPS * 32, 1) stay_kernel(const Args a) {
    extern __shared__ __align__(128) uint8_t ring_all[];
    __shared__ uint64_t full[STAY_WARPS][2];                     // keys, values
    __shared__ int cum[MAX_SEQS + 1], lens[MAX_SEQS], firsts[MAX_SEQS];      // items before a sequence; its length (with a new token) and the token
    __shared__ int abort_flag, taken;
    constexpr int PER = BY_LEAF ? 1 : LEAVES;                    // leaves of an item
    pdl_trigger();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, j = lane & 3;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int w = 0; w < STAY_WARPS; ++w) {
            mbar_init(&full[w][0], 1);
            mbar_init(&full[w][1], 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        int before = 0;
#pragma unroll 1
        for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
            const int b = s0 + lane;
            int mine = 0;
            if (b < a.n_seqs) {
                const Seq s = sequence(a, b);
                if (s.new_tokens > 0 && fits(a, s)) {
                    const int lp = PER * leaf_pages(s.pages, a.n_kv);
                    mine = (s.pages + lp - 1) / lp * a.n_kv;
                }
                lens[b] = s.len;
                firsts[b] = s.first;
            }
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
    const int stop = (int)((int64_t)(blockIdx.x + 1) * cum[a.n_seqs] / gridDim.x);
    pdl_wait();
    uint8_t* tile = ring_all + (size_t)warp * TILE;

    auto take = [&](Item& n, int& ids) {
        int u = 0;
        if (lane == 0) u = atomicAdd(&taken, 1);
        u = __shfl_sync(0xffffffffu, u, 0);
        n.b = -1;
        if (u >= stop) return;
        int lo = 0, hi = a.n_seqs - 1;                           // the last sequence with cum[b] <= u
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cum[mid] <= u) lo = mid;
            else hi = mid - 1;
        }
        n.b = lo;
        const int pages = (lens[lo] + kPage - 1) / kPage, local = u - cum[lo];
        n.lp = leaf_pages(pages, a.n_kv);
        const int items = (pages + PER * n.lp - 1) / (PER * n.lp);
        n.nodes = (pages + LEAVES * n.lp - 1) / (LEAVES * n.lp);
        n.kvh = local / items;
        n.place = local - n.kvh * items;
        n.page = n.place * PER * n.lp;
        n.end = min(pages, n.page + PER * n.lp);
        ids = n.page + lane < n.end ? checked_page(a, a.page_table[(int64_t)lo * a.table_width + n.page + lane]) : 0;
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
    Seq s;
    s.new_tokens = 1;
    s.first = firsts[cn.b];
    Rows<1> w;
    fetch_rows<1>(a, s, cn.kvh, 0, w);
    bool ok = true;
#pragma unroll 1
    while (true) {
        s.len = lens[cn.b];
        s.start = s.len - 1;
        s.first = firsts[cn.b];
        order_rows<1>(a, w);
        w.limit[0][0] = w.limit[0][1] = s.start;
        take(nn, next_ids);
        Fold f[2];
        float o[MT][4];
        f[0].m = f[1].m = -INFINITY;
        f[0].l = f[1].l = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        int held = 0;                                            // of the 32 ids that the lanes have
#pragma unroll 1
        for (int page = cn.page; page < cn.end;) {
            Sum<1> sum;
            const int leaf_end = min(cn.end, page + cn.lp);
            bool fresh = true;
#pragma unroll 1
            for (; page < leaf_end; ++page) {
                int next_id = -1, next_kvh = cn.kvh;
                ok = ok && mbar_wait(&full[warp][0], parity, &abort_flag, a.status, 16);
                leaf_page<1>(a, tile, w, s, page, fresh, sum, [&]() {
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
                    if (next_id >= 0) start_half(next_id, next_kvh, 0);
                    if (page + 1 == cn.end && nn.b >= 0) {       // (the queries are not needed any more: the next item's are asked for)
                        Seq t;
                        t.new_tokens = 1;
                        t.first = firsts[nn.b];
                        fetch_rows<1>(a, t, nn.kvh, 0, w);
                    }
                    ok = mbar_wait(&full[warp][1], parity, &abort_flag, a.status, 16) && ok;
                });
                fresh = false;
                parity ^= 1;
                __syncwarp();
                if (next_id >= 0) start_half(next_id, next_kvh, 1);
                if (!ok) {                                       // (what is on its way has to arrive before this shared memory is somebody else's)
                    for (int h = 0; h < 2 && next_id >= 0; ++h) {
                        int mine = 0;
                        mbar_wait(&full[warp][h], parity, &mine, a.status, 16);
                    }
                    return;
                }
            }
            finish_leaf<1>(sum);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f[c].step(sum.m[0][c], sum.l[0][c]);
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    o[i][c] = f[c].of(o[i][c], sum.o[i][0][c]);
                    o[i][c + 2] = f[c].of(o[i][c + 2], sum.o[i][0][c + 2]);
                }
            }
        }
        const bool whole = cn.end - cn.page == (s.len + kPage - 1) / kPage;      // (the item is all of the sequence)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int64_t flat = 2 * j + c < a.group ? (int64_t)s.first * a.n_heads + cn.kvh * a.group + 2 * j + c : -1;
            if (flat < 0) continue;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if (whole) write_result(a, flat, r * (D / 8) + 2 * i, o[i][c], o[i][c + 2], f[c].l);
                else write_record(a, flat, cn.place, r * (D / 8) + 2 * i, o[i][c], o[i][c + 2]);
            }
            if (!whole && r == 0) write_weights(a, flat, cn.place, f[c].m, f[c].l);
        }
        if (nn.b < 0) return;
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
    const int seen = (s.start + tok - s.first) / kPage + 1, per = (BY_LEAF ? 1 : LEAVES) * leaf_pages(s.pages, a.n_kv), n = (seen + per - 1) / per;
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
// threads' worth of groups).  Everything in 32 bits; a leaf leaves a record.  6 sequences of up to 1,000 positions, 16 heads over 2 of 128: the four warps a
// node that this took the place of 46 us, now 16.
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
    const int lp = leaf_pages(s.pages, a.n_kv), last = (min(row0 + PR, n_rows) - 1) / a.group;
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
    const int64_t rows = (int64_t)max_q * (n_heads / n_kv);
    p.nodes = nodes_of(pages, n_kv);
    p.form = f32 && form == AUTO ? PLAIN : form;
    const bool can_stay = rows <= 8 && n_seqs <= MAX_SEQS, can_tc = D == 128 && n_seqs <= MAX_SEQS;
    p.possible = p.form >= AUTO && p.form <= TC_CLUSTERS && !(f32 && p.form != PLAIN) && !((p.form == STAY || p.form == STAY_LEAVES) && !can_stay) &&
                 !(p.form >= TC && !can_tc) && !((p.form == CLUSTERS || p.form == TC_CLUSTERS) && p.nodes > CLUSTER);
    const int64_t nodes = (int64_t)n_seqs * n_kv * p.nodes;
    if (p.form == AUTO && can_tc && rows > 8)
        p.form = p.nodes <= CLUSTER && nodes <= 2 * sm_count() ? TC_CLUSTERS : TC;
    else if (p.form == AUTO)
        p.form = can_stay && nodes >= 2 * (int64_t)LEAVES * sm_count() ? STAY : (p.nodes <= CLUSTER && nodes <= 2 * sm_count() ? CLUSTERS : RECORDS);
    const bool tc = p.form >= TC;
    p.nt = p.form == PLAIN || rows <= 8 ? 1 : (rows <= 16 || D > 128 ? 2 : 3);
    p.rows = p.form == PLAIN ? 8 : (tc ? (rows <= 8 ? 8 : (rows <= 16 ? 16 : (rows <= 24 ? 24 : 32))) : 8 * p.nt);
    p.tiles = (int)((rows + p.rows - 1) / p.rows);
    p.stages = leaf_pages(pages, n_kv) > 1 || p.nt == 3 ? MAX_STAGES : 1;
    if (p.form == STAY_LEAVES || p.form == PLAIN) p.nodes = (pages + leaf_pages(pages, n_kv) - 1) / leaf_pages(pages, n_kv);      // (places for records)
    p.blocks = p.form == STAY || p.form == STAY_LEAVES || p.form == TC ? sm_count() : (int64_t)n_seqs * n_kv * p.tiles * p.nodes;
    const bool records = p.nodes > 1 && p.form != CLUSTERS && p.form != TC_CLUSTERS;
    p.scratch = records ? (int64_t)n_tokens * n_heads * p.nodes * (D + 2) : 0;
    p.kernels = records ? 2 : 1;
    return p;
}

// Dynamic shared memory beyond what a kernel has without asking.
static int allow(void (*kernel)(Args), int bytes) {
    static void (*asked[8])(Args) = {};                          // (two host threads may both ask: it does no harm)
    for (int i = 0; i < 8; ++i) {
        if (asked[i] == kernel) return 0;
        if (asked[i] == nullptr) {
            WICK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
            asked[i] = kernel;
            return 0;
        }
    }
    return 0;
}

template <typename T>
static int attention(const void* q, int n_tokens, const void* kv, int64_t kv_pages, void* out, const int* cu_seqlens, int n_seqs, const int* start,
                     const int* seq_of_token, const int* page_table, int table_width, int n_heads, int n_kv, int max_q, int kv_bound, float scale,
                     float* scratch, int64_t scratch_size, int form, int* status, void* stream) {
    WICK_REQUIRE(n_tokens >= 0 && n_seqs > 0 && n_heads > 0 && n_kv > 0 && n_heads % n_kv == 0 && table_width > 0 && max_q >= 0 && kv_bound >= 0,
                 "attention_kv4: bad sizes");
    WICK_REQUIRE((((uintptr_t)q | (uintptr_t)kv | (uintptr_t)out | (uintptr_t)scratch) & 15) == 0, "attention_kv4: arrays must begin on multiples of 16 bytes");
    if (n_tokens == 0 || max_q == 0 || kv_bound == 0) return 0;
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
    a.status = status;
    const cudaStream_t st = (cudaStream_t)stream;
    const dim3 grid((unsigned)p.blocks);
    if (p.form == PLAIN) {
        WICK_CUDA(launch(plain_kernel<T>, grid, dim3(256), 0, st, a));
    } else if (p.form >= TC) {
        if (int rc = launch_tc(a, p.rows, p.form == TC_CLUSTERS, p.blocks, st)) return rc;
    } else if (p.form >= STAY) {
        void (*kernel)(Args) = p.form == STAY ? stay_kernel<false> : stay_kernel<true>;
        if (int rc = allow(kernel, STAY_WARPS * TILE)) return rc;
        WICK_CUDA(launch(kernel, grid, dim3(STAY_WARPS * 32), STAY_WARPS * TILE, st, a));
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
        WICK_CUDA(launch(p.form == STAY_LEAVES || p.form == PLAIN ? join_kernel<T, true> : join_kernel<T, false>, dim3((unsigned)(((int64_t)n_tokens * n_heads + 3) / 4)), dim3(128), 0, st, a, seq_of_token, n_tokens));
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
