// Attention over a prefix that groups of sequences share, and over each sequence's own keys behind it (attn_shared.cuh has the
// mathematics and how the shared part is cut).
//
//   1. the shared keys: attn_shared_prefix_kernel here (any head size, bfloat16 and float32, tiles of 16 rows), or the tcgen05 kernel
//      of attn_shared_tc.cu (bfloat16, head sizes 64 and 128, tiles of 128 rows); a record (m, l, o) per run of units;
//   2. attn_shared_own_kernel: a block per sequence, key head and 16 rows (and part of the own keys, where they are many): the
//      own keys, then all parts joined and written.  It starts while the first kernel's last blocks run and waits for them only
//      before it joins;
//   3. where a sequence's own keys are cut into parts: attn_shared_join_kernel.
//
// bfloat16: mma.sync on tiles of 16 rows and 16 keys.  Keys and values go from the cache straight to registers: the inner index of
// q . k is summed over in any order, so a lane takes 16 neighbouring bytes of a key row and the same of its query row as operands of
// two instructions; and a value row's numbers may stand in any order of columns, so a lane takes 16 neighbouring bytes of each of four
// keys' rows and pairs them by byte permutation.  No shared memory, no barrier until the warps' parts are joined.  Weights enter the second
// product rounded to bfloat16, and their sum is taken of the rounded ones, so that a row of equal values keeps them.
// float32: products and sums on the CUDA cores, keys and values through shared memory, 32 keys at a time.
#include "common.cuh"
#include "attn_shared.cuh"

#ifndef WICK_HD
#error "compile with -DWICK_HD=<head_dim>"
#endif

namespace wick {
namespace shared_prefix {

constexpr int HD = WICK_HD;
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head_dim must be a multiple of 16 in [16, 256]");
typedef __nv_bfloat16 bf16;

constexpr int R = 16;                              // rows of a tile
constexpr int W = 4, THREADS = W * 32;
constexpr int REC = R * (HD + 2);                  // floats of a tile's record: [HD / 4][R][4] sums, [R][2] maximum and sum of weights
constexpr int SPLIT = 512;                         // own keys from which on a sequence is cut
constexpr int MAX_SPLITS = 16;
constexpr float LOG2E = 1.4426950408889634f;

__host__ __device__ inline int own_splits(int n) { return n <= SPLIT ? 1 : min(MAX_SPLITS, (n + SPLIT - 1) / SPLIT); }
__host__ __device__ inline int split_keys(int n, int splits) { return ((n + 63) / 64 + splits - 1) / splits * 64; }

// 2^(a - b) for maxima that may be -inf (nothing seen): then the weight is 0.
__device__ __forceinline__ float weight(float a, float b) { return a == -INFINITY ? 0.f : exp2f(a - b); }

// A block's 16 rows, as the cores leave them: in PARTS parts.
template <typename T> struct Work;
template <> struct Work<bf16> {
    static constexpr int PARTS = W;
    float o[W][R][HD];
    float m[W][R], l[W][R];
};
template <> struct Work<float> {
    static constexpr int PARTS = 1;
    static constexpr int KT = 32;                  // keys of a tile
    float o[1][R][HD];
    float q[R][HD];
    float k[2][KT][HD + 4], v[2][KT][HD];
    float p[KT][R];
    float m[1][R], l[1][R], alpha[R];
};

// Which rows a block has: their queries (null: none) and the last key that each sees.
template <typename T> struct Rows {
    const T* q[R];
    int last[R];
};

// ---- bfloat16 ----------------------------------------------------------------
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// N neighbouring 32-bit words (8 N bytes of bfloat16 pairs), as wide as their number allows.
template <int N> __device__ __forceinline__ void load_words(uint32_t* d, const bf16* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 t = *reinterpret_cast<const uint4*>(p + 2 * i);
            d[i] = t.x, d[i + 1] = t.y, d[i + 2] = t.z, d[i + 3] = t.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 t = *reinterpret_cast<const uint2*>(p + 2 * i);
            d[i] = t.x, d[i + 1] = t.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = *reinterpret_cast<const uint32_t*>(p + 2 * i);
    }
}
// A row as the operand of q . k, lane part t = 0 .. 3 of it: chunks of 32 numbers, 8 a part; a last chunk of 16, 4 a part.
// Word 2 s + i is register i of instruction s.
constexpr int KW = HD / 8;
__device__ __forceinline__ void load_row(uint32_t* d, const bf16* row, int t) {
#pragma unroll
    for (int c = 0; c < HD / 32; ++c) load_words<4>(d + 4 * c, row + 32 * c + 8 * t);
    if constexpr (HD % 32 != 0) load_words<2>(d + HD / 32 * 4, row + HD / 32 * 32 + 4 * t);
}
// A value row, lane part n = 0 .. 7 of it: sets of 64 numbers, 8 a part; a last set of 16, 32 or 48.
constexpr int VW = HD / 16, LAST = HD % 64 / 16;   // words of a row a lane holds; those of the last set
__device__ __forceinline__ void load_values(uint32_t* d, const bf16* row, int n) {
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) load_words<4>(d + 4 * c, row + 64 * c + 8 * n);
    if constexpr (LAST > 0) load_words<LAST>(d + HD / 64 * 4, row + HD / 64 * 64 + 2 * LAST * n);
}
// The column that number j (of the HD / 8 a lane's part n has) is.
__device__ __forceinline__ int value_column(int j, int n) { return j < HD / 64 * 8 ? j / 8 * 64 + 8 * n + j % 8 : HD / 64 * 64 + 2 * LAST * n + j - HD / 64 * 8; }

// The rows' attention over the keys [key0, key1) of the sequence whose page ids are tab (key0 a multiple of 16), into w.
// Warps take every fourth step of 16 keys.
__device__ void attend(Work<bf16>& w, const Rows<bf16>& rows, const bf16* __restrict__ kv, int64_t kv_pages, const int* __restrict__ tab, int kvh,
                       int n_kv, int key0, int key1, float scale, int* status) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const float sl2 = scale * LOG2E;
    uint32_t qa[KW * 2];                           // instruction s: words 4 s .. 4 s + 3
    {
        uint32_t a[KW], b[KW];
#pragma unroll
        for (int i = 0; i < KW; ++i) a[i] = b[i] = 0;
        if (rows.q[g]) load_row(a, rows.q[g], t);
        if (rows.q[g + 8]) load_row(b, rows.q[g + 8], t);
#pragma unroll
        for (int s = 0; s < KW / 2; ++s) qa[4 * s] = a[2 * s], qa[4 * s + 1] = b[2 * s], qa[4 * s + 2] = a[2 * s + 1], qa[4 * s + 3] = b[2 * s + 1];
    }
    const int last0 = rows.last[g], last1 = rows.last[g + 8];
    float o[HD / 8][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    const int64_t page_elems = (int64_t)2 * n_kv * kPage * HD;
    const int steps = (key1 - key0 + 15) / 16;
    // the tile of keys of a step (values n_kv tiles of a page further), from its page's id
    auto page_of = [&](int s) { return s < steps ? tab[(key0 + 16 * s) / kPage] : 0; };
    auto tile_of = [&](int s, int page) -> const bf16* {
        if (page < 0 || page >= kv_pages) {
            if (lane == 0) atomicCAS(status, 0, 10);
            page = 0;
        }
        return kv + page * page_elems + ((int64_t)kvh * kPage + (key0 + 16 * s) % kPage) * HD;
    };
    uint32_t kb[2][KW], vb[4][VW];
    auto load_keys = [&](const bf16* tile) {
        load_row(kb[0], tile + (int64_t)g * HD, t);
        load_row(kb[1], tile + (int64_t)(g + 8) * HD, t);
    };
    auto load_vals = [&](const bf16* tile) {
        const bf16* v = tile + (int64_t)n_kv * kPage * HD;
        load_values(vb[0], v + (2 * t) * HD, g);
        load_values(vb[1], v + (2 * t + 1) * HD, g);
        load_values(vb[2], v + (2 * t + 8) * HD, g);
        load_values(vb[3], v + (2 * t + 9) * HD, g);
    };
    int s = warp;
    const bf16* tile = nullptr;
    int page_next = 0;
    if (s < steps) {
        tile = tile_of(s, page_of(s));
        load_keys(tile);
        load_vals(tile);
        page_next = page_of(s + W);
    }
#pragma unroll 1
    for (; s < steps; s += W) {
        const int key = key0 + 16 * s;
        float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int i = 0; i < KW / 2; ++i) {
            mma16816(c[0], qa + 4 * i, kb[0][2 * i], kb[0][2 * i + 1]);
            mma16816(c[1], qa + 4 * i, kb[1][2 * i], kb[1][2 * i + 1]);
        }
        const bf16* next = nullptr;
        if (s + W < steps) {
            next = tile_of(s + W, page_next);
            load_keys(next);
            page_next = page_of(s + 2 * W);
        }
        if (key + 16 > key1) {                     // places behind the last key hold anything: no weight, and zeros for values
#pragma unroll
            for (int i = 0; i < VW; ++i) {
                if (key + 2 * t >= key1) vb[0][i] = 0;
                if (key + 2 * t + 1 >= key1) vb[1][i] = 0;
                if (key + 2 * t + 8 >= key1) vb[2][i] = 0;
                if (key + 2 * t + 9 >= key1) vb[3][i] = 0;
            }
        }
        const int lim0 = min(last0, key1 - 1) - key - 2 * t, lim1 = min(last1, key1 - 1) - key - 2 * t;   // places up to them are seen
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                c[h][i] = 8 * h + i <= lim0 ? c[h][i] * sl2 : -INFINITY;
                c[h][2 + i] = 8 * h + i <= lim1 ? c[h][2 + i] * sl2 : -INFINITY;
            }
        float x0 = fmaxf(fmaxf(c[0][0], c[0][1]), fmaxf(c[1][0], c[1][1])), x1 = fmaxf(fmaxf(c[0][2], c[0][3]), fmaxf(c[1][2], c[1][3]));
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
        }
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float a0 = weight(m0, n0), a1 = weight(m1, n1);
        const float z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
        m0 = n0, m1 = n1;
        uint32_t pa[4];
        l0 *= a0, l1 *= a1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(exp2f(c[h][0] - z0), exp2f(c[h][1] - z0));
            const __nv_bfloat162 r = __floats2bfloat162_rn(exp2f(c[h][2] - z1), exp2f(c[h][3] - z1));
            const float2 pf = __bfloat1622float2(p), rf = __bfloat1622float2(r);
            l0 += pf.x + pf.y, l1 += rf.x + rf.y;
            pa[2 * h] = *reinterpret_cast<const uint32_t*>(&p);
            pa[2 * h + 1] = *reinterpret_cast<const uint32_t*>(&r);
        }
#pragma unroll
        for (int j = 0; j < HD / 8; ++j) {
            o[j][0] *= a0, o[j][1] *= a0, o[j][2] *= a1, o[j][3] *= a1;
            const int i = j / 2;
            const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
            mma16816(o[j], pa, __byte_perm(vb[0][i], vb[1][i], sel), __byte_perm(vb[2][i], vb[3][i], sel));
        }
        if (next) load_vals(next);
    }
#pragma unroll
    for (int d = 1; d <= 2; d <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, d);
        l1 += __shfl_xor_sync(0xffffffffu, l1, d);
    }
    if (t == 0) w.m[warp][g] = m0, w.l[warp][g] = l0, w.m[warp][g + 8] = m1, w.l[warp][g + 8] = l1;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
        const int c0 = value_column(j, 2 * t), c1 = value_column(j, 2 * t + 1);
        w.o[warp][g][c0] = o[j][0], w.o[warp][g][c1] = o[j][1];
        w.o[warp][g + 8][c0] = o[j][2], w.o[warp][g + 8][c1] = o[j][3];
    }
    __syncthreads();
}

// ---- float32 -----------------------------------------------------------------
__device__ __forceinline__ void copy16(void* dst, const void* src, bool there) {
    const int n = there ? 16 : 0;                  // (0: zeros)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(n) : "memory");
}

// A warp has the scores of four rows with a tile's 32 keys, a thread the sums of four rows and four columns.
__device__ void attend(Work<float>& w, const Rows<float>& rows, const float* __restrict__ kv, int64_t kv_pages, const int* __restrict__ tab, int kvh,
                       int n_kv, int key0, int key1, float scale, int* status) {
    constexpr int KT = Work<float>::KT, ITEMS = (HD + THREADS - 1) / THREADS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float sl2 = scale * LOG2E;
    for (int i = tid; i < R * HD / 4; i += THREADS) {
        const float* q = rows.q[i / (HD / 4)];
        *reinterpret_cast<float4*>(&w.q[i / (HD / 4)][i % (HD / 4) * 4]) =
            q ? *reinterpret_cast<const float4*>(q + i % (HD / 4) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    const int64_t page_elems = (int64_t)2 * n_kv * kPage * HD;
    const int tiles = (key1 - key0 + KT - 1) / KT;
    auto fetch = [&](int i) {
        const int key = key0 + i * KT;
        int page = tab[key / kPage];
        if (page < 0 || page >= kv_pages) {
            if (tid == 0) atomicCAS(status, 0, 10);
            page = 0;
        }
        const float* k = kv + page * page_elems + ((int64_t)kvh * kPage + key % kPage) * HD;
        const float* v = k + (int64_t)n_kv * kPage * HD;
        for (int c = tid; c < KT * HD / 4; c += THREADS) {
            const int row = c / (HD / 4), col = c % (HD / 4) * 4;
            const bool there = key + row < key1;
            copy16(&w.k[i & 1][row][col], k + row * HD + col, there);
            copy16(&w.v[i & 1][row][col], v + row * HD + col, there);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    float m[4], l[4], acc[ITEMS][4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int it = 0; it < ITEMS; ++it)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[it][i][0] = acc[it][i][1] = acc[it][i][2] = acc[it][i][3] = 0.f;
    if (tiles > 0) fetch(0);
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
        if (i + 1 < tiles) {
            fetch(i + 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int d = 0; d < HD; d += 4) {
            const float4 k4 = *reinterpret_cast<const float4*>(&w.k[i & 1][lane][d]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 q4 = *reinterpret_cast<const float4*>(&w.q[warp * 4 + r][d]);
                s[r] = fmaf(q4.x, k4.x, s[r]), s[r] = fmaf(q4.y, k4.y, s[r]);
                s[r] = fmaf(q4.z, k4.z, s[r]), s[r] = fmaf(q4.w, k4.w, s[r]);
            }
        }
        const int key = key0 + i * KT + lane;
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float x = key < key1 && key <= rows.last[warp * 4 + r] ? s[r] * sl2 : -INFINITY;
            const float n = fmaxf(m[r], warp_max(x)), a = weight(m[r], n);
            p[r] = weight(x, n);
            l[r] = l[r] * a + warp_sum(p[r]);
            m[r] = n;
            if (lane == 0) w.alpha[warp * 4 + r] = a;
        }
        *reinterpret_cast<float4*>(&w.p[lane][warp * 4]) = make_float4(p[0], p[1], p[2], p[3]);
        __syncthreads();
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int idx = tid + it * THREADS, rg = idx / (HD / 4), c = idx % (HD / 4) * 4;
            if (idx < HD) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float a = w.alpha[rg * 4 + r];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[it][r][e] *= a;
                }
#pragma unroll 4
                for (int key = 0; key < KT; ++key) {
                    const float4 v4 = *reinterpret_cast<const float4*>(&w.v[i & 1][key][c]), p4 = *reinterpret_cast<const float4*>(&w.p[key][rg * 4]);
                    const float pr[4] = {p4.x, p4.y, p4.z, p4.w};
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        acc[it][r][0] = fmaf(pr[r], v4.x, acc[it][r][0]), acc[it][r][1] = fmaf(pr[r], v4.y, acc[it][r][1]);
                        acc[it][r][2] = fmaf(pr[r], v4.z, acc[it][r][2]), acc[it][r][3] = fmaf(pr[r], v4.w, acc[it][r][3]);
                    }
                }
            }
        }
        __syncthreads();
    }
    if (lane == 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r) w.m[0][warp * 4 + r] = m[r], w.l[0][warp * 4 + r] = l[r];
    }
#pragma unroll
    for (int it = 0; it < ITEMS; ++it) {
        const int idx = tid + it * THREADS, rg = idx / (HD / 4), c = idx % (HD / 4) * 4;
        if (idx < HD) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<float4*>(&w.o[0][rg * 4 + r][c]) = make_float4(acc[it][r][0], acc[it][r][1], acc[it][r][2], acc[it][r][3]);
        }
    }
    __syncthreads();
}

// The block's parts of row r joined: the maximum, the sum of weights, and four columns' sums.
template <typename T> __device__ __forceinline__ float max_of(const Work<T>& w, int r) {
    float m = w.m[0][r];
#pragma unroll
    for (int i = 1; i < Work<T>::PARTS; ++i) m = fmaxf(m, w.m[i][r]);
    return m;
}
template <typename T> __device__ __forceinline__ float sum_of(const Work<T>& w, int r, float m) {
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < Work<T>::PARTS; ++i) l = fmaf(w.l[i][r], weight(w.m[i][r], m), l);
    return l;
}
template <typename T> __device__ __forceinline__ float4 columns_of(const Work<T>& w, int r, int c, float m) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < Work<T>::PARTS; ++i) {
        const float a = weight(w.m[i][r], m);
        const float4 o = *reinterpret_cast<const float4*>(&w.o[i][r][c]);
        s.x = fmaf(o.x, a, s.x), s.y = fmaf(o.y, a, s.y), s.z = fmaf(o.z, a, s.z), s.w = fmaf(o.w, a, s.w);
    }
    return s;
}
template <typename T> __device__ __forceinline__ void write_record(const Work<T>& w, float* rec) {
    for (int i = threadIdx.x; i < R * HD / 4; i += THREADS) {
        const int r = i % R, c = i / R;
        *reinterpret_cast<float4*>(rec + i * 4) = columns_of(w, r, c * 4, max_of(w, r));
    }
    if (threadIdx.x < R) {
        const float m = max_of(w, threadIdx.x);
        *reinterpret_cast<float2*>(rec + R * HD + 2 * threadIdx.x) = make_float2(m, sum_of(w, threadIdx.x, m));
    }
}

// ---- 1. the shared keys --------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(THREADS)
attn_shared_prefix_kernel(const T* q, const T* __restrict__ kv, int64_t kv_pages, const Groups G, float scale, int* plan, float* records, int* status) {
    extern __shared__ __align__(16) uint8_t smem[];
    Work<T>& w = *reinterpret_cast<Work<T>*>(smem);
    __shared__ Rows<T> rows;
    pdl_wait();
    pdl_trigger();                                  // (behind the wait: the next kernel reads what this one reads without a wait of its own)
    q = fresh(q);
    Walk walk(G, gridDim.x, blockIdx.x == 0 && threadIdx.x < 32 ? plan : nullptr);
    Segment s;
    while (walk.segment(s)) {                       // (every warp walks the same way)
        __syncthreads();                            // (the rows and the work of the segment before)
        if (threadIdx.x < R) {
            const int idx = s.tile * R + threadIdx.x;
            const bool there = idx < s.n_tok * G.gs;
            rows.q[threadIdx.x] = there ? q + ((int64_t)(s.tok0 + idx / G.gs) * G.heads + s.column * G.gs + idx % G.gs) * HD : nullptr;
            rows.last[threadIdx.x] = there ? s.pages * kPage - 1 : -1;
        }
        __syncthreads();
        attend(w, rows, kv, kv_pages, G.page_table + (int64_t)G.cu_groups[s.g] * G.table_width, s.column / G.per_kv, G.kv_heads,
               s.from * kPage, s.to * kPage, scale, status);
        write_record(w, records + (int64_t)s.record * REC);
    }
}

// ---- 2. the own keys, and all parts joined -----------------------------------------
// What the records of the shared part look like.
struct Shared {
    const int* plan;                               // null: nothing is shared
    const float* records;
    int rows;                                      // that a record has room for
};

// Row `row` of the tile (token tok, head) joined with the shared part's records: the factors of the own part (M -> its weight) and
// of each record are left in f[0] and f[1 ..].  Called by the 8 lanes that share a row; n_seg records from `rec` on, at place r.
struct Joined {
    int first, n, r;                               // records, the row's place in them
};
__device__ __forceinline__ Joined records_of(const Groups& G, const Shared& sh, int g, int tok, int head, int kvh) {
    Joined j = {0, 0, 0};
    if (!sh.plan) return j;
    const Cut c = cut_of(G, g);
    if (c.pages == 0) return j;
    const int *units = sh.plan + 1, *items = sh.plan + 2 + G.n;
    const int S = __ldcg(sh.plan), U = __ldcg(units + G.n);
    const int h = head - kvh * (G.heads / G.kv_heads), column = kvh * G.per_kv + h / G.gs;
    const int idx = (tok - c.tok0) * G.gs + h % G.gs, tile = idx / G.rows, pair = tile / G.pair, w = c.width(G, pair);
    const int u = __ldcg(units + g) + c.before(G, pair, column);
    const int c0 = block_of(u + w - 1, U, S), c1 = block_of(u + w * c.blocks - 1, U, S);
    j.first = (__ldcg(items + g) + pair * G.columns + column + c0) * G.pair + tile - pair * G.pair;
    j.n = c1 - c0 + 1;
    j.r = idx - tile * G.rows;
    return j;
}

// The 16 rows of a tile written: own(r, m, l) gives the own part's maximum and sum, cols(r, c, m) its columns.
template <typename T, typename Own, typename Cols>
__device__ __forceinline__ void finish(const Groups& G, const Shared& sh, T* __restrict__ out, int g, int tok0, int row0, int n_rows, int kvh, Own own,
                                       Cols cols) {
    __shared__ Joined parts[R];
    __shared__ float most[R], over[R];
    const int tid = threadIdx.x, group = G.heads / G.kv_heads, rec_floats = sh.rows * (HD + 2), step = rec_floats * G.pair;   // (of an item's records)
    auto tok_of = [&](int r) { return tok0 + (row0 + r) / group; };
    auto head_of = [&](int r) { return kvh * group + (row0 + r) % group; };
    {
        const int r = tid / 8, k = tid % 8;        // 8 lanes a row
        Joined j = {0, 0, 0};
        float m = -INFINITY, l = 0.f;
        if (r < n_rows) {
            own(r, m, l);
            j = records_of(G, sh, g, tok_of(r), head_of(r), kvh);
        }
        const float m_own = m, l_own = l;
        for (int i = k; i < j.n; i += 8) m = fmaxf(m, __ldcg(sh.records + (int64_t)j.first * rec_floats + (int64_t)i * step + sh.rows * HD + 2 * j.r));
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        l = k == 0 ? l_own * weight(m_own, m) : 0.f;
        for (int i = k; i < j.n; i += 8) {
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(sh.records + (int64_t)j.first * rec_floats + (int64_t)i * step + sh.rows * HD + 2 * j.r));
            l = fmaf(ml.y, weight(ml.x, m), l);
        }
#pragma unroll
        for (int d = 1; d < 8; d <<= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
        if (k == 0) parts[r] = j, most[r] = m, over[r] = l != 0.f ? __fdiv_rn(1.0f, l) : 0.f;     // (a sum that is no number shows)
    }
    __syncthreads();
    for (int i = tid; i < n_rows * (HD / 4); i += THREADS) {
        const int r = i % n_rows, c = i / n_rows;
        const Joined j = parts[r];
        const float m = most[r];
        float4 s = cols(r, c * 4, m);
        const float* rec = sh.records + (int64_t)j.first * rec_floats;
#pragma unroll 4
        for (int k = 0; k < j.n; ++k, rec += step) {
            const float4 o = __ldcg(reinterpret_cast<const float4*>(rec + ((int64_t)c * sh.rows + j.r) * 4));
            const float a = weight(__ldcg(rec + sh.rows * HD + 2 * j.r), m);
            s.x = fmaf(o.x, a, s.x), s.y = fmaf(o.y, a, s.y), s.z = fmaf(o.z, a, s.z), s.w = fmaf(o.w, a, s.w);
        }
        const float f = over[r];
        st4(out + ((int64_t)tok_of(r) * G.heads + head_of(r)) * HD + c * 4, s.x * f, s.y * f, s.z * f, s.w * f);
    }
}

// The own keys of sequence b: their first position and the end, or -1 (with a report) where the description cannot be.
__device__ __forceinline__ int2 own_keys(const Groups& G, int b, int q_len, int* status) {
    const int g = G.group_of[b];
    const int begin = g >= 0 && g < G.n ? pages_of(G, g) * kPage : 0, end = G.start[b] + q_len;
    if (g < 0 || g >= G.n || G.start[b] < begin || (end + kPage - 1) / kPage > G.table_width) {
        if (threadIdx.x == 0) atomicCAS(status, 0, 11);
        return make_int2(-1, -1);
    }
    return make_int2(begin, end);
}

// Blocks (key head and tile of rows, sequence, part of the own keys).
template <typename T>
__global__ void __launch_bounds__(THREADS)
attn_shared_own_kernel(const T* q, const T* __restrict__ kv, int64_t kv_pages, T* __restrict__ out, const Groups G, const Shared sh, float scale,
                       float* own_records, int* status) {
    extern __shared__ __align__(16) uint8_t smem[];
    Work<T>& w = *reinterpret_cast<Work<T>*>(smem);
    __shared__ Rows<T> rows;
    // (With a shared part the kernel before this one is the one that computes it, and has waited for q and the cache.)
    if (!sh.plan) pdl_wait();
    pdl_trigger();
    q = fresh(q);
    const int b = blockIdx.y, kvh = blockIdx.x % G.kv_heads, row0 = blockIdx.x / G.kv_heads * R;
    const int tok0 = G.cu_seqlens[b], q_len = G.cu_seqlens[b + 1] - tok0, group = G.heads / G.kv_heads;
    const int n_rows = min(R, q_len * group - row0);
    if (n_rows <= 0) {
        pdl_wait();                                 // (whoever waits for this kernel waits for the one before it too)
        return;
    }
    const int2 keys = own_keys(G, b, q_len, status);
    const int n = keys.y - keys.x, splits = min(own_splits(n), (int)gridDim.z), per = split_keys(n, splits);
    const int key0 = keys.x + (int)blockIdx.z * per, key1 = min(keys.y, key0 + per);
    if ((int)blockIdx.z >= splits || keys.x < 0) {
        pdl_wait();
        if (keys.x < 0 && blockIdx.z == 0)
            for (int i = threadIdx.x; i < n_rows * HD; i += THREADS)
                st(out + ((int64_t)(tok0 + (row0 + i / HD) / group) * G.heads + kvh * group + (row0 + i / HD) % group) * HD + i % HD, 0.f);
        return;
    }
    if (threadIdx.x < R) {
        const int idx = row0 + threadIdx.x;
        const bool there = (int)threadIdx.x < n_rows;
        rows.q[threadIdx.x] = there ? q + ((int64_t)(tok0 + idx / group) * G.heads + kvh * group + idx % group) * HD : nullptr;
        rows.last[threadIdx.x] = there ? keys.y - q_len + idx / group : -1;
    }
    __syncthreads();
    attend(w, rows, kv, kv_pages, G.page_table + (int64_t)b * G.table_width, kvh, G.kv_heads, key0, key1, scale, status);
    pdl_wait();
    if (splits > 1) {
        write_record(w, own_records + (((int64_t)b * gridDim.x + blockIdx.x) * gridDim.z + blockIdx.z) * REC);
        return;
    }
    finish(G, sh, out, G.group_of[b], tok0, row0, n_rows, kvh,
           [&](int r, float& m, float& l) {
               m = max_of(w, r);
               l = sum_of(w, r, m);
           },
           [&](int r, int c, float m) { return columns_of(w, r, c, m); });
}

// ---- 3. sequences whose own keys were cut ------------------------------------------
// Blocks (key head and tile of rows, sequence); max_splits: parts that there is room for.
template <typename T>
__global__ void __launch_bounds__(THREADS)
attn_shared_join_kernel(T* __restrict__ out, const Groups G, const Shared sh, const float* own_records, int max_splits, int* status) {
    pdl_wait();
    pdl_trigger();
    const int b = blockIdx.y, kvh = blockIdx.x % G.kv_heads, row0 = blockIdx.x / G.kv_heads * R;
    const int tok0 = G.cu_seqlens[b], q_len = G.cu_seqlens[b + 1] - tok0, group = G.heads / G.kv_heads;
    const int n_rows = min(R, q_len * group - row0);
    if (n_rows <= 0) return;
    const int2 keys = own_keys(G, b, q_len, status);
    const int splits = keys.x < 0 ? 1 : min(own_splits(keys.y - keys.x), max_splits);
    if (splits <= 1) return;
    const float* rec = own_records + ((int64_t)b * gridDim.x + blockIdx.x) * max_splits * REC;
    finish(G, sh, out, G.group_of[b], tok0, row0, n_rows, kvh,
           [&](int r, float& m, float& l) {
               for (int i = 0; i < splits; ++i) m = fmaxf(m, __ldcg(rec + (int64_t)i * REC + R * HD + 2 * r));
               for (int i = 0; i < splits; ++i) {
                   const float2 ml = __ldcg(reinterpret_cast<const float2*>(rec + (int64_t)i * REC + R * HD + 2 * r));
                   l = fmaf(ml.y, weight(ml.x, m), l);
               }
           },
           [&](int r, int c, float m) {
               float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
               for (int i = 0; i < splits; ++i) {
                   const float4 o = __ldcg(reinterpret_cast<const float4*>(rec + (int64_t)i * REC + (c / 4 * R + r) * 4));
                   const float a = weight(__ldcg(rec + (int64_t)i * REC + R * HD + 2 * r), m);
                   s.x = fmaf(o.x, a, s.x), s.y = fmaf(o.y, a, s.y), s.z = fmaf(o.z, a, s.z), s.w = fmaf(o.w, a, s.w);
               }
               return s;
           });
}

}  // namespace shared_prefix
}  // namespace wick

using namespace wick;

namespace wick {
namespace shared_prefix {

constexpr int PER_SM = 2;                          // blocks an SM of the kernel for shared keys

struct Call {
    Groups G;
    bool tc;                                       // the shared part's tcgen05 form
    int tiles_own, splits, blocks;                 // tiles of 16 rows of the longest sequence; parts of own keys; blocks for the shared keys
    int64_t plan_words, prefix_floats, own_floats;
};

static int plan_call(Call& c, bool half, int n_tokens, int n_seqs, int n_groups, int heads, int kv_heads, int max_pages, int own_bound, int max_q_len) {
    WICK_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "attention (shared prefix): %d heads over %d kv heads", heads, kv_heads);
    WICK_REQUIRE(n_seqs >= 1 && n_seqs <= 65535 && n_tokens >= 0, "attention (shared prefix): %d sequences, %d tokens", n_seqs, n_tokens);
    WICK_REQUIRE(n_groups >= 1 && n_groups <= MAX_GROUPS, "attention (shared prefix): %d groups (1 to %d)", n_groups, MAX_GROUPS);
    WICK_REQUIRE(max_pages >= 0 && own_bound >= 0 && max_q_len >= 0, "attention (shared prefix): bad bounds");
    const int group = heads / kv_heads;
    c.G.n = n_groups, c.G.n_seqs = n_seqs, c.G.max_pages = max_pages, c.G.heads = heads, c.G.kv_heads = kv_heads;
    c.tc = half && tc_supported();
    if (c.tc) {
        // heads of a tile: all of a key head's, or as many as 128 rows hold of more
        int gs = group;
        for (int n = 2; gs > TC_ROWS; ++n)
            if (group % n == 0) gs = group / n;
        c.G.rows = TC_ROWS / gs * gs, c.G.gs = gs, c.G.per_kv = group / gs, c.G.columns = heads / gs, c.G.block = 2, c.G.pair = 2;
    } else {
        c.G.rows = R, c.G.gs = group, c.G.per_kv = 1, c.G.columns = kv_heads, c.G.block = 1, c.G.pair = 1;
    }
    c.tiles_own = ceil_div((int64_t)max_q_len * group, R);
    WICK_REQUIRE((int64_t)c.tiles_own * kv_heads <= INT32_MAX / 2, "attention (shared prefix): %d tokens of one sequence are too many", max_q_len);
    c.splits = own_splits(own_bound);
    c.blocks = (c.tc ? 1 : PER_SM) * sm_count();
    c.plan_words = max_pages > 0 ? (2 * (n_groups + 1) + 1 + 3) / 4 * 4 : 0;
    const int64_t tiles = ceil_div((int64_t)n_tokens * c.G.gs, c.G.rows) + n_groups;
    c.prefix_floats = max_pages > 0 ? ((tiles / c.G.pair + n_groups) * c.G.columns + c.blocks) * c.G.pair * (c.tc ? TC_ROWS : R) * (HD + 2) : 0;
    c.own_floats = c.splits > 1 ? (int64_t)n_seqs * c.tiles_own * kv_heads * c.splits * REC : 0;
    return 0;
}

template <typename T>
static int attn_shared(const void* q, int n_tokens, const void* kv, int64_t kv_pages, void* out, const int* cu_groups, const int* pages,
                       const int* group_of, int n_groups, const int* cu_seqlens, int n_seqs, const int* start, const int* page_table, int table_width,
                       int heads, int kv_heads, int max_pages, int own_bound, int max_q_len, float scale, float* scratch, int64_t scratch_floats,
                       int* status, cudaStream_t s) {
    Call c = {};
    if (int e = plan_call(c, sizeof(T) == 2, n_tokens, n_seqs, n_groups, heads, kv_heads, max_pages, own_bound, max_q_len)) return e;
    WICK_REQUIRE((((uintptr_t)q | (uintptr_t)kv | (uintptr_t)out | (uintptr_t)scratch) & 15) == 0, "attention (shared prefix): operands must be 16-byte aligned");
    WICK_REQUIRE(scratch_floats >= c.plan_words + c.prefix_floats + c.own_floats, "attention (shared prefix): scratch of %lld floats, %lld needed",
                 (long long)scratch_floats, (long long)(c.plan_words + c.prefix_floats + c.own_floats));
    WICK_REQUIRE(scale >= 0.f, "attention (shared prefix): a negative scale");
    if (n_tokens == 0) return 0;
    Groups& G = c.G;
    G.cu_groups = cu_groups, G.pages = pages, G.group_of = group_of, G.cu_seqlens = cu_seqlens, G.start = start, G.page_table = page_table;
    G.table_width = table_width;
    int* plan = reinterpret_cast<int*>(scratch);
    float *records = scratch + c.plan_words, *own = records + c.prefix_floats;
    constexpr int SMEM = (int)sizeof(Work<T>);
    static bool raised = false;
    if (!raised) {
        WICK_CUDA(cudaFuncSetAttribute(attn_shared_prefix_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        WICK_CUDA(cudaFuncSetAttribute(attn_shared_own_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        raised = true;
    }
    Shared sh = {nullptr, records, c.tc ? TC_ROWS : R};
    if (max_pages > 0) sh.plan = plan;
    if (max_pages > 0 && c.tc) {
        if (int e = launch_tc(q, n_tokens, kv, kv_pages, G, c.blocks, scale, plan, records, status, s)) return e;
    } else if (max_pages > 0) {
        WICK_CUDA(launch(attn_shared_prefix_kernel<T>, dim3(c.blocks), dim3(THREADS), (size_t)SMEM, s, (const T*)q, (const T*)kv, kv_pages, G, scale, plan,
                         records, status));
        if (int e = check_launch("attn_shared_prefix")) return e;
    }
    WICK_CUDA(launch(attn_shared_own_kernel<T>, dim3(c.tiles_own * kv_heads, n_seqs, c.splits), dim3(THREADS), (size_t)SMEM, s, (const T*)q, (const T*)kv,
                     kv_pages, (T*)out, G, sh, scale, own, status));
    if (int e = check_launch("attn_shared_own")) return e;
    if (c.splits > 1) {
        WICK_CUDA(launch(attn_shared_join_kernel<T>, dim3(c.tiles_own * kv_heads, n_seqs), dim3(THREADS), 0, s, (T*)out, G, sh, (const float*)own,
                         c.splits, status));
        if (int e = check_launch("attn_shared_join")) return e;
    }
    return 0;
}

}  // namespace shared_prefix
}  // namespace wick

// float32 words of scratch that a call of these sizes needs (half: of the bfloat16 form; -1: refused, see wick_last_error).
WICK_API long long wick_attn_shared_scratch(int half, int n_tokens, int n_seqs, int n_groups, int heads, int kv_heads, int max_pages, int own_bound, int max_q_len) {
    shared_prefix::Call c = {};
    if (shared_prefix::plan_call(c, half != 0, n_tokens, n_seqs, n_groups, heads, kv_heads, max_pages, own_bound, max_q_len)) return -1;
    return c.plan_words + c.prefix_floats + c.own_floats;
}

// q, out: [n_tokens, heads, HD]; kv: one schedule entry's cache [kv_pages, 2, kv_heads, 64, HD], which holds the new tokens' keys and
// values; cu_groups: int32 [n_groups + 1], the sequences of each group; pages: int32 [n_groups], the leading pages that a group's
// sequences have in common (each holds that many whole pages before this step); group_of: int32 [n_seqs].  max_pages, own_bound,
// max_q_len: upper bounds of pages, of a sequence's positions behind its group's pages, and of a sequence's new tokens.
// status: 10 a page outside the cache, 11 a sequence that does not fit its group or its page table (its rows become zeros).
#define WICK_ATTN_SHARED(NAME, T)                                                                                                                        \
    WICK_API int NAME(const void* q, int n_tokens, const void* kv, int64_t kv_pages, void* out, const int* cu_groups, const int* pages,                   \
                      const int* group_of, int n_groups, const int* cu_seqlens, int n_seqs, const int* start, const int* page_table, int table_width,     \
                      int heads, int kv_heads, int max_pages, int own_bound, int max_q_len, float scale, float* scratch, int64_t scratch_floats,          \
                      int* status, void* s) {                                                                                                             \
        return shared_prefix::attn_shared<T>(q, n_tokens, kv, kv_pages, out, cu_groups, pages, group_of, n_groups, cu_seqlens, n_seqs, start,             \
                                             page_table, table_width, heads, kv_heads, max_pages, own_bound, max_q_len, scale, scratch, scratch_floats,   \
                                             status, (cudaStream_t)s);                                                                                    \
    }
WICK_ATTN_SHARED(wick_attn_shared_bf16, __nv_bfloat16)
WICK_ATTN_SHARED(wick_attn_shared_f32, float)
