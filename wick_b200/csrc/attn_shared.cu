// Attention over a prefix that groups of sequences share, and over each sequence's own keys behind it (attn_shared.cuh has the
// mathematics and how the work is cut): the entry points, and the form for any head size in float32, and in bfloat16 for head sizes
// other than 64 and 128 (those: attn_shared_tc.cu, attn_shared_own.cu).
//
//   1. attn_shared_part_kernel over the sequences' own keys and the groups' shared ones: tiles of 16 rows, a record (m, l, o) per run;
//   2. attn_shared_join_kernel: a row's records joined and written.
//
// bfloat16: mma.sync on tiles of 16 rows and 16 keys.  Keys and values go from the cache straight to registers: the inner index of
// q . k is summed over in any order, so a lane takes 16 neighbouring bytes of a key row and the same of its query row as operands of
// two instructions; and a value row's numbers may stand in any order of columns, so a lane takes 16 neighbouring bytes of each of four
// keys' rows and pairs them by byte permutation.  No shared memory, no barrier until the warps' parts are joined.  Weights enter the second
// product rounded to bfloat16, and their sum is taken of the rounded ones, so that a row of equal values keeps them.
// float32: products and sums on the CUDA cores, keys and values through shared memory, 32 keys at a time: bound by the chain of a page, two
// times 64 rounds through shared memory by four warps (6 sequences behind 1,000 positions, 16 heads over 4 of 128: 12.2 us, 7 MB; the reads
// at the shared memory's rate would be 2).
// The join is bound by a chain (plan, then records that other SMs have just written) and, where there are many, by the records' bytes: 64
// sequences of 32 heads with ten records a row of the shared keys, 11 MB, 7 us; 4 of 16 heads 4.5.
#include "common.cuh"
#include "attn_shared.cuh"
#include "packed.cuh"

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

// A warp has the scores of four rows with a tile's 32 keys, a thread the sums of four rows and four columns.  FEW: where there are four rows at
// most (a token of up to four heads), a warp has a quarter of the tile's keys, a lane one row's score with one of them, then four columns of
// all four rows; the warps' parts are joined at the end (11 sequences of up to 1,085 own positions behind 732, 8 heads of 64 over 8: 24.5 us,
// and 27.8 with a quarter of the warps at work).
template <bool FEW>
__device__ void attend(Work<float>& w, const Rows<float>& rows, const float* __restrict__ kv, int64_t kv_pages, const int* __restrict__ tab, int kvh,
                       int n_kv, int key0, int key1, float scale, int* status) {
    constexpr int KT = Work<float>::KT, ITEMS = FEW ? (HD / 4 + 31) / 32 : (HD + THREADS - 1) / THREADS;
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
        if constexpr (FEW) {
            const int mine = warp * 8 + (lane & 7), row = lane >> 3;
            float t4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(&w.k[i & 1][mine][d]), q4 = *reinterpret_cast<const float4*>(&w.q[row][d]);
                t4[0] = fmaf(q4.x, k4.x, t4[0]), t4[1] = fmaf(q4.y, k4.y, t4[1]), t4[2] = fmaf(q4.z, k4.z, t4[2]), t4[3] = fmaf(q4.w, k4.w, t4[3]);
            }
            const int key = key0 + i * KT + mine;
            const float x = key < key1 && key <= rows.last[row] ? ((t4[0] + t4[1]) + (t4[2] + t4[3])) * sl2 : -INFINITY;
            float n = x;
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) n = fmaxf(n, __shfl_xor_sync(0xffffffffu, n, o));
            n = fmaxf(m[0], n);
            const float a = weight(m[0], n), p = weight(x, n);
            l[0] = l[0] * a + p;                       // (of this lane's keys)
            m[0] = n;
            float ar[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) ar[r] = __shfl_sync(0xffffffffu, a, r * 8);
#pragma unroll
            for (int it = 0; it < ITEMS; ++it)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[it][r][e] *= ar[r];
#pragma unroll
            for (int key = 0; key < 8; ++key) {
                float pr[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) pr[r] = __shfl_sync(0xffffffffu, p, r * 8 + key);
#pragma unroll
                for (int it = 0; it < ITEMS; ++it) {
                    const int c = (it * 32 + lane) * 4;
                    if (c >= HD) continue;
                    const float4 v4 = *reinterpret_cast<const float4*>(&w.v[i & 1][warp * 8 + key][c]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        acc[it][r][0] = fmaf(pr[r], v4.x, acc[it][r][0]), acc[it][r][1] = fmaf(pr[r], v4.y, acc[it][r][1]);
                        acc[it][r][2] = fmaf(pr[r], v4.z, acc[it][r][2]), acc[it][r][3] = fmaf(pr[r], v4.w, acc[it][r][3]);
                    }
                }
            }
            __syncthreads();
            continue;
        }
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
    if constexpr (FEW) {
        // the warps' parts, in the place of the keys: [W][4][HD] sums, [W][4] maxima and sums of weights
        float *parts = &w.k[0][0][0], *ml = parts + W * 4 * HD;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
        if ((lane & 7) == 0) ml[(warp * 4 + (lane >> 3)) * 2] = m[0], ml[(warp * 4 + (lane >> 3)) * 2 + 1] = l[0];
#pragma unroll
        for (int it = 0; it < ITEMS; ++it) {
            const int c = (it * 32 + lane) * 4;
            if (c >= HD) continue;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<float4*>(parts + (warp * 4 + r) * HD + c) = make_float4(acc[it][r][0], acc[it][r][1], acc[it][r][2], acc[it][r][3]);
        }
        __syncthreads();
        for (int idx = tid; idx < 4 * HD; idx += THREADS) {
            const int r = idx / HD, c = idx % HD;
            float mm = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < W; ++k) mm = fmaxf(mm, ml[(k * 4 + r) * 2]);
#pragma unroll
            for (int k = 0; k < W; ++k) sum = fmaf(parts[(k * 4 + r) * HD + c], weight(ml[(k * 4 + r) * 2], mm), sum);
            w.o[0][r][c] = sum;
        }
        if (tid < 4) {
            float mm = -INFINITY, sum = 0.f;
            for (int k = 0; k < W; ++k) mm = fmaxf(mm, ml[(k * 4 + tid) * 2]);
            for (int k = 0; k < W; ++k) sum = fmaf(ml[(k * 4 + tid) * 2 + 1], weight(ml[(k * 4 + tid) * 2], mm), sum);
            w.m[0][tid] = mm, w.l[0][tid] = sum;
        }
        __syncthreads();
        return;
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
template <typename T> __device__ __forceinline__ void write_record(const Work<T>& w, float* rec, int n_rows) {
    for (int i = threadIdx.x; i < R * HD / 4; i += THREADS) {
        const int r = i % R, c = i / R;
        if (r >= n_rows) continue;
        *reinterpret_cast<float4*>(rec + i * 4) = columns_of(w, r, c * 4, max_of(w, r));
    }
    if ((int)threadIdx.x < min(R, n_rows)) {
        const float m = max_of(w, threadIdx.x);
        *reinterpret_cast<float2*>(rec + R * HD + 2 * threadIdx.x) = make_float2(m, sum_of(w, threadIdx.x, m));
    }
}

// ---- the parts ---------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(THREADS)
attn_shared_part_kernel(const T* q, const T* __restrict__ kv, int64_t kv_pages, T* __restrict__ out, const Groups G, int groups, float scale, int* plan,
                        float* records, int* status) {
    extern __shared__ __align__(16) uint8_t smem[];
    Work<T>& w = *reinterpret_cast<Work<T>*>(smem);
    __shared__ Rows<T> rows;
    pdl_trigger();
    const int group = G.heads / G.kv_heads;
    const OwnParts parts{G, R, groups};
    Walk walk(parts, gridDim.x, nullptr);           // (the description may be read before the wait)
    pdl_wait();
    q = fresh(q), kv = fresh(kv);                   // (the step's own keys and values have just been appended)
    Segment s;
    while (walk.segment(s)) {                       // (every warp walks the same way)
        __syncthreads();                            // (the rows and the work of the segment before)
        if (threadIdx.x < R) {
            const int idx = s.tile * R + threadIdx.x, tok = idx / group;
            const bool there = idx < s.cut.n_tok * group;
            rows.q[threadIdx.x] = there ? q + ((int64_t)(s.cut.tok0 + tok) * G.heads + s.column * group + idx - tok * group) * HD : nullptr;
            rows.last[threadIdx.x] = there ? s.last(tok) : -1;
        }
        __syncthreads();
        const int* table = G.page_table + (int64_t)s.cut.seq * G.table_width;
        const int n_rows = s.cut.n_tok * group - s.tile * R, key0 = (s.cut.first + s.from) * kPage, key1 = min((s.cut.first + s.to) * kPage, s.cut.end);
        if constexpr (sizeof(T) == 2) attend(w, rows, kv, kv_pages, table, s.column, G.kv_heads, key0, key1, scale, status);
        else if (n_rows <= 4) attend<true>(w, rows, kv, kv_pages, table, s.column, G.kv_heads, key0, key1, scale, status);
        else attend<false>(w, rows, kv, kv_pages, table, s.column, G.kv_heads, key0, key1, scale, status);
        write_record(w, records + (int64_t)s.record * REC, n_rows);
    }
    if (blockIdx.x == 0 && threadIdx.x < 32) {
        const Walk all(parts, gridDim.x, plan);
        clear_unfit(parts, out, G.heads * HD, all.wrong, status);
    }
}

// ---- the records joined ------------------------------------------------------------
// Where a row's records of one kind are: n of them, `step` floats apart, the row at place r.
struct Source {
    const float* at;
    int n, step, rows, r;
};
__device__ __forceinline__ Source shared_source(const Groups& G, const Records& rec, int g, const Cut& c, int tok, int h, int kvh) {
    Source s = {rec.at, 0, 0, rec.rows, 0};
    if (!rec.plan || c.pages == 0) return s;
    const int idx = (tok - c.tok0) * G.gs + h % G.gs, tile = idx / G.rows, floats = rec.rows * (HD + 2);
    const int run = rec.plan[0];                   // (0, no records: looked at last, beside the other reads)
    const Place p = place_of(G, c, max(run, 1), tile, kvh * G.per_kv + h / G.gs);
    s.at = rec.at + (int64_t)((rec.plan[1 + g] + p.first) * G.pair + tile % G.pair) * floats;
    s.n = run > 0 ? p.n : 0, s.step = floats * G.pair, s.r = idx - tile * G.rows;
    return s;
}
__device__ __forceinline__ Source own_source(const OwnParts& parts, const Records& rec, int b, const Cut& c, int idx, int kvh) {
    if (c.pages == 0) return Source{rec.at, 0, 0, rec.rows, 0};
    const int *units = rec.plan + 1, *items = rec.plan + 2 + parts.n();
    const int workers = rec.plan[0];               // (0, no records: looked at last, beside the other reads)
    const Deal deal(units[parts.n()], max(workers, 1));
    const int tile = idx / parts.rows, item = tile * parts.G.kv_heads + kvh, u = units[b] + item * c.pages, c0 = deal.worker_of(u);
    const int floats = rec.rows * (HD + 2);
    return Source{rec.at + (int64_t)(items[b] + item + c0) * floats, workers > 0 ? deal.worker_of(u + c.pages - 1) - c0 + 1 : 0, floats, rec.rows, idx - tile * parts.rows};
}

// Blocks (four rows, sequence): a thread has a row and four columns (and those 128, 256 .. behind), four neighbouring threads four
// neighbouring rows, whose sums lie side by side in a record.  JN records at a time (16 where all blocks run at once, and 8, for more of them on
// an SM, where they do not), the shared keys' and the own ones' in one
// list, so that all reads of a row that has no more stand side by side: each of the eight threads of a row in a warp finds a weight or two,
// and all read the sums of all JN at once (behind the last one: of that one again, without weight).
constexpr int JT = 128, JR = 4;
template <typename T, int JN>
__global__ void __launch_bounds__(JT)
attn_shared_join_kernel(T* __restrict__ out, const Groups G, const Records shared, const Records own, int groups) {
    const int b = blockIdx.y, row = (int)blockIdx.x * JR + (int)threadIdx.x % JR, group = G.heads / G.kv_heads;
    const OwnParts parts{G, own.rows, groups};
    const Cut mine = parts(b);                      // (the description may be read before the wait)
    const int tok = row / G.heads, head = row - tok * G.heads, kvh = head / group, h = head - kvh * group, g = G.group_of[b];
    const bool there = tok < mine.n_tok && mine.pages > 0;
    Cut c = Cut{};
    if (there) c = groups ? parts(G.n_seqs + g) : SharedParts{G}(g);
    pdl_wait();
    pdl_trigger();
    Source s0 = {shared.at, 0, 0, 0, 0}, s1 = s0;
    if (there) {
        s0 = groups ? own_source(parts, own, G.n_seqs + g, c, (mine.tok0 + tok - c.tok0) * group + h, kvh) : shared_source(G, shared, g, c, mine.tok0 + tok, h, kvh);
        s1 = own_source(parts, own, b, mine, tok * group + h, kvh);
    }
    const int k = (threadIdx.x & 31) / JR, n = s0.n + s1.n;        // k: of the eight threads of a row
    // number `at` of a record of s0's, `at1` of one of s1's, of record i of both
    auto place = [&](int i, int at, int at1) {
        const bool first = i < s0.n;
        return (first ? s0.at + at : s1.at + at1) + (int64_t)(first ? i : i - s0.n) * (first ? s0.step : s1.step);
    };
    const int ml0 = s0.rows * HD + 2 * s0.r, ml1 = s1.rows * HD + 2 * s1.r;
    for (int col = threadIdx.x / JR; col < (HD / 4 + 7) / 8 * 8; col += JT / JR) {     // (whole warps)
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        float m = -INFINITY, l = 0.f;
        const int at0 = (min(col, HD / 4 - 1) * s0.rows + s0.r) * 4, at1 = (min(col, HD / 4 - 1) * s1.rows + s1.r) * 4;
#pragma unroll 1
        for (int i0 = 0; __any_sync(0xffffffffu, i0 < n); i0 += JN) {
            const int left = n - i0;                // (a row without further records: reads the last one again, or none)
            float2 x[JN / 8];
            float4 o[JN];
#pragma unroll
            for (int i = 0; i < JN / 8; ++i) {
                x[i] = make_float2(-INFINITY, 0.f);
                if (k + 8 * i < left) x[i] = *reinterpret_cast<const float2*>(place(i0 + k + 8 * i, ml0, ml1));
            }
#pragma unroll
            for (int i = 0; i < JN; ++i)
                if (left > 0) o[i] = *reinterpret_cast<const float4*>(place(i0 + min(i, left - 1), at0, at1));
            float most = m;
#pragma unroll
            for (int i = 0; i < JN / 8; ++i) most = fmaxf(most, x[i].x);
#pragma unroll
            for (int d = JR; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            const float before = weight(m, most);
            m = most;
            l *= before, s.x *= before, s.y *= before, s.z *= before, s.w *= before;
            float w[JN / 8], add = 0.f;
#pragma unroll
            for (int i = 0; i < JN / 8; ++i) {
                w[i] = weight(x[i].x, m);
                if (k + 8 * i < left) add += x[i].y * w[i];
            }
#pragma unroll
            for (int d = JR; d < 32; d <<= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
            l += add;
#pragma unroll
            for (int i = 0; i < JN; ++i) {
                const float a = __shfl_sync(0xffffffffu, w[i / 8], i % 8 * JR + (threadIdx.x % JR));
                if (i >= left) continue;
                s.x = fmaf(o[i].x, a, s.x), s.y = fmaf(o[i].y, a, s.y), s.z = fmaf(o[i].z, a, s.z), s.w = fmaf(o[i].w, a, s.w);
            }
        }
        const float f = l != 0.f ? __fdiv_rn(1.0f, l) : 0.f;       // (a sum that is no number shows)
        if (there && col < HD / 4) st4(out + ((int64_t)(mine.tok0 + tok) * G.heads + head) * HD + col * 4, s.x * f, s.y * f, s.z * f, s.w * f);
    }
}

}  // namespace shared_prefix
}  // namespace wick

using namespace wick;

namespace wick {
namespace shared_prefix {

constexpr int FEW = 3500 * (HD < 128 ? 2 : 1);
// Thread blocks an SM of the form for any head size: what its shared memory holds (the same: 20.5 us, and 24.5 with two everywhere; 24 sequences
// behind 3,000 positions, 24 heads over 4 of 64, float32: 38.9 and 50.4).
constexpr int PER_SM = HD > 128 ? 1 : 256 / HD < 8 ? 256 / HD : 8;

struct Call {
    Groups G;
    bool fast;                                     // the forms for bfloat16 at head sizes 64 and 128
    bool tc;                                       // the shared keys have a kernel of their own
    int blocks, blocks_own;                        // for the shared keys, for the own ones
    int64_t plan_shared, plan_own, shared_floats, own_floats;
    int64_t all() const { return plan_shared + plan_own + shared_floats + own_floats; }
};

static int plan_call(Call& c, bool half, int n_tokens, int n_seqs, int n_groups, int heads, int kv_heads, int max_pages, int own_bound, int max_q_len) {
    WICK_REQUIRE(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "attention (shared prefix): %d heads over %d kv heads", heads, kv_heads);
    WICK_REQUIRE(n_seqs >= 1 && n_seqs <= 65535 && n_tokens >= 0, "attention (shared prefix): %d sequences, %d tokens", n_seqs, n_tokens);
    WICK_REQUIRE(n_groups >= 1 && n_groups <= MAX_GROUPS, "attention (shared prefix): %d groups (1 to %d)", n_groups, MAX_GROUPS);
    WICK_REQUIRE(max_pages >= 0 && own_bound >= 0 && max_q_len >= 0 && (int64_t)max_q_len * heads <= INT32_MAX / 2, "attention (shared prefix): bad bounds");
    const int group = heads / kv_heads;
    Groups& G = c.G;
    G.n = n_groups, G.n_seqs = n_seqs, G.max_pages = max_pages, G.heads = heads, G.kv_heads = kv_heads;
    G.single = max_q_len == 1 && n_tokens == n_seqs;
    c.fast = half && fast_supported();
    // heads of a tcgen05 tile: all of a key head's, or as many as 128 rows hold of more
    int gs = group;
    for (int n = 2; gs > TC_ROWS; ++n)
        if (group % n == 0) gs = group / n;
    G.rows = TC_ROWS / gs * gs, G.gs = gs, G.per_kv = group / gs, G.columns = heads / gs, G.pair = 2;
    const int sms = sm_count(), rows_own = c.fast ? OWN_ROWS : R, own_per_sm = c.fast ? OWN_WARPS * (128 / HD) : PER_SM;
    const int64_t tiles = (int64_t)ceil_div((int64_t)n_tokens * gs, G.rows) + n_groups, items = (tiles / 2 + n_groups) * G.columns;
    const int64_t units = tiles * G.columns * max_pages;
    const int64_t items_seqs = ((int64_t)ceil_div((int64_t)n_tokens * group, rows_own) + n_seqs) * kv_heads, pages_own = ceil_div(own_bound, kPage);
    const int64_t items_groups = max_pages > 0 ? ((int64_t)ceil_div((int64_t)n_tokens * group, rows_own) + n_groups) * kv_heads : 0;
    WICK_REQUIRE(units <= INT32_MAX / 2 && items_seqs * pages_own + items_groups * max_pages <= INT32_MAX / 2, "attention (shared prefix): too much for one step");
    // The shared keys have a kernel of their own from FEW pages of 8 rows on: fewer take the own keys' kernel, and one launch, less time (16
    // sequences of 32 heads over 8 of 128: behind 2,048 positions 14.6 us together and 16.3 apart, 4,096 20.1 and 18.9; 48 of 24 over 4 of
    // 64: 2,048 17.5 and 19.8, 4,096 24.9 and 21.3; over 120 sizes the better of the two is missed by 0.2 % and 0.7 % on average).
    c.tc = c.fast && items_groups * max_pages > FEW;
    int first = sms, second = own_per_sm * sms;
    if (c.tc) {
        // The own keys' kernel starts as soon as all thread blocks of the first one run, on the SMs that those leave (64 sequences of 370 own
        // positions behind 8,192 shared ones, 32 heads over 8: one behind the other 54 us, half of the SMs each 42; 24 behind 31,000, 64 over
        // 8: 72, and 64 on four fifths and one).  Shares by what each is expected to take: a page of own keys a quarter of a turn
        // of a tile and two pages, which takes 0.6 of one where the tile has both streams.  (Lengths are on the device: groups of equal
        // size are assumed, that share 0.7 of the most pages where there are several, and half of the most own positions.)
        const int per_group = ceil_div(ceil_div(n_tokens, n_groups) * (int64_t)gs, G.rows);
        const double work = (double)n_groups * G.columns * per_group * (per_group == 1 ? 0.6 : 1.0) * ceil_div(max_pages, 2) * (n_groups > 1 ? 0.7 : 1.0);
        const double tiles_own = G.single ? (double)n_seqs * ceil_div(group, OWN_ROWS) : (double)n_tokens * group / OWN_ROWS + 0.5 * n_seqs;
        const double work_own = tiles_own * kv_heads * (0.5 * own_bound / kPage + 0.5) * 0.26;
        first = (int)min((int64_t)max(1, min(sms - 8, (int)(sms * work / (work + work_own)))), max((int64_t)1, units / 2));
        second = own_per_sm * (sms - first);
    }
    // No more thread blocks than there can be runs of work; and few items with many pages are cut into longer runs than one page, since a row's
    // records are joined sixteen at a time (4 sequences of 8 heads of 64 behind 16,384 positions: runs of one page 42 us, of seven 23; 4 of
    // 32 over 8 of 128 behind 4,096: 14.8, 12.1).
    const int64_t items_own = items_seqs + (c.tc ? 0 : items_groups), most = max(pages_own, c.tc ? (int64_t)0 : (int64_t)max_pages);
    const int run = max(1, (int)sqrt(most / 5.0));
    c.blocks = (int)max((int64_t)1, min((int64_t)first, units / 2));
    c.blocks_own = (int)max((int64_t)1, min((int64_t)second, (items_seqs * pages_own + (c.tc ? 0 : items_groups * max_pages)) / run));
    c.plan_shared = c.tc ? (n_groups + 2 + 3) / 4 * 4 : 0;
    c.plan_own = (2 * (n_seqs + n_groups) + 3 + 3) / 4 * 4;
    c.shared_floats = c.tc ? max((int64_t)c.blocks, items) * 2 * TC_ROWS * (HD + 2) : 0;
    c.own_floats = (items_own + c.blocks_own) * rows_own * (HD + 2);
    return 0;
}

template <typename T>
static int attn_shared(const T* q, int n_tokens, const T* kv, int64_t kv_pages, T* out, const int* cu_groups, const int* pages,
                       const int* group_of, int n_groups, const int* cu_seqlens, int n_seqs, const int* start, const int* page_table, int table_width,
                       int heads, int kv_heads, int max_pages, int own_bound, int max_q_len, float scale, float* scratch, int64_t scratch_floats,
                       int* status, cudaStream_t s) {
    Call c = {};
    if (int e = plan_call(c, sizeof(T) == 2, n_tokens, n_seqs, n_groups, heads, kv_heads, max_pages, own_bound, max_q_len)) return e;
    WICK_REQUIRE((((uintptr_t)q | (uintptr_t)kv | (uintptr_t)out | (uintptr_t)scratch) & 15) == 0, "attention (shared prefix): operands must be 16-byte aligned");
    WICK_REQUIRE(scratch_floats >= c.all(), "attention (shared prefix): scratch of %lld floats, %lld needed", (long long)scratch_floats, (long long)c.all());
    WICK_REQUIRE(scale >= 0.f, "attention (shared prefix): a negative scale");
    if (n_tokens == 0) return 0;
    Groups& G = c.G;
    G.cu_groups = cu_groups, G.pages = pages, G.group_of = group_of, G.cu_seqlens = cu_seqlens, G.start = start, G.page_table = page_table;
    G.table_width = table_width;
    int *plan = reinterpret_cast<int*>(scratch), *plan_own = plan + c.plan_shared;
    float *records = scratch + c.plan_shared + c.plan_own, *own = records + c.shared_floats;
    const int groups = c.tc || max_pages == 0 ? 0 : n_groups;      // that the own keys' kernel takes too
    if (fast_supported() && sizeof(T) == 2) {
        if (c.tc)
            if (int e = launch_tc(q, n_tokens, kv, kv_pages, G, c.blocks, scale, plan, records, status, s)) return e;
        if (int e = launch_own(q, kv, kv_pages, out, G, groups, c.tc, c.blocks_own, scale, plan_own, own, status, s)) return e;
    } else if constexpr (sizeof(T) == 4 || (HD != 64 && HD != 128)) {
        constexpr int SMEM = (int)sizeof(Work<T>);
        static bool raised = false;
        if (!raised) {
            WICK_CUDA(cudaFuncSetAttribute(attn_shared_part_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
            raised = true;
        }
        WICK_CUDA(launch(attn_shared_part_kernel<T>, dim3(c.blocks_own), dim3(THREADS), (size_t)SMEM, s, q, kv, kv_pages, out, G, groups, scale, plan_own, own,
                         status));
        if (int e = check_launch("attn_shared_part")) return e;
    }
    const Records sh = {c.tc ? plan : nullptr, records, TC_ROWS}, ow = {plan_own, own, c.fast ? OWN_ROWS : R};
    const dim3 grid(ceil_div((int64_t)max_q_len * heads, JR), n_seqs);
    if ((int64_t)grid.x * grid.y <= 4 * sm_count()) WICK_CUDA(launch(attn_shared_join_kernel<T, 16>, grid, dim3(JT), 0, s, out, G, sh, ow, groups));
    else WICK_CUDA(launch(attn_shared_join_kernel<T, 8>, grid, dim3(JT), 0, s, out, G, sh, ow, groups));
    return check_launch("attn_shared_join");
}

}  // namespace shared_prefix
}  // namespace wick

// float32 words of scratch that a call of these sizes needs (half: of the bfloat16 form; -1: refused, see wick_last_error), and the
// kernels that it launches.
WICK_API long long wick_attn_shared_scratch(int half, int n_tokens, int n_seqs, int n_groups, int heads, int kv_heads, int max_pages, int own_bound, int max_q_len,
                                            int* kernels) {
    shared_prefix::Call c = {};
    if (shared_prefix::plan_call(c, half != 0, n_tokens, n_seqs, n_groups, heads, kv_heads, max_pages, own_bound, max_q_len)) return -1;
    *kernels = n_tokens == 0 ? 0 : 2 + c.tc;
    return c.all();
}

// q, out: [n_tokens, heads, HD]; kv: one schedule entry's cache [kv_pages, 2, kv_heads, 64, HD], which holds the new tokens' keys and
// values; cu_groups: int32 [n_groups + 1], the sequences of each group; pages: int32 [n_groups], the leading pages that a group's
// sequences have in common (each holds that many whole pages before this step); group_of: int32 [n_seqs].  max_pages, own_bound,
// max_q_len: upper bounds of pages, of a sequence's positions behind its group's pages, and of a sequence's new tokens.
// status: 10 a page outside the cache, 11 a sequence that does not fit its group or its page table (its rows become zeros), or groups in no order
// (where the own keys' kernel does them too all rows become zeros, else they lack the shared keys).
#define WICK_ATTN_SHARED(NAME, T)                                                                                                                        \
    WICK_API int NAME(const void* q, int n_tokens, const void* kv, int64_t kv_pages, void* out, const int* cu_groups, const int* pages,                   \
                      const int* group_of, int n_groups, const int* cu_seqlens, int n_seqs, const int* start, const int* page_table, int table_width,     \
                      int heads, int kv_heads, int max_pages, int own_bound, int max_q_len, float scale, float* scratch, int64_t scratch_floats,          \
                      int* status, void* s) {                                                                                                             \
        return shared_prefix::attn_shared<T>((const T*)q, n_tokens, (const T*)kv, kv_pages, (T*)out, cu_groups, pages, group_of, n_groups, cu_seqlens, n_seqs, start,             \
                                             page_table, table_width, heads, kv_heads, max_pages, own_bound, max_q_len, scale, scratch, scratch_floats,   \
                                             status, (cudaStream_t)s);                                                                                    \
    }
WICK_ATTN_SHARED(wick_attn_shared_bf16, __nv_bfloat16)
WICK_ATTN_SHARED(wick_attn_shared_f32, float)
WICK_PACKED(wick_attn_shared_bf16)
WICK_PACKED(wick_attn_shared_f32)
