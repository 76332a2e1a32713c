// The own keys of each sequence behind its group's shared prefix: bfloat16, head sizes 64 and 128.
//
// A thread block is ONE warp that feeds itself; six of them (head size 64: twelve) fill an SM's shared memory.  The pages of all items (a
// sequence's 16 rows of one key head) are dealt to the warps in equal runs (attn_shared.cuh).  A warp has room for one page of keys and
// one of values: the next page's keys are copied (TMA, 128-byte swizzle) while it turns scores into weights and multiplies the values,
// the next values while it multiplies the next keys, from one item into the next.  Queries are on the 16-row side of mma.sync, so that weights
// are the second product's operand as they stand; they enter it rounded to bfloat16, and their sum is taken of the rounded ones.  Every item leaves
// a record per run that has a part of it.
// Bound by the bytes of the keys and values.  (Measured and left: blocks of four or eight warps that shared a page met three times
// a page, 2,000 clocks of latency that two blocks an SM could not hide: 64 sequences of 370 own positions, 8 key heads, 28 us.)
// The kernel of the shared part runs before this one, which starts under its last blocks.
#include "tcgen05.cuh"
#include "attn_shared.cuh"

#ifndef WICK_HD
#error "compile with -DWICK_HD=<head_dim>"
#endif

namespace wick {
namespace shared_prefix {

bool fast_supported() { return WICK_HD == 64 || WICK_HD == 128; }

namespace own {

constexpr bool SUPPORTED = WICK_HD == 64 || WICK_HD == 128;
constexpr int HD = SUPPORTED ? WICK_HD : 64;           // other head sizes: never launched
typedef __nv_bfloat16 bf16;
constexpr int R = OWN_ROWS;
constexpr int PANELS = HD / 64, PANEL_BYTES = kPage * 128, TILE_BYTES = PANELS * PANEL_BYTES;   // a page of keys, or of values
constexpr int KS = HD / 16, NT = HD / 8;               // steps of q . k; tiles of eight value columns
constexpr int REC = R * (HD + 2);

struct Smem {
    uint8_t k[TILE_BYTES], v[TILE_BYTES];
    uint64_t k_full, v_full;
    int abort_flag;
};
constexpr int SMEM_BYTES = (int)sizeof(Smem);
static_assert(OWN_WARPS * (128 / HD) * (SMEM_BYTES + 1024) <= 228 * 1024, "the warps of an SM");

__device__ __forceinline__ void ldsm_x4(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t* r, uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte offset, inside a page's tile, of the 16-byte chunk `chunk` (8 numbers) of row `row`.
__device__ __forceinline__ uint32_t tile_off(int row, int chunk) {
    return (uint32_t)((chunk >> 3) * PANEL_BYTES + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// The page after the one at hand: the run's part it lies in, its place in it.  A lane holds one of 32 page numbers.
struct Ahead {
    Segment s;
    int j, ids;
    bool any;
};

__global__ void __launch_bounds__(32)
attn_shared_own_kernel(const __grid_constant__ CUtensorMap kv_map, const bf16* q, int64_t kv_pages, bf16* __restrict__ out, const Groups G, int after_shared,
                       float scale, int* plan, float* records, int* status) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    const int lane = threadIdx.x, g = lane >> 2, t = lane & 3;
    const int group = G.heads / G.kv_heads;
    const float sl2 = scale * LOG2E;
    if (lane == 0) {
        sm.abort_flag = 0;
        mbar_init(&sm.k_full, 1), mbar_init(&sm.v_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    // (With a shared part the kernel before this one is the one that computes it, and has waited for q and the cache.)
    if (!after_shared) pdl_wait();
    pdl_trigger();
    const OwnParts parts{G, R};
    Walk<OwnParts> walk(parts, gridDim.x, nullptr);
    Ahead next;
    auto know_ids = [&]() {                            // from page next.j on
        const int* table = G.page_table + (int64_t)next.s.cut.seq * G.table_width + next.s.cut.first;
        int id = next.j + lane < next.s.to ? table[next.j + lane] : 0;
        if (id < 0 || id >= kv_pages) {
            atomicCAS(status, 0, 10);
            id = 0;
        }
        next.ids = id;
    };
    auto begin = [&]() {
        next.any = walk.segment(next.s);
        next.j = next.s.from;
        if (next.any) know_ids();
    };
    auto copy = [&](int v) {                           // of the page ahead; its place was read by this warp before
        const int page = __shfl_sync(0xffffffffu, next.ids, (next.j - next.s.from) & 31);
        __syncwarp();
        if (lane == 0) {
            uint64_t* bar = v ? &sm.v_full : &sm.k_full;
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            mbar_expect_tx(bar, TILE_BYTES);
            for (int pn = 0; pn < PANELS; ++pn)
                tma_load_2d(&kv_map, bar, (v ? sm.v : sm.k) + pn * PANEL_BYTES, pn * 64, ((page * 2 + v) * G.kv_heads + next.s.column) * kPage);
        }
        __syncwarp();
    };
    bool ok = (smem_u32(smem_raw) & 1023) == 0;        // (always: the block's dynamic shared memory is all there is)
    if (!ok && lane == 0) atomicCAS(status, 0, 7);
    next.any = false;
    if (ok) begin();
    if (next.any) copy(0), copy(1);

    uint32_t qa[KS][4];
    float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    int last0 = -1, last1 = -1;                        // the last position that rows g and g + 8 see
    bool upper = false;                                // rows 8 to 15 are there
    const uint32_t k_s = smem_u32(sm.k), v_s = smem_u32(sm.v);
#pragma unroll 1
    for (int turn = 0; ok && next.any; turn ^= 1) {
        const bool first = next.j == next.s.from, last = next.j + 1 == next.s.to;
        const int key0 = (next.s.cut.first + next.j) * kPage, valid = next.s.cut.end - key0;     // places of the page that hold a token
        const int record = next.s.record;
        if (first) {
            const int i0 = next.s.tile * R + g, n_rows = next.s.cut.n_tok * group - next.s.tile * R;
            const bool is0 = g < n_rows, is1 = g + 8 < n_rows;
            const int tok0 = i0 / group, tok1 = (i0 + 8) / group, p0 = next.s.cut.end - next.s.cut.n_tok, h = next.s.column * group;
            const bf16* q0 = q + ((int64_t)(next.s.cut.tok0 + tok0) * G.heads + h + i0 - tok0 * group) * HD + 2 * t;
            const bf16* q1 = q + ((int64_t)(next.s.cut.tok0 + tok1) * G.heads + h + i0 + 8 - tok1 * group) * HD + 2 * t;
            last0 = is0 ? p0 + tok0 : -1, last1 = is1 ? p0 + tok1 : -1;
            upper = n_rows > 8;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                qa[i][0] = is0 ? *reinterpret_cast<const uint32_t*>(q0 + i * 16) : 0u;
                qa[i][1] = is1 ? *reinterpret_cast<const uint32_t*>(q1 + i * 16) : 0u;
                qa[i][2] = is0 ? *reinterpret_cast<const uint32_t*>(q0 + i * 16 + 8) : 0u;
                qa[i][3] = is1 ? *reinterpret_cast<const uint32_t*>(q1 + i * 16 + 8) : 0u;
            }
            m0 = m1 = -INFINITY, l0 = l1 = 0.f;
#pragma unroll
            for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        }
        // the page ahead, before this one is waited for
        if (!last) {
            if (((++next.j - next.s.from) & 31) == 0) know_ids();
        } else {
            begin();
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&sm.k_full, turn, &sm.abort_flag, status, 7));
        if (!ok) break;
        float c[kPage / 8][4];
#pragma unroll
        for (int n = 0; n < kPage / 8; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int n = 0; n < kPage / 8; n += 2) {
                uint32_t kb[4];
                ldsm_x4(kb, k_s + tile_off(n * 8 + (lane >> 4) * 8 + (lane & 7), 2 * i + ((lane >> 3) & 1)));
                mma16816(c[n], qa[i], kb[0], kb[1]);
                mma16816(c[n + 1], qa[i], kb[2], kb[3]);
            }
        if (next.any) copy(0);
        // the rows' maxima, weights and sums
        float x0 = -INFINITY, x1 = -INFINITY;
        const int lim0 = last0 - key0 - 2 * t, lim1 = last1 - key0 - 2 * t;        // places up to them are seen
#pragma unroll
        for (int n = 0; n < kPage / 8; ++n) {
            c[n][0] = 8 * n <= lim0 ? c[n][0] * sl2 : -INFINITY, c[n][1] = 8 * n + 1 <= lim0 ? c[n][1] * sl2 : -INFINITY;
            c[n][2] = 8 * n <= lim1 ? c[n][2] * sl2 : -INFINITY, c[n][3] = 8 * n + 1 <= lim1 ? c[n][3] * sl2 : -INFINITY;
            x0 = fmaxf(x0, fmaxf(c[n][0], c[n][1])), x1 = fmaxf(x1, fmaxf(c[n][2], c[n][3]));
        }
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
        }
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float a0 = weight(m0, n0), a1 = weight(m1, n1), z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
        m0 = n0, m1 = n1;
        l0 *= a0, l1 *= a1;
        uint32_t pa[kPage / 16][4];
#pragma unroll
        for (int n = 0; n < kPage / 8; ++n) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(exp2f(c[n][0] - z0), exp2f(c[n][1] - z0));
            const float2 pf = __bfloat1622float2(p);
            l0 += pf.x + pf.y;
            pa[n / 2][(n & 1) * 2] = *reinterpret_cast<const uint32_t*>(&p);
            pa[n / 2][(n & 1) * 2 + 1] = 0u;
        }
        if (upper) {
#pragma unroll
            for (int n = 0; n < kPage / 8; ++n) {
                const __nv_bfloat162 r = __floats2bfloat162_rn(exp2f(c[n][2] - z1), exp2f(c[n][3] - z1));
                const float2 rf = __bfloat1622float2(r);
                l1 += rf.x + rf.y;
                pa[n / 2][(n & 1) * 2 + 1] = *reinterpret_cast<const uint32_t*>(&r);
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) o[i][0] *= a0, o[i][1] *= a0, o[i][2] *= a1, o[i][3] *= a1;
        ok = __all_sync(0xffffffffu, mbar_wait(&sm.v_full, turn, &sm.abort_flag, status, 7));
        if (!ok) break;
#pragma unroll
        for (int ks = 0; ks < kPage / 16; ++ks)
#pragma unroll
            for (int i = 0; i < NT; i += 2) {
                uint32_t vb[4];
                ldsm_x4_trans(vb, v_s + tile_off(ks * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), i + (lane >> 4)));
                if (valid < kPage) {                                   // places without a token may hold anything: zeros
                    const int left = valid - ks * 16 - 2 * t;
                    const uint32_t f0 = left >= 2 ? 0xffffffffu : (left == 1 ? 0xffffu : 0u), f1 = left >= 10 ? 0xffffffffu : (left == 9 ? 0xffffu : 0u);
                    vb[0] &= f0, vb[1] &= f1, vb[2] &= f0, vb[3] &= f1;
                }
                mma16816(o[i], pa[ks], vb[0], vb[1]);
                mma16816(o[i + 1], pa[ks], vb[2], vb[3]);
            }
        if (next.any) copy(1);
        if (last) {
            float* rec = records + (int64_t)record * REC;
            float s0 = l0, s1 = l1;
#pragma unroll
            for (int d = 1; d <= 2; d <<= 1) {
                s0 += __shfl_xor_sync(0xffffffffu, s0, d);
                s1 += __shfl_xor_sync(0xffffffffu, s1, d);
            }
            if (t == 0) {
                *reinterpret_cast<float2*>(rec + R * HD + 2 * g) = make_float2(m0, s0);
                *reinterpret_cast<float2*>(rec + R * HD + 2 * (g + 8)) = make_float2(m1, s1);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                const int c0 = j * 8 + 2 * t;
                if (last0 >= 0) *reinterpret_cast<float2*>(rec + ((c0 >> 2) * R + g) * 4 + (c0 & 3)) = make_float2(o[j][0], o[j][1]);
                if (last1 >= 0) *reinterpret_cast<float2*>(rec + ((c0 >> 2) * R + g + 8) * 4 + (c0 & 3)) = make_float2(o[j][2], o[j][3]);
            }
        }
    }
    if (blockIdx.x == 0) {
        pdl_wait();
        Walk<OwnParts>(parts, gridDim.x, plan);
        clear_unfit(parts, out, G.heads * HD, status);
    }
    pdl_wait();                                        // (whoever waits for this kernel waits for the one before it too)
    if (sm.abort_flag) {
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) __nanosleep(1000);       // copies in flight land before the block leaves
    }
}

}  // namespace own

int launch_own(const void* q, const void* kv, int64_t kv_pages, void* out, const Groups& G, bool after_shared, int blocks, float scale, int* plan,
               float* records, int* status, cudaStream_t s) {
    using namespace own;
    CUtensorMap kv_map;
    if (int e = make_bf16_map(&kv_map, kv, kv_pages * 2 * G.kv_heads * kPage, HD, kPage, "attention (shared prefix)")) return e;
    static bool raised = false;
    if (!raised) {
        WICK_CUDA(cudaFuncSetAttribute(attn_shared_own_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
        raised = true;
    }
    WICK_CUDA(launch(attn_shared_own_kernel, dim3(blocks), dim3(32), (size_t)SMEM_BYTES, s, kv_map, (const bf16*)q, kv_pages, (bf16*)out, G,
                     (int)after_shared, scale, plan, records, status));
    return check_launch("attn_shared_own");
}

}  // namespace shared_prefix
}  // namespace wick
