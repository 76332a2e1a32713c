// The own keys of each sequence behind its group's shared prefix, and shared keys that are too few for a kernel of their own: bfloat16,
// head sizes 64 and 128.
//
// A thread block is ONE warp that feeds itself; six of them (head size 64: twelve) fill an SM's shared memory.  The pages of all items (a
// sequence's 8 rows of one key head) are dealt to the warps in equal runs (attn_shared.cuh).  A warp has room for one page of keys and
// one of values: the next page's keys are copied (TMA, 128-byte swizzle) while it turns scores into weights and multiplies the values,
// the next values while it multiplies the next keys, from one item into the next.  Keys and value columns are on the 16-row side of mma.sync, the
// rows on the 8-wide one (with rows on the 16-row side a page took twice the instructions, of which a token of 4 or 8 heads needs half);
// weights are turned into the second product's operand by movmatrix, rounded to bfloat16; their sum is taken of the rounded ones.  Every item
// leaves a record per run that has a part of it.
// Bound by the bytes of the keys and values: with all SMs a page takes a warp 4 us, 7 TB/s, behind a start of 3 us (the description, then the
// first page); on the 65 SMs that the shared part leaves by one warp's chain, copy - scores - weights - values, 2.2 us a page.  64 sequences of
// 370 own positions, 8 key heads of 128 (97 MB): 23 us there; 4 sequences behind 512 positions, both parts: 5.6 us.
// (Measured and left: blocks of four or eight warps that shared a page met three times a page, 2,000 clocks of latency that two blocks an SM
// could not hide, 28 us; half a page a turn and twice the warps, 24 us in place of 26, but twice the records: steps of few keys lost 10 to
// 25 %.)
// The kernel of the shared part runs before this one, which starts under its last blocks.  A page's place is read by the warp that has the next
// page copied there, before; only where zeros were written there does a fence stand between.
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
constexpr int KS = HD / 16, MT = kPage / 16;           // steps of q . k, and tiles of 16 value columns; tiles of 16 keys
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

// An 8 x 8 matrix of 16-bit numbers, a row in four lanes: the transposed matrix in the same layout.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

// The page after the one at hand: the run's part it lies in, its place in it.  A lane holds one of 32 page numbers.
struct Ahead {
    Segment s;
    int j, ids;
    bool any;
};

__global__ void __launch_bounds__(32)
attn_shared_own_kernel(const __grid_constant__ CUtensorMap kv_map, const bf16* q, int64_t kv_pages, bf16* __restrict__ out, const Groups G, int groups, int after_shared,
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
    // (The description lies ready before the step's kernels start.)
    const OwnParts parts{G, R, groups};
    Walk walk(parts, gridDim.x, nullptr);
    const uint64_t policy = read_once_policy();        // (once for 8 rows: the records, which are read again, are to stay)
    Ahead next = {};
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
            mbar_expect_tx(bar, TILE_BYTES);
            for (int pn = 0; pn < PANELS; ++pn)
                tma_load_2d(&kv_map, bar, (v ? sm.v : sm.k) + pn * PANEL_BYTES, pn * 64, ((page * 2 + v) * G.kv_heads + next.s.column) * kPage, policy);
        }
        __syncwarp();
    };
    bool ok = (smem_u32(smem_raw) & 1023) == 0;        // (always: the block's dynamic shared memory is all there is)
    if (!ok && lane == 0) atomicCAS(status, 0, 7);
    next.any = false;
    if (ok) begin();
    // (With a shared part the kernel before this one is the one that computes it, and has waited for q and the cache.)
    if (!after_shared) pdl_wait();
    pdl_trigger();
    if (next.any) copy(0), copy(1);

    uint32_t qb[KS][2];                                // lane: row g
    float o[KS][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;        // columns 16 i + g and + 8 of rows 2 t and 2 t + 1
    int last0 = -1, last1 = -1;                        // the last position that rows 2 t and 2 t + 1 see
    const uint32_t k_s = smem_u32(sm.k), v_s = smem_u32(sm.v);
#pragma unroll 1
    for (int turn = 0; ok && next.any; turn ^= 1) {
        const bool first = next.j == next.s.from, last = next.j + 1 == next.s.to;
        const int key0 = (next.s.cut.first + next.j) * kPage, valid = next.s.cut.end - key0;     // places of the page that hold a token
        const int record = next.s.record;
        if (first) {
            const int row0 = next.s.tile * R, n_rows = next.s.cut.n_tok * group - row0;
            const int tok = (row0 + g) / group;
            const bf16* q0 = q + ((int64_t)(next.s.cut.tok0 + tok) * G.heads + next.s.column * group + row0 + g - tok * group) * HD + 2 * t;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                qb[i][0] = g < n_rows ? *reinterpret_cast<const uint32_t*>(q0 + i * 16) : 0u;
                qb[i][1] = g < n_rows ? *reinterpret_cast<const uint32_t*>(q0 + i * 16 + 8) : 0u;
            }
            last0 = 2 * t < n_rows ? next.s.last((row0 + 2 * t) / group) : -1, last1 = 2 * t + 1 < n_rows ? next.s.last((row0 + 2 * t + 1) / group) : -1;
            m0 = m1 = -INFINITY, l0 = l1 = 0.f;
#pragma unroll
            for (int i = 0; i < KS; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        }
        // the page ahead, before this one is waited for
        if (!last) {
            if (((++next.j - next.s.from) & 31) == 0) know_ids();
        } else {
            begin();
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&sm.k_full, turn, &sm.abort_flag, status, 7));
        if (!ok) break;
        float c[MT][4];                                // keys 16 m + g and + 8, rows 2 t and 2 t + 1
#pragma unroll
        for (int m = 0; m < MT; ++m) c[m][0] = c[m][1] = c[m][2] = c[m][3] = 0.f;
#pragma unroll
        for (int i = 0; i < KS; ++i)
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                uint32_t ka[4];
                ldsm_x4(ka, k_s + tile_off(m * 16 + (lane & 15), 2 * i + (lane >> 4)));
                mma16816(c[m], ka, qb[i][0], qb[i][1]);
            }
        if (next.any) copy(0);
        // the rows' maxima, weights and sums
        float x0 = -INFINITY, x1 = -INFINITY;
        const int lim0 = last0 - key0 - g, lim1 = last1 - key0 - g;    // places up to them are seen
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            c[m][0] = 16 * m <= lim0 ? c[m][0] * sl2 : -INFINITY, c[m][1] = 16 * m <= lim1 ? c[m][1] * sl2 : -INFINITY;
            c[m][2] = 16 * m + 8 <= lim0 ? c[m][2] * sl2 : -INFINITY, c[m][3] = 16 * m + 8 <= lim1 ? c[m][3] * sl2 : -INFINITY;
            x0 = fmaxf(x0, fmaxf(c[m][0], c[m][2])), x1 = fmaxf(x1, fmaxf(c[m][1], c[m][3]));
        }
#pragma unroll
        for (int d = 4; d <= 16; d <<= 1) {
            x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, d));
            x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, d));
        }
        const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
        const float a0 = weight(m0, n0), a1 = weight(m1, n1), z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
        m0 = n0, m1 = n1;
        l0 *= a0, l1 *= a1;
        uint32_t pb[MT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(exp2f(c[m][2 * h] - z0), exp2f(c[m][2 * h + 1] - z1));
                const float2 pf = __bfloat1622float2(p);
                l0 += pf.x, l1 += pf.y;
                pb[m][h] = transpose8x8(*reinterpret_cast<const uint32_t*>(&p));
            }
#pragma unroll
        for (int i = 0; i < KS; ++i) o[i][0] *= a0, o[i][1] *= a1, o[i][2] *= a0, o[i][3] *= a1;
        ok = __all_sync(0xffffffffu, mbar_wait(&sm.v_full, turn, &sm.abort_flag, status, 7));
        if (!ok) break;
        if (valid < kPage) {                           // places without a token may hold anything: zeros
            for (int i = max(valid, 0) * (HD / 8) + lane; i < kPage * (HD / 8); i += 32)
                *reinterpret_cast<uint4*>(sm.v + tile_off(i / (HD / 8), i % (HD / 8))) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");       // (before the next copy writes there)
            __syncwarp();
        }
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t va[4];
                ldsm_x4_trans(va, v_s + tile_off(m * 16 + (lane >> 4) * 8 + (lane & 7), 2 * i + ((lane >> 3) & 1)));
                mma16816(o[i], va, pb[m][0], pb[m][1]);
            }
        if (next.any) copy(1);
        if (last) {
            float* rec = records + (int64_t)record * REC;
            float s0 = l0, s1 = l1;
#pragma unroll
            for (int d = 4; d <= 16; d <<= 1) {
                s0 += __shfl_xor_sync(0xffffffffu, s0, d);
                s1 += __shfl_xor_sync(0xffffffffu, s1, d);
            }
            if (g == 0) *reinterpret_cast<float4*>(rec + R * HD + 4 * t) = make_float4(m0, s0, m1, s1);
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = 16 * i + 8 * h + g;
                    float* at = rec + ((col >> 2) * R + 2 * t) * 4 + (col & 3);
                    if (last0 >= 0) at[0] = o[i][2 * h];
                    if (last1 >= 0) at[4] = o[i][2 * h + 1];
                }
        }
    }
    if (blockIdx.x == 0) {
        pdl_wait();
        const Walk all(parts, gridDim.x, plan);
        clear_unfit(parts, out, G.heads * HD, all.wrong, status);
    }
    pdl_wait();                                        // (whoever waits for this kernel waits for the one before it too)
    if (sm.abort_flag) {
        const uint64_t t0 = global_ns();
        while (global_ns() - t0 < 2000000ull) __nanosleep(1000);       // copies in flight land before the block leaves
    }
}

}  // namespace own

int launch_own(const void* q, const void* kv, int64_t kv_pages, void* out, const Groups& G, int groups, bool after_shared, int blocks, float scale, int* plan,
               float* records, int* status, cudaStream_t s) {
    using namespace own;
    WICK_REQUIRE(kv_pages * 2 * G.kv_heads * kPage <= INT32_MAX, "attention (shared prefix): a cache of %lld pages is beyond the copies' coordinates", (long long)kv_pages);
    CUtensorMap kv_map;
    if (int e = make_bf16_map(&kv_map, kv, kv_pages * 2 * G.kv_heads * kPage, HD, kPage, "attention (shared prefix)")) return e;
    static bool raised = false;
    if (!raised) {
        WICK_CUDA(cudaFuncSetAttribute(attn_shared_own_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES));
        raised = true;
    }
    WICK_CUDA(launch(attn_shared_own_kernel, dim3(blocks), dim3(32), (size_t)SMEM_BYTES, s, kv_map, (const bf16*)q, kv_pages, (bf16*)out, G,
                     groups, (int)after_shared, scale, plan, records, status));
    return check_launch("attn_shared_own");
}

}  // namespace shared_prefix
}  // namespace wick
