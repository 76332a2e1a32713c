// The own keys of each sequence behind its group's shared prefix: bfloat16, head sizes 64 and 128.
//
// Two persistent thread blocks an SM.  The pages of all items (a sequence's 16 rows of one key head) are dealt to them in equal runs
// (attn_shared.cuh); a producer warp copies a run's pages (TMA, 128-byte swizzle), and an item's query rows with its first page, into a
// ring, from one item into the next, so that copies never stop for the end of an item: the work is bound by the bytes of the
// keys and values.  Four warps compute, a page at a time:
//   * a warp has the scores of the 16 rows with 16 of the page's keys (mma.sync); the warps agree on the rows' maxima;
//   * weights go to shared memory as bfloat16 (their sum is taken of the rounded ones), and each warp multiplies all of the page's
//     with a quarter of the value columns: the sums of a row stay in registers, spread over the warps, and are never joined among them.
// Every item leaves a record per run that has a part of it.  (Joined in place by the thread block that finished an item, a chain of five
// dependent reads an item held up the ring: 64 sequences of 370 own positions behind 8,192 shared ones, 32 heads over 8: 120 us.)
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
constexpr int W = 4, THREADS = (W + 1) * 32;
constexpr int PANELS = HD / 64, PANEL_BYTES = kPage * 128, TILE_BYTES = PANELS * PANEL_BYTES;   // a page of keys, or of values
constexpr int STAGES = HD == 128 ? 3 : 5;              // pages of keys and values in flight
constexpr int KS = HD / 16, NT = HD / 32;              // steps of q . k; tiles of eight value columns a warp has
constexpr int REC = R * (HD + 2);

// What a page in the ring is.
struct Page {
    int first, last;                                   // of its item's part
    int key0, end;                                     // its first position, the end of the sequence's
    int row0, n_rows, n_tok;                           // the item's first row (of the sequence's in this key head), its rows; the sequence's new tokens
    int record;
};
struct Smem {
    uint8_t kv[STAGES][2][TILE_BYTES];
    bf16 q[STAGES][R][HD];
    bf16 p[2][R][kPage];                               // (16-byte chunk c of row r at place c ^ (r & 7))
    float mx[2][W][R], l[W][R];
    Page page[STAGES];
    uint64_t full[STAGES], empty[STAGES];
    int abort_flag;
};
constexpr int SMEM_BYTES = (int)sizeof(Smem);
static_assert(2 * (SMEM_BYTES + 1024) <= 228 * 1024, "two blocks an SM");

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
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
// The four warps that compute meet; any: whether some thread says so (every thread gets the same answer).
__device__ __forceinline__ void sync_warps() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool sync_any(bool mine) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(r) : "r"((uint32_t)mine) : "memory");
    return r != 0;
}

__global__ void __launch_bounds__(THREADS, 2)
attn_shared_own_kernel(const __grid_constant__ CUtensorMap kv_map, const bf16* q, int64_t kv_pages, bf16* __restrict__ out, const Groups G, int after_shared,
                       float scale, int* plan, float* records, int* status) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem& sm = *reinterpret_cast<Smem*>(smem_raw);
    volatile int* abort_flag = &sm.abort_flag;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = G.heads / G.kv_heads;
    if (tid == 0) {
        sm.abort_flag = 0;
        for (int i = 0; i < STAGES; ++i) mbar_init(&sm.full[i], 1), mbar_init(&sm.empty[i], W);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // (With a shared part the kernel before this one is the one that computes it, and has waited for q and the cache.)
    if (!after_shared) pdl_wait();
    pdl_trigger();
    __syncthreads();
    int stage = 0, turn = 0;

    if (warp == W) {
        // ---------------- producer ----------------
        const OwnParts parts{G, R};
        const bool one = elect_one();
        bool ok = (smem_u32(smem_raw) & 1023) == 0;   // (always: the block's dynamic shared memory is all there is)
        if (!ok && one) atomicCAS(status, 0, 7);
        Walk<OwnParts> walk(parts, gridDim.x, nullptr);
        Segment s;
        auto room = [&]() { return turn == 0 || __all_sync(0xffffffffu, mbar_wait(&sm.empty[stage], (turn - 1) & 1, abort_flag, status, 7)); };
#pragma unroll 1
        while (ok && walk.segment(s)) {
            const int* table = G.page_table + (int64_t)s.cut.seq * G.table_width + s.cut.first;
            const int row0 = s.tile * R, n_rows = min(R, s.cut.n_tok * group - row0);
            int ids = 0;
#pragma unroll 1
            for (int j = s.from; j < s.to; ++j) {
                if (((j - s.from) & 31) == 0) {                        // a lane holds one of 32 page numbers
                    ids = j + lane < s.to ? table[j + lane] : 0;
                    if (ids < 0 || ids >= kv_pages) {
                        atomicCAS(status, 0, 10);
                        ids = 0;
                    }
                }
                const int page = __shfl_sync(0xffffffffu, ids, (j - s.from) & 31);
                ok = room();
                if (!ok) break;
                if (one) {
                    const bool first = j == s.from;
                    sm.page[stage] = Page{first, j + 1 == s.to, (s.cut.first + j) * kPage, s.cut.end, row0, n_rows, s.cut.n_tok, s.record};
                    mbar_expect_tx(&sm.full[stage], 2 * TILE_BYTES + (first ? n_rows * HD * 2 : 0));
#pragma unroll
                    for (int v = 0; v < 2; ++v)
                        for (int pn = 0; pn < PANELS; ++pn)
                            tma_load_2d(&kv_map, &sm.full[stage], sm.kv[stage][v] + pn * PANEL_BYTES, pn * 64, ((page * 2 + v) * G.kv_heads + s.column) * kPage);
                    if (first) {
                        for (int r = 0; r < n_rows;) {                 // rows of one token lie side by side
                            const int tok = (row0 + r) / group, h = row0 + r - tok * group, n = min(group - h, n_rows - r);
                            bulk_load(&sm.q[stage][r][0], q + ((int64_t)(s.cut.tok0 + tok) * G.heads + s.column * group + h) * HD, (uint32_t)(n * HD * 2), &sm.full[stage]);
                            r += n;
                        }
                    }
                }
                if (++stage == STAGES) stage = 0, ++turn;
                __syncwarp();
            }
        }
        if (ok && room() && one) {                                     // the end of the run
            sm.page[stage].record = -1;
            mbar_arrive(&sm.full[stage]);
        }
        if (blockIdx.x == 0) {
            pdl_wait();
            Walk<OwnParts>(parts, gridDim.x, plan);
            clear_unfit(parts, out, G.heads * HD, status);
        }
    } else {
        // ---------------- compute ----------------
        const int g = lane >> 2, t = lane & 3, col = warp * (HD / 4) + 2 * t;
        const float sl2 = scale * LOG2E;
        uint32_t qa[KS][4];
        float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        int last0 = -1, last1 = -1;                                    // the last position that rows g and g + 8 see
#pragma unroll 1
        for (int set = 0;; set ^= 1) {                                 // of maxima and weights
            const bool here = __all_sync(0xffffffffu, mbar_wait(&sm.full[stage], turn & 1, abort_flag, status, 7));
            const Page& pg = sm.page[stage];
            if (!here || pg.record < 0) {                              // a warp that gave up waiting, or the end: all leave together
                sync_any(true);
                break;
            }
            const uint32_t k_s = smem_u32(sm.kv[stage][0]), v_s = smem_u32(sm.kv[stage][1]);
            const int key0 = pg.key0, valid = pg.end - key0;           // places of the page that hold a token
            if (pg.first) {
                const uint32_t q_s = smem_u32(&sm.q[stage][0][0]);
#pragma unroll
                for (int i = 0; i < KS; ++i) ldsm_x4(qa[i], q_s + (uint32_t)((((lane >> 3) & 1) * 8 + (lane & 7)) * HD + i * 16 + (lane >> 4) * 8) * 2);
                const int i0 = pg.row0 + g, p0 = pg.end - pg.n_tok;
                last0 = g < pg.n_rows ? p0 + i0 / group : -1, last1 = g + 8 < pg.n_rows ? p0 + (i0 + 8) / group : -1;
                m0 = m1 = -INFINITY, l0 = l1 = 0.f;
#pragma unroll
                for (int j = 0; j < NT; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
            }
            float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                uint32_t kb[4];
                ldsm_x4(kb, k_s + tile_off(warp * 16 + (lane >> 4) * 8 + (lane & 7), 2 * i + ((lane >> 3) & 1)));
                mma16816(c[0], qa[i], kb[0], kb[1]);
                mma16816(c[1], qa[i], kb[2], kb[3]);
            }
            const int mine = key0 + warp * 16 + 2 * t, lim0 = last0 - mine, lim1 = last1 - mine;     // places up to them are seen
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
            if (t == 0) sm.mx[set][warp][g] = x0, sm.mx[set][warp][g + 8] = x1;
            if (sync_any(false)) break;
            float n0 = m0, n1 = m1;
#pragma unroll
            for (int w = 0; w < W; ++w) n0 = fmaxf(n0, sm.mx[set][w][g]), n1 = fmaxf(n1, sm.mx[set][w][g + 8]);
            const float a0 = weight(m0, n0), a1 = weight(m1, n1), z0 = n0 == -INFINITY ? 0.f : n0, z1 = n1 == -INFINITY ? 0.f : n1;
            m0 = n0, m1 = n1;
            l0 *= a0, l1 *= a1;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(exp2f(c[h][0] - z0), exp2f(c[h][1] - z0));
                const __nv_bfloat162 r = __floats2bfloat162_rn(exp2f(c[h][2] - z1), exp2f(c[h][3] - z1));
                const float2 pf = __bfloat1622float2(p), rf = __bfloat1622float2(r);
                l0 += pf.x + pf.y, l1 += rf.x + rf.y;
                const int at = ((warp * 2 + h) ^ g) * 8 + 2 * t;       // (rows g and g + 8 have their chunks in the same places)
                *reinterpret_cast<__nv_bfloat162*>(&sm.p[set][g][at]) = p;
                *reinterpret_cast<__nv_bfloat162*>(&sm.p[set][g + 8][at]) = r;
            }
            sync_warps();
#pragma unroll
            for (int i = 0; i < NT; ++i) o[i][0] *= a0, o[i][1] *= a0, o[i][2] *= a1, o[i][3] *= a1;
            const uint32_t p_s = smem_u32(&sm.p[set][0][0]);
#pragma unroll
            for (int ks = 0; ks < kPage / 16; ++ks) {
                uint32_t pa[4];
                const int pr = ((lane >> 3) & 1) * 8 + (lane & 7);
                ldsm_x4(pa, p_s + (uint32_t)(pr * kPage + ((ks * 2 + (lane >> 4)) ^ (pr & 7)) * 8) * 2);
#pragma unroll
                for (int i = 0; i < NT; i += 2) {
                    uint32_t vb[4];
                    ldsm_x4_trans(vb, v_s + tile_off(ks * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), warp * (HD / 32) + i + (lane >> 4)));
                    if (valid < kPage) {                               // the others may hold anything: zeros
                        const int left = valid - ks * 16 - 2 * t;
                        const uint32_t f0 = left >= 2 ? 0xffffffffu : (left == 1 ? 0xffffu : 0u), f1 = left >= 10 ? 0xffffffffu : (left == 9 ? 0xffffu : 0u);
                        vb[0] &= f0, vb[1] &= f1, vb[2] &= f0, vb[3] &= f1;
                    }
                    mma16816(o[i], pa, vb[0], vb[1]);
                    mma16816(o[i + 1], pa, vb[2], vb[3]);
                }
            }
            if (pg.last) {
                float* rec = records + (int64_t)pg.record * REC;
                const bool is0 = last0 >= 0, is1 = last1 >= 0;
                float s0 = l0, s1 = l1;
#pragma unroll
                for (int d = 1; d <= 2; d <<= 1) {
                    s0 += __shfl_xor_sync(0xffffffffu, s0, d);
                    s1 += __shfl_xor_sync(0xffffffffu, s1, d);
                }
                if (t == 0) sm.l[warp][g] = s0, sm.l[warp][g + 8] = s1;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int cc = col + 8 * j;
                    if (is0) *reinterpret_cast<float2*>(rec + ((cc >> 2) * R + g) * 4 + (cc & 3)) = make_float2(o[j][0], o[j][1]);
                    if (is1) *reinterpret_cast<float2*>(rec + ((cc >> 2) * R + g + 8) * 4 + (cc & 3)) = make_float2(o[j][2], o[j][3]);
                }
                sync_warps();
                if (warp == 0 && t == 0) {                             // (the sums' next use lies behind two further barriers)
                    s0 = s1 = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w) s0 += sm.l[w][g], s1 += sm.l[w][g + 8];
                    *reinterpret_cast<float2*>(rec + R * HD + 2 * g) = make_float2(m0, s0);
                    *reinterpret_cast<float2*>(rec + R * HD + 2 * (g + 8)) = make_float2(m1, s1);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[stage]);
            if (++stage == STAGES) stage = 0, ++turn;
        }
    }
    pdl_wait();                                                        // (whoever waits for this kernel waits for the one before it too)
    __syncthreads();
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
    WICK_CUDA(launch(attn_shared_own_kernel, dim3(blocks), dim3(THREADS), (size_t)SMEM_BYTES, s, kv_map, (const bf16*)q, kv_pages, (bf16*)out, G,
                     (int)after_shared, scale, plan, records, status));
    return check_launch("attn_shared_own");
}

}  // namespace shared_prefix
}  // namespace wick
