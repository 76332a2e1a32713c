// A step's page tables, positions and slots, built on the device from the sequences' lengths.
//
// Sequence b holds start_b positions on held_b = ceil(start_b / 64) pages and gets q_b more; need_b = ceil((start_b + q_b) / 64) -
// held_b pages come from the list of free ones, sequence after sequence:
//   page of its column j:  tables[source][j]                     j < held_b      (source: its own record, or its parent's)
//                          free[head + sum_{b' < b} need_b' + j - held_b]        j < held_b + need_b
//                          0 (the reserved page)                  beyond, and beyond the list's end, which is reported
// and for its token i, at position p = start_b + i: slot = page of column p / 64, times 64, plus p % 64.
//
// Forks read what their parents held BEFORE the call, whatever becomes of the parents in it (two sequences may change places): a call with
// parents first makes the rows from the tables as they are, and writes them into the tables in a second launch.  A fork begins on a page of its
// own (start_b a multiple of 64): in the middle of one, it and its parent would write to the same places.
//
// Every block makes the sums over all sequences for itself (a few thousand numbers from the L2 cache; a launch for them, or blocks that wait
// for one another, would cost more than that), then a warp fills a sequence's row, a thread a token.  Record 0 is the padding's: it gets no
// pages.
// Bound by that chain, and in a large call by its rows, a warp each, whose reads and writes wait for one another: 48 sequences of a token each
// 3.3 to 3.7 us (with parents, and so a second launch, 4.2), 700 with 300 forks and up to 400 tokens each (5 MB written) 10.3.
#include "common.cuh"
#include "packed.cuh"

namespace wick {

constexpr int TT = 256;
constexpr int MAX_TABLE_SEQS = 8192;

struct Tables {
    const int *start, *q_len, *slots, *parent;
    int* tables;                                   // [n_slots, table_width]
    const int *free_pages, *free_head;
    int *page_table, *cu_seqlens, *kv_len, *positions, *seq_of_token, *head_out;
    int64_t* slot_map;
    int n_seqs, n_slots, table_width, width, n_free, n_tokens;

    // The record of sequence b; -1 (reported, no pages): outside the tables, a parent outside them, a fork that begins inside a page.
    __device__ __forceinline__ int slot_of(int b) const {
        const int s = slots[b], p = parent ? parent[b] : -1;
        return s != 0 && (s < 0 || s >= n_slots || p >= n_slots || (p >= 0 && p != s && start[b] % kPage != 0)) ? -1 : s;
    }
    __device__ __forceinline__ int source_of(int b, int slot) const {
        const int p = parent ? parent[b] : -1;
        return p >= 0 && p < n_slots ? p : max(slot, 0);
    }
};

// The rows that step_tables_kernel has made, into the tables: a warp has COLUMNS columns of a sequence, a lane four, read before one is written.
constexpr int COLUMNS = 128;
__global__ void __launch_bounds__(TT) store_tables_kernel(const Tables a, int pieces) {
    const int at = ((int)blockIdx.x * TT + (int)threadIdx.x) >> 5, b = at / pieces;
    int slot = 0, from = 0, to = 0;
    if (b < a.n_seqs) {                            // (what the call was given may be read before the wait: the kernel before has waited for it)
        const int start = max(a.start[b], 0);
        slot = a.slot_of(b);
        if (a.source_of(b, slot) == slot) from = (start + kPage - 1) / kPage;
        to = min((start + max(a.q_len[b], 0) + kPage - 1) / kPage, min(a.width, a.table_width));
    }
    pdl_wait();                                    // (no early start of the next kernel, as below)
    if (slot <= 0) return;
    const int* row = a.page_table + (int64_t)b * a.width;
    const int j0 = (at - b * pieces) * COLUMNS + (int)(threadIdx.x & 31);
    int page[COLUMNS / 32];
#pragma unroll
    for (int k = 0; k < COLUMNS / 32; ++k) page[k] = j0 + 32 * k < to ? row[j0 + 32 * k] : 0;
#pragma unroll
    for (int k = 0; k < COLUMNS / 32; ++k)
        if (j0 + 32 * k >= from && j0 + 32 * k < to) a.tables[(int64_t)slot * a.table_width + j0 + 32 * k] = page[k];
}

__global__ void __launch_bounds__(TT) step_tables_kernel(const Tables a, int* status) {
    extern __shared__ int sums[];
    int* cum_q = sums;                             // tokens of the sequences before each one
    int* cum_n = sums + a.n_seqs + 1;              // pages that they need
    __shared__ int warp_q[TT / 32], warp_n[TT / 32];
    pdl_wait();
    if (a.parent) pdl_trigger();                   // (store_tables_kernel; no other kernel starts early: kernels of a step read these fields before they wait)
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, B = a.n_seqs;
    auto held_of = [&](int b) { return (max(a.start[b], 0) + kPage - 1) / kPage; };
    int base_q = 0, base_n = 0;
    for (int s0 = 0; s0 < B; s0 += TT) {
        const int b = s0 + tid;
        int q = 0, n = 0;
        if (b < B) {
            q = max(a.q_len[b], 0);
            if (a.slot_of(b) > 0) n = (max(a.start[b], 0) + q + kPage - 1) / kPage - held_of(b);
        }
        int uq = q, un = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int tq = __shfl_up_sync(0xffffffffu, uq, o), tn = __shfl_up_sync(0xffffffffu, un, o);
            if (lane >= o) uq += tq, un += tn;
        }
        if (lane == 31) warp_q[warp] = uq, warp_n[warp] = un;
        __syncthreads();
        int wq = 0, wn = 0, all_q = 0, all_n = 0;
#pragma unroll
        for (int w = 0; w < TT / 32; ++w) {
            if (w < warp) wq += warp_q[w], wn += warp_n[w];
            all_q += warp_q[w], all_n += warp_n[w];
        }
        if (b < B) cum_q[b] = base_q + wq + uq - q, cum_n[b] = base_n + wn + un - n;
        base_q += all_q, base_n += all_n;
        __syncthreads();
    }
    if (tid == 0) cum_q[B] = base_q, cum_n[B] = base_n;
    __syncthreads();
    const int head = *a.free_head;

    // What column j of sequence b holds.
    auto page_at = [&](int src, int slot, int held, int total, int first, int j) -> int {
        if (slot <= 0 || j >= total) return 0;
        if (j < held) return j < a.table_width ? a.tables[(int64_t)src * a.table_width + j] : 0;
        const int at = first + j - held;
        return at >= 0 && at < a.n_free ? a.free_pages[at] : 0;
    };

    const int gt = (int)blockIdx.x * TT + tid, step = (int)gridDim.x * TT;
    for (int b = gt; b <= B; b += step) {
        a.cu_seqlens[b] = cum_q[b];
        if (b < B) a.kv_len[b] = max(a.start[b], 0) + cum_q[b + 1] - cum_q[b];
    }
    if (gt == 0) {
        *a.head_out = head + cum_n[B];
        if ((head < 0 || head + cum_n[B] > a.n_free) && cum_n[B] > 0) atomicCAS(status, 0, 12);
        if (cum_q[B] > a.n_tokens) atomicCAS(status, 0, 14);
    }
    for (int b = gt >> 5; b < B; b += step >> 5) {
        const int slot = a.slot_of(b), held = held_of(b), total = held + cum_n[b + 1] - cum_n[b], first = head + cum_n[b], src = a.source_of(b, slot);
        if (lane == 0 && (slot < 0 || (slot > 0 && total > min(a.width, a.table_width)))) atomicCAS(status, 0, 13);
        for (int j = lane; j < a.width; j += 32) {
            const int page = page_at(src, slot, held, total, first, j);
            a.page_table[(int64_t)b * a.width + j] = page;
            if (!a.parent && slot > 0 && j >= held && j < total && j < a.table_width) a.tables[(int64_t)slot * a.table_width + j] = page;
        }
    }
    for (int t = gt; t < a.n_tokens; t += step) {
        int pos = 0, seq = 0;
        int64_t at = -1;
        if (t < cum_q[B]) {
            int lo = 0, hi = B;                    // cum_q[lo] <= t < cum_q[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (cum_q[mid] <= t) lo = mid;
                else hi = mid;
            }
            seq = lo;
            pos = max(a.start[seq], 0) + t - cum_q[seq];
            const int slot = a.slot_of(seq), held = held_of(seq), total = held + cum_n[seq + 1] - cum_n[seq];
            at = (int64_t)page_at(a.source_of(seq, slot), slot, held, total, head + cum_n[seq], pos / kPage) * kPage + pos % kPage;
        }
        a.positions[t] = pos;
        a.seq_of_token[t] = seq;
        a.slot_map[t] = at;
    }
}

}  // namespace wick

using namespace wick;

// Arrays as in struct Tables.  status: 12 the list of free pages is too short, 13 a record, a parent or a length outside the tables, or a fork
// that begins inside a page, 14 more tokens than places.  Two launches with parents, one without.
WICK_API int wick_step_tables(const int* start, const int* q_len, const int* slots, const int* parent, int n_seqs, int* tables, int n_slots,
                              int table_width, const int* free_pages, int n_free, const int* free_head, int* page_table, int width,
                              int* cu_seqlens, int* kv_len, int* positions, int* seq_of_token, void* slot_map, int n_tokens, int* head_out,
                              int* status, void* s) {
    WICK_REQUIRE(n_seqs >= 1 && n_seqs <= MAX_TABLE_SEQS, "step_tables: %d sequences (1 to %d)", n_seqs, MAX_TABLE_SEQS);
    WICK_REQUIRE(n_slots >= 1 && table_width >= 1 && width >= 1 && n_free >= 0 && n_tokens >= 0, "step_tables: bad sizes");
    Tables a = {start, q_len, slots, parent, tables, free_pages, free_head, page_table, cu_seqlens, kv_len, positions, seq_of_token, head_out,
                (int64_t*)slot_map, n_seqs, n_slots, table_width, width, n_free, n_tokens};
    const int pieces = ceil_div(min(width, table_width), COLUMNS);
    WICK_REQUIRE((int64_t)n_seqs * pieces <= INT32_MAX / 32, "step_tables: %d sequences of %d columns", n_seqs, width);
    const int blocks = max(1, min(2 * sm_count(), max(ceil_div((int64_t)n_seqs, TT / 32), ceil_div(n_tokens, TT))));
    const size_t smem = (size_t)(2 * (n_seqs + 1)) * sizeof(int);
    static bool raised = false;
    if (!raised) {
        WICK_CUDA(cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(2 * (MAX_TABLE_SEQS + 1) * sizeof(int))));
        raised = true;
    }
    WICK_CUDA(launch(step_tables_kernel, dim3(blocks), dim3(TT), smem, (cudaStream_t)s, a, status));
    if (int e = check_launch("step_tables")) return e;
    if (!parent) return 0;
    WICK_CUDA(launch(store_tables_kernel, dim3(ceil_div((int64_t)n_seqs * pieces, TT / 32)), dim3(TT), 0, (cudaStream_t)s, a, pieces));
    return check_launch("store_tables");
}
WICK_PACKED(wick_step_tables)
