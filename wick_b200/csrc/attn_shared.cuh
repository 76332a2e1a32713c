// Attention of a step's new tokens where groups of sequences share their first pages: what the kernels agree on.
//
// With L_g the positions of group g's shared pages, a row (a token's query head) at position p is
//   y = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q . k_j,  j = 0 .. p
// and the sum splits at L_g: keys below it are the same for all rows of the group, and are read once for as many rows as a tile
// holds; the rest are the sequence's own.  Each part is kept as (m, l, o) = (maximum, sum of weights, weighted sum of values), all
// in float32, and parts are joined by M = max m_i, l = sum l_i 2^(m_i - M), o likewise (scores in units of log2 e).
//
// Shared keys: a tile (or, where a thread block takes two, a pair of neighbouring tiles) is an ITEM.  An item's pages are cut
// into RUNS of equal length, the shortest that leaves no thread block with two (see Runs): what a run costs besides its pages (its
// start and its record) is as much as ten of them.  Own keys (and shared ones, where they are few): a sequence's 16 or 8 rows
// of one key head are an item, whose pages are dealt to the workers in equal contiguous runs, from one item into the next (see Walk).  Either way a record is
// written per run and item, and who has what follows from the description alone: the kernel that joins finds the records by
// arithmetic, in a fixed order.
#pragma once

#include "common.cuh"

namespace wick {
namespace shared_prefix {

constexpr int MAX_GROUPS = 1024;

// The step's description and how the shared part is cut.
struct Groups {
    const int *cu_groups, *pages, *group_of;       // sequences of group g: cu_groups[g] .. ; its shared pages; the group of a sequence
    const int *cu_seqlens, *start, *page_table;
    int n, n_seqs, table_width, max_pages;
    int single;                                    // every sequence brings one token: token i is sequence i's
    int heads, kv_heads;
    int rows;                                      // of a tile
    int gs, per_kv, columns;                       // heads of a tile; tiles of heads to a key head, in all
    int pair;                                      // tiles of an item, at most
};
__device__ __forceinline__ int pages_of(const Groups& G, int g) { return max(0, min(min(G.pages[g], G.max_pages), G.table_width)); }

// Something whose tiles see the same keys: a group and its shared pages, or a sequence and its own.
struct Cut {
    int pages, tok0, n_tok, tiles;
    int seq, first, end;                           // the row of the page table, its first column, the end of the positions
    // A group that ends before it begins.  Scratch has room for groups that are one behind the other; in any other order a sequence could be in
    // many.  Then nothing is computed for groups, which is reported.
    bool wrong;
};
struct SharedParts {
    const Groups& G;
    __device__ __forceinline__ Cut operator()(int g) const {
        Cut c;
        c.pages = pages_of(G, g);
        const int from = G.cu_groups[g], to = G.cu_groups[g + 1];
        const int a = max(0, min(from, G.n_seqs)), b = max(a, min(to, G.n_seqs));
        c.wrong = to < from;
        c.seq = a, c.first = 0;
        c.tok0 = G.single ? a : G.cu_seqlens[a];
        c.n_tok = (G.single ? b : G.cu_seqlens[b]) - c.tok0;
        c.tiles = c.pages > 0 ? (c.n_tok * G.gs + G.rows - 1) / G.rows : 0;
        c.end = c.pages * kPage;
        return c;
    }
};
// What the workers of the own keys' kernel do: the own keys of each sequence (of one that does not fit its group or its page table:
// none), and behind the last sequence, where no other kernel does them, the shared keys of each group.
struct OwnParts {
    const Groups& G;
    int rows;                                      // of a tile
    int groups;                                    // that come behind the sequences
    __device__ __forceinline__ int n() const { return G.n_seqs + groups; }
    __device__ __forceinline__ bool shared(int i) const { return i >= G.n_seqs; }
    __device__ __forceinline__ bool fits(int b, const Cut& c) const {
        const int g = G.group_of[b];
        return g >= 0 && g < G.n && b >= G.cu_groups[g] && b < G.cu_groups[g + 1] && G.start[b] >= c.first * kPage && (c.end + kPage - 1) / kPage <= G.table_width;
    }
    __device__ __forceinline__ Cut operator()(int i) const {
        Cut c;
        if (shared(i)) {
            c = SharedParts{G}(i - G.n_seqs);
        } else {
            const int g = G.group_of[i];
            c.seq = i, c.wrong = false;
            c.tok0 = G.single ? i : G.cu_seqlens[i];
            c.n_tok = G.single ? 1 : G.cu_seqlens[i + 1] - c.tok0;
            c.first = g >= 0 && g < G.n ? pages_of(G, g) : 0;
            c.end = G.start[i] + c.n_tok;
            c.pages = c.n_tok > 0 && fits(i, c) ? (c.end + kPage - 1) / kPage - c.first : 0;
        }
        c.tiles = c.pages > 0 ? (c.n_tok * (G.heads / G.kv_heads) + rows - 1) / rows : 0;
        return c;
    }
};
// By a warp: the sequences that do not fit are reported, and groups in no order (wrong); the sequences' rows are made zero.
template <typename T> __device__ __forceinline__ void clear_unfit(const OwnParts& parts, T* out, int row_numbers, bool wrong, int* status) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < parts.G.n_seqs; b0 += 32) {
        Cut c = Cut{};
        if (b0 + lane < parts.G.n_seqs) c = parts(b0 + lane);
        unsigned bad = __ballot_sync(0xffffffffu, c.n_tok > 0 && c.pages == 0);
        if ((bad || wrong) && lane == 0) atomicCAS(status, 0, 11);
        for (; bad; bad &= bad - 1) {
            const int l = __ffs(bad) - 1;
            const int64_t at = (int64_t)__shfl_sync(0xffffffffu, c.tok0, l) * row_numbers, n = (int64_t)__shfl_sync(0xffffffffu, c.n_tok, l) * row_numbers;
            for (int64_t i = lane; i < n; i += 32) st(out + at + i, 0.f);
        }
    }
}
// Own pages dealt: worker c of S takes the units (pages of an item) from run_start(c) to run_start(c + 1), U / S of them or one more.
struct Deal {
    int U, S, per, more;                           // more: workers that have one more than per
    __device__ __forceinline__ Deal(int units, int workers) : U(units) {
        S = max(1, min(workers, U));
        per = U / S, more = U - per * S;
    }
    __device__ __forceinline__ int run_start(int c) const { return c * per + min(c, more); }
    __device__ __forceinline__ int worker_of(int u) const { return u < more * (per + 1) ? u / (per + 1) : more + (u - more * (per + 1)) / per; }
};

// A run's part of one item: `tiles` tiles from `tile` on, pages from .. to.
struct Segment {
    Cut cut;
    int tile, tiles, column;
    int from, to;
    int record;
    bool shared;                                   // (Walk) a group's keys: every row sees all of them
    // (Walk) the last position that a row of the thing's token `tok` sees
    __device__ __forceinline__ int last(int tok) const { return shared ? cut.end - 1 : cut.end - cut.n_tok + tok; }
};

// ---- shared keys -------------------------------------------------------------------
// The pages of a run of an item of w tiles: `run` for two tiles, twice as many for one (whose pages cost half).
__device__ __forceinline__ int run_pages(const Groups& G, int run, int w) { return run * G.pair / w; }
// Runs of an item of w tiles, of all items of a group.
__device__ __forceinline__ int runs_of_item(const Groups& G, const Cut& c, int run, int w) {
    const int n = run_pages(G, run, w);
    return (c.pages + n - 1) / n;
}
__device__ __forceinline__ int runs_of(const Groups& G, const Cut& c, int run) {
    const int full = c.tiles / G.pair, rest = c.tiles - full * G.pair;
    return G.columns * (full * runs_of_item(G, c, run, G.pair) + (rest ? runs_of_item(G, c, run, rest) : 0));
}
// Where a tile of a group is: its item's first run (of the group's) and number of runs.
struct Place {
    int first, n;
};
__device__ __forceinline__ Place place_of(const Groups& G, const Cut& c, int run, int tile, int column) {
    const int pair = tile / G.pair, w = min(G.pair, c.tiles - pair * G.pair), n = runs_of_item(G, c, run, w);
    const int before = pair > 0 ? pair * G.columns * runs_of_item(G, c, run, G.pair) : 0;
    return Place{before + column * n, n};
}

// A warp's knowledge of all runs.  A lane knows one group of 32.
struct Runs {
    const Groups& G;
    int run, all;                                  // pages of a run (0: the groups are in no order), all runs
    int g0, before;                                // first of the groups known; runs of the groups before it
    Cut mine;
    int upto;                                      // runs up to this lane's group

    __device__ __forceinline__ void know(int first) {
        g0 = first;
        const int g = g0 + (int)(threadIdx.x & 31);
        mine = Cut{};
        if (g < G.n) mine = SharedParts{G}(g);
    }
    __device__ __forceinline__ void count() {
        int x = mine.tiles > 0 ? runs_of(G, mine, run) : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, x, o);
            if ((int)(threadIdx.x & 31) >= o) x += t;
        }
        upto = before + x;
    }
    __device__ __forceinline__ Runs(const Groups& groups, int blocks) : G(groups), before(0) {
        // the shortest run that leaves no thread block with two; no shorter than an equal share, no longer than the longest item
        int cost = 0, most = 1;
        bool wrong = false;
        for (int g = 0; g < G.n; g += 32) {
            know(g);
            wrong |= mine.wrong;
            cost += __reduce_add_sync(0xffffffffu, (unsigned)(mine.tiles * G.columns * mine.pages));
            most = max(most, (int)__reduce_max_sync(0xffffffffu, (unsigned)(mine.tiles > 0 ? mine.pages : 0)));
        }
        run = max(1, (cost + blocks * G.pair - 1) / (blocks * G.pair));
        for (;; run += 1 + run / 16) {
            all = 0;
            for (int g = 0; g < G.n; g += 32) {
                if (G.n > 32) know(g);
                all += (int)__reduce_add_sync(0xffffffffu, (unsigned)(mine.tiles > 0 ? runs_of(G, mine, run) : 0));
            }
            if (all <= blocks || run >= most) break;
        }
        if (G.n > 32) know(0);
        count();
        if (__any_sync(0xffffffffu, wrong)) all = run = 0;
    }
    // plan: the pages of a run, then the runs before each group.
    __device__ __forceinline__ void write(int* plan, int* status) {
        if ((threadIdx.x & 31) == 0) {
            plan[0] = run, plan[1] = 0;
            if (run == 0) atomicCAS(status, 0, 11);
        }
        if (run == 0) return;
        for (int g = 0; g < G.n; g += 32) {
            if (g > 0) before = __shfl_sync(0xffffffffu, upto, 31), know(g), count();
            if (g + (int)(threadIdx.x & 31) < G.n) plan[2 + g + (threadIdx.x & 31)] = upto;
        }
    }
    // Run r (of those asked for one after the other, in rising order).
    __device__ __forceinline__ Segment segment(int r) {
        while (r >= __shfl_sync(0xffffffffu, upto, 31)) before = __shfl_sync(0xffffffffu, upto, 31), know(g0 + 32), count();
        const int l = __ffs(__ballot_sync(0xffffffffu, r < upto)) - 1;
        Segment s;
        Cut& c = s.cut;
        c.pages = __shfl_sync(0xffffffffu, mine.pages, l), c.tok0 = __shfl_sync(0xffffffffu, mine.tok0, l);
        c.n_tok = __shfl_sync(0xffffffffu, mine.n_tok, l), c.tiles = __shfl_sync(0xffffffffu, mine.tiles, l);
        c.seq = __shfl_sync(0xffffffffu, mine.seq, l);
        c.first = 0, c.end = c.pages * kPage;
        const int local = r - (l > 0 ? __shfl_sync(0xffffffffu, upto, l - 1) : before);
        const int per = G.columns * runs_of_item(G, c, run, G.pair), full = c.tiles / G.pair;
        const int pair = min(full, local / per), w = pair < full ? G.pair : c.tiles - full * G.pair, n = runs_of_item(G, c, run, w), rest = local - pair * per;
        s.column = rest / n;
        s.tile = pair * G.pair, s.tiles = w;
        s.from = (rest - s.column * n) * run_pages(G, run, w), s.to = min(c.pages, s.from + run_pages(G, run, w));
        s.record = r;
        return s;
    }
};

// ---- own keys ----------------------------------------------------------------------
// A worker's way through its run; a worker is `blockIdx.x`.  A lane knows one sequence (or group) of 32.
struct Walk {
    const OwnParts parts;
    Deal deal;
    int u, end;                                    // where it is in its run, the run's end
    int b0, units, items;                          // first of the sequences known; units and items before it
    Cut mine;
    int upto_units, upto_items;                    // ... and up to this lane's
    bool wrong;                                    // the groups are in no order

    __device__ __forceinline__ Cut cut(int first) const {
        const int b = first + (int)(threadIdx.x & 31);
        return b < parts.n() ? parts(b) : Cut{};
    }
    __device__ __forceinline__ void know(int first, const Cut& c) {
        b0 = first, mine = c;
        int y = mine.tiles * parts.G.kv_heads, x = y * mine.pages;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int tx = __shfl_up_sync(0xffffffffu, x, o), ty = __shfl_up_sync(0xffffffffu, y, o);
            if ((int)(threadIdx.x & 31) >= o) x += tx, y += ty;
        }
        upto_units = units + x, upto_items = items + y;
    }
    __device__ __forceinline__ void next(const Cut& c) {       // what was known becomes what lies before
        units = __shfl_sync(0xffffffffu, upto_units, 31), items = __shfl_sync(0xffffffffu, upto_items, 31);
        know(b0 + 32, c);
    }
    // plan: the workers' number (0: the groups are in no order) and the units and items before each sequence are written down there (null: not).
    __device__ __forceinline__ Walk(const OwnParts& p, int workers, int* plan) : parts(p), deal(0, 1), units(0), items(0), wrong(false) {
        const int lane = threadIdx.x & 31;
        know(0, cut(0));
        for (;;) {
            const Cut ahead = b0 + 32 < parts.n() ? cut(b0 + 32) : mine;       // (read beside what is counted now)
            const int b = b0 + lane;
            wrong |= mine.wrong;
            if (plan && b < parts.n()) plan[2 + b] = upto_units, plan[3 + parts.n() + b] = upto_items;
            if (b0 + 32 >= parts.n()) break;
            next(ahead);
        }
        deal = Deal(__shfl_sync(0xffffffffu, upto_units, 31), workers);
        wrong = __any_sync(0xffffffffu, wrong);
        if (plan && lane == 0) plan[0] = wrong ? 0 : deal.S, plan[1] = 0, plan[2 + parts.n()] = 0;
        const bool in = !wrong && deal.U > 0 && (int)blockIdx.x < deal.S;
        u = in ? deal.run_start(blockIdx.x) : 0;
        end = in ? deal.run_start(blockIdx.x + 1) : 0;
        if (u < units) units = items = 0, know(0, cut(0));                     // (else it begins among those known last)
    }
    // The next part of the run; false: there is none.
    __device__ __forceinline__ bool segment(Segment& s) {
        if (u >= end) return false;
        while (u >= __shfl_sync(0xffffffffu, upto_units, 31)) next(cut(b0 + 32));
        const int l = __ffs(__ballot_sync(0xffffffffu, u < upto_units)) - 1, columns = parts.G.kv_heads;
        Cut& c = s.cut;
        c.pages = __shfl_sync(0xffffffffu, mine.pages, l), c.tok0 = __shfl_sync(0xffffffffu, mine.tok0, l);
        c.n_tok = __shfl_sync(0xffffffffu, mine.n_tok, l), c.tiles = __shfl_sync(0xffffffffu, mine.tiles, l);
        c.seq = __shfl_sync(0xffffffffu, mine.seq, l);
        c.first = __shfl_sync(0xffffffffu, mine.first, l), c.end = __shfl_sync(0xffffffffu, mine.end, l);
        const int local = u - __shfl_sync(0xffffffffu, upto_units - mine.tiles * columns * mine.pages, l), item = local / c.pages;
        s.shared = parts.shared(b0 + l);
        s.tile = item / columns, s.tiles = 1, s.column = item - s.tile * columns;
        s.from = local - item * c.pages, s.to = min(c.pages, s.from + end - u);
        // (items and workers rise together along the runs: no two parts share the sum)
        s.record = __shfl_sync(0xffffffffu, upto_items - mine.tiles * columns, l) + item + (int)blockIdx.x;
        u += s.to - s.from;
        return true;
    }
};

// A record: [HD / 4][rows] groups of four sums, then [rows] pairs of maximum and sum.  Records of a kind, and the plan that Runs or Walk wrote
// (null: there are none):
struct Records {
    const int* plan;
    const float* at;
    int rows;                                      // that a record has room for
};

// 2^(a - b) for maxima that may be -inf (nothing seen): then the weight is 0.
__device__ __forceinline__ float weight(float a, float b) { return a == -INFINITY ? 0.f : exp2f(a - b); }

constexpr float LOG2E = 1.4426950408889634f;

// The forms for bfloat16 at head sizes 64 and 128: the shared part on tcgen05 (attn_shared_tc.cu; tiles of up to TC_ROWS rows, two an
// item), and the own keys streamed through shared memory (attn_shared_own.cu).
constexpr int TC_ROWS = 128, OWN_ROWS = 8, OWN_WARPS = 6;    // (warps an SM at head size 128, twice as many at 64)
bool fast_supported();
int launch_tc(const void* q, int n_tokens, const void* kv, int64_t kv_pages, const Groups& G, int blocks, float scale, int* plan, float* records, int* status,
              cudaStream_t s);
int launch_own(const void* q, const void* kv, int64_t kv_pages, void* out, const Groups& G, int groups, bool after_shared, int blocks, float scale, int* plan,
               float* records, int* status, cudaStream_t s);

}  // namespace shared_prefix
}  // namespace wick
