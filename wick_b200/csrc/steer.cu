// What a row's sequence has said so far, and what that and the caller's rules do to its logits.
//
// A row's history is a bit per token of the vocabulary (it occurred, in the prompt or in the output) and a count per token (times
// it was generated; only tokens with their bit set have one above 0).  The bits make the counts' table cheap to keep: a step reads
// the 4 V / 32 bytes of bits and the counts of set bits only, and a row is cleared by its bits.
//
//   l <- seen ? (l > 0 ? l / repetition : l * repetition) : l     (wick src/sampler.rs:76-85)
//   l <- l - (frequency * n + presence * [n > 0])                  n: the count
//   l <- l + bias of the token
//   l <- -inf where the row's mask does not allow the token
//
// Whole numbers are added with atomics, whose order changes nothing.  All arithmetic is in 32 bits, as the logits are.
// Steering is bound by one chain of dependent reads (place, mask, bits, count: 8 rows of 151,936 in 4.5 us, one of 32,768 in 2.6), which in
// large calls every round of blocks goes through: 61 rows of 100,003 tokens, half of them masked, 14.6 us, of which the bytes (4 read and 4
// written a token) are 7.6 and the instructions, some 200 a warp, 4.1.  History calls are a launch (2.4 us each in a graph).
#include "common.cuh"
#include "packed.cuh"

namespace wick {

constexpr int HT = 256;

// Blocks (chunk of words, row of the list).
__global__ void __launch_bounds__(HT)
history_clear_kernel(unsigned* seen, int* counts, const int* rows, int n_rows, int vocab, int words) {
    pdl_trigger();
    pdl_wait();
    seen = fresh(seen), counts = fresh(counts), rows = fresh(rows);
    const int r = rows[blockIdx.y];
    if (r < 0 || r >= n_rows) return;
    for (int i = blockIdx.x * HT + threadIdx.x; i < words; i += gridDim.x * HT) {
        unsigned w = seen[(int64_t)r * words + i];
        if (w == 0) continue;
        seen[(int64_t)r * words + i] = 0;
        while (w) {
            const int v = i * 32 + __ffs(w) - 1;
            if (v < vocab) counts[(int64_t)r * vocab + v] = 0;
            w &= w - 1;
        }
    }
}

__global__ void __launch_bounds__(HT)
history_add_kernel(unsigned* seen, int* counts, const int* tokens, const int* rows, int n, int n_rows, int vocab, int words, int generated) {
    pdl_trigger();
    pdl_wait();
    tokens = fresh(tokens), rows = fresh(rows);    // (the sampler before this kernel has just written the tokens)
    const int i = blockIdx.x * HT + threadIdx.x;
    if (i >= n) return;
    const int r = rows[i], v = tokens[i];
    if (r < 0 || r >= n_rows || v < 0 || v >= vocab) return;
    atomicOr(seen + (int64_t)r * words + (v >> 5), 1u << (v & 31));
    if (generated) atomicAdd(counts + (int64_t)r * vocab + v, 1);
}

struct Steer {
    const float* x;            // logits, rows x_stride apart
    float* y;                  // result, rows y_stride apart (may be x itself)
    int64_t x_stride, y_stride;
    int vocab, words, n_rows, n_masks;
    const int* rows;           // the row's place in the arrays below, or null: its own index
    const unsigned* seen;      // [n_rows, words], or null: no penalties
    const int* counts;         // [n_rows, vocab]
    const float* penalties;    // [n_rows, 3]: repetition, frequency, presence
    const int *bias_cu, *bias_tokens;
    const float* bias_values;  // tokens of one row are distinct
    int n_bias;                // entries there are: ranges end there
    const unsigned* masks;     // [n_masks, words]
    const int* mask_of;        // [n_rows], -1: none
};

// A block takes G tokens a thread of one row: four, or, where that is more than two rounds of blocks, eight, whose bits, block's prologue and
// turn cost half as many instructions, which bound a large call (61 rows of 100,003, half of them masked: 16.1 us and 14.6; 8 of
// 151,936: 4.5 and 5.0).
// VEC: x and y lie alike to 16 bytes, so that four tokens are one load and one store; a row of odd length begins in the middle of four, and
// the bits of a thread's tokens then lie in two words.
template <int G, bool VEC>
__global__ void __launch_bounds__(HT) steer_kernel(const Steer a) {
    constexpr int CH = HT * G;
    constexpr unsigned ALL = (1u << G) - 1;
    __shared__ float bias[CH];
    __shared__ unsigned biased[CH / 32];
    pdl_trigger();
    pdl_wait();
    const int i = blockIdx.y, V = a.vocab;
    const float* x = fresh(a.x) + i * a.x_stride;
    float* y = a.y + i * a.y_stride;
    const int skew = VEC ? (int)(((uintptr_t)x >> 2) & 3) : 0;     // tokens of the first four that lie before the row
    const int e0 = (int)blockIdx.x * CH - skew;                     // the block's first token
    const int r = a.rows ? a.rows[i] : i;
    const bool known = r >= 0 && r < a.n_rows;
    const unsigned* seen = known && a.seen ? a.seen + (int64_t)r * a.words : nullptr;
    const int* counts = a.counts + (int64_t)(known ? r : 0) * V;
    float rep = 1.f, freq = 0.f, pres = 0.f;
    if (seen) rep = a.penalties[r * 3], freq = a.penalties[r * 3 + 1], pres = a.penalties[r * 3 + 2];
    const int which = known && a.masks ? a.mask_of[r] : -1;
    const unsigned* mask = which >= 0 && which < a.n_masks ? a.masks + (int64_t)which * a.words : nullptr;
    int b0 = 0, b1 = 0;
    if (known && a.bias_cu) b0 = max(a.bias_cu[r], 0), b1 = min(a.bias_cu[r + 1], a.n_bias);
    bool biases = false;       // of tokens of this block
    if (b0 < b1) {
        for (int k = threadIdx.x; k < CH / 32; k += HT) biased[k] = 0;
        __syncthreads();
        for (int k = b0 + threadIdx.x; k < b1; k += HT) {
            const int at = a.bias_tokens[k] - e0;
            if (at >= 0 && at < CH) {
                biases = true;
                bias[at] = a.bias_values[k];
                atomicOr(&biased[at >> 5], 1u << (at & 31));
            }
        }
        biases = __syncthreads_or(biases);
    }
    // bits of the G tokens from e on (0 <= e, e + G <= V)
    auto bits = [&](const unsigned* w, int e) -> unsigned {
        const int k = e >> 5, s = e & 31;
        return __funnelshift_r(w[k], s > 32 - G ? w[k + 1] : 0u, s) & ALL;
    };
    auto one = [&](float l, int e, bool is_seen, bool is_biased) -> float {
        if (is_seen) {
            const int n = counts[e];
            l = l > 0.f ? __fdiv_rn(l, rep) : l * rep;
            if (n > 0) l -= fmaf(freq, (float)n, pres);
        }
        return is_biased ? l + bias[e - e0] : l;
    };
    const int at = (int)threadIdx.x * G, e = e0 + at;
    const unsigned biased_bits = biases ? biased[at >> 5] >> (at & 31) & ALL : 0u;
    if (VEC && e >= 0 && e + G <= V) {
        float o[G];
#pragma unroll
        for (int h = 0; h < G; h += 4) {           // (before the bits have come: waiting for them cost more than reading what a mask leaves out)
            const float4 v = *reinterpret_cast<const float4*>(x + e + h);
            o[h] = v.x, o[h + 1] = v.y, o[h + 2] = v.z, o[h + 3] = v.w;
        }
        const unsigned seen_bits = seen ? bits(seen, e) : 0u, allowed = mask ? bits(mask, e) : ALL;
        // Few tokens are seen or biased: a turn for each of the thread's, which is one or none nearly always.
        for (unsigned w = (seen_bits | biased_bits) & allowed; w; w &= w - 1) {
            const int k = __ffs(w) - 1;
            float l = o[0];
#pragma unroll
            for (int i = 1; i < G; ++i) l = k == i ? o[i] : l;
            l = one(l, e + k, seen_bits >> k & 1, biased_bits >> k & 1);
#pragma unroll
            for (int i = 0; i < G; ++i) o[i] = k == i ? l : o[i];
        }
        if (allowed != ALL) {
#pragma unroll
            for (int i = 0; i < G; ++i) o[i] = allowed >> i & 1 ? o[i] : -INFINITY;
        }
#pragma unroll
        for (int h = 0; h < G; h += 4) *reinterpret_cast<float4*>(y + e + h) = make_float4(o[h], o[h + 1], o[h + 2], o[h + 3]);
    } else {
        for (int k = max(e, 0); k < min(e + G, V); ++k) {
            const float l = one(x[k], k, seen && (seen[k >> 5] >> (k & 31) & 1), biased_bits >> (k - e) & 1);
            y[k] = !mask || (mask[k >> 5] >> (k & 31) & 1) ? l : -INFINITY;
        }
    }
}

}  // namespace wick

using namespace wick;

// seen: 32-bit words [n_rows, words]; counts: int32 [n_rows, vocab]; rows: int32 [n], rows outside are left out.
WICK_API int wick_history_clear(void* seen, int* counts, const int* rows, int n, int n_rows, int vocab, int words, void* s) {
    WICK_REQUIRE(vocab > 0 && words == (vocab + 31) / 32 && n >= 0 && n <= 65535, "history_clear: bad sizes");
    if (n == 0) return 0;
    WICK_CUDA(launch(history_clear_kernel, dim3(min(32, ceil_div(words, HT)), n), dim3(HT), 0, (cudaStream_t)s, (unsigned*)seen, counts, rows,
                     n_rows, vocab, words));
    return check_launch("history_clear");
}

// tokens, rows: int32 [n], the row that each token belongs to.  generated: counted, not only marked.
WICK_API int wick_history_add(void* seen, int* counts, const int* tokens, const int* rows, int n, int n_rows, int vocab, int words,
                              int generated, void* s) {
    WICK_REQUIRE(vocab > 0 && words == (vocab + 31) / 32 && n >= 0, "history_add: bad sizes");
    if (n == 0) return 0;
    WICK_CUDA(launch(history_add_kernel, dim3(ceil_div(n, HT)), dim3(HT), 0, (cudaStream_t)s, (unsigned*)seen, counts, tokens, rows, n, n_rows,
                     vocab, words, generated));
    return check_launch("history_add");
}

// x, y: float32 [n, vocab], rows x_stride / y_stride apart; the other arrays as in struct Steer.
WICK_API int wick_steer_logits(const float* x, int64_t x_stride, float* y, int64_t y_stride, int n, int vocab, const int* rows, int n_rows,
                               const void* seen, const int* counts, const float* penalties, const int* bias_cu, const int* bias_tokens,
                               const float* bias_values, int n_bias, const void* masks, const int* mask_of, int n_masks, void* s) {
    WICK_REQUIRE(vocab > 0 && n >= 0 && n <= 65535 && n_bias >= 0, "steer_logits: bad sizes");
    if (n == 0) return 0;
    Steer a = {x, y, x_stride, y_stride, vocab, (vocab + 31) / 32, n_rows, n_masks, rows, (const unsigned*)seen, counts, penalties,
               bias_cu, bias_tokens, bias_values, n_bias, (const unsigned*)masks, mask_of};
    const bool alike = (((uintptr_t)x ^ (uintptr_t)y) & 15) == 0 && (x_stride - y_stride) % 4 == 0;
    const bool eight = alike && (int64_t)ceil_div(vocab, HT * 4) * n > 16 * sm_count();
    const dim3 grid(ceil_div(vocab + (alike ? 3 : 0), HT * (eight ? 8 : 4)), n);
    if (eight) WICK_CUDA(launch(steer_kernel<8, true>, grid, dim3(HT), 0, (cudaStream_t)s, a));
    else if (alike) WICK_CUDA(launch(steer_kernel<4, true>, grid, dim3(HT), 0, (cudaStream_t)s, a));
    else WICK_CUDA(launch(steer_kernel<4, false>, grid, dim3(HT), 0, (cudaStream_t)s, a));
    return check_launch("steer_logits");
}
WICK_PACKED(wick_history_clear)
WICK_PACKED(wick_history_add)
WICK_PACKED(wick_steer_logits)
