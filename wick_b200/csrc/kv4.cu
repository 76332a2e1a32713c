// Writing and reading a cache that holds keys and values in 4 bits (kv4.cuh): the per-head norm and rotation with the append, reading tokens back,
// and opening pages to bfloat16.
#include "kv4.cuh"
#include "packed.cuh"

#ifndef WICK_HD
#error "compile with -DWICK_HD=<head_dim>"
#endif

namespace wick {
namespace kv4 {

constexpr int D = WICK_HD;
static_assert(D % 64 == 0 && D >= 64 && D <= 256, "head sizes of 64, 128, 192 and 256");
typedef __nv_bfloat16 bf16;

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 x = ld4(p), y = ld4(p + 4);
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
}
__device__ __forceinline__ void load8(const bf16* p, float (&v)[8]) {
    Vec16<bf16> t;
    t.load(p);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = t.v[k];
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
    st4(p, v[0], v[1], v[2], v[3]);
    st4(p + 4, v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(bf16* p, const float (&v)[8]) {
    Vec16<bf16> t;
#pragma unroll
    for (int k = 0; k < 8; ++k) t.v[k] = v[k];
    t.store(p);
}

// The page of position pos of sequence b, or -1 (and a report) where the table has no such place or the cache no such page.
__device__ __forceinline__ int64_t page_of(const int* page_table, int table_width, int64_t kv_pages, int b, int pos, int* status) {
    const int j = pos / kPage;
    int64_t page = -1;
    if (pos >= 0 && j < table_width) page = page_table[(int64_t)b * table_width + j];
    if (page < 0 || page >= kv_pages) {
        atomicCAS(status, 0, 15);
        return -1;
    }
    return page;
}

// ---- append --------------------------------------------------------------------
// L lanes per vector (one head of q, k or v of one token): a lane holds 8 neighbouring channels i0 .. and their partners in the rotation, i0 + d / 2 ..;
// four neighbouring lanes hold a group of 32 channels in either half.
//   q:  x / sqrt(mean x^2 + eps) w, rotated, in 32 bits, rounded to the activations' type
//   k:  the same, then codes;   v: codes
// A code is that of the number that 64-bit arithmetic gives (sums over the projection's runs, norm, rotation, range, division).  32 bits would put a few
// numbers in a million, those next to the border between two codes, on the wrong side of it, another few for every other order of the same operations.  So a
// vector is computed in 32 bits with a bound on what they can be off by; where every decision (both scales' roundings, every code) is the same
// anywhere within the bound, it stands, and only where one is not (one key in some 60) the vector is computed again in 64.  4,425 tokens, 32 heads
// over 8 of 128: all in 64 bits 46 us, now 42 (the queries alone 21).
constexpr int L = D == 192 ? 16 : D / 16;

struct Source {                                                  // where a lane's numbers of a key or a value come from, and where its codes go
    const float* parts;                                          // the float32 partial sums, or null
    const void* qkv;                                             // the activations, or null
    int splits;
    int64_t split_stride, base;
    const float *w, *cos_t, *sin_t;                              // of this lane's channels; null: no norm, no rotation
    float eps;
    unsigned mask;                                               // the vector's lanes
    bool is_v;
    uint8_t* head;                                               // the head's part of the page; null: nowhere
    int row, i0;
};

// The sum over a vector's lanes.
template <typename T> __device__ __forceinline__ T vector_sum(T x, unsigned mask) {
    if constexpr (D == 192) {                                    // (12 lanes: each of 4, then the three)
        x += __shfl_xor_sync(mask, x, 1);
        x += __shfl_xor_sync(mask, x, 2);
        const int l0 = (threadIdx.x & 31) / L * L;
        return __shfl_sync(mask, x, l0) + __shfl_sync(mask, x, l0 + 4) + __shfl_sync(mask, x, l0 + 8);
    } else {
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) x += __shfl_xor_sync(mask, x, o);
        return x;
    }
}
__device__ __forceinline__ void store_codes(uint8_t* head, int row, int i0, bool is_v, int half, uint32_t word, uint32_t scale) {
    if (head == nullptr) return;
    if (is_v) word = ((word << 3) & 0xF8F8F8F8u) | ((word >> 5) & 0x07070707u);      // (every byte turned left by 3)
    else word = __funnelshift_l(word, word, 3);
    const int ch = i0 + half * (D / 2), o = ch / 2;
    uint8_t* codes = head + (is_v ? value_codes(D) + row * (D / 2) + value_byte<D>(row, o) : row * (D / 2) + o);
    *reinterpret_cast<uint32_t*>(codes) = word;
    if ((ch & (GROUP - 1)) == 0) *reinterpret_cast<uint32_t*>(head + (is_v ? value_scales(D) : key_scales(D)) + (row * (D / GROUP) + ch / GROUP) * 4) = scale;
}
__device__ __forceinline__ uint32_t pair_of(bf16 a, bf16 b) { return (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16; }
__device__ __forceinline__ int exact_code(double x, double a, double b) { return (int)fmin(fmax(rint((x - b) * 16.0 / a - 16.0), 0.0), 15.0); }
constexpr float LARGEST = 1.7014118346046923e38f;                // 2^127: beyond it values that codes stand for could be infinite

// One half of a vector, 8 numbers a lane, 4 lanes a group, in 64 bits.
__device__ __forceinline__ void encode_exactly(const double (&x)[8], const Source& s, int half) {
    double lo = x[0], hi = x[0];
    bool bad = false;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        lo = fmin(lo, x[k]);
        hi = fmax(hi, x[k]);
        bad |= !isfinite(x[k]);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fmin(lo, __shfl_xor_sync(s.mask, lo, o));
        hi = fmax(hi, __shfl_xor_sync(s.mask, hi, o));
        bad |= __shfl_xor_sync(s.mask, (int)bad, o) != 0;
    }
    // (to bfloat16 by way of 32 bits, as conversions from 64 bits go elsewhere)
    bf16 a = __float2bfloat16_rn((float)((hi - lo) * (16.0 / 15.0)));
    bf16 b = __float2bfloat16_rn((float)(lo - (double)__bfloat162float(a)));
    // (b on its own: from -1.2e38 to 1.2e38, say, a is finite and min - a is not)
    if (bad || fmax(fabs(lo), fabs(hi)) > (double)LARGEST || !isfinite(__bfloat162float(a)) || !isfinite(__bfloat162float(b))) {
        a = __float2bfloat16_rn(0.f);
        b = __ushort_as_bfloat16(0x7FFF);
    }
    const double af = (double)__bfloat162float(a), bf = (double)__bfloat162float(b);
    // 16 (x - b) / a - 16 with 20 bits behind the point, by adding 1.5 2^32: the code is known unless that is next to a half.  There, and where b is so
    // coarse that the number is large, a division: numbers of few bits often lie halfway between two codes, and the quotient is exact there.
    const double inv = af == 0.0 ? 0.0 : 16.0 / af;
    const bool all = fmax(fabs(hi - bf), fabs(lo - bf)) * inv >= 1000.0;
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int up = __double2loint(fma(x[k] - bf, inv, 6442450944.0 - 16.0)) + (1 << 19);
        int code = min(max(up >> 20, 0), 15);
        if (((up + 1) & 0xFFFFF) <= 2 || all) code = exact_code(x[k], af, bf);
        word |= (uint32_t)code << (4 * k);
    }
    if (af == 0.0) word = 0;
    store_codes(s.head, s.row, s.i0, s.is_v, half, word, pair_of(a, b));
}

template <typename T> __device__ __forceinline__ void vector_exactly(const Source& s) {
    double a[8], b[8];
    {
        float fa[8], fb[8];
        if (s.parts) {
            load8(s.parts + s.base, fa);
            load8(s.parts + s.base + D / 2, fb);
        } else {
            load8((const T*)s.qkv + s.base, fa);
            load8((const T*)s.qkv + s.base + D / 2, fb);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a[k] = (double)fa[k];
            b[k] = (double)fb[k];
        }
        for (int sp = 1; s.parts && sp < s.splits; ++sp) {
            load8(s.parts + sp * s.split_stride + s.base, fa);
            load8(s.parts + sp * s.split_stride + s.base + D / 2, fb);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                a[k] += (double)fa[k];
                b[k] += (double)fb[k];
            }
        }
    }
    if (s.w) {
        double ss = 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) ss += a[k] * a[k] + b[k] * b[k];
        ss = vector_sum(ss, s.mask);
        const double scale = 1.0 / sqrt(ss / (double)D + (double)s.eps);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a[k] = (a[k] * scale) * (double)s.w[k];
            b[k] = (b[k] * scale) * (double)s.w[k + D / 2];
        }
    }
    if (s.cos_t) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const double c = (double)s.cos_t[k], sn = (double)s.sin_t[k];
            const double ra = a[k] * c - b[k] * sn, rb = b[k] * c + a[k] * sn;
            a[k] = ra;
            b[k] = rb;
        }
    }
    encode_exactly(a, s, 0);
    encode_exactly(b, s, 1);
}
template <typename T> __device__ __noinline__ void vector_again(const Source* s) { vector_exactly<T>(*s); }

// One half in 32 bits, its numbers off by `off` at most from what 64 bits give.  Returns whether every decision is sure.  With u = 2^-24:
//   range and 16 / 15 of it: 2 off, and four roundings;   min - a: off, and a rounding;   the 64-bit path rounds either to 32 bits before bfloat16: one more;
//   16 (x - b) / a - 16 is taken with 16 bits behind the point from a sum near 192: half of its last place, off 16 / a, and three roundings of at most 48 (its distance from a border is compared with one and a
//   half of that place more).
__device__ __forceinline__ bool encode(const float (&x)[8], float off, unsigned mask, uint32_t& word, uint32_t& scale) {
    constexpr float u = 5.9604645e-8f;
    float lo = x[0], hi = x[0], all = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        lo = fminf(lo, x[k]);
        hi = fmaxf(hi, x[k]);
        all += x[k] * 0.f;                                       // (0, or no number if one of them is infinite or none)
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(mask, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(mask, hi, o));
    }
    const float range = (hi - lo) * (16.0f / 15.0f), da = 2.2f * off + 6.f * u * range;
    const bf16 a = __float2bfloat16_rn(range - da);
    const float af = __bfloat162float(a), least = lo - af, db = 1.1f * off + 3.f * u * fabsf(least);
    const bf16 b = __float2bfloat16_rn(least - db);
    const float bf = __bfloat162float(b), inv = 16.0f / af;
    bool sure = all == 0.f && af >= 1e-30f && fmaxf(fabsf(lo), fabsf(hi)) < 1e38f && fmaxf(fabsf(hi - bf), fabsf(lo - bf)) * inv < 48.f &&
                __bfloat16_as_ushort(a) == __bfloat16_as_ushort(__float2bfloat16_rn(range + da)) &&
                __bfloat16_as_ushort(b) == __bfloat16_as_ushort(__float2bfloat16_rn(least + db));
    const float wide = off * inv * 65536.0f;
    sure = sure && wide < 8000.f;
    const int d = sure ? (int)wide + 2 : 0;
    // The code with 16 bits behind the point, and a half: the low 20 bits of the number's, since 192 has none there; the least distance from a border.
    constexpr int ZERO = 0x43400000;
    int nearest = 0xFFFF;
    word = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int y = __float_as_int(fmaf(x[k] - bf, inv, 176.5f)), kept = min(max(y, ZERO), ZERO + 0xFFFFF);
        nearest = min(nearest, (y + d) & 0xFFFF);
        word |= k < 4 ? (uint32_t)kept >> (16 - 4 * k) & 0xFu << (4 * k) : (uint32_t)kept << (4 * k - 16) & 0xFu << (4 * k);
    }
    scale = pair_of(a, b);
    if (sure && nearest <= 2 * d) {
        if (off != 0.f) return false;
        // (the numbers are what they are, and those of few bits lie on borders)
        word = 0;
#pragma unroll 1
        for (int k = 0; k < 8; ++k) {
            float y = x[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) y = k == e ? x[e] : y;
            word |= (uint32_t)exact_code((double)y, (double)af, (double)bf) << (4 * k);
        }
    }
    return sure;
}

// EXACTLY: all keys and values in 64 bits at once.
template <typename T, bool EXACTLY>
__global__ void __launch_bounds__(128, EXACTLY ? 4 : 8)
append_kernel(const T* __restrict__ qkv, const float* __restrict__ parts, int splits, int64_t split_stride, int n_tokens, int n_heads, int n_kv,
              const float* __restrict__ q_w, const float* __restrict__ k_w, float eps, const float* __restrict__ cos_t,
              const float* __restrict__ sin_t, T* __restrict__ q_out, uint8_t* __restrict__ kv, int64_t kv_pages, const int* __restrict__ page_table,
              int table_width, int n_seqs, const int* __restrict__ seq_of_token, const int* __restrict__ positions, int write_kv, int* status) {
    pdl_trigger();
    pdl_wait();
    qkv = fresh(qkv);
    parts = fresh(parts);
    cos_t = fresh(cos_t);
    sin_t = fresh(sin_t);
    constexpr int half = D / 2;
    const int t = blockIdx.x;
    const int h = (blockIdx.y * blockDim.x + threadIdx.x) / L;
    const int i0 = (threadIdx.x % L) * 8;
    if (h >= n_heads + (write_kv ? 2 * n_kv : 0) || i0 >= half) return;
    // (the lanes of this vector: D / 16 of them, all of which are here)
    const unsigned mask = (D == 256 || D == 192 ? (D == 192 ? 0xFFFu : 0xFFFFu) : (1u << (D / 16)) - 1u) << ((threadIdx.x & 31) / L * L);
    const bool is_q = h < n_heads, is_v = h >= n_heads + n_kv;
    const float* w = is_q ? q_w : (is_v ? nullptr : k_w);
    const bool rotate = !is_v && cos_t != nullptr;
    const int64_t base = ((int64_t)t * (n_heads + 2 * n_kv) + h) * D + i0;
    uint8_t* head = nullptr;                                     // the head's part of the page; null: nowhere
    int row = 0;
    if (!is_q) {
        const int pos = positions[t], seq = seq_of_token[t];
        if (seq < 0 || seq >= n_seqs) {
            atomicCAS(status, 0, 15);
        } else {
            const int64_t page = page_of(page_table, table_width, kv_pages, seq, pos, status);
            if (page >= 0) head = kv + (page * n_kv + (h - n_heads - (is_v ? n_kv : 0))) * head_bytes(D);
        }
        row = pos & (kPage - 1);
    }
    auto source = [&]() {
        Source s;
        s.parts = parts;
        s.qkv = qkv;
        s.splits = splits;
        s.split_stride = split_stride;
        s.base = base;
        s.w = w ? w + i0 : nullptr;
        s.cos_t = rotate ? cos_t + (int64_t)t * half + i0 : nullptr;
        s.sin_t = rotate ? sin_t + (int64_t)t * half + i0 : nullptr;
        s.eps = eps;
        s.mask = mask;
        s.is_v = is_v;
        s.head = head;
        s.row = row;
        s.i0 = i0;
        return s;
    };
    if (EXACTLY && !is_q) {
        vector_exactly<T>(source());
        return;
    }
    float a[8], b[8];
    if (parts) {
        load8(parts + base, a);
        load8(parts + base + half, b);
        if (is_q) {
            for (int sp = 1; sp < splits; ++sp) {
                float da[8], db[8];
                load8(parts + sp * split_stride + base, da);
                load8(parts + sp * split_stride + base + half, db);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    a[k] += da[k];
                    b[k] += db[k];
                }
            }
        } else if (splits > 1) {
            // (in 64 bits: in 32 a sum of large runs of opposite signs would be off by more than a rounding of itself)
            double sa[8], sb[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                sa[k] = (double)a[k];
                sb[k] = (double)b[k];
            }
            for (int sp = 1; sp < splits; ++sp) {
                load8(parts + sp * split_stride + base, a);
                load8(parts + sp * split_stride + base + half, b);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    sa[k] += (double)a[k];
                    sb[k] += (double)b[k];
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                a[k] = (float)sa[k];
                b[k] = (float)sb[k];
            }
        }
    } else {
        load8(qkv + base, a);
        load8(qkv + base + half, b);
    }
    float largest = 0.f, turn = 1.f;                             // of the numbers before the rotation, and of its cosines and sines
    if (w) {
        float wa[8], wb[8];
        load8(w + i0, wa);
        load8(w + i0 + half, wb);
        float scale;
        if (is_q) {
            float ss = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) ss += a[k] * a[k] + b[k] * b[k];
            scale = 1.0f / sqrtf(vector_sum(ss, mask) / (float)D + eps);
        } else {
            // (the sum in 64 bits: in 32 the scale alone would be off by up to 15 roundings, and two to three times as many vectors would not be sure)
            double ss = 0.0;
#pragma unroll
            for (int k = 0; k < 8; ++k) ss += (double)a[k] * (double)a[k] + (double)b[k] * (double)b[k];
            const float mean = (float)(vector_sum(ss, mask) * (1.0 / D) + (double)eps);
            scale = 1.0f / sqrtf(mean);
            // Numbers below the smallest normal one are off by up to 2^-150, however small they are: such a mean proves nothing, and the numbers and their
            // products with the scale are off by that times what they are multiplied by (1.2e-38 of 7.5 roundings and more is above it).
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) top = fmaxf(top, fmaxf(fabsf(wa[k]), fabsf(wb[k])));
            largest = mean < 1.2e-38f ? INFINITY : 1.2e-38f * top * (scale + 1.f);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a[k] = (a[k] * scale) * wa[k];
            b[k] = (b[k] * scale) * wb[k];
        }
    }
    if (!is_q) {
        float size = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) size = fmaxf(size, fmaxf(fabsf(a[k]), fabsf(b[k])));
        largest += size;
    }
    if (rotate) {
        float c[8], sn[8];
        load8(cos_t + (int64_t)t * half + i0, c);
        load8(sin_t + (int64_t)t * half + i0, sn);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            turn = fmaxf(turn, fmaxf(fabsf(c[k]), fabsf(sn[k])));
            const float ra = a[k] * c[k] - b[k] * sn[k], rb = b[k] * c[k] + a[k] * sn[k];
            a[k] = ra;
            b[k] = rb;
        }
    }
    if (is_q) {
        T* dst = q_out + ((int64_t)t * n_heads + h) * D + i0;
        store8(dst, a);
        store8(dst + half, b);
        return;
    }
    // What the numbers can be off by, in roundings u of 32 bits, from what 64 bits give: their own 1 (0 for one run); the scale's 4 (the sum's
    // to 32 bits, of which a root keeps half, root, reciprocal, and what the numbers' do to it); two products 2; the rotation's products and sum 2, of two terms.
    largest = fmaxf(largest, __shfl_xor_sync(mask, largest, 1));
    largest = fmaxf(largest, __shfl_xor_sync(mask, largest, 2));
    turn = fmaxf(turn, __shfl_xor_sync(mask, turn, 1));
    turn = fmaxf(turn, __shfl_xor_sync(mask, turn, 2));
    const float off = (w ? (rotate ? 18.5f : 7.5f) : (parts && splits > 1 ? (rotate ? 6.5f : 1.5f) : (rotate ? 4.5f : 0.f))) * 5.9604645e-8f * largest * turn;
    uint32_t word[2], scale[2];
    bool sure = encode(a, off, mask, word[0], scale[0]);
    sure = encode(b, off, mask, word[1], scale[1]) && sure;
    if (__all_sync(mask, sure)) {
        store_codes(head, row, i0, is_v, 0, word[0], scale[0]);
        store_codes(head, row, i0, is_v, 1, word[1], scale[1]);
        return;
    }
    const Source s = source();
    vector_again<T>(&s);
}

// ---- reading tokens back ---------------------------------------------------------
// Channels 8 w .. 8 w + 7 of row t of a head's part of a page: their codes and scales, and their values.
struct Eight {
    uint32_t codes, scales;
};
__device__ __forceinline__ Eight load_eight(const uint8_t* head, int t, int w, bool is_v) {
    Eight e;
    e.scales = *reinterpret_cast<const uint32_t*>(head + (is_v ? value_scales(D) : key_scales(D)) + (t * (D / GROUP) + w / 4) * 4);
    e.codes = *reinterpret_cast<const uint32_t*>(head + (is_v ? value_codes(D) + t * (D / 2) + value_byte<D>(t, 4 * w) : t * (D / 2) + 4 * w));
    return e;
}
__device__ __forceinline__ uint4 values_of(const Eight& c, bool is_v) {
    const uint32_t a2 = low_halves(c.scales, c.scales), b2 = high_halves(c.scales, c.scales), x = c.codes;
    if (is_v) {
        uint32_t e[4], o[4];                                     // (both halves the same position)
        value_pair<0>(x, x, a2, b2, e[0], o[0]);
        value_pair<1>(x, x, a2, b2, e[1], o[1]);
        value_pair<2>(x, x, a2, b2, e[2], o[2]);
        value_pair<3>(x, x, a2, b2, e[3], o[3]);
        return make_uint4(low_halves(e[0], o[0]), low_halves(e[1], o[1]), low_halves(e[2], o[2]), low_halves(e[3], o[3]));
    }
    uint32_t v[4];
    key_word(x, a2, b2, v);
    return make_uint4(low_halves(v[0], v[1]), low_halves(v[2], v[3]), high_halves(v[0], v[1]), high_halves(v[2], v[3]));
}

__global__ void __launch_bounds__(128)
read_kernel(const uint8_t* __restrict__ kv, int64_t kv_pages, int n_kv, const int* __restrict__ page_table, int table_width, int n_seqs,
            const int* __restrict__ seq_of_token, const int* __restrict__ positions, int n, bf16* __restrict__ out, int* status) {
    pdl_trigger();
    pdl_wait();
    kv = fresh(kv);
    const int t = blockIdx.x, words = n_kv * (D / 8);
    const int i = blockIdx.y * blockDim.x + threadIdx.x;
    if (i >= 2 * words) return;
    const bool is_v = i >= words;
    const int h = (is_v ? i - words : i) / (D / 8), w = i % (D / 8);
    uint4 r = make_uint4(0, 0, 0, 0);
    const int seq = seq_of_token[t], pos = positions[t];
    int64_t page = -1;
    if (seq >= 0 && seq < n_seqs) page = page_of(page_table, table_width, kv_pages, seq, pos, status);
    else atomicCAS(status, 0, 15);
    if (page >= 0) r = values_of(load_eight(kv + (page * n_kv + h) * head_bytes(D), pos % kPage, w, is_v), is_v);
    *reinterpret_cast<uint4*>(out + (((int64_t)(is_v ? n : 0) + t) * n_kv + h) * D + 8 * w) = r;
}

// ---- opening pages ----------------------------------------------------------------
// The pages of all sequences of a step, in order, as bfloat16 pages [2, n_kv, 64, d] one behind the other, and a description of the step over them for the
// attention: the table that names them (every place of it), and the sequences' tokens and starts.  A sequence that does not fit the step or its page table is
// reported and has no pages; its start there is 0 (its results are nothing, and the attention reads within the arrays for it).  Rows behind a sequence's end are
// zeros.  key_scale: the keys are multiplied by 1, -1 or 0 (the attention wants a scale above 0).  A value that is no number would show in earlier tokens'
// rows too (they weigh it with 0, and 0 times it is none): where some token of the step does not see the position, its group is zeros and the position's key
// no number, which shows in every channel of the rows that see it, and in no others.  A block per page and key head.
struct OpenSeq {
    int start, len, pages;                                       // pages: -1 if it does not fit
};
__device__ __forceinline__ OpenSeq open_seq(const int* cu_seqlens, const int* start, int s, int n_tokens, int table_width) {
    const int first = cu_seqlens[s], end = cu_seqlens[s + 1], from = start[s];
    const int64_t len = (int64_t)from + end - first;
    const bool ok = first >= 0 && end >= first && end <= n_tokens && from >= 0 && len <= (int64_t)table_width * kPage;
    return {from, ok ? (int)len : 0, ok ? ((int)len + kPage - 1) / kPage : -1};
}

// Two bfloat16 numbers times -1 or 0 (exact; what is infinite or no number times 0 is none).
__device__ __forceinline__ uint32_t scaled(uint32_t x, int by) {
    if (by < 0) return x ^ 0x80008000u;
    const uint32_t lo = (x & 0x7F80u) == 0x7F80u ? 0x7FFFu : 0u, hi = (x & 0x7F800000u) == 0x7F800000u ? 0x7FFF0000u : 0u;
    return lo | hi;
}

__global__ void __launch_bounds__(256)
open_kernel(const uint8_t* __restrict__ kv, int64_t kv_pages, int n_kv, const int* __restrict__ page_table, int table_width,
            const int* __restrict__ cu_seqlens, const int* __restrict__ start, int n_seqs, int n_tokens, bf16* __restrict__ out,
            int* __restrict__ out_table, int* __restrict__ out_cu, int* __restrict__ out_start, int key_scale, int* status) {
    __shared__ int found[5];
    __shared__ uint8_t none[kPage];
    // (No pdl_trigger: the attention's blocks find their items behind their wait, and started early they only stand in these blocks' way: 48.6 us in place of 49.0
    // for 2,048 tokens, 32 heads over 8 of 128.)
    const int p = blockIdx.x, h = blockIdx.y;
    const bool describes = p == 0 && h == 0;                     // (the block that writes what is not a page's)
    if (threadIdx.x < 32) {
        // the sequence of page p of the step, and its first page's number: a scan over the sequences' pages
        const int lane = threadIdx.x;
        int before = 0, b = -1, j = 0, len = 0, from = 0;
        for (int s0 = 0; s0 < n_seqs; s0 += 32) {
            const int s = s0 + lane;
            const OpenSeq it = s < n_seqs ? open_seq(cu_seqlens, start, s, n_tokens, table_width) : OpenSeq{0, 0, 0};
            const int mine = max(it.pages, 0);
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const int total = __shfl_sync(0xffffffffu, upto, 31);
            if (b < 0 && p < before + total) {
                const int l = __ffs(__ballot_sync(0xffffffffu, p - before < upto)) - 1;
                b = s0 + l;
                j = p - before - __shfl_sync(0xffffffffu, upto - mine, l);
                len = __shfl_sync(0xffffffffu, it.len, l);
                from = __shfl_sync(0xffffffffu, it.start, l);
                if (!describes) break;
            }
            before += total;
        }
        if (lane == 0) {
            found[0] = b;
            found[1] = j;
            found[2] = len;
            found[3] = before;                                   // (where it describes the step: all pages)
            found[4] = from;
        }
    }
    __syncthreads();
    const int b = found[0], j = found[1], len = found[2];
    pdl_wait();
    // All codes of a page are asked for before the first are used (a loop that used them one by one: 42 us for 562 pages of 8 heads of 128, now 30).
    constexpr int STEPS = 2 * kPage * (D / 8) / 256;
    Eight e[STEPS];
    if (b >= 0) {
        kv = fresh(kv);
        int64_t page = page_of(page_table, table_width, kv_pages, b, j * kPage, status);
        if (page < 0) page = 0;
        const uint8_t* head = kv + (page * n_kv + h) * head_bytes(D);
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int i = u * 256 + threadIdx.x;
            e[u] = load_eight(head, i / (D / 8) % kPage, i % (D / 8), u >= STEPS / 2);
        }
        if (h == 0 && threadIdx.x == 0) out_table[(int64_t)b * table_width + j] = p;
        // The places behind a sequence's last page name page 0: the prompt attention copies pages in pairs, the second of an odd number's last pair with them.
        if (h == 0 && (j + 1) * kPage >= len)
            for (int i = j + 1 + threadIdx.x; i < table_width; i += 256) out_table[(int64_t)b * table_width + i] = 0;
    }
    if (describes) {                                             // (while the codes are on their way)
        bool misfit = false;
        for (int s = threadIdx.x; s < n_seqs; s += 256) {
            const int n = open_seq(cu_seqlens, start, s, n_tokens, table_width).pages;
            misfit |= n < 0;
            out_start[s] = n < 0 ? 0 : start[s];
            out_cu[s] = cu_seqlens[s];
            if (s == n_seqs - 1) out_cu[s + 1] = cu_seqlens[s + 1];
            if (n <= 0)
                for (int i = 0; i < table_width; ++i) out_table[(int64_t)s * table_width + i] = 0;
        }
        misfit = __syncthreads_or(misfit);
        if (threadIdx.x == 0 && misfit) {
            // (the tokens in order and within the step)
            atomicCAS(status, 0, 15);
            for (int s = 0, upto = 0; s <= n_seqs; ++s) out_cu[s] = upto = max(upto, min(cu_seqlens[s], n_tokens));
        }
        if (threadIdx.x == 0 && found[3] > (int)gridDim.x) {
            // Pages that there is no room for (the caller counted fewer): said, and named by a page that is there.
            atomicCAS(status, 0, 15);
            int before = 0;
            for (int s = 0; s < n_seqs; ++s) {
                const int n = max(0, open_seq(cu_seqlens, start, s, n_tokens, table_width).pages), room = max(0, (int)gridDim.x - before);
                if (room < n)
                    for (int i = room; i < table_width; ++i) out_table[(int64_t)s * table_width + i] = 0;
                before += n;
            }
        }
    }
    if (b < 0) return;
    const int rows = min(kPage, len - j * kPage), hidden = max(0, found[4] + 1 - j * kPage);        // (from row `hidden` on: not seen by all tokens)
    uint32_t lost = 0;                                           // this thread's values, a bit each, that are no numbers in such rows
    uint4* page_out = reinterpret_cast<uint4*>(out + ((int64_t)p * 2 * n_kv + h) * kPage * D);
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
        const bool is_v = u >= STEPS / 2;
        const int i = u % (STEPS / 2) * 256 + threadIdx.x, t = i / (D / 8);
        if (is_v && t >= hidden && t < rows && no_number(e[u].scales)) {
            e[u].scales = 0;
            lost |= 1u << (u - STEPS / 2);
        }
        uint4 v = values_of(e[u], is_v);
        if (!is_v && key_scale != 1) v = make_uint4(scaled(v.x, key_scale), scaled(v.y, key_scale), scaled(v.z, key_scale), scaled(v.w, key_scale));
        page_out[(is_v ? (int64_t)n_kv * kPage * (D / 8) : 0) + i] = t < rows ? v : make_uint4(0, 0, 0, 0);
    }
    if (hidden < rows && __syncthreads_or(lost != 0)) {
        if (threadIdx.x < kPage) none[threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < STEPS / 2; ++u)
            if (lost >> u & 1) none[(u * 256 + threadIdx.x) / (D / 8)] = 1;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < STEPS / 2; ++u)
            if (none[(u * 256 + threadIdx.x) / (D / 8)]) page_out[u * 256 + threadIdx.x] = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
    }
}

template <typename T>
static int append(const void* qkv, const float* parts, int splits, int n_tokens, int n_heads, int n_kv, const float* q_w, const float* k_w, float eps,
                  const float* cos_t, const float* sin_t, void* q_out, void* kv, int64_t kv_pages, const int* page_table, int table_width, int n_seqs,
                  const int* seq_of_token, const int* positions, int write_kv, int* status, void* stream) {
    WICK_REQUIRE(n_tokens >= 0 && n_heads > 0 && n_kv > 0 && table_width > 0 && n_seqs > 0, "qk_norm_rope_append_kv4: bad sizes");
    WICK_REQUIRE(!parts || splits >= 1, "qk_norm_rope_append_kv4: %d partial sums", splits);
    WICK_REQUIRE((((uintptr_t)qkv | (uintptr_t)parts | (uintptr_t)q_w | (uintptr_t)k_w | (uintptr_t)cos_t | (uintptr_t)sin_t | (uintptr_t)q_out |
                   (uintptr_t)kv) & 15) == 0, "qk_norm_rope_append_kv4: arrays must begin on multiples of 16 bytes");
    const int vectors = n_heads + (write_kv ? 2 * n_kv : 0);
    const int rows = ceil_div(vectors, 128 / L);
    WICK_REQUIRE(rows <= 65535, "qk_norm_rope_append_kv4: %d heads are beyond the grid's limit", vectors);
    if (n_tokens == 0) return 0;
    // (A step of few tokens waits for its slowest vector, which had better not be one that is computed twice: 64 tokens 5.3 us so, 13 with the second look.)
    WICK_CUDA(launch(n_tokens <= 256 ? append_kernel<T, true> : append_kernel<T, false>, dim3(n_tokens, rows), dim3(128), 0, (cudaStream_t)stream, (const T*)qkv, parts, splits,
                     (int64_t)n_tokens * (n_heads + 2 * n_kv) * D, n_tokens, n_heads, n_kv, q_w, k_w, eps, cos_t, sin_t, (T*)q_out, (uint8_t*)kv,
                     kv_pages, page_table, table_width, n_seqs, seq_of_token, positions, write_kv, status));
    return check_launch("qk_norm_rope_append_kv4");
}

}  // namespace kv4
}  // namespace wick

using namespace wick;
typedef __nv_bfloat16 bf16;

#define WICK_KV4_APPEND(NAME, T)                                                                                                                   \
    WICK_API int NAME(const void* qkv, const float* parts, int splits, int n_tokens, int n_heads, int n_kv, const float* q_w, const float* k_w,    \
                      float eps, const float* cos_t, const float* sin_t, void* q_out, void* kv, int64_t kv_pages, const int* page_table,           \
                      int table_width, int n_seqs, const int* seq_of_token, const int* positions, int write_kv, int* status, void* stream) {       \
        return kv4::append<T>(qkv, parts, splits, n_tokens, n_heads, n_kv, q_w, k_w, eps, cos_t, sin_t, q_out, kv, kv_pages, page_table,           \
                              table_width, n_seqs, seq_of_token, positions, write_kv, status, stream);                                            \
    }                                                                                                                                              \
    WICK_PACKED(NAME)
WICK_KV4_APPEND(wick_kv4_append_bf16, bf16)
WICK_KV4_APPEND(wick_kv4_append_f32, float)

// out: bfloat16 [2, n, n_kv, d].
WICK_API int wick_kv4_read(const void* kv, int64_t kv_pages, int n_kv, const int* page_table, int table_width, int n_seqs, const int* seq_of_token,
                           const int* positions, int n, void* out, int* status, void* stream) {
    WICK_REQUIRE(n >= 0 && n_kv > 0 && table_width > 0 && n_seqs > 0, "kv4_read: bad sizes");
    WICK_REQUIRE((((uintptr_t)kv | (uintptr_t)out) & 15) == 0, "kv4_read: arrays must begin on multiples of 16 bytes");
    if (n == 0) return 0;
    const int rows = ceil_div(2 * n_kv * (kv4::D / 8), 128);
    WICK_REQUIRE(rows <= 65535, "kv4_read: %d heads are beyond the grid's limit", n_kv);
    WICK_CUDA(launch(kv4::read_kernel, dim3(n, rows), dim3(128), 0, (cudaStream_t)stream, (const uint8_t*)kv, kv_pages, n_kv, page_table, table_width,
                     n_seqs, seq_of_token, positions, n, (bf16*)out, status));
    return check_launch("kv4_read");
}
WICK_PACKED(wick_kv4_read)

// out: bfloat16 [out_pages, 2, n_kv, 64, d]; out_table: int32 [n_seqs, table_width]; out_cu: int32 [n_seqs + 1]; out_start: int32 [n_seqs]; key_scale: 1, -1 or 0.
WICK_API int wick_kv4_open(const void* kv, int64_t kv_pages, int n_kv, const int* page_table, int table_width, const int* cu_seqlens, const int* start,
                           int n_seqs, int n_tokens, void* out, int out_pages, int* out_table, int* out_cu, int* out_start, int key_scale,
                           int* status, void* stream) {
    WICK_REQUIRE(n_kv > 0 && n_kv <= 65535 && table_width > 0 && table_width <= INT32_MAX / kPage && n_seqs > 0 && n_tokens >= 0 && out_pages > 0,
                 "kv4_open: bad sizes");
    WICK_REQUIRE((((uintptr_t)kv | (uintptr_t)out) & 15) == 0, "kv4_open: arrays must begin on multiples of 16 bytes");
    WICK_REQUIRE(kv_pages > 0, "kv4_open: a cache without pages");
    WICK_CUDA(launch(kv4::open_kernel, dim3(out_pages, n_kv), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)kv, kv_pages, n_kv, page_table,
                     table_width, cu_seqlens, start, n_seqs, n_tokens, (bf16*)out, out_table, out_cu, out_start, key_scale, status));
    return check_launch("kv4_open");
}
WICK_PACKED(wick_kv4_open)
