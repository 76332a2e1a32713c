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
//   k:  the same in 64 bits, then codes;   v: codes
// Codes are decided in 64 bits (sums over the projection's runs, norm, rotation, division): 32 would put a few numbers in a million, those next
// to the border between two codes, on the wrong side of it, another few for every other order of the same operations.
constexpr int L = D == 192 ? 16 : D / 16;

struct Codes {
    uint32_t word[2];                                            // of the lane's channels i0 .. and of their partners
    uint32_t scale[2];                                           // a | b << 16 of their groups
};

// One half of a vector: 8 numbers a lane, 4 lanes a group.
__device__ __forceinline__ void encode(const double (&x)[8], unsigned mask, bool is_v, uint32_t& word, uint32_t& scale) {
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
        lo = fmin(lo, __shfl_xor_sync(mask, lo, o));
        hi = fmax(hi, __shfl_xor_sync(mask, hi, o));
        bad |= __shfl_xor_sync(mask, (int)bad, o) != 0;
    }
    // (to bfloat16 by way of 32 bits, as conversions from 64 bits go elsewhere)
    bf16 a = __float2bfloat16_rn((float)((hi - lo) * (16.0 / 15.0)));
    bf16 b = __float2bfloat16_rn((float)(lo - (double)__bfloat162float(a)));
    // (2^127: so that no value that a code stands for is infinite either)
    if (bad || fmax(fabs(lo), fabs(hi)) > 0x1p127 || !isfinite(__bfloat162float(a))) {
        a = __float2bfloat16_rn(0.f);
        b = __ushort_as_bfloat16(0x7FFF);
        bad = true;
    }
    const double af = (double)__bfloat162float(a), bf = (double)__bfloat162float(b);
    const bool none = bad || af == 0.0;
    // 16 (x - b) / a - 16 with 20 bits behind the point, by adding 1.5 2^32: the code is known unless that is next to a half.  There, and where b is so
    // coarse that the number is large, a division: numbers of few bits often lie halfway between two codes, and the quotient is exact there.
    const double inv = none ? 0.0 : 16.0 / af;
    const bool near_all = fmax(fabs(hi - bf), fabs(lo - bf)) * inv >= 1000.0;
    word = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int up = __double2loint(fma(x[k] - bf, inv, 6442450944.0 - 16.0)) + (1 << 19);
        int code = min(max(up >> 20, 0), 15);
        if (((up + 1) & 0xFFFFF) <= 2 || near_all) code = (int)fmin(fmax(rint((x[k] - bf) * 16.0 / af - 16.0), 0.0), 15.0);
        word |= (uint32_t)code << (4 * k);
    }
    if (none) word = 0;
    if (is_v) word = ((word << 3) & 0xF8F8F8F8u) | ((word >> 5) & 0x07070707u);      // (every byte turned left by 3)
    else word = __funnelshift_l(word, word, 3);
    scale = (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16;
}

template <typename T>
__global__ void __launch_bounds__(128)
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
    float c[8], sn[8], wa[8], wb[8];
    if (rotate) {
        load8(cos_t + (int64_t)t * half + i0, c);
        load8(sin_t + (int64_t)t * half + i0, sn);
    }
    if (w) {
        load8(w + i0, wa);
        load8(w + i0 + half, wb);
    }
    if (is_q) {
        float a[8], b[8];
        if (parts) {
            load8(parts + base, a);
            load8(parts + base + half, b);
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
        } else {
            load8(qkv + base, a);
            load8(qkv + base + half, b);
        }
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) ss += a[k] * a[k] + b[k] * b[k];
            if (D == 192) {                                      // (12 lanes: each of 4, then the three)
                ss += __shfl_xor_sync(mask, ss, 1);
                ss += __shfl_xor_sync(mask, ss, 2);
                const int l0 = (threadIdx.x & 31) / L * L;
                ss = __shfl_sync(mask, ss, l0) + __shfl_sync(mask, ss, l0 + 4) + __shfl_sync(mask, ss, l0 + 8);
            } else {
#pragma unroll
                for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
            }
            const float scale = 1.0f / sqrtf(ss / (float)D + eps);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                a[k] = (a[k] * scale) * wa[k];
                b[k] = (b[k] * scale) * wb[k];
            }
        }
        if (rotate) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float ra = a[k] * c[k] - b[k] * sn[k], rb = b[k] * c[k] + a[k] * sn[k];
                a[k] = ra;
                b[k] = rb;
            }
        }
        T* dst = q_out + ((int64_t)t * n_heads + h) * D + i0;
        store8(dst, a);
        store8(dst + half, b);
        return;
    }
    const int kh = h - n_heads - (is_v ? n_kv : 0), pos = positions[t], seq = seq_of_token[t];
    double a[8], b[8];
    {
        float fa[8], fb[8];
        if (parts) {
            load8(parts + base, fa);
            load8(parts + base + half, fb);
        } else {
            load8(qkv + base, fa);
            load8(qkv + base + half, fb);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a[k] = (double)fa[k];
            b[k] = (double)fb[k];
        }
        for (int sp = 1; parts && sp < splits; ++sp) {
            load8(parts + sp * split_stride + base, fa);
            load8(parts + sp * split_stride + base + half, fb);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                a[k] += (double)fa[k];
                b[k] += (double)fb[k];
            }
        }
    }
    if (w) {
        double ss = 0.0;
#pragma unroll
        for (int k = 0; k < 8; ++k) ss += a[k] * a[k] + b[k] * b[k];
        if (D == 192) {
            ss += __shfl_xor_sync(mask, ss, 1);
            ss += __shfl_xor_sync(mask, ss, 2);
            const int l0 = (threadIdx.x & 31) / L * L;
            ss = __shfl_sync(mask, ss, l0) + __shfl_sync(mask, ss, l0 + 4) + __shfl_sync(mask, ss, l0 + 8);
        } else {
#pragma unroll
            for (int o = L / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
        }
        const double scale = 1.0 / sqrt(ss / (double)D + (double)eps);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            a[k] = (a[k] * scale) * (double)wa[k];
            b[k] = (b[k] * scale) * (double)wb[k];
        }
    }
    if (rotate) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const double ra = a[k] * (double)c[k] - b[k] * (double)sn[k], rb = b[k] * (double)c[k] + a[k] * (double)sn[k];
            a[k] = ra;
            b[k] = rb;
        }
    }
    Codes out;
    encode(a, mask, is_v, out.word[0], out.scale[0]);
    encode(b, mask, is_v, out.word[1], out.scale[1]);
    if (seq < 0 || seq >= n_seqs) {
        atomicCAS(status, 0, 15);
        return;
    }
    const int64_t page = page_of(page_table, table_width, kv_pages, seq, pos, status);
    if (page < 0) return;
    const int row = pos % kPage;
    uint8_t* dst = kv + (page * n_kv + kh) * head_bytes(D);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        const int ch = i0 + s * half, o = ch / 2;
        uint8_t* codes = dst + (is_v ? value_codes(D) + row * half + value_byte<D>(row, o) : row * half + o);
        *reinterpret_cast<uint32_t*>(codes) = out.word[s];
        if ((ch & (GROUP - 1)) == 0)
            *reinterpret_cast<uint32_t*>(dst + (is_v ? value_scales(D) : key_scales(D)) + (row * (D / GROUP) + ch / GROUP) * 4) = out.scale[s];
    }
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
// The pages of all sequences of a step, in order, as bfloat16 pages [2, n_kv, 64, d] one behind the other, and the table that names them there.  Rows
// behind a sequence's end are zeros.  A block per page and key head.
__global__ void __launch_bounds__(256)
open_kernel(const uint8_t* __restrict__ kv, int64_t kv_pages, int n_kv, const int* __restrict__ page_table, int table_width,
            const int* __restrict__ cu_seqlens, const int* __restrict__ start, int n_seqs, bf16* __restrict__ out,
            int* __restrict__ out_table, int* status) {
    // (No pdl_trigger: the kernel behind this one may read the page table before it waits, and this one writes it.)
    __shared__ int found[3];
    const int p = blockIdx.x, h = blockIdx.y;
    if (threadIdx.x < 32) {
        // the sequence of page p of the step, and its first page's number: a scan over the sequences' pages
        const int lane = threadIdx.x;
        int before = 0, b = -1, j = 0, len = 0;
        for (int s0 = 0; s0 < n_seqs; s0 += 32) {
            const int s = s0 + lane;
            const int mine_len = s < n_seqs ? start[s] + cu_seqlens[s + 1] - cu_seqlens[s] : 0;
            const int mine = (mine_len + kPage - 1) / kPage;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const int total = __shfl_sync(0xffffffffu, upto, 31);
            if (p < before + total) {
                const int l = __ffs(__ballot_sync(0xffffffffu, p - before < upto)) - 1;
                b = s0 + l;
                j = p - before - __shfl_sync(0xffffffffu, upto - mine, l);
                len = __shfl_sync(0xffffffffu, mine_len, l);
                break;
            }
            before += total;
        }
        if (lane == 0) {
            found[0] = b;
            found[1] = j;
            found[2] = len;
        }
    }
    __syncthreads();
    const int b = found[0], j = found[1], len = found[2];
    pdl_wait();
    if (b < 0) return;
    kv = fresh(kv);
    int64_t page = page_of(page_table, table_width, kv_pages, b, j * kPage, status);
    if (page < 0) page = 0;
    if (h == 0 && threadIdx.x == 0 && j < table_width) out_table[(int64_t)b * table_width + j] = p;
    if (p == (int)gridDim.x - 1 && h == 0 && threadIdx.x == 0) {
        // Pages that there is no room for (the caller counted fewer): said, and named by a page that is there.
        int before = 0;
        for (int s = 0; s < n_seqs; ++s) {
            const int n = (start[s] + cu_seqlens[s + 1] - cu_seqlens[s] + kPage - 1) / kPage;
            for (int i = max(0, p + 1 - before); i < n; ++i) {
                if (i < table_width) out_table[(int64_t)s * table_width + i] = 0;
                atomicCAS(status, 0, 15);
            }
            before += n;
        }
    }
    const uint8_t* head = kv + (page * n_kv + h) * head_bytes(D);
    const int rows = min(kPage, len - j * kPage);
    // All codes of a page are asked for before the first are used (a loop that used them one by one: 42 us for 562 pages of 8 heads of 128, now 30).
    constexpr int STEPS = 2 * kPage * (D / 8) / 256;
    Eight e[STEPS];
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
        const int i = u * 256 + threadIdx.x;
        e[u] = load_eight(head, i / (D / 8) % kPage, i % (D / 8), u >= STEPS / 2);
    }
#pragma unroll
    for (int u = 0; u < STEPS; ++u) {
        const bool is_v = u >= STEPS / 2;
        const int i = u * 256 + threadIdx.x, t = i / (D / 8) % kPage;
        const uint4 v = values_of(e[u], is_v);
        *reinterpret_cast<uint4*>(out + ((((int64_t)p * 2 + is_v) * n_kv + h) * kPage + t) * D + 8 * (i % (D / 8))) = t < rows ? v : make_uint4(0, 0, 0, 0);
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
    WICK_CUDA(launch(append_kernel<T>, dim3(n_tokens, rows), dim3(128), 0, (cudaStream_t)stream, (const T*)qkv, parts, splits,
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

// out: bfloat16 [out_pages, 2, n_kv, 64, d]; out_table: int32 [n_seqs, table_width].
WICK_API int wick_kv4_open(const void* kv, int64_t kv_pages, int n_kv, const int* page_table, int table_width, const int* cu_seqlens, const int* start,
                           int n_seqs, void* out, int out_pages, int* out_table, int* status, void* stream) {
    WICK_REQUIRE(n_kv > 0 && n_kv <= 65535 && table_width > 0 && n_seqs > 0 && out_pages >= 0, "kv4_open: bad sizes");
    WICK_REQUIRE((((uintptr_t)kv | (uintptr_t)out) & 15) == 0, "kv4_open: arrays must begin on multiples of 16 bytes");
    if (out_pages == 0) return 0;
    WICK_CUDA(launch(kv4::open_kernel, dim3(out_pages, n_kv), dim3(256), 0, (cudaStream_t)stream, (const uint8_t*)kv, kv_pages, n_kv, page_table,
                     table_width, cu_seqlens, start, n_seqs, (bf16*)out, out_table, status));
    return check_launch("kv4_open");
}
WICK_PACKED(wick_kv4_open)
