// A paged key/value cache, gfx950: rows of many sequences in one pool of pages that a table names, what stores a token's rows there and what
// reads them -- attention of one new token of every sequence over all of its rows or over chosen pages, the pages' key bounds, the choice, and
// rows read back as f32.
//
// A pool row is n_kv * hd values (f32, f16, bf16, or Q8_0: int8 codes and an f16 scale for each 32, in the arrays of fhip_kvq_append). Position p of
// sequence i is pool row table[i][p >> shift] << shift | p & (R - 1); a table entry that is no page of the pool is looked up nowhere: its rows are
// dropped by a store and left out by a read.
#include "paged.hpp"

#include <type_traits>

#include "kvblock.hpp"

#include <math.h>

namespace {

using fhip::PagedPost;
using fhip::PagedView;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t NO_PAGE = 0xFFFFFFFFu;

template <int TYPE>
struct Elem {
    static constexpr int BYTES = TYPE == FHIP_F32 ? 4 : TYPE == FHIP_Q8_0 ? 1 : 2;
};

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, bf16x2)); }   // to nearest, ties to even
__device__ __forceinline__ uint32_t pack_f16(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, f16x2)); }

// Four consecutive values starting at value `at` (a multiple of 4) of a pool.
template <int TYPE>
__device__ __forceinline__ f32x4 load4(const void* __restrict__ pool, const uint16_t* __restrict__ scales, size_t at) {
    if constexpr (TYPE == FHIP_F32) {
        return *(const f32x4*)((const float*)pool + at);
    } else if constexpr (TYPE == FHIP_BF16) {
        const uint2 w = *(const uint2*)((const uint16_t*)pool + at);
        return (f32x4){bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
    } else if constexpr (TYPE == FHIP_F16) {
        const uint2 w = *(const uint2*)((const uint16_t*)pool + at);
        const f16x2 a = __builtin_bit_cast(f16x2, w.x), b = __builtin_bit_cast(f16x2, w.y);
        return (f32x4){(float)a.x, (float)a.y, (float)b.x, (float)b.y};
    } else {
        const uint32_t w = *(const uint32_t*)((const int8_t*)pool + at);
        const float d = fhip::kvq_scale(scales[at >> 5]);
        return (f32x4){fhip::kvq_value<FHIP_KVQ_Q8_0>((int8_t)(w & 255u), d, 0.f), fhip::kvq_value<FHIP_KVQ_Q8_0>((int8_t)((w >> 8) & 255u), d, 0.f),
                       fhip::kvq_value<FHIP_KVQ_Q8_0>((int8_t)((w >> 16) & 255u), d, 0.f), fhip::kvq_value<FHIP_KVQ_Q8_0>((int8_t)(w >> 24), d, 0.f)};
    }
}

// Number of pages that hold `len` rows, of those a table row may name.
__device__ __forceinline__ uint32_t pages_of(const PagedView& kv, uint32_t len) { return (uint32_t)(((uint64_t)len + (1u << kv.shift) - 1) >> kv.shift); }
// Rows of sequence i: what the caller says, as far as the table and the host's bound reach.
__device__ __forceinline__ uint32_t rows_of(const PagedView& kv, const uint32_t* __restrict__ lens, uint32_t i, uint32_t max_len) {
    const uint64_t cap = (uint64_t)kv.pages_per_seq << kv.shift;
    uint32_t n = lens[i];
    n = n < max_len ? n : max_len;
    return n < cap ? n : (uint32_t)cap;
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false)); }
template <int CTRL>
__device__ __forceinline__ uint64_t dpp(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xF, 0xF, false), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xF, 0xF, false);
    return (uint64_t)hi << 32 | lo;
}
// over the 16 lanes of a row, in all of them
template <typename T, typename Op>
__device__ __forceinline__ T row16(T v, Op op) {
    v = op(v, dpp<0xB1>(v));    // quad_perm [1,0,3,2]
    v = op(v, dpp<0x4E>(v));    // quad_perm [2,3,0,1]
    v = op(v, dpp<0x141>(v));   // row_half_mirror
    return op(v, dpp<0x140>(v));   // row_mirror
}

// with the other row of a half wave, the other half of the wave: the same in both
template <typename Op>
__device__ __forceinline__ float both_rows(float v, Op op) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
template <typename Op>
__device__ __forceinline__ float both_halves(float v, Op op) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
// what the lane 32 lanes away holds (HD = 128), or 16 (64)
template <int HD>
__device__ __forceinline__ float across(float v, int lane) {
    if constexpr (HD == 128) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(lane & 32 ? a[0] : a[1]);
    } else {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return __uint_as_float(lane & 16 ? a[0] : a[1]);
    }
}

// ---------------------------------------------------------------- storing the rows of new tokens
// values `at` and `at` + 1 of a pool; for Q8_0 the 16 lanes of a block together: d = amax / 127, codes round(v / d) half away from zero, as fhip_kvq_append's
template <int TYPE>
__device__ __forceinline__ void store_pair(const PagedView& kv, bool is_k, size_t at, float2 v, bool placed) {
    void* pool = is_k ? kv.k : kv.v;
    if constexpr (TYPE == FHIP_F32) {
        if (placed) *(float2*)((float*)pool + at) = v;
    } else if constexpr (TYPE == FHIP_BF16) {
        if (placed) *(uint32_t*)((uint16_t*)pool + at) = pack_bf16(v.x, v.y);
    } else if constexpr (TYPE == FHIP_F16) {
        if (placed) *(uint32_t*)((uint16_t*)pool + at) = pack_f16(v.x, v.y);
    } else {
#pragma clang fp contract(off)
        const float amax = row16(fmaxf(fmaxf(0.f, fabsf(v.x)), fabsf(v.y)), [](float a, float b) { return fmaxf(a, b); });
        const float d = amax / 127.0f, inv = d > 0.f ? 1.0f / d : 0.f;
        auto code = [&](float y) {
            const float t = y * inv, q = copysignf(floorf(fabsf(t) + 0.5f), t);
            return q != q ? 0 : (int)fminf(fmaxf(q, -127.0f), 127.0f);
        };
        if (placed) {
            *(uint16_t*)((uint8_t*)pool + at) = (uint16_t)((code(v.x) & 255) | (code(v.y) & 255) << 8);
            if ((threadIdx.x & 15) == 0) (is_k ? kv.k_scales : kv.v_scales)[at >> 5] = __half_as_ushort(__float2half_rn(d));
        }
    }
}
// Row i of the fused projection: + bias, RMS norm of query and key heads, rotation, queries to q_out, keys and values to the row of their page, rounded once.
// The angle pos * base^(-2c / n_rot) is formed in f64, in turns, and only its fraction of a turn is rounded to f32: the f32 product that the contiguous
// caches' post-processing forms is 4e-3 rad off at position 100 000.
// A lane holds two neighbouring dims, so a wave holds 128 values (a slice): one head of 128 or two of 64. TOK tokens a workgroup: with 4 a wave has a
// token to itself and the f64 work of its angles is shared by all of the token's heads; with 1 the waves share a token's slices.
template <int TYPE, int HD, int TOK>
__global__ __launch_bounds__(256) void append_kernel(PagedView kv, PagedPost p, int slices_per_wave) {
    constexpr int LPH = HD / 2;                       // lanes of a head
    constexpr int AHEAD = TOK == 1 ? 1 : 8;           // slices requested together
    __shared__ float2 turns[TOK][HD / 2];             // cos, sin of pair c
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int per_tok = p.n_head + 2 * kv.n_kv, slices = (per_tok * HD + 127) / 128;
    const uint32_t i = TOK == 1 ? blockIdx.x : blockIdx.x * TOK + wave;
    const int s0 = (TOK == 1 ? blockIdx.y * 4 + wave : blockIdx.y) * slices_per_wave;
    const int half = p.n_rot / 2;
    for (int e = tid; e < TOK * half; e += 256) {
        const int j = e / half, c = e - j * half;
        const uint32_t row = blockIdx.x * TOK + j;
        if (row < p.t) {
            double turn = (double)p.pos[row] * (exp((double)c * p.rate) * 0.15915494309189535);      // 1 / (2 pi)
            if (p.freq_scale) turn *= (double)p.freq_scale[c];
            float sn, cs;
            sincospif(2.f * (float)(turn - rint(turn)), &sn, &cs);
            turns[j][c] = make_float2(cs, sn);
        }
    }
    __syncthreads();
    if (i >= p.t) return;
    // the token's place
    const uint32_t seq = p.seqs ? p.seqs[i] : i, pos = p.pos[i], entry = pos >> kv.shift;
    uint32_t page = NO_PAGE;
    if (seq < kv.n_seq && entry < kv.pages_per_seq) page = kv.table[seq * kv.table_stride + entry];
    const bool placed = page < kv.n_pages;
    const size_t row = ((size_t)page << kv.shift) + (pos & ((1u << kv.shift) - 1));
    // this lane's two dims: their pairs' turns and where their partners are
    const int j0 = 2 * (lane % LPH);
    float2 t0 = make_float2(1.f, 0.f), t1 = t0;
    int from = lane;                                  // the lane of the partners (split halves)
    if (j0 < p.n_rot) {
        const float2* turn = turns[TOK == 1 ? 0 : wave];
        if (p.interleaved) {
            t0 = turn[j0 / 2];
        } else {
            const int c0 = j0 < half ? j0 : j0 - half, c1 = j0 + 1 < half ? j0 + 1 : j0 + 1 - half;
            t0 = turn[c0];
            t1 = turn[c1];
            from = lane + (j0 < half ? half / 2 : -(half / 2));
            if (j0 >= half) t0.y = -t0.y;             // the second of a pair: x2 cos + x1 sin
            if (j0 + 1 >= half) t1.y = -t1.y;
        }
    }
    const float* x = p.qkv + (size_t)i * per_tok * HD;
    const float2 one = make_float2(1.f, 1.f), wq = p.q_norm ? *(const float2*)(p.q_norm + j0) : one, wk = p.k_norm ? *(const float2*)(p.k_norm + j0) : one;
    const int s1 = s0 + slices_per_wave < slices ? s0 + slices_per_wave : slices;
    for (int s = s0; s < s1; s += AHEAD) {
        float2 v[AHEAD];
        int head[AHEAD];                              // per_tok and more: none (the last slice of heads of 64 may hold one head only)
#pragma unroll
        for (int e = 0; e < AHEAD; e++) {
            head[e] = s + e < s1 ? (s + e) * (128 / HD) + lane / LPH : per_tok;
            v[e] = head[e] < per_tok ? *(const float2*)(x + (size_t)head[e] * HD + j0) : make_float2(0.f, 0.f);
        }
        if (p.bias) {
            float2 add[AHEAD];
#pragma unroll
            for (int e = 0; e < AHEAD; e++) add[e] = head[e] < per_tok ? *(const float2*)(p.bias + (size_t)head[e] * HD + j0) : make_float2(0.f, 0.f);
#pragma unroll
            for (int e = 0; e < AHEAD; e++) {
                v[e].x += add[e].x;
                v[e].y += add[e].y;
            }
        }
        if (p.q_norm || p.k_norm) {
#pragma unroll
            for (int e = 0; e < AHEAD; e++) {
                float sq = row16(fmaf(v[e].x, v[e].x, v[e].y * v[e].y), [](float a, float b) { return a + b; });
                sq = both_rows(sq, [](float a, float b) { return a + b; });
                if (HD == 128) sq = both_halves(sq, [](float a, float b) { return a + b; });
                const bool is_q = head[e] < p.n_head, normed = is_q ? p.q_norm != nullptr : head[e] < p.n_head + kv.n_kv && p.k_norm;
                const float inv = 1.0f / sqrtf(sq / (float)HD + p.eps);
                if (normed) {
                    v[e].x = v[e].x * inv * (is_q ? wq.x : wk.x);
                    v[e].y = v[e].y * inv * (is_q ? wq.y : wk.y);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < AHEAD; e++) {
            float2 r = v[e];
            if (p.interleaved) {
                if (j0 < p.n_rot) {
                    r.x = fmaf(v[e].x, t0.x, -(v[e].y * t0.y));
                    r.y = fmaf(v[e].y, t0.x, v[e].x * t0.y);
                }
            } else if (half > 0) {
                float2 o;                             // the partners
                if (p.n_rot == HD) {                  // half a head away: 32 lanes, or 16
                    o = make_float2(across<HD>(v[e].x, lane), across<HD>(v[e].y, lane));
                } else if (half & 1) {                // the partner of dim j is dim j +- half, of the other parity
                    const int d = j0 < half ? half : -half, d1 = j0 + 1 < half ? half : -half, base = lane - lane % LPH;
                    o.x = __shfl(v[e].y, base + (((j0 + d) >> 1) & (LPH - 1)));
                    o.y = __shfl(v[e].x, base + (((j0 + 1 + d1) >> 1) & (LPH - 1)));
                } else {
                    o = make_float2(__shfl(v[e].x, from), __shfl(v[e].y, from));
                }
                if (j0 < p.n_rot) {
                    r.x = fmaf(v[e].x, t0.x, -(o.x * t0.y));
                    r.y = fmaf(v[e].y, t1.x, -(o.y * t1.y));
                }
            }
            if (head[e] < p.n_head + kv.n_kv) v[e] = r;
        }
#pragma unroll
        for (int e = 0; e < AHEAD; e++) {
            const int h = head[e];
            if (h < p.n_head) {
                *(float2*)(p.q_out + ((size_t)i * p.n_head + h) * HD + j0) = v[e];
            } else if (h < per_tok) {
                const bool is_k = h < p.n_head + kv.n_kv;
                store_pair<TYPE>(kv, is_k, (row * kv.n_kv + (h - p.n_head - (is_k ? 0 : kv.n_kv))) * HD + j0, v[e], placed);
            }
        }
    }
}

// ---------------------------------------------------------------- rows read back
template <int TYPE>
__global__ __launch_bounds__(256) void rows_kernel(PagedView kv, uint32_t width4, uint32_t seq, size_t row0, size_t rows, float* __restrict__ k_out, float* __restrict__ v_out) {
    const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x, i = id / width4;
    if (i >= rows) return;
    const size_t pos = row0 + i;
    const uint32_t page = kv.table[seq * kv.table_stride + (pos >> kv.shift)];
    if (page >= kv.n_pages) return;
    const size_t col = 4 * (id - i * width4), at = ((((size_t)page << kv.shift) + (pos & ((1u << kv.shift) - 1))) * width4) * 4 + col;
    *(f32x4*)((blockIdx.y ? v_out : k_out) + 4 * id) = load4<TYPE>(blockIdx.y ? kv.v : kv.k, blockIdx.y ? kv.v_scales : kv.k_scales, at);
}

// ---------------------------------------------------------------- bounds of a page's keys
// bounds [n_pages, n_kv, 2, hd]: the smallest and largest value of each dim among the page's keys. The last `fresh` rows of a sequence are new: a page whose
// first row is new starts over, another's bounds widen. One thread a dim; each page of a sequence is one workgroup's, so nothing is added by two.
template <int TYPE>
__global__ void bounds_kernel(PagedView kv, int hd, const uint32_t* __restrict__ lens, const uint32_t* __restrict__ fresh, uint32_t max_new, float* __restrict__ bounds) {
    const uint32_t seq = blockIdx.x / kv.n_kv, head = blockIdx.x % kv.n_kv, R = 1u << kv.shift;
    const uint32_t len = rows_of(kv, lens, seq, 0xFFFFFFFFu);
    uint32_t n = fresh ? fresh[seq] : max_new;
    n = n < max_new ? n : max_new;
    n = n < len ? n : len;
    if (n == 0) return;
    const int d = threadIdx.x;
    for (uint32_t entry = ((len - n) >> kv.shift) + blockIdx.y; entry <= (len - 1) >> kv.shift; entry += gridDim.y) {
        const uint32_t page = kv.table[seq * kv.table_stride + entry];
        if (page >= kv.n_pages) continue;
        const uint32_t start = entry << kv.shift, from = start > len - n ? start : len - n, to = len - start < R ? len : start + R;
        float* b = bounds + ((size_t)page * kv.n_kv + head) * 2 * hd + d;
        float lo = from == start ? INFINITY : b[0], hi = from == start ? -INFINITY : b[hd];
        bool nan = lo != lo || hi != hi;
#pragma unroll 8
        for (uint32_t r = from; r < to; r++) {
            const size_t at = ((((size_t)page << kv.shift) + (r - start)) * kv.n_kv + head) * hd + d;
            const float x = load4<TYPE>(kv.k, kv.k_scales, at & ~(size_t)3)[d & 3];
            nan |= x != x;
            lo = fminf(lo, x);
            hi = fmaxf(hi, x);
        }
        b[0] = nan ? NAN : lo;
        b[hd] = nan ? NAN : hi;
    }
}

// ---------------------------------------------------------------- the choice of pages
// score(page, kv head) = max over its query heads of sum_d max(q_d lo_d, q_d hi_d), the largest product with q that a key within the bounds can have. In f64: the order of
// pages whose scores are next to each other decides what is attended to, and f32 sums would decide it by the order of their additions. As a product: max(q lo, q hi)
// = max(q, 0) hi + min(q, 0) lo. Keys are ordered as unsigned words; a page that is always kept has the largest, a score that is no number the next.
__device__ __forceinline__ uint64_t order_key(double v) {
    if (v != v) return ~0ull - 1;
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return b >> 63 ? ~b : b | 1ull << 63;
}
// On v_mfma_f64_4x4x4_4b_f64, four blocks of 4 pages by 4 queries each: CALLS of them for up to 4 CALLS queries, max(q, 0) and min(q, 0) in f64 in LDS, a lane's bounds four neighbouring dims of
// a page at a time. The bounds' bytes are the floor; the instructions of 16 pages take 1024 CALLS cycles (CALLS = 2: 19.7 TB/s of bounds on the chip). us for 24 sequences' 52 MB of bounds: a wave a page, with a sum over its
// lanes for each of 8 queries, 75; on the 16 x 16 x 4 instruction, whose 16 columns take 4096 cycles whatever is in them, 20; this 18 to 19.5, 2.7 TB/s: of the
// waves' cycles 46 % count as SQ_WAIT_ANY and 43 % as SQ_WAIT_INST_ANY.
template <int HD, int CALLS>
__global__ __launch_bounds__(256) void score_kernel(PagedView kv, const float* __restrict__ q, const uint32_t* __restrict__ lens, uint32_t max_len, const float* __restrict__ bounds,
                                                    int n_head, uint32_t first, uint32_t last, uint64_t* __restrict__ keys, uint32_t key_stride) {
    constexpr int NI = HD / 16;
    __shared__ double up[CALLS][4 * NI][16], down[CALLS][4 * NI][16];      // [..][dim 16 i + 4 k + e as 4 i + e][4 k + query % 4]
    const int lane = threadIdx.x & 63, n = lane & 15, kg = lane >> 4, g = n_head / kv.n_kv, head = blockIdx.y;
    const uint32_t seq = blockIdx.z, pages = pages_of(kv, rows_of(kv, lens, seq, max_len)), groups = (pages + 15) / 16;
    if (blockIdx.x * 4 >= groups) return;
    const uint32_t j = blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t* table = kv.table + seq * kv.table_stride;
    keys += ((size_t)seq * kv.n_kv + head) * key_stride;
    const uint32_t mine = j < groups && 16 * j + n < pages ? table[16 * j + n] : NO_PAGE;
    const float* b = bounds + ((size_t)(mine < kv.n_pages ? mine : 0) * kv.n_kv + head) * 2 * HD + 4 * kg;
    f32x4 lo[NI], hi[NI];
#pragma unroll
    for (int i = 0; i < NI; i++) {
        lo[i] = *(const f32x4*)(b + 16 * i);
        hi[i] = *(const f32x4*)(b + HD + 16 * i);
    }
    __builtin_amdgcn_sched_barrier(0);                // all on their way while the queries are laid out
#pragma unroll
    for (int t = threadIdx.x; t < CALLS * 4 * HD; t += 256) {
        const int query = t / HD, dim = t % HD;
        const float x = query < g ? q[((size_t)seq * n_head + head * g + query) * HD + dim] : 0.f;
        const int at = 4 * (dim / 16) + dim % 4, slot = dim / 4 % 4 * 4 + query % 4;
        up[query / 4][at][slot] = x < 0.f ? 0.0 : (double)x;      // (no number stays one)
        down[query / 4][at][slot] = x < 0.f ? (double)x : 0.0;
    }
    __syncthreads();
    if (j >= groups) return;
    double s[CALLS], s2[CALLS];
#pragma unroll
    for (int c = 0; c < CALLS; c++) s[c] = s2[c] = 0;
    const int slot = 4 * kg + (n & 3);
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int c = 0; c < CALLS; c++) {
                s[c] = __builtin_amdgcn_mfma_f64_4x4x4f64((double)hi[i][e], up[c][4 * i + e][slot], s[c], 0, 0, 0);
                s2[c] = __builtin_amdgcn_mfma_f64_4x4x4f64((double)lo[i][e], down[c][4 * i + e][slot], s2[c], 0, 0, 0);
            }
    // page 16 j + n / 4 * 4 + kg, query 4 c + n % 4
    const int row = (n & ~3) + kg;
    const bool there = __shfl(mine, row) < kv.n_pages;
    uint64_t key = order_key(-INFINITY);
#pragma unroll
    for (int c = 0; c < CALLS; c++) {
        const uint64_t k = order_key(s[c] + s2[c]);
        if (there && 4 * c + (n & 3) < g && k > key) key = k;
    }
    const uint64_t a = dpp<0xB1>(key);                // over the four queries
    key = a > key ? a : key;
    const uint64_t c = dpp<0x4E>(key);
    key = c > key ? c : key;
    const uint32_t page = 16 * j + row;
    if ((n & 3) == 0 && page < pages) keys[page] = page < first || page + last >= pages ? ~0ull : key;
}

// The n_select largest keys of a list, equal ones by their place, as ascending places. One workgroup a list. The key that the last chosen one has is found by counting: the
// interval that holds it is cut into 1024 by its width, and the one of these with it is the next interval.
// T threads; HELD: they keep the keys in registers, up to HELD neighbouring ones each (0, for more than T * HELD: they read them again for each pass). With the keys read
// again for every pass 2048 pages took 16.6 us, from registers of 1024 threads, the 256 first of which had all of them, 13.5.
constexpr int SEL_BINS = 1024, SEL_HELD = 8;
// A wave's inclusive sum.
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);      // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);      // row_bcast 15 into rows 1 and 3, 31 into rows 2 and 3
    v += __builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}
// Over the workgroup: each thread's sum of those in front of it, and of all. buf: a word for each wave.
template <int T>
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* buf, uint32_t& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t upto = wave_upto(v);
    __syncthreads();
    if (lane == 63) buf[wave] = upto;
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        const uint32_t c = buf[w];
        before += w < wave ? c : 0;
        total += c;
    }
    all = total;
    return before + upto - v;
}
template <int T, int HELD>
__global__ __launch_bounds__(T) void select_kernel(PagedView kv, const uint32_t* __restrict__ lens, uint32_t max_len, uint32_t n_select, const uint64_t* __restrict__ keys,
                                                   uint32_t key_stride, uint32_t kept, uint32_t* __restrict__ out) {
    constexpr int BPT = SEL_BINS / T;                 // bins a thread
    __shared__ uint32_t hist[SEL_BINS], buf[T / 64];
    __shared__ uint64_t edge[2][T / 64];
    __shared__ uint32_t found[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t list = blockIdx.x, seq = list / kv.n_kv;
    const uint32_t n = pages_of(kv, rows_of(kv, lens, seq, max_len));
    keys += (size_t)list * key_stride;
    out += (size_t)list * n_select;
    if (n <= n_select) {
        for (uint32_t j = tid; j < n_select; j += T) out[j] = j < n ? j : NO_PAGE;
        return;
    }
    const uint32_t per = (n + T - 1) / T, first = tid * per;      // HELD: this thread's keys are first .. first + per - 1
    uint64_t held[HELD ? HELD : 1];
    if constexpr (HELD > 0)
#pragma unroll
        for (int e = 0; e < HELD; e++) held[e] = (uint32_t)e < per && first + e < n ? keys[first + e] : 0;
    // f(key, place) of this thread's keys, in their order where HELD
    auto each = [&](auto f) {
        if constexpr (HELD > 0) {
#pragma unroll
            for (int e = 0; e < HELD; e++)
                if ((uint32_t)e < per && first + e < n) f(held[e], first + e);
        } else {
            for (uint32_t j = tid; j < n; j += T) f(keys[j], j);
        }
    };
    uint64_t lo = ~0ull, hi = 0;
    each([&](uint64_t k, uint32_t) {
        if (k == ~0ull) return;                       // kept whatever its score
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
    });
    lo = row16(lo, [](uint64_t a, uint64_t b) { return a < b ? a : b; });
    hi = row16(hi, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) {
        const uint64_t a = __shfl_xor((unsigned long long)lo, o), b = __shfl_xor((unsigned long long)hi, o);
        lo = a < lo ? a : lo;
        hi = b > hi ? b : hi;
    }
    if (lane == 0) { edge[0][wave] = lo; edge[1][wave] = hi; }
#pragma unroll
    for (int e = 0; e < BPT; e++) hist[tid + T * e] = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; w++) {
        lo = edge[0][w] < lo ? edge[0][w] : lo;
        hi = edge[1][w] > hi ? edge[1][w] : hi;
    }
    // Chosen are the keys above hi and the largest `want` within [lo, hi]; here n > n_select >= kept, so that holds some. It is over when all that it holds are wanted, or are equal.
    uint32_t want = n_select - kept;
    if (want == 0) lo = hi = ~0ull;
    while (lo < hi) {                                 // (hist is clear here)
        const int bits = 64 - __builtin_clzll(hi - lo), shift = bits > 10 ? bits - 10 : 0;      // (hi - lo) >> shift < 1024
        each([&](uint64_t k, uint32_t) {
            if (k >= lo && k <= hi) atomicAdd(&hist[(uint32_t)((k - lo) >> shift)], 1u);
        });
        __syncthreads();
        uint32_t mine[BPT], sum = 0, all;             // this thread's bins, the highest first
#pragma unroll
        for (int e = 0; e < BPT; e++) {
            const int bin = SEL_BINS - 1 - (tid * BPT + e);
            sum += mine[e] = hist[bin];
            hist[bin] = 0;
        }
        uint32_t above = block_scan<T>(sum, buf, all);
#pragma unroll
        for (int e = 0; e < BPT; e++) {
            if (above < want && above + mine[e] >= want) {
                found[0] = SEL_BINS - 1 - (tid * BPT + e);
                found[1] = want - above;
                found[2] = mine[e];
            }
            above += mine[e];
        }
        __syncthreads();
        const uint64_t bin = found[0];
        if (bin < (hi - lo) >> shift) hi = lo + ((bin + 1) << shift) - 1;
        lo += bin << shift;
        want = found[1];
        if (want == found[2] && lo > 0) {             // all of them: those above lo - 1
            hi = --lo;
            want = 0;
        }
    }
    // places of the keys above lo, and of the first `want` that equal it
    auto above = [&](uint64_t k) { return k == ~0ull || k > lo; };
    auto equal = [&](uint64_t k) { return k == lo && k != ~0ull; };
    uint32_t all;
    if constexpr (HELD > 0) {
        uint32_t same = 0, take = 0;
        each([&](uint64_t k, uint32_t) { same += equal(k); });
        uint32_t rank = block_scan<T>(same, buf, all);
        const uint32_t rank0 = rank;
        each([&](uint64_t k, uint32_t) { take += above(k) || (equal(k) && rank++ < want); });
        uint32_t at = block_scan<T>(take, buf, all);
        rank = rank0;
        each([&](uint64_t k, uint32_t j) {
            if (above(k) || (equal(k) && rank++ < want)) out[at++] = j;
        });
    } else {
        uint32_t done = 0, ties = 0;
        for (uint32_t j0 = 0; j0 < n; j0 += T) {
            const uint32_t j = j0 + tid;
            const uint64_t k = j < n ? keys[j] : 0;
            const bool same = j < n && equal(k);
            const uint32_t rank = ties + block_scan<T>(same, buf, all);
            ties += all;
            const bool take = j < n && (above(k) || (same && rank < want));
            const uint32_t at = done + block_scan<T>(take, buf, all);
            done += all;
            if (take) out[at] = j;
        }
    }
}

// ---------------------------------------------------------------- attention of one token of every sequence
// out[h] = sum_j softmax_j(q_h . K_j / sqrt(hd)) V_j over the rows of the sequence, the g <= 16 query heads of a KV head together on the matrix cores, f32 grade whatever the rows
// are stored in. A wave takes a step of 16 keys (f32) or 32 (two tiles of 16, the other types) at a time.
//
// K q^T puts head n in lane n's column and keys 4 (lane / 16) + r of a tile in its four registers, which is where V^T p^T wants its second operand's keys: nothing is exchanged
// between the two products, and a head's running maximum and sum stay in its column's lanes. Both products are indifferent to which dims or keys share an instruction as
// long as their operands agree, so a lane's loads are of neighbouring bytes of one row: of a key's dims for K, of eight keys' same dims for V.
//   f32    v_mfma_f32_16x16x4_f32 on the rows as they are.
//   bf16   v_mfma_f32_16x16x32_bf16; q and p as three bf16 values each, cut off rather than rounded, so that they add up to the f32 value.
//   f16    v_mfma_f32_16x16x32_f16; q (times a power of two that brings its largest value to 2^14) and p (times 2^15) as two f16 values, 22 bits.
//   Q8_0   keys as f16 holds their codes, q as for f16, a block of 32 dims an instruction, whose sum is multiplied by the block's scale; values c * d, 8 by 11 bits, as the two f16 values
//          whose sum they are, p times 2^15 as two (three products: the two small parts' is 2^-22 of the result). On the f32 instruction, which takes four keys where
//          these take 32, a capped window of 33 sequences, 16 heads of 64, took 69 us.
// What two f16 values do not hold -- weights below 2^-18 of the largest so far, and Q8_0 values whose scale is 512 or more -- takes a step of
// these types to three bf16 values each, which have f32's range. us, every step so | none: 64 sequences of 2000 keys, 8 KV heads of 128 with 5 queries, Q8_0 75 | 62, f16 100 | 99; heads of 64, Q8_0
// 44 | 33, f16 44 | 44; one sequence of 65536 with 8 queries of 128, Q8_0 48 | 39, f16 50 | 49.
// Bound by the rows' bytes. The next step's keys are requested once the current ones are multiplied, its values once the current ones are: eight waves a CU keep 64 KB and more
// on the way without a second set of registers.
//
// Work is dealt out by the device, as only it knows the lengths: the steps of all (sequence, KV head) units in a row are cut into equal ranges, a workgroup each, whatever the
// lengths are. A unit that lies within one range is finished there; of others every workgroup leaves (maximum, sum, weighted rows) in the workspace and join_kernel adds them in order.
// SEL: the steps are those of the listed pages.
constexpr float LOG2E = 1.4426950408889634f;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
union Frag {
    uint32_t w[4];
    bf16x8 b;
    f16x8 h;
};
// the upper halves of two words, the first one's in the lower half
__device__ __forceinline__ uint32_t upper_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t lower_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
// the largest of a column's four lanes, in all of them
__device__ __forceinline__ float column_max(float v) {
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    return both_rows(both_halves(v, larger), larger);
}
// Two codes of a Q8_0 block as f16: byte c + 128 in the bits of 1024 + c + 128, less 1152. sel: 0x04ii04jj for bytes j and i.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, uint32_t sel) {
    const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, sel)) - off);
}
// Two f32 as PARTS 16-bit values each: word i of the result holds part i of both.
template <bool BF>
__device__ __forceinline__ void cut(float a, float b, uint32_t (&w)[3]) {
    if constexpr (BF) {
#pragma unroll
        for (int i = 0; i < 3; i++) {
            w[i] = upper_halves(__float_as_uint(a), __float_as_uint(b));
            a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
            b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
        }
    } else {
        const f16x2 hi = __builtin_bit_cast(f16x2, pack_f16(a, b));
        w[0] = __builtin_bit_cast(uint32_t, hi);
        w[1] = pack_f16(a - (float)hi.x, b - (float)hi.y);
    }
}

// tanh of four scores over their cap, which is small for nearly all of them: its series up to y^17 within 1/2 (what is left out is 9e-10 of it there, a 66th of an f32 rounding), otherwise 1 - 2 / (1 + e^2y), whose
// cancellation costs a factor of two there at most. The library's tanhf has two branches a value, and a wave takes both: the kernel for 33 sequences, window
// 1024, 16 heads of 64 on Q8_0 took 74.5 us with it and 69.2 with this and the bookkeeping in scalar registers.
__device__ __forceinline__ f32x4 tanh4(f32x4 y) {
    const f32x4 z = y * y;
    f32x4 t = z * (6404582.f / 10854718875.f) - 929569.f / 638512875.f;
    t = t * z + 21844.f / 6081075.f;
    t = t * z - 1382.f / 155925.f;
    t = t * z + 62.f / 2835.f;
    t = t * z - 17.f / 315.f;
    t = t * z + 2.f / 15.f;
    t = t * z - 1.f / 3.f;
    t = y * z * t + y;
    float far = 0.f;
#pragma unroll
    for (int r = 0; r < 4; r++) far = fmaxf(far, fabsf(y[r]));
    if (__any(!(far < 0.5f))) {
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const float big = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(fabsf(y[r]) * (2.f * LOG2E)));
            t[r] = fabsf(y[r]) < 0.5f ? t[r] : copysignf(big, y[r]);
        }
    }
    return t;
}

template <int TYPE>
struct Path {
    static constexpr int TILES = TYPE == FHIP_F32 ? 1 : 2;            // of 16 keys a step
    static constexpr int KEYS = 16 * TILES;
    static constexpr int PARTS = TYPE == FHIP_BF16 ? 3 : 2;
    static constexpr bool HALF = TYPE != FHIP_F32;                    // on a 16-bit instruction
    static constexpr float UP = TYPE == FHIP_F16 || TYPE == FHIP_Q8_0 ? 32768.f : 1.f;      // of the weights
};

// Keys of sequence `seq` that are attended to, [lo, len), and the steps that they lie in.
struct Span {
    uint32_t len, lo, first, steps;
};
template <int TYPE, bool SEL>
__device__ __forceinline__ Span span_of(const PagedView& kv, const uint32_t* __restrict__ lens, uint32_t seq, uint32_t max_len, uint32_t window, uint32_t n_select) {
    constexpr int KEYS = Path<TYPE>::KEYS;
    Span s;
    s.len = rows_of(kv, lens, seq, max_len);
    s.lo = window && window < s.len ? s.len - window : 0;
    if constexpr (SEL) {
        const uint32_t pages = pages_of(kv, s.len), listed = pages < n_select ? pages : n_select;
        s.first = 0;
        s.steps = (uint32_t)((((uint64_t)listed << kv.shift) + KEYS - 1) / KEYS);
    } else {
        s.first = s.lo / KEYS;
        s.steps = s.len ? (s.len - 1) / KEYS + 1 - s.first : 0;
    }
    return s;
}
// The same in scalar registers, where it is the same for the whole wave.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) { return (uint64_t)uniform((uint32_t)(v >> 32)) << 32 | uniform((uint32_t)v); }
__device__ __forceinline__ Span uniform(Span s) { return Span{uniform(s.len), uniform(s.lo), uniform(s.first), uniform(s.steps)}; }
struct Attend {
    PagedView kv;
    const float* q;
    const uint32_t* lens;
    const uint32_t* selected;
    float *out, *part;      // part: per workgroup two times g rows of HD, then g (maximum, sum), and 2 g words to keep the next one aligned
    uint32_t* plan;         // per unit: the first and the last workgroup with steps of it, and whether it is the first one's second share; first = last: nothing to join
    uint32_t max_len, n_select, window;
    int n_head;
    float softcap, scale;
    int log_wgs;            // the steps are dealt out to 1 << log_wgs workgroups, MIN_STEPS each at least; < 0: workgroup u has unit u
    uint32_t min_steps;
};

// What a unit costs in steps beside its own: its queries, its first keys' trip and the waves' sums. Without it a workgroup that has many short sequences' units was the last by far: 24 sequences
// of 1 .. 4096 keys on bf16 took 58 us where as many keys in sequences of equal length took 44.
constexpr uint32_t UNIT_COST = 6;
__device__ __forceinline__ uint32_t unit_cost(uint32_t steps) { return steps ? steps + UNIT_COST : 0; }

// Workgroups go round the eight XCDs, each with an L2 of its own. Place of workgroup b of n so that those of an XCD are neighbours: for Q8_0, whose rows' scales are a line for all KV heads of a sequence.
// us with it | without: a window of 33 sequences, 16 heads of 64, 26.5 | 28.3; 8 of 2000 keys 19.7 | 20.4; the other types, whose heads share nothing, are up to 10 % faster spread out (64 of 2000 on
// bf16 100 | 97, 8 of 4096 on f32 60 | 55), but for one of 131072 on bf16, 104.5 | 107.6.
__device__ __forceinline__ uint32_t xcd_neighbours(uint32_t b, uint32_t n) {
    const uint32_t x = b % 8, each = n / 8, more = n % 8;
    return x * each + (x < more ? x : more) + b / 8;
}

template <int TYPE, int HD, bool SEL, int WV>
__global__ __launch_bounds__(64 * WV, HD == 64 ? 3 : 2) void attention_kernel(Attend a) {
    typedef Path<TYPE> P;
    constexpr int TILES = P::TILES, PARTS = P::PARTS, NB = HD / 32, NJ = HD / 16;
    constexpr int IDS = 64 / TILES;                   // steps whose pages a wave looks up at once
    __shared__ float sm_m[WV][16], sm_l[WV][16];
    __shared__ __attribute__((aligned(16))) float sm_o[WV][16][HD + 4];
    const PagedView& kv = a.kv;
    const int lane = threadIdx.x & 63, wave = WV == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, kg = lane >> 4;
    const int g = a.n_head / kv.n_kv;

    uint32_t place = blockIdx.x;
    // this workgroup's steps, and the unit that the first of them belongs to
    uint32_t at = 0, end = 0, unit0 = 0, each = 1;    // places [at, end) of the row of all units (the host has seen that there are fewer than 2^31); unit0: the current unit's first
    uint32_t seq = 0, head = 0, shares = 0;
    Span sp;
    if (a.log_wgs < 0) {
        if (TYPE == FHIP_Q8_0) place = xcd_neighbours(place, gridDim.x);
        seq = place / kv.n_kv;
        head = place % kv.n_kv;
        sp = uniform(span_of<TYPE, SEL>(kv, a.lens, seq, a.max_len, a.window, a.n_select));
    } else {
        // lane l: sequence b + l, what its units cost, and what all up to it do
        Span here;
        uint32_t cost = 0, upto = 0;
        auto costs = [&](uint32_t b) {
            here = Span{0, 0, 0, 0};
            if (b + lane < kv.n_seq) here = span_of<TYPE, SEL>(kv, a.lens, b + lane, a.max_len, a.window, a.n_select);
            cost = unit_cost(here.steps);
            upto = wave_upto(cost * (uint32_t)kv.n_kv);
        };
        uint32_t all = 0;
        for (uint32_t b = (kv.n_seq - 1) & ~63u;; b -= 64) {      // the first 64 stay in hand
            costs(b);
            all += __builtin_amdgcn_readlane(upto, 63);
            if (b == 0) break;
        }
        each = (all + (1u << a.log_wgs) - 1) >> a.log_wgs;
        each = each > a.min_steps ? each : a.min_steps;
        if (TYPE == FHIP_Q8_0 && place * each < all) place = xcd_neighbours(place, (all + each - 1) / each);
        at = place * each;
        end = at + each < all ? at + each : all;
        if (at >= end) return;
        uint32_t before = 0;
        uint64_t found;
        while (!(found = __ballot(before + upto > at))) {
            before += __builtin_amdgcn_readlane(upto, 63);
            seq += 64;
            if (seq >= kv.n_seq) return;              // (lengths that change under the launch)
            costs(seq);
        }
        const int l = __builtin_ctzll(found);
        seq += l;
        sp = Span{(uint32_t)__builtin_amdgcn_readlane(here.len, l), (uint32_t)__builtin_amdgcn_readlane(here.lo, l), (uint32_t)__builtin_amdgcn_readlane(here.first, l),
                  (uint32_t)__builtin_amdgcn_readlane(here.steps, l)};
        before += __builtin_amdgcn_readlane(upto, l);
        const uint32_t its = __builtin_amdgcn_readlane(cost, l);
        before -= its * (uint32_t)kv.n_kv;
        head = (at - before) / its;
        unit0 = before + head * its;
    }
    // to the sequence's next KV head, or the next sequence with any steps, if places of it are this workgroup's
    auto next_unit = [&] {
        unit0 += unit_cost(sp.steps);
        at = unit0;
        if (at + UNIT_COST >= end) return false;
        if (++head == (uint32_t)kv.n_kv) {
            head = 0;
            do {
                if (++seq >= kv.n_seq) return false;
                sp = uniform(span_of<TYPE, SEL>(kv, a.lens, seq, a.max_len, a.window, a.n_select));
            } while (sp.steps == 0);
        }
        return true;
    };

    for (;;) {
        // steps [from, to) of the unit are this workgroup's: those of the places [at, end), of which a unit's first UNIT_COST are none
        auto step_at = [&](uint32_t place) { return place <= unit0 + UNIT_COST ? 0u : place - unit0 - UNIT_COST < sp.steps ? place - unit0 - UNIT_COST : sp.steps; };
        const uint32_t from = step_at(at), to = a.log_wgs < 0 ? sp.steps : step_at(end);
        const bool whole = from == 0 && to == sp.steps;
        if (a.log_wgs >= 0 && to == from) {
            if (!next_unit()) return;
            continue;
        }
        const uint32_t* table = kv.table + seq * kv.table_stride;
        const uint32_t* list = SEL ? a.selected + ((size_t)seq * kv.n_kv + head) * a.n_select : nullptr;
        const uint32_t pages = pages_of(kv, sp.len), row_values = (uint32_t)kv.n_kv * HD;

        float m = -INFINITY, l = 0.f, c2 = a.softcap > 0.f ? a.scale / a.softcap : a.scale * LOG2E;
        f32x4 acc[NJ];
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[j] = (f32x4){0.f, 0.f, 0.f, 0.f};

        const uint32_t mine = to - from > (uint32_t)wave ? (to - from - wave + WV - 1) / WV : 0;      // steps of this wave: from + wave, + WV, ..
        // Lane e: tile e of the steps looked up last, its first key's position and its row's first value in the pools.
        uint32_t tile_pos = NO_PAGE;
        uint64_t tile_at = 0;
        auto look_up = [&](uint32_t k) {              // of steps k .. k + IDS - 1 of this wave
            const uint32_t step = k + lane / TILES;
            uint32_t page = NO_PAGE, entry = 0, start = 0;
            if (step < mine) {
                const uint32_t tile = (sp.first + from + wave + step * WV) * TILES + lane % TILES, slot = tile >> (kv.shift - 4);
                start = (tile & ((1u << (kv.shift - 4)) - 1)) << 4;
                entry = slot;
                if (SEL) entry = slot < a.n_select && slot < pages ? list[slot] : NO_PAGE;
                if (entry < pages) page = table[entry];
            }
            const bool none = page >= kv.n_pages;     // its place in page 0 is read and counts for nothing
            tile_pos = none ? NO_PAGE : (entry << kv.shift) + start;
            tile_at = (((uint64_t)(none ? 0 : page) << kv.shift) + start) * row_values + (uint32_t)head * HD;
        };
        struct Tile {
            uint32_t pos;          // of its first key, a multiple of 16 (NO_PAGE: no key of it counts)
            uint64_t at;           // the KV head's first value of that key
        };
        Tile cur[TILES], nxt[TILES];
        auto find = [&](uint32_t k, Tile (&t)[TILES]) {
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                const uint32_t e = (k % IDS) * TILES + i;
                t[i].pos = __builtin_amdgcn_readlane(tile_pos, e);
                t[i].at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(tile_at >> 32), e) << 32 | (uint32_t)__builtin_amdgcn_readlane((uint32_t)tile_at, e);
            }
        };
        // rows of a tile: K by lane (key n, dims by kg), V by lane (keys 4 kg + r, dims by n)
        constexpr int KW = TYPE == FHIP_F32 ? NJ : TYPE == FHIP_Q8_0 ? (NB + 1) / 2 : NB;      // 16-byte words of a lane's part of a key
        constexpr int VB = HD / 16 * Elem<TYPE>::BYTES;                                       // bytes of a lane's part of a value: 4 .. 32
        constexpr int VW = VB < 4 ? 1 : VB / 4;
        uint32_t kr[TILES][KW * 4], vr[TILES][4][VW];
        uint32_t kd[TYPE == FHIP_Q8_0 ? TILES : 1][4][NB / 2];      // two scales a word
        uint16_t vd[TYPE == FHIP_Q8_0 ? TILES : 1][4];
        const uint32_t k_off = n * row_values * Elem<TYPE>::BYTES + (TYPE == FHIP_Q8_0 ? 8 : 16) * kg;      // of a lane's parts from their tile's first byte
        uint32_t v_off[4], d_off[4];
#pragma unroll
        for (int r = 0; r < 4; r++) {
            v_off[r] = (4 * kg + r) * row_values * Elem<TYPE>::BYTES + (TYPE == FHIP_F32 ? 16 : VB) * n;
            d_off[r] = (4 * kg + r) * (row_values / 16);
        }
        // A tile's bytes from the KV head's first on, as a buffer: the address in scalar registers and a lane's 32-bit offset from it, where a pointer's loads cost an addition of
        // 64 bits a lane each, a tenth of a Q8_0 step's instructions.
        auto tile_bytes = [&](const void* pool, uint64_t bytes) { return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)pool + bytes), 0, (int)(16 * row_values * 4), 0x00027000); };
        auto load_k = [&](const Tile (&t)[TILES]) {
            if constexpr (TYPE == FHIP_Q8_0) {
#pragma unroll
                for (int i = 0; i < TILES; i++) {
                    const auto scales = tile_bytes(kv.k_scales, t[i].at >> 5 << 1), base = tile_bytes(kv.k, t[i].at);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        if constexpr (NB == 4) {
                            const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(scales, d_off[r], 0, 0);
                            kd[i][r][0] = w.x; kd[i][r][1] = w.y;
                        } else {
                            kd[i][r][0] = __builtin_amdgcn_raw_buffer_load_b32(scales, d_off[r], 0, 0);
                        }
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(base, k_off + 32 * b, 0, 0);
                        kr[i][2 * b] = w.x; kr[i][2 * b + 1] = w.y;
                    }
                }
            } else {
                // (the parts of both tiles in turn, as the products take them)
                __amdgpu_buffer_rsrc_t base[TILES];
#pragma unroll
                for (int i = 0; i < TILES; i++) base[i] = tile_bytes(kv.k, t[i].at * Elem<TYPE>::BYTES);
#pragma unroll
                for (int b = 0; b < KW; b++)
#pragma unroll
                    for (int i = 0; i < TILES; i++) {
                        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(base[i], k_off + 64 * b, 0, 0);
                        kr[i][4 * b] = w.x; kr[i][4 * b + 1] = w.y; kr[i][4 * b + 2] = w.z; kr[i][4 * b + 3] = w.w;
                    }
            }
        };
        auto load_v = [&](const Tile (&t)[TILES]) {
#pragma unroll
            for (int i = 0; i < TILES; i++) {
                const auto base = tile_bytes(kv.v, t[i].at * Elem<TYPE>::BYTES);
                const auto scales = tile_bytes(TYPE == FHIP_Q8_0 ? (const void*)kv.v_scales : kv.v, t[i].at >> 5 << 1);
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    if constexpr (TYPE == FHIP_F32) {
#pragma unroll
                        for (int h = 0; h < HD / 64; h++) {
                            const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(base, v_off[r] + 256 * h, 0, 0);
                            vr[i][r][4 * h] = w.x; vr[i][r][4 * h + 1] = w.y; vr[i][r][4 * h + 2] = w.z; vr[i][r][4 * h + 3] = w.w;
                        }
                    } else if constexpr (VB == 16) {
                        const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(base, v_off[r], 0, 0);
                        vr[i][r][0] = w.x; vr[i][r][1] = w.y; vr[i][r][2] = w.z; vr[i][r][3] = w.w;
                    } else if constexpr (VB == 8) {
                        const u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(base, v_off[r], 0, 0);
                        vr[i][r][0] = w.x; vr[i][r][1] = w.y;
                    } else {
                        vr[i][r][0] = __builtin_amdgcn_raw_buffer_load_b32(base, v_off[r], 0, 0);
                    }
                    if constexpr (TYPE == FHIP_Q8_0) vd[i][r] = __builtin_amdgcn_raw_buffer_load_b16(scales, d_off[r] + 2 * (n / (16 / NB)), 0, 0);
                }
            }
        };

        // the unit's queries, as the second operand of K q^T
        f32x4 raw[NJ];
        f32x4 qf[P::HALF ? 1 : NJ];
        Frag qp[P::HALF ? NB : 1][P::HALF ? PARTS : 1];
        auto load_q = [&] {
            const float* qh = a.q + ((size_t)seq * a.n_head + head * g + (n < g ? n : 0)) * HD;
#pragma unroll
            for (int i = 0; i < NJ; i++) raw[i] = *(const f32x4*)(qh + (P::HALF ? 32 * (i / 2) + 8 * kg + 4 * (i & 1) : 16 * i + 4 * kg));
        };
        auto take_q = [&] {
#pragma unroll
            for (int i = 0; i < NJ; i++)
                if (n >= g) raw[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if constexpr (!P::HALF) {
#pragma unroll
                for (int i = 0; i < NJ; i++) qf[i] = raw[i];
            } else {
                float up = 1.f;
                if constexpr (TYPE != FHIP_BF16) {     // the head's largest |q| to [2^14, 2^15)
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < NJ; i++)
#pragma unroll
                        for (int x = 0; x < 4; x++) top = fmaxf(top, fabsf(raw[i][x]));
                    top = column_max(top);
                    const int ex = top > 0.f && top < INFINITY ? 14 - (int)(((__float_as_uint(top) >> 23) & 255u) - 127u) : 0;
                    const int clipped = ex < -126 ? -126 : ex > 126 ? 126 : ex;
                    up = __uint_as_float((uint32_t)(127 + clipped) << 23);
                    c2 *= __uint_as_float((uint32_t)(127 - clipped) << 23);
                }
#pragma unroll
                for (int i = 0; i < NB; i++)
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        uint32_t w[3];
                        cut<TYPE == FHIP_BF16>(raw[2 * i + x / 2][2 * (x & 1)] * up, raw[2 * i + x / 2][2 * (x & 1) + 1] * up, w);
#pragma unroll
                        for (int p = 0; p < PARTS; p++) qp[i][p].w[x] = w[p];
                    }
            }
        };
        // A step, and what it requests of the next one: as two copies, since a request under a condition would be waited for wherever the other path could come from.
        auto work = [&](uint32_t k, auto more) {
            // scores of the step's keys
            f32x4 s[TILES];
#pragma unroll
            for (int i = 0; i < TILES; i++) s[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if constexpr (TYPE == FHIP_F32) {
                f32x4 s2 = (f32x4){0.f, 0.f, 0.f, 0.f};      // two chains: half of the products' latency
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        f32x4& t = e & 1 ? s2 : s[0];
                        t = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[0][4 * j + e]), qf[j][e], t, 0, 0, 0);
                    }
                s[0] += s2;
            } else if constexpr (TYPE == FHIP_Q8_0) {
#pragma unroll
                for (int i = 0; i < TILES; i++)
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        Frag f;                       // eight codes
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint32_t w = kr[i][2 * b + e] ^ 0x80808080u;
                            f.w[2 * e] = codes_f16(w, 0x04010400u);
                            f.w[2 * e + 1] = codes_f16(w, 0x04030402u);
                        }
                        f32x4 t = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int p = PARTS - 1; p >= 0; p--) t = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h, qp[b][p].h, t, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const f16x2 d = __builtin_bit_cast(f16x2, kd[i][r][b / 2]);
                            s[i][r] = fmaf(t[r], (float)(b & 1 ? d.y : d.x), s[i][r]);
                        }
                    }
            } else {
                // the small parts of q first: each chunk's products as its keys come in
#pragma unroll
                for (int b = 0; b < NB; b++)
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; p--)
#pragma unroll
                        for (int i = 0; i < TILES; i++) {
                            Frag f;
#pragma unroll
                            for (int e = 0; e < 4; e++) f.w[e] = kr[i][4 * b + e];
                            if constexpr (TYPE == FHIP_BF16) s[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.b, qp[b][p].b, s[i], 0, 0, 0);
                            else s[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h, qp[b][p].h, s[i], 0, 0, 0);
                        }
            }
            if constexpr (more()) {
                if ((k + 1) % IDS == 0) look_up(k + 1);
                find(k + 1, nxt);
                load_k(nxt);
            }
            // softmax: in units of log2; keys that do not count have no weight, and their values, which may be no numbers, are zero
            if (a.softcap > 0.f) {
#pragma unroll
                for (int i = 0; i < TILES; i++) s[i] = tanh4(s[i] * c2) * (a.softcap * LOG2E);
            } else {
#pragma unroll
                for (int i = 0; i < TILES; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s[i][r] *= c2;
            }
            float least = INFINITY;                   // of the keys that count
#pragma unroll
            for (int i = 0; i < TILES; i++)
                if (cur[i].pos == NO_PAGE || cur[i].pos + 16 > sp.len || cur[i].pos < sp.lo) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t key = cur[i].pos + 4 * kg + r;
                        if (cur[i].pos == NO_PAGE || key >= sp.len || key < sp.lo) {
                            s[i][r] = -INFINITY;
                            if constexpr (TYPE == FHIP_Q8_0) vd[i][r] = 0;      // (codes are numbers whatever lies there)
                            else
#pragma unroll
                                for (int e = 0; e < VW; e++) vr[i][r][e] = 0;
                        } else {
                            least = fminf(least, s[i][r]);
                        }
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 4; r++) least = fminf(least, s[i][r]);
                }
            float top = s[0][0];
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) top = fmaxf(top, s[i][r]);
            top = column_max(top);
            if (__any(top > m)) {                     // a new maximum in some column
                const float now = fmaxf(top, m), f = now == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - now);
                m = now;
                l *= f;
#pragma unroll
                for (int j = 0; j < NJ; j++) acc[j] *= f;
            }
            const float base = m == -INFINITY ? 0.f : m;
            float p[TILES][4];
#pragma unroll
            for (int i = 0; i < TILES; i++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    p[i][r] = __builtin_amdgcn_exp2f(s[i][r] - base);
                    l += p[i][r];
                }
            // weighted rows
            if constexpr (P::HALF) {
                // weights as so many 16-bit values each
                auto cut_weights = [&](auto bf, auto& pp) {
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        uint32_t w[3];
                        cut<bf()>(p[x / 2][2 * (x & 1)] * P::UP, p[x / 2][2 * (x & 1) + 1] * P::UP, w);
#pragma unroll
                        for (int e = 0; e < (int)(sizeof(pp) / sizeof(Frag)); e++) pp[e].w[x] = w[e];
                    }
                };
                uint64_t beyond = 0;                         // lanes with something that two f16 values do not hold:
                uint32_t d2[TYPE == FHIP_Q8_0 ? 4 : 1];      // Q8_0: the scales of keys 2 x and 2 x + 1 in the lane's order
                if constexpr (TYPE != FHIP_BF16) {
                    bool here = least - base < -18.f;        // a weight below 2^-18, whose second part would be smaller than f16's 2^-14, or
                    if constexpr (TYPE == FHIP_Q8_0) {
                        u16x2 most = {0, 0};
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            d2[x] = (uint32_t)vd[x / 2][2 * (x & 1)] | (uint32_t)vd[x / 2][2 * (x & 1) + 1] << 16;
                            most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, d2[x]));
                        }
                        here |= most.x > 0x5FFFu || most.y > 0x5FFFu;      // the values of a scale of 512 and more (or no number)
                    }
                    beyond = __ballot(here);
                    if (beyond) {
                        // weights as three bf16 values each, values as two (f16) or three: all of their products but that of the smallest of three (2^-30 of the whole)
                        constexpr int VALUE_PARTS = TYPE == FHIP_Q8_0 ? 3 : 2;
                        Frag pp[3];
                        cut_weights(std::true_type(), pp);
#pragma unroll
                        for (int j = 0; j < NJ; j++) {
                            float v[8];               // of the lane's keys
#pragma unroll
                            for (int e = 0; e < 8; e++) {
                                if constexpr (TYPE == FHIP_Q8_0) {
                                    const f16x2 d = __builtin_bit_cast(f16x2, d2[e / 2]);
                                    v[e] = (float)(int8_t)(vr[e / 4][e % 4][j / 4] >> 8 * (j % 4)) * (float)(e & 1 ? d.y : d.x);
                                } else {
                                    // (of a vector's two the compiler would keep both, for every row: 49 registers spilled)
                                    v[e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(vr[e / 4][e % 4][j / 2] >> 16 * (j & 1)));
                                }
                            }
#pragma unroll
                            for (int b = 0; b < VALUE_PARTS; b++) {
                                Frag f;
#pragma unroll
                                for (int x = 0; x < 4; x++) f.w[x] = upper_halves(__float_as_uint(v[2 * x]), __float_as_uint(v[2 * x + 1]));
#pragma unroll
                                for (int e = b < 2 ? 2 : 1; e >= 0; e--) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.b, pp[e].b, acc[j], 0, 0, 0);
#pragma unroll
                                for (int e = 0; e < 8; e++) v[e] -= __uint_as_float(__float_as_uint(v[e]) & 0xFFFF0000u);
                            }
                        }
                    }
                    // (two branches: of one with two ways the compiler keeps a set of accumulators each, which costs heads of 64 the third wave of a SIMD)
                    asm volatile("" : "+s"(beyond));
                }
                if (!beyond) {
                    Frag pp[PARTS];
                    cut_weights(std::integral_constant<bool, TYPE == FHIP_BF16>(), pp);
#pragma unroll
                    for (int j = 0; j < NJ; j++) {
                        Frag f, lo;
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const int i = x / 2, r = 2 * (x & 1);
                            if constexpr (TYPE == FHIP_Q8_0) {
                                // values j of two keys: c * d = f + lo, exactly
                                const uint32_t both = __builtin_amdgcn_perm(vr[i][r + 1][j / 4] ^ 0x80808080u, vr[i][r][j / 4] ^ 0x80808080u, (uint32_t)(j % 4) | (uint32_t)(4 + j % 4) << 16 | 0x0C000C00u);
                                const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
                                const f16x2 c = __builtin_bit_cast(f16x2, both | 0x64006400u) - off, d = __builtin_bit_cast(f16x2, d2[x]);
                                const f16x2 hi = c * d;
                                f.w[x] = __builtin_bit_cast(uint32_t, hi);
                                lo.w[x] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(c, d, -hi));
                            } else {
                                const uint32_t u = vr[i][r][j / 2], w = vr[i][r + 1][j / 2];
                                f.w[x] = j & 1 ? upper_halves(u, w) : lower_halves(u, w);
                            }
                        }
                        if constexpr (TYPE == FHIP_Q8_0) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(lo.h, pp[0].h, acc[j], 0, 0, 0);
#pragma unroll
                        for (int e = PARTS - 1; e >= 0; e--) {
                            if constexpr (TYPE == FHIP_BF16) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f.b, pp[e].b, acc[j], 0, 0, 0);
                            else acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h, pp[e].h, acc[j], 0, 0, 0);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int j = 0; j < NJ; j++) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[0][r][j]), p[0][r], acc[j], 0, 0, 0);
            }
            if constexpr (more()) {
                load_v(nxt);
#pragma unroll
                for (int i = 0; i < TILES; i++) cur[i] = nxt[i];
            }
        };
        if (mine > 0) {
            load_q();
            look_up(0);
            find(0, cur);
            load_k(cur);
            __builtin_amdgcn_sched_barrier(0);        // in the loop's order: the wait for the first keys is not one for the values
            load_v(cur);
            __builtin_amdgcn_sched_barrier(0);
            take_q();
            for (uint32_t k = 0; k + 1 < mine; k++) work(k, std::true_type());
            work(mine - 1, std::false_type());
        }
        if constexpr (P::UP != 1.f) {
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[j] *= 1.f / P::UP;
        }

        // the waves' shares joined; element r of acc[j] is dim dim_of(j, 4 kg + r) of head n
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if (kg == 0) { sm_m[wave][n] = m; sm_l[wave][n] = l; }
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int j = 0; j < NJ; j += 4) {
                const int d = TYPE == FHIP_F32 ? 16 * j + 4 * (4 * kg + r) : NJ * (4 * kg + r) + j;
                *(f32x4*)&sm_o[wave][n][d] = (f32x4){acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
            }
        __syncthreads();
        float* part = whole ? nullptr : a.part + ((size_t)place * 2 + shares) * g * (HD + 4);
        if (a.log_wgs >= 0 && from == 0 && threadIdx.x == 0) {       // the unit's first steps are here: who has the others
            const uint32_t last = whole ? place : (unit0 + unit_cost(sp.steps) - 1) / each;
            a.plan[seq * kv.n_kv + head] = place | last << 15 | shares << 30;
        }
        shares += !whole;
        for (int e = threadIdx.x; e < g * (HD / 4); e += 64 * WV) {
            const int h = e / (HD / 4), d = 4 * (e % (HD / 4));
            float top = sm_m[0][h], sum = 0.f;
#pragma unroll
            for (int w = 1; w < WV; w++) top = fmaxf(top, sm_m[w][h]);
            const float base = top == -INFINITY ? 0.f : top;
            f32x4 o = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WV; w++) {
                const float f = __builtin_amdgcn_exp2f(sm_m[w][h] - base);
                sum = fmaf(sm_l[w][h], f, sum);
                o += *(const f32x4*)&sm_o[w][h][d] * f;
            }
            if (whole) {
                const float inv = top == -INFINITY && sum == 0.f ? 0.f : 1.f / sum;      // nothing to attend to: zeros
                *(f32x4*)(a.out + ((size_t)seq * a.n_head + head * g + h) * HD + d) = o * inv;
            } else {
                *(f32x4*)(part + h * HD + d) = o;
                if (d == 0) { part[g * HD + 2 * h] = top; part[g * HD + 2 * h + 1] = sum; }
            }
        }
        if (a.log_wgs < 0 || !next_unit()) return;
        __syncthreads();
    }
}

// What the workgroups of a unit that was cut have left, added in their order; zeros for a unit without keys. A workgroup a query head.
template <int TYPE, int HD, bool SEL>
__global__ __launch_bounds__(256) void join_kernel(Attend a) {
    constexpr int LANES = HD / 4, GROUPS = 256 / LANES;
    __shared__ float sm_m[GROUPS], sm_l[GROUPS];
    __shared__ __attribute__((aligned(16))) float sm_o[GROUPS][HD];
    const PagedView& kv = a.kv;
    const int g = a.n_head / kv.n_kv;
    const uint32_t seq = blockIdx.x / a.n_head, qh = blockIdx.x % a.n_head, head = qh / g, h = qh % g;
    const uint32_t plan = a.plan[seq * kv.n_kv + head];      // (of nobody's making for a unit without steps)
    const Span sp = span_of<TYPE, SEL>(kv, a.lens, seq, a.max_len, a.window, a.n_select);
    float* out = a.out + ((size_t)seq * a.n_head + qh) * HD;
    if (sp.steps == 0) {
        if (threadIdx.x < HD) out[threadIdx.x] = 0.f;
        return;
    }
    const uint32_t wgs = (1u << a.log_wgs) - 1, w0 = plan & wgs, w1 = plan >> 15 & wgs, second = plan >> 30 & 1;      // (within the workspace whatever it holds)
    if (w0 == w1) return;                             // finished where it was
    auto part = [&](uint32_t w) { return a.part + ((size_t)w * 2 + (w == w0 ? second : 0)) * g * (HD + 4); };
    // a group of threads takes every GROUPS-th share; its maximum as it goes
    const int group = threadIdx.x / LANES, d = 4 * (threadIdx.x % LANES);
    f32x4 o = (f32x4){0.f, 0.f, 0.f, 0.f};
    float top = -INFINITY, sum = 0.f;
    for (uint32_t w = w0 + group; w <= w1; w += 4 * GROUPS) {      // four shares requested together
        float m[4], l[4];
        f32x4 v[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const uint32_t at = w + e * GROUPS;
            const float* p = part(at <= w1 ? at : w);
            m[e] = at <= w1 ? p[g * HD + 2 * h] : -INFINITY;
            l[e] = p[g * HD + 2 * h + 1];
            v[e] = *(const f32x4*)(p + h * HD + d);
        }
        float now = top;
#pragma unroll
        for (int e = 0; e < 4; e++) now = fmaxf(now, m[e]);
        const float base = now == -INFINITY ? 0.f : now, f0 = __builtin_amdgcn_exp2f(top - base);
        o *= f0;
        sum *= f0;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float f = w + e * GROUPS <= w1 ? __builtin_amdgcn_exp2f(m[e] - base) : 0.f;
            o += w + e * GROUPS <= w1 ? v[e] * f : (f32x4){0.f, 0.f, 0.f, 0.f};
            sum += w + e * GROUPS <= w1 ? l[e] * f : 0.f;
        }
        top = now;
    }
    *(f32x4*)&sm_o[group][d] = o;
    if (d == 0) { sm_m[group] = top; sm_l[group] = sum; }
    __syncthreads();
    if (threadIdx.x < HD) {
        float all = sm_m[0], v = 0.f, t = 0.f;
#pragma unroll
        for (int i = 1; i < GROUPS; i++) all = fmaxf(all, sm_m[i]);
        const float base = all == -INFINITY ? 0.f : all;
#pragma unroll
        for (int i = 0; i < GROUPS; i++) {
            const float f = __builtin_amdgcn_exp2f(sm_m[i] - base);
            v = fmaf(sm_o[i][threadIdx.x], f, v);
            t = fmaf(sm_l[i], f, t);
        }
        out[threadIdx.x] = all == -INFINITY && t == 0.f ? 0.f : v / t;
    }
}

template <typename Go>
int by_type(uint32_t type, Go go) {
    switch (type) {
        case FHIP_F32: return go(std::integral_constant<int, FHIP_F32>());
        case FHIP_F16: return go(std::integral_constant<int, FHIP_F16>());
        case FHIP_BF16: return go(std::integral_constant<int, FHIP_BF16>());
        default: return go(std::integral_constant<int, FHIP_Q8_0>());
    }
}

}  // namespace

namespace fhip {

int launch_paged_append(uint32_t type, int hd, const PagedView& kv, const PagedPost& p, hipStream_t s) {
    const size_t slices = ((size_t)(p.n_head + 2 * kv.n_kv) * hd + 127) / 128;
    // Few slices go one to a wave. From eight for each of 2048 waves on a wave takes a token's, or as many of them (eight and more) as leave MANY_WAVES. us: 999 tokens of 144
    // heads of 64 25.0 with a slice a wave, 19.8 so; 1200 of 56 of 128 with 4096 waves 19.2, with 16384 16.6.
    constexpr size_t MANY_WAVES = 16384;
    const bool many = p.t * slices >= 8 * 2048;
    const size_t most = (slices + 7) / 8, parts = many ? (p.t >= MANY_WAVES ? 1 : MANY_WAVES / p.t < most ? MANY_WAVES / p.t : most) : 1;
    const int each = many ? (int)((slices + parts - 1) / parts) : 1;
    const dim3 grid(many ? (p.t + 3) / 4 : p.t, many ? (unsigned)parts : (unsigned)((slices + 3) / 4));
    return by_type(type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, kv, p, each); };
        if (hd == 128) many ? go(append_kernel<TYPE, 128, 4>) : go(append_kernel<TYPE, 128, 1>);
        else many ? go(append_kernel<TYPE, 64, 4>) : go(append_kernel<TYPE, 64, 1>);
        return check_hip(hipGetLastError(), "paged_append launch");
    });
}

int launch_paged_rows(uint32_t type, int hd, const PagedView& kv, uint32_t seq, size_t row0, size_t rows, float* k_out, float* v_out, hipStream_t s) {
    const size_t width4 = (size_t)kv.n_kv * hd / 4, grid = (rows * width4 + 255) / 256;
    if (grid > 0xFFFFFFull) return set_error(FHIP_ERR_SHAPE, "fhip_paged_rows: too many rows for one launch");      // 2^32 threads
    return by_type(type, [&](auto ty) {
        hipLaunchKernelGGL((rows_kernel<decltype(ty)::value>), dim3((unsigned)grid, 2), dim3(256), 0, s, kv, (uint32_t)width4, seq, row0, rows, k_out, v_out);
        return check_hip(hipGetLastError(), "paged_rows launch");
    });
}

int launch_paged_key_bounds(uint32_t type, int hd, const PagedView& kv, const uint32_t* lens, const uint32_t* fresh, uint32_t max_new, float* bounds, hipStream_t s) {
    const uint32_t R = 1u << kv.shift;
    uint64_t pages = ((uint64_t)max_new + R - 2) / R + 1;            // that `max_new` rows can touch
    if (pages > kv.pages_per_seq) pages = kv.pages_per_seq;
    return by_type(type, [&](auto ty) {
        hipLaunchKernelGGL((bounds_kernel<decltype(ty)::value>), dim3(kv.n_seq * kv.n_kv, (unsigned)(pages < 65535 ? pages : 65535)), dim3(hd), 0, s, kv, hd, lens, fresh, max_new, bounds);
        return check_hip(hipGetLastError(), "paged_key_bounds launch");
    });
}

static uint32_t pages_at_most(const PagedView& kv, size_t max_len) {
    const size_t pages = (max_len + ((size_t)1 << kv.shift) - 1) >> kv.shift;
    return pages < kv.pages_per_seq ? (uint32_t)pages : kv.pages_per_seq;
}
size_t paged_select_ws_bytes(const PagedView& kv, size_t max_len) { return (size_t)kv.n_seq * kv.n_kv * pages_at_most(kv, max_len) * 8; }
int launch_paged_select(int hd, const PagedView& kv, const float* q, const uint32_t* lens, uint32_t max_len, const float* bounds, int n_head, uint32_t n_select,
                        uint32_t first, uint32_t last, void* ws, uint32_t* out, hipStream_t s) {
    const uint32_t pages = pages_at_most(kv, max_len);
    if (pages > 0) {
        const dim3 grid((pages + 63) / 64, kv.n_kv, kv.n_seq);
        const int calls = (n_head / kv.n_kv + 3) / 4;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, s, kv, q, lens, max_len, bounds, n_head, first, last, (uint64_t*)ws, pages); };
        if (hd == 128) calls == 1 ? go(score_kernel<128, 1>) : calls == 2 ? go(score_kernel<128, 2>) : calls == 3 ? go(score_kernel<128, 3>) : go(score_kernel<128, 4>);
        else calls == 1 ? go(score_kernel<64, 1>) : calls == 2 ? go(score_kernel<64, 2>) : calls == 3 ? go(score_kernel<64, 3>) : go(score_kernel<64, 4>);
    }
    const dim3 lists(kv.n_seq * kv.n_kv);
    auto go = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, lists, dim3(threads), 0, s, kv, lens, max_len, n_select, (const uint64_t*)ws, pages, first + last, out);
    };
    if (pages <= 256 * SEL_HELD) go(select_kernel<256, SEL_HELD>, 256);
    else if (pages <= 1024 * SEL_HELD) go(select_kernel<1024, SEL_HELD>, 1024);
    else go(select_kernel<1024, 0>, 1024);
    return check_hip(hipGetLastError(), "paged_select launch");
}

// Workgroups that the steps are dealt out to, two for each of the chip's 256 CUs.
constexpr int LOG_WGS = 9, MIN_STEPS = 6;
// Whether every unit has a workgroup of its own and nothing is joined: up to four steps for each of its waves; of more units than there are workgroups otherwise up to sixteen, which even
// a single long sequence among short ones walks through in less time than the others' bytes take. us, own | dealt out, heads of 128: bf16 1 sequence of 400 keys and 8 KV heads 8.2 | 9.8, 32 of 400 12.6 | 18.5,
// 64 of 500 28.6 | 33.2, 64 of 2000 97.9 | 103, but 8 of 2000 24.5 | 20.1.
static bool own_workgroups(uint32_t type, const PagedView& kv, size_t keys) {
    const size_t steps = (keys + (type == FHIP_F32 ? 15 : 31)) / (type == FHIP_F32 ? 16 : 32);
    return steps <= 16 || ((size_t)kv.n_seq * kv.n_kv >= ((size_t)1 << LOG_WGS) && steps <= 64);
}
// The deal counts in 32 bits.
static bool too_many_steps(uint32_t type, const PagedView& kv, size_t keys) {
    return (keys / (type == FHIP_F32 ? 16 : 32) + 1 + UNIT_COST) * kv.n_seq * kv.n_kv >= (size_t)1 << 31;
}
// The bound on a sequence's keys, which may be anything, as far as the table reaches.
static size_t within_table(const PagedView& kv, size_t keys) { return keys < (size_t)kv.pages_per_seq << kv.shift ? keys : (size_t)kv.pages_per_seq << kv.shift; }
static size_t plan_floats(const PagedView& kv) { return ((size_t)kv.n_seq * kv.n_kv + 3) / 4 * 4; }
// (of a bound with too many steps as of any other: what a bound needs is enough for every smaller one)
size_t paged_attention_ws_bytes(uint32_t type, const PagedView& kv, int hd, int n_head, size_t max_len) {
    return own_workgroups(type, kv, within_table(kv, max_len)) ? 0 : (plan_floats(kv) + ((size_t)2 << LOG_WGS) * (n_head / kv.n_kv) * (hd + 4)) * sizeof(float);
}
int launch_paged_attention(uint32_t type, int hd, const PagedView& kv, const float* q, const uint32_t* lens, uint32_t max_len, const uint32_t* selected, uint32_t n_select,
                           int n_head, uint32_t window, float softcap, float* ws, float* out, hipStream_t s) {
    const size_t units = (size_t)kv.n_seq * kv.n_kv;
    const size_t bound = within_table(kv, selected ? (size_t)n_select << kv.shift : max_len);
    size_t keys = bound;
    if (window > 0 && (size_t)window + 31 < keys) keys = (size_t)window + 31;      // a window begins and ends within steps
    Attend a;
    a.kv = kv; a.q = q; a.lens = lens; a.selected = selected; a.out = out; a.plan = (uint32_t*)ws; a.part = ws + plan_floats(kv);
    a.max_len = max_len; a.n_select = n_select; a.window = window; a.n_head = n_head; a.softcap = softcap; a.scale = 1.0f / sqrtf((float)hd);
    a.log_wgs = own_workgroups(type, kv, keys) || own_workgroups(type, kv, bound) || too_many_steps(type, kv, keys) ? -1 : LOG_WGS;      // (the second: the caller may have no workspace)
    a.min_steps = MIN_STEPS;
    const bool alone = a.log_wgs < 0 && units > 4 * (size_t)device_cus();      // more units than the chip has waves for by fours: a wave each
    const dim3 grid(a.log_wgs < 0 ? (unsigned)units : 1u << LOG_WGS);
    return by_type(type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        auto go = [&](auto dims, auto sel) {
            constexpr int HD = decltype(dims)::value;
            constexpr bool SEL = decltype(sel)::value;
            if (alone) hipLaunchKernelGGL((attention_kernel<TYPE, HD, SEL, 1>), grid, dim3(64), 0, s, a);
            else hipLaunchKernelGGL((attention_kernel<TYPE, HD, SEL, 4>), grid, dim3(256), 0, s, a);
            if (a.log_wgs >= 0) hipLaunchKernelGGL((join_kernel<TYPE, HD, SEL>), dim3(kv.n_seq * (unsigned)n_head), dim3(256), 0, s, a);
        };
        auto at = [&](auto sel) { hd == 128 ? go(std::integral_constant<int, 128>(), sel) : go(std::integral_constant<int, 64>(), sel); };
        selected ? at(std::true_type()) : at(std::false_type());
        return check_hip(hipGetLastError(), "paged_attention launch");
    });
}

}  // namespace fhip
