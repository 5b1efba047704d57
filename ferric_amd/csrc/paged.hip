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
typedef double f64x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t NO_PAGE = 0xFFFFFFFFu;

template <int TYPE>
struct Elem {
    static constexpr int BYTES = TYPE == FHIP_F32 ? 4 : TYPE == FHIP_Q8_0 ? 1 : 2;
};

__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
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
__device__ __forceinline__ double dpp(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xF, 0xF, false), hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xF, 0xF, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// over the 16 lanes of a row, in all of them
template <typename T, typename Op>
__device__ __forceinline__ T row16(T v, Op op) {
    v = op(v, dpp<0xB1>(v));    // quad_perm [1,0,3,2]
    v = op(v, dpp<0x4E>(v));    // quad_perm [2,3,0,1]
    v = op(v, dpp<0x141>(v));   // row_half_mirror
    return op(v, dpp<0x140>(v));   // row_mirror
}

// ---------------------------------------------------------------- storing the rows of new tokens
// Row i of the fused projection: + bias, RMS norm of query and key heads, rotation, queries to q_out, keys and values to the row of their page, rounded once.
// The angle pos * base^(-2c / n_rot) is formed in f64, in turns, and only its fraction of a turn is rounded to f32: the f32 product that the contiguous
// caches' post-processing forms is 4e-3 rad off at position 100 000.
// A lane holds two neighbouring dims, so a wave holds 128 values (a slice): one head of 128 or two of 64. TOK tokens a workgroup: with 4 a wave has a
// token to itself and the f64 work of its angles is shared by all of the token's heads; with 1 the waves share a token's slices.
template <int TYPE, int HD, int TOK>
__global__ __launch_bounds__(256) void append_kernel(PagedView kv, PagedPost p, int slices_per_wave) {
    constexpr int LPH = HD / 2;                       // lanes of a head
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
    const bool odd = !p.interleaved && (half & 1);    // partners of a lane's two dims in two lanes
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
    for (int s = s0; s < s0 + slices_per_wave && s < slices; s++) {
        const int h = s * (128 / HD) + lane / LPH;    // with heads of 64 the last slice may hold one head only
        const bool live = h < per_tok;
        const bool is_q = h < p.n_head, is_k = !is_q && h < p.n_head + kv.n_kv;
        float2 v = live ? *(const float2*)(x + (size_t)h * HD + j0) : make_float2(0.f, 0.f);
        if (p.bias && live) {
            const float2 b = *(const float2*)(p.bias + (size_t)h * HD + j0);
            v.x += b.x;
            v.y += b.y;
        }
        const float* nw = is_q ? p.q_norm : is_k ? p.k_norm : nullptr;
        float sq = fmaf(v.x, v.x, v.y * v.y);
        sq = row16(sq, [](float a, float b) { return a + b; });
        sq += __shfl_xor(sq, 16);
        if (HD == 128) sq += __shfl_xor(sq, 32);
        if (nw) {
            const float inv = 1.0f / sqrtf(sq / (float)HD + p.eps);
            const float2 w = *(const float2*)(nw + j0);
            v.x = v.x * inv * w.x;
            v.y = v.y * inv * w.y;
        }
        float2 r = v;
        if (p.interleaved) {
            r.x = fmaf(v.x, t0.x, -(v.y * t0.y));
            r.y = fmaf(v.y, t0.x, v.x * t0.y);
        } else if (half > 0) {
            float ox, oy;
            if (odd) {                                // the partner of dim j is dim j +- half, of the other parity
                const int d = j0 < half ? half : -half, d1 = j0 + 1 < half ? half : -half, base = lane - lane % LPH;
                const int f0 = base + (((j0 + d) >> 1) & (LPH - 1)), f1 = base + (((j0 + 1 + d1) >> 1) & (LPH - 1));
                ox = __shfl(v.y, f0);
                oy = __shfl(v.x, f1);
            } else {
                ox = __shfl(v.x, from);
                oy = __shfl(v.y, from);
            }
            if (j0 < p.n_rot) {
                r.x = fmaf(v.x, t0.x, -(ox * t0.y));
                r.y = fmaf(v.y, t1.x, -(oy * t1.y));
            }
        }
        if (is_q || is_k) v = r;
        if (!live) continue;
        if (is_q) {
            *(float2*)(p.q_out + ((size_t)i * p.n_head + h) * HD + j0) = v;
            continue;
        }
        const size_t at = (row * kv.n_kv + (h - p.n_head - (is_k ? 0 : kv.n_kv))) * HD + j0;
        void* pool = is_k ? kv.k : kv.v;
        if constexpr (TYPE == FHIP_F32) {
            if (placed) *(float2*)((float*)pool + at) = v;
        } else if constexpr (TYPE == FHIP_BF16) {
            if (placed) *(uint32_t*)((uint16_t*)pool + at) = pack_bf16(v.x, v.y);
        } else if constexpr (TYPE == FHIP_F16) {
            if (placed) *(uint32_t*)((uint16_t*)pool + at) = pack_f16(v.x, v.y);
        } else {
#pragma clang fp contract(off)
            // a block is the 16 lanes of a row: d = amax / 127, codes round(v / d) half away from zero, as fhip_kvq_append's
            const float amax = row16(fmaxf(fmaxf(0.f, fabsf(v.x)), fabsf(v.y)), [](float a, float b) { return fmaxf(a, b); });
            const float d = amax / 127.0f, inv = d > 0.f ? 1.0f / d : 0.f;
            auto code = [&](float y) {
                const float t = y * inv, q = copysignf(floorf(fabsf(t) + 0.5f), t);
                return q != q ? 0 : (int)fminf(fmaxf(q, -127.0f), 127.0f);
            };
            if (placed) {
                *(uint16_t*)((uint8_t*)pool + at) = (uint16_t)((code(v.x) & 255) | (code(v.y) & 255) << 8);
                if ((lane & 15) == 0) (is_k ? kv.k_scales : kv.v_scales)[at >> 5] = __half_as_ushort(__float2half_rn(d));
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
    const uint32_t entry = ((len - n) >> kv.shift) + blockIdx.y;
    if (entry > (len - 1) >> kv.shift) return;
    const uint32_t page = kv.table[seq * kv.table_stride + entry];
    if (page >= kv.n_pages) return;
    const uint32_t start = entry << kv.shift, from = start > len - n ? start : len - n, to = len - start < R ? len : start + R;
    const int d = threadIdx.x;
    float* b = bounds + ((size_t)page * kv.n_kv + head) * 2 * hd + d;
    float lo = from == start ? INFINITY : b[0], hi = from == start ? -INFINITY : b[hd];
    bool nan = lo != lo || hi != hi;
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

// ---------------------------------------------------------------- the choice of pages
// score(page, kv head) = max over its query heads of sum_d max(q_d lo_d, q_d hi_d), the largest product with q that a key within the bounds can have. In f64: the order of
// pages whose scores are next to each other decides what is attended to, and f32 sums would decide it by the order of their additions. As a product: max(q lo, q hi)
// = max(q, 0) hi + min(q, 0) lo. Keys are ordered as unsigned words; a page that is always kept has the largest, a score that is no number the next.
__device__ __forceinline__ uint64_t order_key(double v) {
    if (v != v) return ~0ull - 1;
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return b >> 63 ? ~b : b | 1ull << 63;
}
template <int HD>
__global__ __launch_bounds__(256) void score_kernel(PagedView kv, const float* __restrict__ q, const uint32_t* __restrict__ lens, uint32_t max_len, const float* __restrict__ bounds,
                                                    int n_head, uint32_t first, uint32_t last, uint64_t* __restrict__ keys, uint32_t key_stride) {
    const int lane = threadIdx.x & 63, g = n_head / kv.n_kv, head = blockIdx.y;
    const uint32_t seq = blockIdx.z, pages = pages_of(kv, rows_of(kv, lens, seq, max_len));
    const uint32_t j = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (j >= pages) return;
    const uint32_t page = kv.table[seq * kv.table_stride + j];
    double best = -INFINITY;
    if (page < kv.n_pages) {
        const float* b = bounds + ((size_t)page * kv.n_kv + head) * 2 * HD;
        for (int e = 0; e < g; e++) {
            double s = 0;
            for (int d = lane; d < HD; d += 64) {
                const double x = q[((size_t)seq * n_head + head * g + e) * HD + d], u = x * (double)b[d], w = x * (double)b[HD + d];
                s += u > w || u != u ? u : w;
            }
            for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
            best = s > best || s != s ? s : best;
        }
    }
    if (lane == 0) keys[((size_t)seq * kv.n_kv + head) * key_stride + j] = j < first || j + last >= pages ? ~0ull : order_key(best);
}

// The n_select largest keys of a list, equal ones by their place, as ascending places. One workgroup a list. The key that the last chosen one has is found by counting: the
// interval that holds it is cut into 1024 by its width, and the one of these with it is the next interval.
constexpr int SEL_T = 512, SEL_BINS = 1024;
__global__ __launch_bounds__(SEL_T) void select_kernel(PagedView kv, const uint32_t* __restrict__ lens, uint32_t max_len, uint32_t n_select, const uint64_t* __restrict__ keys,
                                                       uint32_t key_stride, uint32_t kept, uint32_t* __restrict__ out) {
    __shared__ uint32_t hist[SEL_BINS], counts[2][SEL_T / 64];
    __shared__ uint64_t edge[2][SEL_T / 64];
    __shared__ uint32_t found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint32_t list = blockIdx.x, seq = list / kv.n_kv;
    const uint32_t n = pages_of(kv, rows_of(kv, lens, seq, max_len));
    keys += (size_t)list * key_stride;
    out += (size_t)list * n_select;
    if (n <= n_select) {
        for (uint32_t j = tid; j < n_select; j += SEL_T) out[j] = j < n ? j : NO_PAGE;
        return;
    }
    uint64_t lo = ~0ull, hi = 0;
    for (uint32_t j = tid; j < n; j += SEL_T) {
        const uint64_t k = keys[j];
        if (k == ~0ull) continue;                     // kept whatever its score
        lo = k < lo ? k : lo;
        hi = k > hi ? k : hi;
    }
    for (int o = 32; o; o >>= 1) {
        const uint64_t a = __shfl_xor((unsigned long long)lo, o), b = __shfl_xor((unsigned long long)hi, o);
        lo = a < lo ? a : lo;
        hi = b > hi ? b : hi;
    }
    if (lane == 0) { edge[0][wave] = lo; edge[1][wave] = hi; }
    __syncthreads();
    for (int w = 0; w < SEL_T / 64; w++) {
        lo = edge[0][w] < lo ? edge[0][w] : lo;
        hi = edge[1][w] > hi ? edge[1][w] : hi;
    }
    uint32_t want = n_select - kept;                  // of the keys within [lo, hi], the largest `want` are chosen; here n > n_select >= kept, so it holds some
    while (want > 0 && lo < hi) {
        const int shift = 64 - __builtin_clzll(hi - lo) > 10 ? 64 - __builtin_clzll(hi - lo) - 10 : 0;      // (hi - lo) >> shift < 1024
        for (int b = tid; b < SEL_BINS; b += SEL_T) hist[b] = 0;
        __syncthreads();
        for (uint32_t j = tid; j < n; j += SEL_T) {
            const uint64_t k = keys[j];
            if (k >= lo && k <= hi) atomicAdd(&hist[(uint32_t)((k - lo) >> shift)], 1u);
        }
        __syncthreads();
        if (wave == 0) {                              // a lane has 16 bins, the highest first
            uint32_t mine = 0;
            for (int b = 0; b < 16; b++) mine += hist[SEL_BINS - 1 - (16 * lane + b)];
            uint32_t upto = mine;
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t t = __shfl_up(upto, o);
                if (lane >= o) upto += t;
            }
            uint32_t above = upto - mine;
            if (above < want && upto >= want)
                for (int b = 0; b < 16; b++) {
                    const int bin = SEL_BINS - 1 - (16 * lane + b);
                    const uint32_t c = hist[bin];
                    if (above < want && above + c >= want) {
                        found[0] = (uint32_t)bin;
                        found[1] = want - above;
                    }
                    above += c;
                }
        }
        __syncthreads();
        const uint64_t bin = found[0];
        if (bin < (hi - lo) >> shift) hi = lo + ((bin + 1) << shift) - 1;
        lo += bin << shift;
        want = found[1];
        __syncthreads();
    }
    // places of the keys above it, and of the first `want` that equal it
    uint32_t done = 0, equal = 0;
    for (uint32_t j0 = 0; j0 < n; j0 += SEL_T) {
        const uint32_t j = j0 + tid;
        const uint64_t k = j < n ? keys[j] : 0;
        const bool same = j < n && k == lo && k != ~0ull;
        const uint64_t below = ((uint64_t)1 << lane) - 1, same_mask = __ballot(same);
        if (lane == 0) counts[0][wave] = __popcll(same_mask);
        __syncthreads();
        uint32_t rank = equal + __popcll(same_mask & below);
        for (int w = 0; w < wave; w++) rank += counts[0][w];
        const bool take = (j < n && (k == ~0ull || (want > 0 && k > lo))) || (same && rank < want);
        const uint64_t take_mask = __ballot(take);
        if (lane == 0) counts[1][wave] = __popcll(take_mask);
        __syncthreads();
        uint32_t at = done + __popcll(take_mask & below);
        for (int w = 0; w < wave; w++) at += counts[1][w];
        if (take) out[at] = j;
        for (int w = 0; w < SEL_T / 64; w++) {
            equal += counts[0][w];
            done += counts[1][w];
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- attention of one token of every sequence
// out[h] = sum_j softmax_j(q_h . K_j / sqrt(hd)) V_j over the rows of the sequence, the g query heads of a KV head together, on v_mfma_f32_16x16x4_f32: products of f32
// operands and sums in f32, whatever the rows are stored in. A wave takes 16 keys at a time. K q^T puts head n in lane n's column and keys 4 (lane / 16) + r in its four
// registers, which is where V^T p^T wants its second operand's four keys, one per instruction: nothing is exchanged between the products, and a head's running
// maximum and sum stay in its column's lanes. Lane (m, k = lane / 16) of the first operand holds four neighbouring dims of key m, or four of key 4 k + r for V: both products are
// indifferent to which dims an instruction takes as long as both operands agree, so all loads are of 16 neighbouring bytes.
// SEL: the rows of the listed pages instead of all.
constexpr int ATT_W = 4;
template <int TYPE, int HD, bool SEL>
__global__ __launch_bounds__(64 * ATT_W) void attention_kernel(PagedView kv, const float* __restrict__ q, const uint32_t* __restrict__ lens, uint32_t max_len,
                                                               const uint32_t* __restrict__ selected, uint32_t n_select, int n_head, uint32_t window, float softcap, float scale,
                                                               float* __restrict__ out) {
    constexpr int NI = HD / 16;
    __shared__ float sm_m[ATT_W][16], sm_l[ATT_W][16];
    __shared__ __attribute__((aligned(16))) float sm_o[ATT_W][16][HD + 4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, kg = lane >> 4;
    const int g = n_head / kv.n_kv, head = blockIdx.x % kv.n_kv;
    const uint32_t seq = blockIdx.x / kv.n_kv, R = 1u << kv.shift;
    const uint32_t len = rows_of(kv, lens, seq, max_len), lo = window && window < len ? len - window : 0;
    const uint32_t* table = kv.table + seq * kv.table_stride;
    const uint32_t* list = SEL ? selected + (size_t)blockIdx.x * n_select : nullptr;
    f32x4 qf[NI];
    const float* qh = q + ((size_t)seq * n_head + head * g + (n < g ? n : 0)) * HD;
#pragma unroll
    for (int i = 0; i < NI; i++) {
        qf[i] = *(const f32x4*)(qh + 16 * i + 4 * kg);
        if (n >= g) qf[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
    f32x4 acc[NI];                                    // acc[4 h + c][r]: dim 64 h + 4 (4 kg + r) + c of head n
#pragma unroll
    for (int i = 0; i < NI; i++) acc[i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    const uint32_t first = SEL ? 0 : lo >> 4, tiles = SEL ? n_select << (kv.shift - 4) : (len + 15) >> 4;
    for (uint32_t t = first + wave; t < tiles; t += ATT_W) {
        const uint32_t entry = SEL ? list[t >> (kv.shift - 4)] : t >> (kv.shift - 4);
        const uint32_t start = SEL ? (t & ((R >> 4) - 1)) << 4 : (t << 4) & (R - 1);        // of the tile in its page
        if (SEL && entry >= pages_of(kv, len)) continue;
        const uint32_t page = table[entry], pos = (entry << kv.shift) + start;
        if (page >= kv.n_pages || (SEL && pos >= len)) continue;
        const size_t row = ((size_t)page << kv.shift) + start;
        f32x4 s = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const f32x4 k = load4<TYPE>(kv.k, kv.k_scales, ((row + n) * kv.n_kv + head) * HD + 16 * i + 4 * kg);
#pragma unroll
            for (int e = 0; e < 4; e++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[e], qf[i][e], s, 0, 0, 0);
        }
        float top = m;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            float x = s[r] * scale;
            if (softcap > 0.f) x = softcap * tanhf(x / softcap);
            const uint32_t at = pos + 4 * kg + r;
            s[r] = at < len && at >= lo ? x : -INFINITY;
            top = fmaxf(top, s[r]);
        }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float base = top == -INFINITY ? 0.f : top, f = expf(m - base);
        float p[4];
        l *= f;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            p[r] = expf(s[r] - base);
            l += p[r];
        }
        m = top;
#pragma unroll
        for (int i = 0; i < NI; i++) acc[i] *= f;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint32_t at = pos + 4 * kg + r;
#pragma unroll
            for (int h = 0; h < HD / 64; h++) {
                f32x4 v = load4<TYPE>(kv.v, kv.v_scales, ((row + 4 * kg + r) * kv.n_kv + head) * HD + 64 * h + 4 * n);
                if (!(at < len && at >= lo)) v = (f32x4){0.f, 0.f, 0.f, 0.f};      // what lies behind the last row is no number, maybe
#pragma unroll
                for (int c = 0; c < 4; c++) acc[4 * h + c] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[c], p[r], acc[4 * h + c], 0, 0, 0);
            }
        }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (kg == 0) { sm_m[wave][n] = m; sm_l[wave][n] = l; }
#pragma unroll
    for (int i = 0; i < NI; i++)
#pragma unroll
        for (int r = 0; r < 4; r++) sm_o[wave][n][64 * (i / 4) + 4 * (4 * kg + r) + i % 4] = acc[i][r];
    __syncthreads();
    for (int e = threadIdx.x; e < g * HD; e += 64 * ATT_W) {
        const int h = e / HD, d = e % HD;
        float top = -INFINITY, sum = 0.f, o = 0.f;
        for (int w = 0; w < ATT_W; w++) top = fmaxf(top, sm_m[w][h]);
        const float base = top == -INFINITY ? 0.f : top;
        for (int w = 0; w < ATT_W; w++) {
            const float f = expf(sm_m[w][h] - base);
            sum = fmaf(sm_l[w][h], f, sum);
            o = fmaf(sm_o[w][h][d], f, o);
        }
        out[((size_t)seq * n_head + head * g + h) * HD + d] = top == -INFINITY && sum == 0.f ? 0.f : o / sum;      // nothing to attend to: zeros
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
    // A wave a token once the tokens alone give every CU its waves; fewer tokens leave their slices to more waves.
    const bool many = (size_t)p.t >= 4 * (size_t)device_cus();
    const int each = many ? (int)slices : 1;
    const dim3 grid(many ? (p.t + 3) / 4 : p.t, many ? 1u : (unsigned)((slices + 3) / 4));
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
    if (grid > 0x7FFFFFFFull) return set_error(FHIP_ERR_SHAPE, "fhip_paged_rows: too many rows for one launch");
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
        hipLaunchKernelGGL((bounds_kernel<decltype(ty)::value>), dim3(kv.n_seq * kv.n_kv, (unsigned)pages), dim3(hd), 0, s, kv, hd, lens, fresh, max_new, bounds);
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
        const dim3 grid((pages + 3) / 4, kv.n_kv, kv.n_seq);
        if (hd == 128) hipLaunchKernelGGL((score_kernel<128>), grid, dim3(256), 0, s, kv, q, lens, max_len, bounds, n_head, first, last, (uint64_t*)ws, pages);
        else hipLaunchKernelGGL((score_kernel<64>), grid, dim3(256), 0, s, kv, q, lens, max_len, bounds, n_head, first, last, (uint64_t*)ws, pages);
    }
    hipLaunchKernelGGL(select_kernel, dim3(kv.n_seq * kv.n_kv), dim3(SEL_T), 0, s, kv, lens, max_len, n_select, (const uint64_t*)ws, pages, first + last, out);
    return check_hip(hipGetLastError(), "paged_select launch");
}

size_t paged_attention_ws_bytes(const PagedView&, int, int, size_t) { return 0; }
int launch_paged_attention(uint32_t type, int hd, const PagedView& kv, const float* q, const uint32_t* lens, uint32_t max_len, const uint32_t* selected, uint32_t n_select,
                           int n_head, uint32_t window, float softcap, float* ws, float* out, hipStream_t s) {
    (void)ws;
    const float scale = 1.0f / sqrtf((float)hd);
    const dim3 grid(kv.n_seq * kv.n_kv);
    return by_type(type, [&](auto ty) {
        constexpr int TYPE = decltype(ty)::value;
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(64 * ATT_W), 0, s, kv, q, lens, max_len, selected, n_select, n_head, window, softcap, scale, out); };
        if (hd == 128) selected ? go(attention_kernel<TYPE, 128, true>) : go(attention_kernel<TYPE, 128, false>);
        else selected ? go(attention_kernel<TYPE, 64, true>) : go(attention_kernel<TYPE, 64, false>);
        return check_hip(hipGetLastError(), "paged_attention launch");
    });
}

}  // namespace fhip
