// Launchers of the paged key/value cache (paged.hip); the public description of a cache is fhip_paged.
#pragma once
#include "common.hpp"

namespace fhip {

// A cache as the kernels take it: a row is n_kv * hd values, row p of sequence i lies in page table[i * table_stride + (p >> shift)].
struct PagedView {
    void *k, *v;                    // [n_pages << shift, n_kv * hd]
    uint16_t *k_scales, *v_scales;  // Q8_0: a scale for each 32 values
    const uint32_t* table;
    size_t table_stride;
    uint32_t n_seq, pages_per_seq, n_pages;
    int n_kv, shift;                // pages hold 1 << shift rows
};
struct PagedPost {
    const float *qkv, *bias, *q_norm, *k_norm;   // bias and norms may be null
    const uint32_t *seqs, *pos;                  // seqs null: row i belongs to sequence i
    const float* freq_scale;                     // or null
    float* q_out;
    uint32_t t;
    int n_head, n_rot, interleaved;
    float eps;
    double rate;                                 // pair c turns by pos * exp(c * rate)
};
int launch_paged_append(uint32_t type, int hd, const PagedView& kv, const PagedPost& p, hipStream_t s);
int launch_paged_rows(uint32_t type, int hd, const PagedView& kv, uint32_t seq, size_t row0, size_t rows, float* k_out, float* v_out, hipStream_t s);
int launch_paged_key_bounds(uint32_t type, int hd, const PagedView& kv, const uint32_t* lens, const uint32_t* fresh, uint32_t max_new, float* bounds, hipStream_t s);
size_t paged_select_ws_bytes(const PagedView& kv, size_t max_len);
int launch_paged_select(int hd, const PagedView& kv, const float* q, const uint32_t* lens, uint32_t max_len, const float* bounds, int n_head, uint32_t n_select,
                        uint32_t first, uint32_t last, void* ws, uint32_t* out, hipStream_t s);
// selected: null, or [n_seq, n_kv, n_select] page indices of the sequences
size_t paged_attention_ws_bytes(uint32_t type, const PagedView& kv, int hd, int n_head, size_t max_len);
int launch_paged_attention(uint32_t type, int hd, const PagedView& kv, const float* q, const uint32_t* lens, uint32_t max_len, const uint32_t* selected, uint32_t n_select,
                           int n_head, uint32_t window, float softcap, float* ws, float* out, hipStream_t s);

}  // namespace fhip
