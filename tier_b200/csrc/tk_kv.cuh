// tk_kv.cuh -- the 4-bit key/value cache as the kernels see it: views of
// tk_kvcache / tk_seqs, the checked walk from a packed row to its cached
// token, and the 4-bit numbers.
#pragma once
#include "tk_device.cuh"
#include "tk_internal.h"

namespace tk {

struct KvView {
    uint8_t *kq, *vq;
    __half *ks, *vs;
    int n_pages, page_shift, heads, dim;
};

struct SeqView {
    const int32_t *q_start, *kv_len, *pages;
    int n_seqs, n_tokens, max_new, max_pages;
};

inline KvView kv_view(const tk_kvcache& c) {
    KvView v;
    v.kq = static_cast<uint8_t*>(c.k_q);
    v.vq = static_cast<uint8_t*>(c.v_q);
    v.ks = static_cast<__half*>(c.k_s);
    v.vs = static_cast<__half*>(c.v_s);
    v.n_pages = c.n_pages;
    v.page_shift = 0;
    while ((1 << v.page_shift) < c.page_tokens) ++v.page_shift;
    v.heads = c.n_kv_heads;
    v.dim = c.head_dim;
    return v;
}
inline SeqView seq_view(const tk_seqs& s) {
    return SeqView{s.q_start, s.kv_len, s.pages, s.n_seqs, s.n_tokens, s.max_new, s.max_pages};
}

// One sequence of the batch, its device-side numbers checked: a sequence whose
// numbers do not fit has no new tokens.
struct SeqInfo {
    int row0, n_new, kv;
};
__device__ __forceinline__ SeqInfo seq_info(const SeqView& s, int page_shift, int b, int* status) {
    const int r0 = s.q_start[b], r1 = s.q_start[b + 1], kv = s.kv_len[b];
    SeqInfo i{r0, r1 - r0, kv};
    if (r0 < 0 || r1 < r0 || r1 > s.n_tokens || r1 - r0 > s.max_new || kv < 0 ||
        (long)kv > ((long)s.max_pages << page_shift)) {
        raise_status(status, DEV_INVALID);
        i = SeqInfo{0, 0, 0};
    }
    return i;
}

// Last sequence whose q_start is at or before packed row r (q_start in global
// or shared memory); the caller checks that r lies inside it.
__device__ __forceinline__ int seq_of_row(const int32_t* q_start, int n_seqs, int r) {
    int lo = 0, hi = n_seqs - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (q_start[mid] <= r) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Page holding a sequence's token `pos`: an id outside the cache is reported
// and read as page 0.
__device__ __forceinline__ int page_of(const SeqView& s, const KvView& c, int b, int pos, int* status) {
    const int p = s.pages[(size_t)b * s.max_pages + (pos >> c.page_shift)];
    if ((unsigned)p < (unsigned)c.n_pages) return p;
    raise_status(status, DEV_INVALID);
    return 0;
}
// Index of (page, key/value head, row) among the cache's rows.
__device__ __forceinline__ size_t kv_row(const KvView& c, int page, int head, int pos) {
    return ((((size_t)page * c.heads + head) << c.page_shift) + (pos & ((1 << c.page_shift) - 1)));
}

// The word's value e (0..7), -8..7: fields 0..3 hold values 0, 2, 4, 6 and
// fields 4..7 values 1, 3, 5, 7, so that one mask takes the two fp16 halves of
// a pair of neighbouring values (kv_pairs).
__device__ __forceinline__ int kv_nibble(uint32_t w, int e) {
    const int f = (e >> 1) + 4 * (e & 1);
    return (int)(((w >> (4 * f)) & 15u) ^ 8u) - 8;
}

}  // namespace tk
