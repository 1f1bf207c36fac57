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

// First key of rows at positions `pos` and on: 0 without a window.  (pos may be
// negative, down to minus the new tokens, and a window of any size: from
// position 0 back nothing can overflow, and no key lies before it.)
__host__ __device__ __forceinline__ int kv_first_key(int pos, int window) {
    const int p = pos > 0 ? pos : 0;
    return window > 0 && p >= window ? p - window + 1 : 0;
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
// (false, page 0).
__device__ __forceinline__ bool page_at(const SeqView& s, const KvView& c, int b, int pos, int* status, int& page) {
    page = s.pages[(size_t)b * s.max_pages + (pos >> c.page_shift)];
    if ((unsigned)page < (unsigned)c.n_pages) return true;
    raise_status(status, DEV_INVALID);
    page = 0;
    return false;
}
// The same to read from: page 0 in place of one outside the cache.
__device__ __forceinline__ int page_of(const SeqView& s, const KvView& c, int b, int pos, int* status) {
    int page;
    page_at(s, c, b, pos, status, page);
    return page;
}
// Index of (page, key/value head, row) among the cache's rows.
__device__ __forceinline__ size_t kv_row(const KvView& c, int page, int head, int pos) {
    return ((((size_t)page * c.heads + head) << c.page_shift) + (pos & ((1 << c.page_shift) - 1)));
}

// ---- 4-bit numbers to fp16 -------------------------------------------------
// A word's fields 0..3 hold values 0, 2, 4, 6 and fields 4..7 values 1, 3, 5, 7
// (two's complement), so that one mask takes the two fp16 halves of a pair of
// neighbouring values.  x: four fields of each 16-bit half.  The method is that
// of Kim et al. (2022, "Who Says Elephants Can't Run") for integer weights: an
// fp16 with exponent bits 0x6400 counts in ones from 1024, so OR-ing a field
// n + 8 into its low bits gives 1024 + (n + 8), or 1024 + 16 (n + 8) for the
// second field; the XOR in the same LOP3 turns two's complement n into n + 8.
// Both are brought back to n exactly (|n| <= 8), then scaled: n * d is exact for
// d of 8 significant bits.
__device__ __forceinline__ uint32_t lop_and_xor(uint32_t x, uint32_t mask, uint32_t flip) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(x), "r"(mask), "r"(flip));   // (x & mask) ^ flip
    return r;
}
__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ void kv_fields(uint32_t x, __half2 d, uint32_t (&out)[4]) {
    const __half2 one = as_half2(0xe408e408u);                       // -1032
    const __half2 sixteenth = as_half2(0x2c002c00u), off = as_half2(0xd480d480u);   // 1/16, -72
    const uint32_t y = x >> 8;
    out[0] = as_u32(__hmul2(__hadd2(as_half2(lop_and_xor(x, 0x000f000fu, 0x64086408u)), one), d));
    out[1] = as_u32(__hmul2(__hfma2(as_half2(lop_and_xor(x, 0x00f000f0u, 0x64806480u)), sixteenth, off), d));
    out[2] = as_u32(__hmul2(__hadd2(as_half2(lop_and_xor(y, 0x000f000fu, 0x64086408u)), one), d));
    out[3] = as_u32(__hmul2(__hfma2(as_half2(lop_and_xor(y, 0x00f000f0u, 0x64806480u)), sixteenth, off), d));
}

__device__ __forceinline__ float fast_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}


// ---- attention ---------------------------------------------------------------
struct KvaArgs {
    KvView c;
    SeqView s;
    const void* q;
    void* out;
    long ldq, ldo;
    int n_heads, group, window;
    float scale2;         // scale * log2(e)
    float* part;          // parts of divided rows (workspace)
    int* count;           // finished parts of each divided set of rows, by the block of its first part; zero between calls
    int* status;
};

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int DT>
__device__ __forceinline__ void load_pairs8(const void* p, size_t at, float (&x)[8]) {
    if constexpr (DT == TK_DT_F32) {
        const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
        const float4 u = f[0], v = f[1];
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == TK_DT_BF16) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                x[2 * i] = h2f_bits((uint16_t)(w[i] & 0xffffu));
                x[2 * i + 1] = h2f_bits((uint16_t)(w[i] >> 16));
            }
        }
    }
}
// 2^e with max * 2^e in [2^13, 2^14); 1 for zero and for what is not finite.
__device__ __forceinline__ float q_unit(float max, float& back) {
    const int e = (int)(__float_as_uint(max) >> 23);
    if (e < 14 || e >= 255) { back = 1.0f; return 1.0f; }
    back = __uint_as_float((uint32_t)(e - 13) << 23);             // 2^(e - 127 - 13)
    return __uint_as_float((uint32_t)(254 - (e - 13)) << 23);
}

// A row's softmax weights are 2^(score - reference).  The reference is set `up`
// below the largest score seen and stays until a score passes it by `move`:
// the largest weight lies between 2^up and 2^move, inside fp16's range.  What
// lies below decides how small weights are held, as fp16 ends at 2^-24.
//   fp32 rows, 14 and 15.9: the two parts end at 2^-25, 2^-39 of the largest
//   weight at most; a weight of 2^-22 of it is off by 2^-17 of itself.
//   16-bit rows, 7 and 15: whole fp16 numbers (off by 2^-12 of themselves)
//   down to 2^-21 of the largest, then off by 2^-32 of it.
// A reference that may stay moves less often: 7 for fp32 rows too, off by
// 2^-10 of a weight of 2^-22, took 67.4 us for 8 sequences of 5 rows at 8191
// keys, not 69.4, and 151.4 for two prompts of up to 1537, not 152.3; 14 and 15 for
// 16-bit rows 661 for a prompt of 8192, not 608.
template <bool FP32>
struct KvRef {
    static constexpr float up = FP32 ? 14.0f : 7.0f, move = FP32 ? 15.9f : 15.0f;
    // Minus the reference for a largest score mx, itself rounded: both roundings
    // go down, so that the weight stays below 2^up where a step of fp32 is whole
    // powers of two (from scores of 2^24 on; below 2^27 it is down to 2^20 lower).
    static __device__ __forceinline__ float minus(float mx) {
        return __fsub_rd(up, __fmaf_ru(fabsf(mx), 5.9604644775390625e-08f, mx));
    }
};

// Values e .. e + 3 of an output row (packed row, head): O / l, zero where nothing was seen.
struct KvaRow {
    int row, head;
};
template <int DT, int D>
__device__ __forceinline__ void kv_store_out(const KvaArgs& a, KvaRow r, int e, float4 o, float l) {
    const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
    const size_t at = (size_t)r.row * a.ldo + (size_t)r.head * D + e;
    if (l == 0.0f) o = make_float4(0, 0, 0, 0);
    if constexpr (DT == TK_DT_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    } else {
        uint2 w;
        if constexpr (DT == TK_DT_F16) {
            w.x = (uint32_t)f2h_bits(o.x * inv) | ((uint32_t)f2h_bits(o.y * inv) << 16);
            w.y = (uint32_t)f2h_bits(o.z * inv) | ((uint32_t)f2h_bits(o.w * inv) << 16);
        } else {
            w.x = (uint32_t)f2bf_bits(o.x * inv) | ((uint32_t)f2bf_bits(o.y * inv) << 16);
            w.y = (uint32_t)f2bf_bits(o.z * inv) | ((uint32_t)f2bf_bits(o.w * inv) << 16);
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = w;
    }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Joins the parts of a row set, in the order of the keys, by all `threads` of a
// group (`sync`: its barrier): a part is O of `rows` rows (D values each, of
// ROWS), then (m, l) of each.  at(c): part c, out(r): row r.  Statistics and
// factors go through shared memory (`bytes` of it, rows in batches that fit),
// a warp a row; then 16 parts' O are in flight together.
template <int D, int DT, int ROWS, class At, class Out, class Sync>
__device__ __forceinline__ void kv_join(const KvaArgs& a, int parts, int all_rows, int thread, int threads, uint8_t* smem,
                                        int bytes, At at, Out out, Sync sync) {
    const int some = max(1, min(all_rows, bytes / (8 * parts + 4)));
    const int warp = thread >> 5, lane = thread & 31;
    for (int r0 = 0; r0 < all_rows; r0 += some) {
        const int rows = min(some, all_rows - r0);
        float* fac = reinterpret_cast<float*>(smem);               // [parts][rows] m, then the factor; the same of l; [rows] sums
        float* ls = fac + parts * rows;
        float* sum = ls + parts * rows;
        for (int i = thread; i < parts * rows; i += threads) {
            const int c = i / rows, r = i - c * rows;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(at(c) + ROWS * D) + r0 + r);
            fac[i] = ml.x;
            ls[i] = ml.y;
        }
        sync();
        for (int r = warp; r < rows; r += threads >> 5) {
            float m = -INFINITY, l = 0.0f;
            for (int c = lane; c < parts; c += 32) m = fmaxf(m, fac[c * rows + r]);
            for (int i = 16; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, i));
            const float ref = m == -INFINITY ? 0.0f : m;
            for (int c = lane; c < parts; c += 32) {
                const float f = fast_exp2(fac[c * rows + r] - ref);
                fac[c * rows + r] = f;
                l += ls[c * rows + r] * f;
            }
            for (int i = 16; i; i >>= 1) l += __shfl_xor_sync(~0u, l, i);
            if (lane == 0) sum[r] = l;
        }
        sync();
        for (int i = thread; i < rows * (D / 4); i += threads) {
            const int r = i / (D / 4), e = (i - r * (D / 4)) * 4;
            float4 o = make_float4(0, 0, 0, 0);
            for (int c0 = 0; c0 < parts; c0 += 16) {               // whatever is left of 16
                float4 v[16];
#pragma unroll
                for (int c = 0; c < 16; ++c)
                    v[c] = __ldcg(reinterpret_cast<const float4*>(at(min(c0 + c, parts - 1)) + (r0 + r) * D + e));
#pragma unroll
                for (int c = 0; c < 16; ++c) {
                    const float f = c0 + c < parts ? fac[(c0 + c) * rows + r] : 0.0f;
                    o.x += v[c].x * f; o.y += v[c].y * f; o.z += v[c].z * f; o.w += v[c].w * f;
                }
            }
            kv_store_out<DT, D>(a, out(r0 + r), e, o, sum[r]);
        }
        sync();
    }
}

// tk_kvattn_tc.cu
tk_status launch_kv_prompt(tk_ctx* ctx, KvaArgs& a, int dtype, cudaStream_t st);

}  // namespace tk
