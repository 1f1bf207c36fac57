// tk_rows.cuh -- rows of logits: units of access, the sums of a softmax, its
// dense gradient, and the launch (tk_logprobs.cu, tk_distill.cu).
#pragma once
#include "tk_device.cuh"
#include "tk_f32x2.cuh"
#include "tk_internal.h"

namespace tk {

constexpr int RW_THREADS = 256, RW_WARPS = RW_THREADS / 32;

template <class T> __device__ __forceinline__ float rw_float(T x);
template <> __device__ __forceinline__ float rw_float(float x) { return x; }
template <> __device__ __forceinline__ float rw_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float rw_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T rw_to(float x);
template <> __device__ __forceinline__ float rw_to(float x) { return x; }
template <> __device__ __forceinline__ __half rw_to(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 rw_to(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float rw_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rw_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Weights.  A logit's exponent to the base 2 below the row's largest, m, is
// y = (x - m) * c, c = log2(e) / temperature.  The difference comes first: it is
// exact where it matters, however large the logits are, and a mask of fp32's
// lowest value only makes it -inf, whose weight 2^y is 0.  Where y is also a
// factor it is clamped at RW_LOW, where the weight is 0 too; a NaN stays one (a
// row that holds NaN or +inf has the sum NaN).
constexpr float RW_LOW = -200.0f;

// What a row's sums are relative to before a logit was seen: the lowest
// finite number, so that -inf has the weight 0 and not NaN.
constexpr float RW_LOWEST = -3.402823466e38f;

// ---------------------------------------------------------------------------
// A row in units of 32 bytes (8 fp32 logits, 16 of the 16-bit types), one load
// and one sector of memory each.  What lies before the first boundary and
// behind the last unit, 30 logits at most, are the row's ends.
// ---------------------------------------------------------------------------
template <class XT>
struct RwUnit {
    static constexpr int N = 32 / sizeof(XT);      // logits
    uint32_t w[8];
    __device__ __forceinline__ void load(const XT* p) {
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(p) : "memory");
    }
    __device__ __forceinline__ f32x2 two(int i) const;     // logits 2 i, 2 i + 1
    __device__ __forceinline__ void lowest();              // all -inf
    __device__ __forceinline__ float max(int half) const;  // of its first or second half; NaN is passed over
};
template <> __device__ __forceinline__ f32x2 RwUnit<float>::two(int i) const {
    return pack2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
}
template <> __device__ __forceinline__ f32x2 RwUnit<__nv_bfloat16>::two(int i) const {
    return pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <> __device__ __forceinline__ f32x2 RwUnit<__half>::two(int i) const {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    return pack2(f.x, f.y);
}
template <class XT> __device__ __forceinline__ void RwUnit<XT>::lowest() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = sizeof(XT) == 4 ? 0xff800000u : 0xff80ff80u;
}
template <> __device__ __forceinline__ void RwUnit<__half>::lowest() {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0xfc00fc00u;
}
template <> __device__ __forceinline__ float RwUnit<float>::max(int half) const {
    const float a = fmaxf(__uint_as_float(w[4 * half]), __uint_as_float(w[4 * half + 1]));
    return fmaxf(fmaxf(a, __uint_as_float(w[4 * half + 2])), __uint_as_float(w[4 * half + 3]));
}
template <> __device__ __forceinline__ float RwUnit<__nv_bfloat16>::max(int half) const {
    uint32_t m = w[4 * half];
#pragma unroll
    for (int i = 1; i < 4; ++i) asm("max.bf16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[4 * half + i]));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
}
template <> __device__ __forceinline__ float RwUnit<__half>::max(int half) const {
    uint32_t m = w[4 * half];
#pragma unroll
    for (int i = 1; i < 4; ++i) asm("max.f16x2 %0, %1, %2;" : "=r"(m) : "r"(m), "r"(w[4 * half + i]));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return fmaxf(f.x, f.y);
}
constexpr int RW_BATCH = 4;                        // units that a thread holds at once

// The part of a row that one block of a cluster takes: units [0, n) from x.
template <class XT>
__device__ __forceinline__ int rw_head(const XT* row, int vocab) {      // logits before the first boundary
    constexpr int N = RwUnit<XT>::N;
    return min((int)(-(reinterpret_cast<uintptr_t>(row) / sizeof(XT)) & (N - 1)), vocab);
}
template <class XT>
struct RwPart {
    const XT* x;              // its first unit
    int first;                // that unit's place in the row
    int n;
    __device__ __forceinline__ RwPart(const XT* row, int vocab, int rank, int parts) {
        constexpr int N = RwUnit<XT>::N;
        const int head = rw_head(row, vocab), units = (vocab - head) / N;
        const int each = ((units + parts - 1) / parts + 31) & ~31, u0 = min(rank * each, units);   // (a warp's loads stay whole)
        first = head + N * u0;
        x = row + first;
        n = min(each, units - u0);
    }
};
// A batch: units u0 + tid, and RW_THREADS apart; -inf beyond the part.
template <class XT>
__device__ __forceinline__ void rw_batch(RwUnit<XT> (&u)[RW_BATCH], const RwPart<XT>& p, int u0) {
    constexpr int N = RwUnit<XT>::N;
    const XT* from = p.x + (long)N * (u0 + (int)threadIdx.x);
    if (u0 + RW_THREADS * RW_BATCH <= p.n) {
#pragma unroll
        for (int j = 0; j < RW_BATCH; ++j) u[j].load(from + N * RW_THREADS * j);
    } else {
#pragma unroll
        for (int j = 0; j < RW_BATCH; ++j) {
            if (u0 + j * RW_THREADS + (int)threadIdx.x < p.n) u[j].load(from + N * RW_THREADS * j);
            else u[j].lowest();
        }
    }
}
// The row's ends: how many, and the place of the i-th.
template <class XT>
struct RwEnds {
    int head, skip, n;
    __device__ __forceinline__ RwEnds(const XT* row, int vocab) {
        constexpr int N = RwUnit<XT>::N;
        head = rw_head(row, vocab);
        skip = (vocab - head) / N * N;
        n = vocab - skip;
    }
    __device__ __forceinline__ int place(int i) const { return i < head ? i : i + skip; }
};

// 2^d, d <= 0, for totals, whose reference may move by little many times in a
// long row: where it does, 2^d - 1 comes from a polynomial (through the Chebyshev
// points of [-1/2, 0], off by 2^-24 of itself), so that next to nothing is lost
// each time; larger steps, where the exponential's own error counts, leave
// little of the totals.
__device__ __forceinline__ double rw_move(float d) {
    const float p = fmaf(fmaf(fmaf(fmaf(0.00115544f, d, 0.009542275f), d, 0.05549072f), d, 0.24022567f), d, 0.69314712f);
    return d > -0.5f ? 1.0 + (double)(d * p) : (double)rw_exp2(d);
}

// Running sums of one thread: S of the weights 2^y and A of 2^y y.  m moves only
// when a batch of logits holds a larger one; s and a are sums of at most
// RW_FLUSH batches before they go, in 64 bits, to the totals, which have a
// reference of their own.  A weight that counts is rounded 16 times in its batch
// (of 16-bit logits; 8 of fp32), 3 to bring the lanes together, 7 as other
// batches come, and 7 times is off by 3.4 roundings as m moves (its exponential
// by 2.4 at most, on sm_100 over all floats from -125 to -2^-40; less for small
// steps): 50, and 10 in at most four exponentials as threads, warps and blocks
// come together: 60.  16 batches made it 95, and totals moved by the
// exponential, 64 times in the longest rows, up to 12 * 2^-22 where all rise
// alike (measured; now 1.4).  It costs 1 % of the loss of 300 fp32 rows (29.7 ->
// 30.1 us) and nothing elsewhere; a polynomial for m's own
// moves cost 2 to 3 % of small calls.
constexpr int RW_FLUSH = 8;
template <bool ENT>
struct RwSums {
    float m = RW_LOWEST, s = 0.0f, a = 0.0f, M = RW_LOWEST;
    double S = 0.0, A = 0.0;
    __device__ __forceinline__ void raise(float to, float c) {
        const float d = fmaxf((m - to) * c, RW_LOW), f = rw_exp2(d);
        if (ENT) a = f * fmaf(s, d, a);
        s *= f;
        m = to;
    }
    __device__ __forceinline__ void flush(float c) {
        const float d = fmaxf((M - m) * c, RW_LOW);
        const double f = rw_move(d);
        if (ENT) A = f * (A + S * d) + a;
        S = f * S + s;
        M = m;
        s = a = 0.0f;
    }
    // Two logits: weights to s2, weight times exponent to a2.
    static __device__ __forceinline__ void two(f32x2 x, f32x2 nm, f32x2 c, f32x2& s2, f32x2& a2) {
        const f32x2 y = mul2(add2(x, nm), c);
        float y0, y1;
        unpack2(y, y0, y1);
        if (ENT) {
            y0 = rw_max_nan(y0, RW_LOW);
            y1 = rw_max_nan(y1, RW_LOW);
        }
        const f32x2 e = pack2(rw_exp2(y0), rw_exp2(y1));
        s2 = add2(s2, e);
        if (ENT) a2 = fma2(e, pack2(y0, y1), a2);
    }
    __device__ __forceinline__ void single(float v, float c) {
        if (v > m) raise(v, c);
        f32x2 s2 = 0, a2 = 0;
        float e, none;
        two(pack2(v, -INFINITY), pack2(-m, -m), pack2(c, c), s2, a2);
        unpack2(s2, e, none);
        s += e;
        if (ENT) {
            unpack2(a2, e, none);
            a += e;
        }
    }
    template <class XT, int NB>
    __device__ __forceinline__ void batch(const RwUnit<XT> (&u)[NB], f32x2 c) {     // none above m
        const f32x2 nm = pack2(-m, -m);
        f32x2 s2[2] = {0, 0}, a2[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
            for (int i = 0; i < RwUnit<XT>::N / 2; ++i) two(u[j].two(i), nm, c, s2[i & 1], a2[i & 1]);
        float p, q;
        unpack2(add2(s2[0], s2[1]), p, q);
        s += p + q;
        if (ENT) {
            unpack2(add2(a2[0], a2[1]), p, q);
            a += p + q;
        }
    }
};

// The same variable of another block of the cluster.
template <class T>
__device__ __forceinline__ T* rw_peer(T* mine, int rank) {
    T* p;
    asm("mapa.u64 %0, %1, %2;" : "=l"(p) : "l"(mine), "r"(rank));
    return p;
}

// m, S and A of all parts brought together: threads of a block, blocks of a
// cluster.  A row that holds NaN or +inf has S = NaN by its arithmetic, one of
// nothing above -inf S = 0.
struct RwStat {
    float m;
    double s, a;
};
__device__ __forceinline__ RwStat rw_to_max(const RwStat& v, float m, float c) {
    const float d = fmaxf((v.m - m) * c, RW_LOW);
    const double f = rw_exp2(d);
    return RwStat{m, f * v.s, f * (v.a + v.s * d)};
}
template <bool ENT>
__device__ __forceinline__ RwStat rw_warp_join(RwStat v, float c) {
    float m = v.m;
    for (int i = 16; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, i));
    v = rw_to_max(v, m, c);
    for (int i = 16; i; i >>= 1) {
        v.s += __shfl_xor_sync(~0u, v.s, i);
        if (ENT) v.a += __shfl_xor_sync(~0u, v.a, i);
    }
    return v;
}

// Two numbers, rounded once, as a pair of DT.
template <class DT> __device__ __forceinline__ uint32_t rw_pair(f32x2 v);
template <> __device__ __forceinline__ uint32_t rw_pair<__nv_bfloat16>(f32x2 v) {
    float lo, hi;
    uint32_t r;
    unpack2(v, lo, hi);
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <> __device__ __forceinline__ uint32_t rw_pair<__half>(f32x2 v) {
    float lo, hi;
    uint32_t r;
    unpack2(v, lo, hi);
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void rw_store(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.global.L1::no_allocate.v4.b32 [%4], {%0,%1,%2,%3};" ::"r"(a), "r"(b), "r"(c), "r"(d), "l"(p) : "memory");
}
__device__ __forceinline__ void rw_store(void* p, const uint32_t* w) {
    asm volatile("st.global.L1::no_allocate.L2::evict_first.v8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "l"(p)
                 : "memory");
}

// The gradient of a row is, but for its own few places, 2^y (f + g y) / S with
// factors of the row (1 / S among them): the dense part.
template <bool LIN>
struct RwDense {
    float m, c, f, g;
    __device__ __forceinline__ f32x2 two(f32x2 x) const {
        const f32x2 y = mul2(add2(x, pack2(-m, -m)), pack2(c, c));
        float y0, y1;
        unpack2(y, y0, y1);
        if (LIN) {
            y0 = rw_max_nan(y0, RW_LOW);
            y1 = rw_max_nan(y1, RW_LOW);
        }
        const f32x2 e = pack2(rw_exp2(y0), rw_exp2(y1));
        return mul2(e, LIN ? fma2(pack2(y0, y1), pack2(g, g), pack2(f, f)) : pack2(f, f));
    }
    __device__ __forceinline__ float one(float x) const {
        float lo, hi;
        unpack2(two(pack2(x, x)), lo, hi);
        return lo;
    }
};

// A place that a thread's entry of a list names, if it lies in the block's part
// of the row and no earlier entry names it: the sum of the entries' shares
// there is subtracted (in the list's order).  ids: in shared memory, 16-byte
// aligned, -1 up to a multiple of four.
struct RwListed {
    bool mine;
    int id;
    float share;
};
template <class XT>
__device__ __forceinline__ RwListed rw_listed(const RwPart<XT>& p, const RwEnds<XT>& e, bool ends, const int* ids,
                                              const float* share, int k, int entry) {
    RwListed r{false, entry < k ? ids[entry] : -1, 0.0f};
    r.mine = r.id >= p.first && r.id < p.first + RwUnit<XT>::N * p.n;
    if (ends && r.id >= 0) r.mine |= r.id < e.head || r.id >= e.head + e.skip;
    if (r.mine)
        for (int j = 0; j < k; j += 4) {
            const int4 o = *reinterpret_cast<const int4*>(ids + j);
            const int at[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (at[i] == r.id) {
                    r.mine &= j + i >= entry;
                    r.share += share[j + i];
                }
        }
    return r;
}

// The dense part.  Where dx's units lie on their boundaries as x's do, a batch
// of units (loaded by rw_batch) is written with one or two stores each.
template <class XT, class DT>
__device__ __forceinline__ bool rw_alike(const DT* d) {       // d: at x's first unit
    constexpr int BYTES = RwUnit<XT>::N * sizeof(DT);
    return (reinterpret_cast<uintptr_t>(d) & (BYTES > 32 ? 31 : BYTES - 1)) == 0;
}
template <class XT, class DT, bool LIN, int NB>
__device__ __forceinline__ void rw_write(const RwUnit<XT> (&u)[NB], DT* d, const RwPart<XT>& p, int u0,
                                         const RwDense<LIN>& dense) {
    constexpr int N = RwUnit<XT>::N, BYTES = N * sizeof(DT);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        const int at = u0 + j * RW_THREADS + (int)threadIdx.x;
        if (at >= p.n) break;
        DT* to = d + (long)N * at;
        uint32_t w[BYTES / 4];
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            const f32x2 r = dense.two(u[j].two(i));
            if constexpr (sizeof(DT) == 4) {
                float lo, hi;
                unpack2(r, lo, hi);
                w[2 * i] = __float_as_uint(lo);
                w[2 * i + 1] = __float_as_uint(hi);
            } else
                w[i] = rw_pair<DT>(r);
        }
        if constexpr (BYTES == 16) rw_store(to, w[0], w[1], w[2], w[3]);
        else
#pragma unroll
            for (int i = 0; i < BYTES / 32; ++i) rw_store(reinterpret_cast<char*>(to) + 32 * i, w + 8 * i);
    }
}
// Where they do not: element by element, a warp's side by side.
template <class XT, class DT, bool LIN>
__device__ __forceinline__ void rw_write_other(DT* d, const RwPart<XT>& p, const RwDense<LIN>& dense) {
    const int n = RwUnit<XT>::N * p.n;
    for (int j0 = threadIdx.x; j0 < n; j0 += 8 * RW_THREADS) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = j0 + i * RW_THREADS < n ? rw_float(p.x[j0 + i * RW_THREADS]) : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            float lo, hi;
            unpack2(dense.two(pack2(x[i], x[i + 1])), lo, hi);
            if (j0 + i * RW_THREADS < n) d[j0 + i * RW_THREADS] = rw_to<DT>(lo);
            if (j0 + (i + 1) * RW_THREADS < n) d[j0 + (i + 1) * RW_THREADS] = rw_to<DT>(hi);
        }
    }
}

// dx of one part of a row: the dense part, at the listed places less their
// shares.  dx may be x itself: what a thread writes it has read, and the listed
// logits are read before any is written.
template <class XT, class DT, bool LIN>
__device__ __forceinline__ void rw_gradient(const XT* row, DT* drow, int vocab, const RwPart<XT>& p, bool ends, const int* ids,
                                            const float* share, int k, float scale, const RwDense<LIN>& dense) {
    const RwEnds<XT> e(row, vocab);
    const RwListed l = rw_listed(p, e, ends, ids, share, k, (int)threadIdx.x);
    const float v = l.mine ? rw_float(row[l.id]) : 0.0f;
    const bool end = ends && (int)threadIdx.x < e.n;
    const float v_end = end ? rw_float(row[e.place(threadIdx.x)]) : 0.0f;
    __syncthreads();
    if (end) drow[e.place(threadIdx.x)] = rw_to<DT>(dense.one(v_end));
    DT* d = drow + p.first;
    if (rw_alike<XT>(d)) {
        for (int u0 = 0; u0 < p.n; u0 += RW_THREADS * RW_BATCH) {
            RwUnit<XT> u[RW_BATCH];
            rw_batch<XT>(u, p, u0);
            rw_write<XT>(u, d, p, u0, dense);
        }
    } else
        rw_write_other<XT>(d, p, dense);
    __syncthreads();
    if (l.mine) drow[l.id] = rw_to<DT>(dense.one(v) - scale * l.share);
}
// A part of a row of zeros.
template <class DT>
__device__ __forceinline__ void rw_zero(DT* drow, int vocab, int rank, int parts) {
    const RwPart<DT> p(drow, vocab, rank, parts);
    const uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int u = threadIdx.x; u < p.n; u += RW_THREADS)
        rw_store(const_cast<DT*>(p.x) + (long)RwUnit<DT>::N * u, w);
    if (rank == parts - 1) {
        const RwEnds<DT> e(drow, vocab);
        if ((int)threadIdx.x < e.n) drow[e.place(threadIdx.x)] = rw_to<DT>(0.0f);
    }
}

// Blocks of a row of a gradient: two batches of each thread, or one where that
// still leaves SMs without a block.  2048 rows of 262144 bf16, us, by batches a
// block: 16 340, 8 332, 4 326, 2 317, 1 334; 100 rows of 50257 fp32 (7 batches)
// by blocks a row: 1 9.0, 3 8.8, 4 7.6, 5 8.2, 8 10.5.
template <class XT>
inline int rw_grad_parts(const tk_ctx* ctx, int n_rows, int vocab) {
    const int batch = RW_THREADS * RW_BATCH * RwUnit<XT>::N, batches = (vocab + batch - 1) / batch;
    const int few = 3 * ctx->num_sms / n_rows, half = (batches + 1) / 2;
    return few > half ? few < batches ? few : batches : half;
}

inline bool rw_few(const tk_ctx* ctx, long n_rows, int parts) { return n_rows * parts <= 4L * ctx->num_sms; }

// Launch of n_rows * parts blocks, in clusters of `parts` where they meet, as a
// programmatic dependent: every block waits, first of all, for the kernel before
// to end, and is in its place by then.  Only calls of few blocks let the next
// one's come early; large ones gain nothing.
template <class A>
inline cudaError_t rw_launch(void (*kern)(A), long n_rows, int parts, bool cluster, size_t smem, const A& a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(n_rows * parts));
    cfg.blockDim = dim3(RW_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster && parts > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}

// launch(x, d) with values of the logits' and the gradient's element types.
template <class F>
inline cudaError_t rw_types(int x_dtype, int d_dtype, F launch) {
    const auto with = [&](auto x) {
        return d_dtype == TK_DT_F32 ? launch(x, float()) : d_dtype == TK_DT_F16 ? launch(x, __half()) : launch(x, __nv_bfloat16());
    };
    return x_dtype == TK_DT_F32 ? with(float()) : x_dtype == TK_DT_F16 ? with(__half()) : with(__nv_bfloat16());
}

}  // namespace tk
