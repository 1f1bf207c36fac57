// tk_rows.cuh -- rows of logits: element types, the weights of a softmax, and
// the arguments of the operators on them (tk_logprobs.cu, tk_distill.cu).
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

// A logit's exponent to the base 2 below the row's largest, m.  The difference
// comes first: it is exact where it matters, however large the logits are, and
// a mask of fp32's lowest value only makes it -inf.  Clamped at -200, where the
// weight 2^y is zero in fp32, so that y may be multiplied by the weight; a NaN
// stays one (a row that holds NaN or +inf has the sum NaN).
constexpr float RW_LOW = -200.0f;
__device__ __forceinline__ float rw_exponent(float x, float m, float c) { return rw_max_nan((x - m) * c, RW_LOW); }

// What a row's sums are relative to before a logit was seen: the lowest
// finite number, so that -inf has the weight 0 and not NaN.
constexpr float RW_LOWEST = -3.402823466e38f;

template <class T>
__device__ __forceinline__ T rw_block_sum(T v, T* part) {             // the same in every thread
    for (int i = 16; i; i >>= 1) v += __shfl_xor_sync(~0u, v, i);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < RW_WARPS; ++w) v += part[w];
    return v;
}
__device__ __forceinline__ float rw_block_max(float v, float* part) {   // NaN is passed over
    for (int i = 16; i; i >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, i));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < RW_WARPS; ++w) v = fmaxf(v, part[w]);
    return v;
}

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

// Running sums of one thread.  m moves only when a batch of logits holds a
// larger one; s and a are sums of at most a few batches before they go, in 64
// bits, to the totals, which have a reference of their own.
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
        const double f = rw_exp2(d);
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
    template <class XT>
    __device__ __forceinline__ void batch(const RwUnit<XT> (&u)[RW_BATCH], f32x2 c) {     // none above m
        const f32x2 nm = pack2(-m, -m);
        f32x2 s2[2] = {0, 0}, a2[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < RW_BATCH; ++j)
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

// m, S and A of all parts brought together: threads of a block, blocks of a
// cluster.  A row that holds NaN or +inf has S = NaN by its arithmetic.
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

// m, S = sum 2^y and, relative to it, A = sum 2^y y of a whole row (the same in
// every thread); a row that holds NaN, +inf or nothing above -inf: S = NaN.
template <class XT>
__device__ __forceinline__ RwStat rw_stats(const XT* x, int vocab, float c, double* dpart, float* fpart) {
    float m = RW_LOWEST;
    for (int j = threadIdx.x; j < vocab; j += RW_THREADS) m = fmaxf(m, rw_float(x[j]));
    m = rw_block_max(m, fpart);
    double s = 0.0, a = 0.0;
    for (int j = threadIdx.x; j < vocab; j += RW_THREADS) {
        const float v = rw_float(x[j]), y = rw_exponent(v, m, c), e = v == -INFINITY ? 0.0f : rw_exp2(y);
        s += e;
        a += e * y;
    }
    s = rw_block_sum(s, dpart);
    a = rw_block_sum(a, dpart);
    if (s == 0.0) s = (double)NAN;                 // nothing above -inf
    return RwStat{m, s, a};
}

// dx[j] = dense(x[j]), at the listed places less sub[]: entries of the same
// place are added up in the list's order by the first of them.  dx may be x
// itself: a listed logit is read before any place is written.
template <class XT, class DT, class F>
__device__ __forceinline__ void rw_gradient(const XT* x, DT* dx, int vocab, const int* ids, const float* sub, int k, F dense) {
    const int tid = threadIdx.x;
    bool first = tid < k && ids[tid] >= 0;
    float q = 0.0f, v = 0.0f;
    if (first) {
        v = rw_float(x[ids[tid]]);
        for (int j = 0; j < k; ++j)
            if (ids[j] == ids[tid]) {
                first &= j >= tid;
                q += sub[j];
            }
    }
    __syncthreads();
    for (int j = tid; j < vocab; j += RW_THREADS) dx[j] = rw_to<DT>(dense(rw_float(x[j])));
    __syncthreads();
    if (first) dx[ids[tid]] = rw_to<DT>(dense(v) - q);
}
template <class DT>
__device__ __forceinline__ void rw_zero(DT* dx, int vocab) {
    for (int j = threadIdx.x; j < vocab; j += RW_THREADS) dx[j] = rw_to<DT>(0.0f);
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
