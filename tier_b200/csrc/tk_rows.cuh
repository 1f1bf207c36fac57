// tk_rows.cuh -- rows of logits: element types, the weights of a softmax, and
// the arguments of the operators on them (tk_logprobs.cu, tk_distill.cu).
#pragma once
#include "tk_device.cuh"
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

// m, S = sum 2^y and, relative to it, A = sum 2^y y of a whole row (the same in
// every thread); a row that holds NaN, +inf or nothing above -inf: S = NaN.
struct RwStat {
    float m;
    double s, a;
};
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
