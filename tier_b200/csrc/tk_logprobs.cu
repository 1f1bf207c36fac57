// tk_logprobs.cu -- tk_logprobs, tk_logprobs_grad: log-probabilities of given
// tokens, entropy, the likeliest tokens, and the gradient of the first two.
#include <climits>
#include "tk_rows.cuh"

namespace tk {

struct LpArgs {
    RowArgs r;
    const int32_t* tokens;
    float *logp, *entropy, *rmax, *rsum;
    int top_k;
    int32_t* top_ids;
    float* top_logp;
};

// Order of candidates: larger logits first, then lower places (unique keys).
__device__ __forceinline__ unsigned long long lp_key(float x, int j) {
    const uint32_t b = __float_as_uint(x + 0.0f);   // (-0 and 0 are alike)
    return (unsigned long long)(b ^ ((int)b < 0 ? ~0u : 0x80000000u)) << 32 | (uint32_t)~j;
}

template <class XT>
__global__ void __launch_bounds__(RW_THREADS) lp_kernel(const LpArgs a) {
    __shared__ double dpart[RW_WARPS];
    __shared__ float fpart[RW_WARPS];
    __shared__ unsigned long long best[RW_WARPS];
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, vocab = a.r.vocab;
    const XT* x = static_cast<const XT*>(a.r.x) + row * a.r.ldx;
    const int token = a.tokens ? a.tokens[row] : 0;
    const bool out = token < 0 || token >= vocab;
    if (token >= vocab && tid == 0) raise_status(a.r.status, DEV_INVALID);
    RwStat st{0.0f, 0.0, 0.0};
    if (!out) st = rw_stats(x, vocab, a.r.c, dpart, fpart);
    const bool bad = st.s != st.s;
    const float none = bad ? NAN : 0.0f;
    const double lns = out || bad ? 0.0 : log(st.s);
    if (tid == 0) {
        if (bad) raise_status(a.r.status, DEV_INVALID);
        const bool no = out || bad;
        if (a.logp) a.logp[row] = no ? none : (float)(((double)rw_float(x[token]) - st.m) * a.r.inv_t - lns);
        if (a.entropy) a.entropy[row] = no ? none : (float)(lns - 0.6931471805599453 * st.a / st.s);
        if (a.rmax) a.rmax[row] = no ? none : st.m;
        if (a.rsum) a.rsum[row] = no ? none : (float)st.s;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.top_k; ++k) {
        unsigned long long top = 0;
        if (!out && !bad) {
            for (int j = tid; j < vocab; j += RW_THREADS) {
                const unsigned long long key = lp_key(rw_float(x[j]), j);
                if (key < last && key > top) top = key;
            }
            for (int i = 16; i; i >>= 1) top = max(top, __shfl_xor_sync(~0u, top, i));
            __syncthreads();
            if ((tid & 31) == 0) best[tid >> 5] = top;
            __syncthreads();
            for (int w = 0; w < RW_WARPS; ++w) top = max(top, best[w]);
        }
        if (tid == 0) {
            const int j = (int)~(uint32_t)top;
            a.top_ids[row * a.top_k + k] = out || bad ? -1 : j;
            if (a.top_logp)
                a.top_logp[row * a.top_k + k] = out || bad ? none : (float)(((double)rw_float(x[j]) - st.m) * a.r.inv_t - lns);
        }
        last = top;
    }
}

struct LgArgs {
    RowArgs r;
    const int32_t* tokens;
    const float *rmax, *rsum, *entropy, *d_logp, *d_entropy;
};

template <class XT, class DT>
__global__ void __launch_bounds__(RW_THREADS) lg_kernel(const LgArgs a) {
    const size_t row = blockIdx.x;
    const int vocab = a.r.vocab;
    const XT* x = static_cast<const XT*>(a.r.x) + row * a.r.ldx;
    DT* dx = static_cast<DT*>(a.r.dx) + row * a.r.ldd;
    const int token = a.tokens ? a.tokens[row] : 0;
    const float dl = a.d_logp ? a.d_logp[row] : 0.0f, de = a.d_entropy ? a.d_entropy[row] : 0.0f;
    if (token >= vocab && threadIdx.x == 0) raise_status(a.r.status, DEV_INVALID);
    if (token < 0 || token >= vocab || (dl == 0.0f && de == 0.0f)) {
        rw_zero(dx, vocab);
        return;
    }
    const float m = a.rmax[row], c = a.r.c, s = a.rsum[row];
    // p (-dl - de (ln p + H)) / T = 2^y (f + g y)
    const float h = a.d_entropy ? a.entropy[row] - logf(s) : 0.0f;
    const float f = -(dl + de * h) / s * a.r.inv_t, g = -de * 0.69314718f / s * a.r.inv_t;
    __shared__ int ids[1];
    __shared__ float sub[1];
    if (threadIdx.x == 0) {
        ids[0] = a.d_logp ? token : -1;
        sub[0] = -dl * a.r.inv_t;
    }
    __syncthreads();
    rw_gradient(x, dx, vocab, ids, sub, 1, [=](float v) {
        const float y = rw_exponent(v, m, c);
        return rw_exp2(y) * (f + g * y);
    });
}

template <class XT>
static cudaError_t launch_lp(const LpArgs& a, cudaStream_t s) {
    lp_kernel<XT><<<a.r.n_rows, RW_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}
tk_status launch_logprobs(tk_ctx* ctx, const RowArgs& r, int x_dtype, const int32_t* tokens, float* logp, float* entropy,
                          float* rmax, float* rsum, int top_k, int32_t* top_ids, float* top_logp, cudaStream_t s) {
    const LpArgs a{r, tokens, logp, entropy, rmax, rsum, top_k, top_ids, top_logp};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    const cudaError_t e = x_dtype == TK_DT_F32 ? launch_lp<float>(a, s)
                        : x_dtype == TK_DT_F16 ? launch_lp<__half>(a, s) : launch_lp<__nv_bfloat16>(a, s);
    return cuda_fail(e, "log-probabilities launch");
}

template <class XT, class DT>
static cudaError_t launch_lg(const LgArgs& a, cudaStream_t s) {
    lg_kernel<XT, DT><<<a.r.n_rows, RW_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}
tk_status launch_logprobs_grad(tk_ctx* ctx, const RowArgs& r, int x_dtype, const int32_t* tokens, const float* rmax,
                               const float* rsum, const float* entropy, const float* d_logp, const float* d_entropy,
                               int d_dtype, cudaStream_t s) {
    const LgArgs a{r, tokens, rmax, rsum, entropy, d_logp, d_entropy};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    return cuda_fail(rw_types(x_dtype, d_dtype, [&](auto x, auto d) { return launch_lg<decltype(x), decltype(d)>(a, s); }),
                     "log-probability gradient launch");
}

}  // namespace tk
