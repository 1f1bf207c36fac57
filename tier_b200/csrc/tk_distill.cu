// tk_distill.cu -- tk_distill, tk_distill_grad: distillation from a teacher's
// top logits.
#include "tk_rows.cuh"

namespace tk {

struct DsArgs {
    RowArgs r;
    int k;
    const int32_t* ids;
    const float *teacher, *weight;
    float *loss, *rmax, *rsum;
    const float *in_max, *in_sum;     // tk_distill_grad: of the forward pass
};

// The teacher's row: its entries' places (-1: none), q and (in the entry's own
// thread) ln q.  Returns 0: no entry, 1: entries, 2: NaN or +inf among them.
__device__ __forceinline__ int ds_teacher(const DsArgs& a, size_t row, int* ids, float* q, double& lnq, double* dpart,
                                          float* fpart) {
    const int tid = threadIdx.x;
    int id = -1;
    float t = -INFINITY;
    if (tid < a.k) {
        id = a.ids[row * a.k + tid];
        if (id >= a.r.vocab) {
            raise_status(a.r.status, DEV_INVALID);
            id = -1;
        }
        if (id >= 0) t = a.teacher[row * a.k + tid];
    }
    const bool bad = !(t < INFINITY);
    const float m = rw_block_max(fmaxf(t, RW_LOWEST), fpart);
    const float e = t == -INFINITY ? 0.0f : rw_exp2(rw_exponent(t, m, a.r.c));
    const double s = rw_block_sum((double)e, dpart);
    lnq = ((double)t - m) * a.r.inv_t - log(s);
    if (tid < a.k) {
        ids[tid] = id;
        q[tid] = (float)(e / s);
    }
    const int any_bad = __syncthreads_or(bad), any = __syncthreads_or(e > 0.0f);
    return any_bad ? 2 : any ? 1 : 0;
}

template <class XT, class DT>
__global__ void __launch_bounds__(RW_THREADS) ds_kernel(const DsArgs a) {
    __shared__ double dpart[RW_WARPS];
    __shared__ float fpart[RW_WARPS];
    __shared__ int ids[TK_TOP_MAX];
    __shared__ float q[TK_TOP_MAX];
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, vocab = a.r.vocab;
    const XT* x = static_cast<const XT*>(a.r.x) + row * a.r.ldx;
    DT* dx = a.r.dx ? static_cast<DT*>(a.r.dx) + row * a.r.ldd : nullptr;
    double lnq;
    const int state = ds_teacher(a, row, ids, q, lnq, dpart, fpart);
    const float w = state ? (a.weight ? a.weight[row] : 1.0f) * a.r.inv_t : 0.0f;
    RwStat st{0.0f, 0.0, 0.0};
    if (a.in_max) {
        st.m = a.in_max[row];
        st.s = a.in_sum[row];
        if (state == 2) st.s = (double)NAN;
        if (state == 2 && tid == 0) raise_status(a.r.status, DEV_INVALID);
    } else {
        if (state) st = rw_stats(x, vocab, a.r.c, dpart, fpart);
        if (state == 2) st.s = (double)NAN;
        const bool bad = st.s != st.s;
        double part = 0.0;
        if (state == 1 && tid < a.k && q[tid] > 0.0f)
            part = q[tid] * (lnq - (((double)rw_float(x[ids[tid]]) - st.m) * a.r.inv_t - log(st.s)));
        part = rw_block_sum(part, dpart);
        if (tid == 0) {
            if (bad) raise_status(a.r.status, DEV_INVALID);
            const float none = bad ? NAN : 0.0f;
            const bool no = !state || bad;
            if (a.loss) a.loss[row] = no ? none : (float)part;
            if (a.rmax) a.rmax[row] = no ? none : st.m;
            if (a.rsum) a.rsum[row] = no ? none : (float)st.s;
        }
    }
    if (!dx) return;
    if (w == 0.0f) {
        rw_zero(dx, vocab);
        return;
    }
    if (tid < a.k) q[tid] *= w;
    __syncthreads();
    const float f = (float)(w / st.s), m = st.m, c = a.r.c;
    rw_gradient(x, dx, vocab, ids, q, a.k, [=](float v) { return rw_exp2(rw_exponent(v, m, c)) * f; });
}

template <class XT, class DT>
static cudaError_t launch_ds(const DsArgs& a, cudaStream_t s) {
    ds_kernel<XT, DT><<<a.r.n_rows, RW_THREADS, 0, s>>>(a);
    return cudaGetLastError();
}
tk_status launch_distill(tk_ctx* ctx, const RowArgs& r, int x_dtype, int k, const int32_t* ids, const float* teacher,
                         const float* weight, float* loss, float* rmax, float* rsum, int d_dtype, cudaStream_t s) {
    const DsArgs a{r, k, ids, teacher, weight, loss, rmax, rsum, nullptr, nullptr};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    return cuda_fail(rw_types(x_dtype, d_dtype, [&](auto x, auto d) { return launch_ds<decltype(x), decltype(d)>(a, s); }),
                     "distillation launch");
}
tk_status launch_distill_grad(tk_ctx* ctx, const RowArgs& r, int x_dtype, int k, const int32_t* ids, const float* teacher,
                              const float* rmax, const float* rsum, const float* weight, int d_dtype, cudaStream_t s) {
    const DsArgs a{r, k, ids, teacher, weight, nullptr, nullptr, nullptr, rmax, rsum};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    return cuda_fail(rw_types(x_dtype, d_dtype, [&](auto x, auto d) { return launch_ds<decltype(x), decltype(d)>(a, s); }),
                     "distillation gradient launch");
}

}  // namespace tk
