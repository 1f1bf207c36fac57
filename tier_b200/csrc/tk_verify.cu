// tk_verify.cu -- tk_draft_verify: drafted tokens against the target's logits.
//
// A row's weights are powers of two: with c = log2(e) / temperature (fp32),
// y = x * c, i = floor(y), weight 2^(y - i) * 2^(i - I), I the row's largest
// i.  Only whole exponents are subtracted, so a weight's bits do not depend on
// which part of the row saw the largest logit first: a row can be streamed
// with a running I, and its sum S (64 bits, rounded once to fp32) and its
// probabilities weight / S come out the same for any split.
#include "tk_device.cuh"
#include "tk_internal.h"

namespace tk {

constexpr int DV_THREADS = 512;

struct DvArgs {
    int n_seqs, n_rows, vocab;
    const int32_t* row_start;
    const float *target, *draft;
    long ldt, ldd;
    const int32_t* tokens;
    const float *u_accept, *u_sample;
    float c;              // log2(e) / temperature; temperature 0: log2(e)
    bool greedy;
    int32_t *n_accept, *next;
    float* logp;
    struct DvStat* stat;  // [2][n_rows]: target's rows, then draft's
    int* status;
};
// What a row's pass leaves: the largest whole exponent, the weights' sum, the
// first largest logit; top = INT_MIN: a row without a distribution.
struct DvStat {
    double sum;
    float top;
    int arg;
    int bad;
};

__device__ __forceinline__ float dv_weight(float x, float c, float top) {
    const float y = __fmul_rn(x, c), i = floorf(y);
    if (!(i - top >= -100.0f)) return 0.0f;      // also y = -inf
    return exp2f(y - i) * exp2f(i - top);
}

template <class T, class F>
__device__ __forceinline__ T block_reduce(T v, T* sh, F f) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int i = 16; i; i >>= 1) v = f(v, __shfl_xor_sync(~0u, v, i));
    __syncthreads();
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    v = sh[0];
    for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v = f(v, sh[w]);
    return v;
}

__global__ void __launch_bounds__(DV_THREADS) dv_rows_kernel(const DvArgs a) {
    __shared__ double shd[32];
    __shared__ float shf[32];
    __shared__ int shi[32];
    const int row = blockIdx.x;
    const float* x = blockIdx.y ? a.draft + (size_t)row * a.ldd : a.target + (size_t)row * a.ldt;
    float mx = -INFINITY;
    int arg = INT32_MAX, bad = 0;
    for (int j = threadIdx.x; j < a.vocab; j += DV_THREADS) {
        const float v = x[j];
        if (v != v || v == INFINITY) bad = 1;
        if (v > mx) { mx = v; arg = j; }
    }
    const float big = block_reduce(mx, shf, [](float p, float q) { return fmaxf(p, q); });
    arg = block_reduce(mx == big ? arg : INT32_MAX, shi, [](int p, int q) { return min(p, q); });
    bad = block_reduce(bad, shi, [](int p, int q) { return p | q; });
    const float top = floorf(__fmul_rn(big, a.c));
    if (!(fabsf(top) <= 3.402823466e38f)) bad = 1;
    double sum = 0.0;
    if (!bad)
        for (int j = threadIdx.x; j < a.vocab; j += DV_THREADS) sum += (double)dv_weight(x[j], a.c, top);
    sum = block_reduce(sum, shd, [](double p, double q) { return p + q; });
    if (threadIdx.x == 0) a.stat[(size_t)blockIdx.y * a.n_rows + row] = DvStat{sum, top, arg, bad};
}

__device__ __forceinline__ float dv_prob(const float* x, int j, float c, const DvStat& s) {
    return __fdiv_rn(dv_weight(x[j], c, s.top), (float)s.sum);
}
__device__ __forceinline__ float dv_logp(const float* x, int j, float c, const DvStat& s) {
    return ((__fmul_rn(x[j], c) - s.top) - log2f((float)s.sum)) * 0.693147180559945309f;
}

__global__ void __launch_bounds__(DV_THREADS) dv_pick_kernel(const DvArgs a) {
    __shared__ int sh_stop, sh_bad, sh_tok;
    __shared__ unsigned long long part[DV_THREADS];
    const int b = blockIdx.x, tid = threadIdx.x, V = a.vocab;
    const int r0 = a.row_start[b], r1 = a.row_start[b + 1];
    if (r0 < 0 || r1 <= r0 || r1 > a.n_rows) {
        if (tid == 0) {
            raise_status(a.status, DEV_INVALID);
            a.n_accept[b] = 0;
            a.next[b] = -1;
        }
        return;
    }
    const DvStat* ts = a.stat;
    const DvStat* ds = a.stat + a.n_rows;
    if (tid == 0) {
        int r = r0, bad = 0;
        for (; r < r1; ++r) {
            const bool last = r == r1 - 1;
            if (ts[r].bad || (!last && a.draft && !a.greedy && ds[r].bad)) { bad = 1; break; }
            if (last) break;
            const int x = a.tokens[r + 1];
            if (x < 0 || x >= V) break;
            const float* t = a.target + (size_t)r * a.ldt;
            bool ok;
            if (a.greedy) ok = x == ts[r].arg;
            else {
                const float q = a.draft ? dv_prob(a.draft + (size_t)r * a.ldd, x, a.c, ds[r]) : 1.0f;
                ok = __fmul_rn(a.u_accept[r], q) < dv_prob(t, x, a.c, ts[r]);
            }
            if (!ok) break;
            if (a.logp) a.logp[r] = dv_logp(t, x, a.c, ts[r]);
        }
        sh_stop = r;
        sh_bad = bad;
        sh_tok = -1;
    }
    __syncthreads();
    const int r = sh_stop;
    const bool last = r == r1 - 1;
    const float* t = a.target + (size_t)r * a.ldt;
    if (!sh_bad && a.greedy) {
        if (tid == 0) sh_tok = ts[r].arg;
    } else if (!sh_bad) {
        const float* d = a.draft && !last ? a.draft + (size_t)r * a.ldd : nullptr;
        const int x = last ? -1 : a.tokens[r + 1];
        const DvStat st = ts[r], sd = d ? ds[r] : st;
        const int per = (V + DV_THREADS - 1) / DV_THREADS, j0 = min(V, tid * per), j1 = min(V, j0 + per);
        for (int pass = 0; pass < 2; ++pass) {
            auto weight = [&](int j) -> unsigned long long {
                float w = dv_prob(t, j, a.c, st);
                if (!pass) {
                    if (d) w = fmaxf(w - dv_prob(d, j, a.c, sd), 0.0f);
                    else if (j == x) w = 0.0f;
                }
                return (unsigned long long)(w * 274877906944.0f);
            };
            unsigned long long s = 0;
            for (int j = j0; j < j1; ++j) s += weight(j);
            __syncthreads();
            part[tid] = s;
            __syncthreads();
            unsigned long long before = 0, total = 0;
            for (int i = 0; i < DV_THREADS; ++i) {
                if (i < tid) before += part[i];
                total += part[i];
            }
            if (!total) continue;
            const unsigned long long u = (unsigned long long)(a.u_sample[b] * 16777216.0f);
            const unsigned long long goal = (total * u) >> 24;
            if (before <= goal && before + s > goal) {
                for (int j = j0; j < j1; ++j) {
                    before += weight(j);
                    if (before > goal) { sh_tok = j; break; }
                }
            }
            break;
        }
    }
    __syncthreads();
    if (tid == 0) {
        if (sh_bad) raise_status(a.status, DEV_INVALID);
        a.n_accept[b] = r - r0;
        a.next[b] = sh_tok;
        if (a.logp) {
            a.logp[r] = sh_tok >= 0 ? dv_logp(t, sh_tok, a.c, ts[r]) : 0.0f;
            for (int i = r + 1; i < r1; ++i) a.logp[i] = 0.0f;
        }
    }
}

size_t draft_verify_ws(int n_rows) { return align256(sizeof(DvStat) * 2 * (size_t)n_rows); }

tk_status launch_draft_verify(tk_ctx* ctx, int n_seqs, const int32_t* row_start, int n_rows, int vocab,
                              const float* target, long ldt, const float* draft, long ldd, const int32_t* tokens,
                              const float* u_accept, const float* u_sample, float temperature, int32_t* n_accept,
                              int32_t* next, float* logp, cudaStream_t s) {
    DvArgs a;
    a.n_seqs = n_seqs; a.n_rows = n_rows; a.vocab = vocab;
    a.row_start = row_start;
    a.target = target; a.draft = temperature > 0.0f ? draft : nullptr;
    a.ldt = ldt; a.ldd = ldd;
    a.tokens = tokens;
    a.u_accept = u_accept; a.u_sample = u_sample;
    a.greedy = temperature == 0.0f;
    a.c = (float)(1.4426950408889634 / (a.greedy ? 1.0 : (double)temperature));
    a.n_accept = n_accept; a.next = next; a.logp = logp;
    a.status = ctx->status;
    tk_status st = ws_ensure(ctx, draft_verify_ws(n_rows), s);
    if (st != TK_OK) return st;
    a.stat = static_cast<DvStat*>(ctx->ws);
    ProfScope ps(ctx, s, PK_SERVE);
    dv_rows_kernel<<<dim3(n_rows, a.draft ? 2 : 1), DV_THREADS, 0, s>>>(a);
    dv_pick_kernel<<<n_seqs, DV_THREADS, 0, s>>>(a);
    ctx->launches += 2;
    return cuda_fail(cudaGetLastError(), "draft verify launch");
}

}  // namespace tk
