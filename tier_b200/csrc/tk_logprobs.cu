// tk_logprobs.cu -- tk_logprobs, tk_logprobs_grad: log-probabilities of given
// tokens, entropy, the likeliest tokens, and the gradient of the first two.
#include <climits>
#include "tk_rows.cuh"

namespace tk {

constexpr int LP_GROUPS = 8;          // groups of logits a thread keeps the largest of
constexpr int LP_KEEP = 2048;         // candidates a block can hold
constexpr int LP_MARGIN = 64;         // and hands on beyond top_k
constexpr int LP_CLUSTER = 16;        // blocks of a row at most

struct LpArgs {
    RowArgs r;
    const int32_t* tokens;
    float *logp, *entropy, *rmax, *rsum;
    int top_k;
    int32_t* top_ids;
    float* top_logp;
    int parts;                // blocks of a row (a cluster)
    int batches;              // batches of a group
    bool fine;                // a group is one unit
};

// Order of logits as whole numbers (-0 and 0 are alike).
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((int)b < 0 ? ~0u : 0x80000000u);
}
__device__ __forceinline__ float lp_value(uint32_t o) { return __uint_as_float(o ^ ((int)o < 0 ? 0x80000000u : ~0u)); }
// Order of candidates: larger logits first, then lower places; no two alike.
__device__ __forceinline__ unsigned long long lp_key(uint32_t order, int place) {
    return (unsigned long long)order << 32 | (uint32_t)~place;
}

// Shared memory of the search for the largest logits.
struct LpTop {
    float big[LP_GROUPS][RW_THREADS];              // each group's largest logit
    unsigned long long keep[LP_KEEP];              // candidates
    uint16_t list[LP_GROUPS * RW_THREADS];         // groups to look through again
    int part[2][RW_WARPS];
    int n, listed;
};

// Sum over the block; `turn` alternates between calls (one barrier a call).
__device__ __forceinline__ int lp_count(LpTop& t, int v, int& turn) {
    turn ^= 1;
    v = __reduce_add_sync(~0u, v);
    if ((threadIdx.x & 31) == 0) t.part[turn][threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < RW_WARPS; ++w) v += t.part[turn][w];
    return v;
}

// The k largest of the t.n > k candidates stay; returns the least of them.
__device__ __noinline__ unsigned long long lp_thin(LpTop& t, int k, int& turn) {
    constexpr int EACH = LP_KEEP / RW_THREADS;
    unsigned long long mine[EACH], least = 0;
    const int n = t.n;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int at = i * RW_THREADS + threadIdx.x;
        mine[i] = at < n ? t.keep[at] : 0;
    }
    for (int bit = 63; bit >= 0; --bit) {          // the largest key that k candidates reach
        const unsigned long long to = least | 1ull << bit;
        int c = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) c += mine[i] >= to;
        c = lp_count(t, c, turn);
        if (c >= k) least = to;
        if (c == k) break;
    }
    if (threadIdx.x == 0) t.n = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (mine[i] >= least) t.keep[atomicAdd(&t.n, 1)] = mine[i];
    __syncthreads();
    return least;
}

// The block's candidates: a set that holds the top_k largest logits of its part
// (or all).  With each group's largest known, the top_k-th largest of these is
// a bound that top_k logits reach: only groups that reach it are looked
// through again, about top_k of them, whatever the row looks like; rows of
// many equal logits can make it more.  Candidates that do not fit are thinned
// on the way.
template <class XT>
__device__ void lp_search(LpTop& t, const LpArgs& a, const XT* row, const RwPart<XT>& p, bool ends) {
    constexpr int NB = RwUnit<XT>::BATCH;
    const int tid = threadIdx.x, k = a.top_k;
    const int batches = (p.n + RW_THREADS * NB - 1) / (RW_THREADS * NB);
    const int groups = a.fine ? batches * NB : (batches + a.batches - 1) / a.batches;   // a thread's
    int turn = 0;
    if (tid == 0) t.n = t.listed = 0;
    uint32_t o[LP_GROUPS];
#pragma unroll
    for (int g = 0; g < LP_GROUPS; ++g) o[g] = g < groups ? lp_order(t.big[g][tid]) : 0;
    uint32_t bound = 0;                            // enough groups reach it, and not many too many
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t to = bound | 1u << bit;
        int c = 0;
#pragma unroll
        for (int g = 0; g < LP_GROUPS; ++g) c += o[g] >= to;
        c = lp_count(t, c, turn);
        if (c >= k) bound = to;
        if (c >= k && c <= k + k / 8 + 4) break;
    }
#pragma unroll
    for (int g = 0; g < LP_GROUPS; ++g)
        if (g < groups && o[g] >= bound) t.list[atomicAdd(&t.listed, 1)] = (uint16_t)(g * RW_THREADS + tid);
    __syncthreads();
    if (ends && tid < 16) {
        const RwEnds<XT> e(row, a.r.vocab);
        if (tid < e.n) {
            const int j = e.place(tid);
            t.keep[atomicAdd(&t.n, 1)] = lp_key(lp_order(rw_float(row[j])), j);
        }
    }
    // unit i of the listed groups
    const int each = a.fine ? 1 : a.batches * NB, total = t.listed * each;
    const auto unit_of = [&](int i) {
        const int g = t.list[i / each], who = g % RW_THREADS, part = g / RW_THREADS, in = i % each;
        return (a.fine ? part : part * each + in) * RW_THREADS + who;
    };
    bool full = false;
    for (int i = tid; i < total && !full; i += RW_THREADS) {
        const int u = unit_of(i);
        if (u >= p.n) continue;
        RwUnit<XT> w;
        w.load(p.x + 8L * u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x[2];
            unpack2(w.two(e), x[0], x[1]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (lp_order(x[h]) >= bound) {
                    const int at = atomicAdd(&t.n, 1);
                    if (at < LP_KEEP) t.keep[at] = lp_key(lp_order(x[h]), p.first + 8 * u + 2 * e + h);
                    full |= at >= LP_KEEP;
                }
        }
    }
    if (__syncthreads_or(full)) {                  // too many: once more, thinned on the way
        unsigned long long least = (unsigned long long)bound << 32;
        if (tid == 0) t.n = 0;
        __syncthreads();
        const RwEnds<XT> e(row, a.r.vocab);
        if (ends && tid < e.n) t.keep[atomicAdd(&t.n, 1)] = lp_key(lp_order(rw_float(row[e.place(tid)])), e.place(tid));
        __syncthreads();
        for (int i0 = 0; i0 < total; i0 += RW_THREADS) {
            const int u = i0 + tid < total ? unit_of(i0 + tid) : p.n;
#pragma unroll 1
            for (int j = 0; j < 8; ++j) {
                unsigned long long key = 0;
                if (u < p.n) key = lp_key(lp_order(rw_float(p.x[8L * u + j])), p.first + 8 * u + j);
                const int n = t.n, more = lp_count(t, key >= least, turn);     // (n before the barrier: pushes come after it)
                if (n + more > LP_KEEP) least = lp_thin(t, k, turn);
                if (key >= least) t.keep[atomicAdd(&t.n, 1)] = key;
                __syncthreads();
            }
        }
    }
    if (t.n > k + LP_MARGIN) lp_thin(t, k, turn);
}

// The same variable of another block of the cluster.
template <class T>
__device__ __forceinline__ T* lp_peer(T* mine, int rank) {
    T* p;
    asm("mapa.u64 %0, %1, %2;" : "=l"(p) : "l"(mine), "r"(rank));
    return p;
}

// A cluster of blocks per row, each with one part of it.  Every logit is read
// once, for the sums and for the largest of each group of logits; the blocks'
// sums and candidates meet in shared memory.
template <class XT, bool ENT, bool TOP>
__global__ void __launch_bounds__(RW_THREADS, 4) lp_kernel(const LpArgs a) {
    constexpr int NB = RwUnit<XT>::BATCH;
    extern __shared__ __align__(16) char lp_smem[];
    __shared__ RwStat join[RW_WARPS], part;
    LpTop& t = *reinterpret_cast<LpTop*>(lp_smem);                                       // TOP
    const size_t row = blockIdx.x / a.parts;
    const int tid = threadIdx.x, vocab = a.r.vocab, rank = blockIdx.x % a.parts, k = a.top_k;
    const float c = a.r.c;
    const int token = a.tokens ? a.tokens[row] : 0;
    if (token < 0 || token >= vocab) {             // the whole cluster alike
        if (rank) return;
        if (tid == 0) {
            if (token >= vocab) raise_status(a.r.status, DEV_INVALID);
            if (a.logp) a.logp[row] = 0.0f;
            if (a.entropy) a.entropy[row] = 0.0f;
            if (a.rmax) a.rmax[row] = 0.0f;
            if (a.rsum) a.rsum[row] = 0.0f;
        }
        for (int i = tid; TOP && i < k; i += RW_THREADS) {
            a.top_ids[row * k + i] = -1;
            if (a.top_logp) a.top_logp[row * k + i] = 0.0f;
        }
        return;
    }
    const XT* x = static_cast<const XT*>(a.r.x) + row * a.r.ldx;
    const float given = a.logp ? rw_float(x[token]) : 0.0f;
    const RwPart<XT> p(x, vocab, rank, a.parts);
    const bool ends = rank == a.parts - 1;
    RwSums<ENT> sums;
    if (ends) {
        const RwEnds<XT> e(x, vocab);
        if (tid < e.n) {
            const float v = rw_float(x[e.place(tid)]);
            if (v > sums.m) sums.raise(v, c);
            f32x2 s2 = 0, a2 = 0;
            sums.two(pack2(v, -INFINITY), pack2(-sums.m, -sums.m), pack2(c, c), s2, a2);
            float lo, hi;
            unpack2(s2, sums.s, hi);
            unpack2(a2, lo, hi);
            if (ENT) sums.a = lo;
        }
    }
    const f32x2 c2 = pack2(c, c);
    float big = -INFINITY;
    int in = 0, g = 0;
    for (int u0 = 0; u0 < p.n; u0 += RW_THREADS * NB) {
        RwUnit<XT> u[NB];
        const XT* from = p.x + 8L * (u0 + tid);
        if (u0 + RW_THREADS * NB <= p.n) {
#pragma unroll
            for (int j = 0; j < NB; ++j) u[j].load(from + 8 * RW_THREADS * j);
        } else {
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                if (u0 + j * RW_THREADS + tid < p.n) u[j].load(from + 8 * RW_THREADS * j);
                else u[j].lowest();
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const float v = u[j].max();
            if (TOP && a.fine) t.big[g + j][tid] = v;
            top = fmaxf(top, v);
        }
        if (top > sums.m) sums.raise(top, c);
        sums.batch(u, c2);
        big = fmaxf(big, top);
        if (++in == a.batches) {
            if (TOP && !a.fine) t.big[g++][tid] = big;
            if (TOP && a.fine) g += NB;
            big = -INFINITY;
            in = 0;
            sums.flush(c);
        }
    }
    if (TOP && !a.fine && in) t.big[g][tid] = big;
    sums.flush(c);
    const RwStat w = rw_warp_join<ENT>(RwStat{sums.M, sums.S, sums.A}, c);
    if ((tid & 31) == 0) join[tid >> 5] = w;
    __syncthreads();
    const auto joined = [&](auto get, int n) {     // n of them, the same in every thread
        RwStat v{RW_LOWEST, 0.0, 0.0};
        for (int i = 0; i < n; ++i) v.m = fmaxf(v.m, get(i).m);
        for (int i = 0; i < n; ++i) {
            const RwStat o = rw_to_max(get(i), v.m, c);
            v.s += o.s;
            v.a += o.a;
        }
        return v;
    };
    RwStat st = joined([&](int i) { return join[i]; }, RW_WARPS);
    if (TOP) lp_search(t, a, x, p, ends);
    if (a.parts > 1) {
        if (tid == 0) part = st;
        cluster_sync();
        st = joined([&](int i) { return *lp_peer(&part, i); }, a.parts);
    }
    if (st.s == 0.0) st.s = (double)NAN;           // nothing above -inf
    const bool bad = st.s != st.s;
    const double lns = log(st.s);
    if (rank == 0 && tid == 0) {
        if (bad) raise_status(a.r.status, DEV_INVALID);
        if (a.logp) a.logp[row] = (float)(((double)given - st.m) * a.r.inv_t - lns);
        if (ENT) a.entropy[row] = (float)(lns - 0.6931471805599453 * st.a / st.s);
        if (a.rmax) a.rmax[row] = bad ? NAN : st.m;
        if (a.rsum) a.rsum[row] = (float)st.s;
    }
    if (TOP) {
        int32_t* ids = a.top_ids + row * k;
        float* lp = a.top_logp ? a.top_logp + row * k : nullptr;
        if (bad) {
            for (int i = tid; rank == 0 && i < k; i += RW_THREADS) {
                ids[i] = -1;
                if (lp) lp[i] = NAN;
            }
        } else {
            // a candidate's place in the row's order: how many are before it, in all blocks
            const unsigned long long* all = t.keep;
            int n = t.n;
            if (a.parts > 1) {
                unsigned long long* got = reinterpret_cast<unsigned long long*>(lp_smem + sizeof(LpTop));
                n = 0;
                for (int r = 0; r < a.parts; ++r) {
                    const LpTop& o = *lp_peer(&t, r);
                    const int m = o.n;
                    for (int i = tid; i < m; i += RW_THREADS) got[n + i] = o.keep[i];
                    n += m;
                }
                __syncthreads();
                all = got;
            }
            for (int i = tid >> 5; i < t.n; i += RW_WARPS) {
                const unsigned long long key = t.keep[i];
                int before = 0;
                for (int j = tid & 31; j < n; j += 32) before += all[j] > key;
                before = __reduce_add_sync(~0u, before);
                if (before < k && (tid & 31) == 0) {
                    ids[before] = (int)~(uint32_t)key;
                    if (lp) lp[before] = (float)(((double)lp_value((uint32_t)(key >> 32)) - st.m) * a.r.inv_t - lns);
                }
            }
        }
    }
    __syncwarp();
    if (a.parts > 1) cluster_sync();               // no block ends while another reads its memory
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

// Blocks of a row: enough that the batch fills the GPU, parts of 2^19 logits at
// most and of a batch of units at least.
static int lp_parts(const tk_ctx* ctx, int n_rows, int vocab) {
    int parts = 1;
    while (parts < LP_CLUSTER && (vocab / parts > 1 << 19 || ((long)n_rows * parts < 4L * ctx->num_sms && vocab / parts > 8192)))
        parts *= 2;
    return parts;
}

template <class XT, bool ENT, bool TOP>
static cudaError_t launch_lp(const tk_ctx* ctx, LpArgs& a, cudaStream_t s) {
    a.parts = lp_parts(ctx, a.r.n_rows, a.r.vocab);
    const int per = RW_THREADS * RwUnit<XT>::BATCH;
    const int units = ((a.r.vocab / 8 + a.parts - 1) / a.parts + 31) & ~31, batches = (units + per - 1) / per;
    a.fine = batches * RwUnit<XT>::BATCH <= LP_GROUPS;
    a.batches = a.fine ? 1 : (batches + LP_GROUPS - 1) / LP_GROUPS;
    int smem = TOP ? (int)sizeof(LpTop) : 0;
    if (TOP && a.parts > 1) smem += a.parts * (a.top_k + LP_MARGIN) * (int)sizeof(unsigned long long);
    const auto kern = lp_kernel<XT, ENT, TOP>;
    static std::atomic<uint64_t> attr_smem{0}, attr_size{0};
    constexpr int MOST = (int)sizeof(LpTop) + LP_CLUSTER * (TK_TOP_MAX + LP_MARGIN) * (int)sizeof(unsigned long long);
    cudaError_t e = smem_attr_once(kern, MOST, ctx->device, attr_smem);
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (e == cudaSuccess && !(attr_size.load(std::memory_order_relaxed) & bit)) {   // more than 8 blocks: on request
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) attr_size.fetch_or(bit);
    }
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long)a.r.n_rows * a.parts));
    cfg.blockDim = dim3(RW_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.parts;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, a);
}
tk_status launch_logprobs(tk_ctx* ctx, const RowArgs& r, int x_dtype, const int32_t* tokens, float* logp, float* entropy,
                          float* rmax, float* rsum, int top_k, int32_t* top_ids, float* top_logp, cudaStream_t s) {
    LpArgs a{r, tokens, logp, entropy, rmax, rsum, top_k, top_ids, top_logp, 1, 1, false};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    const auto with = [&](auto x) {
        using XT = decltype(x);
        return entropy ? top_k ? launch_lp<XT, true, true>(ctx, a, s) : launch_lp<XT, true, false>(ctx, a, s)
                       : top_k ? launch_lp<XT, false, true>(ctx, a, s) : launch_lp<XT, false, false>(ctx, a, s);
    };
    const cudaError_t e = x_dtype == TK_DT_F32 ? with(float()) : x_dtype == TK_DT_F16 ? with(__half()) : with(__nv_bfloat16());
    if (e != cudaSuccess) return cuda_fail(e, "log-probabilities launch");
    return cuda_fail(cudaGetLastError(), "log-probabilities launch");
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
