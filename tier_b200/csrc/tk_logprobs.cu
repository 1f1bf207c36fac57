// tk_logprobs.cu -- tk_logprobs, tk_logprobs_grad: log-probabilities of given
// tokens, entropy, the likeliest tokens, and the gradient of the first two.
//
// With y = (l - m) / T and weights e^y, S = sum e^y and A = sum e^y y:
// ln p = y - ln S and the entropy is ln S - A / S, two positive terms.  Both sums
// come from one reading: m is a running maximum of each thread, to which its
// sums are scaled again when it moves, and parts are brought together in 64
// bits.  The bound is memory; for 16-bit rows an exponential a logit (16 a
// clock and SM, 62 % of them busy) and six other instructions come near it.
//
// The largest logits cost little beside that reading: of each 32-byte unit its
// maximum is kept, cut to 16 bits, a bound is found that enough logits reach,
// and only units that reach it are read again.  (Kept per thread and batch
// instead, a list of 128 read a fifth of a bf16 row again: 1024 rows of 262144
// 129 us, now 103; every alternative by a pass of its own 27 ms.)  What the
// search holds in shared memory is small on purpose: loads on their way need
// the L1 (53 KB a block instead of 43: 1024 rows 112 us, 4096 404 instead of 369).
//
// The gradient reads every logit and writes every gradient once.
//
// Measured (us; calls in a graph, L2 warm): 1 row of 262144 fp32, 20
// alternatives 9.8 (of them the reading 3, the search 3, the meeting of 8 blocks
// 1); 48 of 50257, 5 alternatives 9.7; 4095 x 262144 fp32, none 533 (7.2 TB/s;
// from Python on machines that were idle before 535 to 555); 1024 x 262144 bf16
// without 86 (6.3 TB/s), 20 97, 128 103 (from Python 98 without, 104 to 114
// with 128), 256 112. Gradients of 2048 x 131072 bf16, 30 % of the rows left
// out, 141 (6.5 TB/s).
#include "tk_rows.cuh"

namespace tk {

constexpr int LP_SLOTS = 16;          // for the largest logits of a thread's batches
constexpr int LP_LIST = 1024;         // units that can be listed to be looked through again
constexpr int LP_KEEP = 1024;         // candidates a block can hold
constexpr int LP_SORT = 2 * RW_THREADS;   // and puts in order
constexpr int LP_AHEAD = 2;           // units on their way when they are looked through again
constexpr int LP_CLUSTER = 8;         // blocks of a row at most

struct LpArgs {
    RowArgs r;
    const int32_t* tokens;
    float *logp, *entropy, *rmax, *rsum;
    int top_k;
    int32_t* top_ids;
    float* top_logp;
    int parts;                // blocks of a row (a cluster)
    int shift;                // 2^shift batches share a slot
};

// Order of logits as whole numbers (-0 and 0 are alike).
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ ((int)b < 0 ? ~0u : 0x80000000u);
}
constexpr uint32_t LP_NOTHING = 0x007fffffu;       // of -inf
__device__ __forceinline__ float lp_value(uint32_t o) { return __uint_as_float(o ^ ((int)o < 0 ? 0x80000000u : ~0u)); }
// Order of candidates: larger logits first, then lower places; no two alike.
__device__ __forceinline__ unsigned long long lp_key(uint32_t order, int place) {
    return (unsigned long long)order << 32 | (uint32_t)~place;
}

// Shared memory of the search for the largest logits.
struct LpTop {
    uint2 big[LP_SLOTS][RW_THREADS];               // the largest logit of each unit of a batch, upper 16 bits
    unsigned long long keep[LP_KEEP];              // candidates
    uint16_t list[LP_LIST];                        // slots' units to look through again
    uint32_t low[RW_WARPS], high[RW_WARPS];
    int peers[LP_CLUSTER];                         // candidates of the cluster's blocks (which follow this)
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
// (or all).  With v0 and v1, the largest logits of the first and the second
// halves of each thread's units, a bound is found that top_k of these reach, so
// top_k logits do (256 or 512 numbers, one counting barrier a bit); only units
// that reach it are read again, little more than top_k of them for logits in
// any order, a sector of memory each.  Where many logits are alike or the
// largest stand together, candidates that do not fit are thinned on the way; so
// too where fewer than top_k numbers are above -inf, which gives no bound (from
// Python, us: 1 row of 262144 with 8 finite logits of 20 26, 48 of 50257 with 4
// of 5 24.5, 1024 with 100 of 128 255).
template <class XT>
__device__ __forceinline__ void lp_search(LpTop& t, const LpArgs& a, const XT* row, const RwPart<XT>& p, bool ends,
                                          float v0, float v1) {
    constexpr int N = RwUnit<XT>::N;
    const int tid = threadIdx.x, k = a.top_k;
    if (tid == 0) t.n = t.listed = 0;
    const bool both = k > RW_THREADS / 2;          // (256 of 256 would be no bound)
    const uint32_t o0 = lp_order(both ? v0 : fmaxf(v0, v1)), o1 = both ? lp_order(v1) : 0;
    uint32_t low = __reduce_min_sync(~0u, min(o0 > LP_NOTHING ? o0 : ~0u, o1 > LP_NOTHING ? o1 : ~0u));
    uint32_t high = __reduce_max_sync(~0u, max(o0, o1));
    if ((tid & 31) == 0) {
        t.low[tid >> 5] = low;
        t.high[tid >> 5] = high;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < RW_WARPS; ++w) {
        low = min(low, t.low[w]);
        high = max(high, t.high[w]);
    }
    const auto reach = [&](uint32_t to) {
        const int c = __syncthreads_count(o0 >= to);
        return both ? c + __syncthreads_count(o1 >= to) : c;
    };
    // from the highest bit in which they differ; 0 where those above -inf are few
    uint32_t bound = 0;
    if (low <= high && reach(low) >= k) {
        const int bits = 32 - __clz(low ^ high);
        bound = bits < 32 ? low >> bits << bits : 0;
        for (int bit = bits - 1; bit >= 0; --bit) {
            const uint32_t to = bound | 1u << bit;
            const int c = reach(to);
            if (c < k) continue;
            bound = to;
            if (c <= k + k / 8 + 8) break;
        }
    }
    // the row's ends come first, whatever they hold: 30 at most, which fit (behind
    // the units' they might not, and the units' are counted on where they do not fit)
    const RwEnds<XT> e(row, a.r.vocab);
    const bool end = ends && tid < e.n;
    if (end) t.keep[atomicAdd(&t.n, 1)] = lp_key(lp_order(rw_float(row[e.place(tid)])), e.place(tid));
    const float least_x = bound ? lp_value(bound) : -INFINITY;
    if (fmaxf(v0, v1) >= least_x) {
        const float least_16 = __uint_as_float(__float_as_uint(least_x) & 0xffff0000u);   // (cut off as the slots' numbers are)
        const int batches = (p.n + RW_THREADS * RW_BATCH - 1) / (RW_THREADS * RW_BATCH);
        const int slots = (batches + (1 << a.shift) - 1) >> a.shift;
        unsigned long long hits = 0;               // a bit for each of the thread's numbers
#pragma unroll 4
        for (int g = 0; g < slots; ++g) {
            const uint2 m = t.big[g][tid];
            const float v[RW_BATCH] = {__uint_as_float(m.x << 16), __uint_as_float(m.x & 0xffff0000u), __uint_as_float(m.y << 16),
                                       __uint_as_float(m.y & 0xffff0000u)};
            uint32_t h = 0;
#pragma unroll
            for (int j = 0; j < RW_BATCH; ++j) h |= (v[j] >= least_16 ? 1u : 0u) << j;
            hits |= (unsigned long long)h << RW_BATCH * g;
        }
        int at = atomicAdd(&t.listed, __popcll(hits));
        for (; hits; hits &= hits - 1, ++at)
            if (at < LP_LIST) t.list[at] = (uint16_t)((__ffsll(hits) - 1) * RW_THREADS + tid);
    }
    __syncthreads();
    // the i-th unit to look through: of those listed, or (where they are too many) of all
    const bool all = t.listed > LP_LIST;
    const int total = all ? p.n : t.listed << a.shift;
    const auto unit_of = [&](int i) {
        if (all) return i;
        const int g = t.list[i >> a.shift], who = g % RW_THREADS, j = g / RW_THREADS % RW_BATCH, slot = g / RW_THREADS / RW_BATCH;
        return (((slot << a.shift) + (i & ((1 << a.shift) - 1))) * RW_BATCH + j) * RW_THREADS + who;
    };
    bool full = all;
    for (int i0 = tid; i0 < total && !full; i0 += LP_AHEAD * RW_THREADS) {
        RwUnit<XT> w[LP_AHEAD];
        int u[LP_AHEAD];
#pragma unroll
        for (int q = 0; q < LP_AHEAD; ++q) {
            u[q] = i0 + q * RW_THREADS < total ? unit_of(i0 + q * RW_THREADS) : p.n;
            if (u[q] < p.n) w[q].load(p.x + (long)N * u[q]);
        }
#pragma unroll
        for (int q = 0; q < LP_AHEAD; ++q) {
            if (u[q] >= p.n) continue;
            uint32_t reached = 0;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float x[2];
                unpack2(w[q].two(j / 2), x[0], x[1]);
                reached |= (x[j & 1] >= least_x ? 1u : 0u) << j;
            }
            if (!reached) continue;
            int at = atomicAdd(&t.n, __popc(reached));
            full |= at + __popc(reached) > LP_KEEP;
            if (full) continue;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float x[2];
                unpack2(w[q].two(j / 2), x[0], x[1]);
                if (reached >> j & 1) t.keep[at++] = lp_key(lp_order(x[j & 1]), p.first + N * u[q] + j);
            }
        }
    }
    if (__syncthreads_or(full)) {                  // too many: once more, thinned on the way
        unsigned long long least = max((unsigned long long)bound << 32, 1ull);     // (0: no logit)
        int turn = 0;
        if (tid == 0) t.n = 0;
        __syncthreads();
        if (end) t.keep[atomicAdd(&t.n, 1)] = lp_key(lp_order(rw_float(row[e.place(tid)])), e.place(tid));
        __syncthreads();
        for (int i0 = 0; i0 < total; i0 += RW_THREADS) {
            const int u = i0 + tid < total ? unit_of(i0 + tid) : p.n;
            RwUnit<XT> w;
            w.lowest();
            if (u < p.n) w.load(p.x + (long)N * u);
            if (!__syncthreads_or(u < p.n && lp_key(lp_order(fmaxf(w.max(0), w.max(1))), p.first + N * u) >= least)) continue;
#pragma unroll 1
            for (int j = 0; j < N; ++j) {
                unsigned long long key = 0;
                if (u < p.n) key = lp_key(lp_order(rw_float(p.x[(long)N * u + j])), p.first + N * u + j);
                const int n = t.n, more = lp_count(t, key >= least, turn);     // (n before the barrier: pushes come after it)
                if (n + more > LP_KEEP) least = lp_thin(t, k, turn);
                if (key >= least) t.keep[atomicAdd(&t.n, 1)] = key;
                __syncthreads();
            }
        }
    }
    if (t.n > LP_SORT) {
        int turn = 0;
        lp_thin(t, k, turn);
    }
}

// A warp's 32 keys in order, largest first, by compare and exchange.
__device__ __forceinline__ unsigned long long lp_sort32(unsigned long long v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size *= 2)
#pragma unroll
        for (int d = size / 2; d; d /= 2) {
            const unsigned long long o = __shfl_xor_sync(~0u, v, d);
            const bool larger = (lane & d) == 0 ? (lane & size) == 0 : (lane & size) != 0;
            if ((o > v) == larger) v = o;
        }
    return v;
}

// The t.n <= LP_SORT candidates in order, and no more than k of them: runs of
// 32 are sorted by a warp each, and a key's place is the sum of what the runs
// have before it.
__device__ __forceinline__ void lp_ordered(LpTop& t, int k) {
    constexpr int EACH = LP_SORT / RW_THREADS;
    const int tid = threadIdx.x, lane = tid & 31, n = t.n, runs = (n + 31) / 32;
    unsigned long long key[EACH];
    int at[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int j = i * RW_THREADS + tid;
        key[i] = 0;
        if (j - lane >= n) continue;
        key[i] = lp_sort32(j < n ? t.keep[j] : 0);
        t.keep[j] = key[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        at[i] = 0;
        if (i * RW_THREADS + tid - lane >= n) continue;
#pragma unroll 4
        for (int r = 0; r < runs; ++r) {
            const unsigned long long* run = t.keep + 32 * r;
            int b = 0;
#pragma unroll
            for (int d = 16; d; d /= 2)
                if (run[b + d - 1] > key[i]) b += d;
            at[i] += b + (run[b] > key[i] ? 1 : 0);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i)
        if (key[i] && at[i] < k) t.keep[at[i]] = key[i];
    if (tid == 0) t.n = min(n, k);
    __syncthreads();
}

// A cluster of blocks per row, each with one part of it.  Every logit is read
// once, for the sums and for the largest of each unit; the blocks' sums and
// candidates meet in shared memory.
template <class XT, bool ENT, bool TOP>
__global__ void __launch_bounds__(RW_THREADS, 4) lp_kernel(const LpArgs a) {
    extern __shared__ __align__(16) char lp_smem[];
    __shared__ RwStat join[RW_WARPS], parts[LP_CLUSTER];
    LpTop& t = *reinterpret_cast<LpTop*>(lp_smem);                                       // TOP
    pdl_wait();
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
    if (a.parts > 1) cluster_arrive();
    const XT* x = static_cast<const XT*>(a.r.x) + row * a.r.ldx;
    const float given = a.logp ? rw_float(x[token]) : 0.0f;
    const RwPart<XT> p(x, vocab, rank, a.parts);
    const bool ends = rank == a.parts - 1;
    RwSums<ENT> sums;
    if (ends) {
        const RwEnds<XT> e(x, vocab);
        if (tid < e.n) sums.single(rw_float(x[e.place(tid)]), c);
    }
    const f32x2 c2 = pack2(c, c);
    float v0 = -INFINITY, v1 = -INFINITY;
    int batch = 0;
    // (several batches may share a slot)
    const auto keep = [&](const float (&v)[RW_BATCH]) {
        uint2& slot = t.big[batch >> a.shift][tid];
        float m[RW_BATCH] = {v[0], v[1], v[2], v[3]};
        if (batch & ((1 << a.shift) - 1)) {
            const uint2 o = slot;
            m[0] = fmaxf(m[0], __uint_as_float(o.x << 16));
            m[1] = fmaxf(m[1], __uint_as_float(o.x & 0xffff0000u));
            m[2] = fmaxf(m[2], __uint_as_float(o.y << 16));
            m[3] = fmaxf(m[3], __uint_as_float(o.y & 0xffff0000u));
        }
        slot = make_uint2(__byte_perm(__float_as_uint(m[0]), __float_as_uint(m[1]), 0x7632),
                          __byte_perm(__float_as_uint(m[2]), __float_as_uint(m[3]), 0x7632));
    };
    for (int u0 = 0; u0 < p.n; u0 += RW_THREADS * RW_BATCH) {
        RwUnit<XT> u[RW_BATCH];
        rw_batch<XT>(u, p, u0);
        if (batch > 0 && batch % RW_FLUSH == 0) sums.flush(c);      // (while the loads are on their way)
        float v[RW_BATCH], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < RW_BATCH; ++j) {
            const float lo = u[j].max(0), hi = u[j].max(1);
            v[j] = fmaxf(lo, hi);
            if (TOP) {
                v0 = fmaxf(v0, lo);
                v1 = fmaxf(v1, hi);
            }
            top = fmaxf(top, v[j]);
        }
        if (TOP) keep(v);
        if (top > sums.m) sums.raise(top, c);
        sums.batch(u, c2);
        ++batch;
    }
    if (a.r.few) pdl_trigger();                    // (earlier, the next call's blocks would take cache from the loads)
    sums.flush(c);
    const RwStat w = rw_warp_join<ENT>(RwStat{sums.M, sums.S, sums.A}, c);
    if ((tid & 31) == 0) join[tid >> 5] = w;
    __syncthreads();
    const RwStat none{RW_LOWEST, 0.0, 0.0};
    const int lane = tid & 31;
    RwStat st = rw_warp_join<ENT>(lane < RW_WARPS ? join[lane] : none, c);   // (in every warp)
    if (TOP) {
        lp_search(t, a, x, p, ends, v0, v1);
        lp_ordered(t, k);
    }
    // every block gets all blocks' sums and lists
    unsigned long long* lists = reinterpret_cast<unsigned long long*>(lp_smem + sizeof(LpTop));
    if (a.parts > 1) {
        cluster_wait();                            // (all have begun)
        if (tid < a.parts) {
            *rw_peer(&parts[rank], tid) = st;
            if (TOP) *rw_peer(&t.peers[rank], tid) = t.n;
        }
        if (TOP && tid >> 5 < a.parts)
            for (int i = lane; i < t.n; i += 32) rw_peer(lists + rank * k, tid >> 5)[i] = t.keep[i];
        cluster_sync();
        st = rw_warp_join<ENT>(lane < a.parts ? parts[lane] : none, c);
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
            // a key's place in the row: the sum of what each block has before it
            const int n = t.n;
            const unsigned long long key = tid < n ? t.keep[tid] : 0;
            int at = tid;
            if (a.parts > 1 && tid < n) {
                int b[LP_CLUSTER], m[LP_CLUSTER];
#pragma unroll
                for (int r = 0; r < LP_CLUSTER; ++r) {
                    b[r] = 0;
                    m[r] = r < a.parts ? t.peers[r] : 0;
                }
                for (int d = 1 << (31 - __clz(k)); d; d /= 2)
#pragma unroll
                    for (int r = 0; r < LP_CLUSTER; ++r)
                        if ((lists[min(r, a.parts - 1) * k + min(b[r] + d, k) - 1] > key) & (b[r] + d <= m[r])) b[r] += d;
                at = 0;
#pragma unroll
                for (int r = 0; r < LP_CLUSTER; ++r) at += b[r];
            }
            if (tid < n && at < k) {
                ids[at] = (int)~(uint32_t)key;
                if (lp) lp[at] = (float)(((double)lp_value((uint32_t)(key >> 32)) - st.m) * a.r.inv_t - lns);
            }
        }
    }
}

struct LgArgs {
    RowArgs r;
    const int32_t* tokens;
    const float *rmax, *rsum, *entropy, *d_logp, *d_entropy;
    int parts;                // blocks of a row
};

// One pass: every logit is read once, every gradient written once.
template <class XT, class DT, bool ENT>
__global__ void __launch_bounds__(RW_THREADS, 4) lg_kernel(const LgArgs a) {
    __shared__ __align__(16) int ids[4];
    __shared__ float sub[4];
    if (a.r.few) pdl_trigger();
    pdl_wait();
    const size_t row = blockIdx.x / a.parts;
    const int vocab = a.r.vocab, rank = blockIdx.x % a.parts;
    const XT* x = static_cast<const XT*>(a.r.x) + row * a.r.ldx;
    DT* dx = static_cast<DT*>(a.r.dx) + row * a.r.ldd;
    const int token = a.tokens ? a.tokens[row] : 0;
    const float dl = a.d_logp ? a.d_logp[row] : 0.0f, de = ENT ? a.d_entropy[row] : 0.0f;
    const float m = a.rmax[row], s = a.rsum[row], h = ENT ? a.entropy[row] : 0.0f;
    if (token >= vocab && rank == 0 && threadIdx.x == 0) raise_status(a.r.status, DEV_INVALID);
    if (token < 0 || token >= vocab || (dl == 0.0f && de == 0.0f)) {
        rw_zero(dx, vocab, rank, a.parts);
        return;
    }
    if (s != s && rank == 0 && threadIdx.x == 0) raise_status(a.r.status, DEV_INVALID);
    // -p (dl + de (ln p + H)) / T with ln p = y ln 2 - ln S
    const float r = a.r.inv_t / s;
    const RwDense<ENT> dense{m, a.r.c, -(ENT ? fmaf(de, h - logf(s), dl) : dl) * r, -de * 0.69314718f * r};
    if (threadIdx.x < 4) {
        ids[threadIdx.x] = threadIdx.x == 0 && a.d_logp ? token : -1;
        sub[threadIdx.x] = -dl * a.r.inv_t;
    }
    __syncthreads();
    const RwPart<XT> p(x, vocab, rank, a.parts);
    rw_gradient<XT, DT, ENT>(x, dx, vocab, p, rank == a.parts - 1, ids, sub, 1, 1.0f, dense);
}

// Blocks of a row: for few rows as many as the GPU holds at once, of 8192
// logits each at least.  us by blocks a row 1, 2, 4, 8, without and with 20
// alternatives, whose search each block does: 1 row of 262144 fp32 19, 12, 8.4,
// 6.1 and 25, 18, 12.9, 10.4; 32 of them 20, 13, 9.2, 7.8 and 26, 19, 13.5, 12.1;
// 48 of 50257 7.2, 6.6, 6.1, 5.7 and 11.3, 10.9, 10.4, 10.9; 100 of 131072 bf16
// 10.4, 10.7, 9.4, 10.9 and 14.8, 15.6, 14.1, 20.9; 256 of 262144 bf16 32, 30,
// 32, 37 and 38, 37, 43, 57.
static int lp_parts(const tk_ctx* ctx, int n_rows, int vocab) {
    int parts = 1;
    while (parts < LP_CLUSTER && 2L * n_rows * parts <= 4L * ctx->num_sms && vocab / (2 * parts) >= 8192) parts *= 2;
    return parts;
}

template <class XT, bool ENT, bool TOP>
static cudaError_t launch_lp(const tk_ctx* ctx, LpArgs& a, cudaStream_t s) {
    a.parts = lp_parts(ctx, a.r.n_rows, a.r.vocab);
    a.r.few = rw_few(ctx, a.r.n_rows, a.parts);
    const int each = ((a.r.vocab / RwUnit<XT>::N + a.parts - 1) / a.parts + 31) & ~31;
    const int batches = (each + RW_THREADS * RW_BATCH - 1) / (RW_THREADS * RW_BATCH);
    while (batches > LP_SLOTS << a.shift) ++a.shift;
    int smem = TOP ? (int)sizeof(LpTop) : 0;
    if (TOP && a.parts > 1) smem += a.parts * a.top_k * (int)sizeof(unsigned long long);
    const auto kern = lp_kernel<XT, ENT, TOP>;
    static std::atomic<uint64_t> attr_smem{0};
    constexpr int MOST = (int)sizeof(LpTop) + LP_CLUSTER * TK_TOP_MAX * (int)sizeof(unsigned long long);
    const cudaError_t e = TOP ? smem_attr_once(kern, MOST, ctx->device, attr_smem) : cudaSuccess;
    if (e != cudaSuccess) return e;
    return rw_launch(kern, a.r.n_rows, a.parts, true, smem, a, s);
}
tk_status launch_logprobs(tk_ctx* ctx, const RowArgs& r, int x_dtype, const int32_t* tokens, float* logp, float* entropy,
                          float* rmax, float* rsum, int top_k, int32_t* top_ids, float* top_logp, cudaStream_t s) {
    LpArgs a{r, tokens, logp, entropy, rmax, rsum, top_k, top_ids, top_logp, 1, 0};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    const auto with = [&](auto x) {
        using XT = decltype(x);
        return entropy ? top_k ? launch_lp<XT, true, true>(ctx, a, s) : launch_lp<XT, true, false>(ctx, a, s)
                       : top_k ? launch_lp<XT, false, true>(ctx, a, s) : launch_lp<XT, false, false>(ctx, a, s);
    };
    return cuda_fail(x_dtype == TK_DT_F32 ? with(float()) : x_dtype == TK_DT_F16 ? with(__half()) : with(__nv_bfloat16()),
                     "log-probabilities launch");
}

template <class XT, class DT>
static cudaError_t launch_lg(const tk_ctx* ctx, LgArgs& a, cudaStream_t s) {
    a.parts = rw_grad_parts<XT>(ctx, a.r.n_rows, a.r.vocab);
    a.r.few = rw_few(ctx, a.r.n_rows, a.parts);
    return rw_launch(a.d_entropy ? lg_kernel<XT, DT, true> : lg_kernel<XT, DT, false>, a.r.n_rows, a.parts, false, 0, a, s);
}
tk_status launch_logprobs_grad(tk_ctx* ctx, const RowArgs& r, int x_dtype, const int32_t* tokens, const float* rmax,
                               const float* rsum, const float* entropy, const float* d_logp, const float* d_entropy,
                               int d_dtype, cudaStream_t s) {
    LgArgs a{r, tokens, rmax, rsum, entropy, d_logp, d_entropy, 1};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    return cuda_fail(rw_types(x_dtype, d_dtype, [&](auto x, auto d) { return launch_lg<decltype(x), decltype(d)>(ctx, a, s); }),
                     "log-probability gradient launch");
}

}  // namespace tk
