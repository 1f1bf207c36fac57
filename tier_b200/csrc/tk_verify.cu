// tk_verify.cu -- tk_draft_verify: drafted tokens against the target's logits.
//
// A row's weights are powers of two: with c = log2(e) / temperature (fp32),
// y = x * c, i = floor(y), weight 2^(y - i) * 2^(i - I), I the row's largest
// i.  Only whole exponents are subtracted, so a weight's bits do not depend on
// which part of the row saw the largest logit: parts of a row are summed each
// to its own largest exponent, brought together by exact powers of two, and
// the row's sum S is rounded once to fp32 from a sum of 2^-46.  Another division
// into parts (a batch of another size) can turn that one rounding where the sum
// lies within 2^-46 of the middle between two fp32 numbers; else S, and the
// probabilities weight / S with it, come out the same.
//
// Two launches.  dv_rows reads every logit once (the bound: memory) and leaves
// each part's exponent, sum and largest logit.  dv_pick, a cluster of blocks
// per sequence, finds the first refused row from these and draws the next
// token from that one row: whole weights (multiples of 2^-38) summed per 128
// tokens, the blocks' totals exchanged in shared memory, then the one piece
// that holds the draw searched again.
//
// Measured: 24 sequences of up to 8 rows, vocabulary 262144, with draft logits
// (191 MB) 73.3 us, 2.6 TB/s: dv_rows about 40 (4.8 TB/s; an exponential a
// logit and half a dozen packed instructions keep it from the memory's rate),
// the draw the rest (it reads its two rows again in 192 blocks, and its chain
// of sums, exchange and search is latency).  One sequence of 5 rows 18.4 us, 64
// greedy ones of up to 5 rows of 50257 (40.8 MB) 18.4: two dependent launches.
#include <climits>
#include "tk_device.cuh"
#include "tk_f32x2.cuh"
#include "tk_internal.h"

namespace tk {

constexpr int DV_THREADS = 256, DV_QUADS = 8;          // dv_rows: quads (4 logits) a thread holds in registers at most
constexpr int DP_THREADS = 512, DP_CLUSTER = 16, DP_WARPS = DP_THREADS / 32;   // dv_pick: blocks of a cluster at most
constexpr int DP_SUMS = 64, DP_AHEAD = 6;          // sums kept per warp; steps whose logits are on their way

// A part of a row, or a whole one: largest whole exponent, the weights' sum
// relative to it, the largest logit and its first place; bad: NaN, +inf or
// nothing above -inf.
struct DvStat {
    double sum;
    float top, max;
    int arg, bad;
};

struct DvArgs {
    int n_seqs, n_rows, vocab;
    const int32_t* row_start;
    const float *target, *draft;
    long ldt, ldd;
    const int32_t* tokens;
    const float *u_accept, *u_sample;
    float c;                  // log2(e) / temperature; temperature 0: log2(e)
    bool greedy;
    int32_t *n_accept, *next;
    float* logp;
    DvStat* stat;             // [2][n_rows][parts]: target's rows, then draft's
    int parts, part_quads;    // parts of a row, quads of a part
    int cluster;              // blocks of a sequence in dv_pick
    int* status;
};

__device__ __forceinline__ float dv_exp2(float x) {        // x in [0, 1)
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float dv_max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// 2^d for a whole d in [-126, 0]: d + 1.5 * 2^23 has d in its low bits.
__device__ __forceinline__ float dv_scale(float w, float d) {
    const int k = __float_as_int(d + 12582912.0f);
    return __int_as_float(__float_as_int(w) + (int)((uint32_t)k << 23));
}
__device__ __forceinline__ float dv_weight(float x, float c, float top) {
    const float y = __fmul_rn(x, c), i = floorf(y), d = i - top;
    return d >= -100.0f ? dv_scale(dv_exp2(y - i), d) : 0.0f;      // also y = -inf
}
// Two weights at once, for |top| < 2^22 and y no further than 110 below it
// (clamped: what is further down weighs less than 2^-109 of the row).  Adding
// 1.5 * 2^23 - top downwards leaves i - top in the low bits of the sum, which
// shifted up are added to the exponent of 2^(y - i): the bits of dv_weight
// without its conversions and comparisons.  Packed fp32 instructions take
// both at once.
constexpr float DV_NEAR = 4194304.0f;              // |top| below this: dv_weight2
struct DvFast {
    f32x2 c, bias, nbias;
    float low;
};
__device__ __forceinline__ DvFast dv_fast(float c, float top) {
    const float m = 12582912.0f - top;
    return DvFast{pack2(c, c), pack2(m, m), pack2(-m, -m), top - 110.0f};
}
__device__ __forceinline__ f32x2 dv_weight2(float x0, float x1, const DvFast& k) {
    f32x2 y, t;
    float y0, y1, f0, f1, t0, t1;
    unpack2(mul2(pack2(x0, x1), k.c), y0, y1);
    y = pack2(fmaxf(y0, k.low), fmaxf(y1, k.low));
    t = add2_rm(y, k.bias);
    unpack2(sub2(y, add2(t, k.nbias)), f0, f1);
    unpack2(t, t0, t1);
    return pack2(__uint_as_float((__float_as_uint(t0) << 23) + __float_as_uint(dv_exp2(f0))),
                   __uint_as_float((__float_as_uint(t1) << 23) + __float_as_uint(dv_exp2(f1))));
}

// weight / S rounded once.  With r = 1 / S rounded to nearest, q = w r and the
// exact remainder w - q S give the correctly rounded quotient q + (w - q S) r
// for every S whose significand is not all ones (Markstein 1990); for that
// one, and for what is needed only once, the division itself.
struct DvProb {
    DvFast fast;
    f32x2 ns, r;              // -S, 1 / S
    bool quick;               // both of the above hold
};
__device__ __forceinline__ DvProb dv_prepare(const DvStat& st, float c) {
    const float s = (float)st.sum, r = __frcp_rn(s);
    return DvProb{dv_fast(c, st.top), pack2(-s, -s), pack2(r, r),
                  fabsf(st.top) < DV_NEAR && (__float_as_uint(s) & 0x7fffffu) != 0x7fffffu};
}
__device__ __forceinline__ f32x2 dv_prob2(float x0, float x1, const DvProb& k) {
    const f32x2 w = dv_weight2(x0, x1, k.fast), q = mul2(w, k.r);
    return fma2(fma2(q, k.ns, w), k.r, q);
}
__device__ __forceinline__ float dv_prob(float x, float c, const DvStat& s) {
    return __fdiv_rn(dv_weight(x, c, s.top), (float)s.sum);
}
__device__ __forceinline__ float dv_logp(float x, float c, const DvStat& s) {
    return ((__fmul_rn(x, c) - s.top) - log2f((float)s.sum)) * 0.693147180559945309f;
}
// Exact 2^d (whole d <= 0) for the sums.
__device__ __forceinline__ double dv_pow2(float d) {
    return d < -1000.0f ? 0.0 : __longlong_as_double((long long)(1023 + (int)d) << 52);
}
__device__ __forceinline__ DvStat dv_shfl(const DvStat& s, int i) {
    DvStat o;
    o.sum = __shfl_xor_sync(~0u, s.sum, i);
    o.top = __shfl_xor_sync(~0u, s.top, i);
    o.max = __shfl_xor_sync(~0u, s.max, i);
    o.arg = __shfl_xor_sync(~0u, s.arg, i);
    o.bad = __shfl_xor_sync(~0u, s.bad, i);
    return o;
}
// Symmetric in its arguments.
__device__ __forceinline__ DvStat dv_merge(const DvStat& a, const DvStat& b) {
    DvStat r;
    r.top = fmaxf(a.top, b.top);
    r.sum = (a.top == -INFINITY ? 0.0 : a.sum * dv_pow2(a.top - r.top)) +
            (b.top == -INFINITY ? 0.0 : b.sum * dv_pow2(b.top - r.top));
    r.max = fmaxf(a.max, b.max);
    r.arg = a.max > b.max ? a.arg : b.max > a.max ? b.arg : min(a.arg, b.arg);
    r.bad = a.bad | b.bad;
    return r;
}

// Logits 4 q - off .. + 3 of a row whose first lies `off` floats behind a
// 16-byte boundary: one load inside the row, single ones at its ends;
// -inf outside.
__device__ __forceinline__ float4 dv_quad(const float* x, int off, long q, int vocab) {
    const long j = 4 * q - off;
    if (j >= 0 && j + 4 <= vocab) return __ldg(reinterpret_cast<const float4*>(x + j));
    float4 v;
    v.x = j >= 0 && j < vocab ? x[j] : -INFINITY;
    v.y = j + 1 >= 0 && j + 1 < vocab ? x[j + 1] : -INFINITY;
    v.z = j + 2 >= 0 && j + 2 < vocab ? x[j + 2] : -INFINITY;
    v.w = j + 3 >= 0 && j + 3 < vocab ? x[j + 3] : -INFINITY;
    return v;
}
__device__ __forceinline__ int dv_off(const float* x) { return (int)((reinterpret_cast<uintptr_t>(x) >> 2) & 3); }

// A block takes one part of one row into registers (QUADS loads of 16 bytes a
// thread in flight), finds its largest logit, then sums the weights: each
// thread in fp32 with the rounding errors kept beside (exact to 2^-46), the
// block in 64 bits.
template <bool GREEDY, int QUADS>
__global__ void __launch_bounds__(DV_THREADS, 4) dv_rows_kernel(const DvArgs a) {
    __shared__ float smax[DV_THREADS / 32];
    __shared__ double ssum[DV_THREADS / 32];
    __shared__ int sarg[DV_THREADS / 32];
    pdl_trigger();
    const int part = blockIdx.x % a.parts, row = blockIdx.x / a.parts, tid = threadIdx.x;
    const bool isd = row >= a.n_rows;
    if (isd) {                                     // a sequence's last row judges no draft
        bool last = false;
        for (int i = 1 + tid; i <= a.n_seqs; i += DV_THREADS) last |= a.row_start[i] == row - a.n_rows + 1;
        if (__syncthreads_or(last)) {              // (13 % of the draft's rows here: 72.7 -> 70.5 us)
            if (tid == 0) a.stat[(size_t)row * a.parts + part] = DvStat{0.0, -INFINITY, -INFINITY, INT_MAX, 1};
            return;
        }
    }
    const float* x = isd ? a.draft + (size_t)(row - a.n_rows) * a.ldd : a.target + (size_t)row * a.ldt;
    const int off = dv_off(x);
    const long quads = ((long)off + a.vocab + 3) / 4, q0 = (long)part * a.part_quads;
    const int n = (int)max(0L, min((long)a.part_quads, quads - q0));
    float4 v[QUADS];
#pragma unroll
    for (int k = 0; k < QUADS; ++k) v[k] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    if (4 * q0 >= off && 4 * (q0 + n) - off <= a.vocab) {          // no quad reaches over the row's ends
        const float4* from = reinterpret_cast<const float4*>(x + (4 * q0 - off)) + tid;
#pragma unroll
        for (int k = 0; k < QUADS; ++k)
            if (k * DV_THREADS + tid < n) v[k] = __ldg(from + k * DV_THREADS);
    } else {
#pragma unroll
        for (int k = 0; k < QUADS; ++k)
            if (k * DV_THREADS + tid < n) v[k] = dv_quad(x, off, q0 + k * DV_THREADS + tid, a.vocab);
    }
    float mx = -INFINITY, nan = -INFINITY;
    int arg = INT_MAX;
#pragma unroll
    for (int k = 0; k < QUADS; ++k) {
        const float e[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            nan = dv_max_nan(nan, e[i]);
            if (GREEDY && e[i] > mx) { mx = e[i]; arg = 4 * (k * DV_THREADS) + i; }
        }
    }
    const bool bad = !(nan <= 3.402823466e38f);
    float big = bad ? 0.0f : nan;
    for (int i = 16; i; i >>= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, i));
    if ((tid & 31) == 0) smax[tid >> 5] = big;
    const int any_bad = __syncthreads_or(bad);
#pragma unroll
    for (int w = 0; w < DV_THREADS / 32; ++w) big = fmaxf(big, smax[w]);
    const float top = floorf(__fmul_rn(big, a.c));
    double sum = 0.0;
    if (fabsf(top) < DV_NEAR) {
        // sums start above any weight, so that t - s2 and its difference to the weight are exact
        const DvFast fast = dv_fast(a.c, top);
        f32x2 s2 = pack2(2.0f, 2.0f), err = pack2(0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < QUADS; ++k) {
            if (k * DV_THREADS >= n) break;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x2 w = h ? dv_weight2(v[k].z, v[k].w, fast) : dv_weight2(v[k].x, v[k].y, fast), t = add2(s2, w);
                err = add2(err, sub2(w, sub2(t, s2)));
                s2 = t;
            }
        }
        float p0, p1, e0, e1;
        unpack2(s2, p0, p1);
        unpack2(err, e0, e1);
        sum = (((double)p0 - 2.0) + ((double)p1 - 2.0)) + ((double)e0 + (double)e1);
    } else if (top > -3.402823466e38f) {           // logits of such size: one by one
#pragma unroll 1
        for (int q = tid; q < n; q += DV_THREADS) {
            const float4 u = dv_quad(x, off, q0 + q, a.vocab);
            sum += ((double)dv_weight(u.x, a.c, top) + (double)dv_weight(u.y, a.c, top)) +
                   ((double)dv_weight(u.z, a.c, top) + (double)dv_weight(u.w, a.c, top));
        }
    }
    if (GREEDY) {                                  // the first place of the block's largest
        arg = arg != INT_MAX && mx == big ? arg + (int)(4 * (q0 + tid) - off) : INT_MAX;
        arg = __reduce_min_sync(~0u, arg);
    }
    for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
    if ((tid & 31) == 0) {
        ssum[tid >> 5] = sum;
        sarg[tid >> 5] = arg;
    }
    __syncthreads();
    if (tid == 0) {
        DvStat s{0.0, top, big, INT_MAX, any_bad};
#pragma unroll
        for (int w = 0; w < DV_THREADS / 32; ++w) {
            s.sum += ssum[w];
            s.arg = min(s.arg, sarg[w]);
        }
        a.stat[(size_t)row * a.parts + part] = s;
    }
}

__device__ __forceinline__ unsigned long long ld_cluster_u64(uint32_t addr) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// One row's parts joined by a warp (all lanes return it).
__device__ __forceinline__ DvStat dv_row(const DvArgs& a, size_t row) {
    DvStat s{0.0, -INFINITY, -INFINITY, INT_MAX, 0};
    for (int p = threadIdx.x & 31; p < a.parts; p += 32) s = dv_merge(s, a.stat[row * a.parts + p]);
    for (int i = 16; i; i >>= 1) s = dv_merge(s, dv_shfl(s, i));
    if (!(fabsf(s.top) <= 3.402823466e38f)) s.bad = 1;
    return s;
}

__global__ void __launch_bounds__(DP_THREADS, 2) dv_pick_kernel(const DvArgs a) {
    __shared__ DvStat st_t[DP_WARPS], st_d[DP_WARPS];
    __shared__ int verdict[DP_WARPS];              // 0: accepted, 1: the row draws, 2: no distribution
    __shared__ unsigned long long wsum[DP_WARPS][DP_SUMS], wtot[DP_WARPS], ctot[2];
    extern __shared__ float4 ring[];               // [DP_AHEAD][target, draft][DP_THREADS]: each thread's own
    const int cluster = a.cluster, b = blockIdx.x / cluster, rank = (int)cluster_ctarank(), tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int V = a.vocab;
    pdl_wait();
    const int r0 = a.row_start[b], r1 = a.row_start[b + 1];
    if (r0 < 0 || r1 <= r0 || r1 > a.n_rows) {     // the whole cluster
        if (rank == 0 && tid == 0) {
            raise_status(a.status, DEV_INVALID);
            a.n_accept[b] = 0;
            a.next[b] = -1;
        }
        return;
    }
    // ---- the first row that does not accept its drafted token: a warp a row ----
    int r = r0, what = 1, slot = 0;
    for (;; r += DP_WARPS) {
        const int mine = r + warp;
        if (mine < r1) {
            const bool last = mine == r1 - 1;
            const int x = last ? -1 : a.tokens[mine + 1];
            const bool known = x >= 0 && x < V;
            float lt = 0.0f, ld = 0.0f, u = 0.0f;
            if (known && !a.greedy) {
                lt = a.target[(size_t)mine * a.ldt + x];
                if (a.draft) ld = a.draft[(size_t)mine * a.ldd + x];
                u = a.u_accept[mine];
            }
            const DvStat t = dv_row(a, mine), d = a.draft && !last ? dv_row(a, (size_t)a.n_rows + mine) : t;
            int v = 1;
            if (t.bad || d.bad) v = 2;
            else if (known && a.greedy) v = x != t.arg;
            else if (known) v = !(__fmul_rn(u, a.draft ? dv_prob(ld, a.c, d) : 1.0f) < dv_prob(lt, a.c, t));
            if (lane == 0) {
                st_t[warp] = t;
                st_d[warp] = d;
                verdict[warp] = v;
            }
        }
        __syncthreads();
        const int n = min(DP_WARPS, r1 - r);
        for (slot = 0; slot < n && verdict[slot] == 0; ++slot) {}
        if (rank == 0 && a.logp && tid < slot)     // accepted here
            a.logp[r + tid] = dv_logp(a.target[(size_t)(r + tid) * a.ldt + a.tokens[r + tid + 1]], a.c, st_t[tid]);
        if (slot < n) {                            // (the last row always ends the search)
            what = verdict[slot];
            r += slot;
            break;
        }
        __syncthreads();
    }
    const DvStat st = st_t[slot], sd = st_d[slot];
    const bool last = r == r1 - 1;
    const float* t = a.target + (size_t)r * a.ldt;
    if (rank == 0) {
        if (tid == 0) {
            a.n_accept[b] = r - r0;
            if (what == 2) {
                raise_status(a.status, DEV_INVALID);
                a.next[b] = -1;
                if (a.logp) a.logp[r] = 0.0f;
            } else if (a.greedy) {
                a.next[b] = st.arg;
                if (a.logp) a.logp[r] = dv_logp(st.max, a.c, st);
            }
        }
        if (a.logp)
            for (int i = r + 1 + tid; i < r1; i += DP_THREADS) a.logp[i] = 0.0f;
    }
    if (what == 2 || a.greedy) return;             // the whole cluster
    // ---- draw from row r: a warp takes `mine` runs of 128 tokens one after the other, and keeps a sum of every
    // `each` of them ----
    const float* d = a.draft && !last ? a.draft + (size_t)r * a.ldd : nullptr;
    const int x = last ? -1 : a.tokens[r + 1];
    // both rows are read in quads of the target's alignment (a draft row of another alignment value by value)
    const int off = dv_off(t);
    const bool same = !d || dv_off(d) == off;
    const long quads = ((long)off + V + 3) / 4;
    const int mine = (int)(((quads + 31) / 32 + cluster * DP_WARPS - 1) / (cluster * DP_WARPS));
    const int each = max(4, (mine + DP_SUMS - 1) / DP_SUMS), sums = (mine + each - 1) / each;
    const long q0 = (long)(rank * DP_WARPS + warp) * mine * 32 + lane;
    const DvProb pt = dv_prepare(st, a.c), pd = dv_prepare(sd, a.c);
    const bool quick = pt.quick && pd.quick;
    // quad q of a row into a place of the ring: in the background where it lies inside the row
    auto fetch = [&](const float* x, bool aligned, long q, float4* to) {
        const long j = 4 * q - off;
        if (aligned && j >= 0 && j + 4 <= V) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(x + j) : "memory");
        } else {
            float e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = j + i >= 0 && j + i < V ? x[j + i] : -INFINITY;
            *to = make_float4(e[0], e[1], e[2], e[3]);
        }
    };
    // floor(p 2^38) = hi 2^19 + lo: adding 2^23 downwards leaves a whole number in the low bits (above DP_BIAS)
    constexpr uint32_t DP_BIAS = 0x4b000000u;
    const f32x2 k19 = pack2(524288.0f, 524288.0f), k23 = pack2(8388608.0f, 8388608.0f), n23 = pack2(-8388608.0f, -8388608.0f);
    auto weights = [&](long q, bool rest, const float4& tv, const float4& dv, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
        const float e[4] = {tv.x, tv.y, tv.z, tv.w}, o[4] = {dv.x, dv.y, dv.z, dv.w};
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float p0, p1;
            if (quick) {
                f32x2 p = dv_prob2(e[i], e[i + 1], pt);
                if (rest && d) p = sub2(p, dv_prob2(o[i], o[i + 1], pd));
                unpack2(p, p0, p1);
            } else {
                p0 = dv_prob(e[i], a.c, st);
                p1 = dv_prob(e[i + 1], a.c, st);
                if (rest && d) {
                    p0 -= dv_prob(o[i], a.c, sd);
                    p1 -= dv_prob(o[i + 1], a.c, sd);
                }
            }
            if (rest && !d) {
                if (4 * q - off + i == x) p0 = 0.0f;
                if (4 * q - off + i + 1 == x) p1 = 0.0f;
            }
            const f32x2 u = mul2(pack2(fmaxf(p0, 0.0f), fmaxf(p1, 0.0f)), k19);
            const f32x2 h = add2_rm(u, k23), l = fma2_rm(sub2(u, add2(h, n23)), k19, k23);
            float v0, v1;
            unpack2(h, v0, v1);
            hi[i] = __float_as_uint(v0) - DP_BIAS;
            hi[i + 1] = __float_as_uint(v1) - DP_BIAS;
            unpack2(l, v0, v1);
            lo[i] = __float_as_uint(v0) - DP_BIAS;
            lo[i + 1] = __float_as_uint(v1) - DP_BIAS;
        }
    };
    for (int pass = 0; pass < 2; ++pass) {         // what is left of p over q; p itself if that is nothing
        const bool rest = pass == 0 && !last;
        auto issue = [&](int i, int slot) {
            const long q = q0 + 32L * i;
            if (i < mine && q < quads) {
                float4* at = ring + slot * 2 * DP_THREADS + tid;
                fetch(t, true, q, at);
                if (d && rest) fetch(d, same, q, at + DP_THREADS);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        for (int i = 0; i < DP_AHEAD - 1; ++i) issue(i, i);
        uint32_t h = 0, l = 0;
        int k = 0, e = 0;
        unsigned long long own = 0;
#pragma unroll 1
        for (int i = 0; i < mine; ++i) {
            issue(i + DP_AHEAD - 1, (i + DP_AHEAD - 1) % DP_AHEAD);
            asm volatile("cp.async.wait_group %0;" ::"n"(DP_AHEAD - 1) : "memory");
            const long q = q0 + 32L * i;
            if (q < quads) {
                const float4* from = ring + i % DP_AHEAD * 2 * DP_THREADS + tid;
                uint32_t hi[4], lo[4];
                weights(q, rest, from[0], from[DP_THREADS], hi, lo);
                h += hi[0] + hi[1] + hi[2] + hi[3];
                l += lo[0] + lo[1] + lo[2] + lo[3];
            }
            if (++k == each || i == mine - 1) {
                // (a lane's low halves stay below 2^28; 32 lanes' would pass 2^32 in the largest vocabularies)
                h += l >> 19;
                l &= 0x7ffffu;
                const unsigned long long s = ((unsigned long long)__reduce_add_sync(~0u, h) << 19) + __reduce_add_sync(~0u, l);
                if (lane == 0) wsum[warp][e] = s;
                own += s;
                h = l = k = 0;
                ++e;
            }
        }
        if (lane == 0) wtot[warp] = own;
        __syncthreads();
        if (tid == 0) {
            own = 0;
            for (int w = 0; w < DP_WARPS; ++w) own += wtot[w];
            ctot[pass] = own;
        }
        cluster_sync();
        unsigned long long total = lane < cluster ? ld_cluster_u64(mapa_shared(smem_u32(&ctot[pass]), lane)) : 0, before = 0;
        for (int i = 1; i < 32; i <<= 1) {
            const unsigned long long o = __shfl_up_sync(~0u, total, i);
            if (lane >= i) total += o;
        }
        if (rank > 0) before = __shfl_sync(~0u, total, rank - 1);
        total = __shfl_sync(~0u, total, 31);
        if (total == 0 && pass == 0) continue;     // the whole cluster alike
        // [0, 1) in steps of 2^-24
        const unsigned long long u = (unsigned long long)(fminf(fmaxf(a.u_sample[b], 0.0f), 0.99999994f) * 16777216.0f);
        const unsigned long long goal = (total * u) >> 24;
        cluster_arrive();                          // (the totals have been read)
        // the warp that holds it, the sum, the run, the token
        if (goal >= before && goal < before + ctot[pass]) {
            unsigned long long upto = before;
            for (int w = 0; w < warp; ++w) upto += wtot[w];
            if (goal < upto || goal >= upto + wtot[warp]) break;   // another warp's
            unsigned long long left = goal - upto;
            int e = 0;
            while (e < sums - 1 && left >= wsum[warp][e]) left -= wsum[warp][e++];
            for (int i = e * each; i < min(mine, (e + 1) * each); ++i) {
                const long q = q0 + 32L * i;
                unsigned long long w[4] = {0, 0, 0, 0}, s, sum;
                if (q < quads) {
                    uint32_t hi[4], lo[4];
                    fetch(t, false, q, ring + tid);
                    if (d && rest) fetch(d, false, q, ring + DP_THREADS + tid);
                    weights(q, rest, ring[tid], ring[DP_THREADS + tid], hi, lo);
#pragma unroll
                    for (int k2 = 0; k2 < 4; ++k2) w[k2] = ((unsigned long long)hi[k2] << 19) + lo[k2];
                }
                s = sum = w[0] + w[1] + w[2] + w[3];
                for (int i = 1; i < 32; i <<= 1) {
                    const unsigned long long o = __shfl_up_sync(~0u, sum, i);
                    if (lane >= i) sum += o;
                }
                const unsigned hit = __ballot_sync(~0u, left < sum);
                if (!hit) {
                    left -= __shfl_sync(~0u, sum, 31);
                    continue;
                }
                if (lane == __ffs(hit) - 1) {
                    left -= sum - s;
                    int k2 = 0;
                    while (k2 < 3 && left >= w[k2]) left -= w[k2++];
                    const int tok = (int)(4 * q - off) + k2;
                    a.next[b] = tok;
                    if (a.logp) a.logp[r] = dv_logp(t[tok], a.c, st);
                }
                break;
            }
        }
        break;
    }
    cluster_wait();                                // no block ends while another reads its total
}

constexpr int DP_SMEM = DP_AHEAD * 2 * DP_THREADS * (int)sizeof(float4);

// Blocks of a sequence's draw: 16 at most, and 4/3 an SM over all sequences.
// Two an SM would hide more latency, but clusters stay within a GPC, and a size
// whose last cluster finds no place takes two waves.  Measured (4 rows of 262144
// a sequence with draft logits, whole call, us; first the rule's size):
//    8 sequences: 16 blocks 37, 12 41, 8 46     24: 8 72, 7 74, 10 82, 6 79
//   16: 12 65, 10 55, 16 59, 8 60               32: 6 89, 7 86, 8 93, 5 94
//   48: 4 123, 5 117, 3 136, 6 130
// The rule is within 6 % of the best but at 16 sequences (17 %): which sizes fill
// the GPCs depends on the GPU's floor plan, which it does not ask.
static int pick_cluster(const tk_ctx* ctx, int n_seqs, bool greedy) {
    if (greedy) return 1;                          // a greedy row draws nothing
    const int c = ctx->num_sms * 4 / 3 / n_seqs;
    return c < 1 ? 1 : c > DP_CLUSTER ? DP_CLUSTER : c;
}

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
    // parts of at most what a block's registers hold; smaller ones (down to four
    // quads a thread) while that gives every SM four blocks
    const long quads = ((long)vocab + 6) / 4, rows = (long)n_rows * (a.draft ? 2 : 1);
    long part = (quads * rows + 4L * ctx->num_sms - 1) / (4L * ctx->num_sms);
    if (part < 4 * DV_THREADS) part = 4 * DV_THREADS;
    if (part > DV_QUADS * DV_THREADS) part = DV_QUADS * DV_THREADS;
    a.cluster = pick_cluster(ctx, n_seqs, a.greedy);
    static std::atomic<uint64_t> attr_smem{0}, attr_size{0};
    cudaError_t e = smem_attr_once(dv_pick_kernel, DP_SMEM, ctx->device, attr_smem);
    const uint64_t bit = 1ull << (ctx->device & 63);
    if (e == cudaSuccess && !(attr_size.load(std::memory_order_relaxed) & bit)) {   // more than 8 blocks: on request
        e = cudaFuncSetAttribute(dv_pick_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) attr_size.fetch_or(bit);
    }
    if (e != cudaSuccess) return cuda_fail(e, "draft verify attributes");
    const long parts = (quads + part - 1) / part, grid = parts * rows, pick = (long)n_seqs * a.cluster;
    if (grid > INT_MAX || pick > INT_MAX) return fail(TK_ERR_INVALID, "tk_draft_verify: too many rows");
    a.parts = (int)parts;
    a.part_quads = (int)((quads + parts - 1) / parts);
    tk_status st = ws_ensure(ctx, (size_t)grid * sizeof(DvStat), s);
    if (st != TK_OK) return st;
    a.stat = static_cast<DvStat*>(ctx->ws);
    ProfScope ps(ctx, s, PK_SERVE);
    const bool small = a.part_quads <= 4 * DV_THREADS;
    auto kern = a.greedy ? (small ? dv_rows_kernel<true, 4> : dv_rows_kernel<true, DV_QUADS>)
                         : (small ? dv_rows_kernel<false, 4> : dv_rows_kernel<false, DV_QUADS>);
    // (no dependent of what runs before it: blocks that wait would take the draw's clusters their places, 84 against 72 us)
    kern<<<(unsigned)grid, DV_THREADS, 0, s>>>(a);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)pick);
    cfg.blockDim = dim3(DP_THREADS);
    cfg.dynamicSmemBytes = DP_SMEM;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, dv_pick_kernel, a);
    ctx->launches += 2;
    if (e != cudaSuccess) return cuda_fail(e, "draft verify launch");
    return cuda_fail(cudaGetLastError(), "draft verify launch");
}

}  // namespace tk
