// tk_verify.cu -- tk_draft_verify: drafted tokens against the target's logits.
//
// A row's weights are powers of two: with c = log2(e) / temperature (fp32),
// y = x * c, i = floor(y), weight 2^(y - i) * 2^(i - I), I the row's largest
// i.  Only whole exponents are subtracted, so a weight's bits do not depend on
// which part of the row saw the largest logit: parts of a row are summed each
// to its own largest exponent, brought together by exact powers of two, and
// the row's sum S (64 bits, rounded once to fp32) and its probabilities
// weight / S come out the same for any division.
//
// Two launches.  dv_rows reads every logit once (the bound: memory) and leaves
// each part's exponent, sum and largest logit.  dv_pick, a cluster of blocks
// per sequence, finds the first refused row from these and draws the next
// token from that one row: whole weights (multiples of 2^-38) summed per 128
// tokens, the blocks' totals exchanged in shared memory, then the one piece
// that holds the draw searched again.
#include <climits>
#include "tk_device.cuh"
#include "tk_internal.h"

namespace tk {

constexpr int DV_THREADS = 256, DV_QUADS = 16;     // dv_rows: quads (4 logits) a thread holds in registers at most
constexpr int DP_THREADS = 256, DP_CLUSTER = 16, DP_WARPS = DP_THREADS / 32;   // dv_pick: blocks of a cluster at most
constexpr int DP_GROUPS = 128, DP_AHEAD = 8;       // sums kept per warp; of these, groups whose logits are loaded at once

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
// weight / S rounded once.  With r = 1 / S rounded to nearest, q = w r and the
// exact remainder w - q S give the correctly rounded quotient q + (w - q S) r
// for every S whose significand is not all ones (Markstein 1990); for that
// one, and for what is drawn only once, the division itself.
struct DvInv {
    float s, r;
    bool divide;
};
__device__ __forceinline__ DvInv dv_inv(const DvStat& st) {
    const float s = (float)st.sum;
    return DvInv{s, __frcp_rn(s), (__float_as_uint(s) & 0x7fffffu) == 0x7fffffu};
}
__device__ __forceinline__ float dv_quotient(float w, const DvInv& i) {
    if (i.divide) return __fdiv_rn(w, i.s);
    const float q = __fmul_rn(w, i.r);
    return __fmaf_rn(__fmaf_rn(-q, i.s, w), i.r, q);
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
__global__ void __launch_bounds__(DV_THREADS, QUADS > 8 ? 2 : 4) dv_rows_kernel(const DvArgs a) {
    __shared__ float smax[DV_THREADS / 32];
    __shared__ DvStat sst[DV_THREADS / 32];
    pdl_trigger();
    const int part = blockIdx.x % a.parts, row = blockIdx.x / a.parts, tid = threadIdx.x;
    const bool isd = row >= a.n_rows;
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
    if (GREEDY && arg != INT_MAX) arg += (int)(4 * (q0 + tid) - off);
    const bool bad = !(nan <= 3.402823466e38f);
    if (!GREEDY) mx = bad ? 0.0f : nan;
    float big = mx;
    for (int i = 16; i; i >>= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, i));
    if ((tid & 31) == 0) smax[tid >> 5] = big;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < DV_THREADS / 32; ++w) big = fmaxf(big, smax[w]);
    DvStat s{0.0, floorf(__fmul_rn(big, a.c)), mx, arg, bad};
    if (s.top > -3.402823466e38f) {
        // s2 >= any weight from the start, so that t - s2 and its difference to the weight are exact
        float s2 = 2.0f, err = 0.0f;
#pragma unroll
        for (int k = 0; k < QUADS; ++k) {
            if (k * DV_THREADS >= n) break;
            const float e[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float w = dv_weight(e[i], a.c, s.top), t = __fadd_rn(s2, w);
                err = __fadd_rn(err, __fsub_rn(w, __fsub_rn(t, s2)));
                s2 = t;
            }
        }
        s.sum = ((double)s2 - 2.0) + (double)err;
    }
    for (int i = 16; i; i >>= 1) {
        const DvStat o = dv_shfl(s, i);
        s.sum += o.sum;
        s.arg = s.max > o.max ? s.arg : o.max > s.max ? o.arg : min(s.arg, o.arg);
        s.max = fmaxf(s.max, o.max);
        s.bad |= o.bad;
    }
    if ((tid & 31) == 0) sst[tid >> 5] = s;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < DV_THREADS / 32; ++w) {
            const DvStat o = sst[w];
            s.sum += o.sum;
            s.arg = s.max > o.max ? s.arg : o.max > s.max ? o.arg : min(s.arg, o.arg);
            s.max = fmaxf(s.max, o.max);
            s.bad |= o.bad;
        }
        a.stat[(size_t)row * a.parts + part] = s;
    }
}

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
    __shared__ unsigned long long wsum[DP_GROUPS][DP_WARPS], ctot[2];
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
            const DvStat t = dv_row(a, mine), d = a.draft && !last ? dv_row(a, (size_t)a.n_rows + mine) : t;
            const int x = last ? -1 : a.tokens[mine + 1];
            int v = 1;
            if (t.bad || d.bad) v = 2;
            else if (x >= 0 && x < V) {
                const float lt = a.target[(size_t)mine * a.ldt + x];
                if (a.greedy) v = x != t.arg;
                else {
                    const float q = a.draft ? dv_prob(a.draft[(size_t)mine * a.ldd + x], a.c, d) : 1.0f;
                    v = !(__fmul_rn(a.u_accept[mine], q) < dv_prob(lt, a.c, t));
                }
            }
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
    // ---- draw from row r: the block's share is `runs` runs of 128 tokens a warp and group ----
    const float* d = a.draft && !last ? a.draft + (size_t)r * a.ldd : nullptr;
    const int x = last ? -1 : a.tokens[r + 1];
    // both rows are read in quads of the target's alignment
    const int off = dv_off(t);
    const bool same = !d || dv_off(d) == off;
    const long quads = ((long)off + V + 3) / 4;
    const int share = (int)((quads + cluster - 1) / cluster);
    const int runs = (share + DP_GROUPS * DP_THREADS - 1) / (DP_GROUPS * DP_THREADS);
    const int groups = (share + runs * DP_THREADS - 1) / (runs * DP_THREADS);
    const long q0 = (long)rank * groups * runs * DP_THREADS;
    const DvInv it = dv_inv(st), id = dv_inv(sd);
    auto load = [&](long q, bool rest, float4& tv, float4& dv) {
        tv = dv_quad(t, off, q, V);
        dv = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (d && rest) {
            if (same) dv = dv_quad(d, off, q, V);
            else {
                const long j = 4 * q - off;
                if (j >= 0 && j < V) dv.x = d[j];
                if (j + 1 >= 0 && j + 1 < V) dv.y = d[j + 1];
                if (j + 2 >= 0 && j + 2 < V) dv.z = d[j + 2];
                if (j + 3 >= 0 && j + 3 < V) dv.w = d[j + 3];
            }
        }
    };
    // floor(w 2^38) = hi 2^19 + lo: adding 2^23 downwards leaves a whole number in the low bits
    auto weights = [&](long q, bool rest, const float4& tv, const float4& dv, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
        const float e[4] = {tv.x, tv.y, tv.z, tv.w}, f[4] = {dv.x, dv.y, dv.z, dv.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float p = dv_quotient(dv_weight(e[i], a.c, st.top), it);
            if (rest) {
                if (d) p = fmaxf(p - dv_quotient(dv_weight(f[i], a.c, sd.top), id), 0.0f);
                else if (4 * q - off + i == x) p = 0.0f;
            }
            const float u = p * 524288.0f, h = __fadd_rd(u, 8388608.0f);
            hi[i] = __float_as_uint(h) & 0xfffffu;
            lo[i] = __float_as_uint(__fmaf_rd(u - (h - 8388608.0f), 524288.0f, 8388608.0f)) & 0xfffffu;
        }
    };
    for (int pass = 0; pass < 2; ++pass) {         // what is left of p over q; p itself if that is nothing
        const bool rest = pass == 0 && !last;
        unsigned long long own = 0;
        // (more than one run a group: vocabularies beyond 2^19 tokens and a block, whose groups are loaded one by one)
        for (int g0 = 0; g0 < groups; g0 += DP_AHEAD) {
            float4 tv[DP_AHEAD], dv[DP_AHEAD];
            for (int k = 0; k < runs; ++k) {
#pragma unroll
                for (int j = 0; j < DP_AHEAD; ++j) {
                    const long q = q0 + ((long)((g0 + j) * DP_WARPS + warp) * runs + k) * 32 + lane;
                    tv[j] = dv[j] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (g0 + j < groups && q < quads) load(q, rest, tv[j], dv[j]);
                }
#pragma unroll
                for (int j = 0; j < DP_AHEAD; ++j) {
                    if (g0 + j >= groups) break;
                    const long q = q0 + ((long)((g0 + j) * DP_WARPS + warp) * runs + k) * 32 + lane;
                    uint32_t hi[4], lo[4];
                    weights(q, rest, tv[j], dv[j], hi, lo);
                    const uint32_t h = __reduce_add_sync(~0u, hi[0] + hi[1] + hi[2] + hi[3]);
                    const uint32_t l = __reduce_add_sync(~0u, lo[0] + lo[1] + lo[2] + lo[3]);
                    const unsigned long long s = ((unsigned long long)h << 19) + l;
                    if (lane == 0) wsum[g0 + j][warp] = k ? wsum[g0 + j][warp] + s : s;
                }
            }
        }
        __syncthreads();
        if (warp == 0) {
            for (int i = lane; i < groups * DP_WARPS; i += 32) own += wsum[i / DP_WARPS][i % DP_WARPS];
            for (int i = 16; i; i >>= 1) own += __shfl_xor_sync(~0u, own, i);
            if (lane == 0) ctot[pass] = own;
        }
        cluster_sync();
        unsigned long long total = 0, before = 0;
        for (int c = 0; c < cluster; ++c) {
            unsigned long long v;
            asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(&ctot[pass]), c)) : "memory");
            if (c < rank) before += v;
            total += v;
        }
        if (total == 0 && pass == 0) continue;     // the whole cluster alike
        // [0, 1) in steps of 2^-24
        const unsigned long long u = (unsigned long long)(fminf(fmaxf(a.u_sample[b], 0.0f), 0.99999994f) * 16777216.0f);
        const unsigned long long goal = (total * u) >> 24;
        const unsigned long long here = ctot[pass];
        if (warp == 0 && goal >= before && goal < before + here) {
            // the group and warp that hold it: a lane an even run of sums, then within the run
            unsigned long long left = goal - before;
            const int cnt = groups * DP_WARPS, per = (cnt + 31) / 32, i0 = min(cnt, lane * per), i1 = min(cnt, i0 + per);
            unsigned long long s = 0, sum;
            for (int i = i0; i < i1; ++i) s += wsum[i / DP_WARPS][i % DP_WARPS];
            sum = s;
            for (int i = 1; i < 32; i <<= 1) {
                const unsigned long long o = __shfl_up_sync(~0u, sum, i);
                if (lane >= i) sum += o;
            }
            const int src = __ffs(__ballot_sync(~0u, left < sum)) - 1;
            left -= __shfl_sync(~0u, sum - s, src);
            int at = min(cnt, src * per);
            while (left >= wsum[at / DP_WARPS][at % DP_WARPS]) { left -= wsum[at / DP_WARPS][at % DP_WARPS]; ++at; }
            for (int k = 0; k < runs; ++k) {
                const long q = q0 + ((long)at * runs + k) * 32 + lane;
                unsigned long long w[4] = {0, 0, 0, 0};
                if (q < quads) {
                    float4 tv, dv;
                    uint32_t hi[4], lo[4];
                    load(q, rest, tv, dv);
                    weights(q, rest, tv, dv, hi, lo);
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = ((unsigned long long)hi[i] << 19) + lo[i];
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
                    int e = 0;
                    while (e < 3 && left >= w[e]) left -= w[e++];
                    const int tok = (int)(4 * q - off) + e;
                    a.next[b] = tok;
                    if (a.logp) a.logp[r] = dv_logp(t[tok], a.c, st);
                }
                break;
            }
        }
        break;
    }
    cluster_sync();                                // the totals are read by the others
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
    // blocks of a sequence's draw: as many as are resident at once (two an SM), 16 at most
    a.cluster = DP_CLUSTER;
    while (a.cluster > 1 && (long)n_seqs * a.cluster > 2L * ctx->num_sms) a.cluster >>= 1;
    const long parts = (quads + part - 1) / part, grid = parts * rows, pick = (long)n_seqs * a.cluster;
    if (grid > INT_MAX || pick > INT_MAX) return fail(TK_ERR_INVALID, "tk_draft_verify: too many rows");
    a.parts = (int)parts;
    a.part_quads = (int)((quads + parts - 1) / parts);
    tk_status st = ws_ensure(ctx, (size_t)grid * sizeof(DvStat), s);
    if (st != TK_OK) return st;
    a.stat = static_cast<DvStat*>(ctx->ws);
    static std::atomic<uint64_t> attr_done{0};     // clusters of 16 are more than every GPU must offer: per device
    if (!(attr_done.load(std::memory_order_relaxed) >> (ctx->device & 63) & 1)) {
        const cudaError_t e = cudaFuncSetAttribute(dv_pick_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return cuda_fail(e, "draft verify cluster attribute");
        attr_done.fetch_or(1ull << (ctx->device & 63));
    }
    ProfScope ps(ctx, s, PK_SERVE);
    const bool small = a.part_quads <= 4 * DV_THREADS;
    auto kern = a.greedy ? (small ? dv_rows_kernel<true, 4> : dv_rows_kernel<true, DV_QUADS>)
                         : (small ? dv_rows_kernel<false, 4> : dv_rows_kernel<false, DV_QUADS>);
    kern<<<(unsigned)grid, DV_THREADS, 0, s>>>(a);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)pick);
    cfg.blockDim = dim3(DP_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = a.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, dv_pick_kernel, a);
    ctx->launches += 2;
    if (e != cudaSuccess) return cuda_fail(e, "draft verify launch");
    return cuda_fail(cudaGetLastError(), "draft verify launch");
}

}  // namespace tk
