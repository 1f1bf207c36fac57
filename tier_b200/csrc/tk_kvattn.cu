// tk_kvattn.cu -- tk_kv_attend: attention of new tokens over the 4-bit cache.
#include "tk_kv.cuh"

namespace tk {

struct KvaArgs {
    KvView c;
    SeqView s;
    const void* q;
    void* out;
    long ldq, ldo;
    int n_heads, group, window;
    float scale2;         // scale * log2(e)
    float* part;          // parts of divided rows (workspace)
    int* count;           // finished parts of each sequence and key/value head, zero between calls
    int* status;
};

template <int DT>
__device__ __forceinline__ float ld_elem(const void* p, size_t i) {
    if constexpr (DT == TK_DT_F32) return static_cast<const float*>(p)[i];
    else if constexpr (DT == TK_DT_F16) return h2f_bits(static_cast<const uint16_t*>(p)[i]);
    else return __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16);
}
template <int DT>
__device__ __forceinline__ void st_elem(void* p, size_t i, float x) {
    if constexpr (DT == TK_DT_F32) static_cast<float*>(p)[i] = x;
    else if constexpr (DT == TK_DT_F16) static_cast<uint16_t*>(p)[i] = f2h_bits(x);
    else static_cast<uint16_t*>(p)[i] = f2bf_bits(x);
}

// One warp per (row, head): 32 keys at a time, a key per lane for the scores,
// then head_dim / 32 outputs per lane over the 32 probabilities, with the
// running maximum and sum of the softmax.
template <int D, int DT>
__global__ void __launch_bounds__(128) kv_attend_rows_kernel(const KvaArgs a) {
    constexpr int E = D / 32;
    __shared__ float qs[4][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long item = (long)blockIdx.x * 4 + warp;
    if (item >= (long)a.s.n_tokens * a.n_heads) return;
    const int r = (int)(item / a.n_heads), h = (int)(item % a.n_heads), kh = h / a.group;
    const int b = seq_of_row(a.s.q_start, a.s.n_seqs, r);
    const SeqInfo sq = seq_info(a.s, a.c.page_shift, b, a.status);
    if (r < sq.row0 || r - sq.row0 >= sq.n_new) return;
    const int pos = sq.kv - sq.n_new + (r - sq.row0);
    const int first = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    for (int i = lane; i < D; i += 32) qs[warp][i] = ld_elem<DT>(a.q, (size_t)r * a.ldq + (size_t)h * D + i);
    __syncwarp();
    float o[E] = {}, m = -INFINITY, l = 0.0f;
    for (int k0 = first; k0 <= pos; k0 += 32) {
        const int key = k0 + lane;
        float s = -INFINITY;
        size_t row = 0;
        if (key <= pos) {
            row = kv_row(a.c, page_of(a.s, a.c, b, key, a.status), kh, key);
            const uint32_t* w = reinterpret_cast<const uint32_t*>(a.c.kq) + row * (D / 8);
            s = 0.0f;
            for (int g = 0; g < D / 32; ++g) {
                float t = 0.0f;
                for (int j = 0; j < 4; ++j)
                    for (int e = 0; e < 8; ++e) t += qs[warp][g * 32 + j * 8 + e] * (float)kv_nibble(w[g * 4 + j], e);
                s += t * __half2float(a.c.ks[row * (D / 32) + g]);
            }
            s *= a.scale2;
        }
        float mx = s;
        for (int i = 16; i; i >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, i));
        const float mn = fmaxf(m, mx), fix = exp2f(m - mn);
        m = mn;
        const float p = key <= pos ? exp2f(s - m) : 0.0f;
        float sum = p;
        for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
        l = l * fix + sum;
        for (int e = 0; e < E; ++e) o[e] *= fix;
        const int n = min(32, pos - k0 + 1);
        for (int j = 0; j < n; ++j) {
            const float pj = __shfl_sync(~0u, p, j);
            const size_t rj = __shfl_sync(~0u, (unsigned long long)row, j);
            const int e0 = lane * E;
            const uint32_t w = reinterpret_cast<const uint32_t*>(a.c.vq)[rj * (D / 8) + (e0 >> 3)];
            const float pd = pj * __half2float(a.c.vs[rj * (D / 32) + (e0 >> 5)]);
            for (int e = 0; e < E; ++e) o[e] += pd * (float)kv_nibble(w, (e0 & 7) + e);
        }
    }
    for (int e = 0; e < E; ++e)
        st_elem<DT>(a.out, (size_t)r * a.ldo + (size_t)h * D + lane * E + e, l == 0.0f ? 0.0f : o[e] / l);
}

// Output of row r (of the block), values e .. e + 3: O / l, zero where nothing was seen.
template <int DT, int D, class Item>
__device__ __forceinline__ void kv_store_out(const KvaArgs& a, const Item& it, int r, int e, float4 o, float l) {
    const float inv = l == 0.0f ? 0.0f : __fdividef(1.0f, l);
    const size_t at = (size_t)(it.row0 + r / a.group) * a.ldo + (size_t)(it.head * a.group + r % a.group) * D + e;
    if (l == 0.0f) o = make_float4(0, 0, 0, 0);
    if constexpr (DT == TK_DT_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    } else {
        uint2 w;
        if constexpr (DT == TK_DT_F16) {
            w.x = (uint32_t)f2h_bits(o.x * inv) | ((uint32_t)f2h_bits(o.y * inv) << 16);
            w.y = (uint32_t)f2h_bits(o.z * inv) | ((uint32_t)f2h_bits(o.w * inv) << 16);
        } else {
            w.x = (uint32_t)f2bf_bits(o.x * inv) | ((uint32_t)f2bf_bits(o.y * inv) << 16);
            w.y = (uint32_t)f2bf_bits(o.z * inv) | ((uint32_t)f2bf_bits(o.w * inv) << 16);
        }
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = w;
    }
}

// The last of a head's parts to finish joins them, in the order of the keys
// (the result does not depend on which block that is): parts are [16 rows, D]
// of O, then (m, l) of each row.  The counter is left at zero for the next call.
template <int D, int DT, class Item>
__device__ __forceinline__ void kv_join_last(const KvaArgs& a, const Item& it, int live, int* sh_last) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        int* n = a.count + (size_t)it.b * a.c.heads + it.head;
        const int done = atomicAdd(n, 1) + 1;
        *sh_last = done == it.chunks;
        if (done == it.chunks) *n = 0;
    }
    __syncthreads();
    if (!*sh_last) return;
    __threadfence();
    const float* base = a.part + (size_t)it.first * (16 * (D + 2));
    for (int i = threadIdx.x; i < live * (D / 4); i += blockDim.x) {
        const int r = i / (D / 4), e = (i - r * (D / 4)) * 4;
        float m = -INFINITY, l = 0.0f;
        for (int c = 0; c < it.chunks; ++c) m = fmaxf(m, __ldcg(base + (size_t)c * (16 * (D + 2)) + 16 * D + 2 * r));
        const float ref = m == -INFINITY ? 0.0f : m;
        float4 o = make_float4(0, 0, 0, 0);
        for (int c = 0; c < it.chunks; ++c) {
            const float* part = base + (size_t)c * (16 * (D + 2));
            const float f = fast_exp2(__ldcg(part + 16 * D + 2 * r) - ref);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(part + r * D + e));
            l += __ldcg(part + 16 * D + 2 * r + 1) * f;
            o.x += v.x * f; o.y += v.y * f; o.z += v.z * f; o.w += v.w * f;
        }
        kv_store_out<DT, D>(a, it, r, e, o, l);
    }
}

// ---------------------------------------------------------------------------
// Few rows per key/value head (new tokens x heads of the group <= 16, or <= 8
// for fp32): the cache is streamed once, divided among thread blocks.
//
// One warp takes units of 32 keys.  S = Q K^T and O += P V are m16n8k16 fp16
// products: the 16 matrix rows are the query rows (fp32: 8 rows as hi and lo
// fp16 parts, so that q and p keep 22 bits; their products meet in one lane).
// The order of the reduction index is free, so lane (g, t) = (lane / 4,
// lane % 4) uses what it can load in one piece: for K the t-th quarter of a
// key's row (16 bytes at head_dim 128), for V the g-th eighth of rows t and
// t + 4 of each 8 keys.  A key's scale multiplies its fp16 numbers exactly.
//
// The softmax keeps a reference exponent per row that moves only when a unit
// exceeds it by 2^8 (p stays below 2^8, fp16's rounding is relative, and the
// rescaling of O is rare); l is summed per lane in fp32 and joined at the end.
//
// Rows are copied by cp.async.bulk into each warp's own ring (no barrier
// between warps), as far ahead as the ring is deep.
// ---------------------------------------------------------------------------
constexpr int KD_WARPS = 4, KD_STAGES = 4, KD_UNIT = 32;

template <int D>
struct KdGeo {
    static constexpr int QB = KD_UNIT * D / 2, SB = KD_UNIT * D / 16;      // bytes of numbers, of scales
    static constexpr int STAGE = 2 * QB + 2 * SB;
    static constexpr int RING = KD_WARPS * KD_STAGES * STAGE;
    static constexpr int JOIN = KD_WARPS * (16 * (D + 4) * 4 + 16 * 8);    // each warp's O rows, m and l
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;
};

// What one block works on: part `chunk` of `chunks` of one sequence and
// key/value head.  Every block finds its own from the device's lengths: units
// of all sequences and heads are divided so that about `slots` blocks' worth
// of equal parts results, no part below `least` units.
struct KdItem {
    int b, head, chunk, chunks, u0, u1;    // units [u0, u1) of the sequence
    int kv, n_new, row0, lo;               // keys [lo, kv) are seen by some row
    long first;                            // item number of the head's chunk 0
};
__device__ __forceinline__ int kd_units(const SeqInfo& q, int window, int& lo) {
    lo = 0;
    if (q.n_new == 0) return 0;
    const int first = q.kv - q.n_new - window + 1;
    if (window > 0 && first > 0) lo = first;
    const int n = (q.kv + KD_UNIT - 1) / KD_UNIT - lo / KD_UNIT;
    return n > 0 ? n : 1;                  // no key at all: one part that writes zeros
}
__device__ __forceinline__ bool kd_find(const KvaArgs& a, long item, int slots, int least, KdItem& it) {
    const int lane = threadIdx.x & 31;
    long total = 0;
    for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
        int lo, n = 0;
        if (b0 + lane < a.s.n_seqs) n = kd_units(seq_info(a.s, a.c.page_shift, b0 + lane, a.status), a.window, lo);
        total += __reduce_add_sync(~0u, n);
    }
    total *= a.c.heads;
    long per = (total + slots - 1) / slots;
    if (per < least) per = least;
    long before = 0;
    for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
        SeqInfo q{0, 0, 0};
        int lo = 0, n = 0;
        if (b0 + lane < a.s.n_seqs) {
            q = seq_info(a.s, a.c.page_shift, b0 + lane, nullptr);
            n = kd_units(q, a.window, lo);
        }
        const int chunks = (int)((n + per - 1) / per);
        const long mine = (long)chunks * a.c.heads;
        long sum = mine;                   // items up to and with this lane's sequence
        for (int i = 1; i < 32; i <<= 1) {
            const long o = __shfl_up_sync(~0u, sum, i);
            if (lane >= i) sum += o;
        }
        const unsigned hit = __ballot_sync(~0u, item < before + sum);
        if (hit) {
            const int src = __ffs(hit) - 1;
            it.b = b0 + src;
            it.chunks = __shfl_sync(~0u, chunks, src);
            it.kv = __shfl_sync(~0u, q.kv, src);
            it.n_new = __shfl_sync(~0u, q.n_new, src);
            it.row0 = __shfl_sync(~0u, q.row0, src);
            it.lo = __shfl_sync(~0u, lo, src);
            n = __shfl_sync(~0u, n, src);
            const long at = item - before - __shfl_sync(~0u, sum - mine, src);
            it.head = (int)(at / it.chunks);
            it.chunk = (int)(at - (long)it.head * it.chunks);
            it.first = item - it.chunk;
            const int u = it.lo / KD_UNIT;
            it.u0 = u + (int)((long)n * it.chunk / it.chunks);
            it.u1 = u + (int)((long)n * (it.chunk + 1) / it.chunks);
            return true;
        }
        before += __shfl_sync(~0u, sum, 31);
    }
    return false;
}

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <int DT>
__device__ __forceinline__ void load_pairs8(const void* p, size_t at, float (&x)[8]) {
    if constexpr (DT == TK_DT_F32) {
        const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
        const float4 u = f[0], v = f[1];
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == TK_DT_BF16) {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            } else {
                x[2 * i] = h2f_bits((uint16_t)(w[i] & 0xffffu));
                x[2 * i + 1] = h2f_bits((uint16_t)(w[i] >> 16));
            }
        }
    }
}
// 2^e with max * 2^e in [2^13, 2^14); 1 for zero and for what is not finite.
__device__ __forceinline__ float q_unit(float max, float& back) {
    const int e = (int)(__float_as_uint(max) >> 23);
    if (e < 14 || e >= 255) { back = 1.0f; return 1.0f; }
    back = __uint_as_float((uint32_t)(e - 13) << 23);             // 2^(e - 127 - 13)
    return __uint_as_float((uint32_t)(254 - (e - 13)) << 23);
}

template <int D, int DT>
__global__ void __launch_bounds__(KD_WARPS * 32, 3) kv_decode_kernel(const KvaArgs a, int slots, int least) {
    using G = KdGeo<D>;
    constexpr bool SPLIT = DT == TK_DT_F32;
    constexpr int ROWS = SPLIT ? 8 : 16, NR = SPLIT ? 1 : 2;       // query rows of the block, of a lane
    constexpr int KW = D / 32, VW = D / 64;                        // 32-bit words of a lane's piece of a key / value row
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bar[KD_WARPS][KD_STAGES];
    __shared__ int sh_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    KdItem it;
    if (!kd_find(a, blockIdx.x, slots, least, it)) return;
    uint8_t* ring = smem + warp * (KD_STAGES * G::STAGE);
    if (lane == 0) {
        for (int s = 0; s < KD_STAGES; ++s) mbar_init(&bar[warp][s], 1);
        fence_mbar_init();
    }
    __syncwarp();

    // ---- rows: row r of the block is token r / group, head r % group ----
    const int rows = it.n_new * a.group, pos0 = it.kv - it.n_new;
    uint32_t qf[2 * KW][4];
    float sc[NR];
    int limit[NR], from[NR];                                       // keys [from, limit) are seen
    {
        float x[NR][KW][8];
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int r = g + 8 * i;
            float mx = 0.0f;
            limit[i] = from[i] = 0;
            if (r < rows) {
                const int tok = r / a.group;
                limit[i] = pos0 + tok + 1;
                from[i] = a.window > 0 ? limit[i] - a.window : 0;
                const size_t at = (size_t)(it.row0 + tok) * a.ldq + (size_t)(it.head * a.group + r % a.group) * D + t * (D / 4);
#pragma unroll
                for (int w = 0; w < KW; ++w) {
                    load_pairs8<DT>(a.q, at + w * 8, x[i][w]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x[i][w][e]));
                }
            } else {
#pragma unroll
                for (int w = 0; w < KW; ++w)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[i][w][e] = 0.0f;
            }
            mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
            float back;
            const float up = copysignf(q_unit(mx, back), a.scale2);
            sc[i] = back * fabsf(a.scale2);
#pragma unroll
            for (int w = 0; w < KW; ++w)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][w][e] *= up;
        }
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int p = 0; p < 2; ++p) {
                    const int e = 4 * h + 2 * p;
                    const uint32_t hi = pack_half2(x[0][w][e], x[0][w][e + 1]);
                    qf[2 * w + h][2 * p] = hi;
                    if constexpr (SPLIT) {
                        const __half2 hh = as_half2(hi);
                        qf[2 * w + h][2 * p + 1] = pack_half2(x[0][w][e] - __low2float(hh), x[0][w][e + 1] - __high2float(hh));
                    } else {
                        qf[2 * w + h][2 * p + 1] = pack_half2(x[1][w][e], x[1][w][e + 1]);
                    }
                }
    }

    float o[D / 8][4], m[NR], l[NR];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
#pragma unroll
    for (int i = 0; i < NR; ++i) { m[i] = -INFINITY; l[i] = 0.0f; }

    // ---- the warp's units: u0 + warp, + 4, ... ----
    const int mine = it.u1 - it.u0 > warp && it.kv > 0 ? (it.u1 - it.u0 - warp + KD_WARPS - 1) / KD_WARPS : 0;
    const size_t page_rows = (size_t)1 << a.c.page_shift;
    const int ppu = a.c.page_shift < 5 ? 2 : 1;                    // pages per unit (16-token pages: two)
    const int run = KD_UNIT / ppu;
    int pid[2] = {0, 0};
    auto issue = [&](int i) {                                      // whole warp; lane 0 copies
        if (i >= mine) return;
        const int u = it.u0 + warp + i * KD_WARPS, stage = i % KD_STAGES;
        if ((i & 31) == 0) {                                       // page ids of the next 32 units, one a lane
            const int pos = (it.u0 + warp + (i + lane) * KD_WARPS) * KD_UNIT;
#pragma unroll
            for (int p = 0; p < 2; ++p)
                if (p < ppu && pos + p * run < it.kv) pid[p] = page_of(a.s, a.c, it.b, pos + p * run, a.status);
        }
        const int id0 = __shfl_sync(~0u, pid[0], i & 31), id1 = __shfl_sync(~0u, pid[1], i & 31);
        if (lane == 0) {
            const int pos = u * KD_UNIT, n = ppu == 2 && pos + run < it.kv ? 2 : 1;
            uint8_t* dst = ring + stage * G::STAGE;
            mbar_arrive_expect_tx(&bar[warp][stage], (uint32_t)(n * run * (D + D / 8)));
            for (int p = 0; p < n; ++p) {
                const size_t row = ((size_t)(p ? id1 : id0) * a.c.heads + it.head) * page_rows + ((pos + p * run) & (page_rows - 1));
                const int at = p * run;
                bulk_load(dst + at * (D / 2), a.c.kq + row * (D / 2), run * (D / 2), &bar[warp][stage]);
                bulk_load(dst + G::QB + at * (D / 2), a.c.vq + row * (D / 2), run * (D / 2), &bar[warp][stage]);
                bulk_load(dst + 2 * G::QB + at * (D / 16), a.c.ks + row * (D / 32), run * (D / 16), &bar[warp][stage]);
                bulk_load(dst + 2 * G::QB + G::SB + at * (D / 16), a.c.vs + row * (D / 32), run * (D / 16), &bar[warp][stage]);
            }
        }
    };
    for (int i = 0; i < KD_STAGES - 1; ++i) issue(i);

    for (int i = 0; i < mine; ++i) {
        issue(i + KD_STAGES - 1);
        const int stage = i % KD_STAGES, key0 = (it.u0 + warp + i * KD_WARPS) * KD_UNIT;
        if (!__all_sync(~0u, mbar_wait(&bar[warp][stage], (i / KD_STAGES) & 1, a.status))) {
            for (int k = i + 1; k < min(i + KD_STAGES, mine); ++k)  // reported; the copies in flight end first
                mbar_wait(&bar[warp][k % KD_STAGES], (k / KD_STAGES) & 1, a.status);
            break;
        }
        const uint8_t* kq = ring + stage * G::STAGE;
        const uint8_t* vq = kq + G::QB;
        const __half* ks = reinterpret_cast<const __half*>(kq + 2 * G::QB);
        const __half* vs = reinterpret_cast<const __half*>(kq + 2 * G::QB + G::SB);

        // S: matrix column n of tile j is key 8 j + (n >> 1) + 4 (n & 1), so
        // that lane t's two columns are keys t and t + 4 of the 8
        float s[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
            const int key = 8 * j + (g >> 1) + 4 * (g & 1);
            uint32_t w[KW];
            if constexpr (KW == 4) {
                const uint4 u = *reinterpret_cast<const uint4*>(kq + key * (D / 2) + t * 16);
                w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(kq + key * (D / 2) + t * 8);
                w[0] = u.x; w[1] = u.y;
            }
            const __half2 d = __half2half2(ks[key * (D / 32) + (t * D / 128)]);
#pragma unroll
            for (int i2 = 0; i2 < KW; ++i2) {
                uint32_t b[4];
                kv_fields(w[i2], d, b);
                mma_16816(s[j], qf[2 * i2], b[0], b[1]);
                mma_16816(s[j], qf[2 * i2 + 1], b[2], b[3]);
            }
        }
        const bool edge = key0 + KD_UNIT > pos0 + 1 || key0 < it.lo + it.n_new;
        float p[NR][8];
        float top[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            top[r] = -INFINITY;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float v = SPLIT ? s[j >> 1][j & 1] + s[j >> 1][2 + (j & 1)] : s[j >> 1][2 * r + (j & 1)];
                v *= sc[r];
                if (edge) {
                    const int key = key0 + 8 * (j >> 1) + t + 4 * (j & 1);
                    if (key >= limit[r] || key < from[r]) v = -INFINITY;
                }
                p[r][j] = v;
                top[r] = fmaxf(top[r], v);
            }
            top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(~0u, top[r], 2));
        }
        bool move = top[0] > m[0] + 8.0f;
        if constexpr (NR == 2) move |= top[1] > m[1] + 8.0f;
        if (__any_sync(~0u, move)) {
            float f[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const float mn = fmaxf(m[r], top[r]);
                f[r] = mn == -INFINITY ? 1.0f : fast_exp2(m[r] - mn);
                m[r] = mn;
                l[r] *= f[r];
            }
#pragma unroll
            for (int i2 = 0; i2 < D / 8; ++i2) {
                o[i2][0] *= f[0]; o[i2][1] *= f[0];
                o[i2][2] *= f[NR - 1]; o[i2][3] *= f[NR - 1];
            }
        }
        uint32_t pa[2][4];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const float ref = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[r][j] = fast_exp2(p[r][j] - ref);
                l[r] += p[r][j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t hi = pack_half2(p[0][2 * j], p[0][2 * j + 1]);
            pa[j >> 1][2 * (j & 1)] = hi;
            if constexpr (SPLIT) {
                const __half2 hh = as_half2(hi);
                pa[j >> 1][2 * (j & 1) + 1] = pack_half2(p[0][2 * j] - __low2float(hh), p[0][2 * j + 1] - __high2float(hh));
            } else {
                pa[j >> 1][2 * (j & 1) + 1] = pack_half2(p[1][2 * j], p[1][2 * j + 1]);
            }
        }
        // O: matrix column n of tile e' is value (D / 8) n + e' of the head
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t w[4][VW];                                     // keys 16 h + t, + 4, + 8, + 12
            __half d[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int key = 16 * h + 4 * j + t;
                if constexpr (VW == 2) {
                    const uint2 u = *reinterpret_cast<const uint2*>(vq + key * (D / 2) + g * 8);
                    w[j][0] = u.x; w[j][1] = u.y;
                } else {
                    w[j][0] = *reinterpret_cast<const uint32_t*>(vq + key * (D / 2) + g * 4);
                }
                d[j] = vs[key * (D / 32) + (g * D / 256)];
                // a row that nothing sees may hold any scale
                if (edge && (key0 + key >= it.kv || key0 + key < it.lo)) d[j] = __ushort_as_half(0);
            }
            const __half2 d0 = __halves2half2(d[0], d[1]), d1 = __halves2half2(d[2], d[3]);
#pragma unroll
            for (int i2 = 0; i2 < VW; ++i2)
#pragma unroll
                for (int half = 0; half < 2; ++half) {             // fields 0..3: values 0 2 4 6; 4..7: 1 3 5 7
                    uint32_t b0[4], b1[4];
                    const uint32_t sel = half ? 0x7632u : 0x5410u;
                    kv_fields(__byte_perm(w[0][i2], w[1][i2], sel), d0, b0);
                    kv_fields(__byte_perm(w[2][i2], w[3][i2], sel), d1, b1);
#pragma unroll
                    for (int f = 0; f < 4; ++f) mma_16816(o[8 * i2 + 2 * f + half], pa[h], b0[f], b1[f]);
                }
        }
        __syncwarp();                                              // the stage may be overwritten
    }

    // ---- join the warps: lane sums, then O in the ring's memory ----
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        l[r] += __shfl_xor_sync(~0u, l[r], 1);
        l[r] += __shfl_xor_sync(~0u, l[r], 2);
    }
    __syncthreads();                                               // every warp is done with its ring
    constexpr int OLD = D + 4;
    float* osh = reinterpret_cast<float*>(smem);
    float* msh = osh + KD_WARPS * 16 * OLD;
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        float* to = osh + (warp * 16 + g + 8 * r) * OLD;
#pragma unroll
        for (int e = 0; e < D / 8; ++e)
#pragma unroll
            for (int c = 0; c < 2; ++c)
                to[(2 * t + c) * (D / 8) + e] = SPLIT ? o[e][c] + o[e][2 + c] : o[e][2 * r + c];
        if (t == 0) {
            msh[(warp * 16 + g + 8 * r) * 2] = m[r];
            msh[(warp * 16 + g + 8 * r) * 2 + 1] = l[r];
        }
    }
    __syncthreads();
    const bool whole = it.chunks == 1;
    const int live = min(rows, ROWS);
    for (int i = threadIdx.x; i < live * (D / 4); i += KD_WARPS * 32) {
        const int r = i / (D / 4), e = (i - r * (D / 4)) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) mm = fmaxf(mm, msh[(w * 16 + r) * 2]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f;
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
            const float f = fast_exp2(msh[(w * 16 + r) * 2] - ref);
            const float4 v = *reinterpret_cast<const float4*>(osh + (w * 16 + r) * OLD + e);
            ll += msh[(w * 16 + r) * 2 + 1] * f;
            acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        }
        if (whole) kv_store_out<DT, D>(a, it, r, e, acc, ll);
        else {
            float* part = a.part + (size_t)blockIdx.x * (16 * (D + 2));
            *reinterpret_cast<float4*>(part + r * D + e) = acc;
            if (e == 0) {
                part[16 * D + 2 * r] = mm;
                part[16 * D + 2 * r + 1] = ll;
            }
        }
    }
    if (whole) return;
    kv_join_last<D, DT>(a, it, live, &sh_last);
}

template <int D>
static void go_rows(const KvaArgs& a, int dtype, unsigned grid, cudaStream_t st) {
    if (dtype == TK_DT_F32) kv_attend_rows_kernel<D, TK_DT_F32><<<grid, 128, 0, st>>>(a);
    else if (dtype == TK_DT_F16) kv_attend_rows_kernel<D, TK_DT_F16><<<grid, 128, 0, st>>>(a);
    else kv_attend_rows_kernel<D, TK_DT_BF16><<<grid, 128, 0, st>>>(a);
}

// Zeroed counters for the join, grown on demand (synchronizes the device then).
static tk_status count_ensure(tk_ctx* ctx, size_t n) {
    if (n <= ctx->kv_count_len) return TK_OK;
    cudaError_t e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return cuda_fail(e, "tk_kv_attend: counter growth");
    if (ctx->kv_count) cudaFree(ctx->kv_count);
    ctx->kv_count = nullptr;
    ctx->kv_count_len = 0;
    n = (n + 1023) / 1024 * 1024;
    e = cudaMalloc(&ctx->kv_count, n * sizeof(int));
    if (e == cudaSuccess) e = cudaMemset(ctx->kv_count, 0, n * sizeof(int));
    if (e == cudaSuccess) e = cudaDeviceSynchronize();
    if (e != cudaSuccess) return cuda_fail(e, "tk_kv_attend: counters");
    ctx->kv_count_len = n;
    return TK_OK;
}

template <int D, int DT>
static tk_status go_decode_t(tk_ctx* ctx, const KvaArgs& a, unsigned grid, int slots, int least, cudaStream_t st) {
    static std::atomic<uint64_t> attr_done{0};
    auto kern = kv_decode_kernel<D, DT>;
    cudaError_t e = smem_attr_once(kern, KdGeo<D>::SMEM, ctx->device, attr_done);
    if (e != cudaSuccess) return cuda_fail(e, "kv decode smem attribute");
    ProfScope ps(ctx, st, PK_SERVE);
    kern<<<grid, KD_WARPS * 32, KdGeo<D>::SMEM, st>>>(a, slots, least);
    ctx->launches++;
    return cuda_fail(cudaGetLastError(), "kv decode launch");
}

template <int D>
static tk_status go_decode(tk_ctx* ctx, KvaArgs& a, int dtype, cudaStream_t st) {
    const long pairs = (long)a.s.n_seqs * a.c.heads;
    const int slots = 3 * ctx->num_sms, least = KD_WARPS;
    const long grid = slots + pairs;      // no division has more parts: sum of ceil(units / per) < total / per + pairs
    if (grid > INT32_MAX) return fail(TK_ERR_INVALID, "tk_kv_attend: too many sequences");
    tk_status r = ws_ensure(ctx, (size_t)grid * (16 * (D + 2)) * sizeof(float), st);
    if (r == TK_OK) r = count_ensure(ctx, (size_t)pairs);
    if (r != TK_OK) return r;
    a.part = static_cast<float*>(ctx->ws);
    a.count = ctx->kv_count;
    if (dtype == TK_DT_F32) return go_decode_t<D, TK_DT_F32>(ctx, a, (unsigned)grid, slots, least, st);
    if (dtype == TK_DT_F16) return go_decode_t<D, TK_DT_F16>(ctx, a, (unsigned)grid, slots, least, st);
    return go_decode_t<D, TK_DT_BF16>(ctx, a, (unsigned)grid, slots, least, st);
}

tk_status launch_kv_attend(tk_ctx* ctx, const tk_kvcache& c, const tk_seqs& s, const void* q, int dtype, long ldq,
                           int n_heads, float scale, int window, void* out, long ldo, cudaStream_t st) {
    KvaArgs a;
    a.c = kv_view(c);
    a.s = seq_view(s);
    a.q = q; a.out = out;
    a.ldq = ldq; a.ldo = ldo;
    a.n_heads = n_heads;
    a.group = n_heads / c.n_kv_heads;
    a.window = window;
    a.scale2 = (float)((double)scale * 1.4426950408889634);
    a.status = ctx->status;
    const long grid = ((long)s.n_tokens * n_heads + 3) / 4;
    if (grid > INT32_MAX) return fail(TK_ERR_INVALID, "tk_kv_attend: too many rows");
    if ((long)s.max_new * a.group <= (dtype == TK_DT_F32 ? 8 : 16))
        return c.head_dim == 64 ? go_decode<64>(ctx, a, dtype, st) : go_decode<128>(ctx, a, dtype, st);
    ProfScope ps(ctx, st, PK_SERVE);
    if (c.head_dim == 64) go_rows<64>(a, dtype, (unsigned)grid, st);
    else go_rows<128>(a, dtype, (unsigned)grid, st);
    ctx->launches++;
    return cuda_fail(cudaGetLastError(), "kv attend launch");
}

}  // namespace tk
