// tk_kvcache.cu -- tk_kv_append and tk_kv_read: rounding keys and values to
// the 4-bit cache and expanding them again.
#include "tk_f32x2.cuh"
#include "tk_kv.cuh"

namespace tk {

constexpr int KVC_THREADS = 256;

// Eight values as they are in memory, and widened.
template <int DT>
struct Raw8 {
    uint4 u[DT == TK_DT_F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ void widen8(const Raw8<DT>& r, float (&x)[8]) {
    const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
    if constexpr (DT == TK_DT_F32) {
        const uint32_t v[4] = {r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = __uint_as_float(w[i]);
            x[4 + i] = __uint_as_float(v[i]);
        }
    } else {
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

// One item is 8 consecutive values of one token's k or v row; four lanes make
// a group of 32.  A warp takes up to ITEMS * 32 items of one such row: it
// finds the token's place once, and its loads are in flight together.
// Bound: long appends by instructions (issue 75 % busy, the integer pipe 67 %:
// the extreme, the exact rounding, the packing), reading back by the latency of
// its loads (issue 65 %, stalls on them 7.8 an instruction); single
// tokens by the launch.  Measured: 13 thousand bf16 rows of k and v (8
// key/value heads of 128) appended and read back, 117 MB in 32 us, 3.65 TB/s,
// where an item a thread took 79; 16 single fp32 tokens 5.2 us for both calls
// in a graph, 12.6 with their host side.
struct KvcArgs {
    KvView c;
    SeqView s;
    void *k, *v;          // rows in (append) or out (read)
    long ldk, ldv;
    int items, chunks;    // of a row: heads * dim / 8 items; warps
    int* status;
};

// Sequence of packed row r by a warp: 32 starts are compared at once.
__device__ __forceinline__ int seq_of_row_warp(const int32_t* q_start, int n_seqs, int r) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = n_seqs;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + lane * step;
        const unsigned at_or_before = __ballot_sync(~0u, lane * step < n && q_start[at] <= r);
        const int k = at_or_before ? 31 - __clz(at_or_before) : 0;
        n = min(step, n - k * step);
        lo += k * step;
    }
    return lo;
}

// A warp's place: its lane's first item in the packed row, and in the cache.
// Later items are 32 further on: 8 SIZE * 32 bytes of the packed row, 32 * 32 /
// dim * 8 heads (page_tokens rows each) of the cache.
struct Where {
    bool ok;
    int left;             // items of the row from the lane's first on
    uint8_t *x, *q, *s;
    uint32_t qstep, sstep;
};
template <int SIZE>
__device__ __forceinline__ bool where_is(const KvcArgs& a, int items_of_warp, Where& w) {
    const unsigned warp = blockIdx.x * (KVC_THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const unsigned row = warp / a.chunks, token = row >> 1, chunk = warp - row * a.chunks;
    const bool v = row & 1;
    if (token >= (unsigned)a.s.n_tokens) return false;
    const int b = seq_of_row_warp(a.s.q_start, a.s.n_seqs, token);
    const SeqInfo q = seq_info(a.s, a.c.page_shift, b, a.status);
    const int at = (int)token - q.row0, pos = q.kv - q.n_new + at;
    int page = 0;
    w.ok = at >= 0 && at < q.n_new && pos >= 0 && page_at(a.s, a.c, b, pos, a.status, page);   // (alike in all lanes)
    const int shift = a.c.dim == 128 ? 4 : 3;                      // items of a head
    const uint32_t item = chunk * items_of_warp + lane, word = item & ((1u << shift) - 1);
    w.left = a.items - (int)item;
    w.x = static_cast<uint8_t*>(v ? a.v : a.k) + ((size_t)token * (v ? a.ldv : a.ldk) + (size_t)item * 8) * SIZE;
    const size_t held = w.ok ? kv_row(a.c, page, item >> shift, pos) : 0;
    w.q = (v ? a.c.vq : a.c.kq) + held * (a.c.dim >> 1) + word * 4;
    w.s = reinterpret_cast<uint8_t*>(v ? a.c.vs : a.c.ks) + held * (a.c.dim >> 4) + (word >> 2) * 2;
    const uint32_t rows = (32u >> shift) << a.c.page_shift;
    w.qstep = rows * (a.c.dim >> 1);
    w.sstep = rows * (a.c.dim >> 4);
    return true;
}

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float min3_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// The group's value of largest magnitude, the first of several.  Four lanes.
__device__ __forceinline__ float group_extreme(const float (&x)[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (fabsf(x[i]) > fabsf(m)) m = x[i];
#pragma unroll
    for (int step = 1; step < 4; step <<= 1) {
        const float o = __shfl_xor_sync(~0u, m, step);
        if (fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && (threadIdx.x & step))) m = o;
    }
    return m;
}

// The arithmetic is kept short, as it is the bound: the extreme from the group's
// largest and smallest value (value by value only where both are as far from
// zero, or not finite), whole numbers by adding 2^23 downwards, whose bits are
// shifted together.  Four lanes share a group so that every load is 16 or 32
// consecutive bytes a lane and a warp's stores fill whole 32-byte sectors.
template <int DT, int ITEMS>
__global__ void __launch_bounds__(KVC_THREADS) kv_append_kernel(const KvcArgs a) {
    constexpr int SIZE = DT == TK_DT_F32 ? 4 : 2;
    pdl_trigger();
    pdl_wait();
    Where w;
    if (!where_is<SIZE>(a, ITEMS * 32, w) || !w.ok) return;
    const bool holds_scale = (threadIdx.x & 3) == 0;
    Raw8<DT> raw[ITEMS] = {};
#pragma unroll
    for (int t = 0; t < ITEMS; ++t)
        if (t * 32 < w.left) {
            const uint4* from = reinterpret_cast<const uint4*>(w.x + t * (32 * 8 * SIZE));
            raw[t].u[0] = __ldg(from);
            if constexpr (SIZE == 4) raw[t].u[1] = __ldg(from + 1);
        }
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
        float x[8];
        widen8<DT>(raw[t], x);
        float hi = max3_nan(max3_nan(x[0], x[1], x[2]), max3_nan(x[3], x[4], x[5]), max3_nan(x[6], x[7], x[7]));
        float lo = min3_nan(min3_nan(x[0], x[1], x[2]), min3_nan(x[3], x[4], x[5]), min3_nan(x[6], x[7], x[7]));
#pragma unroll
        for (int step = 1; step < 4; step <<= 1) {
            const float h = __shfl_xor_sync(~0u, hi, step), l = __shfl_xor_sync(~0u, lo, step);
            hi = max3_nan(hi, h, h);
            lo = min3_nan(lo, l, l);
        }
        float m = hi > -lo ? hi : lo;
        if (__any_sync(~0u, !(hi <= 3.402823466e38f) || !(lo >= -3.402823466e38f))) {
            bool bad = false;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(fabsf(x[i]) <= 3.402823466e38f)) { x[i] = 0.0f; bad = true; }
            if (bad) raise_status(a.status, DEV_INVALID);
            m = group_extreme(x);
        } else if (__any_sync(~0u, hi == -lo)) {
            m = group_extreme(x);
        }
        // 8 significant bits, so that n * d (up to 3 more) is exact in fp16
        float d = __bfloat162float(__float2bfloat16_rn(__fmul_rn(m, -0.125f)));
        d = fminf(fmaxf(d, -8160.0f), 8160.0f);
        uint16_t dh = __half_as_ushort(__float2half_rn(d));
        if ((dh & 0x7fffu) == 0) dh = 0;                           // a scale that rounds to zero has no sign
        d = h2f_bits(dh);
        const float r = d == 0.0f ? 0.0f : __frcp_rn(d);
        // floor(x r + 8.5) in [0, 15] in the low bits of the sum with 2^23, which
        // is 0x4b000000 + n: shifted together, the constants go at once.  Below
        // zero only a scale far from m / -8 leads (fp16's smallest, 8160).
        const bool far = __any_sync(~0u, fabsf(d) < 6.103515625e-05f || fabsf(d) == 8160.0f);
        uint32_t word = 0;
        constexpr uint32_t BIAS = 0x4b000000u;
        uint32_t bias = 0;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            const int f = 4 * (e >> 1);                            // values e and e + 1: fields f / 4 and f / 4 + 4
            float q0, q1, n0, n1;
            // (scalar products: a packed one would be contracted with the sum, whose ties then fall otherwise)
            unpack2(add2(pack2(__fmul_rn(x[e], r), __fmul_rn(x[e + 1], r)), pack2(8.5f, 8.5f)), q0, q1);
            if (far) {
                q0 = fmaxf(q0, 0.0f);
                q1 = fmaxf(q1, 0.0f);
            }
            unpack2(add2_rm(pack2(fminf(q0, 15.5f), fminf(q1, 15.5f)), pack2(8388608.0f, 8388608.0f)), n0, n1);
            word += (__float_as_uint(n0) << f) + (__float_as_uint(n1) << (f + 16));
            bias += (BIAS << f) + (BIAS << (f + 16));
        }
        word = (word - bias) ^ 0x88888888u;                        // n to two's complement
        if (t * 32 < w.left) {
            *reinterpret_cast<uint32_t*>(w.q + t * w.qstep) = word;
            if (holds_scale) *reinterpret_cast<uint16_t*>(w.s + t * w.sstep) = dh;
        }
    }
}

template <int DT, int ITEMS>
__global__ void __launch_bounds__(KVC_THREADS) kv_read_kernel(const KvcArgs a) {
    constexpr int SIZE = DT == TK_DT_F32 ? 4 : 2;
    pdl_trigger();
    pdl_wait();
    Where w;
    if (!where_is<SIZE>(a, ITEMS * 32, w)) return;
    uint32_t q[ITEMS];
    uint16_t d[ITEMS];
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
        q[t] = 0;
        d[t] = 0;
        if (t * 32 < w.left && w.ok) {
            q[t] = *reinterpret_cast<const uint32_t*>(w.q + t * w.qstep);
            d[t] = *reinterpret_cast<const uint16_t*>(w.s + t * w.sstep);
        }
    }
#pragma unroll
    for (int t = 0; t < ITEMS; ++t) {
        if (t * 32 >= w.left) break;
        uint32_t even[4], odds[4];                                 // values 0 1 | 2 3 | 4 5 | 6 7, exact in fp16
        kv_fields(q[t], __half2half2(__ushort_as_half(d[t])), even);
        uint4* to = reinterpret_cast<uint4*>(w.x + t * (32 * 8 * SIZE));
        if constexpr (DT == TK_DT_F16) {
            to[0] = make_uint4(even[0], even[1], even[2], even[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(as_half2(even[i]));
                if constexpr (DT == TK_DT_F32) {
                    even[i] = __float_as_uint(f.x);
                    odds[i] = __float_as_uint(f.y);
                } else {
                    even[i] = (uint32_t)f2bf_bits(f.x) | ((uint32_t)f2bf_bits(f.y) << 16);
                }
            }
            if constexpr (DT == TK_DT_F32) {
                to[0] = make_uint4(even[0], odds[0], even[1], odds[1]);
                to[1] = make_uint4(even[2], odds[2], even[3], odds[3]);
            } else {
                to[0] = make_uint4(even[0], even[1], even[2], even[3]);
            }
        }
    }
}

template <int ITEMS>
static cudaError_t go_kvc(const KvcArgs& a, int dtype, bool append, unsigned grid, cudaStream_t st) {
    void (*kern)(const KvcArgs);
    if (append)
        kern = dtype == TK_DT_F32   ? kv_append_kernel<TK_DT_F32, ITEMS>
               : dtype == TK_DT_F16 ? kv_append_kernel<TK_DT_F16, ITEMS>
                                    : kv_append_kernel<TK_DT_BF16, ITEMS>;
    else
        kern = dtype == TK_DT_F32   ? kv_read_kernel<TK_DT_F32, ITEMS>
               : dtype == TK_DT_F16 ? kv_read_kernel<TK_DT_F16, ITEMS>
                                    : kv_read_kernel<TK_DT_BF16, ITEMS>;
    return launch_dependent(kern, grid, KVC_THREADS, 0, st, a);
}

static tk_status launch_kvc(tk_ctx* ctx, const tk_kvcache& c, const tk_seqs& s, void* k, void* v, int dtype, long ldk,
                            long ldv, bool append, cudaStream_t st) {
    KvcArgs a;
    a.c = kv_view(c);
    a.s = seq_view(s);
    a.k = k; a.v = v;
    a.ldk = ldk; a.ldv = ldv;
    a.items = c.n_kv_heads * c.head_dim / 8;
    a.status = ctx->status;
    // few tokens: a warp for every 32 items; many: for 4 x 32, which finds its place once for all
    const bool many = (long)s.n_tokens * a.items > 32L * 32 * ctx->num_sms;
    a.chunks = (a.items + (many ? 127 : 31)) / (many ? 128 : 32);
    const long grid = (2L * s.n_tokens * a.chunks + KVC_THREADS / 32 - 1) / (KVC_THREADS / 32);
    if (grid * (KVC_THREADS / 32) > INT32_MAX) return fail(TK_ERR_INVALID, "tk_kv_append / tk_kv_read: too many values");
    ProfScope ps(ctx, st, PK_SERVE);
    const cudaError_t e = many ? go_kvc<4>(a, dtype, append, (unsigned)grid, st) : go_kvc<1>(a, dtype, append, (unsigned)grid, st);
    ctx->launches++;
    return cuda_fail(e, append ? "kv append launch" : "kv read launch");
}

tk_status launch_kv_append(tk_ctx* ctx, const tk_kvcache& c, const tk_seqs& s, const void* k, const void* v, int dtype,
                           long ldk, long ldv, cudaStream_t st) {
    return launch_kvc(ctx, c, s, const_cast<void*>(k), const_cast<void*>(v), dtype, ldk, ldv, true, st);
}
tk_status launch_kv_read(tk_ctx* ctx, const tk_kvcache& c, const tk_seqs& s, void* k, void* v, int dtype, long ldk,
                         long ldv, cudaStream_t st) {
    return launch_kvc(ctx, c, s, k, v, dtype, ldk, ldv, false, st);
}

}  // namespace tk
