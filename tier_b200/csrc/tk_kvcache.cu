// tk_kvcache.cu -- tk_kv_append and tk_kv_read: rounding keys and values to
// the 4-bit cache and expanding them again.
#include "tk_kv.cuh"

namespace tk {

constexpr int KVC_THREADS = 256;

template <int DT>
__device__ __forceinline__ void load8(const void* p, size_t at, float (&x)[8]) {
    if constexpr (DT == TK_DT_F32) {
        const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
        const float4 a = __ldg(f), b = __ldg(f + 1);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    } else {
        const uint4 u = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at));
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

template <int DT>
__device__ __forceinline__ void store8(void* p, size_t at, const float (&x)[8]) {
    if constexpr (DT == TK_DT_F32) {
        float4* f = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
        f[0] = make_float4(x[0], x[1], x[2], x[3]);
        f[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DT == TK_DT_BF16)
                w[i] = (uint32_t)f2bf_bits(x[2 * i]) | ((uint32_t)f2bf_bits(x[2 * i + 1]) << 16);
            else
                w[i] = (uint32_t)f2h_bits(x[2 * i]) | ((uint32_t)f2h_bits(x[2 * i + 1]) << 16);
        }
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// One item is 8 consecutive values of one token's k or v row; four lanes make
// a group of 32.  A token's items are its k row's, then its v row's.
struct KvcArgs {
    KvView c;
    SeqView s;
    void *k, *v;          // rows in (append) or out (read)
    long ldk, ldv;
    int items;            // per token: 2 * heads * dim / 8
    int* status;
};

struct Where {
    bool in_v, ok;
    size_t at;            // element in the k or v array
    size_t row;           // cache row
    int word;             // 32-bit word within it
};
__device__ __forceinline__ Where where_is(const KvcArgs& a, const int32_t* q_start, long idx) {
    Where w;
    const int r = (int)(idx / a.items);
    int i = (int)(idx - (long)r * a.items);
    const int half = a.items >> 1;
    w.in_v = i >= half;
    if (w.in_v) i -= half;
    w.at = (size_t)r * (w.in_v ? a.ldv : a.ldk) + (size_t)i * 8;
    const int per = a.c.dim >> 3, head = i / per;
    w.word = i - head * per;
    const int b = seq_of_row(q_start, a.s.n_seqs, r);
    const SeqInfo q = seq_info(a.s, a.c.page_shift, b, a.status);
    const int pos = q.kv - q.n_new + (r - q.row0);
    w.ok = r >= q.row0 && r - q.row0 < q.n_new && pos >= 0;
    w.row = w.ok ? kv_row(a.c, page_of(a.s, a.c, b, pos, a.status), head, pos) : 0;
    return w;
}

// Bound: memory (each value read once, half a byte and a sixteenth of a scale
// written).  Four lanes share a group so that every load is 16 or 32
// consecutive bytes a lane and a warp's stores fill whole 32-byte sectors.
template <int DT>
__global__ void __launch_bounds__(KVC_THREADS) kv_append_kernel(const KvcArgs a, long total) {
    const long idx = (long)blockIdx.x * KVC_THREADS + threadIdx.x;
    const bool live = idx < total;      // total is a multiple of 4: a group's lanes agree
    float x[8] = {};
    Where w{};
    if (live) {
        w = where_is(a, a.s.q_start, idx);
        load8<DT>(w.in_v ? a.v : a.k, w.at, x);
    }
    bool odd = false;
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (!(fabsf(x[i]) <= 3.402823466e38f)) { odd = true; x[i] = 0.0f; }
        if (fabsf(x[i]) > fabsf(m)) m = x[i];      // the first of several
    }
#pragma unroll
    for (int step = 1; step < 4; step <<= 1) {
        const float o = __shfl_xor_sync(~0u, m, step);
        const bool mine_first = ((threadIdx.x & step) == 0);
        if (fabsf(o) > fabsf(m) || (fabsf(o) == fabsf(m) && !mine_first)) m = o;
    }
    // 8 significant bits, so that n * d (up to 3 more) is exact in fp16
    float d = __bfloat162float(__float2bfloat16_rn(__fmul_rn(m, -0.125f)));
    d = fminf(fmaxf(d, -8160.0f), 8160.0f);
    uint16_t dh = f2h_bits(d);
    if ((dh & 0x7fffu) == 0) dh = 0;      // a scale that rounds to zero has no sign
    d = h2f_bits(dh);
    const float r = d == 0.0f ? 0.0f : __frcp_rn(d);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = fminf(fmaxf(floorf(__fadd_rn(__fmul_rn(x[e], r), 8.5f)), 0.0f), 15.0f);
        word |= (((uint32_t)(int)q ^ 8u) & 15u) << (4 * ((e >> 1) + 4 * (e & 1)));
    }
    if (!live) return;
    if (odd && w.ok) raise_status(a.status, DEV_INVALID);
    if (!w.ok) return;
    reinterpret_cast<uint32_t*>(w.in_v ? a.c.vq : a.c.kq)[w.row * (a.c.dim >> 3) + w.word] = word;
    if ((w.word & 3) == 0)
        reinterpret_cast<uint16_t*>(w.in_v ? a.c.vs : a.c.ks)[w.row * (a.c.dim >> 5) + (w.word >> 2)] = dh;
}

template <int DT>
__global__ void __launch_bounds__(KVC_THREADS) kv_read_kernel(const KvcArgs a, long total) {
    const long idx = (long)blockIdx.x * KVC_THREADS + threadIdx.x;
    if (idx >= total) return;
    const Where w = where_is(a, a.s.q_start, idx);
    float x[8] = {};
    if (w.ok) {
        const uint32_t q = reinterpret_cast<const uint32_t*>(w.in_v ? a.c.vq : a.c.kq)[w.row * (a.c.dim >> 3) + w.word];
        const float d = __half2float((w.in_v ? a.c.vs : a.c.ks)[w.row * (a.c.dim >> 5) + (w.word >> 2)]);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __fmul_rn((float)kv_nibble(q, e), d);
    }
    store8<DT>(w.in_v ? a.v : a.k, w.at, x);
}

static tk_status launch_kvc(tk_ctx* ctx, const tk_kvcache& c, const tk_seqs& s, void* k, void* v, int dtype, long ldk,
                            long ldv, bool append, cudaStream_t st) {
    KvcArgs a;
    a.c = kv_view(c);
    a.s = seq_view(s);
    a.k = k; a.v = v;
    a.ldk = ldk; a.ldv = ldv;
    a.items = 2 * c.n_kv_heads * c.head_dim / 8;
    a.status = ctx->status;
    const long total = (long)s.n_tokens * a.items;
    const long grid = (total + KVC_THREADS - 1) / KVC_THREADS;
    if (grid > INT32_MAX) return fail(TK_ERR_INVALID, "tk_kv_append / tk_kv_read: too many values");
    ProfScope ps(ctx, st, PK_SERVE);
    const dim3 g((unsigned)grid), t(KVC_THREADS);
    if (append) {
        if (dtype == TK_DT_F32) kv_append_kernel<TK_DT_F32><<<g, t, 0, st>>>(a, total);
        else if (dtype == TK_DT_F16) kv_append_kernel<TK_DT_F16><<<g, t, 0, st>>>(a, total);
        else kv_append_kernel<TK_DT_BF16><<<g, t, 0, st>>>(a, total);
    } else {
        if (dtype == TK_DT_F32) kv_read_kernel<TK_DT_F32><<<g, t, 0, st>>>(a, total);
        else if (dtype == TK_DT_F16) kv_read_kernel<TK_DT_F16><<<g, t, 0, st>>>(a, total);
        else kv_read_kernel<TK_DT_BF16><<<g, t, 0, st>>>(a, total);
    }
    ctx->launches++;
    return cuda_fail(cudaGetLastError(), append ? "kv append launch" : "kv read launch");
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
