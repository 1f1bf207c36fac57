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

template <int D>
static void go_rows(const KvaArgs& a, int dtype, unsigned grid, cudaStream_t st) {
    if (dtype == TK_DT_F32) kv_attend_rows_kernel<D, TK_DT_F32><<<grid, 128, 0, st>>>(a);
    else if (dtype == TK_DT_F16) kv_attend_rows_kernel<D, TK_DT_F16><<<grid, 128, 0, st>>>(a);
    else kv_attend_rows_kernel<D, TK_DT_BF16><<<grid, 128, 0, st>>>(a);
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
    ProfScope ps(ctx, st, PK_SERVE);
    if (c.head_dim == 64) go_rows<64>(a, dtype, (unsigned)grid, st);
    else go_rows<128>(a, dtype, (unsigned)grid, st);
    ctx->launches++;
    return cuda_fail(cudaGetLastError(), "kv attend launch");
}

}  // namespace tk
