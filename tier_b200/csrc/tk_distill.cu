// tk_distill.cu -- tk_distill, tk_distill_grad: distillation from a teacher's
// top logits.
//
// loss = sum q (ln q - ln p), of which sum q ln q and sum q l need the listed
// places alone and ln S a reading of the row; the gradient (w / T) (p - q) is
// dense but for q, which a second write puts in at the listed places.
//
// Loss and gradient in one call read the row from memory once and write the
// gradient once; the row's second reading is served on the chip.  The bound is
// memory; what keeps the call from it is the second reading (without it 331 us
// where the call took 409, before a batch was held), blocks that meet between the
// passes, and two exponentials a logit (without them 50 of 753 us, 100 where
// long runs lower the clock).  Tried and slower: blocks that stay and take rows in
// turn (498 to 604 us where this took 425: all read, meet and write at the same
// time), both passes as tasks of a queue, gradients some rows behind the sums
// (485: the rows between them pass the L2), a part's whole length in shared
// memory (no room in the L1 for loads on their way: 506 and more), 512 or 1024
// threads a block (427, 426).
//
// Measured (us; calls in a graph, and from Python on machines that were
// idle before): 4096 x 262144 bf16 750 to 775, 751 to 828 (5.1 TB/s of floor bytes at
// the most), 512 x 262144 fp32 to bf16 135 to 144, 145, 16 x 50257 fp16 7.8, 9.7;
// the loss of 300 x 131072 fp32 29.7, 30; the gradient alone 2048 x 262144 bf16
// 317 (6.8 TB/s), 320.
#include <type_traits>
#include "tk_rows.cuh"

namespace tk {

constexpr int DS_CLUSTER = 8;         // blocks of a row at most

struct DsArgs {
    RowArgs r;
    int k;
    const int32_t* ids;
    const float *teacher, *weight;
    float *loss, *rmax, *rsum;
    const float *in_max, *in_sum;     // tk_distill_grad: of the forward pass
    int parts;                        // blocks of a row
};

// The teacher's row in shared memory: an entry's place (-1: it does not
// count), logit and q = softmax(t / T); the row's own logits there; maximum and
// sum of the teacher's softmax.  state 0: no entry counts, 1: some do, 2: NaN or
// +inf among them.
struct DsTeacher {
    __align__(16) int ids[TK_TOP_MAX];
    float t[TK_TOP_MAX], q[TK_TOP_MAX], x[TK_TOP_MAX];
    float m, s;
    int state;
};
// One warp's registers: entries lane, lane + 32, ...
struct DsEntries {
    static constexpr int EACH = TK_TOP_MAX / 32;
    int id[EACH];
    float t[EACH];
    __device__ __forceinline__ void load(const DsArgs& a, size_t row) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const bool in = 32 * i + lane < a.k;
            id[i] = in ? a.ids[row * a.k + 32 * i + lane] : -1;
            t[i] = in ? a.teacher[row * a.k + 32 * i + lane] : 0.0f;
        }
    }
    __device__ __forceinline__ void softmax(DsTeacher& s, const DsArgs& a, bool report) {
        const int lane = threadIdx.x & 31;
        float m = RW_LOWEST, sum = 0.0f;
        bool some = false, bad = false, beyond = false;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            beyond |= id[i] >= a.r.vocab;
            if (id[i] < 0 || id[i] >= a.r.vocab || t[i] == -INFINITY) {
                id[i] = -1;
                t[i] = -INFINITY;
            }
            some |= id[i] >= 0;
            bad |= !(t[i] < INFINITY);
            m = fmaxf(m, t[i]);
        }
        for (int i = 16; i; i >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, i));
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (32 * i >= a.k) break;
            s.ids[32 * i + lane] = id[i];
            s.t[32 * i + lane] = t[i];
            t[i] = rw_exp2((t[i] - m) * a.r.c);
            sum += t[i];
        }
        for (int i = 16; i; i >>= 1) sum += __shfl_xor_sync(~0u, sum, i);
        const float r = 1.0f / sum;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (32 * i >= a.k) break;
            asm("mul.ftz.f32 %0, %1, %2;" : "=f"(s.q[32 * i + lane]) : "f"(t[i]), "f"(r));   // (below 2^-126: 0)
        }
        some = __any_sync(~0u, some);
        bad = __any_sync(~0u, bad);
        if (report && beyond) raise_status(a.r.status, DEV_INVALID);
        if (lane == 0) {
            s.m = m;
            s.s = sum;
            s.state = bad ? 2 : some;
        }
    }
};

// n sums brought together, in every lane of a warp.
template <class F>
__device__ __forceinline__ RwStat ds_join(F from, int n, float c) {
    RwStat st{RW_LOWEST, 0.0, 0.0};
    for (int i = threadIdx.x & 31; i < n; i += 32) {
        const RwStat o = from(i);
        const float m = fmaxf(st.m, o.m);
        st = RwStat{m, rw_to_max(st, m, c).s + rw_to_max(o, m, c).s, 0.0};
    }
    return rw_warp_join<false>(st, c);
}
// One warp: the row's loss, maximum and sum.
__device__ __forceinline__ void ds_loss(const DsTeacher& t, const DsArgs& a, size_t row, const RwStat& st) {
    const int lane = threadIdx.x & 31;
    const bool bad = st.s != st.s;
    double sum = 0.0, qs = 0.0;                    // (q adds up to 1 but for its roundings)
    for (int i = lane; i < a.k; i += 32) {
        const float q = t.q[i];
        if (q > 0.0f) sum += q * ((((double)t.t[i] - t.m) - ((double)t.x[i] - st.m)) * a.r.inv_t);
        qs += q;
    }
    for (int i = 16; i; i >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, i);
        qs += __shfl_xor_sync(~0u, qs, i);
    }
    if (lane == 0) {
        if (bad) raise_status(a.r.status, DEV_INVALID);
        if (a.loss) a.loss[row] = (float)(sum + qs * (log(st.s) - log((double)t.s)));
        if (a.rmax) a.rmax[row] = bad ? NAN : st.m;
        if (a.rsum) a.rsum[row] = (float)st.s;
    }
}

// A thread's first batch stays in shared memory between the passes: its own
// units, which no other thread reads (16 bytes of a warp's threads side by
// side).  More of them would not help: 6 units instead of 4 left the L1 too
// little room for the loads on their way (384 -> 437 us; 1 unit 413, 2 398).
struct DsHeld {
    uint4 part[RW_BATCH][2][RW_THREADS];
    template <class XT>
    __device__ __forceinline__ void hold(const RwUnit<XT> (&u)[RW_BATCH]) {
#pragma unroll
        for (int j = 0; j < RW_BATCH; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                part[j][h][threadIdx.x] = make_uint4(u[j].w[4 * h], u[j].w[4 * h + 1], u[j].w[4 * h + 2], u[j].w[4 * h + 3]);
    }
    template <class XT>
    __device__ __forceinline__ void take(RwUnit<XT>& u, int j) const {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 q = part[j][h][threadIdx.x];
            u.w[4 * h] = q.x;
            u.w[4 * h + 1] = q.y;
            u.w[4 * h + 2] = q.z;
            u.w[4 * h + 3] = q.w;
        }
    }
};

// A cluster of blocks per row, each with one part of it: the sums of the
// softmax over one reading, the blocks' sums brought together in shared memory;
// then the gradient over a second, which has the first batch in shared memory
// and the last one in registers and finds the others in the L2.
template <class XT, class DT>
__global__ void __launch_bounds__(RW_THREADS, 4) ds_kernel(const DsArgs a) {
    constexpr bool GRAD = !std::is_same<DT, void>::value;
    constexpr int STEP = RW_THREADS * RW_BATCH;
    __shared__ typename std::conditional<GRAD, DsHeld, int>::type held;
    __shared__ DsTeacher t;
    __shared__ RwStat join[DS_CLUSTER * RW_WARPS];
    pdl_wait();
    const size_t row = blockIdx.x / a.parts;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, vocab = a.r.vocab, rank = blockIdx.x % a.parts;
    const float c = a.r.c;
    const XT* x = static_cast<const XT*>(a.r.x) + row * a.r.ldx;
    const RwPart<XT> p(x, vocab, rank, a.parts);
    const RwEnds<XT> e(x, vocab);
    const bool ends = rank == a.parts - 1, end = ends && tid < e.n;
    const float weight = a.weight ? a.weight[row] : 1.0f;
    const f32x2 c2 = pack2(c, c);
    RwSums<false> sums;
    RwUnit<XT> u[RW_BATCH];
    const auto add = [&]() {
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < RW_BATCH; ++j) top = fmaxf(top, fmaxf(u[j].max(0), u[j].max(1)));
        if (top > sums.m) sums.raise(top, c);
        sums.batch(u, c2);
    };
    // the first batch and the teacher's row together
    rw_batch<XT>(u, p, 0);
    if (warp == RW_WARPS - 1) {
        DsEntries entries;
        entries.load(a, row);
        entries.softmax(t, a, rank == 0);
    }
    add();
    __syncthreads();
    const int state = t.state;
    if (state == 0) {                              // the whole cluster alike
        if (rank == 0 && tid == 0) {
            if (a.loss) a.loss[row] = 0.0f;
            if (a.rmax) a.rmax[row] = 0.0f;
            if (a.rsum) a.rsum[row] = 0.0f;
        }
        if constexpr (GRAD) rw_zero(static_cast<DT*>(a.r.dx) + row * a.r.ldd, vocab, rank, a.parts);
        return;
    }
    if (a.parts > 1) cluster_arrive();
    // logits at single places: before any gradient is written
    const int entry = RW_THREADS - 1 - tid, id = entry < a.k ? t.ids[entry] : -1;    // (the first warp has the loss)
    const float listed = id >= 0 ? rw_float(x[id]) : 0.0f;
    const float v_end = end ? rw_float(x[e.place(tid)]) : -INFINITY;
    int u0 = 0, batch = 1;
    while (u0 + STEP < p.n) {
        if constexpr (GRAD)
            if (u0 == 0) held.hold(u);
        u0 += STEP;
        rw_batch<XT>(u, p, u0);
        if (batch++ % RW_FLUSH == 0) sums.flush(c);      // (while the loads are on their way)
        add();
    }
    if (a.r.few) pdl_trigger();
    if (entry < a.k) t.x[entry] = listed;
    sums.single(v_end, c);
    sums.flush(c);
    // every block gets all warps' sums
    const RwStat w = rw_warp_join<false>(RwStat{sums.M, sums.S, 0.0}, c);
    if (a.parts > 1) {
        cluster_wait();                            // (all have begun)
        if (lane < a.parts) *rw_peer(&join[rank * RW_WARPS + warp], lane) = w;
        cluster_sync();
    } else {
        if (lane == 0) join[warp] = w;
        __syncthreads();
    }
    RwStat st = ds_join([&](int i) { return join[i]; }, a.parts * RW_WARPS, c);
    if (st.s == 0.0 || state == 2) st.s = (double)NAN;      // nothing above -inf
    if (rank == 0 && warp == 0) ds_loss(t, a, row, st);
    if constexpr (GRAD) {
        DT* dx = static_cast<DT*>(a.r.dx) + row * a.r.ldd;
        const float wt = weight * a.r.inv_t;
        if (wt == 0.0f) {
            rw_zero(dx, vocab, rank, a.parts);
            return;
        }
        const RwDense<false> dense{st.m, c, wt / (float)st.s, 0.0f};
        DT* d = dx + p.first;
        if (rw_alike<XT>(d)) {
            rw_write<XT>(u, d, p, u0, dense);
            const bool first = u0 > 0;             // there is a held batch
            u0 -= STEP;
            if (u0 > 0) rw_batch<XT>(u, p, u0);
            const auto write_held = [&]() {
#pragma unroll 2
                for (int j = 0; j < RW_BATCH; ++j) {
                    RwUnit<XT> w[1];
                    held.take(w[0], j);
                    rw_write<XT>(w, d, p, j * RW_THREADS, dense);
                }
            };
            // fp32 rows: while the others are on their way (512 x 262144 to bf16 151 ->
            // 144 us; 16-bit rows, whose conversions need the registers, 2048 x 262144
            // 385 -> 392)
            constexpr bool early = sizeof(XT) == 4;
            if (early && first) write_held();
            for (; u0 > 0; u0 -= STEP) {
                rw_write<XT>(u, d, p, u0, dense);
                if (u0 > STEP) rw_batch<XT>(u, p, u0 - STEP);
            }
            if (!early && first) write_held();
        } else
            rw_write_other<XT>(d, p, dense);
        if (end) dx[e.place(tid)] = rw_to<DT>(dense.one(v_end));
        const RwListed l = rw_listed(p, e, ends, t.ids, t.q, a.k, entry);
        __syncthreads();
        if (l.mine) dx[l.id] = rw_to<DT>(dense.one(listed) - wt * l.share);
    }
}

// The gradient alone: one pass.
template <class XT, class DT>
__global__ void __launch_bounds__(RW_THREADS, 4) dg_kernel(const DsArgs a) {
    __shared__ DsTeacher t;
    if (a.r.few) pdl_trigger();
    pdl_wait();
    const size_t row = blockIdx.x / a.parts;
    const int tid = threadIdx.x, vocab = a.r.vocab, rank = blockIdx.x % a.parts;
    const XT* x = static_cast<const XT*>(a.r.x) + row * a.r.ldx;
    DT* dx = static_cast<DT*>(a.r.dx) + row * a.r.ldd;
    const float wt = (a.weight ? a.weight[row] : 1.0f) * a.r.inv_t, m = a.in_max[row], s = a.in_sum[row];
    if (tid < 32) {
        DsEntries entries;
        entries.load(a, row);
        entries.softmax(t, a, rank == 0);
    }
    __syncthreads();
    const int state = t.state;
    if (rank == 0 && tid == 0 && (state == 2 || (state == 1 && wt != 0.0f && s != s))) raise_status(a.r.status, DEV_INVALID);
    if (state == 0 || wt == 0.0f) {
        rw_zero(dx, vocab, rank, a.parts);
        return;
    }
    rw_gradient<XT, DT, false>(x, dx, vocab, RwPart<XT>(x, vocab, rank, a.parts), rank == a.parts - 1, t.ids, t.q, a.k, wt,
                               RwDense<false>{m, a.r.c, state == 2 ? NAN : wt / s, 0.0f});
}

// Blocks of a row: enough for few rows (of 8192 logits each at least); with a
// gradient, one for every 128 KB of it: two batches of a block are then read
// again, and the 148 rows that four blocks an SM hold of 512 KB each stay in the
// L2.  us by blocks a row 1, 2, 4, 8: 2048 rows of 512 KB (bf16) 470, 440, 384,
// 433; 512 of 1 MB (fp32) 207, 196, 177, 150; 300 of 256 KB 41.6, 39.7, 41.6,
// 46.7; 1024 of 64 KB 31, 37, 59, 109; few: 100 of 50257 fp32 13.7, 13.3, 10.9, 15.8.
static int ds_parts(const tk_ctx* ctx, int n_rows, int vocab, long row_bytes, bool grad) {
    int parts = 1;
    while (parts < DS_CLUSTER && vocab / (2 * parts) >= 8192 &&
           (2L * n_rows * parts <= 4L * ctx->num_sms || (grad && row_bytes / parts > 128 << 10)))
        parts *= 2;
    return parts;
}
template <class XT, class DT>
static cudaError_t launch_ds(const tk_ctx* ctx, DsArgs& a, cudaStream_t s) {
    a.parts = ds_parts(ctx, a.r.n_rows, a.r.vocab, (long)a.r.vocab * sizeof(XT), !std::is_same<DT, void>::value);
    a.r.few = rw_few(ctx, a.r.n_rows, a.parts);
    return rw_launch(ds_kernel<XT, DT>, a.r.n_rows, a.parts, true, 0, a, s);
}
tk_status launch_distill(tk_ctx* ctx, const RowArgs& r, int x_dtype, int k, const int32_t* ids, const float* teacher,
                         const float* weight, float* loss, float* rmax, float* rsum, int d_dtype, cudaStream_t s) {
    DsArgs a{r, k, ids, teacher, weight, loss, rmax, rsum, nullptr, nullptr, 1};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    const cudaError_t e = r.dx ? rw_types(x_dtype, d_dtype, [&](auto x, auto d) { return launch_ds<decltype(x), decltype(d)>(ctx, a, s); })
                        : x_dtype == TK_DT_F32 ? launch_ds<float, void>(ctx, a, s)
                        : x_dtype == TK_DT_F16 ? launch_ds<__half, void>(ctx, a, s) : launch_ds<__nv_bfloat16, void>(ctx, a, s);
    return cuda_fail(e, "distillation launch");
}
tk_status launch_distill_grad(tk_ctx* ctx, const RowArgs& r, int x_dtype, int k, const int32_t* ids, const float* teacher,
                              const float* rmax, const float* rsum, const float* weight, int d_dtype, cudaStream_t s) {
    DsArgs a{r, k, ids, teacher, weight, nullptr, nullptr, nullptr, rmax, rsum, 1};
    ProfScope ps(ctx, s, PK_LMHEAD);
    ctx->launches += 1;
    return cuda_fail(rw_types(x_dtype, d_dtype, [&](auto x, auto d) {
        a.parts = rw_grad_parts<decltype(x)>(ctx, a.r.n_rows, a.r.vocab);
        a.r.few = rw_few(ctx, a.r.n_rows, a.parts);
        return rw_launch(dg_kernel<decltype(x), decltype(d)>, a.r.n_rows, a.parts, false, 0, a, s);
    }), "distillation gradient launch");
}

}  // namespace tk
