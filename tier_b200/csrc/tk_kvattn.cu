// tk_kvattn.cu -- tk_kv_attend: attention of new tokens over the 4-bit cache;
// the streaming kernel for few rows (many: tk_kvattn_tc.cu).
#include "tk_kv.cuh"

namespace tk {

// The last of a head's parts to finish joins them (the result does not depend
// on which block that is).  The counter is left at zero for the next call.
template <int D, int DT, int ROWS, class Item>
__device__ __forceinline__ void kv_join_last(const KvaArgs& a, const Item& it, int live, uint8_t* smem, int bytes,
                                             int* sh_last) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        int* n = a.count + it.c0;                                  // no other head in parts begins in that block
        const int done = atomicAdd(n, 1) + 1;
        *sh_last = done == it.chunks;
        if (done == it.chunks) *n = 0;
    }
    __syncthreads();
    if (!*sh_last) return;
    __threadfence();
    kv_join<D, DT, ROWS>(
        a, it.chunks, live, threadIdx.x, blockDim.x, smem, bytes,
        [&](int c) { return a.part + (size_t)(2 * (it.c0 + c) + (c == 0 ? it.odd : 0)) * (ROWS * (D + 2)); },
        [&](int r) { return KvaRow{it.row0 + r / a.group, it.head * a.group + r % a.group}; }, [] { __syncthreads(); });
}

// ---------------------------------------------------------------------------
// Few rows per key/value head (new tokens x heads of the group <= 32): the
// cache is streamed once, divided among thread blocks.
//
// One warp takes units of 32 keys.  S^T = K Q^T and O^T += V^T P^T are
// m16n8k16 fp16 products with the keys, or the values of a head, as the 16
// matrix rows and the query rows as the 8 columns (NT sets of 8): what the
// cache holds is read and turned to fp16 once, and 8 query rows cost 32
// registers of O.  fp32 rows enter as hi and lo fp16 parts (two products), so
// that q and p keep 22 bits.  The order of a reduction index is free, so lane
// (g, t) = (lane / 4, lane % 4) uses what it can load in one piece: of K the
// t-th quarter of a key's row (16 bytes at head_dim 128), of V the g-th eighth
// of two rows of each 8 keys.  A key's scale multiplies its fp16
// numbers exactly.  P^T's fragments are S^T's turned by movmatrix.
//
// The softmax keeps a reference per row that moves only when a unit's largest
// weight would near fp16's largest (KvRef): the rescaling of O is rare, and otherwise
// no lane needs another's maximum.  l is summed per lane in fp32 and joined at
// the end.
//
// Rows are copied by 16-byte cp.async into each warp's own ring (no barrier
// between warps), as far ahead as the ring is deep: nine instructions a unit,
// where bulk copies of the four pieces cost about a hundred in addresses and
// barrier handling.  The keys' order within 8 (kd_key) and an exchange of
// half rows of V keep the fragment loads free of bank conflicts.
//
// Bound: long caches by the instructions that turn 4 bits into fp16 fragments,
// not by memory; few rows by the chain of one unit after another and the join.
// Measured (32 query heads, 8 key/value heads of 128; us, TB/s of cache read):
// one fp16 row at 4097 keys 10.8, 0.44; 32 bf16 rows at up to 16300 each 58.7,
// 3.3; one fp32 row at 131071 54.9, 2.8; 8 sequences of 5 fp32 rows at 8191
// 69.3, 1.1 (three column sets of two parts, 8 warps an SM: six products where
// a bf16 row has one, and few warps to hide their latency).
// ---------------------------------------------------------------------------
constexpr int KD_WARPS = 4, KD_STAGES = 3, KD_UNIT = 32, KD_MAX_ROWS = 32;
// Blocks an SM: registers for 8 or 16 query rows allow three, for 24 or 32 two.
constexpr int kd_blocks(int nt) { return nt <= 2 ? 3 : 2; }
static_assert(kd_blocks(1) < KV_SYNC_PER_SM, "a counter a block behind the flags");

template <int D, int NT>
struct KdGeo {
    static constexpr int QB = KD_UNIT * D / 2, SB = KD_UNIT * D / 16;      // bytes of numbers, of scales
    static constexpr int STAGE = 2 * QB + 2 * SB;
    static constexpr int RING = KD_WARPS * KD_STAGES * STAGE;
    static constexpr int JOIN = KD_WARPS * 8 * NT * ((D + 4) * 4 + 8);     // each warp's O rows, m and l
    static constexpr int SMEM = RING > JOIN ? RING : JOIN;
    static constexpr int PART = 8 * NT * (D + 2);                          // floats of a part: O, then (m, l) of each row
};

// How the units of all sequences and key/value heads are divided among the
// blocks, all of which are resident at once; each block works it out from the
// lengths on the device.  With `per` the equal share of a block:
//   whole parts: every head is cut into ceil(units / p) even parts, one a
//     block, for the smallest p of per, 1.03 per and 1.07 per that leaves no
//     more parts than blocks.  A short batch (p = `least`) is always cut the
//     same way, whatever else it holds.
//   runs: otherwise (many heads of very different length) the units, one head
//     after the other, are cut into equal runs; a run may end one head and
//     begin others.
// A head that lies in several blocks is joined by the last to finish its part.
struct KdSeq {
    int kv, n_new, row0, lo, units;        // keys [lo, kv) are seen by some row
};
struct KdPlan {
    uint32_t total, per;                   // units, or parts with `whole`; per block with runs; units of a part else
    bool whole;
    KdSeq mine;                            // lane's sequence, if there are at most 32
};
struct KdItem {
    int b, head, kv, n_new, row0, lo;
    int u0, u1;                            // units [u0, u1) of the sequence are this block's
    int chunks, slot, c0, odd;             // parts of the head; place of this one; part 0's place is 2 c0 + odd, c's 2 (c0 + c)
};
__device__ __forceinline__ KdSeq kd_seq(const KvaArgs& a, int b, int* status) {
    KdSeq s{0, 0, 0, 0, 0};
    if (b >= a.s.n_seqs) return s;
    const SeqInfo q = seq_info(a.s, a.c.page_shift, b, status);
    if (q.n_new == 0) return s;
    s.kv = q.kv; s.n_new = q.n_new; s.row0 = q.row0;
    s.lo = kv_first_key(q.kv - q.n_new, a.window);
    // no key at all: one unit without keys, whose result is zero
    s.units = max((q.kv + KD_UNIT - 1) / KD_UNIT - s.lo / KD_UNIT, 1);
    return s;
}
// (the host bounds all units by 2^31)
__device__ __forceinline__ KdPlan kd_plan(const KvaArgs& a, uint32_t least) {
    const int lane = threadIdx.x & 31;
    KdPlan p;
    uint32_t total = 0;
    for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
        p.mine = kd_seq(a, b0 + lane, a.status);
        total += __reduce_add_sync(~0u, p.mine.units);
    }
    p.total = total * a.c.heads;
    p.whole = false;
    p.per = max((p.total + gridDim.x - 1) / gridDim.x, least);
    const uint32_t room = gridDim.x / a.c.heads;                   // parts that a head may have, over all sequences
#pragma unroll 1
    for (int k = 0; k < 3; ++k) {
        const uint32_t tried = p.per + (k * p.per + 29) / 30;
        uint32_t parts = 0;
        for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
            const int n = a.s.n_seqs > 32 ? kd_seq(a, b0 + lane, nullptr).units : p.mine.units;
            parts += __reduce_add_sync(~0u, (n + tried - 1) / tried);
        }
        if (parts <= room) {
            p.per = tried;
            p.whole = true;
            p.total = parts * a.c.heads;
            break;
        }
    }
    return p;
}
// The sequence and head of unit (with whole parts: part) x, and what of it lies before `end`.
__device__ __forceinline__ void kd_find(const KvaArgs& a, const KdPlan& plan, uint32_t x, uint32_t end, KdItem& it) {
    const int lane = threadIdx.x & 31;
    uint32_t before = 0;
    for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
        const KdSeq q = a.s.n_seqs > 32 ? kd_seq(a, b0 + lane, nullptr) : plan.mine;
        const uint32_t each = plan.whole ? (q.units + plan.per - 1) / plan.per : q.units, mine = each * a.c.heads;
        uint32_t sum = mine;               // units or parts up to and with this lane's sequence
        if (a.s.n_seqs > 1)
            for (int i = 1; i < 32; i <<= 1) {
                const uint32_t o = __shfl_up_sync(~0u, sum, i);
                if (lane >= i) sum += o;
            }
        const unsigned hit = __ballot_sync(~0u, x < before + sum);
        if (hit) {
            const int src = __ffs(hit) - 1;
            it.b = b0 + src;
            it.kv = __shfl_sync(~0u, q.kv, src);
            it.n_new = __shfl_sync(~0u, q.n_new, src);
            it.row0 = __shfl_sync(~0u, q.row0, src);
            it.lo = __shfl_sync(~0u, q.lo, src);
            const uint32_t n = __shfl_sync(~0u, q.units, src), count = __shfl_sync(~0u, each, src);
            const uint32_t at = x - before - __shfl_sync(~0u, sum - mine, src);
            it.head = at / count;
            const uint32_t off = at - it.head * count;
            const int u = it.lo / KD_UNIT;
            if (plan.whole) {
                // ceil(n / count) or one less units a part
                const uint32_t big = (n + count - 1) / count, cut = n - (big - 1) * count;
                it.u0 = u + off * big - (off > cut ? off - cut : 0);
                it.u1 = it.u0 + big - (off >= cut);
                it.chunks = count;
                it.c0 = blockIdx.x - off;
                it.odd = 0;
                it.slot = 2 * blockIdx.x;
            } else {
                // a block has one part of a head begun before it at most, and one of a head that goes on behind it
                const uint32_t h0 = x - off, h1 = h0 + n;
                it.u0 = u + off;
                it.u1 = u + (min(h1, end) - h0);
                it.c0 = h0 / plan.per;
                it.chunks = (h1 - 1) / plan.per - it.c0 + 1;
                it.odd = 1;
                it.slot = 2 * blockIdx.x + (off == 0);
            }
            return;
        }
        before += __shfl_sync(~0u, sum, 31);
    }
}

// Key of matrix index i within its 8: 0 5 2 7 1 4 3 6.  Neighbours (one fp16
// pair of P^T, two rows of K) differ in parity, so that 64-byte rows fall on
// different banks; the even and the odd four are distinct modulo 4.
__device__ __forceinline__ int kd_key(int i) {
    const int b = ((i & 2) | ((i >> 2) & 1));
    return (i & 1) ? 4 + (b ^ 1) : b;
}

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 8 x 8 fp16 matrix, row lane / 4, columns 2 (lane % 4), + 1: transposed.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
template <int D, int DT, int NT>
__global__ void __launch_bounds__(KD_WARPS * 32, kd_blocks(NT)) kv_decode_kernel(const KvaArgs a, uint32_t least) {
    using G = KdGeo<D, NT>;
    constexpr bool SPLIT = DT == TK_DT_F32;
    constexpr int ROWS = 8 * NT, PARTS = SPLIT ? 2 : 1;            // query rows, fp16 parts of q and p
    constexpr int KW = D / 32, VW = D / 64;                        // 32-bit words of a lane's piece of a key / value row
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr bool QREG = NT == 1;                                 // q's fragments stay in registers
    __shared__ uint4 qsm[NT][PARTS][QREG ? 1 : KW][32];            // or, as the fragments of a word's two steps, here
    __shared__ int sh_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int kg = kd_key(g), k0 = kd_key(2 * t), k1 = kd_key(2 * t + 1);
    pdl_trigger();
    pdl_wait();
    const KdPlan plan = kd_plan(a, least);
    uint32_t x = plan.whole ? blockIdx.x : blockIdx.x * plan.per;
    const uint32_t end = min(x + (plan.whole ? 1 : plan.per), plan.total);
    uint8_t* ring = smem + warp * (KD_STAGES * G::STAGE);

  for (; x < end; ) {
    KdItem it;
    kd_find(a, plan, x, end, it);
    x += plan.whole ? 1 : it.u1 - it.u0;
    // ---- rows: row r of the block is token r / group, head r % group; lane (g, t) loads the t-th quarter of row
    // g (before the copies below queue up in front of it) and keeps the statistics of rows 2 t and 2 t + 1 ----
    const int rows = it.n_new * a.group, pos0 = it.kv - it.n_new;
    float x0[NT][KW][8];
    int lim[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int r = g + 8 * n;
        lim[n] = INT32_MAX;
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
            for (int e = 0; e < 8; ++e) x0[n][w][e] = 0.0f;
        if (r < rows) {
            const int tok = r / a.group;
            lim[n] = max(pos0 + tok + 1, 0);
            const size_t at = (size_t)(it.row0 + tok) * a.ldq + (size_t)(it.head * a.group + r % a.group) * D + t * (D / 4);
#pragma unroll
            for (int w = 0; w < KW; ++w) load_pairs8<DT>(a.q, at + w * 8, x0[n][w]);
        }
    }

    // ---- the warp's units: u0 + warp, + 4, ... ----
    const int mine = it.u1 - it.u0 > warp && it.kv > 0 ? (it.u1 - it.u0 - warp + KD_WARPS - 1) / KD_WARPS : 0;
    const int page_mask = (1 << a.c.page_shift) - 1;
    const long head_rows = (long)it.head << a.c.page_shift, page_rows = (long)a.c.heads << a.c.page_shift;
    const bool small = a.c.page_shift < 5;                         // 16-token pages: two a unit
    constexpr int HALF = G::QB / 1024;                             // copies of 512 bytes in 16 rows
    const uint8_t* kp = a.c.kq + lane * 16;
    const uint8_t* vp = a.c.vq + lane * 16;
    constexpr int SL = G::SB / 16;                                 // lanes that copy one plane's scales
    const uint8_t* sp = reinterpret_cast<const uint8_t*>(lane < SL ? a.c.ks : a.c.vs) + (lane % SL) * 16;
    const uint32_t to0 = smem_u32(ring) + lane * 16, tov = to0 ^ (D == 128 ? (lane & 8) << 2 : 0);
    int pid = 0, pid2 = 0;
    auto issue = [&](int i, int stage) {
        if (i < mine) {
            const int pos = (it.u0 + warp + i * KD_WARPS) * KD_UNIT;
            if ((i & 31) == 0) {                                   // page ids of the next 32 units, one a lane
                const int p = pos + lane * (KD_WARPS * KD_UNIT);
                if (i + lane < mine) {                             // (of two pages the first may lie before every window)
                    pid = small && p + 16 <= it.lo ? 0 : page_of(a.s, a.c, it.b, p, a.status);
                    if (small && p + 16 < it.kv) pid2 = page_of(a.s, a.c, it.b, p + 16, a.status);
                }
            }
            long row = __shfl_sync(~0u, pid, i & 31) * page_rows + head_rows + (pos & page_mask), row2 = row + 16;
            const int last = it.kv - pos > 16 ? 32 : 16;           // whole 16-row pieces: inside the page
            if (small) row2 = __shfl_sync(~0u, pid2, i & 31) * page_rows + head_rows;
            const uint32_t st = stage * G::STAGE;
#pragma unroll
            for (int c = 0; c < HALF; ++c) {
                cp_async16(to0 + st + c * 512, kp + row * (D / 2) + c * 512);
                cp_async16(tov + st + G::QB + c * 512, vp + row * (D / 2) + c * 512);
            }
            if (last == 32)
#pragma unroll
                for (int c = 0; c < HALF; ++c) {
                    cp_async16(to0 + st + (HALF + c) * 512, kp + row2 * (D / 2) + c * 512);
                    cp_async16(tov + st + G::QB + (HALF + c) * 512, vp + row2 * (D / 2) + c * 512);
                }
            const bool second = (lane % SL) * 16 >= 16 * (D / 16);
            if (lane < 2 * SL && (!second || last == 32))
                cp_async16(to0 + st + 2 * G::QB, sp + (second && small ? row2 - 16 : row) * (D / 16));
        }
        cp_async_commit();
    };
    for (int i = 0; i < KD_STAGES - 1; ++i) issue(i, i);

    uint4 qr[PARTS][KW];
    float sc[NT][2];
    int limit[NT][2], from[NT][2];                                 // keys [from, limit) are seen
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float mx = 0.0f;
#pragma unroll
        for (int w = 0; w < KW; ++w)
#pragma unroll
            for (int e = 0; e < 8; ++e) mx = fmaxf(mx, fabsf(x0[n][w][e]));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 2));
        float back;
        const float up = copysignf(q_unit(mx, back), a.scale2);
        back *= fabsf(a.scale2);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            sc[n][c] = __shfl_sync(~0u, back, 4 * (2 * t + c));
            limit[n][c] = __shfl_sync(~0u, lim[n], 4 * (2 * t + c));
            from[n][c] = a.window > 0 && limit[n][c] != INT32_MAX ? max(limit[n][c] - a.window, 0) : 0;
        }
#pragma unroll
        for (int w = 0; w < KW; ++w) {
            if (!QREG && warp != w % KD_WARPS) continue;           // each warp lays out its share
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const float u = x0[n][w][2 * p] * up, v = x0[n][w][2 * p + 1] * up;
                hi[p] = pack_half2(u, v);
                const __half2 hh = as_half2(hi[p]);
                lo[p] = pack_half2(u - __low2float(hh), v - __high2float(hh));
            }
            uint4& to = QREG ? qr[0][w] : qsm[n][0][QREG ? 0 : w][lane];
            to = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (SPLIT) {
                uint4& to2 = QREG ? qr[PARTS - 1][w] : qsm[n][PARTS - 1][QREG ? 0 : w][lane];
                to2 = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
    if constexpr (!QREG) __syncthreads();

    float o[NT][D / 16][4], nm[NT][2], l[NT][2];                   // nm: minus the reference, +inf before the first
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
        nm[n][0] = nm[n][1] = INFINITY;
        l[n][0] = l[n][1] = 0.0f;
    }

    int stage = 0;
    for (int i = 0; i < mine; ++i) {
        issue(i + KD_STAGES - 1, stage == 0 ? KD_STAGES - 1 : stage - 1);
        cp_async_wait<KD_STAGES - 1>();
        __syncwarp();
        const int key0 = (it.u0 + warp + i * KD_WARPS) * KD_UNIT;
        const uint8_t* kq = ring + stage * G::STAGE;
        const uint8_t* vq = kq + G::QB;
        __half* ks = reinterpret_cast<__half*>(ring + stage * G::STAGE + 2 * G::QB);
        __half* vs = ks + G::SB / 2;
        const bool edge = key0 + 32 > pos0 + 1 || key0 < it.lo + it.n_new;
        if (edge) {     // a row that nothing sees may hold any scale
            const int key = key0 + lane;
            if (key >= it.kv || key < it.lo)
#pragma unroll
                for (int e = 0; e < D / 32; ++e) ks[lane * (D / 32) + e] = vs[lane * (D / 32) + e] = __ushort_as_half(0);
            __syncwarp();
        }

        // S^T: matrix row r of an 8-row half is key kd_key(r) of its 8
        float s[NT][2][4];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
            uint32_t w[2][KW];
            __half2 d[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int key = 16 * kt + 8 * j + kg;
                if constexpr (KW == 4) {
                    const uint4 u = *reinterpret_cast<const uint4*>(kq + key * (D / 2) + t * 16);
                    w[j][0] = u.x; w[j][1] = u.y; w[j][2] = u.z; w[j][3] = u.w;
                } else {
                    const uint2 u = *reinterpret_cast<const uint2*>(kq + key * (D / 2) + t * 8);
                    w[j][0] = u.x; w[j][1] = u.y;
                }
                d[j] = __half2half2(ks[key * (D / 32) + (t * D / 128)]);
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) s[n][kt][0] = s[n][kt][1] = s[n][kt][2] = s[n][kt][3] = 0.0f;
#pragma unroll
            for (int i2 = 0; i2 < KW; ++i2) {
                uint32_t fa[4], fb[4];
                kv_fields(w[0][i2], d[0], fa);
                kv_fields(w[1][i2], d[1], fb);
                const uint32_t a0[4] = {fa[0], fb[0], fa[1], fb[1]}, a1[4] = {fa[2], fb[2], fa[3], fb[3]};
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; --p) {         // low parts first
                        const uint4 q = QREG ? qr[p][i2] : qsm[n][p][QREG ? 0 : i2][lane];
                        mma_16816(s[n][kt], a0, q.x, q.y);
                        mma_16816(s[n][kt], a1, q.z, q.w);
                    }
            }
        }
        // exponents: value j of a row is key 8 j + kd_key(g)
        const int at = key0 + kg;
        float v[NT][2][4];
        auto exponents = [&]() {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[n][c][j] = fmaf(s[n][j >> 1][2 * (j & 1) + c], sc[n][c], nm[n][c]);
            if (edge) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const unsigned width = limit[n][c] - from[n][c];
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if ((unsigned)(at + 8 * j - from[n][c]) >= width) v[n][c][j] = -INFINITY;
                    }
            }
        };
        exponents();
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) top = fmaxf(top, v[n][c][j]);
        if (__any_sync(~0u, top > KvRef<SPLIT>::move)) {                     // a row's reference moves
            float old[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) { old[n][c] = nm[n][c]; nm[n][c] = 0.0f; }
            exponents();
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float mx = fmaxf(fmaxf(v[n][c][0], v[n][c][1]), fmaxf(v[n][c][2], v[n][c][3]));
#pragma unroll
                    for (int i2 = 4; i2 < 32; i2 <<= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, i2));
                    const float now = fminf(old[n][c], KvRef<SPLIT>::minus(mx)), f = now == INFINITY ? 1.0f : fast_exp2(now - old[n][c]);
                    nm[n][c] = now;
                    l[n][c] *= f;
#pragma unroll
                    for (int i2 = 0; i2 < D / 16; ++i2) {
                        o[n][i2][c] *= f;
                        o[n][i2][2 + c] *= f;
                    }
                }
            exponents();
#pragma unroll
            for (int n = 0; n < NT; ++n)                           // a row that has seen nothing yet: no weight
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    if (nm[n][c] == INFINITY)
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[n][c][j] = v[n][c][j] != v[n][c][j] ? v[n][c][j] : -INFINITY;
        }
        uint32_t pb[NT][PARTS][4];                                 // P^T fragments of the four 8-key groups
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float p0 = fast_exp2(v[n][0][j]), p1 = fast_exp2(v[n][1][j]);
                l[n][0] += p0;
                l[n][1] += p1;
                const uint32_t hi = pack_half2(p0, p1);
                pb[n][0][j] = turn8x8(hi);
                if constexpr (SPLIT) {
                    const __half2 hh = as_half2(hi);
                    pb[n][PARTS - 1][j] = turn8x8(pack_half2(p0 - __low2float(hh), p1 - __high2float(hh)));
                }
            }
        // O^T: matrix rows g and g + 8 of tile i are values (D / 8) g + 2 i and + 1 of the head. The tensor core cuts what
        // it adds to an accumulator: n products in one lose up to n 2^-24 of it. So the 32 keys' sum is made from zero and
        // added to O here (fp32, 131071 keys: 2 us of 55, where one accumulator for all keys was 2e-6 off).
        uint32_t w[8][VW];                                         // the two keys of lane t, of each 8-key group
        __half2 d[4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = 8 * (j >> 1) + (j & 1 ? k1 : k0);
            if constexpr (VW == 2) {
                const uint2 u = *reinterpret_cast<const uint2*>(vq + key * (D / 2) + ((g * 8) ^ ((k0 & 2) << 4)));
                w[j][0] = u.x; w[j][1] = u.y;
            } else {
                w[j][0] = *reinterpret_cast<const uint32_t*>(vq + key * (D / 2) + g * 4);
            }
            const __half dj = vs[key * (D / 32) + (g * D / 256)];
            d[j >> 1] = j & 1 ? __halves2half2(__low2half(d[j >> 1]), dj) : __half2half2(dj);
        }
#pragma unroll
        for (int i2 = 0; i2 < VW; ++i2) {
            uint32_t fl[8][4];                                     // fields 0..3: values 0 2 4 6; 4..7: 1 3 5 7
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                kv_fields(__byte_perm(w[2 * j][i2], w[2 * j + 1][i2], 0x5410u), d[j], fl[2 * j]);
                kv_fields(__byte_perm(w[2 * j][i2], w[2 * j + 1][i2], 0x7632u), d[j], fl[2 * j + 1]);
            }
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint32_t av[4] = {fl[4 * h][f], fl[4 * h + 1][f], fl[4 * h + 2][f], fl[4 * h + 3][f]};
                            mma_16816(sum, av, pb[n][p][2 * h], pb[n][p][2 * h + 1]);
                        }
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[n][4 * i2 + f][e] += sum[e];
                }
        }
        __syncwarp();                                              // the stage may be overwritten
        if (++stage == KD_STAGES) stage = 0;
    }

    // ---- join the warps: lane sums, then O in the ring's memory ----
    __syncthreads();                                               // every warp is done with its ring
    constexpr int OLD = D + 4;
    float* osh = reinterpret_cast<float*>(smem);
    float* msh = osh + KD_WARPS * ROWS * OLD;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            for (int i = 4; i < 32; i <<= 1) l[n][c] += __shfl_xor_sync(~0u, l[n][c], i);
            const int r = warp * ROWS + 8 * n + 2 * t + c;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                *reinterpret_cast<float2*>(osh + r * OLD + (D / 8) * g + 2 * i) = make_float2(o[n][i][c], o[n][i][2 + c]);
            if (g == 0) {
                msh[r * 2] = -nm[n][c];
                msh[r * 2 + 1] = l[n][c];
            }
        }
    __syncthreads();
    const bool whole = it.chunks == 1;
    const int live = min(rows, ROWS);
    for (int i = threadIdx.x; i < live * (D / 4); i += KD_WARPS * 32) {
        const int r = i / (D / 4), e = (i - r * (D / 4)) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) mm = fmaxf(mm, msh[(w * ROWS + r) * 2]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float ll = 0.0f;
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int w = 0; w < KD_WARPS; ++w) {
            const float f = fast_exp2(msh[(w * ROWS + r) * 2] - ref);
            const float4 v = *reinterpret_cast<const float4*>(osh + (w * ROWS + r) * OLD + e);
            ll += msh[(w * ROWS + r) * 2 + 1] * f;
            acc.x += v.x * f; acc.y += v.y * f; acc.z += v.z * f; acc.w += v.w * f;
        }
        if (whole) kv_store_out<DT, D>(a, KvaRow{it.row0 + r / a.group, it.head * a.group + r % a.group}, e, acc, ll);
        else {
            float* part = a.part + (size_t)it.slot * G::PART;
            *reinterpret_cast<float4*>(part + r * D + e) = acc;
            if (e == 0) {
                part[ROWS * D + 2 * r] = mm;
                part[ROWS * D + 2 * r + 1] = ll;
            }
        }
    }
    if (!whole) kv_join_last<D, DT, ROWS>(a, it, live, smem, G::SMEM, &sh_last);
    __syncthreads();
  }
}

template <int D, int DT, int NT>
static tk_status go_decode_t(tk_ctx* ctx, const KvaArgs& a, unsigned grid, int least, cudaStream_t st) {
    static std::atomic<uint64_t> attr_done{0};
    auto kern = kv_decode_kernel<D, DT, NT>;
    cudaError_t e = smem_attr_once(kern, KdGeo<D, NT>::SMEM, ctx->device, attr_done);
    if (e != cudaSuccess) return cuda_fail(e, "kv decode smem attribute");
    ProfScope ps(ctx, st, PK_SERVE);
    e = launch_dependent(kern, grid, KD_WARPS * 32, KdGeo<D, NT>::SMEM, st, a, (uint32_t)least);
    ctx->launches++;
    return cuda_fail(e, "kv decode launch");
}

template <int D, int DT>
static tk_status go_decode(tk_ctx* ctx, KvaArgs& a, cudaStream_t st) {
    const size_t pairs = (size_t)a.s.n_seqs * a.c.heads;
    const int nt = ((int)a.s.max_new * a.group + 7) / 8;
    const unsigned grid = kd_blocks(nt) * ctx->num_sms;   // what is resident at once
    const int least = KD_WARPS;                           // a unit for every warp
    if (pairs * ((size_t)a.s.max_pages << a.c.page_shift) / KD_UNIT + pairs > (1ull << 31))
        return fail(TK_ERR_UNSUPPORTED, "tk_kv_attend: sequences x heads x table length beyond 2^36 tokens");
    tk_status r = ws_ensure(ctx, (size_t)grid * 2 * (8 * nt * (D + 2)) * sizeof(float), st);
    if (r != TK_OK) return r;
    a.part = static_cast<float*>(ctx->ws);
    a.count = ctx->kv_sync + ctx->num_sms;
    switch (nt) {
        case 1: return go_decode_t<D, DT, 1>(ctx, a, grid, least, st);
        case 2: return go_decode_t<D, DT, 2>(ctx, a, grid, least, st);
        case 3: return go_decode_t<D, DT, 3>(ctx, a, grid, least, st);
        default: return go_decode_t<D, DT, 4>(ctx, a, grid, least, st);
    }
}
template <int D>
static tk_status go_decode_d(tk_ctx* ctx, KvaArgs& a, int dtype, cudaStream_t st) {
    if (dtype == TK_DT_F32) return go_decode<D, TK_DT_F32>(ctx, a, st);
    if (dtype == TK_DT_F16) return go_decode<D, TK_DT_F16>(ctx, a, st);
    return go_decode<D, TK_DT_BF16>(ctx, a, st);
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
    // few rows per key/value head are memory's work, many the tensor cores'
    if ((long)s.max_new * a.group <= KD_MAX_ROWS)
        return c.head_dim == 64 ? go_decode_d<64>(ctx, a, dtype, st) : go_decode_d<128>(ctx, a, dtype, st);
    return launch_kv_prompt(ctx, a, dtype, st);
}

}  // namespace tk
