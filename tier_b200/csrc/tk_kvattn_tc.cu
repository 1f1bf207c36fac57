// tk_kvattn_tc.cu -- tk_kv_attend for many rows per key/value head (prompts,
// chunks of them, long drafts): attention over the 4-bit cache on tcgen05.
//
// A block works on one key/value head of one sequence and up to two sets
// ("streams") of 128 query rows (row = token * group + head of the group), one
// tile of 128 keys after the other:
//   S = Q K^T      both from shared memory, 128 x 128 in TMEM
//   P = 2^(S - m)  one thread a row, written over S as fp16
//   O += P V       P from TMEM, V from shared memory, 128 x head_dim in TMEM
// fp32 rows enter as hi and lo fp16 parts, P too (two products each, one
// stream's rows): 22 bits of each.  The tensor core works on one stream while
// the other's softmax runs.  With at most 128 rows both streams take the same
// rows and every other tile of keys, and are joined at the end.
//
// The keys and values of a tile are turned from 4 bits to fp16 once per block,
// by four warps, a key a thread, one tile ahead in registers, straight into
// the 128-byte-swizzled operand layout (the same bytes serve K, whose
// reduction index is the head's values, and V, where it is the keys).
//
// The tensor core cuts what it adds to an accumulator: n products in one lose
// up to n 2^-24 of it (fp32, 30000 keys: 1.1e-4).  So every SEG steps O is
// added to a sum in fp32, in memory that stays in L2, and begins from zero:
// 128 products (7.6e-6) for fp32, 512 (3.1e-5, of a rounding of 4.9e-4) else.
//
// As in the streaming kernel the softmax's reference moves only when a weight
// would near fp16's largest (KvRef), so that O in TMEM is rarely rescaled.
//
// Warps (512 threads, one block an SM): 0-3 and 4-7 the streams' softmax, 8-11
// the converters, 12 issues the products (13-15 idle: registers are divided by
// groups of four warps).  A row set that would leave SMs idle
// is cut along the keys, and its parts joined by the last block to finish.
//
// Bound: the softmax's instructions (an exponential, a product-sum, an addition
// and half a conversion a score) beside the tensor core's 2 x 128 cycles a
// tile; neither waits long for the other, under a power limit that holds the
// clock at 1.47 GHz of 1.97 in long prompts.  Measured (32 query heads on 8
// key/value heads of 128; calls one after the other): a prompt of 8192, bf16,
// 608 us, 904 TFLOP/s; three chunks of up to 1000 rows behind 6001 keys, window
// 1024, 16 heads on 4 of 64, fp16, 31.5 us; two fp32 prompts of up to 1537 rows,
// 2000 keys, 152 us, 252 TFLOP/s (two parts of q and of P: twice that in the
// tensor core).
#include "tk_f32x2.cuh"
#include "tk_kv.cuh"

namespace tk {
namespace kt {

constexpr int ROWS = 128, KEYS = 128, THREADS = 512;
// registers a thread of each warpgroup: 4 x 128 at launch, 192 + 192 + 80 + 48 = 512 after the split
// (184 + 184 + 88 + 56 spills in the softmax: a prompt of 8192 took 652 us, not 609)
constexpr int REG_SOFTMAX = 192, REG_CONVERT = 80, REG_ISSUE = 48;

template <int D, bool SPLIT>
struct Geo {
    static constexpr int TILE = 128 * D * 2;                       // bytes of 128 rows in fp16
    static constexpr int PANEL = 128 * 128;                        // 64 columns of them
    static constexpr int GROUP = SPLIT ? ROWS : 2 * ROWS;          // query rows of a block
    static constexpr int SMEM = 6 * TILE + 1024;                   // q: 2 sets (or parts), K and V: 2 stages each
    static constexpr uint32_t S = 0, O = 256;                      // TMEM columns: S of stream w at 128 w, O at 256 + D w
    static constexpr int PART = GROUP * (D + 2);                   // floats of a part: O, then (m, l) of each row
    static constexpr int SUM = 2 * ROWS * D;                       // floats of the two streams' sums
    static constexpr int SEG = SPLIT ? 8 : 64;                     // steps between additions to them (a power of two)
};

struct Item {
    int b, head, group, part, parts;
    int kv, n_new, row0, rows;             // rows: of this block, from row group * GROUP of the sequence
    int tok0, sub0;                        // token of the first of them, and head of the group
    int lo, hi, t0, t1;                    // this part's tiles, and the keys [lo, hi) of them that some row may see
};

// What a sequence asks for: its row sets per head, and the tiles of the longest.
struct Need {
    SeqInfo q;
    int groups, tiles;
};
template <int GROUP>
__device__ __forceinline__ Need need(const KvaArgs& a, int b, int* status) {
    Need n{SeqInfo{0, 0, 0}, 0, 0};
    if (b >= a.s.n_seqs) return n;
    n.q = seq_info(a.s, a.c.page_shift, b, status);
    n.groups = (int)(((long)n.q.n_new * a.group + GROUP - 1) / GROUP);
    n.tiles = (n.q.kv + KEYS - 1) / KEYS;
    return n;
}

// Whether row sets are cut into parts: twice as many as there are would fill
// the SMs at most.  (64 bits: packed rows that invalid contents name in many
// sequences are counted in each.)
__host__ __device__ __forceinline__ bool cuts(long sets, int heads, int sms) { return 2 * sets * heads <= sms; }

// Item `x`: sequences in order, within one the last rows (most keys) first,
// heads innermost.  Row sets are cut into parts only while that leaves no more
// blocks than SMs.
template <int GROUP>
__device__ __forceinline__ bool find(const KvaArgs& a, int x, int sms, Item& it) {
    const int lane = threadIdx.x & 31;
    long sets = 0, work = 0;                                       // row sets, their tiles
    const Need first = need<GROUP>(a, lane, a.status);             // kept: mostly there are no others
    for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
        const Need n = b0 ? need<GROUP>(a, b0 + lane, a.status) : first;
        sets += __reduce_add_sync(~0u, n.groups);
        long w = (long)n.groups * n.tiles;
        for (int i = 16; i; i >>= 1) w += __shfl_xor_sync(~0u, w, i);
        work += w;
    }
    int per = INT32_MAX;                                           // tiles of a part
    if (cuts(sets, a.c.heads, sms)) {
        // at most sms / 2 parts are begun and not full, so that twice the even
        // share (six steps of an eighth) always fits
        per = max(1, (int)((work * a.c.heads + sms - 1) / sms));
        for (int step = 0; step < 6; ++step, per += (per + 7) / 8) {
            int parts = 0;
            for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
                const Need n = b0 ? need<GROUP>(a, b0 + lane, nullptr) : first;
                parts += __reduce_add_sync(~0u, n.groups * ((max(n.tiles, 1) + per - 1) / per));
            }
            if (parts * a.c.heads <= sms) break;
        }
        if (per < 2) per = 2;
    }
    int before = 0;
    for (int b0 = 0; b0 < a.s.n_seqs; b0 += 32) {
        const Need n = b0 ? need<GROUP>(a, b0 + lane, nullptr) : first;
        const int parts = per == INT32_MAX ? 1 : (max(n.tiles, 1) + per - 1) / per;
        const int mine = n.groups * a.c.heads * parts;
        int sum = mine;
        for (int i = 1; i < 32; i <<= 1) {
            const int o = __shfl_up_sync(~0u, sum, i);
            if (lane >= i) sum += o;
        }
        const unsigned hit = __ballot_sync(~0u, x < before + sum);
        if (hit) {
            const int src = __ffs(hit) - 1;
            it.b = b0 + src;
            it.kv = __shfl_sync(~0u, n.q.kv, src);
            it.n_new = __shfl_sync(~0u, n.q.n_new, src);
            it.row0 = __shfl_sync(~0u, n.q.row0, src);
            it.parts = __shfl_sync(~0u, parts, src);
            const int groups = __shfl_sync(~0u, n.groups, src);
            const int at = x - before - __shfl_sync(~0u, sum - mine, src);
            it.part = at % it.parts;
            const int set = at / it.parts;
            it.head = set % a.c.heads;
            it.group = groups - 1 - set / a.c.heads;
            it.rows = (int)min((long)GROUP, (long)it.n_new * a.group - (long)it.group * GROUP);
            const int pos0 = it.kv - it.n_new;
            it.tok0 = (int)((long)it.group * GROUP / a.group);
            it.sub0 = (int)((long)it.group * GROUP - (long)it.tok0 * a.group);
            const int front = pos0 + it.tok0, last = front + (int)((unsigned)(it.sub0 + it.rows - 1) / (unsigned)a.group);
            it.hi = max(last + 1, 0);
            it.lo = kv_first_key(front, a.window);
            const int t = it.lo / KEYS, n2 = it.hi > it.lo ? (it.hi + KEYS - 1) / KEYS - t : 0;
            it.t0 = t + (int)((long)n2 * it.part / it.parts);
            it.t1 = t + (int)((long)n2 * (it.part + 1) / it.parts);
            it.hi = min(it.hi, it.t1 * KEYS);                      // (a stream's last tile may lie behind the part)
            return true;
        }
        before += __shfl_sync(~0u, sum, 31);
    }
    return false;
}

__device__ __forceinline__ void tc_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tc_st_32x32b_x8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tc_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// The two softmax warpgroups' own barrier.
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The products' warp stays converged, so that descriptors live in uniform
// registers: one lane (`one`) issues.  With the whole loop in one lane, moving
// each product's operands into place took twice the product's own 64 cycles.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
// D[tmem] (+)= A[smem desc] * B[smem desc]^T, kind::f16.
__device__ __forceinline__ void mma_ss(uint32_t one, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem desc], kind::f16.
__device__ __forceinline__ void mma_ts(uint32_t one, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t one, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
        "r"(one)
        : "memory");
}

// A place for the block's sums: one block an SM is resident, so that of `slots`
// places one is free (its flag is zero between blocks).
__device__ __forceinline__ int take_slot(int* busy, int slots, int* status) {
    uint32_t s;
    asm volatile("mov.u32 %0, %%smid;" : "=r"(s));
    s %= (uint32_t)slots;
    const uint64_t t0 = globaltimer();
    do {
        for (int i = 0; i < slots; ++i, s = s + 1 == (uint32_t)slots ? 0 : s + 1)
            if (atomicCAS(busy + s, 0, 1) == 0) {
                __threadfence();
                return (int)s;
            }
    } while (globaltimer() - t0 < kWaitLimitNs);
    raise_status(status, DEV_TIMEOUT);
    return -1;
}

// The last part of a row set to finish joins them, in the order of the keys
// (by the softmax warpgroups; parts lie by block).
template <int D, int DT>
__device__ __forceinline__ void join_parts(const KvaArgs& a, const Item& it, uint8_t* smem, int* sh_last) {
    using G = Geo<D, DT == TK_DT_F32>;
    __threadfence();
    softmax_sync();
    if (threadIdx.x == 0) {
        int* n = a.count + (blockIdx.x - it.part);                 // (sets in parts have no more blocks than SMs)
        const int done = atomicAdd(n, 1) + 1;
        *sh_last = done == it.parts;
        if (*sh_last) *n = 0;
    }
    softmax_sync();
    if (!*sh_last) return;
    __threadfence();
    const float* base = a.part + (size_t)(blockIdx.x - it.part) * G::PART;
    kv_join<D, DT, G::GROUP>(
        a, it.parts, it.rows, threadIdx.x, 256, smem, G::SMEM - 1024, [&](int c) { return base + (size_t)c * G::PART; },
        [&](int row) {
            const long grow = (long)it.group * G::GROUP + row;
            return KvaRow{it.row0 + (int)(grow / a.group), it.head * a.group + (int)(grow % a.group)};
        },
        [] { softmax_sync(); });
}

template <int D, int DT>
__global__ void __launch_bounds__(THREADS, 1) kv_prompt_kernel(const KvaArgs a, float* sums, int* busy, int sms) {
    constexpr bool SPLIT = DT == TK_DT_F32;
    constexpr int PARTS = SPLIT ? 2 : 1;                           // fp16 parts of q and of P
    using G = Geo<D, SPLIT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], q_full, s_full[2], p_full[2], o_full[2];
    __shared__ uint32_t tmem_slot;
    __shared__ float ml[2][ROWS][2];
    __shared__ int sh_last, sh_slot;
    __shared__ Item it;                                            // (not in registers: the softmax needs them all)
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sq = smem, *sk = smem + 2 * G::TILE, *sv = smem + 4 * G::TILE;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    pdl_trigger();
    pdl_wait();
    Item found;
    if (!find<G::GROUP>(a, blockIdx.x, sms, found)) return;
    // both streams on the same rows, every other tile each
    const bool same = SPLIT || found.rows <= ROWS;
    const int tiles = found.t1 - found.t0;
    const int steps = same ? (tiles + 1) / 2 : tiles;              // tiles of a stream
    if (threadIdx.x == 0) {
        it = found;
        sh_slot = steps > G::SEG ? take_slot(busy, sms, a.status) : -1;
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], 128);
            mbar_init(&v_full[i], 128);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_empty[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 128);
            mbar_init(&o_full[i], 1);
        }
        mbar_init(&q_full, 256);
        fence_mbar_init();
    }
    if (warp == 12) {
        tmem_alloc(&tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;

    const int made = same ? 2 * steps : steps;                     // tiles made (the last may have no keys)
    const int pos0 = it.kv - it.n_new;
    // lane address of a softmax warp's rows
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;

    if (warp < 8) {
        reg_inc<REG_SOFTMAX>();
        float l = 0.0f, nm = INFINITY;                             // nm: minus the reference; +inf before the first
        // ---------------- softmax: thread = row ----------------
        const int w = warp >> 2, r = (warp & 3) * 32 + lane, row = same ? r : w * ROWS + r;
        const bool live = row < it.rows;
        const int tok = it.tok0 + (int)((unsigned)(it.sub0 + row) / (unsigned)a.group);
        const int end = live ? max(pos0 + tok + 1, 0) : 0, from = a.window > 0 ? max(end - a.window, 0) : 0;
        const int limit = min(end, it.hi);                         // keys [from, limit) are this part's and seen
        constexpr int LANES = D / 8, AT_ONCE = 32 / LANES;         // lanes of a row, rows of a warp's instruction
        // packed row and head (within the group) of a row of this block, and of the row AT_ONCE further
        auto place = [&](int x) {
            const unsigned g = (unsigned)(it.sub0 + x), t = g / (unsigned)a.group;
            return KvaRow{it.row0 + it.tok0 + (int)t, (int)(g - t * (unsigned)a.group)};
        };
        auto further = [&](KvaRow& p) {
            for (p.head += AT_ONCE; p.head >= a.group; p.head -= a.group) ++p.row;
        };
        float sc = 0.0f;
        if (steps) {
            // q to fp16 in shared memory: set w, or of a split both parts; the streams of `same` halve the rows. Rows come as
            // they are, all at once, and are turned where they lie by the lanes that copied them, in loops that stay short:
            // this runs once a block, and fetching its instructions is dear (a thread its own row 18000 cycles, a
            // seventh of a prompt of 8192; LANES lanes a row by registers, unrolled, 21000; so 9000).
            float(*unit)[2] = ml[same ? 0 : w];
            const int n = same ? 16 : 32, r0 = (warp & 3) * 32 + (same ? 16 * w : 0) + lane / LANES, c = lane % LANES;
            uint8_t* set = sq + (same ? 0 : w) * G::TILE + (c >> 3) * G::PANEL;
            KvaRow p = place(r0 + (same ? 0 : w * ROWS));
            const int rows = it.rows, head0 = it.head * a.group;
#pragma unroll 2
            for (int i = 0; i < n; i += AT_ONCE, further(p)) {
                const int at = r0 + i, row2 = at + (same ? 0 : w * ROWS);
                uint8_t* to = set + at * 128 + (((c & 7) ^ (at & 7)) << 4);
                if (row2 < rows) {
                    const size_t e = (size_t)p.row * a.ldq + (size_t)(head0 + p.head) * D + c * 8;
                    if constexpr (SPLIT) {
                        cp_async16(smem_u32(to), static_cast<const float*>(a.q) + e);
                        cp_async16(smem_u32(to + G::TILE), static_cast<const float*>(a.q) + e + 4);
                    } else {
                        cp_async16(smem_u32(to), static_cast<const uint16_t*>(a.q) + e);
                    }
                } else {
                    *reinterpret_cast<uint4*>(to) = make_uint4(0, 0, 0, 0);
                    if constexpr (SPLIT) *reinterpret_cast<uint4*>(to + G::TILE) = make_uint4(0, 0, 0, 0);
                }
            }
            cp_async_commit();
            cp_async_wait<0>();
#pragma unroll 1
            for (int i = 0; i < n; i += 2 * AT_ONCE) {             // two rows a lane at once
                float x[2][8], mx[2] = {0.0f, 0.0f};
                auto spot = [&](int k) {
                    const int at = r0 + i + k * AT_ONCE;
                    return set + at * 128 + (((c & 7) ^ (at & 7)) << 4);
                };
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if constexpr (SPLIT) {
                        const float4 u = *reinterpret_cast<const float4*>(spot(k));
                        const float4 v = *reinterpret_cast<const float4*>(spot(k) + G::TILE);
                        x[k][0] = u.x; x[k][1] = u.y; x[k][2] = u.z; x[k][3] = u.w;
                        x[k][4] = v.x; x[k][5] = v.y; x[k][6] = v.z; x[k][7] = v.w;
                    } else {
                        load_pairs8<DT>(spot(k), 0, x[k]);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) mx[k] = fmaxf(mx[k], fabsf(x[k][e]));
                }
#pragma unroll
                for (int e = 1; e < LANES; e <<= 1)
#pragma unroll
                    for (int k = 0; k < 2; ++k) mx[k] = fmaxf(mx[k], __shfl_xor_sync(~0u, mx[k], e));
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    float back;
                    const float up = copysignf(q_unit(mx[k], back), a.scale2);
                    if (c == 0) unit[r0 + i + k * AT_ONCE][0] = back;
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float u = x[k][2 * e] * up, v = x[k][2 * e + 1] * up;
                        hi[e] = pack_half2(u, v);
                        lo[e] = pack_half2(u - __low2float(as_half2(hi[e])), v - __high2float(as_half2(hi[e])));
                    }
                    *reinterpret_cast<uint4*>(spot(k)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    if constexpr (SPLIT) *reinterpret_cast<uint4*>(spot(k) + G::TILE) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
            }
            if (same) softmax_sync();
            else __syncwarp();
            sc = fmaxf(unit[r][0] * fabsf(a.scale2), 1e-37f);      // above zero: masked scores stay -inf
            fence_async_shared();
            mbar_arrive(&q_full);
        }
        const uint32_t ts = tmem + lanes + G::S + w * 128, to = tmem + lanes + G::O + w * D;
        const bool any_live = __any_sync(~0u, live);
        // this row's sum, chunks of four values 128 rows apart, and its factor
        auto total = [&](int c) {
            return reinterpret_cast<float4*>(sums + (size_t)sh_slot * G::SUM) + (w * (D / 4) + c / 4) * ROWS + r;
        };
        float ft = 1.0f;
        const int seg = sh_slot >= 0 ? G::SEG : steps;
        bool ok = true;
        for (int j0 = 0; j0 < steps && ok; j0 += seg) {
            if (j0 > 0 && any_live) {                              // (with S, the last O is there)
                ok = __all_sync(~0u, mbar_wait(&s_full[w], j0 & 1, a.status));
                tc_fence_after();
                if (!ok) break;
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t y[32];
                    float4 t[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        t[i] = j0 > G::SEG ? __ldcg(total(c + 4 * i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    tc_ld_32x32b_x32(to + c, y);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        __stcg(total(c + 4 * i),
                               make_float4(fmaf(t[i].x, ft, __uint_as_float(y[4 * i])),
                                           fmaf(t[i].y, ft, __uint_as_float(y[4 * i + 1])),
                                           fmaf(t[i].z, ft, __uint_as_float(y[4 * i + 2])),
                                           fmaf(t[i].w, ft, __uint_as_float(y[4 * i + 3]))));
                }
                ft = 1.0f;
            }
            const int j1 = min(j0 + seg, steps);
            for (int j = j0; j < j1; ++j) {
                const int key0 = (it.t0 + (same ? 2 * j + w : j)) * KEYS;
                ok = __all_sync(~0u, mbar_wait(&s_full[w], j & 1, a.status));
                if (!ok) break;
                tc_fence_after();
                if (any_live) {
                    const bool edge = __any_sync(~0u, live && (key0 + KEYS > limit || key0 < from));
                    // S of the whole row in registers
                    float x[KEYS];
#pragma unroll
                    for (int c = 0; c < 4; ++c) tc_ld_32x32b_x32(ts + c * 32, *reinterpret_cast<uint32_t(*)[32]>(x + c * 32));
                    tc_wait_ld();
                    if (edge) {                                        // what the row does not see
                        const unsigned width = max(limit - from, 0);
                        const int rel = key0 - from;
#pragma unroll
                        for (int i = 0; i < KEYS; ++i)
                            if ((unsigned)(rel + i) >= width) x[i] = -INFINITY;
                    }
                    float m0 = x[0], m1 = x[1], m2 = x[2], m3 = x[3];
#pragma unroll
                    for (int i = 4; i < KEYS; i += 8) {
                        m0 = max3(m0, x[i], x[i + 1]);
                        m1 = max3(m1, x[i + 2], x[i + 3]);
                        if (i + 4 < KEYS) {
                            m2 = max3(m2, x[i + 4], x[i + 5]);
                            m3 = max3(m3, x[i + 6], x[i + 7]);
                        }
                    }
                    m0 = fmaxf(max3(m0, m1, m2), m3);
                    const bool move = fmaf(m0, sc, nm) > KvRef<SPLIT>::move;   // the largest exponent, as it is taken below
                    if (__any_sync(~0u, move)) {
                        const float now = move ? KvRef<SPLIT>::minus(m0 * sc) : nm;
                        const float f = now == INFINITY ? 1.0f : fast_exp2(now - nm);
                        nm = now;
                        l *= f;
                        ft *= f;
                        if (j > j0) {
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t y[16];
                                tc_ld_32x32b_x16(to + c, y);
                                tc_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) y[i] = __float_as_uint(__uint_as_float(y[i]) * f);
                                tc_st_32x32b_x16(to + c, y);
                            }
                            tc_wait_st();
                        }
                    }
                    const f32x2 sc2 = pack2(sc, sc), ref2 = nm == INFINITY ? pack2(0.0f, 0.0f) : pack2(nm, nm);
                    f32x2 sum = pack2(l, 0.0f);
                    // in place and in three steps, eight pairs apart, so that no
                    // exponential waits for its own operand or its own use
                    auto exponent = [&](int i) {                       // pairs i .. i + 7
#pragma unroll
                        for (int k = i; k < i + 8; ++k)
                            unpack2(fma2(pack2(x[2 * k], x[2 * k + 1]), sc2, ref2), x[2 * k], x[2 * k + 1]);
                    };
                    auto power = [&](int i) {
#pragma unroll
                        for (int k = 2 * i; k < 2 * i + 16; ++k) x[k] = fast_exp2(x[k]);
                    };
                    auto finish = [&](int i) {
                        uint32_t hi[8], lo[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float p0 = x[2 * (i + k)], p1 = x[2 * (i + k) + 1];
                            sum = add2(sum, pack2(p0, p1));
                            hi[k] = pack_half2(p0, p1);
                            if constexpr (SPLIT)
                                lo[k] = pack_half2(p0 - __low2float(as_half2(hi[k])), p1 - __high2float(as_half2(hi[k])));
                        }
                        tc_st_32x32b_x8(ts + i, hi);
                        if constexpr (SPLIT) tc_st_32x32b_x8(ts + 64 + i, lo);
                    };
                    exponent(0);
#pragma unroll
                    for (int i = 0; i < KEYS / 2; i += 8) {
                        power(i);
                        if (i + 8 < KEYS / 2) exponent(i + 8);
                        if (i >= 8) finish(i - 8);
                    }
                    finish(KEYS / 2 - 8);
                    float s0, s1;
                    unpack2(sum, s0, s1);
                    l = s0 + s1;
                    tc_wait_st();
                }
                tc_fence_before();
                mbar_arrive(&p_full[w]);
            }
        }
        if (steps) {
            mbar_wait(&o_full[w], 0, a.status);
            tc_fence_after();
        }
        ml[w][r][0] = -nm;
        ml[w][r][1] = l;
        auto add_total = [&](int c, uint32_t (&x)[32]) {
            if (sh_slot < 0 || !any_live) return;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 t = __ldcg(total(c + 4 * i));
                x[4 * i] = __float_as_uint(fmaf(t.x, ft, __uint_as_float(x[4 * i])));
                x[4 * i + 1] = __float_as_uint(fmaf(t.y, ft, __uint_as_float(x[4 * i + 1])));
                x[4 * i + 2] = __float_as_uint(fmaf(t.z, ft, __uint_as_float(x[4 * i + 2])));
                x[4 * i + 3] = __float_as_uint(fmaf(t.w, ft, __uint_as_float(x[4 * i + 3])));
            }
        };
        if (same) {                                                // the second stream's O of the same rows by way of smem
            float* osh = reinterpret_cast<float*>(smem);           // [128][D + 4]
            softmax_sync();                                        // (both streams' products are done: q, K and V are free)
            if (w == 1 && steps)
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    uint32_t x[32];
                    tc_ld_32x32b_x32(to + c, x);
                    tc_wait_ld();
                    add_total(c, x);
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(osh + r * (D + 4) + c + i) = make_uint4(x[i], x[i + 1], x[i + 2], x[i + 3]);
                }
            softmax_sync();
        }
        float* part = it.parts > 1 ? a.part + (size_t)blockIdx.x * G::PART : nullptr;
        if (!same || w == 0) {
            const float* osh = reinterpret_cast<const float*>(smem);
            float m = -nm, sum = l, f0 = 1.0f, f1 = 0.0f;
            if (same) {
                const float m1 = ml[1][r][0], big = fmaxf(m, m1), ref = big == -INFINITY ? 0.0f : big;
                f0 = fast_exp2(m - ref);
                f1 = fast_exp2(m1 - ref);
                sum = sum * f0 + ml[1][r][1] * f1;
                m = big;
            }
            if (part && live) {
                part[G::GROUP * D + 2 * row] = m;
                part[G::GROUP * D + 2 * row + 1] = sum;
            }
            const bool none = sum == 0.0f && !part;                // sees nothing: zero
            const float inv = part ? 1.0f : none ? 0.0f : __fdividef(1.0f, sum);
            // by halves of the columns through shared memory nothing else uses now, so that whole rows are written, four
            // at once (one at a time, each by a division, 14500 cycles a block; so 10000)
            const KvaRow first = place(row - lane + lane / LANES);
            uint8_t* stage = (same ? sv : sq + w * G::TILE) + (warp & 3) * 32 * (2 * D);
#pragma unroll 1
            for (int half = 0; half < D && any_live; half += D / 2) {
#pragma unroll 1
                for (int c = half; c < half + D / 2; c += 32) {
                    uint32_t x[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) x[i] = 0;
                    if (steps) {                                   // (uniform)
                        tc_ld_32x32b_x32(to + c, x);
                        tc_wait_ld();
                        add_total(c, x);
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float4 o = make_float4(__uint_as_float(x[i]) * f0, __uint_as_float(x[i + 1]) * f0,
                                               __uint_as_float(x[i + 2]) * f0, __uint_as_float(x[i + 3]) * f0);
                        if (same && steps) {
                            const float4 u = *reinterpret_cast<const float4*>(osh + r * (D + 4) + c + i);
                            o.x += u.x * f1; o.y += u.y * f1; o.z += u.z * f1; o.w += u.w * f1;
                        }
                        o = none ? make_float4(0, 0, 0, 0) : make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
                        *reinterpret_cast<float4*>(stage + lane * (2 * D) + ((((c - half + i) >> 2) ^ (lane & 7)) << 4)) = o;
                    }
                }
                __syncwarp();
                KvaRow p = first;
                const int rows = it.rows, head0 = it.head * a.group;
#pragma unroll 1
                for (int i = 0; i < 32; i += 4 * AT_ONCE) {
                    const int q4 = lane % LANES;
                    float4 o[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int from = i + k * AT_ONCE + lane / LANES;
                        o[k] = *reinterpret_cast<const float4*>(stage + from * (2 * D) + ((q4 ^ (from & 7)) << 4));
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k, further(p)) {
                        const int at = row - lane + i + k * AT_ONCE + lane / LANES;
                        if (at >= rows) continue;
                        if (part) *reinterpret_cast<float4*>(part + at * D + half + q4 * 4) = o[k];
                        else kv_store_out<DT, D>(a, KvaRow{p.row, head0 + p.head}, half + q4 * 4, o[k], 1.0f);
                    }
                }
                __syncwarp();
            }
        }
        if (part) join_parts<D, DT>(a, it, smem, &sh_last);
    } else if (warp < 12) {
        reg_dec<REG_CONVERT>();
        // ---------------- converters: thread = key of the tile ----------------
        const int t = threadIdx.x - 256;
        uint4 kr[D / 32], vr[D / 32];
        uint32_t ks[D / 64], vs[D / 64];
        auto fetch = [&](int i) {
            const int pos = (it.t0 + i) * KEYS + t;
            const bool in = i < made && pos >= it.lo && pos < it.hi;   // hi <= kv
            const size_t row = in ? kv_row(a.c, page_of(a.s, a.c, it.b, pos, a.status), it.head, pos) : 0;
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                kr[c] = vr[c] = make_uint4(0, 0, 0, 0);
                if (in) {
                    kr[c] = __ldg(reinterpret_cast<const uint4*>(a.c.kq + row * (D / 2)) + c);
                    vr[c] = __ldg(reinterpret_cast<const uint4*>(a.c.vq + row * (D / 2)) + c);
                }
            }
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                ks[c] = vs[c] = 0;
                if (in) {
                    ks[c] = __ldg(reinterpret_cast<const uint32_t*>(a.c.ks + row * (D / 32)) + c);
                    vs[c] = __ldg(reinterpret_cast<const uint32_t*>(a.c.vs + row * (D / 32)) + c);
                }
            }
        };
        auto store = [&](const uint4 (&x)[D / 32], const uint32_t (&s)[D / 64], uint8_t* to) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
                const __half2 sc2 = as_half2(s[c >> 1]);
                const __half2 d = c & 1 ? __high2half2(sc2) : __low2half2(sc2);
                const uint32_t w4[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t f[4];
                    kv_fields(w4[i], d, f);
                    const int chunk = 4 * c + i;
                    *reinterpret_cast<uint4*>(to + (chunk >> 3) * G::PANEL + t * 128 + (((chunk & 7) ^ (t & 7)) << 4)) =
                        make_uint4(f[0], f[1], f[2], f[3]);
                }
            }
        };
        if (made) fetch(0);
        for (int i = 0; i < made; ++i) {
            const int st = i & 1;
            const uint32_t parity = ((i >> 1) & 1) ^ 1;
            if (!__all_sync(~0u, mbar_wait(&k_empty[st], parity, a.status))) break;
            store(kr, ks, sk + st * G::TILE);
            fence_async_shared();
            mbar_arrive(&k_full[st]);
            if (!__all_sync(~0u, mbar_wait(&v_empty[st], parity, a.status))) break;
            store(vr, vs, sv + st * G::TILE);
            fence_async_shared();
            mbar_arrive(&v_full[st]);
            fetch(i + 1);
        }
    } else {
        reg_dec<REG_ISSUE>();
        if (warp == 12 && steps) {
            // ---------------- products (the whole warp; one lane issues) ----------------
            constexpr uint32_t id_s = idesc_f16(128, KEYS, 0, 0, 0), id_o = idesc_f16(128, D, 0, 0, 1);
            constexpr uint64_t TILE = G::TILE >> 4;                // in a descriptor's address units
            const uint32_t one = elect_one();
            const uint64_t dq = sdesc_sw128(smem_u32(sq), 16, 1024), dk = sdesc_sw128(smem_u32(sk), 16, 1024);
            const uint64_t dv = sdesc_sw128(smem_u32(sv), G::PANEL, 1024);
            auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(~0u, mbar_wait(bar, parity, a.status)); };
            auto product_s = [&](int w, int i) {                   // stream w, tile i of the ring
                const uint64_t kd = dk + (i & 1) * TILE;
#pragma unroll
                for (int p = PARTS - 1; p >= 0; --p) {
                    const uint64_t qd = dq + (SPLIT ? p : same ? 0 : w) * TILE;
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk) {
                        const uint32_t off = ((kk >> 2) * G::PANEL + (kk & 3) * 32) >> 4;
                        mma_ss(one, tmem + G::S + w * 128, qd + off, kd + off, id_s, p != PARTS - 1 || kk > 0);
                    }
                }
                commit(one, &s_full[w]);
                if (same || w == 1) commit(one, &k_empty[i & 1]);
            };
            const bool cut = sh_slot >= 0;
            bool ok = wait(&q_full, 0);
            for (int w = 0; w < 2 && ok; ++w) {
                const int i = same ? w : 0;
                ok = wait(&k_full[i & 1], (i >> 1) & 1);
                tc_fence_after();
                if (ok) product_s(w, i);
            }
            for (int j = 0; j < steps && ok; ++j)
                for (int w = 0; w < 2 && ok; ++w) {
                    const int i = same ? 2 * j + w : j;
                    ok = wait(&v_full[i & 1], (i >> 1) & 1) && wait(&p_full[w], j & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t vd = dv + (i & 1) * TILE;
                    const uint32_t more = cut ? j % G::SEG > 0 : j > 0;
#pragma unroll
                    for (int p = PARTS - 1; p >= 0; --p)
#pragma unroll
                        for (int kk = 0; kk < KEYS / 16; ++kk)
                            mma_ts(one, tmem + G::O + w * D, tmem + G::S + w * 128 + p * 64 + kk * 8, vd + (kk * 2048 >> 4), id_o,
                                   more || p != PARTS - 1 || kk > 0);
                    if (same || w == 1) commit(one, &v_empty[i & 1]);
                    if (j + 1 < steps) {
                        const int n = same ? i + 2 : j + 1;
                        ok = wait(&k_full[n & 1], (n >> 1) & 1);
                        tc_fence_after();
                        if (ok) product_s(w, n);
                    } else {
                        commit(one, &o_full[w]);
                    }
                }
            if (!ok) {  // reported; what was issued ends first
                commit(one, &o_full[0]);
                commit(one, &o_full[1]);
                mbar_wait(&o_full[0], 0, a.status);
                mbar_wait(&o_full[1], 0, a.status);
            }
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x == 0 && sh_slot >= 0) {
        __threadfence();
        atomicExch(busy + sh_slot, 0);
    }
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

template <int D, int DT>
static tk_status go(tk_ctx* ctx, KvaArgs& a, cudaStream_t st) {
    using G = Geo<D, DT == TK_DT_F32>;
    static std::atomic<uint64_t> attr_done{0};
    auto kern = kv_prompt_kernel<D, DT>;
    cudaError_t e = smem_attr_once(kern, G::SMEM, ctx->device, attr_done);
    if (e != cudaSuccess) return cuda_fail(e, "kv prompt smem attribute");
    // no more row sets than whole groups of all rows and one begun per
    // sequence; cut into parts only where there are at most as many as SMs
    const long sets = (((long)a.s.n_tokens * a.group + G::GROUP - 1) / G::GROUP + a.s.n_seqs) * a.c.heads;
    const long grid = sets > ctx->num_sms ? sets : ctx->num_sms;
    if (grid > INT32_MAX) return fail(TK_ERR_INVALID, "tk_kv_attend: too many rows");
    tk_status r = ws_ensure(ctx, (size_t)ctx->num_sms * (G::PART + G::SUM) * sizeof(float), st);
    if (r != TK_OK) return r;
    a.part = static_cast<float*>(ctx->ws);
    float* sums = a.part + (size_t)ctx->num_sms * G::PART;
    int* busy = ctx->kv_sync;
    a.count = busy + ctx->num_sms;
    ProfScope ps(ctx, st, PK_SERVE);
    e = launch_dependent(kern, (unsigned)grid, THREADS, G::SMEM, st, a, sums, busy, ctx->num_sms);
    ctx->launches++;
    return cuda_fail(e, "kv prompt launch");
}

}  // namespace kt

tk_status launch_kv_prompt(tk_ctx* ctx, KvaArgs& a, int dtype, cudaStream_t st) {
    const bool wide = a.c.dim == 128;
    if (dtype == TK_DT_F32) return wide ? kt::go<128, TK_DT_F32>(ctx, a, st) : kt::go<64, TK_DT_F32>(ctx, a, st);
    if (dtype == TK_DT_F16) return wide ? kt::go<128, TK_DT_F16>(ctx, a, st) : kt::go<64, TK_DT_F16>(ctx, a, st);
    return wide ? kt::go<128, TK_DT_BF16>(ctx, a, st) : kt::go<64, TK_DT_BF16>(ctx, a, st);
}

}  // namespace tk
