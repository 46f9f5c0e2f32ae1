// Paged attention of many rows (chunks, whole prompts, image tokens) on the
// 5th-generation tensor cores (sm_100a).
//
// A CTA takes 256 rows (the query heads of one cache head packed with the
// tokens, see attn_paged.cu) as two 128-row tiles and walks the keys that they
// see in steps of 128, each tile in half-steps of 64:
//   S_i = Q_i K^T           tcgen05.mma, both operands in shared memory, S in TMEM
//   P_i = 2^(c S_i - c m)   one thread per row (two warpgroups, one per tile)
//   O_i += P_i V            tcgen05.mma, P_i in TMEM (over S_i), V in shared
//                           memory as it lies in the cache (MN-major operand)
// S_i has a buffer for each half, so its warpgroup goes from one half-step to
// the next without waiting for a product: while it works on one half, the
// tile's issuing warp adds the other to O_i and refills its buffer.  O_i is
// rescaled only when a row's maximum has grown by more than 2^8 since the last
// time (P then stays below 256, exact enough in either 16-bit type), i.e.
// seldom after the first steps, by the warpgroup itself once the product before
// has finished.  The rounding of P to the cache's type is the only one before
// the result's; sums are taken before it.
//
//   warps 0-3, 4-7   softmax of tile 0 / 1, epilogue
//   warps 8, 9       MMA issue of tile 0 / 1; warp 8 allocates TMEM
//   warp 10          TMA producer: K and V tiles of 128 keys through a ring of
//                    stages, one box per page piece and 64-element half, the
//                    boxes of a tile issued by the warp's lanes in parallel
//   warp 11          clears the rows of V that no row sees
//
// TMEM: S_0, S_1 (two halves of 64 columns each), O_0, O_1 (head_dim each).
// Blocks of rows go heaviest first (last rows first).  With few blocks the keys
// are split over CTAs: partial results (column-major, so that the 128 threads of
// a tile store whole lines), which a second kernel joins in order.
//
// What bounds it (2 x 4224 image tokens, 30 heads of 128, f16; 505 us, 1085
// TFLOP/s, in the first milliseconds).  A step takes about 3340 cycles, and as
// many with the exponentials left out: the tensor cores work through four
// products of 128 x 64 keys, which take as long as 128 x 128 ones would (every
// product of a tile reads all its queries from shared memory), and two of
// 128 x head_dim.  The special-function units are busy for 2048 of them (32768
// exponentials).  Besides, a CTA costs about 8 us for finding its work, the
// queries, the first product and the results.  In a loop the GPU's 1000 W cap
// lowers the clock from 1965 to about 1700 MHz: 581 us (944 TFLOP/s, 69 % of
// what cuBLAS sustains there).
// Tried and dropped: one issuer and 128-key steps, where a tile waits for its
// products (the same time on these, 2 % slower on prompts, 2 % faster on one long
// chunk, 216 registers instead of 119); two threads per row; tiles taking turns
// with the special-function units; a quarter or an eighth of the exponentials by
// polynomial (faster by 1 % at best, 7 % slower on the long chunk, where the
// power cap binds most).
//
// Every wait is bounded; on timeout the kernel sets TC_STATUS_TIMEOUT, drains
// its copies and MMAs, frees TMEM and returns.  No multicast.
#include "attn_kernels.cuh"

namespace tc {
namespace {

constexpr int kThreads = 384;
constexpr float kLazy = 8.f;   // log2 of the growth of a maximum that is let pass

template <int DP>
struct ChunkLayout {
    static constexpr uint32_t halves = DP / 64;
    static constexpr uint32_t half_bytes = 128 * 128;            // 128 rows x 64 elements
    static constexpr uint32_t tile_bytes = halves * half_bytes;  // Q tile, K tile, V tile
    static constexpr uint32_t stages = DP == 128 ? 5 : 8;
    static constexpr uint32_t q_off = 0, kv_off = 2 * tile_bytes;
    static constexpr uint32_t bar_off = kv_off + stages * tile_bytes;
    // kv_full[S] kv_empty[S], [tile][half]: s_full p_full pv_done, then q_full fin v_fixed[2]
    static constexpr uint32_t misc_off = bar_off + (2 * stages + 16) * 8;
    static constexpr uint32_t bytes = misc_off + 16 + 1024;
    static constexpr uint32_t s_col = 0, o_col = 256, tmem_cols = 512;
    static_assert(bytes <= 232448, "shared memory per CTA exceeds the sm_100 limit");
};

// Bounded wait of a warp, a few instructions: a wait that gives up (after about
// a second) returns false; the role then ends, and those that wait for it give
// up in turn.  Every phase of a barrier must be waited for, or be known to be
// the current one: a parity two phases back looks the same.
__device__ __forceinline__ bool wait(uint32_t b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .u32 n;\n mov.u32 n, 20000;\n"
        "again_%=:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n @p bra done_%=;\n"
        " sub.u32 n, n, 1;\n setp.ne.u32 q, n, 0;\n @q bra again_%=;\n"
        "done_%=:\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok) : "r"(b), "r"(parity), "r"(50000u) : "memory");
    return __all_sync(0xffffffffu, ok != 0);
}
// One arrival for the warp.
__device__ __forceinline__ void warp_arrive(uint32_t b) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) bar_arrive(b);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// O (and P) are read and written by the row's own thread.
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
          "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
          "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
          "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),
          "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
          "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}

// pk = 16-bit 2^(c s + off) of N scores, sums added to `sum`.
template <bool BF16, int N>
__device__ __forceinline__ void exps(const float *s, uint64_t c2, uint64_t off2, uint32_t *pk, uint64_t (&sum)[2]) {
#pragma unroll
    for (int k = 0; k < N; k += 2) {
        float e0, e1;
        f2unpack(f2fma(f2pack(__float_as_uint(s[k]), __float_as_uint(s[k + 1])), c2, off2), e0, e1);
        e0 = ex2(e0);
        e1 = ex2(e1);
        pk[k / 2] = pack16<BF16>(e0, e1);
        sum[(k / 2) & 1] = f2add(sum[(k / 2) & 1], f2pack(__float_as_uint(e0), __float_as_uint(e1)));
    }
}

// Largest of 64 scores (NaN passed over).
__device__ __forceinline__ float top_of(const float *s) {
    float m[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
    for (int k = 4; k < 60; k += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) asm("max.f32 %0, %0, %1, %2;" : "+f"(m[e]) : "f"(s[k + e]), "f"(s[k + 4 + e]));
    asm("max.f32 %0, %0, %1, %2;" : "+f"(m[0]) : "f"(s[60]), "f"(s[61]));
    asm("max.f32 %0, %0, %1, %2;" : "+f"(m[1]) : "f"(s[62]), "f"(s[63]));
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// A in TMEM, B in shared memory.
__device__ __forceinline__ void mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc));
}
// Shared-memory descriptors with the 128-byte swizzle, as the word that holds
// the address (in 16-byte units) and the constant upper word (8-row groups
// 1024 bytes apart, version 1, layout type 2).  K-major operands (Q, K) have
// the field next to the address unused (1); the [keys x 64] halves of V are
// the MN-major operand, the next 64 elements of N `half` bytes on.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t next) { return (saddr >> 4) | (next << 16); }
__device__ __forceinline__ uint64_t desc(uint32_t low) { return (uint64_t)kDescHigh << 32 | low; }

// What a CTA works on; the same in every thread.
struct Work {
    Request rq;
    uint32_t b, h, part, n_split, split;
    int32_t row0, n_rows;
    int32_t lo[2], hi[2];     // keys that tile i's rows see, within the CTA's share
    int32_t first[2], last[2];   // its half-steps of 64 keys (tile i has none: first == last)
    int32_t begin, end;       // steps of the CTA (keys 128 step ..)
    int32_t seen_lo, seen_hi; // keys that any row sees, within the share
};

// Step j has keys that no row sees (only the first and the last can).
__device__ __forceinline__ bool cut_step(const Work &w, int32_t j) {
    return j * kChunkKeys < w.seen_lo || (j + 1) * kChunkKeys > w.seen_hi;
}

// Share `split` of block `blk` of rows and cache head h; false: there is none.
__device__ __forceinline__ bool find_work(const AttnParams &p, uint32_t blk, uint32_t h, uint32_t split, Work &w) {
    w.h = h;
    w.split = split;
    // Request b's blocks begin at first(b) = rows before it / 256 + b: that
    // leaves room for its partly filled one.
    auto first_block = [&](uint32_t b) {
        return (int64_t)p.batch.new_offsets[b] * p.group / kChunkRows + b;
    };
    if (p.batch.n_seq <= 32) {   // all requests in one round of loads
        const uint32_t lane = threadIdx.x & 31, mine = min(lane, p.batch.n_seq - 1);
        const int32_t begin = p.batch.new_offsets[mine], end = p.batch.new_offsets[mine + 1];
        const int32_t length = p.batch.lengths[mine];
        const bool before = (int64_t)begin * p.group / kChunkRows + mine <= (int64_t)blk;
        w.b = __popc(__ballot_sync(0xffffffffu, before && lane > 0 && lane < p.batch.n_seq));
        w.rq = check_request(p.batch, p.page_shift, __shfl_sync(0xffffffffu, begin, w.b),
                             __shfl_sync(0xffffffffu, end, w.b), __shfl_sync(0xffffffffu, length, w.b), p.status);
    } else {
        w.b = count_prefix(p.batch.n_seq - 1, [&](uint32_t b) { return first_block(b) <= (int64_t)blk; });
        w.rq = load_request(p.batch, p.page_shift, w.b, p.status);
    }
    w.n_rows = w.rq.n_new * (int32_t)p.group;
    const int64_t row0 = ((int64_t)blk - ((int64_t)w.rq.first * p.group / kChunkRows + w.b)) * kChunkRows;
    if (row0 < 0 || row0 >= w.n_rows) return false;
    w.row0 = (int32_t)row0;
    const int32_t place0 = w.rq.length - w.rq.n_new;
    int32_t lo_all = 0x7fffffff, hi_all = -1, unused;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int32_t r0 = w.row0 + 128 * i, r1 = min(r0 + 128, w.n_rows) - 1;
        w.lo[i] = w.hi[i] = 0;
        if (r0 < w.n_rows) {
            visible(place0 + r0 / (int32_t)p.group, w.rq.length, p.causal, p.window, w.lo[i], unused);
            visible(place0 + r1 / (int32_t)p.group, w.rq.length, p.causal, p.window, unused, w.hi[i]);
        }
        if (w.hi[i] <= w.lo[i]) {
            w.lo[i] = w.hi[i] = 0;
        } else {
            lo_all = min(lo_all, w.lo[i]);
            hi_all = max(hi_all, w.hi[i]);
        }
    }
    const int32_t steps = (int32_t)(p.chunk / kChunkKeys);   // of a share
    int32_t s0 = 0, s1 = 0;
    if (hi_all >= 0) {
        s0 = lo_all / kChunkKeys;
        s1 = (hi_all + kChunkKeys - 1) / kChunkKeys;
    }
    w.n_split = p.splits == 1 ? 1u : (uint32_t)max((s1 - s0 + steps - 1) / steps, 1);
    if (w.split >= w.n_split) return false;
    if (w.n_split > p.splits) {   // the launch was sized for a shorter span
        if (threadIdx.x == 0) atomicOr(p.status, kStatusGeometry);
        return false;
    }
    w.begin = s0 + (int32_t)w.split * steps;
    w.end = p.splits == 1 ? s1 : min(s1, w.begin + steps);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        w.lo[i] = max(w.lo[i], w.begin * kChunkKeys);
        w.hi[i] = min(w.hi[i], w.end * kChunkKeys);
        if (w.hi[i] <= w.lo[i]) {
            w.first[i] = w.last[i] = 2 * w.begin;
        } else {
            w.first[i] = w.lo[i] / 64;
            w.last[i] = (w.hi[i] + 63) / 64;
        }
    }
    w.seen_lo = min(w.first[0] < w.last[0] ? w.lo[0] : 0x7fffffff, w.first[1] < w.last[1] ? w.lo[1] : 0x7fffffff);
    w.seen_hi = max(w.hi[0], w.hi[1]);
    w.part = (blk * p.n_kv + w.h) * p.splits + w.split;
    return true;
}

// Normalised elements [c0, c0 + 32) of a row.
template <bool BF16>
__device__ __forceinline__ void store_row32(const AttnParams &p, uint16_t *o, uint32_t c0, const float *v, float inv) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pack16<BF16>(v[2 * i] * inv, v[2 * i + 1] * inv);
    if (p.out_wide >= 32 && c0 + 32 <= p.head_dim) {   // whole sectors
#pragma unroll
        for (int i = 0; i < 16; i += 8)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                         ::"l"(o + c0 + 2 * i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]),
                           "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7]) : "memory");
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t d = c0 + 8 * i;
        if (d >= p.head_dim) break;
        if (p.out_wide) {
            *reinterpret_cast<uint4 *>(o + d) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[d + 2 * k] = (uint16_t)w[4 * i + k];
                o[d + 2 * k + 1] = (uint16_t)(w[4 * i + k] >> 16);
            }
        }
    }
}

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                 const __grid_constant__ AttnParams p) {
    using L = ChunkLayout<DP>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    // Warps by role, as listed above (the block's first four are 8 to 11).
    const uint32_t warp = (threadIdx.x / 32 + 8) % 12, lane = threadIdx.x % 32, tid = warp * 32 + lane;
    Work w;
    {
        const uint32_t id = blockIdx.x / p.n_kv;   // heaviest blocks (last rows) first
        if (!find_work(p, p.n_blocks - 1 - id / p.splits, blockIdx.x % p.n_kv, id % p.splits, w)) return;
    }
    const uint32_t bars = su32(smem + L::bar_off);
    auto kv_full = [&](uint32_t i) { return bars + 8 * i; };
    auto kv_empty = [&](uint32_t i) { return bars + 8 * (L::stages + i); };
    auto s_full = [&](uint32_t i, uint32_t h) { return bars + 8 * (2 * L::stages + 2 * i + h); };
    auto p_full = [&](uint32_t i, uint32_t h) { return bars + 8 * (2 * L::stages + 4 + 2 * i + h); };
    auto pv_done = [&](uint32_t i, uint32_t h) { return bars + 8 * (2 * L::stages + 8 + 2 * i + h); };
    const uint32_t q_full = bars + 8 * (2 * L::stages + 12), fin = q_full + 8, v_fixed = fin + 8;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::misc_off);

    if (tid == 0) {
        for (uint32_t i = 0; i < L::stages; ++i) {
            bar_init(kv_full(i), 1);
            bar_init(kv_empty(i), 3);
        }
        for (uint32_t k = 0; k < 4; ++k) {
            bar_init(s_full(k / 2, k % 2), 1);
            bar_init(p_full(k / 2, k % 2), 4);
            bar_init(pv_done(k / 2, k % 2), 1);
        }
        bar_init(q_full, 8);
        bar_init(fin, 2);
        bar_init(v_fixed, 1);
        bar_init(v_fixed + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(su32(tmem_slot)), "r"(L::tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    // Queries of both tiles, DP / 8 16-byte pieces a row over the 256 softmax
    // threads, all in flight while the block sets up (one after the other they
    // took 10 us of every CTA, in two rounds 3 us).
    constexpr uint32_t q_per = DP / 8, q_rounds = q_per;
    uint32_t qv[q_rounds][4];
    if (warp < 8) {
#pragma unroll
        for (uint32_t k = 0; k < q_rounds; ++k) {
            const uint32_t c = tid + k * 256, r = c / q_per, x = c % q_per;
            const uint32_t row = (uint32_t)w.row0 + r, token = row / p.group;
            const uint16_t *q = p.q + ((uint64_t)w.rq.first + token) * p.ld_q_token +
                                (uint64_t)(w.h * p.group + row - token * p.group) * p.ld_q_head + x * 8;
            const bool on = row < (uint32_t)w.n_rows && x * 8 < p.head_dim;
            if (p.q_wide) {
                const uint4 u = on ? *reinterpret_cast<const uint4 *>(q) : make_uint4(0u, 0u, 0u, 0u);
                qv[k][0] = u.x; qv[k][1] = u.y; qv[k][2] = u.z; qv[k][3] = u.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) qv[k][e] = on ? (uint32_t)q[2 * e] | (uint32_t)q[2 * e + 1] << 16 : 0u;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= 8) {
        if (warp == 10) {
        // ---------------------------------------------------- TMA producer
        const uint32_t box = min((uint32_t)kChunkKeys, 1u << p.page_shift), pieces = kChunkKeys / box;
        const uint32_t piece = lane % pieces, half0 = lane / pieces;   // lanes: 32 / pieces halves at a time
        const int32_t key_first = w.seen_lo, key_end = w.seen_hi;
        uint32_t st = 0, ph = 0, issued = 0;
        bool ok = true;
        for (int32_t j = w.begin; j < w.end; ++j) {
            // this lane's page piece of the step (pages behind the first key seen may
            // have been given back)
            const int32_t pos = j * kChunkKeys + (int32_t)(piece * box);
            const bool on = pos < key_end && pos + (int32_t)box > key_first;
            int32_t page = 0;
            // (an impossible page is -1: a box outside the cache arrives as zeros)
            if (on) page = load_page(p.batch, p.n_pages, w.b, (uint32_t)pos >> p.page_shift, p.status);
            const int token = (int)((uint32_t)pos & ((1u << p.page_shift) - 1));
            const uint32_t n_on = __popc(__ballot_sync(0xffffffffu, on && half0 == 0));
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv) {
                if (!(ok = wait(kv_empty(st), ph ^ 1))) break;
                if (lane == 0) bar_expect_tx(kv_full(st), n_on * box * DP * 2);
                __syncwarp();
                const uint32_t dst = su32(smem + L::kv_off + st * L::tile_bytes) + piece * box * 128;
                if (on)
                    for (uint32_t hf = half0; hf < L::halves; hf += 32 / pieces)
                        tma_load_4d(dst + hf * L::half_bytes, kv ? &vmap : &kmap, kv_full(st), (int)(hf * 64), token,
                                    (int)w.h, page);
                ++issued;
                if (++st == L::stages) { st = 0; ph ^= 1; }
            }
            if (!ok) break;
        }
        __syncwarp();
        // every copy issued has landed before exit
        for (uint32_t n = issued > L::stages ? issued - L::stages : 0; n < issued; ++n)
            ok = wait(kv_full(n % L::stages), (n / L::stages) & 1u) && ok;
        if (!ok && lane == 0) atomicOr(p.status, kStatusTimeout);
        __syncwarp();
        } else if (warp == 8 || warp == 9) {
        // ---------------------------------------------------- MMA issuers, one per tile
        // (the whole warp runs the loop, so that descriptors and bounds stay
        // uniform; one elected lane issues)
        constexpr uint32_t idesc_s = mma_idesc<64, !BF16>();
        constexpr uint32_t idesc_o = mma_idesc<DP, !BF16>() | (1u << 16);   // B is MN-major
        constexpr uint32_t kHalfKeys = 64 * 128 >> 4;                       // 64 keys on, in descriptor units
        auto uniform = [](int32_t v) { return __shfl_sync(0xffffffffu, v, 0); };
        const uint32_t i = uniform(warp - 8);
        const int32_t begin = uniform(w.begin), end = uniform(w.end);
        const int32_t first = uniform(i ? w.first[1] : w.first[0]), last = uniform(i ? w.last[1] : w.last[0]);
        const uint32_t q_low = desc_low(su32(smem + L::q_off) + i * L::tile_bytes, 1);
        const uint32_t k_low = desc_low(su32(smem + L::kv_off), 1);
        const uint32_t v_low = desc_low(su32(smem + L::kv_off), L::half_bytes >> 4);
        const uint32_t s_tmem = tmem + L::s_col + i * 128, o_tmem = tmem + L::o_col + i * DP;
        // ring positions of K and V of step j: 2 (j - begin) and one more
        auto stage_of = [&](uint32_t n) { return n % L::stages; };
        auto wait_kv = [&](uint32_t n) { return wait(kv_full(stage_of(n)), (n / L::stages) & 1u); };
        bool ok = wait(q_full, 0);
        tc_fence_after();
        // Round j: for each half of the keys, O += P(j - 1) V(j - 1), then S(j)
        // over the probabilities just used.  Every K and V of the CTA is
        // released by both issuers and the clearing warp.
        for (int32_t j = begin; ok && j <= end; ++j) {
            const uint32_t n = 2 * (uint32_t)(j - begin);
            if (j > begin) {
                if (!(ok = wait_kv(n - 1))) break;
                if (cut_step(w, j - 1) && !(ok = wait(v_fixed + (j - 1 > begin ? 8 : 0), 0))) break;
            }
            const uint32_t v = v_low + stage_of(n - 1) * (L::tile_bytes >> 4);
            const uint32_t k = k_low + stage_of(n) * (L::tile_bytes >> 4);
#pragma unroll 1
            for (uint32_t h = 0; h < 2; ++h) {
                // half-steps of the product and of the scores, and how many came before
                const int32_t gp = 2 * (j - 1) + (int32_t)h, gs = gp + 2;
                const uint32_t done = (uint32_t)(gp - first);
                if (gp >= first && gp < last) {
                    if (!(ok = wait(p_full(i, h), done >> 1 & 1u))) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t kk = 0; kk < 4; ++kk)
                            mma_f16_ts(o_tmem, s_tmem + h * 64 + kk * 8, desc(v + h * kHalfKeys + kk * (2048 >> 4)),
                                       idesc_o, kk ? 1u : (uint32_t)(done > 0));
                        mma_commit(pv_done(i, h));
                    }
                    __syncwarp();
                }
                if (h == 0 && j < end && !(ok = wait_kv(n))) break;
                if (gs >= first && gs < last) {
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (uint32_t kk = 0; kk < DP / 16; ++kk) {
                            const uint32_t off = ((kk / 4) * L::half_bytes + (kk % 4) * 32) >> 4;
                            mma_f16(s_tmem + h * 64, desc(q_low + off), desc(k + h * kHalfKeys + off), idesc_s,
                                    kk ? 1u : 0u);
                        }
                        mma_commit(s_full(i, h));
                    }
                    __syncwarp();
                }
            }
            if (ok && elect_one()) {
                if (j > begin) mma_commit(kv_empty(stage_of(n - 1)));
                if (j < end) mma_commit(kv_empty(stage_of(n)));
            }
            __syncwarp();
        }
        if (elect_one()) mma_commit(fin);   // every MMA issued has completed before TMEM is freed
        __syncwarp();
        ok = wait(fin, 0) && ok;
        if (!ok && lane == 0) atomicOr(p.status, kStatusTimeout);
        } else if (warp == 11) {
        // ---------------------------------------------------- values that no row sees
        // Rows of V outside the keys seen are cleared before the product reads
        // them: their bytes are whatever the page holds there, and 0 * NaN is NaN.
        // The warp sees every load of the ring and its release with the issuers'
        // (a wait that skipped phases could not tell one from the next but one).
        const int32_t seen_lo = w.seen_lo, seen_hi = w.seen_hi;
        const uint32_t loads = 2 * (uint32_t)(w.end - w.begin);
        for (uint32_t n = 0; n < loads; ++n) {
            if (!wait(kv_full(n % L::stages), (n / L::stages) & 1u)) break;
            const int32_t j = w.begin + (int32_t)(n / 2);
            if (n % 2 == 0 || !cut_step(w, j)) {
                warp_arrive(kv_empty(n % L::stages));
                continue;
            }
            const uint32_t v = su32(smem + L::kv_off) + (n % L::stages) * L::tile_bytes;
            const int32_t key0 = j * kChunkKeys;
            // rows [0, below) and [above, 128), whole 16-byte pieces
            const uint32_t below = (uint32_t)min(max(seen_lo - key0, 0), kChunkKeys);
            const uint32_t above = (uint32_t)min(max(seen_hi - key0, 0), kChunkKeys);
            for (uint32_t c = lane; c < (below + kChunkKeys - above) * (DP / 8); c += 32) {
                const uint32_t rr = c / 8 / L::halves, hf = c / 8 % L::halves;
                const uint32_t r = rr < below ? rr : above + rr - below;
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                             ::"r"(v + hf * L::half_bytes + r * 128 + (c % 8) * 16), "r"(0) : "memory");
            }
            fence_proxy_async();
            warp_arrive(v_fixed + (j > w.begin ? 8 : 0));
            warp_arrive(kv_empty(n % L::stages));
        }
        __syncwarp();
        }
    } else {
        // ---------------------------------------------------- softmax
        const int i = warp / 4;
        const int32_t first = i ? w.first[1] : w.first[0], last = i ? w.last[1] : w.last[0];
        // queries of both tiles into shared memory
        {
#pragma unroll
            for (uint32_t k = 0; k < q_rounds; ++k) {
                const uint32_t c = tid + k * 256, r = c / q_per, x = c % q_per;
                const uint32_t dst = su32(smem + L::q_off) + (r / 128) * L::tile_bytes + (x / 8) * L::half_bytes +
                                     (r % 128) * 128 + (((x % 8) ^ (r % 8)) << 4);
                const uint32_t sign = p.negate_q ? 0x80008000u : 0u;
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                             ::"r"(dst), "r"(qv[k][0] ^ sign), "r"(qv[k][1] ^ sign), "r"(qv[k][2] ^ sign),
                               "r"(qv[k][3] ^ sign) : "memory");
            }
            fence_proxy_async();
            warp_arrive(q_full);
        }
        const uint32_t quad = warp & 3, r = quad * 32 + lane;     // row of the tile = TMEM lane
        const uint32_t t_s = tmem + ((quad * 32) << 16) + L::s_col + i * 128;
        const uint32_t t_o = tmem + ((quad * 32) << 16) + L::o_col + i * DP;
        const int32_t row = w.row0 + 128 * i + (int32_t)r;
        const bool valid = row < w.n_rows;
        int32_t lo = 0, hi = 0;
        const int32_t place = w.rq.length - w.rq.n_new + row / (int32_t)p.group;
        if (valid) visible(place, w.rq.length, p.causal, p.window, lo, hi);
        const float c = p.scale_log2;
        float m = -INFINITY, l = 0.f;   // running maximum (of S), sum
        bool ok = true;
        // half-steps of 64 keys
        for (int32_t g = first; g < last; ++g) {
            const uint32_t h = g & 1, done = (uint32_t)(g - first), parity = done >> 1 & 1u;
            if (!(ok = wait(s_full(i, h), parity))) break;
            tc_fence_after();
            float s[64];
            tmem_ld32_nowait(t_s + h * 64, s);
            tmem_ld32_nowait(t_s + h * 64 + 32, s + 32);
            tmem_wait_ld();
            const int32_t a = lo - g * 64, z = hi - g * 64;   // seen: a <= k < z
            if (__builtin_expect(__any_sync(0xffffffffu, a > 0 || z < 64), 0)) {
#pragma unroll
                for (int k = 0; k < 64; ++k)
                    if (k < a || k >= z) s[k] = -INFINITY;
            }
            const float top = top_of(s);
            const bool grow = m == -INFINITY ? top > m : (top - m) * c > kLazy;
            if (__builtin_expect(__any_sync(0xffffffffu, grow), 0)) {
                const float m_new = grow ? top : m;
                const float alpha = grow ? ex2((m - m_new) * c) : 1.f;
                m = m_new;
                l *= alpha;
                if (done) {
                    // the half-step before has been added to O
                    if (!(ok = wait(pv_done(i, h ^ 1), (done - 1) >> 1 & 1u))) break;
                    tc_fence_after();
#pragma unroll 1
                    for (int k = 0; k < DP; k += 16) {
                        float o[16];
                        tmem_ld16(t_o + k, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[e] *= alpha;
                        tmem_st16(t_o + k, reinterpret_cast<uint32_t *>(o));
                    }
                }
            }
            uint64_t sum2[2] = {0, 0};
            uint32_t pk[32];
            exps<BF16, 64>(s, f2splat(c), f2splat(m == -INFINITY ? 0.f : -m * c), pk, sum2);
            tmem_st32(t_s + h * 64, pk);
            float s0, s1, s2, s3;
            f2unpack(sum2[0], s0, s1);
            f2unpack(sum2[1], s2, s3);
            l += (s0 + s1) + (s2 + s3);
            tmem_wait_st();
            tc_fence_before();
            warp_arrive(p_full(i, h));
        }
        // ---- results of the row
        const bool any = first < last;
        if (any && ok) ok = wait(pv_done(i, (last - 1) & 1), (uint32_t)(last - 1 - first) >> 1 & 1u);
        if (!ok && lane == 0) atomicOr(p.status, kStatusTimeout);
        tc_fence_after();
        const uint64_t token = (uint64_t)w.rq.first + row / (int32_t)p.group;
        const uint32_t head = w.h * p.group + row % (int32_t)p.group;
        uint16_t *out = p.out + token * p.ld_out_token + head * p.ld_out_head;
        if (ok) {
            const float inv = l == 0.f ? 0.f : 1.f / l;   // (a NaN sum stays one)
            if (w.n_split == 1 && valid && p.lse)
                p.lse[token * (p.n_kv * p.group) + head] =
                    l == 0.f ? -INFINITY : (m * c + log2f(l)) * 0.693147180559945309f;
            float *po = p.ws + p.ws_ml + (uint64_t)w.part * DP * kChunkRows + 128 * i + r;
            if (w.n_split > 1)
                __stcg(reinterpret_cast<float2 *>(p.ws) + (uint64_t)w.part * kChunkRows + 128 * i + r,
                       make_float2(m * c, l));
#pragma unroll
            for (uint32_t k = 0; k < DP; k += 32) {
                float o[32] = {};
                if (any) {
                    tmem_ld32_nowait(t_o + k, o);
                    tmem_wait_ld();
                }
                if (w.n_split > 1) {
#pragma unroll
                    for (uint32_t e = 0; e < 32; ++e) __stcg(po + (uint64_t)(k + e) * kChunkRows, o[e]);
                } else if (valid) {
                    if (l == 0.f)
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0.f;
                    store_row32<BF16>(p, out, k, o, inv);
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::tmem_cols));
    }
}

constexpr uint32_t kJoinRows = 32;

// Adds the shares of 32 rows in order.  A warp takes DP / 8 columns, a lane a
// row, so that every load is a whole line of the column-major partial results.
// (Joined by the CTA that finished last, 16 shares of one block took 45 us.)
template <int DP, bool BF16>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ AttnParams p) {
    constexpr uint32_t cols = DP / 8;
    __shared__ float2 stat[kChunkShares][kJoinRows];   // maximum and sum of a share's rows
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, r = blockIdx.y * kJoinRows + lane;
    Work w;
    if (!find_work(p, blockIdx.x / p.n_kv, blockIdx.x % p.n_kv, 0, w) || w.n_split == 1) return;
    const float2 *ml = reinterpret_cast<const float2 *>(p.ws) + (uint64_t)w.part * kChunkRows + r;
    for (uint32_t s = warp; s < w.n_split; s += 8) stat[s][lane] = ml[(uint64_t)s * kChunkRows];
    __syncthreads();
    const int32_t row = w.row0 + (int32_t)r;
    if (row >= w.n_rows) return;
    float m = -INFINITY, l = 0.f;
    for (uint32_t s = 0; s < w.n_split; ++s) m = fmaxf(m, stat[s][lane].x);
    const float base = m == -INFINITY ? 0.f : m;
    const float *po = p.ws + p.ws_ml + ((uint64_t)w.part * DP + warp * cols) * kChunkRows + r;
    float acc[cols] = {};
#pragma unroll 2
    for (uint32_t s = 0; s < w.n_split; ++s) {
        const float2 v = stat[s][lane];
        const float a = v.y == 0.f ? 0.f : ex2(v.x - base);   // (a share that saw nothing has written nothing)
        l += a * v.y;
#pragma unroll
        for (uint32_t e = 0; e < cols; ++e) {
            const float x = po[((uint64_t)s * DP + e) * kChunkRows];
            acc[e] = v.y == 0.f ? acc[e] : fmaf(a, x, acc[e]);
        }
    }
    const uint64_t token = (uint64_t)w.rq.first + row / (int32_t)p.group;
    const uint32_t head = w.h * p.group + row % (int32_t)p.group;
    if (p.lse && warp == 0)
        p.lse[token * (p.n_kv * p.group) + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t *o = p.out + token * p.ld_out_token + head * p.ld_out_head;
#pragma unroll
    for (uint32_t e = 0; e < cols; e += 8) {
        const uint32_t d = warp * cols + e;
        if (d >= p.head_dim) break;
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) u[k] = pack16<BF16>(acc[e + 2 * k] * inv, acc[e + 2 * k + 1] * inv);
        if (p.out_wide) {
            *reinterpret_cast<uint4 *>(o + d) = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                o[d + 2 * k] = (uint16_t)u[k];
                o[d + 2 * k + 1] = (uint16_t)(u[k] >> 16);
            }
        }
    }
}

template <int DP, bool BF16>
cudaError_t launch_inst(const CUtensorMap &km, const CUtensorMap &vm, const AttnParams &p, cudaStream_t s) {
    using L = ChunkLayout<DP>;
    auto kernel = chunk_kernel<DP, BF16>;
    static DeviceCache cache;
    int unused = 0;
    cudaError_t e = per_device(cache, unused, [&](int &) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::bytes);
    });
    if (e != cudaSuccess) return e;
    kernel<<<p.n_blocks * p.n_kv * p.splits, kThreads, L::bytes, s>>>(km, vm, p);
    if (p.splits > 1)
        join_kernel<DP, BF16><<<dim3(p.n_blocks * p.n_kv, kChunkRows / kJoinRows), 256, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_chunk(const CUtensorMap &km, const CUtensorMap &vm, const AttnParams &p, bool bf16,
                         cudaStream_t s) {
    if (p.head_dim <= 64) return bf16 ? launch_inst<64, true>(km, vm, p, s) : launch_inst<64, false>(km, vm, p, s);
    return bf16 ? launch_inst<128, true>(km, vm, p, s) : launch_inst<128, false>(km, vm, p, s);
}

}  // namespace tc
