// Paged attention of many rows (chunks, whole prompts, image tokens) on the
// 5th-generation tensor cores (sm_100a).
//
// A CTA takes 256 rows (the query heads of one cache head packed with the
// tokens, see attn_paged.cu) as two 128-row tiles and walks the keys that they
// see in steps of 128:
//   S_i = Q_i K^T           tcgen05.mma, both operands in shared memory, S in TMEM
//   P_i = 2^(c S_i - c m)   one thread per row (two warpgroups, one per tile)
//   O_i += P_i V            tcgen05.mma, P_i in TMEM (over S_i), V in shared
//                           memory as it lies in the cache (MN-major operand)
// Four 128 x 128 x 128 products a step (2048 tensor cycles at head_dim 128)
// against 32768 exponentials (2048 cycles of the special-function units), so
// the tile not being exponentiated keeps the tensor cores busy: the issuing
// thread orders PV_0(j), S_0(j+1), PV_1(j), S_1(j+1), and a commit behind
// S_i(j+1) also covers PV_i(j), so the warpgroup that finds S_i(j+1) complete
// may rescale O_i itself.  That happens only when a row's maximum has grown by
// more than 2^8 since the last time (P then stays below 256, exact enough in
// either 16-bit type), i.e. seldom after the first steps.
//
//   warps 0-3, 4-7   softmax of tile 0 / 1, epilogue
//   warp 8           TMA producer: K and V tiles of 128 keys through a ring of
//                    stages, one box per page piece and 64-element half, the
//                    boxes of a tile issued by the warp's lanes in parallel
//   warps 10, 11     nothing (they complete the warpgroup that gives up registers)
//   warp 9           TMEM allocation, MMA issue; zeroes the rows of V outside
//                    the keys seen in the first and last step (their bytes are
//                    whatever the page holds there, and 0 * NaN is NaN)
//
// TMEM: S_0, S_1 (128 columns each), O_0, O_1 (head_dim each).  Blocks of rows
// go heaviest first (last rows first).  With few blocks the keys are split
// over CTAs: partial results (column-major, so that the 128 threads of a tile
// store and load whole lines) and the last to finish joins them in order.
//
// Every wait is bounded; on timeout the kernel sets TC_STATUS_TIMEOUT, drains
// its copies and MMAs, frees TMEM and returns.  No multicast.
#include "attn_kernels.cuh"

namespace tc {
namespace {

constexpr int kThreads = 384;
// Registers of a thread: 384 threads launch with 168; the warpgroup of the
// producer and the issuer gives up what the softmax warpgroups (which hold 128
// scores) take.
constexpr int kSoftmaxRegs = 216, kOtherRegs = 72, kLaunchRegs = 168;
static_assert(256 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs, "the shares exceed the launch's registers");
constexpr float kLazy = 8.f;   // log2 of the growth of a maximum that is let pass

template <int DP>
struct ChunkLayout {
    static constexpr uint32_t halves = DP / 64;
    static constexpr uint32_t half_bytes = 128 * 128;            // 128 rows x 64 elements
    static constexpr uint32_t tile_bytes = halves * half_bytes;  // Q tile, K tile, V tile
    static constexpr uint32_t stages = DP == 128 ? 5 : 8;
    static constexpr uint32_t q_off = 0, kv_off = 2 * tile_bytes;
    static constexpr uint32_t bar_off = kv_off + stages * tile_bytes;
    // kv_full[S] kv_empty[S] s_full[2] p_full[2] o_full[2] q_full fin
    static constexpr uint32_t misc_off = bar_off + (2 * stages + 8) * 8;
    static constexpr uint32_t bytes = misc_off + 16 + 1024;
    static constexpr uint32_t s_col = 0, o_col = 256, tmem_cols = 512;
    static_assert(bytes <= 232448, "shared memory per CTA exceeds the sm_100 limit");
};

// bar_wait without a call (a call would fix the caller's registers below the
// softmax warpgroups' share).
__device__ __forceinline__ bool wait(uint32_t b, uint32_t parity, volatile uint32_t *abort_flag, uint32_t *status,
                                     bool honor_abort = true) {
    if (bar_try(b, parity)) return true;
    const uint64_t t0 = gtimer();
    for (;;) {
        if (bar_try_sleep(b, parity, 20000u)) return true;
        if (honor_abort && *abort_flag) return false;
        if (gtimer() - t0 > kTimeoutNs) {
            atomicOr(status, kStatusTimeout);
            *abort_flag = 1u;
            return false;
        }
    }
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

// Barrier of the 256 softmax threads.
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// What a CTA works on; the same in every thread.
struct Work {
    Request rq;
    uint32_t b, h, part, group_index, n_split, split;
    int32_t row0, n_rows;
    int32_t lo[2], hi[2];     // keys that tile i's rows see, within the CTA's share
    int32_t first[2], last[2];   // its steps (tile i has none: first == last)
    int32_t begin, end;       // steps of the CTA (keys 128 step ..)
};

__device__ __forceinline__ bool find_work(const AttnParams &p, Work &w) {
    uint32_t id = blockIdx.x;
    w.h = id % p.n_kv;
    id /= p.n_kv;
    w.split = id % p.splits;
    const uint32_t blk = p.n_blocks - 1 - id / p.splits;
    // Request b's blocks begin at first(b) = rows before it / 256 + b: that
    // leaves room for its partly filled one.
    auto first_block = [&](uint32_t b) {
        return (int64_t)p.batch.new_offsets[b] * p.group / kChunkRows + b;
    };
    w.b = count_prefix(p.batch.n_seq - 1, [&](uint32_t b) { return first_block(b) <= (int64_t)blk; });
    w.rq = load_request(p.batch, p.page_shift, w.b, p.status);
    w.n_rows = w.rq.n_new * (int32_t)p.group;
    const int64_t row0 = ((int64_t)blk - first_block(w.b)) * kChunkRows;
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
            w.first[i] = w.last[i] = w.begin;
        } else {
            w.first[i] = w.lo[i] / kChunkKeys;
            w.last[i] = (w.hi[i] + kChunkKeys - 1) / kChunkKeys;
        }
    }
    w.group_index = blk * p.n_kv + w.h;
    w.part = w.group_index * p.splits + w.split;
    return true;
}

// Normalised elements [c0, c0 + 32) of a row.
template <bool BF16>
__device__ __forceinline__ void store_row32(const AttnParams &p, uint16_t *o, uint32_t c0, const float *v, float inv) {
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = pack16<BF16>(v[2 * i] * inv, v[2 * i + 1] * inv);
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
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    Work w;
    if (!find_work(p, w)) return;
    const uint32_t bars = su32(smem + L::bar_off);
    auto kv_full = [&](uint32_t i) { return bars + 8 * i; };
    auto kv_empty = [&](uint32_t i) { return bars + 8 * (L::stages + i); };
    auto s_full = [&](uint32_t i) { return bars + 8 * (2 * L::stages + i); };
    auto p_full = [&](uint32_t i) { return bars + 8 * (2 * L::stages + 2 + i); };
    auto o_full = [&](uint32_t i) { return bars + 8 * (2 * L::stages + 4 + i); };
    const uint32_t q_full = bars + 8 * (2 * L::stages + 6), fin = q_full + 8;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::misc_off);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    uint32_t *last_flag = tmem_slot + 2;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < L::stages; ++i) {
            bar_init(kv_full(i), 1);
            bar_init(kv_empty(i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(s_full(i), 1);
            bar_init(p_full(i), 128);
            bar_init(o_full(i), 1);
        }
        bar_init(q_full, 256);
        bar_init(fin, 1);
        *abort_flag = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(su32(tmem_slot)), "r"(L::tmem_cols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 8) {
        // ---------------------------------------------------- TMA producer
        const uint32_t box = min((uint32_t)kChunkKeys, 1u << p.page_shift), pieces = kChunkKeys / box;
        const uint32_t piece = lane % pieces, half0 = lane / pieces;   // lanes: 32 / pieces halves at a time
        const int32_t key_end = max(w.hi[0], w.hi[1]);
        uint32_t st = 0, ph = 0, issued = 0;
        for (int32_t j = w.begin; j < w.end; ++j) {
            // this lane's page piece of the step
            const int32_t pos = j * kChunkKeys + (int32_t)(piece * box);
            const bool on = pos < key_end;
            int32_t page = 0;
            if (on) page = max(load_page(p.batch, p.n_pages, w.b, (uint32_t)pos >> p.page_shift, p.status), 0);
            const int token = (int)((uint32_t)pos & ((1u << p.page_shift) - 1));
            const uint32_t n_on = min(pieces, (uint32_t)(key_end - j * kChunkKeys + (int32_t)box - 1) / box);
            bool ok = true;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                ok = wait(kv_empty(st), ph ^ 1, abort_flag, p.status);
                if (!(ok = __all_sync(0xffffffffu, ok))) break;
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
        if (lane == 0)
            // every copy issued has landed before exit
            for (uint32_t n = issued > L::stages ? issued - L::stages : 0; n < issued; ++n)
                wait(kv_full(n % L::stages), (n / L::stages) & 1u, abort_flag, p.status, false);
        __syncwarp();
        } else if (warp == 9) {
        // ---------------------------------------------------- MMA issuer
        constexpr uint32_t idesc_s = mma_idesc<128, !BF16>();
        constexpr uint32_t idesc_o = mma_idesc<DP, !BF16>() | (1u << 16);   // B is MN-major
        const uint32_t q_addr = su32(smem + L::q_off), kv_addr = su32(smem + L::kv_off);
        // ring positions of K and V of step j: 2 (j - begin) and one more
        auto stage_of = [&](uint32_t n) { return n % L::stages; };
        auto phase_of = [&](uint32_t n) { return (n / L::stages) & 1u; };
        auto wait_kv = [&](uint32_t n) {
            return __all_sync(0xffffffffu, wait(kv_full(stage_of(n)), phase_of(n), abort_flag, p.status));
        };
        const uint32_t q_low = desc_low(q_addr, 1), k_low = desc_low(kv_addr, 1);
        const uint32_t v_low = desc_low(kv_addr, L::half_bytes >> 4);
        auto issue_s = [&](int i, uint32_t n) {
            if (lane == 0) {
                const uint32_t q = q_low + i * (L::tile_bytes >> 4), k = k_low + stage_of(n) * (L::tile_bytes >> 4);
#pragma unroll
                for (uint32_t kk = 0; kk < DP / 16; ++kk) {
                    const uint32_t off = ((kk / 4) * L::half_bytes + (kk % 4) * 32) >> 4;
                    mma_f16(tmem + L::s_col + i * 128, desc(q + off), desc(k + off), idesc_s, kk ? 1u : 0u);
                }
                mma_commit(s_full(i));
            }
        };
        const int32_t seen_lo = min(w.first[0] < w.last[0] ? w.lo[0] : 0x7fffffff,
                                    w.first[1] < w.last[1] ? w.lo[1] : 0x7fffffff);
        const int32_t seen_hi = max(w.hi[0], w.hi[1]);
        bool ok = __all_sync(0xffffffffu, wait(q_full, 0, abort_flag, p.status));
        tc_fence_after();
        uint32_t n = 0;   // ring position of K(j)
        if (ok && w.begin < w.end) {
            ok = wait_kv(0);
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (ok && w.first[i] == w.begin && w.first[i] < w.last[i]) issue_s(i, 0);
            if (ok && lane == 0) mma_commit(kv_empty(0));
        }
        for (int32_t j = w.begin; ok && j < w.end; ++j, n += 2) {
            ok = wait_kv(n + 1);
            const int32_t key0 = j * kChunkKeys;
            if (ok && (key0 < seen_lo || key0 + kChunkKeys > seen_hi)) {
                const uint32_t v = kv_addr + stage_of(n + 1) * L::tile_bytes;
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
                __syncwarp();
            }
            bool waited = false;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!ok) break;
                if (j >= w.first[i] && j < w.last[i]) {
                    ok = __all_sync(0xffffffffu,
                                    wait(p_full(i), (uint32_t)(j - w.first[i]) & 1u, abort_flag, p.status));
                    if (!ok) break;
                    tc_fence_after();
                    if (lane == 0) {
                        const uint32_t v = v_low + stage_of(n + 1) * (L::tile_bytes >> 4);
#pragma unroll
                        for (uint32_t kk = 0; kk < kChunkKeys / 16; ++kk)
                            mma_f16_ts(tmem + L::o_col + i * DP, tmem + L::s_col + i * 128 + kk * 8,
                                       desc(v + kk * (2048 >> 4)), idesc_o, j > w.first[i] || kk ? 1u : 0u);
                        if (j + 1 == w.last[i]) mma_commit(o_full(i));
                    }
                }
                if (j + 1 >= w.first[i] && j + 1 < w.last[i]) {
                    if (!waited) {
                        ok = wait_kv(n + 2);
                        if (!ok) break;
                        tc_fence_after();
                        waited = true;
                    }
                    issue_s(i, n + 2);
                }
            }
            if (ok && j + 1 < w.end && !waited) ok = wait_kv(n + 2);
            if (ok && lane == 0) {
                mma_commit(kv_empty(stage_of(n + 1)));
                if (j + 1 < w.end) mma_commit(kv_empty(stage_of(n + 2)));
            }
        }
        if (lane == 0) {
            mma_commit(fin);   // every MMA issued has completed before TMEM is freed
            wait(fin, 0, abort_flag, p.status, false);
        }
        __syncwarp();
        }
    } else {
        // ---------------------------------------------------- softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int i = warp / 4;
        const int32_t first = i ? w.first[1] : w.first[0], last = i ? w.last[1] : w.last[0];
        // queries of both tiles: DP / 8 16-byte pieces a row, all 256 threads
        {
            constexpr uint32_t per = DP / 8;
            for (uint32_t c = threadIdx.x; c < 256 * per; c += 256) {
                const uint32_t r = c / per, x = c % per;
                const int32_t row = w.row0 + (int32_t)r;
                uint32_t v[4] = {};
                if (row < w.n_rows && x * 8 < p.head_dim) {
                    const uint16_t *q = p.q + (uint64_t)(w.rq.first + row / (int32_t)p.group) * p.ld_q_token +
                                        (uint64_t)(w.h * p.group + row % (int32_t)p.group) * p.ld_q_head + x * 8;
                    if (p.q_wide) {
                        const uint4 u = *reinterpret_cast<const uint4 *>(q);
                        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
                    } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] = (uint32_t)q[2 * k] | (uint32_t)q[2 * k + 1] << 16;
                    }
                    if (p.negate_q)
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] ^= 0x80008000u;
                }
                const uint32_t dst = su32(smem + L::q_off) + (r / 128) * L::tile_bytes + (x / 8) * L::half_bytes +
                                     (r % 128) * 128 + (((x % 8) ^ (r % 8)) << 4);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                             ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
            }
            fence_proxy_async();
            bar_arrive(q_full);
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
        for (int32_t j = first; j < last; ++j) {
            ok = wait(s_full(i), (uint32_t)(j - first) & 1u, abort_flag, p.status);
            if (!(ok = __all_sync(0xffffffffu, ok))) break;
            tc_fence_after();
            float s[128];
#pragma unroll
            for (int k = 0; k < 4; ++k) tmem_ld32_nowait(t_s + 32 * k, s + 32 * k);
            tmem_wait_ld();
            const int32_t a = lo - j * kChunkKeys, z = hi - j * kChunkKeys;   // seen: a <= column < z
            if (__any_sync(0xffffffffu, a > 0 || z < kChunkKeys)) {
#pragma unroll
                for (int k = 0; k < 128; ++k)
                    if (k < a || k >= z) s[k] = -INFINITY;
            }
            float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int k = 4; k < 128; k += 4) {
                mx[0] = fmaxf(mx[0], s[k]);
                mx[1] = fmaxf(mx[1], s[k + 1]);
                mx[2] = fmaxf(mx[2], s[k + 2]);
                mx[3] = fmaxf(mx[3], s[k + 3]);
            }
            const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
            const bool grow = m == -INFINITY ? top > m : (top - m) * c > kLazy;
            if (__any_sync(0xffffffffu, grow)) {
                const float m_new = grow ? top : m;
                const float alpha = grow ? ex2((m - m_new) * c) : 1.f;
                m = m_new;
                l *= alpha;
                if (j > first) {
#pragma unroll
                    for (int k = 0; k < DP; k += 32) {
                        float o[32];
                        tmem_ld32_nowait(t_o + k, o);
                        tmem_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] *= alpha;
                        tmem_st32(t_o + k, reinterpret_cast<uint32_t *>(o));
                    }
                }
            }
            const float off = m == -INFINITY ? 0.f : -m * c;
            const uint64_t c2 = f2splat(c), off2 = f2splat(off);
            uint64_t sum2[2] = {0, 0};
#pragma unroll
            for (int k0 = 0; k0 < 128; k0 += 64) {
                uint32_t pk[32];
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    const uint64_t x = f2fma(f2pack(__float_as_uint(s[k0 + k]), __float_as_uint(s[k0 + k + 1])), c2, off2);
                    float e0, e1;
                    f2unpack(x, e0, e1);
                    e0 = ex2(e0);
                    e1 = ex2(e1);
                    pk[k / 2] = pack16<BF16>(e0, e1);
                    sum2[(k / 2) & 1] = f2add(sum2[(k / 2) & 1], f2pack(__float_as_uint(e0), __float_as_uint(e1)));
                }
                tmem_st32(t_s + k0 / 2, pk);
            }
            float s0, s1, s2, s3;
            f2unpack(sum2[0], s0, s1);
            f2unpack(sum2[1], s2, s3);
            l += (s0 + s1) + (s2 + s3);
            tmem_wait_st();
            tc_fence_before();
            bar_arrive(p_full(i));
        }
        // ---- results of the row
        const bool any = first < last;
        if (any && ok) ok = __all_sync(0xffffffffu, wait(o_full(i), 0, abort_flag, p.status));
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
#pragma unroll 1
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
        if (w.n_split > 1) {
            // ---- the share that finishes last adds them all, in order
            __threadfence();
            softmax_sync();
            if (threadIdx.x == 0) {
                const uint32_t before = atomicAdd(p.counters + w.group_index, 1u);
                *last_flag = before + 1 == w.n_split;
                if (before + 1 == w.n_split) p.counters[w.group_index] = 0u;
            }
            softmax_sync();
            if (*last_flag && valid) {
            __threadfence();
            const uint64_t part0 = (uint64_t)w.group_index * p.splits;
            const float2 *ml = reinterpret_cast<const float2 *>(p.ws) + part0 * kChunkRows + threadIdx.x;
            const float *po = p.ws + p.ws_ml + part0 * DP * kChunkRows + threadIdx.x;
            float mm = -INFINITY, ll = 0.f;
            for (uint32_t s = 0; s < w.n_split; ++s) mm = fmaxf(mm, __ldcg(ml + (uint64_t)s * kChunkRows).x);
            const float base = mm == -INFINITY ? 0.f : mm;
            for (uint32_t s = 0; s < w.n_split; ++s) {
                const float2 v = __ldcg(ml + (uint64_t)s * kChunkRows);
                ll += ex2(v.x - base) * v.y;
            }
            if (p.lse)
                p.lse[token * (p.n_kv * p.group) + head] =
                    ll == 0.f ? -INFINITY : (mm + log2f(ll)) * 0.693147180559945309f;
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
        #pragma unroll 1
            for (uint32_t k = 0; k < DP; k += 32) {
                float acc[32] = {};
                for (uint32_t s = 0; s < w.n_split; ++s) {
                    const float2 v = __ldcg(ml + (uint64_t)s * kChunkRows);
                    const float a = ex2(v.x - base);
                    if (v.y == 0.f) continue;   // it saw nothing (a NaN sum is kept)
        #pragma unroll
                    for (uint32_t e = 0; e < 32; ++e)
                        acc[e] = fmaf(a, __ldcg(po + ((uint64_t)s * DP + k + e) * kChunkRows), acc[e]);
                }
                store_row32<BF16>(p, out, k, acc, inv);
            }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(L::tmem_cols));
    }
}

template <int DP, bool BF16>
cudaError_t launch_inst(const CUtensorMap &km, const CUtensorMap &vm, const AttnParams &p, cudaStream_t s) {
    using L = ChunkLayout<DP>;
    auto kernel = chunk_kernel<DP, BF16>;
    static DeviceCache cache;
    int unused = 0;
    cudaError_t e = per_device(cache, unused, [&](int &) {
        // the registers that the warpgroups share out must have been launched
        cudaFuncAttributes attr{};
        const cudaError_t q = cudaFuncGetAttributes(&attr, kernel);
        if (q != cudaSuccess) return q;
        if (attr.numRegs != kLaunchRegs) return cudaErrorInvalidKernelImage;
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::bytes);
    });
    if (e != cudaSuccess) return e;
    kernel<<<p.n_blocks * p.n_kv * p.splits, kThreads, L::bytes, s>>>(km, vm, p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_chunk(const CUtensorMap &km, const CUtensorMap &vm, const AttnParams &p, bool bf16,
                         cudaStream_t s) {
    if (p.head_dim <= 64) return bf16 ? launch_inst<64, true>(km, vm, p, s) : launch_inst<64, false>(km, vm, p, s);
    return bf16 ? launch_inst<128, true>(km, vm, p, s) : launch_inst<128, false>(km, vm, p, s);
}

}  // namespace tc
