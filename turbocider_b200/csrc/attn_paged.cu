// Attention of a step's new tokens over a paged cache
// (tc_cuda_paged_attention): out = softmax(scale q K^T) V.
//
// The query heads that share a cache head are packed with the request's new
// tokens into rows (row r: token r / group, head r % group), so K and V are
// read once for all of them.  This file has the kernel for few rows (single
// tokens, a few drafted ones): bytes bound, the floor is one read of K and V.
//
// A CTA takes up to 16, 32 or 64 rows (mma.sync tiles of 16; with so few rows the
// tensor work is a small part of the memory time, so the padding costs nothing)
// of one cache head and one chunk of the cache; its four warps take steps of 16
// or 32 keys in turn, each with its own running maximum, sum and output in
// registers, so the loop has no CTA-wide synchronisation.  Each warp keeps a
// ring of TMA boxes in flight (64 elements x up to a step's tokens of a page,
// 128-byte swizzle, conflict-free for ldmatrix), a lane issuing each.  The warps'
// results are joined in shared memory, the chunks' by the CTA that finishes last
// (partial outputs in the workspace, added in chunk order, so the result does
// not depend on timing).
//
// A decode step of 96 requests, 1.5 GB of cache: 235 us, 6.52 TB/s (99 % of the
// measured copy).  One token over 3001 positions (12 MB): 9.9 us, bound by one
// CTA's chain: 0.9 us to its pages, 2 us to the first keys, 2 us of steps, 0.6 us to
// join the warps, 1 us for the arrival, 1.5 us to add the shares.
//
// Probabilities are rounded to the cache's 16-bit type for the P V product
// (its relative error, 2^-9 or 2^-12 an element, averages out over the keys);
// their sum is taken before the rounding.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "attn.cuh"
#include "attn_kernels.cuh"

namespace tc {
namespace {

// Keys of a warp's step: 32 for heads of up to 64, where 16 leave too little
// between two waits (with the queries' loads, 23 requests by up to
// 28 rows: 33 -> 20 us).
constexpr int step_keys(int dp, int mt) { return dp == 64 && mt <= 2 ? 32 : 16; }
constexpr int kWarps = 4;
constexpr uint32_t kMaxChunk = 1024;
// CTAs that an SM has room for: by the rings for 16 rows (heads of 256 need 128 KB
// for two stages), by the registers of 32 and 64 rows (all 255 of them with 64,
// where 256 bytes a thread spill).
constexpr int ctas_per_sm(int dp, int mt) { return dp == 256 ? 1 : mt == 1 ? 3 : 2; }

// Rows of a CTA: MT mma tiles of 16.
template <int DP, int MT>
struct FewLayout {
    static constexpr int halves = DP / 64;
    static constexpr int rows = 16 * MT;
    static constexpr int keys = step_keys(DP, MT);
    static constexpr uint32_t kv_bytes = keys * DP * 2;       // K of a step; V follows
    static constexpr uint32_t stage = 2 * kv_bytes;
    // 64 KB of rings (128 for heads of 256).  (Three stages and two CTAs an SM kept
    // as much in flight as two and three but took 265 us, not 245, for 1.5 GB of
    // cache.)
    static constexpr int stages = DP == 64 && keys == 16 ? 4 : 2;
    static constexpr uint32_t ring = stages * stage;           // per warp
    static constexpr uint32_t q_off = kWarps * ring;           // queries: rows x DP, 16-byte pieces swizzled by row
    static constexpr uint32_t bar_off = q_off + rows * DP * 2;
    static constexpr uint32_t page_off = bar_off + kWarps * stages * 8;
    static constexpr uint32_t ml_off = page_off + (kMaxChunk / 8 + 2) * 4;   // [warp][row][m, l]
    static constexpr uint32_t misc_off = ml_off + kWarps * rows * 8;
    static constexpr uint32_t bytes = misc_off + 16 + 1024;
    static constexpr int places = ctas_per_sm(DP, MT);
    static_assert(places * (bytes + 1024) <= 233472, "the CTAs of an SM share its memory");
    static_assert(kWarps * ring >= kWarps * rows * DP * 4, "the join reuses the rings");
    static constexpr uint32_t max_shares = kWarps * ring / (rows * 8);   // whose statistics fit there too
};

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool TRANS>
__device__ __forceinline__ void ldsm4(uint32_t (&v)[4], uint32_t addr) {
    if (TRANS)
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
    else
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr) : "memory");
}

// Adds the n_split shares of a tile in order and stores its rows.  R: rounds of
// 128 threads x 4 elements that the rows take.
template <int DP, int MT, bool BF16, int R>
__device__ __forceinline__ void join_shares(const AttnParams &p, const Request &rq, uint32_t h, uint32_t tile,
                                            int32_t row0, uint32_t rows, uint32_t n_split, float2 *part, float2 *ml) {
    using L = FewLayout<DP, MT>;
    constexpr uint32_t quads = DP / 4, threads = kWarps * 32;
    const float2 *mls = reinterpret_cast<const float2 *>(p.ws) + (uint64_t)tile * p.splits * p.ws_rows;
    const float *os = p.ws + p.ws_ml + (uint64_t)tile * p.splits * p.ws_rows * DP;
    // `part` [share][row] (shared memory): maximum, then weight; sum.  The
    // statistics first, a few threads per row; the first shares' outputs need no
    // weight to travel and are on their way meanwhile.
    constexpr uint32_t lanes = threads / L::rows, ahead = R == 1 ? 8 : 8 / R > 1 ? 8 / R : 1;
    constexpr uint32_t together = R == 1 ? 16 : 16 / R > 1 ? 16 / R : 1;   // shares in flight after them
    auto output = [&](uint32_t s, uint32_t k) {
        const uint32_t e = min(threadIdx.x + k * threads, rows * quads - 1);
        return __ldcg(reinterpret_cast<const float4 *>(
            os + ((uint64_t)min(s, n_split - 1) * p.ws_rows + e / quads) * DP + (e % quads) * 4));
    };
    float4 first[ahead][R];
#pragma unroll
    for (uint32_t s = 0; s < ahead; ++s)
#pragma unroll
        for (uint32_t k = 0; k < R; ++k) first[s][k] = output(s, k);
    const uint32_t r = threadIdx.x / lanes, s0 = threadIdx.x % lanes;
    float mm = -INFINITY, ll = 0.f;
    if (r < rows) {
#pragma unroll 4
        for (uint32_t s = s0; s < n_split; s += lanes) {
            const float2 v = __ldcg(mls + (uint64_t)s * p.ws_rows + r);
            part[s * L::rows + r] = v;
            mm = fmaxf(mm, v.x);
        }
    }
#pragma unroll
    for (uint32_t d = lanes / 2; d > 0; d /= 2) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, d));
    if (r < rows) {
        for (uint32_t s = s0; s < n_split; s += lanes) {
            const float2 v = part[s * L::rows + r];
            const float a = v.x == -INFINITY ? 0.f : exp2f(v.x - mm);
            part[s * L::rows + r].x = a;
            ll += a * v.y;
        }
    }
#pragma unroll
    for (uint32_t d = lanes / 2; d > 0; d /= 2) ll += __shfl_xor_sync(0xffffffffu, ll, d);
    if (s0 == 0 && r < rows) ml[r] = make_float2(mm, ll);
    __syncthreads();
    float4 acc[R] = {};
    auto add = [&](uint32_t s, uint32_t k, const float4 &x) {
        const uint32_t e = min(threadIdx.x + k * threads, rows * quads - 1);
        const float a = part[s * L::rows + e / quads].x;
        acc[k].x += a * x.x;
        acc[k].y += a * x.y;
        acc[k].z += a * x.z;
        acc[k].w += a * x.w;
    };
#pragma unroll
    for (uint32_t s = 0; s < ahead; ++s)
        if (s < n_split)
#pragma unroll
            for (uint32_t k = 0; k < R; ++k) add(s, k, first[s][k]);
    for (uint32_t f = ahead; f < n_split; f += together) {
        float4 x[together][R];
#pragma unroll
        for (uint32_t s = 0; s < together; ++s)
#pragma unroll
            for (uint32_t k = 0; k < R; ++k) x[s][k] = output(f + s, k);
#pragma unroll
        for (uint32_t s = 0; s < together; ++s)
            if (f + s < n_split)
#pragma unroll
                for (uint32_t k = 0; k < R; ++k) add(f + s, k, x[s][k]);
    }
#pragma unroll
    for (uint32_t k = 0; k < R; ++k) {
        const uint32_t e = threadIdx.x + k * threads;
        if (e < rows * quads)
            store_row4<BF16>(p, rq, h, row0 + (int32_t)(e / quads), (e % quads) * 4, acc[k], ml[e / quads].x,
                             ml[e / quads].y);
    }
}

template <int DP, int MT, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, ctas_per_sm(DP, MT))
    few_rows_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                    const __grid_constant__ AttnParams p) {
    using L = FewLayout<DP, MT>;
    constexpr int kKeys = L::keys;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t split = blockIdx.x, h = blockIdx.y, unit = p.first_unit + blockIdx.z;
    const uint32_t b = unit / p.row_tiles, rt = unit % p.row_tiles;
    volatile uint32_t *abort_flag = reinterpret_cast<uint32_t *>(smem + L::misc_off);
    uint32_t *last_flag = reinterpret_cast<uint32_t *>(smem + L::misc_off) + 1;
    const uint32_t bars = su32(smem + L::bar_off) + warp * L::stages * 8;
    if (threadIdx.x < 2)
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(threadIdx.x ? &vmap : &kmap)) : "memory");
    if (threadIdx.x == 0) *abort_flag = 0u;
    if (lane == 0)
        for (int i = 0; i < L::stages; ++i) bar_init(bars + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

    // The entry of the page list that this thread will want if the first key
    // is 0 (no window) travels with the request's values.
    uint32_t guess = (split * p.chunk >> p.page_shift) + threadIdx.x;
    int32_t guessed = -1;
    if (guess < p.batch.table_width && threadIdx.x <= p.chunk >> p.page_shift)
        guessed = p.batch.page_table[(uint64_t)b * p.batch.ld_table + guess];
    else
        guess = ~0u;
    const Request rq = load_request(p.batch, p.page_shift, b, p.status);
    const int32_t n_rows = rq.n_new * (int32_t)p.group, row0 = (int32_t)rt * L::rows;
    if (row0 >= n_rows) return;
    // keys that any row of the tile sees, and this CTA's share
    const int32_t place0 = rq.length - rq.n_new;
    const int32_t tok0 = row0 / (int32_t)p.group, tok1 = (min(row0 + L::rows, n_rows) - 1) / (int32_t)p.group;
    int32_t lo, hi, unused;
    visible(place0 + tok0, rq.length, p.causal, p.window, lo, unused);
    visible(place0 + tok1, rq.length, p.causal, p.window, unused, hi);
    const int32_t base = lo & ~(kKeys - 1);
    const uint32_t n_split = hi > lo ? (uint32_t)(hi - base + (int32_t)p.chunk - 1) / p.chunk : 1u;
    if (split >= n_split) return;
    if (n_split > p.splits) {   // the launch was sized for a shorter span
        if (threadIdx.x == 0) atomicOr(p.status, kStatusGeometry);
        return;
    }
    const int32_t begin = base + (int32_t)(split * p.chunk), end = hi > lo ? min(hi, begin + (int32_t)p.chunk) : begin;

    // ---- page numbers of the chunk, from the one with the first key seen on
    // (earlier ones may have been given back)
    int32_t *pages = reinterpret_cast<int32_t *>(smem + L::page_off);
    if (end > begin) {
        const uint32_t j0 = (uint32_t)begin >> p.page_shift, j1 = (uint32_t)(end - 1) >> p.page_shift;
        for (uint32_t j = ((uint32_t)max(begin, lo) >> p.page_shift) + threadIdx.x; j <= j1; j += kWarps * 32)
            pages[j - j0] = j == guess ? check_page(guessed, p.n_pages, p.status)
                                       : load_page(p.batch, p.n_pages, b, j, p.status);
    }

    __syncthreads();

    const uint32_t ring = su32(smem) + warp * L::ring;
    const int32_t steps = (end - begin + kKeys - 1) / kKeys;
    const uint32_t box = min((uint32_t)kKeys, 1u << p.page_shift);   // tokens of a TMA box
    // Loads of the warp's step i (16 keys from `key`), a lane for each box: K or
    // V, half, and page piece, of the pieces that begin before the chunk's end
    // and end behind the first key seen.
    const uint32_t box_half = lane / 2 % L::halves, box_piece = lane / 2 / L::halves;
    auto issue = [&](int32_t i, uint32_t st) {
        const int32_t key = begin + i * kKeys;
        const uint32_t pieces = min((uint32_t)kKeys / box, (uint32_t)(end - key + (int32_t)box - 1) / box);
        const uint32_t first = (uint32_t)max(lo - key, 0) / box;
        const uint32_t bar = bars + 8 * st;
        if (lane == 0) bar_expect_tx(bar, (pieces - first) * box * DP * 4);
        __syncwarp();
        if (box_piece >= first && box_piece < pieces) {
            const uint32_t pos = (uint32_t)key + box_piece * box;
            // (an impossible page is -1: a box outside the cache arrives as zeros)
            const int page = pages[(pos >> p.page_shift) - ((uint32_t)begin >> p.page_shift)];
            tma_load_4d(ring + st * L::stage + (lane & 1) * L::kv_bytes + box_half * (kKeys * 128) + box_piece * box * 128,
                        lane & 1 ? &vmap : &kmap, bar, (int)box_half * 64, (int)(pos & ((1u << p.page_shift) - 1)),
                        (int)h, page);
        }
    };
    for (int32_t s = 0; s < L::stages; ++s)
        if ((int32_t)warp + s * kWarps < steps) issue((int32_t)warp + s * kWarps, (uint32_t)s);

    // ---- queries through shared memory into row-major A fragments
    const uint32_t g = lane / 4, t4 = lane % 4;
    uint32_t qf[MT][DP / 16][4];
    {
        constexpr uint32_t per = DP / 8, rounds = L::rows * per / (kWarps * 32);
        uint32_t v[rounds][4];
#pragma unroll
        for (uint32_t k = 0; k < rounds; ++k) {
            const uint32_t c = threadIdx.x + k * kWarps * 32, x = c % per, row = (uint32_t)row0 + c / per;
            const uint32_t tok = row / p.group;
            const uint16_t *q = p.q + ((uint64_t)rq.first + tok) * p.ld_q_token +
                                (uint64_t)(h * p.group + row - tok * p.group) * p.ld_q_head + x * 8;
            const bool on = row < (uint32_t)n_rows && x * 8 < p.head_dim;
            if (p.q_wide) {
                const uint4 u = on ? *reinterpret_cast<const uint4 *>(q) : make_uint4(0u, 0u, 0u, 0u);
                v[k][0] = u.x; v[k][1] = u.y; v[k][2] = u.z; v[k][3] = u.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[k][e] = on ? (uint32_t)q[2 * e] | (uint32_t)q[2 * e + 1] << 16 : 0u;
            }
        }
        const uint32_t q_addr = su32(smem + L::q_off);
#pragma unroll
        for (uint32_t k = 0; k < rounds; ++k) {
            const uint32_t c = threadIdx.x + k * kWarps * 32, x = c % per, r = c / per;
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                         ::"r"(q_addr + r * (DP * 2) + ((x ^ (r & 7)) << 4)), "r"(v[k][0]), "r"(v[k][1]), "r"(v[k][2]),
                           "r"(v[k][3]) : "memory");
        }
        __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                const uint32_t r = mt * 16 + (lane & 15), x = ks * 2 + (lane >> 4);
                ldsm4<false>(qf[mt][ks], q_addr + r * (DP * 2) + ((x ^ (r & 7)) << 4));
            }
    }
    int32_t row_lo[MT][2], row_hi[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int32_t r = row0 + mt * 16 + (int32_t)g + 8 * i;
            visible(place0 + r / (int32_t)p.group, rq.length, p.causal, p.window, row_lo[mt][i], row_hi[mt][i]);
            if (r >= n_rows) row_hi[mt][i] = 0;
        }

    float o[MT][DP / 8][4] = {};
    float m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) m[mt][0] = m[mt][1] = -INFINITY, l[mt][0] = l[mt][1] = 0.f;
    uint32_t st = 0, ph = 0;
    for (int32_t i = (int32_t)warp; i < steps; i += kWarps) {
        const int32_t key = begin + i * kKeys;
        const bool okw = bar_wait(bars + 8 * st, ph, abort_flag, p.status);
        if (!__all_sync(0xffffffffu, okw)) break;
        const uint32_t ks_addr = ring + st * L::stage, vs_addr = ks_addr + L::kv_bytes;
        if (key < lo || key + kKeys > hi) {
            // keys outside what the tile sees: their values must not reach the
            // product even as 0 * NaN
            for (uint32_t c = lane; c < kKeys * DP / 8; c += 32) {
                const uint32_t r = c / (DP / 8), x = c % (DP / 8);
                const int32_t j = key + (int32_t)r;
                if (j < lo || j >= hi)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};"
                                 ::"r"(vs_addr + (x >> 3) * (kKeys * 128) + r * 128 + (((x & 7) ^ (r & 7)) << 4)), "r"(0)
                                 : "memory");
            }
            fence_proxy_async();   // before a later copy into the stage
            __syncwarp();
        }
        float s[MT][kKeys / 8][4] = {};
        const uint32_t lr = lane & 7, li = lane >> 3;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
            for (int kg = 0; kg < kKeys / 16; ++kg) {
                const uint32_t x = ks * 2 + (li & 1), kr = kg * 16 + (li >> 1) * 8 + lr;
                uint32_t bf[4];
                ldsm4<false>(bf, ks_addr + (x >> 3) * (kKeys * 128) + kr * 128 + (((x & 7) ^ lr) << 4));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    mma16816<BF16>(s[mt][2 * kg], qf[mt][ks], bf[0], bf[1]);
                    mma16816<BF16>(s[mt][2 * kg + 1], qf[mt][ks], bf[2], bf[3]);
                }
            }
        uint32_t pf[MT][kKeys / 16][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            // scale to powers of two, mask, running maximum
            float mx[2] = {m[mt][0], m[mt][1]};
#pragma unroll
            for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int32_t j = key + n * 8 + (int32_t)t4 * 2 + (c & 1);
                    const bool seen = j >= row_lo[mt][c >> 1] && j < row_hi[mt][c >> 1];
                    s[mt][n][c] = seen ? s[mt][n][c] * p.scale_log2 : -INFINITY;
                    mx[c >> 1] = fmaxf(mx[c >> 1], s[mt][n][c]);
                }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
            }
            if (__any_sync(0xffffffffu, mx[0] > m[mt][0] || mx[1] > m[mt][1])) {
                float al[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    al[r] = mx[r] > m[mt][r] ? exp2f(m[mt][r] - mx[r]) : 1.f;
                    l[mt][r] *= al[r];
                    m[mt][r] = mx[r];
                }
#pragma unroll
                for (int n = 0; n < DP / 8; ++n) {
                    o[mt][n][0] *= al[0];
                    o[mt][n][1] *= al[0];
                    o[mt][n][2] *= al[1];
                    o[mt][n][3] *= al[1];
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float mm = m[mt][r] == -INFINITY ? 0.f : m[mt][r];
#pragma unroll
                for (int kg = 0; kg < kKeys / 16; ++kg) {
                    float e[4];
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int c = 0; c < 2; ++c) e[n * 2 + c] = exp2f(s[mt][2 * kg + n][r * 2 + c] - mm);
                    l[mt][r] += (e[0] + e[1]) + (e[2] + e[3]);
                    pf[mt][kg][r] = pack16<BF16>(e[0], e[1]);
                    pf[mt][kg][r + 2] = pack16<BF16>(e[2], e[3]);
                }
            }
        }
#pragma unroll
        for (int kg = 0; kg < kKeys / 16; ++kg)
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) {
                const uint32_t x = n * 2 + (li >> 1), kr = kg * 16 + (li & 1) * 8 + lr;
                uint32_t bf[4];
                ldsm4<true>(bf, vs_addr + (x >> 3) * (kKeys * 128) + kr * 128 + (((x & 7) ^ lr) << 4));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    mma16816<BF16>(o[mt][2 * n], pf[mt][kg], bf[0], bf[1]);
                    mma16816<BF16>(o[mt][2 * n + 1], pf[mt][kg], bf[2], bf[3]);
                }
            }
        __syncwarp();   // every lane has read the stage
        if (i + L::stages * kWarps < steps) issue(i + L::stages * kWarps, st);
        if (++st == L::stages) { st = 0; ph ^= 1; }
    }
    if (*abort_flag) {   // every copy issued has landed before the memory is reused or the CTA exits
        for (int i = 0; i < L::stages; ++i) {
            bar_wait(bars + 8 * i, 0, abort_flag, p.status, false);
            bar_wait(bars + 8 * i, 1, abort_flag, p.status, false);
        }
    }

    // ---- join the warps
    __syncthreads();   // the rings are free
    float *ow = reinterpret_cast<float *>(smem) + warp * L::rows * DP;
    float2 *ml = reinterpret_cast<float2 *>(smem + L::ml_off);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 1);
            l[mt][r] += __shfl_xor_sync(0xffffffffu, l[mt][r], 2);
            if (t4 == 0) ml[warp * L::rows + mt * 16 + g + 8 * r] = make_float2(m[mt][r], l[mt][r]);
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r)
                *reinterpret_cast<float2 *>(ow + (mt * 16 + g + 8 * r) * DP + ((n * 8 + t4 * 2) ^ ((g & 3) * 8))) =
                    make_float2(o[mt][n][2 * r], o[mt][n][2 * r + 1]);
    }
    __syncthreads();
    const uint32_t rows = (uint32_t)min(L::rows, n_rows - row0);
    const uint32_t tile = blockIdx.z * p.n_kv + h;
    const float *oall = reinterpret_cast<const float *>(smem);
    constexpr uint32_t quads = DP / 4;
    // element e: row e / quads, elements 4 (e % quads) ..
    for (uint32_t e = threadIdx.x; e < rows * quads; e += kWarps * 32) {
        const uint32_t r = e / quads, d = (e % quads) * 4;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, ml[w * L::rows + r].x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float ll = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float2 v = ml[w * L::rows + r];
            const float a = v.x == -INFINITY ? 0.f : exp2f(v.x - mm);
            const float4 x = *reinterpret_cast<const float4 *>(oall + (w * L::rows + r) * DP + (d ^ ((r & 3) * 8)));
            acc.x += a * x.x;
            acc.y += a * x.y;
            acc.z += a * x.z;
            acc.w += a * x.w;
            ll += a * v.y;
        }
        if (n_split == 1) {
            store_row4<BF16>(p, rq, h, row0 + (int32_t)r, d, acc, mm, ll);
        } else {
            const uint64_t part = (uint64_t)tile * p.splits + split;
            __stcg(reinterpret_cast<float4 *>(p.ws + p.ws_ml + (part * p.ws_rows + r) * DP + d), acc);
            if (d == 0) __stcg(reinterpret_cast<float2 *>(p.ws) + part * p.ws_rows + r, make_float2(mm, ll));
        }
    }
    if (n_split == 1) return;

    // ---- the share that finishes last adds them all, in order
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        const uint32_t before = atomicAdd(p.counters + tile, 1u);
        *last_flag = before + 1 == n_split;
        if (before + 1 == n_split) p.counters[tile] = 0u;
        __threadfence();
    }
    __syncthreads();
    if (!*last_flag) return;
    if (n_split <= L::max_shares) {
        constexpr int rounds = L::rows * quads / (kWarps * 32);
        float2 *part = reinterpret_cast<float2 *>(smem);
        if (rows * quads <= kWarps * 32)
            join_shares<DP, MT, BF16, 1>(p, rq, h, tile, row0, rows, n_split, part, ml);
        else
            join_shares<DP, MT, BF16, rounds>(p, rq, h, tile, row0, rows, n_split, part, ml);
        return;
    }
    const float2 *mls = reinterpret_cast<const float2 *>(p.ws) + (uint64_t)tile * p.splits * p.ws_rows;
    const float *os = p.ws + p.ws_ml + (uint64_t)tile * p.splits * p.ws_rows * DP;
    for (uint32_t e = threadIdx.x; e < rows * quads; e += kWarps * 32) {   // very many shares
        const uint32_t r = e / quads, d = (e % quads) * 4;
        float mm = -INFINITY, ll = 0.f;
        for (uint32_t s = 0; s < n_split; ++s) mm = fmaxf(mm, __ldcg(mls + (uint64_t)s * p.ws_rows + r).x);
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (uint32_t s = 0; s < n_split; ++s) {
            const float2 v = __ldcg(mls + (uint64_t)s * p.ws_rows + r);
            const float a = v.x == -INFINITY ? 0.f : exp2f(v.x - mm);
            const float4 x = __ldcg(reinterpret_cast<const float4 *>(os + ((uint64_t)s * p.ws_rows + r) * DP + d));
            acc.x += a * x.x;
            acc.y += a * x.y;
            acc.z += a * x.z;
            acc.w += a * x.w;
            ll += a * v.y;
        }
        store_row4<BF16>(p, rq, h, row0 + (int32_t)r, d, acc, mm, ll);
    }
}

template <int DP, int MT, bool BF16>
cudaError_t launch_few(const CUtensorMap &km, const CUtensorMap &vm, const AttnParams &p, dim3 grid, cudaStream_t s) {
    using L = FewLayout<DP, MT>;
    auto kernel = few_rows_kernel<DP, MT, BF16>;
    static DeviceCache cache;
    int unused = 0;
    cudaError_t e = per_device(cache, unused, [&](int &) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::bytes);
    });
    if (e != cudaSuccess) return e;
    kernel<<<grid, kWarps * 32, L::bytes, s>>>(km, vm, p);
    return cudaGetLastError();
}

template <int DP, int MT>
cudaError_t launch_few_t(const CUtensorMap &km, const CUtensorMap &vm, const AttnParams &p, bool bf16, dim3 grid,
                         cudaStream_t s) {
    return bf16 ? launch_few<DP, MT, true>(km, vm, p, grid, s) : launch_few<DP, MT, false>(km, vm, p, grid, s);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void *ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
        return static_cast<PFN_cuTensorMapEncodeTiled_v12000>(nullptr);
    }();
    return fn;
}

// [page][head][token][d] of K or V as a map of 64-element x box_tokens boxes
// with the 128-byte swizzle; elements past head_dim are filled with zeros.
bool encode_cache(CUtensorMap *map, const uint16_t *base, const CacheView &c, uint32_t box_tokens, bool bf16) {
    auto enc = encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[4] = {c.head_dim, c.page_size, c.n_heads, c.n_pages};
    // the stride of a dimension of one element is never used but must be valid
    const uint64_t any = (uint64_t)c.head_dim * 2;
    const cuuint64_t strides[3] = {c.ld_token * 2, c.n_heads > 1 ? c.ld_head * 2 : any, c.n_pages > 1 ? c.ld_page * 2 : any};
    const cuuint32_t box[4] = {64u, box_tokens, 1u, 1u};
    const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
    return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
               const_cast<uint16_t *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Bytes of partial results that one launch asks the workspace for, at most
// (where one unit of work needs no more).
constexpr uint64_t kWorkspaceMost = 256u << 20;

// A fresh buffer of at least `need` bytes, `want` if there is room.
cudaError_t grown(void **fresh, size_t &want, size_t need) {
    cudaError_t e = cudaMalloc(fresh, want);
    if (e != cudaSuccess && want > need) e = cudaMalloc(fresh, want = need);
    if (e != cudaSuccess) cudaGetLastError();   // reported here, not by the next launch
    return e;
}

// Grows the context's split workspace; the counters start at zero and every
// complete kernel leaves them so.  cudaErrorMemoryAllocation: no room.
cudaError_t ensure_split(tc_cuda_ctx *ctx, size_t floats, size_t counters, cudaStream_t s) {
    constexpr int room = sizeof(ctx->attn_outgrown) / sizeof(ctx->attn_outgrown[0]);
    if (floats > ctx->attn_ws_floats) {
        void *fresh = nullptr;
        size_t bytes = std::max(floats, 2 * ctx->attn_ws_floats) * sizeof(float);
        if (ctx->attn_outgrown_n == room) return cudaErrorMemoryAllocation;   // grown too often
        const cudaError_t e = grown(&fresh, bytes, floats * sizeof(float));
        if (e != cudaSuccess) return e;
        if (ctx->attn_ws) ctx->attn_outgrown[ctx->attn_outgrown_n++] = ctx->attn_ws;
        ctx->attn_ws = static_cast<float *>(fresh);
        ctx->attn_ws_floats = bytes / sizeof(float);
    }
    if (counters > ctx->attn_counters_n) {
        void *fresh = nullptr;
        size_t bytes = std::max(counters, 2 * ctx->attn_counters_n) * sizeof(uint32_t);
        if (ctx->attn_outgrown_n == room) return cudaErrorMemoryAllocation;
        cudaError_t e = grown(&fresh, bytes, counters * sizeof(uint32_t));
        if (e == cudaSuccess && (e = cudaMemsetAsync(fresh, 0, bytes, s)) != cudaSuccess) cudaFree(fresh);
        if (e != cudaSuccess) return e;
        if (ctx->attn_counters) ctx->attn_outgrown[ctx->attn_outgrown_n++] = ctx->attn_counters;
        ctx->attn_counters = static_cast<uint32_t *>(fresh);
        ctx->attn_counters_n = bytes / sizeof(uint32_t);
    }
    return cudaSuccess;
}

// How a call is divided over CTAs, by its sizes alone.
struct AttnPlan {
    bool many;                 // attn_chunk_sm100.cu's kernel, else this file's
    uint32_t dp, mt;           // head_dim padded; mma tiles of a CTA (few rows)
    uint32_t chunk, splits;    // keys of a share, shares
    uint32_t n_blocks;         // many rows: upper bound of the blocks of rows
    uint32_t row_tiles, ws_rows;
    uint64_t units, each;      // few rows: requests x row tiles, of which a launch takes `each`
    uint64_t ws_ml, ws_floats, counters;   // workspace (0: none)
};

const char *plan_attention(const BatchView &bt, uint32_t n_kv, uint64_t group, uint32_t head_dim, uint32_t page_shift,
                           bool causal, int32_t window, uint32_t sm_count, uint64_t workspace_most, AttnPlan &a) {
    a = AttnPlan{};
    // longest span of keys one tile of rows sees (requests that their row of the
    // page table does not cover are not served)
    uint64_t span = std::min<uint64_t>(bt.max_length, (uint64_t)bt.table_width << page_shift);
    if (window) {
        const uint64_t reach = (uint64_t)window * (causal ? 1 : 2) + bt.max_new;
        if (reach < span) span = reach;
    }
    const uint64_t rows_most = group * bt.max_new;
    // mma tiles of a CTA: all rows of a request in one CTA, so that K and V are
    // read once, as far as the registers go; beyond, blocks of 256 rows on the
    // tensor cores.  This kernel against that one in us (caches cold, 4 cache heads):
    //   rows a head       16     32     48-64  |  16     32     48-64   128
    //                     head_dim 128         |  head_dim 64
    //   1 x 500 keys     14/26  18/24   18/24  | 12/24  14/24   19/24   20/22
    //   8 x 500          16/20  21/18   22/18  | 14/18  16/18   22/18   25/16
    //   32 x 500         23/22  27/21   27/22  | 16/19  20/18   30/19   33/18
    //   1 x 4000         20/32  27/32   27/33  | 16/28  20/28   29/28   31/28
    //   8 x 4000         31/42  35/42   43/41  | 21/37  25/36   38/36   55/34
    //   32 x 4000        70/74  80/72  135/74  | 43/70  49/66   99/68  182/53
    // (48 to 64 rows of heads of 64 stay here for the few and short requests; many
    // long ones would be faster there.)
    const uint32_t dp = a.dp = head_dim <= 64 ? 64 : head_dim <= 128 ? 128 : 256;
    const uint32_t mt = a.mt = rows_most <= 16 || dp == 256 ? 1 : rows_most <= 32 || dp == 128 ? 2 : 4;
    a.many = rows_most > mt * 16 && head_dim <= 128;
    if (a.many) {
        const uint64_t rows = (uint64_t)bt.n_tokens * group;
        a.n_blocks = (uint32_t)(rows / kChunkRows + bt.n_seq);
        // Shares of the keys: as many CTAs as make the busiest SM's work least,
        // in steps of 128 keys plus kCtaSteps for what a CTA does besides, one
        // CTA per SM, and the time to join the shares (2 us, 0.5 us a share, and
        // their partial results written and read at 6.5 TB/s, all in quarters of
        // a step of 2 us); no share under kLeastSteps, none for a gain of less than
        // 1 in kLeastGain (a round more or less of thousands of CTAs is within the
        // model's error, gigabytes of partial results are not), and no more than
        // the workspace is to hold.
        constexpr uint64_t kCtaSteps = 3, kLeastSteps = 2, kLeastGain = 32, kQuarterBytes = 3250000;
        const uint64_t steps = (span + kChunkKeys - 1) / kChunkKeys + 1;
        const uint64_t blocks = std::max<uint64_t>((rows + kChunkRows - 1) / kChunkRows, bt.n_seq);
        const uint64_t part_bytes = (uint64_t)n_kv * kChunkRows * (dp + 2) * sizeof(float);   // of a block and share
        uint64_t one = 0, best = 0, share = steps;
        for (uint64_t n = 1; n <= kChunkShares && (n == 1 || steps / n >= kLeastSteps); ++n) {
            const uint64_t each = (steps + n - 1) / n, real = (steps + each - 1) / each;
            if (real > 1 && a.n_blocks * real * part_bytes > workspace_most) break;
            const uint64_t waves = (blocks * n_kv * real + sm_count - 1) / sm_count;
            const uint64_t join = real > 1 ? 4 + real + 2 * blocks * real * part_bytes / kQuarterBytes : 0;
            const uint64_t cost = 4 * waves * (each + kCtaSteps) + join;
            if (n == 1) one = best = cost;
            if (cost < best && cost + one / kLeastGain <= one) {
                best = cost;
                share = each;
            }
        }
        a.chunk = (uint32_t)(share * kChunkKeys);
        a.splits = (uint32_t)((steps + share - 1) / share);
        if ((uint64_t)a.n_blocks * n_kv * a.splits > 0x7fffffffu) return "too many tokens or requests";
        if (a.splits > 1) {
            const uint64_t parts = (uint64_t)a.n_blocks * n_kv * a.splits * kChunkRows;
            a.ws_ml = parts * 2;
            a.ws_floats = a.ws_ml + parts * dp;
        }
        return nullptr;
    }
    a.row_tiles = (uint32_t)((rows_most + 16 * mt - 1) / (16 * mt));
    a.units = (uint64_t)bt.n_seq * a.row_tiles;
    if (a.units > 0x7fffffffu) return "too many tokens or requests";
    span += step_keys((int)dp, (int)mt);   // the first key is rounded down to a step
    // Chunk of the cache per CTA: the least of (rounds of CTAs over the GPU's
    // places) x (a chunk's time + what a CTA costs besides) + the time to join
    // the shares, all in keys: about 100 KB for a CTA's start and end (7 us
    // against 15 GB/s a place), 8 keys a share.  8 requests of 6000 keys of 64 by 28
    // rows: 7 shares, one round, 29 us; 11 shares in two rounds 41 us.
    // For 17 to 32 rows of heads of 64 the rounds are the mean of two: all requests
    // as long as the longest, and three quarters of that on average.  23 drafting
    // requests of 100 to 6000 keys behind a window of 2048: 3 shares, 20.2 us, where
    // the longest alone would give 5 shares and 28.4.  For the other shapes the
    // longest alone is as good or better (decode step of 96 requests 236.5 us
    // against 242.5; heads of 128 with up to 32 rows 2 % on average).
    const uint64_t places = (uint64_t)sm_count * ctas_per_sm((int)dp, (int)mt), cta_keys = 100 * 1024 / (4 * dp);
    const bool uneven = dp == 64 && mt == 2 && bt.n_seq > 1;
    uint64_t chunk = kMaxChunk, best = ~0ull;
    for (uint64_t c = kMaxChunk; c >= 64; c -= 64) {
        const uint64_t n = (span + c - 1) / c, ctas = a.units * n * n_kv, rounds = (ctas + places - 1) / places;
        const uint64_t fewer = uneven ? (ctas * 3 / 4 + places - 1) / places : rounds;
        const uint64_t cost = (rounds + fewer) * (c + cta_keys) / 2 + 8 * n;
        if (cost < best) {
            best = cost;
            chunk = c;
        }
    }
    a.chunk = (uint32_t)chunk;
    a.splits = (uint32_t)((span + chunk - 1) / chunk);
    a.ws_rows = (uint32_t)std::min<uint64_t>(rows_most, 16 * mt);
    // Units of a launch: a dimension of the grid, and no more than their partial
    // results fit the workspace (at 256 MB and 16 KB or so a CTA that leaves tens of
    // rounds over the GPU; launches on a stream take turns with the workspace).
    a.each = std::min<uint64_t>(a.units, 65535);
    if (a.splits > 1) {
        const uint64_t parts = (uint64_t)n_kv * a.splits * a.ws_rows;   // of a unit
        a.each = std::max<uint64_t>(std::min(a.each, workspace_most / (parts * (dp + 2) * sizeof(float))), 1);
        a.ws_ml = (a.each * parts * 2 + 3) / 4 * 4;
        a.ws_floats = a.ws_ml + a.each * parts * dp;
        a.counters = a.each * n_kv;
    }
    return nullptr;
}

int attend(tc_cuda_ctx *ctx, const tc_paged_cache *cache, const tc_paged_batch *batch, const tc_attention *a,
           cudaStream_t s) {
    CacheView c{};
    AttnParams p{};
    if (!ctx || !a) return fail("null argument");
    if (const char *e = check_cache(cache, c)) return fail(e);
    if (const char *e = check_batch(batch, p.batch)) return fail(e);
    if (!a->n_heads || a->n_heads % c.n_heads) return fail("n_heads must be a multiple of the cache's heads");
    if (!(a->scale == a->scale) || std::isinf(a->scale)) return fail("scale must be finite");
    if (a->window < 0) return fail("window must not be negative");
    if (!p.batch.n_tokens) return ok();
    if (!a->q || !a->out) return fail("null argument");
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->out)) % 2 ||
        reinterpret_cast<uintptr_t>(a->lse) % 4)
        return fail("misaligned pointer");
    if ((a->ld_q_token | a->ld_q_head | a->ld_out_token | a->ld_out_head) >> 38)
        return fail("invalid/overlapping head stride");
    if (rows_overlap(p.batch.n_tokens, a->ld_out_token, a->n_heads, a->ld_out_head, c.head_dim))
        return fail("invalid/overlapping head stride");
    if (!p.batch.max_new) return fail("max_new must not be 0 where there are tokens");
    const uint64_t group = a->n_heads / c.n_heads;
    if (c.n_heads > 65535 || group * p.batch.max_new > 0x7fffffffu) return fail("too many heads");
    p.q = static_cast<const uint16_t *>(a->q);
    p.out = static_cast<uint16_t *>(a->out);
    p.lse = a->lse;
    p.ld_q_token = a->ld_q_token;
    p.ld_q_head = a->ld_q_head;
    p.ld_out_token = a->ld_out_token;
    p.ld_out_head = a->ld_out_head;
    p.n_kv = c.n_heads;
    p.group = (uint32_t)group;
    p.head_dim = c.head_dim;
    p.page_shift = c.page_shift;
    p.n_pages = c.n_pages;
    p.causal = a->causal != 0;
    p.window = a->window > kMaxLength ? kMaxLength : a->window;
    p.scale_log2 = a->scale * 1.4426950408889634f;   // exp(x) = 2^(x log2 e)
    p.status = ctx->status;
    p.q_wide = !(reinterpret_cast<uintptr_t>(a->q) % 16) && !(a->ld_q_token % 8) && !(a->ld_q_head % 8);
    p.out_quads = !(reinterpret_cast<uintptr_t>(a->out) % 8) && !(a->ld_out_token % 4) && !(a->ld_out_head % 4);
    const bool bf16 = cache->dtype == TC_DTYPE_BF16;

    CurrentDevice guard(ctx->device);
    AttnPlan plan;
    for (uint64_t most = kWorkspaceMost;;) {
        if (const char *e = plan_attention(p.batch, c.n_heads, group, c.head_dim, c.page_shift, p.causal, p.window,
                                           (uint32_t)ctx->sm_count, most, plan))
            return fail(e);
        const cudaError_t e = plan.ws_floats ? ensure_split(ctx, plan.ws_floats, plan.counters, s) : cudaSuccess;
        if (e == cudaSuccess) break;
        // no room: with what there is (any other error, as in a capture, is one)
        if (e != cudaErrorMemoryAllocation || most != kWorkspaceMost) return cuda_fail("attention workspace allocation", e);
        most = std::min<uint64_t>(ctx->attn_ws_floats * sizeof(float), most - 1);
    }
    p.chunk = plan.chunk;
    p.splits = plan.splits;
    p.n_blocks = plan.n_blocks;
    p.row_tiles = plan.row_tiles;
    p.ws_rows = plan.ws_rows;
    p.ws_ml = plan.ws_ml;
    p.ws = ctx->attn_ws;
    p.counters = ctx->attn_counters;
    const uint32_t dp = plan.dp, mt = plan.mt;
    const uint32_t keys = plan.many ? kChunkKeys : step_keys((int)dp, (int)mt);
    CUtensorMap km, vm;
    const uint32_t box = c.page_size < keys ? c.page_size : keys;
    if (!encode_cache(&km, c.k, c, box, bf16) || !encode_cache(&vm, c.v, c, box, bf16))
        return fail("the cache cannot be described to TMA");
    if (plan.many) {
        const uint64_t out_bits = reinterpret_cast<uintptr_t>(a->out) | a->ld_out_token * 2 | a->ld_out_head * 2;
        p.out_wide = out_bits % 32 == 0 ? 32 : out_bits % 16 == 0 ? 16 : 0;
        p.negate_q = p.scale_log2 < 0.f;
        p.scale_log2 = std::fabs(p.scale_log2);
        if (p.scale_log2 < 1e-30f) p.scale_log2 = 1e-30f;   // 0 * -inf would lose the mask
        const cudaError_t e = launch_chunk(km, vm, p, bf16, s);
        return e == cudaSuccess ? ok() : cuda_fail("paged attention launch", e);
    }
    cudaError_t e = cudaSuccess;
    for (uint64_t first = 0; first < plan.units && e == cudaSuccess; first += plan.each) {
        p.first_unit = (uint32_t)first;
        const dim3 grid(p.splits, c.n_heads, (uint32_t)std::min(plan.each, plan.units - first));
        if (dp == 64)
            e = mt == 1   ? launch_few_t<64, 1>(km, vm, p, bf16, grid, s)
                : mt == 2 ? launch_few_t<64, 2>(km, vm, p, bf16, grid, s)
                          : launch_few_t<64, 4>(km, vm, p, bf16, grid, s);
        else if (dp == 128)
            e = mt == 1 ? launch_few_t<128, 1>(km, vm, p, bf16, grid, s) : launch_few_t<128, 2>(km, vm, p, bf16, grid, s);
        else
            e = launch_few_t<256, 1>(km, vm, p, bf16, grid, s);
    }
    return e == cudaSuccess ? ok() : cuda_fail("paged attention launch", e);
}

}  // namespace
}  // namespace tc

extern "C" int tc_paged_attention_plan(uint32_t sm_count, uint32_t n_heads, uint32_t cache_heads, uint32_t head_dim,
                                       uint32_t page_size, const tc_paged_batch *batch, int32_t causal, int32_t window,
                                       tc_attention_plan *plan) {
    using namespace tc;
    try {
        if (!batch || !plan) return fail("null argument");
        if (!sm_count || !head_dim || head_dim % 8 || head_dim > 256 || !cache_heads || cache_heads > 65535 || !n_heads ||
            n_heads % cache_heads || page_size < 8 || page_size > 65536 || (page_size & (page_size - 1)) || window < 0 ||
            batch->max_length > (uint32_t)kMaxLength || !batch->n_seq || batch->n_seq > 0xffffffu || !batch->n_tokens ||
            batch->n_tokens > 0x7fffffffu || !batch->max_new)
            return fail("sizes that tc_cuda_paged_attention would not take");
        BatchView bt{};
        bt.n_seq = batch->n_seq;
        bt.table_width = batch->table_width;
        bt.n_tokens = batch->n_tokens;
        bt.max_new = std::min(batch->max_new, batch->n_tokens);
        bt.max_length = batch->max_length;
        const uint64_t group = n_heads / cache_heads;
        if (group * bt.max_new > 0x7fffffffu) return fail("too many heads");
        AttnPlan a;
        if (const char *e = plan_attention(bt, cache_heads, group, head_dim, (uint32_t)__builtin_ctz(page_size), causal != 0,
                                           std::min(window, kMaxLength), sm_count, kWorkspaceMost, a))
            return fail(e);
        *plan = tc_attention_plan{};
        plan->many_rows = a.many;
        plan->rows = a.many ? kChunkRows : 16 * a.mt;
        plan->ctas_per_sm = a.many ? 1 : (uint32_t)ctas_per_sm((int)a.dp, (int)a.mt);
        plan->share_keys = a.chunk;
        plan->shares = a.splits;
        plan->launches = a.many ? 1 : (uint32_t)((a.units + a.each - 1) / a.each);
        plan->workspace_bytes = a.ws_floats * sizeof(float);
        return ok();
    } catch (...) {
        return TC_CUDA_FAIL;
    }
}

extern "C" int tc_cuda_paged_attention(tc_cuda_ctx *ctx, const tc_paged_cache *cache, const tc_paged_batch *batch,
                                       const tc_attention *attention, void *stream) {
    try {
        return tc::attend(ctx, cache, batch, attention, static_cast<cudaStream_t>(stream));
    } catch (...) {
        return TC_CUDA_FAIL;
    }
}
