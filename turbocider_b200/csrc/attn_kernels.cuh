// Device pieces shared by the paged-attention kernels.
#pragma once
#include "attn.cuh"
#include "kq_sm100.cuh"

namespace tc {

struct AttnParams {
    const uint16_t *q;
    uint16_t *out;
    float *lse;
    uint64_t ld_q_token, ld_q_head, ld_out_token, ld_out_head;
    BatchView batch;
    uint32_t n_kv, group, head_dim, page_shift, n_pages;
    int causal;
    int32_t window;
    float scale_log2;            // scale * log2(e)
    uint32_t *status;
    // row tiles of a request and chunks of its cache
    uint32_t row_tiles, chunk, splits;
    uint32_t first_unit;         // few rows: request and row tile of the launch's first CTAs
    // partial results: [tile][split][ws_rows] of (maximum, sum), then of the
    // unnormalised outputs from float ws_ml on
    uint32_t ws_rows;
    uint64_t ws_ml;
    float *ws;
    uint32_t *counters;
    bool q_wide, out_quads;      // 16-byte loads of q / 8-byte stores of out are aligned
    uint32_t out_wide;           // bytes of an aligned store of out: 32, 16, or 0 for less
    uint32_t n_blocks;           // many rows: upper bound of the blocks of rows
    bool negate_q;               // many rows: scale_log2 is positive, the sign goes to q
};

// Chunks of many rows (attn_chunk_sm100.cu), head_dim at most 128.
constexpr int kChunkRows = 256;      // rows of a CTA: two tensor-core tiles
constexpr int kChunkKeys = 128;      // keys of a step
constexpr uint32_t kChunkShares = 64;   // shares of the keys, at most
cudaError_t launch_chunk(const CUtensorMap &km, const CUtensorMap &vm, const AttnParams &p, bool bf16,
                         cudaStream_t s);

namespace {

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, uint32_t b, int x, int y, int z,
                                            int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(b) : "memory");
}

// Two floats rounded to one word of 16-bit elements.
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// Final results of row `row` of the request (token row / group), elements
// [d, d + 4): acc / sum, and the row's log-sum with d = 0.
template <bool BF16>
__device__ __forceinline__ void store_row4(const AttnParams &p, const Request &rq, uint32_t h, int32_t row, uint32_t d,
                                           float4 acc, float m, float l) {
    const uint64_t token = (uint64_t)rq.first + row / p.group;
    const uint32_t head = h * p.group + row % p.group;
    if (p.lse && d == 0)
        p.lse[token * (p.n_kv * p.group) + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f;
    if (d >= p.head_dim) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;   // (a NaN sum stays one)
    const uint2 w = make_uint2(pack16<BF16>(acc.x * inv, acc.y * inv), pack16<BF16>(acc.z * inv, acc.w * inv));
    uint16_t *o = p.out + token * p.ld_out_token + head * p.ld_out_head + d;
    if (p.out_quads) {
        *reinterpret_cast<uint2 *>(o) = w;
    } else {
        o[0] = (uint16_t)w.x;
        o[1] = (uint16_t)(w.x >> 16);
        o[2] = (uint16_t)w.y;
        o[3] = (uint16_t)(w.y >> 16);
    }
}

}  // namespace
}  // namespace tc
