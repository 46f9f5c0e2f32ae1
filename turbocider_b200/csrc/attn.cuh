// Shared pieces of the attention operators (attn_heads.cu, attn_paged.cu,
// attn_chunk_sm100.cu): views of the paged cache and of a step's batch, the
// checks of what is read from device memory, and host-side argument checks.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <string>

#include "../../include/turbocider_cuda.h"
#include "tc_internal.h"

namespace tc {

constexpr uint32_t kStatusGeometry = 1u << 3;
constexpr int32_t kMaxLength = 1 << 30;   // cached tokens of one request (sums with a window stay in int32)

// The step of tc_paged_batch, as kernels read it.
struct BatchView {
    const int32_t *new_offsets, *lengths, *page_table;
    uint32_t n_seq, table_width, ld_table, n_tokens, max_new, max_length;
};

struct CacheView {
    uint16_t *k, *v;
    uint64_t ld_page, ld_head, ld_token;
    uint32_t n_pages, page_size, page_shift, n_heads, head_dim;
};

// One request of the step (no rows or length 0 where its values in device
// memory are impossible).
struct Request {
    int32_t first, n_new, length;   // first row of q, new tokens, cached tokens
};

#ifdef __CUDACC__
// A request with its values checked: rows inside q, a length that covers its
// new tokens (0: an unused place) and that its row of the page table covers,
// nothing past the bounds the launch was sized by.
__device__ __forceinline__ Request check_request(const BatchView &bt, uint32_t page_shift, int32_t first, int32_t end,
                                                 int32_t length, uint32_t *status) {
    Request r{first, end - first, length};
    if (first < 0 || end < first || (uint32_t)end > bt.n_tokens) {
        atomicOr(status, kStatusGeometry);
        return Request{0, 0, 0};
    }
    if (length < 0 || (uint32_t)length > bt.max_length || (uint32_t)r.n_new > bt.max_new ||
        ((uint64_t)bt.table_width << page_shift) < (uint64_t)length || (length < r.n_new && length > 0)) {
        atomicOr(status, kStatusGeometry);
        r.length = 0;
        r.n_new = min(r.n_new, (int32_t)bt.max_new);   // rows past it are nobody's
    }
    return r;
}
__device__ __forceinline__ Request load_request(const BatchView &bt, uint32_t page_shift, uint32_t b,
                                                uint32_t *status) {
    return check_request(bt, page_shift, bt.new_offsets[b], bt.new_offsets[b + 1], bt.lengths[b], status);
}

// Page number of entry j of request b's row (j < table_width).  A number
// outside the cache sets TC_STATUS_GEOMETRY and gives -1.
__device__ __forceinline__ int32_t check_page(int32_t p, uint32_t n_pages, uint32_t *status) {
    if (p < 0 || (uint32_t)p >= n_pages) {
        atomicOr(status, kStatusGeometry);
        return -1;
    }
    return p;
}
__device__ __forceinline__ int32_t load_page(const BatchView &bt, uint32_t n_pages, uint32_t b, uint32_t j,
                                             uint32_t *status) {
    return check_page(bt.page_table[(uint64_t)b * bt.ld_table + j], n_pages, status);
}

// How many of the requests 1 .. n satisfy `before` (true for a prefix of
// them), found by the warp 32 at a time.
template <class F>
__device__ __forceinline__ uint32_t count_prefix(uint32_t n, F &&before) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0;   // the answer is in [lo, lo + n]
    while (n > 0) {
        const uint32_t step = (n + 31) / 32, i = (lane + 1) * step;
        const bool yes = before(lo + min(i, n)) && i <= n;
        const uint32_t c = __popc(__ballot_sync(0xffffffffu, yes));
        lo += c * step;
        n = min(n - c * step, step - 1);
    }
    return lo;
}

// Positions [lo, hi) that the new token at cache position p sees.
__device__ __forceinline__ void visible(int32_t p, int32_t length, int causal, int32_t window, int32_t &lo,
                                        int32_t &hi) {
    lo = window > 0 ? max(p - window + 1, 0) : 0;
    hi = causal ? min(p + 1, length) : window > 0 ? min(p + window, length) : length;
}
#endif

// ---- host side of the entry points
inline int fail(const char *reason) {
    set_last_error(reason);
    return TC_CUDA_FAIL;
}
inline int ok() {
    set_last_error("");
    return TC_CUDA_OK;
}
inline int cuda_fail(const char *what, cudaError_t e) {
    set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
    return TC_CUDA_FAIL;
}

// The context's device current for a call, the caller's afterwards.
struct CurrentDevice {
    int previous = -1;
    explicit CurrentDevice(int device) {
        if (cudaGetDevice(&previous) != cudaSuccess) previous = -1;
        if (previous != device) cudaSetDevice(device);
        else previous = -1;
    }
    ~CurrentDevice() {
        if (previous >= 0) cudaSetDevice(previous);
    }
};

// Checks of the arguments; nullptr: fine.
const char *check_cache(const tc_paged_cache *c, CacheView &v);
const char *check_batch(const tc_paged_batch *b, BatchView &v);
// Whether [a][b] rows of `width` elements at strides ld_a, ld_b share elements.
bool rows_overlap(uint64_t a, uint64_t ld_a, uint64_t b, uint64_t ld_b, uint64_t width);

}  // namespace tc
