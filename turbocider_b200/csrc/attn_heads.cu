// Norm and position rotation of query and key heads, alone
// (tc_cuda_qk_norm_rope) or on the way into a paged cache
// (tc_cuda_kv_append).  For a head x of head_dim elements
//     y = x * rsqrt(mean(x^2) + eps) * weight
//     (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t)
// over its rotary pairs, t = position * freq.
//
// Bytes bound: every element is read once and written once (2 + 2 bytes for
// 16-bit types) against about 10 flops.  A head is spread over the smallest
// power-of-two group of lanes that gives each lane one unit of 8 elements: 4
// pairs with both members in the same lane (two 4-element chunks half a
// rotary width apart for the half layout, 8 neighbours for the interleaved
// one), so the rotation needs no exchange and the norm one butterfly over the
// group.  A block takes one token; a thread keeps its unit for all heads it
// visits, so the angles, sines and cosines are formed once per thread and
// serve every head.
//
// The angle: freq / 2 pi is held as a 64-bit binary fraction of a turn and
// multiplied by the position modulo 2^64, i.e. modulo one turn and exactly,
// whatever the position; its top 32 bits go to sincospif.  A table of cosines
// would cost rotary_dim * 4 bytes a token and a size fixed in advance.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include "attn.cuh"

namespace tc {
namespace {

struct HeadsView {
    const void *x;
    void *out;
    const float *weight;
    uint64_t ld_token, ld_head, ld_out_token, ld_out_head;
    uint32_t n_heads;
};

struct HeadsParams {
    HeadsView q, k, v;           // v: copied to the cache (append only)
    uint32_t head_dim, n_tokens, heads_per_block;
    int rms_norm;
    float eps, inv_dim;
    // rotation
    const double *freq;
    const int32_t *positions;
    uint32_t rotary_units, half, n_axes, axis_end[4];
    float amplitude;
    // append
    BatchView batch;
    CacheView cache;
    uint32_t *status;
};

// Four elements in and out of fp32.
__device__ __forceinline__ void unpack4(float4 v, float *f) { f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w; }
template <class T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <class T>
struct alignas(4 * sizeof(T)) Chunk { T v[4]; };

// VEC: 4-element chunks may be moved as one access.
template <class T, bool VEC>
__device__ __forceinline__ Chunk<T> load_chunk(const T *p) {
    if (VEC) return *reinterpret_cast<const Chunk<T> *>(p);
    Chunk<T> c;
#pragma unroll
    for (int i = 0; i < 4; ++i) c.v[i] = p[i];
    return c;
}
template <class T, bool VEC>
__device__ __forceinline__ void store_chunk(T *p, const Chunk<T> &c) {
    if (VEC) {
        *reinterpret_cast<Chunk<T> *>(p) = c;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = c.v[i];
}

// Request of token t: the number of requests that end at or before it
// (n_seq: t belongs to none).
__device__ __forceinline__ uint32_t request_of(const BatchView &bt, int32_t t) {
    return count_prefix(bt.n_seq, [&](uint32_t b) { return bt.new_offsets[b] <= t; });
}

template <class T, bool HALF, bool APPEND, bool VEC>
__global__ void __launch_bounds__(128) heads_kernel(const __grid_constant__ HeadsParams p) {
    const uint32_t units = p.head_dim / 8;
    const uint32_t lanes = units <= 1 ? 1u : 1u << (32 - __clz(units - 1));   // lanes per head
    const uint32_t unit = threadIdx.x & (lanes - 1), slot = threadIdx.x / lanes, slots = blockDim.x / lanes;
    const bool active = unit < units, rotates = unit < p.rotary_units;
    // the unit's two chunks of four elements
    const uint32_t c0 = rotates && HALF ? 4 * unit : 8 * unit;
    const uint32_t c1 = rotates && HALF ? p.half + 4 * unit : 8 * unit + 4;
    const uint32_t n_rot = p.q.n_heads + p.k.n_heads, n_all = n_rot + p.v.n_heads;
    const uint32_t h_end = min((blockIdx.y + 1) * p.heads_per_block, n_all);
    const uint64_t t = blockIdx.x;

    int32_t position = 0;
    uint64_t k_base = 0;          // of head 0 in the cache
    bool store_kv = false;
    if (APPEND) {
        const uint32_t b = request_of(p.batch, (int32_t)t);
        if (b >= p.batch.n_seq) return;
        const Request r = load_request(p.batch, p.cache.page_shift, b, p.status);
        if ((int32_t)t < r.first || (int32_t)t >= r.first + r.n_new) return;
        const int32_t at = r.length - r.n_new + ((int32_t)t - r.first);
        if (r.length > 0 && at >= 0) {
            const int32_t page = load_page(p.batch, p.cache.n_pages, b, (uint32_t)at >> p.cache.page_shift, p.status);
            store_kv = page >= 0;
            k_base = (uint64_t)(page < 0 ? 0 : page) * p.cache.ld_page +
                     ((uint32_t)at & (p.cache.page_size - 1)) * p.cache.ld_token;
        }
        position = max(at, 0);
    }

    float cs[4], sn[4];
    if (rotates) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t pair = 4 * unit + i;
            int32_t pos = position;
            if (p.positions) {
                uint32_t axis = 0;
                while (axis + 1 < p.n_axes && pair >= p.axis_end[axis]) ++axis;
                pos = p.positions[t * p.n_axes + axis];
            }
            // freq in turns as a fraction of 2^64; negative frequencies wrap
            // (two's complement), whole turns fall away
            const double turns = p.freq[pair] * 0.15915494309189533577;   // 1 / (2 pi)
            const uint64_t step = (uint64_t)__double2ull_rn((turns - floor(turns)) * 18446744073709551616.0);
            const uint64_t phase = step * (uint64_t)(int64_t)pos;
            sincospif((float)(int32_t)(phase >> 32) * 4.656612873077392578125e-10f, &sn[i], &cs[i]);   // 2^-31
            sn[i] *= p.amplitude;
            cs[i] *= p.amplitude;
        }
    }

    // heads 0 .. : the queries', then the keys', then the values'
#pragma unroll 4
    for (uint32_t h = blockIdx.y * p.heads_per_block + slot; h < h_end + slot; h += slots) {
        // (every lane runs the loop so that the butterfly below is complete)
        const bool on = active && h < h_end;
        const bool is_q = h < p.q.n_heads, is_v = h >= n_rot;
        const HeadsView &hv = is_q ? p.q : is_v ? p.v : p.k;
        const uint32_t hh = is_q ? h : is_v ? h - n_rot : h - p.q.n_heads;
        const T *x = static_cast<const T *>(hv.x) + t * hv.ld_token + hh * hv.ld_head;
        Chunk<T> a, b;
        if (on) {
            a = load_chunk<T, VEC>(x + c0);
            b = load_chunk<T, VEC>(x + c1);
        }
        T *out;
        if (APPEND && !is_q)
            out = reinterpret_cast<T *>(is_v ? p.cache.v : p.cache.k) + k_base + hh * p.cache.ld_head;
        else
            out = static_cast<T *>(hv.out) + t * hv.ld_out_token + hh * hv.ld_out_head;
        const bool store = on && (!APPEND || is_q || store_kv);
        float fa[4], fb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            fa[i] = on ? to_float<T>(a.v[i]) : 0.f;
            fb[i] = on ? to_float<T>(b.v[i]) : 0.f;
        }
        if (p.rms_norm) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss += fa[i] * fa[i] + fb[i] * fb[i];
            for (uint32_t d = lanes / 2; d > 0; d /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, d);
            if (!is_v) {
                const float r = rsqrtf(ss * p.inv_dim + p.eps);
                float wa[4] = {1.f, 1.f, 1.f, 1.f}, wb[4] = {1.f, 1.f, 1.f, 1.f};
                if (hv.weight && on) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        wa[i] = hv.weight[c0 + i];
                        wb[i] = hv.weight[c1 + i];
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    fa[i] *= r * wa[i];
                    fb[i] *= r * wb[i];
                }
            }
        }
        if (rotates && !is_v) {
            if (HALF) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float u = fa[i], w = fb[i];
                    fa[i] = u * cs[i] - w * sn[i];
                    fb[i] = w * cs[i] + u * sn[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float *e = i < 2 ? fa + 2 * i : fb + 2 * i - 4;
                    const float u = e[0], w = e[1];
                    e[0] = u * cs[i] - w * sn[i];
                    e[1] = w * cs[i] + u * sn[i];
                }
            }
        }
        if (store) {
            if (!is_v) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a.v[i] = from_float<T>(fa[i]);
                    b.v[i] = from_float<T>(fb[i]);
                }
            }
            store_chunk<T, VEC>(out + c0, a);
            store_chunk<T, VEC>(out + c1, b);
        }
    }
}

template <class T, bool APPEND>
cudaError_t launch_heads(HeadsParams &p, bool half, bool vec, int sm_count, cudaStream_t s) {
    const uint32_t n_all = p.q.n_heads + p.k.n_heads + p.v.n_heads;
    uint32_t lanes = 1;
    while (lanes * 8 < p.head_dim) lanes *= 2;
    const uint32_t slots = 128 / lanes;
    // One pass over the heads per block while that leaves the GPU underfilled
    // (each thread then carries one head), all heads of a token per block
    // once there are enough tokens (the angles are formed once per block).
    const uint64_t passes = (n_all + slots - 1) / slots;
    const uint64_t room = (uint64_t)sm_count * 16;   // blocks of 128 resident
    uint64_t per = (passes * p.n_tokens + room - 1) / room;
    if (per < 1) per = 1;
    if (per > passes) per = passes;
    p.heads_per_block = (uint32_t)per * slots;
    const dim3 grid(p.n_tokens, (n_all + p.heads_per_block - 1) / p.heads_per_block);
    if (half) {
        if (vec) heads_kernel<T, true, APPEND, true><<<grid, 128, 0, s>>>(p);
        else heads_kernel<T, true, APPEND, false><<<grid, 128, 0, s>>>(p);
    } else {
        if (vec) heads_kernel<T, false, APPEND, true><<<grid, 128, 0, s>>>(p);
        else heads_kernel<T, false, APPEND, false><<<grid, 128, 0, s>>>(p);
    }
    return cudaGetLastError();
}

int fail(const char *reason) {
    set_last_error(reason);
    return TC_CUDA_FAIL;
}
int ok() {
    set_last_error("");
    return TC_CUDA_OK;
}

HeadsView view_of(const tc_heads *h) {
    return {h->x, h->out, h->weight, h->ld_token, h->ld_head, h->ld_out_token, h->ld_out_head, h->n_heads};
}

// 4-element chunks of `item`-byte elements can move as one access.
bool chunked(const void *p, uint64_t ld_token, uint64_t ld_head, uint32_t item) {
    return !(reinterpret_cast<uintptr_t>(p) % (4 * item)) && !(ld_token % 4) && !(ld_head % 4);
}

// Whether rows of `width` elements at the given strides share elements.
struct Extent { uint64_t count, stride; };
bool overlap(Extent *e, int n, uint64_t width) {
    std::sort(e, e + n, [](const Extent &a, const Extent &b) { return a.stride < b.stride; });
    for (int i = 0; i < n; ++i) {
        if (e[i].count <= 1) continue;
        if (e[i].stride < width) return true;
        width += e[i].stride * (e[i].count - 1);
    }
    return false;
}

const char *check_heads(const tc_heads *h, uint64_t n_tokens, uint32_t head_dim, uint32_t item, bool has_out) {
    if (!h->n_heads) return "no heads";
    if (!h->x || (has_out && !h->out)) return "null argument";
    if (reinterpret_cast<uintptr_t>(h->x) % item || (has_out && reinterpret_cast<uintptr_t>(h->out) % item) ||
        reinterpret_cast<uintptr_t>(h->weight) % 4)
        return "misaligned pointer";
    if ((h->ld_token | h->ld_head | h->ld_out_token | h->ld_out_head) >> 38) return "invalid/overlapping head stride";
    if (has_out) {
        if (rows_overlap(n_tokens, h->ld_out_token, h->n_heads, h->ld_out_head, head_dim)) return "invalid/overlapping head stride";
    }
    return nullptr;
}

// Fills the rotation of `p`; nullptr: fine.
const char *take_rope(HeadsParams &p, const tc_rope *r, uint32_t head_dim, bool own_positions, bool &half) {
    half = true;
    p.amplitude = 1.f;
    if (!r) return nullptr;
    if (!r->freq) return "null argument";
    if (!r->rotary_dim || r->rotary_dim % 8 || r->rotary_dim > head_dim)
        return "rotary_dim must be a multiple of 8, at most head_dim";
    if (r->layout != TC_ROPE_HALF && r->layout != TC_ROPE_INTERLEAVED) return "invalid rotation layout";
    if (r->n_axes < 1 || r->n_axes > 4) return "1 to 4 position axes";
    if (!r->positions && (!own_positions || r->n_axes != 1)) return "the rotation needs positions";
    uint64_t end = 0;
    for (uint32_t a = 0; a < r->n_axes; ++a) {
        end += r->n_axes == 1 ? r->rotary_dim / 2 : r->sections[a];
        p.axis_end[a] = end > 0xffffffffu ? 0xffffffffu : (uint32_t)end;
    }
    if (end != r->rotary_dim / 2) return "the sections must add up to rotary_dim / 2";
    half = r->layout == TC_ROPE_HALF;
    p.freq = r->freq;
    p.positions = r->positions;
    p.rotary_units = r->rotary_dim / 8;
    p.half = r->rotary_dim / 2;
    p.n_axes = r->n_axes;
    p.amplitude = r->amplitude;
    return nullptr;
}

const char *check_dim(uint32_t head_dim) {
    return head_dim && head_dim % 8 == 0 && head_dim <= 256 ? nullptr
                                                              : "head_dim must be a multiple of 8, at most 256";
}

const char *take_norm(HeadsParams &p, int rms_norm, float eps, uint32_t head_dim) {
    if (rms_norm && !(eps >= 0.f)) return "eps must not be negative";
    p.rms_norm = rms_norm != 0;
    p.eps = eps;
    p.inv_dim = 1.f / (float)head_dim;
    p.head_dim = head_dim;
    return nullptr;
}

int cuda_fail(const char *what, cudaError_t e) {
    set_last_error(std::string(what) + ": " + cudaGetErrorString(e));
    return TC_CUDA_FAIL;
}

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

}  // namespace

bool rows_overlap(uint64_t a, uint64_t ld_a, uint64_t b, uint64_t ld_b, uint64_t width) {
    Extent e[2] = {{a, ld_a}, {b, ld_b}};
    return overlap(e, 2, width);
}

const char *check_cache(const tc_paged_cache *c, CacheView &v) {
    if (!c || !c->k || !c->v) return "null argument";
    if (c->dtype != TC_DTYPE_F16 && c->dtype != TC_DTYPE_BF16) return "the cache holds f16 or bf16";
    if (const char *e = check_dim(c->head_dim)) return e;
    if (!c->n_heads || !c->n_pages) return "the cache has no pages or no heads";
    if (c->n_pages > 0x7fffffffu) return "too many pages";
    if (c->page_size < 8 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
        return "page_size must be a power of two from 8 to 65536";
    if ((c->ld_page | c->ld_head | c->ld_token) % 8 || (reinterpret_cast<uintptr_t>(c->k) |
                                                        reinterpret_cast<uintptr_t>(c->v)) % 16)
        return "cache buffers must be 16-byte aligned with strides of multiples of 8 elements";
    if ((c->ld_page | c->ld_head | c->ld_token) >> 38) return "invalid/overlapping cache stride";
    Extent e[3] = {{c->n_pages, c->ld_page}, {c->n_heads, c->ld_head}, {c->page_size, c->ld_token}};
    if (overlap(e, 3, c->head_dim)) return "invalid/overlapping cache stride";
    v.k = static_cast<uint16_t *>(c->k);
    v.v = static_cast<uint16_t *>(c->v);
    v.ld_page = c->ld_page;
    v.ld_head = c->ld_head;
    v.ld_token = c->ld_token;
    v.n_pages = c->n_pages;
    v.page_size = c->page_size;
    v.page_shift = (uint32_t)__builtin_ctz(c->page_size);
    v.n_heads = c->n_heads;
    v.head_dim = c->head_dim;
    return nullptr;
}

const char *check_batch(const tc_paged_batch *b, BatchView &v) {
    if (!b) return "null argument";
    if (b->n_tokens && (!b->n_seq || !b->new_offsets || !b->lengths)) return "null argument";
    if (b->n_tokens && b->table_width && !b->page_table) return "null argument";
    if (b->n_tokens > 0x7fffffffu || b->n_seq > 0xffffffu) return "too many tokens or requests";
    if (b->ld_table < b->table_width) return "invalid/overlapping page table stride";
    if (b->max_length > (uint32_t)kMaxLength) return "a request holds at most 2^30 tokens";
    v.new_offsets = b->new_offsets;
    v.lengths = b->lengths;
    v.page_table = b->page_table;
    v.n_seq = b->n_seq;
    v.table_width = b->table_width;
    v.ld_table = b->ld_table;
    v.n_tokens = b->n_tokens;
    v.max_new = b->max_new < b->n_tokens ? b->max_new : b->n_tokens;
    v.max_length = b->max_length;
    return nullptr;
}

}  // namespace tc

extern "C" {

int tc_rope_freqs(uint32_t rotary_dim, double theta, uint32_t scaling, double factor, double trained_length,
                  double beta_fast, double beta_slow, double *freq, float *amplitude) {
    using namespace tc;
    if (!freq || !amplitude) return fail("null argument");
    if (!rotary_dim || rotary_dim % 2) return fail("rotary_dim must be even");
    if (!(theta > 0.0) || !std::isfinite(theta)) return fail("theta must be positive");
    if (scaling > TC_ROPE_BANDS) return fail("unknown rotation scaling");
    if (scaling != TC_ROPE_PLAIN && (!(factor >= 1.0) || !std::isfinite(factor))) return fail("factor must be at least 1");
    if (scaling == TC_ROPE_NTK && rotary_dim <= 2) return fail("this scaling needs rotary_dim above 2");
    if (scaling == TC_ROPE_YARN || scaling == TC_ROPE_BANDS) {
        if (!(trained_length > 0.0) || !(beta_slow > 0.0) || !(beta_fast > beta_slow))
            return fail("trained_length and beta_fast > beta_slow must be positive");
        if (scaling == TC_ROPE_YARN && !(theta > 1.0)) return fail("this scaling needs theta above 1");
    }
    const double two_pi = 6.283185307179586476925, d = rotary_dim;
    const uint32_t n = rotary_dim / 2;
    if (scaling == TC_ROPE_NTK) theta *= std::pow(factor, d / (d - 2.0));
    double low = 0.0, high = 0.0;
    if (scaling == TC_ROPE_YARN) {
        // pair index that turns beta times in trained_length
        low = std::floor(d * std::log(trained_length / (beta_fast * two_pi)) / (2.0 * std::log(theta)));
        high = std::ceil(d * std::log(trained_length / (beta_slow * two_pi)) / (2.0 * std::log(theta)));
        low = low < 0.0 ? 0.0 : low;
        high = high > d - 1.0 ? d - 1.0 : high;
        if (high <= low) high = low + 0.001;
    }
    *amplitude = scaling == TC_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.f;
    for (uint32_t i = 0; i < n; ++i) {
        double f = std::pow(theta, -2.0 * i / d);
        double keep = 1.0;   // share of the unscaled frequency
        if (scaling == TC_ROPE_LINEAR) keep = 0.0;
        if (scaling == TC_ROPE_YARN) keep = 1.0 - (i - low) / (high - low);
        if (scaling == TC_ROPE_BANDS) keep = (trained_length * f / two_pi - beta_slow) / (beta_fast - beta_slow);
        keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
        if (scaling != TC_ROPE_PLAIN && scaling != TC_ROPE_NTK) f = f * keep + f / factor * (1.0 - keep);
        freq[i] = f;
    }
    return ok();
}

int tc_cuda_qk_norm_rope(tc_cuda_ctx *ctx, const tc_heads *q, const tc_heads *k, uint64_t n_tokens,
                         uint32_t head_dim, int dtype, int rms_norm, float eps, const tc_rope *rope, void *stream) {
    using namespace tc;
    try {
        if (!ctx || !q) return fail("null argument");
        if (dtype < TC_DTYPE_F32 || dtype > TC_DTYPE_BF16) return fail("invalid dtype");
        if (const char *e = check_dim(head_dim)) return fail(e);
        if (n_tokens > 0x7fffffffu) return fail("too many tokens or requests");
        HeadsParams p{};
        bool half;
        if (const char *e = take_norm(p, rms_norm, eps, head_dim)) return fail(e);
        if (const char *e = take_rope(p, rope, head_dim, false, half)) return fail(e);
        if (!n_tokens) return ok();
        const uint32_t item = dtype == TC_DTYPE_F32 ? 4 : 2;
        bool vec = true;
        const tc_heads *both[2] = {q, k};
        for (const tc_heads *h : both) {
            if (!h) continue;
            if (const char *e = check_heads(h, n_tokens, head_dim, item, true)) return fail(e);
            vec = vec && chunked(h->x, h->ld_token, h->ld_head, item) &&
                  chunked(h->out, h->ld_out_token, h->ld_out_head, item);
        }
        if ((uint64_t)q->n_heads + (k ? k->n_heads : 0) > 65535) return fail("too many heads");
        p.q = view_of(q);
        if (k) p.k = view_of(k);
        p.n_tokens = (uint32_t)n_tokens;
        p.status = ctx->status;
        CurrentDevice guard(ctx->device);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        cudaError_t e;
        if (dtype == TC_DTYPE_F32) e = launch_heads<float, false>(p, half, vec, ctx->sm_count, s);
        else if (dtype == TC_DTYPE_F16) e = launch_heads<__half, false>(p, half, vec, ctx->sm_count, s);
        else e = launch_heads<__nv_bfloat16, false>(p, half, vec, ctx->sm_count, s);
        return e == cudaSuccess ? ok() : cuda_fail("norm and rotation launch", e);
    } catch (...) {
        return TC_CUDA_FAIL;
    }
}

int tc_cuda_kv_append(tc_cuda_ctx *ctx, const tc_paged_cache *cache, const tc_paged_batch *batch, const tc_heads *k,
                      const tc_heads *v, const tc_heads *q, int rms_norm, float eps, const tc_rope *rope,
                      void *stream) {
    using namespace tc;
    try {
        if (!ctx || !k || !v) return fail("null argument");
        HeadsParams p{};
        bool half;
        if (const char *e = check_cache(cache, p.cache)) return fail(e);
        if (const char *e = check_batch(batch, p.batch)) return fail(e);
        const uint32_t head_dim = cache->head_dim;
        if (const char *e = take_norm(p, rms_norm, eps, head_dim)) return fail(e);
        if (const char *e = take_rope(p, rope, head_dim, true, half)) return fail(e);
        if (k->n_heads != cache->n_heads || v->n_heads != cache->n_heads)
            return fail("keys and values must have the cache's heads");
        if (!p.batch.n_tokens) return ok();
        // the cache's chunks always move whole: its alignment is checked
        bool vec = true;
        const tc_heads *all[3] = {k, v, q};
        for (const tc_heads *h : all) {
            if (!h) continue;
            if (const char *e = check_heads(h, p.batch.n_tokens, head_dim, 2, h == q)) return fail(e);
            vec = vec && chunked(h->x, h->ld_token, h->ld_head, 2);
            if (h == q) vec = vec && chunked(h->out, h->ld_out_token, h->ld_out_head, 2);
        }
        if ((uint64_t)k->n_heads + v->n_heads + (q ? q->n_heads : 0) > 65535) return fail("too many heads");
        p.k = view_of(k);
        p.v = view_of(v);
        if (q) p.q = view_of(q);
        p.n_tokens = p.batch.n_tokens;
        p.status = ctx->status;
        CurrentDevice guard(ctx->device);
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        const cudaError_t e = cache->dtype == TC_DTYPE_F16
                                  ? launch_heads<__half, true>(p, half, vec, ctx->sm_count, s)
                                  : launch_heads<__nv_bfloat16, true>(p, half, vec, ctx->sm_count, s);
        return e == cudaSuccess ? ok() : cuda_fail("cache append launch", e);
    } catch (...) {
        return TC_CUDA_FAIL;
    }
}

}  // extern "C"
