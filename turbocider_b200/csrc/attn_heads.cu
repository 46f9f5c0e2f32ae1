// Norm and position rotation of query and key heads, alone
// (tc_cuda_qk_norm_rope) or on the way into a paged cache
// (tc_cuda_kv_append).  For a head x of head_dim elements
//     y = x * rsqrt(mean(x^2) + eps) * weight
//     (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t)
// over its rotary pairs, t = position * freq.
//
// Bytes bound: every element is read once and written once (2 + 2 bytes for
// 16-bit types) against about 10 flops.  A head is spread over the smallest
// power-of-two group of lanes that gives each lane one unit of 16 elements (8
// for f32 and for odd sizes): two chunks half a rotary width apart for the
// half layout, half a head apart for the interleaved one (whole sectors per
// access), so that both members of every pair are in one lane, the rotation
// needs no exchange and the norm one butterfly over the group.  A warp takes one
// token and some or all of its heads, kBatch for each lane group at a time; the
// token's sines and cosines are formed once per warp, the norm's weights folded
// into them, and the arithmetic is packed two fp32 to an operation: with 8-byte
// chunks and plain arithmetic half of the time went into issuing instructions.
// 8448 tokens x 60 heads of 128 (260 MB): 53.5 us, 4.9 TB/s; appending 281 MB:
// 58.6 us.  Batches read ahead took 62 and 130 us, four warps a token with shared
// sines and cosines 60 and 80 at best.  The limit of 80 registers (six blocks an
// SM) costs five of the eight 8-element forms 4 to 16 bytes of spills a thread.
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
#include "kq_sm100.cuh"

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
    uint32_t head_dim, n_tokens, groups, heads_per_group;
    int rms_norm;
    float eps, inv_dim;
    // rotation
    const double *freq;
    const int32_t *positions;
    uint32_t half, n_axes, axis_end[4];
    float amplitude;
    // append
    BatchView batch;
    CacheView cache;
    uint32_t *status;
};

// Elements in and out of fp32.
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

// A lane's unit of a head: two chunks of CH elements.
template <class T, int CH>
struct alignas(CH * sizeof(T) < 16 ? CH * sizeof(T) : 16) Chunk { T v[CH]; };
template <class T, int CH>
struct Unit { Chunk<T, CH> c[2]; };

// WIDE: accesses of whole chunks are aligned.
template <class T, int CH, bool WIDE>
__device__ __forceinline__ void load_unit(Unit<T, CH> &u, const T *p, const uint32_t (&at)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (WIDE) u.c[k] = *reinterpret_cast<const Chunk<T, CH> *>(p + at[k]);
        else
#pragma unroll
            for (int i = 0; i < CH; ++i) u.c[k].v[i] = p[at[k] + i];
    }
}
template <class T, int CH, bool WIDE>
__device__ __forceinline__ void store_unit(T *p, const uint32_t (&at)[2], const Unit<T, CH> &u) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (WIDE) *reinterpret_cast<Chunk<T, CH> *>(p + at[k]) = u.c[k];
        else
#pragma unroll
            for (int i = 0; i < CH; ++i) p[at[k] + i] = u.c[k].v[i];
    }
}

// Request of token t: the number of requests that end at or before it
// (n_seq: t belongs to none).
__device__ __forceinline__ uint32_t request_of(const BatchView &bt, int32_t t) {
    return count_prefix(bt.n_seq, [&](uint32_t b) { return bt.new_offsets[b] <= t; });
}

constexpr int kBlocks = 6;   // resident per SM (at most 80 registers a thread)
constexpr int kWarps = 4, kBatch = 2;   // warps of a block; heads that a lane has in flight

// What a lane keeps for every head it visits.
struct Lane {
    uint32_t at[2], lanes, slot, slots;   // elements where its chunks begin
    bool active, rotates[2];              // chunk k is rotated
    uint32_t pair[2];                     // pair of chunk k's first element
};

// Members of a unit's pairs as fp32: a[i], b[i] are elements i of its chunks
// (half layout) or neighbours (the first half of them in chunk 0).
template <class T, int CH, bool HALF>
__device__ __forceinline__ void unpack(const Unit<T, CH> &u, float (&a)[CH], float (&b)[CH]) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        a[i] = to_float<T>(HALF ? u.c[0].v[i] : u.c[2 * i / CH].v[2 * i % CH]);
        b[i] = to_float<T>(HALF ? u.c[1].v[i] : u.c[2 * i / CH].v[2 * i % CH + 1]);
    }
}
template <class T, int CH, bool HALF>
__device__ __forceinline__ void pack(Unit<T, CH> &u, const float (&a)[CH], const float (&b)[CH]) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        (HALF ? u.c[0].v[i] : u.c[2 * i / CH].v[2 * i % CH]) = from_float<T>(a[i]);
        (HALF ? u.c[1].v[i] : u.c[2 * i / CH].v[2 * i % CH + 1]) = from_float<T>(b[i]);
    }
}
// Two fp32 lanes in one operation (sm_100a).
__device__ __forceinline__ uint64_t two(float lo, float hi) {
    return f2pack(__float_as_uint(lo), __float_as_uint(hi));
}

// Heads [begin, end) of one kind, `slots` at a time: norm, rotation, store.
// The heads of a batch are all read before the first is written (out may be x).
template <class T, int CH, bool HALF, bool WIDE>
__device__ __forceinline__ void turn_heads(const HeadsParams &p, const Lane &ln, const float2 *turn, const T *x, uint64_t ld_x, T *out,
                                           uint64_t ld_out, const float *weight, uint32_t begin, uint32_t end,
                                           bool store) {
    if (begin >= end) return;
    // a' = r (a wa cos - b wb sin), b' = r (b wb cos + a wa sin); a chunk past
    // the rotated part keeps a' = r a wa, b' = r b wb
    uint64_t aa[CH / 2], ab[CH / 2], bb[CH / 2], ba[CH / 2];
#pragma unroll
    for (int i = 0; i < CH; i += 2) {
        float wa[2] = {1.f, 1.f}, wb[2] = {1.f, 1.f};
        float2 cs[2] = {{1.f, 0.f}, {1.f, 0.f}};
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int e = i + k, c = HALF ? 0 : 2 * e / CH;   // chunk of a
            if (weight) {
                wa[k] = weight[HALF ? ln.at[0] + e : ln.at[c] + 2 * e % CH];
                wb[k] = weight[HALF ? ln.at[1] + e : ln.at[c] + 2 * e % CH + 1];
            }
            if (ln.rotates[c]) cs[k] = turn[ln.pair[c] + (HALF ? e : e % (CH / 2))];
        }
        aa[i / 2] = two(wa[0] * cs[0].x, wa[1] * cs[1].x);
        ab[i / 2] = two(-wb[0] * cs[0].y, -wb[1] * cs[1].y);
        bb[i / 2] = two(wb[0] * cs[0].x, wb[1] * cs[1].x);
        ba[i / 2] = two(wa[0] * cs[0].y, wa[1] * cs[1].y);
    }
    store = store && ln.active;
    // (every lane runs every round: the butterfly of the norm needs them all)
    for (uint32_t h0 = begin + ln.slot; h0 < end + ln.slot; h0 += kBatch * ln.slots) {
        Unit<T, CH> u[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k)
            load_unit<T, CH, WIDE>(u[k], x + min(h0 + k * ln.slots, end - 1) * ld_x, ln.at);
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const uint32_t h = h0 + k * ln.slots;
            float fa[CH], fb[CH];
            unpack<T, CH, HALF>(u[k], fa, fb);
            uint64_t a[CH / 2], b[CH / 2];
#pragma unroll
            for (int i = 0; i < CH; i += 2) {
                a[i / 2] = two(fa[i], fa[i + 1]);
                b[i / 2] = two(fb[i], fb[i + 1]);
            }
            float r = 1.f;
            if (p.rms_norm) {
                uint64_t s = f2mul(a[0], a[0]);
#pragma unroll
                for (int i = 1; i < CH / 2; ++i) s = f2fma(a[i], a[i], s);
#pragma unroll
                for (int i = 0; i < CH / 2; ++i) s = f2fma(b[i], b[i], s);
                float s0, s1;
                f2unpack(s, s0, s1);
                float ss = ln.active ? s0 + s1 : 0.f;
                for (uint32_t d = ln.lanes / 2; d > 0; d /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, d);
                r = rsqrtf(ss * p.inv_dim + p.eps);
            }
            const uint64_t r2 = f2splat(r);
#pragma unroll
            for (int i = 0; i < CH / 2; ++i) {
                uint64_t ya = f2mul(a[i], aa[i]), yb = f2mul(b[i], bb[i]);
                if (ln.rotates[HALF ? 0 : 4 * i / CH]) {
                    ya = f2fma(b[i], ab[i], ya);
                    yb = f2fma(a[i], ba[i], yb);
                }
                f2unpack(f2mul(ya, r2), fa[2 * i], fa[2 * i + 1]);
                f2unpack(f2mul(yb, r2), fb[2 * i], fb[2 * i + 1]);
            }
            if (store && h < end) {
                pack<T, CH, HALF>(u[k], fa, fb);
                store_unit<T, CH, WIDE>(out + h * ld_out, ln.at, u[k]);
            }
        }
    }
}

template <class T, int CH, bool HALF, bool APPEND, bool WIDE>
__global__ void __launch_bounds__(kWarps * 32, kBlocks) heads_kernel(const __grid_constant__ HeadsParams p) {
    __shared__ float2 turns[kWarps][128];   // cos and sin of the token's pairs
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint64_t task = (uint64_t)blockIdx.x * kWarps + warp;
    const uint64_t t = task / p.groups;
    if (t >= p.n_tokens) return;
    const uint32_t units = p.head_dim / (2 * CH);
    Lane ln;
    ln.lanes = units <= 1 ? 1u : 1u << (32 - __clz(units - 1));   // lanes per head
    ln.slot = lane / ln.lanes;
    ln.slots = 32 / ln.lanes;
    const uint32_t own = lane & (ln.lanes - 1);
    ln.active = own < units;
    // (a lane without a unit reads the first one's and adds and stores nothing)
    const uint32_t unit = ln.active ? own : 0u;
    if (HALF) {
        const uint32_t turned = p.half / CH;   // units that are rotated
        ln.rotates[0] = ln.rotates[1] = unit < turned;
        ln.at[0] = unit < turned ? CH * unit : 2 * p.half + CH * (unit - turned);
        ln.at[1] = ln.at[0] + (unit < turned ? p.half : p.head_dim / 2 - p.half);
        ln.pair[0] = ln.pair[1] = CH * unit;
    } else {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            ln.at[k] = CH * unit + k * (p.head_dim / 2);
            ln.rotates[k] = ln.at[k] < 2 * p.half;
            ln.pair[k] = ln.at[k] / 2;
        }
    }

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
    for (uint32_t pair = lane; pair < p.half; pair += 32) {
        int32_t pos = position;
        if (p.positions) {
            uint32_t axis = 0;
            while (axis + 1 < p.n_axes && pair >= p.axis_end[axis]) ++axis;
            pos = p.positions[t * p.n_axes + axis];
        }
        // freq in turns as a fraction of 2^64 (negative ones wrap, whole turns
        // fall away), times the position modulo 2^64
        const double turn = p.freq[pair] * 0.15915494309189533577;   // 1 / (2 pi)
        const uint64_t step = (uint64_t)__double2ull_rn((turn - floor(turn)) * 18446744073709551616.0);
        const uint64_t phase = step * (uint64_t)(int64_t)pos;
        float s, c;
        sincospif((float)(int32_t)(phase >> 32) * 4.656612873077392578125e-10f, &s, &c);   // 2^-31
        turns[warp][pair] = make_float2(c * p.amplitude, s * p.amplitude);
    }
    __syncwarp();

    // this warp's share of the heads: the queries' come first, then the keys', then the values'
    const uint32_t nq = p.q.n_heads, nk = p.k.n_heads, nv = p.v.n_heads;
    const uint32_t h0 = (uint32_t)(task % p.groups) * p.heads_per_group, h1 = h0 + p.heads_per_group;
    turn_heads<T, CH, HALF, WIDE>(p, ln, turns[warp], static_cast<const T *>(p.q.x) + t * p.q.ld_token, p.q.ld_head,
                                  static_cast<T *>(p.q.out) + t * p.q.ld_out_token, p.q.ld_out_head, p.q.weight,
                                  min(h0, nq), min(h1, nq), true);
    const uint32_t k0 = min(max(h0, nq) - nq, nk), k1 = min(max(h1, nq) - nq, nk);
    turn_heads<T, CH, HALF, WIDE>(p, ln, turns[warp], static_cast<const T *>(p.k.x) + t * p.k.ld_token, p.k.ld_head,
                                  APPEND ? reinterpret_cast<T *>(p.cache.k) + k_base
                                         : static_cast<T *>(p.k.out) + t * p.k.ld_out_token,
                                  APPEND ? p.cache.ld_head : p.k.ld_out_head, p.k.weight, k0, k1,
                                  !APPEND || store_kv);
    if (APPEND && store_kv && ln.active) {   // values as they are
        const uint32_t first = nq + nk, v0 = min(max(h0, first) - first, nv), v1 = min(max(h1, first) - first, nv);
        const T *x = static_cast<const T *>(p.v.x) + t * p.v.ld_token;
        T *out = reinterpret_cast<T *>(p.cache.v) + k_base;
#pragma unroll 2
        for (uint32_t h = v0 + ln.slot; h < v1; h += ln.slots) {
            Unit<T, CH> u;
            load_unit<T, CH, WIDE>(u, x + h * p.v.ld_head, ln.at);
            store_unit<T, CH, WIDE>(out + h * p.cache.ld_head, ln.at, u);
        }
    }
}

template <class T, int CH, bool APPEND>
cudaError_t launch_sized(HeadsParams &p, bool half, bool wide, int sm_count, cudaStream_t s) {
    const uint32_t n_all = p.q.n_heads + p.k.n_heads + p.v.n_heads;
    uint32_t lanes = 1;
    while (lanes * 2 * CH < p.head_dim) lanes *= 2;
    // A warp takes one batch of heads while that leaves the GPU underfilled,
    // all heads of a token once there are enough tokens (the angles are formed
    // once per warp).
    const uint32_t slots = 32 / lanes, batch = slots * kBatch;
    const uint64_t batches = (n_all + batch - 1) / batch;
    const uint64_t room = (uint64_t)sm_count * 32;   // warps resident
    uint64_t per = (batches * p.n_tokens + room - 1) / room;
    if (per < 1) per = 1;
    if (per > batches) per = batches;
    p.heads_per_group = (uint32_t)per * batch;
    p.groups = (n_all + p.heads_per_group - 1) / p.heads_per_group;
    const uint64_t blocks = ((uint64_t)p.n_tokens * p.groups + kWarps - 1) / kWarps;
    if (blocks > 0x7fffffffu) return cudaErrorInvalidValue;
    auto launch = [&](auto kernel) { kernel<<<(unsigned)blocks, kWarps * 32, 0, s>>>(p); };
    if (wide) {
        if (half) launch(heads_kernel<T, CH, true, APPEND, true>);
        else launch(heads_kernel<T, CH, false, APPEND, true>);
    } else if constexpr (CH == 4) {   // (chunks of 8 are taken only where they are aligned)
        if (half) launch(heads_kernel<T, CH, true, APPEND, false>);
        else launch(heads_kernel<T, CH, false, APPEND, false>);
    }
    return cudaGetLastError();
}

// Chunks of 8 elements where the sizes allow it and, for f32, of 4.
template <class T, bool APPEND>
cudaError_t launch_heads(HeadsParams &p, bool half, bool wide, int sm_count, cudaStream_t s) {
    if (sizeof(T) == 2 && wide && p.head_dim % 16 == 0 && p.half % 8 == 0)
        return launch_sized<T, sizeof(T) == 2 ? 8 : 4, APPEND>(p, half, true, sm_count, s);
    return launch_sized<T, 4, APPEND>(p, half, wide, sm_count, s);
}

// (the weight belongs to the norm: without one it has no part)
HeadsView view_of(const tc_heads *h, int rms_norm) {
    return {h->x, h->out, rms_norm ? h->weight : nullptr, h->ld_token, h->ld_head, h->ld_out_token, h->ld_out_head, h->n_heads};
}

// Units of a row can be moved by 16-byte accesses.
bool chunked(const void *p, uint64_t ld_token, uint64_t ld_head, uint32_t item) {
    return !(reinterpret_cast<uintptr_t>(p) % 16) && !(ld_token * item % 16) && !(ld_head * item % 16);
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
    try {
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
    } catch (...) {
        return TC_CUDA_FAIL;
    }
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
        p.q = view_of(q, rms_norm);
        if (k) p.k = view_of(k, rms_norm);
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
        p.k = view_of(k, rms_norm);
        p.v = view_of(v, 0);
        if (q) p.q = view_of(q, rms_norm);
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
