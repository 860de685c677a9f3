// AdamW over many tensors in one launch: float master weights, gradients of any of the three types, optional 16-bit
// working copy, states in float or in 8 bits; loss scale undone on the fly, skipped as a whole by the non-finite flag.
//
//   g = grad / scaling      m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2
//   w = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)          (decoupled weight decay)
//
// The step count t lives on the device and is advanced by the kernel, so that a captured step can be replayed.
//
// 8-bit states: e4m3 codes with one float scale (largest magnitude / 448) per 128 elements of a tensor.  m is rounded
// to nearest.  v moves by a thousandth of the gap to g^2 a step, far less than half a step of a 3-bit mantissa: rounded
// to nearest it would never leave its code (simulated over 1500 steps with drifting gradient scales, the update is then
// 50 % off; with stochastic rounding 15 %).  So v is rounded up with the probability of what is cut off, 16 random
// bits an element from Philox4x32-10 keyed by `seed` and counted by (element, tensor, step); a positive v never
// becomes 0, which would make the update m / eps.
//
// Bound by HBM: 8 B of weight, the gradient, the copy and 16 B (float) or 4.125 B (8-bit) of state per element.
#include "common.cuh"

#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

namespace trb {
namespace {

constexpr int kBlock = 128;              // elements that share a scale
constexpr int kChunk = 4096;             // elements a thread block takes at a time: 32 scale blocks
constexpr int kThreads = 256;
constexpr float kE4m3Max = 448.0f;
constexpr float kSmallest = 1.20370622e-35f;    // 2^-116: below it 448 / max or max / 448 would leave the normal range

struct Tensor {                          // one entry of the plan's device image
    float* w;
    const void* g;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    void* copy;
    int64_t n;
    float weight_decay;
    int32_t vec;                         // every pointer allows 16-byte vectors of floats (8 of the copy)
};

struct Header {
    uint32_t done;                       // blocks of the running step that have ended; 0 between steps
    uint32_t pad[3];
};

struct Chunk { int32_t tensor, index; };

size_t tensors_at() { return sizeof(Header); }
size_t chunks_at(int64_t count) { return align_up((int64_t)(sizeof(Header) + (size_t)count * sizeof(Tensor)), 16); }

struct Hyper {
    float lr;
    const float* lr_dev;                 // used instead of lr when not null
    double log_beta1, log_beta2;
    float beta1, beta2, rest1, rest2;    // rest = 1 - beta, taken in double
    float eps;
    const float* scaling;
    const int32_t* skip_flag;
    int32_t* step;
    uint32_t seed_lo, seed_hi;
};

// per-launch scalars that follow from the step count
struct Scalars { float lr, rate, widen, inv_scale; int32_t step; };

__device__ __forceinline__ Scalars scalars_of(const Hyper& h) {
    Scalars s;
    s.step = *h.step;
    const double t = (double)s.step + 1.0;
    s.lr = h.lr_dev ? *h.lr_dev : h.lr;
    s.rate = (float)((double)s.lr / -expm1(t * h.log_beta1));
    s.widen = (float)rsqrt(-expm1(t * h.log_beta2));
    const float sc = h.scaling ? *h.scaling : 1.0f;
    s.inv_scale = sc != 0.f ? 1.0f / sc : 1.0f;
    return s;
}

// The products are rounded one by one (no fused multiply-add): the states are then the same numbers whatever the
// compiler contracts, and 8-bit codes that sit next to a rounding border come out the same everywhere.
__device__ __forceinline__ void moments(float g, float& m, float& v, const Hyper& h) {
    m = __fadd_rn(__fmul_rn(m, h.beta1), __fmul_rn(g, h.rest1));
    v = __fadd_rn(__fmul_rn(v, h.beta2), __fmul_rn(__fmul_rn(g, g), h.rest2));
}

__device__ __forceinline__ float updated(float w, float m, float v, float decay, const Scalars& s, float eps) {
    return w * decay - s.rate * m / (sqrtf(v) * s.widen + eps);
}

// ---------------------------------------------------------------- loads and stores of four consecutive elements
template <int GT>
__device__ __forceinline__ float4 load_grad4(const void* g, int64_t i) {
    if constexpr (GT == TRB200_DTYPE_F32) {
        return *reinterpret_cast<const float4*>(static_cast<const float*>(g) + i);
    } else {
        const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g) + i);
        const float2 a = unpack2_t<GT == TRB200_DTYPE_BF16>(r.x), b = unpack2_t<GT == TRB200_DTYPE_BF16>(r.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
}

template <int GT>
__device__ __forceinline__ float load_grad(const void* g, int64_t i) {
    if constexpr (GT == TRB200_DTYPE_F32) return static_cast<const float*>(g)[i];
    else return load16_t<GT == TRB200_DTYPE_BF16>(static_cast<const uint16_t*>(g) + i);
}

// CT: type of the copy, -1 for none
template <int CT>
__device__ __forceinline__ void store_copy4(void* c, int64_t i, const float (&w)[4]) {
    if constexpr (CT >= 0) {
        constexpr bool kBf16 = CT == TRB200_DTYPE_BF16;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(c) + i) = make_uint2(pack2_t<kBf16>(w[0], w[1]), pack2_t<kBf16>(w[2], w[3]));
    }
}

template <int CT>
__device__ __forceinline__ void store_copy(void* c, int64_t i, float w) {
    if constexpr (CT >= 0) static_cast<uint16_t*>(c)[i] = round16_t<CT == TRB200_DTYPE_BF16>(w);
}

// ---------------------------------------------------------------- float states
template <int GT, int CT>
__device__ __forceinline__ void chunk_float(const Tensor& t, int64_t i0, int64_t n, const Hyper& h, const Scalars& s) {
    const float decay = 1.0f - s.lr * t.weight_decay;
    float* m_ = static_cast<float*>(t.m);
    float* v_ = static_cast<float*>(t.v);
    int64_t done = i0;
    if (t.vec) {
        for (int64_t i = i0 + 4 * (int64_t)threadIdx.x; i + 4 <= n; i += 4 * kThreads) {
            float w[4], g[4], m[4], v[4];
            *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(t.w + i);
            *reinterpret_cast<float4*>(g) = load_grad4<GT>(t.g, i);
            *reinterpret_cast<float4*>(m) = *reinterpret_cast<const float4*>(m_ + i);
            *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(v_ + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                moments(g[j] * s.inv_scale, m[j], v[j], h);
                w[j] = updated(w[j], m[j], v[j], decay, s, h.eps);
            }
            *reinterpret_cast<float4*>(t.w + i) = *reinterpret_cast<const float4*>(w);
            *reinterpret_cast<float4*>(m_ + i) = *reinterpret_cast<const float4*>(m);
            *reinterpret_cast<float4*>(v_ + i) = *reinterpret_cast<const float4*>(v);
            store_copy4<CT>(t.copy, i, w);
        }
        done = i0 + (n - i0) / 4 * 4;
    }
    for (int64_t i = done + threadIdx.x; i < n; i += kThreads) {
        float m = m_[i], v = v_[i];
        moments(load_grad<GT>(t.g, i) * s.inv_scale, m, v, h);
        const float w = updated(t.w[i], m, v, decay, s, h.eps);
        t.w[i] = w;
        m_[i] = m;
        v_[i] = v;
        store_copy<CT>(t.copy, i, w);
    }
}

// ---------------------------------------------------------------- 8-bit states
struct Philox4 { uint32_t v[4]; };

__device__ __forceinline__ Philox4 philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0,
                                                 uint32_t k1) {
    constexpr uint32_t kM0 = 0xD2511F53u, kM1 = 0xCD9E8D57u, kW0 = 0x9E3779B9u, kW1 = 0xBB67AE85u;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint32_t hi0 = __umulhi(kM0, c0), lo0 = kM0 * c0;
        const uint32_t hi1 = __umulhi(kM1, c2), lo1 = kM1 * c2;
        const uint32_t n0 = hi1 ^ c1 ^ k0, n2 = hi0 ^ c3 ^ k1;
        c0 = n0; c1 = lo1; c2 = n2; c3 = lo0;
        k0 += kW0; k1 += kW1;
    }
    return Philox4{{c0, c1, c2, c3}};
}

__device__ __forceinline__ void unpack_e4m3(uint32_t codes, float scale, float (&f)[4]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> (16 * k)), __NV_E4M3);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h));
        f[2 * k] = a.x * scale;
        f[2 * k + 1] = a.y * scale;
    }
}

__device__ __forceinline__ uint32_t pack_nearest(const float (&f)[4], float up) {
    const auto lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0] * up, f[1] * up), __NV_SATFINITE, __NV_E4M3);
    const auto hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2] * up, f[3] * up), __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)lo | (uint32_t)hi << 16;
}

// e4m3 code of y in [0, 448], rounded up with probability r / 65536 of a step: from 2^-6 on a step is 2^20 in the
// float's bits; below, y + 2^-6 lies in one binade whose steps of 2^20 are the subnormal steps of 2^-9
__device__ __forceinline__ uint32_t code_stochastic(float y, uint32_t r) {
    const bool normal = y >= 0.015625f;
    const float z = normal ? y : y + 0.015625f;
    const uint32_t c = ((__float_as_uint(z) + (r << 4)) >> 20) - (normal ? 960u : 968u);
    return c == 0u && y > 0.f ? 1u : c;
}

// largest of non-negative floats over the warp, NaN above all (bits of such floats order as integers)
__device__ __forceinline__ float warp_top(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v))); }

// an infinite largest value leaves nothing to scale by: NaN, as for a NaN
__device__ __forceinline__ float scale_of(float top) {
    return top < kSmallest ? 0.f : (top == INFINITY ? NAN : __fmul_rn(top, 1.0f / kE4m3Max));
}

// One scale block by one warp: lane l has elements 4l .. 4l + 3; `r` = their random halves.
template <int GT, int CT>
__device__ __forceinline__ void block_8bit(const Tensor& t, int64_t block, int64_t n, const uint32_t (&r)[4], const Hyper& h,
                                           const Scalars& s, float decay) {
    const int lane = threadIdx.x & 31;
    const int64_t i = block * kBlock + 4 * lane;
    uint8_t* m_ = static_cast<uint8_t*>(t.m);
    uint8_t* v_ = static_cast<uint8_t*>(t.v);
    const bool whole = t.vec && (block + 1) * kBlock <= n;      // the same in every lane
    float w[4] = {}, g[4] = {}, m[4] = {}, v[4] = {};
    const float ms = t.m_scale[block], vs = t.v_scale[block];
    if (whole) {
        *reinterpret_cast<float4*>(w) = *reinterpret_cast<const float4*>(t.w + i);
        *reinterpret_cast<float4*>(g) = load_grad4<GT>(t.g, i);
        unpack_e4m3(*reinterpret_cast<const uint32_t*>(m_ + i), ms, m);
        unpack_e4m3(*reinterpret_cast<const uint32_t*>(v_ + i), vs, v);
    } else {
        uint32_t mc = 0, vc = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) {
                w[j] = t.w[i + j];
                g[j] = load_grad<GT>(t.g, i + j);
                mc |= (uint32_t)m_[i + j] << (8 * j);
                vc |= (uint32_t)v_[i + j] << (8 * j);
            }
        unpack_e4m3(mc, ms, m);
        unpack_e4m3(vc, vs, v);
    }
    float mt = 0.f, vt = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        moments(g[j] * s.inv_scale, m[j], v[j], h);
        w[j] = updated(w[j], m[j], v[j], decay, s, h.eps);
        // as integers, so that a NaN is the largest
        mt = __uint_as_float(max(__float_as_uint(mt), __float_as_uint(fabsf(m[j]))));
        vt = __uint_as_float(max(__float_as_uint(vt), __float_as_uint(fabsf(v[j]))));
    }
    mt = warp_top(mt);
    vt = warp_top(vt);
    const float m_up = mt < kSmallest ? 0.f : __fmul_rn(__frcp_rn(mt), kE4m3Max);
    const float v_up = vt < kSmallest ? 0.f : __fmul_rn(__frcp_rn(vt), kE4m3Max);
    const uint32_t mc = pack_nearest(m, m_up);
    uint32_t vc = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) vc |= code_stochastic(fminf(v[j] * v_up, kE4m3Max), r[j]) << (8 * j);
    if (whole) {
        *reinterpret_cast<float4*>(t.w + i) = *reinterpret_cast<const float4*>(w);
        *reinterpret_cast<uint32_t*>(m_ + i) = mc;
        *reinterpret_cast<uint32_t*>(v_ + i) = vc;
        store_copy4<CT>(t.copy, i, w);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < n) {
                t.w[i + j] = w[j];
                m_[i + j] = (uint8_t)(mc >> (8 * j));
                v_[i + j] = (uint8_t)(vc >> (8 * j));
                store_copy<CT>(t.copy, i + j, w[j]);
            }
    }
    if (lane == 0) {
        t.m_scale[block] = scale_of(mt);
        t.v_scale[block] = scale_of(vt);
    }
}

template <int GT, int CT>
__device__ __forceinline__ void chunk_8bit(const Tensor& t, int tensor, int64_t i0, int64_t n, const Hyper& h, const Scalars& s) {
    const float decay = 1.0f - s.lr * t.weight_decay;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // two blocks share a counter: eight elements a lane, sixteen bits each
    for (int64_t pair = i0 / (2 * kBlock) + warp; pair * 2 * kBlock < n; pair += kThreads / 32) {
        const uint64_t group = (uint64_t)pair * 32 + lane;
        const Philox4 x = philox4x32_10((uint32_t)group, (uint32_t)tensor, (uint32_t)s.step, (uint32_t)(group >> 32),
                                        h.seed_lo, h.seed_hi);
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = x.v[j] & 0xffffu;
        block_8bit<GT, CT>(t, 2 * pair, n, r, h, s, decay);
        if ((2 * pair + 1) * kBlock < n) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[j] = x.v[j] >> 16;
            block_8bit<GT, CT>(t, 2 * pair + 1, n, r, h, s, decay);
        }
    }
}

// Persistent blocks over the plan's chunks.  The last block to end advances the step count: by then every block has
// read it.
template <int GT, int CT, bool E8>
__global__ void __launch_bounds__(kThreads)
adamw_kernel(Header* __restrict__ head, const Tensor* __restrict__ tensors, const Chunk* __restrict__ chunks, int count, Hyper h) {
    if (h.skip_flag && *h.skip_flag) return;
    __shared__ Scalars s_scalars;
    if (threadIdx.x == 0) s_scalars = scalars_of(h);
    __syncthreads();
    const Scalars s = s_scalars;
    for (int c = blockIdx.x; c < count; c += gridDim.x) {
        const Chunk ch = chunks[c];
        const Tensor t = tensors[ch.tensor];
        const int64_t i0 = (int64_t)ch.index * kChunk;
        const int64_t n = t.n - i0 < kChunk ? t.n : i0 + kChunk;
        if constexpr (E8) chunk_8bit<GT, CT>(t, ch.tensor, i0, n, h, s);
        else chunk_float<GT, CT>(t, i0, n, h, s);
    }
    if (threadIdx.x == 0 && atomicAdd(&head->done, 1u) == gridDim.x - 1) {
        head->done = 0u;
        *h.step = s.step + 1;
    }
}

template <int GT, int CT>
void launch(bool e8, int grid, cudaStream_t st, Header* head, const Tensor* t, const Chunk* c, int count, const Hyper& h) {
    if (e8) adamw_kernel<GT, CT, true><<<grid, kThreads, 0, st>>>(head, t, c, count, h);
    else adamw_kernel<GT, CT, false><<<grid, kThreads, 0, st>>>(head, t, c, count, h);
}

template <int GT>
void launch(int copy, bool e8, int grid, cudaStream_t st, Header* head, const Tensor* t, const Chunk* c, int count, const Hyper& h) {
    if (copy == TRB200_DTYPE_F16) launch<GT, TRB200_DTYPE_F16>(e8, grid, st, head, t, c, count, h);
    else if (copy == TRB200_DTYPE_BF16) launch<GT, TRB200_DTYPE_BF16>(e8, grid, st, head, t, c, count, h);
    else launch<GT, -1>(e8, grid, st, head, t, c, count, h);
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// chunks of all tensors, or -1 for a bad description
int64_t count_chunks(const trb200_adamw_tensor* tensors, int32_t count) {
    int64_t total = 0;
    for (int32_t i = 0; i < count; ++i) {
        if (tensors[i].n < 0 || tensors[i].n > ((int64_t)1 << 42)) return -1;
        total += chunks_of(tensors[i].n);
    }
    return total;
}

int grad_size(int dtype) { return dtype == TRB200_DTYPE_F32 ? 4 : 2; }

struct Range { uintptr_t from, to; bool written; };

// the tensors' buffers are disjoint, but for gradients, which may share memory among themselves
int check_disjoint(std::vector<Range>& r) {
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t any = 0, written = 0;      // ends of the ranges so far
    for (const Range& x : r) {
        if (x.from < (x.written ? any : written)) return 0;
        any = std::max(any, x.to);
        if (x.written) written = std::max(written, x.to);
    }
    return 1;
}

int write_plan(const trb200_adamw_tensor* in, int32_t count, int32_t grad_dtype, int32_t copy_dtype, int32_t state_bits,
               void* image, size_t image_bytes, trb200_adamw_plan* plan) {
    TRB_REQUIRE(plan && image && (in || count == 0) && count >= 0, TRB200_ERR_INVALID_ARGUMENT, "adamw_plan: null pointer or negative count");
    TRB_REQUIRE(valid_dtype(grad_dtype) || grad_dtype == TRB200_DTYPE_F32, TRB200_ERR_INVALID_ARGUMENT,
                "adamw_plan: unknown gradient dtype %d", grad_dtype);
    TRB_REQUIRE(valid_dtype(copy_dtype) || copy_dtype == TRB200_DTYPE_NONE, TRB200_ERR_INVALID_ARGUMENT,
                "adamw_plan: unknown dtype %d of the copy", copy_dtype);
    TRB_REQUIRE(state_bits == 32 || state_bits == 8, TRB200_ERR_INVALID_ARGUMENT, "adamw_plan: states have 32 or 8 bits, not %d", state_bits);
    const int64_t chunks = count_chunks(in, count);
    TRB_REQUIRE(chunks >= 0 && chunks <= 0x7fffffff, TRB200_ERR_INVALID_ARGUMENT, "adamw_plan: bad tensor size");
    TRB_REQUIRE(image_bytes >= chunks_at(count) + (size_t)chunks * sizeof(Chunk), TRB200_ERR_WORKSPACE, "adamw_plan: image too small");
    const bool e8 = state_bits == 8;
    char* base = static_cast<char*>(image);
    memset(base, 0, chunks_at(count));
    Chunk* ch = reinterpret_cast<Chunk*>(base + chunks_at(count));
    std::vector<Range> ranges;
    ranges.reserve((size_t)count * 7);
    for (int32_t i = 0; i < count; ++i) {
        const trb200_adamw_tensor& t = in[i];
        if (t.n == 0) continue;
        TRB_REQUIRE(t.w && t.g && t.m && t.v && (!e8 || (t.m_scale && t.v_scale)) && (copy_dtype == TRB200_DTYPE_NONE || t.copy),
                    TRB200_ERR_INVALID_ARGUMENT, "adamw_plan: null pointer in tensor %d", i);
        const uintptr_t w = reinterpret_cast<uintptr_t>(t.w), g = reinterpret_cast<uintptr_t>(t.g),
                        m = reinterpret_cast<uintptr_t>(t.m), v = reinterpret_cast<uintptr_t>(t.v),
                        ms = reinterpret_cast<uintptr_t>(t.m_scale), vs = reinterpret_cast<uintptr_t>(t.v_scale),
                        c = reinterpret_cast<uintptr_t>(t.copy);
        const bool copied = copy_dtype != TRB200_DTYPE_NONE;
        TRB_REQUIRE((w & 3u) == 0 && (g & (uintptr_t)(grad_size(grad_dtype) - 1)) == 0 && (e8 || ((m | v) & 3u) == 0) &&
                        (!e8 || ((ms | vs) & 3u) == 0) && (!copied || (c & 1u) == 0),
                    TRB200_ERR_INVALID_ARGUMENT, "adamw_plan: tensor %d is not aligned to its elements", i);
        TRB_REQUIRE(std::isfinite(t.weight_decay) && t.weight_decay >= 0.f, TRB200_ERR_INVALID_ARGUMENT,
                    "adamw_plan: bad weight decay in tensor %d", i);
        const uintptr_t n = (uintptr_t)t.n, state = e8 ? 1 : 4, scales = (n + kBlock - 1) / kBlock * 4;
        ranges.push_back({w, w + 4 * n, true});
        ranges.push_back({g, g + (uintptr_t)grad_size(grad_dtype) * n, false});
        ranges.push_back({m, m + state * n, true});
        ranges.push_back({v, v + state * n, true});
        if (e8) {
            ranges.push_back({ms, ms + scales, true});
            ranges.push_back({vs, vs + scales, true});
        }
        if (copied) ranges.push_back({c, c + 2 * n, true});
        const bool vec = (w & 15u) == 0 && (g & (uintptr_t)(4 * grad_size(grad_dtype) - 1)) == 0 &&
                         ((m | v) & (e8 ? 3u : 15u)) == 0 && (!copied || (c & 7u) == 0);
        const Tensor d{t.w, t.g, t.m, t.v, t.m_scale, t.v_scale, copied ? t.copy : nullptr, t.n, t.weight_decay, vec ? 1 : 0};
        memcpy(base + tensors_at() + (size_t)i * sizeof(Tensor), &d, sizeof(d));
        for (int64_t k = 0; k < chunks_of(t.n); ++k) {
            const Chunk x{i, (int32_t)k};
            memcpy(ch++, &x, sizeof(x));
        }
    }
    TRB_REQUIRE(check_disjoint(ranges), TRB200_ERR_INVALID_ARGUMENT,
                "adamw_plan: a buffer that is written overlaps another one (is a tensor listed twice?)");
    *plan = trb200_adamw_plan{nullptr, count, (int32_t)chunks, grad_dtype, copy_dtype, state_bits};
    return TRB200_OK;
}

}  // namespace
}  // namespace trb

extern "C" size_t trb200_adamw_plan_bytes(const trb200_adamw_tensor* tensors, int32_t count) {
    if (count < 0 || (count > 0 && !tensors)) return 0;
    const int64_t chunks = trb::count_chunks(tensors, count);
    if (chunks < 0 || chunks > 0x7fffffff) return 0;
    return trb::chunks_at(count) + (size_t)chunks * sizeof(trb::Chunk);
}

extern "C" int trb200_adamw_plan_write(const trb200_adamw_tensor* tensors, int32_t count, int32_t grad_dtype,
                                       int32_t copy_dtype, int32_t state_bits, void* host_image, size_t image_bytes,
                                       trb200_adamw_plan* plan) {
    try {
        return trb::write_plan(tensors, count, grad_dtype, copy_dtype, state_bits, host_image, image_bytes, plan);
    } catch (...) {
        return trb::fail(TRB200_ERR_INVALID_ARGUMENT, "adamw_plan: out of host memory");
    }
}

extern "C" int trb200_adamw_step(const trb200_adamw_plan* plan, int32_t* step, float lr, const float* lr_dev, double beta1,
                                 double beta2, float eps, const float* scaling, const int32_t* skip_flag, uint64_t seed,
                                 void* stream) {
    TRB_REQUIRE(plan && plan->image && step, TRB200_ERR_INVALID_ARGUMENT, "adamw_step: null pointer");
    TRB_REQUIRE((reinterpret_cast<uintptr_t>(plan->image) & 15u) == 0, TRB200_ERR_INVALID_ARGUMENT,
                "adamw_step: the plan's image must be 16-byte aligned");
    TRB_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, TRB200_ERR_INVALID_ARGUMENT,
                "adamw_step: beta1 and beta2 must lie in [0, 1)");
    TRB_REQUIRE(eps > 0.f && std::isfinite(eps) && std::isfinite(lr), TRB200_ERR_INVALID_ARGUMENT,
                "adamw_step: eps must be positive, lr finite");
    TRB_REQUIRE(plan->count >= 0 && plan->chunks >= 0 &&
                    (trb::valid_dtype(plan->grad_dtype) || plan->grad_dtype == TRB200_DTYPE_F32) &&
                    (trb::valid_dtype(plan->copy_dtype) || plan->copy_dtype == TRB200_DTYPE_NONE) &&
                    (plan->state_bits == 32 || plan->state_bits == 8),
                TRB200_ERR_INVALID_ARGUMENT, "adamw_step: not a plan that trb200_adamw_plan_write wrote");
    char* base = static_cast<char*>(plan->image);
    auto* head = reinterpret_cast<trb::Header*>(base);
    const auto* tensors = reinterpret_cast<const trb::Tensor*>(base + trb::tensors_at());
    const auto* chunks = reinterpret_cast<const trb::Chunk*>(base + trb::chunks_at(plan->count));
    const trb::Hyper h{lr, lr_dev, std::log(beta1), std::log(beta2), (float)beta1, (float)beta2, (float)(1.0 - beta1),
                       (float)(1.0 - beta2), eps, scaling, skip_flag, step, (uint32_t)seed, (uint32_t)(seed >> 32)};
    int grid = trb::sm_count() * 8;
    if (grid > plan->chunks) grid = plan->chunks;
    if (grid < 1) grid = 1;                                  // no elements: the step still counts
    const bool e8 = plan->state_bits == 8;
    cudaStream_t st = trb::as_stream(stream);
    if (plan->grad_dtype == TRB200_DTYPE_F32)
        trb::launch<TRB200_DTYPE_F32>(plan->copy_dtype, e8, grid, st, head, tensors, chunks, plan->chunks, h);
    else if (plan->grad_dtype == TRB200_DTYPE_F16)
        trb::launch<TRB200_DTYPE_F16>(plan->copy_dtype, e8, grid, st, head, tensors, chunks, plan->chunks, h);
    else
        trb::launch<TRB200_DTYPE_BF16>(plan->copy_dtype, e8, grid, st, head, tensors, chunks, plan->chunks, h);
    TRB_LAUNCH_CHECK("adamw");
    return TRB200_OK;
}
