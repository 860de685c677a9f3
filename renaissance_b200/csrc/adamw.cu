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
// Bound by HBM: 8 B of weight, the gradient, the copy and 16 B (float) or 4.125 B (8-bit) of state per element.  Float
// states reach it: 138 M elements in 652 us, 0.97 of the copy bandwidth.  8-bit ones come near (480 us, 0.80; 25.6 M
// elements with 16-bit gradients 88 us, 0.72): their 61 instructions an element (decoding, the update, the largest
// magnitude of a block, random bits, encoding) take 64 % of the issue slots, and 24 warps an SM do not hide all of a unit's
// chain of them.  So loads have to be on their way all the time (asynchronous copies, three units ahead a warp), and pairs of
// floats go through the packed instructions.
#include "chained.cuh"
#include "common.cuh"
#include "packed.cuh"

#include <cuda_fp8.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>
#include <vector>

namespace trb {
namespace {

constexpr int kBlock = 128;              // elements that share a scale
constexpr int kUnit = 2 * kBlock;        // elements that the work is counted in; a tensor takes whole units
constexpr int kThreads = 256, kWarps = kThreads / 32;
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

// behind the tensors: count + 1 int32, the units in front of each tensor
size_t tensors_at() { return sizeof(Header); }
size_t units_at(int64_t count) { return sizeof(Header) + (size_t)count * sizeof(Tensor); }
size_t image_size(int64_t count) { return align_up((int64_t)(units_at(count) + (size_t)(count + 1) * sizeof(int32_t)), 16); }

struct Hyper {
    float lr;
    const float* lr_dev;                 // used instead of lr when not null
    double log_beta1, log_beta2;
    float beta1, beta2, rest1, rest2;    // rest = 1 - beta, taken in double
    float eps;
    const float* scaling;
    const int32_t* skip_flag;
    int32_t* step;
    int32_t run;                         // units that a block takes at a time
    float one;                           // 1
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

// Four elements as two pairs of floats: the packed instructions do two in one.
struct Quad { uint64_t a, b; };

__device__ __forceinline__ Quad quad(const float4& f) { return {pair_of(f.x, f.y), pair_of(f.z, f.w)}; }
__device__ __forceinline__ float4 single(const Quad& q) {
    const float2 a = split(q.a), b = split(q.b);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ Quad times(const Quad& q, float f) { return {mul2(q.a, twice(f)), mul2(q.b, twice(f))}; }

// The two products are rounded before they are added: the states are then the same numbers whatever the compiler
// contracts, and 8-bit codes that sit next to a rounding border come out the same everywhere.  A packed addition of
// packed products was seen to be contracted; a multiply-add with a one that the compiler cannot see (h.one) is not.
__device__ __forceinline__ uint64_t moment(uint64_t state, uint64_t fresh, float beta, float rest, const Hyper& h) {
    return fma2(mul2(state, twice(beta)), twice(h.one), mul2(fresh, twice(rest)));
}

__device__ __forceinline__ void moments(const Quad& g, Quad& m, Quad& v, const Hyper& h) {
    m = {moment(m.a, g.a, h.beta1, h.rest1, h), moment(m.b, g.b, h.beta1, h.rest1, h)};
    v = {moment(v.a, mul2(g.a, g.a), h.beta2, h.rest2, h), moment(v.b, mul2(g.b, g.b), h.beta2, h.rest2, h)};
}

// Square root and reciprocal are the approximate ones, together good to 2^-21 of the change (the correctly rounded ones
// would be two roundings, 2^-23, for several times the instructions): next to a weight well above lr the weight's own
// rounding hides it, a weight that starts at 0 carries it.  The square root takes subnormal v as they are: flushed to
// zero, v below 2^-126 would leave eps alone in the denominator.
__device__ __forceinline__ uint64_t updated(uint64_t w, uint64_t m, uint64_t v, float decay, const Scalars& s, float eps) {
    float2 f = split(v);
    asm("sqrt.approx.f32 %0, %0;" : "+f"(f.x));
    asm("sqrt.approx.f32 %0, %0;" : "+f"(f.y));
    f = split(fma2(pair_of(f.x, f.y), twice(s.widen), twice(eps)));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(f.y));
    return fma2(mul2(m, twice(-s.rate)), pair_of(f.x, f.y), mul2(w, twice(decay)));
}

__device__ __forceinline__ Quad updated(const Quad& w, const Quad& m, const Quad& v, float decay, const Scalars& s, float eps) {
    return {updated(w.a, m.a, v.a, decay, s, eps), updated(w.b, m.b, v.b, decay, s, eps)};
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
__device__ __forceinline__ void store_copy4(void* c, int64_t i, const float4& w) {
    if constexpr (CT >= 0) {
        constexpr bool kBf16 = CT == TRB200_DTYPE_BF16;
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(c) + i) = make_uint2(pack2_t<kBf16>(w.x, w.y), pack2_t<kBf16>(w.z, w.w));
    }
}

template <int CT>
__device__ __forceinline__ void store_copy(void* c, int64_t i, float w) {
    if constexpr (CT >= 0) static_cast<uint16_t*>(c)[i] = round16_t<CT == TRB200_DTYPE_BF16>(w);
}

// ---------------------------------------------------------------- float states
// elements [i0, end) of a tensor by a thread block
template <int GT, int CT>
__device__ __forceinline__ void range_float(const Tensor& t, int64_t i0, int64_t end, const Hyper& h, const Scalars& s, float decay) {
    float* const m_ = static_cast<float*>(t.m);
    float* const v_ = static_cast<float*>(t.v);
    int64_t done = i0;
    if (t.vec) {
        for (int64_t i = i0 + 4 * (int64_t)threadIdx.x; i + 4 <= end; i += 4 * kThreads) {
            Quad w = quad(*reinterpret_cast<const float4*>(t.w + i)), m = quad(*reinterpret_cast<const float4*>(m_ + i));
            Quad v = quad(*reinterpret_cast<const float4*>(v_ + i));
            moments(times(quad(load_grad4<GT>(t.g, i)), s.inv_scale), m, v, h);
            w = updated(w, m, v, decay, s, h.eps);
            const float4 w4 = single(w);
            *reinterpret_cast<float4*>(t.w + i) = w4;
            *reinterpret_cast<float4*>(m_ + i) = single(m);
            *reinterpret_cast<float4*>(v_ + i) = single(v);
            store_copy4<CT>(t.copy, i, w4);
        }
        done = i0 + (end - i0) / 4 * 4;
    }
    for (int64_t i = done + threadIdx.x; i < end; i += kThreads) {
        Quad m{twice(m_[i]), 0}, v{twice(v_[i]), 0};
        moments({twice(load_grad<GT>(t.g, i) * s.inv_scale), 0}, m, v, h);
        const float w = split(updated(twice(t.w[i]), m.a, v.a, decay, s, h.eps)).x;
        t.w[i] = w;
        m_[i] = split(m.a).x;
        v_[i] = split(v.a).x;
        store_copy<CT>(t.copy, i, w);
    }
}

// ---------------------------------------------------------------- 8-bit states
struct Philox4 { uint32_t v[4]; };

constexpr int kRounds = 10;
struct PhiloxKeys { uint32_t k0[kRounds], k1[kRounds]; };        // of the rounds, from the seed

PhiloxKeys philox_keys(uint64_t seed) {
    PhiloxKeys k;
    for (uint32_t r = 0; r < kRounds; ++r) {
        k.k0[r] = (uint32_t)seed + r * 0x9E3779B9u;
        k.k1[r] = (uint32_t)(seed >> 32) + r * 0xBB67AE85u;
    }
    return k;
}

__device__ __forceinline__ Philox4 philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, const PhiloxKeys& k) {
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k.k0[r];
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k.k1[r];
        c1 = (uint32_t)p1;
        c3 = (uint32_t)p0;
    }
    return Philox4{{c0, c1, c2, c3}};
}

__device__ __forceinline__ Quad unpack_e4m3(uint32_t codes, float scale) {
    const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3);
    const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    return times({pair_of(a.x, a.y), pair_of(b.x, b.y)}, scale);
}

__device__ __forceinline__ uint32_t pack_nearest(const Quad& q, float up) {
    const Quad y = times(q, up);
    const auto lo = __nv_cvt_float2_to_fp8x2(split(y.a), __NV_SATFINITE, __NV_E4M3);
    const auto hi = __nv_cvt_float2_to_fp8x2(split(y.b), __NV_SATFINITE, __NV_E4M3);
    return (uint32_t)lo | (uint32_t)hi << 16;
}

// e4m3 codes of q * up, rounded up with probability r / 65536 of a step; 1 at least for what is above 0.  Times 2^-120
// the smallest normal e4m3 number becomes the smallest normal float: exponent and mantissa of the code are then the
// float's bits from 20 on, in the subnormal range too.  q * up is at most 448 (1 + 2^-22), two steps of a float above the
// largest code's number: random bits that end in four zeros do not carry it further.
__device__ __forceinline__ uint32_t pack_stochastic(const Quad& q, float up, const uint32_t (&r)[4]) {
    const float4 y = single(times(q, up)), f = single(times(times(q, up), 7.52316385e-37f));
    const float ys[4] = {y.x, y.y, y.z, y.w}, fs[4] = {f.x, f.y, f.z, f.w};
    uint32_t codes = 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        codes += max((__float_as_uint(fs[j]) + r[j] * 16u) >> 20, min(__float_as_uint(ys[j]), 1u)) << (8 * j);
    return codes;
}

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// largest of non-negative floats over the warp, a NaN (the positive one) above all: their bits order as integers
__device__ __forceinline__ float warp_top(float v) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu)); }

// an infinite largest value leaves nothing to scale by: NaN, as for a NaN
__device__ __forceinline__ float scale_of(float top) {
    return top < kSmallest ? 0.f : (top == INFINITY ? NAN : __fmul_rn(top, 1.0f / kE4m3Max));
}

// What an infinite v of a block with finite m is stored as: an infinity would take the block's other elements with it.
// Half of the range, so that 448 times its scale does not overflow again: from there it decays like any other.
constexpr float kHalfRange = 1.70141183e38f;    // 2^127
__device__ __forceinline__ uint64_t at_most_half(uint64_t v) {
    const float2 f = split(v);
    return pair_of(fminf(f.x, kHalfRange), fminf(f.y, kHalfRange));
}

// A lane's elements of a scale block, 4 lane .. 4 lane + 3, and the block's scales.
template <int GT>
struct BlockLoad {
    float4 w;
    uint4 g;                // floats, or 16-bit pairs in x and y
    uint32_t m, v;
    float ms, vs;

    // element by element, zeros behind the tensor's end
    __device__ __forceinline__ void load_some(const Tensor& t, int64_t block) {
        const int64_t i = block * kBlock + 4 * (threadIdx.x & 31);
        float* wk = reinterpret_cast<float*>(&w);
        uint32_t* gk = reinterpret_cast<uint32_t*>(&g);
        w = make_float4(0.f, 0.f, 0.f, 0.f);
        g = make_uint4(0u, 0u, 0u, 0u);
        m = v = 0u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i + j < t.n) {
                wk[j] = t.w[i + j];
                if constexpr (GT == TRB200_DTYPE_F32) gk[j] = static_cast<const uint32_t*>(t.g)[i + j];
                else gk[j >> 1] |= (uint32_t) static_cast<const uint16_t*>(t.g)[i + j] << (16 * (j & 1));
                m |= (uint32_t) static_cast<const uint8_t*>(t.m)[i + j] << (8 * j);
                v |= (uint32_t) static_cast<const uint8_t*>(t.v)[i + j] << (8 * j);
            }
        const bool there = block * kBlock < t.n;
        ms = there ? t.m_scale[block] : 0.f;
        vs = there ? t.v_scale[block] : 0.f;
    }

    __device__ __forceinline__ Quad grad() const {
        if constexpr (GT == TRB200_DTYPE_F32) {
            return {pair_of(__uint_as_float(g.x), __uint_as_float(g.y)), pair_of(__uint_as_float(g.z), __uint_as_float(g.w))};
        } else {
            const float2 a = unpack2_t<GT == TRB200_DTYPE_BF16>(g.x), b = unpack2_t<GT == TRB200_DTYPE_BF16>(g.y);
            return {pair_of(a.x, a.y), pair_of(b.x, b.y)};
        }
    }
};

// Whole units on their way: asynchronous copies into shared memory hold no registers, so kAhead units a warp are in
// flight.  A lane copies what it will read itself, but for the four scales of the unit (lanes 0 .. 3).
constexpr int kAhead = 3;

template <int BYTES>
__device__ __forceinline__ void copy_async(void* to, const void* from) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <int GT>
struct Stage {
    using G = std::conditional_t<GT == TRB200_DTYPE_F32, uint4, uint2>;
    float4 w[2][kThreads];
    G g[2][kThreads];
    uint32_t m[2][kThreads], v[2][kThreads];
    float scales[kWarps][4];

    __device__ __forceinline__ void fetch(const Tensor& t, int64_t unit) {
        const int tid = threadIdx.x, lane = tid & 31;
        const int64_t i = unit * kUnit + 4 * lane;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            copy_async<16>(&w[k][tid], t.w + i + k * kBlock);
            copy_async<sizeof(G)>(&g[k][tid], static_cast<const char*>(t.g) + (i + k * kBlock) * (sizeof(G) / 4));
            copy_async<4>(&m[k][tid], static_cast<const uint8_t*>(t.m) + i + k * kBlock);
            copy_async<4>(&v[k][tid], static_cast<const uint8_t*>(t.v) + i + k * kBlock);
        }
        if (lane < 4) copy_async<4>(&scales[tid >> 5][lane], (lane & 1 ? t.v_scale : t.m_scale) + 2 * unit + (lane >> 1));
    }

    __device__ __forceinline__ void read(BlockLoad<GT>& x, int k) const {
        const int tid = threadIdx.x;
        const float2 sc = *reinterpret_cast<const float2*>(&scales[tid >> 5][2 * k]);
        x.ms = sc.x;
        x.vs = sc.y;
        x.w = w[k][tid];
        x.m = m[k][tid];
        x.v = v[k][tid];
        if constexpr (GT == TRB200_DTYPE_F32) x.g = g[k][tid];
        else x.g = make_uint4(g[k][tid].x, g[k][tid].y, 0u, 0u);
    }
};

// One unit by one warp: a whole one from its stage, any other (stage = null) element by element.
template <int GT, int CT, bool WHOLE>
__device__ __forceinline__ void unit_8bit(const Tensor& t, int tensor, int64_t unit, const Stage<GT>* stage, const Hyper& h,
                                          const PhiloxKeys& keys, const Scalars& s, float decay) {
    const int lane = threadIdx.x & 31;
    const int64_t i = unit * kUnit + 4 * lane;                  // and kBlock behind it
    Quad m[2], v[2];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        BlockLoad<GT> x;
        if (WHOLE) stage->read(x, k);
        else x.load_some(t, 2 * unit + k);
        m[k] = unpack_e4m3(x.m, x.ms);
        v[k] = unpack_e4m3(x.v, x.vs);
        moments(times(x.grad(), s.inv_scale), m[k], v[k], h);
        const float4 w = single(updated(quad(x.w), m[k], v[k], decay, s, h.eps)), m4 = single(m[k]), v4 = single(v[k]);
        float mt = max_or_nan(max_or_nan(fabsf(m4.x), fabsf(m4.y)), max_or_nan(fabsf(m4.z), fabsf(m4.w)));
        float vt = max_or_nan(max_or_nan(v4.x, v4.y), max_or_nan(v4.z, v4.w));
        if (WHOLE) {
            *reinterpret_cast<float4*>(t.w + i + k * kBlock) = w;
            store_copy4<CT>(t.copy, i + k * kBlock, w);
        } else {
            const float ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + k * kBlock + j < t.n) {
                    t.w[i + k * kBlock + j] = ws[j];
                    store_copy<CT>(t.copy, i + k * kBlock + j, ws[j]);
                }
        }
        mt = warp_top(mt);
        vt = warp_top(vt);
        if (vt == INFINITY && mt < INFINITY) {                  // seldom: the square of a finite gradient overflowed
            v[k] = {at_most_half(v[k].a), at_most_half(v[k].b)};
            vt = kHalfRange;
        }
        if ((lane & 3) == 2 * k) top = mt;
        if ((lane & 3) == 2 * k + 1) top = vt;
    }
    // lanes 0 .. 3 (and every four behind them): the scale of m and of v, first and second block
    const float up = top < kSmallest ? 0.f : __fmul_rn(__frcp_rn(top), kE4m3Max);
    if (lane < 4 && (WHOLE || (2 * unit + (lane >> 1)) * kBlock < t.n))
        (lane & 1 ? t.v_scale : t.m_scale)[2 * unit + (lane >> 1)] = scale_of(top);
    // the two blocks share a counter: eight elements a lane, sixteen bits each
    const uint64_t group = (uint64_t)unit * 32 + lane;
    const Philox4 bits = philox4x32_10((uint32_t)group, (uint32_t)tensor, (uint32_t)s.step, (uint32_t)(group >> 32), keys);
    uint8_t* const m_ = static_cast<uint8_t*>(t.m);
    uint8_t* const v_ = static_cast<uint8_t*>(t.v);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float m_up = __shfl_sync(0xffffffffu, up, 2 * k), v_up = __shfl_sync(0xffffffffu, up, 2 * k + 1);
        const uint32_t mc = pack_nearest(m[k], m_up);
        uint32_t r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = k == 0 ? bits.v[j] & 0xffffu : bits.v[j] >> 16;
        const uint32_t vc = pack_stochastic(v[k], v_up, r);
        if (WHOLE) {
            *reinterpret_cast<uint32_t*>(m_ + i + k * kBlock) = mc;
            *reinterpret_cast<uint32_t*>(v_ + i + k * kBlock) = vc;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + k * kBlock + j < t.n) {
                    m_[i + k * kBlock + j] = (uint8_t)(mc >> (8 * j));
                    v_[i + k * kBlock + j] = (uint8_t)(vc >> (8 * j));
                }
        }
    }
}

// units [u0, u1) of a tensor by a thread block, a warp a unit
template <int GT, int CT>
__device__ __forceinline__ void range_8bit(const Tensor& t, int tensor, int64_t u0, int64_t u1, Stage<GT>* stages, const Hyper& h,
                                           const PhiloxKeys& keys, const Scalars& s, float decay) {
    const int64_t whole = t.vec ? min(u1, t.n / kUnit) : u0;    // units below it are whole
    int64_t u = u0 + (threadIdx.x >> 5), ahead = u;
    int slot = 0;
#pragma unroll
    for (int i = 0; i < kAhead; ++i, ahead += kWarps) {
        if (ahead < whole) stages[i].fetch(t, ahead);
        copies_commit();
    }
    for (; u < whole; u += kWarps, ahead += kWarps) {
        copies_wait<kAhead - 1>();
        __syncwarp();                                           // the scales are other lanes' copies
        unit_8bit<GT, CT, true>(t, tensor, u, stages + slot, h, keys, s, decay);
        __syncwarp();
        if (ahead < whole) stages[slot].fetch(t, ahead);
        copies_commit();
        slot = slot + 1 == kAhead ? 0 : slot + 1;
    }
    for (; u < u1; u += kWarps) unit_8bit<GT, CT, false>(t, tensor, u, nullptr, h, keys, s, decay);
}

// ---------------------------------------------------------------- the step
// The blocks of the grid take runs of h.run units in turn, whatever tensors they belong to.  The last block to end
// advances the step count: by then every block has read it.
template <int GT, int CT, bool E8>
__global__ void __launch_bounds__(kThreads, 3)
adamw_kernel(Header* head, const Tensor* tensors, const int32_t* units, int count, const __grid_constant__ Hyper h,
             const __grid_constant__ PhiloxKeys keys) {
    extern __shared__ __align__(16) unsigned char s_stages[];   // 8 bit: kAhead stages
    __shared__ Scalars s_scalars;
    ptx::wait_prior_grid();
    if (h.skip_flag && *h.skip_flag) return;
    if (threadIdx.x == 0) s_scalars = scalars_of(h);
    const int64_t total = units[count];
    int tensor = -1;
    int64_t from = 0, to = 0;                                    // units of the tensor
    Tensor t;
    auto go = [&](int64_t u) {                                   // to the last tensor with units[tensor] <= u
        if (u < to) return;
        int lo = tensor + 1, hi = count - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (units[mid] <= u) lo = mid;
            else hi = mid - 1;
        }
        tensor = lo;
        from = units[lo];
        to = units[lo + 1];
        t = tensors[lo];
    };
    int64_t u = (int64_t)blockIdx.x * h.run;
    if (u < total) go(u);                                        // meanwhile the scalars are computed
    __syncthreads();
    const Scalars s = s_scalars;
    for (; u < total; u += (int64_t)(gridDim.x - 1) * h.run) {
        for (const int64_t end = min(total, u + h.run); u < end;) {
            go(u);
            const int64_t stop = min(to, end);
            const float decay = 1.0f - s.lr * t.weight_decay;
            if constexpr (E8)
                range_8bit<GT, CT>(t, tensor, u - from, stop - from, reinterpret_cast<Stage<GT>*>(s_stages), h, keys, s, decay);
            else
                range_float<GT, CT>(t, (u - from) * kUnit, min(t.n, (stop - from) * kUnit), h, s, decay);
            u = stop;
        }
    }
    if (threadIdx.x == 0 && atomicAdd(&head->done, 1u) == gridDim.x - 1) {
        head->done = 0u;
        *h.step = s.step + 1;
    }
}

using Kernel = void (*)(Header*, const Tensor*, const int32_t*, int, const Hyper, const PhiloxKeys);

template <int GT, int CT>
Kernel kernel_of(bool e8) { return e8 ? adamw_kernel<GT, CT, true> : adamw_kernel<GT, CT, false>; }

template <int GT>
Kernel kernel_of(int copy, bool e8) {
    return copy == TRB200_DTYPE_F16 ? kernel_of<GT, TRB200_DTYPE_F16>(e8)
                                    : (copy == TRB200_DTYPE_BF16 ? kernel_of<GT, TRB200_DTYPE_BF16>(e8) : kernel_of<GT, -1>(e8));
}

Kernel kernel_of(int grad, int copy, bool e8) {
    return grad == TRB200_DTYPE_F32 ? kernel_of<TRB200_DTYPE_F32>(copy, e8)
                                    : (grad == TRB200_DTYPE_F16 ? kernel_of<TRB200_DTYPE_F16>(copy, e8) : kernel_of<TRB200_DTYPE_BF16>(copy, e8));
}

// The smallest eps.  A float v is off by 2^-149 / (1 - beta2) at most where it is subnormal, whatever the step (each step
// adds up to 2^-149, and the bias correction is at most 1 / (1 - beta2)), hence the root by 2^-74.5 / sqrt(1 - beta2):
// 2^-19.5 of the smallest eps.  A block of an 8-bit v below kSmallest is stored as zeros, which takes
// 2^-58 / sqrt(1 - beta2) from the root: 2^-5 of the smallest eps, half a step of the codes.  With a smaller eps the
// denominator of such an element could come out as next to nothing, and its change as orders of magnitude too large.
double least_eps(double beta2, bool e8) { return std::ldexp(1.0, e8 ? -53 : -55) / std::sqrt(1.0 - beta2); }
constexpr float kMostEps = 8.50705917e37f;  // 2^126: the reciprocal of anything larger would be flushed to zero

int64_t units_of(int64_t n) { return (n + kUnit - 1) / kUnit; }

// units of all tensors, or -1 for a bad description
int64_t count_units(const trb200_adamw_tensor* tensors, int32_t count) {
    int64_t total = 0;
    for (int32_t i = 0; i < count; ++i) {
        if (tensors[i].n < 0 || tensors[i].n > ((int64_t)1 << 42)) return -1;
        total += units_of(tensors[i].n);
    }
    return total <= 0x7fffffff ? total : -1;
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
    const int64_t units = count_units(in, count);
    TRB_REQUIRE(units >= 0, TRB200_ERR_INVALID_ARGUMENT, "adamw_plan: bad tensor size");
    TRB_REQUIRE(image_bytes >= image_size(count), TRB200_ERR_WORKSPACE, "adamw_plan: image too small");
    const bool e8 = state_bits == 8;
    char* base = static_cast<char*>(image);
    memset(base, 0, image_size(count));
    char* units_out = base + units_at(count);
    int32_t before = 0;
    std::vector<Range> ranges;
    ranges.reserve((size_t)count * 7);
    for (int32_t i = 0; i < count; ++i) {
        const trb200_adamw_tensor& t = in[i];
        before += (int32_t)units_of(t.n);
        memcpy(units_out + (size_t)(i + 1) * sizeof(int32_t), &before, sizeof(before));
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
    }
    TRB_REQUIRE(check_disjoint(ranges), TRB200_ERR_INVALID_ARGUMENT,
                "adamw_plan: a buffer that is written overlaps another one (is a tensor listed twice?)");
    *plan = trb200_adamw_plan{nullptr, count, (int32_t)units, grad_dtype, copy_dtype, state_bits};
    return TRB200_OK;
}

}  // namespace
}  // namespace trb

extern "C" size_t trb200_adamw_plan_bytes(const trb200_adamw_tensor* tensors, int32_t count) {
    if (count < 0 || (count > 0 && !tensors)) return 0;
    return trb::count_units(tensors, count) < 0 ? 0 : trb::image_size(count);
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
    TRB_REQUIRE(trb::aligned4(step, lr_dev, scaling, skip_flag), TRB200_ERR_INVALID_ARGUMENT,
                "adamw_step: step, lr_dev, scaling and skip_flag must be aligned to 4 bytes");
    TRB_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, TRB200_ERR_INVALID_ARGUMENT,
                "adamw_step: beta1 and beta2 must lie in [0, 1)");
    TRB_REQUIRE(std::isfinite(lr), TRB200_ERR_INVALID_ARGUMENT, "adamw_step: lr must be finite");
    TRB_REQUIRE(plan->count >= 0 && plan->units >= 0 &&
                    (trb::valid_dtype(plan->grad_dtype) || plan->grad_dtype == TRB200_DTYPE_F32) &&
                    (trb::valid_dtype(plan->copy_dtype) || plan->copy_dtype == TRB200_DTYPE_NONE) &&
                    (plan->state_bits == 32 || plan->state_bits == 8),
                TRB200_ERR_INVALID_ARGUMENT, "adamw_step: not a plan that trb200_adamw_plan_write wrote");
    const bool e8 = plan->state_bits == 8;
    TRB_REQUIRE(eps >= trb::least_eps(beta2, e8) && eps <= trb::kMostEps, TRB200_ERR_INVALID_ARGUMENT,
                "adamw_step: eps = %g, but with beta2 = %.9g and %d-bit states it must lie in [%.3g, 8.5e37]", (double)eps, beta2,
                (int)plan->state_bits, trb::least_eps(beta2, e8));
    TRB_REQUIRE((reinterpret_cast<uintptr_t>(plan->image) & 15u) == 0, TRB200_ERR_INVALID_ARGUMENT,
                "adamw_step: the plan's image must be 16-byte aligned");
    char* base = static_cast<char*>(plan->image);
    auto* head = reinterpret_cast<trb::Header*>(base);
    const auto* tensors = reinterpret_cast<const trb::Tensor*>(base + trb::tensors_at());
    const auto* units = reinterpret_cast<const int32_t*>(base + trb::units_at(plan->count));
    // Three blocks an SM (138 M elements, float states: 653 us against 690 with four, 710 with two; 8-bit ones 486 against
    // 510 with four).  Runs of 16 units (float) or 64 (8 bit), as even a number for the blocks as that allows; small plans
    // in runs that give every block something to do.  Float runs of 4 take 646 us for one tensor of 138 M elements (655), but
    // 127 us for 160 tensors of 160 000 (121.5); 8-bit ones of 8 take 107 us for 25.6 M elements (87), of 232, the same for
    // every block, 88.
    const int64_t resident = (int64_t)trb::sm_count() * 3, least = e8 ? trb::kWarps : 4, most = e8 ? 64 : 16;
    const int64_t rounds = (plan->units + resident * most - 1) / (resident * most);
    int64_t run = rounds ? (plan->units + resident * rounds - 1) / (resident * rounds) : least;
    run = (run + least - 1) / least * least;
    int grid = (int)std::min(resident, (plan->units + run - 1) / run);
    if (grid < 1) grid = 1;                                  // no elements: the step still counts
    const trb::Hyper h{lr, lr_dev, std::log(beta1), std::log(beta2), (float)beta1, (float)beta2, (float)(1.0 - beta1),
                       (float)(1.0 - beta2), eps, scaling, skip_flag, step, (int32_t)run, 1.0f};
    const size_t smem = !e8 ? 0 : trb::kAhead * (plan->grad_dtype == TRB200_DTYPE_F32 ? sizeof(trb::Stage<TRB200_DTYPE_F32>)
                                                                                     : sizeof(trb::Stage<TRB200_DTYPE_F16>));
    const trb::Kernel kernel = trb::kernel_of(plan->grad_dtype, plan->copy_dtype, e8);
    if (e8) {
        static bool ready[64][3][3] = {};
        int dev = 0;
        TRB_CUDA_TRY(cudaGetDevice(&dev));
        bool* done = dev < 64 ? &ready[dev][plan->grad_dtype][plan->copy_dtype + 1] : nullptr;
        if (!done || !*done) {
            TRB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
            TRB_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, 100));
            if (done) *done = true;
        }
    }
    TRB_CUDA_TRY(trb::launch_chained(kernel, grid, trb::kThreads, 1, smem, trb::as_stream(stream), head, tensors, units, plan->count, h,
                                     trb::philox_keys(seed)));
    TRB_LAUNCH_CHECK("adamw");
    return TRB200_OK;
}
