// Losses that start from the log-probabilities of chosen classes: the log-probabilities themselves, the clipped policy
// loss with a KL term and the paired preference loss, the last two with their gradient with respect to the logits.
// Rows of half, bfloat16 or float logits, float arithmetic.
//
//   m = max_c z_c     s = sum_c exp(z_c - m)     logp = (z_y - m) - log s     lse = m + log s
//
//   policy:      r = exp(logp - old)     kl = exp(ref - logp) - (ref - logp) - 1
//                loss_i = w_i * (-min(r A, clip(r, 1 - lo, 1 + hi) A) + k * kl)
//                d loss_i / d logp = w_i * (-[r A <= clip(r) A] r A + k * (1 - exp(ref - logp)))
//   preference:  S_q = sum of logp over the rows of sequence q     x_p = beta * ((S - ref)_2p - (S - ref)_2p+1)
//                loss_p = (-(1 - e) log sigmoid(x) - e log sigmoid(-x)) / pairs
//                d loss_p / d logp = +-beta * (e sigmoid(x) - (1 - e) sigmoid(-x)) / pairs
//   both:        d logits_c = scaling * (d loss / d logp) * ([c == y] - exp(z_c - m) / s)
//
// A row whose label lies outside [0, classes), whose weight is 0, that belongs to no sequence, or whose logits are all
// minus infinity does not count: it adds nothing to the loss, its gradient is zero and (but for the last kind) its
// logits are not read.
//
// All of it is bound by HBM: per logit one read, and one write where there is a gradient.
#include "chained.cuh"
#include "common.cuh"
#include "packed.cuh"
#include "sm100_ptx.cuh"

#include <cmath>
#include <type_traits>

namespace trb {
namespace {

// log2(e) in two floats: with the first alone every exponent is 1.3e-8 of itself short, and log s, whose terms are all
// off the same way, by 1.3e-7 at 131072 classes (measured; 3e-8 with both), which a sequence of 1000 rows adds up
constexpr float kLog2eHi = 1.44269502f, kLog2eLo = 1.92596303e-8f;

// ---------------------------------------------------------------- storage types (TRB200_DTYPE_*)
template <int DT>
struct Logit {
    using T = uint16_t;
    static constexpr int kVec = 8;              // elements of a 16-byte vector
    static constexpr bool kBf16 = DT == TRB200_DTYPE_BF16;
    static __device__ __forceinline__ float load(const T* p) { return load16_t<kBf16>(p); }
    static __device__ __forceinline__ void store(T* p, float v) { *p = round16_t<kBf16>(v); }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[kVec]) { unpack8_t<kBf16>(v, f); }
    static __device__ __forceinline__ uint4 pack(const float (&f)[kVec]) {
        return make_uint4(pack2_t<kBf16>(f[0], f[1]), pack2_t<kBf16>(f[2], f[3]), pack2_t<kBf16>(f[4], f[5]),
                          pack2_t<kBf16>(f[6], f[7]));
    }
};

template <>
struct Logit<TRB200_DTYPE_F32> {
    using T = float;
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float load(const T* p) { return *p; }
    static __device__ __forceinline__ void store(T* p, float v) { *p = v; }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&f)[kVec]) {
        f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&f)[kVec]) {
        return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    }
};

// A row as whole 16-byte vectors between a few single elements at its ends (rows start anywhere: an odd class count or
// an odd stride moves every row's alignment).
struct RowSplit {
    int head, nvec, tail;       // elements, vectors, elements
    template <typename T>
    __device__ __forceinline__ RowSplit(const T* row, int classes) {
        constexpr int kVec = 16 / (int)sizeof(T);
        const int skew = (int)((reinterpret_cast<uintptr_t>(row) & 15u) / sizeof(T));
        head = min(classes, skew ? kVec - skew : 0);
        nvec = (classes - head) / kVec;
        tail = classes - head - nvec * kVec;
    }
    // single element `tid`, or -1 (there are head + tail, fewer than 2 * 16 / sizeof(T))
    __device__ __forceinline__ int single(int tid, int classes) const {
        if (tid < head) return tid;
        const int t = tid - head;
        return t < tail ? classes - tail + t : -1;
    }
};

// 16 bytes to an address that is aligned for its element type only
__device__ __forceinline__ void store_any(void* p, const uint4& v, int elem) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    if ((a & 15u) == 0) {
        *static_cast<uint4*>(p) = v;
    } else if ((a & 7u) == 0) {
        static_cast<uint2*>(p)[0] = make_uint2(v.x, v.y);
        static_cast<uint2*>(p)[1] = make_uint2(v.z, v.w);
    } else if (elem == 4 || (a & 3u) == 0) {
        uint32_t* q = static_cast<uint32_t*>(p);
        q[0] = v.x; q[1] = v.y; q[2] = v.z; q[3] = v.w;
    } else {
        uint16_t* q = static_cast<uint16_t*>(p);
        q[0] = (uint16_t)v.x; q[1] = (uint16_t)(v.x >> 16); q[2] = (uint16_t)v.y; q[3] = (uint16_t)(v.y >> 16);
        q[4] = (uint16_t)v.z; q[5] = (uint16_t)(v.z >> 16); q[6] = (uint16_t)v.w; q[7] = (uint16_t)(v.w >> 16);
    }
}

// ---------------------------------------------------------------- maximum and sum of exponentials
// exp(z - m) is 2^(d hi + d lo) with d = z - m: the difference first, so that the largest element gives exactly 1, a row
// with one class exactly logp = 0, and the type's lowest value as a mask no overflow.  The exponential is the hardware's,
// 2^-22 off at most: its unit is busy for up to three quarters of the time as it is.
struct MaxSum { float m, s; };       // s: sum of exp(z - m); m = -inf goes with s = 0; a NaN ends up in s

__device__ __forceinline__ float exp_of(float d) { return fast_exp2(fmaf(d, kLog2eLo, d * kLog2eHi)); }

// what differences are taken to: 0 stands in for -inf, so that no difference of infinities is formed
__device__ __forceinline__ float pivot(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b) {
    const float m = fmaxf(a.m, b.m), p = pivot(m);
    return {m, a.s * exp_of(a.m - p) + b.s * exp_of(b.m - p)};
}

template <int N>
__device__ __forceinline__ void take(MaxSum& a, const float (&f)[N]) {
    float m = f[0];
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmaxf(m, f[j]);
    m = fmaxf(m, a.m);
    const float p = pivot(m);
    a = {m, a.s * exp_of(a.m - p)};
#pragma unroll
    for (int j = 0; j < N; ++j) a.s += exp_of(f[j] - p);
}

// the same MaxSum in every thread of a block of T threads; s_red holds T / 32 entries
template <int T>
__device__ __forceinline__ MaxSum block_merge(MaxSum a, MaxSum* s_red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        a = merge(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
    __syncthreads();
    if (lane == 0) s_red[warp] = a;
    __syncthreads();
    a = s_red[0];
#pragma unroll 1
    for (int i = 1; i < T / 32; ++i) a = merge(a, s_red[i]);
    return a;
}

// ---- rows whose maximum lies within +-2^100; the others (infinities, all NaN, numbers of a broken model) leave for the
// code above
constexpr float kFloor = -1.26765060e30f;   // -2^100: stands in for -inf as a thread's maximum

__device__ __forceinline__ bool plain(float m) { return fabsf(m) < -kFloor; }

// Rows whose 16-bit gradient may be taken as slope_vec() does; row_gradient() takes the others.
constexpr float kNear = 256.f;
template <int DT>
__device__ __forceinline__ bool near(float m) { return plain(m) && (DT == TRB200_DTYPE_F32 || fabsf(m) <= kNear); }

__device__ __forceinline__ uint64_t exp2_pair(uint64_t x) {
    const float2 f = split(x);
    return pair_of(fast_exp2(f.x), fast_exp2(f.y));
}
// exp_of() of z - m; `minus` = -m twice
__device__ __forceinline__ uint64_t exp_pair(uint64_t z, uint64_t minus) {
    const uint64_t d = add2(z, minus);
    return exp2_pair(fma2(d, twice(kLog2eLo), mul2(d, twice(kLog2eHi))));
}

// MaxSum over the low N lanes of a warp (N a power of two); the maximum first, so that a lane rescales its sum once
template <int N>
__device__ __forceinline__ MaxSum warp_merge(MaxSum a) {
    float m = a.m;
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float s = a.s * exp_of(a.m - m);
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return {m, s};
}

// Vectors of a row as pairs of floats.
template <int DT>
struct Vec {
    using L = Logit<DT>;
    static constexpr int kPairs = L::kVec / 2;
    // -inf in every element
    static constexpr uint32_t kLow = DT == TRB200_DTYPE_F16 ? 0xfc00fc00u : (DT == TRB200_DTYPE_BF16 ? 0xff80ff80u : 0xff800000u);

    static __device__ __forceinline__ uint64_t pair(const uint4& v, int i) {
        if constexpr (DT == TRB200_DTYPE_F32) {
            return i == 0 ? pair_of(__uint_as_float(v.x), __uint_as_float(v.y)) : pair_of(__uint_as_float(v.z), __uint_as_float(v.w));
        } else {
            const float2 f = unpack2_t<L::kBf16>(i == 0 ? v.x : (i == 1 ? v.y : (i == 2 ? v.z : v.w)));
            return pair_of(f.x, f.y);
        }
    }

    // largest element of N vectors, NaN aside; 16-bit types two at a time
    template <int N>
    static __device__ __forceinline__ float top(const uint4 (&v)[N]) {
        if constexpr (DT == TRB200_DTYPE_F32) {
            float m = __uint_as_float(v[0].x);
#pragma unroll
            for (int i = 0; i < N; ++i)
                m = fmaxf(fmaxf(m, fmaxf(__uint_as_float(v[i].x), __uint_as_float(v[i].y))),
                          fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w)));
            return m;
        } else {
            using H = std::conditional_t<L::kBf16, __nv_bfloat162, __half2>;
            const H* h = reinterpret_cast<const H*>(&v);
            H m[4] = {h[0], h[1], h[2], h[3]};          // four chains
#pragma unroll
            for (int i = 4; i < 4 * N; ++i) m[i & 3] = __hmax2(m[i & 3], h[i]);
            m[0] = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
            return fmaxf(__low2float(m[0]), __high2float(m[0]));
        }
    }
};

// Maximum and sum over vectors that arrive in groups of N.
struct Running {
    float m = kFloor;
    uint64_t s0 = 0, s1 = 0;            // two sums of pairs, to shorten the chains of additions

    __device__ __forceinline__ uint64_t raise(float top) {
        const uint64_t sc = twice(exp_of(m - top));
        m = top;
        s0 = mul2(s0, sc);
        s1 = mul2(s1, sc);
        return twice(-top);
    }

    template <int DT, int N>
    __device__ __forceinline__ void take(const uint4 (&v)[N]) {
        using V = Vec<DT>;
        const uint64_t minus = raise(fmaxf(m, V::top(v)));
#pragma unroll
        for (int k = 0; k < N; ++k) {
#pragma unroll
            for (int i = 0; i < V::kPairs; i += 2) {
                s0 = add2(s0, exp_pair(V::pair(v[k], i), minus));
                s1 = add2(s1, exp_pair(V::pair(v[k], i + 1), minus));
            }
        }
    }

    // one element, -inf for none
    __device__ __forceinline__ void take_one(float z) {
        raise(fmaxf(m, z));
        s0 = add2(s0, pair_of(exp_of(z - m), 0.f));
    }

    __device__ __forceinline__ MaxSum total() const {
        const float2 s = split(add2(s0, s1));
        return {m, s.x + s.y};
    }
};

// What the gradient of a row needs: g_c = coef ([c == y] - exp(z_c - m) / s).  A 16-bit result is one multiply-add and
// one exponential, |coef| p_c = 2^(z_c hi + up) with up = log2(|coef| / s) - m hi (within kNear its rounding is 2^-16
// of the power, next to the 2^-12 or 2^-9 of the result's), and the sign is the conversion's.
struct Slope {
    float m, s, coef, up;
    __device__ __forceinline__ float at(float z, bool label) const {        // one element in full precision
        return fmaf(exp_of(z - m), -coef / s, label ? coef : 0.f);
    }
};

__device__ __forceinline__ Slope slope_of(MaxSum a, float coef) {
    return {a.m, a.s, coef, log2f(fabsf(coef) / a.s) - a.m * kLog2eHi};
}

template <int DT, bool NEG>
__device__ __forceinline__ uint4 slope_vec(const uint4& v, const Slope& g) {
    using V = Vec<DT>;
    if constexpr (DT == TRB200_DTYPE_F32) {
        const uint64_t minus = twice(-g.m), fall = twice(-g.coef / g.s);
        const float2 x = split(mul2(exp_pair(V::pair(v, 0), minus), fall)), y = split(mul2(exp_pair(V::pair(v, 1), minus), fall));
        return make_uint4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
    } else {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = split(exp2_pair(fma2(V::pair(v, i), twice(kLog2eHi), twice(g.up))));
            o[i] = NEG ? pack2_t<V::L::kBf16>(-x.x, -x.y) : pack2_t<V::L::kBf16>(x.x, x.y);
        }
        return make_uint4(o[0], o[1], o[2], o[3]);
    }
}

// ---------------------------------------------------------------- what a row's loss is
struct PolicyArgs {
    const float* old_logp;
    const float* ref_logp;      // may be null: no KL term
    const float* advantages;
    const float* weights;       // may be null: 1 / rows
    const float* scaling;
    float low, high, kl_coef;   // clipping bounds of the ratio
    float even_weight;          // 1 / rows
};

struct PolicyIn { float old_logp, ref_logp, advantage, weight, scaling; };

__device__ __forceinline__ PolicyIn policy_in(const PolicyArgs& a, int row) {
    return {a.old_logp[row], a.ref_logp ? a.ref_logp[row] : 0.f, a.advantages[row],
            a.weights ? a.weights[row] : a.even_weight, a.scaling[0]};
}

// exp(x) - 1 - x with more = exp(x) - 1.  Next to 0 by its series x^2 (1/2 + x/6 + x^2/24 + ...), whose first term left out
// is 2e-9 of it: the difference of the two would keep 2^-24 |x| of a number of size x^2 / 2 (6e-3 of it at |x| = 1e-5).
__device__ __forceinline__ float exp_excess(float x, float more) {
    if (fabsf(x) >= 0.5f) return more == INFINITY ? INFINITY : more - x;        // no inf - inf for a class without chance
    float p = 2.75573192e-6f;                                                   // 1 / 9!
    p = fmaf(p, x, 2.48015873e-5f);
    p = fmaf(p, x, 1.98412698e-4f);
    p = fmaf(p, x, 1.38888889e-3f);
    p = fmaf(p, x, 8.33333333e-3f);
    p = fmaf(p, x, 4.16666667e-2f);
    p = fmaf(p, x, 0.166666667f);
    p = fmaf(p, x, 0.5f);
    return x * x * p;
}

// a - b and what its rounding cut off
__device__ __forceinline__ float minus_with_rest(float a, float b, float& rest) {
    const float d = a - b, back = d - a;
    rest = (a - (d - back)) - (b + back);
    return d;
}

// log-probability of the label with logit zy minus old, which is near it, to 2^-24: ((zy - m) - old) - log s with what the two
// differences cut off, and with s = 2^e f, f in [0.75, 1.5): log s = e ln 2 + log f.  ln 2 is in two floats, the first short
// enough for e ln 2 to be exact.
__device__ __forceinline__ float moved_since(float old, float zy, MaxSum a) {
    constexpr float kLn2Hi = 0.693145751953125f, kLn2Lo = 1.42860682e-6f;
    const int e = (__float_as_int(a.s) - 0x3f400000) >> 23;
    const float log_f = logf(a.s * __int_as_float((127 - e) << 23)), p = (float)e;
    float r1, r2;
    const float d = minus_with_rest(minus_with_rest(zy, a.m, r1), old, r2);
    return (fmaf(-p, kLn2Hi, d) - log_f) + (r1 + fmaf(-p, kLn2Lo, r2));
}

// Weighted loss of a row and scaling * its derivative with respect to logp.  The stored logp is off by half a step of a float
// (5e-7 for 8 to 16), which the ratio would take over.  Where old_logp is that very float the policy has not moved, and the
// ratio is exactly 1.
__device__ __forceinline__ void policy_row(const PolicyArgs& a, const PolicyIn& in, float logp, float zy, MaxSum stats, float& loss,
                                           float& coef) {
    const float adv = in.advantage;
    float moved = logp - in.old_logp;
    if (moved != 0.f && fabsf(moved) < INFINITY) moved = moved_since(in.old_logp, zy, stats);
    const float ratio = expf(moved);
    const float kept = ratio * adv;
    const float cut = fminf(fmaxf(ratio, a.low), a.high) * adv;
    float l, g;
    if (kept <= cut) { l = -kept; g = -kept; }
    else { l = kept > cut ? -cut : NAN; g = kept > cut ? 0.f : NAN; }     // unordered: a NaN stays one
    if (a.ref_logp) {
        const float gap = in.ref_logp - logp;                   // of the floats: 0 where the reference's is the same one
        const float more = expm1f(gap);                         // no cancellation next to gap = 0
        l += a.kl_coef * exp_excess(gap, more);
        g -= a.kl_coef * more;
    }
    loss = l * in.weight;
    coef = g * in.weight * in.scaling;
}

// ---------------------------------------------------------------- what a row kernel is for
template <int DT>
struct Rows {
    using T = typename Logit<DT>::T;
    const T* z;
    int64_t z_stride;
    T* d;                           // gradient
    int64_t d_stride;
    const int32_t* labels;
    int rows, classes;
    __device__ __forceinline__ const T* logits(int row) const { return z + (int64_t)row * z_stride; }
    __device__ __forceinline__ T* gradient(int row) const { return d + (int64_t)row * d_stride; }
};

// log-probability of the label with logit zy, never above 0
__device__ __forceinline__ float label_logp(float zy, MaxSum a) { return (zy - a.m) - logf(a.s); }

// Each purpose says which rows count, takes a counting row's MaxSum to its outputs and, for a gradient, to coef.
struct LogpRows {
    static constexpr bool kGradient = false;
    float* logp;
    float* lse;
    struct In {};
    __device__ __forceinline__ bool counts(int row) const { return true; }
    __device__ __forceinline__ In in(int row) const { return {}; }
    __device__ __forceinline__ void skip(int row) const {
        logp[row] = 0.f;
        if (lse) lse[row] = 0.f;
    }
    __device__ __forceinline__ float finish(int row, const In&, float zy, MaxSum a, bool write) const {
        if (write) {
            const bool none = a.s == 0.f;                           // every logit is -inf
            logp[row] = none ? -INFINITY : label_logp(zy, a);
            if (lse) lse[row] = none ? -INFINITY : a.m + logf(a.s);
        }
        return 0.f;
    }
};

struct PolicyRows {
    static constexpr bool kGradient = true;
    PolicyArgs p;
    float* logp;
    float* loss_partial;
    using In = PolicyIn;
    __device__ __forceinline__ bool counts(int row) const { return !p.weights || p.weights[row] != 0.f; }
    __device__ __forceinline__ In in(int row) const { return policy_in(p, row); }
    __device__ __forceinline__ void skip(int row) const { logp[row] = loss_partial[row] = 0.f; }
    __device__ __forceinline__ float finish(int row, const In& x, float zy, MaxSum a, bool write) const {
        float lp = 0.f, loss = 0.f, coef = 0.f;
        if (a.s != 0.f) {
            lp = label_logp(zy, a);
            policy_row(p, x, lp, zy, a, loss, coef);
        }
        if (write) {
            logp[row] = lp;
            loss_partial[row] = loss;
        }
        return coef;
    }
};

// first pass of the preference loss: statistics of the rows that count; coef starts at 0 for every row
struct PairRows {
    static constexpr bool kGradient = false;
    const int32_t* seq_starts;
    int seqs;
    float* logp;
    double* logp64;                 // what the sequence sums take: the rounding of logp, 3e-7 a row, would add up
    float* row_max;
    float* row_sum;                 // 0: the row does not count
    float* coef;
    struct In {};
    __device__ __forceinline__ bool counts(int row) const { return row >= seq_starts[0] && row < seq_starts[seqs]; }
    __device__ __forceinline__ In in(int row) const { return {}; }
    __device__ __forceinline__ void skip(int row) const {
        logp[row] = row_max[row] = row_sum[row] = coef[row] = 0.f;
        logp64[row] = 0.0;
    }
    __device__ __forceinline__ float finish(int row, const In&, float zy, MaxSum a, bool write) const {
        if (write) {
            logp[row] = a.s != 0.f ? label_logp(zy, a) : 0.f;
            logp64[row] = a.s != 0.f ? ((double)zy - (double)a.m) - log((double)a.s) : 0.0;
            row_max[row] = a.m;
            row_sum[row] = a.s;
            coef[row] = 0.f;
        }
        return 0.f;
    }
};

// ---------------------------------------------------------------- rows that leave the plain path
// 16-bit rows with a maximum beyond 256 read it once more for their gradient, with the difference z - m first: the policy
// loss of 65536 x 1000 halfs takes 111 us where it takes 70 us up to 256, of 4096 x 32000 bfloat16 113 us in place of 94.
//
// maximum and sum of the row over the T threads of the block
template <int DT, int T>
__device__ __forceinline__ MaxSum row_stats(const typename Logit<DT>::T* z, int classes, MaxSum* s_red) {
    using L = Logit<DT>;
    const RowSplit sp(z, classes);
    MaxSum a{-INFINITY, 0.f};
    const int e = sp.single(threadIdx.x, classes);
    if (e >= 0) {
        const float f[1] = {L::load(z + e)};
        take(a, f);
    }
    const uint4* zv = reinterpret_cast<const uint4*>(z + sp.head);
#pragma unroll 1
    for (int v = threadIdx.x; v < sp.nvec; v += T) {
        float f[L::kVec];
        L::unpack(zv[v], f);
        take(a, f);
    }
    return block_merge<T>(a, s_red);
}

// zeros for the row whose gradient is d, by `parts` groups of T threads
template <int DT, int T>
__device__ __forceinline__ void zero_row(typename Logit<DT>::T* d, int classes, int tid, int part, int parts) {
    const RowSplit sp(d, classes);
    if (part == 0)
        for (int i = tid; i < sp.head + sp.tail; i += T) Logit<DT>::store(d + sp.single(i, classes), 0.f);
    uint4* dv = reinterpret_cast<uint4*>(d + sp.head);
#pragma unroll 4
    for (int v = part * T + tid; v < sp.nvec; v += parts * T) __stcs(dv + v, make_uint4(0u, 0u, 0u, 0u));
}

// d = coef * ([c == y] - exp(z - m) / s) by `parts` groups of T threads
template <int DT, int T>
__device__ __forceinline__ void row_gradient(const typename Logit<DT>::T* z, typename Logit<DT>::T* d, int classes,
                                             int y, MaxSum a, float coef, int tid, int part, int parts) {
    using L = Logit<DT>;
    const RowSplit sp(z, classes);
    const float p = pivot(a.m), fall = -coef / a.s;
    for (int i = part == 0 ? tid : sp.head + sp.tail; i < sp.head + sp.tail; i += T) {
        const int e = sp.single(i, classes);
        L::store(d + e, fmaf(exp_of(L::load(z + e) - p), fall, e == y ? coef : 0.f));
    }
    const uint4* zv = reinterpret_cast<const uint4*>(z + sp.head);
#pragma unroll 1
    for (int v = part * T + tid; v < sp.nvec; v += parts * T) {
        float f[L::kVec];
        L::unpack(zv[v], f);
        const int c0 = sp.head + v * L::kVec, jy = y - c0;
#pragma unroll
        for (int j = 0; j < L::kVec; ++j) f[j] = fmaf(exp_of(f[j] - p), fall, j == jy ? coef : 0.f);
        store_any(d + c0, L::pack(f), (int)sizeof(typename L::T));
    }
}

// ---------------------------------------------------------------- short rows: in registers
// G lanes of a warp share a row, K vectors each; what a row costs beside its elements (setting up, merging, the loss
// itself) is paid once for the 32 / G rows of the warp: log-probabilities of 65536 rows of 64 bfloat16 classes take 6.4 us
// with 8 lanes a row, 22.0 us with 32.  65536 x 1000 take 27.3 us (0.74 of the copy bandwidth), the policy loss 70 us.
// Up to 2048 classes: 16383 x 1100 floats take 15.1 us (policy 39.6) here and 21.2 us (40.5) streamed.  Beyond, 16 bits,
// 16384 x 4096: 23.9 us against 28.0, but the policy loss 59 us against 52.4, and all operators have to take the same
// kernel for a length (see launch_rows).
constexpr int kShortThreads = 128;

// The words are to be unpacked again by the next pass: kept as floats they would take twice the registers.
template <int K>
__device__ __forceinline__ void forget(uint4 (&raw)[K]) {
#pragma unroll
    for (int k = 0; k < K; ++k) asm volatile("" : "+r"(raw[k].x), "+r"(raw[k].y), "+r"(raw[k].z), "+r"(raw[k].w));
}

// MaxSum of the plain path over the G lanes of a row, in all of them
template <int G>
__device__ __forceinline__ MaxSum group_merge(MaxSum a) {
    float m = a.m;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    float s = a.s * exp_of(a.m - m);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return {m, s};
}

// the same for any MaxSum, by the lanes of one row alone
template <int G>
__device__ __forceinline__ MaxSum lanes_merge(MaxSum a) {
    const unsigned lanes = (G == 32 ? 0xffffffffu : (1u << (G & 31)) - 1u) << (threadIdx.x & 31 & ~(G - 1));
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1)
        a = merge(a, {__shfl_xor_sync(lanes, a.m, o), __shfl_xor_sync(lanes, a.s, o)});
    // merge(a, b) and merge(b, a) may differ in the last bit: all take the first lane's
    return {__shfl_sync(lanes, a.m, 0, G), __shfl_sync(lanes, a.s, 0, G)};
}

template <int DT, int G, int K, class P>
__global__ void __launch_bounds__(kShortThreads, K >= 16 ? 4 : (K >= 8 ? 5 : 8))
rows_short(Rows<DT> r, P p) {
    using L = Logit<DT>;
    const int lane = threadIdx.x & (G - 1);
    const int row = blockIdx.x * (kShortThreads / G) + threadIdx.x / G;
    ptx::wait_prior_grid();
    ptx::let_next_grid_start();
    const bool there = row < r.rows;                            // lanes without a row, or with one that does not count,
    const int y = there ? r.labels[row] : -1;                   // go along: the shuffles are the whole warp's
    const bool counts = (unsigned)y < (unsigned)r.classes && p.counts(row);
    const auto* z = r.logits(there ? row : 0);
    const RowSplit sp(z, r.classes);
    const uint4* zv = reinterpret_cast<const uint4*>(z + sp.head);
    uint4 raw[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        raw[k] = make_uint4(Vec<DT>::kLow, Vec<DT>::kLow, Vec<DT>::kLow, Vec<DT>::kLow);
        if (counts && lane + G * k < sp.nvec) raw[k] = __ldcs(zv + lane + G * k);
    }
    // single elements: fewer than 16 (half) or 8 (float) a row
    constexpr int kEdges = (2 * L::kVec + G - 1) / G;
    int edge_at[kEdges];
    float edge[kEdges];
#pragma unroll
    for (int i = 0; i < kEdges; ++i) {
        edge_at[i] = counts ? sp.single(lane + G * i, r.classes) : -1;
        edge[i] = edge_at[i] >= 0 ? L::load(z + edge_at[i]) : -INFINITY;
    }
    typename P::In in{};
    float zy = 0.f;
    if (counts) {
        in = p.in(row);
        zy = L::load(z + y);
    }
    Running run;
    run.template take<DT>(raw);
#pragma unroll
    for (int i = 0; i < kEdges; ++i) run.take_one(edge[i]);
    MaxSum a = group_merge<G>(run.total());
    if (counts && !plain(a.m)) {                                // seldom; the same in all lanes of the row
        a = {-INFINITY, 0.f};
        for (int c = lane; c < r.classes; c += G) {
            const float f[1] = {L::load(z + c)};
            take(a, f);
        }
        a = lanes_merge<G>(a);
    }
    if (!there) return;
    if (!counts) {
        if (lane == 0) p.skip(row);
        if constexpr (P::kGradient) zero_row<DT, G>(r.gradient(row), r.classes, lane, 0, 1);
        return;
    }
    const float coef = p.finish(row, in, zy, a, lane == 0);     // the same in all lanes of the row
    if constexpr (P::kGradient) {
        auto* d = r.gradient(row);
        if (coef == 0.f) {
            zero_row<DT, G>(d, r.classes, lane, 0, 1);
        } else if (near<DT>(a.m)) {
            const Slope g = slope_of(a, coef);
            auto* dv = d + sp.head;
            const bool wide = (reinterpret_cast<uintptr_t>(dv) & 15u) == 0, neg = coef > 0.f;
            forget(raw);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int v = lane + G * k;
                if (v >= sp.nvec) continue;
                const uint4 out = neg ? slope_vec<DT, true>(raw[k], g) : slope_vec<DT, false>(raw[k], g);
                if (wide) __stcs(reinterpret_cast<uint4*>(dv) + v, out);
                else store_any(dv + v * L::kVec, out, (int)sizeof(typename L::T));
            }
#pragma unroll
            for (int i = 0; i < kEdges; ++i)
                if (edge_at[i] >= 0) L::store(d + edge_at[i], g.at(edge[i], edge_at[i] == y));
            // the label's element again, by the lane that stored its vector
            const int vy = (y - sp.head) / L::kVec;
            if (y >= sp.head && vy < sp.nvec && (vy & (G - 1)) == lane) L::store(d + y, g.at(zy, true));
        } else {
            row_gradient<DT, G>(z, d, r.classes, y, a, coef, lane, 0, 1);
        }
    }
}

// ---------------------------------------------------------------- longer rows: streamed
// A row is cut into parts by its length alone, up to kMaxParts of them; a cluster of C blocks shares it, `per_block`
// parts each.  Every part has its own maximum and sum, and they are merged in one order whatever C is: a row's
// log-probability is the same number in every batch and in every operator, as long as the row's address modulo 16 bytes
// is the same.  Vectors start at aligned addresses, so that a row that moves to another alignment (odd class counts or
// strides) is summed in another order: of 200 rows of 1001, 2047 or 50021 classes 4 to 10 then came out different, by
// 2e-6 at most.
//
// The gradient reads the row again.  The blocks that are resident at once (six of 256 threads an SM) hold 64 KB of logits
// each, 57 MB in all, so that the second read comes from L2 (4096 x 32000 bfloat16: 269 MB are read from HBM, 262 MB of
// logits).  Shorter rows get smaller blocks: what a row costs beside its elements is paid by every warp of its block
// (log-probabilities, 16384 rows: 2056 classes 25.1 us with 64 threads, 56.9 us with 256; 4096 classes 28.0 and 60.1 us).
//
// Log-probabilities of 6000 x 50021: 88 us, 0.83 of the copy bandwidth.  Policy loss: 4096 x 32000, a quarter of the rows
// masked, 85 us, 0.83; 8192 x 131072, a tenth masked, 750 us, 0.83.  At 4096 x 32000 with every row counting, 11.7
// instructions a logit take 51 % of the issue slots and the exponentials 72 % of their unit; warps wait for loads and for
// the block's barriers.  In a loop the GPU runs into its power limit at 8192 x 131072 (1000 W, 1.6 GHz).
constexpr int kStreamThreads = 1536;         // of an SM, in blocks of 64, 128 or 256
constexpr int kMaxParts = 8;
constexpr int kPartVecs = 4096;             // 64 KB, unless the row has more than kMaxParts of them

template <int DT, int T, class P>
__global__ void __launch_bounds__(T, kStreamThreads / T)
rows_streamed(Rows<DT> r, P p, int C, int parts, int per_block, int part_vecs) {
    using L = Logit<DT>;
    constexpr int kStreamWarps = T / 32;
    __shared__ MaxSum s_red[kMaxParts][kStreamWarps], s_parts[kMaxParts];
    __shared__ Slope s_slope;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row = blockIdx.x / C, rank = blockIdx.x - row * C;
    ptx::wait_prior_grid();
    ptx::let_next_grid_start();
    const int y = r.labels[row];
    const auto* z = r.logits(row);
    if ((unsigned)y >= (unsigned)r.classes || !p.counts(row)) {     // the same in all blocks of the row
        if (tid == 0 && rank == 0) p.skip(row);
        if constexpr (P::kGradient) zero_row<DT, T>(r.gradient(row), r.classes, tid, rank, C);
        return;
    }
    if (C > 1) ptx::cluster_arrive();
    const RowSplit sp(z, r.classes);
    const int part0 = rank * per_block, own = max(0, min(per_block, parts - part0));
    // the last part takes a vector more or less as the row's alignment has it
    auto part_end = [&](int q) { return q == parts - 1 ? sp.nvec : min(sp.nvec, (q + 1) * part_vecs); };
    const uint4* zv = reinterpret_cast<const uint4*>(z + sp.head);
    const int edge_at = rank == 0 ? sp.single(tid, r.classes) : -1;
    for (int q = 0; q < own; ++q) {
        Running run;
        const int end = part_end(part0 + q);
        int v = (part0 + q) * part_vecs + tid;
        for (; v + 3 * T < end; v += 4 * T) {
            const uint4 x[4] = {zv[v], zv[v + T], zv[v + 2 * T], zv[v + 3 * T]};
            run.template take<DT>(x);
        }
        if (v < end) {
            uint4 x[3];
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                x[k] = make_uint4(Vec<DT>::kLow, Vec<DT>::kLow, Vec<DT>::kLow, Vec<DT>::kLow);
                if (v + k * T < end) x[k] = zv[v + k * T];
            }
            run.template take<DT>(x);
        }
        if (part0 + q == 0 && edge_at >= 0) run.take_one(L::load(z + edge_at));
        const MaxSum a = warp_merge<32>(run.total());
        if (lane == 0) s_red[q][warp] = a;
    }
    typename P::In in{};
    float zy = 0.f;
    if (tid == 0) {
        in = p.in(row);
        zy = L::load(z + y);
    }
    __syncthreads();
    MaxSum a{kFloor, 0.f};                                      // in lane q of warp 0: of the block's part q
    if (warp == 0) {
        for (int q = 0; q < own; ++q) {
            const MaxSum b = warp_merge<kStreamWarps>(s_red[q][lane & (kStreamWarps - 1)]);
            if (lane == q) a = b;
        }
    }
    const int at = lane & (kMaxParts - 1);
    if (C == 1) {
        if (warp == 0) a = warp_merge<kMaxParts>({__shfl_sync(0xffffffffu, a.m, at), __shfl_sync(0xffffffffu, a.s, at)});
    } else {
        // every block writes its parts into every peer; the barrier passed first says that the peers run
        ptx::cluster_wait();
        if (warp == 0 && lane < own)
            for (int peer = 0; peer < C; ++peer) {
                const uint32_t to = ptx::map_to_cta(ptx::smem_u32(s_parts + part0 + lane), peer);
                ptx::st_remote_u32(to, __float_as_uint(a.m));
                ptx::st_remote_u32(to + 4, __float_as_uint(a.s));
            }
        ptx::cluster_arrive();
        ptx::cluster_wait();
        if (warp == 0) a = warp_merge<kMaxParts>(at < parts ? s_parts[at] : MaxSum{kFloor, 0.f});
    }
    if (tid == 0) {
        const float coef = plain(a.m) ? p.finish(row, in, zy, a, rank == 0) : 0.f;
        s_slope = P::kGradient ? slope_of(a, coef) : Slope{a.m, a.s, coef, 0.f};
    }
    __syncthreads();
    if (!plain(s_slope.m)) {                                    // seldom: every block takes the whole row
        a = row_stats<DT, T>(z, r.classes, s_red[0]);
        if (tid == 0) s_slope = {a.m, a.s, p.finish(row, in, zy, a, rank == 0), 0.f};
        __syncthreads();
    }
    if constexpr (P::kGradient) {
        const Slope g = s_slope;
        auto* d = r.gradient(row);
        if (g.coef == 0.f) {
            zero_row<DT, T>(d, r.classes, tid, rank, C);
            return;
        }
        if (!near<DT>(g.m)) {
            row_gradient<DT, T>(z, d, r.classes, y, {g.m, g.s}, g.coef, tid, rank, C);
            return;
        }
        auto* dv = d + sp.head;
        const bool wide = (reinterpret_cast<uintptr_t>(dv) & 15u) == 0;
        const int begin = part0 * part_vecs, end = own > 0 ? part_end(part0 + own - 1) : 0;
        auto sweep = [&](auto negative) {
            constexpr bool kNeg = decltype(negative)::value;
            int v = begin + tid;
            if (wide) {
                uint4* o = reinterpret_cast<uint4*>(dv);
                for (; v + 3 * T < end; v += 4 * T) {
                    const uint4 x[4] = {__ldcs(zv + v), __ldcs(zv + v + T), __ldcs(zv + v + 2 * T), __ldcs(zv + v + 3 * T)};
#pragma unroll
                    for (int k = 0; k < 4; ++k) __stcs(o + v + k * T, slope_vec<DT, kNeg>(x[k], g));
                }
                for (; v < end; v += T) __stcs(o + v, slope_vec<DT, kNeg>(__ldcs(zv + v), g));
            } else {
#pragma unroll 2
                for (; v < end; v += T)
                    store_any(dv + (int64_t)v * L::kVec, slope_vec<DT, kNeg>(__ldcs(zv + v), g), (int)sizeof(typename L::T));
            }
        };
        if (g.coef > 0.f) sweep(std::true_type{});
        else sweep(std::false_type{});
        if (edge_at >= 0) L::store(d + edge_at, g.at(L::load(z + edge_at), edge_at == y));
        // the label's element again, by the thread that stored its vector
        const int vy = y < sp.head ? -1 : (y - sp.head) / L::kVec;
        if (vy >= begin && vy < end && (vy - begin) % T == tid) L::store(d + y, g.at(L::load(z + y), true));
    }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// sum over the block's threads, in thread 0; `s_part` holds T / 32 entries
template <int T>
__device__ __forceinline__ double block_sum(double v, double* s_part) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    if (threadIdx.x == 0)
        for (int i = 0; i < T / 32; ++i) v += s_part[i];
    return v;
}

// Sequence sums, the pairs' losses and the rows' coefficients: a block per pair, sums in double in a fixed order.
// Sequence bounds come from device memory: they are clamped to the rows, whatever they say.  Bound by latency (10 us for
// the one pair of 4096 rows; a warp a pair took 70 us).
constexpr int kPairThreads = 1024;

__global__ void __launch_bounds__(kPairThreads)
preference_pairs(const double* logp, const float* row_sum, const int32_t* seq_starts, const float* ref_logp,
                 const float* scaling, double beta, double smoothing, int rows, int pairs, float* seq_logp,
                 float* loss_partial, float* coef) {
    __shared__ double s_part[kPairThreads / 32];
    __shared__ float s_pull;
    const int p = blockIdx.x;
    ptx::wait_prior_grid();
    ptx::let_next_grid_start();
    int lo[2], hi[2];
    double sums[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        lo[k] = min(max(seq_starts[2 * p + k], 0), rows);
        hi[k] = min(max(seq_starts[2 * p + k + 1], 0), rows);
        double t = 0.0;
#pragma unroll 8
        for (int i = lo[k] + threadIdx.x; i < hi[k]; i += kPairThreads) t += logp[i];
        sums[k] = block_sum<kPairThreads>(t, s_part);
    }
    if (threadIdx.x == 0) {
        seq_logp[2 * p] = (float)sums[0];
        seq_logp[2 * p + 1] = (float)sums[1];
        const double ref = ref_logp ? (double)ref_logp[2 * p] - (double)ref_logp[2 * p + 1] : 0.0;
        const double x = beta * (sums[0] - sums[1] - ref);
        // -log sigmoid(x) = max(-x, 0) + log1p(exp(-|x|)); sigmoid from the same exponential of a negative number
        const double tail = exp(-fabs(x)), soft = log1p(tail);
        const double up = x >= 0 ? 1.0 / (1.0 + tail) : tail / (1.0 + tail);        // sigmoid(x)
        const double down = x >= 0 ? tail / (1.0 + tail) : 1.0 / (1.0 + tail);      // sigmoid(-x)
        // a term with the factor 0 is left out: an answer without chance (x infinite) would make it 0 * inf
        const double part = ((smoothing < 1.0 ? (1.0 - smoothing) * (fmax(-x, 0.0) + soft) : 0.0) +
                             (smoothing > 0.0 ? smoothing * (fmax(x, 0.0) + soft) : 0.0)) / pairs;
        loss_partial[p] = (float)(x == x ? part : x);
        s_pull = (float)(beta * (smoothing * up - (1.0 - smoothing) * down) / pairs * (double)scaling[0]);
    }
    __syncthreads();
    const float pull = s_pull;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll 8
        for (int i = lo[k] + threadIdx.x; i < hi[k]; i += kPairThreads) coef[i] = row_sum[i] != 0.f ? (k ? -pull : pull) : 0.f;
    }
}

// Sum of the partial losses in double, in a fixed order, by one block of T threads.
template <int T>
__device__ __forceinline__ void sum_partials(const float* partial, int n, float* loss) {
    __shared__ double s_part[T / 32];
    double t = 0.0;
    for (int i = threadIdx.x; i < n; i += T) t += (double)partial[i];
    t = block_sum<T>(t, s_part);
    if (threadIdx.x == 0) *loss = (float)t;
}

constexpr int kSumThreads = 512;

__global__ void __launch_bounds__(kSumThreads)
partial_loss_sum(const float* partial, int n, float* loss) {
    ptx::wait_prior_grid();
    sum_partials<kSumThreads>(partial, n, loss);
}

// Second pass of the preference loss: every row's maximum, sum and coef are known, nothing is left to wait for.  G threads
// a row, or G = all of the block's for each of the `parts` of a long one; a thread's vectors in batches of four loads.
// The first block also adds up the loss.  Bound by HBM: 4096 x 32000 bfloat16 take 82 us under the profiler, 472 MB at 70 %
// of the DRAM's peak.  Groups of threads against a block a row (whole preference loss): 65536 x 64 31 us against 166 us,
// 16384 x 4096 78 us against 102 us.
constexpr int kSlopeThreads = 256;

template <int DT, int G>
__global__ void __launch_bounds__(kSlopeThreads)
preference_gradient_rows(Rows<DT> r, const float* row_max, const float* row_sum, const float* coef_of, int parts,
                         const float* loss_partial, int pairs, float* loss) {
    using L = Logit<DT>;
    // from the last row down: what the first pass read last is still in L2
    const int tid = threadIdx.x & (G - 1), group = blockIdx.x * (kSlopeThreads / G) + threadIdx.x / G;
    const int back = group / parts, part = group - back * parts, row = r.rows - 1 - back;
    ptx::wait_prior_grid();
    ptx::let_next_grid_start();
    if (blockIdx.x == 0) sum_partials<kSlopeThreads>(loss_partial, pairs, loss);
    if (row < 0) return;
    const float coef = coef_of[row];
    auto* d = r.gradient(row);
    if (coef == 0.f) {
        zero_row<DT, G>(d, r.classes, tid, part, parts);
        return;
    }
    const MaxSum a{row_max[row], row_sum[row]};
    const int y = r.labels[row];
    const auto* z = r.logits(row);
    if (!near<DT>(a.m)) {
        row_gradient<DT, G>(z, d, r.classes, y, a, coef, tid, part, parts);
        return;
    }
    const RowSplit sp(z, r.classes);
    const Slope g = slope_of(a, coef);
    const uint4* zv = reinterpret_cast<const uint4*>(z + sp.head);
    auto* dv = d + sp.head;
    const bool wide = (reinterpret_cast<uintptr_t>(dv) & 15u) == 0, neg = coef > 0.f;
#pragma unroll 1
    for (int v0 = part * 8 * G + tid; v0 < sp.nvec; v0 += parts * 8 * G)
#pragma unroll
        for (int b = 0; b < 8; b += 4) {
            uint4 raw[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (v0 + (b + k) * G < sp.nvec) raw[k] = __ldcs(zv + v0 + (b + k) * G);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int v = v0 + (b + k) * G;
                if (v >= sp.nvec) continue;
                const uint4 out = neg ? slope_vec<DT, true>(raw[k], g) : slope_vec<DT, false>(raw[k], g);
                if (wide) __stcs(reinterpret_cast<uint4*>(dv) + v, out);
                else store_any(dv + (int64_t)v * L::kVec, out, (int)sizeof(typename L::T));
            }
        }
    if (part == 0)
        for (int i = tid; i < sp.head + sp.tail; i += G) {
            const int e = sp.single(i, r.classes);
            L::store(d + e, g.at(L::load(z + e), e == y));
        }
    // the label's element again, by the thread that stored its vector
    const int vy = y < sp.head ? -1 : (y - sp.head) / L::kVec;
    if (vy >= 0 && vy < sp.nvec && vy / (8 * G) % parts == part && vy % G == tid) L::store(d + y, g.at(L::load(z + y), true));
}

// ---------------------------------------------------------------- argument checks
struct LogitArgs {
    const void* logits;
    int64_t logits_stride;
    const int32_t* labels;
    void* dlogits;
    int64_t dlogits_stride;
    int32_t rows, classes, dtype;
};

int elem_size(int dtype) { return dtype == TRB200_DTYPE_F32 ? 4 : 2; }

int check_logits(const LogitArgs& a, bool gradient, const char* who) {
    TRB_REQUIRE(valid_dtype(a.dtype) || a.dtype == TRB200_DTYPE_F32, TRB200_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d",
                who, a.dtype);
    TRB_REQUIRE(a.rows >= 0 && a.classes > 0 && a.logits_stride >= a.classes &&
                    (!gradient || a.dlogits_stride >= a.classes),
                TRB200_ERR_INVALID_ARGUMENT, "%s: bad sizes (rows=%d classes=%d)", who, a.rows, a.classes);
    TRB_REQUIRE(a.classes <= (1 << 30) && a.rows <= (1 << 30), TRB200_ERR_UNSUPPORTED, "%s: more than 2^30 rows or classes", who);
    if (a.rows == 0) return TRB200_OK;
    TRB_REQUIRE(a.logits && a.labels && (!gradient || a.dlogits), TRB200_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
    const uintptr_t mask = (uintptr_t)elem_size(a.dtype) - 1;
    TRB_REQUIRE(((reinterpret_cast<uintptr_t>(a.logits) | (gradient ? reinterpret_cast<uintptr_t>(a.dlogits) : 0)) & mask) == 0,
                TRB200_ERR_INVALID_ARGUMENT, "%s: logits and their gradient must be aligned to their element", who);
    if (gradient) {
        const uintptr_t z0 = reinterpret_cast<uintptr_t>(a.logits), d0 = reinterpret_cast<uintptr_t>(a.dlogits);
        const uintptr_t z1 = z0 + ((uintptr_t)(a.rows - 1) * (uintptr_t)a.logits_stride + a.classes) * elem_size(a.dtype);
        const uintptr_t d1 = d0 + ((uintptr_t)(a.rows - 1) * (uintptr_t)a.dlogits_stride + a.classes) * elem_size(a.dtype);
        TRB_REQUIRE(d1 <= z0 || z1 <= d0, TRB200_ERR_INVALID_ARGUMENT, "%s: the gradient must not overlap the logits", who);
    }
    return TRB200_OK;
}

template <int DT>
Rows<DT> rows_of(const LogitArgs& a) {
    using T = typename Logit<DT>::T;
    return {static_cast<const T*>(a.logits), a.logits_stride, static_cast<T*>(a.dlogits), a.dlogits_stride, a.labels, a.rows, a.classes};
}

// One kernel over the rows.  Which one goes by their length alone, as do the sums in it but for the row's alignment.
template <int DT, class P>
int launch_rows(const Rows<DT>& r, const P& p, cudaStream_t s, const char* who) {
    const int nvec = r.classes / Logit<DT>::kVec;
    if (nvec <= 2048 / Logit<DT>::kVec) {
        const int lanes = nvec <= 32 ? 8 : (nvec <= 128 ? 16 : 32);
        const int grid = (int)(((int64_t)r.rows * lanes + kShortThreads - 1) / kShortThreads);
        auto* kernel = nvec <= 8 ? rows_short<DT, 8, 1, P>
                                 : (nvec <= 32 ? rows_short<DT, 8, 4, P>
                                               : (nvec <= 64 ? rows_short<DT, 16, 4, P>
                                                             : (nvec <= 128 ? rows_short<DT, 16, 8, P> : rows_short<DT, 32, 8, P>)));
        if constexpr (DT == TRB200_DTYPE_F32)
            if (nvec > 256) kernel = rows_short<DT, 32, 16, P>;
        TRB_CUDA_TRY(launch_chained(kernel, grid, kShortThreads, 1, 0, s, r, p));
    } else {
        int parts = (nvec + kPartVecs - 1) / kPartVecs, part_vecs = kPartVecs;
        if (parts > kMaxParts) {
            parts = kMaxParts;
            part_vecs = (nvec + kMaxParts - 1) / kMaxParts;
        }
        // Blocks a row.  A gradient: one for each part, for the second read (see rows_streamed; 8192 x 131072 bfloat16 take
        // 748 us so, 835 us with twice as many blocks and 914 us with one for the row).  Otherwise one for all parts
        // (6000 x 50021: 91 us, two blocks 103 us: the blocks of a cluster start and end together), or one for each where
        // that would leave blocks of the GPU unused.
        const int T = nvec <= 1024 ? 64 : (nvec <= 2048 ? 128 : 256);
        const int64_t resident = (int64_t)sm_count() * (kStreamThreads / T);
        int C = 1;
        while (C < parts && r.rows <= 0x7fffffff / (2 * C) && (P::kGradient || r.rows * (int64_t)C < resident)) C *= 2;
        auto* kernel = T == 64 ? rows_streamed<DT, 64, P> : (T == 128 ? rows_streamed<DT, 128, P> : rows_streamed<DT, 256, P>);
        TRB_CUDA_TRY(launch_chained(kernel, r.rows * C, T, C, 0, s, r, p, C, parts, (parts + C - 1) / C, part_vecs));
    }
    TRB_LAUNCH_CHECK(who);
    return TRB200_OK;
}

}  // namespace

}  // namespace trb

// calls LAUNCH(DT) for the storage type
#define TRB_BY_DTYPE(dtype, LAUNCH)                                   \
    do {                                                              \
        if ((dtype) == TRB200_DTYPE_F16) { LAUNCH(TRB200_DTYPE_F16); } \
        else if ((dtype) == TRB200_DTYPE_BF16) { LAUNCH(TRB200_DTYPE_BF16); } \
        else { LAUNCH(TRB200_DTYPE_F32); }                            \
    } while (0)

extern "C" int trb200_token_logp(const void* logits, int64_t logits_stride, const int32_t* labels, float* logp,
                                 float* lse, int32_t rows, int32_t classes, int32_t dtype, void* stream) {
    const trb::LogitArgs a{logits, logits_stride, labels, nullptr, 0, rows, classes, dtype};
    const int rc = trb::check_logits(a, false, "token_logp");
    if (rc != TRB200_OK) return rc;
    if (rows == 0) return TRB200_OK;
    TRB_REQUIRE(logp, TRB200_ERR_INVALID_ARGUMENT, "token_logp: null pointer");
    TRB_REQUIRE(trb::aligned4(labels, logp, lse), TRB200_ERR_INVALID_ARGUMENT,
                "token_logp: labels, logp and lse must be aligned to 4 bytes");
    const trb::LogpRows p{logp, lse};
#define TRB_LAUNCH(DT) return trb::launch_rows<DT>(trb::rows_of<DT>(a), p, trb::as_stream(stream), "token_logp")
    TRB_BY_DTYPE(dtype, TRB_LAUNCH);
#undef TRB_LAUNCH
}

extern "C" int trb200_policy_loss_fused(const void* logits, int64_t logits_stride, const int32_t* actions,
                                        const float* old_logp, const float* ref_logp, const float* advantages,
                                        const float* weights, const float* scaling, float clip_low, float clip_high,
                                        float kl_coef, void* dlogits, int64_t dlogits_stride, float* logp,
                                        float* loss_partial, float* loss, int32_t rows, int32_t classes, int32_t dtype,
                                        void* stream) {
    const trb::LogitArgs a{logits, logits_stride, actions, dlogits, dlogits_stride, rows, classes, dtype};
    const int rc = trb::check_logits(a, true, "policy_loss");
    if (rc != TRB200_OK) return rc;
    TRB_REQUIRE(loss && scaling, TRB200_ERR_INVALID_ARGUMENT, "policy_loss: null pointer");
    TRB_REQUIRE(clip_low >= 0.f && clip_low <= 1.f && clip_high >= 0.f && std::isfinite(kl_coef),
                TRB200_ERR_INVALID_ARGUMENT, "policy_loss: clip_low must lie in [0, 1], clip_high >= 0, kl_coef finite");
    TRB_REQUIRE(ref_logp || kl_coef == 0.f, TRB200_ERR_INVALID_ARGUMENT, "policy_loss: a KL term needs ref_logp");
    TRB_REQUIRE(rows == 0 || (old_logp && advantages && logp && loss_partial), TRB200_ERR_INVALID_ARGUMENT,
                "policy_loss: null pointer");
    TRB_REQUIRE(trb::aligned4(actions, old_logp, ref_logp, advantages, weights, scaling, logp, loss_partial, loss),
                TRB200_ERR_INVALID_ARGUMENT, "policy_loss: arrays of 4-byte elements must be aligned to them");
    const trb::PolicyArgs p{old_logp, kl_coef != 0.f ? ref_logp : nullptr, advantages, weights, scaling, 1.0f - clip_low,
                            1.0f + clip_high, kl_coef, rows ? 1.0f / (float)rows : 0.f};
    if (rows > 0) {
        const trb::PolicyRows rows_p{p, logp, loss_partial};
        int rc2 = TRB200_OK;
#define TRB_LAUNCH(DT) rc2 = trb::launch_rows<DT>(trb::rows_of<DT>(a), rows_p, trb::as_stream(stream), "policy_loss")
        TRB_BY_DTYPE(dtype, TRB_LAUNCH);
#undef TRB_LAUNCH
        if (rc2 != TRB200_OK) return rc2;
    }
    TRB_CUDA_TRY(trb::launch_chained(trb::partial_loss_sum, 1, trb::kSumThreads, 1, 0, trb::as_stream(stream), loss_partial, rows, loss));
    TRB_LAUNCH_CHECK("partial_loss_sum");
    return TRB200_OK;
}

extern "C" size_t trb200_preference_loss_workspace_bytes(int32_t rows) {
    return rows > 0 ? (size_t)rows * (sizeof(double) + 3 * sizeof(float)) : 0;
}

extern "C" int trb200_preference_loss_fused(const void* logits, int64_t logits_stride, const int32_t* labels,
                                            const int32_t* seq_starts, const float* ref_logp, const float* scaling,
                                            double beta, double label_smoothing, void* dlogits, int64_t dlogits_stride,
                                            float* logp, float* seq_logp, float* loss_partial, float* loss, int32_t rows,
                                            int32_t pairs, int32_t classes, int32_t dtype, void* workspace,
                                            size_t workspace_bytes, void* stream) {
    const trb::LogitArgs a{logits, logits_stride, labels, dlogits, dlogits_stride, rows, classes, dtype};
    const int rc = trb::check_logits(a, true, "preference_loss");
    if (rc != TRB200_OK) return rc;
    TRB_REQUIRE(pairs > 0 && pairs <= (1 << 29), TRB200_ERR_INVALID_ARGUMENT, "preference_loss: bad number of pairs (%d)", pairs);
    TRB_REQUIRE(seq_starts && scaling && seq_logp && loss_partial && loss && (rows == 0 || logp),
                TRB200_ERR_INVALID_ARGUMENT, "preference_loss: null pointer");
    TRB_REQUIRE(trb::aligned4(labels, seq_starts, ref_logp, scaling, logp, seq_logp, loss_partial, loss),
                TRB200_ERR_INVALID_ARGUMENT, "preference_loss: arrays of 4-byte elements must be aligned to them");
    TRB_REQUIRE(std::isfinite(beta) && label_smoothing >= 0.0 && label_smoothing <= 1.0, TRB200_ERR_INVALID_ARGUMENT,
                "preference_loss: beta must be finite and label_smoothing lie in [0, 1]");
    TRB_REQUIRE(rows == 0 || (workspace && workspace_bytes >= trb200_preference_loss_workspace_bytes(rows) &&
                              (reinterpret_cast<uintptr_t>(workspace) & 7u) == 0),
                TRB200_ERR_WORKSPACE, "preference_loss: workspace missing, too small or misaligned");
    cudaStream_t s = trb::as_stream(stream);
    double* logp64 = static_cast<double*>(workspace);
    float* row_max = reinterpret_cast<float*>(logp64 + rows);
    float* row_sum = row_max + rows;
    float* coef = row_sum + rows;
    if (rows > 0) {
        const trb::PairRows p{seq_starts, 2 * pairs, logp, logp64, row_max, row_sum, coef};
        int rc2 = TRB200_OK;
#define TRB_LAUNCH(DT) rc2 = trb::launch_rows<DT>(trb::rows_of<DT>(a), p, s, "preference_loss statistics")
        TRB_BY_DTYPE(dtype, TRB_LAUNCH);
#undef TRB_LAUNCH
        if (rc2 != TRB200_OK) return rc2;
    }
    TRB_CUDA_TRY(trb::launch_chained(trb::preference_pairs, pairs, trb::kPairThreads, 1, 0, s, logp64, row_sum, seq_starts, ref_logp,
                                     scaling, beta, label_smoothing, rows, pairs, seq_logp, loss_partial, coef));
    TRB_LAUNCH_CHECK("preference_pairs");
    if (rows == 0) {
        TRB_CUDA_TRY(trb::launch_chained(trb::partial_loss_sum, 1, trb::kSumThreads, 1, 0, s, loss_partial, pairs, loss));
        TRB_LAUNCH_CHECK("partial_loss_sum");
    }
    if (rows > 0) {
        const int nvec = classes / (16 / trb::elem_size(dtype));
        // eight vectors a thread: 8 threads a row up to 64 vectors, 32 up to 512, then blocks of 2048 vectors each
        const int G = nvec <= 64 ? 8 : (nvec <= 512 ? 32 : 256);
        int parts = G < 256 ? 1 : (nvec + 2047) / 2048;
        if (parts > 0x7fffffff / rows) parts = 0x7fffffff / rows;
        const unsigned grid = (unsigned)(((int64_t)rows * parts * G + trb::kSlopeThreads - 1) / trb::kSlopeThreads);
        cudaError_t err = cudaSuccess;
#define TRB_LAUNCH(DT)                                                                                                \
    auto* kernel = G == 8 ? trb::preference_gradient_rows<DT, 8>                                                      \
                          : (G == 32 ? trb::preference_gradient_rows<DT, 32> : trb::preference_gradient_rows<DT, 256>); \
    err = trb::launch_chained(kernel, grid, trb::kSlopeThreads, 1, 0, s, trb::rows_of<DT>(a), row_max, row_sum, coef, parts, \
                              loss_partial, pairs, loss)
        TRB_BY_DTYPE(dtype, TRB_LAUNCH);
#undef TRB_LAUNCH
        TRB_CUDA_TRY(err);
        TRB_LAUNCH_CHECK("preference_gradient_rows");
    }
    return TRB200_OK;
}
