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
#include "common.cuh"

#include <cmath>

namespace trb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

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
    // the single element of this thread, or -1 (head + tail < 2 * 16 / sizeof(T) <= 16 threads have one)
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
// s counts exponentials against m.  m = -inf goes with s = 0 (nothing but -inf seen); a NaN ends up in s.
struct MaxSum { float m, s; };

// the number exponentials are taken against: 0 stands in for -inf, so that no difference of infinities is formed
__device__ __forceinline__ float pivot(float m) { return m == -INFINITY ? 0.f : m; }

__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b) {
    const float m = fmaxf(a.m, b.m), p = pivot(m);
    return {m, a.s * fast_exp2((a.m - p) * kLog2e) + b.s * fast_exp2((b.m - p) * kLog2e)};
}

template <int N>
__device__ __forceinline__ void take(MaxSum& a, const float (&f)[N]) {
    float m = a.m;
#pragma unroll
    for (int j = 0; j < N; ++j) m = fmaxf(m, f[j]);
    const float p = pivot(m);
    float s = a.s * fast_exp2((a.m - p) * kLog2e);
    // the difference is taken before the scaling: with the type's lowest value as mask, z * log2(e) would overflow
#pragma unroll
    for (int j = 0; j < N; ++j) s += fast_exp2((f[j] - p) * kLog2e);
    a = {m, s};
}

// the same MaxSum in every thread of a block of T threads; s_red holds T / 32 entries
template <int T>
__device__ __forceinline__ MaxSum block_merge(MaxSum a, MaxSum* s_red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        a = merge(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
    if (lane == 0) s_red[warp] = a;
    __syncthreads();
    a = lane < T / 32 ? s_red[lane] : MaxSum{-INFINITY, 0.f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        a = merge(a, {__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o)});
    return a;
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

// weighted loss of a row and its derivative with respect to logp
__device__ __forceinline__ void policy_row(const PolicyArgs& a, int row, float w, float logp, float& loss, float& slope) {
    const float adv = a.advantages[row];
    const float ratio = expf(logp - a.old_logp[row]);
    const float kept = ratio * adv;
    const float cut = fminf(fmaxf(ratio, a.low), a.high) * adv;
    float l, g;
    if (kept <= cut) { l = -kept; g = -kept; }
    else { l = kept > cut ? -cut : NAN; g = kept > cut ? 0.f : NAN; }     // unordered: a NaN stays one
    if (a.ref_logp) {
        const float gap = a.ref_logp[row] - logp;
        const float more = expm1f(gap);                         // no cancellation next to gap = 0
        l += a.kl_coef * (more - gap);
        g -= a.kl_coef * more;
    }
    loss = l * w;
    slope = g * w;
}

// ---------------------------------------------------------------- row kernels
template <int DT>
struct Rows {
    const typename Logit<DT>::T* z;
    int64_t z_stride;
    typename Logit<DT>::T* d;       // gradient
    int64_t d_stride;
    const int32_t* labels;
    int classes;
};

// maximum and sum of the row over the T threads of the block
template <int DT, int T>
__device__ __forceinline__ MaxSum row_stats(const typename Logit<DT>::T* z, int classes, MaxSum* s_red) {
    using L = Logit<DT>;
    const RowSplit sp(z, classes);
    MaxSum a{-INFINITY, 0.f};
    const int e = sp.single(threadIdx.x, classes);
    if (e >= 0) a = {L::load(z + e), 1.0f};
    if (a.m == -INFINITY) a.s = 0.f;
    if (isnan(a.m)) a = {-INFINITY, NAN};
    const uint4* zv = reinterpret_cast<const uint4*>(z + sp.head);
    int v = threadIdx.x;
    for (; v + 3 * T < sp.nvec; v += 4 * T) {           // four loads in flight
        uint4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = zv[v + u * T];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float f[L::kVec];
            L::unpack(raw[u], f);
            take(a, f);
        }
    }
    for (; v < sp.nvec; v += T) {
        float f[L::kVec];
        L::unpack(zv[v], f);
        take(a, f);
    }
    return block_merge<T>(a, s_red);
}

// d = coef * ([c == y] - exp(z - m) / s) over the T threads of the block; coef == 0 writes zeros without reading z
template <int DT, int T>
__device__ __forceinline__ void row_gradient(const typename Logit<DT>::T* z, typename Logit<DT>::T* d, int classes,
                                             int y, float m, float s, float coef) {
    using L = Logit<DT>;
    constexpr int kSize = (int)sizeof(typename L::T);
    if (coef == 0.f) {
        const RowSplit sp(d, classes);
        const int e = sp.single(threadIdx.x, classes);
        if (e >= 0) L::store(d + e, 0.f);
        uint4* dv = reinterpret_cast<uint4*>(d + sp.head);
        for (int v = threadIdx.x; v < sp.nvec; v += T) dv[v] = make_uint4(0u, 0u, 0u, 0u);
        return;
    }
    const RowSplit sp(z, classes);
    const float p = pivot(m), fall = -coef / s;
    const int e = sp.single(threadIdx.x, classes);
    if (e >= 0) L::store(d + e, fmaf(fast_exp2((L::load(z + e) - p) * kLog2e), fall, e == y ? coef : 0.f));
    const uint4* zv = reinterpret_cast<const uint4*>(z + sp.head);
    auto one = [&](const uint4& raw, int v) {
        float f[L::kVec];
        L::unpack(raw, f);
#pragma unroll
        for (int j = 0; j < L::kVec; ++j) f[j] = fast_exp2((f[j] - p) * kLog2e) * fall;
        const int c0 = sp.head + v * L::kVec, jy = y - c0;
        if ((unsigned)jy < (unsigned)L::kVec) {                 // the label sits in at most one vector of the row
#pragma unroll
            for (int j = 0; j < L::kVec; ++j) f[j] += j == jy ? coef : 0.f;
        }
        store_any(d + c0, L::pack(f), kSize);
    };
    int v = threadIdx.x;
    for (; v + 3 * T < sp.nvec; v += 4 * T) {
        uint4 raw[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = zv[v + u * T];
#pragma unroll
        for (int u = 0; u < 4; ++u) one(raw[u], v + u * T);
    }
    for (; v < sp.nvec; v += T) one(zv[v], v);
}

// log-probability of the label; a row that is read has 0 <= y < classes
template <int DT>
__device__ __forceinline__ float label_logp(const typename Logit<DT>::T* z, int y, MaxSum a) {
    return (Logit<DT>::load(z + y) - pivot(a.m)) - logf(a.s);
}

template <int DT, int T>
__global__ void __launch_bounds__(T)
token_logp_rows(Rows<DT> r, float* __restrict__ logp, float* __restrict__ lse) {
    __shared__ MaxSum s_red[T / 32];
    const int row = blockIdx.x;
    const int y = r.labels[row];
    if ((unsigned)y >= (unsigned)r.classes) {
        if (threadIdx.x == 0) {
            logp[row] = 0.f;
            if (lse) lse[row] = 0.f;
        }
        return;
    }
    const auto* z = r.z + (int64_t)row * r.z_stride;
    const MaxSum a = row_stats<DT, T>(z, r.classes, s_red);
    if (threadIdx.x == 0) {
        const bool none = a.s == 0.f;                           // every logit is -inf
        logp[row] = none ? -INFINITY : label_logp<DT>(z, y, a);
        if (lse) lse[row] = none ? -INFINITY : a.m + logf(a.s);
    }
}

template <int DT, int T>
__global__ void __launch_bounds__(T)
policy_loss_rows(Rows<DT> r, PolicyArgs p, float* __restrict__ logp, float* __restrict__ loss_partial) {
    __shared__ MaxSum s_red[T / 32];
    const int row = blockIdx.x;
    const int y = r.labels[row];
    const float w = p.weights ? p.weights[row] : p.even_weight;
    const auto* z = r.z + (int64_t)row * r.z_stride;
    float lp = 0.f, loss = 0.f, coef = 0.f;
    MaxSum a{0.f, 1.f};
    if ((unsigned)y < (unsigned)r.classes && w != 0.f) {
        a = row_stats<DT, T>(z, r.classes, s_red);
        if (a.s != 0.f) {
            lp = label_logp<DT>(z, y, a);
            policy_row(p, row, w, lp, loss, coef);
            coef *= p.scaling[0];
        }
    }
    if (threadIdx.x == 0) {
        logp[row] = lp;
        loss_partial[row] = loss;
    }
    row_gradient<DT, T>(z, r.d + (int64_t)row * r.d_stride, r.classes, y, a.m, a.s, coef);
}

// first pass of the preference loss: statistics of the rows that count; coef starts at 0 for every row
template <int DT, int T>
__global__ void __launch_bounds__(T)
preference_stats_rows(Rows<DT> r, const int32_t* __restrict__ seq_starts, int seqs, float* __restrict__ logp,
                      float* __restrict__ row_max, float* __restrict__ row_sum, float* __restrict__ coef) {
    __shared__ MaxSum s_red[T / 32];
    const int row = blockIdx.x;
    const int y = r.labels[row];
    const bool counts = (unsigned)y < (unsigned)r.classes && row >= seq_starts[0] && row < seq_starts[seqs];
    const auto* z = r.z + (int64_t)row * r.z_stride;
    MaxSum a{0.f, 0.f};
    if (counts) a = row_stats<DT, T>(z, r.classes, s_red);
    if (threadIdx.x == 0) {
        logp[row] = a.s != 0.f ? label_logp<DT>(z, y, a) : 0.f;
        row_max[row] = a.m;
        row_sum[row] = a.s;                                     // 0: the row does not count
        coef[row] = 0.f;
    }
}

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Sequence sums, the pairs' losses and the rows' coefficients: one warp per pair, sums in double in a fixed order.
// Sequence bounds come from device memory: they are clamped to the rows, whatever they say.
__global__ void __launch_bounds__(1024)
preference_pairs(const float* __restrict__ logp, const float* __restrict__ row_sum,
                 const int32_t* __restrict__ seq_starts, const float* __restrict__ ref_logp,
                 const float* __restrict__ scaling, double beta, double smoothing, int rows, int pairs,
                 float* __restrict__ seq_logp, float* __restrict__ loss_partial, float* __restrict__ loss,
                 float* __restrict__ coef) {
    __shared__ double s_loss[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double mine = 0.0;
    for (int p = warp; p < pairs; p += 32) {
        double sums[2];
        int lo[2], hi[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            lo[k] = min(max(seq_starts[2 * p + k], 0), rows);
            hi[k] = min(max(seq_starts[2 * p + k + 1], 0), rows);
            double t = 0.0;
            for (int i = lo[k] + lane; i < hi[k]; i += 32) t += (double)logp[i];
            sums[k] = warp_sum(t);
            if (lane == 0) seq_logp[2 * p + k] = (float)sums[k];
        }
        const double ref = ref_logp ? (double)ref_logp[2 * p] - (double)ref_logp[2 * p + 1] : 0.0;
        const double x = beta * (sums[0] - sums[1] - ref);
        // -log sigmoid(x) = max(-x, 0) + log1p(exp(-|x|)); sigmoid from the same exponential of a negative number
        const double tail = exp(-fabs(x)), soft = log1p(tail);
        const double up = x >= 0 ? 1.0 / (1.0 + tail) : tail / (1.0 + tail);        // sigmoid(x)
        const double down = x >= 0 ? tail / (1.0 + tail) : 1.0 / (1.0 + tail);      // sigmoid(-x)
        const double part = ((1.0 - smoothing) * (fmax(-x, 0.0) + soft) + smoothing * (fmax(x, 0.0) + soft)) / pairs;
        const float pull = (float)(beta * (smoothing * up - (1.0 - smoothing) * down) / pairs * (double)scaling[0]);
        if (lane == 0) loss_partial[p] = (float)(x == x ? part : x);
        mine += x == x ? part : x;
#pragma unroll
        for (int k = 0; k < 2; ++k)
            for (int i = lo[k] + lane; i < hi[k]; i += 32)
                if (row_sum[i] != 0.f) coef[i] = k ? -pull : pull;
    }
    if (lane == 0) s_loss[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 32; ++i) t += s_loss[i];
        *loss = (float)t;
    }
}

template <int DT, int T>
__global__ void __launch_bounds__(T)
preference_gradient_rows(Rows<DT> r, const float* __restrict__ row_max, const float* __restrict__ row_sum,
                         const float* __restrict__ coef) {
    const int row = blockIdx.x;
    row_gradient<DT, T>(r.z + (int64_t)row * r.z_stride, r.d + (int64_t)row * r.d_stride, r.classes, r.labels[row],
                        row_max[row], row_sum[row], coef[row]);
}

// Sum of the rows' losses in double, in a fixed order.
__global__ void __launch_bounds__(1024)
row_loss_sum(const float* __restrict__ partial, int rows, float* __restrict__ loss) {
    __shared__ double s_part[32];
    double t = 0.0;
    for (int i = threadIdx.x; i < rows; i += 1024) t += (double)partial[i];
    t = warp_sum(t);
    if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = t;
    __syncthreads();
    if (threadIdx.x < 32) {
        t = warp_sum(s_part[threadIdx.x]);
        if (threadIdx.x == 0) *loss = (float)t;
    }
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
    TRB_REQUIRE(a.classes <= (1 << 30), TRB200_ERR_UNSUPPORTED, "%s: more than 2^30 classes", who);
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
    return {static_cast<const T*>(a.logits), a.logits_stride, static_cast<T*>(a.dlogits), a.dlogits_stride, a.labels, a.classes};
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
#define TRB_LAUNCH(DT) \
    trb::token_logp_rows<DT, 256><<<rows, 256, 0, trb::as_stream(stream)>>>(trb::rows_of<DT>(a), logp, lse)
    TRB_BY_DTYPE(dtype, TRB_LAUNCH);
#undef TRB_LAUNCH
    TRB_LAUNCH_CHECK("token_logp_rows");
    return TRB200_OK;
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
    const trb::PolicyArgs p{old_logp, kl_coef != 0.f ? ref_logp : nullptr, advantages, weights, scaling, 1.0f - clip_low,
                            1.0f + clip_high, kl_coef, rows ? 1.0f / (float)rows : 0.f};
    if (rows > 0) {
#define TRB_LAUNCH(DT) \
    trb::policy_loss_rows<DT, 256><<<rows, 256, 0, trb::as_stream(stream)>>>(trb::rows_of<DT>(a), p, logp, loss_partial)
        TRB_BY_DTYPE(dtype, TRB_LAUNCH);
#undef TRB_LAUNCH
        TRB_LAUNCH_CHECK("policy_loss_rows");
    }
    trb::row_loss_sum<<<1, 1024, 0, trb::as_stream(stream)>>>(loss_partial, rows, loss);
    TRB_LAUNCH_CHECK("row_loss_sum");
    return TRB200_OK;
}

extern "C" size_t trb200_preference_loss_workspace_bytes(int32_t rows) {
    return rows > 0 ? (size_t)rows * 3 * sizeof(float) : 0;
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
    TRB_REQUIRE(std::isfinite(beta) && label_smoothing >= 0.0 && label_smoothing <= 1.0, TRB200_ERR_INVALID_ARGUMENT,
                "preference_loss: beta must be finite and label_smoothing lie in [0, 1]");
    TRB_REQUIRE(rows == 0 || (workspace && workspace_bytes >= trb200_preference_loss_workspace_bytes(rows) &&
                              (reinterpret_cast<uintptr_t>(workspace) & 3u) == 0),
                TRB200_ERR_WORKSPACE, "preference_loss: workspace missing, too small or misaligned");
    cudaStream_t s = trb::as_stream(stream);
    float* row_max = static_cast<float*>(workspace);
    float* row_sum = row_max + rows;
    float* coef = row_sum + rows;
    if (rows > 0) {
#define TRB_LAUNCH(DT)                                                                                               \
    trb::preference_stats_rows<DT, 256><<<rows, 256, 0, s>>>(trb::rows_of<DT>(a), seq_starts, 2 * pairs, logp, row_max, \
                                                             row_sum, coef)
        TRB_BY_DTYPE(dtype, TRB_LAUNCH);
#undef TRB_LAUNCH
        TRB_LAUNCH_CHECK("preference_stats_rows");
    }
    trb::preference_pairs<<<1, 1024, 0, s>>>(logp, row_sum, seq_starts, ref_logp, scaling, beta, label_smoothing, rows,
                                             pairs, seq_logp, loss_partial, loss, coef);
    TRB_LAUNCH_CHECK("preference_pairs");
    if (rows > 0) {
#define TRB_LAUNCH(DT) \
    trb::preference_gradient_rows<DT, 256><<<rows, 256, 0, s>>>(trb::rows_of<DT>(a), row_max, row_sum, coef)
        TRB_BY_DTYPE(dtype, TRB_LAUNCH);
#undef TRB_LAUNCH
        TRB_LAUNCH_CHECK("preference_gradient_rows");
    }
    return TRB200_OK;
}
