// gk_policy_loss.cu - the policy loss of a training step and its gradient.
//
// For a row of logits z with legal entries L (all of them without a mask),
//   log p_j = z_j - M - log S,  M = max_L z,  S = sum_L exp(z_j - M),
// the row's loss has up to three terms:
//   clipped ratio   -min(q A, clip(q, lo, hi) A),  q = exp(log p_a - old)
//   KL estimate     kl_weight (e^d - d - 1),       d = reference - log p_a
//   target          target_weight sum_j t_j (log t_j - log p_j)
// and its gradient is, with c the derivative by log p_a and T = sum_j t_j,
//   dz_j = (target_weight T - c) p_j - target_weight t_j + c [j = a].
// The loss is the sum of the rows divided by the denominator.
//
// The row statistics, the row terms and the gradient are fp32 (row sums are
// added in double); the gradient is rounded once to the logits' type. exp of
// 16-bit logits uses the hardware's 2^x (relative error about 2^-22, far below
// the 2^-9 of the rounded result); fp32 logits use expf.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>
#include <type_traits>

#include "../../include/gk.h"
#include "gk_act.cuh"
#include "gk_launch.cuh"
#include "gk_row_part.cuh"

namespace gk {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kRowWarps = 8;        // rows per block of the short-row kernel
constexpr int kShortRow = 256;      // longest row that one warp keeps in registers
constexpr int kLongThreads = 256;   // threads per CTA of the long-row kernel
constexpr int kMaxCluster = 8;

struct None {};

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float exp_of(float d) { return ex2(d * 1.4426950408889634f); }

// exp(x - m) for many x of one row. For 16-bit logits it is 2^(x s - m s),
// one multiply-add and one 2^x; `correct` undoes the rounding of m s, which
// all terms share. From 1e5 on 16-bit values are 32 (fp16) or 512 and more
// (bf16) apart: exp is then 1 or nothing, which 2^(x - m) gives without overflow.
template <typename T>
struct Exp {
    float scale, offset, correct;
    __device__ __forceinline__ explicit Exp(float m) {
        scale = fabsf(m) < 1e5f ? 1.4426950408889634f : 1.0f;
        offset = m * scale;
        const float rest = fmaf(m, scale, -offset);
        correct = fabsf(rest) < 1.0f ? ex2(-rest) : 1.0f;  // not a number for an infinite m
    }
    __device__ __forceinline__ float operator()(float x) const { return ex2(fmaf(x, scale, -offset)); }
    __device__ __forceinline__ float term(float x) const { return (*this)(x); }  // of the sum
    __device__ __forceinline__ uint64_t pair(float x, float y) const {          // of both
        float a, b;
        halves(fma2(two(x, y), two(scale, scale), two(-offset, -offset)), a, b);
        return two(ex2(a), ex2(b));
    }
};
// fp32 logits: the difference first, which keeps the exponent's error at the
// last bit of x - m; in the row's sum, which every log-probability is taken
// from, also without the small bias of the quick 2^x.
template <>
struct Exp<float> {
    float m;
    static constexpr float correct = 1.0f;
    __device__ __forceinline__ explicit Exp(float top) : m(top) {}
    __device__ __forceinline__ float operator()(float x) const { return ex2((x - m) * 1.4426950408889634f); }
    __device__ __forceinline__ float term(float x) const { return expf(x - m); }
};

// Elements of one 16-byte vector of logits.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <int BYTES>
struct Raw;
template <>
struct Raw<1> {
    using type = uint8_t;
};
template <>
struct Raw<4> {
    using type = uint32_t;
};
template <>
struct Raw<8> {
    using type = uint2;
};
template <>
struct Raw<16> {
    using type = uint4;
};

// V consecutive entries of a row, masked ones as -inf, with a bit an entry for the legal ones.
template <typename TL, int V>
struct Group {
    static constexpr int kWords = V * (int)sizeof(TL) / 4;
    uint32_t w[V > 1 ? kWords : 1];  // the entries as they lie in memory; V == 1: one entry, as fp32
    uint32_t legal;
    __device__ __forceinline__ float x(int i) const {
        if constexpr (V == 1 || sizeof(TL) == 4) {
            return __uint_as_float(w[i]);
        } else if constexpr (std::is_same<TL, __half>::value) {
            const __half2 h = *reinterpret_cast<const __half2*>(&w[i / 2]);
            return i & 1 ? __high2float(h) : __low2float(h);
        } else {
            // From the word: one shift or mask an entry.
            return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        }
    }
    __device__ __forceinline__ float top() const {
        if constexpr (V == 8) {  // 16-bit logits: in pairs, which keeps them packed
            using P = typename std::conditional<std::is_same<TL, __half>::value, __half2, __nv_bfloat162>::type;
            const P* v = reinterpret_cast<const P*>(w);
            const P m = __hmax2(__hmax2(v[0], v[1]), __hmax2(v[2], v[3]));
            return fmaxf(to_f(m.x), to_f(m.y));
        } else {
            float m = x(0);
#pragma unroll
            for (int i = 1; i < V; ++i) m = fmaxf(m, x(i));
            return m;
        }
    }
    __device__ __forceinline__ void hide(int i) {
        if constexpr (V == 1 || sizeof(TL) == 4)
            w[i] = 0xff800000u;
        else if constexpr (std::is_same<TL, __half>::value)
            w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | 0xfc000000u : (w[i / 2] & 0xffff0000u) | 0xfc00u;
        else
            w[i / 2] = i & 1 ? (w[i / 2] & 0xffffu) | 0xff800000u : (w[i / 2] & 0xffff0000u) | 0xff80u;
    }
    // All V entries lie in the row; `from` is 16-byte aligned if V > 1.
    template <bool MASK>
    __device__ __forceinline__ void load(const TL* from, const uint8_t* mask) {
        legal = (1u << V) - 1u;
        if constexpr (V > 1) {
            const uint4 v = *reinterpret_cast<const uint4*>(from);
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else {
            w[0] = __float_as_uint(to_f(*from));
        }
        if constexpr (MASK) {
            alignas(V) uint8_t m[V];
            using R = typename Raw<V>::type;
            *reinterpret_cast<R*>(m) = __ldg(reinterpret_cast<const R*>(mask));
            legal = 0u;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                legal |= (m[i] != 0 ? 1u : 0u) << i;
                if (m[i] == 0) hide(i);
            }
        }
    }
    // The group at the row's start or end: entries outside [0, cols) count as masked.
    __device__ __forceinline__ void load_edge(const TL* lrow, const uint8_t* mrow, int first, int cols) {
        legal = 0u;
#pragma unroll
        for (int i = 0; i < (V > 1 ? kWords : 1); ++i) w[i] = 0u;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int j = first + i;
            const bool in = j >= 0 && j < cols && (mrow == nullptr || mrow[j] != 0);
            legal |= (in ? 1u : 0u) << i;
            if (!in)
                hide(i);
            else if constexpr (V == 1 || sizeof(TL) == 4)
                w[i] = __float_as_uint(to_f(lrow[j]));
            else
                w[i / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(lrow)[j] << (16 * (i & 1));
        }
    }
};

// The same entries of the target, 0 where `legal` has no bit.
template <typename TT, int V>
__device__ __forceinline__ void load_target(const TT* trow, uint32_t legal, int first, bool edge, float (&t)[V]) {
    if constexpr (std::is_same<TT, None>::value) {
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] = 0.0f;
    } else {
        if (V > 1 && !edge) {
            if constexpr (V > 1) {
                alignas(16) TT tv[V];
#pragma unroll
                for (int k = 0; k < (int)(V * sizeof(TT) / 16); ++k)
                    reinterpret_cast<uint4*>(tv)[k] = __ldg(reinterpret_cast<const uint4*>(trow + first) + k);
#pragma unroll
                for (int i = 0; i < V; ++i) t[i] = (legal >> i) & 1u ? to_f(tv[i]) : 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) t[i] = (legal >> i) & 1u ? to_f(trow[first + i]) : 0.0f;
        }
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pair_of(float lo, float hi) {
    uint32_t v;
    if constexpr (std::is_same<T, __half>::value)
        *reinterpret_cast<__half2*>(&v) = __floats2half2_rn(lo, hi);
    else
        *reinterpret_cast<__nv_bfloat162*>(&v) = __floats2bfloat162_rn(lo, hi);
    return v;
}
template <typename TL, int V>
__device__ __forceinline__ void store_group(TL* grow, int first, int cols, bool edge, const float (&g)[V]) {
    if (V > 1 && !edge) {
        if constexpr (V > 1) {
            uint4 w;
            if constexpr (V == 4)
                w = make_uint4(__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]),
                               __float_as_uint(g[3]));
            else
                w = make_uint4(pair_of<TL>(g[0], g[1]), pair_of<TL>(g[2], g[3]), pair_of<TL>(g[4], g[5]),
                               pair_of<TL>(g[6], g[7]));
            __stcs(reinterpret_cast<uint4*>(grow + first), w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (first + i >= 0 && first + i < cols) grow[first + i] = from_f<TL>(g[i]);
    }
}

// Maximum and sum of exponentials of a part of a row. M starts at the lowest
// finite value, so -inf entries add exp(-inf) = 0 and a row of nothing but the
// lowest value is uniform; S == 0 means that nothing is left.
struct Softmax {
    float m = -FLT_MAX, s = 0.0f;
    // Symmetric, so a butterfly of joins gives every lane the same bits.
    __device__ __forceinline__ void join(float m2, float s2) {
        const float top = fmaxf(m, m2);
        // A part with nothing in it must not scale by exp(lowest - top).
        s = (s == 0.0f ? 0.0f : s * exp_of(m - top)) + (s2 == 0.0f ? 0.0f : s2 * exp_of(m2 - top));
        m = top;
    }
    __device__ __forceinline__ void join_lanes(int lanes) {
        for (int o = lanes >> 1; o; o >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m, o), s2 = __shfl_xor_sync(0xffffffffu, s, o);
            join(m2, s2);
        }
    }
};

struct Row {
    float m, inv_s, log_s, total_t;  // inv_s 0: the row is skipped
    float c;                         // derivative of the row's loss by log p of the action
    float loss;                      // without the target term
    float log_p;
    int64_t action;                  // -1: none
};

// What the row's scalar terms read; fetched before the statistics are known.
struct RowInput {
    int64_t action = -1;
    float x = 0.0f, old = 0.0f, advantage = 0.0f, reference = 0.0f;
    bool legal = false;
};
template <typename TL>
__device__ __forceinline__ RowInput row_input(const gk_policy_loss_t& p, int64_t r, const TL* lrow,
                                              const uint8_t* mrow) {
    RowInput in;
    if (p.actions != nullptr) {
        in.action = p.actions[r];
        in.old = p.old_log_probs[r];
        in.advantage = p.advantages[r];
        if (p.reference_log_probs != nullptr) in.reference = p.reference_log_probs[r];
        in.legal = in.action >= 0 && in.action < p.cols && (mrow == nullptr || mrow[in.action] != 0);
        if (in.legal) in.x = to_f(lrow[in.action]);
    }
    return in;
}

// The row's scalar terms from its statistics. WIDE: a long row's log p is in
// the tens, where the ratio exp(log p - old) would feel the last fp32 bit of
// log p, so the difference is formed in double (by one thread a row).
template <bool WIDE>
__device__ __forceinline__ Row row_terms(const gk_policy_loss_t& p, const RowInput& in, float m, float s,
                                         float total_t) {
    Row o;
    o.m = m;
    o.total_t = total_t;
    o.c = o.loss = o.log_p = 0.0f;
    o.log_s = logf(s);
    o.action = -1;
    bool skip = s == 0.0f;
    if (p.actions != nullptr) {
        skip = skip || in.action < 0;
        if (!skip) {
            if (!in.legal) {
                // There is no log-probability to train on.
                o.c = o.loss = o.log_p = nanf("");
            } else {
                o.action = in.action;
                using W = typename std::conditional<WIDE, double, float>::type;
                W log_s = o.log_s;
                if (WIDE && s < INFINITY) {
                    // s = f 2^k with f in [0.75, 1.5): log f is small, so its last bit is too.
                    const int k = (int)((__float_as_uint(s) + 0x400000u) >> 23) - 127;
                    log_s = (W)k * (W)0.69314718055994531 + (W)logf(__uint_as_float(__float_as_uint(s) - (k << 23)));
                }
                const W log_p = ((W)in.x - (W)m) - log_s;
                o.log_p = (float)log_p;
                const float adv = in.advantage;
                const float q = expf((float)(log_p - (W)in.old));
                const float free = q * adv, held = fminf(fmaxf(q, p.clip_low), p.clip_high) * adv;
                // fminf drops a NaN; the comparisons keep it.
                o.loss = free <= held ? -free : (held < free ? -held : nanf(""));
                o.c = free <= held ? -free : (held < free ? 0.0f : nanf(""));
                if (p.reference_log_probs != nullptr) {
                    const float d = (float)((W)in.reference - log_p);
                    const float e = expm1f(d);
                    o.loss += p.kl_weight * (e - d);
                    o.c -= p.kl_weight * e;
                }
            }
        }
    }
    o.inv_s = skip ? 0.0f : 1.0f / s;
    if (skip) o.total_t = 0.0f;
    return o;
}

__device__ __forceinline__ float inverse_denominator(const gk_policy_loss_t& p) {
    return 1.0f / (p.denominator_ptr != nullptr ? *p.denominator_ptr : p.denominator);
}

// Gradient of a group but for the action's own part: `kp` multiplies exp(x - M), `kt` the target.
template <typename TL, typename TT, int V>
__device__ __forceinline__ void gradient_group(const Group<TL, V>& h, const float (&t)[V], const Exp<TL>& e, float kp,
                                               float kt, float (&g)[V]) {
    if constexpr (V > 1 && sizeof(TL) == 2) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            uint64_t v = mul2(e.pair(h.x(i), h.x(i + 1)), two(kp, kp));
            if constexpr (!std::is_same<TT, None>::value) v = fma2(two(t[i], t[i + 1]), two(-kt, -kt), v);
            halves(v, g[i], g[i + 1]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            g[i] = kp * e(h.x(i));
            if constexpr (!std::is_same<TT, None>::value) g[i] -= kt * t[i];
        }
    }
}

// t (log t - d), with d the entry's log-probability or its distance to a
// maximum; 0 for t = 0 whatever d is, not a number for a t below 0.
__device__ __forceinline__ float target_term(float t, float d) {
    const float term = t * (__logf(t) - d);
    return t == 0.0f ? 0.0f : term;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

__device__ __forceinline__ void write_row(const gk_policy_loss_t& p, int64_t r, const Row& o) {
    reinterpret_cast<float4*>(p.stats)[r] = make_float4(o.m, o.inv_s, o.c, o.total_t);
    if (p.log_probs != nullptr) p.log_probs[r] = o.inv_s == 0.0f ? 0.0f : o.log_p;
}

// The sum of the blocks' sums in their order; one block.
__device__ __forceinline__ void finish_loss(const gk_policy_loss_t& p, double sum) {
    *p.loss = (float)(sum * (1.0 / (double)(p.denominator_ptr != nullptr ? *p.denominator_ptr : p.denominator)));
}

__global__ void __launch_bounds__(256) policy_loss_sum_kernel(gk_policy_loss_t p, int parts) {
    __shared__ double sums[256];
    double v = 0.0;
    for (int i = threadIdx.x; i < parts; i += 256) v += p.partials[i];
    sums[threadIdx.x] = v;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (threadIdx.x < o) sums[threadIdx.x] += sums[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) finish_loss(p, sums[0]);
}

// Rows of at most 32 * NPL entries: a warp holds its row in registers, so
// logits, mask and target are read once and the gradient is written in the
// same pass. Lane l holds entries l, l + 32, ... Bound by instructions (four
// selects by mask and target an entry): 65536 x 82 fp32 with mask and target
// 44 us, 1.6 TB/s of what it has to move; 256 rows 2.7 us.
template <typename TL, typename TT, int NPL>
__global__ void __launch_bounds__(kRowWarps * 32) policy_loss_rows_kernel(gk_policy_loss_t p) {
    __shared__ double sums[kRowWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double sum = 0.0;
    const float inv_n = inverse_denominator(p);
    for (int64_t r = (int64_t)blockIdx.x * kRowWarps + warp; r < p.rows; r += (int64_t)gridDim.x * kRowWarps) {
        const TL* lrow = static_cast<const TL*>(p.logits) + r * p.logits_stride;
        const uint8_t* mrow = p.mask == nullptr ? nullptr : p.mask + r * p.mask_stride;
        const TT* trow = std::is_same<TT, None>::value ? nullptr
                                                       : static_cast<const TT*>(p.target) + r * p.target_stride;
        float x[NPL], t[NPL];
        uint32_t legal = 0u;
        float m = -FLT_MAX, total_t = 0.0f;
        const RowInput in_row = row_input(p, r, lrow, mrow);
#pragma unroll
        for (int k = 0; k < NPL; ++k) {
            const int j = lane + 32 * k;
            const bool in = j < p.cols && (mrow == nullptr || mrow[j] != 0);
            legal |= (in ? 1u : 0u) << k;
            x[k] = in ? to_f(lrow[j]) : -INFINITY;
            t[k] = 0.0f;
            if constexpr (!std::is_same<TT, None>::value) t[k] = in ? to_f(trow[j]) : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < NPL; ++k) {
            m = fmaxf(m, x[k]);
            total_t += t[k];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        const Exp<TL> exp_m(m);
        float e[NPL], s = 0.0f;
#pragma unroll
        for (int k = 0; k < NPL; ++k) {
            e[k] = exp_m.term(x[k]);
            s += e[k];
        }
        s = warp_sum(s) * exp_m.correct;
        if constexpr (!std::is_same<TT, None>::value) total_t = warp_sum(total_t);
        const Row o = row_terms<false>(p, in_row, m, s, total_t);
        float loss = lane == 0 ? o.loss : 0.0f;
        if constexpr (!std::is_same<TT, None>::value) {
            float kl = 0.0f;
#pragma unroll
            for (int k = 0; k < NPL; ++k) kl += target_term(t[k], (x[k] - m) - o.log_s);
            kl = warp_sum(kl);
            if (lane == 0 && o.inv_s != 0.0f) loss += p.target_weight * kl;
        }
        if (lane == 0) {
            sum += (double)loss;
            write_row(p, r, o);
        }
        if (p.grad != nullptr) {
            TL* grow = static_cast<TL*>(p.grad) + r * p.cols;
            const float kp = inv_n * (p.target_weight * o.total_t - o.c) * o.inv_s * exp_m.correct;
            const float kt = inv_n * p.target_weight;
#pragma unroll
            for (int k = 0; k < NPL; ++k) {
                const int j = lane + 32 * k;
                if (j >= p.cols) continue;
                float g = 0.0f;
                if (((legal >> k) & 1u) && o.inv_s != 0.0f) {
                    g = kp * e[k] - kt * t[k];
                    if (j == o.action) g += inv_n * o.c;
                }
                grow[j] = from_f<TL>(g);
            }
        }
    }
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double v = 0.0;
        for (int w = 0; w < kRowWarps; ++w) v += sums[w];
        if (gridDim.x == 1)
            finish_loss(p, v);
        else
            p.partials[blockIdx.x] = v;
    }
}

// The part of a row that one CTA of a cluster takes, and its operands' rows.
template <typename TL, typename TT, int V>
struct Part : RowPart<V> {
    const TL* lrow;
    const uint8_t* mrow;
    const TT* trow;
    __device__ __forceinline__ Part(const gk_policy_loss_t& p, int64_t r, int rank, int log_ranks)
        : RowPart<V>(r, p.logits_stride, (int)p.cols, rank, log_ranks) {
        lrow = static_cast<const TL*>(p.logits) + r * p.logits_stride;
        mrow = p.mask == nullptr ? nullptr : p.mask + r * p.mask_stride;
        trow = std::is_same<TT, None>::value ? nullptr : static_cast<const TT*>(p.target) + r * p.target_stride;
    }
};

__device__ __forceinline__ void copy_async(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
                 : "memory");
}

// Longer rows: a cluster of CTAs takes a row, each CTA a part of it; the parts
// meet through distributed shared memory. STAGED: a CTA's part of the logits
// lies in shared memory, so they are read from HBM once. Each thread copies the
// groups that it reads itself, so no barrier stands between a copy and its use,
// and a slot takes the next row's group as soon as this row's last pass has
// read it: the loads of one row run under the stores of the row before.
// Otherwise (a part past the shared memory, or rows that are not aligned) each
// pass reads the row itself, from L2 where it fits. Three CTAs of 256 threads an
// SM: one's barrier and loads hide under the passes of the others. Issue slots are
// 58% busy (some 17 instructions an entry over its passes, exponentials of 16-bit
// logits in pairs) and HBM runs at three quarters of a copy's rate: 4096 x 128000
// bf16 428 us, 4.9 TB/s; 8192 x 1000 23 us; 1024 x 32771 fp16 with target, which
// reads the target beside, 52 us; 7 x 100003, a few rows' latency, 6.7.
template <typename TL, typename TT, int V, bool STAGED, int THREADS>
__global__ void __launch_bounds__(THREADS, 3 * kLongThreads / THREADS) policy_loss_long_kernel(gk_policy_loss_t p,
                                                                                             int log_ranks) {
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = 1 << log_ranks, rank = log_ranks == 0 ? 0 : (int)cluster.block_rank();
    // Another CTA's shared memory may be written once that CTA runs: all arrive here, and wait for the others
    // under the first row's loads.
    bool all_run = ranks == 1;
    if (!all_run) cluster.barrier_arrive();
    constexpr bool kTarget = !std::is_same<TT, None>::value;
    constexpr int kWarps = THREADS / 32;
    extern __shared__ uint4 staged[];
    // What each warp of the cluster found (maximum, sum, target sum, target
    // term), by turns: written by every CTA, read after the cluster barrier.
    // A slot is written again two rows later, a barrier after its last read.
    __shared__ float4 found[2][kMaxCluster * kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t clusters = gridDim.x >> log_ranks;
    const float inv_n = inverse_denominator(p);
    const int cols = (int)p.cols;
    double sum = 0.0;
    int turn = 0;
    int64_t r = blockIdx.x >> log_ranks;
    Part<TL, TT, V> part(p, r, rank, log_ranks);
    if constexpr (STAGED) {
        const TL* from = part.lrow + (part.full * V - part.shift);
        for (int k = tid; k < part.full_end - part.full; k += THREADS) copy_async(staged + k, from + k * V);
    }
    while (r < p.rows) {
        const RowInput in = row_input(p, r, part.lrow, part.mrow);
        const int base = part.full * V - part.shift, count = part.full_end - part.full;
        // The row's first group where it is an edge is thread 0's, its last the last thread's.
        const bool head = V > 1 && tid == 0 && part.begin < part.full && part.begin < part.end;
        const bool tail = V > 1 && tid == THREADS - 1 && part.full_end < part.end && part.end - 1 >= part.full;
        const TL* from = STAGED ? reinterpret_cast<const TL*>(staged) : part.lrow + base;
        const uint8_t* mask = part.mrow == nullptr ? nullptr : part.mrow + base;
        // f(group, index of its first entry, whether it is an edge) for this thread's groups.
        auto edges = [&](auto&& f) {
            if (head || tail) {
                const int first = (head ? part.begin : part.end - 1) * V - part.shift;
                Group<TL, V> h;
                h.load_edge(part.lrow, part.mrow, first, cols);
                f(h, first, true);
            }
        };
        auto groups = [&](auto&& f) {
            if (part.mrow == nullptr) {
#pragma unroll 4
                for (int k = tid; k < count; k += THREADS) {
                    Group<TL, V> h;
                    h.template load<false>(from + k * V, nullptr);
                    f(h, base + k * V, false);
                }
            } else {
#pragma unroll 4
                for (int k = tid; k < count; k += THREADS) {
                    Group<TL, V> h;
                    h.template load<true>(from + k * V, mask + k * V);
                    f(h, base + k * V, false);
                }
            }
            edges(f);
        };
        if constexpr (STAGED) asm volatile("cp.async.wait_all;" ::: "memory");
        Softmax acc;
        float total_t = 0.0f, kl = 0.0f;
        groups([&](const Group<TL, V>& h, int, bool) { acc.m = fmaxf(acc.m, h.top()); });
#pragma unroll
        for (int o = 16; o; o >>= 1) acc.m = fmaxf(acc.m, __shfl_xor_sync(kFull, acc.m, o));
        {
            const Exp<TL> e(acc.m);
            uint64_t s2 = two(0.0f, 0.0f);
            groups([&](const Group<TL, V>& h, int first, bool edge) {
                if constexpr (V > 1 && sizeof(TL) == 2) {
#pragma unroll
                    for (int i = 0; i < V; i += 2) s2 = add2(s2, e.pair(h.x(i), h.x(i + 1)));
                } else {
#pragma unroll
                    for (int i = 0; i + 1 < V; i += 2) s2 = add2(s2, two(e.term(h.x(i)), e.term(h.x(i + 1))));
                    if constexpr (V == 1) acc.s += e.term(h.x(0));
                }
                if constexpr (kTarget) {
                    float t[V];
                    load_target<TT, V>(part.trow, h.legal, first, edge, t);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        total_t += t[i];
                        kl += target_term(t[i], h.x(i) - acc.m);
                    }
                }
            });
            float even, odd;
            halves(s2, even, odd);
            acc.s = warp_sum(acc.s + even + odd) * e.correct;
        }
        if (kTarget) {
            total_t = warp_sum(total_t);
            kl = warp_sum(kl);
        }
        const float4 mine = make_float4(acc.m, acc.s, total_t, kl);
        if (ranks > 1) {
            if (!all_run) cluster.barrier_wait();
            all_run = true;
            if (lane < ranks) cluster.map_shared_rank(found[turn], lane)[rank * kWarps + warp] = mine;
            cluster.sync();
        } else {
            if (lane == 0) found[turn][warp] = mine;
            __syncthreads();
        }
        // Every warp joins what all found and forms the row's terms for itself.
        const int all = ranks * kWarps;
        const float4 none = make_float4(-FLT_MAX, 0.0f, 0.0f, 0.0f);
        const float4 f0 = lane < all ? found[turn][lane] : none;
        const float4 f1 = kWarps * kMaxCluster > 32 && lane + 32 < all ? found[turn][lane + 32] : none;
        acc.m = f0.x, acc.s = f0.y;
        acc.join(f1.x, f1.y);
        acc.join_lanes(32);
        if (kTarget) {
            total_t = warp_sum(f0.z + f1.z);
            // A warp without mass has no distance to add (and no finite one, if all it saw was -inf).
            kl = warp_sum((f0.z == 0.0f ? f0.w : f0.w + f0.z * (acc.m - f0.x)) +
                          (f1.z == 0.0f ? f1.w : f1.w + f1.z * (acc.m - f1.x)));
        }
        const Row o = row_terms<true>(p, in, acc.m, acc.s, total_t);
        if (rank == 0 && tid == 0) {
            write_row(p, r, o);
            sum += (double)(o.loss + (kTarget && o.inv_s != 0.0f ? p.target_weight * (kl + total_t * o.log_s) : 0.0f));
        }
        // The next row of this CTA: its groups take the slots as the last pass empties them.
        const int64_t next_r = r + clusters;
        const Part<TL, TT, V> next(p, next_r < p.rows ? next_r : r, rank, log_ranks);
        const TL* next_from = next.lrow + (next.full * V - next.shift);
        const int next_count = STAGED && next_r < p.rows ? next.full_end - next.full : 0;
        TL* grow = static_cast<TL*>(p.grad) + r * p.cols;
        if (o.inv_s != 0.0f && p.grad != nullptr) {
            const Exp<TL> e(o.m);
            const float kt = inv_n * p.target_weight;
            const float kp = inv_n * (p.target_weight * o.total_t - o.c) * o.inv_s * e.correct;
            auto finish = [&](const Group<TL, V>& h, int first, bool edge) {
                float t[V], g[V];
                load_target<TT, V>(part.trow, h.legal, first, edge, t);
                gradient_group<TL, TT, V>(h, t, e, kp, kt, g);
                store_group<TL, V>(grow, first, cols, edge, g);
            };
            // The mask's presence is settled outside the loops, so that without one nothing is left of it inside.
            auto last_pass = [&](auto masked) {
                constexpr bool kMask = decltype(masked)::value;
                constexpr int U = 4;
                int k = tid;
                const int whole = next_count > 0 ? min(count, next_count) : count;
                for (; k + (U - 1) * THREADS < whole; k += U * THREADS) {
                    Group<TL, V> h[U];
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        h[u].template load<kMask>(from + (k + u * THREADS) * V, mask + (k + u * THREADS) * V);
#pragma unroll
                    for (int u = 0; u < U; ++u) finish(h[u], base + (k + u * THREADS) * V, false);
                    if (next_count > 0) {
#pragma unroll
                        for (int u = 0; u < U; ++u)
                            copy_async(staged + k + u * THREADS, next_from + (k + u * THREADS) * V);
                    }
                }
                for (; k < count; k += THREADS) {
                    Group<TL, V> h;
                    h.template load<kMask>(from + k * V, mask + k * V);
                    finish(h, base + k * V, false);
                    if (k < next_count) copy_async(staged + k, next_from + k * V);
                }
                fill_past<THREADS>(tid, count, next_count, [&](int q) { copy_async(staged + q, next_from + q * V); });
            };
            if (part.mrow == nullptr)
                last_pass(std::false_type());
            else
                last_pass(std::true_type());
            edges(finish);
            if (o.action >= 0) {
                // The action's own part: the thread that wrote its group writes it again.
                const int q = ((int)o.action + part.shift) / V;
                const bool first = q < part.full, last = q >= part.full_end;
                if (q >= part.begin && q < part.end &&
                    tid == (first ? 0 : (last ? THREADS - 1 : (q - part.full) % THREADS))) {
                    float t = 0.0f;
                    if constexpr (kTarget) t = to_f(part.trow[o.action]);
                    grow[o.action] = from_f<TL>(kp * e(to_f(part.lrow[o.action])) - kt * t + inv_n * o.c);
                }
            }
        } else {
            for (int k = tid; k < next_count; k += THREADS) copy_async(staged + k, next_from + k * V);
            if (p.grad != nullptr)
                for (int j = max(0, part.begin * V - part.shift) + tid; j < min(cols, part.end * V - part.shift);
                     j += THREADS)
                    grow[j] = from_f<TL>(0.0f);
        }
        part = next;
        r = next_r;
        turn ^= 1;
    }
    if (ranks > 1) cluster.sync();  // no CTA leaves while another writes to its shared memory
    if (rank == 0 && tid == 0) {
        if (clusters == 1)
            finish_loss(p, sum);
        else
            p.partials[blockIdx.x >> log_ranks] = sum;
    }
}

// The gradient from the saved row statistics, scaled by the upstream
// gradient. A gradient that the forward pass wrote is for an upstream of one,
// and is left as it is when that holds (`written`: 1.5 to 4 us for the blocks to
// see it). fp16 gradients are made here only, where the upstream gradient (a loss
// scale) is known: 1024 x 32771 with target 44 us, 4.5 TB/s.
template <typename TL, typename TT, int V>
__global__ void __launch_bounds__(256) policy_loss_backward_kernel(gk_policy_loss_t p, const float* upstream,
                                                                   int written) {
    const float up = *upstream;
    if (written && up == 1.0f) return;
    constexpr int kGroups = 4;  // groups a lane takes of a row's chunk
    const float scale = up * inverse_denominator(p);
    const int lane = threadIdx.x & 31, cols = (int)p.cols;
    const int64_t chunks = (p.cols + V - 1 + V * 32 * kGroups - 1) / (V * 32 * kGroups), items = p.rows * chunks;
    const int64_t warps = (int64_t)gridDim.x * 8;
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += warps) {
        const int64_t r = it / chunks;
        const int chunk = (int)(it - r * chunks);
        const Part<TL, TT, V> part(p, r, 0, 0);
        TL* grow = static_cast<TL*>(p.grad) + r * p.cols;
        const float4 st = reinterpret_cast<const float4*>(p.stats)[r];  // maximum, 1 / sum, c, target sum
        const int64_t action = p.actions == nullptr ? -1 : p.actions[r];
        const Exp<TL> e(st.x);
        const float kp = scale * (p.target_weight * st.w - st.z) * st.y * e.correct, kt = scale * p.target_weight;
#pragma unroll
        for (int k = 0; k < kGroups; ++k) {
            const int q = (chunk * kGroups + k) * 32 + lane;
            if (q >= part.end) break;
            const int first = q * V - part.shift;
            const bool edge = q < part.full || q >= part.full_end;
            float t[V], g[V];
            Group<TL, V> h;
            if (edge)
                h.load_edge(part.lrow, part.mrow, first, cols);
            else if (part.mrow == nullptr)
                h.template load<false>(part.lrow + first, nullptr);
            else
                h.template load<true>(part.lrow + first, part.mrow + first);
            load_target<TT, V>(part.trow, h.legal, first, edge, t);
            if (st.y != 0.0f) {
                gradient_group<TL, TT, V>(h, t, e, kp, kt, g);
                const int64_t at = action - first;
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (at == i) g[i] += scale * st.z;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) g[i] = 0.0f;
            }
            store_group<TL, V>(grow, first, cols, edge, g);
        }
    }
}

bool valid(const gk_policy_loss_t* p) {
    if (p == nullptr || p->rows < 0 || p->cols < 1 || p->cols > (1ll << 30)) return false;
    if (p->logits_type < GK_FP32 || p->logits_type > GK_FP16) return false;
    if (p->rows == 0) return p->loss != nullptr;
    if (p->logits == nullptr || p->stats == nullptr || p->partials == nullptr || p->loss == nullptr) return false;
    if (p->target != nullptr && p->target_type != GK_FP32 && p->target_type != p->logits_type) return false;
    if (p->actions == nullptr) {
        if (p->target == nullptr || p->reference_log_probs != nullptr) return false;
    } else if (p->old_log_probs == nullptr || p->advantages == nullptr) {
        return false;
    }
    return true;
}

bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Whether every operand's 16-byte groups fall on the logits' own groups in
// every row: aligned bases, and row lengths that leave the same remainder.
bool vectorised(const gk_policy_loss_t& p, int v) {
    auto same = [&](int64_t stride) { return (stride - p.logits_stride) % v == 0; };
    if (!aligned16(p.logits)) return false;
    if (p.mask != nullptr && !(aligned(p.mask, v) && same(p.mask_stride))) return false;
    if (p.target != nullptr && !(aligned16(p.target) && same(p.target_stride))) return false;
    if (p.grad != nullptr && !(aligned16(p.grad) && same(p.cols))) return false;
    return p.logits_stride >= 0;
}

// How a long row is split and staged. A CTA's part is at most 72 KB, three to
// an SM; the cluster grows until the part fits, and with fewer rows than the
// SMs hold until the grid fills them, but no part gets shorter than two vectors
// a thread. Parts of less take 64 threads, so that more rows are in flight.
struct LongPlan {
    int log_cluster, threads;
    bool staged;
    size_t smem;
};
constexpr int64_t kPartBytes = 72 << 10;
constexpr int kShortThreads = 64;

LongPlan long_plan(const gk_policy_loss_t& p, int v) {
    const int64_t groups = (p.cols + 2 * (v - 1)) / v;  // with the shift of an odd row
    int log = 0;
    auto part = [&](int k) { return (groups + (1 << k) - 1) >> k; };
    while ((1 << log) < kMaxCluster && (part(log) * 16 > kPartBytes || ((p.rows << (log + 1)) <= 3 * kSmCount &&
                                                                        part(log + 1) >= 2 * kLongThreads)))
        ++log;
    LongPlan plan{};
    plan.log_cluster = log;
    plan.staged = v > 1 && part(log) * 16 <= kPartBytes;
    plan.threads = plan.staged && part(log) < 2 * kLongThreads ? kShortThreads : kLongThreads;
    plan.smem = plan.staged ? (size_t)part(log) * 16 : 0;
    return plan;
}

int row_blocks(int64_t rows) { return blocks_for(rows, kRowWarps, kSmCount * 8); }

template <typename TL, typename TT, int V, bool STAGED, int THREADS>
int launch_long(const gk_policy_loss_t& p, const LongPlan& plan, int* clusters, cudaStream_t s) {
    auto* kernel = policy_loss_long_kernel<TL, TT, V, STAGED, THREADS>;
    static bool done[64] = {};
    static int resident[64][4] = {};  // clusters of 1, 2, 4, 8 CTAs that the device holds at once
    int dev = 0;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.blockDim = dim3(THREADS);
    cfg.stream = s;
    if (!once_per_device(done, [&] {
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPartBytes) != cudaSuccess ||
                cudaGetDevice(&dev) != cudaSuccess)
                return false;
            for (int i = 0; i < 4; ++i) {
                attr[0].val.clusterDim.x = 1 << i;
                cfg.gridDim = dim3(8);
                cfg.dynamicSmemBytes = !STAGED ? 0 : (THREADS == kLongThreads ? kPartBytes : 2 * kLongThreads * 16);
                if (cudaOccupancyMaxActiveClusters(&resident[dev][i], kernel, &cfg) != cudaSuccess) return false;
            }
            return true;
        }))
        return setup_failed();
    if (cudaGetDevice(&dev) != cudaSuccess) return setup_failed();
    // GPCs of an odd number of SMs leave some out of a cluster: a grid that is
    // resident at once has no second round for the rest.
    const int64_t most = resident[dev][plan.log_cluster] > 0 ? resident[dev][plan.log_cluster] : 1;
    *clusters = (int)(p.rows < most ? p.rows : most);
    attr[0].val.clusterDim.x = 1 << plan.log_cluster;
    cfg.gridDim = dim3((unsigned)(*clusters << plan.log_cluster));
    cfg.dynamicSmemBytes = plan.smem;
    return (int)cudaLaunchKernelEx(&cfg, kernel, p, plan.log_cluster);
}

template <typename TL, typename TT>
int forward(const gk_policy_loss_t& p, cudaStream_t s) {
    int parts;
    if (p.cols <= kShortRow) {
        parts = row_blocks(p.rows);
        if (p.cols <= 96)
            policy_loss_rows_kernel<TL, TT, 3><<<parts, kRowWarps * 32, 0, s>>>(p);
        else
            policy_loss_rows_kernel<TL, TT, 8><<<parts, kRowWarps * 32, 0, s>>>(p);
    } else {
        constexpr int V = kVec<TL>;
        const bool vec = vectorised(p, V);
        const LongPlan plan = long_plan(p, vec ? V : 1);
        int e;
        if (!vec)
            e = launch_long<TL, TT, 1, false, kLongThreads>(p, plan, &parts, s);
        else if (!plan.staged)
            e = launch_long<TL, TT, V, false, kLongThreads>(p, plan, &parts, s);
        else if (plan.threads == kLongThreads)
            e = launch_long<TL, TT, V, true, kLongThreads>(p, plan, &parts, s);
        else
            e = launch_long<TL, TT, V, true, kShortThreads>(p, plan, &parts, s);
        if (e != 0) return e;
    }
    if (parts > 1) policy_loss_sum_kernel<<<1, 256, 0, s>>>(p, parts);
    return launch_status();
}

template <typename TL, typename TT>
int backward(const gk_policy_loss_t& p, const float* upstream, int written, cudaStream_t s) {
    const bool vec = p.cols > kShortRow && vectorised(p, kVec<TL>);
    const int64_t per = (int64_t)(vec ? kVec<TL> : 1) * 32 * 4;
    const int64_t chunks = (p.cols + (vec ? kVec<TL> : 1) - 1 + per - 1) / per;
    const int grid = blocks_for(p.rows * chunks, 8, kSmCount * 32);
    if (vec)
        policy_loss_backward_kernel<TL, TT, kVec<TL>><<<grid, 256, 0, s>>>(p, upstream, written);
    else
        policy_loss_backward_kernel<TL, TT, 1><<<grid, 256, 0, s>>>(p, upstream, written);
    return launch_status();
}

template <typename F>
int by_type(const gk_policy_loss_t& p, F&& f) {
    const bool same = p.target != nullptr && p.target_type == p.logits_type;
    if (p.logits_type == GK_FP32)
        return p.target == nullptr ? f((float*)0, (None*)0) : f((float*)0, (float*)0);
    if (p.logits_type == GK_BF16)
        return p.target == nullptr ? f((__nv_bfloat16*)0, (None*)0)
                                   : (same ? f((__nv_bfloat16*)0, (__nv_bfloat16*)0) : f((__nv_bfloat16*)0, (float*)0));
    return p.target == nullptr ? f((__half*)0, (None*)0)
                               : (same ? f((__half*)0, (__half*)0) : f((__half*)0, (float*)0));
}

}  // namespace
}  // namespace gk

extern "C" {

int gk_policy_loss_parts(int64_t rows, int64_t cols) {
    if (rows < 1 || cols < 1) return 0;
    if (cols <= gk::kShortRow) return gk::row_blocks(rows);
    const int64_t most = gk::kSmCount * 32;  // clusters of any plan: the CTAs that the SMs hold at most
    return (int)(rows < most ? rows : most);
}

int gk_policy_loss_forward(const gk_policy_loss_t* p, void* stream) {
    using namespace gk;
    if (!valid(p)) return GK_EINVAL;
    cudaStream_t s = as_stream(stream);
    if (p->rows == 0) {
        const cudaError_t e = cudaMemsetAsync(p->loss, 0, sizeof(float), s);
        return (int)e;
    }
    return by_type(*p, [&](auto* l, auto* t) {
        return forward<std::remove_pointer_t<decltype(l)>, std::remove_pointer_t<decltype(t)>>(*p, s);
    });
}

int gk_policy_loss_backward(const gk_policy_loss_t* p, const float* upstream, int written, void* stream) {
    using namespace gk;
    if (!valid(p) || upstream == nullptr) return GK_EINVAL;
    if (p->rows == 0) return 0;
    if (p->grad == nullptr) return GK_EINVAL;
    return by_type(*p, [&](auto* l, auto* t) {
        return backward<std::remove_pointer_t<decltype(l)>, std::remove_pointer_t<decltype(t)>>(
            *p, upstream, written, as_stream(stream));
    });
}

}  // extern "C"
