// gk_linear.cu - the linear operator y = act(x W^T + b + r) and its gradients.
//
//   dz = dy act'(z),  dr = dz,  db = sum_m dz,  dx = dz W,  dW = dz^T x
//
// 16-bit types run their three products on tcgen05 (gk_gemm.cu). fp32 runs on
// the fp32 units: its callers train the network's heads in fp32, and one tf32
// or bf16 product would lose the bits that they keep fp32 for. A product with
// at most eight rows reads each weight once and is bound by that: it runs as
// dot products on the cores, but for weights so wide that tcgen05 streams them
// faster (few_rows_win).
#include <cooperative_groups.h>

#include <type_traits>

#include "../../include/gk.h"
#include "gk_act.cuh"
#include "gk_gemm.cuh"
#include "gk_launch.cuh"

namespace gk {
namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kFewRows = 8;

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// ------------------------------------------------------------ few rows

struct FewRows {
    const void* x;
    const void* w;
    const void* bias;
    const void* residual;
    void* y;
    void* pre;
    int64_t x_stride, w_stride, residual_stride, pre_stride;
    int m, n;
    int64_t k;
    int activation;
    int k_parts;  // warps that share an output along k: 1, 2, 4 or 8
};

// A warp (or k_parts of them) takes R rows of W; its lanes run along k, 16
// bytes of each row at a time where V > 1, and every value of W meets the M
// rows of x (held by L1) in registers. Bound by the bytes of W for one row (4096
// -> 12288 bf16 19 us, 5.3 TB/s; 32000: 5.6 TB/s), then by the loads of x.
// Steps unrolled, measured: 16 bytes at a time 2 for one row (1: 29 us, 4: 25)
// and 1 for more (8 rows of 4096 -> 12288: 43, unrolled 55 us); single values 4
// (4097 -> 12288, one row: 32 us, by 2 152 us).
template <int M, int V>
constexpr int kFewUnroll = V == 1 ? 4 : M == 1 ? 2 : 1;
template <typename T, int M, int R, int V>
__global__ void __launch_bounds__(256) linear_few_kernel(FewRows p) {
    __shared__ float parts[8][R * M];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int teams = 8 / p.k_parts, team = warp / p.k_parts, part = warp % p.k_parts;
    const int64_t n0 = ((int64_t)blockIdx.x * teams + team) * R;
    const T* x = static_cast<const T*>(p.x);
    const T* w = static_cast<const T*>(p.w);
    float acc[R][M];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < M; ++m) acc[r][m] = 0.0f;
    const T* wr[R];
#pragma unroll
    for (int r = 0; r < R; ++r) wr[r] = w + (n0 + r < p.n ? n0 + r : p.n - 1) * p.w_stride;
    const T* xr[M];  // a row that is not there repeats the last: no branch stands between the loads
#pragma unroll
    for (int m = 0; m < M; ++m) xr[m] = x + (m < p.m ? m : p.m - 1) * p.x_stride;
    const int64_t step = (int64_t)32 * V * p.k_parts;
#pragma unroll kFewUnroll<M, V>
    for (int64_t k = ((int64_t)part * 32 + lane) * V; k < p.k; k += step) {
        alignas(16) T wv[R][V];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if constexpr (V > 1)
                *reinterpret_cast<uint4*>(wv[r]) = __ldcs(reinterpret_cast<const uint4*>(wr[r] + k));
            else
                wv[r][0] = __ldg(wr[r] + k);
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
            // Never taken; with one row it keeps the loads of W together (4096 x 12288: 20.8 -> 19.0 us).
            if (M == 1 && p.m < 1) break;
            alignas(16) T xv[V];
            if constexpr (V > 1)
                *reinterpret_cast<uint4*>(xv) = __ldg(reinterpret_cast<const uint4*>(xr[m] + k));
            else
                xv[0] = __ldg(xr[m] + k);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < V; ++i) acc[r][m] = fmaf(as_float<T>(wv[r][i]), as_float<T>(xv[i]), acc[r][m]);
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int m = 0; m < M; ++m) {
            float v = acc[r][m];
#pragma unroll
            for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
            if (lane == 0) parts[warp][r * M + m] = v;
        }
    __syncthreads();
    for (int i = threadIdx.x; i < teams * R * M; i += 256) {
        const int t = i / (R * M), r = (i / M) % R, m = i % M;
        const int64_t n = ((int64_t)blockIdx.x * teams + t) * R + r;
        if (n >= p.n || m >= p.m) continue;
        float v = 0.0f;
        for (int q = 0; q < p.k_parts; ++q) v += parts[t * p.k_parts + q][r * M + m];
        if (p.bias != nullptr) v += as_float<T>(static_cast<const T*>(p.bias)[n]);
        if (p.residual != nullptr) v += as_float<T>(static_cast<const T*>(p.residual)[m * p.residual_stride + n]);
        const float y = act_value<sizeof(T) == 2>(v, p.activation);
        if (p.pre != nullptr) {
            if (p.activation == GK_ACT_TANH)
                static_cast<float*>(p.pre)[m * p.pre_stride + n] = y;
            else
                static_cast<T*>(p.pre)[m * p.pre_stride + n] = rounded<T>(v);
        }
        static_cast<T*>(p.y)[(int64_t)m * p.n + n] = rounded<T>(y);
    }
}

template <typename T>
bool rows_aligned(const void* p, int64_t stride) {
    return aligned16(p) && stride % kVec<T> == 0;
}

template <typename T, int M>
int few_rows(FewRows p, cudaStream_t s) {
    const bool vec = p.k % kVec<T> == 0 && rows_aligned<T>(p.x, p.x_stride) && rows_aligned<T>(p.w, p.w_stride);
    // Four rows of W a warp, for the loads in flight and the reuse of x; fewer
    // outputs than that keeps busy are split along k over the block's warps.
    const int64_t warps = (p.n + 3) / 4;
    p.k_parts = 1;
    while (p.k_parts < 8 && warps * p.k_parts < 16 * kSmCount && p.k >= (int64_t)p.k_parts * 2 * 32 * kVec<T>)
        p.k_parts *= 2;
    const int64_t per_block = 4 * (8 / p.k_parts);
    const unsigned grid = (unsigned)((p.n + per_block - 1) / per_block);
    if (vec)
        linear_few_kernel<T, M, 4, kVec<T>><<<grid, 256, 0, s>>>(p);
    else
        linear_few_kernel<T, M, 4, 1><<<grid, 256, 0, s>>>(p);
    return launch_status();
}

// ------------------------------------------------------------ fp32 products

struct Gemm32 {
    const float* a;
    const void* b;       // of the kernel's type E, like out
    int64_t a_ld, b_ld;  // elements between rows of A and B, or between their k where m or n is contiguous
    void* out;
    const float* bias;
    const float* residual;
    float* pre;
    int64_t out_ld, residual_ld, pre_ld;
    int64_t m, n, k;
    int activation;
    int wide;  // rows of out and pre start on 16 bytes
};

// A tile of B x B outputs, P x P to a thread, k in steps of 16 through two
// shared-memory buffers with the next step's loads in registers. The products
// are packed pairs (two fp32 multiply-adds an instruction, each rounded like
// one of its own). With few tiles a cluster of CTAs shares one along k and adds
// the parts up in rank order through distributed shared memory. Bound by the
// fp32 units where it is large (2048^3 388 us, 44 TFLOP/s) and by the latency of
// its steps where it is small (4096 x 162 -> 82 and its gradients 11 to 15 us each;
// steps of 32 or 64 k gained up to 10% there and lost as much elsewhere).
constexpr int kStep = 16;
template <int B, int P>
struct Tile32 {
    static constexpr int kThreads = (B / P) * (B / P), kPitch = B + 4;
    static constexpr int kSmem = (B * kPitch > 4 * kStep * kPitch ? B * kPitch : 4 * kStep * kPitch) * 4;
    static constexpr int kQuads = B * kStep / 4 / kThreads;  // groups of four elements a thread loads of an operand
};

// One operand's B x 16 step, four neighbours at a time along its contiguous
// dimension: k (K) or the row. VEC: those four are one aligned load. 16-bit
// elements (E) become fp32 as they arrive.
template <typename E, int B, int P, bool K, bool VEC>
struct Loader32 {
    using T = Tile32<B, P>;
    float v[T::kQuads][4];
    const E* at[T::kQuads];  // this thread's first element of each group, now
    int left;                    // rows of the tile
    int64_t step;
    __device__ __forceinline__ static void place(int t, int i, int& row, int& k) {
        const int q = t + i * T::kThreads;
        if (K)
            k = (q % (kStep / 4)) * 4, row = q / (kStep / 4);
        else
            row = (q % (B / 4)) * 4, k = q / (B / 4);
    }
    __device__ __forceinline__ void start(const E* p, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int t) {
        step = K ? kStep : kStep * ld;
        left = rows - row0 < B ? (int)(rows - row0) : B;
#pragma unroll
        for (int i = 0; i < T::kQuads; ++i) {
            int row, k;
            place(t, i, row, k);
            at[i] = K ? p + (row0 + row) * ld + k0 + k : p + (k0 + k) * ld + row0 + row;
        }
    }
    // `k_left`: k elements left from the step's start.
    __device__ __forceinline__ void fetch(int64_t k_left, int t) {
        if (left == B && k_left >= kStep) {
#pragma unroll
            for (int i = 0; i < T::kQuads; ++i) {
                if constexpr (VEC && sizeof(E) == 4) {
                    *reinterpret_cast<float4*>(v[i]) = __ldg(reinterpret_cast<const float4*>(at[i]));
                } else if constexpr (VEC) {
                    alignas(8) E four[4];
                    *reinterpret_cast<uint2*>(four) = __ldg(reinterpret_cast<const uint2*>(at[i]));
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i][j] = as_float<E>(four[j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) v[i][j] = as_float<E>(__ldg(at[i] + j));
                }
                at[i] += step;
            }
            return;
        }
        const int k_end = k_left < kStep ? (int)k_left : kStep;
#pragma unroll
        for (int i = 0; i < T::kQuads; ++i) {
            int row, k;
            place(t, i, row, k);
            const int count = K ? (row < left ? k_end - k : 0) : (k < k_end ? left - row : 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[i][j] = j < count ? as_float<E>(__ldg(at[i] + j)) : 0.0f;
            at[i] += step;
        }
    }
    __device__ __forceinline__ void store(float (*tile)[T::kPitch], int t) const {
#pragma unroll
        for (int i = 0; i < T::kQuads; ++i) {
            int row, k;
            place(t, i, row, k);
            if (K) {
#pragma unroll
                for (int j = 0; j < 4; ++j) tile[k + j][row] = v[i][j];
            } else {
                *reinterpret_cast<float4*>(&tile[k][row]) = *reinterpret_cast<const float4*>(v[i]);
            }
        }
    }
};

__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ void multiply_add(uint64_t& acc, uint64_t a, uint64_t b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}

// Bias, residual, activation and stores of four neighbours of a row.
__device__ __forceinline__ void finish4_fp32(const Gemm32& g, int64_t m, int64_t n, float (&v)[4]) {
    const bool whole = g.wide && n + 4 <= g.n;
    const int count = g.n - n < 4 ? (int)(g.n - n) : 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (j < count) {
            if (g.bias != nullptr) v[j] += __ldg(g.bias + n + j);
            if (g.residual != nullptr) v[j] += __ldg(g.residual + m * g.residual_ld + n + j);
        }
    }
    float* pre = g.pre == nullptr ? nullptr : g.pre + m * g.pre_ld + n;
    float* out = static_cast<float*>(g.out) + m * g.out_ld + n;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = g.activation == GK_ACT_NONE ? v[j] : act_value<false>(v[j], g.activation);
    if (g.activation == GK_ACT_TANH) {  // keeps its value, not the sum
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = y[j];
    }
    if (whole) {
        if (pre != nullptr) *reinterpret_cast<float4*>(pre) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(out) = make_float4(y[0], y[1], y[2], y[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j >= count) break;
            if (pre != nullptr) pre[j] = v[j];
            out[j] = y[j];
        }
    }
}

// 16-bit results are gradients and have nothing but the rounding.
template <typename E>
__device__ __forceinline__ void finish4(const Gemm32& g, int64_t m, int64_t n, float (&v)[4]) {
    if constexpr (sizeof(E) == 4) {
        finish4_fp32(g, m, n, v);
    } else {
        E* out = static_cast<E*>(g.out) + m * g.out_ld + n;
        alignas(8) E four[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) four[j] = rounded<E>(v[j]);
        if (g.wide && n + 4 <= g.n) {
            *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(four);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < g.n) out[j] = four[j];
        }
    }
}

template <typename E, int B, int P, bool AK, bool BK, bool VEC>
__global__ void __launch_bounds__(Tile32<B, P>::kThreads, P == 8 ? 512 / Tile32<B, P>::kThreads : 1)
    gemm32_kernel(Gemm32 g, int tiles_n) {
    extern __shared__ float smem[];
    using T = Tile32<B, P>;
    constexpr int kSide = B / P, kPitch = T::kPitch, kParts = P / 4;
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = cluster.num_blocks(), rank = cluster.block_rank();
    float(*as)[kPitch] = reinterpret_cast<float(*)[kPitch]>(smem);                      // [2 * kStep]
    float(*bs)[kPitch] = reinterpret_cast<float(*)[kPitch]>(smem + 2 * kStep * kPitch);  // [2 * kStep]
    const int t = threadIdx.x, tx = t % kSide, ty = t / kSide;
    const int64_t tile_m = blockIdx.x / tiles_n, tile_n = blockIdx.x - tile_m * tiles_n;
    const int64_t m0 = tile_m * B, n0 = tile_n * B;
    const int64_t steps = (g.k + kStep - 1) / kStep;
    const int64_t s0 = steps * rank / ranks, s1 = steps * (rank + 1) / ranks;
    uint64_t acc[P][P / 2];
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int j = 0; j < P / 2; ++j) acc[i][j] = 0ull;
    Loader32<float, B, P, AK, VEC> la;
    Loader32<E, B, P, BK, VEC> lb;
    la.start(g.a, g.a_ld, m0, g.m, s0 * kStep, t);
    lb.start(static_cast<const E*>(g.b), g.b_ld, n0, g.n, s0 * kStep, t);
    la.fetch(g.k - s0 * kStep, t);
    lb.fetch(g.k - s0 * kStep, t);
    for (int64_t s = s0; s < s1; ++s) {
        const int buf = (int)((s - s0) & 1) * kStep;
        la.store(as + buf, t);
        lb.store(bs + buf, t);
        __syncthreads();
        if (s + 1 < s1) {
            la.fetch(g.k - (s + 1) * kStep, t);
            lb.fetch(g.k - (s + 1) * kStep, t);
        }
#pragma unroll
        for (int k = 0; k < kStep; ++k) {
            float a[P];
            uint64_t b[P / 2];
#pragma unroll
            for (int q = 0; q < kParts; ++q) {
                *reinterpret_cast<float4*>(a + 4 * q) =
                    *reinterpret_cast<float4*>(&as[buf + k][B / kParts * q + ty * 4]);
                *reinterpret_cast<ulonglong2*>(b + 2 * q) =
                    *reinterpret_cast<ulonglong2*>(&bs[buf + k][B / kParts * q + tx * 4]);
            }
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const uint64_t twice = pair_of(a[i], a[i]);
#pragma unroll
                for (int j = 0; j < P / 2; ++j) multiply_add(acc[i][j], twice, b[j]);
            }
        }
    }
    if (ranks == 1) {  // straight from the registers
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int64_t m = m0 + B / kParts * (i / 4) + ty * 4 + i % 4;
            if (m >= g.m) continue;
#pragma unroll
            for (int q = 0; q < kParts; ++q) {
                float v[4];
                *reinterpret_cast<ulonglong2*>(v) = make_ulonglong2(acc[i][2 * q], acc[i][2 * q + 1]);
                finish4<E>(g, m, n0 + B / kParts * q + tx * 4, v);
            }
        }
        return;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
        for (int q = 0; q < kParts; ++q)
            *reinterpret_cast<ulonglong2*>(smem + (B / kParts * (i / 4) + ty * 4 + i % 4) * kPitch + B / kParts * q +
                                           tx * 4) = make_ulonglong2(acc[i][2 * q], acc[i][2 * q + 1]);
    cluster.sync();
    const int quads = B / ranks * (B / 4), first = rank * (B / ranks);
    for (int i = t; i < quads; i += T::kThreads) {
        const int r = first + i / (B / 4), c = i % (B / 4) * 4;
        if (m0 + r >= g.m || n0 + c >= g.n) continue;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < ranks; ++k) {
            const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(smem, k) + r * kPitch + c);
            v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        }
        finish4<E>(g, m0 + r, n0 + c, v);
    }
    cluster.sync();  // no CTA leaves while another reads its part
}

template <typename E, int B, int P, bool AK, bool BK, bool VEC>
int launch_gemm32(const Gemm32& g, cudaStream_t s) {
    using T = Tile32<B, P>;
    auto* kernel = gemm32_kernel<E, B, P, AK, BK, VEC>;
    static bool ready[64] = {};
    if (!once_per_device(ready, [&] {
            return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem) == cudaSuccess &&
                   cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
        }))
        return setup_failed();
    const int64_t tiles_n = (g.n + B - 1) / B, tiles = (g.m + B - 1) / B * tiles_n;
    if (tiles >= (1ll << 31)) return GK_EINVAL;
    const int64_t steps = (g.k + kStep - 1) / kStep;
    // Parts of three steps or more, until there are 512 threads an SM.
    const int64_t most = 512 / T::kThreads * kSmCount;
    int ranks = 1;
    while (ranks < 16 && tiles * ranks * 2 <= most && steps >= ranks * 2 * 3) ranks *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tiles, 1, (unsigned)ranks);
    cfg.blockDim = dim3(T::kThreads);
    cfg.dynamicSmemBytes = T::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = ranks;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, g, (int)tiles_n);
}

template <bool AK, bool BK, bool VEC>
int gemm32(const Gemm32& g, cudaStream_t s) {
    // Measured (us, 128 x 128 | 64 x 64 | 32 x 32 tiles): 2048^3 388 | 467 | 601,
    // 1024^3 55 | 68 | 83, 512 x 4096 x 512 83 | 68 | 91, 300 x 700 x 900
    // 25 | 24 | 25, 4096 x 162 x 82 20 | 19 | 13, 9 x 4000 x 4000 94 | 67 | 48
    // (m x k x n). Large tiles reuse more of what they read; small ones keep the
    // SMs busy on little work and waste less of a ragged edge.
    auto tiles = [&](int64_t b) { return ((g.m + b - 1) / b) * ((g.n + b - 1) / b); };
    const double work = (double)g.m * (double)g.n * (double)g.k;
    const double area128 = 16384.0 * tiles(128), area64 = 4096.0 * tiles(64), area32 = 1024.0 * tiles(32);
    if (work < 134217728.0 || area64 >= 1.5 * area32) return launch_gemm32<float, 32, 4, AK, BK, VEC>(g, s);
    if (tiles(128) >= 32 && area128 <= 1.1 * area64) return launch_gemm32<float, 128, 8, AK, BK, VEC>(g, s);
    return launch_gemm32<float, 64, 8, AK, BK, VEC>(g, s);
}
template <bool AK, bool BK>
int gemm32(Gemm32 g, cudaStream_t s) {
    g.wide = aligned16(g.out) && g.out_ld % 4 == 0 &&
             (g.pre == nullptr || (aligned16(g.pre) && g.pre_ld % 4 == 0));
    const bool vec = aligned16(g.a) && aligned16(g.b) && g.a_ld % 4 == 0 && g.b_ld % 4 == 0;
    return vec ? gemm32<AK, BK, true>(g, s) : gemm32<AK, BK, false>(g, s);
}

// A small product of 16-bit gradients with dz in fp32.
template <typename E, bool AK>
int gemm32_narrow(Gemm32 g, cudaStream_t s) {
    g.wide = aligned16(g.out) && g.out_ld % 4 == 0;
    const bool vec = aligned16(g.a) && aligned16(g.b) && g.a_ld % 4 == 0 && g.b_ld % 4 == 0;
    return vec ? launch_gemm32<E, 32, 4, AK, false, true>(g, s) : launch_gemm32<E, 32, 4, AK, false, false>(g, s);
}

// ------------------------------------------------------------ dz and db

struct Slope {
    const void* dy;
    const void* kept;  // [m, n]; unused without activation
    void* dz;          // or nullptr
    float* dz32;       // dz before its rounding, or nullptr
    float* sums;       // [slabs, n] column sums of each slab of rows, or nullptr
    int64_t dy_stride, kept_stride, dz_stride, dz32_stride;
    int64_t m, n, slab;  // rows of a slab
    int activation;
};

// A warp goes down a slab of rows along 32 V columns; `across` of a block's
// eight warps lie side by side (whole lines of a row next to one another), the
// others take rows in turn. Bound by bytes where the slope is cheap (relu, 8192 x
// 4096 bf16 33 us, 6.1 TB/s) and by instructions for gelu and silu, which take two
// values an instruction where they can (gelu of 8192 x 8192 bf16 92 us, 4.4 TB/s;
// one by one 105).
template <int ACT>
constexpr bool kBends = ACT == GK_ACT_TANH || ACT == GK_ACT_GELU || ACT == GK_ACT_SILU;  // dz has more bits than dy
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(256, 4) linear_slope_kernel(Slope p, int across) {
    constexpr bool kSlope = ACT != GK_ACT_NONE;
    using K = typename std::conditional<ACT == GK_ACT_TANH, float, T>::type;  // tanh keeps fp32
    __shared__ float sums[8][32 * V];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int side = warp % across, down = warp / across, step = 8 / across;
    const int64_t first = (int64_t)blockIdx.x * 32 * V * across;
    const int64_t c = first + (side * 32 + lane) * V, r0 = (int64_t)blockIdx.y * p.slab;
    const int64_t r1 = r0 + p.slab < p.m ? r0 + p.slab : p.m;
    float sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
    if (c < p.n) {
        const T* dyp = static_cast<const T*>(p.dy) + c;
        const K* keptp = static_cast<const K*>(p.kept) + c;
        T* dzp = static_cast<T*>(p.dz) + c;
        constexpr int U = 2;  // rows in flight
        for (int64_t r = r0 + down; r < r1; r += U * step) {
            alignas(16) T dy[U][V];
            alignas(16) K kept[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = r + u * step;
                if (row >= r1) continue;
                if constexpr (V > 1) {
                    *reinterpret_cast<uint4*>(dy[u]) = __ldcs(reinterpret_cast<const uint4*>(dyp + row * p.dy_stride));
                    if constexpr (kSlope) {
#pragma unroll
                        for (int i = 0; i < (int)(V * sizeof(K) / 16); ++i)
                            reinterpret_cast<uint4*>(kept[u])[i] =
                                __ldcs(reinterpret_cast<const uint4*>(keptp + row * p.kept_stride) + i);
                    }
                } else {
                    dy[u][0] = dyp[row * p.dy_stride];
                    if constexpr (kSlope) kept[u][0] = keptp[row * p.kept_stride];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = r + u * step;
                if (row >= r1) continue;
                alignas(16) float z[V];
                if constexpr (V > 1 && sizeof(T) == 2) {  // two values an instruction where there is one
                    constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
                    uint32_t* words = reinterpret_cast<uint32_t*>(dy[u]);
#pragma unroll
                    for (int i = 0; i < V; i += 2) {
                        float up[2], slope[2];
                        unpack16(words[i / 2], bf16, up[0], up[1]);
                        uint64_t v = two(up[0], up[1]);
                        if constexpr (kSlope) {
                            slope[0] = as_float<K>(kept[u][i]), slope[1] = as_float<K>(kept[u][i + 1]);
                            if constexpr (ACT == GK_ACT_GELU) {
                                quick_gelu_slopes(slope[0], slope[1]);
                            } else {
                                slope[0] = act_slope<true>(slope[0], ACT);
                                slope[1] = act_slope<true>(slope[1], ACT);
                            }
                            v = mul2(v, two(slope[0], slope[1]));
                        }
                        halves(v, z[i], z[i + 1]);
                        halves(add2(two(sum[i], sum[i + 1]), v), sum[i], sum[i + 1]);
                        if constexpr (kSlope) words[i / 2] = pack16(z[i], z[i + 1], bf16);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        z[i] = as_float<T>(dy[u][i]);
                        if constexpr (kSlope) {
                            z[i] *= act_slope<sizeof(T) == 2>(as_float<K>(kept[u][i]), ACT);
                            dy[u][i] = rounded<T>(z[i]);
                        }
                        sum[i] += z[i];
                    }
                }
                if constexpr (kBends<ACT> && sizeof(T) == 2) {
                    if (p.dz32 != nullptr) {
                        float* at = p.dz32 + row * p.dz32_stride + c;
                        if constexpr (V > 1) {
#pragma unroll
                            for (int i = 0; i < V; i += 4)
                                *reinterpret_cast<float4*>(at + i) = make_float4(z[i], z[i + 1], z[i + 2], z[i + 3]);
                        } else {
                            at[0] = z[0];
                        }
                    }
                }
                if (p.dz != nullptr) {
                    if constexpr (V > 1)
                        *reinterpret_cast<uint4*>(dzp + row * p.dz_stride) = *reinterpret_cast<uint4*>(dy[u]);
                    else
                        dzp[row * p.dz_stride] = dy[u][0];
                }
            }
        }
    }
    if (p.sums == nullptr) return;
#pragma unroll
    for (int i = 0; i < V; ++i) sums[warp][lane * V + i] = sum[i];
    __syncthreads();
    for (int i = threadIdx.x; i < 32 * V * across; i += 256) {
        const int64_t col = first + i;
        if (col >= p.n) break;
        float v = 0.0f;
        for (int w = 0; w < step; ++w) v += sums[w * across + i / (32 * V)][i % (32 * V)];
        p.sums[(int64_t)blockIdx.y * p.n + col] = v;
    }
}

// db from the slabs' sums: 32 columns a block, eight warps each add every
// eighth slab, then in order.
template <typename T>
__global__ void __launch_bounds__(256) linear_bias_kernel(const float* sums, int64_t n, int slabs, T* db) {
    __shared__ float part[8][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    float v = 0.0f;
    if (c < n) {
#pragma unroll 4
        for (int s = warp; s < slabs; s += 8) v += sums[(int64_t)s * n + c];
    }
    part[warp][lane] = v;
    __syncthreads();
    if (warp == 0 && c < n) {
#pragma unroll
        for (int w = 1; w < 8; ++w) v += part[w][lane];
        db[c] = rounded<T>(v);
    }
}

struct SlopePlan {
    int vec, slabs, across;
    int64_t slab, col_blocks;
};
template <typename T>
SlopePlan slope_plan(int64_t m, int64_t n, bool vec) {
    SlopePlan p{};
    p.vec = vec ? kVec<T> : 1;
    p.across = 1;
    while (p.across < 8 && (int64_t)p.across * 32 * p.vec < n) p.across *= 2;
    p.col_blocks = (n + 32 * p.vec * p.across - 1) / (32 * p.vec * p.across);
    // One round of the four blocks that an SM holds, in slabs of 16 rows or more.
    int64_t slabs = 4 * kSmCount / p.col_blocks;
    if (slabs > (m + 15) / 16) slabs = (m + 15) / 16;
    if (slabs < 1) slabs = 1;
    p.slab = (m + slabs - 1) / slabs;
    p.slabs = (int)((m + p.slab - 1) / p.slab);
    return p;
}

template <typename T, int ACT>
void launch_slope(const Slope& a, dim3 grid, const SlopePlan& plan, cudaStream_t s) {
    if (plan.vec > 1)
        linear_slope_kernel<T, kVec<T>, ACT><<<grid, 256, 0, s>>>(a, plan.across);
    else
        linear_slope_kernel<T, 1, ACT><<<grid, 256, 0, s>>>(a, plan.across);
}
template <typename T>
int launch_slope(const Slope& a, dim3 grid, const SlopePlan& plan, cudaStream_t s) {
    switch (a.activation) {
        case GK_ACT_RELU: launch_slope<T, GK_ACT_RELU>(a, grid, plan, s); break;
        case GK_ACT_TANH: launch_slope<T, GK_ACT_TANH>(a, grid, plan, s); break;
        case GK_ACT_GELU: launch_slope<T, GK_ACT_GELU>(a, grid, plan, s); break;
        case GK_ACT_SILU: launch_slope<T, GK_ACT_SILU>(a, grid, plan, s); break;
        default: launch_slope<T, GK_ACT_NONE>(a, grid, plan, s); break;
    }
    return launch_status();
}

// Rows of a 16-bit matrix to rows that start on 16 bytes, as TMA needs them.
__global__ void __launch_bounds__(256) align_rows_kernel(const uint16_t* from, int64_t stride, int64_t rows,
                                                         int64_t cols, uint16_t* to, int64_t to_stride) {
    // A thread makes one 16-byte chunk; its eight loads are in flight together.
    const int64_t chunks = to_stride / 8, items = rows * chunks;
    for (int64_t it = (int64_t)blockIdx.x * 256 + threadIdx.x; it < items; it += (int64_t)gridDim.x * 256) {
        const int64_t r = it / chunks, c = (it - r * chunks) * 8;
        alignas(16) uint16_t v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? __ldg(from + r * stride + c + i) : (uint16_t)0;
        *reinterpret_cast<uint4*>(to + r * to_stride + c) = *reinterpret_cast<uint4*>(v);
    }
}

// ------------------------------------------------------------ workspaces

int64_t pad8(int64_t n) { return (n + 7) & ~(int64_t)7; }

struct Arena {
    uint8_t* base;
    size_t used = 0;
    explicit Arena(void* p) : base(static_cast<uint8_t*>(p)) {}
    void* take(int64_t bytes) {
        void* p = base == nullptr ? nullptr : base + used;
        used += ((size_t)bytes + 255) & ~(size_t)255;
        return p;
    }
};

bool sizes_ok(int64_t m, int64_t n, int64_t k, int dtype, int activation) {
    const int64_t most = (1ll << 31) - 1;
    return m >= 0 && n >= 1 && k >= 1 && m <= most && n <= most && k <= most && dtype >= GK_FP32 &&
           dtype <= GK_FP16 && activation >= GK_ACT_NONE && activation <= GK_ACT_SILU;
}

bool tma_rows(const void* p, int64_t stride, int64_t cols) {
    return aligned16(p) && stride % 8 == 0 && stride >= cols;
}

// The matrix itself if TMA can read its rows, else an aligned copy in the arena.
struct Operand {
    const void* p;
    int64_t ld;
    bool copied;
};
Operand operand(Arena& arena, const void* p, int64_t stride, int64_t rows, int64_t cols) {
    if (tma_rows(p, stride, cols)) return {p, stride, false};
    return {arena.take(rows * pad8(cols) * 2), pad8(cols), true};
}
int copy_if_needed(const Operand& o, const void* p, int64_t stride, int64_t rows, int64_t cols, cudaStream_t s) {
    if (!o.copied) return 0;
    const int64_t items = rows * (o.ld / 8);
    align_rows_kernel<<<blocks_for(items, 256, kSmCount * 32), 256, 0, s>>>(
        static_cast<const uint16_t*>(p), stride, rows, cols, static_cast<uint16_t*>(const_cast<void*>(o.p)), o.ld);
    return launch_status();
}

// Whether dot products on the cores are the faster form. fp32: up to eight rows.
// 16-bit types, against the thin product on tcgen05 that costs a start of some
// 5 us and then the bytes of W whatever the rows (cores | tcgen05, us): one row
// of 4096 -> 4096 7.9 | 10.6, 8192 -> 8192 23.1 | 24.5, 4096 -> 32000 47 | 43;
// two rows of 4096 -> 4096 8.6 | 10.6, 4096 -> 12288 21 | 20; four of 512 -> 16384
// 7.8 | 7.8, 4096 -> 4096 12.7 | 10.9; eight of 4096 -> 512 4.4 | 6.0, 512 -> 16384
// 11.1 | 8.0. Rows that TMA cannot read have to be copied for it first: one row
// of 4097 -> 12288 32 | 62, four 51 | 64, eight 90 | 64, eight of 517 -> 16384 19 | 18.
bool few_rows_win(const gk_linear_t& p) {
    if (p.m > kFewRows) return false;
    if (p.dtype == GK_FP32) return true;
    const double work = (double)p.m * (double)p.n * (double)p.k;
    if (!tma_rows(p.x, p.x_stride, p.k) || !tma_rows(p.w, p.w_stride, p.k)) return p.m <= 4 || work <= 1 << 26;
    return work <= (p.m == 1 ? 8e7 : 1 << 25);
}

struct ForwardPlan {
    Operand x, w;
    size_t bytes;
    bool few;
};
ForwardPlan forward_plan(const gk_linear_t& p, void* workspace) {
    ForwardPlan f{};
    Arena arena(workspace);
    f.few = few_rows_win(p);
    if (!f.few && p.dtype != GK_FP32) {
        f.x = operand(arena, p.x, p.x_stride, p.m, p.k);
        f.w = operand(arena, p.w, p.w_stride, p.n, p.k);
    }
    f.bytes = arena.used;
    return f;
}

template <typename T>
int few_rows_by_m(const FewRows& f, cudaStream_t s) {
    if (f.m <= 1) return few_rows<T, 1>(f, s);
    if (f.m <= 2) return few_rows<T, 2>(f, s);
    if (f.m <= 4) return few_rows<T, 4>(f, s);
    return few_rows<T, 8>(f, s);
}

bool forward_ok(const gk_linear_t* p) {
    if (p == nullptr || !sizes_ok(p->m, p->n, p->k, p->dtype, p->activation)) return false;
    if (p->m == 0) return true;
    return p->x != nullptr && p->w != nullptr && p->y != nullptr && p->x_stride >= 0 && p->w_stride >= 0 &&
           (p->residual == nullptr || p->residual_stride >= 0) &&
           (p->pre == nullptr || p->pre_stride >= p->n);
}

struct BackwardPlan {
    bool forms_dz;    // dz is another matrix than dy
    Operand x, w, dz;
    // Products of few outputs that take dz before its rounding, on the fp32 units.
    bool narrow_dx, narrow_dw;
    float* dz32;
    void* unpacked;   // x from its codes
    int64_t unpacked_ld;
    float* sums;
    SlopePlan slope;
    bool runs_slope;
    size_t bytes;
};

// The rounding of dz to 16 bits puts an error into a gradient as large as the
// gradient's own rounding, 1.4 times in all; tcgen05 takes 16-bit operands, so a
// product that it runs has to bear that. A narrow one, of few outputs or from
// few dz (a head's, a short batch's), takes as long on the fp32 units and gets
// dz in fp32 there, and its operands as they lie. Measured (us, fp32 units |
// tcgen05 with its aligned copies): 7 x 4756 -> 17 both gradients 5.7 | 12.3, dw of
// 1024 x 4000 -> 4 13.3 | 8.6, of 12616 x 2 -> 4 31 | 14, of 16384 x 128 -> 128 45 | 14,
// dx of 4 x 4096 -> 4096 46 | 10: hence the bounds on the contraction and the work.
bool narrow(int64_t rows, int64_t cols, int64_t contraction, int64_t dz) {
    return (rows * cols <= 1 << 14 || dz <= 1 << 12) && contraction <= 4096 &&
           (double)rows * (double)cols * (double)contraction <= 1 << 23;
}

template <typename T>
BackwardPlan backward_plan(const gk_linear_grad_t& p, void* workspace) {
    constexpr bool k16 = sizeof(T) == 2;
    BackwardPlan b{};
    Arena arena(workspace);
    if (k16 && (p.activation == GK_ACT_TANH || p.activation == GK_ACT_GELU || p.activation == GK_ACT_SILU)) {
        b.narrow_dx = p.dx != nullptr && narrow(p.m, p.k, p.n, p.m * p.n);
        b.narrow_dw = p.dw != nullptr && narrow(p.n, p.k, p.m, p.m * p.n);
        if (b.narrow_dx || b.narrow_dw) b.dz32 = static_cast<float*>(arena.take(p.m * pad8(p.n) * 4));
    }
    const bool products = (p.dx != nullptr && !b.narrow_dx) || (p.dw != nullptr && !b.narrow_dw);
    // Without an activation dz is dy, unless the product needs its rows aligned.
    b.forms_dz = p.activation != GK_ACT_NONE || (k16 && products && !tma_rows(p.dy, p.dy_stride, p.n));
    b.dz = {p.dy, p.dy_stride, false};
    if (b.forms_dz) {
        // The residual's gradient serves as dz where its rows are aligned.
        if (p.dz != nullptr && (!k16 || !products || tma_rows(p.dz, p.n, p.n)))
            b.dz = {p.dz, p.n, false};
        else if ((b.narrow_dx || b.narrow_dw) && !products)  // all who read dz read it in fp32
            b.dz = {nullptr, 0, false};
        else
            b.dz = {arena.take(p.m * pad8(p.n) * (int64_t)sizeof(T)), pad8(p.n), false};
    }
    if (p.dw != nullptr && p.x_codes != nullptr) {
        b.unpacked_ld = k16 ? pad8(p.k) : p.k;
        b.unpacked = arena.take(p.m * b.unpacked_ld * (int64_t)sizeof(T));
    }
    if (k16) {
        if (p.dw != nullptr && !b.narrow_dw && p.x_codes == nullptr)
            b.x = operand(arena, p.x, p.x_stride, p.m, p.k);
        else
            b.x = {p.x, p.x_stride, false};
        b.w = {p.w, p.w_stride, false};
        if (p.dx != nullptr && !b.narrow_dx) b.w = operand(arena, p.w, p.w_stride, p.n, p.k);
    } else {
        b.x = {p.x, p.x_stride, false};
        b.w = {p.w, p.w_stride, false};
    }
    if (b.unpacked_ld > 0) b.x = {b.unpacked, b.unpacked_ld, false};
    b.runs_slope = b.forms_dz || p.db != nullptr;
    const bool vec = aligned16(p.dy) && p.dy_stride % kVec<T> == 0 && p.n % kVec<T> == 0 &&
                     (p.kept == nullptr || (aligned16(p.kept) && p.kept_stride % kVec<T> == 0)) && (p.dz == nullptr || aligned16(p.dz));
    b.slope = slope_plan<T>(p.m, p.n, vec);
    if (p.db != nullptr) b.sums = static_cast<float*>(arena.take((int64_t)b.slope.slabs * p.n * 4));
    b.bytes = arena.used;
    return b;
}

bool backward_ok(const gk_linear_grad_t* p) {
    if (p == nullptr || !sizes_ok(p->m, p->n, p->k, p->dtype, p->activation) || p->m < 1) return false;
    if (p->dy == nullptr || p->dy_stride < 0) return false;
    if (p->activation != GK_ACT_NONE && (p->kept == nullptr || p->kept_stride < 0)) return false;
    if (p->activation == GK_ACT_NONE && p->dz != nullptr) return false;
    if (p->dx != nullptr && (p->w == nullptr || p->w_stride < 0)) return false;
    if (p->dw != nullptr && p->x == nullptr && (p->x_codes == nullptr || p->x_scales == nullptr)) return false;
    return true;
}

template <typename T>
int backward(const gk_linear_grad_t& p, void* workspace, uint32_t* status, cudaStream_t s) {
    constexpr bool k16 = sizeof(T) == 2;
    const BackwardPlan b = backward_plan<T>(p, workspace);
    int e = 0;
    if (b.runs_slope) {
        Slope a{p.dy, p.activation == GK_ACT_NONE ? nullptr : p.kept,
                b.forms_dz ? const_cast<void*>(b.dz.p) : nullptr, b.dz32, b.sums, p.dy_stride, p.kept_stride, b.dz.ld,
                pad8(p.n), p.m, p.n,
                b.slope.slab, p.activation};
        const dim3 grid((unsigned)b.slope.col_blocks, (unsigned)b.slope.slabs);
        if ((e = launch_slope<T>(a, grid, b.slope, s)) != 0) return e;
        if (p.db != nullptr) {
            linear_bias_kernel<T><<<(unsigned)((p.n + 31) / 32), 256, 0, s>>>(b.sums, p.n, b.slope.slabs,
                                                                                 static_cast<T*>(p.db));
            if ((e = launch_status()) != 0) return e;
        }
    }
    if (p.dz != nullptr && b.dz.p != p.dz) {
        // dz lies in aligned rows of the workspace; the residual's gradient has rows of n.
        const cudaError_t c = cudaMemcpy2DAsync(p.dz, p.n * sizeof(T), b.dz.p, b.dz.ld * sizeof(T),
                                                p.n * sizeof(T), p.m, cudaMemcpyDeviceToDevice, s);
        if (c != cudaSuccess) return (int)c;
    }
    if (p.dw != nullptr && p.x_codes != nullptr) {
        e = gk_unpack(p.x_codes, p.x_scales, p.m, p.k, b.unpacked, b.unpacked_ld, p.dtype, s);
        if (e != 0) return e;
    }
    if constexpr (k16) {
        const Gemm32 none{};
        if (b.narrow_dx) {
            Gemm32 g = none;
            g.a = b.dz32, g.b = b.w.p, g.a_ld = pad8(p.n), g.b_ld = b.w.ld, g.out = p.dx, g.out_ld = p.k;
            g.m = p.m, g.n = p.k, g.k = p.n;
            if ((e = gemm32_narrow<T, true>(g, s)) != 0) return e;
        } else if (p.dx != nullptr) {
            if ((e = copy_if_needed(b.w, p.w, p.w_stride, p.n, p.k, s)) != 0) return e;
            GemmArgs g{b.dz.p, b.w.p, b.dz.ld, b.w.ld, 0, 1, p.dx, p.k, nullptr, nullptr, 0, nullptr, 0,
                       p.m, p.k, p.n, p.dtype, GK_ACT_NONE};
            if ((e = gemm16(g, status, s)) != 0) return e;
        }
        if (b.narrow_dw) {
            Gemm32 g = none;
            g.a = b.dz32, g.b = b.x.p, g.a_ld = pad8(p.n), g.b_ld = b.x.ld, g.out = p.dw, g.out_ld = p.k;
            g.m = p.n, g.n = p.k, g.k = p.m;
            if ((e = gemm32_narrow<T, false>(g, s)) != 0) return e;
        } else if (p.dw != nullptr) {
            if (p.x_codes == nullptr && (e = copy_if_needed(b.x, p.x, p.x_stride, p.m, p.k, s)) != 0) return e;
            GemmArgs g{b.dz.p, b.x.p, b.dz.ld, b.x.ld, 1, 1, p.dw, p.k, nullptr, nullptr, 0, nullptr, 0,
                       p.n, p.k, p.m, p.dtype, GK_ACT_NONE};
            if ((e = gemm16(g, status, s)) != 0) return e;
        }
    } else {
        const float* dz = static_cast<const float*>(b.dz.p);
        if (p.dx != nullptr) {
            Gemm32 g{dz, static_cast<const float*>(b.w.p), b.dz.ld, b.w.ld, static_cast<float*>(p.dx),
                     nullptr, nullptr, nullptr, p.k, 0, 0, p.m, p.k, p.n, GK_ACT_NONE, 0};
            if ((e = gemm32<true, false>(g, s)) != 0) return e;
        }
        if (p.dw != nullptr) {
            Gemm32 g{dz, static_cast<const float*>(b.x.p), b.dz.ld, b.x.ld, static_cast<float*>(p.dw),
                     nullptr, nullptr, nullptr, p.k, 0, 0, p.n, p.k, p.m, GK_ACT_NONE, 0};
            if ((e = gemm32<false, false>(g, s)) != 0) return e;
        }
    }
    return 0;
}

}  // namespace
}  // namespace gk

extern "C" {

size_t gk_linear_workspace_bytes(const gk_linear_t* p) {
    return gk::forward_ok(p) && p->m > 0 ? gk::forward_plan(*p, nullptr).bytes : 0;
}

int gk_linear_forward(const gk_linear_t* p, void* workspace, uint32_t* status, void* stream) {
    using namespace gk;
    if (!forward_ok(p) || status == nullptr) return GK_EINVAL;
    if (p->m == 0) return 0;
    const ForwardPlan f = forward_plan(*p, workspace);
    if (f.bytes > 0 && workspace == nullptr) return GK_EINVAL;
    cudaStream_t s = as_stream(stream);
    if (f.few) {
        FewRows r{p->x, p->w, p->bias, p->residual, p->y, p->pre, p->x_stride, p->w_stride, p->residual_stride,
                  p->pre_stride, (int)p->m, (int)p->n, p->k, p->activation, 1};
        if (p->dtype == GK_FP32) return few_rows_by_m<float>(r, s);
        if (p->dtype == GK_BF16) return few_rows_by_m<__nv_bfloat16>(r, s);
        return few_rows_by_m<__half>(r, s);
    }
    if (p->dtype == GK_FP32) {
        Gemm32 g{static_cast<const float*>(p->x), static_cast<const float*>(p->w), p->x_stride, p->w_stride,
                 static_cast<float*>(p->y), static_cast<const float*>(p->bias),
                 static_cast<const float*>(p->residual), static_cast<float*>(p->pre), p->n, p->residual_stride,
                 p->pre_stride,                 p->m, p->n, p->k, p->activation, 0};
        return gemm32<true, true>(g, s);
    }
    int e = copy_if_needed(f.x, p->x, p->x_stride, p->m, p->k, s);
    if (e == 0) e = copy_if_needed(f.w, p->w, p->w_stride, p->n, p->k, s);
    if (e != 0) return e;
    GemmArgs g{f.x.p, f.w.p, f.x.ld, f.w.ld, 0, 0, p->y, p->n, p->bias, p->residual, p->residual_stride, p->pre,
               p->pre_stride, p->m, p->n, p->k, p->dtype, p->activation};
    return gemm16(g, status, s);
}

size_t gk_linear_grad_workspace_bytes(const gk_linear_grad_t* p) {
    using namespace gk;
    if (!backward_ok(p)) return 0;
    return p->dtype == GK_FP32 ? backward_plan<float>(*p, nullptr).bytes : backward_plan<__half>(*p, nullptr).bytes;
}

int gk_linear_backward(const gk_linear_grad_t* p, void* workspace, uint32_t* status, void* stream) {
    using namespace gk;
    if (!backward_ok(p) || status == nullptr) return GK_EINVAL;
    if (workspace == nullptr && gk_linear_grad_workspace_bytes(p) > 0) return GK_EINVAL;
    cudaStream_t s = as_stream(stream);
    if (p->dtype == GK_FP32) return backward<float>(*p, workspace, status, s);
    if (p->dtype == GK_BF16) return backward<__nv_bfloat16>(*p, workspace, status, s);
    return backward<__half>(*p, workspace, status, s);
}

}  // extern "C"
