// gk_pack.cu - activations kept in 8 bits for the backward pass.
//
// A block of 32 values shares a power-of-two scale 2^s with
// 448 2^(s-1) < max |x| <= 448 2^s, so a value x is held as e4m3(x 2^-s): three
// fraction bits (off by at most 2^-4 of itself) down to max |x| 2^-15, then evenly spaced
// to 2^-18 of the maximum, below which it is held as zero. The scale being a
// power of two, every held value is a bf16, fp16 and fp32 value: unpacking
// rounds nothing. Memory traffic bounds both directions: 8192 x 4096 bf16 packed
// in 18 us (5.6 TB/s) and unpacked in 17 (6.0), 4096 x 5184 fp32 in 19 and 15.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/gk.h"
#include "gk_act.cuh"
#include "gk_launch.cuh"

namespace gk {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kBlock = 32;

template <typename T>
constexpr int kLowest = -124;  // least scale exponent: the smallest step 2^(s-9) is a value of T
template <>
constexpr int kLowest<__half> = -15;
template <typename T>
constexpr float kLargest = 3.4028234663852886e38f;
template <>
constexpr float kLargest<__half> = 65504.0f;
template <>
constexpr float kLargest<__nv_bfloat16> = 3.3895313892515355e38f;

// The scale exponent for a block whose largest finite magnitude is `top`.
template <typename T>
__device__ __forceinline__ int scale_exponent(float top) {
    if (top == 0.0f) return max(0, kLowest<T>);
    // top = f 2^e, 1 <= f < 2; 448 = 1.75 2^8. (A subnormal top counts as e = -127, which the least scale covers.)
    const uint32_t bits = __float_as_uint(top);
    const int e = (int)(bits >> 23) - 127;
    return max(kLowest<T>, (bits & 0x7fffffu) > 0x600000u ? e - 7 : e - 8);
}

__device__ __forceinline__ float finite_magnitude(float x) {
    const float a = fabsf(x);
    return a <= 3.4028234663852886e38f ? a : 0.0f;  // also false for NaN
}

__device__ __forceinline__ uint32_t code_of(float x, float inverse) {
    if (!(fabsf(x) <= 3.4028234663852886e38f)) return 0x7fu;
    return __nv_cvt_float_to_fp8(x * inverse, __NV_SATFINITE, __NV_E4M3);
}

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// The value of a code: the code's four exponent and three fraction bits under
// a float's exponent, times 2^120 for the difference of the biases.
__device__ __forceinline__ float value_of(uint32_t code) {
    const uint32_t magnitude = code & 0x7fu;
    if (magnitude == 0x7fu) return __uint_as_float(0x7fc00000u);
    const float v = __uint_as_float(magnitude << 20) * 1.329227995784916e36f;
    return __uint_as_float(__float_as_uint(v) | ((code & 0x80u) << 24));
}

template <typename T>
__device__ __forceinline__ T held(uint32_t code, float scale) {
    const float v = value_of(code) * scale;
    const float most = kLargest<T>;
    return rounded<T>(v > most ? most : (v < -most ? -most : v));
}

// The largest finite magnitude of a warp's lanes: as bits, which order like the magnitudes.
__device__ __forceinline__ float warp_top(float v) {
    return __uint_as_float(__reduce_max_sync(kFull, __float_as_uint(finite_magnitude(v))));
}

// A lane an element, a warp four blocks of 32 at a time along a chunk of a row.
constexpr int64_t kChunk = 4096;  // columns a warp takes of a row
template <typename T>
__device__ __forceinline__ void pack_span(const T* x, int64_t count, uint8_t* codes, uint8_t* scales, int lane) {
    for (int64_t c0 = 0; c0 < count; c0 += 4 * kBlock) {
        float v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t c = c0 + u * kBlock + lane;
            v[u] = c < count ? as_float<T>(x[c]) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t c = c0 + u * kBlock + lane;
            const int s = scale_exponent<T>(warp_top(v[u]));
            if (c < count) codes[c] = (uint8_t)code_of(v[u], power_of_two(-s));
            if (lane == 0 && c < count) scales[c / kBlock] = (uint8_t)(s + 127);
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(256) pack_rows_kernel(const T* x, int64_t stride, int64_t rows, int64_t cols,
                                                        uint8_t* codes, uint8_t* scales) {
    const int lane = threadIdx.x & 31;
    const int64_t per_row = (cols + kBlock - 1) / kBlock, chunks = (cols + kChunk - 1) / kChunk;
    const int64_t items = rows * chunks, warps = (int64_t)gridDim.x * 8;
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += warps) {
        const int64_t r = it / chunks, c0 = (it - r * chunks) * kChunk;
        pack_span(x + r * stride + c0, cols - c0 < kChunk ? cols - c0 : kChunk, codes + r * cols + c0,
                  scales + r * per_row + c0 / kBlock, lane);
    }
}

// The largest magnitude of a vector, with infinities and NaN; 16-bit values stay packed.
template <typename T>
__device__ __forceinline__ float vector_top(uint4 raw);
template <>
__device__ __forceinline__ float vector_top<float>(uint4 raw) {
    // As bits, which order like the magnitudes and put NaN above infinity.
    const uint32_t m = 0x7fffffffu;
    return __uint_as_float(max(max(raw.x & m, raw.y & m), max(raw.z & m, raw.w & m)));
}
template <typename P>
__device__ __forceinline__ P packed_top(uint4 raw) {
    const uint32_t m = 0x7fff7fffu;
    uint32_t w[4] = {raw.x & m, raw.y & m, raw.z & m, raw.w & m};
    const P* v = reinterpret_cast<const P*>(w);
    return __hmax2_nan(__hmax2_nan(v[0], v[1]), __hmax2_nan(v[2], v[3]));
}
__device__ __forceinline__ float greater_or_nan(float a, float b) { return a > b || a != a ? a : b; }
template <>
__device__ __forceinline__ float vector_top<__half>(uint4 raw) {
    const float2 f = __half22float2(packed_top<__half2>(raw));
    return greater_or_nan(f.x, f.y);
}
template <>
__device__ __forceinline__ float vector_top<__nv_bfloat16>(uint4 raw) {
    const float2 f = __bfloat1622float2(packed_top<__nv_bfloat162>(raw));
    return greater_or_nan(f.x, f.y);
}

// Whole blocks of aligned rows: 16 bytes a thread, 32 * sizeof(T) / 16 threads
// a block of 32, four vectors a thread in flight.
template <typename T>
__global__ void __launch_bounds__(256) pack_vectors_kernel(const T* x, int64_t vectors, int tail, uint8_t* codes,
                                                           uint8_t* scales) {
    constexpr int V = 16 / (int)sizeof(T), kTeam = kBlock / V, kUnroll = 4;
    if (tail > 0 && blockIdx.x == gridDim.x - 1) {  // the last, shorter block of 32
        if (threadIdx.x < 32)
            pack_span(x + vectors * V, tail, codes + vectors * V, scales + vectors / kTeam, threadIdx.x);
        return;
    }
    const int64_t start = (int64_t)blockIdx.x * (256 * kUnroll) + threadIdx.x;
    uint4 raw[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = start + u * 256;
        raw[u] = i < vectors ? __ldcs(reinterpret_cast<const uint4*>(x) + i) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = start + u * 256;
        const T* v = reinterpret_cast<const T*>(&raw[u]);
        float top = vector_top<T>(raw[u]);  // not finite if any value is not
#pragma unroll
        for (int o = kTeam / 2; o; o >>= 1) {
            const float other = __shfl_xor_sync(kFull, top, o);
            top = other > top || other != other ? other : top;
        }
        uint32_t word[V / 4];
        int s;
        if (top <= 3.4028234663852886e38f) {
            s = scale_exponent<T>(top);
            const float inverse = power_of_two(-s);
#pragma unroll
            for (int k = 0; k < V / 4; ++k) {
                const float2 a = make_float2(as_float<T>(v[4 * k]) * inverse, as_float<T>(v[4 * k + 1]) * inverse);
                const float2 b = make_float2(as_float<T>(v[4 * k + 2]) * inverse, as_float<T>(v[4 * k + 3]) * inverse);
                word[k] = (uint32_t)__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3) |
                          (uint32_t)__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3) << 16;
            }
        } else {  // the whole team is here: an infinity or a NaN among the block's values
            top = 0.0f;
#pragma unroll
            for (int k = 0; k < V; ++k) top = fmaxf(top, finite_magnitude(as_float<T>(v[k])));
            // Its own lanes, whichever others are here.
            const unsigned team = ((1u << kTeam) - 1u) << (threadIdx.x & 31 & ~(kTeam - 1));
#pragma unroll
            for (int o = kTeam / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(team, top, o));
            s = scale_exponent<T>(top);
            const float inverse = power_of_two(-s);
#pragma unroll
            for (int k = 0; k < V / 4; ++k)
                word[k] = code_of(as_float<T>(v[4 * k]), inverse) | code_of(as_float<T>(v[4 * k + 1]), inverse) << 8 |
                          code_of(as_float<T>(v[4 * k + 2]), inverse) << 16 |
                          code_of(as_float<T>(v[4 * k + 3]), inverse) << 24;
        }
        if (i < vectors) {
            if constexpr (V == 4)
                reinterpret_cast<uint32_t*>(codes)[i] = word[0];
            else
                reinterpret_cast<uint2*>(codes)[i] = make_uint2(word[0], word[1]);
            if ((threadIdx.x & (kTeam - 1)) == 0) scales[i / kTeam] = (uint8_t)(s + 127);
        }
    }
}

template <typename T>
__device__ __forceinline__ void unpack_span(const uint8_t* codes, const uint8_t* scales, int64_t count, T* x,
                                            int lane) {
    for (int64_t c0 = 0; c0 < count; c0 += 4 * kBlock) {
        uint32_t code[4], scale[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t c = c0 + u * kBlock + lane;
            code[u] = c < count ? codes[c] : 0u;
            scale[u] = c < count ? scales[c / kBlock] : 0u;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t c = c0 + u * kBlock + lane;
            if (c < count) x[c] = held<T>(code[u], power_of_two((int)scale[u] - 127));
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(256) unpack_rows_kernel(const uint8_t* codes, const uint8_t* scales, int64_t rows,
                                                          int64_t cols, T* x, int64_t stride) {
    const int lane = threadIdx.x & 31;
    const int64_t per_row = (cols + kBlock - 1) / kBlock, chunks = (cols + kChunk - 1) / kChunk;
    const int64_t items = rows * chunks, warps = (int64_t)gridDim.x * 8;
    for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += warps) {
        const int64_t r = it / chunks, c0 = (it - r * chunks) * kChunk;
        unpack_span(codes + r * cols + c0, scales + r * per_row + c0 / kBlock,
                    cols - c0 < kChunk ? cols - c0 : kChunk, x + r * stride + c0, lane);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) unpack_vectors_kernel(const uint8_t* codes, const uint8_t* scales,
                                                             int64_t vectors, int tail, T* x) {
    constexpr int V = 16 / (int)sizeof(T), kTeam = kBlock / V, kUnroll = 4;
    if (tail > 0 && blockIdx.x == gridDim.x - 1) {  // the last, shorter block of 32
        if (threadIdx.x < 32)
            unpack_span(codes + vectors * V, scales + vectors / kTeam, tail, x + vectors * V, threadIdx.x);
        return;
    }
    const int64_t start = (int64_t)blockIdx.x * (256 * kUnroll) + threadIdx.x;
    uint32_t word[kUnroll][V / 4];
    float scale[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = start + u * 256;
        if (i >= vectors) continue;
        if constexpr (V == 4) {
            word[u][0] = __ldcs(reinterpret_cast<const uint32_t*>(codes) + i);
        } else {
            const uint2 w = __ldcs(reinterpret_cast<const uint2*>(codes) + i);
            word[u][0] = w.x, word[u][V / 4 - 1] = w.y;
        }
        scale[u] = power_of_two((int)scales[i / kTeam] - 127);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const int64_t i = start + u * 256;
        if (i >= vectors) continue;
        alignas(16) T out[V];
        // No value is above 448 scale, so below this scale none has to be cut off.
        if (scale[u] <= kLargest<T> / 512.0f) {
#pragma unroll
            for (int k = 0; k < V; k += 2) {
                const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
                    (__nv_fp8x2_storage_t)(word[u][k / 4] >> (8 * (k % 4))), __NV_E4M3);
                const float2 f = __half22float2(__half2(h));
                out[k] = rounded<T>(f.x * scale[u]);
                out[k + 1] = rounded<T>(f.y * scale[u]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) out[k] = held<T>((word[u][k / 4] >> (8 * (k % 4))) & 0xffu, scale[u]);
        }
        reinterpret_cast<uint4*>(x)[i] = *reinterpret_cast<uint4*>(out);
    }
}

bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

// Rows in whole blocks that follow one another without a gap, or one row: one
// run of vectors, and the row's last block if it is shorter.
bool one_run(int64_t rows, int64_t cols, int64_t stride) {
    return rows == 1 || (cols % kBlock == 0 && stride == cols);
}

template <typename T>
int pack(const void* x, int64_t stride, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scales,
         cudaStream_t s) {
    if (one_run(rows, cols, stride) && aligned16(x) && aligned8(codes)) {
        const int tail = (int)(rows * cols % kBlock);
        const int64_t vectors = (rows * cols - tail) / (16 / (int64_t)sizeof(T));
        const unsigned grid = (unsigned)((vectors + 1023) / 1024) + (tail > 0 ? 1u : 0u);
        pack_vectors_kernel<T><<<grid, 256, 0, s>>>(static_cast<const T*>(x), vectors, tail, codes, scales);
    } else {
        const int64_t items = rows * ((cols + kChunk - 1) / kChunk);
        pack_rows_kernel<T><<<blocks_for(items, 8, kSmCount * 32), 256, 0, s>>>(static_cast<const T*>(x), stride,
                                                                                rows, cols, codes, scales);
    }
    return launch_status();
}

template <typename T>
int unpack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* x, int64_t stride,
           cudaStream_t s) {
    if (one_run(rows, cols, stride) && aligned16(x) && aligned8(codes)) {
        const int tail = (int)(rows * cols % kBlock);
        const int64_t vectors = (rows * cols - tail) / (16 / (int64_t)sizeof(T));
        const unsigned grid = (unsigned)((vectors + 1023) / 1024) + (tail > 0 ? 1u : 0u);
        unpack_vectors_kernel<T><<<grid, 256, 0, s>>>(codes, scales, vectors, tail, static_cast<T*>(x));
    } else {
        const int64_t items = rows * ((cols + kChunk - 1) / kChunk);
        unpack_rows_kernel<T><<<blocks_for(items, 8, kSmCount * 32), 256, 0, s>>>(codes, scales, rows, cols,
                                                                                  static_cast<T*>(x), stride);
    }
    return launch_status();
}

// Sizes whose element count, and grid, stay in range.
bool valid(const void* x, int64_t stride, int64_t rows, int64_t cols, const void* codes, const void* scales) {
    if (rows < 0 || cols < 0) return false;
    if (rows == 0 || cols == 0) return true;
    if (rows > (1ll << 40) / cols || (rows > 1 && stride < cols)) return false;
    return x != nullptr && codes != nullptr && scales != nullptr;
}

}  // namespace
}  // namespace gk

extern "C" {

int gk_pack(const void* x, int64_t stride, int dtype, int64_t rows, int64_t cols, uint8_t* codes, uint8_t* scales,
            void* stream) {
    using namespace gk;
    if (!valid(x, stride, rows, cols, codes, scales) || dtype < GK_FP32 || dtype > GK_FP16) return GK_EINVAL;
    if (rows == 0 || cols == 0) return 0;
    cudaStream_t s = as_stream(stream);
    if (dtype == GK_FP32) return pack<float>(x, stride, rows, cols, codes, scales, s);
    if (dtype == GK_BF16) return pack<__nv_bfloat16>(x, stride, rows, cols, codes, scales, s);
    return pack<__half>(x, stride, rows, cols, codes, scales, s);
}

int gk_unpack(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t cols, void* x, int64_t stride,
              int dtype, void* stream) {
    using namespace gk;
    if (!valid(x, stride, rows, cols, codes, scales) || dtype < GK_FP32 || dtype > GK_FP16) return GK_EINVAL;
    if (rows == 0 || cols == 0) return 0;
    cudaStream_t s = as_stream(stream);
    if (dtype == GK_FP32) return unpack<float>(codes, scales, rows, cols, x, stride, s);
    if (dtype == GK_BF16) return unpack<__nv_bfloat16>(codes, scales, rows, cols, x, stride, s);
    return unpack<__half>(codes, scales, rows, cols, x, stride, s);
}

}  // extern "C"
