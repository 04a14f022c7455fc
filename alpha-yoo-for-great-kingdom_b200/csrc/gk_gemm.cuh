// gk_gemm.cuh - the 16-bit matrix product of the training-step operators.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace gk {

// out[m, n] = act(sum_k A[m, k] B[n, k] + bias[n] + residual[m, n]), fp32
// accumulation, one rounding to the output. Each operand is stored with k
// contiguous (`*_across` 0: row m or n, leading dimension *_ld) or with m or n
// contiguous (`*_across` 1: row k). Operands start on 16 bytes and have leading
// dimensions that are multiples of 8; everything else may be odd.
struct GemmArgs {
    const void* a;
    const void* b;
    int64_t a_ld, b_ld;
    int a_across, b_across;
    void* out;
    int64_t out_ld;
    const void* bias;      // or nullptr
    const void* residual;  // or nullptr
    int64_t residual_ld;
    void* pre;             // the sum before the activation (tanh: its value in fp32), or nullptr
    int64_t pre_ld;
    int64_t m, n, k;       // each below 2^31, k >= 1
    int dtype;             // GK_BF16 or GK_FP16
    int activation;        // GK_ACT_*
};

// 0, GK_EINVAL or a cudaError_t. status: uint32[2], GK_ERR_TIMEOUT convention.
int gemm16(const GemmArgs& g, uint32_t* status, cudaStream_t stream);

}  // namespace gk
