// Arguments and epilogue of the dense products (linear.hip).
#pragma once

#include "lds_ring.h"
#include "moe_common.h"

namespace moe {

constexpr int64_t kMaxLinearWidth = 1 << 20;
constexpr int64_t kMaxLinearTokens = 1 << 21;

struct LinearArgs {
    const uint8_t* x;        // [T, k_bytes] bytes of bf16 or e4m3
    const uint8_t* weight;   // [rows, w_stride bytes]
    const float* x_scales;   // e4m3: [T]
    const float* w_scales;   // e4m3: [rows]
    const void* bias;        // [rows], fp32 or bf16, or null
    const uint16_t* residual;  // [T, n] bf16 or null
    uint16_t* output;        // [T, n] bf16
    int64_t tokens;
    int64_t k_bytes;         // of a row of x
    int64_t w_stride;        // bytes from one weight row to the next
    int64_t n;               // output columns
    int64_t rows;            // weight rows: n, or 2 n for swiglu (gate rows, then up rows)
    bool bias_bf16;
    bool fp8;
    int activation;          // MOE_ACT_*
};

int64_t linear_scratch_bytes(const LinearArgs& a);
int launch_linear(const LinearArgs& a, void* scratch, hipStream_t stream);

}  // namespace moe
