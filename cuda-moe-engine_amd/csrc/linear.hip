// Dense products with their epilogue: y = act(x W^T + b) + residual.
//
//   bf16:  z = sum_k x_tk W_nk,   e4m3:  z = (sum_k x_tk W_nk) sx_t sw_n
//   swiglu: W holds n gate rows, then n up rows; y = silu(z_gate) z_up + residual
//
// Products accumulate in fp32 on MFMA and everything behind them stays in fp32: one rounding
// to bf16. Both types run the same code over bytes: a 128-byte stage of a row is 64 bf16
// (two 16x16x32 products) or 128 e4m3 (one 16x16x128), and any order of k inside it is as
// good as another as long as x and W share it.
#include "linear.h"

namespace moe {

namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));
typedef int intx4 __attribute__((ext_vector_type(4)));

// 16 weight rows by 16 rows of x, 128 bytes of k: lane l holds bytes [32 (l / 16), + 32) of row
// l % 16 of each. Lane l's result: x row l % 16, weight rows 4 (l / 16) + 0..3.
template <bool FP8>
__device__ __forceinline__ floatx4 mma(const intx4 (&w)[2], const intx4 (&x)[2], floatx4 acc) {
    if constexpr (FP8) {
        intx8 a, b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            a[i] = w[0][i];
            a[4 + i] = w[1][i];
            b[i] = x[0][i];
            b[4 + i] = x[1][i];
        }
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, 0, 0, 0);
    } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w[h]),
                                                          __builtin_bit_cast(bf16x8_t, x[h]), acc, 0, 0, 0);
        return acc;
    }
}

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case MOE_ACT_RELU: return z < 0.0f ? 0.0f : z;  // NaN stays
        case MOE_ACT_SILU: return z / (1.0f + expf(-z));
        case MOE_ACT_GELU: return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
        case MOE_ACT_GELU_TANH: return 0.5f * z * (1.0f + tanhf(0.79788456080286536f * (z + 0.044715f * z * z * z)));
        default: return z;
    }
}

__device__ __forceinline__ float bias_at(const LinearArgs& a, int64_t row) {
    if (a.bias == nullptr) return 0.0f;
    return a.bias_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.bias)[row]) : static_cast<const float*>(a.bias)[row];
}

constexpr int kTile = 64, kStage = 128, kPad = 16;

// A 64 x 64 tile on four waves of 32 x 32, one stage in LDS at a time.
template <bool FP8, bool SWIGLU>
__global__ __launch_bounds__(256) void linear_tile_kernel(LinearArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t lx[kTile][kStage + kPad], lw[kTile][kStage + kPad];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t t0 = static_cast<int64_t>(blockIdx.y) * kTile;
    constexpr int COLS = SWIGLU ? kTile / 2 : kTile;
    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * COLS;
    const int wt = (wave >> 1) * 32, wn = (wave & 1) * 32;
    // Weight row of LDS row r: swiglu pairs 16 gate rows with their 16 up rows.
    auto weight_row = [&](int r) -> int64_t {
        if constexpr (SWIGLU) {
            const int64_t col = n0 + (r / 32) * 16 + r % 16;
            return col < a.n ? (r % 32 < 16 ? col : a.n + col) : -1;
        }
        return n0 + r < a.n ? n0 + r : -1;
    };
    floatx4 acc[2][2] = {};
    for (int64_t k = 0; k < a.k_bytes; k += kStage) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kTile * kStage / 16 / 256; ++i) {
            const int at = i * 256 + threadIdx.x, r = at / 8, c = at % 8 * 16;
            uint4 vx = make_uint4(0, 0, 0, 0), vw = vx;
            const int64_t wr = weight_row(r);
            if (k + c < a.k_bytes) {
                if (t0 + r < a.tokens) vx = *reinterpret_cast<const uint4*>(a.x + (t0 + r) * a.k_bytes + k + c);
                if (wr >= 0) vw = *reinterpret_cast<const uint4*>(a.weight + wr * a.w_stride + k + c);
            }
            *reinterpret_cast<uint4*>(&lx[r][c]) = vx;
            *reinterpret_cast<uint4*>(&lw[r][c]) = vw;
        }
        __syncthreads();
        intx4 fx[2][2], fw[2][2];
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int c = (lane >> 4) * 32 + h * 16;
                fx[f][h] = *reinterpret_cast<const intx4*>(&lx[wt + f * 16 + (lane & 15)][c]);
                fw[f][h] = *reinterpret_cast<const intx4*>(&lw[wn + f * 16 + (lane & 15)][c]);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = mma<FP8>(fw[j], fx[i], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int64_t t = t0 + wt + i * 16 + (lane & 15);
        if (t >= a.tokens) continue;
        const float sx = FP8 ? a.x_scales[t] : 1.0f;
#pragma unroll
        for (int j = 0; j < (SWIGLU ? 1 : 2); ++j) {
            const int64_t col = n0 + (SWIGLU ? wn / 2 : wn + j * 16) + 4 * (lane >> 4);
            if (col >= a.n) continue;
            float y[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float z = acc[i][j][r];
                if (FP8) z = z * sx * a.w_scales[col + r];
                z += bias_at(a, col + r);
                if constexpr (SWIGLU) {
                    float up = acc[i][1][r];
                    if (FP8) up = up * sx * a.w_scales[a.n + col + r];
                    up += bias_at(a, a.n + col + r);
                    z = z / (1.0f + expf(-z)) * up;
                } else {
                    z = activate(z, a.activation);
                }
                if (a.residual != nullptr) z += bf16_to_f32(a.residual[t * a.n + col + r]);
                y[r] = z;
            }
            uint2 packed = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
            *reinterpret_cast<uint2*>(a.output + t * a.n + col) = packed;
        }
    }
}

}  // namespace

int64_t linear_scratch_bytes(const LinearArgs&) { return 0; }

int launch_linear(const LinearArgs& a, void*, hipStream_t stream) {
    const bool swiglu = a.activation == MOE_ACT_SWIGLU;
    const int cols = swiglu ? kTile / 2 : kTile;
    const dim3 grid(static_cast<unsigned>((a.n + cols - 1) / cols), static_cast<unsigned>((a.tokens + kTile - 1) / kTile));
    if (a.fp8)
        (swiglu ? linear_tile_kernel<true, true> : linear_tile_kernel<true, false>)<<<grid, 256, 0, stream>>>(a);
    else
        (swiglu ? linear_tile_kernel<false, true> : linear_tile_kernel<false, false>)<<<grid, 256, 0, stream>>>(a);
    return check_launch("linear");
}

}  // namespace moe
