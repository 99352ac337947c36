// Root-mean-square norm of rows, its 8-bit form, and its gradients.
//
//   h = x + residual,  rstd = 1 / sqrt(mean_j h_j^2 + eps),  y_j = h_j rstd w_j
//   8 bits: scale = max(max_j |y_j|, 2^-100) / 448,  q_j = e4m3(y_j / scale)
//   dx = rstd (g w - u mean_j(g_j w_j u_j)) + base,  dw = sum_t g u,  u = x rstd
//
// A row is read once: it waits in registers between its sum of squares, its largest value
// and its output (the norm is taken of the fp32 sum of x and residual, not of its rounded
// copy, so y is rounded once). Bound by the bytes.
#include "row_ops.h"

namespace moe {

namespace {

// 16 bytes of a row a lane.
template <int DT> constexpr int kVec = DT == MOE_DTYPE_F32 ? 4 : 8;

// OP over the WAVES waves of a row, the result in each thread; `at` alternates between the
// two halves of `lds`, so one barrier a reduction is enough.
template <typename OP, int WAVES>
__device__ __forceinline__ float row_reduce(float x, float* lds) {
    x = lanes_reduce<OP>(x);
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
        __syncthreads();
        x = lds[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) x = OP::of(x, lds[w]);
    }
    return x;
}

// Weights of the lane's columns: 1 without a weight; of the rows' type or fp32.
template <int DT, int N>
__device__ __forceinline__ void load_weights(const void* weight, bool same, int at, int n, float (&w)[N]) {
    if (weight == nullptr) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = 1.0f;
    } else if (same) {
        load_row<DT, N>(static_cast<const typename Elem<DT>::T*>(weight), at, n, w);
    } else {
        load_row<MOE_DTYPE_F32, N>(static_cast<const float*>(weight), at, n, w);
    }
}

template <int N>
__device__ __forceinline__ void store_e4m3(uint8_t* row, int at, int n, const float (&in)[N]) {
    uint32_t words[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        int word = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * i], in[4 * i + 1], 0, false);
        words[i] = __builtin_amdgcn_cvt_pk_fp8_f32(in[4 * i + 2], in[4 * i + 3], word, true);
    }
    if (at + N <= n) {
        Unaligned<uint8_t, N> v;
        __builtin_memcpy(&v, words, N);
        *reinterpret_cast<Unaligned<uint8_t, N>*>(row + at) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i < n) row[at + i] = static_cast<uint8_t>(words[i / 4] >> (8 * (i % 4)));
    }
}

// WAVES waves a row (a workgroup of max(WAVES, 4) waves takes 4 / WAVES rows), NV vectors a lane.
// NORM false: the rows are only written in 8 bits (quantize_rows).
template <int DT, int NV, int WAVES, bool QUANT, bool NORM>
__global__ __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64) void rms_norm_kernel(NormArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int N = kVec<DT>;
    constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1;
    static_assert(WAVES == 1 || WAVES >= 4, "rows share no barrier");
    __shared__ float lds[2][WAVES];
    const int thread = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + (WAVES == 1 ? threadIdx.x >> 6 : 0);
    if (row >= a.tokens) return;
    const int n = a.hidden;
    const bool same = a.weight_dtype == DT;
    const T* x = static_cast<const T*>(a.x) + row * n;
    float h[NV][N];
    float sum = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int at = (v * WAVES * 64 + thread) * N;
        if (at < n) {
            load_row<DT, N>(x, at, n, h[v]);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) h[v][i] = 0.0f;
        }
    }
    if constexpr (NORM) {
        if (a.residual != nullptr) {
            const T* r = static_cast<const T*>(a.residual) + row * n;
            T* total = static_cast<T*>(a.total) + row * n;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int at = (v * WAVES * 64 + thread) * N;
                if (at >= n) continue;
                float add[N];
                load_row<DT, N>(r, at, n, add);
#pragma unroll
                for (int i = 0; i < N; ++i) h[v][i] += add[i];
                store_row<DT, N>(total, at, n, h[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) sum += h[v][i] * h[v][i];
        sum = row_reduce<SumOp, WAVES>(sum, lds[0]);
        const float rstd = 1.0f / sqrtf(sum / static_cast<float>(n) + a.eps);
        if (a.rstd != nullptr && thread == 0) a.rstd[row] = rstd;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at >= n) continue;
            float w[N];
            load_weights<DT, N>(a.weight, same, at, n, w);
#pragma unroll
            for (int i = 0; i < N; ++i) h[v][i] = h[v][i] * rstd * w[i];
        }
    }
    float inverse = 1.0f;
    if constexpr (QUANT) {
        float most = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(h[v][i]));
        most = fmaxf(row_reduce<MaxOp, WAVES>(most, lds[1]), kLeastAmax);
        const float scale = most / kE4m3Most;
        if (thread == 0) a.scales[row] = scale;
        inverse = 1.0f / scale;
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int at = (v * WAVES * 64 + thread) * N;
        if (at >= n) continue;
        if constexpr (QUANT) {
            // The largest value may come out a rounding past 448: it is held there.
            // fmed3 would hide a NaN, which the conversion keeps.
            float q[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float y = h[v][i] * inverse;
                q[i] = fabsf(y) > kE4m3Most ? copysignf(kE4m3Most, y) : y;
            }
            store_e4m3<N>(static_cast<uint8_t*>(a.output) + row * n, at, n, q);
        } else {
            store_row<DT, N>(static_cast<T*>(a.output) + row * n, at, n, h[v]);
        }
    }
}

template <int DT, int NV, int WAVES>
void run_norm(const NormArgs& a, bool norm, hipStream_t stream) {
    constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1;
    const dim3 grid(static_cast<unsigned>((a.tokens + ROWS - 1) / ROWS)), block(WAVES < 4 ? 256 : WAVES * 64);
    if (!norm)
        rms_norm_kernel<DT, NV, WAVES, true, false><<<grid, block, 0, stream>>>(a);
    else if (a.scales != nullptr)
        rms_norm_kernel<DT, NV, WAVES, true, true><<<grid, block, 0, stream>>>(a);
    else
        rms_norm_kernel<DT, NV, WAVES, false, true><<<grid, block, 0, stream>>>(a);
}

template <int DT>
void norm_by_width(const NormArgs& a, bool norm, hipStream_t stream) {
    constexpr int lane = kVec<DT>;
    const int vectors = (a.hidden + lane - 1) / lane;  // of the row
    if (vectors <= 64) return run_norm<DT, 1, 1>(a, norm, stream);
    if (vectors <= 128) return run_norm<DT, 2, 1>(a, norm, stream);
    if (vectors <= 256) return run_norm<DT, 1, 4>(a, norm, stream);
    if (vectors <= 512) return run_norm<DT, 2, 4>(a, norm, stream);
    if (vectors <= 1024) return run_norm<DT, 4, 4>(a, norm, stream);
    if (DT != MOE_DTYPE_F32 || vectors <= 2048) return run_norm<DT, 2, 16>(a, norm, stream);
    run_norm<DT, DT == MOE_DTYPE_F32 ? 4 : 2, 16>(a, norm, stream);
}

}  // namespace

static void norm_by_type(const NormArgs& a, bool norm, hipStream_t stream) {
    if (a.dtype == MOE_DTYPE_F32)
        norm_by_width<MOE_DTYPE_F32>(a, norm, stream);
    else if (a.dtype == MOE_DTYPE_F16)
        norm_by_width<MOE_DTYPE_F16>(a, norm, stream);
    else
        norm_by_width<MOE_DTYPE_BF16>(a, norm, stream);
}

int launch_rms_norm(const NormArgs& a, hipStream_t stream) {
    norm_by_type(a, true, stream);
    return check_launch("rms_norm");
}

int launch_quantize_rows(const NormArgs& a, hipStream_t stream) {
    norm_by_type(a, false, stream);
    return check_launch("quantize_rows");
}

// -- gradients ---------------------------------------------------------------

namespace {

constexpr int kGradBlocks = 512;  // partial weight gradients

template <int DT, int NV, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void rms_norm_grad_kernel(NormGradArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int N = kVec<DT>;
    __shared__ float lds[2][WAVES];
    const int thread = threadIdx.x, n = a.hidden;
    const bool same = a.weight_dtype == DT;
    float dw[NV][N];
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int i = 0; i < N; ++i) dw[v][i] = 0.0f;
    int half = 0;
    for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x, half ^= 1) {
        const T* x = static_cast<const T*>(a.x) + row * n;
        const T* g = static_cast<const T*>(a.grad_output) + row * n;
        const float rstd = a.rstd[row];
        float u[NV][N], gw[NV][N];
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at < n) {
                load_row<DT, N>(x, at, n, u[v]);
                load_row<DT, N>(g, at, n, gw[v]);
                float w[N];
                load_weights<DT, N>(a.weight, same, at, n, w);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    u[v][i] *= rstd;
                    dw[v][i] += gw[v][i] * u[v][i];
                    gw[v][i] *= w[i];
                    dot += gw[v][i] * u[v][i];
                }
            }
        }
        if (a.grad_x != nullptr) {
            const float c = row_reduce<SumOp, WAVES>(dot, lds[half]) / static_cast<float>(n);
            const T* base = static_cast<const T*>(a.grad_x_base);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int at = (v * WAVES * 64 + thread) * N;
                if (at >= n) continue;
                float d[N];
                if (base != nullptr) {
                    load_row<DT, N>(base + row * n, at, n, d);
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) d[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < N; ++i) d[i] += rstd * (gw[v][i] - u[v][i] * c);
                store_row<DT, N>(static_cast<T*>(a.grad_x) + row * n, at, n, d);
            }
        }
    }
    if (a.grad_weight != nullptr) {
        float* part = a.scratch + static_cast<int64_t>(blockIdx.x) * n;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at < n) store_row<MOE_DTYPE_F32, N>(part, at, n, dw[v]);
        }
    }
}

// grad_weight[j] = sum of the partial rows, in order: 32 columns by 8 slices a workgroup.
__global__ __launch_bounds__(256) void column_sum_kernel(const float* __restrict__ part, float* __restrict__ out, int rows,
                                                         int n) {
    __shared__ float lds[8][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int j = blockIdx.x * 32 + col;
    float sum = 0.0f;
    if (j < n)
        for (int r = slice; r < rows; r += 8) sum += part[static_cast<int64_t>(r) * n + j];
    lds[slice][col] = sum;
    __syncthreads();
    if (slice == 0 && j < n) {
#pragma unroll
        for (int s = 1; s < 8; ++s) sum += lds[s][col];
        out[j] = sum;
    }
}

int grad_blocks(int64_t tokens) { return static_cast<int>(tokens < kGradBlocks ? tokens : kGradBlocks); }

template <int DT, int NV, int WAVES>
void run_grad(const NormGradArgs& a, hipStream_t stream) {
    rms_norm_grad_kernel<DT, NV, WAVES><<<grad_blocks(a.tokens), WAVES * 64, 0, stream>>>(a);
}

template <int DT>
void grad_by_width(const NormGradArgs& a, hipStream_t stream) {
    constexpr int lane = kVec<DT>;
    const int vectors = (a.hidden + lane - 1) / lane;
    if (vectors <= 64) return run_grad<DT, 1, 1>(a, stream);
    if (vectors <= 256) return run_grad<DT, 1, 4>(a, stream);
    if (vectors <= 512) return run_grad<DT, 2, 4>(a, stream);
    if (vectors <= 1024) return run_grad<DT, 2, 8>(a, stream);
    if (DT != MOE_DTYPE_F32 || vectors <= 2048) return run_grad<DT, 2, 16>(a, stream);
    run_grad<DT, DT == MOE_DTYPE_F32 ? 4 : 2, 16>(a, stream);
}

}  // namespace

int64_t rms_norm_backward_scratch_bytes(int64_t tokens, int64_t hidden) {
    return static_cast<int64_t>(grad_blocks(tokens)) * hidden * 4;
}

int launch_rms_norm_backward(const NormGradArgs& a, hipStream_t stream) {
    if (a.dtype == MOE_DTYPE_F32)
        grad_by_width<MOE_DTYPE_F32>(a, stream);
    else if (a.dtype == MOE_DTYPE_F16)
        grad_by_width<MOE_DTYPE_F16>(a, stream);
    else
        grad_by_width<MOE_DTYPE_BF16>(a, stream);
    if (a.grad_weight != nullptr)
        column_sum_kernel<<<(a.hidden + 31) / 32, 256, 0, stream>>>(a.scratch, a.grad_weight, grad_blocks(a.tokens),
                                                                    a.hidden);
    return check_launch("rms_norm_backward");
}

}  // namespace moe
