// Root-mean-square norm of rows, its 8-bit form, and its gradients.
//
//   h = x + residual,  rstd = 1 / sqrt(mean_j h_j^2 + eps),  y_j = h_j rstd w_j
//   8 bits: scale = max(max_j |y_j|, 2^-100) / 448,  q_j = e4m3(y_j / scale)
//   dx = rstd (g w - u mean_j(g_j w_j u_j)) + base,  dw = sum_t g u,  u = x rstd
//
// A row is read once: it waits in registers between its sum of squares, its largest value
// and its output (the norm is taken of the fp32 sum of x and residual, not of its rounded
// copy, so y is rounded once). Bound by the bytes: 8192 x 4096 bf16 with residual to 8 bits 46 us, 5.1 TB/s (as a
// copy of 1 GiB), rows alone to 8 bits 28672 x 4096 67.6 us, 5.2 TB/s; 4096 x 2048 bf16 forward 8.9 us and gradients 12.2 + 4.5 (the partial rows' sum), 3.5 TB/s in all;
// one row 3.1 us, of which two are any launch's.
#include <algorithm>

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
        typename Bytes<N>::V v;
        __builtin_memcpy(&v, words, N);
        store_bytes<N>(row + at, v);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i < n) row[at + i] = static_cast<uint8_t>(words[i / 4] >> (8 * (i % 4)));
    }
}

// WAVES waves a row, NV vectors a lane; a workgroup of four waves takes four rows at a time where a wave is enough.
// Workgroups walk the rows, the next row's loads in flight while one is summed and written.
// NORM false: the rows are only written in 8 bits (quantize_rows).
template <int DT, int NV, int WAVES, bool QUANT, bool NORM>
__global__ __launch_bounds__(WAVES < 4 ? 256 : WAVES * 64) void rms_norm_kernel(NormArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int N = kVec<DT>;
    constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1;
    static_assert(WAVES == 1 || WAVES >= 4, "rows share no barrier");
    __shared__ float lds[2][2][WAVES];
    const int thread = WAVES == 1 ? threadIdx.x & 63 : threadIdx.x;
    const int n = a.hidden;
    const int64_t stride = static_cast<int64_t>(gridDim.x) * ROWS;
    int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + (WAVES == 1 ? threadIdx.x >> 6 : 0);
    if (row >= a.tokens) return;
    using V = typename Bytes<N * sizeof(T)>::V;
    V xv[NV], rv[NV];
    const bool add = NORM && a.residual != nullptr;
    auto fetch = [&](int64_t at_row) {
        const T* x = static_cast<const T*>(a.x) + at_row * n;
        const T* r = static_cast<const T*>(a.residual) + at_row * n;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at < n) {
                xv[v] = load_vector<T, N>(x, at, n);
                if (add) rv[v] = load_vector<T, N>(r, at, n);
            }
        }
    };
    fetch(row);
    float w[NORM ? NV : 1][N];
    if constexpr (NORM) {
        const bool same = a.weight_dtype == DT;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at < n) load_weights<DT, N>(a.weight, same, at, n, w[v]);
        }
    }
    for (int turn = 0; row < a.tokens; turn ^= 1) {
        float h[NV][N];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at >= n) {
#pragma unroll
                for (int i = 0; i < N; ++i) h[v][i] = 0.0f;
                continue;
            }
            unpack<DT>(xv[v], h[v]);
            if (add) {
                float r[N];
                unpack<DT>(rv[v], r);
#pragma unroll
                for (int i = 0; i < N; ++i) h[v][i] += r[i];
            }
        }
        const int64_t this_row = row;
        row += stride;
        if (row < a.tokens) fetch(row);
        if (add) {
            T* total = static_cast<T*>(a.total) + this_row * n;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int at = (v * WAVES * 64 + thread) * N;
                if (at < n) store_row<DT, N>(total, at, n, h[v]);
            }
        }
        if constexpr (NORM) {
            float sum = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) sum += h[v][i] * h[v][i];
            sum = row_reduce<SumOp, WAVES>(sum, lds[turn][0]);
            const float rstd = 1.0f / sqrtf(sum / static_cast<float>(n) + a.eps);
            if (a.rstd != nullptr && thread == 0) a.rstd[this_row] = rstd;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const int at = (v * WAVES * 64 + thread) * N;
                    if (at < n) h[v][i] = h[v][i] * rstd * w[v][i];
                }
        }
        float inverse = 1.0f, divisor = 1.0f;
        if constexpr (QUANT) {
            float most = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < N; ++i) most = fmaxf(most, fabsf(h[v][i]));
            most = fmaxf(row_reduce<MaxOp, WAVES>(most, lds[turn][1]), kLeastAmax);
            const float scale = most / kE4m3Most;
            if (thread == 0) a.scales[this_row] = scale;
            inverse = 1.0f / scale;
            divisor = scale < __builtin_inff() ? scale : 0.0f;  // of an infinite scale 0 and NaN are left
        }
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at >= n) continue;
            if constexpr (QUANT) {
                // The quotient as division rounds it: the product's error by its remainder. (The product alone is a
                // rounding beside it, which in bf16 rows, where quotients often lie half way between two e4m3
                // values, moves one value in 5000 a step.) The largest value may come out a rounding past
                // 448: it is held there. A minimum would hide a NaN, which the conversion keeps.
                float q[N];
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float near = h[v][i] * inverse;
                    const float y = fmaf(-fmaf(near, divisor, -h[v][i]), inverse, near);  // (-0 stays -0)
                    q[i] = fabsf(y) > kE4m3Most ? copysignf(kE4m3Most, y) : y;
                }
                store_e4m3<N>(static_cast<uint8_t*>(a.output) + this_row * n, at, n, q);
            } else {
                store_row<DT, N>(static_cast<T*>(a.output) + this_row * n, at, n, h[v]);
            }
        }
    }
}

// As many workgroups as the chip holds at 32 waves a CU, an equal number of rows each.
template <int WAVES>
unsigned norm_grid(const NormArgs& a) {
    constexpr int ROWS = WAVES < 4 ? 4 / WAVES : 1;
    const int64_t blocks = (a.tokens + ROWS - 1) / ROWS, most = 256 * (WAVES < 4 ? 8 : 32 / WAVES);
    const int64_t turns = (blocks + most - 1) / most;
    return static_cast<unsigned>((blocks + turns - 1) / turns);
}

template <int DT, int NV, int WAVES>
void run_norm(const NormArgs& a, bool norm, hipStream_t stream) {
    const dim3 grid(norm_grid<WAVES>(a)), block(WAVES < 4 ? 256 : WAVES * 64);
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
    // A vector a lane where 16 waves allow it: 8 waves of one against 4 of two at 8192 x 4096 bf16 in 8
    // bits 41 against 42 us, one row 3.1 against 3.5; a wave for the whole row 94 and 9.2.
    if (vectors <= 64) return run_norm<DT, 1, 1>(a, norm, stream);
    if (vectors <= 128) return run_norm<DT, 2, 1>(a, norm, stream);
    if (vectors <= 256) return run_norm<DT, 1, 4>(a, norm, stream);
    if (vectors <= 512) return run_norm<DT, 1, 8>(a, norm, stream);
    if (vectors <= 1024) return run_norm<DT, 1, 16>(a, norm, stream);
    if (vectors <= 2048) return run_norm<DT, 2, 16>(a, norm, stream);
    if (norm) {
        if constexpr (DT == MOE_DTYPE_F32) run_norm<DT, 4, 16>(a, norm, stream);
        return;
    }
    // Rows that are only quantized may be twice as wide.
    rms_norm_kernel<DT, DT == MOE_DTYPE_F32 ? 8 : 4, 16, true, false><<<norm_grid<16>(a), 1024, 0, stream>>>(a);
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

// WAVES waves a row, NV vectors a lane. A workgroup walks rows and keeps its share of the weight's gradient in
// registers; where a lane has one vector, the weight stays there too and the next row's loads are in flight
// (with two, the registers of 16 waves do not hold that).
template <int DT, int NV, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void rms_norm_grad_kernel(NormGradArgs a) {
    using T = typename Elem<DT>::T;
    constexpr int N = kVec<DT>;
    using V = typename Bytes<N * sizeof(T)>::V;
    __shared__ float lds[2][WAVES];
    const int thread = threadIdx.x, n = a.hidden;
    const bool has_base = a.grad_x_base != nullptr && a.grad_x != nullptr;
    constexpr bool AHEAD = NV == 1;
    float dw[NV][N], kept[AHEAD ? NV : 1][N];
    V xv[NV], gv[NV], bv[AHEAD ? NV : 1];
    float rstd = 0.0f;
    auto fetch = [&](int64_t row) {
        rstd = a.rstd[row];
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at < n) {
                xv[v] = load_vector<T, N>(static_cast<const T*>(a.x) + row * n, at, n);
                gv[v] = load_vector<T, N>(static_cast<const T*>(a.grad_output) + row * n, at, n);
                if constexpr (AHEAD) {
                    if (has_base) bv[v] = load_vector<T, N>(static_cast<const T*>(a.grad_x_base) + row * n, at, n);
                }
            }
        }
    };
    int64_t row = blockIdx.x;
    if constexpr (AHEAD) fetch(row);
    const bool same = a.weight_dtype == DT;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int at = (v * WAVES * 64 + thread) * N;
        if constexpr (AHEAD) {
            if (at < n) load_weights<DT, N>(a.weight, same, at, n, kept[v]);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) dw[v][i] = 0.0f;
    }
    for (int turn = 0; row < a.tokens; turn ^= 1) {
        if constexpr (!AHEAD) fetch(row);
        float u[NV][N], gw[NV][N], d[AHEAD ? NV : 1][N];
        float dot = 0.0f;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = (v * WAVES * 64 + thread) * N;
            if (at < n) {
                float w[N];
                if constexpr (AHEAD) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        w[i] = kept[v][i];
                        d[v][i] = 0.0f;
                    }
                    if (has_base) unpack<DT>(bv[v], d[v]);
                } else {
                    load_weights<DT, N>(a.weight, same, at, n, w);
                }
                unpack<DT>(xv[v], u[v]);
                unpack<DT>(gv[v], gw[v]);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    u[v][i] *= rstd;
                    dw[v][i] += gw[v][i] * u[v][i];
                    gw[v][i] *= w[i];
                    dot += gw[v][i] * u[v][i];
                }
            }
        }
        const int64_t this_row = row;
        const float this_rstd = rstd;
        row += gridDim.x;
        if (AHEAD && row < a.tokens) fetch(row);
        if (a.grad_x != nullptr) {
            const float c = row_reduce<SumOp, WAVES>(dot, lds[turn]) / static_cast<float>(n);
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const int at = (v * WAVES * 64 + thread) * N;
                if (at >= n) continue;
                float out[N];
                if constexpr (AHEAD) {
#pragma unroll
                    for (int i = 0; i < N; ++i) out[i] = d[v][i];
                } else {
#pragma unroll
                    for (int i = 0; i < N; ++i) out[i] = 0.0f;
                    if (has_base)
                        load_row<DT, N>(static_cast<const T*>(a.grad_x_base) + this_row * n, at, n, out);
                }
#pragma unroll
                for (int i = 0; i < N; ++i) out[i] += this_rstd * (gw[v][i] - u[v][i] * c);
                store_row<DT, N>(static_cast<T*>(a.grad_x) + this_row * n, at, n, out);
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

// grad_weight[j] = sum of the partial rows, in a fixed order: 32 columns by 32 slices a workgroup, a
// slice's rows in flight together.
__global__ __launch_bounds__(1024) void column_sum_kernel(const float* __restrict__ part, float* __restrict__ out, int rows,
                                                          int n) {
    constexpr int SLICES = 32, UNROLL = 8;
    __shared__ float lds[SLICES][33];
    const int col = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int j = blockIdx.x * 32 + col;
    float sum = 0.0f;
    if (j < n) {
        for (int r0 = slice; r0 < rows; r0 += SLICES * UNROLL) {
            float v[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int r = r0 + u * SLICES;
                v[u] = r < rows ? part[static_cast<int64_t>(r) * n + j] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) sum += v[u];
        }
    }
    lds[slice][col] = sum;
    __syncthreads();
    // Half a wave a column, a lane a slice.
    const int at = blockIdx.x * 32 + slice;
    sum = lanes_reduce<SumOp, SLICES>(lds[col][slice]);
    if (col == 0 && at < n) out[at] = sum;
}

// Waves a row of the gradient kernel.
int grad_waves(int vectors) {
    if (vectors <= 64) return 1;
    if (vectors <= 128) return 2;
    if (vectors <= 256) return 4;
    return vectors <= 512 ? 8 : 16;
}

// Workgroups, each of which leaves a partial weight gradient: eight rows each, fewer where that leaves CUs
// idle (512 x 4096: 256 workgroups 10.0 us, 64 12.1), and not so many that the partial rows cost what they
// save (4096 x 2048: 512 17.3 us, 1024 19.4; 2048 x 8192: 256 27, 512 30).
int grad_blocks(int64_t tokens, int64_t hidden, int dtype) {
    const int lane = dtype == MOE_DTYPE_F32 ? 4 : 8;
    const int waves = grad_waves(static_cast<int>((hidden + lane - 1) / lane));
    const int64_t most = waves <= 2 ? 2048 / waves : waves <= 8 ? 512 : 256;
    const int64_t blocks = std::max<int64_t>(tokens / 8, std::min<int64_t>(tokens, 256));
    return static_cast<int>(std::min(blocks, most));
}

template <int DT, int NV, int WAVES>
void run_grad(const NormGradArgs& a, hipStream_t stream) {
    rms_norm_grad_kernel<DT, NV, WAVES><<<grad_blocks(a.tokens, a.hidden, a.dtype), WAVES * 64, 0, stream>>>(a);
}

template <int DT>
void grad_by_width(const NormGradArgs& a, hipStream_t stream) {
    constexpr int lane = kVec<DT>;
    const int vectors = (a.hidden + lane - 1) / lane;
    switch (grad_waves(vectors)) {
        case 1: return run_grad<DT, 1, 1>(a, stream);
        case 2: return run_grad<DT, 1, 2>(a, stream);
        case 4: return run_grad<DT, 1, 4>(a, stream);
        case 8: return run_grad<DT, 1, 8>(a, stream);
        default: break;
    }
    if (vectors <= 1024) return run_grad<DT, 1, 16>(a, stream);
    if (DT != MOE_DTYPE_F32 || vectors <= 2048) return run_grad<DT, 2, 16>(a, stream);
    run_grad<DT, DT == MOE_DTYPE_F32 ? 4 : 2, 16>(a, stream);
}

}  // namespace

int64_t rms_norm_backward_scratch_bytes(int64_t tokens, int64_t hidden, int dtype) {
    return static_cast<int64_t>(grad_blocks(tokens, hidden, dtype)) * hidden * 4;
}

int launch_rms_norm_backward(const NormGradArgs& a, hipStream_t stream) {
    if (a.dtype == MOE_DTYPE_F32)
        grad_by_width<MOE_DTYPE_F32>(a, stream);
    else if (a.dtype == MOE_DTYPE_F16)
        grad_by_width<MOE_DTYPE_F16>(a, stream);
    else
        grad_by_width<MOE_DTYPE_BF16>(a, stream);
    if (a.grad_weight != nullptr)
        column_sum_kernel<<<(a.hidden + 31) / 32, 1024, 0, stream>>>(
            a.scratch, a.grad_weight, grad_blocks(a.tokens, a.hidden, a.dtype), a.hidden);
    return check_launch("rms_norm_backward");
}

}  // namespace moe
