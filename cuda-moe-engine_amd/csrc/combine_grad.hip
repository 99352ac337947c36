// Gradients of the transport.
//
//   out_t = sum_k w_tk y[inverse_tk]:  dy[inverse_tk] = w_tk dout_t,  dw_tk = <dout_t, y[inverse_tk]>
//
// One pass: a wave takes a token, reads its dout row once, and each of its K expert rows
// once, writing the row's gradient and keeping K running sums in fp32; the lanes' sums
// meet by shuffles in one order. Bound by the bytes: K rows read and K written a token
// (4096 tokens, top-2, rows of 2048 bf16: 84 MB in 17.5 us beside the dispatch's gradient,
// 14.6 alone, 5.7 TB/s). Four rows in flight a lane instead of two took 22.1 us.
// Every packed row that holds no assignment gets a zero gradient, so that a program's
// expert backward may run over whole spans; with 64 experts and spans of 128 rows that is
// half of the rows (8192 assignments of 4096 in 16384 rows: 155 us with two bytes a lane
// and 64 blocks, 59 with 16 bytes, 55 with 256 blocks).
#include <algorithm>

#include "moe_common.h"

namespace moe {

template <int DT, int VE, int K>
__global__ __launch_bounds__(256) void combine_grad_kernel(
    const typename Elem<DT>::T* __restrict__ grad_output, const typename Elem<DT>::T* __restrict__ y,
    const int32_t* __restrict__ inverse, const float* __restrict__ weights, const int32_t* __restrict__ counts,
    const int32_t* __restrict__ offsets, typename Elem<DT>::T* __restrict__ grad_y, float* __restrict__ grad_weights,
    int64_t tokens, int64_t hidden, int topk, int experts, int64_t rows, int64_t token_blocks) {
    using T = typename Elem<DT>::T;
    using V = Unaligned<T, VE>;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (blockIdx.x >= token_blocks) {
        // The gaps behind each expert's assignments and behind the last span: wave w of
        // these blocks takes rows w, w + waves, ... of each. Lane e reads expert e's gap.
        const int64_t waves = (static_cast<int64_t>(gridDim.x) - token_blocks) * 4;
        const int64_t self = (static_cast<int64_t>(blockIdx.x) - token_blocks) * 4 + wave;
        int lane_from = 0, lane_to = 0;
        if (lane < experts) {
            lane_to = offsets[lane + 1];
            lane_from = min(offsets[lane] + counts[lane], lane_to);
        }
        const int end = offsets[experts];
        for (int e = 0; e <= experts; ++e) {
            const int64_t from = e < experts ? __shfl(lane_from, e) : end;
            const int64_t to = e < experts ? __shfl(lane_to, e) : rows;
            for (int64_t r = (from > 0 ? from : 0) + self; r < to && r < rows; r += waves) {
                T* dst = grad_y + r * hidden;
                const V zeros = {};
                for (int64_t v = lane; v < hidden / VE; v += 64) *reinterpret_cast<V*>(dst + v * VE) = zeros;
                const int64_t j = hidden / VE * VE + lane;
                if (j < hidden) dst[j] = Elem<DT>::store(0.0f);
            }
        }
        return;
    }
    const int64_t t = static_cast<int64_t>(blockIdx.x) * 4 + wave;
    if (t >= tokens) return;
    float w[K], dot[K];
    int64_t row[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        w[k] = dot[k] = 0.0f;
        row[k] = -1;
        if (k < topk) {
            const int r = inverse[t * topk + k];
            w[k] = weights[t * topk + k];
            row[k] = r >= 0 && r < rows ? r : -1;
        }
    }
    const T* g = grad_output + t * hidden;
    const int64_t vectors = hidden / VE;
    for (int64_t v = lane; v < vectors; v += 64) {
        const V go = *reinterpret_cast<const V*>(g + v * VE);
        V in[K];
#pragma unroll
        for (int k = 0; k < K; ++k)
            if (row[k] >= 0) in[k] = *reinterpret_cast<const V*>(y + row[k] * hidden + v * VE);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (row[k] < 0) continue;
            V o;
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float f = Elem<DT>::load(go.v[j]);
                dot[k] += f * Elem<DT>::load(in[k].v[j]);
                o.v[j] = Elem<DT>::store_product(w[k], f);
            }
            *reinterpret_cast<V*>(grad_y + row[k] * hidden + v * VE) = o;
        }
    }
    const int64_t j = vectors * VE + lane;  // fewer than VE <= 64 elements are left
    if (j < hidden) {
        const float f = Elem<DT>::load(g[j]);
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (row[k] < 0) continue;
            dot[k] += f * Elem<DT>::load(y[row[k] * hidden + j]);
            grad_y[row[k] * hidden + j] = Elem<DT>::store_product(w[k], f);
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) dot[k] += __shfl_xor(dot[k], d);
        if (lane == 0 && k < topk) grad_weights[t * topk + k] = dot[k];
    }
}

template <int DT>
static int combine_grad_typed(const void* grad_output, const void* y, const int32_t* inverse, const float* weights,
                              const int32_t* counts, const int32_t* offsets, void* grad_y, float* grad_weights,
                              int64_t tokens, int64_t hidden, int topk, int experts, int64_t rows, hipStream_t stream) {
    using T = typename Elem<DT>::T;
    constexpr int VE = 16 / static_cast<int>(sizeof(T));
    const int64_t token_blocks = (tokens + 3) / 4;
    const int64_t spare = rows - tokens * topk;
    // One block also where every row should be taken: ids out of range leave some free.
    const int64_t pad_blocks = std::clamp<int64_t>((spare + 3) / 4, 1, 256);
    const auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(token_blocks + pad_blocks)), dim3(256), 0, stream,
                           static_cast<const T*>(grad_output), static_cast<const T*>(y), inverse, weights, counts,
                           offsets, static_cast<T*>(grad_y), grad_weights, tokens, hidden, topk, experts, rows,
                           token_blocks);
        return check_launch("combine_grad_kernel");
    };
    if (topk == 1) return run(combine_grad_kernel<DT, VE, 1>);
    if (topk == 2) return run(combine_grad_kernel<DT, VE, 2>);
    if (topk <= 4) return run(combine_grad_kernel<DT, VE, 4>);
    return run(combine_grad_kernel<DT, VE, 8>);
}

int launch_combine_grad(const void* grad_output, const void* y, int dtype, const int32_t* inverse, const float* weights,
                        const int32_t* counts, const int32_t* offsets, void* grad_y, float* grad_weights, int64_t tokens,
                        int64_t hidden, int topk, int experts, int64_t rows, hipStream_t stream) {
    const auto run = [&](auto f) {
        return f(grad_output, y, inverse, weights, counts, offsets, grad_y, grad_weights, tokens, hidden, topk, experts,
                 rows, stream);
    };
    if (dtype == MOE_DTYPE_F32) return run(combine_grad_typed<MOE_DTYPE_F32>);
    if (dtype == MOE_DTYPE_F16) return run(combine_grad_typed<MOE_DTYPE_F16>);
    return run(combine_grad_typed<MOE_DTYPE_BF16>);
}

}  // namespace moe
