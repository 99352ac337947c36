// The router's training losses, and the gradients of logits, x, router weight and bias.
//
//   v = logits + bias, p = softmax(v), lse = log sum exp v, N valid tokens (mask)
//   balance = E sum_e (c_e / (N K)) (sum_t p_te / N),   z = sum_t lse_t^2 / N
//   dv_te = gb E / (N^2 K) p_te (c_e - sum_j p_tj c_j) + gz (2 / N) lse_t p_te
//         + sum_{k: ids_tk = e} w_tk (dw_tk - sum_j w_tj dw_tj),  w_t = softmax of the chosen v
//   dx = base + dv W,  dW = dv^T x,  dbias = sum_t dv
//
// The counts c are whole numbers and have no gradient. A token is a group of G lanes with
// eight experts each, in registers: the tables are a few MB at most, so these kernels are
// launch and latency, and with a lane per expert the shuffles of the softmax were most of
// it (8192 tokens of 64 experts: losses 13.9 us and logits' gradient 12.3, 5.5 and 5.3 now,
// 8.8 with the routing weights' gradient and the bias).
// dx and dW are the skinny products of low_rank.hip with the experts as ranks.
#include <algorithm>

#include "low_rank.h"

namespace moe {

constexpr int kPer = 8;  // experts per lane

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kRor8 = 0x128, kRor4 = 0x124, kRor2 = 0x122,
              kRor1 = 0x121;

__device__ __forceinline__ float max_nan(float a, float b) { return b > a || b != b ? b : a; }  // keeps a NaN

// e^x for x <= 0 (a NaN stays one): 2^t with t = x log2 e rounded, times e^(what the
// rounding left), to first order; the hardware's 2^t is good to about one rounding. Below
// -100 it is 0, as no sum it enters beside e^0 = 1 can tell.
__device__ __forceinline__ float exp_to_0(float x) {
    const float log2e = 1.44269504f, rest = 1.92596303e-8f;  // log2 e, and beyond fp32
    const float t = x * log2e;
    const float left = __builtin_fmaf(x, log2e, -t) + x * rest;
    const float y = __builtin_amdgcn_exp2f(t);
    return x < -100.0f ? 0.0f : __builtin_fmaf(y * left, 0.693147181f, y);
}

// Over the G neighbouring lanes of a token.
template <int G>
__device__ __forceinline__ float token_max(float v) {
    if constexpr (G >= 2) v = max_nan(v, dpp<kXor1>(v));
    if constexpr (G >= 4) v = max_nan(v, dpp<kXor2>(v));
    if constexpr (G >= 8) v = max_nan(v, dpp<kHalfMirror>(v));
    return v;
}
template <int G>
__device__ __forceinline__ float token_sum(float v) {
    if constexpr (G >= 2) v += dpp<kXor1>(v);
    if constexpr (G >= 4) v += dpp<kXor2>(v);
    if constexpr (G >= 8) v += dpp<kHalfMirror>(v);
    return v;
}
// Over a wave's tokens: the lanes of one place in their groups. All lanes are active.
template <int G, typename T>
__device__ __forceinline__ T wave_sum(T v) {
    v += dpp<kRor8>(v);
    if constexpr (G <= 4) v += dpp<kRor4>(v);
    if constexpr (G <= 2) v += dpp<kRor2>(v);
    if constexpr (G <= 1) v += dpp<kRor1>(v);
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
}

// This lane's eight logits of a token (with the bias), -inf past the experts.
__device__ __forceinline__ void load_logits(const float* __restrict__ row, const float (&bias)[kPer], int e0, int experts,
                                            float (&v)[kPer]) {
    using V = Unaligned<float, 4>;
    if (e0 + kPer <= experts) {
        const V a = *reinterpret_cast<const V*>(row + e0), b = *reinterpret_cast<const V*>(row + e0 + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = a.v[j] + bias[j];
            v[4 + j] = b.v[j] + bias[4 + j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) v[j] = e0 + j < experts ? row[e0 + j] + bias[j] : -__builtin_inff();
    }
}

// p and lse of a token. All logits -inf: p = 0 and lse = 0; +inf or NaN logits show in both.
template <int G>
__device__ __forceinline__ void token_softmax(const float (&v)[kPer], float (&p)[kPer], float* lse) {
    float top = v[0];
#pragma unroll
    for (int j = 1; j < kPer; ++j) top = max_nan(top, v[j]);
    top = token_max<G>(top);
    const bool some = top != -__builtin_inff();
    float total = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        p[j] = some ? exp_to_0(v[j] - top) : 0.0f;
        total += p[j];
    }
    total = token_sum<G>(total);
    const float inverse = some ? 1.0f / total : 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) p[j] *= inverse;
    *lse = some ? top + logf(total) : 0.0f;
}

struct LossOut {
    float* losses;    // [2]
    int32_t* stats;   // [E + 1]: counts, valid tokens
};

// One wave, a lane per expert.
__device__ __forceinline__ void write_losses(const LossOut& out, float p, int count, float z, int n, int experts,
                                             int topk) {
    const int lane = threadIdx.x;
    float balance = lane < experts ? static_cast<float>(count) * p : 0.0f;
    balance = wave_sum<1>(balance);
    if (lane < experts) out.stats[lane] = count;
    if (lane > 0) return;
    out.stats[experts] = n;
    const float valid = static_cast<float>(n);
    out.losses[0] = n ? balance / valid * (static_cast<float>(experts) / (valid * topk)) : 0.0f;
    out.losses[1] = n ? z / valid : 0.0f;
}

// A block's sums over its tokens: records[block] = p [E], z, counts [E], tokens (the
// latter as integers), or the losses themselves where it is the only block.
// K: the most experts a token has here.
template <int G, int K>
__global__ __launch_bounds__(256) void router_loss_kernel(const float* __restrict__ logits,
                                                          const float* __restrict__ bias,
                                                          const int32_t* __restrict__ ids,
                                                          const uint8_t* __restrict__ mask, int64_t tokens, int experts,
                                                          int topk, float* __restrict__ records, LossOut out) {
    __shared__ float sp[4][64];
    __shared__ int32_t sc[4][64];
    __shared__ float sz[4];
    __shared__ int32_t sn[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e0 = tid % G * kPer;
    float b[kPer], p_sum[kPer], z_sum = 0.0f;
    int count[kPer], n = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        b[j] = bias && e0 + j < experts ? bias[e0 + j] : 0.0f;
        p_sum[j] = 0.0f;
        count[j] = 0;
    }
    for (int64_t t = (static_cast<int64_t>(blockIdx.x) * 256 + tid) / G; t < tokens;
         t += static_cast<int64_t>(gridDim.x) * (256 / G)) {
        if (mask && !mask[t]) continue;  // the whole group
        float v[kPer], p[kPer], lse;
        int id[K];
#pragma unroll
        for (int k = 0; k < K; ++k) id[k] = k < topk ? ids[t * topk + k] : -1;
        load_logits(logits + t * experts, b, e0, experts, v);
        token_softmax<G>(v, p, &lse);
        z_sum += lse * lse;
        ++n;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            p_sum[j] += p[j];
#pragma unroll
            for (int k = 0; k < K; ++k) count[j] += id[k] == e0 + j;
        }
    }
    // A wave's tokens, then the waves.
    z_sum = wave_sum<G>(z_sum);
    n = wave_sum<G>(n);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        p_sum[j] = wave_sum<G>(p_sum[j]);
        count[j] = wave_sum<G>(count[j]);
        if (lane < G) {
            sp[wave][e0 + j] = p_sum[j];
            sc[wave][e0 + j] = count[j];
        }
    }
    if (lane == 0) {
        sz[wave] = z_sum;
        sn[wave] = n;
    }
    __syncthreads();
    if (wave > 0) return;
    float p_all = 0.0f;
    int count_all = 0;
    if (lane < experts) {
        p_all = (sp[0][lane] + sp[1][lane]) + (sp[2][lane] + sp[3][lane]);
        count_all = sc[0][lane] + sc[1][lane] + sc[2][lane] + sc[3][lane];
    }
    z_sum = (sz[0] + sz[1]) + (sz[2] + sz[3]);
    n = sn[0] + sn[1] + sn[2] + sn[3];
    if (gridDim.x == 1) {
        write_losses(out, p_all, count_all, z_sum, n, experts, topk);
        return;
    }
    float* r = records + static_cast<int64_t>(blockIdx.x) * (2 * experts + 2);
    int32_t* ri = reinterpret_cast<int32_t*>(r + experts + 1);
    if (lane < experts) {
        r[lane] = p_all;
        ri[lane] = count_all;
    }
    if (lane == 0) {
        r[experts] = z_sum;
        ri[experts] = n;
    }
}

constexpr int kLossBlocks = 256;

__global__ __launch_bounds__(1024) void router_loss_sum_kernel(const float* __restrict__ records, int blocks, int experts,
                                                               int topk, LossOut out) {
    // Thread (part, field): the records part, part + 8, ... of one of up to 65 fields,
    // eight of them in flight.
    constexpr int U = 8;
    __shared__ float sf[8][65];
    __shared__ int32_t si[8][65];
    const int field = threadIdx.x & 127, part = threadIdx.x >> 7;
    const int size = 2 * experts + 2;
    if (field <= experts) {
        float f = 0.0f;
        int n = 0;
        for (int r0 = part; r0 < blocks; r0 += 8 * U) {
            float fs[U];
            int ns[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + 8 * u;
                fs[u] = r < blocks ? records[r * size + field] : 0.0f;
                ns[u] = r < blocks ? reinterpret_cast<const int32_t*>(records)[r * size + experts + 1 + field] : 0;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                f += fs[u];
                n += ns[u];
            }
        }
        sf[part][field] = f;
        si[part][field] = n;
    }
    __syncthreads();
    if (threadIdx.x <= static_cast<unsigned>(experts)) {
        float f = sf[0][field];
        int n = si[0][field];
        for (int r = 1; r < 8; ++r) {
            f += sf[r][field];
            n += si[r][field];
        }
        sf[0][field] = f;
        si[0][field] = n;
    }
    __syncthreads();
    if (threadIdx.x < 64)
        write_losses(out, sf[0][field], si[0][field], sf[0][experts], si[0][experts], experts, topk);
}

// dv, and each block's sum over its tokens for the bias (bias_part may be null).
template <int G, int K>
__global__ __launch_bounds__(256) void router_logits_grad_kernel(
    const float* __restrict__ logits, const float* __restrict__ bias, const int32_t* __restrict__ ids,
    const uint8_t* __restrict__ mask, const int32_t* __restrict__ stats, const float* __restrict__ grad_losses,
    const float* __restrict__ grad_weights, int64_t tokens, int experts, int topk, float* __restrict__ grad_logits,
    float* __restrict__ bias_part) {
    __shared__ float sb[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e0 = tid % G * kPer;
    float b[kPer], c[kPer], bias_sum[kPer], balance = 0.0f, z = 0.0f;
    if (grad_losses) {
        const int n = stats[experts];
        const float valid = static_cast<float>(n);
        balance = n ? grad_losses[0] * (static_cast<float>(experts) / (valid * topk)) / valid : 0.0f;
        z = n ? grad_losses[1] * 2.0f / valid : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const bool held = e0 + j < experts;
        b[j] = bias && held ? bias[e0 + j] : 0.0f;
        c[j] = grad_losses && held ? static_cast<float>(stats[e0 + j]) : 0.0f;
        bias_sum[j] = 0.0f;
    }
    for (int64_t t = (static_cast<int64_t>(blockIdx.x) * 256 + tid) / G; t < tokens;
         t += static_cast<int64_t>(gridDim.x) * (256 / G)) {
        float dv[kPer] = {0, 0, 0, 0, 0, 0, 0, 0};
        const float* row = logits + t * experts;
        if (!mask || mask[t]) {
            if (grad_losses) {
                float v[kPer], p[kPer], lse, mean = 0.0f;
                load_logits(row, b, e0, experts, v);
                token_softmax<G>(v, p, &lse);
#pragma unroll
                for (int j = 0; j < kPer; ++j) mean += p[j] * c[j];
                mean = token_sum<G>(mean);
#pragma unroll
                for (int j = 0; j < kPer; ++j) dv[j] = p[j] * (balance * (c[j] - mean) + z * lse);
            }
            if (grad_weights) {
                // The chosen experts' softmax, the same terms in every lane of the token; an
                // id outside the experts was not routed and has no term.
                float chosen[K], dw[K];
                int id[K];
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    id[k] = k < topk ? ids[t * topk + k] : -1;
                    dw[k] = k < topk ? grad_weights[t * topk + k] : 0.0f;
                }
                float top = -__builtin_inff(), total = 0.0f, dot = 0.0f;
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    const bool routed = static_cast<unsigned>(id[k]) < static_cast<unsigned>(experts);
                    chosen[k] = routed ? row[id[k]] + (bias ? bias[id[k]] : 0.0f) : -__builtin_inff();
                    top = max_nan(top, chosen[k]);
                }
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    chosen[k] = chosen[k] == -__builtin_inff() ? 0.0f : chosen[k] == top ? 1.0f : exp_to_0(chosen[k] - top);
                    total += chosen[k];
                    // A chosen expert of weight 0 passes nothing on, whatever its gradient.
                    dot += chosen[k] == 0.0f ? 0.0f : chosen[k] * dw[k];
                }
                if (total != 0.0f) {
                    const float inverse = 1.0f / total;
                    dot *= inverse;
#pragma unroll
                    for (int k = 0; k < K; ++k) {
                        const float term = chosen[k] == 0.0f ? 0.0f : chosen[k] * inverse * (dw[k] - dot);
#pragma unroll
                        for (int j = 0; j < kPer; ++j) dv[j] += id[k] == e0 + j ? term : 0.0f;
                    }
                }
            }
        }
        float* dst = grad_logits + t * experts;
        if (e0 + kPer <= experts) {
            using V = Unaligned<float, 4>;
            *reinterpret_cast<V*>(dst + e0) = V{{dv[0], dv[1], dv[2], dv[3]}};
            *reinterpret_cast<V*>(dst + e0 + 4) = V{{dv[4], dv[5], dv[6], dv[7]}};
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (e0 + j < experts) dst[e0 + j] = dv[j];
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) bias_sum[j] += dv[j];
    }
    if (!bias_part) return;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        bias_sum[j] = wave_sum<G>(bias_sum[j]);
        if (lane < G) sb[wave][e0 + j] = bias_sum[j];
    }
    __syncthreads();
    if (tid < experts)
        bias_part[static_cast<int64_t>(blockIdx.x) * experts + tid] =
            (sb[0][tid] + sb[1][tid]) + (sb[2][tid] + sb[3][tid]);
}

__global__ __launch_bounds__(256) void router_bias_grad_kernel(ColumnSums bias) { sum_columns(bias); }

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
static int group_lanes(int experts) { return experts <= 8 ? 1 : experts <= 16 ? 2 : experts <= 32 ? 4 : 8; }

// Blocks of the token kernels: one for up to four rounds of its lanes, else as many as there
// are tokens for, at most kLossBlocks. The losses of 1024 lanes (1024 tokens of 8 experts) take
// 5.9 us in one block and as long in four with the second launch, 8.6 and 12.1 a call from
// Python; 2048 lanes 8.8 and 5.9, 9.1 and 12.2 a call.
static int token_blocks(int64_t tokens, int experts) {
    const int64_t lanes = tokens * group_lanes(experts);
    return lanes <= 1024 ? 1 : static_cast<int>(std::min<int64_t>((lanes + 255) / 256, kLossBlocks));
}

// f(lanes a token, most experts a token): top-1 and top-2, and the rest.
template <typename F>
static int by_shape(int experts, int topk, F f) {
    const auto with = [&](auto g) {
        return topk <= 2 ? f(g, std::integral_constant<int, 2>{}) : f(g, std::integral_constant<int, kMaxTopk>{});
    };
    switch (group_lanes(experts)) {
        case 1: return with(std::integral_constant<int, 1>{});
        case 2: return with(std::integral_constant<int, 2>{});
        case 4: return with(std::integral_constant<int, 4>{});
        default: return with(std::integral_constant<int, 8>{});
    }
}

int64_t router_loss_scratch_bytes(int64_t tokens, int64_t experts) {
    const int64_t blocks = token_blocks(tokens, static_cast<int>(experts));
    return blocks == 1 ? 0 : blocks * (2 * experts + 2) * 4;
}

int launch_router_loss(const float* logits, const float* bias, const int32_t* ids, const uint8_t* mask, float* losses,
                       int32_t* stats, float* records, int64_t tokens, int experts, int topk, hipStream_t stream) {
    const int blocks = token_blocks(tokens, experts);
    const LossOut out{losses, stats};
    int rc = by_shape(experts, topk, [&](auto g, auto k) {
        hipLaunchKernelGGL((router_loss_kernel<decltype(g)::value, decltype(k)::value>), dim3(blocks), dim3(256), 0,
                           stream, logits, bias, ids, mask, tokens, experts, topk, records, out);
        return check_launch("router_loss_kernel");
    });
    if (rc != MOE_OK || blocks == 1) return rc;
    hipLaunchKernelGGL(router_loss_sum_kernel, dim3(1), dim3(1024), 0, stream, records, blocks, experts, topk, out);
    return check_launch("router_loss_sum_kernel");
}

// With `bias` (its part set by the caller), the blocks' bias sums too: bias->blocks of them,
// left to add up, or none when the only block wrote bias->out.
int launch_router_logits_grad(const float* logits, const float* bias, const int32_t* ids, const uint8_t* mask,
                              const int32_t* stats, const float* grad_losses, const float* grad_weights,
                              float* grad_logits, ColumnSums* sums, int64_t tokens, int experts, int topk,
                              hipStream_t stream) {
    const int blocks = token_blocks(tokens, experts);
    float* part = nullptr;
    if (sums && sums->out) {
        part = blocks == 1 ? sums->out : const_cast<float*>(sums->part);
        sums->rows = blocks == 1 ? 0 : blocks;
        sums->columns = experts;
    }
    return by_shape(experts, topk, [&](auto g, auto k) {
        hipLaunchKernelGGL((router_logits_grad_kernel<decltype(g)::value, decltype(k)::value>), dim3(blocks), dim3(256),
                           0, stream, logits, bias, ids, mask, stats, grad_losses, grad_weights, tokens, experts, topk,
                           grad_logits, part);
        return check_launch("router_logits_grad_kernel");
    });
}

// Scratch of route_backward: grad_logits [T, E], bias sums, outer's partial sums.
static int64_t aligned16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

int64_t route_backward_scratch_bytes(int64_t tokens, int64_t hidden, int64_t experts) {
    const Groups g = one_group(tokens, hidden, experts);
    return aligned16(tokens * experts * 4) + aligned16(static_cast<int64_t>(kLossBlocks) * experts * 4) +
           (g.split_bound > 1 ? g.split_bound * experts * hidden * 4 : 0);
}

int launch_route_backward(const uint16_t* x, const float* router_w, const float* logits, const float* bias,
                          const int32_t* ids, const uint8_t* mask, const int32_t* stats, const float* grad_losses,
                          const float* grad_weights, const uint16_t* grad_x_base, uint16_t* grad_x, float* grad_router_w,
                          float* grad_bias, char* scratch, int64_t tokens, int64_t hidden, int experts, int topk,
                          hipStream_t stream) {
    float* grad_logits = reinterpret_cast<float*>(scratch);
    float* bias_part = reinterpret_cast<float*>(scratch + aligned16(tokens * experts * 4));
    float* partials = reinterpret_cast<float*>(scratch + aligned16(tokens * experts * 4) +
                                               aligned16(static_cast<int64_t>(kLossBlocks) * experts * 4));
    Groups g = one_group(tokens, hidden, experts);
    g.mask = mask;
    ColumnSums sums;
    sums.part = bias_part;
    sums.out = grad_bias;
    int rc = launch_router_logits_grad(logits, bias, ids, mask, stats, grad_losses, grad_weights, grad_logits, &sums,
                                       tokens, experts, topk, stream);
    if (rc == MOE_OK && grad_x)
        rc = launch_spread(grad_logits, 1, router_w, true, nullptr, g, grad_x_base, grad_x, nullptr, tokens, hidden,
                           experts, stream);
    // The bias' last sums ride on the weight gradient's, where there is one.
    const bool apart = sums.rows > 0 && (!grad_router_w || g.split_bound == 1);
    if (rc == MOE_OK && grad_router_w)
        rc = launch_outer({grad_logits, x, partials, grad_router_w, hidden}, {}, nullptr, g, false, tokens, experts, 1,
                          stream, apart ? ColumnSums{} : sums);
    if (rc == MOE_OK && apart) {
        hipLaunchKernelGGL(router_bias_grad_kernel, dim3(1), dim3(256), 0, stream, sums);
        rc = check_launch("router_bias_grad_kernel");
    }
    return rc;
}

}  // namespace moe
