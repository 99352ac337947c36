// The router's training losses, and the gradients of logits, x, router weight and bias.
//
//   v = logits + bias, p = softmax(v), lse = log sum exp v, N valid tokens (mask)
//   balance = E sum_e (c_e / (N K)) (sum_t p_te / N),   z = sum_t lse_t^2 / N
//   dv_te = gb E / (N^2 K) p_te (c_e - sum_j p_tj c_j) + gz (2 / N) lse_t p_te
//         + sum_{k: ids_tk = e} w_tk (dw_tk - sum_j w_tj dw_tj),  w_t = softmax of the chosen v
//   dx = base + dv W,  dW = dv^T x,  dbias = sum_t dv
//
// The counts c are whole numbers and have no gradient. A token is a group of G lanes, one
// expert each (G the power of two from E on); the tables are a few MB at most, so these
// kernels are launch and latency. dx and dW are the skinny products of low_rank.hip with
// the experts as ranks.
#include "low_rank.h"

namespace moe {

// p and lse of one token's group of lanes; v is -inf past the experts. A token whose
// logits are all -inf has p = 0 and lse = 0; +inf or NaN logits make both NaN.
template <int G>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) {
        const float o = __shfl_xor(v, d);
        v = o > v || o != o ? o : v;  // keeps a NaN
    }
    return v;
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) v += __shfl_xor(v, d);
    return v;
}

template <int G>
__device__ __forceinline__ void group_softmax(float v, float* p, float* lse) {
    const float top = group_max<G>(v);
    if (top == -__builtin_inff()) {
        *p = 0.0f;
        *lse = 0.0f;
        return;
    }
    const float e = expf(v - top);
    const float total = group_sum<G>(e);
    *p = e / total;
    *lse = top + logf(total);
}

// A block's sums over its tokens: record[block] = p [E], z, counts [E], tokens (the
// latter as integers), or the losses themselves when it is the only block.
struct LossOut {
    float* losses;    // [2]
    int32_t* stats;   // [E + 1]: counts, valid tokens
};

// One wave, a lane per expert.
__device__ __forceinline__ void write_losses(const LossOut& out, float p, int count, float z, int n, int experts,
                                             int topk) {
    const int lane = threadIdx.x;
    const float balance = group_sum<64>(lane < experts ? static_cast<float>(count) * p : 0.0f);
    if (lane < experts) out.stats[lane] = count;
    if (lane > 0) return;
    out.stats[experts] = n;
    const float valid = static_cast<float>(n);
    out.losses[0] = n ? balance / valid * (static_cast<float>(experts) / (valid * topk)) : 0.0f;
    out.losses[1] = n ? z / valid : 0.0f;
}

template <int G>
__global__ __launch_bounds__(256) void router_loss_kernel(const float* __restrict__ logits,
                                                          const float* __restrict__ bias,
                                                          const int32_t* __restrict__ ids,
                                                          const uint8_t* __restrict__ mask, int64_t tokens, int experts,
                                                          int topk, float* __restrict__ records, LossOut out) {
    constexpr int PER = 256 / G;
    __shared__ float sp[4][64];
    __shared__ int32_t sc[4][64];
    __shared__ float sz[4];
    __shared__ int32_t sn[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e = tid % G;
    const float b = e < experts && bias ? bias[e] : 0.0f;
    float p_sum = 0.0f, z_sum = 0.0f;
    int count = 0, n = 0;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * PER + tid / G; t < tokens;
         t += static_cast<int64_t>(gridDim.x) * PER) {
        if (mask && !mask[t]) continue;  // the whole group
        const float v = e < experts ? logits[t * experts + e] + b : -__builtin_inff();
        float p, lse;
        group_softmax<G>(v, &p, &lse);
        p_sum += p;
        z_sum += lse * lse;
        ++n;
        for (int k = 0; k < topk; ++k) count += ids[t * topk + k] == e;
    }
    // The groups' sums, in one order: the groups of a wave, then the waves.
#pragma unroll
    for (int d = G; d < 64; d <<= 1) {
        p_sum += __shfl_xor(p_sum, d);
        z_sum += __shfl_xor(z_sum, d);
        count += __shfl_xor(count, d);
        n += __shfl_xor(n, d);
    }
    if (lane < G) {
        sp[wave][lane] = p_sum;
        sc[wave][lane] = count;
    }
    if (lane == 0) {
        sz[wave] = z_sum;
        sn[wave] = n;
    }
    __syncthreads();
    if (tid < experts) {
        p_sum = (sp[0][tid] + sp[1][tid]) + (sp[2][tid] + sp[3][tid]);
        count = sc[0][tid] + sc[1][tid] + sc[2][tid] + sc[3][tid];
    }
    z_sum = (sz[0] + sz[1]) + (sz[2] + sz[3]);
    n = sn[0] + sn[1] + sn[2] + sn[3];
    if (gridDim.x > 1) {
        float* r = records + static_cast<int64_t>(blockIdx.x) * (2 * experts + 2);
        int32_t* ri = reinterpret_cast<int32_t*>(r + experts + 1);
        if (tid < experts) {
            r[tid] = p_sum;
            ri[tid] = count;
        }
        if (tid == 0) {
            r[experts] = z_sum;
            ri[experts] = n;
        }
        return;
    }
    if (wave == 0) write_losses(out, p_sum, count, z_sum, n, experts, topk);
}

constexpr int kLossBlocks = 256;

__global__ __launch_bounds__(1024) void router_loss_sum_kernel(const float* __restrict__ records, int blocks, int experts,
                                                               int topk, LossOut out) {
    // Thread (part, field): the records part, part + 8, ... of one of up to 65 fields.
    __shared__ float sf[8][65];
    __shared__ int32_t si[8][65];
    const int field = threadIdx.x & 127, part = threadIdx.x >> 7;
    const int size = 2 * experts + 2;
    if (field <= experts) {
        float f = 0.0f;
        int n = 0;
        for (int r = part; r < blocks; r += 8) {
            f += records[r * size + field];
            n += reinterpret_cast<const int32_t*>(records)[r * size + experts + 1 + field];
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
template <int G>
__global__ __launch_bounds__(256) void router_logits_grad_kernel(
    const float* __restrict__ logits, const float* __restrict__ bias, const int32_t* __restrict__ ids,
    const uint8_t* __restrict__ mask, const int32_t* __restrict__ stats, const float* __restrict__ grad_losses,
    const float* __restrict__ grad_weights, int64_t tokens, int experts, int topk, float* __restrict__ grad_logits,
    float* __restrict__ bias_part) {
    constexpr int PER = 256 / G;
    __shared__ float sb[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, e = tid % G;
    const float b = e < experts && bias ? bias[e] : 0.0f;
    float balance = 0.0f, z = 0.0f, c = 0.0f;
    if (grad_losses) {
        const int n = stats[experts];
        const float valid = static_cast<float>(n);
        balance = n ? grad_losses[0] * (static_cast<float>(experts) / (valid * topk)) / valid : 0.0f;
        z = n ? grad_losses[1] * 2.0f / valid : 0.0f;
        c = e < experts ? static_cast<float>(stats[e]) : 0.0f;
    }
    float bias_sum = 0.0f;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * PER + tid / G; t < tokens;
         t += static_cast<int64_t>(gridDim.x) * PER) {
        float dv = 0.0f;
        if (!mask || mask[t]) {
            const float v = e < experts ? logits[t * experts + e] + b : -__builtin_inff();
            if (grad_losses) {
                float p, lse;
                group_softmax<G>(v, &p, &lse);
                const float mean = group_sum<G>(p * c);
                dv = p * (balance * (c - mean) + z * lse);
            }
            if (grad_weights) {
                // The chosen experts' softmax, the same terms in every lane; an id outside
                // the experts was not routed and has no term.
                float chosen[kMaxTopk], dw[kMaxTopk];
                int id[kMaxTopk];
                float top = -__builtin_inff(), total = 0.0f, dot = 0.0f;
#pragma unroll
                for (int k = 0; k < kMaxTopk; ++k) {
                    if (k >= topk) break;
                    id[k] = ids[t * topk + k];
                    dw[k] = grad_weights[t * topk + k];
                    const bool routed = static_cast<unsigned>(id[k]) < static_cast<unsigned>(experts);
                    const float vk = __shfl(v, (lane & ~(G - 1)) | (routed ? id[k] : 0));
                    chosen[k] = routed ? vk : -__builtin_inff();
                    top = chosen[k] > top || chosen[k] != chosen[k] ? chosen[k] : top;
                }
#pragma unroll
                for (int k = 0; k < kMaxTopk; ++k) {
                    if (k >= topk) break;
                    chosen[k] = chosen[k] == -__builtin_inff() ? 0.0f : chosen[k] == top ? 1.0f : expf(chosen[k] - top);
                    total += chosen[k];
                    // A chosen expert of weight 0 passes nothing on, whatever its gradient.
                    dot += chosen[k] == 0.0f ? 0.0f : chosen[k] * dw[k];
                }
                if (total != 0.0f) {
                    dot /= total;
#pragma unroll
                    for (int k = 0; k < kMaxTopk; ++k) {
                        if (k >= topk) break;
                        if (id[k] == e && chosen[k] != 0.0f) dv += chosen[k] / total * (dw[k] - dot);
                    }
                }
            }
        }
        if (e < experts) grad_logits[t * experts + e] = dv;
        bias_sum += dv;
    }
    if (!bias_part) return;
#pragma unroll
    for (int d = G; d < 64; d <<= 1) bias_sum += __shfl_xor(bias_sum, d);
    if (lane < G) sb[wave][lane] = bias_sum;
    __syncthreads();
    if (tid < experts)
        bias_part[static_cast<int64_t>(blockIdx.x) * experts + tid] =
            (sb[0][tid] + sb[1][tid]) + (sb[2][tid] + sb[3][tid]);
}

__global__ __launch_bounds__(256) void router_bias_grad_kernel(const float* __restrict__ bias_part, int blocks,
                                                               int experts, float* __restrict__ grad_bias) {
    __shared__ float s[4][64];
    const int e = threadIdx.x & 63, part = threadIdx.x >> 6;
    float f = 0.0f;
    if (e < experts)
        for (int r = part; r < blocks; r += 4) f += bias_part[r * experts + e];
    s[part][e] = f;
    __syncthreads();
    if (threadIdx.x < static_cast<unsigned>(experts)) grad_bias[e] = (s[0][e] + s[1][e]) + (s[2][e] + s[3][e]);
}

// ---------------------------------------------------------------------------
// Host launchers
// ---------------------------------------------------------------------------
static int group_lanes(int experts) {
    int g = 1;
    while (g < experts) g <<= 1;
    return g;
}

// Blocks of the token kernels: a few tokens a group, at most kLossBlocks.
static int token_blocks(int64_t tokens, int experts) {
    const int64_t per = 256 / group_lanes(experts) * 4;
    const int64_t blocks = (tokens + per - 1) / per;
    return static_cast<int>(blocks < 1 ? 1 : blocks > kLossBlocks ? kLossBlocks : blocks);
}

template <typename F>
static int by_lanes(int experts, F f) {
    switch (group_lanes(experts)) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 8: return f(std::integral_constant<int, 8>{});
        case 16: return f(std::integral_constant<int, 16>{});
        case 32: return f(std::integral_constant<int, 32>{});
        default: return f(std::integral_constant<int, 64>{});
    }
}

int64_t router_loss_scratch_bytes(int64_t tokens, int64_t experts) {
    return static_cast<int64_t>(token_blocks(tokens, static_cast<int>(experts))) * (2 * experts + 2) * 4;
}

int launch_router_loss(const float* logits, const float* bias, const int32_t* ids, const uint8_t* mask, float* losses,
                       int32_t* stats, float* records, int64_t tokens, int experts, int topk, hipStream_t stream) {
    const int blocks = token_blocks(tokens, experts);
    const LossOut out{losses, stats};
    int rc = by_lanes(experts, [&](auto g) {
        hipLaunchKernelGGL(router_loss_kernel<decltype(g)::value>, dim3(blocks), dim3(256), 0, stream, logits, bias, ids,
                           mask, tokens, experts, topk, records, out);
        return check_launch("router_loss_kernel");
    });
    if (rc != MOE_OK || blocks == 1) return rc;
    hipLaunchKernelGGL(router_loss_sum_kernel, dim3(1), dim3(1024), 0, stream, records, blocks, experts, topk, out);
    return check_launch("router_loss_sum_kernel");
}

int launch_router_logits_grad(const float* logits, const float* bias, const int32_t* ids, const uint8_t* mask,
                              const int32_t* stats, const float* grad_losses, const float* grad_weights,
                              float* grad_logits, float* bias_part, float* grad_bias, int64_t tokens, int experts,
                              int topk, hipStream_t stream) {
    const int blocks = token_blocks(tokens, experts);
    float* part = !grad_bias ? nullptr : blocks == 1 ? grad_bias : bias_part;
    int rc = by_lanes(experts, [&](auto g) {
        hipLaunchKernelGGL(router_logits_grad_kernel<decltype(g)::value>, dim3(blocks), dim3(256), 0, stream, logits,
                           bias, ids, mask, stats, grad_losses, grad_weights, tokens, experts, topk, grad_logits, part);
        return check_launch("router_logits_grad_kernel");
    });
    if (rc != MOE_OK || !grad_bias || blocks == 1) return rc;
    hipLaunchKernelGGL(router_bias_grad_kernel, dim3(1), dim3(256), 0, stream, bias_part, blocks, experts, grad_bias);
    return check_launch("router_bias_grad_kernel");
}

// Scratch of route_backward: grad_logits [T, E], bias sums, outer's partial sums.
static int64_t aligned16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

int64_t route_backward_scratch_bytes(int64_t tokens, int64_t hidden, int64_t experts) {
    const Groups g = one_group(tokens);
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
    const Groups g = one_group(tokens);
    int rc = launch_router_logits_grad(logits, bias, ids, mask, stats, grad_losses, grad_weights, grad_logits, bias_part,
                                       grad_bias, tokens, experts, topk, stream);
    if (rc == MOE_OK && grad_x)
        rc = launch_spread(grad_logits, 1, router_w, true, nullptr, g, grad_x_base, grad_x, nullptr, tokens, hidden,
                           experts, stream);
    if (rc == MOE_OK && grad_router_w)
        rc = launch_outer(grad_logits, x, nullptr, g, partials, grad_router_w, false, tokens, hidden, experts, 1, stream);
    return rc;
}

}  // namespace moe
