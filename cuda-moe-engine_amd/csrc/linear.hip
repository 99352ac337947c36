// Dense products with their epilogue: y = act(x W^T + b) + residual.
//
//   bf16:  z = sum_k x_tk W_nk,   e4m3:  z = (sum_k x_tk W_nk) sx_t sw_n
//   swiglu: W holds n gate rows, then n up rows; y = silu(z_gate) z_up + residual
//
// Products accumulate in fp32 on MFMA and everything behind them stays in fp32: one rounding
// to bf16. Few rows of x are bound by the weight's bytes (linear_few_kernel), many by the matrix
// instructions (linear_ring.h); between them k is split over workgroups, so that every CU has
// a part, and the partial sums are joined by a second launch with the epilogue.
#include <algorithm>

#include "linear_ring.h"

namespace moe {

namespace {

// Up to 16 XF rows of x: a workgroup takes 16 WF weight rows (16 gate and their 16 up rows) and
// its waves split k, stage by stage. The weight goes from memory to registers, each lane 32 bytes of a
// 128-byte line; the waves' sums meet in LDS, in order.
template <bool FP8, LinearAct ACT, int XF, int WF, int WAVES, int UNROLL>
__global__ __launch_bounds__(WAVES * 64) void linear_few_kernel(LinearArgs p, int steps) {
    constexpr bool SWIGLU = ACT == kActSwiglu;
    static_assert(!SWIGLU || WF == 2, "a gate fragment and its up fragment");
    __shared__ floatx4 sums[WAVES][XF * WF][64];
    constexpr int COLS = SWIGLU ? 16 : 16 * WF;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t col0 = static_cast<int64_t>(blockIdx.x) * COLS;
    const auto rw = make_rsrc(p.weight + col0 * p.w_stride, static_cast<uint32_t>((p.rows - col0) * p.w_stride));
    const auto rx = make_rsrc(p.x, static_cast<uint32_t>(p.tokens * p.k_bytes));
    const uint32_t chunk = (lane >> 4) * 32;
    constexpr uint32_t kPast = 0xfffffff0u;
    uint32_t w_off[WF], x_off[XF];
#pragma unroll
    for (int f = 0; f < WF; ++f) {
        const int64_t row = (SWIGLU ? f * p.n : f * 16) + (lane & 15);
        w_off[f] = static_cast<uint32_t>(row * p.w_stride + chunk);
    }
#pragma unroll
    for (int f = 0; f < XF; ++f) {
        const int64_t row = f * 16 + (lane & 15);
        x_off[f] = row < p.tokens ? static_cast<uint32_t>(row * p.k_bytes + chunk) : kPast;
    }
    floatx4 acc[XF][WF] = {};
    auto load = [](auto rsrc, uint32_t off, uint32_t at, bool in) {
        return __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, in ? off : kPast, in ? at : 0u, 0));
    };
    for (int s0 = wave; s0 < steps; s0 += WAVES * UNROLL) {
        intx4 w[UNROLL][WF][2], x[UNROLL][XF][2];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int s = s0 + u * WAVES;
            if (s < steps) {
                const uint32_t at = static_cast<uint32_t>(s) * kStageBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bool in = at + chunk + h * 16 < p.k_bytes;
#pragma unroll
                    for (int f = 0; f < WF; ++f) w[u][f][h] = load(rw, w_off[f] + h * 16 + at, 0u, in);
#pragma unroll
                    for (int f = 0; f < XF; ++f) x[u][f][h] = load(rx, x_off[f] == kPast ? kPast : x_off[f] + h * 16 + at, 0u, in);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (s0 + u * WAVES < steps) {
#pragma unroll
                for (int i = 0; i < XF; ++i)
#pragma unroll
                    for (int j = 0; j < WF; ++j) {
                        if constexpr (FP8) {
                            acc[i][j] = dense_mma<true>(DenseFrag<true>{{w[u][j][0], w[u][j][1]}},
                                                        DenseFrag<true>{{x[u][i][0], x[u][i][1]}}, acc[i][j]);
                        } else {
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                acc[i][j] = dense_mma<false>(DenseFrag<false>{{w[u][j][h]}}, DenseFrag<false>{{x[u][i][h]}},
                                                             acc[i][j]);
                        }
                    }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < XF; ++i)
#pragma unroll
        for (int j = 0; j < WF; ++j) sums[wave][i * WF + j][lane] = acc[i][j];
    __syncthreads();
    // A wave an output block.
    constexpr int BLOCKS = SWIGLU ? XF : XF * WF;
    for (int b = wave; b < BLOCKS; b += WAVES) {
        const int i = SWIGLU ? b : b / WF, j = SWIGLU ? 0 : b % WF;
        float z[4] = {}, up[4] = {};
        for (int w = 0; w < WAVES; ++w) {
            const floatx4 v = sums[w][i * WF + j][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) z[r] += v[r];
            if constexpr (SWIGLU) {
                const floatx4 g = sums[w][i * WF + 1][lane];
#pragma unroll
                for (int r = 0; r < 4; ++r) up[r] += g[r];
            }
        }
        const int64_t row = i * 16 + (lane & 15), col = col0 + j * 16 + 4 * (lane >> 4);
        if (row >= p.tokens || col >= p.n) continue;
        float scale[4], bias[4], up_scale[4] = {}, up_bias[4] = {};
        column_terms<FP8>(p, col, scale, bias);
        if constexpr (SWIGLU) column_terms<FP8>(p, p.n + col, up_scale, up_bias);
        const int64_t at = row * p.n + col;
        uint2 residual = make_uint2(0, 0);
        if (p.residual != nullptr) residual = *reinterpret_cast<const uint2*>(p.residual + at);
        *reinterpret_cast<uint2*>(p.output + at) = finish4<FP8, ACT>(
            z, up, FP8 ? p.x_scales[row] : 1.0f, scale, bias, up_scale, up_bias, p.activation, residual);
    }
}

// Joins the partial sums of k's parts, in order: four columns a thread.
template <bool FP8, LinearAct ACT>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs p, const float* __restrict__ partial, int splits) {
    constexpr bool SWIGLU = ACT == kActSwiglu;
    const int64_t quads = p.n / 4;
    const int64_t index = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (index >= p.tokens * quads) return;
    const int64_t row = index / quads, col = (index - row * quads) * 4;
    float z[4] = {}, up[4] = {};
    for (int s = 0; s < splits; ++s) {
        const float* from = partial + (s * p.tokens + row) * p.rows + col;
        const floatx4 v = *reinterpret_cast<const floatx4*>(from);
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] += v[r];
        if constexpr (SWIGLU) {
            const floatx4 g = *reinterpret_cast<const floatx4*>(from + p.n);
#pragma unroll
            for (int r = 0; r < 4; ++r) up[r] += g[r];
        }
    }
    float scale[4], bias[4], up_scale[4] = {}, up_bias[4] = {};
    column_terms<FP8>(p, col, scale, bias);
    if constexpr (SWIGLU) column_terms<FP8>(p, p.n + col, up_scale, up_bias);
    const int64_t at = row * p.n + col;
    uint2 residual = make_uint2(0, 0);
    if (p.residual != nullptr) residual = *reinterpret_cast<const uint2*>(p.residual + at);
    *reinterpret_cast<uint2*>(p.output + at) = finish4<FP8, ACT>(
        z, up, FP8 ? p.x_scales[row] : 1.0f, scale, bias, up_scale, up_bias, p.activation, residual);
}

void run_few(const LinearArgs& a, hipStream_t stream) {
    const int steps = static_cast<int>((a.k_bytes + kStageBytes - 1) / kStageBytes);
    const unsigned grid = static_cast<unsigned>((a.n + 15) / 16);
    linear_instance(a, [&](auto act, auto fp8) {
        constexpr LinearAct ACT = decltype(act)::value;
        linear_few_kernel<decltype(fp8)::value, ACT, 1, ACT == kActSwiglu ? 2 : 1, 8, 4><<<grid, 512, 0, stream>>>(a, steps);
    });
}

enum Kernel { kFew, kTile64, kTile128, kTile256 };

struct Choice {
    Kernel kernel;
    LinearPlan plan;
    int grid;
};

constexpr int kCus = 256;

Choice choose(const LinearArgs& a) {
    Choice c{};
    LinearPlan& plan = c.plan;
    plan.steps = static_cast<int>((a.k_bytes + kStageBytes - 1) / kStageBytes);
    plan.splits = 1;
    if (a.tokens <= 16) {
        c.kernel = kFew;
        return c;
    }
    const int64_t big = ((a.tokens + 255) / 256) * ((a.rows + 255) / 256);
    const int64_t mid = ((a.tokens + 127) / 128) * ((a.rows + 127) / 128);
    int tile = 64, slots = 3 * kCus;
    c.kernel = kTile64;
    if (big >= kCus) {
        tile = 256, slots = kCus;
        c.kernel = kTile256;
    } else if (mid >= kCus) {
        tile = 128, slots = 2 * kCus;
        c.kernel = kTile128;
    }
    plan.row_tiles = static_cast<int>((a.tokens + tile - 1) / tile);
    plan.col_tiles = static_cast<int>((a.rows + tile - 1) / tile);
    if (a.activation == MOE_ACT_SWIGLU) plan.col_tiles = static_cast<int>((a.n + tile / 2 - 1) / (tile / 2));
    const int64_t tiles = static_cast<int64_t>(plan.row_tiles) * plan.col_tiles;
    // At least eight stages a part.
    if (2 * tiles <= slots)
        plan.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(slots / tiles, plan.steps / 8)));
    plan.split_steps = (plan.steps + plan.splits - 1) / plan.splits;
    plan.splits = (plan.steps + plan.split_steps - 1) / plan.split_steps;
    c.grid = static_cast<int>(std::min<int64_t>(tiles * plan.splits, slots));
    c.grid = std::min((c.grid + kNumXcd - 1) / kNumXcd * kNumXcd, slots);
    return c;
}

}  // namespace

int64_t linear_scratch_bytes(const LinearArgs& a) {
    if (a.tokens == 0) return 0;
    const Choice c = choose(a);
    return c.plan.splits > 1 ? static_cast<int64_t>(c.plan.splits) * a.tokens * a.rows * 4 : 0;
}

int launch_linear(const LinearArgs& a, void* scratch, hipStream_t stream) {
    Choice c = choose(a);
    c.plan.partial = static_cast<float*>(scratch);
    switch (c.kernel) {
        case kFew: run_few(a, stream); break;
        case kTile64: run_dense<64, 64, 53 * 1024, 2>(a, c.plan, c.grid, stream); break;
        case kTile128: run_dense<128, 128, 80 * 1024, 2>(a, c.plan, c.grid, stream); break;
        case kTile256: run_dense<256, 256, 160 * 1024, 2>(a, c.plan, c.grid, stream); break;
    }
    if (c.plan.splits > 1) {
        const unsigned grid = static_cast<unsigned>((a.tokens * (a.n / 4) + 255) / 256);
        linear_instance(a, [&](auto act, auto fp8) {
            linear_join_kernel<decltype(fp8)::value, decltype(act)::value><<<grid, 256, 0, stream>>>(a, c.plan.partial,
                                                                                                    c.plan.splits);
        });
    }
    return check_launch("linear");
}

}  // namespace moe
