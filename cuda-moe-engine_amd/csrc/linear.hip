// Dense products with their epilogue: y = act(x W^T + b) + residual.
//
//   bf16:  z = sum_k x_tk W_nk,   e4m3:  z = (sum_k x_tk W_nk) sx_t sw_n
//   swiglu: W holds n gate rows, then n up rows; y = silu(z_gate) z_up + residual
//
// Products accumulate in fp32 on MFMA and everything behind them stays in fp32: one rounding
// to bf16. Up to 16 rows of x are bound by the weight's bytes (linear_few_kernel: a workgroup for 16 columns, so
// outputs of fewer than 4096 columns leave CUs idle: 14336 to 1024 18.7 us, 1.6 TB/s), many by the matrix
// instructions (linear_ring.h); between them k is split over workgroups, so that every CU has
// a part, and the partial sums are joined by a second launch with the epilogue.
//
// One row of 4096 e4m3 by 2 x 14336 weight rows (SwiGLU) 22.9 us, 5.1 TB/s; 4096 rows of it 340 us, 2830 TFLOP/s;
// 4096 x 14336 x 4096 bf16 with a residual 320 us, 1500 TFLOP/s (a large library product: 1536 bf16, 3090 e4m3; all
// of these within 5% from one card to another, by its power).
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
    const uint32_t chunk = (lane >> 4) * 16;  // of each half of a line
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
    auto load = [](auto rsrc, uint32_t off, bool in) {
        return __builtin_bit_cast(intx4, __builtin_amdgcn_raw_buffer_load_b128(rsrc, in ? off : kPast, 0u, 0));
    };
    // Workgroups start at different k: rows a multiple of 4 KiB apart lie on the same memory channels, and in step
    // all CUs would read the same ones (2 x 14336 rows of 4096 e4m3, one row of x: 24.5 -> 23.9 us).
    const int turn = static_cast<int>(blockIdx.x) % steps;
    for (int s0 = wave; s0 < steps; s0 += WAVES * UNROLL) {
        intx4 w[UNROLL][WF][2], x[UNROLL][XF][2];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int s = s0 + u * WAVES;
            if (s < steps) {
                const uint32_t at = static_cast<uint32_t>(s + turn < steps ? s + turn : s + turn - steps) * kStageBytes;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const bool in = at + chunk + h * 64 < p.k_bytes;
#pragma unroll
                    for (int f = 0; f < WF; ++f) w[u][f][h] = load(rw, w_off[f] + h * 64 + at, in);
#pragma unroll
                    for (int f = 0; f < XF; ++f) x[u][f][h] = load(rx, x_off[f] + h * 64 + at, in && x_off[f] != kPast);
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
    with_activation<ACT>(p.activation, [&](auto act_c) {
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
            *reinterpret_cast<uint2*>(p.output + at) = finish4<FP8, decltype(act_c)::value, false>(
                z, up, FP8 ? p.x_scales[row] : 1.0f, scale, bias, up_scale, up_bias, residual);
        }
    });
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
    with_activation<ACT>(p.activation, [&](auto act_c) {
        *reinterpret_cast<uint2*>(p.output + at) = finish4<FP8, decltype(act_c)::value, false>(
            z, up, FP8 ? p.x_scales[row] : 1.0f, scale, bias, up_scale, up_bias, residual);
    });
}

void run_few(const LinearArgs& a, hipStream_t stream) {
    const int steps = static_cast<int>((a.k_bytes + kStageBytes - 1) / kStageBytes);
    const unsigned grid = static_cast<unsigned>((a.n + 15) / 16);
    linear_instance(a, [&](auto act, auto fp8) {
        constexpr LinearAct ACT = decltype(act)::value;
        linear_few_kernel<decltype(fp8)::value, ACT, 1, ACT == kActSwiglu ? 2 : 1, 8, 4><<<grid, 512, 0, stream>>>(a, steps);
    });
}

// The tile shapes, and what a stage of each costs a CU: 128 bytes of k of TM + BN rows go into LDS and are read from
// there by two waves each, 3 (TM + BN) cycles at 128 bytes a cycle, about 1.25 of that as measured (128 x 128 950
// cycles, 64 x 64 470); the 256 x 256 tile alone is bound by its matrix instructions (2048 cycles).
struct TileShape {
    int tm, bn;
    int cycles;    // a stage
    int overhead;  // first loads and epilogue
};
enum Kernel { kTile64, kTile64x128, kTile96x128, kTile128, kTile256, kFew };
constexpr TileShape kShapes[] = {
    {64, 64, 470, 2500}, {64, 128, 700, 3200}, {96, 128, 830, 3900}, {128, 128, 950, 4500}, {256, 256, 2150, 13000}};

struct Choice {
    Kernel kernel;
    LinearPlan plan;
    int grid;
    bool deep;  // 128 x 128: a CU's whole LDS, where no second tile shares it and k is long (16 stages lose 0.5 us
                // of 16 by it, 64 gain 3 of 38)
};

constexpr int kCus = 256;
constexpr int64_t kMostTiles = 1 << 22;
constexpr int kJoinCycles = 6000;   // the second launch of a split product
constexpr int kJoinBytes = 1800;    // of partial sums a cycle, written and read

// The cheapest shape and split of k: tiles share a CU's LDS, so a CU takes its tiles one after the other whatever
// the ring depths are. Chosen against the best of all shapes and splits, timed: 48 x 14336 x 4096 bf16 four parts
// of 64 x 64 27 us (37 as one part a tile of 128 columns), 333 x 4096 x 4096 64 x 128 21 (27 with 64 x 64), 1024 x 4096 x
// 4096 128 x 128 35, 200 x 1000 x 2744 64 x 64 7.5 (11 with two parts), 2758 x 9344 x 2328
// bf16 256 x 256 in parts 120.
Choice choose(const LinearArgs& a) {
    Choice best{};
    best.plan.steps = static_cast<int>((a.k_bytes + kStageBytes - 1) / kStageBytes);
    best.plan.splits = 1;
    if (a.tokens <= 16) {
        best.kernel = kFew;
        return best;
    }
    const int steps = best.plan.steps;
    const bool element = a.activation != MOE_ACT_NONE && a.activation != MOE_ACT_SWIGLU;
    int64_t least = INT64_MAX;
    for (int k = kTile64; k <= kTile256; ++k) {
        const TileShape& s = kShapes[k];
        const int cols = a.activation == MOE_ACT_SWIGLU ? s.bn / 2 : s.bn;
        const int64_t row_tiles = (a.tokens + s.tm - 1) / s.tm, col_tiles = (a.n + cols - 1) / cols;
        const int64_t tiles = row_tiles * col_tiles;
        if (k != kTile256 && tiles > kMostTiles) continue;  // a workgroup each: a grid's threads stay below 2^32
        const int overhead = element ? 5 * s.overhead / 4 : s.overhead;  // an elementwise activation's part
        for (int splits = 1; splits <= 16 && 8 * splits <= std::max(steps, 8); ++splits) {
            if (splits > 1 && tiles * splits > 2 * kCus) break;
            const int part = (steps + splits - 1) / splits;
            const int64_t rounds = (tiles * splits + kCus - 1) / kCus;
            int64_t cost = rounds * (static_cast<int64_t>(part) * s.cycles + overhead);
            if (splits > 1) cost += kJoinCycles + splits * a.tokens * a.rows * 8 / kJoinBytes;
            if (cost >= least) continue;
            least = cost;
            best.kernel = static_cast<Kernel>(k);
            best.plan.row_tiles = static_cast<int>(row_tiles);
            best.plan.col_tiles = static_cast<int>(col_tiles);
            best.plan.split_steps = part;
            best.plan.splits = (steps + part - 1) / part;
            best.deep = tiles * best.plan.splits <= kCus && part >= 32;
            best.grid = static_cast<int>(
                std::min<int64_t>((tiles * best.plan.splits + kNumXcd - 1) / kNumXcd * kNumXcd, kCus));
        }
    }
    return best;
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
        case kTile64: run_dense<64, 64, 80 * 1024, false>(a, c.plan, c.grid, stream); break;
        case kTile64x128: run_dense<64, 128, 80 * 1024, false>(a, c.plan, c.grid, stream); break;
        case kTile96x128: run_dense<96, 128, 80 * 1024, false>(a, c.plan, c.grid, stream); break;
        case kTile128:
            if (c.deep)
                run_dense<128, 128, 160 * 1024, false>(a, c.plan, c.grid, stream);
            else
                run_dense<128, 128, 80 * 1024, false>(a, c.plan, c.grid, stream);
            break;
        case kTile256: run_dense<256, 256, 160 * 1024, true>(a, c.plan, c.grid, stream); break;
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
