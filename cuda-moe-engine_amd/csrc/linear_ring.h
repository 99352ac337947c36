// Tiles of the dense products (linear.h): operands through an LDS ring, four waves a workgroup.
//
// Work is counted in bytes: a stage is 128 bytes of k of TM rows of x and BN rows of the weight, 64 bf16 or 128
// e4m3, so both types move the same lines and differ in the matrix instruction alone (two
// 16x16x32 bf16 steps or one 16x16x128 e4m3 step a stage, of the same duration).
//
//  * buffer_load ... lds moves 8 rows of one 128-byte line a wave instruction. Rows past the
//    operand's end read as zero through the resource's range; chunks past K in the last stage
//    by an offset past every range, so padding between rows never enters a sum.
//  * Chunk c (16 bytes) of LDS row r lies at chunk c ^ ((r >> 1) & 7): 16 rows read at one chunk
//    touch all banks once.
//  * One barrier a stage. A stage's fragments are read between the matrix instructions of the step
//    before, its slot is refilled from the barrier on that follows its last read.
//  * Persistent workgroups chain tiles: the last windows of one load the next one's first stages.
#pragma once

#include "linear.h"

namespace moe {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef int intx8 __attribute__((ext_vector_type(8)));

constexpr int kStageBytes = 128;
constexpr int kRingWaves = 4;

// A launch's tiles: row tiles fastest, then column tiles, then splits of k.
struct LinearPlan {
    int row_tiles;
    int col_tiles;
    int splits;       // parts of k; more than one: partial sums in `partial`
    int steps;        // stages of a whole row
    int split_steps;  // stages of a part (the last may have fewer)
    float* partial;   // [splits, T, rows] fp32
};

struct LinearTile {
    bool valid;
    int row0, col0, step0, steps, split;  // col0 in weight rows (of the gate half)
};

__device__ __forceinline__ int ring_swizzle(int row) { return (row >> 1) & 7; }

constexpr int dense_stages(uint32_t stage_a, uint32_t stage_b, uint32_t bytes, int cap) {
    const int fit = static_cast<int>(bytes / (stage_a + stage_b));
    return fit < cap ? fit : cap;
}

// What the epilogue applies: nothing, one of the elementwise activations, or the gated one.
enum LinearAct { kActNone, kActElement, kActSwiglu };

template <int TM_, int BN_, LinearAct ACT_, bool FP8_, uint32_t LDS_, bool CHAIN_, int WC_ = 2, int CAP = 6>
struct DenseShape {
    static constexpr int TM = TM_, BN = BN_, WC = WC_;
    static constexpr LinearAct ACT = ACT_;
    // Persistent workgroups that chain tiles, or a workgroup a tile.
    static constexpr bool CHAIN = CHAIN_;
    static constexpr bool SWIGLU = ACT == kActSwiglu, FP8 = FP8_;
    static constexpr uint32_t LDS = LDS_;
    static constexpr int COLS = SWIGLU ? BN / 2 : BN;  // output columns of a tile
    static constexpr int WTM = TM / (kRingWaves / WC), WTN = BN / WC;
    static constexpr int FA = WTM / 16, FB = WTN / 16;
    static constexpr int A_LOADS = TM / 8 / kRingWaves, B_LOADS = BN / 8 / kRingWaves, LOADS = A_LOADS + B_LOADS;
    static constexpr uint32_t A_STAGE = TM * kStageBytes, B_STAGE = BN * kStageBytes;
    // Three or more whole stages where they fit, else two of x and what fits of the weight.
    static constexpr int EQUAL = dense_stages(A_STAGE, B_STAGE, LDS, CAP);
    static constexpr int SB = EQUAL >= 3 ? EQUAL : static_cast<int>((LDS - 2 * A_STAGE) / B_STAGE);
    static constexpr int SA = EQUAL >= 3 ? EQUAL : 2;
    static constexpr uint32_t B_BASE = SA * A_STAGE;
    static constexpr uint32_t FRAG = 16 * kStageBytes;
    // Loads younger than a stage's own when its first read waits for it: A of stage u + SA, then B of
    // stage u + SB are issued in each window.
    static constexpr int VM_STEADY = (SB > SA ? B_LOADS : 0) + (SA - 2) * LOADS;
    static constexpr int VM_FIRST = (SB > SA ? B_LOADS : 0) + (SA - 1) * LOADS;
    // 16-byte stores of a tile's epilogue, none of them behind a branch: as many operations at least are younger than
    // the next tile's first loads, which go out before them.
    static constexpr int STORES = CHAIN ? FA * (SWIGLU ? FB / 2 : FB) / 2 : 0;
    static_assert(A_LOADS >= 1 && B_LOADS >= 1 && FA >= 1 && FB >= 2 && FB % 2 == 0, "tile shape");
    static_assert(SA >= 2 && SB >= SA && SA * A_STAGE + SB * B_STAGE <= LDS, "ring does not fit");
    static_assert(VM_FIRST + STORES < 64, "loads in flight fit the counter");
    static_assert(!CHAIN || FB % 4 == 0, "stores in pairs of blocks");
};

template <typename S>
struct DenseLoads {
    __amdgpu_buffer_rsrc_t ra, rb;
    uint32_t a_off[S::A_LOADS], b_off[S::B_LOADS];
    char* lds;
    int wave;
    bool in_tail[2];  // the lane's chunk of even and odd row groups lies below K in a row's last stage

    struct Rsrc {
        __amdgpu_buffer_rsrc_t a, b;
    };
    static __device__ __forceinline__ Rsrc resources(const LinearArgs& p, const LinearTile& t) {
        const int64_t skip = static_cast<int64_t>(t.step0) * kStageBytes;
        const int64_t rows = min<int64_t>(p.tokens - t.row0, S::TM);
        Rsrc r;
        r.a = make_rsrc(p.x + t.row0 * p.k_bytes + skip, static_cast<uint32_t>(rows * p.k_bytes - skip));
        r.b = make_rsrc(p.weight + t.col0 * p.w_stride + skip,
                        static_cast<uint32_t>((p.rows - t.col0) * p.w_stride - skip));
        return r;
    }
    __device__ __forceinline__ DenseLoads(const LinearArgs& p, char* lds_, const Rsrc& r) : lds(lds_) {
        const int lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        ra = r.a;
        rb = r.b;
        const int lrow = lane >> 3, chunk = lane & 7;
        const int tail = static_cast<int>((p.k_bytes - 1) % kStageBytes) + 1;
#pragma unroll
        for (int g = 0; g < 2; ++g) in_tail[g] = (chunk ^ ring_swizzle(8 * g + lrow)) * 16 < tail;
#pragma unroll
        for (int i = 0; i < S::A_LOADS; ++i) {
            const int row = (wave * S::A_LOADS + i) * 8 + lrow;
            a_off[i] = static_cast<uint32_t>(row * p.k_bytes + (chunk ^ ring_swizzle(row)) * 16);
        }
#pragma unroll
        for (int i = 0; i < S::B_LOADS; ++i) {
            const int row = (wave * S::B_LOADS + i) * 8 + lrow;
            int64_t from = row;
            if constexpr (S::SWIGLU) {
                // A wave's columns: WTN / 2 gate rows, then their up rows.
                const int half = S::WTN / 2, col = row / S::WTN * half + row % half;
                from = row % S::WTN < half ? col : p.n + col;
            }
            b_off[i] = static_cast<uint32_t>(from * p.w_stride + (chunk ^ ring_swizzle(row)) * 16);
        }
    }
    // Load l of stage kt into slot st. `last`: stage kt ends the rows.
    __device__ __forceinline__ void issue_a(__amdgpu_buffer_rsrc_t r, int kt, int st, int l, bool last) const {
        const int g = wave * S::A_LOADS + l;
        dma16(r, lds + st * S::A_STAGE + g * 1024, offset(a_off[l], kt, g, last), static_cast<uint32_t>(kt) * kStageBytes);
    }
    __device__ __forceinline__ void issue_b(__amdgpu_buffer_rsrc_t r, int kt, int st, int l, bool last) const {
        const int g = wave * S::B_LOADS + l;
        dma16(r, lds + S::B_BASE + st * S::B_STAGE + g * 1024, offset(b_off[l], kt, g, last),
              static_cast<uint32_t>(kt) * kStageBytes);
    }
    __device__ __forceinline__ uint32_t offset(uint32_t off, int kt, int g, bool last) const {
        // (Both places by name: with an odd number of loads a wave the parity is the wave's, and an index into two
        // flags would put them in memory.)
        const bool in = g & 1 ? in_tail[1] : in_tail[0];
        return last && !in ? 0xfffffff0u - static_cast<uint32_t>(kt) * kStageBytes : off;
    }
    // The loads of the windows before stage 0, in the loop's order (only the last window's when
    // `chained`: the others went out in the tile before). Stages past the end load the last one again,
    // so that every window counts the same loads.
    __device__ __forceinline__ void prologue(int steps, bool ends, int a0, int b0, bool chained) const {
#pragma unroll
        for (int v = -S::SB; v < 0; ++v) {
            if (chained && v != -1) continue;
            if (v + S::SA >= 0) {
                const int st = a0 + v + S::SA >= S::SA ? a0 + v : a0 + v + S::SA, kt = min(v + S::SA, steps - 1);
#pragma unroll
                for (int l = 0; l < S::A_LOADS; ++l) issue_a(ra, kt, st, l, ends && kt == steps - 1);
            }
            const int st = b0 + v + S::SB >= S::SB ? b0 + v : b0 + v + S::SB, kt = min(v + S::SB, steps - 1);
#pragma unroll
            for (int l = 0; l < S::B_LOADS; ++l) issue_b(rb, kt, st, l, ends && kt == steps - 1);
        }
    }
};

// One 16-row fragment of the current step: 16 bytes a lane (bf16) or 32 (e4m3).
template <bool FP8>
struct DenseFrag {
    intx4 h[FP8 ? 2 : 1];
};

template <bool FP8>
__device__ __forceinline__ floatx4 dense_mma(const DenseFrag<FP8>& w, const DenseFrag<FP8>& x, floatx4 acc) {
    if constexpr (FP8) {
        const intx8 a = __builtin_shufflevector(w.h[0], w.h[1], 0, 1, 2, 3, 4, 5, 6, 7);
        const intx8 b = __builtin_shufflevector(x.h[0], x.h[1], 0, 1, 2, 3, 4, 5, 6, 7);
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, 0, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, w.h[0]),
                                                       __builtin_bit_cast(bf16x8_t, x.h[0]), acc, 0, 0, 0);
    }
}

// -- epilogue ----------------------------------------------------------------

// z / (1 + e^-z) and its like: hardware exp2 and reciprocal, about 1 ulp each and the rounding of the
// exponent, below 2e-6 of the value up to |z| of 30 (where e^-|z| is gone), before bf16's 4e-3.
__device__ __forceinline__ float sigmoid_times(float z, float u) {
    return z * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(u * -1.4426950408889634f));
}

// z Phi(z): with a = |z| / sqrt 2 and t = 1 / (1 + a / 2), erfc(a) = t P(t) e^(-a^2), P of degree 8 by weighted
// least squares over a in [0, 12] (within 3e-7 of erfc in fp32), so that the negative side, where
// 1 + erf cancels, keeps its relative precision.
__device__ __forceinline__ float gelu_erf(float z) {
    const float a = fabsf(z) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.5f * a);
    float p = -0.05936202353897773f;
    p = p * t + 0.28600591597164415f;
    p = p * t - 0.4901644081133491f;
    p = p * t + 0.28145938040851415f;
    p = p * t - 0.028961970795025077f;
    p = p * t + 0.20367457674410538f;
    p = p * t + 0.24285453204440827f;
    p = p * t + 0.2824094757421122f;
    p = p * t + 0.2820844776905523f;
    const float q = 0.5f * t * p * __builtin_amdgcn_exp2f(a * a * -1.4426950408889634f);
    return z * (z < 0.0f ? q : 1.0f - q);  // of infinity 1, and no difference of two infinities
}

template <int ACT>
__device__ __forceinline__ float activated(float z) {
    if constexpr (ACT == MOE_ACT_RELU) return z < 0.0f ? 0.0f : z;  // NaN stays
    if constexpr (ACT == MOE_ACT_SILU) return sigmoid_times(z, z);
    if constexpr (ACT == MOE_ACT_GELU) return gelu_erf(z);
    // z / 2 (1 + tanh u) = z / (1 + e^-2u)
    if constexpr (ACT == MOE_ACT_GELU_TANH) return sigmoid_times(z, 1.5957691216057308f * (z + 0.044715f * z * z * z));
    return z;
}

// f(constant<activation>) of a kernel whose kind of activation is KIND. The choice is made here, outside of an
// epilogue's loops: made for each value, the code of 256 x 256 values and four activations does not stay in the
// instruction cache (12995 rows, k 448, 13232 columns, e4m3 with silu: 315 -> 220 us).
template <LinearAct KIND, typename F>
__device__ __forceinline__ void with_activation(int act, const F& f) {
    if constexpr (KIND == kActElement) {
        if (act == MOE_ACT_RELU)
            f(std::integral_constant<int, MOE_ACT_RELU>{});
        else if (act == MOE_ACT_SILU)
            f(std::integral_constant<int, MOE_ACT_SILU>{});
        else if (act == MOE_ACT_GELU)
            f(std::integral_constant<int, MOE_ACT_GELU>{});
        else
            f(std::integral_constant<int, MOE_ACT_GELU_TANH>{});
    } else if constexpr (KIND == kActSwiglu) {
        f(std::integral_constant<int, MOE_ACT_SWIGLU>{});
    } else {
        f(std::integral_constant<int, MOE_ACT_NONE>{});
    }
}

// Columns col .. col + 3 of the weight row set at `base`: scales (1 for bf16) and bias (0 without).
template <bool FP8>
__device__ __forceinline__ void column_terms(const LinearArgs& p, int64_t row, float (&scale)[4], float (&bias)[4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        scale[r] = 1.0f;
        bias[r] = 0.0f;
    }
    if constexpr (FP8) {
        const auto v = *reinterpret_cast<const Unaligned<float, 4>*>(p.w_scales + row);
#pragma unroll
        for (int r = 0; r < 4; ++r) scale[r] = v.v[r];
    }
    if (p.bias != nullptr) {
        if (p.bias_bf16) {
            const auto v = *reinterpret_cast<const Unaligned<uint16_t, 4>*>(static_cast<const uint16_t*>(p.bias) + row);
#pragma unroll
            for (int r = 0; r < 4; ++r) bias[r] = bf16_to_f32(v.v[r]);
        } else {
            const auto v = *reinterpret_cast<const Unaligned<float, 4>*>(static_cast<const float*>(p.bias) + row);
#pragma unroll
            for (int r = 0; r < 4; ++r) bias[r] = v.v[r];
        }
    }
}

// Four columns of one row of x: sums to bf16, with bias and the residual's four values. Without them (PLAIN) neither
// is added: an epilogue of 256 x 256 is 128 or 256 values a lane, a tenth of a tile of 32 stages.
template <bool FP8, int ACT, bool PLAIN>
__device__ __forceinline__ uint2 finish4(const float (&z)[4], const float (&up)[4], float sx, const float (&scale)[4],
                                         const float (&bias)[4], const float (&up_scale)[4], const float (&up_bias)[4],
                                         uint2 residual) {
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float v = FP8 ? z[r] * sx * scale[r] : z[r];  // (the product of the scales alone may leave fp32)
        if constexpr (!PLAIN) v += bias[r];
        if constexpr (ACT == MOE_ACT_SWIGLU) {
            float u = FP8 ? up[r] * sx * up_scale[r] : up[r];
            if constexpr (!PLAIN) u += up_bias[r];
            y[r] = sigmoid_times(v, v) * u;
        } else {
            y[r] = activated<ACT>(v);
        }
    }
    if constexpr (!PLAIN) {
        y[0] += __uint_as_float(residual.x << 16);
        y[1] += __uint_as_float(residual.x & 0xffff0000u);
        y[2] += __uint_as_float(residual.y << 16);
        y[3] += __uint_as_float(residual.y & 0xffff0000u);
    }
    return make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
}

// What the epilogue reads: the scales of the lane's rows, its columns' terms, and the residual (of two rows at a time
// where tiles are chained). Rows past the end and columns past it (kPastColumns) read as zero through the
// resource's range.
constexpr uint32_t kPastColumns = 0xd0000000u;  // past every range, and a row's offset (below 2^29) added to it as well
template <typename S>
struct DenseExtra {
    static constexpr int OUT = S::SWIGLU ? S::FB / 2 : S::FB;
    static constexpr int KEPT = S::CHAIN ? 2 : S::FA;
    uint32_t residual[KEPT * OUT * 2];
    float sx[S::FA];
    float scale[OUT][4], bias[OUT][4], up_scale[S::SWIGLU ? OUT : 1][4], up_bias[S::SWIGLU ? OUT : 1][4];

    __device__ __forceinline__ void load_columns(const LinearArgs& p, int64_t col0) {
        static_for<OUT>([&](auto j_c) {
            constexpr int j = decltype(j_c)::value;
            const int64_t col = min(col0 + j * 16, p.n - 4);
            column_terms<S::FP8>(p, col, scale[j], bias[j]);
            if constexpr (S::SWIGLU) column_terms<S::FP8>(p, p.n + col, up_scale[j], up_bias[j]);
        });
    }
    __device__ __forceinline__ void load_scales(const LinearArgs& p, const LinearTile& t, int row) {
        if constexpr (S::FP8) {
            const auto r = make_rsrc(p.x_scales + t.row0, static_cast<uint32_t>(min<int64_t>(p.tokens - t.row0, S::TM) * 4));
#pragma unroll
            for (int i = 0; i < S::FA; ++i)
                sx[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, (row + i * 16) * 4, 0, 0));
        } else {
#pragma unroll
            for (int i = 0; i < S::FA; ++i) sx[i] = 1.0f;
        }
    }
    // Row fragment I at byte `at` of the tile's rows, columns from col on.
    template <int I>
    __device__ __forceinline__ void load_row(const LinearArgs& p, __amdgpu_buffer_rsrc_t r, uint32_t at, int col) {
        static_for<OUT>([&](auto j_c) {
            constexpr int j = decltype(j_c)::value;
            const uint32_t c = col + j * 16 < p.n ? static_cast<uint32_t>(col + j * 16) * 2 : kPastColumns;
            const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, at + c, 0, 0);
            residual[(I % KEPT * OUT + j) * 2] = v[0];
            residual[(I % KEPT * OUT + j) * 2 + 1] = v[1];
        });
    }
};
// A tile's rows of the residual or the output; none where there is no residual.
template <typename S>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t tile_rows(const LinearArgs& p, const LinearTile& t, const uint16_t* of) {
    const int64_t rows = min<int64_t>(p.tokens - t.row0, S::TM);
    return make_rsrc(of + t.row0 * p.n, of != nullptr ? static_cast<uint32_t>(rows * p.n * 2) : 0u);
}

__device__ __forceinline__ void to_vgpr(floatx4& v) { asm volatile("" : "+v"(v)); }

// One tile. Its prologue has been issued (`CHAIN`; else it goes out here, behind the epilogue's operands, whose
// latency then hides behind the product); `after`: the stores of the tile before may be in flight (they share the
// loads' counter, and were issued after these, so that a wait may leave them out: this and a tile's row
// scales in one load instead of eight, each behind the row's stores before it, took 4096 x 4096 x 28672 e4m3 with SwiGLU from
// 370 to 355 us in one session). With `chain` the last windows load the first stages of the next tile (resources
// `next`), otherwise its whole prologue goes out in `hook`, once every wave is done with the ring.
template <typename S, typename Hook>
__device__ __forceinline__ void dense_tile(const LinearArgs& p, const LinearPlan& plan, char* lds, const LinearTile& t,
                                           bool after, int sa0, int sb0, bool chain,
                                           typename DenseLoads<S>::Rsrc next, bool next_ends, int next_steps,
                                           const Hook& hook) {
    constexpr bool FP8 = S::FP8, SWIGLU = S::SWIGLU;
    constexpr int FA = S::FA, FB = S::FB, SA = S::SA, SB = S::SB, HB = FB / 2, HM = FA * HB;
    constexpr int A_LOADS = S::A_LOADS, B_LOADS = S::B_LOADS, LOADS = S::LOADS;
    constexpr int SUBS = FP8 ? 1 : 2;         // steps of a stage
    constexpr int SLOTS = 2 * SUBS * HM;      // matrix instructions of a window
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / S::WC, wn = wave % S::WC;
    const DenseLoads<S> ops(p, lds, DenseLoads<S>::resources(p, t));
    const bool ends = t.step0 + t.steps == plan.steps;

    // Lane l reads row l % 16 of a fragment at chunks l / 16 and 4 + l / 16: the two bf16 steps, or an e4m3
    // step's two halves. Fragments 16 rows apart share the swizzle.
    const int ar = wm * S::WTM + (lane & 15), br = wn * S::WTN + (lane & 15), chunk = lane >> 4;
    uint32_t va[2], vb[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        va[h] = static_cast<uint32_t>(ar * kStageBytes + (((4 * h + chunk) ^ ring_swizzle(ar)) << 4));
        vb[h] = S::B_BASE + static_cast<uint32_t>(br * kStageBytes + (((4 * h + chunk) ^ ring_swizzle(br)) << 4));
    }
    floatx4 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[i][j][r] = 0.0f;

    const int lane_row = lane >> 4;
    const int col4 = 4 * lane_row;
    const int tile_row = wm * S::WTM + (lane & 15);
    const int first_col = t.col0 + wn * (SWIGLU ? S::WTN / 2 : S::WTN);
    const uint32_t row_bytes = static_cast<uint32_t>(p.n) * 2;
    DenseExtra<S> extra;
    if constexpr (!S::CHAIN) {
        if (plan.splits == 1) {
            extra.load_columns(p, first_col + col4);
            extra.load_scales(p, t, tile_row);
            const auto r = tile_rows<S>(p, t, p.residual);
            static_for<FA>([&](auto i_c) {
                constexpr int i = decltype(i_c)::value;
                extra.template load_row<i>(p, r, (tile_row + i * 16) * row_bytes, first_col + col4);
            });
        }
        ops.prologue(t.steps, ends, 0, 0, false);
    }

    using Frag = DenseFrag<FP8>;
    // Fragment idx of the step whose (first) address is va[sub] or vb[sub] plus the slot's offset.
    auto read_at = [&](const uint32_t (&v)[2], uint32_t slot, auto sub_c, int idx) {
        Frag f;
        constexpr int sub = decltype(sub_c)::value;
        f.h[0] = *reinterpret_cast<const intx4*>(lds + v[sub] + slot + idx * S::FRAG);
        if constexpr (FP8) f.h[1] = *reinterpret_cast<const intx4*>(lds + v[1] + slot + idx * S::FRAG);
        return f;
    };
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    // The order is pinned instruction by instruction; of e4m3 in pairs, where the second product can start while
    // reads are still being issued (4096 x 4096 x 28672 with SwiGLU 367 -> 353 us; in fours 380, not at all 390).
    auto pin = [&](auto m_c) {
        if constexpr (!FP8 || decltype(m_c)::value % 2 == 1) fence();
    };
    Frag fa[FA], fb[FB];
    struct Refill {
        int kt_a, slot_a, kt_b, slot_b;
        __amdgpu_buffer_rsrc_t ra, rb;
        bool a_last, b_last;
    };
    // Loads of a window: x in its first quarter, the weight in the two after it, where the quarters hold them.
    constexpr bool kQuarters = A_LOADS <= SLOTS / 4 && B_LOADS <= SLOTS / 2;
    auto refill_at = [&](auto g_c, const Refill& r) {
        constexpr int g = decltype(g_c)::value;
        static_for<A_LOADS>([&](auto l_c) {
            constexpr int l = decltype(l_c)::value;
            constexpr int slot = kQuarters ? l * (SLOTS / 4) / A_LOADS : l * SLOTS / LOADS;
            if constexpr (slot == g) ops.issue_a(r.ra, r.kt_a, r.slot_a, l, r.a_last);
        });
        static_for<B_LOADS>([&](auto l_c) {
            constexpr int l = decltype(l_c)::value;
            constexpr int slot = kQuarters ? SLOTS / 4 + l * (SLOTS / 2) / B_LOADS : (A_LOADS + l) * SLOTS / LOADS;
            if constexpr (slot == g) ops.issue_b(r.rb, r.kt_b, r.slot_b, l, r.b_last);
        });
    };
    constexpr auto first_slot = [](int b) constexpr { return 2 * b < HM - 1 ? 2 * b : HM - 1; };
    constexpr auto second_slot = [](int b) constexpr { return 2 * b + 1 < HM - 1 ? 2 * b + 1 : HM - 1; };
    // Weight fragments [0, HB) by every x fragment (in snake order: one operand changes at a time), reading this
    // step's fragments [HB, FB).
    auto first_half = [&](uint32_t slot_b, auto sub_c, auto q_c, const Refill& rf) {
        constexpr int q = decltype(q_c)::value;
        static_for<HM>([&](auto m_c) {
            constexpr int m = decltype(m_c)::value;
            constexpr int i = m / HB, j = (i % 2) ? HB - 1 - m % HB : m % HB;
            if constexpr (q >= 0) refill_at(std::integral_constant<int, q * HM + m>{}, rf);
            acc[i][j] = dense_mma<FP8>(fb[j], fa[i], acc[i][j]);
            static_for<HB>([&](auto b_c) {
                constexpr int b = decltype(b_c)::value;
                if constexpr (first_slot(b) == m) fb[HB + b] = read_at(vb, slot_b, sub_c, HB + b);
            });
            pin(m_c);
        });
    };
    // The other weight fragments, reading the next step's x fragments and weight fragments [0, HB).
    auto second_half = [&](uint32_t slot_a, uint32_t slot_b, auto sub_c, auto last_c, auto q_c, const Refill& rf) {
        constexpr bool last = decltype(last_c)::value;
        constexpr int q = decltype(q_c)::value;
        static_for<HM>([&](auto m_c) {
            constexpr int m = decltype(m_c)::value;
            constexpr int i = m / HB, j = HB + ((i % 2) ? HB - 1 - m % HB : m % HB);
            if constexpr (q >= 0) refill_at(std::integral_constant<int, q * HM + m>{}, rf);
            acc[i][j] = dense_mma<FP8>(fb[j], fa[i], acc[i][j]);
            if constexpr (!last) {
                static_for<HB>([&](auto b_c) {
                    constexpr int b = decltype(b_c)::value;
                    if constexpr (second_slot(b) == m) fb[b] = read_at(vb, slot_b, sub_c, b);
                });
                if constexpr (m % HB == HB - 1) fa[i] = read_at(va, slot_a, sub_c, i);
            }
            pin(m_c);
        });
    };
    using C0 = std::integral_constant<int, 0>;
    using C1 = std::integral_constant<int, 1>;
    using NoLoads = std::integral_constant<int, -1>;
    using More = std::false_type;
    const Refill none{0, 0, 0, 0, ops.ra, ops.rb, false, false};
    const int steps = t.steps;
    const bool stores = S::CHAIN && after && plan.splits == 1;
    if (stores)
        wait_vm_lgkm<S::VM_FIRST + S::STORES>();
    else if (after)
        wait_vm_lgkm<0>();
    else
        wait_vm_lgkm<S::VM_FIRST>();
    ring_barrier();
    fence();
    {
        const uint32_t a0 = sa0 * S::A_STAGE, b0 = sb0 * S::B_STAGE;
#pragma unroll
        for (int b = 0; b < HB; ++b) fb[b] = read_at(vb, b0, C0{}, b);
#pragma unroll
        for (int i = 0; i < FA; ++i) fa[i] = read_at(va, a0, C0{}, i);
        first_half(b0, C0{}, NoLoads{}, none);
        if constexpr (SUBS == 2) {
            second_half(a0, b0, C1{}, More{}, NoLoads{}, none);
            first_half(b0, C1{}, NoLoads{}, none);
        }
    }
    int sa = sa0, sb = sb0;  // slots of the stage whose last half is pending
    auto window = [&](const Refill& rf, int na, int nb, bool behind) {
        const uint32_t a0 = na * S::A_STAGE, b0 = nb * S::B_STAGE;
        fence();
        if (behind)
            wait_vm_lgkm<S::VM_STEADY + S::STORES>();
        else
            wait_vm_lgkm<S::VM_STEADY>();
        ring_barrier();
        fence();
        second_half(a0, b0, C0{}, More{}, C0{}, rf);
        first_half(b0, C0{}, C1{}, rf);
        if constexpr (SUBS == 2) {
            second_half(a0, b0, C1{}, More{}, std::integral_constant<int, 2>{}, rf);
            first_half(b0, C1{}, std::integral_constant<int, 3>{}, rf);
        }
    };
    int u = 0;
    // Refills of this tile's whole stages, without selects; then the last windows in full. (A workgroup of one small
    // tile is bound by LDS and latency, not by the scalar unit, and its code is fetched anew by each launch: one
    // loop.)
    for (; S::CHAIN && u < steps - SB - 1; ++u) {
        const int na = sa + 1 == SA ? 0 : sa + 1, nb = sb + 1 == SB ? 0 : sb + 1;
        window(Refill{u + SA, sa, u + SB, sb, ops.ra, ops.rb, false, false}, na, nb, stores && u == 0);
        sa = na;
        sb = nb;
    }
    for (; u + 1 < steps; ++u) {
        const int na = sa + 1 == SA ? 0 : sa + 1, nb = sb + 1 == SB ? 0 : sb + 1;
        const bool a_next = S::CHAIN && chain && u + SA >= steps, b_next = S::CHAIN && chain && u + SB >= steps;
        const int kt_a = a_next ? u + SA - steps : min(u + SA, steps - 1);
        const int kt_b = b_next ? u + SB - steps : min(u + SB, steps - 1);
        window(Refill{kt_a, sa, kt_b, sb, a_next ? next.a : ops.ra, b_next ? next.b : ops.rb,
                      a_next ? next_ends && kt_a == next_steps - 1 : ends && kt_a == steps - 1,
                      b_next ? next_ends && kt_b == next_steps - 1 : ends && kt_b == steps - 1},
               na, nb, stores && u == 0);
        sa = na;
        sb = nb;
    }
    if constexpr (S::CHAIN) {
        if (plan.splits == 1) {
            extra.load_columns(p, first_col + col4);
            extra.load_scales(p, t, tile_row);
        }
        fence();
    }
    second_half(0u, 0u, C0{}, std::true_type{}, NoLoads{}, none);
    // Also without a next tile: no load may land in this LDS once the workgroup has ended.
    wait_vm_lgkm<0>();
    if constexpr (S::CHAIN) {
        ring_barrier();
        hook();
    }

    // Lane l holds, of each 16 x 16 block, row l % 16 and columns 4 (l / 16) + 0..3. The empty asm moves a row of
    // accumulators to plain registers before the epilogue's pairs could shape their assignment in the loop.
    const int col8 = 8 * (((lane_row & 1) << 1) | (lane_row >> 1));
    constexpr int OUT = DenseExtra<S>::OUT;
    if (plan.splits > 1) {
        // Partial sums of weight rows, as they are.
        static_for<FA>([&](auto i_c) {
            constexpr int i = decltype(i_c)::value;
            const int64_t row = t.row0 + tile_row + i * 16;
            float* to = plan.partial + (t.split * p.tokens + row) * p.rows;
            static_for<FB>([&](auto j_c) {
                constexpr int j = decltype(j_c)::value;
                to_vgpr(acc[i][j]);
                constexpr bool up = SWIGLU && j >= OUT;
                const int col = first_col + (up ? j - OUT : j) * 16 + col4;
                if (row < p.tokens && col < p.n) *reinterpret_cast<floatx4*>(to + (up ? p.n : 0) + col) = acc[i][j];
            });
        });
        return;
    }
    const auto out_rows = tile_rows<S>(p, t, p.output), residual_rows = tile_rows<S>(p, t, p.residual);
    auto finish = [&](auto act_c, auto plain_c) {
        constexpr int ACT = decltype(act_c)::value;
        constexpr bool PLAIN = decltype(plain_c)::value;
        if constexpr (S::CHAIN && !PLAIN) extra.template load_row<0>(p, residual_rows, tile_row * row_bytes, first_col + col4);
        static_for<FA>([&](auto i_c) {
            constexpr int i = decltype(i_c)::value;
            static_for<FB>([&](auto j_c) { to_vgpr(acc[i][decltype(j_c)::value]); });
            const uint32_t at = (tile_row + i * 16) * row_bytes;
            // The next row's residual is in flight while this one is worked out.
            if constexpr (S::CHAIN && !PLAIN && i + 1 < FA)
                extra.template load_row<i + 1>(p, residual_rows, at + 16 * row_bytes, first_col + col4);
            uint2 out[OUT];
            static_for<OUT>([&](auto j_c) {
                constexpr int j = decltype(j_c)::value;
                constexpr int up = SWIGLU ? j + OUT : j, ju = SWIGLU ? j : 0;
                float z[4], v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    z[r] = acc[i][j][r];
                    v[r] = acc[i][up][r];
                }
                const uint32_t* kept = extra.residual + (i % DenseExtra<S>::KEPT * OUT + j) * 2;
                out[j] = finish4<FP8, ACT, PLAIN>(z, v, extra.sx[i], extra.scale[j], extra.bias[j], extra.up_scale[ju],
                                                  extra.up_bias[ju], PLAIN ? make_uint2(0, 0) : make_uint2(kept[0], kept[1]));
            });
            // Lanes 16 apart trade halves of two neighbouring blocks: 16-byte stores of 8 columns.
            static_for<OUT / 2>([&](auto h_c) {
                constexpr int j = 2 * decltype(h_c)::value;
                const auto s0 = __builtin_amdgcn_permlane16_swap(out[j].x, out[j + 1].x, false, false);
                const auto s1 = __builtin_amdgcn_permlane16_swap(out[j].y, out[j + 1].y, false, false);
                const int col = first_col + j * 16 + col8;
                const uint32_t c = col < p.n ? static_cast<uint32_t>(col) * 2 : kPastColumns;
                const intx4 v = {static_cast<int>(s0[0]), static_cast<int>(s1[0]), static_cast<int>(s0[1]),
                                 static_cast<int>(s1[1])};
                __builtin_amdgcn_raw_buffer_store_b128(v, out_rows, at + c, 0, 0);
            });
            if constexpr (OUT % 2 == 1) {
                const int col = first_col + (OUT - 1) * 16 + col4;
                const uint32_t c = col < p.n ? static_cast<uint32_t>(col) * 2 : kPastColumns;
                typedef int intx2 __attribute__((ext_vector_type(2)));
                const intx2 v = {static_cast<int>(out[OUT - 1].x), static_cast<int>(out[OUT - 1].y)};
                __builtin_amdgcn_raw_buffer_store_b64(v, out_rows, at + c, 0, 0);
            }
        });
    };
    with_activation<S::ACT>(p.activation, [&](auto act_c) {
        if constexpr (S::CHAIN) {
            if (p.bias == nullptr && p.residual == nullptr) return finish(act_c, std::true_type{});
        }
        finish(act_c, std::false_type{});
    });
}

// A workgroup a tile. XCD i % 8 has a contiguous share of the tiles, as below.
template <typename S>
__global__ __launch_bounds__(256) void dense_tile_kernel(LinearArgs p, LinearPlan plan) {
    __shared__ __attribute__((aligned(1024))) char lds[S::LDS];
    const int tiles = plan.row_tiles * plan.col_tiles * plan.splits;
    const int per = (tiles + kNumXcd - 1) / kNumXcd;
    const int index = static_cast<int>(blockIdx.x) % kNumXcd * per + static_cast<int>(blockIdx.x) / kNumXcd;
    if (index >= tiles) return;
    const int column = index / plan.row_tiles;
    LinearTile t{};
    t.split = column / plan.col_tiles;
    t.row0 = (index - column * plan.row_tiles) * S::TM;
    t.col0 = (column - t.split * plan.col_tiles) * S::COLS;
    t.step0 = t.split * plan.split_steps;
    t.steps = min(plan.split_steps, plan.steps - t.step0);
    dense_tile<S>(p, plan, lds, t, false, 0, 0, false, {}, false, 0, [] {});
}

// Persistent: workgroups on XCD i % 8 take a contiguous share of the tiles, in order, so that the CUs of one L2
// work on neighbouring rows of x and the same weight rows.
template <typename S>
__global__ __launch_bounds__(256) void dense_ring_kernel(LinearArgs p, LinearPlan plan) {
    __shared__ __attribute__((aligned(1024))) char lds[S::LDS];
    using Loads = DenseLoads<S>;
    const int tiles = plan.row_tiles * plan.col_tiles * plan.splits;
    const int grid = static_cast<int>(gridDim.x);
    const int xcds = grid < kNumXcd ? 1 : kNumXcd;
    // XCD x has tiles [x tiles / xcds, (x + 1) tiles / xcds), its workgroups every (grid / xcds)-th of them.
    const int xcd = blockIdx.x % xcds, per = grid / xcds;
    const int first = static_cast<int>(static_cast<int64_t>(xcd) * tiles / xcds);
    const int end = static_cast<int>(static_cast<int64_t>(xcd + 1) * tiles / xcds);
    auto locate = [&](int index) {
        LinearTile t{false, 0, 0, 0, 0, 0};
        if (index >= end) return t;
        const int column = index / plan.row_tiles;
        t.split = column / plan.col_tiles;
        t.row0 = (index - column * plan.row_tiles) * S::TM;
        t.col0 = (column - t.split * plan.col_tiles) * S::COLS;
        t.step0 = t.split * plan.split_steps;
        t.steps = min(plan.split_steps, plan.steps - t.step0);
        t.valid = true;
        return t;
    };
    int at = first + static_cast<int>(blockIdx.x) / xcds;
    LinearTile cur = locate(at);
    if (!cur.valid) return;
    Loads(p, lds, Loads::resources(p, cur)).prologue(cur.steps, cur.step0 + cur.steps == plan.steps, 0, 0, false);
    bool after = false;
    int sa = 0, sb = 0;
    for (;;) {
        at += per;
        LinearTile nxt = locate(at);
        {
            // Opaque copies: nothing of the next tile is formed early and kept through the loop.
            int v = nxt.valid, r = nxt.row0, c = nxt.col0, k = nxt.step0, n = nxt.steps, s = nxt.split;
            asm volatile("" : "+s"(v), "+s"(r), "+s"(c), "+s"(k), "+s"(n), "+s"(s));
            nxt = LinearTile{v != 0, r, c, k, n, s};
        }
        const bool chain = nxt.valid && cur.steps >= S::SB && nxt.steps >= S::SB;
        const bool next_ends = nxt.step0 + nxt.steps == plan.steps;
        typename Loads::Rsrc next{};
        if (chain) next = Loads::resources(p, nxt);
        const int na = (sa + cur.steps) % S::SA, nb = (sb + cur.steps) % S::SB;
        auto hook = [&] {
            if (!nxt.valid) return;
            const Loads ops(p, lds, Loads::resources(p, nxt));
            ops.prologue(nxt.steps, next_ends, chain ? na : 0, chain ? nb : 0, chain);
        };
        dense_tile<S>(p, plan, lds, cur, after, sa, sb, chain, next, next_ends, nxt.steps, hook);
        if (!nxt.valid) break;
        sa = chain ? na : 0;
        sb = chain ? nb : 0;
        cur = nxt;
        after = true;
    }
}

// f(constant<LinearAct>, constant<FP8>) for these operands.
template <typename F>
void linear_instance(const LinearArgs& a, F&& f) {
    auto by_type = [&](auto act) { a.fp8 ? f(act, std::true_type{}) : f(act, std::false_type{}); };
    if (a.activation == MOE_ACT_SWIGLU)
        by_type(std::integral_constant<LinearAct, kActSwiglu>{});
    else if (a.activation == MOE_ACT_NONE)
        by_type(std::integral_constant<LinearAct, kActNone>{});
    else
        by_type(std::integral_constant<LinearAct, kActElement>{});
}

// The shape's kernel for these operands: `grid` persistent workgroups, or one for each tile.
template <int TM, int BN, uint32_t LDS, bool CHAIN>
void run_dense(const LinearArgs& a, const LinearPlan& plan, int grid, hipStream_t stream) {
    linear_instance(a, [&](auto act, auto fp8) {
        using S = DenseShape<TM, BN, decltype(act)::value, decltype(fp8)::value, LDS, CHAIN>;
        if constexpr (CHAIN) {
            dense_ring_kernel<S><<<grid, 256, 0, stream>>>(a, plan);
        } else {
            const int tiles = plan.row_tiles * plan.col_tiles * plan.splits;
            dense_tile_kernel<S><<<(tiles + kNumXcd - 1) / kNumXcd * kNumXcd, 256, 0, stream>>>(a, plan);
        }
    });
}

extern template void run_dense<256, 256, 160 * 1024, true>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
extern template void run_dense<128, 128, 160 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
extern template void run_dense<128, 128, 80 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
extern template void run_dense<96, 128, 80 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
extern template void run_dense<64, 128, 80 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
extern template void run_dense<64, 64, 80 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);

}  // namespace moe
