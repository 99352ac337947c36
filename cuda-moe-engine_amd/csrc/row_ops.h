// Wave sums, vector access with a short tail, and argument structs shared by the row operators
// (norm.hip, scored_route.hip, clip.hip) and their entry points (abi_layer.hip).
#pragma once

#include "moe_common.h"

namespace moe {

constexpr int64_t kMaxNormWidth = 16384;      // a row stays in a workgroup's registers
constexpr int64_t kMaxLayerTokens = 1 << 21;  // grids of up to 1024 threads a token stay below 2^32
constexpr int kMaxScoredExperts = 512;        // sixteen scores a lane, one wave
constexpr float kE4m3Most = 448.0f;           // largest finite e4m3 value
constexpr float kLeastAmax = 0x1p-100f;       // rows whose largest value is below this have its scale
constexpr int64_t kMaxClipTensors = 1 << 16;
constexpr int64_t kClipPartials = 2048;       // partial sums of squares of one clipping

// The wave's sum and maximum, in every lane: butterflies inside 16 lanes by DPP, across
// them by lane swaps, so no step goes through LDS.
template <int CTRL>
__device__ __forceinline__ float dpp_move(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int kDppXor1 = 0xb1;         // quad_perm 1,0,3,2
constexpr int kDppXor2 = 0x4e;         // quad_perm 2,3,0,1
constexpr int kDppHalfMirror = 0x141;  // lane i of 8 -> 7 - i
constexpr int kDppMirror = 0x140;      // lane i of 16 -> 15 - i

struct SumOp {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct MaxOp {
    static __device__ __forceinline__ float of(float a, float b) { return fmaxf(a, b); }
};

// OP over aligned groups of WIDTH lanes (a power of two up to 64), the result in each lane.
template <typename OP, int WIDTH = kWave>
__device__ __forceinline__ float lanes_reduce(float x) {
    if constexpr (WIDTH >= 2) x = OP::of(x, dpp_move<kDppXor1>(x));
    if constexpr (WIDTH >= 4) x = OP::of(x, dpp_move<kDppXor2>(x));
    if constexpr (WIDTH >= 8) x = OP::of(x, dpp_move<kDppHalfMirror>(x));
    if constexpr (WIDTH >= 16) x = OP::of(x, dpp_move<kDppMirror>(x));
    if constexpr (WIDTH >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = OP::of(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    if constexpr (WIDTH >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = OP::of(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    return x;
}

// Elements [at, at + N) of a row of n, as fp32, 0 past its end. One vector access unless the
// row ends inside it.
template <int DT, int N>
__device__ __forceinline__ void load_row(const typename Elem<DT>::T* row, int at, int n, float (&out)[N]) {
    using T = typename Elem<DT>::T;
    Unaligned<T, N> v;
    if (at + N <= n) {
        v = *reinterpret_cast<const Unaligned<T, N>*>(row + at);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v.v[i] = at + i < n ? row[at + i] : T(0);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = Elem<DT>::load(v.v[i]);
}

template <int DT, int N>
__device__ __forceinline__ void store_row(typename Elem<DT>::T* row, int at, int n, const float (&in)[N]) {
    using T = typename Elem<DT>::T;
    Unaligned<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.v[i] = Elem<DT>::store(in[i]);
    if (at + N <= n) {
        *reinterpret_cast<Unaligned<T, N>*>(row + at) = v;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i < n) row[at + i] = v.v[i];
    }
}

// What the entry points check and the launchers take.
struct NormArgs {
    const void* x;
    const void* residual;
    const void* weight;
    void* total;
    void* output;
    float* scales;  // not null: output is e4m3
    float* rstd;
    int64_t tokens;
    int hidden;
    int dtype;
    int weight_dtype;
    float eps;
};

struct NormGradArgs {
    const void* grad_output;
    const void* x;
    const void* weight;
    const float* rstd;
    const void* grad_x_base;
    void* grad_x;
    float* grad_weight;
    float* scratch;
    int64_t tokens;
    int hidden;
    int dtype;
    int weight_dtype;
};

struct ScoreArgs {
    const float* logits;
    const float* bias;
    int32_t* ids;
    float* weights;
    int64_t tokens;
    int experts;
    int topk;
    int groups;
    int top_groups;
    int group_best;
    bool sigmoid;
    bool renormalize;
    float scale;
};

struct ScoreGradArgs {
    const float* grad_weights;
    const float* logits;
    const int32_t* ids;
    float* grad_logits;
    int64_t tokens;
    int experts;
    int topk;
    bool sigmoid;
    bool renormalize;
    float scale;
};

int launch_rms_norm(const NormArgs& a, hipStream_t stream);
int launch_quantize_rows(const NormArgs& a, hipStream_t stream);
int64_t rms_norm_backward_scratch_bytes(int64_t tokens, int64_t hidden);
int launch_rms_norm_backward(const NormGradArgs& a, hipStream_t stream);
int launch_route_scored(const ScoreArgs& a, hipStream_t stream);
int launch_route_scored_backward(const ScoreGradArgs& a, hipStream_t stream);
int launch_clip_gradients(const void* const* grads, void* const* outputs, const int64_t* elements, const int64_t* dtypes,
                          int64_t tensors, double max_norm, float* norm, double* partials, hipStream_t stream);

}  // namespace moe
