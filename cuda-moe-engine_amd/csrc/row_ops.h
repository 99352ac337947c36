// Wave sums, vector access with a short tail, and argument structs shared by the row operators
// (norm.hip, scored_route.hip, clip.hip) and their entry points (abi_layer.hip).
#pragma once

#include <type_traits>

#include "moe_common.h"

namespace moe {

constexpr int64_t kMaxNormWidth = 16384;      // a row stays in a workgroup's registers
constexpr int64_t kMaxQuantizeWidth = 32768;  // without a weight's registers
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

// The largest of aligned groups of WIDTH lanes, for unsigned integers (which, unlike floats, need no
// quieting of each operand: one instruction a step).
template <int WIDTH>
__device__ __forceinline__ uint32_t lanes_max(uint32_t x) {
    auto step = [&](auto ctrl) {
        const uint32_t other = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 0xf, 0xf, true);
        x = other > x ? other : x;
    };
    if constexpr (WIDTH >= 2) step(std::integral_constant<int, kDppXor1>{});
    if constexpr (WIDTH >= 4) step(std::integral_constant<int, kDppXor2>{});
    if constexpr (WIDTH >= 8) step(std::integral_constant<int, kDppHalfMirror>{});
    if constexpr (WIDTH >= 16) step(std::integral_constant<int, kDppMirror>{});
    if constexpr (WIDTH >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        x = s[0] > s[1] ? s[0] : s[1];
    }
    if constexpr (WIDTH >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        x = s[0] > s[1] ? s[0] : s[1];
    }
    return x;
}

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

// 16, 8 or 4 bytes at any address, as one instruction: a copy through a struct of elements is
// split into narrow loads where its elements are converted one by one (the norm of 8192 x 4096 in 8 bits took
// 68 us with such copies, 41 without).
template <int BYTES> struct Bytes;
template <> struct Bytes<16> {
    typedef uint32_t V __attribute__((ext_vector_type(4)));
    typedef uint32_t At __attribute__((ext_vector_type(4), aligned(1)));
};
template <> struct Bytes<8> {
    typedef uint32_t V __attribute__((ext_vector_type(2)));
    typedef uint32_t At __attribute__((ext_vector_type(2), aligned(1)));
};
template <> struct Bytes<4> {
    typedef uint32_t V;
    typedef uint32_t At __attribute__((aligned(1)));
};

template <int BYTES>
__device__ __forceinline__ typename Bytes<BYTES>::V load_bytes(const void* p) {
    return *static_cast<const typename Bytes<BYTES>::At*>(p);
}

template <int BYTES>
__device__ __forceinline__ void store_bytes(void* p, typename Bytes<BYTES>::V v) {
    *static_cast<typename Bytes<BYTES>::At*>(p) = v;
}

// Elements [at, at + N) of a row of n as they lie, 0 past its end. One access unless the row ends
// inside it.
template <typename T, int N>
__device__ __forceinline__ typename Bytes<N * sizeof(T)>::V load_vector(const T* row, int at, int n) {
    if (at + N <= n) return load_bytes<N * sizeof(T)>(row + at);
    T v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = at + i < n ? row[at + i] : T(0);
    return __builtin_bit_cast(typename Bytes<N * sizeof(T)>::V, v);
}

// The N elements of such a vector as fp32, and back.
template <int DT, int N, typename V>
__device__ __forceinline__ void unpack(V v, float (&out)[N]) {
    using T = typename Elem<DT>::T;
    static_assert(sizeof(V) == N * sizeof(T), "vector");
    T e[N];
    __builtin_memcpy(e, &v, sizeof(V));
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = Elem<DT>::load(e[i]);
}

template <int DT, int N>
__device__ __forceinline__ auto pack(const float (&in)[N]) {
    using T = typename Elem<DT>::T;
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = Elem<DT>::store(in[i]);
    return __builtin_bit_cast(typename Bytes<N * sizeof(T)>::V, e);
}

// As fp32, in accesses of up to 16 bytes.
template <int DT, int N>
__device__ __forceinline__ void load_row(const typename Elem<DT>::T* row, int at, int n, float (&out)[N]) {
    using T = typename Elem<DT>::T;
    constexpr int STEP = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += STEP) {
        float part[STEP];
        unpack<DT>(load_vector<T, STEP>(row, at + i, n), part);
#pragma unroll
        for (int j = 0; j < STEP; ++j) out[i + j] = part[j];
    }
}

template <int DT, int N>
__device__ __forceinline__ void store_row(typename Elem<DT>::T* row, int at, int n, const float (&in)[N]) {
    using T = typename Elem<DT>::T;
    constexpr int STEP = N * sizeof(T) > 16 ? 16 / sizeof(T) : N;
#pragma unroll
    for (int i = 0; i < N; i += STEP) {
        float part[STEP];
#pragma unroll
        for (int j = 0; j < STEP; ++j) part[j] = in[i + j];
        const auto v = pack<DT>(part);
        if (at + i + STEP <= n) {
            store_bytes<STEP * sizeof(T)>(row + at + i, v);
        } else {
            T e[STEP];
            __builtin_memcpy(e, &v, sizeof(v));
#pragma unroll
            for (int j = 0; j < STEP; ++j)
                if (at + i + j < n) row[at + i + j] = e[j];
        }
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
    int group_size;  // set by the launcher: experts of a group,
    int lane_shift;  // log2 of its lanes
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
int64_t rms_norm_backward_scratch_bytes(int64_t tokens, int64_t hidden, int dtype);
int launch_rms_norm_backward(const NormGradArgs& a, hipStream_t stream);
int launch_route_scored(const ScoreArgs& a, hipStream_t stream);
int launch_route_scored_backward(const ScoreGradArgs& a, hipStream_t stream);
int launch_clip_gradients(const void* const* grads, void* const* outputs, const int64_t* elements, const int64_t* dtypes,
                          int64_t tensors, double max_norm, float* norm, double* partials, hipStream_t stream);

}  // namespace moe
