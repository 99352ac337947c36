// The global norm of many gradients, and the gradients scaled so that it is at most max_norm.
//
//   norm = sqrt(sum over all tensors of g^2),  f = min(1, max_norm / (norm + 1e-6)),  out = round(f g)
//
// Two launches for up to kClipTensors tensors (more: a pair per that many): the squares'
// sums of workgroups, then every workgroup of the second adds these partial sums itself and
// scales its share. The tensors' addresses go by value in the launch's arguments, so nothing
// is copied to the device and a captured graph holds them. A square of fp32 is exact in 64
// bits, and all sums are 64 bits: no gradient that is finite makes the norm overflow.
// Bound by the bytes: all tensors read twice and written once.
#include "row_ops.h"

namespace moe {

namespace {

constexpr int kClipTensors = 112;   // of one launch: their table fits the kernel's arguments
constexpr int kChunk = 1 << 15;     // elements a workgroup takes at a time
constexpr int kThreads = 256;

struct ClipTable {
    const void* in[kClipTensors];
    void* out[kClipTensors];
    int64_t elements[kClipTensors];
    int32_t first[kClipTensors + 1];  // chunks before each tensor
    int8_t dtype[kClipTensors];
    int tensors;
};
static_assert(sizeof(ClipTable) + 64 <= 4096, "kernel arguments");

// The tensor of a chunk, by halving.
__device__ __forceinline__ int tensor_of(const ClipTable& t, int chunk) {
    int lo = 0, hi = t.tensors - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (t.first[mid] <= chunk)
            lo = mid;
        else
            hi = mid - 1;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) x += __shfl_xor(x, d);
    return x;
}

__device__ __forceinline__ double block_sum(double x, double* lds) {
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    double sum = lds[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) sum += lds[w];
    return sum;
}

template <int DT>
__device__ __forceinline__ double squares(const void* in, int64_t from, int n) {
    using T = typename Elem<DT>::T;
    constexpr int N = DT == MOE_DTYPE_F32 ? 4 : 8;
    const T* g = static_cast<const T*>(in) + from;
    double sum = 0.0;
    for (int at = threadIdx.x * N; at < n; at += kThreads * N) {
        float v[N];
        load_row<DT, N>(g, at, n, v);
#pragma unroll
        for (int i = 0; i < N; ++i) sum += static_cast<double>(v[i]) * static_cast<double>(v[i]);
    }
    return sum;
}

__global__ __launch_bounds__(kThreads) void clip_norm_kernel(ClipTable t, double* __restrict__ partials) {
    __shared__ double lds[kThreads / kWave];
    double sum = 0.0;
    const int chunks = t.first[t.tensors];
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        const int64_t from = static_cast<int64_t>(chunk - t.first[i]) * kChunk;
        const int n = static_cast<int>(min<int64_t>(kChunk, t.elements[i] - from));
        const int dt = t.dtype[i];
        if (dt == MOE_DTYPE_F32)
            sum += squares<MOE_DTYPE_F32>(t.in[i], from, n);
        else if (dt == MOE_DTYPE_F16)
            sum += squares<MOE_DTYPE_F16>(t.in[i], from, n);
        else
            sum += squares<MOE_DTYPE_BF16>(t.in[i], from, n);
    }
    sum = block_sum(sum, lds);
    if (threadIdx.x == 0) partials[blockIdx.x] = sum;
}

template <int DT>
__device__ __forceinline__ void scale(const void* in, void* out, int64_t from, int n, float factor) {
    using T = typename Elem<DT>::T;
    constexpr int N = DT == MOE_DTYPE_F32 ? 4 : 8;
    const T* g = static_cast<const T*>(in) + from;
    T* o = static_cast<T*>(out) + from;
    for (int at = threadIdx.x * N; at < n; at += kThreads * N) {
        float v[N];
        load_row<DT, N>(g, at, n, v);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= factor;
        store_row<DT, N>(o, at, n, v);
    }
}

// `count` partial sums of all the norm launches; the first launch's first workgroup writes the norm.
__global__ __launch_bounds__(kThreads) void clip_scale_kernel(ClipTable t, const double* __restrict__ partials, int count,
                                                              double max_norm, float* __restrict__ norm_out) {
    __shared__ double lds[kThreads / kWave];
    double sum = 0.0;
    for (int i = threadIdx.x; i < count; i += kThreads) sum += partials[i];
    const double norm = sqrt(block_sum(sum, lds));
    if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = static_cast<float>(norm);
    // A norm that is no number or infinite leaves the gradients as they are.
    const double ratio = max_norm / (norm + 1e-6);
    const float factor = norm < __builtin_inf() && ratio < 1.0 ? static_cast<float>(ratio) : 1.0f;
    const int chunks = t.first[t.tensors];
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        if (factor == 1.0f && t.in[i] == t.out[i]) continue;
        const int64_t from = static_cast<int64_t>(chunk - t.first[i]) * kChunk;
        const int n = static_cast<int>(min<int64_t>(kChunk, t.elements[i] - from));
        const int dt = t.dtype[i];
        if (dt == MOE_DTYPE_F32)
            scale<MOE_DTYPE_F32>(t.in[i], t.out[i], from, n, factor);
        else if (dt == MOE_DTYPE_F16)
            scale<MOE_DTYPE_F16>(t.in[i], t.out[i], from, n, factor);
        else
            scale<MOE_DTYPE_BF16>(t.in[i], t.out[i], from, n, factor);
    }
}

int blocks_of(int chunks, int launches) {
    const int most = static_cast<int>(kClipPartials) / launches;
    return chunks < most ? (chunks < 1 ? 1 : chunks) : most;
}

}  // namespace

// The entry point has bounded tensors and elements, so that chunks fit 32 bits and every
// launch has partial sums of its own.
int launch_clip_gradients(const void* const* grads, void* const* outputs, const int64_t* elements, const int64_t* dtypes,
                          int64_t tensors, double max_norm, float* norm, double* partials, hipStream_t stream) {
    const int launches = tensors <= kClipTensors ? 1 : static_cast<int>((tensors + kClipTensors - 1) / kClipTensors);
    for (int pass = 0; pass < 2; ++pass) {
        int used = 0, total = 0;
        if (pass == 1)
            for (int l = 0; l < launches; ++l) {
                int64_t chunks = 0;
                for (int64_t i = l * kClipTensors; i < tensors && i < (l + 1) * kClipTensors; ++i)
                    chunks += (elements[i] + kChunk - 1) / kChunk;
                total += blocks_of(static_cast<int>(chunks), launches);
            }
        for (int l = 0; l < launches; ++l) {
            ClipTable t;
            t.tensors = 0;
            int chunks = 0;
            for (int64_t i = l * kClipTensors; i < tensors && i < (l + 1) * kClipTensors; ++i) {
                const int k = t.tensors++;
                t.in[k] = grads[i];
                t.out[k] = outputs[i];
                t.elements[k] = elements[i];
                t.dtype[k] = static_cast<int8_t>(dtypes[i]);
                t.first[k] = chunks;
                chunks += static_cast<int>((elements[i] + kChunk - 1) / kChunk);
            }
            t.first[t.tensors] = chunks;
            const int blocks = blocks_of(chunks, launches);
            if (pass == 0) {
                clip_norm_kernel<<<blocks, kThreads, 0, stream>>>(t, partials + used);
                used += blocks;
            } else {
                clip_scale_kernel<<<blocks, kThreads, 0, stream>>>(t, partials, total, max_norm, l == 0 ? norm : nullptr);
            }
        }
    }
    return check_launch("clip_gradients");
}

}  // namespace moe
