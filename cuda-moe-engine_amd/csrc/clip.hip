// The global norm of many gradients, and the gradients scaled so that it is at most max_norm.
//
//   norm = sqrt(sum over all tensors of g^2),  f = min(1, max_norm / (norm + 1e-6)),  out = round(f g)
//
// Two launches for up to kClipTensors tensors (more: a pair per that many): the squares'
// sums of workgroups, then every workgroup of the second adds these partial sums itself and
// scales its share. The tensors' addresses go by value in the launch's arguments, so nothing
// is copied to the device and a captured graph holds them. A square of fp32 is exact in 64
// bits, and all sums are 64 bits: no gradient that is finite makes the norm overflow.
// Bound by the bytes: all tensors read twice and written once. 554 M bf16 elements in 200 tensors (two launches
// of each kernel) 680 us: the squares at 4.8 TB/s, the scaling at 4.9. 24 tensors of 65536 fp32 11 us, launches.
#include "row_ops.h"

namespace moe {

namespace {

constexpr int kClipTensors = 112;   // of one launch: their table fits the kernel's arguments
constexpr int kThreads = 256;
constexpr int kLeastChunk = 1 << 11, kMostChunk = 1 << 16;
constexpr int kUnroll = 4;          // vectors of 16 bytes a lane has in flight

struct ClipTable {
    const void* in[kClipTensors];
    void* out[kClipTensors];
    int64_t elements[kClipTensors];
    int32_t first[kClipTensors + 1];  // chunks before each tensor
    int8_t dtype[kClipTensors];
    int tensors;
    int chunk;  // elements a workgroup takes at a time
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

// f(first element, v[N]) of a chunk of n elements from g, kUnroll vectors a lane in flight: whole
// rounds of the workgroup, then vector by vector, the last one short.
template <int DT, typename F>
__device__ __forceinline__ void each_vector(const typename Elem<DT>::T* g, int n, const F& f) {
    constexpr int N = DT == MOE_DTYPE_F32 ? 4 : 8, STEP = kThreads * N;
    int at = threadIdx.x * N;
    for (; at + (kUnroll - 1) * STEP + N <= n; at += kUnroll * STEP) {
        typename Bytes<16>::V v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) v[u] = load_bytes<16>(g + at + u * STEP);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            float x[N];
            unpack<DT>(v[u], x);
            f(at + u * STEP, x);
        }
    }
    for (; at < n; at += STEP) {
        float x[N];
        load_row<DT, N>(g, at, n, x);
        f(at, x);
    }
}

template <int DT>
__device__ __forceinline__ double squares(const void* in, int64_t from, int n) {
    double sum = 0.0;
    each_vector<DT>(static_cast<const typename Elem<DT>::T*>(in) + from, n, [&](int, const auto& x) {
        for (float v : x) sum += static_cast<double>(v) * static_cast<double>(v);
    });
    return sum;
}

__global__ __launch_bounds__(kThreads) void clip_norm_kernel(ClipTable t, double* __restrict__ partials) {
    __shared__ double lds[kThreads / kWave];
    double sum = 0.0;
    const int chunks = t.first[t.tensors];
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int i = tensor_of(t, chunk);
        const int64_t from = static_cast<int64_t>(chunk - t.first[i]) * t.chunk;
        const int n = static_cast<int>(min<int64_t>(t.chunk, t.elements[i] - from));
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

template <int DT, typename F>
__device__ __forceinline__ void scale(const void* in, void* out, int64_t from, int n, F factor) {
    typename Elem<DT>::T* o = static_cast<typename Elem<DT>::T*>(out) + from;
    each_vector<DT>(static_cast<const typename Elem<DT>::T*>(in) + from, n, [&](int at, auto& x) {
        for (float& v : x) v = static_cast<float>(static_cast<F>(v) * factor);
        store_row<DT>(o, at, n, x);
    });
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
    const double factor = norm < __builtin_inf() && ratio < 1.0 ? ratio : 1.0;
    const int chunks = t.first[t.tensors];
    auto each_chunk = [&](auto f) {
        // Backwards: what the pass before read last may still be in the caches.
        for (int chunk = chunks - 1 - static_cast<int>(blockIdx.x); chunk >= 0; chunk -= gridDim.x) {
            const int i = tensor_of(t, chunk);
            if (f == 1 && t.in[i] == t.out[i]) continue;
            const int64_t from = static_cast<int64_t>(chunk - t.first[i]) * t.chunk;
            const int n = static_cast<int>(min<int64_t>(t.chunk, t.elements[i] - from));
            const int dt = t.dtype[i];
            if (dt == MOE_DTYPE_F32)
                scale<MOE_DTYPE_F32>(t.in[i], t.out[i], from, n, f);
            else if (dt == MOE_DTYPE_F16)
                scale<MOE_DTYPE_F16>(t.in[i], t.out[i], from, n, f);
            else
                scale<MOE_DTYPE_BF16>(t.in[i], t.out[i], from, n, f);
        }
    };
    // Large gradients may need a factor below fp32's normal range (an fp32 one of 3.2e-44 is off by 2%): in 64 bits,
    // which costs fp16 3% where it is always done (500 M elements 616 -> 632 us).
    if (factor < 0x1p-126)
        each_chunk(factor);
    else
        each_chunk(static_cast<float>(factor));
}

// A launch's share of the partial sums bounds its workgroups, in the second pass as well: lists of thousands of tensors
// leave CUs idle (554 M bf16 in 200 tensors 668 us in place, in 2000 1822, in 6000 5810).
int blocks_of(int chunks, int launches) {
    const int most = static_cast<int>(kClipPartials) / launches;
    return chunks < most ? (chunks < 1 ? 1 : chunks) : most;
}

int chunks_of(int64_t elements, int chunk) { return static_cast<int>((elements + chunk - 1) / chunk); }

}  // namespace

// The entry point has bounded tensors and elements, so that chunks fit 32 bits and every
// launch has partial sums of its own.
int launch_clip_gradients(const void* const* grads, void* const* outputs, const int64_t* elements, const int64_t* dtypes,
                          int64_t tensors, double max_norm, float* norm, double* partials, hipStream_t stream) {
    const int launches = tensors <= kClipTensors ? 1 : static_cast<int>((tensors + kClipTensors - 1) / kClipTensors);
    // A chunk for each of kClipPartials workgroups, within bounds: small batches spread over the chip, large
    // ones do not search for their tensor all the time.
    int64_t total = 0;
    for (int64_t i = 0; i < tensors; ++i) total += elements[i];
    int chunk = kLeastChunk;
    while (chunk < kMostChunk && chunk * kClipPartials < total) chunk *= 2;
    int used = 0;
    for (int pass = 0; pass < 2; ++pass) {
        for (int l = 0; l < launches; ++l) {
            ClipTable t;
            t.tensors = 0;
            t.chunk = chunk;
            int chunks = 0;
            for (int64_t i = l * kClipTensors; i < tensors && i < (l + 1) * kClipTensors; ++i) {
                const int k = t.tensors++;
                t.in[k] = grads[i];
                t.out[k] = outputs[i];
                t.elements[k] = elements[i];
                t.dtype[k] = static_cast<int8_t>(dtypes[i]);
                t.first[k] = chunks;
                chunks += chunks_of(elements[i], chunk);
            }
            t.first[t.tensors] = chunks;
            const int blocks = blocks_of(chunks, launches);
            if (pass == 0) {
                clip_norm_kernel<<<blocks, kThreads, 0, stream>>>(t, partials + used);
                used += blocks;
            } else {
                clip_scale_kernel<<<blocks, kThreads, 0, stream>>>(t, partials, used, max_norm, l == 0 ? norm : nullptr);
            }
        }
    }
    return check_launch("clip_gradients");
}

}  // namespace moe
