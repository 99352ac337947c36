// Low-rank adapters of many requests beside a shared projection, and the same skinny
// products for the router's gradient.
//
//   h_i = down_a x_i,   y_i = base_i + s_a up_a^T h_i         (a = the row's adapter)
//   dh_i = s_a up_a dy_i,  dx_i = base_i + down_a^T dh_i
//   ddown_a = sum_i dh_i x_i^T,  dup_a = s_a sum_i h_i dy_i^T
//
// down [N, r, H] and up [N, r, O] are both rank-major, so forward and backward are three
// products: contract (a long row against r rows), spread (r values over a long row) and
// outer (r values times a long row, summed over the rows). All three are bound by the
// long rows' bytes (2r flop per 2 bytes), run on v_mfma_f32_16x16x32_bf16 straight from
// global memory to registers, and use no atomics: every sum has one order.
#include <algorithm>

#include "low_rank.h"

namespace moe {

typedef __bf16 lbf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t mfma(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(lbf16x8_t, a), __builtin_bit_cast(lbf16x8_t, b),
                                                   c, 0, 0, 0);
}

__device__ __forceinline__ u32x4_t load16(const uint16_t* p) { return *reinterpret_cast<const u32x4_t*>(p); }

// What f is beyond its bf16 part: below 2^-8 |f|, and 0 beyond an infinite or NaN part,
// so that two parts hold f to 2^-16 and three exactly.
__device__ __forceinline__ float bf16_rest(float f, uint32_t part) {
    const float rest = f - bf16_to_f32(static_cast<uint16_t>(part));
    return __builtin_isfinite(rest) ? rest : 0.0f;
}

// ---------------------------------------------------------------------------
// Rows sorted by adapter. One workgroup counts the ids in LDS, scans the counts into
// starts, and writes the tile and split tables; then a wave per adapter collects its
// rows in order (ballot ranks: stable, no atomics), in the same launch for up to
// kGroupSmall rows and in a second one for more. A program groups once a step and uses
// the table for all its projections.
// ---------------------------------------------------------------------------
constexpr int kGroupThreads = 1024;
constexpr int kGroupSmall = 4096;

__device__ __forceinline__ int group_of(int id, int adapters) {
    return static_cast<unsigned>(id) < static_cast<unsigned>(adapters) ? id : adapters;
}

// The rows of group a, in order, to order[pos...]; `ids(i)` is row i's group.
template <typename F>
__device__ __forceinline__ void collect_rows(int a, int pos, int end, int tokens, int lane, int32_t* order, F ids) {
    constexpr int U = 4;
    for (int base = 0; base < tokens && pos < end; base += 64 * U) {
        int group[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = base + 64 * u + lane;
            group[u] = i < tokens ? ids(i) : -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const uint64_t found = __ballot(group[u] == a);
            if (group[u] == a) order[pos + __popcll(found & ((1ull << lane) - 1))] = base + 64 * u + lane;
            pos += __popcll(found);
        }
    }
}

__global__ __launch_bounds__(kGroupThreads) void adapter_group_kernel(const int32_t* __restrict__ ids,
                                                                      int32_t* __restrict__ table, TableLayout t,
                                                                      int tokens, int adapters) {
    extern __shared__ int32_t lds[];
    int32_t* counts = lds;                    // [adapters + 1], then the groups' starts
    int32_t* cached = lds + adapters + 1;     // [tokens] groups of a small batch
    __shared__ int32_t wave_sums[3][kGroupThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const bool small = tokens <= kGroupSmall;
    for (int i = tid; i <= adapters; i += kGroupThreads) counts[i] = 0;
    __syncthreads();
    for (int i = tid; i < tokens; i += kGroupThreads) {
        const int a = group_of(ids[i], adapters);
        if (small) cached[i] = a;
        // Rows of a request are neighbours: one add for a wave of one group.
        const uint64_t active = __ballot(1);
        const int first = __builtin_amdgcn_readfirstlane(a);
        if (__ballot(a == first) == active) {
            if (lane == __ffsll(static_cast<unsigned long long>(active)) - 1) atomicAdd(&counts[a], __popcll(active));
        } else {
            atomicAdd(&counts[a], 1);
        }
    }
    __syncthreads();
    // Exclusive scans of rows, tiles and splits over the groups; a thread owns `per` neighbours.
    const int groups = adapters + 1;
    const int per = (groups + kGroupThreads - 1) / kGroupThreads;
    const int g0 = min(tid * per, groups), g1 = min(g0 + per, groups);
    int rows = 0, tiles = 0, splits = 0;
    for (int a = g0; a < g1; ++a) {
        rows += counts[a];
        tiles += (counts[a] + kTileRows - 1) / kTileRows;
        if (a < adapters) splits += (counts[a] + t.split_rows - 1) / t.split_rows;
    }
    int row_end = rows, tile_end = tiles, split_end = splits;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int r = __shfl_up(row_end, d), i = __shfl_up(tile_end, d), s = __shfl_up(split_end, d);
        if (lane >= d) {
            row_end += r;
            tile_end += i;
            split_end += s;
        }
    }
    if (lane == 63) {
        wave_sums[0][wave] = row_end;
        wave_sums[1][wave] = tile_end;
        wave_sums[2][wave] = split_end;
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w) {
        row_end += wave_sums[0][w];
        tile_end += wave_sums[1][w];
        split_end += wave_sums[2][w];
    }
    int row = row_end - rows, tile = tile_end - tiles, split = split_end - splits;
    int32_t* starts = table + t.starts;
    int32_t* split_start = table + t.split_start;
    int4* tile_table = reinterpret_cast<int4*>(table + t.tiles);
    int4* split_table = reinterpret_cast<int4*>(table + t.splits);
    for (int a = g0; a < g1; ++a) {
        const int n = counts[a];
        const int owner = a < adapters ? a : -1;
        starts[a] = row;
        for (int i = 0; i < n; i += kTileRows) tile_table[tile++] = make_int4(owner, row + i, min(kTileRows, n - i), 0);
        if (a < adapters) {
            const int parts = (n + t.split_rows - 1) / t.split_rows;
            split_start[a] = split;
            for (int i = 0; i < n; i += t.split_rows)
                split_table[split++] = make_int4(a, row + i, min(t.split_rows, n - i), parts);
        } else {
            starts[adapters + 1] = tokens;
            split_start[adapters] = split;
            table[0] = tile;
            table[1] = split;
            table[2] = table[3] = 0;
        }
        counts[a] = row;  // this thread's own entry: its start from here on
        row += n;
    }
    if (!small) return;
    __syncthreads();
    for (int a = wave; a < groups; a += kGroupThreads / 64) {
        const int end = a < adapters ? counts[a + 1] : tokens;
        if (counts[a] < end)
            collect_rows(a, counts[a], end, tokens, lane, table + t.order, [&](int i) { return cached[i]; });
    }
}

__global__ __launch_bounds__(256) void adapter_order_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ table,
                                                            TableLayout t, int tokens, int adapters) {
    const int a = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (a > adapters) return;
    const int pos = table[t.starts + a], end = table[t.starts + a + 1];
    if (pos < end)
        collect_rows(a, pos, end, tokens, threadIdx.x & 63, table + t.order,
                     [&](int i) { return group_of(ids[i], adapters); });
}

int launch_adapter_group(const int32_t* ids, void* table, int64_t tokens, int adapters, hipStream_t stream) {
    const TableLayout t = table_layout(tokens, adapters);
    int32_t* base = static_cast<int32_t*>(table);
    const bool small = tokens <= kGroupSmall;
    const size_t lds = (static_cast<size_t>(adapters) + 1 + (small ? tokens : 0)) * 4;
    hipLaunchKernelGGL(adapter_group_kernel, dim3(1), dim3(kGroupThreads), lds, stream, ids, base, t,
                       static_cast<int>(tokens), adapters);
    int rc = check_launch("adapter_group_kernel");
    if (rc != MOE_OK || small) return rc;
    hipLaunchKernelGGL(adapter_order_kernel, dim3((adapters + 4) / 4), dim3(256), 0, stream, ids, base, t,
                       static_cast<int>(tokens), adapters);
    return check_launch("adapter_order_kernel");
}

// ---------------------------------------------------------------------------
// contract: h[i][c] = sum_k x[i][k] w[c][k].
// A workgroup takes a tile of up to 64 rows of one adapter and a slice of k, its four
// waves a quarter of the slice each. Both operands lie along k as the MFMA reads them
// (lane l: row l % 16, 8 k from 8 (l / 16)); k is permuted inside 64 so that a lane
// reads 32 bytes and a step whole 128-byte lines. Rows past the tile and ranks past r
// are read from the last one and not stored (an output depends on its own row and rank
// alone). The waves' sums meet in LDS, the slices' in the consumer, in slice order.
// ---------------------------------------------------------------------------
template <int MF, int NR>
struct ContractStep {
    u32x4_t x[MF][2], w[NR][2];
};

template <int MF, int NR>
__device__ __forceinline__ void contract_load(ContractStep<MF, NR>& s, const uint16_t* const (&xr)[MF],
                                              const uint16_t* const (&wr)[NR], int kk, int k) {
    const u32x4_t zero = {0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = kk + 8 * h;
        if (at < k) {
#pragma unroll
            for (int m = 0; m < MF; ++m) s.x[m][h] = load16(xr[m] + at);
#pragma unroll
            for (int n = 0; n < NR; ++n) s.w[n][h] = load16(wr[n] + at);
        } else {
#pragma unroll
            for (int m = 0; m < MF; ++m) s.x[m][h] = zero;
#pragma unroll
            for (int n = 0; n < NR; ++n) s.w[n][h] = zero;
        }
    }
}

template <int MF, int NR>
__device__ __forceinline__ void contract_tile(const uint16_t* __restrict__ x, const uint16_t* __restrict__ w,
                                              const int32_t* order, int first, int rows, float* __restrict__ part,
                                              int k, int rank, int kb, int ke, float* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l = lane & 15, g = lane >> 4;
    const uint16_t* xr[MF];
    const uint16_t* wr[NR];
#pragma unroll
    for (int m = 0; m < MF; ++m)
        xr[m] = x + static_cast<int64_t>(order[first + min(16 * m + l, rows - 1)]) * k;
#pragma unroll
    for (int n = 0; n < NR; ++n) wr[n] = w + static_cast<int64_t>(min(16 * n + l, rank - 1)) * k;
    f32x4_t acc[MF][NR];
#pragma unroll
    for (int m = 0; m < MF; ++m)
#pragma unroll
        for (int n = 0; n < NR; ++n) acc[m][n] = f32x4_t{0, 0, 0, 0};
    if (kb < ke) {
        ContractStep<MF, NR> cur, next;
        contract_load<MF, NR>(cur, xr, wr, kb + 16 * g, k);
        for (int k0 = kb; k0 < ke; k0 += 64) {
            if (k0 + 64 < ke) contract_load<MF, NR>(next, xr, wr, k0 + 64 + 16 * g, k);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int m = 0; m < MF; ++m)
#pragma unroll
                    for (int n = 0; n < NR; ++n) acc[m][n] = mfma(cur.x[m][h], cur.w[n][h], acc[m][n]);
            cur = next;
        }
    }
    // One 16-row fragment at a time: [wave][row][rank] in LDS, summed in wave order.
    constexpr int C = 16 * NR;
#pragma unroll
    for (int m = 0; m < MF; ++m) {
        if (m > 0) __syncthreads();
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) lds[(wave * 16 + 4 * g + q) * C + 16 * n + l] = acc[m][n][q];
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * C; i += 256) {
            const int row = 16 * m + i / C, c = i % C;
            if (row < rows && c < rank)
                part[static_cast<int64_t>(first + row) * rank + c] =
                    ((lds[i] + lds[i + 16 * C]) + lds[i + 32 * C]) + lds[i + 48 * C];
        }
    }
}

template <int NR>
__global__ __launch_bounds__(256) void contract_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ w,
                                                       Groups gr, float* __restrict__ partials, int64_t tokens, int k,
                                                       int rank, int span) {
    __shared__ float lds[4 * 16 * 16 * NR];
    if (static_cast<int>(blockIdx.x) >= gr.head[0]) return;
    const int4 tile = gr.tiles[blockIdx.x];
    if (tile.x < 0) return;
    const int kb = blockIdx.y * span + static_cast<int>(threadIdx.x >> 6) * (span / 4);
    const int ke = min(kb + span / 4, k);
    const uint16_t* wa = w + static_cast<int64_t>(tile.x) * rank * k;
    float* part = partials + static_cast<int64_t>(blockIdx.y) * tokens * rank;
    if (tile.z > 32)
        contract_tile<4, NR>(x, wa, gr.order, tile.y, tile.z, part, k, rank, kb, ke, lds);
    else if (tile.z > 16)
        contract_tile<2, NR>(x, wa, gr.order, tile.y, tile.z, part, k, rank, kb, ke, lds);
    else
        contract_tile<1, NR>(x, wa, gr.order, tile.y, tile.z, part, k, rank, kb, ke, lds);
}

int contract_slices(int tile_bound, int64_t k) {
    const int64_t most = (k + 255) / 256;
    int64_t s = 1;
    while (s < 16 && s * 2 <= most && s * 2 * tile_bound <= 1024) s <<= 1;
    return static_cast<int>(s);
}

int launch_contract(const uint16_t* x, const uint16_t* w, const Groups& g, float* partials, int slices, int64_t tokens,
                    int64_t k, int rank, hipStream_t stream) {
    const int span = static_cast<int>(((k + slices - 1) / slices + 255) / 256 * 256);
    const dim3 grid(g.tile_bound, slices);
    const auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, x, w, g, partials, tokens, static_cast<int>(k), rank, span);
        return check_launch("contract_kernel");
    };
    if (rank <= 16) return run(contract_kernel<1>);
    if (rank <= 32) return run(contract_kernel<2>);
    if (rank <= 64) return run(contract_kernel<4>);
    return run(contract_kernel<8>);
}

// ---------------------------------------------------------------------------
// spread: out[i][j] = base[i][j] + s sum_c h[i][c] w[c][j].
// A workgroup takes a tile of up to 64 rows and 512 columns, a wave 128 of them. w lies
// across the MFMA's k (the ranks), so a lane loads 16 bytes of 8 rank rows and transposes
// the 8 x 8 block in registers (32 v_perm_b32); MFMA i then covers columns n0 + 8 l + i,
// and a lane ends with 8 neighbouring columns of a row: base and out move 16 bytes a lane.
// h enters as two bf16 parts (rest below 2^-16 of it, under the result's own rounding to
// bf16): for r <= 16 side by side in one MFMA's 32 k, else as two MFMAs on one w.
// ---------------------------------------------------------------------------
// The 8 x 8 block of 16-bit values v[j] (row j, two columns a dword) as B operands:
// column i of all rows.
__device__ __forceinline__ void transpose8(const u32x4_t (&v)[8], u32x4_t (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int p = 0; p < 4; ++p)
            b[i][p] = __builtin_amdgcn_perm(v[2 * p + 1][i / 2], v[2 * p][i / 2], (i & 1) ? 0x07060302u : 0x05040100u);
}

// NK: 32-rank chunks. HALF (r <= 16): one chunk whose k 0-15 are h's first parts and
// 16-31 the rests, w's rows twice. W32: w is fp32, taken as two bf16 parts as well
// (the product of the two rests, below 2^-32 of the term, is left out).
template <int NK, bool HALF, bool W32>
__global__ __launch_bounds__(256) void spread_kernel(const float* __restrict__ partials, int slices, const void* wv,
                                                     const float* __restrict__ scales, Groups gr, const uint16_t* base,
                                                     uint16_t* out, float* __restrict__ h_out, int64_t tokens,
                                                     int64_t width, int rank) {
    constexpr int KP = 32 * NK + 8;  // 16-byte rows, off the banks' period
    __shared__ __attribute__((aligned(16))) uint16_t hi[kTileRows * KP];
    __shared__ __attribute__((aligned(16))) uint16_t lo[HALF ? 8 : kTileRows * KP];
    __shared__ int32_t row_of[kTileRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l = lane & 15, g = lane >> 4;
    int adapter = 0, first = blockIdx.x * kTileRows, rows;
    if (gr.order) {
        if (static_cast<int>(blockIdx.x) >= gr.head[0]) return;
        const int4 tile = gr.tiles[blockIdx.x];
        adapter = tile.x;
        first = tile.y;
        rows = tile.z;
    } else {
        rows = static_cast<int>(min(static_cast<int64_t>(kTileRows), tokens - first));
    }
    if (tid < rows) row_of[tid] = gr.order ? gr.order[first + tid] : first + tid;
    const int64_t col = static_cast<int64_t>(blockIdx.y) * kSpreadCols + wave * 128 + 8 * l;
    const bool inside = col < width;
    const u32x4_t zero = {0, 0, 0, 0};
    if (adapter < 0) {  // no adapter: h is 0, the base as it is
        if (h_out && blockIdx.y == 0)
            for (int i = tid; i < rows * rank; i += 256) h_out[static_cast<int64_t>(first) * rank + i] = 0.0f;
        if (base == out || !out) return;
        __syncthreads();
        if (inside)
            for (int r = g; r < rows; r += 4) {
                const int64_t at = row_of[r] * width + col;
                *reinterpret_cast<u32x4_t*>(out + at) = base ? load16(base + at) : zero;
            }
        return;
    }
    // h: the slices' sums as bf16 parts; zero past the rank and past the rows.
    for (int i = tid; i < kTileRows * (HALF ? 16 : 32 * NK); i += 256) {
        const int row = i / (HALF ? 16 : 32 * NK), c = i % (HALF ? 16 : 32 * NK);
        float h = 0.0f;
        if (row < rows && c < rank) {
            const int64_t at = static_cast<int64_t>(first + row) * rank + c;
            for (int s = 0; s < slices; ++s) h += partials[static_cast<int64_t>(s) * tokens * rank + at];
            if (h_out && blockIdx.y == 0) h_out[at] = h;
        }
        const uint16_t a = f32_to_bf16(h);
        const uint16_t b = f32_to_bf16(bf16_rest(h, a));
        hi[row * KP + c] = a;
        if (HALF)
            hi[row * KP + 16 + c] = b;
        else
            lo[row * KP + c] = b;
    }
    // w's operands.
    u32x4_t b[NK][8], b2[W32 ? NK : 1][8];
#pragma unroll
    for (int n = 0; n < NK; ++n) {
        if (W32) {
            const float* w = static_cast<const float*>(wv);
            f32x4_t v[8][2];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = HALF ? (8 * g + j) & 15 : 32 * n + 8 * g + j;
                v[j][0] = v[j][1] = f32x4_t{0, 0, 0, 0};
                if (inside && c < rank) {
                    const float* src = w + static_cast<int64_t>(c) * width + col;
                    v[j][0] = *reinterpret_cast<const f32x4_t*>(src);
                    v[j][1] = *reinterpret_cast<const f32x4_t*>(src + 4);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float f0 = v[2 * p][i / 4][i % 4], f1 = v[2 * p + 1][i / 4][i % 4];
                    b[n][i][p] = pack_bf16x2(f0, f1);
                    b2[n][i][p] = pack_bf16x2(bf16_rest(f0, b[n][i][p]), bf16_rest(f1, b[n][i][p] >> 16));
                }
        } else {
            const uint16_t* w = static_cast<const uint16_t*>(wv) + static_cast<int64_t>(adapter) * rank * width;
            u32x4_t v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = HALF ? (8 * g + j) & 15 : 32 * n + 8 * g + j;
                v[j] = inside && c < rank ? load16(w + static_cast<int64_t>(c) * width + col) : zero;
            }
            transpose8(v, b[n]);
        }
    }
    if (!out) return;
    const float scale = scales ? scales[adapter] : 1.0f;
    __syncthreads();
#pragma unroll 1
    for (int m = 0; m < (rows + 15) / 16; ++m) {
        u32x4_t old[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = 16 * m + 4 * g + q;
            old[q] = base && inside && r < rows ? load16(base + row_of[r] * width + col) : zero;
        }
        f32x4_t acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            const int at = (16 * m + l) * KP + 32 * n + 8 * g;
            const u32x4_t a = *reinterpret_cast<const u32x4_t*>(hi + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = mfma(a, b[n][i], acc[i]);
            if (!HALF) {
                const u32x4_t a2 = *reinterpret_cast<const u32x4_t*>(lo + at);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = mfma(a2, b[n][i], acc[i]);
            }
            if (W32) {
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = mfma(a, b2[n][i], acc[i]);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = 16 * m + 4 * g + q;
            if (!inside || r >= rows) continue;
            u32x4_t o;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const float b0 = bf16_to_f32(static_cast<uint16_t>(old[q][d]));
                const float b1 = bf16_to_f32(static_cast<uint16_t>(old[q][d] >> 16));
                o[d] = pack_bf16x2(b0 + scale * acc[2 * d][q], b1 + scale * acc[2 * d + 1][q]);
            }
            *reinterpret_cast<u32x4_t*>(out + row_of[r] * width + col) = o;
        }
    }
}

int launch_spread(const float* partials, int slices, const void* w, bool w32, const float* scales, const Groups& g,
                  const uint16_t* base, uint16_t* out, float* h_out, int64_t tokens, int64_t width, int rank,
                  hipStream_t stream) {
    const unsigned columns = static_cast<unsigned>((width + kSpreadCols - 1) / kSpreadCols);
    const dim3 grid(g.tile_bound, out ? columns : 1);  // without out: h_out alone
    const auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, partials, slices, w, scales, g, base, out, h_out, tokens,
                           width, rank);
        return check_launch("spread_kernel");
    };
    if (w32) {  // the router: at most 64 experts
        if (rank <= 16) return run(spread_kernel<1, true, true>);
        if (rank <= 32) return run(spread_kernel<1, false, true>);
        return run(spread_kernel<2, false, true>);
    }
    if (rank <= 16) return run(spread_kernel<1, true, false>);
    if (rank <= 32) return run(spread_kernel<1, false, false>);
    if (rank <= 64) return run(spread_kernel<2, false, false>);
    return run(spread_kernel<4, false, false>);
}

// ---------------------------------------------------------------------------
// outer: out[c][j] = s sum_i h[i][c] x[i][j] over an adapter's rows.
// The rows are the MFMA's k. A workgroup takes a split of one adapter's rows and 128
// columns; its waves take 32 rows in turn. x's 8 x 8 blocks are transposed in registers
// as in spread; h (fp32, read along the ranks) enters as three bf16 parts, which hold
// all its bits, so each product is exact and sums in fp32. The waves' sums meet in LDS;
// an adapter of one split is done, of more its partial sums are added in split order.
// ---------------------------------------------------------------------------
template <bool BF16>
__device__ __forceinline__ void store8(void* out, int64_t at, const float (&v)[8]) {
    if (BF16) {
        u32x4_t o;
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = pack_bf16x2(v[2 * d], v[2 * d + 1]);
        *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(out) + at) = o;
    } else {
        float* p = static_cast<float*>(out) + at;
        *reinterpret_cast<f32x4_t*>(p) = f32x4_t{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
    }
}

template <int NR, bool BF16>
__global__ __launch_bounds__(256) void outer_kernel(const float* __restrict__ h, const uint16_t* __restrict__ x,
                                                    const float* __restrict__ scales, Groups gr,
                                                    float* __restrict__ partials, void* __restrict__ out,
                                                    int64_t tokens, int64_t width, int rank) {
    __shared__ __attribute__((aligned(16))) float lds[4 * 16 * 128];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l = lane & 15, g = lane >> 4;
    int adapter = 0, first = blockIdx.x * gr.split_rows, rows, parts = gr.split_bound;
    if (gr.order) {
        if (static_cast<int>(blockIdx.x) >= gr.head[1]) return;
        const int4 split = gr.splits[blockIdx.x];
        adapter = split.x;
        first = split.y;
        rows = split.z;
        parts = split.w;
    } else {
        rows = static_cast<int>(min(static_cast<int64_t>(gr.split_rows), tokens - first));
    }
    const int64_t col = static_cast<int64_t>(blockIdx.y) * kOuterCols + 8 * l;
    const bool inside = col < width;
    const int c0 = blockIdx.z * 16 * NR;
    const u32x4_t zero = {0, 0, 0, 0};
    f32x4_t acc[NR][8];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[n][i] = f32x4_t{0, 0, 0, 0};
    for (int t0 = 32 * wave; t0 < rows; t0 += 128) {
        u32x4_t v[8];
        float hv[NR][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = t0 + 8 * g + j;
            v[j] = zero;
            if (i < rows && inside) {
                const int64_t row = gr.order ? gr.order[first + i] : first + i;
                v[j] = load16(x + row * width + col);
            }
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int c = c0 + 16 * n + l;
                hv[n][j] = i < rows && c < rank ? h[static_cast<int64_t>(first + i) * rank + c] : 0.0f;
            }
        }
        u32x4_t b[8];
        transpose8(v, b);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            u32x4_t a0, a1, a2;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                float f0 = hv[n][2 * p], f1 = hv[n][2 * p + 1];
                a0[p] = pack_bf16x2(f0, f1);
                f0 = bf16_rest(f0, a0[p]);
                f1 = bf16_rest(f1, a0[p] >> 16);
                a1[p] = pack_bf16x2(f0, f1);
                a2[p] = pack_bf16x2(bf16_rest(f0, a1[p]), bf16_rest(f1, a1[p] >> 16));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[n][i] = mfma(a2, b[i], acc[n][i]);
                acc[n][i] = mfma(a1, b[i], acc[n][i]);
                acc[n][i] = mfma(a0, b[i], acc[n][i]);
            }
        }
    }
    const float scale = scales ? scales[adapter] : 1.0f;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        if (n > 0) __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float* dst = lds + (wave * 16 + 4 * g + q) * 128 + 8 * l;
            *reinterpret_cast<f32x4_t*>(dst) = f32x4_t{acc[n][0][q], acc[n][1][q], acc[n][2][q], acc[n][3][q]};
            *reinterpret_cast<f32x4_t*>(dst + 4) = f32x4_t{acc[n][4][q], acc[n][5][q], acc[n][6][q], acc[n][7][q]};
        }
        __syncthreads();
        const int c = c0 + 16 * n + tid / 16;
        const int64_t j = static_cast<int64_t>(blockIdx.y) * kOuterCols + 8 * (tid & 15);
        if (c < rank && j < width) {
            float v[8];
            const float* src = lds + (tid / 16) * 128 + 8 * (tid & 15);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = scale * (((src[i] + src[i + 2048]) + src[i + 4096]) + src[i + 6144]);
            if (parts == 1)
                store8<BF16>(out, (static_cast<int64_t>(adapter) * rank + c) * width + j, v);
            else
                store8<false>(partials, (static_cast<int64_t>(blockIdx.x) * rank + c) * width + j, v);
        }
    }
}

// An adapter's partial sums in split order, or zeros for one without rows.
template <bool BF16>
__global__ __launch_bounds__(256) void outer_sum_kernel(const float* __restrict__ partials, Groups gr,
                                                        void* __restrict__ out, int64_t elements) {
    const int a = blockIdx.y;
    const int s0 = gr.order ? gr.split_start[a] : 0;
    const int s1 = gr.order ? gr.split_start[a + 1] : gr.split_bound;
    if (s1 - s0 == 1) return;
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 8;
    if (at >= elements) return;
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int s = s0; s < s1; ++s) {
        const float* p = partials + static_cast<int64_t>(s) * elements + at;
        const f32x4_t lo = *reinterpret_cast<const f32x4_t*>(p), hi = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] += lo[i];
            v[4 + i] += hi[i];
        }
    }
    store8<BF16>(out, a * elements + at, v);
}

int launch_outer(const float* h, const uint16_t* x, const float* scales, const Groups& g, float* partials, void* out,
                 bool out_bf16, int64_t tokens, int64_t width, int rank, int adapters, hipStream_t stream) {
    const int nr = rank <= 16 ? 1 : rank <= 32 ? 2 : 4;
    const dim3 grid(g.split_bound, static_cast<unsigned>((width + kOuterCols - 1) / kOuterCols),
                    (rank + 16 * nr - 1) / (16 * nr));
    const auto run = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, h, x, scales, g, partials, out, tokens, width, rank);
        return check_launch("outer_kernel");
    };
    int rc = MOE_OK;
    if (g.split_bound == 0)
        rc = MOE_OK;  // no rows: zeros, below
    else if (out_bf16)
        rc = nr == 1 ? run(outer_kernel<1, true>) : nr == 2 ? run(outer_kernel<2, true>) : run(outer_kernel<4, true>);
    else
        rc = nr == 1 ? run(outer_kernel<1, false>) : nr == 2 ? run(outer_kernel<2, false>) : run(outer_kernel<4, false>);
    if (rc != MOE_OK || (!g.order && g.split_bound == 1)) return rc;
    const int64_t elements = rank * width;
    const dim3 sum_grid(static_cast<unsigned>((elements + 2047) / 2048), adapters);
    if (out_bf16)
        hipLaunchKernelGGL(outer_sum_kernel<true>, sum_grid, dim3(256), 0, stream, partials, g, out, elements);
    else
        hipLaunchKernelGGL(outer_sum_kernel<false>, sum_grid, dim3(256), 0, stream, partials, g, out, elements);
    return check_launch("outer_sum_kernel");
}

// ---------------------------------------------------------------------------
// The operators
// ---------------------------------------------------------------------------
static int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// Forward: contract's partial sums. Backward: those of dh, dh itself, outer's partial sums.
int64_t low_rank_scratch_bytes(int64_t tokens, int64_t hidden, int64_t width, int64_t rank, int64_t adapters,
                               bool backward) {
    const TableLayout t = table_layout(tokens, adapters);
    const int64_t row = tokens * rank * 4;
    if (!backward) return contract_slices(t.tile_bound, hidden) * row;
    return up16(contract_slices(t.tile_bound, width) * row) + up16(row) +
           static_cast<int64_t>(t.split_bound) * rank * std::max(hidden, width) * 4;
}

int launch_low_rank_add(const uint16_t* x, const uint16_t* down, const uint16_t* up, const float* scales,
                        const void* table, const uint16_t* base, uint16_t* output, float* hidden_out, char* scratch,
                        int64_t tokens, int64_t hidden, int64_t width, int rank, int adapters, hipStream_t stream) {
    const Groups g = groups_of(table, tokens, adapters);
    const int slices = contract_slices(g.tile_bound, hidden);
    float* partials = reinterpret_cast<float*>(scratch);
    int rc = launch_contract(x, down, g, partials, slices, tokens, hidden, rank, stream);
    if (rc == MOE_OK)
        rc = launch_spread(partials, slices, up, false, scales, g, base, output, hidden_out, tokens, width, rank, stream);
    return rc;
}

int launch_low_rank_backward(const uint16_t* grad_output, const uint16_t* x, const uint16_t* down, const uint16_t* up,
                             const float* scales, const void* table, const float* hidden_in, const uint16_t* grad_x_base,
                             uint16_t* grad_x, void* grad_down, void* grad_up, bool grad_bf16, char* scratch,
                             int64_t tokens, int64_t hidden, int64_t width, int rank, int adapters, hipStream_t stream) {
    const Groups g = groups_of(table, tokens, adapters);
    const int slices = contract_slices(g.tile_bound, width);
    const int64_t row = tokens * rank * 4;
    float* dh_parts = reinterpret_cast<float*>(scratch);
    float* dh = reinterpret_cast<float*>(scratch + up16(slices * row));
    float* partials = reinterpret_cast<float*>(scratch + up16(slices * row) + up16(row));
    int rc = MOE_OK;
    if (tokens > 0 && (grad_x || grad_down)) {
        rc = launch_contract(grad_output, up, g, dh_parts, slices, tokens, width, rank, stream);
        // dx, and dh's sum for the outer product (the spread alone has no output without grad_x).
        if (rc == MOE_OK)
            rc = launch_spread(dh_parts, slices, down, false, scales, g, grad_x_base, grad_x, dh, tokens, hidden, rank,
                               stream);
    }
    if (rc == MOE_OK && grad_down)
        rc = launch_outer(dh, x, scales, g, partials, grad_down, grad_bf16, tokens, hidden, rank, adapters, stream);
    if (rc == MOE_OK && grad_up)
        rc = launch_outer(hidden_in, grad_output, scales, g, partials, grad_up, grad_bf16, tokens, width, rank, adapters,
                          stream);
    return rc;
}

}  // namespace moe
