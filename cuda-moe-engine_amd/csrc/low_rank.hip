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

// Orders a wave's LDS accesses: what its lanes wrote before is there for all of them after.
// (A wave's LDS operations complete in order; this keeps the compiler from moving them.)
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// ---------------------------------------------------------------------------
// Rows sorted by adapter: a stable counting sort. A wave ranks 64 rows at a time among
// themselves (a ballot per bit of the group number) and behind its earlier rows (its own
// counts in LDS), so that no order depends on timing; the waves' counts are then added up
// in order, the groups scanned, and each row goes to its group's start plus its rank. Up
// to kChunkRows rows are one launch of one workgroup: latency (4096 rows of 8, 256 and
// 4096 adapters 7.5, 9.9 and 26 us, where a wave per adapter that looks through all rows
// took 12, 140 and 910). More rows are counted by chunk, scanned by one workgroup and
// placed by chunk (65536 rows 15, 18 and 46 us, where one workgroup counting took 190 to
// 206). A program groups once a step and uses the table for all its projections.
// ---------------------------------------------------------------------------
constexpr int kGroupThreads = 1024;

__device__ __forceinline__ int group_of(int id, int adapters) {
    return static_cast<unsigned>(id) < static_cast<unsigned>(adapters) ? id : adapters;
}

// This wave's rows of a chunk: each one's group and its rank among the wave's rows of that
// group, group << 16 | rank, and in counts [groups] how many the wave has of each.
template <int STEPS>
__device__ __forceinline__ void rank_rows(const int32_t* __restrict__ ids, int first, int tokens, int adapters,
                                          uint16_t* counts, uint32_t (&ranked)[STEPS]) {
    const int lane = threadIdx.x & 63;
    int group[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int i = first + 64 * s + lane;
        group[s] = i < tokens ? group_of(ids[i], adapters) : 0;
    }
    for (int a = lane; a <= adapters; a += 64) counts[a] = 0;
    wave_lds_order();
    const int bits = 32 - __clz(adapters);  // adapters >= 1: the groups are 0...adapters
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        uint64_t same = __ballot(first + 64 * s + lane < tokens);
        if (same == 0) break;
        const bool held = same >> lane & 1;
        for (int b = 0; b < bits; ++b) {
            const bool bit = group[s] >> b & 1;
            const uint64_t plane = __ballot(bit);
            same &= bit ? plane : ~plane;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int before = held ? counts[group[s]] : 0;
        wave_lds_order();
        if (held && rank == 0) counts[group[s]] = static_cast<uint16_t>(before + __popcll(same));
        wave_lds_order();
        ranked[s] = static_cast<uint32_t>(group[s]) << 16 | static_cast<uint32_t>(before + rank);
    }
}

// The waves' counts of a group become what the waves before them have; returns their sum.
template <int WAVES>
__device__ __forceinline__ int sum_waves(uint16_t* counts, int groups, int a) {
    uint16_t n[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) n[w] = counts[w * groups + a];
    int sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        counts[w * groups + a] = static_cast<uint16_t>(sum);
        sum += n[w];
    }
    return sum;
}

// An adapter's splits, and those of them whose sums are added up (none of an only one) in the
// upper 16 bits: a batch has at most kMaxAdapters + 2 kMaxAdapterTokens / kMaxSplitRows of
// them, and the halves are scanned as one.
__device__ __forceinline__ int split_counts(int rows, const TableLayout& t) {
    const int splits = (rows + t.split_rows - 1) >> __builtin_ctz(t.split_rows);
    return splits > 1 ? splits * 0x10001 : splits;
}

// start [groups + 1] in LDS: the groups' counts in, their starts out. Returns the first
// tile and split (with the first partial sum) of the thread's groups.
__device__ __forceinline__ int2 scan_groups(int32_t* start, const TableLayout& t, int tokens, int groups) {
    __shared__ int32_t wave_sums[3][kGroupThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (groups + kGroupThreads - 1) / kGroupThreads;
    const int g0 = min(tid * per, groups), g1 = min(g0 + per, groups);
    int rows = 0, tiles = 0, splits = 0;
    for (int a = g0; a < g1; ++a) {
        rows += start[a];
        tiles += (start[a] + kTileRows - 1) / kTileRows;
        if (a < groups - 1) splits += split_counts(start[a], t);
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
    int row = row_end - rows;
    for (int a = g0; a < g1; ++a) {
        const int n = start[a];
        start[a] = row;
        row += n;
    }
    if (tid == 0) start[groups] = tokens;
    return make_int2(tile_end - tiles, split_end - splits);
}

// The table's parts but the rows, an entry a thread: a tile's or split's group is found in
// LDS (first_of, twice groups + 1 entries).
__device__ __forceinline__ void write_table(const int32_t* start, int32_t* first_of, int2 first,
                                            int32_t* __restrict__ table, const TableLayout& t, int groups) {
    const int tid = threadIdx.x;
    const int per = (groups + kGroupThreads - 1) / kGroupThreads;
    const int g0 = min(tid * per, groups), g1 = min(g0 + per, groups);
    int32_t *tile_of = first_of, *split_of = first_of + groups + 1;
    int tile = first.x, split = first.y;
    for (int a = g0; a < g1; ++a) {
        const int n = start[a + 1] - start[a];
        tile_of[a] = tile;
        split_of[a] = split;
        tile += (n + kTileRows - 1) / kTileRows;
        if (a < groups - 1) {
            split += split_counts(n, t);
        } else {
            tile_of[groups] = tile;
            split_of[groups] = split;
        }
    }
    __syncthreads();
    for (int a = tid; a <= groups; a += kGroupThreads) table[t.starts + a] = start[a];
    for (int a = tid; a < groups; a += kGroupThreads)
        table[t.partial_start + a] = split_of[a] >> 16 << 1 | (start[a] < start[a + 1]);
    if (tid < 4) table[tid] = tid == 0 ? tile_of[groups] : tid == 1 ? split_of[groups] & 0xffff : 0;
    const auto write = [&](const int32_t* firsts, int mask, int rows, int4* to, auto last) {
        const auto entry = [&](int a) { return firsts[a] & mask; };
        const int count = entry(groups);
        for (int i = tid; i < count; i += kGroupThreads) {
            int low = 0, high = groups;  // entry(low) <= i < entry(high)
            while (high - low > 1) {
                const int mid = (low + high) / 2;
                if (entry(mid) <= i)
                    low = mid;
                else
                    high = mid;
            }
            const int at = start[low] + (i - entry(low)) * rows;
            to[i] = make_int4(low < groups - 1 ? low : -1, at, min(rows, start[low + 1] - at),
                              last(low, i - entry(low)));
        }
    };
    write(tile_of, -1, kTileRows, reinterpret_cast<int4*>(table + t.tiles), [](int, int) { return 0; });
    write(split_of, 0xffff, t.split_rows, reinterpret_cast<int4*>(table + t.splits), [&](int a, int i) {
        return split_of[a + 1] - split_of[a] == 1 ? -1 : (split_of[a] >> 16) + i;  // one split, none added up
    });
}

// All rows of a small batch, ranked by the first WAVES waves.
template <int WAVES>
__global__ __launch_bounds__(kGroupThreads) void adapter_group_kernel(const int32_t* __restrict__ ids,
                                                                      int32_t* __restrict__ table, TableLayout t,
                                                                      int tokens, int adapters) {
    constexpr int STEPS = kChunkRows / (64 * WAVES);
    extern __shared__ int32_t lds[];
    const int groups = adapters + 1;
    int32_t* start = lds;                                              // [groups + 1]
    uint16_t* counts = reinterpret_cast<uint16_t*>(lds + groups + 1);  // [WAVES][groups], then tile_of and split_of
    const int tid = threadIdx.x, wave = tid >> 6;
    const int steps = (tokens + 64 * WAVES - 1) / (64 * WAVES), first = wave * 64 * steps;
    uint32_t ranked[STEPS];
    if (wave < WAVES)
        rank_rows<STEPS>(ids, first, min(first + 64 * steps, tokens), adapters, counts + wave * groups, ranked);
    __syncthreads();
    for (int a = tid; a < groups; a += kGroupThreads) start[a] = sum_waves<WAVES>(counts, groups, a);
    __syncthreads();
    const int2 tables = scan_groups(start, t, tokens, groups);
    __syncthreads();
    if (wave < WAVES) {
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
            const int i = first + 64 * s + (tid & 63), group = ranked[s] >> 16;
            if (s < steps && i < tokens)
                table[t.order + start[group] + counts[wave * groups + group] + (ranked[s] & 0xffff)] = i;
        }
    }
    __syncthreads();
    write_table(start, reinterpret_cast<int32_t*>(counts), tables, table, t, groups);
}

// Larger batches: each chunk's counts,
__global__ __launch_bounds__(256) void adapter_count_kernel(const int32_t* __restrict__ ids, int32_t* __restrict__ table,
                                                            TableLayout t, int tokens, int adapters) {
    extern __shared__ int32_t lds[];
    const int tid = threadIdx.x, groups = adapters + 1;
    for (int a = tid; a < groups; a += 256) lds[a] = 0;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kChunkRows / 256; ++s) {
        const int i = blockIdx.x * kChunkRows + 256 * s + tid;
        if (i >= tokens) break;
        // Rows of a request are neighbours: one add for a wave of one group.
        const int a = group_of(ids[i], adapters);
        const uint64_t active = __ballot(1);
        if (__ballot(a == __builtin_amdgcn_readfirstlane(a)) == active) {
            if ((tid & 63) == 0) atomicAdd(&lds[a], __popcll(active));
        } else {
            atomicAdd(&lds[a], 1);
        }
    }
    __syncthreads();
    for (int a = tid; a < groups; a += 256) table[t.chunks + static_cast<int64_t>(blockIdx.x) * groups + a] = lds[a];
}

// their sums over the chunks before, the starts and the tables,
__global__ __launch_bounds__(kGroupThreads) void adapter_scan_kernel(int32_t* __restrict__ table, TableLayout t, int tokens,
                                                                    int adapters, int chunks) {
    extern __shared__ int32_t lds[];
    const int groups = adapters + 1;
    int32_t *start = lds, *first_of = lds + groups + 1;
    constexpr int U = 16;  // chunks in flight
    for (int a = threadIdx.x; a < groups; a += kGroupThreads) {
        int32_t* count = table + t.chunks + a;
        int sum = 0;
        for (int c0 = 0; c0 < chunks; c0 += U) {
            int n[U];
#pragma unroll
            for (int u = 0; u < U; ++u) n[u] = c0 + u < chunks ? count[static_cast<int64_t>(c0 + u) * groups] : 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (c0 + u < chunks) count[static_cast<int64_t>(c0 + u) * groups] = sum;
                sum += n[u];
            }
        }
        start[a] = sum;
    }
    __syncthreads();
    const int2 tables = scan_groups(start, t, tokens, groups);
    __syncthreads();
    write_table(start, first_of, tables, table, t, groups);
}

// and the rows to their places: never past the table, whatever the ids have become since
// they were counted.
template <int WAVES>
__global__ __launch_bounds__(64 * WAVES) void adapter_place_kernel(const int32_t* __restrict__ ids,
                                                                   int32_t* __restrict__ table, TableLayout t, int tokens,
                                                                   int adapters) {
    constexpr int STEPS = kChunkRows / (64 * WAVES);
    extern __shared__ int32_t lds[];
    const int groups = adapters + 1;
    int32_t* start = lds;
    uint16_t* counts = reinterpret_cast<uint16_t*>(lds + groups + 1);
    const int tid = threadIdx.x, wave = tid >> 6;
    const int first = blockIdx.x * kChunkRows + wave * 64 * STEPS;
    uint32_t ranked[STEPS];
    rank_rows<STEPS>(ids, first, tokens, adapters, counts + wave * groups, ranked);
    __syncthreads();
    for (int a = tid; a < groups; a += 64 * WAVES) {
        start[a] = table[t.starts + a] + table[t.chunks + static_cast<int64_t>(blockIdx.x) * groups + a];
        sum_waves<WAVES>(counts, groups, a);
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        const int i = first + 64 * s + (tid & 63), group = ranked[s] >> 16;
        if (i >= tokens) break;
        const int at = start[group] + counts[wave * groups + group] + (ranked[s] & 0xffff);
        if (at < tokens) table[t.order + at] = i;
    }
}

int launch_adapter_group(const int32_t* ids, void* table, int64_t tokens, int adapters, hipStream_t stream) {
    const TableLayout t = table_layout(tokens, adapters);
    int32_t* base = static_cast<int32_t*>(table);
    const int rows = static_cast<int>(tokens), groups = adapters + 1;
    // Sixteen waves' counts, or four's, within 64 KiB of LDS beside the starts.
    const bool many = groups > 1536;
    const size_t lds = (groups + 1) * 4 + std::max((many ? 4 : 16) * groups * 2, 2 * (groups + 1) * 4);
    if (t.chunk_count == 0) {
        const auto kernel = many ? adapter_group_kernel<4> : adapter_group_kernel<16>;
        hipLaunchKernelGGL(kernel, dim3(1), dim3(kGroupThreads), lds, stream, ids, base, t, rows, adapters);
        return check_launch("adapter_group_kernel");
    }
    const dim3 chunks(t.chunk_count);
    hipLaunchKernelGGL(adapter_count_kernel, chunks, dim3(256), groups * 4, stream, ids, base, t, rows, adapters);
    int rc = check_launch("adapter_count_kernel");
    if (rc != MOE_OK) return rc;
    hipLaunchKernelGGL(adapter_scan_kernel, dim3(1), dim3(kGroupThreads), 3 * (groups + 1) * 4, stream, base, t, rows,
                       adapters, t.chunk_count);
    rc = check_launch("adapter_scan_kernel");
    if (rc != MOE_OK) return rc;
    if (many)
        hipLaunchKernelGGL(adapter_place_kernel<4>, chunks, dim3(256), lds, stream, ids, base, t, rows, adapters);
    else
        hipLaunchKernelGGL(adapter_place_kernel<16>, chunks, dim3(1024), lds, stream, ids, base, t, rows, adapters);
    return check_launch("adapter_place_kernel");
}

// ---------------------------------------------------------------------------
// contract: h[i][c] = sum_k x[i][k] w[c][k].
// A workgroup takes a tile of up to 64 rows of one adapter and a slice of k. A wave takes
// 16 rows and the slice, or for r > 32, where w's lines are the more, 32 rows and half of
// it; with fewer rows in the tile more waves share them and split the slice. Up to 64 ranks
// take eight waves and half the slices (rank 16 in eight waves spills: 29.4 -> 32.5 us with
// spread). Eight lanes load a 128-byte line of a row, D steps of 64 k ahead, and the wave
// turns the step over in LDS of its own into the MFMA's operands (lane l: row l % 16, 8 k
// from 8 (l / 16); k is permuted inside 64). Loaded as operands, neighbouring lanes hold different rows and each
// 16 bytes is a line of its own to the L1: T=4096, H=4096, r=16 and 64 took 17.2 and 38.6
// us, 11.1 and 15.9 now. Its 33.5 MB of x are 6.5 us at a copy's rate, and outer reads as
// many in 8.8: no bound is known for the rest. Rows
// past the tile and ranks past r are read from the last one and not stored (an output
// depends on its own row and rank alone). Waves on one row meet in LDS, slices in the
// consumer, both in order. Past 64 ranks (21.7 us at r=128) the LDS that turns w's lines
// over for 32 rows takes longer than x's bytes.
// ---------------------------------------------------------------------------
// 16 rows of 64 k: lane i loads piece i % 8 (8 k) of rows i / 8 and i / 8 + 8.
struct LineRows {
    const uint16_t* row[2];
};
struct Lines {
    u32x4_t v[2];
};

__device__ __forceinline__ void load_lines(Lines& s, const LineRows& r, int at, int k) {
    const u32x4_t zero = {0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) s.v[h] = at < k ? load16(r.row[h] + at) : zero;
}
// Of `rows` rows: the others are zeros that cost no traffic (decoding 8.1 -> 7.9 us, 777 rows
// 12.6 -> 12.4; contract, whose loads wait on HBM, gains nothing).
__device__ __forceinline__ void load_lines(Lines& s, const LineRows& r, int at, int k, int rows, int lane) {
    const u32x4_t zero = {0, 0, 0, 0};
#pragma unroll
    for (int h = 0; h < 2; ++h) s.v[h] = at < k && lane / 8 + 8 * h < rows ? load16(r.row[h] + at) : zero;
}

// A wave's 2 KiB: piece p of row r lies at slot p ^ (r % 8) of its 128 bytes, so that the
// operands' 16 rows fall on different banks.
__device__ __forceinline__ void put_lines(uint16_t* lds, const Lines& s, int lane) {
    const int row = lane / 8, slot = (lane % 8) ^ row;
    *reinterpret_cast<u32x4_t*>(lds + row * 64 + slot * 8) = s.v[0];
    *reinterpret_cast<u32x4_t*>(lds + (row + 8) * 64 + slot * 8) = s.v[1];
}
__device__ __forceinline__ u32x4_t get_operand(const uint16_t* lds, int l, int g, int h) {
    return *reinterpret_cast<const u32x4_t*>(lds + l * 64 + (((2 * g + h) ^ (l & 7)) * 8));
}

// NR: 16-rank fragments. F: 16-row fragments a wave. W: waves.
template <int NR, int F, int W>
__global__ __launch_bounds__(64 * W) void contract_kernel(const uint16_t* __restrict__ x, const uint16_t* __restrict__ w,
                                                       Groups gr, float* __restrict__ partials, int64_t tokens, int k,
                                                       int rank, int span) {
    constexpr int D = NR <= 2 ? 6 : NR == 4 ? 3 : 2;  // steps in flight
    constexpr int C = 16 * NR;
    constexpr int kWaveHalfs = 1024 * (F + NR);  // x's fragments and w's
    __shared__ __attribute__((aligned(16))) uint16_t lines[W * kWaveHalfs];
    const int4 tile = gr.tiles[blockIdx.x];
    if (static_cast<int>(blockIdx.x) >= gr.head[0] || tile.x < 0) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int l = lane & 15, g = lane >> 4;
    const int first = tile.y, rows = tile.z;
    // Waves on the same rows, this wave's rows and its part of the slice.
    const int kw = (rows > 32 ? F : rows > 16 ? 2 * F : 4) * (W / 4);
    const int m = wave / kw, kpart = wave % kw;
    const bool two = F == 2 && rows - 32 * m > 16;
    const int kb = blockIdx.y * span + kpart * (span / kw);
    const int ke = 16 * F * m < rows ? min(kb + span / kw, k) : 0;
    f32x4_t acc[F][NR];
#pragma unroll
    for (int f = 0; f < F; ++f)
#pragma unroll
        for (int n = 0; n < NR; ++n) acc[f][n] = f32x4_t{0, 0, 0, 0};
    if (kb < ke) {
        LineRows xr[F], wr[NR];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = lane / 8 + 8 * h;
#pragma unroll
            for (int f = 0; f < F; ++f)
                xr[f].row[h] = x + static_cast<int64_t>(gr.order[first + min(16 * (F * m + f) + r, rows - 1)]) * k;
#pragma unroll
            for (int n = 0; n < NR; ++n)
                wr[n].row[h] = w + (static_cast<int64_t>(tile.x) * rank + min(16 * n + r, rank - 1)) * k;
        }
        struct Step {
            Lines x[F], w[NR];
        };
        Step ring[D];
        const auto fetch = [&](Step& s, int k0) {
            const int at = k0 + 8 * (lane % 8);
            load_lines(s.x[0], xr[0], at, k);
            if (two) load_lines(s.x[F - 1], xr[F - 1], at, k);
#pragma unroll
            for (int n = 0; n < NR; ++n) load_lines(s.w[n], wr[n], at, k);
        };
        uint16_t* mine = lines + wave * kWaveHalfs;
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (kb + 64 * d < ke) fetch(ring[d], kb + 64 * d);
        for (int k0 = kb; k0 < ke; k0 += 64 * D)
#pragma unroll
            for (int d = 0; d < D; ++d)
                if (k0 + 64 * d < ke) {
                    put_lines(mine, ring[d].x[0], lane);
                    if (two) put_lines(mine + 1024, ring[d].x[F - 1], lane);
#pragma unroll
                    for (int n = 0; n < NR; ++n) put_lines(mine + 1024 * (F + n), ring[d].w[n], lane);
                    wave_lds_order();
                    const int ahead = k0 + 64 * (d + D);
                    if (ahead < ke) fetch(ring[d], ahead);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const u32x4_t a = get_operand(mine, l, g, h);
                        u32x4_t b[NR];
#pragma unroll
                        for (int n = 0; n < NR; ++n) {
                            b[n] = get_operand(mine + 1024 * (F + n), l, g, h);
                            acc[0][n] = mfma(a, b[n], acc[0][n]);
                        }
                        if (two) {
                            const u32x4_t a1 = get_operand(mine + 1024, l, g, h);
#pragma unroll
                            for (int n = 0; n < NR; ++n) acc[F - 1][n] = mfma(a1, b[n], acc[F - 1][n]);
                        }
                    }
                    wave_lds_order();
                }
    }
    // The other waves of the rows pass their sums to the first, a fragment at a time
    // through the same LDS.
    float* lds = reinterpret_cast<float*>(lines);
    float* part = partials + (static_cast<int64_t>(blockIdx.y) * tokens + first + 16 * F * m) * rank;
#pragma unroll
    for (int f = 0; f < F; ++f) {
        if (kw > 1) __syncthreads();
        if (kpart > 0) {
            float* dst = lds + (m * (kw - 1) + kpart - 1) * 16 * C;
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q) dst[(4 * g + q) * C + 16 * n + l] = acc[f][n][q];
        }
        if (kw > 1) __syncthreads();
        if (kpart > 0) continue;
        for (int p = 1; p < kw; ++p) {
            const float* src = lds + (m * (kw - 1) + p - 1) * 16 * C;
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q) acc[f][n][q] += src[(4 * g + q) * C + 16 * n + l];
        }
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int r = 16 * f + 4 * g + q;
                if (16 * F * m + r < rows && 16 * n + l < rank) part[r * rank + 16 * n + l] = acc[f][n][q];
            }
    }
}

// Up to about 600 workgroups of the tiles that the table could hold; past 32 ranks, where
// spread reads each slice's sums again for every 256 columns, 512, or one a CU of the eight
// waves of up to 64 ranks (contract and spread of 8192 x 4096 to 4096, rank 16: 46.9 us, with
// 512 50.5; of 4096 rows, rank 64: 45.5 with three slices, 46.3 with two, 46.8 with four of
// four waves; of 1024 rows 20.1 and 22.6; of 16384, rank 128: 158, with 600 168). The host
// knows the bank and not how many of its adapters a batch uses, so few adapters of a large one
// get few slices (contract and spread of 4096 rows of six adapters beside 8, 64 and 256, rank
// 16: 25.5, 30.3 and 55.4 us, rank 64: 38.7, 49.7 and 74.1). Ranks 17 to 32 and past 64 keep
// fewer workgroups on a CU than their rule supposes (186 registers; one workgroup).
int contract_slices(int tile_bound, int64_t k, int64_t rank) {
    const bool wide = rank > 32 && rank <= 64;
    const int64_t most = wide ? (k + 511) / 512 : (k + 255) / 256;
    const int64_t workgroups = rank <= 32 ? 600 : wide ? 256 : 512;
    int best = 1;
    for (int s : {2, 3, 4, 8, 16})
        if (s <= most && static_cast<int64_t>(s) * tile_bound <= workgroups) best = s;
    return best;
}

int launch_contract(const uint16_t* x, const uint16_t* w, const Groups& g, float* partials, int slices, int64_t tokens,
                    int64_t k, int rank, hipStream_t stream) {
    const dim3 grid(g.tile_bound, slices);
    const auto run = [&](auto kernel, int waves) {
        const int unit = 64 * waves;  // whole steps for every wave
        const int span = static_cast<int>(((k + slices - 1) / slices + unit - 1) / unit * unit);
        hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, stream, x, w, g, partials, tokens, static_cast<int>(k),
                           rank, span);
        return check_launch("contract_kernel");
    };
    if (rank <= 16) return run(contract_kernel<1, 1, 4>, 4);
    if (rank <= 32) return run(contract_kernel<2, 1, 4>, 4);
    if (rank <= 64) return run(contract_kernel<4, 2, 8>, 8);
    return run(contract_kernel<8, 2, 4>, 4);
}

// Workgroup b as (column part, row part), the column parts of a row part next to each
// other on one XCD (b % 8 is its XCD): an XCD then meets few adapters, whose w stays in
// its L2 (T=4096, 4096 columns, r=64 of eight adapters: 24.8 -> 22.8 us).
__device__ __forceinline__ bool part_of(int columns, int rows, int* column, int* row) {
    const int per = gridDim.x / kNumXcd;
    const int i = (blockIdx.x % kNumXcd) * per + blockIdx.x / kNumXcd;
    *column = i % columns;
    *row = i / columns;
    return *row < rows;
}
static unsigned part_grid(int64_t columns, int64_t rows) {
    return static_cast<unsigned>((columns * rows + kNumXcd - 1) / kNumXcd * kNumXcd);
}

// ---------------------------------------------------------------------------
// spread: out[i][j] = base[i][j] + s sum_c h[i][c] w[c][j].
// A workgroup takes a tile of up to 64 rows and 512 columns (256), a wave 128 of them. w
// lies across the MFMA's k (the ranks), so a lane loads 8 (4) columns of 8 rank rows and
// transposes the block in registers (v_perm_b32); MFMA i then covers columns n0 + 8 l + i,
// and a lane ends with 8 neighbouring columns of a row: base and out move 16 bytes a lane.
// h enters as two bf16 parts (rest below 2^-16 of it, under the result's own rounding to
// bf16): for r <= 16 side by side in one MFMA's 32 k, else as two MFMAs on one w. Bound by
// base's and out's bytes: 67 MB (T=4096, 4096 columns) at r=16 in 17.9 us on average and 14.1
// at best inside a training pass, 3.8 and 4.8 TB/s; at r=64 22.8 and at r=128 35, where
// every column part reads the slices' sums of h again.
// ---------------------------------------------------------------------------
// The 8 x N block of 16-bit values v[j] (row j, two columns a dword) as B operands:
// column i of all rows.
template <int N, typename V>
__device__ __forceinline__ void transpose8(const V (&v)[8], u32x4_t (&b)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int p = 0; p < 4; ++p)
            b[i][p] = __builtin_amdgcn_perm(v[2 * p + 1][i / 2], v[2 * p][i / 2], (i & 1) ? 0x07060302u : 0x05040100u);
}

// NK: 32-rank chunks. HALF (r <= 16): one chunk whose k 0-15 are h's first parts and
// 16-31 the rests, w's rows twice. W32: w is fp32, taken as two bf16 parts as well
// (the product of the two rests, below 2^-16 of the term, is left out). A workgroup takes
// `fragments` 16-row fragments of a tile, blockIdx.z the first: the whole tile, or 2 or 1
// where whole tiles would leave CUs idle. base's rows are on their way one fragment ahead.
// COLS: columns a lane, 8, or 4 where w's operands for 8 would leave a SIMD one wave
// (r > 32, fp32 w). STREAM: base is read past the caches.
template <int NK, bool HALF, bool W32, int COLS, bool STREAM>
__global__ __launch_bounds__(256, NK == 1 && !W32 ? 3 : 1) void spread_kernel(
    const float* __restrict__ partials, int slices, const void* wv, const float* __restrict__ scales, Groups gr,
    const uint16_t* base, uint16_t* out, float* __restrict__ h_out, int64_t tokens, int64_t width, int rank,
    int fragments, int columns) {
    constexpr int KP = 32 * NK + 8;  // 16-byte rows, off the banks' period
    constexpr int C = HALF ? 16 : 32 * NK;
    constexpr int R = W32 && NK == 2 ? kWideTileRows : kTileRows;
    __shared__ __attribute__((aligned(16))) uint16_t hi[R * KP];
    __shared__ __attribute__((aligned(16))) uint16_t lo[HALF ? 8 : R * KP];
    __shared__ int32_t row_of[R];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l = lane & 15, g = lane >> 4;
    int chunk, at_tile;
    if (!part_of(columns, gr.tile_bound, &chunk, &at_tile)) return;
    int adapter = 0, first = at_tile * R, rows;
    if (gr.order) {
        const int4 tile = gr.tiles[at_tile];
        if (at_tile >= gr.head[0]) return;
        adapter = tile.x;
        first = tile.y;
        rows = tile.z;
    } else {
        rows = static_cast<int>(min(static_cast<int64_t>(R), tokens - first));
    }
    first += 16 * fragments * blockIdx.z;
    rows = min(rows - static_cast<int>(16 * fragments * blockIdx.z), 16 * fragments);
    if (rows <= 0) return;
    const int64_t col = static_cast<int64_t>(chunk) * (64 * COLS) + (wave * 16 + l) * COLS;
    const bool inside = col < width;
    typedef uint32_t cols_t __attribute__((ext_vector_type(COLS / 2)));  // 16-bit columns
    typedef float wide_t __attribute__((ext_vector_type(COLS)));
    const cols_t zero = {};
    // What a workgroup asks memory for, in this order and without a wait between but the one
    // for its first rows' numbers: row numbers, w, base's first rows, h.
    const auto listed = [&](int r) { return gr.order ? gr.order[first + r] : first + r; };
    const auto kept = [&](int r) { return row_of[r]; };
    const int own_row = tid < rows ? listed(tid) : 0;
    int first_rows[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) first_rows[q] = listed(min(4 * g + q, rows - 1));
    const auto from_base = [](const uint16_t* p) {
        const cols_t* v = reinterpret_cast<const cols_t*>(p);
        if constexpr (STREAM) return __builtin_nontemporal_load(v);
        return *v;
    };
    // This lane's rows of a fragment, 16 m + 4 g + q, and what base has there.
    int64_t at[4];
    cols_t old[4];
    const auto fetch = [&](int m, auto row) {
#pragma unroll
        for (int q = 0; q < 4; ++q) at[q] = row(min(16 * m + 4 * g + q, rows - 1)) * width + col;
#pragma unroll
        for (int q = 0; q < 4; ++q) old[q] = base && inside ? from_base(base + at[q]) : zero;
    };
    if (adapter < 0) {  // no adapter: h is 0, the base as it is
        if (h_out && chunk == 0)
            for (int i = tid; i < rows * rank; i += 256) h_out[static_cast<int64_t>(first) * rank + i] = 0.0f;
        if (base == out || !out || !inside) return;
        for (int m = 0; 16 * m < rows; ++m) {
            fetch(m, listed);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (16 * m + 4 * g + q < rows) *reinterpret_cast<cols_t*>(out + at[q]) = old[q];
        }
        return;
    }
    u32x4_t b[NK][COLS], b2[W32 ? NK : 1][COLS];
    cols_t raw[W32 ? 1 : NK][8];
    wide_t raw32[W32 ? NK : 1][8];
    const int64_t skip = static_cast<int64_t>(adapter) * rank * width;
    const uint16_t* wa = static_cast<const uint16_t*>(wv) + skip;
    const float* wf = static_cast<const float*>(wv) + skip;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = HALF ? (8 * g + j) & 15 : 32 * n + 8 * g + j;
            // A scalar base and a 32-bit offset (rank * width is below 2^28).
            const uint32_t from = static_cast<uint32_t>(c) * static_cast<uint32_t>(width) + static_cast<uint32_t>(col);
            const bool held = inside && c < rank;
            if constexpr (W32)
                raw32[n][j] = held ? *reinterpret_cast<const wide_t*>(wf + from) : wide_t{};
            else
                raw[n][j] = held ? *reinterpret_cast<const cols_t*>(wa + from) : zero;
        }
    if (out) {
#pragma unroll
        for (int q = 0; q < 4; ++q) at[q] = first_rows[q] * width + col;
#pragma unroll
        for (int q = 0; q < 4; ++q) old[q] = base && inside ? from_base(base + at[q]) : zero;
    }
    // h: the slices' sums as bf16 parts; zero past the rank and past the rows, up to a
    // whole fragment. A thread takes four ranks of a row, U rows and S slices in flight.
    constexpr int Q = C / 4;
    const int filled = (rows + 15) / 16 * 16 * Q;
    const int64_t slice = tokens * rank;
    const auto stage = [&](auto count) {
        constexpr int S = decltype(count)::value, U = C >= 64 && S <= 4 && S != 3 ? 2 : 1;
        using V = Unaligned<float, 4>;
#pragma unroll 1
        for (int i0 = tid; i0 < filled; i0 += 256 * U) {
            float h[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) h[u][j] = 0.0f;
#pragma unroll 1
            for (int s0 = 0; s0 < slices; s0 += S) {
                V part[U][S];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + 256 * u, row = i / Q, c = i % Q * 4;
                    const uint32_t from = static_cast<uint32_t>(first + row) * rank + c;  // below 2^28
#pragma unroll
                    for (int s = 0; s < S; ++s) {
                        part[u][s] = V{{0, 0, 0, 0}};
                        if (row < rows) {
                            const float* src = partials + (s0 + s) * slice + from;
                            if (c + 4 <= rank) {
                                part[u][s] = *reinterpret_cast<const V*>(src);
                            } else {
#pragma unroll
                                for (int j = 0; j < 3; ++j)
                                    if (c + j < rank) part[u][s].v[j] = src[j];
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
#pragma unroll
                    for (int s = 0; s < S; ++s)
#pragma unroll
                        for (int j = 0; j < 4; ++j) h[u][j] += part[u][s].v[j];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 256 * u, row = i / Q, c = i % Q * 4;
                if (i >= filled) break;
                uint16_t a[4], rest[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (h_out && chunk == 0 && row < rows && c + j < rank)
                        h_out[static_cast<uint32_t>(first + row) * rank + c + j] = h[u][j];
                    a[j] = f32_to_bf16(h[u][j]);
                    rest[j] = f32_to_bf16(bf16_rest(h[u][j], a[j]));
                }
                const auto two = [](uint16_t x, uint16_t y) { return x | static_cast<uint32_t>(y) << 16; };
                uint16_t* other = HALF ? hi + row * KP + 16 + c : lo + row * KP + c;
                *reinterpret_cast<uint2*>(hi + row * KP + c) = make_uint2(two(a[0], a[1]), two(a[2], a[3]));
                *reinterpret_cast<uint2*>(other) = make_uint2(two(rest[0], rest[1]), two(rest[2], rest[3]));
            }
        }
    };
    if constexpr (W32)  // the router's gradient is one
        stage(std::integral_constant<int, 1>{});
    else switch (slices) {
        case 1: stage(std::integral_constant<int, 1>{}); break;
        case 2: stage(std::integral_constant<int, 2>{}); break;
        case 3: stage(std::integral_constant<int, 3>{}); break;
        case 4: stage(std::integral_constant<int, 4>{}); break;
        default: stage(std::integral_constant<int, 8>{}); break;
    }
    if (!out) return;
    if (tid < rows) row_of[tid] = own_row;
    const float scale = scales ? scales[adapter] : 1.0f;
    __syncthreads();
    const int last = (rows - 1) / 16;
#pragma unroll
    for (int n = 0; n < NK; ++n) {
        if constexpr (W32) {
#pragma unroll
            for (int i = 0; i < COLS; ++i)
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    const float f0 = raw32[n][2 * p][i], f1 = raw32[n][2 * p + 1][i];
                    b[n][i][p] = pack_bf16x2(f0, f1);
                    b2[n][i][p] = pack_bf16x2(bf16_rest(f0, b[n][i][p]), bf16_rest(f1, b[n][i][p] >> 16));
                }
        } else {
            transpose8(raw[n], b[n]);
        }
    }
#pragma unroll 1
    for (int m = 0; m <= last; ++m) {
        int64_t now[4];
        cols_t there[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            now[q] = at[q];
            there[q] = old[q];
        }
        if (m < last) fetch(m + 1, kept);
        f32x4_t acc[COLS];
#pragma unroll
        for (int i = 0; i < COLS; ++i) acc[i] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            const int from = (16 * m + l) * KP + 32 * n + 8 * g;
            const u32x4_t a = *reinterpret_cast<const u32x4_t*>(hi + from);
#pragma unroll
            for (int i = 0; i < COLS; ++i) acc[i] = mfma(a, b[n][i], acc[i]);
            if (!HALF) {
                const u32x4_t a2 = *reinterpret_cast<const u32x4_t*>(lo + from);
#pragma unroll
                for (int i = 0; i < COLS; ++i) acc[i] = mfma(a2, b[n][i], acc[i]);
            }
            if (W32) {
#pragma unroll
                for (int i = 0; i < COLS; ++i) acc[i] = mfma(a, b2[n][i], acc[i]);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (!inside || 16 * m + 4 * g + q >= rows) continue;
            cols_t o;
#pragma unroll
            for (int d = 0; d < COLS / 2; ++d) {
                const float b0 = bf16_to_f32(static_cast<uint16_t>(there[q][d]));
                const float b1 = bf16_to_f32(static_cast<uint16_t>(there[q][d] >> 16));
                o[d] = pack_bf16x2(b0 + scale * acc[2 * d][q], b1 + scale * acc[2 * d + 1][q]);
            }
            __builtin_nontemporal_store(o, reinterpret_cast<cols_t*>(out + now[q]));
        }
    }
}

// Results are stored past the caches, which then hold what the next workgroups read (1024
// rows of 4096 columns with contract, rank 16: 15.2 -> 14.2 us; 4096 rows 29.5 -> 30.8 with
// nothing in the caches, the same behind the kernels that wrote x and base), and from 48 MB
// of base on it is read that way too (8192 rows behind those kernels, rank 16 and 64: 46.8
// -> 39.7 and 68 -> 61, 71 -> 70 with nothing in the caches; at 32 MB and less it lost up to
// 8%).
constexpr int64_t kStreamElements = 24 << 20;

int launch_spread(const float* partials, int slices, const void* w, bool w32, const float* scales, const Groups& g,
                  const uint16_t* base, uint16_t* out, float* h_out, int64_t tokens, int64_t width, int rank,
                  hipStream_t stream) {
    const auto run = [&](auto kernel, int cols) {
        // Without out: h_out alone.
        const int columns = out ? static_cast<int>((width + 64 * cols - 1) / (64 * cols)) : 1;
        const int64_t parts = static_cast<int64_t>(g.tile_bound) * columns;
        const int whole = g.order ? kTileRows / 16 : group_tile_rows(rank) / 16;
        // Whole tiles read w once a tile, parts of them fill the card: 512 rows of 4096
        // columns at rank 64 (272 parts) 13.6 us with whole tiles, 10.9 with 2; 1024 rows at
        // rank 16 (200) 10.8 with 1, 8.2 with 2; 256 rows at rank 64 (144) 8.5 and 7.7 with 1.
        const int fragments = parts > 384 ? whole : parts > 192 ? 2 : 1;
        hipLaunchKernelGGL(kernel, dim3(part_grid(columns, g.tile_bound), 1, whole / fragments), dim3(256), 0, stream,
                           partials, slices, w, scales, g, base, out, h_out, tokens, width, rank, fragments, columns);
        return check_launch("spread_kernel");
    };
    const auto by_rank = [&](auto streamed) {
        constexpr bool S = decltype(streamed)::value;
        if (w32) {  // the router: at most 64 experts
            if (rank <= 16) return run(spread_kernel<1, true, true, 8, S>, 8);
            if (rank <= 32) return run(spread_kernel<1, false, true, 8, S>, 8);
            return run(spread_kernel<2, false, true, 4, S>, 4);
        }
        if (rank <= 16) return run(spread_kernel<1, true, false, 8, S>, 8);
        if (rank <= 32) return run(spread_kernel<1, false, false, 8, S>, 8);
        if (rank <= 64) return run(spread_kernel<2, false, false, 4, S>, 4);
        return run(spread_kernel<4, false, false, 4, S>, 4);
    };
    return tokens * width >= kStreamElements ? by_rank(std::true_type{}) : by_rank(std::false_type{});
}

// ---------------------------------------------------------------------------
// contract and spread in one launch, for small batches: decoding steps are launch and
// latency. A workgroup takes 16 rows of a tile and up to 1024 columns a turn; its eight
// waves split all of k, add up in LDS, and each spread 128 columns. Every column part
// computes h again, from w in the L2, so that nothing is handed over between workgroups.
// The sums' order is k's over eight waves: results differ from the two launches' in fp32
// rounding. Latency, not bytes: one row of 4096 -> 4096 at rank 16 takes 7.5 us under replay
// and 8.3 a call (two launches 7.2, and 11.5 with the host's second launch and scratch), of
// 512 -> 512 4.6; 64 rows of 16 adapters 10.6. Loads five to seven steps ahead took 8.4 to
// 8.7 where four took 8.1, sixteen waves of 64 columns 9.8 (their registers spill).
// ---------------------------------------------------------------------------
constexpr int kFusedWaves = 8;
constexpr int kFusedCols = kFusedWaves * 128;

template <int NR>
__global__ __launch_bounds__(64 * kFusedWaves) void fused_kernel(
    const uint16_t* __restrict__ x, const uint16_t* __restrict__ down, const uint16_t* __restrict__ up,
    const float* __restrict__ scales, Groups gr, const uint16_t* base, uint16_t* out, float* __restrict__ h_out, int k,
    int64_t width, int rank, int turns) {
    constexpr bool HALF = NR == 1;
    constexpr int NK = 1, C = 16 * NR, KP = 32 * NK + 8;
    constexpr int D = 4;
    constexpr int kStepHalfs = 1024 * (1 + NR), kWaveHalfs = 2 * kStepHalfs;  // two steps' lines a wave
    __shared__ __attribute__((aligned(16))) uint16_t lines[kFusedWaves * kWaveHalfs];
    __shared__ __attribute__((aligned(16))) uint16_t hi[16 * KP];
    __shared__ __attribute__((aligned(16))) uint16_t lo[HALF ? 8 : 16 * KP];
    const int4 tile = gr.tiles[blockIdx.x / 4];
    if (static_cast<int>(blockIdx.x / 4) >= gr.head[0]) return;
    const int skip = 16 * (blockIdx.x % 4);
    const int adapter = tile.x, first = tile.y + skip, rows = min(tile.z - skip, 16);
    if (rows <= 0) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l = lane & 15, g = lane >> 4;
    int64_t row_at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) row_at[q] = gr.order[first + min(4 * g + q, rows - 1)] * width;
    int64_t col = static_cast<int64_t>(blockIdx.y) * turns * kFusedCols + wave * 128 + 8 * l;
    const u32x4_t zero = {0, 0, 0, 0};
    if (adapter < 0) {  // no adapter: h is 0, the base as it is
        if (h_out && blockIdx.y == 0)
            for (int i = tid; i < rows * rank; i += 64 * kFusedWaves) h_out[static_cast<int64_t>(first) * rank + i] = 0.0f;
        if (base == out || !out) return;
        for (int turn = 0; turn < turns && col < width; ++turn, col += kFusedCols)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (4 * g + q < rows)
                    *reinterpret_cast<u32x4_t*>(out + row_at[q] + col) = base ? load16(base + row_at[q] + col) : zero;
        return;
    }
    // The first turn's rows of up and base are on their way while h is made.
    const uint16_t* wa = up + static_cast<int64_t>(adapter) * rank * width;
    u32x4_t raw[NK][8], old[4];
    const auto fetch = [&] {
        const bool inside = col < width;
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = HALF ? (8 * g + j) & 15 : 32 * n + 8 * g + j;
                const uint32_t from = static_cast<uint32_t>(c) * static_cast<uint32_t>(width) + static_cast<uint32_t>(col);
                raw[n][j] = inside && c < rank ? load16(wa + from) : zero;
            }
#pragma unroll
        for (int q = 0; q < 4; ++q) old[q] = base && inside ? load16(base + row_at[q] + col) : zero;
    };
    if (out) fetch();
    f32x4_t acc[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) acc[n] = f32x4_t{0, 0, 0, 0};
    uint16_t* mine = lines + wave * kWaveHalfs;
    {
        // A wave's share of k: whole steps of 64.
        const int steps = (k + 63) / 64, share = (steps + kFusedWaves - 1) / kFusedWaves * 64;
        const int kb = wave * share, ke = min(kb + share, k);
        LineRows xr, wr[NR];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = lane / 8 + 8 * h;
            xr.row[h] = x + static_cast<int64_t>(gr.order[first + min(r, rows - 1)]) * k;
#pragma unroll
            for (int n = 0; n < NR; ++n)
                wr[n].row[h] = down + (static_cast<int64_t>(adapter) * rank + min(16 * n + r, rank - 1)) * k;
        }
        struct Step {
            Lines x, w[NR];
        };
        Step ring[D];
        const auto load = [&](Step& s, int k0) {
            const int at = k0 + 8 * (lane % 8);
            load_lines(s.x, xr, at, k, rows, lane);
#pragma unroll
            for (int n = 0; n < NR; ++n) load_lines(s.w[n], wr[n], at, k);
        };
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (kb + 64 * d < ke) load(ring[d], kb + 64 * d);
        const auto put = [&](const Step& s, int parity) {
            uint16_t* to = mine + parity * kStepHalfs;
            put_lines(to, s.x, lane);
#pragma unroll
            for (int n = 0; n < NR; ++n) put_lines(to + 1024 * (1 + n), s.w[n], lane);
        };
        // A step's lines are in LDS before the one before it is read.
        if (kb < ke) put(ring[0], 0);
        for (int k0 = kb; k0 < ke; k0 += 64 * D)
#pragma unroll
            for (int d = 0; d < D; ++d)
                if (k0 + 64 * d < ke) {
                    const int ahead = k0 + 64 * (d + D);
                    if (ahead < ke) load(ring[d], ahead);
                    wave_lds_order();
                    if (k0 + 64 * (d + 1) < ke) put(ring[(d + 1) % D], (d + 1) % 2);
                    const uint16_t* from = mine + d % 2 * kStepHalfs;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const u32x4_t a = get_operand(from, l, g, h);
#pragma unroll
                        for (int n = 0; n < NR; ++n) acc[n] = mfma(a, get_operand(from + 1024 * (1 + n), l, g, h), acc[n]);
                    }
                    wave_lds_order();
                }
    }
    // The waves' sums, each in its own lines, added in wave order.
    float* sums = reinterpret_cast<float*>(mine);
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q) sums[(4 * g + q) * C + 16 * n + l] = acc[n][q];
    __syncthreads();
    for (int i = tid; i < 16 * (HALF ? 16 : 32 * NK); i += 64 * kFusedWaves) {
        const int row = i / C, c = i % C;
        float h = 0.0f;
        if (row < rows && c < rank) {
#pragma unroll
            for (int p = 0; p < kFusedWaves; ++p) h += reinterpret_cast<const float*>(lines + p * kWaveHalfs)[i];
            if (h_out && blockIdx.y == 0) h_out[static_cast<int64_t>(first + row) * rank + c] = h;
        }
        const uint16_t a = f32_to_bf16(h), rest = f32_to_bf16(bf16_rest(h, a));
        hi[row * KP + c] = a;
        if (HALF)
            hi[row * KP + 16 + c] = rest;
        else
            lo[row * KP + c] = rest;
    }
    if (!out) return;
    __syncthreads();
    const float scale = scales ? scales[adapter] : 1.0f;
    for (int turn = 0; turn < turns; ++turn) {
        u32x4_t b[NK][8], there[4];
#pragma unroll
        for (int n = 0; n < NK; ++n) transpose8(raw[n], b[n]);
#pragma unroll
        for (int q = 0; q < 4; ++q) there[q] = old[q];
        const int64_t now = col;
        col += kFusedCols;
        if (turn + 1 < turns) fetch();
        f32x4_t sum[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = f32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            const int from = l * KP + 32 * n + 8 * g;
            const u32x4_t a = *reinterpret_cast<const u32x4_t*>(hi + from);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] = mfma(a, b[n][i], sum[i]);
            if (!HALF) {
                const u32x4_t a2 = *reinterpret_cast<const u32x4_t*>(lo + from);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] = mfma(a2, b[n][i], sum[i]);
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (now >= width || 4 * g + q >= rows) continue;
            u32x4_t o;
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const float b0 = bf16_to_f32(static_cast<uint16_t>(there[q][d]));
                const float b1 = bf16_to_f32(static_cast<uint16_t>(there[q][d] >> 16));
                o[d] = pack_bf16x2(b0 + scale * sum[2 * d][q], b1 + scale * sum[2 * d + 1][q]);
            }
            *reinterpret_cast<u32x4_t*>(out + row_at[q] + now) = o;
        }
    }
}

// Workgroups of a fused launch's column parts, or 0 where two launches take less time. A call
// from Python pays 3 us for the second launch and its scratch, a replay nothing, and the rule
// is for calls. The parts' repeated reads of x and w (16 rows and the ranks, of k) may come
// to kFusedBytes: 64 rows of 16 adapters, 4096 to 4096 at rank 16, take 10.8 us a call and
// 11.7 in two launches (replayed 10.6 and 7.8), 256 rows of 8 adapters 12.1 and 12.5 (12.2 and
// 8.6); with 64 MB, 48 rows of 64 adapters took 23.6 where two launches take 12.0 (23.1 and
// 8.6). A workgroup walks all of k, so rank * k is limited too: one row of 4096 columns at
// rank 16, at the limit, 8.3 us a call and 11.5 in two launches (7.5 and 7.2); of 8192, past
// it, 10.9 and 11.6 (10.6 and 7.3); of 4096 at rank 32, 9.5 and 11.6 (9.1 and 7.7).
constexpr int64_t kFusedBytes = 32 << 20;
constexpr int64_t kFusedElements = 64 << 10;

static int fused_parts(int64_t tokens, int64_t k, int64_t width, int rank, int adapters) {
    // No registers for up's rows beside the loads of h past 32 ranks; and one CU streams
    // a long w slower than two launches over all of them take.
    if (rank > 32 || rank * k > kFusedElements) return 0;
    const int64_t fragments = tokens / 16 + std::min<int64_t>(adapters + 1, tokens);
    if (fragments == 0) return 0;
    const int64_t columns = (width + kFusedCols - 1) / kFusedCols;
    const int64_t parts = std::clamp<int64_t>(512 / fragments, 1, columns);
    return fragments * parts * (rank + 16) * k * 2 <= kFusedBytes ? static_cast<int>(parts) : 0;
}

// contract and spread: h of x and down, then up; one launch for small batches. Without
// out: h_out alone, with the same sums.
static int launch_through(const uint16_t* x, const uint16_t* down, const uint16_t* up, const float* scales,
                          const Groups& g, const uint16_t* base, uint16_t* out, float* h_out, float* partials,
                          int64_t tokens, int64_t k, int64_t width, int rank, int adapters, hipStream_t stream) {
    if (const int parts = fused_parts(tokens, k, width, rank, adapters)) {
        const int columns = out ? static_cast<int>((width + kFusedCols - 1) / kFusedCols) : 1;
        const int turns = (columns + parts - 1) / parts;
        const dim3 grid(4 * g.tile_bound, (columns + turns - 1) / turns);
        const auto run = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, grid, dim3(64 * kFusedWaves), 0, stream, x, down, up, scales, g, base, out, h_out,
                               static_cast<int>(k), width, rank, turns);
            return check_launch("fused_kernel");
        };
        return rank <= 16 ? run(fused_kernel<1>) : run(fused_kernel<2>);
    }
    const int slices = contract_slices(g.tile_bound, k, rank);
    const int rc = launch_contract(x, down, g, partials, slices, tokens, k, rank, stream);
    if (rc != MOE_OK) return rc;
    return launch_spread(partials, slices, up, false, scales, g, base, out, h_out, tokens, width, rank, stream);
}

// ---------------------------------------------------------------------------
// outer: out[c][j] = s sum_i h[i][c] x[i][j] over an adapter's rows.
// The rows are the MFMA's k. A workgroup takes a split of one adapter's rows and 128
// columns; its waves take 32 rows in turn. x's 8 x 8 blocks are transposed in registers
// as in spread; h (fp32, read along the ranks) enters as three bf16 parts, which hold
// all its bits, so each product is exact and sums in fp32. The waves' sums meet in LDS;
// an adapter of one split is done, of more its partial sums are added in split order.
// Bound by x's bytes: both products of 4096 rows of 4096 columns, 67 MB, in 14.4 us at
// r=16 and 18 at r=32, and 4 us for the splits' sums.
// ---------------------------------------------------------------------------
template <bool BF16>
__device__ __forceinline__ void store4(void* out, int64_t at, f32x4_t v) {
    if (BF16)
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) =
            make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
    else
        *reinterpret_cast<f32x4_t*>(static_cast<float*>(out) + at) = v;
}

// Eight fp32 values as three bf16 operands: their significands' 24 bits, eight at a time,
// cut off and not rounded, so that each rest is exact (an infinite value leaves NaN).
__device__ __forceinline__ void split3(const float (&f)[8], u32x4_t (&a)[3]) {
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        float f0 = f[2 * p], f1 = f[2 * p + 1];
#pragma unroll
        for (int n = 0; n < 3; ++n) {
            const uint32_t b0 = __float_as_uint(f0), b1 = __float_as_uint(f1);
            a[n][p] = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
            f0 -= __uint_as_float(b0 & 0xffff0000u);
            f1 -= __uint_as_float(b1 & 0xffff0000u);
        }
    }
}

// Up to 32 ranks: a wave holds NR 16-rank fragments of 128 columns, the waves share the
// rows. The split's row numbers are in LDS before the first row is asked
// for: read from the table beside each step's rows, every step waited for memory twice
// (4096 rows of 4096 columns, rank 16, both products: 22.4 us, 14.8 now; loads one or two
// steps ahead then gain nothing).
// A launch does up to two products on the same groups (an adapter's two gradients).
struct OuterJobs {
    OuterJob job[2];
    int columns[2];  // column parts of each; the grid has both
};

// A workgroup's split, job and columns.
struct OuterPart {
    OuterJob job;
    int column, adapter, first, rows, partial;
};
__device__ __forceinline__ bool outer_part(const OuterJobs& jobs, const Groups& gr, int64_t tokens, OuterPart* p) {
    const bool second = static_cast<int>(blockIdx.y) >= jobs.columns[0];
    p->job = jobs.job[second];
    p->column = (blockIdx.y - (second ? jobs.columns[0] : 0)) * kOuterCols;
    if (gr.order) {
        const int4 split = gr.splits[blockIdx.x];
        p->adapter = split.x;
        p->first = split.y;
        p->rows = split.z;
        p->partial = split.w;
        return static_cast<int>(blockIdx.x) < gr.head[1];
    }
    p->adapter = 0;
    p->first = blockIdx.x * gr.split_rows;
    p->rows = static_cast<int>(min(static_cast<int64_t>(gr.split_rows), tokens - p->first));
    p->partial = gr.split_bound > 1 ? static_cast<int>(blockIdx.x) : -1;
    return true;
}

// The split's rows, up to whole 64s. -1: past its end, or a masked row, which may hold
// anything (its h is 0, and 0 times NaN is not).
__device__ __forceinline__ void list_rows(int32_t* row_of, const Groups& gr, const OuterPart& p) {
    for (int i = threadIdx.x; i < (p.rows + 63) / 64 * 64; i += blockDim.x) {
        const int at = p.first + i;
        row_of[i] = i >= p.rows ? -1 : gr.order ? gr.order[at] : gr.mask && !gr.mask[at] ? -1 : at;
    }
}

// Four columns of a rank: the result, or this split's share of it.
template <bool BF16>
__device__ __forceinline__ void store_outer(const OuterPart& p, int rank, int c, int64_t j, f32x4_t sum) {
    if (c >= rank || j >= p.job.width) return;
    if (p.partial < 0)
        store4<BF16>(p.job.out, (static_cast<int64_t>(p.adapter) * rank + c) * p.job.width + j, sum);
    else
        store4<false>(p.job.partials, (static_cast<int64_t>(p.partial) * rank + c) * p.job.width + j, sum);
}

template <int NR, bool BF16>
__global__ __launch_bounds__(256, 3) void outer_kernel(OuterJobs jobs, const float* __restrict__ scales, Groups gr,
                                                    int64_t tokens, int rank) {
    constexpr int W = 4;
    __shared__ __attribute__((aligned(16))) float lds[W * 16 * kOuterCols];
    __shared__ int32_t row_of[kMaxSplitRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l = lane & 15, g = lane >> 4;
    OuterPart part;
    if (!outer_part(jobs, gr, tokens, &part)) return;
    list_rows(row_of, gr, part);
    const int rows = part.rows;
    const int64_t width = part.job.width;
    const int64_t col = part.column + 8 * l;
    const bool inside = col < width;
    const u32x4_t zero = {0, 0, 0, 0};
    f32x4_t acc[NR][8];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[n][i] = f32x4_t{0, 0, 0, 0};
    __syncthreads();
    for (int t0 = 32 * wave; t0 < rows; t0 += 32 * W) {
        u32x4_t v[8];
        float hv[NR][8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = t0 + 8 * g + j;
            const int row = i < rows ? row_of[i] : -1;
            v[j] = row >= 0 && inside ? load16(part.job.x + row * width + col) : zero;
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const int c = 16 * n + l;
                hv[n][j] = i < rows && c < rank ? part.job.h[static_cast<int64_t>(part.first + i) * rank + c] : 0.0f;
            }
        }
        u32x4_t b[8];
        transpose8(v, b);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            u32x4_t a[3];
            split3(hv[n], a);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                acc[n][i] = mfma(a[2], b[i], acc[n][i]);
                acc[n][i] = mfma(a[1], b[i], acc[n][i]);
                acc[n][i] = mfma(a[0], b[i], acc[n][i]);
            }
        }
    }
    const float scale = scales ? scales[part.adapter] : 1.0f;
    // One fragment of every wave at a time: [wave][rank][column] in LDS, the waves summed
    // in order; a thread takes four columns of two ranks.
#pragma unroll
    for (int n = 0; n < NR; ++n) {
        if (n > 0) __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float* dst = lds + (wave * 16 + 4 * g + q) * kOuterCols + 8 * l;
            *reinterpret_cast<f32x4_t*>(dst) = f32x4_t{acc[n][0][q], acc[n][1][q], acc[n][2][q], acc[n][3][q]};
            *reinterpret_cast<f32x4_t*>(dst + 4) = f32x4_t{acc[n][4][q], acc[n][5][q], acc[n][6][q], acc[n][7][q]};
        }
        __syncthreads();
#pragma unroll
        for (int r0 = 0; r0 < 16; r0 += 8) {
            const int r = r0 + tid / 32;
            const float* src = lds + r * kOuterCols + 4 * (tid & 31);
            f32x4_t sum = *reinterpret_cast<const f32x4_t*>(src);
#pragma unroll
            for (int w = 1; w < W; ++w) sum += *reinterpret_cast<const f32x4_t*>(src + w * 16 * kOuterCols);
            store_outer<BF16>(part, rank, 16 * n + r, part.column + 4 * (tid & 31), sum * scale);
        }
    }
}

// More than 32 ranks: every wave would load and transpose the same x, and each column part
// split the same h, once per 32 ranks (4096 rows of 4096 columns, rank 64 and 128, both
// products: 41.9 and 74.4 us). Here eight waves stage 64 rows a step in LDS as operands,
// a wave eight of them (x transposed, h split), while the next rows' loads are on their
// way; then a wave multiplies its quarter of the ranks and half of the columns: 23 and 46 us.
// RF: 16-rank fragments, 4 or 8.
template <int RF, bool BF16>
__global__ __launch_bounds__(512, 4) void outer_wide_kernel(OuterJobs jobs, const float* __restrict__ scales, Groups gr,
                                                            int64_t tokens, int rank) {
    constexpr int R = 16 * RF, NR = RF / 4, HL = R / 64;
    // [32 rows][8 of them][column, or rank], 16 bytes each: eight rows of a column or rank.
    // Column c of a half lies at 16 (c % 4) + c / 4, so that a lane ends with four
    // neighbours.
    __shared__ u32x4_t xs[2][4][kOuterCols];
    __shared__ u32x4_t hs[2][3][4][R];
    __shared__ __attribute__((aligned(16))) int32_t row_of[kMaxSplitRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int l = lane & 15, g = lane >> 4;
    OuterPart part;
    if (!outer_part(jobs, gr, tokens, &part)) return;
    list_rows(row_of, gr, part);
    const int rows = part.rows;
    const int64_t width = part.job.width;
    const bool inside = part.column + 2 * lane < width;
    const int rank0 = wave % 4 * 16 * NR, half = wave / 4;
    f32x4_t acc[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[n][i] = f32x4_t{0, 0, 0, 0};
    // This wave's eight rows of a step: two columns and a rank (two) a lane. Addresses are
    // a scalar row and a lane's offset; rows of none are read from row 0 (and the last h) and
    // taken as zeros of x.
    const uint32_t x_at = inside ? 2 * lane : 0;
    uint32_t xv[8], valid;
    float hv[HL][8];
    const int own = __builtin_amdgcn_readfirstlane(8 * wave);
    const uint16_t* x0 = part.job.x + part.column;
    const auto fetch = [&](int t0) {
        valid = 0;
        const int4 listed[2] = {*reinterpret_cast<const int4*>(row_of + t0 + own),
                                *reinterpret_cast<const int4*>(row_of + t0 + own + 4)};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = min(t0 + own + j, rows - 1);
            const int row = __builtin_amdgcn_readfirstlane(reinterpret_cast<const int*>(listed)[j]);
            valid |= static_cast<uint32_t>(row >= 0) << j;
            xv[j] = *reinterpret_cast<const uint32_t*>(x0 + max(row, 0) * width + x_at);
            const float* h = part.job.h + static_cast<int64_t>(part.first + i) * rank;
#pragma unroll
            for (int n = 0; n < HL; ++n) hv[n][j] = h[min(64 * n + lane, rank - 1)];
        }
    };
    __syncthreads();
    fetch(0);
    for (int t0 = 0; t0 < rows; t0 += 64) {
        const int group = wave / 4, eight = wave % 4;
#pragma unroll
        for (int j = 0; j < 8; ++j) xv[j] = valid >> j & 1 ? xv[j] : 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            u32x4_t b;
#pragma unroll
            for (int p = 0; p < 4; ++p)
                b[p] = __builtin_amdgcn_perm(xv[2 * p + 1], xv[2 * p], i ? 0x07060302u : 0x05040100u);
            const int c = 2 * lane + i;
            xs[group][eight][(c & 64) + 16 * (c & 3) + (c & 63) / 4] = b;
        }
#pragma unroll
        for (int n = 0; n < HL; ++n) {
            u32x4_t a[3];
            split3(hv[n], a);
#pragma unroll
            for (int p = 0; p < 3; ++p) hs[group][p][eight][64 * n + lane] = a[p];
        }
        __syncthreads();
        if (t0 + 64 < rows) fetch(t0 + 64);
        if (rank0 < rank) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                u32x4_t b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] = xs[k][g][64 * half + 16 * i + l];
#pragma unroll
                for (int n = 0; n < NR; ++n)
#pragma unroll
                    for (int p = 2; p >= 0; --p) {
                        const u32x4_t a = hs[k][p][g][rank0 + 16 * n + l];
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][i] = mfma(a, b[i], acc[n][i]);
                    }
            }
        }
        __syncthreads();
    }
    const float scale = scales ? scales[part.adapter] : 1.0f;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            store_outer<BF16>(part, rank, rank0 + 16 * n + 4 * g + q, part.column + 64 * half + 4 * l,
                              f32x4_t{acc[n][0][q], acc[n][1][q], acc[n][2][q], acc[n][3][q]} * scale);
}

// An adapter's partial sums in split order, or zeros for one without rows.
template <bool BF16>
__global__ __launch_bounds__(256) void outer_sum_kernel(OuterJobs jobs, Groups gr, int rank, ColumnSums extra) {
    const int a = blockIdx.y;
    const int64_t blocks0 = (jobs.job[0].width * rank + 1023) / 1024;
    const int64_t blocks1 = (jobs.job[1].width * rank + 1023) / 1024;
    if (static_cast<int64_t>(blockIdx.x) >= blocks0 + blocks1) {
        sum_columns(extra);
        return;
    }
    const bool second = static_cast<int64_t>(blockIdx.x) >= blocks0;
    const OuterJob job = jobs.job[second];
    const int64_t elements = job.width * rank;
    const int first = gr.order ? gr.partial_start[a] : 0;
    const int s0 = first >> 1, s1 = gr.order ? gr.partial_start[a + 1] >> 1 : gr.split_bound;
    if (s0 == s1 && (first & 1)) return;  // its one split wrote the result
    const int64_t at = ((static_cast<int64_t>(blockIdx.x) - (second ? blocks0 : 0)) * 256 + threadIdx.x) * 4;
    if (at >= elements) return;
    f32x4_t sum = {0, 0, 0, 0};
    constexpr int U = 8;  // splits in flight
    for (int s = s0; s < s1; s += U) {
        f32x4_t v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            v[u] = *reinterpret_cast<const f32x4_t*>(job.partials + static_cast<int64_t>(min(s + u, s1 - 1)) * elements + at);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s + u < s1) sum += v[u];
    }
    store4<BF16>(job.out, a * elements + at, sum);
}

int launch_outer(const OuterJob& first, const OuterJob& second, const float* scales, const Groups& g, bool out_bf16,
                 int64_t tokens, int rank, int adapters, hipStream_t stream, ColumnSums extra) {
    OuterJobs jobs;
    jobs.job[0] = first;
    jobs.job[1] = second;
    for (int i = 0; i < 2; ++i) jobs.columns[i] = static_cast<int>((jobs.job[i].width + kOuterCols - 1) / kOuterCols);
    const dim3 grid(g.split_bound, jobs.columns[0] + jobs.columns[1]);
    const auto run = [&](auto kernel, int waves) {
        hipLaunchKernelGGL(kernel, grid, dim3(64 * waves), 0, stream, jobs, scales, g, tokens, rank);
        return check_launch("outer_kernel");
    };
    const auto by_rank = [&](auto bf16) {
        constexpr bool B = decltype(bf16)::value;
        if (rank <= 16) return run(outer_kernel<1, B>, 4);
        if (rank <= 32) return run(outer_kernel<2, B>, 4);
        if (rank <= 64) return run(outer_wide_kernel<4, B>, 8);
        return run(outer_wide_kernel<8, B>, 8);
    };
    int rc = MOE_OK;
    if (g.split_bound > 0) rc = out_bf16 ? by_rank(std::true_type{}) : by_rank(std::false_type{});
    if (rc != MOE_OK || (!g.order && g.split_bound == 1)) return rc;
    // One more block for the extra sums (of the router, whose rows are one group).
    const int64_t blocks = (first.width * rank + 1023) / 1024 + (second.width * rank + 1023) / 1024 + (extra.rows > 0);
    const dim3 sum_grid(static_cast<unsigned>(blocks), adapters);
    if (out_bf16)
        hipLaunchKernelGGL(outer_sum_kernel<true>, sum_grid, dim3(256), 0, stream, jobs, g, rank, extra);
    else
        hipLaunchKernelGGL(outer_sum_kernel<false>, sum_grid, dim3(256), 0, stream, jobs, g, rank, extra);
    return check_launch("outer_sum_kernel");
}

// ---------------------------------------------------------------------------
// The operators
// ---------------------------------------------------------------------------
static int64_t up16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

// contract's partial sums, none where one launch does.
static int64_t through_bytes(int64_t tokens, int64_t k, int64_t width, int64_t rank, int64_t adapters) {
    if (fused_parts(tokens, k, width, static_cast<int>(rank), static_cast<int>(adapters))) return 0;
    return contract_slices(table_layout(tokens, adapters).tile_bound, k, rank) * tokens * rank * 4;
}

int64_t low_rank_add_scratch_bytes(int64_t tokens, int64_t hidden, int64_t width, int64_t rank, int64_t adapters) {
    return through_bytes(tokens, hidden, width, rank, adapters);
}

// Where the backward pass' scratch lies: contract's sums of dh and dh itself (for grad_x and
// grad_down), and the partial sums of the products that are wanted.
struct BackwardScratch {
    int64_t dh, down, up, bytes;
};
static BackwardScratch backward_scratch(int64_t tokens, int64_t hidden, int64_t width, int64_t rank, int64_t adapters,
                                        bool want_x, bool want_down, bool want_up) {
    const int64_t rows = static_cast<int64_t>(table_layout(tokens, adapters).partial_bound) * rank;
    BackwardScratch s{};
    if (want_x || want_down) {
        s.dh = up16(through_bytes(tokens, width, hidden, rank, adapters));
        s.down = s.dh + up16(tokens * rank * 4);
    }
    s.up = s.down + (want_down ? rows * hidden * 4 : 0);
    s.bytes = s.up + (want_up ? rows * width * 4 : 0);
    return s;
}
int64_t low_rank_backward_scratch_bytes(int64_t tokens, int64_t hidden, int64_t width, int64_t rank, int64_t adapters,
                                        bool want_x, bool want_down, bool want_up) {
    return backward_scratch(tokens, hidden, width, rank, adapters, want_x, want_down, want_up).bytes;
}

int launch_low_rank_add(const uint16_t* x, const uint16_t* down, const uint16_t* up, const float* scales,
                        const void* table, const uint16_t* base, uint16_t* output, float* hidden_out, char* scratch,
                        int64_t tokens, int64_t hidden, int64_t width, int rank, int adapters, hipStream_t stream) {
    const Groups g = groups_of(table, tokens, adapters);
    return launch_through(x, down, up, scales, g, base, output, hidden_out, reinterpret_cast<float*>(scratch), tokens,
                          hidden, width, rank, adapters, stream);
}

int launch_low_rank_backward(const uint16_t* grad_output, const uint16_t* x, const uint16_t* down, const uint16_t* up,
                             const float* scales, const void* table, const float* hidden_in, const uint16_t* grad_x_base,
                             uint16_t* grad_x, void* grad_down, void* grad_up, bool grad_bf16, char* scratch,
                             int64_t tokens, int64_t hidden, int64_t width, int rank, int adapters, hipStream_t stream) {
    const Groups g = groups_of(table, tokens, adapters);
    const BackwardScratch at = backward_scratch(tokens, hidden, width, rank, adapters, grad_x, grad_down, grad_up);
    float* dh_parts = reinterpret_cast<float*>(scratch);
    float* dh = reinterpret_cast<float*>(scratch + at.dh);
    int rc = MOE_OK;
    // dx, and dh for its outer product.
    if (tokens > 0 && (grad_x || grad_down))
        rc = launch_through(grad_output, up, down, scales, g, grad_x_base, grad_x, dh, dh_parts, tokens, width, hidden,
                            rank, adapters, stream);
    if (rc == MOE_OK && (grad_down || grad_up)) {
        OuterJob jobs[2];
        if (grad_down) jobs[0] = {dh, x, reinterpret_cast<float*>(scratch + at.down), grad_down, hidden};
        if (grad_up) jobs[1] = {hidden_in, grad_output, reinterpret_cast<float*>(scratch + at.up), grad_up, width};
        rc = launch_outer(jobs[0], jobs[1], scales, g, grad_bf16, tokens, rank, adapters, stream);
    }
    return rc;
}

}  // namespace moe
