// Row grouping by adapter and the three products of low-rank adapters (contract,
// spread, outer), shared by low_rank.hip and router_grad.hip.
#pragma once

#include "moe_common.h"

namespace moe {

constexpr int kMaxAdapters = 4096;
constexpr int kMaxRank = 128;
constexpr int64_t kMaxAdapterTokens = 1 << 21;  // tiles and adapters within a grid's 65535
constexpr int64_t kMaxLowRankWidth = 1 << 20;
constexpr int kChunkRows = 4096;  // rows that one workgroup sorts by adapter
constexpr int kTileRows = 64;     // rows of one adapter per tile (contract, spread)
// Rows per tile of one group of more than 32 ranks (the router's experts): their fp32
// weights are taken apart into bf16 parts once a tile (dx of 64 experts with the logits'
// gradient, 8192 x 2048: 21.2 us, with 64 rows 23.4; 16384 x 4096: 66.5 and 72.0).
constexpr int kWideTileRows = 128;
inline int group_tile_rows(int64_t rank) { return rank > 32 ? kWideTileRows : kTileRows; }
constexpr int kOuterCols = 128;   // columns per workgroup of outer
constexpr int kMaxSplitRows = 1024;

// Where the parts of an adapter table lie, in int32 from its start:
//   head         [4]     tiles, splits, 0, 0
//   order        [T]     rows sorted by adapter (stable); rows of no adapter last
//   starts       [N + 2] first sorted row of each adapter, of the rows of none, T
//   partial_start [N + 1] twice the first partial sum of each adapter (a split's, of the adapters
//                        that have several), plus 1 where the adapter has rows
//   tiles        [tile_bound]  {adapter (-1: none), first sorted row, rows <= kTileRows, 0}
//   splits       [split_bound] {adapter, first sorted row, rows <= split_rows, partial sum (-1: the
//                        adapter's only split)}
//   chunks       [chunk_count][N + 1]  while it is made, of a batch of more rows than a chunk:
//                        each chunk's rows of each adapter, then those of the chunks before
struct TableLayout {
    int64_t order, starts, partial_start, tiles, splits, chunks, ints;
    int tile_bound, split_bound, partial_bound, split_rows, chunk_count;
};

// Rows per split of the outer product: a split's partial result is written and read
// back once (4 * rank * width bytes twice), so few of them, but enough workgroups
// (splits * width / 128) to fill the card: about 8 splits of a batch. Both gradients of 4
// adapters from and to 4096 columns, dh's contract included, with 8, 4 and 16 splits: 4096
// rows at rank 16 31.8, 37.0 and 34.7 us, at rank 64 46.4, 58.2 and 53.5; 1024 rows at rank
// 16 20.5 with 8 and 19.3 with 4.
inline int outer_split_rows(int64_t tokens) {
    int rows = 128;
    while (rows < kMaxSplitRows && rows * 8 < tokens) rows <<= 1;
    return rows;
}

inline TableLayout table_layout(int64_t tokens, int64_t adapters) {
    TableLayout t{};
    const auto up4 = [](int64_t n) { return (n + 3) / 4 * 4; };
    t.split_rows = outer_split_rows(tokens);
    // Each group has at most one partial tile (split).
    t.tile_bound = static_cast<int>(tokens / kTileRows + (adapters + 1 < tokens ? adapters + 1 : tokens));
    t.split_bound = static_cast<int>(tokens / t.split_rows + (adapters < tokens ? adapters : tokens));
    // An adapter of n > split_rows rows has fewer than 2 n / split_rows splits; the others' one
    // split writes the result itself, so that a large bank asks for no more partial sums.
    const int64_t partials = tokens > t.split_rows ? 2 * tokens / t.split_rows : 0;
    t.partial_bound = partials < t.split_bound ? static_cast<int>(partials) : t.split_bound;
    t.order = 4;
    t.starts = t.order + up4(tokens);
    t.partial_start = t.starts + up4(adapters + 2);
    t.tiles = t.partial_start + up4(adapters + 1);
    t.splits = t.tiles + 4 * static_cast<int64_t>(t.tile_bound);
    t.chunks = t.splits + 4 * static_cast<int64_t>(t.split_bound);
    t.chunk_count = tokens > kChunkRows ? static_cast<int>((tokens + kChunkRows - 1) / kChunkRows) : 0;
    t.ints = t.chunks + up4(t.chunk_count * (adapters + 1));
    return t;
}

// Device view of a table. A null order stands for one group of all rows in order.
struct Groups {
    const int32_t* head = nullptr;
    const int32_t* order = nullptr;
    const int32_t* partial_start = nullptr;
    const int4* tiles = nullptr;
    const int4* splits = nullptr;
    int tile_bound = 0, split_bound = 0, split_rows = 0;
    const uint8_t* mask = nullptr;  // one group: outer takes no row of x whose byte is 0
};

inline Groups groups_of(const void* table, int64_t tokens, int64_t adapters) {
    const TableLayout t = table_layout(tokens, adapters);
    const int32_t* base = static_cast<const int32_t*>(table);
    Groups g;
    g.head = base;
    g.order = base + t.order;
    g.partial_start = base + t.partial_start;
    g.tiles = reinterpret_cast<const int4*>(base + t.tiles);
    g.splits = reinterpret_cast<const int4*>(base + t.splits);
    g.tile_bound = t.tile_bound;
    g.split_bound = t.split_bound;
    g.split_rows = t.split_rows;
    return g;
}

// The splits of one group may follow the width and rank too: about 512 workgroups, or 256
// of the eight waves that more than 32 ranks take (router dW with the logits' gradient, the
// same workgroups, twice and half as many: 4096 x 4096 of 8 experts 15.1, 16.7 and 15.4 us,
// 8192 x 2048 of 64 experts 22.0, 22.6 and 30.0).
inline Groups one_group(int64_t tokens, int64_t width, int64_t rank) {
    Groups g;
    const int64_t columns = (width + kOuterCols - 1) / kOuterCols;
    const int64_t most = rank > 32 ? 256 : 512;
    g.split_rows = 128;
    while (g.split_rows < kMaxSplitRows && tokens * columns > g.split_rows * most) g.split_rows <<= 1;
    const int rows = group_tile_rows(rank);
    g.tile_bound = static_cast<int>((tokens + rows - 1) / rows);
    g.split_bound = static_cast<int>((tokens + g.split_rows - 1) / g.split_rows);
    return g;
}

// out[c] = sum over rows of part[row][c], c < columns <= 64; nothing when rows is 0.
struct ColumnSums {
    const float* part = nullptr;
    float* out = nullptr;
    int rows = 0, columns = 0;
};

// By one block of 256 threads: thread (quarter, column) takes every fourth row, sixteen of
// them in flight, and the quarters are added in order.
__device__ __forceinline__ void sum_columns(const ColumnSums& c) {
    constexpr int U = 16;
    __shared__ float quarter[4][64];
    const int column = threadIdx.x & 63, q = threadIdx.x >> 6;
    float f = 0.0f;
    if (column < c.columns)
        for (int r0 = q; r0 < c.rows; r0 += 4 * U) {
            float v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = r0 + 4 * u < c.rows ? c.part[(r0 + 4 * u) * c.columns + column] : 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u) f += v[u];
        }
    quarter[q][column] = f;
    __syncthreads();
    if (threadIdx.x < static_cast<unsigned>(c.columns))
        c.out[column] = (quarter[0][column] + quarter[1][column]) + (quarter[2][column] + quarter[3][column]);
}

// K slices of contract for this shape; partials holds that many [tokens, rank] sums.
int contract_slices(int tile_bound, int64_t k, int64_t rank);

// partials[s][i][c] = sum over slice s of x[order[i]][k] * w[adapter][c][k]; rows of no
// adapter are not written.
int launch_contract(const uint16_t* x, const uint16_t* w, const Groups& g, float* partials, int slices, int64_t tokens,
                    int64_t k, int rank, hipStream_t stream);

// out[order[i]][j] = base[order[i]][j] + scale * sum_c h[i][c] * w[adapter][c][j], h the sum
// of `slices` partials; rows of no adapter: out = base. base may be null (0) or out.
// w is bf16, or fp32 for w32. h_out (may be null) receives h.
int launch_spread(const float* partials, int slices, const void* w, bool w32, const float* scales, const Groups& g,
                  const uint16_t* base, uint16_t* out, float* h_out, int64_t tokens, int64_t width, int rank,
                  hipStream_t stream);

// out[a][c][j] = scale_a * sum over a's rows of h[i][c] * x[order[i]][j], fp32 or bf16;
// 0 for an adapter without rows. partials: partial_bound * rank * width fp32 (one group:
// split_bound, none where that is 1).
struct OuterJob {
    const float* h = nullptr;
    const uint16_t* x = nullptr;
    float* partials = nullptr;
    void* out = nullptr;
    int64_t width = 0;  // 0: no job
};

// One or two such products on the same groups. `extra` sums ride on the launch that adds
// the splits up (one group: only where it has several).
int launch_outer(const OuterJob& first, const OuterJob& second, const float* scales, const Groups& g, bool out_bf16,
                 int64_t tokens, int rank, int adapters, hipStream_t stream, ColumnSums extra = {});

}  // namespace moe
