// Attention of single tokens over ranges of a paged cache (ranges.hip): the
// windowed decode and the decode of sequences that share their leading pages.
#pragma once

#include <algorithm>
#include <vector>

#include "sa_internal.h"

namespace sa {

// Rows (sequences) of one launch see, in order, the tokens of their group's
// source and of a source of their own.  A source is the token ranges [0, a1)
// and [b0, b1) of one cache row (a1 <= b0).
struct RangeSource {
    int32_t cache_row, a1, b0, b1;
};

// One call: n_rows rows of q [n_rows][n_q][D]; row i's own source own[i];
// n_groups runs of consecutive rows, run g of group_rows[g] rows seeing
// group[g] as well (n_groups 0: none).  Groups of more than kRowsPerLaunch
// rows are attended kRowsPerLaunch at a time.
struct RangePlan {
    int n_rows;
    const RangeSource* own;
    int n_groups;
    const int32_t* group_rows;
    const RangeSource* group;
};

// Head sizes the kernels take.
inline bool ranges_head_dim(int d) { return d == 64 || d == 128; }
constexpr int kRangesMaxRep = 64;   // query heads per KV head
// Workspace for any call of n_rows rows whose own sources have at most
// own_tokens tokens and whose groups' have at most group_tokens.
size_t ranges_ws(int n_rows, int n_q, int d, long long own_tokens, long long group_tokens);
sa_status decode_ranges(const PagedView& c, const float* q, int n_q, const RangePlan& plan, float scale, float* out,
                        void* ws, size_t ws_bytes, hipStream_t st);

// A chunk of n new tokens, appended at positions len .. len + n - 1 of a cache row,
// each seeing what came before it and itself; first: its first row of q and out.
struct ChunkSeq {
    int32_t cache_row, len, n, first;
};

// The last of n (1 .. 64) chunks whose rows begin at or before row, for all lanes of a
// wave alike; row is at or behind the first chunk's.
__device__ __forceinline__ int chunk_of(const ChunkSeq* seqs, int n, int row) {
    if (n == 1) return 0;
    const int lane = threadIdx.x & (kWave - 1);
    return __popcll(__ballot(lane < n && seqs[lane].first <= row)) - 1;
}

// Launches launch(grid, first row) over the partials of rows query rows, 256 / (D / 4) of them
// per workgroup of 256; a grid has fewer than 2^32 threads.
template <int D, class Launch>
sa_status merge_rows(long long rows, const Launch& launch) {
    constexpr long long per = 256 / (D / 4), most = per << 23;
    for (long long row = 0; row < rows; row += most) {
        launch(dim3((unsigned)((std::min(most, rows - row) + per - 1) / per)), row);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}

// Attention of chunks of new tokens: q and out [rows][n_q][D], fp32 or (q16) bf16.
// extend_rows_ws: for n <= kRowsPerLaunch of them, enough for any lengths of at most
// max_tokens.
size_t extend_rows_ws(int n, const int32_t* counts, int n_q, int n_kv, int d, bool f32, long long max_tokens);
sa_status extend_rows(const PagedView& c, const void* q, bool q16, int n_q, const ChunkSeq* seqs, int n, float scale,
                      void* out, void* ws, size_t ws_bytes, hipStream_t st);

// The same for chunks of many query rows (extend.hip), and which of a call's chunks
// (none of them empty) go which way.
void split_chunks(sa_dtype kv, int rep, int n_kv, const ChunkSeq* seqs, int n, std::vector<ChunkSeq>* many,
                  std::vector<ChunkSeq>* few);
size_t extend_blocks_ws(int n, const int32_t* counts, int n_q, int n_kv, int d, long long max_tokens);
sa_status extend_blocks(const PagedView& c, const void* q, bool q16, int n_q, const ChunkSeq* seqs, int n, float scale,
                        void* out, void* ws, size_t ws_bytes, hipStream_t st);

}  // namespace sa
