// Attention of single tokens over ranges of a paged cache (ranges.hip): the
// windowed decode and the decode of sequences that share their leading pages.
#pragma once

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

}  // namespace sa
