// Paged KV cache for gfx950 and the fused q/k RMSNorm + RoPE + K/V append.
//
// Storage: one device allocation holding, per layer, a K pool and a V pool of
// [num_pages][n_kv_heads][64][head_dim] elements (fp32, bf16 or 8-bit codes, the
// codes' scales in pools of their own).  A page of one
// head is 64 consecutive rows, so the decode kernel streams 8-32 KiB of
// contiguous memory per page.  Pages are handed out from a host free list;
// block_table[seq][j] names the page holding tokens 64j..64j+63 (-1: none).
//
// The reference keeps a dense [B, Hkv, max_seq, D] fp32 tensor per layer and
// copies it out on every step (reference tensor_cpp/include/tensor_cpp/kv_cache.h:27-238);
// here the cache stays resident and the decode kernel reads it in place.
//
// Ordering: the host decides (page_table.cpp) and publishes the table rows and
// lengths with small kernels on the stream the caller passes, so a reset,
// reserve, set_pages, append, decode and commit issued on one stream run in
// the order they were called.
#include "sa_internal.h"
#include "page_table.h"
#include "ranges.h"

#include <algorithm>
#include <cmath>
#include <functional>
#include <initializer_list>
#include <new>
#include <vector>

struct sa_kvcache {
    sa_kv_desc desc{};
    int device = 0;
    char* pool = nullptr;          // [layers][2][num_pages][n_kv][64][D]
    uint8_t* scales = nullptr;     // 8 bits: [layers][2][num_pages][n_kv][64], else NULL
    size_t scale_bytes = 0;        // K and V scales of one layer
    size_t elem_bytes = 4;
    size_t page_bytes = 0;         // one page of one of K / V: n_kv * 64 * D * elem
    size_t layer_bytes = 0;        // K pool + V pool of one layer
    size_t total_bytes = 0;
    int32_t* d_table = nullptr;    // [max_seqs][max_pages_per_seq]
    int32_t* d_lens = nullptr;     // [max_seqs]
    sa::PageTable pt;              // host decisions; the device arrays follow them
};

namespace sa {
namespace {

__global__ void fill_i32_kernel(int32_t* p, size_t n, int32_t v) {
    size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) p[i] = v;
}

__global__ void fill_zero_u128_kernel(uint4* p, size_t n) {
    size_t stride = (size_t)gridDim.x * blockDim.x;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += stride)
        p[i] = make_uint4(0, 0, 0, 0);
}

// Row [first, first + n) of the block table, values passed by value.
struct TableRow {
    int32_t v[64];
};

__global__ void write_table_kernel(int32_t* dst, TableRow row, int n) {
    if ((int)threadIdx.x < n) dst[threadIdx.x] = row.v[threadIdx.x];
}

// seq_lens[rows[i]] = add ? seq_lens[rows[i]] + val : val
__global__ void update_lens_kernel(int32_t* lens, RowList rows, int n, int val, int add) {
    int i = threadIdx.x;
    if (i < n) lens[rows.row[i]] = add ? lens[rows.row[i]] + val : val;
}

// seq_lens[rows[i]] = to[i]
__global__ void write_lens_kernel(int32_t* lens, RowList rows, RowList to, int n) {
    const int i = threadIdx.x;
    if (i < n) lens[rows.row[i]] = to.row[i];
}

__global__ void add_lens_range_kernel(int32_t* lens, int n, int val) {
    int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) lens[i] += val;
}

// Publish entries [first, n) of seq's host table row (the others are on the
// device already).
sa_status write_table_row(sa_kvcache* c, int seq, int first, int n, hipStream_t st) {
    const int mp = c->desc.max_pages_per_seq;
    const int32_t* src = c->pt.row(seq);
    for (int j0 = first; j0 < n; j0 += 64) {
        TableRow row;
        const int m = std::min(64, n - j0);
        for (int j = 0; j < m; ++j) row.v[j] = src[j0 + j];
        hipLaunchKernelGGL(write_table_kernel, dim3(1), dim3(64), 0, st,
                           c->d_table + (size_t)seq * mp + j0, row, m);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}

// Set (add = 0) or add to (add = 1) the device lengths of rows[0, n)
// (rows == NULL: 0 .. n-1).
sa_status publish_lens(sa_kvcache* c, const int32_t* rows, int n, int val, int add, hipStream_t st) {
    for (int i0 = 0; i0 < n; i0 += kRowsPerLaunch) {
        RowList rl;
        const int m = std::min(kRowsPerLaunch, n - i0);
        for (int i = 0; i < m; ++i) rl.row[i] = rows ? rows[i0 + i] : i0 + i;
        hipLaunchKernelGGL(update_lens_kernel, dim3(1), dim3(kRowsPerLaunch), 0, st, c->d_lens, rl, m, val, add);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}

sa_status refused(const Verdict& v) { return fail(v.status, v.msg); }

// ---------------------------------------------------------------------------
// Publishing a fork or a reorder: table entries, lengths and page copies of
// several rows in one launch.  Rows that share their prompt differ in a few
// entries behind it, so only entries that change are sent; a fork's shared
// entries are copied on the device.
// ---------------------------------------------------------------------------
constexpr int kEdits = 160, kCopies = 64;
struct TableEdit {
    int32_t row, col, page;
};
struct RowsArgs {
    int32_t* table;
    int32_t* lens;
    char* pool;
    uint8_t* scales;                              // 8 bits, else NULL
    size_t layer_bytes, scale_bytes;
    int max_pages, n_kv, head_bytes, row_bytes;   // head_bytes: 64 rows of one head of a page
    int n_edits, n_lens, n_copies;
    int like_dst, like_src, like_n;               // a fork: row dst's first n entries are row src's
    TableEdit edit[kEdits];
    int32_t len_row[kRowsPerLaunch], len[kRowsPerLaunch];
    PageCopy copy[kCopies];
};
static_assert(sizeof(RowsArgs) <= 4096, "kernel arguments");

// Block (x, y) copies head slice x (layer, K or V, head) of page pair y.  No
// page is both read and written in a launch.  Bound: for a few pages the latency
// of a round trip, hidden behind the host's part (28 layers, 8 heads of 128, bf16:
// a reorder of 4 rows 9 us a call, of 64 rows behind 2,000 tokens 25, a fork 6.7).
__global__ void __launch_bounds__(256) update_rows_kernel(RowsArgs a) {
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        for (int i = threadIdx.x; i < a.like_n; i += 256)
            a.table[(size_t)a.like_dst * a.max_pages + i] = a.table[(size_t)a.like_src * a.max_pages + i];
        for (int i = threadIdx.x; i < a.n_edits; i += 256)
            a.table[(size_t)a.edit[i].row * a.max_pages + a.edit[i].col] = a.edit[i].page;
        if ((int)threadIdx.x < a.n_lens) a.lens[a.len_row[threadIdx.x]] = a.len[threadIdx.x];
    }
    if ((int)blockIdx.y >= a.n_copies) return;
    const PageCopy cp = a.copy[blockIdx.y];
    const int head = blockIdx.x % a.n_kv, half = blockIdx.x / a.n_kv;   // half: 2 layer + (V)
    char* base = a.pool + (size_t)half * (a.layer_bytes / 2);
    const uint4* src = reinterpret_cast<const uint4*>(base + ((size_t)cp.src * a.n_kv + head) * a.head_bytes);
    uint4* dst = reinterpret_cast<uint4*>(base + ((size_t)cp.dst * a.n_kv + head) * a.head_bytes);
    const int n = cp.tokens * a.row_bytes / 16;
    for (int i = threadIdx.x; i < n; i += 256) dst[i] = src[i];
    if (a.scales && (int)threadIdx.x < cp.tokens) {
        uint8_t* sc = a.scales + (size_t)half * (a.scale_bytes / 2) + (size_t)head * SA_PAGE_TOKENS + threadIdx.x;
        const size_t page = (size_t)a.n_kv * SA_PAGE_TOKENS;
        sc[cp.dst * page] = sc[cp.src * page];
    }
}

// The device side of what fork and reorder decided for rows[0, n): `before`
// holds each row's table entries as they were.  like: the row whose first
// `alike` entries the one row of a fork has, which the device copies itself.
// Nothing is allocated: the page table has changed already, and the device's has
// to follow.
sa_status publish_rows(sa_kvcache* c, const std::vector<int32_t>& rows,
                       const std::vector<std::vector<int32_t>>& before, const std::vector<PageCopy>& copies,
                       hipStream_t st, int like = 0, int alike = 0) {
    // The next entry that changes: column ej of row ei (ei = rows.size(): none).
    size_t ei = 0;
    int ej = alike;
    auto seek = [&]() {
        for (; ei < rows.size(); ++ei, ej = alike) {
            const int32_t* now = c->pt.row(rows[ei]);
            const int old_n = (int)before[ei].size(), n = std::max(old_n, c->pt.npages(rows[ei]));
            for (; ej < n; ++ej)
                if (now[ej] != (ej < old_n ? before[ei][ej] : -1)) return;
        }
    };
    seek();
    size_t l = 0, k = 0;   // a changed row has a length to publish: one launch at least
    while (ei < rows.size() || l < rows.size() || k < copies.size()) {
        RowsArgs a{};
        a.table = c->d_table; a.lens = c->d_lens; a.pool = c->pool; a.layer_bytes = c->layer_bytes;
        a.scales = c->scales; a.scale_bytes = c->scale_bytes;
        a.max_pages = c->desc.max_pages_per_seq; a.n_kv = c->desc.num_kv_heads;
        a.row_bytes = (int)(c->desc.head_dim * c->elem_bytes);
        a.head_bytes = SA_PAGE_TOKENS * a.row_bytes;
        if (l == 0 && alike > 0) {
            a.like_dst = rows[0]; a.like_src = like; a.like_n = alike;
        }
        for (; a.n_edits < kEdits && ei < rows.size(); ++ej, seek())
            a.edit[a.n_edits++] = TableEdit{rows[ei], ej, c->pt.row(rows[ei])[ej]};
        for (; a.n_lens < kRowsPerLaunch && l < rows.size(); ++l) {
            a.len_row[a.n_lens] = rows[l];
            a.len[a.n_lens++] = c->pt.len(rows[l]);
        }
        for (; a.n_copies < kCopies && k < copies.size(); ++k) a.copy[a.n_copies++] = copies[k];
        const dim3 grid(a.n_copies ? 2 * c->desc.num_layers * a.n_kv : 1, std::max(1, a.n_copies));
        hipLaunchKernelGGL(update_rows_kernel, grid, dim3(256), 0, st, a);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}

// Entry points that allocate host memory: nothing is thrown across the C ABI.
template <class F>
sa_status no_throw(F&& body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return fail(SA_ENOMEM, "out of host memory");
    }
}

// ---------------------------------------------------------------------------
// Fused QK-norm + RoPE + append.  A head row (query, key or value) of a prompt is
// served by D/8 lanes (16 at most), 16 bytes of each half per lane, so RoPE needs
// no lane exchange and a wave moves 4 rows of 128 elements per load; the rows of a
// small launch by D/2 lanes (64 at most; kAppendNarrow).
//
// Bound: HBM for prompts: the 29.4 MB of 1024 tokens (16 query and 8 KV heads of
// 128, bf16 cache) take 4.7 us at 6.3 TB/s; the launch takes 7.1 us, 4096 tokens
// 22.5 (rows of 64 lanes with 4-byte loads, two per wave of keys: 7.9 and 25.1).  K and V
// of 8192 tokens into an 8-bit cache, 84 MB: 16.
// ---------------------------------------------------------------------------
struct AppendArgs {
    const float* q; const float* k; const float* v;
    float* q_out;
    float* k_out;              // optional: K normed and rotated, as q_out
    // Optional: q, k and v are the sum of part_S split-K partials of rows
    // part_row0 + a token's place in q, k and v, of a [part_M][(n_q + 2 n_kv) * D] projection;
    // v also goes to v_out.
    const float* part;
    int part_S, part_M, part_row0;
    float* v_out;
    const float* wq; const float* wk;
    const float* cos_t; const float* sin_t;
    RowList rows;              // cache row of each sequence of this launch
    const int32_t* seq_lens;
    const int32_t* table;
    char* k_pool; char* v_pool;
    uint8_t* k_scale; uint8_t* v_scale;   // 8 bits
    int n_q, n_kv, max_pages, rope_max_pos;
    int s0, n_s;               // tokens [s0, s0 + n_s) of each sequence
    int S;                     // tokens of each sequence; 0: as first[] says
    float eps;
    int32_t first[kRowsPerLaunch + 1];    // sequence i's tokens are first[i] .. first[i + 1] - 1 of q, k and v
};

// What a row of an 8-bit cache is held by: codes of x 2^-e, ties to even, and the
// byte e + 127, where 2^e is the smallest power of two, from 2^-100 on, with amax <=
// 448 2^e.  A scale that is a power of two costs a floating format no accuracy, and
// products with it are exact: what is held is code 2^e to the last bit, in bf16
// too, and a row that is read back and appended again holds the same values.
struct RowScale {
    uint32_t byte;
    float up, top;   // 2^-e; the largest code's value
    __device__ __forceinline__ explicit RowScale(float amax) {
        const uint32_t u = __float_as_uint(amax);
        // 448 = 1.75 2^8
        const int e = max(-100, (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u));
        byte = (uint32_t)(e + 127);
        up = __uint_as_float((uint32_t)(127 - e) << 23);
        // 2^e 256 is beyond fp32's range where e is largest
        top = e < 120 ? 448.f : 240.f;
    }
    // Four codes, the first in the lowest byte.  Infinities and NaN become NaN.
    __device__ __forceinline__ uint32_t codes(float a, float b, float c, float d) const {
        const uint32_t lo = __builtin_amdgcn_cvt_pk_fp8_f32(fit(a), fit(b), 0, false);
        return __builtin_amdgcn_cvt_pk_fp8_f32(fit(c), fit(d), (int)lo, true);
    }
    __device__ __forceinline__ float fit(float x) const {
        const float y = x * up;
        return fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(y, -top, top) : __uint_as_float(0x7fc00000u);
    }
    // The larger of m and |x|, where x is finite.
    static __device__ __forceinline__ float larger(float m, float x) {
        return fabsf(x) < INFINITY ? fmaxf(m, fabsf(x)) : m;
    }
};

template <int D>
__global__ void __launch_bounds__(256)
qk_norm_rope_kernel(const float* x, int n_rows, const int32_t* pos, const float* w, float eps,
                    bool eps_outside, const float* cos_t, const float* sin_t, int max_pos, float* y) {
    const int lane = threadIdx.x & (kWave - 1);
    const int row = blockIdx.x * 4 + threadIdx.x / kWave;
    if (row >= n_rows) return;
    RowPairs<D> r;
    r.load(x + (size_t)row * D, lane);
    if (w) r.rms_norm(w, eps, lane, eps_outside);
    const int p = pos ? pos[row] : 0;
    if (cos_t && p >= 0 && p < max_pos) r.rope(cos_t, sin_t, p, lane);
    r.store(y + (size_t)row * D, lane);
}

// A head row over LANES lanes: lane j holds elements i .. i + E - 1 and their
// rotate-half partners i + D/2 .. for i = E j + 64 c.  The arithmetic is RowPairs'
// (the same sums in the same order), so all give the same bits.
template <int D, int E, bool VEC>
struct LaneRow {
    static_assert(E == 4 || (E == 1 && !VEC), "one or four elements");
    static constexpr int H = D / 2;
    static constexpr int LANES = (H < kWave ? H : kWave) / E;
    static constexpr int NC = (H + kWave - 1) / kWave;
    float lo[NC][E], hi[NC][E];

    // E floats; VEC: 16-byte aligned.
    __device__ static __forceinline__ void load_e(const float* x, float (&v)[E]) {
        if constexpr (VEC) {
            const float4 f = *reinterpret_cast<const float4*>(x);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = x[e];
        }
    }
    __device__ static __forceinline__ void store_e(float* y, const float (&v)[E]) {
        if constexpr (VEC) {
            *reinterpret_cast<float4*>(y) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) y[e] = v[e];
        }
    }
    __device__ __forceinline__ void load(const float* x, int j) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            load_e(x + E * j + kWave * c, lo[c]);
            load_e(x + E * j + kWave * c + H, hi[c]);
        }
    }
    // The sum, in split order, of S split-K partial rows x[t * split] ...
    __device__ __forceinline__ void load_sum(const float* x, size_t split, int S, int j) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) lo[c][e] = hi[c][e] = 0.f;
#pragma unroll 4
        for (int t = 0; t < S; ++t) {
            LaneRow p;
            p.load(x + t * split, j);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    lo[c][e] += p.lo[c][e];
                    hi[c][e] += p.hi[c][e];
                }
        }
    }
    __device__ __forceinline__ void rms_norm(const float* w, float eps, int j) {
#pragma clang fp contract(off)
        LaneRow g;
        g.load(w, j);
        float t[E] = {};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) t[e] = fmaf(lo[c][e], lo[c][e], fmaf(hi[c][e], hi[c][e], t[e]));
        float ss = t[0];
        if constexpr (E == 4) ss = (t[0] + t[1]) + (t[2] + t[3]);
        ss = group_reduce<OpSum, 1, LANES>(ss);
        const float rms = sqrtf(ss / (float)D + eps);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                lo[c][e] = (lo[c][e] / rms) * g.lo[c][e];
                hi[c][e] = (hi[c][e] / rms) * g.hi[c][e];
            }
    }
    __device__ __forceinline__ void rope(const float* cos_t, const float* sin_t, int pos, int j) {
#pragma clang fp contract(off)
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float cs[E], sn[E];
            load_e(cos_t + (size_t)pos * H + E * j + kWave * c, cs);
            load_e(sin_t + (size_t)pos * H + E * j + kWave * c, sn);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float l2 = lo[c][e] * cs[e] - hi[c][e] * sn[e];
                const float h2 = hi[c][e] * cs[e] + lo[c][e] * sn[e];
                lo[c][e] = l2;
                hi[c][e] = h2;
            }
        }
    }
    __device__ __forceinline__ void store(float* y, int j) const {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            store_e(y + E * j + kWave * c, lo[c]);
            store_e(y + E * j + kWave * c + H, hi[c]);
        }
    }
    // Row `row` of the cache pools (scale: of the scales), 16-byte aligned.
    template <int KV>
    __device__ __forceinline__ void store_pool(char* pool, uint8_t* scale, size_t at_row, int j) const {
        const size_t row = at_row * D;
        if constexpr (KV == SA_DTYPE_FP8) {
            float amax = 0.f;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int e = 0; e < E; ++e) amax = RowScale::larger(RowScale::larger(amax, lo[c][e]), hi[c][e]);
            const RowScale rs(group_reduce<OpMax, 1, LANES>(amax));
            uint8_t* d = reinterpret_cast<uint8_t*>(pool) + row;
            auto put = [&](int at, const float (&v)[E]) {
                if constexpr (E == 4) *reinterpret_cast<uint32_t*>(d + at) = rs.codes(v[0], v[1], v[2], v[3]);
                else d[at] = (uint8_t)rs.codes(v[0], 0.f, 0.f, 0.f);
            };
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                put(E * j + kWave * c, lo[c]);
                put(E * j + kWave * c + H, hi[c]);
            }
            if (j == 0) scale[at_row] = (uint8_t)rs.byte;
        } else if constexpr (KV == SA_DTYPE_BF16) {
            uint16_t* d = reinterpret_cast<uint16_t*>(pool) + row;
            auto put = [&](int at, const float (&v)[E]) {
                if constexpr (E == 4) {
                    uint32_t b[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        b[e] = f32_to_bf16_rne(v[2 * e]) | (uint32_t)f32_to_bf16_rne(v[2 * e + 1]) << 16;
                    *reinterpret_cast<uint2*>(d + at) = make_uint2(b[0], b[1]);
                } else {
                    d[at] = f32_to_bf16_rne(v[0]);
                }
            };
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                put(E * j + kWave * c, lo[c]);
                put(E * j + kWave * c + H, hi[c]);
            }
        } else {
            float* d = reinterpret_cast<float*>(pool) + row;
            auto put = [&](int at, const float (&v)[E]) {
                if constexpr (E == 4) *reinterpret_cast<float4*>(d + at) = make_float4(v[0], v[1], v[2], v[3]);
                else d[at] = v[0];
            };
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                put(E * j + kWave * c, lo[c]);
                put(E * j + kWave * c + H, hi[c]);
            }
        }
    }
};

// VEC: q, k, v, the partials, weights, tables and outputs are 16-byte aligned.
template <int D, int KV, int E, bool VEC>
__global__ void __launch_bounds__(256)
qknorm_rope_append_kernel(AppendArgs a) {
    using Row = LaneRow<D, E, VEC>;
    const int j = threadIdx.x % Row::LANES;
    const unsigned idx = blockIdx.x * (256u / Row::LANES) + threadIdx.x / Row::LANES;
    const unsigned per_token = a.n_q + 2 * a.n_kv;
    const int s = a.s0 + (int)(idx / per_token);
    const int id = (int)(idx % per_token);   // query heads, key heads, value heads
    const int i_seq = blockIdx.y;
    int first = i_seq * a.S, end = a.s0 + a.n_s;
    if (a.S == 0) {
        first = a.first[i_seq];
        end = min(end, a.first[i_seq + 1] - first);
    }
    if (s >= end) return;
    const bool is_q = id < a.n_q, is_k = !is_q && id < a.n_q + a.n_kv;
    const int head = is_q ? id : is_k ? id - a.n_q : id - a.n_q - a.n_kv;
    const size_t token = (size_t)first + s;
    const size_t src = (token * (is_q ? a.n_q : a.n_kv) + head) * D;
    const int cache_row = a.rows.row[i_seq];
    const int pos = a.seq_lens[cache_row] + s;
    Row r;
    if (a.part) {
        const size_t cols = (size_t)per_token * D;
        r.load_sum(a.part + (a.part_row0 + token) * cols + (size_t)id * D, (size_t)a.part_M * cols, a.part_S, j);
    } else {
        r.load((is_q ? a.q : is_k ? a.k : a.v) + src, j);
    }
    // The host has checked that every row has a page there; these tests only
    // keep a device length that disagrees with the host from writing out of
    // bounds.  Looked up here, so that its round trip overlaps the others.
    const bool paged = !is_q && pos < a.max_pages * 64;
    const int page = paged ? a.table[(size_t)cache_row * a.max_pages + (pos >> 6)] : -1;
    if (is_q || is_k) {
        const float* w = is_q ? a.wq : a.wk;
        if (w) r.rms_norm(w, a.eps, j);
        if (a.cos_t && pos < a.rope_max_pos) r.rope(a.cos_t, a.sin_t, pos, j);
    }
    float* copy = is_q ? a.q_out : is_k ? a.k_out : a.v_out;
    if (copy) r.store(copy + src, j);
    if (page < 0) return;
    r.template store_pool<KV>(is_k ? a.k_pool : a.v_pool, is_k ? a.k_scale : a.v_scale,
                              ((size_t)page * a.n_kv + head) * 64 + (pos & 63), j);
}

// Tokens [t0, t1) of the dense copy [n_kv][len][D] of one sequence (fp32 out): E
// elements of a row per thread, the layer's K and V (blockIdx.z) of head blockIdx.y.  Bound: HBM; 8192
// tokens, 8 heads of 128, 8 bits 84 MB, 15 us (an element per thread and load: 22).
template <int KV, int E>
__global__ void __launch_bounds__(256)
gather_kernel(const char* k_pool, const char* v_pool, const uint8_t* k_scale, const uint8_t* v_scale,
              const int32_t* table_row, int n_kv, int D, int t0, int t1, int len, float* k_out, float* v_out) {
    float* out = blockIdx.z ? v_out : k_out;
    const unsigned idx = blockIdx.x * 256u + threadIdx.x, per_row = D / E;
    const int t = t0 + (int)(idx / per_row), i = (int)(idx % per_row) * E, h = blockIdx.y;
    if (t >= t1 || !out) return;
    const int page = table_row[t >> 6];
    const size_t at = ((size_t)page * n_kv + h) * 64 + (t & 63), row = at * D + i;
    const char* pool = blockIdx.z ? v_pool : k_pool;
    float v[E];
    if constexpr (KV == SA_DTYPE_FP8) {
        const float scale = __uint_as_float((uint32_t)(blockIdx.z ? v_scale : k_scale)[at] << 23);
        const uint8_t* p = reinterpret_cast<const uint8_t*>(pool) + row;
        if constexpr (E == 4) {
            const int x = *reinterpret_cast<const int*>(p);
            v[0] = __builtin_amdgcn_cvt_f32_fp8(x, 0) * scale;
            v[1] = __builtin_amdgcn_cvt_f32_fp8(x, 1) * scale;
            v[2] = __builtin_amdgcn_cvt_f32_fp8(x, 2) * scale;
            v[3] = __builtin_amdgcn_cvt_f32_fp8(x, 3) * scale;
        } else {
            v[0] = __builtin_amdgcn_cvt_f32_fp8((int)p[0], 0) * scale;
        }
    } else if constexpr (KV == SA_DTYPE_BF16) {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(pool) + row;
        if constexpr (E == 4) {
            const uint2 x = *reinterpret_cast<const uint2*>(p);
            v[0] = bf16_lo(x.x); v[1] = bf16_hi(x.x); v[2] = bf16_lo(x.y); v[3] = bf16_hi(x.y);
        } else {
            v[0] = bf16_lo(p[0]);
        }
    } else {
        const float* p = reinterpret_cast<const float*>(pool) + row;
        if constexpr (E == 4) {
            const float4 x = *reinterpret_cast<const float4*>(p);
            v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        } else {
            v[0] = p[0];
        }
    }
    float* dst = out + ((size_t)h * len + t) * D + i;
    if constexpr (E == 4) *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
    else dst[0] = v[0];
}

bool valid_cache(const sa_kvcache* c) { return c && c->pool; }

char* k_pool_of(const sa_kvcache* c, int layer) { return c->pool + (size_t)layer * c->layer_bytes; }
char* v_pool_of(const sa_kvcache* c, int layer) {
    return c->pool + (size_t)layer * c->layer_bytes + c->layer_bytes / 2;
}
uint8_t* k_scales_of(const sa_kvcache* c, int layer) {
    return c->scales ? c->scales + (size_t)layer * c->scale_bytes : nullptr;
}
uint8_t* v_scales_of(const sa_kvcache* c, int layer) {
    return c->scales ? c->scales + (size_t)layer * c->scale_bytes + c->scale_bytes / 2 : nullptr;
}

PagedView view_of(const sa_kvcache* c, int layer) {
    PagedView pv;
    pv.k_pool = k_pool_of(c, layer); pv.v_pool = v_pool_of(c, layer);
    pv.k_scale = k_scales_of(c, layer); pv.v_scale = v_scales_of(c, layer);
    pv.block_table = c->d_table; pv.seq_lens = c->d_lens;
    pv.n_kv = c->desc.num_kv_heads; pv.d = c->desc.head_dim;
    pv.max_pages = c->desc.max_pages_per_seq; pv.num_pages = c->desc.num_pages;
    pv.kv = c->desc.kv_dtype;
    pv.bf16 = c->desc.kv_dtype == SA_DTYPE_BF16;
    return pv;
}

// Kernels of a cache run on its own device; a call made while another one is
// current is refused.
sa_status on_cache_device(const sa_kvcache* c) {
    int dev = 0;
    SA_HIP_TRY(hipGetDevice(&dev));
    if (dev != c->device) return fail(SA_EINVAL, "the cache lives on another device than the current one");
    return SA_OK;
}

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" sa_status sa_kvcache_create(const sa_kv_desc* d, sa_kvcache** out) {
    clear_error();
    if (!d || !out) return fail(SA_EINVAL, "null pointer");
    *out = nullptr;
    if (d->num_layers <= 0 || d->num_kv_heads <= 0 || d->max_seqs <= 0 ||
        d->max_pages_per_seq <= 0 || d->num_pages <= 0)
        return fail(SA_EINVAL, "cache dimensions must be positive");
    if (d->max_pages_per_seq > (1 << 18))
        return fail(SA_EINVAL, "max_pages_per_seq must be at most 262144 (16M tokens)");
    if (d->head_dim != 8 && d->head_dim != 16 && d->head_dim != 32 && d->head_dim != 64 && d->head_dim != 128 &&
        d->head_dim != 256)
        return fail(SA_EINVAL, "head_dim must be 8, 16, 32, 64, 128 or 256");
    if (d->kv_dtype != SA_DTYPE_F32 && d->kv_dtype != SA_DTYPE_BF16 && d->kv_dtype != SA_DTYPE_FP8)
        return fail(SA_EINVAL, "kv_dtype must be F32, BF16 or FP8");
    const bool fp8 = d->kv_dtype == SA_DTYPE_FP8;
    if (fp8 && !ranges_head_dim(d->head_dim)) return fail(SA_EINVAL, "caches in 8 bits take head_dim 64 or 128");
    int device = 0;
    const hipError_t de = hipGetDevice(&device);
    if (de != hipSuccess) return hip_fail(de, "hipGetDevice");
    auto* c = new sa_kvcache();
    c->desc = *d;
    c->device = device;
    c->elem_bytes = fp8 ? 1 : d->kv_dtype == SA_DTYPE_BF16 ? 2 : 4;
    c->page_bytes = (size_t)d->num_kv_heads * 64 * d->head_dim * c->elem_bytes;
    c->layer_bytes = 2 * c->page_bytes * (size_t)d->num_pages;
    c->total_bytes = c->layer_bytes * (size_t)d->num_layers;
    c->scale_bytes = fp8 ? 2 * (size_t)d->num_kv_heads * SA_PAGE_TOKENS * (size_t)d->num_pages : 0;
    const size_t all_scales = c->scale_bytes * (size_t)d->num_layers;
    const size_t n_table = (size_t)d->max_seqs * d->max_pages_per_seq;
    hipError_t e = hipMalloc(&c->pool, c->total_bytes);
    if (e != hipSuccess) {
        delete c;
        return fail(SA_ENOMEM, "KV pool allocation failed");
    }
    e = hipMalloc(&c->d_table, n_table * sizeof(int32_t));
    if (e == hipSuccess) e = hipMalloc(&c->d_lens, (size_t)d->max_seqs * sizeof(int32_t));
    if (e == hipSuccess && fp8) e = hipMalloc(&c->scales, all_scales);
    if (e != hipSuccess) {
        (void)hipFree(c->pool);
        (void)hipFree(c->scales);
        (void)hipFree(c->d_table);
        (void)hipFree(c->d_lens);
        delete c;
        return fail(SA_ENOMEM, "KV table allocation failed");
    }
    c->pt.init(d->max_seqs, d->max_pages_per_seq, d->num_pages);
    *out = c;
    sa_status st = sa_kvcache_reset(c, nullptr);
    if (st == SA_OK) {
        hipError_t se = hipStreamSynchronize(nullptr);
        if (se != hipSuccess) st = hip_fail(se, "hipStreamSynchronize");
    }
    if (st != SA_OK) {
        sa_kvcache_destroy(c);
        *out = nullptr;
    }
    return st;
}

extern "C" sa_status sa_kvcache_destroy(sa_kvcache* c) {
    clear_error();
    if (!c) return SA_OK;
    // Best effort: work still queued on the cache must finish before its
    // memory goes; a failure here leaves nothing else to do.
    (void)hipDeviceSynchronize();
    (void)hipFree(c->pool);
    (void)hipFree(c->scales);
    (void)hipFree(c->d_table);
    (void)hipFree(c->d_lens);
    delete c;
    return SA_OK;
}

extern "C" sa_status sa_kvcache_reset(sa_kvcache* c, sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    hipStream_t st = as_stream(stream);
    const size_t n_table = (size_t)c->desc.max_seqs * c->desc.max_pages_per_seq;
    c->pt.reset();
    hipLaunchKernelGGL(fill_i32_kernel, dim3((n_table + 255) / 256), dim3(256), 0, st, c->d_table,
                       n_table, -1);
    SA_CHECK_LAUNCH();
    hipLaunchKernelGGL(fill_i32_kernel, dim3((c->desc.max_seqs + 255) / 256), dim3(256), 0, st,
                       c->d_lens, (size_t)c->desc.max_seqs, 0);
    SA_CHECK_LAUNCH();
    const size_t n16 = c->total_bytes / 16;
    hipLaunchKernelGGL(fill_zero_u128_kernel, dim3(4096), dim3(256), 0, st,
                       reinterpret_cast<uint4*>(c->pool), n16);
    SA_CHECK_LAUNCH();
    if (c->scales) {
        hipLaunchKernelGGL(fill_zero_u128_kernel, dim3(256), dim3(256), 0, st, reinterpret_cast<uint4*>(c->scales),
                           c->scale_bytes * (size_t)c->desc.num_layers / 16);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}

extern "C" sa_status sa_kvcache_reserve(sa_kvcache* c, int seq, int n_tokens, sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    const int before = c->pt.valid_seq(seq) ? c->pt.npages(seq) : 0;
    const Verdict v = c->pt.reserve(seq, n_tokens);
    if (!v.ok()) return refused(v);
    if (c->pt.npages(seq) == before) return SA_OK;
    return write_table_row(c, seq, before, c->pt.npages(seq), as_stream(stream));   // pages are only added
}

extern "C" sa_status sa_kvcache_set_pages(sa_kvcache* c, int seq, const int32_t* pages, int n_pages,
                                          sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    const int before = c->pt.valid_seq(seq) ? c->pt.npages(seq) : 0;
    bool len_cut = false;
    const Verdict v = c->pt.set_pages(seq, pages, n_pages, &len_cut);
    if (!v.ok()) return refused(v);
    hipStream_t st = as_stream(stream);
    // Entries past the new list become -1 on the device too.
    SA_TRY(write_table_row(c, seq, 0, std::max(before, n_pages), st));
    if (len_cut) {
        const int32_t row = seq;
        SA_TRY(publish_lens(c, &row, 1, c->pt.len(seq), 0, st));
    }
    return SA_OK;
}

extern "C" sa_status sa_kvcache_set_len(sa_kvcache* c, int seq, int len, sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    const Verdict v = c->pt.set_len(seq, len);
    if (!v.ok()) return refused(v);
    const int32_t row = seq;
    return publish_lens(c, &row, 1, len, 0, as_stream(stream));
}

extern "C" sa_status sa_kvcache_set_lens(sa_kvcache* c, const int32_t* seqs, const int32_t* lens, int n,
                                         sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    if (n < 0) return fail(SA_EINVAL, "negative sequence count");
    if (n > 0 && (!seqs || !lens)) return fail(SA_EINVAL, "null seqs or lens");
    return no_throw([&]() -> sa_status {
        SA_TRY(on_cache_device(c));
        const Verdict v = c->pt.set_lens(seqs, lens, n);
        if (!v.ok()) return refused(v);
        for (int i0 = 0; i0 < n; i0 += kRowsPerLaunch) {
            const int m = std::min(kRowsPerLaunch, n - i0);
            RowList rows, to;
            std::copy(seqs + i0, seqs + i0 + m, rows.row);
            std::copy(lens + i0, lens + i0 + m, to.row);
            hipLaunchKernelGGL(write_lens_kernel, dim3(1), dim3(kRowsPerLaunch), 0, as_stream(stream), c->d_lens, rows,
                               to, m);
            SA_CHECK_LAUNCH();
        }
        return SA_OK;
    });
}

extern "C" int sa_kvcache_len(const sa_kvcache* c, int seq) {
    if (!valid_cache(c) || !c->pt.valid_seq(seq)) return -1;
    return c->pt.len(seq);
}

extern "C" int sa_kvcache_capacity(const sa_kvcache* c, int seq) {
    if (!valid_cache(c) || !c->pt.valid_seq(seq)) return -1;
    return c->pt.capacity(seq);
}

extern "C" sa_status sa_kvcache_commit(sa_kvcache* c, const int32_t* seqs, int n_seqs, int n,
                                       sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    const Verdict v = c->pt.commit(seqs, n_seqs, n);
    if (!v.ok()) return refused(v);
    hipStream_t st = as_stream(stream);
    if (!seqs) {
        hipLaunchKernelGGL(add_lens_range_kernel, dim3((n_seqs + 255) / 256), dim3(256), 0, st,
                           c->d_lens, n_seqs, n);
        SA_CHECK_LAUNCH();
        return SA_OK;
    }
    return publish_lens(c, seqs, n_seqs, n, 1, st);
}

extern "C" sa_status sa_kvcache_fork(sa_kvcache* c, int dst, int src, int n_tokens, sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    return no_throw([&]() -> sa_status {
        SA_TRY(on_cache_device(c));
        const std::vector<int32_t> rows{dst};
        std::vector<std::vector<int32_t>> before(1);
        if (c->pt.valid_seq(dst)) before[0].assign(c->pt.row(dst), c->pt.row(dst) + c->pt.npages(dst));
        std::vector<PageCopy> copies;
        const Verdict v = c->pt.fork(dst, src, n_tokens, &copies);
        if (!v.ok()) return refused(v);
        return publish_rows(c, rows, before, copies, as_stream(stream), src, n_tokens / SA_PAGE_TOKENS);
    });
}

extern "C" sa_status sa_kvcache_reorder(sa_kvcache* c, const int32_t* rows, const int32_t* parents, int n,
                                        sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    return no_throw([&]() -> sa_status {
        SA_TRY(on_cache_device(c));
        std::vector<int32_t> changed;
        std::vector<std::vector<int32_t>> before;
        for (int i = 0; rows && parents && i < n; ++i) {
            if (!c->pt.valid_seq(rows[i])) return fail(SA_ERANGE, "sequence index out of range");
            if (rows[i] == parents[i]) continue;
            changed.push_back(rows[i]);
            before.emplace_back(c->pt.row(rows[i]), c->pt.row(rows[i]) + c->pt.npages(rows[i]));
        }
        std::vector<PageCopy> copies;
        const Verdict v = c->pt.reorder(rows, parents, n, &copies);
        if (!v.ok()) return refused(v);
        return publish_rows(c, changed, before, copies, as_stream(stream));
    });
}

extern "C" sa_status sa_kvcache_get_desc(const sa_kvcache* c, sa_kv_desc* out) {
    clear_error();
    if (!valid_cache(c) || !out) return fail(SA_EINVAL, "invalid cache or null output");
    *out = c->desc;
    return SA_OK;
}

extern "C" void* sa_kvcache_k_pool(sa_kvcache* c, int layer) {
    if (!valid_cache(c) || layer < 0 || layer >= c->desc.num_layers) return nullptr;
    return k_pool_of(c, layer);
}
extern "C" void* sa_kvcache_v_pool(sa_kvcache* c, int layer) {
    if (!valid_cache(c) || layer < 0 || layer >= c->desc.num_layers) return nullptr;
    return v_pool_of(c, layer);
}
extern "C" uint8_t* sa_kvcache_k_scales(sa_kvcache* c, int layer) {
    if (!valid_cache(c) || layer < 0 || layer >= c->desc.num_layers) return nullptr;
    return k_scales_of(c, layer);
}
extern "C" uint8_t* sa_kvcache_v_scales(sa_kvcache* c, int layer) {
    if (!valid_cache(c) || layer < 0 || layer >= c->desc.num_layers) return nullptr;
    return v_scales_of(c, layer);
}
extern "C" int32_t* sa_kvcache_block_table(sa_kvcache* c) { return valid_cache(c) ? c->d_table : nullptr; }
extern "C" int32_t* sa_kvcache_seq_lens(sa_kvcache* c) { return valid_cache(c) ? c->d_lens : nullptr; }
extern "C" size_t sa_kvcache_bytes(const sa_kvcache* c) {
    return valid_cache(c) ? c->total_bytes + c->scale_bytes * (size_t)c->desc.num_layers : 0;
}

extern "C" sa_status sa_rope_table_init(float* d_cos, float* d_sin, int max_pos, int head_dim,
                                        float theta, sa_stream_t stream) {
    clear_error();
    if (!d_cos || !d_sin) return fail(SA_EINVAL, "null pointer");
    if (max_pos <= 0 || head_dim <= 0 || head_dim % 2) return fail(SA_EINVAL, "bad table size");
    const int half = head_dim / 2;
    // Same fp32 arithmetic as the reference (powf, then cosf / sinf of the
    // fp32 angle), evaluated once on the host with the C library.
    std::vector<float> inv(half), cs((size_t)max_pos * half), sn((size_t)max_pos * half);
    for (int i = 0; i < half; ++i)
        inv[i] = 1.0f / std::pow(theta, static_cast<float>(i) / static_cast<float>(head_dim));
    for (int p = 0; p < max_pos; ++p) {
        for (int i = 0; i < half; ++i) {
            const float ang = static_cast<float>(p) * inv[i];
            cs[(size_t)p * half + i] = std::cos(ang);
            sn[(size_t)p * half + i] = std::sin(ang);
        }
    }
    hipStream_t st = as_stream(stream);
    SA_HIP_TRY(hipMemcpyAsync(d_cos, cs.data(), cs.size() * sizeof(float), hipMemcpyHostToDevice, st));
    SA_HIP_TRY(hipMemcpyAsync(d_sin, sn.data(), sn.size() * sizeof(float), hipMemcpyHostToDevice, st));
    SA_HIP_TRY(hipStreamSynchronize(st));
    return SA_OK;
}

namespace sa {

namespace {

// Head rows of a launch up to which a row takes 64 lanes (at most 12 waves a CU
// of 256): alone a launch is the latency of one row, and eight divisions per
// lane are a longer chain than two.  us, 64 lanes / 16 / the launch of one wave
// per query or key-and-value row before: 64 sequences of one token, bf16 cache,
// 2.55 / 3.06 / 2.66, 64 tokens 2.56 / 2.87 / 2.65, 128 tokens (4096 rows) 2.93 / 2.94 /
// 2.91, 256 tokens 3.99 / 3.50 / 3.57, 1024 tokens 10.6 / 7.1 / 7.9.
constexpr long long kAppendNarrow = 3000;

template <int D, int KV>
void launch_append_kv(bool wide, bool vec, dim3 grid, hipStream_t st, const AppendArgs& a) {
    if (vec) hipLaunchKernelGGL((qknorm_rope_append_kernel<D, KV, 4, true>), grid, dim3(256), 0, st, a);
    else if (wide) hipLaunchKernelGGL((qknorm_rope_append_kernel<D, KV, 4, false>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((qknorm_rope_append_kernel<D, KV, 1, false>), grid, dim3(256), 0, st, a);
}
template <int D>
void launch_append(sa_dtype kv, bool wide, bool vec, dim3 grid, hipStream_t st, const AppendArgs& a) {
    if constexpr (D == 64 || D == 128)   // the head sizes of 8-bit caches
        if (kv == SA_DTYPE_FP8) return launch_append_kv<D, SA_DTYPE_FP8>(wide, vec, grid, st, a);
    if (kv == SA_DTYPE_BF16) launch_append_kv<D, SA_DTYPE_BF16>(wide, vec, grid, st, a);
    else launch_append_kv<D, SA_DTYPE_F32>(wide, vec, grid, st, a);
}

// Shared by the entry points below: q/k/v given (part == NULL), or summed from
// the n_part split-K partials of the projection at part (q, k, v NULL).
// counts: the sequences' new tokens where they differ (host), else NULL and S each.
sa_status append_impl(sa_kvcache* c, int layer, const float* q, const float* k, const float* v, const float* part,
                      int n_part, int n_seq, int S, const int32_t* counts, const int32_t* seq_ids, int n_q_heads,
                      const float* q_norm_w, const float* k_norm_w, float eps, const float* rope_cos,
                      const float* rope_sin, int rope_max_pos, float* q_out, float* k_out, float* v_out,
                      hipStream_t st) {
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    if (layer < 0 || layer >= c->desc.num_layers) return fail(SA_ERANGE, "Layer index out of range");
    const bool none = counts && n_seq > 0 && std::all_of(counts, counts + n_seq, [](int32_t m) { return m == 0; });
    if (part ? n_part <= 0 : (!k || !v) && !none) return fail(SA_EINVAL, "null k or v");
    if ((q || part) && ((!q_out && !none) || n_q_heads <= 0)) return fail(SA_EINVAL, "q needs q_out and n_q_heads > 0");
    if (n_seq <= 0 || (!counts && S <= 0)) return fail(SA_EINVAL, "n_seq and S must be positive");
    if ((rope_cos == nullptr) != (rope_sin == nullptr)) return fail(SA_EINVAL, "cos and sin go together");
    if (rope_cos && rope_max_pos <= 0) return fail(SA_EINVAL, "RoPE table needs rope_max_pos > 0");
    const Verdict vd = counts ? c->pt.check_append(seq_ids, n_seq, counts, rope_cos ? rope_max_pos : 0)
                              : c->pt.check_append(seq_ids, n_seq, S, rope_cos ? rope_max_pos : 0);
    if (!vd.ok()) return refused(vd);
    if (counts) SA_TRY(on_cache_device(c));
    long long tokens = 0;
    for (int i = 0; i < n_seq; ++i) tokens += counts ? counts[i] : S;
    if (tokens > 0x7fffffffLL) return fail(SA_EINVAL, "more than 2^31 - 1 new tokens");
    AppendArgs a{};
    a.q_out = q_out;
    a.part = part; a.part_S = n_part; a.part_M = (int)tokens;
    a.wq = q_norm_w; a.wk = k_norm_w; a.cos_t = rope_cos; a.sin_t = rope_sin;
    a.seq_lens = c->d_lens; a.table = c->d_table;
    a.k_pool = k_pool_of(c, layer); a.v_pool = v_pool_of(c, layer);
    a.k_scale = k_scales_of(c, layer); a.v_scale = v_scales_of(c, layer);
    a.n_q = q || part ? n_q_heads : 0; a.n_kv = c->desc.num_kv_heads;
    a.max_pages = c->desc.max_pages_per_seq; a.rope_max_pos = rope_max_pos; a.eps = eps;
    a.S = counts ? 0 : S;
    const int rows = a.n_q + 2 * a.n_kv;
    const int D = c->desc.head_dim;
    const sa_dtype kv = c->desc.kv_dtype;
    // Up to kRowsPerLaunch sequences per launch, their cache rows by value.
    size_t at = 0;   // the launch's first token
    for (int i0 = 0; i0 < n_seq; i0 += kRowsPerLaunch) {
        const int m = std::min(kRowsPerLaunch, n_seq - i0);
        int most = 0;
        a.first[0] = 0;
        for (int i = 0; i < m; ++i) {
            const int n = counts ? counts[i0 + i] : S;
            a.rows.row[i] = seq_ids ? seq_ids[i0 + i] : i0 + i;
            a.first[i + 1] = a.first[i] + n;
            most = std::max(most, n);
        }
        a.q = q ? q + at * n_q_heads * D : nullptr;
        a.q_out = a.n_q ? q_out + at * n_q_heads * D : nullptr;
        a.k = k ? k + at * a.n_kv * D : nullptr;
        a.k_out = k_out ? k_out + at * a.n_kv * D : nullptr;
        a.v = v ? v + at * a.n_kv * D : nullptr;
        a.v_out = v_out ? v_out + at * a.n_kv * D : nullptr;
        a.part_row0 = (int)at;
        at += a.first[m];
        const bool wide = (long long)rows * a.first[m] > kAppendNarrow;
        bool vec = wide;   // the launch's pointers allow 16-byte accesses
        for (const void* p : std::initializer_list<const void*>{a.q, a.k, a.v, a.part, a.q_out, a.k_out, a.v_out, a.wq,
                                                                a.wk, a.cos_t, a.sin_t})
            vec = vec && aligned16(p);
        const int lanes = std::min(D / 2, kWave) / (wide ? 4 : 1);
        const int step = tokens_per_launch(rows, lanes);
        for (a.s0 = 0; a.s0 < most; a.s0 += a.n_s) {
            a.n_s = std::min(step, most - a.s0);
            const dim3 grid((unsigned)(((long long)rows * a.n_s * lanes + 255) / 256), m);
            switch (D) {
                case 8: launch_append<8>(kv, wide, vec, grid, st, a); break;
                case 16: launch_append<16>(kv, wide, vec, grid, st, a); break;
                case 32: launch_append<32>(kv, wide, vec, grid, st, a); break;
                case 64: launch_append<64>(kv, wide, vec, grid, st, a); break;
                case 128: launch_append<128>(kv, wide, vec, grid, st, a); break;
                case 256: launch_append<256>(kv, wide, vec, grid, st, a); break;
                default: return fail(SA_EINVAL, "head_dim");
            }
            SA_CHECK_LAUNCH();
        }
    }
    return SA_OK;
}

}  // namespace

sa_status qknorm_rope_append(sa_kvcache* c, int layer, const float* q, const float* k, const float* v, int n_seq,
                             int S, const int32_t* seq_ids, int n_q_heads, const float* q_norm_w,
                             const float* k_norm_w, float eps, const float* rope_cos, const float* rope_sin,
                             int rope_max_pos, float* q_out, float* k_out, hipStream_t st) {
    return append_impl(c, layer, q, k, v, nullptr, 0, n_seq, S, nullptr, seq_ids, n_q_heads, q_norm_w, k_norm_w, eps,
                       rope_cos, rope_sin, rope_max_pos, q_out, k_out, nullptr, st);
}

sa_status qknorm_rope_append_partials(sa_kvcache* c, int layer, const float* part, int n_part, int n_seq, int S,
                                      int n_q_heads, const float* q_norm_w, const float* k_norm_w, float eps,
                                      const float* rope_cos, const float* rope_sin, int rope_max_pos, float* q_out,
                                      float* k_out, float* v_out, hipStream_t st) {
    if (!part) return fail(SA_EINVAL, "null partials");
    return append_impl(c, layer, nullptr, nullptr, nullptr, part, n_part, n_seq, S, nullptr, nullptr, n_q_heads,
                       q_norm_w, k_norm_w, eps, rope_cos, rope_sin, rope_max_pos, q_out, k_out, v_out, st);
}

sa_status append_partials_ragged(sa_kvcache* c, int layer, const float* part, int n_part, int n_seq,
                                 const int32_t* counts, int n_q_heads, const float* q_norm_w, const float* k_norm_w,
                                 float eps, const float* rope_cos, const float* rope_sin, int rope_max_pos,
                                 float* q_out, hipStream_t st) {
    if (!part) return fail(SA_EINVAL, "null partials");
    return append_impl(c, layer, nullptr, nullptr, nullptr, part, n_part, n_seq, 0, counts, nullptr, n_q_heads,
                       q_norm_w, k_norm_w, eps, rope_cos, rope_sin, rope_max_pos, q_out, nullptr, nullptr, st);
}

}  // namespace sa

extern "C" sa_status sa_qknorm_rope_append(sa_kvcache* c, int layer, const float* q, const float* k,
                                           const float* v, int n_seq, int S, const int32_t* seq_ids,
                                           int n_q_heads, const float* q_norm_w,
                                           const float* k_norm_w, float eps, const float* rope_cos,
                                           const float* rope_sin, int rope_max_pos, float* q_out,
                                           sa_stream_t stream) {
    clear_error();
    return qknorm_rope_append(c, layer, q, k, v, n_seq, S, seq_ids, n_q_heads, q_norm_w, k_norm_w, eps, rope_cos,
                              rope_sin, rope_max_pos, q_out, nullptr, as_stream(stream));
}

extern "C" sa_status sa_qknorm_rope_append_ragged(sa_kvcache* c, int layer, const float* q, const float* k,
                                                  const float* v, int n_seq, const int32_t* counts,
                                                  const int32_t* seq_ids, int n_q_heads, const float* q_norm_w,
                                                  const float* k_norm_w, float eps, const float* rope_cos,
                                                  const float* rope_sin, int rope_max_pos, float* q_out,
                                                  sa_stream_t stream) {
    clear_error();
    if (!counts) return fail(SA_EINVAL, "null counts");
    return no_throw([&] {
        return append_impl(c, layer, q, k, v, nullptr, 0, n_seq, 0, counts, seq_ids, n_q_heads, q_norm_w, k_norm_w,
                           eps, rope_cos, rope_sin, rope_max_pos, q_out, nullptr, nullptr, as_stream(stream));
    });
}

namespace sa {
namespace {

// A step's queries, normed and rotated, before the partials of a decode over an
// 8-bit cache.
size_t step_q_bytes(const sa_kvcache* c, int n_seq, int n_q_heads) {
    return ((size_t)n_seq * n_q_heads * c->desc.head_dim * sizeof(float) + 255) / 256 * 256;
}

sa_status check_ranges(const sa_kvcache* c, int layer, const void* q, int n_seq, int n_q_heads, const void* out,
                       const void* ws, size_t ws_bytes, size_t ws_need);

// Decode over an 8-bit cache: every row's tokens as one range.
sa_status decode_fp8(const sa_kvcache* c, int layer, const float* q, int n_seq, const int32_t* seq_ids, int n_q_heads,
                     int n_pending, float scale, float* out, void* ws, size_t ws_bytes, hipStream_t st) {
    const size_t need = ranges_ws(n_seq, n_q_heads, c->desc.head_dim,
                                  (long long)c->desc.max_pages_per_seq * SA_PAGE_TOKENS, 0);
    SA_TRY(check_ranges(c, layer, q, n_seq, n_q_heads, out, ws, ws_bytes, need));
    const Verdict vd = c->pt.check_decode(seq_ids, n_seq, n_pending, nullptr, nullptr);
    if (!vd.ok()) return refused(vd);
    std::vector<RangeSource> own(n_seq);
    for (int i = 0; i < n_seq; ++i) {
        const int row = seq_ids ? seq_ids[i] : i;
        own[i] = RangeSource{row, 0, 0, c->pt.len(row) + n_pending};
    }
    return decode_ranges(view_of(c, layer), q, n_q_heads, RangePlan{n_seq, own.data(), 0, nullptr, nullptr}, scale, out,
                         ws, ws_bytes, st);
}

}  // namespace
}  // namespace sa

extern "C" size_t sa_paged_decode_ws_bytes(const sa_kvcache* c, int n_seq, int n_q_heads) {
    if (!valid_cache(c) || n_seq <= 0 || n_q_heads <= 0) return 0;
    if (c->scales)
        return step_q_bytes(c, n_seq, n_q_heads) +
               ranges_ws(n_seq, n_q_heads, c->desc.head_dim, (long long)c->desc.max_pages_per_seq * SA_PAGE_TOKENS, 0);
    return paged_ws(n_seq, n_q_heads, c->desc.num_kv_heads, c->desc.head_dim, c->desc.max_pages_per_seq);
}

extern "C" sa_status sa_paged_decode(const sa_kvcache* c, int layer, const float* q, int n_seq,
                                     const int32_t* seq_ids, int n_q_heads, int n_pending, float scale,
                                     float* out, void* ws, size_t ws_bytes, sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    if (layer < 0 || layer >= c->desc.num_layers) return fail(SA_ERANGE, "Layer index out of range");
    if (n_seq <= 0) return fail(SA_EINVAL, "n_seq must be positive");
    return no_throw([&]() -> sa_status {
        if (c->scales)
            return decode_fp8(c, layer, q, n_seq, seq_ids, n_q_heads, n_pending, scale, out, ws, ws_bytes,
                              as_stream(stream));
        int max_len = 0;
        long long total = 0;
        const Verdict vd = c->pt.check_decode(seq_ids, n_seq, n_pending, &max_len, &total);
        if (!vd.ok()) return refused(vd);
        const PagedView pv = view_of(c, layer);
        std::vector<int32_t> lens(n_seq);
        for (int i = 0; i < n_seq; ++i) lens[i] = c->pt.len(seq_ids ? seq_ids[i] : i);
        return decode_paged(pv, q, n_seq, seq_ids, lens.data(), n_q_heads, n_pending, max_len, total, scale, out, ws,
                            ws_bytes, as_stream(stream));
    });
}

namespace sa {
namespace {

// What the decodes over ranges share: the checks of their arguments and the
// view of a layer's pools.
sa_status check_ranges(const sa_kvcache* c, int layer, const void* q, int n_seq, int n_q_heads, const void* out,
                       const void* ws, size_t ws_bytes, size_t ws_need) {
    if (layer < 0 || layer >= c->desc.num_layers) return fail(SA_ERANGE, "Layer index out of range");
    if (!q || !out) return fail(SA_EINVAL, "null pointer");
    if (n_seq <= 0) return fail(SA_EINVAL, "n_seq must be positive");
    if (n_q_heads <= 0 || n_q_heads % c->desc.num_kv_heads) return fail(SA_EINVAL, "bad head counts");
    if (n_q_heads / c->desc.num_kv_heads > kRangesMaxRep || n_q_heads > 65535)
        return fail(SA_EINVAL, "at most 64 query heads per KV head");
    if (!ranges_head_dim(c->desc.head_dim)) return fail(SA_EINVAL, "head_dim must be 64 or 128");
    if (!aligned16(q) || !aligned16(out) || !aligned16(ws))
        return fail(SA_EINVAL, "q, out and ws must be 16-byte aligned");
    // A call of one launch is refused by that launch, which may need less.
    if (n_seq > kRowsPerLaunch && ws_need > 0 && (!ws || ws_bytes < ws_need))
        return fail(SA_ENOMEM, "workspace too small for the partials");
    return on_cache_device(c);
}

}  // namespace
}  // namespace sa

sa_status sa::check_append(const sa_kvcache* c, int n, int S, int max_pos) {
    const Verdict v = c->pt.check_append(nullptr, n, S, max_pos);
    return v.ok() ? SA_OK : refused(v);
}

sa_status sa::check_append_ragged(const sa_kvcache* c, int n, const int32_t* counts, int max_pos) {
    const Verdict v = c->pt.check_append(nullptr, n, counts, max_pos);
    return v.ok() ? on_cache_device(c) : refused(v);
}

long long sa::shared_tokens_saved(const sa_kvcache* c, const int32_t* sizes, int n_groups) {
    long long saved = 0;
    for (int g = 0, at = 0; g < n_groups; at += sizes[g], ++g)
        saved += (long long)(sizes[g] - 1) * c->pt.shared_tokens(nullptr, at, sizes[g], 1);
    return saved;
}

extern "C" size_t sa_paged_decode_window_ws_bytes(const sa_kvcache* c, int n_seq, int n_q_heads, int window,
                                                  int n_sink) {
    if (!valid_cache(c) || n_seq <= 0 || n_q_heads <= 0 || window <= 0 || n_sink < 0) return 0;
    const long long seen = std::min<long long>((long long)c->desc.max_pages_per_seq * SA_PAGE_TOKENS,
                                               (long long)window + n_sink);
    return ranges_ws(n_seq, n_q_heads, c->desc.head_dim, seen, 0);
}

extern "C" sa_status sa_paged_decode_window(const sa_kvcache* c, int layer, const float* q, int n_seq,
                                            const int32_t* seq_ids, int n_q_heads, int n_pending, int window,
                                            int n_sink, float scale, float* out, void* ws, size_t ws_bytes,
                                            sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    if (window <= 0) return fail(SA_EINVAL, "window must be positive");
    if (n_sink < 0) return fail(SA_EINVAL, "n_sink must be >= 0");
    return no_throw([&]() -> sa_status {
        SA_TRY(check_ranges(c, layer, q, n_seq, n_q_heads, out, ws, ws_bytes,
                            sa_paged_decode_window_ws_bytes(c, n_seq, n_q_heads, window, n_sink)));
        const Verdict vd = c->pt.check_decode(seq_ids, n_seq, n_pending, nullptr, nullptr);
        if (!vd.ok()) return refused(vd);
        std::vector<RangeSource> own(n_seq);
        for (int i = 0; i < n_seq; ++i) {
            const int row = seq_ids ? seq_ids[i] : i;
            const int len = c->pt.len(row) + n_pending, first = std::max(0, len - window);
            // sinks that reach the window leave one range
            own[i] = n_sink < first ? RangeSource{row, n_sink, first, len} : RangeSource{row, 0, 0, len};
        }
        return decode_ranges(view_of(c, layer), q, n_q_heads, RangePlan{n_seq, own.data(), 0, nullptr, nullptr}, scale,
                             out, ws, ws_bytes, as_stream(stream));
    });
}

extern "C" size_t sa_paged_decode_shared_ws_bytes(const sa_kvcache* c, int n_seq, int n_q_heads) {
    if (!valid_cache(c) || n_seq <= 0 || n_q_heads <= 0) return 0;
    const long long tokens = (long long)c->desc.max_pages_per_seq * SA_PAGE_TOKENS;
    return ranges_ws(n_seq, n_q_heads, c->desc.head_dim, tokens, tokens);
}

extern "C" sa_status sa_paged_decode_shared(const sa_kvcache* c, int layer, const float* q, int n_seq,
                                            const int32_t* seq_ids, const int32_t* group_sizes, int n_groups,
                                            int n_q_heads, int n_pending, float scale, float* out, void* ws,
                                            size_t ws_bytes, sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    if (group_sizes ? n_groups <= 0 : n_groups != 0) return fail(SA_EINVAL, "group_sizes and n_groups go together");
    return no_throw([&]() -> sa_status {
        SA_TRY(check_ranges(c, layer, q, n_seq, n_q_heads, out, ws, ws_bytes,
                            sa_paged_decode_shared_ws_bytes(c, n_seq, n_q_heads)));
        const Verdict vd = c->pt.check_decode(seq_ids, n_seq, n_pending, nullptr, nullptr);
        if (!vd.ok()) return refused(vd);
        const std::vector<int32_t> sizes = group_sizes ? std::vector<int32_t>(group_sizes, group_sizes + n_groups)
                                                       : std::vector<int32_t>{n_seq};
        long long rows = 0;
        for (int32_t n : sizes) {
            if (n <= 0) return fail(SA_EINVAL, "group sizes must be positive");
            rows += n;
        }
        if (rows != n_seq) return fail(SA_EINVAL, "group sizes must add up to n_seq");
        std::vector<RangeSource> own(n_seq), group;
        bool any = false;
        int at = 0;
        for (int32_t n : sizes) {
            const int first = seq_ids ? seq_ids[at] : at;
            const int shared = c->pt.shared_tokens(seq_ids ? seq_ids + at : nullptr, first, n, n_pending);
            group.push_back(RangeSource{first, shared, shared, shared});
            any = any || shared > 0;
            for (int i = at; i < at + n; ++i) {
                const int row = seq_ids ? seq_ids[i] : i;
                own[i] = RangeSource{row, 0, shared, c->pt.len(row) + n_pending};
            }
            at += n;
        }
        return decode_ranges(view_of(c, layer), q, n_q_heads,
                             RangePlan{n_seq, own.data(), any ? (int)sizes.size() : 0, sizes.data(), group.data()},
                             scale, out, ws, ws_bytes, as_stream(stream));
    });
}

extern "C" size_t sa_paged_extend_ws_bytes(const sa_kvcache* c, int n_seq, const int32_t* counts, int n_q_heads) {
    if (!valid_cache(c) || n_seq <= 0 || !counts || n_q_heads <= 0 || n_q_heads % c->desc.num_kv_heads ||
        !ranges_head_dim(c->desc.head_dim) || n_q_heads / c->desc.num_kv_heads > kRangesMaxRep)
        return 0;
    for (int i = 0; i < n_seq; ++i)
        if (counts[i] < 0) return 0;
    const long long tokens = (long long)c->desc.max_pages_per_seq * SA_PAGE_TOKENS;
    const bool f32 = c->desc.kv_dtype == SA_DTYPE_F32;
    // Whichever way the sequences go: a launch of either takes up to kRowsPerLaunch of
    // them, which need no more than the largest.
    int32_t most[kRowsPerLaunch];
    if (n_seq > kRowsPerLaunch) {
        std::partial_sort_copy(counts, counts + n_seq, most, most + kRowsPerLaunch, std::greater<int32_t>());
        counts = most;
        n_seq = kRowsPerLaunch;
    }
    return std::max(extend_rows_ws(n_seq, counts, n_q_heads, c->desc.num_kv_heads, c->desc.head_dim, f32, tokens),
                    extend_blocks_ws(n_seq, counts, n_q_heads, c->desc.num_kv_heads, c->desc.head_dim, tokens));
}

extern "C" sa_status sa_paged_extend(const sa_kvcache* c, int layer, const void* q, sa_dtype q_dtype, int n_seq,
                                     const int32_t* seq_ids, const int32_t* counts, int n_q_heads, float scale,
                                     void* out, void* ws, size_t ws_bytes, sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    if (q_dtype != SA_DTYPE_F32 && q_dtype != SA_DTYPE_BF16) return fail(SA_EINVAL, "q_dtype must be F32 or BF16");
    if (q_dtype == SA_DTYPE_BF16 && c->desc.kv_dtype == SA_DTYPE_F32)
        return fail(SA_EINVAL, "bf16 queries take a bf16 or 8-bit cache");
    if (!counts) return fail(SA_EINVAL, "null counts");
    return no_throw([&]() -> sa_status {
        const Verdict vd = c->pt.check_rows(seq_ids, n_seq, false);
        if (!vd.ok()) return refused(vd);
        // nothing to do needs no tensors
        if (n_seq > 0 && std::all_of(counts, counts + n_seq, [](int32_t k) { return k == 0; })) return SA_OK;
        const size_t need = sa_paged_extend_ws_bytes(c, n_seq, counts, n_q_heads);
        SA_TRY(check_ranges(c, layer, q, n_seq, n_q_heads, out, ws, ws_bytes, need));
        // Sequences of few and of many query rows go their own ways, one behind the
        // other, in the same workspace.
        const PagedView view = view_of(c, layer);
        const bool q16 = q_dtype == SA_DTYPE_BF16;
        std::vector<ChunkSeq> seqs, few, many;
        seqs.reserve(n_seq);
        long long rows = 0;
        for (int i = 0; i < n_seq; ++i) {
            const int row = seq_ids ? seq_ids[i] : i, len = c->pt.len(row);
            if (counts[i] < 0) return fail(SA_EINVAL, "counts must be >= 0");
            if (rows + counts[i] > kMaxNewTokens) return fail(SA_EINVAL, "more than 2^20 new tokens");
            if ((long long)len + counts[i] > c->pt.capacity(row))
                return fail(SA_ERANGE, "Requested seq_len exceeds cached length");
            if (counts[i]) seqs.push_back(ChunkSeq{row, len, counts[i], (int)rows});
            rows += counts[i];
        }
        const size_t bytes = (size_t)rows * n_q_heads * view.d * (q16 ? 2 : 4), used = std::min(ws_bytes, need);
        if (overlap(out, bytes, q, bytes) || overlap(ws, used, q, bytes) || overlap(ws, used, out, bytes))
            return fail(SA_EINVAL, "q, out and ws must not overlap");
        split_chunks(view.kv, n_q_heads / view.n_kv, view.n_kv, seqs.data(), (int)seqs.size(), &many, &few);
        // The second way's launch must not be refused behind the first's.
        if (!many.empty() && !few.empty() && need > 0 && (!ws || ws_bytes < need))
            return fail(SA_ENOMEM, "workspace too small for the partials");
        if (!many.empty())
            SA_TRY(extend_blocks(view, q, q16, n_q_heads, many.data(), (int)many.size(), scale, out, ws, ws_bytes,
                                 as_stream(stream)));
        if (few.empty()) return SA_OK;
        return extend_rows(view, q, q16, n_q_heads, few.data(), (int)few.size(), scale, out, ws, ws_bytes,
                           as_stream(stream));
    });
}

namespace sa {
namespace {

// sa_append_decode; with part set, q, k and v come from the projection's
// split-K partials instead (FusedAppend::part).
sa_status append_decode_impl(sa_kvcache* c, int layer, const float* q, const float* k, const float* v,
                             const float* part, int n_part, int n_seq, const int32_t* seq_ids, int n_q_heads,
                             const float* q_norm_w, const float* k_norm_w, float eps, const float* rope_cos,
                             const float* rope_sin, int rope_max_pos, float scale, float* out, float* q_out,
                             void* ws, size_t ws_bytes, int commit, hipStream_t stream,
                             DecodeParts* parts = nullptr) {
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    if (layer < 0 || layer >= c->desc.num_layers) return fail(SA_ERANGE, "Layer index out of range");
    if (!out || (part ? n_part <= 0 : (!q || !k || !v))) return fail(SA_EINVAL, "null q, k, v or out");
    if (n_seq <= 0) return fail(SA_EINVAL, "n_seq must be positive");
    if (n_q_heads <= 0 || n_q_heads % c->desc.num_kv_heads) return fail(SA_EINVAL, "bad head counts");
    if ((rope_cos == nullptr) != (rope_sin == nullptr)) return fail(SA_EINVAL, "cos and sin go together");
    if (rope_cos && rope_max_pos <= 0) return fail(SA_EINVAL, "RoPE table needs rope_max_pos > 0");
    if (c->desc.head_dim < 64) return fail(SA_EINVAL, "the fused decode step takes head_dim 64, 128 or 256");
    Verdict vd = c->pt.check_append(seq_ids, n_seq, 1, rope_cos ? rope_max_pos : 0);
    if (!vd.ok()) return refused(vd);
    if (c->scales) {
        // The append and the decode as launches of their own, the normed, rotated
        // queries where the caller wants them or before the partials.
        const size_t head = q_out ? 0 : step_q_bytes(c, n_seq, n_q_heads);
        float* q_step = q_out ? q_out : static_cast<float*>(ws);
        if (!q_out && (!ws || ws_bytes < head)) return fail(SA_ENOMEM, "workspace too small for the queries");
        if (n_q_heads / c->desc.num_kv_heads > kRangesMaxRep || n_q_heads > 65535)
            return fail(SA_EINVAL, "at most 64 query heads per KV head");
        if (!aligned16(out) || !aligned16(q_step) || !aligned16(ws))
            return fail(SA_EINVAL, "out, q_out and ws must be 16-byte aligned");
        const size_t need = sa_paged_decode_ws_bytes(c, n_seq, n_q_heads);
        if (need > 0 && (!ws || ws_bytes < need)) return fail(SA_ENOMEM, "workspace too small for the partials");
        SA_TRY(on_cache_device(c));
        SA_TRY(append_impl(c, layer, q, k, v, part, n_part, n_seq, 1, nullptr, seq_ids, n_q_heads, q_norm_w, k_norm_w,
                           eps, rope_cos, rope_sin, rope_max_pos, q_step, nullptr, nullptr, stream));
        SA_TRY(decode_fp8(c, layer, q_step, n_seq, seq_ids, n_q_heads, 1, scale, out,
                          ws ? static_cast<char*>(ws) + head : nullptr, ws_bytes - head, stream));
        return commit ? sa_kvcache_commit(c, seq_ids, n_seq, 1, stream) : SA_OK;
    }
    int max_len = 0;
    long long total = 0;
    vd = c->pt.check_decode(seq_ids, n_seq, 1, &max_len, &total);
    if (!vd.ok()) return refused(vd);
    std::vector<int32_t> pos(n_seq);
    for (int i = 0; i < n_seq; ++i) pos[i] = c->pt.len(seq_ids ? seq_ids[i] : i);
    const PagedView pv = view_of(c, layer);
    FusedAppend f{};
    f.k = k; f.v = v; f.wq = q_norm_w; f.wk = k_norm_w; f.eps = eps;
    f.cos_t = rope_cos; f.sin_t = rope_sin; f.rope_max_pos = rope_max_pos;
    // One launch (up to kRowsPerLaunch rows) commits inside the kernel.  A
    // call of more rows takes several launches; their lengths are published
    // by one pass after the last launch is enqueued, so a launch that fails
    // leaves every device length as it was.
    const bool in_kernel_commit = commit && n_seq <= kRowsPerLaunch;
    f.q_out = q_out; f.lens = c->d_lens; f.pos = pos.data(); f.commit = in_kernel_commit;
    f.part = part; f.part_S = n_part; f.part_M = n_seq;
    f.parts = parts;
    SA_TRY(decode_paged_fused(pv, q, n_seq, seq_ids, n_q_heads, f, max_len, total, scale, out, ws, ws_bytes,
                              stream));
    if (commit) {
        if (!in_kernel_commit) SA_TRY(publish_lens(c, seq_ids, n_seq, 1, 1, stream));
        vd = c->pt.commit(seq_ids, n_seq, 1);   // checked above: cannot be refused
        if (!vd.ok()) return refused(vd);
    }
    return SA_OK;
}

}  // namespace

sa_status append_decode_partials(sa_kvcache* c, int layer, const float* part, int n_part, int n_seq,
                                 const int32_t* seq_ids, int n_q_heads, const float* q_norm_w,
                                 const float* k_norm_w, float eps, const float* rope_cos, const float* rope_sin,
                                 int rope_max_pos, float scale, float* out, float* q_out, void* ws,
                                 size_t ws_bytes, int commit, hipStream_t st, DecodeParts* parts) {
    if (!part) return fail(SA_EINVAL, "null projection partials");
    return append_decode_impl(c, layer, nullptr, nullptr, nullptr, part, n_part, n_seq, seq_ids, n_q_heads,
                              q_norm_w, k_norm_w, eps, rope_cos, rope_sin, rope_max_pos, scale, out, q_out, ws,
                              ws_bytes, commit, st, parts);
}

}  // namespace sa

extern "C" sa_status sa_append_decode(sa_kvcache* c, int layer, const float* q, const float* k, const float* v,
                                      int n_seq, const int32_t* seq_ids, int n_q_heads, const float* q_norm_w,
                                      const float* k_norm_w, float eps, const float* rope_cos,
                                      const float* rope_sin, int rope_max_pos, float scale, float* out,
                                      float* q_out, void* ws, size_t ws_bytes, int commit, sa_stream_t stream) {
    clear_error();
    if (!q || !k || !v) return fail(SA_EINVAL, "null q, k, v or out");
    return no_throw([&] {
        return append_decode_impl(c, layer, q, k, v, nullptr, 0, n_seq, seq_ids, n_q_heads, q_norm_w, k_norm_w, eps,
                                  rope_cos, rope_sin, rope_max_pos, scale, out, q_out, ws, ws_bytes, commit,
                                  as_stream(stream));
    });
}

extern "C" sa_status sa_append_decode_partials(sa_kvcache* c, int layer, const float* part, int n_part,
                                               int n_seq, const int32_t* seq_ids, int n_q_heads,
                                               const float* q_norm_w, const float* k_norm_w, float eps,
                                               const float* rope_cos, const float* rope_sin, int rope_max_pos,
                                               float scale, float* out, float* q_out, void* ws, size_t ws_bytes,
                                               int commit, sa_stream_t stream) {
    clear_error();
    return no_throw([&] {
        return append_decode_partials(c, layer, part, n_part, n_seq, seq_ids, n_q_heads, q_norm_w, k_norm_w, eps,
                                      rope_cos, rope_sin, rope_max_pos, scale, out, q_out, ws, ws_bytes, commit,
                                      as_stream(stream));
    });
}

extern "C" sa_status sa_kvcache_gather(const sa_kvcache* c, int layer, int seq, int len, float* k_out,
                                       float* v_out, sa_stream_t stream) {
    clear_error();
    if (!valid_cache(c)) return fail(SA_EINVAL, "invalid cache");
    if (layer < 0 || layer >= c->desc.num_layers) return fail(SA_ERANGE, "Layer index out of range");
    if (seq < 0 || seq >= c->desc.max_seqs) return fail(SA_ERANGE, "sequence index out of range");
    if (len < 0 || len > c->pt.len(seq)) return fail(SA_ERANGE, "Requested seq_len exceeds cached length");
    if (len == 0) return SA_OK;
    if (!k_out && !v_out) return fail(SA_EINVAL, "null outputs");
    const int32_t* row = c->d_table + (size_t)seq * c->desc.max_pages_per_seq;
    hipStream_t st = as_stream(stream);
    const PagedView pv = view_of(c, layer);
    const bool vec = aligned16(k_out) && aligned16(v_out);   // pools are
    const int per_row = c->desc.head_dim / (vec ? 4 : 1), step = tokens_per_launch(1, per_row);
    auto launch = [&](auto kernel) {
        for (int t0 = 0; t0 < len; t0 += step) {
            const int t1 = std::min(len - t0, step) + t0;
            const dim3 grid((unsigned)(((long long)(t1 - t0) * per_row + 255) / 256), c->desc.num_kv_heads, 2);
            hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, k_pool_of(c, layer), v_pool_of(c, layer), pv.k_scale,
                               pv.v_scale, row, c->desc.num_kv_heads, c->desc.head_dim, t0, t1, len, k_out, v_out);
        }
    };
    switch (c->desc.kv_dtype) {
        case SA_DTYPE_FP8: vec ? launch(gather_kernel<SA_DTYPE_FP8, 4>) : launch(gather_kernel<SA_DTYPE_FP8, 1>); break;
        case SA_DTYPE_BF16: vec ? launch(gather_kernel<SA_DTYPE_BF16, 4>) : launch(gather_kernel<SA_DTYPE_BF16, 1>); break;
        default: vec ? launch(gather_kernel<SA_DTYPE_F32, 4>) : launch(gather_kernel<SA_DTYPE_F32, 1>);
    }
    SA_CHECK_LAUNCH();
    return SA_OK;
}

extern "C" sa_status sa_qk_norm_rope_ex(const float* x, int n_rows, int D, const int32_t* pos,
                                        const float* norm_w, float eps, sa_norm_mode mode,
                                        const float* rope_cos, const float* rope_sin, int rope_max_pos,
                                        float* y, sa_stream_t stream) {
    clear_error();
    if (!x || !y) return fail(SA_EINVAL, "null pointer");
    if (n_rows < 0) return fail(SA_EINVAL, "n_rows must be >= 0");
    if (mode != SA_NORM_EPS_INSIDE && mode != SA_NORM_EPS_OUTSIDE) return fail(SA_EINVAL, "unknown norm mode");
    if ((rope_cos == nullptr) != (rope_sin == nullptr)) return fail(SA_EINVAL, "cos and sin go together");
    if (rope_cos && !pos) return fail(SA_EINVAL, "RoPE needs positions");
    if (n_rows == 0) return SA_OK;
    hipStream_t st = as_stream(stream);
    const dim3 grid((n_rows + 3) / 4);
    const bool outside = mode == SA_NORM_EPS_OUTSIDE;
    switch (D) {
#define SA_NORM_ROPE_CASE(DD)                                                                          \
    case DD:                                                                                           \
        hipLaunchKernelGGL(qk_norm_rope_kernel<DD>, grid, dim3(256), 0, st, x, n_rows, pos, norm_w, eps, \
                           outside, rope_cos, rope_sin, rope_max_pos, y);                              \
        break;
        SA_NORM_ROPE_CASE(8)
        SA_NORM_ROPE_CASE(16)
        SA_NORM_ROPE_CASE(32)
        SA_NORM_ROPE_CASE(64)
        SA_NORM_ROPE_CASE(128)
        SA_NORM_ROPE_CASE(256)
#undef SA_NORM_ROPE_CASE
        default:
            return fail(SA_EINVAL, "head_dim must be 8, 16, 32, 64, 128 or 256");
    }
    SA_CHECK_LAUNCH();
    return SA_OK;
}

extern "C" sa_status sa_qk_norm_rope(const float* x, int n_rows, int D, const int32_t* pos,
                                     const float* norm_w, float eps, const float* rope_cos,
                                     const float* rope_sin, int rope_max_pos, float* y,
                                     sa_stream_t stream) {
    return sa_qk_norm_rope_ex(x, n_rows, D, pos, norm_w, eps, SA_NORM_EPS_INSIDE, rope_cos, rope_sin,
                              rope_max_pos, y, stream);
}
