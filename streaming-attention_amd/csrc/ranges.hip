// Attention of single tokens, and of few new tokens in a row, over ranges of a paged
// cache, on bf16 MFMA.
//
// A row (sequence) of a launch sees the tokens of up to two sources: its
// group's (a prefix whose pages several rows list, read once for all of them)
// and its own (the tokens behind the prefix, or the sinks and the window of a
// windowed decode).  A source's tokens are cut into chunks; one workgroup
// takes a chunk of one KV head for all query rows of the source (rows of the
// group x query heads of the KV head, up to Geo::ROWS at a time) and leaves a
// partial (m, l, O) per query row; a second launch joins a row's partials,
// O = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c.  A row with one partial
// is written by the first launch, and a launch of such rows has no second.
//
// Arithmetic: fp32 throughout.  q (scaled by scale * log2 e) and the softmax
// weights enter the products as the exact sum of three bf16 terms; cached bf16
// values are one term, cached fp32 ones three, split where they are used.  Of
// the products of three by three terms the six largest are taken: what is left
// out is below 2^-24 of the product, the rounding of an fp32 one.  fp32 values
// that only one tile of 16 query rows uses are not split: fp32 MFMA takes them as
// they are (4 searches of 4 beams behind 1500 - 2100 tokens 19.4 us against 19.8).
// A chunk's row whose sums are not finite is computed anew without terms
// (plain_row.h), so that infinities and values near fp32's limit come out as in
// the paged decode that does not split.
//
// An 8-bit cache's codes are one bf16 term each, 2^e times the code: widened with their
// row's scale on the way from LDS into registers, exactly (K read as rows, V
// transposed as bytes, ds_read_tr8_b64).
//
// Chunks of new tokens (at most some dozen query rows each; extend.hip takes longer ones):
// the query rows of a source are then the new tokens x query heads of the KV head,
// and a token's own place is its mask's last key, so only tiles at the end are masked.
//
// Layout: v_mfma_f32_16x16x32_bf16 with S^T = K Q^T (rows: keys, columns: query
// rows), so that a lane's eight scores of a 32-key tile are the operand that
// O^T += V^T P^T takes.  Four waves: RG of them take 16 RT query
// rows each (RT 1, fp32 also 2), and KG = 4 / RG groups of RG waves take every KG-th tile of the chunk.
//   RG = 1 (up to 16 RT rows): a wave reads its own tiles and never waits for
//     another; the next tile's K load into LDS while P V is computed, the next
//     tile's V while the scores are.
//   RG > 1: the waves of a key group share its tiles, a ring of RG of them.
//
// Bound, 16 / 8 heads of 128: HBM for many rows (64 rows, window 4096 and 4 sinks,
// bf16: 992 MB in 157 us, 6.3 TB/s); the products and the softmax between for many
// rows behind one prefix (64 behind 32768 tokens, bf16: 75 us, MFMA 42 % and VALU
// 45 % busy; loads alone 55, computing alone 66, of both 15 for launches, queries
// and partials); the latency of the tiles for few rows (4 x 4 beams, fp32: 19.4 us,
// 2.65 per tile of a wave; 4 rows behind 512 tokens, bf16: 9.0).  Over 8 bits 64 rows of
// 512 - 32768 tokens, 2.12 GB, take 341 us (6.2 TB/s; MFMA 31 % and VALU 52 % busy), one row
// of 5000 14.1; chunks of 5 tokens of each of 64 sequences of 512 - 16384, bf16, 2.18 GB, 363
// (6.0 TB/s), 5 tokens behind 1000, fp32, 12.6 - 13.4 (9.2 and 4.4 alone under the kernel
// tracer: arguments, table, page ids to LDS and a barrier, K, scores, V, a reduction
// across the waves, each waiting for the one before it; then the joining launch).
#include "ranges.h"

#include <algorithm>
#include <type_traits>
#include <utility>
#include <vector>

#include "bf16_terms.h"
#include "plain_row.h"
#include "prefill_shared.h"

namespace sa {
namespace {

using pf::lds_s16x4_t;
using pf::lds_u8_t;
using pf::s16x4_t;
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef int s32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s32x2_t lds_s32x2_t;

constexpr int kTile = 32;                    // keys per tile; divides a page
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kMaxChunks = 64;               // chunks of one source
constexpr int kChunkTiles = 1024;            // tiles of one chunk, whose page ids sit in LDS
constexpr int kSources = 2 * kRowsPerLaunch;
constexpr float kRaiseAt = 65536.f;          // a lane's sum of weights that raises the running max

// What every launch over a cache has.
struct CacheArgs {
    const void* q;           // [rows][n_q][D], fp32 or (chunks of tokens) bf16
    const void* k;           // pool [pages][n_kv][64][D]
    const void* v;
    const uint8_t* k_scale;  // 8 bits: [pages][n_kv][64]
    const uint8_t* v_scale;
    const int32_t* table;    // [max_seqs][max_pages]
    void* out;               // like q
    float* part_o;           // [partial rows][n_kv][D]
    float* part_ml;          // [partial rows][n_kv][2]
    int n_kv, n_q, rep, max_pages, num_pages;
    uint32_t rep_inv;                        // ceil(2^20 / rep): j / rep = j rep_inv >> 20 for query rows j
    float sl2;                               // scale * log2(e)
};

struct RangeArgs : CacheArgs {
    int n_groups, n_rows;
    int row_block;                           // query rows of a workgroup
    int chunk_group, chunk_own;              // tiles
    uint64_t single;                         // rows with one partial, which is the output
    // Sources 0 .. n_groups - 1 are the groups', n_groups + i is row i's own.
    RangeSource src[kSources];
    int32_t start[kSources + 1];             // a source's first workgroup in the grid
    int32_t base[kSources];                  // its first partial row
    // 32-bit, as every array here: for a byte array and a dword array indexed
    // alike, the compiler split a scalar address into parts that are no
    // multiples of 4, whose low bits the scalar load drops.
    int32_t first[kRowsPerLaunch + 1];       // a group's first row; first[n_groups] = n_rows
    int32_t group_of[kRowsPerLaunch];        // a row's group
};
static_assert(sizeof(RangeArgs) <= 4096, "kernel arguments");
static_assert(kRowsPerLaunch <= 64, "a bit of `single` per row");

// The tiles of a source: those of [0, a1), then those of [b0, b1).
__host__ __device__ inline int tiles_a(const RangeSource& s) { return (s.a1 + kTile - 1) / kTile; }
__host__ __device__ inline int tiles_of(const RangeSource& s) {
    return tiles_a(s) + (s.b1 > s.b0 ? (s.b1 - 1) / kTile - s.b0 / kTile + 1 : 0);
}
struct TileSpan {
    int t0, lo, hi;   // the tile's first token, and the tokens of it that the source has
};
__device__ __forceinline__ TileSpan tile_span(const RangeSource& s, int u) {
    const int na = tiles_a(s);
    TileSpan r;
    if (u < na) {
        r.t0 = u * kTile;
        r.lo = r.t0;
        r.hi = min(r.t0 + kTile, s.a1);
    } else {
        r.t0 = (s.b0 / kTile + u - na) * kTile;
        r.lo = max(r.t0, s.b0);
        r.hi = min(r.t0 + kTile, s.b1);
    }
    return r;
}

// The cached values' type, as the cache's sa_dtype.
constexpr int kF32 = SA_DTYPE_F32, kBf16 = SA_DTYPE_BF16, kFp8 = SA_DTYPE_FP8;

template <int D, int KV>
struct Geo {
    static constexpr bool BF16 = KV == kBf16, FP8 = KV == kFp8;
    static constexpr int ROWB = D * (FP8 ? 1 : BF16 ? 2 : 4);   // bytes of one key's row
    static constexpr int HALF = kTile * ROWB;         // K or V of a tile
    static constexpr int SCALES = 2 * kTile;          // 8 bits: bytes of the tile's scales, K's, then V's
    static constexpr int TILEB = 2 * HALF + (FP8 ? SCALES : 0);
    static constexpr int MORE = FP8 ? 1 : 0;          // wave loads of the scales
    static constexpr int CPR = ROWB / 16;             // 16-byte chunks of a row
    static constexpr int RPL = kWave / CPR;           // rows per wave load
    static constexpr int NL = kTile / RPL;            // wave loads per half
    static constexpr int KS = D / 32, DB = D / 16;
    static constexpr int NT = KV == kF32 ? kTerms : 1;   // terms of a cached value
    static constexpr int RT = KV == kF32 ? 2 : 1;     // most tiles of 16 query rows of a wave
    static constexpr int ROWS = kWaves * RT * 16;     // query rows of a workgroup
    // LDS: one tile per wave, or the partials of the waves' query rows at the end.
    static constexpr int LDS = kWaves * (TILEB > 16 * RT * D * 4 ? TILEB : 16 * RT * D * 4);

    // Chunk c of row r sits at chunk c ^ swz(r) of the row: the 16 rows 8a + 4kb
    // + b (a, b < 4) of a K fragment read, and the rows of a V^T read (bf16: 8g
    // + 4u + b with b < 4 and g of one half wave; fp32: 8g + e, g < 4), fall on
    // different banks; for fp32 products (F32) 16 neighbouring rows, and 4g + e.
    // 8 bits: the 16 rows of a K fragment read as above (16 codes a lane), rows 8g + s / 2
    // (s < 16, 8 codes a lane) of a V^T read.
    template <bool F32>
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (F32) return r & 15;
        else if constexpr (FP8) return (CPR == 8 ? ((r >> 1) & 1) << 2 : 0) | (((r >> 4) ^ (r >> 2)) & 1) << 1 | ((r >> 3) & 1);
        else if constexpr (!BF16) return (((r >> 3) & 3) << 2) | (r & 3);
        else if constexpr (CPR == 16) return ((r & 3) << 2) | (((r >> 3) & 1) << 1) | ((r >> 4) & 1);
        else return (((r >> 1) & 1) << 2) | (((r >> 3) & 1) << 1) | ((r >> 4) & 1);
    }
    template <bool F32>
    static __device__ __forceinline__ int off(int r, int c) { return r * ROWB + ((c ^ swz<F32>(r)) << 4); }
};

__device__ __forceinline__ f32x4_t lds_f4(const lds_u8_t* p) {
    return *reinterpret_cast<const __attribute__((address_space(3))) f32x4_t*>(p);
}

// pf::dma16 for data that is read once: non-temporal.
__device__ __forceinline__ void dma16_nt(const void* g, lds_u8_t* dst) {
    const uint32_t m = static_cast<uint32_t>(reinterpret_cast<size_t>(dst));
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt" ::"v"(g), "s"(m) : "memory", "m0");
}

// The same of 4 bytes per lane.
__device__ __forceinline__ void dma4_nt(const void* g, lds_u8_t* dst) {
    const uint32_t m = static_cast<uint32_t>(reinterpret_cast<size_t>(dst));
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off nt" ::"v"(g), "s"(m) : "memory", "m0");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ float row_sum(float v) { return group_reduce<OpSum, 16, kWave>(v); }
__device__ __forceinline__ float row_max(float v) { return group_reduce<OpMax, 16, kWave>(v); }

// The state of one wave: 16 RT query rows, lane (g = lane / 16, r16 = lane %
// 16) holds row r16 of each tile of 16.
template <int D, int KV, int RT>
struct WaveState {
    using G = Geo<D, KV>;
    static constexpr bool BF16 = G::BF16, FP8 = G::FP8;
    static constexpr int PAIRS = KV == kF32 ? 6 : 3;
    // fp32 values whose split into terms would serve one tile of query rows only:
    // v_mfma_f32_16x16x4_f32 instead.
    static constexpr bool F32 = KV == kF32 && RT == 1;
    static __device__ __forceinline__ int off(int r, int c) { return G::template off<F32>(r, c); }
    // Terms of the cached and of the other operand of a product, largest first.
    static constexpr int pair_a(int pr) { return KV != kF32 ? 0 : (pr == 2 || pr == 4 ? 1 : pr == 5 ? 2 : 0); }
    static constexpr int pair_b(int pr) { return KV != kF32 ? pr : (pr == 1 || pr == 4 ? 1 : pr == 3 ? 2 : 0); }

    bf16x8_t q[RT][G::KS][kTerms];
    f32x4_t qf[D / 16], pf[2];   // F32: q from D / 4 g on, the weights
    f32x4_t acc[RT][G::DB];
    float m[RT];     // running max (log2 domain) at the last raise
    float b[RT];     // -m once finite: the score chain's start
    float l[RT];     // this lane's part of the sum of weights
    float cap[RT];   // kRaiseAt once m is finite: the first tile always raises
    bf16x8_t p[RT][kTerms];
    int g, r16;

    __device__ __forceinline__ void init(int lane) {
        g = lane >> 4;
        r16 = lane & 15;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
            for (int db = 0; db < G::DB; ++db) acc[rt][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
            m[rt] = -INFINITY;
            b[rt] = 0.f;
            l[rt] = 0.f;
            cap[rt] = -1.f;
        }
    }
    // 8 bits: a lane reads 16 codes of a key at once, which two products take, so
    // product ks multiplies d = 64 (ks / 2) + 16 g + 8 (ks % 2) ...
    template <class T>
    __device__ __forceinline__ void load_q(int rt, const T* row, float sl2) {
        if constexpr (sizeof(T) == 2) {
            static_assert(!F32, "bf16 queries of fp32 caches");
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                const int d = FP8 ? 64 * (ks / 2) + 16 * g + 8 * (ks % 2) : 32 * ks + 8 * g;
                const u32x4_t x = *reinterpret_cast<const u32x4_t*>(row + d);
                split_terms(f32x4_t{bf16_lo(x[0]), bf16_hi(x[0]), bf16_lo(x[1]), bf16_hi(x[1])} * sl2,
                            f32x4_t{bf16_lo(x[2]), bf16_hi(x[2]), bf16_lo(x[3]), bf16_hi(x[3])} * sl2, q[rt][ks]);
            }
            return;
        } else {
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) qf[i] = *reinterpret_cast<const f32x4_t*>(row + D / 4 * g + 4 * i) * sl2;
            return;
        }
        f32x4_t x[G::KS][2];
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = FP8 ? 64 * (ks / 2) + 16 * g + 8 * (ks % 2) : 32 * ks + 8 * g;
                x[ks][i] = *reinterpret_cast<const f32x4_t*>(row + d + 4 * i);
            }
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks) split_terms(x[ks][0] * sl2, x[ks][1] * sl2, q[rt][ks]);
        }
    }

    // Scores of the tile whose K sits at kb, masked to its tokens [lo, hi) and, in a
    // chunk (CAUSAL), to those before limit[rt], and
    // the weights p = 2^(s - m) as three bf16 terms.  Element 4 h + e of a lane
    // is key 8 g + 4 h + e (F32: 16 h + 4 g + e, the operand of V^T P^T as it is;
    // the products take d in the order that lets a lane read 16 bytes of K).
    template <bool CAUSAL>
    __device__ __forceinline__ void scores(const lds_u8_t* kb, const TileSpan& sp, const int (&limit)[RT], int first_limit) {
        float vs[8];   // 8 bits: the scales of V's rows, which the weights take
        if constexpr (FP8) {
            const u32x2_t b = *reinterpret_cast<const __attribute__((address_space(3))) u32x2_t*>(kb + 2 * G::HALF + kTile + 8 * g);
#pragma unroll
            for (int j = 0; j < 8; ++j) vs[j] = scale_of(b[j >> 2] >> (8 * (j & 3)) & 255u);
        }
        f32x4_t s[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) s[rt][0] = s[rt][1] = f32x4_t{b[rt], b[rt], b[rt], b[rt]};
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                f32x4_t kf[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) kf[h] = lds_f4(kb + off(16 * h + r16, D / 16 * g + i));
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        s[0][h] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[h][e], qf[i][e], s[0][h], 0, 0, 0);
            }
        }
#pragma unroll
        for (int ks = 0; ks < (F32 ? 0 : G::KS); ++ks) {
            bf16x8_t kf[2][G::NT];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = 8 * (r16 >> 2) + 4 * h + (r16 & 3);
                if constexpr (FP8) {
                    const u32x4_t x = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(
                        kb + off(r, 4 * (ks / 2) + g));
                    kf[h][0] = codes_bf16x8(x[2 * (ks & 1)], x[2 * (ks & 1) + 1], scale_of(kb[2 * G::HALF + r]));
                } else if constexpr (BF16) {
                    kf[h][0] = *reinterpret_cast<const __attribute__((address_space(3))) bf16x8_t*>(
                        kb + off(r, 4 * ks + g));
                } else {
                    split_terms(lds_f4(kb + off(r, 8 * ks + 2 * g)), lds_f4(kb + off(r, 8 * ks + 2 * g + 1)),
                                kf[h]);
                }
            }
#pragma unroll
            for (int pr = 0; pr < PAIRS; ++pr)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        s[rt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[h][pair_a(pr)], q[rt][ks][pair_b(pr)],
                                                                           s[rt][h], 0, 0, 0);
        }
        const bool ragged = sp.hi - sp.lo < kTile || (CAUSAL && sp.hi > first_limit);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (ragged) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int t = sp.t0 + (F32 ? 16 * (j >> 2) + 4 * g + (j & 3) : 8 * g + j);
                    if (t < sp.lo || t >= sp.hi || (CAUSAL && t >= limit[rt])) s[rt][j >> 2][j & 3] = -INFINITY;
                    if (FP8 && (t < sp.lo || t >= sp.hi)) vs[j] = 0.f;   // a byte that no row has written
                }
            }
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(s[rt][j >> 2][j & 3]);
            float sum = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
            if (__any(!(sum <= cap[rt]))) {
                float mt = s[rt][0][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) mt = fmaxf(mt, s[rt][j >> 2][j & 3]);
                const float m_new = fmaxf(m[rt], row_max(mt) - b[rt]);
                const float alpha = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - m_new);
#pragma unroll
                for (int db = 0; db < G::DB; ++db) acc[rt][db] *= alpha;
                l[rt] *= alpha;
                const float b_new = m_new == -INFINITY ? 0.f : -m_new;
                const float delta = b_new - b[rt];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __builtin_amdgcn_exp2f(s[rt][j >> 2][j & 3] + delta);
                sum = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                m[rt] = m_new;
                b[rt] = b_new;
                cap[rt] = m_new == -INFINITY ? -1.f : kRaiseAt;
            }
            l[rt] += sum;
            if constexpr (FP8)
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] *= vs[j];
            pf[0] = f32x4_t{w[0], w[1], w[2], w[3]};
            pf[1] = f32x4_t{w[4], w[5], w[6], w[7]};
            if constexpr (!F32) split_terms(pf[0], pf[1], p[rt]);
        }
    }

    // O^T += V^T P^T for the tile whose V sits at vb.
    __device__ __forceinline__ void weigh(const lds_u8_t* vb) {
        // ND d blocks at a time: consecutive MFMAs do not wait for each other
        constexpr int ND = 2;
#pragma unroll
        for (int d0 = 0; d0 < G::DB; d0 += ND) {
            if constexpr (F32) {
                float x[ND][8];
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        x[d][j] = *reinterpret_cast<const __attribute__((address_space(3))) float*>(
                            vb + off(16 * (j >> 2) + 4 * g + (j & 3), 4 * (d0 + d) + (r16 >> 2)) + (r16 & 3) * 4);
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        acc[0][d0 + d] =
                            __builtin_amdgcn_mfma_f32_16x16x4f32(x[d][j], pf[j >> 2][j & 3], acc[0][d0 + d], 0, 0, 0);
                continue;
            }
            bf16x8_t vf[ND][G::NT];
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                if constexpr (FP8) {
                    // Lane s of a group of 16 reads row 8 g + s / 2, columns 16 db + 8 (s %
                    // 2) ..; lane r16 receives the codes V[8 g + e][16 db + r16].
                    const s32x2_t x = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                        (lds_s32x2_t*)(vb + off(8 * g + (r16 >> 1), d0 + d) + (r16 & 1) * 8));
                    vf[d][0] = codes_bf16x8(x[0], x[1], 1.f);
                } else if constexpr (BF16) {
                    // Lane s of a group of 16 reads row 8 g + 4 u + s / 4, columns
                    // 16 db + 4 (s % 4) ..; lane r16 receives V[8 g + 4 u + e][16 db + r16].
                    const int c = 2 * (d0 + d) + ((r16 & 3) >> 1), h8 = (r16 & 1) * 8;
                    const int r = 8 * g + (r16 >> 2);
                    const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vb + off(r, c) + h8));
                    const s16x4_t y =
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vb + off(r + 4, c) + h8));
                    vf[d][0] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
                } else {
                    f32x4_t x[2];
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        x[j >> 2][j & 3] = *reinterpret_cast<const __attribute__((address_space(3))) float*>(
                            vb + off(8 * g + j, 4 * (d0 + d) + (r16 >> 2)) + (r16 & 3) * 4);
                    split_terms(x[0], x[1], vf[d]);
                }
            }
#pragma unroll
            for (int pr = 0; pr < PAIRS; ++pr)
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        acc[rt][d0 + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            vf[d][pair_a(pr)], p[rt][pair_b(pr)], acc[rt][d0 + d], 0, 0, 0);
        }
    }
};

// A workgroup's place in the launch.
struct Item {
    RangeSource src;
    int kvh;
    int u0, u1;        // its tiles of the source
    int row0, rows;    // the source's first row of the launch, and its query rows
    int q0, q1;        // the workgroup's query rows of those
    int part0;         // the chunk's first partial row
    uint64_t single;   // RangeArgs::single from row0 on
    int limit0;        // a chunk of new tokens: row r sees tokens before limit0 + r
};

// Query row j of an item: row row0 + j / rep of the launch, head j % rep of the
// KV head.  j <= 64 rep and rep <= 64, so j rep < 2^20 and the product's quotient
// is exact.
static_assert(kRowsPerLaunch * kRangesMaxRep * kRangesMaxRep < (1 << 20), "query rows divided by a product");
__device__ __forceinline__ int row_of(const CacheArgs& a, int j) { return (int)(((uint32_t)j * a.rep_inv) >> 20); }

__device__ __forceinline__ int group_chunks(const RangeArgs& a, int g) {
    const int rows = (a.first[g + 1] - a.first[g]) * a.rep;
    return (a.start[g + 1] - a.start[g]) / ((rows + a.row_block - 1) / a.row_block);
}
__device__ __forceinline__ int own_chunks(const RangeArgs& a, int row) {
    return a.start[a.n_groups + row + 1] - a.start[a.n_groups + row];
}

// O (unnormalised), m and l of query row j of an item: the output itself if it
// is the row's only partial.  c: float4 column.
template <int D, class T>
__device__ __forceinline__ void put(const CacheArgs& a, const Item& it, int j, int c, f32x4_t o, float m, float l) {
    const int r = row_of(a, j);
    if (it.single >> r & 1) {
        const int head = it.kvh * a.rep + j - r * a.rep;
        store4(static_cast<T*>(a.out) + ((size_t)(it.row0 + r) * a.n_q + head) * D + 4 * c, o * (1.0f / l));
        return;
    }
    const size_t at = (size_t)(it.part0 + j) * a.n_kv + it.kvh;
    *reinterpret_cast<f32x4_t*>(a.part_o + at * D + 4 * c) = o;
    if (c == 0) *reinterpret_cast<f32x2_t*>(a.part_ml + at * 2) = f32x2_t{m, l};
}

// Returns the query rows, from it.q0 (RG = 4: the wave's first) on a bit each, that
// the wave has to compute anew: their sums are not finite and nothing was put.
// T: the queries' and the output's type; CAUSAL: the rows are a chunk of new tokens.
template <int D, int KV, int RG, int RT, class T, bool CAUSAL>
__device__ __forceinline__ uint64_t attend(const CacheArgs& a, const Item& it, lds_u8_t* smem, const int32_t* pages,
                                       float (*ml)[2]) {
    using G = Geo<D, KV>;
    constexpr int KG = kWaves / RG;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int kg = wave / RG, rg = wave % RG;
    const int q_base = it.q0 + rg * 16 * RT;

    WaveState<D, KV, RT> w;
    w.init(lane);
    int limit[RT];
    const int first_limit = CAUSAL ? it.limit0 + row_of(a, it.q0) : 0;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
        limit[rt] = CAUSAL ? it.limit0 + row_of(a, min(q_base + 16 * rt + w.r16, it.q1 - 1)) : 0;

    // Wave loads [first, first + N) of the 2 NL of tile u (K's, then V's) into the
    // tile at dst.  Rows outside the source's tokens read the nearest one inside.
    auto load = [&](int u, lds_u8_t* dst, int first, auto n_c) {
        const TileSpan sp = tile_span(it.src, u);
        const size_t at = (((size_t)pages[u - it.u0] * a.n_kv + it.kvh) * SA_PAGE_TOKENS) * G::ROWB;
#pragma unroll
        for (int i = 0; i < decltype(n_c)::value; ++i) {
            const bool is_v = first + i >= G::NL;
            const int r = (first + i - (is_v ? G::NL : 0)) * G::RPL + lane / G::CPR;
            const int tok = min(max(sp.t0 + r, sp.lo), sp.hi - 1) & (SA_PAGE_TOKENS - 1);
            const int col = ((lane % G::CPR) ^ G::template swz<decltype(w)::F32>(r)) * 16;
            const char* pool = static_cast<const char*>(is_v ? a.v : a.k);
            dma16_nt(pool + at + (size_t)tok * G::ROWB + col, dst + (first + i) * 1024);
        }
    };
    // 8 bits: the tile's scales, 8 lanes for K's and 8 for V's, behind its V at dst.
    auto load_scales = [&](int u, lds_u8_t* dst) {
        if constexpr (G::FP8) {
            const size_t at = ((size_t)pages[u - it.u0] * a.n_kv + it.kvh) * SA_PAGE_TOKENS +
                              (tile_span(it.src, u).t0 & (SA_PAGE_TOKENS - 1));
            const uint8_t* s = (lane < 8 ? a.k_scale : a.v_scale) + at + 4 * (lane & 7);
            if (lane < 16) dma4_nt(s, dst);
        }
    };
    auto load_queries = [&]() {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int j = min(q_base + 16 * rt + w.r16, it.q1 - 1), r = row_of(a, j);
            w.load_q(rt, static_cast<const T*>(a.q) + ((size_t)(it.row0 + r) * a.n_q + it.kvh * a.rep + j - r * a.rep) * D,
                     a.sl2);
        }
    };

    if constexpr (RG == 1) {
        using Half = std::integral_constant<int, G::NL>;
        lds_u8_t* const kb = smem + wave * G::TILEB;
        lds_u8_t* const vb = kb + G::HALF;
        int u = it.u0 + kg;
        if (u < it.u1) {
            load_scales(u, kb + 2 * G::HALF);
            load(u, kb, 0, Half{});
            load(u, kb, G::NL, Half{});
        }
        load_queries();   // behind the first tile's loads, so that the two latencies are one
        for (; u < it.u1; u += KG) {
            const bool more = u + KG < it.u1;
            wait_loads<G::NL>();                               // K; V may be in flight
            w.template scores<CAUSAL>(kb, tile_span(it.src, u), limit, first_limit);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // K and the scales have been read
            if (more) {
                load_scales(u + KG, kb + 2 * G::HALF);
                load(u + KG, kb, 0, Half{});
                wait_loads<G::NL + G::MORE>();                 // V; the next K may be in flight
            } else {
                wait_loads<0>();
            }
            w.weigh(vb);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (more) load(u + KG, kb, G::NL, Half{});
        }
    } else {
        // RG stages per key group; each wave loads its share of a tile.
        constexpr int MINE = 2 * G::NL / RG;
        static_assert(MINE * RG == 2 * G::NL, "a tile's loads are shared evenly");
        using Mine = std::integral_constant<int, MINE>;
        lds_u8_t* const ring = smem + kg * RG * G::TILEB;
        const int n_all = (it.u1 - it.u0 + KG - 1) / KG;                  // steps of the workgroup
        const int n = it.u0 + kg < it.u1 ? (it.u1 - it.u0 - kg + KG - 1) / KG : 0;   // of this key group
        auto load_tile = [&](int t) {
            lds_u8_t* dst = ring + (t % RG) * G::TILEB;
            load_scales(it.u0 + kg + t * KG, dst + 2 * G::HALF);   // every wave, so that all wait for as many loads
            load(it.u0 + kg + t * KG, dst, rg * MINE, Mine{});
        };
        for (int t = 0; t < RG - 1; ++t)
            if (t < n) load_tile(t);
        load_queries();
        for (int t = 0; t < n_all; ++t) {
            // tiles t .. t + RG - 2 are in flight where the chunk has them
            if (t + RG - 1 <= n) wait_loads<(RG - 2) * (MINE + G::MORE)>();
            else wait_loads<0>();
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (t + RG - 1 < n) load_tile(t + RG - 1);
            if (t < n) {
                const lds_u8_t* kb = ring + (t % RG) * G::TILEB;
                w.template scores<CAUSAL>(kb, tile_span(it.src, it.u0 + kg + t * KG), limit, first_limit);
                w.weigh(kb + G::HALF);
            }
        }
    }

    float l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) l[rt] = row_sum(w.l[rt]);
    uint64_t anew = 0;
    if constexpr (KG == 1) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int j = q_base + 16 * rt + w.r16;
            const bool fine = l[rt] + row_sum(not_finite<G::DB>(w.acc[rt])) < INFINITY;
            anew |= (__ballot(j < it.q1 && !fine) & 0xffff) << (16 * rt);
            if (j < it.q1 && fine) {
#pragma unroll
                for (int db = 0; db < G::DB; ++db) put<D, T>(a, it, j, 4 * db + w.g, w.acc[rt][db], w.m[rt], l[rt]);
            }
        }
    } else {
        // The key groups' partials meet in LDS, over the tiles (all consumed).
        constexpr int ROWS = RG * RT * 16;
        __syncthreads();
        auto* po = reinterpret_cast<__attribute__((address_space(3))) f32x4_t*>(smem);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const int j = (rg * RT + rt) * 16 + w.r16;
#pragma unroll
            for (int db = 0; db < G::DB; ++db) po[(kg * ROWS + j) * (D / 4) + 4 * db + w.g] = w.acc[rt][db];
            if (w.g == 0) {
                ml[kg * ROWS + j][0] = w.m[rt];
                ml[kg * ROWS + j][1] = l[rt];
            }
        }
        __syncthreads();
        constexpr int C = D / 4;
        const int c = lane % C;
        for (int j0 = wave * (kWave / C); j0 < ROWS; j0 += kThreads / C) {   // the wave's rows
            if (it.q0 + j0 >= it.q1) break;
            const int j = j0 + lane / C;
            float M = ml[j][0];
#pragma unroll
            for (int k = 1; k < KG; ++k) M = fmaxf(M, ml[k * ROWS + j][0]);
            f32x4_t o = {0.f, 0.f, 0.f, 0.f};
            float L = 0.f;
#pragma unroll
            for (int k = 0; k < KG; ++k) {
                const float mk = ml[k * ROWS + j][0];
                const float wk = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - M);
                o += po[(k * ROWS + j) * C + c] * wk;
                L += ml[k * ROWS + j][1] * wk;
            }
            const bool mine = it.q0 + j < it.q1;
            const uint64_t bad = __ballot(mine && !(L + not_finite<1>(&o) < INFINITY));
            constexpr uint64_t row = (1ull << C) - 1;
            static_assert(ROWS <= 64, "a bit per row");
            if (mine && !(bad >> (lane / C * C) & row)) put<D, T>(a, it, it.q0 + j, c, o, M, L);
#pragma unroll
            for (int g = 0; g < kWave / C; ++g)
                if (bad >> (g * C) & row) anew |= 1ull << (j0 + g);
        }
    }
    return anew;
}

// Query row j of an item without matrix instructions.
template <int D, int KV, class T, bool CAUSAL>
__device__ __forceinline__ void attend_plain(const CacheArgs& a, const Item& it, const int32_t* pages, int j) {
    using E = std::conditional_t<KV == kFp8, uint8_t, std::conditional_t<KV == kBf16, uint16_t, float>>;
    const int lane = threadIdx.x & (kWave - 1);
    const int r = row_of(a, j), head = it.kvh * a.rep + j - r * a.rep;
    const size_t row = ((size_t)(it.row0 + r) * a.n_q + head) * D;
    PlainRow<D> p;
    for (int u = it.u0; u < it.u1 && !p.lost(); ++u) {
        TileSpan sp = tile_span(it.src, u);
        if (CAUSAL) sp.hi = min(sp.hi, it.limit0 + r);
        if (CAUSAL && sp.hi <= sp.lo) break;
        const size_t key = ((size_t)pages[u - it.u0] * a.n_kv + it.kvh) * SA_PAGE_TOKENS + (sp.lo & (SA_PAGE_TOKENS - 1));
        const size_t at = key * D;
        auto value = [&](const void* pool, int i) { return static_cast<const E*>(pool) + at + (size_t)i * D; };
        auto scale = [&](const uint8_t* s, int i) {
            if constexpr (KV == kFp8) return scale_of(s[key + i]);
            else return 1.f;
        };
        p.keys(sp.hi - sp.lo, static_cast<const T*>(a.q) + row, a.sl2, [&](int i) { return value(a.k, i); },
               [&](int i) { return value(a.v, i); }, [&](int i) { return scale(a.k_scale, i); },
               [&](int i) { return scale(a.v_scale, i); });
    }
    if (it.single >> r & 1) {
#pragma unroll
        for (int e = 0; e < p.E; ++e) {
            const float v = p.o[e] / p.l;
            if constexpr (sizeof(T) == 2) static_cast<T*>(a.out)[row + lane * p.E + e] = f32_to_bf16_rne(v);
            else static_cast<T*>(a.out)[row + lane * p.E + e] = v;
        }
        return;
    }
    const size_t at = (size_t)(it.part0 + j) * a.n_kv + it.kvh;
#pragma unroll
    for (int e = 0; e < p.E; ++e) a.part_o[at * D + lane * p.E + e] = p.o[e];
    if (lane == 0) {
        a.part_ml[at * 2] = p.m;
        a.part_ml[at * 2 + 1] = p.l;
    }
}

// The tiles' pages; an id outside the pool (a table entry that was never set) is
// clamped so that no load can fault.
__device__ __forceinline__ void stage_pages(const CacheArgs& a, const Item& it, int32_t* pages) {
    const int32_t* trow = a.table + (size_t)it.src.cache_row * a.max_pages;
    for (int i = threadIdx.x; i < it.u1 - it.u0; i += kThreads)
        pages[i] = min(max(trow[tile_span(it.src, it.u0 + i).t0 / SA_PAGE_TOKENS], 0), a.num_pages - 1);
    __syncthreads();
}

// An item's query rows by as many waves as they need.
template <int D, int KV, class T, bool CAUSAL>
__device__ __forceinline__ void attend_item(const CacheArgs& a, const Item& it, lds_u8_t* smem, const int32_t* pages,
                                            float (*ml)[2]) {
    const int rows = it.q1 - it.q0;
    uint64_t anew;
    int first = it.q0;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if constexpr (KV != kF32) {
        if (rows <= 16) anew = attend<D, KV, 1, 1, T, CAUSAL>(a, it, smem, pages, ml);
        else if (rows <= 32) anew = attend<D, KV, 2, 1, T, CAUSAL>(a, it, smem, pages, ml);
        else anew = attend<D, KV, 4, 1, T, CAUSAL>(a, it, smem, pages, ml), first += 16 * wave;
    } else {
        if (rows <= 16) anew = attend<D, KV, 1, 1, T, CAUSAL>(a, it, smem, pages, ml);
        else if (rows <= 32) anew = attend<D, KV, 1, 2, T, CAUSAL>(a, it, smem, pages, ml);
        else if (rows <= 64) anew = attend<D, KV, 2, 2, T, CAUSAL>(a, it, smem, pages, ml);
        else anew = attend<D, KV, 4, 2, T, CAUSAL>(a, it, smem, pages, ml), first += 32 * wave;
    }
    for (; anew; anew &= anew - 1) attend_plain<D, KV, T, CAUSAL>(a, it, pages, first + __builtin_ctzll(anew));
}

template <int D, int KV>
__global__ void __launch_bounds__(kThreads, KV == kFp8 ? 3 : 1) range_attn_kernel(RangeArgs a) {
    using G = Geo<D, KV>;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ int32_t pages[kChunkTiles];
    __shared__ float ml[G::ROWS][2];
    lds_u8_t* const smem = (lds_u8_t*)smem_raw;

    // The KV head varies fastest: with 8 of them each XCD has one head's chunks.
    Item it;
    it.kvh = blockIdx.x;
    const int n_src = a.n_groups + a.n_rows;
    // The last source that starts at or before blockIdx.y: every lane looks at
    // one or two of them.
    const int lane = threadIdx.x & (kWave - 1);
    int lo = __popcll(__ballot(lane < n_src && a.start[lane] <= (int)blockIdx.y)) - 1;
    if (n_src > kWave) lo += __popcll(__ballot(lane + kWave < n_src && a.start[lane + kWave] <= (int)blockIdx.y));
    it.src = a.src[lo];
    const bool grouped = lo < a.n_groups;
    it.row0 = grouped ? a.first[lo] : lo - a.n_groups;
    it.rows = (grouped ? a.first[lo + 1] - a.first[lo] : 1) * a.rep;
    const int nb = (it.rows + G::ROWS - 1) / G::ROWS;
    const int local = blockIdx.y - a.start[lo];
    const int chunk = local / nb, tiles = grouped ? a.chunk_group : a.chunk_own;
    it.u0 = chunk * tiles;
    it.u1 = min(it.u0 + tiles, tiles_of(it.src));
    it.q0 = (local % nb) * G::ROWS;
    it.q1 = min(it.q0 + G::ROWS, it.rows);
    it.part0 = a.base[lo] + chunk * it.rows;
    it.single = a.single >> it.row0;

    it.limit0 = 0;
    stage_pages(a, it, pages);
    attend_item<D, KV, float, false>(a, it, smem, pages, ml);
}

// Joins the partials of row blockIdx.y's query head blockIdx.x: thread (s, c)
// takes float4 column c of every S-th partial.  A row with none is zero.
template <int D>
__global__ void __launch_bounds__(256) range_merge_kernel(RangeArgs a) {
    constexpr int C = D / 4, S = 256 / C;
    const int head = blockIdx.x, row = blockIdx.y;
    if (a.single >> row & 1) return;
    const int kvh = head / a.rep;
    const int no = own_chunks(a, row);
    int ng = 0, gbase = 0, grows = 0, gj = 0;
    if (a.n_groups) {
        const int g = a.group_of[row];
        ng = group_chunks(a, g);
        grows = (a.first[g + 1] - a.first[g]) * a.rep;
        gj = (row - a.first[g]) * a.rep + head % a.rep;
        gbase = a.base[g];
    }
    const int n = ng + no;
    const int c = threadIdx.x % C, s = threadIdx.x / C;
    const int obase = a.base[a.n_groups + row];
    float M = -INFINITY, L = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    for (int i = s; i < n; i += S) {
        const int pr = i < ng ? gbase + i * grows + gj : obase + (i - ng) * a.rep + head % a.rep;
        const size_t at = (size_t)pr * a.n_kv + kvh;
        const f32x2_t ml = *reinterpret_cast<const f32x2_t*>(a.part_ml + at * 2);
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part_o + at * D + 4 * c);
        const float m_new = fmaxf(M, ml[0]);
        const float w0 = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - m_new);
        const float w1 = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - m_new);
        o = o * w0 + x * w1;
        L = L * w0 + ml[1] * w1;
        M = m_new;
    }
    __shared__ f32x4_t so[S][C];
    __shared__ float sm[S][2];
    so[s][c] = o;
    if (c == 0) {
        sm[s][0] = M;
        sm[s][1] = L;
    }
    __syncthreads();
    if (s) return;
    float all = sm[0][0];
#pragma unroll
    for (int k = 1; k < S; ++k) all = fmaxf(all, sm[k][0]);
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
    L = 0.f;
#pragma unroll
    for (int k = 0; k < S; ++k) {
        const float wk = sm[k][0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[k][0] - all);
        o += so[k][c] * wk;
        L += sm[k][1] * wk;
    }
    float* dst = static_cast<float*>(a.out) + ((size_t)row * a.n_q + head) * D + 4 * c;
    *reinterpret_cast<f32x4_t*>(dst) = n ? o * (1.0f / L) : f32x4_t{0.f, 0.f, 0.f, 0.f};
}

template <int D, int KV>
sa_status launch(const RangeArgs& a, bool merge, hipStream_t st) {
    const int n_src = a.n_groups + a.n_rows;
    if (a.start[n_src] > 0) {
        constexpr int lds = Geo<D, KV>::LDS;
        constexpr auto kernel = range_attn_kernel<D, KV>;
        SA_TRY(pf::opt_in_lds<kernel>(lds));
        hipLaunchKernelGGL(kernel, dim3(a.n_kv, a.start[n_src]), dim3(kThreads), lds, st, a);
        SA_CHECK_LAUNCH();
    }
    if (merge) {
        hipLaunchKernelGGL((range_merge_kernel<D>), dim3(a.n_q, a.n_rows), dim3(256), 0, st, a);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}

int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// Tiles per chunk: the shortest chunk whose workgroups are about one round (2
// per CU in bf16, 1 in fp32; the groups' sources half a round at least, what the
// rows' own leave otherwise), since a workgroup costs 5 us besides its tiles (16
// rows in 4 groups behind 1500 - 2100 tokens, fp32: 12 tiles 20.3, 8 25.7, 4 30.8
// us), and kLongChunk where that would be longer (64 rows of 4100 tokens, bf16: 16
// tiles 158.3, 24 155.3, 32 156.2, 64 158.6, one round 174 us; 64 rows behind 32768
// shared tokens: 16 tiles 82, 24 76, 32 74, 48 75 us).
// A launch without groups whose rows have few tiles gives each row one chunk,
// which saves the second launch: up to four tiles per wave (7 rows of 403 tokens,
// bf16, d = 64: 6.7 against 7.8 us in four chunks; 16 query rows of 512 tokens,
// d = 128: a second, third and fourth tile per wave cost 0.8, 1.7 and 2.7 us, the
// second launch 3.5), in fp32 two (a tile per wave costs 2.65 us).
// Tiles of an 8-bit cache are half as long: kLongChunk8 (64 rows of 512 - 32768 tokens:
// 32 tiles 352 us, 48 343, 64 340), and so are the longest of chunks of new tokens (5 of each
// of 64 sequences of 512 - 16384, bf16: 32 tiles 373 us, 64 368).
constexpr int kLongChunk = 32, kLongChunk8 = 64;
template <class F>
int pick_tiles(long long round, long long work, const F& workgroups, int longest) {
    for (int t = kWaves; t < longest; t += kWaves)
        if (work <= round * t && workgroups(t) <= round) return t;
    return longest;
}

}  // namespace

size_t ranges_ws(int n_rows, int n_q, int d, long long own_tokens, long long group_tokens) {
    if (n_rows <= 0 || n_q <= 0) return 0;
    // Two ranges have at most two partly filled tiles more than their tokens' worth.
    auto chunks = [](long long tokens) -> long long {
        const long long tiles = tokens / kTile + 3;
        return tokens <= 0 ? 0 : std::min<long long>(tiles, std::max(kMaxChunks, ceil_div(tiles, kChunkTiles)));
    };
    const long long per_row = chunks(own_tokens) + chunks(group_tokens);
    return (size_t)(std::min(n_rows, kRowsPerLaunch) * per_row) * n_q * (d + 2) * sizeof(float);
}

namespace {

void set_cache(CacheArgs& a, const PagedView& c, int n_q, float scale) {
    a.k = c.k_pool; a.v = c.v_pool; a.k_scale = c.k_scale; a.v_scale = c.v_scale; a.table = c.block_table;
    a.n_kv = c.n_kv; a.n_q = n_q; a.rep = n_q / c.n_kv;
    a.max_pages = c.max_pages; a.num_pages = c.num_pages;
    a.sl2 = scale * pf::kLog2eP;
    a.rep_inv = ((1u << 20) + a.rep - 1) / a.rep;
}

}  // namespace

sa_status decode_ranges(const PagedView& c, const float* q, int n_q, const RangePlan& plan, float scale, float* out,
                        void* ws, size_t ws_bytes, hipStream_t st) {
    RangeArgs a{};
    set_cache(a, c, n_q, scale);
    const bool f32 = c.kv == SA_DTYPE_F32;
    const int long_chunk = c.kv == SA_DTYPE_FP8 ? kLongChunk8 : kLongChunk;
    a.row_block = f32 ? Geo<128, kF32>::ROWS : Geo<128, kBf16>::ROWS;
    int g = 0, done = 0;   // the group of the launch's first row, and its rows already attended
    for (int i0 = 0; i0 < plan.n_rows; i0 += kRowsPerLaunch) {
        a.n_rows = std::min(kRowsPerLaunch, plan.n_rows - i0);
        a.n_groups = 0;
        if (plan.n_groups) {
            for (int i = 0; i < a.n_rows;) {
                const int n = std::min(plan.group_rows[g] - done, a.n_rows - i);
                a.src[a.n_groups] = plan.group[g];
                a.first[a.n_groups] = i;
                for (int r = i; r < i + n; ++r) a.group_of[r] = a.n_groups;
                ++a.n_groups;
                i += n;
                done += n;
                if (done == plan.group_rows[g]) {
                    ++g;
                    done = 0;
                }
            }
        }
        a.first[a.n_groups] = a.n_rows;
        for (int i = 0; i < a.n_rows; ++i) a.src[a.n_groups + i] = plan.own[i0 + i];

        // Chunks of the sources, at most kMaxChunks each (more only where
        // kChunkTiles asks for it).
        const int n_src = a.n_groups + a.n_rows;
        auto rows_of = [&](int s) { return (s < a.n_groups ? a.first[s + 1] - a.first[s] : 1) * a.rep; };
        auto blocks_of = [&](int s) { return ceil_div(rows_of(s), a.row_block); };
        // Chunks of the sources first .. last - 1 for about `round` workgroups.
        auto pick = [&](int first, int last, long long round, bool whole) {
            int longest = 0;
            long long work = 0;
            for (int s = first; s < last; ++s) {
                longest = std::max(longest, tiles_of(a.src[s]));
                work += (long long)tiles_of(a.src[s]) * blocks_of(s) * a.n_kv;
            }
            auto workgroups = [&](int tiles) {
                long long n = 0;
                for (int s = first; s < last; ++s)
                    n += (long long)ceil_div(tiles_of(a.src[s]), tiles) * blocks_of(s) * a.n_kv;
                return n;
            };
            int chunk = whole && longest <= (f32 ? 2 : 4) * kWaves ? std::max(1, longest)
                                                                      : pick_tiles(round, work, workgroups, long_chunk);
            if (attn_kv_block() > 0) chunk = attn_kv_block() / kTile;
            chunk = std::min(std::max(chunk, ceil_div(longest, kMaxChunks)), kChunkTiles);
            return std::pair<int, long long>(chunk, workgroups(chunk));
        };
        const long long slots = (f32 ? 1LL : c.kv == SA_DTYPE_FP8 ? 3LL : 2LL) * device_cu_count(), round = slots + slots / 4;
        const auto own = pick(a.n_groups, n_src, round, a.n_groups == 0);
        a.chunk_own = own.first;
        a.chunk_group = pick(0, a.n_groups, std::max(round - own.second, round / 2), false).first;
        // Own chunks as long as the groups' end before them, with fewer workgroups (64
        // rows of up to 512 tokens behind 8192 shared ones, bf16: 36.3 us against
        // 39.1; 2 x 4 behind 10000, up to 1000 of their own: 25.8 against 26.2, but
        // 8 x 8 behind 4000 - 8000: 68.3 against 67.1).
        if (a.n_groups) a.chunk_own = std::max(a.chunk_own, a.chunk_group);

        long long parts = 0;
        std::vector<int> chunks(n_src);
        a.start[0] = 0;
        for (int s = 0; s < n_src; ++s) {
            chunks[s] = ceil_div(tiles_of(a.src[s]), s < a.n_groups ? a.chunk_group : a.chunk_own);
            a.base[s] = (int)parts;
            parts += (long long)chunks[s] * rows_of(s);
            a.start[s + 1] = a.start[s] + chunks[s] * blocks_of(s);
        }
        if (a.start[n_src] > 65535) return fail(SA_EINVAL, "too many tokens for one call");   // the grid's y
        a.single = 0;
        for (int i = 0; i < a.n_rows; ++i)
            if (chunks[a.n_groups + i] + (a.n_groups ? chunks[a.group_of[i]] : 0) == 1) a.single |= 1ull << i;
        const bool merge = a.single != (a.n_rows < 64 ? (1ull << a.n_rows) - 1 : ~0ull);
        if (merge) {
            const size_t need = (size_t)parts * a.n_kv * (c.d + 2) * sizeof(float);
            if (need > 0 && (!ws || ws_bytes < need)) return fail(SA_ENOMEM, "workspace too small for the partials");
            a.part_o = static_cast<float*>(ws);
            a.part_ml = a.part_o + (size_t)parts * a.n_kv * c.d;
        }
        a.q = q + (size_t)i0 * n_q * c.d;
        a.out = out + (size_t)i0 * n_q * c.d;
        if (c.d == 64) SA_TRY(c.kv == SA_DTYPE_FP8    ? (launch<64, kFp8>(a, merge, st))
                              : c.kv == SA_DTYPE_BF16 ? (launch<64, kBf16>(a, merge, st))
                                                      : (launch<64, kF32>(a, merge, st)));
        else SA_TRY(c.kv == SA_DTYPE_FP8    ? (launch<128, kFp8>(a, merge, st))
                    : c.kv == SA_DTYPE_BF16 ? (launch<128, kBf16>(a, merge, st))
                                            : (launch<128, kF32>(a, merge, st)));
    }
    return SA_OK;
}

// ---------------------------------------------------------------- chunks of new tokens

namespace {

// Blocks of consecutive tokens of a sequence (as many query rows as a workgroup
// takes) whose keys are cut into chunks of tiles; a workgroup takes a chunk of one
// KV head for a block.
struct ChunkArgs : CacheArgs {
    int n_seq;
    int block;                               // tokens of a block
    int tiles;                               // of a chunk
    ChunkSeq seq[kRowsPerLaunch];
    int32_t start[kRowsPerLaunch + 1];       // a sequence's first item, of blocks x chunks
    int32_t base[kRowsPerLaunch];            // its first partial row
    int32_t chunks[kRowsPerLaunch];          // of its last block
};
static_assert(sizeof(ChunkArgs) <= 4096, "kernel arguments");
static_assert(kRowsPerLaunch <= kWave, "a lane per sequence");

// Tiles that the tokens of block b of a sequence see.
__host__ __device__ inline int block_tiles(const ChunkSeq& s, int b, int block) {
    return (s.len + (s.n < (b + 1) * block ? s.n : (b + 1) * block) - 1) / kTile + 1;
}

template <int D, int KV, class T>
__global__ void __launch_bounds__(kThreads) chunk_attn_kernel(ChunkArgs a) {
    using G = Geo<D, KV>;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    __shared__ int32_t pages[kChunkTiles];
    __shared__ float ml[G::ROWS][2];
    const int lane = threadIdx.x & (kWave - 1);
    const int item = blockIdx.x / a.n_kv;
    // The last sequence that starts at or before the item (those without tokens
    // start where the next one does).
    // One sequence's arguments come with the others, not behind a search.
    ChunkSeq sq = a.seq[0];
    int chunks = a.chunks[0], local = item, base = 0;
    if (a.n_seq > 1) {
        const int i = __popcll(__ballot(lane < a.n_seq && a.start[lane] <= item)) - 1;
        sq = a.seq[i];
        chunks = a.chunks[i];
        local = item - a.start[i];
        base = a.base[i];
    }
    const int b = local / chunks, c = local % chunks;
    Item it;
    it.kvh = blockIdx.x % a.n_kv;
    it.u0 = c * a.tiles;
    it.u1 = min(it.u0 + a.tiles, block_tiles(sq, b, a.block));
    if (it.u0 >= it.u1) return;
    const int t0 = b * a.block, n = min(a.block, sq.n - t0);
    it.src = RangeSource{sq.cache_row, 0, 0, sq.len + t0 + n};
    it.row0 = sq.first + t0;
    it.rows = n * a.rep;
    it.q0 = 0;
    it.q1 = it.rows;
    it.part0 = base + (c * sq.n + t0) * a.rep;
    it.single = chunks == 1 ? ~0ull : 0;
    it.limit0 = sq.len + t0 + 1;
    stage_pages(a, it, pages);
    attend_item<D, KV, T, true>(a, it, (lds_u8_t*)smem_raw, pages, ml);
}

// Joins the partials of (token, head) rows from the launch's first token on, D / 4
// lanes each.
template <int D, class T>
__global__ void __launch_bounds__(256) chunk_merge_kernel(ChunkArgs a, long long row0, long long rows) {
    constexpr int C = D / 4;
    const long long first = row0 + (long long)blockIdx.x * (256 / C), at_row = first + threadIdx.x / C;
    const int i0 = chunk_of(a.seq, a.n_seq, a.seq[0].first + (int)(first / a.n_q));
    if (at_row >= rows) return;
    const int head = (int)(at_row % a.n_q), row = a.seq[0].first + (int)(at_row / a.n_q);
    int i = i0;
    while (i + 1 < a.n_seq && a.seq[i + 1].first <= row) ++i;
    const ChunkSeq sq = a.seq[i];
    const int t = row - sq.first;
    if (a.chunks[i] == 1 || t >= sq.n) return;   // written already, or a row of another launch
    const int n = (block_tiles(sq, t / a.block, a.block) + a.tiles - 1) / a.tiles;
    const int kvh = head / a.rep, c = threadIdx.x % C;
    float M = -INFINITY, L = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
        const size_t at = (size_t)(a.base[i] + (k * sq.n + t) * a.rep + head % a.rep) * a.n_kv + kvh;
        const f32x2_t ml = *reinterpret_cast<const f32x2_t*>(a.part_ml + at * 2);
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part_o + at * D + 4 * c);
        const float m_new = fmaxf(M, ml[0]);
        const float w0 = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - m_new);
        const float w1 = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - m_new);
        o = o * w0 + x * w1;
        L = L * w0 + ml[1] * w1;
        M = m_new;
    }
    store4(static_cast<T*>(a.out) + ((size_t)row * a.n_q + head) * D + 4 * c, o * (1.0f / L));
}

template <int D, int KV, class T>
sa_status launch_chunks(const ChunkArgs& a, int rows, bool merge, hipStream_t st) {
    constexpr int lds = Geo<D, KV>::LDS;
    constexpr auto kernel = chunk_attn_kernel<D, KV, T>;
    SA_TRY(pf::opt_in_lds<kernel>(lds));
    hipLaunchKernelGGL(kernel, dim3((unsigned)a.start[a.n_seq] * a.n_kv), dim3(kThreads), lds, st, a);
    SA_CHECK_LAUNCH();
    if (!merge) return SA_OK;
    const long long n = (long long)rows * a.n_q;
    return merge_rows<D>(n, [&](dim3 grid, long long row0) {
        hipLaunchKernelGGL((chunk_merge_kernel<D, T>), grid, dim3(256), 0, st, a, row0, n);
    });
}

template <int D>
sa_status dispatch_chunks(const ChunkArgs& a, sa_dtype kv, bool q16, int rows, bool merge, hipStream_t st) {
    if (kv == SA_DTYPE_F32) return launch_chunks<D, kF32, float>(a, rows, merge, st);
    if (kv == SA_DTYPE_BF16)
        return q16 ? launch_chunks<D, kBf16, uint16_t>(a, rows, merge, st)
                   : launch_chunks<D, kBf16, float>(a, rows, merge, st);
    return q16 ? launch_chunks<D, kFp8, uint16_t>(a, rows, merge, st) : launch_chunks<D, kFp8, float>(a, rows, merge, st);
}

// Tokens of a block: the query rows that a workgroup takes, at most 64 tokens (a
// bit of Item::single each).
int block_tokens(bool f32, int rep) {
    return std::max(1, std::min(64, (f32 ? Geo<128, kF32>::ROWS : Geo<128, kBf16>::ROWS) / rep));
}
// Workgroups that a launch of chunks aims at: a round and a quarter of them.
long long chunk_round(bool f32) {
    const long long slots = (f32 ? 1LL : 2LL) * device_cu_count();
    return slots + slots / 4;
}
constexpr int kChunkRounds = 4;   // of workgroups that long contexts are cut into

}  // namespace

size_t extend_rows_ws(int n, const int32_t* counts, int n_q, int n_kv, int d, bool f32, long long max_tokens) {
    const int rep = n_q / n_kv, block = block_tokens(f32, rep);
    const long long tiles = (max_tokens + kTile - 1) / kTile;
    const long long most = std::min<long long>(tiles, std::max<long long>(kMaxChunks, ceil_div(tiles, kChunkTiles)));
    if (most <= 1) return 0;
    long long rows = 0, blocks = 0, widest = 0;
    for (int i = 0; i < n; ++i) {
        rows += (long long)counts[i] * n_q;
        blocks += ceil_div(counts[i], block);
        widest = std::max<long long>(widest, std::min(counts[i], block) * rep);
    }
    // By chunks of a sequence, and by workgroups of the launch.
    const long long by_chunks = rows * most;
    const long long forced = tiles > kChunkTiles ? blocks * n_kv * ceil_div(tiles, kChunkTiles) : 0;
    const long long by_groups = std::max(kChunkRounds * chunk_round(f32), forced) * widest;
    return (size_t)std::max(rows, std::min(by_chunks, by_groups)) * (d + 2) * sizeof(float);
}

sa_status extend_rows(const PagedView& c, const void* q, bool q16, int n_q, const ChunkSeq* seqs, int n, float scale,
                      void* out, void* ws, size_t ws_bytes, hipStream_t st) {
    ChunkArgs a{};
    set_cache(a, c, n_q, scale);
    a.q = q;
    a.out = out;
    const bool f32 = c.kv == SA_DTYPE_F32;
    a.block = block_tokens(f32, a.rep);
    for (int i0 = 0; i0 < n; i0 += kRowsPerLaunch) {
        a.n_seq = std::min(kRowsPerLaunch, n - i0);
        long long work = 0;
        int longest = 0;
        for (int i = 0; i < a.n_seq; ++i) {
            a.seq[i] = seqs[i0 + i];
            const int blocks = ceil_div(a.seq[i].n, a.block);
            for (int b = 0; b < blocks; ++b) work += block_tiles(a.seq[i], b, a.block);
            if (blocks) longest = std::max(longest, block_tiles(a.seq[i], blocks - 1, a.block));
        }
        if (longest == 0) continue;
        work *= a.n_kv;
        auto items = [&](int tiles) {
            long long k = 0;
            for (int i = 0; i < a.n_seq; ++i) {
                const int blocks = ceil_div(a.seq[i].n, a.block);
                if (blocks) k += (long long)blocks * ceil_div(block_tiles(a.seq[i], blocks - 1, a.block), tiles);
            }
            return k;
        };
        const long long round = chunk_round(f32);
        int tiles = longest <= (f32 ? 2 : 4) * kWaves
                        ? longest
                        : std::max<int>(pick_tiles(round, work, [&](int t) { return items(t) * a.n_kv; }, kLongChunk8),
                                        (int)std::min<long long>(longest, work / (kChunkRounds * round)));
        // no more partials than extend_rows_ws counts on
        while (tiles < longest && items(tiles) * a.n_kv > kChunkRounds * round) tiles += kWaves;
        tiles = std::min(std::max(tiles, ceil_div(longest, kMaxChunks)), kChunkTiles);
        a.tiles = tiles;
        long long parts = 0, at = 0;
        bool merge = false;
        for (int i = 0; i < a.n_seq; ++i) {
            const int blocks = ceil_div(a.seq[i].n, a.block);
            a.chunks[i] = blocks ? ceil_div(block_tiles(a.seq[i], blocks - 1, a.block), tiles) : 1;
            a.start[i] = (int)at;
            a.base[i] = (int)parts;
            at += (long long)blocks * a.chunks[i];
            if (a.chunks[i] > 1) {
                parts += (long long)a.chunks[i] * a.seq[i].n * a.rep;
                merge = true;
            }
        }
        a.start[a.n_seq] = (int)at;
        const int rows = a.seq[a.n_seq - 1].first + a.seq[a.n_seq - 1].n - a.seq[0].first;
        // a grid has fewer than 2^32 threads
        if (at * a.n_kv >= (1LL << 32) / kThreads)
            return fail(SA_EINVAL, "too many tokens for one call");
        if (merge) {
            const size_t need = (size_t)parts * a.n_kv * (c.d + 2) * sizeof(float);
            if (!ws || ws_bytes < need) return fail(SA_ENOMEM, "workspace too small for the partials");
            a.part_o = static_cast<float*>(ws);
            a.part_ml = a.part_o + (size_t)parts * a.n_kv * c.d;
        }
        SA_TRY(c.d == 64 ? dispatch_chunks<64>(a, c.kv, q16, rows, merge, st)
                         : dispatch_chunks<128>(a, c.kv, q16, rows, merge, st));
    }
    return SA_OK;
}

}  // namespace sa
