// Attention of chunks of many new tokens over a paged cache, on bf16 MFMA.
//
// A chunk's query rows (new tokens x query heads of a KV head, in that order) are cut
// into blocks of 32 per wave; token j of a sequence of len committed tokens sees keys
// 0 .. len + j.  A workgroup takes a block of one KV head and a range of its key
// tiles, a tile being a page's 64 keys, and leaves its rows' output, or where a
// block's tiles are cut a partial (m, l, O) per row for a second launch to join.
//
// bf16 queries (and output) over a bf16 or 8-bit cache: v_mfma_f32_32x32x16_bf16 and
// the softmax of bf16_wave.h; the roundings are P to bf16 (2^-8 of each weight, the
// sums taken of the rounded ones) and the output's.  A bf16 page is loaded straight
// into LDS; codes of an 8-bit page are widened on the way, times their row's scale,
// which is exact, once per workgroup rather than once per wave.
//
// fp32 queries (and output): every operand as the exact sum of bf16 terms, three for
// fp32 values, one for what bf16 and 8-bit caches hold; of the products of three by
// three terms the six largest are taken (what is left out is below 2^-24 of the
// product), of one by three all; v_mfma_f32_16x16x32_bf16, a wave owns 16 rows,
// tiles of 32 keys become terms on their way into LDS.
//
// Whole blocks, or blocks cut into parts of equal lengths, keep the CUs evenly busy where they
// make many rounds or fit them; for fp32 queries there is a third way, all blocks'
// tiles in a row cut into as many equal lengths as workgroups run at a time, each
// going from block to block (700 fp32 tokens behind 4000, 16 / 8 heads of 128: 200 -> 137
// us).  bf16 queries gain nothing by it: what a further block costs to begin, 8 us with
// eight waves, is more than they lose by rounds.
//
// Rows whose sums are not finite are computed anew over what they see (plain_row.h).
//
// Bound, 16 / 8 heads of 128: MFMA and the softmax's VALU work beside it.  2048 bf16 tokens
// behind 30720, 533 GF: 505 - 523 us, 1.02 - 1.06 PFLOP/s of 1.6 that a large product
// reaches, MFMA 53 % and VALU 44 % busy, the second launch 17 of them.  512 fp32 tokens behind
// 3584, 16.1 GF x 6: 92 - 94 us, 1.03 - 1.05 PFLOP/s of products, MFMA 51 %, VALU 39 %; fp32 over
// bf16 or 8 bits, three products, 2048 behind 8192: 426 - 432 us, 1.08.  Seven chunks of
// 1 - 700 tokens over 8 bits, 32 / 8 heads of 64, 82.9 GF: 130 - 134 us; at 64 the softmax is as
// long as the products (VALU 63 %, MFMA 40 %), the joining launch takes 15, and rounds of
// workgroups of unequal lengths cost a tenth.
#include <algorithm>
#include <cmath>
#include <vector>

#include "bf16_terms.h"
#include "bf16_wave.h"
#include "plain_row.h"
#include "ranges.h"

namespace sa {
namespace {

constexpr int kSortedBlocks = 128;   // of a launch whose parts have an order or equal lengths

struct BlockArgs {
    const void* q;
    const void* k;
    const void* v;
    const uint8_t* k_scale;
    const uint8_t* v_scale;
    const int32_t* table;
    void* out;
    float* part_o;
    float* part_ml;
    int n_kv, n_q, rep, max_pages, num_pages;
    int n_seq;
    int rows;                                // query rows of a block
    int tile;                                // keys of a tile
    int tiles;                               // key tiles of a workgroup
    float sl2;                               // |scale| log2(e)
    float factor;                            // scale log2(e)
    uint32_t q_sign;                         // 0x80008000 for a negative scale
    ChunkSeq seq[kRowsPerLaunch];
    int32_t start[kRowsPerLaunch + 1];       // a sequence's first item, of blocks x parts
    // Several sequences' parts in the order of their lengths: first the `full` ones of
    // a.tiles, block k's from full_at[k] on, then rest[..], the blocks that leave a shorter
    // one, longest first; start[i] is then sequence i's first block.  n_blocks 0: sequence
    // behind sequence.
    int n_blocks, full;
    uint16_t full_at[kSortedBlocks + 1];
    uint8_t rest[kSortedBlocks];
    // Tiles cut evenly: even > 0 tiles per workgroup of the blocks' tiles in a row,
    // block_at[k] before block k; start[i] is then sequence i's first block.
    int even;
    union {
        struct {
            int32_t base[kRowsPerLaunch];    // its first partial row
            int32_t parts[kRowsPerLaunch];   // of its last block
        };
        int32_t block_at[kSortedBlocks + 1];
    };
};
static_assert(sizeof(BlockArgs) <= 4096, "kernel arguments");

// Key tiles that block b of a sequence sees.
__host__ __device__ inline int block_key_tiles(const ChunkSeq& s, int b, int rows, int rep, int tile) {
    const long long end = (long long)(b + 1) * rows, all = (long long)s.n * rep;
    return (int)((s.len + ((end < all ? end : all) - 1) / rep) / tile) + 1;
}

// A workgroup's place.
struct Block {
    ChunkSeq sq;
    int kvh, r0, row_end;   // query rows [r0, row_end) of the sequence
    int u0, u1;             // key tiles
    bool whole;             // the output itself
    long long part0;        // partial row of query row 0
    const __attribute__((address_space(4))) int32_t* pages;
};
// Where workgroup `item` leaves its partial of a block whose tiles begin at from: of the
// blocks that it has a part of only its first and its last may be others' too.
__device__ __forceinline__ long long even_part(int item, int from, int even) {
    return 2LL * item + (from > item * even);
}
// The next block of a workgroup where tiles are cut evenly, while there is one; at: -1, then
// where it begins.
__device__ __forceinline__ bool place_even(const BlockArgs& a, Block& w, int& at) {
    const int lane = threadIdx.x & (kWave - 1), item = blockIdx.x / a.n_kv;
    const int first = item * a.even, end = min(first + a.even, a.block_at[a.n_blocks]);
    if (at < 0) at = first;
    if (at >= end) return false;
    int k = -1, i = 0;
    for (int j = lane; j - lane < a.n_blocks; j += kWave) k += __popcll(__ballot(j < a.n_blocks && a.block_at[j] <= at));
    if (a.n_seq > 1) i = __popcll(__ballot(lane < a.n_seq && a.start[lane] <= k)) - 1;
    w.sq = a.seq[i];
    w.kvh = blockIdx.x % a.n_kv;
    const int all = w.sq.n * a.rep, from = a.block_at[k], to = a.block_at[k + 1];
    w.r0 = ((all + a.rows - 1) / a.rows - 1 - (k - a.start[i])) * a.rows;
    w.row_end = min(all, w.r0 + a.rows);
    w.u0 = at - from;
    w.u1 = min(to, end) - from;
    w.whole = w.u0 == 0 && to <= end;
    w.part0 = even_part(item, from, a.even) * a.rows - w.r0;
    w.pages = (const __attribute__((address_space(4))) int32_t*)(a.table + (size_t)w.sq.cache_row * a.max_pages);
    at = from + w.u1;
    return true;
}
template <int TILE>
__device__ __forceinline__ bool place(const BlockArgs& a, Block& w) {
    const int lane = threadIdx.x & (kWave - 1);
    const int item = blockIdx.x / a.n_kv;   // the KV head varies fastest: with 8 of them each XCD has one
    // One sequence: its arguments with the others', not behind a search (arguments may be
    // a trip to host memory away).
    int parts = a.parts[0], local = item, base = 0;
    w.sq = a.seq[0];
    if (a.n_blocks) {
        int k = -1;
        if (item < a.full)
            for (int j = lane; j - lane < a.n_blocks; j += kWave)
                k += __popcll(__ballot(j < a.n_blocks && a.full_at[j] <= item));
        else
            k = __builtin_amdgcn_readfirstlane(a.rest[item - a.full]);
        const int c = item < a.full ? item - a.full_at[k] : a.full_at[k + 1] - a.full_at[k];
        const int i = __popcll(__ballot(lane < a.n_seq && a.start[lane] <= k)) - 1;
        w.sq = a.seq[i];
        parts = a.parts[i];
        local = (k - a.start[i]) * parts + c;
        base = a.base[i];
    } else if (a.n_seq > 1) {
        const int i = __popcll(__ballot(lane < a.n_seq && a.start[lane] <= item)) - 1;
        w.sq = a.seq[i];
        parts = a.parts[i];
        local = item - a.start[i];
        base = a.base[i];
    }
    w.kvh = blockIdx.x % a.n_kv;
    const int all = w.sq.n * a.rep;
    // the longest blocks first
    const int blocks = (all + a.rows - 1) / a.rows, b = blocks - 1 - local / parts, c = local % parts;
    w.r0 = b * a.rows;
    w.row_end = min(all, w.r0 + a.rows);
    w.u0 = c * a.tiles;
    w.u1 = min(w.u0 + a.tiles, block_key_tiles(w.sq, b, a.rows, a.rep, TILE));
    w.whole = parts == 1;
    w.part0 = base + (long long)c * all;
    // read with scalar loads
    w.pages = (const __attribute__((address_space(4))) int32_t*)(a.table + (size_t)w.sq.cache_row * a.max_pages);
    return w.u0 < w.u1;
}
// The page of a sequence's 64 keys from 64 j on; an id outside the pool (an entry
// that was never set) is clamped so that no load can fault.
__device__ __forceinline__ int page_of(const BlockArgs& a, const Block& w, int j) {
    return min(max(w.pages[j], 0), a.num_pages - 1);
}
__device__ __forceinline__ size_t out_row(const BlockArgs& a, const Block& w, int row) {
    const int t = row / a.rep;
    return ((size_t)(w.sq.first + t) * a.n_q + w.kvh * a.rep + row - t * a.rep);
}

// Query row `row` over the workgroup's keys without matrix instructions, one wave.
template <int D, int KV, int TILE, class T>
__device__ __forceinline__ void block_plain(const BlockArgs& a, const Block& w, int row) {
    using E = std::conditional_t<KV == SA_DTYPE_FP8, uint8_t, std::conditional_t<KV == SA_DTYPE_BF16, uint16_t, float>>;
    const int lane = threadIdx.x & (kWave - 1);
    const int end = w.sq.len + row / a.rep + 1;   // keys that it sees
    const size_t o = out_row(a, w, row) * D;
    PlainRow<D> p;
    for (int u = w.u0; u < w.u1 && u * TILE < end && !p.lost(); ++u) {
        const int k0 = u * TILE;
        const size_t key = ((size_t)page_of(a, w, k0 / SA_PAGE_TOKENS) * a.n_kv + w.kvh) * SA_PAGE_TOKENS +
                           k0 % SA_PAGE_TOKENS;
        auto value = [&](const void* pool, int i) { return static_cast<const E*>(pool) + (key + i) * D; };
        auto scale = [&](const uint8_t* s, int i) {
            if constexpr (KV == SA_DTYPE_FP8) return scale_of(s[key + i]);
            else return 1.f;
        };
        p.keys(min(TILE, end - k0), static_cast<const T*>(a.q) + o, a.factor,
               [&](int i) { return value(a.k, i); }, [&](int i) { return value(a.v, i); },
               [&](int i) { return scale(a.k_scale, i); }, [&](int i) { return scale(a.v_scale, i); });
    }
    const size_t at = (size_t)(w.part0 + row) * a.n_kv + w.kvh;
#pragma unroll
    for (int e = 0; e < p.E; ++e) {
        const int d = lane * p.E + e;
        if (!w.whole) a.part_o[at * D + d] = p.o[e];
        else if constexpr (sizeof(T) == 2) static_cast<T*>(a.out)[o + d] = f32_to_bf16_rne(p.o[e] / p.l);
        else static_cast<T*>(a.out)[o + d] = p.o[e] / p.l;
    }
    if (!w.whole && lane == 0) {
        a.part_ml[at * 2] = p.m;
        a.part_ml[at * 2 + 1] = p.l;
    }
}

// ---------------------------------------------------------------- bf16

template <int D, int W, bool FP8>
__global__ void __launch_bounds__(W * kWave, W == 8 && D == 64 ? 4 : 1) extend_bf16_kernel(BlockArgs a) {
    using G = BfGeo<D>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    lds_u8_t* const smem = (lds_u8_t*)smem_raw;
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<size_t>(smem));
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    Block b;
    if (!place<kBfTile>(a, b)) return;
    const int last_key = b.sq.len + b.sq.n - 1;   // of the sequence: keys behind it are not read

    // ---- a bf16 tile straight into LDS, two tiles ahead ----
    // Load i of a wave copies RPL rows, this lane's 16 bytes of them at off[i] from
    // the page's first row; rows behind the sequence repeat its last.
    constexpr int NI = G::NL / W > 0 ? G::NL / W : 1;
    int row[NI], col[NI];
    uint32_t off[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        row[i] = (wave * NI + i) * G::RPL + lane / G::CPR;
        col[i] = 16 * ((lane % G::CPR) ^ G::swz(row[i] & 15));
        off[i] = row[i] * G::ROWB + col[i];
    }
    auto load_bf16 = [&](int u, int page) {
        if (G::NL < W && wave >= G::NL) return;
        const size_t at = ((size_t)page * a.n_kv + b.kvh) * G::HALF;
        const char* kt = static_cast<const char*>(a.k) + at;
        const char* vt = static_cast<const char*>(a.v) + at;
        lds_u8_t* dst = smem + (u & 1) * G::STAGE;
        const int most = last_key - u * kBfTile;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            uint32_t o = off[i];
            if (most < kBfTile - 1) o = min(row[i], most) * G::ROWB + col[i];
            dma16_from(kt, o, dst + (wave * NI + i) * 1024);
            dma16_from(vt, o, dst + G::HALF + (wave * NI + i) * 1024);
        }
    };
    // ---- an 8-bit tile through registers, one tile ahead ----
    constexpr int PIECES = kBfTile * D / 16;             // of 16 codes
    constexpr int NP = PIECES / (W * kWave) > 0 ? PIECES / (W * kWave) : 1;
    const bool loads = PIECES >= W * kWave || threadIdx.x < PIECES;
    u32x4_t rk[NP], rv[NP];
    uint32_t sk[NP], sv[NP];
    auto load_fp8 = [&](int u, int page) {
        if (!loads) return;
        const size_t at = ((size_t)page * a.n_kv + b.kvh) * kBfTile;
        const int most = last_key - u * kBfTile;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int idx = threadIdx.x + i * W * kWave;
            const size_t r = at + min(idx / (D / 16), most);
            rk[i] = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(a.k) + r * D + 16 * (idx % (D / 16)));
            rv[i] = *reinterpret_cast<const u32x4_t*>(static_cast<const char*>(a.v) + r * D + 16 * (idx % (D / 16)));
            sk[i] = a.k_scale[r];
            sv[i] = a.v_scale[r];
        }
    };
    auto store_fp8 = [&](int u) {
        if (!loads) return;
        lds_u8_t* dst = smem + (u & 1) * G::STAGE;
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int idx = threadIdx.x + i * W * kWave;
            const int r = idx / (D / 16), c = 2 * (idx % (D / 16));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                lds_u8_t* at = dst + r * G::ROWB + (((c + h) ^ G::swz(r & 15)) << 4);
                *reinterpret_cast<__attribute__((address_space(3))) bf16x8_t*>(at) =
                    codes_bf16x8(rk[i][2 * h], rk[i][2 * h + 1], scale_of(sk[i]));
                *reinterpret_cast<__attribute__((address_space(3))) bf16x8_t*>(at + G::HALF) =
                    codes_bf16x8(rv[i][2 * h], rv[i][2 * h + 1], scale_of(sv[i]));
            }
        }
    };

    int page = page_of(a, b, b.u0), next = b.u0 + 1 < b.u1 ? page_of(a, b, b.u0 + 1) : 0;
    if constexpr (FP8) load_fp8(b.u0, page);
    else load_bf16(b.u0, page);
    // This wave's 32 query rows, and the tokens that they belong to.
    const int w0 = b.r0 + wave * 32;
    const int my_row = min(w0 + (lane & 31), b.row_end - 1);
    const bool active = w0 < b.row_end;
    const int q_lo = b.sq.len + min(w0, b.row_end - 1) / a.rep, q_hi = b.sq.len + min(w0 + 31, b.row_end - 1) / a.rep;
    const int q_mine = b.sq.len + my_row / a.rep;   // the last key that this lane's row sees
    BfWave<D> w;
    w.init(static_cast<const uint16_t*>(a.q) + out_row(a, b, my_row) * D, a.sl2, a.q_sign, w0, lane);
    if constexpr (FP8) {
        store_fp8(b.u0);
        if (b.u0 + 1 < b.u1) load_fp8(b.u0 + 1, next);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    } else if (b.u0 + 1 < b.u1) {
        load_bf16(b.u0 + 1, next);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NI) : "memory");   // the first tile
    } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    next = b.u0 + 2 < b.u1 ? page_of(a, b, b.u0 + 2) : 0;
    // Tile u has been computed by this wave.
    auto end_tile = [&](int u) {
        if constexpr (FP8) {
            if (u + 1 < b.u1) store_fp8(u + 1);           // where tile u - 1 was
            if (u + 2 < b.u1) load_fp8(u + 2, next);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (u + 2 < b.u1) load_bf16(u + 2, next);
        }
        if (u + 3 < b.u1) next = page_of(a, b, u + 3);
    };
    auto edge_tile = [&](int u) {
        const uint32_t sb = lds_at + (u & 1) * G::STAGE;
        if (active) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int k = u * kBfTile + 32 * kb;
                const uint32_t hb = sb + kb * 32 * G::ROWB;
                if (k > q_hi) continue;
                // Eight waves come here only with the tiles at the diagonal: one form, with
                // the mask, is enough, and without the other the registers do (2048
                // tokens behind none 71 -> 45 us), but for five that heads of 64 over 8 bits
                // still spill around the ping-pong.
                f32x16_t s = w.scores(hb);
                if (W == 4 && k + 31 <= q_lo) {
                    w.template weigh<false>(s, hb);
                } else {
                    const int last = q_mine - k - 8 * w.hh;
#pragma unroll
                    for (int j = 0; j < 16; ++j) s[j] = 16 * (j / 8) + j % 8 > last ? -INFINITY : s[j] * w.c;
                    w.template weigh<true>(s, hb);
                }
            }
        }
        end_tile(u);
    };
    int u = b.u0;
    if constexpr (W == 8) {
        // The tiles that every row of the workgroup sees whole, in ping-pong: waves w and
        // w + 4 share a SIMD, and each half tile is a block of MFMAs (the half before's P
        // V, this half's scores) and a softmax.  Waves 4 - 7 take the half's barrier
        // between the two, waves 0 - 3 behind both, so that on every SIMD one wave's
        // softmax runs under the other's MFMAs.
        const int hi = min(b.u1, (b.sq.len + b.r0 / a.rep + 1) / kBfTile);
        if (u < hi) {
            const bool late = wave >= W / 2;
            if (!late) __builtin_amdgcn_s_setprio(1);
            bf16x8_t vf[G::NDB][2], pb[2];
#pragma unroll
            for (int db = 0; db < G::NDB; ++db) vf[db][0] = vf[db][1] = bf16x8_t{};
            pb[0] = pb[1] = bf16x8_t{};
            auto pv = [&]() {
#pragma unroll
                for (int db = 0; db < G::NDB; ++db)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
                        w.acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db][t], pb[t], w.acc[db], 0, 0, 0);
            };
            for (; u < hi; ++u) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const uint32_t hb = lds_at + (u & 1) * G::STAGE + kb * 32 * G::ROWB;
                    bf16x8_t kf[G::NKS];
#pragma unroll
                    for (int ks = 0; ks < G::NKS; ++ks) kf[ks] = w.k_frag(hb, ks);
                    pv();
#pragma unroll
                    for (int db = 0; db < G::NDB; ++db)
#pragma unroll
                        for (int t = 0; t < 2; ++t) vf[db][t] = w.v_frag(hb, db, t);
                    f32x16_t s = {};
#pragma unroll
                    for (int ks = 0; ks < G::NKS; ++ks)
                        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[ks], w.qf[ks], s, 0, 0, 0);
                    auto sync = [&]() {
                        __builtin_amdgcn_sched_barrier(0);
                        if (kb == 0) asm volatile("s_barrier" ::: "memory");
                        else end_tile(u);
                        __builtin_amdgcn_sched_barrier(0);
                    };
                    if (late) sync();
                    w.template softmax<false>(s, pb);
                    if (!late) sync();
                }
            }
            pv();
            __builtin_amdgcn_s_setprio(0);
        }
    }
    for (; u < b.u1; ++u) edge_tile(u);

    const int rows = b.row_end - w0;   // of the wave, where positive
    uint32_t anew;
    if (b.whole) {
        // The output through LDS, 32 rows per wave, so that stores are whole rows.
        anew = w.store(b.row_end, [&](int r) { return static_cast<uint16_t*>(a.out) + out_row(a, b, r) * D; },
                       smem + wave * 32 * G::ROWB, lane);
    } else {
        const float l = w.l + xor32(w.l);
        float zero = 0.f;   // NaN where an accumulator is not finite
#pragma unroll
        for (int db = 0; db < G::NDB; ++db)
#pragma unroll
            for (int j = 0; j < 16; ++j) zero = fmaf(w.acc[db][j], 0.f, zero);
        const uint64_t bad = __ballot(w.n < rows && !(l + zero < INFINITY));
        anew = (uint32_t)bad | (uint32_t)(bad >> 32);
        if (w.n < rows && !(anew >> w.n & 1)) {
            const size_t at = (size_t)(b.part0 + w0 + w.n) * a.n_kv + b.kvh;
            float* o = a.part_o + at * D + 4 * w.hh;
#pragma unroll
            for (int db = 0; db < G::NDB; ++db)
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
                    *reinterpret_cast<f32x4_t*>(o + 32 * db + 8 * jj) =
                        f32x4_t{w.acc[db][4 * jj], w.acc[db][4 * jj + 1], w.acc[db][4 * jj + 2], w.acc[db][4 * jj + 3]};
            if (w.hh == 0) *reinterpret_cast<f32x2_t*>(a.part_ml + at * 2) = f32x2_t{w.m, l};
        }
    }
    for (; anew; anew &= anew - 1)
        block_plain<D, FP8 ? SA_DTYPE_FP8 : SA_DTYPE_BF16, kBfTile, uint16_t>(a, b, w0 + __builtin_ctz(anew));
}

// ---------------------------------------------------------------- fp32

constexpr int kTermTile = 32;

template <int D, int KV>
struct TermGeo {
    static constexpr int NT = KV == SA_DTYPE_F32 ? kTerms : 1;   // terms of a cached value
    static constexpr int PAIRS = KV == SA_DTYPE_F32 ? 6 : 3;
    static constexpr int ROWB = 2 * D;                  // a row of one term
    static constexpr int TERM = kTermTile * ROWB;       // one term of K or V
    static constexpr int STAGE = 2 * NT * TERM;         // K's terms, then V's
    static constexpr int CPR = ROWB / 16;
    static constexpr int KS = D / 32, DB = D / 16;
    // Terms of the cached and of the other operand of a product, largest first.
    static constexpr int pair_a(int pr) { return NT == 1 ? 0 : (pr == 2 || pr == 4 ? 1 : pr == 5 ? 2 : 0); }
    static constexpr int pair_b(int pr) { return NT == 1 ? pr : (pr == 1 || pr == 4 ? 1 : pr == 3 ? 2 : 0); }
    // Chunk c of row r at c ^ swz(r): rows 8a + 4kb + b of a K fragment read and rows
    // 8g + 4u + b of a half wave's V^T read on different banks.
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (CPR == 16) return ((r & 3) << 2) | (((r >> 3) & 1) << 1) | ((r >> 4) & 1);
        else return (((r >> 1) & 1) << 2) | (((r >> 3) & 1) << 1) | ((r >> 4) & 1);
    }
    static __device__ __forceinline__ int off(int r, int c) { return r * ROWB + ((c ^ swz(r)) << 4); }
};

// Eight cached values on their way into LDS.
template <int KV>
struct Staged {
    u32x4_t x[KV == SA_DTYPE_F32 ? 2 : 1];
    uint32_t scale;
    __device__ __forceinline__ void load(const void* pool, const uint8_t* scales, size_t row, size_t at) {
        if constexpr (KV == SA_DTYPE_F32) {
            x[0] = *reinterpret_cast<const u32x4_t*>(static_cast<const float*>(pool) + at);
            x[1] = *reinterpret_cast<const u32x4_t*>(static_cast<const float*>(pool) + at + 4);
        } else if constexpr (KV == SA_DTYPE_BF16) {
            x[0] = *reinterpret_cast<const u32x4_t*>(static_cast<const uint16_t*>(pool) + at);
        } else {
            const uint2 c = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at);
            x[0][0] = c.x;
            x[0][1] = c.y;
            scale = scales[row];
        }
    }
    template <int N>
    __device__ __forceinline__ void terms(bf16x8_t (&t)[N]) const {
        if constexpr (KV == SA_DTYPE_F32)
            split_terms(__builtin_bit_cast(f32x4_t, x[0]), __builtin_bit_cast(f32x4_t, x[1]), t);
        else if constexpr (KV == SA_DTYPE_BF16) t[0] = __builtin_bit_cast(bf16x8_t, x[0]);
        else t[0] = codes_bf16x8(x[0][0], x[0][1], scale_of(scale));
    }
};

template <int D, int W, int KV, bool EVEN>
__global__ void __launch_bounds__(W * kWave) extend_f32_kernel(BlockArgs a) {
    using G = TermGeo<D, KV>;
    constexpr int THREADS = W * kWave;
    constexpr int C8 = D / 8;                           // 8-element pieces of a row
    constexpr int NC = kTermTile * C8 / THREADS > 0 ? kTermTile * C8 / THREADS : 1;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    lds_u8_t* const smem = (lds_u8_t*)smem_raw;
    Block b;
    auto block = [&]() {
        uint32_t tid = threadIdx.x;
        if constexpr (EVEN) asm volatile("" : "+v"(tid));   // nothing of a block stays in registers for the next
        const int lane = tid & (kWave - 1);
        const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
        const int r16 = lane & 15, g = lane >> 4;
        const int last_key = b.sq.len + b.sq.n - 1;   // of the sequence: keys behind it are not read

        // ---- tiles: as cached in registers one tile ahead, bf16 terms in LDS ----
        const bool loads = kTermTile * C8 >= THREADS || (int)tid < kTermTile * C8;
        Staged<KV> sk[NC], sv[NC];
        auto load = [&](int u, int page) {
            if (!loads) return;
            const int k0 = u * kTermTile;
            const size_t first = ((size_t)page * a.n_kv + b.kvh) * SA_PAGE_TOKENS + k0 % SA_PAGE_TOKENS;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int idx = tid + i * THREADS;
                const size_t row = first + min(idx / C8, last_key - k0), at = row * D + 8 * (idx % C8);
                sk[i].load(a.k, a.k_scale, row, at);
                sv[i].load(a.v, a.v_scale, row, at);
            }
        };
        auto store_tile = [&](int u) {
            if (!loads) return;
            lds_u8_t* base = smem + (u & 1) * G::STAGE;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const int idx = tid + i * THREADS;
                const int off = G::off(idx / C8, idx % C8);
                bf16x8_t t[G::NT];
                sk[i].terms(t);
#pragma unroll
                for (int x = 0; x < G::NT; ++x)
                    *reinterpret_cast<__attribute__((address_space(3))) bf16x8_t*>(base + x * G::TERM + off) = t[x];
                sv[i].terms(t);
#pragma unroll
                for (int x = 0; x < G::NT; ++x)
                    *reinterpret_cast<__attribute__((address_space(3))) bf16x8_t*>(base + (G::NT + x) * G::TERM + off) =
                        t[x];
            }
        };
        auto page_at = [&](int u) { return page_of(a, b, u * kTermTile / SA_PAGE_TOKENS); };
        load(b.u0, page_at(b.u0));
        int next = b.u0 + 1 < b.u1 ? page_at(b.u0 + 1) : 0;

        const int w0 = b.r0 + wave * 16;
        const int my_row = min(w0 + r16, b.row_end - 1);
        const bool active = w0 < b.row_end;
        const int q_lo = b.sq.len + min(w0, b.row_end - 1) / a.rep, q_hi = b.sq.len + min(w0 + 15, b.row_end - 1) / a.rep;
        const int q_mine = b.sq.len + my_row / a.rep;   // the last key that this lane's row sees
        bf16x8_t qf[G::KS][kTerms];
        {
            const float* row = static_cast<const float*>(a.q) + out_row(a, b, my_row) * D + 8 * g;
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks)
                split_terms(*reinterpret_cast<const f32x4_t*>(row + 32 * ks) * a.factor,
                            *reinterpret_cast<const f32x4_t*>(row + 32 * ks + 4) * a.factor, qf[ks]);
        }
        f32x4_t acc[G::DB];
#pragma unroll
        for (int db = 0; db < G::DB; ++db) acc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        float m = -INFINITY, bias = 0.f, l = 0.f, cap = -1.f;

        auto compute = [&](int k0, const lds_u8_t* sb, bool mask) {
            // element 4 kb + e of a lane: key 8 g + 4 kb + e
            f32x4_t s[2] = {f32x4_t{bias, bias, bias, bias}, f32x4_t{bias, bias, bias, bias}};
#pragma unroll
            for (int ks = 0; ks < G::KS; ++ks) {
                bf16x8_t kf[2][G::NT];
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int t = 0; t < G::NT; ++t)
                        kf[kb][t] = *reinterpret_cast<const __attribute__((address_space(3))) bf16x8_t*>(
                            sb + t * G::TERM + G::off(8 * (r16 >> 2) + 4 * kb + (r16 & 3), 4 * ks + g));
#pragma unroll
                for (int pr = 0; pr < G::PAIRS; ++pr)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
                        s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kb][G::pair_a(pr)], qf[ks][G::pair_b(pr)], s[kb],
                                                                        0, 0, 0);
            }
            if (mask) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k0 + 8 * g + j > q_mine) s[j >> 2][j & 3] = -INFINITY;
            }
            float p[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(s[j >> 2][j & 3]);
            float sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            if (__any(!(sum <= cap))) {
                float mt = s[0][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) mt = fmaxf(mt, s[j >> 2][j & 3]);
                const float m_new = fmaxf(m, group_reduce<OpMax, 16, kWave>(mt) - bias);
                const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
#pragma unroll
                for (int db = 0; db < G::DB; ++db) acc[db] *= alpha;
                l *= alpha;
                const float b_new = m_new == -INFINITY ? 0.f : -m_new;
                const float delta = b_new - bias;
#pragma unroll
                for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(s[j >> 2][j & 3] + delta);
                sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                m = m_new;
                bias = b_new;
                cap = m_new == -INFINITY ? -1.f : kBfRaiseAt;
            }
            l += sum;
            bf16x8_t pt[kTerms];
            split_terms(f32x4_t{p[0], p[1], p[2], p[3]}, f32x4_t{p[4], p[5], p[6], p[7]}, pt);
#pragma unroll
            for (int db = 0; db < G::DB; ++db) {
                bf16x8_t vf[G::NT];
                const int c = 2 * db + ((r16 & 3) >> 1), r = 8 * g + (r16 >> 2), h8 = (r16 & 1) * 8;
#pragma unroll
                for (int t = 0; t < G::NT; ++t) {
                    const lds_u8_t* vb = sb + (G::NT + t) * G::TERM + h8;
                    const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vb + G::off(r, c)));
                    const s16x4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vb + G::off(r + 4, c)));
                    vf[t] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
                }
#pragma unroll
                for (int pr = 0; pr < G::PAIRS; ++pr)
                    acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[G::pair_a(pr)], pt[G::pair_b(pr)], acc[db], 0, 0,
                                                                      0);
            }
        };

        store_tile(b.u0);
        if (b.u0 + 1 < b.u1) load(b.u0 + 1, next);
        next = b.u0 + 2 < b.u1 ? page_at(b.u0 + 2) : 0;
        lds_barrier();
        for (int u = b.u0; u < b.u1; ++u) {
            const int k0 = u * kTermTile;
            if (active && k0 <= q_hi) compute(k0, smem + (u & 1) * G::STAGE, k0 + kTermTile - 1 > q_lo);
            if (u + 1 < b.u1) {
                store_tile(u + 1);   // where tile u - 1 was
                if (u + 2 < b.u1) load(u + 2, next);
                if (u + 3 < b.u1) next = page_at(u + 3);
            }
            lds_barrier();
        }

        const float sum = group_reduce<OpSum, 16, kWave>(l);
        const float fine = sum + group_reduce<OpSum, 16, kWave>(not_finite<G::DB>(acc));
        const bool mine = w0 + r16 < b.row_end, ok = fine < INFINITY;
        if (mine && ok) {
            if (b.whole) {
                const float inv = 1.0f / sum;
                float* o = static_cast<float*>(a.out) + out_row(a, b, my_row) * D + 4 * g;
#pragma unroll
                for (int db = 0; db < G::DB; ++db) *reinterpret_cast<f32x4_t*>(o + 16 * db) = acc[db] * inv;
            } else {
                const size_t at = (size_t)(b.part0 + my_row) * a.n_kv + b.kvh;
#pragma unroll
                for (int db = 0; db < G::DB; ++db)
                    *reinterpret_cast<f32x4_t*>(a.part_o + at * D + 16 * db + 4 * g) = acc[db];
                if (g == 0) *reinterpret_cast<f32x2_t*>(a.part_ml + at * 2) = f32x2_t{m, sum};
            }
        }
        for (uint32_t anew = __ballot(mine && !ok) & 0xffff; anew; anew &= anew - 1)
            block_plain<D, KV, kTermTile, float>(a, b, w0 + __builtin_ctz(anew));
    };
    if constexpr (EVEN) {
        for (int at = -1; place_even(a, b, at);) block();
    } else {
        if (place<kTermTile>(a, b)) block();
    }
}

// ---------------------------------------------------------------- partials

// O = sum_c 2^(m_c - M) O_c / sum_c 2^(m_c - M) l_c, D / 4 lanes per row of 256 D / 4
// consecutive (token, head) rows from the launch's first token on.
template <int D, class T, bool EVEN>
__global__ void __launch_bounds__(256) block_merge_kernel(BlockArgs a, long long row0, long long n) {
    constexpr int C = D / 4, ROWS = 256 / C;
    const long long first = row0 + (long long)blockIdx.x * ROWS, r = first + threadIdx.x / C;
    const int i0 = chunk_of(a.seq, a.n_seq, a.seq[0].first + (int)(first / a.n_q));
    if (r >= n) return;
    const int token = a.seq[0].first + (int)(r / a.n_q), head = (int)(r % a.n_q), c = threadIdx.x % C;
    int i = i0;
    while (i + 1 < a.n_seq && a.seq[i + 1].first <= token) ++i;
    const ChunkSeq sq = a.seq[i];
    const int t = token - sq.first;
    if (t >= sq.n) return;                      // a row of another launch
    const int kvh = head / a.rep, row = t * a.rep + head % a.rep;
    const int b = row / a.rows;
    int parts;
    long long first_part, others, step;   // part p's row: first_part or, where p > 0, others + p step
    if constexpr (EVEN) {
        const int k = a.start[i] + (sq.n * a.rep + a.rows - 1) / a.rows - 1 - b;
        const int from = a.block_at[k], item = from / a.even;
        parts = (a.block_at[k + 1] - 1) / a.even - item + 1;
        if (parts == 1) return;                 // written already
        first_part = even_part(item, from, a.even) * a.rows + row - b * a.rows;
        others = even_part(item, item * a.even, a.even) * a.rows + row - b * a.rows;
        step = 2 * a.rows;
    } else {
        if (a.parts[i] == 1) return;
        parts = (block_key_tiles(sq, b, a.rows, a.rep, a.tile) + a.tiles - 1) / a.tiles;
        first_part = others = a.base[i] + row;
        step = (long long)sq.n * a.rep;
    }
    float M = -INFINITY, L = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
        const size_t at = (size_t)(EVEN && p == 0 ? first_part : others + p * step) * a.n_kv + kvh;
        const f32x2_t ml = *reinterpret_cast<const f32x2_t*>(a.part_ml + at * 2);
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part_o + at * D + 4 * c);
        const float m_new = fmaxf(M, ml[0]);
        const float w0 = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - m_new);
        const float w1 = ml[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[0] - m_new);
        o = o * w0 + x * w1;
        L = L * w0 + ml[1] * w1;
        M = m_new;
    }
    store4(static_cast<T*>(a.out) + ((size_t)token * a.n_q + head) * D + 4 * c, o * (1.0f / L));
}

// ---------------------------------------------------------------- launch

constexpr int kMaxRounds = 4;    // of workgroups that a launch's tiles are cut into
// What a workgroup costs besides its tiles, in tiles: its beginning and its output, or
// where a block is cut a partial written and read again (bf16, 6 for both head sizes: 7 chunks
// of 1 - 700 tokens, heads of 128, 216 us, 191 with 9; 16 of 100 - 1000, heads of 64, 397, 331 with
// 4, which 9 leaves at 397).
constexpr int kWholeTiles = 2, kCutBf16 = 9, kCutBf16Narrow = 4, kCutF32 = 4, kCutTerms = 7;
// And a workgroup's further blocks where tiles are cut evenly.
constexpr int kNextF32 = 4, kNextTerms = 14;

// Workgroups of a kind that share a CU (by registers, and for fp32 caches by LDS: 96 KiB
// at D = 128, 48 at 64), and what a tile of one takes of a full CU's time, in those of
// eight waves (measured, 2048 tokens behind 8192, 16 / 8 heads, us in workgroups of eight
// and four waves: bf16, D = 128 169 / 276, 64 100 / 132; fp32 cache 803 / 1178, 410 / 469; fp32
// over a bf16 cache 413 / 402, 273 / 218, so in four waves always), and where no CU has
// more than one.
struct Kind {
    int per_cu;
    double tile, alone;
};
Kind kind_of(bool q16, sa_dtype kv, int d, int waves) {
    if (q16 && d == 64) return waves == 8 ? Kind{2, 1.0, 1.2} : Kind{2, 0.66, 0.78};
    if (q16) return waves == 8 ? Kind{1, 1.0, 1.0} : Kind{2, 0.82, 0.7};
    if (kv != SA_DTYPE_F32) return d == 64 ? Kind{3, 0.5, 0.9} : Kind{2, 0.5, 0.6};
    if (d == 64) return waves == 8 ? Kind{2, 1.0, 1.2} : Kind{3, 0.57, 1.0};
    return waves == 8 ? Kind{1, 1.0, 1.0} : Kind{1, 0.73, 0.73};
}

template <auto KERNEL>
sa_status launch_blocks(const BlockArgs& a, int waves, int items, int lds, hipStream_t st) {
    SA_TRY(pf::opt_in_lds<KERNEL>(lds));
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)items * a.n_kv), dim3(waves * kWave), lds, st, a);
    SA_CHECK_LAUNCH();
    return SA_OK;
}
template <int D, int KV>
sa_status launch_f32(const BlockArgs& a, int waves, int items, hipStream_t st) {
    constexpr int lds = 2 * TermGeo<D, KV>::STAGE;
    if constexpr (KV == SA_DTYPE_F32)
        if (waves == 8)
            return a.even ? launch_blocks<extend_f32_kernel<D, 8, KV, true>>(a, 8, items, lds, st)
                          : launch_blocks<extend_f32_kernel<D, 8, KV, false>>(a, 8, items, lds, st);
    return a.even ? launch_blocks<extend_f32_kernel<D, 4, KV, true>>(a, 4, items, lds, st)
                  : launch_blocks<extend_f32_kernel<D, 4, KV, false>>(a, 4, items, lds, st);
}
template <int D, bool FP8>
sa_status launch_bf16(const BlockArgs& a, int waves, int items, hipStream_t st) {
    constexpr int lds = 2 * BfGeo<D>::STAGE;
    return waves == 8 ? launch_blocks<extend_bf16_kernel<D, 8, FP8>>(a, 8, items, lds, st)
                      : launch_blocks<extend_bf16_kernel<D, 4, FP8>>(a, 4, items, lds, st);
}
template <int D>
sa_status dispatch_blocks(const BlockArgs& a, sa_dtype kv, bool q16, int waves, int items, bool merge, long long rows,
                          hipStream_t st) {
    if (q16) SA_TRY(kv == SA_DTYPE_FP8 ? (launch_bf16<D, true>(a, waves, items, st))
                                       : (launch_bf16<D, false>(a, waves, items, st)));
    else SA_TRY(kv == SA_DTYPE_F32    ? (launch_f32<D, SA_DTYPE_F32>(a, waves, items, st))
                : kv == SA_DTYPE_BF16 ? (launch_f32<D, SA_DTYPE_BF16>(a, waves, items, st))
                                      : (launch_f32<D, SA_DTYPE_FP8>(a, waves, items, st)));
    if (!merge) return SA_OK;
    return merge_rows<D>(rows, [&](dim3 grid, long long row0) {
        if (q16) hipLaunchKernelGGL((block_merge_kernel<D, uint16_t, false>), grid, dim3(256), 0, st, a, row0, rows);
        else if (a.even) hipLaunchKernelGGL((block_merge_kernel<D, float, true>), grid, dim3(256), 0, st, a, row0, rows);
        else hipLaunchKernelGGL((block_merge_kernel<D, float, false>), grid, dim3(256), 0, st, a, row0, rows);
    });
}

long long blocks_of(long long rows, int block) { return (rows + block - 1) / block; }

}  // namespace

// Blocks for sequences of kBlockRows query rows of a KV head, where a call has enough
// of them: below it the rows' launch with its smaller pieces is quicker.  us, rows /
// blocks, 16 / 8 heads of 128, queries and cache bf16: 256 rows over 1128 keys 19.6 / 20.7,
// 512 over 1256 31.6 / 24.7, 64 over 8032 36.1 / 29.8, 768 over 384 15.0 / 17.3; fp32 (always
// blocks): 64 over 32 13.2 / 6.8, over 1032 22.0 / 19.0; 32 sequences of 32 rows over 2016
// 116 / 146.  Other sequences join the blocks where they cost an eighth of them at most,
// which saves their launches.
void split_chunks(sa_dtype kv, int rep, int n_kv, const ChunkSeq* seqs, int n, std::vector<ChunkSeq>* many,
                  std::vector<ChunkSeq>* few) {
    constexpr long long kBlockRows = 64, kBlockWork = 3000000, kJoinRows = 256 / 8;
    long long work = 0, others = 0;   // query rows x keys; keys
    for (int i = 0; i < n; ++i) {
        const long long rows = (long long)seqs[i].n * rep, keys = (long long)seqs[i].len + seqs[i].n;
        if (rows >= kBlockRows) work += rows * keys;
        else others += keys;
    }
    const bool blocks = work > 0 && (kv == SA_DTYPE_F32 || work * n_kv >= kBlockWork), join = others * kJoinRows <= work;
    for (int i = 0; i < n; ++i)
        (blocks && (join || (long long)seqs[i].n * rep >= kBlockRows) ? many : few)->push_back(seqs[i]);
}

namespace {

// The parts of several sequences by their lengths, so that the last to begin are the
// shortest: seven chunks of 1 - 700 tokens over 8 bits 137 -> 130 us, eight of 100 - 1000
// behind up to 16000, bf16, 16 / 8 heads of 64 393 -> 285.  The search costs 0.6 us.
void sort_parts(BlockArgs& a, long long* items) {
    struct Rest { int tiles, block; } rest[kSortedBlocks];
    int k = 0, n_rest = 0;
    long long full = 0, blocks = 0;
    for (int i = 0; i < a.n_seq; ++i) blocks += blocks_of((long long)a.seq[i].n * a.rep, a.rows);
    if (blocks > kSortedBlocks) return;
    int32_t start[kRowsPerLaunch];
    for (int i = 0; i < a.n_seq; ++i) {
        start[i] = k;
        for (int b = (int)blocks_of((long long)a.seq[i].n * a.rep, a.rows) - 1; b >= 0; --b, ++k) {
            const int tiles = block_key_tiles(a.seq[i], b, a.rows, a.rep, a.tile);
            a.full_at[k] = (uint16_t)full;
            full += tiles / a.tiles;
            if (full > 0xffff) return;
            if (tiles % a.tiles) rest[n_rest++] = {tiles % a.tiles, k};
        }
    }
    a.full_at[k] = (uint16_t)full;
    std::sort(rest, rest + n_rest, [](const Rest& x, const Rest& y) {
        return x.tiles != y.tiles ? x.tiles > y.tiles : x.block < y.block;
    });
    for (int r = 0; r < n_rest; ++r) a.rest[r] = (uint8_t)rest[r].block;
    std::copy(start, start + a.n_seq, a.start);
    a.n_blocks = k;
    a.full = (int)full;
    *items = full + n_rest;
}

}  // namespace

size_t extend_blocks_ws(int n, const int32_t* counts, int n_q, int n_kv, int d, long long max_tokens) {
    const long long tiles = (max_tokens + kTermTile - 1) / kTermTile;
    if (tiles <= 1) return 0;
    long long rows = 0;
    for (int i = 0; i < n; ++i) rows += (long long)counts[i] * n_q;
    // at most as many workgroups as extend_blocks cuts into
    return (size_t)std::min(rows * tiles, kMaxRounds * device_cu_count() * 256LL) * (d + 2) * sizeof(float);
}

sa_status extend_blocks(const PagedView& c, const void* q, bool q16, int n_q, const ChunkSeq* seqs, int n, float scale,
                        void* out, void* ws, size_t ws_bytes, hipStream_t st) {
    BlockArgs a{};
    a.q = q; a.out = out;
    a.k = c.k_pool; a.v = c.v_pool; a.k_scale = c.k_scale; a.v_scale = c.v_scale; a.table = c.block_table;
    a.n_kv = c.n_kv; a.n_q = n_q; a.rep = n_q / c.n_kv;
    a.max_pages = c.max_pages; a.num_pages = c.num_pages;
    a.factor = scale * pf::kLog2eP;
    a.sl2 = std::fabs(a.factor);
    a.q_sign = scale < 0 ? 0x80008000u : 0u;
    for (int i0 = 0; i0 < n; i0 += kRowsPerLaunch) {
        a.n_seq = std::min(kRowsPerLaunch, n - i0);
        long long most = 0;
        for (int i = 0; i < a.n_seq; ++i) {
            a.seq[i] = seqs[i0 + i];
            most = std::max(most, (long long)a.seq[i].n * a.rep);
        }
        a.tile = q16 ? kBfTile : kTermTile;
        const int per_wave = q16 ? 32 : 16;
        int longest = 1;
        auto last_tiles = [&](int i) {
            const int last = (int)blocks_of((long long)a.seq[i].n * a.rep, a.rows) - 1;
            return block_key_tiles(a.seq[i], last, a.rows, a.rep, a.tile);
        };
        auto parts_of = [&](int i, int tiles) { return (last_tiles(i) + tiles - 1) / tiles; };
        auto workgroups = [&](int tiles) {
            long long k = 0;
            for (int i = 0; i < a.n_seq; ++i) k += blocks_of((long long)a.seq[i].n * a.rep, a.rows) * parts_of(i, tiles);
            return k * a.n_kv;
        };
        // Eight or four waves, and the tiles of a workgroup: what is estimated cheapest, in
        // tiles of a workgroup of eight waves on a CU of its own.
        const long long cus = device_cu_count();
        const int cut = q16 ? (c.d == 128 ? kCutBf16 : kCutBf16Narrow) : c.kv == SA_DTYPE_F32 ? kCutF32 : kCutTerms;
        const bool terms = !q16 && c.kv != SA_DTYPE_F32;   // in four waves always
        int waves = 8;
        double best = INFINITY;
        a.even = 0;
        long long rows_all = 0;
        int keys = 0;
        for (int i = 0; i < a.n_seq; ++i) {
            rows_all += (long long)a.seq[i].n * n_q;
            keys = std::max(keys, a.seq[i].len + a.seq[i].n);
        }
        // extend_blocks_ws's rows
        const long long room = std::min(rows_all * ((keys + kTermTile - 1) / kTermTile), kMaxRounds * cus * 256);
        for (int w = 8; w >= 4; w -= 4) {
            if (w == 8 && (most <= 4 * per_wave || terms)) continue;
            a.rows = w * per_wave;
            longest = 1;
            const Kind kind = kind_of(q16, c.kv, c.d, w);
            // a sequence's blocks by four of them
            struct Some { double blocks; int tiles; } some[4 * kRowsPerLaunch];
            int n_some = 0;
            double work = 0.0;
            for (int i = 0; i < a.n_seq; ++i) {
                longest = std::max(longest, last_tiles(i));
                const int blocks = (int)blocks_of((long long)a.seq[i].n * a.rep, a.rows), k = std::min(blocks, 4);
                for (int j = 0; j < k; ++j) {
                    const int b = (int)((2LL * j + 1) * blocks / (2 * k));
                    some[n_some] = {(double)blocks / k * a.n_kv, block_key_tiles(a.seq[i], b, a.rows, a.rep, a.tile)};
                    work += some[n_some].blocks * some[n_some].tiles;
                    ++n_some;
                }
            }
            for (int p = 1, t = 0; p <= longest; ++p) {
                if (t == (longest + p - 1) / p) continue;
                t = (longest + p - 1) / p;
                const double wgs = (double)workgroups(t), slots = (double)(kind.per_cu * cus);
                if (p > 1 && wgs > kMaxRounds * cus) break;
                // Parts of more than half of t in rounds (no two in one's time), or all of the work
                // evenly, whichever is longer.
                double big = 0.0, big_tiles = 0.0;
                for (int j = 0; j < n_some; ++j) {
                    const int whole = some[j].tiles / t, rest = some[j].tiles % t;
                    const bool more = 2 * rest > t;
                    big += some[j].blocks * (whole + more);
                    big_tiles += some[j].blocks * ((double)whole * t + (more ? rest : 0));
                }
                const double rounds = big > 0.0 ? std::ceil(big / slots) * (big_tiles / big) : 0.0;
                const double tile = wgs > cus ? kind.per_cu * kind.tile : kind.alone;
                const double cost = (std::max({rounds, work / slots, (double)t}) +
                                     (p > 1 ? cut : kWholeTiles) * std::max(1.0, wgs / slots)) * tile;
                if (cost < best) best = cost, waves = w, a.tiles = t, a.even = 0;
            }
            // All blocks' tiles in a row, cut evenly.
            long long blocks = 0, total = 0;
            for (int i = 0; i < a.n_seq; ++i) blocks += blocks_of((long long)a.seq[i].n * a.rep, a.rows);
            if (q16 || blocks > kSortedBlocks || (w == 8 && c.d == 64)) continue;
            for (int i = 0; i < a.n_seq; ++i)
                for (int b = 0, k = (int)blocks_of((long long)a.seq[i].n * a.rep, a.rows); b < k; ++b)
                    total += block_key_tiles(a.seq[i], b, a.rows, a.rep, a.tile);
            for (int per : {kind.per_cu, 1}) {
                const long long most_wgs = std::min(total, per * cus / a.n_kv);
                if (most_wgs < 1) continue;
                const int t = (int)((total + most_wgs - 1) / most_wgs);
                const long long wgs = (total + t - 1) / t;
                if (2 * wgs * a.rows * a.n_kv > room) continue;
                const double cost = (t + cut + (terms ? kNextTerms : kNextF32) * (double)blocks / wgs) *
                                    (wgs * a.n_kv > cus ? kind.per_cu * kind.tile : kind.alone);
                if (cost < best) best = cost, waves = w, a.even = t;
            }
        }
        a.rows = waves * per_wave;
        long long at = 0, parts = 0;
        if (a.even) {
            int k = 0, sum = 0;
            for (int i = 0; i < a.n_seq; ++i) {
                a.start[i] = k;
                for (int b = (int)blocks_of((long long)a.seq[i].n * a.rep, a.rows) - 1; b >= 0; --b) {
                    a.block_at[k++] = sum;
                    sum += block_key_tiles(a.seq[i], b, a.rows, a.rep, a.tile);
                }
            }
            a.start[a.n_seq] = a.n_blocks = k;
            a.block_at[k] = sum;
            at = (sum + a.even - 1) / a.even;
            parts = 2 * at * a.rows;
        }
        if (!a.even) a.n_blocks = 0;
        for (int i = 0; i < a.n_seq && !a.even; ++i) {
            a.parts[i] = parts_of(i, a.tiles);
            a.start[i] = (int)at;
            a.base[i] = (int)parts;
            at += blocks_of((long long)a.seq[i].n * a.rep, a.rows) * a.parts[i];
            if (a.parts[i] > 1) parts += (long long)a.parts[i] * a.seq[i].n * a.rep;
        }
        if (!a.even) a.start[a.n_seq] = (int)at;
        if (!a.even && a.n_seq > 1) sort_parts(a, &at);
        const long long tokens = a.seq[a.n_seq - 1].first + a.seq[a.n_seq - 1].n - a.seq[0].first;
        // a grid has fewer than 2^32 threads
        if (at * a.n_kv >= (1LL << 32) / (waves * kWave) || parts > 0x7fffffffLL)
            return fail(SA_EINVAL, "too many tokens for one call");
        if (parts) {
            const size_t need = (size_t)parts * a.n_kv * (c.d + 2) * sizeof(float);
            if (!ws || ws_bytes < need) return fail(SA_ENOMEM, "workspace too small for the partials");
            a.part_o = static_cast<float*>(ws);
            a.part_ml = a.part_o + (size_t)parts * a.n_kv * c.d;
        }
        SA_TRY(c.d == 64 ? dispatch_blocks<64>(a, c.kv, q16, waves, (int)at, parts > 0, tokens * n_q, st)
                         : dispatch_blocks<128>(a, c.kv, q16, waves, (int)at, parts > 0, tokens * n_q, st));
    }
    return SA_OK;
}

}  // namespace sa
