// Causal prefill attention with a sliding window and sinks on gfx950 MFMA.
//
// Query i sees key j <= i when i - j < window or j < n_sink.  A workgroup
// serves a tile of consecutive queries of the heads that share a KV head and
// walks the key tiles that some query of it sees: those of the sinks that lie
// before the window, then those from the window's start of its first query to
// its last query.  Scores are computed transposed, S^T = K Q^T, so that a lane
// owns one query column and the weights come out as the operand of O^T += V^T
// P^T; softmax runs in the log2 domain with a running max that is raised only
// when a lane's sum of weights exceeds kRaiseAt (every weight is then below
// it, and relative errors do not depend on it).  A tile that every query of a
// wave sees whole takes no mask; one that none sees is skipped.
//
// bf16: v_mfma_f32_32x32x16_bf16, a wave owns 32 queries, tiles of 64 keys
// loaded straight into LDS one tile ahead.  q enters as given and the scale is
// applied to the fp32 scores, so the roundings are P to bf16 (2^-9 of each
// weight, the sums taken of the rounded ones) and the output's.
//
// fp32: every operand as the exact sum of three bf16 terms, of whose products
// the six largest are taken (what is left out is below 2^-24 of the product),
// v_mfma_f32_16x16x32_bf16; a wave owns 16 queries, tiles of 32 keys are split
// into terms on their way into LDS.
//
// A hidden key's weight of 0 makes NaN of an infinite or NaN value, and a split
// makes NaN of an infinity: rows whose sums are not finite are computed anew over
// the keys that they see (plain_row.h).
//
// Bound: MFMA, with the softmax between.  16 / 8 heads of 128: 8192 queries,
// window 1024, 4 sinks, bf16 87 us (64.7 GF of visible products, 0.74 PFLOP/s;
// at a large product's rate 40): two rounds of a workgroup per CU, whose queries,
// first tile and stores nothing covers.  2048 queries, window 512, fp32 54.6 us (7.6
// GF, six products each: 0.83 PFLOP/s; 28): every key is split by each query tile
// that sees it.  3 prompts of 777, window 200, 16 / 4 heads of 64, bf16 10.4 us: a
// launch and a wave's chain of five tiles.
#include <algorithm>
#include <cmath>

#include "bf16_terms.h"
#include "plain_row.h"
#include "prefill_shared.h"

namespace sa {
namespace {

using pf::f32x16_t;
using pf::lds_s16x4_t;
using pf::lds_u8_t;
using pf::s16x4_t;

constexpr float kRaiseAt = 65536.f;

struct WindowArgs : pf::PrefillArgs {
    void* dst;        // the output, in the inputs' type
    int window, sink;
};

// The key tiles of KT keys that queries [q0, q1] see: ns tiles from 0 on, then
// n - ns from w0 on.
struct TileList {
    int ns, w0, n;
    __device__ __forceinline__ int operator()(int i) const { return i < ns ? i : w0 + i - ns; }
};
template <int KT>
__device__ __forceinline__ TileList tile_list(const WindowArgs& a, int q0, int q1) {
    TileList t;
    t.w0 = max(0, q0 - a.window + 1) / KT;   // window <= L, so nothing overflows
    t.ns = min((a.sink + KT - 1) / KT, t.w0);
    t.n = t.ns + q1 / KT - t.w0 + 1;
    return t;
}
// How queries [q0, q1] see keys [k0, k1]: none of them, all of them, or a part.
enum Seen { kNone, kAll, kSome };
__device__ __forceinline__ Seen seen(const WindowArgs& a, int q0, int q1, int k0, int k1) {
    if (k0 > q1 || (q0 - k1 >= a.window && k0 >= a.sink)) return kNone;
    if (k1 <= q0 && (q1 - k0 < a.window || k1 < a.sink)) return kAll;
    return kSome;
}
__device__ __forceinline__ bool hidden(const WindowArgs& a, int q, int k) {
    return k > q || (q - k >= a.window && k >= a.sink);
}

// Query row `row` of the workgroup's head h0 + dh without matrix instructions, one
// wave.  The launch's arguments (the kernel's first) are read anew, so that no
// register holds them until here.
template <int D, class T>
__device__ __forceinline__ void window_plain(int dh, int row) {
    const int lane = threadIdx.x & (kWave - 1);
    auto args = (const __attribute__((address_space(4))) WindowArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    int block = blockIdx.x;
    asm volatile("" : "+s"(args), "+s"(block));
    const WindowArgs& a = *(const WindowArgs*)args;
    const float factor = a.q_sign ? -a.sl2 : a.sl2;   // bf16: the sign went to q
    const pf::Work wk = pf::map_work(a, block);
    const T* Q = static_cast<const T*>(a.q) + wk.b * a.qs[0] + (wk.h0 + dh) * a.qs[1];
    const T* K = static_cast<const T*>(a.k) + wk.b * a.kvs[0] + wk.kvh * a.kvs[1];
    const T* V = static_cast<const T*>(a.v) + wk.b * a.kvs[0] + wk.kvh * a.kvs[1];
    T* out = static_cast<T*>(a.dst) + wk.b * a.os[0] + (wk.h0 + dh) * a.os[1];
    const int from = max(0, row - a.window + 1);
    PlainRow<D> p;
    auto span = [&](int k0, int k1) {
        for (int k = k0; k < k1 && !p.lost(); k += kWave)
            p.keys(min(kWave, k1 - k), Q + row * a.qs[2], factor, [&](int i) { return K + (k + i) * a.kvs[2]; },
                   [&](int i) { return V + (k + i) * a.kvs[2]; });
    };
    span(0, min(a.sink, from));
    span(from, row + 1);
#pragma unroll
    for (int e = 0; e < p.E; ++e) {
        const float v = p.o[e] / p.l;
        if constexpr (sizeof(T) == 2) out[row * a.os[2] + lane * p.E + e] = f32_to_bf16_rne(v);
        else out[row * a.os[2] + lane * p.E + e] = v;
    }
}

// pf::dma16 with a uniform base and a byte offset per lane.
__device__ __forceinline__ void dma16_from(const void* base, uint32_t off, lds_u8_t* dst) {
    const uint32_t m = static_cast<uint32_t>(reinterpret_cast<size_t>(dst));
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m)
                 : "memory", "m0");
}

// ---------------------------------------------------------------- bf16

constexpr int kBfTile = 64;

template <int D>
struct BfGeo {
    static constexpr int ROWB = 2 * D;
    static constexpr int CPR = ROWB / 16;               // 16-byte chunks of a row
    static constexpr int RPL = kWave / CPR;             // rows per wave load
    static constexpr int NL = kBfTile / RPL;            // wave loads per tensor and tile
    static constexpr int HALF = kBfTile * ROWB;
    static constexpr int STAGE = 2 * HALF;              // K, then V
    static constexpr int NKS = D / 16, NDB = D / 32;
    // Chunk c of row r sits at c ^ swz(r): the K fragment reads (16 rows, one
    // chunk) and the V transpose reads (4 rows, 4 chunks) of a cycle fall on
    // different banks.
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (CPR == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
        else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    }
};

template <int D>
struct BfWave {
    using G = BfGeo<D>;
    int n, hh, q0;
    bf16x8_t qf[G::NKS];
    f32x16_t acc[G::NDB];
    float m, nm, l, cap;   // running max, -m once finite (else 0), this lane's part of the sum, raise bound
    float c;               // |scale| log2(e)
    // Where this lane's fragments start in a half tile.  Chunk numbers meet the
    // rows' permutation by exclusive or, so fragment ks of K is at k_at ^ 32 ks, and
    // that of d block db of V at v_at ^ 64 db: one instruction, and no register each.
    int k_at, v_at[2];

    __device__ __forceinline__ void init(const WindowArgs& a, const uint16_t* Q, int q_first, int lane) {
        n = lane & 31;
        hh = lane >> 5;
        q0 = q_first;
        c = a.sl2;
        const uint16_t* row = Q + min(q0 + n, a.L - 1) * a.qs[2] + 8 * hh;
#pragma unroll
        for (int ks = 0; ks < G::NKS; ++ks) {
            u32x4_t raw = *reinterpret_cast<const u32x4_t*>(row + ks * 16);
            raw ^= a.q_sign;
            qf[ks] = __builtin_bit_cast(bf16x8_t, raw);
        }
#pragma unroll
        for (int db = 0; db < G::NDB; ++db) acc[db] = f32x16_t{};
        m = -INFINITY;
        nm = 0.f;
        l = 0.f;
        cap = -1.f;
        const int r = pf::swap_bits23(n);
        k_at = r * G::ROWB + ((hh ^ G::swz(r & 15)) << 4);
        const int g = lane >> 4, j = lane & 15;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int vr = 8 * hh + 4 * u + j / 4;
            v_at[u] = vr * G::ROWB + (((2 * (g & 1) + ((j & 3) >> 1)) ^ G::swz(vr & 15)) << 4) + (j & 1) * 8;
        }
    }

    // Scores times c (first: -inf times a factor of 0 would be NaN), those of keys
    // that this lane's query does not see -inf.  Element j is key base + 16 (j / 8)
    // + j % 8, so that all comparisons are with constants.
    __device__ __forceinline__ void hide(const WindowArgs& a, int k0, int q1, f32x16_t& s) const {
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] *= c;
        const int base = k0 + 8 * hh, q = q0 + n;
        if (k0 + 31 > q0) {                       // some query lies before some key
            const int last = q - base;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (16 * (j / 8) + j % 8 > last) s[j] = -INFINITY;
        }
        if (q1 - k0 >= a.window) {                // some key lies before some query's window
            const int first = q - a.window + 1 - base, sink = a.sink - base;
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (16 * (j / 8) + j % 8 < first && 16 * (j / 8) + j % 8 >= sink) s[j] = -INFINITY;
        }
    }

    // hb, the half's K rows, is a multiple of 256 bytes into LDS.
    __device__ __forceinline__ bf16x8_t k_frag(uint32_t hb, int ks) const {
        return *reinterpret_cast<const __attribute__((address_space(3))) bf16x8_t*>((hb + k_at) ^ (ks << 5));
    }
    __device__ __forceinline__ bf16x8_t v_frag(uint32_t hb, int db, int t) const {
        const uint32_t more = G::HALF + t * 16 * G::ROWB;
        const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(((hb + v_at[0]) ^ (db << 6)) + more));
        const s16x4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(((hb + v_at[1]) ^ (db << 6)) + more));
        return __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    }

    // The weights of 32 scores as two operands of P V, and their part of the row
    // sum; raises the running max where needed (rescaling O and the sum).
    template <bool MASK>
    __device__ __forceinline__ void softmax(const f32x16_t& s, bf16x8_t (&pb)[2]) {
        float p[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) p[j] = __builtin_amdgcn_exp2f(MASK ? s[j] + nm : fmaf(s[j], c, nm));
        pb[0] = pf::pack_bf16x8(p);
        pb[1] = pf::pack_bf16x8(p + 8);
        float sum = pf::sum_bf16x8(pb[1], 0.f) + pf::sum_bf16x8(pb[0], 0.f);
        if (__any(!(sum <= cap))) {
            float mt = s[0];
#pragma unroll
            for (int j = 1; j < 16; ++j) mt = fmaxf(mt, s[j]);
            if constexpr (!MASK) mt *= c;
            mt = fmaxf(mt, xor32(mt));
            const float m_new = fmaxf(m, mt);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
#pragma unroll
            for (int db = 0; db < G::NDB; ++db) acc[db] *= alpha;
            l *= alpha;
            m = m_new;
            nm = m_new == -INFINITY ? 0.f : -m_new;
            cap = m_new == -INFINITY ? -1.f : kRaiseAt;
#pragma unroll
            for (int j = 0; j < 16; ++j) p[j] = __builtin_amdgcn_exp2f(MASK ? s[j] + nm : fmaf(s[j], c, nm));
            pb[0] = pf::pack_bf16x8(p);
            pb[1] = pf::pack_bf16x8(p + 8);
            sum = pf::sum_bf16x8(pb[1], 0.f) + pf::sum_bf16x8(pb[0], 0.f);
        }
        l += sum;
    }

    // The 32 keys from k0 on, their K rows at hb.
    template <bool MASK>
    __device__ __forceinline__ void half(const WindowArgs& a, int k0, int q1, uint32_t hb) {
        f32x16_t s = {};
#pragma unroll
        for (int ks = 0; ks < G::NKS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(hb, ks), qf[ks], s, 0, 0, 0);
        if constexpr (MASK) hide(a, k0, q1, s);
        bf16x8_t pb[2];
        softmax<MASK>(s, pb);
#pragma unroll
        for (int db = 0; db < G::NDB; ++db)
#pragma unroll
            for (int t = 0; t < 2; ++t)
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v_frag(hb, db, t), pb[t], acc[db], 0, 0, 0);
    }

    // O / l: every lane's columns into the wave's part of LDS (chunks of a row
    // permuted as the tiles' are), then rows of 16-byte pieces to memory.  Returns
    // the rows, a bit each, that are not finite and not written.
    __device__ __forceinline__ uint32_t store(uint16_t* head, long long row, int L, lds_u8_t* buf, int lane) const {
        const float inv = 1.0f / (l + xor32(l));
        const bf16x2_t one = {(__bf16)1.0f, (__bf16)1.0f};
        float sum[4] = {};   // of the outputs: finite where they are
#pragma unroll
        for (int db = 0; db < G::NDB; ++db)
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                const f32x2_t x = {acc[db][4 * jj] * inv, acc[db][4 * jj + 1] * inv};
                const f32x2_t y = {acc[db][4 * jj + 2] * inv, acc[db][4 * jj + 3] * inv};
                const bf16x2_t bx = __builtin_convertvector(x, bf16x2_t), by = __builtin_convertvector(y, bf16x2_t);
                sum[jj] = __builtin_amdgcn_fdot2_f32_bf16(bx, one, sum[jj], false);
                sum[jj] = __builtin_amdgcn_fdot2_f32_bf16(by, one, sum[jj], false);
                *reinterpret_cast<__attribute__((address_space(3))) uint64_t*>(
                    buf + n * G::ROWB + (((4 * db + jj) ^ G::swz(n & 15)) << 4) + 8 * hh) =
                    (uint64_t)__builtin_bit_cast(uint32_t, by) << 32 | __builtin_bit_cast(uint32_t, bx);
            }
        const uint64_t bad = __ballot(q0 + n < L && !(fabsf((sum[0] + sum[1]) + (sum[2] + sum[3])) < INFINITY));
        const uint32_t anew = (uint32_t)bad | (uint32_t)(bad >> 32);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // a wave's own part: no barrier
#pragma unroll
        for (int i = 0; i < 32 / G::RPL; ++i) {
            const int r = i * G::RPL + lane / G::CPR, ch = lane % G::CPR;
            const u32x4_t v = *reinterpret_cast<const __attribute__((address_space(3))) u32x4_t*>(
                buf + r * G::ROWB + ((ch ^ G::swz(r & 15)) << 4));
            if (q0 + r < L && !(anew >> r & 1)) *reinterpret_cast<u32x4_t*>(head + (q0 + r) * row + 8 * ch) = v;
        }
        return anew;
    }
};

// W waves: W / gh query blocks of 32 for each of gh heads.  Eight at D = 64: the registers
// of four waves per SIMD, two workgroups of eight per CU.
template <int D, int W>
__global__ void __launch_bounds__(W * kWave, W == 8 && D == 64 ? 4 : 1) window_bf16_kernel(WindowArgs a) {
    using G = BfGeo<D>;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    lds_u8_t* const smem = (lds_u8_t*)smem_raw;
    const uint32_t lds_at = static_cast<uint32_t>(reinterpret_cast<size_t>(smem));
    const pf::Work wk = pf::map_work(a, blockIdx.x);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int wph = W / a.gh;
    const int h = wk.h0 + wave / wph;
    const uint16_t* Q = static_cast<const uint16_t*>(a.q) + wk.b * a.qs[0] + h * a.qs[1];
    const uint16_t* K = static_cast<const uint16_t*>(a.k) + wk.b * a.kvs[0] + wk.kvh * a.kvs[1];
    const uint16_t* V = static_cast<const uint16_t*>(a.v) + wk.b * a.kvs[0] + wk.kvh * a.kvs[1];
    const int q_first = wk.qt * wph * 32, q_last = min(a.L, q_first + wph * 32) - 1;
    const TileList tiles = tile_list<kBfTile>(a, q_first, q_last);

    // Load i of a wave copies RPL rows, this lane's 16 bytes of them at off[i] from
    // the tile's first row; rows past the sequence repeat its last.
    constexpr int NI = G::NL / W > 0 ? G::NL / W : 1;
    const int row_bytes = (int)a.kvs[2] * 2;
    int row[NI], col[NI];
    uint32_t off[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        row[i] = (wave * NI + i) * G::RPL + lane / G::CPR;
        col[i] = 16 * ((lane % G::CPR) ^ G::swz(row[i] & 15));
        off[i] = row[i] * row_bytes + col[i];
    }
    auto load = [&](int it) {
        if (G::NL < W && wave >= G::NL) return;
        const int k0 = tiles(it) * kBfTile;
        const uint16_t* kt = K + k0 * a.kvs[2];
        const uint16_t* vt = V + k0 * a.kvs[2];
        lds_u8_t* dst = smem + (it & 1) * G::STAGE;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            uint32_t o = off[i];
            if (k0 + kBfTile > a.L) o = min(row[i], a.L - 1 - k0) * row_bytes + col[i];
            dma16_from(kt, o, dst + (wave * NI + i) * 1024);
            dma16_from(vt, o, dst + G::HALF + (wave * NI + i) * 1024);
        }
    };
    load(0);
    BfWave<D> w;
    w.init(a, Q, q_first + (wave % wph) * 32, lane);
    const int q1 = min(w.q0 + 31, a.L - 1);
    if (tiles.n > 1) {
        load(1);
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NI) : "memory");   // tile 0
    } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    // Tile it has been computed by every wave: its stage takes tile it + 2.
    auto end_tile = [&](int it) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (it + 2 < tiles.n) load(it + 2);
    };
    // A tile whose halves a wave's queries see whole, in part or not at all.
    auto edge_tile = [&](int it) {
        const int k0 = tiles(it) * kBfTile;
        const uint32_t sb = lds_at + (it & 1) * G::STAGE;
        if (w.q0 < a.L) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const int k = k0 + 32 * kb;
                const Seen sn = seen(a, w.q0, q1, k, k + 31);
                if (sn == kAll) w.template half<false>(a, k, q1, sb + kb * 32 * G::ROWB);
                else if (sn == kSome) w.template half<true>(a, k, q1, sb + kb * 32 * G::ROWB);
            }
        }
        end_tile(it);
    };
    int it = 0;
    if constexpr (W == 8) {
        // The tiles that every query of the workgroup sees whole, in ping-pong:
        // waves w and w + 4 share a SIMD, and each half tile is a block of MFMAs
        // (the half before's P V, this half's scores) and a softmax.  Waves 4 - 7
        // take the half's barrier between the two, waves 0 - 3 behind both, so that
        // on every SIMD one wave's softmax runs under the other's MFMAs (8192
        // queries, window 1024, when written: 90 us against 96 with all tiles as edge
        // tiles; 103 with all tiles in this loop, whose masks then cost it registers).
        const int lo = min(tiles.n, tiles.ns + max(0, (q_last - a.window + kBfTile) / kBfTile - tiles.w0));
        const int hi = tiles.ns + (q_first + 1) / kBfTile - tiles.w0;
        for (; it < lo; ++it) edge_tile(it);
        if (lo < hi) {
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
            for (; it < hi; ++it) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const uint32_t hb = lds_at + (it & 1) * G::STAGE + kb * 32 * G::ROWB;
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
                        else end_tile(it);
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
    for (; it < tiles.n; ++it) edge_tile(it);
    // The output through LDS, 32 rows per wave, so that stores are whole rows.
    uint32_t anew = w.store(static_cast<uint16_t*>(a.dst) + wk.b * a.os[0] + h * a.os[1], a.os[2], a.L,
                            smem + wave * 32 * G::ROWB, lane);
    for (; anew; anew &= anew - 1)
        window_plain<D, uint16_t>(wave / wph, w.q0 + __builtin_ctz(anew));
}

// ---------------------------------------------------------------- fp32

constexpr int kF32Tile = 32;

template <int D>
struct F32Geo {
    static constexpr int ROWB = 2 * D;                  // a row of one term
    static constexpr int TERM = kF32Tile * ROWB;        // one term of K or V
    static constexpr int STAGE = 6 * TERM;              // K terms 0 - 2, V terms 0 - 2
    static constexpr int CPR = ROWB / 16;
    static constexpr int KS = D / 32, DB = D / 16;
    // Chunk c of row r at c ^ swz(r): rows 8a + 4kb + b of a K fragment read and
    // rows 8g + 4u + b of a half wave's V^T read on different banks.
    static __device__ __forceinline__ int swz(int r) {
        if constexpr (CPR == 16) return ((r & 3) << 2) | (((r >> 3) & 1) << 1) | ((r >> 4) & 1);
        else return (((r >> 1) & 1) << 2) | (((r >> 3) & 1) << 1) | ((r >> 4) & 1);
    }
    static __device__ __forceinline__ int off(int r, int c) { return r * ROWB + ((c ^ swz(r)) << 4); }
};

constexpr int kPairs = 6;
__host__ __device__ constexpr int pair_a(int pr) { return pr == 2 || pr == 4 ? 1 : pr == 5 ? 2 : 0; }
__host__ __device__ constexpr int pair_b(int pr) { return pr == 1 || pr == 4 ? 1 : pr == 3 ? 2 : 0; }

template <int D, int W>
__global__ void __launch_bounds__(W * kWave) window_f32_kernel(WindowArgs a) {
    using G = F32Geo<D>;
    constexpr int NT = W * kWave;
    constexpr int C8 = D / 8;                           // 8-element pieces of a row
    constexpr int NC = kF32Tile * C8 / NT > 0 ? kF32Tile * C8 / NT : 1;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    lds_u8_t* const smem = (lds_u8_t*)smem_raw;
    const pf::Work wk = pf::map_work(a, blockIdx.x);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r16 = lane & 15, g = lane >> 4;
    const int wph = W / a.gh;
    const int h = wk.h0 + wave / wph;
    const float* Q = static_cast<const float*>(a.q) + wk.b * a.qs[0] + h * a.qs[1];
    const float* K = static_cast<const float*>(a.k) + wk.b * a.kvs[0] + wk.kvh * a.kvs[1];
    const float* V = static_cast<const float*>(a.v) + wk.b * a.kvs[0] + wk.kvh * a.kvs[1];
    const int q_first = wk.qt * wph * 16, q_last = min(a.L, q_first + wph * 16) - 1;
    const TileList tiles = tile_list<kF32Tile>(a, q_first, q_last);

    // ---- tiles: fp32 in registers one tile ahead, three bf16 terms in LDS ----
    const bool loads = kF32Tile * C8 >= NT || threadIdx.x < kF32Tile * C8;
    f32x4_t sk[NC][2], sv[NC][2];
    auto load = [&](int it) {
        if (!loads) return;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int idx = threadIdx.x + i * NT;
            const long long e = (long long)min(tiles(it) * kF32Tile + idx / C8, a.L - 1) * a.kvs[2] + 8 * (idx % C8);
            sk[i][0] = *reinterpret_cast<const f32x4_t*>(K + e);
            sk[i][1] = *reinterpret_cast<const f32x4_t*>(K + e + 4);
            sv[i][0] = *reinterpret_cast<const f32x4_t*>(V + e);
            sv[i][1] = *reinterpret_cast<const f32x4_t*>(V + e + 4);
        }
    };
    auto store_tile = [&](int it) {
        if (!loads) return;
        lds_u8_t* base = smem + (it & 1) * G::STAGE;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int idx = threadIdx.x + i * NT;
            const int off = G::off(idx / C8, idx % C8);
            bf16x8_t t[kTerms];
            split_terms(sk[i][0], sk[i][1], t);
#pragma unroll
            for (int x = 0; x < kTerms; ++x)
                *reinterpret_cast<__attribute__((address_space(3))) bf16x8_t*>(base + x * G::TERM + off) = t[x];
            split_terms(sv[i][0], sv[i][1], t);
#pragma unroll
            for (int x = 0; x < kTerms; ++x)
                *reinterpret_cast<__attribute__((address_space(3))) bf16x8_t*>(base + (3 + x) * G::TERM + off) = t[x];
        }
    };
    load(0);

    const int q0 = q_first + (wave % wph) * 16;
    const int q1 = min(q0 + 15, a.L - 1);
    bf16x8_t qf[G::KS][kTerms];
    {
        const float* row = Q + (long long)min(q0 + r16, a.L - 1) * a.qs[2] + 8 * g;
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks)
            split_terms(*reinterpret_cast<const f32x4_t*>(row + 32 * ks) * a.sl2,
                        *reinterpret_cast<const f32x4_t*>(row + 32 * ks + 4) * a.sl2, qf[ks]);
    }
    f32x4_t acc[G::DB];
#pragma unroll
    for (int db = 0; db < G::DB; ++db) acc[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, b = 0.f, l = 0.f, cap = -1.f;

    auto compute = [&](int k0, const lds_u8_t* sb, bool mask) {
        // element 4 kb + e of a lane: key 8 g + 4 kb + e
        f32x4_t s[2] = {f32x4_t{b, b, b, b}, f32x4_t{b, b, b, b}};
#pragma unroll
        for (int ks = 0; ks < G::KS; ++ks) {
            bf16x8_t kf[2][kTerms];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int t = 0; t < kTerms; ++t)
                    kf[kb][t] = *reinterpret_cast<const __attribute__((address_space(3))) bf16x8_t*>(
                        sb + t * G::TERM + G::off(8 * (r16 >> 2) + 4 * kb + (r16 & 3), 4 * ks + g));
#pragma unroll
            for (int pr = 0; pr < kPairs; ++pr)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    s[kb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf[kb][pair_a(pr)], qf[ks][pair_b(pr)], s[kb], 0, 0,
                                                                    0);
        }
        if (mask) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (hidden(a, q0 + r16, k0 + 8 * g + j)) s[j >> 2][j & 3] = -INFINITY;
        }
        float p[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(s[j >> 2][j & 3]);
        float sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
        if (__any(!(sum <= cap))) {
            float mt = s[0][0];
#pragma unroll
            for (int j = 1; j < 8; ++j) mt = fmaxf(mt, s[j >> 2][j & 3]);
            const float m_new = fmaxf(m, group_reduce<OpMax, 16, kWave>(mt) - b);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
#pragma unroll
            for (int db = 0; db < G::DB; ++db) acc[db] *= alpha;
            l *= alpha;
            const float b_new = m_new == -INFINITY ? 0.f : -m_new;
            const float delta = b_new - b;
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(s[j >> 2][j & 3] + delta);
            sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            m = m_new;
            b = b_new;
            cap = m_new == -INFINITY ? -1.f : kRaiseAt;
        }
        l += sum;
        bf16x8_t pt[kTerms];
        split_terms(f32x4_t{p[0], p[1], p[2], p[3]}, f32x4_t{p[4], p[5], p[6], p[7]}, pt);
#pragma unroll
        for (int db = 0; db < G::DB; ++db) {
            bf16x8_t vf[kTerms];
            const int c = 2 * db + ((r16 & 3) >> 1), r = 8 * g + (r16 >> 2), h8 = (r16 & 1) * 8;
#pragma unroll
            for (int t = 0; t < kTerms; ++t) {
                const lds_u8_t* vb = sb + (3 + t) * G::TERM + h8;
                const s16x4_t x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vb + G::off(r, c)));
                const s16x4_t y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vb + G::off(r + 4, c)));
                vf[t] = __builtin_bit_cast(bf16x8_t, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
            }
#pragma unroll
            for (int pr = 0; pr < kPairs; ++pr)
                acc[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf[pair_a(pr)], pt[pair_b(pr)], acc[db], 0, 0, 0);
        }
    };

    store_tile(0);
    if (tiles.n > 1) load(1);
    __syncthreads();
    for (int it = 0; it < tiles.n; ++it) {
        if (q0 < a.L) {
            const int k0 = tiles(it) * kF32Tile;
            const Seen sn = seen(a, q0, q1, k0, k0 + kF32Tile - 1);
            if (sn != kNone) compute(k0, smem + (it & 1) * G::STAGE, sn == kSome);
        }
        if (it + 1 < tiles.n) {
            store_tile(it + 1);
            if (it + 2 < tiles.n) load(it + 2);
        }
        __syncthreads();
    }

    const float sum = group_reduce<OpSum, 16, kWave>(l + not_finite<G::DB>(acc)), inv = 1.0f / sum;
    const bool fine = sum < INFINITY;
    if (q0 + r16 < a.L && fine) {
        float* o = static_cast<float*>(a.dst) + wk.b * a.os[0] + h * a.os[1] + (long long)(q0 + r16) * a.os[2] + 4 * g;
#pragma unroll
        for (int db = 0; db < G::DB; ++db) *reinterpret_cast<f32x4_t*>(o + 16 * db) = acc[db] * inv;
    }
    for (uint32_t anew = __ballot(q0 + r16 < a.L && !fine) & 0xffff; anew; anew &= anew - 1)
        window_plain<D, float>(wave / wph, q0 + __builtin_ctz(anew));
}

// ---------------------------------------------------------------- launch

// Waves per workgroup, the heads it serves and its query tile: eight waves where
// that fills the CUs (8192 queries, bf16, 512 workgroups: 87 us against 92.5 in
// workgroups of four; 2048, fp32, 256: 54.6 against 83.5), else four (3 x 777, bf16,
// 300 against 156: 10.4 us against 13.1 in eight).
struct WindowShape {
    int waves, gh, q_tile;
};
WindowShape window_shape(bool bf16, int batch, int Hq, int Hkv, int L) {
    const int G = Hq / Hkv, per_wave = bf16 ? 32 : 16;
    WindowShape s{8, 1, 0};
    for (;; s.waves = 4) {
        // All heads that share a KV head where they divide the waves: a
        // workgroup's tiles are window + query tile keys for waves x per_wave rows.
        s.gh = 1;
        while (s.gh * 2 <= s.waves && G % (s.gh * 2) == 0) s.gh *= 2;
        s.q_tile = s.waves / s.gh * per_wave;
        const long long wgs = (long long)batch * (Hq / s.gh) * ((L + s.q_tile - 1) / s.q_tile);
        if (s.waves == 4 || wgs >= device_cu_count()) return s;
    }
}

template <auto KERNEL>
sa_status launch_window(const WindowArgs& a, int batch, const WindowShape& s, int lds, hipStream_t st) {
    SA_TRY(pf::opt_in_lds<KERNEL>(lds));
    const long long grid = (long long)batch * (a.Hq / s.gh) * a.n_qt;
    hipLaunchKernelGGL(KERNEL, dim3((unsigned)grid), dim3(s.waves * kWave), lds, st, a);
    SA_CHECK_LAUNCH();
    return SA_OK;
}

template <int D>
sa_status dispatch_window(const WindowArgs& a, bool bf16, int batch, const WindowShape& s, hipStream_t st) {
    if (bf16)
        return s.waves == 8 ? launch_window<window_bf16_kernel<D, 8>>(a, batch, s, 2 * BfGeo<D>::STAGE, st)
                            : launch_window<window_bf16_kernel<D, 4>>(a, batch, s, 2 * BfGeo<D>::STAGE, st);
    return s.waves == 8 ? launch_window<window_f32_kernel<D, 8>>(a, batch, s, 2 * F32Geo<D>::STAGE, st)
                        : launch_window<window_f32_kernel<D, 4>>(a, batch, s, 2 * F32Geo<D>::STAGE, st);
}

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" sa_status sa_prefill_window(const void* q, const void* k, const void* v, sa_dtype dtype, int batch,
                                       int n_q_heads, int n_kv_heads, int L, int D, const int64_t q_strides[3],
                                       const int64_t kv_strides[3], const int64_t out_strides[3], int window,
                                       int n_sink, float scale, void* out, sa_stream_t stream) {
    clear_error();
    if (dtype != SA_DTYPE_F32 && dtype != SA_DTYPE_BF16) return fail(SA_EINVAL, "dtype must be F32 or BF16");
    if (batch <= 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads) return fail(SA_EINVAL, "bad head counts");
    if (L < 0 || L > (1 << 30)) return fail(SA_EINVAL, "L must be 0 to 2^30");
    if (D != 64 && D != 128) return fail(SA_EINVAL, "head_dim must be 64 or 128");
    if (window <= 0) return fail(SA_EINVAL, "window must be positive");
    if (n_sink < 0) return fail(SA_EINVAL, "n_sink must be >= 0");
    if ((q_strides == nullptr) != (kv_strides == nullptr) || (q_strides == nullptr) != (out_strides == nullptr))
        return fail(SA_EINVAL, "strides are given for all tensors or for none");
    if (L == 0) return SA_OK;
    if (!q || !k || !v || !out) return fail(SA_EINVAL, "null pointer");
    const bool bf16 = dtype == SA_DTYPE_BF16;
    const int elem = bf16 ? 2 : 4;
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
        return fail(SA_EINVAL, "tensors must be 16-byte aligned");
    WindowArgs a{};
    a.q = q; a.k = k; a.v = v; a.dst = out;
    const long long LD = (long long)L * D;
    const long long dense_q[3] = {n_q_heads * LD, LD, D}, dense_kv[3] = {n_kv_heads * LD, LD, D};
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = q_strides ? q_strides[i] : dense_q[i];
        a.kvs[i] = kv_strides ? kv_strides[i] : dense_kv[i];
        a.os[i] = out_strides ? out_strides[i] : dense_q[i];
        for (long long s : {a.qs[i], a.kvs[i], a.os[i]})
            if (s < 0 || s * elem % 16) return fail(SA_EINVAL, "strides must be multiples of 16 bytes, not negative");
    }
    if (a.kvs[2] >= (1 << 24)) return fail(SA_EINVAL, "the row stride of k and v must be below 2^24 elements");
    a.Hq = n_q_heads; a.Hkv = n_kv_heads; a.L = L;
    a.window = std::min(window, L);
    a.sink = std::min(n_sink, L);
    const WindowShape s = window_shape(bf16, batch, n_q_heads, n_kv_heads, L);
    a.gh = s.gh;
    a.q_tile = s.q_tile;
    a.n_qt = (L + s.q_tile - 1) / s.q_tile;
    // a grid has fewer than 2^32 threads
    if ((long long)batch * (n_q_heads / s.gh) * a.n_qt >= (1LL << 32) / (s.waves * kWave))
        return fail(SA_EINVAL, "too many query tiles");
    const long long groups = (long long)batch * n_kv_heads;
    a.xcd_groups = groups % 8 == 0 ? (int)(groups / 8) : 0;
    // bf16: the sign goes to q, so that the scores' factor is not negative
    a.sl2 = (bf16 ? std::fabs(scale) : scale) * pf::kLog2eP;
    a.q_sign = bf16 && scale < 0 ? 0x80008000u : 0u;
    return D == 64 ? dispatch_window<64>(a, bf16, batch, s, as_stream(stream))
                   : dispatch_window<128>(a, bf16, batch, s, as_stream(stream));
}
