// A wave's part of causal attention on v_mfma_f32_32x32x16_bf16: 32 query rows
// against tiles of 64 keys whose K and V rows lie in LDS as bf16, chunks permuted.
// Scores are computed transposed, S^T = K Q^T, so that a lane owns one query column
// and the weights come out as the operand of O^T += V^T P^T; softmax in the log2
// domain with a running max that is raised only when a lane's sum of weights exceeds
// kRaiseAt.  Shared by the windowed prefill and the chunks over a paged cache.
#pragma once

#include "bf16_terms.h"
#include "prefill_shared.h"

namespace sa {

using pf::f32x16_t;
using pf::lds_s16x4_t;
using pf::lds_u8_t;
using pf::s16x4_t;

constexpr float kBfRaiseAt = 65536.f;

// pf::dma16 with a uniform base and a byte offset per lane.
__device__ __forceinline__ void dma16_from(const void* base, uint32_t off, lds_u8_t* dst) {
    const uint32_t m = static_cast<uint32_t>(reinterpret_cast<size_t>(dst));
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m)
                 : "memory", "m0");
}

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

    // q: row n of the wave's 32; sl2, q_sign: pf::PrefillArgs.
    __device__ __forceinline__ void init(const uint16_t* q, float sl2, uint32_t q_sign, int q_first, int lane) {
        n = lane & 31;
        hh = lane >> 5;
        q0 = q_first;
        c = sl2;
        const uint16_t* row = q + 8 * hh;
#pragma unroll
        for (int ks = 0; ks < G::NKS; ++ks) {
            u32x4_t raw = *reinterpret_cast<const u32x4_t*>(row + ks * 16);
            raw ^= q_sign;
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
            cap = m_new == -INFINITY ? -1.f : kBfRaiseAt;
#pragma unroll
            for (int j = 0; j < 16; ++j) p[j] = __builtin_amdgcn_exp2f(MASK ? s[j] + nm : fmaf(s[j], c, nm));
            pb[0] = pf::pack_bf16x8(p);
            pb[1] = pf::pack_bf16x8(p + 8);
            sum = pf::sum_bf16x8(pb[1], 0.f) + pf::sum_bf16x8(pb[0], 0.f);
        }
        l += sum;
    }

    // The scores of 32 keys whose K rows are at hb: element j is key 16 (j / 8) + 8 hh + j % 8.
    __device__ __forceinline__ f32x16_t scores(uint32_t hb) const {
        f32x16_t s = {};
#pragma unroll
        for (int ks = 0; ks < G::NKS; ++ks) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k_frag(hb, ks), qf[ks], s, 0, 0, 0);
        return s;
    }

    // The values of those keys by the scores' weights.  MASK: the caller has scaled the
    // scores by c (first: -inf times a factor of 0 would be NaN) and made those that are
    // not seen -inf.  Masks are the callers' own code between the two calls: as a
    // function passed in here they cost the windowed prefill 15 registers and 2 % of its time.
    template <bool MASK>
    __device__ __forceinline__ void weigh(f32x16_t& s, uint32_t hb) {
        bf16x8_t pb[2];
        softmax<MASK>(s, pb);
#pragma unroll
        for (int db = 0; db < G::NDB; ++db)
#pragma unroll
            for (int t = 0; t < 2; ++t)
                acc[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v_frag(hb, db, t), pb[t], acc[db], 0, 0, 0);
    }

    // O / l: every lane's columns into the wave's part of LDS (chunks of a row
    // permuted as the tiles' are), then rows of 16-byte pieces to memory, row q0 + r < L
    // to dst(q0 + r).  Returns the rows r, a bit each, that are not finite and not written.
    template <class Dst>
    __device__ __forceinline__ uint32_t store(int L, const Dst& dst, lds_u8_t* buf, int lane) const {
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
            if (q0 + r < L && !(anew >> r & 1)) *reinterpret_cast<u32x4_t*>(dst(q0 + r) + 8 * ch) = v;
        }
        return anew;
    }
};

}  // namespace sa
