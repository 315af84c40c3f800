// Attention of one query row in plain fp32 arithmetic, for the rows whose
// result on the matrix cores is not finite.
//
// There an infinity loses its meaning: its split into bf16 terms is {inf, NaN,
// NaN} (as is that of an fp32 value beyond bf16's largest), weights of several
// terms meet it with both signs, and a hidden key's weight of 0 times an infinity
// or NaN is NaN.  A kernel therefore looks at each row's sums once at the end (a
// NaN never leaves them) and computes the rows that are not finite anew here,
// over the keys that the row sees and no others.  Ordinary rows pay for the look
// alone, an FMA per accumulator (decode over ranges, 16 / 8 heads of 128: 4 x 4 rows
// in fp32 20.7 -> 20.8 us, one row 10.7 -> 10.9, 64 rows behind 32768 shared tokens
// 75.3 -> 75.4; windowed prefill of 3 x 777 in bf16 10.3 -> 10.4, of 8192 86.5 as
// before).  Rows computed anew: 64 behind 32768 tokens, all values NaN, 6.4 ms.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bf16_terms.h"
#include "sa_internal.h"

namespace sa {

__device__ __forceinline__ float plain_value(float v) { return v; }
__device__ __forceinline__ float plain_value(uint16_t v) { return bf16_lo(v); }
__device__ __forceinline__ float plain_value(uint8_t v) { return __builtin_amdgcn_cvt_f32_fp8(v, 0); }   // e4m3

// Eight values from a 16-byte aligned place.
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const f32x4_t x = reinterpret_cast<const f32x4_t*>(p)[h];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * h + i] = x[i];
    }
}
__device__ __forceinline__ void load8(const uint16_t* p, float (&v)[8]) {
    const u32x4_t x = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = bf16_lo(x[i]);
        v[2 * i + 1] = bf16_hi(x[i]);
    }
}

// Eight codes in e4m3 from an 8-byte aligned place.
__device__ __forceinline__ void load8(const uint8_t* p, float (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int x = reinterpret_cast<const int*>(p)[h];
        v[4 * h] = __builtin_amdgcn_cvt_f32_fp8(x, 0);
        v[4 * h + 1] = __builtin_amdgcn_cvt_f32_fp8(x, 1);
        v[4 * h + 2] = __builtin_amdgcn_cvt_f32_fp8(x, 2);
        v[4 * h + 3] = __builtin_amdgcn_cvt_f32_fp8(x, 3);
    }
}

struct NoScale {
    __device__ __forceinline__ float operator()(int) const { return 1.f; }
};

// 0 where all values are finite, else NaN.
template <int N>
__device__ __forceinline__ float not_finite(const f32x4_t* v) {
    f32x4_t x = v[0] * 0.f;
#pragma unroll
    for (int i = 1; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = fmaf(v[i][e], 0.f, x[e]);
    return (x[0] + x[1]) + (x[2] + x[3]);
}

// One wave: running maximum (log2 domain) and sum of weights, and columns E lane
// .. E lane + E - 1 of the unnormalised output.
template <int D>
struct PlainRow {
    static constexpr int E = D / kWave;
    float m = -INFINITY, l = 0.f;
    float o[E] = {};

    // A NaN among the weights makes one of every column, whatever else there is.
    __device__ __forceinline__ bool lost() const { return l != l; }

    // n keys (1 .. 64), lane i's score is that of key i: c sum_d q[d] key(i)[d].
    // key(i), value(i): where key or value i starts, for i < n; ks(i), vs(i): a
    // power of two that its elements are times.
    template <class T, class Key, class Value, class KeyScale = NoScale, class ValueScale = NoScale>
    __device__ __forceinline__ void keys(int n, const T* q, float c, const Key& key, const Value& value,
                                         const KeyScale& ks = {}, const ValueScale& vs = {}) {
        const int lane = threadIdx.x & (kWave - 1);
        const auto* k = key(min(lane, n - 1));
        float s = 0.f;
#pragma unroll 4
        for (int d = 0; d < D; d += 8) {
            float x[8], y[8];
            load8(k + d, x);
            load8(q + d, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) s = fmaf(x[i], y[i], s);
        }
        s = lane < n ? s * ks(min(lane, n - 1)) * c : -INFINITY;
        const float top = group_reduce<OpMax, 1, kWave>(s);   // leaves NaN out, which the sums then hold
        const float m_new = fmaxf(m, top);
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - m_new);
        float p = m_new == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(s - m_new);
        if (s != s) p = s;
        if (lane >= n) p = 0.f;
        l = l * alpha + group_reduce<OpSum, 1, kWave>(p);
        // Before the first finite score there is nothing to scale, but what a
        // weight of 0 has made of an infinity (NaN) stays.
        if (m != -INFINITY)
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] *= alpha;
        m = m_new;
#pragma unroll 8
        for (int i = 0; i < n; ++i) {
            const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), i));
            const auto* v = value(i) + lane * E;
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] = fmaf(w, plain_value(v[e]) * vs(i), o[e]);
        }
    }
};

}  // namespace sa
