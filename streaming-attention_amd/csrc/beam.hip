// Selection of a beam search: of all continuations (beam b, token t) of a
// group's beams, the n_select with the largest accumulated log probability
//   c(b, t) = score_b + x_bt - log sum_t' exp(x_bt'),
// of equal ones the lowest b * vocab + t.
//
// Two launches.  The first streams the logits once: every row is cut into
// segments, and each leaves its largest logit and its sum of exponentials
// relative to it (fp32, at most 512 values a sum; longer segments are joined in 64
// bits).  The second, a workgroup
// per group, joins the sums in 64 bits and selects.  c is non-decreasing in x,
// so with tau a value that at least n_select segment maxima reach, only
// segments whose maximum reaches tau hold candidates, and only their elements
// that reach tau are candidates: a few dozen, put in order by counting for
// each how many precede it.  Comparisons with tau are in fp32 (rounding is
// monotone, so nothing is lost); the order is decided in 64 bits, so that a beam's
// own candidates keep theirs.  Those of different beams are apart by their
// normalisers' errors too.
// Where equal maxima make the lists overflow, the selection goes in n_select
// rounds over (c, index) instead.
//
// Bound: HBM for the first launch (64 rows of 151,936: 38.9 MB in 8.3 us), latency
// for the second: a lone workgroup per search fetches every instruction that it
// runs once, 7.7 us for 4 beams and 10.8 for 8 x 8.  Both, graph-replayed: 4 beams
// of 151,936 tokens 10.9 us, 8 searches of 8 21.4, 3 of 5 beams of 32,003 11.8.
#include "sa_internal.h"

#include <algorithm>

namespace sa {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kMaxBeams = 64, kMaxSelect = 64;
constexpr int kMaxGroups = 1 << 20;                      // a grid has fewer than 2^32 threads
constexpr int kFewSlots = 4, kMaxSlots = 8;              // segments of a thread of the second launch
constexpr int kBeamsPerWave = kMaxBeams / kSelWaves;
constexpr int kBlock = 8 * kWave;                        // elements of a wave's step
constexpr int kWays = 4;                                 // thresholds tried at once
constexpr int kTopLanes = kSelThreads / kWave;           // lanes of a first guess
static_assert(kWays * kSelWaves == kWave && kSelWaves == 16, "a lane per threshold and wave");
static_assert(kMaxSelect <= kWave, "a first guess for every place");
constexpr int kSegList = 256, kCandList = 1024, kGather = 8;
static_assert(kMaxSelect <= kSegList, "the rounds fill the segment list");
constexpr float kNone = -INFINITY;

struct BeamArgs {
    const float* logits;     // [groups * beams] rows of vocab, row_stride apart
    const float* scores;     // [groups][beams]
    float2* seg;             // [groups * beams][n_seg]: largest logit, sum of exp(x - it)
    float* out_scores;       // [groups][n_select]
    int32_t* out_tokens;
    int32_t* out_beams;
    long long row_stride;
    int n_groups, n_beams, vocab, n_select;
    int n_seg, seg_len;      // segments of a row, elements of a segment
    int steps;               // steps of kBlock elements per wave
    int wg_per_row;
    // Second launch: a beam's segments on waves_per_beam waves, or
    // beams_per_wave beams on a wave, per_beam segments of a beam per thread.
    int waves_per_beam, beams_per_wave, per_beam;
};

// exp(d) for d <= 0; log2(e) in two parts, so that the argument's rounding
// does not bias long sums.
__device__ __forceinline__ float exp_diff(float d) {
    return __builtin_amdgcn_exp2f(fmaf(d, 1.44269502162933349609f, d * 1.92596299112661746887e-8f));
}

// The sum over a wave, in 64 bits: lane exchanges inside 16 lanes with DPP
// (after each step groups are uniform, so the mirrors act as xor 4 and 8), then
// halves of 32 and of the wave.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
    v += dpp_f64<kDppXor1>(v);
    v += dpp_f64<kDppXor2>(v);
    v += dpp_f64<kDppHalfMirror>(v);
    v += dpp_f64<kDppMirror>(v);
    v += __shfl_xor(v, 16, kWave);
    v += __shfl_xor(v, 32, kWave);
    return v;
}

// A wave takes `steps` steps of kBlock consecutive elements of a row, four
// neighbouring ones per lane and load (VEC: rows start 16-byte aligned, else
// four loads).  VPT < 8: the 64 VPT elements of 16 VPT lanes are a segment, so
// one reduction serves all segments of a load; VPT = 8: the wave's steps are one,
// whose maxima and sums the lanes keep, a step each, until 64 of them are joined
// in 64 bits (a running fp32 sum, rescaled at each step, would carry an error of
// its own per step).
template <int VPT, bool VEC>
__global__ void __launch_bounds__(256) beam_scan_kernel(BeamArgs a) {
    constexpr int LANES = VPT < 4 ? 16 * VPT : kWave;   // lanes of a segment
    constexpr int JOIN = VPT == 8 ? 2 : 1;              // loads of a segment
    const int row = blockIdx.x / a.wg_per_row;
    const int block = (blockIdx.x % a.wg_per_row) * 4 + threadIdx.x / kWave;
    const int lane = threadIdx.x & (kWave - 1);
    const long long first = (long long)block * a.steps * kBlock;
    if (first >= a.vocab) return;
    const float* x = a.logits + (long long)row * a.row_stride;
    float m_run = kNone, m_of = kNone, l_of = 0.f;   // m_of, l_of: this lane's step
    double l_run = 0.0;
    for (int s = 0; s < a.steps; ++s) {
        const long long at = first + (long long)s * kBlock;
        float v[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long long i = at + j * 4 * kWave + 4 * lane;
            if (VEC && i + 4 <= a.vocab) {
                const float4 q = *reinterpret_cast<const float4*>(x + i);
                v[j][0] = q.x; v[j][1] = q.y; v[j][2] = q.z; v[j][3] = q.w;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[j][e] = i + e < a.vocab ? x[i + e] : kNone;
            }
        }
#pragma unroll
        for (int g = 0; g < 2; g += JOIN) {
            float m = kNone;
#pragma unroll
            for (int j = g; j < g + JOIN; ++j) m = fmaxf(m, fmaxf(fmaxf(v[j][0], v[j][1]), fmaxf(v[j][2], v[j][3])));
            m = group_reduce<OpMax, 1, LANES>(m);
            const float from = m == kNone ? 0.f : m;   // -inf itself adds 0
            float l = 0.f;
#pragma unroll
            for (int j = g; j < g + JOIN; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) l += exp_diff(v[j][e] - from);
            l = group_reduce<OpSum, 1, LANES>(l);
            if constexpr (VPT < 8) {
                const long long seg = (at + g * 4 * kWave + 4 * lane) / (kWave * VPT);
                if (lane % LANES == 0 && seg < a.n_seg) a.seg[(long long)row * a.n_seg + seg] = make_float2(m, l);
            } else {
                if (a.steps == 1) {
                    m_run = m;
                    l_run = l;
                    continue;
                }
                if (lane == s % kWave) {
                    m_of = m;
                    l_of = l;
                }
                if ((s + 1) % kWave && s + 1 < a.steps) continue;
                const float top = fmaxf(m_run, group_reduce<OpMax, 1, kWave>(m_of));
                const double sum = wave_sum_f64(m_of == kNone ? (double)l_of : (double)l_of * (double)exp_diff(m_of - top));
                l_run = (m_run == kNone ? l_run : l_run * (double)exp_diff(m_run - top)) + sum;
                m_run = top;
                m_of = kNone;
                l_of = 0.f;
            }
        }
    }
    if constexpr (VPT == 8) {
        if (lane == 0) a.seg[(long long)row * a.n_seg + block] = make_float2(m_run, (float)l_run);
    }
}

// Floats as unsigned integers of the same order (NaN aside), and back.
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t u = __float_as_uint(f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// A beam's segment in one integer of the segments' order.
constexpr int kSegBits = 16;
static_assert(kSelWaves * kWave * kMaxSlots <= 1 << kSegBits, "segments of a beam");
__device__ __forceinline__ int segment_id(int beam, int seg) { return beam << kSegBits | seg; }
__device__ __forceinline__ int beam_of(int id) { return id >> kSegBits; }
__device__ __forceinline__ int seg_of(int id) { return id & ((1 << kSegBits) - 1); }

struct alignas(16) Candidate {
    double c;
    int idx, beam;
};

// Candidate order: larger value first, of equal ones the lower index.
__device__ __forceinline__ bool ahead(double v, int i, double w, int j) { return v > w || (v == w && i < j); }

// The first candidate of the workgroup in that order; idx < 0: none.
__device__ void first_of_all(double& v, int& idx, double* sv, int* si) {
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const double w = __shfl_xor(v, d, kWave);
        const int j = __shfl_xor(idx, d, kWave);
        if (j >= 0 && (idx < 0 || ahead(w, j, v, idx))) {
            v = w;
            idx = j;
        }
    }
    const int wave = threadIdx.x / kWave;
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == 0) {
        sv[wave] = v;
        si[wave] = idx;
    }
    __syncthreads();
    for (int w = 0; w < kSelWaves; ++w)
        if (si[w] >= 0 && (idx < 0 || ahead(sv[w], si[w], v, idx))) {
            v = sv[w];
            idx = si[w];
        }
}

template <int SLOTS>
__global__ void __launch_bounds__(kSelThreads) beam_pick_kernel(BeamArgs a) {
    __shared__ double base[kMaxBeams];              // score - log sum exp; NaN: the beam offers nothing
    __shared__ float wave_max[kSelWaves][kBeamsPerWave];
    __shared__ double wave_sum[kSelWaves][kBeamsPerWave];
    __shared__ float tops[kWave], ranked[kWave];    // the largest segment maximum of 16 lanes each
    __shared__ float counts[2][kWays * kSelWaves];
    __shared__ int seg_list[kSegList];
    __shared__ Candidate cand[kCandList];
    __shared__ int n_segs, n_cand;
    __shared__ double red_v[kSelWaves];
    __shared__ int red_i[kSelWaves];

    const int group = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    const float2* seg = a.seg + (long long)group * a.n_beams * a.n_seg;
    const int want = a.n_select;
    if (tid == 0) {
        n_segs = 0;
        n_cand = 0;
    }

    // ---- this thread's segments: slot j is part j % per_beam of its wave's beam
    // j / per_beam, whose segments are dealt out to the beam's waves first ----
    // A search's scores are read here and its results written at the end: they may
    // share their place, while no search's results may fall on another's scores.
    const float score = tid < a.n_beams ? a.scores[(long long)group * a.n_beams + tid] : 0.f;
    float2 sg[SLOTS];
    int id[SLOTS];      // segment of the beam, -1: none
    int of[SLOTS];      // the beam's place in the wave (uniform)
    const int n_slots = a.per_beam * a.beams_per_wave;
    const int beam0 = a.beams_per_wave > 1 ? wave * a.beams_per_wave : wave / a.waves_per_beam;
    {
        int bi = 0, k = 0;
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
            const int s = (k * kWave + lane) * a.waves_per_beam + wave % a.waves_per_beam;
            of[j] = bi;
            id[j] = j < n_slots && beam0 + bi < a.n_beams && s < a.n_seg ? s : -1;
            sg[j] = id[j] >= 0 ? seg[(beam0 + bi) * a.n_seg + s] : make_float2(kNone, 0.f);
            if (++k == a.per_beam) {
                k = 0;
                ++bi;
            }
        }
    }

    // ---- the beams' normalisers ----
    auto first_of = [&](int b) { return a.beams_per_wave > 1 ? b / a.beams_per_wave : b * a.waves_per_beam; };
    auto place_of = [&](int b) { return a.beams_per_wave > 1 ? b % a.beams_per_wave : 0; };
    for (int bi = 0; bi < a.beams_per_wave; ++bi) {
        float m = kNone;
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) m = of[j] == bi ? fmaxf(m, sg[j].x) : m;
        m = group_reduce<OpMax, 1, kWave>(m);
        double l = 0.0;
#pragma unroll
        for (int j = 0; j < SLOTS; ++j)
            if (j < n_slots && of[j] == bi) l += sg[j].x == kNone ? sg[j].y : (double)(sg[j].y * exp_diff(sg[j].x - m));
        l = wave_sum_f64(l);
        if (lane == 0) {
            wave_max[wave][bi] = m;
            wave_sum[wave][bi] = l;
        }
    }
    __syncthreads();
    if (tid < a.n_beams) {
        const int w0 = first_of(tid), bi = place_of(tid);
        float m = kNone;
        double l = 0.0;
        for (int w = w0; w < w0 + a.waves_per_beam; ++w) {
            const float x = wave_max[w][bi], y = fmaxf(m, x);
            l = (m == kNone ? l : l * (double)exp_diff(m - y)) +
                (x == kNone ? wave_sum[w][bi] : wave_sum[w][bi] * (double)exp_diff(x - y));
            m = y;
        }
        const double lse = (double)m + log(l);
        base[tid] = isfinite(lse) ? (double)score - lse : (double)NAN;
    }
    __syncthreads();

    // ---- tau: a value that at least `want`, and rarely more than twice as many,
    // of the threads' largest segment maxima reach (-inf: fewer threads have one).
    // The first guesses are largest values of 16 lanes each, of which the want-th
    // largest is seldom reached by many more threads; then kWays thresholds at once,
    // equal parts of the range that is left, by the values' bit patterns. ----
    float key[SLOTS];
    float best = kNone;
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
        key[j] = kNone;
        if (j < n_slots && beam0 + of[j] < a.n_beams) {
            const float k = (float)(base[beam0 + of[j]] + (double)sg[j].x);
            if (k > kNone) key[j] = k;   // also leaves NaN out
        }
        best = fmaxf(best, key[j]);
    }
    {
        const float m = group_reduce<OpMax, 1, kTopLanes>(best);
        if (lane % kTopLanes == 0) tops[tid / kTopLanes] = m;
    }
    __syncthreads();
    const float a_top = tops[lane];
    // tops in order, largest first: each wave finds the places of its own four.
#pragma unroll
    for (int j = 0; j < kWave / kSelWaves; ++j) {
        const int i = wave * (kWave / kSelWaves) + j;
        const float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(a_top), i));
        const int place = __popcll(__ballot(a_top > v || (a_top == v && lane < i)));
        if (lane == 0) ranked[place] = v;
    }
    __syncthreads();
    const float most = ranked[0];
    const uint32_t mine = ordered(best);
    int parity = 0;
    // Threads whose best is at least v[0], .., v[kWays - 1] (increasing).  Lanes 16 i
    // .. add up the waves' counts for v[i] (whole numbers, exact in fp32).
    auto reach = [&](const uint32_t (&v)[kWays], int (&n)[kWays]) {
#pragma unroll
        for (int i = 0; i < kWays; ++i) {
            const int here = __popcll(__ballot(mine >= v[i]));
            if (lane == 0) counts[parity][i * kSelWaves + wave] = (float)here;
        }
        __syncthreads();
        const float all = group_reduce<OpSum, 1, kSelWaves>(counts[parity][lane]);
#pragma unroll
        for (int i = 0; i < kWays; ++i)
            n[i] = (int)__uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(all), i * kSelWaves));
        parity ^= 1;
    };
    float t = kNone;
    if (most > kNone) {
        const uint32_t bottom = ordered(kNone) + 1;
        uint32_t v[kWays] = {max(bottom, ordered(ranked[want - 1])), max(bottom, ordered(ranked[(want - 1) / 2])),
                             max(bottom, ordered(ranked[(want - 1) / 4])), ordered(most)};
        uint32_t lo = bottom, hi = ordered(most) + 1;
        int n[kWays];
        reach(v, n);
        bool go = n[0] >= want;      // else every value is wanted
        while (go) {
#pragma unroll
            for (int i = 0; i < kWays; ++i) {
                if (n[i] >= want) lo = v[i];
                if (n[i] >= want && n[i] <= 2 * want) go = false;
                if (n[i] < want) hi = min(hi, v[i]);
            }
            t = unordered(lo);
            if (!go || hi - lo <= 1) break;
            const uint32_t step = (hi - lo) / (kWays + 1);
#pragma unroll
            for (int i = 0; i < kWays; ++i) v[i] = lo + (step ? (i + 1) * step : min(i + 1u, hi - 1 - lo));
            reach(v, n);
        }
    }

    // ---- the segments and elements that reach it ----
#pragma unroll
    for (int j = 0; j < SLOTS; ++j) {
        if (key[j] > kNone && key[j] >= t) {
            const int at = atomicAdd(&n_segs, 1);
            if (at < kSegList) seg_list[at] = segment_id(beam0 + of[j], id[j]);
        }
    }
    __syncthreads();
    const float* x = a.logits + (long long)group * a.n_beams * a.row_stride;
    auto value = [&](int s, int off, int& idx) -> double {
        const int b = beam_of(s);
        const long long tok = (long long)seg_of(s) * a.seg_len + off;
        idx = -1;
        if (tok >= a.vocab) return 0.0;
        const double c = base[b] + (double)x[b * a.row_stride + tok];
        if (c > (double)kNone) idx = b * a.vocab + (int)tok;
        return c;
    };
    if (n_segs <= kSegList) {
        // all their elements at once, kGather per thread in flight
        const int shift = 31 - __clz(a.seg_len);
        const long long n = (long long)n_segs << shift;
        for (long long at0 = tid; at0 < n; at0 += kGather * kSelThreads) {
            float v[kGather];
            int idx[kGather], beam[kGather];
#pragma unroll
            for (int j = 0; j < kGather; ++j) {
                const long long at = at0 + j * kSelThreads;
                idx[j] = -1;
                if (at < n) {
                    const int s = seg_list[at >> shift];
                    beam[j] = beam_of(s);
                    const long long tok = ((long long)seg_of(s) << shift) + (at & (a.seg_len - 1));
                    if (tok < a.vocab) {
                        idx[j] = beam[j] * a.vocab + (int)tok;
                        v[j] = x[beam[j] * a.row_stride + tok];
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < kGather; ++j) {
                if (idx[j] < 0) continue;
                const double c = base[beam[j]] + (double)v[j];
                if (c > (double)kNone && (float)c >= t) {
                    const int at = atomicAdd(&n_cand, 1);
                    if (at < kCandList) cand[at] = Candidate{c, idx[j], beam[j]};
                }
            }
        }
    }
    __syncthreads();
    const long long out0 = (long long)group * a.n_select;
    auto put = [&](int r, double c, int idx, int beam) {
        a.out_scores[out0 + r] = idx < 0 ? kNone : (float)c;
        a.out_tokens[out0 + r] = idx < 0 ? -1 : idx - beam * a.vocab;
        a.out_beams[out0 + r] = idx < 0 ? -1 : beam;
    };
    if (n_segs <= kSegList && n_cand <= kCandList) {
        const int n = n_cand;
        if (tid < n) {
            const Candidate mine = cand[tid];
            int r = 0;
#pragma unroll 8
            for (int j = 0; j < n; ++j) r += ahead(cand[j].c, cand[j].idx, mine.c, mine.idx);
            if (r < a.n_select) put(r, mine.c, mine.idx, mine.beam);
        }
        if (tid >= n && tid < a.n_select) put(tid, 0.0, -1, -1);
        return;
    }

    // ---- many equal values: rounds, first over segments in the order of (largest
    // c, first index), of which the first `want` hold the selection ----
    double last_v = INFINITY;
    int last_i = -1, picked = 0;
    for (; picked < want; ++picked) {
        double v = 0.0;
        int idx = -1;
#pragma unroll
        for (int j = 0; j < SLOTS; ++j) {
            if (!(key[j] > kNone)) continue;
            const int s = segment_id(beam0 + of[j], id[j]);
            const double c = base[beam0 + of[j]] + (double)sg[j].x;
            if (picked && !ahead(last_v, last_i, c, s)) continue;
            if (idx < 0 || ahead(c, s, v, idx)) {
                v = c;
                idx = s;
            }
        }
        first_of_all(v, idx, red_v, red_i);
        if (idx < 0) break;
        last_v = v;
        last_i = idx;
        if (tid == 0) seg_list[picked] = idx;
    }
    __syncthreads();
    const long long n = (long long)picked * a.seg_len;
    bool more = true;
    for (int r = 0; r < a.n_select; ++r) {
        double v = 0.0;
        int idx = -1;
        for (long long i = tid; more && i < n; i += kSelThreads) {
            int at;
            const double c = value(seg_list[i / a.seg_len], (int)(i % a.seg_len), at);
            if (at < 0 || (r && !ahead(last_v, last_i, c, at))) continue;
            if (idx < 0 || ahead(c, at, v, idx)) {
                v = c;
                idx = at;
            }
        }
        first_of_all(v, idx, red_v, red_i);
        more = idx >= 0;
        last_v = v;
        last_i = idx;
        if (tid == 0) put(r, v, idx, idx / a.vocab);
    }
}

struct BeamShape {
    int slots, vpt, steps, n_seg;
    int waves_per_beam, beams_per_wave, per_beam;
};
// The shortest segments that the second launch's threads hold: in four slots
// each where segments of 256 elements do, since its time is mostly that of
// fetching its instructions (when written, 4 beams of 151,936 tokens 12.0 us
// against 12.5 in eight, 3 x 5 of 32,003 12.7 against 13.3), else in eight (8 x 8
// of 151,936 21.7 against 24.2 us).
BeamShape beam_shape(int n_beams, int vocab) {
    BeamShape s{kFewSlots, 1, 1, 0, std::max(1, kSelWaves / n_beams), (n_beams + kSelWaves - 1) / kSelWaves, 0};
    for (;;) {
        const long long len = (long long)kWave * s.vpt * s.steps;
        s.n_seg = (int)((vocab + len - 1) / len);
        s.per_beam = (s.n_seg + kWave * s.waves_per_beam - 1) / (kWave * s.waves_per_beam);
        if (s.per_beam * s.beams_per_wave <= s.slots) return s;
        if (s.slots == kFewSlots && s.vpt == 4) s.slots = kMaxSlots, s.vpt = 1;
        else if (s.vpt < 8) s.vpt *= 2;
        else s.steps *= 2;
    }
}

bool beam_sizes_ok(int n_groups, int n_beams, int vocab, int n_select) {
    return n_groups > 0 && n_beams > 0 && n_beams <= kMaxBeams && vocab > 0 && n_select > 0 && n_select <= kMaxSelect &&
           (long long)n_beams * vocab < (1LL << 31) && n_groups <= kMaxGroups;
}

}  // namespace
}  // namespace sa

using namespace sa;

sa_status sa::check_beam_scores(const float* scores, const float* out_scores, int n_groups, int n_beams, int n_select) {
    if (n_groups <= 0 || n_beams <= 0 || n_select <= 0) return SA_OK;   // refused as sizes
    if (out_scores == scores && (n_select == n_beams || n_groups == 1)) return SA_OK;
    const uintptr_t in = reinterpret_cast<uintptr_t>(scores), out = reinterpret_cast<uintptr_t>(out_scores);
    const unsigned long long n = n_groups;
    if (in < out + n * n_select * sizeof(float) && out < in + n * n_beams * sizeof(float))
        return fail(SA_EINVAL, "out_scores may be scores itself for as many selected as beams, or for one search, "
                               "and not overlap it otherwise");
    return SA_OK;
}

extern "C" size_t sa_beam_select_ws_bytes(int n_groups, int n_beams, int vocab, int n_select) {
    if (!beam_sizes_ok(n_groups, n_beams, vocab, n_select)) return 0;
    return (size_t)n_groups * n_beams * beam_shape(n_beams, vocab).n_seg * sizeof(float2);
}

extern "C" sa_status sa_beam_select(const float* logits, int64_t row_stride, const float* scores, int n_groups,
                                    int n_beams, int vocab, int n_select, float* out_scores, int32_t* out_tokens,
                                    int32_t* out_beams, void* ws, size_t ws_bytes, sa_stream_t stream) {
    clear_error();
    if (!logits || !scores || !out_scores || !out_tokens || !out_beams) return fail(SA_EINVAL, "null pointer");
    if (!beam_sizes_ok(n_groups, n_beams, vocab, n_select))
        return fail(SA_EINVAL, "beam selection takes 1 to 64 beams, 1 to 64 selected, n_beams * vocab < 2^31, 2^20 groups");
    if (row_stride < vocab) return fail(SA_EINVAL, "row_stride must be at least vocab");
    SA_TRY(check_beam_scores(scores, out_scores, n_groups, n_beams, n_select));
    const BeamShape sh = beam_shape(n_beams, vocab);
    if (!ws || ws_bytes < sa_beam_select_ws_bytes(n_groups, n_beams, vocab, n_select))
        return fail(SA_ENOMEM, "workspace too small for the segments");
    if (reinterpret_cast<uintptr_t>(ws) & 7u) return fail(SA_EINVAL, "ws must be 8-byte aligned");
    BeamArgs a{};
    a.logits = logits; a.scores = scores; a.seg = static_cast<float2*>(ws);
    a.out_scores = out_scores; a.out_tokens = out_tokens; a.out_beams = out_beams;
    a.row_stride = row_stride;
    a.n_groups = n_groups; a.n_beams = n_beams; a.vocab = vocab; a.n_select = n_select;
    a.waves_per_beam = sh.waves_per_beam; a.beams_per_wave = sh.beams_per_wave; a.per_beam = sh.per_beam;
    a.n_seg = sh.n_seg; a.seg_len = kWave * sh.vpt * sh.steps; a.steps = sh.steps;
    const long long per_wave = (long long)kBlock * sh.steps;
    a.wg_per_row = (int)((vocab + 4 * per_wave - 1) / (4 * per_wave));
    hipStream_t st = as_stream(stream);
    const long long wgs = (long long)n_groups * n_beams * a.wg_per_row;
    if (wgs >= (1LL << 24)) return fail(SA_EINVAL, "too many logits for one call");
    const dim3 grid((unsigned)wgs);
    const bool vec = aligned16(logits) && row_stride % 4 == 0;
    switch (sh.vpt) {
#define SA_BEAM_SCAN(VV)                                                                              \
    case VV:                                                                                          \
        if (vec) hipLaunchKernelGGL((beam_scan_kernel<VV, true>), grid, dim3(256), 0, st, a);         \
        else hipLaunchKernelGGL((beam_scan_kernel<VV, false>), grid, dim3(256), 0, st, a);            \
        break;
        SA_BEAM_SCAN(1)
        SA_BEAM_SCAN(2)
        SA_BEAM_SCAN(4)
        SA_BEAM_SCAN(8)
#undef SA_BEAM_SCAN
    }
    SA_CHECK_LAUNCH();
    if (sh.slots == kFewSlots) hipLaunchKernelGGL(beam_pick_kernel<kFewSlots>, dim3(n_groups), dim3(kSelThreads), 0, st, a);
    else hipLaunchKernelGGL(beam_pick_kernel<kMaxSlots>, dim3(n_groups), dim3(kSelThreads), 0, st, a);
    SA_CHECK_LAUNCH();
    return SA_OK;
}
