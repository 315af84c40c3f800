// Selection of a beam search: of all continuations (beam b, token t) of a
// group's beams, the n_select with the largest accumulated log probability
//   c(b, t) = score_b + x_bt - log sum_t' exp(x_bt'),
// of equal ones the lowest b * vocab + t.
//
// Two launches.  The first streams the logits once: every row is cut into
// segments, and each leaves its largest logit and its sum of exponentials
// relative to it (fp32, at most 64 VPT values a sum).  The second, a workgroup
// per group, joins the sums in 64 bits and selects.  c is non-decreasing in x,
// so with tau a value that at least n_select segment maxima reach, only
// segments whose maximum reaches tau hold candidates, and only their elements
// that reach tau are candidates: a few dozen, put in order by counting for
// each how many precede it.  Comparisons with tau are in fp32 (rounding is
// monotone, so nothing is lost); the order is decided in 64 bits, since
// candidates of different beams may lie closer than fp32 sums are exact.
// Where equal maxima make the lists overflow, the selection goes in n_select
// rounds over (c, index) instead.
//
// Bound: HBM, the logits read once.
#include "sa_internal.h"

#include <algorithm>

namespace sa {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWaves = kSelThreads / kWave;
constexpr int kMaxBeams = 64, kMaxSelect = 64;
constexpr int kSlots = 8;                                // segments of a thread of the second launch
constexpr int kBeamsPerWave = kMaxBeams / kSelWaves;
constexpr int kBlock = 8 * kWave;                        // elements of a wave's step
constexpr int kSegList = 256, kCandList = 1024;
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

// A wave takes `steps` steps of kBlock consecutive elements of a row.  VPT < 8:
// every VPT rows of 64 elements are a segment; VPT = 8: the wave's steps are
// one segment.
template <int VPT>
__global__ void __launch_bounds__(256) beam_scan_kernel(BeamArgs a) {
    constexpr int SEGS = 8 / VPT;
    const int row = blockIdx.x / a.wg_per_row;
    const int block = (blockIdx.x % a.wg_per_row) * 4 + threadIdx.x / kWave;
    const int lane = threadIdx.x & (kWave - 1);
    const long long first = (long long)block * a.steps * kBlock;
    if (first >= a.vocab) return;
    const float* x = a.logits + (long long)row * a.row_stride;
    float m_run = kNone, l_run = 0.f;
    for (int s = 0; s < a.steps; ++s) {
        const long long at = first + (long long)s * kBlock;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const long long i = at + j * kWave + lane;
            v[j] = i < a.vocab ? x[i] : kNone;
        }
#pragma unroll
        for (int g = 0; g < SEGS; ++g) {
            float m = v[g * VPT];
#pragma unroll
            for (int j = 1; j < VPT; ++j) m = fmaxf(m, v[g * VPT + j]);
            m = group_reduce<OpMax, 1, kWave>(m);
            float l = 0.f;
#pragma unroll
            for (int j = 0; j < VPT; ++j) l += m == kNone && v[g * VPT + j] == kNone ? 0.f : exp_diff(v[g * VPT + j] - m);
            l = group_reduce<OpSum, 1, kWave>(l);
            if constexpr (VPT < 8) {
                const long long seg = at / (kWave * VPT) + g;
                if (lane == 0 && seg < a.n_seg) a.seg[(long long)row * a.n_seg + seg] = make_float2(m, l);
            } else {
                const float mn = fmaxf(m_run, m);
                l_run = (m_run == kNone ? l_run : l_run * exp_diff(m_run - mn)) + (m == kNone ? l : l * exp_diff(m - mn));
                m_run = mn;
            }
        }
    }
    if constexpr (VPT == 8) {
        if (lane == 0) a.seg[(long long)row * a.n_seg + block] = make_float2(m_run, l_run);
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

__global__ void __launch_bounds__(kSelThreads) beam_pick_kernel(BeamArgs a) {
    __shared__ double base[kMaxBeams];              // score - log sum exp; NaN: the beam offers nothing
    __shared__ float wave_max[kSelWaves][kBeamsPerWave];
    __shared__ double wave_sum[kSelWaves][kBeamsPerWave];
    __shared__ float beam_max[kMaxBeams];
    __shared__ float top[kSelWaves];
    __shared__ int counts[2][kSelWaves];
    __shared__ int seg_list[kSegList];
    __shared__ double cand_v[kCandList];
    __shared__ int cand_i[kCandList];
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
    float2 sg[kSlots];
    int id[kSlots];      // beam * n_seg + segment, -1: none
    int of[kSlots];      // the beam's place in the wave
    {
        int bi = 0, k = 0;
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
            const int beam = a.beams_per_wave > 1 ? wave * a.beams_per_wave + bi : wave / a.waves_per_beam;
            const int s = (k * kWave + lane) * a.waves_per_beam + wave % a.waves_per_beam;
            of[j] = bi;
            id[j] = bi < a.beams_per_wave && beam < a.n_beams && s < a.n_seg ? beam * a.n_seg + s : -1;
            sg[j] = id[j] >= 0 ? seg[id[j]] : make_float2(kNone, 0.f);
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
        for (int j = 0; j < kSlots; ++j) m = of[j] == bi ? fmaxf(m, sg[j].x) : m;
        m = group_reduce<OpMax, 1, kWave>(m);
        if (lane == 0) wave_max[wave][bi] = m;
    }
    __syncthreads();
    for (int bi = 0; bi < a.beams_per_wave; ++bi) {
        const int w0 = a.beams_per_wave > 1 ? wave : wave / a.waves_per_beam * a.waves_per_beam;
        float m = kNone;
        for (int w = w0; w < min(w0 + a.waves_per_beam, kSelWaves); ++w) m = fmaxf(m, wave_max[w][bi]);
        double l = 0.0;
#pragma unroll
        for (int j = 0; j < kSlots; ++j)
            if (id[j] >= 0 && of[j] == bi) l += (double)(sg[j].y * exp_diff(sg[j].x - m));
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) l += __shfl_xor(l, d, kWave);
        const int beam = a.beams_per_wave > 1 ? wave * a.beams_per_wave + bi : wave / a.waves_per_beam;
        if (lane == 0) {
            wave_sum[wave][bi] = l;
            if (wave == w0 && beam < a.n_beams) beam_max[beam] = m;
        }
    }
    __syncthreads();
    if (tid < a.n_beams) {
        const int w0 = first_of(tid), bi = place_of(tid);
        double l = 0.0;
        for (int w = w0; w < w0 + a.waves_per_beam; ++w) l += wave_sum[w][bi];
        const double lse = (double)beam_max[tid] + log(l);
        base[tid] = isfinite(lse) ? (double)a.scores[(long long)group * a.n_beams + tid] - lse : (double)NAN;
    }
    __syncthreads();

    // ---- tau: a value that at least `want`, and rarely more than twice as many,
    // of the threads' largest segment maxima reach (-inf: fewer threads have one).
    // Bisection over the values' bit patterns, from 16 below the largest on. ----
    float key[kSlots];
    float best = kNone;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
        const float k = id[j] >= 0 ? (float)(base[id[j] / a.n_seg] + (double)sg[j].x) : kNone;
        key[j] = k > kNone ? k : kNone;   // also leaves NaN out
        best = fmaxf(best, key[j]);
    }
    {
        const float m = group_reduce<OpMax, 1, kWave>(best);
        if (lane == 0) top[wave] = m;
    }
    __syncthreads();
    float most = top[0];
#pragma unroll
    for (int w = 1; w < kSelWaves; ++w) most = fmaxf(most, top[w]);
    const uint32_t mine = ordered(best);
    int parity = 0;
    auto reach = [&](uint32_t v) {   // threads whose best is at least v
        const int n = __popcll(__ballot(mine >= v));
        if (lane == 0) counts[parity][wave] = n;
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < kSelWaves; ++w) all += counts[parity][w];
        parity ^= 1;
        return all;
    };
    uint32_t lo = ordered(kNone) + 1, hi = ordered(most) + 1;
    float t = kNone;
    if (most > kNone && reach(lo) >= want) {
        const uint32_t near = ordered(most - 16.f);
        if (near > lo && reach(near) >= want) lo = near;
        while (hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int n = reach(mid);
            if (n >= want) lo = mid;
            else hi = mid;
            if (n >= want && n <= 2 * want) break;
        }
        t = unordered(lo);
    }


    // ---- the segments and elements that reach it ----
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
        if (key[j] > kNone && key[j] >= t) {
            const int at = atomicAdd(&n_segs, 1);
            if (at < kSegList) seg_list[at] = id[j];
        }
    }
    __syncthreads();
    const float* x = a.logits + (long long)group * a.n_beams * a.row_stride;
    auto value = [&](int s, int off, int& idx) -> double {
        const int b = s / a.n_seg;
        const long long tok = (long long)(s % a.n_seg) * a.seg_len + off;
        idx = -1;
        if (tok >= a.vocab) return 0.0;
        const double c = base[b] + (double)x[b * a.row_stride + tok];
        if (c > (double)kNone) idx = b * a.vocab + (int)tok;
        return c;
    };
    if (n_segs <= kSegList) {
        // a wave per segment, four rows of 64 elements in flight
        for (int i = wave; i < n_segs; i += kSelWaves) {
            const int s = seg_list[i];
            const int b = s / a.n_seg;
            const long long tok0 = (long long)(s % a.n_seg) * a.seg_len;
            const float* xr = x + b * a.row_stride + tok0;
            const int left = (int)min((long long)a.seg_len, a.vocab - tok0);
            const double bb = base[b];
            for (int o = 0; o < left; o += 4 * kWave) {
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = o + j * kWave + lane < left ? xr[o + j * kWave + lane] : kNone;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const double c = bb + (double)v[j];
                    if (c > (double)kNone && (float)c >= t) {
                        const int at = atomicAdd(&n_cand, 1);
                        if (at < kCandList) {
                            cand_v[at] = c;
                            cand_i[at] = b * a.vocab + (int)tok0 + o + j * kWave + lane;
                        }
                    }
                }
            }
        }
    }
    __syncthreads();
    const long long out0 = (long long)group * a.n_select;
    auto put = [&](int r, double c, int idx) {
        a.out_scores[out0 + r] = idx < 0 ? kNone : (float)c;
        a.out_tokens[out0 + r] = idx < 0 ? -1 : idx % a.vocab;
        a.out_beams[out0 + r] = idx < 0 ? -1 : idx / a.vocab;
    };
    if (n_segs <= kSegList && n_cand <= kCandList) {
        const int n = n_cand;
        if (tid < n) {
            const double c = cand_v[tid];
            const int idx = cand_i[tid];
            int r = 0;
            for (int j = 0; j < n; ++j) r += ahead(cand_v[j], cand_i[j], c, idx);
            if (r < a.n_select) put(r, c, idx);
        }
        if (tid >= n && tid < a.n_select) put(tid, 0.0, -1);
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
        for (int j = 0; j < kSlots; ++j) {
            const int s = id[j];
            if (!(key[j] > kNone)) continue;
            const double c = base[s / a.n_seg] + (double)sg[j].x;
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
        if (tid == 0) put(r, v, idx);
    }
}

struct BeamShape {
    int vpt, steps, n_seg;
    int waves_per_beam, beams_per_wave, per_beam;
};
// The shortest segments that the second launch's threads hold.
BeamShape beam_shape(int n_beams, int vocab) {
    BeamShape s{1, 1, 0, std::max(1, kSelWaves / n_beams), (n_beams + kSelWaves - 1) / kSelWaves, 0};
    for (;;) {
        const long long len = (long long)kWave * s.vpt * s.steps;
        s.n_seg = (int)((vocab + len - 1) / len);
        s.per_beam = (s.n_seg + kWave * s.waves_per_beam - 1) / (kWave * s.waves_per_beam);
        if (s.per_beam * s.beams_per_wave <= kSlots) return s;
        if (s.vpt < 8) s.vpt *= 2;
        else s.steps *= 2;
    }
}

bool beam_sizes_ok(int n_groups, int n_beams, int vocab, int n_select) {
    return n_groups > 0 && n_beams > 0 && n_beams <= kMaxBeams && vocab > 0 && n_select > 0 && n_select <= kMaxSelect &&
           (long long)n_beams * vocab < (1LL << 31) && (long long)n_groups * n_beams < (1LL << 24);
}

}  // namespace
}  // namespace sa

using namespace sa;

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
        return fail(SA_EINVAL, "beam selection takes 1 to 64 beams, 1 to 64 selected, n_beams * vocab < 2^31");
    if (row_stride < vocab) return fail(SA_EINVAL, "row_stride must be at least vocab");
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
    if (wgs >= (1LL << 31)) return fail(SA_EINVAL, "too many rows");
    const dim3 grid((unsigned)wgs);
    switch (sh.vpt) {
        case 1: hipLaunchKernelGGL(beam_scan_kernel<1>, grid, dim3(256), 0, st, a); break;
        case 2: hipLaunchKernelGGL(beam_scan_kernel<2>, grid, dim3(256), 0, st, a); break;
        case 4: hipLaunchKernelGGL(beam_scan_kernel<4>, grid, dim3(256), 0, st, a); break;
        default: hipLaunchKernelGGL(beam_scan_kernel<8>, grid, dim3(256), 0, st, a); break;
    }
    SA_CHECK_LAUNCH();
    hipLaunchKernelGGL(beam_pick_kernel, dim3(n_groups), dim3(kSelThreads), 0, st, a);
    SA_CHECK_LAUNCH();
    return SA_OK;
}
