// Verification of drafted tokens against the target model's logits, from given
// uniform numbers; without drafts, sampling.
//
// A sequence has n drafted tokens x_0 .. x_{n-1}, target logits at n + 1 places and,
// from a draft model, draft logits at n.  With p = softmax(target / T) and q =
// softmax(draft / T) (without draft logits all of x_i's probability on x_i), x_i is
// accepted while u_i q(x_i) < p(x_i); one more token is then drawn from w = max(p - q,
// 0) at the first rejected place, or from w = p behind the last: the first t with
// sum_{t' <= t} w > u sum w.  T = 0: x_i is accepted while it is the largest logit's,
// whose token also follows.
//
// A sum of probabilities decides which token is drawn, and tokens of a large
// vocabulary lie as close as 1e-6: sums and exponentials are in 64 bits, off by some
// 1e-13.
//
// Launches: (1) every row is cut into segments of 2048 logits, a wave's each, or where a
// call has fewer than 4096 of them a workgroup's, which leave a logit that no other
// exceeds by far and the sum of exponentials relative to it (T = 0: the largest and its
// token); (2) with draft logits, what is accepted, a workgroup per sequence, and the
// rejected places' sums of w per segment; (3) a workgroup per sequence finds the
// segment that the uniform number falls into, then the token (without (2), after
// deciding what is accepted).
//
// Bound: 64-bit arithmetic of the first launch, per logit ten FMAs (2.33 ns per wave and
// SIMD), four additions and a conversion (1.95) among some 21 instructions, VALU 95 % busy
// (its reads alone would be 54 us); in the others a workgroup's chain of dependent reads,
// scans and barriers.  64 sequences of 4 drafts, 576 rows of 151,936 logits, 350 MB: 100 -
// 108 us; one sequence 17.6 - 18.2; 5 sequences of looked-up drafts, 32,003 logits, 11.7.
// Alone under the kernel tracer, gaps between and the clock lower, the launches take 73, 5,
// 21 and 8; 4.6, 4.4, 4.0 and 6.0; 4.1 and 8.4.
#include "sa_internal.h"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <new>
#include <type_traits>

namespace sa {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kQuads = 2;                        // 16-byte pieces of a lane in a step
constexpr int kStep = 4 * kQuads * kWave;        // logits that a wave takes at once
constexpr int kSteps = 4;                        // of a segment
constexpr int kSeg = kSteps * kStep;             // logits of a segment
constexpr int kDraw = 512;                       // threads that look for a token, four logits each
static_assert(kSeg == 4 * kDraw, "a piece per thread");
constexpr int kMaxDraft = 64;                    // drafted tokens of a sequence (a lane each)

struct Segment {
    double sum;     // of exp((x - top) / T)
    float top;      // a logit that no other exceeds by far (T = 0: the largest); -inf if there is none
    int32_t at;     // T = 0: its token
};

// What is drawn from.
enum Source { kTarget, kRest, kRestOfOne, kNothing };

struct VerifyArgs {
    const float* target;      // rows first[i] + i .. first[i + 1] + i of sequence i
    const float* draft;       // rows first[i] ..; NULL: none
    const int32_t* tokens;    // [drafts]
    const float* u_accept;    // [drafts]
    const float* u_sample;    // [sequences]
    long long target_stride, draft_stride;
    Segment* seg;             // [target rows, then draft rows][n_seg]
    double* rest;             // [sequences of the launch][n_seg]: sums of w
    struct Decision* decided; // [sequences of the launch], with draft logits
    int32_t* out_accepted;    // [sequences]
    int32_t* out_tokens;      // [sequences][out_stride]
    int n_target, n_draft;    // rows
    int vocab, n_seg, n_seq, out_stride;
    int groups;               // workgroups per sequence of the second launch
    double factor;            // log2(e) / T
    int seq0;                 // the launch's first sequence
    int32_t first[kRowsPerLaunch + 1];   // sequences' first drafts
};
static_assert(sizeof(VerifyArgs) <= 4096, "kernel arguments");

// 2^f, |f| <= 1/2, within 3.7e-14 of it: 1 + f times the polynomial of degree 8 that
// equals (2^f - 1) / f at the nine Chebyshev nodes of the interval.
__device__ __forceinline__ double exp2_half(double f) {
    double s = 1.0203121294865924e-07;
    s = fma(s, f, 1.3255224885529674e-06);
    s = fma(s, f, 1.525268684524423e-05);
    s = fma(s, f, 1.540345585242065e-04);
    s = fma(s, f, 1.3333558179044404e-03);
    s = fma(s, f, 9.618129159402609e-03);
    s = fma(s, f, 5.550410866476042e-02);
    s = fma(s, f, 0.2402265069581299);
    s = fma(s, f, 0.6931471805599453);
    return fma(s, f, 1.0);
}
// exp((x - top) / T); 0 for a logit of -inf, NaN for one of NaN.
__device__ __forceinline__ double weight(float x, float top, double factor) {
    double t = ((double)x - (double)top) * factor;
    t = t < -1100.0 ? -1100.0 : t;   // 2^-1100 is 0; t is below 1000
    const double n = __builtin_rint(t);
    return __builtin_ldexp(exp2_half(t - n), (int)n);
}
// The same for sums, in fewer instructions: logits of 2^-1000 of the reference's weight
// and less, and NaN, count as much.  The argument is a single FMA, off by 2^-53 of
// ref / T log2(e), so that has to be small (fine).
constexpr double kFineRef = 1024.0;
struct SumWeight {
    double factor, shift;
    float least;
    bool fine;
    __device__ __forceinline__ SumWeight(float ref, double f) : factor(f), shift(-(double)ref * f) {
        least = (float)((double)ref - 1000.0 / f);
        fine = fabs(shift) <= kFineRef && least > -3e38f;
    }
    __device__ __forceinline__ double operator()(float x) const {
        constexpr double kRound = 6755399441055744.0;   // 1.5 2^52: a sum's low word is t rounded
        const double t = fma((double)fmaxf(x, least), factor, shift);
        const double r = t + kRound;
        const double s = exp2_half(t - (r - kRound));
        return __hiloint2double(__double2hiint(s) + (__double2loint(r) << 20), __double2loint(s));
    }
};
constexpr double kNothingLeft = 1e-280;   // sums of weights that are all about 2^-1000 or 0 stay below it

template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, false);
    return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
__device__ __forceinline__ double wave_sum(double v) {
    v += dpp_f64<kDppXor1>(v);
    v += dpp_f64<kDppXor2>(v);
    v += dpp_f64<kDppHalfMirror>(v);
    v += dpp_f64<kDppMirror>(v);
    v += __shfl_xor(v, 16, kWave);
    v += __shfl_xor(v, 32, kWave);
    return v;
}

// A row's logits by segments.  Segment s holds tokens kSeg s - off .. of the row, off
// the row's distance from the 16-byte boundary before it, so that rows of any
// alignment are read in 16-byte pieces.
struct Row {
    const float* x;
    int off, vocab;
    __device__ __forceinline__ Row(const float* row, int v)
        : x(row), off((int)(reinterpret_cast<uintptr_t>(row) >> 2 & 3)), vocab(v) {}
    // The four tokens from first() on; places outside the row are none.
    __device__ __forceinline__ long long first(int s, int quad) const { return (long long)kSeg * s + 4 * quad - off; }
    __device__ __forceinline__ void load(int s, int quad, float none, float (&v)[4]) const {
        load_at(first(s, quad), none, v);
    }
    // Whether segment s lies inside the row, and its pieces then.
    __device__ __forceinline__ bool inside(int s) const {
        return (s > 0 || off == 0) && (long long)kSeg * (s + 1) - off <= vocab;
    }
    __device__ __forceinline__ void load_inside(int s, int quad, float (&v)[4]) const {
        const float4 f = *reinterpret_cast<const float4*>(x + first(s, quad));
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    }
    // Tokens i .. i + 3, wherever another row's pieces start.
    __device__ __forceinline__ void load_at(long long i, float none, float (&v)[4]) const {
        if (i >= 0 && i + 4 <= vocab && (i + off) % 4 == 0) {
            const float4 f = *reinterpret_cast<const float4*>(x + i);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = i + e >= 0 && i + e < vocab ? x[i + e] : none;
        }
    }
};

__device__ __forceinline__ const float* target_row(const VerifyArgs& a, long long r) { return a.target + r * a.target_stride; }
__device__ __forceinline__ const float* draft_row(const VerifyArgs& a, long long r) { return a.draft + r * a.draft_stride; }

// A part's sum relative to the largest logit of the whole.
__device__ __forceinline__ double joined(const Segment& g, float top, double factor) {
    return g.top == -INFINITY ? g.sum : g.sum * weight(g.top, top, factor);   // 0 or NaN without a largest logit
}

// Sums of exponentials of a wave's logits, a step at a time, relative to one of the
// first step's logits: 64 bits hold what exceeds it by 2^kFar, and only then is
// another one taken.
constexpr double kFar = 600.0;
struct WaveSum {
    double sum = 0.0;
    float ref = -INFINITY, top = -INFINITY;   // top: this lane's largest
    bool lost = false;                        // a NaN or +inf
    __device__ __forceinline__ void add(const float (&v)[kQuads][4], double factor) {
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                m = fmaxf(m, v[j][e]);
                lost = lost || !(v[j][e] < INFINITY);
            }
        top = fmaxf(top, m);
        if (ref == -INFINITY || __any(((double)m - (double)ref) * factor > kFar)) {
            const float now = group_reduce<OpMax, 1, kWave>(top);
            if (now < INFINITY) {
                if (ref != -INFINITY) sum *= weight(ref, now, factor);
                ref = now;
            }
        }
        if (ref == -INFINITY) return;
        const SumWeight w(ref, factor);
        if (w.fine) {
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += w(v[j][e]);
        } else {
            for (int j = 0; j < kQuads; ++j)
                for (int e = 0; e < 4; ++e) sum += weight(v[j][e], ref, factor);
        }
    }
    __device__ __forceinline__ Segment done() {
        Segment g{wave_sum(sum), ref, 0};
        if (__any(lost)) g.sum = NAN;
        return g;
    }
};
struct WaveTop {
    float top = -INFINITY;
    int at = 0x7fffffff;
    __device__ __forceinline__ void add(const float (&v)[kQuads][4], const int (&t)[kQuads]) {
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[j][e] > top) top = v[j][e], at = t[j] + e;   // tokens ascend
    }
    __device__ __forceinline__ Segment done() {
#pragma unroll
        for (int mask = 1; mask < kWave; mask *= 2) {
            const float ot = __shfl_xor(top, mask, kWave);
            const int oi = __shfl_xor(at, mask, kWave);
            if (better(ot, oi, top, at)) top = ot, at = oi;
        }
        return Segment{0.0, top, at};
    }
};

// A wave per segment of a row, or (SPLIT) a workgroup, a step per wave: few rows.
template <bool GREEDY, bool SPLIT>
__global__ void __launch_bounds__(kThreads) verify_segments_kernel(VerifyArgs a) {
    __shared__ Segment part[kWaves];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const long long item = SPLIT ? (long long)blockIdx.x : (long long)blockIdx.x * kWaves + wave;
    const int row = (int)(item / a.n_seg), s = (int)(item % a.n_seg);
    if (row >= a.n_target + a.n_draft) return;
    const Row r(row < a.n_target ? target_row(a, row) : draft_row(a, row - a.n_target), a.vocab);
    std::conditional_t<GREEDY, WaveTop, WaveSum> w;
    auto load = [&](int k, float (&v)[kQuads][4]) {
#pragma unroll
        for (int j = 0; j < kQuads; ++j) r.load(s, (k * kQuads + j) * kWave + lane, -INFINITY, v[j]);
    };
    auto load_inside = [&](int k, float (&v)[kQuads][4]) {
#pragma unroll
        for (int j = 0; j < kQuads; ++j) r.load_inside(s, (k * kQuads + j) * kWave + lane, v[j]);
    };
    auto add = [&](int k, const float (&v)[kQuads][4]) {
        if constexpr (GREEDY) {
            int t[kQuads];
#pragma unroll
            for (int j = 0; j < kQuads; ++j) t[j] = (int)r.first(s, (k * kQuads + j) * kWave + lane);
            w.add(v, t);
        } else {
            w.add(v, a.factor);
        }
    };
    float v[2][kQuads][4];
    if constexpr (SPLIT) {
        load(wave, v[0]);
        add(wave, v[0]);
    } else if (r.inside(s)) {
        load_inside(0, v[0]);
        for (int k = 0; k < kSteps; k += 2) {   // the next step's loads in flight under a step's sums
            load_inside(k + 1, v[1]);
            add(k, v[0]);
            if (k + 2 < kSteps) load_inside(k + 2, v[0]);
            add(k + 1, v[1]);
        }
    } else {
        for (int k = 0; k < kSteps; ++k) {
            load(k, v[0]);
            add(k, v[0]);
        }
    }
    Segment out = w.done();
    if constexpr (SPLIT) {
        if (lane == 0) part[wave] = out;
        __syncthreads();
        if (wave) return;
        out = part[lane & 3];
        if constexpr (GREEDY) {
#pragma unroll
            for (int mask = 1; mask < kWaves; mask *= 2) {
                const float ot = __shfl_xor(out.top, mask, kWave);
                const int oi = __shfl_xor(out.at, mask, kWave);
                if (better(ot, oi, out.top, out.at)) out.top = ot, out.at = oi;
            }
        } else {
            const float top = group_reduce<OpMax, 1, kWaves>(out.top);
            double sum = joined(out, top, a.factor);
            sum += dpp_f64<kDppXor1>(sum);
            sum += dpp_f64<kDppXor2>(sum);
            out = Segment{sum, top, 0};
        }
    }
    if (lane == 0) a.seg[item] = out;
}

// A row's largest logit and its sum of exponentials relative to it; a row whose sum
// is 0 or not finite has no distribution.
struct Norm {
    double sum;
    float top;
    __device__ __forceinline__ bool ok() const { return sum > 0.0 && sum < INFINITY; }
};
// Lanes' segments of a row, loaded ahead of their use; rows of more segments than
// lanes are read again.
__device__ __forceinline__ Segment load_segment(const VerifyArgs& a, long long row) {
    const int lane = threadIdx.x & (kWave - 1);
    return lane < a.n_seg ? a.seg[row * a.n_seg + lane] : Segment{0.0, -INFINITY, 0};
}
__device__ __forceinline__ Norm row_norm(const VerifyArgs& a, long long row, const Segment& mine) {
    const int lane = threadIdx.x & (kWave - 1);
    const Segment* seg = a.seg + row * a.n_seg;
    float top = mine.top;
    for (int s = lane + kWave; s < a.n_seg; s += kWave) top = fmaxf(top, seg[s].top);
    top = group_reduce<OpMax, 1, kWave>(top);
    double sum = joined(mine, top, a.factor);
    for (int s = lane + kWave; s < a.n_seg; s += kWave) sum += joined(seg[s], top, a.factor);
    return Norm{wave_sum(sum), top};
}

// What a sequence's uniform numbers decide.
struct Decision {
    Norm p, q;            // of the place that the next token comes from
    long long row, drow;  // of the target, of the draft
    int accepted;
    Source source;
    int token;            // kRestOfOne: the rejected token
};
struct Shared {
    Norm p[kMaxDraft + 1], q[kMaxDraft];
    int accepted;
};

// The same for every thread of the workgroup.
template <int WAVES>
__device__ __forceinline__ Decision decide(const VerifyArgs& a, int i, Shared& sh) {
    const int first = a.first[i], n = a.first[i + 1] - first;
    const long long row0 = (long long)first + a.seq0 + i;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x & (kWave - 1);
    const int rows = n + 1 + (a.draft ? n : 0);
    auto row_of = [&](int r) { return r <= n ? row0 + r : (long long)a.n_target + first + r - n - 1; };
    // The drafted tokens' logits, beside the rows' segments.
    int x = -1;
    float u = 0.f, tx = 0.f, dx = 0.f;
    bool drafted = false;
    if (wave == 0 && lane < n) {
        x = a.tokens[first + lane];
        u = a.u_accept[first + lane];
        drafted = x >= 0 && x < a.vocab;
        if (drafted) {
            tx = target_row(a, row0 + lane)[x];
            if (a.draft) dx = draft_row(a, first + lane)[x];
        }
    }
    constexpr int kAhead = 3;
    for (int r0 = wave; r0 < rows; r0 += kAhead * WAVES) {
        Segment g[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) g[k] = load_segment(a, row_of(min(r0 + k * WAVES, rows - 1)));
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int r = r0 + k * WAVES;
            if (r >= rows) break;
            const Norm m = row_norm(a, row_of(r), g[k]);
            if (lane == 0) (r <= n ? sh.p[r] : sh.q[r - n - 1]) = m;
        }
    }
    __syncthreads();
    if (wave == 0) {
        bool ok = false;
        if (drafted && sh.p[lane].ok()) {
            double qx = 1.0;
            if (a.draft) qx = sh.q[lane].ok() ? weight(dx, sh.q[lane].top, a.factor) / sh.q[lane].sum : NAN;
            ok = (double)u * qx < weight(tx, sh.p[lane].top, a.factor) / sh.p[lane].sum;
        }
        const int accepted = __ffsll((long long)~__ballot(ok)) - 1;
        if (lane == 0) sh.accepted = accepted < 0 ? kMaxDraft : accepted;
    }
    __syncthreads();
    Decision d;
    d.accepted = sh.accepted;
    d.p = sh.p[d.accepted];
    d.row = row0 + d.accepted;
    d.drow = first + d.accepted;
    d.source = kTarget;
    d.token = -1;
    d.q = Norm{0.0, 0.f};
    if (!d.p.ok()) {
        d.source = kNothing;
    } else if (d.accepted < n) {
        if (a.draft) {
            d.q = sh.q[d.accepted];
            if (d.q.ok()) d.source = kRest;
        } else {
            d.token = a.tokens[d.drow];
            if (d.token >= 0 && d.token < a.vocab) d.source = kRestOfOne;
        }
    }
    return d;
}

// w of the four tokens of a place of a segment.
struct Weigher {
    const VerifyArgs& a;
    const Decision& d;
    Row p, q;
    double pi, qi;
    __device__ __forceinline__ Weigher(const VerifyArgs& args, const Decision& dec)
        : a(args), d(dec), p(target_row(args, dec.row), args.vocab),
          q(dec.source == kRest ? draft_row(args, dec.drow) : nullptr, args.vocab), pi(1.0 / dec.p.sum),
          qi(dec.source == kRest ? 1.0 / dec.q.sum : 0.0) {}
    __device__ __forceinline__ void operator()(int s, int quad, double (&w)[4]) const {
        float x[4];
        p.load(s, quad, -INFINITY, x);
        const long long t = p.first(s, quad);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = weight(x[e], d.p.top, a.factor) * pi;
        if (d.source == kRest) {
            float y[4];
            q.load_at(t, -INFINITY, y);
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = fmax(0.0, w[e] - weight(y[e], d.q.top, a.factor) * qi);
        } else if (d.source == kRestOfOne) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (t + e == d.token) w[e] = 0.0;
        }
    }
};

// What is accepted: a workgroup per sequence.
__global__ void __launch_bounds__(kDraw) verify_decide_kernel(VerifyArgs a) {
    __shared__ Shared sh;
    const Decision d = decide<kDraw / kWave>(a, blockIdx.x, sh);
    if (threadIdx.x == 0) a.decided[blockIdx.x] = d;
}

// The sums of w per segment at the rejected places.
__global__ void __launch_bounds__(kThreads) verify_rest_kernel(VerifyArgs a) {
    __shared__ double part[kWaves];
    const int i = blockIdx.x / a.groups, g = blockIdx.x % a.groups;
    const Decision d = a.decided[i];
    if (d.source != kRest) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x & (kWave - 1);
    const Row p(target_row(a, d.row), a.vocab), q(draft_row(a, d.drow), a.vocab);
    const double pi = 1.0 / d.p.sum, qi = 1.0 / d.q.sum;
    const SumWeight pw(d.p.top, a.factor), qw(d.q.top, a.factor);
    for (int s = g; s < a.n_seg; s += a.groups) {
        float x[kQuads][4], y[kQuads][4];
#pragma unroll
        for (int j = 0; j < kQuads; ++j) {
            const int quad = (wave * kQuads + j) * kWave + lane;
            p.load(s, quad, -INFINITY, x[j]);
            q.load_at(p.first(s, quad), -INFINITY, y[j]);
        }
        double sum = 0.0;
        if (pw.fine && qw.fine) {
#pragma unroll
            for (int j = 0; j < kQuads; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum += fmax(0.0, pw(x[j][e]) * pi - qw(y[j][e]) * qi);
        } else {
            for (int j = 0; j < kQuads; ++j)
                for (int e = 0; e < 4; ++e)
                    sum += fmax(0.0, weight(x[j][e], d.p.top, a.factor) * pi - weight(y[j][e], d.q.top, a.factor) * qi);
        }
        sum = wave_sum(sum);
        __syncthreads();
        if (lane == 0) part[wave] = sum;
        __syncthreads();
        if (threadIdx.x == 0) a.rest[(long long)i * a.n_seg + s] = (part[0] + part[1]) + (part[2] + part[3]);
    }
}

// The sum of the threads' values before this one's, and of all.
template <int N>
__device__ __forceinline__ double scan(double v, double (&part)[N], double* all) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    double sum = v;
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) {
        const double o = __shfl_up(sum, k, kWave);
        if (lane >= k) sum += o;
    }
    __syncthreads();
    if (lane == kWave - 1) part[wave] = sum;
    __syncthreads();
    double before = 0.0;
    *all = 0.0;
    for (int k = 0; k < N; ++k) {
        if (k < wave) before += part[k];
        *all += part[k];
    }
    return before + (sum - v);
}

// The smallest of the threads' values.
template <int N>
__device__ __forceinline__ int least(int v, int (&part)[N]) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int k = 1; k < kWave; k *= 2) v = min(v, __shfl_xor(v, k, kWave));
    __syncthreads();
    if (lane == 0) part[wave] = v;
    __syncthreads();
    for (int k = 0; k < N; ++k) v = min(v, part[k]);
    return v;
}

// A workgroup per sequence: the token that u falls on, and the results.
__global__ void __launch_bounds__(kDraw) verify_draw_kernel(VerifyArgs a) {
    __shared__ Shared sh;
    __shared__ double part[kDraw / kWave];
    __shared__ int ipart[kDraw / kWave];
    const int i = blockIdx.x, seq = a.seq0 + i, tid = threadIdx.x;
    Decision d = a.decided ? a.decided[i] : decide<kDraw / kWave>(a, i, sh);
    constexpr int kNone = 0x7fffffff;
    int token = -1;
    if (d.source != kNothing) {
        const Segment* seg = a.seg + d.row * a.n_seg;
        const double* rest = a.rest + (long long)i * a.n_seg;
        // The segment of a rejected token without a distribution is summed anew without
        // it: a difference would lose the others' digits.
        int without = -1;
        double without_sum = 0.0;
        if (d.source == kRestOfOne) {
            const Weigher w(a, d);
            without = (d.token + w.p.off) / kSeg;
            double v[4];
            w(without, tid, v);
            scan((v[0] + v[1]) + (v[2] + v[3]), part, &without_sum);
        }
        auto sum_of = [&](int s) -> double {
            if (d.source == kRest) return rest[s];
            if (d.source == kRestOfOne && s == without) return without_sum;
            const Segment g = seg[s];
            return g.top == -INFINITY ? 0.0 : g.sum * weight(g.top, d.p.top, a.factor) / d.p.sum;
        };
        const int per = (a.n_seg + kDraw - 1) / kDraw;
        double mine = 0.0, all, before;
        auto sums = [&]() {
            mine = 0.0;
            for (int s = tid * per; s < min(a.n_seg, (tid + 1) * per); ++s) mine += sum_of(s);
            before = scan(mine, part, &all);
        };
        sums();
        if (!(all > kNothingLeft)) {   // p is nowhere above q
            d.source = kTarget;
            sums();
        }
        const double goal = (double)a.u_sample[seq] * all;
        // The first segment whose sums reach beyond the goal, else the last that has any.
        int found = kNone, last = -1;
        double sum = before;
        double start = 0.0;
        for (int s = tid * per; s < min(a.n_seg, (tid + 1) * per); ++s) {
            const double v = sum_of(s);
            if (v > kNothingLeft) {
                last = s;
                if (found == kNone && sum + v > goal) found = s, start = sum;
            }
            sum += v;
        }
        int s = least(found, ipart);
        if (s == kNone) {
            s = -least(-last, ipart);
            if (s == last) found = s, start = sum - sum_of(s);
        }
        __shared__ double s_start;
        if (found == s) s_start = start;
        __syncthreads();
        const Weigher w(a, d);
        double v[4], whole;
        w(s, tid, v);
        double c = s_start + scan((v[0] + v[1]) + (v[2] + v[3]), part, &whole);
        found = kNone;
        last = -1;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c += v[e];
            if (v[e] > 0.0) {
                last = (int)w.p.first(s, tid) + e;
                if (found == kNone && c > goal) found = last;
            }
        }
        token = least(found, ipart);
        if (token == kNone) token = -least(-last, ipart);
    }
    const int n = a.first[i + 1] - a.first[i];
    if (tid == 0) a.out_accepted[seq] = d.accepted;
    for (int k = tid; k < a.out_stride; k += kDraw)
        a.out_tokens[(long long)seq * a.out_stride + k] =
            k < d.accepted && k < n ? a.tokens[a.first[i] + k] : k == d.accepted ? token : -1;
}

// T = 0, a wave per sequence.
__global__ void __launch_bounds__(kWave) verify_greedy_kernel(VerifyArgs a) {
    const int i = blockIdx.x, seq = a.seq0 + i, lane = threadIdx.x;
    const int first = a.first[i], n = a.first[i + 1] - first;
    int accepted = 0, token = -1;
    for (;; ++accepted) {
        const Segment* seg = a.seg + ((long long)first + seq + accepted) * a.n_seg;
        float top = -INFINITY;
        int at = 0x7fffffff;
        for (int s = lane; s < a.n_seg; s += kWave) {
            const Segment g = seg[s];
            if (g.top > top) top = g.top, at = g.at;   // segments ascend
        }
#pragma unroll
        for (int mask = 1; mask < kWave; mask *= 2) {
            const float ot = __shfl_xor(top, mask, kWave);
            const int oi = __shfl_xor(at, mask, kWave);
            if (better(ot, oi, top, at)) top = ot, at = oi;
        }
        token = at == 0x7fffffff ? -1 : at;
        if (accepted == n || token < 0 || a.tokens[first + accepted] != token) break;
    }
    if (lane == 0) a.out_accepted[seq] = accepted;
    for (int k = lane; k < a.out_stride; k += kWave)
        a.out_tokens[(long long)seq * a.out_stride + k] =
            k < accepted ? a.tokens[first + k] : k == accepted ? token : -1;
}

bool verify_sizes_ok(int n_seq, const int32_t* counts, int vocab, long long* drafts) {
    *drafts = 0;
    if (n_seq <= 0 || n_seq > (1 << 20) || vocab <= 0 || vocab > (1 << 30)) return false;
    for (int i = 0; counts && i < n_seq; ++i) {
        if (counts[i] < 0 || counts[i] > kMaxDraft) return false;
        *drafts += counts[i];
    }
    return true;
}

int segments_of(int vocab) { return (vocab + 3 + kSeg - 1) / kSeg; }   // rows start up to 3 logits into the first

}  // namespace
}  // namespace sa

using namespace sa;

extern "C" size_t sa_draft_verify_ws_bytes(int n_seq, const int32_t* counts, int vocab) {
    long long n;
    if (!verify_sizes_ok(n_seq, counts, vocab, &n)) return 0;
    const size_t segs = segments_of(vocab);
    return (size_t)(2 * n + n_seq) * segs * sizeof(Segment) +
           (size_t)std::min(n_seq, kRowsPerLaunch) * (segs * sizeof(double) + sizeof(Decision));
}

extern "C" sa_status sa_draft_verify(const float* target, int64_t target_stride, const float* draft,
                                     int64_t draft_stride, const int32_t* tokens, const float* u_accept,
                                     const float* u_sample, int n_seq, const int32_t* counts, int vocab,
                                     float temperature, int32_t* out_accepted, int32_t* out_tokens, int out_stride,
                                     void* ws, size_t ws_bytes, sa_stream_t stream) {
    clear_error();
    long long n;
    if (!verify_sizes_ok(n_seq, counts, vocab, &n))
        return fail(SA_EINVAL, "verification takes 1 to 2^20 sequences, 0 to 64 drafted tokens each, vocab 1 to 2^30");
    if (!(temperature >= 0.f) || !(temperature < INFINITY)) return fail(SA_EINVAL, "temperature must be >= 0 and finite");
    static_assert(sizeof(Segment) == 16 && sizeof(Decision) % 8 == 0, "the workspace's parts are aligned");
    const bool greedy = temperature == 0.f;
    if (greedy) draft = nullptr;   // unused
    if (!target || !out_accepted || !out_tokens || (n > 0 && !tokens)) return fail(SA_EINVAL, "null pointer");
    if (!greedy && (!u_sample || (n > 0 && !u_accept))) return fail(SA_EINVAL, "null uniform numbers");
    if (target_stride < vocab || (draft && draft_stride < vocab)) return fail(SA_EINVAL, "row strides must be at least vocab");
    int most = 0;
    for (int i = 0; counts && i < n_seq; ++i) most = std::max(most, counts[i]);
    if (out_stride < most + 1) return fail(SA_EINVAL, "out_stride must be above the most drafted tokens");
    const size_t out_n = (size_t)n_seq * out_stride * sizeof(int32_t), acc_n = (size_t)n_seq * sizeof(int32_t);
    const size_t target_n = ((size_t)(n + n_seq - 1) * target_stride + vocab) * sizeof(float);
    const size_t draft_n = n ? ((size_t)(n - 1) * draft_stride + vocab) * sizeof(float) : 0;
    struct { const void* p; size_t n; } in[] = {{target, target_n}, {draft, draft_n}, {tokens, (size_t)n * 4},
                                                {greedy ? nullptr : u_accept, (size_t)n * 4},
                                                {greedy ? nullptr : u_sample, (size_t)n_seq * 4}};
    for (const auto& x : in)
        if (overlap(out_tokens, out_n, x.p, x.n) || overlap(out_accepted, acc_n, x.p, x.n))
            return fail(SA_EINVAL, "outputs must not overlap inputs");
    if (overlap(out_tokens, out_n, out_accepted, acc_n)) return fail(SA_EINVAL, "outputs must not overlap each other");
    if (!draft) draft_stride = 0;
    VerifyArgs a{};
    a.n_target = (int)(n + n_seq);
    a.n_draft = draft ? (int)n : 0;
    a.n_seg = segments_of(vocab);
    const long long segs = (long long)(a.n_target + a.n_draft) * a.n_seg;
    // a workgroup per segment while that leaves CUs without one
    const bool split = segs < 4LL * kWaves * 256;
    const long long wgs = split ? segs : (segs + kWaves - 1) / kWaves;
    // a grid has fewer than 2^32 threads
    if (wgs >= (1LL << 32) / kThreads) return fail(SA_EINVAL, "too many logits for one call");
    const size_t need = sa_draft_verify_ws_bytes(n_seq, counts, vocab);
    if (!ws || ws_bytes < need) return fail(SA_ENOMEM, "workspace too small for the segments");
    if (!aligned16(ws)) return fail(SA_EINVAL, "ws must be 16-byte aligned");
    for (const auto& x : in)
        if (overlap(ws, need, x.p, x.n)) return fail(SA_EINVAL, "ws must not overlap inputs");
    if (overlap(ws, need, out_tokens, out_n) || overlap(ws, need, out_accepted, acc_n))
        return fail(SA_EINVAL, "ws must not overlap outputs");
    a.target = target; a.draft = draft; a.tokens = tokens; a.u_accept = u_accept; a.u_sample = u_sample;
    a.target_stride = target_stride; a.draft_stride = draft_stride;
    a.seg = static_cast<Segment*>(ws);
    a.rest = reinterpret_cast<double*>(a.seg + (size_t)(2 * n + n_seq) * a.n_seg);
    a.out_accepted = out_accepted; a.out_tokens = out_tokens; a.out_stride = out_stride;
    a.vocab = vocab;
    a.factor = greedy ? 0.0 : 1.4426950408889634074 / (double)temperature;
    hipStream_t st = as_stream(stream);
    const auto kernel = greedy ? (split ? verify_segments_kernel<true, true> : verify_segments_kernel<true, false>)
                               : (split ? verify_segments_kernel<false, true> : verify_segments_kernel<false, false>);
    hipLaunchKernelGGL(kernel, dim3((unsigned)wgs), dim3(kThreads), 0, st, a);
    SA_CHECK_LAUNCH();
    int at = 0;
    for (a.seq0 = 0; a.seq0 < n_seq; a.seq0 += kRowsPerLaunch) {
        a.n_seq = std::min(kRowsPerLaunch, n_seq - a.seq0);
        a.first[0] = at;
        for (int i = 0; i < a.n_seq; ++i) a.first[i + 1] = a.first[i] + (counts ? counts[a.seq0 + i] : 0);
        at = a.first[a.n_seq];
        if (greedy) {
            hipLaunchKernelGGL(verify_greedy_kernel, dim3(a.n_seq), dim3(kWave), 0, st, a);
            SA_CHECK_LAUNCH();
            continue;
        }
        a.decided = nullptr;
        if (draft && at > a.first[0]) {
            a.decided = reinterpret_cast<Decision*>(a.rest + (size_t)std::min(n_seq, kRowsPerLaunch) * a.n_seg);
            a.groups = std::max(1, std::min(a.n_seg, 8 * device_cu_count() / a.n_seq));
            hipLaunchKernelGGL(verify_decide_kernel, dim3(a.n_seq), dim3(kDraw), 0, st, a);
            SA_CHECK_LAUNCH();
            hipLaunchKernelGGL(verify_rest_kernel, dim3(a.n_seq * a.groups), dim3(kThreads), 0, st, a);
            SA_CHECK_LAUNCH();
        }
        hipLaunchKernelGGL(verify_draw_kernel, dim3(a.n_seq), dim3(kDraw), 0, st, a);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}
