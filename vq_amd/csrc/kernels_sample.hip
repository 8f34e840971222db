// Sampling from rows of scores (vqhip_sample_device in include/vqhip.h).  For a row l of V scores (NaN counts as -inf), with
// m = max l and w_j = exp((l_j - m) / T), in the order of falling l, equal ones by index:
//     S1  the first top_k                                                                  Z1 = sum of w over S1
//     S2  those of S1 whose mass before them is below top_p Z1 (the first always)
//     S3  those of S2 with w_j >= min_p                                                    Z  = sum of w over S3
//     idx = the smallest j of S3 with  sum over { i in S3, i <= j } of w_i  >  u Z,        prob = w_idx / Z
// Every filter keeps a beginning of the order, so S3 is { l > t } and the first r (by index) of { l = t }, and w >= min_p: no
// sort is needed, only the threshold t and the count r, and the draw goes by index, not by order.
//
// Numbers.  The index is an exact answer, so what decides it is computed in more than 32 bits: w in f64, sums in f64 in a fixed
// order, and where masses are added by atomics (the histogram of k_sample_block) as integers, whose sums do not depend on
// the order (w 2^s rounded, s chosen so that V of them fit 63 bits).  Two correct evaluations still part where u Z or top_p Z1
// falls within ~1e-11 of a border.
//
// Two kernels.  Up to 1024 scores: k_sample_wave, a wave per row, the row in registers, no LDS.  Longer rows:
// k_sample_block, a workgroup per row, which first cuts the row down to the few hundred scores the filters are decided
// among and hands those to the same code as a wave's row.
#include <algorithm>
#include <type_traits>

#include "codes_device.h"

namespace vq {

namespace {

struct SampleArgs {
    const void *S;
    uint64_t N, ld;
    uint32_t V;
    int mass_bits;                      // s above
    float temperature, top_p, min_p;    // for every row ...
    uint32_t top_k;
    const float *temperatures, *top_ps, *min_ps;       // ... or one per row, where not null
    const uint32_t *top_ks;
    const float *u;
    uint32_t *idx;
    float *prob;
};

// ---------------------------------------------------------------------------------------------- keys, weights, wave sums
constexpr uint32_t KEY_LEAST = 0x007FFFFFu;            // key of -inf: masked scores and NaN

// Floats in the order of their values as unsigned numbers; -0 and NaN are folded into +0 and -inf.
__device__ __forceinline__ uint32_t key_of(float l)
{
    const uint32_t b = __float_as_uint(l + 0.0f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return l == l ? k : KEY_LEAST;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// exp(x) for x <= 0 (0 for -inf and NaN), relative error below 4e-16: x = n ln 2 + r, |r| <= ln 2 / 2, and the exponential series of
// r to r^12 / 12! (the next term is 1.7e-16)
__device__ __forceinline__ double exp_down(double x)
{
    x = fmax(x, -800.0);
    const double n = rint(x * 1.4426950408889634);
    double r = fma(n, -0.693147180369123816490, x);
    r = fma(n, -1.90821492927058770002e-10, r);
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}

struct Weigh {
    uint32_t top_key;
    double top, inv_t;
    __device__ __forceinline__ double operator()(uint32_t k) const
    {
        const double w = exp_down(((double)value_of(k) - top) * inv_t);
        return k == top_key ? 1.0 : w;                 // (also where the maximum is +inf)
    }
};

// Lanes below move up within the wave by data-parallel primitives: rows of 16 by shifts, then across rows.  Lanes without a
// source add `none`.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t none, uint32_t v)
{
    return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = dpp<CTRL, ROWS>(0u, (uint32_t)b), hi = dpp<CTRL, ROWS>(0u, (uint32_t)(b >> 32));
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double last_lane(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, 63), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63);
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double lane_of(double v, int l)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, l), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
    return __longlong_as_double((long long)(((uint64_t)hi << 32) | lo));
}
__device__ __forceinline__ double wave_scan(double v)              // inclusive
{
    v += dpp<0x111, 0xf>(v);
    v += dpp<0x112, 0xf>(v);
    v += dpp<0x114, 0xf>(v);
    v += dpp<0x118, 0xf>(v);
    v += dpp<0x142, 0xa>(v);
    v += dpp<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v)
{
    v += dpp<0x111, 0xf>(0u, v);
    v += dpp<0x112, 0xf>(0u, v);
    v += dpp<0x114, 0xf>(0u, v);
    v += dpp<0x118, 0xf>(0u, v);
    v += dpp<0x142, 0xa>(0u, v);
    v += dpp<0x143, 0xc>(0u, v);
    return v;
}
__device__ __forceinline__ double wave_total(double v) { return last_lane(wave_scan(v)); }
__device__ __forceinline__ uint32_t wave_total(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(v), 63); }
__device__ __forceinline__ uint32_t wave_max(uint32_t v)
{
    v = max(v, dpp<0x111, 0xf>(0u, v));
    v = max(v, dpp<0x112, 0xf>(0u, v));
    v = max(v, dpp<0x114, 0xf>(0u, v));
    v = max(v, dpp<0x118, 0xf>(0u, v));
    v = max(v, dpp<0x142, 0xa>(0u, v));
    v = max(v, dpp<0x143, 0xc>(0u, v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t wave_min(uint32_t v) { return ~wave_max(~v); }

// ---------------------------------------------------------------------------------------------- a wave's set of scores
// 64 E scores in the order of their index, lane i holding E consecutive ones, weights beside them: a weight of 0 is a score
// that is out (masked, filtered, or padding).  All members are called by the whole wave; what they return is uniform.
template <int E>
struct WaveSet {
    uint32_t key[E];
    double w[E];

    // A step of the search for a threshold inside [lo, hi], lo < hi: the middle of the values, which splits an even spread of
    // scores in half; after `many` steps the middle of the keys, which ends after 32 more however the scores lie.
    __device__ static uint32_t middle(uint32_t lo, uint32_t hi, int step)
    {
        const uint32_t half = lo + (hi - lo) / 2;
        if (step >= 24) return half;
        const uint32_t m = key_of(0.5f * value_of(lo) + 0.5f * value_of(hi));
        return m >= lo && m < hi ? m : half;
    }
    __device__ uint32_t count_above(uint32_t k) const
    {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) n += __popcll(__ballot(w[e] > 0.0 && key[e] > k));
        return n;
    }
    __device__ double mass_above(uint32_t k) const
    {
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) s += key[e] > k ? w[e] : 0.0;
        return wave_total(s);
    }
    __device__ uint32_t least_key() const
    {
        uint32_t m = 0xFFFFFFFFu;
#pragma unroll
        for (int e = 0; e < E; ++e) m = min(m, w[e] > 0.0 ? key[e] : 0xFFFFFFFFu);
        return wave_min(m);
    }
    __device__ uint32_t count_equal(uint32_t k) const
    {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) n += __popcll(__ballot(w[e] > 0.0 && key[e] == k));
        return n;
    }

    // The threshold of the first k in the order; more than k scores are in.
    __device__ void cut_count(uint32_t k, uint32_t top_key, uint32_t &t, uint32_t &r) const
    {
        uint32_t lo = least_key(), hi = top_key;       // fewer than k above hi, k or more above lo - 1
        for (int step = 0; lo < hi; ++step) {
            const uint32_t m = middle(lo, hi, step), n = count_above(m);
            if (n == k) {
                t = m;
                r = 0;
                return;
            }
            if (n < k)
                hi = m;
            else
                lo = m + 1;
        }
        t = lo;
        r = k - count_above(t);
    }

    // The threshold of those whose mass before them in the order is below `border` (> 0): the first always.
    __device__ void cut_mass(double border, uint32_t top_key, uint32_t &t, uint32_t &r, uint32_t &ties) const
    {
        uint32_t lo = least_key(), hi = top_key;       // mass above hi is below the border
        for (int step = 0; lo < hi; ++step) {
            const uint32_t m = middle(lo, hi, step);
            if (mass_above(m) < border)
                hi = m;
            else
                lo = m + 1;
            uint32_t n = 0, some = 0;                  // a single score left inside: it is the threshold
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool in = w[e] > 0.0 && key[e] >= lo && key[e] <= hi;
                n += __popcll(__ballot(in));
                some = max(some, in ? key[e] : 0u);
            }
            if (n == 1) {
                lo = hi = wave_max(some);
                break;
            }
        }
        t = lo;
        ties = count_equal(t);
        double wt = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) wt = key[e] == t ? fmax(wt, w[e]) : wt;
        const uint64_t has = __ballot(wt > 0.0);
        wt = lane_of(wt, __ffsll((unsigned long long)has) - 1);
        const double above = mass_above(t);
        // the j-th of the equal ones (from 0) is kept while above + j wt < border
        r = equal_kept(border - above, wt, ties);
    }
    // The least r in [1, ties] with r wt >= room.
    __device__ static uint32_t equal_kept(double room, double wt, uint32_t ties)
    {
        const double q = ceil(room / wt);
        uint32_t r = q < 1.0 ? 1u : q > (double)ties ? ties : (uint32_t)q;
        if (r > 1 && (double)(r - 1) * wt >= room) --r;
        if (r < ties && (double)r * wt < room) ++r;
        return r;
    }

    // Weights of scores behind the threshold become 0.
    __device__ void apply(uint32_t t, uint32_t r)
    {
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += w[e] > 0.0 && key[e] == t;
        uint32_t before = 0;
        const bool all = wave_total(mine) <= r;
        if (!all) before = wave_scan(mine) - mine;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool eq = w[e] > 0.0 && key[e] == t;
            if (key[e] < t || (eq && !all && before >= r)) w[e] = 0.0;
            before += eq;
        }
    }

    // The filters, then the draw.  -> place of the index drawn in the set, its weight, the sum of the weights.
    __device__ uint32_t draw(uint32_t top_key, uint32_t top_k, float top_p, float min_p, float u, double &drawn, double &total)
    {
        if (top_k > 0 && count_above(KEY_LEAST) > top_k) {
            uint32_t t, r;
            cut_count(top_k, top_key, t, r);
            apply(t, r);
        }
        if (top_p < 1.0f) {
            uint32_t t, r, ties;
            cut_mass((double)top_p * mass_above(KEY_LEAST), top_key, t, r, ties);
            apply(t, r);
        }
        if (min_p > 0.0f) {
            const double least = (double)fminf(min_p, 1.0f);
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = w[e] >= least ? w[e] : 0.0;
        }
        double mine = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += w[e];
        const double upto = wave_scan(mine);
        total = last_lane(upto);
        const double target = (double)u * total;
        // the first lane past the target; should rounding leave the target at the very end, the last lane that holds anything
        const uint64_t some = __ballot(mine > 0.0), hit = __ballot(mine > 0.0 && upto > target);
        const int l = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll(some);
        double before = lane_of(upto - mine, l);
        uint32_t at = 0;
        bool done = false;
        drawn = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const double x = w[e];
            before += x;
            if (!done && x > 0.0) {
                at = e;
                drawn = x;
                done = before > target;
            }
        }
        // (only lane l's walk counts: it started from that lane's own sum)
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, l);
        drawn = lane_of(drawn, l);
        return (uint32_t)l * E + at;
    }
};

struct RowParams {
    float temperature, top_p, min_p, u;
    uint32_t top_k;
    bool greedy;
    __device__ RowParams(const SampleArgs &a, uint64_t i)
    {
        temperature = a.temperatures ? a.temperatures[i] : a.temperature;
        top_p = a.top_ps ? a.top_ps[i] : a.top_p;
        min_p = a.min_ps ? a.min_ps[i] : a.min_p;
        top_k = a.top_ks ? a.top_ks[i] : a.top_k;
        const float v = a.u[i];
        u = v > 0.0f ? fminf(v, 0x1.fffffep-1f) : 0.0f;
        greedy = !(temperature > 0.0f && temperature < INFINITY) || top_k == 1 || top_p <= 0.0f;
        if (!(top_p < 1.0f)) top_p = 1.0f;
        if (!(min_p > 0.0f)) min_p = 0.0f;
    }
};

// ---------------------------------------------------------------------------------------------- a wave per row
constexpr int WAVE_THREADS = 256;

// E consecutive scores per lane; VEC: the rows allow loads of 16 bytes (or of all E where they are fewer)
template <class T, int E, bool VEC>
__global__ void __launch_bounds__(WAVE_THREADS) k_sample_wave(const SampleArgs a)
{
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t waves = (uint64_t)gridDim.x * (WAVE_THREADS / 64);
    for (uint64_t i = (uint64_t)blockIdx.x * (WAVE_THREADS / 64) + (threadIdx.x >> 6); i < a.N; i += waves) {
        const T *row = (const T *)a.S + i * a.ld;
        WaveSet<E> set;
        constexpr int LOAD = 16 / (int)sizeof(T) < E ? 16 / (int)sizeof(T) : E;
        const uint32_t j0 = lane * E;
#pragma unroll
        for (int c = 0; c < E; c += LOAD) {
            if (VEC && j0 + c + LOAD <= a.V) {
                const Pack<T, LOAD * (int)sizeof(T)> v = *(const Pack<T, LOAD * (int)sizeof(T)> *)(row + j0 + c);
#pragma unroll
                for (int e = 0; e < LOAD; ++e) set.key[c + e] = key_of(widen(v.v[e]));
            } else {
#pragma unroll
                for (int e = 0; e < LOAD; ++e) set.key[c + e] = j0 + c + e < a.V ? key_of(widen(row[j0 + c + e])) : KEY_LEAST;
            }
        }
        const RowParams p(a, i);
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) most = max(most, set.key[e]);
        most = wave_max(most);
        uint32_t at = 0;
        float prob = 0.0f;
        if (most > KEY_LEAST) {
            if (p.greedy) {
                uint32_t e1 = E;
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if (set.key[e] == most) e1 = e;
                const int l = __ffsll((unsigned long long)__ballot(e1 < E)) - 1;
                at = (uint32_t)l * E + (uint32_t)__builtin_amdgcn_readlane((int)e1, l);
                prob = 1.0f;
            } else {
                const Weigh weigh{most, (double)value_of(most), 1.0 / (double)p.temperature};
#pragma unroll
                for (int e = 0; e < E; ++e) set.w[e] = weigh(set.key[e]);
                double drawn, total;
                at = set.draw(most, p.top_k, p.top_p, p.min_p, p.u, drawn, total);
                prob = (float)(drawn / total);
            }
        }
        if (lane == 0) {
            a.idx[i] = at;
            if (a.prob) a.prob[i] = prob;
        }
    }
}

// ---------------------------------------------------------------------------------------------- a workgroup per row
constexpr uint32_t LIST = 512;                         // scores the filters are decided among: a wave's set of 8 per lane
constexpr uint32_t SEGMENT = 256;                      // of them from one wave's part of the row
constexpr uint32_t BINS = 2048;                        // histogram of masses, even steps of the score

template <int THREADS>
struct BlockShared {
    static constexpr int WAVES = THREADS / 64;
    union {
        unsigned long long mass[BINS];
        struct {
            uint32_t key[WAVES * SEGMENT], at[WAVES * SEGMENT];
        } segment;
    };
    uint32_t list_key[LIST], list_at[LIST];
    unsigned long long wide[WAVES];
    double sums[WAVES];
    uint32_t words[WAVES];
    uint32_t hist[256];
    unsigned long long hist_mass[256];
    uint32_t n, t, r, ties;
    unsigned long long above;
};

// One row, worked on by a workgroup: all members are called by all its lanes.  The row is dealt to the waves in consecutive
// ranges, a range in steps of 64 PER scores, PER consecutive ones per lane: order of index = (wave, step, lane, place).
template <class T, int THREADS, bool VEC>
struct BlockRow {
    static constexpr int WAVES = THREADS / 64;
    static constexpr int PER = VEC ? 16 / (int)sizeof(T) : 1;
    static constexpr uint32_t STEP = 64 * PER;
    using Shared = BlockShared<THREADS>;

    Shared &sh;
    const T *row;
    uint32_t V;
    int s;
    Weigh weigh;

    __device__ static uint32_t wave() { return threadIdx.x >> 6; }
    __device__ static uint32_t lane() { return threadIdx.x & 63; }
    // this wave's part of [lo, hi)
    __device__ static void part(uint32_t &lo, uint32_t &hi)
    {
        const uint32_t steps = (hi - lo + STEP - 1) / STEP, len = (steps + WAVES - 1) / WAVES * STEP;
        const uint64_t from = (uint64_t)lo + (uint64_t)wave() * len;
        const uint32_t end = hi;
        lo = (uint32_t)min(from, (uint64_t)end);
        hi = (uint32_t)min(from + len, (uint64_t)end);
    }
    // This lane's scores of one step; what lies behind `hi` is a masked score.
    using Piece = Pack<T, PER * (int)sizeof(T)>;
    __device__ __forceinline__ Piece load(uint32_t base, uint32_t hi) const
    {
        const uint32_t j = base + lane() * PER;
        Piece v;
        if (j + PER <= hi) {
            v = *(const Piece *)(row + j);
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e) v.v[e] = j + e < hi ? row[j + e] : (T)-INFINITY;
        }
        return v;
    }
    // f(index of the first, keys) for this lane's scores of one step
    template <class F>
    __device__ __forceinline__ void step_of(uint32_t base, const Piece &v, F &&f) const
    {
        uint32_t key[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) key[e] = key_of(widen(v.v[e]));
        f(base + lane() * PER, key);
    }
    // ... and of all steps of [lo, hi).  FLIGHT steps are on their way at a time: 4 where f is a few instructions; where it
    // computes weights, the one next is, which its hundreds of instructions cover.
    template <uint32_t FLIGHT, class F>
    __device__ __forceinline__ void each(uint32_t lo, uint32_t hi, F &&f) const
    {
        uint32_t base = lo;
        if (FLIGHT == 1) {
            if (base >= hi) return;
            Piece v = load(base, hi);
#pragma unroll 1
            for (; base < hi; base += STEP) {
                const Piece now = v;
                if (hi - base > STEP) v = load(base + STEP, hi);
                step_of(base, now, f);
            }
            return;
        }
#pragma unroll 1
        for (; base < hi && hi - base >= FLIGHT * STEP; base += FLIGHT * STEP) {
            Piece v[FLIGHT];
#pragma unroll
            for (uint32_t q = 0; q < FLIGHT; ++q) v[q] = *(const Piece *)(row + base + q * STEP + lane() * PER);
#pragma unroll
            for (uint32_t q = 0; q < FLIGHT; ++q) step_of(base + q * STEP, v[q], f);
        }
#pragma unroll 1
        for (; base < hi; base += STEP) step_of(base, load(base, hi), f);
    }

    __device__ unsigned long long fixed(double w) const
    {
        // w 2^s + 2^52 has the rounded integer in its mantissa (s <= 51, w <= 1)
        const double d = fma(w, __longlong_as_double((long long)(1023 + s) << 52), 0x1p52);
        return (unsigned long long)__double_as_longlong(d) & 0xFFFFFFFFFFFFFull;
    }

    // Maximum of the row; mine: of what this lane has seen.
    __device__ uint32_t find_top(uint32_t &mine)
    {
        uint32_t lo = 0, hi = V, m = 0;
        part(lo, hi);
        each<4>(lo, hi, [&](uint32_t, const uint32_t (&k)[PER]) {
#pragma unroll
            for (int e = 0; e < PER; ++e) m = max(m, k[e]);
        });
        mine = m;
        m = wave_max(m);
        if (lane() == 0) sh.words[wave()] = m;
        __syncthreads();
        for (int k = 0; k < WAVES; ++k) m = max(m, sh.words[k]);
        __syncthreads();
        return m;
    }

    // The k-th largest (1 <= k <= THREADS) of one key per lane, by 8 bits at a time.
    __device__ uint32_t kth_largest(uint32_t key, uint32_t k)
    {
        uint32_t prefix = 0;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (threadIdx.x < 256) sh.hist[threadIdx.x] = 0;
            __syncthreads();
            if (shift == 24 || (key >> (shift + 8)) == prefix) atomicAdd(&sh.hist[(key >> shift) & 255], 1u);
            __syncthreads();
            uint32_t above;
            const uint32_t b = border_bin(k, above);
            prefix = (prefix << 8) | b;
            k -= above;
            __syncthreads();
        }
        return prefix;
    }
    // Over sh.hist: the bin that holds the k-th from the top, and how many lie in the bins above it.  Every wave for itself.
    __device__ uint32_t border_bin(uint32_t k, uint32_t &above) const
    {
        uint32_t c[4], mine = 0;                       // lane l: bins 255 - 4 l down to 252 - 4 l
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] = sh.hist[255 - 4 * lane() - e];
            mine += c[e];
        }
        const uint32_t upto = wave_scan(mine);
        const uint64_t hit = __ballot(upto >= k);
        const int l = hit ? __ffsll((unsigned long long)hit) - 1 : 63;
        uint32_t run = upto - mine, at = 3, before = run;
        bool done = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (!done) {
                at = e;
                before = run;
                run += c[e];
                done = run >= k;
            }
        }
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, l);
        above = (uint32_t)__builtin_amdgcn_readlane((int)before, l);
        return 255 - 4 * l - at;
    }

    // The scores `in` says, in the order of their index, into the list.  False if they do not fit.
    template <class P>
    __device__ bool collect(P &&in)
    {
        uint32_t lo = 0, hi = V, n = 0;
        part(lo, hi);
        const uint32_t w = wave();
        each<4>(lo, hi, [&](uint32_t j, const uint32_t (&k)[PER]) {
            uint32_t mask = 0;
#pragma unroll
            for (int e = 0; e < PER; ++e) mask |= in(k[e]) ? 1u << e : 0u;
            if (__ballot(mask != 0) == 0) return;
            const uint32_t c = __popc(mask), upto = wave_scan(c);
            uint32_t to = n + upto - c;
#pragma unroll
            for (int e = 0; e < PER; ++e)
                if ((mask >> e) & 1) {
                    if (to < SEGMENT) {
                        sh.segment.key[w * SEGMENT + to] = k[e];
                        sh.segment.at[w * SEGMENT + to] = j + e;
                    }
                    ++to;
                }
            n += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
        });
        if (lane() == 0) sh.words[w] = n;
        __syncthreads();
        uint32_t all = 0, before = 0;
        bool fits = true;
        for (int k = 0; k < WAVES; ++k) {
            before += k < (int)w ? sh.words[k] : 0;
            all += sh.words[k];
            fits = fits && sh.words[k] <= SEGMENT;
        }
        fits = fits && all <= LIST;
        if (fits)
            for (uint32_t q = lane(); q < n; q += 64) {
                sh.list_key[before + q] = sh.segment.key[w * SEGMENT + q];
                sh.list_at[before + q] = sh.segment.at[w * SEGMENT + q];
            }
        if (threadIdx.x == 0) sh.n = all;
        __syncthreads();
        return fits;
    }

    // The list as a wave's set.
    template <int E>
    __device__ void load_list(WaveSet<E> &set) const
    {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t q = lane() * E + e;
            set.key[e] = q < sh.n ? sh.list_key[q] : KEY_LEAST;
            set.w[e] = weigh(set.key[e]);
        }
    }
    template <int E>
    __device__ void draw_from_list(const RowParams &p, uint32_t &at, float &prob)
    {
        WaveSet<E> set;
        load_list(set);
        double drawn, total;
        at = sh.list_at[set.draw(weigh.top_key, p.top_k, p.top_p, p.min_p, p.u, drawn, total)];
        prob = (float)(drawn / total);
    }
    template <int E>
    __device__ void cut_list(double border, uint32_t &t, uint32_t &r, uint32_t &ties)
    {
        WaveSet<E> set;
        load_list(set);
        set.cut_mass(border, weigh.top_key, t, r, ties);
    }

    // Radix selection over the whole row, 8 bits of the key at a time, for the rows the list does not serve (top_k beyond it,
    // a border among more equal or nearly equal scores than it holds).  Kept so far: keys above t and r of those equal to t;
    // on return the shorter beginning.  By count: the first `border`.  By mass: those whose mass before them is below it.
    template <bool MASS>
    __device__ void cut(unsigned long long border, uint32_t &t, uint32_t &r, uint32_t &ties)
    {
        uint32_t prefix = 0, found = 0;
        bool first = true;
        unsigned long long before = 0;
        // the low bits of a widened 16-bit score follow from its sign: 16 of them for bf16, 13 for f16
        constexpr int LAST = sizeof(T) == 4 ? 0 : std::is_same<T, __bf16>::value ? 16 : 8;
        for (int shift = 24; shift >= LAST; shift -= 8) {
            if (threadIdx.x < 256) {
                sh.hist[threadIdx.x] = 0;
                sh.hist_mass[threadIdx.x] = 0;
            }
            __syncthreads();
            uint32_t lo = 0, hi = V;
            part(lo, hi);
            each<1>(lo, hi, [&](uint32_t, const uint32_t (&k)[PER]) {
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    if (k[e] < t || k[e] <= KEY_LEAST || (!first && (k[e] >> (shift + 8)) != prefix)) continue;
                    const uint32_t b = (k[e] >> shift) & 255;
                    atomicAdd(&sh.hist[b], 1u);
                    if (MASS && k[e] > t) atomicAdd(&sh.hist_mass[b], fixed(weigh(k[e])));
                }
            });
            __syncthreads();
            if (threadIdx.x == 0) {
                // of the keys equal to t only r are left
                if (MASS && r != 0 && t > KEY_LEAST && (first || (t >> (shift + 8)) == prefix)) sh.hist_mass[(t >> shift) & 255] += (unsigned long long)r * fixed(weigh(t));
                // the bin of the last element kept: the lowest whose total above it is below the border
                unsigned long long run = before, above = before;
                uint32_t pick = 0;
                bool any = false;
                for (int b = 255; b >= 0; --b) {
                    if (sh.hist[b] == 0) continue;
                    if (run >= border && any) break;
                    any = true;
                    pick = b;
                    above = run;
                    run += MASS ? sh.hist_mass[b] : sh.hist[b];
                }
                sh.n = pick;
                sh.above = above;
                sh.ties = any ? sh.hist[pick] : 0;
            }
            __syncthreads();
            prefix = (prefix << 8) | sh.n;
            before = sh.above;
            found = sh.ties;
            first = false;
            __syncthreads();
        }
        if (found == 0) return;
        uint32_t nt = prefix << LAST;
        if (!(nt >> 31)) nt |= (1u << LAST) - 1u;        // a negative score: the folded bits are ones
        ties = found;
        const uint32_t most = nt == t ? min(found, r) : found;               // the border of an earlier cut
        uint32_t nr;
        if (MASS) {
            const unsigned long long w = fixed(weigh(nt));
            nr = border <= before ? 1 : w == 0 ? most : (uint32_t)min((unsigned long long)most, (border - before + w - 1) / w);
            nr = max(nr, 1u);
        } else {
            nr = (uint32_t)min((unsigned long long)most, border - before);
        }
        t = nt;
        r = nr;
    }

    // Index of the r-th (r >= 1) score equal to t.
    __device__ uint32_t nth_equal(uint32_t t, uint32_t r)
    {
        uint32_t lo = 0, hi = V, n = 0;
        part(lo, hi);
        each<4>(lo, hi, [&](uint32_t, const uint32_t (&k)[PER]) {
#pragma unroll
            for (int e = 0; e < PER; ++e) n += k[e] == t;
        });
        n = wave_total(n);
        if (lane() == 0) sh.words[wave()] = n;
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t k = 0; k < wave(); ++k) before += sh.words[k];
        if (before < r && before + n >= r) {              // this wave's part holds it
            for (uint32_t base = lo; base < hi; base += STEP) {
                bool done = false;
                step_of(base, load(base, hi), [&](uint32_t j, const uint32_t (&k)[PER]) {
                    uint32_t c = 0;
#pragma unroll
                    for (int e = 0; e < PER; ++e) c += k[e] == t;
                    const uint32_t upto = wave_scan(c), here = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
                    if (before + here >= r) {
                        uint32_t at = before + upto - c;
#pragma unroll
                        for (int e = 0; e < PER; ++e) {
                            at += k[e] == t;
                            if (k[e] == t && at == r) sh.n = j + e;
                        }
                        done = true;
                    }
                    before += here;
                });
                if (done) break;
            }
        }
        __syncthreads();
        const uint32_t at = sh.n;
        __syncthreads();
        return at;
    }

    // The draw among keys above t and those equal to t up to index last_equal, with weights of at least `least`.
    __device__ void draw(uint32_t t, uint32_t last_equal, double least, float u, uint32_t &at, float &prob)
    {
        const uint32_t floor_key = max(t, KEY_LEAST + 1);
        auto kept = [&](uint32_t k, uint32_t j) -> double {
            if (k < floor_key || (k == t && j > last_equal)) return 0.0;
            const double x = weigh(k);
            return x >= least ? x : 0.0;
        };
        uint32_t lo = 0, hi = V;
        double before = 0.0, target = 0.0, total = 0.0;
        // sums of the waves' parts, the part the target falls in, its parts, ... down to one step
        for (bool whole = true; whole || hi - lo > STEP; whole = false) {
            uint32_t a = lo, b = hi;
            part(a, b);
            double mine = 0.0;
            each<1>(a, b, [&](uint32_t j, const uint32_t (&k)[PER]) {
#pragma unroll
                for (int e = 0; e < PER; ++e) mine += kept(k[e], j + e);
            });
            mine = wave_total(mine);
            if (lane() == 0) sh.sums[wave()] = mine;
            __syncthreads();
            if (whole) {
                for (int k = 0; k < WAVES; ++k) total += sh.sums[k];
                target = (double)u * total;
            }
            int pick = -1;
            for (int k = 0; k < WAVES; ++k) {
                if (sh.sums[k] == 0.0) continue;
                if (pick >= 0) before += sh.sums[pick];
                pick = k;
                if (before + sh.sums[k] > target) break;
            }
            const uint32_t steps = (hi - lo + STEP - 1) / STEP, len = (steps + WAVES - 1) / WAVES * STEP;
            lo += (uint32_t)pick * len;
            hi = (uint32_t)min((uint64_t)lo + len, (uint64_t)hi);
            __syncthreads();
        }
        step_of(lo, load(lo, hi), [&](uint32_t j, const uint32_t (&k)[PER]) {
            double x[PER], mine = 0.0;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                x[e] = kept(k[e], j + e);
                mine += x[e];
            }
            const double upto = before + wave_scan(mine);
            const uint64_t some = __ballot(mine > 0.0), hit = __ballot(mine > 0.0 && upto > target);
            const int l = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll(some);
            double run = upto - mine, drawn = 0.0;
            uint32_t place = 0;
            bool done = false;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                run += x[e];
                if (!done && x[e] > 0.0) {
                    place = e;
                    drawn = x[e];
                    done = run > target;
                }
            }
            at = (uint32_t)__builtin_amdgcn_readlane((int)(j + place), l);
            prob = (float)(lane_of(drawn, l) / total);
        });
    }
};

template <class T, int THREADS, bool VEC>
__global__ void __launch_bounds__(THREADS) k_sample_block(const SampleArgs a)
{
    using Row = BlockRow<T, THREADS, VEC>;
    constexpr int WAVES = THREADS / 64;
    __shared__ typename Row::Shared sh;
    for (uint64_t i = blockIdx.x; i < a.N; i += gridDim.x) {
        Row row{sh, (const T *)a.S + i * a.ld, a.V, a.mass_bits, {}};
        const RowParams p(a, i);
        uint32_t at = 0, mine;
        float prob = 0.0f;
        const uint32_t top = row.find_top(mine);
        row.weigh = Weigh{top, (double)value_of(top), 1.0 / (double)p.temperature};
        if (top > KEY_LEAST && p.greedy) {
            at = row.nth_equal(top, 1);
            prob = 1.0f;
        } else if (top > KEY_LEAST) {
            uint32_t t = KEY_LEAST, r = 0, ties = 0;
            bool done = false;
            if (p.top_k > 0 && p.top_k < a.V) {
                // The k-th largest of the lanes' own maxima: at least k scores reach it, and few more do, since the largest
                // scores rarely share a lane.
                if (p.top_k <= (THREADS < 1024 ? THREADS / 2 : 256)) {
                    const uint32_t least = max(row.kth_largest(mine, p.top_k), KEY_LEAST + 1);
                    if (row.collect([&](uint32_t k) { return k >= least; })) {
                        if (threadIdx.x < 64) {
                            if (sh.n <= 256)
                                row.template draw_from_list<4>(p, at, prob);
                            else
                                row.template draw_from_list<8>(p, at, prob);
                        }
                        done = true;
                    }
                }
                if (!done) row.template cut<false>(p.top_k, t, r, ties);
            }
            if (!done) {
                if (p.top_p < 1.0f) {
                    // masses by even steps of the score from the maximum down.  All scores more than ln(V / (1 - p)) below it (in
                    // units of T) together weigh less than 1 - p, so the border lies above: that is where the steps are.
                    const float reach = (logf((float)a.V) - logf(fmaxf(1.0f - p.top_p, 0x1p-24f)) + 1.0f) * p.temperature;
                    const float per = (float)BINS / reach, high = value_of(top);
                    auto bin = [&](uint32_t k) {
                        const float below = high - value_of(k);
                        return below > 0.0f ? (uint32_t)fminf(below * per, (float)(BINS - 1)) : 0u;
                    };
                    for (uint32_t b = threadIdx.x; b < BINS; b += THREADS) sh.mass[b] = 0;
                    __syncthreads();
                    uint32_t lo = 0, hi = a.V;
                    row.part(lo, hi);
                    row.template each<1>(lo, hi, [&](uint32_t, const uint32_t (&k)[Row::PER]) {
#pragma unroll
                        for (int e = 0; e < Row::PER; ++e) {
                            if (k[e] <= t) continue;                       // (of the scores equal to t, r are left: added below)
                            const unsigned long long f = row.fixed(row.weigh(k[e]));
                            if (f) atomicAdd(&sh.mass[bin(k[e])], f);
                        }
                    });
                    __syncthreads();
                    if (r != 0 && threadIdx.x == 0) sh.mass[bin(t)] += (unsigned long long)r * row.fixed(row.weigh(t));
                    __syncthreads();
                    // running totals of the bins
                    constexpr uint32_t EACH = BINS / THREADS;
                    unsigned long long sum = 0;
#pragma unroll
                    for (uint32_t e = 0; e < EACH; ++e) sum += sh.mass[threadIdx.x * EACH + e];
                    unsigned long long upto = sum;
                    for (int o = 1; o < 64; o <<= 1) {
                        const unsigned long long y = __shfl_up(upto, o);
                        if ((int)row.lane() >= o) upto += y;
                    }
                    if (row.lane() == 63) sh.wide[row.wave()] = upto;
                    __syncthreads();
                    unsigned long long before = upto - sum, z = 0;
                    for (int k = 0; k < WAVES; ++k) {
                        before += k < (int)row.wave() ? sh.wide[k] : 0;
                        z += sh.wide[k];
                    }
                    const unsigned long long border = (unsigned long long)ceil((double)p.top_p * (double)z);
                    if (before < border && border <= before + sum) {
                        uint32_t b = threadIdx.x * EACH;
                        while (before + sh.mass[b] < border) before += sh.mass[b++];
                        sh.t = b;
                        sh.above = before;
                    }
                    __syncthreads();
                    const uint32_t at_bin = sh.t;
                    const unsigned long long above = sh.above;
                    const bool listed = r == 0 && row.collect([&](uint32_t k) { return k > KEY_LEAST && bin(k) == at_bin; });
                    if (listed) {
                        if (threadIdx.x < 64) {
                            const double room = (double)(border - above) * __longlong_as_double((long long)(1023 - a.mass_bits) << 52);
                            uint32_t t1, r1, n1;
                            if (sh.n <= 256)
                                row.template cut_list<4>(room, t1, r1, n1);
                            else
                                row.template cut_list<8>(room, t1, r1, n1);
                            if (threadIdx.x == 0) {
                                sh.t = t1;
                                sh.r = r1;
                                sh.ties = n1;
                            }
                        }
                        __syncthreads();
                        t = sh.t;
                        r = sh.r;
                        ties = sh.ties;
                    } else {
                        row.template cut<true>(border, t, r, ties);
                    }
                }
                uint32_t last_equal = a.V;
                if (t > KEY_LEAST && r < ties) last_equal = row.nth_equal(t, r);
                __syncthreads();
                row.draw(t, last_equal, p.min_p > 0.0f ? (double)fminf(p.min_p, 1.0f) : 0.0, p.u, at, prob);
            }
        }
        if (threadIdx.x == 0) {
            a.idx[i] = at;
            if (a.prob) a.prob[i] = prob;
        }
        __syncthreads();
    }
}

template <class T, int E>
hipError_t run_wave(const SampleArgs &a, hipStream_t s)
{
    constexpr int LOAD = 16 / (int)sizeof(T) < E ? 16 / (int)sizeof(T) : E;
    const uint64_t align = LOAD * sizeof(T) - 1;
    const bool vec = (((uint64_t)(uintptr_t)a.S | a.ld * sizeof(T)) & align) == 0;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((a.N + WAVE_THREADS / 64 - 1) / (WAVE_THREADS / 64), 1u << 20);
    if (vec)
        hipLaunchKernelGGL((k_sample_wave<T, E, true>), dim3(blocks), dim3(WAVE_THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_sample_wave<T, E, false>), dim3(blocks), dim3(WAVE_THREADS), 0, s, a);
    return hipGetLastError();
}

template <class T, int THREADS>
hipError_t run_block(const SampleArgs &a, hipStream_t s)
{
    const bool vec = (((uint64_t)(uintptr_t)a.S | a.ld * sizeof(T)) & 15) == 0;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(a.N, 1u << 20);
    if (vec)
        hipLaunchKernelGGL((k_sample_block<T, THREADS, true>), dim3(blocks), dim3(THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_sample_block<T, THREADS, false>), dim3(blocks), dim3(THREADS), 0, s, a);
    return hipGetLastError();
}

template <class T>
hipError_t run_sample(const SampleArgs &a, hipStream_t s)
{
    if (a.V <= 256) return run_wave<T, 4>(a, s);
    if (a.V <= 1024) return run_wave<T, 16>(a, s);
    if (a.V <= 8192) return run_block<T, 256>(a, s);
    return run_block<T, 1024>(a, s);
}

}  // namespace

hipError_t launch_sample(const void *dS, int dtype, uint64_t N, uint32_t V, uint64_t ld, const vqhip_sampling &how, const float *du, uint32_t *didx,
                         float *dprob, hipStream_t s)
{
    int log2v = 0;
    while ((1ull << log2v) < V) ++log2v;
    const SampleArgs a{dS, N, ld, V, std::min(51, 62 - log2v), how.temperature, how.top_p, how.min_p, how.top_k, how.dtemperature, how.dtop_p, how.dmin_p,
                       how.dtop_k, du, didx, dprob};
    if (dtype == VQHIP_F32) return run_sample<float>(a, s);
    if (dtype == VQHIP_BF16) return run_sample<__bf16>(a, s);
    return run_sample<_Float16>(a, s);
}

}  // namespace vq
