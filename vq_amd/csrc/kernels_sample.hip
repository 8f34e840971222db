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
// the order: in units of 2^-s of the largest weight a step of the histogram can hold, s chosen so that V of them fit 63 bits.  (Of the
// row's largest weight they would lose long tails: 2^22 scores of weight 2^-42 beside a 1 are 1e-6 of the row, each below half a unit.)
// Two correct evaluations still part where u Z or top_p Z1 falls within ~1e-14 of a border, or V 2^-61 where that is more.
//
// Three kernels.  Up to 64 scores: k_sample_quad, four lanes per row.  Up to 1024: k_sample_wave, a wave per row.  Both hold the row in
// registers and read it once.  Longer rows: k_sample_block, a workgroup per row, which first cuts the row down to the few
// hundred scores the filters are decided among and hands those to the same code as a wave's row; it reads the row three or
// four times, all but the first from the caches.
//
// What bounds them: the vector units, not memory.  A weight in f64 is 23 instructions.  400000 x 256 f32 with top_p 0.9: 233 us, 356 vector
// instructions a row, 92 of them the weights, the units busy all the time (reading the scores once is 89 us at the rate of a large copy).
// 256 x 131072 bf16 with top_p 0.9: 98 us, the units busy 71 %, 74 instructions a score over the four passes, 46 of them its two
// weights.  1 x 131072 bf16 with top_k 50 and top_p 0.9: 19 us, one workgroup's latency.
#include <algorithm>
#include <cfloat>
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

using u32x4s = uint32_t __attribute__((ext_vector_type(4)));
// 16 bytes from any multiple of an element's size
typedef uint32_t words_by4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t words_by2 __attribute__((ext_vector_type(4), aligned(2)));

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

// w = exp((l - top) / T) = 2^z, z = (l - top) log2(e) / T <= 0: 2^n by the exponent, 2^f, |f| <= 1/2, by the exponential series of
// f ln 2 to its 12th power (the next term is 1.7e-16); 0 for -inf and NaN, 1 for the maximum itself, also where that is +inf.
// p f + c with c in scalar registers: left to itself the compiler keeps the constants of a loop in vector registers and copies each
// before a multiply-add that overwrites it, which is half as many instructions again.
__device__ __forceinline__ double horner(double p, double f, double c)
{
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(p), "v"(f), "s"(c));
    return r;
}

// 1 / x to ~2^-46 for x in [2^-149, 2^128): the instruction's 23 bits and one step of Newton's.  A division is eleven instructions.
__device__ __forceinline__ double inverse(double x)
{
    const double r = __builtin_amdgcn_rcp(x);
    return fma(fma(-x, r, 1.0), r, r);
}

struct Weigh {
    float top;
    double scale;                       // log2(e) / T
    __device__ Weigh() {}
    __device__ Weigh(float maximum, float temperature) : top(maximum)
    {
        const double r = inverse((double)temperature), q = 1.4426950408889634 * r;
        scale = fma(fma(-(double)temperature, q, 1.4426950408889634), r, q);
    }
    // FINITE: the maximum is
    template <bool FINITE = false>
    __device__ __forceinline__ double of(float l) const
    {
        const double z = fmax(((double)l - (double)top) * scale, -1100.0), n = rint(z), f = z - n;
        double p = 2.5678435993488206e-11;              // ln2^k / k!
        p = horner(p, f, 4.4455382718708116e-10);
        p = horner(p, f, 7.0549116208011233e-09);
        p = horner(p, f, 1.0178086009239700e-07);
        p = horner(p, f, 1.3215486790144309e-06);
        p = horner(p, f, 1.5252733804059840e-05);
        p = horner(p, f, 1.5403530393381609e-04);
        p = horner(p, f, 1.3333558146428443e-03);
        p = horner(p, f, 9.6181291076284772e-03);
        p = horner(p, f, 5.5504108664821580e-02);
        p = horner(p, f, 2.4022650695910071e-01);
        p = horner(p, f, 6.9314718055994531e-01);
        p = fma(p, f, 1.0);
        p = ldexp(p, (int)n);
        if (FINITE) return p;
        const uint64_t w = (uint64_t)__double_as_longlong(p);
        const uint32_t hi = l == top ? 0x3FF00000u : (uint32_t)(w >> 32);      // (the low half is 0 for the maximum either way)
        return __longlong_as_double((long long)((uint64_t)hi << 32 | (uint32_t)w));
    }
    __device__ __forceinline__ double operator()(float l) const { return of(l); }
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
    // (zero where a lane has no source; rows left out keep what they are given, another zero)
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, ROWS == 0xf);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, ROWS == 0xf);
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
__device__ __forceinline__ double wave_total(double v)
{
    // (as the scan, but that only the last lane has to be right: the rows in between may add what they like)
    v += dpp<0x111, 0xf>(v);
    v += dpp<0x112, 0xf>(v);
    v += dpp<0x114, 0xf>(v);
    v += dpp<0x118, 0xf>(v);
    v += dpp<0x142, 0xf>(v);
    v += dpp<0x143, 0xf>(v);
    return last_lane(v);
}
__device__ __forceinline__ uint32_t wave_total(uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan(v), 63); }
// A lane without a source keeps its own value.  (In assembler, where the shift is part of the comparison; a value written by the
// instruction before needs two cycles until other lanes may read it.)
#define WAVE_EXTREME(op)                                                                                                                          \
    "s_nop 1\n" op " %0, %0, %0 row_shr:1 row_mask:0xf bank_mask:0xf\n"                                                                           \
    "s_nop 1\n" op " %0, %0, %0 row_shr:2 row_mask:0xf bank_mask:0xf\n"                                                                           \
    "s_nop 1\n" op " %0, %0, %0 row_shr:4 row_mask:0xf bank_mask:0xf\n"                                                                           \
    "s_nop 1\n" op " %0, %0, %0 row_shr:8 row_mask:0xf bank_mask:0xf\n"                                                                           \
    "s_nop 1\n" op " %0, %0, %0 row_bcast:15 row_mask:0xa bank_mask:0xf\n"                                                                        \
    "s_nop 1\n" op " %0, %0, %0 row_bcast:31 row_mask:0xc bank_mask:0xf\n"                                                                        \
    "s_nop 1"
__device__ __forceinline__ float wave_max(float v)
{
    asm(WAVE_EXTREME("v_max_f32_dpp") : "+v"(v));
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}
__device__ __forceinline__ float wave_min(float v)
{
    asm(WAVE_EXTREME("v_min_f32_dpp") : "+v"(v));
    return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}
#undef WAVE_EXTREME

// ---------------------------------------------------------------------------------------------- a wave's set of scores
// 64 E scores in the order of their index, lane i holding E consecutive ones, weights beside them.  A score that is out (masked,
// filtered, of no weight, or padding) is -inf and weighs 0.  All members are called by the whole wave; what they return is uniform.
constexpr int SET_BINS = 256;

template <int E>
struct WaveSet {
    float l[E];
    double w[E];

    template <bool FINITE = false>
    __device__ __forceinline__ void weigh_all(const Weigh &weigh)
    {
#pragma unroll
        for (int e = 0; e < E; ++e) w[e] = weigh.of<FINITE>(l[e]);
    }
    __device__ __forceinline__ void drop_weightless()
    {
#pragma unroll
        for (int e = 0; e < E; ++e) l[e] = w[e] > 0.0 ? l[e] : -INFINITY;
    }
    __device__ uint32_t count_above(float x) const
    {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) n += __popcll(__ballot(l[e] > x));
        return n;
    }
    __device__ uint32_t count_equal(float x) const
    {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) n += __popcll(__ballot(l[e] == x));
        return n;
    }
    __device__ double mass() const
    {
        double s = w[0];
#pragma unroll
        for (int e = 1; e < E; ++e) s += w[e];
        return wave_total(s);
    }
    __device__ double mass_above(float x) const
    {
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) s += l[e] > x ? w[e] : 0.0;
        return wave_total(s);
    }
    // the largest score not above x, the least one above x
    __device__ float snap_down(float x) const
    {
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, l[e] <= x ? l[e] : -INFINITY);
        return wave_max(m);
    }
    __device__ float snap_up(float x) const
    {
        float m = INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) m = fminf(m, l[e] > x ? l[e] : INFINITY);
        return wave_min(m);
    }

    // A bracket for cut_mass (by MASS) or cut_count by a histogram over even steps of the score, `span` of it in all, from the maximum `high` down.  Its
    // masses are integers, w 2^21 rounded, which at most 1024 of them put at most 512 off: with 600 to spare on either side
    // the border lies in the bins found, whatever their order of addition; counts are exact.  True if they hold one score alone, the last one
    // kept: hi.
    template <bool MASS>
    __device__ __forceinline__ bool narrow(double border, float high, float span, float &lo, float &hi, uint32_t *bins) const
    {
        static_assert(E <= 16, "at most 1024 scores");
        const float per = (float)SET_BINS * __builtin_amdgcn_rcpf(span);
        const uint32_t lane = threadIdx.x & 63;
        *(uint4 *)&bins[4 * lane] = make_uint4(0, 0, 0, 0);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        uint32_t bin[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            // (a maximum or a step beyond all bounds: inf - inf and 0 * inf go to the first bin)
            bin[e] = (uint32_t)fminf(fmaxf((high - l[e]) * per, 0.0f), (float)(SET_BINS - 1));
            const uint32_t f = MASS ? (uint32_t)fma(w[e], 0x1p21, 0.5) : l[e] > -INFINITY ? 1u : 0u;
            if (bin[e] < SET_BINS - 1) atomicAdd(&bins[bin[e]], f);          // (the last bin holds what the others do not, and is not asked)
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const uint4 c = *(const uint4 *)&bins[4 * lane];
        const uint32_t p0 = c.x, p1 = p0 + c.y, p2 = p1 + c.z, p3 = p2 + c.w, base = wave_scan(p3) - p3;
        auto first = [&](uint32_t x) -> uint32_t {                      // the first bin that brings the total to x
            const uint64_t hit = __ballot(base + p3 >= x);
            if (!hit) return SET_BINS - 1;
            const int q = __ffsll((unsigned long long)hit) - 1;
            const uint32_t in = (base + p0 < x) + (base + p1 < x) + (base + p2 < x);
            return 4 * q + (uint32_t)__builtin_amdgcn_readlane((int)in, q);
        };
        uint32_t b0, b1;
        if (MASS) {
            const double units = border * 0x1p21;
            b0 = first(units > 600.0 ? (uint32_t)(units - 600.0) : 0u);
            b1 = first((uint32_t)fmin(units + 600.0, 4294967295.0));
        } else {
            b0 = b1 = first((uint32_t)border);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        uint64_t lanes = 0;
        uint32_t n = 0;
        float one = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool in = bin[e] - b0 <= b1 - b0;
            const uint64_t m = __ballot(in);
            lanes |= m;
            n += __popcll(m);
            one = in ? l[e] : one;
        }
        if (n == 1) {
            hi = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(one), __ffsll((unsigned long long)lanes) - 1));
            return true;
        }
        float top = -INFINITY, below = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            top = fmaxf(top, bin[e] >= b0 ? l[e] : -INFINITY);
            below = fmaxf(below, bin[e] > b1 ? l[e] : -INFINITY);
        }
        hi = wave_max(top);
        lo = wave_max(below);
        return false;
    }

    // The first k in the order end with the score t, of which r of `ties` are among them; more than k scores are in.
    __device__ void cut_count(uint32_t k, float &t, uint32_t &r, uint32_t &ties, uint32_t *bins) const
    {
        // fewer than k above hi, k or more above lo; hi is one of the scores.  Every step takes at least one value out of the bracket
        // and, where scores are spread evenly, half of them.
        float lo, hi;
        const float high = snap_down(INFINITY);
        if (narrow<false>((double)k, high, high - snap_up(-INFINITY), lo, hi, bins)) {
            t = hi;
            r = ties = 1;
            return;
        }
        for (;;) {
            const float least = snap_up(lo);
            if (least >= hi) break;
            float m = 0.5f * least + 0.5f * hi;
            if (!(m >= least && m < hi)) m = least;
            const uint32_t n = count_above(m);
            if (n == k) {
                t = snap_up(m);
                r = ties = count_equal(t);
                return;
            }
            if (n < k)
                hi = snap_down(m);
            else
                lo = m;
        }
        t = hi;
        ties = count_equal(t);
        r = k - count_above(t);
    }

    // Those whose mass before them in the order is below `border` (> 0), the first always: they end with the score t, of which r of
    // `ties` are among them.  high: the largest score that is in.
    __device__ __forceinline__ void cut_mass(double border, float high, float span, float &t, uint32_t &r, uint32_t &ties, uint32_t *bins) const
    {
        float lo = -INFINITY, hi = high;               // mass above hi below the border, mass above lo not
        if (narrow<true>(border, high, span, lo, hi, bins)) {
            t = hi;
            r = ties = 1;
            return;
        }
        for (;;) {
            const float least = snap_up(lo);
            if (least >= hi) break;
            float m = 0.5f * least + 0.5f * hi;
            if (!(m >= least && m < hi)) m = least;
            if (mass_above(m) < border)
                hi = snap_down(m);
            else
                lo = m;
        }
        t = hi;
        ties = count_equal(t);
        double wt = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) wt = l[e] == t ? w[e] : wt;
        const uint64_t has = __ballot(wt > 0.0);
        wt = lane_of(wt, __ffsll((unsigned long long)has) - 1);
        // the j-th of the equal ones (from 0) is kept while (mass above) + j wt < border
        r = ties == 1 ? 1u : equal_kept(border - mass_above(t), wt, ties);
    }
    // The least r in [1, ties] with r wt >= room.
    __device__ static uint32_t equal_kept(double room, double wt, uint32_t ties)
    {
        const double q = ceil(room / wt);
        uint32_t r = q < 1.0 ? 1u : q > (double)ties ? ties : (uint32_t)q;
        if (r > 1 && (double)(r - 1) * wt >= room) --r;
        if (r < ties && (double)r * wt < room) ++r;
        return (uint32_t)__builtin_amdgcn_readfirstlane((int)r);
    }

    // Scores behind the threshold go out.
    __device__ __forceinline__ void apply(float t, uint32_t r, uint32_t ties)
    {
        if (r < ties) {                                // by index, of the equal ones
            uint32_t mine = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) mine += l[e] == t;
            uint32_t before = wave_scan(mine) - mine;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool eq = l[e] == t;
                if (eq && before >= r) {
                    l[e] = -INFINITY;
                    w[e] = 0.0;
                }
                before += eq;
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool in = l[e] >= t;
            l[e] = in ? l[e] : -INFINITY;
            w[e] = in ? w[e] : 0.0;
        }
    }

    // The filters, then the draw.  -> place of the index drawn in the set, its weight, the sum of the weights.
    __device__ __forceinline__ uint32_t draw(float top, uint32_t top_k, float top_p, float min_p, float u, float reach, uint32_t *bins, double &drawn,
                                             double &total)
    {
        if (top_k > 0) {
            drop_weightless();
            if (count_above(-INFINITY) > top_k) {
                float t;
                uint32_t r, ties;
                cut_count(top_k, t, r, ties, bins);
                apply(t, r, ties);
            }
        }
        if (top_p < 1.0f) {
            float t;
            uint32_t r, ties;
            cut_mass((double)top_p * mass(), top, reach, t, r, ties, bins);
            apply(t, r, ties);
        }
        if (min_p > 0.0f) {
            const double least = (double)fminf(min_p, 1.0f);
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = w[e] >= least ? w[e] : 0.0;
        }
        double mine = w[0];
#pragma unroll
        for (int e = 1; e < E; ++e) mine += w[e];
        const double upto = wave_scan(mine);
        total = last_lane(upto);
        const double target = (double)u * total;
        // the first lane past the target, the first of its scores past it
        const uint64_t past = __ballot(upto > target);
        uint32_t at = E;
        double run = upto - mine;
        drawn = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            run += w[e];
            const bool here = at == E && run > target;
            at = here ? e : at;
            drawn = here ? w[e] : drawn;
        }
        int q = past ? __ffsll((unsigned long long)past) - 1 : 0;
        if (lane_of(drawn, q) > 0.0) {
            at = (uint32_t)__builtin_amdgcn_readlane((int)at, q);
            drawn = lane_of(drawn, q);
            return (uint32_t)q * E + at;
        }
        // rounding has left the target at the very end of a lane's scores, or of all: among those that weigh something, the last where
        // none is past it
        const uint64_t some = __ballot(mine > 0.0), hit = __ballot(mine > 0.0 && upto > target);
        q = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll(some);
        run = upto - mine;
        at = 0;
        bool done = false;
        drawn = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const double x = w[e];
            run += x;
            if (!done && x > 0.0) {
                at = e;
                drawn = x;
                done = run > target;
            }
        }
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, q);
        drawn = lane_of(drawn, q);
        return (uint32_t)q * E + at;
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
    // How far below the maximum the border of a nucleus among V scores lies at most: all scores more than ln(V / (1 - p)) below
    // it (in units of T) together weigh less than 1 - p.
    __device__ float reach(uint32_t V) const { return octaves(V) * 0.6932f * temperature; }
    // ... in powers of two of the weight, a little less (0.6932 > ln 2)
    __device__ float octaves(uint32_t V) const { return __builtin_amdgcn_logf((float)V) - __builtin_amdgcn_logf(fmaxf(1.0f - top_p, 0x1p-24f)) + 1.5f; }
};

// ---------------------------------------------------------------------------------------------- a wave per row
constexpr int WAVE_THREADS = 256;

// E consecutive scores per lane; VEC: the rows allow loads of 16 bytes (or of all E where they are fewer)
template <class T, int E, bool VEC>
__global__ void __launch_bounds__(WAVE_THREADS) k_sample_wave(const SampleArgs a)
{
    // (a wave has turned its row before it needs the bins)
    union PerWave {
        uint32_t bins[SET_BINS];
        float turn[VEC ? 1 : 64 * (E + 1)];
    };
    __shared__ __attribute__((aligned(16))) PerWave sh[WAVE_THREADS / 64];
    PerWave &mine = sh[threadIdx.x >> 6];
    const uint32_t lane = threadIdx.x & 63, j0 = lane * E;
    const uint64_t waves = (uint64_t)gridDim.x * (WAVE_THREADS / 64);
    uint64_t i = (uint64_t)blockIdx.x * (WAVE_THREADS / 64) + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (i >= a.N) return;

    // A row's scores as they come: E consecutive ones a lane, or (where rows do not allow wide loads) 64 consecutive ones a load
    T raw[E];
    auto request = [&](uint64_t at) {
        const T *row = (const T *)a.S + at * a.ld;
        if constexpr (VEC) {
            constexpr int LOAD = 16 / (int)sizeof(T) < E ? 16 / (int)sizeof(T) : E;
#pragma unroll
            for (int c = 0; c < E; c += LOAD) {
                if (j0 + c + LOAD <= a.V) {
                    const Pack<T, LOAD * (int)sizeof(T)> v = *(const Pack<T, LOAD * (int)sizeof(T)> *)(row + j0 + c);
#pragma unroll
                    for (int e = 0; e < LOAD; ++e) raw[c + e] = v.v[e];
                } else {
#pragma unroll
                    for (int e = 0; e < LOAD; ++e) raw[c + e] = j0 + c + e < a.V ? row[j0 + c + e] : (T)-INFINITY;
                }
            }
        } else {
#pragma unroll
            for (int c = 0; c < E; ++c) raw[c] = c * 64 + lane < a.V ? row[c * 64 + lane] : (T)-INFINITY;
        }
    };
    request(i);
    for (;;) {
        WaveSet<E> set;
        if constexpr (VEC) {
#pragma unroll
            for (int e = 0; e < E; ++e) set.l[e] = fmaxf(widen(raw[e]), -INFINITY);                       // (NaN: -inf)
        } else {
            // turned in LDS to E consecutive ones a lane (rows a word longer, so that the lanes' rows begin in different banks)
            float *turn = mine.turn;
#pragma unroll
            for (int c = 0; c < E; ++c) {
                const uint32_t j = c * 64 + lane;
                turn[j / E * (E + 1) + j % E] = fmaxf(widen(raw[c]), -INFINITY);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
            for (int e = 0; e < E; ++e) set.l[e] = turn[lane * (E + 1) + e];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        const bool more = i + waves < a.N;
        if (more) request(i + waves);                  // on its way while this row is worked on
        const RowParams p(a, i);
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, set.l[e]);
        top = wave_max(top);
        uint32_t at = 0;
        float prob = 0.0f;
        if (top > -INFINITY) {
            if (p.greedy) {
                uint32_t e1 = E;
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if (set.l[e] == top) e1 = e;
                const int q = __ffsll((unsigned long long)__ballot(e1 < E)) - 1;
                at = (uint32_t)q * E + (uint32_t)__builtin_amdgcn_readlane((int)e1, q);
                prob = 1.0f;
            } else {
                if (top == INFINITY) {                 // the rows' own order, with a finite maximum
#pragma unroll
                    for (int e = 0; e < E; ++e) set.l[e] = set.l[e] == top ? 0.0f : -INFINITY;
                    top = 0.0f;
                }
                set.template weigh_all<true>(Weigh(top, p.temperature));
                double drawn, total;
                at = set.draw(top, p.top_k, p.top_p, p.min_p, p.u, p.reach(a.V), mine.bins, drawn, total);
                prob = (float)(drawn * inverse(total));
            }
        }
        if (lane == 0) {
            a.idx[i] = at;
            if (a.prob) a.prob[i] = prob;
        }
        if (!more) return;
        i += waves;
    }
}

// ---------------------------------------------------------------------------------------------- four lanes per row
// Short rows: a wave works on 16 of them at once, so that what a row costs beside its weights (sums, extremes, the search for a
// border) is shared by 16.  What the lanes of a row exchange are permutations within four lanes; rows of a wave part ways in
// loops and branches, the lanes of one never do.
template <int CTRL>
__device__ __forceinline__ uint32_t quad(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <int CTRL>
__device__ __forceinline__ float quad(float v) { return __uint_as_float(quad<CTRL>(__float_as_uint(v))); }
template <int CTRL>
__device__ __forceinline__ double quad(double v)
{
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return __longlong_as_double((long long)((uint64_t)quad<CTRL>((uint32_t)(b >> 32)) << 32 | quad<CTRL>((uint32_t)b)));
}
constexpr int NEIGHBOUR = 0xB1, OPPOSITE = 0x4E, LANE = 0x55;        // the lane beside, the pair beside; k LANE: lane k
template <class V>
__device__ __forceinline__ V quad_sum(V v)                           // (the same bits in all four: both sides add the same two)
{
    v += quad<NEIGHBOUR>(v);
    return v + quad<OPPOSITE>(v);
}
__device__ __forceinline__ float quad_max(float v)
{
    v = fmaxf(v, quad<NEIGHBOUR>(v));
    return fmaxf(v, quad<OPPOSITE>(v));
}
__device__ __forceinline__ float quad_min(float v)
{
    v = fminf(v, quad<NEIGHBOUR>(v));
    return fminf(v, quad<OPPOSITE>(v));
}
__device__ __forceinline__ uint32_t quad_min(uint32_t v)
{
    v = min(v, quad<NEIGHBOUR>(v));
    return min(v, quad<OPPOSITE>(v));
}

// A row of up to 4 E scores, lane i of its four holding E consecutive ones, with WaveSet's conventions.
template <int E>
struct QuadSet {
    float l[E];
    double w[E];

    __device__ __forceinline__ uint32_t count_above(float x) const
    {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) n += l[e] > x;
        return quad_sum(n);
    }
    __device__ __forceinline__ uint32_t count_equal(float x) const
    {
        uint32_t n = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) n += l[e] == x;
        return quad_sum(n);
    }
    __device__ __forceinline__ double mass_above(float x) const
    {
        double s = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) s += l[e] > x ? w[e] : 0.0;
        return quad_sum(s);
    }
    __device__ __forceinline__ float snap_down(float x) const
    {
        float m = -INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) m = fmaxf(m, l[e] <= x ? l[e] : -INFINITY);
        return quad_max(m);
    }
    __device__ __forceinline__ float snap_up(float x) const
    {
        float m = INFINITY;
#pragma unroll
        for (int e = 0; e < E; ++e) m = fminf(m, l[e] > x ? l[e] : INFINITY);
        return quad_min(m);
    }
    // Halves the bracket (lo, hi] of scores until hi is the only one in it: below(m) tells that the border lies
    // at or below m.
    template <class Below>
    __device__ __forceinline__ float border(float lo, float hi, Below &&below) const
    {
        for (;;) {
            const float least = snap_up(lo);
            if (least >= hi) return hi;
            float m = 0.5f * least + 0.5f * hi;
            if (!(m >= least && m < hi)) m = least;
            if (below(m))
                hi = snap_down(m);
            else
                lo = m;
        }
    }
    // Scores behind the r-th of those equal to t go out.
    __device__ __forceinline__ void apply(float t, uint32_t r, uint32_t ties)
    {
        if (r < ties) {
            uint32_t mine = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) mine += l[e] == t;
            const uint32_t q = threadIdx.x & 3, n0 = quad<0>(mine), n1 = quad<LANE>(mine), n2 = quad<2 * LANE>(mine);
            uint32_t before = (q > 0 ? n0 : 0) + (q > 1 ? n1 : 0) + (q > 2 ? n2 : 0);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool eq = l[e] == t;
                if (eq && before >= r) {
                    l[e] = -INFINITY;
                    w[e] = 0.0;
                }
                before += eq;
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool in = l[e] >= t;
            l[e] = in ? l[e] : -INFINITY;
            w[e] = in ? w[e] : 0.0;
        }
    }

    // The filters, then the draw: its place in the row and its weight in the lane that holds it (true there).
    __device__ __forceinline__ bool draw(float top, uint32_t top_k, float top_p, float min_p, float u, float reach, uint32_t &place, double &drawn, double &total)
    {
        const uint32_t q = threadIdx.x & 3;
        if (top_k > 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) l[e] = w[e] > 0.0 ? l[e] : -INFINITY;
            if (count_above(-INFINITY) > top_k) {
                const float t = border(-INFINITY, top, [&](float m) { return count_above(m) < top_k; });
                apply(t, top_k - count_above(t), count_equal(t));
            }
        }
        if (top_p < 1.0f) {
            const double room = (double)top_p * mass_above(-INFINITY);
            // (what lies further below the maximum cannot hold the border; the second term: rounding of the difference)
            const float t = border(top - reach - fabsf(top) * 0x1p-22f, top, [&](float m) { return mass_above(m) < room; });
            const uint32_t ties = count_equal(t);
            uint32_t r = 1;
            if (ties > 1) {
                double wt = 0.0;
#pragma unroll
                for (int e = 0; e < E; ++e) wt = l[e] == t ? w[e] : wt;
                // (lanes without one of them have 0, the others the same weight)
                wt = fmax(wt, quad<NEIGHBOUR>(wt));
                wt = fmax(wt, quad<OPPOSITE>(wt));
                const double left = room - mass_above(t), n = ceil(left / wt);
                r = n < 1.0 ? 1u : n > (double)ties ? ties : (uint32_t)n;
                if (r > 1 && (double)(r - 1) * wt >= left) --r;
                if (r < ties && (double)r * wt < left) ++r;
            }
            apply(t, r, ties);
        }
        if (min_p > 0.0f) {
            const double least = (double)fminf(min_p, 1.0f);
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = w[e] >= least ? w[e] : 0.0;
        }
        double mine = w[0];
#pragma unroll
        for (int e = 1; e < E; ++e) mine += w[e];
        const double m0 = quad<0>(mine), m1 = quad<LANE>(mine), m2 = quad<2 * LANE>(mine), m3 = quad<3 * LANE>(mine);
        const double before = (q > 0 ? m0 : 0.0) + (q > 1 ? m1 : 0.0) + (q > 2 ? m2 : 0.0);
        total = m0 + m1 + m2 + m3;
        const double target = (double)u * total;
        // the first lane past the target (u < 1: there is one); should rounding leave the target at the end of its scores, the last of them
        const uint32_t at = quad_min(mine > 0.0 && before + mine > target ? q : 4u);
        double run = before;
        bool done = false;
        place = 0;
        drawn = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const double x = w[e];
            run += x;
            if (!done && x > 0.0) {
                place = q * E + e;
                drawn = x;
                done = run > target;
            }
        }
        return q == at;
    }
};

constexpr int QUAD_THREADS = 256;

// VEC: the rows allow loads of 16 bytes (or of all E where they are fewer)
template <class T, int E, bool VEC>
__global__ void __launch_bounds__(QUAD_THREADS) k_sample_quad(const SampleArgs a)
{
    constexpr int LOAD = VEC ? (16 / (int)sizeof(T) < E ? 16 / (int)sizeof(T) : E) : 1;
    const uint32_t q = threadIdx.x & 3, j0 = q * E;
    for (uint64_t i = (uint64_t)blockIdx.x * (QUAD_THREADS / 4) + (threadIdx.x >> 2); i < a.N; i += (uint64_t)gridDim.x * (QUAD_THREADS / 4)) {
        const T *row = (const T *)a.S + i * a.ld;
        QuadSet<E> set;
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < E; c += LOAD) {
            T raw[LOAD];
            if (j0 + c + LOAD <= a.V) {
                const Pack<T, LOAD * (int)sizeof(T)> v = *(const Pack<T, LOAD * (int)sizeof(T)> *)(row + j0 + c);
#pragma unroll
                for (int e = 0; e < LOAD; ++e) raw[e] = v.v[e];
            } else {
#pragma unroll
                for (int e = 0; e < LOAD; ++e) raw[e] = j0 + c + e < a.V ? row[j0 + c + e] : (T)-INFINITY;
            }
#pragma unroll
            for (int e = 0; e < LOAD; ++e) {
                set.l[c + e] = fmaxf(widen(raw[e]), -INFINITY);                                              // (NaN: -inf)
                top = fmaxf(top, set.l[c + e]);
            }
        }
        top = quad_max(top);
        const RowParams p(a, i);
        uint32_t at = 0;
        float prob = 0.0f;
        bool own = q == 0;
        if (top > -INFINITY) {
            if (p.greedy) {
                at = 4 * E;
#pragma unroll
                for (int e = E - 1; e >= 0; --e)
                    if (set.l[e] == top) at = j0 + e;
                at = quad_min(at);
                prob = 1.0f;
            } else {
                if (top == INFINITY) {                 // the rows' own order, with a finite maximum
#pragma unroll
                    for (int e = 0; e < E; ++e) set.l[e] = set.l[e] == top ? 0.0f : -INFINITY;
                    top = 0.0f;
                }
                const Weigh weigh(top, p.temperature);
#pragma unroll
                for (int e = 0; e < E; ++e) set.w[e] = weigh.of<true>(set.l[e]);
                double drawn, total;
                own = set.draw(top, p.top_k, p.top_p, p.min_p, p.u, p.reach(a.V), at, drawn, total);
                prob = (float)(drawn * inverse(total));
            }
        }
        if (own) {
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
            float l[WAVES * SEGMENT];
            uint32_t at[WAVES * SEGMENT];
        } segment;
    };
    float list_l[LIST];
    uint32_t list_at[LIST];
    unsigned long long wide[WAVES], above, own;
    double sums[WAVES], room;
    float queue[WAVES][64 + 64 * 8];    // scores of the draw on their way to a full wave
    uint32_t words[WAVES], hist[256];
    __attribute__((aligned(16))) uint32_t bins[SET_BINS];
    uint32_t n, pick, found;
    float t;
};
// One per workgroup, the same for the kernel and the functions it calls.
template <class T, int THREADS>
__device__ __forceinline__ BlockShared<THREADS> &block_shared()
{
    __shared__ BlockShared<THREADS> sh;
    return sh;
}

// Scalars that are the same in all lanes, told to the compiler (arguments of a called function are not).
__device__ __forceinline__ uint32_t same(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ float same(float v) { return __uint_as_float(same(__float_as_uint(v))); }
__device__ __forceinline__ uint64_t same(uint64_t v) { return (uint64_t)same((uint32_t)(v >> 32)) << 32 | same((uint32_t)v); }
__device__ __forceinline__ double same(double v) { return __longlong_as_double((long long)same((uint64_t)__double_as_longlong(v))); }

// A cut of the order: it ends with the score t, of which r of `ties` are kept, the last of them at position `last` (EVERY: all of
// them; UNKNOWN: it has to be looked for).  t = -inf: not cut.
constexpr uint32_t EVERY = 0xFFFFFFFFu, UNKNOWN = 0xFFFFFFFEu;
struct Cut {
    float t;
    uint32_t r, ties, last;
};
struct Drawn {
    uint32_t at;
    float prob;
};

// Even steps of the score, BINS of them over `reach` from the maximum down, what lies further down in the last.
struct Steps {
    float high, per;                    // per: steps per unit of the score
    uint32_t fall;                      // powers of two that a weight falls by in a step, in units of 2^-20
    __device__ Steps() : high(0.0f), per(0.0f), fall(0) {}
    __device__ Steps(float maximum, float reach, float octaves) : high(maximum), per(fminf((float)BINS / reach, FLT_MAX)), fall((uint32_t)(octaves * (0x1p20f / (float)BINS))) {}
    __device__ __forceinline__ uint32_t of(float l) const { return (uint32_t)fminf(fmaxf((high - l) * per, 0.0f), (float)(BINS - 1)); }      // (inf - inf: the first)
    // Weights of step b are at most 2^-down(b), but for rounding: the step's largest or, where `per` was cut, less.
    __device__ __forceinline__ int down(uint32_t b) const { return (int)(b * fall >> 20); }
};

// One row, worked on by a workgroup: all members are called by all its lanes.  The row is dealt to the waves in consecutive
// ranges, a range in steps of 64 PER scores, PER consecutive ones per lane: order of index = (wave, step, lane, place).  Rows
// begin anywhere, and are read 16 bytes at a time from there on: how a row is dealt, and with it the last bits of its sums, does not
// depend on where it lies.
template <class T, int THREADS>
struct BlockRow {
    static constexpr int WAVES = THREADS / 64;
    static constexpr int PER = 16 / (int)sizeof(T);
    static constexpr uint32_t STEP = 64 * PER;
    using Piece = Pack<T, PER * (int)sizeof(T)>;
    using GlobalT = const __attribute__((address_space(1))) T;
    using Global16 = const __attribute__((address_space(1))) typename std::conditional<sizeof(T) == 4, words_by4, words_by2>::type;

    uint64_t row;                       // address of the first score in global memory
    uint32_t V;
    int s;
    Weigh weigh;

    __device__ __forceinline__ static BlockShared<THREADS> &shared() { return block_shared<T, THREADS>(); }
    __device__ __forceinline__ BlockRow uniform() const
    {
        BlockRow b;
        b.row = same(row);
        b.V = same(V);
        b.s = (int)same((uint32_t)s);
        b.weigh.top = same(weigh.top);
        b.weigh.scale = same(weigh.scale);
        return b;
    }
    __device__ __forceinline__ static uint32_t wave() { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }
    __device__ __forceinline__ static uint32_t lane() { return threadIdx.x & 63; }
    // this wave's part of [lo, hi)
    __device__ __forceinline__ static void part(uint32_t &lo, uint32_t &hi)
    {
        const uint32_t steps = (hi - lo + STEP - 1) / STEP, len = (steps + WAVES - 1) / WAVES * STEP;
        const uint64_t from = (uint64_t)lo + (uint64_t)wave() * len;
        const uint32_t end = hi;
        lo = (uint32_t)min(from, (uint64_t)end);
        hi = (uint32_t)min(from + len, (uint64_t)end);
    }
    __device__ __forceinline__ Piece load_whole(uint32_t j) const { return __builtin_bit_cast(Piece, (u32x4s)*(Global16 *)(row + (uint64_t)j * sizeof(T))); }
    // This lane's scores of one step; what lies behind `hi` is a masked score.
    __device__ __forceinline__ Piece load(uint32_t base, uint32_t hi) const
    {
        const uint32_t j = base + lane() * PER;
        if (j + PER <= hi) return load_whole(j);
        Piece v;
#pragma unroll
        for (int e = 0; e < PER; ++e) v.v[e] = j + e < hi ? ((GlobalT *)row)[j + e] : (T)-INFINITY;
        return v;
    }
    // f(position of the first, scores) for this lane's scores of one step
    template <class F>
    __device__ __forceinline__ void step_of(uint32_t base, const Piece &v, F &&f) const
    {
        float l[PER];
#pragma unroll
        for (int e = 0; e < PER; ++e) l[e] = widen(v.v[e]);
        f(base + lane() * PER, l);
    }
    // ... and of all steps of [lo, hi).  FLIGHT steps are on their way at a time: 8 where f is a few instructions; where it
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
            for (uint32_t q = 0; q < FLIGHT; ++q) v[q] = load_whole(base + q * STEP + lane() * PER);
#pragma unroll
            for (uint32_t q = 0; q < FLIGHT; ++q) step_of(base + q * STEP, v[q], f);
        }
#pragma unroll 1
        for (; base < hi; base += STEP) step_of(base, load(base, hi), f);
    }

    // A weight of step b in units of 2^-(s + down(b)).
    __device__ __forceinline__ unsigned long long fixed(double w, const Steps &steps, uint32_t b) const
    {
        // w 2^(s + down) + 2^52 has the rounded integer in its mantissa (s <= 51); the power's exponent is s + b fall's whole part
        const uint32_t power = (__umul24(b, steps.fall) + ((uint32_t)(1023 + s) << 20)) & 0xFFF00000u;
        const double d = fma(w, __longlong_as_double((long long)((uint64_t)power << 32)), 0x1p52);
        return (unsigned long long)__double_as_longlong(d) & 0xFFFFFFFFFFFFFull;
    }

    // Maximum of the row; mine: of what this lane has seen.  (fmaxf passes NaN over.)
    __device__ __forceinline__ float find_top(float &mine) const
    {
        auto &sh = shared();
        uint32_t lo = 0, hi = V;
        part(lo, hi);
        float high = -INFINITY;
        each<8>(lo, hi, [&](uint32_t, const float (&l)[PER]) {
#pragma unroll
            for (int e = 0; e < PER; ++e) high = fmaxf(high, l[e]);
        });
        mine = high;
        high = wave_max(high);
        if (lane() == 0) sh.words[wave()] = __float_as_uint(high);
        __syncthreads();
        for (int k = 0; k < WAVES; ++k) high = fmaxf(high, __uint_as_float(sh.words[k]));
        __syncthreads();
        return same(high + 0.0f);
    }

    // The k-th largest (1 <= k <= THREADS) of one key per lane, by 8 bits at a time.
    __device__ __forceinline__ uint32_t kth_largest(uint32_t key, uint32_t k) const
    {
        auto &sh = shared();
        uint32_t prefix = 0;
#pragma unroll 1
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
    __device__ __forceinline__ uint32_t border_bin(uint32_t k, uint32_t &above) const
    {
        auto &sh = shared();
        uint32_t c[4], mine = 0;                       // lane l: bins 255 - 4 l down to 252 - 4 l
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            c[e] = sh.hist[255 - 4 * lane() - e];
            mine += c[e];
        }
        const uint32_t upto = wave_scan(mine);
        const uint64_t hit = __ballot(upto >= k);
        const int q = hit ? __ffsll((unsigned long long)hit) - 1 : 63;
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
        at = (uint32_t)__builtin_amdgcn_readlane((int)at, q);
        above = (uint32_t)__builtin_amdgcn_readlane((int)before, q);
        return 255 - 4 * q - at;
    }

    // Over sh.mass, whose bins are in the order of falling scores: this lane's consecutive bins, what lies in front of them and the sum
    // of all.
    struct Totals {
        unsigned long long before, own, all;
    };
    __device__ __forceinline__ Totals totals() const
    {
        auto &sh = shared();
        constexpr uint32_t EACH = BINS / THREADS;
        Totals n{0, 0, 0};
#pragma unroll
        for (uint32_t e = 0; e < EACH; ++e) n.own += sh.mass[threadIdx.x * EACH + e];
        unsigned long long upto = n.own;
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned long long y = __shfl_up(upto, o);
            if ((int)lane() >= o) upto += y;
        }
        if (lane() == 63) sh.wide[wave()] = upto;
        __syncthreads();
        n.before = upto - n.own;
        for (int k = 0; k < WAVES; ++k) {
            n.before += k < (int)wave() ? sh.wide[k] : 0;
            n.all += sh.wide[k];
        }
        return n;
    }
    // The bin that brings the running total to `border` (1 <= border <= the sum of all), what lies in front of it, and its own.
    __device__ __forceinline__ uint32_t border_of(const Totals &n, unsigned long long border, unsigned long long &above, unsigned long long &own) const
    {
        auto &sh = shared();
        if (n.before < border && border <= n.before + n.own) {
            unsigned long long before = n.before;
            uint32_t b = threadIdx.x * (BINS / THREADS);
            while (before + sh.mass[b] < border) before += sh.mass[b++];
            sh.pick = b;
            sh.above = before;
            sh.own = sh.mass[b];
        }
        __syncthreads();
        const uint32_t at = same(sh.pick);
        above = same((uint64_t)sh.above);
        own = same((uint64_t)sh.own);
        __syncthreads();
        return at;
    }

    // The scores in [least, most] that `in` says, in the order of their index, into the list.  False if they do not fit.
    template <class P>
    __device__ __forceinline__ bool collect(float least, float most, P &&in) const
    {
        auto &sh = shared();
        uint32_t lo = 0, hi = V, n = 0;
        part(lo, hi);
        const uint32_t w = wave();
        each<8>(lo, hi, [&](uint32_t j, const float (&l)[PER]) {
            bool some = false;
#pragma unroll
            for (int e = 0; e < PER; ++e) some |= l[e] >= least && l[e] <= most;
            if (__ballot(some) == 0) return;
            uint32_t mask = 0;
#pragma unroll
            for (int e = 0; e < PER; ++e) mask |= l[e] >= least && l[e] <= most && in(l[e]) ? 1u << e : 0u;
            const uint32_t c = __popc(mask), upto = wave_scan(c);
            uint32_t to = n + upto - c;
#pragma unroll
            for (int e = 0; e < PER; ++e)
                if ((mask >> e) & 1) {
                    if (to < SEGMENT) {
                        sh.segment.l[w * SEGMENT + to] = l[e];
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
                sh.list_l[before + q] = sh.segment.l[w * SEGMENT + q];
                sh.list_at[before + q] = sh.segment.at[w * SEGMENT + q];
            }
        if (threadIdx.x == 0) sh.n = all;
        __syncthreads();
        return same((uint32_t)fits) != 0;
    }

    // The list as a wave's set.
    template <int E, bool WEIGH = true>
    __device__ __forceinline__ void load_list(WaveSet<E> &set) const
    {
        auto &sh = shared();
        const uint32_t n = same(sh.n);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t q = lane() * E + e;
            set.l[e] = q < n ? sh.list_l[q] : -INFINITY;
        }
        if (WEIGH) {
            set.weigh_all(weigh);
            set.drop_weightless();
        }
    }
};

// The parts of a row's work that a row needs once at most, as functions of their own: one kernel with all of them in line does not
// fit its registers.
template <class Row, int E>
__device__ __attribute__((noinline)) Drawn list_draw(const Row r, const RowParams p)
{
    const Row row = r.uniform();
    WaveSet<E> set;
    row.load_list(set);
    double drawn, total;
    const uint32_t q = set.draw(row.weigh.top, same(p.top_k), same(p.top_p), same(p.min_p), same(p.u), same(p.reach(row.V)), Row::shared().bins, drawn, total);
    return {Row::shared().list_at[q], (float)(drawn * inverse(total))};
}

template <class Row, int E, bool MASS>
__device__ __attribute__((noinline)) Cut list_cut(const Row r, double border)
{
    const Row row = r.uniform();
    WaveSet<E> set;
    row.template load_list<E, MASS>(set);
    Cut c;
    if (MASS) {
        const float high = set.snap_down(INFINITY), low = set.snap_up(-INFINITY);
        set.cut_mass(same(border), high, high > low ? high - low : 1.0f, c.t, c.r, c.ties, Row::shared().bins);
    } else {
        set.cut_count((uint32_t)same(border), c.t, c.r, c.ties, Row::shared().bins);
    }
    c.last = EVERY;
    if (c.r < c.ties) {                                // (all of the row's scores equal to t are in the list)
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) mine += set.l[e] == c.t;
        uint32_t before = wave_scan(mine) - mine, at = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool eq = set.l[e] == c.t;
            before += eq;
            if (eq && before == c.r) at = Row::lane() * E + e + 1;
        }
        const uint64_t hit = __ballot(at != 0);
        c.last = Row::shared().list_at[(uint32_t)__builtin_amdgcn_readlane((int)at, __ffsll((unsigned long long)hit) - 1) - 1];
    }
    return c;
}

// The cut among the scores of the list, by the first wave, told to all.
template <class Row, bool MASS>
__device__ __forceinline__ Cut cut_of_list(const Row row, double border)
{
    auto &sh = Row::shared();
    if (threadIdx.x < 64) {
        const Cut c = sh.n <= 256 ? list_cut<Row, 4, MASS>(row, border) : list_cut<Row, 8, MASS>(row, border);
        if (threadIdx.x == 0) {
            sh.t = c.t;
            sh.pick = c.r;
            sh.found = c.ties;
            sh.n = c.last;
        }
    }
    __syncthreads();
    const Cut c{same(sh.t), same(sh.pick), same(sh.found), same(sh.n)};
    __syncthreads();
    return c;
}

// Radix selection over the whole row, up to 11 bits of the ordered key at a time, for the rows the list does not serve at once
// (top_k beyond it, a border among more equal or nearly equal scores than it holds).  `old`: an earlier cut.  By count: the
// first `border`; by mass: those whose mass before them is below it.  (Digits of 8 bits are the sign and seven of the exponent
// first: a handful of bins, at whose addresses the additions queue.)  By mass: among the scores of step `at`, in its units.
template <class Row, class T, int THREADS, bool MASS>
__device__ __attribute__((noinline)) Cut radix_cut(const Row r0, unsigned long long border, const Cut o, const Steps st, uint32_t at)
{
    const Row row = r0.uniform();
    auto &sh = Row::shared();
    border = same((uint64_t)border);
    at = same(at);
    Steps steps;
    steps.high = same(st.high);
    steps.per = same(st.per);
    steps.fall = same(st.fall);
    const Cut old{same(o.t), same(o.r), same(o.ties), 0};
    const uint32_t t = key_of(old.t);
    // the low bits of a widened 16-bit score follow from its sign: 16 of them for bf16, 13 for f16
    constexpr int LAST = sizeof(T) == 4 ? 0 : std::is_same<T, __bf16>::value ? 16 : 13;
    uint32_t prefix = 0;
    unsigned long long above = 0, own = 0;
    int shift = 32;
    bool listed = false;
#pragma unroll 1
    while (shift > LAST) {
        const int from = shift, bits = min(11, from - LAST);
        shift -= bits;
        for (uint32_t b = threadIdx.x; b < BINS; b += THREADS) sh.mass[b] = 0;
        __syncthreads();
        const uint32_t mask = (1u << bits) - 1;
        auto ours = [&](uint32_t k) { return from == 32 || (k >> (from & 31)) == prefix; };
        uint32_t lo = 0, hi = row.V;
        Row::part(lo, hi);
        row.template each<MASS ? 1 : 4>(lo, hi, [&](uint32_t, const float (&l)[Row::PER]) {
#pragma unroll
            for (int e = 0; e < Row::PER; ++e) {
                const uint32_t k = key_of(l[e]);
                if (k <= KEY_LEAST || k < t || (MASS && (k == t || steps.of(l[e]) != at)) || !ours(k)) continue;
                atomicAdd(&sh.mass[mask - ((k >> shift) & mask)], MASS ? row.fixed(row.weigh(l[e]), steps, at) : 1ull);
            }
        });
        __syncthreads();
        if (MASS && old.r != 0 && steps.of(old.t) == at && ours(t)) {       // of the scores equal to t only r are left
            if (threadIdx.x == 0) sh.mass[mask - ((t >> shift) & mask)] += (unsigned long long)old.r * row.fixed(row.weigh(old.t), steps, at);
            __syncthreads();
        }
        const typename Row::Totals n = row.totals();
        const unsigned long long rest = border - above;
        if (rest > n.all) return o;                    // (by count: the row has no more)
        unsigned long long front;
        const uint32_t d = mask - row.border_of(n, rest, front, own);
        prefix = from == 32 ? d : prefix << bits | d;
        above += front;
        if (!MASS && shift > LAST && own <= LIST && !listed) {               // few are left: to the list (once: one wave may hold too many of them)
            listed = true;
            const uint32_t first = max(prefix << shift, KEY_LEAST + 1), last = min(prefix << shift | ((1u << shift) - 1), key_of(INFINITY));
            if (row.collect(value_of(first), value_of(last), [&](float l) { return key_of(l) >> shift == prefix; })) return cut_of_list<Row, false>(row, (double)(border - above));
        }
    }
    uint32_t nt = prefix << LAST;
    if (!(nt >> 31)) nt |= (1u << LAST) - 1u;          // a negative score: the folded bits are ones
    Cut c{value_of(nt), 0, 0, EVERY};
    uint32_t lo = 0, hi = row.V, ties = 0;
    if (MASS) {
        Row::part(lo, hi);
        row.template each<8>(lo, hi, [&](uint32_t, const float (&l)[Row::PER]) {
#pragma unroll
            for (int e = 0; e < Row::PER; ++e) ties += l[e] == c.t;
        });
        ties = wave_total(ties);
        if (Row::lane() == 0) sh.words[Row::wave()] = ties;
        __syncthreads();
        for (int k = 0; k < Row::WAVES; ++k) c.ties += sh.words[k];
        __syncthreads();
        c.ties = same(c.ties);
        const uint32_t most = nt == t ? min(c.ties, old.r) : c.ties;         // the border of an earlier cut
        const unsigned long long w = row.fixed(row.weigh(c.t), steps, at);
        c.r = (uint32_t)min((unsigned long long)most, (border - above + w - 1) / max(w, 1ull));
        c.r = max(c.r, 1u);
    } else {
        c.ties = (uint32_t)own;
        c.r = (uint32_t)(border - above);
    }
    if (c.r < c.ties) c.last = UNKNOWN;
    return c;
}

// Position of the r-th (r >= 1) score equal to v.
template <class Row>
__device__ __attribute__((noinline)) uint32_t nth_equal(const Row r0, float v, uint32_t r)
{
    const Row row = r0.uniform();
    auto &sh = Row::shared();
    v = same(v);
    r = same(r);
    uint32_t lo = 0, hi = row.V, n = 0;
    Row::part(lo, hi);
    row.template each<8>(lo, hi, [&](uint32_t, const float (&l)[Row::PER]) {
#pragma unroll
        for (int e = 0; e < Row::PER; ++e) n += l[e] == v;
    });
    n = wave_total(n);
    if (Row::lane() == 0) sh.words[Row::wave()] = n;
    __syncthreads();
    uint32_t before = 0;
    for (uint32_t k = 0; k < Row::wave(); ++k) before += sh.words[k];
    before = same(before);
    if (before < r && before + n >= r) {                  // this wave's part holds it
        for (uint32_t base = lo; base < hi; base += Row::STEP) {
            bool done = false;
            row.step_of(base, row.load(base, hi), [&](uint32_t j, const float (&l)[Row::PER]) {
                uint32_t c = 0;
#pragma unroll
                for (int e = 0; e < Row::PER; ++e) c += l[e] == v;
                const uint32_t upto = wave_scan(c), here = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
                if (before + here >= r) {
                    uint32_t at = before + upto - c;
#pragma unroll
                    for (int e = 0; e < Row::PER; ++e) {
                        at += l[e] == v;
                        if (l[e] == v && at == r) sh.n = j + e;
                    }
                    done = true;
                }
                before += here;
            });
            if (done) break;
        }
    }
    __syncthreads();
    const uint32_t at = same(sh.n);
    __syncthreads();
    return at;
}

// The draw among scores above `edge` and those equal to it up to position last_equal (edge = -inf: all), with weights of at least
// `least`, which scores below `from` do not have.
template <class Row, int THREADS>
__device__ __attribute__((noinline)) Drawn row_draw(const Row r0, float edge, uint32_t last_equal, double least, float from, float u)
{
    constexpr int WAVES = THREADS / 64, PER = Row::PER;
    const Row row = r0.uniform();
    auto &sh = Row::shared();
    edge = same(edge);
    last_equal = same(last_equal);
    least = same(least);
    u = same(u);
    const bool all = edge == -INFINITY && least == 0.0;
    const float floor = fmaxf(fmaxf(edge, -FLT_MAX), same(from));
    auto in = [&](float l, uint32_t j) { return l >= floor && !(l == edge && j > last_equal); };
    auto weight = [&](float l) {
        const double x = row.weigh(l);
        return x >= least ? x : 0.0;
    };
    uint32_t lo = 0, hi = row.V;
    double before = 0.0, target = 0.0, total = 0.0;
    // sums of the waves' parts, the part the target falls in, its parts, ... down to one step
    for (bool whole = true; whole || hi - lo > Row::STEP; whole = false) {
        uint32_t a = lo, b = hi;
        Row::part(a, b);
        double mine = 0.0;
        if (all) {
            row.template each<1>(a, b, [&](uint32_t, const float (&l)[PER]) {
#pragma unroll
                for (int e = 0; e < PER; ++e) mine += row.weigh(l[e]);
            });
        } else {
            // few scores are in: they queue up until a whole wave of them can be weighed at once
            float *queue = sh.queue[Row::wave()];
            uint32_t n = 0;
            row.template each<4>(a, b, [&](uint32_t j, const float (&l)[PER]) {
#pragma unroll
                for (int e = 0; e < PER; ++e) {
                    bool is = l[e] >= floor;
                    if (last_equal != EVERY) is = is && !(l[e] == edge && j + e > last_equal);
                    const uint64_t m = __ballot(is);
                    if (is) queue[n + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0))] = l[e];
                    n += __popcll(m);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                while (n >= 64) {                      // from the end: what stays is in front
                    n -= 64;
                    mine += weight(queue[n + Row::lane()]);
                }
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            });
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (Row::lane() < n) mine += weight(queue[Row::lane()]);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        mine = wave_total(mine);
        if (Row::lane() == 0) sh.sums[Row::wave()] = mine;
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
        pick = max(pick, 0);                           // (the maximum is always in: there is a sum)
        const uint32_t steps = (hi - lo + Row::STEP - 1) / Row::STEP, len = (steps + WAVES - 1) / WAVES * Row::STEP;
        lo = same(lo + (uint32_t)pick * len);
        hi = same((uint32_t)min((uint64_t)lo + len, (uint64_t)hi));
        __syncthreads();
    }
    Drawn d;
    row.step_of(lo, row.load(lo, hi), [&](uint32_t j, const float (&l)[PER]) {
        double x[PER], mine = 0.0;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            x[e] = in(l[e], j + e) ? weight(l[e]) : 0.0;
            mine += x[e];
        }
        const double upto = before + wave_scan(mine);
        const uint64_t some = __ballot(mine > 0.0), hit = __ballot(mine > 0.0 && upto > target);
        const int q = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll(some);
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
        d.at = (uint32_t)__builtin_amdgcn_readlane((int)(j + place), q);
        d.prob = (float)(lane_of(drawn, q) * inverse(total));
    });
    return d;
}

// The nucleus of a row with none or a count cut: masses by even steps of the score, from the maximum down to where the border
// can be; then the scores of the step it falls in.
template <class Row, class T, int THREADS>
__device__ __attribute__((noinline)) Cut mass_cut(const Row r0, float top_p, float reach, float octaves, const Cut o)
{
    const Row row = r0.uniform();
    auto &sh = Row::shared();
    const Cut old{same(o.t), same(o.r), same(o.ties), 0};
    top_p = same(top_p);
    const Steps steps(row.weigh.top, same(reach), same(octaves));
    for (uint32_t b = threadIdx.x; b < BINS; b += THREADS) sh.mass[b] = 0;
    __syncthreads();
    // the last bin, most of a row's scores, in registers: its additions would queue at one address
    unsigned long long rest = 0;
    uint32_t lo = 0, hi = row.V;
    Row::part(lo, hi);
    row.template each<1>(lo, hi, [&](uint32_t, const float (&l)[Row::PER]) {
#pragma unroll
        for (int e = 0; e < Row::PER; ++e) {
            const uint32_t b = steps.of(l[e]);
            const unsigned long long f = row.fixed(row.weigh(l[e] > old.t ? l[e] : -INFINITY), steps, b);  // (of the scores equal to old.t, r are left: added below)
            if (b < BINS - 1)
                atomicAdd(&sh.mass[b], f);
            else
                rest += f;
        }
    });
    if (rest) atomicAdd(&sh.mass[BINS - 1], rest);
    __syncthreads();
    if (old.r != 0 && threadIdx.x == 0) {
        const uint32_t b = steps.of(old.t);
        sh.mass[b] += (unsigned long long)old.r * row.fixed(row.weigh(old.t), steps, b);
    }
    __syncthreads();
    // The bins' masses as numbers, summed in a fixed order: the border, the bin that reaches it and the mass in front of that.  (Bins without
    // mass are passed over, also where a rounding would stop at one.)
    constexpr uint32_t EACH = BINS / THREADS;
    const auto mass = [&](uint32_t b) { return ldexp((double)sh.mass[b], -(row.s + steps.down(b))); };
    double own = 0.0;
#pragma unroll
    for (uint32_t e = 0; e < EACH; ++e) own += mass(threadIdx.x * EACH + e);
    const double upto = wave_scan(own);
    if (Row::lane() == 63) sh.sums[Row::wave()] = upto;
    __syncthreads();
    double front = 0.0, all = 0.0;
    for (int k = 0; k < Row::WAVES; ++k) {
        front += k < (int)Row::wave() ? sh.sums[k] : 0.0;
        all += sh.sums[k];
    }
    const double border = (double)top_p * all;
    const uint64_t past = __ballot(own > 0.0 && front + upto >= border);
    if (Row::lane() == 0) sh.words[Row::wave()] = past != 0;
    __syncthreads();
    int w = 0;
    while (w + 1 < Row::WAVES && sh.words[w] == 0) ++w;
    if (w == (int)Row::wave() && past && Row::lane() == (uint32_t)__ffsll((unsigned long long)past) - 1) {      // (top_p < 1: there is one)
        double run = front + upto - own;
        for (uint32_t e = 0; e < EACH; ++e) {
            const uint32_t b = threadIdx.x * EACH + e;
            if (sh.mass[b] == 0) continue;
            sh.pick = b;
            sh.room = border - run;
            sh.own = sh.mass[b];
            run += mass(b);
            if (run >= border) break;
        }
    }
    __syncthreads();
    const uint32_t at_bin = same(sh.pick);
    const double room = fmax(same(sh.room), DBL_MIN);
    const unsigned long long in = same((uint64_t)sh.own);
    __syncthreads();
    // (half a bin to spare on either side: the exact answer is steps.of()'s)
    const float step = 1.0f / steps.per, most = steps.high - ((float)at_bin - 0.5f) * step;
    const float least = steps.high == INFINITY ? INFINITY : at_bin + 1 < BINS ? steps.high - ((float)at_bin + 1.5f) * step : -FLT_MAX;   // (inf - inf: no such bound)
    // (where the border of an earlier cut is in the step too, not all that are equal to it are in)
    if ((old.r != 0 && steps.of(old.t) == at_bin) || !row.collect(least, most, [&](float l) { return steps.of(l) == at_bin; })) {
        const double units = ceil(ldexp(room, row.s + steps.down(at_bin)));
        return radix_cut<Row, T, THREADS, true>(row, min(max((unsigned long long)fmin(units, 0x1p62), 1ull), in), old, steps, at_bin);
    }
    return cut_of_list<Row, true>(row, room);
}

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_sample_block(const SampleArgs a)
{
    using Row = BlockRow<T, THREADS>;
    auto &sh = Row::shared();
    for (uint64_t i = blockIdx.x; i < a.N; i += gridDim.x) {
        Row row{(uint64_t)((const T *)a.S + i * a.ld), a.V, a.mass_bits, Weigh()};
        const RowParams p(a, i);
        Drawn d{0, 0.0f};
        float mine;
        const float top = row.find_top(mine);
        row.weigh = Weigh(top, p.temperature);
        if (top > -INFINITY && p.greedy) {
            d = Drawn{nth_equal(row, top, 1), 1.0f};
        } else if (top > -INFINITY) {
            Cut c{-INFINITY, 0, 0, EVERY};
            bool done = false;
            if (p.top_k > 0 && p.top_k < a.V) {
                // The k-th largest of the lanes' own maxima: at least k scores reach it, and few more do, since the largest
                // scores rarely share a lane: of scores in no order -n ln(1 - k / n) for n lanes, which is 430 of the 512 the
                // list holds at these k.
                if (p.top_k <= (THREADS == 256 ? 208 : THREADS == 512 ? 290 : 352)) {
                    const uint32_t least = max(row.kth_largest(key_of(mine), p.top_k), KEY_LEAST + 1);
                    if (row.collect(value_of(least), INFINITY, [](float) { return true; })) {
                        if (threadIdx.x < 64) d = sh.n <= 256 ? list_draw<Row, 4>(row, p) : list_draw<Row, 8>(row, p);
                        done = true;
                    }
                }
                if (!done) c = radix_cut<Row, T, THREADS, false>(row, p.top_k, c, Steps(), 0);
            }
            if (!done) {
                if (p.top_p < 1.0f) c = mass_cut<Row, T, THREADS>(row, p.top_p, p.reach(a.V), p.octaves(a.V), c);
                const uint32_t last_equal = c.last == UNKNOWN ? nth_equal(row, c.t, c.r) : c.last;
                // scores this far below the maximum miss min_p whatever the rounding
                const double least = p.min_p > 0.0f ? (double)fminf(p.min_p, 1.0f) : 0.0;
                const float from = p.min_p > 0.0f && top < INFINITY ? top + p.temperature * (__logf((float)least) * 1.001f - 0.001f) : -INFINITY;
                d = row_draw<Row, THREADS>(row, c.t, last_equal, least, from, p.u);
            }
        }
        if (threadIdx.x == 0) {
            a.idx[i] = d.at;
            if (a.prob) a.prob[i] = d.prob;
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
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((a.N + WAVE_THREADS / 64 - 1) / (WAVE_THREADS / 64), 16384);     // row after row, the next on its way
    if (vec)
        hipLaunchKernelGGL((k_sample_wave<T, E, true>), dim3(blocks), dim3(WAVE_THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_sample_wave<T, E, false>), dim3(blocks), dim3(WAVE_THREADS), 0, s, a);
    return hipGetLastError();
}

template <class T, int E>
hipError_t run_quad(const SampleArgs &a, hipStream_t s)
{
    constexpr int LOAD = 16 / (int)sizeof(T) < E ? 16 / (int)sizeof(T) : E;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((a.N + QUAD_THREADS / 4 - 1) / (QUAD_THREADS / 4), 1u << 20);
    if ((((uint64_t)(uintptr_t)a.S | a.ld * sizeof(T)) & (LOAD * sizeof(T) - 1)) == 0)
        hipLaunchKernelGGL((k_sample_quad<T, E, true>), dim3(blocks), dim3(QUAD_THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_sample_quad<T, E, false>), dim3(blocks), dim3(QUAD_THREADS), 0, s, a);
    return hipGetLastError();
}

template <class T, int THREADS>
hipError_t run_block(const SampleArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL((k_sample_block<T, THREADS>), dim3((uint32_t)std::min<uint64_t>(a.N, 1u << 20)), dim3(THREADS), 0, s, a);
    return hipGetLastError();
}

template <class T>
hipError_t run_sample(const SampleArgs &a, uint64_t rows, hipStream_t s)
{
    // Four lanes per row up to 64 scores: us for 400000 rows, f32, top_p 0.9 (with a wave per row): 10 scores 28 (216), 32 48
    // (230), 64 94 (237); with parameters per row 64 130 (387)
    if (a.V <= 16) return run_quad<T, 4>(a, s);
    if (a.V <= 32) return run_quad<T, 8>(a, s);
    if (a.V <= 64) return run_quad<T, 16>(a, s);
    // A wave per row, all of it in registers, up to 1024 scores, with room for no more than it takes.  us, f32, top_p 0.9: 65536 x 256
    // 54 (with room for 1024 160), 400000 x 100 187 (with room for 256 247), 32768 x 512 49 (91; by workgroups 314), 32768 x 1000 103 (345)
    if (a.V <= 128) return run_wave<T, 2>(a, s);
    if (a.V <= 256) return run_wave<T, 4>(a, s);
    if (a.V <= 512) return run_wave<T, 8>(a, s);
    if (a.V <= 1024) return run_wave<T, 16>(a, s);
    // A small workgroup wastes less at its barriers, a large one is done sooner where there are fewer rows than CUs, or long ones.  us at
    // 256 / 512 / 1024 lanes, top_p 0.9: 8192 x 4096 151 / 241 / 481; 256 x 16384 31 / 24 / 26, 1024 x 16384 60 / 62 / 99; 256 x 50000
    // 76 / 58 / 54, 512 x 50000 98 / 84 / 102; bf16 256 x 131072 177 / 114 / 98, 512 x 131072 219 / 220 / 188
    if (a.V <= 8192) return run_block<T, 256>(a, s);
    if (a.V <= 32768 || (a.V <= 65536 && rows > 256)) return run_block<T, 512>(a, s);
    return run_block<T, 1024>(a, s);
}

}  // namespace

hipError_t launch_sample(const void *dS, int dtype, uint64_t N, uint32_t V, uint64_t ld, const vqhip_sampling &how, const float *du, uint32_t *didx,
                         float *dprob, uint64_t rows, hipStream_t s)
{
    int log2v = 0;
    while ((1ull << log2v) < V) ++log2v;
    const SampleArgs a{dS, N, ld, V, std::min(51, 62 - log2v), how.temperature, how.top_p, how.min_p, how.top_k, how.dtemperature, how.dtop_p, how.dmin_p,
                       how.dtop_k, du, didx, dprob};
    if (dtype == VQHIP_F32) return run_sample<float>(a, rows, s);
    if (dtype == VQHIP_BF16) return run_sample<__bf16>(a, rows, s);
    return run_sample<_Float16>(a, rows, s);
}

}  // namespace vq
