// Sampling from rows of scores (vqhip_sample_device in include/vqhip.h).  For a row l of V scores (NaN counts as -inf), with
// m = max l and w_j = exp((l_j - m) / T), in the order of falling l, equal ones by index:
//     S1  the first top_k                                                                  Z1 = sum of w over S1
//     S2  those of S1 whose mass before them is below top_p Z1 (the first always)
//     S3  those of S2 with w_j >= min_p                                                    Z  = sum of w over S3
//     idx = the smallest j of S3 with  sum over { i in S3, i <= j } of w_i  >  u Z,        prob = w_idx / Z
// Every filter keeps a beginning of the order, so S3 is { l > t } and the first r (by index) of { l = t }, and w >= min_p: no
// sort is needed, only the threshold t and the count r.  They are found by radix selection on the ordered bits of l: a
// histogram of 8 bits at a time (counts for top_k, masses for top_p), the bin the border falls in, then the next 8 bits of
// that bin alone.
//
// Numbers.  The index is an exact answer, so what decides it is computed in more than 32 bits: w in f64; the masses of the
// histogram as integers (w 2^s, s chosen so that V of them fit 63 bits), because their additions are atomic and integer sums do
// not depend on their order; the sums of the draw in f64 in a fixed order.  Two correct evaluations still part where u Z falls
// within ~1e-15 of a border.
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

constexpr uint32_t KEY_LEAST = 0x007FFFFFu;            // key of -inf: masked scores and NaN

// Floats in the order of their values as unsigned numbers; -0 and NaN are folded into +0 and -inf.
__device__ __forceinline__ uint32_t key_of(float l)
{
    if (!(l == l)) return KEY_LEAST;
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

template <class V>
__device__ __forceinline__ V wave_sum(V v)
{
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
template <class V>
__device__ __forceinline__ V wave_scan(V v)            // inclusive
{
    for (int o = 1; o < 64; o <<= 1) {
        const V y = __shfl_up(v, o);
        if ((int)(threadIdx.x & 63) >= o) v += y;
    }
    return v;
}

// One row, worked on by a workgroup.  Everything below is called by all its lanes.
template <class T, int THREADS>
struct Row {
    static constexpr int WAVES = THREADS / 64;
    struct Shared {
        unsigned long long mass[256];
        uint32_t count[256];
        double sums[WAVES];
        uint32_t words[WAVES];
        uint32_t pick;
        unsigned long long above;
        uint32_t found;
    };
    Shared &sh;
    const T *row;
    uint32_t V;
    int s;
    uint32_t top_key;                   // of the maximum
    double top, inv_t;

    __device__ uint32_t key(uint32_t j) const { return key_of(widen(row[j])); }
    __device__ double weight(uint32_t k) const
    {
        if (k == top_key) return 1.0;
        if (k <= KEY_LEAST) return 0.0;
        return exp(((double)value_of(k) - top) * inv_t);
    }
    __device__ unsigned long long fixed(double w) const { return (unsigned long long)rint(ldexp(w, s)); }

    __device__ uint32_t block_max(uint32_t v)
    {
        for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor(v, o));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh.words[threadIdx.x >> 6] = v;
        __syncthreads();
        for (int k = 0; k < WAVES; ++k) v = max(v, sh.words[k]);
        return v;
    }

    __device__ void find_top()
    {
        uint32_t m = 0;
        for (uint32_t j = threadIdx.x; j < V; j += THREADS) m = max(m, key(j));
        top_key = block_max(m);
        top = (double)value_of(top_key);
    }

    // The order cut where a running total crosses a border: by count (top_k) or by mass (top_p).  Kept so far: keys above t,
    // and `r` of the keys equal to t.  On return they describe the shorter beginning.
    //   by count: the first `border` of the order.   by mass: those whose mass before them is below `border` (fixed point).
    template <bool MASS>
    __device__ void cut(unsigned long long border, uint32_t &t, uint32_t &r)
    {
        uint32_t prefix = 0, fixed_bits = 0;             // the bits of the threshold found so far
        unsigned long long before = 0;                   // count or mass above the prefix
        // the low bits of a widened 16-bit score follow from its sign: 16 of them for bf16, 13 for f16
        constexpr int LAST = sizeof(T) == 4 ? 0 : std::is_same<T, __bf16>::value ? 16 : 8;
        uint32_t ties = 0;
        for (int shift = 24; shift >= LAST; shift -= 8) {
            for (int b = threadIdx.x; b < 256; b += THREADS) {
                sh.count[b] = 0;
                sh.mass[b] = 0;
            }
            __syncthreads();
            for (uint32_t j = threadIdx.x; j < V; j += THREADS) {
                const uint32_t k = key(j);
                if (k < t || k <= KEY_LEAST || (fixed_bits && (k >> (shift + 8)) != prefix)) continue;
                const uint32_t b = (k >> shift) & 255;
                atomicAdd(&sh.count[b], 1u);
                if (MASS && k > t) atomicAdd(&sh.mass[b], fixed(weight(k)));
            }
            __syncthreads();
            if (MASS && threadIdx.x == 0 && r != 0 && t > KEY_LEAST) {
                // of the keys equal to t only r are left
                if (!fixed_bits || (t >> (shift + 8)) == prefix) sh.mass[(t >> shift) & 255] += (unsigned long long)r * fixed(weight(t));
            }
            __syncthreads();
            if (threadIdx.x == 0) {
                // the bin that holds the last element kept: the lowest whose total above it is below the border
                unsigned long long run = before, above = before;
                uint32_t pick = 256;
                for (int b = 255; b >= 0; --b) {
                    if (sh.count[b] == 0) continue;
                    if (run >= border && pick != 256) break;
                    pick = b;
                    above = run;
                    run += MASS ? sh.mass[b] : sh.count[b];
                }
                sh.pick = pick;
                sh.above = above;
                sh.found = pick < 256 ? sh.count[pick] : 0;
            }
            __syncthreads();
            if (sh.pick == 256) return;                  // nothing there at all: nothing to cut
            prefix = (prefix << 8) | sh.pick;
            fixed_bits += 8;
            before = sh.above;
            ties = sh.found;
            __syncthreads();
        }
        uint32_t nt = prefix << LAST;
        if (!(nt >> 31)) nt |= (1u << LAST) - 1u;        // a negative score: the folded bits are ones
        if (nt == t) ties = min(ties, r);                // the border of an earlier cut
        uint32_t nr;
        if (MASS) {
            const unsigned long long w = fixed(weight(nt));
            // the j-th of the equal ones is kept while before + j w < border
            nr = border <= before ? 1 : w == 0 ? ties : (uint32_t)min((unsigned long long)ties, (border - before + w - 1) / w);
            nr = max(nr, 1u);
        } else {
            nr = (uint32_t)min((unsigned long long)ties, border - before);
        }
        t = nt;
        r = nr;
    }

    // Elements of the row are dealt to the waves in consecutive ranges for everything that goes by index.
    __device__ uint32_t range() const { return ((V + THREADS - 1) / THREADS) * 64; }

    // Index of the r-th (r >= 1) element equal to t.
    __device__ uint32_t nth_equal(uint32_t t, uint32_t r)
    {
        const uint32_t w = threadIdx.x >> 6, lane = threadIdx.x & 63, len = range();
        uint32_t n = 0;
        const uint32_t lo = w * len, hi = min(V, lo + len);
        for (uint32_t j = lo + lane; j < hi; j += 64) n += key(j) == t;
        n = wave_sum(n);
        __syncthreads();
        if (lane == 0) sh.words[w] = n;
        __syncthreads();
        uint32_t before = 0;
        for (uint32_t k = 0; k < w; ++k) before += sh.words[k];
        if (before < r && before + n >= r) {              // this wave's range holds it
            for (uint32_t base = lo; base < hi; base += 64) {
                const bool is = base + lane < hi && key(base + lane) == t;
                const uint64_t all = __ballot(is);
                const uint32_t here = __popcll(all);
                if (before + here >= r) {
                    const uint32_t mine = before + __popcll(all & ((1ull << lane) - 1)) + 1;
                    if (is && mine == r) sh.found = base + lane;
                    break;
                }
                before += here;
            }
        }
        __syncthreads();
        return sh.found;
    }
};

template <class T, int THREADS>
__global__ void __launch_bounds__(THREADS) k_sample(const SampleArgs a)
{
    using R = Row<T, THREADS>;
    __shared__ typename R::Shared sh;
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (uint64_t i = blockIdx.x; i < a.N; i += gridDim.x) {
        __syncthreads();
        R row{sh, (const T *)a.S + i * a.ld, a.V, a.mass_bits, 0, 0.0, 0.0};
        const float temperature = a.temperatures ? a.temperatures[i] : a.temperature;
        const float top_p = a.top_ps ? a.top_ps[i] : a.top_p, min_p = a.min_ps ? a.min_ps[i] : a.min_p;
        const uint32_t top_k = a.top_ks ? a.top_ks[i] : a.top_k;
        row.find_top();
        if (row.top_key <= KEY_LEAST) {                                        // nothing to draw from
            if (threadIdx.x == 0) {
                a.idx[i] = 0;
                if (a.prob) a.prob[i] = 0.0f;
            }
            continue;
        }
        if (!(temperature > 0.0f && temperature < INFINITY) || top_k == 1 || top_p <= 0.0f) {        // the first maximum
            const uint32_t first = row.nth_equal(row.top_key, 1);
            if (threadIdx.x == 0) {
                a.idx[i] = first;
                if (a.prob) a.prob[i] = 1.0f;
            }
            continue;
        }
        row.inv_t = 1.0 / (double)temperature;

        uint32_t t = KEY_LEAST, r = 0;                                         // everything above -inf
        if (top_k > 0 && top_k < a.V) row.template cut<false>(top_k, t, r);
        if (top_p < 1.0f) {
            // Z1 in fixed point, then the border
            unsigned long long z = 0;
            for (uint32_t j = threadIdx.x; j < a.V; j += THREADS) {
                const uint32_t k = row.key(j);
                if (k > t) z += row.fixed(row.weight(k));
            }
            z = wave_sum(z);
            __syncthreads();
            if (lane == 0) sh.mass[w] = z;
            __syncthreads();
            z = (unsigned long long)r * row.fixed(row.weight(t));
            for (int k = 0; k < R::WAVES; ++k) z += sh.mass[k];
            __syncthreads();
            row.template cut<true>((unsigned long long)ceil((double)top_p * (double)z), t, r);
        }
        const double least = min_p > 0.0f ? (double)fminf(min_p, 1.0f) : 0.0;
        const uint32_t last_equal = t > KEY_LEAST ? row.nth_equal(t, r) : 0;    // equal to t and kept: up to here
        auto kept = [&](uint32_t j) -> double {
            const uint32_t k = row.key(j);
            if (k < t || (k == t && (j > last_equal || t <= KEY_LEAST))) return 0.0;
            const double x = row.weight(k);
            return x >= least ? x : 0.0;
        };

        // the draw: sums of the waves' ranges, the range the target falls in, then along that range 64 at a time
        const uint32_t len = row.range(), lo = w * len, hi = min(a.V, lo + len);
        double mine = 0.0;
        for (uint32_t j = lo + lane; j < hi; j += 64) mine += kept(j);
        mine = wave_sum(mine);
        __syncthreads();
        if (lane == 0) sh.sums[w] = mine;
        __syncthreads();
        double total = 0.0;
        for (int k = 0; k < R::WAVES; ++k) total += sh.sums[k];
        float u = a.u[i];
        u = u > 0.0f ? fminf(u, 0x1.fffffep-1f) : 0.0f;
        const double target = (double)u * total;
        double before = 0.0;
        int pick = -1;
        for (int k = 0; k < R::WAVES; ++k) {
            if (sh.sums[k] == 0.0) continue;
            if (pick >= 0) before += sh.sums[pick];
            pick = k;
            if (before + sh.sums[k] > target) break;
        }
        if ((int)w == pick) {
            uint32_t at = 0;
            double at_w = 0.0;
            for (uint32_t base = lo; base < hi; base += 64) {
                const double x = base + lane < hi ? kept(base + lane) : 0.0;
                const double c = before + wave_scan(x);
                const uint64_t some = __ballot(x > 0.0), hit = __ballot(x > 0.0 && c > target);
                if (some) {
                    // the last element seen so far stands in should rounding leave the target at the very end
                    const int sl = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll(some);
                    at = base + sl;
                    at_w = __shfl(x, sl);
                    if (hit) break;
                }
                before = __shfl(c, 63);
            }
            if (lane == 0) {
                a.idx[i] = at;
                if (a.prob) a.prob[i] = (float)(at_w / total);
            }
        }
    }
}

template <class T>
hipError_t run_sample(const SampleArgs &a, hipStream_t s)
{
    const uint32_t blocks = (uint32_t)std::min<uint64_t>(a.N, 1u << 20);
    // lanes of a row: a wave for a row it walks in a few steps, more where the row is long enough to keep them busy
    if (a.V <= 1024)
        hipLaunchKernelGGL((k_sample<T, 64>), dim3(blocks), dim3(64), 0, s, a);
    else if (a.V <= 8192)
        hipLaunchKernelGGL((k_sample<T, 256>), dim3(blocks), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((k_sample<T, 1024>), dim3(blocks), dim3(1024), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const void *dS, int dtype, uint64_t N, uint32_t V, uint64_t ld, const vqhip_sampling &how, const float *du, uint32_t *didx,
                         float *dprob, hipStream_t s)
{
    int log2v = 0;
    while ((1ull << log2v) < V) ++log2v;
    const SampleArgs a{dS, N, ld, V, std::min(52, 62 - log2v), how.temperature, how.top_p, how.min_p, how.top_k, how.dtemperature, how.dtop_p, how.dmin_p,
                       how.dtop_k, du, didx, dprob};
    if (dtype == VQHIP_F32) return run_sample<float>(a, s);
    if (dtype == VQHIP_BF16) return run_sample<__bf16>(a, s);
    return run_sample<_Float16>(a, s);
}

}  // namespace vq
