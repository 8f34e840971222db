// Scores of a batch (vqhip_scores_device in include/vqhip.h): S[i][j] = - sum_d (x[i][d] - w[j][d])^2, N x K in f32: the
// squared distances of euclidean_distance (src/helpers.rs:18-20) without the root.
//
// Three kernels.  Few prototypes: k_scores_few, a lane per sample.  Rows of up to DIRECT_D values: k_scores_direct, a tile a
// workgroup, 8 x 8 scores a lane, so that 16 values read from LDS feed 128 vector instructions.  Both are the formula as it stands
// on the vector units.  Longer rows: k_scores_mfma, where the two vector instructions per (sample, prototype, value) of the
// direct form would bound it, the products run on the bf16 matrix cores, six of exact three-piece splits (bf16x6,
// mfma_device.h), in the expanded form
//     |x - w|^2 = |x - c|^2 + |w - c|^2 - 2 (x - c).(w - c)
// with c the mean prototype, so that an offset all values share (pixels) does not cost digits.  Its rounding errors are those
// of the two norms, so the pairs whose distance is small beside them (below CLOSE of their sum: a sample and the few
// prototypes next to it) are measured again in the direct form, by 4 lanes a pair, or a square of pairs where they are many.  Which
// form a pair takes and the order of its sums depend on the pair alone, not on the tile or the pairs beside it: a score has the same
// bits whatever other rows a call has.  500000 x 128 against 256, us: no pair close 261, a close prototype for each sample 318, half of
// all pairs close 1250.
//
// What bounds them: the matrix cores where rows are long (20011 x 784 against 1000 179 us, 1050 TFLOP/s over the six products; a
// library's bf16 product reaches 1195 here), staging, products and the stores of a tile in turn where they are short (500000 x 128 against
// 256 245 us, 3.1 TB/s, the matrix pipe busy 40 %), the scores' stores where the prototypes are few (500000 x 4 against 256 92 us, 5.6 TB/s).
#include <algorithm>
#include <type_traits>

#include "mfma_device.h"
#include "vq_common.h"

namespace vq {

namespace {

constexpr int SC_THREADS = 256, SC_K = 16;
// Workgroups of a launch: a grid holds fewer than 2^32 lanes, larger problems are several launches (or steps of a loop)
constexpr uint32_t GRID = 1u << 22;

// Four floats in one access of 16 bytes, which has to begin at a multiple of 4 only
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

struct ScoreArgs {
    const float *X, *W, *C;           // C: the mean prototype, D values (any would do for the result; near the mean they keep its digits)
    float *S;
    uint64_t N, ld;
    uint32_t K, D;
    const uint32_t *img;              // k_scores_image: the prototypes' pieces; behind them their norms and their mean
    const float *norms;
    uint32_t blocks;                  // of 64 prototypes
    uint32_t colTiles;
};

// Reduction values d0 .. d0 + 3 of one row, zero behind D or behind the last row (a pair of zeros adds nothing).
__device__ __forceinline__ float4 load4(const float *base, uint64_t row, bool on, uint32_t D, uint32_t d0)
{
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!on || d0 >= D) return v;
    const float *p = base + row * D + d0;
    if (d0 + 4 <= D) {
        const float4u q = *(const float4u *)p;
        return make_float4(q.x, q.y, q.z, q.w);
    }
    v.x = p[0];
    if (d0 + 1 < D) v.y = p[1];
    if (d0 + 2 < D) v.z = p[2];
    return v;
}
__device__ __forceinline__ void store4(float *to, float x, float y, float z, float w)
{
    const float4u v = {x, y, z, w};
    *(float4u *)to = v;
}

// TX lanes side by side, 8 prototypes each: 128, 64 or 32 prototypes a tile, 8 samples each of the 256 / TX lanes above another.
template <int TX>
__global__ void __launch_bounds__(SC_THREADS, 2) k_scores_direct(const ScoreArgs a)
{
    constexpr int SC_M = SC_THREADS / TX * 8, SC_N = TX * 8, XPARTS = SC_M / 64, WPARTS = (SC_N + 63) / 64;
    // (a row of the tile per reduction value, moved 4 banks on from the one before)
    __shared__ __attribute__((aligned(16))) float lx[2][SC_K][SC_M + 4], lw[2][SC_K][SC_N + 4];
    const uint64_t tile = blockIdx.x;
    const uint64_t row0 = tile / a.colTiles * SC_M;
    const uint32_t col0 = (uint32_t)(tile % a.colTiles) * SC_N;
    const int t = threadIdx.x;
    // staging: lane t moves values 4 (t & 3) .. + 3 of rows (t >> 2), (t >> 2) + 64, ... of both operands
    const int sr = t >> 2, sd = (t & 3) * 4;
    const int ty = t / TX, tx = t % TX;
    float acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;

    float4 px[XPARTS], pw[WPARTS];
    auto fetch = [&](uint32_t d) {
#pragma unroll
        for (int h = 0; h < XPARTS; ++h) {
            const uint64_t r = row0 + sr + 64 * h;
            px[h] = load4(a.X, r, r < a.N, a.D, d + sd);
        }
#pragma unroll
        for (int h = 0; h < WPARTS; ++h) {
            const uint32_t c = col0 + sr + 64 * h;
            pw[h] = load4(a.W, c, c < a.K, a.D, d + sd);
        }
    };
    auto put = [&](float *to, int ld, const float4 &v) {
        to[0] = v.x;
        to[ld] = v.y;
        to[2 * ld] = v.z;
        to[3 * ld] = v.w;
    };
    auto stage = [&](int b) {
#pragma unroll
        for (int h = 0; h < XPARTS; ++h) put(&lx[b][sd][sr + 64 * h], SC_M + 4, px[h]);
#pragma unroll
        for (int h = 0; h < WPARTS; ++h)
            if (SC_N >= 64 || sr < SC_N) put(&lw[b][sd][sr + 64 * h], SC_N + 4, pw[h]);
    };
    fetch(0);
    stage(0);
    __syncthreads();
    int b = 0;
    for (uint32_t d = 0; d < a.D; d += SC_K, b ^= 1) {
        const bool more = d + SC_K < a.D;
        if (more) fetch(d + SC_K);
        const int values = min(SC_K, (int)(a.D - d + 3) & ~3);
#pragma unroll 4
        for (int k = 0; k < values; ++k) {
            float x[8], w[8];
            *(float4 *)&x[0] = *(const float4 *)&lx[b][k][ty * 4];
            *(float4 *)&x[4] = *(const float4 *)&lx[b][k][SC_M / 2 + ty * 4];
            *(float4 *)&w[0] = *(const float4 *)&lw[b][k][tx * 4];
            *(float4 *)&w[4] = *(const float4 *)&lw[b][k][SC_N / 2 + tx * 4];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float e = x[i] - w[j];
                    acc[i][j] = fmaf(e, e, acc[i][j]);
                }
        }
        if (more) stage(b ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint64_t r = row0 + (i >> 2) * (SC_M / 2) + ty * 4 + (i & 3);
        if (r >= a.N) continue;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const uint32_t c = col0 + g * (SC_N / 2) + tx * 4;
            float *out = a.S + r * a.ld + c;
            if (c + 4 <= a.K) {
                store4(out, -acc[i][g * 4], -acc[i][g * 4 + 1], -acc[i][g * 4 + 2], -acc[i][g * 4 + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < a.K) out[e] = -acc[i][g * 4 + e];
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- few prototypes
// A lane per sample, its values in registers; the prototypes' values are the same for all lanes and come through the scalar
// cache, so that nothing is staged and nobody waits at a barrier.  Tiles of 128 prototypes would be mostly empty here.
template <int DP>
__global__ void __launch_bounds__(SC_THREADS) k_scores_few(const ScoreArgs a)
{
    using Uniform = const __attribute__((address_space(4))) float;
    const uint64_t r = (uint64_t)blockIdx.x * SC_THREADS + threadIdx.x;
    if (r >= a.N) return;
    const float *row = a.X + r * a.D;
    float x[DP];
#pragma unroll
    for (int d = 0; d < DP; d += 4) {
        if ((uint32_t)d + 4 <= a.D) {
            const float4u v = *(const float4u *)(row + d);
            x[d] = v.x;
            x[d + 1] = v.y;
            x[d + 2] = v.z;
            x[d + 3] = v.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[d + e] = (uint32_t)(d + e) < a.D ? row[d + e] : 0.0f;
        }
    }
    float *out = a.S + r * a.ld;
    for (uint32_t j = 0; j < a.K; j += 4) {
        // (behind the last prototype: that one again, not stored)
        Uniform *w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) w[q] = (Uniform *)a.W + (size_t)min(j + q, a.K - 1) * a.D;
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int d = 0; d < DP; d += 4) {
            if ((uint32_t)d >= a.D) break;
            if ((uint32_t)d + 4 <= a.D) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float f = x[d + e] - w[q][d + e];
                        s[q] = fmaf(f, f, s[q]);
                    }
            } else {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if ((uint32_t)(d + e) < a.D)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float f = x[d + e] - w[q][d + e];
                            s[q] = fmaf(f, f, s[q]);
                        }
            }
        }
        if (j + 4 <= a.K) {
            store4(out + j, -s[0], -s[1], -s[2], -s[3]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (j + q < a.K) out[j + q] = -s[q];
        }
    }
}

// ---------------------------------------------------------------------------------------------- matrix cores
// Which kernel.  us for 500000 samples (a lane per sample / direct tiles of 32, 64 or 128 prototypes / matrix cores):
//     16 values: 3 prototypes 7.2 / 24 / 28, 16 prototypes 23 / 26 / 34, 32 prototypes 51 / 28 / 35, 64 prototypes 119 / 36 / 35,
//                256 prototypes 438 / 137 / 120
//      8 values: 16 prototypes 16 / 19 / 35, 64 prototypes 122 / 30 / 36, 256 prototypes 361 / 100 / 124
//     32 values: 16 prototypes 36 / 44 / 35, 256 prototypes 524 / 224 / 135
// The lanes of k_scores_few store K apart, which is what it costs: K^2 D up to 4096.  The direct form is kept to 16 values, where the
// matrix cores are ahead against many prototypes: it has the smaller error.
constexpr uint32_t FEW_D = 32, FEW_K = 32;      // k_scores_few
constexpr uint32_t DIRECT_D = 16;               // k_scores_direct
// Of |x - c|^2 + |w - c|^2; distances below it are measured directly.  The products' error is a few 2^-24 of the norms, so at 1/16
// a distance is within a few 1e-6 of itself (the bar of this library is 1e-5); at 1/8 the samples of a codebook would take
// their own prototype's way through the direct form too, 55 us more on 500k x 128 against 256.
constexpr float CLOSE = 0.0625f;
constexpr int MF_K = 16;
// Norms above this become NaN, and with them every score made from them, so that such pairs are measured directly: the sum of two norms up
// to here and the score itself (four times a norm at most) stay finite.  What is beyond f32 is decided by the direct form alone.
constexpr float NORM_MOST = 0x1p125f;
__device__ __forceinline__ float finite_norm(float x) { return x <= NORM_MOST ? x : NAN; }

// The sum over 4 consecutive lanes, in all of them
__device__ __forceinline__ float quad_sum(float v)
{
    auto other = [](float x, auto ctrl) { return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true)); };
    v += other(v, std::integral_constant<int, 0xB1>());              // lane ^ 1
    return v + other(v, std::integral_constant<int, 0x4E>());        // lane ^ 2
}
// Four more squares of a pair that is measured directly.  What such a pair's score is does not depend on the pairs beside it: lane l of
// 4 takes the values 4 l .. 4 l + 3 of every 16 in their order, quad_sum joins the 4 sums.
__device__ __forceinline__ void add_squares(float &s, const float4 &x, const float4 &w)
{
    const float e0 = x.x - w.x, e1 = x.y - w.y, e2 = x.z - w.z, e3 = x.w - w.w;
    s = fmaf(e0, e0, fmaf(e1, e1, fmaf(e2, e2, fmaf(e3, e3, s))));
}

// The prototypes as the matrix cores read them, made once per model: per step of 16 reduction values and block of 64 prototypes
// three pieces of 64 rows of 16 bf16 (6 KiB, what a workgroup copies to LDS as it is), zero behind the last prototype and
// value.  A row of a piece is two 16-byte halves, swapped in every other group of 8 rows, so that 16 lanes reading the same half
// of 16 rows touch 16 different 16-byte slots of the 64 banks.
constexpr uint32_t IMG_BLOCK = 3 * 64 * 8;             // dwords
constexpr uint32_t IMG_PAD = 256;                      // prototypes the image is filled up to a multiple of: the widest tile

__device__ __forceinline__ int piece_slot(int row, int quad) { return (((quad >> 1) ^ (row >> 3)) & 1) * 4 + (quad & 1) * 2; }
inline uint32_t image_blocks(uint32_t K) { return (uint32_t)(((uint64_t)K + IMG_PAD - 1) / IMG_PAD * (IMG_PAD / 64)); }

// The mean prototype, 16 values a workgroup, rows dealt to its 64 groups of 16 lanes; 0 where it is not finite
__global__ void __launch_bounds__(1024) k_scores_mean(const float *W, uint32_t K, uint32_t D, float *C)
{
    __shared__ double part[64][16];
    const uint32_t v = threadIdx.x & 15, g = threadIdx.x >> 4;
    for (uint64_t base = (uint64_t)blockIdx.x * 16; base < D; base += (uint64_t)gridDim.x * 16) {
        const uint64_t d = base + v;
        double s = 0.0;
        if (d < D)
#pragma unroll 8
            for (uint64_t k = g; k < K; k += 64) s += (double)W[k * D + d];
        part[g][v] = s;
        __syncthreads();
        if (g == 0 && d < D) {
            for (int q = 1; q < 64; ++q) s += part[q][v];
            const float mean = (float)(s / K);
            C[d] = fabsf(mean) < INFINITY ? mean : 0.0f;
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) k_scores_image(const float *W, const float *C, uint32_t K, uint32_t D, uint32_t blocks, uint32_t steps, uint32_t *img)
{
    const int row = threadIdx.x >> 2, quad = threadIdx.x & 3;
    for (uint64_t at = blockIdx.x; at < (uint64_t)blocks * steps; at += gridDim.x) {         // at: step, then block
        const uint64_t k = at % blocks * 64 + row;
        const uint32_t d = (uint32_t)(at / blocks) * MF_K + quad * 4;
        const float4 w = load4(W, k, k < K, D, d), c = load4(C, 0, k < K, D, d);
        uint32_t p[3], q[3];
        split3(w.x - c.x, w.y - c.y, p[0], p[1], p[2]);
        split3(w.z - c.z, w.w - c.w, q[0], q[1], q[2]);
        uint32_t *to = img + at * IMG_BLOCK + row * 8 + piece_slot(row, quad);
#pragma unroll
        for (int i = 0; i < 3; ++i) *(uint2 *)(to + i * 64 * 8) = make_uint2(p[i], q[i]);
    }
}

// |w - c|^2, a wave per prototype; 0 behind the last
__global__ void __launch_bounds__(64) k_scores_norms(const float *W, const float *C, uint32_t K, uint32_t D, uint64_t rows, float *norms)
{
    for (uint64_t k = blockIdx.x; k < rows; k += gridDim.x) {
        float s = 0.0f;
        if (k < K)
            for (uint32_t d = threadIdx.x; d < D; d += 64) {
                const float e = W[k * D + d] - C[d];
                s = fmaf(e, e, s);
            }
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (threadIdx.x == 0) norms[k] = s;
    }
}

// A workgroup of WR x WC waves, a wave 32 RW x 32 CW scores in RW x CW accumulators of v_mfma_f32_32x32x16_bf16.  A operand: lane l
// holds sample l & 31, B operand: prototype l & 31; lanes 0-31 the reduction values 0 .. 7 of a step, lanes 32-63 8 .. 15.
// Result: lane l holds prototype l & 31 and samples 8 g + 4 (l >> 5) + e.  The samples are centred and split on their way to LDS;
// both operands are double buffered there.
constexpr uint32_t CLOSE_LIST = 512;                   // close pairs a wave measures one by one at most; more: squares of its tile

template <int RW, int CW, int WR, int WC, int PER_SIMD>
__global__ void __launch_bounds__(WR * WC * 64, PER_SIMD) k_scores_mfma(const ScoreArgs a)
{
    constexpr int THREADS = WR * WC * 64, TM = 32 * RW * WR, TN = 32 * CW * WC, MT = 32 * RW, NT = 32 * CW;
    constexpr int XROWS = THREADS / 4, XPARTS = TM / XROWS;                         // staging: 4 lanes a sample
    constexpr int COPY = TN / 64 * (int)IMG_BLOCK / 4, COPIES = (COPY + THREADS - 1) / THREADS;     // 16-byte pieces of the image
    static_assert(TM % XROWS == 0 && TM % 64 == 0 && TN % 64 == 0, "whole blocks of 64 rows");
    constexpr int XSTAGE = TM * 3 * 8, WSTAGE = TN * 3 * 8;
    __shared__ __attribute__((aligned(16))) uint32_t lx[2][XSTAGE], lw[2][WSTAGE];
    __shared__ __attribute__((aligned(16))) float nx[TM], nw[TN];
    __shared__ uint16_t lists[WR * WC][CLOSE_LIST];
    // workgroups are dealt to the 8 XCDs in turn: each takes a consecutive share of the tiles, so that the column tiles of the same
    // samples meet in one L2
    const uint32_t share = (gridDim.x + 7) / 8, tile = blockIdx.x % 8 * share + blockIdx.x / 8;
    const uint64_t row0 = (uint64_t)(tile / a.colTiles) * TM;
    const uint32_t col0 = tile % a.colTiles * TN;
    if (row0 >= a.N) return;
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5, l31 = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6), wr = wave / WC, wc = wave % WC;
    const int sr = t >> 2, sd = (t & 3) * 4;          // staging: values sd .. + 3 of rows sr, sr + XROWS, ...
    const int slot = piece_slot(sr, t & 3);           // ... and where they go, in dwords of the row's piece
    const int swap = ((half ^ (l31 >> 3)) & 1) * 4;   // which half of a row's piece this lane reads
    const u32x4 *img = (const u32x4 *)(a.img + (size_t)(col0 / 64) * IMG_BLOCK);
    const size_t imgStep = (size_t)a.blocks * (IMG_BLOCK / 4);

    const uint32_t steps = (a.D + MF_K - 1) / MF_K;

    // Samples are requested PREFETCH steps ahead of their use (HBM), the image one (L2), and the image first: loads are waited for
    // in the order of their issue.  None of them is conditional (a count of loads on their way that depends on a branch is
    // waited for as a whole): what lies behind the last sample or value is read inside instead, and dropped.
    constexpr int PREFETCH = 2;
    float4 px[PREFETCH][XPARTS], pc;
    u32x4 pw[COPIES];
    float sx[XPARTS];
    const float *xrow[XPARTS];
#pragma unroll
    for (int i = 0; i < XPARTS; ++i) {
        sx[i] = 0.0f;
        xrow[i] = a.X + min(row0 + sr + XROWS * i, a.N - 1) * a.D;
    }
    auto values = [&](const float *row, uint32_t step) -> float4 {
        const uint32_t d = step * MF_K + sd;
        const float4u v = *(const float4u *)(row + min(d, a.D - 4));               // (the last four where there are fewer left)
        return make_float4(v.x, v.y, v.z, v.w);
    };
    auto samples = [&](int u, uint32_t step) {
#pragma unroll
        for (int i = 0; i < XPARTS; ++i) px[u][i] = values(xrow[i], step);
    };
    auto fetch = [&](uint32_t step) {
        pc = values(a.C, step);
#pragma unroll
        for (int i = 0; i < COPIES; ++i) pw[i] = img[COPY % THREADS == 0 ? t + i * THREADS : min(t + i * THREADS, COPY - 1)];
        if (step + 1 < steps) img += imgStep;
    };
    auto stage = [&](int b, int u, uint32_t step, auto whole) {
#pragma unroll
        for (int i = 0; i < COPIES; ++i)
            if (COPY % THREADS == 0 || t + i * THREADS < COPY) *(u32x4 *)&lw[b][4 * (t + i * THREADS)] = pw[i];
#pragma unroll
        for (int i = 0; i < XPARTS; ++i) {
            const float4 v = px[u][i];
            float4 x = make_float4(v.x - pc.x, v.y - pc.y, v.z - pc.z, v.w - pc.w);
            if (!decltype(whole)::value && (step + 1) * MF_K > a.D) {
                const uint32_t d = step * MF_K + sd;
                const uint32_t over = d + 4 > a.D ? d + 4 - a.D : 0;               // values behind the last: what is here is that far ahead
                x = over == 0 ? x : over == 1 ? make_float4(x.y, x.z, x.w, 0.0f) : over == 2 ? make_float4(x.z, x.w, 0.0f, 0.0f) : over == 3 ? make_float4(x.w, 0.0f, 0.0f, 0.0f) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            sx[i] = fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(x.z, x.z, fmaf(x.w, x.w, sx[i]))));
            uint32_t p[3], q[3];
            split3(x.x, x.y, p[0], p[1], p[2]);
            split3(x.z, x.w, q[0], q[1], q[2]);
            const int row = sr + XROWS * i;
#pragma unroll
            for (int c = 0; c < 3; ++c) *(uint2 *)&lx[b][((row / 64 * 3 + c) * 64 + row % 64) * 8 + slot] = make_uint2(p[c], q[c]);
        }
    };
    // (both operands lie as blocks of 64 rows, three pieces each)
    auto piece = [&](const uint32_t *l, int row, int c) { return *(const u32x4 *)&l[((row / 64 * 3 + c) * 64 + row % 64) * 8 + swap]; };
    f32x16 acc[RW][CW];
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
        for (int j = 0; j < CW; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

    fetch(0);
#pragma unroll
    for (int u = 0; u < PREFETCH; ++u) samples(u, u);
    stage(0, 0, 0, std::false_type());
    fetch(min(1u, steps - 1));
    samples(0, PREFETCH);
    __syncthreads();
    auto multiply = [&](int b) {
        u32x4 fx[RW][3];
#pragma unroll
        for (int i = 0; i < RW; ++i)
#pragma unroll
            for (int c = 0; c < 3; ++c) fx[i][c] = piece(lx[b], wr * MT + i * 32 + l31, c);
#pragma unroll
        for (int j = 0; j < CW; ++j) {
            u32x4 fw[3];
#pragma unroll
            for (int c = 0; c < 3; ++c) fw[c] = piece(lw[b], wc * NT + j * 32 + l31, c);
            // the six products that matter, the smallest first
            constexpr int PX[6] = {2, 0, 1, 1, 0, 0}, PW[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
            for (int p = 0; p < 6; ++p)
#pragma unroll
                for (int i = 0; i < RW; ++i) acc[i][j] = mma_bf(fx[i][PX[p]], fw[PW[p]], acc[i][j]);
        }
    };
    // Steps whose successor is whole, without a branch, so that the next step's staging is scheduled among the products: 20011
    // x 784 against 1000 192 us, with the branch 205
    const uint32_t whole = a.D / MF_K;
    uint32_t k0 = 0;
    for (; k0 + PREFETCH < whole; k0 += PREFETCH) {
#pragma unroll
        for (int u = 0; u < PREFETCH; ++u) {
            const int next = (u + 1) % PREFETCH;
            multiply(u & 1);
            stage((u & 1) ^ 1, next, k0 + u + 1, std::true_type());
            fetch(k0 + u + 2);
            samples(next, k0 + u + 1 + PREFETCH);
            __syncthreads();
        }
    }
    for (; k0 < steps; k0 += PREFETCH) {
#pragma unroll
        for (int u = 0; u < PREFETCH; ++u) {
            const uint32_t k = k0 + u;
            if (k >= steps) break;
            const int next = (u + 1) % PREFETCH;
            multiply(u & 1);
            if (k + 1 < steps) {
                stage((u & 1) ^ 1, next, k + 1, std::false_type());
                fetch(k + 2);
                samples(next, k + 1 + PREFETCH);
            }
            __syncthreads();
        }
    }
    // the samples' norms: 4 lanes hold the parts of a row
#pragma unroll
    for (int i = 0; i < XPARTS; ++i) {
        float x = sx[i];
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) x += __shfl_xor(x, o);
        if ((t & 3) == 0) nx[sr + XROWS * i] = finite_norm(x);
    }
    for (int q = t; q < TN; q += THREADS) nw[q] = finite_norm(a.norms[col0 + q]);
    __syncthreads();

    // scores, and a bit for each of this wave's close pairs, 32 prototypes a word, where the samples were staged
    static_assert(TM * TN / 32 <= 2 * XSTAGE, "a bit for every pair of the tile");
    uint32_t *close = &lx[0][0] + wave * MT * CW;
    for (int q = lane; q < MT * CW; q += 64) close[q] = 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint64_t wrow = row0 + wr * MT;
    const uint32_t wcol = col0 + wc * NT;
    auto finish = [&](auto bounded) {
        float *const out = a.S + wrow * a.ld + wcol;
        const size_t at = 4 * half * a.ld + l31;
#pragma unroll
        for (int j = 0; j < CW; ++j) {
            const float w2 = nw[wc * NT + j * 32 + l31];
#pragma unroll
            for (int i = 0; i < RW; ++i)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 x2 = *(const float4 *)&nx[wr * MT + i * 32 + 8 * g + 4 * half];
                    const float fx2[4] = {x2.x, x2.y, x2.z, x2.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t lr = i * 32 + 8 * g + 4 * half + e, lc = j * 32 + l31;
                        const float both = fx2[e] + w2, s = fmaf(2.0f, acc[i][j][4 * g + e], -both);
                        float *const to = out + (size_t)(i * 32 + 8 * g + e) * a.ld + j * 32;
                        const bool on = !decltype(bounded)::value || (wrow + lr < a.N && wcol + lc < a.K);
                        const bool far = s <= -CLOSE * both;                          // (not so where a norm is NaN)
                        const uint64_t m = __ballot(!far);
                        if (m == 0) {
                            if (on) to[at] = s;
                        } else {
                            if (on && far) to[at] = s;
                            const uint64_t c = __ballot(on && !far);
                            if (l31 == 0) close[lr * CW + j] = (uint32_t)(half ? c >> 32 : c);
                        }
                    }
                }
        }
    };
    if (row0 + TM <= a.N && col0 + TN <= a.K)
        finish(std::false_type());
    else
        finish(std::true_type());
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    constexpr int WORDS = (MT * CW + 63) / 64;             // a lane's
    uint32_t word[WORDS], own = 0;
#pragma unroll
    for (int k = 0; k < WORDS; ++k) {
        word[k] = lane + 64 * k < MT * CW ? close[lane + 64 * k] : 0;
        own += __popc(word[k]);
    }
    if (__ballot(own != 0) == 0) return;
    uint32_t upto = own;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t v = __shfl_up(upto, o);
        if (lane >= o) upto += v;
    }
    const uint32_t n = (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    if (n <= MT * NT / 32) {
        // a list of them: sample << 8 | prototype, inside this wave's tile
        static_assert(MT * NT / 32 <= (int)CLOSE_LIST, "the pairs measured one by one are all in the list");
        uint16_t *list = lists[wave];
        uint32_t to = upto - own;
#pragma unroll
        for (int k = 0; k < WORDS; ++k)
            for (uint32_t left = word[k]; left; left &= left - 1)
                list[to++] = (uint16_t)((lane + 64 * k) / CW << 8 | ((lane + 64 * k) % CW * 32 + __ffs(left) - 1));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        // 4 lanes a pair
        const uint32_t gl = lane & 3;
        for (uint32_t p = lane >> 2; p < n; p += 16) {
            const uint32_t q = list[p];
            const float *x = a.X + (wrow + (q >> 8)) * a.D, *w = a.W + (uint64_t)(wcol + (q & 255)) * a.D;
            float s = 0.0f;
            for (uint32_t d = gl * 4; d < a.D; d += 64) {
                // (64 values on their way at once; what lies behind the row is 0 - 0)
                float4 u[4], v[4];
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    u[h] = load4(x, 0, true, a.D, d + 16 * h);
                    v[h] = load4(w, 0, true, a.D, d + 16 * h);
                }
#pragma unroll
                for (int h = 0; h < 4; ++h) add_squares(s, u[h], v[h]);
            }
            s = quad_sum(s);
            if (gl == 0) a.S[(wrow + (q >> 8)) * a.ld + wcol + (q & 255)] = -s;
        }
        return;
    }
    // many: Q x Q pairs per 4 lanes, squares of the tile without a close one left out; a lane's sums are those of a pair measured alone
    constexpr int Q = 4 * RW, ACROSS = NT / Q;
    static_assert(32 % Q == 0, "a square's bits lie in one word a row");
    const uint32_t gl = lane & 3;
#pragma unroll 1
    for (uint32_t b = lane >> 2; b < MT / Q * ACROSS; b += 16) {
        const uint32_t r0 = b / ACROSS * Q, c0 = b % ACROSS * Q;
        uint64_t pairs = 0;                                // bit i Q + j: sample r0 + i, prototype c0 + j
#pragma unroll
        for (int i = 0; i < Q; ++i) pairs |= (uint64_t)(close[(r0 + i) * CW + c0 / 32] >> (c0 % 32) & ((1u << Q) - 1)) << (i * Q);
        if (pairs == 0) continue;
        float sum[Q][Q];
#pragma unroll
        for (int i = 0; i < Q; ++i)
#pragma unroll
            for (int j = 0; j < Q; ++j) sum[i][j] = 0.0f;
        for (uint32_t d = gl * 4; d < a.D; d += 16) {
            float4 x[Q], w[Q];
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                x[i] = load4(a.X, wrow + r0 + i, wrow + r0 + i < a.N, a.D, d);
                w[i] = load4(a.W, wcol + c0 + i, wcol + c0 + i < a.K, a.D, d);
            }
#pragma unroll
            for (int i = 0; i < Q; ++i)
#pragma unroll
                for (int j = 0; j < Q; ++j) add_squares(sum[i][j], x[i], w[j]);
        }
        // lane l of the 4 stores the pairs l, l + 4, ...
#pragma unroll
        for (int p = 0; p < Q * Q; p += 4) {
            float mine = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float s = quad_sum(sum[(p + e) / Q][(p + e) % Q]);
                mine = gl == (uint32_t)e ? s : mine;
            }
            const uint32_t j = p % Q + gl;
            if (pairs >> (p + gl) & 1) a.S[(wrow + r0 + p / Q) * a.ld + wcol + c0 + j] = -mine;
        }
    }
}

// launch(part, workgroups) for parts of the scores that a launch can hold, of whole tiles of TM samples and TN prototypes; colTiles is set
template <uint32_t TM, uint32_t TN, class Launch>
hipError_t in_parts(const ScoreArgs &all, Launch &&launch)
{
    const uint64_t wide = (uint64_t)GRID * TN;
    for (uint64_t col = 0; col < all.K; col += wide) {
        ScoreArgs a = all;
        a.K = (uint32_t)std::min<uint64_t>(all.K - col, wide);
        a.colTiles = (uint32_t)(((uint64_t)a.K + TN - 1) / TN);
        a.W = all.W + col * all.D;
        a.img = all.img + col / 64 * IMG_BLOCK;
        a.norms = all.norms + col;
        const uint64_t most = (uint64_t)(GRID / a.colTiles) * TM;
        for (uint64_t row = 0; row < all.N; row += most) {
            a.X = all.X + row * all.D;
            a.S = all.S + row * all.ld + col;
            a.N = std::min(all.N - row, most);
            const hipError_t e = launch(a, (uint32_t)((a.N + TM - 1) / TM * a.colTiles));
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}

template <int TX>
hipError_t run_direct(const ScoreArgs &all, hipStream_t s)
{
    return in_parts<SC_THREADS / TX * 8, TX * 8>(all, [&](const ScoreArgs &a, uint32_t tiles) {
        hipLaunchKernelGGL(k_scores_direct<TX>, dim3(tiles), dim3(SC_THREADS), 0, s, a);
        return hipGetLastError();
    });
}

template <int RW, int CW, int WR, int WC, int PER_SIMD>
hipError_t run_mfma(const ScoreArgs &all, hipStream_t s)
{
    constexpr uint32_t TM = 32 * RW * WR, TN = 32 * CW * WC;
    static_assert(IMG_PAD % TN == 0, "the image covers every tile");
    return in_parts<TM, TN>(all, [&](const ScoreArgs &a, uint32_t tiles) {
        hipLaunchKernelGGL((k_scores_mfma<RW, CW, WR, WC, PER_SIMD>), dim3((tiles + 7) / 8 * 8), dim3(WR * WC * 64), 0, s, a);
        return hipGetLastError();
    });
}

bool is_few(uint32_t K, uint32_t D) { return K <= FEW_K && D <= FEW_D && K * K * D <= 4096; }

}  // namespace

// The layout's parts: pieces, norms, mean
struct ScoresImage {
    uint32_t blocks, steps;
    size_t norms, mean, bytes;
    ScoresImage(uint32_t K, uint32_t D) : blocks(image_blocks(K)), steps((uint32_t)(((uint64_t)D + MF_K - 1) / MF_K))
    {
        norms = (size_t)steps * blocks * IMG_BLOCK * 4;
        mean = norms + (size_t)blocks * 64 * 4;
        bytes = mean + (size_t)D * 4;
    }
};

size_t scores_image_bytes(uint32_t K, uint32_t D) { return D <= DIRECT_D || is_few(K, D) ? 0 : ScoresImage(K, D).bytes; }

hipError_t launch_scores_image(const float *dW, uint32_t K, uint32_t D, void *dImg, hipStream_t s)
{
    const ScoresImage image(K, D);
    float *const mean = (float *)((char *)dImg + image.mean);
    hipLaunchKernelGGL(k_scores_mean, dim3(std::min(D / 16 + 1, GRID / 4)), dim3(1024), 0, s, dW, K, D, mean);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_scores_image, dim3((uint32_t)std::min<uint64_t>((uint64_t)image.blocks * image.steps, GRID)), dim3(256), 0, s, dW, mean, K, D, image.blocks, image.steps, (uint32_t *)dImg);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    const uint64_t rows = (uint64_t)image.blocks * 64;
    hipLaunchKernelGGL(k_scores_norms, dim3((uint32_t)std::min<uint64_t>(rows, GRID)), dim3(64), 0, s, dW, mean, K, D, rows, (float *)((char *)dImg + image.norms));
    return hipGetLastError();
}

hipError_t launch_scores(const float *dX, uint64_t N, uint32_t D, const float *dW, const void *dImg, uint32_t K, float *dS, uint64_t ld, hipStream_t s)
{
    const ScoresImage image(K, D);
    ScoreArgs a{dX, dW, (const float *)((const char *)dImg + image.mean), dS, N, ld, K, D, (const uint32_t *)dImg, (const float *)((const char *)dImg + image.norms), image.blocks, 0};
    if (is_few(K, D)) {
        const uint64_t most = (uint64_t)GRID * SC_THREADS;
        for (uint64_t off = 0; off < N; off += most) {
            a.X = dX + off * D;
            a.S = dS + off * ld;
            a.N = std::min(N - off, most);
            const dim3 blocks((uint32_t)((a.N + SC_THREADS - 1) / SC_THREADS));
            if (D <= 4)
                hipLaunchKernelGGL(k_scores_few<4>, blocks, dim3(SC_THREADS), 0, s, a);
            else if (D <= 16)
                hipLaunchKernelGGL(k_scores_few<16>, blocks, dim3(SC_THREADS), 0, s, a);
            else
                hipLaunchKernelGGL(k_scores_few<32>, blocks, dim3(SC_THREADS), 0, s, a);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    }
    if (D > DIRECT_D) {
        // Larger tiles read both operands less often, smaller ones leave fewer of the 512 places (two workgroups a CU) empty in the last
        // round.  us, 128 x 256 / 128 x 128 / 64 x 64 tiles: 500k x 128 against 256 (3907 wide tiles) 256 / 274 / 342, 500k x 64 187 / 191 /
        // 242, 20011 x 784 against 1000 (628) 194 / 176 / 237
        // Where prototypes would leave a large part of a wide tile empty, a narrower one is taken: what a tile of each kind costs per
        // column is 1 / 1.1 / 1.5.
        const uint64_t rows = (N + 127) / 128, c64 = ((uint64_t)K + 63) / 64, c128 = (c64 + 1) / 2, c256 = (c64 + 3) / 4;
        const uint64_t wide = c256 * 40, middle = c128 * 22, slim = c64 * 15;
        if (rows * c256 >= 2048 && wide <= middle && wide <= slim) return run_mfma<2, 4, 2, 2, 2>(a, s);
        if (rows * c128 >= 512 && middle <= slim) return run_mfma<2, 2, 2, 2, 2>(a, s);
        return run_mfma<1, 1, 2, 2, 5>(a, s);
    }
    // (the narrowest tile that pads the prototypes least)
    if (K <= 32) return run_direct<4>(a, s);
    return ((uint64_t)K + 63) / 64 % 2 ? run_direct<8>(a, s) : run_direct<16>(a, s);
}

}  // namespace vq
