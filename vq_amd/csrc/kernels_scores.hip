// Scores of a batch (vqhip_scores_device in include/vqhip.h): S[i][j] = - sum_d (x[i][d] - w[j][d])^2, N x K in f32.
//
// The direct form of euclidean_distance without the root (src/helpers.rs:18-20), as the rest of this library measures its
// distances: |x|^2 - 2 x.w + |w|^2 on the matrix cores would cancel for the prototypes nearest a sample, which are the ones a
// draw is made of.  Two vector instructions per (sample, prototype, value) bound it: no matrix instruction subtracts first.
//
// A workgroup computes a 128 x 128 tile, a lane 8 x 8 of it in registers, so 16 values read from LDS feed 128 vector
// instructions; the next 16 values of the reduction are on their way from memory meanwhile.
#include <algorithm>

#include "vq_common.h"

namespace vq {

namespace {

constexpr int SC_THREADS = 256, SC_M = 128, SC_N = 128, SC_K = 16;
constexpr int SC_LD = SC_M + 4;       // a row of the tile per reduction value, moved 4 banks on from the one before

struct ScoreArgs {
    const float *X, *W;
    float *S;
    uint64_t N, ld;
    uint32_t K, D;
    uint32_t colTiles;
    int vecX, vecW, vecS;             // rows may be moved 16 bytes at a time
};

// Reduction values d0 .. d0 + 3 of one row, zero behind D or behind the last row (a pair of zeros adds nothing).
__device__ __forceinline__ float4 load4(const float *base, uint64_t row, bool on, uint32_t D, uint32_t d0, int vec)
{
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (!on || d0 >= D) return v;
    const float *p = base + row * D + d0;
    if (vec) return *(const float4 *)p;
    v.x = p[0];
    if (d0 + 1 < D) v.y = p[1];
    if (d0 + 2 < D) v.z = p[2];
    if (d0 + 3 < D) v.w = p[3];
    return v;
}

__global__ void __launch_bounds__(SC_THREADS) k_scores(const ScoreArgs a)
{
    __shared__ __attribute__((aligned(16))) float lx[2][SC_K][SC_LD], lw[2][SC_K][SC_LD];
    const uint64_t tile = blockIdx.x;
    const uint64_t row0 = tile / a.colTiles * SC_M;
    const uint32_t col0 = (uint32_t)(tile % a.colTiles) * SC_N;
    const int t = threadIdx.x;
    // staging: lane t moves values 4 (t & 3) .. + 3 of rows (t >> 2) and (t >> 2) + 64, of both operands
    const int sr = t >> 2, sd = (t & 3) * 4;
    const int ty = t >> 4, tx = t & 15;
    float acc[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;

    float4 px[2], pw[2];
    auto fetch = [&](uint32_t d) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint64_t r = row0 + sr + 64 * h;
            const uint32_t c = col0 + sr + 64 * h;
            px[h] = load4(a.X, r, r < a.N, a.D, d + sd, a.vecX);
            pw[h] = load4(a.W, c, c < a.K, a.D, d + sd, a.vecW);
        }
    };
    auto stage = [&](int b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float fx[4] = {px[h].x, px[h].y, px[h].z, px[h].w}, fw[4] = {pw[h].x, pw[h].y, pw[h].z, pw[h].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                lx[b][sd + e][sr + 64 * h] = fx[e];
                lw[b][sd + e][sr + 64 * h] = fw[e];
            }
        }
    };
    fetch(0);
    stage(0);
    __syncthreads();
    int b = 0;
    for (uint32_t d = 0; d < a.D; d += SC_K, b ^= 1) {
        const bool more = d + SC_K < a.D;
        if (more) fetch(d + SC_K);
#pragma unroll
        for (int k = 0; k < SC_K; ++k) {
            float x[8], w[8];
            *(float4 *)&x[0] = *(const float4 *)&lx[b][k][ty * 4];
            *(float4 *)&x[4] = *(const float4 *)&lx[b][k][64 + ty * 4];
            *(float4 *)&w[0] = *(const float4 *)&lw[b][k][tx * 4];
            *(float4 *)&w[4] = *(const float4 *)&lw[b][k][64 + tx * 4];
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
        const uint64_t r = row0 + (i >> 2) * 64 + ty * 4 + (i & 3);
        if (r >= a.N) continue;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const uint32_t c = col0 + g * 64 + tx * 4;
            float *out = a.S + r * a.ld + c;
            if (a.vecS && c + 4 <= a.K) {
                *(float4 *)out = make_float4(-acc[i][g * 4], -acc[i][g * 4 + 1], -acc[i][g * 4 + 2], -acc[i][g * 4 + 3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < a.K) out[e] = -acc[i][g * 4 + e];
            }
        }
    }
}

}  // namespace

hipError_t launch_scores(const float *dX, uint64_t N, uint32_t D, const float *dW, uint32_t K, float *dS, uint64_t ld, hipStream_t s)
{
    ScoreArgs a{dX, dW, dS, N, ld, K, D, (K + SC_N - 1) / SC_N, 0, 0, 0};
    const bool rows = D % 4 == 0;
    a.vecX = rows && ((uintptr_t)dX & 15) == 0;
    a.vecW = rows && ((uintptr_t)dW & 15) == 0;
    a.vecS = ld % 4 == 0 && ((uintptr_t)dS & 15) == 0;
    // one grid holds fewer than 2^31 workgroups
    const uint64_t most = ((1ull << 30) / a.colTiles) * SC_M;
    for (uint64_t off = 0; off < N; off += most) {
        a.X = dX + off * D;
        a.S = dS + off * ld;
        a.N = std::min(N - off, most);
        const uint64_t blocks = (a.N + SC_M - 1) / SC_M * a.colTiles;
        hipLaunchKernelGGL(k_scores, dim3((uint32_t)blocks), dim3(SC_THREADS), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace vq
