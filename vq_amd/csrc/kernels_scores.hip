// Scores of a batch (vqhip_scores_device in include/vqhip.h): S[i][j] = - sum_d (x[i][d] - w[j][d])^2, N x K in f32: the
// squared distances of euclidean_distance (src/helpers.rs:18-20) without the root.
//
// Two kernels.  Rows of up to DIRECT_D values: k_scores_direct, the formula as it stands on the vector units, a 128 x 128 tile a
// workgroup, 8 x 8 a lane, so that 16 values read from LDS feed 128 vector instructions.  Longer rows: k_scores_mfma, where the
// two vector instructions per (sample, prototype, value) of the direct form would bound it, the products run on the bf16
// matrix cores, six of exact three-piece splits (bf16x6, mfma_device.h), in the expanded form
//     |x - w|^2 = |x - c|^2 + |w - c|^2 - 2 (x - c).(w - c)
// with c the mean prototype, so that an offset all values share (pixels) does not cost digits.  Its rounding errors are those
// of the two norms, so the pairs whose distance is small beside them (below CLOSE of their sum: a sample and the few
// prototypes next to it) are measured again in the direct form: by 16 lanes a pair, or as a whole tile where they are many.
#include <algorithm>
#include <type_traits>

#include "mfma_device.h"
#include "vq_common.h"

namespace vq {

namespace {

constexpr int SC_THREADS = 256, SC_M = 128, SC_N = 128, SC_K = 16;
constexpr int SC_LD = SC_M + 4;       // a row of the tile per reduction value, moved 4 banks on from the one before

struct ScoreArgs {
    const float *X, *W, *C;           // C: the mean prototype, D values
    float *S;
    uint64_t N, ld;
    uint32_t K, D;
    uint32_t colTiles;
    int vecX, vecW, vecS, vecC;       // rows may be moved 16 bytes at a time
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

__global__ void __launch_bounds__(SC_THREADS, 2) k_scores_direct(const ScoreArgs a)
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
#pragma unroll 4
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

// ---------------------------------------------------------------------------------------------- matrix cores
constexpr uint32_t DIRECT_D = 32;     // rows up to this length: k_scores_direct
constexpr float CLOSE = 0.125f;       // of |x - c|^2 + |w - c|^2; distances below it are measured directly
constexpr int MF_THREADS = 256, MF_K = 16;

// The sum over 16 consecutive lanes, in the last of them
__device__ __forceinline__ float row_sum(float v)
{
    auto up = [](float x, auto ctrl) { return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, false)); };
    v += up(v, std::integral_constant<int, 0x111>());
    v += up(v, std::integral_constant<int, 0x112>());
    v += up(v, std::integral_constant<int, 0x114>());
    v += up(v, std::integral_constant<int, 0x118>());
    return v;
}

// A workgroup: 64 R x 64 R scores, a wave 32 R x 32 R of them in R x R accumulators of v_mfma_f32_32x32x16_bf16.  A operand: lane
// l holds sample l & 31, B operand: prototype l & 31; lanes 0-31 the reduction values 0 .. 7 of a step, lanes 32-63 8 .. 15.
// Result: lane l holds prototype l & 31 and samples 8 g + 4 (l >> 5) + e.
// LDS: a piece of a row is 16 bf16 = two 16-byte halves, swapped in every other group of 8 rows, so that 16 lanes reading the same
// half of 16 rows touch 16 different 16-byte slots of the 64 banks.
template <int R>
__global__ void __launch_bounds__(MF_THREADS, 2) k_scores_mfma(const ScoreArgs a)
{
    constexpr int TILE = 64 * R, WT = 32 * R;
    __shared__ __attribute__((aligned(16))) uint32_t lds[2][2][3][TILE][8];        // samples, prototypes; two buffers; three pieces
    auto &lx = lds[0], &lw = lds[1];
    __shared__ __attribute__((aligned(16))) float nx[TILE], nw[TILE];
    // workgroups are dealt to the 8 XCDs in turn: each takes a consecutive share of the tiles, so that the column tiles of the same
    // samples meet in one L2
    const uint32_t share = (gridDim.x + 7) / 8, tile = blockIdx.x % 8 * share + blockIdx.x / 8;
    const uint64_t row0 = (uint64_t)(tile / a.colTiles) * TILE;
    const uint32_t col0 = tile % a.colTiles * TILE;
    if (row0 >= a.N) return;
    const int t = threadIdx.x, lane = t & 63, half = lane >> 5, l31 = lane & 31, wr = t >> 7, wc = (t >> 6) & 1;
    const int sr = t >> 2, sd = (t & 3) * 4;          // staging: values sd .. + 3 of rows sr, sr + 64
    const int slot = ((((t & 3) >> 1) ^ (sr >> 3)) & 1) * 4 + (t & 1) * 2;       // ... and where they go, in dwords of the row's piece
    const int swap = (half ^ (l31 >> 3)) & 1;         // which slot this lane reads

    float4 px[R], pw[R], pc;
    float sx[R], sw[R];
#pragma unroll
    for (int i = 0; i < R; ++i) sx[i] = sw[i] = 0.0f;
    auto fetch = [&](uint32_t d) {
        pc = load4(a.C, 0, true, a.D, d + sd, a.vecC);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const uint64_t r = row0 + sr + 64 * i;
            const uint32_t c = col0 + sr + 64 * i;
            px[i] = load4(a.X, r, r < a.N, a.D, d + sd, a.vecX);
            pw[i] = load4(a.W, c, c < a.K, a.D, d + sd, a.vecW);
        }
    };
    auto put = [&](uint32_t (&to)[3][TILE][8], int row, const float4 &v) {
        uint32_t p[3], q[3];
        split3(v.x, v.y, p[0], p[1], p[2]);
        split3(v.z, v.w, q[0], q[1], q[2]);
#pragma unroll
        for (int c = 0; c < 3; ++c) *(uint2 *)&to[c][row][slot] = make_uint2(p[c], q[c]);
    };
    auto stage = [&](int b) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float4 x = make_float4(px[i].x - pc.x, px[i].y - pc.y, px[i].z - pc.z, px[i].w - pc.w);
            const float4 w = make_float4(pw[i].x - pc.x, pw[i].y - pc.y, pw[i].z - pc.z, pw[i].w - pc.w);
            sx[i] = fmaf(x.x, x.x, fmaf(x.y, x.y, fmaf(x.z, x.z, fmaf(x.w, x.w, sx[i]))));
            sw[i] = fmaf(w.x, w.x, fmaf(w.y, w.y, fmaf(w.z, w.z, fmaf(w.w, w.w, sw[i]))));
            put(lx[b], sr + 64 * i, x);
            put(lw[b], sr + 64 * i, w);
        }
    };
    f32x16 acc[R][R];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0.0f;

    fetch(0);
    stage(0);
    __syncthreads();
    int b = 0;
    for (uint32_t d = 0; d < a.D; d += MF_K, b ^= 1) {
        const bool more = d + MF_K < a.D;
        if (more) fetch(d + MF_K);
        u32x4 fx[R][3], fw[R][3];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < 3; ++c) {
                fx[i][c] = *(const u32x4 *)&lx[b][c][wr * WT + i * 32 + l31][swap * 4];
                fw[i][c] = *(const u32x4 *)&lw[b][c][wc * WT + i * 32 + l31][swap * 4];
            }
        // the six products that matter, the smallest first
        constexpr int PX[6] = {2, 0, 1, 1, 0, 0}, PW[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for (int p = 0; p < 6; ++p)
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < R; ++j) acc[i][j] = mma_bf(fx[i][PX[p]], fw[j][PW[p]], acc[i][j]);
        if (more) stage(b ^ 1);
        __syncthreads();
    }
    // the norms: 4 lanes hold the parts of a row
#pragma unroll
    for (int i = 0; i < R; ++i) {
        float x = sx[i], w = sw[i];
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            x += __shfl_xor(x, o);
            w += __shfl_xor(w, o);
        }
        if ((t & 3) == 0) {
            nx[sr + 64 * i] = x;
            nw[sr + 64 * i] = w;
        }
    }
    __syncthreads();

    // scores, and this wave's list of close pairs (sample << 8 | prototype, inside its tile) in the staging memory
    uint16_t *list = (uint16_t *)&lds[0][0][0][0][0] + (t >> 6) * (WT * WT);
    static_assert(sizeof lds >= 4 * WT * WT * sizeof(uint16_t), "a list of all pairs of the four waves fits");
    uint32_t n = 0;
    const bool inside = row0 + TILE <= a.N && col0 + TILE <= a.K;
    float *const out = a.S + (row0 + wr * WT) * a.ld + col0 + wc * WT;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const uint32_t lc = j * 32 + l31;
        const float w2 = nw[wc * WT + lc];
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const uint32_t lr0 = i * 32 + 8 * g + 4 * half;
                const float4 x2 = *(const float4 *)&nx[wr * WT + lr0];
                const float fx2[4] = {x2.x, x2.y, x2.z, x2.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t lr = lr0 + e;
                    const float both = fx2[e] + w2, s = fmaf(2.0f, acc[i][j][4 * g + e], -both);
                    const bool on = inside || (row0 + wr * WT + lr < a.N && col0 + wc * WT + lc < a.K);
                    const bool close = on && !(-s >= CLOSE * both);               // (also where anything is not finite)
                    if (on && !close) out[lr * a.ld + lc] = s;
                    const uint64_t m = __ballot(close);
                    if (m) {
                        if (close) list[n + __popcll(m & ((1ull << lane) - 1))] = (uint16_t)(lr << 8 | lc);
                        n += __popcll(m);
                    }
                }
            }
    }
    if (n == 0) return;
    const uint64_t wrow = row0 + wr * WT;
    const uint32_t wcol = col0 + wc * WT;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (n <= WT * WT / 32) {
        // 16 lanes a pair, two pairs at a time
        const uint32_t g = lane >> 4, gl = lane & 15;
        for (uint32_t p = g; p < n; p += 8) {
            const bool two = p + 4 < n;
            const uint32_t q0 = list[p], q1 = list[two ? p + 4 : p];
            const float *x0 = a.X + (wrow + (q0 >> 8)) * a.D, *w0 = a.W + (uint64_t)(wcol + (q0 & 255)) * a.D;
            const float *x1 = a.X + (wrow + (q1 >> 8)) * a.D, *w1 = a.W + (uint64_t)(wcol + (q1 & 255)) * a.D;
            float s0 = 0.0f, s1 = 0.0f;
            for (uint32_t d = gl * 4; d < a.D; d += 64) {
                const float4 u0 = load4(x0, 0, true, a.D, d, a.vecX), v0 = load4(w0, 0, true, a.D, d, a.vecW);
                const float4 u1 = load4(x1, 0, true, a.D, d, a.vecX), v1 = load4(w1, 0, true, a.D, d, a.vecW);
                const float e0 = u0.x - v0.x, e1 = u0.y - v0.y, e2 = u0.z - v0.z, e3 = u0.w - v0.w;
                const float f0 = u1.x - v1.x, f1 = u1.y - v1.y, f2 = u1.z - v1.z, f3 = u1.w - v1.w;
                s0 = fmaf(e0, e0, fmaf(e1, e1, fmaf(e2, e2, fmaf(e3, e3, s0))));
                s1 = fmaf(f0, f0, fmaf(f1, f1, fmaf(f2, f2, fmaf(f3, f3, s1))));
            }
            s0 = row_sum(s0);
            s1 = row_sum(s1);
            if (gl == 15) {
                a.S[(wrow + (q0 >> 8)) * a.ld + wcol + (q0 & 255)] = -s0;
                if (two) a.S[(wrow + (q1 >> 8)) * a.ld + wcol + (q1 & 255)] = -s1;
            }
        }
        return;
    }
    // the wave's whole tile, 4 R x 4 R scores a lane
    __threadfence();                                   // (its scores so far are written, before others lanes write some of them again)
    const int ty = lane >> 3, tx = lane & 7;
    float sum[4 * R][4 * R];
#pragma unroll
    for (int i = 0; i < 4 * R; ++i)
#pragma unroll
        for (int j = 0; j < 4 * R; ++j) sum[i][j] = 0.0f;
    for (uint32_t d = 0; d < a.D; d += 4) {
        float4 x[4 * R], w[4 * R];
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) {
            x[i] = load4(a.X, wrow + ty + 8 * i, wrow + ty + 8 * i < a.N, a.D, d, a.vecX);
            w[i] = load4(a.W, wcol + tx + 8 * i, wcol + tx + 8 * i < a.K, a.D, d, a.vecW);
        }
#pragma unroll
        for (int i = 0; i < 4 * R; ++i)
#pragma unroll
            for (int j = 0; j < 4 * R; ++j) {
                const float e0 = x[i].x - w[j].x, e1 = x[i].y - w[j].y, e2 = x[i].z - w[j].z, e3 = x[i].w - w[j].w;
                sum[i][j] = fmaf(e3, e3, fmaf(e2, e2, fmaf(e1, e1, fmaf(e0, e0, sum[i][j]))));
            }
    }
#pragma unroll
    for (int i = 0; i < 4 * R; ++i)
#pragma unroll
        for (int j = 0; j < 4 * R; ++j) {
            const uint64_t r = wrow + ty + 8 * i;
            const uint32_t c = wcol + tx + 8 * j;
            if (r < a.N && c < a.K) a.S[r * a.ld + c] = -sum[i][j];
        }
}

template <int R>
hipError_t run_mfma(ScoreArgs a, hipStream_t s)
{
    constexpr uint32_t TILE = 64 * R;
    a.colTiles = (a.K + TILE - 1) / TILE;
    const uint64_t N = a.N, most = std::max<uint64_t>(1, (1u << 30) / a.colTiles) * TILE;        // a grid holds fewer than 2^31 workgroups
    const float *X = a.X;
    float *S = a.S;
    for (uint64_t off = 0; off < N; off += most) {
        a.X = X + off * a.D;
        a.S = S + off * a.ld;
        a.N = std::min(N - off, most);
        const uint64_t tiles = (a.N + TILE - 1) / TILE * a.colTiles;
        hipLaunchKernelGGL((k_scores_mfma<R>), dim3((uint32_t)((tiles + 7) / 8 * 8)), dim3(MF_THREADS), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

hipError_t launch_scores(const float *dX, uint64_t N, uint32_t D, const float *dW, const float *dC, uint32_t K, float *dS, uint64_t ld, hipStream_t s)
{
    ScoreArgs a{dX, dW, dC, dS, N, ld, K, D, (K + SC_N - 1) / SC_N, 0, 0, 0, 0};
    const bool rows = D % 4 == 0;
    a.vecX = rows && ((uintptr_t)dX & 15) == 0;
    a.vecW = rows && ((uintptr_t)dW & 15) == 0;
    a.vecC = rows && ((uintptr_t)dC & 15) == 0;
    a.vecS = ld % 4 == 0 && ((uintptr_t)dS & 15) == 0;
    if (D > DIRECT_D) {
        // the large tile reads every operand half as often; the small one fills the card with fewer scores
        const uint64_t large = (N + 127) / 128 * ((K + 127) / 128);
        return large >= 512 ? run_mfma<2>(a, s) : run_mfma<1>(a, s);
    }
    // one grid holds fewer than 2^31 workgroups
    const uint64_t most = ((1ull << 30) / a.colTiles) * SC_M;
    for (uint64_t off = 0; off < N; off += most) {
        a.X = dX + off * D;
        a.S = dS + off * ld;
        a.N = std::min(N - off, most);
        const uint64_t blocks = (a.N + SC_M - 1) / SC_M * a.colTiles;
        hipLaunchKernelGGL(k_scores_direct, dim3((uint32_t)blocks), dim3(SC_THREADS), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace vq
