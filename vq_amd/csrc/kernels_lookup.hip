// Codebook lookup and its gradient (vqhip_lookup_device, vqhip_lookup_gradient_device in include/vqhip.h).
//
//     lookup     Y[i] = scale * T[idx[i]]                               (a zero row where idx[i] is outside [0, K))
//     gradient   G[k] (+)= scale * sum over { i : idx[i] = k } dY[i]    and how many rows each sum has
//
// The reference keeps its prototypes in a Vec and reads `prototypes[idx].vector` one sample at a time (src/glvq/glvq.rs:231
// reads the name beside it); these are that read for a batch of indices and the transposed operation, which no part of the
// reference has.
//
// The gradient is a scatter-add.  Atomic additions would make the order of the sums, and so their last bits, differ from run
// to run, and they serialise on crowded rows.  Instead the rows are put in the order of their indices (a stable radix sort of
// (index, row) pairs: 8 bytes per row against D values per row) and each run of equal indices is summed in that order, so the
// same inputs give the same bits on every call:
//     (few rows and a table that is not large: all of it in one launch, k_grad_single)
//     sort     k_sort_small (one workgroup, all in LDS) or k_sort_count / k_sort_scan / k_sort_move per digit
//     reduce   k_grad_reduce: the sorted positions are cut into equal chunks whatever the runs are, so one crowded index
//              costs no more than many rare ones.  A run inside one chunk is finished there; the parts of a run that crosses
//              chunk borders go to the workspace in f32
//     join     k_grad_join: adds up the parts of those runs in order, writes the rows no index names, and the counts
//
// What bounds them: memory.  Lookup of 2000000 rows of 128 out of 256, f32: 177 us, stores at 5.8 TB/s (a fill of this card: 6.8).
// Gradient of 2000000 rows of 128 over 256, f32: 242 us, of which the sums are 195 at 5.2 TB/s, read in the order of the indices, and
// the sort 36.  16384 rows of 4096 over 65536, bf16 to f32: 266 us, of which clearing the rows nobody names is about 165 at
// 5.6 TB/s, the sums 50 at 6 TB/s.
#include <algorithm>
#include <type_traits>

#include "codes_device.h"

namespace vq {

namespace {

using u32x4 = uint32_t __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------------------------- lookup
struct LookupArgs {
    const void *T;
    uint64_t ldt;
    const uint32_t *idx;
    uint64_t N;
    uint32_t K, D;
    float scale;
    void *Y;
    uint64_t ldy;
    int log2g;              // 2^log2g lanes per row and column step
};

constexpr int LOOK_THREADS = 256;

// 16 bytes of consecutive elements, from any multiple of an element's size: rows of any length and pitch are moved alike.  Stores
// do not stay in the caches: what is written here is read once at best, and the table is read over and over.
typedef uint32_t words_by4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t words_by2 __attribute__((ext_vector_type(4), aligned(2)));
template <class T>
struct Piece {
    static constexpr int E = 16 / (int)sizeof(T);
    using words = typename std::conditional<sizeof(T) == 4, words_by4, words_by2>::type;
    T v[E];
};
template <class T>
__device__ __forceinline__ Piece<T> load_piece(const T *p) { return __builtin_bit_cast(Piece<T>, (u32x4)*(const typename Piece<T>::words *)p); }
template <class T>
__device__ __forceinline__ void store_piece(T *p, const Piece<T> &v) { __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (typename Piece<T>::words *)p); }

// 2^log2g lanes share a row; blockIdx.y picks the column step.  U rows are in flight per lane: index -> row -> store is a
// chain of two memory latencies, and nothing else hides them.
template <class T, int U>
__global__ void __launch_bounds__(LOOK_THREADS) k_lookup(const LookupArgs a)
{
    using P = Piece<T>;
    const int g = 1 << a.log2g;
    const uint32_t col = ((uint32_t)blockIdx.y * g + (threadIdx.x & (g - 1))) * P::E;
    if (col >= a.D) return;
    const uint32_t rows = LOOK_THREADS >> a.log2g;                   // rows of one step of the block
    const T *table = (const T *)a.T + col;
    T *out = (T *)a.Y + col;
    const uint32_t left = a.D - col;                                 // elements of the row from here on
    auto work = [&](auto whole) {
        constexpr bool W = decltype(whole)::value;
        for (uint64_t base = (uint64_t)blockIdx.x * rows * U + (threadIdx.x >> a.log2g); base < a.N; base += (uint64_t)gridDim.x * rows * U) {
            uint32_t k[U];
            P v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t i = base + (uint64_t)u * rows;
                k[u] = i < a.N ? a.idx[i] : a.K;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const T *row = table + (uint64_t)k[u] * a.ldt;
                if (W && k[u] < a.K) {
                    v[u] = load_piece(row);
                } else {
#pragma unroll
                    for (int e = 0; e < P::E; ++e) v[u].v[e] = !W && k[u] < a.K && (uint32_t)e < left ? row[e] : (T)0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint64_t i = base + (uint64_t)u * rows;
                if (i >= a.N) break;
                if (k[u] < a.K) {
#pragma unroll
                    for (int e = 0; e < P::E; ++e) v[u].v[e] = narrow<T>(widen(v[u].v[e]) * a.scale);
                }
                T *to = out + i * a.ldy;
                if (W) {
                    store_piece(to, v[u]);
                } else {
#pragma unroll
                    for (int e = 0; e < P::E; ++e)
                        if ((uint32_t)e < left) to[e] = v[u].v[e];
                }
            }
        }
    };
    if (left >= P::E)
        work(std::true_type());
    else
        work(std::false_type());
}

template <class T>
hipError_t run_lookup(LookupArgs a, hipStream_t s)
{
    const uint32_t steps = (a.D + Piece<T>::E - 1) / Piece<T>::E;
    a.log2g = 0;
    while ((1u << a.log2g) < steps && a.log2g < 8) ++a.log2g;
    const uint32_t cols = (steps + (1u << a.log2g) - 1) >> a.log2g;
    const uint64_t rows = LOOK_THREADS >> a.log2g;
    // four rows in flight per lane once that still leaves every CU several workgroups
    const bool four = (a.N + 4 * rows - 1) / (4 * rows) * cols >= 2048;
    const uint64_t per = four ? 4 * rows : rows;
    const uint32_t blocks = (uint32_t)std::min<uint64_t>((a.N + per - 1) / per, 1u << 20);
    if (four)
        hipLaunchKernelGGL((k_lookup<T, 4>), dim3(blocks, cols), dim3(LOOK_THREADS), 0, s, a);
    else
        hipLaunchKernelGGL((k_lookup<T, 1>), dim3(blocks, cols), dim3(LOOK_THREADS), 0, s, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------- sort
// Stable: equal keys stay in the order of their rows.  A workgroup owns a tile of consecutive positions, a wave a consecutive
// part of the tile, and takes 64 of them at a time, so (wave, step, lane) is the order of the positions.  The place of an
// element among those with its digit: how many the waves before it hold (a table per wave, summed once), how many the steps
// before it held (the table's running count), and how many lanes below it hold the same digit (a ballot per digit bit).
constexpr int SORT_MAX_BITS = 11;                                   // bits of one pass
constexpr uint32_t NONE = 0xFFFFFFFFu;

// The lanes whose digit of `bits` <= MAX bits is this lane's
template <int MAX>
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits)
{
    uint32_t lo = ~0u, hi = ~0u;
#pragma unroll
    for (int b = 0; b < MAX; ++b) {
        if (b < bits) {                                                     // (the same in all lanes)
            const uint64_t v = __ballot((d >> b) & 1);
            const uint32_t mine = (uint32_t)((int32_t)(d << (31 - b)) >> 31);
            lo &= ~((uint32_t)v ^ mine);
            hi &= ~((uint32_t)(v >> 32) ^ mine);
        }
    }
    return (uint64_t)hi << 32 | lo;
}

// Exclusive prefix sum over the n <= 2048 entries of `a` (LDS), by the whole workgroup of THREADS lanes.
template <int THREADS>
__device__ void scan_bins(uint32_t *a, uint32_t n, uint32_t *tmp)
{
    const uint32_t t = threadIdx.x, per = (n + THREADS - 1) / THREADS;
    uint32_t sum = 0;
    for (uint32_t j = 0; j < per; ++j)
        if (t * per + j < n) sum += a[t * per + j];
    uint32_t x = sum;
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t y = __shfl_up(x, o);
        if ((int)(t & 63) >= o) x += y;
    }
    if ((t & 63) == 63) tmp[t >> 6] = x;
    __syncthreads();
    uint32_t before = x - sum;
    for (uint32_t w = 0; w < t >> 6; ++w) before += tmp[w];
    for (uint32_t j = 0; j < per; ++j)
        if (t * per + j < n) {
            const uint32_t v = a[t * per + j];
            a[t * per + j] = before;
            before += v;
        }
    __syncthreads();
}

// Rows of zeros where start[k] is NONE, 2^log2g lanes a row, 16 bytes a lane and store; 2 where rows are no whole words
struct ZeroArgs {
    char *G;
    uint64_t pitch, bytes;          // of a row, in bytes
    int words;
    int log2g;
    uint32_t blocks;                // workgroups that do it, behind the others; 0: none
};

__device__ __forceinline__ void zero_rows(const ZeroArgs &z, const uint32_t *start, uint32_t K, uint32_t block, uint32_t threads)
{
    const uint32_t gl = threadIdx.x & ((1u << z.log2g) - 1), groups = threads >> z.log2g;
    const words_by4 zero = {0, 0, 0, 0};
    for (uint64_t k = (uint64_t)block * groups + (threadIdx.x >> z.log2g); k < K; k += (uint64_t)z.blocks * groups) {
        if (start[k] != NONE) continue;
        char *row = z.G + k * z.pitch;
        if (z.words) {
            for (uint64_t at = gl * 16; at + 16 <= z.bytes; at += 16ull << z.log2g) __builtin_nontemporal_store(zero, (words_by4 *)(row + at));
            for (uint64_t at = (z.bytes & ~15ull) + gl * 4; at < z.bytes; at += 4ull << z.log2g) __builtin_nontemporal_store(0u, (uint32_t *)(row + at));
        } else {
            for (uint64_t at = gl * 2; at < z.bytes; at += 2ull << z.log2g) __builtin_nontemporal_store((uint16_t)0, (uint16_t *)(row + at));
        }
    }
}

struct SortArgs {
    const uint32_t *idx;            // first pass: keys are min(idx, K), rows their positions; null later
    const uint32_t *keys_in, *rows_in;
    uint32_t *keys, *rows;          // result of the pass
    uint32_t *hist;                 // [bins][tiles]
    uint32_t *total;                // [bins]
    uint32_t *start;                // K entries: NONE in the first pass, then (with `mark`) 0 where an index occurs
    const uint32_t *mark;           // the indices, or null
    uint32_t N, K, tiles;
    int shift, bits;
    int scanned;                    // k_sort_scan has summed hist; otherwise every tile of a move does
    ZeroArgs zero;                  // rows to clear beside the first move
};

__device__ __forceinline__ uint32_t load_key(const SortArgs &a, uint32_t i)
{
    return a.idx ? min(a.idx[i], a.K) : a.keys_in[i];
}
__device__ __forceinline__ void mark_present(const SortArgs &a, uint64_t from, uint64_t step)
{
    for (uint64_t i = from; i < a.N; i += step) {
        const uint32_t k = a.mark[i];
        if (k < a.K) a.start[k] = 0;
    }
}

// THREADS x ITEMS positions a workgroup
template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) k_sort_count(const SortArgs a)
{
    __shared__ uint32_t bins[1 << SORT_MAX_BITS];
    constexpr uint32_t TILE = THREADS * ITEMS;
    const uint32_t nb = 1u << a.bits, tile = blockIdx.x;
    for (uint32_t b = threadIdx.x; b < nb; b += THREADS) bins[b] = 0;
    if (a.idx)
        for (uint64_t k = (uint64_t)tile * THREADS + threadIdx.x; k < a.K; k += (uint64_t)gridDim.x * THREADS) a.start[k] = NONE;
    __syncthreads();
    const uint32_t base = tile * TILE, end = min(a.N - base, TILE);
    uint32_t key[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) key[j] = threadIdx.x + j * THREADS < end ? load_key(a, base + threadIdx.x + j * THREADS) : 0;
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
        if (threadIdx.x + j * THREADS < end) atomicAdd(&bins[(key[j] >> a.shift) & (nb - 1)], 1u);
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < nb; b += THREADS) a.hist[(size_t)b * a.tiles + tile] = bins[b];
}

// One workgroup per bin: exclusive prefix sum over the tiles, in place, and the bin's total.
// Workgroups behind the bins': which indices occur.
__global__ void __launch_bounds__(256) k_sort_scan(const SortArgs a)
{
    __shared__ uint32_t part[4];
    const uint32_t nb = 1u << a.bits, tiles = a.tiles;
    if (blockIdx.x >= nb) return mark_present(a, (uint64_t)(blockIdx.x - nb) * 256 + threadIdx.x, (uint64_t)(gridDim.x - nb) * 256);
    uint32_t *h = a.hist + (size_t)blockIdx.x * tiles, *total = a.total;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t carry = 0;
    for (uint32_t base = 0; base < tiles; base += 256) {
        const uint32_t i = base + threadIdx.x, v = i < tiles ? h[i] : 0;
        uint32_t x = v;
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        if (lane == 63) part[w] = x;
        __syncthreads();
        uint32_t before = carry + x - v;
        for (int k = 0; k < w; ++k) before += part[k];
        if (i < tiles) h[i] = before;
        carry += part[0] + part[1] + part[2] + part[3];
        __syncthreads();
    }
    if (threadIdx.x == 0) total[blockIdx.x] = carry;
}

// Ranks `ITEMS` elements per lane (held in registers, wave-consecutive) by their digit; on return rank[j] is the element's
// place inside the tile and first[d] the first place of digit d.  `count`: WAVES tables of nb counters.
template <int WAVES, int ITEMS, int MAX>
__device__ __forceinline__ void rank_tile(const uint32_t (&key)[ITEMS], uint32_t valid, int shift, int bits, uint16_t *count, uint32_t *first, uint32_t *tmp,
                                          uint32_t (&rank)[ITEMS])
{
    const uint32_t nb = 1u << bits, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    for (uint32_t b = threadIdx.x; b < nb * WAVES / 2; b += WAVES * 64) ((uint32_t *)count)[b] = 0;
    __syncthreads();
    uint16_t *mine = count + w * nb;
    uint64_t same[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const bool on = (w * ITEMS + j) * 64 + lane < valid;
        same[j] = same_digit<MAX + 1>(on ? (key[j] >> shift) & (nb - 1) : nb, bits + 1);    // (bit `bits` set: no digit of the tile)
    }
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const bool on = (w * ITEMS + j) * 64 + lane < valid;
        const uint32_t d = (key[j] >> shift) & (nb - 1);
        const uint32_t below = __builtin_amdgcn_mbcnt_hi((uint32_t)(same[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same[j], 0));
        uint32_t had = 0;
        if (on) had = mine[d];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");              // every lane has read before the first of them adds
        if (on && below == 0) mine[d] = (uint16_t)(had + __popcll(same[j]));
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        rank[j] = had + below;
    }
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < nb; b += WAVES * 64) {
        uint32_t c[WAVES], run = 0;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) c[k] = count[k * nb + b];
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            count[k * nb + b] = (uint16_t)run;
            run += c[k];
        }
        first[b] = run;
    }
    __syncthreads();
    scan_bins<WAVES * 64>(first, nb, tmp);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
        if ((w * ITEMS + j) * 64 + lane < valid) {
            const uint32_t d = (key[j] >> shift) & (nb - 1);
            rank[j] += first[d] + mine[d];
        }
}

template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) k_sort_move(const SortArgs a)
{
    constexpr int WAVES = THREADS / 64;
    constexpr uint32_t TILE = THREADS * ITEMS;
    __shared__ uint32_t lkey[TILE], lrow[TILE], tmp[WAVES];
    extern __shared__ uint32_t tables[];                                    // per bin: first, base, and WAVES 2-byte counters
    const uint32_t nb = 1u << a.bits, tile = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (tile >= a.tiles) return zero_rows(a.zero, a.start, a.K, tile - a.tiles, THREADS);
    uint32_t *first = tables, *base = tables + nb;
    uint16_t *count = (uint16_t *)(tables + 2 * nb);
    const uint32_t begin = tile * TILE, valid = min(a.N - begin, TILE);
    uint32_t key[ITEMS], row[ITEMS], rank[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const uint32_t p = (w * ITEMS + j) * 64 + lane;
        key[j] = p < valid ? load_key(a, begin + p) : 0;
        row[j] = p < valid ? (a.idx ? begin + p : a.rows_in[begin + p]) : 0;
    }
    constexpr int EACH = (1 << SORT_MAX_BITS) / THREADS;
    uint32_t before[EACH];                                                  // of this lane's bins: in the tiles in front of this one
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const uint32_t b = threadIdx.x + j * THREADS;
        before[j] = 0;
        if (b < nb) {
            const uint32_t *h = a.hist + (size_t)b * a.tiles;
            if (a.scanned) {
                before[j] = h[tile];
                base[b] = a.total[b];
            } else {
                uint32_t all = 0;
                for (uint32_t i = 0; i < a.tiles; ++i) {
                    const uint32_t v = h[i];
                    before[j] += i < tile ? v : 0;
                    all += v;
                }
                base[b] = all;
            }
        }
    }
    __syncthreads();
    scan_bins<THREADS>(base, nb, tmp);
    rank_tile<WAVES, ITEMS, SORT_MAX_BITS>(key, valid, a.shift, a.bits, count, first, tmp, rank);
    // where this tile's elements of a digit go, less their first place in the tile
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const uint32_t b = threadIdx.x + j * THREADS;
        if (b < nb) base[b] += before[j] - first[b];
    }
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
        if ((w * ITEMS + j) * 64 + lane < valid) {
            lkey[rank[j]] = key[j];
            lrow[rank[j]] = row[j];
        }
    __syncthreads();
    // through LDS in the order of the places, so that the elements of a digit leave as one consecutive piece
    for (uint32_t p = threadIdx.x; p < valid; p += THREADS) {
        const uint32_t k = lkey[p], to = base[(k >> a.shift) & (nb - 1)] + p;
        a.keys[to] = k;
        a.rows[to] = lrow[p];
    }
}

// All passes in one workgroup and one launch, for at most THREADS x ITEMS rows.
constexpr uint32_t SMALL_TILE = 8192;
constexpr int SMALL_MAX_BITS = 9;                                    // 256 indices and one for the rows without a place: one pass

template <int THREADS, int ITEMS>
__device__ __forceinline__ void sort_in_lds(const SortArgs &a, int key_bits, uint32_t *lkey, uint32_t *lrow, uint16_t *count, uint32_t *first, uint32_t *tmp)
{
    constexpr int WAVES = THREADS / 64;
    const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t key[ITEMS], row[ITEMS], rank[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const uint32_t p = (w * ITEMS + j) * 64 + lane;
        key[j] = p < a.N ? load_key(a, p) : 0;
        row[j] = p;
    }
    const int passes = (key_bits + SMALL_MAX_BITS - 1) / SMALL_MAX_BITS, bits = (key_bits + passes - 1) / passes;
    for (int pass = 0; pass < passes; ++pass) {
        rank_tile<WAVES, ITEMS, SMALL_MAX_BITS>(key, a.N, pass * bits, bits, count, first, tmp, rank);
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
            if ((w * ITEMS + j) * 64 + lane < a.N) {
                lkey[rank[j]] = key[j];
                lrow[rank[j]] = row[j];
            }
        __syncthreads();
        if (pass + 1 < passes) {
#pragma unroll
            for (int j = 0; j < ITEMS; ++j) {
                const uint32_t p = (w * ITEMS + j) * 64 + lane;
                if (p < a.N) {
                    key[j] = lkey[p];
                    row[j] = lrow[p];
                }
            }
            __syncthreads();
        }
    }
}

template <int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) k_sort_small(const SortArgs a, int key_bits)
{
    constexpr int WAVES = THREADS / 64;
    constexpr uint32_t TILE = THREADS * ITEMS;
    __shared__ uint32_t lkey[TILE], lrow[TILE];                             // 64 KiB at most
    __shared__ __attribute__((aligned(4))) uint16_t count[WAVES << SMALL_MAX_BITS];
    __shared__ uint32_t first[1 << SMALL_MAX_BITS], tmp[WAVES];
    if (blockIdx.x != 0) {                                                  // the other workgroups only set `start`, or clear rows
        if (a.zero.blocks) return zero_rows(a.zero, a.start, a.K, blockIdx.x - 1, THREADS);
        for (uint64_t k = (uint64_t)(blockIdx.x - 1) * THREADS + threadIdx.x; k < a.K; k += (uint64_t)(gridDim.x - 1) * THREADS) a.start[k] = NONE;
        return;
    }
    sort_in_lds<THREADS, ITEMS>(a, key_bits, lkey, lrow, count, first, tmp);
    for (uint32_t p = threadIdx.x; p < a.N; p += THREADS) {
        a.keys[p] = lkey[p];
        a.rows[p] = lrow[p];
    }
}

template <int THREADS, int ITEMS>
void run_sort_small(const SortArgs &a, int key_bits, hipStream_t s)
{
    const uint32_t fill = a.zero.blocks ? a.zero.blocks : std::min<uint32_t>((a.K + THREADS - 1) / THREADS, 256);
    hipLaunchKernelGGL((k_sort_small<THREADS, ITEMS>), dim3(1 + fill), dim3(THREADS), 0, s, a, key_bits);
}

template <int THREADS, int ITEMS>
void run_sort_pass(SortArgs a, hipStream_t s)
{
    const uint32_t nb = 1u << a.bits, marks = a.mark ? std::min<uint32_t>((a.N + 255) / 256, 1024) : 0;
    // a launch less where the table of counts is small (32 KiB at most) and a row of it short: every tile sums it for itself.  us: 9000
    // rows of 64 over 256 23.5 / 21.4, 20000 of 64 over 30000 (two passes) 38.9 / 35.5; 49 tiles, 100000 of 8 over 30: 31.9 / 36.7
    a.scanned = marks || a.tiles > 16 || (uint64_t)nb * a.tiles > 8192;
    hipLaunchKernelGGL((k_sort_count<THREADS, ITEMS>), dim3(a.tiles), dim3(THREADS), 0, s, a);
    if (a.scanned) hipLaunchKernelGGL(k_sort_scan, dim3(nb + marks), dim3(256), 0, s, a);
    hipLaunchKernelGGL((k_sort_move<THREADS, ITEMS>), dim3(a.tiles + a.zero.blocks), dim3(THREADS), nb * (8 + THREADS / 64 * 2), s, a);
}

__global__ void __launch_bounds__(256) k_mark(const SortArgs a) { mark_present(a, (uint64_t)blockIdx.x * 256 + threadIdx.x, (uint64_t)gridDim.x * 256); }

__global__ void k_fill_u32(uint32_t *p, uint64_t n, uint32_t v)
{
    for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (uint64_t)gridDim.x * blockDim.x) p[i] = v;
}

// ---------------------------------------------------------------------------------------------- reduce and join
struct GradArgs {
    const void *dY;
    uint64_t ldy;
    const uint32_t *keys, *rows;    // sorted
    uint32_t N, K, D;
    float scale;
    void *G;
    uint64_t ldg;
    int accumulate, cleared;        // cleared: the rows no index names are zero already
    uint32_t *start, *end;          // K each: first place and place behind the last of every index that occurs
    uint32_t *counts;               // nullable
    float *parts;                   // [chunks][2][dpad]: head (a run that began in an earlier chunk), tail (one that goes on)
    uint32_t dpad, chunk, chunks, slabs;
    int log2g;
};

constexpr int GRAD_THREADS = 256;
constexpr int GRAD_FLIGHT = 8;      // rows a lane has in flight

// A lane's columns of a row: E of them from `at` on, the first `skip` of which are its neighbour's (the last lane of a row whose
// length is no multiple of E begins earlier, so that every load is a whole one).
template <int E>
struct Columns {
    uint32_t at, skip;
    bool mine;
    __device__ Columns(uint32_t first, uint32_t D) : at(first + E <= D ? first : D - E), skip(first - at), mine(first < D) {}
};
template <class T, int E>
__device__ __forceinline__ Pack<T, E * (int)sizeof(T)> load_columns(const T *p)              // from any multiple of an element's size
{
    Pack<T, E * (int)sizeof(T)> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}
template <class T, int E>
__device__ __forceinline__ void store_columns(T *p, const Pack<T, E * (int)sizeof(T)> &v, uint32_t skip)
{
    if (E > 1 && skip == 0) {
        static_assert(E == 1 || E * sizeof(T) == 16, "one element or 16 bytes");
        if constexpr (E > 1) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, v), (typename Piece<T>::words *)p);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if ((uint32_t)e >= skip) p[e] = v.v[e];
    }
}

// One finished row piece: G (+)= scale * sum, rounded once.
template <class TO, int E>
__device__ __forceinline__ void store_grad(const GradArgs &a, uint32_t k, const Columns<E> &c, const float (&acc)[E])
{
    TO *g = (TO *)a.G + (uint64_t)k * a.ldg + c.at;
    Pack<TO, E * (int)sizeof(TO)> o;
    if (a.accumulate) {
        o = load_columns<TO, E>(g);
#pragma unroll
        for (int e = 0; e < E; ++e) o.v[e] = narrow<TO>(fmaf(acc[e], a.scale, widen(o.v[e])));
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) o.v[e] = narrow<TO>(acc[e] * a.scale);
    }
    store_columns<TO, E>(g, o, c.skip);
}
template <class TO, int E>
__device__ __forceinline__ void store_zeros(const GradArgs &a, uint64_t k, const Columns<E> &c)
{
    Pack<TO, E * (int)sizeof(TO)> zero;
#pragma unroll
    for (int e = 0; e < E; ++e) zero.v[e] = (TO)0.0f;
    store_columns<TO, E>((TO *)a.G + k * a.ldg + c.at, zero, c.skip);
}

// Sums the runs of the sorted places [p0, p1) over this lane's E columns (at dY; none of its own: !mine) in their order.  done(k,
// from, upto, sum) for every run of an index inside the table, at its end or the range's.
template <class T, int E, class Keys, class Done>
__device__ __forceinline__ void sum_runs(const Keys keys, const Keys rows, uint32_t p0, uint32_t p1, uint32_t K, const T *dY, uint64_t ldy, const Done &done)
{
    float acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
    uint32_t cur = keys[p0], from = p0;
    for (uint32_t p = p0; p < p1; p += GRAD_FLIGHT) {
        uint32_t key[GRAD_FLIGHT], row[GRAD_FLIGHT];
        Pack<T, E * (int)sizeof(T)> v[GRAD_FLIGHT];
#pragma unroll
        for (int j = 0; j < GRAD_FLIGHT; ++j) {
            const uint32_t q = min(p + j, p1 - 1);
            key[j] = keys[q];
            row[j] = rows[q];
        }
        if (key[0] >= K) {                                         // sorted: nothing but rows without a place from here on
            if (cur < K) done(cur, from, p, acc);
            return;
        }
#pragma unroll
        for (int j = 0; j < GRAD_FLIGHT; ++j)                      // (a row without a place is not read: its batch's first is, again)
            v[j] = load_columns<T, E>(dY + (uint64_t)(key[j] < K ? row[j] : row[0]) * ldy);
#pragma unroll
        for (int j = 0; j < GRAD_FLIGHT; ++j) {
            if (p + j < p1) {
                if (key[j] != cur) {
                    if (cur < K) done(cur, from, p + j, acc);
                    cur = key[j];
                    from = p + j;
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
                }
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += widen(v[j].v[e]);
            }
        }
    }
    if (cur < K) done(cur, from, p1, acc);
}

// 2^log2g lanes own one chunk of sorted places and E * 2^log2g columns of it.
template <class T, class TO, int E>
__global__ void __launch_bounds__(GRAD_THREADS) k_grad_reduce(const GradArgs a)
{
    const uint64_t group = ((uint64_t)blockIdx.x * GRAD_THREADS + threadIdx.x) >> a.log2g;
    const uint32_t c = (uint32_t)(group / a.slabs), slab = (uint32_t)(group % a.slabs);
    if (c >= a.chunks) return;
    const uint32_t gl = threadIdx.x & ((1u << a.log2g) - 1);
    const Columns<E> cols(((slab << a.log2g) + gl) * E, a.D);
    const bool first = slab == 0 && gl == 0;
    const uint32_t p0 = c * a.chunk, p1 = min(a.N, p0 + a.chunk);
    const bool left = p0 > 0 && a.keys[p0 - 1] == a.keys[p0];     // the first run began in an earlier chunk
    const uint32_t behind = p1 < a.N ? a.keys[p1] : NONE;
    sum_runs<T, E>(a.keys, a.rows, p0, p1, a.K, (const T *)a.dY + (cols.mine ? cols.at : 0), a.ldy, [&](uint32_t k, uint32_t from, uint32_t upto, const float (&acc)[E]) {
        const bool l = from == p0 && left, r = upto == p1 && behind == k;
        if (first) {
            if (!l) a.start[k] = from;
            if (!r) a.end[k] = upto;
        }
        if (!cols.mine) return;
        if (!l && !r) {
            store_grad<TO, E>(a, k, cols, acc);
        } else {
            float *part = a.parts + ((size_t)c * 2 + (l ? 0 : 1)) * a.dpad + cols.at;
#pragma unroll
            for (int e = 0; e < E; ++e) part[e] = acc[e];
        }
    });
}

// Blocks [0, chunks * slabs): the run that begins in the chunk and goes on behind it, if there is one: its parts summed in a
// fixed order (each group of lanes a consecutive share of them, the shares in order).  The other blocks: rows no index names,
// and the counts.
template <class TO, int E>
__global__ void __launch_bounds__(GRAD_THREADS) k_grad_join(const GradArgs a, uint32_t join_blocks)
{
    __shared__ float share[GRAD_THREADS * E];
    const uint32_t gsize = 1u << a.log2g, gl = threadIdx.x & (gsize - 1), gi = threadIdx.x >> a.log2g, groups = GRAD_THREADS >> a.log2g;
    if (blockIdx.x < join_blocks) {
        const uint32_t c = blockIdx.x / a.slabs, slab = blockIdx.x % a.slabs;
        const uint32_t p1 = min(a.N, c * a.chunk + a.chunk);
        if (p1 >= a.N) return;
        const uint32_t k = a.keys[p1 - 1];
        if (k >= a.K || a.keys[p1] != k || a.start[k] < c * a.chunk) return;
        const uint32_t more = (a.end[k] - 1) / a.chunk - c;                        // chunks behind this one that the run reaches
        const Columns<E> cols((slab * gsize + gl) * E, a.D);
        const uint32_t per = (more + groups - 1) / groups;
        float acc[E];
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.0f;
        if (cols.mine) {
            const uint32_t lo = gi * per, hi = min(more, lo + per);
#pragma unroll 8
            for (uint32_t j = lo; j < hi; ++j) {
                const float *part = a.parts + (size_t)(c + 1 + j) * 2 * a.dpad + cols.at;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += part[e];
            }
        }
#pragma unroll
        for (int e = 0; e < E; ++e) share[(gi * gsize + gl) * E + e] = acc[e];
        __syncthreads();
        if (gi != 0 || !cols.mine) return;
        const float *tail = a.parts + ((size_t)c * 2 + 1) * a.dpad + cols.at;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = tail[e];
        for (uint32_t g = 0; g < groups && g * per < more; ++g)
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += share[(g * gsize + gl) * E + e];
        store_grad<TO, E>(a, k, cols, acc);
        return;
    }
    const uint64_t lanes = (uint64_t)(gridDim.x - join_blocks) * groups;
    for (uint64_t k = (uint64_t)(blockIdx.x - join_blocks) * groups + gi; k < a.K; k += lanes) {
        const uint32_t s = a.start[k];
        if (a.counts && gl == 0) a.counts[k] = s == NONE ? 0 : a.end[k] - s;
        if (s != NONE || a.accumulate || a.cleared) continue;
        for (uint32_t col = gl * E; col < a.D; col += gsize * E) store_zeros<TO, E>(a, k, Columns<E>(col, a.D));
    }
}

// ---------------------------------------------------------------------------------------------- all in one launch
// For few rows and a table that is not large: every workgroup sorts all indices for itself (a few us, instead of two more launches
// with their partial sums in memory between them) and then does one column slab of one part of the table.
constexpr uint32_t SINGLE_ROWS = 8192;                              // indices
constexpr uint64_t SINGLE_BYTES = 32u << 20;                        // of the table
constexpr uint32_t SINGLE_PART = 32768;                             // rows of a part

// The first place in the sorted keys[0 .. n) that is not below k
__device__ __forceinline__ uint32_t lower_place(const uint32_t *keys, uint32_t n, uint32_t k)
{
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
        const uint32_t m = (lo + hi) / 2;
        if (keys[m] < k)
            lo = m + 1;
        else
            hi = m;
    }
    return lo;
}

template <class T, class TO, int E, int THREADS, int ITEMS>
__global__ void __launch_bounds__(THREADS) k_grad_single(const GradArgs a, const uint32_t *idx, int key_bits, uint32_t parts)
{
    constexpr int WAVES = THREADS / 64;
    constexpr uint32_t TILE = THREADS * ITEMS;
    __shared__ uint32_t lkey[TILE], lrow[TILE], present[SINGLE_PART / 32];
    __shared__ __attribute__((aligned(4))) uint16_t count[WAVES << SMALL_MAX_BITS];
    __shared__ uint32_t first[1 << SMALL_MAX_BITS], tmp[WAVES];
    __shared__ float part[2][THREADS * E];                           // head and tail of every group of lanes
    const uint32_t slab = blockIdx.x % a.slabs, which = blockIdx.x / a.slabs;
    const uint32_t k0 = (uint32_t)((uint64_t)a.K * which / parts), k1 = (uint32_t)((uint64_t)a.K * (which + 1) / parts);
    SortArgs q{};
    q.idx = idx;
    q.N = a.N;
    q.K = a.K;
    for (uint32_t b = threadIdx.x; b < (k1 - k0 + 31) / 32; b += THREADS) present[b] = 0;
    sort_in_lds<THREADS, ITEMS>(q, key_bits, lkey, lrow, count, first, tmp);

    const uint32_t lo = lower_place(lkey, a.N, k0), hi = lower_place(lkey, a.N, k1);
    const uint32_t gsize = 1u << a.log2g, gl = threadIdx.x & (gsize - 1), g = threadIdx.x >> a.log2g, groups = THREADS >> a.log2g;
    const Columns<E> cols((slab * gsize + gl) * E, a.D);
    const bool mine = cols.mine;
    const uint32_t per = (hi - lo + groups - 1) / groups;
    const uint32_t p0 = min(hi, lo + g * per), p1 = min(hi, p0 + per);
    for (uint32_t p = lo + threadIdx.x; p < hi; p += THREADS) {
        const uint32_t k = lkey[p];
        atomicOr(&present[(k - k0) / 32], 1u << ((k - k0) % 32));
        if (a.counts && slab == 0 && (p == 0 || lkey[p - 1] != k)) a.counts[k] = lower_place(lkey, a.N, k + 1) - p;
    }
    if (p0 < p1) {
        const bool left = p0 > 0 && lkey[p0 - 1] == lkey[p0];
        const uint32_t behind = p1 < a.N ? lkey[p1] : NONE;
        sum_runs<T, E>(lkey, lrow, p0, p1, a.K, (const T *)a.dY + (cols.mine ? cols.at : 0), a.ldy, [&](uint32_t k, uint32_t from, uint32_t upto, const float (&acc)[E]) {
            const bool l = from == p0 && left, r = upto == p1 && behind == k;
            if (!l && !r) {
                if (mine) store_grad<TO, E>(a, k, cols, acc);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) part[l ? 0 : 1][threadIdx.x * E + e] = acc[e];
            }
        });
    }
    __syncthreads();
    // the run that begins among this group's places and goes on behind them
    if (p0 < p1 && p1 < hi && mine) {
        const uint32_t k = lkey[p1 - 1];
        if (lkey[p1] == k && !(p0 > 0 && lkey[p0 - 1] == k && lkey[p0] == k)) {
            float acc[E];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = part[1][threadIdx.x * E + e];
            uint32_t at = p1;
            for (uint32_t h = 1; at < hi && lkey[at] == k; ++h, at += per)
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += part[0][(threadIdx.x + h * gsize) * E + e];
            store_grad<TO, E>(a, k, cols, acc);
        }
    }
    for (uint32_t k = k0 + g; k < k1; k += groups) {
        if ((present[(k - k0) / 32] >> ((k - k0) % 32)) & 1) continue;
        if (a.counts && slab == 0 && gl == 0) a.counts[k] = 0;
        if (!a.accumulate && mine) store_zeros<TO, E>(a, k, cols);
    }
}

// ---------------------------------------------------------------------------------------------- plan of one gradient call
struct GradPlan {
    uint32_t tile, tiles, chunk, chunks, dpad;
    int key_bits, passes, bits;
    bool small;
    size_t keys[2], rows[2], hist, total, start, end, parts, bytes;      // offsets into the workspace
};

GradPlan plan_gradient(uint64_t N, uint32_t K, uint32_t D)
{
    GradPlan p{};
    p.small = N <= SMALL_TILE;
    p.key_bits = 32 - __builtin_clz(K);                                   // indices 0 .. K - 1, and K for the rows without a place
    p.passes = (p.key_bits + SORT_MAX_BITS - 1) / SORT_MAX_BITS;
    p.bits = (p.key_bits + p.passes - 1) / p.passes;
    // small tiles spread a sort over the card; of very many rows they would make the table of counts large
    p.tile = N <= (4u << 20) ? 2048 : 8192;
    p.tiles = (uint32_t)((N + p.tile - 1) / p.tile);
    // chunks: enough groups of lanes to fill the card (8192 waves) however the runs lie, at least 8 rows each, so that the
    // parts of runs that cross chunk borders stay a small share of the rows read
    const uint64_t units = N * ((D + 255) / 256);
    p.chunk = (uint32_t)std::min<uint64_t>(std::max<uint64_t>((units + 8191) / 8192, 8), 4096);
    p.chunks = (uint32_t)((N + p.chunk - 1) / p.chunk);
    p.dpad = (D + 7) / 8 * 8;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t o = at;
        at += (bytes + 255) / 256 * 256;
        return o;
    };
    for (int j = 0; j < 2; ++j) {
        const bool used = j == 0 || (!p.small && p.passes > 1);
        p.keys[j] = take(used ? N * 4 : 0);
        p.rows[j] = take(used ? N * 4 : 0);
    }
    p.hist = take(p.small ? 0 : ((size_t)p.tiles << p.bits) * 4);
    p.total = take(p.small ? 0 : (size_t)4 << p.bits);
    p.start = take((size_t)K * 4);
    p.end = take((size_t)K * 4);
    p.parts = take((size_t)p.chunks * 2 * p.dpad * 4);
    p.bytes = at;
    return p;
}

template <class T, class TO, int E>
hipError_t run_reduce(const GradArgs &a, const uint32_t *single, uint32_t parts, int key_bits, hipStream_t s)
{
    if (single) {
        if (a.N <= 1024)
            hipLaunchKernelGGL((k_grad_single<T, TO, E, 256, 4>), dim3(a.slabs * parts), dim3(256), 0, s, a, single, key_bits, parts);
        else if (a.N <= 4096)
            hipLaunchKernelGGL((k_grad_single<T, TO, E, 1024, 4>), dim3(a.slabs * parts), dim3(1024), 0, s, a, single, key_bits, parts);
        else
            hipLaunchKernelGGL((k_grad_single<T, TO, E, 1024, 8>), dim3(a.slabs * parts), dim3(1024), 0, s, a, single, key_bits, parts);
        return hipGetLastError();
    }
    const uint32_t groups = GRAD_THREADS >> a.log2g;
    if (a.N) {
        const uint64_t blocks = ((uint64_t)a.chunks * a.slabs + groups - 1) / groups;
        hipLaunchKernelGGL((k_grad_reduce<T, TO, E>), dim3((uint32_t)blocks), dim3(GRAD_THREADS), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    const uint32_t join_blocks = a.N ? a.chunks * a.slabs : 0;
    const uint32_t fill_blocks = std::min<uint32_t>((a.K + groups - 1) / groups, 8192);
    hipLaunchKernelGGL((k_grad_join<TO, E>), dim3(join_blocks + fill_blocks), dim3(GRAD_THREADS), 0, s, a, join_blocks);
    return hipGetLastError();
}

template <class T, class TO>
hipError_t run_reduce_width(const GradArgs &a, int e, const uint32_t *single, uint32_t parts, int key_bits, hipStream_t s)
{
    constexpr int E = 16 / (int)sizeof(TO);
    return e == E ? run_reduce<T, TO, E>(a, single, parts, key_bits, s) : run_reduce<T, TO, 1>(a, single, parts, key_bits, s);
}

size_t elem_bytes(int dtype) { return dtype == VQHIP_F32 ? 4 : 2; }

}  // namespace

hipError_t launch_lookup(const void *dT, int dtype, uint64_t ldt, uint32_t K, uint32_t D, const uint32_t *didx, uint64_t N, float scale, void *dY,
                         uint64_t ldy, hipStream_t s)
{
    const LookupArgs a{dT, ldt, didx, N, K, D, scale, dY, ldy, 0};
    if (dtype == VQHIP_F32) return run_lookup<float>(a, s);
    if (dtype == VQHIP_BF16) return run_lookup<__bf16>(a, s);
    return run_lookup<_Float16>(a, s);
}

size_t lookup_gradient_workspace(uint64_t N, uint32_t K, uint32_t D) { return plan_gradient(N, K, D).bytes; }

hipError_t launch_lookup_gradient(const void *dG, int dtype, uint64_t ldg, const uint32_t *didx, uint64_t N, float scale, uint32_t K, uint32_t D, void *dT,
                                  int out_dtype, uint64_t ldt, bool accumulate, uint32_t *dcounts, void *dwork, hipStream_t s)
{
    const GradPlan p = plan_gradient(N, K, D);
    char *w = (char *)dwork;
    auto at = [&](size_t o) { return (uint32_t *)(w + o); };
    const size_t bi = elem_bytes(dtype), bo = elem_bytes(out_dtype);
    GradArgs a{dG, ldg, at(p.keys[0]), at(p.rows[0]), (uint32_t)N, K, D, scale, dT, ldt, accumulate ? 1 : 0, 0, at(p.start), at(p.end), dcounts,
               (float *)(w + p.parts), p.dpad, p.chunk, p.chunks, 0, 0};
    const int wide = (int)(16 / bo);
    int n = 0;                                                              // elements a lane takes at once
    uint32_t parts = 0;
    bool one = false;
    auto shape = [&](int elements) {
        n = elements;
        const uint32_t steps = (D + n - 1) / n;
        a.log2g = 0;
        while ((1u << a.log2g) < steps && a.log2g < 6) ++a.log2g;
        a.slabs = (steps + (1u << a.log2g) - 1) >> a.log2g;
        // One launch: about one workgroup a CU, each with 64 rows of the table or more and no more than 128 KiB to read, which is a few
        // us.  3001 rows of 515 over 997: 23 us in three launches, 17 in one; 8000 of 256 over 30000 32 and 25.
        parts = std::max(std::max(1u, std::min(256 / std::min(a.slabs, 256u), (K + 63) / 64)), (K + SINGLE_PART - 1) / SINGLE_PART);
        one = N > 0 && N <= SINGLE_ROWS && (uint64_t)K * D * bo <= SINGLE_BYTES && N * D * bi <= (uint64_t)a.slabs * parts * (128u << 10);
    };
    // 16 bytes of the table, or one element where they do not divide the row and it is short or the launch the only one: a row's
    // last lane then stores by elements.  us by 16 bytes / by one: 300000 rows of 203 over 5000 bf16 70 / 108, 50000 of 1001 over
    // 1000 f32 63 / 90; 1000000 of 5 over 100 f32 76 / 56, 3001 of 515 over 997 f16 (one launch) 20.5 / 16.5
    shape(D % wide == 0 ? wide : 1);
    if (!one && D >= 32) shape(wide);
    const uint32_t *single = one ? didx : nullptr;
    // Rows no index names are cleared beside the sort, whose few workgroups leave the memory idle, where clearing takes longer
    // than telling the rows apart beforehand (two small launches; 16384 rows of 4096 over 65536: 334 us without, 270 with).
    const bool early = N > 0 && !accumulate && (uint64_t)K * D * bo > SINGLE_BYTES;
    SortArgs q{didx, nullptr, nullptr, at(p.keys[0]), at(p.rows[0]), at(p.hist), at(p.total), at(p.start), nullptr, (uint32_t)N, K, p.tiles, 0, p.bits, 0, {}};
    const bool words = (((uint64_t)(uintptr_t)dT | ldt * bo | (uint64_t)D * bo) & 3) == 0;
    ZeroArgs zero{(char *)dT, ldt * bo, (uint64_t)D * bo, words, 0, 0};
    while (((words ? 16ull : 2ull) << zero.log2g) < zero.bytes && zero.log2g < 8) ++zero.log2g;
    // A row to a workgroup where rows are 2 KiB or more, and the next one from another: 1000 rows of 512 over 131072 54 us, by 4096
    // workgroups 65; short rows by 4096: 5000 of 64 over 1000000 68 us, by 65536 133.
    const uint64_t shares = zero.bytes >= 2048 ? std::min<uint64_t>((((uint64_t)K << zero.log2g) + 255) / 256, 65536) : std::min<uint64_t>((K + 15) / 16, 4096);
    zero.blocks = early ? (uint32_t)shares : 0;
    const uint32_t few = std::min<uint32_t>((K + 255) / 256, 4096);
    a.cleared = early ? 1 : 0;
    if (one) {
        // (sorts for itself)
    } else if (N == 0) {
        hipLaunchKernelGGL(k_fill_u32, dim3(few), dim3(256), 0, s, q.start, (uint64_t)K, NONE);
    } else if (p.small) {
        if (early) {
            q.mark = didx;
            hipLaunchKernelGGL(k_fill_u32, dim3(few), dim3(256), 0, s, q.start, (uint64_t)K, NONE);
            hipLaunchKernelGGL(k_mark, dim3((uint32_t)(N + 255) / 256), dim3(256), 0, s, q);
            q.zero = zero;
        }
        if (N <= 1024)
            run_sort_small<256, 4>(q, p.key_bits, s);
        else if (N <= 4096)
            run_sort_small<1024, 4>(q, p.key_bits, s);
        else
            run_sort_small<1024, 8>(q, p.key_bits, s);
    } else {
        for (int pass = 0; pass < p.passes; ++pass) {
            const int to = (p.passes - 1 - pass) & 1;                       // the last pass ends in buffer 0
            q.idx = pass == 0 ? didx : nullptr;
            q.keys_in = at(p.keys[to ^ 1]);
            q.rows_in = at(p.rows[to ^ 1]);
            q.keys = at(p.keys[to]);
            q.rows = at(p.rows[to]);
            q.shift = pass * p.bits;
            q.mark = early && pass == 0 ? didx : nullptr;
            q.zero = pass == 0 ? zero : ZeroArgs{};
            if (p.tile == 2048)
                run_sort_pass<256, 8>(q, s);
            else
                run_sort_pass<512, 16>(q, s);
        }
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (dtype == VQHIP_F32) return run_reduce_width<float, float>(a, n, single, parts, p.key_bits, s);
    if (dtype == VQHIP_BF16) return out_dtype == VQHIP_F32 ? run_reduce_width<__bf16, float>(a, n, single, parts, p.key_bits, s) : run_reduce_width<__bf16, __bf16>(a, n, single, parts, p.key_bits, s);
    return out_dtype == VQHIP_F32 ? run_reduce_width<_Float16, float>(a, n, single, parts, p.key_bits, s) : run_reduce_width<_Float16, _Float16>(a, n, single, parts, p.key_bits, s);
}

}  // namespace vq
