// Which key blocks a query block attends to: block means (sfast_hip_block_means) and the choice by their products (sfast_hip_block_topk).
//
// Sums and products run in 64 bits: a choice stands on which of two scores is larger. Products of two fp32 means are exact then, and sums lose
// 2^-53 a step, so the order of the additions (which differs between the score kernels below) can decide only between scores that agree to about
// 2^-53 of their terms' magnitudes. Within a call all blocks' scores are summed in one order: equal means give equal scores.
#include "common.h"
#include <math.h>

namespace sfast {

namespace {

// ---- block means ------------------------------------------------------------------------------------------------------------------------
// Bound by reading x. A workgroup owns one block and 32 runs of V elements (512 bytes of a contiguous token); 8 groups of threads share its
// rows, each thread keeps several 16-byte loads in flight, and the groups' sums are added in LDS in a fixed order.
// (57600 x 10 rows of 64 in f16: 13.4 us, 5.6 TB/s; 4 x 8191 x 8 rows of 128, ragged: 9.7 us, of which 2 are the launch.)
struct MeansArgs {
    const void *x;
    const int32_t *lengths;
    float *out;
    int B, S, H, D, block, n, runs;  // runs = H * D / V
    int64_t xs[3];
};

template <typename T, int V> struct alignas(sizeof(T) * V) MeanVec {
    T e[V];
};

template <typename T, int V> __global__ void __launch_bounds__(256) block_means_kernel(const MeansArgs a) {
    __shared__ double part[8][32 * V];
    const int tid = threadIdx.x, col = tid & 31, grp = tid >> 5;
    const int cols = (a.runs + 31) / 32;
    const int unit = (int)(blockIdx.x / (uint32_t)cols);
    const int run = (int)(blockIdx.x - (uint32_t)unit * cols) * 32 + col;
    const int b = unit / a.n, j = unit - b * a.n;
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
    const int rows = min(max(len - j * a.block, 0), a.block);  // (j * block <= S)
    double sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0;
    const int e = run * V;  // H * D has 31 bits
    const int h = e / a.D, d = e - h * a.D;
    if (run < a.runs) {
        const T *x = (const T *)a.x + b * a.xs[0] + (int64_t)j * a.block * a.xs[1] + h * a.xs[2] + d;
        int r = grp;
        for (; r + 24 < rows; r += 32) {
            MeanVec<T, V> v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const MeanVec<T, V> *>(x + (int64_t)(r + 8 * i) * a.xs[1]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int k = 0; k < V; ++k) sum[k] += (double)(float)v[i].e[k];
        }
        for (; r < rows; r += 8) {
            const MeanVec<T, V> v = *reinterpret_cast<const MeanVec<T, V> *>(x + (int64_t)r * a.xs[1]);
#pragma unroll
            for (int k = 0; k < V; ++k) sum[k] += (double)(float)v.e[k];
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) part[grp][i * 32 + col] = sum[i];
    __syncthreads();
    // output element i of run c: the workgroup's 32 * V elements are neighbours in memory
    const int first = (int)(blockIdx.x - (uint32_t)unit * cols) * 32 * V;
    for (int i = tid; i < 32 * V; i += 256) {
        const int c = i / V, k = i - c * V;
        if (first + i >= a.H * a.D) continue;
        double s = 0.0;
#pragma unroll
        for (int g = 0; g < 8; ++g) s += part[g][k * 32 + c];
        a.out[(int64_t)unit * a.H * a.D + first + i] = rows > 0 ? (float)(s / rows) : 0.f;
    }
}

// ---- scores -------------------------------------------------------------------------------------------------------------------------------
// 64-bit MFMAs (16x16x4) on operands read from memory as fp32: a lane reads four consecutive head-dim elements of its row at a time, and the
// four products of such a group take them in the order the lanes hold them -- any order of the head dim will do as long as both operands
// share it. A wave owns 16 x MI query blocks and 16 x NJ key blocks; a workgroup's four waves share the query blocks.
// 450 x 900 blocks of 10 heads of 64 take 22 us: the matrix pipe is busy for 7.3 of them (64 cycles an instruction, all waves in step), the
// rest is the first loads' way from memory, the keys' way out (32 MB) and the ends of the grid; without the products it still takes 20 us,
// without the stores 19.
typedef double f64x4 __attribute__((ext_vector_type(4)));

struct TopkArgs {
    const float *qm, *km;
    const int32_t *klen;
    uint32_t *high, *low;  // [B, Hk, nQ, nK]: the halves of the scores' keys
    int32_t *out;     // [B, Hk, nQ, topk]
    int B, nQ, nK, H, Hk, G, D, topk, bk;
};

__device__ __forceinline__ int topk_count(const TopkArgs &a, int b) {
    if (!a.klen) return a.nK;
    const uint32_t n = ((uint32_t)max(a.klen[b], 0) + (uint32_t)(a.bk - 1)) / (uint32_t)a.bk;
    return (int)min(n, (uint32_t)a.nK);
}

// a score as a 64-bit key whose order is the score's (NaN above all, -0 and 0 alike, 0 is no key)
__device__ __forceinline__ uint64_t topk_key(double s) {
    s += 0.0;  // -0 and 0 are one score
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    if (s != s) return ~0ull;
    return (u >> 63) ? ~u : (u | (1ull << 63));
}

// the upper halves decide nearly always: they are kept apart, and the lower ones are read only where they do not
__device__ __forceinline__ void put_key(const TopkArgs &a, int64_t at, double s) {
    const uint64_t k = topk_key(s);
    a.high[at] = (uint32_t)(k >> 32);
    a.low[at] = (uint32_t)k;
}

template <int MI, int NJ> __global__ void __launch_bounds__(256, 4) block_score_kernel(const TopkArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l15 = lane & 15, l4 = lane >> 4;
    const int pair = blockIdx.z, hk = pair % a.Hk, b = pair / a.Hk;
    const int i0 = blockIdx.y * 16 * MI, j0 = (blockIdx.x * 4 + wave) * 16 * NJ;
    const int count = topk_count(a, b);
    if (j0 >= count) return;
    f64x4 acc[MI][NJ];
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int y = 0; y < NJ; ++y) acc[x][y] = f64x4{0.0, 0.0, 0.0, 0.0};
    // rows outside read row 0: their products land in results that nobody stores
    const float *kp[NJ], *qp[MI];
#pragma unroll
    for (int y = 0; y < NJ; ++y) {
        const int j = j0 + 16 * y + l15;
        kp[y] = a.km + (((int64_t)b * a.nK + (j < count ? j : 0)) * a.Hk + hk) * a.D + 4 * l4;
    }
#pragma unroll
    for (int x = 0; x < MI; ++x) {
        const int i = i0 + 16 * x + l15;
        qp[x] = a.qm + (((int64_t)b * a.nQ + (i < a.nQ ? i : 0)) * a.H + hk * a.G) * a.D + 4 * l4;
    }
    f32x4 k[NJ], q[MI];
    const auto load = [&](int d0) __attribute__((always_inline)) {
        const bool in = d0 + 4 * l4 < a.D;
#pragma unroll
        for (int y = 0; y < NJ; ++y) k[y] = in ? *reinterpret_cast<const f32x4 *>(kp[y] + d0) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < MI; ++x) q[x] = in ? *reinterpret_cast<const f32x4 *>(qp[x] + d0) : f32x4{0.f, 0.f, 0.f, 0.f};
    };
    load(0);
    for (int d0 = 0; d0 < a.D; d0 += 16) {
        double kd[NJ][4], qd[MI][4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int y = 0; y < NJ; ++y) kd[y][t] = (double)k[y][t];
#pragma unroll
            for (int x = 0; x < MI; ++x) qd[x][t] = (double)q[x][t];
        }
        const bool in = d0 + 4 * l4 < a.D;
        for (int g = 1; g < a.G; ++g)
#pragma unroll
            for (int x = 0; x < MI; ++x) {
                const f32x4 v = in ? *reinterpret_cast<const f32x4 *>(qp[x] + (int64_t)g * a.D + d0) : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int t = 0; t < 4; ++t) qd[x][t] += (double)v[t];
            }
        if (d0 + 16 < a.D) load(d0 + 16);  // under the products of this group
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int x = 0; x < MI; ++x)
#pragma unroll
                for (int y = 0; y < NJ; ++y) acc[x][y] = __builtin_amdgcn_mfma_f64_16x16x4f64(qd[x][t], kd[y][t], acc[x][y], 0, 0, 0);
    }
    // result register r of a lane: query block 4 r + lane / 16, key block lane % 16
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 16 * x + 4 * r + l4;
            if (i >= a.nQ) continue;
            const int64_t row = ((int64_t)pair * a.nQ + i) * a.nK;
#pragma unroll
            for (int y = 0; y < NJ; ++y) {
                const int j = j0 + 16 * y + l15;
                if (j < count) put_key(a, row + j, acc[x][y][r]);
            }
        }
}

// One or a few query blocks (a token): bound by reading the key means, not worth a matrix tile. Eight lanes share a key block (128 bytes of its
// row at a time), a wave holds 32 key blocks in registers, and the query sums wait in LDS as 64-bit numbers.
constexpr int SCORE_FEW = 4, SCORE_FEW_D = 128;
__global__ void __launch_bounds__(256) block_score_few_kernel(const TopkArgs a) {
    __shared__ __attribute__((aligned(16))) double qs[SCORE_FEW][SCORE_FEW_D];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l7 = lane & 7, l8 = lane >> 3;
    const int pair = blockIdx.z, hk = pair % a.Hk, b = pair / a.Hk;
    const int count = topk_count(a, b);
    const int j0 = (blockIdx.x * 4 + wave) * 32;
    if ((int)blockIdx.x * 128 >= count) return;
    f32x4 k[4][4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
        const int j = j0 + 8 * y + l8;
        const float *row = a.km + (((int64_t)b * a.nK + (j < count ? j : 0)) * a.Hk + hk) * a.D;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = 32 * c + 4 * l7;
            k[y][c] = d < a.D ? *reinterpret_cast<const f32x4 *>(row + d) : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    for (int e = tid; e < a.nQ * a.D; e += 256) {
        const int i = e / a.D, d = e - i * a.D;
        const float *q = a.qm + (((int64_t)b * a.nQ + i) * a.H + hk * a.G) * a.D + d;
        double s = 0.0;
        for (int g = 0; g < a.G; ++g) s += (double)q[(int64_t)g * a.D];
        qs[i][d] = s;
    }
    __syncthreads();
    for (int i = 0; i < a.nQ; ++i) {
        double s[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = 32 * c + 4 * l7;
            if (d < a.D) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const double q = qs[i][d + t];
#pragma unroll
                    for (int y = 0; y < 4; ++y) s[y] = fma(q, (double)k[y][c][t], s[y]);
                }
            }
        }
        const int64_t row = ((int64_t)pair * a.nQ + i) * a.nK;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
#pragma unroll
            for (int off = 4; off >= 1; off >>= 1) s[y] += __shfl_xor(s[y], off, 64);
            const int j = j0 + 8 * y + l8;
            if (l7 == 0 && j < count) put_key(a, row + j, s[y]);
        }
    }
}

// ---- the topk best of a row ---------------------------------------------------------------------------------------------------------------
// WAVES waves hold a row's scores in registers as order-preserving 64-bit keys (0 = not there) and find the topk-th largest bit by bit from
// the top: a bit stays set while at least topk keys reach the candidate, and the search ends as soon as exactly topk do. It starts below the
// bits that all keys in question share and looks at the upper 31 bits first: those settle all but near-ties, for two instructions a key and bit (a
// comparison's mask would cost wait states on top). Keys equal to the threshold are taken in the order of their index.
// 4500 rows of 900 take 12 us: about 12 bits of 52 instructions each, and the keys' way in; 64 rows of 2048 (four waves) 8 us.
// sum / maximum over a wave, the same in every lane (row shifts by 1, 2, 4, 8, then across the rows of 16: lane 63 holds the result)
template <int CTRL> __device__ __forceinline__ uint32_t topk_dpp(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ uint32_t topk_wave_sum(uint32_t v) {
    v += topk_dpp<0x111>(v), v += topk_dpp<0x112>(v), v += topk_dpp<0x114>(v), v += topk_dpp<0x118>(v);
    v += topk_dpp<0x142>(v), v += topk_dpp<0x143>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t topk_wave_or(uint32_t v) {
    v |= topk_dpp<0x111>(v), v |= topk_dpp<0x112>(v), v |= topk_dpp<0x114>(v), v |= topk_dpp<0x118>(v);
    v |= topk_dpp<0x142>(v), v |= topk_dpp<0x143>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t topk_wave_max(uint32_t v) {
    v = max(v, topk_dpp<0x111>(v)), v = max(v, topk_dpp<0x112>(v)), v = max(v, topk_dpp<0x114>(v)), v = max(v, topk_dpp<0x118>(v));
    v = max(v, topk_dpp<0x142>(v)), v = max(v, topk_dpp<0x143>(v));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}

template <int WAVES, int NPL> __global__ void __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) block_topk_kernel(const TopkArgs a, int n_rows) {
    __shared__ uint32_t sums[2][WAVES];
    __shared__ int above_s[WAVES], equal_s[WAVES];
    const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : threadIdx.x >> 6;
    const int row_id = (int)(WAVES == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x);  // (less than 2^26 rows)
    if (row_id >= n_rows) return;
    const int64_t row = row_id;
    const int count = topk_count(a, row_id / a.nQ / a.Hk);
    const int j0 = wave * 64 * NPL + lane;
    uint32_t up[NPL];  // the upper 31 bits of the keys
#pragma unroll
    for (int n = 0; n < NPL; ++n) up[n] = a.high[row * a.nK + min(j0 + 64 * n, a.nK - 1)];  // all in flight, whether they count or not
#pragma unroll
    for (int n = 0; n < NPL; ++n) up[n] = j0 + 64 * n < count ? up[n] >> 1 : 0u;
    int turn = 0;
    const auto over_waves = [&](uint32_t mine, bool most, bool any = false) __attribute__((always_inline)) -> uint32_t {
        if (WAVES == 1) return mine;
        turn ^= 1;
        if (lane == 0) sums[turn][wave] = mine;
        __syncthreads();
        uint32_t s = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s = any ? s | sums[turn][w] : most ? max(s, sums[turn][w]) : s + sums[turn][w];
        return s;
    };
    int32_t *out = a.out + row * a.topk;
    for (int i = count + (WAVES == 1 ? lane : (int)threadIdx.x); i < a.topk; i += WAVES == 1 ? 64 : WAVES * 64) out[i] = -1;
    const uint64_t below = (1ull << lane) - 1;
    uint32_t edge_up = 0;
    bool exact = count <= a.topk;  // everything that is there is chosen (and is not 0 in its upper bits: only keys that are not there are)
    if (!exact) {
        const uint32_t want = (uint32_t)a.topk;
        uint32_t big = 0, small = 0;  // largest upper part, largest complement of one (of a key that is there)
#pragma unroll
        for (int n = 0; n < NPL; ++n) {
            big = max(big, up[n]);
            small = max(small, j0 + 64 * n < count ? ~up[n] : 0u);
        }
        big = over_waves(topk_wave_max(big), true);
        small = ~over_waves(topk_wave_max(small), true);
        const auto reach_up = [&](uint32_t cand) __attribute__((always_inline)) -> uint32_t {
            // 31-bit numbers: the sign of the difference tells which is less; the signs are collected and counted at the end
            uint32_t less = 0;
#pragma unroll
            for (int n = 0; n < NPL; ++n) less = __builtin_amdgcn_alignbit(less, up[n] - cand, 31);
            return (uint32_t)(64 * NPL * WAVES) - over_waves(topk_wave_sum(__builtin_popcount(less)), false);
        };
        // the topk-th key is mostly within two powers of two of the largest (19 bits of the upper part are its fraction's): one look there
        // saves the search through the exponents
        const uint32_t probe = big - (2u << 19);
        if (big > (2u << 19) && probe > small) {
            const uint32_t have = reach_up(probe);
            exact = have == want;
            if (have >= want)
                small = edge_up = probe;
            else
                big = probe - 1;
        }
        const uint32_t differ = big ^ small;
        const int top = differ ? 31 - __builtin_clz(differ) : -1;
        if (!exact) edge_up = top < 0 ? big : big & ~((2u << top) - 1u);
        for (int bit = top; bit >= 0 && !exact; --bit) {
            const uint32_t cand = edge_up | (1u << bit), have = reach_up(cand);
            if (have >= want) edge_up = cand;
            exact = have == want;
        }
    }
    if (exact) {
        // positions: chosen keys of earlier waves, earlier registers, lower lanes
        const uint32_t from = max(edge_up, 1u);
        int at = 0;
        if (WAVES > 1) {
            int mine = 0;
#pragma unroll
            for (int n = 0; n < NPL; ++n) mine += __popcll(__ballot(up[n] >= from));
            if (lane == 0) above_s[wave] = mine;
            __syncthreads();
            for (int w = 0; w < wave; ++w) at += above_s[w];
        }
#pragma unroll
        for (int n = 0; n < NPL; ++n) {
            const bool take = up[n] >= from;
            const uint64_t some = __ballot(take);
            if (take) out[at + __popcll(some & below)] = j0 + 64 * n;
            at += __popcll(some);
        }
        return;
    }
    // Scores that agree in their upper 31 bits stand at the border: the topk-th key has the upper bits edge_up, the other 33 decide, then the
    // index. The keys are read again as they are needed, and the search starts below the bits that the ones at the border share (equal scores
    // need none).
    const uint32_t want = (uint32_t)a.topk;
    const auto key = [&](int n) __attribute__((always_inline)) -> uint64_t {
        const int64_t at = row * a.nK + min(j0 + 64 * n, a.nK - 1);
        return j0 + 64 * n < count ? ((uint64_t)a.high[at] << 32) | a.low[at] : 0ull;
    };
    const auto reach = [&](uint64_t from) __attribute__((always_inline)) -> uint32_t {
        uint32_t mine = 0;
#pragma unroll 4
        for (int n = 0; n < NPL; ++n) mine += key(n) >= from ? 1u : 0u;
        return over_waves(topk_wave_sum(mine), false);
    };
    uint32_t share_hi = 0, share_lo = 0, miss_hi = 0, miss_lo = 0;
#pragma unroll 4
    for (int n = 0; n < NPL; ++n) {
        const uint64_t k = key(n);
        if ((uint32_t)(k >> 33) == edge_up && k != 0) {
            share_hi |= (uint32_t)(k >> 32), share_lo |= (uint32_t)k;       // bits that some key has
            miss_hi |= ~(uint32_t)(k >> 32), miss_lo |= ~(uint32_t)k;       // bits that some key lacks
        }
    }
    share_hi = over_waves(topk_wave_or(share_hi), true, true), share_lo = over_waves(topk_wave_or(share_lo), true, true);
    miss_hi = over_waves(topk_wave_or(miss_hi), true, true), miss_lo = over_waves(topk_wave_or(miss_lo), true, true);
    const uint64_t shared = ((uint64_t)share_hi << 32) | share_lo, differ = shared & (((uint64_t)miss_hi << 32) | miss_lo);
    const int top = differ ? 63 - __builtin_clzll(differ) : -1;  // below 33
    uint64_t edge = top < 0 ? shared : shared & ~((2ull << top) - 1ull);
    bool all = false;  // exactly topk keys reach the edge
    for (int bit = top; bit >= 0 && !all; --bit) {
        const uint64_t cand = edge | (1ull << bit);
        const uint32_t have = reach(cand);
        if (have >= want) edge = cand;
        all = have == want;
    }
    const int limit = all ? 0x7fffffff : (int)(want - (edge == ~0ull ? 0u : reach(edge + 1)));  // how many of those at the edge
    int above0 = 0, equal0 = 0;
    if (WAVES > 1) {
        int ab = 0, eq = 0;
#pragma unroll 4
        for (int n = 0; n < NPL; ++n) {
            const uint64_t k = key(n);
            ab += __popcll(__ballot(k > edge));
            eq += __popcll(__ballot(k == edge));
        }
        if (lane == 0) above_s[wave] = ab, equal_s[wave] = eq;
        __syncthreads();
        for (int w = 0; w < wave; ++w) above0 += above_s[w], equal0 += equal_s[w];
    }
#pragma unroll 4
    for (int n = 0; n < NPL; ++n) {
        const uint64_t k = key(n), ab = __ballot(k > edge), eq = __ballot(k == edge);
        const int rank = equal0 + __popcll(eq & below);
        const bool take = k > edge || (k == edge && rank < limit);
        if (take) out[above0 + __popcll(ab & below) + min(rank, limit)] = j0 + 64 * n;
        above0 += __popcll(ab);
        equal0 += __popcll(eq);
    }
}

template <int WAVES, int NPL> int launch_topk(const TopkArgs &a, hipStream_t st) {
    const int64_t rows = (int64_t)a.B * a.Hk * a.nQ;
    const dim3 grid((unsigned)(WAVES == 1 ? ceil_div64(rows, 4) : rows));
    hipLaunchKernelGGL((block_topk_kernel<WAVES, NPL>), grid, dim3(WAVES == 1 ? 256 : WAVES * 64), 0, st, a, (int)rows);
    return check_launch("block_topk");
}

static int check_topk(const sfast_block_topk_params *p) {
    SFAST_REQUIRE(p, SFAST_ERR_INVALID, "block_topk: null argument");
    SFAST_REQUIRE(p->B > 0 && p->nQ > 0 && p->nK > 0 && p->H > 0 && p->Hk > 0 && p->D > 0 && p->topk > 0 && p->block_k > 0, SFAST_ERR_INVALID,
                  "block_topk: bad shape");
    SFAST_REQUIRE(p->H % p->Hk == 0, SFAST_ERR_INVALID, "block_topk: %d query heads are no multiple of %d key heads", p->H, p->Hk);
    SFAST_REQUIRE(p->D % 4 == 0, SFAST_ERR_UNSUPPORTED, "block_topk: head dim %d is no multiple of 4", p->D);
    SFAST_REQUIRE(p->nK <= 32768 && p->topk <= 32768, SFAST_ERR_UNSUPPORTED, "block_topk: %d of %d key blocks (up to 32768)", p->topk, p->nK);
    SFAST_REQUIRE((int64_t)p->B * p->Hk <= 65535 && p->nQ <= (1 << 20) &&
                      fits_launch((int64_t)p->B * p->Hk * p->nQ, p->nK <= 2048 ? 64 : 1024), SFAST_ERR_UNSUPPORTED, "block_topk: too many rows");
    return SFAST_OK;
}

}  // namespace

template <typename T> static int means_launch(MeansArgs &a, int run, hipStream_t st) {
    a.runs = a.H * (a.D / run);
    const int64_t blocks = (int64_t)a.B * a.n * ceil_div(a.runs, 32);
    SFAST_REQUIRE(fits_launch(blocks, 256) && (int64_t)a.H * a.D <= (1ll << 30), SFAST_ERR_UNSUPPORTED, "block_means: too many blocks");
    const dim3 grid((unsigned)blocks);
    set_kernel_name("block_means[V=%d]", run);
    constexpr int MOST = 16 / sizeof(T);
    if (run == MOST)
        hipLaunchKernelGGL((block_means_kernel<T, MOST>), grid, dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((block_means_kernel<T, 1>), grid, dim3(256), 0, st, a);
    return check_launch("block_means");
}

}  // namespace sfast

using namespace sfast;

extern "C" int sfast_hip_block_means(const void *x, const int32_t *lengths, float *out, const sfast_block_means_params *p, sfast_stream_t stream) {
    SFAST_REQUIRE(p && x && out, SFAST_ERR_INVALID, "block_means: null argument");
    SFAST_REQUIRE(p->B > 0 && p->S > 0 && p->H > 0 && p->D > 0, SFAST_ERR_INVALID, "block_means: bad shape");
    SFAST_REQUIRE(p->block >= 1 && p->block <= 1024, SFAST_ERR_INVALID, "block_means: blocks of %d rows (1 to 1024)", p->block);
    SFAST_REQUIRE(p->dtype == SFAST_F16 || p->dtype == SFAST_BF16 || p->dtype == SFAST_F32, SFAST_ERR_UNSUPPORTED, "block_means: bad dtype %d", p->dtype);
    MeansArgs a{};
    a.x = x, a.lengths = lengths, a.out = out;
    a.B = p->B, a.S = p->S, a.H = p->H, a.D = p->D, a.block = p->block, a.n = (int)ceil_div64(p->S, p->block);
    // 16-byte loads where head dim, strides and address allow them, else element by element
    const int es = (int)dtype_bytes(p->dtype);
    int run = 16 / es;
    bool vec = p->D % run == 0 && aligned16(x);
    for (int i = 0; i < 3; ++i) {
        a.xs[i] = p->xs[i];
        vec = vec && p->xs[i] % run == 0;
    }
    if (!vec) run = 1;
    hipStream_t st = (hipStream_t)stream;
    if (p->dtype == SFAST_F16) return means_launch<f16>(a, run, st);
    if (p->dtype == SFAST_BF16) return means_launch<bf16>(a, run, st);
    return means_launch<float>(a, run, st);
}

extern "C" size_t sfast_hip_block_topk_workspace_bytes(const sfast_block_topk_params *p) {
    if (check_topk(p) != SFAST_OK) return 0;
    return (size_t)p->B * p->Hk * p->nQ * p->nK * 8;
}

extern "C" int sfast_hip_block_topk(const float *qm, const float *km, const int32_t *key_lengths, int32_t *out, const sfast_block_topk_params *p,
                                    void *workspace, size_t workspace_bytes, sfast_stream_t stream) {
    SFAST_REQUIRE(qm && km && out, SFAST_ERR_INVALID, "block_topk: null argument");
    int rc = check_topk(p);
    if (rc != SFAST_OK) return rc;
    SFAST_REQUIRE(aligned16(qm) && aligned16(km), SFAST_ERR_UNSUPPORTED, "block_topk: means must be 16-byte aligned");
    SFAST_REQUIRE(workspace && aligned8(workspace) && workspace_bytes >= sfast_hip_block_topk_workspace_bytes(p), SFAST_ERR_WORKSPACE,
                  "block_topk: workspace too small");
    TopkArgs a{};
    a.qm = qm, a.km = km, a.klen = key_lengths, a.out = out, a.high = (uint32_t *)workspace;
    a.low = a.high + (size_t)p->B * p->Hk * p->nQ * p->nK;
    a.B = p->B, a.nQ = p->nQ, a.nK = p->nK, a.H = p->H, a.Hk = p->Hk, a.G = p->H / p->Hk, a.D = p->D, a.topk = p->topk, a.bk = p->block_k;
    hipStream_t st = (hipStream_t)stream;
    const unsigned pairs = (unsigned)(p->B * p->Hk);
    // a few query blocks (a token has one): the key means are read once, no matrix tile; up to 16: one row tile, the four waves side by side
    // along the key blocks
    if (p->nQ <= SCORE_FEW && p->D <= SCORE_FEW_D)
        hipLaunchKernelGGL(block_score_few_kernel, dim3((unsigned)ceil_div(p->nK, 128), 1, pairs), dim3(256), 0, st, a);
    else if (p->nQ <= 16)
        hipLaunchKernelGGL((block_score_kernel<1, 1>), dim3((unsigned)ceil_div(p->nK, 64), 1, pairs), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((block_score_kernel<2, 2>), dim3((unsigned)ceil_div(p->nK, 128), (unsigned)ceil_div(p->nQ, 32), pairs), dim3(256), 0, st, a);
    rc = check_launch("block_score");
    if (rc) return rc;
    set_kernel_name("block_topk[nK=%d]", p->nK);
    // a row's keys stay in registers: one wave up to 2048 of them (four from 1025 on where rows are few: 23.8 against 25.9 us for 64 rows of
    // 2048, but 43.9 against 37.1 for 4500 of 900), sixteen waves beyond
    if (p->nK > 1024 && p->nK <= 2048 && (int64_t)pairs * p->nQ <= 512) return launch_topk<4, 8>(a, st);
    if (p->nK <= 256) return launch_topk<1, 4>(a, st);
    if (p->nK <= 1024) return launch_topk<1, 16>(a, st);
    if (p->nK <= 2048) return launch_topk<1, 32>(a, st);
    if (p->nK <= 8192) return launch_topk<16, 8>(a, st);
    return launch_topk<16, 32>(a, st);
}
