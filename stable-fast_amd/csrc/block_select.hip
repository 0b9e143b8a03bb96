// Which key blocks a query block attends to: block means (sfast_hip_block_means) and the choice by their products (sfast_hip_block_topk).
//
// Sums and products run in 64 bits: a choice stands on which of two scores is larger, and in 64 bits the order of the additions does not
// decide that (products of two fp32 means are exact, sums lose 2^-53). The cost is hidden: the means read x once, and the scores are few.
#include "common.h"
#include <math.h>

namespace sfast {

namespace {

// ---- block means ------------------------------------------------------------------------------------------------------------------------
// Bound by reading x. A workgroup owns one block and 32 runs of V elements (512 bytes of a contiguous token); 8 groups of threads share its
// rows, each thread keeps several 16-byte loads in flight, and the groups' sums are added in LDS in a fixed order.
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
    const int64_t unit = blockIdx.x / cols;
    const int run = (int)(blockIdx.x - unit * cols) * 32 + col;
    const int j = (int)(unit % a.n), b = (int)(unit / a.n);
    const int len = a.lengths ? min(max(a.lengths[b], 0), a.S) : a.S;
    const int rows = min(max(len - j * a.block, 0), a.block);
    double sum[V];
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0;
    const int64_t e = (int64_t)run * V;
    const int h = (int)(e / a.D), d = (int)(e - (int64_t)h * a.D);
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
    const int64_t first = (int64_t)(blockIdx.x - unit * cols) * 32 * V;
    for (int i = tid; i < 32 * V; i += 256) {
        const int c = i / V, k = i - c * V;
        if (first + i >= (int64_t)a.H * a.D) continue;
        double s = 0.0;
#pragma unroll
        for (int g = 0; g < 8; ++g) s += part[g][k * 32 + c];
        a.out[unit * a.H * a.D + first + i] = rows > 0 ? (float)(s / rows) : 0.f;
    }
}

// ---- scores -------------------------------------------------------------------------------------------------------------------------------
// 64-bit MFMAs (16x16x4) on operands read from memory as fp32: a lane reads four consecutive head-dim elements of its row at a time, and the
// four products of such a group take them in the order the lanes hold them -- any order of the head dim will do as long as both operands
// share it. A wave owns 16 x MI query blocks and 16 x NJ key blocks; a workgroup's four waves share the query blocks.
typedef double f64x4 __attribute__((ext_vector_type(4)));

struct TopkArgs {
    const float *qm, *km;
    const int32_t *klen;
    double *score;    // [B, Hk, nQ, nK]
    int32_t *out;     // [B, Hk, nQ, topk]
    int B, nQ, nK, H, Hk, G, D, topk, bk;
};

__device__ __forceinline__ int topk_count(const TopkArgs &a, int b) {
    if (!a.klen) return a.nK;
    const int64_t n = ((int64_t)max(a.klen[b], 0) + a.bk - 1) / a.bk;
    return (int)min(n, (int64_t)a.nK);
}

template <int MI, int NJ> __global__ void __launch_bounds__(256) block_score_kernel(const TopkArgs a) {
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
    for (int d0 = 0; d0 < a.D; d0 += 16) {
        const int d = d0 + 4 * l4;
        double q[MI][4], k[NJ][4];
#pragma unroll
        for (int y = 0; y < NJ; ++y) {
            const int j = j0 + 16 * y + l15;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
            if (d < a.D && j < count) v = *reinterpret_cast<const f32x4 *>(a.km + (((int64_t)b * a.nK + j) * a.Hk + hk) * a.D + d);
#pragma unroll
            for (int t = 0; t < 4; ++t) k[y][t] = (double)v[t];
        }
#pragma unroll
        for (int x = 0; x < MI; ++x) {
            const int i = i0 + 16 * x + l15;
#pragma unroll
            for (int t = 0; t < 4; ++t) q[x][t] = 0.0;
            if (d < a.D && i < a.nQ) {
                const float *row = a.qm + (((int64_t)b * a.nQ + i) * a.H + hk * a.G) * a.D + d;
                for (int g = 0; g < a.G; ++g) {
                    const f32x4 v = *reinterpret_cast<const f32x4 *>(row + g * a.D);
#pragma unroll
                    for (int t = 0; t < 4; ++t) q[x][t] += (double)v[t];
                }
            }
        }
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int x = 0; x < MI; ++x)
#pragma unroll
                for (int y = 0; y < NJ; ++y) acc[x][y] = __builtin_amdgcn_mfma_f64_16x16x4f64(q[x][t], k[y][t], acc[x][y], 0, 0, 0);
    }
    // result register r of a lane: query block 4 r + lane / 16, key block lane % 16
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int i = i0 + 16 * x + 4 * r + l4;
            if (i >= a.nQ) continue;
            double *row = a.score + ((int64_t)pair * a.nQ + i) * a.nK;
#pragma unroll
            for (int y = 0; y < NJ; ++y) {
                const int j = j0 + 16 * y + l15;
                if (j < count) row[j] = acc[x][y][r];
            }
        }
}

// ---- the topk best of a row ---------------------------------------------------------------------------------------------------------------
// WAVES waves hold a row's scores in registers as order-preserving 64-bit keys (0 = not there) and find the topk-th largest bit by bit from
// the top: a bit stays set while at least topk keys reach the candidate, and the search ends as soon as exactly topk do. Keys equal to the
// threshold are taken in the order of their index.
__device__ __forceinline__ uint64_t topk_key(double s) {
    s += 0.0;  // -0 and 0 are one score
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    if (s != s) return ~0ull;
    return (u >> 63) ? ~u : (u | (1ull << 63));
}

template <int WAVES, int NPL> __global__ void __launch_bounds__(WAVES == 1 ? 256 : WAVES * 64) block_topk_kernel(const TopkArgs a, int64_t n_rows) {
    __shared__ int sums[2][WAVES], above_s[WAVES], equal_s[WAVES];
    const int lane = threadIdx.x & 63, wave = WAVES == 1 ? 0 : threadIdx.x >> 6;
    const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
    if (row >= n_rows) return;
    const int64_t pair = row / a.nQ;
    const int count = topk_count(a, (int)(pair / a.Hk));
    const int j0 = wave * 64 * NPL + lane;
    uint64_t key[NPL];
#pragma unroll
    for (int n = 0; n < NPL; ++n) key[n] = j0 + 64 * n < count ? topk_key(a.score[row * a.nK + j0 + 64 * n]) : 0ull;
    int turn = 0;
    const auto total = [&](int mine) -> int {
        if (WAVES == 1) return mine;
        turn ^= 1;
        if (lane == 0) sums[turn][wave] = mine;
        __syncthreads();
        int s = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += sums[turn][w];
        return s;
    };
    uint64_t edge = 1;     // keys above it (or at it, in order) are chosen
    int at_edge = 0;       // how many of those at it; 0: all
    if (count > a.topk) {
        edge = 0;
        bool exact = false;
        for (int bit = 63; bit >= 0; --bit) {
            const uint64_t cand = edge | (1ull << bit);
            int mine = 0;
#pragma unroll
            for (int n = 0; n < NPL; ++n) mine += __popcll(__ballot(key[n] >= cand));
            const int have = total(mine);
            if (have >= a.topk) edge = cand;
            if (have == a.topk) {
                exact = true;
                break;
            }
        }
        if (!exact) {
            int mine = 0;
#pragma unroll
            for (int n = 0; n < NPL; ++n) mine += __popcll(__ballot(key[n] > edge));
            at_edge = a.topk - total(mine);
        }
    }
    // positions: chosen keys of earlier waves, earlier registers, lower lanes
    const uint64_t below = (1ull << lane) - 1;
    int above0 = 0, equal0 = 0;
    if (WAVES > 1) {
        int ab = 0, eq = 0;
#pragma unroll
        for (int n = 0; n < NPL; ++n) {
            ab += __popcll(__ballot(key[n] > edge));
            eq += __popcll(__ballot(key[n] == edge));
        }
        if (lane == 0) above_s[wave] = ab, equal_s[wave] = eq;
        __syncthreads();
        for (int w = 0; w < wave; ++w) above0 += above_s[w], equal0 += equal_s[w];
    }
    const int limit = at_edge ? at_edge : 0x7fffffff;
    int32_t *out = a.out + row * a.topk;
#pragma unroll
    for (int n = 0; n < NPL; ++n) {
        const uint64_t ab = __ballot(key[n] > edge), eq = __ballot(key[n] == edge);
        const int rank = equal0 + __popcll(eq & below);
        const bool take = key[n] > edge || (key[n] == edge && rank < limit);
        if (take) out[above0 + __popcll(ab & below) + min(rank, limit)] = j0 + 64 * n;
        above0 += __popcll(ab);
        equal0 += __popcll(eq);
    }
    for (int i = count + (WAVES == 1 ? lane : (int)threadIdx.x); i < a.topk; i += WAVES == 1 ? 64 : WAVES * 64) out[i] = -1;
}

template <int WAVES, int NPL> int launch_topk(const TopkArgs &a, hipStream_t st) {
    const int64_t rows = (int64_t)a.B * a.Hk * a.nQ;
    const dim3 grid((unsigned)(WAVES == 1 ? ceil_div64(rows, 4) : rows));
    hipLaunchKernelGGL((block_topk_kernel<WAVES, NPL>), grid, dim3(WAVES == 1 ? 256 : WAVES * 64), 0, st, a, rows);
    return check_launch("block_topk");
}

static int check_topk(const sfast_block_topk_params *p) {
    SFAST_REQUIRE(p, SFAST_ERR_INVALID, "block_topk: null argument");
    SFAST_REQUIRE(p->B > 0 && p->nQ > 0 && p->nK > 0 && p->H > 0 && p->Hk > 0 && p->D > 0 && p->topk > 0 && p->block_k > 0, SFAST_ERR_INVALID,
                  "block_topk: bad shape");
    SFAST_REQUIRE(p->H % p->Hk == 0, SFAST_ERR_INVALID, "block_topk: %d query heads are no multiple of %d key heads", p->H, p->Hk);
    SFAST_REQUIRE(p->D % 4 == 0, SFAST_ERR_UNSUPPORTED, "block_topk: head dim %d is no multiple of 4", p->D);
    SFAST_REQUIRE(p->nK <= 32768, SFAST_ERR_UNSUPPORTED, "block_topk: %d key blocks (up to 32768)", p->nK);
    SFAST_REQUIRE((int64_t)p->B * p->Hk <= 65535 && p->nQ <= (1 << 20) && (int64_t)p->B * p->Hk * p->nQ <= (1ll << 30), SFAST_ERR_UNSUPPORTED, "block_topk: too many rows");
    return SFAST_OK;
}

}  // namespace

template <typename T> static int means_launch(MeansArgs &a, int run, hipStream_t st) {
    a.runs = a.H * (a.D / run);
    const int64_t blocks = (int64_t)a.B * a.n * ceil_div(a.runs, 32);
    SFAST_REQUIRE(blocks <= (1ll << 31) - 1, SFAST_ERR_UNSUPPORTED, "block_means: too many blocks");
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
    a.B = p->B, a.S = p->S, a.H = p->H, a.D = p->D, a.block = p->block, a.n = ceil_div(p->S, p->block);
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
    a.qm = qm, a.km = km, a.klen = key_lengths, a.out = out, a.score = (double *)workspace;
    a.B = p->B, a.nQ = p->nQ, a.nK = p->nK, a.H = p->H, a.Hk = p->Hk, a.G = p->H / p->Hk, a.D = p->D, a.topk = p->topk, a.bk = p->block_k;
    hipStream_t st = (hipStream_t)stream;
    const unsigned pairs = (unsigned)(p->B * p->Hk);
    // up to 16 query blocks (a token has one): one row tile, the four waves side by side along the key blocks
    if (p->nQ <= 16)
        hipLaunchKernelGGL((block_score_kernel<1, 1>), dim3((unsigned)ceil_div(p->nK, 64), 1, pairs), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((block_score_kernel<2, 2>), dim3((unsigned)ceil_div(p->nK, 128), (unsigned)ceil_div(p->nQ, 32), pairs), dim3(256), 0, st, a);
    rc = check_launch("block_score");
    if (rc) return rc;
    set_kernel_name("block_topk[nK=%d]", p->nK);
    // a row's keys stay in registers: one wave up to 2048 of them, sixteen waves beyond
    if (p->nK <= 256) return launch_topk<1, 4>(a, st);
    if (p->nK <= 1024) return launch_topk<1, 16>(a, st);
    if (p->nK <= 2048) return launch_topk<1, 32>(a, st);
    if (p->nK <= 8192) return launch_topk<16, 8>(a, st);
    return launch_topk<16, 32>(a, st);
}
