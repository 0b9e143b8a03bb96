// Attention over chosen key blocks, forward (sfast_hip_block_attention).
//
// A query block of bq rows attends to the keys of the blocks its list names: o = softmax(scale q k^T) v with a running maximum and sum in
// fp32, lse = log of the sum. Per row and key 4 D flops on the matrix pipe against ~6 VALU operations for the softmax; K and V of a head are
// re-read by every query block that names them and live in L2 (each XCD walks a contiguous range of (batch, head, query block)).
//
//   * a workgroup is one query block: bq / 32 waves of 32 rows (Q in registers), which stream 64-key K and V tiles through two LDS stages
//     filled by LDS-DMA (no staging registers); V stays row-major and is read transposed by ds_read_b64_tr_b16.
//   * few query rows (a token against a long cache): the rows of all heads of a group share a wave (the group shares its list, K and V are
//     read once), and a list is split over workgroups whose partial results a second launch joins.
//
// Measured, bf16: 32760 x 24 rows of 128 against 64 blocks of 64 each 1.64 ms, 1005 TFLOP/s (a library's matrix product of 8192^3: 1406);
// 14400 x 20 rows of 64 against 32 blocks 176 us, 858 TFLOP/s. No single part bounds the first: without the exponentials (1540 us), the loads,
// the LDS reads, or either product (1320 - 1360 each) it is faster by less than that part alone takes; by the counters (8192 x 24 rows of 128) the
// matrix pipe is busy 48 % of the time and the VALU 38 %, for heads of 64 38 % and 60 %. With heads of 64 the VALU has the more to do (32 exponentials at 16 cycles, 32 fused products and 32 additions a tile
// of 64 keys and wave, 960 cycles against 512 of products). 4 x 8 rows of a token (32 heads) against 64 blocks of a long cache: 16 + 4 us, 50 MB.
// Tried and left: a tile's products under the next tile's softmax, raised wave priorities, the reference as the products' start
// (the compiler copies the registers), four waves a SIMD for heads of 64 (177 -> 195 us).
#include "block_attn.h"
#include <type_traits>

namespace sfast {

namespace {

constexpr int BA_MAX_LIST = 1024;  // entries of one workgroup's (part of a) list: 2048 tiles

template <int DP, int NS> constexpr int ba_fwd_lds() { return NS * 2 * BaTile<DP>::BYTES + BA_MAX_LIST * 2 * 4 + 16; }

// NS: LDS stages, NS - 1 tiles are on their way while one is used. KW = 2: two waves share the rows and take a half of every tile's keys each
// (joined through LDS at the end): where compute units are not full, a tile's chain of products, softmax and products is what takes time, and
// with 64 rows a workgroup its LDS leaves room for half the waves otherwise (16384 x 16 rows of 128, blocks of 64: 410 -> 340 us; with 128
// rows the waves are there anyway and the second set of them costs more than it hides, 177 -> 195 us for 14400 x 20 rows of 64).
// PACK: rows are (query, head of the group) pairs, row = s * G + g, one unit per key head; else one unit per query head.
constexpr int ba_key_waves(int NW, int NS, bool PACK) { return PACK || NS > 2 || NW == 2 ? 2 : 1; }

template <typename T, int DP, int NW, int NS, bool PACK, int KW = ba_key_waves(NW, NS, PACK)>
__global__ void __launch_bounds__(NW * KW * 64, 2) block_attn_fwd_kernel(const BlockAttnArgs a) {
    using vec8 = typename Elem<T>::vec8;
    constexpr int KD = DP / 16, DB = DP / 32, TILE = BaTile<DP>::BYTES, KBN = 2 / KW;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int *tiles = reinterpret_cast<int *>(smem + NS * 2 * TILE);
    int *ntiles_p = tiles + 2 * BA_MAX_LIST;

    const int lin = (blockIdx.x & 7) * a.chunk + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= a.chunk || lin >= a.nblk) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, hi = lane >> 5;
    // order of the work: (batch, key head, query block, head of the group | part of the list)
    const int inner = PACK ? a.nsplit : a.G * a.nsplit;
    const int in = lin % inner, u = lin / inner;
    const int sp = in % a.nsplit, g0 = PACK ? 0 : in / a.nsplit;
    const int qb = u % a.nQ, pair = u / a.nQ;
    const int hk = pair % a.Hk, b = pair / a.Hk;
    const int klen = a.klen ? min(max(a.klen[b], 0), a.Sk) : a.Sk;
    const int qlen = a.qlen ? min(max(a.qlen[b], 0), a.Sq) : a.Sq;

    const int half = KW == 1 ? 0 : wave / NW;  // the half of the keys
    const int r = (KW == 1 ? wave : wave % NW) * 32 + l31;
    const int s = PACK ? r / a.G : qb * a.bq + r;
    const int h = hk * a.G + (PACK ? r - s * a.G : g0);
    const bool inside = PACK ? s < a.Sq : (r < a.bq && s < a.Sq);  // a row of the output
    const bool row_ok = inside && s < qlen;

    if (wave == 0) {
        int n = 0;
        if ((PACK ? 0 : qb * a.bq) < qlen) {
            const int e0 = (int)((int64_t)a.topk * sp / a.nsplit), e1 = (int)((int64_t)a.topk * (sp + 1) / a.nsplit);
            n = ba_tiles(a.blocks + ((int64_t)pair * a.nQ + qb) * a.topk, e0, e1, a.bk, klen, lane, tiles);
        }
        if (lane == 0) *ntiles_p = n;
    }

    // Q: B operand, column = the lane's row
    const T *Qp = (const T *)a.q + (int64_t)b * a.qs[0] + (int64_t)s * a.qs[1] + (int64_t)h * a.qs[2];
    vec8 qf[KD];
#pragma unroll
    for (int kd = 0; kd < KD; ++kd) {
        const int d0 = kd * 16 + hi * 8;
        u32x4 raw = {0u, 0u, 0u, 0u};
        if (row_ok && d0 < a.D) raw = *reinterpret_cast<const u32x4 *>(Qp + d0);
        qf[kd] = __builtin_bit_cast(vec8, raw);
    }

    const T *Kp = (const T *)a.k + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[2];
    const T *Vp = (const T *)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[2];
    BaLoader<DP, NW * KW> kl, vl;
    kl.init(wave, lane, a.ks[1], a.D);
    vl.init(wave, lane, a.vs[1], a.D);

    f32x16 o[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m = -INFINITY, l = 0.f;  // reference of the row (log2 units) and the lane's share of the sum
    const float c = a.c;

    __syncthreads();
    const int n = __builtin_amdgcn_readfirstlane(*ntiles_p);
    const auto request = [&](int t) __attribute__((always_inline)) {
        const int tile = __builtin_amdgcn_readfirstlane(tiles[t]);
        char *st = smem + (t % NS) * (2 * TILE);
        kl.load(Kp, a.ks[1], a.D, tile * 64, klen - tile * 64, st, wave);
        vl.load(Vp, a.vs[1], a.D, tile * 64, klen - tile * 64, st + TILE, wave);
    };
#pragma unroll
    for (int t = 0; t < NS - 1; ++t)
        if (t < n) request(t);
    for (int t = 0; t < n; ++t) {
        const int cur = __builtin_amdgcn_readfirstlane(tiles[t]);
        char *Ks = smem + (t % NS) * (2 * TILE), *Vs = Ks + TILE;
        // tile t has landed (NS - 2 later ones may be on their way), every wave is done with the stage that is requested next
        if (NS > 2 && t + NS - 2 < n)
            ba_sync<(NS - 2) * 2 * BaLoader<DP, NW * KW>::N>();
        else
            ba_sync();
        if (t + NS - 1 < n) request(t + NS - 1);
        // scores: all K fragments are requested before the first product (the two key halves alternate: independent accumulators)
        vec8 kf[KBN][KD];
#pragma unroll
        for (int kd = 0; kd < KD; ++kd)
#pragma unroll
            for (int kb = 0; kb < KBN; ++kb) kf[kb][kd] = ba_row_frag<T, DP>(Ks, (half + kb) * 32 + l31, kd, hi);
        __builtin_amdgcn_sched_barrier(0);
        f32x16 sc[KBN];
#pragma unroll
        for (int kb = 0; kb < KBN; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[kb][i] = 0.f;
#pragma unroll
        for (int kd = 0; kd < KD; ++kd)
#pragma unroll
            for (int kb = 0; kb < KBN; ++kb) sc[kb] = ba_mfma(kf[kb][kd], qf[kd], sc[kb]);
        __builtin_amdgcn_sched_barrier(0);
        // V^T fragments of the first half of the keys arrive under the softmax
        vec8 vf[2 * KBN][DB];
#pragma unroll
        for (int g = 0; g < KBN; ++g)
#pragma unroll
            for (int db = 0; db < DB; ++db) vf[g][db] = ba_col_frag<T, DP>(Vs, lane, db, half * 32 + g * 16);
        __builtin_amdgcn_sched_barrier(0);
        const int left = klen - cur * 64;
        if (left < 64) {
#pragma unroll
            for (int kb = 0; kb < KBN; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if ((half + kb) * 32 + (i & 3) + 8 * (i >> 2) + 4 * hi >= left) sc[kb][i] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < KBN; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kb][i]);
        mx = ba_xor32_max(mx) * c;
        // the reference follows the maximum only when that has grown 256-fold: o / l does not depend on it, and sums and products have the
        // range for it (f16 probabilities up to 256)
        if (__any(mx > m + 8.f)) {
            const float mn = fmaxf(m, mx);
            const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
        }
        const float ref = m == -INFINITY ? 0.f : m;  // a row whose scores are all -inf keeps the sum 0
        // the sum takes the probabilities in fp32, the product with V takes them rounded to the type: half a step each, so that out is off by 1.1
        // times (5 keys) to 1.4 times (many) what its own rounding alone would give
        vec8 p[2 * KBN];
#pragma unroll
        for (int kb = 0; kb < KBN; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(fmaf(sc[kb][i], c, -ref));
                l += e;
                p[kb * 2 + (i >> 3)][i & 7] = Elem<T>::from_f32(e);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int g = KBN; g < 2 * KBN; ++g)
#pragma unroll
            for (int db = 0; db < DB; ++db) vf[g][db] = ba_col_frag<T, DP>(Vs, lane, db, half * 32 + g * 16);
#pragma unroll
        for (int g = 0; g < 2 * KBN; ++g)
#pragma unroll
            for (int db = 0; db < DB; ++db) o[db] = ba_mfma(vf[g][db], p[g], o[db]);
    }
    l = ba_xor32_sum(l);
    if constexpr (KW == 2) {
        // the second half's sums come through LDS (the stages are free, the list is no longer needed)
        __syncthreads();
        const int rw = wave % NW;
        float *const so = reinterpret_cast<float *>(smem) + rw * (DB * 16 * 64) + lane, *const sml = reinterpret_cast<float *>(tiles) + rw * 128 + lane;
        if (half == 1) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) so[(db * 16 + i) * 64] = o[db][i];
            sml[0] = m, sml[64] = l;
        }
        __syncthreads();
        if (half == 1) return;
        const float m1 = sml[0], top = fmaxf(m, m1), base = top == -INFINITY ? 0.f : top;
        const float w0 = __builtin_amdgcn_exp2f(m - base), w1 = __builtin_amdgcn_exp2f(m1 - base);
        m = top, l = l * w0 + sml[64] * w1;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] = o[db][i] * w0 + so[(db * 16 + i) * 64] * w1;
    }
    if (!inside) return;
    if (!row_ok) {  // a row behind its sequence: nothing
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    }

    if (a.nsplit > 1) {
        const int64_t row = (((int64_t)u * (PACK ? 1 : a.G) + g0) * a.nsplit + sp) * (NW * 32) + r;
        float *po = a.part_o + row * a.D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = db * 32 + 8 * i + 4 * hi;
                if (d < a.D) *reinterpret_cast<f32x4 *>(po + d) = f32x4{o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]};
            }
        if (hi == 0) *reinterpret_cast<float2 *>(a.part_ml + row * 2) = make_float2(m, l);
        return;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;  // no key (or all scores -inf): zeros
    const int64_t at = (int64_t)b * a.os[0] + (int64_t)s * a.os[1] + (int64_t)h * a.os[2];
    T *Op = (T *)a.out + at;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = db * 32 + 8 * i + 4 * hi;
            if (d < a.D) {
                const float x[4] = {o[db][4 * i] * inv, o[db][4 * i + 1] * inv, o[db][4 * i + 2] * inv, o[db][4 * i + 3] * inv};
                const u32x2 y = pack4<T>(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<u32x2 *>(Op + d) = y;
                if (a.out_rest) {
                    float z[4];
                    unpack4<T>(y, z);
                    *reinterpret_cast<u32x2 *>((T *)a.out_rest + at + d) = pack4<T>(x[0] - z[0], x[1] - z[1], x[2] - z[2], x[3] - z[3]);
                }
            }
        }
    if (hi == 0) {
        float v = -INFINITY;
        if (!(l == 0.f)) v = (m + __log2f(l)) * 0.69314718055994530942f;
        a.lse[((int64_t)b * a.H + h) * a.Sq + s] = v;
    }
}

// joins the parts of a row: o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s. One wave a row: lane p has part p's weight (64 parts at a time),
// every lane two columns, eight parts in flight.
template <typename T, bool PACK> __global__ void __launch_bounds__(256) block_attn_join_kernel(const BlockAttnArgs a, int rows, int n_rows) {
    const int lane = threadIdx.x & 63;
    const int id = blockIdx.x * 4 + (threadIdx.x >> 6);   // (b, hk, qb, g, row of the block) | (b, hk, row)
    if (id >= n_rows) return;
    const int per = PACK ? a.Sq * a.G : a.bq;
    const int unit = id / per, r = id - unit * per;
    int x = unit, g = 0, qb = 0;
    if (!PACK) g = x % a.G, x /= a.G, qb = x % a.nQ, x /= a.nQ;
    const int b = x / a.Hk, hk = x - b * a.Hk;
    const int s = PACK ? r / a.G : qb * a.bq + r;
    const int h = hk * a.G + (PACK ? r - s * a.G : g);
    if (s >= a.Sq) return;
    const int64_t first = (int64_t)unit * a.nsplit * rows + r;
    const float *ml = a.part_ml + first * 2;
    const float *po = a.part_o + first * a.D;
    const int64_t ml_step = (int64_t)rows * 2, po_step = (int64_t)rows * a.D;
    const int d = lane * 2 < a.D ? lane * 2 : 0;
    float M = -INFINITY, L = 0.f, x0 = 0.f, x1 = 0.f;
    for (int p0 = 0; p0 < a.nsplit; p0 += 64) {
        const int n = min(64, a.nsplit - p0);
        float2 mine = make_float2(-INFINITY, 0.f);
        if (lane < n) mine = *reinterpret_cast<const float2 *>(ml + (p0 + lane) * ml_step);
        const float top = fmaxf(M, wave_max(mine.x));
        const float ref = top == -INFINITY ? 0.f : top;
        const float old = __builtin_amdgcn_exp2f(M - ref);  // (-inf: nothing was summed yet)
        const float w = __builtin_amdgcn_exp2f(mine.x - ref);
        M = top;
        L = L * old + wave_sum(w * mine.y);
        x0 *= old, x1 *= old;
#pragma unroll 1
        for (int p = 0; p < n; p += 8) {
            float2 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const float2 *>(po + (int64_t)(p0 + min(p + i, n - 1)) * po_step + d);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float wi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), min(p + i, 63)));
                if (p + i >= n) wi = 0.f, v[i] = make_float2(0.f, 0.f);
                x0 = fmaf(wi, v[i].x, x0);
                x1 = fmaf(wi, v[i].y, x1);
            }
        }
    }
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
    const int64_t at = (int64_t)b * a.os[0] + (int64_t)s * a.os[1] + (int64_t)h * a.os[2];
    if (lane * 2 < a.D) {
        const T y0 = Elem<T>::from_f32(x0 * inv), y1 = Elem<T>::from_f32(x1 * inv);
        const typename Elem<T>::vec2 y = {y0, y1};
        *reinterpret_cast<typename Elem<T>::vec2 *>((T *)a.out + at + d) = y;
        if (a.out_rest) {
            const typename Elem<T>::vec2 z = {Elem<T>::from_f32(x0 * inv - (float)y0), Elem<T>::from_f32(x1 * inv - (float)y1)};
            *reinterpret_cast<typename Elem<T>::vec2 *>((T *)a.out_rest + at + d) = z;
        }
    }
    if (lane == 0) {
        float v = -INFINITY;
        if (!(L == 0.f)) v = (M + __log2f(L)) * 0.69314718055994530942f;
        a.lse[((int64_t)b * a.H + h) * a.Sq + s] = v;
    }
}

template <typename T, int DP, int NW, int NS, bool PACK> int set_attr() {
    auto kern = block_attn_fwd_kernel<T, DP, NW, NS, PACK>;
    const hipError_t e = hipFuncSetAttribute((const void *)kern, hipFuncAttributeMaxDynamicSharedMemorySize, ba_fwd_lds<DP, NS>());
    if (e != hipSuccess) {
        set_error("hipFuncSetAttribute(block_attn_fwd): %s", hipGetErrorString(e));
        return SFAST_ERR_LAUNCH;
    }
    return 0;
}

struct Plan {
    bool pack, deep;
    int nw, nsplit;
    int64_t units, nblk;
};

// How a call is cut into workgroups.
//  * Packed rows: all query rows of a group fit 64 rows of one or two waves.
//  * A list is split over workgroups where that is shorter. Measured: a workgroup takes 1.1 us a tile while compute units are free (512
//    workgroups are two on each), 0.8 us with two waves for the keys; a split adds 4 us for the second launch and the partial results' way
//    through memory at 3.2 bytes / ps (8 heads of 1000 rows of 128 against 64 blocks: 33.5 us, with 0.8 bytes / ps in this sum 45.5).
//  * deep: four LDS stages instead of two and two waves for the keys, for grids that leave one workgroup to a compute unit anyway
//    (2 x 6 x 1000 rows against 8 blocks of 64: 11.7 us, with two stages and one wave 14.7). Not for
//    packed rows: 4 x 8 of them with lists cut in eight take 19.9 us with four stages, 19.0 with two.
static Plan make_plan(const sfast_block_attn_params *p) {
    Plan pl{};
    const int G = p->H / p->Hk;
    const int nQ = ceil_div(p->Sq, p->block_q);
    pl.pack = nQ == 1 && (int64_t)p->Sq * G <= 64;
    pl.nw = pl.pack ? (p->Sq * G <= 32 ? 1 : 2) : p->block_q / 32;
    pl.units = (int64_t)p->B * p->Hk * nQ * (pl.pack ? 1 : G);
    // (SFAST_BATCH_INVARIANT: a sample's parts are those of the reference batch, common.h)
    const int64_t units = g_batch_ref > 0 ? pl.units / p->B * g_batch_ref : pl.units;
    const int64_t tiles = (int64_t)p->topk * (p->block_k / 64);
    const int64_t least = ceil_div64(p->topk, BA_MAX_LIST - 1);  // a part holds at most BA_MAX_LIST entries
    int64_t ns = least;
    if (units < 256) {
        const double rows = pl.pack ? (double)p->Sq * G : pl.nw * 32;
        const double part = 2.0 * units * rows * p->D * 4 / 3.2e6;  // us a part, written and read
        const auto tile_us = [&](int64_t blocks) { return pl.pack || blocks <= 256 ? 0.8 : 1.1; };
        double best = tile_us(units * least) * (double)ceil_div64(tiles, least) + (least > 1 ? 4.0 + part * least : 0.0);
        for (int64_t x = least + 1; x <= p->topk && x <= tiles / 2 && x * units <= 1024; x += 1 + x / 32) {
            const double rounds = (double)ceil_div64(x * units, 512);
            const double t = tile_us(x * units) * (double)ceil_div64(tiles, x) * rounds + 4.0 + part * (double)x;
            if (t < best) best = t, ns = x;
        }
    }
    pl.nsplit = (int)ns;
    pl.nblk = pl.units * ns;
    pl.deep = !pl.pack && units * ns <= 256;  // (decides how many waves share a row's keys: the order of its sums)
    return pl;
}

template <typename T, int DP> int launch(const BlockAttnArgs &a, const Plan &pl, hipStream_t st) {
    const dim3 grid((unsigned)(8 * a.chunk));
    const auto go = [&](auto NW, auto NS, auto PACK) {
        constexpr int nw = decltype(NW)::value, ns = decltype(NS)::value;
        hipLaunchKernelGGL((block_attn_fwd_kernel<T, DP, nw, ns, decltype(PACK)::value>), grid, dim3(nw * ba_key_waves(nw, ns, decltype(PACK)::value) * 64),
                           (ba_fwd_lds<DP, ns>()), st, a);
    };
    const auto with = [&](auto NW) {
        if (pl.deep)
            go(NW, std::integral_constant<int, 4>{}, std::false_type{});
        else
            go(NW, std::integral_constant<int, 2>{}, std::false_type{});
    };
    if (pl.pack && pl.nw == 1)
        go(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{}, std::true_type{});
    else if (pl.pack)
        go(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{}, std::true_type{});
    else if (pl.nw == 2)
        with(std::integral_constant<int, 2>{});
    else
        with(std::integral_constant<int, 4>{});
    int rc = check_launch("block_attention");
    if (rc || pl.nsplit == 1) return rc;
    const int per = pl.pack ? a.Sq * a.G : a.bq;
    const int rows = (int)(pl.units * per);  // (the entry point holds units * 128 rows of a split call below 2^26)
    const dim3 jgrid((unsigned)ceil_div(rows, 4));
    if (pl.pack)
        hipLaunchKernelGGL((block_attn_join_kernel<T, true>), jgrid, dim3(256), 0, st, a, pl.nw * 32, rows);
    else
        hipLaunchKernelGGL((block_attn_join_kernel<T, false>), jgrid, dim3(256), 0, st, a, pl.nw * 32, rows);
    return check_launch("block_attention join");
}

}  // namespace

int block_attn_check(const sfast_block_attn_params *p) {
    SFAST_REQUIRE(p, SFAST_ERR_INVALID, "block_attention: null argument");
    SFAST_REQUIRE(p->dtype == SFAST_F16 || p->dtype == SFAST_BF16, SFAST_ERR_UNSUPPORTED, "block_attention: f16 / bf16 only");
    SFAST_REQUIRE(p->B > 0 && p->H > 0 && p->Hk > 0 && p->Sq > 0 && p->Sk > 0 && p->D > 0 && p->topk > 0, SFAST_ERR_INVALID, "block_attention: bad shape");
    SFAST_REQUIRE(p->H % p->Hk == 0, SFAST_ERR_INVALID, "block_attention: %d query heads are no multiple of %d key heads", p->H, p->Hk);
    SFAST_REQUIRE(p->D % 8 == 0 && p->D <= 128, SFAST_ERR_UNSUPPORTED, "block_attention: head dim %d (a multiple of 8 up to 128 is supported)", p->D);
    SFAST_REQUIRE((p->block_q == 64 || p->block_q == 128) && (p->block_k == 64 || p->block_k == 128), SFAST_ERR_UNSUPPORTED,
                  "block_attention: blocks of 64 or 128 rows, got %d / %d", p->block_q, p->block_k);
    // (the gradients hold lse / scale in fp32)
    SFAST_REQUIRE(p->scale >= 0x1p-100f && p->scale < INFINITY, SFAST_ERR_UNSUPPORTED, "block_attention: the scale must be positive (2^-100 and more) and finite");
    SFAST_REQUIRE(p->Sq <= (1 << 30) && p->Sk <= (1 << 30), SFAST_ERR_UNSUPPORTED, "block_attention: more than 2^30 rows");
    for (int i = 0; i < 3; ++i)
        SFAST_REQUIRE(p->qs[i] >= 0 && p->ks[i] >= 0 && p->vs[i] >= 0 && p->qs[i] % 8 == 0 && p->ks[i] % 8 == 0 && p->vs[i] % 8 == 0, SFAST_ERR_UNSUPPORTED,
                      "block_attention: strides must be multiples of 8 elements");
    // offsets inside one 64-row tile have 32 bits, bit 31 marks an element outside
    SFAST_REQUIRE(p->ks[1] < (1 << 23) && p->vs[1] < (1 << 23) && p->qs[1] < (1 << 23), SFAST_ERR_UNSUPPORTED, "block_attention: row stride too long");
    // what lies behind a tile's last row is cut off by its address: rows must not overlap
    SFAST_REQUIRE(p->ks[1] >= p->D && p->vs[1] >= p->D && p->qs[1] >= p->D, SFAST_ERR_UNSUPPORTED, "block_attention: rows overlap");
    return SFAST_OK;
}

int block_attn_init() {
    int rc = 0;
#define SFAST_BA_ATTR(T, DP)                                                         \
    if (!rc) rc = set_attr<T, DP, 1, 2, true>();                                     \
    if (!rc) rc = set_attr<T, DP, 2, 2, true>();                                     \
    if (!rc) rc = set_attr<T, DP, 2, 2, false>();                                    \
    if (!rc) rc = set_attr<T, DP, 4, 2, false>();                                    \
    if (!rc) rc = set_attr<T, DP, 2, 4, false>();                                    \
    if (!rc) rc = set_attr<T, DP, 4, 4, false>();
    SFAST_BA_ATTR(f16, 64)
    SFAST_BA_ATTR(f16, 128)
    SFAST_BA_ATTR(bf16, 64)
    SFAST_BA_ATTR(bf16, 128)
#undef SFAST_BA_ATTR
    return rc;
}

}  // namespace sfast

using namespace sfast;

extern "C" size_t sfast_hip_block_attention_workspace_bytes(const sfast_block_attn_params *p) {
    if (block_attn_check(p) != SFAST_OK) return 0;
    const Plan pl = make_plan(p);
    if (pl.nsplit == 1) return 0;
    return (size_t)pl.nblk * (pl.nw * 32) * (p->D + 2) * 4;
}

extern "C" int sfast_hip_block_attention(const void *q, const void *k, const void *v, const int32_t *blocks, const int32_t *key_lengths,
                                         const int32_t *query_lengths, void *out, float *lse, void *out_rest, const sfast_block_attn_params *p,
                                         void *workspace, size_t workspace_bytes, sfast_stream_t stream) {
    SFAST_REQUIRE(q && k && v && blocks && out && lse, SFAST_ERR_INVALID, "block_attention: null argument");
    int rc = block_attn_check(p);
    if (rc != SFAST_OK) return rc;
    SFAST_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned8(out) && aligned8(out_rest), SFAST_ERR_UNSUPPORTED,
                  "block_attention: operands must be 16-byte aligned");
    for (int i = 0; i < 3; ++i) SFAST_REQUIRE(p->os[i] % 4 == 0, SFAST_ERR_UNSUPPORTED, "block_attention: output strides must be multiples of 4 elements");
    const Plan pl = make_plan(p);
    // (the join gives a wave to a row: bq rows of a unit)
    SFAST_REQUIRE(fits_launch(pl.nblk + 7, pl.nw * 128) && (pl.nsplit == 1 || fits_launch(pl.units * 128, 64)), SFAST_ERR_UNSUPPORTED,
                  "block_attention: too many query blocks");
    BlockAttnArgs a{};
    a.q = q, a.k = k, a.v = v, a.blocks = blocks, a.klen = key_lengths, a.qlen = query_lengths, a.out = out, a.out_rest = out_rest, a.lse = lse;
    a.B = p->B, a.H = p->H, a.Hk = p->Hk, a.G = p->H / p->Hk, a.Sq = p->Sq, a.Sk = p->Sk, a.D = p->D, a.topk = p->topk;
    a.bq = p->block_q, a.bk = p->block_k, a.nQ = ceil_div(p->Sq, p->block_q), a.nK = ceil_div(p->Sk, p->block_k);
    for (int i = 0; i < 3; ++i) a.qs[i] = p->qs[i], a.ks[i] = p->ks[i], a.vs[i] = p->vs[i], a.os[i] = p->os[i];
    a.scale = p->scale;
    a.c = p->scale * 1.44269504088896340736f;
    a.nsplit = pl.nsplit;
    a.nblk = (int)pl.nblk;
    a.chunk = (int)ceil_div64(pl.nblk, 8);
    if (pl.nsplit > 1) {
        SFAST_REQUIRE(workspace && workspace_bytes >= sfast_hip_block_attention_workspace_bytes(p) && aligned16(workspace), SFAST_ERR_WORKSPACE,
                      "block_attention: workspace too small");
        a.part_o = (float *)workspace;
        a.part_ml = a.part_o + (size_t)pl.nblk * (pl.nw * 32) * p->D;
    }
    hipStream_t st = (hipStream_t)stream;
    set_kernel_name("block_attn_fwd[DP=%d,rows=%d,stages=%d,split=%d%s]", p->D <= 64 ? 64 : 128, pl.nw * 32, pl.deep ? 4 : 2, pl.nsplit,
                    pl.pack ? ",packed" : "");
    if (p->dtype == SFAST_F16) return p->D <= 64 ? launch<f16, 64>(a, pl, st) : launch<f16, 128>(a, pl, st);
    return p->D <= 64 ? launch<bf16, 64>(a, pl, st) : launch<bf16, 128>(a, pl, st);
}
