// Attention over chosen key blocks, gradients (sfast_hip_block_attention_backward).
//
// With P = exp(s - lse): dV = P^T dO, dP = dO V^T, dS = P (dP - delta), dQ = scale dS K, dK = scale dS^T Q, delta = rowsum(dO O) - dlse.
// Bound by the matrix pipe (seven products a tile pair: the scores and dP are made twice) together with the VALU (an exponential a pair and
// kernel). bf16: 14400 x 20 rows of 64 against 32 blocks of 64 take 565 us, 935 TFLOP/s over the seven products (dkv takes 3 parts of 5);
// 32760 x 24 rows of 128 against 64 blocks 6.6 ms, 878 TFLOP/s.
//
//   * two kernels instead of atomics, so that the same call gives the same bits: one streams the listed key blocks past a query block (dQ),
//     one streams the query blocks past a key block (dK, dV).
//   * the second needs the lists the other way round: a small kernel counts, per key block, how often each query block names it (integer
//     atomics: their order changes nothing), and the workgroup of a key block walks its row of counts.
//   * both keep their own rows' operands and sums in registers and read the streamed tiles from LDS as rows (scores, dP) and transposed (sums).
//   * dkv of 64-key blocks and heads of 64: four waves a workgroup, two for the keys, two for the halves of each tile's rows. The same LDS then
//     serves twice the waves (three a SIMD): 594 -> 576 us for the 14400 x 20 rows. Heads of 128 fill the registers: one wave a SIMD (dq in
//     256 registers spills: 6.6 -> 7.2 ms).
#include "block_attn.h"
#include <algorithm>
#include <type_traits>

namespace sfast {

namespace {

constexpr int BB_LIST = 1024, BB_NAMES = 256;  // list entries, query blocks held in LDS at a time (three dkv workgroups of D <= 64 and more fit a compute unit)
constexpr float LOG2E = 1.44269504088896340736f;

template <int DP> constexpr int bb_dq_lds() { return 4 * BaTile<DP>::BYTES + BB_LIST * 2 * 4 + 16; }
template <int DP> constexpr int bb_halves() { return DP == 64 ? 2 : 1; }  // waves that share the rows of a dkv tile (64-key blocks)
template <int DP> constexpr int bb_dkv_lds() { return 4 * BaTile<DP>::BYTES + 2 * 1024 + BB_NAMES * 2 * 4 + 16; }

// What a row's statistics enter the products as: -lse / scale (dkv) and -delta (both), each as four numbers of the type times fixed powers of
// two (one more matrix instruction starts the accumulators from their sums), each number what the ones before it left.
//  * bf16 has fp32's range: powers of 1, and the numbers hold all of an fp32 value down to bf16's smallest normal number, 2^-126.
//  * f16: powers 2^15 to 2^-14, from 2^31 down to steps of 2^-28 (a delta below 2^-28 counts as 0; dout is f16 too, in steps of 2^-24, and so
//    are the gradients). A finite number beyond them (2^31, where q . k holds no more than its leading digits unless scale is tiny) becomes
//    NaN: a gradient that cannot be had is not 0.
// Parts below the type's normal numbers are left to the next one, so that nothing depends on how subnormals are multiplied.
template <typename T> struct BbParts;
template <> struct BbParts<f16> {
    static constexpr float POWER[4] = {32768.f, 16.f, 1.f / 128.f, 1.f / 16384.f}, LEAST = 0x1p-14f;
};
template <> struct BbParts<bf16> {
    static constexpr float POWER[4] = {1.f, 1.f, 1.f, 1.f}, LEAST = 0x1p-126f;
};
template <typename T> __device__ __forceinline__ u32x2 bb_parts(float x) {
    typename Elem<T>::vec4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a = x * (1.f / BbParts<T>::POWER[i]);
        if (fabsf(a) < BbParts<T>::LEAST) a = 0.f;
        v[i] = Elem<T>::from_f32(a);
        if (i == 0 && fabsf(x) < INFINITY && fabsf((float)v[0]) == INFINITY) v[0] = Elem<T>::from_f32(NAN);
        const float taken = (float)v[i];
        x = taken != taken || fabsf(taken) == INFINITY ? 0.f : fmaf(-taken, BbParts<T>::POWER[i], x);
    }
    return __builtin_bit_cast(u32x2, v);
}

// the operand that the parts meet: its elements 0 .. 3 of the 16 summed ones are the powers, the rest 0
template <typename T> __device__ __forceinline__ typename Elem<T>::vec8 bb_powers(int hi) {
    typename Elem<T>::vec8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = Elem<T>::from_f32(i < 4 && hi == 0 ? BbParts<T>::POWER[i & 3] : 0.f);
    return v;
}

// A row's delta (LPR lanes, 8 elements each) and parts; rows up to whole query blocks exist and are marked empty. Clears the counts as well.
// Bound by reading out, what its rounding left, and its gradient once (14400 x 20 rows of 64: 24 us, 111 MB, 4.6 TB/s).
template <typename T, int LPR> __global__ void __launch_bounds__(256) block_attn_delta_kernel(const BlockAttnArgs a, int64_t cells) {
    const int64_t blocks = (int64_t)gridDim.x * gridDim.y;
    for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < cells; i += blocks * 256) a.cnt[i] = 0;
    const uint32_t row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR;  // (s, h) of sequence b
    const int d = (threadIdx.x % LPR) * 8, b = blockIdx.y;
    const int Sp = a.nQ * a.bq;
    if (row >= (uint32_t)Sp * (uint32_t)a.H) return;
    const int s = (int)(row / (uint32_t)a.H), h = (int)(row - (uint32_t)s * (uint32_t)a.H);
    const int qlen = a.qlen ? min(max(a.qlen[b], 0), a.Sq) : a.Sq;
    float sum = 0.f;
    if (s < qlen && d < a.D) {
        const int64_t at = b * a.os[0] + s * a.os[1] + h * a.os[2] + d;
        const u32x4 g = *reinterpret_cast<const u32x4 *>((const T *)a.dout + b * a.dos[0] + s * a.dos[1] + h * a.dos[2] + d);
        const u32x4 o = *reinterpret_cast<const u32x4 *>((const T *)a.o + at);
        u32x4 z = {0u, 0u, 0u, 0u};
        // out to 16 more bits: in a row that attends to few keys dP - delta cancels
        if (a.o_rest) z = *reinterpret_cast<const u32x4 *>((const T *)a.o_rest + at);
        float x[8], y[8], w[8];
        unpack8<T>(g, x);
        unpack8<T>(o, y);
        unpack8<T>(z, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[i], y[i], sum);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum = fmaf(x[i], w[i], sum);
    }
#pragma unroll
    for (int off = LPR / 2; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
    if (d >= 16) return;
    // the first lane writes lse's parts, the second delta and its parts
    const int64_t at = ((int64_t)b * a.H + h) * a.Sq + s;
    float x;
    if (d == 0) {
        const float L = s < qlen ? a.lse[at] : -INFINITY;
        x = L == -INFINITY ? -INFINITY : -L / a.scale;  // a row without keys: probabilities 0
    } else {
        if (a.dlse && s < qlen) sum -= a.dlse[at];
        x = -sum;
    }
    reinterpret_cast<u32x2 *>(a.stat + ((int64_t)b * a.H + h) * Sp + s)[d == 0 ? 0 : 1] = bb_parts<T>(x);
}

// cnt[pair][key block][query block] += 1 for every entry that names something
__global__ void __launch_bounds__(256) block_attn_count_kernel(const BlockAttnArgs a) {
    const int e = blockIdx.x * 256 + threadIdx.x;  // entry of the lists of one (batch, key head)
    if (e >= a.nQ * a.topk) return;
    const int pair = blockIdx.y, qb = e / a.topk, b = pair / a.Hk;
    const int klen = a.klen ? min(max(a.klen[b], 0), a.Sk) : a.Sk;
    const int j = a.blocks[(int64_t)pair * a.nQ * a.topk + e];
    if (j >= 0 && (int64_t)j * a.bk < klen) atomicAdd(a.cnt + ((int64_t)pair * a.nK + j) * a.nQ + qb, 1);
}

// Probabilities and dS are rounded to the type for the products that sum them, which doubles the square of a gradient's error: 1.42 times one
// rounding's, measured alike for lists of 1 to 30 blocks and for 5 keys. With FINE the part that this rounding cuts off takes part as well, in
// products of its own: the gradient keeps its last rounding alone. The rule is what that costs. Calls of one query or one key block have it:
// their time is that of a chain of small steps (100 x 16 query rows of 64 against 16 blocks of 64: 43.5 -> 47 us). Whole grids would pay a third.
// f16: a dS below 2^-14 loses digits and below 2^-25 is 0 (the cut-off part is smaller still), so small losses want a scale, as for any f16 gradient.
template <typename T, bool FINE> struct BbRounded {
    typename Elem<T>::vec8 v, rest;
    __device__ __forceinline__ void set(int i, float x) {
        v[i] = Elem<T>::from_f32(x);
        if (FINE) rest[i] = Elem<T>::from_f32(x - (float)v[i]);
    }
    __device__ __forceinline__ f32x16 times(typename Elem<T>::vec8 a, f32x16 c) const {
        if (FINE) c = ba_mfma(a, rest, c);
        return ba_mfma(a, v, c);
    }
};

// dQ of one query block: the forward's streams, K read as rows (scores) and transposed (dQ), V as rows (dP)
template <typename T, int DP, int NW, bool FINE>
__global__ void __launch_bounds__(NW * 64, DP == 128 ? 1 : NW == 4 ? 3 : 2) block_attn_dq_kernel(const BlockAttnArgs a) {
    using vec8 = typename Elem<T>::vec8;
    constexpr int KD = DP / 16, DB = DP / 32, TILE = BaTile<DP>::BYTES;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    int *tiles = reinterpret_cast<int *>(smem + 4 * TILE);
    int *ntiles_p = tiles + 2 * BB_LIST;

    const int lin = (blockIdx.x & 7) * a.chunk + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= a.chunk || lin >= a.nblk) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, hi = lane >> 5;
    const int unit = lin / a.nsplit, sp = lin - unit * a.nsplit;
    const int g0 = unit % a.G, u = unit / a.G;
    const int qb = u % a.nQ, pair = u / a.nQ;
    const int hk = pair % a.Hk, b = pair / a.Hk, h = hk * a.G + g0;
    const int klen = a.klen ? min(max(a.klen[b], 0), a.Sk) : a.Sk;
    const int qlen = a.qlen ? min(max(a.qlen[b], 0), a.Sq) : a.Sq;
    const int s = qb * a.bq + wave * 32 + l31;
    const bool row_ok = s < qlen;

    const T *Qp = (const T *)a.q + (int64_t)b * a.qs[0] + (int64_t)s * a.qs[1] + (int64_t)h * a.qs[2];
    const T *Gp = (const T *)a.dout + (int64_t)b * a.dos[0] + (int64_t)s * a.dos[1] + (int64_t)h * a.dos[2];
    vec8 qf[KD], gf[KD];
#pragma unroll
    for (int kd = 0; kd < KD; ++kd) {
        const int d0 = kd * 16 + hi * 8;
        u32x4 x = {0u, 0u, 0u, 0u}, y = {0u, 0u, 0u, 0u};
        if (row_ok && d0 < a.D) {
            x = *reinterpret_cast<const u32x4 *>(Qp + d0);
            y = *reinterpret_cast<const u32x4 *>(Gp + d0);
        }
        qf[kd] = __builtin_bit_cast(vec8, x);
        gf[kd] = __builtin_bit_cast(vec8, y);
    }
    float L = INFINITY;  // a row without keys: probabilities 0
    u32x4 dparts = {0u, 0u, 0u, 0u};
    if (row_ok) {
        const float v = a.lse[((int64_t)b * a.H + h) * a.Sq + s];
        if (v != -INFINITY) L = v * LOG2E;
        const u32x4 parts = a.stat[((int64_t)b * a.H + h) * (a.nQ * a.bq) + s];
        if (hi == 0) dparts = u32x4{parts[2], parts[3], 0u, 0u};
    }
    const vec8 powers = bb_powers<T>(hi);
    const T *Kp = (const T *)a.k + (int64_t)b * a.ks[0] + (int64_t)hk * a.ks[2];
    const T *Vp = (const T *)a.v + (int64_t)b * a.vs[0] + (int64_t)hk * a.vs[2];
    BaLoader<DP, NW> kl, vl;
    kl.init(wave, lane, a.ks[1], a.D);
    vl.init(wave, lane, a.vs[1], a.D);
    f32x16 dq[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) dq[db][i] = 0.f;
    const float c = a.c;

    const int e_all = qb * a.bq < qlen ? (int)((int64_t)a.topk * (sp + 1) / a.nsplit) : 0;
    for (int e0 = (int)((int64_t)a.topk * sp / a.nsplit); e0 < e_all; e0 += BB_LIST) {
        __syncthreads();
        if (wave == 0) {
            const int n = ba_tiles(a.blocks + ((int64_t)pair * a.nQ + qb) * a.topk, e0, min(e0 + BB_LIST, e_all), a.bk, klen, lane, tiles);
            if (lane == 0) *ntiles_p = n;
        }
        __syncthreads();
        const int n = __builtin_amdgcn_readfirstlane(*ntiles_p);
        int next = n > 0 ? __builtin_amdgcn_readfirstlane(tiles[0]) : 0;
        if (n > 0) {
            kl.load(Kp, a.ks[1], a.D, next * 64, klen - next * 64, smem, wave);
            vl.load(Vp, a.vs[1], a.D, next * 64, klen - next * 64, smem + TILE, wave);
        }
        for (int t = 0; t < n; ++t) {
            const int cur = next;
            char *Ks = smem + (t & 1) * (2 * TILE), *Vs = Ks + TILE;
            if (t + 1 < n) next = __builtin_amdgcn_readfirstlane(tiles[t + 1]);
            ba_sync();
            if (t + 1 < n) {
                char *Kn = smem + ((t + 1) & 1) * (2 * TILE);
                kl.load(Kp, a.ks[1], a.D, next * 64, klen - next * 64, Kn, wave);
                vl.load(Vp, a.vs[1], a.D, next * 64, klen - next * 64, Kn + TILE, wave);
            }
            const int left = klen - cur * 64;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                // all fragments of a product are requested ahead of it, K^T's under the exponentials
                vec8 kf[KD], vf[KD], kt[2][DB];
#pragma unroll
                for (int kd = 0; kd < KD; ++kd) {
                    kf[kd] = ba_row_frag<T, DP>(Ks, kb * 32 + l31, kd, hi);
                    vf[kd] = ba_row_frag<T, DP>(Vs, kb * 32 + l31, kd, hi);
                }
                __builtin_amdgcn_sched_barrier(0);
                f32x16 sc, dp;
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = 0.f, dp[i] = 0.f;
                dp = ba_mfma(powers, __builtin_bit_cast(vec8, dparts), dp);  // dP - delta
#pragma unroll
                for (int kd = 0; kd < KD; ++kd) {
                    sc = ba_mfma(kf[kd], qf[kd], sc);
                    dp = ba_mfma(vf[kd], gf[kd], dp);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int db = 0; db < DB; ++db) kt[g][db] = ba_col_frag<T, DP>(Ks, lane, db, kb * 32 + g * 16);
                __builtin_amdgcn_sched_barrier(0);
                if (left < 64) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (kb * 32 + (i & 3) + 8 * (i >> 2) + 4 * hi >= left) sc[i] = -INFINITY;
                }
                BbRounded<T, FINE> ds[2];
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i >> 3].set(i & 7, __builtin_amdgcn_exp2f(fmaf(sc[i], c, -L)) * dp[i]);
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int db = 0; db < DB; ++db) dq[db] = ds[g].times(kt[g][db], dq[db]);
            }
        }
    }
    if (a.nsplit > 1) {
        float *po = a.part_o + ((int64_t)lin * (NW * 32) + wave * 32 + l31) * a.D;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = db * 32 + 8 * i + 4 * hi;
                if (d < a.D) *reinterpret_cast<f32x4 *>(po + d) = f32x4{dq[db][4 * i], dq[db][4 * i + 1], dq[db][4 * i + 2], dq[db][4 * i + 3]};
            }
        return;
    }
    if (s >= a.Sq) return;
    T *Op = (T *)a.dq + (int64_t)b * a.dqs[0] + (int64_t)s * a.dqs[1] + (int64_t)h * a.dqs[2];
    const float k = row_ok ? a.scale : 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = db * 32 + 8 * i + 4 * hi;
            if (d < a.D)
                *reinterpret_cast<u32x2 *>(Op + d) = pack4<T>(dq[db][4 * i] * k, dq[db][4 * i + 1] * k, dq[db][4 * i + 2] * k, dq[db][4 * i + 3] * k);
        }
}

// dK and dV of one key block: NW waves of 32 keys (K and V in registers as the lanes' columns), streaming 64-row tiles of Q and dO of the query
// blocks that name it, of all heads of the group
template <typename T, int DP, int NW, int RS, bool FINE>
__global__ void __launch_bounds__(NW * RS * 64, DP == 128 ? 1 : FINE ? 2 : RS + 1) block_attn_dkv_kernel(const BlockAttnArgs a) {
    using vec8 = typename Elem<T>::vec8;
    constexpr int KD = DP / 16, DB = DP / 32, TILE = BaTile<DP>::BYTES;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    char *const stat = smem + 4 * TILE;                           // two stages of 64 rows' parts
    int *names = reinterpret_cast<int *>(stat + 2 * 1024);        // query block, log2 of how often it names the key block
    int *n_p = names + 2 * BB_NAMES;

    const int lin = (blockIdx.x & 7) * a.chunk + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= a.chunk || lin >= a.nblk) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), l31 = lane & 31, hi = lane >> 5;
    const int piece = lin / a.nsplit, sp = lin - piece * a.nsplit;
    // a block's 128 keys may be two workgroups' work
    const int pieces = a.bk / (NW * 32), unit = piece / pieces, k0 = (piece - unit * pieces) * (NW * 32);
    const int j = unit % a.nK, pair = unit / a.nK;
    const int hk = pair % a.Hk, b = pair / a.Hk;
    const int klen = a.klen ? min(max(a.klen[b], 0), a.Sk) : a.Sk;
    const int qlen = a.qlen ? min(max(a.qlen[b], 0), a.Sq) : a.Sq;
    const int kw = RS == 1 ? wave : wave % NW, half = RS == 1 ? 0 : wave / NW;
    const int64_t first_key = (int64_t)j * a.bk + k0, key = first_key + kw * 32 + l31;
    const bool key_ok = key < klen;
    const int32_t *cnt = a.cnt + ((int64_t)pair * a.nK + j) * a.nQ;
    const int i_first = (int)((int64_t)a.nQ * sp / a.nsplit);
    int i_all = first_key < klen ? min((qlen + a.bq - 1) / a.bq, (int)((int64_t)a.nQ * (sp + 1) / a.nsplit)) : 0;
    // few query blocks leave most of a long cache unnamed: its keys are not read (3 x 13 heads of one token, 21108 keys of 80: 223 -> 127 us)
    if (i_all - i_first <= 64 && __ballot(i_first + lane < i_all && cnt[i_first + lane] > 0) == 0) i_all = 0;

    const T *Kp = (const T *)a.k + (int64_t)b * a.ks[0] + key * a.ks[1] + (int64_t)hk * a.ks[2];
    const T *Vp = (const T *)a.v + (int64_t)b * a.vs[0] + key * a.vs[1] + (int64_t)hk * a.vs[2];
    vec8 kf[KD], vf[KD];
#pragma unroll
    for (int kd = 0; kd < KD; ++kd) {
        const int d0 = kd * 16 + hi * 8;
        u32x4 x = {0u, 0u, 0u, 0u}, y = {0u, 0u, 0u, 0u};
        if (key_ok && i_all > 0 && d0 < a.D) {
            x = *reinterpret_cast<const u32x4 *>(Kp + d0);
            y = *reinterpret_cast<const u32x4 *>(Vp + d0);
        }
        kf[kd] = __builtin_bit_cast(vec8, x);
        vf[kd] = __builtin_bit_cast(vec8, y);
    }
    BaLoader<DP, NW * RS> ql, gl;
    ql.init(wave, lane, a.qs[1], a.D);
    gl.init(wave, lane, a.dos[1], a.D);
    const vec8 powers = bb_powers<T>(hi);
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) dk[db][i] = 0.f, dv[db][i] = 0.f;
    const float c = a.c;
    const int subs = a.bq >> 6;

    // the step that is requested next: entry e of the list (query block qb, log2 of its count), head g of the group, 64-row tile sub of the block
    int e = 0, g = 0, sub = 0, qb = 0, often = 0, entries = 0;
    const T *Qh = nullptr, *Gh = nullptr;  // the head's rows
    const u32x4 *Sh = nullptr;
    const auto entry = [&]() __attribute__((always_inline)) {
        qb = __builtin_amdgcn_readfirstlane(names[2 * e]), often = __builtin_amdgcn_readfirstlane(names[2 * e + 1]);
    };
    const auto first_head = [&]() __attribute__((always_inline)) {
        const int64_t h = (int64_t)hk * a.G;
        Qh = (const T *)a.q + (int64_t)b * a.qs[0] + h * a.qs[2];
        Gh = (const T *)a.dout + (int64_t)b * a.dos[0] + h * a.dos[2];
        Sh = a.stat + ((int64_t)b * a.H + h) * (a.nQ * a.bq);
    };
    const auto request = [&](int stage) __attribute__((always_inline)) {
        const int s0 = qb * a.bq + sub * 64;
        char *Qs = smem + stage * (2 * TILE);
        ql.load(Qh, a.qs[1], a.D, s0, qlen - s0, Qs, wave);
        gl.load(Gh, a.dos[1], a.D, s0, qlen - s0, Qs + TILE, wave);
        if (wave == NW * RS - 1) ba_dma(ba_rsrc(Sh + s0, 1024), (ba_lds_t)(stat + stage * 1024), lane * 16);
        if (++sub == subs) {
            sub = 0;
            if (++g == a.G) {
                g = 0, ++e;
                first_head();
                if (e < entries) entry();
            } else {
                Qh += a.qs[2], Gh += a.dos[2], Sh += a.nQ * a.bq;
            }
        }
    };

    for (int i0 = i_first; i0 < i_all; i0 += BB_NAMES) {
        __syncthreads();
        if (wave == 0) {
            int n = 0;
            for (int i = i0; i < min(i0 + BB_NAMES, i_all); i += 64) {
                const int m = i + lane < min(i0 + BB_NAMES, i_all) ? cnt[i + lane] : 0;
                const uint64_t some = __ballot(m > 0);
                const int at = n + __popcll(some & ((1ull << lane) - 1));
                if (m > 0) names[2 * at] = i + lane, names[2 * at + 1] = __float_as_int(__log2f((float)m));
                n += __popcll(some);
            }
            if (lane == 0) *n_p = n;
        }
        __syncthreads();
        entries = __builtin_amdgcn_readfirstlane(*n_p);
        const int steps = entries * (a.G * subs);
        e = 0, g = 0, sub = 0;
        first_head();
        int often_now = 0, often_next = 0;
        if (steps > 0) {
            entry();
            often_next = often;
            request(0);
        }
        for (int x = 0; x < steps; ++x) {
            const char *Qs = smem + (x & 1) * (2 * TILE), *Gs = Qs + TILE;
            const char *Ls = stat + (x & 1) * 1024;
            ba_sync();
            often_now = often_next, often_next = often;
            const float times = __int_as_float(often_now);  // exp2(x + times) = count exp2(x)
            if (x + 1 < steps) request((x + 1) & 1);
#pragma unroll
            for (int y = 0; y < 2 / RS; ++y) {
                const int rb = RS == 1 ? y : half;
                vec8 qf[KD], gt[2][DB];
#pragma unroll
                for (int kd = 0; kd < KD; ++kd) qf[kd] = ba_row_frag<T, DP>(Qs, rb * 32 + l31, kd, hi);
                const u32x4 parts = *reinterpret_cast<const u32x4 *>(Ls + (rb * 32 + l31) * 16);
                f32x16 sc, dp;
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = 0.f;
                // s - lse / scale
                sc = ba_mfma(__builtin_bit_cast(vec8, u32x4{hi ? 0u : parts[0], hi ? 0u : parts[1], 0u, 0u}), powers, sc);
#pragma unroll
                for (int kd = 0; kd < KD; ++kd) sc = ba_mfma(qf[kd], kf[kd], sc);
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int db = 0; db < DB; ++db) gt[g][db] = ba_col_frag<T, DP>(Gs, lane, db, rb * 32 + g * 16);
                BbRounded<T, FINE> p8[2], ds[2];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[i] = __builtin_amdgcn_exp2f(fmaf(sc[i], c, times));
                    p8[i >> 3].set(i & 7, sc[i]);
                }
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int db = 0; db < DB; ++db) dv[db] = p8[g].times(gt[g][db], dv[db]);
                vec8 gf[KD], qt[2][DB];
#pragma unroll
                for (int kd = 0; kd < KD; ++kd) gf[kd] = ba_row_frag<T, DP>(Gs, rb * 32 + l31, kd, hi);
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] = 0.f;
                // dP - delta
                dp = ba_mfma(__builtin_bit_cast(vec8, u32x4{hi ? 0u : parts[2], hi ? 0u : parts[3], 0u, 0u}), powers, dp);
#pragma unroll
                for (int kd = 0; kd < KD; ++kd) dp = ba_mfma(gf[kd], vf[kd], dp);
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int db = 0; db < DB; ++db) qt[g][db] = ba_col_frag<T, DP>(Qs, lane, db, rb * 32 + g * 16);
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i >> 3].set(i & 7, sc[i] * dp[i]);
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int db = 0; db < DB; ++db) dk[db] = ds[g].times(qt[g][db], dk[db]);
            }
        }
    }
    if constexpr (RS == 2) {
        // the second half's sums come through LDS (the stages are free)
        __syncthreads();
        float *const so = reinterpret_cast<float *>(smem) + kw * (2 * DB * 16 * 64) + lane;
        if (half == 1) {
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) so[(db * 16 + i) * 64] = dk[db][i], so[((DB + db) * 16 + i) * 64] = dv[db][i];
        }
        __syncthreads();
        if (half == 1) return;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) dk[db][i] += so[(db * 16 + i) * 64], dv[db][i] += so[((DB + db) * 16 + i) * 64];
    }
    if (a.nsplit > 1) {
        float *po = a.part_o + ((int64_t)lin * (NW * 32) + kw * 32 + l31) * (2 * a.D);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = db * 32 + 8 * i + 4 * hi;
                if (d < a.D) {
                    *reinterpret_cast<f32x4 *>(po + d) = f32x4{dk[db][4 * i], dk[db][4 * i + 1], dk[db][4 * i + 2], dk[db][4 * i + 3]};
                    *reinterpret_cast<f32x4 *>(po + a.D + d) = f32x4{dv[db][4 * i], dv[db][4 * i + 1], dv[db][4 * i + 2], dv[db][4 * i + 3]};
                }
            }
        return;
    }
    if (key >= a.Sk) return;
    T *Kg = (T *)a.dk + (int64_t)b * a.dks[0] + key * a.dks[1] + (int64_t)hk * a.dks[2];
    T *Vg = (T *)a.dv + (int64_t)b * a.dvs[0] + key * a.dvs[1] + (int64_t)hk * a.dvs[2];
    const float k = a.scale;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = db * 32 + 8 * i + 4 * hi;
            if (d < a.D) {
                u32x2 x = pack4<T>(dk[db][4 * i] * k, dk[db][4 * i + 1] * k, dk[db][4 * i + 2] * k, dk[db][4 * i + 3] * k);
                u32x2 y = pack4<T>(dv[db][4 * i], dv[db][4 * i + 1], dv[db][4 * i + 2], dv[db][4 * i + 3]);
                if (!key_ok) x = u32x2{0u, 0u}, y = u32x2{0u, 0u};  // a key behind the sequence
                *reinterpret_cast<u32x2 *>(Kg + d) = x;
                *reinterpret_cast<u32x2 *>(Vg + d) = y;
            }
        }
}

// the sum of a row's parts, four elements a thread (KV: a key's dk, then its dv)
template <typename T, bool KV> __global__ void __launch_bounds__(256) block_attn_add_parts_kernel(const BlockAttnArgs a, int rows, int n_rows) {
    const int runs = (KV ? 2 : 1) * a.D / 4;
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int row = (int)(id / runs), run = (int)(id - (int64_t)row * runs);
    if (row >= n_rows) return;
    const int unit = row / rows, r = row - unit * rows;  // a query block of a head | a piece of a key block
    int b, at, h, d = run * 4;
    bool there;
    if (KV) {
        const int pieces = a.bk / rows, block = unit / pieces, pair = block / a.nK;
        h = pair % a.Hk, b = pair / a.Hk, at = (block - pair * a.nK) * a.bk + (unit - block * pieces) * rows + r;
        if (at >= a.Sk) return;
        there = at < (a.klen ? min(max(a.klen[b], 0), a.Sk) : a.Sk);
    } else {
        const int g = unit % a.G, u = unit / a.G, qb = u % a.nQ, pair = u / a.nQ;
        h = pair % a.Hk * a.G + g, b = pair / a.Hk, at = qb * a.bq + r;
        if (at >= a.Sq) return;
        there = at < (a.qlen ? min(max(a.qlen[b], 0), a.Sq) : a.Sq);
    }
    const float *p = a.part_o + ((int64_t)unit * a.nsplit * rows + r) * (runs * 4) + d;
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < a.nsplit; ++i) sum += *reinterpret_cast<const f32x4 *>(p + (int64_t)i * rows * (runs * 4));
    const bool value = KV && d >= a.D;
    if (value) d -= a.D;
    const float k = value ? 1.f : a.scale;
    u32x2 x = pack4<T>(sum[0] * k, sum[1] * k, sum[2] * k, sum[3] * k);
    if (!there) x = u32x2{0u, 0u};  // behind the sequence
    T *out = (T *)(KV ? value ? a.dv : a.dk : a.dq);
    const int64_t *st = KV ? value ? a.dvs : a.dks : a.dqs;
    *reinterpret_cast<u32x2 *>(out + b * st[0] + at * st[1] + h * st[2] + d) = x;
}

// How the two products of a call are cut: nq, nk parts of a query block's list and of a key block's query blocks (their sums in fp32 meet in
// the workspace), few: 64 keys a workgroup and halved tiles.
struct BwdPlan {
    int nq, nk;
    bool few;
    int64_t units_q, units_k, part_floats;
};

// A workgroup's chain of tiles is the time where there are fewer workgroups than compute units: it is cut so that they fill them, into parts of
// eight tiles (about 10 us, against 5 for the second launch) and more. (24 heads of 16217 rows of 40 against one block of 120 keys: 372 -> 155 us;
// 4 x 2 heads of 56 rows of 96 against 47 blocks of 128: 208 -> 63.)
static BwdPlan bwd_plan(const sfast_block_attn_params *p) {
    BwdPlan pl{};
    const int64_t nQ = ceil_div(p->Sq, p->block_q), nK = ceil_div(p->Sk, p->block_k), G = p->H / p->Hk;
    const int64_t B = g_batch_ref > 0 ? g_batch_ref : p->B;  // (SFAST_BATCH_INVARIANT: a sample's parts are those of the reference batch, common.h)
    pl.few = B * p->Hk * nK * (p->block_k / 64) <= 256;
    pl.units_q = (int64_t)p->B * p->H * nQ, pl.units_k = (int64_t)p->B * p->Hk * nK * (pl.few ? p->block_k / 64 : 1);
    const auto parts = [&](int64_t units, int64_t steps, int64_t most) {
        const int64_t n = std::min(std::min(256 / std::max<int64_t>(units / p->B * B, 1), steps / 8), most);
        return (int)std::max<int64_t>(n, 1);
    };
    pl.nq = parts(pl.units_q, (int64_t)p->topk * (p->block_k / 64), p->topk);
    pl.nk = parts(pl.units_k, nQ * std::min<int64_t>(p->topk, nK) / nK * (p->block_q / 64) * G, nQ);
    const int64_t keys = pl.few ? 64 : p->block_k;
    pl.part_floats = std::max(pl.nq > 1 ? pl.units_q * pl.nq * p->block_q * p->D : 0, pl.nk > 1 ? pl.units_k * pl.nk * keys * 2 * p->D : 0);
    return pl;
}

template <typename T, int DP, bool FINE> int set_attr() {
    hipError_t e = hipSuccess;
    const auto one = [&](const void *kern, int bytes) {
        if (e == hipSuccess) e = hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    one((const void *)block_attn_dq_kernel<T, DP, 2, FINE>, bb_dq_lds<DP>());
    one((const void *)block_attn_dq_kernel<T, DP, 4, FINE>, bb_dq_lds<DP>());
    one((const void *)block_attn_dkv_kernel<T, DP, 2, bb_halves<DP>(), FINE>, bb_dkv_lds<DP>());
    one((const void *)block_attn_dkv_kernel<T, DP, 2, 2, FINE>, bb_dkv_lds<DP>());
    one((const void *)block_attn_dkv_kernel<T, DP, 4, 1, FINE>, bb_dkv_lds<DP>());
    if (e != hipSuccess) {
        set_error("hipFuncSetAttribute(block_attn_bwd): %s", hipGetErrorString(e));
        return SFAST_ERR_LAUNCH;
    }
    return 0;
}

template <typename T, int DP, bool FINE> int launch(BlockAttnArgs a, const BwdPlan &pl, hipStream_t st) {
    const int64_t cells = (int64_t)a.B * a.Hk * a.nK * a.nQ;
    const int64_t rows = (int64_t)a.nQ * a.bq * a.H;
    if (DP == 64)
        hipLaunchKernelGGL((block_attn_delta_kernel<T, 8>), dim3((unsigned)ceil_div64(rows, 32), a.B), dim3(256), 0, st, a, cells);
    else
        hipLaunchKernelGGL((block_attn_delta_kernel<T, 16>), dim3((unsigned)ceil_div64(rows, 16), a.B), dim3(256), 0, st, a, cells);
    int rc = check_launch("block_attention_backward delta");
    if (rc) return rc;
    hipLaunchKernelGGL(block_attn_count_kernel, dim3((unsigned)ceil_div(a.nQ * a.topk, 256), a.B * a.Hk), dim3(256), 0, st, a);
    rc = check_launch("block_attention_backward count");
    if (rc) return rc;
    const auto add_parts = [&](auto KV, int64_t units, int rows) {
        constexpr bool kv = decltype(KV)::value;
        const int n_rows = (int)(units * rows);
        const dim3 grid((unsigned)ceil_div64((int64_t)n_rows * ((kv ? 2 : 1) * a.D / 4), 256));
        hipLaunchKernelGGL((block_attn_add_parts_kernel<T, kv>), grid, dim3(256), 0, st, a, rows, n_rows);
        return check_launch("block_attention_backward add parts");
    };
    a.nsplit = pl.nq;
    a.nblk = (int)pl.units_q * pl.nq;
    a.chunk = ceil_div(a.nblk, 8);
    if (a.bq == 64)
        hipLaunchKernelGGL((block_attn_dq_kernel<T, DP, 2, FINE>), dim3(8 * a.chunk), dim3(128), bb_dq_lds<DP>(), st, a);
    else
        hipLaunchKernelGGL((block_attn_dq_kernel<T, DP, 4, FINE>), dim3(8 * a.chunk), dim3(256), bb_dq_lds<DP>(), st, a);
    rc = check_launch("block_attention_backward dq");
    if (!rc && pl.nq > 1) rc = add_parts(std::false_type{}, pl.units_q, a.bq);
    if (rc) return rc;
    // Where 64 keys a workgroup leave compute units free, the chain of a workgroup's steps is the time: blocks of 128 are two workgroups' work and
    // every tile's rows are halved (whole backward of 2 x 4 x 9 blocks of 128 keys of 64: 49 -> 42 us; of 8 x 16 blocks of 64 keys of 128: 57 ->
    // 46; of 8 x 16 blocks of 128 keys of 128: 98 -> 75).
    a.nsplit = pl.nk;
    a.nblk = (int)pl.units_k * pl.nk;
    a.chunk = ceil_div(a.nblk, 8);
    const auto dkv = [&](auto NW, auto RS) {
        constexpr int nw = decltype(NW)::value, rs = decltype(RS)::value;
        hipLaunchKernelGGL((block_attn_dkv_kernel<T, DP, nw, rs, FINE>), dim3(8 * a.chunk), dim3(nw * rs * 64), bb_dkv_lds<DP>(), st, a);
    };
    if (pl.few)
        dkv(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
    else if (a.bk == 64)
        dkv(std::integral_constant<int, 2>{}, std::integral_constant<int, bb_halves<DP>()>{});
    else
        dkv(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    rc = check_launch("block_attention_backward dkv");
    return rc || pl.nk == 1 ? rc : add_parts(std::true_type{}, pl.units_k, pl.few ? 64 : a.bk);
}

static int64_t padded_rows(const sfast_block_attn_params *p) { return (int64_t)p->B * p->H * ceil_div(p->Sq, p->block_q) * p->block_q; }
static int64_t cells(const sfast_block_attn_params *p) {
    return (int64_t)p->B * p->Hk * ceil_div(p->Sk, p->block_k) * ceil_div(p->Sq, p->block_q);
}

}  // namespace

int block_attn_bwd_init() {
    int rc = 0;
#define SFAST_BB_ATTR(T, DP)                           \
    if (!rc) rc = set_attr<T, DP, false>();            \
    if (!rc) rc = set_attr<T, DP, true>();
    SFAST_BB_ATTR(f16, 64)
    SFAST_BB_ATTR(f16, 128)
    SFAST_BB_ATTR(bf16, 64)
    SFAST_BB_ATTR(bf16, 128)
#undef SFAST_BB_ATTR
    return rc;
}

}  // namespace sfast

using namespace sfast;

extern "C" size_t sfast_hip_block_attention_backward_workspace_bytes(const sfast_block_attn_params *p) {
    if (block_attn_check(p) != SFAST_OK) return 0;
    return (size_t)padded_rows(p) * 16 + (size_t)(cells(p) + 3) / 4 * 16 + (size_t)bwd_plan(p).part_floats * 4;
}

extern "C" int sfast_hip_block_attention_backward(const void *q, const void *k, const void *v, const int32_t *blocks, const int32_t *key_lengths,
                                                  const int32_t *query_lengths, const void *out, const void *out_rest, const float *lse, const void *dout,
                                                  const float *dlse, void *dq, void *dk, void *dv, const sfast_block_attn_params *p,
                                                  void *workspace, size_t workspace_bytes, sfast_stream_t stream) {
    SFAST_REQUIRE(q && k && v && blocks && out && lse && dout && dq && dk && dv, SFAST_ERR_INVALID, "block_attention_backward: null argument");
    int rc = block_attn_check(p);
    if (rc != SFAST_OK) return rc;
    SFAST_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(out) && aligned16(out_rest) && aligned16(dout) && aligned8(dq) &&
                      aligned8(dk) && aligned8(dv),
                  SFAST_ERR_UNSUPPORTED, "block_attention_backward: operands must be 16-byte aligned");
    for (int i = 0; i < 3; ++i) {
        SFAST_REQUIRE(p->os[i] % 8 == 0 && p->dos[i] % 8 == 0 && p->os[i] >= 0 && p->dos[i] >= 0, SFAST_ERR_UNSUPPORTED,
                      "block_attention_backward: strides must be multiples of 8 elements");
        SFAST_REQUIRE(p->dqs[i] % 4 == 0 && p->dks[i] % 4 == 0 && p->dvs[i] % 4 == 0, SFAST_ERR_UNSUPPORTED,
                      "block_attention_backward: gradient strides must be multiples of 4 elements");
    }
    SFAST_REQUIRE(p->dos[1] >= p->D && p->dos[1] < (1 << 23), SFAST_ERR_UNSUPPORTED, "block_attention_backward: rows overlap, or their stride is too long");
    const BwdPlan pl = bwd_plan(p);
    SFAST_REQUIRE(fits_launch(pl.units_q * pl.nq + 7, 256) && fits_launch(pl.units_k * pl.nk + 7, 256) &&
                      fits_launch(padded_rows(p) / p->B / 16 + 1, 256) && p->B <= 65535 && (int64_t)p->B * p->Hk <= 65535 &&
                      (int64_t)ceil_div(p->Sq, p->block_q) * p->topk <= (1ll << 30),
                  SFAST_ERR_UNSUPPORTED, "block_attention_backward: too many rows");
    SFAST_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= sfast_hip_block_attention_backward_workspace_bytes(p), SFAST_ERR_WORKSPACE,
                  "block_attention_backward: workspace too small");
    BlockAttnArgs a{};
    a.q = q, a.k = k, a.v = v, a.o = out, a.o_rest = out_rest, a.dout = dout, a.lse = const_cast<float *>(lse), a.dlse = dlse, a.dq = dq, a.dk = dk, a.dv = dv;
    a.blocks = blocks, a.klen = key_lengths, a.qlen = query_lengths;
    a.stat = (u32x4 *)workspace;
    a.cnt = (int32_t *)(a.stat + padded_rows(p));
    a.part_o = (float *)(a.cnt + (cells(p) + 3) / 4 * 4);
    a.B = p->B, a.H = p->H, a.Hk = p->Hk, a.G = p->H / p->Hk, a.Sq = p->Sq, a.Sk = p->Sk, a.D = p->D, a.topk = p->topk;
    a.bq = p->block_q, a.bk = p->block_k, a.nQ = ceil_div(p->Sq, p->block_q), a.nK = ceil_div(p->Sk, p->block_k);
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = p->qs[i], a.ks[i] = p->ks[i], a.vs[i] = p->vs[i], a.os[i] = p->os[i], a.dos[i] = p->dos[i];
        a.dqs[i] = p->dqs[i], a.dks[i] = p->dks[i], a.dvs[i] = p->dvs[i];
    }
    a.scale = p->scale;
    a.c = p->scale * LOG2E;
    hipStream_t st = (hipStream_t)stream;
    const bool fine = a.nQ == 1 || a.nK == 1;
    const int dp = p->D <= 64 ? 64 : 128;
    set_kernel_name("block_attn_bwd[DP=%d,rows=%d,keys=%d,halves=%d,parts=%d+%d%s]", dp, a.bq, pl.few ? 64 : a.bk,
                    pl.few ? 2 : a.bk == 64 ? (dp == 64 ? bb_halves<64>() : bb_halves<128>()) : 1, pl.nq, pl.nk, fine ? ",fine" : "");
#define SFAST_BB(T)                                                                    \
    if (p->D <= 64) return fine ? launch<T, 64, true>(a, pl, st) : launch<T, 64, false>(a, pl, st); \
    return fine ? launch<T, 128, true>(a, pl, st) : launch<T, 128, false>(a, pl, st);
    if (p->dtype == SFAST_F16) { SFAST_BB(f16) }
    SFAST_BB(bf16)
#undef SFAST_BB
}
