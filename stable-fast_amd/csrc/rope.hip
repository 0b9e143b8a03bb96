// Rotary positions with several axes (sfast_hip_rope_nd): q and k of a call in one launch, forward and (inverse = 1) backward.
//
// Pair (x0, x1) of a token turns by its axis' position times theta^(-2 i / d): y0 = x0 cos - x1 sin, y1 = x0 sin + x1 cos. Nothing but
// reading and writing q and k once costs anything: a workgroup makes the table of its tokens' cosines and sines in LDS -- once per token and
// pair, for all heads of q and k -- in 64 bits (an angle of 10^6 radians keeps 10 digits), rounded to fp32 once, and then streams rows
// through registers, four in flight a thread.
//
// Bound by memory (bf16, q and k): 57600 tokens x 24 heads of 128 take 265 us, 5.3 TB/s (a copy reaches 4.9); with section widths that allow
// no run longer than a pair 307 us; 10 heads of 64 leave few rows to a token's table, 64 us, 4.6 TB/s (95 in single pairs). No
// thread divides 64-bit numbers: a workgroup's tokens belong to one sequence (with a division a token those 64 us are 89). 4 tokens of 24 + 8
// heads are a launch.
// Tried: rows of all tokens flattened with the first loads ahead of the table (the table is then read per row: 335 and 92 us); four tokens in
// flight (247 us, but 75 for the heads of 64 and 330 in single pairs: its registers cost waves).
#include "common.h"
#include <math.h>

namespace sfast {

namespace {

constexpr int ROPE_MAX_PAIRS = 128, ROPE_MAX_TOK = 4;

struct RopeArgs {
    const void *q, *k, *pos;
    void *qo, *ko;
    int B, S, H, Hk, D, pairs;   // pairs = D / 2; those behind the sections are copied
    int n_axes, pos_type, inverse;
    int half0[5];                // first pair of axis a's section (half0[n_axes] = rotated pairs), tail included as a last section
    int64_t qs[3], ks[3], qos[3], kos[3], ps[2];
    int tok, chunks;             // tokens of a workgroup (of one sequence), workgroups of a sequence
    double turn[ROPE_MAX_PAIRS]; // theta^(-2 i / d) / (2 pi) of every pair: angles in turns
};

__device__ __forceinline__ double rope_pos(const void *p, int type, int64_t i) {
    switch (type) {
    case SFAST_POS_I32: return (double)((const int32_t *)p)[i];
    case SFAST_POS_I64: return (double)((const int64_t *)p)[i];
    case SFAST_POS_F32: return (double)((const float *)p)[i];
    default: return ((const double *)p)[i];
    }
}

template <typename T, int V> struct alignas(sizeof(T) * V) RopeVec {
    T e[V];
};

// V pairs a thread: one run of 2 V elements (INTER) or two runs of V elements, half a section apart. TAIL: there are elements behind the
// sections, whose bits are copied (a turn by 0 would carry an infinity to its neighbour). Without one nothing is selected: 10 heads of 64 take
// 62 us, with the selection 70.
template <typename T, int V, bool INTER, bool TAIL> __global__ void __launch_bounds__(256) rope_kernel(const RopeArgs a) {
    __shared__ float2 table[ROPE_MAX_TOK * ROPE_MAX_PAIRS];
    const int tid = threadIdx.x;
    const int b = (int)(blockIdx.x / (uint32_t)a.chunks), s0 = (int)(blockIdx.x - (uint32_t)b * a.chunks) * a.tok;
    const int ntok = min(a.tok, a.S - s0);
    for (int i = tid; i < ntok * a.pairs; i += 256) {
        const int t = i / a.pairs, p = i - t * a.pairs;
        float2 cs = make_float2(1.f, 0.f);
        if (p < a.half0[a.n_axes]) {
            int axis = 0;
#pragma unroll
            for (int x = 1; x < SFAST_ROPE_MAX_AXES; ++x) axis += x < a.n_axes && p >= a.half0[x];
            const double x = rope_pos(a.pos, a.pos_type, b * a.ps[0] + (s0 + t) * a.ps[1] + axis) * a.turn[p];
            double sn, c;
            sincospi(2.0 * (x - rint(x)), &sn, &c);
            cs = make_float2((float)c, a.inverse ? (float)-sn : (float)sn);
        }
        table[t * a.pairs + p] = cs;
    }
    __syncthreads();

    const int items = a.pairs / V, rpp = 256 / items;  // items of a row; rows the workgroup moves at a time (items <= 128)
    const int row0 = tid / items, item = tid - row0 * items;
    if (row0 >= rpp) return;
    const int p0 = item * V;
    int off0, off1 = 0;
    if (INTER) {
        off0 = p0 * 2;
    } else {
        // the section that holds pair p0 (a tail behind the last axis is a section of its own)
        int first = 0, next = a.half0[1];
#pragma unroll
        for (int x = 1; x <= SFAST_ROPE_MAX_AXES; ++x)
            if (x <= a.n_axes && p0 >= a.half0[x]) first = a.half0[x], next = x < a.n_axes ? a.half0[x + 1] : a.pairs;
        off0 = 2 * first + (p0 - first);
        off1 = off0 + (next - first);
    }
    const int heads = a.H + a.Hk, rotated = a.half0[a.n_axes];
    for (int t = 0; t < ntok; ++t) {
        const int s = s0 + t;
        const T *Q = (const T *)a.q + b * a.qs[0] + s * a.qs[1], *K = (const T *)a.k + b * a.ks[0] + s * a.ks[1];
        T *Qo = (T *)a.qo + b * a.qos[0] + s * a.qos[1], *Ko = (T *)a.ko + b * a.kos[0] + s * a.kos[1];
        float2 cs[V];
#pragma unroll
        for (int i = 0; i < V; ++i) cs[i] = table[t * a.pairs + p0 + i];
        for (int h0 = row0; h0 < heads; h0 += 4 * rpp) {
            RopeVec<T, INTER ? 2 * V : V> x0[4], x1[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int h = h0 + j * rpp;
                if (h >= heads) break;
                const T *row = h < a.H ? Q + h * a.qs[2] : K + (h - a.H) * a.ks[2];
                x0[j] = *reinterpret_cast<const RopeVec<T, INTER ? 2 * V : V> *>(row + off0);
                if (!INTER) x1[j] = *reinterpret_cast<const RopeVec<T, INTER ? 2 * V : V> *>(row + off1);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int h = h0 + j * rpp;
                if (h >= heads) break;
                T *row = h < a.H ? Qo + h * a.qos[2] : Ko + (h - a.H) * a.kos[2];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    T &r0 = INTER ? x0[j].e[2 * i] : x0[j].e[i], &r1 = INTER ? x0[j].e[2 * i + 1] : x1[j].e[i];
                    const float u = (float)r0, v = (float)r1;
                    const T y0 = Elem<T>::from_f32(fmaf(u, cs[i].x, -v * cs[i].y)), y1 = Elem<T>::from_f32(fmaf(u, cs[i].y, v * cs[i].x));
                    const bool turns = !TAIL || p0 + i < rotated;
                    r0 = turns ? y0 : r0, r1 = turns ? y1 : r1;
                }
                *reinterpret_cast<RopeVec<T, INTER ? 2 * V : V> *>(row + off0) = x0[j];
                if (!INTER) *reinterpret_cast<RopeVec<T, INTER ? 2 * V : V> *>(row + off1) = x1[j];
            }
        }
    }
}

template <typename T, int V> static int launch(const RopeArgs &a, bool inter, hipStream_t st) {
    const dim3 grid((unsigned)(a.B * a.chunks));
    const bool tail = a.half0[a.n_axes] < a.pairs;
    constexpr int MOST = 16 / sizeof(T);  // elements of one access
    if constexpr (2 * V <= MOST) {
        if (inter && tail)
            hipLaunchKernelGGL((rope_kernel<T, V, true, true>), grid, dim3(256), 0, st, a);
        else if (inter)
            hipLaunchKernelGGL((rope_kernel<T, V, true, false>), grid, dim3(256), 0, st, a);
    }
    if constexpr (V <= MOST) {
        if (!inter && tail)
            hipLaunchKernelGGL((rope_kernel<T, V, false, true>), grid, dim3(256), 0, st, a);
        else if (!inter)
            hipLaunchKernelGGL((rope_kernel<T, V, false, false>), grid, dim3(256), 0, st, a);
    }
    return check_launch("rope_nd");
}

}  // namespace

}  // namespace sfast

using namespace sfast;

extern "C" int sfast_hip_rope_nd(const void *q, const void *k, const void *positions, void *q_out, void *k_out, const sfast_rope_params *p,
                                 sfast_stream_t stream) {
    SFAST_REQUIRE(p && q && positions && q_out, SFAST_ERR_INVALID, "rope_nd: null argument");
    SFAST_REQUIRE(p->B > 0 && p->S > 0 && p->H > 0 && p->Hk >= 0 && p->D > 0, SFAST_ERR_INVALID, "rope_nd: bad shape");
    SFAST_REQUIRE(p->Hk == 0 || (k && k_out), SFAST_ERR_INVALID, "rope_nd: null key tensor");
    SFAST_REQUIRE(p->D % 2 == 0 && p->D <= 2 * ROPE_MAX_PAIRS, SFAST_ERR_UNSUPPORTED, "rope_nd: head dim %d (even, up to %d)", p->D, 2 * ROPE_MAX_PAIRS);
    SFAST_REQUIRE(p->n_axes >= 1 && p->n_axes <= SFAST_ROPE_MAX_AXES, SFAST_ERR_UNSUPPORTED, "rope_nd: %d axes (1 to %d)", p->n_axes, SFAST_ROPE_MAX_AXES);
    SFAST_REQUIRE(p->dtype == SFAST_F16 || p->dtype == SFAST_BF16 || p->dtype == SFAST_F32, SFAST_ERR_UNSUPPORTED, "rope_nd: bad dtype %d", p->dtype);
    SFAST_REQUIRE(p->pos_type >= SFAST_POS_I32 && p->pos_type <= SFAST_POS_F64, SFAST_ERR_UNSUPPORTED, "rope_nd: bad position type %d", p->pos_type);
    SFAST_REQUIRE(p->theta > 0.0 && p->theta < INFINITY, SFAST_ERR_INVALID, "rope_nd: theta must be positive and finite");
    const int es = (int)dtype_bytes(p->dtype);
    RopeArgs a{};
    a.q = q, a.k = k, a.pos = positions, a.qo = q_out, a.ko = k_out;
    a.B = p->B, a.S = p->S, a.H = p->H, a.Hk = p->Hk, a.D = p->D, a.pairs = p->D / 2;
    a.n_axes = p->n_axes, a.pos_type = p->pos_type, a.inverse = p->inverse;
    // V pairs a thread: 16 bytes in one access (neighbouring pairs) or in each of two (halves). Shorter runs where a section, a stride or an
    // address does not allow that.
    int run = 16 / es;  // elements of one access
    const auto fits = [&](int64_t v) { while (run > 1 && v % run) run >>= 1; };
    int at = 0;
    const double octaves = log2(p->theta);
    for (int x = 0; x < p->n_axes; ++x) {
        const int d = p->sections[x];
        SFAST_REQUIRE(d > 0 && d % 2 == 0 && d <= p->D - at, SFAST_ERR_INVALID, "rope_nd: section %d has %d of %d elements left (even, positive)", x, d,
                      p->D - at);
        a.half0[x] = at / 2;
        for (int i = 0; i < d / 2; ++i) a.turn[at / 2 + i] = exp2(-2.0 * i / d * octaves) * (0.5 / M_PI);
        if (!p->interleaved) fits(d / 2);
        at += d;
    }
    a.half0[p->n_axes] = at / 2;
    if (!p->interleaved) fits((p->D - at) / 2);
    fits(p->D);
    const auto base = [&](const void *ptr) { while (run > 1 && ((uintptr_t)ptr) % (run * es)) run >>= 1; };
    base(q), base(q_out);
    if (p->Hk) base(k), base(k_out);
    for (int i = 0; i < 3; ++i) {
        fits(p->qs[i]), fits(p->qos[i]);
        if (p->Hk) fits(p->ks[i]), fits(p->kos[i]);
        a.qs[i] = p->qs[i], a.ks[i] = p->ks[i], a.qos[i] = p->qos[i], a.kos[i] = p->kos[i];
    }
    SFAST_REQUIRE(!p->interleaved || run >= 2, SFAST_ERR_UNSUPPORTED, "rope_nd: neighbouring pairs need addresses and strides of whole pairs");
    a.ps[0] = p->ps[0], a.ps[1] = p->ps[1];
    // tokens of a workgroup: enough to give every thread a table entry, few enough to leave eight workgroups for each compute unit
    a.tok = 1;
    while (a.tok < ROPE_MAX_TOK && a.tok < p->S && (int64_t)p->B * p->S / (2 * a.tok) >= 2048) a.tok *= 2;
    a.chunks = (int)ceil_div64(p->S, a.tok);
    SFAST_REQUIRE(fits_launch((int64_t)p->B * a.chunks, 256), SFAST_ERR_UNSUPPORTED, "rope_nd: too many tokens");
    hipStream_t st = (hipStream_t)stream;
    const int v = p->interleaved ? run / 2 : run;
    set_kernel_name("rope_nd[%s,V=%d]", p->interleaved ? "pairs" : "halves", v);
#define SFAST_ROPE(T)                                         \
    switch (v) {                                              \
    case 8: return launch<T, 8>(a, p->interleaved, st);       \
    case 4: return launch<T, 4>(a, p->interleaved, st);       \
    case 2: return launch<T, 2>(a, p->interleaved, st);       \
    default: return launch<T, 1>(a, p->interleaved, st);      \
    }
    if (p->dtype == SFAST_F16) { SFAST_ROPE(f16) }
    if (p->dtype == SFAST_BF16) { SFAST_ROPE(bf16) }
    SFAST_ROPE(float)
#undef SFAST_ROPE
}
