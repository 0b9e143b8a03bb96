// Shared by block_attn.hip (attention over chosen key blocks: forward, split form) and block_attn_bwd.hip (its gradients): arguments, the
// LDS image of a 64-row tile, MFMA operand reads.
//
// All products are 32x32x16 MFMAs in "swapped" form: the result tile holds the streamed rows (keys in the forward) along its registers and
// the wave's own rows (queries) along its lanes -- S^T = K . Q^T -- so that a row's statistics live in one lane pair (lane, lane ^ 32) and
// the probabilities come out in the layout that the second product reads as its B operand: register j of 16-row group g of a lane in
// half hi is streamed row 16 g + (j & 3) + 8 (j >> 2) + 4 hi. The A operand of the second product (V^T: 16 streamed rows of one head-dim
// column per lane pair) uses the same order of rows, read straight from the row-major tile with the transposing 8-byte LDS read.
#pragma once
#include "common.h"
#include <math.h>

namespace sfast {

struct BlockAttnArgs {
    const void *q, *k, *v, *dout, *o, *o_rest;
    void *out, *out_rest, *dq, *dk, *dv;  // out_rest: what the rounding of out left, or NULL
    float *lse;                // [B, H, Sq], natural log
    const float *dlse;         // gradient of lse, or NULL
    const int32_t *blocks;     // [B, Hk, nQ, topk]
    const int32_t *klen, *qlen;  // [B] or NULL
    u32x4 *stat;               // backward: [B, H, nQ * bq] a row's lse and delta = rowsum(dout * o) - dlse as parts (block_attn_bwd.hip)
    int32_t *cnt;              // backward: [B, Hk, nK, nQ] how often query block i names key block j
    float *part_o, *part_ml;   // split form: unnormalised partial results, (reference, sum) pairs
    int B, H, Hk, G, Sq, Sk, D, nQ, nK, topk, bq, bk, nsplit;
    int64_t qs[3], ks[3], vs[3], os[3], dos[3], dqs[3], dks[3], dvs[3];  // element strides (b, s, h), head-dim stride 1
    float c;                   // scale * log2(e): probabilities are exp2(c * s - m)
    float scale;
    int nblk, chunk;           // workgroups of work, workgroups given to one XCD
};

typedef __attribute__((address_space(3))) void *ba_lds_t;

__device__ __forceinline__ f32x16 ba_mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 ba_mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// A 64-row x DP tile in LDS: rows of DP * 2 bytes without padding (LDS-DMA writes 1 KB runs), 16-byte chunks XOR-permuted inside a row.
// The permutation spreads both reads over the 64 banks: 16 rows at one chunk (operand reads, 16 bytes a lane) and 4 consecutive rows at two
// neighbouring chunk pairs (transposing reads, 8 bytes a lane).
template <int DP> struct BaTile {
    static_assert(DP == 64 || DP == 128, "head dims are padded to 64 or 128");
    static constexpr int CH = DP / 8;
    static constexpr int BYTES = 64 * DP * 2;
    static __device__ __forceinline__ int swz(int row) {
        return DP == 128 ? (((row & 3) << 2) | ((row >> 2) & 3)) : ((((row >> 1) & 1) << 2) | (((row >> 2) & 1) << 1) | ((row >> 3) & 1));
    }
    static __device__ __forceinline__ int off(int row, int chunk) { return row * (DP * 2) + ((chunk ^ swz(row)) << 4); }
};

// 16-byte operand fragment: row `row`, head-dim elements kd * 16 + hi * 8 .. + 7
template <typename T, int DP> __device__ __forceinline__ typename Elem<T>::vec8 ba_row_frag(const char *tile, int row, int kd, int hi) {
    return *reinterpret_cast<const typename Elem<T>::vec8 *>(tile + BaTile<DP>::off(row, kd * 2 + hi));
}

typedef short ba_s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) ba_s4 *ba_tr_ptr;
// transposing read: lane l of the wave gets head-dim column db * 32 + (l & 31) of the streamed rows row0 + 4 hi + 0 .. 3 (inside a
// 16-lane group, result lane 4 a + b receives element b of source lanes a, a + 4, a + 8, a + 12: source lane s supplies four columns of row s >> 2)
template <int DP> __device__ __forceinline__ int ba_tr_off(int lane, int db, int row0) {
    const int s = lane & 15, gl = lane >> 4;
    const int row = row0 + 4 * (gl >> 1) + (s >> 2);
    const int chunk = db * 4 + (gl & 1) * 2 + ((s & 3) >> 1);
    return BaTile<DP>::off(row, chunk) + (s & 1) * 8;
}
// (`tile` is __restrict__ so that the compiler does not order the read behind the LDS-DMA requests for the OTHER stage: without it every
// transposing read waits for all of them; ba_sync() orders the stages)
// A operand (head-dim columns db * 32 + (lane & 31)) x (16 streamed rows from row0, in the order of the probabilities)
template <typename T, int DP> __device__ __forceinline__ typename Elem<T>::vec8 ba_col_frag(const char *__restrict__ tile, int lane, int db, int row0) {
    const ba_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ba_tr_ptr)(tile + ba_tr_off<DP>(lane, db, row0)));
    const ba_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((ba_tr_ptr)(tile + ba_tr_off<DP>(lane, db, row0 + 8)));
    typedef short s8 __attribute__((ext_vector_type(8)));
    const s8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(typename Elem<T>::vec8, both);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t ba_rsrc(const void *base, uint32_t bytes) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)base);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uintptr_t)base >> 32));
    return __builtin_amdgcn_make_buffer_rsrc((void *)(((uintptr_t)hi << 32) | lo), 0, (int)__builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

__device__ __forceinline__ void ba_dma(const __amdgpu_buffer_rsrc_t rsrc, ba_lds_t dst, uint32_t off) {  // 16 bytes a lane
#ifdef __HIP_DEVICE_COMPILE__  // (the host pass refuses gfx950's 16-byte form)
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, dst, 16, off, 0, 0, 0);
#endif
}

// One matrix's share of a tile load: NW waves move 64 rows x DP elements from memory to LDS (16 bytes a lane, 1 KB an instruction). Rows
// behind the last valid one and head-dim elements behind D lie outside the buffer descriptor and arrive as zeros. A tile's base address
// is 64-bit (its own descriptor), so a cache may be longer than 4 GB; inside a tile offsets have 32 bits.
template <int DP, int NW> struct BaLoader {
    static constexpr int N = BaTile<DP>::CH / NW;
    static_assert(N >= 1, "");
    uint32_t voff[N];
    __device__ __forceinline__ void init(int wave, int lane, int64_t stride, int D) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int slot = (i * NW + wave) * 64 + lane;
            const int row = slot / BaTile<DP>::CH, chunk = (slot % BaTile<DP>::CH) ^ BaTile<DP>::swz(row);
            voff[i] = chunk * 8 < D ? (uint32_t)row * (uint32_t)stride * 2u + (uint32_t)chunk * 16u : 0x80000000u;
        }
    }
    __device__ __forceinline__ void load(const void *base, int64_t stride, int D, int row0, int rows, char *lds, int wave) const {
        rows = min(rows, 64);
        const uint32_t bytes = rows > 0 ? ((uint32_t)(rows - 1) * (uint32_t)stride + (uint32_t)D) * 2u : 0u;
        const __amdgpu_buffer_rsrc_t r = ba_rsrc((const char *)base + (int64_t)row0 * stride * 2, bytes);
#pragma unroll
        for (int i = 0; i < N; ++i)
            ba_dma(r, (ba_lds_t)(lds + (i * NW + wave) * 1024), voff[i]);
    }
};

__device__ __forceinline__ float ba_xor32_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const uint32_t x = r[0], y = r[1];
    return fmaxf(__uint_as_float(x), __uint_as_float(y));
}
__device__ __forceinline__ float ba_xor32_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const uint32_t x = r[0], y = r[1];
    return __uint_as_float(x) + __uint_as_float(y);
}

// Every wave's LDS-DMA requests have landed and every wave is done reading what the next requests overwrite. (The compiler's barrier waits
// for LDS operations, not for LDS-DMA: that wait is spelled out.)
// LEFT: requests of this wave that may still be on their way (they return in order).
template <int LEFT = 0> __device__ __forceinline__ void ba_sync() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT > 63 ? 63 : LEFT) : "memory");
    __syncthreads();
}

// the tiles (64 keys each) that the entries [e0, e1) of one list name, in the order of the list, into LDS; entries outside the sequence
// name nothing. Run by one wave; returns their number.
__device__ __forceinline__ int ba_tiles(const int32_t *list, int e0, int e1, int bk, int klen, int lane, int *tiles) {
    int n = 0;
    const int sub = bk >> 6;
#pragma unroll 1
    for (int e = e0; e < e1; e += 64) {
        const int j = e + lane < e1 ? list[e + lane] : -1;
        const int64_t first = (int64_t)j * bk;
        const bool one = j >= 0 && first < klen, two = one && sub == 2 && first + 64 < klen;
        const uint64_t m1 = __ballot(one), m2 = __ballot(two), below = (1ull << lane) - 1;
        int at = n + __popcll(m1 & below) + __popcll(m2 & below);
        if (one) tiles[at] = j * sub;
        if (two) tiles[at + 1] = j * sub + 1;
        n += __popcll(m1) + __popcll(m2);
    }
    return n;
}

int block_attn_check(const sfast_block_attn_params *p);  // what both calls ask of their parameters
int block_attn_init();
int block_attn_bwd_init();

}  // namespace sfast
