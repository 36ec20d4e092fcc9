// Tiles and arguments shared by the differential-attention kernels (forward and backward).
#pragma once
#include "blk_common.h"

namespace ndb {

// A tile of ROWS rows of RB bytes in LDS, filled by loads that go straight there (16 bytes a lane).  Piece c of row r lies at
// c ^ swz(r): 16 rows read at one piece (row fragments) cover all 64 banks, and so do the 4 rows x 64 bytes of a transposed
// bf16 read or the two rows of a column read in fp32.
template <typename T, int RB>
struct Tile {
    static constexpr int ES = (int)sizeof(T);

    static __device__ __forceinline__ int swz(int r) {
        if constexpr (ES == 2 && RB == 128) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        if constexpr (ES == 2) return ((r & 3) << 2) | ((r >> 2) & 3);
        return (((r >> 2) & 1) << 3) | (((r >> 3) & 1) << 2) | (r & 3);
    }

    // Lane bases.  Everything else of an address is a constant: an exclusive-or in the bits of the piece and an offset.
    // row(): piece c + lh of row r0 + l31 (c even, r0 a multiple of 32)
    static __device__ __forceinline__ int row_base(int lane) { return (lane & 31) * RB + ((swz(lane & 31) ^ (lane >> 5)) << 4); }
    static __device__ __forceinline__ u32x4 row(const char* t, int base, int r0, int c) {
        return *reinterpret_cast<const u32x4*>(t + (base ^ ((c & 15) << 4)) + (c >> 4) * 256 + r0 * RB);
    }

    // columns: bf16 cols(): lane (d = col + l31) gets rows r0 + 4 lh + 0 .. 3 and r0 + 8 + 4 lh + 0 .. 3 (the k order in which an
    // accumulator's registers serve as the other operand); fp32 one(): row r0 + (e & 3) + 8 (e >> 2) + 4 lh.  col a multiple of
    // 32, r0 of 16 (bf16) / 32.
    static __device__ __forceinline__ int col_base(int lane) {
        const int lh = lane >> 5;
        if constexpr (ES == 2) {
            const int i = lane & 15, r = 4 * lh + (i >> 2);
            return r * RB + ((((lane & 16) / 8 + ((i & 3) >> 1)) ^ swz(r)) << 4) + (i & 1) * 8;
        }
        return 4 * lh * RB + ((((lane & 31) >> 2) ^ swz(4 * lh)) << 4) + (lane & 3) * 4;
    }
    static __device__ __forceinline__ u32x4 cols(const char* t, int base, int r0, int col) {
        u32x4 v;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const char* a = t + (base ^ (((col / 8 & 15) ^ (2 * h)) << 4)) + (col / 128) * 256 + (r0 + 8 * h) * RB;
            union { s16x4 h4; unsigned u[2]; } c;
            c.h4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
            v[2 * h] = c.u[0], v[2 * h + 1] = c.u[1];
        }
        return v;
    }
    static __device__ __forceinline__ float one(const char* t, int base, int r0, int e, int col) {
        const int r = (e & 3) + 8 * (e >> 2);
        return *reinterpret_cast<const float*>(t + (base ^ (((col / 4 & 15) ^ swz(r)) << 4)) + (col / 64) * 256 + (r0 + r) * RB);
    }
};

// keep the addresses made from a lane base inside the loop: hoisted, they would take a register each
__device__ __forceinline__ int in_loop(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// this wave's share of filling such a tile
template <typename T, int RB, int ROWS, int NW>
struct TileLoad {
    static constexpr int PPR = RB / 16, NI = ROWS * PPR / 64 / NW;
    static_assert(NI >= 1 && NI * 64 * NW == ROWS * PPR, "the waves share the pieces evenly");
    unsigned off[NI];

    // rows of two halves of HB bytes in LDS (HB = RB: one), of which `dim` bytes each are real and lie side by side in memory
    template <int HB>
    __device__ __forceinline__ void init(int64_t stride_b, int dim, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int lin = (i * NW + wave) * 64 + lane, r = lin / PPR, c = (lin % PPR) ^ Tile<T, RB>::swz(r);
            const int half = c * 16 / HB, in = c * 16 - half * HB;
            off[i] = in < dim ? (unsigned)(r * stride_b) + (unsigned)(half * dim + in) : 0xfffffff0u;
        }
    }
    // `left`: bytes from base to the end of the rows that count; pieces past it become zero (buffer range check)
    __device__ __forceinline__ void load(char* t, const void* base, int64_t left, int wave) const {
        const uint64_t n = left < 0 ? 0 : (left < 0xfffffff0LL ? (uint64_t)left : 0xfffffff0ull);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)(unsigned)n, 0x00020000);
#pragma unroll
        for (int i = 0; i < NI; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(t + (i * NW + wave) * 1024), 16, (int)off[i], 0, 0, 0);
    }
};

// one 32 x 32 block of weights (rows: what is summed over, columns: a lane's own) as the second operand of a product
template <typename T>
struct Probs;
template <>
struct Probs<__bf16> {
    bf16x8 f[2];
    __device__ __forceinline__ void set(int e, float v) { f[e >> 3][e & 7] = (__bf16)v; }
    // the sum of what the product multiplies
    __device__ __forceinline__ float sum() const {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bf16x2 one = {(__bf16)1.f, (__bf16)1.f}, p = {f[i >> 2][2 * (i & 3)], f[i >> 2][2 * (i & 3) + 1]};
            t = __builtin_amdgcn_fdot2_f32_bf16(p, one, t, false);
        }
        return t;
    }
};
template <>
struct Probs<float> {
    float f[16];
    __device__ __forceinline__ void set(int e, float v) { f[e] = v; }
    __device__ __forceinline__ float sum() const {
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) t += f[i];
        return t;
    }
};

// acc[d][column] += sum over the 32 rows r0 .. of tile[row][col0 + d] * p[row][column]
template <typename T, int RB>
__device__ __forceinline__ f32x16 mma_cols(const char* t, int base, int r0, int col, const Probs<T>& p, f32x16 acc) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            union { u32x4 u; bf16x8 h; } a;
            a.u = Tile<T, RB>::cols(t, base, r0 + 16 * s, col);
            acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, p.f[s], acc, 0, 0, 0);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(Tile<T, RB>::one(t, base, r0, e, col), p.f[e], acc, 0, 0, 0);
    }
    return acc;
}

struct DiffTensor {       // [batch, token, head, channel], channels contiguous
    const void* p;
    int64_t sb, st, sh;   // elements
};

struct DiffArgs {
    DiffTensor q, k, v;
    const void* lam_vec[4];       // lq1, lk1, lq2, lk2: [D], or [H, D] with lam_sh = D
    int64_t lam_sh;
    float lam_init;
    const int* lengths;           // [B] or null (Tk each)
    void* out;                    // [B, Tq, H, Dv]
    void *o1, *o2;                // training: the two maps' own outputs, like out
    float* lse;                   // training: [2][B, Tq, H], log2 of the softmax denominators (+inf: nothing seen)
    float* part;                  // splits: [splits][B * Hk * Tq * g][2 Dv + 4]
    int B, Tq, Tk, H, Hk, g, D, Dv, causal;
    int splits, chunk;            // keys per split
    float c;                      // scale * log2(e)
    float scale;
};

__device__ __forceinline__ int diff_length(const int* lengths, int b, int Tk) {
    if (!lengths) return Tk;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > Tk ? Tk : n);
}

// exp(lq1 . lk1) and exp(lq2 . lk2) of one head, by one wave
template <typename T>
__device__ __forceinline__ void diff_lambda(const DiffArgs& p, int head, int lane, float& e1, float& e2) {
    const T* v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<const T*>(p.lam_vec[i]) + head * p.lam_sh;
    float a = 0.f, b = 0.f;
    for (int d = lane; d < p.D; d += 64) {
        a = fmaf((float)v[0][d], (float)v[1][d], a);
        b = fmaf((float)v[2][d], (float)v[3][d], b);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    e1 = expf(a);
    e2 = expf(b);
}

constexpr int DIFF_MAX_GROUP = 64;

// consecutive workgroup ids go to the 8 XCDs in turn: give each a contiguous run, so that the readers of one head's keys share an L2
__device__ __forceinline__ int xcd_run(int lin, int total) {
    const int q = total >> 3, r = total & 7, x = lin & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (lin >> 3);
}

}  // namespace ndb
