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

    // columns: bf16 cols2(): lane (d = col + l31) gets, of k-step s, rows r0 + 16 s + 4 lh + 0 .. 3 and 8 further (the k order in
    // which an accumulator's registers serve as the other operand); fp32 one(): row r0 + (e & 3) + 8 (e >> 2) + 4 lh.  col a multiple of
    // 32, r0 of 16 (bf16) / 32.
    static __device__ __forceinline__ int col_base(int lane) {
        const int lh = lane >> 5;
        if constexpr (ES == 2) {
            const int i = lane & 15, r = 4 * lh + (i >> 2);
            return r * RB + ((((lane & 16) / 8 + ((i & 3) >> 1)) ^ swz(r)) << 4) + (i & 1) * 8;
        }
        return 4 * lh * RB + ((((lane & 31) >> 2) ^ swz(4 * lh)) << 4) + (lane & 3) * 4;
    }
    // the fragments of two 32-column blocks col, col + 32 for rows r0 .. r0 + 31: f[block][k-step].  Eight transposed reads and their
    // wait in one piece of assembly: of the builtin the compiler believes that it may read what a load in flight to the other
    // stage writes, and waits for that load.
    static __device__ __forceinline__ void cols2(const char* t, int base, int r0, int col, u32x4 (&f)[2][2]) {
        const int at = (int)(uintptr_t)(__attribute__((address_space(3))) const char*)t + r0 * RB;
        u32x2 v[2][2][2];          // [block][k-step][rows + 8]
        const int a0 = at + (base ^ ((col / 8 & 15) << 4)), a1 = at + (base ^ (((col / 8 & 15) ^ 2) << 4));
        const int b0 = at + (base ^ (((col + 32) / 8 & 15) << 4)), b1 = at + (base ^ ((((col + 32) / 8 & 15) ^ 2) << 4));
        const int ca = (col / 128) * 256, cb = ((col + 32) / 128) * 256;
        static_assert(24 * RB + 512 < 65536, "offsets fit the instruction");
        if (ca == 0 && cb == 0) cols2_asm<0, 0>(v, a0, a1, b0, b1);
        else cols2_asm<256, 256>(v, a0, a1, b0, b1);
#pragma unroll
        for (int d = 0; d < 2; ++d)
#pragma unroll
            for (int s = 0; s < 2; ++s) f[d][s] = u32x4{v[d][s][0][0], v[d][s][0][1], v[d][s][1][0], v[d][s][1][1]};
    }
    template <int CA, int CB>
    static __device__ __forceinline__ void cols2_asm(u32x2 (&v)[2][2][2], int a0, int a1, int b0, int b1) {
        asm volatile(
            "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
            "ds_read_b64_tr_b16 %1, %9 offset:%13\n\t"
            "ds_read_b64_tr_b16 %2, %8 offset:%14\n\t"
            "ds_read_b64_tr_b16 %3, %9 offset:%15\n\t"
            "ds_read_b64_tr_b16 %4, %10 offset:%16\n\t"
            "ds_read_b64_tr_b16 %5, %11 offset:%17\n\t"
            "ds_read_b64_tr_b16 %6, %10 offset:%18\n\t"
            "ds_read_b64_tr_b16 %7, %11 offset:%19\n\t"
            "s_waitcnt lgkmcnt(0)"
            : "=&v"(v[0][0][0]), "=&v"(v[0][0][1]), "=&v"(v[0][1][0]), "=&v"(v[0][1][1]), "=&v"(v[1][0][0]), "=&v"(v[1][0][1]),
              "=&v"(v[1][1][0]), "=&v"(v[1][1][1])
            : "v"(a0), "v"(a1), "v"(b0), "v"(b1), "n"(CA), "n"(CA + 8 * RB), "n"(CA + 16 * RB), "n"(CA + 24 * RB), "n"(CB),
              "n"(CB + 8 * RB), "n"(CB + 16 * RB), "n"(CB + 24 * RB));
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

// over the two lanes (halves) that hold a column of an accumulator
__device__ __forceinline__ float half_max(float v) {
    union { float f; unsigned u; } x;
    x.f = v;
    const auto r = __builtin_amdgcn_permlane32_swap(x.u, x.u, false, false);
    union { unsigned u; float f; } a, b;
    a.u = r[0], b.u = r[1];
    return fmaxf(a.f, b.f);
}
__device__ __forceinline__ float half_sum(float v) {
    union { float f; unsigned u; } x;
    x.f = v;
    const auto r = __builtin_amdgcn_permlane32_swap(x.u, x.u, false, false);
    union { unsigned u; float f; } a, b;
    a.u = r[0], b.u = r[1];
    return a.f + b.f;
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

// acc[n][d][column] += sum over the 32 rows r0 .. of tile[row][col + 32 n + d] * p[row][column], for N blocks of columns, of which
// the first `real` columns count (fp32 leaves out blocks past them, D > 64 excepted: see no_step)
template <typename T, int RB, int N>
__device__ __forceinline__ void mma_cols(const char* t, int base, int r0, int col, int real, const Probs<T>& p, f32x16 (&acc)[N]) {
    if constexpr (sizeof(T) == 2) {
        static_assert(N % 2 == 0, "blocks in pairs");
#pragma unroll
        for (int n = 0; n < N; n += 2) {
            u32x4 f[2][2];
            Tile<T, RB>::cols2(t, base, r0, col + 32 * n, f);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    union { u32x4 u; bf16x8 h; } a;
                    a.u = f[i][s];
                    acc[n + i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, p.f[s], acc[n + i], 0, 0, 0);
                }
        }
    } else {
        if constexpr (RB < 1024) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if (n && 32 * n >= real) break;
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    acc[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(Tile<T, RB>::one(t, base, r0, e, col + 32 * n), p.f[e], acc[n], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
#pragma unroll
                for (int n = 0; n < N; ++n)
                    acc[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(Tile<T, RB>::one(t, base, r0, e, col + 32 * n), p.f[e], acc[n], 0, 0, 0);
        }
    }
}

// both maps' products with the halves of one tile: acc[m][d][column] += sum over rows of tile[row][m HD + 32 d ..] * p[m][row][column]
template <typename T, int RB, int HD>
__device__ __forceinline__ void mma_halves(const char* t, int base, int real, const Probs<T>& p0, const Probs<T>& p1, f32x16 (&acc)[2][HD / 32]) {
    if constexpr (sizeof(T) == 2 && HD == 32) {              // one block of each half: a pair
        u32x4 f[2][2];
        Tile<T, RB>::cols2(t, base, 0, 0, f);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            union { u32x4 u; bf16x8 h; } a, b;
            a.u = f[0][s], b.u = f[1][s];
            acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, p0.f[s], acc[0][0], 0, 0, 0);
            acc[1][0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b.h, p1.f[s], acc[1][0], 0, 0, 0);
        }
    } else {
        mma_cols<T, RB>(t, base, 0, 0, real, p0, acc[0]);
        mma_cols<T, RB>(t, base, 0, HD, real, p1, acc[1]);
    }
}

// fp32: step c of a product over `real` channels (8 a step) has none left.  A branch costs little beside a step's 256 cycles
// (D = 48, Dv = 96: 123 us for 140), but not where the registers are full already (D > 64: 255 us for 222 at 128).
template <typename T, int HD>
__device__ __forceinline__ bool no_step(int c, int real) { return sizeof(T) == 4 && HD < 128 && c && 8 * c >= real; }

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

// A ring of NST stages: fetch(i, stage) requests tile i (PER vector-memory operations a wave, always as many), NST - 1 tiles ahead
// of compute(i, stage).  Other such operations in between only make the wait for a tile stricter.
template <int NST, int PER, class Fetch, class Compute>
__device__ __forceinline__ void ring(char* stages, int bytes, int n, Fetch&& fetch, Compute&& compute) {
    static_assert((NST - 2) * PER < 64, "the counter's range");
#pragma unroll
    for (int i = 0; i < NST - 1; ++i)
        if (i < n) fetch(i, stages + i * bytes);
    int now = 0;
    for (int i = 0; i < n; ++i) {
        // tile i has landed (the NST - 2 behind it may be under way) ...
        if (i + NST - 1 <= n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NST - 2) * PER) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();                         // ... in all waves, and they are through with tile i - 1
        asm volatile("" ::: "memory");
        if (i + NST - 1 < n) fetch(i + NST - 1, stages + (now == 0 ? NST - 1 : now - 1) * bytes);
        compute(i, stages + now * bytes);
        now = now + 1 == NST ? 0 : now + 1;
    }
}

constexpr int DIFF_MAX_GROUP = 64;

// consecutive workgroup ids go to the 8 XCDs in turn: give each a contiguous run, so that the readers of one head's keys share an L2
__device__ __forceinline__ int xcd_run(int lin, int total) {
    const int q = total >> 3, r = total & 7, x = lin & 7;
    return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (lin >> 3);
}

// workgroup -> (batch and key head, index within).  Consecutive ids go to the 8 XCDs in turn; each XCD gets whole (batch, key head)s,
// whose readers then share an L2.  Units of equal length: one after the other.  Causal ones (index 0 the longest): the longest
// of all of them first, so that the short ones fill the end.
__device__ __forceinline__ void unit_of(int lin, int total, int units, int causal, int& unit, int& index) {
    if (causal && units % 8 == 0) {
        const int per = units >> 3, j = lin >> 3;
        index = j / per;
        unit = (lin & 7) * per + j - index * per;
    } else if (causal) {
        index = lin / units;
        unit = lin - index * units;
    } else {
        const int id = xcd_run(lin, total), per = total / units;
        unit = id / per;
        index = id - unit * per;
    }
}

}  // namespace ndb
