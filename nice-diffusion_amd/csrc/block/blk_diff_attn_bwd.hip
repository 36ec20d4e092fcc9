// Differential attention, backward.  With P1, P2 the two maps (rebuilt from the scores and the kept log denominators), dP = dO V^T
// and, per row, D1 = dO . O1, D2 = dO . O2 (the maps' own outputs, kept by the forward pass):
//   dV = (P1 - lam P2)^T dO     dS1 = P1 (dP - D1)     dS2 = -lam P2 (dP - D2)
//   dq_i = s dS_i k_i           dk_i = s dS_i^T q_i    dlam = -sum P2 dP, which scales the gradients of the four vectors
//
// Two launches without atomics: queries (a wave owns 32 rows, the keys pass by: D1, D2 and dq), then keys (a wave owns 32 keys, the
// rows of all query heads pass by: dk, dv and its share of dlam), and a small one for the vectors.  Both rebuild the scores: 28 D T^2 operations for Dv = 2 D in all
// where 20 would do with the maps kept, but nothing of T x T is stored.  Scores and dP come out of the matrix unit in the layout
// in which dS is the next product's operand; the transposed operands are column reads of the same row-major tiles.
// dlam is summed from fp32 P2 and dP, not from the rounded O2: it is one number and may cancel.  Rounding to bf16 besides the
// outputs: P1 - lam P2, dS1, dS2 as operands, O1 and O2.  A sequence of one key has constant maps: dq and dk are made exactly zero.
//
// Measured, bf16, 8 x 2048^2 x 8 heads of 64 + 128, causal: keys 230 us, queries (with D1 and D2) 161 us (0.52 and 0.50 PFLOP/s of
// matrix operations); what bounds them is what bounds the forward pass, with two exponentials and ~12 vector operations a score, and
// LDS reads that no phase starts under the one before it (phase(), below).  Vector registers spilled: 26 by that key kernel (8 waves),
// 10 by the one of bf16 D <= 32; fp32 with D > 64: 125 by the query kernel, 15 by the key kernel.
#include "blk_diff_attn.h"

namespace ndb {

int diff_head_dim(int D, int Dv);
int diff_parts(int64_t units, int slots, int64_t length, int64_t grain, double per, double bytes, int causal, int64_t& share);
int diff_check(const char* fn, const DiffArgs& a, int dtype);

struct DiffBwdArgs {
    DiffArgs f;
    DiffTensor dout;              // [B, Tq, H, Dv]
    const void *o1, *o2;
    const float* lse;             // [2][B, Tq, H]
    float* dots;                  // [2][B, Tq, H]: D1, D2
    float* dlam_part;             // [B * Hk][key blocks][row splits][waves][g]
    void *dq, *dk, *dv;           // contiguous
    void* dvec[4];
    int key_blocks, waves;        // of the key kernel: waves * 32 keys a workgroup
    int row_splits;               // its rows over this many workgroups: fp32 partials [row_splits][B * Tk * Hk][2 D + Dv]
    int key_splits, chunk;        // the query kernel's keys: fp32 partials [key_splits][B * Tq * H][2 D]
    float *part_kv, *part_q;
};

// d += x . y over 16 bytes
template <typename T>
__device__ __forceinline__ void dot16(u32x4 x, u32x4 y, float& d) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 2) {
            union { unsigned u; bf16x2 h; } a, b;
            a.u = x[i], b.u = y[i];
            d = __builtin_amdgcn_fdot2_f32_bf16(a.h, b.h, d, false);
        } else {
            union { unsigned u; float f; } a, b;
            a.u = x[i], b.u = y[i];
            d = fmaf(a.f, b.f, d);
        }
    }
}

template <typename T, int HD>
struct DiffBwdShape {
    static constexpr int ES = (int)sizeof(T), DV = 2 * HD, RB = 2 * HD * ES;      // q / k rows and dO / v rows: equally long
    static constexpr int PH = HD * ES / 16, NS = PH / 2, NSV = RB / 32;
    static constexpr int KT = RB == 1024 ? 32 : 64;                               // keys of a tile (query kernel)
    static constexpr int RT = RB <= 256 ? 64 : 32;                                // rows of a tile (key kernel)
    static constexpr bool V_LDS = RB <= 512;                                      // key kernel: its 128 value rows in LDS, else in registers
};

// the compiler may not move work across: gathered, the operands of all phases do not fit the registers
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

// DK, DV: which gradients this launch makes.  Wide heads take two launches: the outputs and operands of both do not fit the registers
template <typename T, int HD, int NW, bool DK, bool DVG>
__global__ void __launch_bounds__(64 * NW, (HD * (int)sizeof(T) == 64 ? 3 : (NW == 8 ? 2 : 1))) diff_dkv_kernel(const DiffBwdArgs p) {
    using S = DiffBwdShape<T, HD>;
    using TR = Tile<T, S::RB>;
    constexpr int RT = S::RT, STAT = 4 * 64 * 4, STAGE = 2 * RT * S::RB + STAT;     // q rows, dO rows, [lse1, lse2, D1, D2][64]
    constexpr int KEYS = 32 * NW, VB = DK && S::V_LDS ? KEYS * S::RB : 16;
    constexpr int NST = S::RB == 128 || 3 * STAGE + VB > 150 * 1024 ? 2 : 3;      // 128-byte rows: three workgroups a CU instead
    __shared__ __attribute__((aligned(16))) char stages[NST * STAGE], v_rows[VB];
    __shared__ float lam_s[DIFF_MAX_GROUP];
    const DiffArgs& f = p.f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, lh = lane >> 5;
    int bh, kb;
    unit_of(blockIdx.x, gridDim.x, f.B * f.Hk, f.causal, bh, kb);
    const int at_part = bh * p.key_blocks * p.row_splits + kb, rs = kb % p.row_splits;
    kb /= p.row_splits;
    const int b = bh / f.Hk, hk = bh - b * f.Hk;
    const int len = diff_length(f.lengths, b, f.Tk);
    const int key0 = kb * KEYS, key = key0 + wave * 32 + l31;
    const bool kin = key < len;

    for (int h = wave; h < f.g; h += NW) {
        float e1, e2;
        diff_lambda<T>(f, hk * f.g + h, lane, e1, e2);
        if (lane == 0) lam_s[h] = e1 - e2 + f.lam_init;
    }
    u32x4 kf[2][S::NS], vf[DK && !S::V_LDS ? S::NSV : 1];
    {
        const int kr = kin ? key : 0;
        const char* kp = reinterpret_cast<const char*>(static_cast<const T*>(f.k.p) + b * f.k.sb + (int64_t)kr * f.k.st + hk * f.k.sh);
        const char* vp = reinterpret_cast<const char*>(static_cast<const T*>(f.v.p) + b * f.v.sb + (int64_t)kr * f.v.st + hk * f.v.sh);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int c = 0; c < S::NS; ++c) {
                const int by = (2 * c + lh) * 16;
                kf[m][c] = u32x4{0u, 0u, 0u, 0u};
                if (kin && by < f.D * S::ES) kf[m][c] = *reinterpret_cast<const u32x4*>(kp + m * f.D * S::ES + by);
            }
        if constexpr (DK && !S::V_LDS) {
#pragma unroll
            for (int c = 0; c < S::NSV; ++c) {
                const int by = (2 * c + lh) * 16;
                vf[c] = u32x4{0u, 0u, 0u, 0u};
                if (kin && by < f.Dv * S::ES) vf[c] = *reinterpret_cast<const u32x4*>(vp + by);
            }
        }
    }
    if constexpr (DK && S::V_LDS) {                            // keys past the sequence's end become zero rows
        TileLoad<T, S::RB, KEYS, NW> lv;
        lv.template init<S::RB>(f.v.st * S::ES, f.Dv * S::ES, wave, lane);
        lv.load(v_rows, static_cast<const T*>(f.v.p) + b * f.v.sb + (int64_t)key0 * f.v.st + hk * f.v.sh, ((int64_t)(len - key0 - 1) * f.v.st + f.Dv) * S::ES, wave);
    }
    f32x16 dk[2][DK ? HD / 32 : 1], dv[DVG ? S::DV / 32 : 1];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
#pragma unroll
        for (int d = 0; d < (DK ? HD / 32 : 1); ++d) dk[0][d][e] = dk[1][d][e] = 0.f;
#pragma unroll
        for (int d = 0; d < (DVG ? S::DV / 32 : 1); ++d) dv[d][e] = 0.f;
    }

    TileLoad<T, S::RB, RT, NW> lq, lo;
    lq.template init<S::RB / 2>(f.q.st * S::ES, f.D * S::ES, wave, lane);
    lo.template init<S::RB>(p.dout.st * S::ES, f.Dv * S::ES, wave, lane);
    const int row_base = TR::row_base(lane), col_base = TR::col_base(lane);
    const int nt = (f.Tq + RT - 1) / RT;
    int tile0 = 0;                                            // causal: the first tile with a row that sees this block's first key
    if (f.causal) {
        const int t = key0 - len + f.Tq;
        tile0 = t > 0 ? t / RT : 0;
    }
    const int per_head = (key0 < len && tile0 < nt) ? nt - tile0 : 0, total = per_head * f.g;
    const int share = (total + p.row_splits - 1) / p.row_splits, i0 = rs * share, n = total - i0 < share ? total - i0 : share;
    const int hg0 = n > 0 ? i0 / per_head : 0, hg1 = n > 0 ? (i0 + n - 1) / per_head : -1;       // heads of this workgroup's tiles
    const int64_t rows_all = (int64_t)f.B * f.Tq * f.H;
    // the statistics of a tile's rows, a kind a wave (waves past the fourth repeat them)
    const int kind = wave & 3;
    const float* const stats = (kind < 2 ? p.lse : p.dots) + (kind & 1) * rows_all;
    const unsigned soff = lane < RT ? (unsigned)lane * (unsigned)f.H * 4u : 0xfffffff0u;
    // tiles are requested and used in the same order: all of a head's rows, then the next head's
    int f_hg = hg0, f_t0 = (tile0 + i0 - hg0 * per_head) * RT, c_hg = f_hg, c_t0 = f_t0;
    const T* const qb = static_cast<const T*>(f.q.p) + b * f.q.sb + (int64_t)hk * f.g * f.q.sh;
    const T* const ob = static_cast<const T*>(p.dout.p) + b * p.dout.sb + (int64_t)hk * f.g * p.dout.sh;
    auto fetch = [&](int, char* at) {
        const int hg = f_hg, t0 = f_t0, head = hk * f.g + hg;
        f_t0 += RT;
        if (f_t0 >= f.Tq) {
            f_t0 = tile0 * RT;
            ++f_hg;
        }
        const int left = f.Tq - t0;
        lq.load(at, qb + (int64_t)t0 * f.q.st + hg * f.q.sh, ((left - 1) * f.q.st + 2 * f.D) * S::ES, wave);
        lo.load(at + RT * S::RB, ob + (int64_t)t0 * p.dout.st + hg * p.dout.sh, ((left - 1) * p.dout.st + f.Dv) * S::ES, wave);
        const int64_t first = ((int64_t)b * f.Tq + t0) * f.H + head;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(stats + first), 0, ((left < RT ? left : RT) - 1) * f.H * 4 + 4, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(at + 2 * RT * S::RB + kind * 256), 4, (int)soff, 0, 0, 0);
    };
    float dl = 0.f;
    auto compute = [&](int i, const char* tq) {
        const int hg = c_hg, t0 = c_t0;
        c_t0 += RT;
        const float lam = lam_s[hg];
        const char* to = tq + RT * S::RB;
        const float* st = reinterpret_cast<const float*>(tq + 2 * RT * S::RB) + 4 * lh;
#pragma unroll 1
        for (int r32 = 0; r32 < RT; r32 += 32) {
            const int rb = in_loop(row_base), cb = in_loop(col_base);
            const char* q32 = tq + r32 * S::RB;
            const char* o32 = to + r32 * S::RB;
            f32x16 s[2], dp;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[m][e] = 0.f;
#pragma unroll
                for (int c = 0; c < S::NS; ++c)
                    if (!no_step<T, HD>(c, f.D)) s[m] = mma_step<T>(TR::row(q32, rb, 0, m * S::PH + 2 * c), kf[m][c], s[m]);
            }
            // rows that see this lane's key: from `first` on (causal), no row past the last, none for a key past the sequence's end
            const int r_first = t0 + r32 + len - f.Tq;        // causal: the first row of the block sees the keys up to this one
            if (key0 + wave * 32 + 31 >= len || (f.causal && key0 + wave * 32 + 31 > r_first) || t0 + r32 + 32 > f.Tq) {
                const int first = kin ? (f.causal ? key - r_first - 4 * lh : -0x40000000) : 0x40000000, rows_in = f.Tq - t0 - r32 - 4 * lh;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool in = (e & 3) + 8 * (e >> 2) >= first && (e & 3) + 8 * (e >> 2) < rows_in;
                    s[0][e] = in ? s[0][e] : -INFINITY;
                    s[1][e] = in ? s[1][e] : -INFINITY;
                }
            }
            Probs<T> pd;
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const f32x4 l1 = *reinterpret_cast<const f32x4*>(st + r32 + 8 * g4), l2 = *reinterpret_cast<const f32x4*>(st + 64 + r32 + 8 * g4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = 4 * g4 + j;
                    s[0][e] = __builtin_amdgcn_exp2f(fmaf(s[0][e], f.c, -l1[j]));
                    s[1][e] = __builtin_amdgcn_exp2f(fmaf(s[1][e], f.c, -l2[j]));
                    if constexpr (DVG) pd.set(e, fmaf(-lam, s[1][e], s[0][e]));
                }
            }
            phase();
            if constexpr (DVG) mma_cols<T, S::RB>(o32, cb, 0, 0, f.Dv, pd, dv);
            if constexpr (DK) {
                phase();
#pragma unroll
                for (int e = 0; e < 16; ++e) dp[e] = 0.f;
#pragma unroll
                for (int c = 0; c < S::NSV; ++c) {
                    if (no_step<T, HD>(c, f.Dv)) break;
                    u32x4 v;
                    if constexpr (S::V_LDS) v = TR::row(v_rows + wave * 32 * S::RB, rb, 0, 2 * c);
                    else v = vf[c];
                    dp = mma_step<T>(TR::row(o32, rb, 0, 2 * c), v, dp);
                }
                phase();
                Probs<T> d1, d2;
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const f32x4 c1 = *reinterpret_cast<const f32x4*>(st + 128 + r32 + 8 * g4), c2 = *reinterpret_cast<const f32x4*>(st + 192 + r32 + 8 * g4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int e = 4 * g4 + j;
                        dl = fmaf(s[1][e], dp[e], dl);
                        d1.set(e, s[0][e] * (dp[e] - c1[j]));
                        d2.set(e, lam * s[1][e] * (c2[j] - dp[e]));
                    }
                }
                mma_halves<T, S::RB, HD>(q32, cb, f.D, d1, d2, dk);
            }
        }
        const bool through = c_t0 >= f.Tq;                    // this head's rows
        if (through) {
            c_t0 = tile0 * RT;
            ++c_hg;
        }
        if (DK && (through || i + 1 == n)) {
#pragma unroll
            for (int o = 32; o; o >>= 1) dl += __shfl_xor(dl, o, 64);
            if (lane == 0) p.dlam_part[((int64_t)at_part * NW + wave) * f.g + hg] = -dl;
            dl = 0.f;
        }
    };
    ring<NST, 2 * decltype(lq)::NI + 1>(stages, STAGE, n, fetch, compute);
    if constexpr (DK) {
        for (int h = lane; h < f.g; h += 64)
            if (h < hg0 || h > hg1) p.dlam_part[((int64_t)at_part * NW + wave) * f.g + h] = 0.f;
    }
    if (key >= f.Tk) return;
    if (!kin) {                                               // its weights are zero, but zero times a row's NaN is none
#pragma unroll
        for (int e = 0; e < 16; ++e) {
#pragma unroll
            for (int d = 0; d < (DK ? HD / 32 : 1); ++d) dk[0][d][e] = dk[1][d][e] = 0.f;
#pragma unroll
            for (int d = 0; d < (DVG ? S::DV / 32 : 1); ++d) dv[d][e] = 0.f;
        }
    }
    const int64_t krow = ((int64_t)b * f.Tk + key) * f.Hk + hk;
    const float scale = p.row_splits > 1 ? 1.f : (len == 1 ? 0.f : f.scale);
    float* const part = p.part_kv + ((int64_t)rs * f.B * f.Tk * f.Hk + krow) * (2 * f.D + f.Dv);
    if constexpr (DK) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int dd = d * 32 + 8 * g4 + 4 * lh;
                    const float v[4] = {dk[m][d][4 * g4] * scale, dk[m][d][4 * g4 + 1] * scale, dk[m][d][4 * g4 + 2] * scale, dk[m][d][4 * g4 + 3] * scale};
                    if (dd >= f.D) continue;
                    if (p.row_splits > 1) store_vec<float, 4>(part + m * f.D + dd, v);
                    else store_vec<T, 4>(static_cast<T*>(p.dk) + krow * 2 * f.D + m * f.D + dd, v);
                }
    }
    if constexpr (DVG) {
#pragma unroll
        for (int d = 0; d < S::DV / 32; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int dd = d * 32 + 8 * g4 + 4 * lh;
                const float v[4] = {dv[d][4 * g4], dv[d][4 * g4 + 1], dv[d][4 * g4 + 2], dv[d][4 * g4 + 3]};
                if (dd >= f.Dv) continue;
                if (p.row_splits > 1) store_vec<float, 4>(part + 2 * f.D + dd, v);
                else store_vec<T, 4>(static_cast<T*>(p.dv) + krow * f.Dv + dd, v);
            }
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(256, (HD * (int)sizeof(T) >= 256 ? 1 : 2)) diff_dq_kernel(const DiffBwdArgs p) {
    using S = DiffBwdShape<T, HD>;
    using TR = Tile<T, S::RB>;
    constexpr int KT = S::KT, STAGE = 2 * KT * S::RB;
    __shared__ __attribute__((aligned(16))) char stages[2 * STAGE];
    __shared__ float lam_s[DIFF_MAX_GROUP];
    const DiffArgs& f = p.f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, lh = lane >> 5;
    const int rows = f.Tq * f.g, tiles = (rows + 127) / 128;
    int bh, tile;
    unit_of(blockIdx.x, gridDim.x, f.B * f.Hk, f.causal, bh, tile);
    const int ks = tile % p.key_splits;
    tile = tiles - 1 - tile / p.key_splits;                   // longest rows first
    const int b = bh / f.Hk, hk = bh - b * f.Hk;
    const int len = diff_length(f.lengths, b, f.Tk);
    const int r0 = tile * 128 + wave * 32, r = r0 + l31 < rows ? r0 + l31 : rows - 1;
    const int t = r / f.g, hg = r - t * f.g, head = hk * f.g + hg;
    const int seen = f.causal ? t + len - f.Tq + 1 : len;
    int kend = len;
    if (f.causal) {
        const int rl = (tile + 1) * 128 - 1 < rows ? (tile + 1) * 128 - 1 : rows - 1;
        kend = rl / f.g + len - f.Tq + 1;
    }
    const int kbeg = ks * p.chunk;
    if (kend > kbeg + p.chunk) kend = kbeg + p.chunk;
    for (int h = wave; h < f.g; h += 4) {
        float e1, e2;
        diff_lambda<T>(f, hk * f.g + h, lane, e1, e2);
        if (lane == 0) lam_s[h] = e1 - e2 + f.lam_init;
    }
    u32x4 q[2][S::NS], go[S::NSV];
    {
        const char* qp = reinterpret_cast<const char*>(static_cast<const T*>(f.q.p) + b * f.q.sb + t * f.q.st + head * f.q.sh);
        const char* gp = reinterpret_cast<const char*>(static_cast<const T*>(p.dout.p) + b * p.dout.sb + t * p.dout.st + head * p.dout.sh);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int c = 0; c < S::NS; ++c) {
                const int by = (2 * c + lh) * 16;
                q[m][c] = u32x4{0u, 0u, 0u, 0u};
                if (by < f.D * S::ES) q[m][c] = *reinterpret_cast<const u32x4*>(qp + m * f.D * S::ES + by);
            }
#pragma unroll
        for (int c = 0; c < S::NSV; ++c) {
            const int by = (2 * c + lh) * 16;
            go[c] = u32x4{0u, 0u, 0u, 0u};
            if (by < f.Dv * S::ES) go[c] = *reinterpret_cast<const u32x4*>(gp + by);
        }
    }
    const int64_t orow = ((int64_t)b * f.Tq + t) * f.H + head, rows_all = (int64_t)f.B * f.Tq * f.H;
    const float l1 = p.lse[orow], l2 = p.lse[rows_all + orow];
    float c1 = 0.f, c2 = 0.f;                                 // D1, D2: kept for the key kernel
    {
        const char* p1 = reinterpret_cast<const char*>(static_cast<const T*>(p.o1) + orow * f.Dv);
        const char* p2 = reinterpret_cast<const char*>(static_cast<const T*>(p.o2) + orow * f.Dv);
#pragma unroll
        for (int c = 0; c < S::NSV; ++c) {
            const int by = (2 * c + lh) * 16;
            if (by < f.Dv * S::ES) {
                dot16<T>(go[c], *reinterpret_cast<const u32x4*>(p1 + by), c1);
                dot16<T>(go[c], *reinterpret_cast<const u32x4*>(p2 + by), c2);
            }
        }
        c1 = half_sum(c1);
        c2 = half_sum(c2);
        if (ks == 0 && lh == 0 && r0 + l31 < rows) {
            p.dots[orow] = c1;
            p.dots[rows_all + orow] = c2;
        }
    }
    __syncthreads();
    const float nlam = -lam_s[hg];
    f32x16 dq[2][HD / 32];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) dq[m][d][e] = 0.f;

    TileLoad<T, S::RB, KT, 4> lk, lv;
    lk.template init<S::RB / 2>(f.k.st * S::ES, f.D * S::ES, wave, lane);
    lv.template init<S::RB>(f.v.st * S::ES, f.Dv * S::ES, wave, lane);
    const T* kp = static_cast<const T*>(f.k.p) + b * f.k.sb + hk * f.k.sh;
    const T* vp = static_cast<const T*>(f.v.p) + b * f.v.sb + hk * f.v.sh;
    auto fetch = [&](int i, char* at) {
        const int key = kbeg + i * KT;
        const int64_t n = len - key;
        lk.load(at, kp + (int64_t)key * f.k.st, ((n - 1) * f.k.st + 2 * f.D) * S::ES, wave);
        lv.load(at + KT * S::RB, vp + (int64_t)key * f.v.st, ((n - 1) * f.v.st + f.Dv) * S::ES, wave);
    };
    const int row_base = TR::row_base(lane), col_base = TR::col_base(lane);
    auto compute = [&](int i, const char* tile_k) {
        const int key0 = kbeg + i * KT;
#pragma unroll 1
        for (int k32 = 0; k32 < KT; k32 += 32) {
            const int kb = key0 + k32;
            if (kb >= kend) break;
            const char* tk = tile_k + k32 * S::RB;
            const char* tv = tk + KT * S::RB;
            const int rb = in_loop(row_base), cb = in_loop(col_base);
            f32x16 s[2], dp;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[m][e] = 0.f;
#pragma unroll
                for (int c = 0; c < S::NS; ++c)
                    if (!no_step<T, HD>(c, f.D)) s[m] = mma_step<T>(TR::row(tk, rb, 0, m * S::PH + 2 * c), q[m][c], s[m]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] = 0.f;
#pragma unroll
            for (int c = 0; c < S::NSV; ++c)
                if (!no_step<T, HD>(c, f.Dv)) dp = mma_step<T>(TR::row(tv, rb, 0, 2 * c), go[c], dp);
            const int left = seen - kb - 4 * lh;              // keys of this block the row sees
            if (f.causal ? kb + 32 > r0 / f.g + len - f.Tq + 1 : kb + 32 > len) {
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const bool in = (e & 3) + 8 * (e >> 2) < left;
                    s[0][e] = in ? s[0][e] : -INFINITY;
                    s[1][e] = in ? s[1][e] : -INFINITY;
                }
            }
            Probs<T> d1, d2;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][e], f.c, -l1)), p2 = __builtin_amdgcn_exp2f(fmaf(s[1][e], f.c, -l2));
                d1.set(e, p1 * (dp[e] - c1));
                d2.set(e, nlam * p2 * (dp[e] - c2));
            }
            mma_halves<T, S::RB, HD>(tk, cb, f.D, d1, d2, dq);
        }
    };
    ring<2, decltype(lk)::NI + decltype(lv)::NI>(stages, STAGE, kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0, fetch, compute);
    if (r0 + l31 >= rows) return;
    const float scale = p.key_splits > 1 ? 1.f : (len == 1 ? 0.f : f.scale);
    float* const part = p.part_q + ((int64_t)ks * rows_all + orow) * 2 * f.D;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int dd = d * 32 + 8 * g4 + 4 * lh;
                const float v[4] = {dq[m][d][4 * g4] * scale, dq[m][d][4 * g4 + 1] * scale, dq[m][d][4 * g4 + 2] * scale, dq[m][d][4 * g4 + 3] * scale};
                if (dd >= f.D) continue;
                if (p.key_splits > 1) store_vec<float, 4>(part + m * f.D + dd, v);
                else store_vec<T, 4>(static_cast<T*>(p.dq) + orow * 2 * f.D + m * f.D + dd, v);
            }
}

// the splits' partials in order: 8 columns of a key's dk | dv or of a row's dq a thread
template <typename T>
__global__ void __launch_bounds__(256) diff_bwd_join_kernel(const DiffBwdArgs p) {
    const DiffArgs& f = p.f;
    const int64_t krows = (int64_t)f.B * f.Tk * f.Hk, qrows = (int64_t)f.B * f.Tq * f.H;
    const int ck = (2 * f.D + f.Dv) / 8, cq = 2 * f.D / 8;
    const int64_t nk = p.row_splits > 1 ? krows * ck : 0, nq = p.key_splits > 1 ? qrows * cq : 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nk + nq; i += (int64_t)gridDim.x * 256) {
        const bool kv = i < nk;
        const int64_t j = kv ? i : i - nk, row = j / (kv ? ck : cq);
        const int c = (int)(j - row * (kv ? ck : cq)) * 8, width = kv ? 2 * f.D + f.Dv : 2 * f.D, splits = kv ? p.row_splits : p.key_splits;
        const float* src = (kv ? p.part_kv : p.part_q) + row * width + c;
        const int64_t step = (kv ? krows : qrows) * width;
        float v[8] = {};
        for (int s = 0; s < splits; ++s) {
            float t[8];
            load_vec<float, 8>(src + s * step, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += t[e];
        }
        const int b = (int)(row / (kv ? (int64_t)f.Tk * f.Hk : (int64_t)f.Tq * f.H));
        const float scale = c >= 2 * f.D ? 1.f : (diff_length(f.lengths, b, f.Tk) == 1 ? 0.f : f.scale);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= scale;
        if (!kv) store_vec<T, 8>(static_cast<T*>(p.dq) + row * 2 * f.D + c, v);
        else if (c < 2 * f.D) store_vec<T, 8>(static_cast<T*>(p.dk) + row * 2 * f.D + c, v);
        else store_vec<T, 8>(static_cast<T*>(p.dv) + row * f.Dv + c - 2 * f.D, v);
    }
}

// The four vectors' gradients from the partial dlam, summed in a fixed order: a workgroup per head, or one for all heads where they
// share the vectors.
template <typename T>
__global__ void __launch_bounds__(1024) diff_dvec_kernel(const DiffBwdArgs p) {
    __shared__ float red[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, head = blockIdx.x, per = p.key_blocks * p.row_splits * p.waves;
    float t = 0.f;
    if (p.f.lam_sh) {
        const int hk = head / p.f.g, hg = head - hk * p.f.g;
        for (int i = threadIdx.x; i < p.f.B * per; i += 1024) {
            const int b = i / per, j = i - b * per;
            t += p.dlam_part[(((int64_t)b * p.f.Hk + hk) * per + j) * p.f.g + hg];
        }
    } else {
        const int64_t all = (int64_t)p.f.B * p.f.Hk * per * p.f.g;
#pragma unroll 4
        for (int64_t i = threadIdx.x; i < all; i += 1024) t += p.dlam_part[i];
    }
    float e1, e2;
    diff_lambda<T>(p.f, head, lane, e1, e2);
#pragma unroll
    for (int o = 32; o; o >>= 1) t += __shfl_xor(t, o, 64);
    if (lane == 0) red[wave] = t;
    __syncthreads();
    if (wave) return;
    float dlam = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) dlam += red[w];
    const int64_t at = head * p.f.lam_sh;
    for (int d = lane; d < p.f.D; d += 64) {
        const T* v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = static_cast<const T*>(p.f.lam_vec[i]) + at + d;
        if (p.dvec[0]) static_cast<T*>(p.dvec[0])[at + d] = (T)(dlam * e1 * (float)*v[1]);
        if (p.dvec[1]) static_cast<T*>(p.dvec[1])[at + d] = (T)(dlam * e1 * (float)*v[0]);
        if (p.dvec[2]) static_cast<T*>(p.dvec[2])[at + d] = (T)(-dlam * e2 * (float)*v[3]);
        if (p.dvec[3]) static_cast<T*>(p.dvec[3])[at + d] = (T)(-dlam * e2 * (float)*v[2]);
    }
}

template <typename T, int HD, int NW, bool DK, bool DVG>
static int launch_dkv(const char* fn, const DiffBwdArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((diff_dkv_kernel<T, HD, NW, DK, DVG>), dim3((unsigned)(a.f.B * a.f.Hk * a.key_blocks * a.row_splits)), dim3(64 * NW), 0, st, a);
    return check_launch(fn);
}

template <typename T, int HD>
static int launch_diff_bwd(const char* fn, const DiffBwdArgs& a, hipStream_t st) {
    const int tiles = (a.f.Tq * a.f.g + 127) / 128;
    hipLaunchKernelGGL((diff_dq_kernel<T, HD>), dim3((unsigned)(a.f.B * a.f.Hk * tiles * a.key_splits)), dim3(256), 0, st, a);
    if constexpr (HD == 128) {
        if (int rc = launch_dkv<T, HD, 4, true, false>(fn, a, st)) return rc;
        if (int rc = launch_dkv<T, HD, 4, false, true>(fn, a, st)) return rc;
    } else if (HD * (int)sizeof(T) == 128 && a.waves == 8) {
        if (int rc = launch_dkv<T, HD, HD * (int)sizeof(T) == 128 ? 8 : 4, true, true>(fn, a, st)) return rc;
    } else {
        if (int rc = launch_dkv<T, HD, 4, true, true>(fn, a, st)) return rc;
    }
    if (a.row_splits > 1 || a.key_splits > 1) hipLaunchKernelGGL((diff_bwd_join_kernel<T>), dim3(1024), dim3(256), 0, st, a);
    if (a.dvec[0] || a.dvec[1] || a.dvec[2] || a.dvec[3])
        hipLaunchKernelGGL((diff_dvec_kernel<T>), dim3((unsigned)(a.f.lam_sh ? a.f.H : 1)), dim3(1024), 0, st, a);
    return check_launch(fn);
}

struct DiffBwdPlan {
    int waves, key_blocks, row_splits, key_splits, chunk;
    int64_t dots, dlam, kv, q;    // floats of workspace
};

// Rows of 256 bytes (D 33 .. 64 in bf16, to 32 in fp32): 8 waves share the rows that pass by, two to a SIMD in one workgroup a CU,
// where that still fills the chip (8 x 2048^2 x 8 heads: 390 us for 440 with 4); others 4.  Loops divided as diff_parts says and
// joined in order.  Key kernel: a CU holds three workgroups of 128-byte rows, one of longer ones (134 KB of LDS, with 4 waves too:
// counting two of those divides one drawn shape in 13 otherwise, and 24 such shapes took 1.5 to 2 % longer).  Query kernel: two, one
// from 512-byte rows on; three of 128-byte rows would fit, but counting them chose no better (24 shapes: 0.3 % longer).
static DiffBwdPlan diff_bwd_plan(int B, int Tq, int Tk, int H, int Hk, int D, int Dv, int es, int causal) {
    DiffBwdPlan pl{};
    const int g = H / Hk;
    const int64_t units = (int64_t)B * Hk, rows = (int64_t)B * Tq * H, krows = (int64_t)B * Tk * Hk;
    pl.waves = diff_head_dim(D, Dv) * es == 128 && units * ((Tk + 255) / 256) >= 256 ? 8 : 4;
    pl.key_blocks = (Tk + 32 * pl.waves - 1) / (32 * pl.waves);
    // a tile of rows (all heads of the group pass by) in the key kernel, 64 keys in the query kernel, in cycles per row / key
    const int hd = diff_head_dim(D, Dv), rt = hd * es <= 64 * 2 ? 64 : 32;
    int64_t share;
    pl.row_splits = diff_parts(units * pl.key_blocks, 256 * (hd * es == 64 ? 3 : 1), (int64_t)g * ((Tq + rt - 1) / rt), 1,
                               rt * (pl.waves / 4) * (es == 4 ? 12.0 : 2.0) * hd, (double)krows * (2 * D + Dv) * 4, causal, share);
    pl.key_splits = diff_parts(units * (((int64_t)Tq * g + 127) / 128), hd * es >= 256 ? 256 : 512, Tk, 64, (es == 4 ? 8.0 : 1.3) * hd, (double)rows * 2 * D * 4, causal, share);
    pl.chunk = (int)share;
    pl.dots = 2 * rows;
    pl.dlam = (units * pl.key_blocks * pl.row_splits * pl.waves * g + 3) / 4 * 4;
    pl.kv = pl.row_splits > 1 ? pl.row_splits * krows * (2 * D + Dv) : 0;
    pl.q = pl.key_splits > 1 ? pl.key_splits * rows * 2 * D : 0;
    pl.dots = (pl.dots + 3) / 4 * 4;
    return pl;
}

// What a backward pass of these sizes needs beyond diff_check; a forward pass that keeps its statistics asks too, so that no step
// ends between the two.  The output's gradient may come contiguous, with token rows of H Dv elements.
int diff_bwd_check(const char* fn, const DiffArgs& a, int dtype) {
    const DiffBwdPlan pl = diff_bwd_plan(a.B, a.Tq, a.Tk, a.H, a.Hk, a.D, a.Dv, dtype == ND_DT_BF16 ? 2 : 4, a.causal);
    const int64_t units = (int64_t)a.B * a.Hk, tiles = ((int64_t)a.Tq * (a.H / a.Hk) + 127) / 128;
    NDB_REQUIRE(grid_fits(units * pl.key_blocks * pl.row_splits, 64 * pl.waves) && grid_fits(units * tiles * pl.key_splits, 256), fn,
                "too many workgroups for one launch of the backward pass");
    NDB_REQUIRE(a.Tq == 1 || (int64_t)a.H * a.Dv <= (1 << 22), fn, "the output's gradient: more than 2^22 elements a token");
    return ND_OK;
}

template <typename T>
static int dispatch_diff_bwd(const char* fn, const DiffBwdArgs& a, hipStream_t st) {
    switch (diff_head_dim(a.f.D, a.f.Dv)) {
        case 32: return launch_diff_bwd<T, 32>(fn, a, st);
        case 64: return launch_diff_bwd<T, 64>(fn, a, st);
        default: return launch_diff_bwd<T, 128>(fn, a, st);
    }
}

}  // namespace ndb

using namespace ndb;

extern "C" int64_t nd_diff_attention_bwd_workspace_floats(int B, int Tq, int Tk, int H, int Hk, int D, int Dv, int dtype) {
    if (B <= 0 || Tq <= 0 || Tk <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0 || D > 128 || Dv <= 0 || Dv > 256) return -1;
    int64_t most = 0;
    for (int causal = 0; causal < 2; ++causal) {
        const DiffBwdPlan pl = diff_bwd_plan(B, Tq, Tk, H, Hk, D, Dv, dtype == ND_DT_BF16 ? 2 : 4, causal);
        const int64_t n = pl.dots + pl.dlam + pl.kv + pl.q;
        most = n > most ? n : most;
    }
    return most;
}

extern "C" int nd_diff_attention_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                                     int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const void* lambda_q1,
                                     const void* lambda_k1, const void* lambda_q2, const void* lambda_k2, int64_t lambda_sh,
                                     float lambda_init, const int* key_lengths, const void* out1, const void* out2, const float* lse,
                                     const void* dout, int64_t do_sb, int64_t do_st, int64_t do_sh, void* dq, void* dk, void* dv,
                                     void* dlambda_q1, void* dlambda_k1, void* dlambda_q2, void* dlambda_k2, float* workspace, int B,
                                     int Tq, int Tk, int H, int Hk, int D, int Dv, float scale, int flags, int dtype, nd_stream_t stream) {
    const char* fn = "nd_diff_attention_bwd";
    DiffBwdArgs p{};
    DiffArgs& a = p.f;
    a.q = {q, q_sb, q_st, q_sh}, a.k = {k, k_sb, k_st, k_sh}, a.v = {v, v_sb, v_st, v_sh};
    a.lam_vec[0] = lambda_q1, a.lam_vec[1] = lambda_k1, a.lam_vec[2] = lambda_q2, a.lam_vec[3] = lambda_k2;
    a.lam_sh = lambda_sh, a.lam_init = lambda_init, a.lengths = key_lengths;
    a.B = B, a.Tq = Tq, a.Tk = Tk, a.H = H, a.Hk = Hk, a.D = D, a.Dv = Dv, a.causal = flags & ND_ATTN_CAUSAL;
    a.scale = scale, a.c = scale * 1.4426950408889634f;
    if (int rc = diff_check(fn, a, dtype)) return rc;
    if (int rc = diff_bwd_check(fn, a, dtype)) return rc;
    a.g = H / Hk;
    NDB_REQUIRE(out1 && out2 && lse && dout && dq && dk && dv && workspace, fn, "null pointer");
    const int per = dtype == ND_DT_BF16 ? 8 : 4;
    NDB_REQUIRE(aligned_to(dout, 16) && do_sb % per == 0 && do_st % per == 0 && do_sh % per == 0 && do_st >= 0 && do_st <= (1 << 22), fn,
                "rows of the output's gradient must be 16-byte aligned");
    NDB_REQUIRE(aligned_to(out1, 16) && aligned_to(out2, 16) && aligned_to(dq, 16) && aligned_to(dk, 16) && aligned_to(dv, 16), fn, "pointers must be 16-byte aligned");
    const DiffBwdPlan pl = diff_bwd_plan(B, Tq, Tk, H, Hk, D, Dv, dtype == ND_DT_BF16 ? 2 : 4, a.causal);
    p.waves = pl.waves, p.key_blocks = pl.key_blocks, p.row_splits = pl.row_splits, p.key_splits = pl.key_splits, p.chunk = pl.chunk;
    NDB_REQUIRE(aligned_to(workspace, 16), fn, "workspace must be 16-byte aligned");
    p.dout = {dout, do_sb, do_st, do_sh};
    p.o1 = out1, p.o2 = out2, p.lse = lse, p.dq = dq, p.dk = dk, p.dv = dv;
    p.dvec[0] = dlambda_q1, p.dvec[1] = dlambda_k1, p.dvec[2] = dlambda_q2, p.dvec[3] = dlambda_k2;
    p.dots = workspace;
    p.dlam_part = workspace + pl.dots;
    p.part_kv = workspace + pl.dots + pl.dlam;
    p.part_q = p.part_kv + pl.kv;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return dtype == ND_DT_BF16 ? dispatch_diff_bwd<__bf16>(fn, p, st) : dispatch_diff_bwd<float>(fn, p, st);
}
