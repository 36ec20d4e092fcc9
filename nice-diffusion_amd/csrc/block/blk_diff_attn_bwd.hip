// Differential attention, backward.  With P1, P2 the two maps (rebuilt from the scores and the kept log denominators), dP = dO V^T
// and, per row, D1 = dO . O1, D2 = dO . O2 (the maps' own outputs, kept by the forward pass):
//   dV = (P1 - lam P2)^T dO     dS1 = P1 (dP - D1)     dS2 = -lam P2 (dP - D2)
//   dq_i = s dS_i k_i           dk_i = s dS_i^T q_i    dlam = -sum P2 dP, which scales the gradients of the four vectors
//
// Three launches without atomics: D1 / D2; keys (a wave owns 32 keys, the rows of all query heads pass by: dk, dv and its share
// of dlam); queries (a wave owns 32 rows, the keys pass by: dq).  Both rebuild the scores: 28 D T^2 operations for Dv = 2 D in all
// where 20 would do with the maps kept, but nothing of T x T is stored.  Scores and dP come out of the matrix unit in the layout
// in which dS is the next product's operand; the transposed operands are column reads of the same row-major tiles.
// dlam is summed from fp32 P2 and dP, not from the rounded O2: it is one number and may cancel.  Rounding to bf16 besides the
// outputs: P1 - lam P2, dS1, dS2 as operands, O1 and O2.  A sequence of one key has constant maps: dq and dk are made exactly zero.
#include "blk_diff_attn.h"

namespace ndb {

int diff_head_dim(int D, int Dv);
int diff_check(const char* fn, const DiffArgs& a, int dtype);

struct DiffBwdArgs {
    DiffArgs f;
    DiffTensor dout;              // [B, Tq, H, Dv]
    const void *o1, *o2;
    const float* lse;             // [2][B, Tq, H]
    float* dots;                  // [2][B, Tq, H]: D1, D2
    float* dlam_part;             // [B * Hk][key blocks][4 waves][g]
    float* dlam;                  // [H]
    void *dq, *dk, *dv;           // contiguous
    void* dvec[4];
    int key_blocks;
};

// D1, D2 of a row: 16 lanes, 8 channels at a time
template <typename T>
__global__ void __launch_bounds__(256) diff_dots_kernel(const DiffBwdArgs p) {
    const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4, all = (int64_t)p.f.B * p.f.Tq * p.f.H;
    if (row >= all) return;
    const int lane = threadIdx.x & 15;
    const int h = (int)(row % p.f.H);
    const int64_t bt = row / p.f.H;
    const int b = (int)(bt / p.f.Tq), t = (int)(bt - (int64_t)b * p.f.Tq);
    const T* g = static_cast<const T*>(p.dout.p) + b * p.dout.sb + t * p.dout.st + h * p.dout.sh;
    float d1 = 0.f, d2 = 0.f;
    for (int d = lane * 8; d < p.f.Dv; d += 128) {
        float x[8], y[8], z[8];
        load_vec<T, 8>(g + d, x);
        load_vec<T, 8>(static_cast<const T*>(p.o1) + row * p.f.Dv + d, y);
        load_vec<T, 8>(static_cast<const T*>(p.o2) + row * p.f.Dv + d, z);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            d1 = fmaf(x[e], y[e], d1);
            d2 = fmaf(x[e], z[e], d2);
        }
    }
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        d1 += __shfl_xor(d1, o, 64);
        d2 += __shfl_xor(d2, o, 64);
    }
    if (lane == 0) {
        p.dots[row] = d1;
        p.dots[all + row] = d2;
    }
}

template <typename T, int HD>
struct DiffBwdShape {
    static constexpr int ES = (int)sizeof(T), DV = 2 * HD, RB = 2 * HD * ES;      // q / k rows and dO / v rows: equally long
    static constexpr int PH = HD * ES / 16, NS = PH / 2, NSV = RB / 32;
    static constexpr int RT = (ES == 4 && HD == 128) ? 32 : 64;                   // rows (or keys) of a tile
    static constexpr int STAGE = 2 * RT * RB;
};

template <typename T, int HD>
constexpr int diff_dkv_lds() { return 2 * DiffBwdShape<T, HD>::STAGE + 2 * 4 * DiffBwdShape<T, HD>::RT * 4 + DIFF_MAX_GROUP * 4; }

// DK, DV: which gradients this launch makes.  Wide heads take two launches: the outputs and operands of both do not fit the registers
template <typename T, int HD, bool DK, bool DVG>
__global__ void __launch_bounds__(256, (HD == 32 ? 2 : 1)) diff_dkv_kernel(const DiffBwdArgs p) {
    using S = DiffBwdShape<T, HD>;
    using TR = Tile<T, S::RB>;
    constexpr int RT = S::RT;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* const stat = reinterpret_cast<float*>(smem + 2 * S::STAGE);            // [2][lse1, lse2, D1, D2][RT]
    float* const lam_s = stat + 2 * 4 * RT;
    const DiffArgs& f = p.f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, lh = lane >> 5;
    int id = xcd_run(blockIdx.x, gridDim.x);
    const int bh = id / p.key_blocks, kb = id - bh * p.key_blocks;
    const int b = bh / f.Hk, hk = bh - b * f.Hk;
    const int len = diff_length(f.lengths, b, f.Tk);
    const int key0 = kb * 128, key = key0 + wave * 32 + l31;
    const bool kin = key < len;

    for (int h = wave; h < f.g; h += 4) {
        float e1, e2;
        diff_lambda<T>(f, hk * f.g + h, lane, e1, e2);
        if (lane == 0) lam_s[h] = e1 - e2 + f.lam_init;
    }
    u32x4 kf[2][S::NS], vf[DK ? S::NSV : 1];
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
        if constexpr (DK) {
#pragma unroll
            for (int c = 0; c < S::NSV; ++c) {
                const int by = (2 * c + lh) * 16;
                vf[c] = u32x4{0u, 0u, 0u, 0u};
                if (kin && by < f.Dv * S::ES) vf[c] = *reinterpret_cast<const u32x4*>(vp + by);
            }
        }
    }
    f32x16 dk[2][DK ? HD / 32 : 1], dv[DVG ? S::DV / 32 : 1];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
#pragma unroll
        for (int d = 0; d < (DK ? HD / 32 : 1); ++d) dk[0][d][e] = dk[1][d][e] = 0.f;
#pragma unroll
        for (int d = 0; d < (DVG ? S::DV / 32 : 1); ++d) dv[d][e] = 0.f;
    }

    TileLoad<T, S::RB, RT, 4> lq, lo;
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
    const int64_t rows_all = (int64_t)f.B * f.Tq * f.H;
    float sv = 0.f;                                           // this thread's row statistic of the stage in flight
    auto fetch = [&](int i, int stage) {
        const int hg = i / per_head, t0 = (tile0 + i - hg * per_head) * RT, head = hk * f.g + hg;
        char* at = smem + stage * S::STAGE;
        const int64_t n = f.Tq - t0;
        lq.load(at, static_cast<const T*>(f.q.p) + b * f.q.sb + (int64_t)t0 * f.q.st + head * f.q.sh, ((n - 1) * f.q.st + 2 * f.D) * S::ES, wave);
        lo.load(at + RT * S::RB, static_cast<const T*>(p.dout.p) + b * p.dout.sb + (int64_t)t0 * p.dout.st + head * p.dout.sh,
                ((n - 1) * p.dout.st + f.Dv) * S::ES, wave);
        const int which = threadIdx.x / RT, t = t0 + (int)threadIdx.x - which * RT;
        sv = which < 2 ? INFINITY : 0.f;
        if (which < 4 && t < f.Tq) {
            const int64_t row = ((int64_t)b * f.Tq + t) * f.H + head;
            sv = (which < 2 ? p.lse : p.dots)[(which & 1) * rows_all + row];
        }
    };
    float dl = 0.f;
    if (total) fetch(0, 0);
    for (int i = 0; i < total; ++i) {
        const int stage = i & 1;
        if ((int)threadIdx.x < 4 * RT) stat[stage * 4 * RT + threadIdx.x] = sv;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (i + 1 < total) fetch(i + 1, stage ^ 1);
        const int hg = i / per_head, t0 = (tile0 + i - hg * per_head) * RT;
        const float lam = lam_s[hg];
        const char* tq = smem + stage * S::STAGE;
        const char* to = tq + RT * S::RB;
        const float* st = stat + stage * 4 * RT + 4 * lh;
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
                for (int c = 0; c < S::NS; ++c) s[m] = mma_step<T>(TR::row(q32, rb, 0, m * S::PH + 2 * c), kf[m][c], s[m]);
            }
            if constexpr (DK) {
#pragma unroll
                for (int e = 0; e < 16; ++e) dp[e] = 0.f;
#pragma unroll
                for (int c = 0; c < S::NSV; ++c) dp = mma_step<T>(TR::row(o32, rb, 0, 2 * c), vf[c], dp);
            }
            // rows that see this lane's key: from `first` on (causal), none past the sequence's end
            const int first = kin ? (f.causal ? key - len + f.Tq - t0 - r32 - 4 * lh : -0x40000000) : 0x40000000;
            Probs<T> pd, d1, d2;
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const f32x4 l1 = *reinterpret_cast<const f32x4*>(st + r32 + 8 * g4), l2 = *reinterpret_cast<const f32x4*>(st + RT + r32 + 8 * g4);
                const f32x4 c1 = *reinterpret_cast<const f32x4*>(st + 2 * RT + r32 + 8 * g4), c2 = *reinterpret_cast<const f32x4*>(st + 3 * RT + r32 + 8 * g4);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int e = 4 * g4 + j;
                    const bool in = j + 8 * g4 >= first;
                    float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][e], f.c, -l1[j])), p2 = __builtin_amdgcn_exp2f(fmaf(s[1][e], f.c, -l2[j]));
                    p1 = in ? p1 : 0.f;
                    p2 = in ? p2 : 0.f;
                    if constexpr (DVG) pd.set(e, p1 - lam * p2);
                    if constexpr (DK) {
                        dl = fmaf(p2, dp[e], dl);
                        d1.set(e, p1 * (dp[e] - c1[j]));
                        d2.set(e, -lam * p2 * (dp[e] - c2[j]));
                    }
                }
            }
            if constexpr (DVG) {
#pragma unroll
                for (int d = 0; d < S::DV / 32; ++d) dv[d] = mma_cols<T, S::RB>(o32, cb, 0, d * 32, pd, dv[d]);
            }
            if constexpr (DK) {
#pragma unroll
                for (int d = 0; d < HD / 32; ++d) {
                    dk[0][d] = mma_cols<T, S::RB>(q32, cb, 0, d * 32, d1, dk[0][d]);
                    dk[1][d] = mma_cols<T, S::RB>(q32, cb, 0, HD + d * 32, d2, dk[1][d]);
                }
            }
        }
        if (DK && i + 1 == (hg + 1) * per_head) {             // this head's rows are through
#pragma unroll
            for (int o = 32; o; o >>= 1) dl += __shfl_xor(dl, o, 64);
            if (lane == 0) p.dlam_part[(((int64_t)bh * p.key_blocks + kb) * 4 + wave) * f.g + hg] = -dl;
            dl = 0.f;
        }
    }
    if (DK && total == 0)
        for (int h = lane; h < f.g; h += 64) p.dlam_part[(((int64_t)bh * p.key_blocks + kb) * 4 + wave) * f.g + h] = 0.f;
    if (key >= f.Tk) return;
    const int64_t krow = ((int64_t)b * f.Tk + key) * f.Hk + hk;
    const float scale = len == 1 ? 0.f : f.scale;
    if constexpr (DK) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int d = 0; d < HD / 32; ++d)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int dd = d * 32 + 8 * g4 + 4 * lh;
                    const float v[4] = {dk[m][d][4 * g4] * scale, dk[m][d][4 * g4 + 1] * scale, dk[m][d][4 * g4 + 2] * scale, dk[m][d][4 * g4 + 3] * scale};
                    if (dd < f.D) store_vec<T, 4>(static_cast<T*>(p.dk) + krow * 2 * f.D + m * f.D + dd, v);
                }
    }
    if constexpr (DVG) {
#pragma unroll
        for (int d = 0; d < S::DV / 32; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int dd = d * 32 + 8 * g4 + 4 * lh;
                const float v[4] = {dv[d][4 * g4], dv[d][4 * g4 + 1], dv[d][4 * g4 + 2], dv[d][4 * g4 + 3]};
                if (dd < f.Dv) store_vec<T, 4>(static_cast<T*>(p.dv) + krow * f.Dv + dd, v);
            }
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(256, (HD * (int)sizeof(T) >= 256 ? 1 : 2)) diff_dq_kernel(const DiffBwdArgs p) {
    using S = DiffBwdShape<T, HD>;
    using TR = Tile<T, S::RB>;
    constexpr int KT = S::RT;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    float* const lam_s = reinterpret_cast<float*>(smem + 2 * S::STAGE);
    const DiffArgs& f = p.f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, lh = lane >> 5;
    const int rows = f.Tq * f.g, tiles = (rows + 127) / 128;
    const int id = xcd_run(blockIdx.x, gridDim.x);
    const int bh = id / tiles, tile = f.causal ? tiles - 1 - (id - bh * tiles) : id - bh * tiles;
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
    const float l1 = p.lse[orow], l2 = p.lse[rows_all + orow], c1 = p.dots[orow], c2 = p.dots[rows_all + orow];
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
    auto fetch = [&](int key, int stage) {
        char* at = smem + stage * S::STAGE;
        const int64_t n = len - key;
        lk.load(at, kp + (int64_t)key * f.k.st, ((n - 1) * f.k.st + 2 * f.D) * S::ES, wave);
        lv.load(at + KT * S::RB, vp + (int64_t)key * f.v.st, ((n - 1) * f.v.st + f.Dv) * S::ES, wave);
    };
    const int row_base = TR::row_base(lane), col_base = TR::col_base(lane);
    if (0 < kend) fetch(0, 0);
    int stage = 0;
    for (int key0 = 0; key0 < kend; key0 += KT, stage ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (key0 + KT < kend) fetch(key0 + KT, stage ^ 1);
#pragma unroll 1
        for (int k32 = 0; k32 < KT; k32 += 32) {
            const int kb = key0 + k32;
            if (kb >= kend) break;
            const char* tk = smem + stage * S::STAGE + k32 * S::RB;
            const char* tv = tk + KT * S::RB;
            const int rb = in_loop(row_base), cb = in_loop(col_base);
            f32x16 s[2], dp;
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int e = 0; e < 16; ++e) s[m][e] = 0.f;
#pragma unroll
                for (int c = 0; c < S::NS; ++c) s[m] = mma_step<T>(TR::row(tk, rb, 0, m * S::PH + 2 * c), q[m][c], s[m]);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) dp[e] = 0.f;
#pragma unroll
            for (int c = 0; c < S::NSV; ++c) dp = mma_step<T>(TR::row(tv, rb, 0, 2 * c), go[c], dp);
            Probs<T> d1, d2;
            const int left = seen - kb - 4 * lh;              // keys of this block the row sees
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const bool in = (e & 3) + 8 * (e >> 2) < left;
                float p1 = __builtin_amdgcn_exp2f(fmaf(s[0][e], f.c, -l1)), p2 = __builtin_amdgcn_exp2f(fmaf(s[1][e], f.c, -l2));
                p1 = in ? p1 : 0.f;
                p2 = in ? p2 : 0.f;
                d1.set(e, p1 * (dp[e] - c1));
                d2.set(e, nlam * p2 * (dp[e] - c2));
            }
#pragma unroll
            for (int d = 0; d < HD / 32; ++d) {
                dq[0][d] = mma_cols<T, S::RB>(tk, cb, 0, d * 32, d1, dq[0][d]);
                dq[1][d] = mma_cols<T, S::RB>(tk, cb, 0, HD + d * 32, d2, dq[1][d]);
            }
        }
    }
    if (r0 + l31 >= rows) return;
    const float scale = len == 1 ? 0.f : f.scale;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int d = 0; d < HD / 32; ++d)
#pragma unroll
            for (int g4 = 0; g4 < 4; ++g4) {
                const int dd = d * 32 + 8 * g4 + 4 * lh;
                const float v[4] = {dq[m][d][4 * g4] * scale, dq[m][d][4 * g4 + 1] * scale, dq[m][d][4 * g4 + 2] * scale, dq[m][d][4 * g4 + 3] * scale};
                if (dd < f.D) store_vec<T, 4>(static_cast<T*>(p.dq) + orow * 2 * f.D + m * f.D + dd, v);
            }
}

// dlam[h]: the partials of one head in a fixed order
__global__ void __launch_bounds__(256) diff_dlam_kernel(const DiffBwdArgs p) {
    __shared__ float red[256];
    const int head = blockIdx.x, hk = head / p.f.g, hg = head - hk * p.f.g, per = p.key_blocks * 4;
    float t = 0.f;
    for (int i = threadIdx.x; i < p.f.B * per; i += 256) {
        const int b = i / per, j = i - b * per;
        t += p.dlam_part[(((int64_t)b * p.f.Hk + hk) * per + j) * p.f.g + hg];
    }
    red[threadIdx.x] = t;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) p.dlam[head] = red[0];
}

// the four vectors' gradients: one wave per head, or one for all heads where they share the vectors
template <typename T>
__global__ void __launch_bounds__(64) diff_dvec_kernel(const DiffBwdArgs p) {
    const int lane = threadIdx.x;
    float e1, e2;
    diff_lambda<T>(p.f, p.f.lam_sh ? (int)blockIdx.x : 0, lane, e1, e2);
    float dlam = 0.f;
    if (p.f.lam_sh)
        dlam = p.dlam[blockIdx.x];
    else
        for (int h = 0; h < p.f.H; ++h) dlam += p.dlam[h];
    const int64_t at = blockIdx.x * p.f.lam_sh;
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

template <typename T, int HD, bool DK, bool DVG>
static int launch_dkv(const char* fn, const DiffBwdArgs& a, hipStream_t st) {
    auto kern = diff_dkv_kernel<T, HD, DK, DVG>;
    static bool attr_set[kMaxDevices] = {};
    if (int rc = ensure_max_lds(reinterpret_cast<const void*>(kern), attr_set, fn)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.f.B * a.f.Hk * a.key_blocks)), dim3(256), (diff_dkv_lds<T, HD>()), st, a);
    return check_launch(fn);
}

template <typename T, int HD>
static int launch_diff_bwd(const char* fn, const DiffBwdArgs& a, hipStream_t st) {
    const int64_t rows = (int64_t)a.f.B * a.f.Tq * a.f.H;
    hipLaunchKernelGGL((diff_dots_kernel<T>), dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a);
    if constexpr (HD == 128) {
        if (int rc = launch_dkv<T, HD, true, false>(fn, a, st)) return rc;
        if (int rc = launch_dkv<T, HD, false, true>(fn, a, st)) return rc;
    } else {
        if (int rc = launch_dkv<T, HD, true, true>(fn, a, st)) return rc;
    }
    auto kern = diff_dq_kernel<T, HD>;
    static bool attr_set[kMaxDevices] = {};
    if (int rc = ensure_max_lds(reinterpret_cast<const void*>(kern), attr_set, fn)) return rc;
    const int tiles = (a.f.Tq * a.f.g + 127) / 128;
    hipLaunchKernelGGL(kern, dim3((unsigned)(a.f.B * a.f.Hk * tiles)), dim3(256), 2 * (DiffBwdShape<T, HD>::STAGE) + DIFF_MAX_GROUP * 4, st, a);
    if (a.dvec[0] || a.dvec[1] || a.dvec[2] || a.dvec[3]) {
        hipLaunchKernelGGL(diff_dlam_kernel, dim3((unsigned)a.f.H), dim3(256), 0, st, a);
        hipLaunchKernelGGL((diff_dvec_kernel<T>), dim3((unsigned)(a.f.lam_sh ? a.f.H : 1)), dim3(64), 0, st, a);
    }
    return check_launch(fn);
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

extern "C" int64_t nd_diff_attention_bwd_workspace_floats(int B, int Tq, int Tk, int H, int Hk) {
    if (B <= 0 || Tq <= 0 || Tk <= 0 || H <= 0 || Hk <= 0 || H % Hk) return -1;
    return 2LL * B * Tq * H + (int64_t)B * H * ((Tk + 127) / 128) * 4 + H;
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
    a.g = H / Hk;
    NDB_REQUIRE(out1 && out2 && lse && dout && dq && dk && dv && workspace, fn, "null pointer");
    const int per = dtype == ND_DT_BF16 ? 8 : 4;
    NDB_REQUIRE(aligned_to(dout, 16) && do_sb % per == 0 && do_st % per == 0 && do_sh % per == 0 && do_st >= 0 && do_st <= (1 << 22), fn,
                "rows of the output's gradient must be 16-byte aligned");
    NDB_REQUIRE(aligned_to(out1, 16) && aligned_to(out2, 16) && aligned_to(dq, 16) && aligned_to(dk, 16) && aligned_to(dv, 16), fn, "pointers must be 16-byte aligned");
    p.key_blocks = (Tk + 127) / 128;
    NDB_REQUIRE((int64_t)B * Hk * p.key_blocks <= (1 << 24) && (int64_t)B * Hk * (((int64_t)Tq * a.g + 127) / 128) <= (1 << 24), fn, "too many workgroups for one launch");
    p.dout = {dout, do_sb, do_st, do_sh};
    p.o1 = out1, p.o2 = out2, p.lse = lse, p.dq = dq, p.dk = dk, p.dv = dv;
    p.dvec[0] = dlambda_q1, p.dvec[1] = dlambda_k1, p.dvec[2] = dlambda_q2, p.dvec[3] = dlambda_k2;
    p.dots = workspace;
    p.dlam_part = workspace + 2LL * B * Tq * H;
    p.dlam = p.dlam_part + (int64_t)B * H * p.key_blocks * 4;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return dtype == ND_DT_BF16 ? dispatch_diff_bwd<__bf16>(fn, p, st) : dispatch_diff_bwd<float>(fn, p, st);
}
