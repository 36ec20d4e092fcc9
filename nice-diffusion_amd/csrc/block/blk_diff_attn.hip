// Differential attention, forward:  o = (softmax(s q1 k1^T) - lam softmax(s q2 k2^T)) v,  lam = exp(lq1.lk1) - exp(lq2.lk2) + lam_init
//
// q [B, Tq, H, 2D], k [B, Tk, Hk, 2D]: the two halves of a head's channels are the two maps' queries and keys; v [B, Tk, Hk, Dv].
// The query heads of one key head are rows beside each other: row r of a (batch, key head) is token r / g, head r % g, so one
// pass over the keys serves all of them.
//
// One pass with running maxima and sums for both maps: per 32 keys x 32 rows  S^T = K Q^T  twice, exponentials, O^T += V^T P^T
// twice (the V fragments are read once).  As in the plain attention kernels a lane holds one row's scores (accumulator as the
// next product's operand); V^T comes from transposed LDS reads of the row-major tile.  The two outputs stay apart to the end:
// their scales are only known then.  Alternatively the maps could be joined before the product (two thirds of its operations),
// at the price of a pass over the scores for the statistics: the same matrix operations and twice the exponentials.
//   prefill    4 waves x 32 rows, tiles of 64 keys (fp32 with D > 64: 32), a ring of two (bf16, D <= 32: three), loads straight to
//              LDS.  bf16, 8 x 2048^2 x 8 heads of 64 + 128: 227 us (0.91 PFLOP/s of matrix operations), causal 132 (141 with what the
//              backward pass reads written too); 64 x 1024^2 x 6 heads of 32 + 64: 212 us.  Bound by the SIMD's issue: matrix operations
//              and the softmax's vector operations add up rather than overlap (a fused multiply-add 2.5 cycles beside them, an
//              exponential 2.8 to 8)
//   few rows   (g Tq <= 32: single tokens) a kernel of its own: diff_few_kernel
//   wide heads (D > 64) 128 value channels a workgroup, the scores made twice when Dv is above that: both maps' outputs and the
//              queries of 256 channels do not fit the registers (measured: 290 spilled)
//   splits     when (batch, key head, row tile) does not fill the chip the keys are divided over workgroups; fp32 partial
//              outputs, joined in split order by a second launch
// No maximum is taken of a tile as a rule: its weights are made against the row's reference of before, and only where their sum
// passes 2^10 (or nothing was seen so far) the reference moves to the tile's maximum and they are made again: a weight stays
// below 2^10, as exact in floating point as one below 1.  Rounding to bf16 besides the output: the weights p as the second product's
// operand; their sum is taken from the rounded values.
#include "blk_diff_attn.h"

namespace ndb {

template <typename T, int HD>
struct DiffShape {
    static constexpr int ES = (int)sizeof(T), DV = HD == 128 ? 128 : 2 * HD;      // value channels of a workgroup
    static constexpr int RBK = 2 * HD * ES, RBV = DV * ES;
    static constexpr int PH = HD * ES / 16;                  // pieces of one half of a key row
    static constexpr int NS = PH / 2;                        // steps of a score product
    static constexpr int NDT = DV / 32;
    static constexpr int KT_MANY = (ES == 4 && HD == 128) ? 32 : 64;
    // few rows: each wave has a tile of 32 keys of its own, up to 128 KiB together
    static constexpr int TILE_FEW = 32 * (RBK + RBV);
    static constexpr int NW_FEW = TILE_FEW <= 16384 ? 8 : (TILE_FEW <= 32768 ? 4 : 2);
};

// four channels dd .. of output row `orow` from both maps' sums and their statistics (maximum, sum of weights, twice)
template <typename T>
__device__ __forceinline__ void diff_store(const DiffArgs& p, int64_t orow, int dd, const f32x4 (&o)[2], const f32x4& st, float lam, bool first) {
    float a[4], c[4], y[4];
    const float i1 = st[1] != 0.f ? 1.f / st[1] : 0.f, i2 = st[3] != 0.f ? 1.f / st[3] : 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        a[e] = o[0][e] * i1;
        c[e] = o[1][e] * i2;
        y[e] = a[e] - lam * c[e];
    }
    store_vec<T, 4>(static_cast<T*>(p.out) + orow * p.Dv + dd, y);
    if (p.o1) {
        store_vec<T, 4>(static_cast<T*>(p.o1) + orow * p.Dv + dd, a);
        store_vec<T, 4>(static_cast<T*>(p.o2) + orow * p.Dv + dd, c);
    }
    if (p.lse && first) {
        p.lse[orow] = st[1] != 0.f ? st[0] + log2f(st[1]) : INFINITY;
        p.lse[(int64_t)p.B * p.Tq * p.H + orow] = st[3] != 0.f ? st[2] + log2f(st[3]) : INFINITY;
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(256, (HD * (int)sizeof(T) >= 256 ? 1 : (HD == 32 && sizeof(T) == 2 ? 3 : 2))) diff_attn_kernel(const DiffArgs p) {
    using S = DiffShape<T, HD>;
    constexpr int KT = S::KT_MANY, NW = 4;                    // keys of a tile, waves
    constexpr int NJ = 1;                                     // 32-key blocks at a time (2 at D <= 32: 181 registers for 142, no faster)
    constexpr int STAGE = KT * (S::RBK + S::RBV);
    constexpr int NST = HD == 32 && S::ES == 2 ? 3 : 2;       // tiles in LDS
    using TK = Tile<T, S::RBK>;
    using TV = Tile<T, S::RBV>;
    __shared__ __attribute__((aligned(16))) char stages[NST * STAGE];
    __shared__ float lam_s[DIFF_MAX_GROUP];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, lh = lane >> 5;

    const int rows = p.Tq * p.g, tiles = (rows + 127) / 128;
    int bh, id;
    unit_of(blockIdx.x, gridDim.x, p.B * p.Hk, p.causal, bh, id);
    const int vb = HD == 128 ? id / (tiles * p.splits) : 0, dv0 = vb * S::DV, dvn = p.Dv - dv0 < S::DV ? p.Dv - dv0 : S::DV;
    id -= vb * tiles * p.splits;
    const int sp = id / tiles, tile = tiles - 1 - (id - sp * tiles);      // longest rows first
    const int b = bh / p.Hk, hk = bh - b * p.Hk;
    const int len = diff_length(p.lengths, b, p.Tk);

    // this lane's row
    const int r0 = tile * 128 + wave * 32;
    const int r = r0 + l31 < rows ? r0 + l31 : rows - 1;
    const int t = r / p.g, hg = r - t * p.g, head = hk * p.g + hg;
    const int seen = p.causal ? t + len - p.Tq + 1 : len;      // keys this row sees (<= 0: none)
    int last = len;                                            // keys the workgroup needs
    if (p.causal) {
        const int rl = (tile + 1) * 128 - 1 < rows ? (tile + 1) * 128 - 1 : rows - 1;
        last = rl / p.g + len - p.Tq + 1;
    }
    const int kbeg = sp * p.chunk;
    int kend = kbeg + p.chunk < last ? kbeg + p.chunk : last;

    for (int h = wave; h < (p.splits == 1 ? p.g : 0); h += NW) {      // divided keys: the join makes them
        float e1, e2;
        diff_lambda<T>(p, hk * p.g + h, lane, e1, e2);
        if (lane == 0) lam_s[h] = e1 - e2 + p.lam_init;
    }

    u32x4 q[2][S::NS];
    {
        const char* qp = reinterpret_cast<const char*>(static_cast<const T*>(p.q.p) + b * p.q.sb + t * p.q.st + head * p.q.sh);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int c = 0; c < S::NS; ++c) {
                const int by = (2 * c + lh) * 16;
                q[m][c] = u32x4{0u, 0u, 0u, 0u};
                if (by < p.D * S::ES) q[m][c] = *reinterpret_cast<const u32x4*>(qp + m * p.D * S::ES + by);
            }
    }
    f32x16 o[2][S::NDT];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int d = 0; d < S::NDT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[m][d][e] = 0.f;
    float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    TileLoad<T, S::RBK, KT, NW> lk;
    TileLoad<T, S::RBV, KT, NW> lv;
    lk.template init<S::RBK / 2>(p.k.st * S::ES, p.D * S::ES, wave, lane);
    lv.template init<S::RBV>(p.v.st * S::ES, dvn * S::ES, wave, lane);
    const T* kp = static_cast<const T*>(p.k.p) + b * p.k.sb + hk * p.k.sh;
    const T* vp = static_cast<const T*>(p.v.p) + b * p.v.sb + hk * p.v.sh + dv0;
    auto fetch = [&](int i, char* at) {                       // keys at or past the sequence's end become zero rows
        const int key = kbeg + i * KT;
        const int64_t n = len - key;
        lk.load(at, kp + (int64_t)key * p.k.st, ((n - 1) * p.k.st + 2 * p.D) * S::ES, wave);
        lv.load(at + KT * S::RBK, vp + (int64_t)key * p.v.st, ((n - 1) * p.v.st + dvn) * S::ES, wave);
    };
    const int row_base = TK::row_base(lane), col_base = TV::col_base(lane);
    auto compute = [&](int i, const char* tk) {
        const int key0 = kbeg + i * KT;
        const char* tv = tk + KT * S::RBK;
#pragma unroll 1
        for (int sub = 0; sub < KT / 32; sub += NJ) {
            const int kb = key0 + sub * 32;
            if (kb >= kend) break;
            const int rb = in_loop(row_base), cb = in_loop(col_base);
            const char* k32 = tk + sub * 32 * S::RBK;
            const char* v32 = tv + sub * 32 * S::RBV;
            f32x16 s[2][NJ];
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int m = 0; m < 2; ++m) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[m][j][e] = 0.f;
#pragma unroll
                    for (int c = 0; c < S::NS; ++c)
                        if (!no_step<T, HD>(c, p.D)) s[m][j] = mma_step<T>(TK::row(k32, rb, 32 * j, m * S::PH + 2 * c), q[m][c], s[m][j]);
                }
            // scores past what a row sees: only in the tile that holds a row's end
            const bool cut = p.causal ? kb + 32 * NJ > r0 / p.g + len - p.Tq + 1 : kb + 32 * NJ > len;
            if (cut) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const bool in = kb + 32 * j + (e & 3) + 8 * (e >> 2) + 4 * lh < seen;
                        s[0][j][e] = in ? s[0][j][e] : -INFINITY;
                        s[1][j][e] = in ? s[1][j][e] : -INFINITY;
                    }
            }
            Probs<T> pr[2][NJ];
            float sum[2];
            auto weights = [&](int m) {                       // sum: this lane half's keys; the halves meet at the end
                const float ref = mx[m] == -INFINITY ? 0.f : mx[m];
                sum[m] = 0.f;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) pr[m][j].set(e, __builtin_amdgcn_exp2f(fmaf(s[m][j][e], p.c, -ref)));
                    sum[m] += pr[m][j].sum();
                }
            };
            weights(0);
            weights(1);
            const bool again = mx[0] == -INFINITY || mx[1] == -INFINITY || fmaxf(sum[0], sum[1]) > 1024.f;
            if (__builtin_amdgcn_ballot_w64(again) != 0) {
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    float top = -INFINITY;
#pragma unroll
                    for (int j = 0; j < NJ; ++j)
#pragma unroll
                        for (int e = 0; e < 16; e += 2) top = fmaxf(fmaxf(s[m][j][e], s[m][j][e + 1]), top);
                    top = half_max(top) * p.c;
                    const bool move = top > mx[m];
                    const float a = move ? __builtin_amdgcn_exp2f(mx[m] - top) : 1.f;
                    mx[m] = move ? top : mx[m];
                    l[m] *= a;
#pragma unroll
                    for (int d = 0; d < S::NDT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[m][d][e] *= a;
                    weights(m);
                }
            }
            l[0] += sum[0];
            l[1] += sum[1];
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                if constexpr (S::ES == 2) {
#pragma unroll
                    for (int d = 0; d < S::NDT; d += 2) {     // the value fragments serve both maps
                        u32x4 f[2][2];
                        TV::cols2(v32, cb, 32 * j, d * 32, f);
#pragma unroll
                        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
                            for (int x = 0; x < 2; ++x)
#pragma unroll
                                for (int m = 0; m < 2; ++m) {
                                    union { u32x4 u; bf16x8 h; } a;
                                    a.u = f[x][s2];
                                    o[m][d + x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.h, pr[m][j].f[s2], o[m][d + x], 0, 0, 0);
                                }
                    }
                } else {
#pragma unroll
                    for (int d = 0; d < S::NDT; ++d) {
                        if (HD < 128 && d && 32 * d >= dvn) break;
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float a = TV::one(v32, cb, 32 * j, e, d * 32);
                            o[0][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, pr[0][j].f[e], o[0][d], 0, 0, 0);
                            o[1][d] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, pr[1][j].f[e], o[1][d], 0, 0, 0);
                        }
                    }
                }
            }
        }
    };
    ring<NST, decltype(lk)::NI + decltype(lv)::NI>(stages, STAGE, kend > kbeg ? (kend - kbeg + KT - 1) / KT : 0, fetch, compute);
    l[0] = half_sum(l[0]);
    l[1] = half_sum(l[1]);
    __syncthreads();                                          // lam_s is written; the stages are free

    if (r0 + l31 >= rows) return;
    if (p.splits > 1) {
        float* at = p.part + ((int64_t)sp * p.B * p.Hk * rows + (int64_t)bh * rows + r) * (2 * p.Dv + 4);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int d = 0; d < S::NDT; ++d)
#pragma unroll
                for (int g4 = 0; g4 < 4; ++g4) {
                    const int dd = d * 32 + 8 * g4 + 4 * lh;
                    const f32x4 v = {o[m][d][4 * g4], o[m][d][4 * g4 + 1], o[m][d][4 * g4 + 2], o[m][d][4 * g4 + 3]};
                    if (dd < dvn) *reinterpret_cast<f32x4*>(at + m * p.Dv + dv0 + dd) = v;
                }
        if (lh == 0 && vb == 0) *reinterpret_cast<f32x4*>(at + 2 * p.Dv) = f32x4{mx[0], l[0], mx[1], l[1]};
        return;
    }
    const f32x4 st = {mx[0], l[0], mx[1], l[1]};
    const int64_t orow = ((int64_t)b * p.Tq + t) * p.H + head;
#pragma unroll
    for (int d = 0; d < S::NDT; ++d)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const int dd = d * 32 + 8 * g4 + 4 * lh;
            f32x4 sum[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) sum[m] = f32x4{o[m][d][4 * g4], o[m][d][4 * g4 + 1], o[m][d][4 * g4 + 2], o[m][d][4 * g4 + 3]};
            if (dd < dvn) diff_store<T>(p, orow, dv0 + dd, sum, st, lam_s[hg], dd == 0 && vb == 0);
        }
}

// Few rows: a read of the cache.  8 waves (fewer for wide tiles), each with a tile of 32 keys of its own, no barrier; the next keys
// are requested when the scores are made, the next values when the outputs are, so about 3/4 of 128 KiB a CU is under way.
// A row's two maps are two columns of the products (column 16 m + row: 16 rows a workgroup), so one exponential a key and lane and
// one product with the values serve both; the scores are made with either half of the keys, and a lane takes those of its own map.
// What the bf16 weights leave out is a second bf16 operand here (49.3 us becomes 50.0, and the error is the output's rounding alone).
// 16 tokens, 16 heads on 4, 64 + 128 channels, ragged caches up to 8192 (197 MB, 38 us as a copy): 48.5 us with the join; with 128-key
// tiles for the whole workgroup in two stages 62, four 32-key stages for each of 2 waves 81, accumulators for either map 51.
template <typename T, int HD>
__global__ void __launch_bounds__((64 * DiffShape<T, HD>::NW_FEW), (HD * (int)sizeof(T) >= 256 ? 1 : 2)) diff_few_kernel(const DiffArgs p) {
    using S = DiffShape<T, HD>;
    using TK = Tile<T, S::RBK>;
    using TV = Tile<T, S::RBV>;
    constexpr int NW = S::NW_FEW, STAGE = S::TILE_FEW;
    constexpr bool REST = S::ES == 2;
    static_assert(S::NDT * 4096 <= STAGE, "a wave's part of the join fits its tile");
    __shared__ __attribute__((aligned(16))) char stages[NW * STAGE];
    __shared__ float ml[NW][32][2], lam_s[DIFF_MAX_GROUP];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, lh = lane >> 5, map = l31 >> 4;

    // nothing to share: the (batch, key head)s in turn, so that every XCD has long and short sequences
    const int rows = p.Tq * p.g, tiles = (rows + 15) / 16;
    int id = blockIdx.x / (p.B * p.Hk);
    const int bh = blockIdx.x - id * (p.B * p.Hk);
    const int vb = HD == 128 ? id / (tiles * p.splits) : 0, dv0 = vb * S::DV, dvn = p.Dv - dv0 < S::DV ? p.Dv - dv0 : S::DV;
    id -= vb * tiles * p.splits;
    const int sp = id / tiles, tile = id - sp * tiles;
    const int b = bh / p.Hk, hk = bh - b * p.Hk;
    const int len = diff_length(p.lengths, b, p.Tk);

    const int r0 = tile * 16, r = r0 + (l31 & 15) < rows ? r0 + (l31 & 15) : rows - 1;
    const int t = r / p.g, hg = r - t * p.g;
    const int seen = p.causal ? t + len - p.Tq + 1 : len;      // keys this row sees (<= 0: none)
    const int cut_from = p.causal ? r0 / p.g + len - p.Tq + 1 : len;      // keys from here on are not seen by every row
    const int rl = r0 + 15 < rows ? r0 + 15 : rows - 1;
    const int last = p.causal ? rl / p.g + len - p.Tq + 1 : len;
    const int kbeg = sp * p.chunk, kend = kbeg + p.chunk < last ? kbeg + p.chunk : last;

    for (int h = wave; h < (p.splits == 1 ? p.g : 0); h += NW) {      // divided keys: the join makes them
        float e1, e2;
        diff_lambda<T>(p, hk * p.g + h, lane, e1, e2);
        if (lane == 0) lam_s[h] = e1 - e2 + p.lam_init;
    }
    u32x4 q[S::NS];
    {
        const char* qp = reinterpret_cast<const char*>(static_cast<const T*>(p.q.p) + b * p.q.sb + t * p.q.st + (hk * p.g + hg) * p.q.sh + map * p.D);
#pragma unroll
        for (int c = 0; c < S::NS; ++c) {
            const int by = (2 * c + lh) * 16;
            q[c] = u32x4{0u, 0u, 0u, 0u};
            if (by < p.D * S::ES) q[c] = *reinterpret_cast<const u32x4*>(qp + by);
        }
    }
    f32x16 o[S::NDT];
#pragma unroll
    for (int d = 0; d < S::NDT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float mx = -INFINITY, l = 0.f;

    TileLoad<T, S::RBK, 32, 1> lk;
    TileLoad<T, S::RBV, 32, 1> lv;
    lk.template init<S::RBK / 2>(p.k.st * S::ES, p.D * S::ES, 0, lane);
    lv.template init<S::RBV>(p.v.st * S::ES, dvn * S::ES, 0, lane);
    const T* kp = static_cast<const T*>(p.k.p) + b * p.k.sb + hk * p.k.sh;
    const T* vp = static_cast<const T*>(p.v.p) + b * p.v.sb + hk * p.v.sh + dv0;
    char* const tk = stages + wave * STAGE;
    char* const tv = tk + 32 * S::RBK;
    const int first = kbeg + wave * 32, n = kend > first ? (kend - first + 32 * NW - 1) / (32 * NW) : 0;      // the waves take tiles in turn
    auto fetch_k = [&](int i) {                               // keys at or past the sequence's end become zero rows
        const int key = first + i * 32 * NW;
        lk.load(tk, kp + (int64_t)key * p.k.st, ((int64_t)(len - key - 1) * p.k.st + 2 * p.D) * S::ES, 0);
    };
    auto fetch_v = [&](int i) {
        const int key = first + i * 32 * NW;
        lv.load(tv, vp + (int64_t)key * p.v.st, ((int64_t)(len - key - 1) * p.v.st + dvn) * S::ES, 0);
    };
    constexpr int NK = decltype(lk)::NI, NV = decltype(lv)::NI;
    const int row_base = TK::row_base(lane), col_base = TV::col_base(lane);
    if (n > 0) {
        fetch_k(0);
        fetch_v(0);
    }
    for (int i = 0; i < n; ++i) {
        const int kb = first + i * 32 * NW;
        const int rb = in_loop(row_base), cb = in_loop(col_base);
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NV) : "memory");      // the tile's keys are there
        f32x16 s, s2;
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = s2[e] = 0.f;
#pragma unroll
        for (int c = 0; c < S::NS; ++c)
            if (!no_step<T, HD>(c, p.D)) {
                s = mma_step<T>(TK::row(tk, rb, 0, 2 * c), q[c], s);
                s2 = mma_step<T>(TK::row(tk, rb, 0, S::PH + 2 * c), q[c], s2);
            }
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = map ? s2[e] : s[e];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + 1 < n) {                                      // the next tile's keys after the scores, its values after the outputs
            fetch_k(i + 1);
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NK) : "memory");      // this tile's values are there
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (kb + 32 > cut_from) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[e] = kb + (e & 3) + 8 * (e >> 2) + 4 * lh < seen ? s[e] : -INFINITY;
        }
        Probs<T> pr, rest;
        float sum;
        auto weights = [&] {                                  // sum: this lane half's keys; the halves meet at the end
            const float ref = mx == -INFINITY ? 0.f : mx;
            sum = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[e], p.c, -ref));
                sum += w;
                pr.set(e, w);
                if constexpr (REST) rest.set(e, w - (float)(__bf16)w);
            }
        };
        weights();
        const bool again = mx == -INFINITY || sum > 1024.f;
        if (__builtin_amdgcn_ballot_w64(again) != 0) {
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; e += 2) top = fmaxf(fmaxf(s[e], s[e + 1]), top);
            top = half_max(top) * p.c;
            const bool move = top > mx;
            const float a = move ? __builtin_amdgcn_exp2f(mx - top) : 1.f;
            mx = move ? top : mx;
            l *= a;
#pragma unroll
            for (int d = 0; d < S::NDT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= a;
            weights();
        }
        l += sum;
        mma_cols<T, S::RBV>(tv, cb, 0, 0, dvn, pr, o);
        if constexpr (REST) mma_cols<T, S::RBV>(tv, cb, 0, 0, dvn, rest, o);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (i + 1 < n) fetch_v(i + 1);
    }
    l = half_sum(l);

    // join the waves: a common maximum, then the outputs added in wave order, each element by one thread
    if (lh == 0) {
        ml[wave][l31][0] = mx;
        ml[wave][l31][1] = l;
    }
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < NW; ++w) top = fmaxf(top, ml[w][l31][0]);
    const float f = __builtin_amdgcn_exp2f(mx - (top == -INFINITY ? 0.f : top));
#pragma unroll
    for (int d = 0; d < S::NDT; ++d)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4)
            *reinterpret_cast<f32x4*>(tk + l31 * (S::NDT * 128) + (((d * 8 + 2 * g4 + lh) ^ (l31 & 7)) << 4)) =
                f32x4{o[d][4 * g4] * f, o[d][4 * g4 + 1] * f, o[d][4 * g4 + 2] * f, o[d][4 * g4 + 3] * f};
    __syncthreads();
    constexpr int PC = S::NDT * 8;                            // 16-byte pieces of a row and map
    const int here = rows - r0 < 16 ? rows - r0 : 16;
    for (int e = threadIdx.x; e < here * PC; e += NW * 64) {
        const int row = e / PC, pc = e - row * PC, dd = pc * 4;
        if (dd >= dvn) continue;
        f32x4 out[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, st;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int col = 16 * m + row;
            float tp = -INFINITY, sum = 0.f;
            for (int w = 0; w < NW; ++w) tp = fmaxf(tp, ml[w][col][0]);
            for (int w = 0; w < NW; ++w) {
                sum += ml[w][col][1] * __builtin_amdgcn_exp2f(ml[w][col][0] - (tp == -INFINITY ? 0.f : tp));
                out[m] += *reinterpret_cast<const f32x4*>(stages + w * STAGE + col * (S::NDT * 128) + ((pc ^ (col & 7)) << 4));
            }
            st[2 * m] = tp;
            st[2 * m + 1] = sum;
        }
        const bool lead = dd == 0 && vb == 0;
        if (p.splits > 1) {
            float* at = p.part + ((int64_t)sp * p.B * p.Hk * rows + (int64_t)bh * rows + r0 + row) * (2 * p.Dv + 4);
            *reinterpret_cast<f32x4*>(at + dv0 + dd) = out[0];
            *reinterpret_cast<f32x4*>(at + p.Dv + dv0 + dd) = out[1];
            if (lead) *reinterpret_cast<f32x4*>(at + 2 * p.Dv) = st;
            continue;
        }
        const int tt = (r0 + row) / p.g, h = r0 + row - tt * p.g;
        diff_store<T>(p, ((int64_t)b * p.Tq + tt) * p.H + hk * p.g + h, dv0 + dd, out, st, lam_s[h], lead);
    }
}

// Joins the splits of a row: a group of G lanes, 4 channels a lane.  The lanes share the reads that come before the outputs (the
// lambda vectors, the splits' statistics), which by one lane each were the launch's whole time; from 8 splits on all groups of the
// workgroup share a row (1 token, 32768 keys, 64 splits: 45 us of the call's 64 before).
template <typename T>
__global__ void __launch_bounds__(256) diff_join_kernel(const DiffArgs p, int G, int groups) {
    __shared__ float part[256][10];
    const int rows = p.Tq * p.g, lane = threadIdx.x & (G - 1), dd = lane * 4, group = groups > 1 ? threadIdx.x / G : 0;
    const int64_t all = (int64_t)p.B * p.Hk * rows, row = groups > 1 ? blockIdx.x : ((int64_t)blockIdx.x * 256 + threadIdx.x) / G;
    if (row >= all) return;                                   // whole groups; whole workgroups where they share
    const int bh = (int)(row / rows), r = (int)(row - (int64_t)bh * rows), b = bh / p.Hk, hk = bh - b * p.Hk;
    const int t = r / p.g, head = hk * p.g + (r - t * p.g);
    const int LD = 2 * p.Dv + 4;
    const float* at = p.part + row * LD;
    const int64_t step = all * LD;
    float e1 = 0.f, e2 = 0.f, top[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    {
        const T* v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = static_cast<const T*>(p.lam_vec[i]) + head * p.lam_sh;
        for (int d = lane; d < p.D; d += G) {
            e1 = fmaf((float)v[0][d], (float)v[1][d], e1);
            e2 = fmaf((float)v[2][d], (float)v[3][d], e2);
        }
    }
    for (int s = lane; s < p.splits; s += G) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(at + s * step + 2 * p.Dv);
        top[0] = fmaxf(top[0], v[0]);
        top[1] = fmaxf(top[1], v[2]);
    }
    for (int o = 1; o < G; o <<= 1) {
        e1 += __shfl_xor(e1, o, 64);
        e2 += __shfl_xor(e2, o, 64);
        top[0] = fmaxf(top[0], __shfl_xor(top[0], o, 64));
        top[1] = fmaxf(top[1], __shfl_xor(top[1], o, 64));
    }
    f32x4 o[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    if (dd < p.Dv) {
#pragma unroll 4
        for (int s = group; s < p.splits; s += groups) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(at + s * step + 2 * p.Dv);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float f = __builtin_amdgcn_exp2f(v[2 * m] - (top[m] == -INFINITY ? 0.f : top[m]));
                l[m] += v[2 * m + 1] * f;
                o[m] += *reinterpret_cast<const f32x4*>(at + s * step + m * p.Dv + dd) * f;
            }
        }
    }
    if (groups > 1) {                                         // in group order
#pragma unroll
        for (int m = 0; m < 2; ++m) {
#pragma unroll
            for (int e = 0; e < 4; ++e) part[threadIdx.x][5 * m + e] = o[m][e];
            part[threadIdx.x][5 * m + 4] = l[m];
        }
        __syncthreads();
        if (group) return;
        for (int g = 1; g < groups; ++g)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
#pragma unroll
                for (int e = 0; e < 4; ++e) o[m][e] += part[g * G + lane][5 * m + e];
                l[m] += part[g * G + lane][5 * m + 4];
            }
    }
    if (dd >= p.Dv) return;
    const f32x4 st = {top[0], l[0], top[1], l[1]};
    diff_store<T>(p, ((int64_t)b * p.Tq + t) * p.H + head, dd, o, st, expf(e1) - expf(e2) + p.lam_init, dd == 0);
}

// padded head dim of the kernels: the smallest of 32 / 64 / 128 that holds D and half of Dv
int diff_head_dim(int D, int Dv) {
    const int n = D > (Dv + 1) / 2 ? D : (Dv + 1) / 2;
    return n <= 32 ? 32 : (n <= 64 ? 64 : 128);
}

int diff_bwd_check(const char* fn, const DiffArgs& a, int dtype);      // blk_diff_attn_bwd.hip

struct DiffPlan {
    bool few;
    int splits, chunk;
};

// Into how many parts `length` (keys, rows) is divided: the fewest rounds of workgroups x their time, plus the join.  `units`
// workgroups without a division, `slots` of them on the chip at a time, `per` cycles of a CU per unit of length and workgroup,
// `bytes` of fp32 partials per part, written and read at ~5 TB/s (2.3 KiB a cycle); shares are multiples of `grain`.  Causal ones
// are of all lengths and start with the longest, so rounds say little: none from 256 workgroups on (8 x 2048^2 x 8 heads with
// gradients: 540 us, 710 divided), else about 512 (1 x 4096^2, 4 heads on one: 190 us, 246 by the rounds).  Against the best of ten
// divisions (profiles/block_attention_divisions.txt) the choices take 4 and 2 % longer on the mean (rows and keys of the backward pass,
// 11 shapes in three types and widths each), causal ones 14, 10 and 8 % (forward, rows, keys; 12 shapes), most where 256 workgroups
// are those of a few long sequences (1 x 8192^2 x 4 heads: 288 us, 168 in three parts).
int diff_parts(int64_t units, int slots, int64_t length, int64_t grain, double per, double bytes, int causal, int64_t& share) {
    double best_t = 1e300;
    int best = 1;
    share = length;
    if (causal) {
        int64_t n = units < 256 ? 512 / units : 1, most = (int64_t)((double)length * per / 24000.0) + 1;      // no share under 24000 cycles
        n = n < 1 ? 1 : (n < 16 ? n : 16);
        n = n < most ? n : most;
        share = ((length + n - 1) / n + grain - 1) / grain * grain;
        return (int)((length + share - 1) / share);
    }
    for (int want = 1; want <= 64; ++want) {
        const int64_t chunk = ((length + want - 1) / want + grain - 1) / grain * grain, parts = (length + chunk - 1) / chunk;
        if (parts != want) continue;
        const int64_t rounds = (units * parts + slots - 1) / slots, active = units * parts < slots ? (units * parts + 255) / 256 : slots / 256;
        double t = (double)rounds * ((double)chunk * per * active + 6000.0);
        if (parts > 1) t += 9000.0 + 300.0 * (double)parts + 2.0 * (double)parts * bytes / 2340.0;
        if (t < best_t) best_t = t, best = (int)parts, share = chunk;
    }
    return best;
}

// Few rows: ~256 workgroups, one for each CU (the case above: 50 us; 512 even out ragged lengths, but a second start and join cost
// more: 58 us, 1024: 74), no split under two tiles for each wave (4 x 8 heads, 2048 keys: 18 us for 20 with one).  fp32: 118 us for
// 393 MB there (76 us as a copy).  The form ends at 32 rows of a key head: 4 sequences, 16 heads on 4, 8192 keys, causal, 8 new tokens
// 22.9 us, 9 tokens 33.9, 128 tokens 97 (24.8 of matrix operations).  Many: a workgroup's 32 keys take its CU ~30 HD cycles, fp32
// ~190 HD.
static DiffPlan diff_plan(int B, int Tq, int Tk, int H, int Hk, int D, int Dv, int es, int causal) {
    const int g = H / Hk, rows = Tq * g, hd = diff_head_dim(D, Dv);
    DiffPlan pl{rows <= 32, 1, Tk};
    const int64_t units = (int64_t)B * Hk * (pl.few ? (rows + 15) / 16 : (rows + 127) / 128) * (hd == 128 ? (Dv + 127) / 128 : 1);
    if (pl.few) {
        const int tile = 32 * (2 * hd + (hd == 128 ? 128 : 2 * hd)) * es, grain = 32 * (tile <= 16384 ? 8 : (tile <= 32768 ? 4 : 2));      // a tile for each wave
        int64_t n = 256 / units, most = (Tk + 2 * grain - 1) / (2 * grain);
        n = n < most ? n : most;
        n = n < 1 ? 1 : (n < 64 ? n : 64);
        const int64_t chunk = ((Tk + n - 1) / n + grain - 1) / grain * grain;
        pl.chunk = (int)chunk;
        pl.splits = (int)((Tk + chunk - 1) / chunk);
    } else {
        int64_t chunk;
        const int slots = 256 * (es == 4 ? (hd == 32 ? 2 : 1) : (hd == 32 ? 3 : (hd == 64 ? 2 : 1)));
        pl.splits = diff_parts(units, slots, Tk, 64, es == 4 ? 6.0 * hd : 0.95 * hd, (double)B * Tq * H * (2 * Dv + 4) * 4, causal, chunk);
        pl.chunk = (int)chunk;
    }
    return pl;
}

template <typename T, int HD>
static int launch_diff(const char* fn, const DiffArgs& a, bool few, hipStream_t st) {
    const int rows = a.Tq * a.g, per = few ? 16 : 128;
    const int vblocks = (a.Dv + DiffShape<T, HD>::DV - 1) / DiffShape<T, HD>::DV;
    const int64_t blocks = (int64_t)a.B * a.Hk * ((rows + per - 1) / per) * a.splits * vblocks;
    NDB_REQUIRE(grid_fits(blocks, few ? 64 * DiffShape<T, HD>::NW_FEW : 256), fn, "too many workgroups for one launch");
    if (few) hipLaunchKernelGGL((diff_few_kernel<T, HD>), dim3((unsigned)blocks), dim3(64 * DiffShape<T, HD>::NW_FEW), 0, st, a);
    else hipLaunchKernelGGL((diff_attn_kernel<T, HD>), dim3((unsigned)blocks), dim3(256), 0, st, a);
    if (a.splits > 1) {
        const int G = a.Dv <= 64 ? 16 : (a.Dv <= 128 ? 32 : 64);
        const int64_t all = (int64_t)a.B * a.Hk * rows;
        const int groups = a.splits >= 8 && all <= 16384 ? 256 / G : 1;
        hipLaunchKernelGGL((diff_join_kernel<T>), dim3((unsigned)(groups > 1 ? all : (all * G + 255) / 256)), dim3(256), 0, st, a, G, groups);
    }
    return check_launch(fn);
}

template <typename T>
static int dispatch_diff(const char* fn, const DiffArgs& a, bool few, hipStream_t st) {
    switch (diff_head_dim(a.D, a.Dv)) {
        case 32: return launch_diff<T, 32>(fn, a, few, st);
        case 64: return launch_diff<T, 64>(fn, a, few, st);
        default: return launch_diff<T, 128>(fn, a, few, st);
    }
}

int diff_check(const char* fn, const DiffArgs& a, int dtype) {
    NDB_REQUIRE(dtype == ND_DT_F32 || dtype == ND_DT_BF16, fn, "dtype must be ND_DT_F32 or ND_DT_BF16");
    NDB_REQUIRE(a.B > 0 && a.Tq > 0 && a.Tk > 0 && a.H > 0 && a.Hk > 0, fn, "sizes must be positive");
    NDB_REQUIRE(a.H % a.Hk == 0 && a.H / a.Hk <= DIFF_MAX_GROUP, fn, "query heads must be a multiple of the key heads, at most 64 times as many");
    NDB_REQUIRE(a.H <= (1 << 20), fn, "more than 2^20 heads");
    NDB_REQUIRE(a.D > 0 && a.D % 8 == 0 && a.D <= 128, fn, "head dim must be a multiple of 8 and at most 128");
    NDB_REQUIRE(a.Dv > 0 && a.Dv % 8 == 0 && a.Dv <= 256, fn, "value dim must be a multiple of 8 and at most 256");
    NDB_REQUIRE((int64_t)a.Tq * a.H < (1LL << 30) && a.Tk < (1 << 30), fn, "too many tokens");
    NDB_REQUIRE(a.scale > 0.f, fn, "scale must be positive");
    const int per = dtype == ND_DT_BF16 ? 8 : 4;
    const DiffTensor* t[3] = {&a.q, &a.k, &a.v};
    for (const DiffTensor* x : t) {
        NDB_REQUIRE(x->p, fn, "null pointer");
        NDB_REQUIRE(aligned_to(x->p, 16) && x->sb % per == 0 && x->st % per == 0 && x->sh % per == 0, fn, "rows must be 16-byte aligned");
        NDB_REQUIRE(x->st >= 0 && x->st <= (1 << 22), fn, "token stride must be 0 .. 2^22 elements");
    }
    for (const void* v : a.lam_vec) NDB_REQUIRE(v && aligned_to(v, 16), fn, "lambda vectors must be given, 16-byte aligned");
    return ND_OK;
}

}  // namespace ndb

using namespace ndb;

extern "C" int64_t nd_diff_attention_workspace_floats(int B, int Tq, int Tk, int H, int Hk, int D, int Dv, int dtype) {
    if (B <= 0 || Tq <= 0 || Tk <= 0 || H <= 0 || Hk <= 0 || H % Hk || D <= 0 || D > 128 || Dv <= 0 || Dv > 256) return -1;
    int splits = 1;
    for (int causal = 0; causal < 2; ++causal) {
        const DiffPlan pl = diff_plan(B, Tq, Tk, H, Hk, D, Dv, dtype == ND_DT_BF16 ? 2 : 4, causal);
        splits = pl.splits > splits ? pl.splits : splits;
    }
    return splits > 1 ? (int64_t)splits * B * Tq * H * (2 * Dv + 4) : 0;
}

extern "C" int nd_diff_attention(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                                 int64_t k_sh, const void* v, int64_t v_sb, int64_t v_st, int64_t v_sh, const void* lambda_q1,
                                 const void* lambda_k1, const void* lambda_q2, const void* lambda_k2, int64_t lambda_sh, float lambda_init,
                                 const int* key_lengths, void* out, void* out1, void* out2, float* lse, float* workspace, int B, int Tq,
                                 int Tk, int H, int Hk, int D, int Dv, float scale, int flags, int dtype, nd_stream_t stream) {
    const char* fn = "nd_diff_attention";
    DiffArgs a{};
    a.q = {q, q_sb, q_st, q_sh}, a.k = {k, k_sb, k_st, k_sh}, a.v = {v, v_sb, v_st, v_sh};
    a.lam_vec[0] = lambda_q1, a.lam_vec[1] = lambda_k1, a.lam_vec[2] = lambda_q2, a.lam_vec[3] = lambda_k2;
    a.lam_sh = lambda_sh, a.lam_init = lambda_init, a.lengths = key_lengths;
    a.out = out, a.o1 = out1, a.o2 = out2, a.lse = lse, a.part = workspace;
    a.B = B, a.Tq = Tq, a.Tk = Tk, a.H = H, a.Hk = Hk, a.D = D, a.Dv = Dv, a.causal = flags & ND_ATTN_CAUSAL;
    a.scale = scale, a.c = scale * 1.4426950408889634f;
    if (int rc = diff_check(fn, a, dtype)) return rc;
    a.g = H / Hk;
    NDB_REQUIRE(out && aligned_to(out, 16) && (!out1 || (out2 && lse && aligned_to(out1, 16) && aligned_to(out2, 16))), fn, "outputs missing or not 16-byte aligned");
    if (int rc = lse ? diff_bwd_check(fn, a, dtype) : ND_OK) return rc;
    const DiffPlan pl = diff_plan(B, Tq, Tk, H, Hk, D, Dv, dtype == ND_DT_BF16 ? 2 : 4, a.causal);
    a.splits = pl.splits, a.chunk = pl.chunk;
    NDB_REQUIRE(pl.splits == 1 || (workspace && aligned_to(workspace, 16)), fn, "workspace missing");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    return dtype == ND_DT_BF16 ? dispatch_diff<__bf16>(fn, a, pl.few, st) : dispatch_diff<float>(fn, a, pl.few, st);
}
