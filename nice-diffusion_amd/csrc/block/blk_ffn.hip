// Gated feed-forward block, forward and backward:
//   [a | u] = x w_in^T + b_in,   h = act(a) u,   y = residual + h w_out^T + b_out            (x [M, C], w_in [2F, C], w_out [C, F])
//   dh = dy w_out;  da = dh u act'(a);  du = dh act(a);  dx = [da | du] w_in;
//   dw_in = [da | du]^T x;  dw_out = dy^T h;  db_in, db_out: column sums of [da | du], dy
//
// Six matrix products on the engine of blk_gemm.h.  The first makes the gate and the up columns of the same f in one wave, so
// activation and product happen on the fp32 accumulators; its backward twin (dh) applies the derivative the same way.  MFMA
// bound for long inputs: 6 M C F operations forward, 12 backward.
//
// Roundings to bf16 besides the outputs: h (operand of the second product), a and u where a backward pass will want them
// (they are what it reads instead of repeating the first product: 2/9 of its operations), da and du (operands of two
// products).  Each is off by half a unit, 2^-8 relative; fp32 calls round nothing to fewer bits.  In either type silu, gelu_tanh and the
// slope of gelu take the hardware's exponential (its argument rounded to fp32 first) and reciprocal, 1 ulp each.
//
// Measured, bf16: 16384 x 1024 x 4096 with gradients 1250 us (0.99 PFLOP/s; six products alone by the library: 1240), 65536 x 384 x
// 1024 forward with gelu 233 us (0.66; 215 replayed on one input).  The parts are at the kernels and launch choices below.
#include "blk_gemm.h"

namespace ndb {

// f = act(a), df = act'(a).  The normal distribution of gelu: fp32 calls take the library's error function; in bf16 calls, whose
// results carry 8 bits, Hastings' rational form serves both it and the slope with one exponential (Abramowitz and Stegun 7.1.26:
// erfc(x) = t P(t) exp(-x^2), t = 1 / (1 + 0.3275911 x), to 1.5e-7): with erff the epilogue took 60 of the 265 us of the first
// product of ffn at 65536 x 384 x 1024.
template <typename T, int ACT>
__device__ __forceinline__ void act_and_slope(float a, float& f, float& df) {
    if constexpr (ACT == ND_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-a));
        f = a * s;
        df = s * (1.f + a * (1.f - s));
    } else if constexpr (ACT == ND_ACT_GELU) {
        float cdf, pdf = __expf(-0.5f * a * a);
        if constexpr (sizeof(T) == 2) {
            const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, fabsf(a), 1.f));
            const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f);
            const float tail = 0.5f * poly * pdf;             // of the normal distribution beyond |a|
            cdf = a < 0.f ? tail : 1.f - tail;
        } else {
            cdf = 0.5f * (1.f + erff(a * 0.70710678118654752f));
        }
        f = a * cdf;
        df = fmaf(a * 0.3989422804014327f, pdf, cdf);
    } else {      // 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z)),  z = sqrt(2 / pi) (a + 0.044715 a^3)
        const float z2 = 1.5957691216057308f * a * (1.f + 0.044715f * a * a);
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z2));
        f = a * s;
        df = s + a * s * (1.f - s) * 1.5957691216057308f * (1.f + 0.134145f * a * a);
    }
}

// Epilogues: columns(n) what a lane needs for its 8 columns, row(m, n) what it reads for one row of them (requested ahead of the
// row's turn), store(...) the rest.
struct None {};

template <typename T>
struct Eight {            // 8 elements as they lie
    u32x4 r[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) r[i] = reinterpret_cast<const u32x4*>(p)[i];
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 2) {
            union { unsigned u; float f; } c;
            const unsigned w = r[0][i >> 1];
            c.u = i & 1 ? w & 0xffff0000u : w << 16;
            return c.f;
        } else {
            union { unsigned u; float f; } c;
            c.u = r[i >> 2][i & 3];
            return c.f;
        }
    }
};

template <typename T, int ACT>
struct EpiGate {          // h = act(a) u, and a | u where they are kept
    static constexpr bool GATED = true;
    using Row = None;
    struct Cols { float a[8], u[8]; };
    const T* bias;
    T* h;
    T* au;
    int F;
    __device__ __forceinline__ Cols columns(int f) const {
        Cols c;
        if (bias) {
            load_vec<T, 8>(bias + f, c.a);
            load_vec<T, 8>(bias + F + f, c.u);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) c.a[e] = c.u[e] = 0.f;
        }
        return c;
    }
    __device__ __forceinline__ Row row(int, int) const { return Row{}; }
    __device__ __forceinline__ void store(int m, int f, int, float (&a)[8], float (&u)[8], const Cols& c, const Row&) const {
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            a[e] += c.a[e];
            u[e] += c.u[e];
            float v, d;
            act_and_slope<T, ACT>(a[e], v, d);
            r[e] = v * u[e];
        }
        store_vec<T, 8>(h + (int64_t)m * F + f, r);
        if (au) {
            store_vec<T, 8>(au + (int64_t)m * 2 * F + f, a);
            store_vec<T, 8>(au + (int64_t)m * 2 * F + F + f, u);
        }
    }
};

template <typename T, int ACT>
struct EpiGateBwd {       // dh -> da | du
    static constexpr bool GATED = false;
    using Cols = None;
    struct Row { Eight<T> a, u; };
    const T* au;
    T* dau;
    int F;
    __device__ __forceinline__ Cols columns(int) const { return Cols{}; }
    __device__ __forceinline__ Row row(int m, int f) const {
        Row r;
        r.a.load(au + (int64_t)m * 2 * F + f);
        r.u.load(au + (int64_t)m * 2 * F + F + f);
        return r;
    }
    __device__ __forceinline__ void store(int m, int f, int, float (&dh)[8], float (&)[8], const Cols&, const Row& r) const {
        float da[8], du[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float v, d;
            act_and_slope<T, ACT>(r.a[e], v, d);
            da[e] = dh[e] * r.u[e] * d;
            du[e] = dh[e] * v;
        }
        store_vec<T, 8>(dau + (int64_t)m * 2 * F + f, da);
        store_vec<T, 8>(dau + (int64_t)m * 2 * F + F + f, du);
    }
};

template <typename T>
struct EpiOut {           // bias, residual, one rounding
    static constexpr bool GATED = false;
    struct Cols { float b[8]; };
    struct Row { Eight<T> r; };
    const T* bias;
    const T* res;
    T* out;
    int64_t ldr, ldo;
    __device__ __forceinline__ Cols columns(int n) const {
        Cols c;
        if (bias) {
            load_vec<T, 8>(bias + n, c.b);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) c.b[e] = 0.f;
        }
        return c;
    }
    __device__ __forceinline__ Row row(int m, int n) const {
        Row r;
        if (res) r.r.load(res + m * ldr + n);
        return r;
    }
    __device__ __forceinline__ void store(int m, int n, int, float (&v)[8], float (&)[8], const Cols& c, const Row& r) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += c.b[e];
        if (res) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += r.r[e];
        }
        store_vec<T, 8>(out + m * ldo + n, v);
    }
};

struct EpiPart {          // one split's fp32 partial
    static constexpr bool GATED = false;
    using Cols = None;
    using Row = None;
    float* out;
    int64_t ld, split;
    __device__ __forceinline__ Cols columns(int) const { return Cols{}; }
    __device__ __forceinline__ Row row(int, int) const { return Row{}; }
    __device__ __forceinline__ void store(int m, int n, int sp, float (&v)[8], float (&)[8], const Cols&, const Row&) const {
        store_vec<float, 8>(out + sp * split + m * ld + n, v);
    }
};

// the partials of a split product in split order, then the epilogue; 8 columns a thread
template <typename T>
__global__ void __launch_bounds__(256) gemm_join_kernel(const float* part, int splits, int M, int N, const EpiOut<T> epi) {
    const int64_t units = (int64_t)M * (N / 8);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < units; i += (int64_t)gridDim.x * 256) {
        const int m = (int)(i / (N / 8)), n = (int)(i - (int64_t)m * (N / 8)) * 8;
        const float* p = part + (int64_t)m * N + n;
        const auto c = epi.columns(n);
        const auto r = epi.row(m, n);
        float v[8];
        load_vec<float, 8>(p, v);
#pragma unroll 4
        for (int s = 1; s < splits; ++s) {
            float t[8];
            load_vec<float, 8>(p + s * (int64_t)M * N, t);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += t[e];
        }
        epi.store(m, n, 0, v, v, c, r);
    }
}

// Column sums of one or two matrices [M, N] at once: 8 columns a thread, 8 rows side by side a block; a partial row per block, then
// the rows in order.  (Both bias gradients in two launches instead of four:
// 139 us for 147 at 2355 x 264 x 680 in fp32, with all gradients.)
template <typename T>
struct ColSum {
    const T* src;
    int64_t ld;
    int N, rows;              // columns, row blocks
    float* part;              // [rows][N]
    T* out;
};

template <typename T>
__global__ void __launch_bounds__(256) colsum_kernel(const ColSum<T> first, const ColSum<T> second, int M) {
    __shared__ float red[8][257];
    const int blocks = (first.N + 255) / 256;
    const bool other = (int)blockIdx.x >= blocks;
    const ColSum<T>& p = other ? second : first;
    if ((int)blockIdx.y >= p.rows) return;
    const int bx = other ? blockIdx.x - blocks : blockIdx.x;
    const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, n = (bx * 32 + cx) * 8;
    float s[8] = {};
    if (n < p.N) {
#pragma unroll 4
        for (int m = blockIdx.y * 8 + ry; m < M; m += p.rows * 8) {
            float v[8];
            load_vec<T, 8>(p.src + m * p.ld + n, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += v[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[ry][cx * 8 + e] = s[e];
    __syncthreads();
    const int c = bx * 256 + threadIdx.x;
    if (c < p.N) {
        float t = 0.f;
#pragma unroll
        for (int r = 0; r < 8; ++r) t += red[r][threadIdx.x];
        p.part[(int64_t)blockIdx.y * p.N + c] = t;
    }
}

template <typename T>
__global__ void __launch_bounds__(1024) colsum_join_kernel(const ColSum<T> first, const ColSum<T> second) {
    __shared__ float red[32][33];
    const int blocks = (first.N + 31) / 32;
    const bool other = (int)blockIdx.x >= blocks;
    const ColSum<T>& p = other ? second : first;
    const int n = (other ? blockIdx.x - blocks : blockIdx.x) * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
    float t = 0.f;
    if (n < p.N)
        for (int r = lane; r < p.rows; r += 32) t += p.part[(int64_t)r * p.N + n];
    red[lane][threadIdx.x & 31] = t;
    __syncthreads();
    if (lane == 0 && n < p.N) {
        float u = 0.f;
        for (int l = 0; l < 32; ++l) u += red[l][threadIdx.x & 31];
        p.out[n] = (T)u;
    }
}

// ------------------------------------------------------------------------------------------------------------ few rows
// Up to 32 rows: a read of the weights.  A workgroup makes 16 columns (gated: the gate and the up columns of 16 f) of
// [M, N] = x w^T with 16 x 16 products, the weights' rows as their first operand; its waves take 128-byte pieces of the rows in
// turn, straight to registers, UNITS pieces requested at a time (bf16 4, fp32 2: 23 us for 24 at 1 x 1024 x 4096), and are summed
// in wave order.  Both operands take the channels of a piece in the same order, 16 bytes a lane.  Where columns are few (no more
// than one workgroup a CU) 8 columns: half of the operand stays empty, but twice the CUs read: 12.8 us for 13.9.
// The block at C 1024, F 4096, bf16 (25 MB, 4.9 us as a copy), replayed: 1 row 10.8 us (fp32 21.2), this form / the tiles at 4 rows
// 11.7 / 15.4, 16 rows 14.3 / 15.7, 32 rows 19.0 / 19.2.  Narrower weights gain up to 32 rows (384 / 1024: 9.3 / 12.7), wider ones lose
// from 17 on (2048 / 8192 at 32 rows: 41 / 31, fp32 93 / 61).
// What is left are two launches that each start, read for 2 to 3 us and drain.
constexpr int FEW_ROWS = 32, FEW_NARROW = 2048;

template <typename T, int NW, int MT, int COLS, class Epi>
__global__ void __launch_bounds__(NW * 64) few_rows_kernel(const T* x, int64_t ldx, const T* w, int M, int N, int K, const Epi epi) {
    constexpr int G = Epi::GATED ? 2 : 1, PIECE = 128 / (int)sizeof(T), LANE = 16 / (int)sizeof(T), UNITS = sizeof(T) == 2 ? 4 : 2;
    __shared__ __attribute__((aligned(16))) float red[NW][G][16 * MT][20];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l15 = lane & 15, l4 = lane >> 4, n0 = blockIdx.x * COLS;
    const T* rows[G];
#pragma unroll
    for (int g = 0; g < G; ++g) rows[g] = w + ((int64_t)g * N + n0 + l15) * K + l4 * LANE;
    const bool in_n = l15 < COLS && n0 + l15 < N;
    const int pieces = (K + PIECE - 1) / PIECE;
    f32x4 acc[MT][G];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int g = 0; g < G; ++g) acc[t][g] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int p0 = wave; p0 < pieces; p0 += NW * UNITS) {
        u32x4 a[UNITS][2][G], b[UNITS][2][MT];
#pragma unroll
        for (int i = 0; i < UNITS; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = (p0 + i * NW) * PIECE + h * (PIECE / 2);
                const bool in_k = k + l4 * LANE < K;
#pragma unroll
                for (int g = 0; g < G; ++g) {
                    a[i][h][g] = u32x4{0u, 0u, 0u, 0u};
                    if (in_k && in_n) a[i][h][g] = *reinterpret_cast<const u32x4*>(rows[g] + k);
                }
#pragma unroll
                for (int t = 0; t < MT; ++t) {
                    b[i][h][t] = u32x4{0u, 0u, 0u, 0u};
                    if (in_k && 16 * t + l15 < M) b[i][h][t] = *reinterpret_cast<const u32x4*>(x + (16 * t + l15) * ldx + l4 * LANE + k);
                }
            }
#pragma unroll
        for (int i = 0; i < UNITS; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        if constexpr (sizeof(T) == 2) {
                            union { u32x4 u; bf16x8 v; } p, q;
                            p.u = a[i][h][g], q.u = b[i][h][t];
                            acc[t][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(p.v, q.v, acc[t][g], 0, 0, 0);
                        } else {
                            union { u32x4 u; float f[4]; } p, q;
                            p.u = a[i][h][g], q.u = b[i][h][t];
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc[t][g] = __builtin_amdgcn_mfma_f32_16x16x4f32(p.f[e], q.f[e], acc[t][g], 0, 0, 0);
                        }
                    }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int g = 0; g < G; ++g) *reinterpret_cast<f32x4*>(&red[wave][g][16 * t + l15][l4 * 4]) = acc[t][g];
    const int m = threadIdx.x / (COLS / 8), c8 = (threadIdx.x % (COLS / 8)) * 8, n = n0 + c8;
    const bool mine = m < M && n < N;                         // 8 columns of a row (N is a multiple of 8)
    typename Epi::Cols cols{};
    typename Epi::Row row{};
    if (mine) {
        cols = epi.columns(n);
        row = epi.row(m, n);
    }
    __syncthreads();
    if (!mine) return;
    float v[G][8];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            f32x4 t = *reinterpret_cast<const f32x4*>(&red[0][g][m][c8 + e]);
#pragma unroll
            for (int u = 1; u < NW; ++u) t += *reinterpret_cast<const f32x4*>(&red[u][g][m][c8 + e]);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[g][e + j] = t[j];
        }
    epi.store(m, n, 0, v[0], v[G - 1], cols, row);
}

template <typename T, int NW, class Epi>
static int run_few(const char* fn, const T* x, int64_t ldx, const T* w, int M, int N, int K, const Epi& epi, hipStream_t st) {
    const int cols = N <= FEW_NARROW ? 8 : 16;
    auto kern = M <= 16 ? (cols == 8 ? few_rows_kernel<T, NW, 1, 8, Epi> : few_rows_kernel<T, NW, 1, 16, Epi>)
                        : (cols == 8 ? few_rows_kernel<T, NW, 2, 8, Epi> : few_rows_kernel<T, NW, 2, 16, Epi>);
    hipLaunchKernelGGL(kern, dim3((N + cols - 1) / cols), dim3(NW * 64), 0, st, x, ldx, w, M, N, K, epi);
    return check_launch(fn);
}

// ------------------------------------------------------------------------------------------------------ launch choices
struct Plan {
    int ti;               // tiles of 64 ti x 64 ti
    int splits, k_tiles;
};

// Time of a product in cycles of a CU (2.2 GHz), the constants fitted to 198 products of 33 feed-forward shapes, each timed with every
// tile and several divisions (profiles/block_products_by_tile.txt: the choices cost 1.6 % on the mean over the best ones).  A workgroup's stage (128
// bytes of k): bf16 3200 / 1120 / 380 at ti 4 / 2 / 1 (LDS and L2 traffic per operation: 275 GFLOP, 16384 x 1024 x 8192, took
// 230 / 265 / 484 us), fp32 the matrix units' 1024 ti^2, ti 1 a fifth more.  4 / ti workgroups share a CU; a stage takes ~850 to
// arrive.  What the epilogue moves (`moved`, bytes) goes at ~5 TB/s, worse where one workgroup has the CU to itself and nothing
// overlaps it (so does gelu's arithmetic: 65536 x 384 x 1024 forward, replayed, 233 us with ti 4, 215 with 2): the gate's backward product at 16384 x 4096 x 1024 takes 266 / 214 / 272 us, its forward one 283 / 305 / 418.
static Plan plan_gemm(int64_t M, int64_t N, int64_t K, int es, bool gated, bool gelu, bool may_split, double moved) {
    const int kt = 128 / es;
    const int64_t stages = (K + kt - 1) / kt;
    Plan best{};
    double best_t = 1e300;
    for (int ti = 4; ti; ti /= 2) {
        const int tile = 64 * ti;
        const int64_t tiles = ((M + tile - 1) / tile) * ((N + (gated ? tile / 2 : tile) - 1) / (gated ? tile / 2 : tile));
        const double stage = es == 4 ? (ti == 1 ? 1220.0 : 1024.0 * ti * ti) : (ti == 4 ? 3200.0 : (ti == 2 ? 1120.0 : 380.0));
        const double epilogue = moved / 2340.0 * (ti == 4 ? 1.2 : (ti == 2 ? 0.8 : 0.7));
        for (int want = 1; want <= (may_split ? 64 : 1); want *= 2) {
            const int64_t per = (stages + want - 1) / want;
            const int64_t splits = (stages + per - 1) / per;
            if (want > 1 && (per < 4 || splits * M * N > (1LL << 28))) break;
            if (ti < 4 && !grid_fits(tiles * splits, GEMM_THREADS)) break;
            const int64_t each = (tiles * splits + 255) / 256, rounds = (each + 4 / ti - 1) / (4 / ti);      // workgroups a CU
            const double work = (double)each * per * stage, wait = (double)rounds * per * 850.0;
            double t = (work > wait ? work : wait) + (double)rounds * (ti == 4 ? 8200.0 : (ti == 2 ? 4600.0 : 2600.0)) + epilogue;
            if (gelu) t += (double)each * (ti == 4 ? 14000.0 : (ti == 2 ? 600.0 : 150.0));
            // the join moves splits + 1 fp32 copies at ~1.7 KiB a cycle over the chip, and is a launch of its own
            if (splits > 1) t += 11000.0 + (double)(splits + 1) * M * N * 4 / 1700.0;
            if (t < best_t) {
                best_t = t;
                best = {ti, (int)splits, (int)per};
            }
        }
    }
    return best;
}

template <typename T, int TI, bool XK, bool WK, class Epi>
static int launch_gemm(const char* fn, const GemmSide<T>& x, const GemmSide<T>& w, int K, const Plan& pl, int gate, const Epi& epi, hipStream_t st) {
    constexpr int tile = 64 * TI;
    GemmArgs<T> a{};
    a.x = x, a.w = w, a.K = K, a.k_tiles = pl.k_tiles, a.splits = pl.splits, a.gate_rows = gate;
    a.tiles_m = (x.n + tile - 1) / tile;
    const int per_n = gate ? tile / 2 : tile, cols = gate ? gate : w.n;
    a.tiles_n = (cols + per_n - 1) / per_n;
    const int64_t blocks = (int64_t)a.tiles_m * a.tiles_n * pl.splits;
    NDB_REQUIRE(grid_fits(blocks, GEMM_THREADS), fn, "too many tiles for one launch");
    auto kern = gemm_kernel<T, TI, XK, WK, Epi>;
    static bool attr_set[kMaxDevices] = {};
    if (int rc = ensure_max_lds(reinterpret_cast<const void*>(kern), attr_set, fn)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)blocks), dim3(GEMM_THREADS), gemm_lds_bytes<TI>(), st, a, epi);
    return check_launch(fn);
}

template <typename T, bool XK, bool WK, class Epi>
static int run_gemm(const char* fn, const GemmSide<T>& x, const GemmSide<T>& w, int K, const Plan& pl, int gate, const Epi& epi, hipStream_t st) {
    switch (pl.ti) {
        case 4: return launch_gemm<T, 4, XK, WK>(fn, x, w, K, pl, gate, epi, st);
        case 2: return launch_gemm<T, 2, XK, WK>(fn, x, w, K, pl, gate, epi, st);
        default: return launch_gemm<T, 1, XK, WK>(fn, x, w, K, pl, gate, epi, st);
    }
}

// a product whose contraction may be split: straight to the output, or partials and their join
template <typename T, bool XK, bool WK>
static int run_gemm_out(const char* fn, const GemmSide<T>& x, const GemmSide<T>& w, int K, float* ws, const EpiOut<T>& epi, hipStream_t st) {
    const Plan pl = plan_gemm(x.n, w.n, K, sizeof(T), false, false, true, (double)x.n * w.n * sizeof(T));
    if (pl.splits == 1) return run_gemm<T, XK, WK>(fn, x, w, K, pl, 0, epi, st);
    NDB_REQUIRE(ws, fn, "workspace missing");
    const EpiPart part{ws, w.n, (int64_t)x.n * w.n};
    if (int rc = run_gemm<T, XK, WK>(fn, x, w, K, pl, 0, part, st)) return rc;
    const int64_t units = (int64_t)x.n * (w.n / 8);
    const int64_t blocks = (units + 255) / 256;
    hipLaunchKernelGGL((gemm_join_kernel<T>), dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(256), 0, st, ws, pl.splits, x.n, w.n, epi);
    return check_launch(fn);
}

static int64_t split_floats(int64_t M, int64_t N, int64_t K, int es) {
    const Plan pl = plan_gemm(M, N, K, es, false, false, true, (double)M * N * es);
    return pl.splits > 1 ? pl.splits * M * N : 0;
}

static int colsum_blocks(int64_t M, int64_t N) {
    const int64_t cols = (N + 255) / 256, rows = (M + 63) / 64;
    int64_t b = (2048 + cols - 1) / cols;
    if (b > rows) b = rows;
    return (int)(b < 1 ? 1 : (b > 1024 ? 1024 : b));
}

template <typename T>
static int run_colsum(const char* fn, const ColSum<T>& first, const ColSum<T>& second, int M, hipStream_t st) {
    const int rows = first.rows > second.rows ? first.rows : second.rows;
    hipLaunchKernelGGL((colsum_kernel<T>), dim3((first.N + 255) / 256 + (second.N + 255) / 256, rows), dim3(256), 0, st, first, second, M);
    hipLaunchKernelGGL((colsum_join_kernel<T>), dim3((first.N + 31) / 32 + (second.N + 31) / 32), dim3(1024), 0, st, first, second);
    return check_launch(fn);
}

template <typename T>
struct Ffn {
    const T *x, *w_in, *b_in, *w_out, *b_out, *res;
    T *y, *h, *au;
    int64_t ldx, ldr, ldy;
    float* ws;
    int M, C, F;
};

template <typename T, int ACT>
static int ffn_forward(const char* fn, const Ffn<T>& a, hipStream_t st) {
    const EpiGate<T, ACT> gate{a.b_in, a.h, a.au, a.F};
    const EpiOut<T> down{a.b_out, a.res, a.y, a.ldr, a.ldy};
    if (a.M <= FEW_ROWS) {
        if (int rc = run_few<T, 8>(fn, a.x, a.ldx, a.w_in, a.M, a.F, a.C, gate, st)) return rc;
        return run_few<T, 16>(fn, a.h, a.F, a.w_out, a.M, a.C, a.F, down, st);
    }
    const Plan pl = plan_gemm(a.M, a.F, a.C, sizeof(T), true, ACT != ND_ACT_SILU, false, (a.au ? 3.0 : 1.0) * a.M * a.F * sizeof(T));
    if (int rc = run_gemm<T, true, true>(fn, GemmSide<T>{a.x, a.ldx, a.M}, GemmSide<T>{a.w_in, a.C, 2 * a.F}, a.C, pl, a.F, gate, st))
        return rc;
    return run_gemm_out<T, true, true>(fn, GemmSide<T>{a.h, a.F, a.M}, GemmSide<T>{a.w_out, a.F, a.C}, a.F, a.ws, down, st);
}

template <typename T>
struct FfnBwd {
    const T *dy, *x, *w_in, *w_out, *au, *h;
    T *dx, *dw_in, *db_in, *dw_out, *db_out, *dau;
    int64_t lddy, ldx;
    float* ws;
    int M, C, F;
};

template <typename T, int ACT>
static int ffn_backward(const char* fn, const FfnBwd<T>& a, hipStream_t st) {
    const int M = a.M, C = a.C, F = a.F;
    if (a.dau) {
        const Plan pl = plan_gemm(M, F, C, sizeof(T), false, ACT != ND_ACT_SILU, false, 4.0 * M * F * sizeof(T));
        if (int rc = run_gemm<T, true, false>(fn, GemmSide<T>{a.dy, a.lddy, M}, GemmSide<T>{a.w_out, F, F}, C, pl, 0,
                                              EpiGateBwd<T, ACT>{a.au, a.dau, F}, st))
            return rc;
    }
    if (a.dx)
        if (int rc = run_gemm_out<T, true, false>(fn, GemmSide<T>{a.dau, 2 * F, M}, GemmSide<T>{a.w_in, C, C}, 2 * F, a.ws,
                                                  EpiOut<T>{nullptr, nullptr, a.dx, 0, C}, st))
            return rc;
    if (a.dw_in)
        if (int rc = run_gemm_out<T, false, false>(fn, GemmSide<T>{a.dau, 2 * F, 2 * F}, GemmSide<T>{a.x, a.ldx, C}, M, a.ws,
                                                   EpiOut<T>{nullptr, nullptr, a.dw_in, 0, C}, st))
            return rc;
    if (a.dw_out)
        if (int rc = run_gemm_out<T, false, false>(fn, GemmSide<T>{a.dy, a.lddy, C}, GemmSide<T>{a.h, F, F}, M, a.ws,
                                                   EpiOut<T>{nullptr, nullptr, a.dw_out, 0, F}, st))
            return rc;
    if (a.db_in || a.db_out) {
        ColSum<T> in{a.dau, 2 * F, a.db_in ? 2 * F : 0, a.db_in ? colsum_blocks(M, 2 * F) : 0, a.ws, a.db_in};
        ColSum<T> out{a.dy, a.lddy, a.db_out ? C : 0, a.db_out ? colsum_blocks(M, C) : 0, a.ws + (int64_t)in.rows * in.N, a.db_out};
        if (int rc = run_colsum<T>(fn, in, out, M, st)) return rc;
    }
    return ND_OK;
}

static int ffn_check(const char* fn, int M, int C, int F, int act, int dtype) {
    NDB_REQUIRE(M > 0 && C > 0 && F > 0, fn, "sizes must be positive");
    NDB_REQUIRE(M <= (1 << 30), fn, "more than 2^30 rows");      // a row index and the step behind it fit 32 bits
    NDB_REQUIRE(C % 8 == 0 && F % 8 == 0, fn, "channels and hidden channels must be multiples of 8");
    NDB_REQUIRE((int64_t)C * F <= (1LL << 28) && C <= (1 << 20) && F <= (1 << 20), fn, "weights of more than 2^28 elements, or more than 2^20 channels");
    NDB_REQUIRE(act >= ND_ACT_SILU && act <= ND_ACT_GELU_TANH, fn, "unknown activation");
    NDB_REQUIRE(dtype == ND_DT_F32 || dtype == ND_DT_BF16, fn, "dtype must be ND_DT_F32 or ND_DT_BF16");
    return ND_OK;
}

static bool row_ok(const void* p, int64_t ld, int cols, int es) { return !p || (aligned_to(p, 16) && ld * es % 16 == 0 && ld >= cols && ld <= (1 << 21)); }

}  // namespace ndb

using namespace ndb;

extern "C" int64_t nd_gated_ffn_workspace_floats(int M, int C, int F, int dtype) {
    if (M <= 0 || C <= 0 || F <= 0) return -1;
    return M <= FEW_ROWS ? 0 : split_floats(M, C, F, dtype == ND_DT_BF16 ? 2 : 4);
}

extern "C" int nd_gated_ffn(const void* x, int64_t ldx, const void* w_in, const void* b_in, const void* w_out, const void* b_out,
                            const void* residual, int64_t ldr, void* y, int64_t ldy, void* h, void* au, float* workspace, int M, int C,
                            int F, int act, int dtype, nd_stream_t stream) {
    const char* fn = "nd_gated_ffn";
    if (int rc = ffn_check(fn, M, C, F, act, dtype)) return rc;
    const int es = dtype == ND_DT_BF16 ? 2 : 4;
    NDB_REQUIRE(x && w_in && w_out && y && h, fn, "null pointer");
    NDB_REQUIRE(row_ok(x, ldx, C, es) && row_ok(residual, ldr, C, es) && row_ok(y, ldy, C, es), fn, "rows must be 16-byte aligned and no shorter than C");
    NDB_REQUIRE(aligned_to(w_in, 16) && aligned_to(w_out, 16) && aligned_to(b_in, 16) && aligned_to(b_out, 16) && aligned_to(h, 16) && aligned_to(au, 16), fn,
                "pointers must be 16-byte aligned");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        const Ffn<T> a{static_cast<const T*>(x), static_cast<const T*>(w_in), static_cast<const T*>(b_in), static_cast<const T*>(w_out),
                       static_cast<const T*>(b_out), static_cast<const T*>(residual), static_cast<T*>(y), static_cast<T*>(h), static_cast<T*>(au),
                       ldx, ldr, ldy, workspace, M, C, F};
        return act == ND_ACT_SILU ? ffn_forward<T, ND_ACT_SILU>(fn, a, st)
                                  : (act == ND_ACT_GELU ? ffn_forward<T, ND_ACT_GELU>(fn, a, st) : ffn_forward<T, ND_ACT_GELU_TANH>(fn, a, st));
    };
    return dtype == ND_DT_BF16 ? go(__bf16{}) : go(float{});
}

extern "C" int64_t nd_gated_ffn_bwd_workspace_floats(int M, int C, int F, int dtype) {
    if (M <= 0 || C <= 0 || F <= 0) return -1;
    const int es = dtype == ND_DT_BF16 ? 2 : 4;
    int64_t n = split_floats(M, C, 2LL * F, es);
    const int64_t more[3] = {split_floats(2LL * F, C, M, es), split_floats(C, F, M, es),
                             (int64_t)colsum_blocks(M, 2LL * F) * 2 * F + (int64_t)colsum_blocks(M, C) * C};
    for (int64_t v : more) n = v > n ? v : n;
    return n;
}

extern "C" int nd_gated_ffn_bwd(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w_in, const void* w_out,
                                const void* au, const void* h, void* dx, void* dw_in, void* db_in, void* dw_out, void* db_out, void* dau,
                                float* workspace, int M, int C, int F, int act, int dtype, nd_stream_t stream) {
    const char* fn = "nd_gated_ffn_bwd";
    if (int rc = ffn_check(fn, M, C, F, act, dtype)) return rc;
    const int es = dtype == ND_DT_BF16 ? 2 : 4;
    NDB_REQUIRE(dy && (!dw_out || h) && (!dw_in || x) && (!dx || w_in), fn, "null pointer");
    NDB_REQUIRE(!(dx || dw_in || db_in) || (dau && au && w_out), fn, "dx, dw_in and db_in need au, w_out and the dau buffer");
    NDB_REQUIRE(workspace, fn, "workspace missing");
    NDB_REQUIRE(row_ok(dy, lddy, C, es) && row_ok(x, ldx, C, es), fn, "rows must be 16-byte aligned and no shorter than C");
    for (const void* p : {w_in, w_out, au, h, (const void*)dx, (const void*)dw_in, (const void*)dw_out, (const void*)dau, (const void*)workspace})
        NDB_REQUIRE(aligned_to(p, 16), fn, "pointers must be 16-byte aligned");
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        const FfnBwd<T> a{static_cast<const T*>(dy), static_cast<const T*>(x), static_cast<const T*>(w_in), static_cast<const T*>(w_out),
                          static_cast<const T*>(au), static_cast<const T*>(h), static_cast<T*>(dx), static_cast<T*>(dw_in),
                          static_cast<T*>(db_in), static_cast<T*>(dw_out), static_cast<T*>(db_out), dx || dw_in || db_in ? static_cast<T*>(dau) : nullptr,
                          lddy, ldx, workspace, M, C, F};
        return act == ND_ACT_SILU ? ffn_backward<T, ND_ACT_SILU>(fn, a, st)
                                  : (act == ND_ACT_GELU ? ffn_backward<T, ND_ACT_GELU>(fn, a, st) : ffn_backward<T, ND_ACT_GELU_TANH>(fn, a, st));
    };
    return dtype == ND_DT_BF16 ? go(__bf16{}) : go(float{});
}
