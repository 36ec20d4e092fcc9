// The matrix product engine of the feed-forward operators: out[m][n] = sum_k X(m, k) W(n, k), bf16 or fp32, both operands in
// either order ("K-major": rows of consecutive k; otherwise rows of consecutive m / n), the epilogue a functor.
//
// A workgroup of 4 waves (2 x 2) makes a tile of 64 TI x 64 TI outputs, a wave 32 TI x 32 TI: TI = 4 (256 x 256, one
// workgroup a CU), 2 (128 x 128, two) or 1 (64 x 64, four: small products, and fp32, whose matrix rate leaves LDS time to spare).  Both operands go straight from memory to LDS (buffer loads with the LDS
// destination, 16 bytes a lane) in two stages of 128 bytes of k; a wave reads one 16-byte piece a lane and k-step for each
// of its 32-row fragments, 2 TI of them for TI^2 matrix instructions.  The weights are the first operand of the matrix
// instruction, so a lane ends with 4 consecutive n of one m.
//
//   LDS images   K-major: [row][8 pieces of 16 bytes], piece c of row r at c ^ (r >> 1 & 7): 16 rows read at one piece cover
//                all 64 banks.  Otherwise [k][row], bf16 read back transposed (ds_read_b64_tr_b16: 4 k of 16 rows), piece c
//                of k at c ^ (k & 3) << 2 (TI = 1, rows of half the banks: c ^ (k >> 1 & 1) << 2); fp32 read one float a lane, piece c at
//                c ^ (k >> 2 & 1) << 3: conflict-free too.
//   bf16 k-step  16 k: lane half lh holds k = 8 lh + 0 .. 7 of its row (v_mfma_f32_32x32x16_bf16).
//   fp32 k-step  8 k:  lane half lh holds k = 4 lh + 0 .. 3; four v_mfma_f32_32x32x2_f32, each taking one k of either half.
//   Loop         the fragments of a k-step are requested one step ahead; behind the last request of a stage one barrier
//                hands that stage over to the loads of the tile after next, which then have a whole tile's time to arrive.
//                With one wave a SIMD nothing else fills the matrix pipe, so every request sits between two matrix
//                instructions (a fence after each keeps the compiler from gathering them).
//   K tails      pieces past the end are made zero by the buffer range check (offset past the descriptor's size); rows past
//                M or N hold whatever lies there inside the tensor, and their outputs are not stored.
//   Epilogue     through LDS, 32 rows a wave at a time, so that a lane gets 8 consecutive n and a row's stores are whole lines.
//
// Measured, bf16 product alone at 16384 x 1024 x 8192 (275 GFLOP): 231 us K-major, 236 us with W [k][n] (1.19 / 1.16 PFLOP/s; the
// library's product of 8192^3 runs at 1.39); 4096 x 4096 x 8192 with both [k][.] 216 us (1.27).  What bounds it: with the loads
// taken out 189 us, the matrix instructions alone 137 us, the LDS reads alone 75 us (100 transposed), the loads alone 100 (rows of
// 512 bytes) to 190 us (rows of 128): the LDS is written and read about two thirds of the time, which is what keeps the matrix pipe
// from its rate.  Steps on the way, same product: requests in a bunch behind the barrier 282 us; 64-byte rows in a ring of 3, 4 or 5
// stages 240 us, the depth making no difference; transposed reads that the compiler cannot tell from the loads in flight
// (it then waits for them) 282 us.
#pragma once
#include <type_traits>
#include "blk_common.h"

namespace ndb {

template <typename T>
struct GemmSide {
    const T* p;
    int64_t ld;      // elements between rows (K-major: rows of m / n; otherwise rows of k)
    int n;           // rows of m / n
};

template <typename T>
struct GemmArgs {
    GemmSide<T> x, w;
    int K;           // whole contraction
    int k_tiles;     // stages of 128 bytes per split
    int tiles_m, tiles_n, splits;
    int gate_rows;   // 0, or F: the W tile is 32 TI rows of the gate half and the same 32 TI of the up half
};

constexpr int GEMM_THREADS = 256;

// block -> (tile_m, tile_n, split): consecutive workgroup ids go to the 8 XCDs in turn; each XCD gets one contiguous run of
// tiles, and a run walks groups of 8 tile rows column by column, so what its CUs hold at a time shares operand tiles in L2
__device__ __forceinline__ void gemm_tile(int lin, int total, int tiles_m, int tiles_n, int& tm, int& tn, int& sp) {
    const int q = total >> 3, r = total & 7, xcd = lin & 7;
    int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (lin >> 3);
    const int per = tiles_m * tiles_n;
    sp = id / per;
    id -= sp * per;
    const int group = 8 * tiles_n, g = id / group, first = g * 8;
    const int rows = tiles_m - first < 8 ? tiles_m - first : 8;
    id -= g * group;
    tn = id / rows;
    tm = first + id - tn * rows;
}

// one operand of a workgroup tile: its share of the loads, and its fragments
template <typename T, int TI, bool KMAJOR>
struct GemmOperand {
    static constexpr int ES = (int)sizeof(T), TILE = 64 * TI, KT = 128 / ES, PIECE = 16 / ES;
    static constexpr int NL = 2 * TI;                        // loads of 1 KiB per wave and stage
    static constexpr int STAGE = TILE * 128;                 // bytes
    static constexpr int ROWB = TILE * ES;                   // not K-major: bytes of a k row

    unsigned off[NL];
    int piece;                                               // K-major: k piece of this lane's loads
    uint64_t base;
    unsigned num;                                            // bytes that a whole stage may touch (descriptor size)
    unsigned ldb, tailw;                                     // not K-major: bytes of a k row, and from the tile's first column to its end
    unsigned soff;                                           // K-major: bytes along k
    int64_t step;
    int frag0;

    __device__ __forceinline__ void init(const GemmSide<T>& s, int K, int row0, int k0, int wave, int lane, int wbase, int gate) {
        const int64_t lb = s.ld * ES;
        soff = 0;
        ldb = (unsigned)lb;
        if constexpr (KMAJOR) {
            piece = (lane & 7) ^ (((lane >> 3) >> 1) & 7);
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int r8 = (wave * NL + i) * 8;
                int row = r8 + (lane >> 3);
                if (gate) {                                  // wave column of 32 TI rows: first half gate, second half up
                    const int wn = r8 / (32 * TI), in = r8 - wn * (32 * TI);
                    row = wn * (16 * TI) + (in & (16 * TI - 1)) + (in >= 16 * TI ? gate : 0) + (lane >> 3);
                }
                off[i] = (unsigned)(row * lb) + (unsigned)((i & 1 ? piece ^ 4 : piece) << 4);
            }
            base = reinterpret_cast<uint64_t>(s.p) + (uint64_t)(row0 * lb + (int64_t)k0 * ES);
            const uint64_t left = (uint64_t)((s.n - 1 - row0) * lb + (int64_t)(K - k0) * ES);
            num = left < 0xfffffff0ull ? (unsigned)left : 0xfffffff0u;
            const int l31 = lane & 31, lh = lane >> 5;
            frag0 = (wbase + l31) * 128 + ((lh ^ ((l31 >> 1) & 7)) << 4);
        } else {
            constexpr int CPR = ROWB / 16, RPL = 64 / CPR;   // pieces per k row, k rows per load
            static_assert(CPR <= 64, "a load covers whole k rows");
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int k = (wave * NL + i) * RPL + lane / CPR;
                const int c = (lane & (CPR - 1)) ^ swz(k);
                off[i] = (unsigned)(k * lb) + (unsigned)(c << 4);
            }
            base = reinterpret_cast<uint64_t>(s.p) + (uint64_t)((int64_t)k0 * lb + (int64_t)row0 * ES);
            tailw = (unsigned)(s.n - row0) * ES;
            num = (KT - 1) * ldb + tailw;
            step = (int64_t)KT * lb;
            frag0 = wbase;
        }
    }

    static __device__ __forceinline__ int swz(int k) { return ES == 4 ? ((k >> 2) & 1) << 3 : (TI == 1 ? ((k >> 1) & 1) << 2 : (k & 3) << 2); }

    __device__ __forceinline__ void one(char* stage, int wave, int i, unsigned n, unsigned o) const {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base), 0, (int)n, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(stage + (wave * NL + i) * 1024), 16, (int)o, (int)soff, 0, 0);
    }
    __device__ __forceinline__ void advance() {
        if constexpr (KMAJOR) soff += 128;
        else base += (uint64_t)step;
    }
    // request a stage of which krem >= 1 k are left
    __device__ __forceinline__ void load(char* stage, int wave, int krem) {
        unsigned n = num;
        if (!KMAJOR && krem < KT) n = (unsigned)(krem - 1) * ldb + tailw;
#pragma unroll
        for (int i = 0; i < NL; ++i) one(stage, wave, i, n, KMAJOR && (i & 1 ? piece ^ 4 : piece) * PIECE >= krem ? 0xfffffff0u : off[i]);
        advance();
    }

    // 16 bytes a lane: row wbase + 32 t + l31, k-step s (lane half lh)
    __device__ __forceinline__ u32x4 frag(const char* stage, int lane, int t, int s) const {
        if constexpr (KMAJOR) {
            return *reinterpret_cast<const u32x4*>(stage + ((frag0 ^ (s << 5)) + t * 4096));
        } else if constexpr (ES == 2) {
            const int lh = lane >> 5, i = lane & 15;
            const int m = frag0 + 32 * t + (lane & 16) + (i & 3) * 4;
            u32x4 v;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = 16 * s + 8 * lh + 4 * h + (i >> 2);
                const char* a = stage + k * ROWB + (((m >> 3) ^ swz(i >> 2)) << 4) + (m & 4) * 2;
                const s16x4 r = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
                union { s16x4 h4; unsigned u[2]; } c;
                c.h4 = r;
                v[2 * h] = c.u[0], v[2 * h + 1] = c.u[1];
            }
            return v;
        } else {
            const int lh = lane >> 5, m = frag0 + 32 * t + (lane & 31);
            u32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = 8 * s + 4 * lh + j;
                v[j] = *reinterpret_cast<const unsigned*>(stage + k * ROWB + (((m >> 2) ^ (lh << 3)) << 4) + (m & 3) * 4);
            }
            return v;
        }
    }
};

template <int TI>
constexpr int gemm_lds_bytes() { return 2 * 2 * 64 * TI * 128; }

#define NDB_SB __builtin_amdgcn_sched_barrier(0x6)
// one k-step of a stage: the matrix instructions of fragments c, and between them the fragments of the next step from `src` and
// (REQ) the requests of a whole stage into `dst`
template <typename T, int TI, class X, class W, int c, int s, bool REQ>
__device__ __forceinline__ void gemm_step(const char* src, char* dst, const X& x, const W& w, u32x4 (&fx)[2][TI], u32x4 (&fw)[2][TI], f32x16 (&acc)[TI][TI], int wave, int lane) {
    constexpr int SZ = X::STAGE, PER = X::NL + W::NL;
#pragma unroll
    for (int a = 0; a < TI; ++a)
#pragma unroll
        for (int b = 0; b < TI; ++b) {
            acc[a][b] = mma_step<T>(fw[c][a], fx[c][b], acc[a][b]);
            NDB_SB;
            const int i = a * TI + b;
            if (i < TI) fw[c ^ 1][i] = w.frag(src + SZ, lane, i, s);
            else if (i < 2 * TI) fx[c ^ 1][i - TI] = x.frag(src, lane, i - TI, s);
            if (TI == 1) fx[c ^ 1][0] = x.frag(src, lane, 0, s);
            if (REQ) {
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    if (j * TI * TI / PER != i) continue;              // spread over the matrix instructions
                    if (j < X::NL) x.one(dst, wave, j, x.num, x.off[j % X::NL]);
                    else w.one(dst + SZ, wave, j - X::NL, w.num, w.off[(j - X::NL) % W::NL]);
                }
            }
            NDB_SB;
        }
}
// every read of this stage has returned and the next stage has landed, in all waves
__device__ __forceinline__ void gemm_sync() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070);                       // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// Whole stages with a whole stage to request, two at a time; returns how many.  The stages are restrict pointers: the compiler
// then knows that the fragments it reads are not those that a load in flight will write, and does not wait for it.
template <typename T, int TI, class X, class W>
__device__ __forceinline__ int gemm_loop(char* __restrict__ sa, char* __restrict__ sb, X& x, W& w, u32x4 (&fx)[2][TI], u32x4 (&fw)[2][TI], f32x16 (&acc)[TI][TI], int end, int wave, int lane) {
    int kt = 0;
    for (; kt + 1 < end; kt += 2) {
        gemm_step<T, TI, X, W, 0, 1, false>(sa, sa, x, w, fx, fw, acc, wave, lane);
        gemm_step<T, TI, X, W, 1, 2, false>(sa, sa, x, w, fx, fw, acc, wave, lane);
        gemm_step<T, TI, X, W, 0, 3, false>(sa, sa, x, w, fx, fw, acc, wave, lane);
        gemm_sync();
        gemm_step<T, TI, X, W, 1, 0, true>(sb, sa, x, w, fx, fw, acc, wave, lane);
        x.advance();
        w.advance();
        gemm_step<T, TI, X, W, 0, 1, false>(sb, sb, x, w, fx, fw, acc, wave, lane);
        gemm_step<T, TI, X, W, 1, 2, false>(sb, sb, x, w, fx, fw, acc, wave, lane);
        gemm_step<T, TI, X, W, 0, 3, false>(sb, sb, x, w, fx, fw, acc, wave, lane);
        gemm_sync();
        gemm_step<T, TI, X, W, 1, 0, true>(sa, sb, x, w, fx, fw, acc, wave, lane);
        x.advance();
        w.advance();
    }
    return kt;
}
#undef NDB_SB

template <typename T, int TI, bool XK, bool WK, class Epi>
__global__ void __launch_bounds__(GEMM_THREADS, 4 / TI) gemm_kernel(const GemmArgs<T> p, const Epi epi) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    using X = GemmOperand<T, TI, XK>;
    using W = GemmOperand<T, TI, WK>;
    constexpr int KT = X::KT, SZ = X::STAGE;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave & 1, wn = wave >> 1;
    int tm, tn, sp;
    gemm_tile(blockIdx.x, gridDim.x, p.tiles_m, p.tiles_n, tm, tn, sp);
    const int kt0 = sp * p.k_tiles;
    const int all = (p.K + KT - 1) / KT;
    const int nt = all - kt0 < p.k_tiles ? all - kt0 : p.k_tiles;
    const int k0 = kt0 * KT, m0 = tm * X::TILE, n0 = tn * (p.gate_rows ? X::TILE / 2 : X::TILE);
    X x;
    W w;
    x.init(p.x, p.K, m0, k0, wave, lane, wm * 32 * TI, 0);
    w.init(p.w, p.K, n0, k0, wave, lane, wn * 32 * TI, p.gate_rows);

    f32x16 acc[TI][TI];          // [n][m]
#pragma unroll
    for (int a = 0; a < TI; ++a)
#pragma unroll
        for (int b = 0; b < TI; ++b)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[a][b][e] = 0.f;

    auto ax = [&](int st) { return smem + st * 2 * SZ; };
    constexpr int PER = X::NL + W::NL;
    x.load(ax(0), wave, p.K - k0);
    w.load(ax(0) + SZ, wave, p.K - k0);
    asm volatile("" ::: "memory");
    if (nt > 1) {
        x.load(ax(1), wave, p.K - k0 - KT);
        w.load(ax(1) + SZ, wave, p.K - k0 - KT);
    }
    u32x4 fx[2][TI], fw[2][TI];
    if (nt > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PER) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int t = 0; t < TI; ++t) {
        fx[0][t] = x.frag(ax(0), lane, t, 0);
        fw[0][t] = w.frag(ax(0) + SZ, lane, t, 0);
    }
    int kt = gemm_loop<T, TI, X, W>(ax(0), ax(1), x, w, fx, fw, acc, nt - ((p.K - k0) % KT ? 3 : 2), wave, lane);
    for (; kt < nt; ++kt) {          // the last few: nothing or a cut stage to request
        char* const cs = ax(kt & 1);
        char* const ns = ax((kt & 1) ^ 1);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int c = s & 1;
            if (s < 3) {
#pragma unroll
                for (int t = 0; t < TI; ++t) {
                    fx[c ^ 1][t] = x.frag(cs, lane, t, s + 1);
                    fw[c ^ 1][t] = w.frag(cs + SZ, lane, t, s + 1);
                }
            } else if (kt + 1 < nt) {
                gemm_sync();
                if (kt + 2 < nt) {
                    const int krem = p.K - k0 - (kt + 2) * KT;
                    x.load(cs, wave, krem);
                    w.load(cs + SZ, wave, krem);
                }
#pragma unroll
                for (int t = 0; t < TI; ++t) {
                    fx[c ^ 1][t] = x.frag(ns, lane, t, 0);
                    fw[c ^ 1][t] = w.frag(ns + SZ, lane, t, 0);
                }
            }
#pragma unroll
            for (int a = 0; a < TI; ++a)
#pragma unroll
                for (int b = 0; b < TI; ++b) acc[a][b] = mma_step<T>(fw[c][a], fx[c][b], acc[a][b]);
        }
    }
    __builtin_amdgcn_s_barrier();                             // every wave is through with the stages
    asm volatile("" ::: "memory");
    // 32 rows at a time: registers -> LDS [row][32 TI fp32, pieces of 4 at piece ^ row] -> 8 consecutive n a lane
    constexpr int PPR = 8 * TI, LPR = Epi::GATED ? 2 * TI : 4 * TI, RPI = 64 / LPR, NIT = 32 / RPI;
    const int l31 = lane & 31, lh = lane >> 5, col = lane & (LPR - 1);
    char* const mine = smem + wave * (32 * 32 * TI * 4);
    const int n = Epi::GATED ? n0 + wn * 16 * TI + col * 8 : n0 + wn * 32 * TI + col * 8;
    const bool n_in = n < (Epi::GATED ? p.gate_rows : p.w.n);
    const auto cols = epi.columns(n_in ? n : 0);
    auto piece_at = [&](int r, int c) { return reinterpret_cast<f32x4*>(mine + r * (128 * TI) + ((c ^ (r & (PPR - 1))) << 4)); };
#pragma unroll
    for (int b = 0; b < TI; ++b) {
        const int mb = m0 + wm * 32 * TI + b * 32;
        typename Epi::Row extra[NIT];
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
            const int m = mb + it * RPI + lane / LPR;
            if (n_in && m < p.x.n) extra[it] = epi.row(m, n);
        }
#pragma unroll
        for (int a = 0; a < TI; ++a)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *piece_at(l31, a * 8 + 2 * g + lh) = f32x4{acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
#pragma unroll
        for (int it = 0; it < NIT; ++it) {
            const int r = it * RPI + lane / LPR, m = mb + r;
            float v[8], u[8];
            const f32x4 v0 = *piece_at(r, 2 * col), v1 = *piece_at(r, 2 * col + 1);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = v0[e], v[4 + e] = v1[e];
            if constexpr (Epi::GATED) {
                const f32x4 u0 = *piece_at(r, PPR / 2 + 2 * col), u1 = *piece_at(r, PPR / 2 + 2 * col + 1);
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = u0[e], u[4 + e] = u1[e];
            }
            if (n_in && m < p.x.n) epi.store(m, n, sp, v, u, cols, extra[it]);
        }
    }
}

}  // namespace ndb
