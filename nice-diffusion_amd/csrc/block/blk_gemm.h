// The matrix product engine of the feed-forward operators: out[m][n] = sum_k X(m, k) W(n, k), bf16 or fp32, both operands in
// either order ("K-major": rows of consecutive k; otherwise rows of consecutive m / n), the epilogue a functor.
//
// A workgroup of 4 waves (2 x 2) makes a tile of 64 TI x 64 TI outputs, a wave 32 TI x 32 TI: TI = 4 (256 x 256, one
// workgroup a CU) or 2 (128 x 128, two).  Both operands go straight from memory to LDS (buffer loads with the LDS
// destination, 16 bytes a lane) in two stages of 128 bytes of k; a wave reads one 16-byte piece a lane and k-step for each
// of its 32-row fragments, 2 TI of them for TI^2 matrix instructions: LDS bandwidth is what a smaller wave tile would run
// out of first.  The weights are the first operand of the matrix instruction, so a lane ends with 4 consecutive n of one m.
//
//   LDS images   K-major: [row][8 pieces of 16 bytes], piece c of row r at c ^ (r >> 1 & 7): 16 rows read at one piece cover
//                all 64 banks.  Otherwise [k][row], bf16 read back transposed (ds_read_b64_tr_b16: 4 k of 16 rows), piece c
//                of k at c ^ (k & 3) << 2; fp32 read one float a lane, piece c at c ^ (k >> 2 & 1) << 3: conflict-free too.
//   bf16 k-step  16 k: lane half lh holds k = 8 lh + 0 .. 7 of its row (v_mfma_f32_32x32x16_bf16).
//   fp32 k-step  8 k:  lane half lh holds k = 4 lh + 0 .. 3; four v_mfma_f32_32x32x2_f32, each taking one k of either half.
//   Loop         the fragments of a k-step are requested one step ahead; behind the last request of a stage one barrier
//                hands that stage over to the loads of the tile after next, which then have a whole tile's time to arrive.
//   K tails      pieces past the end are made zero by the buffer range check (offset past the descriptor's size); rows past
//                M or N hold whatever lies there inside the tensor, and their outputs are not stored.
#pragma once
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
    int piece;                                               // K-major: k piece of the even loads; the odd ones have piece ^ 4
    uint64_t base;
    uint64_t left;                                           // bytes from base to the end of the tensor
    int64_t step;                                            // bytes from one stage to the next
    int frag0;

    __device__ __forceinline__ void init(const GemmSide<T>& s, int K, int row0, int k0, int wave, int lane, int wbase, int gate) {
        const int64_t ldb = s.ld * ES;
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
                off[i] = (unsigned)(row * ldb) + (unsigned)((i & 1 ? piece ^ 4 : piece) << 4);
            }
            base = reinterpret_cast<uint64_t>(s.p) + (uint64_t)(row0 * ldb + (int64_t)k0 * ES);
            left = (uint64_t)((s.n - 1 - row0) * ldb + (int64_t)(K - k0) * ES);
            step = 128;
            const int l31 = lane & 31, lh = lane >> 5;
            frag0 = wbase * 128 + l31 * 128 + ((lh ^ ((l31 >> 1) & 7)) << 4);
        } else {
            constexpr int CPR = ROWB / 16, RPL = 64 / CPR;   // pieces per k row, k rows per load
            static_assert(CPR <= 64, "a load covers whole k rows");
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int k = (wave * NL + i) * RPL + lane / CPR;
                const int c = (lane & (CPR - 1)) ^ swz(k);
                off[i] = (unsigned)(k * ldb) + (unsigned)(c << 4);
            }
            base = reinterpret_cast<uint64_t>(s.p) + (uint64_t)((int64_t)k0 * ldb + (int64_t)row0 * ES);
            left = (uint64_t)((int64_t)(K - 1 - k0) * ldb + (int64_t)(s.n - row0) * ES);
            step = (int64_t)KT * ldb;
            frag0 = wbase;
        }
    }

    static __device__ __forceinline__ int swz(int k) { return ES == 2 ? (k & 3) << 2 : ((k >> 2) & 1) << 3; }

    // request a stage; krem: k left from this stage's first (K-major tails)
    __device__ __forceinline__ void load(char* stage, int wave, int krem) {
        const uint64_t cap = left < 0xfffffff0ull ? left : 0xfffffff0ull;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base), 0, (int)(unsigned)cap, 0x00020000);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            unsigned o = off[i];
            if (KMAJOR && krem < KT) {
                const int pc = i & 1 ? piece ^ 4 : piece;
                o = pc * PIECE < krem ? o : 0xfffffff0u;
            }
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(stage + (wave * NL + i) * 1024), 16, (int)o, 0, 0, 0);
        }
        base += (uint64_t)step;
        left = left > (uint64_t)step ? left - (uint64_t)step : 0;
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
                const char* a = stage + k * ROWB + (((m >> 3) ^ ((i >> 2) << 2)) << 4) + (m & 4) * 2;
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

template <typename T, int TI, bool XK, bool WK, class Epi>
__global__ void __launch_bounds__(GEMM_THREADS, TI == 4 ? 1 : 2) gemm_kernel(const GemmArgs<T> p, const Epi epi) {
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

    char* const sx[2] = {smem, smem + SZ};
    char* const sw[2] = {smem + 2 * SZ, smem + 3 * SZ};
    x.load(sx[0], wave, p.K - k0);
    w.load(sw[0], wave, p.K - k0);
    asm volatile("" ::: "memory");          // the count below tells the two stages' loads apart by their order
    if (nt > 1) {
        x.load(sx[1], wave, p.K - k0 - KT);
        w.load(sw[1], wave, p.K - k0 - KT);
    }
    u32x4 fx[2][TI], fw[2][TI];
    if (nt > 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(X::NL + W::NL) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int t = 0; t < TI; ++t) {
        fx[0][t] = x.frag(sx[0], lane, t, 0);
        fw[0][t] = w.frag(sw[0], lane, t, 0);
    }
    for (int kt = 0; kt < nt; ++kt) {
        const int cur = kt & 1;
        char* const cx = smem + cur * SZ;
        char* const cw = smem + 2 * SZ + cur * SZ;
        char* const nx = smem + (cur ^ 1) * SZ;
        char* const nw = smem + 2 * SZ + (cur ^ 1) * SZ;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int c = s & 1, n = c ^ 1;
            if (s < 3) {
#pragma unroll
                for (int t = 0; t < TI; ++t) {
                    fx[n][t] = x.frag(cx, lane, t, s + 1);
                    fw[n][t] = w.frag(cw, lane, t, s + 1);
                }
            } else if (kt + 1 < nt) {
                // every read of this stage has returned and the next stage has landed, in all waves
                asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
                if (kt + 2 < nt) {
                    const int krem = p.K - k0 - (kt + 2) * KT;
                    x.load(cx, wave, krem);
                    w.load(cw, wave, krem);
                }
#pragma unroll
                for (int t = 0; t < TI; ++t) {
                    fx[n][t] = x.frag(nx, lane, t, 0);
                    fw[n][t] = w.frag(nw, lane, t, 0);
                }
            }
#pragma unroll
            for (int a = 0; a < TI; ++a)
#pragma unroll
                for (int b = 0; b < TI; ++b) acc[a][b] = mma_step<T>(fw[c][a], fx[c][b], acc[a][b]);
        }
    }
    // a lane's piece: row m, columns n .. n + 3
    const int l31 = lane & 31, lh = lane >> 5;
#pragma unroll
    for (int b = 0; b < TI; ++b) {
        const int m = m0 + wm * 32 * TI + b * 32 + l31;
        if (m >= p.x.n) continue;
        if constexpr (Epi::GATED) {
#pragma unroll
            for (int a = 0; a < TI / 2; ++a)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int f = n0 + wn * 16 * TI + a * 32 + 8 * g + 4 * lh;
                    const f32x4 u = {acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
                    const f32x4 v = {acc[a + TI / 2][b][4 * g], acc[a + TI / 2][b][4 * g + 1], acc[a + TI / 2][b][4 * g + 2],
                                     acc[a + TI / 2][b][4 * g + 3]};
                    if (f < p.gate_rows) epi(m, f, u, v);
                }
        } else {
#pragma unroll
            for (int a = 0; a < TI; ++a)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int n = n0 + wn * 32 * TI + a * 32 + 8 * g + 4 * lh;
                    const f32x4 u = {acc[a][b][4 * g], acc[a][b][4 * g + 1], acc[a][b][4 * g + 2], acc[a][b][4 * g + 3]};
                    if (n < p.w.n) epi(m, n, sp, u);
                }
        }
    }
}

}  // namespace ndb
