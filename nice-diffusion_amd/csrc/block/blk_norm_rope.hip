// RMS norm of every query and key head with the rotation by position in the same pass, forward and backward.
//
//   n = x r w,  r = (mean_d x^2 + eps)^-1/2          (one head of one token: D channels)
//   y = n with each pair (a, b) of the first R channels turned:  (a cos - b sin, b cos + a sin)
//   dn = dy with each pair turned back;  dw = sum over rows of dn x r;  dx = r (dn w) - x r^3 / D * sum_d(dn w x)
//
// HBM-bound: each element is read once (twice in the backward: x and dy) and written once, ~12 operations in between, all in
// fp32 and rounded once at the store.  A row is held by a group of G lanes (a power of two); a lane holds whole PAIRS (two
// chunks of VEC channels, 16 bytes each where the sizes and addresses allow it), so the rotation needs no exchange and the
// row sums are log2(G) lane swaps.  Rows are ordered (token, head): the groups of a wave mostly belong to one token and
// read the same cos / sin.  Both tensors go in one launch.  The weight gradient is summed without atomics: fixed rows per
// block, lanes -> block -> one partial row per block in the workspace, added in block order by a second launch.
//
// Measured, bf16: 64 x 1024 tokens, 6 + 6 heads of 64 out of a packed qkv row, 45 us for 201 MB (4.4 TB/s; a copy of 1 GiB runs at
// 5.15); 16 x 4096 tokens, 12 + 4 heads of 128, forward and backward 260 us for 1.34 GB (5.2 TB/s).
#include "blk_common.h"

namespace ndb {

struct NormRopeSide {
    const void* x;       // input
    const void* dy;      // backward: gradient of the output
    void* out;           // forward: y; backward: dx
    const void* w;       // [D] or null (all ones)
    int64_t xb, xt, xh;  // strides in elements: batch, token, head
    int64_t gb, gt, gh;  // strides of dy
    int64_t ob, ot, oh;  // strides of out
    int H;
};

struct NormRopeArgs {
    NormRopeSide s[2];
    const float* cos;
    const float* sin;
    int64_t cb;          // batch stride of the tables (0: shared); token stride R / 2
    float* part;         // backward: [blocks][D] partial weight gradients, those of the query blocks first
    int B, T, D, R, G;   // G: lanes per row
    int PC, RC;          // chunks of VEC pairs per row, and how many of them rotate
    float eps;
    int blocks_q;        // backward: blocks that walk the query rows
    long rows;           // forward: B * T * (Hq + Hk)
};

// the two channel offsets of chunk c
template <int VEC, bool INTER>
__device__ __forceinline__ void chunk_at(const NormRopeArgs& p, int c, int& a, int& b) {
    if constexpr (INTER) {
        a = c < p.RC ? 2 * c * VEC : p.R + 2 * (c - p.RC) * VEC;
        b = a + VEC;
    } else {
        a = c < p.RC ? c * VEC : p.R + (c - p.RC) * VEC;
        b = a + (c < p.RC ? p.R / 2 : (p.D - p.R) / 2);
    }
}

// pair i of a chunk: elements (lo, hi) of the 2 * VEC values
template <int VEC, bool INTER>
__device__ __forceinline__ constexpr int lo_of(int i) { return INTER ? 2 * i : i; }
template <int VEC, bool INTER>
__device__ __forceinline__ constexpr int hi_of(int i) { return INTER ? 2 * i + 1 : i + VEC; }

template <typename T, int VEC>
__device__ __forceinline__ void load_pair(const T* p, int a, int b, float (&v)[2 * VEC]) {
    float t[VEC];
    load_vec<T, VEC>(p + a, t);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = t[i];
    load_vec<T, VEC>(p + b, t);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[VEC + i] = t[i];
}

template <typename T, int VEC>
__device__ __forceinline__ void store_pair(T* p, int a, int b, const float (&v)[2 * VEC]) {
    float t[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = v[i];
    store_vec<T, VEC>(p + a, t);
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = v[VEC + i];
    store_vec<T, VEC>(p + b, t);
}

__device__ __forceinline__ float group_sum(float v, int G) {
    for (int o = 1; o < G; o <<= 1) v += __shfl_xor(v, o, 64);
    return v;
}

constexpr int NR_THREADS = 256;

template <typename T, int VEC, int NI, bool INTER>
__global__ void __launch_bounds__(NR_THREADS) norm_rope_kernel(const NormRopeArgs p) {
    const int j = threadIdx.x & (p.G - 1);
    const int heads = p.s[0].H + p.s[1].H, per = NR_THREADS / p.G;
    // whole groups leave the loop together: the swaps below stay inside a group
    for (long row = (long)blockIdx.x * per + threadIdx.x / p.G; row < p.rows; row += (long)gridDim.x * per) {
        const unsigned tok = p.rows <= 0x7fffffffL ? (unsigned)row / (unsigned)heads : (unsigned)(row / heads);   // B * T < 2^31
        int h = (int)(row - (long)tok * heads);
        const int b = (int)(tok / (unsigned)p.T), t = (int)(tok - (unsigned)b * (unsigned)p.T);
        const NormRopeSide& s = p.s[h >= p.s[0].H];
        if (h >= p.s[0].H) h -= p.s[0].H;
        const T* x = static_cast<const T*>(s.x) + b * s.xb + t * s.xt + h * s.xh;
        T* out = static_cast<T*>(s.out) + b * s.ob + t * s.ot + h * s.oh;
        const float* cs = p.cos + b * p.cb + (long)t * (p.R / 2);
        const float* sn = p.sin + b * p.cb + (long)t * (p.R / 2);
        const T* w = static_cast<const T*>(s.w);

        float v[NI][2 * VEC];
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = j + i * p.G;
            if (c < p.PC) {
                int a, bb;
                chunk_at<VEC, INTER>(p, c, a, bb);
                load_pair<T, VEC>(x, a, bb, v[i]);
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e) ss = fmaf(v[i][e], v[i][e], ss);
            }
        }
        const float r = rsqrtf(group_sum(ss, p.G) / (float)p.D + p.eps);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = j + i * p.G;
            if (c < p.PC) {
                int a, bb;
                chunk_at<VEC, INTER>(p, c, a, bb);
                float wv[2 * VEC];
                if (w) {
                    load_pair<T, VEC>(w, a, bb, wv);
#pragma unroll
                    for (int e = 0; e < 2 * VEC; ++e) v[i][e] = v[i][e] * r * wv[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 2 * VEC; ++e) v[i][e] *= r;
                }
                if (c < p.RC) {
                    float co[VEC], si[VEC];
                    load_vec<float, VEC>(cs + c * VEC, co);
                    load_vec<float, VEC>(sn + c * VEC, si);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float lo = v[i][lo_of<VEC, INTER>(e)], hi = v[i][hi_of<VEC, INTER>(e)];
                        v[i][lo_of<VEC, INTER>(e)] = lo * co[e] - hi * si[e];
                        v[i][hi_of<VEC, INTER>(e)] = hi * co[e] + lo * si[e];
                    }
                }
                store_pair<T, VEC>(out, a, bb, v[i]);
            }
        }
    }
}

template <typename T, int VEC, int NI, bool INTER>
__global__ void __launch_bounds__(NR_THREADS) norm_rope_bwd_kernel(const NormRopeArgs p) {
    extern __shared__ float red[];                    // [NR_THREADS / G][D]
    const int j = threadIdx.x & (p.G - 1), grp = threadIdx.x / p.G, groups = NR_THREADS / p.G;
    const int side = (int)blockIdx.x >= p.blocks_q;
    const NormRopeSide& s = p.s[side];
    const long blk = (long)blockIdx.x - (side ? p.blocks_q : 0);
    const long nblk = side ? (long)gridDim.x - p.blocks_q : p.blocks_q;
    const long rows = (long)p.B * p.T * s.H;
    const T* w = static_cast<const T*>(s.w);
    float wv[NI][2 * VEC], dw[NI][2 * VEC];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int c = j + i * p.G;
#pragma unroll
        for (int e = 0; e < 2 * VEC; ++e) {
            wv[i][e] = 1.f;
            dw[i][e] = 0.f;
        }
        if (w && c < p.PC) {
            int a, bb;
            chunk_at<VEC, INTER>(p, c, a, bb);
            load_pair<T, VEC>(w, a, bb, wv[i]);
        }
    }
    for (long row = blk * groups + grp; row < rows; row += nblk * groups) {
        const unsigned tok = rows <= 0x7fffffffL ? (unsigned)row / (unsigned)s.H : (unsigned)(row / s.H);
        const int h = (int)(row - (long)tok * s.H);
        const int b = (int)(tok / (unsigned)p.T), t = (int)(tok - (unsigned)b * (unsigned)p.T);
        const T* x = static_cast<const T*>(s.x) + b * s.xb + t * s.xt + h * s.xh;
        const T* dy = static_cast<const T*>(s.dy) + b * s.gb + t * s.gt + h * s.gh;
        T* out = static_cast<T*>(s.out) + b * s.ob + t * s.ot + h * s.oh;
        const float* cs = p.cos + b * p.cb + (long)t * (p.R / 2);
        const float* sn = p.sin + b * p.cb + (long)t * (p.R / 2);
        float v[NI][2 * VEC], g[NI][2 * VEC];
        float ss = 0.f, sg = 0.f;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = j + i * p.G;
            if (c < p.PC) {
                int a, bb;
                chunk_at<VEC, INTER>(p, c, a, bb);
                load_pair<T, VEC>(x, a, bb, v[i]);
                load_pair<T, VEC>(dy, a, bb, g[i]);
                if (c < p.RC) {
                    float co[VEC], si[VEC];
                    load_vec<float, VEC>(cs + c * VEC, co);
                    load_vec<float, VEC>(sn + c * VEC, si);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const float lo = g[i][lo_of<VEC, INTER>(e)], hi = g[i][hi_of<VEC, INTER>(e)];
                        g[i][lo_of<VEC, INTER>(e)] = lo * co[e] + hi * si[e];
                        g[i][hi_of<VEC, INTER>(e)] = hi * co[e] - lo * si[e];
                    }
                }
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e) {
                    ss = fmaf(v[i][e], v[i][e], ss);
                    sg = fmaf(g[i][e] * wv[i][e], v[i][e], sg);
                }
            }
        }
        for (int o = 1; o < p.G; o <<= 1) {
            ss += __shfl_xor(ss, o, 64);
            sg += __shfl_xor(sg, o, 64);
        }
        const float r = rsqrtf(ss / (float)p.D + p.eps);
        const float k = r * r * (sg / (float)p.D);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int c = j + i * p.G;
            if (c < p.PC) {
                int a, bb;
                chunk_at<VEC, INTER>(p, c, a, bb);
#pragma unroll
                for (int e = 0; e < 2 * VEC; ++e) {
                    dw[i][e] = fmaf(g[i][e], v[i][e] * r, dw[i][e]);
                    v[i][e] = r * (g[i][e] * wv[i][e] - v[i][e] * k);
                }
                store_pair<T, VEC>(out, a, bb, v[i]);
            }
        }
    }
    if (p.part == nullptr) return;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const int c = j + i * p.G;
        if (c < p.PC) {
            int a, bb;
            chunk_at<VEC, INTER>(p, c, a, bb);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                red[grp * p.D + a + e] = dw[i][e];
                red[grp * p.D + bb + e] = dw[i][VEC + e];
            }
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += NR_THREADS) {
        float t = 0.f;
        for (int gi = 0; gi < groups; ++gi) t += red[gi * p.D + d];
        p.part[(long)blockIdx.x * p.D + d] = t;
    }
}

// dw[d] = sum of the partial rows of one side, in a fixed order: 32 channels x 32 row lanes a block
template <typename T>
__global__ void __launch_bounds__(1024) norm_rope_dw_kernel(const float* part, int rows_q, int rows_k, int D, T* dwq, T* dwk) {
    __shared__ float red[32][33];
    const int side = blockIdx.y, d = blockIdx.x * 32 + (threadIdx.x & 31), lane = threadIdx.x >> 5;
    const float* src = part + (side ? (long)rows_q * D : 0);
    const int rows = side ? rows_k : rows_q;
    T* dst = side ? dwk : dwq;
    float t = 0.f;
    if (d < D && dst) {
#pragma unroll 8
        for (int r = lane; r < rows; r += 32) t += src[(long)r * D + d];
    }
    red[lane][threadIdx.x & 31] = t;
    __syncthreads();
    if (lane == 0 && d < D && dst) {
        float u = 0.f;
        for (int l = 0; l < 32; ++l) u += red[l][threadIdx.x & 31];
        dst[d] = (T)u;
    }
}

// widest access that the channel counts and every address allow
template <typename T>
static int norm_rope_vec(const NormRopeArgs& a, bool inter, bool bwd) {
    for (int v = 16 / (int)sizeof(T); v > 1; v >>= 1) {
        const int bytes = v * (int)sizeof(T);
        const int unit = inter ? 2 * v : v;
        const int rot = inter ? a.R : a.R / 2, rest = inter ? a.D - a.R : (a.D - a.R) / 2;
        bool ok = rot % unit == 0 && rest % unit == 0;
        if (a.R) ok = ok && aligned_to(a.cos, v >= 4 ? 16 : 4 * v) && aligned_to(a.sin, v >= 4 ? 16 : 4 * v) && a.cb % (v >= 4 ? 4 : v) == 0;
        for (int i = 0; i < 2; ++i) {
            const NormRopeSide& s = a.s[i];
            if (!s.H) continue;
            ok = ok && aligned_to(s.x, bytes) && aligned_to(s.out, bytes) && aligned_to(s.w, bytes);
            ok = ok && s.xb % v == 0 && s.xt % v == 0 && s.xh % v == 0 && s.ob % v == 0 && s.ot % v == 0 && s.oh % v == 0;
            if (bwd) ok = ok && aligned_to(s.dy, bytes) && s.gb % v == 0 && s.gt % v == 0 && s.gh % v == 0;
        }
        if (ok) return v;
    }
    return 1;
}

constexpr int NR_MAX_D = 512;

// D <= 512: one chunk a lane covers a row of <= 64 chunks at VEC >= 4, two at VEC 2, four at VEC 1
template <typename T, int VEC, bool INTER>
static void launch_norm_rope(NormRopeArgs& a, bool bwd, int blocks, hipStream_t st) {
    constexpr int NI = VEC >= 4 ? 1 : (VEC == 2 ? 2 : 4);
    a.PC = a.D / 2 / VEC;
    a.RC = a.R / 2 / VEC;
    a.G = 1;
    while (a.G * NI < a.PC) a.G <<= 1;
    if (bwd) {
        const size_t lds = a.part ? (size_t)(NR_THREADS / a.G) * a.D * sizeof(float) : 0;
        hipLaunchKernelGGL((norm_rope_bwd_kernel<T, VEC, NI, INTER>), dim3(blocks), dim3(NR_THREADS), lds, st, a);
    } else {
        const long per = NR_THREADS / a.G;
        const long n = (a.rows + per - 1) / per;      // beyond 2^20 blocks each takes several rows a group
        hipLaunchKernelGGL((norm_rope_kernel<T, VEC, NI, INTER>), dim3((unsigned)(n < (1L << 20) ? n : (1L << 20))), dim3(NR_THREADS), 0, st, a);
    }
}

template <typename T>
static void dispatch_norm_rope(NormRopeArgs& a, bool inter, bool bwd, int blocks, hipStream_t st) {
    const int v = norm_rope_vec<T>(a, inter, bwd);
#define NDB_CASE(V)                                                        \
    if (v == V) {                                                          \
        if (inter)                                                         \
            launch_norm_rope<T, V, true>(a, bwd, blocks, st);              \
        else                                                               \
            launch_norm_rope<T, V, false>(a, bwd, blocks, st);             \
        return;                                                            \
    }
    if constexpr (sizeof(T) == 2) {
        NDB_CASE(8)
    }
    NDB_CASE(4)
    NDB_CASE(2)
    NDB_CASE(1)
#undef NDB_CASE
}

// backward blocks of one side: enough rows a block (>= 32) that the partial rows stay a small part of what is moved, and at
// most 2048 of them
static int norm_rope_bwd_blocks(long rows) {
    const long n = (rows + 31) / 32;
    return (int)(n < 1 ? 1 : (n > 2048 ? 2048 : n));
}

static int norm_rope_check(const char* fn, int B, int T, int Hq, int Hk, int D, int R, const void* cos, const void* sin, int dtype) {
    NDB_REQUIRE(B > 0 && T > 0 && Hq > 0 && Hk >= 0, fn, "sizes must be positive");
    NDB_REQUIRE(D > 0 && D % 2 == 0 && D <= NR_MAX_D, fn, "head dim must be even and at most 512");
    NDB_REQUIRE(R >= 0 && R % 2 == 0 && R <= D, fn, "rotated channels must be even and at most the head dim");
    NDB_REQUIRE(R == 0 || (cos && sin), fn, "cos / sin tables missing");
    NDB_REQUIRE(dtype == ND_DT_F32 || dtype == ND_DT_BF16, fn, "dtype must be ND_DT_F32 or ND_DT_BF16");
    NDB_REQUIRE((long)B * T <= 0x7fffffffL && (long)B * T * (Hq + Hk) <= (1L << 34), fn, "too many rows for one launch");
    return ND_OK;
}

// Rows of `bytes` bytes at p + sum_i x_i s[i], 0 <= x_i < n[i]
struct RowBox {
    uint64_t p;
    int64_t n[3], s[3], bytes;
};

static RowBox row_box(const void* p, int64_t sb, int64_t st, int64_t sh, int64_t B, int64_t T, int64_t H, int64_t D, int64_t es) {
    RowBox r{reinterpret_cast<uintptr_t>(p), {B, T, H}, {sb * es, st * es, sh * es}, D * es};
    for (int i = 0; i < 3; ++i) {
        if (r.n[i] == 1) r.s[i] = 0;
        if (r.s[i] < 0) r.p += (uint64_t)(r.s[i] * (r.n[i] - 1)), r.s[i] = -r.s[i];
    }
    return r;
}

// Is there sum_i x_i s[i] + c = delta with lo[i] <= x_i <= hi[i] and c_lo <= c <= c_hi (and some x_i not 0)?  s descending and
// positive, so that few x_i are left to try at each level; after `visits` of them the answer is yes.
static bool row_meet(const int64_t* s, const int64_t* lo, const int64_t* hi, int dims, int64_t delta, int64_t c_lo, int64_t c_hi, bool moved, int& visits) {
    if (dims == 0) return moved && delta >= c_lo && delta <= c_hi;
    int64_t r_lo = c_lo, r_hi = c_hi;                          // what the dimensions behind this one reach
    for (int i = 1; i < dims; ++i) r_lo += lo[i] * s[i], r_hi += hi[i] * s[i];
    auto div_down = [](int64_t a, int64_t b) { return a / b - (a % b < 0); };
    int64_t from = -div_down(r_hi - delta, s[0]), to = div_down(delta - r_lo, s[0]);
    from = from > lo[0] ? from : lo[0];
    to = to < hi[0] ? to : hi[0];
    for (int64_t x = from; x <= to; ++x) {
        if (--visits < 0) return true;
        if (row_meet(s + 1, lo + 1, hi + 1, dims - 1, delta - x * s[0], c_lo, c_hi, moved || x != 0, visits)) return true;
    }
    return false;
}

// Do the rows of a and b (b null: two rows of a) have a byte in common?  Exact for equal strides; otherwise yes if their ranges meet.
static bool rows_overlap(const RowBox& a, const RowBox* b) {
    int64_t s[3], lo[3], hi[3];
    int dims = 0;
    if (b) {
        uint64_t ea = a.p + (uint64_t)a.bytes, eb = b->p + (uint64_t)b->bytes;
        for (int i = 0; i < 3; ++i) ea += (uint64_t)((a.n[i] - 1) * a.s[i]), eb += (uint64_t)((b->n[i] - 1) * b->s[i]);
        if (ea <= b->p || eb <= a.p) return false;
    }
    for (int i = 0; i < 3; ++i) {
        const int64_t na = a.n[i], nb = b ? b->n[i] : na, sa = a.s[i], sb = b ? b->s[i] : sa, st = na > 1 ? sa : sb;
        if (na > 1 && nb > 1 && sa != sb) return true;
        if (st == 0) {
            if (!b && na > 1) return true;
            continue;
        }
        int j = dims++;
        for (; j > 0 && s[j - 1] < st; --j) s[j] = s[j - 1], lo[j] = lo[j - 1], hi[j] = hi[j - 1];
        s[j] = st, lo[j] = -(nb - 1), hi[j] = na - 1;
    }
    int visits = 4096;
    const int64_t delta = b ? (int64_t)(b->p - a.p) : 0, rb = b ? b->bytes : a.bytes;
    return row_meet(s, lo, hi, dims, delta, -(rb - 1), a.bytes - 1, b != nullptr, visits);
}

static bool rows_same(const RowBox& a, const RowBox& b) {
    for (int i = 0; i < 3; ++i)
        if (a.n[i] != b.n[i] || a.s[i] != b.s[i]) return false;
    return a.p == b.p && a.bytes == b.bytes;
}

// An output may be its own input; any other common address is a race between the workgroups.
static bool norm_rope_outputs_apart(const NormRopeArgs& a, int es) {
    RowBox in[2], out[2];
    const int sides = a.s[1].H ? 2 : 1;
    for (int i = 0; i < sides; ++i) {
        const NormRopeSide& s = a.s[i];
        in[i] = row_box(s.x, s.xb, s.xt, s.xh, a.B, a.T, s.H, a.D, es);
        out[i] = row_box(s.out, s.ob, s.ot, s.oh, a.B, a.T, s.H, a.D, es);
    }
    if (sides == 2 && rows_overlap(out[0], &out[1])) return false;
    for (int i = 0; i < sides; ++i) {
        if (rows_overlap(out[i], nullptr)) return false;
        for (int j = 0; j < sides; ++j) {
            if (!(i == j && rows_same(out[i], in[j])) && !(i != j && rows_same(out[j], in[j])) && rows_overlap(out[i], &in[j])) return false;
            const RowBox w = row_box(a.s[j].w, 0, 0, 0, 1, 1, 1, a.D, es);
            if (a.s[j].w && rows_overlap(out[i], &w)) return false;
        }
        for (const float* t : {a.cos, a.sin}) {
            const RowBox c = row_box(t, a.cb, a.R / 2, 0, a.B, a.T, 1, a.R / 2, 4);
            if (a.R && rows_overlap(out[i], &c)) return false;
        }
    }
    return true;
}

}  // namespace ndb

using namespace ndb;

extern "C" int nd_rows_overlap(const void* a, int64_t a_sb, int64_t a_st, int64_t a_sh, int Ha, const void* b, int64_t b_sb, int64_t b_st,
                               int64_t b_sh, int Hb, int B, int T, int D, int es) {
    if (B <= 0 || T <= 0 || D <= 0 || es <= 0 || Ha <= 0 || (b && Hb <= 0)) return 0;
    const RowBox x = row_box(a, a_sb, a_st, a_sh, B, T, Ha, D, es);
    if (!b) return rows_overlap(x, nullptr);
    const RowBox y = row_box(b, b_sb, b_st, b_sh, B, T, Hb, D, es);
    return rows_overlap(x, &y);
}

extern "C" int nd_qk_norm_rope(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                               int64_t k_sh, const void* q_weight, const void* k_weight, const float* cos, const float* sin,
                               int64_t table_sb, void* q_out, int64_t qo_sb, int64_t qo_st, int64_t qo_sh, void* k_out, int64_t ko_sb,
                               int64_t ko_st, int64_t ko_sh, int B, int T, int Hq, int Hk, int D, int R, float eps, int flags,
                               int dtype, nd_stream_t stream) {
    const char* fn = "nd_qk_norm_rope";
    if (int rc = norm_rope_check(fn, B, T, Hq, Hk, D, R, cos, sin, dtype)) return rc;
    NDB_REQUIRE(q && q_out && (Hk == 0 || (k && k_out)), fn, "null pointer");
    NormRopeArgs a{};
    a.s[0] = {q, nullptr, q_out, q_weight, q_sb, q_st, q_sh, 0, 0, 0, qo_sb, qo_st, qo_sh, Hq};
    a.s[1] = {k, nullptr, k_out, k_weight, k_sb, k_st, k_sh, 0, 0, 0, ko_sb, ko_st, ko_sh, Hk};
    a.cos = cos, a.sin = sin, a.cb = table_sb;
    a.B = B, a.T = T, a.D = D, a.R = R, a.eps = eps;
    a.rows = (long)B * T * (Hq + Hk);
    NDB_REQUIRE(norm_rope_outputs_apart(a, dtype == ND_DT_BF16 ? 2 : 4), fn, "outputs overlap each other, themselves or what is read (other than their own input)");
    const bool inter = flags & ND_ROPE_INTERLEAVED;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    if (dtype == ND_DT_BF16)
        dispatch_norm_rope<__bf16>(a, inter, false, 0, st);
    else
        dispatch_norm_rope<float>(a, inter, false, 0, st);
    return check_launch(fn);
}

extern "C" int64_t nd_qk_norm_rope_bwd_workspace_floats(int B, int T, int Hq, int Hk, int D) {
    if (B <= 0 || T <= 0 || Hq <= 0 || Hk < 0 || D <= 0) return -1;
    return (int64_t)(norm_rope_bwd_blocks((long)B * T * Hq) + (Hk ? norm_rope_bwd_blocks((long)B * T * Hk) : 0)) * D;
}

extern "C" int nd_qk_norm_rope_bwd(const void* q, int64_t q_sb, int64_t q_st, int64_t q_sh, const void* k, int64_t k_sb, int64_t k_st,
                                   int64_t k_sh, const void* q_weight, const void* k_weight, const float* cos, const float* sin,
                                   int64_t table_sb, const void* dq_out, int64_t dqo_sb, int64_t dqo_st, int64_t dqo_sh,
                                   const void* dk_out, int64_t dko_sb, int64_t dko_st, int64_t dko_sh, void* dq, int64_t dq_sb,
                                   int64_t dq_st, int64_t dq_sh, void* dk, int64_t dk_sb, int64_t dk_st, int64_t dk_sh, void* dq_weight,
                                   void* dk_weight, float* workspace, int B, int T, int Hq, int Hk, int D, int R, float eps,
                                   int flags, int dtype, nd_stream_t stream) {
    const char* fn = "nd_qk_norm_rope_bwd";
    if (int rc = norm_rope_check(fn, B, T, Hq, Hk, D, R, cos, sin, dtype)) return rc;
    NDB_REQUIRE(q && dq_out && dq && (Hk == 0 || (k && dk_out && dk)), fn, "null pointer");
    const bool weights = dq_weight || dk_weight;
    NDB_REQUIRE(!weights || workspace, fn, "the weight gradients need a workspace");
    NormRopeArgs a{};
    a.s[0] = {q, dq_out, dq, q_weight, q_sb, q_st, q_sh, dqo_sb, dqo_st, dqo_sh, dq_sb, dq_st, dq_sh, Hq};
    a.s[1] = {k, dk_out, dk, k_weight, k_sb, k_st, k_sh, dko_sb, dko_st, dko_sh, dk_sb, dk_st, dk_sh, Hk};
    a.cos = cos, a.sin = sin, a.cb = table_sb;
    a.B = B, a.T = T, a.D = D, a.R = R, a.eps = eps;
    a.part = weights ? workspace : nullptr;
    a.blocks_q = norm_rope_bwd_blocks((long)B * T * Hq);
    const int blocks_k = Hk ? norm_rope_bwd_blocks((long)B * T * Hk) : 0;
    const bool inter = flags & ND_ROPE_INTERLEAVED;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const dim3 gdw((D + 31) / 32, Hk ? 2 : 1);
    if (dtype == ND_DT_BF16) {
        dispatch_norm_rope<__bf16>(a, inter, true, a.blocks_q + blocks_k, st);
        if (weights)
            hipLaunchKernelGGL((norm_rope_dw_kernel<__bf16>), gdw, dim3(1024), 0, st, workspace, a.blocks_q, blocks_k, D,
                               static_cast<__bf16*>(dq_weight), static_cast<__bf16*>(dk_weight));
    } else {
        dispatch_norm_rope<float>(a, inter, true, a.blocks_q + blocks_k, st);
        if (weights)
            hipLaunchKernelGGL((norm_rope_dw_kernel<float>), gdw, dim3(1024), 0, st, workspace, a.blocks_q, blocks_k, D,
                               static_cast<float*>(dq_weight), static_cast<float*>(dk_weight));
    }
    return check_launch(fn);
}
