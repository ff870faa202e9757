// Orthogonalised updates (Newton-Schulz products, as the Muon optimiser takes them) for many matrices at once.
//
// X0 = U / (|U|_F + eps);  per step  A = X X^T,  B = b A + c A A,  X <- a X + B X   (X [m, n], m <= n: the shorter side of
// U in front);  the result is X in U's orientation, in bf16.  With the usual (a, b, c) every singular value of U ends
// near 1.
//
// Number formats.  The operands of the matrix instructions are fp16: every |x| is at most the largest singular value
// (about 1.2), so the range that bf16 pays three bits for is not needed; X, A, B are kept times powers of two that put
// them in the middle of fp16's range (X's by the matrix: an update that is small against eps starts at |U| / eps and
// ends at most `gain` = prod max(1, a) times that, so it is held 2^e times larger).  All sums are fp32 (the norm's fp64).
// A rounding of X in step i is noise in every direction, and grows by a^(steps - 1 - i) in those of small singular
// values (3.44^4 = 140 from the first of five steps), against an answer that is O(1) there.  While that factor is above
// SPLIT_ABOVE, X is a hi + lo pair of fp16 (22 bits) in X <- B X: two products.  A and B need no more than fp16: their
// roundings, multiplied by X, stay in the directions that X has.  On an update of four strong directions over 0.01 of
// noise the result is 0.0018 off 64 bits with pairs in three of five steps (0.0053 in two, 0.0010 in four), 0.042
// without, 0.33 with bf16 throughout; its own rounding to bf16 is 0.0017.
#include <math.h>
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "common.h"

namespace {

typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void* lptr_t;

constexpr int BK = 32, NTHR = 256;
constexpr int ITEMS = 16;                       // items described by one launch of the norm kernel
constexpr int BLK = 6;                          // tiles' order: by blocks of 6 x 6
constexpr float SX = 4096.f;                    // X is stored times this
constexpr double SPLIT_ABOVE = 8.0;

// One item: `batch` matrices of one shape.  Offsets in elements of the region of their kind.
struct Mat {
    const void* in;
    void* out;
    int64_t in_batch, in_ld, out_batch, out_ld, xoff, aoff;
    int rows, cols, batch, dtype;
    int tall, m, n, mp, np;                     // m <= n; mp, np: padded to 64 (zeros)
    int parts, part0, mat0;                     // partial sums of the norm: per matrix, first index; first matrix
    int preps;                                  // 64 x 64 tiles that a workgroup of the preparing kernel takes
    int sym0, rect0, prep0;                     // first tile of each kind
};
// One tile of a product: everything a workgroup needs to start on it, in one load.
struct Tile {
    int64_t xo, ao;                             // the matrix in the X and A / B regions (elements)
    int mp, np, m0, n0, item, mat;              // mat: index within the item
    int all, pad;                               // index of the matrix over all items
};
// (read as constant memory, that is through scalar loads: it was written by an earlier launch)
DEVI Tile load_tile(const Tile* p) {
    typedef const __attribute__((address_space(4))) u32x4* cptr_t;
    struct { u32x4 w[3]; } t;
#pragma unroll
    for (int i = 0; i < 3; ++i) t.w[i] = ((cptr_t)(uintptr_t)p)[i];
    return __builtin_bit_cast(Tile, t);
}
DEVI float load_const(const float* p) { return *(const __attribute__((address_space(4))) float*)(uintptr_t)p; }
struct Setup {
    Mat it[ITEMS];
    int wg0[ITEMS + 1];                         // first workgroup of each item
    int count, first;                           // items here, index of the first
};
// X, A, B lie as panels of 32 columns: element (r, c) of a matrix of mp rows at ((c / 32) mp + r) 32 + c % 32.
struct Ws {                                     // regions of the workspace
    Mat* mats;
    Tile *sym, *rect;                           // tiles of the symmetric products / of the update
    int* map_prep;                              // workgroup of the preparing kernel -> item
    double* parts;
    float* exps;                                // 2^-e of each matrix
    int tsym, trect;                            // tile sizes
    f16 *x[2][2], *a, *b;                       // X: [buffer][hi / lo]
};

DEVI double block_sum_f64(double v, double* red) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    double r = 0;
    for (int i = 0; i < (int)(blockDim.x >> 6); ++i) r += red[i];
    return r;
}

// squares of rows [r0, r1): V elements a thread and load, four loads in flight, rows one behind the other
template <typename T, int V> DEVI double rows_sq(const T* p, int64_t ld, int cols, int r0, int r1) {
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T) * V)));
    const int g = (cols + V - 1) / V, dr = NTHR / g, dc = NTHR % g;         // vectors a row; a step of NTHR of them
    int r = r0 + (int)threadIdx.x / g, c = (int)threadIdx.x % g;
    double s = 0;
    while (r < r1) {
        float v[4][V];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const T* x = p + r * ld + c * V;
#pragma unroll
            for (int i = 0; i < V; ++i) v[u][i] = 0.f;
            if (r < r1) {
                if (V == 1 || c * V + V <= cols) {
                    const vec w = *(const vec*)x;
#pragma unroll
                    for (int i = 0; i < V; ++i) v[u][i] = (float)w[i];
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (c * V + i < cols) v[u][i] = (float)x[i];
                }
            }
            r += dr;
            c += dc;
            if (c >= g) { c -= g; ++r; }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) s = fma((double)v[u][i], (double)v[u][i], s);
    }
    return s;
}
template <typename T> DEVI double rows_sq(const void* in, int64_t at, int64_t ld, int cols, int r0, int r1) {
    const T* p = (const T*)in + at;
    if (((uintptr_t)p | (uint64_t)(ld * sizeof(T))) % (4 * sizeof(T)) == 0) return rows_sq<T, 4>(p, ld, cols, r0, r1);
    return rows_sq<T, 1>(p, ld, cols, r0, r1);
}

DEVI int prep_groups(const Mat& q) { return (((q.mp + 63) / 64) * ((q.np + 63) / 64) + q.preps - 1) / q.preps; }

// Partial sums of squares (fp64: neither 1e-30 nor 1e30 leaves the range), and the tables that the
// following launches read: items, the map of the preparing kernel, the products' tiles.
__global__ __launch_bounds__(NTHR) void ortho_norm_kernel(const Setup su, const Ws ws) {
    __shared__ double red[4];
    int i = 0;
    while (i + 1 < su.count && (int)blockIdx.x >= su.wg0[i + 1]) ++i;
    const Mat& q = su.it[i];
    const int w = blockIdx.x - su.wg0[i], nw = su.wg0[i + 1] - su.wg0[i], id = su.first + i;
    if (w == 0 && threadIdx.x == 0) ws.mats[id] = q;
    const int t0 = w * NTHR + threadIdx.x, ts = nw * NTHR;
    const int np_ = q.batch * prep_groups(q);
    for (int t = t0; t < np_; t += ts) ws.map_prep[q.prep0 + t] = id;
    // the tiles of the products
    const int sm = (q.mp + ws.tsym - 1) / ws.tsym, ns = sm * (sm + 1) / 2;
    const int rm = (q.mp + ws.trect - 1) / ws.trect, nr = rm * ((q.np + ws.trect - 1) / ws.trect);
    for (int t = t0; t < q.batch * (ns + nr); t += ts) {
        const bool sym = t < q.batch * ns;
        const int u = sym ? t : t - q.batch * ns, mat = u / (sym ? ns : nr);
        int k = u - mat * (sym ? ns : nr);
        Tile d{q.xoff + (int64_t)mat * q.mp * q.np, q.aoff + (int64_t)mat * q.mp * q.mp, q.mp, q.np, 0, 0, id, mat, q.mat0 + mat, 0};
        // Tiles that follow each other, which the 32 CUs of one XCD take, share rows and columns in its L2 (the head MLP's 2048 x
        // 2048: 455 us in all by whole rows, 446 by blocks; matrices of up to 6 tiles a side have the same order either way).
        if (sym) {                           // BLK x BLK at a time
            int r = 0, c = 0;
            for (;;) {
                const int h = min(BLK, sm - r), n = r == c ? h * (h + 1) / 2 : h * min(BLK, sm - c);
                if (k < n) break;
                k -= n;
                c += BLK;
                if (c >= sm) { r += BLK; c = r; }
            }
            if (r == c) {
                const int h = min(BLK, sm - r);
                int i = 0;
                while (k >= h - i) { k -= h - i; ++i; }
                r += i;
                c += i + k;
            } else {
                const int w = min(BLK, sm - c);
                r += k / w;
                c += k % w;
            }
            d.m0 = r * ws.tsym;
            d.n0 = c * ws.tsym;
            ws.sym[q.sym0 + u] = d;
        } else {                             // BLK rows of tiles at a time, column by column
            const int rn = nr / rm, r = k / (BLK * rn) * BLK, h = min(BLK, rm - r), e = k - r * rn;
            d.m0 = (r + e % h) * ws.trect;
            d.n0 = (e / h) * ws.trect;
            ws.rect[q.rect0 + u] = d;
        }
    }
    const int b = w / q.parts, part = w - b * q.parts, per = (q.rows + q.parts - 1) / q.parts;
    const int r0 = part * per, r1 = min(q.rows, r0 + per);
    const double s = q.dtype == DINO_F32 ? rows_sq<float>(q.in, b * q.in_batch, q.in_ld, q.cols, r0, r1)
                                         : rows_sq<bf16>(q.in, b * q.in_batch, q.in_ld, q.cols, r0, r1);
    const double tot = block_sum_f64(s, red);
    if (threadIdx.x == 0) ws.parts[q.part0 + w] = tot;
}

// X0 = U * SX 2^e / (|U| + eps) as hi + lo in panels, shorter side in front, padding cleared; 64 x 64 elements at a time,
// through LDS where U is tall.  VEC: U's rows start at multiples of four elements.
template <typename T, bool VEC> DEVI void prep_tiles(const Mat& q, const T* u, f16* xh, f16* xl, int t0, int t1, float pre, float scale, float (&tile)[64][66]) {
    const int tn = (q.np + 63) / 64, c4 = (threadIdx.x & 15) * 4, r0 = threadIdx.x >> 4;
    for (int t = t0; t < t1; ++t) {
        const int m0 = (t / tn) * 64, n0 = (t % tn) * 64;
        float v[4][4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {            // row ur, columns uc .. uc + 3 of U
            const int ur = (q.tall ? n0 : m0) + r0 + 16 * p, uc = (q.tall ? m0 : n0) + c4;
            const T* x = u + ur * q.in_ld + uc;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[p][k] = 0.f;
            if (ur < q.rows) {
                if (VEC && uc + 4 <= q.cols) load4<T>(x, v[p]);
                else {
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (uc + k < q.cols) v[p][k] = to_f32<T>(x[k]);
                }
            }
        }
        if (q.tall) {
            __syncthreads();
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k) tile[r0 + 16 * p][c4 + k] = v[p][k];
            __syncthreads();
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[p][k] = tile[c4 + k][r0 + 16 * p];
        }
        const int n = n0 + c4;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int m = m0 + r0 + 16 * p;
            if (m >= q.mp || n >= q.np) continue;
            const int64_t at = ((int64_t)(n >> 5) * q.mp + m) * 32 + (n & 31);
            f16x4 h, l;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float x = v[p][k] * pre * scale;
                h[k] = (f16)x;
                l[k] = (f16)(x - (float)h[k]);
            }
            *(f16x4*)(xh + at) = h;
            if (xl) *(f16x4*)(xl + at) = l;
        }
    }
}
__global__ __launch_bounds__(NTHR) void ortho_prep_kernel(const Ws ws, double eps, double gain, int lo) {
    __shared__ double red[4];
    __shared__ float tile[64][66];
    const int id = ws.map_prep[blockIdx.x];
    const Mat& q = ws.mats[id];
    const int per = prep_groups(q), w = blockIdx.x - q.prep0, b = w / per, part = w - b * per;
    double s = 0;
    for (int p = threadIdx.x; p < q.parts; p += NTHR) s += ws.parts[q.part0 + b * q.parts + p];
    const double norm = sqrt(block_sum_f64(s, red)), end = gain * (norm / (norm + eps));
    const int e = end > 0.0 && end < 1.0 ? min(120, ilogb(1.0 / end)) : 0;
    // in two factors where one would leave fp32: a norm below 1e-35 with an eps as small
    const double whole = ldexp((double)SX, e) / (norm + eps);
    const float pre = whole > 0x1p100 ? 0x1p64f : 1.f, scale = (float)(whole / pre);
    if (part == 0 && threadIdx.x == 0) ws.exps[q.mat0 + b] = ldexpf(1.f, -e);
    const int nt = ((q.mp + 63) / 64) * ((q.np + 63) / 64), t0 = part * q.preps, t1 = min(nt, t0 + q.preps);
    const int64_t xo = q.xoff + (int64_t)b * q.mp * q.np;
    f16 *xh = ws.x[0][0] + xo, *xl = lo ? ws.x[0][1] + xo : nullptr;
    if (q.dtype == DINO_F32) {
        const float* u = (const float*)q.in + b * q.in_batch;
        if ((((uintptr_t)u | (uint64_t)(q.in_ld * 4)) & 15) == 0) prep_tiles<float, true>(q, u, xh, xl, t0, t1, pre, scale, tile);
        else prep_tiles<float, false>(q, u, xh, xl, t0, t1, pre, scale, tile);
    } else {
        const bf16* u = (const bf16*)q.in + b * q.in_batch;
        if ((((uintptr_t)u | (uint64_t)(q.in_ld * 2)) & 7) == 0) prep_tiles<bf16, true>(q, u, xh, xl, t0, t1, pre, scale, tile);
        else prep_tiles<bf16, false>(q, u, xh, xl, t0, t1, pre, scale, tile);
    }
}

struct GemmArgs {
    Ws ws;
    int src, split_next, ntiles;     // X buffer read; the next step's operands are pairs; tiles of this launch
    float c0, c1, ca;                // epilogue: c0 * (elementwise operand) + c1 * product, + ca on the diagonal
};

DEVI int fsw(int x) { return (4 - (x & 3)) & 3; }
template <int N> DEVI void wait_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// T x T tiles of a product, a workgroup of eight waves (2 x 4, each T/2 x T/4; T = 64: 4 x 2) walking its share of them.
//   GRAM    A = X X^T               rows of X against rows of X; tiles on and above the diagonal, written twice
//   POLY    B = a I + b A + c A A   A symmetric: rows against rows again
//   UPDATE  X' = B X                rows of B against COLUMNS of X (transposing LDS reads)
//   FINAL   the last UPDATE: into the caller's matrix as bf16
// (a on B's diagonal instead of a X in the update: no second read of X.)
// Operands go global -> LDS by DMA in a ring of S stages of 32 along the contraction, one stream of stages over all tiles of
// the workgroup: the next tile's first stages are on their way while this one's results leave.  With SPLIT (an UPDATE) a
// stage holds the hi and the lo part of X and feeds two products.
// What bounds it, for X' of ViT-L's 144 matrices (0.62 TFLOP; 0.9 GB to read, 0.6 GB to write): 590 us = 1050 TFLOP/s (a large
// library product reaches 1306 here); of pairs (1.24 TFLOP) 1030 us = 1200.  The matrix pipes are busy in 57 % of the cycles (pairs:
// 66 %), at 1.9 GHz under this load; a stage's fragments and DMAs are 128 KB of LDS, without a bank conflict, as long at 128
// bytes a cycle as its products.  A tile's results, which all CUs write at about the same time, take a fifth of the time.
// Small matrices are bound by the launches: 2 + 3 a step, 4.2 us each.
// The two waves of a SIMD work in opposite phases, a barrier apart: one reads its fragments from LDS while the other
// multiplies.  Waves 4..7 ("late") run one phase behind waves 0..3: stage s is read in phases 2s and 2s + 1, its slot is
// refilled from phase 2s + 2 on, and both groups write a finished tile's results in the phase after its last read.  A phase
// is short (32 products of 16 cycles), so what stands between two barriers beside them is kept small: 20 scalar
// instructions in front of the products were 5 % of the whole.
enum { GRAM, POLY, UPDATE, FINAL };
template <int T, bool SPLIT> struct Cfg {
    static constexpr int WM = T == 64 ? 4 : 2, WN = 8 / WM;         // waves along rows and columns
    static constexpr int MI = T / 16 / WM, NI = T / 16 / WN;        // fragments of 16 x 16 a wave
    // parts of a stage: KB panels of P and of Q (SPLIT: Q's hi, then its lo).  Two panels for T <= 128: half the phases,
    // whose fixed part (barrier, LDS latency: about 0.25 us) is otherwise longer than their products
    static constexpr int KB = T <= 128 ? 2 : 1, PP = KB, QP = SPLIT ? 2 * KB : KB;
    static constexpr int OPB = T * BK * 2, STAGE = (PP + QP) * OPB;
    static constexpr int S = T == 128 ? (SPLIT ? 3 : 2) : SPLIT && T == 256 ? 3 : 4;
    static constexpr int PIECES = T / 16;                           // DMAs a part, of 16 rows of P each
    static constexpr int NP = PP * PIECES / 8, NQ = QP * PIECES / 8;    // ... a wave and stage
    static constexpr int SUBM = 16 * MI, SUBN = 16 * NI;            // a wave's part of the tile
    static constexpr int IMG = SPLIT ? 0 : 16 * SUBM * 2;           // image of 16 columns of it (UPDATE has none)
    static constexpr int SMEM = S * STAGE + 8 * IMG;                // T = 256: 160 KB (SPLIT: 144), 128: 80 (144), 64: 68 (96)
    static constexpr int PER_CU = T <= 128 && !SPLIT ? 2 : 1;       // workgroups a CU: LDS and registers allow so many
};
// The DMA is written in assembly: behind the builtin the compiler waits for ALL requests before every transposing LDS
// read, which may alias what is being filled for all it knows.  It has no register result; the waits are landed()'s.
// M0 is written nowhere else.
DEVI u32x4 rsrc(const void* p, int bytes) {
    const uint64_t a = (uint64_t)p;
    u32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((unsigned)a);
    r[1] = __builtin_amdgcn_readfirstlane((unsigned)(a >> 32));
    r[2] = __builtin_amdgcn_readfirstlane(bytes);         // offsets past the end are dropped
    r[3] = 0x00020000;
    return r;
}
DEVI void dma16(unsigned lds, int voff, const u32x4& rs, int soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
                 ::"s"(lds), "v"(voff), "s"(rs), "s"(soff) : "memory");
}
// chunk permutation of a [32 rows][4 chunks] panel: the eight rows (8 apart in two groups of four) that half a wave's
// transposing read touches lie in different banks
DEVI int tkey(int row) { return 2 * ((row >> 3) & 1); }

// odd rows of 16 lanes of w[0], w[1] trade places with even rows of w[2], w[3] (its own inverse)
DEVI u32x4 swap16(const u32x4& w) {
    const auto x = __builtin_amdgcn_permlane16_swap(w[0], w[2], false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(w[1], w[3], false, false);
    return u32x4{x[0], y[0], x[1], y[1]};
}
// eight 16-bit values, of which `left` lie inside the row; addresses are multiples of `align` bytes
DEVI void store8x16(uint16_t* o, const u32x4& w, int align, int left) {
    if (align >= 16 && left >= 8) *(u32x4*)o = w;
    else if (align >= 8 && left >= 8) {
        *(u32x2*)o = u32x2{w[0], w[1]};
        *(u32x2*)(o + 4) = u32x2{w[2], w[3]};
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < left) o[k] = (uint16_t)(k & 1 ? w[k / 2] >> 16 : w[k / 2] & 0xffffu);
    }
}
template <bool TOBF> DEVI unsigned pack2(float a, float b) {
    if (TOBF) {
        const bf16x2 v = {(bf16)a, (bf16)b};
        return __builtin_bit_cast(unsigned, v);
    }
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {(f16)a, (f16)b};
    return __builtin_bit_cast(unsigned, v);
}

template <int MODE, int T, bool SPLIT>
__global__ __launch_bounds__(512, (2 * Cfg<T, SPLIT>::PER_CU)) void ortho_gemm_kernel(const GemmArgs ga) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Cfg<T, SPLIT> C;
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    constexpr int S = C::S, MI = C::MI, NI = C::NI, KB = C::KB, PP = C::PP, QP = C::QP, NP = C::NP, NQ = C::NQ;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / C::WN, wn = wave % C::WN, i = lane & 15, g = lane >> 4;
    int late = wave >> 2;
    asm volatile("" : "+s"(late));             // (an integer to the compiler, compared by scalar instructions)
    const Ws& ws = ga.ws;
    const Tile* tiles = SYM ? ws.sym : ws.rect;
    // workgroup -> tiles b, b + G, ...: in every round an XCD has neighbouring tiles
    const int G = gridDim.x, b0 = xcd_remap(blockIdx.x, G);
    const int nmine = (ga.ntiles - b0 + G - 1) / G;

    // ---- stages: 32 columns of T rows of P ([row][4 chunks of 16 B]), and of Q either the same or, for UPDATE, 32 rows
    // of T columns (T / 32 panels of [32 rows][4 chunks]).  The operands lie in memory as panels of 32 columns, so every
    // DMA of a wave moves 1 KB in one piece.  Chunks are permuted by a key of the row so that no read meets itself
    // in a bank.  Rows behind the matrix read zeros or the next panel, panels behind it the last one: only their own
    // results, which are not stored, see them.  (A request never starts behind its buffer: the range check subtracts the
    // uniform part of the offset from the size.)  A wave moves pieces wave, wave + 8, ...: first P's, then Q's.
    // Piece e = wave + 8 n of an operand is piece e % PIECES of its part e / PIECES.
    constexpr int ND = C::PIECES >= 8 ? C::PIECES / 8 : 1;   // different pieces of a part that a wave takes
    int voP[ND], voQ[ND];
#pragma unroll
    for (int u = 0; u < ND; ++u) {
        const int e = (wave + 8 * u) % C::PIECES, r = e * 16 + (lane >> 2), t = (e & 1) * 16 + (lane >> 2);
        voP[u] = r * 64 + (((lane & 3) ^ fsw(r >> 2)) << 4);
        voQ[u] = SYM ? voP[u] : t * 64 + (((lane & 3) ^ tkey(t)) << 4);
    }
    u32x4 rsP, rsQ[SPLIT ? 2 : 1];
    const unsigned lds0 = (unsigned)(uintptr_t)(lptr_t)smem + wave * 1024;
    // the next stage to request: its tile's index, stages left in the tile, LDS address, offsets in P and Q, their steps
    int ji = 0, left = 0, soP = 0, soQ[ND], panel = 0, stepQ = 0;
    unsigned iat = lds0;
    Tile tn = load_tile(tiles + b0);                       // the tile after the one being requested
    auto open = [&]() {                        // start requesting tile tn
        panel = tn.mp * 64;
        stepQ = KB * (SYM ? panel : 2048);
        soP = tn.m0 * 64;
#pragma unroll
        for (int u = 0; u < ND; ++u)
            soQ[u] = SYM ? tn.n0 * 64 : min((tn.n0 >> 5) + (((wave + 8 * u) % C::PIECES) >> 1), (tn.np >> 5) - 1) * panel;
        left = (MODE == GRAM ? tn.np : tn.mp) / (BK * KB);
        rsP = rsrc(MODE == GRAM ? ws.x[ga.src][0] + tn.xo : MODE == POLY ? ws.a + tn.ao : ws.b + tn.ao,
                   tn.mp * (MODE == GRAM ? tn.np : tn.mp) * 2);
#pragma unroll
        for (int h = 0; h < (SPLIT ? 2 : 1); ++h)
            rsQ[h] = rsrc(MODE == POLY ? ws.a + tn.ao : ws.x[ga.src][h] + tn.xo, tn.mp * (MODE == POLY ? tn.mp : tn.np) * 2);
        if (ji + 1 < nmine) tn = load_tile(tiles + b0 + (ji + 1) * G);
    };
    open();
    constexpr int NREQ = NP + NQ;                          // requests of a wave and stage
    static_assert(QP * MI >= NREQ, "multiply() takes one request a row");
    auto part_of = [&](int n) { return C::PIECES >= 8 ? 8 * n / C::PIECES : (wave + 8 * n) / C::PIECES; };
    auto request = [&](int n) {
        if (n < NP) {
            const int h = part_of(n);
            dma16(iat + n * 8192, voP[n % ND], rsP, soP + h * panel);
        } else {
            n -= NP;
            const int h = part_of(n);                      // (h % KB: panel along the contraction)
            dma16(iat + PP * C::OPB + n * 8192, voQ[n % ND], rsQ[SPLIT ? 8 * n / (C::PIECES * KB) : 0],
                  soQ[n % ND] + (h % KB) * (SYM ? panel : 2048));
        }
    };
    // (Behind the last tile the requests go on, to the last matrix's first rows: a stage is always NREQ of them.)
    auto requested = [&]() {
        soP += KB * panel;
#pragma unroll
        for (int u = 0; u < ND; ++u) soQ[u] += stepQ;
        iat += C::STAGE;
        if (iat == lds0 + S * C::STAGE) iat = lds0;
        if (--left == 0) {
            if (++ji < nmine) open();
            else {
                soP = panel = stepQ = 0;
#pragma unroll
                for (int u = 0; u < ND; ++u) soQ[u] = 0;
            }
        }
    };
    auto issue = [&]() {
#pragma unroll
        for (int n = 0; n < NREQ; ++n) request(n);
        requested();
    };
    // my DMAs of the next stage to read are done: at most S - 2 stages are younger
    auto landed = [&]() { wait_vmcnt<NREQ * (S - 2)>(); };

    f32x4 acc[MI][NI];
    auto clear = [&]() {
#pragma unroll
        for (int a = 0; a < MI; ++a)
#pragma unroll
            for (int c = 0; c < NI; ++c) acc[a][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    };
    clear();
    const int rp = wm * C::SUBM + i, offP = rp * 64 + ((g ^ fsw(rp >> 2)) << 4);
    const int rq = wn * C::SUBN + i, offQ = PP * C::OPB + rq * 64 + ((g ^ fsw(rq >> 2)) << 4);
    int offT[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
        const int row = 8 * g + (i >> 2), col = wn * C::SUBN + ni * 16, ch = (col & 31) / 8 + ((i & 3) >> 1);
        offT[ni] = PP * C::OPB + (col >> 5) * 2048 + row * 64 + ((ch ^ tkey(row)) << 4) + (i & 1) * 8;
    }
    // LATER: a slot is refilled a phase later than its last read (one phase less ahead), and no wait for that read stands in
    // front of the barrier: the products wait for their own operands as they come.  X' of pairs of ViT-L's matrices 1205 ->
    // 1056 us when it was built.  With two stages there is no phase to spare.
    constexpr bool LATER = S > 2;
    u32x4 fp[PP][MI], fq[QP][NI];
    int slot = 0;
    auto read = [&]() {
        const char* st = smem + slot * C::STAGE;
        slot = slot + 1 == S ? 0 : slot + 1;
#pragma unroll
        for (int h = 0; h < QP; ++h)
#pragma unroll
            for (int x = 0; x < NI; ++x) {
                const char* sh = st + h * C::OPB;
                if (SYM) fq[h][x] = *(const u32x4*)(sh + offQ + x * 1024);
                else {
                    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(sh + offT[x])));
                    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(sh + offT[x] + 256)));
                    fq[h][x] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                }
            }
#pragma unroll
        for (int h = 0; h < PP; ++h)
#pragma unroll
            for (int x = 0; x < MI; ++x) fp[h][x] = *(const u32x4*)(st + h * C::OPB + offP + x * 1024);
        if (!LATER) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    // with the requests of a stage between the products, whose time they then do not take
    auto multiply = [&](bool req) {
#pragma unroll
        for (int h = QP - 1; h >= 0; --h)
#pragma unroll
            for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        __builtin_bit_cast(f16x8, fq[h][ni]), __builtin_bit_cast(f16x8, fp[h % KB][mi]), acc[mi][ni], 0, 0, 0);
                const int n = (QP - 1 - h) * MI + mi;
                if (n < NREQ && req) request(n);
                if (n == NREQ && req) requested();
            }
        if (QP * MI == NREQ && req) requested();
    };
    auto phase = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
    };

    // ---- results of a tile.  Lane (i, g) holds columns 16 ni + 4 g + r of row 16 mi + i of its wave's part.
    char* img = smem + S * C::STAGE + wave * C::IMG;
    auto finish = [&](const Tile& d, float e1) {
        const int mp = d.mp, np = d.np;
        // the matrix's own exponent: products of two stored X (A) carry 2^2e, of two A's 2^4e too much; B is kept without
        const float e2 = e1 * e1;
        const float c0 = ga.c0 * e2, c1 = MODE == POLY ? ga.c1 * e2 * e2 : MODE == FINAL ? ga.c1 * e1 : ga.c1;
        const int wm0 = d.m0 + wm * C::SUBM, wn0 = d.n0 + wn * C::SUBN;
        const int nend = SYM ? mp : np;
        // Where fragment (mi, ni) lies in a matrix of panels: a lane's part and a uniform one (mp is a multiple of 64, so a
        // fragment is inside as a whole or outside as a whole).
        // A store or load takes 16 bytes a lane: the two fragments of a panel trade halves between lanes 16 apart, after
        // which lane (i, g) holds columns 8 (g / 2) .. + 7 of fragment ni + g % 2 -- 64 bytes of a row from four lanes,
        // 1 KB in one piece from the wave.
        const int vlane = i * 64 + (g & 1) * 32 + (g >> 1) * 16;
        auto upart = [&](int ni) { return (min((wn0 + 16 * ni) >> 5, (nend >> 5) - 1) * mp + min(wm0, mp - 16)) * 64; };
        // (ni even; + 1024 mi)
        if (MODE == POLY) {
            // (loads without a branch, so that they are in flight together: a fragment behind the matrix reads another one or
            // zero and is not stored)
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)(ws.a + d.ao), 0, mp * mp * 2, 0x00020000);
            constexpr int PART = (MI + 1) / 2;
#pragma unroll
            for (int q = 0; q < MI; q += PART) {
                u32x4 el[PART][NI / 2];
#pragma unroll
                for (int mi = 0; mi < PART; ++mi)
#pragma unroll
                    for (int ni = 0; ni < NI; ni += 2)
                        el[mi][ni / 2] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, vlane + (q + mi) * 1024, upart(ni), 0));
#pragma unroll
                for (int mi = 0; mi < PART; ++mi)
#pragma unroll
                    for (int ni = 0; ni < NI; ni += 2) {
                        const u32x4 w = swap16(el[mi][ni / 2]);
                        const f16x4 x0 = __builtin_bit_cast(f16x4, u32x2{w[0], w[1]}), x1 = __builtin_bit_cast(f16x4, u32x2{w[2], w[3]});
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            acc[q + mi][ni][r] = fmaf(c0, (float)x0[r], acc[q + mi][ni][r] * c1);
                            acc[q + mi][ni + 1][r] = fmaf(c0, (float)x1[r], acc[q + mi][ni + 1][r] * c1);
                        }
                    }
            }
            if (d.m0 == d.n0) {
                int off = wm0 + i - wn0 - 4 * g;
                asm volatile("" : "+v"(off));        // (or the 128 comparisons, the same for every tile, are kept in registers)
#pragma unroll
                for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                    for (int ni = 0; ni < NI; ++ni)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[mi][ni][r] += off == 16 * (ni - mi) + r ? ga.ca : 0.f;
            }
        } else {
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[mi][ni][r] *= c1;
        }
        // the fragments (mi, ni) and (mi, ni + 1) as 16 bytes a lane
        auto pair = [&](auto tobf_c, int mi, int ni) {
            constexpr bool TOBF = decltype(tobf_c)::value;
            const f32x4 a = acc[mi][ni], b = acc[mi][ni + 1];
            return swap16(u32x4{pack2<TOBF>(a[0], a[1]), pack2<TOBF>(a[2], a[3]), pack2<TOBF>(b[0], b[1]), pack2<TOBF>(b[2], b[3])});
        };
        auto put = [&](f16* dst) {
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)dst, 0, mp * nend * 2, 0x00020000);
#pragma unroll
            for (int ni = 0; ni < NI; ni += 2) {
                if (wn0 + 16 * ni >= nend) continue;
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) {
                    if (wm0 + 16 * mi >= mp) continue;
                    __builtin_amdgcn_raw_buffer_store_b128(pair(std::false_type{}, mi, ni), rs, vlane + mi * 1024, upart(ni), 0);
                }
            }
        };
        // ... by columns (a mirrored tile, a tall matrix of the caller's) through an image of 16 columns at a time in LDS, so
        // that a store covers rows of the destination; a wave reads only what it wrote.
        auto put_columns = [&](auto tobf_c, uint16_t* dst, int64_t ld, int rows, int cols, int align) {
            constexpr bool TOBF = decltype(tobf_c)::value;
            constexpr int RB = C::SUBM * 2;
            auto at = [&](int c, int m) { return c * RB + ((m * 2) ^ ((c >> 1 & (C::SUBM / 16 - 1)) << 5)); };
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) {
                    // lanes i and i ^ 1 (rows m, m + 1) trade: the even one gets columns r = 0, 1 of both, the odd one 2, 3
                    const f32x4 v = acc[mi][ni];
                    const bool odd = i & 1;
                    const float x0 = dpp_mov<0xB1>(odd ? v[0] : v[2]), x1 = dpp_mov<0xB1>(odd ? v[1] : v[3]);
                    const int c = 4 * g + (odd ? 2 : 0), m = mi * 16 + (i & ~1);
                    *(unsigned*)(img + at(c, m)) = odd ? pack2<TOBF>(x0, v[2]) : pack2<TOBF>(v[0], x0);
                    *(unsigned*)(img + at(c + 1, m)) = odd ? pack2<TOBF>(x1, v[3]) : pack2<TOBF>(v[1], x1);
                }
                for (int e = lane; e < 2 * C::SUBM; e += 64) {
                    // panels: up to 64 bytes of each of the 16 columns; else whole columns
                    constexpr int CH = C::SUBM < 32 ? C::SUBM / 8 : 4;
                    const int c = TOBF ? e / (C::SUBM / 8) : (e / CH) & 15;
                    const int m = TOBF ? (e - c * (C::SUBM / 8)) * 8 : e / (16 * CH) * 32 + e % CH * 8;
                    const u32x4 w = *(const u32x4*)(img + at(c, m));
                    const int dr = wn0 + ni * 16 + c, dc = wm0 + m;
                    if (dr >= rows || dc >= cols) continue;
                    uint16_t* o = dst + (TOBF ? dr * ld + dc : ((int64_t)(dc >> 5) * ld + dr) * 32 + (dc & 31));
                    store8x16(o, w, TOBF ? align : 16, cols - dc);
                }
            }
        };
        auto take_hi = [&]() {       // what the fp16 just written has left of the values
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[mi][ni][r] -= (float)(f16)acc[mi][ni][r];
        };
        if (SYM) {
            f16* o = (MODE == GRAM ? ws.a : ws.b) + d.ao;
            put(o);
            if (d.m0 != d.n0) put_columns(std::false_type{}, (uint16_t*)o, mp, mp, mp, 16);
        } else if (MODE == UPDATE) {
            put(ws.x[ga.src ^ 1][0] + d.xo);
            if (SPLIT && ga.split_next) {          // (pairs are used from the first step on)
                take_hi();
                put(ws.x[ga.src ^ 1][1] + d.xo);
            }
        } else {
            const Mat& q = ws.mats[d.item];
            bf16* out = (bf16*)q.out + d.mat * q.out_batch;
            const uint64_t bits = (uintptr_t)out | (uint64_t)(q.out_ld * 2);
            const int al = (bits & 15) == 0 ? 16 : (bits & 7) == 0 ? 8 : 2;
            if (q.tall) put_columns(std::true_type{}, (uint16_t*)out, q.out_ld, q.n, q.m, al);
            else {
#pragma unroll
                for (int mi = 0; mi < MI; ++mi) {
                    const int m = wm0 + mi * 16 + i;
#pragma unroll
                    for (int ni = 0; ni < NI; ni += 2) {
                        const u32x4 w = pair(std::true_type{}, mi, ni);
                        const int n = wn0 + 16 * ni + (g & 1) * 16 + (g >> 1) * 8;
                        if (m < q.m && n < q.n) store8x16((uint16_t*)out + m * q.out_ld + n, w, al, q.n - n);
                    }
                }
            }
        }
        clear();
    };

    // ---- the stream of stages.  Early waves read stage s in phase 2s and multiply in 2s + 1, late ones a phase later; a
    // tile that ended with s is finished by both in phase 2s + 2.  Stage s + S is requested into the slot of s in phase
    // 2s + 2, LATER in 2s + 3: early waves' reads are waited for by their products in 2s + 1, late ones' in 2s + 2 (or at
    // the end of 2s + 1).
    for (int s = 0; s < S - 1; ++s) issue();
    Tile cur = load_tile(tiles + b0), nxt = load_tile(tiles + b0 + (nmine > 1 ? G : 0));
    int total = (MODE == GRAM ? cur.np : cur.mp) / (BK * KB), j = 0, k = 0;
    float e1 = load_const(ws.exps + cur.all);
    landed();
    phase();
    if (!LATER) issue();
    if (late) phase();
    for (;;) {
        read();
        if (late) {
            if (LATER) issue();
            landed();
        }
        phase();
        multiply(LATER ? !late : late);
        if (!late) {
            landed();
            phase();
            if (!LATER) issue();
        }
        if (++k == total) {
            finish(cur, e1);
            if (++j == nmine) break;
            cur = nxt;
            e1 = load_const(ws.exps + cur.all);
            if (j + 1 < nmine) nxt = load_tile(tiles + b0 + (j + 1) * G);
            total = (MODE == GRAM ? cur.np : cur.mp) / (BK * KB);
            k = 0;
        }
        if (late) phase();
    }
    wait_vmcnt<0>();                            // no request outlives the workgroup's LDS
#endif
}

// ---- host side ------------------------------------------------------------------------------------------------
int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

struct Layout {
    int64_t bytes, mats, sym, rect, map, parts, exps, x, a;      // byte offsets; x / a: first region, xbytes / abytes apart
    int64_t xbytes, abytes, ntile[3];
    int tile[2];                                    // of the symmetric products, of the update
};

int describe(const dino_ortho_item* items, int count, Mat* out, Layout& L) {
    int64_t xo = 0, ao = 0, sym = 0, rect = 0, prep = 0, parts = 0, nmat = 0;
    for (int i = 0; i < count; ++i) {
        const dino_ortho_item& s = items[i];
        if (s.rows <= 0 || s.cols <= 0 || s.batch < 0 || (s.dtype != DINO_F32 && s.dtype != DINO_BF16)) return DINO_ERR_BADARG;
        if (s.rows > 32768 || s.cols > 32768) return DINO_ERR_TOO_LARGE;   // a matrix is one buffer below 2^31 bytes
        Mat q{};
        q.in = s.in; q.out = s.out;
        q.in_batch = s.in_batch; q.in_ld = s.in_ld; q.out_batch = s.out_batch; q.out_ld = s.out_ld;
        q.rows = s.rows; q.cols = s.cols; q.batch = s.batch; q.dtype = s.dtype;
        q.tall = s.rows > s.cols;
        q.m = q.tall ? s.cols : s.rows;
        q.n = q.tall ? s.rows : s.cols;
        q.mp = (int)up(q.m, 64);
        q.np = (int)up(q.n, 64);
        if ((int64_t)q.mp * q.np * 2 >= (1ll << 31)) return DINO_ERR_TOO_LARGE;
        // elements a workgroup of the norm: few where many would leave CUs idle (with 16384 throughout and one load in flight:
        // one of 192 x 192 7 us, now 5; one of 1024 x 588 and small ones 12, now 5; the head MLP's 13, now 11)
        const int64_t each = (int64_t)s.batch * q.m * q.n > (1 << 22) ? 16384 : 4096;
        int64_t p = ((int64_t)q.m * q.n + each - 1) / each;
        if (p > 256) p = 256;
        q.parts = (int)(p > q.rows ? q.rows : p);
        const int64_t pt = (int64_t)((q.mp + 63) / 64) * ((q.np + 63) / 64);
        q.preps = (int)(pt * s.batch > 16384 ? 8 : pt * s.batch > 4096 ? 2 : 1);
        q.mat0 = (int)nmat;
        q.part0 = (int)parts; q.xoff = xo; q.aoff = ao; q.prep0 = (int)prep;
        parts += (int64_t)s.batch * q.parts;
        xo += (int64_t)s.batch * q.mp * q.np;
        ao += (int64_t)s.batch * q.mp * q.mp;
        prep += (int64_t)s.batch * ((pt + q.preps - 1) / q.preps);
        nmat += s.batch;
        if (prep >= (1 << 24) || parts >= (1 << 24)) return DINO_ERR_TOO_LARGE;    // 256 threads each, < 2^32 a launch
        if (out) out[i] = q;
    }
    // Tile size of the symmetric products and of the update, each the one of least estimated time: rounds of tiles over
    // the 256 CUs, a tile of 256 costing 256 a stage, one of 128 (two share a CU and overlap their starts and ends) 83.  Tiles of
    // 64 have the shorter phases, but read twice as much for a product; two of them on a CU cost 53 (symmetric: less of the
    // matrix twice) or 78.  So 64 is taken where all of them run at once.  Measured (us): a launch with 256 / 128: ViT-L's matrices A 371 / 391, B 219 / 231, X' 590 / 763,
    // of pairs 1010 / 1300; ViT-S's A 46 / 31, B 22 / 15, X' 30 / 29, of pairs 51 / 49; the head MLP's A 52 / 24, X' 48 / 34, of
    // pairs 83 / 42.  A launch with 128 / 64: one of 192 x 192 5.5 / 4.4; one of 1024 x 588 and small ones A 13 / 8, B 11 / 6;
    // the head's A 24 / 33; ViT-S's X' 31 / 45.  A whole call: one of 1024 x 1024 225 / 145, of 512 x 512 147 / 100,
    // 48 of 192 x 192 and 24 of 768 x 192 172 / 154 (64 for A and B only), 24 and 12 of 384 292 / 324.
    for (int kind = 0; kind < 2; ++kind) {
        double best = 0;
        for (int T = 256; T >= 64; T /= 2) {
            double work = 0, tiles = 0;
            for (int i = 0; i < count; ++i) {
                const int64_t m = up(items[i].rows < items[i].cols ? items[i].rows : items[i].cols, 64);
                const int64_t n = up(items[i].rows < items[i].cols ? items[i].cols : items[i].rows, 64);
                const double tm = (double)((m + T - 1) / T), tn = (double)((n + T - 1) / T);
                const double k = kind ? tm * tn * items[i].batch : tm * (tm + 1) / 2 * items[i].batch;
                tiles += k;
                work += k * (double)(kind ? m : n + m);
            }
            if (tiles == 0) tiles = 1;
            const double cost = work / tiles * (T == 64 ? ceil(tiles / 512) * (kind ? 78 : 53) : ceil(tiles / 256) * (T == 256 ? 256 : 83));
            if (T == 256 || cost < best) { best = cost; L.tile[kind] = T; }
        }
    }
    // tiles with the longest contraction first: the last round then ends evenly
    int* order = (int*)malloc(sizeof(int) * (size_t)(count + 1));
    if (!order) return DINO_ERR_TOO_LARGE;
    for (int i = 0; i < count; ++i) order[i] = i;
    auto lo_side = [&](int i) { return items[i].rows < items[i].cols ? items[i].rows : items[i].cols; };
    auto hi_side = [&](int i) { return items[i].rows < items[i].cols ? items[i].cols : items[i].rows; };
    for (int kind = 0; kind < 2; ++kind) {
        std::stable_sort(order, order + count, [&](int a, int b) { return kind ? lo_side(a) > lo_side(b) : hi_side(a) > hi_side(b); });
        for (int o = 0; o < count; ++o) {
            const int i = order[o], T = L.tile[kind];
            const int64_t m = up(lo_side(i), 64), n = up(hi_side(i), 64), tm = (m + T - 1) / T;
            int64_t& at = kind ? rect : sym;
            if (out) (kind ? out[i].rect0 : out[i].sym0) = (int)at;
            at += items[i].batch * (kind ? tm * ((n + T - 1) / T) : tm * (tm + 1) / 2);
        }
    }
    free(order);
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t r = at; at = up(at + bytes, 256); return r; };
    L.ntile[0] = sym; L.ntile[1] = rect; L.ntile[2] = prep;
    L.mats = take((int64_t)sizeof(Mat) * count);
    L.sym = take((int64_t)sizeof(Tile) * sym);
    L.rect = take((int64_t)sizeof(Tile) * rect);
    L.map = take(4 * prep);
    L.parts = take(8 * parts);
    L.exps = take(4 * nmat);
    L.xbytes = up(2 * xo, 256);
    L.abytes = up(2 * ao, 256);
    L.x = take(4 * L.xbytes);
    L.a = take(2 * L.abytes);
    L.bytes = at;
    return DINO_OK;
}

// largest |p(x)| and |q| over singular values x up to `top`,  p = x q,  q = a + b x^2 + c x^4: at the ends or where a
// derivative is 0  (q' = 2 x (b + 2 c y),  p' = a + 3 b y + 5 c y^2,  y = x^2)
void poly_bounds(const float* co, double top, double& px, double& qx) {
    const double a = co[0], b = co[1], c = co[2], end = top * top, disc = 9 * b * b - 20 * a * c;
    double y[5] = {0, end, -1, -1, -1};
    if (c != 0) {
        y[2] = -b / (2 * c);
        if (disc >= 0) {
            y[3] = (-3 * b + sqrt(disc)) / (10 * c);
            y[4] = (-3 * b - sqrt(disc)) / (10 * c);
        }
    } else if (b != 0) y[3] = -a / (3 * b);
    px = qx = 0;
    for (double v : y) {
        if (!(v >= 0 && v <= end)) continue;
        const double q = fabs(a + b * v + c * v * v);
        px = fmax(px, q * sqrt(v));
        qx = fmax(qx, q);
    }
}

template <int MODE, int T, bool SPLIT> int launch_as(const GemmArgs& ga, hipStream_t st) {
    constexpr int smem = Cfg<T, SPLIT>::SMEM;
    static bool ready[64];                            // by device; two threads may both set it, to the same
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return (int)e;
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        e = hipFuncSetAttribute((const void*)ortho_gemm_kernel<MODE, T, SPLIT>, hipFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != hipSuccess) return (int)e;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    const int most = 256 * Cfg<T, SPLIT>::PER_CU;     // what the CUs hold at once
    hipLaunchKernelGGL((ortho_gemm_kernel<MODE, T, SPLIT>), dim3(ga.ntiles < most ? ga.ntiles : most), dim3(512), smem, st, ga);
    return dino_launch_status();
}
template <int MODE> int launch_gemm(GemmArgs& ga, int T, bool split, int64_t tiles, hipStream_t st) {
    ga.ntiles = (int)tiles;
    if (MODE == UPDATE && split)
        return T == 256 ? launch_as<UPDATE, 256, true>(ga, st) : T == 128 ? launch_as<UPDATE, 128, true>(ga, st) : launch_as<UPDATE, 64, true>(ga, st);
    return T == 256 ? launch_as<MODE, 256, false>(ga, st) : T == 128 ? launch_as<MODE, 128, false>(ga, st) : launch_as<MODE, 64, false>(ga, st);
}

}  // namespace

extern "C" int dino_ortho_workspace(const dino_ortho_item* items, int count, int64_t* bytes) {
    DINO_CHECK_ARG(bytes && count >= 0 && (count == 0 || items));
    Layout L;
    const int rc = describe(items, count, nullptr, L);
    if (rc == DINO_OK) *bytes = L.bytes;
    return rc;
}

extern "C" int dino_ortho(const dino_ortho_item* items, int count, int steps, const float* coeffs, double eps,
                          void* workspace, int64_t workspace_bytes, void* stream) {
    DINO_CHECK_ARG(count >= 0 && (count == 0 || items) && steps >= 1 && steps <= DINO_ORTHO_MAX_STEPS && coeffs);
    DINO_CHECK_ARG(eps >= 0.0 && eps < 1e30);
    // How far the singular values (at most 1 at first) can get, step by step: fp16 holds X times SX
    double top = 1.0, sa[DINO_ORTHO_MAX_STEPS], sb[DINO_ORTHO_MAX_STEPS], grow[DINO_ORTHO_MAX_STEPS];
    for (int s = 0; s < steps; ++s) {
        double px, qx;
        for (int k = 0; k < 3; ++k) DINO_CHECK_ARG(fabsf(coeffs[3 * s + k]) < 1e4f);
        poly_bounds(coeffs + 3 * s, top * 1.01, px, qx);
        DINO_CHECK_ARG(px < 12.0);
        sa[s] = exp2(floor(log2(30000.0 / (top * top * 1.1))));
        sb[s] = exp2(floor(log2(30000.0 / fmax(qx * 1.1, 1e-3))));
        if (sb[s] > 4096.0) sb[s] = 4096.0;
        top = fmax(px, 1e-3);
    }
    double gain = 1.0;
    for (int s = steps - 1; s >= 0; --s) {
        grow[s] = gain;                           // growth of an error made in step s
        gain *= fmax(1.0, fabs((double)coeffs[3 * s]));
    }
    int total = 0;
    for (int i = 0; i < count; ++i) total += items[i].batch > 0;
    if (total == 0) return DINO_OK;
    Mat* mats = (Mat*)malloc(sizeof(Mat) * (size_t)count);
    if (!mats) return DINO_ERR_TOO_LARGE;
    Layout L;
    int rc = describe(items, count, mats, L);
    for (int i = 0; rc == DINO_OK && i < count; ++i)
        if (items[i].batch > 0 && (!items[i].in || !items[i].out || items[i].in_ld < items[i].cols || items[i].out_ld < items[i].cols))
            rc = DINO_ERR_BADARG;
    if (rc == DINO_OK && (!workspace || workspace_bytes < L.bytes || ((uintptr_t)workspace & 255))) rc = DINO_ERR_BADARG;
    if (rc != DINO_OK) { free(mats); return rc; }
    char* w = (char*)workspace;
    Ws ws;
    ws.mats = (Mat*)(w + L.mats);
    ws.sym = (Tile*)(w + L.sym);
    ws.rect = (Tile*)(w + L.rect);
    ws.map_prep = (int*)(w + L.map);
    ws.parts = (double*)(w + L.parts);
    ws.exps = (float*)(w + L.exps);
    ws.tsym = L.tile[0];
    ws.trect = L.tile[1];
    for (int k = 0; k < 2; ++k)
        for (int h = 0; h < 2; ++h) ws.x[k][h] = (f16*)(w + L.x + (2 * k + h) * L.xbytes);
    ws.a = (f16*)(w + L.a);
    ws.b = (f16*)(w + L.a + L.abytes);
    const hipStream_t st = (hipStream_t)stream;
    for (int i0 = 0; i0 < count; i0 += ITEMS) {
        Setup su;
        su.first = i0;
        su.count = count - i0 < ITEMS ? count - i0 : ITEMS;
        int wg = 0;
        for (int i = 0; i < su.count; ++i) {
            su.it[i] = mats[i0 + i];
            su.wg0[i] = wg;
            wg += su.it[i].batch * su.it[i].parts;
        }
        su.wg0[su.count] = wg;
        if (wg) hipLaunchKernelGGL(ortho_norm_kernel, dim3(wg), dim3(NTHR), 0, st, su, ws);
    }
    free(mats);
    auto split = [&](int s) { return s < steps && grow[s] > SPLIT_ABOVE; };
    hipLaunchKernelGGL(ortho_prep_kernel, dim3((unsigned)L.ntile[2]), dim3(NTHR), 0, st, ws, eps, gain, (int)split(0));
    rc = dino_launch_status();
    for (int s = 0; s < steps && rc == DINO_OK; ++s) {
        const float* c = coeffs + 3 * s;
        GemmArgs ga{ws, s & 1, split(s + 1), 0, 0.f, (float)(sa[s] / ((double)SX * SX)), 0.f};
        rc = launch_gemm<GRAM>(ga, L.tile[0], false, L.ntile[0], st);
        if (rc != DINO_OK) break;
        ga.c0 = (float)(c[1] * sb[s] / sa[s]);
        ga.c1 = (float)(c[2] * sb[s] / (sa[s] * sa[s]));
        ga.ca = (float)(c[0] * sb[s]);
        rc = launch_gemm<POLY>(ga, L.tile[0], false, L.ntile[0], st);
        if (rc != DINO_OK) break;
        ga.c1 = (float)((s + 1 == steps ? 1.0 / SX : 1.0) / sb[s]);
        rc = s + 1 == steps ? launch_gemm<FINAL>(ga, L.tile[1], false, L.ntile[1], st)   // (the last step's errors do not grow)
                            : launch_gemm<UPDATE>(ga, L.tile[1], split(s), L.ntile[1], st);
    }
    return rc;
}
