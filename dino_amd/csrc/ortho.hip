// Orthogonalised updates (Newton-Schulz products, as the Muon optimiser takes them) for many matrices at once.
//
// X0 = U / (|U|_F + eps);  per step  A = X X^T,  B = b A + c A A,  X <- a X + B X   (X [m, n], m <= n: the shorter side of
// U in front);  the result is X in U's orientation, in bf16.  With the usual (a, b, c) every singular value of U ends
// near 1.
//
// Number formats.  The operands of the matrix instructions are fp16: every |x| is at most the largest singular value
// (about 1.2), so the range that bf16 pays three bits for is not needed; X, A, B are kept times powers of two that put
// them in the middle of fp16's range (X's by the matrix: an update that is small against eps starts at |U| / eps and
// ends at most `gain` = prod max(1, a) times that, so it is held 2^e times larger).  All sums are fp32 (the norm's fp64).  A rounding error made in step i grows by
// a^(steps - 1 - i) in the directions of small singular values (3.44^4 = 140 from the first of five steps), against an
// answer that is O(1) there.  While that factor is above SPLIT_ABOVE the operands are hi + lo pairs of fp16 (22 bits;
// products hi hi + hi lo + lo hi, three passes of the same loop); after that plain fp16.  On an update of four strong
// directions over noise the result is then 0.003 off 64 bits, with plain fp16 throughout 0.04, with bf16 0.33.
#include <math.h>
#include <stdlib.h>

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
constexpr float SX = 4096.f;                    // X is stored times this
constexpr double SPLIT_ABOVE = 16.0;

// One item: `batch` matrices of one shape.  Offsets in elements of the region of their kind.
struct Mat {
    const void* in;
    void* out;
    int64_t in_batch, in_ld, out_batch, out_ld, xoff, aoff;
    int rows, cols, batch, dtype;
    int tall, m, n, mp, np;                     // m <= n; mp, np: padded to 32 (zeros)
    int parts, part0, mat0;                     // partial sums of the norm: per matrix, first index; first matrix
    int sym0, rect0, prep0, nsym, nrect;        // first global tile of each kind; tiles of the whole item
};
struct Setup {
    Mat it[ITEMS];
    int wg0[ITEMS + 1];                         // first workgroup of each item
    int count, first;                           // items here, index of the first
};
// X, A, B lie as panels of 32 columns: element (r, c) of a matrix of mp rows at ((c / 32) mp + r) 32 + c % 32.
struct Ws {                                     // regions of the workspace
    Mat* mats;
    int *map_sym, *map_rect, *map_prep;         // tile -> item
    double* parts;
    float* exps;                                // per matrix: 2^-e
    f16 *x[2][2], *a[2], *b[2];                 // [buffer][hi / lo]
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

// squares of rows [r0, r1): a wave a row; V elements a lane and load
template <typename T, int V> DEVI double rows_sq(const T* p, int64_t ld, int cols, int r0, int r1) {
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T) * V)));
    const int lane = threadIdx.x & 63;
    double s = 0;
    for (int r = r0 + (threadIdx.x >> 6); r < r1; r += NTHR / 64) {
        const T* x = p + r * ld;
        for (int c = lane * V; c < cols; c += 64 * V) {
            if (V == 1 || c + V <= cols) {
                const vec v = *(const vec*)(x + c);
#pragma unroll
                for (int i = 0; i < V; ++i) { const double d = (double)(float)v[i]; s = fma(d, d, s); }
            } else {
                for (int i = c; i < cols; ++i) { const double d = (double)(float)x[i]; s = fma(d, d, s); }
            }
        }
    }
    return s;
}
template <typename T> DEVI double rows_sq(const void* in, int64_t at, int64_t ld, int cols, int r0, int r1) {
    const T* p = (const T*)in + at;
    if (((uintptr_t)p | (uint64_t)(ld * sizeof(T))) % (4 * sizeof(T)) == 0) return rows_sq<T, 4>(p, ld, cols, r0, r1);
    return rows_sq<T, 1>(p, ld, cols, r0, r1);
}

// Partial sums of squares (fp64: neither 1e-30 nor 1e30 leaves the range), and the item table with the tile -> item maps
// that the following launches read.
__global__ __launch_bounds__(NTHR) void ortho_norm_kernel(const Setup su, const Ws ws) {
    __shared__ double red[4];
    int i = 0;
    while (i + 1 < su.count && (int)blockIdx.x >= su.wg0[i + 1]) ++i;
    const Mat& q = su.it[i];
    const int w = blockIdx.x - su.wg0[i], nw = su.wg0[i + 1] - su.wg0[i], id = su.first + i;
    if (w == 0 && threadIdx.x == 0) ws.mats[id] = q;
    const int t0 = w * NTHR + threadIdx.x, ts = nw * NTHR;
    for (int t = t0; t < q.nsym; t += ts) ws.map_sym[q.sym0 + t] = id;
    for (int t = t0; t < q.nrect; t += ts) ws.map_rect[q.rect0 + t] = id;
    const int np_ = q.batch * ((q.mp + 63) / 64) * ((q.np + 63) / 64);
    for (int t = t0; t < np_; t += ts) ws.map_prep[q.prep0 + t] = id;
    const int b = w / q.parts, part = w - b * q.parts, per = (q.rows + q.parts - 1) / q.parts;
    const int r0 = part * per, r1 = min(q.rows, r0 + per);
    const double s = q.dtype == DINO_F32 ? rows_sq<float>(q.in, b * q.in_batch, q.in_ld, q.cols, r0, r1)
                                         : rows_sq<bf16>(q.in, b * q.in_batch, q.in_ld, q.cols, r0, r1);
    const double tot = block_sum_f64(s, red);
    if (threadIdx.x == 0) ws.parts[q.part0 + w] = tot;
}

// X0 = U * SX / (|U| + eps) as hi + lo, shorter side in front, padding cleared: 64 x 64 tiles through LDS where U is tall.
__global__ __launch_bounds__(NTHR) void ortho_prep_kernel(const Ws ws, double eps, double gain, int lo) {
    __shared__ double red[4];
    __shared__ float tile[64][65];
    const int id = ws.map_prep[blockIdx.x];
    const Mat& q = ws.mats[id];
    const int tm = (q.mp + 63) / 64, tn = (q.np + 63) / 64;
    int t = blockIdx.x - q.prep0;
    const int b = t / (tm * tn);
    t -= b * tm * tn;
    const int m0 = (t / tn) * 64, n0 = (t % tn) * 64;
    double s = 0;
    for (int p = threadIdx.x; p < q.parts; p += NTHR) s += ws.parts[q.part0 + b * q.parts + p];
    const double norm = sqrt(block_sum_f64(s, red)), end = gain * (norm / (norm + eps));
    const int e = end > 0.0 && end < 1.0 ? min(80, ilogb(1.0 / end)) : 0;
    const float scale = (float)(ldexp((double)SX, e) / (norm + eps));
    if (t == 0 && threadIdx.x == 0) ws.exps[q.mat0 + b] = ldexpf(1.f, -e);
    const int c = threadIdx.x & 63, r0 = threadIdx.x >> 6;
    for (int r = r0; r < 64; r += 4) {       // rows of U: m0.. of X, or n0.. where U is tall
        const int ur = (q.tall ? n0 : m0) + r, uc = (q.tall ? m0 : n0) + c;
        float v = 0.f;
        if (ur < q.rows && uc < q.cols) {
            const int64_t at = b * q.in_batch + ur * q.in_ld + uc;
            v = (q.dtype == DINO_F32 ? ((const float*)q.in)[at] : (float)((const bf16*)q.in)[at]) * scale;
        }
        tile[r][c] = v;
    }
    __syncthreads();
    f16* xh = ws.x[0][0] + q.xoff + (int64_t)b * q.mp * q.np;
    f16* xl = ws.x[0][1] + q.xoff + (int64_t)b * q.mp * q.np;
    for (int r = r0; r < 64; r += 4) {
        if (m0 + r >= q.mp || n0 + c >= q.np) continue;
        const float v = q.tall ? tile[c][r] : tile[r][c];
        const int64_t at = ((int64_t)((n0 + c) >> 5) * q.mp + m0 + r) * 32 + ((n0 + c) & 31);
        const f16 h = (f16)v;
        xh[at] = h;
        if (lo) xl[at] = (f16)(v - (float)h);
    }
}

struct GemmArgs {
    Ws ws;
    int src, split_next;             // X buffer read; the next step's operands are pairs
    float c0, c1;                    // epilogue: c0 * (elementwise operand) + c1 * product
};

DEVI int fsw(int x) { return (4 - (x & 3)) & 3; }
template <int N> DEVI void wait_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// T x T tile of a product per workgroup of eight waves (2 x 4, each T/2 x T/4).
//   GRAM    A = X X^T             rows of X against rows of X; tiles on and above the diagonal, written twice
//   POLY    B = b A + c A A       A symmetric: rows against rows again
//   UPDATE  X' = a X + B X        rows of B against COLUMNS of X (transposing LDS reads)
//   FINAL   the last UPDATE: into the caller's matrix as bf16
// Operands go global -> LDS by DMA in a ring of stages of 32 along the contraction; with SPLIT a stage holds the hi and lo
// parts of both and feeds three products (hi hi, hi lo, lo hi): 3 products for 2 loads.  The path from L2 to the CUs
// bounds these products (about 10 TB/s: T operations a byte), hence the large tiles and the shared split stages.
// The two waves of a SIMD work in opposite phases, a barrier apart: one reads its fragments from LDS while the other
// multiplies.  Waves 4..7 (B) run one phase behind waves 0..3 (A); stage s is read in phases 2s (A) and 2s + 1 (B), its
// slot is refilled from phase 2s + 2 on.
enum { GRAM, POLY, UPDATE, FINAL };
template <int T, bool SPLIT> struct Cfg {
    static constexpr int MI = T / 32, NI = T / 64;                  // fragments of 16 x 16 a wave
    static constexpr int OPB = T * BK * 2, STAGE = (SPLIT ? 4 : 2) * OPB;
    static constexpr int S = T == 256 ? (SPLIT ? 2 : 4) : T == 192 ? (SPLIT ? 3 : 5) : (SPLIT ? 2 : 4);
    static constexpr int ND = T / 64;                               // DMAs a wave, stage and part (hi / lo)
    static constexpr int SUBM = 16 * MI, SUBN = 16 * NI;            // a wave's part of the tile
    static constexpr int LDT = SUBM + 4, LDN = SUBN + 4;            // rows of its image in LDS (elements), by column / row
    static constexpr int IMG = (LDT * SUBN > LDN * SUBM ? LDT * SUBN : LDN * SUBM) * 2;
    static constexpr int SMEM = S * STAGE > 8 * IMG ? S * STAGE : 8 * IMG;
};
// chunk permutation of a [32 rows][4 chunks] panel: the eight rows (8 apart in two groups of four) that half a wave's
// transposing read touches lie in different banks
DEVI int tkey(int row) { return 2 * ((row >> 3) & 1); }

DEVI unsigned pack2(float a, float b, bool to_bf16) {
    if (to_bf16) {
        const bf16x2 v = {(bf16)a, (bf16)b};
        return __builtin_bit_cast(unsigned, v);
    }
    typedef f16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 v = {(f16)a, (f16)b};
    return __builtin_bit_cast(unsigned, v);
}

template <int MODE, int T, bool SPLIT>
__global__ __launch_bounds__(512, T == 128 ? 4 : 2) void ortho_gemm_kernel(const GemmArgs ga) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef Cfg<T, SPLIT> C;
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    constexpr int S = C::S, MI = C::MI, NI = C::NI, ND = C::ND, NP = SPLIT ? 2 : 1;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave >> 2, wn = wave & 3, i = lane & 15, g = lane >> 4;
    const bool late = wave >= 4;
    const int bid = xcd_remap(blockIdx.x, gridDim.x);
    const Ws& ws = ga.ws;
    const int id = SYM ? ws.map_sym[bid] : ws.map_rect[bid];
    const Mat& q = ws.mats[id];
    const int mp = q.mp, np = q.np;
    const int tm = (mp + T - 1) / T, tn = (np + T - 1) / T;
    int t = bid - (SYM ? q.sym0 : q.rect0);
    const int per = SYM ? tm * (tm + 1) / 2 : tm * tn;
    const int b = t / per;
    t -= b * per;
    int ti, tj;
    if (SYM) {
        ti = 0;
        while (t >= tm - ti) { t -= tm - ti; ++ti; }
        tj = ti + t;
    } else {
        tj = t / tm;                 // the tiles of one column panel follow each other: it stays in L2
        ti = t - tj * tm;
    }
    const int m0 = ti * T, n0 = tj * T;
    const int64_t xo = q.xoff + (int64_t)b * mp * np, ao = q.aoff + (int64_t)b * mp * mp;
    const int total = (MODE == GRAM ? np : mp) / BK;
    const float e1 = ws.exps[q.mat0 + b], e2 = e1 * e1;

    // ---- stages: 32 columns of T rows of P ([row][4 chunks of 16 B]), and of Q either the same or, for UPDATE, 32 rows
    // of T columns (T / 32 panels of [32 rows][4 chunks]).  The operands lie in memory as panels of 32 columns, so every
    // DMA of a wave moves 1 KB in one piece.  Chunks are permuted by a key of the row so that no read meets itself
    // in a bank.  Rows and columns behind the matrix read zeros or neighbours: only their own results, which are not
    // stored, see them.  A wave moves pieces wave, wave + 8, ...: first P's, then Q's.
    __amdgpu_buffer_rsrc_t rsP[NP], rsQ[NP];
#pragma unroll
    for (int h = 0; h < NP; ++h) {
        const f16* P = MODE == GRAM ? ws.x[ga.src][h] + xo : MODE == POLY ? ws.a[h] + ao : ws.b[h] + ao;
        const f16* Q = MODE == POLY ? ws.a[h] + ao : ws.x[ga.src][h] + xo;
        rsP[h] = __builtin_amdgcn_make_buffer_rsrc((void*)P, 0, mp * (MODE == GRAM ? np : mp) * 2, 0x00020000);
        rsQ[h] = __builtin_amdgcn_make_buffer_rsrc((void*)Q, 0, mp * (MODE == POLY ? mp : np) * 2, 0x00020000);
    }
    int vo[ND];
#pragma unroll
    for (int u = 0; u < ND; ++u) {
        const int d = wave + 8 * u;
        const bool isP = d < T / 16;
        const int e = isP ? d : d - T / 16;
        if (isP || SYM) {
            const int r = e * 16 + (lane >> 2);
            vo[u] = r * 64 + (((lane & 3) ^ fsw(r >> 2)) << 4);
        } else {
            const int r = (e & 1) * 16 + (lane >> 2);
            vo[u] = (e >> 1) * mp * 64 + r * 64 + (((lane & 3) ^ tkey(r)) << 4);
        }
    }
    int inext = 0, islot = 0;
    auto issue = [&]() {
        if (inext < total) {
            const int soP = (inext * mp + m0) * 64;
            const int soQ = SYM ? (inext * mp + n0) * 64 : ((n0 >> 5) * mp + inext * 32) * 64;
#pragma unroll
            for (int h = 0; h < NP; ++h)
#pragma unroll
                for (int u = 0; u < ND; ++u) {
                    const int d = wave + 8 * u;
                    const bool isP = d < T / 16;
                    const int at = islot * C::STAGE + h * 2 * C::OPB + d * 1024;
                    __builtin_amdgcn_raw_ptr_buffer_load_lds(isP ? rsP[h] : rsQ[h], (lptr_t)(smem + at), 16, vo[u],
                                                             isP ? soP : soQ, 0, 0);
                }
        }
        ++inext;
        islot = islot + 1 == S ? 0 : islot + 1;
    };
    auto landed = [&](int s) {       // my DMAs of stage s are done (inext: stages requested)
        const int younger = min(inext, total) - 1 - s;
        if (younger >= S - 1) wait_vmcnt<NP * ND * (S - 1)>();
        else if (S > 2 && younger == S - 2) wait_vmcnt<NP * ND * (S - 2)>();
        else if (S > 3 && younger == S - 3) wait_vmcnt<NP * ND * (S - 3)>();
        else wait_vmcnt<0>();
    };

    f32x4 acc[MI][NI];
#pragma unroll
    for (int a = 0; a < MI; ++a)
#pragma unroll
        for (int c = 0; c < NI; ++c) acc[a][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int rp = wm * C::SUBM + i, offP = rp * 64 + ((g ^ fsw(rp >> 2)) << 4);
    const int rq = wn * C::SUBN + i, offQ = C::OPB + rq * 64 + ((g ^ fsw(rq >> 2)) << 4);
    int offT[NI];
#pragma unroll
    for (int ni = 0; ni < NI; ++ni) {
        const int row = 8 * g + (i >> 2), col = wn * C::SUBN + ni * 16, ch = (col & 31) / 8 + ((i & 3) >> 1);
        offT[ni] = C::OPB + (col >> 5) * 2048 + row * 64 + ((ch ^ tkey(row)) << 4) + (i & 1) * 8;
    }
    u32x4 fp[NP][MI], fq[NP][NI];
    auto read = [&](const char* st) {
#pragma unroll
        for (int h = 0; h < NP; ++h) {
            const char* sh = st + h * 2 * C::OPB;
#pragma unroll
            for (int x = 0; x < NI; ++x) {
                if (SYM) fq[h][x] = *(const u32x4*)(sh + offQ + x * 1024);
                else {
                    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(sh + offT[x])));
                    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(sh + offT[x] + 256)));
                    fq[h][x] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                }
            }
#pragma unroll
            for (int x = 0; x < MI; ++x) fp[h][x] = *(const u32x4*)(sh + offP + x * 1024);
        }
    };
    auto multiply = [&]() {
        auto mm = [&](int hp, int hq) {
#pragma unroll
            for (int mi = 0; mi < MI; ++mi)
#pragma unroll
                for (int ni = 0; ni < NI; ++ni)
                    acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        __builtin_bit_cast(f16x8, fq[hq][ni]), __builtin_bit_cast(f16x8, fp[hp][mi]), acc[mi][ni], 0, 0, 0);
        };
        if (SPLIT) {
            mm(NP - 1, 0);
            mm(0, NP - 1);
        }
        mm(0, 0);
    };
    auto phase = [&]() {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
    };

    for (int s = 0; s < S - 1; ++s) issue();
    landed(0);
    phase();                                                   // phase 0 begins
    if (late) {
        issue();
        phase();
    }
    int slot = 0;
    for (int s = 0; s < total; ++s) {
        if (!late) issue();                                    // stage s + S - 1, into the slot that s - 1 has left
        read(smem + slot * C::STAGE);
        slot = slot + 1 == S ? 0 : slot + 1;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (late) landed(s + 1);
        phase();
        if (late) issue();
        multiply();
        if (!late) landed(s + 1);
        if (!late || s + 1 < total) phase();
    }

    // ---- epilogue.  Lane (i, g) holds columns 16 ni + 4 g + r of row 16 mi + i of its wave's part.
    // The matrix's own exponent: products of two (A) or three (B X) stored operands carry 2^2e too much.
    const float c1 = MODE == GRAM ? ga.c1 : MODE == FINAL ? ga.c1 * e2 * e1 : ga.c1 * e2;
    const float c0 = MODE == FINAL ? ga.c0 * e1 : ga.c0;
    const int wm0 = m0 + wm * C::SUBM, wn0 = n0 + wn * C::SUBN;
    const int nend = SYM ? mp : np;
#pragma unroll
    for (int mi = 0; mi < MI; ++mi) {
        const int m = wm0 + mi * 16 + i;
#pragma unroll
        for (int ni = 0; ni < NI; ++ni) {
            const int n = wn0 + 16 * ni + 4 * g;
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[mi][ni][r] *= c1;
            if (MODE != GRAM && m < mp && n < nend) {
                const int64_t at = (MODE == POLY ? ao : xo) + ((int64_t)(n >> 5) * mp + m) * 32 + (n & 31);
                const f16* eh = MODE == POLY ? ws.a[0] : ws.x[ga.src][0];
                const f16* el = MODE == POLY ? ws.a[1] : ws.x[ga.src][1];
                const f16x4 h = *(const f16x4*)(eh + at);
                f16x4 l{};
                if (SPLIT) l = *(const f16x4*)(el + at);
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[mi][ni][r] = fmaf(c0, (float)h[r] + (float)l[r], acc[mi][ni][r]);
            }
        }
    }
    // fp16 results go to panels: 32 bytes of 16 rows a store
    auto put = [&](f16* dst) {
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
            const int m = wm0 + mi * 16 + i;
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                const int n = wn0 + 16 * ni + 4 * g;
                const f32x4 v = acc[mi][ni];
                if (m < mp && n < nend)
                    *(u32x2*)(dst + ((int64_t)(n >> 5) * mp + m) * 32 + (n & 31)) = u32x2{pack2(v[0], v[1], false), pack2(v[2], v[3], false)};
            }
        }
    };
    // ... mirrored ones, and the caller's bf16, through an image of the wave's part in LDS (all stages are done with; a
    // wave reads only what it wrote), by rows or by columns, so that every store covers rows of the destination.
    char* img = smem + wave * C::IMG;
    constexpr bool TOBF = MODE == FINAL;
    auto emit = [&](auto by_col_c, void* dst, int64_t ld, int rows, int cols, bool aligned) {
        constexpr bool COL = decltype(by_col_c)::value;       // destination rows are columns of the tile
        constexpr int LDI = COL ? C::LDT : C::LDN;            // elements a row of the image
        constexpr int NR = COL ? C::SUBN : C::SUBM, NC = COL ? C::SUBM : C::SUBN;
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < NI; ++ni) {
                const f32x4 v = acc[mi][ni];
                if (!COL) {
                    const u32x2 w = {pack2(v[0], v[1], TOBF), pack2(v[2], v[3], TOBF)};
                    *(u32x2*)(img + ((mi * 16 + i) * LDI + ni * 16 + 4 * g) * 2) = w;
                } else {
                    // lanes i and i ^ 1 (rows m, m + 1) trade: the even one gets columns r = 0, 1 of both, the odd one 2, 3
                    const bool odd = i & 1;
                    const float x0 = dpp_mov<0xB1>(odd ? v[0] : v[2]), x1 = dpp_mov<0xB1>(odd ? v[1] : v[3]);
                    const int c = ni * 16 + 4 * g + (odd ? 2 : 0), m = mi * 16 + (i & ~1);
                    *(unsigned*)(img + (c * LDI + m) * 2) = odd ? pack2(x0, v[2], TOBF) : pack2(v[0], x0, TOBF);
                    *(unsigned*)(img + ((c + 1) * LDI + m) * 2) = odd ? pack2(x1, v[3], TOBF) : pack2(v[1], x1, TOBF);
                }
            }
        const int r0 = COL ? wn0 : wm0, q0 = COL ? wm0 : wn0;  // destination of the image's origin
        constexpr int LPR = NC / 4;                            // lanes a row, four elements each
        for (int e = lane; e < NR * LPR; e += 64) {
            int r = e / LPR, c = (e - r * LPR) * 4;
            if (!TOBF) {                                       // panels: 64 bytes of one row after the other
                const int pan = e / (8 * NR), f = e - pan * (8 * NR);
                r = f >> 3;
                c = pan * 32 + (f & 7) * 4;
            }
            const u32x2 w = *(const u32x2*)(img + (r * LDI + c) * 2);
            const int dr = r0 + r, dc = q0 + c;
            if (dr >= rows || dc >= cols) continue;
            uint16_t* o = (uint16_t*)dst + (TOBF ? dr * ld + dc : ((int64_t)(dc >> 5) * ld + dr) * 32 + (dc & 31));
            if (aligned && dc + 4 <= cols) *(u32x2*)o = w;
            else {
                const unsigned x[4] = {w[0] & 0xffffu, w[0] >> 16, w[1] & 0xffffu, w[1] >> 16};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (dc + k < cols) o[k] = (uint16_t)x[k];
            }
        }
    };
    auto take_hi = [&]() {           // what the fp16 of the image has left of the values
#pragma unroll
        for (int mi = 0; mi < MI; ++mi)
#pragma unroll
            for (int ni = 0; ni < NI; ++ni)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[mi][ni][r] -= (float)(f16)acc[mi][ni][r];
    };
    if (SYM) {
        f16* const* o = MODE == GRAM ? ws.a : ws.b;
        put(o[0] + ao);
        if (ti != tj) emit(std::true_type{}, o[0] + ao, mp, mp, mp, true);
        if (SPLIT) {
            take_hi();
            put(o[1] + ao);
            if (ti != tj) emit(std::true_type{}, o[1] + ao, mp, mp, mp, true);
        }
    } else if (MODE == UPDATE) {
        put(ws.x[ga.src ^ 1][0] + xo);
        if (SPLIT && ga.split_next) {
            take_hi();
            put(ws.x[ga.src ^ 1][1] + xo);
        }
    } else {
        bf16* out = (bf16*)q.out + b * q.out_batch;
        const bool al = (((uintptr_t)out | (uint64_t)(q.out_ld * 2)) & 7) == 0;
        if (q.tall) emit(std::true_type{}, out, q.out_ld, q.n, q.m, al);
        else emit(std::false_type{}, out, q.out_ld, q.m, q.n, al);
    }
#endif
}

// ---- host side ------------------------------------------------------------------------------------------------
int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

struct Layout {
    int64_t bytes, mats, maps[3], parts, exps, x, a;      // byte offsets; x / a: first region, xbytes / abytes apart
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
        q.mp = (int)up(q.m, 32);
        q.np = (int)up(q.n, 32);
        if ((int64_t)q.mp * q.np * 2 >= (1ll << 31)) return DINO_ERR_TOO_LARGE;
        int64_t p = ((int64_t)q.m * q.n + 16383) / 16384;
        if (p > 256) p = 256;
        q.parts = (int)(p > q.rows ? q.rows : p);
        q.part0 = (int)parts; q.mat0 = (int)nmat; q.xoff = xo; q.aoff = ao; q.prep0 = (int)prep;
        parts += (int64_t)s.batch * q.parts;
        nmat += s.batch;
        xo += (int64_t)s.batch * q.mp * q.np;
        ao += (int64_t)s.batch * q.mp * q.mp;
        prep += (int64_t)s.batch * ((q.mp + 63) / 64) * ((q.np + 63) / 64);
        if (prep >= (1 << 24) || parts >= (1 << 24)) return DINO_ERR_TOO_LARGE;    // 256 threads each, < 2^32 a launch
        if (out) out[i] = q;
    }
    // Tile size of the symmetric products and of the update, each the one of least estimated time: rounds of tiles over
    // the CUs, a tile costing its area over the rate that the path from L2 allows (T operations a byte, and no
    // more than about two thirds of the matrix pipes).
    for (int kind = 0; kind < 2; ++kind) {
        double best = 0;
        const int sizes[3] = {256, 192, 128};
        for (int z = 0; z < 3; ++z) {
            const int T = sizes[z];
            double work = 0, tiles = 0;
            for (int i = 0; i < count; ++i) {
                int64_t m = up(items[i].rows < items[i].cols ? items[i].rows : items[i].cols, 32);
                int64_t n = up(items[i].rows < items[i].cols ? items[i].cols : items[i].rows, 32);
                const double tm = (double)((m + T - 1) / T), tn = (double)((n + T - 1) / T);
                const double k = kind ? tm * tn * items[i].batch : tm * (tm + 1) / 2 * items[i].batch;
                tiles += k;
                work += k * (double)(kind ? m : n + m);
            }
            if (tiles == 0) tiles = 1;
            const double cost = work / tiles * ceil(tiles / (T == 128 ? 512.0 : 256.0)) * T * T / (T == 256 ? 1.0 : T == 192 ? 0.8 : 0.35);
            if (z == 0 || cost < best) { best = cost; L.tile[kind] = T; }
        }
        static const char* force[2] = {getenv("OT_SYM"), getenv("OT_RECT")};
        if (force[kind]) L.tile[kind] = atoi(force[kind]);
    }
    for (int i = 0; i < count; ++i) {
        int64_t m = up(items[i].rows < items[i].cols ? items[i].rows : items[i].cols, 32);
        int64_t n = up(items[i].rows < items[i].cols ? items[i].cols : items[i].rows, 32);
        const int64_t ts = (m + L.tile[0] - 1) / L.tile[0], tm = (m + L.tile[1] - 1) / L.tile[1], tn = (n + L.tile[1] - 1) / L.tile[1];
        const int64_t ns = items[i].batch * (ts * (ts + 1) / 2), nr = items[i].batch * tm * tn;
        if (out) {
            out[i].sym0 = (int)sym; out[i].rect0 = (int)rect;
            out[i].nsym = (int)ns; out[i].nrect = (int)nr;
        }
        sym += ns;
        rect += nr;
    }
    int64_t at = 0;
    auto take = [&](int64_t bytes) { const int64_t r = at; at = up(at + bytes, 256); return r; };
    L.ntile[0] = sym; L.ntile[1] = rect; L.ntile[2] = prep;
    L.mats = take((int64_t)sizeof(Mat) * count);
    for (int k = 0; k < 3; ++k) L.maps[k] = take(4 * L.ntile[k]);
    L.parts = take(8 * parts);
    L.exps = take(4 * nmat);
    L.xbytes = up(2 * xo, 256);
    L.abytes = up(2 * ao, 256);
    L.x = take(4 * L.xbytes);
    L.a = take(4 * L.abytes);
    L.bytes = at;
    return DINO_OK;
}

// largest |p(x)| and |b x^2 + c x^4| over singular values up to `top`
void poly_bounds(const float* c, double top, double& px, double& qx) {
    px = qx = 0;
    for (int k = 0; k <= 512; ++k) {
        const double x = top * k / 512, x2 = x * x, q = c[1] * x2 + c[2] * x2 * x2;
        px = fmax(px, fabs((c[0] + q) * x));
        qx = fmax(qx, fabs(q));
    }
}

template <int MODE, int T, bool SPLIT> int launch_as(const GemmArgs& ga, int64_t grid, hipStream_t st) {
    constexpr int smem = Cfg<T, SPLIT>::SMEM;
    static const hipError_t set = hipFuncSetAttribute((const void*)ortho_gemm_kernel<MODE, T, SPLIT>,
                                                      hipFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (set != hipSuccess) return (int)set;
    hipLaunchKernelGGL((ortho_gemm_kernel<MODE, T, SPLIT>), dim3((unsigned)grid), dim3(512), smem, st, ga);
    return dino_launch_status();
}
template <int MODE> int launch_gemm(const GemmArgs& ga, int T, bool split, int64_t grid, hipStream_t st) {
    if (T == 256) return split ? launch_as<MODE, 256, true>(ga, grid, st) : launch_as<MODE, 256, false>(ga, grid, st);
    if (T == 192) return split ? launch_as<MODE, 192, true>(ga, grid, st) : launch_as<MODE, 192, false>(ga, grid, st);
    return split ? launch_as<MODE, 128, true>(ga, grid, st) : launch_as<MODE, 128, false>(ga, grid, st);
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
    ws.map_sym = (int*)(w + L.maps[0]);
    ws.map_rect = (int*)(w + L.maps[1]);
    ws.map_prep = (int*)(w + L.maps[2]);
    ws.parts = (double*)(w + L.parts);
    ws.exps = (float*)(w + L.exps);
    for (int k = 0; k < 2; ++k)
        for (int h = 0; h < 2; ++h) ws.x[k][h] = (f16*)(w + L.x + (2 * k + h) * L.xbytes);
    for (int h = 0; h < 2; ++h) {
        ws.a[h] = (f16*)(w + L.a + h * L.abytes);
        ws.b[h] = (f16*)(w + L.a + (2 + h) * L.abytes);
    }
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
        GemmArgs ga{ws, s & 1, split(s + 1), 0.f, (float)(sa[s] / ((double)SX * SX))};
        rc = launch_gemm<GRAM>(ga, L.tile[0], split(s), L.ntile[0], st);
        if (rc != DINO_OK) break;
        ga.c0 = (float)(c[1] * sb[s] / sa[s]);
        ga.c1 = (float)(c[2] * sb[s] / (sa[s] * sa[s]));
        rc = launch_gemm<POLY>(ga, L.tile[0], split(s), L.ntile[0], st);
        if (rc != DINO_OK) break;
        const double o = s + 1 == steps ? 1.0 / SX : 1.0;
        ga.c0 = (float)(c[0] * o);
        ga.c1 = (float)(o / sb[s]);
        rc = s + 1 == steps ? launch_gemm<FINAL>(ga, L.tile[1], split(s), L.ntile[1], st)
                            : launch_gemm<UPDATE>(ga, L.tile[1], split(s), L.ntile[1], st);
    }
    return rc;
}
