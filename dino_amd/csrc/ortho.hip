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

#include "common.h"

namespace {

typedef _Float16 f16;
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) void* lptr_t;

constexpr int TILE = 128, BK = 32, S = 4, NTHR = 256;
constexpr int OPB = TILE * BK * 2;              // bytes of one operand's stage
constexpr int STAGE = 2 * OPB;                  // 16 KB
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
    int tm, tn, sym0, rect0, prep0, ntiles_sym; // tiles of 128; first global tile of each kind
};
struct Setup {
    Mat it[ITEMS];
    int wg0[ITEMS + 1];                         // first workgroup of each item
    int count, first;                           // items here, index of the first
};
struct Ws {                                     // regions of the workspace
    Mat* mats;
    int *map_sym, *map_rect, *map_prep;         // tile -> item
    double* parts;
    float* exps;                                // per matrix: 2^-e
    f16 *x[2][2], *a[2], *b[2];                 // [buffer][hi / lo]
};

DEVI void split_store(f16* hi, f16* lo, const float (&v)[4]) {
    f16x4 h, l;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        h[r] = (f16)v[r];
        l[r] = (f16)(v[r] - (float)h[r]);
    }
    *(f16x4*)hi = h;
    if (lo) *(f16x4*)lo = l;
}

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

template <typename T> DEVI double row_range_sq(const T* p, int64_t ld, int cols, int64_t e0, int64_t e1) {
    double s = 0;
    for (int64_t e = e0 + threadIdx.x; e < e1; e += NTHR) {
        const int64_t r = e / cols;
        const double x = (double)to_f32<T>(p[r * ld + (e - r * cols)]);
        s += x * x;
    }
    return s;
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
    for (int t = t0; t < q.batch * q.ntiles_sym; t += ts) ws.map_sym[q.sym0 + t] = id;
    for (int t = t0; t < q.batch * q.tm * q.tn; t += ts) ws.map_rect[q.rect0 + t] = id;
    const int np_ = q.batch * ((q.mp + 63) / 64) * ((q.np + 63) / 64);
    for (int t = t0; t < np_; t += ts) ws.map_prep[q.prep0 + t] = id;
    const int b = w / q.parts, part = w - b * q.parts;
    const int64_t n = (int64_t)q.rows * q.cols, per = (n + q.parts - 1) / q.parts;
    const int64_t e0 = part * per, e1 = e0 + per < n ? e0 + per : n;
    const double s = q.dtype == DINO_F32
                         ? row_range_sq<float>((const float*)q.in + b * q.in_batch, q.in_ld, q.cols, e0, e1)
                         : row_range_sq<bf16>((const bf16*)q.in + b * q.in_batch, q.in_ld, q.cols, e0, e1);
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
        const int64_t at = (int64_t)(m0 + r) * q.np + n0 + c;
        const f16 h = (f16)v;
        xh[at] = h;
        if (lo) xl[at] = (f16)(v - (float)h);
    }
}

struct GemmArgs {
    Ws ws;
    int src, split, split_next;      // X buffer read, operands are pairs, the next step's operands are pairs
    float c0, c1;                    // epilogue: c0 * (elementwise operand) + c1 * product
};

DEVI int fsw(int x) { return (4 - (x & 3)) & 3; }
DEVI int tkey(int row) { return 2 * ((row & 3) | (((row >> 3) & 1) << 2)); }
template <int N> DEVI void wait_vmcnt() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// 128 x 128 tile of a product per workgroup (2 x 2 waves of 64 x 64).
//   GRAM    A = X X^T             rows of X against rows of X; tiles on and above the diagonal, written twice
//   POLY    B = b A + c A A       A symmetric: rows against rows again
//   UPDATE  X' = a X + B X        rows of B against COLUMNS of X (transposing LDS reads)
//   FINAL   the last UPDATE: into the caller's matrix as bf16
// Operands go global -> LDS by DMA in a ring of S stages of 32 along the contraction; split operands are three passes
// (hi hi, hi lo, lo hi) of one stream of stages.
enum { GRAM, POLY, UPDATE, FINAL };
template <int MODE> __global__ __launch_bounds__(NTHR, 2) void ortho_gemm_kernel(const GemmArgs ga) {
#if defined(__HIP_DEVICE_COMPILE__)
    constexpr bool SYM = MODE == GRAM || MODE == POLY;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = wave >> 1, wn = wave & 1, i = lane & 15, g = lane >> 4;
    const int bid = xcd_remap(blockIdx.x, gridDim.x);
    const Ws& ws = ga.ws;
    const int id = SYM ? ws.map_sym[bid] : ws.map_rect[bid];
    const Mat& q = ws.mats[id];
    const int mp = q.mp, np = q.np;
    int t = bid - (SYM ? q.sym0 : q.rect0);
    const int per = SYM ? q.ntiles_sym : q.tm * q.tn;
    const int b = t / per;
    t -= b * per;
    int ti, tj;
    if (SYM) {
        ti = 0;
        while (t >= q.tm - ti) { t -= q.tm - ti; ++ti; }
        tj = ti + t;
    } else {
        tj = t / q.tm;               // the tiles of one column panel follow each other: it stays in L2
        ti = t - tj * q.tm;
    }
    const int m0 = ti * TILE, n0 = tj * TILE;
    const int64_t xo = q.xoff + (int64_t)b * mp * np, ao = q.aoff + (int64_t)b * mp * mp;
    const int ldp = MODE == GRAM ? np : mp, ldq = MODE == GRAM ? np : MODE == POLY ? mp : np;
    const int K = MODE == GRAM ? np : mp;
    const f16* P[2];
    const f16* Q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        P[h] = MODE == GRAM ? ws.x[ga.src][h] + xo : MODE == POLY ? ws.a[h] + ao : ws.b[h] + ao;
        Q[h] = MODE == POLY ? ws.a[h] + ao : ws.x[ga.src][h] + xo;
    }
    const int pbytes = mp * ldp * 2, qbytes = mp * ldq * 2;

    // ---- stages: 32 columns of 128 rows of P ([row][4 chunks of 16 B]), and of Q either the same or, for UPDATE, 32 rows
    // of 128 columns ([k][16 chunks]); chunks are permuted by a key of the row so that neither kind of read meets
    // itself in a bank.  Rows and columns behind the matrix read zeros or neighbours: only their own results, which
    // are not stored, see them.
    const int wv = __builtin_amdgcn_readfirstlane(wave);
    int voP[2], voQ[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const int L = tid + NTHR * u;
        const int r = L >> 2, c = L & 3;
        voP[u] = (r * ldp + ((c ^ fsw(r >> 2)) << 3)) * 2;
        if (SYM) voQ[u] = (r * ldq + ((c ^ fsw(r >> 4)) << 3)) * 2;
        else {
            const int kr = L >> 4, kc = L & 15;
            voQ[u] = (kr * ldq + ((kc ^ tkey(kr)) << 3)) * 2;
        }
    }
    const int nk = K / BK, nseg = ga.split ? 3 : 1, total = nk * nseg;
    int iseg = 0, ik = 0, islot = 0;
    __amdgpu_buffer_rsrc_t rsP = __builtin_amdgcn_make_buffer_rsrc((void*)P[0], 0, pbytes, 0x00020000);
    __amdgpu_buffer_rsrc_t rsQ = __builtin_amdgcn_make_buffer_rsrc((void*)Q[0], 0, qbytes, 0x00020000);
    auto issue = [&]() {
        const int sa = islot * STAGE + wv * 1024;
        const int k = ik * BK;
        const int soP = (m0 * ldp + k) * 2;
        const int soQ = SYM ? (n0 * ldq + k) * 2 : (k * ldq + n0) * 2;
#pragma unroll
        for (int u = 0; u < 2; ++u)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsP, (lptr_t)(smem + sa + u * 4096), 16, voP[u], soP, 0, 0);
#pragma unroll
        for (int u = 0; u < 2; ++u)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsQ, (lptr_t)(smem + sa + OPB + u * 4096), 16, voQ[u], soQ, 0, 0);
        islot = islot + 1 == S ? 0 : islot + 1;
        if (++ik == nk) {
            ik = 0;
            ++iseg;                                   // 0: hi hi, 1: hi lo, 2: lo hi
            rsP = __builtin_amdgcn_make_buffer_rsrc((void*)P[iseg == 2], 0, pbytes, 0x00020000);
            rsQ = __builtin_amdgcn_make_buffer_rsrc((void*)Q[iseg == 1], 0, qbytes, 0x00020000);
        }
    };
    int issued = 0;
#pragma unroll
    for (int s = 0; s < S - 1; ++s)
        if (issued < total) { issue(); ++issued; }

    f32x4 acc[4][4];
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[a][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int ra0 = wm * 64 + i, rb0 = wn * 64 + 16 * (i >> 2) + (i & 3);
    const int offP = ra0 * 64 + ((g ^ fsw(ra0 >> 2)) << 4);
    const int offQ = OPB + rb0 * 64 + ((g ^ fsw(rb0 >> 4)) << 4);
    int offT[4];
#pragma unroll
    for (int ni = 0; ni < 4; ++ni) {
        const int row = 8 * g + (i >> 2), ch = (wn * 64 + ni * 16) / 8 + ((i & 3) >> 1);
        offT[ni] = OPB + row * 256 + ((ch ^ tkey(row)) << 4) + (i & 1) * 8;
    }

    int cslot = 0;
    for (int s = 0; s < total; ++s) {
        if (total - 1 - s >= S - 2) wait_vmcnt<4 * (S - 2)>();
        else wait_vmcnt<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (issued < total) { issue(); ++issued; }
        const char* st = smem + cslot * STAGE;
        u32x4 fp[4], fq[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            if (SYM) fq[x] = *(const u32x4*)(st + offQ + x * 256);
            else {
                const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + offT[x])));
                const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(st + offT[x] + 1024)));
                fq[x] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) fp[x] = *(const u32x4*)(st + offP + x * 1024);
#pragma unroll
        for (int mi = 0; mi < 4; ++mi)
#pragma unroll
            for (int ni = 0; ni < 4; ++ni)
                acc[mi][ni] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, fq[ni]),
                                                                     __builtin_bit_cast(f16x8, fp[mi]), acc[mi][ni], 0, 0, 0);
        cslot = cslot + 1 == S ? 0 : cslot + 1;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // before a wave may refill this slot
    }

    // the matrix's own exponent: products of two (A) or three (B X) stored operands carry 2^2e too much
    const float e1 = ws.exps[q.mat0 + b], e2 = e1 * e1;
    const float c1 = MODE == GRAM ? ga.c1 : MODE == FINAL ? ga.c1 * e2 * e1 : ga.c1 * e2;
    const float c0 = MODE == FINAL ? ga.c0 * e1 : ga.c0;
    // ---- epilogue: lane holds four consecutive columns of row m per fragment
#pragma unroll
    for (int mi = 0; mi < 4; ++mi) {
        const int m = m0 + wm * 64 + mi * 16 + i;
        if (m >= mp) continue;
#pragma unroll
        for (int ni = 0; ni < 4; ++ni) {
            const int n = n0 + wn * 64 + (SYM ? 16 * g + 4 * ni : 16 * ni + 4 * g);
            if (n >= (SYM ? mp : np)) continue;
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = c1 * acc[mi][ni][r];
            if (MODE != GRAM) {
                const int64_t at = MODE == POLY ? ao + (int64_t)m * mp + n : xo + (int64_t)m * np + n;
                const f16* eh = MODE == POLY ? ws.a[0] : ws.x[ga.src][0];
                const f16* el = MODE == POLY ? ws.a[1] : ws.x[ga.src][1];
                const f16x4 h = *(const f16x4*)(eh + at);
                f16x4 l{};
                if (ga.split) l = *(const f16x4*)(el + at);
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = fmaf(c0, (float)h[r] + (float)l[r], v[r]);
            }
            if (SYM) {
                f16* oh = (MODE == GRAM ? ws.a[0] : ws.b[0]) + ao;
                f16* ol = (MODE == GRAM ? ws.a[1] : ws.b[1]) + ao;
                split_store(oh + (int64_t)m * mp + n, ga.split ? ol + (int64_t)m * mp + n : nullptr, v);
                if (ti != tj) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const f16 h = (f16)v[r];
                        oh[(int64_t)(n + r) * mp + m] = h;
                        if (ga.split) ol[(int64_t)(n + r) * mp + m] = (f16)(v[r] - (float)h);
                    }
                }
            } else if (MODE == UPDATE) {
                const int64_t at = xo + (int64_t)m * np + n;
                split_store(ws.x[ga.src ^ 1][0] + at, ga.split_next ? ws.x[ga.src ^ 1][1] + at : nullptr, v);
            } else {
                if (m >= q.m) continue;
                bf16* out = (bf16*)q.out + b * q.out_batch;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (n + r < q.n) out[q.tall ? (int64_t)(n + r) * q.out_ld + m : (int64_t)m * q.out_ld + n + r] = (bf16)v[r];
            }
        }
    }
#endif
}

// ---- host side ------------------------------------------------------------------------------------------------
int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

struct Layout {
    int64_t bytes, mats, maps[3], parts, exps, x, a;      // byte offsets; x / a: first region, xbytes / abytes apart
    int64_t xbytes, abytes, ntile[3];
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
        q.tm = (q.mp + TILE - 1) / TILE;
        q.tn = (q.np + TILE - 1) / TILE;
        q.ntiles_sym = q.tm * (q.tm + 1) / 2;
        int64_t p = ((int64_t)q.m * q.n + 16383) / 16384;
        q.parts = (int)(p > 256 ? 256 : p);
        q.part0 = (int)parts; q.mat0 = (int)nmat; q.xoff = xo; q.aoff = ao; q.sym0 = (int)sym; q.rect0 = (int)rect; q.prep0 = (int)prep;
        parts += (int64_t)s.batch * q.parts;
        nmat += s.batch;
        xo += (int64_t)s.batch * q.mp * q.np;
        ao += (int64_t)s.batch * q.mp * q.mp;
        sym += (int64_t)s.batch * q.ntiles_sym;
        rect += (int64_t)s.batch * q.tm * q.tn;
        prep += (int64_t)s.batch * ((q.mp + 63) / 64) * ((q.np + 63) / 64);
        if (prep >= (1 << 24) || parts >= (1 << 24)) return DINO_ERR_TOO_LARGE;    // 256 threads each, < 2^32 a launch
        if (out) out[i] = q;
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

template <int MODE> int launch_gemm(const GemmArgs& ga, int64_t grid, hipStream_t st) {
    constexpr int smem = S * STAGE;
    hipLaunchKernelGGL((ortho_gemm_kernel<MODE>), dim3((unsigned)grid), dim3(NTHR), smem, st, ga);
    return dino_launch_status();
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
        GemmArgs ga{ws, s & 1, split(s), split(s + 1), 0.f, (float)(sa[s] / ((double)SX * SX))};
        rc = launch_gemm<GRAM>(ga, L.ntile[0], st);
        if (rc != DINO_OK) break;
        ga.c0 = (float)(c[1] * sb[s] / sa[s]);
        ga.c1 = (float)(c[2] * sb[s] / (sa[s] * sa[s]));
        rc = launch_gemm<POLY>(ga, L.ntile[0], st);
        if (rc != DINO_OK) break;
        const double o = s + 1 == steps ? 1.0 / SX : 1.0;
        ga.c0 = (float)(c[0] * o);
        ga.c1 = (float)(o / sb[s]);
        rc = s + 1 == steps ? launch_gemm<FINAL>(ga, L.ntile[1], st) : launch_gemm<UPDATE>(ga, L.ntile[1], st);
    }
    return rc;
}
