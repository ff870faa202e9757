// Log probabilities of given prototypes, entropy and the best prototypes of rows of logits, and their gradient.
//
// With d = x - c (c: the centre, or 0), tau the temperature and md = max_k d_k of a row:
//   zs_k = (d_k - md) / tau,  s = sum e^zs,  t = sum zs e^zs
//   log p_k = zs_k - log s,   H = -sum p log p = log s - t / s
// Everything is taken relative to md BEFORE the division by tau: neither a masked logit of the type's lowest value nor
// a small tau can overflow, and log p has no cancellation of two large numbers (m / tau against its log-sum-exp).
// Rows that are all -inf: log p = -inf, H = 0, gradient 0.  NaN or +inf in a row: NaN for the row's results.
// Best prototypes are ordered by d, equal ones by their index, NaN first; the order uses 64-bit keys
// (order-preserving bits of d, ~index), so there are no ties left and the result does not depend on the schedule.
#include "common.h"

namespace {

typedef bf16 bf16x8u __attribute__((ext_vector_type(8), aligned(2)));   // rows may start at any element
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr float NEG_INF = -__builtin_inff();
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float Z_MIN = -300.f;  // e^Z_MIN and 2^Z_MIN are 0 in fp32: 0 * (-inf) becomes 0 * Z_MIN
constexpr int CAP = 256;        // candidates a chunk can hold for its best k before it falls back to k rounds
constexpr int MAX_K = 64, MAX_CHUNKS = 64;
constexpr int CHUNK_MAX = 16384;

template <typename T> DEVI void load8u(const T* p, float (&v)[8]);
template <> DEVI void load8u<float>(const float* p, float (&v)[8]) {
    const f32x4u a = *(const f32x4u*)p, b = *(const f32x4u*)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
}
template <> DEVI void load8u<bf16>(const bf16* p, float (&v)[8]) {
    const bf16x8u a = *(const bf16x8u*)p;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
}
template <typename T> DEVI void store8u(T* p, const float (&v)[8]);
template <> DEVI void store8u<float>(float* p, const float (&v)[8]) {
    f32x4u a, b;
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = v[i]; b[i] = v[4 + i]; }
    *(f32x4u*)p = a;
    *(f32x4u*)(p + 4) = b;
}
template <> DEVI void store8u<bf16>(bf16* p, const float (&v)[8]) {
    bf16x8u a;
#pragma unroll
    for (int i = 0; i < 8; ++i) a[i] = (bf16)v[i];
    *(bf16x8u*)p = a;
}

// eight elements as loaded: kept packed while they are in flight
template <typename T> struct Raw8;
template <> struct Raw8<bf16> {
    bf16x8u v;
    DEVI void load(const bf16* p) { v = *(const bf16x8u*)p; }
    DEVI float at(int i) const { return (float)v[i]; }
};
template <> struct Raw8<float> {
    f32x4u lo, hi;
    DEVI void load(const float* p) { lo = *(const f32x4u*)p; hi = *(const f32x4u*)(p + 4); }
    DEVI float at(int i) const { return i < 4 ? lo[i & 3] : hi[i & 3]; }
};

// order-preserving bits: a < b  <=>  ord(a) < ord(b); -0 counts as +0, every NaN above +inf
DEVI unsigned ord_bits(float d) {
    const unsigned b = __builtin_bit_cast(unsigned, d + 0.f);
    if (d != d) return 0xFFC00000u;
    return b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
}
DEVI float ord_float(unsigned o) {
    return __builtin_bit_cast(float, (o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}
typedef unsigned long long u64;
DEVI u64 make_key(float d, int idx) { return ((u64)ord_bits(d) << 32) | (unsigned)~idx; }
DEVI u64 wave_max_u64(u64 v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned hi = __shfl_xor((unsigned)(v >> 32), o, 64), lo = __shfl_xor((unsigned)v, o, 64);
        const u64 w = ((u64)hi << 32) | lo;
        v = w > v ? w : v;
    }
    return v;
}

struct Part {        // one chunk of one row; `keys` (topk of them, best first) follow in their own array
    float m, s, t, pad;
};

struct FwdArgs {
    const void* x;
    int64_t ld, rows;
    int K, S, chunk, T, topk;
    const float* center;
    float inv_temp;
    const int64_t* targets;
    float* log_prob;
    float* entropy;
    float* stats;
    float* top_lp;
    int64_t* top_idx;
    Part* parts;
    u64* keys;
};

// log p of one value of d under a row's (md, log s)
DEVI float log_p(float d, float md, float logs, float inv_temp) {
    if (md == NEG_INF && logs == NEG_INF) return NEG_INF;      // nothing in the row
    return (d - md) * inv_temp - logs;
}

// writes the results of a finished row; called by one whole wave
template <typename T> DEVI void finish_row(const FwdArgs& a, int64_t row, float md, float s, float t2, int lane) {
    const float logs = logf(s);
    if (lane == 0) {
        const bool none = md == NEG_INF && s == 0.f;
        a.entropy[row] = none ? 0.f : logs - t2 * LN2 / s;
        a.stats[2 * row] = md;
        a.stats[2 * row + 1] = logs;
    }
    const T* x = (const T*)a.x + row * a.ld;
    for (int j = lane; j < a.T; j += 64) {
        const int64_t at = a.targets[row * a.T + j];
        float v = 0.f;
        if (at >= 0 && at < a.K) {
            const float d = to_f32<T>(x[at]) - (a.center ? a.center[at] : 0.f);
            v = log_p(d, md, logs, a.inv_temp);
        } else if (at != -1) v = __builtin_nanf("");
        a.log_prob[row * a.T + j] = v;
    }
}
DEVI void put_top(const FwdArgs& a, int64_t row, int j, u64 key, float md, float s) {
    a.top_idx[row * a.topk + j] = (int64_t)(int)~(unsigned)key;
    a.top_lp[row * a.topk + j] = log_p(ord_float((unsigned)(key >> 32)), md, logf(s), a.inv_temp);
}

// One workgroup of NT threads takes one chunk (at most NT * 8 * NV columns) of one row, held in registers: read
// once, then the maximum, the sums and the best k come from registers.
// Bound: memory, with about 12 vector instructions and an exp2 an element close behind (50 us of the 85 below).  MI355X:
// 2560 rows of 65536 bf16 (336 MB) 59 us one call after another = 5.7 TB/s, 80 .. 86 beside the gradient's writes; with a centre,
// read from L2 by every workgroup, 91.  Best prototypes: one 3 us more, eight 24 (their lower bound and the list of candidates are
// 200 instructions a wave).  512 rows with a centre and 8 best 22 us + the join; 12608 of 4096 with 2 best (103 MB) 25 us =
// 4.1 TB/s; 333 fp32 rows of 8191, a third of them -inf, 9.7 us.
// Splitting a row over workgroups of 256 threads leaves 32 values a thread in registers, five waves a SIMD or more.
template <typename T, int NT, int NV, bool CEN>
__global__ __launch_bounds__(NT) void logprob_fwd_kernel(const FwdArgs a) {
    constexpr int NW = NT / 64;
    __shared__ float red[3 * NW];
    __shared__ u64 cand[CAP];
    __shared__ u64 best[MAX_K];
    __shared__ u64 rkey[NW];
    __shared__ int ncand;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / a.S;
    const int ch = (int)(blockIdx.x - row * a.S);
    const int c0 = ch * a.chunk, c1 = min(a.K, c0 + a.chunk);
    const T* x = (const T*)a.x + row * a.ld;

    float d[NV][8];
    if (c0 + NT * 8 * NV <= c1) {        // a whole chunk: no column behind the end
        Raw8<T> raw[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) raw[j].load(x + c0 + (j * NT + tid) * 8);
        if (CEN) {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float c[8];
                load8u<float>(a.center + c0 + (j * NT + tid) * 8, c);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[j][i] = raw[j].at(i) - c[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) d[j][i] = raw[j].at(i);
        }
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = c0 + (j * NT + tid) * 8;
            if (at + 8 <= c1) {
                load8u<T>(x + at, d[j]);
                if (CEN) {
                    float c[8];
                    load8u<float>(a.center + at, c);
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[j][i] -= c[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    d[j][i] = at + i < c1 ? to_f32<T>(x[at + i]) - (CEN ? a.center[at + i] : 0.f) : NEG_INF;
            }
        }
    }
    float vm[NV], tm = NEG_INF;                                    // NaNs pass by: they show in the sums
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        vm[j] = d[j][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) vm[j] = fmaxf(vm[j], d[j][i]);
        tm = fmaxf(tm, vm[j]);
    }

    float md = wave_max(tm);
    if (NW > 1) {
        if (lane == 0) red[wave] = md;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) md = fmaxf(md, red[w]);
    }
    // (d - ref) / tau in units of log 2.  One fma an element: z = d sc - fl(ref sc), whose offset against the exact
    // (d - ref) sc is the same dz for every element of the chunk and is taken out of the sums below.  dz is half a step of
    // ref sc: at most 1/4 below 2^22.  Rows further from zero (masked by -1e9 or the type's lowest value throughout) form
    // the difference first.
    const float ref = md == NEG_INF ? 0.f : md, sc = a.inv_temp * LOG2E, off = ref * sc;
    float s = 0.f, t2 = 0.f;
    if (fabsf(off) < 4194304.f) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = fmaf(d[j][i], sc, -off);
                const float e = __builtin_amdgcn_exp2f(z);
                s += e;
                t2 = fmaf(e, fmaxf(z, Z_MIN), t2);                 // e = 0 meets z = -inf
            }
        const float dz = fmaf(ref, sc, -off), f = __builtin_amdgcn_exp2f(-dz);
        t2 = f * fmaf(-dz, s, t2);
        s *= f;
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = (d[j][i] - ref) * sc;
                const float e = __builtin_amdgcn_exp2f(z);
                s += e;
                t2 = fmaf(e, fmaxf(z, Z_MIN), t2);
            }
    }
    s = wave_sum(s);
    t2 = wave_sum(t2);
    if (NW > 1) {
        if (lane == 0) { red[NW + wave] = s; red[2 * NW + wave] = t2; }
        if (tid == 0) ncand = 0;
        __syncthreads();
        s = t2 = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) { s += red[NW + w]; t2 += red[2 * NW + w]; }
    } else if (tid == 0) ncand = 0;

    if (a.topk > 0) {
        const int k = a.topk;
        // lower bound of the k-th best: the maximum itself for one; else the k-th best of a wave's 64 thread maxima (16 leading
        // bits of the order, by bisection over ballots), the larger of the waves'
        float T_ = md;
        __syncthreads();
        if (k > 1) {
            const unsigned key16 = ord_bits(tm) >> 16;
            unsigned th = 0;
#pragma unroll
            for (int b = 15; b >= 0; --b) {
                const unsigned c = th | (1u << b);
                if (__popcll(__ballot(key16 >= c)) >= k) th = c;
            }
            if (NW > 1) {
                if (lane == 0) red[wave] = __builtin_bit_cast(float, th);
                __syncthreads();
#pragma unroll
                for (int w = 0; w < NW; ++w) th = max(th, __builtin_bit_cast(unsigned, red[w]));
            }
            T_ = th <= 0x007Fu ? NEG_INF : ord_float(th << 16);
        }
        const bool nan = s != s;             // a NaN is no maximum of its vector: such a chunk takes the rounds below
        // (columns behind the chunk's end hold -inf and are told by their index)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            if (vm[j] >= T_ && !nan) {
                const int at = c0 + (j * NT + tid) * 8;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (d[j][i] >= T_ && at + i < c1) {
                        const int p = atomicAdd(&ncand, 1);
                        if (p < CAP) cand[p] = make_key(d[j][i], at + i);
                    }
            }
        }
        __syncthreads();
        const int n = ncand;
        if (n <= CAP && !nan) {
            for (int q = tid; q < MAX_K; q += NT) best[q] = 0;
            __syncthreads();
            for (int q = tid; q < n; q += NT) {
                const u64 key = cand[q];
                int rank = 0;
                for (int r = 0; r < n; ++r) rank += cand[r] > key;
                if (rank < k) best[rank] = key;
            }
            __syncthreads();
        } else if (md == NEG_INF && !nan) {          // nothing but -inf: the first ones
            for (int q = tid; q < k; q += NT) best[q] = c0 + q < c1 ? make_key(NEG_INF, c0 + q) : 0;
            __syncthreads();
        } else {
            // many equal or masked values, or a NaN: k rounds of the next best key.  The columns are read again, eight loads at
            // a time: d kept alive to here costs registers in every row (12608 rows of 4096: 25.3 us without, 28.7 with)
            u64 last = ~0ull;
            for (int q = 0; q < k; ++q) {
                u64 mine = 0;
                for (int b = c0 + tid; b < c1; b += 8 * NT) {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int at = min(b + i * NT, c1 - 1);
                        v[i] = to_f32<T>(x[at]) - (CEN ? a.center[at] : 0.f);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const u64 key = make_key(v[i], min(b + i * NT, c1 - 1));
                        if (key < last && key > mine) mine = key;
                    }
                }
                mine = wave_max_u64(mine);
                if (NW > 1) {
                    if (lane == 0) rkey[wave] = mine;
                    __syncthreads();
#pragma unroll
                    for (int w = 0; w < NW; ++w) mine = rkey[w] > mine ? rkey[w] : mine;
                    __syncthreads();
                }
                if (tid == 0) best[q] = mine;
                last = mine;
            }
            __syncthreads();
        }
    }
    if (a.S == 1) {
        if (wave == 0) finish_row<T>(a, row, md, s, t2, lane);
        if (tid < a.topk) put_top(a, row, tid, best[tid], md, s);
    } else {
        const int64_t p = row * a.S + ch;
        if (tid == 0) a.parts[p] = Part{md, s, t2, 0.f};
        if (tid < a.topk) a.keys[p * a.topk + tid] = best[tid];
    }
}

// Joins the chunks of a row: one wave per row, lane = chunk (at most 64).  Up to 64 keys are ranked against each other, a key a
// lane; more are merged, a round a result (ranked too, 160 took 6.6 us instead of 4).  4 .. 5 us, a launch's latency (512 rows of
// 8 chunks with 8 best each: 6 by rounds).
template <typename T> __global__ __launch_bounds__(64) void logprob_join_kernel(const FwdArgs a) {
    __shared__ u64 all[64];
    const int lane = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int n = a.S * a.topk;
    const u64* keys = a.keys + row * n;
    Part q{NEG_INF, 0.f, 0.f, 0.f};
    if (lane < a.S) q = a.parts[row * a.S + lane];
    u64 cur = 0;
    if (n <= 64) {
        if (lane < n) cur = keys[lane];
        all[lane] = cur;
    }
    const float md = wave_max(q.m);
    const float sc = a.inv_temp * LOG2E;
    const float dl = q.m == NEG_INF ? 0.f : (q.m - md) * sc;       // an empty chunk has s = t = 0 (or NaN)
    const float f = __builtin_amdgcn_exp2f(dl);
    const float s = wave_sum(q.s * f);
    const float t2 = wave_sum(f * fmaf(q.s, fmaxf(dl, Z_MIN), q.t));
    finish_row<T>(a, row, md, s, t2, lane);
    if (n <= 64) {
        __syncthreads();
        int rank = 0;
#pragma unroll 8
        for (int r = 0; r < n; ++r) rank += all[r] > cur;
        if (cur && rank < a.topk) put_top(a, row, rank, cur, md, s);       // (0: no key, a chunk of fewer columns)
        return;
    }
    int head = 0;
    keys += lane * a.topk;
    if (lane < a.S) cur = keys[0];
    for (int j = 0; j < a.topk; ++j) {
        const u64 b = wave_max_u64(cur);
        if (cur == b && b != 0) {
            put_top(a, row, j, b, md, s);
            ++head;
            cur = head < a.topk ? keys[head] : 0;
        }
    }
}

struct BwdArgs {
    const void* x;
    int64_t ld, rows;
    int K, S, chunk, T, topk;
    const float* center;
    float inv_temp;
    const float* stats;
    const float* entropy;
    const int64_t* targets;
    const float* dlp;
    const float* dent;
    const int64_t* top_idx;
    const float* dtop;
    void* dx;
    int64_t ldd;
};

constexpr int BNT = 256, BNV = 4, BCHUNK = BNT * 8 * BNV;

// dx_k = (sum_j g_j [k = idx_j] - p_k (sum_j g_j + gH (log p_k + H))) / tau; the (index, gradient) pairs of the row that
// fall into the chunk are compacted in their order, so a repeated index adds up the same way every time.
// Bound: memory.  One read, one write: 2560 rows of 65536 bf16 (671 MB) 113 us = 5.9 TB/s; 12608 of 4096 (207 MB) 38 us.
template <typename T>
__global__ __launch_bounds__(BNT) void logprob_bwd_kernel(const BwdArgs a) {
    extern __shared__ __attribute__((aligned(8))) char smem[];
    int* lidx = (int*)smem;
    float* lg = (float*)(lidx + a.T + a.topk);
    __shared__ int ln;
    __shared__ float lsum;
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t row = blockIdx.x / a.S;
    const int c0 = (int)(blockIdx.x - row * a.S) * BCHUNK, c1 = min(a.K, c0 + BCHUNK);
    const T* x = (const T*)a.x + row * a.ld;
    T* dx = (T*)a.dx + row * a.ldd;
    const float md = a.stats[2 * row], logs = a.stats[2 * row + 1];
    const bool none = md == NEG_INF && logs == NEG_INF;

    float d[BNV][8];
#pragma unroll
    for (int j = 0; j < BNV; ++j) {
        const int at = c0 + (j * BNT + tid) * 8;
        if (at + 8 <= c1) {
            load8u<T>(x + at, d[j]);
            if (a.center) {
                float c[8];
                load8u<float>(a.center + at, c);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[j][i] -= c[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                d[j][i] = at + i < c1 ? to_f32<T>(x[at + i]) - (a.center ? a.center[at + i] : 0.f) : NEG_INF;
        }
    }
    if (tid < 64) {
        float sum = 0.f;
        int n = 0;
        for (int b = 0; b < a.T + a.topk; b += 64) {
            const int j = b + lane;
            int64_t at = -1;
            float g = 0.f;
            if (j < a.T) {
                if (a.dlp) {
                    at = a.targets[row * a.T + j];
                    g = a.dlp[row * a.T + j];
                }
            } else if (j < a.T + a.topk && a.dtop) {
                at = a.top_idx[row * a.topk + j - a.T];
                g = a.dtop[row * a.topk + j - a.T];
            }
            if (at < 0 || at >= a.K) g = 0.f;
            sum += wave_sum(g);
            const bool in = at >= c0 && at < c1;
            const u64 m = __ballot(in);
            if (in) {
                const int p = n + __popcll(m & ((1ull << lane) - 1));
                lidx[p] = (int)at;
                lg[p] = g;
            }
            n += __popcll(m);
        }
        if (lane == 0) {
            ln = n;
            lsum = sum;
        }
    }
    __syncthreads();
    const int n = ln;
    const float gH = a.dent ? a.dent[row] : 0.f, H = a.entropy[row];
    const float base = lsum + gH * H;
#pragma unroll
    for (int j = 0; j < BNV; ++j) {
        const int at = c0 + (j * BNT + tid) * 8;
        if (at >= c1) continue;
        float g[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float lp = (d[j][i] - md) * a.inv_temp - logs;
            const float p = __builtin_amdgcn_exp2f(lp * LOG2E);
            g[i] = none ? 0.f : -p * fmaf(gH, fmaxf(lp, Z_MIN), base);
        }
        if (!none)
            for (int q = 0; q < n; ++q) {
                const int o = lidx[q] - at;
                if (o >= 0 && o < 8) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (i == o) g[i] += lg[q];
                }
            }
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] *= a.inv_temp;
        if (at + 8 <= c1) store8u<T>(dx + at, g);
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at + i < c1) dx[at + i] = from_f32<T>(g[i]);
        }
    }
}

// Columns per workgroup.  A row of up to 16384 is one workgroup's, up to 64 columns a thread (one wave's up to 2048): no
// second launch.  Two chunks and a join against it, us on MI355X: 333 rows of 8191 (fp32, topk 5) 10.4 / 6.8; of 16384, bf16
// with topk 5: 1 row 8.5 / 6.9, 512 13.4 / 9.4, 2560 28.2 / 23.8, 12608 125 / 113.
// Longer rows are cut into chunks of 8192, 32 columns a thread (512 rows of 65536 bf16, centred, topk 8: 26 us; chunks of
// 16384: 27), joined by a second kernel; of 16384 where 64 chunks would not reach the end.
struct Plan {
    int nt, nv, chunk, S;
};
Plan plan_of(int64_t rows, int K) {
    Plan p;
    p.nt = K <= 2048 ? 64 : K <= 4096 ? 128 : 256;
    p.nv = 1;
    const int most = K > 16384 && K <= 8192 * MAX_CHUNKS ? 4 : 8;
    while (p.nv < most && p.nt * 8 * p.nv < K) p.nv *= 2;
    // few rows: shorter chunks, so that a row is read by many CUs (1 row of 65536: 32 chunks of 2048)
    if (K > 16384)
        while (p.nv > 1) {
            const int64_t next = (K + p.nt * 4 * p.nv - 1) / (p.nt * 4 * p.nv);
            if (next > MAX_CHUNKS || rows * next > 1024) break;
            p.nv /= 2;
        }
    p.chunk = p.nt * 8 * p.nv;
    p.S = (K + p.chunk - 1) / p.chunk;
    return p;
}

template <typename T, bool CEN> int run_fwd(const FwdArgs& a, const Plan& p, hipStream_t st) {
    const dim3 grid((unsigned)(a.rows * p.S));
#define LAUNCH(NT_, NV_) \
    if (p.nt == NT_ && p.nv == NV_) hipLaunchKernelGGL((logprob_fwd_kernel<T, NT_, NV_, CEN>), grid, dim3(NT_), 0, st, a)
    LAUNCH(64, 1);
    LAUNCH(64, 2);
    LAUNCH(64, 4);
    LAUNCH(128, 4);
    LAUNCH(256, 1);
    LAUNCH(256, 2);
    LAUNCH(256, 4);
    LAUNCH(256, 8);
#undef LAUNCH
    int rc = dino_launch_status();
    if (rc == DINO_OK && p.S > 1) {
        hipLaunchKernelGGL((logprob_join_kernel<T>), dim3((unsigned)a.rows), dim3(64), 0, st, a);
        rc = dino_launch_status();
    }
    return rc;
}

int64_t ws_bytes(int64_t rows, int K, int topk) {
    const Plan p = plan_of(rows, K);
    return p.S > 1 ? rows * p.S * (int64_t)(sizeof(Part) + 8 * topk) : 0;
}

}  // namespace

extern "C" int dino_logprob_workspace(int64_t rows, int K, int topk, int64_t* bytes) {
    DINO_CHECK_ARG(bytes && rows >= 0 && K > 0 && topk >= 0 && topk <= MAX_K && topk <= K);
    if (K > CHUNK_MAX * MAX_CHUNKS) return DINO_ERR_TOO_LARGE;
    *bytes = ws_bytes(rows, K, topk);
    return DINO_OK;
}

extern "C" int dino_logprob_fwd(int dtype, const void* logits, int64_t ld, int64_t rows, int K, const float* center,
                                float inv_temp, const int64_t* targets, int T, int topk, float* log_prob,
                                float* entropy, float* stats, float* top_log_prob, int64_t* top_index,
                                void* workspace, int64_t workspace_bytes, void* stream) {
    DINO_CHECK_ARG(dtype == DINO_F32 || dtype == DINO_BF16);
    DINO_CHECK_ARG(rows >= 0 && K > 0 && ld >= K && T >= 0 && topk >= 0 && topk <= MAX_K && topk <= K);
    DINO_CHECK_ARG(inv_temp > 0.f && inv_temp <= 3.4e38f);
    if (rows == 0) return DINO_OK;
    DINO_CHECK_ARG(logits && entropy && stats && (T == 0 || (targets && log_prob)) &&
                   (topk == 0 || (top_log_prob && top_index)));
    if (K > CHUNK_MAX * MAX_CHUNKS) return DINO_ERR_TOO_LARGE;
    const Plan p = plan_of(rows, K);
    // fewer than 2^32 threads a launch (the joining kernel: 64 a row)
    if (rows >= (1ll << 26) || rows * p.S * p.nt >= (1ll << 32)) return DINO_ERR_TOO_LARGE;
    DINO_CHECK_ARG(p.S == 1 || (workspace && workspace_bytes >= ws_bytes(rows, K, topk)));
    FwdArgs a{logits, ld, rows, K, p.S, p.chunk, T, topk, center, inv_temp, targets, log_prob, entropy, stats,
              top_log_prob, top_index, (Part*)workspace,
              p.S > 1 ? (u64*)((char*)workspace + rows * p.S * (int64_t)sizeof(Part)) : nullptr};
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == DINO_BF16) return center ? run_fwd<bf16, true>(a, p, st) : run_fwd<bf16, false>(a, p, st);
    return center ? run_fwd<float, true>(a, p, st) : run_fwd<float, false>(a, p, st);
}

extern "C" int dino_logprob_bwd(int dtype, const void* logits, int64_t ld, int64_t rows, int K, const float* center,
                                float inv_temp, const float* stats, const float* entropy, const int64_t* targets, int T,
                                const float* dlog_prob, const float* dentropy, const int64_t* top_index, int topk,
                                const float* dtop_log_prob, void* dlogits, int64_t ldd, void* stream) {
    DINO_CHECK_ARG(dtype == DINO_F32 || dtype == DINO_BF16);
    DINO_CHECK_ARG(rows >= 0 && K > 0 && ld >= K && ldd >= K && T >= 0 && topk >= 0 && topk <= MAX_K);
    DINO_CHECK_ARG(inv_temp > 0.f && inv_temp <= 3.4e38f);
    if (rows == 0) return DINO_OK;
    DINO_CHECK_ARG(logits && stats && entropy && dlogits && (!dlog_prob || T == 0 || targets) &&
                   (!dtop_log_prob || topk == 0 || top_index));
    if (K > CHUNK_MAX * MAX_CHUNKS || T > 4096) return DINO_ERR_TOO_LARGE;
    const int S = (K + BCHUNK - 1) / BCHUNK;
    if (rows >= (1ll << 31) || rows * S * BNT >= (1ll << 32)) return DINO_ERR_TOO_LARGE;
    const BwdArgs a{logits, ld, rows, K, S, BCHUNK, dlog_prob ? T : 0, dtop_log_prob ? topk : 0, center, inv_temp,
                    stats, entropy, targets, dlog_prob, dentropy, top_index, dtop_log_prob, dlogits, ldd};
    const int smem = (a.T + a.topk) * 8;
    const dim3 grid((unsigned)(rows * S));
    if (dtype == DINO_BF16)
        hipLaunchKernelGGL((logprob_bwd_kernel<bf16>), grid, dim3(BNT), smem, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL((logprob_bwd_kernel<float>), grid, dim3(BNT), smem, (hipStream_t)stream, a);
    return dino_launch_status();
}
