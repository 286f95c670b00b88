// Row soft-max of attention scores with a learned relative position bias, and its gradient.
//
// Rows are (sample b, head h, query i), columns are keys j; queries and keys sit on grids qh x qw and kh x kw (1 x L for a
// sequence).  The bias depends on the offset of the key from the query only: slot (jy - iy + qh - 1, jx - ix + qw - 1) of a
// (qh + kh - 1) x (qw + kw - 1) map of buckets, and a table [bucket][head]:
//   v = scale * x + table[bucket(slot)][h];  a column is out where the key mask is 0 or v is -inf;  y = exp(v - max) / sum,
//   0 in columns that are out and in rows where every column is; a NaN among a row's scores makes the whole row NaN
//   p = exp(v - max) / sum from the scores again (never from the rounded y),  ds = p * (dy - sum p dy),  dx = scale * ds,
//   dtable[k][h] = sum of ds over the samples and the pairs whose slot has bucket k
//
// exp(d) of a difference d <= 0 is the hardware's 2^(d log2 e): two instructions where a library exponential takes a dozen.  That is off by
// |d| / 2 steps of float relative to itself, which 16-bit outputs do not see; float outputs (float probabilities, gradients of float scores)
// take six more instructions that put the lost part back (rs_exp).
//
// Bytes bind: every score is read once and every output written once; a row stays in registers in between.  The table is expanded once
// per call to [head][slot], where the bias of a row is a window whose rows are contiguous.  Four forms, by the row's length M:
//   M <= 128           16 lanes per row, four rows per wave side by side: the row's sums are four DPP steps, and nothing is done
//                      four times over that one wave instruction can do for four rows
//   M <= 8192, and columns in fours do not cross a row of the key grid (kw % 4 == 0 or a sequence), more than one query per row of
//   queries            rs_*_vec: a lane takes four neighbouring columns of two or four neighbouring queries: the 16 biases of
//                      four are 7 neighbouring words of the map, their 16 gradients fall into 7 slots
//   M <= 16384         a lane takes columns t, t + T, ...: neighbouring lanes read neighbouring words whatever the pitch, the
//                      alignment and the width of the key grid
//   longer             tiles of 8192 columns, two launches: sums of the tiles, then the tiles again
//
// Gradient of the table: a workgroup takes the rows of a tile of RX x RY neighbouring queries (of several samples) of one head and
// adds every ds into its slot of a slab in LDS.  In one row every column has a slot of its own, so the adds need no atomics, only
// an order between rows (the barrier of the row's sum; wave_order() and a slab per unit where one wave has whole rows).  Slabs are written out, summed by slot and then
// by bucket in a fixed order, in double: a bucket may collect millions of terms.
//
// Measured on one MI355X (copy of 1 GiB: 5.2 TB/s), float scores, bfloat16 probabilities: 28672 rows of 1792 (32 x 56 map) 59 us =
// 5.2 TB/s; 8160 rows of 8160 (68 x 120) forward 91 us = 4.4 TB/s, backward 146 us = 4.6 TB/s with the adds into the slabs, 23 + 5 us
// for the sums over slabs and buckets; the whole step with float probabilities 326 us for 1.33 GB in two passes.  117600 rows of 49 (7 x 7 windows, half):
// forward 13.6 us, backward 20.6 (1.7 TB/s: instructions bind, a row has 49 columns for 64 places).  Key rows that fours would cross
// (67 x 121): 125 us forward, column by column, the step 367 us.  Rows in tiles, 544 of 40000 keys: the step 223 us, x and dy read twice.
#pragma once
#include "row_ops.h"

#define RS_BLOCK 256
#define RS_TILE 8192            // columns of a workgroup where rows are split
// keeps the compiler from taking the first accesses of a rare path and of the usual one together (a vector access would fall apart)
#ifndef GVFI_HOSTSIM
#define RS_APART() asm volatile("" ::: "memory")
// a value that the compiler must not work with ahead of this place: conditions of rare paths, kept over the loop, would take the scalar
// registers of the usual one
#define RS_OPAQUE(x) asm volatile("" : "+v"(x))
#else
#define RS_APART() ((void)0)
#define RS_OPAQUE(x) ((void)0)
#endif
#define RS_LONGEST 16384        // longest row that one workgroup keeps

// division of numbers below 2^31 by an invariant: a product and a shift (gvfi_magic_div)
struct RsDiv { unsigned mul, sh; };
__device__ __forceinline__ unsigned rs_div(unsigned x, RsDiv d) { return (__umulhi(x, d.mul) + x) >> d.sh; }
static inline RsDiv rs_divisor(unsigned d) {
    RsDiv r;
    gvfi_magic_div(d, r.mul, r.sh);
    return r;
}

struct RsArgs {
    const void* x; long long ldx;
    const void* dy; long long lddy;
    void* y; long long ldy; int zero_to;      // output: y, or dx in the backward pass
    const float* table; const int* bucket_of;
    const float* bias;                        // [heads][slots]: the table by offset
    const unsigned char* mask;                // [B][M] or NULL
    float* stats;                             // [rows][2]: max, 1 / sum (0, 0: nothing in the row)
    float* part;                              // split rows: [rows][tiles][2]
    float* slab;                              // [heads][batch chunk][tile y][tile x][slab]
    double* dslot;                            // [zparts][heads][slots]
    const int* order; const int* starts;      // slots sorted by bucket, where each bucket starts
    float* dtable;
    float scale;
    long long rows;
    int B, heads, qh, qw, kh, kw, Q, M, nx, slots, buckets;
    RsDiv by_kw, by_Q, by_heads, by_qw, by_qh, by_gx;      // gx: groups of queries in a row of the query grid (rs_forward_vec)
    int per;                                  // forward: rows (rs_forward_vec: groups of four) of a unit of lanes
    int RX, RY, BC, tx, ty, tb, sw, slab_n;   // backward: tile of queries, samples of a workgroup, their numbers; slab width, size
    int zparts;                               // sums of a slot, joined with its bucket
    int tiles;                                // split rows: tiles of RS_TILE columns
};

__device__ __forceinline__ int rs_row_of(const RsArgs& a, int j) { return (int)rs_div((unsigned)j, a.by_kw); }

// exp(d), d <= 0 (-inf: 0; a NaN stays one).  OUT: the type of what is computed from it.  For float the rounding of t = d log2 e and the tail
// of the constant, |d| / 2 steps of the result together, are put back (two steps are left); an output of 16 bits does not see them.
template <typename OUT> __device__ __forceinline__ float rs_exp(float d) {
    const float t = d * 1.44269504f, y = exp2_hw(t);
    if constexpr (sizeof(OUT) == 2) return y;
    const float lost = fmaf(d, 1.92596299e-8f, fmaf(d, 1.44269504f, -t)) * 0.69314718f;
    return fmaf(y, t >= -150.f ? lost : 0.f, y);            // (-inf, and a t that overflowed: lost is a NaN, y is 0)
}

// position of a row, advanced row by row
struct RsPos {
    int b, h, iy, ix;
    __device__ __forceinline__ void next(const RsArgs& a) {
        if (++ix == a.qw) {
            ix = 0;
            if (++iy == a.qh) {
                iy = 0;
                if (++h == a.heads) { h = 0; ++b; }
            }
        }
    }
};
__device__ __forceinline__ RsPos rs_pos(const RsArgs& a, long long r) {
    RsPos p;
    const unsigned q = rs_div((unsigned)r, a.by_Q), i = (unsigned)r - q * (unsigned)a.Q;
    p.b = (int)rs_div(q, a.by_heads);
    p.h = (int)(q - (unsigned)p.b * (unsigned)a.heads);
    p.iy = (int)rs_div(i, a.by_qw);
    p.ix = (int)(i - (unsigned)p.iy * (unsigned)a.qw);
    return p;
}
// where a row's bias starts: column j has p[(j / kw) * nx + j % kw]
__device__ __forceinline__ const float* rs_bias_row(const RsArgs& a, int h, int iy, int ix) {
    return a.bias + (long long)h * a.slots + (long long)(a.qh - 1 - iy) * a.nx + (a.qw - 1 - ix);
}

// sum / maximum over the T lanes of a row: 16 (a DPP row) or whole waves (each wave its own)
template <int T> __device__ __forceinline__ float rs_sum(float v) {
    if constexpr (T >= 64) return wave_sum(v);
    else return row_sum(v);
}
template <int T> __device__ __forceinline__ float rs_max(float v) {
    if constexpr (T >= 64) return wave_max(v);
    else return row_max(v);
}
// joins the waves of a row: (m, s) of a wave -> of the row, and the factor exp(max of the wave - max of the row).  Lane l of every 16
// takes wave l's pair.  red: two buffers in turn (a wave writes one again only after the barrier of the other)
template <typename OUT, int WAVES> __device__ __forceinline__ float rs_join(float& m, float& s, const float (*red)[2]) {
    static_assert(WAVES <= 16, "a pair per lane of a DPP row");
    const int l = threadIdx.x & 15;
    const float ml = l < WAVES ? red[l & (WAVES - 1)][0] : -INFINITY, sl = l < WAVES ? red[l & (WAVES - 1)][1] : 0.f;
    const float top = row_max(ml), z = top == -INFINITY ? 0.f : top;
    const float f = rs_exp<OUT>(m - z);
    m = top;
    s = row_sum(sl * rs_exp<OUT>(ml - z));
    return f;
}
// the same for plain sums
template <int WAVES> __device__ __forceinline__ float rs_join_sum(const float* red) {
    const int l = threadIdx.x & 15;
    return row_sum(l < WAVES ? red[l & (WAVES - 1)] : 0.f);
}
__device__ __forceinline__ int rs_col(const RsArgs& a, int j) { return j < a.M ? j : a.M - 1; }
// which of a lane's columns are there
template <int T, int NV> __device__ __forceinline__ void rs_mask(const RsArgs& a, int b, int t, int c0, bool (&in)[NV]) {
    if (a.mask) {
        const unsigned char* mask = a.mask + (long long)b * a.M;
        unsigned char m[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) m[i] = mask[rs_col(a, c0 + t + i * T)];
#pragma unroll
        for (int i = 0; i < NV; ++i) in[i] = c0 + t + i * T < a.M && m[i] != 0;
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) in[i] = c0 + t + i * T < a.M;
    }
}

// ---- forward: T lanes per row, ROWS rows in flight
template <typename TX, typename TY, int T, int NV, int ROWS>
__global__ __launch_bounds__(T < RS_BLOCK ? RS_BLOCK : T) void rs_forward_kernel(RsArgs a) {
    constexpr int WAVES = T >= 64 ? T / 64 : 1, UNITS = T < RS_BLOCK ? RS_BLOCK / T : 1;
    __shared__ float red[2][ROWS][WAVES][2];
    const int t = threadIdx.x % T;
    const long long r0 = ((long long)blockIdx.x * UNITS + threadIdx.x / T) * a.per;
    const long long r1 = r0 + a.per < a.rows ? r0 + a.per : a.rows;
    int co[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = rs_col(a, t + i * T);
        co[i] = rs_row_of(a, j) * (a.nx - a.kw) + j;
    }
    RsPos pos = rs_pos(a, r0 < a.rows ? r0 : 0);
    int par = 0;
    // (every unit makes the same number of turns: the lanes of a wave stay together)
    for (int k = 0; k < a.per; k += ROWS, par ^= 1) {
        const long long r = r0 + k;
        float v[ROWS][NV], m[ROWS], s[ROWS];
        RsPos p = pos;
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            // (loads without branches: a lane past the end reads the last column, a row past the end the first row)
            const bool live = r + q < r1;
            const TX* x = (const TX*)a.x + (live ? r + q : 0) * a.ldx;
            const float* bias = rs_bias_row(a, live ? p.h : 0, live ? p.iy : 0, live ? p.ix : 0);
            bool in[NV];
            rs_mask<T, NV>(a, live ? p.b : 0, t, 0, in);
#pragma unroll
            for (int i = 0; i < NV; ++i) v[q][i] = fmaf(Elem<TX>::ld(x + rs_col(a, t + i * T)), a.scale, bias[co[i]]);
#pragma unroll
            for (int i = 0; i < NV; ++i) v[q][i] = live && in[i] ? v[q][i] : -INFINITY;
            p.next(a);
        }
        pos = p;
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            m[q] = v[q][0];
#pragma unroll
            for (int i = 1; i < NV; ++i) m[q] = fmaxf(m[q], v[q][i]);
            m[q] = rs_max<T>(m[q]);                         // (passes over NaN, which comes back in the sum)
            const float top = m[q] == -INFINITY ? 0.f : m[q];
            s[q] = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                v[q][i] = rs_exp<TY>(v[q][i] - top);
                s[q] += v[q][i];
            }
            s[q] = rs_sum<T>(s[q]);
            if (WAVES > 1 && (threadIdx.x & 63) == 0) {
                red[par][q][threadIdx.x >> 6][0] = m[q];
                red[par][q][threadIdx.x >> 6][1] = s[q];
            }
        }
        if (WAVES > 1) __syncthreads();
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            float f = 1.f;
            if constexpr (WAVES > 1) f = rs_join<TY, WAVES>(m[q], s[q], red[par][q]);
            if (r + q >= r1) continue;
            const float inv = s[q] == 0.f ? 0.f : 1.f / s[q];
            f *= inv;
            TY* y = (TY*)a.y + (r + q) * a.ldy;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (t + i * T < a.M) y[t + i * T] = to_elem<TY>(v[q][i] * f);
            for (int j = a.M + t; j < a.zero_to; j += T) y[j] = to_elem<TY>(0.f);
            if (a.stats && t == 0) {
                a.stats[2 * (r + q)] = m[q] == -INFINITY ? 0.f : m[q];
                a.stats[2 * (r + q) + 1] = inv;
            }
        }
    }
}

// Four neighbouring elements wherever they lie: the hardware takes vector accesses at any element's alignment.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Four { T e[4]; };
template <typename T> __device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
    const Four<T> q = *(const Four<T>*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = Elem<T>::ld(&q.e[e]);
}
template <typename T> __device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
    Four<T> q;
#pragma unroll
    for (int e = 0; e < 4; ++e) q.e[e] = to_elem<T>(v[e]);
    *(Four<T>*)p = q;
}
// A lane's chunk of four columns j .. j + 3.  Loads have no branches: a chunk over the row's end (nv < 4) loads the row's last four and
// moves them `sh` places to the left, one behind the end loads them too (M > 128).  What it holds from column M on is to be ignored.
struct RsChunk {
    int j, at, nv;
    __device__ __forceinline__ RsChunk(const RsArgs& a, int column) {
        j = column;
        at = j + 4 <= a.M ? j : a.M - 4;
        nv = a.M - j < 4 ? (a.M - j > 0 ? a.M - j : 0) : 4;
    }
    static __device__ __forceinline__ RsChunk rare(const RsArgs& a, int column) {
        RS_OPAQUE(column);
        return RsChunk(a, column);
    }
    // the columns that are over the end, after the load
    __device__ __forceinline__ void settle(float (&v)[4]) const {
        if (at != j)
#pragma unroll
            for (int k = 0; k < 3; ++k)
                if (at + k < j) { v[0] = v[1]; v[1] = v[2]; v[2] = v[3]; }
    }
    template <typename T> __device__ __forceinline__ void store(T* row, const float (&v)[4]) const {
        if (nv == 4) {
            store4<T>(row + j, v);
        } else if (nv > 0) {
            RS_APART();
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < nv) row[j + e] = to_elem<T>(v[e]);
        }
    }
    // which columns are there
    __device__ __forceinline__ void mask(const unsigned char* m, bool (&in)[4]) const {
        if (m) {
            float v[4];
            const Four<unsigned char> q = *(const Four<unsigned char>*)(m + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)q.e[e];
            settle(v);
#pragma unroll
            for (int e = 0; e < 4; ++e) in[e] = e < nv && v[e] != 0.f;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) in[e] = e < nv;
        }
    }
};
// the biases of four columns and NQ neighbouring queries: column e of query q has w[NQ - 1 - q + e].  p: the first column's, query 0.
// (Where fewer queries or columns are left, a few words before or behind the map are read: RS_MARGIN.)
template <int NQ> __device__ __forceinline__ void load_window(const float* p, float (&w)[8]) {
    float lo[4], hi[4];
    load4<float>(p - (NQ - 1), lo);
    if (NQ > 2) load4<float>(p - (NQ - 1) + 4, hi);
    else hi[0] = p[3], hi[1] = hi[2] = hi[3] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        w[e] = lo[e];
        w[4 + e] = hi[e];
    }
}

// all chunks i of this wave are whole (one scalar comparison)
#define RS_FULL(i) (((T == 64 ? 0 : wave * 64) + 63 + (i) * T) * 4 + 4 <= a.M)
// NQ queries ix .. ix + NQ - 1 of one row of the query grid at a time; a lane has NC chunks of four columns.
template <typename TX, typename TY, int T, int NC, int NQ>
__global__ __launch_bounds__(T < RS_BLOCK ? RS_BLOCK : T) void rs_forward_vec_kernel(RsArgs a) {
    constexpr int WAVES = T / 64, UNITS = T < RS_BLOCK ? RS_BLOCK / T : 1;
    __shared__ float red[2][NQ][WAVES][2];
    const int t = threadIdx.x % T, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const unsigned gx = (unsigned)(a.qw + NQ - 1) / NQ;                     // groups of a row of queries
    const long long groups = a.rows / a.qw * gx;
    const long long g0 = ((long long)blockIdx.x * UNITS + (T == 64 ? wave : 0)) * a.per;
    int co[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const RsChunk c(a, (t + i * T) * 4);
        const int j = c.nv > 0 ? c.j : c.at;
        co[i] = rs_row_of(a, j) * (a.nx - a.kw) + j;
    }
    int par = 0;
    for (int k = 0; k < a.per; ++k, par ^= 1) {
        const long long g = g0 + k;
        if (g >= groups) break;                                              // (the whole unit, in whole waves)
        const unsigned line = rs_div((unsigned)g, a.by_gx);                            // row of queries of all heads and samples
        const int ix = (int)((unsigned)g - line * gx) * NQ;
        const int nq = a.qw - ix < NQ ? a.qw - ix : NQ;
        const unsigned bh = rs_div(line, a.by_qh);
        const int iy = (int)(line - bh * (unsigned)a.qh), b = (int)rs_div(bh, a.by_heads), h = (int)(bh - (unsigned)b * (unsigned)a.heads);
        const long long r = (long long)line * a.qw + ix;
        const float* bias = rs_bias_row(a, h, iy, ix);
        const unsigned char* mask = a.mask ? a.mask + (long long)b * a.M : nullptr;
        float v[NQ][NC][4], m[NQ], s[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const TX* x = (const TX*)a.x + (r + (q < nq ? q : 0)) * a.ldx;   // (a query that is not there: the first again)
#pragma unroll
            for (int i = 0; i < NC; ++i) load4<TX>(x + RsChunk(a, (t + i * T) * 4).at, v[q][i]);
        }
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float w[8];
            load_window<NQ>(bias + co[i], w);
            if (!mask && RS_FULL(i)) {                       // no selects
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[q][i][e] = fmaf(v[q][i][e], a.scale, w[NQ - 1 - q + e]);
            } else {
                const RsChunk c = RsChunk::rare(a, (t + i * T) * 4);
                bool in[4];
                c.mask(mask, in);
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    c.settle(v[q][i]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[q][i][e] = in[e] ? fmaf(v[q][i][e], a.scale, w[NQ - 1 - q + e]) : -INFINITY;
                }
            }
        }
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            m[q] = -INFINITY;
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) m[q] = fmaxf(m[q], v[q][i][e]);
            m[q] = wave_max(m[q]);
            const float top = m[q] == -INFINITY ? 0.f : m[q];
            s[q] = 0.f;
#pragma unroll
            for (int i = 0; i < NC; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[q][i][e] = rs_exp<TY>(v[q][i][e] - top);
                    s[q] += v[q][i][e];
                }
            s[q] = wave_sum(s[q]);
            if (WAVES > 1 && (threadIdx.x & 63) == 0) {
                red[par][q][threadIdx.x >> 6][0] = m[q];
                red[par][q][threadIdx.x >> 6][1] = s[q];
            }
        }
        if (WAVES > 1) __syncthreads();
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            float f = 1.f;
            if constexpr (WAVES > 1) f = rs_join<TY, WAVES>(m[q], s[q], red[par][q]);
            if (q >= nq) continue;
            const float inv = s[q] == 0.f ? 0.f : 1.f / s[q];
            f *= inv;
            TY* y = (TY*)a.y + (r + q) * a.ldy;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[q][i][e] *= f;
                if (RS_FULL(i)) store4<TY>(y + (t + i * T) * 4, v[q][i]);
                else RsChunk::rare(a, (t + i * T) * 4).store(y, v[q][i]);
            }
            for (int j = a.M + t; j < a.zero_to; j += T) y[j] = to_elem<TY>(0.f);
            if (a.stats && t == 0) {
                a.stats[2 * (r + q)] = m[q] == -INFINITY ? 0.f : m[q];
                a.stats[2 * (r + q) + 1] = inv;
            }
        }
    }
}

// ---- split rows: tiles of RS_TILE columns.  Phase 0: (max, sum) of a tile; phase 1: joins a row's tiles and writes
template <typename TX, typename TY, int PHASE> __global__ __launch_bounds__(512) void rs_forward_split_kernel(RsArgs a) {
    constexpr int T = 512, NV = RS_TILE / T;
    __shared__ float red[T / 64];
    const long long r = blockIdx.x / (unsigned)a.tiles;
    const int tile = (int)(blockIdx.x - r * a.tiles), t = threadIdx.x;
    const RsPos p = rs_pos(a, r);
    const TX* x = (const TX*)a.x + r * a.ldx;
    const float* bias = rs_bias_row(a, p.h, p.iy, p.ix);
    float v[NV], m = -INFINITY, s = 0.f, inv = 0.f;
    bool in[NV];
    rs_mask<T, NV>(a, p.b, t, tile * RS_TILE, in);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = rs_col(a, tile * RS_TILE + t + i * T);
        v[i] = fmaf(Elem<TX>::ld(x + j), a.scale, bias[rs_row_of(a, j) * (a.nx - a.kw) + j]);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) v[i] = in[i] ? v[i] : -INFINITY;
    float* part = a.part + r * a.tiles * 2;
    if (PHASE == 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) m = fmaxf(m, v[i]);
        m = wave_max(m);
        if ((t & 63) == 0) red[t >> 6] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < T / 64; ++w) m = fmaxf(m, red[w]);
        __syncthreads();
    } else {
        for (int k = 0; k < a.tiles; ++k) m = fmaxf(m, part[2 * k]);
    }
    const float top = m == -INFINITY ? 0.f : m;
    if (PHASE == 1) {
        double all = 0.0;                                    // (a row may have 2^17 tiles)
        for (int k = 0; k < a.tiles; ++k) all += (double)(part[2 * k + 1] * rs_exp<TY>(part[2 * k] - top));
        s = (float)all;
        inv = s == 0.f ? 0.f : 1.f / s;
        TY* y = (TY*)a.y + r * a.ldy;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int j = tile * RS_TILE + t + i * T;
            if (j < a.M) y[j] = to_elem<TY>(rs_exp<TY>(v[i] - top) * inv);
        }
        if (tile == a.tiles - 1)
            for (int j = a.M + t; j < a.zero_to; j += T) y[j] = to_elem<TY>(0.f);
        if (a.stats && tile == 0 && t == 0) {
            a.stats[2 * r] = top;
            a.stats[2 * r + 1] = inv;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) s += rs_exp<TY>(v[i] - top);
    s = wave_sum(s);
    if ((t & 63) == 0) red[t >> 6] = s;
    __syncthreads();
    if (t == 0) {
        s = 0.f;
        for (int w = 0; w < T / 64; ++w) s += red[w];
        part[2 * tile] = m;
        part[2 * tile + 1] = s;
    }
}

// ---- backward.  SPLIT false: whole rows, PHASE unused.  SPLIT true: a tile of columns; PHASE 0 sums p dy of the tile into part,
// PHASE 1 takes the rows' sums from there.  T = 16: 16 units of 16 lanes, each with a run of the tile's rows and a slab of its own.
struct RsTile { int tile, h, x0, y0, b0, nxr, nyr, nbr; unsigned out; };
__device__ __forceinline__ RsTile rs_tile(const RsArgs& a, bool split) {
    RsTile c;
    unsigned u = blockIdx.x;
    c.tile = split ? (int)(u % (unsigned)a.tiles) : 0;
    if (split) u /= (unsigned)a.tiles;
    c.out = u;
    c.x0 = (int)(u % (unsigned)a.tx) * a.RX; u /= (unsigned)a.tx;
    c.y0 = (int)(u % (unsigned)a.ty) * a.RY; u /= (unsigned)a.ty;
    c.b0 = (int)(u % (unsigned)a.tb) * a.BC;
    c.h = (int)(u / (unsigned)a.tb);
    c.nxr = a.qw - c.x0 < a.RX ? a.qw - c.x0 : a.RX;
    c.nyr = a.qh - c.y0 < a.RY ? a.qh - c.y0 : a.RY;
    c.nbr = a.B - c.b0 < a.BC ? a.B - c.b0 : a.BC;
    return c;
}
template <typename TX, typename TY, int T, int NV, int ROWS, bool SPLIT, int PHASE>
__global__ __launch_bounds__(T < 64 ? RS_BLOCK : T) void rs_backward_kernel(RsArgs a) {
    constexpr int WAVES = T >= 64 ? T / 64 : 1, UNITS = T < 64 ? RS_BLOCK / T : 1, LANES = T * UNITS;
    __shared__ float red[2][ROWS][WAVES];
    GVFI_DYN_SMEM(smem);
    const int t = threadIdx.x % T, unit = threadIdx.x / T;
    float* slab = (float*)smem + unit * a.slab_n;
    const RsTile c = rs_tile(a, SPLIT);
    const int c0 = c.tile * RS_TILE;
    const bool adds = a.dtable != nullptr && !(SPLIT && PHASE == 0);
    if (adds) {
        for (int i = threadIdx.x; i < a.slab_n * UNITS; i += LANES) ((float*)smem)[i] = 0.f;
        __syncthreads();
    }
    const int jy0 = SPLIT ? rs_row_of(a, c0) : 0;
    int co[NV], so[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int j = rs_col(a, c0 + t + i * T), jy = rs_row_of(a, j);
        co[i] = jy * (a.nx - a.kw) + j;
        // (split: a tile's columns side by side, RX - 1 words more where a row of the key grid ends; RY is 1)
        so[i] = SPLIT ? j - c0 + (jy - jy0) * (a.RX - 1) : jy * a.sw + (j - jy * a.kw);
    }
    const int n = c.nxr * c.nyr * c.nbr, per = UNITS == 1 ? n : (n + UNITS - 1) / UNITS;
    const int k1 = unit * per + per < n ? unit * per + per : n;
    int k = unit * per, ix = 0, iy = 0, ib = 0, par = 0;
    if (UNITS > 1) {
        const int l = k / c.nxr;
        ix = k - l * c.nxr;
        ib = l / c.nyr;
        iy = l - ib * c.nyr;
    }
    for (int turn = 0; turn < per; turn += ROWS, k += ROWS, par ^= 1) {
        float p[ROWS][NV], d[ROWS][NV], dot[ROWS];
        int sb[ROWS];
        long long row[ROWS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            const bool live = k + q < k1;
            const int lb = c.b0 + (live ? ib : 0), ly = c.y0 + (live ? iy : 0), lx = c.x0 + (live ? ix : 0);
            row[q] = ((long long)lb * a.heads + c.h) * a.Q + (long long)ly * a.qw + lx;
            sb[q] = (a.RY - 1 - iy) * a.sw + a.RX - 1 - ix;
            dot[q] = 0.f;
            // (loads without branches, as in the forward pass)
            const TX* x = (const TX*)a.x + row[q] * a.ldx;
            const TY* dy = (const TY*)a.dy + row[q] * a.lddy;
            const float* bias = rs_bias_row(a, c.h, ly, lx);
            const float top = a.stats[2 * row[q]], inv = a.stats[2 * row[q] + 1];
            bool in[NV];
            rs_mask<T, NV>(a, lb, t, c0, in);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int j = rs_col(a, c0 + t + i * T);
                p[q][i] = fmaf(Elem<TX>::ld(x + j), a.scale, bias[co[i]]);
                d[q][i] = Elem<TY>::ld(dy + j);
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float v = live && in[i] ? p[q][i] : -INFINITY;
                p[q][i] = rs_exp<TX>(v - top) * inv;
                d[q][i] = v == -INFINITY ? 0.f : d[q][i];
                dot[q] += p[q][i] * d[q][i];
            }
            if (live && ++ix == c.nxr) {
                ix = 0;
                if (++iy == c.nyr) { iy = 0; ++ib; }
            }
        }
        if (SPLIT && PHASE == 1) {
            double all = 0.0;
            for (int w = 0; w < a.tiles; ++w) all += (double)a.part[row[0] * a.tiles + w];
            dot[0] = (float)all;
            if (adds) __syncthreads();
        } else {
#pragma unroll
            for (int q = 0; q < ROWS; ++q) dot[q] = rs_sum<T>(dot[q]);
            if (WAVES > 1) {
                // (two buffers in turn; the barrier is also the one between the adds of two rows)
#pragma unroll
                for (int q = 0; q < ROWS; ++q)
                    if ((threadIdx.x & 63) == 0) red[par][q][threadIdx.x >> 6] = dot[q];
                __syncthreads();
#pragma unroll
                for (int q = 0; q < ROWS; ++q) dot[q] = rs_join_sum<WAVES>(red[par][q]);
            }
        }
        if (SPLIT && PHASE == 0) {
            if (t == 0) a.part[row[0] * a.tiles + c.tile] = dot[0];
            continue;
        }
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            if (k + q < k1) {
                TX* dx = (TX*)a.y + row[q] * a.ldy;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int j = c0 + t + i * T;
                    if (j < a.M) {
                        const float ds = p[q][i] * (d[q][i] - dot[q]);
                        dx[j] = to_elem<TX>(ds * a.scale);
                        if (adds) slab[so[i] + sb[q]] += ds;
                    }
                }
            }
            // (of two rows, different lanes add to one word; several waves have the barrier of the row's sum in between)
            if (WAVES == 1 && !SPLIT) wave_order();
        }
    }
    if (adds) {
        __syncthreads();
        float* o = a.slab + ((long long)c.out * (SPLIT ? a.tiles : 1) + c.tile) * a.slab_n;
        for (int i = threadIdx.x; i < a.slab_n; i += LANES) {
            float s = ((float*)smem)[i];
            for (int u = 1; u < UNITS; ++u) s += ((float*)smem)[u * a.slab_n + i];
            o[i] = s;
        }
    }
}

// (the first slot of a chunk is a multiple of NQ: RX, the rows of the slab and the columns are multiples of four)
template <int NQ> __device__ __forceinline__ void slab_add(float* p, float a, float b, float c, float d) {
    if constexpr (NQ == 4) {
        float4 f = *(const float4*)p;
        f.x += a; f.y += b; f.z += c; f.w += d;
        *(float4*)p = f;
    } else {
        float2 f = ((const float2*)p)[0], g = ((const float2*)p)[1];
        f.x += a; f.y += b; g.x += c; g.y += d;
        ((float2*)p)[0] = f;
        ((float2*)p)[1] = g;
    }
}
// NQ queries at a time, four columns per chunk (rs_forward_vec_kernel): the 16 gradients of a chunk are joined to 7 neighbouring
// slots w[NQ - 1 - q + e] and added 16 bytes at a time -- the first four, which no other lane has, then, behind a barrier, the other three,
// which are the first of the next chunk.  RX, the slab's rows and so the chunks' first slots are multiples of four.
template <typename TX, typename TY, int T, int NC, int NQ> __global__ __launch_bounds__(T, 4) void rs_backward_vec_kernel(RsArgs a) {
    constexpr int WAVES = T / 64;
    __shared__ float red[2][NQ][WAVES];
    GVFI_DYN_SMEM(smem);
    float* slab = (float*)smem;
    const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const RsTile c = rs_tile(a, false);
    const bool adds = a.dtable != nullptr;
    if (adds) {
        for (int i = t; i < a.slab_n; i += T) slab[i] = 0.f;
        __syncthreads();
    }
    int co[NC], so[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const RsChunk k(a, (t + i * T) * 4);
        const int j = k.nv > 0 ? k.j : k.at, jy = rs_row_of(a, j);
        co[i] = jy * (a.nx - a.kw) + j;
        so[i] = k.nv > 0 ? jy * a.sw + (j - jy * a.kw) : -1;
    }
    int par = 0;
    for (int ib = 0; ib < c.nbr; ++ib)
        for (int iy = 0; iy < c.nyr; ++iy)
            for (int ix = 0; ix < c.nxr; ix += NQ, par ^= 1) {
                const int nq = c.nxr - ix < NQ ? c.nxr - ix : NQ;
                const long long r = (((long long)(c.b0 + ib)) * a.heads + c.h) * a.Q + (long long)(c.y0 + iy) * a.qw + c.x0 + ix;
                const float* bias = rs_bias_row(a, c.h, c.y0 + iy, c.x0 + ix);
                const unsigned char* mask = a.mask ? a.mask + (long long)(c.b0 + ib) * a.M : nullptr;
                float p[NQ][NC][4], d[NQ][NC][4], dot[NQ], top[NQ], inv[NQ];
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    const long long rq = r + (q < nq ? q : 0);               // (a query that is not there: the first again)
                    const TX* x = (const TX*)a.x + rq * a.ldx;
                    const TY* dy = (const TY*)a.dy + rq * a.lddy;
                    top[q] = a.stats[2 * rq];
                    inv[q] = q < nq ? a.stats[2 * rq + 1] : 0.f;
                    dot[q] = 0.f;
#pragma unroll
                    for (int i = 0; i < NC; ++i) {
                        const int at = RsChunk(a, (t + i * T) * 4).at;
                        load4<TX>(x + at, p[q][i]);
                        load4<TY>(dy + at, d[q][i]);
                    }
                }
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    float w[8];
                    load_window<NQ>(bias + co[i], w);
                    if (mask || nq < NQ || !RS_FULL(i)) {
                        const RsChunk k = RsChunk::rare(a, (t + i * T) * 4);
                        bool in[4];
                        k.mask(mask, in);
#pragma unroll
                        for (int q = 0; q < NQ; ++q) {
                            k.settle(p[q][i]);
                            k.settle(d[q][i]);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                p[q][i][e] = q < nq && in[e] ? fmaf(p[q][i][e], a.scale, w[NQ - 1 - q + e]) : -INFINITY;
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < NQ; ++q)
#pragma unroll
                            for (int e = 0; e < 4; ++e) p[q][i][e] = fmaf(p[q][i][e], a.scale, w[NQ - 1 - q + e]);
                    }
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float v = p[q][i][e];
                            p[q][i][e] = rs_exp<TX>(v - top[q]) * inv[q];
                            d[q][i][e] = v == -INFINITY ? 0.f : d[q][i][e];
                            dot[q] = fmaf(p[q][i][e], d[q][i][e], dot[q]);
                        }
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    dot[q] = wave_sum(dot[q]);
                    if (WAVES > 1 && (t & 63) == 0) red[par][q][t >> 6] = dot[q];
                }
                __syncthreads();                             // (also between the second adds of the group before and the first of this)
                if (WAVES > 1)
#pragma unroll
                    for (int q = 0; q < NQ; ++q) dot[q] = rs_join_sum<WAVES>(red[par][q]);
                const int sb = (a.RY - 1 - iy) * a.sw + a.RX - NQ - ix;
                float late[NC][4];
#pragma unroll
                for (int i = 0; i < NC; ++i) {
                    float w[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = 0.f;
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[q][i][e] *= d[q][i][e] - dot[q];
                        if (nq == NQ && RS_FULL(i)) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[NQ - 1 - q + e] += p[q][i][e];
                        } else {
                            // (selected: beside a NaN a column or a query that is not there has a NaN too, and its slot is another's)
                            const int nv = RsChunk::rare(a, (t + i * T) * 4).nv;
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[NQ - 1 - q + e] += q < nq && e < nv ? p[q][i][e] : 0.f;
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) p[q][i][e] *= a.scale;
                        TX* dx = (TX*)a.y + (r + q) * a.ldy;
                        if (q >= nq) continue;
                        if (RS_FULL(i)) store4<TX>(dx + (t + i * T) * 4, p[q][i]);
                        else RsChunk::rare(a, (t + i * T) * 4).store(dx, p[q][i]);
                    }
                    if (adds && (RS_FULL(i) || so[i] >= 0)) slab_add<NQ>(slab + so[i] + sb, w[0], w[1], w[2], w[3]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) late[i][e] = w[4 + e];
                }
                if (adds) {
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < NC; ++i)
                        if (RS_FULL(i) || so[i] >= 0) {
                            if (NQ == 4) slab_add<4>(slab + so[i] + sb + 4, late[i][0], late[i][1], late[i][2], 0.f);
                            else slab[so[i] + sb + 4] += late[i][0];
                        }
                }
            }
    if (adds) {
        __syncthreads();
        float* o = a.slab + (long long)c.out * a.slab_n;
        for (int i = t; i < a.slab_n; i += T) o[i] = slab[i];
    }
}

// ---- launches of one pair of element types (instantiated in a file of its own)
#define RS_MARGIN 4            // words before and behind the expanded table that load_window may touch
// whether rs_*_vec takes the rows (see the head of this file)
static inline bool rs_vec(const RsArgs& a) {
    return a.M > 128 && a.M <= 8192 && a.qw > 1 && (a.kh == 1 || a.kw % 4 == 0);
}
template <typename TX, typename TY> void rs_forward_launch(RsArgs a, hipStream_t st);
template <typename TX, typename TY> void rs_backward_launch(const RsArgs& a, hipStream_t st);

#ifdef RS_INSTANTIATE
// lanes of a row and columns per lane by the row's length: 16 lanes for short rows, then enough lanes for 16 columns or fewer in each
#define RS_BY_LENGTH(GO)                     \
    do {                                     \
        if (a.M <= 16) GO(16, 1, 4);         \
        else if (a.M <= 64) GO(16, 4, 2);    \
        else if (a.M <= 128) GO(16, 8, 1);   \
        else if (a.M <= 512) GO(64, 8, 1);   \
        else if (a.M <= 2048) GO(256, 8, 1); \
        else if (a.M <= 8192) GO(512, 16, 1); \
        else GO(1024, 16, 1);                \
    } while (0)

// the same for rs_*_vec: lanes, chunks of four columns per lane, queries at a time.  Two queries for the longest rows, whose workgroups
// would otherwise need the registers of a whole CU and leave it without work at every barrier.
#define RS_VEC_FORWARD(GO)                   \
    do {                                     \
        if (a.M <= 256) GO(64, 1, 4);        \
        else if (a.M <= 512) GO(64, 2, 4);   \
        else if (a.M <= 1024) GO(256, 1, 4); \
        else if (a.M <= 2048) GO(256, 2, 4); \
        else if (a.M <= 4096) GO(512, 2, 4); \
        else GO(512, 4, 2);                  \
    } while (0)
// The backward pass keeps twice as much per lane, so it takes more lanes, and above 256 columns two queries at a time.  40 M float scores with
// bfloat16 gradients, four queries | two, us: 200 columns 108 | 116; 401 114 | 105; 1000 106 | 110; 1500 113 | 110; 2400 123 | 121; 3500 117 | 114;
// 8160 288 | 181.  bfloat16 scores: 200 86 | 89; 401 80 | 78; 1000 69 | 71; 1500 81 | 81; 2400 92 | 83; 3500 80 | 74; 8160 234 | 134.
#define RS_VEC_BACKWARD(GO)                  \
    do {                                     \
        if (a.M <= 256) GO(64, 1, 4);        \
        else if (a.M <= 512) GO(128, 1, 2);  \
        else if (a.M <= 1024) GO(256, 1, 2); \
        else if (a.M <= 2048) GO(512, 1, 2); \
        else if (a.M <= 4096) GO(512, 2, 2); \
        else GO(512, 4, 2);                  \
    } while (0)

// rows (or groups) of a unit, at most 16: the chip's lanes are filled twice over while there are enough rows, by 16-lane units once (their
// start, divisions lane by lane, costs as much as a row)
static long long rs_per(long long rows, int lanes) {
    const long long units = (lanes < 64 ? 1 : 2) * 256LL * 2048 / lanes;
    const long long per = (rows + units - 1) / units;
    return per > 16 ? 16 : per;
}
template <typename TX, typename TY> void rs_forward_launch(RsArgs a, hipStream_t st) {
    if (a.tiles > 1) {
        const dim3 grid((unsigned)(a.rows * a.tiles));
        GVFI_LAUNCH_COOP((rs_forward_split_kernel<TX, TY, 0>), grid, dim3(512), st, a);
        GVFI_LAUNCH_COOP((rs_forward_split_kernel<TX, TY, 1>), grid, dim3(512), st, a);
        return;
    }
    if (rs_vec(a)) {
#define RS_GO(T, N, NQ)                                                                                               \
    do {                                                                                                              \
        const long long groups = a.rows / a.qw * ((a.qw + NQ - 1) / NQ);                                              \
        const long long per = rs_per(groups, T), pb = per * (T < RS_BLOCK ? RS_BLOCK / T : 1);                        \
        a.per = (int)per;                                                                                             \
        a.by_gx = rs_divisor((unsigned)((a.qw + NQ - 1) / NQ));                                                       \
        GVFI_LAUNCH_COOP((rs_forward_vec_kernel<TX, TY, T, N, NQ>), dim3((unsigned)((groups + pb - 1) / pb)),         \
                         dim3(T < RS_BLOCK ? RS_BLOCK : T), st, a);                                                   \
    } while (0)
        RS_VEC_FORWARD(RS_GO);
#undef RS_GO
        return;
    }
#define RS_GO(T, N, R)                                                                                                \
    do {                                                                                                              \
        long long per = rs_per(a.rows, T);                                                                            \
        per = (per + R - 1) / R * R;                                                                                  \
        const long long pb = per * (T < RS_BLOCK ? RS_BLOCK / T : 1);                                                 \
        a.per = (int)per;                                                                                             \
        GVFI_LAUNCH_COOP((rs_forward_kernel<TX, TY, T, N, R>), dim3((unsigned)((a.rows + pb - 1) / pb)),              \
                         dim3(T < RS_BLOCK ? RS_BLOCK : T), st, a);                                                   \
    } while (0)
    RS_BY_LENGTH(RS_GO);
#undef RS_GO
}
template <typename TX, typename TY> void rs_backward_launch(const RsArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((long long)a.heads * a.tb * a.ty * a.tx * a.tiles));
    const int shm = a.dtable ? a.slab_n * 4 * (a.M <= 128 ? 16 : 1) : 16;
    if (a.tiles > 1) {
        GVFI_LAUNCH_COOP_SHM((rs_backward_kernel<TX, TY, 512, RS_TILE / 512, 1, true, 0>), grid, dim3(512), 16, st, a);
        GVFI_LAUNCH_COOP_SHM((rs_backward_kernel<TX, TY, 512, RS_TILE / 512, 1, true, 1>), grid, dim3(512), shm, st, a);
        return;
    }
    if (rs_vec(a)) {
#define RS_GO(T, N, NQ) GVFI_LAUNCH_COOP_SHM((rs_backward_vec_kernel<TX, TY, T, N, NQ>), grid, dim3(T), shm, st, a)
        RS_VEC_BACKWARD(RS_GO);
#undef RS_GO
        return;
    }
#define RS_GO(T, N, R) GVFI_LAUNCH_COOP_SHM((rs_backward_kernel<TX, TY, T, N, R, false, 1>), grid, dim3(T < 64 ? RS_BLOCK : T), shm, st, a)
    RS_BY_LENGTH(RS_GO);
#undef RS_GO
}
#endif
