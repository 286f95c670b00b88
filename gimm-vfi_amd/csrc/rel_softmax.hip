// Biased row soft-max: the C ABI, the kernels without an element type, the tile of the backward pass (rel_softmax.h has the rest).
#include "rel_softmax.h"

__global__ __launch_bounds__(RS_BLOCK) void rs_expand_kernel(RsArgs a, float* bias) {
    const int i = blockIdx.x * RS_BLOCK + threadIdx.x, h = blockIdx.y;
    if (i >= a.slots) return;
    const int k = a.bucket_of[i];
    bias[(long long)h * a.slots + i] = (unsigned)k < (unsigned)a.buckets ? a.table[(long long)k * a.heads + h] : 0.f;
}

// The sum of a slot over the slabs that hold it, over parts w, w + P, ... of the (sample chunk, tile of query rows) pairs
__device__ __forceinline__ double rs_slot_sum(const RsArgs& a, int h, int s, int w, int P) {
    double acc = 0.0;
    const int sy = s / a.nx, sx = s - sy * a.nx;         // offset of the key from the query, from the smallest
    // in the slab of tile tx the slot has column sx - qw + (tx + 1) RX, which is in [0, kw + RX - 2]; rows likewise
    const int x0 = a.qw - sx > a.RX ? (a.qw - sx + a.RX - 1) / a.RX - 1 : 0, x1 = (a.kw + a.qw - 2 - sx) / a.RX;
    const int y0 = a.qh - sy > a.RY ? (a.qh - sy + a.RY - 1) / a.RY - 1 : 0, y1 = (a.kh + a.qh - 2 - sy) / a.RY;
    const unsigned nx = (unsigned)((x1 < a.tx ? x1 : a.tx - 1) - x0 + 1), ny = (unsigned)((y1 < a.ty ? y1 : a.ty - 1) - y0 + 1);
    const int ly1 = sy - a.qh + a.RY, lx1 = sx - a.qw + a.RX;               // row and column in the slab of tile 0
    const unsigned pairs = ny * (unsigned)a.tb;
    if (a.tiles == 1 && pairs >= (unsigned)P) {
        for (unsigned u = (unsigned)w; u < pairs; u += P) {
            const unsigned b = u / ny;
            const int ty = y0 + (int)(u - b * ny);
            // (from tile to tile the slot moves by a slab and RX words)
            const float* p = a.slab + ((((long long)h * a.tb + b) * a.ty + ty) * a.tx + x0) * a.slab_n + (ly1 + ty * a.RY) * a.sw + lx1 + x0 * a.RX;
#pragma unroll 8
            for (unsigned k = 0; k < nx; ++k) acc += (double)p[(long long)k * (a.slab_n + a.RX)];
        }
        return acc;
    }
    // few pairs (sequences have one row of queries): the parts take the tiles
    for (unsigned long long i = (unsigned)w; i < (unsigned long long)pairs * nx; i += P) {
        const unsigned u = (unsigned)(i / nx), b = u / ny;
        const int tx = x0 + (int)(i - (unsigned long long)u * nx), ty = y0 + (int)(u - b * ny), lx = lx1 + tx * a.RX;
        const long long blk = (((long long)h * a.tb + b) * a.ty + ty) * a.tx + tx;
        if (a.tiles == 1) {
            acc += (double)a.slab[blk * a.slab_n + (ly1 + ty * a.RY) * a.sw + lx];
            continue;
        }
        // split rows (RY is 1): the tiles that hold a column of this key row whose slab has the slot: jx in [lx - RX + 1, lx]
        const int jy = sy - (a.qh - 1) + ty;
        const int from = jy * a.kw + (lx - a.RX + 1 > 0 ? lx - a.RX + 1 : 0), to = jy * a.kw + (lx < a.kw - 1 ? lx : a.kw - 1);
        for (int tl = from / RS_TILE; tl <= to / RS_TILE; ++tl) {
            const int c0 = tl * RS_TILE, k0 = rs_row_of(a, c0);
            acc += (double)a.slab[(blk * a.tiles + tl) * a.slab_n + jy * a.kw - c0 + (jy - k0) * (a.RX - 1) + lx];
        }
    }
    return acc;
}

// Workgroups of the sums behind the slabs: a launch has fewer than 2^32 lanes, the workgroups loop over what is left
#ifndef GVFI_HOSTSIM
#define RS_MOST_GROUPS (1LL << 23)
#else
#define RS_MOST_GROUPS 7LL      // (the emulator's tests take the loops)
#endif
static unsigned rs_groups(long long n) { return (unsigned)(n < RS_MOST_GROUPS ? n : RS_MOST_GROUPS); }

// 16 slots x 16 of the parts of the slabs; gridDim.z workgroups share the slabs of 16 slots and leave a sum each
__global__ __launch_bounds__(RS_BLOCK) void rs_slots_kernel(RsArgs a) {
    __shared__ double red[16][16];
    const int l = threadIdx.x & 15, w = threadIdx.x >> 4, h = blockIdx.y;
    for (int s0 = (int)blockIdx.x * 16; s0 < a.slots; s0 += (int)gridDim.x * 16) {        // (slots < 2^30, the step at most 2^27)
        const int s = s0 + l;
        red[w][l] = s < a.slots ? rs_slot_sum(a, h, s, (int)blockIdx.z * 16 + w, 16 * a.zparts) : 0.0;
        __syncthreads();
        if (w == 0 && s < a.slots) {
            double acc = 0.0;
            for (int k = 0; k < 16; ++k) acc += red[k][l];
            a.dslot[((long long)blockIdx.z * a.heads + h) * a.slots + s] = acc;
        }
        __syncthreads();
    }
}

// sum of a bucket over its slots: P lanes per (bucket, head); with P = RS_BLOCK in `parts` workgroups, which leave their shares in `share`
template <int P> __global__ __launch_bounds__(RS_BLOCK) void rs_buckets_kernel(RsArgs a, int parts, double* share) {
    __shared__ double red[RS_BLOCK];
    const int t = threadIdx.x % P, h = blockIdx.y;
    const long long units = (long long)a.buckets * parts;
    for (long long u0 = (long long)blockIdx.x * (RS_BLOCK / P); u0 < units; u0 += (long long)gridDim.x * (RS_BLOCK / P)) {
        const long long unit = u0 + threadIdx.x / P;
        const long long k = unit / parts;
        const int part = (int)(unit - k * parts);
        double s = 0.0;
        if (k < a.buckets)
            for (int i = a.starts[k] + part * P + t; i < a.starts[k + 1]; i += P * parts) {
                const int slot = a.order[i];
                if ((unsigned)slot < (unsigned)a.slots)
                    for (int z = 0; z < a.zparts; ++z) s += a.dslot[((long long)z * a.heads + h) * a.slots + slot];
            }
        red[threadIdx.x] = s;
        for (int o = P / 2; o > 0; o >>= 1) {
            __syncthreads();
            if (t < o) red[threadIdx.x] += red[threadIdx.x + o];
        }
        if (t == 0 && k < a.buckets) {
            if (parts == 1) a.dtable[k * a.heads + h] = (float)red[threadIdx.x];
            else share[(k * a.heads + h) * parts + part] = red[threadIdx.x];
        }
        __syncthreads();
    }
}
__global__ __launch_bounds__(RS_BLOCK) void rs_shares_kernel(RsArgs a, int parts, const double* share) {
    const long long i = (long long)blockIdx.x * RS_BLOCK + threadIdx.x;
    if (i >= (long long)a.buckets * a.heads) return;
    double s = 0.0;
    for (int p = 0; p < parts; ++p) s += share[i * parts + p];
    a.dtable[i] = (float)s;
}
#define RS_SHARES (1024 * 64)
// Workgroups per bucket where the buckets are few and the slots many: logarithmic buckets put nearly all of a long sequence into one
static int rs_parts(const RsArgs& a, int buckets) {
    const int p = buckets <= 1024 ? a.slots / 4096 : 1;
    return p < 1 ? 1 : p > 64 ? 64 : p;
}

// Few slots: a workgroup sums a bucket straight from the slabs (16 x 7 x 7 windows: one launch of 4 us instead of 11 + 4)
#define RS_FEW_SLOTS 2048
__global__ __launch_bounds__(RS_BLOCK) void rs_direct_kernel(RsArgs a) {
    __shared__ double red[RS_BLOCK];
    const int k = blockIdx.x, h = blockIdx.y, t = threadIdx.x;
    double s = 0.0;
    for (int i = a.starts[k]; i < a.starts[k + 1]; ++i) {
        const int slot = a.order[i];
        if ((unsigned)slot < (unsigned)a.slots) s += rs_slot_sum(a, h, slot, t, RS_BLOCK);
    }
    red[t] = s;
    for (int o = RS_BLOCK / 2; o > 0; o >>= 1) {
        __syncthreads();
        if (t < o) red[t] += red[t + o];
    }
    if (t == 0) a.dtable[(long long)k * a.heads + h] = (float)red[0];
}

// ---- host
static int rs_check(RsArgs& a, long long B, int heads, int qh, int qw, int kh, int kw, int buckets, int x_dtype, int dtype) {
    if (!gvfi_dtype_ok(dtype) || (x_dtype != dtype && x_dtype != GVFI_F32)) return -2;
    if (B < 0 || B >= (1LL << 31) || heads <= 0 || heads > 65535 || qh <= 0 || qw <= 0 || kh <= 0 || kw <= 0 || buckets <= 0) return -2;
    const long long Q = (long long)qh * qw, M = (long long)kh * kw, slots = ((long long)qh + kh - 1) * ((long long)qw + kw - 1);
    if (Q >= (1LL << 30) || M >= (1LL << 30) || slots >= (1LL << 30)) return -2;
    a.B = (int)B; a.heads = heads; a.qh = qh; a.qw = qw; a.kh = kh; a.kw = kw; a.Q = (int)Q; a.M = (int)M;
    a.nx = qw + kw - 1; a.slots = (int)slots; a.buckets = buckets;
    a.rows = B * heads * Q;
    a.by_kw = rs_divisor((unsigned)kw); a.by_Q = rs_divisor((unsigned)Q); a.by_heads = rs_divisor((unsigned)heads);
    a.by_qw = rs_divisor((unsigned)qw); a.by_qh = rs_divisor((unsigned)qh);
    a.tiles = M <= RS_LONGEST ? 1 : (int)((M + RS_TILE - 1) / RS_TILE);
    // A launch has fewer than 2^32 lanes: workgroups of 512 for rows in tiles, else T lanes (RS_BY_LENGTH) for 16 rows
    const long long T = a.tiles > 1 ? 512 * 16 : M <= 128 ? 16 : M <= 512 ? 64 : M <= 2048 ? 256 : M <= 8192 ? 512 : 1024;
    return a.rows < (1LL << 31) && a.rows * a.tiles * T < (1LL << 36) ? 0 : -2;
}
// Tile of queries and samples of a workgroup of the backward pass.  More rows per slab spread the cost of clearing, writing and
// reading it again (about 12 bytes per slot against 10 per element of every row); more workgroups fill the chip.
static void rs_backward_plan(RsArgs& a) {
    const bool vec = rs_vec(a);
    const int units = a.M <= 128 ? 16 : 1;                                         // slabs of a workgroup
    const long long target = a.rows / 2048;                                        // rows of a workgroup for 2048 of them
    const long long least = units > 1 ? 64 : 8, most = target < least ? least : target > 256 ? 256 : target;
    const long long nky = a.tiles == 1 ? a.kh : (RS_TILE - 1) / a.kw + 2 < a.kh ? (RS_TILE - 1) / a.kw + 2 : a.kh;   // key rows of a tile
    const long long room = units > 1 ? 1024 : 36 * 1024;                           // floats of LDS of a slab
    const int kw = vec ? (a.kw + 3) / 4 * 4 : a.kw, step = vec ? 4 : 1;
    auto width = [&](long long rx) { return vec ? kw + rx : kw + rx - 1; };        // (vec: whole fours, and the words behind the last chunk)
    auto slab = [&](long long rx, long long ry) {
        return a.tiles > 1 ? RS_TILE + nky * (rx - 1) : (nky + ry - 1) * width(rx);
    };
    long long rx = a.qw < most ? a.qw : most;
    rx = (rx + step - 1) / step * step;
    while (rx > step && slab(rx, 1) > room) rx = ((rx + 1) / 2 + step - 1) / step * step;
    a.RX = (int)rx;
    a.RY = 1;
    if (a.RX >= a.qw && a.tiles == 1)
        while (a.RY < a.qh && (long long)(a.RY + 1) * a.qw <= most && slab(a.RX, a.RY + 1) <= room) ++a.RY;
    a.BC = 1;
    if (a.RX >= a.qw && a.RY == a.qh) {
        const long long bc = most / ((long long)a.qw * a.RY);
        a.BC = (int)(bc < 1 ? 1 : bc < a.B ? bc : a.B);
    }
    a.tx = (a.qw + a.RX - 1) / a.RX;
    a.ty = (a.qh + a.RY - 1) / a.RY;
    a.tb = (a.B + a.BC - 1) / a.BC;
    a.sw = (int)width(a.RX);
    a.slab_n = (int)slab(a.RX, a.RY);
    // workgroups that share the slabs of 16 slots: enough to fill the chip, each with work for its 16 parts
    const long long groups = ((long long)a.slots + 15) / 16 * a.heads, shares = (long long)a.ty * a.tb * ((a.kw + a.RX - 2) / a.RX + 1) / 64;
    long long z = 4096 / groups;
    z = z > shares ? shares : z;
    a.zparts = (int)(z < 1 ? 1 : z > 16 ? 16 : z);
}
// the expanded table with its margins, in whole 16 bytes
static long long rs_bias_floats(const RsArgs& a) { return ((long long)a.heads * a.slots + 2 * RS_MARGIN + 3) / 4 * 4; }
static long long rs_workgroups(const RsArgs& a) { return (long long)a.heads * a.tb * a.ty * a.tx * a.tiles; }
// whether the backward pass is a launch of fewer than 2^32 lanes (workgroups of at most 256 lanes up to 1024 columns, of 512 up to 8192 and
// in tiles, else of 1024)
static bool rs_backward_fits(const RsArgs& a) {
    return rs_workgroups(a) * (a.M <= 1024 ? 256 : a.M <= 8192 || a.tiles > 1 ? 512 : 1024) < (1LL << 32);
}
static long long rs_slab_floats(const RsArgs& a) { return rs_workgroups(a) * a.slab_n; }
extern "C" long long gvfi_softmax_rel_bias_workspace(long long B, int heads, int qh, int qw, int kh, int kw, int backward) {
    RsArgs a = {};
    if (rs_check(a, B, heads, qh, qw, kh, kw, 1, GVFI_F32, GVFI_F32)) return -2;
    const long long nb = rs_bias_floats(a), np = a.tiles > 1 ? a.rows * a.tiles * 2 : 0;
    if (!backward || B == 0) return nb + np;
    rs_backward_plan(a);
    if (!rs_backward_fits(a)) return -2;
    return nb + 2LL * a.zparts * heads * a.slots + 1 + np + rs_slab_floats(a) + (a.slots < 8192 ? 0 : RS_SHARES * 2LL * heads);
}
#define RS_DISPATCH(...)                                                                              \
    do {                                                                                              \
        if (x_dtype == GVFI_F32) GVFI_DISPATCH_T(dtype, typedef float TX; typedef T TY; __VA_ARGS__); \
        else if (dtype == GVFI_F16) { typedef f16_t TX; typedef f16_t TY; __VA_ARGS__; }              \
        else { typedef bf16_t TX; typedef bf16_t TY; __VA_ARGS__; }                                   \
    } while (0)
extern "C" int gvfi_softmax_rel_bias(const void* x, int x_dtype, long long ldx, const float* table, const int* bucket_of, int buckets,
                                     const unsigned char* key_mask, float scale, void* y, long long ldy, int zero_to, float* stats,
                                     long long B, int heads, int qh, int qw, int kh, int kw, float* workspace, int dtype,
                                     void* stream) {
    RsArgs a = {};
    if (rs_check(a, B, heads, qh, qw, kh, kw, buckets, x_dtype, dtype)) return -2;
    if (B == 0) return 0;
    if (!x || !y || !table || !bucket_of || !workspace || ldx < a.M || ldy < a.M || zero_to < a.M || zero_to > ldy) return -2;
    a.x = x; a.ldx = ldx; a.y = y; a.ldy = ldy; a.zero_to = zero_to; a.table = table; a.bucket_of = bucket_of;
    a.mask = key_mask; a.stats = stats; a.scale = scale; a.bias = workspace + RS_MARGIN;
    hipStream_t st = (hipStream_t)stream;
    a.part = workspace + rs_bias_floats(a);
    GVFI_LAUNCH_SIMPLE(rs_expand_kernel, dim3((unsigned)((a.slots + RS_BLOCK - 1) / RS_BLOCK), (unsigned)heads), dim3(RS_BLOCK), st, a, workspace + RS_MARGIN);
    RS_DISPATCH((rs_forward_launch<TX, TY>(a, st)));
    return (int)hipGetLastError();
}
extern "C" int gvfi_softmax_rel_bias_backward(const void* dy, long long lddy, const void* x, int x_dtype, long long ldx,
                                              const float* table, const int* bucket_of, int buckets, const int* order,
                                              const int* starts, const unsigned char* key_mask, float scale, const float* stats,
                                              void* dx, long long lddx, float* dtable, long long B, int heads, int qh, int qw, int kh,
                                              int kw, float* workspace, int dtype, void* stream) {
    RsArgs a = {};
    if (rs_check(a, B, heads, qh, qw, kh, kw, buckets, x_dtype, dtype)) return -2;
    if (B == 0) return 0;
    if (!x || !dy || !dx || !table || !bucket_of || !stats || !workspace || ldx < a.M || lddy < a.M || lddx < a.M) return -2;
    if (dtable && (!order || !starts)) return -2;
    rs_backward_plan(a);
    if (!rs_backward_fits(a)) return -2;
    a.x = x; a.ldx = ldx; a.dy = dy; a.lddy = lddy; a.y = dx; a.ldy = lddx; a.zero_to = a.M; a.table = table;
    a.bucket_of = bucket_of; a.mask = key_mask; a.stats = (float*)stats; a.scale = scale; a.dtable = dtable;
    a.order = order; a.starts = starts;
    const long long nb = rs_bias_floats(a), np = a.tiles > 1 ? a.rows * a.tiles * 2 : 0;
    a.bias = workspace + RS_MARGIN; a.slab = workspace + nb; a.part = a.slab + rs_slab_floats(a);
    a.dslot = (double*)(((uintptr_t)(a.part + np) + 7) & ~(uintptr_t)7);
    double* share = a.dslot + (long long)a.zparts * heads * a.slots;      // (where rs_parts may be above 1)
    hipStream_t st = (hipStream_t)stream;
    GVFI_LAUNCH_SIMPLE(rs_expand_kernel, dim3((unsigned)((a.slots + RS_BLOCK - 1) / RS_BLOCK), (unsigned)heads), dim3(RS_BLOCK), st, a, workspace + RS_MARGIN);
    RS_DISPATCH((rs_backward_launch<TX, TY>(a, st)));
    if (dtable && a.slots <= RS_FEW_SLOTS && a.slots / buckets < 8 && buckets <= 4096 && (long long)a.ty * a.tb >= 64) {
        GVFI_LAUNCH_COOP(rs_direct_kernel, dim3((unsigned)buckets, (unsigned)heads), dim3(RS_BLOCK), st, a);
    } else if (dtable) {
        GVFI_LAUNCH_COOP(rs_slots_kernel, dim3(rs_groups((a.slots + 15LL) / 16), (unsigned)heads, (unsigned)a.zparts), dim3(RS_BLOCK), st, a);
        if (buckets <= 1024) {
            const int parts = rs_parts(a, buckets);
            GVFI_LAUNCH_COOP((rs_buckets_kernel<RS_BLOCK>), dim3(rs_groups((long long)buckets * parts), (unsigned)heads), dim3(RS_BLOCK), st, a, parts,
                             share);
            if (parts > 1)
                GVFI_LAUNCH_SIMPLE(rs_shares_kernel, dim3((unsigned)(((long long)buckets * heads + RS_BLOCK - 1) / RS_BLOCK)), dim3(RS_BLOCK), st,
                                   a, parts, (const double*)share);
        } else {
            GVFI_LAUNCH_COOP((rs_buckets_kernel<16>), dim3(rs_groups((buckets + 15LL) / 16), (unsigned)heads), dim3(RS_BLOCK), st, a, 1, share);
        }
    }
    return (int)hipGetLastError();
}
