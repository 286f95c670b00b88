// Group norm with an activation: the C ABI, the kernels without an element type, the choice of form (group_norm.h has the rest).
#include "group_norm.h"

// sum over the workgroup, in every lane, in double
__device__ __forceinline__ double gn_block_sum(double v, double* red) {
    __syncthreads();
    red[threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.x < 16) {
        v = 0.0;
#pragma unroll
        for (int k = 0; k < GN_BLOCK / 16; ++k) v += red[threadIdx.x + 16 * k];
        red[threadIdx.x] = v;
    }
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int k = 0; k < 16; ++k) v += red[k];
    return v;
}

// joins the chunks of a group, and its channels where they come one by one (cols = C values per chunk, `per_group` of them a group's)
__global__ __launch_bounds__(GN_BLOCK) void gn_stats_kernel(const float* part, float* stats, long long HW, long long per, int cols,
                                                            int G, int per_group, int Cg, int chunks, float eps) {
    __shared__ double red[GN_BLOCK];
    const int n = blockIdx.x / G, g = blockIdx.x - n * G;
    const float* w = part + (long long)n * chunks * 2 * cols + g * per_group;
    const long long items = (long long)chunks * per_group;
    const double share = (double)(Cg / per_group);           // values of a pixel in an item
    double s = 0.0;
    for (long long i = threadIdx.x; i < items; i += GN_BLOCK) {
        const long long k = per_group == 1 ? i : i / per_group;
        const double cnt = share * (double)(k + 1 < chunks ? per : HW - k * per);
        s += cnt * (double)w[k * 2 * cols + (i - k * per_group)];
    }
    const double m = (double)HW * (double)Cg;
    const double mean = gn_block_sum(s, red) / m;
    double q = 0.0;
    for (long long i = threadIdx.x; i < items; i += GN_BLOCK) {
        const long long k = per_group == 1 ? i : i / per_group;
        const double cnt = share * (double)(k + 1 < chunks ? per : HW - k * per);
        const double d = (double)w[k * 2 * cols + (i - k * per_group)] - mean;
        q += (double)w[(k * 2 + 1) * cols + (i - k * per_group)] + cnt * d * d;
    }
    const float var = (float)(gn_block_sum(q, red) / m);
    if (threadIdx.x == 0) {
        stats[((long long)n * G + g) * 2] = (float)mean;
        stats[((long long)n * G + g) * 2 + 1] = 1.f / sqrtf(var + eps);
    }
}

// sums of an image's channels over its chunks, and A, B of the group
__global__ __launch_bounds__(GN_BLOCK) void gn_bwd_group_kernel(GnArgs a) {
    __shared__ double sh[2][GN_BLOCK];
    const int n = blockIdx.x / a.G, g = blockIdx.x - n * a.G;
    int cp = 1;                                     // channels side by side, the chunks in GN_BLOCK / cp parts
    while (cp < a.Cg && cp < GN_BLOCK) cp <<= 1;
    const int cl = threadIdx.x & (cp - 1), part = threadIdx.x / cp, parts = GN_BLOCK / cp;
    const float* w = a.part + (long long)n * a.chunks * 2 * a.C + g * a.Cg;
    double ga = 0.0, gb = 0.0;
    for (int cb = 0; cb < a.Cg; cb += cp) {
        const int c = cb + cl;
        double s = 0.0, q = 0.0;
        if (c < a.Cg)
            for (int k = part; k < a.chunks; k += parts) {
                s += (double)w[(long long)k * 2 * a.C + c];
                q += (double)w[((long long)k * 2 + 1) * a.C + c];
            }
        __syncthreads();
        sh[0][threadIdx.x] = s;
        sh[1][threadIdx.x] = q;
        __syncthreads();
        if (part == 0 && c < a.Cg) {
            s = q = 0.0;
            for (int k = 0; k < parts; ++k) {
                s += sh[0][k * cp + cl];
                q += sh[1][k * cp + cl];
            }
            const int cc = g * a.Cg + c;
            a.sums[(long long)n * 2 * a.C + cc] = (float)s;
            a.sums[((long long)n * 2 + 1) * a.C + cc] = (float)q;
            const double gm = a.gamma ? (double)a.gamma[cc] : 1.0;
            ga += gm * s;
            gb += gm * q;
        }
    }
    ga = gn_block_sum(ga, sh[0]);
    gb = gn_block_sum(gb, sh[1]);
    if (threadIdx.x == 0) {
        const double m = (double)a.HW * (double)a.Cg;
        a.ab[((long long)n * a.G + g) * 2] = (float)(ga / m);
        a.ab[((long long)n * a.G + g) * 2 + 1] = (float)(gb / m);
    }
}

// Steps of the parameters' gradients (gn_params_part): a step leaves one row of sums per GN_IMAGES of the rows before it
__global__ __launch_bounds__(GN_BLOCK) void gn_params_kernel(const float* sums, long long rows, int C, float* out, float* dgamma,
                                                             float* dbeta) {
    gn_params_part(blockIdx.x, sums, rows, C, out, dgamma, dbeta);
}
static void gn_params(const GnArgs& a, hipStream_t st) {
    const float* from = a.sums;
    float* to = a.part;                                      // (the chunks' sums are used up: N * 2 * C floats at least)
    long long rows = a.N;
    for (;;) {
        const long long next = (rows + GN_IMAGES - 1) / GN_IMAGES;
        const dim3 grid((unsigned)((a.C + 15) / 16 * next));
        GVFI_LAUNCH_COOP(gn_params_kernel, grid, dim3(GN_BLOCK), st, from, rows, a.C, next > 1 ? to : nullptr, a.dgamma, a.dbeta);
        if (next == 1) return;
        from = to;
        to = to == a.part ? a.sums : a.part;
        rows = next;
    }
}

void gn_launch_stats(const GnArgs& a, float* stats, float eps, hipStream_t st) {
    GVFI_LAUNCH_COOP(gn_stats_kernel, dim3((unsigned)a.N * (unsigned)a.G), dim3(GN_BLOCK), st, (const float*)a.part, stats, a.HW, a.per,
                     a.whole ? a.G : a.C, a.G, a.whole ? 1 : a.Cg, a.Cg, a.chunks, eps);
}
void gn_launch_group(const GnArgs& a, hipStream_t st) {
    GVFI_LAUNCH_COOP(gn_bwd_group_kernel, dim3((unsigned)a.N * (unsigned)a.G), dim3(GN_BLOCK), st, a);
}

// ---- host
static int gn_check(int C, int G, long long N, long long HW, int act, int dtype) {
    if (!gvfi_dtype_ok(dtype) || C <= 0 || C > (1 << 24) || G <= 0 || C % G || N < 0 || HW < 0) return -2;
    if (act < 0 || act == GVFI_ACT_PRELU || act == GVFI_ACT_SIN || act > GVFI_ACT_SILU) return -2;
    return 0;
}
// Pixels per workgroup: as many workgroups as the CUs hold at once (five of the applying kernels on each; a second round for the rest
// costs more than a longer first one), at least two octets per lane and at most GN_FOLD * GN_MOST
#ifndef GVFI_HOSTSIM
#define GN_WORKGROUPS 1280
#else
#define GN_WORKGROUPS 16        // (the emulator's tests reach long chunks)
#endif
static bool gn_plan(GnArgs& a) {
    const int oct = (a.C + 7) / 8, o = oct < GN_MAXOCT ? oct : GN_MAXOCT;
    a.octp = 1;
    while (a.octp < o) a.octp <<= 1;
    const long long lanes = GN_BLOCK / a.octp, zs = (oct + GN_MAXOCT - 1) / GN_MAXOCT;
    const long long images = a.N > 0 ? (long long)a.N * zs : 1;
    long long want = (GN_WORKGROUPS + images - 1) / images;                       // chunks of an image
    long long per = (a.HW + want - 1) / want;
    if (per < lanes * 2) per = lanes * 2;
    if (per > lanes * GN_FOLD * GN_MOST) per = lanes * GN_FOLD * GN_MOST;
    a.per = (per + lanes - 1) / lanes * lanes;
    const long long chunks = (a.HW + a.per - 1) / a.per;
    if (chunks >= (1LL << 23)) return false;
    a.chunks = (int)chunks;
    a.whole = a.C <= GN_MAXOCT * 8 || GN_MAXOCT * 8 % (a.C / a.G) == 0;
    // (a launch has fewer than 2^32 lanes: 2^23 workgroups of 512, the images of the one-launch form rounded up to eights; 2^24 of 256
    // in gn_params)
    const long long n = a.N;
    return n * a.chunks < (1LL << 23) && (n + 7) * a.G < (1LL << 23) && (a.C + 15) / 16 * ((n + GN_IMAGES - 1) / GN_IMAGES) < (1LL << 24);
}
// Groups of a workgroup of the one-launch form, and the octets of a lane (0: the image does not fit, or streaming is faster; bytes: what the
// pass reads).  As few groups as give whole
// octets while the workgroups are few (every workgroup's share is latency then); more, for longer runs of bytes, while there are
// more than 1024 of them.
static int gn_slab_plan(const GnArgs& a, int most, double bytes, GnSlab& b, int& threads) {
    int g = 1;
    while (g < a.G && (g * a.Cg) % 8) ++g;
    if ((g * a.Cg) % 8) return 0;
    while ((long long)a.N * ((a.G + 2 * g - 1) / (2 * g)) >= 1024 && 2 * g * a.Cg <= 64 && 2 * g <= a.G) g *= 2;
    b.gpb = g;
    b.oct = g * a.Cg / 8;
    if (b.oct > 16) return 0;
    b.octp = 1;
    while (b.octp < b.oct) b.octp <<= 1;
    b.runs = (a.G + g - 1) / g;
    b.images8 = a.N >= 8 ? (a.N + 7) / 8 : 0;
    threads = a.HW * b.octp <= 1024 ? 256 : 512;
    const long long r = (a.HW * b.octp + threads - 1) / threads;
    // Up to 4 octets of a lane (a workgroup's time is then below that of the other launches of the streaming form) always: 16 x 448 pixels x 128
    // bfloat16 channels 12.6 us against 18.3, 8 x 2048 x 256 12.8 against 23.3 (forward with the call; backward likewise).  More only where not
    // reading twice pays although a workgroup takes 16 bytes of every pixel and its neighbours the rest of the same lines:
    //   workgroups for half of the CUs    8 images x 7168 x 32 channels, 32 workgroups, backward 26.3 against 19.8; from 128 on 33.8 against 43.1
    //   a whole image on one XCD          (8 images, dealt) else every XCD fetches the lines: 6 x 7168 x 512 channels 91.8 against 40.5, 4 x 7168 x
    //                                     512 57.3 against 35.1; 8 x 7168 x 512 42.6 against 45.3
    //   XCDs with the same load           9 images x 7168 x 512 72.4 against 50.0 (seven XCDs wait for the one with two)
    //   128 MB read at most               what the last-level cache holds between one run's visit to a line and the next: 32 x 7168 x 128 (58 MB)
    //                                     forward 39.9 against 45.2, backward (117 MB) 71.9 against 78.0; 64 x 7168 x 128 backward (235 MB) 174
    //                                     against 130
    if (r > 4 && ((long long)a.N * b.runs < 128 || a.N < 8 || 4LL * a.N < 3 * 8 * b.images8 || bytes > 128e6)) return 0;
    return r <= most ? (int)r : 0;
}
extern "C" long long gvfi_group_norm_workspace(int C, int G, long long N, long long HW) {
    if (gn_check(C, G, N, HW, 0, GVFI_F32) || N >= (1LL << 30)) return -2;
    GnArgs a;
    a.C = C; a.G = G; a.N = (int)N; a.HW = HW;
    if (!gn_plan(a)) return -2;
    return N * a.chunks * 2 * C + N * 2 * C + N * 2 * G;
}
extern "C" int gvfi_group_norm(const void* x, long long ldx, int C, int G, long long N, long long HW, const float* gamma,
                               const float* beta, float eps, int act, void* y, long long ldy, float* stats, float* workspace,
                               int dtype, void* stream) {
    if (gn_check(C, G, N, HW, act, dtype)) return -2;
    if (N == 0 || HW == 0) return 0;
    if (!x || !y || !stats || !workspace || ldx < C || ldy < C) return -2;
    GnArgs a = {};
    a.x = x; a.ldx = ldx; a.y = y; a.ldy = ldy; a.gamma = gamma; a.beta = beta; a.stats = stats; a.part = workspace;
    a.HW = HW; a.C = C; a.G = G; a.Cg = C / G; a.N = (int)N; a.act = gn_act_of(act);
    if (N >= (1LL << 30) || !gn_plan(a)) return -2;
    const int es = gvfi_esize(dtype);
    const bool al = C % 8 == 0 && gvfi_rows_aligned(x, ldx, es) && gvfi_rows_aligned(y, ldy, es);
    GnSlab b = {};
    int threads = 0;
    const int r = al ? gn_slab_plan(a, dtype == GVFI_F32 ? 8 : 16, (double)N * HW * C * es, b, threads) : 0;
    GVFI_DISPATCH_T(dtype, gn_forward_launch<T>(a, b, threads, r, al, stats, eps, (hipStream_t)stream));
    return (int)hipGetLastError();
}
extern "C" int gvfi_group_norm_backward(const void* dy, long long lddy, const void* x, long long ldx, int C, int G, long long N,
                                        long long HW, const float* gamma, const float* beta, const float* stats, int act, void* dx,
                                        long long lddx, float* dgamma, float* dbeta, float* workspace, int dtype, void* stream) {
    if (gn_check(C, G, N, HW, act, dtype)) return -2;
    if (N == 0 || HW == 0) return 0;
    if (!x || !dy || !dx || !stats || !workspace || ldx < C || lddy < C || lddx < C) return -2;
    GnArgs a = {};
    a.x = x; a.ldx = ldx; a.dy = dy; a.lddy = lddy; a.y = dx; a.ldy = lddx; a.gamma = gamma; a.beta = beta; a.stats = stats;
    a.HW = HW; a.C = C; a.G = G; a.Cg = C / G; a.N = (int)N; a.act = gn_act_of(act); a.dgamma = dgamma; a.dbeta = dbeta;
    if (N >= (1LL << 30) || !gn_plan(a)) return -2;
    a.part = workspace;
    a.sums = workspace + N * a.chunks * 2 * C;
    a.ab = a.sums + N * 2 * C;
    const int es = gvfi_esize(dtype);
    const bool al = C % 8 == 0 && gvfi_rows_aligned(x, ldx, es) && gvfi_rows_aligned(dy, lddy, es) && gvfi_rows_aligned(dx, lddx, es);
    GnSlab b = {};
    int threads = 0;
    const int r = al ? gn_slab_plan(a, dtype == GVFI_F32 ? 8 : 16, (double)N * HW * C * es * 2, b, threads) : 0;
    hipStream_t st = (hipStream_t)stream;
    GVFI_DISPATCH_T(dtype, gn_backward_launch<T>(a, b, threads, r, al, st));
    if ((dgamma || dbeta) && (r || N > GN_IMAGES)) gn_params(a, st);       // (else the last launch above has done it)
    return (int)hipGetLastError();
}
