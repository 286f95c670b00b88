// Group norm with an activation, channels last, forward and backward.
//
//   xhat = (x - mean) * rstd over the m = HW * C/G values of a group of one image,  z = xhat * gamma + beta,  y = act(z)
//   dz = dy * act'(z),  dbeta = sum dz,  dgamma = sum dz * xhat,
//   dx = rstd * (gamma dz - A - xhat B),  A = mean over the group of gamma dz,  B = mean over the group of gamma dz xhat
//
// The work is a few operations per element: bytes bind.  A workgroup covers a run of pixels of one image and up to 64 octets of
// channels; a lane keeps its octet, so everything that depends on the channel stays in registers.  Statistics: for every GN_FOLD pixels a
// lane sums x - k and (x - k)^2 with k the first of these values -- k is one of the values, so (k - mean)^2 <= M2 and the difference
// sum (x-k)^2 - (sum (x-k))^2 / n loses at most a factor GN_FOLD + 1, whatever the mean.  Means and centred sums
// (M2 = sum (x - mean)^2) are then joined as  mean = sum n_i mean_i / n,  M2 = sum M2_i + n_i (mean_i - mean)^2, always in the same
// order: two runs give the same bits.  No chain of float additions is longer than GN_FOLD + GN_MOST: a lane folds its sums every GN_FOLD
// pixels and has at most GN_FOLD * GN_MOST of them, the sums over chunks are in double.
//
// Measured on one MI355X, whose copy of 1 GiB reaches 5.2 TB/s.  Streaming form, 16 images of 128 x 224 x 64 bfloat16 with ReLU: sums
// 15.1 us (3.9 TB/s), joining 3.9, applying 24.6 (4.8 TB/s, part of its reads from the caches); a training step 121 us, of 2 images of
// 1088 x 1920 x 64 907 us (eight passes over 535 MB: 4.7 TB/s).  One-launch form, 16 images of 64 x 112 x 96 bfloat16 with SiLU: forward 26 us, backward 36
// (44 and 66 MB): every lane takes 16 bytes of a 192-byte pixel, so a line of 128 bytes is asked of the L2 eight times (1.38 M and 2.75 M
// requests), and the L1 waits for them 0.6 and 0.55 of the time; vector instructions fill 0.4 and 0.5.  2 images of 16 x 28 x 128: 6.2.
#pragma once
#include "row_ops.h"

#define GN_BLOCK 256
#define GN_MAXOCT 64           // octets of a workgroup: 512 channels
#define GN_U 4                 // pixels of a lane in flight, forward
#define GN_UB 2                // ... and backward (two tensors)
#define GN_FOLD 64             // pixels of a lane whose sums are added up before they are joined with its others
#define GN_MOST 64             // such runs of a lane

// Activations in four classes, so that a kernel holds the code of one and no branch per element:
//   0  max(z, 0) + p0 min(z, 0): none (1), ReLU (0), LeakyReLU (0.1)
//   1  sigmoid s(z), and SiLU = z s(z) (p0 = 1)
//   2  GELU (erf)
//   3  tanh
// Every value and derivative is accurate relative to itself, not to 1: a small tanh, a far tail of GELU or a saturated sigmoid's derivative
// keeps its digits (but for a derivative's own zero crossing).  float tensors take the library's exponential, erfc, tanh and an exact
// division: the value's error is a few steps.  Tensors of 16 bits take 2^t and 1 / x of the hardware and an erfc of this file, together below
// 2^-16 of the value, where half's own rounding is up to 2^-11: the library's functions cost five times the instructions, which the
// backward pass of a 16-bit tensor was bound by.
struct GnAct { int cls; float p0; };
static inline GnAct gn_act_of(int act) {
    switch (act) {
        case GVFI_ACT_RELU: return {0, 0.f};
        case GVFI_ACT_LRELU: return {0, 0.1f};
        case GVFI_ACT_SIGMOID: return {1, 0.f};
        case GVFI_ACT_SILU: return {1, 1.f};
        case GVFI_ACT_GELU: return {2, 0.f};
        case GVFI_ACT_TANH: return {3, 0.f};
        default: return {0, 1.f};
    }
}
// 1 / x and exp(-x) for tensors of type T
template <typename T> __device__ __forceinline__ float gn_rcp(float x) {
#ifndef GVFI_HOSTSIM
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_rcpf(x);
#endif
    return 1.f / x;
}
template <typename T> __device__ __forceinline__ float gn_exp_neg(float x) {
    if constexpr (sizeof(T) == 2) return exp2_hw(x * -1.44269504f);
    else return expf(-x);
}
// with e = exp(-|z|): r = 1 / (1 + e) is s(|z|), e r is s(-|z|), and the derivative of s is their product at either sign
struct GnSig { float s, slope; };
template <typename T> __device__ __forceinline__ GnSig gn_sig(float z) {
    const float e = gn_exp_neg<T>(fabsf(z)), r = gn_rcp<T>(1.f + e);
    return {z < 0.f ? e * r : r, e * r * r};
}
// Phi(z) = erfc(-z / sqrt 2) / 2 and phi(z) = exp(-z^2 / 2) / sqrt(2 pi).  For 16 bits erfc(x) exp(x^2) on x >= 0 is a polynomial in
// t = 1 / (1 + 0.44 x), fitted over [0, 9.5] to the least largest relative error, 5.2e-6 = 2^-17.5
template <typename T> __device__ __forceinline__ void gn_phi(float z, float& cdf, float& pdf) {
    if constexpr (sizeof(T) == 4) {
        cdf = 0.5f * erfcf(z * -0.70710678118654752f);
        pdf = 0.3989422804014327f * expf(-0.5f * z * z);
    } else {
        const float x = fabsf(z) * 0.70710678118654752f;
        const float t = gn_rcp<T>(fmaf(0.44f, x, 1.f));
        const float e = gn_exp_neg<T>(x * x);
        float h = fmaf(t, -0.14610421f, 0.35064869f);
        h = fmaf(t, h, 0.04073489f);
        h = fmaf(t, h, 0.26358454f);
        h = fmaf(t, h, 0.24256996f);
        h = fmaf(t, h, 0.24856098f) * (0.5f * t) * e;
        cdf = z < 0.f ? h : 1.f - h;
        pdf = 0.3989422804014327f * e;
    }
}
// tanh(z) = (1 - e) / (1 + e), e = exp(-2 |z|); below 1/8, where 1 - e loses digits, z - z^3 / 3 + 2 z^5 / 15 (the next term is 17 z^6 / 315 of it)
template <typename T> __device__ __forceinline__ float gn_tanh(float z) {
    if constexpr (sizeof(T) == 4) return tanhf(z);
    const float a = fabsf(z), e = gn_exp_neg<T>(2.f * a), q = z * z;
    const float far = copysignf((1.f - e) * gn_rcp<T>(1.f + e), z), near = z * fmaf(q, fmaf(q, 2.f / 15.f, -1.f / 3.f), 1.f);
    return a < 0.125f ? near : far;
}
template <typename T, int CLS> __device__ __forceinline__ float gn_act(float z, const GnAct& f) {
    if constexpr (CLS == 0) return z > 0.f ? z : f.p0 == 0.f ? (z != z ? z : 0.f) : z * f.p0;
    else if constexpr (CLS == 1) {
        const float s = gn_sig<T>(z).s;
        return f.p0 == 0.f ? s : z * s;
    } else if constexpr (CLS == 2) {
        float cdf, pdf;
        gn_phi<T>(z, cdf, pdf);
        return z * cdf;
    } else return gn_tanh<T>(z);
}
template <typename T, int CLS> __device__ __forceinline__ float gn_slope(float z, const GnAct& f) {
    if constexpr (CLS == 0) return z > 0.f ? 1.f : z != z ? z : f.p0;
    else if constexpr (CLS == 1) {
        const GnSig g = gn_sig<T>(z);
        return f.p0 == 0.f ? g.slope : fmaf(z, g.slope, g.s);
    } else if constexpr (CLS == 2) {
        float cdf, pdf;
        gn_phi<T>(z, cdf, pdf);
        return fmaf(z, pdf, cdf);
    } else return 4.f * gn_sig<T>(2.f * z).slope;
}

struct GnArgs {
    const void* x; long long ldx;
    const void* dy; long long lddy;
    void* y; long long ldy;          // output: y, or dx in the backward pass
    const float* gamma; const float* beta;
    const float* stats;              // [N][G][2] mean, rstd
    float* part;                     // [N][chunks][2][C], or [N][chunks][2][G] where a workgroup covers whole groups (forward)
    float* sums;                     // [N][2][C]     (backward: sum dz, sum dz xhat)
    float* ab;                       // [N][G][2]     (backward: A, B)
    float* dgamma; float* dbeta;
    long long HW, per;               // pixels of an image, pixels of a chunk
    int C, G, Cg, N, chunks, whole, octp;   // whole: workgroups cover whole groups; octp: their octets
                                     // rounded up to a power of two
    GnAct act;
};

// sum of v[8] over the pixel lanes of an octet, in every lane; red: [4 waves][octp * 8] floats
__device__ __forceinline__ void gn_reduce(float (&v)[8], int octp, float* red) {
    for (int off = octp; off < 64; off <<= 1)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += __shfl_xor(v[e], off);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    __syncthreads();
    if (lane < octp)
#pragma unroll
        for (int e = 0; e < 8; ++e) red[(w * GN_MAXOCT + lane) * 8 + e] = v[e];
    __syncthreads();
    const int o = threadIdx.x & (octp - 1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < GN_BLOCK / 64; ++k) s += red[(k * GN_MAXOCT + o) * 8 + e];
        v[e] = s;
    }
}

template <typename T, bool AL> __global__ __launch_bounds__(GN_BLOCK) void gn_partial_kernel(GnArgs a) {
    constexpr int U = GN_U;
    __shared__ float red[GN_BLOCK / 64 * GN_MAXOCT * 8];
    __shared__ float kept[16][GN_BLOCK];           // what a lane has joined so far: mean, M2 (in registers they would cost a third of the waves)
    const int o = threadIdx.x & (a.octp - 1), pl = threadIdx.x / a.octp, lanes = GN_BLOCK / a.octp;
    const int c0 = (blockIdx.y * GN_MAXOCT + o) * 8;
    const int nv = a.C - c0 < 8 ? a.C - c0 : 8;
    const int n = blockIdx.x / a.chunks, chunk = blockIdx.x - n * a.chunks;
    const long long p0 = (long long)chunk * a.per;
    const long long p1 = p0 + a.per < a.HW ? p0 + a.per : a.HW;
    const T* x = (const T*)a.x + (long long)n * a.HW * a.ldx + c0;
    float k[8], s[8], q[8], mean[8], m2[8], tot[8], n1 = 0.f, cnt = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) k[e] = s[e] = q[e] = 0.f;
    // joins the sums (s, q) of n1 pixels to what `kept` has of cnt pixels
    auto join = [&]() {
        const float in = n1 > 0.f ? 1.f / n1 : 0.f, f = n1 / (cnt + n1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            m2[e] = fmaxf(q[e] - s[e] * s[e] * in, 0.f);
            if (q[e] != q[e]) m2[e] = q[e];
            mean[e] = k[e] + s[e] * in;
            if (cnt > 0.f) {
                const float mk = kept[e][threadIdx.x], d = mean[e] - mk;
                mean[e] = n1 > 0.f ? fmaf(d, f, mk) : mk;
                m2[e] = kept[8 + e][threadIdx.x] + (n1 > 0.f ? fmaf(d * d, cnt * f, m2[e]) : 0.f);
            }
        }
        cnt += n1;
    };
    if (nv > 0 && p0 + pl < p1) {
        long long pivot = p0 + pl;
        load8<T, AL>(x + pivot * a.ldx, nv, k);
        int turns = 0;
        for (long long p = p0 + pl; p < p1; p += U * lanes) {
            float v[U][8];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long r = p + u * lanes;
                load8<T, AL>(x + (r < p1 ? r : pivot) * a.ldx, nv, v[u]);          // (past the end: the pivot again, difference 0)
                n1 += r < p1 ? 1.f : 0.f;
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float d = v[u][e] - k[e];
                    s[e] += d;
                    q[e] = fmaf(d, d, q[e]);
                }
            if (++turns == GN_FOLD / U) {
                join();
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    kept[e][threadIdx.x] = mean[e];
                    kept[8 + e][threadIdx.x] = m2[e];
                    s[e] = q[e] = 0.f;
                }
                n1 = 0.f;
                turns = 0;
                if (p + U * lanes < p1) {
                    pivot = p + U * lanes;
                    load8<T, AL>(x + pivot * a.ldx, nv, k);
                }
            }
        }
    }
    join();
#pragma unroll
    for (int e = 0; e < 8; ++e) tot[e] = mean[e] * cnt;
    gn_reduce(tot, a.octp, red);
    const float in = 1.f / (float)(p1 - p0);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        tot[e] *= in;
        const float d = mean[e] - tot[e];
        m2[e] += cnt * d * d;
    }
    gn_reduce(m2, a.octp, red);
    if (!a.whole) {
        if (pl == 0) {
            float* w = a.part + (long long)blockIdx.x * 2 * a.C + c0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < nv) {
                    w[e] = tot[e];
                    w[a.C + e] = m2[e];
                }
        }
        return;
    }
    // the channels of a group (all of them have p1 - p0 values)
    __syncthreads();
    float* mc = red;
    float* qc = red + GN_MAXOCT * 8;
    if (pl == 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            mc[o * 8 + e] = tot[e];
            qc[o * 8 + e] = m2[e];
        }
    __syncthreads();
    const int cb = blockIdx.y * GN_MAXOCT * 8, ng = ((a.C - cb < GN_MAXOCT * 8 ? a.C - cb : GN_MAXOCT * 8)) / a.Cg;
    float* w = a.part + (long long)blockIdx.x * 2 * a.G + cb / a.Cg;
    const float cn = (float)(p1 - p0), ig = 1.f / (float)a.Cg;
    if (a.Cg <= 16) {
        for (int g = threadIdx.x; g < ng; g += GN_BLOCK) {
            float mean = 0.f, q2 = 0.f;
            for (int c = 0; c < a.Cg; ++c) mean += mc[g * a.Cg + c];
            mean *= ig;
            for (int c = 0; c < a.Cg; ++c) {
                const float d = mc[g * a.Cg + c] - mean;
                q2 += qc[g * a.Cg + c] + cn * d * d;
            }
            w[g] = mean;
            w[a.G + g] = q2;
        }
    } else {
        const int lane = threadIdx.x & 63;
        for (int g = threadIdx.x >> 6; g < ng; g += GN_BLOCK / 64) {
            float mean = 0.f, q2 = 0.f;
            for (int c = lane; c < a.Cg; c += 64) mean += mc[g * a.Cg + c];
            mean = wave_sum(mean) * ig;
            for (int c = lane; c < a.Cg; c += 64) {
                const float d = mc[g * a.Cg + c] - mean;
                q2 += qc[g * a.Cg + c] + cn * d * d;
            }
            q2 = wave_sum(q2);
            if (lane == 0) {
                w[g] = mean;
                w[a.G + g] = q2;
            }
        }
    }
}

// The pass that comes second takes the workgroups backwards: what the first pass read last is still in the caches.  By eights, so that a
// chunk stays with its XCD and that XCD's L2.
__device__ __forceinline__ unsigned gn_backwards(unsigned n) {
    const unsigned n8 = n >> 3 << 3, i = blockIdx.x;
    return i < n8 ? n8 - 8 - (i & ~7u) + (i & 7u) : i;
}

// what a lane keeps of its octet's channels
struct GnChan { float mean[8], rstd[8], k[8], be[8]; };          // z = (x - mean) * k + beta, k = rstd * gamma
__device__ __forceinline__ void gn_channels(const GnArgs& a, int n, int c0, int nv, GnChan& ch) {
    int g = c0 / a.Cg, left = (g + 1) * a.Cg - c0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int c = e < nv ? c0 + e : 0;
        const float* st = a.stats + ((long long)n * a.G + (e < nv ? g : 0)) * 2;
        if (--left == 0) { ++g; left = a.Cg; }
        ch.mean[e] = st[0];
        ch.rstd[e] = st[1];
        ch.k[e] = a.gamma ? st[1] * a.gamma[c] : st[1];
        ch.be[e] = a.beta ? a.beta[c] : 0.f;
    }
}

template <typename T, bool AL, int CLS> __global__ __launch_bounds__(GN_BLOCK) void gn_apply_kernel(GnArgs a) {
    const int o = threadIdx.x & (a.octp - 1), pl = threadIdx.x / a.octp, lanes = GN_BLOCK / a.octp;
    const int c0 = (blockIdx.y * GN_MAXOCT + o) * 8;
    const int nv = a.C - c0 < 8 ? a.C - c0 : 8;
    if (nv <= 0) return;
    const unsigned blk = gn_backwards((unsigned)a.N * (unsigned)a.chunks);
    const int n = blk / a.chunks, chunk = blk - n * a.chunks;
    GnChan ch;
    gn_channels(a, n, c0, nv, ch);
    const long long p0 = (long long)chunk * a.per;
    const long long p1 = p0 + a.per < a.HW ? p0 + a.per : a.HW;
    const T* x = (const T*)a.x + (long long)n * a.HW * a.ldx + c0;
    T* y = (T*)a.y + (long long)n * a.HW * a.ldy + c0;
    for (long long p = p0 + pl; p < p1; p += GN_U * lanes) {
        float v[GN_U][8];
#pragma unroll
        for (int u = 0; u < GN_U; ++u)
            if (p + u * lanes < p1) load8<T, AL>(x + (p + u * lanes) * a.ldx, nv, v[u]);
#pragma unroll
        for (int u = 0; u < GN_U; ++u)
            if (p + u * lanes < p1) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[u][e] = gn_act<T, CLS>(fmaf(v[u][e] - ch.mean[e], ch.k[e], ch.be[e]), a.act);
                store8<T, AL>(y + (p + u * lanes) * a.ldy, nv, v[u]);
            }
    }
}

// ---- backward
template <typename T, bool AL, int CLS> __global__ __launch_bounds__(GN_BLOCK) void gn_bwd_partial_kernel(GnArgs a) {
    __shared__ float red[GN_BLOCK / 64 * GN_MAXOCT * 8];
    __shared__ float kept[16][GN_BLOCK];           // a lane's sums of the pixels before the last GN_FOLD
    const int o = threadIdx.x & (a.octp - 1), pl = threadIdx.x / a.octp, lanes = GN_BLOCK / a.octp;
    const int c0 = (blockIdx.y * GN_MAXOCT + o) * 8;
    const int nv = a.C - c0 < 8 ? a.C - c0 : 8;
    const int n = blockIdx.x / a.chunks, chunk = blockIdx.x - n * a.chunks;
    const long long p0 = (long long)chunk * a.per;
    const long long p1 = p0 + a.per < a.HW ? p0 + a.per : a.HW;
    float s[8], q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = q[e] = 0.f;
    if (nv > 0) {
        GnChan ch;
        gn_channels(a, n, c0, nv, ch);
        const T* x = (const T*)a.x + (long long)n * a.HW * a.ldx + c0;
        const T* dy = (const T*)a.dy + (long long)n * a.HW * a.lddy + c0;
        int turns = 0;
        bool folded = false;
        for (long long p = p0 + pl; p < p1; p += GN_UB * lanes) {
            float v[GN_UB][8], d[GN_UB][8];
#pragma unroll
            for (int u = 0; u < GN_UB; ++u)
                if (p + u * lanes < p1) {
                    load8<T, AL>(x + (p + u * lanes) * a.ldx, nv, v[u]);
                    load8<T, AL>(dy + (p + u * lanes) * a.lddy, nv, d[u]);
                }
#pragma unroll
            for (int u = 0; u < GN_UB; ++u)
                if (p + u * lanes < p1)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x0 = v[u][e] - ch.mean[e];
                        const float dz = d[u][e] * gn_slope<T, CLS>(fmaf(x0, ch.k[e], ch.be[e]), a.act);
                        s[e] += dz;
                        q[e] = fmaf(dz, x0, q[e]);
                    }
            if (++turns == GN_FOLD / GN_UB) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    kept[e][threadIdx.x] = folded ? kept[e][threadIdx.x] + s[e] : s[e];
                    kept[8 + e][threadIdx.x] = folded ? kept[8 + e][threadIdx.x] + q[e] : q[e];
                    s[e] = q[e] = 0.f;
                }
                turns = 0;
                folded = true;
            }
        }
        if (folded)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s[e] += kept[e][threadIdx.x];
                q[e] += kept[8 + e][threadIdx.x];
            }
#pragma unroll
        for (int e = 0; e < 8; ++e) q[e] *= ch.rstd[e];
    }
    gn_reduce(s, a.octp, red);
    gn_reduce(q, a.octp, red);
    if (pl == 0) {
        float* w = a.part + (long long)blockIdx.x * 2 * a.C + c0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < nv) {
                w[e] = s[e];
                w[a.C + e] = q[e];
            }
    }
}

// The parameters' gradients: sums over the images, 16 channels x 16 parts of GN_IMAGES images per workgroup
#define GN_IMAGES 128
__device__ __forceinline__ void gn_params_part(unsigned unit, const float* sums, long long rows, int C, float* out, float* dgamma,
                                               float* dbeta) {
    __shared__ float red[2][16][16];
    const unsigned cb = (unsigned)(C + 15) / 16, step = unit / cb;
    const int l = threadIdx.x & 15, w = threadIdx.x >> 4, c = (int)(unit - step * cb) * 16 + l;
    const long long n0 = (long long)step * GN_IMAGES, n1 = n0 + GN_IMAGES < rows ? n0 + GN_IMAGES : rows;
    float s = 0.f, q = 0.f;
    if (c < C)
        for (long long n = n0 + w; n < n1; n += 16) {
            s += sums[n * 2 * C + c];
            q += sums[(n * 2 + 1) * C + c];
        }
    red[0][w][l] = s;
    red[1][w][l] = q;
    __syncthreads();
    if (threadIdx.x < 32 && c < C) {
        float v = 0.f;
        for (int k = 0; k < 16; ++k) v += red[w][k][l];
        if (out) out[(step * 2LL + w) * C + c] = v;
        else if (float* o = w == 0 ? dbeta : dgamma) o[c] = v;
    }
}

// dx; the workgroups behind the last image's sum the parameters' gradients of up to GN_IMAGES images
template <typename T, bool AL, int CLS> __global__ __launch_bounds__(GN_BLOCK) void gn_bwd_apply_kernel(GnArgs a) {
    if (blockIdx.x >= (unsigned)a.N * (unsigned)a.chunks) {
        if (blockIdx.y == 0) gn_params_part(blockIdx.x - (unsigned)a.N * (unsigned)a.chunks, a.sums, a.N, a.C, nullptr, a.dgamma, a.dbeta);
        return;
    }
    const int o = threadIdx.x & (a.octp - 1), pl = threadIdx.x / a.octp, lanes = GN_BLOCK / a.octp;
    const int c0 = (blockIdx.y * GN_MAXOCT + o) * 8;
    const int nv = a.C - c0 < 8 ? a.C - c0 : 8;
    if (nv <= 0) return;
    const unsigned blk = gn_backwards((unsigned)a.N * (unsigned)a.chunks);
    const int n = blk / a.chunks, chunk = blk - n * a.chunks;
    GnChan ch;
    gn_channels(a, n, c0, nv, ch);
    float A[8], B[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float* ab = a.ab + ((long long)n * a.G + (e < nv ? c0 + e : 0) / a.Cg) * 2;
        A[e] = ch.rstd[e] * ab[0];                           // dx = k dz - rstd A - (x - mean) rstd^2 B
        B[e] = ch.rstd[e] * ch.rstd[e] * ab[1];
    }
    const long long p0 = (long long)chunk * a.per;
    const long long p1 = p0 + a.per < a.HW ? p0 + a.per : a.HW;
    const T* x = (const T*)a.x + (long long)n * a.HW * a.ldx + c0;
    const T* dy = (const T*)a.dy + (long long)n * a.HW * a.lddy + c0;
    T* dx = (T*)a.y + (long long)n * a.HW * a.ldy + c0;
    for (long long p = p0 + pl; p < p1; p += GN_UB * lanes) {
        float v[GN_UB][8], d[GN_UB][8];
#pragma unroll
        for (int u = 0; u < GN_UB; ++u)
            if (p + u * lanes < p1) {
                load8<T, AL>(x + (p + u * lanes) * a.ldx, nv, v[u]);
                load8<T, AL>(dy + (p + u * lanes) * a.lddy, nv, d[u]);
            }
#pragma unroll
        for (int u = 0; u < GN_UB; ++u)
            if (p + u * lanes < p1) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x0 = v[u][e] - ch.mean[e];
                    const float dz = d[u][e] * gn_slope<T, CLS>(fmaf(x0, ch.k[e], ch.be[e]), a.act);
                    v[u][e] = fmaf(ch.k[e], dz, -fmaf(x0, B[e], A[e]));
                }
                store8<T, AL>(dx + (p + u * lanes) * a.ldy, nv, v[u]);
            }
    }
}

// ---- a group's pixels in the registers of one workgroup: x (and dy) are read once and there is one launch
//
// Workgroup = (image, run of gpb groups, `oct` octets wide); R octets of a lane stay in registers between the sums and the output.
struct GnSlab { int gpb, oct, octp, runs, images8; };      // images8: images of one XCD (images dealt to the 8 XCDs), 0: not dealt

// An octet as it lies in memory.  gn_opaque makes the compiler forget what it knows of the words: without it the unpacked floats of
// the first pass are kept for the second, twice the registers.
template <typename T> struct GnRaw { static constexpr int N = 8 * (int)sizeof(T) / 4; uint32_t w[N]; };
template <typename T> __device__ __forceinline__ void gn_raw_load(GnRaw<T>& r, const T* p) {
#pragma unroll
    for (int h = 0; h < GnRaw<T>::N / 4; ++h) {
        const uint4 q = ((const uint4*)p)[h];
        r.w[4 * h] = q.x; r.w[4 * h + 1] = q.y; r.w[4 * h + 2] = q.z; r.w[4 * h + 3] = q.w;
    }
}
template <typename T> __device__ __forceinline__ float gn_raw(const GnRaw<T>& r, int e);
template <> __device__ __forceinline__ float gn_raw<float>(const GnRaw<float>& r, int e) {
    union { uint32_t u; float f; } c;
    c.u = r.w[e];
    return c.f;
}
template <> __device__ __forceinline__ float gn_raw<bf16_t>(const GnRaw<bf16_t>& r, int e) {
    union { uint32_t u; float f; } c;
    c.u = e & 1 ? r.w[e >> 1] & 0xffff0000u : r.w[e >> 1] << 16;
    return c.f;
}
template <> __device__ __forceinline__ float gn_raw<f16_t>(const GnRaw<f16_t>& r, int e) {
    f16_t h;
    h.v = (uint16_t)(e & 1 ? r.w[e >> 1] >> 16 : r.w[e >> 1] & 0xffffu);
    return h2f(h);
}
template <typename T> __device__ __forceinline__ void gn_opaque(GnRaw<T>& r) {
#ifndef GVFI_HOSTSIM
    if constexpr (sizeof(T) == 2)
#pragma unroll
        for (int k = 0; k < GnRaw<T>::N; ++k) asm volatile("" : "+v"(r.w[k]));
#endif
}
// sums of v[8] over a workgroup's pixel lanes: tot[octet * 8 + e]; buf: 8 * T floats.  Few octets: through LDS, a wave per channel (six
// rounds of shuffles of eight values would take three times as long); from four on the shuffles are few.
template <int T_> __device__ __forceinline__ void gn_channel_sums(const float (&v)[8], int octp, float* buf, float* tot) {
    const int t = threadIdx.x, lane = t & 63;
    __syncthreads();
    if (octp >= 4) {
        float s[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = v[e];
        for (int off = octp; off < 64; off <<= 1)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += __shfl_xor(s[e], off);
        if (lane < octp)
#pragma unroll
            for (int e = 0; e < 8; ++e) buf[((t >> 6) * octp + lane) * 8 + e] = s[e];
        __syncthreads();
        for (int c = t; c < octp * 8; c += T_) {
            float a = 0.f;
            for (int w = 0; w < T_ / 64; ++w) a += buf[w * octp * 8 + c];
            tot[c] = a;
        }
        __syncthreads();
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) buf[e * T_ + t] = v[e];
    __syncthreads();
    const int lanes = T_ / octp;
    for (int col = t >> 6; col < octp * 8; col += T_ / 64) {
        const int o = col >> 3, e = col & 7;
        float s = 0.f;
        for (int k = lane; k < lanes; k += 64) s += buf[e * T_ + k * octp + o];
        s = wave_sum(s);
        if (lane == 0) tot[col] = s;
    }
    __syncthreads();
}
// sums of v[8] over each channel's group, in v.  OCT: groups are whole octets
template <int T_, bool OCT> __device__ __forceinline__ void gn_group_sums(float (&v)[8], const GnArgs& a, const GnSlab& b, int o, float* buf,
                                                                            float* tot) {
    if (OCT) {
        float s = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        const int lane = threadIdx.x & 63;
        if (b.octp == 1) s = wave_sum(s);
        else
            for (int off = b.octp; off < 64; off <<= 1) s += __shfl_xor(s, off);
        __syncthreads();
        if (lane < b.octp) buf[(threadIdx.x >> 6) * b.octp + lane] = s;
        __syncthreads();
        const int og = a.Cg / 8, o0 = o / og * og;
        s = 0.f;
        for (int w = 0; w < T_ / 64; ++w)
            for (int k = 0; k < og; ++k) s += buf[w * b.octp + ((o0 + k) & (b.octp - 1))];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s;
    } else {
        gn_channel_sums<T_>(v, b.octp, buf, tot);
        for (int g = threadIdx.x; g < b.gpb; g += T_) {
            float s = 0.f;
            for (int c = 0; c < a.Cg; ++c) s += tot[g * a.Cg + c];
            buf[g] = s;
        }
        __syncthreads();
        int g = o * 8 / a.Cg, left = (g + 1) * a.Cg - o * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = g < b.gpb ? buf[g] : 0.f;
            if (--left == 0) { ++g; left = a.Cg; }
        }
    }
}
__device__ __forceinline__ bool gn_slab_block(const GnArgs& a, const GnSlab& b, int& n, int& run) {
    unsigned i = blockIdx.x;
    if (b.images8) {                                       // workgroups i, i + 8, ... run on one XCD: whole images to each
        const unsigned j = i >> 3;
        n = (int)((i & 7) + 8 * (j / (unsigned)b.runs));
        run = (int)(j % (unsigned)b.runs);
        return n < a.N;
    }
    n = (int)(i / (unsigned)b.runs);
    run = (int)(i % (unsigned)b.runs);
    return true;
}

template <typename T, int T_, int R, bool OCT, int CLS> __global__ __launch_bounds__(T_) void gn_slab_kernel(GnArgs a, GnSlab b, float* stats, float eps) {
    __shared__ float buf[OCT ? T_ / 64 * 16 : 8 * T_];
    __shared__ float tot[OCT ? 1 : 128];
    int n, run;
    if (!gn_slab_block(a, b, n, run)) return;
    const int o = threadIdx.x & (b.octp - 1), pl = threadIdx.x / b.octp, lanes = T_ / b.octp;
    const int c0 = run * b.gpb * a.Cg + o * 8;
    const bool on = o < b.oct && c0 < a.C;
    const T* x = (const T*)a.x + (long long)n * a.HW * a.ldx + c0;
    GnRaw<T> raw[R];
    float s[8], mean[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (on && pl + i * lanes < a.HW) gn_raw_load<T>(raw[i], x + (pl + i * lanes) * a.ldx);
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (on && pl + i * lanes < a.HW)
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] += gn_raw<T>(raw[i], e);
#pragma unroll
    for (int i = 0; i < R; ++i) gn_opaque<T>(raw[i]);
    gn_group_sums<T_, OCT>(s, a, b, o, buf, tot);
    const float im = 1.f / ((float)a.HW * (float)a.Cg);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        mean[e] = s[e] * im;
        s[e] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (on && pl + i * lanes < a.HW)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = gn_raw<T>(raw[i], e) - mean[e];
                s[e] = fmaf(d, d, s[e]);
            }
#pragma unroll
    for (int i = 0; i < R; ++i) gn_opaque<T>(raw[i]);
    gn_group_sums<T_, OCT>(s, a, b, o, buf, tot);
    if (!on) return;
    float ga[8], be[8];
    int g = c0 / a.Cg, left = (g + 1) * a.Cg - c0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float rstd = 1.f / sqrtf(s[e] * im + eps);
        if (pl == 0 && left == a.Cg) {                     // the group's first channel
            stats[((long long)n * a.G + g) * 2] = mean[e];
            stats[((long long)n * a.G + g) * 2 + 1] = rstd;
        }
        if (--left == 0) { ++g; left = a.Cg; }
        ga[e] = a.gamma ? rstd * a.gamma[c0 + e] : rstd;
        be[e] = a.beta ? a.beta[c0 + e] : 0.f;
    }
    T* y = (T*)a.y + (long long)n * a.HW * a.ldy + c0;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (pl + i * lanes < a.HW) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = gn_act<T, CLS>(fmaf(gn_raw<T>(raw[i], e) - mean[e], ga[e], be[e]), a.act);
            store8<T, true>(y + (pl + i * lanes) * a.ldy, 8, v);
        }
}

template <typename T, int T_, int R, int CLS> __global__ __launch_bounds__(T_) void gn_slab_bwd_kernel(GnArgs a, GnSlab b) {
    __shared__ float buf[8 * T_];
    __shared__ float tot[2][128], ab[2][128];
    int n, run;
    if (!gn_slab_block(a, b, n, run)) return;
    const int o = threadIdx.x & (b.octp - 1), pl = threadIdx.x / b.octp, lanes = T_ / b.octp;
    const int cb = run * b.gpb * a.Cg, c0 = cb + o * 8;
    const bool on = o < b.oct && c0 < a.C;
    const T* x = (const T*)a.x + (long long)n * a.HW * a.ldx + c0;
    const T* dy = (const T*)a.dy + (long long)n * a.HW * a.lddy + c0;
    GnRaw<T> rx[R], rd[R];
    GnChan ch;
    gn_channels(a, n, on ? c0 : 0, 8, ch);
    float s[8], q[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = q[e] = 0.f;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (on && pl + i * lanes < a.HW) {
            gn_raw_load<T>(rx[i], x + (pl + i * lanes) * a.ldx);
            gn_raw_load<T>(rd[i], dy + (pl + i * lanes) * a.lddy);
        }
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (on && pl + i * lanes < a.HW)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x0 = gn_raw<T>(rx[i], e) - ch.mean[e];
                const float dz = gn_raw<T>(rd[i], e) * gn_slope<T, CLS>(fmaf(x0, ch.k[e], ch.be[e]), a.act);
                s[e] += dz;
                q[e] = fmaf(dz, x0, q[e]);
            }
#pragma unroll
    for (int e = 0; e < 8; ++e) q[e] *= ch.rstd[e];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        gn_opaque<T>(rx[i]);
        gn_opaque<T>(rd[i]);
    }
    gn_channel_sums<T_>(s, b.octp, buf, tot[0]);
    gn_channel_sums<T_>(q, b.octp, buf, tot[1]);
    for (int c = threadIdx.x; c < b.oct * 8 && cb + c < a.C; c += T_) {
        a.sums[(long long)n * 2 * a.C + cb + c] = tot[0][c];
        a.sums[((long long)n * 2 + 1) * a.C + cb + c] = tot[1][c];
    }
    for (int g = threadIdx.x; g < 2 * b.gpb; g += T_) {    // A of the groups, then B
        const int w = g >= b.gpb, gg = g - (w ? b.gpb : 0);
        float v = 0.f;
        if (cb + gg * a.Cg < a.C)
            for (int c = 0; c < a.Cg; ++c) v += (a.gamma ? a.gamma[cb + gg * a.Cg + c] : 1.f) * tot[w][gg * a.Cg + c];
        ab[w][gg] = v / ((float)a.HW * (float)a.Cg);
    }
    __syncthreads();
    if (!on) return;
    float A[8], B[8];
    int g = o * 8 / a.Cg, left = (g + 1) * a.Cg - o * 8;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        A[e] = ch.rstd[e] * ab[0][g];
        B[e] = ch.rstd[e] * ch.rstd[e] * ab[1][g];
        if (--left == 0) { if (g + 1 < b.gpb) ++g; left = a.Cg; }
    }
    T* dx = (T*)a.y + (long long)n * a.HW * a.ldy + c0;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (pl + i * lanes < a.HW) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x0 = gn_raw<T>(rx[i], e) - ch.mean[e];
                const float dz = gn_raw<T>(rd[i], e) * gn_slope<T, CLS>(fmaf(x0, ch.k[e], ch.be[e]), a.act);
                v[e] = fmaf(ch.k[e], dz, -fmaf(x0, B[e], A[e]));
            }
            store8<T, true>(dx + (pl + i * lanes) * a.ldy, 8, v);
        }
}

// ---- launches of one element type (instantiated per type in a file of its own)
void gn_launch_stats(const GnArgs& a, float* stats, float eps, hipStream_t st);
void gn_launch_group(const GnArgs& a, hipStream_t st);
template <typename T> void gn_forward_launch(const GnArgs& a, const GnSlab& b, int threads, int r, bool al, float* stats, float eps,
                                             hipStream_t st);
template <typename T> void gn_backward_launch(const GnArgs& a, const GnSlab& b, int threads, int r, bool al, hipStream_t st);

#define GN_BY_CLASS(GO)              \
    do {                             \
        if (a.act.cls == 0) GO(0);   \
        else if (a.act.cls == 1) GO(1); \
        else if (a.act.cls == 2) GO(2); \
        else GO(3);                  \
    } while (0)
#ifdef GN_INSTANTIATE
template <typename T> void gn_forward_launch(const GnArgs& a, const GnSlab& b, int threads, int r, bool al, float* stats, float eps,
                                             hipStream_t st) {
    if (r) {
        const dim3 gs((unsigned)((b.images8 ? 8LL * b.images8 : (long long)a.N) * b.runs));
#define GN_GO3(T_, R, O, K) GVFI_LAUNCH_COOP((gn_slab_kernel<T, T_, R, O, K>), gs, dim3(T_), st, a, b, stats, eps)
#define GN_GO2(O, K)                                   \
    do {                                               \
        if (threads == 256) GN_GO3(256, 4, O, K);      \
        else if (r <= 8) GN_GO3(512, 8, O, K);         \
        else if constexpr (sizeof(T) == 2) GN_GO3(512, 16, O, K); \
    } while (0)
#define GN_GO1(K) do { if (a.Cg % 8 == 0) GN_GO2(true, K); else GN_GO2(false, K); } while (0)
        GN_BY_CLASS(GN_GO1);
        return;
    }
    const dim3 grid((unsigned)((long long)a.N * a.chunks), (unsigned)((a.C + GN_MAXOCT * 8 - 1) / (GN_MAXOCT * 8)));
    if (al) GVFI_LAUNCH_COOP((gn_partial_kernel<T, true>), grid, dim3(GN_BLOCK), st, a);
    else GVFI_LAUNCH_COOP((gn_partial_kernel<T, false>), grid, dim3(GN_BLOCK), st, a);
    gn_launch_stats(a, stats, eps, st);
#define GN_GO(K)                                                                                                    \
    do {                                                                                                            \
        if (al) GVFI_LAUNCH_SIMPLE((gn_apply_kernel<T, true, K>), grid, dim3(GN_BLOCK), st, a);                     \
        else GVFI_LAUNCH_SIMPLE((gn_apply_kernel<T, false, K>), grid, dim3(GN_BLOCK), st, a);                       \
    } while (0)
    GN_BY_CLASS(GN_GO);
#undef GN_GO
}
template <typename T> void gn_backward_launch(const GnArgs& a, const GnSlab& b, int threads, int r, bool al, hipStream_t st) {
    if (r) {
        const dim3 gs((unsigned)((b.images8 ? 8LL * b.images8 : (long long)a.N) * b.runs));
#define GN_GO2B(T_, R, K) GVFI_LAUNCH_COOP((gn_slab_bwd_kernel<T, T_, R, K>), gs, dim3(T_), st, a, b)
#define GN_GO1B(K)                                 \
    do {                                           \
        if (threads == 256) GN_GO2B(256, 4, K);    \
        else if (r <= 8) GN_GO2B(512, 8, K);       \
        else if constexpr (sizeof(T) == 2) GN_GO2B(512, 16, K); \
    } while (0)
        GN_BY_CLASS(GN_GO1B);
        return;
    }
    const dim3 grid((unsigned)((long long)a.N * a.chunks), (unsigned)((a.C + GN_MAXOCT * 8 - 1) / (GN_MAXOCT * 8)));
    const dim3 gridp(grid.x + ((a.dgamma || a.dbeta) && a.N <= GN_IMAGES ? (unsigned)(a.C + 15) / 16 : 0u), grid.y);
#define GN_GO(K)                                                                                                    \
    do {                                                                                                            \
        if (al) GVFI_LAUNCH_COOP((gn_bwd_partial_kernel<T, true, K>), grid, dim3(GN_BLOCK), st, a);                 \
        else GVFI_LAUNCH_COOP((gn_bwd_partial_kernel<T, false, K>), grid, dim3(GN_BLOCK), st, a);                   \
        gn_launch_group(a, st);                                                                                     \
        if (al) GVFI_LAUNCH_COOP((gn_bwd_apply_kernel<T, true, K>), gridp, dim3(GN_BLOCK), st, a);                  \
        else GVFI_LAUNCH_COOP((gn_bwd_apply_kernel<T, false, K>), gridp, dim3(GN_BLOCK), st, a);                    \
    } while (0)
    GN_BY_CLASS(GN_GO);
#undef GN_GO
}
#endif
