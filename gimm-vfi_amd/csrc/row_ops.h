// Helpers shared by the kernels that stream rows of channels (group_norm.hip, dropout.hip, rel_softmax.hip).
#pragma once
#include "common.h"

// float -> element, round to nearest even, overflow to infinity: gradients of a scaled loss are looked through for infinities, so
// these operators do not saturate as Elem<f16_t>::st does.
template <typename T> __device__ __forceinline__ T to_elem(float f);
template <> __device__ __forceinline__ float to_elem<float>(float f) { return f; }
template <> __device__ __forceinline__ bf16_t to_elem<bf16_t>(float f) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(bf16_t, (__bf16)f);       // v_cvt_pk_bf16_f32
#else
    return f2bf(f);
#endif
}
template <> __device__ __forceinline__ f16_t to_elem<f16_t>(float f) {
#if defined(__HIP_DEVICE_COMPILE__)
    f16_t r;
    r.v = __builtin_bit_cast(uint16_t, (_Float16)f);
    return r;
#else
    f16_t r = f2h(f);
    if (f >= 65520.f || f <= -65520.f) r.v = f > 0 ? 0x7c00 : 0xfc00;
    return r;
#endif
}

// Eight consecutive elements ("octet": one 16-byte vector of a 16-bit type, two of float) as floats.
// AL: every octet is whole and 16-byte aligned.  Else whole octets are still taken as vectors -- the hardware's vector accesses need
// no more than the element's alignment -- and of others the first nv elements one by one, the rest are 0.
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Oct { T e[8]; };
template <typename T, bool AL> __device__ __forceinline__ void load8(const T* p, int nv, float (&v)[8]) {
    if constexpr (AL) {
        constexpr int VE = Elem<T>::VE;
        struct alignas(16) Q { T e[VE]; };
#pragma unroll
        for (int h = 0; h < 8 / VE; ++h) {
            const Q q = ((const Q*)p)[h];
#pragma unroll
            for (int e = 0; e < VE; ++e) v[h * VE + e] = Elem<T>::ld(&q.e[e]);
        }
    } else if (nv >= 8) {
        const Oct<T> q = *(const Oct<T>*)p;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = Elem<T>::ld(&q.e[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < nv ? Elem<T>::ld(p + e) : 0.f;
    }
}
template <typename T, bool AL> __device__ __forceinline__ void store8(T* p, int nv, const float (&v)[8]) {
    if constexpr (AL) {
        constexpr int VE = Elem<T>::VE;
        struct alignas(16) Q { T e[VE]; };
#pragma unroll
        for (int h = 0; h < 8 / VE; ++h) {
            Q q;
#pragma unroll
            for (int e = 0; e < VE; ++e) q.e[e] = to_elem<T>(v[h * VE + e]);
            ((Q*)p)[h] = q;
        }
    } else if (nv >= 8) {
        Oct<T> q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q.e[e] = to_elem<T>(v[e]);
        *(Oct<T>*)p = q;
    } else {
#pragma unroll
        for (int e = 0; e < 7; ++e)
            if (e < nv) p[e] = to_elem<T>(v[e]);
    }
}

// Sum / maximum over a wave, in every lane (all 64 lanes take part).  The 16 lanes of a row by DPP, the four rows by reading a lane of
// each: vector instructions only, where shuffles would queue at the LDS unit.
#ifndef GVFI_HOSTSIM
template <int CTRL> __device__ __forceinline__ float dpp_f(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_f(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// ... over the 16 lanes of a DPP row
__device__ __forceinline__ float row_sum(float v) {
    v += dpp_f<0xB1>(v);        // quad_perm 1 0 3 2
    v += dpp_f<0x4E>(v);        // quad_perm 2 3 0 1
    v += dpp_f<0x141>(v);       // row_half_mirror
    v += dpp_f<0x140>(v);       // row_mirror
    return v;
}
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dpp_f<0xB1>(v));
    v = fmaxf(v, dpp_f<0x4E>(v));
    v = fmaxf(v, dpp_f<0x141>(v));
    v = fmaxf(v, dpp_f<0x140>(v));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    v = row_sum(v);
    return (lane_f(v, 0) + lane_f(v, 16)) + (lane_f(v, 32) + lane_f(v, 48));
}
__device__ __forceinline__ float wave_max(float v) {
    v = row_max(v);
    return fmaxf(fmaxf(lane_f(v, 0), lane_f(v, 16)), fmaxf(lane_f(v, 32), lane_f(v, 48)));
}
#else
__device__ __forceinline__ float row_sum(float v) {
    for (int off = 1; off < 16; off <<= 1) v += __shfl_xor(v, off);
    return v;
}
__device__ __forceinline__ float row_max(float v) {
    for (int off = 1; off < 16; off <<= 1) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
    for (int off = 1; off < 64; off <<= 1) v = fmaxf(v, __shfl_xor(v, off));
    return v;
}
#endif

// A wave's accesses to memory before this place happen before those after it, whichever of its lanes make them.  No instruction: a wave's LDS
// operations are carried out in order, what this stops is the compiler moving them.
__device__ __forceinline__ void wave_order() {
#ifndef GVFI_HOSTSIM
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#else
    emu::wave_sync();
#endif
}

// 2^x of the hardware: about one step of float; 0 below 2^-126; 2^-inf = 0, a NaN stays one
__device__ __forceinline__ float exp2_hw(float x) {
#ifndef GVFI_HOSTSIM
    return __builtin_amdgcn_exp2f(x);
#else
    return exp2f(x);
#endif
}

// every row of `ld` elements of size `es` starts on a 16-byte boundary
static inline bool gvfi_rows_aligned(const void* p, long long ld, int es) {
    return (((uintptr_t)p) & 15) == 0 && ((ld * es) & 15) == 0;
}
static inline int gvfi_esize(int dtype) { return dtype == GVFI_F32 ? 4 : 2; }
static inline bool gvfi_dtype_ok(int dtype) { return dtype == GVFI_F32 || dtype == GVFI_BF16 || dtype == GVFI_F16; }
