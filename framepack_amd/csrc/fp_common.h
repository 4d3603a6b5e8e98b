// Shared device helpers for the gfx950 (CDNA4, wave64) kernels of the FramePack DiT hot path.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef __bf16 bf16;
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

#define FP_CHECK_LAUNCH()                        \
    do {                                         \
        hipError_t e__ = hipGetLastError();      \
        if (e__ != hipSuccess) return (int)e__;  \
    } while (0)

// Argument errors are reported as hipErrorInvalidValue (1); the host mirror turns them into ValueError.
#define FP_REQUIRE(cond)                               \
    do {                                               \
        if (!(cond)) return (int)hipErrorInvalidValue; \
    } while (0)

__device__ __forceinline__ float bf16_bits_to_f32(unsigned short b) { return __uint_as_float(((unsigned)b) << 16); }

// sum over the 64 lanes of a wave (result in every lane)
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// sum over aligned groups of 16 lanes
__device__ __forceinline__ float group16_sum(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// K3's sum of squared deviations (its 16-bit and its e4m3 form have to give the same bits): every square is rounded before it is
// added, under every compiler option.
__device__ __forceinline__ float k3_add_square(float ss, float d) {
#pragma clang fp contract(off)
    return ss + d * d;
}

// K2's arithmetic between its rounding points (norm_kernels.hip and the GEMM epilogue that replaces it, gemm_w4.h, have to give
// the same bits): what is fused and what is not is written out, so that no compiler option decides it for one of them alone.
__device__ __forceinline__ float k2_sum_of_squares(const float (&f)[8]) {
#pragma clang fp contract(off)
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
    return ss;
}
__device__ __forceinline__ float k2_rstd(float row_ss, float eps) { return rsqrtf(__builtin_fmaf(row_ss, 1.f / 128.f, eps)); }
// Rotary pair p of a lane's four, (re, im): (re c0 - im s0, im c1 + re s1).  Both products of the last pair are rounded before they
// are added, of the others' only the one with the sine: the results that these kernels have given from the start.
__device__ __forceinline__ float k2_rot_re(int p, float re, float im, float c0, float s0) {
#pragma clang fp contract(off)
    return p == 3 ? re * c0 - im * s0 : __builtin_fmaf(re, c0, -(im * s0));
}
__device__ __forceinline__ float k2_rot_im(int p, float re, float im, float c1, float s1) {
#pragma clang fp contract(off)
    return p == 3 ? im * c1 + re * s1 : __builtin_fmaf(im, c1, re * s1);
}

// Bijective XCD-aware remap (blocks b and b+8 share an XCD's L2): gives each XCD a contiguous run of
// work items so that neighbours in work order share operands through one L2.
__device__ __forceinline__ int xcd_remap(int bid, int nwg) {
    const int q = nwg >> 3, r = nwg & 7, xcd = bid & 7;
    const int base = (xcd < r) ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q;
    return base + (bid >> 3);
}
