// K13, internal: the matrix-core launches of gated_ff_mfma.hip that gated_ff.hip's entry points use.
#pragma once
#include "fp_common.h"

enum { FF_BF16 = 0, FF_F16 = 1, FF_E4M3 = 2 };

// h = act(x . wg^T * scales + bg) * (x . wu^T * scales + bu); x, wg, wu 16-byte aligned with row strides of multiples of 16
// bytes, K a multiple of 64 (e4m3: 128); gate / up: the projections, or null.
__attribute__((visibility("hidden"))) int fpi_glu(int type, const void* x, int64_t ldx, const float* xs, const void* wg, int64_t ldwg,
                                                  const float* gs, const void* wu, int64_t ldwu, const float* us, const void* bg,
                                                  const void* bu, void* h, int64_t ldh, void* gate, void* up, int64_t ldp, int M,
                                                  int F, int K, int act, hipStream_t st);

// part[s] [M, N] fp32 = a [M, K] . w [N, K]^T over the K tiles (64) of part s: ks_per each, the last part the rest;
// narrow: 256 x 128 tiles instead of 256 x 256
__attribute__((visibility("hidden"))) int fpi_gemm_parts(int type, bool narrow, const void* a, int64_t lda, const void* w, int64_t ldw, float* part,
                                                         int M, int N, int K, int splits, int ks_per, hipStream_t st);
