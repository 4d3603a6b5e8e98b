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

// The same in fp32 parts of K, without scales, biases and activation: part[s] [M, 2 Fp], x . wg^T from column 0, x . wu^T from
// column Fp = F rounded up to 8 on, over the K tiles (128 bytes) of part s: ks_per each, the last part the rest.
__attribute__((visibility("hidden"))) int fpi_glu_parts(int type, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu,
                                                        int64_t ldwu, float* part, int M, int F, int K, int splits, int ks_per,
                                                        hipStream_t st);

// The gradient's products: out [M, N] = a [M, K] . w with w's K tiles as they lie, 64 rows of N each; tile t at w + t tiles,
// + d1 bytes from tile s1 on, + d2 from tile s2 on (gemm_w4.h, TrArgs).  out in 16 bits (splits = 0; row stride N, 16-byte
// aligned) or fp32 parts [splits][M, N] over ks_per K tiles each.  narrow: 256 x 128 tiles instead of 256 x 256 (as the
// parts have).  K % 64 == 0, N % 8 == 0.
struct GradProduct {
    bool narrow;
    const void *a, *w;
    int64_t lda, ldw, d1, d2;
    int s1, s2, M, N, K, splits, ks_per;
    void* out;
};
__attribute__((visibility("hidden"))) int fpi_grad_product(int type, const GradProduct& p, hipStream_t st);
// Two in one launch of 256 x 128 tiles: `first` (splits > 0), then `second`.
__attribute__((visibility("hidden"))) int fpi_grad_pair(int type, const GradProduct& first, const GradProduct& second, hipStream_t st);
