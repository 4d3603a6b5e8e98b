// K13's forward product on the matrix cores: instances of gemm_w4.h (see GluArgs there; figures in gated_ff.hip).
#include "gated_ff.h"
#include "gemm_w4.h"

using namespace fp_gemm;

int fpi_glu(int type, const void* x, int64_t ldx, const float* xs, const void* wg, int64_t ldwg, const float* gs, const void* wu,
            int64_t ldwu, const float* us, const void* bg, const void* bu, void* h, int64_t ldh, void* gate, void* up, int64_t ldp,
            int M, int F, int K, int act, hipStream_t st) {
    const GluArgs glu{wu, bu, ldwu, us, gate, up, ldp, act};
    const int ntm = (M + BM - 1) / BM;
    FP_REQUIRE((int64_t)ntm * ((F + 63) / 64) < (1ll << 31));
    // tile walk (ConvGeom::gm): 4 column tiles x all row tiles where there are many, else 8 row tiles x all column tiles (19385
    // rows, [4096, 14336]: 3.23 against 3.35 ms; 4096 rows: 0.676 either way; 8000 rows, [1152, 4304]: 155 against 153 us)
    ConvGeom cg{};
    cg.gm = ntm >= 48 ? -4 : 8;
    // fewer 256 x 128 tiles than half the CUs: 256 x 64 ones, twice as many at about 0.6 of the time each (as K5)
    const bool narrow = (int64_t)ntm * ((F + 127) / 128) <= persistent_grid() / 2;
#define FP_GLU(T, TO, NT, KEEP)                                                                                                   \
    return launch_w4<T, 0, 0, TO, NT, 0, 0, 0, 1, KEEP>(x, ldx, 0, K, wg, ldwg, bg, h, ldh, M, F, K, 0, nullptr, 0, nullptr, cg, st, \
                                                        xs, gs, QkNormArgs{}, Rows2{}, glu)
    if (type == FF_E4M3) {
        if (narrow) FP_GLU(fp8e4, bf16, 4, 0);
        FP_GLU(fp8e4, bf16, 8, 0);
    }
    if (type == FF_BF16) {
        if (gate) {
            if (narrow) FP_GLU(bf16, bf16, 4, 1);
            FP_GLU(bf16, bf16, 8, 1);
        }
        if (narrow) FP_GLU(bf16, bf16, 4, 0);
        FP_GLU(bf16, bf16, 8, 0);
    }
    if (gate) {
        if (narrow) FP_GLU(_Float16, _Float16, 4, 1);
        FP_GLU(_Float16, _Float16, 8, 1);
    }
    if (narrow) FP_GLU(_Float16, _Float16, 4, 0);
    FP_GLU(_Float16, _Float16, 8, 0);
#undef FP_GLU
}

int fpi_glu_parts(int type, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu, float* part, int M, int F,
                  int K, int splits, int ks_per, hipStream_t st) {
    const int64_t Fp = (F + 7) & ~7;
    const GluArgs glu{wu, nullptr, ldwu, nullptr, nullptr, nullptr, Fp, 0};
    const SplitArgs sp{splits, ks_per};
    const ConvGeom cg{};
    const int nk = K / (type == FF_E4M3 ? 128 : 64);
    FP_REQUIRE((int64_t)((M + BM - 1) / BM) * ((F + 63) / 64) * splits < (1ll << 31));
    FP_REQUIRE(splits > 0 && (int64_t)(splits - 1) * ks_per < nk && (int64_t)splits * ks_per >= nk);
#define FP_PARTS(T)                                                                                                                     \
    return launch_w4<T, 0, 0, float, 4, 0, 0, 0, 1, 0, 1>(x, ldx, 0, K, wg, ldwg, nullptr, part, 2 * Fp, M, F, K, 0, nullptr, 0, nullptr, cg, \
                                                          st, nullptr, nullptr, QkNormArgs{}, Rows2{}, glu, sp)
    if (type == FF_E4M3) FP_PARTS(fp8e4);
    if (type == FF_BF16) FP_PARTS(bf16);
    FP_PARTS(_Float16);
#undef FP_PARTS
}
