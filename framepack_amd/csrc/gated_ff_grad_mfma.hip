// K13's gradient products on the matrix cores: instances of gemm_w4.h (see TrArgs, SplitArgs and PartsArgs there; figures in
// gated_ff.hip).  W by rows of K is read as it lies: transposed copies of Wg, Wu and x would move 213 MB each way at 4096 rows
// of [4096, 11008], where either product takes 535 us.
#include "gated_ff.h"
#include "gemm_w4.h"

using namespace fp_gemm;

static bool fits(const GradProduct& p) {
    return p.K % BK == 0 && p.N % 8 == 0 && (int64_t)(p.M / 256 + 1) * (p.N / 128 + 1) * (p.splits > 0 ? p.splits : 1) < (1ll << 30) &&
           (p.splits == 0 || ((int64_t)(p.splits - 1) * p.ks_per < p.K / BK && (int64_t)p.splits * p.ks_per >= p.K / BK));
}

template <typename T>
static int run(const GradProduct& p, hipStream_t st) {
    const TrArgs tr{p.s1, p.s2, p.d1, p.d2};
    const SplitArgs sp{p.splits, p.ks_per};
    const ConvGeom cg{};
    FP_REQUIRE(fits(p));
#define FP_TR(TO, NT, SPLIT)                                                                                                         \
    return launch_w4<T, 0, 0, TO, NT, 0, 0, 0, 0, 0, SPLIT, 1>(p.a, p.lda, 0, p.K, p.w, p.ldw, nullptr, p.out, p.N, p.M, p.N, p.K, 0, \
                                                               nullptr, 0, nullptr, cg, st, nullptr, nullptr, QkNormArgs{}, Rows2{},  \
                                                               GluArgs{}, sp, tr)
    if (p.splits > 0) FP_TR(float, 4, 1);
    if (p.narrow) FP_TR(T, 4, 0);
    FP_TR(T, 8, 0);
#undef FP_TR
}

template <typename T>
static int run_pair(const GradProduct& q, const GradProduct& p, hipStream_t st) {
    FP_REQUIRE(fits(q) && fits(p) && q.splits > 0);
    const ConvGeom cg{};
    const PartsArgs pp{q.a, q.w, (float*)q.out, q.lda, q.ldw, {q.s1, q.s2, q.d1, q.d2}, q.M, q.N, q.K, (q.M + BM - 1) / BM, (q.N + 127) / 128,
                       {q.splits, q.ks_per}};
#define FP_PAIR(TO, SPLIT)                                                                                                          \
    return launch_w4<T, 0, 0, TO, 4, 0, 0, 0, 0, 0, SPLIT, 1, 1>(p.a, p.lda, 0, p.K, p.w, p.ldw, nullptr, p.out, p.N, p.M, p.N, p.K, 0, \
                                                                nullptr, 0, nullptr, cg, st, nullptr, nullptr, QkNormArgs{}, Rows2{}, \
                                                                GluArgs{}, SplitArgs{p.splits, p.ks_per},                             \
                                                                TrArgs{p.s1, p.s2, p.d1, p.d2}, pp)
    if (p.splits > 0) FP_PAIR(float, 1);
    FP_PAIR(T, 0);
#undef FP_PAIR
}

int fpi_grad_product(int type, const GradProduct& p, hipStream_t st) {
    return type == FF_BF16 ? run<bf16>(p, st) : run<_Float16>(p, st);
}

int fpi_grad_pair(int type, const GradProduct& first, const GradProduct& second, hipStream_t st) {
    return type == FF_BF16 ? run_pair<bf16>(first, second, st) : run_pair<_Float16>(first, second, st);
}
