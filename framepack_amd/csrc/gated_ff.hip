// K13: the gated feed-forward block's first half, h = act(x . Wg^T + bg) * (x . Wu^T + bu), act = SiLU or tanh-GELU, in
// bf16 / f16 and on e4m3 operands, and its gradient.  gfx950 / wave64; C-ABI entry points at the bottom, declarations in
// include/framepack_hip.h.
//
//   dg = dh u act'(g)   du = dh act(g)   dx = dg . Wg + du . Wu   dWg = dg^T . x   dWu = du^T . x   db = column sums
//
// Up to 48 rows both weights stream through registers once (glu_few_kernel; bound by their bytes), above that gemm_w4.h's tile
// multiplies 256 rows by both projections' columns and joins them in its epilogue (bound by the matrix pipe; where there are few
// tiles, by the operands' way into LDS).  The gradient: one element-wise pass that writes dg | du as rows and as columns (HBM),
// then two products on the same tile, which read Wg, Wu and x as they lie.  A large copy runs at 4.9 TB/s on this card, a large
// product at 1440 TFLOP/s in bf16 and 2370 in e4m3.  Measured, [K, F], us:
//   1 row, [4096, 14336], bf16           44      5.3 TB/s of weights
//   16 rows, the same, e4m3              23      5.2 TB/s
//   64 - 256 rows, the same, bf16        59 - 67 4.0 - 3.5 TB/s (128 bytes of a row a K tile)
//   729 rows, [1152, 4304], f16          22      (204 tiles on 256 CUs; 10 of it first loads and epilogue)
//   4096 rows, [4096, 14336], e4m3       388     2480 TFLOP/s
//   19385 rows, [4096, 14336], bf16      3190    1430 TFLOP/s (matrix pipe 78 % busy at 1.82 GHz)
//   gradient, 729 rows, [1152, 4304]     61      element-wise 14.5, products 41, parts 5
//   gradient, 4096 rows, [4096, 11008]   1185    element-wise 109 (5.8 TB/s), products 2 x 535 (1380 TFLOP/s)
// (calls one after the other for half a second, by when the clock has settled: the first some twenty of the long ones after a pause
// take up to a fifth more or less.)
#include <algorithm>
#include <type_traits>
#include "gated_ff.h"
#include "gemm_pipeline.h"
#include "row_access.h"

extern "C" int64_t fp_gated_ff_workspace_bytes(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                                               int M, int F, int K);
extern "C" int64_t fp_gated_ff_backward_workspace_bytes(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up,
                                                        int64_t ldwu, int M, int F, int K);

namespace {

using fp_gemm::fp8e4;
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma16(h16x8 a, h16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v)); }

// act(v) = v s(v) with s = sigmoid(v) (SiLU) or sigmoid(2 sqrt(2/pi) (v + 0.044715 v^3)) (tanh-GELU)
__device__ __forceinline__ float act_of(float v, int act) {
    constexpr float k = 2.f * 0.7978845608028654f;
    return v * sigmoid(act ? v * __builtin_fmaf(v * v, 0.044715f * k, k) : v);
}
// act(v) and act'(v) = s + v s (1 - s) z'(v).  Where s has run into 0 or 1 the second term is 0, also where z' is inf.
__device__ __forceinline__ void act_grad(float v, int act, float& a, float& da) {
    constexpr float k = 2.f * 0.7978845608028654f;
    const float z = act ? v * __builtin_fmaf(v * v, 0.044715f * k, k) : v;
    const float dz = act ? __builtin_fmaf(v * v, 3.f * 0.044715f * k, k) : 1.f;
    const float s = sigmoid(z), p = s * (1.f - s);
    a = v * s;
    da = s + (p == 0.f ? 0.f : v * p * dz);
}

struct GluCall {
    const void* x;
    int64_t ldx;
    const float* xs;
    const void *w[2];               // gate, up
    int64_t ldw[2];
    const float* ws[2];
    const void* b[2];
    void* h;
    int64_t ldh;
    void* pre[2];
    int64_t ldp;
    int M, F, K, act;
};

// ---- few rows: both weights stream through once -------------------------------------------------------------------
// 16 NC output columns a workgroup: its 4 waves share out K in steps of 128 bytes a row (neighbouring waves read
// neighbouring lines), each multiplying 2 NC tiles of 16 weight rows by MT x 16 tokens straight from registers - no weight
// is used twice, so nothing goes through LDS but the waves' sums at the end.  A lane holds twice 16 bytes of one row a step;
// which bytes is the same for weights and tokens, so the order of K inside a step does not matter.  Bound by the weights'
// bytes and, from 16 tokens on, by the tokens' lines, which every workgroup reads again from the L2: NC = 2 halves them.
// Loads need the type's alignment only; the last, partial step of K goes element by element.
__device__ __forceinline__ f32x4 mma(bf16, const u32x4& w, const u32x4& x, f32x4 c) {
    return mfma16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, x), c);
}
__device__ __forceinline__ f32x4 mma(_Float16, const u32x4& w, const u32x4& x, f32x4 c) {
    return mfma16(__builtin_bit_cast(h16x8, w), __builtin_bit_cast(h16x8, x), c);
}
// e4m3: the matrix instructions (this one and the 16x16x128 of gemm_w4.h alike) cut each product, towards zero, at 2^-13 of the
// binade of the largest of eight neighbours in K, and add in 32 bits from there on: sums are 1.4e-5 of their size off (K = 4096 and
// 8192, normal values), where the same values as bf16 are 2.5e-8 off.  The output's own rounding to bf16 is a hundred times that.
// Exact products would take the bf16 instructions: half the rate above 48 rows (4096 rows: 388 us against some 680).
__device__ __forceinline__ f32x4 mma(fp8e4, const u32x4& w, const u32x4& x, f32x4 c) {
    typedef long l2 __attribute__((ext_vector_type(2)));
    const l2 a = __builtin_bit_cast(l2, w), b = __builtin_bit_cast(l2, x);
    c = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a[0], b[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a[1], b[1], c, 0, 0, 0);
}
// PARTS: blockIdx.y takes per_part steps of K and leaves both projections' sums, [part][M][2 Fp] (see glu_finish_kernel).
template <typename TI, typename TO, int MT, int NC, int STEPS, bool PARTS>
__global__ __launch_bounds__(256) void glu_few_kernel(GluCall q, float* __restrict__ parts, int per_part) {
    constexpr int NW = 4;
    typedef u32x4 Q __attribute__((aligned(1)));
    constexpr int STEP = 128 / (int)sizeof(TI), E = 16 / (int)sizeof(TI);      // elements of a step, of a 16-byte load
    constexpr int G = 2 * NC;                                                  // weight tiles: tile g is matrix g & 1, columns 16 (g >> 1)
    __shared__ float red[NW][G][MT][16 * 17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = lane & 15, ch = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NC);
    const TI *pw[G], *px[MT];
#pragma unroll
    for (int g = 0; g < G; ++g)
        pw[g] = reinterpret_cast<const TI*>(q.w[g & 1]) + min(n0 + (g >> 1) * 16 + row, (int64_t)q.F - 1) * q.ldw[g & 1] + ch * E;
#pragma unroll
    for (int t = 0; t < MT; ++t) px[t] = reinterpret_cast<const TI*>(q.x) + (int64_t)min(t * 16 + row, q.M - 1) * q.ldx + ch * E;
    f32x4 acc[G][MT] = {};
    const int steps = q.K / STEP;                              // whole ones
    const int first = PARTS ? (int)blockIdx.y * per_part : 0, end = PARTS ? min(steps, first + per_part) : steps;
    auto run = [&](auto U_, int s) {                           // the loads of U steps go out together
        constexpr int U = decltype(U_)::value;
        u32x4 w[U][G][2], x[U][MT][2];
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int64_t at = (int64_t)(s + i * NW) * STEP + c * (STEP / 2);
#pragma unroll
                for (int g = 0; g < G; ++g) w[i][g][c] = *reinterpret_cast<const Q*>(pw[g] + at);
#pragma unroll
                for (int t = 0; t < MT; ++t) x[i][t][c] = *reinterpret_cast<const Q*>(px[t] + at);
            }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int g = 0; g < G; ++g)
#pragma unroll
                    for (int t = 0; t < MT; ++t) acc[g][t] = mma(TI{}, w[i][g][c], x[i][t][c], acc[g][t]);
    };
    int s = first + wave;
    if constexpr (STEPS > 1)
        for (; s + (STEPS - 1) * NW < end; s += STEPS * NW) run(std::integral_constant<int, STEPS>{}, s);
    for (; s < end; s += NW) run(std::integral_constant<int, 1>{}, s);
    if (steps * STEP < q.K && end == steps && wave == steps % NW && (!PARTS || blockIdx.y == gridDim.y - 1)) {
        auto part = [&](const TI* p, int c) {                  // 16 bytes of the step, zeros past the end of the row
            TI v[E];
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[j] = TI{};
                if (steps * STEP + c * (STEP / 2) + ch * E + j < q.K) v[j] = p[(int64_t)steps * STEP + c * (STEP / 2) + j];
            }
            u32x4 o;
            __builtin_memcpy(&o, v, 16);
            return o;
        };
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            u32x4 xv[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) xv[t] = part(px[t], c);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const u32x4 wv = part(pw[g], c);
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[g][t] = mma(TI{}, wv, xv[t], acc[g][t]);
            }
        }
    }
    // accumulators: the lane's low bits are the token, its four registers four columns
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) red[wave][g][t][(ch * 4 + e) * 17 + row] = acc[g][t][e];
    __syncthreads();
    for (int i = tid; i < NC * MT * 256; i += NW * 64) {
        const int col = i & 15, nc = (i >> 4) % NC, tok = (i / (16 * NC)) & 15, t = i / (256 * NC);
        const int64_t m = t * 16 + tok, nn = n0 + nc * 16 + col;
        if (m >= q.M || nn >= q.F) continue;
        float v[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            v[g] = red[0][2 * nc + g][t][col * 17 + tok];
#pragma unroll
            for (int w = 1; w < NW; ++w) v[g] += red[w][2 * nc + g][t][col * 17 + tok];
            if constexpr (PARTS) {
                const int64_t Fp = (q.F + 7) & ~7;
                parts[((int64_t)blockIdx.y * q.M + m) * (2 * Fp) + g * Fp + nn] = v[g];
                continue;
            }
            if (sizeof(TI) == 1) v[g] *= q.xs[m] * q.ws[g][nn];
            if (q.b[g]) v[g] += (float)reinterpret_cast<const TO*>(q.b[g])[nn];
            if (q.pre[g]) reinterpret_cast<TO*>(q.pre[g])[m * q.ldp + nn] = (TO)v[g];
        }
        if constexpr (!PARTS) reinterpret_cast<TO*>(q.h)[m * q.ldh + nn] = (TO)(act_of(v[0], q.act) * v[1]);
    }
}

// h (and the projections) from the parts of K [splits][M][2 Fp], Fp = F rounded up to 8: added up in their order, then what the
// one-pass kernels do at their ends.  A lane takes four columns.
template <typename TO, bool SCALED>
__global__ __launch_bounds__(256) void glu_finish_kernel(GluCall q, const float* __restrict__ parts, int splits) {
    typedef TO A4 __attribute__((ext_vector_type(4), aligned(2)));
    const int64_t Fp = (q.F + 7) & ~7, per = Fp / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= q.M * per) return;
    const int64_t m = i / per;
    const int n = (int)(i - m * per) * 4;
    f32x4 v[2];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const float* p = parts + m * (2 * Fp) + g * Fp + n;
        v[g] = *reinterpret_cast<const f32x4*>(p);
        for (int s = 1; s < splits; ++s) v[g] += *reinterpret_cast<const f32x4*>(p + (int64_t)s * q.M * (2 * Fp));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (n + j >= q.F) continue;
            if (SCALED) v[g][j] *= q.xs[m] * q.ws[g][n + j];
            if (q.b[g]) v[g][j] += (float)reinterpret_cast<const TO*>(q.b[g])[n + j];
        }
    }
    const A4 o = {(TO)(act_of(v[0][0], q.act) * v[1][0]), (TO)(act_of(v[0][1], q.act) * v[1][1]), (TO)(act_of(v[0][2], q.act) * v[1][2]),
                  (TO)(act_of(v[0][3], q.act) * v[1][3])};
    auto put = [&](TO* to, const A4& a) {
        if (n + 4 <= q.F) {
            *reinterpret_cast<A4*>(to) = a;
        } else {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (n + j < q.F) to[j] = a[j];
        }
    };
    put(reinterpret_cast<TO*>(q.h) + m * q.ldh + n, o);
#pragma unroll
    for (int g = 0; g < 2; ++g)
        if (q.pre[g]) put(reinterpret_cast<TO*>(q.pre[g]) + m * q.ldp + n, A4{(TO)v[g][0], (TO)v[g][1], (TO)v[g][2], (TO)v[g][3]});
}

// ---- the gradient -------------------------------------------------------------------------------------------------
// The products of the gradient contract over F (dx) and over the rows (dWg, dWu): along the rows of the weights, of x and of
// dg | du.  The matrix-core kernel takes one such operand as it lies and transposes it on the way into registers (gemm_w4.h,
// TrArgs): the weights and x.  dg | du is written both ways round by the kernel that computes it.  4096 rows, [4096, 11008]: the
// two products take 537 us each, with weights and x transposed beforehand 516 us each and 95 us more for that; with dg | du
// transposed in registers too 622 us for dW (those reads run at half the rate and both operands' fill the LDS pipe) against
// 29 us for writing it twice.
// What is contracted is padded to whole K tiles of 64: dg | du by the kernel that computes it, the others' last tile by a
// copy of its own.
constexpr int64_t up64(int64_t v) { return (v + 63) & ~(int64_t)63; }
constexpr int64_t up8(int64_t v) { return (v + 7) & ~(int64_t)7; }

// Up to three matrices of the same width into zero-padded rows of their own stride.
struct Copies {
    const void* src[3];
    void* dst[3];
    int64_t ld_src[3], ld_dst[3];
    int rows[3], rows_p[3];         // rows of the source, rows written (0: not this one)
    int cols, cols_p;               // columns of the source, columns written (a multiple of 8)
    int64_t chunks;                 // of all of them: 8 columns each
};
template <typename T> __device__ __forceinline__ void copy_rows_of(const Copies& q, int64_t block, int64_t blocks) {
    const int per = q.cols_p / 8;
    const int64_t n0 = (int64_t)q.rows_p[0] * per, n1 = n0 + (int64_t)q.rows_p[1] * per;
    for (int64_t i = block * 256 + threadIdx.x; i < q.chunks; i += blocks * 256) {
        const int k = i < n0 ? 0 : i < n1 ? 1 : 2;
        const int64_t at = i - (k == 0 ? 0 : k == 1 ? n0 : n1), r = at / per;
        const int c = (int)(at - r * per) * 8;
        typename vec8<T>::type v = {};
        if (r < q.rows[k]) {
            v = load8(reinterpret_cast<const T*>(q.src[k]) + r * q.ld_src[k], c, q.cols);
            fit(v, c, q.cols);
        }
        *reinterpret_cast<typename vec8<T>::type*>(reinterpret_cast<T*>(q.dst[k]) + r * q.ld_dst[k] + c) = v;
    }
}
template <typename T>
__global__ __launch_bounds__(256) void copy_rows_kernel(Copies q) {
    copy_rows_of<T>(q, blockIdx.x, gridDim.x);
}
constexpr int64_t COPY_BLOCKS = 2048;       // at most
void count(Copies& c, int cols, int cols_p) {
    c.cols = cols;
    c.cols_p = cols_p;
    c.chunks = ((int64_t)c.rows_p[0] + c.rows_p[1] + c.rows_p[2]) * (cols_p / 8);
}

// The biases' gradients: db [2 F] = sum of the row tiles' column sums [tiles][2 Fp], 64 columns a block.
struct ColumnSums {
    const float* sums;
    int tiles, F, Fp;
    void* db;
    __host__ unsigned blocks() const { return sums ? 2 * (unsigned)((F + 63) / 64) : 0; }
};
template <typename T> __device__ __forceinline__ void column_sums_of(const ColumnSums& q, int b) {
    __shared__ float red[4][64];
    const int per = (q.F + 63) / 64, half = b / per, l = threadIdx.x & 63, c = (b - half * per) * 64 + l, w = threadIdx.x >> 6;
    float s = 0.f;
    if (c < q.F)
        for (int i = w; i < q.tiles; i += 4) s += q.sums[(int64_t)i * (2 * q.Fp) + half * q.Fp + c];
    red[w][l] = s;
    __syncthreads();
    if (w == 0 && c < q.F) reinterpret_cast<T*>(q.db)[half * q.F + c] = (T)((red[0][l] + red[1][l]) + (red[2][l] + red[3][l]));
}

template <typename T>
__global__ __launch_bounds__(256) void column_sums_kernel(ColumnSums q) {
    column_sums_of<T>(q, blockIdx.x);
}

// A 64 x 64 tile in LDS, written by rows and read by columns: 16-byte chunks, the chunk index XORed with row / 8 so that the
// eight rows a lane gathers a column chunk from and the lanes' neighbouring columns fall into different banks.
template <typename T>
__device__ __forceinline__ void tile_put(T* t, int row, int chunk, const typename vec8<T>::type& v) {
    *reinterpret_cast<typename vec8<T>::type*>(t + row * 64 + ((chunk ^ (row >> 3)) << 3)) = v;
}
template <typename T>
__device__ __forceinline__ typename vec8<T>::type tile_get_t(const T* t, int col, int rchunk) {      // rows 8 rchunk .. + 7 of a column
    typename vec8<T>::type v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = t[(rchunk * 8 + j) * 64 + (((col >> 3) ^ rchunk) << 3) + (col & 7)];
    return v;
}

// dg and du are rounded to the type here, as the operands of the matrix instructions have to be.  With x, the weights and the
// results rounded as well that makes the gradients' error 1.4 times that of products of unrounded dg and du (bf16 2.34e-3 against
// 1.65e-3 of their norm, f16 2.93e-4 against 2.07e-4: one rounding more of the same size).  Kept, because the next better form, each
// value as the sum of two, doubles the products (4096 rows, [4096, 11008]: 1070 of 1185 us).  In f16 a dg or du past 65504 becomes
// infinite, and with it the gradients that take it, as any f16 gradient does there: callers scale their loss for that.
//
// dg | du as rows [M, 2 Fp] in K tiles of 64 - `whole` tiles of dg, as many of du, then the last of dg and of du if there is one
// more, zeros behind column F - and as columns [2 F, Mp], zeros behind row M; colsum: the tile's column sums [row tile][2 Fp]
// (or null).  Grid (Fp / 64, Mp / 64 + rows of blocks for the copies).  One read of dh, g, u; two writes of dg and du.
template <typename T>
__global__ __launch_bounds__(256) void glu_grad_kernel(const T* __restrict__ dh, int64_t ldh, const T* __restrict__ gate, int64_t ldg,
                                                       const T* __restrict__ up, int64_t ldu, T* __restrict__ dgu, T* __restrict__ dgut,
                                                       float* __restrict__ colsum, int M, int F, int Fp, int Mp, int whole, int act,
                                                       Copies copies) {
    typedef typename vec8<T>::type V;
    __shared__ __attribute__((aligned(16))) T tg[64 * 64], tu[64 * 64];
    __shared__ float cs[2][4][64];
    const int row_tiles = Mp / 64;
    if ((int)blockIdx.y >= row_tiles) {
        copy_rows_of<T>(copies, (int64_t)(blockIdx.y - row_tiles) * gridDim.x + blockIdx.x, (int64_t)(gridDim.y - row_tiles) * gridDim.x);
        return;
    }
    const int64_t m0 = (int64_t)blockIdx.y * 64;
    const int f0 = blockIdx.x * 64, ch = threadIdx.x & 7, c = f0 + ch * 8;
    float sg[8] = {}, su[8] = {};
    V dv[2], gv[2], uv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {                           // all loads first
        const int64_t m = min(m0 + (threadIdx.x >> 3) + 32 * i, (int64_t)M - 1);
        dv[i] = load8(dh + m * ldh, c, F);
        gv[i] = load8(gate + m * ldg, c, F);
        uv[i] = load8(up + m * ldu, c, F);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = (threadIdx.x >> 3) + 32 * i;
        const int64_t m = m0 + r;
        V og = {}, ou = {};
        if (m < M) {
            V &d = dv[i], &g = gv[i], &u = uv[i];
            fit(d, c, F);
            fit(g, c, F);
            fit(u, c, F);
#pragma unroll
            for (int j = 0; j < 8; ++j) {                   // (zeros behind column F: dg = du = 0 there)
                float a, da;
                act_grad((float)g[j], act, a, da);
                const float vg = (float)d[j] * (float)u[j] * da, vu = (float)d[j] * a;
                sg[j] += vg;
                su[j] += vu;
                og[j] = (T)vg;
                ou[j] = (T)vu;
            }
            T* row = dgu + m * (2 * (int64_t)Fp) + ch * 8;
            const int tile = blockIdx.x;
            *reinterpret_cast<V*>(row + (tile < whole ? tile : 2 * whole) * 64) = og;
            *reinterpret_cast<V*>(row + (tile < whole ? whole + tile : 2 * whole + 1) * 64) = ou;
        }
        tile_put(tg, r, ch, og);
        tile_put(tu, r, ch, ou);
    }
    if (colsum) {       // over the 8 rows of a wave and pass, then over the waves, in a fixed order
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int o = 8; o < 64; o <<= 1) {
                sg[j] += __shfl_xor(sg[j], o, 64);
                su[j] += __shfl_xor(su[j], o, 64);
            }
            if ((threadIdx.x & 63) < 8) {
                cs[0][threadIdx.x >> 6][ch * 8 + j] = sg[j];
                cs[1][threadIdx.x >> 6][ch * 8 + j] = su[j];
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int f = (threadIdx.x >> 3) + 32 * i;
        if (f0 + f >= F) break;
        *reinterpret_cast<V*>(dgut + (int64_t)(f0 + f) * Mp + m0 + ch * 8) = tile_get_t(tg, f, ch);
        *reinterpret_cast<V*>(dgut + (int64_t)(F + f0 + f) * Mp + m0 + ch * 8) = tile_get_t(tu, f, ch);
    }
    if (colsum && threadIdx.x < 128) {
        const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
        colsum[(int64_t)blockIdx.y * (2 * Fp) + w * Fp + f0 + l] = (cs[w][0][l] + cs[w][1][l]) + (cs[w][2][l] + cs[w][3][l]);
    }
}
// out [M, N] = sum of the parts [splits][M, Np] (Np % 8 == 0), rounded once; a lane takes four columns, from chunk i0 on.
struct PartSum {
    const float* part;
    void* out;
    int64_t M, i0;
    int splits, N, Np;
    unsigned blocks;
};
template <typename T> __device__ __forceinline__ void add_parts_of(const PartSum& q, unsigned block) {
    const int64_t i = q.i0 + (int64_t)block * 256 + threadIdx.x;
    const int per = q.Np / 4;
    if (i >= q.M * per) return;
    const int64_t m = i / per;
    const int n = (int)(i - m * per) * 4;
    f32x4 s = *reinterpret_cast<const f32x4*>(q.part + m * q.Np + n);
    for (int k = 1; k < q.splits; ++k) s += *reinterpret_cast<const f32x4*>(q.part + ((int64_t)k * q.M + m) * q.Np + n);
    T* to = reinterpret_cast<T*>(q.out) + m * q.N + n;
    typedef T A4 __attribute__((ext_vector_type(4), aligned(2)));
    if (n + 4 <= q.N) {
        *reinterpret_cast<A4*>(to) = A4{(T)s[0], (T)s[1], (T)s[2], (T)s[3]};
    } else {
#pragma unroll
        for (int j = 0; j < 3; ++j)
            if (n + j < q.N) to[j] = (T)s[j];
    }
}
// Up to two such sums, and column sums by the blocks behind theirs.
template <typename T>
__global__ __launch_bounds__(256) void add_parts_kernel(PartSum a, PartSum b, ColumnSums cs) {
    const unsigned i = blockIdx.x;
    if (i < a.blocks) add_parts_of<T>(a, i);
    else if (i < a.blocks + b.blocks) add_parts_of<T>(b, i - a.blocks);
    else column_sums_of<T>(cs, (int)(i - a.blocks - b.blocks));
}

// How a product [M, N] over K (a multiple of 64) is cut: whole (0 parts: straight to 16 bits) where its 256 x 256 tiles fill
// half the chip, else 256 x 128 tiles in parts of K of at least 8 tiles, as many as there are CUs.  N % 8 != 0: always
// through 32 bits (the 16-bit stores are 16 bytes wide).
struct Cut {
    int splits, ks_per;
    bool narrow;
};
Cut cut(int64_t M, int N, int K) {
    const int64_t tm = (M + 255) / 256;
    const int nk = K / 64;
    const bool narrow = tm * ((N + 255) / 256) < 128;
    int64_t s = 1;
    if (narrow) {
        s = 256 / (tm * ((N + 127) / 128));
        if (s > nk / 8) s = nk / 8;
        if (s < 1) s = 1;
    }
    const int per = (int)((nk + s - 1) / s);
    const int splits = (nk + per - 1) / per;
    return {splits == 1 && N % 8 == 0 ? 0 : splits, per, narrow};
}
int64_t cut_bytes(int64_t M, int N, int K) { return (int64_t)cut(M, N, K).splits * M * up8(N) * 4; }

// Both products of the gradient in one launch (fpi_grad_pair): dx in parts of K first, then dw, in parts too if dw.splits > 0.
// Workgroup i takes items i, i + 256, .. of 256 x 128 tiles: the cuts are those that leave the longest workgroup the fewest K
// tiles of about 0.7 us; an item counts 3 more (its first loads, its stores), what goes through 32 bits its traffic and launch.
// Taken where dx's 256 x 256 tiles fill less than half the chip and dw's are no more than 384: the whole gradient, one launch /
// two launches, us: 129 rows, [K, F] = [256, 512] 17 / 28; 729, [1152, 4304] (170 tiles) 62 / 71; 8000, [256, 1024] 66 / 80; 512,
// [2048, 5504] (344) 82 / 86; 1024, [2048, 8192] (512) 189 / 177: there 256 x 256 tiles, which stage less a product, win.
struct Pair {
    Cut dx, dw;                     // dx.splits == 0: not this way
};
Pair pair(int M, int F, int K) {
    const int nk = (int)up64(F) / 32, nk_w = (int)up64(M) / 64, tn = (K + 127) / 128;
    const int64_t t = (int64_t)((M + 255) / 256) * tn, t_w = (2 * (int64_t)F + 255) / 256 * tn;
    Pair best{{0, nk, true}, {0, nk_w, true}};
    if (!cut(M, K, 64 * nk).narrow || (2 * (int64_t)F + 255) / 256 * ((K + 255) / 256) > 384) return best;
    double least = 1e30;
    auto trial = [&](int s, int s_w) {
        const int per = (nk + s - 1) / s, per_w = (nk_w + s_w - 1) / s_w;
        const unsigned n = (unsigned)(t * ((nk + per - 1) / per)), n_w = (unsigned)(t_w * ((nk_w + per_w - 1) / per_w));
        const unsigned all = (n + n_w + 255) / 256, up = (n + 255) / 256, down = n / 256, rest = (n + n_w - n % 256 + 255) / 256;
        // workgroup 0, and the first with an item of dx less
        const unsigned most = std::max(up * (per + 3) + (all - up) * (per_w + 3), down * (per + 3) + (rest - down) * (per_w + 3));
        const bool parts_w = s_w > 1 || K % 8 != 0;        // (the 16-bit stores are 16 bytes wide)
        const double cost = most + (2.3e-6 * s * M * K) + (parts_w ? 2 + 2.3e-6 * s_w * 2 * F * K : 0);
        if (cost < least) {
            least = cost;
            best.dx = {(nk + per - 1) / per, per, true};
            best.dw = {parts_w ? (nk_w + per_w - 1) / per_w : 0, per_w, true};
        }
    };
    const int most_w = (int)std::min<int64_t>(nk_w / 8, 256 / t_w);
    for (int s = 1; s <= 32 && (s == 1 || nk / s >= 8); ++s) {
        trial(s, 1);
        if (most_w > 1) trial(s, most_w);
        if (most_w > 3) trial(s, most_w / 2);
    }
    return best;
}

// Rows up to which the weights are streamed (glu_few_kernel).  Streamed / matrix-core kernel, us, at 16, 32, 48 and 64 rows (64: with
// a fourth token tile, which is not built):
//   [K, F]         bf16                                          e4m3
//   [1152, 4304]   9.2 / 15   11.2 / 15   13.4 / 15   16 / 16    6.6 / 12   7.9 / 12   9.1 / 12   11 / 13
//   [2048, 5504]   15 / 18    17.6 / 19   21.5 / 19   26 / 20    8.8 / 17   10.7 / 18  13 / 18    15 / 19
//   [4096, 4096]   15 / 26    18.5 / 25   22 / 26     26 / 27    12 / 17    13 / 17    14 / 18    16 / 18
//   [4096, 11008]  48 / 51    53 / 52     60 / 53     69 / 53    23 / 30    27 / 32    33 / 32    37 / 33
//   [4096, 14336]  48 / 60    53 / 58     62 / 58     94 / 59    25 / 34    28 / 33    34 / 34    47 / 34
// One number for all: within 1 - 13 % of the better form at 33 - 48 rows in 16 bits, ahead of it or level in 8.
constexpr int FEW = 48;
constexpr int64_t FAR = int64_t(1) << 22;   // gemm_w4.h: 32-bit offsets within a tile
constexpr int MOST_F = 1 << 27;             // glu_few_kernel's lanes, 16 a column, have to stay below 2^32
constexpr int LIMIT = (1 << 20) - 64;      // M, F, K of the gradient: row strides of 2 F and 4 K stay below gemm_w4.h's limit of 2^22

bool aligned2(const void* p) { return ((uintptr_t)p & 1) == 0; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool wide_rows(const void* p, int64_t ld, int K) { return aligned16(p) && ld % 8 == 0 && ld < FAR && K % 64 == 0; }
// rows that the gradient's products read as they lie (K is not contracted there); their last K tile's copy has their stride
bool plain_rows(const void* p, int64_t ld, int K) { return aligned16(p) && ld % 8 == 0 && K % 8 == 0 && ld >= K && ld <= 4 * (int64_t)K; }

struct GradSpace {                  // byte offsets in the workspace, each a multiple of 256
    bool plain_x, plain_w;
    int64_t ldx, ldw;               // row strides as the products see them
    int64_t dgu, dgut, x, w, colsum, parts, end;         // x, w (gate, then up): the last K tile, or (not plain) all of it
};
GradSpace grad_space(const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu, int64_t M, int64_t F, int K) {
    const int64_t Fp = up64(F), Mp = up64(M), Kp = up8(K);
    GradSpace g;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += (bytes + 255) & ~(int64_t)255;
        return o;
    };
    g.plain_x = plain_rows(x, ldx, K);
    g.plain_w = plain_rows(wg, ldwg, K) && plain_rows(wu, ldwu, K) && ldwg == ldwu;
    g.ldx = g.plain_x ? ldx : Kp;
    g.ldw = g.plain_w ? ldwg : Kp;
    g.dgu = take(M * 2 * Fp * 2);
    g.dgut = take(2 * F * Mp * 2);
    g.x = take((g.plain_x ? (M % 64 ? 64 : 0) : Mp) * g.ldx * 2);
    g.w = take(2 * (g.plain_w ? (F % 64 ? 64 : 0) : Fp) * g.ldw * 2);
    g.colsum = take(Mp / 64 * 2 * Fp * 4);
    const Pair both = pair((int)M, (int)F, K);
    g.parts = take(both.dx.splits > 0 ? (both.dx.splits * M + both.dw.splits * 2 * F) * Kp * 4
                                      : std::max(cut_bytes(M, K, (int)(2 * Fp)), cut_bytes(2 * F, K, (int)Mp)));
    g.end = at;
    return g;
}

// out [M, N] = sum of the parts [splits][M, up8(N)], `also` with it; sums: taken along by the (first) launch, `sums.sums` is null
// from then on.  A launch's lanes have to stay below 2^32.
PartSum part_sum(const float* parts, int splits, void* out, int64_t M, int N) {
    const int64_t lanes = M * (up8(N) / 4);
    return {parts, out, M, 0, splits, N, (int)up8(N), (unsigned)((std::min(lanes, int64_t(1) << 30) + 255) / 256)};
}
template <typename T>
int add_parts(PartSum q, PartSum also, ColumnSums& sums, hipStream_t st) {
    for (PartSum* one : {&also, &q}) {                      // the rest of a sum of more lanes than one launch is given
        const int64_t lanes = one->M * (one->Np / 4);
        for (PartSum more = *one; (more.i0 += int64_t(1) << 30) < lanes;) {
            more.blocks = (unsigned)((std::min(lanes - more.i0, int64_t(1) << 30) + 255) / 256);
            add_parts_kernel<T><<<dim3(more.blocks), dim3(256), 0, st>>>(more, PartSum{}, ColumnSums{});
            FP_CHECK_LAUNCH();
        }
    }
    add_parts_kernel<T><<<dim3(q.blocks + also.blocks + sums.blocks()), dim3(256), 0, st>>>(q, also, sums);
    FP_CHECK_LAUNCH();
    sums.sums = nullptr;
    return 0;
}

// out [M, N] = the product, through fp32 parts where it is cut
template <typename T>
int product(GradProduct p, T* out, int N, float* parts, ColumnSums& sums, hipStream_t st) {
    const Cut c = cut(p.M, N, p.K);
    p.narrow = c.narrow;
    p.splits = c.splits;
    p.ks_per = c.ks_per;
    p.N = (int)up8(N);
    p.out = c.splits ? (void*)parts : (void*)out;
    if (int rc = fpi_grad_product(__is_same(T, bf16) ? FF_BF16 : FF_F16, p, st)) return rc;
    return c.splits == 0 ? 0 : add_parts<T>(part_sum(parts, c.splits, out, p.M, N), PartSum{}, sums, st);
}

// How a forward call runs.  e: bytes of an operand's element.
struct Plan {
    bool few, two;                  // stream the weights; two column tiles a workgroup
    bool x_fits, g_fits, u_fits;    // (not few) what the matrix-core kernel can read as it lies
    int splits, per;                // parts of K, steps (few) or K tiles of each; 1: no parts
    int64_t parts, bytes;           // where the parts begin in the workspace, and its end
};
Plan plan(int e, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu, int64_t M, int64_t F, int K) {
    Plan p{};
    p.few = M <= FEW;
    // two column tiles where that leaves a workgroup per CU; one for the fewest tokens in 16 bits
    p.two = F >= 8192 && (M > 8 || e == 1);
    p.x_fits = p.g_fits = p.u_fits = true;
    if (!p.few && e == 2) p.x_fits = wide_rows(x, ldx, K), p.g_fits = wide_rows(wg, ldwg, K), p.u_fits = wide_rows(wu, ldwu, K);
    // Parts of K where the output's tiles leave CUs idle and K is long enough to pay for the second launch: as many as there are
    // CUs, of at least 8 steps.  One launch / in parts, us: rows, [K, F] = 128, [4096, 4096] 49 / 28; 87, [6784, 120] 62 / 18;
    // 300, [2048, 1024] 24 / 20; 300, [1024, 1024] 15.3 / 16.4; streamed: 16, [8192, 1024] 24 / 14; 1, [2048, 1024] 6.4 / 7.4.
    const int64_t nk = (p.few ? (int64_t)K : up64(K)) * e / 128, tiles = p.few ? (F + 15) / 16 : (M + 255) / 256 * ((F + 63) / 64);
    int64_t s = 1;
    if (p.few ? tiles <= 64 && nk >= 64 : tiles <= 128 && nk >= 24) s = std::min(256 / tiles, nk / 8);
    p.per = (int)((nk + s - 1) / s);
    p.splits = p.per > 0 ? (int)((nk + p.per - 1) / p.per) : 1;
    const int64_t copied = (p.x_fits ? 0 : M) + (p.g_fits ? 0 : F) + (p.u_fits ? 0 : F);
    p.parts = (copied * up64(K) * 2 + 255) & ~(int64_t)255;
    p.bytes = p.splits > 1 ? p.parts + (int64_t)p.splits * M * 2 * up8(F) * 4 : copied * up64(K) * 2;
    return p;
}

template <typename TI, typename TO>
int ff_launch(const void* x, int64_t ldx, const float* xs, const void* wg, int64_t ldwg, const float* gs, const void* wu, int64_t ldwu,
              const float* us, const void* bg, const void* bu, void* h, int64_t ldh, void* gate, void* up, int64_t ldp, int M, int F,
              int K, int act, void* ws, int64_t ws_bytes, void* stream) {
    FP_REQUIRE(x && wg && wu && h && M >= 0 && F > 0 && K > 0 && (act == 0 || act == 1) && !bg == !bu && !gate == !up);
    FP_REQUIRE(M <= 1 << 30 && F <= MOST_F && K <= 1 << 30);
    FP_REQUIRE(ldx >= 0 && ldwg >= K && ldwu >= K && ldh >= F && (!gate || ldp >= F));
    FP_REQUIRE(sizeof(TI) == 1 || (aligned2(x) && aligned2(wg) && aligned2(wu) && aligned2(h) && aligned2(bg) && aligned2(bu) &&
                                   aligned2(gate) && aligned2(up)));
    if (M == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    constexpr int type = sizeof(TI) == 1 ? FF_E4M3 : __is_same(TI, bf16) ? FF_BF16 : FF_F16;
    const GluCall q{x, ldx, xs, {wg, wu}, {ldwg, ldwu}, {gs, us}, {bg, bu}, h, ldh, {gate, up}, ldp, M, F, K, act};
    const Plan p = plan(sizeof(TI), x, ldx, wg, ldwg, wu, ldwu, M, F, K);
    FP_REQUIRE(p.bytes == 0 || (ws && aligned16(ws) && ws_bytes >= p.bytes));
    float* parts = (float*)((char*)ws + p.parts);
    if (p.few) {
        const int mt = (M + 15) / 16;
#define FP_FEW(MT, NC, STEPS, PARTS)                                                                                                        \
    glu_few_kernel<TI, TO, MT, NC, STEPS, PARTS><<<dim3((unsigned)((F + 16 * NC - 1) / (16 * NC)), PARTS ? p.splits : 1), dim3(256), 0, st>>>( \
        q, parts, p.per)
        if (p.splits > 1) {
            if (mt == 1) FP_FEW(1, 1, 2, true);
            else if (mt == 2) FP_FEW(2, 1, 1, true);
            else FP_FEW(3, 1, 1, true);
        } else if (mt == 1) {
            if (p.two) FP_FEW(1, 2, 1, false);
            else FP_FEW(1, 1, 2, false);
        } else if (mt == 2) {
            if (p.two) FP_FEW(2, 2, 1, false);
            else FP_FEW(2, 1, 1, false);
        } else {
            if (p.two) FP_FEW(3, 2, 1, false);
            else FP_FEW(3, 1, 1, false);
        }
#undef FP_FEW
        FP_CHECK_LAUNCH();
    } else {
        // The matrix-core kernel stages its operands 16 bytes a lane and in whole K tiles, with 32-bit offsets inside a tile:
        // what does not fit that is copied into rows that do.
        int Kp = K;
        if constexpr (sizeof(TI) == 2) {
            if (!p.x_fits || !p.g_fits || !p.u_fits) {
                FP_REQUIRE(K <= LIMIT);
                Kp = (int)up64(K);
                TI *xp = (TI*)ws, *gp = xp + (p.x_fits ? 0 : (int64_t)M * Kp), *upk = gp + (p.g_fits ? 0 : (int64_t)F * Kp);
                Copies c{{x, wg, wu}, {xp, gp, upk}, {ldx, ldwg, ldwu}, {Kp, Kp, Kp}};
                c.rows[0] = c.rows_p[0] = p.x_fits ? 0 : M;
                c.rows[1] = c.rows_p[1] = p.g_fits ? 0 : F;
                c.rows[2] = c.rows_p[2] = p.u_fits ? 0 : F;
                count(c, K, Kp);
                copy_rows_kernel<TI><<<dim3((unsigned)std::min((c.chunks + 255) / 256, COPY_BLOCKS)), dim3(256), 0, st>>>(c);
                FP_CHECK_LAUNCH();
                if (!p.x_fits) x = xp, ldx = Kp;
                if (!p.g_fits) wg = gp, ldwg = Kp;
                if (!p.u_fits) wu = upk, ldwu = Kp;
            }
        }
        if (p.splits == 1)
            return fpi_glu(type, x, ldx, xs, wg, ldwg, gs, wu, ldwu, us, bg, bu, h, ldh, gate, up, ldp, M, F, Kp, act, st);
        if (int rc = fpi_glu_parts(type, x, ldx, wg, ldwg, wu, ldwu, parts, M, F, Kp, p.splits, p.per, st)) return rc;
    }
    if (p.splits > 1) {
        const int64_t lanes = (int64_t)M * (up8(F) / 4);
        glu_finish_kernel<TO, sizeof(TI) == 1><<<dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, st>>>(q, parts, p.splits);
        FP_CHECK_LAUNCH();
    }
    return 0;
}

template <typename T>
int ff_grad_launch(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
                   const void* gate, int64_t ldg, const void* up, int64_t ldu, void* dx, void* dw, void* db, int M, int F, int K, int act, void* ws, int64_t ws_bytes, void* stream) {
    FP_REQUIRE(dh && x && wg && wu && gate && up && dx && dw && (act == 0 || act == 1));
    FP_REQUIRE(aligned2(dh) && aligned2(x) && aligned2(wg) && aligned2(wu) && aligned2(gate) && aligned2(up) && aligned2(db));
    FP_REQUIRE(aligned16(dx) && aligned16(dw));
    FP_REQUIRE(M > 0 && F > 0 && K > 0 && ldh >= 0 && ldx >= 0 && ldg >= 0 && ldu >= 0 && ldwg >= K && ldwu >= K);
    FP_REQUIRE(M <= LIMIT && F <= LIMIT && K <= LIMIT);
    const GradSpace g = grad_space(x, ldx, wg, ldwg, wu, ldwu, M, F, K);
    FP_REQUIRE(ws && aligned16(ws) && ws_bytes >= g.end);
    hipStream_t st = (hipStream_t)stream;
    const int Fp = (int)up64(F), Mp = (int)up64(M), Kp = (int)up8(K);
    char* base = (char*)ws;
    T *dgu = (T*)(base + g.dgu), *dgut = (T*)(base + g.dgut), *xc = (T*)(base + g.x), *wc = (T*)(base + g.w);
    float *colsum = db ? (float*)(base + g.colsum) : nullptr, *parts = (float*)(base + g.parts);
    const int whole = g.plain_w ? F / 64 : Fp / 64, x_whole = g.plain_x ? M / 64 : Mp / 64, wc_rows = g.plain_w ? 64 : Fp;
    // what the products cannot read as it lies: all of it, or the rows of a partial last K tile
    const int xr = M % 64, wr = F % 64;
    Copies c{{x, wg, wu}, {xc, wc, wc + wc_rows * g.ldw}, {ldx, ldwg, ldwu}, {g.ldx, g.ldw, g.ldw}};
    if (g.plain_x) c.src[0] = (const T*)x + (int64_t)(M - xr) * ldx;
    if (g.plain_w) c.src[1] = (const T*)wg + (int64_t)(F - wr) * ldwg, c.src[2] = (const T*)wu + (int64_t)(F - wr) * ldwu;
    c.rows[0] = g.plain_x ? xr : M;
    c.rows_p[0] = g.plain_x ? (xr ? 64 : 0) : Mp;
    c.rows[1] = c.rows[2] = g.plain_w ? wr : F;
    c.rows_p[1] = c.rows_p[2] = g.plain_w ? (wr ? 64 : 0) : Fp;
    count(c, K, Kp);
    const int64_t copy_rows = (std::min((c.chunks + 255) / 256, COPY_BLOCKS) + Fp / 64 - 1) / (Fp / 64);       // of blocks
    glu_grad_kernel<T><<<dim3((unsigned)(Fp / 64), (unsigned)(Mp / 64 + copy_rows)), dim3(256), 0, st>>>(
        (const T*)dh, ldh, (const T*)gate, ldg, (const T*)up, ldu, dgu, dgut, colsum, M, F, Fp, Mp, whole, act, c);
    FP_CHECK_LAUNCH();
    ColumnSums sums{colsum, Mp / 64, F, Fp, db};
    const T *w0 = g.plain_w ? (const T*)wg : wc, *w1 = g.plain_w ? (const T*)wu : wc + wc_rows * g.ldw, *x0 = g.plain_x ? (const T*)x : xc;
    // where K tile t lies if one matrix went on: w0's tiles, w1's from tile `whole` on, the copies' from tile 2 whole on
    auto jump = [](const T* to, const T* from, int64_t tiles, int64_t ld) { return ((intptr_t)to - (intptr_t)from) - tiles * 64 * ld * 2; };
    GradProduct p{}, q{};
    p.a = dgu, p.lda = 2 * Fp, p.w = w0, p.ldw = g.ldw;
    p.s1 = whole, p.d1 = jump(w1, w0, whole, g.ldw);
    p.s2 = 2 * whole, p.d2 = jump(wc, w0, 2 * whole, g.ldw) - p.d1;
    p.M = M, p.K = 2 * Fp;
    q.a = dgut, q.lda = Mp, q.w = x0, q.ldw = g.ldx;
    q.s1 = x_whole, q.d1 = jump(xc, x0, x_whole, g.ldx);
    q.s2 = 1 << 30, q.d2 = 0;
    q.M = 2 * F, q.K = Mp;
    if (const Pair both = pair(M, F, K); both.dx.splits > 0) {
        float* parts_w = parts + (int64_t)both.dx.splits * M * Kp;
        p.splits = both.dx.splits, p.ks_per = both.dx.ks_per, p.out = parts;
        q.splits = both.dw.splits, q.ks_per = both.dw.ks_per, q.out = both.dw.splits > 0 ? (void*)parts_w : dw;
        p.N = q.N = Kp;
        if (int rc = fpi_grad_pair(__is_same(T, bf16) ? FF_BF16 : FF_F16, p, q, st)) return rc;
        return add_parts<T>(part_sum(parts, both.dx.splits, dx, M, K),
                            both.dw.splits > 0 ? part_sum(parts_w, both.dw.splits, dw, 2 * F, K) : PartSum{}, sums, st);
    }
    if (int rc = product<T>(p, (T*)dx, K, parts, sums, st)) return rc;
    if (int rc = product<T>(q, (T*)dw, K, parts, sums, st)) return rc;
    if (sums.sums) {
        column_sums_kernel<T><<<dim3(sums.blocks()), dim3(256), 0, st>>>(sums);
        FP_CHECK_LAUNCH();
    }
    return 0;
}

}  // namespace

extern "C" int64_t fp_gated_ff_workspace_bytes(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                                               int M, int F, int K) {
    if (M <= 0 || F <= 0 || K <= 0 || M > 1 << 30 || F > MOST_F || K > 1 << 30) return 0;
    return plan(2, x, ldx, w_gate, ldwg, w_up, ldwu, M, F, K).bytes;
}

extern "C" int64_t fp_gated_ff_fp8_workspace_bytes(int M, int F, int K) {
    if (M <= 0 || F <= 0 || K <= 0 || M > 1 << 30 || F > MOST_F || K > 1 << 30) return 0;
    return plan(1, nullptr, 0, nullptr, 0, nullptr, 0, M, F, K).bytes;
}

extern "C" int fp_gated_ff_bf16(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                                const void* b_gate, const void* b_up, void* h, int64_t ldh, void* gate, void* up, int64_t ldp, int M,
                                int F, int K, int act, void* workspace, int64_t workspace_bytes, void* stream) {
    return ff_launch<bf16, bf16>(x, ldx, nullptr, w_gate, ldwg, nullptr, w_up, ldwu, nullptr, b_gate, b_up, h, ldh, gate, up, ldp, M, F,
                                 K, act, workspace,
                                 workspace_bytes, stream);
}

extern "C" int fp_gated_ff_f16(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                               const void* b_gate, const void* b_up, void* h, int64_t ldh, void* gate, void* up, int64_t ldp, int M,
                               int F, int K, int act, void* workspace, int64_t workspace_bytes, void* stream) {
    return ff_launch<_Float16, _Float16>(x, ldx, nullptr, w_gate, ldwg, nullptr, w_up, ldwu, nullptr, b_gate, b_up, h, ldh, gate, up,
                                         ldp, M, F, K, act, workspace,
                                 workspace_bytes, stream);
}

extern "C" int fp_gated_ff_fp8(const void* x, int64_t ldx, const void* x_scale, const void* w_gate, int64_t ldwg, const void* wg_scale,
                               const void* w_up, int64_t ldwu, const void* wu_scale, const void* b_gate, const void* b_up, void* h,
                               int64_t ldh, int M, int F, int K, int act, void* workspace, int64_t workspace_bytes, void* stream) {
    FP_REQUIRE(x_scale && wg_scale && wu_scale && K > 0 && K % 128 == 0 && F > 0 && F % 8 == 0);
    FP_REQUIRE(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(h) && ldx % 16 == 0 && ldwg % 16 == 0 &&
               ldwu % 16 == 0 && ldh % 8 == 0 && ldx >= 0);
    FP_REQUIRE(((uintptr_t)x_scale & 3) == 0 && aligned16(wg_scale) && aligned16(wu_scale) && aligned16(b_gate) && aligned16(b_up));
    return ff_launch<fp8e4, bf16>(x, ldx, (const float*)x_scale, w_gate, ldwg, (const float*)wg_scale, w_up, ldwu,
                                  (const float*)wu_scale, b_gate, b_up, h, ldh, nullptr, nullptr, 0, M, F, K, act, workspace, workspace_bytes, stream);
}

extern "C" int64_t fp_gated_ff_backward_workspace_bytes(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up,
                                                        int64_t ldwu, int M, int F, int K) {
    if (M <= 0 || F <= 0 || K <= 0 || M > LIMIT || F > LIMIT || K > LIMIT) return 0;
    return grad_space(x, ldx, w_gate, ldwg, w_up, ldwu, M, F, K).end;
}

extern "C" int fp_gated_ff_backward_bf16(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* w_gate, int64_t ldwg,
                                         const void* w_up, int64_t ldwu, const void* gate, int64_t ldg, const void* up, int64_t ldu,
                                         void* dx, void* dw, void* db, int M, int F, int K, int act,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
    return ff_grad_launch<bf16>(dh, ldh, x, ldx, w_gate, ldwg, w_up, ldwu, gate, ldg, up, ldu, dx, dw, db, M, F, K,
                                act, workspace, workspace_bytes, stream);
}

extern "C" int fp_gated_ff_backward_f16(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* w_gate, int64_t ldwg,
                                        const void* w_up, int64_t ldwu, const void* gate, int64_t ldg, const void* up, int64_t ldu,
                                        void* dx, void* dw, void* db, int M, int F, int K, int act,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
    return ff_grad_launch<_Float16>(dh, ldh, x, ldx, w_gate, ldwg, w_up, ldwu, gate, ldg, up, ldu, dx, dw, db, M,
                                    F, K, act, workspace, workspace_bytes, stream);
}
