// K13: the gated feed-forward block's first half, h = act(x . Wg^T + bg) * (x . Wu^T + bu), act = SiLU or tanh-GELU, in
// bf16 / f16 and on e4m3 operands, and its gradient.  gfx950 / wave64; C-ABI entry points at the bottom, declarations in
// include/framepack_hip.h.
//
//   dg = dh u act'(g)   du = dh act(g)   dx = dg . Wg + du . Wu   dWg = dg^T . x   dWu = du^T . x   db = column sums
#include <type_traits>
#include "gated_ff.h"
#include "gemm_pipeline.h"
#include "row_access.h"

extern "C" int64_t fp_gated_ff_workspace_bytes(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                                               int M, int F, int K);
extern "C" int64_t fp_gated_ff_backward_workspace_bytes(int M, int F, int K);
extern "C" int fp_gemm_bf16(const void*, int64_t, const void*, int, const void*, int64_t, const void*, void*, int64_t, int, int, int, int,
                            int, const void*, int64_t, const void*, void*);
extern "C" int fp_gemm_f16(const void*, int64_t, const void*, int, const void*, int64_t, const void*, void*, int64_t, int, int, int, int,
                           int, const void*, int64_t, const void*, void*);

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
__device__ __forceinline__ f32x4 mma(fp8e4, const u32x4& w, const u32x4& x, f32x4 c) {
    typedef long l2 __attribute__((ext_vector_type(2)));
    const l2 a = __builtin_bit_cast(l2, w), b = __builtin_bit_cast(l2, x);
    c = __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a[0], b[0], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_fp8_fp8(a[1], b[1], c, 0, 0, 0);
}
template <typename TI, typename TO, int MT, int NC, int STEPS>
__global__ __launch_bounds__(256) void glu_few_kernel(GluCall q) {
    constexpr int NW = 4;
    typedef u32x4 Q __attribute__((aligned(1)));
    constexpr int STEP = 128 / (int)sizeof(TI), E = 16 / (int)sizeof(TI);      // elements of a step, of a 16-byte load
    constexpr int G = 2 * NC;                                                  // weight tiles: tile g is matrix g & 1, columns 16 (g >> 1)
    __shared__ float red[NW][G][MT][16 * 17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = lane & 15, ch = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * (16 * NC);
    const int m0 = blockIdx.y * (MT * 16);
    const TI *pw[G], *px[MT];
#pragma unroll
    for (int g = 0; g < G; ++g)
        pw[g] = reinterpret_cast<const TI*>(q.w[g & 1]) + min(n0 + (g >> 1) * 16 + row, (int64_t)q.F - 1) * q.ldw[g & 1] + ch * E;
#pragma unroll
    for (int t = 0; t < MT; ++t) px[t] = reinterpret_cast<const TI*>(q.x) + (int64_t)min(m0 + t * 16 + row, q.M - 1) * q.ldx + ch * E;
    f32x4 acc[G][MT] = {};
    const int steps = q.K / STEP;
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
    int s = wave;
    if constexpr (STEPS > 1)
        for (; s + (STEPS - 1) * NW < steps; s += STEPS * NW) run(std::integral_constant<int, STEPS>{}, s);
    for (; s < steps; s += NW) run(std::integral_constant<int, 1>{}, s);
    if (steps * STEP < q.K && wave == steps % NW) {
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
        const int64_t m = m0 + t * 16 + tok, nn = n0 + nc * 16 + col;
        if (m >= q.M || nn >= q.F) continue;
        float v[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            v[g] = red[0][2 * nc + g][t][col * 17 + tok];
#pragma unroll
            for (int w = 1; w < NW; ++w) v[g] += red[w][2 * nc + g][t][col * 17 + tok];
            if (sizeof(TI) == 1) v[g] *= q.xs[m] * q.ws[g][nn];
            if (q.b[g]) v[g] += (float)reinterpret_cast<const TO*>(q.b[g])[nn];
            if (q.pre[g]) reinterpret_cast<TO*>(q.pre[g])[m * q.ldp + nn] = (TO)v[g];
        }
        reinterpret_cast<TO*>(q.h)[m * q.ldh + nn] = (TO)(act_of(v[0], q.act) * v[1]);
    }
}

// ---- the gradient -------------------------------------------------------------------------------------------------
// The products of the gradient contract over F (dx) and over the rows (dWg, dWu), the matrix-core kernel over the unit
// stride of both operands: so dg | du is laid out both ways round by the kernel that computes it, and the weights and x
// are transposed.  Contracted lengths are zero-padded to whole K tiles of 64 in the workspace, which also takes care of
// sizes and strides that the wide loads cannot read.
constexpr int64_t up64(int64_t v) { return (v + 63) & ~(int64_t)63; }
constexpr int64_t up8(int64_t v) { return (v + 7) & ~(int64_t)7; }

// Up to three matrices of the same width into rows of Kp elements (a multiple of 64), zeros behind column K
struct Copies {
    const void* src[3];
    void* dst[3];
    int64_t ld[3];
    int rows[3];                    // 0: not this one
};
template <typename T>
__global__ __launch_bounds__(256) void copy_rows_kernel(Copies q, int K, int Kp) {
    const int per = Kp / 8;
    const int64_t n0 = (int64_t)q.rows[0] * per, n1 = n0 + (int64_t)q.rows[1] * per, n2 = n1 + (int64_t)q.rows[2] * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n2; i += (int64_t)gridDim.x * 256) {
        const int k = i < n0 ? 0 : i < n1 ? 1 : 2;
        const int64_t at = i - (k == 0 ? 0 : k == 1 ? n0 : n1), r = at / per;
        const int c = (int)(at - r * per) * 8;
        const T* src = reinterpret_cast<const T*>(k == 0 ? q.src[0] : k == 1 ? q.src[1] : q.src[2]);
        T* dst = reinterpret_cast<T*>(k == 0 ? q.dst[0] : k == 1 ? q.dst[1] : q.dst[2]);
        typename vec8<T>::type v = load8(src + r * (k == 0 ? q.ld[0] : k == 1 ? q.ld[1] : q.ld[2]), c, K);
        fit(v, c, K);
        *reinterpret_cast<typename vec8<T>::type*>(dst + r * Kp + c) = v;
    }
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

// dst[c][r] = src[r][c] for r < rows_p (a multiple of 8; zeros from `rows` on) and c < cols_p (zeros from cols on)
struct Transposes {                 // three of them in one launch, one after the other in blockIdx.x, 64 x 64 tiles
    const void* src[3];
    void* dst[3];
    int64_t ld_src[3], ld_dst[3];
    int rows[3], rows_p[3], tiles[3], cols, cols_p, col_tiles;
};
// behind them (if wanted) the biases' gradients: db = sum of the row tiles' column sums, 64 columns a block
struct ColumnSums {
    const float* sums;              // [tiles][2 S] (or null)
    int tiles, F, S;
    void *dbg, *dbu;
};
template <typename T>
__global__ __launch_bounds__(256) void transpose_kernel(Transposes t, ColumnSums cs) {
    __shared__ __attribute__((aligned(16))) T tile[64 * 64];
    int b = blockIdx.x, k = 0;
    while (k < 3 && b >= t.tiles[k]) b -= t.tiles[k++];
    if (k == 3) {
        float(*red)[64] = reinterpret_cast<float(*)[64]>(tile);
        const int per = (cs.F + 63) / 64, half = b / per, l = threadIdx.x & 63, c = (b - half * per) * 64 + l, q = threadIdx.x >> 6;
        float s = 0.f;
        if (c < cs.F)
            for (int i = q; i < cs.tiles; i += 4) s += cs.sums[(int64_t)i * (2 * cs.S) + half * cs.S + c];
        red[q][l] = s;
        __syncthreads();
        if (q == 0 && c < cs.F) reinterpret_cast<T*>(half ? cs.dbu : cs.dbg)[c] = (T)((red[0][l] + red[1][l]) + (red[2][l] + red[3][l]));
        return;
    }
    const T* src = reinterpret_cast<const T*>(t.src[k]);
    T* dst = reinterpret_cast<T*>(t.dst[k]);
    const int64_t r0 = (int64_t)(b / t.col_tiles) * 64;
    const int c0 = b % t.col_tiles * 64;
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int r = i >> 3, ch = i & 7;
        typename vec8<T>::type v = {};
        if (r0 + r < t.rows[k]) {
            v = load8(src + (r0 + r) * t.ld_src[k], c0 + ch * 8, t.cols);
            fit(v, c0 + ch * 8, t.cols);
        }
        tile_put(tile, r, ch, v);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {
        const int c = i >> 3, ch = i & 7;
        if (c0 + c < t.cols_p && r0 + ch * 8 < t.rows_p[k])
            *reinterpret_cast<typename vec8<T>::type*>(dst + (int64_t)(c0 + c) * t.ld_dst[k] + r0 + ch * 8) = tile_get_t(tile, c, ch);
    }
}

// dg | du as rows [M, Kd] - dg from column 0, du from column S on, S = F rounded up to 8, zeros in the gaps and behind them
// up to Kd - and as columns [2 S, Mp], zeros behind row M; colsum: the tile's column sums [row tile][2 S] (or null).
// Grid (ceil(S / 64), Mp / 64).  One read of dh, g, u; two writes of dg and du.
template <typename T>
__global__ __launch_bounds__(256) void glu_grad_kernel(const T* __restrict__ dh, int64_t ldh, const T* __restrict__ gate, int64_t ldg,
                                                       const T* __restrict__ up, int64_t ldu, T* __restrict__ dgu, T* __restrict__ dgut,
                                                       float* __restrict__ colsum, int M, int F, int S, int Kd, int Mp, int act) {
    typedef typename vec8<T>::type V;
    __shared__ __attribute__((aligned(16))) T tg[64 * 64], tu[64 * 64];
    __shared__ float cs[2][4][64];
    const int64_t m0 = (int64_t)blockIdx.y * 64;
    const int f0 = blockIdx.x * 64, ch = threadIdx.x & 7, c = f0 + ch * 8;
    const bool last = blockIdx.x == gridDim.x - 1;
    float sg[8] = {}, su[8] = {};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = (threadIdx.x >> 3) + 32 * i;
        const int64_t m = m0 + r;
        V og = {}, ou = {};
        if (m < M) {
            V d = load8(dh + m * ldh, c, F), g = load8(gate + m * ldg, c, F), u = load8(up + m * ldu, c, F);
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
            T* row = dgu + m * Kd;
            if (c < S) {
                *reinterpret_cast<V*>(row + c) = og;
                *reinterpret_cast<V*>(row + S + c) = ou;
            }
            if (last && 2 * S + ch * 8 < Kd) *reinterpret_cast<V*>(row + 2 * S + ch * 8) = V{};
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
        if (f0 + f >= S) break;
        *reinterpret_cast<V*>(dgut + (int64_t)(f0 + f) * Mp + m0 + ch * 8) = tile_get_t(tg, f, ch);
        *reinterpret_cast<V*>(dgut + (int64_t)(S + f0 + f) * Mp + m0 + ch * 8) = tile_get_t(tu, f, ch);
    }
    if (colsum && threadIdx.x < 128) {
        const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
        if (f0 + l < S)
            colsum[(int64_t)blockIdx.y * (2 * S) + w * S + f0 + l] = (cs[w][0][l] + cs[w][1][l]) + (cs[w][2][l] + cs[w][3][l]);
    }
}
// out [M, N] = sum of the parts [splits][M, Np] (Np % 8 == 0), rounded once; a lane takes four columns
template <typename T>
__global__ __launch_bounds__(256) void add_parts_kernel(const float* __restrict__ part, int splits, T* __restrict__ out, int64_t M, int N, int Np) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int per = Np / 4;
    if (i >= M * per) return;
    const int64_t m = i / per;
    const int n = (int)(i - m * per) * 4;
    f32x4 s = *reinterpret_cast<const f32x4*>(part + m * Np + n);
    for (int k = 1; k < splits; ++k) s += *reinterpret_cast<const f32x4*>(part + ((int64_t)k * M + m) * Np + n);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (n + j < N) out[m * N + n + j] = (T)s[j];
}

// How a product [M, N] over K (a multiple of 64) is cut: whole (0 parts: straight to 16 bits) where its 256 x 256 tiles fill
// half the chip, else 256 x 128 tiles in parts of K of at least 8 tiles, as many as there are CUs.  N % 8 != 0: always
// through 32 bits (the 16-bit stores are 16 bytes wide).
struct Cut {
    int splits, ks_per;
};
Cut cut(int64_t M, int N, int K) {
    const int64_t tm = (M + 255) / 256;
    const int nk = K / 64;
    int64_t s = 1;
    if (tm * ((N + 255) / 256) < 128) {
        s = 256 / (tm * ((N + 127) / 128));
        if (s > nk / 8) s = nk / 8;
        if (s < 1) s = 1;
    }
    const int per = (int)((nk + s - 1) / s);
    const int splits = (nk + per - 1) / per;
    return {splits == 1 && N % 8 == 0 ? 0 : splits, per};
}
int64_t cut_bytes(int64_t M, int N, int K) { return (int64_t)cut(M, N, K).splits * M * up8(N) * 4; }

struct GradSpace {                  // byte offsets in the workspace, each a multiple of 256
    int64_t dgu, dgut, wt, xt, colsum, parts, end;
};
GradSpace grad_space(int64_t M, int64_t F, int64_t K) {
    const int64_t S = up8(F), Kd = up64(2 * S), Mp = up64(M), Kp = up8(K);
    GradSpace g;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t o = at;
        at += (bytes + 255) & ~(int64_t)255;
        return o;
    };
    g.dgu = take(M * Kd * 2);
    g.dgut = take(2 * S * Mp * 2);
    g.wt = take(Kp * Kd * 2);
    g.xt = take(Kp * Mp * 2);
    g.colsum = take(Mp / 64 * 2 * S * 4);
    const int64_t a = cut_bytes(M, (int)K, (int)Kd), b = cut_bytes(F, (int)K, (int)Mp), c = cut_bytes(2 * F, (int)K, (int)Mp);
    g.parts = take(a > b ? (a > c ? a : c) : (b > c ? b : c));
    g.end = at;
    return g;
}

// out [M, N] = a [M, K] . w [up8(N), K]^T, K a multiple of 64 and everything in the workspace's layout
template <typename T>
int product(const T* a, int64_t lda, const T* w, int64_t ldw, T* out, int M, int N, int K, float* parts, hipStream_t st) {
    constexpr int type = sizeof(T) == 2 && __is_same(T, bf16) ? FF_BF16 : FF_F16;
    const Cut c = cut(M, N, K);         // (splits > 1 means few tiles: the narrow tile)
    if (c.splits == 0)
        return (type == FF_BF16 ? fp_gemm_bf16 : fp_gemm_f16)(a, lda, nullptr, 0, w, ldw, nullptr, out, N, M, N, K, 0, 0, nullptr, 0, nullptr, st);
    const int Np = (int)up8(N);
    if (int rc = fpi_gemm_parts(type, c.splits > 1, a, lda, w, ldw, parts, M, Np, K, c.splits, c.ks_per, st)) return rc;
    add_parts_kernel<T><<<dim3((unsigned)(((int64_t)M * (Np / 4) + 255) / 256)), dim3(256), 0, st>>>(parts, c.splits, out, M, N, Np);
    FP_CHECK_LAUNCH();
    return 0;
}

// Rows up to which the weights are streamed (glu_few_kernel).  [K, F] = [4096, 14336], streamed / matrix-core kernel, us:
// bf16 45 / 70 at 1 row, 56 / 69 at 32, 64 / 71 at 48, 70 / 73 at 64; e4m3 21 / 30 at 1, 32 / 34 at 48, 37 / 35 at 64.
constexpr int FEW = 48;
constexpr int64_t FAR = int64_t(1) << 22;   // gemm_w4.h: 32-bit offsets within a tile
constexpr int LIMIT = (1 << 21) - 64;      // M, F, K of the gradient: Kd and Mp stay below gemm_w4.h's limit of 2^22 for a row stride

bool aligned2(const void* p) { return ((uintptr_t)p & 1) == 0; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool wide_rows(const void* p, int64_t ld, int K) { return aligned16(p) && ld % 8 == 0 && ld < FAR && K % 64 == 0; }

template <typename TI, typename TO>
int ff_launch(const void* x, int64_t ldx, const float* xs, const void* wg, int64_t ldwg, const float* gs, const void* wu, int64_t ldwu,
              const float* us, const void* bg, const void* bu, void* h, int64_t ldh, void* gate, void* up, int64_t ldp, int M, int F,
              int K, int act, void* ws, int64_t ws_bytes, void* stream) {
    FP_REQUIRE(x && wg && wu && h && M >= 0 && F > 0 && K > 0 && (act == 0 || act == 1) && !bg == !bu && !gate == !up);
    FP_REQUIRE(ldx >= 0 && ldwg >= K && ldwu >= K && ldh >= F && (!gate || ldp >= F));
    FP_REQUIRE(sizeof(TI) == 1 || (aligned2(x) && aligned2(wg) && aligned2(wu) && aligned2(h) && aligned2(bg) && aligned2(bu) &&
                                   aligned2(gate) && aligned2(up)));
    if (M == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    constexpr int type = sizeof(TI) == 1 ? FF_E4M3 : __is_same(TI, bf16) ? FF_BF16 : FF_F16;
    const GluCall q{x, ldx, xs, {wg, wu}, {ldwg, ldwu}, {gs, us}, {bg, bu}, h, ldh, {gate, up}, ldp, M, F, K, act};
    if (M <= FEW) {
        const int mt = (M + 15) / 16;
        // two column tiles a workgroup where that leaves a workgroup per CU; one for the fewest tokens in 16 bits
        const bool two = F >= 8192 && (M > 8 || sizeof(TI) == 1);
#define FP_FEW(MT, NC, STEPS) glu_few_kernel<TI, TO, MT, NC, STEPS><<<dim3((unsigned)((F + 16 * NC - 1) / (16 * NC))), dim3(256), 0, st>>>(q)
        if (mt == 1) {
            if (two) FP_FEW(1, 2, 1);
            else FP_FEW(1, 1, 2);
        } else if (mt == 2) {
            if (two) FP_FEW(2, 2, 1);
            else FP_FEW(2, 1, 1);
        } else {
            if (two) FP_FEW(3, 2, 1);
            else FP_FEW(3, 1, 1);
        }
#undef FP_FEW
        FP_CHECK_LAUNCH();
        return 0;
    }
    // The matrix-core kernel stages its operands 16 bytes a lane and in whole K tiles, with 32-bit offsets inside a tile: what
    // does not fit that is copied into rows that do.
    if constexpr (sizeof(TI) == 2) {
        const bool x_fits = wide_rows(x, ldx, K), g_fits = wide_rows(wg, ldwg, K), u_fits = wide_rows(wu, ldwu, K);
        if (!x_fits || !g_fits || !u_fits) {
            const int64_t Kp = up64(K);
            FP_REQUIRE(K <= LIMIT && F <= LIMIT && ws && aligned16(ws) &&
                       ws_bytes >= fp_gated_ff_workspace_bytes(x, ldx, wg, ldwg, wu, ldwu, M, F, K));
            TI *xp = (TI*)ws, *gp = xp + (x_fits ? 0 : M * Kp), *upk = gp + (g_fits ? 0 : F * Kp);
            const Copies c{{x, wg, wu}, {xp, gp, upk}, {ldx, ldwg, ldwu}, {x_fits ? 0 : M, g_fits ? 0 : F, u_fits ? 0 : F}};
            const int64_t chunks = ((int64_t)c.rows[0] + c.rows[1] + c.rows[2]) * (Kp / 8);
            copy_rows_kernel<TI><<<dim3((unsigned)(chunks < 2048 * 256 ? (chunks + 255) / 256 : 2048)), dim3(256), 0, st>>>(c, K, (int)Kp);
            FP_CHECK_LAUNCH();
            return fpi_glu(type, x_fits ? x : xp, x_fits ? ldx : Kp, xs, g_fits ? wg : gp, g_fits ? ldwg : Kp, gs, u_fits ? wu : upk,
                           u_fits ? ldwu : Kp, us, bg, bu, h, ldh, gate, up, ldp, M, F, (int)Kp, act, st);
        }
    }
    return fpi_glu(type, x, ldx, xs, wg, ldwg, gs, wu, ldwu, us, bg, bu, h, ldh, gate, up, ldp, M, F, K, act, st);
}

template <typename T>
int ff_grad_launch(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
                   const void* gate, int64_t ldg, const void* up, int64_t ldu, void* dx, void* dwg, void* dwu, void* dbg, void* dbu,
                   int M, int F, int K, int act, void* ws, int64_t ws_bytes, void* stream) {
    FP_REQUIRE(dh && x && wg && wu && gate && up && dx && dwg && dwu && !dbg == !dbu && (act == 0 || act == 1));
    FP_REQUIRE(aligned2(dh) && aligned2(x) && aligned2(wg) && aligned2(wu) && aligned2(gate) && aligned2(up) && aligned2(dbg) && aligned2(dbu));
    FP_REQUIRE(aligned16(dx) && aligned16(dwg) && (K % 8 != 0 ? aligned2(dwu) : aligned16(dwu)));
    FP_REQUIRE(M > 0 && F > 0 && K > 0 && ldh >= 0 && ldx >= 0 && ldg >= 0 && ldu >= 0 && ldwg >= K && ldwu >= K);
    FP_REQUIRE(M <= LIMIT && F <= LIMIT && K <= LIMIT);
    FP_REQUIRE(ws && aligned16(ws) && ws_bytes >= fp_gated_ff_backward_workspace_bytes(M, F, K));
    hipStream_t st = (hipStream_t)stream;
    const GradSpace g = grad_space(M, F, K);
    const int S = (int)up8(F), Kd = (int)up64(2 * S), Mp = (int)up64(M), Kp = (int)up8(K), ktiles = (Kp + 63) / 64;
    char* base = (char*)ws;
    T *dgu = (T*)(base + g.dgu), *dgut = (T*)(base + g.dgut), *wt = (T*)(base + g.wt), *xt = (T*)(base + g.xt);
    float *colsum = dbg ? (float*)(base + g.colsum) : nullptr, *parts = (float*)(base + g.parts);
    glu_grad_kernel<T><<<dim3((unsigned)((S + 63) / 64), (unsigned)(Mp / 64)), dim3(256), 0, st>>>(
        (const T*)dh, ldh, (const T*)gate, ldg, (const T*)up, ldu, dgu, dgut, colsum, M, F, S, Kd, Mp, act);
    FP_CHECK_LAUNCH();
    const int up_rows = Kd - S;
    const Transposes t{{wg, wu, x}, {wt, wt + S, xt}, {ldwg, ldwu, ldx}, {Kd, Kd, Mp}, {F, F, M}, {S, up_rows, Mp},
                       {(S + 63) / 64 * ktiles, (up_rows + 63) / 64 * ktiles, Mp / 64 * ktiles}, K, Kp, ktiles};
    const ColumnSums cs{colsum, Mp / 64, F, S, dbg, dbu};
    transpose_kernel<T><<<dim3((unsigned)(t.tiles[0] + t.tiles[1] + t.tiles[2] + (dbg ? 2 * ((F + 63) / 64) : 0))), dim3(256), 0, st>>>(t, cs);
    FP_CHECK_LAUNCH();
    if (int rc = product<T>(dgu, Kd, wt, Kd, (T*)dx, M, K, Kd, parts, st)) return rc;
    // (dWg over dWu in one product where they are the halves of one matrix)
    if (S == F && (T*)dwu == (T*)dwg + (int64_t)F * K) return product<T>(dgut, Mp, xt, Mp, (T*)dwg, 2 * F, K, Mp, parts, st);
    if (int rc = product<T>(dgut, Mp, xt, Mp, (T*)dwg, F, K, Mp, parts, st)) return rc;
    return product<T>(dgut + (int64_t)S * Mp, Mp, xt, Mp, (T*)dwu, F, K, Mp, parts, st);
}

}  // namespace

extern "C" int64_t fp_gated_ff_workspace_bytes(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                                               int M, int F, int K) {
    if (M <= FEW || F <= 0 || K <= 0 || F > LIMIT || K > LIMIT) return 0;
    const int64_t rows = (wide_rows(x, ldx, K) ? 0 : (int64_t)M) + (wide_rows(w_gate, ldwg, K) ? 0 : (int64_t)F) +
                         (wide_rows(w_up, ldwu, K) ? 0 : (int64_t)F);
    return rows * up64(K) * 2;
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
                               int64_t ldh, int M, int F, int K, int act, void* stream) {
    FP_REQUIRE(x_scale && wg_scale && wu_scale && K > 0 && K % 128 == 0 && F > 0 && F % 8 == 0);
    FP_REQUIRE(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(h) && ldx % 16 == 0 && ldwg % 16 == 0 &&
               ldwu % 16 == 0 && ldh % 8 == 0 && ldx >= 0);
    FP_REQUIRE(((uintptr_t)x_scale & 3) == 0 && aligned16(wg_scale) && aligned16(wu_scale) && aligned16(b_gate) && aligned16(b_up));
    return ff_launch<fp8e4, bf16>(x, ldx, (const float*)x_scale, w_gate, ldwg, (const float*)wg_scale, w_up, ldwu,
                                  (const float*)wu_scale, b_gate, b_up, h, ldh, nullptr, nullptr, 0, M, F, K, act, nullptr, 0, stream);
}

extern "C" int64_t fp_gated_ff_backward_workspace_bytes(int M, int F, int K) {
    if (M <= 0 || F <= 0 || K <= 0 || M > LIMIT || F > LIMIT || K > LIMIT) return 0;
    return grad_space(M, F, K).end;
}

extern "C" int fp_gated_ff_backward_bf16(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* w_gate, int64_t ldwg,
                                         const void* w_up, int64_t ldwu, const void* gate, int64_t ldg, const void* up, int64_t ldu,
                                         void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, int M, int F, int K, int act,
                                         void* workspace, int64_t workspace_bytes, void* stream) {
    return ff_grad_launch<bf16>(dh, ldh, x, ldx, w_gate, ldwg, w_up, ldwu, gate, ldg, up, ldu, dx, dw_gate, dw_up, db_gate, db_up, M, F, K,
                                act, workspace, workspace_bytes, stream);
}

extern "C" int fp_gated_ff_backward_f16(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* w_gate, int64_t ldwg,
                                        const void* w_up, int64_t ldwu, const void* gate, int64_t ldg, const void* up, int64_t ldu,
                                        void* dx, void* dw_gate, void* dw_up, void* db_gate, void* db_up, int M, int F, int K, int act,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
    return ff_grad_launch<_Float16>(dh, ldh, x, ldx, w_gate, ldwg, w_up, ldwu, gate, ldg, up, ldu, dx, dw_gate, dw_up, db_gate, db_up, M,
                                    F, K, act, workspace, workspace_bytes, stream);
}
