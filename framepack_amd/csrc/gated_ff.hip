// K13: the gated feed-forward block's first half, h = act(x . Wg^T + bg) * (x . Wu^T + bu), act = SiLU or tanh-GELU, in
// bf16 / f16 and on e4m3 operands, and its gradient.  gfx950 / wave64; C-ABI entry points at the bottom, declarations in
// include/framepack_hip.h.
//
//   dg = dh u act'(g)   du = dh act(g)   dx = dg . Wg + du . Wu   dWg = dg^T . x   dWu = du^T . x   db = column sums
#include "gemm_pipeline.h"

extern "C" int64_t fp_gated_ff_backward_workspace_bytes(int M, int F, int K);

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

// ---- any size, any strides: 64 x 64 output tiles, one element per load -------------------------------------------
// GLU:  c = act(a . b0^T + bias0) * (a . b1^T + bias1)        (p0, p1: the two projections, or null)
// else: c = a . b0^T (+ a1 . b1^T)
// a[m][k] = a[m * a_rs + k * a_ks] and so on: every orientation of the gradient's products is one call.
// e4m3 operands are widened to bf16, which holds them exactly; a_scale [M], b_scale0/1 [N] (or null).
template <typename TI> struct widen {
    typedef TI type;
    typedef TI vec8 __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ TI of(TI v) { return v; }
};
template <> struct widen<fp8e4> {
    typedef bf16 type;
    typedef bf16x8 vec8;
    static __device__ __forceinline__ bf16 of(fp8e4 v) { return (bf16)__builtin_amdgcn_cvt_f32_fp8((int)v.bits, 0); }
};
struct Operand {
    const void* p;
    int64_t rs, ks;
};
template <typename TI, typename TO, bool GLU>
__global__ __launch_bounds__(256) void any_gemm_kernel(Operand a, Operand b0, Operand a1, Operand b1, const float* __restrict__ a_scale,
                                                       const float* __restrict__ s0, const float* __restrict__ s1,
                                                       const TO* __restrict__ bias0, const TO* __restrict__ bias1,
                                                       TO* __restrict__ c, int64_t ldc, TO* __restrict__ p0, TO* __restrict__ p1,
                                                       int64_t ldp, int M, int N, int K, int act) {
    typedef typename widen<TI>::type TM;
    typedef typename widen<TI>::vec8 TM8;
    __shared__ __attribute__((aligned(16))) TM sa[64][40], sb[2][64][40];      // rows of 32, padded to 80 B
    const int64_t m0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
    f32x4 acc[2][2][2] = {};
    auto stage = [&](TM (*dst)[40], const Operand& o, int64_t r0, int rows, int k0) {
        const TI* p = reinterpret_cast<const TI*>(o.p);
        // the axis with unit stride goes along the lanes
        const bool kfast = o.ks == 1;
        for (int i = tid; i < 64 * 32; i += 256) {
            const int r = kfast ? i >> 5 : i & 63, k = kfast ? i & 31 : i >> 6;
            TM v = (TM)0.f;
            if (r0 + r < rows && k0 + k < K) v = widen<TI>::of(p[(r0 + r) * o.rs + (int64_t)(k0 + k) * o.ks]);
            dst[r][k] = v;
        }
    };
    const int segs = !GLU && a1.p ? 2 : 1;
    for (int seg = 0; seg < segs; ++seg)
        for (int k0 = 0; k0 < K; k0 += 32) {
            stage(sa, seg ? a1 : a, m0, M, k0);
            stage(sb[0], seg ? b1 : b0, n0, N, k0);
            if constexpr (GLU) stage(sb[1], b1, n0, N, k0);
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const TM8 av = *reinterpret_cast<const TM8*>(&sa[wm + i * 16 + (lane & 15)][(lane >> 4) * 8]);
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int g = 0; g < (GLU ? 2 : 1); ++g)
                        acc[g][i][j] = mfma16(*reinterpret_cast<const TM8*>(&sb[g][wn + j * 16 + (lane & 15)][(lane >> 4) * 8]), av,
                                              acc[g][i][j]);
            }
            __syncthreads();
        }
    // (operands swapped: the lane's low bits are the row, its four registers four columns)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t m = m0 + wm + i * 16 + (lane & 15), n = n0 + wn + j * 16 + (lane >> 4) * 4 + e;
                if (m >= M || n >= N) continue;
                float v = acc[0][i][j][e];
                if constexpr (GLU) {
                    const float as = a_scale ? a_scale[m] : 1.f;
                    const float g = v * (s0 ? as * s0[n] : 1.f) + (bias0 ? (float)bias0[n] : 0.f);
                    const float u = acc[1][i][j][e] * (s1 ? as * s1[n] : 1.f) + (bias1 ? (float)bias1[n] : 0.f);
                    if (p0) p0[m * ldp + n] = (TO)g;
                    if (p1) p1[m * ldp + n] = (TO)u;
                    v = act_of(g, act) * u;
                }
                c[m * ldc + n] = (TO)v;
            }
}

// dg, du [M, F] (row stride F) from dh and the two projections; grid (ceil(F / 256), rows)
template <typename T>
__global__ __launch_bounds__(256) void glu_grad_kernel(const T* __restrict__ dh, int64_t ldh, const T* __restrict__ gate, int64_t ldg,
                                                       const T* __restrict__ up, int64_t ldu, T* __restrict__ dg,
                                                       T* __restrict__ du, int M, int F, int act) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= F) return;
    for (int64_t m = blockIdx.y; m < M; m += gridDim.y) {
        float a, da;
        act_grad((float)gate[m * ldg + c], act, a, da);
        const float d = (float)dh[m * ldh + c];
        dg[m * F + c] = (T)(d * (float)up[m * ldu + c] * da);
        du[m * F + c] = (T)(d * a);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void bias_grad_kernel(const T* __restrict__ dg, const T* __restrict__ du, T* __restrict__ dbg,
                                                        T* __restrict__ dbu, int M, int F) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= F) return;
    const T* p = blockIdx.y ? du : dg;
    float s = 0.f;
    for (int64_t m = 0; m < M; ++m) s += (float)p[m * F + c];
    (blockIdx.y ? dbu : dbg)[c] = (T)s;
}

bool aligned2(const void* p) { return ((uintptr_t)p & 1) == 0; }
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename TI, typename TO, bool GLU>
int any_gemm(Operand a, Operand b0, Operand a1, Operand b1, const float* as, const float* s0, const float* s1, const void* bias0,
             const void* bias1, void* c, int64_t ldc, void* p0, void* p1, int64_t ldp, int M, int N, int K, int act, hipStream_t st) {
    const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((M + 63) / 64));
    FP_REQUIRE(grid.y < 65536);
    any_gemm_kernel<TI, TO, GLU><<<grid, dim3(256), 0, st>>>(a, b0, a1, b1, as, s0, s1, (const TO*)bias0, (const TO*)bias1, (TO*)c, ldc,
                                                             (TO*)p0, (TO*)p1, ldp, M, N, K, act);
    FP_CHECK_LAUNCH();
    return 0;
}

template <typename TI, typename TO>
int ff_launch(const void* x, int64_t ldx, const float* xs, const void* wg, int64_t ldwg, const float* gs, const void* wu, int64_t ldwu,
              const float* us, const void* bg, const void* bu, void* h, int64_t ldh, void* gate, void* up, int64_t ldp, int M, int F,
              int K, int act, void* stream) {
    FP_REQUIRE(x && wg && wu && h && M >= 0 && F > 0 && K > 0 && (act == 0 || act == 1) && !bg == !bu && !gate == !up);
    FP_REQUIRE(ldx >= 0 && ldwg >= K && ldwu >= K && ldh >= F && (!gate || ldp >= F));
    FP_REQUIRE(sizeof(TI) == 1 || (aligned2(x) && aligned2(wg) && aligned2(wu) && aligned2(h) && aligned2(bg) && aligned2(bu) &&
                                   aligned2(gate) && aligned2(up)));
    if (M == 0) return 0;
    return any_gemm<TI, TO, true>({x, ldx, 1}, {wg, ldwg, 1}, {nullptr, 0, 0}, {wu, ldwu, 1}, xs, gs, us, bg, bu, h, ldh, gate, up, ldp,
                                  M, F, K, act, (hipStream_t)stream);
}

template <typename T>
int ff_grad_launch(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* wg, int64_t ldwg, const void* wu, int64_t ldwu,
                   const void* gate, int64_t ldg, const void* up, int64_t ldu, void* dx, int64_t lddx, void* dwg, void* dwu,
                   int64_t lddw, void* dbg, void* dbu, int M, int F, int K, int act, void* ws, int64_t ws_bytes, void* stream) {
    FP_REQUIRE(dh && x && wg && wu && gate && up && dx && dwg && dwu && !dbg == !dbu && (act == 0 || act == 1));
    FP_REQUIRE(aligned2(dh) && aligned2(x) && aligned2(wg) && aligned2(wu) && aligned2(gate) && aligned2(up) && aligned2(dx) &&
               aligned2(dwg) && aligned2(dwu) && aligned2(dbg) && aligned2(dbu));
    FP_REQUIRE(M > 0 && F > 0 && K > 0 && ldh >= 0 && ldx >= 0 && ldg >= 0 && ldu >= 0 && ldwg >= K && ldwu >= K && lddx >= K && lddw >= K);
    FP_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= fp_gated_ff_backward_workspace_bytes(M, F, K));
    hipStream_t st = (hipStream_t)stream;
    T* dg = (T*)ws;
    T* du = dg + (int64_t)M * F;
    glu_grad_kernel<T><<<dim3((unsigned)((F + 255) / 256), (unsigned)(M < 16384 ? M : 16384)), dim3(256), 0, st>>>(
        (const T*)dh, ldh, (const T*)gate, ldg, (const T*)up, ldu, dg, du, M, F, act);
    FP_CHECK_LAUNCH();
    const Operand none{nullptr, 0, 0};
    if (int rc = any_gemm<T, T, false>({dg, F, 1}, {wg, 1, ldwg}, {du, F, 1}, {wu, 1, ldwu}, nullptr, nullptr, nullptr, nullptr, nullptr,
                                       dx, lddx, nullptr, nullptr, 0, M, K, F, 0, st))
        return rc;
    for (int i = 0; i < 2; ++i)
        if (int rc = any_gemm<T, T, false>({i ? du : dg, 1, F}, {x, 1, ldx}, none, none, nullptr, nullptr, nullptr, nullptr, nullptr,
                                           i ? dwu : dwg, lddw, nullptr, nullptr, 0, F, K, M, 0, st))
            return rc;
    if (dbg) {
        bias_grad_kernel<T><<<dim3((unsigned)((F + 255) / 256), 2), dim3(256), 0, st>>>(dg, du, (T*)dbg, (T*)dbu, M, F);
        FP_CHECK_LAUNCH();
    }
    return 0;
}

}  // namespace

extern "C" int fp_gated_ff_bf16(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                                const void* b_gate, const void* b_up, void* h, int64_t ldh, void* gate, void* up, int64_t ldp, int M,
                                int F, int K, int act, void* stream) {
    return ff_launch<bf16, bf16>(x, ldx, nullptr, w_gate, ldwg, nullptr, w_up, ldwu, nullptr, b_gate, b_up, h, ldh, gate, up, ldp, M, F,
                                 K, act, stream);
}

extern "C" int fp_gated_ff_f16(const void* x, int64_t ldx, const void* w_gate, int64_t ldwg, const void* w_up, int64_t ldwu,
                               const void* b_gate, const void* b_up, void* h, int64_t ldh, void* gate, void* up, int64_t ldp, int M,
                               int F, int K, int act, void* stream) {
    return ff_launch<_Float16, _Float16>(x, ldx, nullptr, w_gate, ldwg, nullptr, w_up, ldwu, nullptr, b_gate, b_up, h, ldh, gate, up,
                                         ldp, M, F, K, act, stream);
}

extern "C" int fp_gated_ff_fp8(const void* x, int64_t ldx, const void* x_scale, const void* w_gate, int64_t ldwg, const void* wg_scale,
                               const void* w_up, int64_t ldwu, const void* wu_scale, const void* b_gate, const void* b_up, void* h,
                               int64_t ldh, int M, int F, int K, int act, void* stream) {
    FP_REQUIRE(x_scale && wg_scale && wu_scale && K > 0 && K % 128 == 0 && F > 0 && F % 8 == 0);
    FP_REQUIRE(aligned16(x) && aligned16(w_gate) && aligned16(w_up) && aligned16(h) && ldx % 16 == 0 && ldwg % 16 == 0 &&
               ldwu % 16 == 0 && ldh % 8 == 0 && ldx >= 0);
    FP_REQUIRE(((uintptr_t)x_scale & 3) == 0 && aligned16(wg_scale) && aligned16(wu_scale) && aligned16(b_gate) && aligned16(b_up));
    return ff_launch<fp8e4, bf16>(x, ldx, (const float*)x_scale, w_gate, ldwg, (const float*)wg_scale, w_up, ldwu,
                                  (const float*)wu_scale, b_gate, b_up, h, ldh, nullptr, nullptr, 0, M, F, K, act, stream);
}

extern "C" int64_t fp_gated_ff_backward_workspace_bytes(int M, int F, int K) {
    if (M <= 0 || F <= 0 || K <= 0) return 0;
    return ((int64_t)M * F * 4 + 15) & ~(int64_t)15;
}

extern "C" int fp_gated_ff_backward_bf16(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* w_gate, int64_t ldwg,
                                         const void* w_up, int64_t ldwu, const void* gate, int64_t ldg, const void* up, int64_t ldu,
                                         void* dx, int64_t lddx, void* dw_gate, void* dw_up, int64_t lddw, void* db_gate, void* db_up,
                                         int M, int F, int K, int act, void* workspace, int64_t workspace_bytes, void* stream) {
    return ff_grad_launch<bf16>(dh, ldh, x, ldx, w_gate, ldwg, w_up, ldwu, gate, ldg, up, ldu, dx, lddx, dw_gate, dw_up, lddw, db_gate,
                                db_up, M, F, K, act, workspace, workspace_bytes, stream);
}

extern "C" int fp_gated_ff_backward_f16(const void* dh, int64_t ldh, const void* x, int64_t ldx, const void* w_gate, int64_t ldwg,
                                        const void* w_up, int64_t ldwu, const void* gate, int64_t ldg, const void* up, int64_t ldu,
                                        void* dx, int64_t lddx, void* dw_gate, void* dw_up, int64_t lddw, void* db_gate, void* db_up,
                                        int M, int F, int K, int act, void* workspace, int64_t workspace_bytes, void* stream) {
    return ff_grad_launch<_Float16>(dh, ldh, x, ldx, w_gate, ldwg, w_up, ldwu, gate, ldg, up, ldu, dx, lddx, dw_gate, dw_up, lddw,
                                    db_gate, db_up, M, F, K, act, workspace, workspace_bytes, stream);
}
