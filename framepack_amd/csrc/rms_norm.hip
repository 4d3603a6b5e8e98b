// K12: RMSNorm of a residual sum (the pre-norm of a language model's layer), with a 16-bit or an e4m3 output, and its
// gradient.  gfx950 / wave64; C-ABI entry points at the bottom, declarations in include/framepack_hip.h.
//
//   h = resid + x        r = 1 / sqrt(mean(h^2) + eps)        y = h r w
//   dx = dresid = dh + r (dn - n mean(dn n)),  n = h r,  dn = dy w;        dw = sum over rows of dy n
#include "fp_common.h"

extern "C" int64_t fp_rmsnorm_residual_backward_workspace_bytes(int rows, int cols);

namespace {

constexpr float FP8_MAX = 448.f;

// sum / max over the 256 lanes of a workgroup, the result in every lane (red: 4 floats of LDS, free on return)
__device__ __forceinline__ float block_sum(float v, float* red) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return v;
}
__device__ __forceinline__ float block_max(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    __syncthreads();
    return v;
}

// y / scale to e4m3: the quotient by one Newton step on y * (1 / scale), so that it rounds as a division does
__device__ __forceinline__ unsigned char to_e4m3(float y, float scale, float inv) {
    const float q = y * inv;
    const float v = __builtin_fmaf(__builtin_fmaf(-q, scale, y), inv, q);
    return (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(v, 0.f, 0, false) & 0xff);
}
// The row's scale.  A row of zeros gets 1; below the smallest normal number 1 / scale would overflow.
__device__ __forceinline__ float row_scale(float amax) { return amax > 0.f ? fmaxf(amax / FP8_MAX, 0x1p-126f) : 1.f; }

// One workgroup per row, three passes over it (the second and third from the caches).  The sum h is held in 32 bits for
// the norm and rounded once where it is stored.
// (y and h may lie on x and resid: those four are not __restrict__, and a lane reads an element before it writes it)
template <typename T, bool Q8>
__global__ __launch_bounds__(256) void rmsnorm_rows_kernel(const T* x, int64_t x_rs, const T* resid, int64_t r_rs,
                                                           const T* __restrict__ w, T* y, int64_t y_rs,
                                                           float* __restrict__ q_scale, T* h, int64_t h_rs, int cols, float eps) {
    __shared__ float red[4];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * x_rs;
    const T* rr = resid ? resid + row * r_rs : nullptr;
    auto at = [&](int c) { return (float)xr[c] + (rr ? (float)rr[c] : 0.f); };
    float ss = 0.f;
    for (int c = threadIdx.x; c < cols; c += 256) {
        const float v = at(c);
        ss += v * v;
    }
    const float r = 1.f / sqrtf(block_sum(ss, red) / (float)cols + eps);
    float scale = 1.f, inv = 1.f;
    if constexpr (Q8) {
        float m = 0.f;
        for (int c = threadIdx.x; c < cols; c += 256) m = fmaxf(m, fabsf(at(c) * r * (float)w[c]));
        scale = row_scale(block_max(m, red));
        inv = 1.f / scale;
        if (threadIdx.x == 0) q_scale[row] = scale;
    }
    for (int c = threadIdx.x; c < cols; c += 256) {
        const float v = at(c), o = v * r * (float)w[c];
        if constexpr (Q8) reinterpret_cast<unsigned char*>(y)[row * y_rs + c] = to_e4m3(o, scale, inv);
        else y[row * y_rs + c] = (T)o;
        if (rr) h[row * h_rs + c] = (T)v;
    }
}

// dx of one row per workgroup (dx may lie on dh); the row's r is left in `rstd` for the weight's gradient
template <typename T>
__global__ __launch_bounds__(256) void rmsnorm_grad_rows_kernel(const T* __restrict__ dy, int64_t dy_rs, const T* __restrict__ h,
                                                                int64_t h_rs, const T* dh, int64_t dh_rs,
                                                                const T* __restrict__ w, T* dx, int64_t dx_rs,
                                                                float* __restrict__ rstd, int cols, float eps) {
    __shared__ float red[4];
    const int64_t row = blockIdx.x;
    float ss = 0.f, dot = 0.f;
    for (int c = threadIdx.x; c < cols; c += 256) {
        const float v = (float)h[row * h_rs + c];
        ss += v * v;
        dot += (float)dy[row * dy_rs + c] * (float)w[c] * v;
    }
    const float r = 1.f / sqrtf(block_sum(ss, red) / (float)cols + eps);
    const float k = block_sum(dot, red) * r * r / (float)cols;      // mean(dn n) r
    for (int c = threadIdx.x; c < cols; c += 256) {
        const float up = dh ? (float)dh[row * dh_rs + c] : 0.f;
        dx[row * dx_rs + c] = (T)(up + r * ((float)dy[row * dy_rs + c] * (float)w[c] - (float)h[row * h_rs + c] * k));
    }
    if (threadIdx.x == 0) rstd[row] = r;
}

// partial[g][c] = sum of dy n over the rows of group g (a contiguous run); grid (ceil(cols / 256), groups)
template <typename T>
__global__ __launch_bounds__(256) void rmsnorm_dweight_partial_kernel(const T* __restrict__ dy, int64_t dy_rs,
                                                                      const T* __restrict__ h, int64_t h_rs,
                                                                      const float* __restrict__ rstd, float* __restrict__ part,
                                                                      int rows, int cols) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    const int per = (rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = (int64_t)blockIdx.y * per, r1 = min(r0 + per, (int64_t)rows);
    float s = 0.f;
    for (int64_t r = r0; r < r1; ++r) s += (float)dy[r * dy_rs + c] * ((float)h[r * h_rs + c] * rstd[r]);
    part[(int64_t)blockIdx.y * cols + c] = s;
}
template <typename T>
__global__ __launch_bounds__(256) void rmsnorm_dweight_reduce_kernel(const float* __restrict__ part, int groups, int cols,
                                                                     T* __restrict__ dw) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    float s = 0.f;
    for (int g = 0; g < groups; ++g) s += part[(int64_t)g * cols + c];
    dw[c] = (T)s;
}

bool aligned2(const void* p) { return ((uintptr_t)p & 1) == 0; }

constexpr int GROUPS = 256;       // of rows, in the weight's gradient
int grad_groups(int rows) { return rows < GROUPS ? rows : GROUPS; }

template <typename T, bool Q8>
int norm_launch(const void* x, int64_t x_rs, const void* resid, int64_t r_rs, const void* w, void* y, int64_t y_rs,
                void* q_scale, void* h, int64_t h_rs, int rows, int cols, float eps, void* stream) {
    FP_REQUIRE(x && w && y && rows >= 0 && cols > 0 && x_rs >= 0 && y_rs >= cols);
    FP_REQUIRE(!resid == !h && (!resid || (r_rs >= 0 && h_rs >= cols)) && eps >= 0.f);
    FP_REQUIRE(aligned2(x) && aligned2(resid) && aligned2(w) && (Q8 || aligned2(y)) && aligned2(h));
    FP_REQUIRE(!Q8 || (q_scale && ((uintptr_t)q_scale & 3) == 0));
    if (rows == 0) return 0;
    rmsnorm_rows_kernel<T, Q8><<<dim3((unsigned)rows), dim3(256), 0, (hipStream_t)stream>>>(
        (const T*)x, x_rs, (const T*)resid, r_rs, (const T*)w, (T*)y, y_rs, (float*)q_scale, (T*)h, h_rs, cols, eps);
    FP_CHECK_LAUNCH();
    return 0;
}

template <typename T>
int grad_launch(const void* dy, int64_t dy_rs, const void* h, int64_t h_rs, const void* dh, int64_t dh_rs, const void* w,
                void* dx, int64_t dx_rs, void* dw, int rows, int cols, float eps, void* ws, int64_t ws_bytes, void* stream) {
    FP_REQUIRE(dy && h && w && dx && dw && rows > 0 && cols > 0 && dy_rs >= 0 && h_rs >= 0 && dx_rs >= cols && eps >= 0.f);
    FP_REQUIRE(!dh || dh_rs >= 0);
    FP_REQUIRE(aligned2(dy) && aligned2(h) && aligned2(dh) && aligned2(w) && aligned2(dx) && aligned2(dw));
    FP_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= fp_rmsnorm_residual_backward_workspace_bytes(rows, cols));
    hipStream_t st = (hipStream_t)stream;
    float* rstd = (float*)ws;
    float* part = rstd + ((rows + 3) & ~3);
    const int groups = grad_groups(rows);
    rmsnorm_grad_rows_kernel<T><<<dim3((unsigned)rows), dim3(256), 0, st>>>((const T*)dy, dy_rs, (const T*)h, h_rs, (const T*)dh,
                                                                           dh_rs, (const T*)w, (T*)dx, dx_rs, rstd, cols, eps);
    FP_CHECK_LAUNCH();
    const unsigned cb = (unsigned)((cols + 255) / 256);
    rmsnorm_dweight_partial_kernel<T><<<dim3(cb, (unsigned)groups), dim3(256), 0, st>>>((const T*)dy, dy_rs, (const T*)h, h_rs, rstd,
                                                                                       part, rows, cols);
    FP_CHECK_LAUNCH();
    rmsnorm_dweight_reduce_kernel<T><<<dim3(cb), dim3(256), 0, st>>>(part, groups, cols, (T*)dw);
    FP_CHECK_LAUNCH();
    return 0;
}

}  // namespace

extern "C" int fp_rmsnorm_residual_bf16(const void* x, int64_t x_row_stride, const void* resid, int64_t resid_row_stride,
                                        const void* weight, void* y, int64_t y_row_stride, void* h, int64_t h_row_stride,
                                        int rows, int cols, float eps, void* stream) {
    return norm_launch<bf16, false>(x, x_row_stride, resid, resid_row_stride, weight, y, y_row_stride, nullptr, h, h_row_stride,
                                    rows, cols, eps, stream);
}

extern "C" int fp_rmsnorm_residual_f16(const void* x, int64_t x_row_stride, const void* resid, int64_t resid_row_stride,
                                       const void* weight, void* y, int64_t y_row_stride, void* h, int64_t h_row_stride,
                                       int rows, int cols, float eps, void* stream) {
    return norm_launch<_Float16, false>(x, x_row_stride, resid, resid_row_stride, weight, y, y_row_stride, nullptr, h,
                                        h_row_stride, rows, cols, eps, stream);
}

extern "C" int fp_rmsnorm_residual_fp8(const void* x, int64_t x_row_stride, const void* resid, int64_t resid_row_stride,
                                       const void* weight, void* q, int64_t ldq, void* q_scale, void* h, int64_t h_row_stride,
                                       int rows, int cols, float eps, void* stream) {
    return norm_launch<bf16, true>(x, x_row_stride, resid, resid_row_stride, weight, q, ldq, q_scale, h, h_row_stride, rows, cols,
                                   eps, stream);
}

extern "C" int64_t fp_rmsnorm_residual_backward_workspace_bytes(int rows, int cols) {
    if (rows <= 0 || cols <= 0) return 0;
    return ((int64_t)((rows + 3) & ~3) + (int64_t)grad_groups(rows) * cols) * 4;
}

extern "C" int fp_rmsnorm_residual_backward_bf16(const void* dy, int64_t dy_row_stride, const void* h, int64_t h_row_stride,
                                                 const void* dh, int64_t dh_row_stride, const void* weight, void* dx,
                                                 int64_t dx_row_stride, void* dweight, int rows, int cols, float eps,
                                                 void* workspace, int64_t workspace_bytes, void* stream) {
    return grad_launch<bf16>(dy, dy_row_stride, h, h_row_stride, dh, dh_row_stride, weight, dx, dx_row_stride, dweight, rows, cols,
                             eps, workspace, workspace_bytes, stream);
}

extern "C" int fp_rmsnorm_residual_backward_f16(const void* dy, int64_t dy_row_stride, const void* h, int64_t h_row_stride,
                                                const void* dh, int64_t dh_row_stride, const void* weight, void* dx,
                                                int64_t dx_row_stride, void* dweight, int rows, int cols, float eps,
                                                void* workspace, int64_t workspace_bytes, void* stream) {
    return grad_launch<_Float16>(dy, dy_row_stride, h, h_row_stride, dh, dh_row_stride, weight, dx, dx_row_stride, dweight, rows,
                                 cols, eps, workspace, workspace_bytes, stream);
}
