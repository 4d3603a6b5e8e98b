// K12: RMSNorm of a residual sum (the pre-norm of a language model's layer), with a 16-bit or an e4m3 output, and its
// gradient.  gfx950 / wave64; C-ABI entry points at the bottom, declarations in include/framepack_hip.h.
//
//   h = resid + x        r = 1 / sqrt(mean(h^2) + eps)        y = h r w
//   dx = dresid = dh + r (dn - n mean(dn n)),  n = h r,  dn = dy w;        dw = sum over rows of dy n
//
// All of it is bound by HBM: the row stays in registers between its sums and its last use, so every matrix is read or written
// once.  Measured in bf16 (a large copy runs at 4.9 TB/s on the same card), us and TB/s of those bytes:
//   rows x cols      y and h        e4m3 and h     gradient
//   19385 x 4096     113  5.6       100  5.6       127  5.0
//   19385 x 4095     135  4.7       119  4.7       152  4.2     (rows that begin at any 2 bytes: lines shared between lanes' loads)
//   8191 x 4096      44   6.1       41   5.7       55   4.9
//   512 x 4096       5.2            5.6            11           (two launches)
//   1 x 4096         2.6            3.2            6            (latency; the call from Python takes 9 - 14 us on the host)
#include "row_access.h"

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

// e4m3: q = 448 t / top with t = h w, top = max|t|, and the row's scale r top / 448.  The norm's factor r is one of the scale
// alone (in q it would cancel, but for its roundings), unless it is 0, infinite or NaN: then t has it and the scale has not.
// A row of zeros has top = 448, scale 1; between the bounds neither top / 448 nor its reciprocal is infinite.
__device__ __forceinline__ float in_q(float r) { return r > 0.f && r < __builtin_inff() ? 1.f : r; }
__device__ __forceinline__ float row_top(float amax) {
    return amax > 0.f ? fminf(fmaxf(amax, FP8_MAX * 0x1p-126f), 0x1.fffffep127f) : FP8_MAX;
}
__device__ __forceinline__ float row_scale(float amax, float top, float r) {
    return top / FP8_MAX * (amax > 0.f && in_q(r) == 1.f ? r : 1.f);
}
// 448 t / top = 7 t / m with m = top / 64 (exact), inv = 1 / m: the remainder 7 t - q m, taken as (8 t - q m) - t, corrects the
// first quotient, so that one rounding is left in front of that to 8 bits.
__device__ __forceinline__ float quotient(float t, float m, float inv) {
    const float q = t * (7.f * inv);
    return __builtin_fmaf(__builtin_fmaf(-q, m, 8.f * t) - t, inv, q);
}

typedef unsigned int any_u32x2 __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned int any_u32 __attribute__((aligned(1)));
typedef unsigned short any_u16 __attribute__((aligned(1)));

// sum over the TPR lanes of a row (a wave, or the workgroup: red holds a float per wave)
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
    v = wave_sum(v);
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) v += red[i];
    }
    return v;
}
template <int TPR>
__device__ __forceinline__ float row_max(float v, float* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    if constexpr (TPR > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = red[0];
#pragma unroll
        for (int i = 1; i < TPR / 64; ++i) v = fmaxf(v, red[i]);
    }
    return v;
}

// TPR lanes per row (64: four rows a workgroup), the row in registers (NCH chunks of 8 a lane) between the sum of squares
// and the write: one read of x and resid, one write of y and h.  The sum h is held in 32 bits for the norm and rounded
// once where it is stored.  (y and h may lie on x and resid: those four are not __restrict__.  A lane has read its own elements
// before it writes them.  The lane with the row's partial last chunk also reads up to 7 elements in front of its own, as load8
// does; their lane, of another wave perhaps, may have overwritten them by then, and `fit` drops them before anything uses them.)
template <typename T, bool Q8, int TPR, int NCH>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rmsnorm_kernel(const T* x, int64_t x_rs, const T* resid, int64_t r_rs,
                                                                        const T* __restrict__ w, T* y, int64_t y_rs,
                                                                        float* __restrict__ q_scale, T* h, int64_t h_rs, int rows,
                                                                        int cols, float eps) {
    typedef typename vec8<T>::type V;
    __shared__ float red[2][TPR / 64];
    const int lane = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (TPR < 256 ? 256 / TPR : 1) + threadIdx.x / TPR;
    if (TPR == 64 && row >= rows) return;                  // (whole waves; TPR > 64: the grid is the rows)
    const T* xr = x + row * x_rs;
    V xv[NCH], rv[NCH], wv[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) xv[i] = load8(xr, (i * TPR + lane) * 8, cols);
    if (resid) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) rv[i] = load8(resid + row * r_rs, (i * TPR + lane) * 8, cols);
    }
#pragma unroll
    for (int i = 0; i < NCH; ++i) wv[i] = load8(w, (i * TPR + lane) * 8, cols);
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        if ((i + 1) * TPR * 8 <= cols) continue;            // (uniform: a whole chunk in every lane)
        fit(xv[i], (i * TPR + lane) * 8, cols);
        if (resid) fit(rv[i], (i * TPR + lane) * 8, cols);
        fit(wv[i], (i * TPR + lane) * 8, cols);
    }
    float v[NCH][8], ss = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[i][j] = (float)xv[i][j];
            if (resid) v[i][j] += (float)rv[i][j];
            ss += v[i][j] * v[i][j];
        }
    const float r = 1.f / sqrtf(row_sum<TPR>(ss, red[0]) / (float)cols + eps);
    if (resid) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            V o;
#pragma unroll
            for (int j = 0; j < 8; ++j) o[j] = (T)v[i][j];
            store8(h + row * h_rs, (i * TPR + lane) * 8, cols, o);
        }
    }
    float m = 0.f;
    const float f = Q8 ? in_q(r) : r;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        V o;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[i][j] = v[i][j] * f * (float)wv[i][j];
            if constexpr (Q8) m = fmaxf(m, fabsf(v[i][j]));
            else o[j] = (T)v[i][j];
        }
        if constexpr (!Q8) store8(y + row * y_rs, (i * TPR + lane) * 8, cols, o);
    }
    if constexpr (Q8) {
        const float amax = row_max<TPR>(m, red[1]), top = row_top(amax), m64 = top * 0x1p-6f, inv = 1.f / m64;
        if (lane == 0) q_scale[row] = row_scale(amax, top, r);
        unsigned char* qr = reinterpret_cast<unsigned char*>(y) + row * y_rs;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = (i * TPR + lane) * 8;
            u32x2 o;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                int p = 0;
                p = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(v[i][4 * k], m64, inv), quotient(v[i][4 * k + 1], m64, inv), p, false);
                p = __builtin_amdgcn_cvt_pk_fp8_f32(quotient(v[i][4 * k + 2], m64, inv), quotient(v[i][4 * k + 3], m64, inv), p, true);
                o[k] = (unsigned)p;
            }
            if (c + 8 <= cols) {
                *reinterpret_cast<any_u32x2*>(qr + c) = o;
            } else if (c < cols) {
                const int n = cols & 7;
                const unsigned t = n & 4 ? o[1] : o[0];     // behind a whole first half, or the half itself
                if (n & 4) *reinterpret_cast<any_u32*>(qr + c) = o[0];
                if (n & 2) *reinterpret_cast<any_u16*>(qr + c + (n & 4)) = (unsigned short)t;
                if (n & 1) qr[c + n - 1] = (unsigned char)(n & 2 ? t >> 16 : t);
            }
        }
    }
}

// Rows of more than 65536 columns: one workgroup per row, two or three passes over it (all but the first from the caches).
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
    const float f = Q8 ? in_q(r) : r;
    float m64 = 1.f, inv = 1.f;
    if constexpr (Q8) {
        float m = 0.f;
        for (int c = threadIdx.x; c < cols; c += 256) m = fmaxf(m, fabsf(at(c) * f * (float)w[c]));
        const float amax = block_max(m, red);
        const float top = row_top(amax);
        m64 = top * 0x1p-6f;
        inv = 1.f / m64;
        if (threadIdx.x == 0) q_scale[row] = row_scale(amax, top, r);
    }
    for (int c = threadIdx.x; c < cols; c += 256) {
        const float v = at(c), o = v * f * (float)w[c];
        if constexpr (Q8) reinterpret_cast<unsigned char*>(y)[row * y_rs + c] = (unsigned char)(__builtin_amdgcn_cvt_pk_fp8_f32(quotient(o, m64, inv), 0.f, 0, false) & 0xff);
        else y[row * y_rs + c] = (T)o;
        if (rr) h[row * h_rs + c] = (T)v;
    }
}

// The gradient.  TPR lanes per row as above; a workgroup takes rows blockIdx.x, + gridDim.x, ..., keeps the weight's gradient
// of its columns in registers over all of them and leaves one partial row of it: one read of dy, h and dh, one write of dx.
// DW = false (longer rows, whose share of dweight does not fit the registers as well): the row's r is left in part[row].
// AHEAD: the next row is loaded before the current one's sums, so that the loads of two rows are in flight at every barrier
// (where the registers hold them).  dx may lie on dh: what holds for rmsnorm_kernel's partial last chunk holds for dh's here.
template <typename T, int TPR, int NCH, bool AHEAD, bool DW>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rmsnorm_grad_kernel(const T* __restrict__ dy, int64_t dy_rs, const T* __restrict__ h,
                                                                             int64_t h_rs, const T* dh, int64_t dh_rs,
                                                                             const T* __restrict__ w, T* dx, int64_t dx_rs,
                                                                             float* __restrict__ part, int rows, int cols, float eps) {
    typedef typename vec8<T>::type V;
    constexpr int RPB = TPR < 256 ? 256 / TPR : 1;         // rows a workgroup has in hand
    __shared__ float red[2][2][TPR / 64];                  // (alternating: one barrier a row)
    const int lane = threadIdx.x % TPR;
    const int sub = threadIdx.x / TPR;
    const int64_t step = (int64_t)gridDim.x * RPB;
    int64_t row = (int64_t)blockIdx.x * RPB + sub;
    V yv[NCH], hv[NCH], uv[NCH], wv[NCH];
    float dw[DW ? NCH : 1][8] = {};
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = (i * TPR + lane) * 8;
            yv[i] = load8(dy + r * dy_rs, c, cols);
            hv[i] = load8(h + r * h_rs, c, cols);
            if (dh) uv[i] = load8(dh + r * dh_rs, c, cols);
        }
    };
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
        wv[i] = load8(w, (i * TPR + lane) * 8, cols);
        fit(wv[i], (i * TPR + lane) * 8, cols);
    }
    if (AHEAD && row < rows) fetch(row);
    for (int k = 0; row < rows; row += step, k ^= 1) {     // (TPR > 64: the same row in all lanes of the workgroup)
        if (!AHEAD) fetch(row);
        V yc[NCH], hc[NCH], uc[NCH];
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            yc[i] = yv[i];
            hc[i] = hv[i];
            if (dh) uc[i] = uv[i];
        }
        if (AHEAD && row + step < rows) fetch(row + step);
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            if ((i + 1) * TPR * 8 > cols) {                 // (uniform)
                fit(yc[i], (i * TPR + lane) * 8, cols);
                fit(hc[i], (i * TPR + lane) * 8, cols);
                if (dh) fit(uc[i], (i * TPR + lane) * 8, cols);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ss += (float)hc[i][j] * (float)hc[i][j];
                dot += (float)yc[i][j] * (float)wv[i][j] * (float)hc[i][j];
            }
        }
        if constexpr (TPR > 64) {
            ss = wave_sum(ss);
            dot = wave_sum(dot);
            if ((threadIdx.x & 63) == 0) {
                red[k][0][threadIdx.x >> 6] = ss;
                red[k][1][threadIdx.x >> 6] = dot;
            }
            __syncthreads();
            ss = red[k][0][0];
            dot = red[k][1][0];
#pragma unroll
            for (int i = 1; i < TPR / 64; ++i) {
                ss += red[k][0][i];
                dot += red[k][1][i];
            }
        } else {
            ss = wave_sum(ss);
            dot = wave_sum(dot);
        }
        const float r = 1.f / sqrtf(ss / (float)cols + eps);
        const float kk = dot * r * r / (float)cols;        // mean(dn n) r
        if (!DW && lane == 0) part[row] = r;
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int c = (i * TPR + lane) * 8;
            V o;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float g = (float)yc[i][j], v = (float)hc[i][j];
                if constexpr (DW) dw[i][j] += g * (v * r);
                o[j] = (T)((dh ? (float)uc[i][j] : 0.f) + r * (g * (float)wv[i][j] - v * kk));
            }
            store8(dx + row * dx_rs, c, cols, o);
        }
    }
    if constexpr (DW) {
        const int ld = (cols + 7) & ~7;
        float* pr = part + (int64_t)blockIdx.x * ld;
        if constexpr (RPB > 1) {                            // the waves' shares are added up here, in their order
            __shared__ f32x4 all[RPB][NCH][2][TPR];
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                all[sub][i][0][lane] = f32x4{dw[i][0], dw[i][1], dw[i][2], dw[i][3]};
                all[sub][i][1][lane] = f32x4{dw[i][4], dw[i][5], dw[i][6], dw[i][7]};
            }
            __syncthreads();
            for (int i = sub; i < 2 * NCH; i += RPB) {
                const int c = ((i >> 1) * TPR + lane) * 8 + (i & 1) * 4;
                f32x4 s = all[0][i >> 1][i & 1][lane];
#pragma unroll
                for (int k = 1; k < RPB; ++k) s += all[k][i >> 1][i & 1][lane];
                if (c < ld) *reinterpret_cast<f32x4*>(pr + c) = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int c = (i * TPR + lane) * 8;
                if (c < cols) {
                    *reinterpret_cast<f32x4*>(pr + c) = f32x4{dw[i][0], dw[i][1], dw[i][2], dw[i][3]};
                    *reinterpret_cast<f32x4*>(pr + c + 4) = f32x4{dw[i][4], dw[i][5], dw[i][6], dw[i][7]};
                }
            }
        }
    }
}

// Rows of more than 32768 columns: dx of one row per workgroup in two passes (dx may lie on dh), the row's r left in `rstd`.
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
// part[g][c] = sum of dy n over the rows of group g (a contiguous run) from the rows' r; 8 columns a lane, grid
// (ceil(cols / 2048), groups)
template <typename T>
__global__ __launch_bounds__(256) void rmsnorm_dweight_rows_kernel(const T* __restrict__ dy, int64_t dy_rs, const T* __restrict__ h,
                                                                   int64_t h_rs, const float* __restrict__ rstd, float* __restrict__ part,
                                                                   int rows, int cols) {
    typedef typename vec8<T>::type V;
    const int c = (blockIdx.x * 256 + threadIdx.x) * 8;
    const int per = (rows + gridDim.y - 1) / gridDim.y;
    const int64_t r0 = (int64_t)blockIdx.y * per, r1 = min(r0 + per, (int64_t)rows);
    float s[8] = {};
#pragma unroll 2
    for (int64_t r = r0; r < r1; ++r) {
        V y = load8(dy + r * dy_rs, c, cols), v = load8(h + r * h_rs, c, cols);
        fit(y, c, cols);
        fit(v, c, cols);
        const float k = rstd[r];
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] += (float)y[j] * ((float)v[j] * k);
    }
    if (c < cols) {
        float* pr = part + (int64_t)blockIdx.y * ((cols + 7) & ~7) + c;
        *reinterpret_cast<f32x4*>(pr) = f32x4{s[0], s[1], s[2], s[3]};
        *reinterpret_cast<f32x4*>(pr + 4) = f32x4{s[4], s[5], s[6], s[7]};
    }
}
// dw = sum of the partial rows: a workgroup takes 32 columns, 32 groups of 8 lanes take every 32nd row each and are added
// up in a fixed order
template <typename T>
__global__ __launch_bounds__(256) void rmsnorm_dweight_kernel(const float* __restrict__ part, int parts, int cols, T* __restrict__ dw) {
    __shared__ f32x4 red[32][8];
    const int q = threadIdx.x & 7, g = threadIdx.x >> 3, c = blockIdx.x * 32 + q * 4, ld = (cols + 7) & ~7;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (c < ld) {
#pragma unroll 8
        for (int i = g; i < parts; i += 32) s += *reinterpret_cast<const f32x4*>(part + (int64_t)i * ld + c);
    }
    red[g][q] = s;
    __syncthreads();
    if (g == 0) {
#pragma unroll
        for (int i = 1; i < 32; ++i) s += red[i][q];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < cols) dw[c + j] = (T)s[j];
    }
}

bool aligned2(const void* p) { return ((uintptr_t)p & 1) == 0; }

constexpr int MOST_COLS = 1 << 28;   // 32-bit columns, and a launch's lanes below 2^32 (rmsnorm_dweight_kernel: 8 a column)
constexpr int MOST = 1 << 21;        // rows of a launch with a workgroup per row: its lanes have to stay below 2^32
constexpr int REG_COLS = 65536;      // the longest row that is held in registers (1024 lanes, 8 chunks each)
// Lanes per row: a wave where half of a workgroup's would have nothing to do and the rows alone fill the chip, else a workgroup
// (us, wave / workgroup: 20000 x 1024 29 / 34; 19385 x 4096 118 / 114; 1 x 4096 4.4 / 2.6), of 1024 lanes where 256 would hold
// more than 4 chunks each (1000 x 8192, 256 / 1024 lanes: 12.8 / 16.0).
constexpr int WAVE_COLS = 1024, GROUP_COLS = 8192;

// The gradient's partial rows of dweight.  As many workgroups as are resident at once (by the kernels' registers), but at
// least two rows each: a partial row is written and read again, as much as half a row of the matrices.
constexpr int GRAD_COLS = 16384;     // the longest row of the gradient's one-pass form (512 lanes, 4 chunks each)
int grad_parts(int rows, int cols) {
    if (cols > GRAD_COLS) return rows < 64 ? rows : 64;
    const int64_t rpb = cols <= 1024 ? 4 : 1, most = cols <= 2048 ? 1024 : cols <= 4096 ? 768 : cols <= 8192 ? 512 : 256;
    const int64_t groups = (rows + 2 * rpb - 1) / (2 * rpb);
    return (int)(groups < most ? groups : most);
}

template <typename T, bool Q8>
int norm_rows(const T* x, int64_t x_rs, const T* resid, int64_t r_rs, const T* w, T* y, int64_t y_rs, float* q_scale, T* h, int64_t h_rs,
              int rows, int cols, float eps, hipStream_t st) {
#define FP_NORM(TPR, NCH)                                                                                                         \
    rmsnorm_kernel<T, Q8, TPR, NCH><<<dim3((unsigned)(TPR < 256 ? (rows + 3) / 4 : rows)), dim3(TPR < 256 ? 256 : TPR), 0, st>>>( \
        x, x_rs, resid, r_rs, w, y, y_rs, q_scale, h, h_rs, rows, cols, eps)
    const int nch = (cols + 7) / 8;
    if (cols <= 512) {
        FP_NORM(64, 1);
    } else if (cols <= WAVE_COLS && rows >= 2048) {
        FP_NORM(64, 2);
    } else if (cols <= GROUP_COLS) {
        if (nch <= 256) FP_NORM(256, 1);
        else if (nch <= 512) FP_NORM(256, 2);
        else FP_NORM(256, 4);
    } else if (cols <= REG_COLS) {
        if (nch <= 2048) FP_NORM(1024, 2);
        else if (nch <= 4096) FP_NORM(1024, 4);
        else FP_NORM(1024, 8);
    } else {
        rmsnorm_rows_kernel<T, Q8><<<dim3((unsigned)rows), dim3(256), 0, st>>>(x, x_rs, resid, r_rs, w, y, y_rs, q_scale, h, h_rs, cols, eps);
    }
#undef FP_NORM
    FP_CHECK_LAUNCH();
    return 0;
}

template <typename T, bool Q8>
int norm_launch(const void* x, int64_t x_rs, const void* resid, int64_t r_rs, const void* w, void* y, int64_t y_rs,
                void* q_scale, void* h, int64_t h_rs, int rows, int cols, float eps, void* stream) {
    FP_REQUIRE(x && w && y && rows >= 0 && cols > 0 && cols <= MOST_COLS && x_rs >= 0 && y_rs >= cols);
    FP_REQUIRE(!resid == !h && (!resid || (r_rs >= 0 && h_rs >= cols)) && eps >= 0.f);
    FP_REQUIRE(aligned2(x) && aligned2(resid) && aligned2(w) && (Q8 || aligned2(y)) && aligned2(h));
    FP_REQUIRE(!Q8 || (q_scale && ((uintptr_t)q_scale & 3) == 0));
    if (rows == 0) return 0;
    hipStream_t st = (hipStream_t)stream;
    for (int64_t r = 0; r < rows; r += MOST) {
        // (y_rs counts bytes where y is e4m3)
        T* yr = Q8 ? (T*)((unsigned char*)y + r * y_rs) : (T*)y + r * y_rs;
        if (int rc = norm_rows<T, Q8>((const T*)x + r * x_rs, x_rs, resid ? (const T*)resid + r * r_rs : nullptr, r_rs, (const T*)w, yr, y_rs,
                                      Q8 ? (float*)q_scale + r : nullptr, h ? (T*)h + r * h_rs : nullptr, h_rs,
                                      rows - r < MOST ? (int)(rows - r) : MOST, cols, eps, st))
            return rc;
    }
    return 0;
}

template <typename T>
int grad_launch(const void* dy, int64_t dy_rs, const void* h, int64_t h_rs, const void* dh, int64_t dh_rs, const void* w,
                void* dx, int64_t dx_rs, void* dw, int rows, int cols, float eps, void* ws, int64_t ws_bytes, void* stream) {
    FP_REQUIRE(cols <= MOST_COLS);
    FP_REQUIRE(dy && h && w && dx && dw && rows > 0 && cols > 0 && dy_rs >= 0 && h_rs >= 0 && dx_rs >= cols && eps >= 0.f);
    FP_REQUIRE(!dh || dh_rs >= 0);
    FP_REQUIRE(aligned2(dy) && aligned2(h) && aligned2(dh) && aligned2(w) && aligned2(dx) && aligned2(dw));
    FP_REQUIRE(ws && ((uintptr_t)ws & 15) == 0 && ws_bytes >= fp_rmsnorm_residual_backward_workspace_bytes(rows, cols));
    hipStream_t st = (hipStream_t)stream;
    const int parts = grad_parts(rows, cols);
    float* part = (float*)ws;
    float* rstd = part + (int64_t)parts * ((cols + 7) & ~7);
#define FP_GRAD(TPR, NCH, AHEAD, DW, GRID, R, N, PART)                                                                            \
    rmsnorm_grad_kernel<T, TPR, NCH, AHEAD, DW><<<dim3((unsigned)(GRID)), dim3(TPR < 256 ? 256 : TPR), 0, st>>>(                  \
        (const T*)dy + (R) * dy_rs, dy_rs, (const T*)h + (R) * h_rs, h_rs, dh ? (const T*)dh + (R) * dh_rs : nullptr, dh_rs,      \
        (const T*)w, (T*)dx + (R) * dx_rs, dx_rs, PART, N, cols, eps)
    const int nch = (cols + 7) / 8;
    if (nch <= 64) FP_GRAD(64, 1, true, true, parts, 0, rows, part);
    else if (nch <= 128) FP_GRAD(64, 2, true, true, parts, 0, rows, part);
    else if (nch <= 256) FP_GRAD(256, 1, true, true, parts, 0, rows, part);
    else if (nch <= 512) FP_GRAD(256, 2, true, true, parts, 0, rows, part);
    else if (nch <= 1024) FP_GRAD(256, 4, true, true, parts, 0, rows, part);
    else if (nch <= 2048) FP_GRAD(512, 4, false, true, parts, 0, rows, part);
    else {
        for (int64_t r = 0; r < rows; r += MOST) {
            const int n = rows - r < MOST ? (int)(rows - r) : MOST;
            if (nch <= 4096) FP_GRAD(1024, 4, false, false, n, r, n, rstd + r);
            else rmsnorm_grad_rows_kernel<T><<<dim3((unsigned)n), dim3(256), 0, st>>>(
                (const T*)dy + r * dy_rs, dy_rs, (const T*)h + r * h_rs, h_rs, dh ? (const T*)dh + r * dh_rs : nullptr, dh_rs,
                (const T*)w, (T*)dx + r * dx_rs, dx_rs, rstd + r, cols, eps);
            FP_CHECK_LAUNCH();
        }
        rmsnorm_dweight_rows_kernel<T><<<dim3((unsigned)((nch + 255) / 256), (unsigned)parts), dim3(256), 0, st>>>(
            (const T*)dy, dy_rs, (const T*)h, h_rs, rstd, part, rows, cols);
    }
#undef FP_GRAD
    FP_CHECK_LAUNCH();
    rmsnorm_dweight_kernel<T><<<dim3((unsigned)((cols + 31) / 32)), dim3(256), 0, st>>>(part, parts, cols, (T*)dw);
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
    if (rows <= 0 || cols <= 0 || cols > MOST_COLS) return 0;
    return ((int64_t)grad_parts(rows, cols) * (((int64_t)cols + 7) & ~7) + (cols > GRAD_COLS ? (int64_t)rows : 0)) * 4;
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
