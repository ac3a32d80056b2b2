// Group normalisation with an activation for NHWC activations on gfx950.
//
// A sample's P pixels x C channels are cut into G groups of D = C / G neighbouring channels; a group's M = P * D values
// share one mean and one variance:
//   xhat = (x - mean) * rstd,  z = scale_c * xhat + shift_c,  y = act(z) [+ residual]
// Backward, with g = dy * act'(z):
//   dshift_c = sum_{n,p} g,  dscale_c = sum_{n,p} g * xhat
//   dx = rstd * (scale_c g - m1 - xhat * m2),  m1 = sum(scale_c g) / M,  m2 = sum(scale_c g xhat) / M over the group
// One block per (sample, group) forward, three passes over its values; backward sums per (sample, channel) first.
// Statistics and sums are fp32, no atomics.
#include "common.hpp"

namespace stmi {

struct GnGeom {
    int N, P, C, G, D;
};

__device__ __forceinline__ float gn_sigmoid(float z) { return 1.f / (1.f + __expf(-z)); }

// NaN stays NaN in every activation (a maximum with zero would drop it)
__device__ __forceinline__ float gn_act(float z, int act) {
    if (act == STMI_ACT_RELU) return z < 0.f ? 0.f : z;
    if (act == STMI_ACT_SIGMOID) return gn_sigmoid(z);
    if (act == STMI_ACT_SILU) return z * gn_sigmoid(z);
    return z;
}

__device__ __forceinline__ float gn_act_grad(float z, int act) {
    if (act == STMI_ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
    if (act == STMI_ACT_SIGMOID) {
        const float s = gn_sigmoid(z);
        return s * (1.f - s);
    }
    if (act == STMI_ACT_SILU) {
        const float s = gn_sigmoid(z);
        return s * (1.f + z * (1.f - s));
    }
    return 1.f;
}

__device__ __forceinline__ float gn_block_sum(float v, float* red) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const float r = red[0] + red[1] + red[2] + red[3];
    __syncthreads();
    return r;
}

template <typename T>
__global__ __launch_bounds__(256) void gn_fwd_kernel(const T* x, const float* __restrict__ scale,
                                                     const float* __restrict__ shift, const T* residual, T* y,
                                                     float* __restrict__ stats, float eps, int act, GnGeom g) {
    __shared__ float red[4];
    const int n = blockIdx.x / g.G, gr = blockIdx.x % g.G;
    const long base = (long)n * g.P * g.C + (long)gr * g.D, m = (long)g.P * g.D;
    float s = 0.f;
    for (long i = threadIdx.x; i < m; i += 256) s += to_f32<T>(x[base + i / g.D * g.C + i % g.D]);
    const float mean = gn_block_sum(s, red) / (float)m;
    s = 0.f;
    for (long i = threadIdx.x; i < m; i += 256) {
        const float d = to_f32<T>(x[base + i / g.D * g.C + i % g.D]) - mean;
        s += d * d;
    }
    const float rstd = 1.f / sqrtf(gn_block_sum(s, red) / (float)m + eps);
    if (threadIdx.x == 0) {
        stats[(long)blockIdx.x * 2] = mean;
        stats[(long)blockIdx.x * 2 + 1] = rstd;
    }
    for (long i = threadIdx.x; i < m; i += 256) {
        const long at = base + i / g.D * g.C + i % g.D;
        const int c = gr * g.D + (int)(i % g.D);
        float v = gn_act((to_f32<T>(x[at]) - mean) * (scale[c] * rstd) + shift[c], act);
        if (residual) v += to_f32<T>(residual[at]);
        y[at] = from_f32<T>(v);
    }
}

// rows[n][0][c] = sum_p g, rows[n][1][c] = sum_p g * xhat: one block per (sample, channel)
template <typename T>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                          const float* __restrict__ stats, const float* __restrict__ scale,
                                                          const float* __restrict__ shift, float* __restrict__ rows,
                                                          int act, GnGeom g) {
    __shared__ float red[4];
    const int n = blockIdx.x / g.C, c = blockIdx.x % g.C;
    const float mean = stats[((long)n * g.G + c / g.D) * 2], rstd = stats[((long)n * g.G + c / g.D) * 2 + 1];
    const long base = (long)n * g.P * g.C + c;
    float s1 = 0.f, s2 = 0.f;
    for (int p = threadIdx.x; p < g.P; p += 256) {
        const float d = to_f32<T>(x[base + (long)p * g.C]) - mean;
        const float gv = to_f32<T>(dy[base + (long)p * g.C]) * gn_act_grad(d * (scale[c] * rstd) + shift[c], act);
        s1 += gv;
        s2 += gv * (d * rstd);
    }
    s1 = gn_block_sum(s1, red);
    s2 = gn_block_sum(s2, red);
    if (threadIdx.x == 0) {
        rows[((long)n * 2) * g.C + c] = s1;
        rows[((long)n * 2 + 1) * g.C + c] = s2;
    }
}

template <typename T>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(const T* x, const T* dy, const float* __restrict__ stats,
                                                           const float* __restrict__ scale, const float* __restrict__ shift,
                                                           const float* __restrict__ rows, T* dx, int act, GnGeom g) {
    const int n = blockIdx.x / g.G, gr = blockIdx.x % g.G;
    const long base = (long)n * g.P * g.C + (long)gr * g.D, m = (long)g.P * g.D;
    const float mean = stats[(long)blockIdx.x * 2], rstd = stats[(long)blockIdx.x * 2 + 1];
    float m1 = 0.f, m2 = 0.f;
    for (int c = gr * g.D; c < (gr + 1) * g.D; c++) {
        m1 += scale[c] * rows[((long)n * 2) * g.C + c];
        m2 += scale[c] * rows[((long)n * 2 + 1) * g.C + c];
    }
    m1 /= (float)m;
    m2 /= (float)m;
    for (long i = threadIdx.x; i < m; i += 256) {
        const long at = base + i / g.D * g.C + i % g.D;
        const int c = gr * g.D + (int)(i % g.D);
        const float d = to_f32<T>(x[at]) - mean;
        const float gv = to_f32<T>(dy[at]) * gn_act_grad(d * (scale[c] * rstd) + shift[c], act);
        dx[at] = from_f32<T>(rstd * (scale[c] * gv - m1 - d * rstd * m2));
    }
}

// dshift[c] (+)= sum over samples of rows[n][0][c], dscale[c] (+)= of rows[n][1][c], in sample order
__global__ __launch_bounds__(256) void gn_param_grads_kernel(const float* __restrict__ rows, float* __restrict__ dscale,
                                                             float* __restrict__ dshift, int n, int C, int accumulate) {
    const int o = blockIdx.x * 256 + threadIdx.x;
    if (o >= 2 * C) return;
    float s = 0.f;
    for (int i = 0; i < n; i++) s += rows[(long)i * 2 * C + o];
    float* dst = o < C ? dshift + o : dscale + (o - C);
    *dst = accumulate ? *dst + s : s;
}

long gn_ws_floats(int n, int h, int w, int c, int groups, int dtype) { return (long)n * 2 * c; }

template <typename T>
static int gn_fwd_t(const T* x, float* stats, float eps, const float* scale, const float* shift, const T* residual, T* y,
                    int act, const GnGeom& g, hipStream_t s) {
    hipLaunchKernelGGL(gn_fwd_kernel<T>, dim3((unsigned)(g.N * g.G)), dim3(256), 0, s, x, scale, shift, residual, y, stats, eps, act, g);
    STMI_LAUNCH_CHECK("gn_fwd_kernel");
    return STMI_OK;
}

int gn_fwd_impl(const void* x, float* ws, float* stats, float eps, const float* scale, const float* shift,
                const void* residual, void* y, int act, int n, int h, int w, int c, int groups, int dtype, hipStream_t s) {
    const GnGeom g{n, h * w, c, groups, c / groups};
    if (dtype == STMI_BF16)
        return gn_fwd_t((const bf16_t*)x, stats, eps, scale, shift, (const bf16_t*)residual, (bf16_t*)y, act, g, s);
    return gn_fwd_t((const float*)x, stats, eps, scale, shift, (const float*)residual, (float*)y, act, g, s);
}

template <typename T>
static int gn_bwd_t(const T* x, const T* dy, const float* stats, const float* scale, const float* shift, T* dx, float* ws,
                    int act, const GnGeom& g, hipStream_t s) {
    hipLaunchKernelGGL(gn_bwd_sums_kernel<T>, dim3((unsigned)(g.N * g.C)), dim3(256), 0, s, x, dy, stats, scale, shift, ws, act, g);
    STMI_LAUNCH_CHECK("gn_bwd_sums_kernel");
    hipLaunchKernelGGL(gn_bwd_apply_kernel<T>, dim3((unsigned)(g.N * g.G)), dim3(256), 0, s, x, dy, stats, scale, shift,
                       (const float*)ws, dx, act, g);
    STMI_LAUNCH_CHECK("gn_bwd_apply_kernel");
    return STMI_OK;
}

int gn_bwd_impl(const void* x, const void* dy, const float* stats, const float* scale, const float* shift, void* dx,
                float* dscale, float* dshift, int accumulate, float* ws, int act, int n, int h, int w, int c, int groups,
                int dtype, hipStream_t s) {
    const GnGeom g{n, h * w, c, groups, c / groups};
    if (n > 0) {
        const int rc = dtype == STMI_BF16
                           ? gn_bwd_t((const bf16_t*)x, (const bf16_t*)dy, stats, scale, shift, (bf16_t*)dx, ws, act, g, s)
                           : gn_bwd_t((const float*)x, (const float*)dy, stats, scale, shift, (float*)dx, ws, act, g, s);
        if (rc) return rc;
    }
    if (dscale) {
        hipLaunchKernelGGL(gn_param_grads_kernel, dim3(ceil_div(2L * c, 256)), dim3(256), 0, s, (const float*)ws, dscale, dshift, n, c, accumulate);
        STMI_LAUNCH_CHECK("gn_param_grads_kernel");
    }
    return STMI_OK;
}

}  // namespace stmi
