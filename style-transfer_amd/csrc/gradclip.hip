// The global L2 norm over many gradient tensors, and clipping by it, on gfx950 (HBM-bound).
//   norm = sqrt(sum_i sum g_i^2),  factor = max_norm / max(norm, max_norm),  out_i = factor * g_i
// The tensors are cut into chunks of at most kChunk elements; a device table names every chunk, so one launch covers any
// number of tensors of any lengths and types.  Squares are summed in double: a finite fp32 gradient can neither overflow
// nor vanish in the sum, and a block's partial sum in `ws` is added up in a fixed order (no atomics).
#include "common.hpp"

namespace stmi {

constexpr int kChunk = 8192;

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// sum over a 256-thread block, valid in every thread; red: 4 doubles of shared memory
__device__ __forceinline__ double block_sum_d(double v, double* red) {
    v = wave_sum_d(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const double r = (red[0] + red[1]) + (red[2] + red[3]);
    __syncthreads();
    return r;
}

// the sum of squares from the partial sums, in the same order in every block and every kernel
__device__ __forceinline__ double fold_squares(const double* __restrict__ ws, double* red) {
    double v = 0.0;
    for (int i = threadIdx.x; i < STMI_GRAD_WS_DOUBLES; i += 256) v += ws[i];
    return block_sum_d(v, red);
}

// max_norm / max(norm, max_norm); NaN where the norm is not finite
__device__ __forceinline__ float clip_factor(double norm, float max_norm) {
    if (!(norm <= 1.7976931348623157e308)) return __builtin_nanf("");
    return norm > (double)max_norm ? (float)((double)max_norm / norm) : 1.f;
}

template <typename T>
__device__ __forceinline__ double chunk_squares(const T* src, int count) {
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += 256) {
        const double v = (double)to_f32<T>(src[i]);
        s += v * v;
    }
    return s;
}

__global__ __launch_bounds__(256) void grad_squares_kernel(const stmi_grad_chunk* __restrict__ table, int nchunks,
                                                           double* __restrict__ ws) {
    __shared__ double red[4];
    double s = 0.0;
    for (int k = blockIdx.x; k < nchunks; k += gridDim.x) {
        const stmi_grad_chunk ch = table[k];
        s += ch.dtype == STMI_BF16 ? chunk_squares((const bf16_t*)ch.src, ch.count) : chunk_squares((const float*)ch.src, ch.count);
    }
    s = block_sum_d(s, red);
    if (threadIdx.x == 0) ws[blockIdx.x] = s;
    if (blockIdx.x == 0)
        for (int i = gridDim.x + threadIdx.x; i < STMI_GRAD_WS_DOUBLES; i += 256) ws[i] = 0.0;
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* __restrict__ ws, float* __restrict__ norm) {
    __shared__ double red[4];
    const double s = fold_squares(ws, red);
    if (threadIdx.x == 0) norm[0] = (float)sqrt(s);
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const T* src, T* dst, int count, float f) {
    for (int i = threadIdx.x; i < count; i += 256) dst[i] = from_f32<T>(to_f32<T>(src[i]) * f);
}

__global__ __launch_bounds__(256) void grad_scale_kernel(const stmi_grad_chunk* __restrict__ table, int nchunks,
                                                         const double* __restrict__ ws, float max_norm,
                                                         float* __restrict__ norm_out) {
    __shared__ double red[4];
    const double norm = sqrt(fold_squares(ws, red));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
    const float f = clip_factor(norm, max_norm);
    for (int k = blockIdx.x; k < nchunks; k += gridDim.x) {
        const stmi_grad_chunk ch = table[k];
        if (f == 1.f && ch.src == ch.dst) continue;
        if (ch.dtype == STMI_BF16)
            chunk_scale((const bf16_t*)ch.src, (bf16_t*)ch.dst, ch.count, f);
        else
            chunk_scale((const float*)ch.src, (float*)ch.dst, ch.count, f);
    }
}

long grad_list_chunks(const long* counts, int n) {
    long k = 0;
    for (int i = 0; i < n; i++) k += (counts[i] + kChunk - 1) / kChunk;
    return k;
}

void grad_list_fill(const void* const* srcs, void* const* dsts, const long* counts, const int* dtypes, int n,
                    stmi_grad_chunk* table) {
    long k = 0;
    for (int i = 0; i < n; i++) {
        const long size = dtypes[i] == STMI_BF16 ? 2 : 4;
        for (long at = 0; at < counts[i]; at += kChunk, k++) {
            table[k].src = (const char*)srcs[i] + at * size;
            table[k].dst = (char*)dsts[i] + at * size;
            table[k].count = (int)(counts[i] - at < kChunk ? counts[i] - at : kChunk);
            table[k].dtype = dtypes[i];
        }
    }
}

static dim3 chunk_grid(int nchunks) {
    return dim3((unsigned)(nchunks < 1 ? 1 : nchunks < STMI_GRAD_WS_DOUBLES ? nchunks : STMI_GRAD_WS_DOUBLES));
}

int grad_squares_impl(const stmi_grad_chunk* table, int nchunks, double* ws, hipStream_t s) {
    hipLaunchKernelGGL(grad_squares_kernel, chunk_grid(nchunks), dim3(256), 0, s, table, nchunks, ws);
    STMI_LAUNCH_CHECK("grad_squares_kernel");
    return STMI_OK;
}

int grad_norm_impl(const double* ws, float* norm, hipStream_t s) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, s, ws, norm);
    STMI_LAUNCH_CHECK("grad_norm_kernel");
    return STMI_OK;
}

int grad_scale_impl(const stmi_grad_chunk* table, int nchunks, const double* ws, float max_norm, float* norm, hipStream_t s) {
    hipLaunchKernelGGL(grad_scale_kernel, chunk_grid(nchunks), dim3(256), 0, s, table, nchunks, ws, max_norm, norm);
    STMI_LAUNCH_CHECK("grad_scale_kernel");
    return STMI_OK;
}

// ------------------------------------------------------------------ Adam with clipping
// The update of stmi_adam_tf1 with g' = g * grad_scale * factor, factor from the norm of g * grad_scale: clipping costs
// no pass of its own.
__global__ __launch_bounds__(256) void adam_clip_kernel(float* __restrict__ p, const float* __restrict__ g,
                                                        float* __restrict__ m, float* __restrict__ v, long count, float lr,
                                                        float b1, float b2, float eps, float grad_scale,
                                                        const double* __restrict__ ws, float max_norm,
                                                        float* __restrict__ norm_out, const int* step_dev, int t_host) {
    __shared__ double red[4];
    __shared__ float sh;
    const double norm = sqrt(fold_squares(ws, red)) * fabs((double)grad_scale);
    if (threadIdx.x == 0) {
        const int t = step_dev ? step_dev[0] : t_host;
        sh = (float)((double)lr * sqrt(1.0 - pow((double)b2, (double)t)) / (1.0 - pow((double)b1, (double)t)));
        if (norm_out && blockIdx.x == 0) norm_out[0] = (float)norm;
    }
    __syncthreads();
    const float lr_t = sh, gs = grad_scale * clip_factor(norm, max_norm);
    for (long i = blockIdx.x * 256L + threadIdx.x; i < count; i += gridDim.x * 256L) {
        const float gi = g[i] * gs;
        const float mi = b1 * m[i] + (1.f - b1) * gi;
        const float vi = b2 * v[i] + (1.f - b2) * gi * gi;
        m[i] = mi;
        v[i] = vi;
        p[i] -= lr_t * mi / (sqrtf(vi) + eps);
    }
}

__global__ void bump_step_kernel(int* step);

int adam_clip_impl(float* p, const float* g, float* m, float* v, long count, float lr, float b1, float b2, float eps,
                   float grad_scale, const double* ws, float max_norm, float* norm, int* step_dev, int t, hipStream_t s) {
    if (step_dev && t >= 0) {
        hipLaunchKernelGGL(bump_step_kernel, dim3(1), dim3(64), 0, s, step_dev);
        STMI_LAUNCH_CHECK("bump_step_kernel");
    }
    const long blocks = (count + 255) / 256;
    hipLaunchKernelGGL(adam_clip_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, s, p, g, m, v, count,
                       lr, b1, b2, eps, grad_scale, ws, max_norm, norm, (const int*)step_dev, t);
    STMI_LAUNCH_CHECK("adam_clip_kernel");
    return STMI_OK;
}

}  // namespace stmi
