// The global L2 norm over many gradient tensors, clipping by it, and Adam with the clipping inside, on gfx950 (HBM-bound).
//   norm = sqrt(sum_i sum g_i^2),  factor = max_norm / max(norm, max_norm),  out_i = factor * g_i
// The tensors are cut into chunks of at most kChunkBytes; a device table names every chunk, so one launch covers any number
// of tensors of any lengths and types, and a block takes the chunks blockIdx, blockIdx + gridDim, ...  A chunk is four
// 16-byte accesses a thread, at the elements' alignment (global memory takes them at any address).
// Squares are summed in double: a finite fp32 gradient can neither overflow nor vanish in the sum, and the long sum costs
// no accuracy; v_fma_f64 runs at the fp32 rate here, so the pass stays bound by its bytes.  A block leaves one partial sum
// in ws; every kernel that needs the norm adds the partial sums up itself, in one fixed order (no atomics, no launch of its
// own).
#include "common.hpp"

namespace stmi {

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

constexpr int kChunkBytes = 16384, kVecs = kChunkBytes / 16 / 256;   // 16-byte accesses of a thread
// Chunks (32 MB) from which the outputs go past the caches: the second reading of the tensors then still finds them in the
// last-level cache (600 ragged tensors, 223 MB read and written: 71 us with ordinary stores, 57 without).
constexpr int kStreamChunks = (32 << 20) / kChunkBytes;

template <bool kNt>
__device__ __forceinline__ u32x4 load16(const void* p) {
    typedef u32x4 __attribute__((aligned(2))) loose;
    const loose* q = static_cast<const loose*>(p);
    if constexpr (kNt) return __builtin_nontemporal_load(q);
    return *q;
}

template <bool kNt>
__device__ __forceinline__ void store16(void* p, const u32x4& v) {
    typedef u32x4 __attribute__((aligned(2))) loose;
    loose* q = static_cast<loose*>(p);
    if constexpr (kNt) __builtin_nontemporal_store(v, q);
    else *q = v;
}

// sum over a 256-thread block, valid in every thread; red: 4 doubles of shared memory
__device__ __forceinline__ double block_sum_d(double v, double* red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

// the sum of squares from the partial sums, in the same order in every block and every kernel
__device__ __forceinline__ double fold_squares(const double* __restrict__ ws, int nparts, double* red) {
    double v = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < nparts; i += 256) v += ws[i];
    return block_sum_d(v, red);
}

// scale * max_norm / max(norm, max_norm) as a product of two fp32 factors; NaN where the norm is not finite.
// b is 1 unless the factor is below 2^-120 (norms of finite gradients reach 2^128 and more), too little for one fp32 number.  A
// normal result then needs |g| > 2^-6, and g * 2^-120 is still a normal number: nothing is lost before the last product.
struct ClipFactor {
    float a, b;
    __device__ __forceinline__ ClipFactor(double norm, float max_norm, double scale) : b(1.f) {
        const double f = norm > (double)max_norm ? scale * ((double)max_norm / norm) : scale;
        const bool tiny = fabs(f) < 0x1p-120 && f != 0.0;
        a = !(norm <= 1.7976931348623157e308) ? __builtin_nanf("") : tiny ? 0x1p-120f : (float)f;
        if (tiny) b = (float)(f * 0x1p120);
    }
    __device__ __forceinline__ float operator()(float g) const { return g * a * b; }
};

// the vectors of a chunk that thread i owns
struct Chunk {
    const char* src;
    char* dst;
    int count, vecs;   // elements, whole 16-byte vectors
    bool half;         // bf16
    __device__ __forceinline__ explicit Chunk(const stmi_grad_chunk& c)
        : src((const char*)c.src), dst((char*)c.dst), count(c.count), half(c.dtype == STMI_BF16) {
        vecs = half ? count >> 3 : count >> 2;
    }
    __device__ __forceinline__ void load(u32x4 (&raw)[kVecs]) const {
#pragma unroll
        for (int u = 0; u < kVecs; u++) {
            const int i = threadIdx.x + u * 256;
            if (i < vecs) raw[u] = load16<false>(src + i * 16);
        }
    }
};

__device__ __forceinline__ float bf16_lo(unsigned w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float bf16_hi(unsigned w) { return __builtin_bit_cast(float, w & 0xffff0000u); }
__device__ __forceinline__ unsigned bf16_pair(float lo, float hi) {
    bf16_t e[2] = {(bf16_t)lo, (bf16_t)hi};
    unsigned w;
    __builtin_memcpy(&w, e, 4);
    return w;
}

// 600 tensors, 112 MB: 21 us, 5.2 TB/s
__global__ __launch_bounds__(256) void grad_squares_kernel(const stmi_grad_chunk* __restrict__ table, int nchunks,
                                                           double* __restrict__ ws) {
    __shared__ double red[4];
    double s0 = 0.0, s1 = 0.0;
    for (int k = blockIdx.x; k < nchunks; k += gridDim.x) {
        const Chunk ch(table[k]);
        u32x4 raw[kVecs];
        ch.load(raw);
#pragma unroll
        for (int u = 0; u < kVecs; u++) {
            if (threadIdx.x + u * 256 >= (unsigned)ch.vecs) continue;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned w = raw[u][j];
                if (ch.half) {
                    const double lo = bf16_lo(w), hi = bf16_hi(w);
                    s0 = __builtin_fma(lo, lo, s0);
                    s1 = __builtin_fma(hi, hi, s1);
                } else {
                    const double v = __builtin_bit_cast(float, w);
                    if (j & 1) s1 = __builtin_fma(v, v, s1);
                    else s0 = __builtin_fma(v, v, s0);
                }
            }
        }
        const int at = (ch.half ? ch.vecs << 3 : ch.vecs << 2) + threadIdx.x;   // what does not fill a vector
        if (at < ch.count) {
            const double v = ch.half ? (double)to_f32<bf16_t>(((const bf16_t*)ch.src)[at]) : (double)((const float*)ch.src)[at];
            s0 = __builtin_fma(v, v, s0);
        }
    }
    s0 = block_sum_d(s0 + s1, red);
    if (threadIdx.x == 0) ws[blockIdx.x] = s0;
}

__global__ __launch_bounds__(256) void grad_norm_kernel(const double* __restrict__ ws, int nparts, float* __restrict__ norm) {
    __shared__ double red[4];
    const double s = fold_squares(ws, nparts, red);
    if (threadIdx.x == 0) norm[0] = (float)sqrt(s);
}

// The chunks are taken from the last to the first: what grad_squares_kernel read last is the likeliest to be in a cache
// still.  The loads of a block's first chunk are on their way while it folds the partial sums.
// 600 tensors, 223 MB read and written: 36 us, 6.2 TB/s
template <bool kNt>
__global__ __launch_bounds__(256) void grad_scale_kernel(const stmi_grad_chunk* __restrict__ table, int nchunks,
                                                         const double* __restrict__ ws, int nparts, float max_norm,
                                                         float* __restrict__ norm_out) {
    __shared__ double red[4];
    u32x4 raw[kVecs];
    int k = nchunks - 1 - (int)blockIdx.x;
    if (k >= 0) Chunk(table[k]).load(raw);
    const double norm = sqrt(fold_squares(ws, nparts, red));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
    const ClipFactor f(norm, max_norm, 1.0);
    for (bool first = true; k >= 0; k -= gridDim.x, first = false) {
        const Chunk ch(table[k]);
        if (f.a == 1.f && ch.src == ch.dst) continue;
        if (!first) ch.load(raw);
#pragma unroll
        for (int u = 0; u < kVecs; u++) {
            const int i = threadIdx.x + u * 256;
            if (i >= ch.vecs) continue;
            u32x4 o;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const unsigned w = raw[u][j];
                o[j] = ch.half ? bf16_pair(f(bf16_lo(w)), f(bf16_hi(w))) : __builtin_bit_cast(unsigned, f(__builtin_bit_cast(float, w)));
            }
            store16<kNt>(ch.dst + i * 16, o);
        }
        const int at = (ch.half ? ch.vecs << 3 : ch.vecs << 2) + threadIdx.x;
        if (at < ch.count) {
            if (ch.half) ((bf16_t*)ch.dst)[at] = (bf16_t)f(to_f32<bf16_t>(((const bf16_t*)ch.src)[at]));
            else ((float*)ch.dst)[at] = f(((const float*)ch.src)[at]);
        }
    }
}

static long chunk_elems(int dtype) { return kChunkBytes / (dtype == STMI_BF16 ? 2 : 4); }

long grad_list_chunks(const long* counts, const int* dtypes, int n) {
    long k = 0;
    for (int i = 0; i < n; i++) k += (counts[i] + chunk_elems(dtypes[i]) - 1) / chunk_elems(dtypes[i]);
    return k;
}

void grad_list_fill(const void* const* srcs, void* const* dsts, const long* counts, const int* dtypes, int n,
                    stmi_grad_chunk* table) {
    long k = 0;
    for (int i = 0; i < n; i++) {
        const long size = dtypes[i] == STMI_BF16 ? 2 : 4, most = chunk_elems(dtypes[i]);
        for (long at = 0; at < counts[i]; at += most, k++) {
            table[k].src = (const char*)srcs[i] + at * size;
            table[k].dst = (char*)dsts[i] + at * size;
            table[k].count = (int)(counts[i] - at < most ? counts[i] - at : most);
            table[k].dtype = dtypes[i];
        }
    }
}

static int chunk_blocks(int nchunks) { return nchunks < 1 ? 1 : nchunks < STMI_GRAD_WS_DOUBLES ? nchunks : STMI_GRAD_WS_DOUBLES; }

int grad_squares_impl(const stmi_grad_chunk* table, int nchunks, double* ws, hipStream_t s) {
    hipLaunchKernelGGL(grad_squares_kernel, dim3(chunk_blocks(nchunks)), dim3(256), 0, s, table, nchunks, ws);
    STMI_LAUNCH_CHECK("grad_squares_kernel");
    return STMI_OK;
}

int grad_norm_impl(const double* ws, int nchunks, float* norm, hipStream_t s) {
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(256), 0, s, ws, chunk_blocks(nchunks), norm);
    STMI_LAUNCH_CHECK("grad_norm_kernel");
    return STMI_OK;
}

int grad_scale_impl(const stmi_grad_chunk* table, int nchunks, const double* ws, float max_norm, float* norm, hipStream_t s) {
    const int blocks = chunk_blocks(nchunks);
    if (nchunks > kStreamChunks)
        hipLaunchKernelGGL(grad_scale_kernel<true>, dim3(blocks), dim3(256), 0, s, table, nchunks, ws, blocks, max_norm, norm);
    else
        hipLaunchKernelGGL(grad_scale_kernel<false>, dim3(blocks), dim3(256), 0, s, table, nchunks, ws, blocks, max_norm, norm);
    STMI_LAUNCH_CHECK("grad_scale_kernel");
    return STMI_OK;
}

// ------------------------------------------------------------------ Adam with clipping
// The update of stmi_adam_tf1 with g' = g * (grad_scale * factor), factor from the norm of g * grad_scale: clipping costs
// no pass of its own.  The rates come in double: 1 - beta2 and 1 - beta2^t of an fp32 0.999 are 1.3e-5 off, and the step
// with them.  (stmi_adam_tf1 keeps fp32 rates: the two updates agree to 1.3e-5 where nothing is clipped, not to the bit.)  28 bytes a parameter; four parameters a thread and access, and the loads of a thread's first ones
// are on their way while the block folds the partial sums and one thread of its last wave works out the step size.
// 20 M parameters (561 MB): 95 us, 5.9 TB/s with the gradients still cached; 1.7 M (47 MB) 12 us.

// b^t for t >= 0 by squaring: t times 2^-53 off at most, and shorter than two pow()
__device__ __forceinline__ double pow_int(double b, unsigned t) {
    double r = 1.0;
    for (; t; t >>= 1, b *= b)
        if (t & 1) r *= b;
    return r;
}

template <bool kNt>
__global__ __launch_bounds__(256) void adam_clip_kernel(float* __restrict__ p, const float* __restrict__ g,
                                                        float* __restrict__ m, float* __restrict__ v, long count, double lr,
                                                        double beta1, double beta2, float eps, float grad_scale,
                                                        const double* __restrict__ ws, int nparts, float max_norm,
                                                        float* __restrict__ norm_out, const int* step_dev, int t_host) {
    __shared__ double red[4];
    __shared__ float sh;
    const long quads = count >> 2, stride = gridDim.x * 256L;
    long q = blockIdx.x * 256L + threadIdx.x;
    u32x4 rg, rp, rm, rv;
    if (q < quads) {
        rg = load16<false>(g + q * 4);
        rm = load16<kNt>(m + q * 4);
        rv = load16<kNt>(v + q * 4);
        rp = load16<kNt>(p + q * 4);
    }
    if (threadIdx.x == 255) {
        const unsigned t = step_dev ? step_dev[0] : t_host;
        sh = (float)(lr * sqrt(1.0 - pow_int(beta2, t)) / (1.0 - pow_int(beta1, t)));
    }
    const float b1 = (float)beta1, b2 = (float)beta2, c1 = (float)(1.0 - beta1), c2 = (float)(1.0 - beta2);
    const double norm = sqrt(fold_squares(ws, nparts, red)) * fabs((double)grad_scale);   // its barrier is sh's too
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) norm_out[0] = (float)norm;
    const float lr_t = sh;
    const ClipFactor factor(norm, max_norm, grad_scale);
    auto update = [&](float gi, float& mi, float& vi, float& pi) {
        gi = factor(gi);
        mi = b1 * mi + c1 * gi;
        vi = b2 * vi + c2 * gi * gi;
        pi -= lr_t * mi / (sqrtf(vi) + eps);
    };
    for (bool first = true; q < quads; q += stride, first = false) {
        if (!first) {
            rg = load16<false>(g + q * 4);
            rm = load16<kNt>(m + q * 4);
            rv = load16<kNt>(v + q * 4);
            rp = load16<kNt>(p + q * 4);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const unsigned wg = rg[j], wm = rm[j], wv = rv[j], wp = rp[j];
            float mi = __builtin_bit_cast(float, wm), vi = __builtin_bit_cast(float, wv), pi = __builtin_bit_cast(float, wp);
            update(__builtin_bit_cast(float, wg), mi, vi, pi);
            rm[j] = __builtin_bit_cast(unsigned, mi);
            rv[j] = __builtin_bit_cast(unsigned, vi);
            rp[j] = __builtin_bit_cast(unsigned, pi);
        }
        store16<kNt>(m + q * 4, rm);
        store16<kNt>(v + q * 4, rv);
        store16<kNt>(p + q * 4, rp);
    }
    if (blockIdx.x == gridDim.x - 1) {
        const long i = (quads << 2) + threadIdx.x;
        if (i < count) update(g[i], m[i], v[i], p[i]);
    }
}

__global__ void bump_step_kernel(int* step);

int adam_clip_impl(float* p, const float* g, float* m, float* v, long count, double lr, double b1, double b2, float eps,
                   float grad_scale, const double* ws, int nchunks, float max_norm, float* norm, int* step_dev, int t,
                   hipStream_t s) {
    if (step_dev && t >= 0) {
        hipLaunchKernelGGL(bump_step_kernel, dim3(1), dim3(64), 0, s, step_dev);
        STMI_LAUNCH_CHECK("bump_step_kernel");
    }
    const long blocks = (count / 4 + 255) / 256;
    const dim3 grid((unsigned)(blocks < 1 ? 1 : blocks < 2048 ? blocks : 2048));
    // parameters and moments beyond the last-level cache (256 MB) go past it: the gradients, read a moment ago, stay there
    auto f = count * 28 > (256L << 20) ? adam_clip_kernel<true> : adam_clip_kernel<false>;
    hipLaunchKernelGGL(f, grid, dim3(256), 0, s, p, g, m, v, count, lr, b1, b2, eps, grad_scale, ws, chunk_blocks(nchunks), max_norm,
                       norm, (const int*)step_dev, t);
    STMI_LAUNCH_CHECK("adam_clip_kernel");
    return STMI_OK;
}

}  // namespace stmi
