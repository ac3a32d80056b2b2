// Group normalisation with an activation for NHWC activations on gfx950 (HBM-bound).
//
// A sample's P pixels x C channels are cut into G groups of D = C / G neighbouring channels; a group's M = P * D values
// share one mean and one variance:
//   xhat = (x - mean) * rstd,  z = scale_c * xhat + shift_c,  y = act(z) [+ residual]
// Backward, with g = dy * act'(z):
//   dshift_c = sum_{n,p} g,  dscale_c = sum_{n,p} g * xhat
//   dx = rstd * (scale_c g - m1 - xhat * m2),  m1 = sum(scale_c g) / M,  m2 = sum(scale_c g xhat) / M over the group
//
// Two launches a direction: a reduction over slices of the samples leaves one partial result per slice and group, and the
// blocks of the second launch fold the partials of their sample and stream the tensor once more.
//
// Layout of the work: a sample is a flat run of P * C elements, cut into rows of L = lcm(C, V) elements (V: the elements
// of a 16-byte access), so that a thread that owns one 16-byte column of a row sees the SAME V channels in every row
// whatever C is.  What does not fill a row behind the last one is the tail; it belongs to the last slice.  The cut depends
// on the sample's own size alone, and accesses need only the elements' alignment (global memory takes 16-byte accesses at
// any address): a sample's bits depend neither on its batch nor on its place.
// Statistics are merged as (count, mean, sum of squared deviations) with the means of the parts (Chan et al.): no
// cancellation however large the mean is next to the deviation.  Sums are fp32, no atomics: bit-reproducible.
#include "common.hpp"

#include <type_traits>

namespace stmi {

constexpr int kGnT = 512;      // threads of a block
constexpr int kGnSlices = 512; // most slices of a sample
constexpr int kGnFold = 8192;  // partials (slices x groups) of a sample that the apply blocks fold themselves

struct GnGeom {
    int N, P, C, G, D;
    int L, Q, R;     // elements and V-wide columns of a row, whole rows of a sample
    int QT, tiles;   // columns a block owns, blocks side by side in a row
    int S, rows;     // slices of a sample, rows of a slice
};

// ------------------------------------------------------------------ activations
template <int A>
__device__ __forceinline__ float gn_act(float z) {
    if constexpr (A == STMI_ACT_RELU) return z < 0.f ? 0.f : z;   // NaN stays NaN
    if constexpr (A == STMI_ACT_SIGMOID) return __builtin_amdgcn_rcpf(1.f + __expf(-z));
    if constexpr (A == STMI_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return z;
}

template <int A>
__device__ __forceinline__ float gn_act_grad(float z) {
    if constexpr (A == STMI_ACT_RELU) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
    if constexpr (A == STMI_ACT_SIGMOID) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
        return s * (1.f - s);
    }
    if constexpr (A == STMI_ACT_SILU) {
        const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
        return s * (1.f + z * (1.f - s));
    }
    return 1.f;
}

// f is compiled once per activation, outside its loops
template <typename F>
__device__ __forceinline__ void gn_with_act(int act, F&& f) {
    if (act == STMI_ACT_RELU) f(std::integral_constant<int, STMI_ACT_RELU>{});
    else if (act == STMI_ACT_SIGMOID) f(std::integral_constant<int, STMI_ACT_SIGMOID>{});
    else if (act == STMI_ACT_SILU) f(std::integral_constant<int, STMI_ACT_SILU>{});
    else f(std::integral_constant<int, STMI_ACT_NONE>{});
}

// ------------------------------------------------------------------ merged statistics
struct GnPart {
    float n, mean, m2;
};

__device__ __forceinline__ GnPart gn_merge(const GnPart& a, const GnPart& b) {
    const float n = a.n + b.n, r = n > 0.f ? b.n / n : 0.f, d = b.mean - a.mean;
    if (b.n == 0.f) return a;
    if (a.n == 0.f) return b;
    return GnPart{n, a.mean + d * r, a.m2 + b.m2 + d * d * (a.n * r)};
}

// lanes of a team (a power of two, within a wave) end with the merge of all of them, in one fixed order
__device__ __forceinline__ GnPart gn_merge_team(GnPart a, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) {
        const GnPart b{__shfl_xor(a.n, o, 64), __shfl_xor(a.mean, o, 64), __shfl_xor(a.m2, o, 64)};
        a = (threadIdx.x & o) ? gn_merge(b, a) : gn_merge(a, b);
    }
    return a;
}

__device__ __forceinline__ int gn_team_lanes(int teams) {   // power of two
    int k = 64;
    while (k > 1 && k * teams > kGnT) k >>= 1;
    return k;
}

// 16 bytes at an element's alignment
template <typename T, int V>
__device__ __forceinline__ void gn_load(const T* p, float (&out)[V]) {
    uint4 raw;
    __builtin_memcpy(&raw, p, 16);
    unpack_vec<T, V>(raw, out);
}

template <typename T, int V>
__device__ __forceinline__ void gn_store(T* p, const float (&in)[V]) {
    T e[V];
#pragma unroll
    for (int i = 0; i < V; i++) e[i] = from_f32<T>(in[i]);
    __builtin_memcpy(p, e, 16);
}

// a block's sample, slice and column tile, and what the calling thread owns of the tile
struct GnPlace {
    int n, s, c0, QT, slots, col, slot, r0, r1;
    bool on;
    long base, end0;   // the sample's first element; the tail's, behind the rows, within the sample
    __device__ __forceinline__ explicit GnPlace(const GnGeom& g) {
        const int per = g.S * g.tiles, t = blockIdx.x % per;
        n = blockIdx.x / per;
        s = t / g.tiles;
        c0 = t % g.tiles * g.QT;
        QT = min(g.QT, g.Q - c0);
        slots = kGnT / QT;
        slot = threadIdx.x / QT;
        col = c0 + threadIdx.x % QT;
        on = slot < slots;
        r0 = min(s * g.rows, g.R);
        r1 = min(r0 + g.rows, g.R);
        base = (long)n * g.P * g.C;
        end0 = (long)g.R * g.L;
    }
    __device__ __forceinline__ bool owns_tail(const GnGeom& g) const { return s == g.S - 1 && c0 == 0; }
};

// ------------------------------------------------------------------ forward, first launch
// ws[n][slice * tiles + tile][3][G]: (count, mean, sum of squared deviations) of the block's values of each group.
// A thread keeps a mean and a sum of squared deviations per channel of its column: a batch of kB values is summed as
// deviations from the mean so far (from the first value in the first batch), then mean += s1 / n, m2 += s2 - s1^2 / n
// with n the count behind the batch.  That shift is a value of the plane or a mean of some, so s2 exceeds the sum it
// stands for by no more than the batch's share of the total, and the short batches keep partial sums short.
template <typename T, int V>
__global__ __launch_bounds__(kGnT) void gn_stats_kernel(const T* __restrict__ x, float* __restrict__ ws, const GnGeom g) {
    constexpr int kB = 8;
    extern __shared__ float sh[];   // [V][kGnT] means, [V][kGnT] sums of squares, [kGnT] counts
    const GnPlace p(g);
    const T* xs = x + p.base;
    float mean[V], m2[V];
#pragma unroll
    for (int j = 0; j < V; j++) mean[j] = m2[j] = 0.f;
    int cnt = 0;
    if (p.on) {
        const T* xc = xs + (long)p.col * V;
        for (int row = p.r0 + p.slot; row < p.r1; row += p.slots * kB) {
            float v[kB][V];
            int m = 0;
#pragma unroll
            for (int u = 0; u < kB; u++) {
                if (row + u * p.slots < p.r1) {
                    gn_load<T, V>(xc + (long)(row + u * p.slots) * g.L, v[u]);
                    m++;
                }
            }
            if (cnt == 0) {
#pragma unroll
                for (int j = 0; j < V; j++) mean[j] = v[0][j];
            }
            cnt += m;
            const float rn = 1.f / (float)cnt;
#pragma unroll
            for (int j = 0; j < V; j++) {
                float s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int u = 0; u < kB; u++) {
                    const float d = u < m ? v[u][j] - mean[j] : 0.f;
                    s1 += d;
                    s2 += d * d;
                }
                const float e = s1 * rn;
                mean[j] += e;
                m2[j] += s2 - s1 * e;
            }
        }
    }
    // V neighbouring channels of one group are merged in the thread
    const bool whole = g.D % V == 0;
    if (whole) {
#pragma unroll
        for (int w = 1; w < V; w <<= 1)
#pragma unroll
            for (int j = 0; j < V; j += 2 * w) {
                const GnPart a = gn_merge(GnPart{(float)(cnt * w), mean[j], m2[j]}, GnPart{(float)(cnt * w), mean[j + w], m2[j + w]});
                mean[j] = a.mean;
                m2[j] = a.m2;
            }
    }
    float* lm = sh;
    float* l2 = sh + V * kGnT;
    int* lc = reinterpret_cast<int*>(sh + 2 * V * kGnT);
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (j && whole) break;
        lm[j * kGnT + threadIdx.x] = mean[j];
        l2[j * kGnT + threadIdx.x] = m2[j];
    }
    lc[threadIdx.x] = p.on ? cnt : 0;
    __syncthreads();
    // a team of lanes merges the entries of one group: `units` per row (channels, or whole columns), every slot
    const int K = gn_team_lanes(g.G), teams = kGnT / K, lane = threadIdx.x & (K - 1);
    const int step = whole ? V : 1, reps = g.L / g.C, units = g.D / step, total = units * reps * p.slots;
    float* out = ws + (((long)p.n * g.S + p.s) * g.tiles + p.c0 / g.QT) * 3 * g.G;
    for (int gr = threadIdx.x / K; gr < (g.G + teams - 1) / teams * teams; gr += teams) {
        GnPart a{0.f, 0.f, 0.f};
        if (gr < g.G) {
            for (int e = lane; e < total; e += K) {
                const int slot = e / (units * reps), rest = e - slot * (units * reps), rep = rest / units;
                const int pos = gr * g.D + (rest - rep * units) * step + rep * g.C;
                const int col = pos / V - p.c0;
                if (col < 0 || col >= p.QT) continue;
                const int t = slot * p.QT + col, j = pos % V;
                a = gn_merge(a, GnPart{(float)(lc[t] * step), lm[j * kGnT + t], l2[j * kGnT + t]});
            }
            if (p.owns_tail(g)) {
                const int tail = (g.P - (int)(p.end0 / g.C)) * g.D;   // rows are whole pixels
                for (int e = lane; e < tail; e += K) {
                    const long at = p.end0 + (long)(e / g.D) * g.C + gr * g.D + e % g.D;
                    a = gn_merge(a, GnPart{1.f, to_f32<T>(xs[at]), 0.f});
                }
            }
        }
        a = gn_merge_team(a, K);
        if (gr < g.G && lane == 0) {
            out[gr] = a.n;
            out[g.G + gr] = a.mean;
            out[2 * g.G + gr] = a.m2;
        }
    }
}

// (mean, 1/sqrt(var + eps)) of group gr of sample n from its partials; every lane of the team ends with them
__device__ __forceinline__ void gn_fold(const float* __restrict__ ws, const GnGeom& g, int n, int gr, int K, float eps,
                                        float& mean, float& rstd) {
    GnPart a{0.f, 0.f, 0.f};
    const int parts = g.S * g.tiles;
    if (gr < g.G) {
        const float* w = ws + (long)n * parts * 3 * g.G + gr;
#pragma unroll 4
        for (int s = threadIdx.x & (K - 1); s < parts; s += K) {
            const float* r = w + (long)s * 3 * g.G;
            a = gn_merge(a, GnPart{r[0], r[g.G], r[2 * g.G]});
        }
    }
    a = gn_merge_team(a, K);
    mean = a.mean;
    rstd = 1.f / sqrtf(a.m2 / a.n + eps);
}

// many partials and groups: folded once by a launch of its own.  grid (N, groups / teams)
__global__ __launch_bounds__(kGnT) void gn_fold_kernel(const float* __restrict__ ws, float* __restrict__ stats, float eps,
                                                       const GnGeom g, int K) {
    const int gr = blockIdx.y * (kGnT / K) + threadIdx.x / K;
    float mean, rstd;
    gn_fold(ws, g, blockIdx.x, gr, K, eps, mean, rstd);
    if (gr < g.G && (threadIdx.x & (K - 1)) == 0) {
        stats[((long)blockIdx.x * g.G + gr) * 2] = mean;
        stats[((long)blockIdx.x * g.G + gr) * 2 + 1] = rstd;
    }
}

// table[2 gr], table[2 gr + 1]: mean and rstd of every group of sample n, in shared memory; ws: folded here (and left in
// stats by the sample's first block), or NULL: read from stats
__device__ __forceinline__ void gn_table(float* table, const float* __restrict__ ws, float* __restrict__ stats, float eps,
                                         const GnGeom& g, int n, bool first) {
    if (ws) {
        const int K = gn_team_lanes(g.G), teams = kGnT / K;
        for (int gr = threadIdx.x / K; gr < (g.G + teams - 1) / teams * teams; gr += teams) {
            float mean, rstd;
            gn_fold(ws, g, n, gr, K, eps, mean, rstd);
            if (gr < g.G && (threadIdx.x & (K - 1)) == 0) {
                table[2 * gr] = mean;
                table[2 * gr + 1] = rstd;
                if (first) {
                    stats[((long)n * g.G + gr) * 2] = mean;
                    stats[((long)n * g.G + gr) * 2 + 1] = rstd;
                }
            }
        }
    } else {
        for (int i = threadIdx.x; i < 2 * g.G; i += kGnT) table[i] = stats[(long)n * g.G * 2 + i];
    }
    __syncthreads();
}

// ------------------------------------------------------------------ forward, second launch
// A slice is walked from its end: what the first launch read last is the likeliest to be in a cache still.
template <typename T, int V>
__global__ __launch_bounds__(kGnT) void gn_apply_kernel(const T* x, const float* __restrict__ ws, float* __restrict__ stats,
                                                        float eps, const float* __restrict__ scale,
                                                        const float* __restrict__ shift, const T* residual, T* y, int act,
                                                        const GnGeom g) {
    constexpr int kU = 4;
    extern __shared__ float table[];
    const GnPlace p(g);
    gn_table(table, ws, stats, eps, g, p.n, p.s == 0 && p.c0 == 0);
    const T* xs = x + p.base;
    const T* rs = residual ? residual + p.base : nullptr;
    T* ys = y + p.base;
    gn_with_act(act, [&](auto A) {
        constexpr int kA = decltype(A)::value;
        if (p.on) {
            float mean[V], a[V], b[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const int c = (p.col * V + j) % g.C, gr = c / g.D;
                mean[j] = table[2 * gr];
                a[j] = scale[c] * table[2 * gr + 1];
                b[j] = shift[c];
            }
            const long off = (long)p.col * V;
            for (int row = p.r1 - 1 - p.slot; row >= p.r0; row -= p.slots * kU) {
                float v[kU][V], r[kU][V];
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    const int rw = row - u * p.slots;
                    if (rw < p.r0) continue;
                    gn_load<T, V>(xs + off + (long)rw * g.L, v[u]);
                    if (rs) gn_load<T, V>(rs + off + (long)rw * g.L, r[u]);
                }
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    const int rw = row - u * p.slots;
                    if (rw < p.r0) continue;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        v[u][j] = gn_act<kA>((v[u][j] - mean[j]) * a[j] + b[j]);
                        if (rs) v[u][j] += r[u][j];
                    }
                    gn_store<T, V>(ys + off + (long)rw * g.L, v[u]);
                }
            }
        }
        if (p.owns_tail(g)) {
            const int tail = (int)((long)g.P * g.C - p.end0);
            for (int e = threadIdx.x; e < tail; e += kGnT) {
                const long at = p.end0 + e;
                const int c = e % g.C, gr = c / g.D;
                float v = gn_act<kA>((to_f32<T>(xs[at]) - table[2 * gr]) * (scale[c] * table[2 * gr + 1]) + shift[c]);
                if (rs) v += to_f32<T>(rs[at]);
                ys[at] = from_f32<T>(v);
            }
        }
    });
}

// ------------------------------------------------------------------ backward, first launch
// rows[n][slice * tiles + tile][2][C]: the block's sums of g and of g * xhat per channel (the parameter gradients' parts);
// grows[...][2][G]: the same times scale, per group.  A thread's sums are kept in two levels (kB values, then the rest).
template <typename T, int V>
__global__ __launch_bounds__(kGnT) void gn_bwd_sums_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                           const float* __restrict__ stats, const float* __restrict__ scale,
                                                           const float* __restrict__ shift, float* __restrict__ rows,
                                                           float* __restrict__ grows, int act, const GnGeom g) {
    constexpr int kB = 4;
    extern __shared__ float sh[];   // [V][kGnT] sums of g, [V][kGnT] of g * xhat, [2][C] the block's sums per channel
    const GnPlace p(g);
    const T* xs = x + p.base;
    const T* ds = dy + p.base;
    const float* st = stats + (long)p.n * g.G * 2;
    float* l1 = sh;
    float* l2 = sh + V * kGnT;
    float* ch = sh + 2 * V * kGnT;
    gn_with_act(act, [&](auto A) {
        constexpr int kA = decltype(A)::value;
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
        if (p.on) {
            float mean[V], rstd[V], a[V], b[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const int c = (p.col * V + j) % g.C, gr = c / g.D;
                mean[j] = st[2 * gr];
                rstd[j] = st[2 * gr + 1];
                a[j] = scale[c] * rstd[j];
                b[j] = shift[c];
            }
            const long off = (long)p.col * V;
            for (int row = p.r0 + p.slot; row < p.r1; row += p.slots * kB) {
                float v[kB][V], d[kB][V];
#pragma unroll
                for (int u = 0; u < kB; u++) {
                    const int rw = row + u * p.slots;
                    if (rw >= p.r1) continue;
                    gn_load<T, V>(xs + off + (long)rw * g.L, v[u]);
                    gn_load<T, V>(ds + off + (long)rw * g.L, d[u]);
                }
#pragma unroll
                for (int j = 0; j < V; j++) {
                    float t1 = 0.f, t2 = 0.f;
#pragma unroll
                    for (int u = 0; u < kB; u++) {
                        if (row + u * p.slots >= p.r1) continue;
                        const float xm = v[u][j] - mean[j];
                        const float gv = d[u][j] * gn_act_grad<kA>(xm * a[j] + b[j]);
                        t1 += gv;
                        t2 += gv * xm;
                    }
                    s1[j] += t1;
                    s2[j] += t2 * rstd[j];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
            l1[j * kGnT + threadIdx.x] = s1[j];
            l2[j * kGnT + threadIdx.x] = s2[j];
        }
        __syncthreads();
        // teams of lanes: one channel each
        const int K = gn_team_lanes(g.C), teams = kGnT / K, lane = threadIdx.x & (K - 1);
        const int reps = g.L / g.C, total = reps * p.slots;
        for (int c = threadIdx.x / K; c < (g.C + teams - 1) / teams * teams; c += teams) {
            float t1 = 0.f, t2 = 0.f;
            if (c < g.C) {
                for (int e = lane; e < total; e += K) {
                    const int slot = e / reps, pos = c + (e - slot * reps) * g.C, col = pos / V - p.c0;
                    if (col < 0 || col >= p.QT) continue;
                    const int t = slot * p.QT + col, j = pos % V;
                    t1 += l1[j * kGnT + t];
                    t2 += l2[j * kGnT + t];
                }
                if (p.owns_tail(g)) {
                    const int pixels = g.P - (int)(p.end0 / g.C), gr = c / g.D;
                    for (int e = lane; e < pixels; e += K) {
                        const long at = p.end0 + (long)e * g.C + c;
                        const float xm = to_f32<T>(xs[at]) - st[2 * gr];
                        const float gv = to_f32<T>(ds[at]) * gn_act_grad<kA>(xm * (scale[c] * st[2 * gr + 1]) + shift[c]);
                        t1 += gv;
                        t2 += gv * (xm * st[2 * gr + 1]);
                    }
                }
            }
            for (int o = 1; o < K; o <<= 1) {
                t1 += __shfl_xor(t1, o, 64);
                t2 += __shfl_xor(t2, o, 64);
            }
            if (c < g.C && lane == 0) {
                ch[c] = t1;
                ch[g.C + c] = t2;
            }
        }
        __syncthreads();
    });
    const long part = ((long)p.n * g.S + p.s) * g.tiles + p.c0 / g.QT;
    for (int i = threadIdx.x; i < 2 * g.C; i += kGnT) rows[part * 2 * g.C + i] = ch[i];
    const int K = gn_team_lanes(g.G), teams = kGnT / K, lane = threadIdx.x & (K - 1);
    for (int gr = threadIdx.x / K; gr < (g.G + teams - 1) / teams * teams; gr += teams) {
        float t1 = 0.f, t2 = 0.f;
        if (gr < g.G) {
            for (int c = gr * g.D + lane; c < (gr + 1) * g.D; c += K) {
                t1 += scale[c] * ch[c];
                t2 += scale[c] * ch[g.C + c];
            }
        }
        for (int o = 1; o < K; o <<= 1) {
            t1 += __shfl_xor(t1, o, 64);
            t2 += __shfl_xor(t2, o, 64);
        }
        if (gr < g.G && lane == 0) {
            grows[part * 2 * g.G + gr] = t1;
            grows[part * 2 * g.G + g.G + gr] = t2;
        }
    }
}

// m[2 gr], m[2 gr + 1] = m1, m2 of group gr of sample n; every lane of the team ends with them
__device__ __forceinline__ void gn_fold_sums(const float* __restrict__ grows, const GnGeom& g, int n, int gr, int K, float& m1,
                                             float& m2) {
    const int parts = g.S * g.tiles;
    m1 = m2 = 0.f;
    if (gr < g.G) {
        const float* w = grows + (long)n * parts * 2 * g.G + gr;
#pragma unroll 4
        for (int s = threadIdx.x & (K - 1); s < parts; s += K) {
            m1 += w[(long)s * 2 * g.G];
            m2 += w[(long)s * 2 * g.G + g.G];
        }
    }
    for (int o = 1; o < K; o <<= 1) {
        m1 += __shfl_xor(m1, o, 64);
        m2 += __shfl_xor(m2, o, 64);
    }
    const float M = (float)g.P * (float)g.D;
    m1 /= M;
    m2 /= M;
}

__global__ __launch_bounds__(kGnT) void gn_fold_sums_kernel(const float* __restrict__ grows, float* __restrict__ m,
                                                            const GnGeom g, int K) {
    const int gr = blockIdx.y * (kGnT / K) + threadIdx.x / K;
    float m1, m2;
    gn_fold_sums(grows, g, blockIdx.x, gr, K, m1, m2);
    if (gr < g.G && (threadIdx.x & (K - 1)) == 0) {
        m[((long)blockIdx.x * g.G + gr) * 2] = m1;
        m[((long)blockIdx.x * g.G + gr) * 2 + 1] = m2;
    }
}

// dshift / dscale from the partial rows: outputs o of [0, 2C), 64 a block, eight row groups each, in one fixed order
__device__ __forceinline__ void gn_param_grads(const float* __restrict__ rows, int nrows, float* __restrict__ dscale,
                                               float* __restrict__ dshift, int accumulate, int C, int block, float* tmp) {
    const int o = block * 64 + (threadIdx.x & 63), rg = threadIdx.x >> 6;
    float s = 0.f;
    if (o < 2 * C) {
#pragma unroll 8
        for (int i = rg; i < nrows; i += kGnT / 64) s += rows[(long)i * 2 * C + o];
    }
    tmp[threadIdx.x] = s;
    __syncthreads();
    if (rg == 0 && o < 2 * C) {
        s = 0.f;
        for (int k = 0; k < kGnT / 64; k++) s += tmp[k * 64 + threadIdx.x];
        float* dst = o < C ? dshift + o : dscale + (o - C);
        *dst = accumulate ? *dst + s : s;
    }
}

// ------------------------------------------------------------------ backward, second launch
// The last blocks fold the parameter gradients, the others write dx.
template <typename T, int V>
__global__ __launch_bounds__(kGnT) void gn_bwd_apply_kernel(const T* x, const T* dy, const float* __restrict__ stats,
                                                            const float* __restrict__ scale, const float* __restrict__ shift,
                                                            const float* __restrict__ grows, const float* __restrict__ msums,
                                                            const float* __restrict__ rows, T* dx, float* dscale, float* dshift,
                                                            int accumulate, int act, const GnGeom g) {
    constexpr int kU = 2;
    extern __shared__ float table[];   // [2G] m1, m2 (512 floats at least)
    const int main_blocks = g.N * g.S * g.tiles;
    if ((int)blockIdx.x >= main_blocks) {
        gn_param_grads(rows, main_blocks, dscale, dshift, accumulate, g.C, blockIdx.x - main_blocks, table);
        return;
    }
    const GnPlace p(g);
    const T* xs = x + p.base;
    const T* ds = dy + p.base;
    T* os = dx + p.base;
    const float* st = stats + (long)p.n * g.G * 2;
    if (msums) {
        for (int i = threadIdx.x; i < 2 * g.G; i += kGnT) table[i] = msums[(long)p.n * g.G * 2 + i];
    } else {
        const int K = gn_team_lanes(g.G), teams = kGnT / K;
        for (int gr = threadIdx.x / K; gr < (g.G + teams - 1) / teams * teams; gr += teams) {
            float m1, m2;
            gn_fold_sums(grows, g, p.n, gr, K, m1, m2);
            if (gr < g.G && (threadIdx.x & (K - 1)) == 0) {
                table[2 * gr] = m1;
                table[2 * gr + 1] = m2;
            }
        }
    }
    __syncthreads();
    gn_with_act(act, [&](auto A) {
        constexpr int kA = decltype(A)::value;
        if (p.on) {
            // dx = a g - k1 - (x - mean) k2 with a = scale rstd, k1 = rstd m1, k2 = rstd^2 m2
            float mean[V], a[V], b[V], k1[V], k2[V];
#pragma unroll
            for (int j = 0; j < V; j++) {
                const int c = (p.col * V + j) % g.C, gr = c / g.D;
                const float rstd = st[2 * gr + 1];
                mean[j] = st[2 * gr];
                a[j] = scale[c] * rstd;
                b[j] = shift[c];
                k1[j] = rstd * table[2 * gr];
                k2[j] = rstd * rstd * table[2 * gr + 1];
            }
            const long off = (long)p.col * V;
            for (int row = p.r1 - 1 - p.slot; row >= p.r0; row -= p.slots * kU) {
                float v[kU][V], d[kU][V];
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    const int rw = row - u * p.slots;
                    if (rw < p.r0) continue;
                    gn_load<T, V>(xs + off + (long)rw * g.L, v[u]);
                    gn_load<T, V>(ds + off + (long)rw * g.L, d[u]);
                }
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    const int rw = row - u * p.slots;
                    if (rw < p.r0) continue;
#pragma unroll
                    for (int j = 0; j < V; j++) {
                        const float xm = v[u][j] - mean[j];
                        v[u][j] = d[u][j] * gn_act_grad<kA>(xm * a[j] + b[j]) * a[j] - k1[j] - xm * k2[j];
                    }
                    gn_store<T, V>(os + off + (long)rw * g.L, v[u]);
                }
            }
        }
        if (p.owns_tail(g)) {
            const int tail = (int)((long)g.P * g.C - p.end0);
            for (int e = threadIdx.x; e < tail; e += kGnT) {
                const long at = p.end0 + e;
                const int c = e % g.C, gr = c / g.D;
                const float rstd = st[2 * gr + 1], a = scale[c] * rstd, xm = to_f32<T>(xs[at]) - st[2 * gr];
                os[at] = from_f32<T>(to_f32<T>(ds[at]) * gn_act_grad<kA>(xm * a + shift[c]) * a - rstd * table[2 * gr] -
                                     xm * (rstd * rstd * table[2 * gr + 1]));
            }
        }
    });
}

__global__ __launch_bounds__(256) void gn_zero_kernel(float* a, float* b, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) a[i] = b[i] = 0.f;
}

// ------------------------------------------------------------------ launches
static int gcd_int(int a, int b) { return b ? gcd_int(b, a % b) : a; }

static GnGeom gn_geom(int n, int P, int c, int groups, int V) {
    GnGeom g;
    g.N = n; g.P = P; g.C = c; g.G = groups; g.D = c / groups;
    g.L = c / gcd_int(c, V) * V;
    g.Q = g.L / V;
    g.QT = g.Q < kGnT ? g.Q : kGnT;
    g.tiles = ceil_div(g.Q, g.QT);
    const int slots = kGnT / g.QT;
    g.R = (int)((long)P * c / g.L);
    // four rows a thread at least; a sample is cut the same way whatever its batch
    int S = ceil_div(kGnSlices, g.tiles);
    if (S > g.R / (slots * 4)) S = g.R / (slots * 4);
    if (S < 1) S = 1;
    g.rows = ceil_div(g.R, S);
    if (g.rows < 1) g.rows = 1;
    g.S = ceil_div(g.R, g.rows);
    if (g.S < 1) g.S = 1;
    return g;
}

static bool gn_folds_itself(const GnGeom& g) { return (long)g.S * g.tiles * g.G <= kGnFold; }

// enough for either direction
long gn_ws_floats(int n, int h, int w, int c, int groups, int dtype) {
    const GnGeom g = gn_geom(n, h * w, c, groups, dtype == STMI_BF16 ? 8 : 4);
    const long parts = (long)n * g.S * g.tiles;
    return parts * 2 * c + parts * 3 * groups + (long)n * 2 * groups;
}

template <typename T, int V>
static int gn_fwd_t(const T* x, float* ws, float* stats, float eps, const float* scale, const float* shift, const T* residual,
                    T* y, int act, int n, int P, int c, int groups, hipStream_t s) {
    const GnGeom g = gn_geom(n, P, c, groups, V);
    const dim3 grid((unsigned)(g.N * g.S * g.tiles));
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), grid, dim3(kGnT), (2 * V + 1) * kGnT * sizeof(float), s, x, ws, g);
    STMI_LAUNCH_CHECK("gn_stats_kernel");
    const float* fold = ws;
    if (!gn_folds_itself(g)) {
        hipLaunchKernelGGL(gn_fold_kernel, dim3(g.N, ceil_div(g.G, kGnT / 64)), dim3(kGnT), 0, s, (const float*)ws, stats, eps, g, 64);
        STMI_LAUNCH_CHECK("gn_fold_kernel");
        fold = nullptr;
    }
    hipLaunchKernelGGL((gn_apply_kernel<T, V>), grid, dim3(kGnT), 2 * g.G * sizeof(float), s, x, fold, stats, eps, scale, shift,
                       residual, y, act, g);
    STMI_LAUNCH_CHECK("gn_apply_kernel");
    return STMI_OK;
}

int gn_fwd_impl(const void* x, float* ws, float* stats, float eps, const float* scale, const float* shift,
                const void* residual, void* y, int act, int n, int h, int w, int c, int groups, int dtype, hipStream_t s) {
    if (dtype == STMI_BF16)
        return gn_fwd_t<bf16_t, 8>((const bf16_t*)x, ws, stats, eps, scale, shift, (const bf16_t*)residual, (bf16_t*)y, act, n, h * w, c, groups, s);
    return gn_fwd_t<float, 4>((const float*)x, ws, stats, eps, scale, shift, (const float*)residual, (float*)y, act, n, h * w, c, groups, s);
}

template <typename T, int V>
static int gn_bwd_t(const T* x, const T* dy, const float* stats, const float* scale, const float* shift, T* dx, float* dscale,
                    float* dshift, int accumulate, float* ws, int act, int n, int P, int c, int groups, hipStream_t s) {
    const GnGeom g = gn_geom(n, P, c, groups, V);
    const long parts = (long)g.N * g.S * g.tiles;
    float* rows = ws;
    float* grows = rows + parts * 2 * g.C;
    float* msums = grows + parts * 2 * g.G;
    const int lds = (2 * V * kGnT + 2 * g.C) * (int)sizeof(float);
    STMI_DYN_LDS((gn_bwd_sums_kernel<T, V>), (2 * V * kGnT + 2 * STMI_GN_MAX_C) * (int)sizeof(float), "gn_bwd_sums_kernel");
    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V>), dim3((unsigned)parts), dim3(kGnT), lds, s, x, dy, stats, scale, shift, rows, grows, act, g);
    STMI_LAUNCH_CHECK("gn_bwd_sums_kernel");
    const float* m = nullptr;
    if (!gn_folds_itself(g)) {
        hipLaunchKernelGGL(gn_fold_sums_kernel, dim3(g.N, ceil_div(g.G, kGnT / 64)), dim3(kGnT), 0, s, (const float*)grows, msums, g, 64);
        STMI_LAUNCH_CHECK("gn_fold_sums_kernel");
        m = msums;
    }
    const int pblocks = dscale ? ceil_div(2L * g.C, 64) : 0;
    const int table = 2 * g.G > kGnT ? 2 * g.G : kGnT;
    hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V>), dim3((unsigned)(parts + pblocks)), dim3(kGnT), table * sizeof(float), s, x, dy,
                       stats, scale, shift, (const float*)grows, m, (const float*)rows, dx, dscale, dshift, accumulate, act, g);
    STMI_LAUNCH_CHECK("gn_bwd_apply_kernel");
    return STMI_OK;
}

int gn_bwd_impl(const void* x, const void* dy, const float* stats, const float* scale, const float* shift, void* dx,
                float* dscale, float* dshift, int accumulate, float* ws, int act, int n, int h, int w, int c, int groups,
                int dtype, hipStream_t s) {
    if (n == 0) {
        if (dscale && !accumulate) {
            hipLaunchKernelGGL(gn_zero_kernel, dim3(ceil_div(c, 256)), dim3(256), 0, s, dscale, dshift, c);
            STMI_LAUNCH_CHECK("gn_zero_kernel");
        }
        return STMI_OK;
    }
    if (dtype == STMI_BF16)
        return gn_bwd_t<bf16_t, 8>((const bf16_t*)x, (const bf16_t*)dy, stats, scale, shift, (bf16_t*)dx, dscale, dshift, accumulate,
                                   ws, act, n, h * w, c, groups, s);
    return gn_bwd_t<float, 4>((const float*)x, (const float*)dy, stats, scale, shift, (float*)dx, dscale, dshift, accumulate, ws, act,
                              n, h * w, c, groups, s);
}

}  // namespace stmi
