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
// blocks of the second launch fold the partials of their sample and stream the tensor once more.  Samples whose groups fit
// the registers of a block take one launch (at the end of the file).
//
// Layout of the work: a sample is a flat run of P * C elements, cut into rows of L = lcm(C, V) elements (V: the elements
// of a 16-byte access), so that a thread that owns one 16-byte column of a row sees the SAME V channels in every row
// whatever C is.  What does not fill a row behind the last one is the tail; it belongs to the last slice.  The cut depends
// on the sample's own size alone, and accesses need only the elements' alignment (global memory takes 16-byte accesses at
// any address): a sample's bits depend neither on its batch nor on its place.
// A mean is formed first and deviations from it are summed then, within a batch of loads, over a block's threads and over
// the slices: no cancellation however large the mean is next to the deviation.  Means are themselves sums of deviations, from
// a value of the group, and every term enters a sum with its weight 1 / M: equal values give their own value and no deviation,
// and nothing leaves fp32 unless a deviation's square does.  Sums are fp32, no atomics: bit-reproducible.
// What the launches of small tensors cost is instructions, not bytes: divisions by the geometry's numbers are done by the
// host (gn_div), constants of the channels come from a table in shared memory that a block makes once, reductions over
// lanes use DPP.
#include "common.hpp"

#include <type_traits>

namespace stmi {

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;

constexpr int kGnT = 512;        // threads of a block
constexpr int kGnSlices = 512;   // most slices of a sample (64 lanes of kGnFoldLane fold them)
constexpr int kGnFoldLane = 8;   // partials a lane folds
constexpr int kGnUnitFwd = 1024, kGnUnitBwd = 512;   // most threads of a unit's block

struct GnGeom {
    int N, P, C, G, D;
    int L, Q, R;         // elements and V-wide columns of a row, whole rows of a sample
    int QT, tiles;       // columns a block owns, blocks side by side in a row
    int S, rows;         // slices of a sample, rows of a slice
    int S2, rows2;       // the same for the second launch
    int slots;           // rows a block walks at once (one tile)
    int parts;           // S * tiles: partial results of a sample, blocks of a sample
    int lgG, lgC;        // log2 of the lanes that reduce one group, one channel
    int U;               // gcd(V, D): neighbouring channels of a column that are always of one group
    int tail;            // elements behind the rows
    bool over_slots;     // lanes of a group's team run over the slots, not over the entries of one
    unsigned rC, rD, rQT, rUnits;   // gn_div's reciprocals
    float rM;                // 1 / M
    float share, share_last; // of a group's values: in a slice, in the last slice with the tail (one tile)
};

// x / d for x < 2^16, d <= 2^16 with r = ceil(2^32 / d): r d exceeds 2^32 by less than d, so x r / 2^32 exceeds x / d by
// less than 2^-16 <= 1 / d
__device__ __forceinline__ int gn_div(int x, unsigned r) { return r ? (int)__umulhi((unsigned)x, r) : x; }   // r == 0: d == 1

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

// ------------------------------------------------------------------ lanes
template <int kCtrl>
__device__ __forceinline__ float gn_dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kCtrl, 0xf, 0xf, true));
}

// the sum of an exchange's two results (copied first: this compiler's bit cast of a vector's element reads element 0)
__device__ __forceinline__ float gn_add_pair(u32x2 r) {
    const unsigned lo = r[0], hi = r[1];
    return __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
}

// sum over a team of 2^lg neighbouring lanes, the same bits in every lane of it: partners at distance 1, 2 (within a
// quad), 4, 8 (mirrored: the lanes of the other half hold equal values), 16, 32 (rows exchanged)
__device__ __forceinline__ float gn_team_sum(float v, int lg) {
    if (lg > 0) v += gn_dpp<0xB1>(v);
    if (lg > 1) v += gn_dpp<0x4E>(v);
    if (lg > 2) v += gn_dpp<0x141>(v);
    if (lg > 3) v += gn_dpp<0x140>(v);
    if (lg > 4) {
        const unsigned b = __builtin_bit_cast(unsigned, v);
        v = gn_add_pair(__builtin_amdgcn_permlane16_swap(b, b, false, false));
    }
    if (lg > 5) {
        const unsigned b = __builtin_bit_cast(unsigned, v);
        v = gn_add_pair(__builtin_amdgcn_permlane32_swap(b, b, false, false));
    }
    return v;
}

// 1 / sqrt(v): the hardware's value (one unit in its last place) and one Newton step
__device__ __forceinline__ float gn_rsqrt(float v) {
    const float r = __builtin_amdgcn_rsqf(v);
    return r + 0.5f * r * (1.f - v * r * r);
}

// ------------------------------------------------------------------ memory
// 16 bytes at an element's alignment; the address is a block's (scalar) and a thread's offset in bytes; kNt: not kept in
// the caches
template <bool kNt>
__device__ __forceinline__ u32x4 gn_load(const void* p, unsigned own) {
    typedef u32x4 __attribute__((aligned(2))) loose;
    const loose* q = reinterpret_cast<const loose*>(static_cast<const char*>(p) + own);
    if constexpr (kNt) return __builtin_nontemporal_load(q);
    return *q;
}

template <bool kNt, typename T, int V>
__device__ __forceinline__ void gn_store(void* p, unsigned own, const float (&in)[V]) {
    typedef u32x4 __attribute__((aligned(2))) loose;
    loose* q = reinterpret_cast<loose*>(static_cast<char*>(p) + own);
    T e[V];
#pragma unroll
    for (int i = 0; i < V; i++) e[i] = from_f32<T>(in[i]);
    u32x4 raw;
    __builtin_memcpy(&raw, e, 16);
    if constexpr (kNt) __builtin_nontemporal_store(raw, q);
    else *q = raw;
}

template <typename T, int V>
__device__ __forceinline__ void gn_unpack(const u32x4& raw, float (&out)[V]) {
    T e[V];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int i = 0; i < V; i++) out[i] = to_f32<T>(e[i]);
}

// ------------------------------------------------------------------ places
// Blocks run over the parts of a sample first: neighbouring blocks read neighbouring memory.
constexpr int kGnGridY = 32768;
__device__ __forceinline__ int gn_sample() { return blockIdx.z * kGnGridY + blockIdx.y; }
static dim3 gn_grid(int parts, int n) {
    return dim3((unsigned)parts, (unsigned)(n < kGnGridY ? n : kGnGridY), (unsigned)((n + kGnGridY - 1) / kGnGridY));
}

// a block's sample, slice and column tile, and what the calling thread owns of the tile.  kTiled: a row has more columns
// than a block has threads
template <bool kTiled>
struct GnPlace {
    int n, s, tile, c0, QT, slots, col, slot, rows;
    long first;        // the slice's first element
    long end0;         // the tail's first element
    unsigned own;      // the thread's first element in the slice
    bool last;         // the last slice: the tail is its
    __device__ __forceinline__ GnPlace(const GnGeom& g, int V, int S, int slice_rows) {
        n = gn_sample();
        s = blockIdx.x;
        tile = c0 = 0;
        QT = g.QT;
        slots = g.slots;
        if constexpr (kTiled) {
            tile = s % g.tiles;
            s /= g.tiles;
            c0 = tile * g.QT;
            QT = min(g.QT, g.Q - c0);
            slots = kGnT / QT;
            slot = threadIdx.x / QT;
        } else {
            slot = gn_div(threadIdx.x, g.rQT);
        }
        col = c0 + threadIdx.x - slot * QT;
        const int r0 = min(s * slice_rows, g.R);
        rows = min(slice_rows, g.R - r0);
        last = s == S - 1 && tile == 0;
        const long base = (long)n * g.P * g.C;
        first = base + (long)r0 * g.L;
        end0 = base + (long)g.R * g.L;
        own = slot * g.L + col * V;
    }
    __device__ __forceinline__ bool on() const { return slot < slots; }
    __device__ __forceinline__ long part(const GnGeom& g) const { return (long)n * g.parts + blockIdx.x; }
};

// the entries of a per-channel table in shared memory that belong to a column
template <int V>
__device__ __forceinline__ void gn_column(const float* tab, const GnGeom& g, int col, float (&out)[V]) {
    if (g.L == g.C) {   // whole columns in a pixel: 16-byte reads
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const f32x4 q = *reinterpret_cast<const f32x4*>(tab + col * V + j);
#pragma unroll
            for (int i = 0; i < 4; i++) out[j + i] = q[i];
        }
    } else {
        int c = col * V - gn_div(col * V, g.rC) * g.C;
#pragma unroll
        for (int j = 0; j < V; j++) {
            out[j] = tab[c];
            c = c + 1 == g.C ? 0 : c + 1;
        }
    }
}

// ------------------------------------------------------------------ forward, first launch
// ws[n][slice * tiles + tile][G][2]: (mean, sum of squared deviations / M) of the block's values of each group; their number
// follows from the cut (gn_share).
// A thread keeps a mean and a sum of squared deviations per channel of its column: a batch of kB values is summed as
// deviations from the mean so far (from the first value in the first batch), then mean += s1 / n, m2 += s2 - s1^2 / n
// with n the count behind the batch.  That shift is a value of the plane or a mean of some, so s2 exceeds the sum it
// stands for by no more than the batch's share of the total, and the short batches keep partial sums short.
// Bound by reading: 16 x 1080 x 1920 x 32 bf16 (2.1 GB) in 312 us, 6.8 TB/s; 4 x 256 x 256 x 32 (17 MB) in 7.0 us, 5.4 where the
// tensor is in the last-level cache: 256 blocks, a block's loads, reductions and partial result one after the other.
template <typename T, int V, bool kNt, bool kTiled>
__global__ __launch_bounds__(kGnT, 4) void gn_stats_kernel(const T* __restrict__ x, float2* __restrict__ ws, const GnGeom g) {
    constexpr int kB = 8;
    extern __shared__ float sh[];   // [V][kGnT] means, [V][kGnT] sums of squares, [kGnT] counts
    const GnPlace<kTiled> p(g, V, g.S, g.rows);
    if (p.n >= g.N) return;
    // the group's first value in the sample, from which the block's means deviate: on its way during the sums
    const T* x0 = x + (long)p.n * g.P * g.C;
    const float first = to_f32<T>(x0[min((int)threadIdx.x >> g.lgG, g.G - 1) * g.D]);
    float mean[V], m2[V];   // m2: divided by M
#pragma unroll
    for (int j = 0; j < V; j++) mean[j] = m2[j] = 0.f;
    int cnt = 0;
    if (p.on()) {
        const T* xb = x + p.first;
        const unsigned own = p.own * (unsigned)sizeof(T);
        const int step = p.slots * g.L, batch = kB * p.slots;
        auto flush = [&](const float (&s1)[V], const float (&s2)[V]) {
            const float rn = __builtin_amdgcn_rcpf((float)cnt);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float e = s1[j] * rn;
                mean[j] += e;
                m2[j] += (s2[j] - s1[j] * e) * g.rM;
            }
        };
        auto add = [&](const u32x4& raw, float (&s1)[V], float (&s2)[V]) {
            float v[V];
            gn_unpack<T, V>(raw, v);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = v[j] - mean[j];
                s1[j] += d;
                s2[j] += d * d;
            }
        };
        int left = p.rows;
        for (; left >= batch; left -= batch, xb += kB * (long)step) {
            u32x4 raw[kB];
#pragma unroll
            for (int u = 0; u < kB; u++) raw[u] = gn_load<kNt>(xb + u * (long)step, own);
            if (cnt == 0) gn_unpack<T, V>(raw[0], mean);
            float s1[V], s2[V];
#pragma unroll
            for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
#pragma unroll
            for (int u = 0; u < kB; u++) add(raw[u], s1, s2);
            cnt += kB;
            flush(s1, s2);
        }
        if (p.slot < left) {   // the last, shorter batch
            u32x4 raw[kB];
            float s1[V], s2[V];
#pragma unroll
            for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
#pragma unroll
            for (int u = 0; u < kB; u++)
                if (p.slot < left - u * p.slots) raw[u] = gn_load<kNt>(xb + u * (long)step, own);
            if (cnt == 0) gn_unpack<T, V>(raw[0], mean);
#pragma unroll
            for (int u = 0; u < kB; u++) {
                if (p.slot < left - u * p.slots) {
                    add(raw[u], s1, s2);
                    cnt++;
                }
            }
            flush(s1, s2);
        }
    }
    // neighbouring channels of one group are merged in the thread: pairs of equal counts
#pragma unroll
    for (int w = 1; w < V; w <<= 1) {
        if (w < g.U) {
#pragma unroll
            for (int j = 0; j < V; j += 2 * w) {
                const float d = mean[j + w] - mean[j];
                mean[j] += 0.5f * d;
                m2[j] += m2[j + w] + d * d * (0.5f * (float)(cnt * w) * g.rM);
            }
        }
    }
    float* lm = sh;
    float* l2 = sh + V * kGnT;
    float* lc = sh + 2 * V * kGnT;
#pragma unroll
    for (int j = 0; j < V; j++) {
        if (j & (g.U - 1)) continue;
        lm[j * kGnT + threadIdx.x] = mean[j];
        l2[j * kGnT + threadIdx.x] = m2[j];
    }
    lc[threadIdx.x] = (float)(cnt * g.U) * g.rM;   // the entry's share of the group
    __syncthreads();
    // a team of lanes adds the entries of one group up, the means first, then the deviations from their mean
    const int K = 1 << g.lgG, lane = threadIdx.x & (K - 1);
    const int units = g.D / g.U, entries = units * (g.L / g.C);
    const int en0 = g.over_slots ? 0 : lane, enstep = g.over_slots ? 1 : K, sl0 = g.over_slots ? lane : 0, slstep = g.over_slots ? K : 1;
    float2* out = ws + p.part(g) * g.G;
    for (int gr0 = 0; gr0 < g.G; gr0 += kGnT >> g.lgG) {
        const int gr = gr0 + (threadIdx.x >> g.lgG);
        const bool live = gr < g.G;
        const float from = gr0 == 0 ? first : live ? to_f32<T>(x0[gr * g.D]) : 0.f;
        // f(share, mean, sum of squared deviations / M) of every entry of the group
        auto each = [&](auto f) {
            for (int en = en0; en < entries; en += enstep) {
                const int rep = gn_div(en, g.rUnits);
                const int pos = gr * g.D + (en - rep * units) * g.U + rep * g.C, col = pos / V - p.c0, j = pos % V;
                if (kTiled && (col < 0 || col >= p.QT)) continue;
                for (int slot = sl0; slot < p.slots; slot += slstep) {
                    const int t = slot * p.QT + col;
                    f(lc[t], lm[j * kGnT + t], l2[j * kGnT + t]);
                }
            }
            if (g.tail && p.last) {
                for (int e = lane; e < g.tail / g.C * g.D; e += K)
                    f(g.rM, to_f32<T>(x[p.end0 + e / g.D * g.C + gr * g.D + e % g.D]), 0.f);
            }
        };
        float n = 0.f, s1 = 0.f, s2 = 0.f;
        if (live) each([&](float c, float m, float) { n += c; s1 += c * (m - from); });
        n = gn_team_sum(n, g.lgG);
        s1 = gn_team_sum(s1, g.lgG);
        const float mu = n > 0.f ? from + s1 / n : from;
        if (live) each([&](float c, float m, float q) { const float d = c > 0.f ? m - mu : 0.f; s2 += q + c * d * d; });
        s2 = gn_team_sum(s2, g.lgG);
        if (live && lane == 0) out[gr] = make_float2(mu, s2);
    }
}

// the share of group gr's values that partial i holds (0 behind the last)
template <bool kTiled>
__device__ __forceinline__ float gn_share(const GnGeom& g, int gr, int i) {
    if constexpr (!kTiled) return i < g.S - 1 ? g.share : i == g.S - 1 ? g.share_last : 0.f;
    if (i >= g.parts) return 0.f;
    const int s = i / g.tiles, t = i - s * g.tiles, rows = max(0, min(g.R, (s + 1) * g.rows) - s * g.rows);
    // positions of the row before e that hold a channel of the group
    const int V = g.L / g.Q, e0 = t * g.QT * V, e1 = min(g.Q, (t + 1) * g.QT) * V;
    const int per = e1 / g.C * g.D + min(max(e1 % g.C - gr * g.D, 0), g.D) - e0 / g.C * g.D - min(max(e0 % g.C - gr * g.D, 0), g.D);
    float n = (float)rows * (float)per;
    if (s == g.S - 1 && t == 0) n += (float)(g.tail / g.C) * (float)g.D;
    return n * g.rM;
}

// (mean, 1/sqrt(var + eps)) of group gr of sample n from its partials, NK at most a lane of the team, in two passes: the
// mean first (from the first partial's), then the deviations from it.  Every lane ends with the result.
template <int NK, bool kTiled>
__device__ __forceinline__ void gn_fold_n(const float2* __restrict__ w, const GnGeom& g, int gr, int lg, float eps, float& mean,
                                          float& rstd) {
    const int K = 1 << lg, lane = threadIdx.x & (K - 1);
    float2 r[NK];
#pragma unroll
    for (int k = 0; k < NK; k++) r[k] = w[(unsigned)(min(lane + (k << lg), g.parts - 1) * g.G)];
    const float from = w[0].x;
    float share[NK], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NK; k++) {
        share[k] = gn_share<kTiled>(g, gr, lane + (k << lg));
        s1 += share[k] > 0.f ? share[k] * (r[k].x - from) : 0.f;
    }
    mean = from + gn_team_sum(s1, lg);
#pragma unroll
    for (int k = 0; k < NK; k++) {
        const float d = r[k].x - mean;
        s2 += share[k] > 0.f ? r[k].y + share[k] * d * d : 0.f;
    }
    rstd = gn_rsqrt(gn_team_sum(s2, lg) + eps);
}

template <bool kTiled>
__device__ __forceinline__ void gn_fold(const float2* __restrict__ ws, const GnGeom& g, int n, int gr, int lg, float eps,
                                        float& mean, float& rstd) {
    const float2* w = ws + ((long)n * g.parts * g.G + min(gr, g.G - 1));
    if (g.parts <= 1 << lg) gn_fold_n<1, kTiled>(w, g, gr, lg, eps, mean, rstd);
    else if (g.parts <= 2 << lg) gn_fold_n<2, kTiled>(w, g, gr, lg, eps, mean, rstd);
    else if (g.parts <= 4 << lg) gn_fold_n<4, kTiled>(w, g, gr, lg, eps, mean, rstd);
    else gn_fold_n<kGnFoldLane, kTiled>(w, g, gr, lg, eps, mean, rstd);
}

// more partials than the second launch's blocks fold: folded once by a launch of its own.  grid (groups / 8, samples)
template <bool kTiled>
__global__ __launch_bounds__(kGnT) void gn_fold_kernel(const float2* __restrict__ ws, float* __restrict__ stats, float eps,
                                                       const GnGeom g) {
    const int n = gn_sample(), gr = blockIdx.x * (kGnT / 64) + (threadIdx.x >> 6);
    if (n >= g.N) return;
    float mean, rstd;
    gn_fold<kTiled>(ws, g, n, gr, 6, eps, mean, rstd);
    if (gr < g.G && (threadIdx.x & 63) == 0) {
        stats[((long)n * g.G + gr) * 2] = mean;
        stats[((long)n * g.G + gr) * 2 + 1] = rstd;
    }
}

// ------------------------------------------------------------------ forward, second launch
// ws: the partials, folded here (the sample's first block leaves the statistics), or NULL: statistics come from stats.
// A slice is walked from its end: what the first launch read last is the likeliest to be in a cache still.  The loads of a
// thread's first rows are on their way while the block folds the partials and makes its table (mean, scale * rstd, shift of
// every channel), those of the next rows while it computes.
// 16 x 1080 x 1920 x 32 bf16 (4.2 GB read and written): 778 us, 5.5 TB/s, a copy's rate; 4 x 256 x 256 x 32 (34 MB) 7.2 us.
template <typename T, int V, bool kNt, bool kPut, bool kRes, bool kTiled>
__global__ __launch_bounds__(kGnT, 4) void gn_apply_kernel(const T* x, const float2* __restrict__ ws, float* __restrict__ stats,
                                                        float eps, const float* __restrict__ scale,
                                                        const float* __restrict__ shift, const T* residual, T* y, int act,
                                                        const GnGeom g) {
    constexpr int kU = 4;
    extern __shared__ float tab[];   // [3][C] mean, scale * rstd, shift; [2G]
    const GnPlace<kTiled> p(g, V, g.S2, g.rows2);
    if (p.n >= g.N) return;
    const int batch = p.slots * kU, full = p.rows / batch, rest = p.rows - full * batch;
    const int step = p.slots * g.L;
    const unsigned own = p.own * (unsigned)sizeof(T);
    const bool on = p.on();
    long at = p.first + (long)full * kU * step;   // the rest of the rows is walked first, then the batches before it
    u32x4 raw[kU];
#pragma unroll
    for (int u = 0; u < kU; u++)
        if (on && p.slot < rest - u * p.slots) raw[u] = gn_load<kNt>(x + at + u * (long)step, own);
    u32x4 next[kU];
    if (on && full > 0) {
#pragma unroll
        for (int u = 0; u < kU; u++) next[u] = gn_load<kNt>(x + at - (kU - u) * (long)step, own);
    }
    float sc = 0.f, sf = 0.f;
    if ((int)threadIdx.x < g.C) {
        sc = scale[threadIdx.x];
        sf = shift[threadIdx.x];
    }
    float* grp = tab + 3 * g.C;
    if (ws) {
        for (int gr0 = 0; gr0 < g.G; gr0 += kGnT >> g.lgG) {
            const int gr = gr0 + (threadIdx.x >> g.lgG);
            float mean, rstd;
            gn_fold<kTiled>(ws, g, p.n, gr, g.lgG, eps, mean, rstd);
            if (gr < g.G && (threadIdx.x & ((1 << g.lgG) - 1)) == 0) {
                grp[2 * gr] = mean;
                grp[2 * gr + 1] = rstd;
                if (blockIdx.x == 0) {
                    stats[((long)p.n * g.G + gr) * 2] = mean;
                    stats[((long)p.n * g.G + gr) * 2 + 1] = rstd;
                }
            }
        }
    } else {
        for (int i = threadIdx.x; i < 2 * g.G; i += kGnT) grp[i] = stats[(long)p.n * g.G * 2 + i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < g.C; c += kGnT) {
        const int gr = gn_div(c, g.rD);
        tab[c] = grp[2 * gr];
        tab[g.C + c] = (c < kGnT ? sc : scale[c]) * grp[2 * gr + 1];
        tab[2 * g.C + c] = c < kGnT ? sf : shift[c];
    }
    __syncthreads();
    gn_with_act(act, [&](auto A) {
        constexpr int kA = decltype(A)::value;
        if (on) {
            float mean[V], a[V], bb[V];
            gn_column<V>(tab, g, p.col, mean);
            gn_column<V>(tab + g.C, g, p.col, a);
            gn_column<V>(tab + 2 * g.C, g, p.col, bb);
            auto put = [&](const u32x4& in, const u32x4& res, long where) {
                float v[V];
                gn_unpack<T, V>(in, v);
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = gn_act<kA>((v[j] - mean[j]) * a[j] + bb[j]);
                if constexpr (kRes) {
                    float r[V];
                    gn_unpack<T, V>(res, r);
#pragma unroll
                    for (int j = 0; j < V; j++) v[j] += r[j];
                }
                gn_store<kPut, T, V>(y + where, own, v);
            };
            u32x4 res[kU];
            if (p.slot < rest) {
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    if (p.slot < rest - u * p.slots) {
                        if constexpr (kRes) res[u] = gn_load<kNt>(residual + at + u * (long)step, own);
                        put(raw[u], res[u], at + u * (long)step);
                    }
                }
            }
            for (int b = full; b > 0; b--) {
                at -= kU * (long)step;
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    raw[u] = next[u];
                    if constexpr (kRes) res[u] = gn_load<kNt>(residual + at + u * (long)step, own);
                }
                if (b > 1) {
#pragma unroll
                    for (int u = 0; u < kU; u++) next[u] = gn_load<kNt>(x + at - (kU - u) * (long)step, own);
                }
#pragma unroll
                for (int u = 0; u < kU; u++) put(raw[u], res[u], at + u * (long)step);
            }
        }
        if (g.tail && p.last) {
            for (int e = threadIdx.x; e < g.tail; e += kGnT) {
                const long q = p.end0 + e;
                const int c = e % g.C;
                float v = gn_act<kA>((to_f32<T>(x[q]) - tab[c]) * tab[g.C + c] + tab[2 * g.C + c]);
                if constexpr (kRes) v += to_f32<T>(residual[q]);
                y[q] = from_f32<T>(v);
            }
        }
    });
}

// ------------------------------------------------------------------ backward, first launch
// rows[n][slice * tiles + tile][2][C]: the block's sums of g and of g * xhat per channel (the parameter gradients' parts);
// grows[...][G][2]: the same times scale, per group.  (A thread adds few values: 32 of a 1080p plane.)
// 4 x 1080 x 1920 x 32 bf16 with SiLU (1.06 GB): 199 us, 5.3 TB/s; its derivative costs an exponential and a reciprocal a value,
// 12 instructions in all, about half of what the vector units could issue in that time.
template <typename T, int V, bool kNt, bool kTiled>
__global__ __launch_bounds__(kGnT, 4) void gn_bwd_sums_kernel(const T* __restrict__ x, const T* __restrict__ dy,
                                                           const float* __restrict__ stats, const float* __restrict__ scale,
                                                           const float* __restrict__ shift, float* __restrict__ rows,
                                                           float2* __restrict__ grows, int act, const GnGeom g) {
    constexpr int kB = 2;
    extern __shared__ float sh[];   // [3][C] mean, scale * rstd, shift, then [V][kGnT] sums of g, [V][kGnT] of g (x - mean);
                                    // behind the larger of the two: [2][C] the block's sums per channel
    const GnPlace<kTiled> p(g, V, g.S, g.rows);
    if (p.n >= g.N) return;
    const float* st = stats + (long)p.n * g.G * 2;
    for (int c = threadIdx.x; c < g.C; c += kGnT) {
        const int gr = gn_div(c, g.rD);
        sh[c] = st[2 * gr];
        sh[g.C + c] = scale[c] * st[2 * gr + 1];
        sh[2 * g.C + c] = shift[c];
    }
    __syncthreads();
    float mean[V], a[V], bb[V];
    if (p.on()) {
        gn_column<V>(sh, g, p.col, mean);
        gn_column<V>(sh + g.C, g, p.col, a);
        gn_column<V>(sh + 2 * g.C, g, p.col, bb);
    }
    __syncthreads();
    float* l1 = sh;
    float* l2 = sh + V * kGnT;
    float* ch = sh + max(2 * V * kGnT, 3 * g.C);
    const unsigned own = p.own * (unsigned)sizeof(T);
    const int step = p.slots * g.L, batch = kB * p.slots;
    gn_with_act(act, [&](auto A) {
        constexpr int kA = decltype(A)::value;
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
        if (p.on()) {
            auto add = [&](const u32x4& vr, const u32x4& dr) {
                float v[V], d[V];
                gn_unpack<T, V>(vr, v);
                gn_unpack<T, V>(dr, d);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xm = v[j] - mean[j];
                    const float gv = d[j] * gn_act_grad<kA>(xm * a[j] + bb[j]);
                    s1[j] += gv;
                    s2[j] += gv * xm;
                }
            };
            // two batches of rows: one on its way, one in the computation
            u32x4 vr[kB], dr[kB], vn[kB], dn[kB];
            auto load = [&](u32x4 (&v)[kB], u32x4 (&d)[kB], int left, long at) {
#pragma unroll
                for (int u = 0; u < kB; u++) {
                    if (p.slot < left - u * p.slots) {
                        v[u] = gn_load<kNt>(x + at + u * (long)step, own);
                        d[u] = gn_load<kNt>(dy + at + u * (long)step, own);
                    }
                }
            };
            long at = p.first;
            load(vr, dr, p.rows, at);
            for (int left = p.rows; left > 0; left -= batch) {
                at += kB * (long)step;
                load(vn, dn, left - batch, at);
#pragma unroll
                for (int u = 0; u < kB; u++) {
                    if (p.slot < left - u * p.slots) add(vr[u], dr[u]);
                    vr[u] = vn[u];
                    dr[u] = dn[u];
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
        const int K = 1 << g.lgC, lane = threadIdx.x & (K - 1), reps = g.L / g.C;
        for (int cc = 0; cc < g.C; cc += kGnT >> g.lgC) {
            const int c = cc + (threadIdx.x >> g.lgC);
            const bool live = c < g.C;
            const int gr = gn_div(live ? c : 0, g.rD);
            float t1 = 0.f, t2 = 0.f;
            if (live) {
                for (int rep = 0; rep < reps; rep++) {
                    const int pos = c + rep * g.C, col = pos / V - p.c0, j = pos % V;
                    if (kTiled && (col < 0 || col >= p.QT)) continue;
                    for (int slot = lane; slot < p.slots; slot += K) {
                        t1 += l1[j * kGnT + slot * p.QT + col];
                        t2 += l2[j * kGnT + slot * p.QT + col];
                    }
                }
                if (g.tail && p.last) {
                    for (int e = lane; e < g.tail / g.C; e += K) {
                        const long q = p.end0 + e * g.C + c;
                        const float xm = to_f32<T>(x[q]) - st[2 * gr];
                        const float gv = to_f32<T>(dy[q]) * gn_act_grad<kA>(xm * (scale[c] * st[2 * gr + 1]) + shift[c]);
                        t1 += gv;
                        t2 += gv * xm;
                    }
                }
            }
            t1 = gn_team_sum(t1, g.lgC);
            t2 = gn_team_sum(t2, g.lgC);
            if (live && lane == 0) {
                ch[c] = t1;
                ch[g.C + c] = t2 * st[2 * gr + 1];
            }
        }
        __syncthreads();
    });
    const long part = p.part(g);
    for (int i = threadIdx.x; i < 2 * g.C; i += kGnT) rows[part * 2 * g.C + i] = ch[i];
    const int K = 1 << g.lgG, lane = threadIdx.x & (K - 1);
    for (int gr0 = 0; gr0 < g.G; gr0 += kGnT >> g.lgG) {
        const int gr = gr0 + (threadIdx.x >> g.lgG);
        float t1 = 0.f, t2 = 0.f;
        if (gr < g.G) {
            for (int c = gr * g.D + lane; c < (gr + 1) * g.D; c += K) {
                t1 += scale[c] * ch[c];
                t2 += scale[c] * ch[g.C + c];
            }
        }
        t1 = gn_team_sum(t1, g.lgG);
        t2 = gn_team_sum(t2, g.lgG);
        if (gr < g.G && lane == 0) grows[part * g.G + gr] = make_float2(t1, t2);
    }
}

// m1, m2 of a group from its partials, as gn_fold
template <int NK>
__device__ __forceinline__ void gn_fold_sums_n(const float2* __restrict__ w, const GnGeom& g, int lg, float& m1, float& m2) {
    const int lane = threadIdx.x & ((1 << lg) - 1);
    float2 r[NK];
#pragma unroll
    for (int k = 0; k < NK; k++) r[k] = w[(unsigned)(min(lane + (k << lg), g.parts - 1) * g.G)];
    m1 = m2 = 0.f;
#pragma unroll
    for (int k = 0; k < NK; k++) {
        if (lane + (k << lg) < g.parts) {
            m1 += r[k].x;
            m2 += r[k].y;
        }
    }
    m1 = gn_team_sum(m1, lg) * g.rM;
    m2 = gn_team_sum(m2, lg) * g.rM;
}

__device__ __forceinline__ void gn_fold_sums(const float2* __restrict__ grows, const GnGeom& g, int n, int gr, int lg, float& m1,
                                             float& m2) {
    const float2* w = grows + ((long)n * g.parts * g.G + min(gr, g.G - 1));
    if (g.parts <= 1 << lg) gn_fold_sums_n<1>(w, g, lg, m1, m2);
    else if (g.parts <= 2 << lg) gn_fold_sums_n<2>(w, g, lg, m1, m2);
    else if (g.parts <= 4 << lg) gn_fold_sums_n<4>(w, g, lg, m1, m2);
    else gn_fold_sums_n<kGnFoldLane>(w, g, lg, m1, m2);
}

__global__ __launch_bounds__(kGnT) void gn_fold_sums_kernel(const float2* __restrict__ grows, float* __restrict__ m, const GnGeom g) {
    const int n = gn_sample(), gr = blockIdx.x * (kGnT / 64) + (threadIdx.x >> 6);
    if (n >= g.N) return;
    float m1, m2;
    gn_fold_sums(grows, g, n, gr, 6, m1, m2);
    if (gr < g.G && (threadIdx.x & 63) == 0) {
        m[((long)n * g.G + gr) * 2] = m1;
        m[((long)n * g.G + gr) * 2 + 1] = m2;
    }
}

// dshift / dscale from the partial rows: outputs o of [0, 2C), 64 a block, eight row groups each, in one fixed order.  Added in
// double: thousands of samples make long runs (131075 equal terms in fp32 were 1.6e-4 off, now 2e-8).  tmp: a number a thread
__device__ __forceinline__ void gn_param_grads(const float* __restrict__ rows, long nrows, float* __restrict__ dscale,
                                               float* __restrict__ dshift, int accumulate, int C, int block, double* tmp) {
    const int o = block * 64 + (threadIdx.x & 63), rg = threadIdx.x >> 6;
    double s = 0.0;
    if (o < 2 * C) {
        long i = rg;
        for (; i + 15 * (kGnT / 64) < nrows; i += 16 * (kGnT / 64)) {
#pragma unroll
            for (int u = 0; u < 16; u++) s += rows[(i + u * (kGnT / 64)) * 2 * C + o];
        }
#pragma unroll 8
        for (; i < nrows; i += kGnT / 64) s += rows[i * 2 * C + o];
    }
    tmp[threadIdx.x] = s;
    __syncthreads();
    if (rg == 0 && o < 2 * C) {
        s = 0.0;
        for (int k = 0; k < kGnT / 64; k++) s += tmp[k * 64 + threadIdx.x];
        float* dst = o < C ? dshift + o : dscale + (o - C);
        *dst = accumulate ? *dst + (float)s : (float)s;
    }
}

// ------------------------------------------------------------------ backward, second launch
// The last blocks fold the parameter gradients, the others write dx.  As in the forward pass a slice is walked from its
// end, and loads are on their way during the fold and the computation of the rows before.
// 4 x 1080 x 1920 x 32 bf16 with SiLU (1.6 GB): 287 us, 5.5 TB/s.
template <typename T, int V, bool kNt, bool kPut, bool kTiled>
__global__ __launch_bounds__(kGnT, 4) void gn_bwd_apply_kernel(const T* x, const T* dy, const float* __restrict__ stats,
                                                            const float* __restrict__ scale, const float* __restrict__ shift,
                                                            const float2* __restrict__ grows, const float* __restrict__ msums,
                                                            const float* __restrict__ rows, T* dx, float* dscale, float* dshift,
                                                            int accumulate, int act, const GnGeom g) {
    constexpr int kU = 2;
    // [5][C] mean, scale * rstd, shift, k1 = rstd m1, k2 = rstd^2 m2 with dx = scale rstd g - k1 - (x - mean) k2; [2G] m1, m2
    // (512 doubles at least)
    extern __shared__ float tab[];
    const int blocks2 = g.S2 * g.tiles;
    if ((int)blockIdx.x >= blocks2) {
        const long q = (long)(blockIdx.x - blocks2) * g.N + gn_sample();
        if (gn_sample() < g.N && q * 64 < 2 * g.C)
            gn_param_grads(rows, (long)g.N * g.parts, dscale, dshift, accumulate, g.C, (int)q, (double*)tab);
        return;
    }
    const GnPlace<kTiled> p(g, V, g.S2, g.rows2);
    if (p.n >= g.N) return;
    const int batch = p.slots * kU, full = p.rows / batch, rest = p.rows - full * batch;
    const int step = p.slots * g.L;
    const unsigned own = p.own * (unsigned)sizeof(T);
    const bool on = p.on();
    long at = p.first + (long)full * kU * step;
    u32x4 vr[kU], dr[kU], vn[kU], dn[kU];
#pragma unroll
    for (int u = 0; u < kU; u++) {
        if (on && p.slot < rest - u * p.slots) {
            vr[u] = gn_load<kNt>(x + at + u * (long)step, own);
            dr[u] = gn_load<kNt>(dy + at + u * (long)step, own);
        }
    }
    if (on && full > 0) {
#pragma unroll
        for (int u = 0; u < kU; u++) {
            vn[u] = gn_load<kNt>(x + at - (kU - u) * (long)step, own);
            dn[u] = gn_load<kNt>(dy + at - (kU - u) * (long)step, own);
        }
    }
    const float* st = stats + (long)p.n * g.G * 2;
    float* grp = tab + 5 * g.C;
    if (msums) {
        for (int i = threadIdx.x; i < 2 * g.G; i += kGnT) grp[i] = msums[(long)p.n * g.G * 2 + i];
    } else {
        for (int gr0 = 0; gr0 < g.G; gr0 += kGnT >> g.lgG) {
            const int gr = gr0 + (threadIdx.x >> g.lgG);
            float m1, m2;
            gn_fold_sums(grows, g, p.n, gr, g.lgG, m1, m2);
            if (gr < g.G && (threadIdx.x & ((1 << g.lgG) - 1)) == 0) {
                grp[2 * gr] = m1;
                grp[2 * gr + 1] = m2;
            }
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < g.C; c += kGnT) {
        const int gr = gn_div(c, g.rD);
        const float rstd = st[2 * gr + 1];
        tab[c] = st[2 * gr];
        tab[g.C + c] = scale[c] * rstd;
        tab[2 * g.C + c] = shift[c];
        tab[3 * g.C + c] = rstd * grp[2 * gr];
        tab[4 * g.C + c] = rstd * rstd * grp[2 * gr + 1];
    }
    __syncthreads();
    gn_with_act(act, [&](auto A) {
        constexpr int kA = decltype(A)::value;
        if (on) {
            float mean[V], a[V], bb[V], k1[V], k2[V];
            gn_column<V>(tab, g, p.col, mean);
            gn_column<V>(tab + g.C, g, p.col, a);
            gn_column<V>(tab + 2 * g.C, g, p.col, bb);
            gn_column<V>(tab + 3 * g.C, g, p.col, k1);
            gn_column<V>(tab + 4 * g.C, g, p.col, k2);
            auto put = [&](const u32x4& vi, const u32x4& di, long where) {
                float v[V], d[V];
                gn_unpack<T, V>(vi, v);
                gn_unpack<T, V>(di, d);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xm = v[j] - mean[j];
                    v[j] = d[j] * gn_act_grad<kA>(xm * a[j] + bb[j]) * a[j] - k1[j] - xm * k2[j];
                }
                gn_store<kPut, T, V>(dx + where, own, v);
            };
            if (p.slot < rest) {
#pragma unroll
                for (int u = 0; u < kU; u++)
                    if (p.slot < rest - u * p.slots) put(vr[u], dr[u], at + u * (long)step);
            }
            for (int b = full; b > 0; b--) {
                at -= kU * (long)step;
#pragma unroll
                for (int u = 0; u < kU; u++) {
                    vr[u] = vn[u];
                    dr[u] = dn[u];
                }
                if (b > 1) {
#pragma unroll
                    for (int u = 0; u < kU; u++) {
                        vn[u] = gn_load<kNt>(x + at - (kU - u) * (long)step, own);
                        dn[u] = gn_load<kNt>(dy + at - (kU - u) * (long)step, own);
                    }
                }
#pragma unroll
                for (int u = 0; u < kU; u++) put(vr[u], dr[u], at + u * (long)step);
            }
        }
        if (g.tail && p.last) {
            for (int e = threadIdx.x; e < g.tail; e += kGnT) {
                const long q = p.end0 + e;
                const int c = e % g.C;
                const float xm = to_f32<T>(x[q]) - tab[c], sa = tab[g.C + c];
                dx[q] = from_f32<T>(to_f32<T>(dy[q]) * gn_act_grad<kA>(xm * sa + tab[2 * g.C + c]) * sa - tab[3 * g.C + c] -
                                    xm * tab[4 * g.C + c]);
            }
        }
    });
}

// ------------------------------------------------------------------ small samples: one launch
// A unit is one group, or the V / D groups of one 16-byte column where D < V; its P pixels x DV columns stay in the
// registers of ONE block: read once, the mean first, then the deviations from it, then the result.  Neighbouring units
// share cache lines: the block numbers are dealt so that they run on one XCD (one L2): 16 samples of 32 x 32 x 512 bf16 in 32
// groups 18.5 -> 11.0 us forward, 31.6 -> 19.5 backward.  One launch of 1 x 16 x 16 x 512 takes 4.4 us, bound by latency.
struct GnUnit {
    int n, unit, DV, Ta, col, pix, dpix;
    long at;   // the thread's first vector, in elements
    __device__ __forceinline__ GnUnit(const GnGeom& g, int V) {
        const unsigned w = max(g.D, V), units = g.C / w, lin = (blockIdx.x & 7) * (gridDim.x / 8) + (blockIdx.x >> 3);
        n = lin / units;
        unit = lin - n * units;
        DV = w / V;
        dpix = blockDim.x / DV;
        Ta = dpix * DV;
        pix = gn_div(threadIdx.x, g.rQT);   // the launcher's: of DV
        col = threadIdx.x - pix * DV;
        if ((int)threadIdx.x >= Ta) pix = g.P;
        at = ((long)n * g.P + pix) * g.C + (long)unit * w + col * V;
    }
};

// sums of NS values over the block, in every thread; red: [16][NS]
template <int NS>
__device__ __forceinline__ void gn_block_sums(float (&v)[NS], float* red) {
    const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int k = 0; k < NS; k++) v[k] = gn_team_sum(v[k], 6);
    if (waves == 1) return;
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int k = 0; k < NS; k++) red[wave * NS + k] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NS; k++) v[k] = 0.f;
    for (int w = 0; w < waves; w++)
#pragma unroll
        for (int k = 0; k < NS; k++) v[k] += red[w * NS + k];
}

template <typename T, int V, int NS, int kU>
__global__ __launch_bounds__(1024) void gn_unit_fwd_kernel(const T* x, float* __restrict__ stats, float eps,
                                                           const float* __restrict__ scale, const float* __restrict__ shift,
                                                           const T* residual, T* y, int act, const GnGeom g) {
    constexpr int W = V / NS;   // channels of a column that share a group
    __shared__ float red[16 * NS];
    const GnUnit u_(g, V);
    if (u_.n >= g.N) return;
    const long step = (long)u_.dpix * g.C;
    u32x4 raw[kU];
#pragma unroll
    for (int u = 0; u < kU; u++)
        if (u_.pix + u * u_.dpix < g.P) raw[u] = gn_load<false>(x + u_.at + u * step, 0);
    const int c0 = u_.unit * max(g.D, V) + u_.col * V;
    // the unit's first 16 bytes: its groups' first values, from which the mean deviates
    const u32x4 first = gn_load<false>(x + ((long)u_.n * g.P * g.C + (long)u_.unit * max(g.D, V)), 0);
    float a[V], b[V];
    if (u_.pix < g.P) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            a[j] = scale[c0 + j];
            b[j] = shift[c0 + j];
        }
    }
    const float rM = g.rM;
    float x0[V], mean[NS], rstd[NS];
    gn_unpack<T, V>(first, x0);
#pragma unroll
    for (int k = 0; k < NS; k++) mean[k] = rstd[k] = 0.f;
#pragma unroll
    for (int u = 0; u < kU; u++) {
        if (u_.pix + u * u_.dpix < g.P) {
            float v[V];
            gn_unpack<T, V>(raw[u], v);
#pragma unroll
            for (int j = 0; j < V; j++) mean[j / W] += (v[j] - x0[j / W * W]) * rM;
        }
    }
    gn_block_sums<NS>(mean, red);
#pragma unroll
    for (int k = 0; k < NS; k++) mean[k] += x0[k * W];
#pragma unroll
    for (int u = 0; u < kU; u++) {
        if (u_.pix + u * u_.dpix < g.P) {
            float v[V];
            gn_unpack<T, V>(raw[u], v);
#pragma unroll
            for (int j = 0; j < V; j++) {
                const float d = v[j] - mean[j / W];
                rstd[j / W] += d * rM * d;
            }
        }
    }
    gn_block_sums<NS>(rstd, red);
#pragma unroll
    for (int k = 0; k < NS; k++) {
        rstd[k] = gn_rsqrt(rstd[k] + eps);
        if (threadIdx.x == 0) {
            float* st = stats + ((long)u_.n * g.G + u_.unit * NS + k) * 2;
            st[0] = mean[k];
            st[1] = rstd[k];
        }
    }
#pragma unroll
    for (int j = 0; j < V; j++) a[j] *= rstd[j / W];
    gn_with_act(act, [&](auto A) {
        constexpr int kA = decltype(A)::value;
#pragma unroll
        for (int u = 0; u < kU; u++) {
            if (u_.pix + u * u_.dpix < g.P) {
                float v[V];
                gn_unpack<T, V>(raw[u], v);
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = gn_act<kA>((v[j] - mean[j / W]) * a[j] + b[j]);
                if (residual) {
                    float r[V];
                    gn_unpack<T, V>(gn_load<false>(residual + u_.at + u * step, 0), r);
#pragma unroll
                    for (int j = 0; j < V; j++) v[j] += r[j];
                }
                gn_store<false, T, V>(y + u_.at + u * step, 0, v);
            }
        }
    });
}

// rows[n][2][C]: the sample's sums of g and g * xhat per channel; for one sample the parameter gradients themselves
template <typename T, int V, int NS, int kU>
__global__ __launch_bounds__(512) void gn_unit_bwd_kernel(const T* x, const T* dy, const float* __restrict__ stats,
                                                          const float* __restrict__ scale, const float* __restrict__ shift,
                                                          T* dx, float* __restrict__ rows, float* dscale, float* dshift,
                                                          int accumulate, int act, const GnGeom g) {
    constexpr int W = V / NS;
    extern __shared__ float sh[];   // [2][V][blockDim] the threads' sums
    __shared__ float red[8 * 2 * NS];
    const GnUnit u_(g, V);
    if (u_.n >= g.N) return;
    const int T_ = blockDim.x, wide = max(g.D, V), c0 = u_.unit * wide;
    const long step = (long)u_.dpix * g.C;
    u32x4 vr[kU], dr[kU];
#pragma unroll
    for (int u = 0; u < kU; u++) {
        if (u_.pix + u * u_.dpix < g.P) {
            vr[u] = gn_load<false>(x + u_.at + u * step, 0);
            dr[u] = gn_load<false>(dy + u_.at + u * step, 0);
        }
    }
    float a[V], b[V], mean[NS], rstd[NS];
#pragma unroll
    for (int k = 0; k < NS; k++) {
        const float* st = stats + ((long)u_.n * g.G + u_.unit * NS + k) * 2;
        mean[k] = st[0];
        rstd[k] = st[1];
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        a[j] = scale[c0 + u_.col * V + j] * rstd[j / W];
        b[j] = shift[c0 + u_.col * V + j];
    }
    gn_with_act(act, [&](auto A) {
        constexpr int kA = decltype(A)::value;
        float s1[V], s2[V];
#pragma unroll
        for (int j = 0; j < V; j++) s1[j] = s2[j] = 0.f;
#pragma unroll
        for (int u = 0; u < kU; u++) {
            if (u_.pix + u * u_.dpix < g.P) {
                float v[V], d[V];
                gn_unpack<T, V>(vr[u], v);
                gn_unpack<T, V>(dr[u], d);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xm = v[j] - mean[j / W];
                    const float gv = d[j] * gn_act_grad<kA>(xm * a[j] + b[j]);
                    s1[j] += gv;
                    s2[j] += gv * xm;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < V; j++) {
            sh[j * T_ + threadIdx.x] = s1[j];
            sh[(V + j) * T_ + threadIdx.x] = s2[j] * rstd[j / W];
        }
        // m1, m2: scale times the sums over the unit's channels, straight from the threads' sums
        float m[2 * NS];
#pragma unroll
        for (int k = 0; k < 2 * NS; k++) m[k] = 0.f;
#pragma unroll
        for (int j = 0; j < V; j++) {
            m[j / W] += a[j] * s1[j];            // rstd times the wanted sum
            m[NS + j / W] += a[j] * s2[j];       // the wanted sum: the product with rstd makes xhat
        }
        gn_block_sums<2 * NS>(m, red);
        const float rM = g.rM;
        // dx = a g - k1 - (x - mean) k2,  k1 = rstd m1,  k2 = rstd^2 m2
#pragma unroll
        for (int k = 0; k < NS; k++) {
            m[k] *= rM;
            m[NS + k] = m[NS + k] * rM * rstd[k] * rstd[k];   // in this order: the product alone may be below 2^-126
        }
#pragma unroll
        for (int u = 0; u < kU; u++) {
            if (u_.pix + u * u_.dpix < g.P) {
                float v[V], d[V];
                gn_unpack<T, V>(vr[u], v);
                gn_unpack<T, V>(dr[u], d);
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const float xm = v[j] - mean[j / W];
                    v[j] = d[j] * gn_act_grad<kA>(xm * a[j] + b[j]) * a[j] - m[j / W] - xm * m[NS + j / W];
                }
                gn_store<false, T, V>(dx + u_.at + u * step, 0, v);
            }
        }
    });
    if (!rows && !dscale) return;
    __syncthreads();
    // per channel: a team of lanes adds the slots' sums
    const int K = 1 << g.lgC, lane = threadIdx.x & (K - 1), teams = T_ >> g.lgC;   // lgC: the launcher's, of max(D, V)
    for (int cc = 0; cc < wide; cc += teams) {
        const int c = cc + (threadIdx.x >> g.lgC);
        float t1 = 0.f, t2 = 0.f;
        if (c < wide) {
            for (int slot = lane; slot < u_.dpix; slot += K) {
                t1 += sh[(c % V) * T_ + slot * u_.DV + c / V];
                t2 += sh[(V + c % V) * T_ + slot * u_.DV + c / V];
            }
        }
        t1 = gn_team_sum(t1, g.lgC);
        t2 = gn_team_sum(t2, g.lgC);
        if (c < wide && lane == 0) {
            if (rows) {
                rows[((long)u_.n * 2) * g.C + c0 + c] = t1;
                rows[((long)u_.n * 2 + 1) * g.C + c0 + c] = t2;
            } else {
                dshift[c0 + c] = accumulate ? dshift[c0 + c] + t1 : t1;
                dscale[c0 + c] = accumulate ? dscale[c0 + c] + t2 : t2;
            }
        }
    }
}

__global__ __launch_bounds__(kGnT) void gn_param_grads_kernel(const float* __restrict__ rows, long nrows, float* dscale,
                                                              float* dshift, int accumulate, int C) {
    __shared__ double tmp[kGnT];
    gn_param_grads(rows, nrows, dscale, dshift, accumulate, C, blockIdx.x, tmp);
}

__global__ __launch_bounds__(256) void gn_zero_kernel(float* a, float* b, int n) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < n) a[i] = b[i] = 0.f;
}

// ------------------------------------------------------------------ launches
// log2 of the lanes (64 at most) that `teams` teams of a block of `threads` have each
static int gn_lg_lanes(int teams, int threads) {
    int lg = 6;
    while (lg > 0 && (teams << lg) > threads) lg--;
    return lg;
}

static unsigned gn_recip(int d) { return d == 1 ? 0u : (unsigned)(((1UL << 32) + d - 1) / d); }

static int gcd_int(int a, int b) { return b ? gcd_int(b, a % b) : a; }

static GnGeom gn_geom(int n, int P, int c, int groups, int V, bool backward) {
    GnGeom g;
    g.N = n; g.P = P; g.C = c; g.G = groups; g.D = c / groups;
    g.L = c / gcd_int(c, V) * V;
    g.Q = g.L / V;
    g.U = gcd_int(V, g.D);
    g.QT = g.Q < kGnT ? g.Q : kGnT;
    g.tiles = ceil_div(g.Q, g.QT);
    g.slots = kGnT / g.QT;
    g.R = (int)((long)P * c / g.L);
    g.tail = (int)((long)P * c - (long)g.R * g.L);
    g.lgG = gn_lg_lanes(groups, kGnT);
    g.lgC = gn_lg_lanes(c, kGnT);
    // `deep` rows a thread of a sample, cut into slices of k: the same way whatever its batch.  Four to eight rows (32 to 64
    // KB a slice): with fewer rows, more blocks for a lone sample; with more, fewer fixed costs (fold, tables, reductions)
    // for a batch.  Forward, 1 and 16 samples of 256 x 256 x 32 bf16: four rows 9.9 and 40.6 us, eight 10.1 and 35.6;
    // backward (with forward) 21.5 and 110, 25.3 and 98.6.
    const int deep = ceil_div(g.R, g.slots), most = backward ? 128 : 64;
    int k = deep <= 4 * most ? 4 : deep <= 8 * most ? ceil_div(deep, most) : 8;
    // few enough partials for the second launch to fold, unless the sample is large (32 MB) or would be cut in too few
    const int few = (kGnFoldLane << g.lgG) / g.tiles, all = kGnSlices / g.tiles;
    if (few >= 64 && (long)P * c / V * 16 <= (32L << 20) && k < ceil_div(deep, few)) k = ceil_div(deep, few);
    if (k < ceil_div(deep, all)) k = ceil_div(deep, all);
    g.rows = g.slots * k;
    g.S = g.R ? ceil_div(g.R, g.rows) : 1;
    g.parts = g.S * g.tiles;
    // The second launch's cut changes no sum: one block a CU where its fold and table are a good part of the work, many where
    // the tensor is large (16 x 1080 x 1920 x 32 bf16, forward: 2048 blocks 1248 us, 4096 1099, 8192 1092), four rows a thread
    // at least.
    const long mb = (long)n * P * c / V * 16 >> 20;
    const int blocks2 = mb > 256 ? 8192 : mb > 48 || backward ? 512 : 256;
    const int k2 = ceil_div((long)deep * g.tiles * (n > 0 ? n : 1), blocks2);
    g.rows2 = g.slots * (k2 > 4 ? k2 : 4);
    g.S2 = g.R ? ceil_div(g.R, g.rows2) : 1;
    const int units = g.D / g.U, entries = units * (g.L / c), K = 1 << g.lgG;
    g.over_slots = entries * ceil_div(g.slots, K) <= g.slots * ceil_div(entries, K);
    g.rC = gn_recip(c);
    g.rD = gn_recip(g.D);
    g.rQT = gn_recip(g.QT);
    g.rUnits = gn_recip(units);
    const double M = (double)P * g.D, pixels = (double)g.L / c;
    const int last = g.R - (g.S - 1) * g.rows;
    g.rM = (float)(1.0 / M);
    g.share = (float)(g.rows * pixels * g.D / M);
    g.share_last = (float)((last * pixels + g.tail / c) * g.D / M);
    return g;
}

// the second launch's blocks fold the partials themselves
static bool gn_folds_itself(const GnGeom& g) { return g.parts <= kGnFoldLane << g.lgG; }

// One block per unit, if a unit's vectors fit its registers: threads and vectors a thread, or false.
// STMI_NO_GN_UNITS: never (tests compare the two forms).
static bool gn_in_units(const GnGeom& g, int V, int most_threads, int* threads, int* u) {
    if (g.C % V || (g.D % V && V % g.D) || STMI_ENV_SET("STMI_NO_GN_UNITS")) return false;
    const int DV = (g.D > V ? g.D : V) / V;
    const long nv = (long)g.P * DV;
    // A unit 16 bytes wide reads every cache line in pieces.  Graph of 20 calls, us, one block per unit / slices: 2025 pixels
    // 16 bytes wide 6.0 / 8.8 forward and 8.5 / 12.2 backward (one sample of 64 channels), 4096 pixels 8.9 / 8.7 and 13.1 / 11.5;
    // 32 bytes wide, 4096 pixels 12.2 / 11.2 (one sample of 512 channels), 33.7 / 51.8 (16 samples), 64 bytes 22.1 / 47.2.
    if (DV == 1 && nv > 2048) return false;
    for (*u = 2; *u <= 8; *u *= 2)
        for (*threads = 64; *threads <= most_threads; *threads *= 2)
            if ((long)(*threads / DV * DV) * *u >= nv) return true;
    return false;
}

// Samples of one launch of `units` blocks a sample: a grid has less than 2^32 threads, 131072 samples of one pixel and 4096
// channels fill it.
static int gn_unit_samples(int units, int threads) { return (int)((1L << 31) / threads / units); }

long gn_ws_floats(int n, int h, int w, int c, int groups, int dtype, int backward) {
    const int V = dtype == STMI_BF16 ? 8 : 4;
    const GnGeom g = gn_geom(n, h * w, c, groups, V, backward);
    const long parts = (long)n * g.parts;
    int threads, u;
    if (gn_in_units(g, V, backward ? kGnUnitBwd : kGnUnitFwd, &threads, &u)) return backward && n > 1 ? (long)n * 2 * c : 0;
    return backward ? parts * 2 * c + parts * 2 * groups + (long)n * 2 * groups : parts * 2 * groups;
}

// f(groups of a column, vectors of a thread) as compile-time constants.  Units 16 bytes wide have 2048 vectors at most
// (gn_in_units): two a thread forward (1024 threads), two or four backward (512).
template <int V, int kNarrow, typename F>
static void gn_unit_launch(const GnGeom& g, int u, F&& f) {
    const int ns = g.D >= V ? 1 : V / g.D;
    auto narrow = [&](auto NS) {
        if (kNarrow == 2 || u == 2) f(NS, std::integral_constant<int, 2>{});
        else f(NS, std::integral_constant<int, kNarrow>{});
    };
    if (ns == 1) {
        std::integral_constant<int, 1> one;
        if (u == 2) f(one, std::integral_constant<int, 2>{});
        else if (u == 4) f(one, std::integral_constant<int, 4>{});
        else f(one, std::integral_constant<int, 8>{});
    } else if (ns == 2) narrow(std::integral_constant<int, 2>{});
    else if (ns == 4) narrow(std::integral_constant<int, 4>{});
    else narrow(std::integral_constant<int, V>{});
}

// Streaming past the caches.  Outputs do from 64 MB of tensors on (below that the next operator may find them in the L2s):
// what was read stays in the last-level cache (256 MB) for the second launch.  16 x 540 x 960 x 32 bf16 cut to 1, 3 and 4
// samples, forward: 22.9 / 63 / 82 us with ordinary stores, 21.3 / 54 / 71 without.  Inputs that do not fit that cache are
// not kept in it either: a 2.1 GB tensor is read at 7.1 TB/s instead of 6.2.
struct GnStream {
    bool loads, stores;
    GnStream(int read, int others, int n, int P, int c, int size) {
        const long one = (long)n * P * c * size;
        loads = read * one > (224L << 20);
        stores = (read + others) * one > (64L << 20);
    }
};

// f(kNt, kPut, kTiled) as compile-time constants; rows of several tiles are rare (more than 512
// columns: channel counts above 512 V, or above 512 and no multiple of V): one form
template <typename F>
static int gn_with_form(const GnStream& st, const GnGeom& g, F&& f) {
    if (g.tiles > 1) return f(std::false_type{}, std::false_type{}, std::true_type{});
    if (st.loads) return f(std::true_type{}, std::true_type{}, std::false_type{});
    if (st.stores) return f(std::false_type{}, std::true_type{}, std::false_type{});
    return f(std::false_type{}, std::false_type{}, std::false_type{});
}

template <typename T, int V>
static int gn_fwd_t(const T* x, float* ws, float* stats, float eps, const float* scale, const float* shift, const T* residual,
                    T* y, int act, int n, int P, int c, int groups, hipStream_t s) {
    GnGeom g = gn_geom(n, P, c, groups, V, false);
    int threads, u;
    if (gn_in_units(g, V, kGnUnitFwd, &threads, &u)) {
        const int wide = g.D > V ? g.D : V;
        g.rQT = gn_recip(wide / V);
        const int most = gn_unit_samples(c / wide, threads);
        for (long n0 = 0; n0 < n; n0 += most) {
            const long at = n0 * P * c;
            g.N = n - n0 < most ? (int)(n - n0) : most;
            const dim3 grid((unsigned)ceil_div((long)g.N * (c / wide), 8) * 8);
            gn_unit_launch<V, 2>(g, u, [&](auto NS, auto U) {
                hipLaunchKernelGGL((gn_unit_fwd_kernel<T, V, decltype(NS)::value, decltype(U)::value>), grid, dim3(threads), 0, s, x + at,
                                   stats + n0 * groups * 2, eps, scale, shift, residual ? residual + at : nullptr, y + at, act, g);
            });
            STMI_LAUNCH_CHECK("gn_unit_fwd_kernel");
        }
        return STMI_OK;
    }
    return gn_with_form(GnStream(1, residual ? 2 : 1, n, P, c, sizeof(T)), g, [&](auto NT, auto PT, auto TL) -> int {
        constexpr bool kNt = decltype(NT)::value, kPut = decltype(PT)::value, kTiled = decltype(TL)::value;
        const dim3 grid = gn_grid(g.parts, n), grid2 = gn_grid(g.S2 * g.tiles, n);
        hipLaunchKernelGGL((gn_stats_kernel<T, V, kNt, kTiled>), grid, dim3(kGnT), (2 * V + 1) * kGnT * sizeof(float), s, x, (float2*)ws, g);
        STMI_LAUNCH_CHECK("gn_stats_kernel");
        const float2* fold = (const float2*)ws;
        if (!gn_folds_itself(g)) {
            hipLaunchKernelGGL((gn_fold_kernel<kTiled>), gn_grid(ceil_div(groups, kGnT / 64), n), dim3(kGnT), 0, s, fold, stats, eps, g);
            STMI_LAUNCH_CHECK("gn_fold_kernel");
            fold = nullptr;
        }
        const int lds = (3 * c + 2 * groups) * (int)sizeof(float), most = 5 * STMI_GN_MAX_C * (int)sizeof(float);
        if (residual) {
            STMI_DYN_LDS((gn_apply_kernel<T, V, kNt, kPut, true, kTiled>), most, "gn_apply_kernel");
            hipLaunchKernelGGL((gn_apply_kernel<T, V, kNt, kPut, true, kTiled>), grid2, dim3(kGnT), lds, s, x, fold, stats, eps, scale, shift,
                               residual, y, act, g);
        } else {
            STMI_DYN_LDS((gn_apply_kernel<T, V, kNt, kPut, false, kTiled>), most, "gn_apply_kernel");
            hipLaunchKernelGGL((gn_apply_kernel<T, V, kNt, kPut, false, kTiled>), grid2, dim3(kGnT), lds, s, x, fold, stats, eps, scale, shift,
                               residual, y, act, g);
        }
        STMI_LAUNCH_CHECK("gn_apply_kernel");
        return STMI_OK;
    });
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
    GnGeom g = gn_geom(n, P, c, groups, V, true);
    int threads, u;
    if (gn_in_units(g, V, kGnUnitBwd, &threads, &u)) {
        const int wide = g.D > V ? g.D : V;
        g.rQT = gn_recip(wide / V);
        g.lgC = gn_lg_lanes(wide, threads);
        float* r = dscale && n > 1 ? ws : nullptr;
        const int most = gn_unit_samples(c / wide, threads);
        for (long n0 = 0; n0 < n; n0 += most) {
            const long at = n0 * P * c;
            g.N = n - n0 < most ? (int)(n - n0) : most;
            const dim3 grid((unsigned)ceil_div((long)g.N * (c / wide), 8) * 8);
            gn_unit_launch<V, 4>(g, u, [&](auto NS, auto U) {
                hipLaunchKernelGGL((gn_unit_bwd_kernel<T, V, decltype(NS)::value, decltype(U)::value>), grid, dim3(threads),
                                   2 * V * threads * sizeof(float), s, x + at, dy + at, stats + n0 * groups * 2, scale, shift, dx + at,
                                   r ? r + n0 * 2 * c : nullptr, dscale, dshift, accumulate, act, g);
            });
            STMI_LAUNCH_CHECK("gn_unit_bwd_kernel");
        }
        if (r) {
            hipLaunchKernelGGL(gn_param_grads_kernel, dim3(ceil_div(2L * c, 64)), dim3(kGnT), 0, s, (const float*)r, (long)n, dscale,
                               dshift, accumulate, c);
            STMI_LAUNCH_CHECK("gn_param_grads_kernel");
        }
        return STMI_OK;
    }
    return gn_with_form(GnStream(2, 1, n, P, c, sizeof(T)), g, [&](auto NT, auto PT, auto TL) -> int {
        constexpr bool kNt = decltype(NT)::value, kPut = decltype(PT)::value, kTiled = decltype(TL)::value;
        const long parts = (long)n * g.parts;
        float* rows = ws;
        float2* grows = (float2*)(rows + parts * 2 * c);
        float* msums = (float*)(grows + parts * groups);
        const int entries = 2 * V * kGnT, lds = ((entries > 3 * c ? entries : 3 * c) + 2 * c) * (int)sizeof(float);
        STMI_DYN_LDS((gn_bwd_sums_kernel<T, V, kNt, kTiled>), 5 * STMI_GN_MAX_C * (int)sizeof(float), "gn_bwd_sums_kernel");
        hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, kNt, kTiled>), gn_grid(g.parts, n), dim3(kGnT), lds, s, x, dy, stats, scale, shift,
                           rows, grows, act, g);
        STMI_LAUNCH_CHECK("gn_bwd_sums_kernel");
        const float* m = nullptr;
        if (!gn_folds_itself(g)) {
            hipLaunchKernelGGL(gn_fold_sums_kernel, gn_grid(ceil_div(groups, kGnT / 64), n), dim3(kGnT), 0, s, (const float2*)grows, msums, g);
            STMI_LAUNCH_CHECK("gn_fold_sums_kernel");
            m = msums;
        }
        const int pblocks = dscale ? ceil_div(2L * c, 64) : 0, table = 5 * c + 2 * groups > 2 * kGnT ? 5 * c + 2 * groups : 2 * kGnT;
        STMI_DYN_LDS((gn_bwd_apply_kernel<T, V, kNt, kPut, kTiled>), 7 * STMI_GN_MAX_C * (int)sizeof(float), "gn_bwd_apply_kernel");
        hipLaunchKernelGGL((gn_bwd_apply_kernel<T, V, kNt, kPut, kTiled>), gn_grid(g.S2 * g.tiles + ceil_div(pblocks, n), n), dim3(kGnT),
                           table * sizeof(float), s, x, dy, stats, scale, shift, (const float2*)grows, m, (const float*)rows, dx, dscale,
                           dshift, accumulate, act, g);
        STMI_LAUNCH_CHECK("gn_bwd_apply_kernel");
        return STMI_OK;
    });
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
