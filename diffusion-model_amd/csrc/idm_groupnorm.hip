// Group normalisation with an activation, channels last, forward and backward (the norms of the bit-flip UNet's ResBlocks,
// mnist_diffusion/mnist_diffusion.py:168-193, as training needs them: any group count, statistics kept, gradients).
//
//   u = x + shift[b, c]                       (the block's time vector; optional)
//   xhat = (u - mean) * rstd                  mean, rstd over the pixels and channels of a group
//   z = xhat * gamma[c] + beta[c],  y = z  or  z * sigmoid(z)
//   dz = dy * y'(z);  dbeta = sum dz;  dgamma = sum dz * xhat
//   dx = rstd * (dz * gamma - A - xhat * B)   A = mean over the group of dz * gamma, B = of dz * gamma * xhat
//   dshift[b, c] = sum over the pixels of dx = rstd * (gamma * sum dz - pixels * A - B * sum xhat)
//
// All arithmetic between the load and the store is float32; y and dx are rounded once, to the type of x.
//
// Two launches per direction: partial statistics of (sample, pixel chunk, channel tile), then a kernel that joins a sample's
// partials and applies.  The weight gradients are partial sums per (sample, chunk) joined by two more small launches, in a
// fixed order: no atomics, so results do not depend on the order in which workgroups run.
#include "../../include/isingdiff.h"
#include "idm_internal.h"
#include "idm_device.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int THREADS = 256;

template <typename T, int V> struct VecOf { typedef __attribute__((ext_vector_type(V))) T type; };
template <typename T> struct VecOf<T, 1> { typedef T type; };

// V consecutive channels as float32
template <typename T, int V> DEVI void load_vec(const T *p, float out[V])
{
    const typename VecOf<T, V>::type v = *(const typename VecOf<T, V>::type *)p;
    if constexpr (V == 1) {
        out[0] = (float)v;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = (float)v[j];
    }
}

template <typename T, int V> DEVI void store_vec(T *p, const float in[V])
{
    if constexpr (V == 1) {
        *p = (T)in[0];
    } else {
        typename VecOf<T, V>::type v;
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (T)in[j];
        *(typename VecOf<T, V>::type *)p = v;
    }
}

// V consecutive float32 of an optional per-channel array (nullptr: the value it stands for)
template <int V> DEVI void load_chan(const float *p, int c, float missing, float out[V])
{
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = p ? p[c + j] : missing;
}

DEVI float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.4426950408889634f)); }

// Count, mean and sum of squared distances from it, of a set of values; join() is the union of two sets.  Sums of raw squares
// would lose the variance of values that lie far from zero.
struct Moments {
    float n, mean, m2;
};
DEVI Moments join(const Moments &a, const Moments &b)
{
    const float n = a.n + b.n;
    if (n == 0.0f) return a;
    const float w = b.n / n, d = b.mean - a.mean;
    return {n, a.mean + d * w, a.m2 + b.m2 + d * d * (a.n * w)};
}

// How the kernels cut a tensor.  A channel tile is at most THREADS vectors of V channels: gpt whole groups, or (groups wider
// than that) one of the tpg parts of a group.
struct Geometry {
    int64_t batch, pixels, x_sample, x_pixel, dy_sample, dy_pixel, shift_sample;
    int channels, groups, gc;     // gc: channels of a group
    int gpt, tpg, ntile;
    int nchunk;
    int64_t chunk;                // pixels of a chunk (the last may be shorter)
    float eps;
    const float *gamma, *beta, *shift;
};

struct Place {
    int64_t b, p0, p1;
    int chunk, tile, c0, width, g0, ng;   // tile's first channel, channels, first group, groups (1 where a group spans tiles)
};

DEVI Place place_of(const Geometry &g, int64_t block, int part_channels)
{
    Place w;
    w.tile = (int)(block % g.ntile);
    const int64_t r = block / g.ntile;
    w.chunk = (int)(r % g.nchunk);
    w.b = r / g.nchunk;
    w.p0 = w.chunk * g.chunk;
    w.p1 = w.p0 + g.chunk < g.pixels ? w.p0 + g.chunk : g.pixels;
    if (g.tpg == 1) {
        w.g0 = w.tile * g.gpt;
        w.ng = g.groups - w.g0 < g.gpt ? g.groups - w.g0 : g.gpt;
        w.c0 = w.g0 * g.gc;
        w.width = w.ng * g.gc;
    } else {
        w.g0 = w.tile / g.tpg;
        w.ng = 1;
        const int at = (w.tile - w.g0 * g.tpg) * part_channels;
        w.c0 = w.g0 * g.gc + at;
        w.width = g.gc - at < part_channels ? g.gc - at : part_channels;
    }
    return w;
}

// Partial statistics: partial[(b * nchunk + chunk) * tpg + part][group] = (n, mean, m2) as three planes' worth of floats.
template <typename T, int V>
__global__ __launch_bounds__(THREADS) void gn_stats_kernel(Geometry g, const T *__restrict__ x, float *__restrict__ partial)
{
    constexpr int U = 4;   // vectors taken together: their mean first, then the squared distances from it
    __shared__ Moments sh[THREADS];
    const Place w = place_of(g, blockIdx.x, THREADS * V);
    const int q = w.width / V, rows = THREADS / q, r = threadIdx.x / q, cq = threadIdx.x - r * q;
    Moments mine = {0.0f, 0.0f, 0.0f};
    if (r < rows) {
        const int c = w.c0 + cq * V;
        const T *xp = x + w.b * g.x_sample + c;
        float add[V];
        load_chan<V>(g.shift ? g.shift + w.b * g.shift_sample : nullptr, c, 0.0f, add);
        int64_t p = w.p0 + r;
        for (; p + (U - 1) * (int64_t)rows < w.p1; p += U * (int64_t)rows) {
            float v[U][V], s = 0.0f, d2 = 0.0f;
#pragma unroll
            for (int k = 0; k < U; ++k) load_vec<T, V>(xp + (p + k * (int64_t)rows) * g.x_pixel, v[k]);
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) s += v[k][j] += add[j];
            const float mean = s * (1.0f / (U * V));
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float d = v[k][j] - mean;
                    d2 = __builtin_fmaf(d, d, d2);
                }
            mine = join(mine, {(float)(U * V), mean, d2});
        }
        for (; p < w.p1; p += rows) {
            float v[V], s = 0.0f, d2 = 0.0f;
            load_vec<T, V>(xp + p * g.x_pixel, v);
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[j] += add[j];
            const float mean = s * (1.0f / V);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[j] - mean;
                d2 = __builtin_fmaf(d, d, d2);
            }
            mine = join(mine, {(float)V, mean, d2});
        }
    }
    sh[threadIdx.x] = mine;
    __syncthreads();
    // wavefront k joins groups k, k + 4, ...: entry e of a group is thread (e / qg) * q + group * qg + e % qg
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, qg = q / w.ng, entries = rows * qg;
    for (int k = wave; k < w.ng; k += THREADS / 64) {
        Moments t = {0.0f, 0.0f, 0.0f};
        for (int e = lane; e < entries; e += 64) t = join(t, sh[(e / qg) * q + k * qg + e % qg]);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1)
            t = join(t, {__shfl_xor(t.n, off, 64), __shfl_xor(t.mean, off, 64), __shfl_xor(t.m2, off, 64)});
        if (lane == 0) {
            const int part = g.tpg == 1 ? 0 : w.tile % g.tpg;
            float *o = partial + (((w.b * g.nchunk + w.chunk) * g.tpg + part) * g.groups + w.g0 + k) * 3;
            o[0] = t.n;
            o[1] = t.mean;
            o[2] = t.m2;
        }
    }
}

template <typename T, int V, bool SWISH>
__global__ __launch_bounds__(THREADS) void gn_apply_kernel(Geometry g, const T *__restrict__ x, const float *__restrict__ partial,
                                                           T *__restrict__ y, float *__restrict__ mean_out,
                                                           float *__restrict__ rstd_out)
{
    __shared__ float s_mean[THREADS], s_rstd[THREADS];
    const Place w = place_of(g, blockIdx.x, THREADS * V);
    const int np = g.nchunk * g.tpg;
    for (int k = threadIdx.x; k < w.ng; k += THREADS) {
        const float *pp = partial + (w.b * np * g.groups + w.g0 + k) * 3;
        Moments t = {0.0f, 0.0f, 0.0f};
        for (int i = 0; i < np; ++i, pp += (int64_t)g.groups * 3) t = join(t, {pp[0], pp[1], pp[2]});
        const float rstd = 1.0f / sqrtf(t.m2 / t.n + g.eps);
        s_mean[k] = t.mean;
        s_rstd[k] = rstd;
        if (w.chunk == 0 && (g.tpg == 1 || w.tile % g.tpg == 0)) {
            mean_out[w.b * g.groups + w.g0 + k] = t.mean;
            rstd_out[w.b * g.groups + w.g0 + k] = rstd;
        }
    }
    __syncthreads();
    const int q = w.width / V, rows = THREADS / q, r = threadIdx.x / q, cq = threadIdx.x - r * q;
    if (r >= rows) return;
    const int c = w.c0 + cq * V, k = g.tpg == 1 ? cq * V / g.gc : 0;
    float add[V], a[V], sh[V];
    load_chan<V>(g.shift ? g.shift + w.b * g.shift_sample : nullptr, c, 0.0f, add);
    load_chan<V>(g.gamma, c, 1.0f, a);
    load_chan<V>(g.beta, c, 0.0f, sh);
    const float mean = s_mean[k], rstd = s_rstd[k];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        add[j] -= mean;
        a[j] *= rstd;
    }
    const T *xp = x + w.b * g.x_sample + c;
    T *yp = y + w.b * g.pixels * g.channels + c;
#pragma unroll 4
    for (int64_t p = w.p0 + r; p < w.p1; p += rows) {
        float v[V];
        load_vec<T, V>(xp + p * g.x_pixel, v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float z = __builtin_fmaf(v[j] + add[j], a[j], sh[j]);
            v[j] = SWISH ? z * sigmoid(z) : z;
        }
        store_vec<T, V>(yp + p * g.channels, v);
    }
}

// xhat and dz of V channels of a pixel
template <int V, bool SWISH>
DEVI void grad_z(const float u[V], const float dy[V], const float add[V], float rstd, const float gamma[V], const float beta[V],
                 float xhat[V], float dz[V])
{
#pragma unroll
    for (int j = 0; j < V; ++j) {
        xhat[j] = (u[j] + add[j]) * rstd;
        dz[j] = dy[j];
        if constexpr (SWISH) {
            const float z = __builtin_fmaf(xhat[j], gamma[j], beta[j]), s = sigmoid(z);
            dz[j] *= s * __builtin_fmaf(z, 1.0f - s, 1.0f);
        }
    }
}

// Per-channel partial sums of dz, dz * xhat and (for the gradient of shift) xhat: three planes of (batch * nchunk, channels).
template <typename T, int V, bool SWISH>
__global__ __launch_bounds__(THREADS) void gn_grad_sums_kernel(Geometry g, const T *__restrict__ dy, const T *__restrict__ x,
                                                               const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                               float *__restrict__ sums, bool with_xhat)
{
    __shared__ float sh[THREADS * V];
    const Place w = place_of(g, blockIdx.x, THREADS * V);
    const int q = w.width / V, rows = THREADS / q, r = threadIdx.x / q, cq = threadIdx.x - r * q;
    float acc[3][V];
#pragma unroll
    for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) acc[i][j] = 0.0f;
    if (r < rows) {
        const int c = w.c0 + cq * V, grp = c / g.gc;
        const float mean = mean_in[w.b * g.groups + grp], rstd = rstd_in[w.b * g.groups + grp];
        float add[V], gamma[V], beta[V];
        load_chan<V>(g.shift ? g.shift + w.b * g.shift_sample : nullptr, c, 0.0f, add);
        load_chan<V>(g.gamma, c, 1.0f, gamma);
        load_chan<V>(g.beta, c, 0.0f, beta);
#pragma unroll
        for (int j = 0; j < V; ++j) add[j] -= mean;
        const T *xp = x + w.b * g.x_sample + c, *dp = dy + w.b * g.dy_sample + c;
#pragma unroll 4
        for (int64_t p = w.p0 + r; p < w.p1; p += rows) {
            float u[V], d[V], xhat[V], dz[V];
            load_vec<T, V>(xp + p * g.x_pixel, u);
            load_vec<T, V>(dp + p * g.dy_pixel, d);
            grad_z<V, SWISH>(u, d, add, rstd, gamma, beta, xhat, dz);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                acc[0][j] += dz[j];
                acc[1][j] = __builtin_fmaf(dz[j], xhat[j], acc[1][j]);
                acc[2][j] += xhat[j];
            }
        }
    }
    const int64_t plane = g.batch * g.nchunk * g.channels, row = (w.b * g.nchunk + w.chunk) * g.channels;
    for (int i = 0; i < (with_xhat ? 3 : 2); ++i) {
        __syncthreads();
        if (r < rows)
#pragma unroll
            for (int j = 0; j < V; ++j) sh[(r * q + cq) * V + j] = acc[i][j];
        __syncthreads();
        for (int c = threadIdx.x; c < w.width; c += THREADS) {
            float s = 0.0f;
            for (int k = 0; k < rows; ++k) s += sh[k * w.width + c];
            sums[i * plane + row + w.c0 + c] = s;
        }
    }
}

template <typename T, int V, bool SWISH>
__global__ __launch_bounds__(THREADS) void gn_grad_apply_kernel(Geometry g, const T *__restrict__ dy, const T *__restrict__ x,
                                                                const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                                const float *__restrict__ sums, T *__restrict__ dx,
                                                                float *__restrict__ dshift)
{
    __shared__ float s_a[THREADS], s_b[THREADS];
    const Place w = place_of(g, blockIdx.x, THREADS * V);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t plane = g.batch * g.nchunk * g.channels;
    const float *sb = sums + w.b * g.nchunk * g.channels;
    const float inv_n = 1.0f / ((float)g.pixels * (float)g.gc);
    for (int k = wave; k < w.ng; k += THREADS / 64) {
        const int gc0 = (w.g0 + k) * g.gc;
        float a = 0.0f, b = 0.0f;
        for (int c = lane; c < g.gc; c += 64) {
            float t0 = 0.0f, t1 = 0.0f;
            for (int i = 0; i < g.nchunk; ++i) {
                const float *o = sb + (int64_t)i * g.channels + gc0 + c;
                t0 += o[0];
                t1 += o[plane];
            }
            const float gm = g.gamma ? g.gamma[gc0 + c] : 1.0f;
            a = __builtin_fmaf(gm, t0, a);
            b = __builtin_fmaf(gm, t1, b);
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) {
            a += __shfl_xor(a, off, 64);
            b += __shfl_xor(b, off, 64);
        }
        if (lane == 0) {
            s_a[k] = a * inv_n;
            s_b[k] = b * inv_n;
        }
    }
    __syncthreads();
    if (dshift && w.chunk == 0) {
        for (int c = threadIdx.x; c < w.width; c += THREADS) {
            const int ch = w.c0 + c, k = g.tpg == 1 ? c / g.gc : 0;
            float t0 = 0.0f, t2 = 0.0f;
            for (int i = 0; i < g.nchunk; ++i) {
                t0 += sb[(int64_t)i * g.channels + ch];
                t2 += sb[2 * plane + (int64_t)i * g.channels + ch];
            }
            const float gm = g.gamma ? g.gamma[ch] : 1.0f, rstd = rstd_in[w.b * g.groups + ch / g.gc];
            dshift[w.b * g.channels + ch] = rstd * (gm * t0 - (float)g.pixels * s_a[k] - s_b[k] * t2);
        }
    }
    const int q = w.width / V, rows = THREADS / q, r = threadIdx.x / q, cq = threadIdx.x - r * q;
    if (r >= rows) return;
    const int c = w.c0 + cq * V, grp = c / g.gc, k = g.tpg == 1 ? cq * V / g.gc : 0;
    const float mean = mean_in[w.b * g.groups + grp], rstd = rstd_in[w.b * g.groups + grp], ga = s_a[k], gb = s_b[k];
    float add[V], gamma[V], beta[V];
    load_chan<V>(g.shift ? g.shift + w.b * g.shift_sample : nullptr, c, 0.0f, add);
    load_chan<V>(g.gamma, c, 1.0f, gamma);
    load_chan<V>(g.beta, c, 0.0f, beta);
#pragma unroll
    for (int j = 0; j < V; ++j) add[j] -= mean;
    const T *xp = x + w.b * g.x_sample + c, *dp = dy + w.b * g.dy_sample + c;
    T *op = dx + w.b * g.pixels * g.channels + c;
#pragma unroll 4
    for (int64_t p = w.p0 + r; p < w.p1; p += rows) {
        float u[V], d[V], xhat[V], dz[V];
        load_vec<T, V>(xp + p * g.x_pixel, u);
        load_vec<T, V>(dp + p * g.dy_pixel, d);
        grad_z<V, SWISH>(u, d, add, rstd, gamma, beta, xhat, dz);
#pragma unroll
        for (int j = 0; j < V; ++j) d[j] = rstd * (dz[j] * gamma[j] - ga - xhat[j] * gb);
        store_vec<T, V>(op + p * g.channels, d);
    }
}

// Column sums of (rows, cols): block (column tile of 64, split s) adds rows s, s + splits, ... to out[s][col].
__global__ __launch_bounds__(256) void gn_columns_kernel(const float *__restrict__ in, int64_t rows, int cols, int splits,
                                                         float *__restrict__ out)
{
    __shared__ float sh[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (col < cols)
        for (int64_t r = blockIdx.y + (int64_t)wave * splits; r < rows; r += 4 * (int64_t)splits) s += in[r * cols + col];
    sh[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && col < cols) out[(int64_t)blockIdx.y * cols + col] = (sh[0][lane] + sh[1][lane]) + (sh[2][lane] + sh[3][lane]);
}

constexpr int kSplits = 64;

int elem_bytes(int dtype) { return dtype == IDM_DT_F32 ? 4 : 2; }

// Vector width: at most 16 bytes, dividing a group, and aligned in every tensor of the call.
int vec_of(const idm_group_norm_desc &d, bool backward, std::initializer_list<const void *> ptrs)
{
    const int e = elem_bytes(d.dtype), gc = d.channels / d.groups;
    for (int v = 16 / e; v > 1; v >>= 1) {
        if (gc % v || d.channels % v || d.x_sample % v || d.x_pixel % v) continue;
        if (backward && (d.dy_sample % v || d.dy_pixel % v)) continue;
        bool ok = true;
        for (const void *p : ptrs) ok = ok && (uintptr_t)p % (size_t)(v * e) == 0;
        if (ok) return v;
    }
    return 1;
}

Geometry geometry_of(const idm_group_norm_desc &d, int v)
{
    Geometry g = {};
    g.batch = d.batch; g.pixels = d.pixels;
    g.x_sample = d.x_sample; g.x_pixel = d.x_pixel; g.dy_sample = d.dy_sample; g.dy_pixel = d.dy_pixel; g.shift_sample = d.shift_sample;
    g.channels = d.channels; g.groups = d.groups; g.gc = d.channels / d.groups;
    g.eps = d.eps;
    const int qg = g.gc / v;
    if (qg <= THREADS) {
        g.gpt = std::min(g.groups, THREADS / qg);
        g.tpg = 1;
        g.ntile = (g.groups + g.gpt - 1) / g.gpt;
    } else {
        g.gpt = 1;
        g.tpg = (qg + THREADS - 1) / THREADS;
        g.ntile = g.groups * g.tpg;
    }
    // enough workgroups to fill the chip, none with less than a few vectors per thread
    const int rows = std::max(1, THREADS / std::min(THREADS, g.gpt * qg));
    const int64_t most = std::max<int64_t>(1, g.pixels / (8 * rows)), want = (2048 + g.batch * g.ntile - 1) / (g.batch * g.ntile);
    int64_t n = std::max<int64_t>(1, std::min<int64_t>({most, want, 1024}));
    g.chunk = (g.pixels + n - 1) / n;
    g.nchunk = (int)((g.pixels + g.chunk - 1) / g.chunk);
    return g;
}

// The vector width depends on pointers, which the size query does not have: the smallest tiles (V = 1) and most chunks bound it.
size_t workspace_floats(const idm_group_norm_desc &d, bool backward)
{
    size_t most = 0;
    for (int v = 16 / elem_bytes(d.dtype); v >= 1; v >>= 1) {
        if ((d.channels / d.groups) % v) continue;
        const Geometry g = geometry_of(d, v);
        const size_t rows = (size_t)g.batch * g.nchunk;
        most = std::max(most, backward ? 3 * rows * g.channels : rows * g.tpg * g.groups * 3);
    }
    if (backward) most += (size_t)kSplits * d.channels + (d.shift_sample == 0 ? (size_t)d.batch * d.channels : 0);
    return most;
}

int check_desc(const idm_group_norm_desc *d, bool backward)
{
    if (!d) return idm_set_error(IDM_ERR_INVALID, "group norm: null descriptor");
    if (d->dtype != IDM_DT_F32 && d->dtype != IDM_DT_BF16 && d->dtype != IDM_DT_F16)
        return idm_set_error(IDM_ERR_INVALID, "group norm: unknown dtype");
    if (d->activation != IDM_ACT_NONE && d->activation != IDM_ACT_SWISH)
        return idm_set_error(IDM_ERR_INVALID, "group norm: unknown activation");
    if (d->batch < 0 || d->pixels < 0 || d->channels <= 0 || d->groups <= 0 || d->channels % d->groups)
        return idm_set_error(IDM_ERR_INVALID, "group norm: channels must be a positive multiple of groups, batch and pixels not negative");
    if (!(d->eps >= 0.0f) || std::isinf(d->eps)) return idm_set_error(IDM_ERR_INVALID, "group norm: eps must be finite and not negative");
    if (d->channels > (1 << 20) || d->pixels > ((int64_t)1 << 40) || d->batch > ((int64_t)1 << 31))
        return idm_set_error(IDM_ERR_INVALID, "group norm: more than 2^20 channels, 2^40 pixels or 2^31 samples");
    if (d->x_pixel < d->channels || (backward && d->dy_pixel < d->channels))
        return idm_set_error(IDM_ERR_INVALID, "group norm: a pixel's stride is less than its channels");
    if (d->x_sample < 0 || d->shift_sample < 0 || (backward && d->dy_sample < 0))
        return idm_set_error(IDM_ERR_INVALID, "group norm: negative stride");
    return IDM_OK;
}

int check_launch(const char *what)
{
    return hipGetLastError() == hipSuccess ? IDM_OK : idm_set_error(IDM_ERR_HIP, what);
}

template <typename T, int V>
int forward_launch(const idm_group_norm_desc &d, const Geometry &g, const void *x, void *y, float *mean, float *rstd, float *ws,
                   hipStream_t s)
{
    const int64_t blocks = g.batch * g.nchunk * g.ntile;
    if (blocks > 0x7fffffff) return idm_set_error(IDM_ERR_INVALID, "group norm: batch too large");
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), dim3((unsigned)blocks), dim3(THREADS), 0, s, g, (const T *)x, ws);
    if (d.activation == IDM_ACT_SWISH)
        hipLaunchKernelGGL((gn_apply_kernel<T, V, true>), dim3((unsigned)blocks), dim3(THREADS), 0, s, g, (const T *)x, ws, (T *)y, mean, rstd);
    else
        hipLaunchKernelGGL((gn_apply_kernel<T, V, false>), dim3((unsigned)blocks), dim3(THREADS), 0, s, g, (const T *)x, ws, (T *)y, mean, rstd);
    return check_launch("group norm: launch failed");
}

// out[c] = sum of column c of (rows, cols); part: kSplits * cols floats
void column_sums(const float *in, int64_t rows, int cols, float *part, float *out, hipStream_t s)
{
    const unsigned ct = (unsigned)((cols + 63) / 64);
    const int splits = (int)std::min<int64_t>(kSplits, (rows + 15) / 16);
    if (splits > 1) {
        hipLaunchKernelGGL(gn_columns_kernel, dim3(ct, (unsigned)splits), dim3(256), 0, s, in, rows, cols, splits, part);
        hipLaunchKernelGGL(gn_columns_kernel, dim3(ct, 1), dim3(256), 0, s, (const float *)part, (int64_t)splits, cols, 1, out);
    } else {
        hipLaunchKernelGGL(gn_columns_kernel, dim3(ct, 1), dim3(256), 0, s, in, rows, cols, 1, out);
    }
}

template <typename T, int V, bool SWISH>
int backward_launch(const Geometry &g, const void *dy, const void *x, const float *mean, const float *rstd, void *dx, float *dgamma,
                    float *dbeta, float *dshift, float *ws, hipStream_t s)
{
    const int64_t blocks = g.batch * g.nchunk * g.ntile, rows = g.batch * g.nchunk, plane = rows * g.channels;
    if (blocks > 0x7fffffff) return idm_set_error(IDM_ERR_INVALID, "group norm: batch too large");
    hipLaunchKernelGGL((gn_grad_sums_kernel<T, V, SWISH>), dim3((unsigned)blocks), dim3(THREADS), 0, s, g, (const T *)dy, (const T *)x, mean,
                       rstd, ws, dshift != nullptr);
    float *part = ws + 3 * plane, *per_sample = nullptr;
    if (dshift && g.shift_sample == 0) per_sample = part + (size_t)kSplits * g.channels;   // one row for all samples: summed below
    hipLaunchKernelGGL((gn_grad_apply_kernel<T, V, SWISH>), dim3((unsigned)blocks), dim3(THREADS), 0, s, g, (const T *)dy, (const T *)x, mean,
                       rstd, (const float *)ws, (T *)dx, per_sample ? per_sample : dshift);
    if (dbeta) column_sums(ws, rows, g.channels, part, dbeta, s);
    if (dgamma) column_sums(ws + plane, rows, g.channels, part, dgamma, s);
    if (per_sample) column_sums(per_sample, g.batch, g.channels, part, dshift, s);
    return check_launch("group norm backward: launch failed");
}

template <typename F> int by_type(int dtype, int v, F &&f)
{
    switch (dtype) {
    case IDM_DT_F32:
        return v == 4 ? f(float{}, std::integral_constant<int, 4>{}) : v == 2 ? f(float{}, std::integral_constant<int, 2>{})
                                                                              : f(float{}, std::integral_constant<int, 1>{});
    case IDM_DT_BF16:
        return v == 8   ? f(__bf16{}, std::integral_constant<int, 8>{})
               : v == 4 ? f(__bf16{}, std::integral_constant<int, 4>{})
               : v == 2 ? f(__bf16{}, std::integral_constant<int, 2>{})
                        : f(__bf16{}, std::integral_constant<int, 1>{});
    default:
        return v == 8   ? f(_Float16{}, std::integral_constant<int, 8>{})
               : v == 4 ? f(_Float16{}, std::integral_constant<int, 4>{})
               : v == 2 ? f(_Float16{}, std::integral_constant<int, 2>{})
                        : f(_Float16{}, std::integral_constant<int, 1>{});
    }
}

}  // namespace

extern "C" {

int idm_group_norm_workspace(const idm_group_norm_desc *d, int backward, size_t *bytes)
{
    const int rc = check_desc(d, backward != 0);
    if (rc != IDM_OK) return rc;
    if (!bytes) return idm_set_error(IDM_ERR_INVALID, "group norm: null size");
    *bytes = d->batch == 0 || d->pixels == 0 ? 0 : workspace_floats(*d, backward != 0) * sizeof(float);
    return IDM_OK;
}

int idm_group_norm_forward(int device, const idm_group_norm_desc *d, const void *x_dev, const float *gamma_dev, const float *beta_dev,
                           const float *shift_dev, void *y_dev, float *mean_dev, float *rstd_dev, void *workspace_dev,
                           size_t workspace_bytes, void *stream)
{
    int rc = check_desc(d, false);
    if (rc != IDM_OK) return rc;
    if (d->batch == 0 || d->pixels == 0) return IDM_OK;
    if (!x_dev || !y_dev || !mean_dev || !rstd_dev || !workspace_dev) return idm_set_error(IDM_ERR_INVALID, "group norm: null argument");
    if (workspace_bytes < workspace_floats(*d, false) * sizeof(float)) return idm_set_error(IDM_ERR_INVALID, "group norm: workspace too small");
    if (hipSetDevice(device) != hipSuccess) return idm_set_error(IDM_ERR_HIP, "group norm: no such device");
    const int v = vec_of(*d, false, {x_dev, y_dev});
    Geometry g = geometry_of(*d, v);
    g.gamma = gamma_dev; g.beta = beta_dev; g.shift = shift_dev;
    return by_type(d->dtype, v, [&](auto t, auto w) {
        return forward_launch<decltype(t), decltype(w)::value>(*d, g, x_dev, y_dev, mean_dev, rstd_dev, (float *)workspace_dev, (hipStream_t)stream);
    });
}

int idm_group_norm_backward(int device, const idm_group_norm_desc *d, const void *dy_dev, const void *x_dev, const float *mean_dev,
                            const float *rstd_dev, const float *gamma_dev, const float *beta_dev, const float *shift_dev, void *dx_dev,
                            float *dgamma_dev, float *dbeta_dev, float *dshift_dev, void *workspace_dev, size_t workspace_bytes,
                            void *stream)
{
    int rc = check_desc(d, true);
    if (rc != IDM_OK) return rc;
    if (d->batch == 0 || d->pixels == 0) return IDM_OK;
    if (!dy_dev || !x_dev || !mean_dev || !rstd_dev || !dx_dev || !workspace_dev)
        return idm_set_error(IDM_ERR_INVALID, "group norm backward: null argument");
    if (workspace_bytes < workspace_floats(*d, true) * sizeof(float))
        return idm_set_error(IDM_ERR_INVALID, "group norm backward: workspace too small");
    if (hipSetDevice(device) != hipSuccess) return idm_set_error(IDM_ERR_HIP, "group norm backward: no such device");
    const int v = vec_of(*d, true, {dy_dev, x_dev, dx_dev});
    Geometry g = geometry_of(*d, v);
    g.gamma = gamma_dev; g.beta = beta_dev; g.shift = shift_dev;
    return by_type(d->dtype, v, [&](auto t, auto w) {
        auto *f = d->activation == IDM_ACT_SWISH ? &backward_launch<decltype(t), decltype(w)::value, true>
                                                 : &backward_launch<decltype(t), decltype(w)::value, false>;
        return f(g, dy_dev, x_dev, mean_dev, rstd_dev, dx_dev, dgamma_dev, dbeta_dev, dshift_dev, (float *)workspace_dev, (hipStream_t)stream);
    });
}

}  // extern "C"
