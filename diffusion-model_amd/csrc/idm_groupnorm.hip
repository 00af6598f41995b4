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
// All arithmetic between the load and the store is float32; y and dx are rounded once, to the type of x.  Sums run in a fixed order,
// no atomics: equal inputs give equal bits.
//
// Memory bounds both directions: x in, y out (forward), x and dy in, dx out (backward); a large copy on this card moves 4.9 TB/s.  Next
// comes the vector unit: a value costs about 18 of its slots forward (exp and rcp are four each) and 32 backward (1 024 x 14 x 14 x 192
// bf16: 18 and 32 us), half to two thirds of the time of its memory.  Two forms:
//   units   one launch; a workgroup holds a channel tile of one sample (or of several small ones) in registers, so memory is touched
//           once.  Backward adds a small launch for the weight gradients.  Forward 1 024 x 28 x 28 x 96 bf16: 77-83 us (3.9 TB/s; 105 in
//           chunks); 4 096 x 7 x 7 x 128 bf16 22 us (4.6 TB/s; 42); backward 1 024 x 14 x 14 x 192 bf16: 60-63 us and 5 of that launch (3.5 TB/s; 93).
//   chunks  two launches over chunks of pixels: partial sums, then their join and the result; x (and dy) are read twice, the second
//           time mostly from the caches.  For maps that a compute unit cannot hold, few large ones, and calls whose pointers, strides
//           or channels are no multiples of 16 bytes.  4 x 128 x 128 x 64 fp16: 14 us forward; 3 x 127 x 125 x 64 fp16: 15 us backward.
// plan_unit() chooses.
#include "../../include/isingdiff.h"
#include "idm_internal.h"
#include "idm_device.h"

#include <algorithm>
#include <cmath>

namespace {

constexpr int THREADS = 256;

template <typename T, int V> struct VecOf { typedef __attribute__((ext_vector_type(V))) T type; };
template <typename T> struct VecOf<T, 1> { typedef T type; };

template <typename T, int V> DEVI void widen_vec(const typename VecOf<T, V>::type &v, float out[V])
{
    if constexpr (V == 1) {
        out[0] = (float)v;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) out[j] = (float)v[j];
    }
}

// V consecutive channels as float32
template <typename T, int V> DEVI void load_vec(const T *p, float out[V]) { widen_vec<T, V>(*(const typename VecOf<T, V>::type *)p, out); }

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

// i / n from inv = 1 / n, for the small numbers of a workgroup (i < 2^13, n <= 2^10): (i + 1/2) * inv is off by less than 2^-10 / n, and the
// nearest integer 1 / 2n away
DEVI int quotient(int i, float inv) { return (int)(((float)i + 0.5f) * inv); }

// s / n with r near 1 / n: exact wherever the quotient is a float (a constant group's mean is its value)
DEVI float over(float s, float n, float r)
{
    const float m = s * r;
    return __builtin_fmaf(__builtin_fmaf(-m, n, s), r, m);
}

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

// The union of many sets, spread over `lanes` lanes: count and mean first, then the squared distances from that mean; no division but
// one.  get(i) is set i.
template <typename F> DEVI Moments join_all(int sets, int lane, int lanes, F &&get)
{
    float n = 0.0f, sum = 0.0f, m2 = 0.0f;
#pragma unroll 4
    for (int i = lane; i < sets; i += lanes) {
        const Moments t = get(i);
        n += t.n;
        sum = __builtin_fmaf(t.n, t.mean, sum);
    }
    for (int off = lanes >> 1; off >= 1; off >>= 1) {
        n += __shfl_xor(n, off, 64);
        sum += __shfl_xor(sum, off, 64);
    }
    const float mean = sum / n;
#pragma unroll 4
    for (int i = lane; i < sets; i += lanes) {
        const Moments t = get(i);
        const float d = t.mean - mean;
        m2 += __builtin_fmaf(t.n * d, d, t.m2);
    }
    for (int off = lanes >> 1; off >= 1; off >>= 1) m2 += __shfl_xor(m2, off, 64);
    return {n, mean, m2};
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

// Grid: x chunks and tiles, y and z samples
DEVI Place place_of(const Geometry &g, int part_channels)
{
    Place w;
    w.chunk = (int)blockIdx.x / g.ntile;
    w.tile = (int)blockIdx.x - w.chunk * g.ntile;
    w.b = (int64_t)blockIdx.z * gridDim.y + blockIdx.y;
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

// ---- chunks ---------------------------------------------------------------------------------------------------------------
//
// Partial statistics of (sample, chunk, tile): (n, mean, m2) of each group at ((b * groups + group) * nchunk + chunk) * tpg + part,
// so that the lanes which join a group read neighbours.
template <typename T, int V>
__global__ __launch_bounds__(THREADS) void gn_stats_kernel(Geometry g, const T *__restrict__ x, float *__restrict__ partial)
{
    constexpr int U = 4;   // vectors taken together: their mean first, then the squared distances from it
    __shared__ Moments sh[THREADS];
    const Place w = place_of(g, THREADS * V);
    if (w.b >= g.batch) return;
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
    const float inv_qg = 1.0f / (float)qg;
    for (int k = wave; k < w.ng; k += THREADS / 64) {
        const Moments t = join_all(entries, lane, 64, [&](int e) {
            const int er = quotient(e, inv_qg);
            return sh[er * q + k * qg + e - er * qg];
        });
        if (lane == 0) {
            const int part = g.tpg == 1 ? 0 : w.tile % g.tpg, np = g.nchunk * g.tpg;
            float *o = partial + ((w.b * g.groups + w.g0 + k) * np + w.chunk * g.tpg + part) * 3;
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
    const Place w = place_of(g, THREADS * V);
    if (w.b >= g.batch) return;
    // the partials of a group are joined by `lanes` lanes, all groups of the tile at once where there are few
    const int np = g.nchunk * g.tpg;
    int lanes = 64;
    while (lanes > 8 && lanes * w.ng > THREADS) lanes >>= 1;
    const int lane = threadIdx.x & (lanes - 1);
    for (int k0 = 0; k0 < w.ng; k0 += THREADS / lanes) {
        const int k = k0 + (int)threadIdx.x / lanes;
        const float *pp = partial + (w.b * g.groups + w.g0 + k) * np * 3;
        const Moments t = join_all(k < w.ng ? np : 0, lane, lanes, [&](int i) {
            const float *o = pp + i * 3;
            return Moments{o[0], o[1], o[2]};
        });
        if (k >= w.ng || lane) continue;
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

// Column sums of one plane (rows, cols) for 16 columns: rows split, split + splits, ... by 256 threads
DEVI void sum_columns(const float *in, int64_t rows, int cols, int col0, int split, int splits, float *out)
{
    __shared__ float sh[16][17];
    const int lane = threadIdx.x & 15, row = threadIdx.x >> 4, col = col0 + lane;
    const float *p = in + col;
    float s = 0.0f;
    if (col < cols)
#pragma unroll 8
        for (int64_t r = split + (int64_t)row * splits; r < rows; r += 16 * (int64_t)splits) s += p[r * cols];
    sh[row][lane] = s;
    __syncthreads();
    if (row == 0 && col < cols) {
        float t[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) t[k] = sh[k][lane];
#pragma unroll
        for (int w = 8; w >= 1; w >>= 1)
#pragma unroll
            for (int k = 0; k < w; ++k) t[k] += t[k + w];
        out[(int64_t)split * cols + col] = t[0];
    }
}

constexpr int kLoads = 4;

// Calls use(p, vectors of x, vectors of dy) for a thread's pixels p, p + rows, ... (kLoads of them, below p1).  The last ones are loaded
// together as well, with the first in place of those behind the end: a loop of single loads for them took 56 of 80 us on 300 x 28 x 28 x
// 96 bf16.
template <typename T, int V, typename F>
DEVI void for_pixels(const Place &w, int r, int rows, const T *x, int64_t xpitch, const T *dy, int64_t dpitch, F &&use)
{
    for (int64_t p = w.p0 + r; p < w.p1; p += kLoads * (int64_t)rows) {
        typename VecOf<T, V>::type u[kLoads], d[kLoads];
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const int64_t at = p + k * (int64_t)rows, from = at < w.p1 ? at : p;
            u[k] = *(const typename VecOf<T, V>::type *)(x + from * xpitch);
            d[k] = *(const typename VecOf<T, V>::type *)(dy + from * dpitch);
        }
        use(p, u, d);
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

// Sums over the rows of buf, whose value (row, column) is at at(row, column): done(c, sum) by one thread for each column.  Needs a
// barrier before and leaves with one.
template <typename G, typename F> DEVI void sum_rows(float *buf, int rows, int width, G &&at, F &&done)
{
    const int TH = (int)blockDim.x, split = TH / width < rows ? TH / width : rows;
    if (split > 1) {
        const int c = threadIdx.x % width, s = threadIdx.x / width;
        float t = 0.0f;
        if (s < split)
            for (int k = s; k < rows; k += split) t += buf[at(k, c)];
        __syncthreads();
        if (s < split) buf[at(s, c)] = t;
        __syncthreads();
        rows = split;
    }
    for (int c = threadIdx.x; c < width; c += TH) {
        float t = 0.0f;
        for (int k = 0; k < rows; ++k) t += buf[at(k, c)];
        done(c, t);
    }
    __syncthreads();
}

// Per-channel partial sums of dz, dz * xhat and (for the gradient of shift) xhat: three planes of (batch * nchunk, channels).
template <typename T, int V, bool SWISH>
__global__ __launch_bounds__(THREADS) void gn_grad_sums_kernel(Geometry g, const T *__restrict__ dy, const T *__restrict__ x,
                                                               const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                               float *__restrict__ sums, float2 *__restrict__ groups, bool with_xhat)
{
    __shared__ float sh[THREADS * V], by_channel[2][THREADS * V];
    const Place w = place_of(g, THREADS * V);
    if (w.b >= g.batch) return;
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
        for_pixels<T, V>(w, r, rows, xp, g.x_pixel, dp, g.dy_pixel, [&](int64_t p, auto &raw, auto &up) {
#pragma unroll
            for (int k = 0; k < kLoads; ++k) {
                if (p + k * (int64_t)rows >= w.p1) continue;
                float u[V], d[V], xhat[V], dz[V];
                widen_vec<T, V>(raw[k], u);
                widen_vec<T, V>(up[k], d);
                grad_z<V, SWISH>(u, d, add, rstd, gamma, beta, xhat, dz);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    acc[0][j] += dz[j];
                    acc[1][j] = __builtin_fmaf(dz[j], xhat[j], acc[1][j]);
                    acc[2][j] += xhat[j];
                }
            }
        });
    }
    const int64_t plane = g.batch * g.nchunk * g.channels, row = (w.b * g.nchunk + w.chunk) * g.channels;
    for (int i = 0; i < (with_xhat ? 3 : 2); ++i) {
        if (r < rows)
#pragma unroll
            for (int j = 0; j < V; ++j) sh[(r * q + cq) * V + j] = acc[i][j];
        __syncthreads();
        sum_rows(sh, rows, w.width, [&](int k, int c) { return k * w.width + c; }, [&](int c, float s) {
            sums[i * plane + row + w.c0 + c] = s;
            if (i < 2) by_channel[i][c] = (g.gamma ? g.gamma[w.c0 + c] : 1.0f) * s;
        });
    }
    // a group's share of this chunk: the next kernel reads these instead of every channel's
    const int part = g.tpg == 1 ? 0 : w.tile % g.tpg, per = g.tpg == 1 ? g.gc : w.width;
    for (int k = threadIdx.x; k < w.ng; k += THREADS) {
        float2 t = {0.0f, 0.0f};
        for (int c = k * per; c < (k + 1) * per; ++c) {
            t.x += by_channel[0][c];
            t.y += by_channel[1][c];
        }
        groups[(w.b * g.groups + w.g0 + k) * (g.nchunk * g.tpg) + w.chunk * g.tpg + part] = t;
    }
}

template <typename T, int V, bool SWISH>
__global__ __launch_bounds__(THREADS) void gn_grad_apply_kernel(Geometry g, const T *__restrict__ dy, const T *__restrict__ x,
                                                                const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                                                const float *__restrict__ sums, const float2 *__restrict__ groups,
                                                                T *__restrict__ dx, float *__restrict__ dshift, float *dbeta, float *dgamma)
{
    __shared__ float s_a[THREADS], s_b[THREADS];
    if ((int)blockIdx.x >= g.nchunk * g.ntile) {   // blocks behind the chunks add up the weight gradients
        if (blockIdx.y || blockIdx.z) return;
        const int64_t rows = g.batch * g.nchunk;
        const int at = ((int)blockIdx.x - g.nchunk * g.ntile) * 16, per = (g.channels + 15) / 16 * 16, plane = at >= per;
        float *out = plane ? dgamma : dbeta;
        if (out) sum_columns(sums + plane * rows * g.channels, rows, g.channels, at - plane * per, 0, 1, out);
        return;
    }
    const Place w = place_of(g, THREADS * V);
    if (w.b >= g.batch) return;
    const int64_t plane = g.batch * g.nchunk * g.channels;
    const float *sb = sums + w.b * g.nchunk * g.channels;
    const float inv_n = 1.0f / ((float)g.pixels * (float)g.gc);
    const int np = g.nchunk * g.tpg;
    int lanes = 64;
    while (lanes > 8 && lanes * w.ng > THREADS) lanes >>= 1;
    const int lane = threadIdx.x & (lanes - 1);
    for (int k0 = 0; k0 < w.ng; k0 += THREADS / lanes) {
        const int k = k0 + (int)threadIdx.x / lanes;
        float2 t = {0.0f, 0.0f};
        if (k < w.ng) {
            const float2 *pp = groups + (w.b * g.groups + w.g0 + k) * np;
#pragma unroll 4
            for (int i = lane; i < np; i += lanes) {
                const float2 o = pp[i];
                t.x += o.x;
                t.y += o.y;
            }
        }
        for (int off = lanes >> 1; off >= 1; off >>= 1) {
            t.x += __shfl_xor(t.x, off, 64);
            t.y += __shfl_xor(t.y, off, 64);
        }
        if (k < w.ng && lane == 0) {
            s_a[k] = t.x * inv_n;
            s_b[k] = t.y * inv_n;
        }
    }
    __syncthreads();
    if (dshift && w.chunk == 0) {
        for (int c = threadIdx.x; c < w.width; c += THREADS) {
            const int ch = w.c0 + c, k = g.tpg == 1 ? c / g.gc : 0;
            float t0 = 0.0f, t2 = 0.0f;
#pragma unroll 8
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
    for_pixels<T, V>(w, r, rows, xp, g.x_pixel, dp, g.dy_pixel, [&](int64_t p, auto &raw, auto &up) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            if (p + k * (int64_t)rows >= w.p1) continue;
            float u[V], d[V], xhat[V], dz[V];
            widen_vec<T, V>(raw[k], u);
            widen_vec<T, V>(up[k], d);
            grad_z<V, SWISH>(u, d, add, rstd, gamma, beta, xhat, dz);
#pragma unroll
            for (int j = 0; j < V; ++j) d[j] = rstd * (dz[j] * gamma[j] - ga - xhat[j] * gb);
            store_vec<T, V>(op + (p + k * (int64_t)rows) * g.channels, d);
        }
    });
}

// ---- one launch: a unit (sample, channel tile) held in the registers of one workgroup ---------------------------------
//
// Sixteen bytes of a pixel are V consecutive channels; thread (r, cq) holds vector cq of pixels r, r + rows, ... (at most NV).  A
// vector is cut into P pieces that never straddle a group: P = 1 where a group is whole vectors, 2 where half vectors fit, else
// V.  x is read once; mean, then the squared distances from it, both over the registers.

typedef __attribute__((ext_vector_type(4))) unsigned u32x4;

template <typename T> constexpr int vec16 = 16 / (int)sizeof(T);

// The values of a raw vector.  The empty asm keeps the compiler from holding the widened copy between two uses.
template <typename T> DEVI void widen(u32x4 raw, float out[vec16<T>])
{
    asm volatile("" : "+v"(raw));
    const auto v = __builtin_bit_cast(typename VecOf<T, vec16<T>>::type, raw);
#pragma unroll
    for (int j = 0; j < vec16<T>; ++j) out[j] = (float)v[j];
}

template <typename T> DEVI u32x4 narrow(const float in[vec16<T>])
{
    typename VecOf<T, vec16<T>>::type v;
#pragma unroll
    for (int j = 0; j < vec16<T>; ++j) v[j] = (T)in[j];
    return __builtin_bit_cast(u32x4, v);
}

// A block's memory as a buffer of kNowhere bytes from p on: the plan takes no unit that reaches so far, and a load at kNowhere gives
// zero, a store there is dropped, so pixels that a thread does not have need no branch.  The whole offset is in the checked
// (vector) part.
constexpr int kNowhere = 1 << 30;
DEVI __amdgpu_buffer_rsrc_t unit_buffer(const void *p, int64_t bytes)
{
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)bytes, 0x00020000);
}
DEVI u32x4 load16(__amdgpu_buffer_rsrc_t b, int at) { return __builtin_amdgcn_raw_buffer_load_b128(b, at, 0, 0); }
DEVI void store16(__amdgpu_buffer_rsrc_t b, int at, u32x4 v) { __builtin_amdgcn_raw_buffer_store_b128(v, b, at, 0, 0); }

// A block is `pack` samples times one tile of ng groups; a sample's part is rows * q threads (`seats`), row r has pixels r, r + rows, ...:
// full of them, one more where r < more.
struct UnitArgs {
    int64_t batch, x_sample, x_pixel, dy_sample, dy_pixel, shift_sample;
    int pixels, channels, groups, gc, ng, q, qg, rows, full, more, seats, pack, swish;
    float inv_q, inv_qg, inv_ng, inv_seats, eps, n, inv_n;   // n: values of a group
    const float *gamma, *beta, *shift;
};
constexpr int kTileVecs = 64;   // vectors of a tile, unless one group (or the fewest whole groups that are whole vectors) is wider

// V consecutive float32 from a 16-byte aligned place
template <int V> DEVI void load_chan16(const float *p, int c, float missing, float out[V])
{
#pragma unroll
    for (int i = 0; i < V; i += 4) {
        const f32x4 v = p ? *(const f32x4 *)(p + c + i) : f32x4{missing, missing, missing, missing};
#pragma unroll
        for (int j = 0; j < 4; ++j) out[i + j] = v[j];
    }
}

// sum += the values of each of a vector's P pieces (1 or 2), squares += their squares, both in float32 and two values at a time
template <int P> DEVI void add_pairs(u32x4 raw, _Float16, float sum[P], float squares[P])
{
    typedef __attribute__((ext_vector_type(2))) _Float16 half2_;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned w = raw[j];   // (a copy: the cast of an element itself takes the first one)
        const half2_ v = __builtin_bit_cast(half2_, w);
        sum[j * P / 4] = __builtin_amdgcn_fdot2(v, half2_{1, 1}, sum[j * P / 4], false);
        squares[j * P / 4] = __builtin_amdgcn_fdot2(v, v, squares[j * P / 4], false);
    }
}
template <int P> DEVI void add_pairs(u32x4 raw, __bf16, float sum[P], float squares[P])
{
    typedef __attribute__((ext_vector_type(2))) __bf16 bf2;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const unsigned w = raw[j];
        const bf2 v = __builtin_bit_cast(bf2, w);
        sum[j * P / 4] = __builtin_amdgcn_fdot2_f32_bf16(v, bf2{(__bf16)1.0f, (__bf16)1.0f}, sum[j * P / 4], false);
        squares[j * P / 4] = __builtin_amdgcn_fdot2_f32_bf16(v, v, squares[j * P / 4], false);
    }
}

struct Seat {
    int64_t b;                 // sample
    int sub, r, cq, c, mine;   // sample of the pack, row, vector of the row, its first channel, pixels
    bool active;
};
template <int V> DEVI Seat seat_of(const UnitArgs &g, int64_t pack, int tile)
{
    Seat s;
    s.sub = quotient(threadIdx.x, g.inv_seats);
    const int l = threadIdx.x - s.sub * g.seats;
    s.r = quotient(l, g.inv_q);
    s.cq = l - s.r * g.q;
    s.c = (tile * g.q + s.cq) * V;
    s.b = pack * g.pack + s.sub;
    s.active = s.sub < g.pack && s.b < g.batch;
    s.mine = s.active ? g.full + (s.r < g.more) : 0;
    return s;
}

// Joins the pieces of each group of the block: `lanes` (a power of two) lanes take one group together, as many as let all groups be
// joined at once, four at least (2 x 100 x 24 in 3-channel groups, bf16, forward: 8.4 us; 15.4 with 64 lanes to each in turn).  load(entry of part, row) and
// add work on a lane's running value, done(sub, group of the tile, value) runs on one lane of each group.  Pieces of a group are qg
// consecutive ones of each row of `row` pieces.
template <typename A, typename B, typename C> DEVI void fold_groups(const UnitArgs &g, int P, A &&first, B &&second, C &&done)
{
    const int entries = g.rows * g.qg, row = g.q * P, all = g.pack * g.ng;
    int lanes = 1;
    while (lanes < 64 && lanes < entries) lanes <<= 1;
    while (lanes > 4 && lanes * all > (int)blockDim.x) lanes >>= 1;
    const int lane = threadIdx.x & (lanes - 1), step = (int)blockDim.x / lanes;
    for (int k0 = 0; k0 < all; k0 += step) {
        const int k = k0 + (int)threadIdx.x / lanes, sub = quotient(k, g.inv_ng), grp = k - sub * g.ng;
        const bool on = k < all;
        const int base = sub * g.seats * P + grp * g.qg;
        auto sum = [&](auto &&term) {
            float2 t = {0.0f, 0.0f};
            if (on)
                for (int e = lane; e < entries; e += lanes) {
                    const int r = quotient(e, g.inv_qg);
                    term(t, base + r * row + e - r * g.qg, r);
                }
            for (int w = lanes >> 1; w >= 1; w >>= 1) {
                t.x += __shfl_xor(t.x, w, 64);
                t.y += __shfl_xor(t.y, w, 64);
            }
            return t;
        };
        const float2 a = sum(first);
        const float2 b = second(a, sum);
        if (on && lane == 0) done(sub, grp, k, b);
    }
}

// Grid: x samples (or packs) that are neighbours, y tiles, z the next ones.  Consecutive blocks go to the eight dies in turn, so
// x = 8 keeps the tiles of one sample on one die, whose cache joins their parts of a line.
template <typename T, int P, int TH, int NV>
__global__ __launch_bounds__(TH) void gn_unit_forward_kernel(UnitArgs g, const T *__restrict__ x, T *__restrict__ y,
                                                             float *__restrict__ mean_out, float *__restrict__ rstd_out)
{
    constexpr int V = vec16<T>, PS = V / P, E = sizeof(T);
    extern __shared__ float lds[];
    float2 *const part = (float2 *)lds, *const stat = part + blockDim.x * P;
    const int64_t pack = (int64_t)blockIdx.z * gridDim.x + blockIdx.x, b0 = pack * g.pack;
    if (b0 >= g.batch) return;
    const Seat s = seat_of<V>(g, pack, blockIdx.y);
    const int c0 = blockIdx.y * g.q * V;
    u32x4 raw[NV];
    {
        const auto xb = unit_buffer(x + b0 * g.x_sample + c0, kNowhere);
        const int pitch = (int)g.x_pixel * E, at = (int)(s.sub * g.x_sample) * E + s.r * pitch + s.cq * 16;
#pragma unroll
        for (int k = 0; k < NV; ++k) raw[k] = load16(xb, k < s.mine ? at + k * g.rows * pitch : kNowhere);
    }
    float add[V], mean[P] = {}, m2[P] = {};
    load_chan16<V>(g.shift && s.active ? g.shift + s.b * g.shift_sample : nullptr, s.c, 0.0f, add);
    // The thread's own mean and squared distances from it, then the group's from all of its threads'.  A sum of squares around zero
    // would lose the variance of values far from it, so the distances are summed; only where 16-bit values come without a shift,
    // and the thread's mean turns out to be within four of its deviations, do sum and sum of squares (two instructions for two
    // values instead of eight) stand: that loses less than five bits.  Each piece decides for itself: what one group holds does not change
    // another's bits.
    const float own = (float)(s.mine ? s.mine * PS : 1), share = __builtin_amdgcn_rcpf(own);
    bool sure[P] = {}, all = false;
    if constexpr (E == 2 && P <= 2) {
        if (!g.shift) {
            float sum[P], squares[P];
#pragma unroll
            for (int i = 0; i < P; ++i) sum[i] = squares[i] = 0.0f;
#pragma unroll
            for (int k = 0; k < NV; ++k) add_pairs<P>(raw[k], T{}, sum, squares);
            all = true;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                mean[i] = over(sum[i], own, share);
                m2[i] = squares[i] - sum[i] * mean[i];
                sure[i] = squares[i] < 0x1p126f && !(m2[i] * 16.0f < sum[i] * mean[i]);   // (not where squares overflow)
                all = all && sure[i];
            }
        }
    }
    if (!all) {
        float mean_[P], m2_[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            mean_[i] = m2_[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < PS; ++j) mean_[i] += add[i * PS + j];
            mean_[i] *= (float)s.mine;
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            float v[V];
            widen<T>(raw[k], v);
#pragma unroll
            for (int j = 0; j < V; ++j) mean_[j / PS] += v[j];
        }
#pragma unroll
        for (int i = 0; i < P; ++i) mean_[i] = over(mean_[i], own, share);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (k >= s.mine) continue;
            float v[V];
            widen<T>(raw[k], v);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = v[j] + (add[j] - mean_[j / PS]);
                m2_[j / PS] = __builtin_fmaf(d, d, m2_[j / PS]);
            }
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            mean[i] = sure[i] ? mean[i] : mean_[i];
            m2[i] = sure[i] ? m2[i] : m2_[i];
        }
    }
#pragma unroll
    for (int i = 0; i < P; ++i) part[threadIdx.x * P + i] = float2{mean[i], m2[i]};
    __syncthreads();
    const auto count = [&](int r) { return (float)((g.full + (r < g.more)) * PS); };
    fold_groups(
        g, P, [&](float2 &t, int at, int r) { t.x = __builtin_fmaf(count(r), part[at].x, t.x); },
        [&](float2 sum, auto &&again) {
            const float m = over(sum.x, g.n, g.inv_n);
            const float2 d2 = again([&](float2 &t, int at, int r) {
                const float2 o = part[at];
                const float d = o.x - m;
                t.x += __builtin_fmaf(count(r) * d, d, o.y);
            });
            return float2{m, 1.0f / sqrtf(d2.x * g.inv_n + g.eps)};
        },
        [&](int sub, int grp, int k, float2 v) {
            stat[k] = v;
            if (b0 + sub < g.batch) {
                const int64_t o = (b0 + sub) * g.groups + blockIdx.y * g.ng + grp;
                mean_out[o] = v.x;
                rstd_out[o] = v.y;
            }
        });
    __syncthreads();
    // z = (x + add) * a + sh in float32.  (Never add * a folded into sh, one instruction for a value less: its rounding is 2^-24 of |mean| rstd,
    // which has no bound where a group is nearly constant, 0.12 of y for 60 000 and eps = 1e-3.  1 024 x 784 x 96 bf16 89 us, folded 88.)
    float a[V], sh[V];
    load_chan16<V>(s.active ? g.gamma : nullptr, s.c, 1.0f, a);
    load_chan16<V>(s.active ? g.beta : nullptr, s.c, 0.0f, sh);
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const float2 t = stat[s.active ? s.sub * g.ng + quotient(s.cq * P + i, g.inv_qg) : 0];
#pragma unroll
        for (int j = i * PS; j < (i + 1) * PS; ++j) {
            add[j] -= t.x;
            a[j] *= t.y;
        }
    }
    const int pitch = g.channels * E, at = (s.sub * g.pixels + s.r) * pitch + s.cq * 16;
    const auto yb = unit_buffer(y + b0 * g.pixels * g.channels + c0, kNowhere);
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        float v[V];
        widen<T>(raw[k], v);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = __builtin_fmaf(v[j] + add[j], a[j], sh[j]);
        if (g.swish)
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] *= sigmoid(v[j]);
        store16(yb, k < s.mine ? at + k * g.rows * pitch : kNowhere, narrow<T>(v));
    }
}

// Backward of a unit: x and dy are read once; dz stays in the registers in float32 between the group sums and dx.  A block walks
// over packs `walker`, walker + walkers, ... of one tile and keeps the tile's weight gradients (in LDS, a thread's own sums); it
// writes them once, as row `walker` of two planes (walkers, channels).
template <typename T, int P, int TH, int NV>
__global__ __launch_bounds__(TH, NV == 8 ? sizeof(T) == 4 && P == 1 ? 3 : 2 : sizeof(T) == 4 ? 4 : 3) void gn_unit_backward_kernel(
    UnitArgs g, int walkers, const T *__restrict__ dy, const T *__restrict__ x, const float *__restrict__ mean_in,
    const float *__restrict__ rstd_in, T *__restrict__ dx, float *__restrict__ sums, float *__restrict__ dshift)
{
    constexpr int V = vec16<T>, PS = V / P, E = sizeof(T);
    constexpr bool AHEAD = E == 2 && NV == 4 && P <= 2;
    extern __shared__ __attribute__((aligned(16))) float lds[];
    float *const total[2] = {lds, lds + blockDim.x * V}, *const buf = lds + 2 * blockDim.x * V;
    float2 *const part = (float2 *)buf, *const stat = (float2 *)(buf + blockDim.x * (V > 2 * P ? V : 2 * P));
    const int walker = blockIdx.z * gridDim.x + blockIdx.x;
    if (walker >= walkers) return;
    // A thread's V values stand in 16-byte pieces, [V / 4][threads][4], so that a wavefront's accesses meet no bank twice.  Written one
    // by one with eight vectors: registers that are neighbours are one demand too many there (512 x 784 x 64 float32: 85 us, 88).
    const auto own = [&](float *b, const float v[V], bool add) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            float *const q = b + (j / 4 * (int)blockDim.x + (int)threadIdx.x) * 4;
            if constexpr (NV == 4) {
                const f32x4 w = {v[j], v[j + 1], v[j + 2], v[j + 3]};
                *(f32x4 *)q = add ? *(const f32x4 *)q + w : w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) q[i] = add ? q[i] + v[j + i] : v[j + i];
            }
        }
    };
    const auto at = [&](int row, int c) { return ((c % V) / 4 * (int)blockDim.x + row * g.q + c / V) * 4 + c % 4; };
    const int width = g.q * V, c0 = blockIdx.y * width;
    const int xpitch = (int)g.x_pixel * E, dpitch = (int)g.dy_pixel * E, opitch = g.channels * E;
    {
        const float zero[V] = {};
        own(total[0], zero, false);
        own(total[1], zero, false);
    }
    // Vector k of a pack (of one behind the last, nothing).  AHEAD: a vector's registers are free once it is used, so the next pack's is
    // loaded into them there and then; memory works while the block computes, though a compute unit holds one such block only
    // (1 024 x 14 x 14 x 192 bf16: 64 us, 70 without; 1 024 x 28 x 28 x 96: 156, 169).  With eight vectors, whose registers are short, and
    // in float32, where two blocks take turns, it costs more than it gives (1 024 x 784 x 64 bf16: 100, 95; 512 x 784 x 64 float32: 98, 83).
    u32x4 raw[NV], up[NV];
    const auto load = [&](const Seat &n, int64_t pack, int first, int last, bool of_x, bool of_dy) {
        const auto xb = unit_buffer(x + pack * g.pack * g.x_sample + c0, kNowhere), db = unit_buffer(dy + pack * g.pack * g.dy_sample + c0, kNowhere);
        const int xat = (int)(n.sub * g.x_sample) * E + n.r * xpitch + n.cq * 16, dat = (int)(n.sub * g.dy_sample) * E + n.r * dpitch + n.cq * 16;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (k < first || k >= last) continue;
            if (of_x) raw[k] = load16(xb, k < n.mine ? xat + k * g.rows * xpitch : kNowhere);
            if (of_dy) up[k] = load16(db, k < n.mine ? dat + k * g.rows * dpitch : kNowhere);
        }
    };
    Seat next;
    if constexpr (AHEAD) {
        next = seat_of<V>(g, walker, blockIdx.y);
        load(next, walker, 0, NV, true, true);
    }
    for (int64_t pack = walker; pack * g.pack < g.batch; pack += walkers) {
        const Seat s = AHEAD ? next : seat_of<V>(g, pack, blockIdx.y);
        const int64_t b0 = pack * g.pack;
        if constexpr (AHEAD) next = seat_of<V>(g, pack + walkers, blockIdx.y);
        else load(s, pack, 0, NV, true, true);
        // u = x + add, xhat = u * rstd, z = u * a + sh; the loop sums dz and dz * u.  (Never the mean folded into sh: where a group is
        // nearly constant its part of z, |mean| rstd, has no bound.  One addition for a value and loop: 1 024 x 196 x 192 bf16 76 us either
        // way, 4 096 x 784 x 32 177 and 168, 700 x 400 x 80 53 either way.)
        float add[V], rstd[P], a[V], sh[V];
        load_chan16<V>(g.shift && s.active ? g.shift + s.b * g.shift_sample : nullptr, s.c, 0.0f, add);
        const float *gamma = g.gamma, *beta = g.beta;
        asm volatile("" : "+s"(gamma), "+s"(beta));   // (read again for each pack: no registers to hold them)
        load_chan16<V>(s.active ? gamma : nullptr, s.c, 1.0f, a);
        load_chan16<V>(s.active ? beta : nullptr, s.c, 0.0f, sh);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int64_t at = s.active ? s.b * g.groups + blockIdx.y * g.ng + quotient(s.cq * P + i, g.inv_qg) : 0;
            const float mean = mean_in[at];
            rstd[i] = rstd_in[at];
#pragma unroll
            for (int j = i * PS; j < (i + 1) * PS; ++j) {
                add[j] -= mean;
                a[j] *= rstd[i];
            }
        }
        float dz[NV][V], s0[V], s1[V];
#pragma unroll
        for (int j = 0; j < V; ++j) s0[j] = s1[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (k < s.mine) {
                float u[V];
                widen<T>(raw[k], u);
                widen<T>(up[k], dz[k]);
#pragma unroll
                for (int j = 0; j < V; ++j) u[j] += add[j];
                if (g.swish)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float z = __builtin_fmaf(u[j], a[j], sh[j]), sg = sigmoid(z);
                        dz[k][j] *= __builtin_fmaf(z * sg, 1.0f - sg, sg);
                    }
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s0[j] += dz[k][j];
                    s1[j] = __builtin_fmaf(dz[k][j], u[j], s1[j]);
                }
            }
            if constexpr (AHEAD) load(next, pack + walkers, k, k + 1, false, true);
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s1[j] *= rstd[j / PS];
#pragma unroll
        for (int i = 0; i < P; ++i) {   // gamma * dz and gamma * dz * xhat, times rstd
            float2 t = {0.0f, 0.0f};
#pragma unroll
            for (int j = i * PS; j < (i + 1) * PS; ++j) {
                t.x = __builtin_fmaf(a[j], s0[j], t.x);
                t.y = __builtin_fmaf(a[j], s1[j], t.y);
            }
            part[threadIdx.x * P + i] = t;
        }
        if (s.active) {
            own(total[0], s0, true);
            own(total[1], s1, true);
        }
        __syncthreads();
        fold_groups(
            g, P,
            [&](float2 &t, int at, int) {
                const float2 o = part[at];
                t.x += o.x;
                t.y += o.y;
            },
            [&](float2 t, auto &&) { return float2{t.x * g.inv_n, t.y * g.inv_n}; },
            [&](int, int, int k, float2 v) { stat[k] = v; });
        __syncthreads();
        // dx = dz * a - (A + B * xhat) with rstd in A and B: dz * a + u * cx + c0
        float cx[P], cc[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float2 t = stat[s.active ? s.sub * g.ng + quotient(s.cq * P + i, g.inv_qg) : 0];
            cx[i] = -rstd[i] * t.y;
            cc[i] = -t.x;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s0[j] = 0.0f;
        const auto ob = unit_buffer(dx + b0 * g.pixels * g.channels + c0, kNowhere);
        const int oat = (s.sub * g.pixels + s.r) * opitch + s.cq * 16;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (k < s.mine) {
                float u[V];
                widen<T>(raw[k], u);
#pragma unroll
                for (int j = 0; j < V; ++j) u[j] = __builtin_fmaf(dz[k][j], a[j], __builtin_fmaf(u[j] + add[j], cx[j / PS], cc[j / PS]));
                if (dshift)
#pragma unroll
                    for (int j = 0; j < V; ++j) s0[j] += u[j];
                store16(ob, oat + k * g.rows * opitch, narrow<T>(u));
            }
            if constexpr (AHEAD) load(next, pack + walkers, k, k + 1, true, false);
        }
        if (dshift) {
            own(buf, s0, false);
            __syncthreads();
            if (g.pack == 1) {
                sum_rows(buf, g.rows, width, at, [&](int k, float t) { dshift[b0 * g.channels + c0 + k] = t; });
            } else {   // few rows each
                for (int i = threadIdx.x; i < g.pack * width; i += blockDim.x) {
                    const int sub = i / width, k = i - sub * width;
                    float t = 0.0f;
                    for (int r = 0; r < g.rows; ++r) t += buf[at(sub * g.rows + r, k)];
                    if (b0 + sub < g.batch) dshift[(b0 + sub) * g.channels + c0 + k] = t;
                }
                __syncthreads();
            }
        }
    }
    __syncthreads();
    for (int i = 0; i < 2; ++i)
        sum_rows(total[i], g.rows * g.pack, width, at, [&](int k, float t) { sums[((int64_t)i * walkers + walker) * g.channels + c0 + k] = t; });
}

// Grid: x 16 columns, y planes, z splits
__global__ __launch_bounds__(256) void gn_columns_kernel(const float *__restrict__ in, int64_t rows, int cols, int splits, float *__restrict__ out0,
                                                         float *__restrict__ out1)
{
    float *out = blockIdx.y ? out1 : out0;
    if (out) sum_columns(in + (int64_t)blockIdx.y * rows * cols, rows, cols, blockIdx.x * 16, blockIdx.z, splits, out);
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

Geometry geometry_of(const idm_group_norm_desc &d, bool backward, int v)
{
    Geometry g = {};
    g.batch = d.batch; g.pixels = d.pixels;
    g.x_sample = d.x_sample; g.x_pixel = d.x_pixel; g.dy_sample = d.dy_sample; g.dy_pixel = d.dy_pixel; g.shift_sample = d.shift_sample;
    g.channels = d.channels; g.groups = d.groups; g.gc = d.channels / d.groups;
    g.eps = d.eps;
    const int qg = g.gc / v;
    if (qg <= THREADS) {
        // Few samples: tiles of 256 bytes, so that blocks come from the channels before they come from more chunks, which all have
        // to be joined (1 x 4 096 x 512 float32, forward: 11 us, whole pixels 26).  Many: whole pixels, whose lines are read once.
        const int wide = g.batch < 256 ? 256 / elem_bytes(d.dtype) / v : THREADS;
        g.gpt = std::min(g.groups, std::max(1, wide / qg));
        g.tpg = 1;
        g.ntile = (g.groups + g.gpt - 1) / g.gpt;
        g.gpt = (g.groups + g.ntile - 1) / g.ntile;   // tiles of one width, nearly
        g.ntile = (g.groups + g.gpt - 1) / g.gpt;
    } else {
        g.gpt = 1;
        g.tpg = (qg + THREADS - 1) / THREADS;
        g.ntile = g.groups * g.tpg;
    }
    // Workgroups for the chip (backward some more: 1 024 x 784 x 90 fp16 180 us, with 1 024 of them 209; forward fewer: 8 x 65 536 x
    // 32 bf16 24 us, with 1 536 of them 26), none with less than four vectors per thread, nor with more to join (12 bytes for a chunk
    // and group) than it has to read itself; chunks of whole fours
    const int rows = std::max(1, THREADS / std::min(THREADS, g.gpt * qg));
    const int64_t most = std::max<int64_t>(1, g.pixels / (4 * rows)), tiles = g.batch * g.ntile, want = ((backward ? 1536 : 1024) + tiles - 1) / tiles;
    const int64_t join = (int64_t)std::sqrt((double)g.pixels * g.gc * elem_bytes(d.dtype) / 12.0);
    int64_t n = std::max<int64_t>(1, std::min<int64_t>({most, want, join, 1024}));
    g.chunk = (g.pixels + n - 1) / n;
    if (n > 1) g.chunk = (g.chunk + 4 * rows - 1) / (4 * rows) * (4 * rows);
    g.nchunk = (int)((g.pixels + g.chunk - 1) / g.chunk);
    return g;
}

// Column sums of one plane (out1 null) or two; part: 2 * kSplits * cols floats
void column_sums(const float *in, int64_t rows, int cols, float *part, float *out0, float *out1, int planes, hipStream_t s)
{
    const unsigned ct = (unsigned)((cols + 15) / 16);
    const int splits = rows > 2048 ? kSplits : 1;
    if (splits > 1) {
        hipLaunchKernelGGL(gn_columns_kernel, dim3(ct, planes, splits), dim3(256), 0, s, in, rows, cols, splits, part, part + (size_t)kSplits * cols);
        hipLaunchKernelGGL(gn_columns_kernel, dim3(ct, planes, 1), dim3(256), 0, s, (const float *)part, (int64_t)splits, cols, 1, out0, out1);
    } else {
        hipLaunchKernelGGL(gn_columns_kernel, dim3(ct, planes, 1), dim3(256), 0, s, in, rows, cols, 1, out0, out1);
    }
}

// ---- the one-launch form: which calls take it, with which instance and tile
struct UnitPlan {
    int pieces, threads, nv, tiles, ng, q, rows, pack;
    int64_t walkers;    // backward: blocks that share the samples of a tile
};

struct Instance { int threads, nv; };            // most threads, vectors of a thread
constexpr Instance kForward[] = {{1024, 8}, {1024, 16}, {1024, 4}};
constexpr Instance kBackward[] = {{512, 8}, {768, 4}};

// Does not look at pointers: `aligned` says whether they are 16-byte aligned.
bool plan_unit(const idm_group_norm_desc &d, bool backward, bool aligned, UnitPlan &u)
{
    const int e = elem_bytes(d.dtype), v = 16 / e, gc = d.channels / d.groups;
    if (!aligned || d.channels % v || d.shift_sample % 4 || d.x_sample % v || d.x_pixel % v || (backward && (d.dy_sample % v || d.dy_pixel % v))) return false;
    const int64_t pitch = std::max<int64_t>({d.x_pixel, d.channels, backward ? d.dy_pixel : 0});
    const int64_t apart = std::max<int64_t>({d.x_sample, d.pixels * d.channels, backward ? d.dy_sample : 0});
    if (d.pixels > 1024 * 16 || d.pixels * pitch * e >= kNowhere / 2) return false;
    u = {};
    u.pieces = gc % v == 0 ? 1 : gc % (v / 2) == 0 ? 2 : v;
    int whole = 1;                                   // fewest groups that are whole vectors
    while (whole * gc % v) ++whole;
    const int wide = whole * gc / v, units = d.groups / whole;
    const Instance *list = backward ? kBackward : kForward;
    auto fits = [&](int tiles, int i) {
        if (units % tiles) return false;
        const int t = units / tiles, q = t * wide;
        if (q > kTileVecs && t > 1) return false;
        const int64_t rows = (d.pixels + list[i].nv - 1) / list[i].nv, seats = rows * q;
        if (seats > list[i].threads) return false;
        // small maps: several samples to a block, of a wavefront's work at least
        int64_t pack = std::max<int64_t>(1, std::min<int64_t>(128 / seats, d.batch * tiles / 1024));
        if (pack * apart * e >= kNowhere / 2) pack = 1;
        u.threads = (int)((seats * pack + 63) / 64 * 64);
        u.nv = list[i].nv;
        u.ng = t * whole;
        u.tiles = tiles;
        u.q = q;
        u.rows = (int)rows;
        u.pack = (int)pack;
        return true;
    };
    // The best of all tiles and instances by what part of the chip's time they use, estimated as the product of
    //  - the seats that hold values (rows are cut to whole wavefronts, the last vector of a thread may be empty);
    //  - the wavefronts at work: a block takes ceil(waves / 4) of a SIMD's places (forward 6 with 8 vectors, 4 with 16, 8 with 4; backward 2
    //    and 3, float32 3 and 4); 12 of them (backward 8) keep the memory busy; a block alone loads, computes and stores in turn;
    //  - what a thread does besides its vectors (a fifth more with 4 of them, unless the joining of many small groups outweighs it; 16
    //    leave fewer wavefronts);
    //  - the parts of a pixel: blocks of one sample share its 128-byte lines, and parts that are no whole 32 bytes share sectors too
    //    (of less weight in calls that do not fill the chip);
    //  - blocks for all compute units, and whole turns of the walkers.
    // Measured on three sets in turn, us, bf16: forward 1 024 x 784 x 96 in 12-channel groups, tiles of 48 / 96 / 192 bytes 83 / 77 / 83;
    // 1 024 x 784 x 64, tiles of 32 / 64 / 128 bytes 55 / 44 / 49; backward 1 024 x 196 x 192, tiles of 48 / 96 / 192 bytes 79 / 76 / 69,
    // 4 096 x 49 x 128, tiles of 32 / 64 / 128 bytes 62 / 47 / 45.
    const int64_t pixel = (int64_t)d.channels * e;
    float best = 0.0f, worth = 0.0f;
    UnitPlan chosen = u;
    for (int i = 0; i < (backward ? 2 : 3); ++i)
        for (int tiles = 1; tiles <= std::min(units, 4096); ++tiles) {
            if (!fits(tiles, i)) continue;
            const int waves = u.threads / 64, many = backward ? 8 : 12;
            const int places = backward ? (i == 0 ? 2 : 3) + (e == 4 && u.pieces == 1) : u.nv == 8 ? 6 : u.nv == 16 ? 4 : 8;
            const int most = waves < 4 ? places * 4 / waves : places / ((waves + 3) / 4);
            const int64_t packs = (d.batch + u.pack - 1) / u.pack, part = (int64_t)u.q * 16;
            const float seats = (float)(u.rows * u.q * u.pack) / (float)u.threads * (float)d.pixels / (float)(u.rows * u.nv);
            const float shared = (float)std::min<int64_t>(128, pixel) / (float)part;
            const float lines = std::max(0.5f, shared > 1.0f ? 1.0f - 0.06f * (shared - 1.0f) : 1.0f) * (part < 32 ? 0.5f : part % 32 ? 0.85f : 1.0f);
            const float fill = std::min(1.0f, (float)(packs * tiles) / 256.0f);
            for (int blocks = backward ? 1 : most; blocks <= most; ++blocks) {
                float use = seats * (1.0f - (1.0f - lines) * fill) * std::min(1.0f, (float)(blocks * waves) / (float)many) * (blocks > 1 + !backward ? 1.0f : blocks > 1 ? 0.97f : backward ? 0.9f : 0.85f) *
                            (u.nv == 4 && (backward || u.pieces <= 2) ? 0.8f : u.nv == 16 ? 0.95f : 1.0f);
                const int64_t want = std::max(1, 256 * blocks / tiles), turns = (packs + want - 1) / want, n = (packs + turns - 1) / turns;
                if (backward) use *= (float)packs / (float)(turns * std::min(want, packs));
                if (use * std::sqrt(fill) > best) {   // (few blocks: their own time counts, not the chip's)
                    best = use * std::sqrt(fill);
                    worth = use * fill;
                    chosen = u;
                    chosen.walkers = n;
                }
            }
        }
    u = chosen;
    // Few large units: the form that cuts a sample into chunks fills the chip (16 x 4 096 x 64 bf16, backward: 17.4 us against 23.6;
    // 16 x 16 384 x 32 float32, forward: 23 against 41).  Small units are done before its second launch has begun (16 x 784 x 32
    // float32, backward: 12.3 against 14.1), unless groups straddle vectors (23 x 784 x 48 in 3-channel groups, bf16: 18 against 14).
    const int64_t bytes = d.pixels * u.q * 16;
    return worth > (backward ? 0.5f : 0.3f) || (best > 0.0f && bytes <= (backward ? u.pieces == 1 ? 40960 : 16384 : u.q == 1 ? 65535 : 131072));
}

// What a call needs.  Unless the caller says that all pointers are aligned, the size query does not know which form and vector width
// the call will take: the largest of all.
size_t workspace_floats(const idm_group_norm_desc &d, bool backward)
{
    UnitPlan u;
    const bool unit = plan_unit(d, backward, true, u);
    size_t most = unit && backward ? (size_t)2 * u.walkers * d.channels : 0;
    if (!(unit && d.aligned))
        for (int v = 16 / elem_bytes(d.dtype); v >= 1; v >>= 1) {
            if ((d.channels / d.groups) % v) continue;
            const Geometry g = geometry_of(d, backward, v);
            const size_t rows = (size_t)g.batch * g.nchunk;
            most = std::max(most, backward ? rows * (3 * g.channels + 2 * g.tpg * g.groups) : rows * g.tpg * g.groups * 3);
        }
    if (backward) most += (size_t)2 * kSplits * d.channels + (d.shift_sample == 0 ? (size_t)d.batch * d.channels : 0);
    return most;
}

UnitArgs unit_args(const idm_group_norm_desc &d, const UnitPlan &u)
{
    UnitArgs a = {};
    a.batch = d.batch; a.x_sample = d.x_sample; a.x_pixel = d.x_pixel; a.dy_sample = d.dy_sample; a.dy_pixel = d.dy_pixel;
    a.shift_sample = d.shift_sample; a.pixels = (int)d.pixels; a.channels = d.channels; a.groups = d.groups;
    a.gc = d.channels / d.groups; a.swish = d.activation == IDM_ACT_SWISH;
    a.ng = u.ng; a.q = u.q; a.rows = u.rows; a.pack = u.pack; a.seats = u.rows * u.q;
    a.qg = u.q * u.pieces / u.ng;
    a.full = a.pixels / u.rows; a.more = a.pixels % u.rows;
    a.inv_q = 1.0f / (float)a.q; a.inv_qg = 1.0f / (float)a.qg; a.inv_ng = 1.0f / (float)a.ng; a.inv_seats = 1.0f / (float)a.seats;
    a.eps = d.eps; a.n = (float)d.pixels * (float)a.gc; a.inv_n = 1.0f / a.n;
    return a;
}

constexpr int64_t kGridZ = 65535;

// n samples (or packs, or walkers) in a grid: eight neighbours in x where there are enough of them
dim3 unit_grid(int64_t n, int tiles)
{
    const unsigned x = n >= 64 ? 8 : (unsigned)n;
    return dim3(x, tiles, (unsigned)((n + x - 1) / x));
}

template <typename T, int P>
int unit_forward(const UnitPlan &u, UnitArgs a, const void *x, void *y, float *mean, float *rstd, hipStream_t s)
{
    const size_t lds = ((size_t)u.threads * P + (size_t)u.pack * u.ng) * sizeof(float2);
    const int64_t most = kGridZ * 8 * u.pack, all = a.batch;   // samples of one launch
    for (int64_t b = 0; b < all; b += most) {
        a.batch = std::min(most, all - b);
        const dim3 grid = unit_grid((a.batch + u.pack - 1) / u.pack, u.tiles);
        const T *xb = (const T *)x + b * a.x_sample;
        T *yb = (T *)y + b * a.pixels * a.channels;
        UnitArgs ab = a;
        if (ab.shift) ab.shift += b * a.shift_sample;
#define IDM_GN_UNIT(TH, NV)                                                                                                       \
    if (u.nv == NV)                                                                                                               \
        hipLaunchKernelGGL((gn_unit_forward_kernel<T, P, TH, NV>), grid, dim3(u.threads), lds, s, ab, xb, yb, mean + b * a.groups, \
                           rstd + b * a.groups)
        IDM_GN_UNIT(1024, 4); else IDM_GN_UNIT(1024, 8); else IDM_GN_UNIT(1024, 16);
#undef IDM_GN_UNIT
    }
    return hipGetLastError() == hipSuccess ? IDM_OK : idm_set_error(IDM_ERR_HIP, "group norm: launch failed");
}

template <typename T, int P>
int unit_backward(const UnitPlan &u, const UnitArgs &a, const void *dy, const void *x, const float *mean, const float *rstd, void *dx,
                  float *dgamma, float *dbeta, float *dshift, float *ws, hipStream_t s)
{
    const size_t lds = (size_t)u.threads * (2 * vec16<T> + std::max(vec16<T>, 2 * P)) * sizeof(float) + (size_t)u.pack * u.ng * sizeof(float2);
    float *part = ws + 2 * u.walkers * a.channels, *rows = dshift;
    if (dshift && a.shift_sample == 0) rows = part + (size_t)2 * kSplits * a.channels;   // one row for all samples: summed below
#define IDM_GN_UNIT(TH, NV)                                                                                                         \
    if (u.nv == NV)                                                                                                                 \
        hipLaunchKernelGGL((gn_unit_backward_kernel<T, P, TH, NV>), unit_grid(u.walkers, u.tiles), dim3(u.threads), lds, s, a,          \
                           (int)u.walkers, (const T *)dy, (const T *)x, mean, rstd, (T *)dx, ws, rows)
    IDM_GN_UNIT(768, 4); else IDM_GN_UNIT(512, 8);
#undef IDM_GN_UNIT
    if (dbeta || dgamma) column_sums(ws, u.walkers, a.channels, part, dbeta, dgamma, 2, s);
    if (rows != dshift) column_sums(rows, a.batch, a.channels, part, dshift, nullptr, 1, s);
    return hipGetLastError() == hipSuccess ? IDM_OK : idm_set_error(IDM_ERR_HIP, "group norm backward: launch failed");
}

template <typename F> int by_piece(int dtype, int pieces, F &&f)
{
    auto go = [&](auto t) {
        constexpr int V = vec16<decltype(t)>;
        return pieces == 1 ? f(t, std::integral_constant<int, 1>{}) : pieces == 2 ? f(t, std::integral_constant<int, 2>{})
                                                                                  : f(t, std::integral_constant<int, V>{});
    };
    switch (dtype) {
    case IDM_DT_F32: return go(float{});
    case IDM_DT_BF16: return go(__bf16{});
    default: return go(_Float16{});
    }
}

bool aligned_to(size_t n, std::initializer_list<const void *> ptrs)
{
    for (const void *p : ptrs)
        if ((uintptr_t)p % n) return false;
    return true;
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
    if (d->channels > (1 << 20) || d->pixels > ((int64_t)1 << 40) || d->batch > ((int64_t)1 << 30))
        return idm_set_error(IDM_ERR_INVALID, "group norm: more than 2^20 channels, 2^40 pixels or 2^30 samples");
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

// samples in y and z; `more` blocks behind the chunks and tiles
dim3 chunk_grid(const Geometry &g, int more)
{
    const int64_t y = std::min<int64_t>(g.batch, 32768);
    return dim3((unsigned)(g.nchunk * g.ntile + more), (unsigned)y, (unsigned)((g.batch + y - 1) / y));
}

template <typename T, int V>
int forward_launch(const idm_group_norm_desc &d, const Geometry &g, const void *x, void *y, float *mean, float *rstd, float *ws,
                   hipStream_t s)
{
    const dim3 blocks = chunk_grid(g, 0);
    hipLaunchKernelGGL((gn_stats_kernel<T, V>), blocks, dim3(THREADS), 0, s, g, (const T *)x, ws);
    if (d.activation == IDM_ACT_SWISH)
        hipLaunchKernelGGL((gn_apply_kernel<T, V, true>), blocks, dim3(THREADS), 0, s, g, (const T *)x, ws, (T *)y, mean, rstd);
    else
        hipLaunchKernelGGL((gn_apply_kernel<T, V, false>), blocks, dim3(THREADS), 0, s, g, (const T *)x, ws, (T *)y, mean, rstd);
    return check_launch("group norm: launch failed");
}

template <typename T, int V, bool SWISH>
int backward_launch(const Geometry &g, const void *dy, const void *x, const float *mean, const float *rstd, void *dx, float *dgamma,
                    float *dbeta, float *dshift, float *ws, hipStream_t s)
{
    const int64_t rows = g.batch * g.nchunk, plane = rows * g.channels;
    float2 *groups = (float2 *)ws;
    float *sums = ws + 2 * rows * g.tpg * g.groups, *part = sums + 3 * plane, *per_sample = nullptr;
    if (dshift && g.shift_sample == 0) per_sample = part + (size_t)2 * kSplits * g.channels;   // one row for all samples: summed below
    hipLaunchKernelGGL((gn_grad_sums_kernel<T, V, SWISH>), chunk_grid(g, 0), dim3(THREADS), 0, s, g, (const T *)dy, (const T *)x, mean, rstd,
                       sums, groups, dshift != nullptr);
    const bool here = (dbeta || dgamma) && rows <= 2048;   // few rows: the weight gradients in the same launch
    hipLaunchKernelGGL((gn_grad_apply_kernel<T, V, SWISH>), chunk_grid(g, here ? (g.channels + 15) / 16 * 2 : 0), dim3(THREADS), 0, s, g,
                       (const T *)dy, (const T *)x, mean, rstd, (const float *)sums, (const float2 *)groups, (T *)dx,
                       per_sample ? per_sample : dshift, dbeta, dgamma);
    if ((dbeta || dgamma) && !here) column_sums(sums, rows, g.channels, part, dbeta, dgamma, 2, s);
    if (per_sample) column_sums(per_sample, g.batch, g.channels, part, dshift, nullptr, 1, s);
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
    const size_t need = workspace_floats(*d, false) * sizeof(float);
    if (!x_dev || !y_dev || !mean_dev || !rstd_dev || (need && !workspace_dev)) return idm_set_error(IDM_ERR_INVALID, "group norm: null argument");
    if (workspace_bytes < need) return idm_set_error(IDM_ERR_INVALID, "group norm: workspace too small");
    if (!aligned_to(elem_bytes(d->dtype), {x_dev, y_dev}) || !aligned_to(4, {gamma_dev, beta_dev, shift_dev, mean_dev, rstd_dev}) ||
        !aligned_to(8, {workspace_dev}))
        return idm_set_error(IDM_ERR_INVALID, "group norm: a pointer is not aligned to its elements, or the workspace to 8 bytes");
    const bool aligned = aligned_to(16, {x_dev, y_dev, gamma_dev, beta_dev, shift_dev});
    if (d->aligned && !aligned) return idm_set_error(IDM_ERR_INVALID, "group norm: a pointer is not aligned to 16 bytes as the descriptor says");
    if (hipSetDevice(device) != hipSuccess) return idm_set_error(IDM_ERR_HIP, "group norm: no such device");
    UnitPlan u;
    if (plan_unit(*d, false, aligned, u)) {
        UnitArgs a = unit_args(*d, u);
        a.gamma = gamma_dev; a.beta = beta_dev; a.shift = shift_dev;
        return by_piece(d->dtype, u.pieces, [&](auto t, auto p) {
            return unit_forward<decltype(t), decltype(p)::value>(u, a, x_dev, y_dev, mean_dev, rstd_dev, (hipStream_t)stream);
        });
    }
    const int v = vec_of(*d, false, {x_dev, y_dev});
    Geometry g = geometry_of(*d, false, v);
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
    if (!aligned_to(elem_bytes(d->dtype), {dy_dev, x_dev, dx_dev}) || !aligned_to(8, {workspace_dev}) ||
        !aligned_to(4, {mean_dev, rstd_dev, gamma_dev, beta_dev, shift_dev, dgamma_dev, dbeta_dev, dshift_dev}))
        return idm_set_error(IDM_ERR_INVALID, "group norm backward: a pointer is not aligned to its elements, or the workspace to 8 bytes");
    const bool aligned = aligned_to(16, {dy_dev, x_dev, dx_dev, gamma_dev, beta_dev, shift_dev});
    if (d->aligned && !aligned)
        return idm_set_error(IDM_ERR_INVALID, "group norm backward: a pointer is not aligned to 16 bytes as the descriptor says");
    if (hipSetDevice(device) != hipSuccess) return idm_set_error(IDM_ERR_HIP, "group norm backward: no such device");
    UnitPlan u;
    if (plan_unit(*d, true, aligned, u)) {
        UnitArgs a = unit_args(*d, u);
        a.gamma = gamma_dev; a.beta = beta_dev; a.shift = shift_dev;
        return by_piece(d->dtype, u.pieces, [&](auto t, auto p) {
            return unit_backward<decltype(t), decltype(p)::value>(u, a, dy_dev, x_dev, mean_dev, rstd_dev, dx_dev, dgamma_dev, dbeta_dev,
                                                                  dshift_dev, (float *)workspace_dev, (hipStream_t)stream);
        });
    }
    const int v = vec_of(*d, true, {dy_dev, x_dev, dx_dev});
    Geometry g = geometry_of(*d, true, v);
    g.gamma = gamma_dev; g.beta = beta_dev; g.shift = shift_dev;
    return by_type(d->dtype, v, [&](auto t, auto w) {
        auto *f = d->activation == IDM_ACT_SWISH ? &backward_launch<decltype(t), decltype(w)::value, true>
                                                 : &backward_launch<decltype(t), decltype(w)::value, false>;
        return f(g, dy_dev, x_dev, mean_dev, rstd_dev, dx_dev, dgamma_dev, dbeta_dev, dshift_dev, (float *)workspace_dev, (hipStream_t)stream);
    });
}

}  // extern "C"
