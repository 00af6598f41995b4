// One AdamW step over many tensors, moments held in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g            v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Every product and sum is rounded to float32 separately (built with -ffp-contract=off): the moments are float32 numbers by
// definition, so the codes of the 8-bit form are the same in every build.
//
// 8-bit moments.  A code is a float32 cut to three mantissa bits, counted in eighths of a binade from a base that its block of
// 256 entries shares: value(code) = float32 bits (code + base) << 20, code 0 is zero.  m: a sign and codes 0..127 (16 binades under
// the block's largest entry), v: codes 0..255 (32 binades).  No scale is divided by, the window moves with the block's largest
// entry, and an entry's precision does not depend on its size (a linear code would lose the small second moments, whose roots
// divide).  The twenty bits that are cut off are rounded with the dither (i * A + t * B mod 2^32) >> 12, A and B the golden-ratio
// constants of two dimensions (2^32 / p, 2^32 / p^2, p^3 = p + 1; swapped for v): equidistributed over the steps of one entry,
// so that a second moment that changes by 0.1 % a step, a hundredth of a code, moves by one code in about a hundred steps, where
// rounding to nearest would never move it.  A second moment of 2^-129 and more never gets code zero.  Entries that are not finite take the
// largest code and leave their block's window to the others.
//
// Memory bounds it: parameter, gradient and moments are read once, parameter and moments written once, 28 bytes an entry with all of them
// float32, 10 with 16-bit parameters and gradients and codes.  50 M entries float32: 268 us (5.2 TB/s; a large copy reaches 4.9, a sum of
// two arrays 5.8), with codes 157 (5.1 TB/s); 100 M bf16 with codes: 218 us (4.6 TB/s; the codes' arithmetic is hidden to two thirds), their
// decoding 164 us (6.1 TB/s).
// All tensors go in one launch for each 96: a workgroup takes 4 096 entries of one of them and finds it by bisection in a table that
// travels with the arguments, so nothing is copied to the device first.  The step is counted and the bias corrected on the device, so
// that a captured step goes on counting: by a kernel of one thread before a large step (4.8 us), within a small one.
#include "../../include/isingdiff.h"
#include "idm_internal.h"
#include "idm_device.h"

#include <algorithm>
#include <cmath>
#include <vector>

namespace {

typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
constexpr int BLOCK = IDM_ADAMW_BLOCK;      // entries that share a window
constexpr int CHUNK = 4096;                 // entries of one workgroup
constexpr int64_t LAUNCH = (1 << 24) - 1;   // workgroups of one launch: fewer than 2^32 threads
constexpr int TENSORS = 96;                 // tensors of one launch (their table travels in the kernel arguments, at most 4 KB)
constexpr uint32_t ROT_A = 0xC13FA9A9u, ROT_B = 0x91E10DA5u;

struct Table {
    void *p[TENSORS];
    const void *g[TENSORS];
    int64_t n[TENSORS];                     // entries
    uint32_t at[TENSORS];                   // block of the first one in the moments
    int32_t first[TENSORS + 1];             // first chunk
    float keep[TENSORS];                    // 1 - lr wd
    int count;
};

struct Coef {
    float size, root;                       // lr / (1 - b1^t), -1 where the count is none; 1 / sqrt(1 - b2^t)
    uint32_t t, unused;
};

// Where the step count stands, and what the coefficients of a step follow from (log1, log2: binary logarithms of the betas)
struct Clock {
    int64_t *step;
    double lr, log1, log2;
};

DEVI Coef coef_of(int64_t t, const Clock &c)
{
    if (t <= 0) return {-1.0f, 0.0f, 0, 0};   // the count before it was negative
    return {(float)(c.lr / (1.0 - exp2((double)t * c.log1))), (float)(1.0 / sqrt(1.0 - exp2((double)t * c.log2))), (uint32_t)t, 0};
}

// A step of one launch of at most kOnce workgroups counts itself: they all read the count, and each adds one to the bits above it when
// it has done so; the last of them moves the count on and clears those bits.  (A negative count stays one until somebody adds, and nobody
// who sees one adds.)  Larger steps begin with a kernel of one thread: the additions go one after the other (in a graph: one workgroup
// 6.5 us instead of 7.1, 128 of them 8.1 and 8.3, 256 11.4 and 9.4, 960 29 and 22; the host takes 1 to 2 us less).
constexpr int kOnce = 256, kCountBits = 53;

__global__ void adamw_begin_kernel(Clock clock, Coef *c)
{
    const int64_t t = *clock.step < 0 ? 0 : *clock.step + 1;
    if (t) *clock.step = t;
    *c = coef_of(t, clock);
}

DEVI float value_m(uint32_t code, int base)
{
    const uint32_t c = code & 127u;
    return __uint_as_float((c ? (c + (uint32_t)base) << 20 : 0u) | (code & 128u) << 24);
}
DEVI float value_v(uint32_t code, int base) { return __uint_as_float(code ? (code + (uint32_t)base) << 20 : 0u); }

// The float32 bits of |x|, rounded to a multiple of 2^20 by the dither: eighths of a binade
DEVI uint32_t place(uint32_t size, uint32_t turn) { return (size + (turn >> 12)) >> 20; }
// The same where x may not be finite (2047), or may round up to what infinity has
DEVI uint32_t place_any(uint32_t size, uint32_t turn)
{
    const uint32_t q = place(size, turn);
    return size >= 0x7f800000u ? 2047u : q < 2039u ? q : 2039u;
}

// N entries of a thread.  `full`: all are there and the address is aligned; else one by one, those below n only.
template <typename T, int N> DEVI void load_entries(const T *p, int64_t i, int64_t n, bool full, float out[N])
{
    typedef __attribute__((ext_vector_type(N))) T vec;
    if (full) {
        const vec v = *(const vec *)(p + i);
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) out[j] = i + j < n ? (float)p[i + j] : 0.0f;
    }
}
template <typename T, int N> DEVI void store_entries(T *p, int64_t i, int64_t n, bool full, const float in[N])
{
    typedef __attribute__((ext_vector_type(N))) T vec;
    if (full) {
        vec v;
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] = (T)in[j];
        *(vec *)(p + i) = v;
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (i + j < n) p[i + j] = (T)in[j];
    }
}

// sqrt and 1 / x by the instructions (one unit in the last place each: the update has 16 roundings of float32 in line at most; the moments
// do not depend on them).  v_sqrt_f32 takes
// denormals for zero, hence the scale.
DEVI float root_of(float v)
{
    const bool small = v < 0x1p-90f;
    const float r = __builtin_amdgcn_sqrtf(small ? v * 0x1p64f : v);
    return small ? r * 0x1p-32f : r;
}

// Moments are not looked at again before the next step.  Where a step's tensors exceed the 256 MB of cache (FAR), 32-bit ones pass
// it by and leave it to parameters and gradients, which the passes before and after the step share.
template <bool FAR, typename V> DEVI V take(const V *p)
{
    if constexpr (FAR) return __builtin_nontemporal_load(p);
    else return *p;
}
template <bool FAR, typename V> DEVI void put(V *p, V v)
{
    if constexpr (FAR) __builtin_nontemporal_store(v, p);
    else *p = v;
}

template <typename PT, typename GT, bool EIGHT, bool FAR>
__global__ __launch_bounds__(256) void adamw_kernel(Table tab, Clock clock, const Coef *__restrict__ coef, float b1, float c1, float b2, float c2,
                                                    float eps, void *__restrict__ m_all, void *__restrict__ v_all,
                                                    int16_t *__restrict__ m_base, int16_t *__restrict__ v_base)
{
    constexpr int N = EIGHT ? 8 : 4;           // entries of a thread: 16-byte loads of 16-bit parameters beside 8-byte ones of codes
    constexpr int LANES = BLOCK / N;           // that share a window
    const int chunk = blockIdx.x;
    int k = 0, hi = tab.count;   // the tensor whose chunks hold this one
    while (hi - k > 1) {
        const int mid = (k + hi) >> 1;
        if (tab.first[mid] <= chunk) k = mid; else hi = mid;
    }
    PT *p = (PT *)tab.p[k];
    const GT *g = (const GT *)tab.g[k];
    const int64_t n = tab.n[k], at = (int64_t)tab.at[k] * BLOCK, i0 = (int64_t)(chunk - tab.first[k]) * CHUNK;
    const bool aligned = ((uintptr_t)p % (N * sizeof(PT)) | (uintptr_t)g % (N * sizeof(GT))) == 0;
    const int64_t count = coef ? 0 : *clock.step, steps = count < 0 ? 0 : (count & (((int64_t)1 << kCountBits) - 1)) + 1;
    const Coef now = coef ? *coef : coef_of(steps, clock);
    const float keep = tab.keep[k], size = now.size, root = now.root;
    const uint32_t t = now.t;
#pragma unroll 2
    for (int64_t i = i0 + threadIdx.x * N; i < i0 + CHUNK; i += 256 * N) {
        if (i / BLOCK * BLOCK >= n) break;     // (the same for all lanes of a block)
        const bool full = aligned && i + N <= n;
        float pv[N], gv[N], m[N], v[N];
        load_entries<PT, N>(p, i, n, full, pv);
        load_entries<GT, N>(g, i, n, full, gv);
        const int64_t w = (at + i) / BLOCK;    // the block among the moments
        if (size < 0.0f) break;                // (all threads or none; here, where the loads are on their way)
        if constexpr (EIGHT) {
            const u32x2 cm = take<FAR>((const u32x2 *)((const uint8_t *)m_all + at + i)), cv = take<FAR>((const u32x2 *)((const uint8_t *)v_all + at + i));
            const int bm = m_base[w], bv = v_base[w];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                m[j] = value_m(cm[j / 4] >> 8 * (j & 3) & 255u, bm);
                v[j] = value_v(cv[j / 4] >> 8 * (j & 3) & 255u, bv);
            }
        } else {
            const f32x4 mm = take<FAR>((const f32x4 *)((const float *)m_all + at + i)), vv = take<FAR>((const f32x4 *)((const float *)v_all + at + i));
#pragma unroll
            for (int j = 0; j < N; ++j) { m[j] = mm[j]; v[j] = vv[j]; }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            m[j] = m[j] * b1 + gv[j] * c1;
            v[j] = v[j] * b2 + (gv[j] * gv[j]) * c2;
            pv[j] = pv[j] * keep - size * (m[j] * __builtin_amdgcn_rcpf(root_of(v[j]) * root + eps));
        }
        store_entries<PT, N>(p, i, n, full, pv);
        if constexpr (EIGHT) {
            typedef __attribute__((ext_vector_type(2))) unsigned short u16x2;
            uint32_t qm[N], qv[N], top = 0, tm = 0, tv = 0;
            const uint32_t id = (uint32_t)(at + i), ta = id * ROT_A + t * ROT_B, tb = id * ROT_B + t * ROT_A;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const uint32_t sm = __float_as_uint(m[j]) & 0x7fffffffu, sv = __float_as_uint(v[j]) & 0x7fffffffu;
                qm[j] = place(sm, ta + j * ROT_A);
                qv[j] = place(sv, tb + j * ROT_B);
                tm = qm[j] > tm ? qm[j] : tm;
                tv = qv[j] > tv ? qv[j] : tv;
            }
            if ((tm > tv ? tm : tv) >= 2039u) {   // rare: near the largest float32 or not finite
                tm = tv = 0;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    qm[j] = place_any(__float_as_uint(m[j]) & 0x7fffffffu, ta + j * ROT_A);
                    qv[j] = place_any(__float_as_uint(v[j]) & 0x7fffffffu, tb + j * ROT_B);
                    if (qm[j] < 2047u) tm = qm[j] > tm ? qm[j] : tm;
                    if (qv[j] < 2047u) tv = qv[j] > tv ? qv[j] : tv;
                }
            }
            top = tm | tv << 16;                  // both maxima in one exchange
#pragma unroll
            for (int off = LANES / 2; off >= 1; off >>= 1)
                top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                                             __builtin_bit_cast(u16x2, (uint32_t)__shfl_xor((int)top, off, 64))));
            const int bm = max((int)(top & 0xffffu) - 127, 0), bv = max((int)(top >> 16) - 255, 0);
            uint32_t cm[2] = {0, 0}, cv[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int a = min(max((int)qm[j] - bm, 0), 127), b = min(max((int)qv[j] - bv, min((int)qv[j], 1)), 255);
                cm[j >> 2] |= ((uint32_t)a | (__float_as_uint(m[j]) >> 24 & 128u)) << 8 * (j & 3);
                cv[j >> 2] |= (uint32_t)b << 8 * (j & 3);
            }
            put<FAR>((u32x2 *)((uint8_t *)m_all + at + i), u32x2{cm[0], cm[1]});
            put<FAR>((u32x2 *)((uint8_t *)v_all + at + i), u32x2{cv[0], cv[1]});
            if ((threadIdx.x & (LANES - 1)) == 0) {
                m_base[w] = (int16_t)bm;
                v_base[w] = (int16_t)bv;
            }
        } else {
            put<FAR>((f32x4 *)((float *)m_all + at + i), f32x4{m[0], m[1], m[2], m[3]});
            put<FAR>((f32x4 *)((float *)v_all + at + i), f32x4{v[0], v[1], v[2], v[3]});
        }
    }
    if (!coef && size >= 0.0f) {
        __syncthreads();   // all wavefronts have read the count
        if (threadIdx.x == 0) {
            typedef unsigned long long word;
            const word before = __hip_atomic_fetch_add((word *)clock.step, (word)1 << kCountBits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (before >> kCountBits == gridDim.x - 1) __hip_atomic_store((word *)clock.step, (word)steps, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
}

__global__ __launch_bounds__(256) void adamw_moments_kernel(const uint8_t *__restrict__ m, const uint8_t *__restrict__ v,
                                                            const int16_t *__restrict__ m_base, const int16_t *__restrict__ v_base,
                                                            float *__restrict__ m_out, float *__restrict__ v_out, int64_t n)
{
    for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)gridDim.x * 1024) {
        const uint32_t cm = *(const uint32_t *)(m + i), cv = *(const uint32_t *)(v + i);
        const int bm = m_base[i / BLOCK], bv = v_base[i / BLOCK];
        f32x4 a, b;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            a[j] = value_m(cm >> 8 * j & 255u, bm);
            b[j] = value_v(cv >> 8 * j & 255u, bv);
        }
        *(f32x4 *)(m_out + i) = a;
        *(f32x4 *)(v_out + i) = b;
    }
}

template <typename F> int by_types(int pt, int gt, F &&f)
{
    auto with_g = [&](auto p) {
        switch (gt) {
        case IDM_DT_F32: return f(p, float{});
        case IDM_DT_BF16: return f(p, __bf16{});
        default: return f(p, _Float16{});
        }
    };
    switch (pt) {
    case IDM_DT_F32: return with_g(float{});
    case IDM_DT_BF16: return with_g(__bf16{});
    default: return with_g(_Float16{});
    }
}

bool known_dtype(int t) { return t == IDM_DT_F32 || t == IDM_DT_BF16 || t == IDM_DT_F16; }
int64_t room_of(int64_t n) { return (n + BLOCK - 1) / BLOCK * BLOCK; }

}  // namespace

extern "C" {

int idm_adamw_step(int device, const idm_adamw_cfg *cfg, int64_t n_tensors, void *const *params_dev, const void *const *grads_dev,
                   const int64_t *sizes, const float *weight_decay, void *m_dev, void *v_dev, int16_t *m_base_dev, int16_t *v_base_dev,
                   int64_t moments, int64_t *step_dev, void *scratch_dev, void *stream)
try {
    if (!cfg || n_tensors < 0 || (n_tensors > 0 && (!params_dev || !grads_dev || !sizes || !weight_decay)) || !step_dev || !scratch_dev)
        return idm_set_error(IDM_ERR_INVALID, "adamw: null argument");
    if ((uintptr_t)step_dev % 8 || (uintptr_t)scratch_dev % 8) return idm_set_error(IDM_ERR_INVALID, "adamw: step count and scratch must be aligned to 8 bytes");
    if (!known_dtype(cfg->param_dtype) || !known_dtype(cfg->grad_dtype)) return idm_set_error(IDM_ERR_INVALID, "adamw: unknown dtype");
    if (cfg->moment_bits != 32 && cfg->moment_bits != 8) return idm_set_error(IDM_ERR_INVALID, "adamw: moments have 32 or 8 bits");
    const bool eight = cfg->moment_bits == 8;
    if (!(cfg->lr >= 0) || std::isinf(cfg->lr) || !(cfg->beta1 >= 0 && cfg->beta1 < 1) || !(cfg->beta2 >= 0 && cfg->beta2 < 1) ||
        !(cfg->eps >= 0) || std::isinf(cfg->eps))
        return idm_set_error(IDM_ERR_INVALID, "adamw: lr and eps must be finite and not negative, the betas in [0, 1)");
    int64_t total = 0, work = 0, tensors = 0;   // entries of the moments, workgroups, tensors with gradients
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;   // what the step writes
    const auto writes = [&](const void *p, size_t bytes) {
        if (bytes) spans.push_back({(uintptr_t)p, (uintptr_t)p + bytes});
    };
    const size_t pb = cfg->param_dtype == IDM_DT_F32 ? 4 : 2, gb = cfg->grad_dtype == IDM_DT_F32 ? 4 : 2;
    for (int64_t i = 0; i < n_tensors; ++i) {
        if (sizes[i] < 0 || sizes[i] > LAUNCH * CHUNK) return idm_set_error(IDM_ERR_INVALID, "adamw: tensor size out of range");
        if (!(weight_decay[i] >= 0) || std::isinf(weight_decay[i]))
            return idm_set_error(IDM_ERR_INVALID, "adamw: weight decay must be finite and not negative");
        total += room_of(sizes[i]);
        if (!sizes[i] || !grads_dev[i]) continue;
        if (!params_dev[i]) return idm_set_error(IDM_ERR_INVALID, "adamw: null parameter");
        if ((uintptr_t)params_dev[i] % pb || (uintptr_t)grads_dev[i] % gb) return idm_set_error(IDM_ERR_INVALID, "adamw: misaligned tensor");
        work += (sizes[i] + CHUNK - 1) / CHUNK;
        writes(params_dev[i], (size_t)sizes[i] * pb);
        ++tensors;
    }
    if (total / BLOCK > 0xffffffff) return idm_set_error(IDM_ERR_INVALID, "adamw: more than 2^40 entries");
    if (total != moments) return idm_set_error(IDM_ERR_INVALID, "adamw: the moments were made for other tensors (each takes its size rounded up to 256 entries)");
    if (total && (!m_dev || !v_dev || (eight && (!m_base_dev || !v_base_dev)))) return idm_set_error(IDM_ERR_INVALID, "adamw: null moments");
    if ((uintptr_t)m_dev % 16 || (uintptr_t)v_dev % 16 || (eight && ((uintptr_t)m_base_dev % 2 || (uintptr_t)v_base_dev % 2)))
        return idm_set_error(IDM_ERR_INVALID, "adamw: moments must be aligned to 16 bytes, their bases to 2");
    for (const void *p : {(const void *)m_dev, (const void *)v_dev}) writes(p, (size_t)total * (eight ? 1 : 4));
    for (const void *p : {(const void *)m_base_dev, (const void *)v_base_dev}) writes(p, eight ? (size_t)(total / BLOCK) * 2 : 0);
    writes(step_dev, 8);
    writes(scratch_dev, 16);
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        if (spans[i].first < spans[i - 1].second)
            return idm_set_error(IDM_ERR_INVALID, "adamw: two of parameters, moments, bases, step count and scratch share memory");
    for (int64_t i = 0; i < n_tensors; ++i) {   // workgroups read gradients while others write parameters and state
        if (!sizes[i] || !grads_dev[i]) continue;
        const uintptr_t lo = (uintptr_t)grads_dev[i], hi = lo + (size_t)sizes[i] * gb;
        auto after = std::lower_bound(spans.begin(), spans.end(), std::make_pair(hi, (uintptr_t)0));   // the first one from hi on
        for (; after != spans.begin() && (after - 1)->second > lo; --after)
            if ((after - 1)->first != lo || params_dev[i] != grads_dev[i] || pb != gb)
                return idm_set_error(IDM_ERR_INVALID, "adamw: a gradient shares memory with a parameter or the state");
    }
    if (hipSetDevice(device) != hipSuccess) return idm_set_error(IDM_ERR_HIP, "adamw: no such device");
    hipStream_t s = (hipStream_t)stream;
    const Clock clock = {step_dev, cfg->lr, std::log2(cfg->beta1), std::log2(cfg->beta2)};
    Coef *coef = work && tensors <= TENSORS && work <= kOnce ? nullptr : (Coef *)scratch_dev;
    if (coef) hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1), 0, s, clock, coef);
    const float b1 = (float)cfg->beta1, c1 = (float)(1 - cfg->beta1), b2 = (float)cfg->beta2, c2 = (float)(1 - cfg->beta2);
    // 1 / x of a subnormal x is infinite, and 0 times that no number.  Above zero a root is at least 2^-75, so eps does not count down there
    const float eps = cfg->eps > 0 ? std::max((float)cfg->eps, 0x1p-126f) : 0.0f;
    // (50 M float32: 267 us, 278 through the cache; 33 M: 140 and 190; below the limit it costs up to a twentieth, and codes gain nothing)
    const bool far = !eight && total * (int64_t)(pb + gb + 8) > (int64_t)1 << 28;
    int64_t at = 0;
    Table tab;
    int64_t chunks = 0;
    tab.count = 0;
    auto flush = [&]() -> int {
        if (!tab.count) return IDM_OK;
        tab.first[tab.count] = (int32_t)chunks;
        auto go = [&](auto p, auto g) {
            using PT = decltype(p);
            using GT = decltype(g);
            auto kernel = eight ? &adamw_kernel<PT, GT, true, false> : far ? &adamw_kernel<PT, GT, false, true> : &adamw_kernel<PT, GT, false, false>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)chunks), dim3(256), 0, s, tab, clock, (const Coef *)coef, b1, c1, b2, c2, eps, m_dev,
                               v_dev, m_base_dev, v_base_dev);
            return IDM_OK;
        };
        by_types(cfg->param_dtype, cfg->grad_dtype, go);
        tab.count = 0;
        chunks = 0;
        return hipGetLastError() == hipSuccess ? IDM_OK : idm_set_error(IDM_ERR_HIP, "adamw: launch failed");
    };
    for (int64_t i = 0; i < n_tensors; at += room_of(sizes[i]), ++i) {
        if (!sizes[i] || !grads_dev[i]) continue;      // no gradient: the tensor and its moments stay as they are
        const int64_t c = (sizes[i] + CHUNK - 1) / CHUNK;
        if (tab.count == TENSORS || chunks + c > LAUNCH) {
            const int rc = flush();
            if (rc != IDM_OK) return rc;
        }
        const int k = tab.count++;
        tab.p[k] = params_dev[i];
        tab.g[k] = grads_dev[i];
        tab.n[k] = sizes[i];
        tab.at[k] = (uint32_t)(at / BLOCK);
        tab.first[k] = (int32_t)chunks;
        tab.keep[k] = (float)(1.0 - cfg->lr * (double)weight_decay[i]);
        chunks += c;
    }
    return flush();
} catch (...) {   // the table of memory spans is the only thing that can throw
    return idm_set_error(IDM_ERR_NOMEM, "adamw: host allocation failed");
}

int idm_adamw_moments(int device, const uint8_t *m_dev, const uint8_t *v_dev, const int16_t *m_base_dev, const int16_t *v_base_dev,
                      float *m_out_dev, float *v_out_dev, int64_t moments, void *stream)
{
    if (moments < 0 || moments % BLOCK || moments > ((int64_t)1 << 40))
        return idm_set_error(IDM_ERR_INVALID, "adamw: the moments are whole blocks of 256 entries");
    if (!moments) return IDM_OK;
    if (!m_dev || !v_dev || !m_base_dev || !v_base_dev || !m_out_dev || !v_out_dev) return idm_set_error(IDM_ERR_INVALID, "adamw: null argument");
    if ((uintptr_t)m_dev % 16 || (uintptr_t)v_dev % 16 || (uintptr_t)m_out_dev % 16 || (uintptr_t)v_out_dev % 16)
        return idm_set_error(IDM_ERR_INVALID, "adamw: moments must be aligned to 16 bytes");
    const size_t n = (size_t)moments, bytes[6] = {n, n, n / BLOCK * 2, n / BLOCK * 2, 4 * n, 4 * n};
    const void *const at[6] = {m_dev, v_dev, m_base_dev, v_base_dev, m_out_dev, v_out_dev};
    for (int i = 4; i < 6; ++i)
        for (int k = 0; k < i; ++k)
            if ((uintptr_t)at[i] < (uintptr_t)at[k] + bytes[k] && (uintptr_t)at[k] < (uintptr_t)at[i] + bytes[i])
                return idm_set_error(IDM_ERR_INVALID, "adamw: the moments' values share memory with their codes or each other");
    if (hipSetDevice(device) != hipSuccess) return idm_set_error(IDM_ERR_HIP, "adamw: no such device");
    const int64_t blocks = std::min<int64_t>((moments + 1023) / 1024, 1 << 20);   // (one pass up to 2^30 entries)
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, m_dev, v_dev,
                       m_base_dev, v_base_dev, m_out_dev, v_out_dev, moments);
    return hipGetLastError() == hipSuccess ? IDM_OK : idm_set_error(IDM_ERR_HIP, "adamw: launch failed");
}

}  // extern "C"
