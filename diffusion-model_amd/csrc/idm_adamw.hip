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
// rounding to nearest would never move it.  A second moment above zero never gets code zero.  Entries that are not finite take the
// largest code and leave their block's window to the others.
#include "../../include/isingdiff.h"
#include "idm_internal.h"
#include "idm_device.h"

#include <algorithm>
#include <cmath>
#include <vector>

namespace {

constexpr int BLOCK = IDM_ADAMW_BLOCK;      // entries that share a window = 4 per lane of one wavefront
constexpr int CHUNK = 4096;                 // entries of one workgroup
constexpr int TENSORS = 64;                 // tensors of one launch (their table travels in the kernel arguments)
constexpr uint32_t ROT_A = 0xC13FA9A9u, ROT_B = 0x91E10DA5u;

struct Table {
    void *p[TENSORS];
    const void *g[TENSORS];
    int64_t n[TENSORS], at[TENSORS];        // entries; index of the first one in the moments
    int64_t first[TENSORS + 1];             // first chunk
    float keep[TENSORS];                    // 1 - lr wd
    int count;
};

struct Coef {
    float size, root;                       // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
    uint32_t t, unused;
};

__global__ void adamw_begin_kernel(int64_t *step, double lr, double b1, double b2, Coef *c)
{
    const int64_t t = *step + 1;
    *step = t;
    c->size = (float)(lr / (1.0 - pow(b1, (double)t)));
    c->root = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
    c->t = (uint32_t)t;
}

// The float32 bits of |x|, rounded to a multiple of 2^20 by the dither: eighths of a binade.  Not finite: 2047.
DEVI int place(uint32_t bits, uint32_t turn)
{
    const uint32_t size = bits & 0x7fffffffu;
    const uint32_t q = (size + (turn >> 12)) >> 20;
    return size < 0x7f800000u ? (int)(q < 2039u ? q : 2039u) : 2047;
}

DEVI float value_m(uint32_t code, int base)
{
    const uint32_t c = code & 127u;
    return __uint_as_float((c ? (c + (uint32_t)base) << 20 : 0u) | (code & 128u) << 24);
}
DEVI float value_v(uint32_t code, int base) { return __uint_as_float(code ? (code + (uint32_t)base) << 20 : 0u); }

DEVI int wave_max(int x)
{
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const int o = __shfl_xor(x, off, 64);
        x = o > x ? o : x;
    }
    return x;
}

template <typename PT, typename GT, bool EIGHT>
__global__ __launch_bounds__(256) void adamw_kernel(Table tab, const Coef *__restrict__ coef, float b1, float c1, float b2, float c2,
                                                    float eps, void *__restrict__ m_all, void *__restrict__ v_all,
                                                    int16_t *__restrict__ m_base, int16_t *__restrict__ v_base)
{
    const int64_t chunk = blockIdx.x;
    int k = 0, hi = tab.count;   // the tensor whose chunks hold this one
    while (hi - k > 1) {
        const int mid = (k + hi) >> 1;
        if (tab.first[mid] <= chunk) k = mid; else hi = mid;
    }
    PT *p = (PT *)tab.p[k];
    const GT *g = (const GT *)tab.g[k];
    const int64_t n = tab.n[k], at = tab.at[k], i0 = (chunk - tab.first[k]) * CHUNK;
    const float keep = tab.keep[k], size = coef->size, root = coef->root;
    const uint32_t t = coef->t;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int blk = wave; blk < CHUNK / BLOCK; blk += 4) {
        const int64_t i = i0 + blk * BLOCK + lane * 4;
        if (i0 + blk * BLOCK >= n) break;          // (the same for the whole wavefront)
        float pv[4], gv[4], m[4], v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = i + j < n;
            pv[j] = in ? (float)p[i + j] : 0.0f;
            gv[j] = in ? (float)g[i + j] : 0.0f;
        }
        const int64_t w = (at + i0) / BLOCK + blk;   // the block among the moments
        if constexpr (EIGHT) {
            const uint32_t cm = *(const uint32_t *)((const uint8_t *)m_all + at + i), cv = *(const uint32_t *)((const uint8_t *)v_all + at + i);
            const int bm = m_base[w], bv = v_base[w];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                m[j] = value_m(cm >> 8 * j & 255u, bm);
                v[j] = value_v(cv >> 8 * j & 255u, bv);
            }
        } else {
            const f32x4 mm = *(const f32x4 *)((const float *)m_all + at + i), vv = *(const f32x4 *)((const float *)v_all + at + i);
#pragma unroll
            for (int j = 0; j < 4; ++j) { m[j] = mm[j]; v[j] = vv[j]; }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m[j] = m[j] * b1 + gv[j] * c1;
            v[j] = v[j] * b2 + (gv[j] * gv[j]) * c2;
            pv[j] = pv[j] * keep - size * (m[j] / (sqrtf(v[j]) * root + eps));
            if (i + j < n) p[i + j] = (PT)pv[j];
        }
        if constexpr (EIGHT) {
            int qm[4], qv[4], tm = 0, tv = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t id = (uint32_t)(at + i + j);
                qm[j] = place(__float_as_uint(m[j]), id * ROT_A + t * ROT_B);
                qv[j] = place(__float_as_uint(v[j]), id * ROT_B + t * ROT_A);
                tm = qm[j] < 2047 && qm[j] > tm ? qm[j] : tm;
                tv = qv[j] < 2047 && qv[j] > tv ? qv[j] : tv;
            }
            tm = wave_max(tm);
            tv = wave_max(tv);
            const int bm = tm > 127 ? tm - 127 : 0, bv = tv > 255 ? tv - 255 : 0;
            uint32_t cm = 0, cv = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                int a = qm[j] - bm, b = qv[j] - bv;
                a = a < 0 ? 0 : a > 127 ? 127 : a;
                b = qv[j] == 0 ? 0 : b < 1 ? 1 : b > 255 ? 255 : b;
                cm |= ((uint32_t)a | __float_as_uint(m[j]) >> 31 << 7) << 8 * j;
                cv |= (uint32_t)b << 8 * j;
            }
            *(uint32_t *)((uint8_t *)m_all + at + i) = cm;
            *(uint32_t *)((uint8_t *)v_all + at + i) = cv;
            if (lane == 0) {
                m_base[w] = (int16_t)bm;
                v_base[w] = (int16_t)bv;
            }
        } else {
            *(f32x4 *)((float *)m_all + at + i) = f32x4{m[0], m[1], m[2], m[3]};
            *(f32x4 *)((float *)v_all + at + i) = f32x4{v[0], v[1], v[2], v[3]};
        }
    }
}

__global__ __launch_bounds__(256) void adamw_moments_kernel(const uint8_t *__restrict__ m, const uint8_t *__restrict__ v,
                                                            const int16_t *__restrict__ m_base, const int16_t *__restrict__ v_base,
                                                            float *__restrict__ m_out, float *__restrict__ v_out, int64_t n)
{
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n) return;
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

template <bool EIGHT, typename F> int by_types(int pt, int gt, F &&f)
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
    if (!known_dtype(cfg->param_dtype) || !known_dtype(cfg->grad_dtype)) return idm_set_error(IDM_ERR_INVALID, "adamw: unknown dtype");
    if (cfg->moment_bits != 32 && cfg->moment_bits != 8) return idm_set_error(IDM_ERR_INVALID, "adamw: moments have 32 or 8 bits");
    const bool eight = cfg->moment_bits == 8;
    if (!(cfg->lr >= 0) || std::isinf(cfg->lr) || !(cfg->beta1 >= 0 && cfg->beta1 < 1) || !(cfg->beta2 >= 0 && cfg->beta2 < 1) ||
        !(cfg->eps >= 0) || std::isinf(cfg->eps))
        return idm_set_error(IDM_ERR_INVALID, "adamw: lr and eps must be finite and not negative, the betas in [0, 1)");
    int64_t total = 0;
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    const size_t pb = cfg->param_dtype == IDM_DT_F32 ? 4 : 2, gb = cfg->grad_dtype == IDM_DT_F32 ? 4 : 2;
    for (int64_t i = 0; i < n_tensors; ++i) {
        if (sizes[i] < 0 || sizes[i] > ((int64_t)1 << 40)) return idm_set_error(IDM_ERR_INVALID, "adamw: tensor size out of range");
        if (!(weight_decay[i] >= 0) || std::isinf(weight_decay[i]))
            return idm_set_error(IDM_ERR_INVALID, "adamw: weight decay must be finite and not negative");
        total += room_of(sizes[i]);
        if (!sizes[i] || !grads_dev[i]) continue;
        if (!params_dev[i]) return idm_set_error(IDM_ERR_INVALID, "adamw: null parameter");
        if ((uintptr_t)params_dev[i] % pb || (uintptr_t)grads_dev[i] % gb) return idm_set_error(IDM_ERR_INVALID, "adamw: misaligned tensor");
        spans.push_back({(uintptr_t)params_dev[i], (uintptr_t)params_dev[i] + (size_t)sizes[i] * pb});
    }
    if (total != moments) return idm_set_error(IDM_ERR_INVALID, "adamw: the moments were made for other tensors (each takes its size rounded up to 256 entries)");
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i)
        if (spans[i].first < spans[i - 1].second) return idm_set_error(IDM_ERR_INVALID, "adamw: two parameters share memory");
    if (total && (!m_dev || !v_dev || (eight && (!m_base_dev || !v_base_dev)))) return idm_set_error(IDM_ERR_INVALID, "adamw: null moments");
    if ((uintptr_t)m_dev % 16 || (uintptr_t)v_dev % 16) return idm_set_error(IDM_ERR_INVALID, "adamw: moments must be aligned to 16 bytes");
    if (hipSetDevice(device) != hipSuccess) return idm_set_error(IDM_ERR_HIP, "adamw: no such device");
    hipStream_t s = (hipStream_t)stream;
    Coef *coef = (Coef *)scratch_dev;
    hipLaunchKernelGGL(adamw_begin_kernel, dim3(1), dim3(1), 0, s, step_dev, cfg->lr, cfg->beta1, cfg->beta2, coef);
    const float b1 = (float)cfg->beta1, c1 = (float)(1 - cfg->beta1), b2 = (float)cfg->beta2, c2 = (float)(1 - cfg->beta2);
    int64_t at = 0;
    Table tab;
    int64_t chunks = 0;
    tab.count = 0;
    auto flush = [&]() -> int {
        if (!tab.count) return IDM_OK;
        tab.first[tab.count] = chunks;
        auto go = [&](auto p, auto g) {
            using PT = decltype(p);
            using GT = decltype(g);
            auto kernel = eight ? &adamw_kernel<PT, GT, true> : &adamw_kernel<PT, GT, false>;
            hipLaunchKernelGGL(kernel, dim3((unsigned)chunks), dim3(256), 0, s, tab, (const Coef *)coef, b1, c1, b2, c2, (float)cfg->eps, m_dev,
                               v_dev, m_base_dev, v_base_dev);
            return IDM_OK;
        };
        by_types<true>(cfg->param_dtype, cfg->grad_dtype, go);
        tab.count = 0;
        chunks = 0;
        return hipGetLastError() == hipSuccess ? IDM_OK : idm_set_error(IDM_ERR_HIP, "adamw: launch failed");
    };
    for (int64_t i = 0; i < n_tensors; at += room_of(sizes[i]), ++i) {
        if (!sizes[i] || !grads_dev[i]) continue;      // no gradient: the tensor and its moments stay as they are
        // a tensor of more chunks than one launch has workgroups is cut
        const int64_t most = (int64_t)1 << 30;
        for (int64_t lo = 0; lo < sizes[i]; lo += most * CHUNK) {
            const int64_t n = std::min<int64_t>(sizes[i] - lo, most * CHUNK), c = (n + CHUNK - 1) / CHUNK;
            if (tab.count == TENSORS || chunks + c > 0x7fffffff) {
                const int rc = flush();
                if (rc != IDM_OK) return rc;
            }
            const int k = tab.count++;
            tab.p[k] = (char *)params_dev[i] + lo * pb;
            tab.g[k] = (const char *)grads_dev[i] + lo * gb;
            tab.n[k] = n;
            tab.at[k] = at + lo;
            tab.first[k] = chunks;
            tab.keep[k] = (float)(1.0 - cfg->lr * (double)weight_decay[i]);
            chunks += c;
        }
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
    if (hipSetDevice(device) != hipSuccess) return idm_set_error(IDM_ERR_HIP, "adamw: no such device");
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)((moments / 4 + 255) / 256)), dim3(256), 0, (hipStream_t)stream, m_dev, v_dev,
                       m_base_dev, v_base_dev, m_out_dev, v_out_dev, moments);
    return hipGetLastError() == hipSuccess ? IDM_OK : idm_set_error(IDM_ERR_HIP, "adamw: launch failed");
}

}  // extern "C"
