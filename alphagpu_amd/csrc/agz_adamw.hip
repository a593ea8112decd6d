// agz_adamw.hip — one AdamW step over many tensors (include/agz.h agz_adamw_step), states in 32 or in 8 bits.
#include "agz_ops.hpp"
#include <cmath>

namespace agz {
namespace ops {

static thread_local char g_ops_error[512];
int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_ops_error, sizeof g_ops_error, fmt, ap);
    va_end(ap);
    return code;
}

// tensors of one launch, in the kernel's arguments (no table in device memory to keep, copy or wait for): 96 x 32 bytes
constexpr int AW_MAX = 96;
constexpr int AW_BLOCK = 128;            // elements per scale
struct AwTensor { void* p; const void* g; uint32_t n_lo, n_hi, chunk0, block0; };   // chunk0, block0: of this launch
struct AwTable { AwTensor t[AW_MAX]; };
struct AwPar {
    float b1, b2, c1, c2, eps, keep;          // c1 = 1 - b1, c2 = 1 - b2; keep = 1 - lr decay
    float step_size, inv_root;                // lr / (1 - b1^t), 1 / sqrt(1 - b2^t): of the host's t
    double b1d, b2d, lrd;                     // ... and what a t in device memory needs
    const int64_t* step_dev;
    int64_t step;
    uint32_t seed, tensor0;
    int count;
};

__host__ __device__ __forceinline__ uint32_t aw_mix(uint32_t h) {
    h *= 0x9E3779B1u; h ^= h >> 16; h *= 0xB504F335u; return h ^ (h >> 16);
}
__host__ __device__ __forceinline__ uint32_t aw_key(uint32_t seed, uint32_t step, uint32_t tensor) { return aw_mix(aw_mix(aw_mix(seed + 0x3C6EF372u) ^ step) + tensor); }

__device__ __forceinline__ double aw_pow(double b, uint64_t t) { double r = 1.0; for (; t; t >>= 1, b *= b) if (t & 1) r *= b; return r; }

// y in [0, 448] to a value of e4m3: up with the probability of its place between its two neighbours (u: 16 random bits).  Below the
// normal numbers the spacing is that of 2^-6: added before, taken off after.
__device__ __forceinline__ float aw_round(float y, uint32_t u) {
    const float low = y < 0.015625f ? 0.015625f : 0.0f;
    const uint32_t t = (__float_as_uint(y + low) + (u << 4)) & ~0xFFFFFu;
    return __uint_as_float(t) - low;
}

// the simple form: one wave per block of 128 elements, two elements per lane
template <typename P, typename G, int BITS>
__global__ __launch_bounds__(256) void k_adamw(AwTable tab, AwPar a, void* mp, void* vp, uint8_t* ms, uint8_t* vs) {
    const int lane = threadIdx.x & 63;
    const uint32_t chunk = blockIdx.x * 4 + (threadIdx.x >> 6);
    int lo = 0, hi = a.count;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (tab.t[mid].chunk0 <= chunk) lo = mid; else hi = mid; }
    const AwTensor t = tab.t[lo];
    const int64_t n = (int64_t)((uint64_t)t.n_hi << 32 | t.n_lo);
    const int64_t blk = chunk - t.chunk0;
    if (blk * AW_BLOCK >= n) return;
    int64_t step = a.step;
    float step_size = a.step_size, inv_root = a.inv_root;
    if (a.step_dev) {
        step = *a.step_dev;
        step_size = (float)(a.lrd / (1.0 - aw_pow(a.b1d, step)));
        inv_root = (float)(1.0 / sqrt(1.0 - aw_pow(a.b2d, step)));
    }
    const uint32_t key = aw_key(a.seed, (uint32_t)step, a.tensor0 + lo);
    const int64_t state0 = ((int64_t)t.block0 + blk) * AW_BLOCK;
    float m[2], r[2], v[2];
    float m_scale = 1.0f, r_scale = 1.0f;
    if (BITS == 8) { m_scale = scale_of(ms[t.block0 + blk]); r_scale = scale_of(vs[t.block0 + blk]); }
    for (int k = 0; k < 2; ++k) {
        const int64_t i = blk * AW_BLOCK + lane * 2 + k, si = state0 + lane * 2 + k;
        const bool in = i < n;
        const float g = in ? to_f(((const G*)t.g)[i]) : 0.0f;
        if (BITS == 32) { m[k] = ((const float*)mp)[si]; v[k] = ((const float*)vp)[si]; }
        else {
            m[k] = __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)mp)[si], 0) * m_scale;
            const float rr = __builtin_amdgcn_cvt_f32_fp8((int)((const uint8_t*)vp)[si], 0) * r_scale;
            v[k] = rr * rr;
        }
        m[k] = m[k] * a.b1 + g * a.c1;
        v[k] = v[k] * a.b2 + (g * g) * a.c2;
        r[k] = sqrtf(v[k]);
        if (in) {
            P* p = (P*)t.p + i;
            *p = from_f<P>(to_f(*p) * a.keep - (m[k] * step_size) / (r[k] * inv_root + a.eps));
        }
        if (BITS == 32) { ((float*)mp)[si] = m[k]; ((float*)vp)[si] = v[k]; }
    }
    if (BITS == 8) {
        float am = 0.0f, ar = 0.0f;
        for (int k = 0; k < 2; ++k) { am = fmaxf(am, fabsf(m[k]) < INFINITY ? fabsf(m[k]) : 0.0f); ar = fmaxf(ar, r[k] < INFINITY ? r[k] : 0.0f); }
        const int bm = scale_byte(wave_max(am)), br = scale_byte(wave_max(ar));
        const float im = inv_scale_of(bm), ir = inv_scale_of(br);
        for (int k = 0; k < 2; ++k) {
            const int64_t i = blk * AW_BLOCK + lane * 2 + k, si = state0 + lane * 2 + k;
            const uint32_t h = aw_mix((uint32_t)i ^ (key + (uint32_t)(i >> 32) * 0x9E3779B1u));
            const float ym = fabsf(m[k]) * im, yr = r[k] * ir;
            float qm = ym < INFINITY ? copysignf(aw_round(ym, h & 0xFFFFu), m[k]) : NAN;
            float qr = yr < INFINITY ? aw_round(yr, h >> 16) : NAN;
            if (yr > 0.0f) qr = fmaxf(qr, 0.001953125f);
            if (!(yr < INFINITY)) qr = NAN;
            const int w = __builtin_amdgcn_cvt_pk_fp8_f32(qm, qr, 0, false);
            ((uint8_t*)mp)[si] = (uint8_t)(w & 0xFF);
            ((uint8_t*)vp)[si] = (uint8_t)(w >> 8 & 0xFF);
        }
        if (lane == 0) { ms[t.block0 + blk] = (uint8_t)bm; vs[t.block0 + blk] = (uint8_t)br; }
    }
}

}  // namespace ops
}  // namespace agz

using namespace agz::ops;

extern "C" {

const char* agz_ops_last_error(void) { return g_ops_error; }

int64_t agz_adamw_state_elements(int count, const int64_t* numel) {
    if (count < 0 || (count > 0 && !numel)) return -1;
    int64_t blocks = 0;
    for (int i = 0; i < count; ++i) {
        if (numel[i] < 0 || numel[i] > ((int64_t)1 << 46)) return -1;
        blocks += cdiv(numel[i], AW_BLOCK);
    }
    return blocks * AW_BLOCK;
}

int agz_adamw_step(int device, void* stream, const agz_adamw_options* o, int count, void* const* params, const void* const* grads, const int64_t* numel,
                   void* m, void* v, void* m_scale, void* v_scale) {
    if (!o) return fail(AGZ_ERR_ARG, "agz_adamw_step: no options");
    if (count < 0 || (count > 0 && (!params || !grads || !numel || !m || !v))) return fail(AGZ_ERR_ARG, "agz_adamw_step: null argument");
    if (!good_dtype(o->param_dtype) || !good_dtype(o->grad_dtype)) return fail(AGZ_ERR_ARG, "agz_adamw_step: unknown dtype");
    if (o->bits != 8 && o->bits != 32) return fail(AGZ_ERR_ARG, "agz_adamw_step: states of %d bits (8 or 32)", o->bits);
    if (o->bits == 8 && count > 0 && (!m_scale || !v_scale)) return fail(AGZ_ERR_ARG, "agz_adamw_step: 8-bit states need their scales");
    if (!o->step_dev && o->step < 1) return fail(AGZ_ERR_ARG, "agz_adamw_step: step %lld (from 1 on)", (long long)o->step);
    if (!(o->beta1 >= 0 && o->beta1 < 1) || !(o->beta2 >= 0 && o->beta2 < 1) || !(o->eps >= 0) || !(o->lr >= 0) || !(o->weight_decay >= 0))
        return fail(AGZ_ERR_ARG, "agz_adamw_step: lr, eps, weight_decay >= 0 and betas in [0, 1)");
    if (agz_adamw_state_elements(count, numel) < 0) return fail(AGZ_ERR_ARG, "agz_adamw_step: a negative or far too large tensor");
    if (count > 0 && (!aligned(m, 16) || !aligned(v, 16))) return fail(AGZ_ERR_ARG, "agz_adamw_step: the states have to begin at a multiple of 16 bytes");
    for (int i = 0; i < count; ++i) {
        if (numel[i] == 0 || !grads[i]) continue;
        if (!params[i]) return fail(AGZ_ERR_ARG, "agz_adamw_step: tensor %d is null", i);
        if (!aligned(params[i], esize(o->param_dtype)) || !aligned(grads[i], esize(o->grad_dtype))) return fail(AGZ_ERR_ARG, "agz_adamw_step: tensor %d is not aligned to its type", i);
    }
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;

    AwPar a{};
    a.b1 = (float)o->beta1; a.b2 = (float)o->beta2; a.c1 = (float)(1.0 - o->beta1); a.c2 = (float)(1.0 - o->beta2);
    a.eps = (float)o->eps; a.keep = (float)(1.0 - o->lr * o->weight_decay);
    a.b1d = o->beta1; a.b2d = o->beta2; a.lrd = o->lr; a.step_dev = o->step_dev; a.step = o->step_dev ? 0 : o->step;
    if (!o->step_dev) {
        a.step_size = (float)(o->lr / (1.0 - std::pow(a.b1d, (double)o->step)));
        a.inv_root = (float)(1.0 / std::sqrt(1.0 - std::pow(a.b2d, (double)o->step)));
    }
    a.seed = o->seed;
    // launches of at most AW_MAX tensors and 2^30 blocks; a tensor of more is cut at a block (its hash index would not be: such a tensor is refused)
    int i = 0;
    int64_t state_block = 0;
    while (i < count) {
        AwTable tab;
        uint32_t chunks = 0;
        const int64_t base = state_block;
        int k = 0;
        const int first = i;
        for (; i < count && k < AW_MAX; ++i) {
            const int64_t blocks = cdiv(numel[i], AW_BLOCK);
            if (blocks > (1ll << 29)) return fail(AGZ_ERR_ARG, "agz_adamw_step: tensor %d has more than 2^36 elements", i);
            if (k > 0 && (state_block - base) + blocks > (1ll << 30)) break;
            tab.t[k++] = AwTensor{params[i], grads[i], (uint32_t)numel[i], (uint32_t)(numel[i] >> 32), chunks, (uint32_t)(state_block - base)};
            chunks += grads[i] ? (uint32_t)blocks : 0;
            state_block += blocks;
        }
        if (chunks == 0) continue;
        a.count = k;
        a.tensor0 = (uint32_t)(o->tensor_base + first);
        const int bytes = o->bits == 32 ? 4 : 1;
        void* mp = (char*)m + base * AW_BLOCK * bytes;
        void* vp = (char*)v + base * AW_BLOCK * bytes;
        uint8_t* ms = o->bits == 8 ? (uint8_t*)m_scale + base : nullptr;
        uint8_t* vs = o->bits == 8 ? (uint8_t*)v_scale + base : nullptr;
        const int rc = by_dtype(o->param_dtype, [&](auto P) { return by_dtype(o->grad_dtype, [&](auto G) {
            return o->bits == 8 ? launch(k_adamw<decltype(P), decltype(G), 8>, dim3((chunks + 3) / 4), dim3(256), 0, stream, tab, a, mp, vp, ms, vs)
                                : launch(k_adamw<decltype(P), decltype(G), 32>, dim3((chunks + 3) / 4), dim3(256), 0, stream, tab, a, mp, vp, ms, vs);
        }); });
        if (rc != AGZ_OK) return rc;
    }
    return AGZ_OK;
}

}  // extern "C"
