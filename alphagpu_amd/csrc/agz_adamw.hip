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
struct AwTensor { void* p; const void* g; uint32_t n_lo; uint16_t n_hi, count; uint32_t chunk0, block0; };   // count: which of AwPar's; chunk0, block0: of this launch
struct AwTable { AwTensor t[AW_MAX]; };
// what the number of steps that a tensor has taken comes to: tensors with equal numbers share one, and a launch has AW_COUNTS of them (most have one: no tensor missed a gradient)
constexpr int AW_COUNTS = 16;
struct AwCount { float step_size, inv_root; uint32_t t; };    // lr / (1 - b1^t), 1 / sqrt(1 - b2^t)
struct AwPar {
    float b1, b2, c1, c2, eps, keep;          // c1 = 1 - b1, c2 = 1 - b2; keep = 1 - lr decay
    AwCount c[AW_COUNTS];                     // of the host's t
    double b1d, b2d, lrd;                     // ... and what a t in device memory needs
    const int64_t *step_dev, *missed_dev;     // (missed_dev: of this launch's first tensor)
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

// A workgroup takes AW_CHUNK neighbouring elements of one tensor, a lane AW_TURNS times four of them: every access is 16 (8, 4) bytes a lane and whole lines a
// wave, and all of a lane's loads are under way before the first is used.  A block of 128 is half a wave: its largest is a reduction over 32 lanes.
constexpr int AW_TURNS = 2, AW_CHUNK = 256 * 4 * AW_TURNS, AW_BLOCKS = AW_CHUNK / AW_BLOCK;
constexpr int64_t AW_MOST = 1ll << 27;      // blocks of a launch: 2^23 workgroups of 256 lanes, and one more a tensor (a launch has fewer than 2^32 lanes)

template <typename T> __device__ __forceinline__ void load4(float* to, const T* from, int64_t i, int64_t n) {
    if (i + 4 <= n) {
        const Span<T, 4> v = *(const Span<T, 4>*)(from + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = to_f(v.e[e]);
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e) to[e] = i + e < n ? to_f(from[i + e]) : 0.0f;
}
// what is held for four elements in 8 bits: rounded as aw_round says; NaN for what is not finite (a block's scale counts its finite entries)
template <bool FLOOR> __device__ __forceinline__ uint32_t aw_hold(const float* x, const uint32_t* u, uint8_t* scale, bool first) {
    float m = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
    if (__any(m == INFINITY)) {
        m = 0.0f;
        for (int e = 0; e < 4; ++e) m = fmaxf(m, fabsf(x[e]) < INFINITY ? fabsf(x[e]) : 0.0f);
    }
    const int b = scale_byte(lanes_max<32>(m));
    if (first) *scale = (uint8_t)b;
    const float inv = inv_scale_of(b);
    float q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float y = fabsf(x[e]) * inv;
        q[e] = aw_round(y, u[e]);
        if (FLOOR) q[e] = y > 0.0f ? fmaxf(q[e], 0.001953125f) : q[e];
        else q[e] = copysignf(q[e], x[e]);
        if (!(y < INFINITY)) q[e] = NAN;
    }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
}

// One pass: every tensor, gradient and state is read and written once.  Bound by memory: 67 M weights in 32 bits 348 us (1.88 GB, 5.4 TB/s), states in 8 bits with bf16
// gradients 176-186 us in a run of calls (942 MB, 5.1-5.4 TB/s; launches in a row under a profiler 165 us at first, up to 280 us later); the eleven tensors of a
// 128-wide network 4.4-5.0 us, the launch.
template <typename P, typename G, int BITS>
__global__ __launch_bounds__(256) void k_adamw(AwTable tab, AwPar a, void* mp, void* vp, uint8_t* ms, uint8_t* vs) {
    const int tid = threadIdx.x;
    int lo = 0, hi = a.count;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (tab.t[mid].chunk0 <= blockIdx.x) lo = mid; else hi = mid; }
    const AwTensor t = tab.t[lo];
    const int64_t n = (int64_t)((uint64_t)t.n_hi << 32 | t.n_lo), chunk = blockIdx.x - t.chunk0;
    const int64_t full = (n + AW_BLOCK - 1) / AW_BLOCK * AW_BLOCK;          // the states go to the end of the last block
    const int64_t i0 = chunk * AW_CHUNK + tid * 4, s0 = (int64_t)t.block0 * AW_BLOCK;
    float p[AW_TURNS][4], g[AW_TURNS][4], m[AW_TURNS][4], v[AW_TURNS][4];
    uint32_t mq[AW_TURNS], vq[AW_TURNS];
    uint8_t mb[AW_TURNS], vb[AW_TURNS];
#pragma unroll
    for (int k = 0; k < AW_TURNS; ++k) {
        const int64_t i = i0 + k * 1024;
        if (i >= full) continue;
        if (BITS == 32) {
            *(float4*)m[k] = *(const float4*)((const float*)mp + s0 + i);
            *(float4*)v[k] = *(const float4*)((const float*)vp + s0 + i);
        } else {
            mq[k] = *(const uint32_t*)((const uint8_t*)mp + s0 + i);
            vq[k] = *(const uint32_t*)((const uint8_t*)vp + s0 + i);
            mb[k] = ms[(s0 + i) / AW_BLOCK];
            vb[k] = vs[(s0 + i) / AW_BLOCK];
        }
        load4(g[k], (const G*)t.g, i, n);
        load4(p[k], (const P*)t.p, i, n);
    }
    AwCount c = a.c[t.count];
    if (a.step_dev) {
        const int64_t step = *a.step_dev - (a.missed_dev ? a.missed_dev[lo] : 0);
        c = {(float)(a.lrd / (1.0 - aw_pow(a.b1d, step))), (float)(1.0 / sqrt(1.0 - aw_pow(a.b2d, step))), (uint32_t)step};
    }
    const uint32_t key = aw_key(a.seed, c.t, a.tensor0 + lo);
#pragma unroll
    for (int k = 0; k < AW_TURNS; ++k) {
        const int64_t i = i0 + k * 1024;
        if (i >= full) continue;                               // (a whole half wave: blocks begin at multiples of 32 lanes)
        if (BITS == 8) {
            const float fm = scale_of(mb[k]), fv = scale_of(vb[k]);
            const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mq[k], false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mq[k], true);
            const auto v01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vq[k], false), v23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vq[k], true);
            m[k][0] = m01[0] * fm; m[k][1] = m01[1] * fm; m[k][2] = m23[0] * fm; m[k][3] = m23[1] * fm;
            v[k][0] = v01[0] * fv; v[k][1] = v01[1] * fv; v[k][2] = v23[0] * fv; v[k][3] = v23[1] * fv;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[k][e] *= v[k][e];
        }
        float r[4];
        uint32_t um[4], ur[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            m[k][e] = m[k][e] * a.b1 + g[k][e] * a.c1;
            v[k][e] = v[k][e] * a.b2 + (g[k][e] * g[k][e]) * a.c2;
            r[e] = sqrtf(v[k][e]);
            p[k][e] = p[k][e] * a.keep - (m[k][e] * c.step_size) / (r[e] * c.inv_root + a.eps);
            if (BITS == 8) {
                const uint32_t h = aw_mix((uint32_t)(i + e) ^ (key + (uint32_t)(i >> 32) * 0x9E3779B1u));
                um[e] = h & 0xFFFFu; ur[e] = h >> 16;
            }
        }
        if (i + 4 <= n) {
            Span<P, 4> o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o.e[e] = from_f<P>(p[k][e]);
            *(Span<P, 4>*)((P*)t.p + i) = o;
        } else
#pragma unroll
            for (int e = 0; e < 4; ++e) if (i + e < n) ((P*)t.p)[i + e] = from_f<P>(p[k][e]);
        if (BITS == 32) {
            *(float4*)((float*)mp + s0 + i) = make_float4(m[k][0], m[k][1], m[k][2], m[k][3]);
            *(float4*)((float*)vp + s0 + i) = make_float4(v[k][0], v[k][1], v[k][2], v[k][3]);
        } else {
            const bool first = (tid & 31) == 0;
            *(uint32_t*)((uint8_t*)mp + s0 + i) = aw_hold<false>(m[k], um, ms + (s0 + i) / AW_BLOCK, first);
            *(uint32_t*)((uint8_t*)vp + s0 + i) = aw_hold<true>(r, ur, vs + (s0 + i) / AW_BLOCK, first);
        }
    }
}

// one more missed step for the tensors of a launch that have no gradient
struct AwMissing { uint32_t bit[AW_MAX / 32]; };
__global__ __launch_bounds__(AW_MAX) void k_adamw_missed(AwMissing b, int64_t* missed) {
    const int i = threadIdx.x;
    if (b.bit[i >> 5] >> (i & 31) & 1) ++missed[i];
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
    return agz_adamw_step_missed(device, stream, o, nullptr, nullptr, count, params, grads, numel, m, v, m_scale, v_scale);
}

int agz_adamw_step_missed(int device, void* stream, const agz_adamw_options* o, const int64_t* missed, int64_t* missed_dev, int count, void* const* params, const void* const* grads,
                          const int64_t* numel, void* m, void* v, void* m_scale, void* v_scale) {
    if (!o) return fail(AGZ_ERR_ARG, "agz_adamw_step: no options");
    if (count < 0 || (count > 0 && (!params || !grads || !numel))) return fail(AGZ_ERR_ARG, "agz_adamw_step: null argument");
    if (!good_dtype(o->param_dtype) || !good_dtype(o->grad_dtype)) return fail(AGZ_ERR_ARG, "agz_adamw_step: unknown dtype");
    if (o->bits != 8 && o->bits != 32) return fail(AGZ_ERR_ARG, "agz_adamw_step: states of %d bits (8 or 32)", o->bits);
    const int64_t elements = agz_adamw_state_elements(count, numel);
    if (elements < 0) return fail(AGZ_ERR_ARG, "agz_adamw_step: a negative or far too large tensor");
    if (elements > 0 && (!m || !v)) return fail(AGZ_ERR_ARG, "agz_adamw_step: null argument");
    if (o->bits == 8 && elements > 0 && (!m_scale || !v_scale)) return fail(AGZ_ERR_ARG, "agz_adamw_step: 8-bit states need their scales");
    if (!o->step_dev && o->step < 1) return fail(AGZ_ERR_ARG, "agz_adamw_step: step %lld (from 1 on)", (long long)o->step);
    if (!o->step_dev && missed_dev) return fail(AGZ_ERR_ARG, "agz_adamw_step: missed_dev goes with step_dev");
    if (!aligned(o->step_dev, 8) || !aligned(missed_dev, 8)) return fail(AGZ_ERR_ARG, "agz_adamw_step: step_dev and missed_dev are not aligned to 8 bytes");
    if (o->step_dev) missed = nullptr;
    if (missed) for (int i = 0; i < count; ++i)
        if (missed[i] < 0 || missed[i] >= o->step) return fail(AGZ_ERR_ARG, "agz_adamw_step: tensor %d missed %lld of the %lld steps before this one", i, (long long)missed[i], (long long)o->step - 1);
    if (!(o->beta1 >= 0 && o->beta1 < 1) || !(o->beta2 >= 0 && o->beta2 < 1) || !(o->eps >= 0) || !(o->lr >= 0) || !(o->weight_decay >= 0))
        return fail(AGZ_ERR_ARG, "agz_adamw_step: lr, eps, weight_decay >= 0 and betas in [0, 1)");
    if (!aligned(m, 16) || !aligned(v, 16)) return fail(AGZ_ERR_ARG, "agz_adamw_step: the states have to begin at a multiple of 16 bytes");
    for (int i = 0; i < count; ++i) {
        if (cdiv(numel[i], AW_BLOCK) > AW_MOST) return fail(AGZ_ERR_ARG, "agz_adamw_step: tensor %d has more than 2^34 elements", i);
        if (numel[i] == 0 || !grads[i]) continue;
        if (!params[i]) return fail(AGZ_ERR_ARG, "agz_adamw_step: tensor %d is null", i);
        if (!aligned(params[i], esize(o->param_dtype)) || !aligned(grads[i], esize(o->grad_dtype))) return fail(AGZ_ERR_ARG, "agz_adamw_step: tensor %d is not aligned to its type", i);
    }
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;

    AwPar a{};
    a.b1 = (float)o->beta1; a.b2 = (float)o->beta2; a.c1 = (float)(1.0 - o->beta1); a.c2 = (float)(1.0 - o->beta2);
    a.eps = (float)o->eps; a.keep = (float)(1.0 - o->lr * o->weight_decay);
    a.b1d = o->beta1; a.b2d = o->beta2; a.lrd = o->lr; a.step_dev = o->step_dev;
    a.seed = o->seed;
    // launches of at most AW_MAX tensors, AW_MOST blocks and AW_COUNTS numbers of steps
    int64_t at[AW_COUNTS];                       // the numbers of steps of this launch (with step_dev: none)
    int i = 0;
    int64_t state_block = 0;
    while (i < count) {
        AwTable tab;
        AwMissing missing{};
        uint32_t chunks = 0;
        const int64_t base = state_block;
        int k = 0, counts = 0;
        const int first = i;
        for (; i < count && k < AW_MAX; ++i) {
            const int64_t blocks = cdiv(numel[i], AW_BLOCK);
            if (k > 0 && (state_block - base) + blocks > AW_MOST) break;
            int c = 0;
            if (!grads[i]) missing.bit[k >> 5] |= 1u << (k & 31);
            else if (!o->step_dev) {
                const int64_t t = o->step - (missed ? missed[i] : 0);
                while (c < counts && at[c] != t) ++c;
                if (c == AW_COUNTS) break;
                if (c == counts) {
                    at[counts++] = t;
                    a.c[c] = {(float)(o->lr / (1.0 - std::pow(a.b1d, (double)t))), (float)(1.0 / std::sqrt(1.0 - std::pow(a.b2d, (double)t))), (uint32_t)t};
                }
            }
            tab.t[k++] = AwTensor{params[i], grads[i], (uint32_t)numel[i], (uint16_t)(numel[i] >> 32), (uint16_t)c, chunks, (uint32_t)(state_block - base)};
            chunks += grads[i] ? (uint32_t)cdiv(blocks, AW_BLOCKS) : 0;
            state_block += blocks;
        }
        a.missed_dev = missed_dev ? missed_dev + first : nullptr;
        if (missed_dev && (missing.bit[0] | missing.bit[1] | missing.bit[2]))
            if (const int rc = launch(k_adamw_missed, dim3(1), dim3(AW_MAX), 0, stream, missing, missed_dev + first)) return rc;
        if (chunks == 0) continue;
        a.count = k;
        a.tensor0 = (uint32_t)(o->tensor_base + first);
        const int bytes = o->bits == 32 ? 4 : 1;
        void* mp = (char*)m + base * AW_BLOCK * bytes;
        void* vp = (char*)v + base * AW_BLOCK * bytes;
        uint8_t* ms = o->bits == 8 ? (uint8_t*)m_scale + base : nullptr;
        uint8_t* vs = o->bits == 8 ? (uint8_t*)v_scale + base : nullptr;
        const int rc = by_dtype(o->param_dtype, [&](auto P) { return by_dtype(o->grad_dtype, [&](auto G) {
            return o->bits == 8 ? launch(k_adamw<decltype(P), decltype(G), 8>, dim3(chunks), dim3(256), 0, stream, tab, a, mp, vp, ms, vs)
                                : launch(k_adamw<decltype(P), decltype(G), 32>, dim3(chunks), dim3(256), 0, stream, tab, a, mp, vp, ms, vs);
        }); });
        if (rc != AGZ_OK) return rc;
    }
    return AGZ_OK;
}

}  // extern "C"
