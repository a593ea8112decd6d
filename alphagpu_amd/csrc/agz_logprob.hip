// agz_logprob.hip — log probabilities of given moves, entropy, best alternatives and the policy term of a loss, with their gradient
// (include/agz.h agz_logprob_forward / _backward; the softmax of mcts_gpu.jl:417 and the policy loss of train.jl:12-15).
#include "agz_ops.hpp"
#include <type_traits>

namespace agz {
namespace ops {

constexpr float LOG2E = 1.4426950408889634f;

struct LpPar {
    int64_t n; int32_t a, top;
    const void* x; int64_t ld;
    const uint8_t* mask; int64_t ld_mask;
    const int64_t* moves;
    const float* target; int64_t ld_target;
    float *move_logp, *entropy, *target_logp, *top_logp;
    int32_t* top_move;
    float* stats;
    const float *g_move, *g_entropy, *g_target, *g_top;
    void* dx; int64_t ldd;
};

// ---------------------------------------------------------------------------------------------------------------------------------------
// A row, or a part of one, in the registers of G neighbouring lanes: lane l of the group holds the elements VEC (l + G i) .. + VEC - 1 of
// i = 0 .. NV - 1, read as one span each (16 bytes for VEC = 16 / sizeof(T); an element that is not allowed is -inf).  The last span is the VEC elements that
// end with the row; of those the ones before the span's own start belong to the span before it and count as not there.
// ---------------------------------------------------------------------------------------------------------------------------------------
template <typename T, int VEC, int G, int NV> struct Row {
    float x[NV * VEC];
    int32_t at[NV];                                            // index of x[i * VEC]; its own elements are those from VEC (l + G i) on

    __device__ __forceinline__ void load(const T* row, const uint8_t* mask, int32_t first, int32_t a, int l) {
        Span<T, VEC> v[NV];
        Span<uint8_t, VEC> m[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int32_t own = first + VEC * (l + G * i);
            at[i] = own < a - VEC ? own : a - VEC;
            if (own < a) {
                v[i] = *(const Span<T, VEC>*)(row + at[i]);
                if (mask) m[i] = *(const Span<uint8_t, VEC>*)(mask + at[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int32_t own = first + VEC * (l + G * i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const bool in = own < a && at[i] + e >= own && (!mask || m[i].e[e]);
                x[i * VEC + e] = in ? to_f(v[i].e[e]) : -INFINITY;
            }
        }
    }
};

// what a row or a part of one adds up to: largest entry, sum of e^d and of d e^d (d = x - largest), of t d and of t
struct Sums { float mx, s, sd, tx, ts; };
__device__ __forceinline__ float base_of(float mx) { return mx == -INFINITY ? 0.0f : mx; }

template <typename T, int VEC, int G, int NV>
__device__ __forceinline__ Sums row_sums(const Row<T, VEC, G, NV>& r, const float* target, int32_t first, int32_t a, int l) {
    Span<float, VEC> t[NV];
    if (target)
#pragma unroll
        for (int i = 0; i < NV; ++i) if (first + VEC * (l + G * i) < a) t[i] = *(const Span<float, VEC>*)(target + r.at[i]);
    Sums o{-INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < NV * VEC; ++k) o.mx = fmaxf(o.mx, r.x[k]);
    o.mx = lanes_max<G>(o.mx);
    const float base = base_of(o.mx);
#pragma unroll
    for (int k = 0; k < NV * VEC; ++k) {
        const float d = r.x[k] - base, e = __builtin_amdgcn_exp2f(d * LOG2E);
        o.s += e;
        o.sd += e * fmaxf(d, -3.0e38f);                        // (0 * -inf)
    }
    o.s = lanes_sum<G>(o.s);
    o.sd = lanes_sum<G>(o.sd);
    if (target) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int32_t own = first + VEC * (l + G * i);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float w = own < a && r.at[i] + e >= own ? t[i].e[e] : 0.0f;
                o.ts += w;
                o.tx += w != 0.0f ? w * (r.x[i * VEC + e] - base) : 0.0f;
            }
        }
        o.tx = lanes_sum<G>(o.tx);
        o.ts = lanes_sum<G>(o.ts);
    }
    return o;
}

// The next best entry of what G lanes hold, taken out of it: its value (-inf: none is left) and its index.  Equal entries by index: every lane offers the
// first of its largest, the lowest index among the lanes whose offer is the largest wins.
template <int N> struct Offer { float v; uint32_t j; int k; };
template <typename T, int VEC, int G, int NV> __device__ __forceinline__ Offer<0> offer(const Row<T, VEC, G, NV>& r) {
    Offer<0> o{-INFINITY, 0xFFFFFFFFu, -1};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
            if (r.x[i * VEC + e] > o.v) { o.v = r.x[i * VEC + e]; o.j = (uint32_t)(r.at[i] + e); o.k = i * VEC + e; }
    return o;
}
template <typename T, int VEC, int G, int NV> __device__ __forceinline__ float take_best(Row<T, VEC, G, NV>& r, Offer<0>& o, uint32_t& j) {
    const float best = lanes_max<G>(o.v);
    j = lanes_min_u<G>(o.v == best ? o.j : 0xFFFFFFFFu);
    if (best > -INFINITY && o.j == j) {
#pragma unroll
        for (int k = 0; k < NV * VEC; ++k) if (k == o.k) r.x[k] = -INFINITY;
        o = offer(r);
    }
    return best;
}

// a row's results from its sums; every lane of the group has them
struct Done { float ls, h; bool bad; };
__device__ __forceinline__ Done finish(const LpPar& p, int64_t i, const Sums& q, float xm, bool given, bool writes) {
    const bool none = q.s == 0.0f, bad = !(q.s < INFINITY);
    const float ls = none ? 0.0f : (bad ? NAN : logf(q.s)), base = base_of(q.mx);
    const float h = none ? 0.0f : ls - q.sd / q.s;
    if (writes) {
        *(float4*)(p.stats + i * 4) = make_float4(base, ls, h, q.ts);
        if (p.entropy) p.entropy[i] = h;
        if (p.target_logp) p.target_logp[i] = q.tx - ls * q.ts;
        if (p.move_logp) p.move_logp[i] = bad ? NAN : (given ? xm - base - ls : 0.0f);
    }
    return {ls, h, bad};
}
// the logit of the given move (-inf: not allowed)
template <typename T> __device__ __forceinline__ float given_logit(const LpPar& p, const T* x, const uint8_t* mask, int64_t i, bool& given) {
    const int64_t mv = p.move_logp ? p.moves[i] : -1;
    given = mv >= 0 && mv < p.a;
    if (!given) return 0.0f;
    const float v = to_f(x[mv]);
    return !mask || mask[mv] ? v : -INFINITY;
}

// A row per group of G lanes: rows of up to G NV VEC actions.  One pass: the row is read once and stays in registers.
template <typename T, int VEC, int G, int NV> __global__ __launch_bounds__(256) void k_logprob(LpPar p) {
    const int l = threadIdx.x & (G - 1);
    const int64_t i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (i >= p.n) return;
    const T* x = (const T*)p.x + i * p.ld;
    const uint8_t* mask = p.mask ? p.mask + i * p.ld_mask : nullptr;
    bool given;
    const float xm = given_logit(p, x, mask, i, given);
    Row<T, VEC, G, NV> r;
    r.load(x, mask, 0, p.a, l);
    const Sums q = row_sums(r, p.target ? p.target + i * p.ld_target : nullptr, 0, p.a, l);
    const Done f = finish(p, i, q, xm, given, l == 0);
    if (p.top > 0) {
        const float off = base_of(q.mx);
        auto o = offer(r);
        for (int k = 0; k < p.top; ++k) {
            uint32_t j;
            const float v = take_best(r, o, j);
            if (l == 0) {
                const bool some = v > -INFINITY && !f.bad;
                if (p.top_move) p.top_move[i * p.top + k] = some ? (int32_t)j : -1;
                if (p.top_logp) p.top_logp[i * p.top + k] = some ? v - off - f.ls : (f.bad ? NAN : -INFINITY);
            }
        }
    }
}

// Longer rows: one wave per part of PART elements leaves the part's sums and best alternatives (as keys) in the workspace, a second launch joins
// the parts of a row.  Parts of one size whatever the number of rows: one row of 131072 is 64 waves, 4096 rows of 50001 are 102400.
constexpr int PART = 2048;
struct PartOut { Sums q; float pad[3]; };

// order of the alternatives as one unsigned number: larger logits first, then lower indices; 0 = none
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t j) {
    uint32_t b = __float_as_uint(x + 0.0f);                  // (-0 -> +0: equal logits)
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (uint64_t)b << 32 | (uint32_t)~j;
}
__device__ __forceinline__ float lp_key_value(uint64_t k) {
    const uint32_t b = (uint32_t)(k >> 32);
    return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}
__device__ __forceinline__ uint64_t wave_max_u64(uint64_t x) {
    const uint32_t hi = lanes_reduce<64>((uint32_t)(x >> 32), [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    const uint32_t lo = lanes_reduce<64>((uint32_t)(x >> 32) == hi ? (uint32_t)x : 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
    return (uint64_t)hi << 32 | lo;
}

template <typename T, int VEC, int NV> __global__ __launch_bounds__(256) void k_logprob_part(LpPar p, int32_t parts, PartOut* part, uint64_t* keys) {
    const int l = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t i = w / parts;
    if (i >= p.n) return;
    const int32_t first = (int32_t)(w - i * parts) * PART;
    const int32_t end = p.a - first > PART ? first + PART : p.a;
    const T* x = (const T*)p.x + i * p.ld;
    Row<T, VEC, 64, NV> r;
    r.load(x, p.mask ? p.mask + i * p.ld_mask : nullptr, first, end, l);
    const Sums q = row_sums(r, p.target ? p.target + i * p.ld_target : nullptr, first, end, l);
    if (l == 0) part[w].q = q;
    if (p.top > 0) {
        auto o = offer(r);
        for (int k = 0; k < p.top; ++k) {
            uint32_t j;
            const float v = take_best(r, o, j);
            if (l == 0) keys[w * p.top + k] = v > -INFINITY ? lp_key(v, j) : 0;
        }
    }
}

template <typename T> __global__ __launch_bounds__(256) void k_logprob_join(LpPar p, int32_t parts, const PartOut* part, const uint64_t* keys) {
    const int l = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= p.n) return;
    const T* x = (const T*)p.x + i * p.ld;
    bool given;
    const float xm = given_logit(p, x, p.mask ? p.mask + i * p.ld_mask : nullptr, i, given);
    part += i * parts;
    float mx = -INFINITY;
    for (int32_t k = l; k < parts; k += 64) mx = fmaxf(mx, part[k].q.mx);
    mx = wave_max(mx);
    Sums q{mx, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int32_t k = l; k < parts; k += 64) {
        const Sums t = part[k].q;
        const float d = base_of(t.mx) - base_of(mx), e = t.s == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(d * LOG2E);   // (a part without entries: base 0)
        q.s += t.s * e;
        q.sd += e > 0.0f ? e * (t.sd + d * t.s) : 0.0f;      // (a part of lowest values: d * s may be infinite, e is 0)
        q.tx += t.ts == 0.0f && t.tx == 0.0f ? 0.0f : t.tx + d * t.ts;
        q.ts += t.ts;
    }
    q.s = wave_sum(q.s); q.sd = wave_sum(q.sd); q.tx = wave_sum(q.tx); q.ts = wave_sum(q.ts);
    const Done f = finish(p, i, q, xm, given, l == 0);
    if (p.top > 0) {
        keys += i * parts * p.top;
        const int64_t total = (int64_t)parts * p.top;
        uint64_t last = ~0ull;
        for (int k = 0; k < p.top; ++k) {
            uint64_t best = 0;
            if (last) for (int64_t c = l; c < total; c += 64) { const uint64_t v = keys[c]; if (v < last && v > best) best = v; }
            best = wave_max_u64(best);
            if (l == 0) {
                const bool some = best && !f.bad;
                if (p.top_move) p.top_move[i * p.top + k] = some ? (int32_t)~(uint32_t)best : -1;
                if (p.top_logp) p.top_logp[i * p.top + k] = some ? lp_key_value(best) - base_of(mx) - f.ls : (f.bad ? NAN : -INFINITY);
            }
            last = best;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// the gradient: one pass that reads the row and writes the gradient; a row (or part) per group of G lanes as above
// ---------------------------------------------------------------------------------------------------------------------------------------
struct GradRow { float mx, ls, h, gh, gt, gm, whole; int32_t mv; };
__device__ __forceinline__ float grad_at(const GradRow& c, float v, float t, bool hot) {
    const float lp = v - c.mx - c.ls, pr = __builtin_amdgcn_exp2f(lp * LOG2E);
    float g = c.gt * t - pr * (c.whole + c.gh * fmaxf(lp + c.h, -1.0e30f)) + (hot ? c.gm : 0.0f);     // (0 * -inf)
    return v == -INFINITY ? 0.0f : g;
}
template <typename T, int VEC, int G, int NV> __global__ __launch_bounds__(256) void k_logprob_grad(LpPar p, int32_t parts) {
    const int l = threadIdx.x & (G - 1);
    const int64_t w = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, i = parts == 1 ? w : w / parts;
    if (i >= p.n) return;
    const int32_t first = parts == 1 ? 0 : (int32_t)(w - i * parts) * PART;
    const int32_t end = parts == 1 || p.a - first <= PART ? p.a : first + PART;
    const T* x = (const T*)p.x + i * p.ld;
    T* dx = (T*)p.dx + i * p.ldd;
    const uint8_t* mask = p.mask ? p.mask + i * p.ld_mask : nullptr;
    const float* target = p.target && p.g_target ? p.target + i * p.ld_target : nullptr;
    Row<T, VEC, G, NV> r;
    r.load(x, mask, first, end, l);
    Span<float, VEC> t[NV];
    if (target)
#pragma unroll
        for (int k = 0; k < NV; ++k) if (first + VEC * (l + G * k) < end) t[k] = *(const Span<float, VEC>*)(target + r.at[k]);
    const float4 st = *(const float4*)(p.stats + i * 4);
    GradRow c{st.x, st.y, st.z, p.g_entropy ? p.g_entropy[i] : 0.0f, target ? p.g_target[i] : 0.0f, 0.0f, 0.0f, -1};
    if (p.moves && p.g_move) {
        const int64_t mv = p.moves[i];
        if (mv >= 0 && mv < p.a) { c.mv = (int32_t)mv; c.gm = p.g_move[i]; }
    }
    c.whole = c.gm + c.gt * st.w;
    if (p.g_top) for (int k = 0; k < p.top; ++k) if (p.top_move[i * p.top + k] >= 0) c.whole += p.g_top[i * p.top + k];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (first + VEC * (l + G * k) >= end) continue;
        const int32_t own = first + VEC * (l + G * k);
        Span<T, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.e[e] = from_f<T>(grad_at(c, r.x[k * VEC + e], target ? t[k].e[e] : 0.0f, r.at[k] + e == c.mv));
        if (r.at[k] == own) *(Span<T, VEC>*)(dx + own) = o;
        else
#pragma unroll
            for (int e = 0; e < VEC; ++e) if (r.at[k] + e >= own) dx[r.at[k] + e] = o.e[e];
    }
    if (p.g_top) {                                             // the alternatives' own entries, written once more with their cotangents
        __threadfence_block();
        for (int k = l; k < p.top; k += G) {
            const int32_t j = p.top_move[i * p.top + k];
            if (j < first || j >= end) continue;
            GradRow d = c;
            d.gm = p.g_top[i * p.top + k] + (j == c.mv ? c.gm : 0.0f);
            dx[j] = from_f<T>(grad_at(d, to_f(x[j]), target ? target[j] : 0.0f, true));
        }
    }
}

static int check(const char* who, const agz_logprob_args* q) {
    if (!q) return fail(AGZ_ERR_ARG, "%s: no arguments", who);
    if (q->n < 0 || q->a < 1 || q->a > (1ll << 30)) return fail(AGZ_ERR_ARG, "%s: %lld rows of %lld actions (rows >= 0, 1 <= actions <= 2^30)", who, (long long)q->n, (long long)q->a);
    if (!good_dtype(q->dtype)) return fail(AGZ_ERR_ARG, "%s: unknown dtype %d", who, q->dtype);
    if (q->top < 0 || q->top > AGZ_TOP_MAX) return fail(AGZ_ERR_ARG, "%s: %d alternatives (0 to %d)", who, q->top, AGZ_TOP_MAX);
    if (q->ld < 0 || q->ld_mask < 0 || q->ld_target < 0) return fail(AGZ_ERR_ARG, "%s: a negative stride", who);
    if (q->n == 0) return AGZ_OK;
    if (!q->logits || !q->stats) return fail(AGZ_ERR_ARG, "%s: logits and stats are required", who);
    if (!aligned(q->logits, esize(q->dtype)) || !aligned(q->target, 4) || !aligned(q->moves, 8) || !aligned(q->stats, 16) || !aligned(q->top_logp, 4) || !aligned(q->top_move, 4) ||
        !aligned(q->move_logp, 4) || !aligned(q->entropy, 4) || !aligned(q->target_logp, 4))
        return fail(AGZ_ERR_ARG, "%s: a pointer is not aligned to its type (stats: to 16 bytes)", who);
    return AGZ_OK;
}

static LpPar pack(const agz_logprob_args* q) {
    LpPar p{};
    p.n = q->n; p.a = (int32_t)q->a; p.top = q->top; p.x = q->logits; p.ld = q->ld; p.mask = q->mask; p.ld_mask = q->ld_mask;
    p.moves = q->moves; p.target = q->target; p.ld_target = q->ld_target; p.move_logp = q->move_logp; p.entropy = q->entropy;
    p.target_logp = q->target_logp; p.top_logp = q->top_logp; p.top_move = q->top_move; p.stats = q->stats;
    return p;
}

}  // namespace ops
}  // namespace agz

using namespace agz::ops;

// f(Row shape) for rows of `a` actions: lanes per row, spans per lane, elements per span; parts: rows longer than PART
template <typename T, typename F> static int by_length(int64_t a, F&& f) {
    constexpr int V = 16 / sizeof(T);
    using std::integral_constant;
    auto go = [&](auto vec, auto g, auto nv) { return f(vec, g, nv); };
#define AGZ_LP(VEC, G, NV) go(integral_constant<int, VEC>{}, integral_constant<int, G>{}, integral_constant<int, NV>{})
    if (a < V) return AGZ_LP(1, 8, 1);
    if (a <= 8 * V) return AGZ_LP(V, 8, 1);
    if (a <= 16 * V) return AGZ_LP(V, 8, 2);
    if (a <= 24 * V) return AGZ_LP(V, 8, 3);
    if (a <= 32 * V) return AGZ_LP(V, 8, 4);
    if (a <= 64 * V) return AGZ_LP(V, 64, 1);
    if (a <= 128 * V) return AGZ_LP(V, 64, 2);
    if (a <= 256 * V && 256 * V < PART) return AGZ_LP(V, 64, 4);
    return AGZ_LP(V, 64, PART / 64 / V);
#undef AGZ_LP
}
static int64_t part_count(int64_t a) { return cdiv(a, PART); }
static bool too_many(int64_t groups) { return cdiv(groups, 4) > 0x7fffffffll; }

extern "C" {

int64_t agz_logprob_workspace(int64_t n, int64_t a, int32_t top) {
    if (n < 0 || a < 1 || a > (1ll << 30) || top < 0 || top > AGZ_TOP_MAX) return -1;
    if (a <= PART) return 0;
    return n * part_count(a) * (int64_t)(sizeof(PartOut) + 8 * top);
}

int agz_logprob_forward(int device, void* stream, const agz_logprob_args* q) {
    if (int rc = check("agz_logprob_forward", q)) return rc;
    if (q->n > 0 && q->move_logp && !q->moves) return fail(AGZ_ERR_ARG, "agz_logprob_forward: move_logp without moves");
    if (q->n > 0 && q->target_logp && !q->target) return fail(AGZ_ERR_ARG, "agz_logprob_forward: target_logp without a target");
    const int64_t need = agz_logprob_workspace(q->n, q->a, q->top);
    if (need > 0 && (!q->workspace || q->workspace_bytes < need || !aligned(q->workspace, 16)))
        return fail(AGZ_ERR_ARG, "agz_logprob_forward: a workspace of %lld bytes, 16-byte aligned", (long long)need);
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    if (q->n == 0) return AGZ_OK;
    const LpPar p = pack(q);
    const int64_t parts = part_count(p.a);
    if (too_many(p.n * parts)) return fail(AGZ_ERR_ARG, "agz_logprob_forward: too many rows");
    return by_dtype(q->dtype, [&](auto t) {
        using T = decltype(t);
        if (parts == 1)
            return by_length<T>(p.a, [&](auto vec, auto g, auto nv) {
                return launch(k_logprob<T, vec(), g(), nv()>, dim3((uint32_t)cdiv(p.n, 256 / g())), dim3(256), 0, stream, p);
            });
        constexpr int V = 16 / sizeof(T);
        PartOut* part = (PartOut*)q->workspace;
        uint64_t* keys = (uint64_t*)(part + p.n * parts);
        if (int rc = launch(k_logprob_part<T, V, PART / 64 / V>, dim3((uint32_t)cdiv(p.n * parts, 4)), dim3(256), 0, stream, p, (int32_t)parts, part, keys)) return rc;
        return launch(k_logprob_join<T>, dim3((uint32_t)cdiv(p.n, 4)), dim3(256), 0, stream, p, (int32_t)parts, part, keys);
    });
}

int agz_logprob_backward(int device, void* stream, const agz_logprob_args* q, const float* g_move, const float* g_entropy, const float* g_target, const float* g_top, void* dx, int64_t ldd) {
    if (int rc = check("agz_logprob_backward", q)) return rc;
    if (q->n > 0) {
        if (!dx || ldd < q->a || !aligned(dx, esize(q->dtype))) return fail(AGZ_ERR_ARG, "agz_logprob_backward: dlogits with a row stride of at least %lld", (long long)q->a);
        if (g_move && !q->moves) return fail(AGZ_ERR_ARG, "agz_logprob_backward: g_move without moves");
        if (g_target && !q->target) return fail(AGZ_ERR_ARG, "agz_logprob_backward: g_target without a target");
        if (g_top && (q->top == 0 || !q->top_move)) return fail(AGZ_ERR_ARG, "agz_logprob_backward: g_top without alternatives");
    }
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    if (q->n == 0) return AGZ_OK;
    LpPar p = pack(q);
    p.g_move = g_move; p.g_entropy = g_entropy; p.g_target = g_target; p.g_top = g_top; p.dx = dx; p.ldd = ldd;
    const int64_t parts = part_count(p.a);
    if (too_many(p.n * parts)) return fail(AGZ_ERR_ARG, "agz_logprob_backward: too many rows");
    return by_dtype(q->dtype, [&](auto t) {
        using T = decltype(t);
        return by_length<T>(p.a, [&](auto vec, auto g, auto nv) {
            return launch(k_logprob_grad<T, vec(), g(), nv()>, dim3((uint32_t)cdiv(p.n * parts, 256 / g())), dim3(256), 0, stream, p, (int32_t)parts);
        });
    });
}

}  // extern "C"
