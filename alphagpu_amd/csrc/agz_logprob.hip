// agz_logprob.hip — log probabilities of given moves, entropy, best alternatives and the policy term of a loss, with their gradient
// (include/agz.h agz_logprob_forward / _backward; the softmax of mcts_gpu.jl:417 and the policy loss of train.jl:12-15).
#include "agz_ops.hpp"

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

// the simple form: one wave per row, the row read once for its maximum, once for its sums and once per alternative
template <typename T> __global__ __launch_bounds__(256) void k_logprob(LpPar p) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= p.n) return;
    const T* x = (const T*)p.x + i * p.ld;
    const uint8_t* mask = p.mask ? p.mask + i * p.ld_mask : nullptr;
    const float* t = p.target ? p.target + i * p.ld_target : nullptr;
    float mx = -INFINITY, any = 0.0f;
    for (int j = lane; j < p.a; j += 64) {
        const float v = to_f(x[j]);
        const bool in = (!mask || mask[j]) && v != -INFINITY;
        if (in) { mx = fmaxf(mx, v); any = 1.0f; }
    }
    mx = wave_max(mx);
    any = wave_max(any);
    float s = 0.0f, sd = 0.0f, tx = 0.0f, ts = 0.0f;
    for (int j = lane; j < p.a; j += 64) {
        const float v = to_f(x[j]);
        const bool in = (!mask || mask[j]) && v != -INFINITY;
        const float d = v - mx;
        if (in) { const float e = exp2f(d * LOG2E); s += e; sd += e > 0.0f || d != d ? e * d : 0.0f; }
        if (t) { const float w = t[j]; ts += w; if (w != 0.0f) tx += in ? w * d : w * -INFINITY; }
    }
    s = wave_sum(s); sd = wave_sum(sd); tx = wave_sum(tx); ts = wave_sum(ts);
    const bool none = any == 0.0f, bad = !none && !(s < INFINITY);
    const float ls = none ? 0.0f : (bad ? NAN : logf(s));
    const float h = none ? 0.0f : ls - sd / s;
    if (lane == 0) {
        float* st = p.stats + i * 4;
        st[0] = mx; st[1] = ls; st[2] = h; st[3] = ts;
        if (p.entropy) p.entropy[i] = h;
        if (p.target_logp) p.target_logp[i] = tx - ls * ts;
        if (p.move_logp) {
            const int64_t mv = p.moves[i];
            float lp = 0.0f;
            if (mv >= 0 && mv < p.a) {
                const float v = to_f(x[mv]);
                lp = (!mask || mask[mv]) && v != -INFINITY ? v - mx - ls : -INFINITY;
            }
            p.move_logp[i] = bad ? NAN : lp;
        }
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        uint64_t best = 0;
        if (!none && !bad)
            for (int j = lane; j < p.a; j += 64) {
                const float v = to_f(x[j]);
                if ((!mask || mask[j]) && v != -INFINITY) { const uint64_t key = lp_key(v, j); if (key < last && key > best) best = key; }
            }
        for (int o = 32; o; o >>= 1) { const uint64_t q = __shfl_xor(best, o); best = q > best ? q : best; }
        if (lane == 0) {
            if (p.top_move) p.top_move[i * p.top + k] = best ? (int32_t)~(uint32_t)best : -1;
            if (p.top_logp) p.top_logp[i * p.top + k] = best ? lp_key_value(best) - mx - ls : (bad ? NAN : -INFINITY);
        }
        last = best ? best : 0;
        if (!best) last = 1;                                   // nothing is below: the rest stays empty
    }
}

template <typename T> __global__ __launch_bounds__(256) void k_logprob_grad(LpPar p) {
    const int lane = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= p.n) return;
    const T* x = (const T*)p.x + i * p.ld;
    T* dx = (T*)p.dx + i * p.ldd;
    const uint8_t* mask = p.mask ? p.mask + i * p.ld_mask : nullptr;
    const float* t = p.target ? p.target + i * p.ld_target : nullptr;
    const float* st = p.stats + i * 4;
    const float mx = st[0], ls = st[1], h = st[2], ts = st[3];
    const float gh = p.g_entropy ? p.g_entropy[i] : 0.0f, gt = p.g_target && t ? p.g_target[i] : 0.0f;
    int64_t mv = p.moves && p.g_move ? p.moves[i] : -1;
    if (mv >= p.a) mv = -1;
    const float gm = mv >= 0 ? p.g_move[i] : 0.0f;
    float whole = gm + gt * ts;
    if (p.g_top) for (int k = 0; k < p.top; ++k) if (p.top_move[i * p.top + k] >= 0) whole += p.g_top[i * p.top + k];
    for (int j = lane; j < p.a; j += 64) {
        const float v = to_f(x[j]);
        const bool in = (!mask || mask[j]) && v != -INFINITY;
        const float lp = v - mx - ls, pr = exp2f(lp * LOG2E);
        float g = -pr * whole;
        if (gh != 0.0f && !(pr == 0.0f)) g -= gh * pr * (lp + h);
        if (t) g += gt * t[j];
        if (j == mv) g += gm;
        if (p.g_top) for (int k = 0; k < p.top; ++k) if (p.top_move[i * p.top + k] == j) g += p.g_top[i * p.top + k];
        if (ls != ls) g = NAN;
        dx[j] = from_f<T>(in ? g : 0.0f);
    }
}

static int check(const char* who, const agz_logprob_args* q) {
    if (!q) return fail(AGZ_ERR_ARG, "%s: no arguments", who);
    if (q->n < 0 || q->a < 1 || q->a >= (1ll << 31)) return fail(AGZ_ERR_ARG, "%s: %lld rows of %lld actions (rows >= 0, 1 <= actions < 2^31)", who, (long long)q->n, (long long)q->a);
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

extern "C" {

int64_t agz_logprob_workspace(int64_t n, int64_t a, int32_t top) {
    if (n < 0 || a < 1 || a >= (1ll << 31) || top < 0 || top > AGZ_TOP_MAX) return -1;
    return 0;
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
    if (cdiv(p.n, 4) > 0x7fffffffll) return fail(AGZ_ERR_ARG, "agz_logprob_forward: too many rows");
    return by_dtype(q->dtype, [&](auto T) { return launch(k_logprob<decltype(T)>, dim3((uint32_t)cdiv(p.n, 4)), dim3(256), 0, stream, p); });
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
    if (cdiv(p.n, 4) > 0x7fffffffll) return fail(AGZ_ERR_ARG, "agz_logprob_backward: too many rows");
    return by_dtype(q->dtype, [&](auto T) { return launch(k_logprob_grad<decltype(T)>, dim3((uint32_t)cdiv(p.n, 4)), dim3(256), 0, stream, p); });
}

}  // extern "C"
