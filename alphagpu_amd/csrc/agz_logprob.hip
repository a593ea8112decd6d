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
        o.sd = __builtin_fmaf(e, fmaxf(d, -3.0e38f), o.sd);     // (0 * -inf)
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
// the places of a list of different keys in LDS: emit(place, key) for the first `top`, emit(place, 0) for the places that nobody has
template <typename E> __device__ __forceinline__ void wave_list_ranks(const uint64_t* list, int count, int top, E&& emit) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int lane = threadIdx.x & 63;
    for (int q = lane; q < count; q += 64) {
        const uint64_t mine = list[q];
        int before = 0;
#pragma unroll 8
        for (int o = 0; o < count; ++o) before += list[o] > mine ? 1 : 0;
        if (before < top) emit(before, mine);
    }
    for (int k = count + lane; k < top; k += 64) emit(k, (uint64_t)0);
}

// The `top` best entries of what a wave holds (NE per lane, -inf: not allowed), largest first: emit(rank, key) from the lane that finds it, emit(rank, 0) behind
// the last.  Every lane's best: the top-th largest of these 64 is a lower bound of the top-th largest entry.  The entries from that bound on (at most top lanes'
// shares) go into a list in LDS, and an entry's place is the number of entries before it: all comparisons are independent, where taking the best again and
// again is a chain of `top` reductions (20 of a row of 131072: part launch 41.5 us so, 9-10 us this way).
constexpr int LIST = AGZ_TOP_MAX * 32;
template <int NE, typename J, typename E> __device__ __forceinline__ void wave_top(const float (&x)[NE], J&& index, int top, uint64_t* list, E&& emit) {
    static_assert(NE <= 32, "the list holds the shares of AGZ_TOP_MAX lanes");
    const int lane = threadIdx.x & 63;
    float v = -INFINITY;
    uint32_t j = 0;
#pragma unroll
    for (int k = 0; k < NE; ++k) if (x[k] > v) { v = x[k]; j = index(k); }
    const uint64_t mine = v > -INFINITY ? lp_key(v, j) : 0;
    const uint32_t hi = (uint32_t)(mine >> 32), lo = (uint32_t)mine;
    int before = 0;
#pragma unroll 8
    for (int o = 0; o < 64; ++o) {
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, o) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, o);
        before += other > mine ? 1 : 0;
    }
    const uint64_t at = __ballot(mine != 0 && before == top - 1);
    uint64_t bound = 1;                                        // fewer than `top` lanes with an entry: every entry
    if (at) {
        const int o = __builtin_ctzll(at);
        bound = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, o) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, o);
    }
    int count = 0;
#pragma unroll
    for (int k = 0; k < NE; ++k) {
        const uint64_t key = x[k] > -INFINITY ? lp_key(x[k], index(k)) : 0;
        const uint64_t in = __ballot(key >= bound);
        if (in) {
            if (key >= bound) list[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0))] = key;
            count += __popcll(in);
        }
    }
    wave_list_ranks(list, count, top, emit);
}

// The next best entry of what G lanes hold, taken out of it: its value (-inf: none is left) and its index.  Equal entries by index: every lane offers the
// first of its largest, the lowest index among the lanes whose offer is the largest wins.  (The largest first and its place behind it: 65536 rows of 81 with five
// alternatives 14.6 -> 12.2 us against keeping value, index and place together.)
template <int N> struct Offer { float v; uint32_t j; int k; };
template <typename T, int VEC, int G, int NV> __device__ __forceinline__ Offer<0> offer(const Row<T, VEC, G, NV>& r, int l, int32_t last) {
    Offer<0> o{-INFINITY, 0xFFFFFFFFu, -1};
#pragma unroll
    for (int k = 0; k < NV * VEC; ++k) o.v = fmaxf(o.v, r.x[k]);
#pragma unroll
    for (int k = NV * VEC - 1; k >= 0; --k) o.k = r.x[k] == o.v ? k : o.k;
    const int32_t own = VEC * l + G * (o.k & ~(VEC - 1));                // (r.at[o.k / VEC], worked out: an index that is no constant would put it into memory)
    if (o.v > -INFINITY) o.j = (uint32_t)((own < last ? own : last) + (o.k & (VEC - 1)));
    return o;
}
template <typename T, int VEC, int G, int NV> __device__ __forceinline__ float take_best(Row<T, VEC, G, NV>& r, Offer<0>& o, uint32_t& j, int l, int32_t last, bool more) {
    const float best = lanes_max<G>(o.v);
    j = lanes_min_u<G>(o.v == best ? o.j : 0xFFFFFFFFu);
    if (more && best > -INFINITY && o.j == j) {
#pragma unroll
        for (int k = 0; k < NV * VEC; ++k) if (k == o.k) r.x[k] = -INFINITY;
        o = offer(r, l, last);
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
        if (p.stats) *(float4*)(p.stats + i * 4) = make_float4(base, ls, h, q.ts);
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

// A row per group of G lanes: rows of up to G NV VEC actions.  One pass over memory: logp_j = d_j - log s and entropy = log s - (sum d e^d) / s with
// d = x - largest, so the row is not read again once the largest is known.
// PLAIN: without mask, target and alternatives (fewer registers).  The other builds of fewer than 64 lanes a row and 24 or 32 elements a lane (rows of 129 to
// 1024 actions) hold most of the row in private memory, 56 and 100 bytes a lane, in all calls: take_best takes an element out at a place that only the run knows.
// That goes through the caches: 32768 rows with mask and target in 32 bits (bf16) take, of 169 actions 15.2 (14.1) us where the bytes take 10.5 (8.2) at the rate of a
// copy, of 225 16.9 (16.1) for 14.0 (10.9), of 361 22.2 (20.1) for 22.3 (17.4), of 500 30.8 (27.5) for 30.9 (24.0), of 1000 68.6 (51.1) for 61.6 (47.9).
// Bound by memory where rows are many, by launch and reductions where they are few.  32768 rows of 81 in 32 bits with mask and five alternatives: 8.0-8.7 us
// (13 MB read; 4.3 us without the alternatives); 65536 with mask and target: 10.4 us (48 MB read, 4.6 TB/s; a copy of large tensors reaches 4.8 TB/s on the same card).
template <typename T, int VEC, int G, int NV, bool PLAIN> __global__ __launch_bounds__(256) void k_logprob(LpPar p) {
    const int l = threadIdx.x & (G - 1);
    const int64_t i = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (i >= p.n) return;
    const T* x = (const T*)p.x + i * p.ld;
    const uint8_t* mask = !PLAIN && p.mask ? p.mask + i * p.ld_mask : nullptr;
    bool given;
    const float xm = given_logit(p, x, mask, i, given);
    Row<T, VEC, G, NV> r;
    r.load(x, mask, 0, p.a, l);
    const Sums q = row_sums(r, !PLAIN && p.target ? p.target + i * p.ld_target : nullptr, 0, p.a, l);
    const Done f = finish(p, i, q, xm, given, l == 0);
    if (!PLAIN && p.top > 0) {
        const float off = base_of(q.mx);
        auto put = [&](int k, bool some, float v, uint32_t j) {
            some = some && !f.bad;
            if (p.top_move) p.top_move[i * p.top + k] = some ? (int32_t)j : -1;
            if (p.top_logp) p.top_logp[i * p.top + k] = some ? v - off - f.ls : (f.bad ? NAN : -INFINITY);
        };
        if constexpr (G == 64) {
            __shared__ uint64_t list[4][LIST];
            wave_top(r.x, [&](int k) { return (uint32_t)(r.at[k / VEC] + k % VEC); }, p.top, list[threadIdx.x >> 6], [&](int k, uint64_t key) { put(k, key != 0, lp_key_value(key), ~(uint32_t)key); });
        } else {
            auto o = offer(r, l, p.a - VEC);
            for (int k = 0; k < p.top; ++k) {
                uint32_t j;
                const float v = take_best(r, o, j, l, p.a - VEC, k + 1 < p.top);
                if (l == 0) put(k, v > -INFINITY, v, j);
            }
        }
    }
}

// Longer rows: one wave per part leaves the part's sums and best alternatives (as keys) in the workspace, a second launch joins the parts of a row.  A part
// is one block of PART elements where alternatives are wanted or rows are few, up to MOST blocks where there are waves enough without: a lane then carries its
// own maximum and sums from block to block (the sums rescaled where the maximum grows), the next block's loads under way behind them,
// and the lanes are joined once.  (4096 rows of 50001 bf16: a block a wave 221 us.)
// Without mask and target the spans lie on 16-byte borders of memory wherever the row begins: the first one begins up to seven elements before the row (and is read
// from the row's start, the elements that are not its own left out), since unaligned spans cost a tenth (50001 against 50000 bf16).
// Bound by memory, and by waves that do not come out even: 4096 rows of 50001 bf16 121 us (3.4 TB/s), 12288 waves where 5120 fit on the card at a time; one row of
// 131072 with 20 alternatives 9-10 us, 64 waves: launch and wave_top.
constexpr int PART = 2048, MOST = 16, WAVES_ENOUGH = 8192, MOST_PAD = 7;
template <typename T, int VEC> __device__ __forceinline__ int pad_of(const T* row) { return (int)((uintptr_t)row / sizeof(T) & (VEC - 1)); }
__device__ __forceinline__ int64_t span_at(int64_t own, int64_t last) { return own < 0 ? 0 : (own < last ? own : last); }     // last: a - VEC
struct PartOut { Sums q; float pad[3]; };

// blocks of a part and parts of a row
struct Parts { int32_t blocks, parts; };
static Parts parts_of(int64_t n, int64_t a, int top, bool plain) {
    const int64_t all = cdiv(plain ? a + MOST_PAD : a, PART);
    int64_t blocks = top > 0 ? 1 : n * all / WAVES_ENOUGH;
    blocks = blocks < 1 ? 1 : (blocks > MOST ? MOST : blocks);
    const int64_t parts = cdiv(all, blocks);
    return {(int32_t)cdiv(all, parts), (int32_t)parts};
}

// sums relative to `mx` brought to `to` >= mx
__device__ __forceinline__ void rebase(Sums& q, float to) {
    const float d = base_of(q.mx) - base_of(to), e = q.mx == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(d * LOG2E);
    q.sd = e > 0.0f ? e * (q.sd + d * q.s) : 0.0f;             // (lowest values: d * s may be infinite, e is 0)
    q.s *= e;
    q.tx += q.ts == 0.0f ? 0.0f : d * q.ts;
    q.mx = to;
}

template <typename T, int VEC, int NV, bool PLAIN> __global__ __launch_bounds__(256) void k_logprob_part(LpPar p, Parts s, PartOut* part, uint64_t* keys) {
    const int l = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t i = w / s.parts;
    if (i >= p.n) return;
    const T* x = (const T*)p.x + i * p.ld;
    const int64_t begin = (w - i * s.parts) * s.blocks * PART - (PLAIN ? pad_of<T, VEC>(x) : 0), stop = begin + (int64_t)s.blocks * PART < p.a ? begin + (int64_t)s.blocks * PART : p.a;
    if constexpr (PLAIN) {                                     // no mask, no target, no alternatives
        Span<T, VEC> v[NV], u[NV];
        auto fetch = [&](Span<T, VEC> (&to)[NV], int64_t first) {
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                to[k] = *(const Span<T, VEC>*)(x + span_at(first + VEC * (l + 64 * k), p.a - VEC));
            }
        };
        Sums q{-INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
        fetch(v, begin);
        for (int64_t first = begin; first < stop; first += PART) {
            if (first + PART < stop) fetch(u, first + PART);
            float f[NV * VEC], mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < NV * VEC; ++k) f[k] = to_f(v[k / VEC].e[k % VEC]);
            if (first < 0 || first + PART > p.a) {             // the row's first and last block: entries that are not the span's own count as not there
#pragma unroll
                for (int k = 0; k < NV; ++k) {
                    const int64_t own = first + VEC * (l + 64 * k), at = span_at(own, p.a - VEC);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) f[k * VEC + e] = at + e >= own && at + e < own + VEC ? f[k * VEC + e] : -INFINITY;
                }
            }
#pragma unroll
            for (int k = 0; k < NV * VEC; ++k) mx = fmaxf(mx, f[k]);
            if (mx > q.mx) rebase(q, mx);
            const float base = base_of(q.mx);
#pragma unroll
            for (int k = 0; k < NV * VEC; ++k) {
                const float d = f[k] - base, e = __builtin_amdgcn_exp2f(d * LOG2E);
                q.s += e;
                q.sd = __builtin_fmaf(e, fmaxf(d, -3.0e38f), q.sd);
            }
#pragma unroll
            for (int k = 0; k < NV; ++k) v[k] = u[k];
        }
        const float mx = wave_max(q.mx);
        rebase(q, mx);
        q.s = wave_sum(q.s);
        q.sd = wave_sum(q.sd);
        if (l == 0) part[w].q = q;
    } else {
        Sums all{-INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
        for (int64_t first = begin; first < stop; first += PART) {
            const int32_t end = (int32_t)(stop - first > PART ? first + PART : stop);
            Row<T, VEC, 64, NV> r;
            r.load(x, p.mask ? p.mask + i * p.ld_mask : nullptr, (int32_t)first, end, l);
            Sums q = row_sums(r, p.target ? p.target + i * p.ld_target : nullptr, (int32_t)first, end, l);
            if (s.blocks > 1) {
                const float mx = fmaxf(all.mx, q.mx);
                rebase(all, mx);
                rebase(q, mx);
                all.s += q.s; all.sd += q.sd; all.tx += q.tx; all.ts += q.ts;
            } else all = q;
            if (p.top > 0) {
                __shared__ uint64_t list[4][LIST];
                wave_top(r.x, [&](int k) { return (uint32_t)(r.at[k / VEC] + k % VEC); }, p.top, list[threadIdx.x >> 6], [&](int k, uint64_t key) { keys[w * p.top + k] = key; });
            }
        }
        if (l == 0) part[w].q = all;
    }
}

// The parts of a row joined by a wave: sums brought to the largest entry of all, alternatives by the bound of wave_top over the parts' keys.  Bound by the launch and
// two dependent reads: 5.7 us for 4096 rows of three parts, 6.6 us for one row of 64 parts with 20 alternatives each.
constexpr int JOIN_LIST = 1024;
template <typename T> __global__ __launch_bounds__(256) void k_logprob_join(LpPar p, int32_t parts, const PartOut* part, const uint64_t* keys) {
    const int l = threadIdx.x & 63;
    const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= p.n) return;
    const T* x = (const T*)p.x + i * p.ld;
    bool given;
    const float xm = given_logit(p, x, p.mask ? p.mask + i * p.ld_mask : nullptr, i, given);
    part += i * parts;
    Sums q{-INFINITY, 0.0f, 0.0f, 0.0f, 0.0f};
    for (int32_t k = l; k < parts; k += 64) {
        Sums t = part[k].q;
        const float mx = fmaxf(q.mx, t.mx);
        rebase(q, mx);
        rebase(t, mx);
        q.s += t.s; q.sd += t.sd; q.tx += t.tx; q.ts += t.ts;
    }
    const float mx = wave_max(q.mx);
    rebase(q, mx);
    q.s = wave_sum(q.s); q.sd = wave_sum(q.sd); q.tx = wave_sum(q.tx); q.ts = wave_sum(q.ts);
    const Done f = finish(p, i, q, xm, given, l == 0);
    if (p.top == 0) return;
    __shared__ uint64_t lists[4][JOIN_LIST];
    uint64_t* list = lists[threadIdx.x >> 6];
    keys += i * parts * p.top;
    const int64_t total = (int64_t)parts * p.top;
    auto emit = [&](int k, uint64_t key) {
        const bool some = key != 0 && !f.bad;
        if (p.top_move) p.top_move[i * p.top + k] = some ? (int32_t)~(uint32_t)key : -1;
        if (p.top_logp) p.top_logp[i * p.top + k] = some ? lp_key_value(key) - base_of(mx) - f.ls : (f.bad ? NAN : -INFINITY);
    };
    // the bound as in wave_top, over the lanes' shares of the parts' keys; up to SHARE keys a lane (SHARE * 64 in all) stay in its registers
    constexpr int SHARE = 32;
    uint64_t held[SHARE], mine = 0;
#pragma unroll
    for (int k = 0; k < SHARE; ++k) held[k] = l + 64 * k < total ? keys[l + 64 * k] : 0;
#pragma unroll
    for (int k = 0; k < SHARE; ++k) mine = held[k] > mine ? held[k] : mine;
    for (int64_t c = l + 64 * SHARE; c < total; c += 64) { const uint64_t v = keys[c]; mine = v > mine ? v : mine; }
    const uint32_t hi = (uint32_t)(mine >> 32), lo = (uint32_t)mine;
    int before = 0;
#pragma unroll 8
    for (int o = 0; o < 64; ++o) {
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, o) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, o);
        before += other > mine ? 1 : 0;
    }
    const uint64_t at = __ballot(mine != 0 && before == p.top - 1);
    uint64_t bound = 1;
    if (at) {
        const int o = __builtin_ctzll(at);
        bound = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, o) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)lo, o);
    }
    int count = 0;
    auto note = [&](uint64_t key) {
        const uint64_t in = __ballot(key >= bound);
        if (in) {
            const int to = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
            if (key >= bound && to < JOIN_LIST) list[to] = key;
            count += __popcll(in);
        }
    };
#pragma unroll
    for (int k = 0; k < SHARE; ++k) if (64 * k < total) note(held[k]);
    for (int64_t c0 = 64 * SHARE; c0 < total; c0 += 64) note(c0 + l < total ? keys[c0 + l] : 0);
    if (count <= JOIN_LIST) {
        wave_list_ranks(list, count, p.top, emit);
        return;
    }
    uint64_t last = ~0ull;                                     // (thousands of parts whose best ones fall to few lanes: one after the other)
    for (int k = 0; k < p.top; ++k) {
        uint64_t best = 0;
        for (int64_t c = l; c < total; c += 64) { const uint64_t v = keys[c]; if (v < last && v > best) best = v; }
        const uint32_t bh = lanes_reduce<64>((uint32_t)(best >> 32), [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        const uint32_t bl = lanes_reduce<64>((uint32_t)(best >> 32) == bh ? (uint32_t)best : 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
        last = (uint64_t)bh << 32 | bl;
        if (l == 0) emit(k, last);
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// the gradient: one pass that reads the row and writes the gradient; a row (or part) per group of G lanes as above.  With the forward pass's largest entry, log sum and
// entropy every entry stands for itself: g_j = c_j - p_j (sum c + g_entropy (logp_j + entropy)).  Bound by memory: 65536 rows of 81 in 32 bits with mask and target
// 13.1 us (69 MB, partly from the caches: 5.3 TB/s)
// ---------------------------------------------------------------------------------------------------------------------------------------
struct GradRow { float mx, ls, gh, gt, gm, whole; int32_t mv; };         // whole: the sum of the cotangents, and gh times the entropy
__device__ __forceinline__ float grad_at(const GradRow& c, float v, float t, bool hot) {
    const float lp = v - c.mx - c.ls, pr = __builtin_amdgcn_exp2f(lp * LOG2E);
    float g = c.gt * t - pr * __builtin_fmaf(c.gh, fmaxf(lp, -1.0e30f), c.whole);      // (0 * -inf)
    g = hot ? g + c.gm : g;
    return v == -INFINITY ? 0.0f : g;
}
template <typename T, int VEC, int G, int NV, bool PLAIN> __global__ __launch_bounds__(256) void k_logprob_grad(LpPar p, int32_t parts) {   // parts: blocks of PART elements of a row
    const int l = threadIdx.x & (G - 1);
    const int64_t w = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G, i = parts == 1 ? w : w / parts;
    if (i >= p.n) return;
    const int32_t first = parts == 1 ? 0 : (int32_t)(w - i * parts) * PART;
    const int32_t end = parts == 1 || p.a - first <= PART ? p.a : first + PART;
    const T* x = (const T*)p.x + i * p.ld;
    T* dx = (T*)p.dx + i * p.ldd;
    const uint8_t* mask = !PLAIN && p.mask ? p.mask + i * p.ld_mask : nullptr;
    const float* target = !PLAIN && p.g_target ? p.target + i * p.ld_target : nullptr;
    Row<T, VEC, G, NV> r;
    r.load(x, mask, first, end, l);
    Span<float, VEC> t[NV];
    if (target)
#pragma unroll
        for (int k = 0; k < NV; ++k) if (first + VEC * (l + G * k) < end) t[k] = *(const Span<float, VEC>*)(target + r.at[k]);
    const float4 st = *(const float4*)(p.stats + i * 4);
    GradRow c{st.x, st.y, p.g_entropy ? p.g_entropy[i] : 0.0f, target ? p.g_target[i] : 0.0f, 0.0f, 0.0f, -1};
    if (p.moves && p.g_move) {
        const int64_t mv = p.moves[i];
        if (mv >= 0 && mv < p.a) { c.mv = (int32_t)mv; c.gm = p.g_move[i]; }
    }
    c.whole = c.gm + c.gt * st.w;
    if (!PLAIN && p.g_top) for (int k = 0; k < p.top; ++k) if (p.top_move[i * p.top + k] >= 0) c.whole += p.g_top[i * p.top + k];
    c.whole += c.gh * st.z;
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
    if (!PLAIN && p.g_top) {                                   // the alternatives' own entries, written once more with their cotangents
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

// ... of long rows without mask, target and cotangents of alternatives: a wave per block, spans on 16-byte borders as in the forward pass (the gradient's rows lie
// like the logits' where their strides agree): 4096 rows of 50001 bf16 144-153 us (819 MB, 5.4-5.7 TB/s; spans that begin where the row begins: 194 us)
template <typename T, int VEC, int NV> __global__ __launch_bounds__(256) void k_logprob_grad_part(LpPar p, int32_t parts) {
    const int l = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), i = w / parts;
    if (i >= p.n) return;
    const T* x = (const T*)p.x + i * p.ld;
    T* dx = (T*)p.dx + i * p.ldd;
    const int64_t first = (w - i * parts) * PART - pad_of<T, VEC>(x);
    Span<T, VEC> v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) v[k] = *(const Span<T, VEC>*)(x + span_at(first + VEC * (l + 64 * k), p.a - VEC));
    const float4 st = *(const float4*)(p.stats + i * 4);
    GradRow c{st.x, st.y, p.g_entropy ? p.g_entropy[i] : 0.0f, 0.0f, 0.0f, 0.0f, -1};
    if (p.moves && p.g_move) {
        const int64_t mv = p.moves[i];
        if (mv >= 0 && mv < p.a) { c.mv = (int32_t)mv; c.gm = p.g_move[i]; }
    }
    c.whole = c.gm + c.gh * st.z;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int64_t own = first + VEC * (l + 64 * k), at = span_at(own, p.a - VEC);
        Span<T, VEC> o;
#pragma unroll
        for (int e = 0; e < VEC; ++e) o.e[e] = from_f<T>(grad_at(c, to_f(v[k].e[e]), 0.0f, at + e == c.mv));
        if (at == own) *(Span<T, VEC>*)(dx + own) = o;
        else
#pragma unroll
            for (int e = 0; e < VEC; ++e) if (at + e >= own && at + e < own + VEC) dx[at + e] = o.e[e];
    }
}

// a launch has fewer than 2^32 lanes: 2^24 - 1 workgroups of 256, and at most 32 rows a workgroup
constexpr int64_t MOST_GROUPS = (1ll << 24) - 1, MOST_ROWS = MOST_GROUPS * 32;

static int check(const char* who, const agz_logprob_args* q) {
    if (!q) return fail(AGZ_ERR_ARG, "%s: no arguments", who);
    if (q->n < 0 || q->a < 1 || q->a > (1ll << 30)) return fail(AGZ_ERR_ARG, "%s: %lld rows of %lld actions (rows >= 0, 1 <= actions <= 2^30)", who, (long long)q->n, (long long)q->a);
    if (q->n > MOST_ROWS) return fail(AGZ_ERR_ARG, "%s: too many rows", who);
    if (!good_dtype(q->dtype)) return fail(AGZ_ERR_ARG, "%s: unknown dtype %d", who, q->dtype);
    if (q->top < 0 || q->top > AGZ_TOP_MAX) return fail(AGZ_ERR_ARG, "%s: %d alternatives (0 to %d)", who, q->top, AGZ_TOP_MAX);
    if (q->ld < 0 || q->ld_mask < 0 || q->ld_target < 0) return fail(AGZ_ERR_ARG, "%s: a negative stride", who);
    if (q->n == 0) return AGZ_OK;
    if (!q->logits) return fail(AGZ_ERR_ARG, "%s: logits are required", who);
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

// f(elements per span, lanes per row, spans per lane) for rows of `a` actions: 32 elements a lane at most, and as few lanes as hold the row, since the
// reductions over them are what short rows spend their time on (200000 rows of 500 bf16: 106 us with 64 lanes a row, 37 us with 16).  A row above 128
// actions of which more than four alternatives are wanted gets a whole wave: wave_top finds them in one go (40000 rows of 500, 20 alternatives: 64 us,
// 180 us with 16 lanes that take one after the other; one alternative costs the few lanes less).  TOPS: alternatives may be wanted.
template <typename T, bool TOPS, typename F> static int by_length(int64_t a, int top, F&& f) {
    constexpr int V = 16 / sizeof(T), F4 = 32 / V, F3 = F4 * 3 / 4, F2 = F4 / 2, F1 = F4 / 4;
    using std::integral_constant;
#define AGZ_LP(VEC, G, NV) f(integral_constant<int, VEC>{}, integral_constant<int, G>{}, integral_constant<int, NV>{})
    if (a < V) return AGZ_LP(1, 8, 1);
    if (a <= 8 * V * F1) return AGZ_LP(V, 8, F1);
    if constexpr (sizeof(T) == 4) if (a > 8 * V * F1 && a <= 8 * V * 3) return AGZ_LP(V, 8, 3);      // (65 to 96 actions in 32 bits: three spans a lane, not four)
    if (a <= 8 * V * F2) return AGZ_LP(V, 8, F2);
    if constexpr (TOPS) if (top > 4 && a > 128) {
        if (a <= 64 * V * F1) return AGZ_LP(V, 64, F1);
        if (a <= 64 * V * F2) return AGZ_LP(V, 64, F2);
        return a <= 64 * V * F3 ? AGZ_LP(V, 64, F3) : AGZ_LP(V, 64, F4);
    }
    if (a <= 8 * V * F4) return AGZ_LP(V, 8, F4);
    if (a <= 16 * V * F3) return AGZ_LP(V, 16, F3);
    if (a <= 16 * V * F4) return AGZ_LP(V, 16, F4);
    if (a <= 32 * V * F3) return AGZ_LP(V, 32, F3);
    if (a <= 32 * V * F4) return AGZ_LP(V, 32, F4);
    if (a <= 64 * V * F3) return AGZ_LP(V, 64, F3);
    return AGZ_LP(V, 64, F4);
#undef AGZ_LP
}
// workgroups of a call on rows that are `parts` waves each, or (1) as by_length says
static int64_t groups_of(int dtype, int64_t n, int64_t a, int top, int64_t parts) {
    int64_t groups = cdiv(n * parts, 4);
    if (parts == 1) by_dtype(dtype, [&](auto t) { return by_length<decltype(t), true>(a, top, [&](auto, auto g, auto) { groups = cdiv(n, 256 / g()); return 0; }); });
    return groups;
}

extern "C" {

int64_t agz_logprob_workspace(int64_t n, int64_t a, int32_t top) {
    if (n < 0 || n > MOST_ROWS || a < 1 || a > (1ll << 30) || top < 0 || top > AGZ_TOP_MAX) return -1;
    if (a <= PART) return 0;
    const int64_t p = parts_of(n, a, top, true).parts, q = parts_of(n, a, top, false).parts;     // (one block more may be longer parts, and fewer)
    return n * (p > q ? p : q) * (int64_t)(sizeof(PartOut) + 8 * top);
}

int agz_logprob_forward(int device, void* stream, const agz_logprob_args* q) {
    if (int rc = check("agz_logprob_forward", q)) return rc;
    if (q->n > 0 && q->move_logp && !q->moves) return fail(AGZ_ERR_ARG, "agz_logprob_forward: move_logp without moves");
    if (q->n > 0 && q->target_logp && !q->target) return fail(AGZ_ERR_ARG, "agz_logprob_forward: target_logp without a target");
    const int64_t need = agz_logprob_workspace(q->n, q->a, q->top);
    if (need > 0 && (!q->workspace || q->workspace_bytes < need || !aligned(q->workspace, 16)))
        return fail(AGZ_ERR_ARG, "agz_logprob_forward: a workspace of %lld bytes, 16-byte aligned", (long long)need);
    const LpPar p = pack(q);
    const bool plain = !p.mask && !p.target && p.top == 0;
    const Parts w = parts_of(p.n, p.a, p.top, plain);
    if (groups_of(q->dtype, p.n, p.a, p.top, p.a <= PART ? 1 : w.parts) > MOST_GROUPS) return fail(AGZ_ERR_ARG, "agz_logprob_forward: too many rows");
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    if (q->n == 0) return AGZ_OK;
    return by_dtype(q->dtype, [&](auto t) {
        using T = decltype(t);
        auto whole = [&](auto is_plain) {
            return by_length<T, !is_plain()>(p.a, p.top, [&](auto vec, auto g, auto nv) {
                return launch(k_logprob<T, vec(), g(), nv(), is_plain()>, dim3((uint32_t)cdiv(p.n, 256 / g())), dim3(256), 0, stream, p);
            });
        };
        if (p.a <= PART) return plain ? whole(std::true_type{}) : whole(std::false_type{});
        constexpr int V = 16 / sizeof(T);
        PartOut* part = (PartOut*)q->workspace;
        uint64_t* keys = (uint64_t*)(part + p.n * w.parts);
        if (int rc = launch(plain ? k_logprob_part<T, V, PART / 64 / V, true> : k_logprob_part<T, V, PART / 64 / V, false>, dim3((uint32_t)cdiv(p.n * w.parts, 4)), dim3(256), 0, stream, p, w, part, keys)) return rc;
        return launch(k_logprob_join<T>, dim3((uint32_t)cdiv(p.n, 4)), dim3(256), 0, stream, p, w.parts, part, keys);
    });
}

int agz_logprob_backward(int device, void* stream, const agz_logprob_args* q, const float* g_move, const float* g_entropy, const float* g_target, const float* g_top, void* dx, int64_t ldd) {
    if (int rc = check("agz_logprob_backward", q)) return rc;
    if (q->n > 0) {
        if (!q->stats) return fail(AGZ_ERR_ARG, "agz_logprob_backward: the forward call's stats are required");
        if (!dx || ldd < q->a || !aligned(dx, esize(q->dtype))) return fail(AGZ_ERR_ARG, "agz_logprob_backward: dlogits with a row stride of at least %lld", (long long)q->a);
        if (g_move && !q->moves) return fail(AGZ_ERR_ARG, "agz_logprob_backward: g_move without moves");
        if (g_target && !q->target) return fail(AGZ_ERR_ARG, "agz_logprob_backward: g_target without a target");
        if (g_top && (q->top == 0 || !q->top_move)) return fail(AGZ_ERR_ARG, "agz_logprob_backward: g_top without alternatives");
    }
    LpPar p = pack(q);
    p.g_move = g_move; p.g_entropy = g_entropy; p.g_target = g_target; p.g_top = g_top; p.dx = dx; p.ldd = ldd;
    const bool plain = !p.mask && !g_target && !g_top;
    const int64_t parts = p.a <= PART ? 1 : cdiv(plain ? p.a + MOST_PAD : p.a, PART);
    if (groups_of(q->dtype, p.n, p.a, 0, parts) > MOST_GROUPS) return fail(AGZ_ERR_ARG, "agz_logprob_backward: too many rows");
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    if (q->n == 0) return AGZ_OK;
    return by_dtype(q->dtype, [&](auto t) {
        using T = decltype(t);
        constexpr int V = 16 / sizeof(T);
        if (plain && parts > 1) return launch(k_logprob_grad_part<T, V, PART / 64 / V>, dim3((uint32_t)cdiv(p.n * parts, 4)), dim3(256), 0, stream, p, (int32_t)parts);
        return by_length<T, false>(p.a, 0, [&](auto vec, auto g, auto nv) {
            return launch(plain ? k_logprob_grad<T, vec(), g(), nv(), true> : k_logprob_grad<T, vec(), g(), nv(), false>, dim3((uint32_t)cdiv(p.n * parts, 256 / g())), dim3(256), 0, stream, p, (int32_t)parts);
        });
    });
}

}  // extern "C"
