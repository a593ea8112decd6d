// agz_fp8.hip — matrices in 8 bits (e4m3 with one power-of-two scale per block of 128) and their product on the matrix units
// (include/agz.h agz_fp8_quantize / agz_fp8_matmul): the layers of the network, forward and backward (DenseNet.jl:161-198, 294-304).
#include "agz_ops.hpp"
#include <type_traits>

namespace agz {
namespace ops {

constexpr int FB = 128;                        // a block: 128 along the contracted axis

struct QuantPar {
    const void *x, *gate;
    int64_t rows, cols, ld;
    uint8_t *q, *s, *qt, *st;
    int64_t pitch, spitch, tpitch, tspitch;     // of q, s and of qt, st
    float* part;                                // column sums of a tile of rows: [row tiles][cols]
};

// eight values times inv (a power of two: exact), rounded to e4m3 to the nearest; the conversion turns NaN and infinities into NaN
__device__ __forceinline__ uint2 enc8(const float* v, float inv) {
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}
// values of the 4 groups of 16 lanes combined (lane l with l ^ 16 and l ^ 32)
template <typename F> __device__ __forceinline__ float groups_reduce(float x, F&& f) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// One workgroup per tile of 128 x 128, all of it in registers: wave w, lane l hold rows 32 w + 8 (l / 16) + 0..7 of columns 8 (l % 16) + 0..7, read and
// written eight at a time both ways (8 x 8 values: the transpose is a matter of which eight are packed).  A row's largest is a reduction over
// 16 lanes, a column's one over 4 lanes and, through LDS, the 4 waves.  fmaxf passes NaN over; a largest of infinity means that the block has one, and its largest
// finite entry is looked for again.
// Bound by memory: 32768 x 512 bf16 both ways 17.0 us (67 MB, 4.0 TB/s), with the gate and column sums 22.0 us (101 MB, 4.6 TB/s); 8192 x 8192 bf16 both ways with column
// sums 62-65 us (270 MB, 4.1-4.4 TB/s); 8192 x 4096 in 32 bits, blocks of 128 x 128, 42-47 us (201 MB, 4.3-4.8 TB/s).
template <typename T, int BR, bool ROW, bool COL, bool GATE, bool NARROW>
__global__ __launch_bounds__(256) void k_quantize(QuantPar p) {
    __shared__ __attribute__((aligned(16))) float red[4][FB];
    __shared__ uint2 turn[COL ? FB : 1][16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, l16 = lane & 15;
    const int64_t r0 = (int64_t)blockIdx.y * FB + w * 32 + (lane >> 4) * 8, c0 = (int64_t)blockIdx.x * FB, c = c0 + l16 * 8;
    // Straight-line loads, all under way at once: rows behind the last read the last one, and where the matrix ends inside a lane's eight columns the eight
    // that end with it are read and moved down; what is outside counts as 0.
    float v[8][8];
    const bool whole = c0 + FB <= p.cols && ((int64_t)blockIdx.y + 1) * FB <= p.rows;      // (of the workgroup)
    {
        const int64_t cl = c < p.cols - 8 ? c : p.cols - 8;
        Span<T, 8> x[8], y[8];
        if constexpr (!NARROW) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int64_t at = (r0 + k < p.rows ? r0 + k : p.rows - 1) * p.ld + cl;
                x[k] = *(const Span<T, 8>*)((const T*)p.x + at);
                if (GATE) y[k] = *(const Span<T, 8>*)((const T*)p.gate + at);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int64_t at = (r0 + k < p.rows ? r0 + k : p.rows - 1) * p.ld + (e < p.cols ? e : p.cols - 1);
                    x[k].e[e] = ((const T*)p.x)[at];
                    if (GATE) y[k].e[e] = ((const T*)p.gate)[at];
                }
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[k][e] = to_f(x[k].e[e]);
                if (GATE && !(to_f(y[k].e[e]) > 0.0f)) v[k][e] = 0.0f;
            }
        if (!whole) {
            const int down = !NARROW ? (int)(c - cl < 8 ? c - cl : 8) : 0, n = (int)(c >= p.cols ? 0 : (p.cols - c < 8 ? p.cols - c : 8));
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
                for (int s = 4; s; s >>= 1)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[k][e] = (down & s) ? (e + s < 8 ? v[k][e + s] : 0.0f) : v[k][e];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] = e < n && r0 + k < p.rows ? v[k][e] : 0.0f;
            }
        }
    }
    auto max2 = [](float a, float b) { return fmaxf(a, b); };
    auto finite = [](float x) { return fabsf(x) < INFINITY ? fabsf(x) : 0.0f; };
    int tile_byte = 0;
    if (BR == FB) {
        float m = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[k][e]));
        if (__any(m == INFINITY)) {
            m = 0.0f;
            for (int k = 0; k < 8; ++k) for (int e = 0; e < 8; ++e) m = fmaxf(m, finite(v[k][e]));
        }
        m = wave_max(m);
        if (lane == 0) red[w][0] = m;
        __syncthreads();
        tile_byte = scale_byte(fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0])));
    }
    if (ROW) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            int b = tile_byte;
            if (BR == 1) {
                float m = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[k][e]));
                if (__any(m == INFINITY)) {
                    m = 0.0f;
                    for (int e = 0; e < 8; ++e) m = fmaxf(m, finite(v[k][e]));
                }
                b = scale_byte(lanes_max<16>(m));
            }
            if (r0 + k < p.rows) {
                *(uint2*)(p.q + (r0 + k) * p.pitch + c) = enc8(v[k], inv_scale_of(b));
                if (l16 == 0) p.s[(r0 + k) * p.spitch + blockIdx.x] = (uint8_t)b;
                if (blockIdx.x == gridDim.x - 1 && l16 > 0 && blockIdx.x + l16 < p.spitch) p.s[(r0 + k) * p.spitch + blockIdx.x + l16] = 127;
            }
        }
    }
    if (COL) {
        float inv[8];
        if (BR == 1) {
            float m[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                m[e] = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) m[e] = fmaxf(m[e], fabsf(v[k][e]));
                if (__any(m[e] == INFINITY)) {
                    m[e] = 0.0f;
                    for (int k = 0; k < 8; ++k) m[e] = fmaxf(m[e], finite(v[k][e]));
                }
                m[e] = groups_reduce(m[e], max2);
            }
            if (lane < 16) {
                *(float4*)&red[w][l16 * 8] = make_float4(m[0], m[1], m[2], m[3]);
                *(float4*)&red[w][l16 * 8 + 4] = make_float4(m[4], m[5], m[6], m[7]);
            }
            __syncthreads();
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float4 t = *(const float4*)&red[0][l16 * 8 + 4 * h];
#pragma unroll
                for (int o = 1; o < 4; ++o) {
                    const float4 u = *(const float4*)&red[o][l16 * 8 + 4 * h];
                    t = make_float4(fmaxf(t.x, u.x), fmaxf(t.y, u.y), fmaxf(t.z, u.z), fmaxf(t.w, u.w));
                }
                m[4 * h] = t.x; m[4 * h + 1] = t.y; m[4 * h + 2] = t.z; m[4 * h + 3] = t.w;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int b = scale_byte(m[e]);
                inv[e] = inv_scale_of(b);
                if (threadIdx.x < 16 && c + e < p.cols) {
                    uint8_t* st = p.st + (c + e) * p.tspitch + blockIdx.y;
                    st[0] = (uint8_t)b;
                    if (blockIdx.y == gridDim.y - 1) for (int k = 1; blockIdx.y + k < p.tspitch; ++k) st[k] = 127;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                inv[e] = inv_scale_of(tile_byte);
                if (threadIdx.x < 16 && c + e < p.cols) {
                    uint8_t* st = p.st + (c + e) * p.tspitch + blockIdx.y;
                    st[0] = (uint8_t)tile_byte;
                    if (blockIdx.y == gridDim.y - 1) for (int k = 1; blockIdx.y + k < p.tspitch; ++k) st[k] = 127;
                }
            }
        }
        // through LDS, so that a column's 128 bytes leave as one line: piece j (8 bytes) of column c lies at piece j + c / 8 of its 16, which spreads a store's
        // 16 columns, eight apart, over all banks
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t[8] = {v[0][e], v[1][e], v[2][e], v[3][e], v[4][e], v[5][e], v[6][e], v[7][e]};
            turn[l16 * 8 + e][(w * 4 + (lane >> 4) + l16) & 15] = enc8(t, inv[e]);
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int col = k * 32 + (threadIdx.x >> 3), j = (threadIdx.x & 7) * 2 + (col >> 3);
            const uint2 lo = turn[col][j & 15], hi = turn[col][(j + 1) & 15];
            if (c0 + col < p.cols) *(uint4*)(p.qt + (c0 + col) * p.tpitch + (int64_t)blockIdx.y * FB + (threadIdx.x & 7) * 16) = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        if (p.part) {
            float sum[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sum[e] = ((v[0][e] + v[1][e]) + (v[2][e] + v[3][e])) + ((v[4][e] + v[5][e]) + (v[6][e] + v[7][e]));
                sum[e] = groups_reduce(sum[e], [](float a, float b) { return a + b; });
            }
            __syncthreads();
            if (lane < 16) {
                *(float4*)&red[w][l16 * 8] = make_float4(sum[0], sum[1], sum[2], sum[3]);
                *(float4*)&red[w][l16 * 8 + 4] = make_float4(sum[4], sum[5], sum[6], sum[7]);
            }
            __syncthreads();
            const int t = threadIdx.x;
            if (t < FB && c0 + t < p.cols) p.part[(int64_t)blockIdx.y * p.cols + c0 + t] = (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]);
        }
    }
}

// the tiles' column sums added up in a fixed order: 64 columns and 16 shares of the tiles per workgroup.  Bound by the launch: 4.6 us for 256 tiles of 512 columns
__global__ __launch_bounds__(1024) void k_colsum(const float* part, int64_t tiles, int64_t cols, void* out, int out_dtype) {
    __shared__ float red[16][64];
    const int x = threadIdx.x & 63, y = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + x;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int64_t i = y; i < tiles; i += 16) s += part[i * cols + c];
    }
    red[y][x] = s;
    __syncthreads();
    if (y == 0 && c < cols) {
#pragma unroll
        for (int k = 1; k < 16; ++k) s += red[k][x];
        if (out_dtype == AGZ_F32) ((float*)out)[c] = s;
        else if (out_dtype == AGZ_BF16) ((bf16*)out)[c] = from_f<bf16>(s);
        else ((f16*)out)[c] = from_f<f16>(s);
    }
}

typedef __attribute__((ext_vector_type(8))) int i32x8;
typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef __attribute__((ext_vector_type(4))) float f32x4;

struct MatPar {
    const uint8_t *qa, *sa, *qb, *sb;
    int64_t m, n, k, pitch, spitch;
    const void* bias; int bias_dtype, relu;
    void* out; int out_dtype; int64_t ldo;
    int slices; float* part;                    // slices of the k axis; above one: their results, [slices][m][n]
};

__device__ __forceinline__ float load_as(const void* p, int dtype, int64_t i) {
    return dtype == AGZ_F32 ? ((const float*)p)[i] : dtype == AGZ_BF16 ? to_f(((const bf16*)p)[i]) : to_f(((const f16*)p)[i]);
}
__device__ __forceinline__ i32x8 load32(const uint8_t* p) {
    const i32x4 a = *(const i32x4*)p, b = *(const i32x4*)(p + 16);
    return i32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// v_mfma_scale_f32_16x16x128_f8f6f4: lane l holds 32 of the 128 k of row l % 16 of A and of B — the same 32 for both, so which does not matter —
// and one scale byte for them (byte SEL of a word); all four lanes of a row have the block's.  Result: column l % 16, rows 4 (l / 16) + i.
template <int SEL> __device__ __forceinline__ f32x4 mma(i32x8 a, i32x8 b, f32x4 c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, SEL, sa, SEL, sb);
}

// The matrix unit adds the products of 8 values in groups of eight, cut off at 2^-13 of the group's largest (measured: beside a product of 2^16 one of 2^3
// in the same eight counts, one of 2^2 does not; between groups it keeps 24 bits): 3e-5 of the result's norm on normally distributed values, a
// seventieth of the rounding of a 16-bit result.  Two kinds of results need more: those in 32 bits, and those behind a relu, whose signs decide which
// gradients pass (measured on 32768 x 512 x 512: with the products of 8 bits some signs next to 0 change and dw is 2.4e-3 off, with these it is not).
// Their values become bf16 on the way (exact, the scale applied: 4 bits of mantissa, 8 of exponent) for v_mfma_f32_16x16x32_bf16, at half the rate.
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8_t;
struct Wide { bf16x8_t v[4]; };
__device__ __forceinline__ Wide widen(i32x8 q, int byte) {
    Wide o;
    const float s = __uint_as_float((uint32_t)byte << 23);       // (the conversion takes the exponent's bits: 2^(byte - 127), also for byte 0)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)q[2 * i + h], s, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)q[2 * i + h], s, true);
            o.v[i][4 * h] = lo[0]; o.v[i][4 * h + 1] = lo[1]; o.v[i][4 * h + 2] = hi[0]; o.v[i][4 * h + 3] = hi[1];
        }
    return o;
}
__device__ __forceinline__ f32x4 mma_wide(const Wide& a, const Wide& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v[i], b.v[i], c, 0, 0, 0);
    return c;
}

// ---------------------------------------------------------------------------------------------------------------------------------------
// Tiles of BM x BN, the k axis in steps of one block of 128: both operands' rows of a step (128 bytes each) go from memory straight into LDS
// (global_load_lds, 16 bytes a lane), two steps deep, one barrier per step.  The 16-byte piece c of row r lies at piece c ^ (r & 7), so that the
// eight lanes that a ds_read_b128 serves at a time, eight rows of one piece, meet all banks once (the permutation is on the memory side: the DMA
// writes lanes in order).  WM x WN waves, each BM / WM x BN / WN in tiles of 16 x 16; B is the first operand, so that a lane ends with four
// neighbouring columns of one row.  Rows and columns outside are read from the last one and not stored.  Scales: a word holds a row's bytes of four steps; the words
// go through LDS too (a load to registers inside the loop would have to be waited for, and with it the next step's loads).
// Bound by the matrix unit and, for long k, by the clock, which falls under its load: a product alone is faster than the same among others.  Tiles of 256:
// 8192 x 4096 x 8192 (m x n x k) 221 us alone = 2.49 PFLOP/s, 237 us in a learning step = 2.32 (the library's product with one scale for each whole matrix, without blocks:
// 3.3 alone), 8192 x 8192 x 4096 259-261 us = 2.11 (2.76), to 32 bits 405 us alone = 1.36, 438 us in a step = 1.26 (the library's bf16 product: 1.57).  They hold 256
// registers, and spill 27 or 28 of them in front of their results.  Tiles of 128: 32768 x 512 x 512 21.9 us, behind a relu 30.9 us, where loading the four steps, products
// and results (50 MB) overlap only between the two workgroups of a CU; four workgroups a CU with one buffer each: 23 and 30 us where two took 20.5 and 26.4, with 23 to
// 41 registers spilled.
// ---------------------------------------------------------------------------------------------------------------------------------------
typedef __attribute__((address_space(1))) const void gvoid;
typedef __attribute__((address_space(3))) void lvoid;

template <typename O> __device__ __forceinline__ void store4(O* to, f32x4 v, int valid) {
    if (valid >= 4) {
        Span<O, 4> s;
#pragma unroll
        for (int e = 0; e < 4; ++e) s.e[e] = from_f<O>(v[e]);
        *(Span<O, 4>*)to = s;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e) if (e < valid) to[e] = from_f<O>(v[e]);
    }
}
__device__ __forceinline__ f32x4 bias4(const MatPar& p, int64_t c) {
    f32x4 b = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < 4; ++e) if (p.bias && c + e < p.n) b[e] = load_as(p.bias, p.bias_dtype, c + e);
    return b;
}
__device__ __forceinline__ f32x4 finish4(const MatPar& p, f32x4 v, f32x4 b) {
    v += b;
    if (p.relu)
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = v[e] < 0.0f ? 0.0f : v[e];        // (NaN stays NaN)
    return v;
}
__device__ __forceinline__ void store_row4(const MatPar& p, int64_t r, int64_t c, f32x4 v) {
    const int valid = (int)(p.n - c < 4 ? p.n - c : 4);
    v = finish4(p, v, bias4(p, c));
    const int64_t at = r * p.ldo + c;
    if (p.out_dtype == AGZ_F32) store4((float*)p.out + at, v, valid);
    else if (p.out_dtype == AGZ_BF16) store4((bf16*)p.out + at, v, valid);
    else store4((f16*)p.out + at, v, valid);
}

template <int BM, int BN, int WM, int WN, bool WIDE> struct Tile {
    static constexpr int NT = WM * WN * 64, FM = BM / WM / 16, FN = BN / WN / 16, PA = BM * 8 / NT, PB = BN * 8 / NT;
    static constexpr bool TURNS = WM * WN == 8 && !WIDE;
    static constexpr int STEP = (BM + BN) * FB, ROW = BN * 2 + 16, OUT = BM * ROW;         // bytes of a step, of a row and of all rows of a 16-bit result
    static constexpr int IN = 2 * STEP + 2 * (BM + BN) * 4, LDS = IN > OUT ? IN : OUT;     // two steps and two groups of scale words
    static_assert((BM + BN) % NT == 0 && BM % 64 == 0 && NT % 128 == 0 && PA * NT == BM * 8 && PB * NT == BN * 8, "whole pieces");
};

// a tile's results: through LDS (rows padded by 16 bytes, so that the 16 rows that a store covers meet different banks), then whole rows to memory;
// a result in 32 bits in two halves, by rows of waves
template <typename O, typename TL, int BM, int BN, int WM, int WN>
__device__ __forceinline__ void store_tile(uint8_t* lds, const f32x4 (&acc)[TL::FM][TL::FN], O* out, int64_t ld, int64_t m, int64_t n, int64_t m0, int64_t n0) {
    constexpr int HALVES = sizeof(O) == 4 ? 2 : 1, RB = BM / HALVES, ROW = BN * sizeof(O) + 16, EV = 16 / sizeof(O), CHUNKS = BN / EV;
    static_assert(WM % HALVES == 0 && RB * ROW <= TL::LDS, "a half of the tile fits");
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l16 = lane & 15, g = lane >> 4;
    const int wm = (w / WN) * (BM / WM), wn = (w % WN) * (BN / WN);
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        __syncthreads();
        if (wm / RB == h) {
#pragma unroll
            for (int i = 0; i < TL::FM; ++i)
#pragma unroll
                for (int j = 0; j < TL::FN; ++j) {
                    Span<O, 4> s;
#pragma unroll
                    for (int e = 0; e < 4; ++e) s.e[e] = from_f<O>(acc[i][j][e]);
                    __builtin_memcpy(__builtin_assume_aligned(lds + (wm - h * RB + i * 16 + l16) * ROW + (wn + j * 16 + g * 4) * (int)sizeof(O), 8), &s, sizeof s);
                }
        }
        __syncthreads();
        for (int x = tid; x < RB * CHUNKS; x += TL::NT) {
            const int r = x / CHUNKS, c = x % CHUNKS * EV;
            const int64_t row = m0 + h * RB + r, col = n0 + c;
            if (row >= m || col >= n) continue;
            Span<O, EV> s;
            __builtin_memcpy(&s, __builtin_assume_aligned(lds + r * ROW + c * (int)sizeof(O), 16), 16);
            O* to = out + row * ld + col;
            if (col + EV <= n) *(Span<O, EV>*)to = s;
            else
#pragma unroll
                for (int e = 0; e < EV - 1; ++e) if (col + e < n) to[e] = s.e[e];
        }
    }
}

template <int BM, int BN, int WM, int WN, bool WIDE>
__global__ __launch_bounds__(WM * WN * 64) void k_matmul_fp8(MatPar p) {
    using TL = Tile<BM, BN, WM, WN, WIDE>;
    constexpr int NT = TL::NT, FM = TL::FM, FN = TL::FN, PA = TL::PA, PB = TL::PB;
    __shared__ __attribute__((aligned(16))) uint8_t lds[TL::LDS];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
    // workgroups of one XCD (every eighth id) take neighbouring tiles: eight rows of tiles by all columns, so that their L2 holds the operands they share
    const uint32_t tm = (uint32_t)((p.m + BM - 1) / BM), tn = (uint32_t)((p.n + BN - 1) / BN), tiles = tm * tn;
    uint32_t id = blockIdx.x % tiles;
    const uint32_t slice = blockIdx.x / tiles;
    {
        const uint32_t per = tiles / 8, rest = tiles % 8, x = id % 8, o = id / 8;
        id = x * per + (x < rest ? x : rest) + o;
    }
    const uint32_t band = id / (8 * tn), rows = tm - band * 8 < 8 ? tm - band * 8 : 8, in = id - band * 8 * tn;
    const int64_t m0 = (int64_t)(band * 8 + in % rows) * BM, n0 = (int64_t)(in / rows) * BN;
    const int wm = (w / WN) * (BM / WM), wn = (w % WN) * (BN / WN);
    const int kb = (int)((p.k + FB - 1) / FB);
    const int k0 = (int)((int64_t)kb * slice / p.slices), k1 = (int)((int64_t)kb * (slice + 1) / p.slices);

    // this thread's pieces of a step: piece tid + i NT of the tile's (BM + BN) * 8, whole waves in A or in B; offsets from the tile's first row
    const uint32_t lastm = (uint32_t)(p.m - 1 - m0 < BM ? p.m - 1 - m0 : BM - 1), lastn = (uint32_t)(p.n - 1 - n0 < BN ? p.n - 1 - n0 : BN - 1);
    const uint32_t pitch = (uint32_t)p.pitch, spitch = (uint32_t)p.spitch;
    const uint8_t *qa = p.qa + m0 * p.pitch, *qb = p.qb + n0 * p.pitch, *sa = p.sa + m0 * p.spitch, *sb = p.sb + n0 * p.spitch;
    // the pieces of a step that a thread fetches: FT threads (with turns, those of the first half of the waves), piece tid + i FT; further pieces are FT / 8 rows
    // apart, a multiple of 8: the same place in the row.  The offsets are worked out anew each time (kept, they would cost a register each).
    constexpr int FT = TL::TURNS ? NT / 2 : NT;
    auto fetch = [&](int k, int buf) {
        uint32_t row0 = tid >> 3;
        asm volatile("" : "+v"(row0));
        const uint32_t piece0 = ((tid & 7) ^ (row0 & 7)) * 16;
        const uint8_t *a = qa + (int64_t)k * FB, *b = qb + (int64_t)k * FB;
        asm volatile("" : "+s"(a), "+s"(b));
        const uint32_t to = (uint32_t)buf * TL::STEP + w * 1024;
#pragma unroll
        for (int i = 0; i < BM * 8 / FT; ++i) {
            const uint32_t r = row0 + i * (FT / 8);
            __builtin_amdgcn_global_load_lds((gvoid*)(a + (__umul24(r < lastm ? r : lastm, pitch) + piece0)), (lvoid*)(lds + to + i * FT * 16), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < BN * 8 / FT; ++i) {
            const uint32_t r = row0 + i * (FT / 8);
            __builtin_amdgcn_global_load_lds((gvoid*)(b + (__umul24(r < lastn ? r : lastn, pitch) + piece0)), (lvoid*)(lds + BM * FB + to + i * FT * 16), 16, 0, 0);
        }
    };
    // scale words of a group of four steps: one per row of the tile, BM + BN of them, into the buffer of the group's parity
    auto fetch_scales = [&](int word) {
#pragma unroll
        for (int i = 0; i < (BM + BN) / FT; ++i) {
            uint32_t x = tid + i * FT;
            asm volatile("" : "+v"(x));
            const bool ofa = w * 64 + i * FT < BM;               // (a whole wave in one of them)
            const uint32_t r = ofa ? x : x - BM, last = ofa ? lastm : lastn;
            __builtin_amdgcn_global_load_lds((gvoid*)((ofa ? sa : sb) + word * 4 + (r < last ? r : last) * spitch), (lvoid*)(lds + 2 * TL::STEP + (word & 1) * (BM + BN) * 4 + i * FT * 4 + w * 256), 4, 0, 0);
        }
    };
    f32x4 acc[FM][FN] = {};
    uint32_t as[FM], bs[FN];
    if (k0 < k1 && w < FT / 64) {
        fetch_scales(k0 >> 2);
        fetch(k0, 0);
    }
    const int p0 = (g ^ (l16 & 7)) * 16, p1 = p0 ^ 64;
    auto frag = [&](const uint8_t* base, int i) {
        const i32x4 x = *(const i32x4*)(base + i * 16 * FB + p0), y = *(const i32x4*)(base + i * 16 * FB + p1);
        return i32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };
    auto take_scales = [&](int k) {                              // the step's bytes at the bottom of the words
        if (k == k0 || (k & 3) == 0) {
            const uint32_t* words = (const uint32_t*)(lds + 2 * TL::STEP + ((k >> 2) & 1) * (BM + BN) * 4) + l16;
#pragma unroll
            for (int i = 0; i < FM; ++i) as[i] = words[wm + i * 16] >> 8 * (k & 3);
#pragma unroll
            for (int j = 0; j < FN; ++j) bs[j] = words[BM + wn + j * 16] >> 8 * (k & 3);
        } else {
#pragma unroll
            for (int i = 0; i < FM; ++i) as[i] >>= 8;
#pragma unroll
            for (int j = 0; j < FN; ++j) bs[j] >>= 8;
        }
    };
    auto fetch_next = [&](int k) {
        if (k + 1 < k1) {
            if (((k + 1) & 3) == 0) fetch_scales((k + 1) >> 2);
            fetch(k + 1, (k + 1 - k0) & 1);
        }
    };
    if constexpr (TL::TURNS) {
        // The two waves of a SIMD (w and w + 4) take turns: while one reads its operands of a step from LDS, all of them, into registers, the other multiplies.
        // Phase 2 k: the first four waves read step k, the others multiply step k - 1; phase 2 k + 1: the other way round; a barrier between phases.  The first
        // four, whose registers are free then, fetch step k + 1 from phase 2 k on (its buffer was last read in phase 2 k - 1) and has to be there at the end of phase 2 k + 1.
        i32x8 av[FM], bv[FN];
        auto read = [&](int k) {
            const uint8_t* la = lds + ((k - k0) & 1) * TL::STEP + (wm + l16) * FB;
            const uint8_t* lb = lds + ((k - k0) & 1) * TL::STEP + BM * FB + (wn + l16) * FB;
#pragma unroll
            for (int j = 0; j < FN; ++j) bv[j] = frag(lb, j);
#pragma unroll
            for (int i = 0; i < FM; ++i) av[i] = frag(la, i);
            take_scales(k);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        auto multiply = [&]() {
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = mma<0>(bv[j], av[i], acc[i][j], (int)bs[j], (int)as[i]);
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
        };
        if (w < WM * WN / 2) {
            for (int k = k0; k < k1; ++k) {
                __syncthreads();
                fetch_next(k);
                read(k);
                __builtin_amdgcn_s_barrier();
                multiply();
            }
        } else {
            for (int k = k0; k < k1; ++k) {
                __syncthreads();
                if (k > k0) multiply();
                __builtin_amdgcn_s_barrier();
                read(k);
            }
            if (k0 < k1) multiply();
        }
    } else {
        for (int k = k0; k < k1; ++k) {
            __syncthreads();                                     // step k is in LDS, and everybody is done with the buffer of step k - 1
            fetch_next(k);
            take_scales(k);
            const uint8_t* la = lds + ((k - k0) & 1) * TL::STEP + (wm + l16) * FB;
            const uint8_t* lb = lds + ((k - k0) & 1) * TL::STEP + BM * FB + (wn + l16) * FB;
            // (the scheduler would move a row's read behind the products of the row before it, into the same registers: the barriers keep it one row ahead)
            if constexpr (WIDE) {
                Wide bw[FN];
#pragma unroll
                for (int j = 0; j < FN; ++j) bw[j] = widen(frag(lb, j), bs[j] & 0xFF);
                i32x8 av = frag(la, 0);
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    const Wide aw = widen(av, as[i] & 0xFF);
                    if (i + 1 < FM) av = frag(la, i + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mma_wide(bw[j], aw, acc[i][j]);
                }
            } else {
                i32x8 bv[FN], av[2];
                av[0] = frag(la, 0);
#pragma unroll
                for (int j = 0; j < FN; ++j) bv[j] = frag(lb, j);
#pragma unroll
                for (int i = 0; i < FM; ++i) {
                    if (i + 1 < FM) av[(i + 1) & 1] = frag(la, i + 1);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = 0; j < FN; ++j) acc[i][j] = mma<0>(bv[j], av[i & 1], acc[i][j], (int)bs[j], (int)as[i]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
    if (p.slices > 1) {
        store_tile<float, TL, BM, BN, WM, WN>(lds, acc, p.part + (int64_t)slice * p.m * p.n, p.n, p.m, p.n, m0, n0);
        return;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const f32x4 b = bias4(p, n0 + wn + j * 16 + g * 4);
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[i][j] = finish4(p, acc[i][j], b);
    }
    if (p.out_dtype == AGZ_F32) { if constexpr (WIDE) store_tile<float, TL, BM, BN, WM, WN>(lds, acc, (float*)p.out, p.ldo, p.m, p.n, m0, n0); }
    else if (p.out_dtype == AGZ_BF16) store_tile<bf16, TL, BM, BN, WM, WN>(lds, acc, (bf16*)p.out, p.ldo, p.m, p.n, m0, n0);
    else store_tile<f16, TL, BM, BN, WM, WN>(lds, acc, (f16*)p.out, p.ldo, p.m, p.n, m0, n0);
}

// the slices of the k axis added up, in order.  Bound by memory: 32 slices of 512 x 512 6.6 us (34 MB, 5.1 TB/s)
__global__ __launch_bounds__(256) void k_matmul_join(MatPar p) {
    const int64_t quads = (p.n + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x, r = i / quads, c = (i - r * quads) * 4;
    if (r >= p.m) return;
    const int valid = (int)(p.n - c < 4 ? p.n - c : 4);
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    const float* at = p.part + r * p.n + c;
    const int64_t next = p.m * p.n;
    if (valid == 4) {
        int s = 0;
        for (; s + 8 <= p.slices; s += 8) {                      // eight loads under way
            Span<float, 4> t[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) t[u] = *(const Span<float, 4>*)(at + (s + u) * next);
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += t[u].e[e];
        }
        for (; s < p.slices; ++s) {
            const Span<float, 4> t = *(const Span<float, 4>*)(at + s * next);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += t.e[e];
        }
    } else
        for (int s = 0; s < p.slices; ++s)
#pragma unroll
            for (int e = 0; e < 3; ++e) if (e < valid) v[e] += at[s * next + e];
    store_row4(p, r, c, v);
}

// 32 values of a block of 128 that four neighbouring lanes share, held in 8 bits: what k_quantize would have written, and the byte of the scale.  n: how many
// of the 32 there are (the others count as 0).
template <typename T> __device__ __forceinline__ int quantize32(const T* x, int n, uint8_t* to) {
    float v[32];
    if (n >= 32) {
        Span<T, 8> s[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) s[k] = *(const Span<T, 8>*)(x + 8 * k);
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = to_f(s[k / 8].e[k % 8]);
    } else
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = k < n ? to_f(x[k]) : 0.0f;
    float m = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) m = fmaxf(m, fabsf(v[k]));
    if (__any(m == INFINITY)) {
        m = 0.0f;
        for (int k = 0; k < 32; ++k) m = fmaxf(m, fabsf(v[k]) < INFINITY ? fabsf(v[k]) : 0.0f);
    }
    const int byte = scale_byte(lanes_max<4>(m));
    const float inv = inv_scale_of(byte);
#pragma unroll
    for (int k = 0; k < 4; ++k) *(uint2*)(to + 8 * k) = enc8(v + 8 * k, inv);
    return byte;
}

// Few rows (up to 16): the weights are read once, straight into the matrix unit's registers, and that is all the time there is.  A wave takes 16
// columns and every FEW_WAVES-th group of four steps; the waves of a workgroup add up through LDS.  T: uint8_t for a matrix in 8 bits, or the type of
// x, which every workgroup then holds in 8 bits itself, in LDS (a launch less; as long as its rows are short, x comes from the caches:
// one row of 8192 and 8192 columns 19.7 us in two launches, 14.7-15.4 us in one: 67 MB of weights, 4.4-4.6 TB/s).
constexpr int FEW_WAVES = 4, FEW_DEEP = 4, FEW_LDS = 32768;
template <typename T, bool WIDE> __global__ __launch_bounds__(FEW_WAVES * 64) void k_matmul_fp8_few(MatPar p, const T* x, int64_t ldx) {
    __shared__ f32x4 sum[FEW_WAVES][64];
    constexpr bool READY = std::is_same<T, uint8_t>::value;
    __shared__ __attribute__((aligned(16))) uint8_t held[READY ? 16 : FEW_LDS];
    __shared__ uint8_t held_scale[READY ? 1 : FEW_LDS / FB];
    // (the wave's number as one value of the wave: the matrix unit takes no heed of a lane condition, so none may stand around its instructions)
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g = lane >> 4;
    const int64_t n0 = (int64_t)blockIdx.x * 16;
    const int r = l16 < p.m ? l16 : (int)p.m - 1;
    const int64_t c = n0 + l16 < p.n ? n0 + l16 : p.n - 1;
    const uint8_t *a = READY ? p.qa + r * p.pitch + g * 32 : held + r * p.pitch + g * 32, *b = p.qb + c * p.pitch + g * 32;
    const int *sa = READY ? (const int*)(p.sa + r * p.spitch) : nullptr, *sb = (const int*)(p.sb + c * p.spitch);
    const int kb = (int)((p.k + FB - 1) / FB), whole = kb / FEW_DEEP;
    const uint8_t* sl = held_scale + r * kb;
    i32x8 bv[FEW_DEEP];
    int bs = 0;
    auto weights = [&](int q) {
#pragma unroll
        for (int k = 0; k < FEW_DEEP; ++k) bv[k] = load32(b + (int64_t)(q * FEW_DEEP + k) * FB);
        bs = sb[q];
    };
    if (w < whole) weights(w);
    if constexpr (!READY) {
        for (int t = threadIdx.x; t < (int)p.m * kb * 4; t += FEW_WAVES * 64) {      // (m pitch <= FEW_LDS)
            const int row = t / (kb * 4), at = t - row * kb * 4;
            const int64_t left = p.k - at * 32;
            const int byte = quantize32(x + row * ldx + at * 32, (int)(left < 0 ? 0 : (left < 32 ? left : 32)), held + row * p.pitch + at * 32);
            if ((at & 3) == 0) held_scale[row * kb + (at >> 2)] = (uint8_t)byte;
        }
        __syncthreads();
    }
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    auto one = [&](i32x8 av, i32x8 bw, int as, int bws) {
        if constexpr (WIDE) acc = mma_wide(widen(bw, bws & 0xFF), widen(av, as & 0xFF), acc);
        else acc = mma<0>(bw, av, acc, bws, as);
    };
    for (int q = w; q < whole; q += FEW_WAVES) {                 // FEW_DEEP = 4 steps: one word of scales
        if (q > w) weights(q);
        i32x8 av[FEW_DEEP];
        int as[FEW_DEEP];
#pragma unroll
        for (int k = 0; k < FEW_DEEP; ++k) av[k] = load32(a + (int64_t)(q * FEW_DEEP + k) * FB);
        if constexpr (READY) {
            const int word = sa[q];
#pragma unroll
            for (int k = 0; k < FEW_DEEP; ++k) as[k] = word >> 8 * k;
        } else {
#pragma unroll
            for (int k = 0; k < FEW_DEEP; ++k) as[k] = sl[q * FEW_DEEP + k];
        }
#pragma unroll
        for (int k = 0; k < FEW_DEEP; ++k) one(av[k], bv[k], as[k], bs >> 8 * k);
    }
    if (w == (whole & (FEW_WAVES - 1)))
        for (int k = whole * FEW_DEEP; k < kb; ++k)
            one(load32(a + (int64_t)k * FB), load32(b + (int64_t)k * FB), READY ? sa[k >> 2] >> 8 * (k & 3) : (int)sl[k], sb[k >> 2] >> 8 * (k & 3));
    sum[w][lane] = acc;
    __syncthreads();
    if (w == 0 && l16 < p.m && n0 + g * 4 < p.n) {
#pragma unroll
        for (int k = 1; k < FEW_WAVES; ++k) acc += sum[k][lane];
        store_row4(p, l16, n0 + g * 4, acc);
    }
}

// More rows on ready weights where the k axis has up to SHORT_STEPS steps: one launch too.  A workgroup turns its SHORT_M rows of x into 8 bits on their way into LDS (the
// same bits that k_quantize writes, 16 lanes a row and step), the weights' 128 rows come straight from memory, all steps at once; then products and results as in the
// tiles above.  Bound by latency where a workgroup or two a CU do it all (20001 x 162 -> 128 bf16, relu: 10.2 us a call in a graph, 11.9 us the launch under a profiler, 11.6 MB), by memory above:
// 200000 x 128 -> 128 30.6 us (102 MB, 3.3 TB/s).
constexpr int SHORT_STEPS = 4, SHORT_M = 64, SHORT_N = 128;
template <int KB> struct Short {
    static constexpr int NT = 256, FM = 2, FN = 4, STEP = (SHORT_M + SHORT_N) * FB, IN = KB * STEP + KB * SHORT_M, OUT = SHORT_M * (SHORT_N * 2 + 16), LDS = IN > OUT ? IN : OUT;
};
template <typename T, int KB, bool WIDE> __global__ __launch_bounds__(256) void k_linear_short(MatPar p, const T* x, int64_t ldx) {
    using TL = Short<KB>;
    constexpr int FM = TL::FM, FN = TL::FN, PASSES = SHORT_M / 16;
    __shared__ __attribute__((aligned(16))) uint8_t lds[TL::LDS];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), l16 = lane & 15, g = lane >> 4;
    const int64_t m0 = (int64_t)blockIdx.x * SHORT_M, n0 = (int64_t)blockIdx.y * SHORT_N;
    const int wm = (w >> 1) * 32, wn = (w & 1) * 64;
    // x: pass s of step k reads row 16 s + tid / 16, eight entries from column 128 k + 8 (tid % 16) on; entry by entry where the row ends inside the eight
    Span<T, 8> raw[KB][PASSES];
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int s = 0; s < PASSES; ++s) {
            const int64_t r = m0 + s * 16 + (tid >> 4) < p.m ? m0 + s * 16 + (tid >> 4) : p.m - 1;
            const T* row = x + r * ldx;
            const int at = k * FB + (tid & 15) * 8;
            if (k + 1 < KB || at + 8 <= (int)p.k) raw[k][s] = *(const Span<T, 8>*)(row + at);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) raw[k][s].e[e] = at + e < (int)p.k ? row[at + e] : from_f<T>(0.0f);
        }
    // the weights' rows: their pieces as in the tiles above, and a word of scales for all steps
    const uint32_t lastn = (uint32_t)(p.n - 1 - n0 < SHORT_N ? p.n - 1 - n0 : SHORT_N - 1), pitch = (uint32_t)p.pitch;
    const uint8_t* qb = p.qb + n0 * p.pitch;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int i = 0; i < SHORT_N * 8 / 256; ++i) {
            const uint32_t r = (tid >> 3) + i * 32, piece = ((tid & 7) ^ (r & 7)) * 16;
            __builtin_amdgcn_global_load_lds((gvoid*)(qb + k * FB + (r < lastn ? r : lastn) * pitch + piece), (lvoid*)(lds + k * TL::STEP + SHORT_M * FB + i * 4096 + w * 1024), 16, 0, 0);
        }
    uint32_t bs[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const uint32_t c = wn + j * 16 + l16;
        bs[j] = *(const uint32_t*)(p.sb + (n0 + (c < lastn ? c : lastn)) * p.spitch);
    }
    uint8_t* scale = lds + KB * TL::STEP;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int s = 0; s < PASSES; ++s) {
            float v[8], m = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) { v[e] = to_f(raw[k][s].e[e]); m = fmaxf(m, fabsf(v[e])); }
            if (__any(m == INFINITY)) {
                m = 0.0f;
                for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.0f);
            }
            const int byte = scale_byte(lanes_max<16>(m)), r = s * 16 + (tid >> 4);
            *(uint2*)(lds + k * TL::STEP + r * FB + (((tid & 15) >> 1) ^ (r & 7)) * 16 + (tid & 1) * 8) = enc8(v, inv_scale_of(byte));
            if ((tid & 15) == 0) scale[k * SHORT_M + r] = (uint8_t)byte;
        }
    __syncthreads();
    f32x4 acc[FM][FN] = {};
    const int p0 = (g ^ (l16 & 7)) * 16, p1 = p0 ^ 64;
    auto frag = [&](const uint8_t* base, int i) {
        const i32x4 x = *(const i32x4*)(base + i * 16 * FB + p0), y = *(const i32x4*)(base + i * 16 * FB + p1);
        return i32x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    };
#pragma unroll
    for (int k = 0; k < KB; ++k) {
        const uint8_t *la = lds + k * TL::STEP + (wm + l16) * FB, *lb = lds + k * TL::STEP + SHORT_M * FB + (wn + l16) * FB;
        i32x8 av[FM];
        int as[FM];
#pragma unroll
        for (int i = 0; i < FM; ++i) { av[i] = frag(la, i); as[i] = scale[k * SHORT_M + wm + i * 16 + l16]; }
        Wide aw[WIDE ? FM : 1];
        if constexpr (WIDE)
#pragma unroll
            for (int i = 0; i < FM; ++i) aw[i] = widen(av[i], as[i]);
#pragma unroll
        for (int j = 0; j < FN; ++j) {
            const i32x8 bv = frag(lb, j);
            if constexpr (WIDE) {
                const Wide bw = widen(bv, bs[j] >> 8 * k & 0xFF);
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[i][j] = mma_wide(bw, aw[i], acc[i][j]);
            } else
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[i][j] = mma<0>(bv, av[i], acc[i][j], (int)(bs[j] >> 8 * k), as[i]);
        }
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
        const f32x4 b = bias4(p, n0 + wn + j * 16 + g * 4);
#pragma unroll
        for (int i = 0; i < FM; ++i) acc[i][j] = finish4(p, acc[i][j], b);
    }
    store_tile<T, TL, SHORT_M, SHORT_N, 2, 2>(lds, acc, (T*)p.out, p.ldo, p.m, p.n, m0, n0);
}

}  // namespace ops
}  // namespace agz

using namespace agz::ops;

static bool too_large(int64_t a) { return a > (1ll << 31) - 256; }
static bool too_deep(int64_t k) { return k > (1ll << 24) - FB; }       // 255 rows of a tile and their pitch in 32 bits

// How a product runs: `few` rows, or tiles of 256 or 128 a side and slices of the k axis.  A tile of 256 reads half as much per operation and needs a whole CU; where
// there are fewer of them than CUs, or the k axis has fewer than eight steps (the loads of one tile and the results of another then overlap:
// 32768 x 512 x 512 23.3 -> 20.5 us, behind a relu 28.1 -> 26.4 us), tiles of 128, two a CU; and where these leave CUs idle too, the k axis is cut so that there are
// about two workgroups a CU, of at least four steps each (64 x 8192 x 8192: 22 us, with four a CU 31 us; 512 x 512 x 32768 to 32 bits: 32 us, 45 us).
namespace {
constexpr int CUS = 256;
struct Plan { bool few; int tile, slices; };
Plan plan(int64_t m, int64_t n, int64_t k) {
    if (m <= 16) return {true, 16, 1};
    const int64_t big = cdiv(m, 256) * cdiv(n, 256), small = cdiv(m, 128) * cdiv(n, 128), steps = cdiv(k, FB);
    if (big >= CUS && steps >= 8) return {false, 256, 1};
    int64_t slices = small < CUS ? 2 * CUS / small : 1;
    if (slices > steps / 4) slices = steps / 4;
    return {false, 128, (int)(slices < 1 ? 1 : slices)};
}
}

// the work of the entry points below, on the current device, arguments checked
namespace {
struct Mat8 { uint8_t *q, *s; };                 // a matrix in 8 bits
int quantize(void* stream, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* gate, int block_rows, Mat8 a, Mat8 t, void* colsum, int colsum_dtype, float* part) {
    if (cols == 0) return AGZ_OK;
    if (rows > 0) {
        const QuantPar p{x, gate, rows, cols, ld, a.q, a.s, t.q, t.s, up(cols, FB), up(cdiv(cols, FB), 4), up(rows, FB), up(cdiv(rows, FB), 4), colsum ? part : nullptr};
        const dim3 grid((uint32_t)cdiv(cols, FB), (uint32_t)cdiv(rows, FB));
        const int rc = by_dtype(dtype, [&](auto T) {
            using X = decltype(T);
            auto go = [&](auto br, auto gated) {
                if (cols < 8)
                    return a.q && t.q ? launch(k_quantize<X, br(), true, true, gated(), true>, grid, dim3(256), 0, stream, p)
                         : a.q ? launch(k_quantize<X, br(), true, false, gated(), true>, grid, dim3(256), 0, stream, p)
                               : launch(k_quantize<X, br(), false, true, gated(), true>, grid, dim3(256), 0, stream, p);
                if (a.q && t.q) return launch(k_quantize<X, br(), true, true, gated(), false>, grid, dim3(256), 0, stream, p);
                if (a.q) return launch(k_quantize<X, br(), true, false, gated(), false>, grid, dim3(256), 0, stream, p);
                return launch(k_quantize<X, br(), false, true, gated(), false>, grid, dim3(256), 0, stream, p);
            };
            using std::integral_constant;
            if (block_rows == 1) return gate ? go(integral_constant<int, 1>{}, std::true_type{}) : go(integral_constant<int, 1>{}, std::false_type{});
            return gate ? go(integral_constant<int, FB>{}, std::true_type{}) : go(integral_constant<int, FB>{}, std::false_type{});
        });
        if (rc != AGZ_OK) return rc;
    }
    if (!colsum) return AGZ_OK;
    return launch(k_colsum, dim3((uint32_t)cdiv(cols, 64)), dim3(1024), 0, stream, (const float*)part, cdiv(rows, FB), cols, colsum, colsum_dtype);
}

int product(void* stream, int64_t m, int64_t n, int64_t k, Mat8 a, Mat8 b, const void* bias, int bias_dtype, int relu, void* out, int out_dtype, int64_t ldo, void* ws) {
    if (m == 0 || n == 0) return AGZ_OK;
    const Plan w = plan(m, n, k);
    const MatPar p{a.q, a.s, b.q, b.s, m, n, k, up(k, FB), up(cdiv(k, FB), 4), bias, bias_dtype, relu, out, out_dtype, ldo, w.slices, (float*)ws};
    const bool wide = out_dtype == AGZ_F32 || relu;
    if (w.few) return launch(wide ? k_matmul_fp8_few<uint8_t, true> : k_matmul_fp8_few<uint8_t, false>, dim3((uint32_t)cdiv(n, 16)), dim3(FEW_WAVES * 64), 0, stream, p, (const uint8_t*)nullptr, (int64_t)0);
    const int64_t groups = cdiv(m, w.tile) * cdiv(n, w.tile) * w.slices;
    if (groups > 0x7fffffffll) return fail(AGZ_ERR_ARG, "a product of more than 2^31 tiles");
    const int rc = w.tile == 256 ? launch(wide ? k_matmul_fp8<256, 256, 2, 4, true> : k_matmul_fp8<256, 256, 2, 4, false>, dim3((uint32_t)groups), dim3(512), 0, stream, p)
                                 : launch(wide ? k_matmul_fp8<128, 128, 2, 2, true> : k_matmul_fp8<128, 128, 2, 2, false>, dim3((uint32_t)groups), dim3(256), 0, stream, p);
    if (rc != AGZ_OK || w.slices == 1) return rc;
    return launch(k_matmul_join, dim3((uint32_t)cdiv(m * cdiv(n, 4), 256)), dim3(256), 0, stream, p);
}

// matrices in 8 bits one behind the other in a buffer (every part at a multiple of 256 bytes); without a buffer it only counts
struct Carve {
    uint8_t* base; int64_t at = 0;
    uint8_t* take(int64_t bytes) { uint8_t* p = base ? base + at : nullptr; at += up(bytes, 256); return p; }
    Mat8 matrix(int64_t rows, int64_t cols) { Mat8 m; m.q = take(rows * up(cols, FB)); m.s = take(rows * up(cdiv(cols, FB), 4)); return m; }
};
bool good_sizes(int64_t m, int64_t n, int64_t k) { return m >= 0 && n >= 0 && k >= 0 && !too_large(m) && !too_large(n) && !too_deep(k) && cdiv(m, FB) <= 65535 && cdiv(n, FB) <= 65535; }
struct Forward { Mat8 a, b; void* ws; };
Forward forward_ws(Carve& c, int64_t m, int64_t n, int64_t k) { return {c.matrix(m, k), c.matrix(n, k), c.take(agz_fp8_matmul_workspace(m, n, k))}; }
// a layer on weights in 8 bits: x in 8 bits first, or on the way where its rows are few
struct Apply { Mat8 a; void* ws; };
bool at_once(int64_t m, int64_t n, int64_t k) { return plan(m, n, k).few && m * up(k, FB) <= FEW_LDS; }
// ... or, where the k axis is short too, x in 8 bits in the product's own launch.  Every 128 columns turn x into 8 bits again: up to 256 of them, or up to eight workgroups a
// CU; with four steps a workgroup fills a CU's LDS, and more than one a CU wait for each other.  In one launch and in two: 20001 x 162 -> 128 bf16 10.2 and 15.0 us,
// 1000 x 128 -> 128 5.8 and 10.4, 200000 x 128 -> 128 30.6 and 44.8, 32768 x 256 -> 512 25.7 and 29.4; but -> 1024 46.1 and 43.9, 8192 x 512 -> 512 16.7 and 15.0,
// 65536 x 512 -> 128 43.4 and 37.3.
bool in_one(int64_t m, int64_t n, int64_t k) {
    const int64_t steps = cdiv(k, FB), across = cdiv(n, SHORT_N), groups = cdiv(m, SHORT_M) * across;
    if (m <= 16 || k == 0 || steps > SHORT_STEPS) return false;
    return steps == SHORT_STEPS ? groups <= CUS : across <= 2 || groups <= 8 * CUS;
}
int layer_in_one(void* stream, const agz_linear_fp8_args* q, Mat8 b, void* y) {
    const MatPar p{nullptr, nullptr, b.q, b.s, q->m, q->n, q->k, up(q->k, FB), up(cdiv(q->k, FB), 4), q->bias, q->bias_dtype, q->relu, y, q->dtype, q->n, 1, nullptr};
    return by_dtype(q->dtype, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kb) {
            return launch(q->relu || q->dtype == AGZ_F32 ? k_linear_short<T, kb(), true> : k_linear_short<T, kb(), false>,
                          dim3((uint32_t)cdiv(p.m, SHORT_M), (uint32_t)cdiv(p.n, SHORT_N)), dim3(256), 0, stream, p, (const T*)q->x, q->ldx);
        };
        using std::integral_constant;
        switch (cdiv(p.k, FB)) {
            case 1: return go(integral_constant<int, 1>{});
            case 2: return go(integral_constant<int, 2>{});
            case 3: return go(integral_constant<int, 3>{});
            default: return go(integral_constant<int, 4>{});
        }
    });
}
Apply apply_ws(Carve& c, int64_t m, int64_t n, int64_t k) {
    if (at_once(m, n, k) || in_one(m, n, k)) return {};
    Apply w;
    w.a = c.matrix(m, k);
    w.ws = c.take(agz_fp8_matmul_workspace(m, n, k));
    return w;
}
struct Saved { Mat8 at, bt; };
Saved saved_of(Carve& c, int64_t m, int64_t n, int64_t k, bool need_dx, bool need_dw) {
    Saved s{};
    if (need_dw) s.at = c.matrix(k, m);
    if (need_dx) s.bt = c.matrix(k, n);
    return s;
}
struct Backward { Mat8 d, t; void *ws; float* part; };
Backward backward_ws(Carve& c, int64_t m, int64_t n, int64_t k, bool need_dx, bool need_dw, bool need_db) {
    Backward w{};
    if (need_dx) w.d = c.matrix(m, n);
    if (need_dw || need_db) w.t = c.matrix(n, m);
    if (need_db) w.part = (float*)c.take(agz_fp8_colsum_ws(m, n));
    const int64_t x = need_dx ? agz_fp8_matmul_workspace(m, k, n) : 0, y = need_dw ? agz_fp8_matmul_workspace(n, k, m) : 0;
    w.ws = c.take(x > y ? x : y);                // (one after the other on the stream)
    return w;
}
int check_linear(const char* who, const agz_linear_fp8_args* q) {
    if (!q) return fail(AGZ_ERR_ARG, "%s: no arguments", who);
    if (!good_sizes(q->m, q->n, q->k)) return fail(AGZ_ERR_ARG, "%s: %lld x %lld x %lld", who, (long long)q->m, (long long)q->n, (long long)q->k);
    if (!good_dtype(q->dtype) || !good_dtype(q->w_dtype) || (q->bias && !good_dtype(q->bias_dtype))) return fail(AGZ_ERR_ARG, "%s: unknown dtype", who);
    if (q->ldx < 0 || q->ldw < 0) return fail(AGZ_ERR_ARG, "%s: a negative stride", who);
    if (!aligned(q->x, esize(q->dtype)) || !aligned(q->w, esize(q->w_dtype)) || (q->bias && !aligned(q->bias, esize(q->bias_dtype)))) return fail(AGZ_ERR_ARG, "%s: a pointer is not aligned to its type", who);
    return AGZ_OK;
}
}  // namespace

extern "C" {

int64_t agz_fp8_pitch(int64_t cols) { return cols < 0 ? -1 : up(cols, FB); }
int64_t agz_fp8_scale_pitch(int64_t cols) { return cols < 0 ? -1 : up(cdiv(cols, FB), 4); }
int64_t agz_fp8_colsum_ws(int64_t rows, int64_t cols) { return rows < 0 || cols < 0 ? -1 : cdiv(rows, FB) * cols * 4; }

int agz_fp8_quantize(int device, void* stream, const void* x, int dtype, int64_t rows, int64_t cols, int64_t ld, const void* gate, int block_rows,
                     void* q, void* s, void* qt, void* st, float* colsum, void* ws, int64_t ws_bytes) {
    if (!good_dtype(dtype)) return fail(AGZ_ERR_ARG, "agz_fp8_quantize: unknown dtype %d", dtype);
    if (rows < 0 || cols < 0 || too_large(rows) || too_large(cols)) return fail(AGZ_ERR_ARG, "agz_fp8_quantize: %lld x %lld", (long long)rows, (long long)cols);
    if (ld < 0) return fail(AGZ_ERR_ARG, "agz_fp8_quantize: a negative stride");
    if (block_rows != 1 && block_rows != FB) return fail(AGZ_ERR_ARG, "agz_fp8_quantize: blocks of %d rows (1 or 128)", block_rows);
    if (rows > 0 && cols > 0 && (!q != !s || !qt != !st || (!q && !qt))) return fail(AGZ_ERR_ARG, "agz_fp8_quantize: q with s and / or qt with st");
    if (colsum && rows > 0 && cols > 0 && (!qt || !ws || ws_bytes < agz_fp8_colsum_ws(rows, cols) || !aligned(ws, 16))) return fail(AGZ_ERR_ARG, "agz_fp8_quantize: colsum needs qt and its workspace");
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    if (cols == 0 || (rows == 0 && !colsum)) return AGZ_OK;
    if (rows > 0 && (!x || !aligned(x, esize(dtype)) || !aligned(gate, esize(dtype)) || !aligned(q, 16) || !aligned(s, 4) || !aligned(qt, 16) || !aligned(st, 4)))
        return fail(AGZ_ERR_ARG, "agz_fp8_quantize: x missing, or a pointer that is not aligned (q, qt: to 16 bytes, scales: to 4)");
    if (cdiv(rows, FB) > 65535) return fail(AGZ_ERR_ARG, "agz_fp8_quantize: more than 65535 x 128 rows");
    return quantize(stream, x, dtype, rows, cols, ld, gate, block_rows, {(uint8_t*)q, (uint8_t*)s}, {(uint8_t*)qt, (uint8_t*)st}, colsum, AGZ_F32, (float*)ws);
}

int64_t agz_fp8_matmul_workspace(int64_t m, int64_t n, int64_t k) {
    if (m < 0 || n < 0 || k < 0 || too_large(m) || too_large(n) || too_deep(k)) return -1;
    if (m == 0 || n == 0) return 0;
    const Plan w = plan(m, n, k);
    return w.slices > 1 ? w.slices * m * n * 4 : 0;
}

int agz_fp8_matmul(int device, void* stream, int64_t m, int64_t n, int64_t k, const void* qa, const void* sa, const void* qb, const void* sb,
                   const void* bias, int bias_dtype, int relu, void* out, int out_dtype, int64_t ldo, void* ws, int64_t ws_bytes) {
    const int64_t need = agz_fp8_matmul_workspace(m, n, k);
    if (need < 0) return fail(AGZ_ERR_ARG, "agz_fp8_matmul: %lld x %lld x %lld", (long long)m, (long long)n, (long long)k);
    if (!good_dtype(out_dtype) || (bias && !good_dtype(bias_dtype))) return fail(AGZ_ERR_ARG, "agz_fp8_matmul: unknown dtype");
    if (need > 0 && (!ws || ws_bytes < need || !aligned(ws, 16))) return fail(AGZ_ERR_ARG, "agz_fp8_matmul: a workspace of %lld bytes, 16-byte aligned", (long long)need);
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    if (m == 0 || n == 0) return AGZ_OK;
    if (!out || ldo < n || !aligned(out, esize(out_dtype)) || (bias && !aligned(bias, esize(bias_dtype)))) return fail(AGZ_ERR_ARG, "agz_fp8_matmul: out with a row stride of at least %lld, aligned to its type", (long long)n);
    if (k > 0 && (!qa || !sa || !qb || !sb || !aligned(qa, 16) || !aligned(qb, 16) || !aligned(sa, 4) || !aligned(sb, 4)))
        return fail(AGZ_ERR_ARG, "agz_fp8_matmul: values aligned to 16 bytes and scales to 4");
    return product(stream, m, n, k, {(uint8_t*)qa, (uint8_t*)sa}, {(uint8_t*)qb, (uint8_t*)sb}, bias, bias_dtype, relu, out, out_dtype, ldo, ws);
}

int64_t agz_linear_fp8_workspace(int64_t m, int64_t n, int64_t k) {
    if (!good_sizes(m, n, k)) return -1;
    Carve c{nullptr};
    forward_ws(c, m, n, k);
    return c.at;
}
int64_t agz_linear_fp8_apply_workspace(int64_t m, int64_t n, int64_t k) {
    if (!good_sizes(m, n, k)) return -1;
    Carve c{nullptr};
    apply_ws(c, m, n, k);
    return c.at;
}
int64_t agz_linear_fp8_saved(int64_t m, int64_t n, int64_t k, int need_dx, int need_dw) {
    if (!good_sizes(m, n, k)) return -1;
    Carve c{nullptr};
    saved_of(c, m, n, k, need_dx, need_dw);
    return c.at;
}
int64_t agz_linear_fp8_backward_workspace(int64_t m, int64_t n, int64_t k, int need_dx, int need_dw, int need_db) {
    if (!good_sizes(m, n, k)) return -1;
    Carve c{nullptr};
    backward_ws(c, m, n, k, need_dx, need_dw, need_db);
    return c.at;
}

int agz_linear_fp8_forward(int device, void* stream, const agz_linear_fp8_args* q, void* y, void* saved, int need_dx, int need_dw, void* ws, int64_t ws_bytes) {
    if (int rc = check_linear("agz_linear_fp8_forward", q)) return rc;
    const int64_t need = agz_linear_fp8_workspace(q->m, q->n, q->k);
    if (need > 0 && (!ws || ws_bytes < need || !aligned(ws, 256))) return fail(AGZ_ERR_ARG, "agz_linear_fp8_forward: a workspace of %lld bytes, 256-byte aligned", (long long)need);
    if ((need_dx || need_dw) && (!aligned(saved, 256) || (!saved && agz_linear_fp8_saved(q->m, q->n, q->k, need_dx, need_dw) > 0))) return fail(AGZ_ERR_ARG, "agz_linear_fp8_forward: saved, 256-byte aligned");
    if ((q->m > 0 && q->n > 0 && (!y || !aligned(y, esize(q->dtype)))) || (q->m > 0 && q->k > 0 && !q->x) || (q->n > 0 && q->k > 0 && !q->w)) return fail(AGZ_ERR_ARG, "agz_linear_fp8_forward: x, w and y are required");
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    Carve c{(uint8_t*)ws}, d{(uint8_t*)saved};
    const Forward f = forward_ws(c, q->m, q->n, q->k);
    const Saved s = saved_of(d, q->m, q->n, q->k, need_dx, need_dw);
    if (int rc = quantize(stream, q->w, q->w_dtype, q->n, q->k, q->ldw, nullptr, FB, f.b, s.bt, nullptr, 0, nullptr)) return rc;
    if (!need_dw && q->m > 0 && q->n > 0 && in_one(q->m, q->n, q->k)) return layer_in_one(stream, q, f.b, y);
    if (int rc = quantize(stream, q->x, q->dtype, q->m, q->k, q->ldx, nullptr, 1, f.a, s.at, nullptr, 0, nullptr)) return rc;
    return product(stream, q->m, q->n, q->k, f.a, f.b, q->bias, q->bias_dtype, q->relu, y, q->dtype, q->n, f.ws);
}

int agz_linear_fp8_apply(int device, void* stream, const agz_linear_fp8_args* q, const void* qw, const void* sw, void* y, void* ws, int64_t ws_bytes) {
    if (int rc = check_linear("agz_linear_fp8_apply", q)) return rc;
    const int64_t m = q->m, n = q->n, k = q->k, need = agz_linear_fp8_apply_workspace(m, n, k);
    if (need > 0 && (!ws || ws_bytes < need || !aligned(ws, 256))) return fail(AGZ_ERR_ARG, "agz_linear_fp8_apply: a workspace of %lld bytes, 256-byte aligned", (long long)need);
    if ((m > 0 && n > 0 && (!y || !aligned(y, esize(q->dtype)))) || (m > 0 && k > 0 && !q->x) || (n > 0 && k > 0 && (!qw || !sw || !aligned(qw, 16) || !aligned(sw, 4))))
        return fail(AGZ_ERR_ARG, "agz_linear_fp8_apply: x, y and the weights (values aligned to 16 bytes, scales to 4) are required");
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    if (m == 0 || n == 0) return AGZ_OK;
    Carve c{(uint8_t*)ws};
    const Apply w = apply_ws(c, m, n, k);
    const Mat8 b{(uint8_t*)qw, (uint8_t*)sw};
    if (in_one(m, n, k)) return layer_in_one(stream, q, b, y);
    if (!at_once(m, n, k)) {
        if (int rc = quantize(stream, q->x, q->dtype, m, k, q->ldx, nullptr, 1, w.a, {}, nullptr, 0, nullptr)) return rc;
        return product(stream, m, n, k, w.a, b, q->bias, q->bias_dtype, q->relu, y, q->dtype, n, w.ws);
    }
    const MatPar p{nullptr, nullptr, b.q, b.s, m, n, k, up(k, FB), up(cdiv(k, FB), 4), q->bias, q->bias_dtype, q->relu, y, q->dtype, n, 1, nullptr};
    return by_dtype(q->dtype, [&](auto t) {
        using T = decltype(t);
        return launch(q->relu || q->dtype == AGZ_F32 ? k_matmul_fp8_few<T, true> : k_matmul_fp8_few<T, false>, dim3((uint32_t)cdiv(n, 16)), dim3(FEW_WAVES * 64), 0, stream, p, (const T*)q->x, q->ldx);
    });
}

int agz_linear_fp8_backward(int device, void* stream, const agz_linear_fp8_args* q, const void* dy, const void* y, const void* saved, int saved_dx, int saved_dw, void* dx, void* dw, void* db, void* ws, int64_t ws_bytes) {
    if (int rc = check_linear("agz_linear_fp8_backward", q)) return rc;
    const int64_t m = q->m, n = q->n, k = q->k, need = agz_linear_fp8_backward_workspace(m, n, k, !!dx, !!dw, !!db);
    if ((dx && !saved_dx) || (dw && !saved_dw)) return fail(AGZ_ERR_ARG, "agz_linear_fp8_backward: the forward call did not save what this needs");
    if (need > 0 && (!ws || ws_bytes < need || !aligned(ws, 256))) return fail(AGZ_ERR_ARG, "agz_linear_fp8_backward: a workspace of %lld bytes, 256-byte aligned", (long long)need);
    if (!aligned(saved, 256) || (!saved && agz_linear_fp8_saved(m, n, k, saved_dx, saved_dw) > 0)) return fail(AGZ_ERR_ARG, "agz_linear_fp8_backward: saved, 256-byte aligned");
    if (m > 0 && n > 0 && (!dy || (q->relu && !y) || !aligned(dy, esize(q->dtype)) || !aligned(y, esize(q->dtype)))) return fail(AGZ_ERR_ARG, "agz_linear_fp8_backward: dy, and y behind a relu, are required");
    if (!aligned(dx, esize(q->dtype)) || !aligned(dw, esize(q->w_dtype)) || (db && (!good_dtype(q->bias_dtype) || !aligned(db, esize(q->bias_dtype))))) return fail(AGZ_ERR_ARG, "agz_linear_fp8_backward: a pointer is not aligned to its type");
    OnDevice on(device);
    if (on.rc != AGZ_OK) return on.rc;
    Carve c{(uint8_t*)ws}, d{(uint8_t*)saved};
    const Backward b = backward_ws(c, m, n, k, dx, dw, db);
    const Saved s = saved_of(d, m, n, k, saved_dx, saved_dw);
    if (dx || dw || db) if (int rc = quantize(stream, dy, q->dtype, m, n, n, q->relu ? y : nullptr, 1, b.d, b.t, db, q->bias_dtype, b.part)) return rc;
    if (dx) if (int rc = product(stream, m, k, n, b.d, s.bt, nullptr, 0, 0, dx, q->dtype, k, b.ws)) return rc;
    if (dw) return product(stream, n, k, m, b.t, s.at, nullptr, 0, 0, dw, q->w_dtype, k, b.ws);
    return AGZ_OK;
}

}  // extern "C"
