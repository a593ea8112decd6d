// agz_ops.hpp — what the operators on device tensors (agz_logprob.hip, agz_fp8.hip, agz_adamw.hip) share: errors, the caller's device,
// launches, conversions between the tensor types and 32-bit floats, wave reductions.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <tuple>
#include <utility>
#include "../../include/agz.h"

namespace agz {
namespace ops {

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));    // sets agz_ops_last_error() of this thread, returns code

// the call's device for the time of the call: the caller's current device is put back at the end
struct OnDevice {
    int prev = -1, rc = AGZ_OK;
    explicit OnDevice(int device) {
        int n = 0;
        if (hipGetDeviceCount(&n) != hipSuccess || n == 0) { (void)hipGetLastError(); rc = fail(AGZ_ERR_HIP, "no HIP device (libagz has no CPU path)"); return; }
        if (device < 0 || device >= n) { rc = fail(AGZ_ERR_ARG, "device %d of %d", device, n); return; }
        int cur = -1;
        if (hipGetDevice(&cur) != hipSuccess) { rc = fail(AGZ_ERR_HIP, "hipGetDevice failed"); return; }
        if (cur != device) {
            if (hipSetDevice(device) != hipSuccess) { (void)hipGetLastError(); rc = fail(AGZ_ERR_HIP, "hipSetDevice(%d) failed", device); return; }
            prev = cur;
        }
    }
    ~OnDevice() { if (prev >= 0) (void)hipSetDevice(prev); }
    OnDevice(const OnDevice&) = delete;
    OnDevice& operator=(const OnDevice&) = delete;
};

// a launch that reports its own status (hipGetLastError would also report an error that somebody else's call left behind)
template <typename... P, typename... A> int launch(void (*k)(P...), dim3 grid, dim3 block, size_t lds, void* stream, A&&... a) {
    if ((uint64_t)grid.x * block.x > 0xFFFFFFFFull || grid.y > 65535) return fail(AGZ_ERR_ARG, "a launch of %u x %u workgroups: too large", grid.x, grid.y);
    std::tuple<P...> args(static_cast<P>(a)...);
    hipError_t e = std::apply([&](auto&... x) { void* p[] = {(void*)&x...}; return hipLaunchKernel((const void*)k, grid, block, p, lds, (hipStream_t)stream); }, args);
    if (e == hipSuccess) return AGZ_OK;
    (void)hipGetLastError();
    return fail(AGZ_ERR_HIP, "kernel launch: %s", hipGetErrorString(e));
}

inline bool aligned(const void* p, uintptr_t to) { return ((uintptr_t)p & (to - 1)) == 0; }
inline int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
inline int64_t cdiv(int64_t x, int64_t by) { return (x + by - 1) / by; }
inline int esize(int dtype) { return dtype == AGZ_F32 ? 4 : 2; }
inline bool good_dtype(int d) { return d == AGZ_F32 || d == AGZ_BF16 || d == AGZ_F16; }

struct bf16 { uint16_t u; };
typedef _Float16 f16;

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f(float x) { return x; }
template <> __device__ __forceinline__ float to_f(bf16 x) { return __uint_as_float((uint32_t)x.u << 16); }
template <> __device__ __forceinline__ float to_f(f16 x) { return (float)x; }
template <typename T> __device__ __forceinline__ T from_f(float x);      // to the nearest, ties to even; NaN stays NaN
template <> __device__ __forceinline__ float from_f(float x) { return x; }
template <> __device__ __forceinline__ bf16 from_f(float x) { __bf16 b = (__bf16)x; bf16 r; __builtin_memcpy(&r, &b, 2); return r; }
template <> __device__ __forceinline__ f16 from_f(float x) { return (f16)x; }

// reductions over G neighbouring lanes, the result in all of them: DPP inside a row of 16 lanes, register swaps between rows (no LDS)
template <int CTRL> __device__ __forceinline__ uint32_t dpp(uint32_t x) { return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false); }
template <int G, typename F> __device__ __forceinline__ uint32_t lanes_reduce(uint32_t x, F&& f) {
    if constexpr (G >= 2) x = f(x, dpp<0xB1>(x));            // quad_perm 1 0 3 2
    if constexpr (G >= 4) x = f(x, dpp<0x4E>(x));            // quad_perm 2 3 0 1
    if constexpr (G >= 8) x = f(x, dpp<0x141>(x));           // row_half_mirror
    if constexpr (G >= 16) x = f(x, dpp<0x140>(x));          // row_mirror
    if constexpr (G >= 32) { const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false); x = f(r[0], r[1]); }
    if constexpr (G >= 64) { const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false); x = f(r[0], r[1]); }
    return x;
}
template <int G> __device__ __forceinline__ float lanes_max(float x) {
    return __uint_as_float(lanes_reduce<G>(__float_as_uint(x), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
template <int G> __device__ __forceinline__ float lanes_sum(float x) {
    return __uint_as_float(lanes_reduce<G>(__float_as_uint(x), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
template <int G> __device__ __forceinline__ uint32_t lanes_min_u(uint32_t x) {
    return lanes_reduce<G>(x, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
__device__ __forceinline__ float wave_max(float x) { return lanes_max<64>(x); }
__device__ __forceinline__ float wave_sum(float x) { return lanes_sum<64>(x); }

// N neighbouring elements at any address that suits one element (the memory unit takes such addresses)
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Span { T e[N]; };

// the byte of the smallest power-of-two scale 2^(byte - 127) with amax <= 448 * scale (amax finite, >= 0; 448 = 1.75 * 2^8: the exponent less
// eight, one more where the mantissa is above 1.75); 127, a scale of one, for a block of zeros.  Subnormal amax: byte 0, 2^-127.
__device__ __forceinline__ int scale_byte(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return b == 0 ? 127 : (e < 0 ? 0 : e);
}
// 2^(byte - 127) and 2^(127 - byte): 2^-127 is below the normal numbers, 2^127 is the largest power
__device__ __forceinline__ float scale_of(int byte) { return byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float((uint32_t)byte << 23); }
__device__ __forceinline__ float inv_scale_of(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }   // byte <= 247: amax < 2^128

// dispatch on a dtype: f(T{})
template <typename F> int by_dtype(int d, F&& f) {
    switch (d) {
        case AGZ_F32: return f(float{});
        case AGZ_BF16: return f(bf16{});
        default: return f(f16{});
    }
}

}  // namespace ops
}  // namespace agz
