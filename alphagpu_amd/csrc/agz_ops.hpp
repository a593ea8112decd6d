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

__device__ __forceinline__ float wave_max(float x) { for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o)); return x; }
__device__ __forceinline__ float wave_sum(float x) { for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o); return x; }

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
