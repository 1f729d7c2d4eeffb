// Block-scaled fp8 codes: a thread has 8 consecutive channels of a row as four float pairs, 16 lanes hold the 128 channels of one scale.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "sm100_ptx.cuh"

namespace feather {
namespace f8 {

constexpr int kBlock = 128;        // channels per scale
constexpr int kVec = 8;            // channels per thread and step

template <bool kE5M2>
struct Code {
    static constexpr float kTop = kE5M2 ? 57344.0f : 448.0f;
    static constexpr float kLeast = static_cast<float>(1e-30 * static_cast<double>(kTop));
};

using Pairs = float2[kVec / 2];   // 8 channels

template <bool kFp16>
__device__ __forceinline__ void unpack8(const uint4& p, Pairs& v) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kFp16) {
            v[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        } else {
            v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
        }
    }
}

template <bool kFp16>
__device__ __forceinline__ uint4 pack8(const Pairs& v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kFp16) {
            const __half2 h = __float22half2_rn(v[i]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __float22bfloat162_rn(v[i]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// max(a, |b|, |c|), NaN if any of them is
__device__ __forceinline__ float max_magnitude(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
    return d;
}

__device__ __forceinline__ float max_magnitude(const Pairs& v) {
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) top = max_magnitude(top, v[i].x, v[i].y);
    return top;
}

// The largest magnitude of 8 packed 16-bit values; the comparison is exact in their own type.
template <bool kFp16>
__device__ __forceinline__ float max_magnitude_packed(const uint4& p) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
    if constexpr (kFp16) {
        __half2 top = __habs2(*reinterpret_cast<const __half2*>(&w[0]));
#pragma unroll
        for (int i = 1; i < 4; ++i) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __half2*>(&w[i])));
        return __half2float(__hmax_nan(__low2half(top), __high2half(top)));
    } else {
        __nv_bfloat162 top = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
        for (int i = 1; i < 4; ++i) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
        return __bfloat162float(__hmax_nan(__low2bfloat16(top), __high2bfloat16(top)));
    }
}

// The 16 lanes of a block agree on its maximum and turn their values into codes. Every lane of the warp takes part; lanes past
// the row's end bring zeros.
template <bool kE5M2>
__device__ __forceinline__ uint2 encode_block(const Pairs& v, float top, float& scale) {
#pragma unroll
    for (int step = 8; step > 0; step >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, top, step);
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(other));
    }
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(Code<kE5M2>::kLeast));
    const float2 inverse = both(Code<kE5M2>::kTop * __frcp_rn(top));
    scale = top * (1.0f / Code<kE5M2>::kTop);
    constexpr __nv_fp8_interpretation_t kind = kE5M2 ? __NV_E5M2 : __NV_E4M3;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __nv_cvt_float2_to_fp8x2(__fmul2_rn(v[i], inverse), __NV_SATFINITE, kind);
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// 16 bytes of an input, by a kernel that may start before the one ahead has finished writing them
__device__ __forceinline__ uint4 load16(const uint16_t* p) { return ld_global_v4(p); }

// ... by an ordinary launch
__device__ __forceinline__ uint4 load16_readonly(const uint16_t* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

}  // namespace f8
}  // namespace feather
