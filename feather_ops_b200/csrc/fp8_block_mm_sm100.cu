// Block-scaled fp8 x fp8 product: activation codes with one float32 scale per row and 128 channels, weight codes with one
// per 128 x 128 block.
//   forward   C[m, n] = sum_b sa[b, m] sw[n / 128, b] (A[m, block b] . W[n, block b]) + bias[n]
//   backward  C[m, k] = sum_b sa[b, m] sw[b, k / 128] (A[m, block b] . W[block b, k])
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "feather_host.h"

namespace feather {
namespace {

constexpr int kBlock = 128;

struct Args {
    const uint8_t* a;
    const float* a_scale;
    const uint8_t* w;
    const float* w_scale;
    const uint16_t* bias;
    uint16_t* c;
    int64_t M, N, K;  // N and K: the weight's axes
    bool transposed_b, a_e5m2, w_e5m2, out_bf16;
};

__device__ __forceinline__ float decode(uint8_t v, bool e5m2) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, e5m2 ? __NV_E5M2 : __NV_E4M3)));
}

// 64 x 64 outputs per CTA, 4 x 4 per thread, on the CUDA cores.
__global__ void __launch_bounds__(256) simple_kernel(const Args p) {
    __shared__ float sa[32][65], sw[32][65];
    const int64_t width = p.transposed_b ? p.K : p.N;
    const int64_t depth = p.transposed_b ? p.N : p.K;
    const int64_t scale_pitch = (p.K + kBlock - 1) / kBlock;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * 64, n0 = static_cast<int64_t>(blockIdx.x) * 64;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float total[4][4] = {};
    for (int64_t b = 0; b * kBlock < depth; ++b) {
        float part[4][4] = {};
        for (int64_t d0 = b * kBlock; d0 < depth && d0 < (b + 1) * kBlock; d0 += 32) {
            __syncthreads();
            for (int i = threadIdx.x; i < 64 * 32; i += 256) {
                const int64_t m = m0 + i / 32, d = d0 + i % 32;
                sa[i % 32][i / 32] = m < p.M && d < depth ? decode(p.a[m * depth + d], p.a_e5m2) : 0.0f;
                const int64_t n = n0 + (p.transposed_b ? i % 64 : i / 32), dw = d0 + (p.transposed_b ? i / 64 : i % 32);
                const bool live = n < width && dw < depth;
                const float v = live ? decode(p.transposed_b ? p.w[dw * p.K + n] : p.w[n * p.K + dw], p.w_e5m2) : 0.0f;
                sw[dw - d0][n - n0] = v;
            }
            __syncthreads();
            for (int d = 0; d < 32; ++d) {
                for (int i = 0; i < 4; ++i) {
                    for (int j = 0; j < 4; ++j) part[i][j] = fmaf(sa[d][ty * 4 + i], sw[d][tx * 4 + j], part[i][j]);
                }
            }
        }
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + ty * 4 + i;
            for (int j = 0; j < 4; ++j) {
                const int64_t n = n0 + tx * 4 + j;
                if (m < p.M && n < width) {
                    const float s = p.w_scale[p.transposed_b ? b * scale_pitch + n / kBlock : n / kBlock * scale_pitch + b];
                    total[i][j] = fmaf(part[i][j], p.a_scale[b * p.M + m] * s, total[i][j]);
                }
            }
        }
    }
    for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty * 4 + i;
        for (int j = 0; j < 4; ++j) {
            const int64_t n = n0 + tx * 4 + j;
            if (m >= p.M || n >= width) continue;
            float v = total[i][j];
            if (p.bias != nullptr) {
                v += p.out_bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.bias)[n]) : __half2float(reinterpret_cast<const __half*>(p.bias)[n]);
            }
            if (p.out_bf16) {
                reinterpret_cast<__nv_bfloat16*>(p.c)[m * width + n] = __float2bfloat16_rn(v);
            } else {
                reinterpret_cast<__half*>(p.c)[m * width + n] = __float2half_rn(v);
            }
        }
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace feather

using namespace feather;

extern "C" bool launch_fp8_block_mm(const uint8_t* a, const float* a_scale, const uint8_t* w, const float* w_scale, const uint16_t* bias, uint16_t* c,
                                    int64_t M, int64_t N, int64_t K, bool transposed_b, int a_e5m2, int w_e5m2, int output_dtype,
                                    cudaStream_t stream) {
    constexpr int64_t kMost = 0x7fffffff - 256;
    if (M < 0 || N <= 0 || K <= 0 || M > kMost || N > kMost || K > kMost || N % 16 != 0 || K % 16 != 0) return false;
    if (transposed_b && bias != nullptr) return false;
    if (output_dtype != 0 && output_dtype != 1) return false;
    if (M == 0) return true;
    if (a == nullptr || a_scale == nullptr || w == nullptr || w_scale == nullptr || c == nullptr) return false;
    if (!aligned16(a) || !aligned16(w) || !aligned16(c)) return false;
    const Args args{a, a_scale, w, w_scale, bias, c, M, N, K, transposed_b, a_e5m2 != 0, w_e5m2 != 0, output_dtype == 1};
    const int64_t width = transposed_b ? K : N;
    if ((M + 63) / 64 > 65535) return false;
    simple_kernel<<<dim3(static_cast<unsigned>((width + 63) / 64), static_cast<unsigned>((M + 63) / 64)), 256, 0, stream>>>(args);
    return cudaGetLastError() == cudaSuccess;
}
