// The row-wise operators around the block-scaled fp8 products: the activation quantizer, RMS norm (+ residual) and
// silu(gate) * up with their outputs in 8 bits, and the backward passes of the last two.
//
// Block scales. Every 128 consecutive channels of a row share one float32 scale:
//     t = max(max |y|, 1e-30 * top),  scale = t / top,  code = fp8(y * (top / t)),  top = 448 (e4m3) or 57344 (e5m2).
// One division per block and one product per element; the floor on t keeps the inverse finite for blocks of zeros. The
// maximum is taken on the bit patterns of |y|, where a NaN is larger than any number, so a block that holds an infinity
// or a NaN gets a scale that is not finite and never reads back as ordinary numbers.
// The scales are laid out [ceil(K / 128), M]: the product's epilogue wants the scales of consecutive rows at one block.
//
// Every kernel may start while the one ahead in its stream ends (programmatic dependent launch), waits for it before it
// reads or writes memory, and lets the next one start likewise.
//
// All five kernels are bound by HBM: a thread moves 8 consecutive channels (one 16-byte load, one 8-byte store of codes),
// 16 lanes hold one block, and its maximum is four shuffles.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "feather_host.h"
#include "sm100_ptx.cuh"

namespace feather {
namespace {

constexpr int kBlock = 128;        // channels per scale
constexpr int kVec = 8;            // channels per thread and step
constexpr int kWarpChannels = 32 * kVec;
constexpr int kMaxNormThreads = 1024;
constexpr int kMaxNormChunks = 4;  // 8-channel chunks of a row per thread
constexpr int64_t kMaxNormWidth = static_cast<int64_t>(kMaxNormThreads) * kMaxNormChunks * kVec;

template <bool kE5M2>
struct Code {
    static constexpr float kTop = kE5M2 ? 57344.0f : 448.0f;
    static constexpr float kLeast = static_cast<float>(1e-30 * static_cast<double>(kTop));
};

template <bool kFp16>
__device__ __forceinline__ void unpack8(const uint4& p, float (&v)[kVec]) {
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kFp16) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

template <bool kFp16>
__device__ __forceinline__ uint4 pack8(const float (&v)[kVec]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (kFp16) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The 16 lanes of a block agree on its maximum (as the bits of |y|) and turn their values into codes. Every lane of the
// warp takes part; lanes past the row's end bring zeros.
template <bool kE5M2>
__device__ __forceinline__ uint2 encode_block(const float (&v)[kVec], float& scale) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kVec; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
    for (int step = 8; step > 0; step >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, step));
    const float t = __uint_as_float(max(top, __float_as_uint(Code<kE5M2>::kLeast)));
    const float inverse = Code<kE5M2>::kTop / t;
    scale = t / Code<kE5M2>::kTop;
    constexpr __nv_fp8_interpretation_t kind = kE5M2 ? __NV_E5M2 : __NV_E4M3;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        w[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inverse, v[2 * i + 1] * inverse), __NV_SATFINITE, kind);
    }
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// The next kernel's blocks are let in at once (they take what room is left and wait as this one does), then this one waits.
__device__ __forceinline__ void start_after_kernel_ahead() {
    grid_launch_dependents();
    grid_dependency_wait();
}

__device__ __forceinline__ uint4 load16(const uint16_t* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

// ---------------------------------------------------------------------------------------------------------
// Activation quantizer and the gate: a warp takes 256 channels of kRows rows, so a thread has kRows (or 2 * kRows)
// independent loads in flight and the scales it writes are consecutive in memory.
// ---------------------------------------------------------------------------------------------------------
constexpr int kTileWarps = 8;

template <bool kFp16, bool kE5M2, bool kGate, int kRows>
__global__ void __launch_bounds__(32 * kTileWarps) tile_quantize_kernel(const uint16_t* __restrict__ x, uint8_t* __restrict__ q,
                                                                        float* __restrict__ scale, int64_t M, int64_t K, int column_warps) {
    start_after_kernel_ahead();
    const int lane = threadIdx.x & 31;
    const int64_t task = static_cast<int64_t>(blockIdx.x) * kTileWarps + (threadIdx.x >> 5);
    const int64_t row0 = task / column_warps * kRows;
    const int64_t column = task % column_warps * kWarpChannels + lane * kVec;
    if (row0 >= M) return;
    const bool live = column < K;
    const int64_t pitch = kGate ? 2 * K : K;
    uint4 a[kRows], b[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const bool here = live && row0 + r < M;
        const uint16_t* const src = x + (row0 + r) * pitch + column;
        a[r] = here ? load16(src) : make_uint4(0, 0, 0, 0);
        if constexpr (kGate) b[r] = here ? load16(src + K) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        float v[kVec];
        unpack8<kFp16>(a[r], v);
        if constexpr (kGate) {
            float up[kVec];
            unpack8<kFp16>(b[r], up);
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[i] = v[i] * sigmoid(v[i]) * up[i];
        }
        float s;
        const uint2 codes = encode_block<kE5M2>(v, s);
        if (live && row0 + r < M) {
            *reinterpret_cast<uint2*>(q + (row0 + r) * K + column) = codes;
            if ((lane & 15) == 0) scale[column / kBlock * M + row0 + r] = s;
        }
    }
}

// d/dgate = g u s (1 + gate (1 - s)), d/dup = g gate s, with s = sigmoid(gate).
template <bool kFp16>
__global__ void __launch_bounds__(256) silu_mul_dgrad_kernel(const uint16_t* __restrict__ grad, const uint16_t* __restrict__ gate_up,
                                                             uint16_t* __restrict__ out, int64_t chunks, int64_t row_chunks) {
    start_after_kernel_ahead();
    const int64_t chunk = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (chunk >= chunks) return;
    const int64_t row = chunk / row_chunks;
    const int64_t F = row_chunks * kVec;
    const int64_t column = (chunk - row * row_chunks) * kVec;
    const int64_t at = row * 2 * F + column;
    const uint4 pg = load16(grad + row * F + column);
    const uint4 pa = load16(gate_up + at);
    const uint4 pu = load16(gate_up + at + F);
    float g[kVec], gate[kVec], up[kVec];
    unpack8<kFp16>(pg, g);
    unpack8<kFp16>(pa, gate);
    unpack8<kFp16>(pu, up);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const float s = sigmoid(gate[i]);
        const float gs = g[i] * s;
        const float d_up = gs * gate[i];
        gate[i] = gs * up[i] * (1.0f + gate[i] * (1.0f - s));
        up[i] = d_up;
    }
    *reinterpret_cast<uint4*>(out + at) = pack8<kFp16>(gate);
    *reinterpret_cast<uint4*>(out + at + F) = pack8<kFp16>(up);
}

// ---------------------------------------------------------------------------------------------------------
// RMS norm: one row per CTA, the row stays in registers (packed, it is 16-bit data) between the two passes.
// ---------------------------------------------------------------------------------------------------------
// Sum over the CTA in a fixed order, the same value in every thread. `slots` holds one float per warp; two barriers, so
// the caller may come back at once with the same slots.
__device__ __forceinline__ float block_sum(float v, float* slots) {
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    const int lane = threadIdx.x & 31;
    __syncthreads();
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? slots[lane] : 0.0f;
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
    return v;
}

template <bool kFp16, bool kWeightF32>
__device__ __forceinline__ void load_weight(const void* weight, int64_t column, float (&w)[kVec]) {
    if constexpr (kWeightF32) {
        const float4* const p = reinterpret_cast<const float4*>(static_cast<const float*>(weight) + column);
        const float4 lo = __ldg(p), hi = __ldg(p + 1);
        w[0] = lo.x, w[1] = lo.y, w[2] = lo.z, w[3] = lo.w;
        w[4] = hi.x, w[5] = hi.y, w[6] = hi.z, w[7] = hi.w;
    } else {
        unpack8<kFp16>(load16(static_cast<const uint16_t*>(weight) + column), w);
    }
}

struct NormParams {
    const uint16_t* x;
    const uint16_t* residual;  // may be null
    const void* weight;
    uint16_t* stream;          // x + residual; null without a residual
    uint8_t* q;
    float* scale;
    float* rstd;
    int64_t M, K;
    float eps;
};

template <bool kFp16, bool kWeightF32, bool kE5M2, int kChunks>
__global__ void __launch_bounds__(kMaxNormThreads) rms_norm_fp8_kernel(const NormParams p) {
    __shared__ float slots[32];
    start_after_kernel_ahead();
    const int64_t row = blockIdx.x;
    const int64_t base = row * p.K;
    const int step = blockDim.x * kVec;
    const int lane = threadIdx.x & 31;
    uint4 h[kChunks];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int64_t column = threadIdx.x * kVec + c * step;
        h[c] = column < p.K ? load16(p.x + base + column) : make_uint4(0, 0, 0, 0);
    }
    if (p.residual != nullptr) {
        uint4 r[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t column = threadIdx.x * kVec + c * step;
            r[c] = column < p.K ? load16(p.residual + base + column) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t column = threadIdx.x * kVec + c * step;
            float a[kVec], b[kVec];
            unpack8<kFp16>(h[c], a);
            unpack8<kFp16>(r[c], b);
#pragma unroll
            for (int i = 0; i < kVec; ++i) a[i] += b[i];
            h[c] = pack8<kFp16>(a);  // the stream is kept in 16 bits, and the norm is taken of what is kept
            if (column < p.K) *reinterpret_cast<uint4*>(p.stream + base + column) = h[c];
        }
    }
    float squares = 0.0f;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        float v[kVec];
        unpack8<kFp16>(h[c], v);
#pragma unroll
        for (int i = 0; i < kVec; ++i) squares = fmaf(v[i], v[i], squares);
    }
    const float rstd = rsqrtf(block_sum(squares, slots) / static_cast<float>(p.K) + p.eps);
    if (threadIdx.x == 0) p.rstd[row] = rstd;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int64_t column = threadIdx.x * kVec + c * step;
        const bool live = column < p.K;
        float v[kVec], w[kVec];
        unpack8<kFp16>(h[c], v);
        if (live) {
            load_weight<kFp16, kWeightF32>(p.weight, column, w);
#pragma unroll
            for (int i = 0; i < kVec; ++i) v[i] = v[i] * rstd * w[i];
        }
        float s;
        const uint2 codes = encode_block<kE5M2>(v, s);
        if (live) {
            *reinterpret_cast<uint2*>(p.q + base + column) = codes;
            if ((lane & 15) == 0) p.scale[column / kBlock * p.M + row] = s;
        }
    }
}

struct NormGradParams {
    const uint16_t* grad;
    const uint16_t* x;
    const void* weight;
    const float* rstd;
    const uint16_t* grad_residual;  // may be null
    uint16_t* grad_x;
    float* partials;                // [gridDim.x][K]
    int64_t M, K;
};

// n = x rstd, u = grad w:  dx = rstd (u - n mean(u n)) + grad_residual,  dw = sum over rows of grad n.
// A CTA walks rows blockIdx.x, + gridDim.x, ... and keeps its share of dw in registers, so that dw costs one row of
// partials per CTA; a second kernel adds those in CTA order (the same bits on every run).
template <bool kFp16, bool kWeightF32, int kChunks>
__global__ void __launch_bounds__(kMaxNormThreads) rms_norm_dgrad_kernel(const NormGradParams p) {
    __shared__ float slots[32];
    start_after_kernel_ahead();
    const int step = blockDim.x * kVec;
    float dw[kChunks][kVec];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int i = 0; i < kVec; ++i) dw[c][i] = 0.0f;
    }
    for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
        const int64_t base = row * p.K;
        const float rstd = __ldg(p.rstd + row);
        uint4 x[kChunks], g[kChunks], r[kChunks];
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t column = threadIdx.x * kVec + c * step;
            const bool live = column < p.K;
            x[c] = live ? load16(p.x + base + column) : make_uint4(0, 0, 0, 0);
            g[c] = live ? load16(p.grad + base + column) : make_uint4(0, 0, 0, 0);
            r[c] = live && p.grad_residual != nullptr ? load16(p.grad_residual + base + column) : make_uint4(0, 0, 0, 0);
        }
        float dot = 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t column = threadIdx.x * kVec + c * step;
            if (column < p.K) {
                float n[kVec], u[kVec], w[kVec];
                unpack8<kFp16>(x[c], n);
                unpack8<kFp16>(g[c], u);
                load_weight<kFp16, kWeightF32>(p.weight, column, w);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    n[i] *= rstd;
                    dw[c][i] = fmaf(u[i], n[i], dw[c][i]);
                    dot = fmaf(u[i] * w[i], n[i], dot);
                }
            }
        }
        const float mean = block_sum(dot, slots) / static_cast<float>(p.K);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int64_t column = threadIdx.x * kVec + c * step;
            if (column < p.K) {
                float n[kVec], u[kVec], w[kVec], res[kVec];
                unpack8<kFp16>(x[c], n);
                unpack8<kFp16>(g[c], u);
                unpack8<kFp16>(r[c], res);
                load_weight<kFp16, kWeightF32>(p.weight, column, w);
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    const float d = u[i] * w[i] - n[i] * rstd * mean;
                    u[i] = p.grad_residual != nullptr ? fmaf(d, rstd, res[i]) : d * rstd;
                }
                *reinterpret_cast<uint4*>(p.grad_x + base + column) = pack8<kFp16>(u);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int64_t column = threadIdx.x * kVec + c * step;
        if (column < p.K) {
            float4* const to = reinterpret_cast<float4*>(p.partials + blockIdx.x * p.K + column);
            to[0] = make_float4(dw[c][0], dw[c][1], dw[c][2], dw[c][3]);
            to[1] = make_float4(dw[c][4], dw[c][5], dw[c][6], dw[c][7]);
        }
    }
}

// out[k] = sum over the rows of partials, row groups first (one per warp), then the groups in order.
constexpr int kSumWarps = 8;
__global__ void __launch_bounds__(32 * kSumWarps) column_sum_kernel(const float* __restrict__ partials, float* __restrict__ out, int rows, int64_t K) {
    __shared__ float part[kSumWarps][33];
    start_after_kernel_ahead();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float sum = 0.0f;
    if (column < K) {
        for (int r = warp; r < rows; r += kSumWarps) sum += partials[r * K + column];
    }
    part[warp][lane] = sum;
    __syncthreads();
    if (warp == 0 && column < K) {
        for (int w = 1; w < kSumWarps; ++w) sum += part[w][lane];
        out[column] = sum;
    }
}

// `overlap`: may start while the kernel ahead in the stream still runs
template <class... Params, class... Args>
bool launch_kernel(void (*kernel)(Params...), int64_t grid, int threads, cudaStream_t stream, bool overlap, Args... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(grid));
    config.blockDim = dim3(static_cast<unsigned>(threads));
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = overlap ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...) == cudaSuccess;
}

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Threads and chunks per thread for one row per CTA: as few chunks as 1024 threads allow when there are few rows (a row
// is then a matter of latency), four per thread otherwise (independent loads, few threads at the barrier).
struct RowShape {
    int threads, chunks;
};

RowShape row_shape(int64_t M, int64_t K, int wanted) {
    const int64_t vectors = K / kVec;
    int chunks = M <= 2 * device_info().sm_count ? 1 : wanted;
    while (chunks > 1 && vectors < static_cast<int64_t>(chunks) * 32) chunks >>= 1;
    while ((vectors + chunks - 1) / chunks > kMaxNormThreads) chunks <<= 1;
    const int64_t threads = (vectors + chunks - 1) / chunks;
    return {static_cast<int>((threads + 31) / 32 * 32), chunks};
}

template <bool kFp16, bool kE5M2, bool kGate>
bool launch_tile(const void* x, void* q, float* scale, int64_t M, int64_t K, cudaStream_t stream, bool overlap) {
    const int64_t column_warps = (K + kWarpChannels - 1) / kWarpChannels;
    const int rows = M * column_warps > 16LL * device_info().sm_count * kTileWarps ? 4 : 1;
    const int64_t tasks = (M + rows - 1) / rows * column_warps;
    const int64_t grid = (tasks + kTileWarps - 1) / kTileWarps;
    if (column_warps > 0x7fffffff || grid > 0x7fffffff) return false;
    const auto kernel = rows == 4 ? tile_quantize_kernel<kFp16, kE5M2, kGate, 4> : tile_quantize_kernel<kFp16, kE5M2, kGate, 1>;
    return launch_kernel(kernel, grid, 32 * kTileWarps, stream, overlap, static_cast<const uint16_t*>(x), static_cast<uint8_t*>(q), scale, M, K,
                         static_cast<int>(column_warps));
}

template <bool kGate>
bool dispatch_tile(const void* x, void* q, float* scale, int64_t M, int64_t K, bool fp16, bool e5m2, cudaStream_t stream, bool overlap = true) {
    if (M < 0 || K <= 0 || K % 16 != 0) return false;
    if (M == 0) return true;
    if (x == nullptr || q == nullptr || scale == nullptr || !aligned(x, 16) || !aligned(q, 16) || !aligned(scale, 4)) return false;
    if (fp16) return e5m2 ? launch_tile<true, true, kGate>(x, q, scale, M, K, stream, overlap) : launch_tile<true, false, kGate>(x, q, scale, M, K, stream, overlap);
    return e5m2 ? launch_tile<false, true, kGate>(x, q, scale, M, K, stream, overlap) : launch_tile<false, false, kGate>(x, q, scale, M, K, stream, overlap);
}

template <bool kFp16, bool kWeightF32, bool kE5M2>
bool launch_norm(const NormParams& p, cudaStream_t stream) {
    const RowShape shape = row_shape(p.M, p.K, 4);
    const auto kernel = shape.chunks == 1   ? rms_norm_fp8_kernel<kFp16, kWeightF32, kE5M2, 1>
                        : shape.chunks == 2 ? rms_norm_fp8_kernel<kFp16, kWeightF32, kE5M2, 2>
                                            : rms_norm_fp8_kernel<kFp16, kWeightF32, kE5M2, 4>;
    return launch_kernel(kernel, p.M, shape.threads, stream, true, p);
}

template <bool kFp16, bool kWeightF32>
bool launch_norm_grad(const NormGradParams& p, int grid, cudaStream_t stream) {
    const RowShape shape = row_shape(p.M, p.K, 2);
    const auto kernel = shape.chunks == 1   ? rms_norm_dgrad_kernel<kFp16, kWeightF32, 1>
                        : shape.chunks == 2 ? rms_norm_dgrad_kernel<kFp16, kWeightF32, 2>
                                            : rms_norm_dgrad_kernel<kFp16, kWeightF32, 4>;
    return launch_kernel(kernel, grid, shape.threads, stream, true, p);
}

// CTAs of the norm's backward pass: at most two per SM of a B200 (their registers hold two), at least four rows each. A
// constant and not the device's count, so that the size of the scratch and the order of the sums do not depend on the device.
constexpr int64_t kNormGradCtas = 296;
int norm_grad_grid(int64_t M) {
    const int64_t wanted = (M + 3) / 4;
    return static_cast<int>(wanted < kNormGradCtas ? wanted : kNormGradCtas);
}

}  // namespace

bool launch_fp8_block_quantize_ahead(const void* x, void* q, float* scale, int64_t M, int64_t K, int input_fp16, int use_e5m2, cudaStream_t stream) {
    return dispatch_tile<false>(x, q, scale, M, K, input_fp16 != 0, use_e5m2 != 0, stream, false);
}

}  // namespace feather

using namespace feather;

extern "C" bool launch_fp8_block_quantize(const void* x, void* q, float* scale, int64_t M, int64_t K, int input_fp16, int use_e5m2,
                                          cudaStream_t stream) {
    return dispatch_tile<false>(x, q, scale, M, K, input_fp16 != 0, use_e5m2 != 0, stream);
}

extern "C" bool launch_silu_mul_fp8(const void* gate_up, void* q, float* scale, int64_t M, int64_t F, int input_fp16, int use_e5m2,
                                    cudaStream_t stream) {
    return dispatch_tile<true>(gate_up, q, scale, M, F, input_fp16 != 0, use_e5m2 != 0, stream);
}

extern "C" bool launch_silu_mul_dgrad(const void* grad, const void* gate_up, void* grad_gate_up, int64_t M, int64_t F, int input_fp16,
                                      cudaStream_t stream) {
    if (M < 0 || F <= 0 || F % 16 != 0) return false;
    if (M == 0) return true;
    if (grad == nullptr || gate_up == nullptr || grad_gate_up == nullptr) return false;
    if (!aligned(grad, 16) || !aligned(gate_up, 16) || !aligned(grad_gate_up, 16)) return false;
    const int64_t row_chunks = F / kVec;
    const int64_t chunks = M * row_chunks;
    const int64_t grid = (chunks + 255) / 256;
    if (grid > 0x7fffffff) return false;
    const auto kernel = input_fp16 != 0 ? silu_mul_dgrad_kernel<true> : silu_mul_dgrad_kernel<false>;
    return launch_kernel(kernel, grid, 256, stream, true, static_cast<const uint16_t*>(grad), static_cast<const uint16_t*>(gate_up),
                         static_cast<uint16_t*>(grad_gate_up), chunks, row_chunks);
}

extern "C" bool launch_rms_norm_fp8(const void* x, const void* residual, const void* weight, void* residual_out, void* q, float* scale, float* rstd,
                                    int64_t M, int64_t K, float eps, int input_fp16, int weight_f32, int use_e5m2, cudaStream_t stream) {
    if (M < 0 || M > 0x7fffffff || K <= 0 || K % 16 != 0 || K > kMaxNormWidth) return false;
    if (M == 0) return true;
    if (x == nullptr || weight == nullptr || q == nullptr || scale == nullptr || rstd == nullptr || (residual == nullptr) != (residual_out == nullptr)) return false;
    if (!aligned(x, 16) || !aligned(residual, 16) || !aligned(weight, 16) || !aligned(residual_out, 16) || !aligned(q, 16)) return false;
    const NormParams p{static_cast<const uint16_t*>(x), static_cast<const uint16_t*>(residual), weight, static_cast<uint16_t*>(residual_out),
                       static_cast<uint8_t*>(q), scale, rstd, M, K, eps};
    
    switch ((input_fp16 != 0 ? 4 : 0) | (weight_f32 != 0 ? 2 : 0) | (use_e5m2 != 0 ? 1 : 0)) {
        case 0: return launch_norm<false, false, false>(p, stream);
        case 1: return launch_norm<false, false, true>(p, stream);
        case 2: return launch_norm<false, true, false>(p, stream);
        case 3: return launch_norm<false, true, true>(p, stream);
        case 4: return launch_norm<true, false, false>(p, stream);
        case 5: return launch_norm<true, false, true>(p, stream);
        case 6: return launch_norm<true, true, false>(p, stream);
        default: return launch_norm<true, true, true>(p, stream);
    }
}

extern "C" int64_t feather_rms_norm_dgrad_partial_floats(int64_t M, int64_t K) {
    return M <= 0 || K <= 0 ? 0 : norm_grad_grid(M) * K;
}

extern "C" bool launch_rms_norm_dgrad(const void* grad, const void* x, const void* weight, const float* rstd, const void* grad_residual, void* grad_x,
                                      float* grad_weight, float* partials, int64_t M, int64_t K, int input_fp16, int weight_f32, cudaStream_t stream) {
    if (M <= 0 || M > 0x7fffffff || K <= 0 || K % 16 != 0 || K > kMaxNormWidth) return false;
    if (grad == nullptr || x == nullptr || weight == nullptr || rstd == nullptr || grad_x == nullptr || grad_weight == nullptr || partials == nullptr) return false;
    if (!aligned(grad, 16) || !aligned(x, 16) || !aligned(weight, 16) || !aligned(grad_residual, 16) || !aligned(grad_x, 16) || !aligned(partials, 16)) return false;
    const NormGradParams p{static_cast<const uint16_t*>(grad), static_cast<const uint16_t*>(x), weight, rstd, static_cast<const uint16_t*>(grad_residual),
                           static_cast<uint16_t*>(grad_x), partials, M, K};
    
    const int grid = norm_grad_grid(M);
    bool ok;
    if (input_fp16 != 0) {
        ok = weight_f32 != 0 ? launch_norm_grad<true, true>(p, grid, stream) : launch_norm_grad<true, false>(p, grid, stream);
    } else {
        ok = weight_f32 != 0 ? launch_norm_grad<false, true>(p, grid, stream) : launch_norm_grad<false, false>(p, grid, stream);
    }
    if (!ok) return false;
    return launch_kernel(column_sum_kernel, (K + 31) / 32, 32 * kSumWarps, stream, true, static_cast<const float*>(partials), grad_weight, grid, K);
}
