// The row-wise operators around the block-scaled fp8 products: the activation quantizer, RMS norm (+ residual) and
// silu(gate) * up with their outputs in 8 bits, and the backward passes of the last two.
//
// Block scales. Every 128 consecutive channels of a row share one float32 scale:
//     t = max(max |y|, 1e-30 * top),  scale = t * (1 / top),  code = fp8(y * (top * (1 / t))),  top = 448 (e4m3) or 57344 (e5m2).
// One reciprocal per block and one product per element; the floor on t keeps the inverse finite for blocks of zeros. The maximum
// keeps NaN, so a block that holds an infinity or a NaN never reads back as ordinary numbers.
// The scales are laid out [ceil(K / 128), M]: the product wants the scales of consecutive rows at one block.
//
// Every kernel but the norm's backward pass may start while the one ahead in its stream ends (programmatic dependent launch),
// waits for it before it reads or writes memory, and lets the next one start likewise.
//
// All kernels move a few bytes per element through HBM, so few instructions per element are left: at 6.5 TB/s an SM gets 4 to 13
// elements per clock and issues 4 warp instructions, i.e. 10 to 30 instructions per element. A thread has 8 consecutive channels
// (one 16-byte load, one 8-byte store of codes) as four float pairs for the packed fp32 arithmetic; 16 lanes hold one block, and
// its maximum is four shuffles. Measured, inputs from HBM: quantizer 8192 x 4096 16.6 us (6.1 TB/s of 6.46 that a copy reaches), gate
// 4096 x 12288 41 to 44 (5.7 to 6.1), norm 8192 x 4096 with a residual 37.7 to 38.5 (6.2), its backward pass 50.3 (5.3). The gate's backward pass takes 72
// at 4096 x 12288, which for its 503 MB is above a copy's rate: a quarter of what it writes is still in L2 when it ends.
#include <cuda_runtime.h>

#include <cstdint>

#include "feather_host.h"
#include "fp8_block.cuh"
#include "sm100_ptx.cuh"

namespace feather {
namespace {

using namespace f8;

constexpr int kWarpChannels = 32 * kVec;
constexpr int kMaxNormThreads = 1024;
constexpr int kMaxNormChunks = 4;  // 8-channel chunks of a row per thread
constexpr int64_t kMaxNormWidth = static_cast<int64_t>(kMaxNormThreads) * kMaxNormChunks * kVec;

// The next kernel's blocks are let in at once (they take what room is left and wait as this one does), then this one waits.
__device__ __forceinline__ void start_after_kernel_ahead() {
    grid_launch_dependents();
    grid_dependency_wait();
}

// 1 / (1 + exp(-x)), each of the two special functions once
__device__ __forceinline__ float2 sigmoid(float2 x) {
    const float2 e = __fmul2_rn(x, both(-1.44269504f));   // -log2(e) x
    float2 d;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d.x) : "f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(d.y) : "f"(e.y));
    d = __fadd2_rn(d, both(1.0f));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.y));
    return d;
}

// ---------------------------------------------------------------------------------------------------------
// Activation quantizer and the gate: a warp takes 256 channels of kRows rows, so a thread has kRows (or 2 * kRows)
// independent loads in flight and the scales it writes are consecutive in memory.
// ---------------------------------------------------------------------------------------------------------
constexpr int kTileWarps = 8;

template <bool kFp16, bool kE5M2, bool kGate, int kRows>
__global__ void __launch_bounds__(32 * kTileWarps) tile_quantize_kernel(const uint16_t* x, uint8_t* q,
                                                                        float* scale, int64_t M, int64_t K, int column_warps) {
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
        Pairs v;
        unpack8<kFp16>(a[r], v);
        float s;
        uint2 codes;
        if constexpr (kGate) {
            Pairs up;
            unpack8<kFp16>(b[r], up);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __fmul2_rn(__fmul2_rn(v[i], sigmoid(v[i])), up[i]);
            codes = encode_block<kE5M2>(v, max_magnitude(v), s);
        } else {
            codes = encode_block<kE5M2>(v, max_magnitude_packed<kFp16>(a[r]), s);
        }
        if (live && row0 + r < M) {
            *reinterpret_cast<uint2*>(q + (row0 + r) * K + column) = codes;
            if ((lane & 15) == 0) scale[column / kBlock * M + row0 + r] = s;
        }
    }
}

// d/dgate = g u s (1 + gate (1 - s)), d/dup = g gate s, with s = sigmoid(gate).
template <bool kFp16>
__global__ void __launch_bounds__(256) silu_mul_dgrad_kernel(const uint16_t* grad, const uint16_t* gate_up,
                                                             uint16_t* out, int64_t chunks, int64_t row_chunks) {
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
    Pairs g, gate, up;
    unpack8<kFp16>(pg, g);
    unpack8<kFp16>(pa, gate);
    unpack8<kFp16>(pu, up);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 s = sigmoid(gate[i]);
        const float2 gs = __fmul2_rn(g[i], s);
        const float2 d_up = __fmul2_rn(gs, gate[i]);
        const float2 rest = __ffma2_rn(s, both(-1.0f), both(1.0f));   // 1 - s
        gate[i] = __fmul2_rn(__fmul2_rn(gs, up[i]), __ffma2_rn(gate[i], rest, both(1.0f)));
        up[i] = d_up;
    }
    *reinterpret_cast<uint4*>(out + at) = pack8<kFp16>(gate);
    *reinterpret_cast<uint4*>(out + at + F) = pack8<kFp16>(up);
}

// ---------------------------------------------------------------------------------------------------------
// RMS norm. A row belongs to blockDim.x threads: one warp up to 1024 channels (blockDim.y rows per CTA, no barrier), else
// the whole CTA. Between the two passes it stays in registers, packed (it is 16-bit data).
// ---------------------------------------------------------------------------------------------------------
constexpr int kWarpRowWidth = 1024;   // a row of at most this many channels is one warp's
constexpr int kRowsPerCta = 8;        // ... with so many of them in a CTA

// Sum over the row's threads in a fixed order, the same value in every thread. `slots`: 32 floats that nobody else uses until the
// next barrier after this call's.
__device__ __forceinline__ float row_sum(float v, float* slots) {
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    const int lane = threadIdx.x & 31;
    if (lane == 0) slots[threadIdx.x >> 5] = v;
    __syncthreads();
    v = lane < warps ? slots[lane] : 0.0f;
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) v += __shfl_xor_sync(0xffffffffu, v, step);
    return v;
}

// kReadonly: by an ordinary launch (see load16_readonly)
template <bool kFp16, bool kWeightF32, bool kReadonly>
__device__ __forceinline__ void load_weight(const void* weight, int64_t column, Pairs& w) {
    const auto load = [](const uint16_t* p) { return kReadonly ? load16_readonly(p) : load16(p); };
    if constexpr (kWeightF32) {
        const uint16_t* const p = reinterpret_cast<const uint16_t*>(static_cast<const float*>(weight) + column);
        const uint4 lo = load(p), hi = load(p + 8);
        w[0] = make_float2(__uint_as_float(lo.x), __uint_as_float(lo.y)), w[1] = make_float2(__uint_as_float(lo.z), __uint_as_float(lo.w));
        w[2] = make_float2(__uint_as_float(hi.x), __uint_as_float(hi.y)), w[3] = make_float2(__uint_as_float(hi.z), __uint_as_float(hi.w));
    } else {
        unpack8<kFp16>(load(static_cast<const uint16_t*>(weight) + column), w);
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

// kRows rows at a time, so that without a residual there are as many loads in flight as with one.
template <bool kFp16, bool kWeightF32, bool kE5M2, int kChunks, int kRows>
__global__ void __launch_bounds__(kMaxNormThreads) rms_norm_fp8_kernel(const NormParams p) {
    __shared__ float slots[kRows * 32];
    start_after_kernel_ahead();
    const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y) * kRows;
    if (row0 >= p.M) return;   // a whole warp, and with more than one warp per row the whole CTA
    const int column0 = threadIdx.x * kVec;
    const int step = blockDim.x * kVec;
    const int width = static_cast<int>(p.K);
    uint4 h[kRows][kChunks];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const bool live = column0 + c * step < width && row0 + r < p.M;
            h[r][c] = live ? load16(p.x + (row0 + r) * p.K + column0 + c * step) : make_uint4(0, 0, 0, 0);
        }
    }
    if (p.residual != nullptr) {
        uint4 add[kRows][kChunks];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const bool live = column0 + c * step < width && row0 + r < p.M;
                add[r][c] = live ? load16(p.residual + (row0 + r) * p.K + column0 + c * step) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                Pairs a, b;
                unpack8<kFp16>(h[r][c], a);
                unpack8<kFp16>(add[r][c], b);
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = __fadd2_rn(a[i], b[i]);
                h[r][c] = pack8<kFp16>(a);  // the stream is kept in 16 bits, and the norm is taken of what is kept
                if (column0 + c * step < width && row0 + r < p.M) *reinterpret_cast<uint4*>(p.stream + (row0 + r) * p.K + column0 + c * step) = h[r][c];
            }
        }
    }
    float sum[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        float2 squares = both(0.0f);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            Pairs v;
            unpack8<kFp16>(h[r][c], v);
#pragma unroll
            for (int i = 0; i < 4; ++i) squares = __ffma2_rn(v[i], v[i], squares);
        }
        sum[r] = squares.x + squares.y;
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) sum[r] = row_sum(sum[r], slots + r * 32);
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        sum[r] = rsqrtf(sum[r] / static_cast<float>(width) + p.eps);
        if (threadIdx.x == 0 && row0 + r < p.M) p.rstd[row0 + r] = sum[r];
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int column = column0 + c * step;
        const bool live = column < width;
        Pairs w = {};
        if (live) load_weight<kFp16, kWeightF32, false>(p.weight, column, w);
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            Pairs v;
            unpack8<kFp16>(h[r][c], v);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __fmul2_rn(__fmul2_rn(v[i], both(sum[r])), w[i]);
            float s;
            const uint2 codes = encode_block<kE5M2>(v, max_magnitude(v), s);
            if (live && row0 + r < p.M) {
                *reinterpret_cast<uint2*>(p.q + (row0 + r) * p.K + column) = codes;
                if ((threadIdx.x & 15) == 0) p.scale[column / kBlock * p.M + row0 + r] = s;
            }
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
// A persistent grid: every CTA walks its rows and keeps its share of dw in registers, so that dw costs one row of partials per
// CTA; a second kernel adds those in CTA order (the same bits on every run). A row is a chain of latencies (loads, ten shuffles, a
// barrier), so what counts is how many rows an SM has on their way: two per CTA with the next row in registers (kAhead), else, at 64 registers, four CTAs
// of 256 threads. (Copying the next rows to shared memory ahead of time was slower at the two or three CTAs that fit then: 68 to 75 us at
// 8192 x 4096 with a residual, and so was every variant whose registers spill there.) Above 16384 channels 1024 threads have four chunks each and the registers do
// spill (460 bytes stored and 400 loaded a thread, 924 and 864 with a float32 weight): 4096 x 32768 with a residual 352 us and 522 to 608, where the bytes take 166;
// 4096 x 16384 106 and 110 (83).
template <bool kFp16, bool kWeightF32, int kChunks, int kThreads, bool kAhead>
__global__ void __launch_bounds__(kThreads) rms_norm_dgrad_kernel(const NormGradParams p) {
    __shared__ float slots[2][32];
    extern __shared__ float total[];   // the width, with several rows per CTA
    const int column0 = threadIdx.x * kVec;
    const int step = blockDim.x * kVec;
    const int width = static_cast<int>(p.K);
    const int64_t row_step = static_cast<int64_t>(gridDim.x) * blockDim.y;
    float2 dw[kChunks][4];
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) dw[c][i] = both(0.0f);
    }
    bool odd = false;
    struct Row {
        uint4 x[kChunks], g[kChunks], res[kChunks];
        float rstd;
    };
    const auto load = [&](int64_t row, Row& r) {
        const bool live = row < p.M;
        const int64_t base = row * p.K;
        r.rstd = live ? __ldg(p.rstd + row) : 0.0f;
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int column = column0 + c * step;
            r.x[c] = r.g[c] = r.res[c] = make_uint4(0, 0, 0, 0);
            if (live && column < width) {
                r.x[c] = load16_readonly(p.x + base + column);
                r.g[c] = load16_readonly(p.grad + base + column);
                if (p.grad_residual != nullptr) r.res[c] = load16_readonly(p.grad_residual + base + column);
            }
        }
    };
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    Row ahead;
    if constexpr (kAhead) load(row0, ahead);
    for (int64_t row = row0; row < p.M; row += row_step) {
        Row now;
        if constexpr (kAhead) {
            now = ahead;
            load(row + row_step, ahead);
        } else {
            load(row, now);
        }
        const int64_t base = row * p.K;
        const float rstd = now.rstd;
        const uint4(&x)[kChunks] = now.x;
        const uint4(&g)[kChunks] = now.g;
        const uint4(&res)[kChunks] = now.res;
        float2 dots = both(0.0f);
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int column = column0 + c * step;
            if (column < width) {
                Pairs n, u, w;
                unpack8<kFp16>(x[c], n);
                unpack8<kFp16>(g[c], u);
                load_weight<kFp16, kWeightF32, true>(p.weight, column, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    n[i] = __fmul2_rn(n[i], both(rstd));
                    dw[c][i] = __ffma2_rn(u[i], n[i], dw[c][i]);
                    dots = __ffma2_rn(__fmul2_rn(u[i], w[i]), n[i], dots);
                }
            }
        }
        const float dot = row_sum(dots.x + dots.y, slots[odd ? 1 : 0]);   // two sets of slots: a thread may still read the other one
        odd = !odd;
        const float2 back = both(-rstd * rstd * (dot / static_cast<float>(width)));
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const int column = column0 + c * step;
            if (column < width) {
                Pairs n, u, w, r;
                unpack8<kFp16>(x[c], n);
                unpack8<kFp16>(g[c], u);
                unpack8<kFp16>(res[c], r);
                load_weight<kFp16, kWeightF32, true>(p.weight, column, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = __ffma2_rn(n[i], back, __ffma2_rn(__fmul2_rn(u[i], w[i]), both(rstd), r[i]));
                *reinterpret_cast<uint4*>(p.grad_x + base + column) = pack8<kFp16>(r);
            }
        }
    }
    grid_launch_dependents();
    if (blockDim.y > 1) {
        // the CTA's rows first: one warp after the other adds its share in shared memory
        for (int y = 0; y < static_cast<int>(blockDim.y); ++y) {
            __syncthreads();
            if (static_cast<int>(threadIdx.y) == y) {
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int column = column0 + c * step;
                    if (column < width) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float2* const sum = reinterpret_cast<float2*>(total + column) + i;
                            if (y > 0) dw[c][i] = __fadd2_rn(dw[c][i], *sum);
                            *sum = dw[c][i];
                        }
                    }
                }
            }
        }
        if (threadIdx.y + 1 != blockDim.y) return;
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        const int column = column0 + c * step;
        if (column < width) {
            float4* const to = reinterpret_cast<float4*>(p.partials + blockIdx.x * p.K + column);
            to[0] = make_float4(dw[c][0].x, dw[c][0].y, dw[c][1].x, dw[c][1].y);
            to[1] = make_float4(dw[c][2].x, dw[c][2].y, dw[c][3].x, dw[c][3].y);
        }
    }
}

// The same for few rows, in one launch and without partials: `rstd` is given, so dw needs nothing of a row but its values. The first M
// CTAs have a row each and write dx, the others 64 channels each and add grad n over the rows: 8 threads abreast, blockDim.x / 8 rows at a
// time, then the lanes and the warps in order. The inputs are read twice, the second time from L2. At 333 x 2576 a call costs the host
// 8 us instead of 11.5, and the device less too.
constexpr int kFewRows = 1024;
constexpr int kFewNarrowRows = 512;                 // with less than 512 channels there are too few of the channels' CTAs
constexpr int kFewWidth = kMaxNormThreads * kVec;   // one chunk per thread
constexpr int kFewThreads = 512;                    // at least, for the channels' CTAs (1000 x 1024: 7.5 us, 9.8 with 256, 10.3 with 1024)
constexpr int kColumnTile = 64;

template <bool kFp16, bool kWeightF32>
__global__ void __launch_bounds__(kMaxNormThreads) rms_norm_dgrad_few_kernel(const NormGradParams p, float* grad_weight) {
    __shared__ float slots[32];
    __shared__ float2 sums[32][kColumnTile / 2];
    start_after_kernel_ahead();
    const int width = static_cast<int>(p.K);
    const int rows = static_cast<int>(p.M);
    if (static_cast<int>(blockIdx.x) < rows) {
        const int64_t row = blockIdx.x;
        const int column = threadIdx.x * kVec;
        const bool live = column < width;
        const float rstd = ld_global_f32(p.rstd + row);
        Pairs n = {}, u = {}, r = {};
        float2 dots = both(0.0f);
        if (live) {
            Pairs w;
            unpack8<kFp16>(load16(p.x + row * p.K + column), n);
            unpack8<kFp16>(load16(p.grad + row * p.K + column), u);
            if (p.grad_residual != nullptr) unpack8<kFp16>(load16(p.grad_residual + row * p.K + column), r);
            load_weight<kFp16, kWeightF32, false>(p.weight, column, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                n[i] = __fmul2_rn(n[i], both(rstd));
                u[i] = __fmul2_rn(u[i], w[i]);
                dots = __ffma2_rn(u[i], n[i], dots);
            }
        }
        const float2 back = both(-rstd * (row_sum(dots.x + dots.y, slots) / static_cast<float>(width)));
        if (live) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = __ffma2_rn(n[i], back, __ffma2_rn(u[i], both(rstd), r[i]));
            *reinterpret_cast<uint4*>(p.grad_x + row * p.K + column) = pack8<kFp16>(r);
        }
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int column = (blockIdx.x - rows) * kColumnTile + lane % 8 * kVec;
    Pairs sum = {};
    if (column < width) {
#pragma unroll 4
        for (int row = threadIdx.x / 8; row < rows; row += blockDim.x / 8) {
            Pairs n, g;
            unpack8<kFp16>(load16(p.x + static_cast<int64_t>(row) * p.K + column), n);
            unpack8<kFp16>(load16(p.grad + static_cast<int64_t>(row) * p.K + column), g);
            const float2 rstd = both(ld_global_f32(p.rstd + row));
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = __ffma2_rn(g[i], __fmul2_rn(n[i], rstd), sum[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int step = 8; step < 32; step <<= 1) {
            sum[i].x += __shfl_xor_sync(0xffffffffu, sum[i].x, step);
            sum[i].y += __shfl_xor_sync(0xffffffffu, sum[i].y, step);
        }
        if (lane < 8) sums[warp][lane * 4 + i] = sum[i];
    }
    __syncthreads();
    const int pair = threadIdx.x;
    const int first = (blockIdx.x - rows) * kColumnTile + 2 * pair;
    if (pair < kColumnTile / 2 && first < width) {
        float2 total = sums[0][pair];
        for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) total = __fadd2_rn(total, sums[w][pair]);
        *reinterpret_cast<float2*>(grad_weight + first) = total;
    }
}

// out[k] = sum over the rows of partials, row groups first (one per warp), then the groups in order.
constexpr int kSumWarps = 8;
__global__ void __launch_bounds__(32 * kSumWarps) column_sum_kernel(const float* partials, float* out, int rows, int64_t K) {
    __shared__ float part[kSumWarps][33];
    grid_dependency_wait();   // launched behind the kernel that writes the partials, as its dependent
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    float sum = 0.0f;
    if (column < K) {
#pragma unroll 8
        for (int r = warp; r < rows; r += kSumWarps) sum += ld_global_f32(partials + r * K + column);
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
bool launch_kernel(void (*kernel)(Params...), int64_t grid, dim3 block, size_t smem, cudaStream_t stream, bool overlap, Args... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(grid));
    config.blockDim = block;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = overlap ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...) == cudaSuccess;
}

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// The threads of a row and the 8-channel chunks that each of them has. One warp up to 1024 channels; beyond, two chunks per
// thread, one where there are few rows (a row is then a matter of latency), and four where 1024 threads need them. The numbers
// come from the sizes alone, and with them the order of the sums.
struct RowShape {
    int threads, rows, chunks;   // blockDim.x, blockDim.y
};

constexpr int kSms = 148;   // of a B200: a constant, since the scratch's size is asked for without a device too

RowShape row_shape(int64_t M, int64_t K) {
    const int64_t vectors = K / kVec;
    const bool few = M <= 2 * kSms;
    if (K <= kWarpRowWidth && !few) return {32, kRowsPerCta, vectors <= 32 ? 1 : vectors <= 64 ? 2 : 4};
    int chunks = few ? 1 : 2;
    while ((vectors + chunks - 1) / chunks > kMaxNormThreads) chunks <<= 1;
    const int64_t threads = (vectors + chunks - 1) / chunks;
    return {static_cast<int>((threads + 31) / 32 * 32), 1, chunks};
}

// The norm's backward pass has a row's successor on its way in registers (128 a thread, so 512 threads on an SM) where a row is a CTA's and those
// CTAs leave no more than a quarter of the 512 threads unused. Measured (us, with a residual; without the next row): 20000 x 1280 46.0 (69.5), 8192 x
// 2048 30.2 (38.6), 8192 x 4096 50.4 (52.9), 4096 x 6144 43.3 (46.7), 4096 x 8192 50.3 (54.5); 8192 x 5120, 320 threads, 73.0 (64.8); rows of a warp 20000 x 1024
// 40.4 (37.3), 20000 x 256 15.6 (14.7).
constexpr int kAheadThreads = 512;

bool next_row_ahead(const RowShape& shape) {
    return shape.rows == 1 && shape.chunks == 2 && shape.threads <= kAheadThreads && kAheadThreads / shape.threads * shape.threads >= kAheadThreads / 4 * 3;
}

// CTAs of the norm's backward pass: what an SM holds (without the next row: at 64 registers a thread, twice that with four chunks per warp; four at
// most), and two rows each at least.
int norm_grad_grid(int64_t M, const RowShape& shape) {
    int64_t per_sm = (next_row_ahead(shape) ? kAheadThreads : 1024) / (shape.threads * shape.rows);
    if (!next_row_ahead(shape) && per_sm > 4) per_sm = 4;
    if (per_sm < 1) per_sm = 1;
    if (shape.rows > 1 && shape.chunks == 4) per_sm = 2;
    const int64_t wanted = (M + 2 * shape.rows - 1) / (2 * shape.rows);
    return static_cast<int>(wanted < kSms * per_sm ? wanted : kSms * per_sm);
}

template <bool kFp16, bool kE5M2, bool kGate>
bool launch_tile(const void* x, void* q, float* scale, int64_t M, int64_t K, cudaStream_t stream, bool overlap) {
    const int64_t column_warps = (K + kWarpChannels - 1) / kWarpChannels;
    const int rows = M * column_warps > 16LL * device_info().sm_count * kTileWarps ? 4 : 1;
    const int64_t tasks = (M + rows - 1) / rows * column_warps;
    const int64_t grid = (tasks + kTileWarps - 1) / kTileWarps;
    if (column_warps > 0x7fffffff || grid > 0x7fffffff) return false;
    const auto kernel = rows == 4 ? tile_quantize_kernel<kFp16, kE5M2, kGate, 4> : tile_quantize_kernel<kFp16, kE5M2, kGate, 1>;
    return launch_kernel(kernel, grid, dim3(32 * kTileWarps), 0, stream, overlap, static_cast<const uint16_t*>(x), static_cast<uint8_t*>(q), scale, M, K,
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
    const RowShape shape = row_shape(p.M, p.K);
    // Two rows at once where there are rows enough to fill the SMs all the same: 8192 x 4096 with a residual 41.4 against 38.4 us,
    // without 26.1 against 25.1; 500 x 5120 5.1 against 5.7.
    const bool two = p.M >= 2048 && shape.rows == 1 && shape.chunks <= 2;
    const auto kernel = shape.chunks == 1   ? (two ? rms_norm_fp8_kernel<kFp16, kWeightF32, kE5M2, 1, 2> : rms_norm_fp8_kernel<kFp16, kWeightF32, kE5M2, 1, 1>)
                        : shape.chunks == 2 ? (two ? rms_norm_fp8_kernel<kFp16, kWeightF32, kE5M2, 2, 2> : rms_norm_fp8_kernel<kFp16, kWeightF32, kE5M2, 2, 1>)
                                            : rms_norm_fp8_kernel<kFp16, kWeightF32, kE5M2, 4, 1>;
    const int64_t rows = shape.rows * (two ? 2 : 1);
    return launch_kernel(kernel, (p.M + rows - 1) / rows, dim3(shape.threads, shape.rows), 0, stream, true, p);
}

// Measured against the persistent kernel: 1000 x 1024 7.5 against 9.2 us, 1024 x 4096 13.4 / 15.0, 2000 x 1024 18.5 / 10.9, 1000 x 256 7.2 / 5.1.
bool few_rows(int64_t M, int64_t K) { return M <= (K < 512 ? kFewNarrowRows : kFewRows) && K <= kFewWidth; }

template <bool kFp16, bool kWeightF32>
bool launch_norm_grad(const NormGradParams& p, float* grad_weight, cudaStream_t stream) {
    if (few_rows(p.M, p.K)) {
        const int threads = static_cast<int>((p.K / kVec + 31) / 32 * 32);
        return launch_kernel(rms_norm_dgrad_few_kernel<kFp16, kWeightF32>, p.M + (p.K + kColumnTile - 1) / kColumnTile,
                             dim3(threads < kFewThreads ? kFewThreads : threads), 0, stream, true, p, grad_weight);
    }
    const RowShape shape = row_shape(p.M, p.K);
    const int grid = norm_grad_grid(p.M, shape);
    const auto kernel = next_row_ahead(shape) ? rms_norm_dgrad_kernel<kFp16, kWeightF32, 2, kAheadThreads, true>
                        : shape.chunks == 1   ? rms_norm_dgrad_kernel<kFp16, kWeightF32, 1, kMaxNormThreads, false>
                        : shape.chunks == 2   ? rms_norm_dgrad_kernel<kFp16, kWeightF32, 2, kMaxNormThreads, false>
                        : shape.rows > 1      ? rms_norm_dgrad_kernel<kFp16, kWeightF32, 4, 32 * kRowsPerCta, false>
                                              : rms_norm_dgrad_kernel<kFp16, kWeightF32, 4, kMaxNormThreads, false>;
    const size_t smem = shape.rows > 1 ? static_cast<size_t>(p.K) * 4 : 0;
    // An ordinary launch: a persistent grid that starts among the CTAs of the kernel ahead is spread unevenly over the SMs (84 against 68 us
    // at 8192 x 4096).
    if (!launch_kernel(kernel, grid, dim3(shape.threads, shape.rows), smem, stream, false, p)) return false;
    return launch_kernel(column_sum_kernel, (p.K + 31) / 32, dim3(32 * kSumWarps), 0, stream, true, static_cast<const float*>(p.partials), grad_weight, grid, p.K);
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
    return launch_kernel(kernel, grid, dim3(256), 0, stream, true, static_cast<const uint16_t*>(grad), static_cast<const uint16_t*>(gate_up),
                         static_cast<uint16_t*>(grad_gate_up), chunks, row_chunks);
}

extern "C" bool launch_rms_norm_fp8(const void* x, const void* residual, const void* weight, void* residual_out, void* q, float* scale, float* rstd,
                                    int64_t M, int64_t K, float eps, int input_fp16, int weight_f32, int use_e5m2, cudaStream_t stream) {
    if (M < 0 || M > 0x7fffffff || K <= 0 || K % 16 != 0 || K > kMaxNormWidth) return false;
    if (M == 0) return true;
    if (x == nullptr || weight == nullptr || q == nullptr || scale == nullptr || rstd == nullptr || (residual == nullptr) != (residual_out == nullptr)) return false;
    if (!aligned(x, 16) || !aligned(residual, 16) || !aligned(weight, 16) || !aligned(residual_out, 16) || !aligned(q, 16) || !aligned(scale, 4) || !aligned(rstd, 4)) return false;
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
    if (M <= 0 || K <= 0 || K > kMaxNormWidth || few_rows(M, K)) return 0;
    return norm_grad_grid(M, row_shape(M, K)) * K;
}

extern "C" bool launch_rms_norm_dgrad(const void* grad, const void* x, const void* weight, const float* rstd, const void* grad_residual, void* grad_x,
                                      float* grad_weight, float* partials, int64_t M, int64_t K, int input_fp16, int weight_f32, cudaStream_t stream) {
    if (M <= 0 || M > 0x7fffffff || K <= 0 || K % 16 != 0 || K > kMaxNormWidth) return false;
    if (grad == nullptr || x == nullptr || weight == nullptr || rstd == nullptr || grad_x == nullptr || grad_weight == nullptr || (partials == nullptr && !few_rows(M, K))) return false;
    if (!aligned(grad, 16) || !aligned(x, 16) || !aligned(weight, 16) || !aligned(grad_residual, 16) || !aligned(grad_x, 16) || !aligned(grad_weight, 8) || !aligned(partials, 16) || !aligned(rstd, 4)) return false;
    const NormGradParams p{static_cast<const uint16_t*>(grad), static_cast<const uint16_t*>(x), weight, rstd, static_cast<const uint16_t*>(grad_residual),
                           static_cast<uint16_t*>(grad_x), partials, M, K};
    if (input_fp16 != 0) {
        return weight_f32 != 0 ? launch_norm_grad<true, true>(p, grad_weight, stream) : launch_norm_grad<true, false>(p, grad_weight, stream);
    }
    return weight_f32 != 0 ? launch_norm_grad<false, true>(p, grad_weight, stream) : launch_norm_grad<false, false>(p, grad_weight, stream);
}
