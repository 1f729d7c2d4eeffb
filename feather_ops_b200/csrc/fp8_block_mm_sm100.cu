// Block-scaled fp8 x fp8 product: activation codes with one float32 scale per row and 128 channels, weight codes with one
// per 128 x 128 block.
//   forward   C[m, n] = sum_b sa[b, m] sw[n / 128, b] (A[m, block b] . W[n, block b]) + bias[n]
//   backward  C[m, k] = sum_b sa[b, m] sw[b, k / 128] (A[m, block b] . W[block b, k])
// The tensor cores multiply the codes of one 128-deep block (four UMMAs, a fresh fp32 accumulator in tensor memory), and
// the epilogue warps scale each block's product into float32 registers while the next block is multiplied.
//
// The copy engine's boxes of the row-major weight are operands as they land: 128 bytes along K are a K-major row forward,
// and backward, where the contraction runs over the weight's rows, the same box is an MN-major operand.
//
// Two kernels, picked by `plan`:
//   * small_kernel: the weight is the M side of the UMMA (128 outputs per CTA) and 16 to 128 tokens its N side, so a few
//     tokens cost no padding to 128 rows. K is split over the CTAs of a cluster, which add their partial sums through
//     distributed shared memory in a fixed order.
//   * pair_kernel: 256 tokens x up to 256 outputs per CTA pair, persistent.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "feather_host.h"
#include "sm100_ptx.cuh"

namespace feather {
namespace f8mm {

constexpr int kBlock = 128;          // depth of a k block = channels per scale
constexpr int kTileBytes = 128 * 128;

__device__ uint32_t g_status[2];

struct Params {
    const float* a_scale;
    const float* w_scale;
    const uint16_t* bias;
    uint16_t* c;
    int64_t w_scale_block;   // step of the weight's scale from one block of the contraction to the next
    int64_t w_scale_out;     // ... and from one block of outputs to the next
    int M, width, num_kb;
    int tiles_m, tiles_n;
    int splits;              // small kernel: CTAs of a cluster along the contraction
    int tile_n, band;        // pair kernel: outputs per tile, row tiles per band of the walk
    uint32_t idesc;
};

struct Ring {
    uint32_t idx = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void advance(uint32_t depth) {
        if (++idx == depth) {
            idx = 0;
            phase ^= 1u;
        }
    }
};

template <bool kOutBf16>
__device__ __forceinline__ float bits_to_float(uint16_t v) {
    if constexpr (kOutBf16) {
        return __uint_as_float(static_cast<uint32_t>(v) << 16);
    } else {
        return __half2float(__ushort_as_half(v));
    }
}

template <bool kOutBf16>
__device__ __forceinline__ uint16_t float_to_bits(float v) {
    if constexpr (kOutBf16) {
        return __bfloat16_as_ushort(__float2bfloat16_rn(v));
    } else {
        return __half_as_ushort(__float2half_rn(v));
    }
}

template <bool kOutBf16>
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
    if constexpr (kOutBf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// Every lane waits; the warp goes on together or not at all.
__device__ __forceinline__ bool warp_wait(const WaitGuard& guard, uint64_t* bar, uint32_t parity, uint32_t site) {
    return __all_sync(0xffffffffu, guard.wait(bar, parity, site));
}

// A wait has run out somewhere in the CTA: copies in flight get time to land before the CTA gives up its shared memory.
__device__ __forceinline__ void let_copies_land(const WaitGuard& guard) {
    if (guard.aborted()) {
        const long long start = clock64();
        while (clock64() - start < 2000000LL) {
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// A few tokens: D[128 outputs, T tokens]
// ---------------------------------------------------------------------------------------------------------
constexpr int kSmallThreads = 192;   // warps 0-3 epilogue (their lane quarters of tensor memory), 4 loads, 5 multiplies
constexpr int kScaleAhead = 4;       // k blocks that the scales are fetched ahead

template <int T>
struct SmallSmem {
    static constexpr int kStageBytes = kTileBytes + T * 128;
    static constexpr int kStages = T <= 16 ? 6 : T == 32 ? 5 : T == 64 ? 4 : 3;   // two CTAs per SM
    static constexpr int kSlots = T <= 64 ? 4 : 2;                              // accumulators in tensor memory
    static constexpr int kScaleOff = kStages * kStageBytes;                     // [4 warps][2][T] floats
    static constexpr int kBarOff = kScaleOff + 4 * 2 * T * 4;
    static constexpr int kNumBars = 2 * kStages + 2 * kSlots;
    static constexpr int kTotal = kBarOff + kNumBars * 8 + 16;
    static constexpr int kDynamic = kTotal + 1024;
    static constexpr int kTmemColumns = kSlots * T < 32 ? 32 : kSlots * T;
    static_assert(T * 512 <= kStages * kStageBytes, "the partial sums are exchanged in the operand ring");
    static_assert(2 * (kDynamic + 1024) <= 228 * 1024 && 2 * kTmemColumns <= 512, "two CTAs per SM");
};

template <int T, bool kBackward, bool kOutBf16>
__global__ void __launch_bounds__(kSmallThreads, 2) small_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const Params p) {
    using L = SmallSmem<T>;
    extern __shared__ uint8_t smem_dyn[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* const full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);
    uint64_t* const empty = full + L::kStages;
    uint64_t* const tmem_full = empty + L::kStages;
    uint64_t* const tmem_empty = tmem_full + L::kSlots;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(full + L::kNumBars);
    volatile uint32_t* const abort_flag = tmem_slot + 1;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const WaitGuard guard{abort_flag, g_status};

    if (threadIdx.x == 0) {
        *abort_flag = 0u;
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < L::kSlots; ++s) {
            mbar_init(&tmem_full[s], 1);
            mbar_init(&tmem_empty[s], 4);
        }
        mbar_init_fence();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_w);
    }
    if (warp == 5) {
        tmem_alloc(tmem_slot, L::kTmemColumns);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    const int splits = p.splits;
    const int rank = static_cast<int>(blockIdx.x) % splits;
    const int tile = static_cast<int>(blockIdx.x) / splits;
    const int m0 = tile % p.tiles_m * T;         // row tiles fastest: the CTAs that share a weight tile run together
    const int tile_n = tile / p.tiles_m;
    const int n0 = tile_n * 128;
    const int kb_begin = static_cast<int>(static_cast<int64_t>(p.num_kb) * rank / splits);
    const int kb_end = static_cast<int>(static_cast<int64_t>(p.num_kb) * (rank + 1) / splits);
    const int row = warp < 4 ? warp * 32 + lane : 0;   // epilogue: output n0 + row
    float acc[T];

    if (warp == 4) {
        if (elect_one()) {
            grid_dependency_wait();
            Ring slot;
            for (int kb = kb_begin; kb < kb_end; ++kb) {
                if (!guard.wait(&empty[slot.idx], slot.phase ^ 1u, kSiteLoadEmpty)) break;
                uint8_t* const w_tile = smem + slot.idx * L::kStageBytes;
                mbar_arrive_expect_tx(&full[slot.idx], L::kStageBytes);
                if constexpr (kBackward) {
                    tma_load_2d(w_tile, &map_w, &full[slot.idx], n0, kb * kBlock);
                } else {
                    tma_load_2d(w_tile, &map_w, &full[slot.idx], kb * kBlock, n0);
                }
                tma_load_2d(w_tile + kTileBytes, &map_a, &full[slot.idx], kb * kBlock, m0);
                slot.advance(L::kStages);
            }
        }
        __syncwarp();
    } else if (warp == 5) {
        if (elect_one()) {
            Ring slot, out;
            for (int kb = kb_begin; kb < kb_end; ++kb) {
                if (!guard.wait(&tmem_empty[out.idx], out.phase ^ 1u, kSiteTmemEmpty)) break;
                if (!guard.wait(&full[slot.idx], slot.phase, kSiteLoadFull)) break;
                tc_fence_after_sync();
                const uint32_t w_addr = smem_u32(smem + slot.idx * L::kStageBytes);
                const uint32_t a_addr = w_addr + kTileBytes;
#pragma unroll
                for (int k = 0; k < kBlock / 32; ++k) {
                    const uint64_t desc_w = kBackward ? make_desc_sw128_mnmajor(w_addr + k * 32 * 128) : make_desc_sw128_kmajor(w_addr + k * 32);
                    umma_f8(tmem_base + out.idx * T, desc_w, make_desc_sw128_kmajor(a_addr + k * 32), p.idesc, k != 0 ? 1u : 0u);
                }
                umma_commit(&empty[slot.idx]);
                umma_commit(&tmem_full[out.idx]);
                slot.advance(L::kStages);
                out.advance(L::kSlots);
            }
        }
        __syncwarp();
    } else {
        constexpr int kPerLane = (T + 31) / 32;   // token scales that a lane fetches per k block
        float* const scales = reinterpret_cast<float*>(smem + L::kScaleOff) + warp * 2 * T;
        float sa[kScaleAhead][kPerLane], sw[kScaleAhead];
        const float* const w_scale = p.w_scale + tile_n * p.w_scale_out;
        const auto fetch = [&](int kb, int at) {
            if (kb >= kb_end) return;
            sw[at] = __ldg(w_scale + kb * p.w_scale_block);
#pragma unroll
            for (int j = 0; j < kPerLane; ++j) {
                const int token = j * 32 + lane;
                sa[at][j] = token < T && m0 + token < p.M ? __ldg(p.a_scale + static_cast<int64_t>(kb) * p.M + m0 + token) : 0.0f;
            }
        };
        grid_dependency_wait();
#pragma unroll
        for (int t = 0; t < T; ++t) acc[t] = 0.0f;
#pragma unroll
        for (int i = 0; i < kScaleAhead; ++i) fetch(kb_begin + i, i);
        Ring out;
        bool ok = true;
        for (int kb0 = kb_begin; ok && kb0 < kb_end; kb0 += kScaleAhead) {
#pragma unroll
            for (int i = 0; i < kScaleAhead; ++i) {
                if (!ok || kb0 + i >= kb_end) continue;
                float* const here = scales + (i & 1) * T;
#pragma unroll
                for (int j = 0; j < kPerLane; ++j) {
                    if (j * 32 + lane < T) here[j * 32 + lane] = sa[i][j] * sw[i];
                }
                fetch(kb0 + i + kScaleAhead, i);
                __syncwarp();
                ok = warp_wait(guard, &tmem_full[out.idx], out.phase, kSiteTmemFull);
                if (!ok) continue;
                tc_fence_after_sync();
                const uint32_t taddr = tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + out.idx * T;
#pragma unroll
                for (int c = 0; c < T / 16; ++c) {
                    uint32_t v[16];
                    tmem_ld_32x16(taddr + c * 16, v);
                    tmem_wait_ld();
                    if (c == T / 16 - 1) {
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&tmem_empty[out.idx]);
                    }
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const float4 s = *reinterpret_cast<const float4*>(here + c * 16 + g * 4);
                        acc[c * 16 + g * 4] = fmaf(__uint_as_float(v[g * 4]), s.x, acc[c * 16 + g * 4]);
                        acc[c * 16 + g * 4 + 1] = fmaf(__uint_as_float(v[g * 4 + 1]), s.y, acc[c * 16 + g * 4 + 1]);
                        acc[c * 16 + g * 4 + 2] = fmaf(__uint_as_float(v[g * 4 + 2]), s.z, acc[c * 16 + g * 4 + 2]);
                        acc[c * 16 + g * 4 + 3] = fmaf(__uint_as_float(v[g * 4 + 3]), s.w, acc[c * 16 + g * 4 + 3]);
                    }
                }
                out.advance(L::kSlots);
            }
        }
    }

    const int column = n0 + row;
    if (splits > 1) {
        // CTA r of the cluster owns tokens [r T / splits, ...): everybody's partial sums of them go into its operand ring
        // ([source][token][output]), which is free in every CTA once all have met here.
        const int share = T / splits;
        __syncthreads();
        cluster_sync_all();
        if (warp < 4) {
            const uint32_t local = smem_u32(smem) + (rank * share * 128 + row) * 4;
#pragma unroll
            for (int t = 0; t < T; ++t) {
                const int owner = t / share;
                st_shared_cluster_f32(map_to_cta(local + (t - owner * share) * 512, owner), acc[t]);
            }
        }
        cluster_sync_all();
        if (warp < 4 && column < p.width && !guard.aborted()) {
            const float bias = p.bias != nullptr ? bits_to_float<kOutBf16>(__ldg(p.bias + column)) : 0.0f;
            const float* const part = reinterpret_cast<const float*>(smem) + row;
            for (int t = 0; t < share; ++t) {
                const int token = m0 + rank * share + t;
                if (token >= p.M) break;
                float sum = part[t * 128];
                for (int s = 1; s < splits; ++s) sum += part[(s * share + t) * 128];
                p.c[static_cast<int64_t>(token) * p.width + column] = float_to_bits<kOutBf16>(sum + bias);
            }
        }
    } else if (warp < 4 && column < p.width && !guard.aborted()) {
        const float bias = p.bias != nullptr ? bits_to_float<kOutBf16>(__ldg(p.bias + column)) : 0.0f;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            if (m0 + t < p.M) p.c[static_cast<int64_t>(m0 + t) * p.width + column] = float_to_bits<kOutBf16>(acc[t] + bias);
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    let_copies_land(guard);
    if (warp == 5) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, L::kTmemColumns);
    }
}

// ---------------------------------------------------------------------------------------------------------
// Many tokens: 256 tokens x tile_n outputs per CTA pair
// ---------------------------------------------------------------------------------------------------------
constexpr int kPairStages = 6;
constexpr int kPairN = 256;
constexpr int kPairEpilogueWarps = 8;                              // two groups of four, one per half of the outputs
constexpr int kPairThreads = 32 * (4 + kPairEpilogueWarps);        // warps 0-3: load, multiply, relay, idle
constexpr int kImageBytes = 32 * 64;                               // 32 rows x 32 outputs of 16 bits

struct PairSmem {
    static constexpr int kStageBytes = 2 * kTileBytes;             // this CTA's 128 activation rows and its half of the outputs
    static constexpr int kImageOff = kPairStages * kStageBytes;    // two images per epilogue warp
    static constexpr int kBarOff = kImageOff + 2 * kPairEpilogueWarps * kImageBytes;
    static constexpr int kNumBars = 3 * kPairStages + 4;
    static constexpr int kTotal = kBarOff + kNumBars * 8 + 16;
    static constexpr int kDynamic = kTotal + 1024;
    static_assert(kDynamic <= 227 * 1024, "the pair kernel's shared memory exceeds an SM's");
};

template <bool kBackward, bool kOutBf16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_c, const Params p) {
    using L = PairSmem;
    extern __shared__ uint8_t smem_dyn[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~static_cast<uintptr_t>(1023));
    uint64_t* const load_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);   // this CTA's boxes have landed
    uint64_t* const load_empty = load_full + kPairStages;                         // signalled in both CTAs by CTA 0's commits
    uint64_t* const both_full = load_empty + kPairStages;                         // CTA 0 only: both CTAs' boxes have landed
    uint64_t* const tmem_full = both_full + kPairStages;
    uint64_t* const tmem_empty = tmem_full + 2;                                   // CTA 0 only
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(load_full + L::kNumBars);
    volatile uint32_t* const abort_flag = tmem_slot + 1;
    const int warp = static_cast<int>(threadIdx.x) / 32;
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const uint32_t cta = cluster_cta_rank();
    const WaitGuard guard{abort_flag, g_status};

    if (threadIdx.x == 0) {
        *abort_flag = 0u;
        for (int s = 0; s < kPairStages; ++s) {
            mbar_init(&load_full[s], 1);
            mbar_init(&load_empty[s], 1);
            mbar_init(&both_full[s], 2);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&tmem_full[s], 1);
            mbar_init(&tmem_empty[s], 2 * kPairEpilogueWarps);
        }
        mbar_init_fence();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_w);
        tma_prefetch_desc(&map_c);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 2 * kPairN);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;

    const int num_tiles = p.tiles_m * p.tiles_n;
    const int first_tile = static_cast<int>(blockIdx.x) / 2;
    const int tile_step = static_cast<int>(gridDim.x) / 2;
    const int half_n = p.tile_n / 2;

    if (warp < 4) {
        registers_decrease<56>();
        if (warp == 0 && elect_one()) {
            // ------------------------------------------------------------------ loads (this CTA's halves)
            grid_dependency_wait();
            const uint32_t stage_bytes = kTileBytes + (kBackward ? kTileBytes : half_n * 128);
            Ring slot;
            bool ok = true;
            for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
                int tile_m, tile_n;
                banded_tile(tile, p.tiles_m, p.tiles_n, p.band, tile_m, tile_n);
                const int m0 = tile_m * 256 + static_cast<int>(cta) * 128;
                const int n0 = tile_n * p.tile_n + static_cast<int>(cta) * half_n;
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    ok = guard.wait(&load_empty[slot.idx], slot.phase ^ 1u, kSiteLoadEmpty);
                    if (!ok) break;
                    uint8_t* const stage = smem + slot.idx * L::kStageBytes;
                    mbar_arrive_expect_tx(&load_full[slot.idx], stage_bytes);
                    tma_load_2d(stage, &map_a, &load_full[slot.idx], kb * kBlock, m0);
                    if constexpr (kBackward) {
                        tma_load_2d(stage + kTileBytes, &map_w, &load_full[slot.idx], n0, kb * kBlock);
                    } else {
                        tma_load_2d(stage + kTileBytes, &map_w, &load_full[slot.idx], kb * kBlock, n0);
                    }
                    slot.advance(kPairStages);
                }
            }
        } else if (warp == 1 && cta == 0 && elect_one()) {
            // ------------------------------------------------------------------ UMMA issuer of the pair
            Ring slot, out;
            bool ok = true;
            for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    ok = guard.wait(&tmem_empty[out.idx], out.phase ^ 1u, kSiteTmemEmpty) && guard.wait(&both_full[slot.idx], slot.phase, kSiteOperandFull);
                    if (!ok) break;
                    tc_fence_after_sync();
                    const uint32_t a_addr = smem_u32(smem + slot.idx * L::kStageBytes);
                    const uint32_t w_addr = a_addr + kTileBytes;
#pragma unroll
                    for (int k = 0; k < kBlock / 32; ++k) {
                        const uint64_t desc_w = kBackward ? make_desc_sw128_mnmajor(w_addr + k * 32 * 128) : make_desc_sw128_kmajor(w_addr + k * 32);
                        umma_f8_pair(tmem_base + out.idx * kPairN, make_desc_sw128_kmajor(a_addr + k * 32), desc_w, p.idesc, k != 0 ? 1u : 0u);
                    }
#pragma unroll
                    for (uint32_t dst = 0; dst < 2; ++dst) umma_commit_pair(map_to_cta(smem_u32(&load_empty[slot.idx]), dst));
#pragma unroll
                    for (uint32_t dst = 0; dst < 2; ++dst) umma_commit_pair(map_to_cta(smem_u32(&tmem_full[out.idx]), dst));
                    slot.advance(kPairStages);
                    out.advance(2);
                }
            }
        } else if (warp == 2 && elect_one()) {
            // ------------------------------------------------------------------ tells CTA 0 that this CTA's boxes have landed
            Ring slot;
            bool ok = true;
            for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    ok = guard.wait(&load_full[slot.idx], slot.phase, kSiteLoadFull);
                    if (!ok) break;
                    mbar_arrive_cluster(map_to_cta(smem_u32(&both_full[slot.idx]), 0));
                    slot.advance(kPairStages);
                }
            }
        }
    } else {
        registers_increase<216>();
        // ---------------------------------------------------------------------- epilogue: this CTA's 128 rows, half of the outputs per group
        const int epi_warp = warp - 4;
        const int quarter = warp % 4;
        const int half = epi_warp / 4;
        const int chunks = half_n / 32;
        const int twist = (lane >> 1) & 3;   // 64-byte swizzle: the 16-byte chunk index is XORed with bits 7-8 of the address
        uint8_t* const images = smem + L::kImageOff + epi_warp * 2 * kImageBytes;
        uint32_t stores = 0;
        Ring out;
        bool ok = true;
        grid_dependency_wait();
        for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
            int tile_m, tile_n;
            banded_tile(tile, p.tiles_m, p.tiles_n, p.band, tile_m, tile_n);
            const int row0 = tile_m * 256 + static_cast<int>(cta) * 128 + quarter * 32;
            const int col0 = tile_n * p.tile_n + half * half_n;
            // half_n is a multiple of 32 and at most 128: the columns meet at most two blocks of the weight's scales, and the
            // border lies between two chunks
            const int block_lo = col0 / kBlock;
            const int border = ((block_lo + 1) * kBlock - col0) / 32;   // first chunk of the second block
            const bool two = border < chunks && (block_lo + 1) * kBlock < p.width;
            const float* const a_scale = p.a_scale + (row0 + lane < p.M ? row0 + lane : 0);
            const float* const w_lo = p.w_scale + (col0 < p.width ? block_lo : 0) * p.w_scale_out;
            const float* const w_hi = two ? w_lo + p.w_scale_out : w_lo;
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
            float sa[kScaleAhead], lo[kScaleAhead], hi[kScaleAhead];
            const auto fetch = [&](int kb, int at) {
                if (kb >= p.num_kb) return;
                sa[at] = __ldg(a_scale + static_cast<int64_t>(kb) * p.M);
                lo[at] = __ldg(w_lo + kb * p.w_scale_block);
                hi[at] = __ldg(w_hi + kb * p.w_scale_block);
            };
#pragma unroll
            for (int i = 0; i < kScaleAhead; ++i) fetch(i, i);
            for (int kb0 = 0; ok && kb0 < p.num_kb; kb0 += kScaleAhead) {
#pragma unroll
                for (int i = 0; i < kScaleAhead; ++i) {
                    if (!ok || kb0 + i >= p.num_kb) continue;
                    const float s_lo = sa[i] * lo[i], s_hi = sa[i] * hi[i];
                    fetch(kb0 + i + kScaleAhead, i);
                    ok = warp_wait(guard, &tmem_full[out.idx], out.phase, kSiteTmemFull);
                    if (!ok) continue;
                    tc_fence_after_sync();
                    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + out.idx * kPairN + half * half_n;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (c < chunks) {
                            uint32_t v[32];
                            tmem_ld_32x32(taddr + c * 32, v);
                            tmem_wait_ld();
                            const float s = c < border ? s_lo : s_hi;
#pragma unroll
                            for (int j = 0; j < 32; ++j) acc[c * 32 + j] = fmaf(__uint_as_float(v[j]), s, acc[c * 32 + j]);
                        }
                    }
                    tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(map_to_cta(smem_u32(&tmem_empty[out.idx]), 0));
                    out.advance(2);
                }
            }
            if (!ok) break;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int column = col0 + c * 32;
                if (c >= chunks || column >= p.width || row0 >= p.M) continue;
                if (p.bias != nullptr) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        if (column + j < p.width) acc[c * 32 + j] += bits_to_float<kOutBf16>(__ldg(p.bias + column + j));
                    }
                }
                if (stores >= 2) {   // the image's earlier store has been read
                    if (lane == 0) tma_store_wait_read<1>();
                    __syncwarp();
                }
                uint8_t* const image = images + (stores & 1u) * kImageBytes;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float* const v = acc + c * 32 + g * 8;
                    *reinterpret_cast<uint4*>(image + lane * 64 + ((g ^ twist) << 4)) =
                        make_uint4(pack_out<kOutBf16>(v[0], v[1]), pack_out<kOutBf16>(v[2], v[3]), pack_out<kOutBf16>(v[4], v[5]), pack_out<kOutBf16>(v[6], v[7]));
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    tma_store_2d(&map_c, image, column, row0);   // clipped at M and width
                    tma_store_commit();
                }
                ++stores;
            }
        }
        if (lane == 0) tma_store_wait<0>();
        __syncwarp();
    }

    // ---------------------------------------------------------------------- teardown
    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    let_copies_land(guard);
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, 2 * kPairN);
    }
}

// ---------------------------------------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------------------------------------
struct Args {
    const uint8_t* a;
    const float* a_scale;
    const uint8_t* w;
    const float* w_scale;
    const uint16_t* bias;
    uint16_t* c;
    int64_t M, N, K;   // N and K: the weight's axes
    bool transposed_b, a_e5m2, w_e5m2, out_bf16;
    bool after_quantizer;   // the kernel before this one in the stream signals its dependents
    cudaStream_t stream;

    int64_t width() const { return transposed_b ? K : N; }
    int64_t depth() const { return transposed_b ? N : K; }
};

Params make_params(const Args& args) {
    Params p{};
    const int64_t scale_pitch = (args.K + kBlock - 1) / kBlock;
    p.a_scale = args.a_scale;
    p.w_scale = args.w_scale;
    p.bias = args.bias;
    p.c = args.c;
    p.w_scale_block = args.transposed_b ? scale_pitch : 1;
    p.w_scale_out = args.transposed_b ? 1 : scale_pitch;
    p.M = static_cast<int>(args.M);
    p.width = static_cast<int>(args.width());
    p.num_kb = static_cast<int>((args.depth() + kBlock - 1) / kBlock);
    return p;
}

bool make_maps(const Args& args, int a_rows, int w_rows, CUtensorMap& map_a, CUtensorMap& map_w) {
    const uint64_t a_dims[2] = {static_cast<uint64_t>(args.depth()), static_cast<uint64_t>(args.M)};
    const uint64_t a_strides[1] = {static_cast<uint64_t>(args.depth())};
    const uint32_t a_box[2] = {kBlock, static_cast<uint32_t>(a_rows)};
    const uint64_t w_dims[2] = {static_cast<uint64_t>(args.K), static_cast<uint64_t>(args.N)};
    const uint64_t w_strides[1] = {static_cast<uint64_t>(args.K)};
    const uint32_t w_box[2] = {128, static_cast<uint32_t>(w_rows)};
    return encode_map(&map_a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, args.a, a_dims, a_strides, a_box, CU_TENSOR_MAP_SWIZZLE_128B) &&
           encode_map(&map_w, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, args.w, w_dims, w_strides, w_box, CU_TENSOR_MAP_SWIZZLE_128B);
}

uint32_t format(bool e5m2) { return e5m2 ? kFmtE5M2 : kFmtE4M3; }

template <int T, bool kBackward, bool kOutBf16>
bool launch_small_instance(const Args& args, int splits) {
    using L = SmallSmem<T>;
    auto* const kernel = &small_kernel<T, kBackward, kOutBf16>;
    static PerDeviceState ready;
    if (ready.get([&] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynamic) == cudaSuccess ? 1 : 0; }) <= 0) return false;
    CUtensorMap map_a, map_w;
    if (!make_maps(args, T, 128, map_a, map_w)) return false;
    Params p = make_params(args);
    const int64_t tiles_m = (args.M + T - 1) / T, tiles_n = (args.width() + 127) / 128;
    if (tiles_m * tiles_n * splits > 0x7fffffff) return false;
    p.tiles_m = static_cast<int>(tiles_m);
    p.tiles_n = static_cast<int>(tiles_n);
    p.splits = splits;
    p.idesc = make_idesc(kAccF32, format(args.w_e5m2), format(args.a_e5m2), 128, T) | (kBackward ? kIdescAMajorMN : 0u);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(tiles_m * tiles_n * splits));
    config.blockDim = dim3(kSmallThreads);
    config.dynamicSmemBytes = L::kDynamic;
    config.stream = args.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = args.after_quantizer ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, map_a, map_w, p) == cudaSuccess;
}

template <bool kBackward, bool kOutBf16>
bool launch_small(const Args& args, int tokens, int splits) {
    switch (tokens) {
        case 16: return launch_small_instance<16, kBackward, kOutBf16>(args, splits);
        case 32: return launch_small_instance<32, kBackward, kOutBf16>(args, splits);
        case 64: return launch_small_instance<64, kBackward, kOutBf16>(args, splits);
        default: return launch_small_instance<128, kBackward, kOutBf16>(args, splits);
    }
}

template <bool kBackward, bool kOutBf16>
bool launch_pair(const Args& args, int tile_n) {
    using L = PairSmem;
    auto* const kernel = &pair_kernel<kBackward, kOutBf16>;
    static PerDeviceState resident_pairs;
    const int pairs = resident_pairs.get([&] {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynamic) != cudaSuccess) return 0;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(static_cast<unsigned>(device_info().sm_count / 2 * 2));
        config.blockDim = dim3(kPairThreads);
        config.dynamicSmemBytes = L::kDynamic;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        config.attrs = attr;
        config.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess || clusters <= 0) {
            (void)cudaGetLastError();
            clusters = device_info().sm_count / 2;
        }
        return clusters;
    });
    if (pairs <= 0) return false;
    CUtensorMap map_a, map_w, map_c;
    if (!make_maps(args, 128, kBackward ? 128 : tile_n / 2, map_a, map_w)) return false;
    const uint64_t c_dims[2] = {static_cast<uint64_t>(args.width()), static_cast<uint64_t>(args.M)};
    const uint64_t c_strides[1] = {static_cast<uint64_t>(args.width()) * 2};
    const uint32_t c_box[2] = {32, 32};
    if (!encode_map(&map_c, kOutBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, args.c, c_dims, c_strides, c_box, CU_TENSOR_MAP_SWIZZLE_64B)) return false;
    Params p = make_params(args);
    const int64_t tiles_m = (args.M + 255) / 256, tiles_n = (args.width() + tile_n - 1) / tile_n;
    if (tiles_m * tiles_n > 0x7fffffff) return false;
    p.tiles_m = static_cast<int>(tiles_m);
    p.tiles_n = static_cast<int>(tiles_n);
    p.tile_n = tile_n;
    int64_t band = (32ll << 20) / (256 * args.depth());   // about 32 MB of activations stay in L2 while a band sweeps the weight
    if (band < 4) band = 4;
    p.band = static_cast<int>(band < tiles_m ? band : tiles_m);
    p.idesc = make_idesc(kAccF32, format(args.a_e5m2), format(args.w_e5m2), 256, static_cast<uint32_t>(tile_n)) | (kBackward ? kIdescBMajorMN : 0u);
    cudaLaunchConfig_t config = {};
    const int64_t tiles = tiles_m * tiles_n;
    config.gridDim = dim3(static_cast<unsigned>(2 * (tiles < pairs ? tiles : pairs)));
    config.blockDim = dim3(kPairThreads);
    config.dynamicSmemBytes = L::kDynamic;
    config.stream = args.stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = args.after_quantizer ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, map_a, map_w, map_c, p) == cudaSuccess;
}

// Which kernel a product gets.
struct Plan {
    int tokens;   // small kernel: tokens per tile; 0: pair kernel
    int splits;   // small kernel: K splits (1, 2, 4 or 8)
    int tile_n;   // pair kernel: outputs per tile
};

Plan plan(int64_t M, int64_t width, int64_t depth, int sms) {
    const int64_t num_kb = (depth + kBlock - 1) / kBlock;
    const int64_t pair_tiles = (M + 255) / 256 * ((width + 255) / 256);
    if (M > 128 && pair_tiles * 4 >= sms) return {0, 1, 256};
    const int tokens = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const int64_t tiles = (M + tokens - 1) / tokens * ((width + 127) / 128);
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= 2 * sms && num_kb >= 4 * splits) splits *= 2;
    return {tokens, splits, 0};
}

template <bool kBackward, bool kOutBf16>
bool launch(const Args& args) {
    const Plan pick = plan(args.M, args.width(), args.depth(), device_info().sm_count);
    return pick.tokens == 0 ? launch_pair<kBackward, kOutBf16>(args, pick.tile_n) : launch_small<kBackward, kOutBf16>(args, pick.tokens, pick.splits);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace f8mm
}  // namespace feather

extern "C" bool launch_fp8_block_mm(const uint8_t* a, const float* a_scale, const uint8_t* w, const float* w_scale, const uint16_t* bias, uint16_t* c,
                                    int64_t M, int64_t N, int64_t K, bool transposed_b, int a_e5m2, int w_e5m2, int output_dtype, cudaStream_t stream) {
    using namespace feather::f8mm;
    constexpr int64_t kMost = 1 << 30;
    if (M < 0 || N <= 0 || K <= 0 || M > kMost || N > kMost || K > kMost || N % 16 != 0 || K % 16 != 0) return false;
    if (transposed_b && bias != nullptr) return false;
    if (output_dtype != 0 && output_dtype != 1) return false;
    if (M == 0) return true;
    if (a == nullptr || a_scale == nullptr || w == nullptr || w_scale == nullptr || c == nullptr) return false;
    if (!aligned16(a) || !aligned16(w) || !aligned16(c)) return false;
    const Args args{a, a_scale, w, w_scale, bias, c, M, N, K, transposed_b, a_e5m2 != 0, w_e5m2 != 0, output_dtype == 1, false, stream};
    if (transposed_b) return args.out_bf16 ? launch<true, true>(args) : launch<true, false>(args);
    return args.out_bf16 ? launch<false, true>(args) : launch<false, false>(args);
}

// Reads and clears the product's wait-status record (see feather_scaled_mm_status).
extern "C" int feather_fp8_block_mm_status(uint32_t* out) {
    uint32_t zero[2] = {0u, 0u};
    if (cudaDeviceSynchronize() != cudaSuccess) return 1;
    if (cudaMemcpyFromSymbol(out, feather::f8mm::g_status, sizeof(zero)) != cudaSuccess) return 1;
    if (cudaMemcpyToSymbol(feather::f8mm::g_status, zero, sizeof(zero)) != cudaSuccess) return 1;
    return 0;
}
