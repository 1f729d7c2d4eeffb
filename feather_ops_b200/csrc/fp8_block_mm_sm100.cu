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
// Two kernels, picked by `launch`:
//   * small_kernel: 128 outputs x 16, 32 or 128 tokens per CTA; for up to 32 tokens the weight is the M side of the UMMA,
//     so that a few tokens cost no padding to 128 rows. K is split over the CTAs of a cluster, which add their partial sums through
//     distributed shared memory in a fixed order. Bound by the pace of a CTA's k blocks (0.28 to 0.33 us each whatever their bytes) and, at these sizes,
//     by what a launch, the first loads and the exchange take: 1 x 12288 x 4096 12.1 to 12.6 us (50 MB, 4.0 TB/s; the weight alone is 7.8 from HBM, and with
//     the weight in L2 it takes 9.6), 24 x 5120 x 5120 10.5, 512 x 4096 x 4096 14.7.
//   * pair_kernel: 256 tokens x 256 outputs per CTA pair, persistent. 8192 x 12288 x 4096 397 to 410 us as the power cap allows
//     (2.0 PFLOP/s), 4096 x 4096 x 4096 68 in bursts of four launches, 75 to 76 in a sustained loop under that cap.
#include <cuda_runtime.h>

#include <cstdint>

#include "feather_host.h"
#include "fp8_block.cuh"
#include "sm100_ptx.cuh"

namespace feather {

// The activation quantizer as an ordinary launch that signals its dependents (fp8_block_quantize_sm100.cu).
bool launch_fp8_block_quantize_ahead(const void* x, void* q, float* scale, int64_t M, int64_t K, int input_fp16, int use_e5m2, cudaStream_t stream);

namespace f8mm {

using f8::kBlock;                    // depth of a k block = channels per scale
constexpr int kTileBytes = 128 * 128;
constexpr int kQuantizeRows = 8;     // up to so many tokens the product quantizes its activation itself ...
constexpr int kQuantizeWarps = 8;    // ... with so many warps, a k block each in turn
constexpr int kMaxSplits = 8;        // CTAs of a cluster along the contraction (the largest portable cluster)

__device__ uint32_t g_status[2];

struct Params {
    const uint16_t* x;       // small kernel that quantizes: the 16-bit activation
    int depth;
    bool x_fp16, x_e5m2;
    const float* a_scale;
    const float* w_scale;
    const uint16_t* bias;
    uint16_t* c;
    int64_t w_scale_block;   // step of the weight's scale from one block of the contraction to the next
    int64_t w_scale_out;     // ... and from one block of outputs to the next
    int M, width, num_kb;
    int tiles_m, tiles_n;
    int splits;              // small kernel: CTAs of a cluster along the contraction
    int band;                // pair kernel: row tiles per band of the walk
    bool weight_ready;       // small kernel: the weight may be read before the kernel ahead has finished
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
__device__ __forceinline__ uint32_t pack_out(float a, float b) {
    if constexpr (kOutBf16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&v);
    }
}

// The warp goes on together or not at all. The first poll is everybody's; a barrier that is not there yet is left to one
// lane, whose polls do not crowd the shared memory that the UMMAs read their operands from.
__device__ __forceinline__ bool warp_wait_longer(const WaitGuard& guard, uint64_t* bar, uint32_t parity, uint32_t site) {
    bool ok = true;
    if (threadIdx.x % 32 == 0) ok = guard.wait(bar, parity, site);
    return __shfl_sync(0xffffffffu, ok, 0);
}

__device__ __forceinline__ bool warp_wait(const WaitGuard& guard, uint64_t* bar, uint32_t parity, uint32_t site) {
    const bool ok = __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || warp_wait_longer(guard, bar, parity, site);
    __syncwarp();
    return ok;
}

// A wait has run out somewhere in the CTA: copies in flight get time to land before the CTA gives up its shared memory.
__device__ __forceinline__ void let_copies_land(const WaitGuard& guard) {
    if (guard.aborted()) {
        const long long start = clock64();
        while (clock64() - start < 2000000LL) {
        }
    }
}

// Scales. A load into a register that is used some k blocks later does not work: the loads of all the k blocks in between
// share the warp's few scoreboards, so the first use waits for the newest of them (3 loads per k block, fetched four ahead,
// cost the pair kernel 200 of 620 us at 8192 x 12288 x 4096). So a warp (two in the small kernel, a batch each in turn)
// brings the scales of k block after k block into shared memory with asynchronous copies, some blocks early, and writes the products
// sa * sw for the epilogue warps. Its arrival is the second one on the accumulator's "full" barrier, so the epilogue waits for both
// at once. It has to be quick: four-byte accesses, and its own next copies issued before the arrival, set the pace of both
// kernels (4096 x 4096 x 4096 69.6 us, then 64.9, and 63.2 without scales; 512 x 4096 x 4096 15.3, 14.1 and 13.8).
constexpr int kScaleAhead = 6;
constexpr int kScaleRing = 8;   // raw scales: more than kScaleAhead, a lane may still read the one before

// [kRows activation scales (zeros from `live` on), two weight scales] into `raw`
template <int kRows>
__device__ __forceinline__ void fetch_scales(float* raw, const float* a_scale, int live, const float* w0, const float* w1) {
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const uint32_t to = smem_u32(raw);
#pragma unroll
    for (int r = lane; r < kRows; r += 32) cp_async_4(to + r * 4, r < live ? a_scale + r : a_scale, r < live);
    if (lane < 2) cp_async_4(to + (kRows + lane) * 4, lane == 0 ? w0 : w1, true);
}

// Two accumulators at once: d += v * s, element by element. Volatile: the order with the tensor memory loads around it is the
// one that the registers were counted for.
__device__ __forceinline__ void fma2(float2& d, uint32_t v0, uint32_t v1, float s0, float s1) {
    asm volatile("{\n\t"
        ".reg .b64 a, b, c;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%0, %1};\n\t"
        "fma.rn.f32x2 c, a, b, c;\n\t"
        "mov.b64 {%0, %1}, c;\n\t"
        "}"
        : "+f"(d.x), "+f"(d.y)
        : "r"(v0), "r"(v1), "f"(s0), "f"(s1));
}

// Codes of one k block of the activation into the swizzled rows of an operand tile, and sa * sw of its tokens. Two tokens per pass, 16
// lanes each; no branch between the passes, so that their chains of shuffles overlap.
constexpr int kQuantizePasses = kQuantizeRows / 2;

template <bool kFp16, bool kE5M2>
__device__ __forceinline__ void quantize_passes(const uint4 (&in)[kQuantizePasses], int live, float sw, uint8_t* rows, float* product) {
    const int lane = static_cast<int>(threadIdx.x) % 32;
    const int chunk = lane % 16;
    uint2 codes[kQuantizePasses];
    float scale[kQuantizePasses];
#pragma unroll
    for (int t = 0; t < kQuantizePasses; ++t) {
        f8::Pairs v;
        f8::unpack8<kFp16>(in[t], v);
        codes[t] = f8::encode_block<kE5M2>(v, f8::max_magnitude_packed<kFp16>(in[t]), scale[t]);
    }
#pragma unroll
    for (int t = 0; t < kQuantizePasses; ++t) {
        const int token = 2 * t + lane / 16;
        if (token < live) {
            *reinterpret_cast<uint2*>(rows + sw128_offset(token, chunk / 2) + chunk % 2 * 8) = codes[t];
            if (chunk == 0) product[token] = scale[t] * sw;
        }
    }
}

// ---------------------------------------------------------------------------------------------------------
// A few tokens: D[128 outputs, T tokens]
// ---------------------------------------------------------------------------------------------------------
// T tokens per tile. With kQuantize (at most 8 tokens) the activation comes in 16 bits and eight warps write its codes into the operand
// ring themselves, a k block each in turn: every CTA quantizes the tokens again, which costs no time beside the weight, and a launch is
// saved, 3.4 us of the host's 11. With more tokens it does not keep up (24 x 5120 x 5120 17.3 us, 12.4 with a quantizer in front).
// Up to 32 tokens the weight is the UMMA's M side: lanes of tensor memory are outputs, columns tokens,
// and a column's scale comes from shared memory. With T = 128 the tokens are the M side, so that a lane has one scale per
// k block and the registers of a warp are outputs. (64 tokens as columns were never faster than 128 lanes: 64 x 5120 x 5120
// in three K splits 13.0 us against 10.9.)
// Loads, UMMAs and accumulators are handed over in steps: two k blocks each up to 32 tokens, where a hand-over costs as much as the
// block's UMMAs (1 x 12288 x 4096 12.7 us, 13.4 with one; 24 x 12288 x 4096 backward without a K split 23.0 and 24.7 at the time), one with 128 tokens (128 x 4096 x 4096
// 11.0, 11.4 with two; 888 x 2352 x 992 7.6 and 7.9). What is left at 16 x 12288 x 4096: 12.1 us, 9.6 with the weight in
// L2 (HBM would need 7.8 for it): 32 k blocks on each of 96 CTAs at their own pace, and launch, first loads and drain. Tiles of fewer outputs on more SMs, with as
// many k blocks each, take as long.
template <int T, bool kQuantize>
struct SmallShape {
    static constexpr bool kTokenLanes = T == 128;
    static constexpr int kWidth = kTokenLanes ? 128 : T;                 // columns of an accumulator
    static constexpr int kColumns = kTokenLanes ? 64 : T;                // ... that an epilogue warp scales
    static constexpr int kGroups = kWidth / kColumns;
    static constexpr int kTeams = kTokenLanes ? 1 : 2;                   // teams take the k blocks in turn
    static constexpr int kWarps = 4 * kGroups * kTeams;
    static constexpr int kScaleWarps = kQuantize ? kQuantizeWarps : 2;
    static constexpr int kThreads = 32 * (kWarps + 2 + kScaleWarps);     // the last ones load, multiply, and bring the scales or quantize
    static constexpr int kDeep = kTokenLanes ? 1 : 2;                    // k blocks per step
    static constexpr int kStageBytes = kDeep * (kTileBytes + T * 128);   // weight tiles, then activation tiles
    static constexpr int kActivationOff = kDeep * kTileBytes;
    static constexpr int kStages = T == 32 ? 5 : 6;
    static constexpr int kSlots = 4;                                     // steps whose accumulators are in tensor memory
    static constexpr int kSlotColumns = kDeep * kWidth;
    static constexpr int kTmemColumns = kSlots * kSlotColumns;
    static constexpr int kPitch = kTokenLanes ? 132 : 128;               // floats of a token's partial sums (lanes are tokens: no bank twice)
    static constexpr int kRaw = T + 4;                                   // floats: T token scales, the weight's, padding
    static constexpr int kRawOff = kStages * kStageBytes;
    static constexpr int kBatch = kSlots / 2;                            // steps that a scale warp does at a time
    static constexpr int kRawRing = kQuantize ? 1 : 4 * kScaleWarps * kBatch * kDeep;   // k blocks, a warp's fetched two batches ahead
    static constexpr int kProducts = 2 * kSlots * kDeep;                 // k blocks whose products are kept
    static constexpr int kScaleOff = kRawOff + kRawRing * kRaw * 4;      // [kProducts][T]
    static constexpr int kBarOff = kScaleOff + kProducts * T * 4;
    static constexpr int kNumBars = 2 * kStages + 2 * kSlots;
    static constexpr int kTotal = kBarOff + kNumBars * 8 + 16;
    static constexpr int kDynamic = kTotal + 1024;
    static_assert(kTeams * T * kPitch * 4 <= kStages * kStageBytes, "the partial sums are laid out in the operand ring");
    static_assert(kDynamic <= 227 * 1024 && kTmemColumns <= 512, "what an SM holds");
    static_assert(!kQuantize || T == 16, "the warps that quantize have registers for 8 tokens");
    static_assert(kSlots % kTeams == 0, "a team's accumulators are its own");
};

template <int T, bool kBackward, bool kOutBf16, bool kQuantize>
__global__ void __launch_bounds__((SmallShape<T, kQuantize>::kThreads), 1)
small_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w, const Params p) {
    using L = SmallShape<T, kQuantize>;
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
            mbar_init(&full[s], kQuantize ? 1 + L::kDeep : 1);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < L::kSlots; ++s) {
            mbar_init(&tmem_full[s], kQuantize ? 1 + L::kDeep : 2);
            mbar_init(&tmem_empty[s], 4 * L::kGroups);
        }
        mbar_init_fence();
    }
    if (warp == L::kWarps) {
        if (elect_one()) {
            if constexpr (!kQuantize) tma_prefetch_desc(&map_a);
            tma_prefetch_desc(&map_w);
        }
        __syncwarp();
    } else if (warp == L::kWarps + 1) {
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
    const int live = p.M - m0 < T ? p.M - m0 : T;
    const int kb_begin = static_cast<int>(static_cast<int64_t>(p.num_kb) * rank / splits);
    const int blocks = static_cast<int>(static_cast<int64_t>(p.num_kb) * (rank + 1) / splits) - kb_begin;
    constexpr int kDeep = L::kDeep;
    const int steps = (blocks + kDeep - 1) / kDeep;   // the last one may have fewer k blocks

    if (warp == L::kWarps) {
        // ---------------------------------------------------------------------- loads
        if (elect_one()) {
            const auto load_weight = [&](int i, int slot) {
                const int here = blocks - i * kDeep < kDeep ? blocks - i * kDeep : kDeep;
                uint8_t* const stage = smem + slot * L::kStageBytes;
                mbar_arrive_expect_tx(&full[slot], here * (kTileBytes + (kQuantize ? 0 : T * kBlock)));
#pragma unroll
                for (int d = 0; d < kDeep; ++d) {
                    const int depth0 = (kb_begin + i * kDeep + d) * kBlock;
                    if (d < here) tma_load_2d(stage + d * kTileBytes, &map_w, &full[slot], kBackward ? n0 : depth0, kBackward ? depth0 : n0);
                }
            };
            // behind the quantizer the weight fills the ring while that runs
            const int early = p.weight_ready ? (steps < L::kStages ? steps : L::kStages) : 0;
            for (int i = 0; i < early; ++i) load_weight(i, i);
            grid_dependency_wait();
            Ring slot;
            for (int i = 0; i < steps; ++i) {
                if (!guard.wait(&empty[slot.idx], slot.phase ^ 1u, kSiteLoadEmpty)) break;
                if (i >= early) load_weight(i, static_cast<int>(slot.idx));
                if constexpr (!kQuantize) {
#pragma unroll
                    for (int d = 0; d < kDeep; ++d) {
                        const int at = i * kDeep + d;
                        if (at < blocks) tma_load_2d(smem + slot.idx * L::kStageBytes + L::kActivationOff + d * T * kBlock, &map_a, &full[slot.idx], (kb_begin + at) * kBlock, m0);
                    }
                }
                slot.advance(L::kStages);
            }
        }
    } else if (warp == L::kWarps + 1) {
        // ---------------------------------------------------------------------- multiplies
        if (elect_one()) {
            grid_dependency_wait();
            Ring slot, out;
            for (int i = 0; i < steps; ++i) {
                if (!guard.wait(&tmem_empty[out.idx], out.phase ^ 1u, kSiteTmemEmpty)) break;
                if (!guard.wait(&full[slot.idx], slot.phase, kSiteLoadFull)) break;
                tc_fence_after_sync();
                const uint32_t stage = smem_u32(smem + slot.idx * L::kStageBytes);
#pragma unroll
                for (int d = 0; d < kDeep; ++d) {
                    if (i * kDeep + d >= blocks) break;
                    const uint32_t w_addr = stage + d * kTileBytes;
                    const uint32_t a_addr = stage + L::kActivationOff + d * T * kBlock;
#pragma unroll
                    for (int k = 0; k < kBlock / 32; ++k) {
                        const uint64_t desc_w = kBackward ? make_desc_sw128_mnmajor(w_addr + k * 32 * 128) : make_desc_sw128_kmajor(w_addr + k * 32);
                        const uint64_t desc_a = make_desc_sw128_kmajor(a_addr + k * 32);
                        umma_f8(tmem_base + out.idx * L::kSlotColumns + d * L::kWidth, L::kTokenLanes ? desc_a : desc_w, L::kTokenLanes ? desc_w : desc_a, p.idesc, k != 0 ? 1u : 0u);
                    }
                }
                if (i + L::kStages < steps) umma_commit(&empty[slot.idx]);   // no arrival that nobody waits for: the CTA might be gone by then
                umma_commit(&tmem_full[out.idx]);
                slot.advance(L::kStages);
                out.advance(L::kSlots);
            }
        }
    } else if (kQuantize && warp >= L::kWarps + 2) {
        // ---------------------------------------------------------------------- codes and scales, a k block per warp in turn
        const int first = warp - (L::kWarps + 2);
        float* const products = reinterpret_cast<float*>(smem + L::kScaleOff);
        const float* const w_scale = p.w_scale + tile_n * p.w_scale_out + kb_begin * p.w_scale_block;
        const int chunk = lane % 16;                          // 8 channels of the block
        const uint16_t* const x = p.x + static_cast<int64_t>(m0) * p.depth + chunk * 8;
        uint4 in[kQuantizePasses];
        float sw = 0.0f;
        const auto fetch = [&](int i) {
            if (i >= blocks) return;
            const int column = (kb_begin + i) * kBlock;
            sw = ld_global_f32(w_scale + i * p.w_scale_block);
#pragma unroll
            for (int t = 0; t < kQuantizePasses; ++t) {
                const int token = 2 * t + lane / 16;
                in[t] = token < live && column + chunk * 8 < p.depth ? f8::load16(x + static_cast<int64_t>(token) * p.depth + column) : make_uint4(0, 0, 0, 0);
            }
        };
        // the ring's rows past the last token are zero, once and for all
        const int spare = (T - live) * 8;
        for (int i = first * 32 + lane; i < spare * L::kStages * kDeep; i += 32 * L::kScaleWarps) {
            const int tile_at = i / spare;
            *reinterpret_cast<uint4*>(smem + tile_at / kDeep * L::kStageBytes + L::kActivationOff + (tile_at % kDeep * T + live) * kBlock + i % spare * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        asm volatile("bar.sync 1, %0;" ::"n"(32 * L::kScaleWarps) : "memory");
        grid_dependency_wait();
        fetch(first);
        for (int i = first; i < steps * kDeep; i += L::kScaleWarps) {   // past the last block: arrivals only
            const int at = i / kDeep, slot = at % L::kStages, before = at - L::kSlots;
            if (!warp_wait(guard, &empty[slot], (static_cast<uint32_t>(at / L::kStages) & 1u) ^ 1u, kSiteOperandEmpty)) break;
            // the slot's previous products are complete, as for the scale warp below
            if (before >= 0 && !warp_wait(guard, &tmem_full[before % L::kSlots], static_cast<uint32_t>(before / L::kSlots) & 1u, kSiteTmemFull)) break;
            uint8_t* const rows = smem + slot * L::kStageBytes + L::kActivationOff + i % kDeep * T * kBlock;
            float* const product = products + i % L::kProducts * T;
            if (p.x_fp16) {
                p.x_e5m2 ? quantize_passes<true, true>(in, live, sw, rows, product) : quantize_passes<true, false>(in, live, sw, rows, product);
            } else {
                p.x_e5m2 ? quantize_passes<false, true>(in, live, sw, rows, product) : quantize_passes<false, false>(in, live, sw, rows, product);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&full[slot]);
                mbar_arrive(&tmem_full[at % L::kSlots]);
            }
            fetch(i + L::kScaleWarps);
        }
    } else if (warp >= L::kWarps + 2) {
        // ---------------------------------------------------------------------- scales, kBatch steps at a time, the warps in turn
        constexpr int kBatch = L::kBatch, kFetch = kBatch * kDeep;   // steps, k blocks
        constexpr int kTurn = L::kScaleWarps * kBatch;
        float* const raw = reinterpret_cast<float*>(smem + L::kRawOff);
        float* const products = reinterpret_cast<float*>(smem + L::kScaleOff);
        const float* const a_scale = p.a_scale + static_cast<int64_t>(kb_begin) * p.M + m0;
        const float* const w_scale = p.w_scale + tile_n * p.w_scale_out + kb_begin * p.w_scale_block;
        const auto fetch = [&](int i0) {
#pragma unroll
            for (int j = 0; j < kFetch; ++j) {
                const int at = i0 * kDeep + j;
                if (at < blocks) {
                    const float* const w = w_scale + at * p.w_scale_block;
                    fetch_scales<T>(raw + at % L::kRawRing * L::kRaw, a_scale + static_cast<int64_t>(at) * p.M, live, w, w);
                }
            }
            cp_async_commit();
        };
        grid_dependency_wait();
        const int first = (warp - (L::kWarps + 2)) * kBatch;
        fetch(first);
        fetch(first + kTurn);
        for (int i0 = first; i0 < steps; i0 += kTurn) {
            cp_async_wait<1>();
            __syncwarp();
            // Every slot's previous products are complete (nothing orders the arrivals of two commits): these arrivals
            // count for the next ones, and the scales of two turns ago, which stood where these go, have been read.
            bool complete = true;
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const int before = i0 + j - L::kSlots;
                if (before >= 0 && complete) complete = warp_wait(guard, &tmem_full[before % L::kSlots], static_cast<uint32_t>(before / L::kSlots) & 1u, kSiteTmemFull);
            }
            if (!complete) break;
#pragma unroll
            for (int j = 0; j < kFetch; ++j) {
                const int at = i0 * kDeep + j;
                const float* const from = raw + at % L::kRawRing * L::kRaw;
                const float w = from[T];   // of blocks past the end: whatever stands there, nobody reads the products
                if (lane < T / 4) {
                    const float4 a = reinterpret_cast<const float4*>(from)[lane];
                    reinterpret_cast<float4*>(products + at % L::kProducts * T)[lane] = make_float4(a.x * w, a.y * w, a.z * w, a.w * w);
                }
            }
            __syncwarp();
            if (lane < kBatch && i0 + lane < steps) mbar_arrive(&tmem_full[(i0 + lane) % L::kSlots]);
            fetch(i0 + 2 * kTurn);
        }
        cp_async_wait<0>();
    } else {
        // ---------------------------------------------------------------------- epilogue
        constexpr int kColumns = L::kColumns;
        const int quarter = warp % 4;
        const int column0 = warp / 4 % L::kGroups * kColumns;
        const int team = warp / (4 * L::kGroups);
        const int token = quarter * 32 + lane;   // token lanes
        const float* const products = reinterpret_cast<const float*>(smem + L::kScaleOff);
        const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + column0;
        float2 acc[kColumns / 2];
#pragma unroll
        for (int t = 0; t < kColumns / 2; ++t) acc[t] = make_float2(0.0f, 0.0f);
        bool ok = true;
        grid_dependency_wait();
#pragma unroll 1
        for (int i = team; i < steps; i += L::kTeams) {
            const int at = i % L::kSlots;
            ok = warp_wait(guard, &tmem_full[at], static_cast<uint32_t>(i / L::kSlots) & 1u, kSiteTmemFull);
            if (!ok) break;
            tc_fence_after_sync();
            const float* const scales = products + i * kDeep % L::kProducts * T;
            const uint32_t from = taddr + at * L::kSlotColumns;
            if constexpr (L::kTokenLanes) {
                static_assert(kColumns == 64, "two loads of 32 columns");
#pragma unroll
                for (int d = 0; d < kDeep; ++d) {
                    if (i * kDeep + d >= blocks) break;
                    uint32_t v[2][32];
                    tmem_ld_32x32(from + d * L::kWidth, v[0]);
                    tmem_ld_32x32(from + d * L::kWidth + 32, v[1]);
                    const float s = scales[d * T + token];
                    tmem_wait_ld();
#pragma unroll
                    for (int g = 0; g < 64; g += 2) fma2(acc[g / 2], v[g / 32][g % 32], v[g / 32][g % 32 + 1], s, s);
                }
            } else {
                // All of the step's loads before the first product. Past the last block stands whatever was there: not used.
                uint32_t v[kDeep * T / 16][16];
#pragma unroll
                for (int c = 0; c < kDeep * T / 16; ++c) tmem_ld_32x16(from + c * 16, v[c]);
                tmem_wait_ld();
#pragma unroll
                for (int d = 0; d < kDeep; ++d) {
                    if (i * kDeep + d >= blocks) break;
#pragma unroll
                    for (int t = 0; t < T; t += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(scales + d * T + t);
                        const uint32_t* const c = v[(d * T + t) / 16] + t % 16;
                        fma2(acc[t / 2], c[0], c[1], f.x, f.y);
                        fma2(acc[t / 2 + 1], c[2], c[3], f.z, f.w);
                    }
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tmem_empty[at]);
        }
        // Every team's sums go into this CTA's operand ring, [team][token][output]. A team may be ahead of the last block's
        // UMMAs, which still read the ring.
        if (ok && steps > 0) {
            const int last = steps - 1;
            (void)warp_wait(guard, &tmem_full[last % L::kSlots], static_cast<uint32_t>(last / L::kSlots) & 1u, kSiteTmemFull);
        }
        float* const part = reinterpret_cast<float*>(smem) + team * T * L::kPitch;
        if constexpr (L::kTokenLanes) {
            float4* const to = reinterpret_cast<float4*>(part + token * L::kPitch + column0);
            if (token < live) {
#pragma unroll
                for (int g = 0; g < kColumns / 4; ++g) to[g] = make_float4(acc[2 * g].x, acc[2 * g].y, acc[2 * g + 1].x, acc[2 * g + 1].y);
            }
        } else {
#pragma unroll
            for (int t = 0; t < kColumns; ++t) {
                if (column0 + t < live) part[(column0 + t) * L::kPitch + quarter * 32 + lane] = t % 2 == 0 ? acc[t / 2].x : acc[t / 2].y;
            }
        }
    }

    // The cluster's CTAs share the tile's tokens out and add all partial sums of theirs: split by split, team by team.
    // One whose wait has run out has none to add, so it takes the whole cluster along, and the outputs stay unwritten.
    __syncwarp();
    __syncthreads();
    if (splits > 1) {
        if (warp == 0 && lane < splits && guard.aborted()) st_shared_cluster_u32(map_to_cta(smem_u32(tmem_slot + 1), static_cast<uint32_t>(lane)), 1u);
        __syncwarp();
        cluster_sync_all();
    }
    const int share = (live + splits - 1) / splits;
    const int token_end = (rank + 1) * share < live ? (rank + 1) * share : live;
    const int column = n0 + 4 * lane;
    if (column < p.width && !guard.aborted()) {
        float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (p.bias != nullptr) {
#pragma unroll
            for (int j = 0; j < 4; ++j) bias[j] = bits_to_float<kOutBf16>(ld_global_u16(p.bias + column + j));
        }
        for (int t = rank * share + warp; t < token_end; t += L::kThreads / 32) {
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int s = 0; s < splits; ++s) {
                const uint32_t part = map_to_cta(smem_u32(smem), static_cast<uint32_t>(s)) + (t * L::kPitch + 4 * lane) * 4;
#pragma unroll
                for (int team = 0; team < L::kTeams; ++team) {
                    const float4 v = ld_shared_cluster_f32x4(part + team * T * L::kPitch * 4);
                    sum.x += v.x;
                    sum.y += v.y;
                    sum.z += v.z;
                    sum.w += v.w;
                }
            }
            *reinterpret_cast<uint2*>(p.c + static_cast<int64_t>(m0 + t) * p.width + column) =
                make_uint2(pack_out<kOutBf16>(sum.x + bias[0], sum.y + bias[1]), pack_out<kOutBf16>(sum.z + bias[2], sum.w + bias[3]));
        }
    }

    __syncwarp();
    tc_fence_before_sync();
    __syncthreads();
    let_copies_land(guard);
    if (splits > 1) cluster_sync_all();   // nobody leaves while a peer reads its sums
    if (warp == L::kWarps + 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, L::kTmemColumns);
    }
}

// ---------------------------------------------------------------------------------------------------------
// Many tokens: 256 tokens x 256 outputs per CTA pair
// ---------------------------------------------------------------------------------------------------------
// What bounds it is the way of an accumulator from the tensor core through the epilogue's registers and back to the tensor
// core once per 128-deep block. So a k block's product is two UMMA groups of half the tile's outputs (h = 0, 1: rows
// h * seg .. of both CTAs' weight boxes), each with two accumulators, barriers and four epilogue warps of its own: the warps of one
// half load accumulators from tensor memory while those of the other scale theirs. A k block takes some 700
// clocks, and the tensor core works 62 % of them (4096 x 4096 x 4096): UMMAs and commit behind those of the other half, load, scale and release by the
// epilogue, and the issuer's wait form a ring of two accumulators. At 4096 x 4096 x 4096 (64.5 us then) a quarter of the UMMAs would save 8 us, no
// loads 7, no scaling 5, all three together 15. Other groups: four of 64 outputs take 16 to 24 % longer (8192 x 12288 x 4096 486 us, 390
// with two), one of 256 with one issuer 13 to 25 % (486). 16 epilogue warps: 18 % (half the registers, so loads and products take turns).
// Tiles of 128 outputs with four accumulators: 25 % (82.3 against 65.7), and slower than small_kernel where that is picked (512 x 4096 x 4096 16.0, 14.0).
constexpr int kPairStages = 4;
constexpr int kPairN = 256;
constexpr int kPairEpilogueWarps = 8;                              // [half][lane quarter]
constexpr int kPairThreads = 32 * (4 + kPairEpilogueWarps);        // warps 0-3: load, multiply h = 0 and 1, scales
constexpr int kImageBytes = 32 * 64;                               // 32 rows x 32 outputs of 16 bits
// Registers a thread, out of the 168 that a CTA of 384 threads starts with. With 56 for the first four warps the issuers and the scale warp spill (52 bytes
// stored and 48 loaded, 4 and 12 with 64; 4096 x 4096 x 4096 77.6 us, 76.0 with 64, both in a sustained loop), 72 spill as much as 64.
constexpr int kPairOtherRegisters = 64, kPairEpilogueRegisters = 216;
static_assert(4 * kPairOtherRegisters + kPairEpilogueWarps * kPairEpilogueRegisters <= (4 + kPairEpilogueWarps) * 168, "an increase would wait for good");

struct PairSmem {
    static constexpr int kStageBytes = 2 * kTileBytes;             // this CTA's 128 activation rows and its half of the outputs
    static constexpr int kImageOff = kPairStages * kStageBytes;    // [epilogue warp][4 chunks]
    static constexpr int kRaw = 132;                               // floats: 128 row scales, two of the weight's, padding
    static constexpr int kRawOff = kImageOff + kPairEpilogueWarps * 4 * kImageBytes;
    static constexpr int kScaleOff = kRawOff + kScaleRing * kRaw * 4;   // products [4 k blocks][2 weight blocks][128 rows]
    static constexpr int kBarOff = kScaleOff + 4 * 2 * 128 * 4;
    static constexpr int kNumBars = 3 * kPairStages + 8;
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
    uint64_t* const load_full = reinterpret_cast<uint64_t*>(smem + L::kBarOff);   // CTA 1: its boxes have landed
    uint64_t* const load_empty = load_full + kPairStages;                         // signalled in both CTAs by the commits of both halves
    uint64_t* const both_full = load_empty + kPairStages;                         // CTA 0: its own boxes have landed, and CTA 1's
    uint64_t* const tmem_full = both_full + kPairStages;                          // [half][accumulator]
    uint64_t* const tmem_empty = tmem_full + 4;                                   // CTA 0 only
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
            mbar_init(&load_empty[s], 2);
            mbar_init(&both_full[s], 2);
        }
        for (int s = 0; s < 4; ++s) {
            mbar_init(&tmem_full[s], 2);
            mbar_init(&tmem_empty[s], kPairEpilogueWarps);   // the half's four warps of both CTAs
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
    constexpr int half_n = kPairN / 2;   // outputs whose weight rows (backward: columns) this CTA loads
    constexpr int seg = half_n / 2;      // of these, the ones in one UMMA group

    if (warp < 4) {
        registers_decrease<kPairOtherRegisters>();
        // k blocks of all tiles of this pair
        const uint32_t turns = first_tile < num_tiles ? static_cast<uint32_t>((num_tiles - 1 - first_tile) / tile_step + 1) * static_cast<uint32_t>(p.num_kb) : 0u;
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
                const int n0 = tile_n * kPairN + static_cast<int>(cta) * half_n;
                for (int kb = 0; kb < p.num_kb; ++kb) {
                    ok = guard.wait(&load_empty[slot.idx], slot.phase ^ 1u, kSiteLoadEmpty);
                    if (!ok) break;
                    uint8_t* const stage = smem + slot.idx * L::kStageBytes;
                    uint64_t* const landed = cta == 0 ? &both_full[slot.idx] : &load_full[slot.idx];
                    mbar_arrive_expect_tx(landed, stage_bytes);
                    tma_load_2d(stage, &map_a, landed, kb * kBlock, m0);
                    tma_load_2d(stage + kTileBytes, &map_w, landed, kBackward ? n0 : kb * kBlock, kBackward ? kb * kBlock : n0);
                    slot.advance(kPairStages);
                }
            }
        } else if ((warp == 1 || warp == 2) && cta == 0 && elect_one()) {
            // ------------------------------------------------------------------ UMMA issuers of the pair, one per half of the outputs. A wait,
            // even on a barrier that is there, takes the issuing thread 75 clocks and a group with its commits 200. (One thread for both
            // halves, which then wait for one another: 4096 x 4096 x 4096 83.7 us, 81.7 with two.)
            const int h = warp - 1;
            grid_dependency_wait();
            Ring slot, out;
            bool ok = true;
            uint32_t left = turns;
            for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
                for (int kb = 0; kb < p.num_kb; ++kb, --left) {
                    // backward the weight box is MN-major: the group's outputs are bytes h * seg .. of its 128-byte rows
                    const uint32_t a_addr = smem_u32(smem + slot.idx * L::kStageBytes);
                    const uint32_t w_addr = a_addr + kTileBytes + h * (kBackward ? seg : seg * 128);
                    ok = guard.wait(&both_full[slot.idx], slot.phase, kSiteOperandFull) && guard.wait(&tmem_empty[2 * h + out.idx], out.phase ^ 1u, kSiteTmemEmpty);
                    if (!ok) break;
                    tc_fence_after_sync();
#pragma unroll
                    for (int k = 0; k < kBlock / 32; ++k) {
                        const uint64_t desc_w = kBackward ? make_desc_sw128_mnmajor(w_addr + k * 32 * 128) : make_desc_sw128_kmajor(w_addr + k * 32);
                        umma_f8_pair(tmem_base + out.idx * kPairN + h * kPairN / 2, make_desc_sw128_kmajor(a_addr + k * 32), desc_w, p.idesc, k != 0 ? 1u : 0u);
                    }
#pragma unroll
                    for (uint32_t dst = 0; dst < 2; ++dst) umma_commit_pair(map_to_cta(smem_u32(&tmem_full[2 * h + out.idx]), dst));
                    if (left > kPairStages) {   // no arrival that nobody waits for: the CTA might be gone by then
#pragma unroll
                        for (uint32_t dst = 0; dst < 2; ++dst) umma_commit_pair(map_to_cta(smem_u32(&load_empty[slot.idx]), dst));
                    }
                    slot.advance(kPairStages);
                    out.advance(2);
                }
            }
        } else if (warp == 1 && cta == 1 && elect_one()) {
            // ------------------------------------------------------------------ tells CTA 0 that this CTA's boxes have landed
            grid_dependency_wait();
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
        } else if (warp == 3) {
            // ------------------------------------------------------------------ scales of this CTA's rows
            float* const raw = reinterpret_cast<float*>(smem + L::kRawOff);
            float* const products = reinterpret_cast<float*>(smem + L::kScaleOff);
            // the block that is fetched next, kScaleAhead blocks before the one that is multiplied: it may be of the next tile
            int tile = first_tile, kb = 0, live = 0;
            const float *a_scale = p.a_scale, *w0 = p.w_scale, *w1 = p.w_scale;
            const auto enter = [&]() {
                if (tile >= num_tiles) return;
                int tile_m, tile_n;
                banded_tile(tile, p.tiles_m, p.tiles_n, p.band, tile_m, tile_n);
                const int row0 = tile_m * 256 + static_cast<int>(cta) * 128, col0 = tile_n * kPairN;
                live = p.M - row0;
                a_scale = p.a_scale + (live > 0 ? row0 : 0);
                // half_n is a block: the outputs of a CTA's weight rows have one block of weight scales
                w0 = p.w_scale + col0 / kBlock * p.w_scale_out;
                w1 = col0 + half_n < p.width ? p.w_scale + (col0 + half_n) / kBlock * p.w_scale_out : w0;
            };
            const auto fetch = [&](uint32_t turn) {
                if (tile < num_tiles) {
                    fetch_scales<128>(raw + turn % kScaleRing * L::kRaw, a_scale, live, w0, w1);
                    a_scale += p.M;
                    w0 += p.w_scale_block;
                    w1 += p.w_scale_block;
                    if (++kb == p.num_kb) {
                        kb = 0;
                        tile += tile_step;
                        enter();
                    }
                }
                cp_async_commit();
            };
            grid_dependency_wait();
            enter();
            for (uint32_t i = 0; i < kScaleAhead; ++i) fetch(i);
            for (uint32_t turn = 0; turn < turns; ++turn) {
                cp_async_wait<kScaleAhead - 1>();
                __syncwarp();
                const uint32_t slot = turn & 1u;
                // the accumulators' previous products are complete: this arrival counts for the next ones, and the scales of four
                // blocks ago, which stood where these go, have been read
                if (turn >= 2 && !(warp_wait(guard, &tmem_full[slot], ((turn >> 1) - 1) & 1u, kSiteTmemFull) &&
                                   warp_wait(guard, &tmem_full[2 + slot], ((turn >> 1) - 1) & 1u, kSiteTmemFull))) {
                    break;
                }
                const float* const from = raw + turn % kScaleRing * L::kRaw;
                const float4 a = reinterpret_cast<const float4*>(from)[lane];
                const float s0 = from[128], s1 = from[129];
                float4* const to = reinterpret_cast<float4*>(products + (turn & 3u) * 256) + lane;
                to[0] = make_float4(a.x * s0, a.y * s0, a.z * s0, a.w * s0);
                to[32] = make_float4(a.x * s1, a.y * s1, a.z * s1, a.w * s1);
                __syncwarp();
                if (lane < 2) mbar_arrive(&tmem_full[2 * lane + slot]);
                fetch(turn + kScaleAhead);
            }
            cp_async_wait<0>();
        }
    } else {
        registers_increase<kPairEpilogueRegisters>();
        // ---------------------------------------------------------------------- epilogue: this CTA's 128 rows
        const int quarter = warp % 4;
        const int half = (warp - 4) / 4;
        constexpr int kChunks = 2 * seg / 32;   // of 32 outputs: those of CTA 0's weight rows, then CTA 1's
        const int twist = (lane >> 1) & 3;   // 64-byte swizzle: the 16-byte chunk index is XORed with bits 7-8 of the address
        uint8_t* const images = smem + L::kImageOff + (warp - 4) * kChunks * kImageBytes;
        // the outputs of CTA 0's weight rows come first, then CTA 1's
        const auto chunk_column = [&](int col0, int c) { return col0 + half * seg + (2 * c >= kChunks ? half_n + (c - kChunks / 2) * 32 : c * 32); };
        const float* const products = reinterpret_cast<const float*>(smem + L::kScaleOff) + quarter * 32 + lane;
        const uint32_t empty0 = map_to_cta(smem_u32(tmem_empty + 2 * half), 0);
        const uint32_t taddr0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + half * (kPairN / 2);
        uint32_t turn = 0;   // k blocks so far: their accumulators alternate
        bool ok = true;
        grid_dependency_wait();   // the kernel before this one may still read what this one writes
        for (int tile = first_tile; ok && tile < num_tiles; tile += tile_step) {
            int tile_m, tile_n;
            banded_tile(tile, p.tiles_m, p.tiles_n, p.band, tile_m, tile_n);
            const int row0 = tile_m * 256 + static_cast<int>(cta) * 128 + quarter * 32;
            const int col0 = tile_n * kPairN;
            float2 acc[kChunks][16];
#pragma unroll
            for (int i = 0; i < 16 * kChunks; ++i) acc[i / 16][i % 16] = make_float2(0.0f, 0.0f);
            // Four chunks of 32 columns per k block, one being loaded while the one before is scaled, across
            // k blocks too: the last chunk of a block is scaled while the first of the next one comes.
            uint32_t v[2][32];
            ok = warp_wait(guard, &tmem_full[2 * half + (turn & 1u)], (turn >> 1) & 1u, kSiteTmemFull);
            if (!ok) break;
            tc_fence_after_sync();
            tmem_ld_32x32(taddr0 + (turn & 1u) * kPairN, v[0]);
#pragma unroll 1
            for (int kb = 0; kb < p.num_kb; ++kb) {
                const uint32_t slot = turn & 1u;
                const uint32_t taddr = taddr0 + slot * kPairN;
                const float s0 = products[(turn & 3u) * 256], s1 = products[(turn & 3u) * 256 + 128];
                ++turn;
#pragma unroll
                for (int c = 0; c < 3; ++c) {
                    tmem_wait_ld();
                    tmem_ld_32x32(taddr + (c + 1) * 32, v[(c + 1) % 2]);
                    const float s = 2 * c < kChunks ? s0 : s1;
#pragma unroll
                    for (int j = 0; j < 16; ++j) fma2(acc[c][j], v[c % 2][2 * j], v[c % 2][2 * j + 1], s, s);
                }
                tmem_wait_ld();
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(empty0 + slot * 8);
                if (kb + 1 < p.num_kb) {
                    ok = warp_wait(guard, &tmem_full[2 * half + (turn & 1u)], (turn >> 1) & 1u, kSiteTmemFull);
                    if (!ok) break;
                    tc_fence_after_sync();
                    tmem_ld_32x32(taddr0 + (turn & 1u) * kPairN, v[0]);
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) fma2(acc[kChunks - 1][j], v[1][2 * j], v[1][2 * j + 1], s1, s1);
            }
            if (!ok) break;
            // Output: an image per chunk, so that the warp waits for nothing but the last tile's stores, long done. (With one image per warp
            // the end of a tile held the tensor core up for 3000 clocks.)
            if (lane == 0) tma_store_wait_read<0>();
            __syncwarp();
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int column = chunk_column(col0, c);
                if (p.bias != nullptr) {
                    // a lane loads one output's, and hands it to the others
                    const float bias = column + lane < p.width ? bits_to_float<kOutBf16>(ld_global_u16(p.bias + column + lane)) : 0.0f;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        acc[c][j].x += __shfl_sync(0xffffffffu, bias, 2 * j);
                        acc[c][j].y += __shfl_sync(0xffffffffu, bias, 2 * j + 1);
                    }
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float2* const f = acc[c] + g * 4;
                    *reinterpret_cast<uint4*>(images + c * kImageBytes + lane * 64 + ((g ^ twist) << 4)) =
                        make_uint4(pack_out<kOutBf16>(f[0].x, f[0].y), pack_out<kOutBf16>(f[1].x, f[1].y), pack_out<kOutBf16>(f[2].x, f[2].y), pack_out<kOutBf16>(f[3].x, f[3].y));
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.M) {
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int column = chunk_column(col0, c);
                    if (column < p.width) tma_store_2d(&map_c, images + c * kImageBytes, column, row0);   // clipped at M and width
                }
                tma_store_commit();
            }
            __syncwarp();
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
// Launch. Both kernels are programmatic dependents: they may start while the kernel ahead in the stream ends, and wait for it
// (griddepcontrol.wait) before they read what it may have written. That is everything, except in the call that quantizes and
// multiplies: its quantizer is an ordinary launch, so by the time it runs nothing older can still write the weight.
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
    bool weight_ready;   // the kernel ahead in the stream is this library's quantizer, launched in the same call after all else had finished
    const uint16_t* x;   // not null: the small kernel quantizes it (a and a_scale are unused)
    bool x_fp16;
    cudaStream_t stream;

    int64_t width() const { return transposed_b ? K : N; }
    int64_t depth() const { return transposed_b ? N : K; }
};

Params make_params(const Args& args) {
    Params p{};
    p.x = args.x;
    p.depth = static_cast<int>(args.depth());
    p.x_fp16 = args.x_fp16;
    p.x_e5m2 = args.a_e5m2;
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

bool make_map_a(const Args& args, int rows, CUtensorMap& map) {
    const uint64_t dims[2] = {static_cast<uint64_t>(args.depth()), static_cast<uint64_t>(args.M)};
    const uint64_t strides[1] = {static_cast<uint64_t>(args.depth())};
    const uint32_t box[2] = {kBlock, static_cast<uint32_t>(rows)};
    return encode_map(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, args.a, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

bool make_map_w(const Args& args, int rows, CUtensorMap& map) {
    const uint64_t dims[2] = {static_cast<uint64_t>(args.K), static_cast<uint64_t>(args.N)};
    const uint64_t strides[1] = {static_cast<uint64_t>(args.K)};
    const uint32_t box[2] = {128, static_cast<uint32_t>(rows)};
    return encode_map(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, args.w, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

uint32_t format(bool e5m2) { return e5m2 ? kFmtE5M2 : kFmtE4M3; }

template <int T, bool kQuantize>
cudaLaunchConfig_t small_config(cudaLaunchAttribute* attr, int64_t grid, int splits) {
    using L = SmallShape<T, kQuantize>;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(grid));
    config.blockDim = dim3(L::kThreads);
    config.dynamicSmemBytes = L::kDynamic;
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    return config;
}

// How many clusters of `splits` CTAs the device holds at once (0: none, or the kernel cannot be prepared). Asked once per
// device: clusters live within a GPC, so 148 SMs hold 45 clusters of three and 15 of eight.
template <int T, bool kBackward, bool kOutBf16, bool kQuantize>
int small_clusters(int splits) {
    static PerDeviceState resident[kMaxSplits + 1];
    return resident[splits].get([&] {
        auto* const kernel = &small_kernel<T, kBackward, kOutBf16, kQuantize>;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SmallShape<T, kQuantize>::kDynamic) != cudaSuccess) return 0;
        cudaLaunchAttribute attr[2];
        const cudaLaunchConfig_t config = small_config<T, kQuantize>(attr, device_info().sm_count / splits * splits, splits);
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &config) != cudaSuccess) {
            (void)cudaGetLastError();
            clusters = 0;
        }
        return clusters;
    });
}

template <int T, bool kBackward, bool kOutBf16, bool kQuantize>
bool launch_small(const Args& args, int splits) {
    if (small_clusters<T, kBackward, kOutBf16, kQuantize>(splits) <= 0) return false;
    CUtensorMap map_a, map_w;
    if (!make_map_w(args, 128, map_w)) return false;
    if constexpr (kQuantize) {
        map_a = map_w;   // unused
    } else {
        if (!make_map_a(args, T, map_a)) return false;
    }
    Params p = make_params(args);
    const int64_t tiles_m = (args.M + T - 1) / T, tiles_n = (args.width() + 127) / 128;
    if (tiles_m * tiles_n * splits > 0x7fffffff) return false;
    p.tiles_m = static_cast<int>(tiles_m);
    p.tiles_n = static_cast<int>(tiles_n);
    p.splits = splits;
    p.weight_ready = args.weight_ready;
    p.idesc = SmallShape<T, kQuantize>::kTokenLanes ? make_idesc(kAccF32, format(args.a_e5m2), format(args.w_e5m2), 128, 128) | (kBackward ? kIdescBMajorMN : 0u)
                                         : make_idesc(kAccF32, format(args.w_e5m2), format(args.a_e5m2), 128, T) | (kBackward ? kIdescAMajorMN : 0u);
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t config = small_config<T, kQuantize>(attr, tiles_m * tiles_n * splits, splits);
    config.stream = args.stream;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, &small_kernel<T, kBackward, kOutBf16, kQuantize>, map_a, map_w, p) == cudaSuccess;
}

template <bool kBackward, bool kOutBf16>
bool launch_pair(const Args& args) {
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
    if (!make_map_a(args, 128, map_a) || !make_map_w(args, kBackward ? 128 : kPairN / 2, map_w)) return false;
    const uint64_t c_dims[2] = {static_cast<uint64_t>(args.width()), static_cast<uint64_t>(args.M)};
    const uint64_t c_strides[1] = {static_cast<uint64_t>(args.width()) * 2};
    const uint32_t c_box[2] = {32, 32};
    if (!encode_map(&map_c, kOutBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, args.c, c_dims, c_strides, c_box, CU_TENSOR_MAP_SWIZZLE_64B)) return false;
    Params p = make_params(args);
    const int64_t tiles_m = (args.M + 255) / 256, tiles_n = (args.width() + kPairN - 1) / kPairN;
    if (tiles_m * tiles_n > 0x7fffffff) return false;
    p.tiles_m = static_cast<int>(tiles_m);
    p.tiles_n = static_cast<int>(tiles_n);
    int64_t band = (32ll << 20) / (256 * args.depth());   // about 32 MB of activations stay in L2 while a band sweeps the weight
    if (band < 4) band = 4;
    p.band = static_cast<int>(band < tiles_m ? band : tiles_m);
    p.idesc = make_idesc(kAccF32, format(args.a_e5m2), format(args.w_e5m2), 256, static_cast<uint32_t>(kPairN / 2)) | (kBackward ? kIdescBMajorMN : 0u);
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
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, map_a, map_w, map_c, p) == cudaSuccess;
}

// What a product is expected to cost, in microseconds, and the K splits that give it. Fitted to single launches over weights in HBM
// (M 1 .. 3600, N 512 .. 12288, K 512 .. 4096): a launch 0.6, a round of CTAs its start and end and a time per k block, the exchange of
// the partial sums of a split.
struct Choice {
    double cost;
    int splits;
};

template <int T, bool kBackward, bool kOutBf16, bool kQuantize>
Choice small_choice(const Args& args) {
    constexpr double kRound = T == 16 ? 2.6 : T == 32 ? 2.8 : 5.0;
    constexpr double kPerBlock = T == 16 ? 0.28 : T == 32 ? 0.33 : 0.33;
    constexpr double kExchange = T == 16 ? 2.0 : 1.8;
    const int64_t num_kb = (args.depth() + kBlock - 1) / kBlock;
    const int64_t tiles = (args.M + T - 1) / T * ((args.width() + 127) / 128);
    Choice best{1e30, 1};
    for (int splits = 1; splits <= kMaxSplits && splits <= num_kb; ++splits) {
        const int clusters = small_clusters<T, kBackward, kOutBf16, kQuantize>(splits);
        if (clusters <= 0 || (splits > 1 && tiles > clusters)) continue;   // a split pays only where all clusters are resident at once
        const double rounds = static_cast<double>((tiles + clusters - 1) / clusters);
        const double blocks = static_cast<double>((num_kb + splits - 1) / splits);
        const double cost = 0.6 + rounds * (kRound + kPerBlock * blocks) + (splits == 1 ? 0.0 : kExchange);
        if (cost < best.cost) best = {cost, splits};
    }
    return best;
}

// A round of the pair kernel's tiles, 0.43 a k block.
double pair_cost(const Args& args) {
    const int64_t pairs = device_info().sm_count / 2;
    const int64_t tiles = (args.M + 255) / 256 * ((args.width() + kPairN - 1) / kPairN);
    const int64_t num_kb = (args.depth() + kBlock - 1) / kBlock;
    return 4.2 + static_cast<double>((tiles + pairs - 1) / pairs) * (1.3 + 0.43 * static_cast<double>(num_kb));
}

// Up to 16 tokens one tile of 16. Above, the cheapest of tiles of 16 (up to 64 tokens), of 32 (up to 128), of 128 and the pair kernel. Measured
// (us): 47 x 608 x 3888 backward 5.3 with tiles of 16 and 5.8 of 32, 26 x 10880 x 1568 13.3 and 7.8; 78 x 6016 x 640 5.2 with tiles of 32 and 6.0 of
// 128, 64 x 5120 x 5120 13.5 and 10.9; 512 x 4096 x 4096 14.1 with tiles of 128 and 20 on the pair kernel, 744 x 7872 x 560 22.0 and 12.6, 1024 x 4096 x
// 4096 29 and 21 to 24.
template <bool kBackward, bool kOutBf16>
bool launch(const Args& args) {
    if (args.x != nullptr) return launch_small<16, kBackward, kOutBf16, true>(args, small_choice<16, kBackward, kOutBf16, true>(args).splits);
    if (args.M <= 16) return launch_small<16, kBackward, kOutBf16, false>(args, small_choice<16, kBackward, kOutBf16, false>(args).splits);
    Choice least{1e30, 1}, narrow{1e30, 1}, wide{1e30, 1};
    double pair = 1e30;
    if (args.M <= 64) least = small_choice<16, kBackward, kOutBf16, false>(args);
    if (args.M <= 128) narrow = small_choice<32, kBackward, kOutBf16, false>(args);
    if (args.M > 32) {
        wide = small_choice<128, kBackward, kOutBf16, false>(args);
        pair = pair_cost(args);
    }
    if (least.cost < narrow.cost && least.cost < wide.cost && least.cost < pair) return launch_small<16, kBackward, kOutBf16, false>(args, least.splits);
    if (narrow.cost <= wide.cost && narrow.cost <= pair) return launch_small<32, kBackward, kOutBf16, false>(args, narrow.splits);
    if (wide.cost <= pair) return launch_small<128, kBackward, kOutBf16, false>(args, wide.splits);
    return launch_pair<kBackward, kOutBf16>(args);
}

bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

bool valid(const Args& args) {
    constexpr int64_t kMost = 1 << 30;
    if (args.M < 0 || args.N <= 0 || args.K <= 0 || args.M > kMost || args.N > kMost || args.K > kMost || args.N % 16 != 0 || args.K % 16 != 0) return false;
    if (args.transposed_b && args.bias != nullptr) return false;
    if (args.M == 0) return true;
    const bool codes = args.a != nullptr && args.a_scale != nullptr && aligned(args.a, 16) && aligned(args.a_scale, 4);
    if (!(args.x != nullptr ? aligned(args.x, 16) : codes) || args.w == nullptr || args.w_scale == nullptr || args.c == nullptr) return false;
    return aligned(args.w, 16) && aligned(args.c, 16) && aligned(args.w_scale, 4) && aligned(args.bias, 2);
}

bool launch(const Args& args) {
    if (args.M == 0) return true;
    if (args.transposed_b) return args.out_bf16 ? launch<true, true>(args) : launch<true, false>(args);
    return args.out_bf16 ? launch<false, true>(args) : launch<false, false>(args);
}

}  // namespace f8mm
}  // namespace feather

extern "C" bool launch_fp8_block_mm(const uint8_t* a, const float* a_scale, const uint8_t* w, const float* w_scale, const uint16_t* bias, uint16_t* c,
                                    int64_t M, int64_t N, int64_t K, bool transposed_b, int a_e5m2, int w_e5m2, int output_dtype, cudaStream_t stream) {
    using namespace feather::f8mm;
    if (output_dtype != 0 && output_dtype != 1) return false;
    const Args args{a, a_scale, w, w_scale, bias, c, M, N, K, transposed_b, a_e5m2 != 0, w_e5m2 != 0, output_dtype == 1, false, nullptr, false, stream};
    return valid(args) && launch(args);
}

extern "C" int64_t feather_fp8_block_linear_scratch_bytes(int64_t M, int64_t depth) {
    using namespace feather::f8mm;
    return M <= kQuantizeRows || depth <= 0 ? 0 : M * (depth + 4 * ((depth + kBlock - 1) / kBlock));
}

extern "C" bool launch_fp8_block_linear(const void* x, void* scratch, const uint8_t* w, const float* w_scale, const uint16_t* bias, uint16_t* c, int64_t M,
                                        int64_t N, int64_t K, bool transposed_b, int input_fp16, int q_e5m2, int w_e5m2, int output_dtype,
                                        cudaStream_t stream) {
    using namespace feather::f8mm;
    if (output_dtype != 0 && output_dtype != 1) return false;
    Args args{nullptr, nullptr, w, w_scale, bias, c, M, N, K, transposed_b, q_e5m2 != 0, w_e5m2 != 0, output_dtype == 1, false, nullptr, input_fp16 != 0, stream};
    if (M <= kQuantizeRows) {
        args.x = static_cast<const uint16_t*>(x);
        return valid(args) && launch(args);
    }
    uint8_t* const q = static_cast<uint8_t*>(scratch);
    float* const q_scale = reinterpret_cast<float*>(q + M * args.depth());   // a row is a multiple of 16 bytes
    args.a = q;
    args.a_scale = q_scale;
    args.weight_ready = true;
    return valid(args) && feather::launch_fp8_block_quantize_ahead(x, q, q_scale, M, args.depth(), input_fp16, q_e5m2, stream) && launch(args);
}

// Reads and clears the product's wait-status record (see feather_scaled_mm_status).
extern "C" int feather_fp8_block_mm_status(uint32_t* out) {
    uint32_t zero[2] = {0u, 0u};
    if (cudaDeviceSynchronize() != cudaSuccess) return 1;
    if (cudaMemcpyFromSymbol(out, feather::f8mm::g_status, sizeof(zero)) != cudaSuccess) return 1;
    if (cudaMemcpyToSymbol(feather::f8mm::g_status, zero, sizeof(zero)) != cudaSuccess) return 1;
    return 0;
}
