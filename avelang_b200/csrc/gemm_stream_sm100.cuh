// The dense products for a handful of tokens (M <= 16): bound by reading the weights once.
//
//   D[m, n] = epilogue( sum_k X[m, k] W[n, k] ),  X (M,K) and W (N,K) bf16 or int8, optionally two weights (gated).
//
// One persistent CTA per SM owns an even share of the weight rows, in groups of 8, over the whole of K: nothing is exchanged
// between CTAs, so there is no workspace, no counter, and the sums have the same order on every call.  A producer warp copies
// units of 16 rows, 4 KB of K per row and stage, into two shared-memory stages of 64 KB with plain bulk copies (no tensor
// map: a row's piece is contiguous), which keeps 128 KB in flight per SM; a third stage where the activations leave room in L1.
// Sixteen warps split each stage's K, 256 bytes of every row each, and add up in shared memory at the end of a unit.
//
// What the shape was chosen by (one token, us): int8 28672 x 8192 59 with units of 32 rows, 1 KB pieces and 8 warps, 50 with
// 16 rows and 2 KB, 40 with 16 warps, 39 with 4 KB pieces (floor 35.8); gated int8 2 x 28672 x 8192 110, 79, 73 and 71 (floor
// 71.5).  With 8 warps a warp's chain of loads and instructions per stage is longer than the stage takes to arrive.
//
// The consumers use mma.sync with 8 weight rows as the n of the instruction and 16 token rows as its m.  The order of K inside
// an instruction is free as long as both operands use the same one, so 16 bytes of a row serve as the B fragments of two
// instructions as they are, one 16-byte shared-memory load per lane; the activations (A) are read with the same pattern
// through L1.  The tensor pipe is far from the limit here (one instruction per 256 bytes of weights), and a tcgen05 tile of
// 128 weight rows would need K split between CTAs to occupy all SMs.
#pragma once

#include "activations.cuh"
#include "sm100_ptx.cuh"

namespace avefp4 {

struct StreamParams {
    const uint8_t* x;                // rows of ld bytes
    const uint8_t* w[2];
    long long ldx, ldw[2];           // row strides in bytes
    long long ldd, ld_gate, ld_up;   // in elements
    int m, n, k_bytes;               // k_bytes: bytes of K per row, a multiple of 16
    const float* x_scale;            // int8: one per token / per weight row
    const float* w_scale[2];
    const __nv_bfloat16* bias;
    int act;
    int stages;                      // of the ring
    __nv_bfloat16* d;
    __nv_bfloat16* gate;             // gated: both products as bf16, or nullptr
    __nv_bfloat16* up;
    int* status;
};

constexpr int kStreamWarps = 16;             // consumers
constexpr int kStreamThreads = 32 * (kStreamWarps + 1);
constexpr int kStreamRows = 16;              // weight rows of a unit at most
constexpr int kPieces = 4;                   // 64-byte pieces of a row that a warp takes of a stage
constexpr int kStreamSpan = 64 * kPieces * kStreamWarps;      // bytes of K per stage
// A row of a stage lies 64 bytes past a multiple of 128: a quarter warp's 16-byte loads (two rows, 64 bytes each) then meet
// all banks once.
constexpr int kStreamRowStride = kStreamSpan + 64;
constexpr int kStreamStageBytes = kStreamRows * kStreamRowStride;

template <bool M8>
struct StreamConfig {
    static constexpr int kTokens = M8 ? 8 : 16;
    static constexpr int kPitch = kStreamRows + 1;
    static constexpr int kMaxStages = M8 ? 3 : 2;
    static constexpr int kPartWords = kStreamWarps * kTokens * kPitch;      // every warp's sums of a unit
    static constexpr int kOffPart = 2 * 8 * kMaxStages + 16;                // after the barriers
    static constexpr int kOffRing = (kOffPart + 2 * 4 * kPartWords + 127) / 128 * 128;
    static constexpr int smem_bytes(int stages) { return kOffRing + stages * kStreamStageBytes; }
    static_assert(kOffRing + kMaxStages * kStreamStageBytes <= 232448, "shared memory budget");
};

// contiguous bytes from memory to this CTA's shared memory, both 16-byte aligned, completion on `bar`; read once: evict first
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(kL2EvictFirst)
                 : "memory");
}

template <bool INT8>
__device__ __forceinline__ void mma_16x8(uint32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (INT8) {
        asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

__device__ __forceinline__ float activate_any(float x, int act) {
    switch (act) {
        case AVE_FP4_ACT_RELU: return act_value<AVE_FP4_ACT_RELU>(x);
        case AVE_FP4_ACT_GELU: return act_value<AVE_FP4_ACT_GELU>(x);
        case AVE_FP4_ACT_GELU_TANH: return act_value<AVE_FP4_ACT_GELU_TANH>(x);
        case AVE_FP4_ACT_SILU: return act_value<AVE_FP4_ACT_SILU>(x);
        default: return x;
    }
}

// M8: at most 8 tokens.  Gated: a unit's rows are up to two groups of w[0] followed by the same groups of w[1].
template <bool INT8, bool GATED, bool M8>
__global__ void __launch_bounds__(kStreamThreads, 1)
gemm_stream_kernel(const StreamParams p) {
    constexpr int kSlots = kStreamRows / 8;                       // groups of a unit in shared memory
    constexpr int kUnit = GATED ? kSlots / 2 : kSlots;            // result groups of a unit
    using Cfg = StreamConfig<M8>;
    constexpr int kTokens = Cfg::kTokens;
    const int stages = p.stages;
    constexpr int kPitch = Cfg::kPitch;
    extern __shared__ __align__(128) uint8_t stream_smem[];
    uint32_t* part = reinterpret_cast<uint32_t*>(stream_smem + Cfg::kOffPart);      // [2][warp][token][row]
    uint8_t* smem = stream_smem + Cfg::kOffRing;
    const uint32_t ring = smem_u32(smem);
    const uint32_t bar_full = smem_u32(stream_smem);
    const uint32_t bar_empty = bar_full + Cfg::kMaxStages * 8;
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const int groups = (p.n + 7) / 8;
    const int first = static_cast<int>(static_cast<long long>(blockIdx.x) * groups / gridDim.x);
    const int last = static_cast<int>(static_cast<long long>(blockIdx.x + 1) * groups / gridDim.x);
    const int steps = (p.k_bytes + kStreamSpan - 1) / kStreamSpan;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(bar_full + s * 8, 1);
            mbar_init(bar_empty + s * 8, kStreamWarps);
        }
        fence_mbar_init();
    }
    __syncthreads();
    if (threadIdx.x == 0) pdl_launch_dependents();
    pdl_wait_prior_grid();

    if (warp == kStreamWarps) {
        // ---------------------------------------------------------------- producer: a lane per row
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int g0 = first; g0 < last && ok; g0 += kUnit) {
            const int got = min(kUnit, last - g0);
            const int half = got * 8;
            const int rows = GATED ? 2 * half : half;
            const bool second = GATED && lane >= half;
            const int n = min(g0 * 8 + (second ? lane - half : lane), p.n - 1);
            const uint8_t* src = p.w[second ? 1 : 0] + n * p.ldw[second ? 1 : 0];
            for (int k = 0; k < steps; ++k) {
                if (!mbar_wait(bar_empty + stage * 8, phase ^ 1u)) {
                    if (lane == 0) atomicCAS(p.status, 0, 101);
                    ok = false;
                    break;
                }
                const uint32_t bytes = static_cast<uint32_t>(min(kStreamSpan, p.k_bytes - k * kStreamSpan));
                if (lane == 0) mbar_arrive_expect_tx(bar_full + stage * 8, bytes * rows);
                __syncwarp();
                if (lane < rows)
                    bulk_load(ring + stage * kStreamStageBytes + lane * kStreamRowStride, src + k * kStreamSpan, bytes, bar_full + stage * 8);
                if (++stage == stages) { stage = 0; phase ^= 1u; }
            }
        }
        // wait until the consumers have taken every stage: no copy is in flight when the CTA exits
        for (int i = 0; i < stages && ok; ++i) {
            if (!mbar_wait(bar_empty + stage * 8, phase ^ 1u)) {
                if (lane == 0) atomicCAS(p.status, 0, 101);
                ok = false;
            }
            if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
        return;
    }

    // ------------------------------------------------------------------- consumers
    const int g = lane >> 2, t = lane & 3;
    const int k_mine = warp * 64 * kPieces + t * 16;            // this lane's first byte of a stage's K; the second is 64 further
    const bool lo = g < p.m, hi = !M8 && g + 8 < p.m;
    const uint8_t* xlo = p.x + (lo ? g : 0) * p.ldx + k_mine;
    const uint8_t* xhi = p.x + (hi ? g + 8 : 0) * p.ldx + k_mine;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint4 a[kPieces], b[kPieces];
    auto load_x = [&](int k) {
#pragma unroll
        for (int s = 0; s < kPieces; ++s) {
            const int at = k * kStreamSpan + s * 64;
            const bool in = at + k_mine < p.k_bytes;   // k_bytes % 16 == 0
            a[s] = load_16(xlo + at, in && lo);
            if constexpr (!M8) b[s] = load_16(xhi + at, in && hi);
            else b[s] = zero;
        }
    };
    load_x(0);
    int stage = 0, unit = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int g0 = first; g0 < last; g0 += kUnit, ++unit) {
        const int got = min(kUnit, last - g0);
        const int slots = GATED ? 2 * got : got;
        uint32_t acc[kSlots][4];
#pragma unroll
        for (int j = 0; j < kSlots; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[j][i] = 0u;
        for (int k = 0; k < steps; ++k) {
            // after a wait that ran out the warp goes on without waiting (its results are void), so that none of the CTA's
            // warps is left behind at the barrier below
            if (ok && !mbar_wait(bar_full + stage * 8, phase)) {
                if (lane == 0) atomicCAS(p.status, 0, 103);
                ok = false;
            }
            const uint8_t* tile = smem + stage * kStreamStageBytes + g * kStreamRowStride + k_mine;
            const int at = k * kStreamSpan + k_mine;
#pragma unroll
            for (int s = 0; s < kPieces; ++s) {
                // past the end of K the stage holds whatever was there before
                const bool in = at + s * 64 < p.k_bytes;
#pragma unroll
                for (int j = 0; j < kSlots; ++j) {
                    if (j >= slots) break;
                    const uint4 w = in ? *reinterpret_cast<const uint4*>(tile + j * 8 * kStreamRowStride + s * 64) : zero;
                    mma_16x8<INT8>(acc[j], a[s].x, b[s].x, a[s].y, b[s].y, w.x, w.y);
                    mma_16x8<INT8>(acc[j], a[s].z, b[s].z, a[s].w, b[s].w, w.z, w.w);
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_empty + stage * 8);
            if (++stage == stages) { stage = 0; phase ^= 1u; }
            load_x(k + 1 < steps ? k + 1 : 0);         // the next stage's activations, ahead of its weights
        }
        // c0, c1: token g, weight rows 2t and 2t + 1; c2, c3: token g + 8.  The buffers alternate: a warp that writes one again
        // has passed the barrier of the unit between, and with it everybody's reads of this one.
        uint32_t* mine = part + (unit & 1) * Cfg::kPartWords + warp * kTokens * kPitch;
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
            mine[g * kPitch + j * 8 + 2 * t] = acc[j][0];
            mine[g * kPitch + j * 8 + 2 * t + 1] = acc[j][1];
            if constexpr (!M8) {
                mine[(g + 8) * kPitch + j * 8 + 2 * t] = acc[j][2];
                mine[(g + 8) * kPitch + j * 8 + 2 * t + 1] = acc[j][3];
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * kStreamWarps) : "memory");
        const uint32_t* all = part + (unit & 1) * Cfg::kPartWords;
        const int cols = got * 8;
        for (int i = threadIdx.x; i < p.m * cols; i += 32 * kStreamWarps) {
            const int m = i / cols, c = i - m * cols, n = g0 * 8 + c;
            if (n >= p.n) continue;
            auto total = [&](int col) {
                if constexpr (INT8) {
                    int sum = 0;
#pragma unroll
                    for (int w = 0; w < kStreamWarps; ++w) sum += static_cast<int>(all[(w * kTokens + m) * kPitch + col]);
                    return __int2float_rn(sum);
                } else {
                    float sum = 0.0f;
#pragma unroll
                    for (int w = 0; w < kStreamWarps; ++w) sum += __uint_as_float(all[(w * kTokens + m) * kPitch + col]);
                    return sum;
                }
            };
            float y = total(c);
            float sx = 1.0f;
            if constexpr (INT8) {
                sx = load_f32(p.x_scale + m);
                y = y * load_f32(p.w_scale[0] + n) * sx;
            }
            if constexpr (GATED) {
                float u = total(cols + c);
                if constexpr (INT8) u = u * load_f32(p.w_scale[1] + n) * sx;
                if (p.gate != nullptr) {
                    p.gate[m * p.ld_gate + n] = __float2bfloat16_rn(y);
                    p.up[m * p.ld_up + n] = __float2bfloat16_rn(u);
                }
                y = activate_any(y, p.act) * u;
            } else {
                if (p.bias != nullptr) y += __bfloat162float(p.bias[n]);
                y = activate_any(y, p.act);
            }
            p.d[m * p.ldd + n] = __float2bfloat16_rn(y);
        }
    }
}

}  // namespace avefp4
