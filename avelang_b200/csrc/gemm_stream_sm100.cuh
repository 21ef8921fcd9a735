// The dense products for a handful of tokens (M <= 16): bound by reading the weights once.
//
//   D[m, n] = epilogue( sum_k X[m, k] W[n, k] ),  X (M,K) and W (N,K) bf16 or int8, optionally two weights (gated).
//
// Every CTA owns ROWS weight rows over the whole of K and its warps split K, so nothing is exchanged between CTAs: no
// workspace, no counters, the same sums in the same order on every call.  Weights go straight from memory to the
// registers of mma.sync: a warp takes 8 weight rows (the n of the instruction) and 64 bytes of K at a time, each
// lane one 16-byte load.  The order of K inside an instruction is free as long as both operands use the same one, so the
// 16 bytes of a lane serve as its B fragments of two instructions as they are, and the activations (A, 16 token rows)
// are loaded with the same pattern, through L1, which all CTAs of an SM share.  The tensor pipe is far from the limit here
// (one instruction per 256 bytes of weights), and a tcgen05 tile of 128 weight rows would leave 20 SMs without work at
// N = 16384 or need K split between CTAs.
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
    int pdl;
    __nv_bfloat16* d;
    __nv_bfloat16* gate;             // gated: both products as bf16, or nullptr
    __nv_bfloat16* up;
};

constexpr int kStreamWarps = 8;

__device__ __forceinline__ uint4 ld_stream(const void* p) {      // read once: not kept in L1
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
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

// GATED: the ROWS weight rows are ROWS / 2 rows of w[0] and the same rows of w[1].  M8: at most 8 tokens.
template <bool INT8, bool GATED, bool M8, int ROWS>
__global__ void __launch_bounds__(kStreamWarps * 32)
gemm_stream_kernel(const StreamParams p) {
    constexpr int kGroups = ROWS / 8;                     // groups of 8 weight rows, one mma n each
    constexpr int kOut = GATED ? ROWS / 2 : ROWS;         // result columns of this CTA
    constexpr int kSpan = 256;                            // bytes of K a warp takes before it moves on
    __shared__ uint32_t part[kStreamWarps][16][ROWS + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * kOut;

    if (p.pdl) {
        pdl_launch_dependents();
        pdl_wait_prior_grid();
    }
    uint32_t acc[kGroups][4];
    const uint8_t* wrow[kGroups];
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0u;
        const int which = GATED ? (j >= kGroups / 2) : 0;
        int row = n0 + (GATED ? (j % (kGroups / 2)) * 8 : j * 8) + g;
        row = min(row, p.n - 1);                          // past the end: a row that exists, its sums are not written
        wrow[j] = p.w[which] + row * p.ldw[which] + t * 16;
    }
    const bool lo = g < p.m, hi = !M8 && g + 8 < p.m;
    const uint8_t* xlo = p.x + (lo ? g : 0) * p.ldx + t * 16;
    const uint8_t* xhi = p.x + (hi ? g + 8 : 0) * p.ldx + t * 16;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);

    for (int k0 = warp * kSpan; k0 < p.k_bytes; k0 += kStreamWarps * kSpan) {
        uint4 w[kGroups][4], a[4], b[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = k0 + s * 64;
            const bool in = k + t * 16 < p.k_bytes;       // k_bytes % 16 == 0
#pragma unroll
            for (int j = 0; j < kGroups; ++j) w[j][s] = in ? ld_stream(wrow[j] + k) : zero;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k = k0 + s * 64;
            const bool in = k + t * 16 < p.k_bytes;
            a[s] = (in && lo) ? __ldg(reinterpret_cast<const uint4*>(xlo + k)) : zero;
            if constexpr (!M8) b[s] = (in && hi) ? __ldg(reinterpret_cast<const uint4*>(xhi + k)) : zero;
            else b[s] = zero;
        }
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int j = 0; j < kGroups; ++j) {
                mma_16x8<INT8>(acc[j], a[s].x, b[s].x, a[s].y, b[s].y, w[j][s].x, w[j][s].y);
                mma_16x8<INT8>(acc[j], a[s].z, b[s].z, a[s].w, b[s].w, w[j][s].z, w[j][s].w);
            }
    }
    // c0, c1: token g, weight rows 2t and 2t + 1; c2, c3: token g + 8
#pragma unroll
    for (int j = 0; j < kGroups; ++j) {
        part[warp][g][j * 8 + 2 * t] = acc[j][0];
        part[warp][g][j * 8 + 2 * t + 1] = acc[j][1];
        if constexpr (!M8) {
            part[warp][g + 8][j * 8 + 2 * t] = acc[j][2];
            part[warp][g + 8][j * 8 + 2 * t + 1] = acc[j][3];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < (M8 ? 8 : 16) * kOut; i += kStreamWarps * 32) {
        const int m = i / kOut, c = i % kOut, n = n0 + c;
        if (m >= p.m || n >= p.n) continue;
        auto total = [&](int col) {
            if constexpr (INT8) {
                int s = 0;
#pragma unroll
                for (int w = 0; w < kStreamWarps; ++w) s += static_cast<int>(part[w][m][col]);
                return __int2float_rn(s);
            } else {
                float s = 0.0f;
#pragma unroll
                for (int w = 0; w < kStreamWarps; ++w) s += __uint_as_float(part[w][m][col]);
                return s;
            }
        };
        float y = total(c);
        float sx = 1.0f;
        if constexpr (INT8) {
            sx = __ldg(p.x_scale + m);
            y = y * __ldg(p.w_scale[0] + n) * sx;
        }
        if constexpr (GATED) {
            float u = total(kOut + c);
            if constexpr (INT8) u = u * __ldg(p.w_scale[1] + n) * sx;
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

}  // namespace avefp4
