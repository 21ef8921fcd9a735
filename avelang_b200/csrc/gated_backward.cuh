// First step of the gated block's backward pass: from dH (M,F) and the kept G = X Wg^T, U = X Wu^T
//
//   dU = dH * act(G),   dG = dH * U * act'(G)
//
// in fp32, rounded to bf16: they are the tensor-core operands of the two products that follow (dX = dG Wg + dU Wu and
// dW = [dG dU]^T X), which take bf16; the rounding, at most 2^-8 of each element, averages out over the
// sums of those products to about that of their own rounding to bf16 (the gradients are off by 2.3e-3 to 2.4e-3 of their norm instead of
// 1.7e-3; a second, lower bf16 part of dG and dU would keep that and double the products).  Bound by memory: three matrices read,
// two written, 10 bytes per element.
#pragma once

#include "activations.cuh"
#include "sm100_ptx.cuh"

namespace avefp4 {

template <int ACT>
__device__ __forceinline__ void gated_backward_pair(uint32_t d, uint32_t g, uint32_t u, uint32_t& dg, uint32_t& du) {
    float v0, s0, v1, s1;
    act_value_slope<ACT>(bf16_lo(g), v0, s0);
    act_value_slope<ACT>(bf16_hi(g), v1, s1);
    du = pack_bf16(bf16_lo(d) * v0, bf16_hi(d) * v1);
    dg = pack_bf16(bf16_lo(d) * bf16_lo(u) * s0, bf16_hi(d) * bf16_hi(u) * s1);
}

// One 16-byte piece (8 columns) of each matrix per thread and step; f8 = F / 8.
template <int ACT>
__global__ void __launch_bounds__(256)
gated_backward_kernel(const __nv_bfloat16* dout, long long ld_dout, const __nv_bfloat16* gate, long long ld_gate, const __nv_bfloat16* up,
                      long long ld_up, __nv_bfloat16* d_gate, __nv_bfloat16* d_up, long long ld, long long rows, int f8) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const long long total = rows * f8;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
        const long long r = i / f8;
        const long long c = (i - r * f8) * 8;
        const uint4 d = load_16<true>(dout + r * ld_dout + c);
        const uint4 g = load_16<true>(gate + r * ld_gate + c);
        const uint4 u = load_16<true>(up + r * ld_up + c);
        uint4 dg, du;
        gated_backward_pair<ACT>(d.x, g.x, u.x, dg.x, du.x);
        gated_backward_pair<ACT>(d.y, g.y, u.y, dg.y, du.y);
        gated_backward_pair<ACT>(d.z, g.z, u.z, dg.z, du.z);
        gated_backward_pair<ACT>(d.w, g.w, u.w, dg.w, du.w);
        *reinterpret_cast<uint4*>(d_gate + r * ld + c) = dg;
        *reinterpret_cast<uint4*>(d_up + r * ld + c) = du;
    }
}

}  // namespace avefp4
