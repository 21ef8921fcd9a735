// Rows of a bf16 matrix -> 8-bit integers with one fp32 scale per row (a token's activations, a channel's weights):
//
//   top = max_k |x[r, k]|,  scale[r] = top / 127,  q[r, k] = rint(127 x[r, k] / top), ties to even
//
// top = 0 is taken as 127 (scale 1, all codes 0).  A row with an infinity or a NaN gets a NaN scale and codes of 0, so that
// whatever is computed from it is NaN and does not pass for a number.
//
// The codes are exact although no division is done per element.  x and top are bf16, so 127 x / top is a quotient of
// integers below 2^15 and 2^8, times a power of two: it is a tie between two codes exactly, or at least 2^-16 of its
// value away from one.  x * (127 / top), two roundings, is within 2^-22 of its value; rounding that to 19 significant bits
// brings every tie back to the tie itself (its 9 bits fit) and carries nothing across (2^-19 + 2^-22 < 2^-16).
//
// Bound by memory: 2 bytes read and 1 written per element.  A row stays in registers between the maximum and the
// rounding, so it is read once; rows of up to 1024 elements take one warp, longer ones one CTA, rows beyond
// 16384 elements are read twice.
#pragma once

#include "activations.cuh"
#include "sm100_ptx.cuh"

namespace avefp4 {

constexpr int kInt8Threads = 256;

// larger of the magnitudes of two bf16 pairs, as unsigned 16-bit integers: finite values order like integers, and
// infinities and NaN stay above all of them
__device__ __forceinline__ uint32_t max_magnitude(uint32_t top, uint32_t pair) { return __vmaxu2(top, pair & 0x7fff7fffu); }

__device__ __forceinline__ uint32_t max_magnitude(uint32_t top, const uint4& v) {
    return max_magnitude(max_magnitude(max_magnitude(max_magnitude(top, v.x), v.y), v.z), v.w);
}

// The code as the low byte of the word: adding 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the low bits.
__device__ __forceinline__ uint32_t int8_code(float x, float recip) {
    const float q = __fmul_rn(x, recip);
    const float c = __fmul_rn(q, 33.0f);           // q (2^5 + 1): the difference below keeps the upper 19 bits of q
    const float r = __fsub_rn(c, __fsub_rn(c, q));
    return __float_as_uint(__fadd_rn(r, 12582912.0f));
}

// Rows whose largest magnitude is below 2^-100 are taken 2^100 times as large, or 127 / top would overflow.
constexpr float kTinyTop = 7.88860905221011805e-31f, kTinyScale = 1.26765060022822940e30f;

template <bool TINY>
__device__ __forceinline__ uint32_t int8_codes4(uint32_t w0, uint32_t w1, float recip) {
    const float s = TINY ? kTinyScale : 1.0f;
    const uint32_t a = int8_code(bf16_lo(w0) * s, recip), b = int8_code(bf16_hi(w0) * s, recip);
    const uint32_t c = int8_code(bf16_lo(w1) * s, recip), d = int8_code(bf16_hi(w1) * s, recip);
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

struct RowScale {
    float scale, recip;    // recip: 127 / top, of the enlarged row if it is tiny
    bool tiny, finite;
};

// top: the row's largest magnitude as bf16 bits
__device__ __forceinline__ RowScale int8_row_scale(uint32_t top) {
    RowScale r;
    const float t = (top == 0u) ? 127.0f : __uint_as_float(top << 16);
    r.finite = top < 0x7f80u;
    r.tiny = t < kTinyTop;
    r.scale = r.finite ? __fdiv_rn(t, 127.0f) : __uint_as_float(0x7fc00000u);
    r.recip = __fdiv_rn(127.0f, r.tiny ? t * kTinyScale : t);
    return r;
}

__device__ __forceinline__ uint2 int8_codes8(const uint4& v, const RowScale& r) {
    if (!r.finite) return make_uint2(0u, 0u);
    if (r.tiny) return make_uint2(int8_codes4<true>(v.x, v.y, r.recip), int8_codes4<true>(v.z, v.w, r.recip));
    return make_uint2(int8_codes4<false>(v.x, v.y, r.recip), int8_codes4<false>(v.z, v.w, r.recip));
}

// NV 16-byte pieces per thread.  CTA_ROW: one row per CTA, else one per warp.  NV == 0: a row of any length, read twice.
template <int NV, bool CTA_ROW>
__global__ void __launch_bounds__(kInt8Threads)
quantize_int8_kernel(const __nv_bfloat16* x, long long rows, int k, long long ldx, int8_t* values, long long ldv, float* scales) {
    constexpr int kRowThreads = CTA_ROW ? kInt8Threads : 32;
    constexpr int kKeep = NV > 0 ? NV : 1;
    __shared__ uint32_t warp_top[kInt8Threads / 32];
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long row = CTA_ROW ? blockIdx.x : static_cast<long long>(blockIdx.x) * (kInt8Threads / 32) + warp;
    if (!CTA_ROW && row >= rows) return;
    const int i0 = CTA_ROW ? threadIdx.x : lane;
    const int pieces = k / 8;                        // k % 8 == 0
    const uint4* src = reinterpret_cast<const uint4*>(x + row * ldx);
    uint2* dst = reinterpret_cast<uint2*>(values + row * ldv);

    uint4 v[kKeep];
    uint32_t top = 0u;
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = i0 + j * kRowThreads;
            v[j] = load_16<true>(src + i, i < pieces);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) top = max_magnitude(top, v[j]);
    } else {
        for (int i = i0; i < pieces; i += kRowThreads) top = max_magnitude(top, load_16(src + i));
    }
    top = max(top >> 16, top & 0xffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (CTA_ROW) {
        if (lane == 0) warp_top[warp] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kInt8Threads / 32; ++w) top = max(top, warp_top[w]);
    }
    const RowScale r = int8_row_scale(top);
    if (i0 == 0) scales[row] = r.scale;
    if constexpr (NV > 0) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int i = i0 + j * kRowThreads;
            if (i < pieces) dst[i] = int8_codes8(v[j], r);
        }
    } else {
        for (int i = i0; i < pieces; i += kRowThreads) dst[i] = int8_codes8(load_16(src + i), r);
    }
}

}  // namespace avefp4
