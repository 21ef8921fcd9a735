/*
 * C ABI of libavefp4, second part: products on 8-bit integers, the gated feed-forward block on bf16 and int8, and the
 * gradients of the bf16 products.  Conventions as in ave_fp4.h: device pointers, everything enqueued on `stream` of the
 * current device without synchronising (safe inside graph capture), nothing allocated, 0 / negative argument error /
 * positive cudaError_t returned, message in ave_fp4_last_error(); ave_fp4_init(device) comes first.
 *
 * Matrices are row-major with a row stride in elements (ld...).  Pointers and row strides are multiples of 16 bytes
 * (a matrix of one row has no row stride to check), bias and scale vectors are contiguous and 16-byte aligned.
 * `activation` is AVE_FP4_ACT_*.  Results may not overlap operands.  No counterpart in the reference, whose one operator is
 * the bf16 product (python/avelang_kernels/amdgpu_gemm.py:458-494).
 */
#ifndef AVE_DENSE_H_
#define AVE_DENSE_H_

#include <stdint.h>

#include "ave_fp4.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Longest K of an integer product: K * 128 * 128 stays below 2^31. */
#define AVE_INT8_MAX_K 131056

/*
 * Rows of a bf16 matrix to 8-bit integers: top = max |x[r,:]|, scales[r] = top / 127 (fp32), values[r,k] =
 * rint(127 x[r,k] / top), ties to even, exactly.  top = 0 counts as 127.  A row holding an infinity or NaN gets scale NaN
 * and codes 0.  k % 16 == 0; `scales` holds `rows` fp32.
 */
int ave_int8_quantize(const void* x_bf16, int64_t rows, int64_t k, int64_t ldx, void* values, int64_t ldv, void* scales,
                      void* stream);

/*
 * D (m, n) bf16 = act(a_scales[row] * b_scales[col] * (A (m, k) B (n, k)^T) + bias[col]) on int8 operands; the integer sums
 * are exact (k <= AVE_INT8_MAX_K), the rest is fp32, rounded to bf16 once.  k % 16 == 0, n % 8 == 0.  bias_bf16 may be NULL.
 * `workspace` (here and in the two gated products): the bytes that the _workspace_bytes function gives for these sizes on the
 * current device, 256-byte aligned; 0 of them whenever m <= 8 or a row of K is shorter than AVE_DENSE_MIN_CUT_BYTES, and for most
 * other sizes.  It holds partial sums during the call and no state between calls.
 */
#define AVE_DENSE_MIN_CUT_BYTES 4096
int64_t ave_int8_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k);
int ave_int8_gemm(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb, const void* b_scales,
                  const void* bias_bf16, int activation, void* d_bf16, int64_t ldd, void* workspace, int64_t workspace_bytes,
                  int64_t m, int64_t n, int64_t k, void* stream);

/* D (m, f) bf16 = act(A Wg^T) * (A Wu^T), int8 operands with scales as above, one pass. */
int64_t ave_int8_gemm_gated_workspace_bytes(int64_t m, int64_t f, int64_t k);
int ave_int8_gemm_gated(const void* a, int64_t lda, const void* a_scales, const void* w_gate, int64_t ld_wg, const void* gate_scales,
                        const void* w_up, int64_t ld_wu, const void* up_scales, int activation, void* d_bf16, int64_t ldd,
                        void* workspace, int64_t workspace_bytes, int64_t m, int64_t f, int64_t k, void* stream);

/*
 * D (m, f) = act(X Wg^T) * (X Wu^T) on bf16: X (m, h), Wg and Wu (f, h); both products in one kernel, fp32 up to the one
 * rounding.  gate_bf16 and up_bf16 (both or neither NULL) receive X Wg^T and X Wu^T, for the backward pass.  h % 8 == 0, f % 8 == 0.
 */
int64_t ave_bf16_gemm_gated_workspace_bytes(int64_t m, int64_t f, int64_t h);
int ave_bf16_gemm_gated(const void* x, int64_t ldx, const void* w_gate, int64_t ld_wg, const void* w_up, int64_t ld_wu, int activation,
                        void* d_bf16, int64_t ldd, void* gate_bf16, int64_t ld_gate, void* up_bf16, int64_t ld_up,
                        void* workspace, int64_t workspace_bytes, int64_t m, int64_t f, int64_t h, void* stream);

/*
 * Backward pass of ave_bf16_gemm_gated from dD (m, f) and the kept products gate and up:
 *   dG = dD * up * act'(gate), dU = dD * act(gate)    (rounded to bf16: operands of the products)
 *   dx (m, h) = dG Wg + dU Wu,   dw_gate (f, h) = dG^T X,   dw_up (f, h) = dU^T X.
 * dx, or dw_gate and dw_up together, may be NULL.  `workspace`: ave_bf16_gated_backward_workspace_bytes(...) bytes (for the
 * current device; want_dx / want_dw: whether those results are not NULL), 256-byte aligned; it holds dG and dU, and partial sums
 * where K is cut into ranges, during the call, and no state between calls.  m == 0 writes zeros to dw_gate and dw_up.
 */
int64_t ave_bf16_gated_backward_workspace_bytes(int64_t m, int64_t f, int64_t h, int want_dx, int want_dw);
int ave_bf16_gated_backward(const void* dd, int64_t ld_dd, const void* x, int64_t ldx, const void* w_gate, int64_t ld_wg,
                            const void* w_up, int64_t ld_wu, const void* gate, int64_t ld_gate, const void* up, int64_t ld_up,
                            int activation, void* dx, int64_t ld_dx, void* dw_gate, void* dw_up, int64_t ld_dw, void* workspace,
                            int64_t workspace_bytes, int64_t m, int64_t f, int64_t h, void* stream);

/*
 * Gradients of D = A B^T (ave_bf16_gemm): da (m, k) = dD B, db (n, k) = dD^T A, for dD (m, n), A (m, k), B (n, k), read as
 * they lie in memory.  da or db may be NULL.  n % 8 == 0, k % 8 == 0; m == 0 writes zeros to db, n == 0 to da.  `workspace`:
 * ave_bf16_gemm_backward_workspace_bytes(...) bytes (for the current device; 0 for most sizes), 256-byte aligned, holds partial
 * sums during the call.
 */
int64_t ave_bf16_gemm_backward_workspace_bytes(int64_t m, int64_t n, int64_t k, int want_da, int want_db);
int ave_bf16_gemm_backward(const void* dd, int64_t ld_dd, const void* a, int64_t lda, const void* b, int64_t ldb, void* da,
                           int64_t ld_da, void* db, int64_t ld_db, void* workspace, int64_t workspace_bytes, int64_t m, int64_t n, int64_t k,
                           void* stream);

#ifdef __cplusplus
}
#endif

#endif /* AVE_DENSE_H_ */
