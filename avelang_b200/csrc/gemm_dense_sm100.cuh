// Persistent tcgen05 tile kernel of the dense products that come with something around them:
//
//   kOpInt8    C = A B^T       A (M,K), B (N,K) int8, both K-contiguous; int32 accumulators (tcgen05.mma kind::i8)
//   kOpBf16    C = A B^T       the same for bf16 (kind::f16, fp32 accumulators)
//   kOpBf16Nn  C = A B         A (M,K), B (K,N) bf16 as they lie in memory: B is read as an MN-major operand
//   kOpBf16Tn  C = A^T B       A (K,M), B (K,N) bf16: both operands MN-major
//
// and, per kernel, one epilogue:
//
//   kDensePlain   D = bf16(C)
//   kDenseScaled  D = bf16(act(C * a_scale[row] * b_scale[col] + bias[col]))
//   kDenseGated   two weights of F rows each: D = bf16(act(G) * U), G = A Wg^T, U = A Wu^T (with scales for int8);
//                 optionally G and U are written as bf16 as well, for the backward pass
//
// The gated form costs no more than a plain product with 2F columns: half of an accumulator tile's columns are rows of
// Wg and the other half the rows of Wu with the same numbers, so that the epilogue finds both factors of an output
// in one thread's TMEM lane.  With CTA pairs this takes no extra load: each CTA supplies half of the B tile, one of
// them from Wg, the other from Wu.
//
// Structure: warps 0 and 2 TMA producers (A and B), warp 1 MMA issuer, 8 or 16 epilogue warps; a ring of shared-memory stages
// of one or two K blocks of 128 bytes per row (128-byte swizzle); two accumulators of up to 256 columns in TMEM, so a tile's
// epilogue runs under the next tile's main loop.  The tile is 128 rows per CTA (one, or a pair on one instruction) by block_n
// columns, and block_n is a run-time value: the number of columns goes into the instruction descriptor, so the host picks
// it, and cuts of K for long sums of few tiles, by an estimate of the launch's clocks (plan_dense in ave_dense_api.cu).
//
// Measured on a B200, operands not in L2 (burst; back to back the power cap takes some 15 %): int8 8192^3 327 us (3.36 POP/s,
// twice the rate of cuBLAS in bf16), gated int8 4096 x 28672 x 8192 1.09 ms (3.53 POP/s), gated bf16 4096 x 16384 x 4096 665 us
// (1.65 PFLOP/s), both gradients of 8192 x 4096 x 16384 1.34 ms (1.64 PFLOP/s): bound by the tensor pipe.  int8 16 x 28672 x 8192
// 41 us (5.7 TB/s) and gated bf16 128 x 14336 x 8192 82 us (5.7 TB/s): bound by reading the weights.  In tiles narrower than 256
// columns the operands' way from L2 is the limit (50 to 85 bytes a clock and SM, less the more SMs ask), and below some 10 us the
// launch is: 0.8 us until the first operands are there, 0.3 until the first accumulator, 0.5 to 1 for the epilogue and 0.3 to 0.7
// to leave.
//
// An MN-major operand tile is kept as boxes of 64 elements (one swizzled 128-byte row) x 64 K rows, 8 KB each: the
// matrix descriptor steps 8 KB from one box to the next along MN (leading offset) and 1 KB from one group of eight
// K rows to the next (stride offset); an MMA's 16 K rows are two such groups.
#pragma once

#include "activations.cuh"
#include "sm100_ptx.cuh"

namespace avefp4 {

enum DenseOperands : int { kOpBf16 = 0, kOpInt8 = 1, kOpBf16Nn = 2, kOpBf16Tn = 3 };
enum DenseEpilogue : int { kDensePlain = 0, kDenseScaled = 1, kDenseGated = 2 };

struct DenseParams {
    long long ldd, ld_gate, ld_up;   // row strides in elements
    int m, n;                        // rows and columns of one result (gated: n = F)
    int num_kb;                      // stages of K of one segment
    int kb_stage;                    // K blocks of 128 bytes per row (64 bf16 or 128 int8 elements) in a stage: 1 or 2
    int segments;                    // 2: C = A0 B0 + A1 B1, two operand pairs of the same sizes
    int kb_split;                    // stages of K in a range
    int splits;                      // > 1: K is cut into that many ranges whose sums (fp32, or int32 of int8) go to `partial`,
                                     // [split][result, or gate and up][m][n]; another kernel adds them up
    int batches;                     // 2: two results, C0 from A0 and C1 from A1, B shared; tile rows of C1 follow those of C0
    int tiles_m, tiles_n;            // tiles of one result
    int block_n;                     // columns of a tile, a multiple of 8 (one CTA) or 32 (pair)
    int b_rows;                      // rows of B in a K block: block_n per CTA, or for an MN-major B the whole boxes of 64 that hold them
    int stages;                      // stages of the ring that fit with this block_n
    int a_rows;                      // rows of A in a K block: 128, or with fewer than that in all, those, to a multiple of 8
    int band;                        // tile rows per band of the schedule
    __nv_bfloat16* d[2];
    uint32_t* partial;
    const float* a_scale;            // one per row of A
    const float* b_scale[2];         // one per row of B; gated: of Wg and Wu
    const __nv_bfloat16* bias;
    int act;
    int wait_late;                   // the previous kernel in the stream writes nothing that this one reads or writes: run beside
                                     // its tail and wait for it (so that whoever waits for this one has waited for both) at the end
    int early, early_items;          // of a wait_late launch: its first `early` clusters start ahead of the others, on SMs that the
                                     // previous kernel has left or not used, and take so many tiles each before the rest is dealt out
    int direct;                      // scaled: rows and tiles of D lie on 32 bytes, a thread stores its row's 16 columns as it has them
    int trigger_late;                // let the next kernel start only once the previous one has finished (the next is wait_late)
    __nv_bfloat16* gate;             // gated: where to keep G and U, or nullptr
    __nv_bfloat16* up;
    int* status;
};

struct DenseConfig {
    static constexpr int kRingBytes = 192 * 1024;        // stages of kb_stage * (a_rows + b_rows) * 128 bytes
    static constexpr int kMaxStages = 16;
    static constexpr int kMaxEpiWarps = 16;
    static constexpr int kEpiBufBytes = 32 * 64;
    static constexpr int kOffEpi = kRingBytes;
    static constexpr int kOffBar = kOffEpi + kMaxEpiWarps * kEpiBufBytes;
    static constexpr int kOffTmemPtr = kOffBar + (2 * kMaxStages + 4) * 8;
    static constexpr int kSmemBytes = kOffTmemPtr + 16 + 1024;
    static constexpr int threads(int epi_warps) { return 96 + 32 * epi_warps; }
    static constexpr int stages(int a_rows, int b_rows, int kb_stage) {
        const int n = kRingBytes / (kb_stage * (a_rows + b_rows) * 128);
        return n < kMaxStages ? n : kMaxStages;
    }
    static_assert(kSmemBytes <= 232448, "shared memory budget");
};

// Tiled load with an L2 policy chosen at run time.
template <int CG>
__device__ __forceinline__ void tma_load(uint32_t dst, const void* tmap, uint32_t bar, int x, int y, uint64_t policy) {
    if constexpr (CG == 1) {
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
            ::"r"(dst), "l"(tmap), "r"(bar), "r"(x), "r"(y), "l"(policy)
            : "memory");
    } else {
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
            ::"r"(dst), "l"(tmap), "r"(bar), "r"(x), "r"(y), "l"(policy)
            : "memory");
    }
}

// Instruction descriptor of kind::f16 / kind::i8: bits 4-5 accumulator (1 fp32, 2 int32), 7-9 / 10-12 operand formats
// (kind::f16: 1 = bf16; kind::i8: 1 = signed), 15 / 16 A / B MN-major, 17-22 N >> 3, 24-28 M >> 4.
__device__ __forceinline__ uint32_t make_idesc_dense(bool int8, bool a_mn, bool b_mn, int mma_m, int mma_n) {
    return ((int8 ? 2u : 1u) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(a_mn) << 15) |
           (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(mma_n >> 3) << 17) |
           (static_cast<uint32_t>(mma_m >> 4) << 24);
}

template <int CG>
__device__ __forceinline__ void mma_int8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1) {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    }
}

// Work item -> (tile row, tile column, K range): ranges slowest; bands of `band` tile rows, rows fastest inside a band, so that
// the CTAs running at the same time share a few A panels and a few B panels in L2.
__device__ __forceinline__ void dense_tile(int t, int rows, int cols, int band, int& tm, int& tn, int& split) {
    split = 0;
    for (const int one = rows * cols; t >= one; t -= one) ++split;       // a few ranges at most
    const int per_band = band * cols;
    const int g = t / per_band;
    const int first = g * band;
    const int in_band = min(rows - first, band);
    const int r = t - g * per_band;
    tm = first + r % in_band;
    tn = r / in_band;
}

// What the epilogue needs of 16 columns beside their accumulators.
template <bool INT8, int EPI>
struct ColumnTerms {
    float4 s0[INT8 ? 4 : 1], s1[INT8 && EPI == kDenseGated ? 4 : 1];
    uint4 bias[EPI == kDenseScaled ? 2 : 1];
};

// Scales and bias of 16 columns from `col` on, in two halves: n is a multiple of 8, and where a half lies past the last column any
// other stands in for it.
template <bool INT8, int EPI>
__device__ __forceinline__ void load_terms(ColumnTerms<INT8, EPI>& t, const float* sb0, const float* sb1, const __nv_bfloat16* bias, int col, int n) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = min(col + 8 * h, n - 8);
        if constexpr (INT8) {
            t.s0[2 * h] = load_f32x4(sb0 + at);
            t.s0[2 * h + 1] = load_f32x4(sb0 + at + 4);
            if constexpr (EPI == kDenseGated) {
                t.s1[2 * h] = load_f32x4(sb1 + at);
                t.s1[2 * h + 1] = load_f32x4(sb1 + at + 4);
            }
        }
        if constexpr (EPI == kDenseScaled) t.bias[h] = (bias != nullptr) ? load_16(bias + at) : make_uint4(0u, 0u, 0u, 0u);
    }
}

// 16 accumulator columns of this thread's row -> 8 words of bf16 pairs.  (16 and not more at a time keeps the code of five
// activations small: a short launch runs it from a cold instruction cache.)
template <bool INT8, int EPI, int ACT>
__device__ __forceinline__ void dense_convert(const uint32_t (&v)[16], const uint32_t (&u)[16], uint32_t (&w)[8], float sa,
                                              const ColumnTerms<INT8, EPI>& t) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float c0[4], c1[4], b[4], y[4];
        if constexpr (INT8) { c0[0] = t.s0[q].x; c0[1] = t.s0[q].y; c0[2] = t.s0[q].z; c0[3] = t.s0[q].w; }
        if constexpr (INT8 && EPI == kDenseGated) { c1[0] = t.s1[q].x; c1[1] = t.s1[q].y; c1[2] = t.s1[q].z; c1[3] = t.s1[q].w; }
        if constexpr (EPI == kDenseScaled) {
            const uint32_t lo = (q & 1) ? t.bias[q >> 1].z : t.bias[q >> 1].x, hi = (q & 1) ? t.bias[q >> 1].w : t.bias[q >> 1].y;
            b[0] = bf16_lo(lo); b[1] = bf16_hi(lo); b[2] = bf16_lo(hi); b[3] = bf16_hi(hi);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            // int32 -> fp32 rounds to nearest: 2^-24 of the sum, far below the one rounding to bf16.  The channel's scale comes
            // first: weights are of ordinary size, so the product with a large token's scale overflows only if the result does.
            float g = __uint_as_float(v[4 * q + i]);
            if constexpr (INT8 && EPI == kDenseScaled) g = fmaf(__int2float_rn(static_cast<int>(v[4 * q + i])) * c0[i], sa, b[i]);
            else if constexpr (INT8) g = __int2float_rn(static_cast<int>(v[4 * q + i])) * c0[i] * sa;
            y[i] = act_value<ACT>(g);
            if constexpr (EPI == kDenseGated && INT8) y[i] *= __int2float_rn(static_cast<int>(u[4 * q + i])) * c1[i] * sa;
            if constexpr (EPI == kDenseGated && !INT8) y[i] *= __uint_as_float(u[4 * q + i]);
        }
        w[2 * q] = pack_bf16(y[0], y[1]);
        w[2 * q + 1] = pack_bf16(y[2], y[3]);
    }
}

// 16 columns of a row, on 32 bytes
__device__ __forceinline__ void store_16(__nv_bfloat16* at, const uint32_t (&w)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// A warp's 2 KB transpose buffer: 64 bytes per row, 16-byte piece q of row r in place q ^ (r / 2 & 3), so that eight lanes
// meet all banks once both when each writes its own row and when four read one row.
__device__ __forceinline__ uint32_t piece_addr(uint32_t sbuf, int row, int q) { return sbuf + row * 64 + ((q ^ ((row >> 1) & 3)) << 4); }

__device__ __forceinline__ void stage_piece(uint32_t sbuf, int row, int q, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_addr(sbuf, row, q)), "r"(w0), "r"(w1), "r"(w2), "r"(w3) : "memory");
}

__device__ __forceinline__ uint4 staged_piece(uint32_t sbuf, int row, int q) {
    uint4 w;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(piece_addr(sbuf, row, q)) : "memory");
    return w;
}

template <int CG, int OP, int EPI>
__global__ void __launch_bounds__(608, 1)
gemm_dense_kernel(const __grid_constant__ CUtensorMap tm_a0, const __grid_constant__ CUtensorMap tm_a1,
                  const __grid_constant__ CUtensorMap tm_b0, const __grid_constant__ CUtensorMap tm_b1, const DenseParams p) {
    using Cfg = DenseConfig;
    constexpr bool kInt8 = (OP == kOpInt8);
    constexpr bool kAMn = (OP == kOpBf16Tn);
    constexpr bool kBMn = (OP == kOpBf16Nn || OP == kOpBf16Tn);
    constexpr bool kGated = (EPI == kDenseGated);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));

    // warp-uniform values through a shuffle, so that the issue loops keep them in uniform registers
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const int rank = (CG == 2) ? static_cast<int>(__shfl_sync(0xffffffffu, cluster_ctarank(), 0)) : 0;
    const bool is_leader = (rank == 0);
    const int cluster_id = blockIdx.x / CG;
    const int num_clusters = gridDim.x / CG;
    const int tile_rows = p.tiles_m * p.batches;
    const int num_tiles = tile_rows * p.tiles_n * p.splits;
    const int all_kb = p.num_kb * p.segments;
    const int stages = p.stages;
    const int epi_warps = static_cast<int>(blockDim.x) / 32 - 3;
    const int bn_cta = p.block_n / CG;                            // columns of the tile whose B one CTA loads
    const int b_bytes = p.b_rows * 128;                           // whole 1 KB swizzle groups
    const int a_bytes = p.a_rows * 128;
    const int kbs = p.kb_stage;
    const uint32_t ring_b = smem_base + stages * kbs * a_bytes;
    const int out_cols = kGated ? p.block_n / 2 : p.block_n;      // result columns of a tile

    const uint32_t bar_full = smem_base + Cfg::kOffBar;
    const uint32_t bar_empty = bar_full + Cfg::kMaxStages * 8;
    const uint32_t bar_tfull = bar_empty + Cfg::kMaxStages * 8;
    const uint32_t bar_tempty = bar_tfull + 2 * 8;
    const uint32_t tmem_ptr_smem = smem_base + Cfg::kOffTmemPtr;
    volatile uint32_t* tmem_ptr_gen = reinterpret_cast<volatile uint32_t*>(smem_gen + Cfg::kOffTmemPtr);

    if (threadIdx.x == 0) {
        prefetch_tensormap(&tm_a0);
        prefetch_tensormap(&tm_b0);
        prefetch_tensormap(&tm_a1);
        prefetch_tensormap(&tm_b1);
        for (int s = 0; s < stages; ++s) {
            mbar_init(bar_full + s * 8, 2);      // both producers of the leader
            mbar_init(bar_empty + s * 8, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(bar_tfull + a * 8, 1);
            mbar_init(bar_tempty + a * 8, epi_warps * CG);
        }
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<CG>(tmem_ptr_smem, 512);
        tmem_relinquish<CG>();
    }
    tcgen05_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();
    tcgen05_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr_gen, 0);

    // This cluster's first work item, and the step from its i-th one to the next: the early clusters share out the first items among
    // themselves, then all of them take turns.
    const int ahead = cluster_id < p.early ? p.early_items : 0;
    const int first_item = cluster_id < p.early ? cluster_id : cluster_id + (p.early_items - 1) * p.early;
    auto step = [&](int i) { return i + 1 < ahead ? p.early : num_clusters; };

    // Operands may come from the previous kernel.  All roles wait for it here, so that none of the bounded waits below counts its time.
    if (threadIdx.x == 0 && !p.trigger_late) pdl_launch_dependents();
    if (!p.wait_late) pdl_wait_prior_grid();
    if (threadIdx.x == 0 && p.trigger_late) pdl_launch_dependents();

    if (warp == 0 || warp == 2) {
        // ------------------------------------------------------- TMA producers: warp 0 loads A, warp 2 loads B
        // Each walks the whole schedule; with one warp for both, the issue loop and not the copies set the pace of narrow tiles.
        const bool for_a = (warp == 0);
        const bool issuer = elect_one_sync();
        // operands that other CTAs read as well stay in L2; with a single tile row B passes through once
        const uint64_t policy = (!for_a && tile_rows == 1) ? kL2EvictFirst : kL2EvictLast;
        const uint32_t bytes = static_cast<uint32_t>(for_a ? a_bytes : b_bytes);
        const uint32_t dst0 = for_a ? smem_base : ring_b;
        const uint32_t peer = (CG == 2) ? mapa_shared(bar_full, 0) - bar_full : 0u;   // the leader's barriers count both CTAs' bytes
        const uint32_t bar_end = bar_full + stages * 8;
        uint32_t dst = dst0, full = bar_full, empty = bar_empty;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = 0, t = first_item; t < num_tiles && ok; t += step(i++)) {
            int tm, tn, split;
            dense_tile(t, tile_rows, p.tiles_n, p.band, tm, tn, split);
            const bool second = tm >= p.tiles_m;                  // tile of the second result
            const int row_a = ((second ? tm - p.tiles_m : tm) * CG + rank) * 128;
            const int row_b = tn * out_cols + (kGated ? 0 : rank * bn_cta);
            int at = split * p.kb_split;
            const int end = min(at + p.kb_split, all_kb);
            int seg = (at >= p.num_kb) ? 1 : 0;
            for (int kb = at - seg * p.num_kb; at < end; ++at, ++kb) {
                if (kb == p.num_kb) { kb = 0; seg = 1; }
                const CUtensorMap* map = for_a ? ((second || seg) ? &tm_a1 : &tm_a0)
                                               : ((seg || (kGated && CG == 2 && rank)) ? &tm_b1 : &tm_b0);
                if (!mbar_wait(empty, phase ^ 1u)) {
                    if (issuer) atomicCAS(p.status, 0, 101);
                    ok = false;
                    break;
                }
                if (issuer) {
                    if (is_leader) mbar_arrive_expect_tx(full, CG * kbs * bytes);
                    const uint32_t bar = full + peer;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        if (u == kbs) break;
                        const int k = kb * kbs + u;             // past the end of K a load brings zeros
                        const uint32_t to = dst + u * bytes;
                        if (for_a) {
                            if constexpr (kAMn) {
                                tma_load<CG>(to, map, bar, row_a * 2, k * 64, policy);
                                tma_load<CG>(to + 8192, map, bar, row_a * 2 + 128, k * 64, policy);
                            } else {
                                tma_load<CG>(to, map, bar, k * 128, row_a, policy);
                            }
                        } else if constexpr (kBMn) {
#pragma unroll
                            for (int c = 0; c < 256 / CG; c += 64)
                                if (c < bn_cta) tma_load<CG>(to + c * 128, map, bar, (row_b + c) * 2, k * 64, policy);
                        } else {
                            tma_load<CG>(to, map, bar, k * 128, row_b, policy);
                            if constexpr (kGated && CG == 1) tma_load<CG>(to + out_cols * 128, &tm_b1, bar, k * 128, row_b, policy);
                        }
                    }
                }
                dst += kbs * bytes;
                full += 8;
                empty += 8;
                if (full == bar_end) { dst = dst0; full = bar_full; empty = bar_empty; phase ^= 1u; }
            }
        }
        // wait until every filled stage has been consumed: no copy or signal is outstanding when the CTA exits
        for (int i = 0; i < stages && ok; ++i) {
            if (!mbar_wait(empty, phase ^ 1u)) {
                if (issuer) atomicCAS(p.status, 0, 101);
                ok = false;
            }
            full += 8;
            empty += 8;
            if (full == bar_end) { full = bar_full; empty = bar_empty; phase ^= 1u; }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------------------- MMA issuer
        if (is_leader) {
            const bool issuer = elect_one_sync();
            // The instruction's columns come in 16s.  Where the tile has 8 fewer it reads on into whatever follows in the ring,
            // as it does for rows of A that are not there: that reaches accumulator columns past the tile's last, which nobody uses.
            const uint32_t idesc = make_idesc_dense(kInt8, kAMn, kBMn, 128 * CG, (p.block_n + 15) / 16 * 16);
            const uint32_t bar_end = bar_full + stages * 8;
            uint32_t sa = smem_base, sb = ring_b, full = bar_full, empty = bar_empty;
            uint32_t phase = 0;
            int tile_iter = 0;
            bool ok = true;
            for (int t = first_item; t < num_tiles && ok; t += step(tile_iter++)) {
                const int acc = tile_iter & 1;
                const uint32_t acc_phase = static_cast<uint32_t>(tile_iter >> 1) & 1u;
                if (!mbar_wait(bar_tempty + acc * 8, acc_phase ^ 1u)) {
                    if (issuer) atomicCAS(p.status, 0, 102);
                    ok = false;
                    break;
                }
                tcgen05_fence_after();
                const uint32_t d_tmem = tmem_base + acc * 256;
                int tm, tn, split;
                dense_tile(t, tile_rows, p.tiles_n, p.band, tm, tn, split);
                const int steps = min(p.kb_split, all_kb - split * p.kb_split);
                for (int i = 0; i < steps; ++i) {
                    if (!mbar_wait(full, phase)) {
                        if (issuer) atomicCAS(p.status, 0, 102);
                        ok = false;
                        break;
                    }
                    tcgen05_fence_after();
                    if (issuer) {
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            if (u == kbs) break;
                            const uint32_t ua = sa + u * a_bytes, ub = sb + u * b_bytes;
                            const uint64_t a_desc = kAMn ? make_smem_desc(ua, 8192, 1024, 2) : make_desc_k_sw128(ua);
                            const uint64_t b_desc = kBMn ? make_smem_desc(ub, 8192, 1024, 2) : make_desc_k_sw128(ub);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                // descriptor addresses count 16 bytes: a K step is 32 bytes along a K-major row, or 16 K rows
                                // (2 KB) of an MN-major tile
                                const uint64_t ad = a_desc + static_cast<uint64_t>(j * (kAMn ? 128 : 2));
                                const uint64_t bd = b_desc + static_cast<uint64_t>(j * (kBMn ? 128 : 2));
                                const uint32_t accumulate = (i > 0 || u > 0 || j > 0) ? 1u : 0u;
                                if constexpr (kInt8) mma_int8<CG>(d_tmem, ad, bd, idesc, accumulate);
                                else mma_bf16<CG>(d_tmem, ad, bd, idesc, accumulate);
                            }
                        }
                        tcgen05_commit<CG>(empty);
                    }
                    sa += kbs * a_bytes;
                    sb += kbs * b_bytes;
                    full += 8;
                    empty += 8;
                    if (full == bar_end) { sa = smem_base; sb = ring_b; full = bar_full; empty = bar_empty; phase ^= 1u; }
                }
                if (ok && issuer) tcgen05_commit<CG>(bar_tfull + acc * 8);
                __syncwarp();
            }
        }
    } else {
        // --------------------------------------------------------------- epilogue
        const int quad = warp & 3;             // TMEM lane quadrant this warp may access
        const int part = (warp - 3) >> 2;      // of the 2 or 4 warps of a quadrant, which take groups of 32 result columns in turn
        const int parts = epi_warps >> 2;
        const uint32_t sbuf = smem_base + Cfg::kOffEpi + (warp - 3) * Cfg::kEpiBufBytes;
        const uint32_t tempty0 = (CG == 2) ? mapa_shared(bar_tempty, 0) : bar_tempty;
        const int results = (kGated && p.gate != nullptr) ? 3 : 1;
        int tile_iter = 0;
        for (int t = first_item; t < num_tiles; t += step(tile_iter++)) {
            int tm, tn, split;
            dense_tile(t, tile_rows, p.tiles_n, p.band, tm, tn, split);
            const bool second = tm >= p.tiles_m;
            const int acc = tile_iter & 1;
            const uint32_t acc_phase = static_cast<uint32_t>(tile_iter >> 1) & 1u;
            const int row0 = ((second ? tm - p.tiles_m : tm) * CG + rank) * 128 + quad * 32;
            const int col0 = tn * out_cols;
            float sa = 1.0f;
            // the row's scale and the first columns' scales and bias come while the products still run
            if constexpr (kInt8) sa = (row0 + lane < p.m) ? load_f32(p.a_scale + row0 + lane) : 0.0f;
            ColumnTerms<kInt8, EPI> terms;
            load_terms(terms, p.b_scale[0], p.b_scale[1], p.bias, col0 + part * 32, p.n);
            if (!mbar_wait(bar_tfull + acc * 8, acc_phase)) {
                if (lane == 0) atomicCAS(p.status, 0, 103);
                break;
            }
            tcgen05_fence_after();
            const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + acc * 256;
            if (p.splits > 1) {
                // sums of a K range, 16 columns (64 bytes) at a time
                constexpr int kSlabs = kGated ? 2 : 1;
                for (int slab = 0; slab < kSlabs; ++slab) {
                    uint32_t* base = p.partial + static_cast<long long>(split * (kGated ? 2 : p.batches) + (kGated ? slab : second ? 1 : 0)) * p.m * p.n;
                    for (int c0 = part * 16; c0 < out_cols; c0 += parts * 16) {
                        uint32_t v[16];
                        tmem_ld_32x32b_x16(t_acc + slab * out_cols + c0, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int q = 0; q < 4; ++q) stage_piece(sbuf, lane, q, v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                        __syncwarp();
                        const int c = c0 + (lane & 3) * 4;
                        const bool col_ok = (c < out_cols) && (col0 + c < p.n);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int rr = i * 8 + (lane >> 2);
                            const uint4 w = staged_piece(sbuf, rr, lane & 3);
                            if (col_ok && row0 + rr < p.m) *reinterpret_cast<uint4*>(base + static_cast<long long>(row0 + rr) * p.n + col0 + c) = w;
                        }
                        __syncwarp();
                    }
                }
            } else {
                for (int c0 = part * 32; c0 < out_cols; c0 += parts * 32) {
                    const int c1 = min(c0 + 32, out_cols);
                    for (int r = 0; r < results; ++r) {
                        // 32 rows x up to 32 columns through a transpose in shared memory, so that a row's part of the result is
                        // stored by neighbouring lanes.  Or directly, in whole 32-byte sectors: at the tensor pipe's full rate its
                        // operands take all of shared memory's 128 bytes a clock, and the transpose slows it down.  int8 with gelu_tanh and
                        // bias, transposed / direct, us: 2048 x 8192 x 1024 25.9 / 24.3 (at 1.9 GHz), 8192 x 8192 x 512 76 / 72, 8192 x 8192 x 1024
                        // 82.7 / 78.9 (63.3 / 65.1 without an activation), 8192^3 the same; gated int8 4096 x 8192 x 1024 56.5 / 55.8, gated
                        // bf16 4096 x 16384 x 4096 805 / 808, and gradients of 512 x 8192 x 8192, bound by writing, 110 / 117, so the
                        // others keep to the transpose.
#pragma unroll 1
                        for (int c = c0; c < c1; c += 16) {
                            uint32_t v[16], u[16], w[8];
                            tmem_ld_32x32b_x16(t_acc + c + ((kGated && r == 2) ? out_cols : 0), v);
                            if (kGated && r == 0) tmem_ld_32x32b_x16(t_acc + out_cols + c, u);
                            tmem_ld_wait();
                            if (EPI == kDensePlain || r > 0) {
                                dense_convert<false, kDensePlain, AVE_FP4_ACT_NONE>(v, v, w, sa, ColumnTerms<false, kDensePlain>{});
                            } else {
                                switch (p.act) {   // warp-uniform
                                    case AVE_FP4_ACT_RELU: dense_convert<kInt8, EPI, AVE_FP4_ACT_RELU>(v, u, w, sa, terms); break;
                                    case AVE_FP4_ACT_GELU: dense_convert<kInt8, EPI, AVE_FP4_ACT_GELU>(v, u, w, sa, terms); break;
                                    case AVE_FP4_ACT_GELU_TANH: dense_convert<kInt8, EPI, AVE_FP4_ACT_GELU_TANH>(v, u, w, sa, terms); break;
                                    case AVE_FP4_ACT_SILU: dense_convert<kInt8, EPI, AVE_FP4_ACT_SILU>(v, u, w, sa, terms); break;
                                    default: dense_convert<kInt8, EPI, AVE_FP4_ACT_NONE>(v, u, w, sa, terms); break;
                                }
                            }
                            if constexpr (kInt8) {      // the next 16 columns' terms: in this group, or the first of the next one
                                const int next = (c + 16 < c1) ? c + 16 : c0 + parts * 32;
                                load_terms(terms, p.b_scale[0], p.b_scale[1], p.bias, col0 + next, p.n);
                            }
                            if constexpr (EPI == kDenseScaled) {
                                if (p.direct) {
                                    const int col = col0 + c;
                                    __nv_bfloat16* at = p.d[0] + (row0 + lane) * p.ldd + col;
                                    if (row0 + lane < p.m) {
                                        if (col + 16 <= p.n) store_16(at, w);
                                        else if (col < p.n) *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
                                    }
                                    continue;
                                }
                            }
                            const int q0 = (c - c0) / 8;
#pragma unroll
                            for (int q = 0; q < 2; ++q) stage_piece(sbuf, lane, q0 + q, w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
                        }
                        if (EPI == kDenseScaled && p.direct) continue;
                        __syncwarp();
                        __nv_bfloat16* d = p.d[second ? 1 : 0];
                        long long ld = p.ldd;
                        if (kGated && r == 1) { d = p.gate; ld = p.ld_gate; }
                        if (kGated && r == 2) { d = p.up; ld = p.ld_up; }
                        const int c = c0 + (lane & 3) * 8;
                        const bool col_ok = (c < c1) && (col0 + c < p.n);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int rr = i * 8 + (lane >> 2);
                            const uint4 w = staged_piece(sbuf, rr, lane & 3);
                            if (col_ok && row0 + rr < p.m) __stcs(reinterpret_cast<uint4*>(d + (row0 + rr) * ld + col0 + c), w);
                        }
                        __syncwarp();
                    }
                }
            }
            tcgen05_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2) mbar_arrive_cluster(tempty0 + acc * 8);
                else mbar_arrive(bar_tempty + acc * 8);
            }
        }
    }

    if (p.wait_late) pdl_wait_prior_grid();
    tcgen05_fence_before();
    __syncthreads();
    if constexpr (CG == 2) cluster_sync_all();
    if (warp == 1) tmem_dealloc<CG>(tmem_base, 512);
}

// Adds up the K ranges of up to three plain results and rounds once: one thread takes 8 columns of a row.
struct SplitSum {
    const uint32_t* partial;     // first range; `stride` words to the next
    long long stride;
    __nv_bfloat16* d;
    long long ldd;
    long long pieces;            // rows * n / 8
    int n8;                      // n / 8
    int splits;
};
struct SplitSums {
    SplitSum job[3];
};

// 8 columns of a K range added to the sums so far
template <bool INT8>
__device__ __forceinline__ void add_range(uint32_t (&acc)[8], const uint32_t* src) {
    const uint4 lo = load_16<true>(src), hi = load_16<true>(src + 4);
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (INT8) acc[i] += w[i];
        else acc[i] = __float_as_uint(__uint_as_float(acc[i]) + __uint_as_float(w[i]));
    }
}

__global__ void __launch_bounds__(256)
sum_splits_kernel(const SplitSums p) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
#pragma unroll 1
    for (int j = 0; j < 3; ++j) {
        const SplitSum& s = p.job[j];
        for (long long i = blockIdx.x * 256ll + threadIdx.x; i < s.pieces; i += gridDim.x * 256ll) {
            uint32_t acc[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
            for (int r = 0; r < s.splits; ++r) add_range<false>(acc, s.partial + r * s.stride + i * 8);
            const long long row = i / s.n8;
            const long long col = (i - row * s.n8) * 8;
            uint32_t w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) w[c] = pack_bf16(__uint_as_float(acc[2 * c]), __uint_as_float(acc[2 * c + 1]));
            *reinterpret_cast<uint4*>(s.d + row * s.ldd + col) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
}

// The same for a scaled or gated result, with the tile kernel's epilogue.  That takes 16 columns; a thread here has 8, and the other
// half of its work falls away in the compiler.
template <bool INT8, int EPI>
__global__ void __launch_bounds__(256)
finish_splits_kernel(const DenseParams p) {
    pdl_launch_dependents();
    pdl_wait_prior_grid();
    const int n8 = p.n / 8;
    const long long pieces = static_cast<long long>(p.m) * n8;
    const long long slab = static_cast<long long>(p.m) * p.n;
    for (long long i = blockIdx.x * 256ll + threadIdx.x; i < pieces; i += gridDim.x * 256ll) {
        const int row = static_cast<int>(i / n8);
        const int col = static_cast<int>(i - static_cast<long long>(row) * n8) * 8;
        uint32_t g[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u}, u[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
        for (int r = 0; r < p.splits; ++r) {
            const uint32_t* src = p.partial + (EPI == kDenseGated ? 2 * r : r) * slab + i * 8;
            add_range<INT8>(g, src);
            if constexpr (EPI == kDenseGated) add_range<INT8>(u, src + slab);
        }
        const float sa = INT8 ? load_f32(p.a_scale + row) : 1.0f;
        ColumnTerms<INT8, EPI> terms;
        load_terms(terms, p.b_scale[0], p.b_scale[1], p.bias, col, p.n);
        uint32_t v16[16], u16[16], w[8];
#pragma unroll
        for (int c = 0; c < 16; ++c) { v16[c] = g[c & 7]; u16[c] = u[c & 7]; }
        switch (p.act) {
            case AVE_FP4_ACT_RELU: dense_convert<INT8, EPI, AVE_FP4_ACT_RELU>(v16, u16, w, sa, terms); break;
            case AVE_FP4_ACT_GELU: dense_convert<INT8, EPI, AVE_FP4_ACT_GELU>(v16, u16, w, sa, terms); break;
            case AVE_FP4_ACT_GELU_TANH: dense_convert<INT8, EPI, AVE_FP4_ACT_GELU_TANH>(v16, u16, w, sa, terms); break;
            case AVE_FP4_ACT_SILU: dense_convert<INT8, EPI, AVE_FP4_ACT_SILU>(v16, u16, w, sa, terms); break;
            default: dense_convert<INT8, EPI, AVE_FP4_ACT_NONE>(v16, u16, w, sa, terms); break;
        }
        *reinterpret_cast<uint4*>(p.d[0] + row * p.ldd + col) = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (EPI == kDenseGated && !INT8) {
            if (p.gate != nullptr) {
                dense_convert<false, kDensePlain, AVE_FP4_ACT_NONE>(v16, v16, w, 1.0f, ColumnTerms<false, kDensePlain>{});
                *reinterpret_cast<uint4*>(p.gate + row * p.ld_gate + col) = make_uint4(w[0], w[1], w[2], w[3]);
                dense_convert<false, kDensePlain, AVE_FP4_ACT_NONE>(u16, u16, w, 1.0f, ColumnTerms<false, kDensePlain>{});
                *reinterpret_cast<uint4*>(p.up + row * p.ld_up + col) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

}  // namespace avefp4
