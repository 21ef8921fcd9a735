// Host side of include/ave_dense.h: argument checks, tile choice and launches of the integer, gated and gradient kernels.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <cstring>

#include "../../include/ave_dense.h"
#include "gated_backward.cuh"
#include "gemm_dense_sm100.cuh"
#include "gemm_stream_sm100.cuh"
#include "host_shared.h"
#include "quantize_int8.cuh"

namespace {

using namespace avefp4;

int fail(const char* fmt, ...) {
    char text[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof(text), fmt, ap);
    va_end(ap);
    return host_fail(-AVE_FP4_ERR_ARG, text);
}

#define AVE_CUDA(call)                                              \
    do {                                                            \
        cudaError_t e__ = (call);                                   \
        if (e__ != cudaSuccess) return host_fail_cuda(e__, #call);  \
    } while (0)

constexpr int64_t kMaxDim = int64_t(1) << 28;     // keeps byte coordinates of a tensor map inside 32 bits

bool sizes_ok(int64_t a, int64_t b, int64_t c) {
    return a >= 0 && b >= 0 && c >= 0 && a <= kMaxDim && b <= kMaxDim && c <= kMaxDim;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A row-major matrix of `elem`-byte elements: pointer and row stride on 16 bytes, rows not overlapping.
int check_matrix(const char* fn, const char* name, const void* p, int64_t rows, int64_t cols, int64_t ld, int elem) {
    if (p == nullptr || !aligned16(p)) return fail("%s: %s is null or not 16-byte aligned", fn, name);
    if (rows > 1 && (ld < cols || ld % (16 / elem) != 0 || ld > (int64_t(1) << 36)))
        return fail("%s: the row stride of %s must be at least %lld and a multiple of %d, got %lld", fn, name, static_cast<long long>(cols),
                    16 / elem, static_cast<long long>(ld));
    return 0;
}

int check_vector(const char* fn, const char* name, const void* p) {
    if (p == nullptr || !aligned16(p)) return fail("%s: %s is null or not 16-byte aligned", fn, name);
    return 0;
}

int check_workspace(const char* fn, const void* workspace, int64_t have, int64_t need) {
    if (need > 0 && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0 || have < need))
        return fail("%s: the workspace must be 256-byte aligned and hold %lld bytes", fn, static_cast<long long>(need));
    return 0;
}

int check_activation(const char* fn, int act) {
    if (act < AVE_FP4_ACT_NONE || act > AVE_FP4_ACT_SILU) return fail("%s: unknown activation %d", fn, act);
    return 0;
}

int64_t row_stride(int64_t rows, int64_t cols, int64_t ld) { return rows > 1 ? ld : cols; }

// Launch attributes: CTA pairs, and the next kernel's launch and set-up under this one's tail (each kernel here waits for the
// previous grid on the device before it touches global memory).
struct Launch {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    Launch(int64_t grid, int threads, size_t smem, int cluster, cudaStream_t stream) {
        memset(&cfg, 0, sizeof(cfg));
        cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
        cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = cluster > 1 ? 2 : 1;
    }
};

// ------------------------------------------------------------------------------- tile kernel
struct Operand {
    const void* p;
    int64_t ld;
};

// What a launch of the tile kernel is made of.
struct DensePlan {
    int cg;          // CTAs of a tile
    int block_n;
    int splits;      // ranges of K, of kb_split stages each (the last may be shorter)
    int kb_split;
    int a_rows, b_rows, kb_stage, stages;
    int64_t items;   // tiles times ranges
    int64_t clk;     // estimate of one
    int64_t sums;    // estimate of writing and reading the ranges' sums
    int sms;         // SMs it runs on
    int early, early_items;      // of the second product of a backward pass: see DenseParams
};

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Tile width, CTA pairs or single CTAs, and cuts of K: the smallest estimate of the launch's time, in SM clocks.
//
// A K block of 128 bytes per row takes a CTA the longest of: 2 block_n clocks of the tensor pipe (128 rows, 4 instructions);
// 2 (a_rows + b_rows) to bring the operands from L2 (64 bytes a clock, what 256 x 256 tiles sustain on all SMs); 140 of issue;
// and with one tile row, whose weights come from memory, the share of 3400 bytes a clock (less by up to a seventh with SMs
// left out), at most 40 of them for one SM.  Work comes in waves of all CTAs.  Cutting K into S ranges costs writing and reading S fp32
// results (2600 bytes a clock) and a launch.  Against sweeps of widths and cuts at 27 sizes the choice was within 14 % of
// the best one, within 5 % for most.
//
// each_plan calls f(plan) for every tile width, CTA pairs or not and number of ranges.
constexpr int64_t kSumsLaunch = 5500;

template <class F>
void each_plan(int sms, int64_t m, int64_t cols, int64_t k_bytes, int segments, int batches, bool a_mn, bool b_mn, bool gated, bool may_split,
               F f) {
    for (int cg = (m <= 128 ? 1 : 2); cg >= 1; --cg) {
        const int64_t clusters = sms / cg;
        const int64_t tile_rows = ceil_div(m, 128 * cg) * batches;
        const int a_rows = (a_mn || m >= 128) ? 128 : static_cast<int>(ceil_div(m, 8) * 8);
        const int step = cg == 2 ? 32 : gated ? 16 : 8;
        for (int bn = 256; bn >= 32; bn -= step) {
            const int b_rows = b_mn ? static_cast<int>(ceil_div(bn / cg, 64) * 64) : bn / cg;
            const int64_t tiles = tile_rows * ceil_div(cols, bn);
            int64_t clk = 2 * bn;
            if (2 * (a_rows + b_rows) > clk) clk = 2 * (a_rows + b_rows);
            if (clk < 140) clk = 140;
            if (tile_rows == 1) {
                const int64_t active = (tiles < clusters ? tiles : clusters) * cg;
                const int64_t rate = 2900 + 500 * active / sms;
                const int64_t all = b_rows * 128 * active / rate, one = b_rows * 128 / 40;
                if (all > clk) clk = all;
                if (one > clk) clk = one;
            }
            const int kbs = bn <= 128 ? 2 : 1;
            const int64_t steps = ceil_div(k_bytes, 128 * kbs) * segments;
            for (int64_t splits = 1; splits <= (may_split ? 8 : 1) && splits <= steps; ++splits) {
                if (splits > 1 && tiles * (splits - 1) >= clusters) break;       // a wave is full without more of them
                const int64_t kb_split = ceil_div(steps, splits);
                const int64_t ranges = ceil_div(steps, kb_split);
                f(DensePlan{cg, bn, static_cast<int>(ranges), static_cast<int>(kb_split), a_rows, b_rows, kbs,
                            DenseConfig::stages(a_rows, b_rows, kbs), tiles * ranges, kb_split * kbs * clk + 400,
                            ranges > 1 ? ranges * m * batches * cols * 8 / 2600 : 0, sms, 0, 0});
            }
        }
    }
}

int64_t launch_clocks(const DensePlan& p) {
    return ceil_div(p.items, p.sms / p.cg) * p.clk + (p.splits > 1 ? p.sums + kSumsLaunch : 0);
}

DensePlan plan_dense(int sms, int64_t m, int64_t cols, int64_t k_bytes, bool gated, bool may_split) {
    DensePlan best{};
    int64_t best_cost = INT64_MAX;
    each_plan(sms, m, cols, k_bytes, 1, 1, false, false, gated, may_split, [&](const DensePlan& p) {
        const int64_t cost = launch_clocks(p);
        if (cost < best_cost) {
            best_cost = cost;
            best = p;
        }
    });
    return best;
}

template <int OP>
constexpr int64_t elem_bytes() { return OP == kOpInt8 ? 1 : 2; }

// Forward products cut K only from here on: below they ask for no workspace, and a caller need not ask.
bool forward_may_cut(int64_t m, int64_t k_bytes) { return m > 8 && k_bytes >= AVE_DENSE_MIN_CUT_BYTES; }

// A plan depends on the sizes alone and takes as long to find as a small product runs, a few microseconds: each host thread keeps the
// last ones it made, in slots by a hash of the sizes.
constexpr int kPlanSlots = 64;

int plan_slot(int64_t m, int64_t n, int64_t k) {
    const uint64_t h = (static_cast<uint64_t>(m) * 0x9E3779B97F4A7C15ull) ^ (static_cast<uint64_t>(n) * 0xC2B2AE3D27D4EB4Full) ^ static_cast<uint64_t>(k);
    return static_cast<int>(((h * 0xD6E8FEB86659FD93ull) >> 32) % kPlanSlots);
}

// A forward product's plan.
template <int OP, int EPI>
DensePlan plan_for(const HostDevice& dev, int64_t m, int64_t n, int64_t k) {
    struct Slot {
        int64_t m, n, k;
        int sms;
        DensePlan plan;
    };
    thread_local Slot slots[kPlanSlots] = {};
    Slot& slot = slots[plan_slot(m, n, k)];
    if (slot.m != m || slot.n != n || slot.k != k || slot.sms != dev.sm_count) {
        slot.plan = plan_dense(dev.sm_count, m, EPI == kDenseGated ? 2 * n : n, k * elem_bytes<OP>(), EPI == kDenseGated, forward_may_cut(m, k * elem_bytes<OP>()));
        slot.m = m;
        slot.n = n;
        slot.k = k;
        slot.sms = dev.sm_count;
    }
    return slot.plan;
}

template <int CG, int OP, int EPI>
int launch_dense_cg(const HostDevice& dev, const DensePlan& plan, const Operand (&a)[2], const Operand (&b)[2], int64_t m, int64_t n, int64_t k,
                    DenseParams p, cudaStream_t stream) {
    using Cfg = DenseConfig;
    constexpr bool kAMn = (OP == kOpBf16Tn), kBMn = (OP == kOpBf16Nn || OP == kOpBf16Tn);
    constexpr int64_t kElem = elem_bytes<OP>();
    const int out_cols = (EPI == kDenseGated) ? plan.block_n / 2 : plan.block_n;
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.block_n = plan.block_n;
    p.a_rows = plan.a_rows;
    p.b_rows = plan.b_rows;
    p.kb_stage = plan.kb_stage;
    p.stages = plan.stages;
    p.splits = plan.splits;
    p.kb_split = plan.kb_split;
    p.num_kb = static_cast<int>(ceil_div(k * kElem, 128 * plan.kb_stage));
    p.tiles_m = static_cast<int>(ceil_div(m, 128 * CG));
    p.tiles_n = static_cast<int>(ceil_div(n, out_cols));
    // Tile rows of a band: their A panels, some 32 MB, stay in L2 while the band goes through B.  Back to back under the power cap,
    // bands of 8 / 16 rows: int8 8192^3 391 / 379 us, gated int8 4096 x 28672 x 8192 1288 / 1266, gated bf16 4096 x 16384 x 4096 840 /
    // 814, 8192^3 1640 / 1698; the gradients of 8192 x 4096 x 16384 (operands as they lie in memory) 1627 / 1666.
    p.band = kBMn ? 8 : static_cast<int>((int64_t(32) << 20) / (128 * CG * k * kElem));
    if (p.band < 8) p.band = 8;
    if (p.band > 16) p.band = 16;
    p.direct = EPI == kDenseScaled && out_cols % 16 == 0 && p.ldd % 16 == 0 && (reinterpret_cast<uintptr_t>(p.d[0]) & 31u) == 0;
    p.status = dev.status;

    CUtensorMap ta[2], tb[2];
    const int b_box = (EPI == kDenseGated) ? out_cols : plan.block_n / CG;
    for (int i = 0; i < 2; ++i) {
        int rc;
        if (kAMn) rc = host_encode_bytes(&ta[i], a[i].p, m * kElem, k, a[i].ld * kElem, 64, "A");
        else rc = host_encode_bytes(&ta[i], a[i].p, k * kElem, m, a[i].ld * kElem, p.a_rows, "A");
        if (rc) return rc;
        if (kBMn) rc = host_encode_bytes(&tb[i], b[i].p, n * kElem, k, b[i].ld * kElem, 64, "B");
        else rc = host_encode_bytes(&tb[i], b[i].p, k * kElem, n, b[i].ld * kElem, b_box, "B");
        if (rc) return rc;
    }
    const int64_t items = int64_t(p.tiles_m) * p.batches * p.tiles_n * p.splits;
    const int64_t clusters = plan.sms / CG;
    // 16 epilogue warps hide more latency (int8 8192 x 8192 x 1024 78 -> 63 us), 8 start sooner (64 x 64 x 64 3.6 against 4.0 us):
    // tiles of up to 64 result columns keep two warps of a quadrant busy and no more, and the plain epilogue is short.
    const int threads = Cfg::threads(EPI != kDensePlain && out_cols > 64 ? 16 : 8);
    Launch launch((items < clusters ? items : clusters) * CG, threads, Cfg::kSmemBytes, CG, stream);
    AVE_CUDA(cudaLaunchKernelEx(&launch.cfg, gemm_dense_kernel<CG, OP, EPI>, ta[0], ta[1], tb[0], tb[1], p));
    return 0;
}

// a[1] / b[1]: second operand of two segments, two results, or the second weight of the gated form
template <int OP, int EPI>
int launch_dense(const HostDevice& dev, const DensePlan& plan, const Operand (&a)[2], const Operand (&b)[2], int64_t m, int64_t n, int64_t k,
                 const DenseParams& p, cudaStream_t stream) {
    if (plan.cg == 1) return launch_dense_cg<1, OP, EPI>(dev, plan, a, b, m, n, k, p, stream);
    return launch_dense_cg<2, OP, EPI>(dev, plan, a, b, m, n, k, p, stream);
}

// Two products in a row, the second of which needs nothing of the first (DenseParams::wait_late): it starts on the SMs that the
// first one's last wave leaves out, one of the first one's items ahead of the rest.  How many tiles those clusters take before the
// rest is dealt out to all: what ends the launch soonest.
// A tile of the second product takes its products' time or, with a short sum, its share of writing the result: 2100 bytes a clock,
// 4.1 TB/s (without the latter 64x8192x8192 went from 62 to 92 us).
// Returns the clocks from the start of the first one's last wave on.
int64_t deal_early(int sms, const DensePlan& first, DensePlan& second) {
    const int64_t clusters = sms / first.cg, grid = sms / second.cg;
    const int64_t rest = first.items % clusters;
    const int64_t early = rest == 0 ? 0 : (clusters - rest) * first.cg / second.cg;
    const int64_t active = second.items < grid ? second.items : grid;
    const int64_t write = int64_t(128) * second.cg * second.block_n * (second.splits > 1 ? 4 : 2) * active / 2100;
    const int64_t clk = second.clk > write ? second.clk : write;
    second.early = second.early_items = 0;
    if (second.items <= early) return first.clk > clk ? first.clk : clk;
    int64_t best = first.clk + ceil_div(second.items, grid) * clk;
    if (early == 0 || early >= grid || second.items <= grid) return best;
    for (int64_t ahead = 1; ahead <= first.clk / clk + 1 && ahead * early < second.items; ++ahead) {
        const int64_t left = second.items - ahead * early, rounds = left / grid, more = left % grid;
        const int64_t late_end = first.clk + (rounds + (more > 0 ? 1 : 0)) * clk;
        const int64_t early_end = (ahead + rounds + (more > grid - early ? 1 : 0)) * clk;
        const int64_t end = late_end > early_end ? late_end : early_end;
        if (end < best) {
            best = end;
            second.early_items = static_cast<int>(ahead);
            second.early = static_cast<int>(early);
        }
    }
    return best;
}

// Plans of two such products, found together: what the first leaves idle the second fills, so a cut of the first one's K that would
// pay for it alone often does not.  And plans of each alone, with the same ranges of K: a gradient's bits do not depend on
// whether the other is asked for.
struct PairPlan {
    DensePlan first, second, first_alone, second_alone;
};

// Choices for one of them: for every number of ranges, the ones that take the least time alone.
struct PlanChoices {
    static constexpr int kEach = 4;
    DensePlan plan[8][kEach];
    int64_t cost[8][kEach];
    int count[8] = {};

    void add(const DensePlan& p) {
        const int64_t c = launch_clocks(p);
        DensePlan(&plans)[kEach] = plan[p.splits - 1];
        int64_t(&costs)[kEach] = cost[p.splits - 1];
        int& n = count[p.splits - 1];
        if (n == kEach && c >= costs[kEach - 1]) return;
        int at = n < kEach ? n++ : kEach - 1;
        for (; at > 0 && costs[at - 1] > c; --at) {
            costs[at] = costs[at - 1];
            plans[at] = plans[at - 1];
        }
        costs[at] = c;
        plans[at] = p;
    }
    template <class F>
    void each(F f) const {
        for (int s = 0; s < 8; ++s)
            for (int i = 0; i < count[s]; ++i) f(plan[s][i]);
    }
};

// Both products in turn, each planned alone / both together, us: gated backward 1003x2744x1048 41.5 / 36.9, 1144x1040x216 21.6 / 17.7,
// product gradients 744x7384x248 21.5 / 16.0, 6480x584x216 19.8 / 13.7; the worst of 220 sizes 880x1800x160 11.1 / 12.3, on average
// 1.7 % less.  Left as planned alone: what memory bounds for half of the time or more (8x11504x2264 31 / 43, for all SMs share that
// however the tiles lie), and what would gain less than 5 % by the estimate (gated backward 2048x4096x1024 69 / 73).
// Where memory bounds the products of a few rows, one of which reads the weights and the other writes their gradients, they run
// beside each other, each on half of the SMs: copying goes at 6.2 TB/s, writing alone at 4.  The second's CTAs are single ones, for
// pairs find no two free neighbours, and take 85 % of its tiles before the first is done.  One after the other / beside each other,
// us: product gradients 64x8192x8192 61 / 54, 64x4096x4096 25.9 / 19.9, 32x20064x4048 72.5 / 67; gated backward 16x14336x4096 104 / 93,
// 64x4096x4096 38.6 / 36.4; with two tile rows, 256x8192x8192 73.9 / 75.1, not.  Ranges that suit half of the SMs and cost the product
// far more when it is asked for alone (32x20064x4048 30 / 47) give way to those it would have alone.
//
// C0 = A B with m0 x n0 results over `segments` sums of length k0, and C1 = A^T B with `batches` results of m1 x n1 and sums of length k1
PairPlan plan_pair(int sms, int64_t m0, int64_t n0, int64_t k0, int segments, int64_t m1, int64_t n1, int64_t k1, int batches) {
    auto each_first = [&](int on, auto f) { each_plan(on, m0, n0, 2 * k0, segments, 1, false, true, false, true, f); };
    auto each_second = [&](auto f) { each_plan(sms, m1, n1, 2 * k1, 1, batches, true, true, false, true, f); };
    auto take = [](DensePlan& least, const DensePlan& p) { if (least.cg == 0 || launch_clocks(p) < launch_clocks(least)) least = p; };
    // (a segment of an odd number of K blocks ends inside a stage of two)
    const bool odd = segments == 2 && ceil_div(k0, 64) % 2 != 0;
    auto same_ranges = [odd](const DensePlan& p, const DensePlan& q) {
        if (odd && p.splits > 1 && p.kb_stage != q.kb_stage) return false;
        return p.splits == q.splits && (p.splits == 1 || p.kb_stage * p.kb_split == q.kb_stage * q.kb_split);
    };
    auto together = [&](const DensePlan& first, DensePlan& second) {
        return (ceil_div(first.items, sms / first.cg) - 1) * first.clk + first.sums + deal_early(sms, first, second) + second.sums +
               (first.splits > 1 || second.splits > 1 ? kSumsLaunch : 0);
    };
    PairPlan best{};
    PlanChoices a, b;
    each_first(sms, [&](const DensePlan& p) { a.add(p); take(best.first, p); });
    each_second([&](const DensePlan& p) { b.add(p); take(best.second, p); });
    const int64_t memory = 2 * segments * k0 * (m0 + n0) / 3300 + 2 * (m0 * n0 + batches * m1 * n1) / 2100;
    const bool by_memory = 2 * memory > launch_clocks(best.first) + launch_clocks(best.second);
    if (by_memory && m0 <= 128) {
        const int half = sms / 2;
        const DensePlan whole = best.first;
        DensePlan alone{};
        best.first = DensePlan{};
        each_first(half, [&](const DensePlan& p) { take(best.first, p); });
        each_first(sms, [&](const DensePlan& p) { if (same_ranges(p, best.first)) take(alone, p); });
        if (launch_clocks(alone) * 10 > launch_clocks(whole) * 13) {      // ranges that would cost it too much alone
            best.first = whole;
            best.first.sms = half;
            each_first(half, [&](const DensePlan& p) { if (same_ranges(p, whole)) take(best.first, p); });
        }
        best.second = DensePlan{};
        each_second([&](const DensePlan& p) { if (p.cg == 1) take(best.second, p); });
        best.second.early_items = static_cast<int>(best.second.items * 85 / 100 / (sms - half));
        best.second.early = best.second.early_items > 0 ? sms - half : 0;
    } else {
        int64_t best_cost = together(best.first, best.second) * 19 / 20;
        if (!by_memory) a.each([&](const DensePlan& first) {
            b.each([&](const DensePlan& choice) {
                DensePlan second = choice;
                const int64_t cost = together(first, second);
                if (cost < best_cost) {
                    best_cost = cost;
                    best.first = first;
                    best.second = second;
                }
            });
        });
    }
    each_first(sms, [&](const DensePlan& p) { if (same_ranges(p, best.first)) take(best.first_alone, p); });
    each_second([&](const DensePlan& p) { if (same_ranges(p, best.second)) take(best.second_alone, p); });
    return best;
}

// As plan_for: found once for a size and kept by each host thread, those of gated blocks and of products in slots of their own.
const PairPlan& pair_for(const HostDevice& dev, int64_t m, int64_t n, int64_t k, bool gated) {
    struct Slot {
        int64_t m, n, k;
        int sms;
        PairPlan plan;
    };
    thread_local Slot slots[2][kPlanSlots] = {};
    Slot& slot = slots[gated ? 1 : 0][plan_slot(m, n, k)];
    if (slot.m != m || slot.n != n || slot.k != k || slot.sms != dev.sm_count) {
        // gated: dX (m, k) = dG Wg + dU Wu over n, dWg and dWu (n, k) over m; else dA (m, k) over n and dB (n, k) over m
        slot.plan = plan_pair(dev.sm_count, m, k, n, gated ? 2 : 1, n, k, m, gated ? 2 : 1);
        slot.m = m;
        slot.n = n;
        slot.k = k;
        slot.sms = dev.sm_count;
    }
    return slot.plan;
}

int64_t split_words(const DensePlan& plan, int64_t rows, int64_t n) { return plan.splits > 1 ? plan.splits * rows * n : 0; }

SplitSum split_sum(const DensePlan& plan, const uint32_t* partial, int64_t stride, void* d, int64_t ldd, int64_t rows, int64_t n) {
    return SplitSum{partial, stride, static_cast<__nv_bfloat16*>(d), ldd, plan.splits > 1 ? rows * n / 8 : 0, static_cast<int>(n / 8), plan.splits};
}

int launch_sums(const HostDevice& dev, const SplitSums& sums, cudaStream_t stream) {
    int64_t most = 0;
    for (const SplitSum& s : sums.job) if (s.pieces > most) most = s.pieces;
    if (most == 0) return 0;
    int64_t grid = ceil_div(most, 256);
    if (grid > int64_t(dev.sm_count) * 8) grid = int64_t(dev.sm_count) * 8;
    Launch launch(grid, 256, 0, 1, stream);
    AVE_CUDA(cudaLaunchKernelEx(&launch.cfg, sum_splits_kernel, sums));
    return 0;
}

// The streaming kernel works in units of 16 weight rows, of about a microsecond each however short K is, and takes K in steps of
// 4 KB; the tile kernel needs a long K to fill its pipeline, and does without either.  us, streaming / tile: int8 1 x 1600 x 8192
// 5.7 / 11.6, 1 x 4800 x 8192 11.3 / 12.4, 1 x 9600 x 8192 17.7 / 17.3, 1 x 28672 x 4096 24.2 / 23.1, 6 x 28672 x 6144 37.6 / 32.2,
// 1 x 28672 x 8192 39.2 / 42.3, gated 1 x 28672 x 8192 72 / 77.  So with more than two units an SM it takes whole steps only, two of
// them, or for one token up to four: longer activations do not stay in what the ring leaves of L1.  int8, K in bytes, 28672 weight rows:
//   one token     8192 39.7 / 42.1, 12288 55.9 / 57.8, 16384 72.6 / 75.5, 24576 109.2 / 107.6, 28672 126.9 / 125.1
//   eight         8192 42.8 / 42.9, 12288 60.1 / 58.3, 16384 77.8 / 76.3, 24576 112.8 / 109.1, 28672 134.1 / 126.5 (9600 rows 53.2 / 46.6)
//   one token, a step in part    8208 49.6 / 43.7, 10240 50.5 / 49.7, 11008 52.1 / 53.0, 13824 65.8 / 64.5, 14336 71.3 / 66.1,
//                                15360 70.8 / 71.1, 18944 86.0 / 92.8 (the most it would gain), 27648 129 / 121
//   eight, a step in part        8208 52.7 / 44.4, 11008 57.9 / 53.7, 14336 73.4 / 66.5, 18944 99.6 / 94.1, 27648 135 / 122
// bf16 gated 14336, K in bytes: one token 8192 38.8 / 40.9, 16384 72.0 / 73.6; eight 8192 40.5 / 41.0, 16384 77.4 / 74.0.
// For 9 to 16 rows its activations do not fit L1 beside the ring: 16 x 1024 x 8192 6.1 / 13.3, 16 x 4096 x 4096 8.0 / 7.7,
// 16 x 28672 x 8192 48.6 / 42.5.
bool stream_rows(const HostDevice& dev, int64_t m, int64_t weight_rows, int64_t k_bytes) {
    const int64_t units = (weight_rows + 15) / 16;
    if (m <= 8) return units <= 2 * dev.sm_count || k_bytes == 8192 || (k_bytes > 8192 && k_bytes % 4096 == 0 && m * k_bytes <= 16384);
    return m <= 16 && units <= dev.sm_count;
}

// A scaled or gated product, with its sums over K cut into ranges where the plan says so.
template <int OP, int EPI>
int launch_forward(const HostDevice& dev, const char* fn, const Operand (&a)[2], const Operand (&b)[2], int64_t m, int64_t n, int64_t k,
                   DenseParams p, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
    const DensePlan plan = plan_for<OP, EPI>(dev, m, n, k);
    int rc = check_workspace(fn, workspace, workspace_bytes, 4 * split_words(plan, m, EPI == kDenseGated ? 2 * n : n));
    if (rc) return rc;
    p.partial = static_cast<uint32_t*>(workspace);
    rc = launch_dense<OP, EPI>(dev, plan, a, b, m, n, k, p, stream);
    if (rc || plan.splits == 1) return rc;
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.splits = plan.splits;
    int64_t grid = ceil_div(m * (n / 8), 256);
    if (grid > int64_t(dev.sm_count) * 8) grid = int64_t(dev.sm_count) * 8;
    Launch launch(grid, 256, 0, 1, stream);
    AVE_CUDA(cudaLaunchKernelEx(&launch.cfg, finish_splits_kernel<OP == kOpInt8, EPI>, p));
    return 0;
}

template <int OP, int EPI>
int64_t forward_workspace(const char* fn, int64_t m, int64_t n, int64_t k) {
    HostDevice dev;
    if (!sizes_ok(m, n, k)) return fail("%s: size out of range", fn);
    if (m == 0 || n == 0 || k == 0) return 0;
    const int rc = host_device(&dev);
    if (rc) return rc < 0 ? rc : -rc;
    const int64_t cols = EPI == kDenseGated ? 2 * n : n;
    if (!forward_may_cut(m, k * elem_bytes<OP>()) || stream_rows(dev, m, cols, k * elem_bytes<OP>())) return 0;
    return 4 * split_words(plan_for<OP, EPI>(dev, m, n, k), m, cols);
}

DenseParams dense_params() {
    DenseParams p;
    memset(&p, 0, sizeof(p));
    p.segments = 1;
    p.batches = 1;
    return p;
}

// ------------------------------------------------------------------------------ a few tokens
template <bool INT8, bool GATED>
int launch_stream(const HostDevice& dev, StreamParams p, cudaStream_t stream) {
    const int64_t groups = (p.n + 7) / 8;
    p.status = dev.status;
    const bool m8 = p.m <= 8;
    // The activations are read through what the ring leaves of L1: a third stage takes that down to some 30 KB.  It is worth 4 to
    // 7 % for one token on a chip at 1.4 GHz under its power cap (nothing at 1.9), and costs 8 tokens of 8 KB 10 %.
    p.stages = (m8 && static_cast<int64_t>(p.m) * p.k_bytes <= (24 << 10)) ? 3 : 2;
    Launch launch(groups < dev.sm_count ? groups : dev.sm_count, kStreamThreads, m8 ? StreamConfig<true>::smem_bytes(p.stages) : StreamConfig<false>::smem_bytes(p.stages), 1, stream);
    if (m8) AVE_CUDA(cudaLaunchKernelEx(&launch.cfg, gemm_stream_kernel<INT8, GATED, true>, p));
    else AVE_CUDA(cudaLaunchKernelEx(&launch.cfg, gemm_stream_kernel<INT8, GATED, false>, p));
    return 0;
}

StreamParams stream_params(const void* x, int64_t ldx_bytes, int64_t m, int64_t n, int64_t k_bytes, int act, void* d, int64_t ldd) {
    StreamParams p;
    memset(&p, 0, sizeof(p));
    p.x = static_cast<const uint8_t*>(x);
    p.ldx = ldx_bytes;
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(n);
    p.k_bytes = static_cast<int>(k_bytes);
    p.act = act;
    p.d = static_cast<__nv_bfloat16*>(d);
    p.ldd = ldd;
    return p;
}

template <int NV, bool CTA_ROW>
int launch_quantize(const void* x, int64_t rows, int64_t k, int64_t ldx, void* values, int64_t ldv, void* scales, cudaStream_t stream) {
    const int64_t per_cta = CTA_ROW ? 1 : kInt8Threads / 32;
    Launch launch((rows + per_cta - 1) / per_cta, kInt8Threads, 0, 1, stream);
    AVE_CUDA(cudaLaunchKernelEx(&launch.cfg, quantize_int8_kernel<NV, CTA_ROW>, static_cast<const __nv_bfloat16*>(x),
                                static_cast<long long>(rows), static_cast<int>(k), static_cast<long long>(ldx), static_cast<int8_t*>(values),
                                static_cast<long long>(ldv), static_cast<float*>(scales)));
    return 0;
}

template <int ACT>
int launch_gated_backward(const HostDevice& dev, const void* dd, int64_t ld_dd, const void* gate, int64_t ld_gate, const void* up,
                          int64_t ld_up, void* d_gate, void* d_up, int64_t ld, int64_t m, int64_t f, cudaStream_t stream) {
    const int64_t pieces = m * (f / 8);
    const int64_t most = int64_t(dev.sm_count) * 8;
    int64_t grid = (pieces + 255) / 256;
    if (grid > most) grid = most;
    Launch launch(grid, 256, 0, 1, stream);
    AVE_CUDA(cudaLaunchKernelEx(&launch.cfg, gated_backward_kernel<ACT>, static_cast<const __nv_bfloat16*>(dd), static_cast<long long>(ld_dd),
                                static_cast<const __nv_bfloat16*>(gate), static_cast<long long>(ld_gate), static_cast<const __nv_bfloat16*>(up),
                                static_cast<long long>(ld_up), static_cast<__nv_bfloat16*>(d_gate), static_cast<__nv_bfloat16*>(d_up),
                                static_cast<long long>(ld), static_cast<long long>(m), static_cast<int>(f / 8)));
    return 0;
}

int zero_matrix(void* d, int64_t rows, int64_t cols, int64_t ld, cudaStream_t stream) {
    if (rows == 0 || cols == 0) return 0;
    AVE_CUDA(cudaMemset2DAsync(d, static_cast<size_t>(row_stride(rows, cols, ld)) * 2, 0, static_cast<size_t>(cols) * 2, static_cast<size_t>(rows), stream));
    return 0;
}

}  // namespace

namespace avefp4 {

cudaError_t prepare_dense_kernels() {
    cudaError_t e;
#define PREP(CG, OP, EPI)                                                                                                              \
    if ((e = cudaFuncSetAttribute(gemm_dense_kernel<CG, OP, EPI>, cudaFuncAttributeMaxDynamicSharedMemorySize, DenseConfig::kSmemBytes)) != cudaSuccess) \
        return e;
    PREP(1, kOpInt8, kDenseScaled)
    PREP(2, kOpInt8, kDenseScaled)
    PREP(1, kOpInt8, kDenseGated)
    PREP(2, kOpInt8, kDenseGated)
    PREP(1, kOpBf16, kDenseGated)
    PREP(2, kOpBf16, kDenseGated)
    PREP(1, kOpBf16Nn, kDensePlain)
    PREP(2, kOpBf16Nn, kDensePlain)
    PREP(1, kOpBf16Tn, kDensePlain)
    PREP(2, kOpBf16Tn, kDensePlain)
#undef PREP
#define PREP(INT8, GATED, M8)                                                                                                          \
    if ((e = cudaFuncSetAttribute(gemm_stream_kernel<INT8, GATED, M8>, cudaFuncAttributeMaxDynamicSharedMemorySize, StreamConfig<M8>::smem_bytes(StreamConfig<M8>::kMaxStages))) != cudaSuccess) \
        return e;
    PREP(true, false, true)
    PREP(true, false, false)
    PREP(true, true, true)
    PREP(true, true, false)
    PREP(false, true, true)
    PREP(false, true, false)
#undef PREP
    // the others are only looked at, so that their code is on the device before a first call inside a stream capture
    cudaFuncAttributes attr;
#define PREP(...) \
    if ((e = cudaFuncGetAttributes(&attr, __VA_ARGS__)) != cudaSuccess) return e;
    PREP(quantize_int8_kernel<1, false>)
    PREP(quantize_int8_kernel<2, false>)
    PREP(quantize_int8_kernel<4, false>)
    PREP(quantize_int8_kernel<1, true>)
    PREP(quantize_int8_kernel<2, true>)
    PREP(quantize_int8_kernel<4, true>)
    PREP(quantize_int8_kernel<8, true>)
    PREP(quantize_int8_kernel<0, true>)
    PREP(gated_backward_kernel<AVE_FP4_ACT_NONE>)
    PREP(gated_backward_kernel<AVE_FP4_ACT_RELU>)
    PREP(gated_backward_kernel<AVE_FP4_ACT_GELU>)
    PREP(gated_backward_kernel<AVE_FP4_ACT_GELU_TANH>)
    PREP(gated_backward_kernel<AVE_FP4_ACT_SILU>)
    PREP(sum_splits_kernel)
    PREP(finish_splits_kernel<true, kDenseScaled>)
    PREP(finish_splits_kernel<true, kDenseGated>)
    PREP(finish_splits_kernel<false, kDenseGated>)
#undef PREP
    return cudaSuccess;
}

}  // namespace avefp4

#define CHECK(x)              \
    do {                      \
        int rc__ = (x);       \
        if (rc__) return rc__; \
    } while (0)

extern "C" {

int ave_int8_quantize(const void* x_bf16, int64_t rows, int64_t k, int64_t ldx, void* values, int64_t ldv, void* scales,
                      void* stream) {
    static const char* fn = "ave_int8_quantize";
    HostDevice dev;
    if (!sizes_ok(rows, k, 0)) return fail("%s: size out of range", fn);
    if (k == 0 || k % 16 != 0) return fail("%s: K must be a positive multiple of 16, got %lld", fn, static_cast<long long>(k));
    if (rows == 0) return 0;
    CHECK(check_matrix(fn, "x", x_bf16, rows, k, ldx, 2));
    CHECK(check_matrix(fn, "values", values, rows, k, ldv, 1));
    CHECK(check_vector(fn, "scales", scales));
    CHECK(host_device(&dev));
    ldx = row_stride(rows, k, ldx);
    ldv = row_stride(rows, k, ldv);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (k <= 256) return launch_quantize<1, false>(x_bf16, rows, k, ldx, values, ldv, scales, s);
    if (k <= 512) return launch_quantize<2, false>(x_bf16, rows, k, ldx, values, ldv, scales, s);
    if (k <= 1024) return launch_quantize<4, false>(x_bf16, rows, k, ldx, values, ldv, scales, s);
    if (k <= 2048) return launch_quantize<1, true>(x_bf16, rows, k, ldx, values, ldv, scales, s);
    if (k <= 4096) return launch_quantize<2, true>(x_bf16, rows, k, ldx, values, ldv, scales, s);
    if (k <= 8192) return launch_quantize<4, true>(x_bf16, rows, k, ldx, values, ldv, scales, s);
    if (k <= 16384) return launch_quantize<8, true>(x_bf16, rows, k, ldx, values, ldv, scales, s);
    return launch_quantize<0, true>(x_bf16, rows, k, ldx, values, ldv, scales, s);
}

int64_t ave_int8_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k) {
    return forward_workspace<kOpInt8, kDenseScaled>("ave_int8_gemm_workspace_bytes", m, n, k);
}

int ave_int8_gemm(const void* a, int64_t lda, const void* a_scales, const void* b, int64_t ldb, const void* b_scales,
                  const void* bias_bf16, int activation, void* d_bf16, int64_t ldd, void* workspace, int64_t workspace_bytes,
                  int64_t m, int64_t n, int64_t k, void* stream) {
    static const char* fn = "ave_int8_gemm";
    HostDevice dev;
    if (!sizes_ok(m, n, k)) return fail("%s: size out of range", fn);
    if (n % 8 != 0) return fail("%s: N must be a multiple of 8, got %lld", fn, static_cast<long long>(n));
    if (k == 0 || k % 16 != 0 || k > AVE_INT8_MAX_K)
        return fail("%s: K must be a positive multiple of 16, at most %d, got %lld", fn, AVE_INT8_MAX_K, static_cast<long long>(k));
    CHECK(check_activation(fn, activation));
    if (m == 0 || n == 0) return 0;
    CHECK(check_matrix(fn, "A", a, m, k, lda, 1));
    CHECK(check_matrix(fn, "B", b, n, k, ldb, 1));
    CHECK(check_matrix(fn, "D", d_bf16, m, n, ldd, 2));
    CHECK(check_vector(fn, "the scales of A", a_scales));
    CHECK(check_vector(fn, "the scales of B", b_scales));
    if (bias_bf16 != nullptr) CHECK(check_vector(fn, "the bias", bias_bf16));
    CHECK(host_device(&dev));
    lda = row_stride(m, k, lda);
    ldb = row_stride(n, k, ldb);
    ldd = row_stride(m, n, ldd);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (stream_rows(dev, m, n, k)) {
        StreamParams p = stream_params(a, lda, m, n, k, activation, d_bf16, ldd);
        p.w[0] = static_cast<const uint8_t*>(b);
        p.ldw[0] = ldb;
        p.x_scale = static_cast<const float*>(a_scales);
        p.w_scale[0] = static_cast<const float*>(b_scales);
        p.bias = static_cast<const __nv_bfloat16*>(bias_bf16);
        return launch_stream<true, false>(dev, p, s);
    }
    DenseParams p = dense_params();
    p.a_scale = static_cast<const float*>(a_scales);
    p.b_scale[0] = p.b_scale[1] = static_cast<const float*>(b_scales);
    p.bias = static_cast<const __nv_bfloat16*>(bias_bf16);
    p.act = activation;
    p.d[0] = p.d[1] = static_cast<__nv_bfloat16*>(d_bf16);
    p.ldd = ldd;
    return launch_forward<kOpInt8, kDenseScaled>(dev, fn, {{a, lda}, {a, lda}}, {{b, ldb}, {b, ldb}}, m, n, k, p, workspace, workspace_bytes, s);
}

int64_t ave_int8_gemm_gated_workspace_bytes(int64_t m, int64_t f, int64_t k) {
    return forward_workspace<kOpInt8, kDenseGated>("ave_int8_gemm_gated_workspace_bytes", m, f, k);
}

int ave_int8_gemm_gated(const void* a, int64_t lda, const void* a_scales, const void* w_gate, int64_t ld_wg, const void* gate_scales,
                        const void* w_up, int64_t ld_wu, const void* up_scales, int activation, void* d_bf16, int64_t ldd,
                        void* workspace, int64_t workspace_bytes, int64_t m, int64_t f, int64_t k, void* stream) {
    static const char* fn = "ave_int8_gemm_gated";
    HostDevice dev;
    if (!sizes_ok(m, f, k)) return fail("%s: size out of range", fn);
    if (f % 8 != 0) return fail("%s: F must be a multiple of 8, got %lld", fn, static_cast<long long>(f));
    if (k == 0 || k % 16 != 0 || k > AVE_INT8_MAX_K)
        return fail("%s: K must be a positive multiple of 16, at most %d, got %lld", fn, AVE_INT8_MAX_K, static_cast<long long>(k));
    CHECK(check_activation(fn, activation));
    if (m == 0 || f == 0) return 0;
    CHECK(check_matrix(fn, "A", a, m, k, lda, 1));
    CHECK(check_matrix(fn, "W_gate", w_gate, f, k, ld_wg, 1));
    CHECK(check_matrix(fn, "W_up", w_up, f, k, ld_wu, 1));
    CHECK(check_matrix(fn, "D", d_bf16, m, f, ldd, 2));
    CHECK(check_vector(fn, "the scales of A", a_scales));
    CHECK(check_vector(fn, "the scales of W_gate", gate_scales));
    CHECK(check_vector(fn, "the scales of W_up", up_scales));
    CHECK(host_device(&dev));
    lda = row_stride(m, k, lda);
    ld_wg = row_stride(f, k, ld_wg);
    ld_wu = row_stride(f, k, ld_wu);
    ldd = row_stride(m, f, ldd);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (stream_rows(dev, m, 2 * f, k)) {
        StreamParams p = stream_params(a, lda, m, f, k, activation, d_bf16, ldd);
        p.w[0] = static_cast<const uint8_t*>(w_gate);
        p.w[1] = static_cast<const uint8_t*>(w_up);
        p.ldw[0] = ld_wg;
        p.ldw[1] = ld_wu;
        p.x_scale = static_cast<const float*>(a_scales);
        p.w_scale[0] = static_cast<const float*>(gate_scales);
        p.w_scale[1] = static_cast<const float*>(up_scales);
        return launch_stream<true, true>(dev, p, s);
    }
    DenseParams p = dense_params();
    p.a_scale = static_cast<const float*>(a_scales);
    p.b_scale[0] = static_cast<const float*>(gate_scales);
    p.b_scale[1] = static_cast<const float*>(up_scales);
    p.act = activation;
    p.d[0] = p.d[1] = static_cast<__nv_bfloat16*>(d_bf16);
    p.ldd = ldd;
    return launch_forward<kOpInt8, kDenseGated>(dev, fn, {{a, lda}, {a, lda}}, {{w_gate, ld_wg}, {w_up, ld_wu}}, m, f, k, p, workspace, workspace_bytes, s);
}

int64_t ave_bf16_gemm_gated_workspace_bytes(int64_t m, int64_t f, int64_t h) {
    return forward_workspace<kOpBf16, kDenseGated>("ave_bf16_gemm_gated_workspace_bytes", m, f, h);
}

int ave_bf16_gemm_gated(const void* x, int64_t ldx, const void* w_gate, int64_t ld_wg, const void* w_up, int64_t ld_wu, int activation,
                        void* d_bf16, int64_t ldd, void* gate_bf16, int64_t ld_gate, void* up_bf16, int64_t ld_up,
                        void* workspace, int64_t workspace_bytes, int64_t m, int64_t f, int64_t h, void* stream) {
    static const char* fn = "ave_bf16_gemm_gated";
    HostDevice dev;
    if (!sizes_ok(m, f, h)) return fail("%s: size out of range", fn);
    if (f % 8 != 0) return fail("%s: F must be a multiple of 8, got %lld", fn, static_cast<long long>(f));
    if (h == 0 || h % 8 != 0) return fail("%s: H must be a positive multiple of 8, got %lld", fn, static_cast<long long>(h));
    CHECK(check_activation(fn, activation));
    if ((gate_bf16 == nullptr) != (up_bf16 == nullptr)) return fail("%s: gate and up are kept together or not at all", fn);
    if (m == 0 || f == 0) return 0;
    CHECK(check_matrix(fn, "x", x, m, h, ldx, 2));
    CHECK(check_matrix(fn, "W_gate", w_gate, f, h, ld_wg, 2));
    CHECK(check_matrix(fn, "W_up", w_up, f, h, ld_wu, 2));
    CHECK(check_matrix(fn, "D", d_bf16, m, f, ldd, 2));
    if (gate_bf16 != nullptr) {
        CHECK(check_matrix(fn, "gate", gate_bf16, m, f, ld_gate, 2));
        CHECK(check_matrix(fn, "up", up_bf16, m, f, ld_up, 2));
    }
    CHECK(host_device(&dev));
    ldx = row_stride(m, h, ldx);
    ld_wg = row_stride(f, h, ld_wg);
    ld_wu = row_stride(f, h, ld_wu);
    ldd = row_stride(m, f, ldd);
    ld_gate = row_stride(m, f, ld_gate);
    ld_up = row_stride(m, f, ld_up);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (stream_rows(dev, m, 2 * f, 2 * h)) {
        StreamParams p = stream_params(x, ldx * 2, m, f, h * 2, activation, d_bf16, ldd);
        p.w[0] = static_cast<const uint8_t*>(w_gate);
        p.w[1] = static_cast<const uint8_t*>(w_up);
        p.ldw[0] = ld_wg * 2;
        p.ldw[1] = ld_wu * 2;
        p.gate = static_cast<__nv_bfloat16*>(gate_bf16);
        p.up = static_cast<__nv_bfloat16*>(up_bf16);
        p.ld_gate = ld_gate;
        p.ld_up = ld_up;
        return launch_stream<false, true>(dev, p, s);
    }
    DenseParams p = dense_params();
    p.act = activation;
    p.d[0] = p.d[1] = static_cast<__nv_bfloat16*>(d_bf16);
    p.ldd = ldd;
    p.gate = static_cast<__nv_bfloat16*>(gate_bf16);
    p.up = static_cast<__nv_bfloat16*>(up_bf16);
    p.ld_gate = ld_gate;
    p.ld_up = ld_up;
    return launch_forward<kOpBf16, kDenseGated>(dev, fn, {{x, ldx}, {x, ldx}}, {{w_gate, ld_wg}, {w_up, ld_wu}}, m, f, h, p, workspace, workspace_bytes, s);
}

}  // extern "C"

namespace {

// Workspace of the gated block's backward pass: dG and dU with rows padded to whole 128-byte lines (a box row of a TMA load
// then touches one line), and what cuts of K in either product need.
struct GatedBackwardPlan {
    DensePlan dx, dw;
    int64_t ld, half, dx_words, dw_words;
    int64_t bytes() const { return 2 * half + 4 * (dx_words + dw_words); }
};

GatedBackwardPlan plan_gated_backward(const HostDevice& dev, int64_t m, int64_t f, int64_t h, bool want_x, bool want_w) {
    GatedBackwardPlan p{};
    p.ld = ceil_div(f, 64) * 64;
    p.half = ceil_div(m * p.ld * 2, 256) * 256;
    const PairPlan& pair = pair_for(dev, m, f, h, true);
    p.dx = want_w ? pair.first : pair.first_alone;
    p.dw = want_x ? pair.second : pair.second_alone;
    if (want_x) p.dx_words = split_words(p.dx, m, h);
    if (want_w) p.dw_words = split_words(p.dw, 2 * f, h);
    return p;
}

struct ProductBackwardPlan {
    DensePlan da, db;
    int64_t da_words, db_words;
    int64_t bytes() const { return 4 * (da_words + db_words); }
};

ProductBackwardPlan plan_product_backward(const HostDevice& dev, int64_t m, int64_t n, int64_t k, bool want_a, bool want_b) {
    ProductBackwardPlan p{};
    const PairPlan& pair = pair_for(dev, m, n, k, false);
    p.da = want_b ? pair.first : pair.first_alone;
    p.db = want_a ? pair.second : pair.second_alone;
    if (want_a) p.da_words = split_words(p.da, m, k);
    if (want_b) p.db_words = split_words(p.db, n, k);
    return p;
}

}  // namespace

extern "C" {

int64_t ave_bf16_gated_backward_workspace_bytes(int64_t m, int64_t f, int64_t h, int want_dx, int want_dw) {
    HostDevice dev;
    if (!sizes_ok(m, f, h)) return fail("ave_bf16_gated_backward_workspace_bytes: size out of range");
    if (m == 0 || f == 0 || h == 0 || !(want_dx || want_dw)) return 0;
    const int rc = host_device(&dev);
    if (rc) return rc < 0 ? rc : -rc;
    return plan_gated_backward(dev, m, f, h, want_dx != 0, want_dw != 0).bytes();
}

int ave_bf16_gated_backward(const void* dd, int64_t ld_dd, const void* x, int64_t ldx, const void* w_gate, int64_t ld_wg,
                            const void* w_up, int64_t ld_wu, const void* gate, int64_t ld_gate, const void* up, int64_t ld_up,
                            int activation, void* dx, int64_t ld_dx, void* dw_gate, void* dw_up, int64_t ld_dw, void* workspace,
                            int64_t workspace_bytes, int64_t m, int64_t f, int64_t h, void* stream) {
    static const char* fn = "ave_bf16_gated_backward";
    HostDevice dev;
    if (!sizes_ok(m, f, h)) return fail("%s: size out of range", fn);
    if (f % 8 != 0) return fail("%s: F must be a multiple of 8, got %lld", fn, static_cast<long long>(f));
    if (h == 0 || h % 8 != 0) return fail("%s: H must be a positive multiple of 8, got %lld", fn, static_cast<long long>(h));
    CHECK(check_activation(fn, activation));
    if ((dw_gate == nullptr) != (dw_up == nullptr)) return fail("%s: dW_gate and dW_up are computed together or not at all", fn);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool want_x = dx != nullptr, want_w = dw_gate != nullptr;
    if (want_x && m > 0) CHECK(check_matrix(fn, "dx", dx, m, h, ld_dx, 2));
    if (want_w && f > 0) {
        CHECK(check_matrix(fn, "dW_gate", dw_gate, f, h, ld_dw, 2));
        CHECK(check_matrix(fn, "dW_up", dw_up, f, h, ld_dw, 2));
    }
    if (m == 0 || f == 0) {
        if (want_x) CHECK(zero_matrix(dx, m, h, ld_dx, s));
        if (want_w) {
            CHECK(zero_matrix(dw_gate, f, h, ld_dw, s));
            CHECK(zero_matrix(dw_up, f, h, ld_dw, s));
        }
        return 0;
    }
    CHECK(check_matrix(fn, "dD", dd, m, f, ld_dd, 2));
    CHECK(check_matrix(fn, "x", x, m, h, ldx, 2));
    CHECK(check_matrix(fn, "W_gate", w_gate, f, h, ld_wg, 2));
    CHECK(check_matrix(fn, "W_up", w_up, f, h, ld_wu, 2));
    CHECK(check_matrix(fn, "gate", gate, m, f, ld_gate, 2));
    CHECK(check_matrix(fn, "up", up, m, f, ld_up, 2));
    if (!want_x && !want_w) return 0;
    CHECK(host_device(&dev));
    const GatedBackwardPlan plan = plan_gated_backward(dev, m, f, h, want_x, want_w);
    CHECK(check_workspace(fn, workspace, workspace_bytes, plan.bytes()));
    ld_dd = row_stride(m, f, ld_dd);
    ldx = row_stride(m, h, ldx);
    ld_wg = row_stride(f, h, ld_wg);
    ld_wu = row_stride(f, h, ld_wu);
    ld_gate = row_stride(m, f, ld_gate);
    ld_up = row_stride(m, f, ld_up);
    const int64_t ld = plan.ld;
    void* d_gate = workspace;
    void* d_up = static_cast<uint8_t*>(workspace) + plan.half;
    uint32_t* dx_partial = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + 2 * plan.half);
    uint32_t* dw_partial = dx_partial + plan.dx_words;
    SplitSums sums{};
    switch (activation) {
        case AVE_FP4_ACT_RELU: CHECK(launch_gated_backward<AVE_FP4_ACT_RELU>(dev, dd, ld_dd, gate, ld_gate, up, ld_up, d_gate, d_up, ld, m, f, s)); break;
        case AVE_FP4_ACT_GELU: CHECK(launch_gated_backward<AVE_FP4_ACT_GELU>(dev, dd, ld_dd, gate, ld_gate, up, ld_up, d_gate, d_up, ld, m, f, s)); break;
        case AVE_FP4_ACT_GELU_TANH: CHECK(launch_gated_backward<AVE_FP4_ACT_GELU_TANH>(dev, dd, ld_dd, gate, ld_gate, up, ld_up, d_gate, d_up, ld, m, f, s)); break;
        case AVE_FP4_ACT_SILU: CHECK(launch_gated_backward<AVE_FP4_ACT_SILU>(dev, dd, ld_dd, gate, ld_gate, up, ld_up, d_gate, d_up, ld, m, f, s)); break;
        default: CHECK(launch_gated_backward<AVE_FP4_ACT_NONE>(dev, dd, ld_dd, gate, ld_gate, up, ld_up, d_gate, d_up, ld, m, f, s)); break;
    }
    if (want_x) {
        DenseParams p = dense_params();
        p.segments = 2;
        p.d[0] = p.d[1] = static_cast<__nv_bfloat16*>(dx);
        p.ldd = row_stride(m, h, ld_dx);
        p.partial = dx_partial;
        p.trigger_late = want_w;
        CHECK((launch_dense<kOpBf16Nn, kDensePlain>(dev, plan.dx, {{d_gate, ld}, {d_up, ld}}, {{w_gate, ld_wg}, {w_up, ld_wu}}, m, h, f, p, s)));
        sums.job[0] = split_sum(plan.dx, dx_partial, m * h, dx, p.ldd, m, h);
    }
    if (want_w) {
        DenseParams p = dense_params();
        p.batches = 2;
        p.d[0] = static_cast<__nv_bfloat16*>(dw_gate);
        p.d[1] = static_cast<__nv_bfloat16*>(dw_up);
        p.ldd = row_stride(f, h, ld_dw);
        p.partial = dw_partial;
        p.wait_late = want_x;
        p.early = plan.dw.early;
        p.early_items = plan.dw.early_items;
        CHECK((launch_dense<kOpBf16Tn, kDensePlain>(dev, plan.dw, {{d_gate, ld}, {d_up, ld}}, {{x, ldx}, {x, ldx}}, f, h, m, p, s)));
        sums.job[1] = split_sum(plan.dw, dw_partial, 2 * f * h, dw_gate, p.ldd, f, h);
        sums.job[2] = split_sum(plan.dw, dw_partial + f * h, 2 * f * h, dw_up, p.ldd, f, h);
    }
    return launch_sums(dev, sums, s);
}

int64_t ave_bf16_gemm_backward_workspace_bytes(int64_t m, int64_t n, int64_t k, int want_da, int want_db) {
    HostDevice dev;
    if (!sizes_ok(m, n, k)) return fail("ave_bf16_gemm_backward_workspace_bytes: size out of range");
    if (m == 0 || n == 0 || k == 0 || !(want_da || want_db)) return 0;
    const int rc = host_device(&dev);
    if (rc) return rc < 0 ? rc : -rc;
    return plan_product_backward(dev, m, n, k, want_da != 0, want_db != 0).bytes();
}

int ave_bf16_gemm_backward(const void* dd, int64_t ld_dd, const void* a, int64_t lda, const void* b, int64_t ldb, void* da,
                           int64_t ld_da, void* db, int64_t ld_db, void* workspace, int64_t workspace_bytes, int64_t m, int64_t n, int64_t k,
                           void* stream) {
    static const char* fn = "ave_bf16_gemm_backward";
    HostDevice dev;
    if (!sizes_ok(m, n, k)) return fail("%s: size out of range", fn);
    if (n % 8 != 0) return fail("%s: N must be a multiple of 8, got %lld", fn, static_cast<long long>(n));
    if (k == 0 || k % 8 != 0) return fail("%s: K must be a positive multiple of 8, got %lld", fn, static_cast<long long>(k));
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (da != nullptr && m > 0) CHECK(check_matrix(fn, "dA", da, m, k, ld_da, 2));
    if (db != nullptr && n > 0) CHECK(check_matrix(fn, "dB", db, n, k, ld_db, 2));
    if (m == 0 || n == 0) {
        if (da != nullptr) CHECK(zero_matrix(da, m, k, ld_da, s));
        if (db != nullptr) CHECK(zero_matrix(db, n, k, ld_db, s));
        return 0;
    }
    CHECK(check_matrix(fn, "dD", dd, m, n, ld_dd, 2));
    CHECK(check_matrix(fn, "A", a, m, k, lda, 2));
    CHECK(check_matrix(fn, "B", b, n, k, ldb, 2));
    CHECK(host_device(&dev));
    ld_dd = row_stride(m, n, ld_dd);
    lda = row_stride(m, k, lda);
    ldb = row_stride(n, k, ldb);
    const ProductBackwardPlan plan = plan_product_backward(dev, m, n, k, da != nullptr, db != nullptr);
    CHECK(check_workspace(fn, workspace, workspace_bytes, plan.bytes()));
    uint32_t* da_partial = static_cast<uint32_t*>(workspace);
    uint32_t* db_partial = da_partial + plan.da_words;
    SplitSums sums{};
    if (da != nullptr) {
        DenseParams p = dense_params();
        p.d[0] = p.d[1] = static_cast<__nv_bfloat16*>(da);
        p.ldd = row_stride(m, k, ld_da);
        p.partial = da_partial;
        p.trigger_late = db != nullptr;
        CHECK((launch_dense<kOpBf16Nn, kDensePlain>(dev, plan.da, {{dd, ld_dd}, {dd, ld_dd}}, {{b, ldb}, {b, ldb}}, m, k, n, p, s)));
        sums.job[0] = split_sum(plan.da, da_partial, m * k, da, p.ldd, m, k);
    }
    if (db != nullptr) {
        DenseParams p = dense_params();
        p.d[0] = p.d[1] = static_cast<__nv_bfloat16*>(db);
        p.ldd = row_stride(n, k, ld_db);
        p.partial = db_partial;
        p.wait_late = da != nullptr;
        p.early = plan.db.early;
        p.early_items = plan.db.early_items;
        CHECK((launch_dense<kOpBf16Tn, kDensePlain>(dev, plan.db, {{dd, ld_dd}, {dd, ld_dd}}, {{a, lda}, {a, lda}}, n, k, m, p, s)));
        sums.job[1] = split_sum(plan.db, db_partial, n * k, db, p.ldd, n, k);
    }
    return launch_sums(dev, sums, s);
}

}  // extern "C"
