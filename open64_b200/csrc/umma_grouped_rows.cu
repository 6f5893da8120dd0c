// Products grouped by expert, and the block-scaled e4m3 product, for few rows: every weight is read once
// for a handful of rows of A, so the weights' way from HBM is all that counts.
//
// The operands change places: 128 rows of a weight are the MMA's M and the rows of A its N (16, 32, 64 or 128),
// so that nothing is spent on rows that are not there - shared memory, TMEM reads and sums go by 16 rows, not
// by 128 - and the ring holds nearly 200 KB of weights on their way per SM.  A thread then owns one column
// of C (one weight row) and all rows of the tile.  With the SwiGLU tail a tile is 128 gate and the 128
// matching up rows: two accumulators, joined through shared memory.
//
// Tiles go group by group, a group's row tiles next to each other (they share the weight block in L2).  When
// there are too few of them to fill the GPU, a cluster of S CTAs divides a tile's K blocks; the partial sums
// meet in distributed shared memory and are added in rank order, each CTA finishing its share of the rows.
//
// Bound by HBM where every weight is read once: 8 experts 4096 x 14336 bf16 for 16 rows 139-143 us = 6.7 TB/s; 32 experts
// 2 x 2048 x 4096 e4m3 for 96 rows 63-65 us = 5.5 TB/s; 1 x 8192 x 8192 e4m3 14 us (graph) = 4.7 TB/s, of which about 4 us
// are launch, first data and the exchange.
//
// Warps: 0 loads, 1 issues the MMAs, 2 fetches scales, 4.. add (four for each weight block).  Launched so that
// its set-up overlaps the previous kernel of the stream (it waits before it touches memory).  That kernel may write what
// is read here while this one already exists, so scales and offsets come by ordinary loads: the read-only path is for
// memory that nobody writes during a kernel's life.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <type_traits>

#include "grouped.cuh"

namespace o64 {

namespace {

constexpr int kGrBufs = 4;  // accumulator buffers
constexpr int kGrScaleSlots = 8;

template <int NB, int TOK>
struct RowsLayout {
    static constexpr int kWBytes = NB * 128 * kRowBytes;
    static constexpr int kXBytes = TOK * kRowBytes;
    static constexpr int kStageBytes = kWBytes + kXBytes;
    static constexpr int kXchBytes = NB == 2 ? TOK * 128 * 4 : 0;  // up values on their way to the gate warps
    static constexpr int kRoom = 200 * 1024 - kXchBytes;
    static constexpr int kStages = kRoom / kStageBytes > 12 ? 12 : kRoom / kStageBytes;
    static constexpr int kRing = kStages * kStageBytes;
    static constexpr int kXch = kRing;
    static constexpr int kScales = kXch + kXchBytes;  // [slot][NB][TOK]
    static constexpr int kAmax = kScales + kGrScaleSlots * NB * TOK * 4;  // [2][4][TOK]
    static constexpr int kBars = kAmax + 2 * 4 * TOK * 4;
    static constexpr int kNumBars = 2 * kStages + 2 * kGrBufs + 2 * kGrScaleSlots + 9;
    static constexpr int kTmemPtr = kBars + 8 * kNumBars;
    static constexpr int kAbort = kTmemPtr + 4;
    static constexpr int kDynamic = kAbort + 4 + 1024;
    static constexpr int kThreads = 128 + 128 * NB;
    static constexpr uint32_t kTmemCols = kGrBufs * NB * TOK;
    static_assert(kDynamic <= 227 * 1024, "shared memory");
    static_assert(kStageBytes % 1024 == 0 && kWBytes % 1024 == 0, "swizzle atoms");
    static_assert(kRing >= 128 * NB * 8 * 16 && kRing >= 128 * NB * TOK * 4, "the ring receives the partial sums");
    static_assert(kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0 && kTmemCols >= 32, "TMEM columns");
};

struct RowsTile {
    int g, begin, end;  // rows of this tile: [begin, end), at most TOK
    int nb;
};

struct RowsWalk {
    int g = 0;
    int base = 0;
    int top = 0;  // the end of the groups before g
};

template <int TOK>
__device__ __forceinline__ bool next_rows_tile(const GroupedParams &p, RowsWalk &w, int t, RowsTile &tile) {
    for (; w.g < p.G; ++w.g) {
        int begin, end;
        group_rows<true>(p, w.g, w.top, begin, end);
        const int tt = (end - begin + TOK - 1) / TOK;
        const int tiles = tt * p.num_n_tiles;
        if (t < w.base + tiles) {
            const int r = t - w.base;
            tile.g = w.g;
            tile.begin = begin + (r % tt) * TOK;
            tile.end = min(tile.begin + TOK, end);
            tile.nb = r / tt;
            return true;
        }
        w.base += tiles;
        w.top = end;
    }
    return false;
}

// The e4m3 tail of a warp's 32 columns: `amax` holds the four warps' largest magnitudes of each row ([4][TOK],
// as integers).  Lane l works out the scales of rows l and l + 32, for all columns of the warp.
template <int TOK, int ROWS>
__device__ __forceinline__ void store_e4m3_rows(const uint32_t *amax, const float (&h)[ROWS], int rows, uint8_t *dst, long long ld, float *scales,
                                                long long ld_scales, bool write_scales) {
    const int lane = threadIdx.x & 31;
    constexpr int kPer = (ROWS + 31) / 32;
    float inv[kPer], back[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int j = i * 32 + lane;
        inv[i] = back[i] = 1.0f;
        if (j < rows) {
            const uint32_t m = max(max(amax[j], amax[TOK + j]), max(amax[2 * TOK + j], amax[3 * TOK + j]));
            const float scale = block_scale_of(__uint_as_float(m));
            if (write_scales) scales[j * ld_scales] = scale;
            inv[i] = 1.0f / scale;
            back[i] = remainder_scale(scale);
        }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        if (j >= rows) break;
        const float f = __shfl_sync(0xffffffffu, inv[j / 32], j % 32), b = __shfl_sync(0xffffffffu, back[j / 32], j % 32);
        dst[j * ld] = (uint8_t)__nv_cvt_float_to_fp8(quotient(h[j], b, f), __NV_SATFINITE, __NV_E4M3);
    }
}

__device__ __forceinline__ void st_cluster_f32x4(uint32_t addr, float2 a, float2 b) {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y) : "memory");
}
__device__ __forceinline__ void st_cluster_f32x2(uint32_t addr, float2 a) {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(addr), "f"(a.x), "f"(a.y) : "memory");
}

}  // namespace

// p.num_n_tiles counts blocks of 128 columns of C; p.split: CTAs a cluster (> 1: one tile per cluster).
// KN: the weight lies [K,N], the first operand with M contiguous.
template <int KIND, int EPI, int TOK, bool KN>
__global__ void __launch_bounds__(RowsLayout<gepi_swiglu(EPI) ? 2 : 1, TOK>::kThreads, 1)
grouped_rows_kernel(const __grid_constant__ CUtensorMap tm_x, const __grid_constant__ CUtensorMap tm_w,
                    const __grid_constant__ GroupedParams p) {
    constexpr bool kSwiglu = gepi_swiglu(EPI);
    constexpr int NB = kSwiglu ? 2 : 1;
    using L = RowsLayout<NB, TOK>;
    constexpr bool kScaled = KIND == MMA_F8F6F4;
    constexpr int kElem = KIND == MMA_F16 ? 2 : 1;
    constexpr int kBlockK = kRowBytes / kElem;
    constexpr int kKnCols = kRowBytes / kElem;          // columns in a 128-byte row of a [K,N] weight
    constexpr int kKnGroupBytes = kBlockK * kRowBytes;  // kBlockK such rows
    static_assert(!KN || !kSwiglu, "gate and up weights are [N,K]");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bar_base = smem_base + L::kBars;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (L::kStages + s); };
    auto acc_full_bar = [&](int b) { return bar_base + 8u * (2 * L::kStages + b); };
    auto acc_empty_bar = [&](int b) { return bar_base + 8u * (2 * L::kStages + kGrBufs + b); };
    auto scale_full_bar = [&](int s) { return bar_base + 8u * (2 * L::kStages + 2 * kGrBufs + s); };
    auto scale_empty_bar = [&](int s) { return bar_base + 8u * (2 * L::kStages + 2 * kGrBufs + kGrScaleSlots + s); };
    const uint32_t extra = bar_base + 8u * (2 * L::kStages + 2 * kGrBufs + 2 * kGrScaleSlots);
    auto up_full_bar = [&](int q) { return extra + 8u * q; };
    auto up_empty_bar = [&](int q) { return extra + 8u * (4 + q); };
    const uint32_t amax_bar = extra + 8u * 8;
    volatile uint32_t *tmem_ptr_smem = reinterpret_cast<volatile uint32_t *>(smem_gen + L::kTmemPtr);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + L::kAbort);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int S = p.split;
    const int rank = S > 1 ? (int)cluster_ctarank() : 0;
    const int first = S > 1 ? (int)(blockIdx.x / S) : (int)blockIdx.x;
    const int step = S > 1 ? (int)(gridDim.x / S) : (int)gridDim.x;
    const int kb_begin = (int)((long long)p.num_k_blocks * rank / S);
    const int kb_end = (int)((long long)p.num_k_blocks * (rank + 1) / S);

    griddep_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < L::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < kGrBufs; ++b) {
            mbar_init(acc_full_bar(b), 1);
            mbar_init(acc_empty_bar(b), 4 * NB);
        }
        for (int s = 0; s < kGrScaleSlots; ++s) {
            mbar_init(scale_full_bar(s), 1);
            mbar_init(scale_empty_bar(s), 4 * NB);
        }
        for (int q = 0; q < 4; ++q) {
            mbar_init(up_full_bar(q), 1);
            mbar_init(up_empty_bar(q), 1);
        }
        mbar_init(amax_bar, 4);
        *abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_x);
        tma_prefetch_desc(&tm_w);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(smem_gen + L::kTmemPtr), L::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    griddep_wait();
    if (p.offsets && blockIdx.x == 0 && warp == 3) {  // offsets that are not ascending within 0 .. T are reported
        for (int g = lane; g < p.G; g += 32) {
            int b, e;
            bool bad;
            group_rows<true>(p, g, 0, b, e, &bad);
            if (bad) atomicCAS(p.status, 0, kBadOffsets);
        }
    }

    float2 acc[TOK / 2];
    RowsTile last;  // split: the one tile of this cluster
    bool have = false;

    if (warp == 0) {
        // ------------------------------ loads -------------------------------------------
        const bool leader = elect_one();
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        RowsWalk walk;
        RowsTile t;
        for (int i = first; ok && next_rows_tile<TOK>(p, walk, i, t); i += step) {
            for (int kb = kb_begin; kb < kb_end; ++kb) {
                ok = mbar_wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, p.status, kWaitGroupProducer, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (leader) {
                    const uint32_t w_dst = smem_base + stage * L::kStageBytes;
                    mbar_arrive_expect_tx(full_bar(stage), L::kStageBytes);
                    if constexpr (KN) {
#pragma unroll
                        for (int c = 0; c < 128 / kKnCols; ++c)
                            tma_load_3d(w_dst + c * kKnGroupBytes, &tm_w, t.nb * 128 + c * kKnCols, kb * kBlockK, t.g, full_bar(stage));
                    } else {
#pragma unroll
                        for (int b = 0; b < NB; ++b)
                            tma_load_3d(w_dst + b * 128 * kRowBytes, &tm_w, kb * kBlockK, t.nb * 128 + b * p.N, t.g, full_bar(stage));
                    }
                    tma_load_2d(w_dst + L::kWBytes, &tm_x, kb * kBlockK, t.begin, full_bar(stage));
                }
                __syncwarp();
                if (++stage == L::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------ MMA ---------------------------------------------
        const bool leader = elect_one();
        constexpr uint32_t fmt = KIND == MMA_F8F6F4 ? 0u : 1u;
        constexpr uint32_t idesc = make_idesc(1u, fmt, fmt, 0u, 128, TOK) | (KN ? 1u << 15 : 0u);
        constexpr uint32_t kWAdvance = KN ? (32 / kElem * kRowBytes) >> 4 : 2;
        int stage = 0;
        uint32_t phase = 0, uses = 0;
        bool ok = true;
        RowsWalk walk;
        RowsTile t;
        // the barriers of the next K block are probed before this one's MMAs are issued: a probe takes about 100
        // cycles, and a loop that waits for its two in turn took 590 a block, 260 of them for the issue
        uint32_t acc_ready = 1, full_ready = mbar_test_wait(full_bar(0), 0);
        auto take = [&]() __attribute__((always_inline)) {
            if (!acc_ready)
                ok = mbar_wait_bounded(acc_empty_bar(uses % kGrBufs), ((uses / kGrBufs) & 1) ^ 1u, abort_flag, p.status, kWaitGroupAccEmpty,
                                       p.wait_ns);
        };
        for (int i = first; ok && next_rows_tile<TOK>(p, walk, i, t); i += step) {
            if (kb_begin == kb_end) continue;
            if (!kScaled) {
                acc_ready = 0;
                take();
            }
            for (int kb = kb_begin; ok && kb < kb_end; ++kb) {
                if (kScaled) take();
                if (!full_ready)
                    ok = mbar_wait_bounded(full_bar(stage), phase, abort_flag, p.status, kWaitGroupFull, p.wait_ns) && ok;
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                const int next_stage = stage + 1 == L::kStages ? 0 : stage + 1;
                const uint32_t next_phase = stage + 1 == L::kStages ? phase ^ 1u : phase;
                if (kScaled) acc_ready = mbar_test_wait(acc_empty_bar((uses + 1) % kGrBufs), (((uses + 1) / kGrBufs) & 1) ^ 1u);
                full_ready = mbar_test_wait(full_bar(next_stage), next_phase);
                tc_fence_after();
                const uint32_t w_addr = smem_base + stage * L::kStageBytes;
                const uint64_t x_desc = make_smem_desc(w_addr + L::kWBytes, 16, 1024);
                const uint32_t d = tmem_base + (uses % kGrBufs) * NB * TOK;
                if (leader) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const uint64_t w_desc = make_smem_desc(w_addr + b * 128 * kRowBytes, KN ? kKnGroupBytes : 16, 1024);
#pragma unroll
                        for (int k = 0; k < kRowBytes / 32; ++k)
                            tc_mma<KIND>(d + b * TOK, w_desc + kWAdvance * k, x_desc + 2u * k, idesc,
                                         (kScaled ? k : ((kb - kb_begin) | k)) != 0 ? 1u : 0u);
                    }
                    tc_commit(empty_bar(stage));
                    if (kScaled) tc_commit(acc_full_bar(uses % kGrBufs));
                }
                __syncwarp();
                if (kScaled) ++uses;
                stage = next_stage;
                phase = next_phase;
            }
            if (!kScaled) {
                if (ok && leader) tc_commit(acc_full_bar(uses % kGrBufs));
                __syncwarp();
                ++uses;
            }
        }
        __syncwarp();
    } else if (kScaled && warp == 2) {
        // ------------------------------ scales ------------------------------------------
        float *ring = reinterpret_cast<float *>(smem_gen + L::kScales);
        constexpr int kPer = (TOK + 31) / 32;  // rows a lane carries
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        RowsWalk walk;
        RowsTile t;
        // four K blocks at a time, the next four (of this tile or of the next one) always on their way
        const float *sa[kPer], *sb0 = nullptr, *sb1 = nullptr;
        const long long sb_step = KN ? p.ldsb : 1;
        float next[kPer][4], b0[4], b1[4];
        int tile = first, kb0 = kb_begin;
        auto fetch = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool in = kb0 + u < kb_end;
#pragma unroll
                for (int r = 0; r < kPer; ++r) next[r][u] = in ? sa[r][kb0 + u] : 0.0f;
                b0[u] = in ? sb0[(kb0 + u) * sb_step] : 0.0f;
                b1[u] = kSwiglu && in ? sb1[kb0 + u] : 0.0f;
            }
        };
        auto begin_tile = [&]() __attribute__((always_inline)) {
            if (!next_rows_tile<TOK>(p, walk, tile, t)) return false;
#pragma unroll
            for (int r = 0; r < kPer; ++r) sa[r] = p.scale_a + (long long)min(t.begin + r * 32 + lane, t.end - 1) * p.ldsa;
            const float *sb = p.scale_b + (long long)t.g * p.stride_sb;
            sb0 = KN ? sb + t.nb : sb + t.nb * p.ldsb;
            sb1 = sb + (long long)((p.N >> 7) + t.nb) * p.ldsb;
            kb0 = kb_begin;
            fetch();
            return true;
        };
        bool more = kb_begin < kb_end && begin_tile();
        while (ok && more) {
            float now[NB][kPer][4];
            const int got = min(4, kb_end - kb0);
#pragma unroll
            for (int r = 0; r < kPer; ++r)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    now[0][r][u] = next[r][u] * b0[u];
                    if constexpr (kSwiglu) now[NB - 1][r][u] = next[r][u] * b1[u];
                }
            kb0 += 4;
            if (kb0 < kb_end) {
                fetch();
            } else {
                tile += step;
                more = begin_tile();
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (u >= got) break;
                ok = mbar_wait_bounded(scale_empty_bar(slot), phase ^ 1u, abort_flag, p.status, kWaitGroupScales, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int r = 0; r < kPer; ++r)
                        if (r * 32 + lane < TOK) ring[(slot * NB + b) * TOK + r * 32 + lane] = now[b][r][u];
                __syncwarp();
                if (lane == 0) mbar_arrive(scale_full_bar(slot));
                if (++slot == kGrScaleSlots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------ sums and tails ----------------------------------
        const int quarter = warp & 3;
        const int blk = (warp - 4) >> 2;  // SwiGLU: 0 = gate, 1 = up
        const int n_in = quarter * 32 + lane;
        const uint32_t t_lane = tmem_base + (uint32_t(quarter * 32) << 16) + blk * TOK;
        const float *ring = reinterpret_cast<const float *>(smem_gen + L::kScales);
        uint32_t uses = 0, slot_phase = 0, tiles = 0;
        int slot = 0;
        bool ok = true;
        RowsWalk walk;
        RowsTile t;
        constexpr int kCols = TOK < 64 ? TOK : 64;  // accumulator columns in flight
        auto fetch = [&](uint32_t (&v)[kCols], uint32_t use, int half) __attribute__((always_inline)) {
            const uint32_t taddr = t_lane + (use % kGrBufs) * NB * TOK + half * kCols;
            if constexpr (TOK == 16) {
                tmem_ld_32x16(taddr, v);
            } else {
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) tmem_ld_32x32(taddr + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&v[32 * c]));
            }
        };
        auto release = [&]() __attribute__((always_inline)) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(acc_empty_bar(uses % kGrBufs));
        };
        for (int i = first; ok && next_rows_tile<TOK>(p, walk, i, t); i += step, ++tiles) {
#pragma unroll
            for (int j = 0; j < TOK / 2; ++j) acc[j] = make_float2(0.0f, 0.0f);
            if constexpr (kScaled) {
                // U K blocks at a time: their waits and their way out of tensor memory overlap.  The barriers of the
                // next ones are probed while these are added.
                auto scales_there = [&](int u) __attribute__((always_inline)) {
                    return mbar_test_wait(scale_full_bar((slot + u) % kGrScaleSlots), slot + u < kGrScaleSlots ? slot_phase : slot_phase ^ 1u);
                };
                auto sums_there = [&](int u) __attribute__((always_inline)) {
                    return mbar_test_wait(acc_full_bar((uses + u) % kGrBufs), ((uses + u) / kGrBufs) & 1);
                };
                uint32_t ready_s = 0, ready_a = 0;  // (of the first of the next blocks)
                auto blocks = [&](auto count) __attribute__((always_inline)) {
                    constexpr int U = decltype(count)::value;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int sl = (slot + u) % kGrScaleSlots;
                        if (u > 0 || !ready_s)
                            ok = mbar_wait_bounded(scale_full_bar(sl), slot + u < kGrScaleSlots ? slot_phase : slot_phase ^ 1u, abort_flag, p.status,
                                                   kWaitGroupScales, p.wait_ns) && ok;
                        if (u > 0 || !ready_a)
                            ok = mbar_wait_bounded(acc_full_bar((uses + u) % kGrBufs), ((uses + u) / kGrBufs) & 1, abort_flag, p.status,
                                                   kWaitGroupAccFull, p.wait_ns) && ok;
                    }
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) return;
                    tc_fence_after();
#pragma unroll
                    for (int half = 0; half < TOK / kCols; ++half) {
                        uint32_t v[U][kCols];
#pragma unroll
                        for (int u = 0; u < U; ++u) fetch(v[u], uses + u, half);
                        // the first 16 rows' scales of each block set out with the sums
                        const float4 *s[U];
                        float4 f[U][4];
#pragma unroll
                        for (int u = 0; u < U; ++u) {
                            s[u] = reinterpret_cast<const float4 *>(ring + (((slot + u) % kGrScaleSlots) * NB + blk) * TOK + half * kCols);
#pragma unroll
                            for (int q = 0; q < 4; ++q) f[u][q] = s[u][q];
                        }
                        tmem_ld_wait();
                        if (half == TOK / kCols - 1) {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) {
#pragma unroll
                                for (int u = 0; u < U; ++u) mbar_arrive(acc_empty_bar((uses + u) % kGrBufs));
                            }
                            ready_s = scales_there(U);
                            ready_a = sums_there(U);
                        }
#pragma unroll
                        for (int u = 0; u < U; ++u) {
#pragma unroll
                            for (int q = 0; q < kCols / 4; ++q) {
                                const float4 x = f[u][q & 3];
                                if (q + 4 < kCols / 4) f[u][q & 3] = s[u][q + 4];
                                float2 *sum = acc + (half * kCols + 4 * q) / 2;
                                sum[0] = __ffma2_rn(make_float2(__uint_as_float(v[u][4 * q]), __uint_as_float(v[u][4 * q + 1])), make_float2(x.x, x.y), sum[0]);
                                sum[1] = __ffma2_rn(make_float2(__uint_as_float(v[u][4 * q + 2]), __uint_as_float(v[u][4 * q + 3])), make_float2(x.z, x.w), sum[1]);
                            }
                        }
                    }
                    __syncwarp();
                    if (lane == 0) {
#pragma unroll
                        for (int u = 0; u < U; ++u) mbar_arrive(scale_empty_bar((slot + u) % kGrScaleSlots));
                    }
                    uses += U;
                    slot += U;
                    if (slot >= kGrScaleSlots) {
                        slot -= kGrScaleSlots;
                        slot_phase ^= 1u;
                    }
                };
                constexpr int kAtOnce = (NB == 1 && TOK <= 64) || TOK <= 32 ? 2 : 1;  // what the registers hold
                int kb = kb_begin;
#pragma unroll 1
                for (; ok && kb + kAtOnce <= kb_end; kb += kAtOnce) blocks(std::integral_constant<int, kAtOnce>());
                if (ok && kb < kb_end) blocks(std::integral_constant<int, 1>());
                if (!ok) break;
            } else if (kb_begin < kb_end) {
                ok = mbar_wait_bounded(acc_full_bar(uses % kGrBufs), (uses / kGrBufs) & 1, abort_flag, p.status, kWaitGroupAccFull, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int half = 0; half < TOK / kCols; ++half) {
                    uint32_t v[kCols];
                    fetch(v, uses, half);
                    tmem_ld_wait();
                    if (half == TOK / kCols - 1) release();
#pragma unroll
                    for (int j = 0; j < kCols / 2; ++j)
                        acc[half * kCols / 2 + j] = make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                }
                ++uses;
            }
            if (!ok) break;
            last = t;
            have = true;
            if (S > 1) break;  // the partial sums meet below

            const int rows = t.end - t.begin;
            const int col = t.nb * 128 + n_in;
            if constexpr (!kSwiglu) {
                if (col < p.N) {
                    __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(p.C) + (long long)t.begin * p.ldc + col;
#pragma unroll
                    for (int j = 0; j < TOK; ++j)
                        if (j < rows) dst[j * p.ldc] = __float2bfloat16_rn((j & 1) ? acc[j / 2].y : acc[j / 2].x);
                }
            } else {
                float *xch = reinterpret_cast<float *>(smem_gen + L::kXch);
                if (blk == 1) {
                    // up: hand the sums to the gate warp of the same rows
                    if (lane == 0)
                        ok = mbar_wait_bounded(up_empty_bar(quarter), (tiles & 1) ^ 1u, abort_flag, p.status, kWaitGroupHalf, p.wait_ns);
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    __syncwarp();  // (orders memory, which the shuffle does not: the other lanes read what lane 0 has waited for)
                    if (!ok) break;
#pragma unroll
                    for (int j = 0; j < TOK; ++j) xch[j * 128 + n_in] = (j & 1) ? acc[j / 2].y : acc[j / 2].x;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(up_full_bar(quarter));
                } else {
                    if (lane == 0)
                        ok = mbar_wait_bounded(up_full_bar(quarter), tiles & 1, abort_flag, p.status, kWaitGroupHalf, p.wait_ns);
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    __syncwarp();  // (orders memory, which the shuffle does not: the other lanes read what lane 0 has waited for)
                    if (!ok) break;
#pragma unroll
                    for (int j = 0; j < TOK / 2; ++j) acc[j] = silu_mul2(acc[j], make_float2(xch[(2 * j) * 128 + n_in], xch[(2 * j + 1) * 128 + n_in]));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(up_empty_bar(quarter));
                    if constexpr (EPI == GEPI_SWIGLU_BF16) {
                        __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(p.C) + (long long)t.begin * p.ldc + col;
#pragma unroll
                        for (int j = 0; j < TOK; ++j)
                            if (j < rows) dst[j * p.ldc] = __float2bfloat16_rn((j & 1) ? acc[j / 2].y : acc[j / 2].x);
                    } else {
                        // the largest magnitude of each row's 128 columns: as integers, whose order is the same and
                        // where a NaN is above everything
                        uint32_t *amax = reinterpret_cast<uint32_t *>(smem_gen + L::kAmax) + (tiles & 1) * 4 * TOK;
#pragma unroll
                        for (int j = 0; j < TOK; ++j) {
                            const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint((j & 1) ? acc[j / 2].y : acc[j / 2].x) & 0x7fffffffu);
                            if (lane == (j & 31)) amax[quarter * TOK + j] = m;
                        }
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(amax_bar);
                            ok = mbar_wait_bounded(amax_bar, tiles & 1, abort_flag, p.status, kWaitGroupHalf, p.wait_ns);
                        }
                        ok = __shfl_sync(0xffffffffu, ok, 0);
                        __syncwarp();  // (orders memory, which the shuffle does not: the other lanes read what lane 0 has waited for)
                        if (!ok) break;
                        float h[TOK];
#pragma unroll
                        for (int j = 0; j < TOK; ++j) h[j] = (j & 1) ? acc[j / 2].y : acc[j / 2].x;
                        store_e4m3_rows<TOK>(amax, h, rows, static_cast<uint8_t *>(p.C) + (long long)t.begin * p.ldc + col, p.ldc,
                                             p.scale_c + (long long)t.begin * p.ldsc + t.nb, p.ldsc, quarter == 0);
                    }
                }
            }
        }
    }

    if (S > 1) {
        // ---- partial sums of one tile: rows r of it belong to CTA r / (TOK / S) of the cluster ----
        __syncwarp();
        cluster_sync_all();  // every ring is idle
        const int shift = __ffs(TOK / S) - 1, per = 1 << shift;  // S and TOK are powers of two
        // what a CTA receives: [rank][four rows at a time][NB * 128 columns], 16 bytes a column, so that a warp's
        // store and its loads are 512 contiguous bytes (with a column's rows side by side the exchange of 64 rows
        // took 10000 cycles)
        const int chunks = per >= 4 ? per >> 2 : 1;
        constexpr uint32_t kChunkBytes = NB * 128 * 16;
        const int n_in = (warp & 3) * 32 + lane;
        if (warp >= 4 && have) {
            const uint32_t base = smem_base + rank * chunks * kChunkBytes + ((warp - 4) / 4 * 128 + n_in) * 16;
            if (per >= 4) {
#pragma unroll
                for (int j = 0; j < TOK; j += 4)
                    if (j < last.end - last.begin)
                        st_cluster_f32x4(map_to_cta(base + ((j & (per - 1)) >> 2) * kChunkBytes, j >> shift), acc[j / 2], acc[j / 2 + 1]);
            } else {
#pragma unroll
                for (int j = 0; j < TOK; j += 2)  // per == 2
                    if (j < last.end - last.begin)
                        st_cluster_f32x2(map_to_cta(base, j >> shift), acc[j / 2]);
            }
        }
        __syncwarp();
        cluster_sync_all();
        const bool mine = warp >= 4 && warp < 8 && have;
        const int col = mine ? last.nb * 128 + n_in : 0;
        const int row0 = mine ? last.begin + (rank << shift) : 0;
        const int rows = mine ? min(per, last.end - row0) : 0;
        // this column's sums of four rows, over all ranks in their order
        auto total4 = [&](int chunk, int blk) __attribute__((always_inline)) {
            const uint8_t *src = smem_gen + chunk * kChunkBytes + (blk * 128 + n_in) * 16;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                if (r >= S) break;
                const float4 x = *reinterpret_cast<const float4 *>(src + r * chunks * kChunkBytes);
                sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
            }
            return sum;
        };
        constexpr int kMostChunks = TOK / 2 / 4;
        float h[kMostChunks * 4];
#pragma unroll
        for (int c = 0; c < kMostChunks; ++c) {
            if (c >= chunks || c * 4 >= rows) break;
            float4 x = total4(c, 0);
            if constexpr (kSwiglu) {
                const float4 u = total4(c, 1);
                const float2 a = silu_mul2(make_float2(x.x, x.y), make_float2(u.x, u.y)), b = silu_mul2(make_float2(x.z, x.w), make_float2(u.z, u.w));
                x = make_float4(a.x, a.y, b.x, b.y);
            }
            h[4 * c] = x.x, h[4 * c + 1] = x.y, h[4 * c + 2] = x.z, h[4 * c + 3] = x.w;
        }
        if constexpr (EPI == GEPI_SWIGLU_E4M3) {
            uint32_t *amax = reinterpret_cast<uint32_t *>(smem_gen + L::kAmax);  // [4][TOK]
#pragma unroll
            for (int c = 0; c < kMostChunks; ++c) {
                if (c * 4 >= rows) break;
                uint32_t m[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) m[e] = __reduce_max_sync(0xffffffffu, __float_as_uint(h[4 * c + e]) & 0x7fffffffu);
                if (lane == 0) *reinterpret_cast<uint4 *>(amax + (warp & 3) * TOK + 4 * c) = make_uint4(m[0], m[1], m[2], m[3]);
            }
            __syncthreads();
            store_e4m3_rows<TOK>(amax, h, rows, static_cast<uint8_t *>(p.C) + (long long)row0 * p.ldc + col, p.ldc,
                                 p.scale_c + (long long)row0 * p.ldsc + (mine ? last.nb : 0), p.ldsc, warp == 4);
        } else if (col < p.N) {
            __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(p.C) + (long long)row0 * p.ldc + col;
#pragma unroll
            for (int j = 0; j < kMostChunks * 4; ++j) {
                if (j >= rows) break;
                dst[j * p.ldc] = __float2bfloat16_rn(h[j]);
            }
        }
    }

    // ------------------------------ teardown --------------------------------------------
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (*abort_flag) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
        }
        tc_fence_after();
        tmem_dealloc(tmem_base, L::kTmemCols);
    }
}

template <int KIND, int EPI, int TOK, bool KN>
static int launch_rows(const GroupedCall &c, GroupedParams p) {
    constexpr int NB = gepi_swiglu(EPI) ? 2 : 1;
    using L = RowsLayout<NB, TOK>;
    constexpr int kElem = KIND == MMA_F16 ? 2 : 1;
    constexpr int kBlockK = kRowBytes / kElem;
    auto kern = grouped_rows_kernel<KIND, EPI, TOK, KN>;
    // per size of cluster: how many the device holds at once (the SMs of a GPC do not divide by every size)
    static KernelSetup ks[4];
    int most_clusters[4] = {c.num_sms, 0, 0, 0};
    int rc = O64_OK;
    for (int i = 0; i < 4 && !rc; ++i)
        rc = ks[i].once(
            [&](int *clusters) {
                if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kDynamic) != cudaSuccess) return (int)O64_ERR_CUDA;
                cudaLaunchConfig_t q = {};
                q.gridDim = dim3(1u << i, 1, 1);
                q.blockDim = dim3(L::kThreads, 1, 1);
                q.dynamicSmemBytes = L::kDynamic;
                cudaLaunchAttribute a;
                a.id = cudaLaunchAttributeClusterDimension;
                a.val.clusterDim.x = 1u << i;
                a.val.clusterDim.y = a.val.clusterDim.z = 1;
                q.attrs = &a;
                q.numAttrs = 1;
                int n = 0;
                if (cudaOccupancyMaxActiveClusters(&n, kern, &q) != cudaSuccess) {
                    (void)cudaGetLastError();
                    n = 0;
                }
                *clusters = n;
                return (int)O64_OK;
            },
            &most_clusters[i]);
    if (rc) return rc;
    CUtensorMap tx, tw;
    rc = encode_2d(&tx, c.kind, c.A, c.T, c.K, c.lda, kBlockK, TOK);
    if (!rc)
        rc = KN ? encode_3d(&tw, kElem, c.B, c.N, c.K, c.G, c.ldb, c.stride_b, kRowBytes / kElem, kBlockK, true)
                : encode_3d(&tw, kElem, c.B, c.K, NB * c.N, c.G, c.ldb, c.stride_b, kBlockK, 128, true);
    if (rc) return rc;
    p.num_n_tiles = (int)((c.N + 127) / 128);
    // at most this many tiles (the groups' sizes are on the device)
    const long long most = (c.T / TOK + (c.G < c.T ? c.G : c.T)) * p.num_n_tiles;
    if (most > INT32_MAX - 4 * c.num_sms) return O64_ERR_RANK;
    const long long tiles = c.offsets ? most : (c.T + TOK - 1) / TOK * p.num_n_tiles;
    // Too few tiles for the GPU: the K blocks of each are divided over a cluster, as long as a CTA keeps four
    // of them.
    int S = 1;
    for (int i = 1; i < 4; ++i)
        if (tiles <= most_clusters[i] && p.num_k_blocks >= 4 << i) S = 1 << i;
    p.split = S;
    const int grid = (int)(S > 1 ? tiles * S : (tiles < c.num_sms ? tiles : c.num_sms));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3(L::kThreads, 1, 1);
    cfg.dynamicSmemBytes = L::kDynamic;
    cfg.stream = c.stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)S;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    if (cudaLaunchKernelEx(&cfg, kern, tx, tw, p) != cudaSuccess) {
        (void)cudaGetLastError();
        return O64_ERR_CUDA;
    }
    return O64_OK;
}

// Which kernel, and how many rows of A a tile: the cheaper of  waves * K blocks / S * (time of a K block)  over the
// tiles that the groups' mean size makes (their sizes are on the device).  Microseconds a K block of 128 bytes,
// measured with one to eight waves of tiles at N, K of 2048 to 8192:
//   e4m3 128 x 16 / 32 / 64 / 128 rows: 0.30 / 0.33 / 0.42 / 0.55    two weight blocks (SwiGLU): 0.42 / 0.45 / 0.60
//   bf16 128 x 16 ... 64 rows: 0.26                                   CTA pairs, 256 x 256: e4m3 0.48, bf16 0.46
// e.g. 128 x 8192 x 8192 e4m3: 24 us here on clusters of two, 35 us on pairs; 256 rows: 38 and 36.
int grouped_rows_tile(const GroupedCall &c) {
    if (c.wgrad || c.epi == GEPI_F32 || c.T <= 0) return 0;
    const bool fp8 = c.kind == O64_KIND_FP8, swiglu = gepi_swiglu(c.epi);
    const int64_t groups = c.G < c.T ? c.G : c.T;
    const int64_t mean = (c.T + groups - 1) / groups;
    const int64_t kbs = (c.K * (fp8 ? 1 : 2) + kRowBytes - 1) / kRowBytes;
    const int64_t pair_cols = swiglu ? 128 : 256;
    const int64_t pair_tiles = groups * ((mean + 255) / 256) * ((c.N + pair_cols - 1) / pair_cols);
    const int pairs = c.num_sms / 2;
    double best = (double)((pair_tiles + pairs - 1) / pairs) * kbs * (fp8 ? 0.48 : 0.46);
    static const double us[3][4] = {{0.30, 0.33, 0.42, 0.55}, {0.42, 0.45, 0.60, 0}, {0.26, 0.26, 0.26, 0}};
    int tok = 0;
    for (int i = 0; i < (fp8 && !swiglu ? 4 : 3); ++i) {
        const int64_t tiles = groups * ((mean + (16 << i) - 1) / (16 << i)) * ((c.N + 127) / 128);
        int S = 1;
        while (S < 8 && tiles * S * 2 <= c.num_sms * 9 / 10 && kbs >= 8 * S) S *= 2;
        const double cost = (double)((tiles * S + c.num_sms - 1) / c.num_sms) * kbs / S * us[fp8 ? (swiglu ? 1 : 0) : 2][i];
        if (cost < best) {
            best = cost;
            tok = 16 << i;
        }
    }
    return tok;
}

template <int KIND, int EPI, bool KN = false>
static int launch_rows_tok(const GroupedCall &c, const GroupedParams &p, int tok) {
    if constexpr (KIND == MMA_F8F6F4 && !gepi_swiglu(EPI))
        if (tok == 128) return launch_rows<KIND, EPI, 128, KN>(c, p);
    if (tok == 16) return launch_rows<KIND, EPI, 16, KN>(c, p);
    if (tok == 32) return launch_rows<KIND, EPI, 32, KN>(c, p);
    return launch_rows<KIND, EPI, 64, KN>(c, p);
}

int grouped_rows_launch(const GroupedCall &c, const GroupedParams &p, int tok) {
    if (c.kind == O64_KIND_BF16) {
        if (c.epi == GEPI_BF16) return c.b_kn ? launch_rows_tok<MMA_F16, GEPI_BF16, true>(c, p, tok) : launch_rows_tok<MMA_F16, GEPI_BF16>(c, p, tok);
    } else if (c.kind == O64_KIND_FP8) {
        if (c.epi == GEPI_BF16) return c.b_kn ? launch_rows_tok<MMA_F8F6F4, GEPI_BF16, true>(c, p, tok) : launch_rows_tok<MMA_F8F6F4, GEPI_BF16>(c, p, tok);
        if (c.epi == GEPI_SWIGLU_BF16) return launch_rows_tok<MMA_F8F6F4, GEPI_SWIGLU_BF16>(c, p, tok);
        if (c.epi == GEPI_SWIGLU_E4M3) return launch_rows_tok<MMA_F8F6F4, GEPI_SWIGLU_E4M3>(c, p, tok);
    }
    return O64_ERR_DTYPE;
}

}  // namespace o64
