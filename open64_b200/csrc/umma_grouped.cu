// Products grouped by expert, and the e4m3 product with a scale for each block of 128, on CTA pairs:
// two SMs compute one 256 x 256 tile with tcgen05.mma.cta_group::2, each loading its own 128 rows of
// the first operand and half of the second (as umma_gemm_2cta.cu does for one dense product).
//
//   C[r, :] = A[r, :] * op(B[g])          for the rows r of group g         (forward, input gradient)
//   dB[g]   = dC[rows of g]^T * A[rows of g]                                 (weight gradient)
//   C[m, n] = sum over K blocks b of  sA[m, b] * sB[n / 128, b] * (A8 * B8^T over block b)[m, n]
//
// Groups are ragged and their bounds live in device memory: every CTA walks the same list of tiles,
// group by group, and takes every num_pairs-th one.  A tile never spans two groups; its last rows may
// read the next group's rows (each row of the product depends on its own row of A only) and are not
// stored.  In the weight gradient the rows are the sum's index, so the last block of a group is cut to
// whole K = 16 steps and the rows behind the group's end are cleared in shared memory first.
//
// With block scales the tensor cores never add across K blocks: a block's products go to one of two
// buffers in tensor memory, and eight warps add them, scaled, to sums they keep in registers (128 a
// thread) while the next block is multiplied.  A thread owns one row and two runs of 64 columns 128
// apart, so that each run has one scale per block (and, with the SwiGLU tail, the first run is gate and
// the second the matching up columns).  One packed multiply-add serves two values: 64 of them a thread
// and block against 512 cycles of MMA.
//
// The scales reach the adding warps through a small ring in shared memory that a warp of its own fills four
// K blocks ahead: fetched by each thread for itself two blocks ahead, they cost 600 to 800 cycles a block
// (32 rows are 32 sectors, and the move from one pipeline register to the next waits for the load).
//
// Warp roles (three warpgroups a CTA): 0 loads, 1 issues the MMAs (first CTA of the pair), 2 fetches scales or, in the
// weight gradient, clears the cut last blocks, 4..11 add and store.
// The sums take 128 registers of a thread and two chunks on their way from tensor memory 64 more, so the
// first warpgroup gives its registers up (setmaxnreg: 128 x 56 + 256 x 224 = the 384 x 168 of the launch).
//
// Measured: bf16, one group, 4096 x 8192 x 8192: 324 us = 1696 TFLOP/s (bound by the tensor pipe, busy 95 % of the time);
// its weight gradient 340 us; e4m3 with block scales 248 us = 2215 TFLOP/s, 870 cycles a K block: MMA, commit, the way
// through registers (350 cycles) and the release across the pair are one chain over two buffers (the product without
// block scales: 194 us).  Two MMAs of 128 columns a block with four buffers: 263 us (their issue and A's second read).
// Every wait is bounded, as in the other kernels.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <type_traits>

#include "grouped.cuh"

namespace o64 {

namespace {

constexpr int kGpThreads = 384;
constexpr int kGpLoaderRegs = 56, kGpAdderRegs = 224;
static_assert(128 * kGpLoaderRegs + 256 * kGpAdderRegs <= kGpThreads * 168, "registers of the launch");
constexpr int kGpStages = 6;
constexpr int kGpTileM = 256, kGpTileN = 256;
constexpr int kGpStageBytes = 2 * kABytes;  // this CTA's 128 rows of A and its 128 of B
constexpr int kGpRing = kGpStages * kGpStageBytes;
constexpr int kGpStaging = kGpRing;                       // 8 warps x 4 KB
constexpr int kGpScaleSlots = 3;
constexpr int kGpScaleFloats = 132;  // this CTA's 128 rows, then the two column blocks
constexpr int kGpScales = kGpStaging + 8 * kEpiStagingBytesPerWarp;
constexpr int kGpBars = kGpScales + kGpScaleSlots * kGpScaleFloats * 4;
constexpr int kGpNumBars = 4 * kGpStages + 8 + 2 * kGpScaleSlots;
static_assert(kGpBars % 8 == 0, "barriers");
constexpr int kGpTmemPtr = kGpBars + 8 * kGpNumBars;
constexpr int kGpAbort = kGpTmemPtr + 4;
constexpr int kGpLoaded = kGpAbort + 4;  // the tile that this CTA's loader is at
constexpr int kGpTotal = kGpLoaded + 4;
constexpr int kGpDynamic = kGpTotal + 1024;
static_assert(kGpDynamic <= 227 * 1024, "shared memory");

struct GroupTile {
    int g, begin, end;  // the group's rows
    int mb, nb;
    int kbs;            // K blocks of this tile
};

// The tile list, walked forward only.
struct TileWalk {
    int g = 0;
    int base = 0;  // tiles before group g
    int top = 0;   // the end of the groups before it
};

template <bool WGRAD>
__device__ __forceinline__ bool next_tile(const GroupedParams &p, TileWalk &w, int t, int block_k, GroupTile &tile) {
    for (; w.g < p.G; ++w.g) {
        group_rows<false>(p, w.g, w.top, tile.begin, tile.end);
        const int rows = tile.end - tile.begin;
        const int mt = WGRAD ? p.num_m_tiles : (rows + kGpTileM - 1) / kGpTileM;
        const int tiles = mt * p.num_n_tiles;  // (the host has checked that all of them together fit an int)
        if (t < w.base + tiles) {
            // bands of eight row tiles, rows fastest: a band's rows of A and one column block of B stay in L2
            const int r = t - w.base;
            const int per_band = 8 * p.num_n_tiles;
            const int band = r / per_band, in = r - band * per_band;
            const int height = min(mt - band * 8, 8);
            tile.g = w.g;
            tile.mb = band * 8 + in % height;
            tile.nb = in / height;
            tile.kbs = WGRAD ? (rows + block_k - 1) / block_k : p.num_k_blocks;
            return true;
        }
        w.base += tiles;
        w.top = tile.end;
    }
    return false;
}

// idesc with both operands' majors (make_idesc knows the second operand's only)
__host__ __device__ constexpr uint32_t grouped_idesc(uint32_t fmt, bool a_mn, bool b_mn) {
    return make_idesc(1u, fmt, fmt, b_mn ? 1u : 0u, kGpTileM, kGpTileN) | ((a_mn ? 1u : 0u) << 15);
}

// Waits as mbar_wait_bounded does for a phase that may be many tiles away: the budget starts anew whenever *progress
// has moved.
__device__ __forceinline__ bool mbar_wait_following(uint32_t bar, uint32_t parity, const volatile uint32_t *progress,
                                                    volatile int *abort_flag, int *status_word, int code, uint64_t budget_ns) {
    uint32_t probes = 0, seen = *progress;
    uint64_t t0 = globaltimer_ns();
    while (!mbar_try_wait(bar, parity)) {
        if ((++probes & 255u) != 0) continue;
        if (*abort_flag) return false;
        const uint32_t at = *progress;
        const uint64_t now = globaltimer_ns();
        if (at != seen) {
            seen = at;
            t0 = now;
        } else if (now - t0 > budget_ns) {
            atomicCAS(status_word, 0, code);
            *abort_flag = 1;
            return false;
        }
    }
    return true;
}

}  // namespace

// KIND: MMA_F16 (bf16) or MMA_F8F6F4 (e4m3 with block scales).  WGRAD: both operands lie with the sum's
// index outermost.  B_KN: the second operand does.
template <int KIND, bool WGRAD, bool B_KN, int EPI>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGpThreads, 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                    const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ GroupedParams p) {
    constexpr bool kScaled = KIND == MMA_F8F6F4;
    constexpr int kElem = KIND == MMA_F16 ? 2 : 1;
    constexpr int kBlockK = kRowBytes / kElem;
    constexpr int kMmaK = 32 / kElem;
    constexpr bool kSwiglu = gepi_swiglu(EPI);
    constexpr bool kBMn = WGRAD || B_KN;
    constexpr int kKnCols = kRowBytes / kElem;              // columns in a 128-byte row of an MN-major operand
    constexpr int kKnGroupBytes = kBlockK * kRowBytes;      // kBlockK such rows
    constexpr int kKnGroups = 128 / kKnCols;
    constexpr int kOutN = kSwiglu ? kGpTileN / 2 : kGpTileN;
    constexpr uint32_t kTmemCols = 512;
    static_assert(!kScaled || !WGRAD, "the weight gradient is a bf16 product");

    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bar_base = smem_base + kGpBars;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kGpStages + s); };
    auto acc_full_bar = [&](int b) { return bar_base + 8u * (2 * kGpStages + b); };
    auto acc_empty_bar = [&](int b) { return bar_base + 8u * (2 * kGpStages + 2 + b); };
    auto half_bar = [&](int quarter) { return bar_base + 8u * (2 * kGpStages + 4 + quarter); };
    auto scale_full_bar = [&](int s) { return bar_base + 8u * (2 * kGpStages + 8 + s); };
    auto scale_empty_bar = [&](int s) { return bar_base + 8u * (2 * kGpStages + 8 + kGpScaleSlots + s); };
    // a group's cut last block: this CTA's half has come; first CTA: the second's half is cleared
    auto tail_bar = [&](int s) { return bar_base + 8u * (2 * kGpStages + 8 + 2 * kGpScaleSlots + s); };
    auto cleared_bar = [&](int s) { return bar_base + 8u * (3 * kGpStages + 8 + 2 * kGpScaleSlots + s); };
    // WGRAD: a tile's K blocks that need no clearing (rows up to a whole K step; what lies behind is not multiplied)
    [[maybe_unused]] auto whole_blocks = [](const GroupTile &t) {
        return (t.end - t.begin) % kMmaK == 0 ? t.kbs : (t.end - t.begin) / kBlockK;
    };
    volatile uint32_t *tmem_ptr_smem = reinterpret_cast<volatile uint32_t *>(smem_gen + kGpTmemPtr);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem_gen + kGpAbort);

    [[maybe_unused]] volatile uint32_t *loaded = reinterpret_cast<volatile uint32_t *>(smem_gen + kGpLoaded);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const int pair_id = (int)cluster_id_x();
    const int num_pairs = (int)num_clusters_x();

    if (threadIdx.x == 0) {
        for (int s = 0; s < kGpStages; ++s) {
            mbar_init(full_bar(s), 1);  // first CTA: its loader's arrival
            mbar_init(empty_bar(s), 1);
            mbar_init(tail_bar(s), 1);
            mbar_init(cleared_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full_bar(b), 1);
            mbar_init(acc_empty_bar(b), 16);  // eight warps in each CTA
        }
        for (int s = 0; s < kGpScaleSlots; ++s) {
            mbar_init(scale_full_bar(s), 1);
            mbar_init(scale_empty_bar(s), 8);
        }
        for (int q = 0; q < 4; ++q) mbar_init(half_bar(q), 2);  // the two warps that share 32 rows
        *abort_flag = 0;
        *loaded = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tm_a);
        tma_prefetch_desc(&tm_b);
        if (p.tma_store) tma_prefetch_desc(&tm_c);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(smem_gen + kGpTmemPtr), kTmemCols);
        tmem_relinquish();
    }
    if (p.offsets && blockIdx.x == 0 && warp == 2) {  // offsets that are not ascending within 0 .. T are reported
        for (int g = lane; g < p.G; g += 32) {
            int b, e;
            bool bad;
            group_rows<false>(p, g, 0, b, e, &bad);
            if (bad) atomicCAS(p.status, 0, kBadOffsets);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_ptr_smem;
    if (threadIdx.x == 0 && (tmem_base & 0xffffu) != 0) {  // all 512 columns: always at zero
        atomicCAS(p.status, 0, kWaitGroupAccEmpty | (int)((tmem_base & 0xfffu) << 12));
        *abort_flag = 1;
    }

    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kGpLoaderRegs));
    if (warp == 0) {
        // ------------------------------ loads (both CTAs) -----------------------------------
        const bool leader = elect_one();
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        TileWalk walk;
        GroupTile t;
        for (int i = pair_id; ok && next_tile<WGRAD>(p, walk, i, kBlockK, t); i += num_pairs) {
            const int m0 = t.mb * kGpTileM + (int)rank * kBlockM;
            const int n0 = t.nb * kOutN;
            // WGRAD: the maps count the columns in groups of 64 or, where the last group is not whole, one by one (two
            // boxes a stage instead of four: the issuing thread needs about 100 cycles for each)
            [[maybe_unused]] const int xa = p.a_groups ? 0 : m0, za = p.a_groups ? m0 / kKnCols : 0;
            [[maybe_unused]] const int xb = p.b_groups ? 0 : n0 + (int)rank * 128, zb = p.b_groups ? (n0 + (int)rank * 128) / kKnCols : 0;
            auto load_block = [&](int kb, auto cut) __attribute__((always_inline)) {
                ok = mbar_wait_bounded(empty_bar(stage), phase ^ 1u, abort_flag, p.status, kWaitGroupProducer, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                const uint32_t a_dst = smem_base + stage * kGpStageBytes;
                const uint32_t b_dst = a_dst + kABytes;
                if (leader) {
                    uint32_t bar;
                    if constexpr (decltype(cut)::value) {  // the clearing warps pass it on
                        mbar_arrive_expect_tx(tail_bar(stage), kGpStageBytes);
                        bar = map_to_cta(tail_bar(stage), rank);
                    } else {
                        if (rank == 0) mbar_arrive_expect_tx(full_bar(stage), 2 * kGpStageBytes);
                        bar = map_to_cta(full_bar(stage), 0);
                    }
                    if constexpr (WGRAD) {
                        const int row = t.begin + kb * kBlockK;
                        tma_load_3d_pair(a_dst, &tm_a, xa, row, za, bar);
                        tma_load_3d_pair(b_dst, &tm_b, xb, row, zb, bar);
                        if (!p.a_groups) tma_load_3d_pair(a_dst + kKnGroupBytes, &tm_a, xa + kKnCols, row, 0, bar);
                        if (!p.b_groups) tma_load_3d_pair(b_dst + kKnGroupBytes, &tm_b, xb + kKnCols, row, 0, bar);
                    } else {
                        tma_load_2d_pair(a_dst, &tm_a, kb * kBlockK, t.begin + m0, bar);
                        if constexpr (B_KN) {
#pragma unroll
                            for (int c = 0; c < kKnGroups; ++c)
                                tma_load_3d_pair(b_dst + c * kKnGroupBytes, &tm_b, n0 + (int)rank * 128 + c * kKnCols, kb * kBlockK, t.g, bar);
                        } else {
                            // SwiGLU: the first CTA holds gate rows, the second the matching up rows
                            const int y = kSwiglu ? n0 + (rank ? p.N : 0) : n0 + (int)rank * 128;
                            tma_load_3d_pair(b_dst, &tm_b, kb * kBlockK, y, t.g, bar);
                        }
                    }
                }
                __syncwarp();
                if (++stage == kGpStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            if constexpr (WGRAD) {
                if (leader) *loaded = (uint32_t)i + 1;
                const int whole = whole_blocks(t);
                for (int kb = 0; ok && kb < whole; ++kb) load_block(kb, std::false_type());
                if (ok && whole < t.kbs) load_block(whole, std::true_type());
            } else {
                for (int kb = 0; ok && kb < t.kbs; ++kb) load_block(kb, std::false_type());
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------ MMA (first CTA) -------------------------------------
        if (rank == 0) {
            const bool leader = elect_one();
            constexpr uint32_t idesc = grouped_idesc(KIND == MMA_F8F6F4 ? 0u : 1u, WGRAD, kBMn);
            constexpr uint32_t kAAdvance = WGRAD ? (kMmaK * kRowBytes) >> 4 : 2;
            constexpr uint32_t kBAdvance = kBMn ? (kMmaK * kRowBytes) >> 4 : 2;
            int stage = 0;
            uint32_t phase = 0;
            uint32_t uses = 0;  // accumulator buffers taken so far
            bool ok = true;
            // the next stage's barrier is probed before this stage's MMAs are issued, so that the probe's
            // latency opens no gap between them
            uint32_t ready = mbar_test_wait(full_bar(0), 0);
            TileWalk walk;
            GroupTile t;
            uint32_t acc_ready = 0;
            auto take = [&] {
                if (!acc_ready)
                ok = mbar_wait_bounded(acc_empty_bar(uses & 1), (uint32_t)((uses >> 1) & 1) ^ 1u, abort_flag, p.status,
                                       kWaitGroupAccEmpty, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
            };
            for (int i = pair_id; ok && next_tile<WGRAD>(p, walk, i, kBlockK, t); i += num_pairs) {
                if (!kScaled && t.kbs > 0) take();
                for (int kb = 0; ok && kb < t.kbs; ++kb) {
                    if (kScaled) {
                        take();
                        if (!ok) break;
                    }
                    if (!__all_sync(0xffffffffu, ready)) {
                        ok = mbar_wait_bounded(full_bar(stage), phase, abort_flag, p.status, kWaitGroupFull, p.wait_ns);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                    }
                    const int next_stage = (stage + 1 == kGpStages) ? 0 : stage + 1;
                    const uint32_t next_phase = (stage + 1 == kGpStages) ? (phase ^ 1u) : phase;
                    const uint32_t next_ready = mbar_test_wait(full_bar(next_stage), next_phase);
                    if (kScaled) acc_ready = mbar_test_wait(acc_empty_bar((uses + 1) & 1), (uint32_t)(((uses + 1) >> 1) & 1) ^ 1u);
                    tc_fence_after();
                    const uint32_t a_addr = smem_base + stage * kGpStageBytes;
                    const uint32_t b_addr = a_addr + kABytes;
                    const uint64_t a_desc = make_smem_desc(a_addr, WGRAD ? kKnGroupBytes : 16, 1024);
                    const uint64_t b_desc = make_smem_desc(b_addr, kBMn ? kKnGroupBytes : 16, 1024);
                    const uint32_t d_tmem = tmem_base + (uint32_t)(uses & 1) * kGpTileN;
                    int steps = kRowBytes / 32;
                    if constexpr (WGRAD) steps = min(steps, (t.end - t.begin - kb * kBlockK + kMmaK - 1) / kMmaK);
                    if (leader) {
                        if (steps == kRowBytes / 32) {
#pragma unroll
                            for (int k = 0; k < kRowBytes / 32; ++k)
                                tc_mma_pair<KIND>(d_tmem, a_desc + kAAdvance * k, b_desc + kBAdvance * k, idesc,
                                                  (kScaled ? k : (kb | k)) != 0 ? 1u : 0u);
                        } else {
                            for (int k = 0; k < steps; ++k)
                                tc_mma_pair<KIND>(d_tmem, a_desc + kAAdvance * k, b_desc + kBAdvance * k, idesc, (kb | k) != 0 ? 1u : 0u);
                        }
                        tc_commit_pair_mask(empty_bar(stage), 3);
                        if (kScaled) tc_commit_pair_mask(acc_full_bar(uses & 1), 3);
                    }
                    __syncwarp();
                    if (kScaled) ++uses;
                    stage = next_stage;
                    phase = next_phase;
                    ready = next_ready;
                }
                if (!kScaled && t.kbs > 0) {
                    if (ok && leader) tc_commit_pair_mask(acc_full_bar(uses & 1), 3);
                    __syncwarp();
                    ++uses;
                }
            }
        }
        __syncwarp();
    } else if (WGRAD && warp == 2) {
        // ------------------------------ cut last blocks (both CTAs) --------------------------
        // The rows from a group's end to the next whole K step are cleared in both operands (whatever lies behind the
        // group may be NaN).  The second CTA says so to the first, whose arrival on the stage's full barrier stands for
        // both.  Every barrier of this way is the stage's own: nobody speaks on one again before the stage is free
        // again, so before it has been heard.  (On one barrier for all stages the second CTA could be two tails ahead,
        // whose parity is that of none.)  A warp of its own, since the loading warp stands still meanwhile and longer for
        // the arrival that publishes plain writes to the other CTA: 8192 rows, 8 experts of 4096 x 14336, 900-1000 us with
        // the clearing there, 850-875 us here.
        uint32_t phases = 0;  // a bit for each stage
        int done = 0;         // blocks before this tile, modulo the ring
        bool ok = true;
        TileWalk walk;
        GroupTile t;
        for (int i = pair_id; ok && next_tile<WGRAD>(p, walk, i, kBlockK, t); i += num_pairs) {
            const int stage = (done + t.kbs - 1 + kGpStages) % kGpStages;
            done = (done + t.kbs) % kGpStages;
            if (whole_blocks(t) == t.kbs) continue;
            const uint32_t phase = (phases >> stage) & 1u;
            phases ^= 1u << stage;
            ok = mbar_wait_following(tail_bar(stage), phase, loaded, abort_flag, p.status, kWaitGroupTail, p.wait_ns);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            const int first = (t.end - t.begin) % kBlockK, last = (first + kMmaK - 1) / kMmaK * kMmaK;
            uint8_t *at = smem_gen + stage * kGpStageBytes;
            for (int c = 0; c < 2 * kKnGroups; ++c)
                for (int q = first * 8 + lane; q < last * 8; q += 32)
                    reinterpret_cast<uint4 *>(at + c * kKnGroupBytes)[q] = make_uint4(0, 0, 0, 0);
            fence_proxy_async_smem();
            __syncwarp();
            if (rank == 1) {
                if (lane == 0) mbar_arrive_release_cluster(map_to_cta(cleared_bar(stage), 0));
            } else {
                ok = mbar_wait_bounded(cleared_bar(stage), phase, abort_flag, p.status, kWaitGroupTail, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                mbar_acquire_cluster(cleared_bar(stage), phase);
                if (lane == 0) mbar_arrive(full_bar(stage));
            }
            __syncwarp();
        }
        __syncwarp();
    } else if (kScaled && warp == 2) {
        // ------------------------------ scales (both CTAs) ----------------------------------
        float *ring = reinterpret_cast<float *>(smem_gen + kGpScales);
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        TileWalk walk;
        GroupTile t;
        // lane l carries rows l, l + 32, l + 64, l + 96 and, for l < 2, one of the two runs of columns; four K
        // blocks at a time, the next four (of this tile or of the next one) always on their way
        const float *sa[4], *sb = nullptr;
        const long long sb_step = B_KN ? p.ldsb : 1;
        float next[5][4];
        int tile = pair_id, kb0 = 0;
        auto fetch = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (p.sa_vec && kb0 + 4 <= t.kbs) {
                    const float4 x = __ldg(reinterpret_cast<const float4 *>(sa[r] + kb0));
                    next[r][0] = x.x, next[r][1] = x.y, next[r][2] = x.z, next[r][3] = x.w;
                } else {
#pragma unroll
                    for (int u = 0; u < 4; ++u) next[r][u] = kb0 + u < t.kbs ? __ldg(sa[r] + kb0 + u) : 0.0f;
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) next[4][u] = lane < 2 && kb0 + u < t.kbs ? __ldg(sb + (kb0 + u) * sb_step) : 0.0f;
        };
        auto begin_tile = [&]() __attribute__((always_inline)) {
            if (!next_tile<WGRAD>(p, walk, tile, kBlockK, t)) return false;
            const int n0 = t.nb * kOutN;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                sa[r] = p.scale_a + (long long)min(t.begin + t.mb * kGpTileM + (int)rank * kBlockM + r * 32 + lane, t.end - 1) * p.ldsa;
            // the block of 128 columns of C (SwiGLU: of gate, or of up) behind run `lane`
            const int blk = kSwiglu ? ((lane & 1 ? p.N + n0 : n0) >> 7) : min((n0 >> 7) + (lane & 1), (p.N - 1) >> 7);
            sb = p.scale_b + (long long)t.g * p.stride_sb + (B_KN ? (long long)blk : blk * p.ldsb);
            kb0 = 0;
            fetch();
            return true;
        };
        bool more = begin_tile();
        while (ok && more) {
            float now[5][4];
            const int have = min(4, t.kbs - kb0);
#pragma unroll
            for (int r = 0; r < 5; ++r)
#pragma unroll
                for (int u = 0; u < 4; ++u) now[r][u] = next[r][u];
            kb0 += 4;
            if (kb0 < t.kbs) {
                fetch();
            } else {
                tile += num_pairs;
                more = begin_tile();
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                if (u >= have) break;
                ok = mbar_wait_bounded(scale_empty_bar(slot), phase ^ 1u, abort_flag, p.status, kWaitGroupScales, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                float *dst = ring + slot * kGpScaleFloats;
#pragma unroll
                for (int r = 0; r < 4; ++r) dst[r * 32 + lane] = now[r][u];
                if (lane < 2) dst[128 + lane] = now[4][u];
                __syncwarp();
                if (lane == 0) mbar_arrive(scale_full_bar(slot));
                if (++slot == kGpScaleSlots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
        }
        __syncwarp();
    }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kGpAdderRegs));
        // ------------------------------ sums, tails and stores (both CTAs) ------------------
        const int quarter = warp & 3;
        const int half = (warp - 4) >> 2;
        uint8_t *staging = smem_gen + kGpStaging + (warp - 4) * kEpiStagingBytesPerWarp;
        uint4 *patch = reinterpret_cast<uint4 *>(staging);
        const int sw = lane & 7;
        const uint32_t t_lane = tmem_base + (uint32_t(quarter * 32) << 16) + half * 64;
        uint32_t uses = 0;
        bool ok = true;
        [[maybe_unused]] uint32_t half_phase = 0, slot_phase = 0;
        [[maybe_unused]] int slot = 0;
        TileWalk walk;
        GroupTile t;
        for (int i = pair_id; ok && next_tile<WGRAD>(p, walk, i, kBlockK, t); i += num_pairs) {
            const int n0 = t.nb * kOutN;
            const int slab0 = t.mb * kGpTileM + (int)rank * kBlockM + quarter * 32;  // of the group's rows (or of dB's)
            float2 acc[2][32];
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int j = 0; j < 32; ++j) acc[r][j] = make_float2(0.0f, 0.0f);

            if constexpr (kScaled) {
                const float *ring = reinterpret_cast<const float *>(smem_gen + kGpScales);
                uint32_t scale_ready = 0;  // the next block's scales, probed while this one is added
#pragma unroll 1
                for (int kb = 0; kb < t.kbs; ++kb, ++uses) {
                    // the block's scales first: they are there long before its products are
                    if (!scale_ready) ok = mbar_wait_bounded(scale_full_bar(slot), slot_phase, abort_flag, p.status, kWaitGroupScales, p.wait_ns);
                    const float s = ring[slot * kGpScaleFloats + quarter * 32 + lane];
                    const float2 sb = *reinterpret_cast<const float2 *>(ring + slot * kGpScaleFloats + 128);
                    const float f0 = s * sb.x, f1 = s * sb.y;
                    ok = mbar_wait_bounded(acc_full_bar(uses & 1), (uint32_t)((uses >> 1) & 1), abort_flag, p.status, kWaitGroupAccFull,
                                           p.wait_ns) && ok;
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t t_row = t_lane + (uint32_t)(uses & 1) * kGpTileN;
                    // 64 columns at a time; the second 64 set out as soon as the registers of the first are free
                    uint32_t va[32], vb[32];
                    tmem_ld_32x32(t_row, va);
                    tmem_ld_32x32(t_row + 32, vb);
                    auto add = [&](const uint32_t(&v)[32], float2(&sum)[32], int at, float f) __attribute__((always_inline)) {
#pragma unroll
                        for (int j = 0; j < 16; ++j)
                            sum[at + j] = __ffma2_rn(make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1])),
                                                     make_float2(f, f), sum[at + j]);
                    };
                    tmem_ld_wait();
                    add(va, acc[0], 0, f0);
                    tmem_ld_32x32(t_row + 128, va);
                    add(vb, acc[0], 16, f0);
                    tmem_ld_32x32(t_row + 160, vb);
                    tmem_ld_wait();
                    tc_fence_before();  // everything of this buffer is in registers
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive_cluster(map_to_cta(acc_empty_bar(uses & 1), 0));
                        mbar_arrive(scale_empty_bar(slot));
                    }
                    if (++slot == kGpScaleSlots) {
                        slot = 0;
                        slot_phase ^= 1u;
                    }
                    scale_ready = mbar_test_wait(scale_full_bar(slot), slot_phase);
                    add(va, acc[1], 0, f1);
                    add(vb, acc[1], 16, f1);
                }
            } else if (t.kbs > 0) {
                if (lane == 0)
                    ok = mbar_wait_bounded(acc_full_bar(uses & 1), (uint32_t)((uses >> 1) & 1), abort_flag, p.status,
                                           kWaitGroupAccFull, p.wait_ns);
                ok = __shfl_sync(0xffffffffu, ok, 0);
                __syncwarp();  // (orders memory, which the shuffle does not: the other lanes read what lane 0 has waited for)
                if (!ok) break;
                tc_fence_after();
                const uint32_t t_row = t_lane + (uint32_t)(uses & 1) * kGpTileN;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t v[32];
                    tmem_ld_32x32(t_row + (c >> 1) * 128 + (c & 1) * 32, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        acc[c >> 1][(c & 1) * 16 + j] = make_float2(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(map_to_cta(acc_empty_bar(uses & 1), 0));
                ++uses;
            }
            if (!ok) break;

            // ---- the tile leaves: 32 rows x 128 bytes at a time through this warp's patch ----
            const int rows_here = (WGRAD ? p.rows_m : t.end - t.begin) - slab0;  // rows of this warp's slab that exist
            const long long grow0 = (WGRAD ? 0 : t.begin) + slab0;
            constexpr int kOutElem = gepi_bytes(EPI);
            uint8_t *c_group = static_cast<uint8_t *>(p.C) + (WGRAD ? (long long)t.g * p.stride_c * kOutElem : 0);
            // sends the patch out: `cols` result columns from column `col` on, kOutElem bytes each
            auto send = [&](int col, int cols) __attribute__((always_inline)) {
                const int bytes = cols * kOutElem;
                if (p.tma_store && bytes == 128 && rows_here >= 32 && col + cols <= p.N) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        tma_store_3d(&tm_c, smem_base + kGpStaging + (warp - 4) * kEpiStagingBytesPerWarp, col * kOutElem, (int)grow0,
                                     WGRAD ? t.g : 0);
                        bulk_commit_group();
                    }
                    return;
                }
                __syncwarp();
                const int pieces = bytes / 16;  // 8 or 4
                for (int q = lane; q < 32 * pieces; q += 32) {
                    const int r = q / pieces, piece = q % pieces;
                    if (r < rows_here) {
                        const uint4 val = patch[r * 8 + (piece ^ (r & 7))];
                        uint8_t *dst = c_group + ((grow0 + r) * p.ldc + col) * kOutElem + piece * 16;
                        const int have = (p.N - col) * kOutElem - piece * 16;  // bytes of this piece inside the row
                        if (p.vec_ok && have >= 16) {
                            *reinterpret_cast<uint4 *>(dst) = val;
                        } else if (have > 0) {
                            const uint32_t w[4] = {val.x, val.y, val.z, val.w};
#pragma unroll
                            for (int b = 0; b < 16 / kOutElem; ++b)
                                if (b * kOutElem < have) {
                                    if constexpr (kOutElem == 4)
                                        reinterpret_cast<uint32_t *>(dst)[b] = w[b];
                                    else if constexpr (kOutElem == 2)
                                        reinterpret_cast<uint16_t *>(dst)[b] = (uint16_t)(w[b >> 1] >> (16 * (b & 1)));
                                    else
                                        dst[b] = (uint8_t)(w[b >> 2] >> (8 * (b & 3)));
                                }
                        }
                    }
                }
                __syncwarp();
            };
            auto patch_free = [&] {  // the bulk store of the patch's last contents has read it
                if (p.tma_store) {
                    if (lane == 0) bulk_wait_read_all();
                    __syncwarp();
                }
            };
            if constexpr (EPI == GEPI_SWIGLU_E4M3) {
                // the two warps that share these rows (a bounded wait like all others: no named barrier)
                auto meet = [&] {
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(half_bar(quarter));
                        ok = mbar_wait_bounded(half_bar(quarter), half_phase, abort_flag, p.status, kWaitGroupHalf, p.wait_ns);
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    __syncwarp();  // (orders memory, which the shuffle does not: the other lanes read what lane 0 has waited for)
                    half_phase ^= 1u;
                };
                float amax = 0.0f;
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    float2 &h = acc[0][j];
                    h = silu_mul2(h, acc[1][j]);
                    amax = max_nan(amax, max_nan(fabsf(h.x), fabsf(h.y)));
                }
                // the row's other 64 columns are with the warp of the other half
                patch_free();
                reinterpret_cast<float *>(patch)[lane] = amax;
                meet();
                if (!ok) break;
                amax = max_nan(amax, reinterpret_cast<const float *>(smem_gen + kGpStaging + ((half ^ 1) * 4 + (warp & 3)) * kEpiStagingBytesPerWarp)[lane]);
                meet();  // read before the values overwrite it
                if (!ok) break;
                const float scale = block_scale_of(amax);
                if (half == 0 && lane < rows_here) p.scale_c[(grow0 + lane) * p.ldsc + t.nb] = scale;
                const float inv = 1.0f / scale, back = remainder_scale(scale);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = quant2(acc[0][q * 8 + e * 2], back, inv) | quant2(acc[0][q * 8 + e * 2 + 1], back, inv) << 16;
                    patch[lane * 8 + (q ^ sw)] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                if (rows_here > 0) send(n0 + half * 64, 64);
            } else if constexpr (EPI == GEPI_F32) {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    patch_free();
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const float2 a = acc[s >> 1][(s & 1) * 16 + 2 * q], b = acc[s >> 1][(s & 1) * 16 + 2 * q + 1];
                        patch[lane * 8 + (q ^ sw)] =
                            make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
                    }
                    if (rows_here > 0) send(n0 + (s >> 1) * 128 + half * 64 + (s & 1) * 32, 32);
                }
            } else {
                if constexpr (EPI == GEPI_SWIGLU_BF16) {
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        acc[0][j] = silu_mul2(acc[0][j], acc[1][j]);
                }
#pragma unroll
                for (int s = 0; s < (kSwiglu ? 1 : 2); ++s) {
                    patch_free();
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        patch[lane * 8 + (q ^ sw)] = make_uint4(
                            pack_bf16x2(acc[s][4 * q].x, acc[s][4 * q].y), pack_bf16x2(acc[s][4 * q + 1].x, acc[s][4 * q + 1].y),
                            pack_bf16x2(acc[s][4 * q + 2].x, acc[s][4 * q + 2].y), pack_bf16x2(acc[s][4 * q + 3].x, acc[s][4 * q + 3].y));
                    if (rows_here > 0) send(n0 + s * 128 + half * 64, 64);
                }
            }
        }
        if (p.tma_store && lane == 0) bulk_wait_all();
    }

    // ------------------------------ teardown --------------------------------------------
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        if (*abort_flag) {
            const uint64_t t0 = globaltimer_ns();
            while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
        }
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// Sets a rectangle of rows of each group (or of each dB) to the empty sum.
__global__ void grouped_zero_kernel(const GroupedParams p, int elem, int wgrad) {
    for (int g = blockIdx.y; g < p.G; g += gridDim.y) {
        int b = 0, e = p.rows_m;
        if (!wgrad) group_rows<false>(p, g, 0, b, e);
        uint8_t *c = static_cast<uint8_t *>(p.C) + (wgrad ? (long long)g * p.stride_c * elem : 0);
        for (long long r = b + blockIdx.x; r < e; r += gridDim.x) {
            for (long long i = threadIdx.x; i < (long long)p.N * elem; i += blockDim.x) c[r * p.ldc * elem + i] = 0;
            if (p.scale_c)
                for (int i = threadIdx.x; i < (p.N + 127) / 128; i += blockDim.x) p.scale_c[r * p.ldsc + i] = 1.0f;
        }
    }
}

static GroupedParams grouped_params(const GroupedCall &c) {
    GroupedParams p;
    p.G = (int)c.G;
    p.T = (int)c.T;
    p.K = (int)c.K;
    p.N = (int)(c.wgrad ? c.K : c.N);
    p.rows_m = (int)c.N;
    p.C = c.C;
    p.ldc = c.ldc;
    p.stride_c = c.stride_c;
    p.scale_a = c.scale_a;
    p.scale_b = c.scale_b;
    p.ldsa = c.ldsa;
    p.ldsb = c.ldsb;
    p.stride_sb = c.stride_sb;
    p.scale_c = c.scale_c;
    p.ldsc = c.ldsc;
    p.offsets = c.offsets;
    p.status = c.status_word;
    p.wait_ns = c.wait_ns ? c.wait_ns : kDefaultWaitNs;
    const int elem = gepi_bytes(c.epi);
    p.vec_ok = (reinterpret_cast<uintptr_t>(c.C) & 15u) == 0 && (c.ldc * elem) % 16 == 0 && (c.stride_c * elem) % 16 == 0;
    p.tma_store = 0;
    p.split = 1;
    p.a_groups = p.b_groups = 0;
    p.sa_vec = (reinterpret_cast<uintptr_t>(c.scale_a) & 15u) == 0 && c.ldsa % 4 == 0;
    p.num_m_tiles = (int)((c.N + kGpTileM - 1) / kGpTileM);
    const int out_n = gepi_swiglu(c.epi) ? kGpTileN / 2 : kGpTileN;
    p.num_n_tiles = (int)((p.N + out_n - 1) / out_n);
    const int block_k = kRowBytes / (c.kind == O64_KIND_BF16 ? 2 : 1);
    p.num_k_blocks = (int)((c.K + block_k - 1) / block_k);
    return p;
}

int grouped_zero_launch(const GroupedCall &c) {
    GroupedParams p = grouped_params(c);
    const dim3 grid(256, (unsigned)(c.G < 64 ? c.G : 64));
    grouped_zero_kernel<<<grid, 256, 0, c.stream>>>(p, gepi_bytes(c.epi), c.wgrad ? 1 : 0);
    return cudaGetLastError() == cudaSuccess ? O64_OK : O64_ERR_CUDA;
}

template <int KIND, bool WGRAD, bool B_KN, int EPI>
static int launch_grouped(const CUtensorMap &ta, const CUtensorMap &tb, const CUtensorMap &tc, const GroupedParams &p, int num_sms,
                          cudaStream_t stream) {
    auto kern = grouped_pair_kernel<KIND, WGRAD, B_KN, EPI>;
    static KernelSetup ks;
    const int rc = ks.once(
        [&](int *) {
            return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGpDynamic) == cudaSuccess
                       ? (int)O64_OK
                       : (int)O64_ERR_CUDA;
        },
        nullptr);
    if (rc) return rc;
    // one pair per two SMs; no more than there can be tiles
    const long long most = WGRAD ? (long long)p.G * p.num_m_tiles * p.num_n_tiles
                                 : ((long long)p.T / kGpTileM + (p.G < p.T ? p.G : p.T)) * p.num_n_tiles;
    if (most > INT32_MAX - num_sms) return O64_ERR_RANK;  // the walk counts tiles in 32 bits
    const int pairs = (int)(most < num_sms / 2 ? (most < 1 ? 1 : most) : num_sms / 2);
    kern<<<2 * pairs, kGpThreads, kGpDynamic, stream>>>(ta, tb, tc, p);
    return cudaGetLastError() == cudaSuccess ? O64_OK : O64_ERR_CUDA;
}

int grouped_launch(const GroupedCall &c) {
    GroupedParams p = grouped_params(c);
    if (const int tok = grouped_rows_tile(c)) return grouped_rows_launch(c, p, tok);
    const int elem = c.kind == O64_KIND_BF16 ? 2 : 1;
    const int block_k = kRowBytes / elem;
    CUtensorMap ta, tb, tc;
    int rc;
    if (c.wgrad) {
        // an operand whose columns come in whole groups of 64 as [group][row][64]: a box of two groups is what a
        // CTA holds of it.  (A last group that is not whole would be read past the rows' ends.)
        auto encode = [&](CUtensorMap *tm, const void *base, int64_t cols, int64_t ld, int *groups) {
            *groups = cols % 64 == 0;
            return *groups ? encode_3d(tm, 2, base, 64, c.T, cols / 64, ld, 64, 64, 64, true, 2)
                           : encode_3d(tm, 2, base, cols, c.T, 1, ld, 0, 64, 64, true);
        };
        rc = encode(&ta, c.A, c.N, c.lda, &p.a_groups);
        if (!rc) rc = encode(&tb, c.B, c.K, c.ldb, &p.b_groups);
    } else {
        const int64_t b_out = gepi_swiglu(c.epi) ? 2 * c.N : c.N;
        rc = encode_2d(&ta, c.kind, c.A, c.T, c.K, c.lda, block_k, kBlockM);
        if (!rc)
            rc = c.b_kn ? encode_3d(&tb, elem, c.B, b_out, c.K, c.G, c.ldb, c.stride_b, block_k, block_k, true)
                        : encode_3d(&tb, elem, c.B, c.K, b_out, c.G, c.ldb, c.stride_b, block_k, 128, true);
    }
    if (rc) return rc;
    tc = ta;
    const int out_elem = gepi_bytes(c.epi);
    if (p.vec_ok && (int64_t)p.N * out_elem >= 128) {
        const int64_t rows = c.wgrad ? c.N : c.T;
        rc = encode_3d(&tc, 1, c.C, (int64_t)p.N * out_elem, rows, c.wgrad ? c.G : 1, c.ldc * out_elem, c.stride_c * out_elem, 128, 32, false);
        if (rc) return rc;
        p.tma_store = 1;
    }
#define O64_GROUPED(KIND, WG, KN, EPI_) return launch_grouped<KIND, WG, KN, EPI_>(ta, tb, tc, p, c.num_sms, c.stream)
    if (c.kind == O64_KIND_BF16) {
        if (c.wgrad) {
            if (c.epi == GEPI_BF16) O64_GROUPED(MMA_F16, true, false, GEPI_BF16);
            if (c.epi == GEPI_F32) O64_GROUPED(MMA_F16, true, false, GEPI_F32);
        } else if (c.epi == GEPI_BF16) {
            if (c.b_kn) O64_GROUPED(MMA_F16, false, true, GEPI_BF16);
            O64_GROUPED(MMA_F16, false, false, GEPI_BF16);
        }
    } else if (c.kind == O64_KIND_FP8) {
        if (c.epi == GEPI_BF16) {
            if (c.b_kn) O64_GROUPED(MMA_F8F6F4, false, true, GEPI_BF16);
            O64_GROUPED(MMA_F8F6F4, false, false, GEPI_BF16);
        }
        if (!c.b_kn && c.epi == GEPI_SWIGLU_BF16) O64_GROUPED(MMA_F8F6F4, false, false, GEPI_SWIGLU_BF16);
        if (!c.b_kn && c.epi == GEPI_SWIGLU_E4M3) O64_GROUPED(MMA_F8F6F4, false, false, GEPI_SWIGLU_E4M3);
    }
#undef O64_GROUPED
    return O64_ERR_DTYPE;
}

}  // namespace o64
