// RMS norm in front of (and, in training, behind) the products: the residual's addition, the norm and
// the 8-bit operand the next product reads, in one pass over the row.
//
//   s = x + r          h[j] = s[j] / sqrt(mean(s^2) + eps) * w[j]
//   e4m3: scale = max |h| over 128 columns (or the row) / 448, q = e4m3(h / scale)
//
// A row of at most 32768 columns stays in the registers of one group of threads between the two
// things that need all of it (the mean, the largest value), so every operand crosses HBM once.  The
// norm is taken of the sum in fp32; the stream s that goes on to the next layer is that sum rounded
// to bf16 once.
//
// Bound by HBM: 16384 x 8192 with the residual to e4m3 153 to 174 us on several B200s = 5.4 to 6.1 TB/s (0.83 to 0.94 of a
// copy), backward 8192 x 8192 with the residual 94 us = 5.7 TB/s.  Many rows run on a few blocks per SM that stay: rows come in by bulk copies, a ring of
// three ahead, so that loads go on while a row is reduced, converted and stored, and a thread keeps its
// columns of w.  Few rows run on a block per row that loads for itself.
//
// Gradient, with n = s * rstd, g = dy * w:   dx = rstd * (g - n * mean(g n)) + dr   (x and r receive
// the same one),   dw[j] = sum over rows of dy n.  The sum over rows runs in two fixed stages (a
// partial row per thread group, then one addition per column), so that it does not depend on timing.
#include <cuda_bf16.h>

#include <algorithm>

#include "e4m3.cuh"
#include "norm.cuh"
#include "ptx_sm100.cuh"
#include "umma_common.cuh"

namespace o64 {

namespace {

constexpr int kNormMaxThreads = 512;
// Narrower rows run on the block-per-row kernel.  (A measured choice only above: 65536 x 256 to e4m3 84 us there and 48 on the ring.
// Below, the ring would take less as well, 65536 x 192 48 us and not 85, backward 40 and not 46, but for unaligned rows backward,
// 127 columns 61 us and not 52.)
constexpr int kRingCols = 256;

// Eight consecutive bf16 values of a row; columns >= n read as zero.
template <bool VEC>
__device__ __forceinline__ void load8(const __nv_bfloat16 *row, int col, int n, float (&v)[8]) {
    if constexpr (VEC) {
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (col < n) raw = *reinterpret_cast<const uint4 *>(row + col);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = col + i < n ? __bfloat162float(row[col + i]) : 0.0f;
    }
}

template <bool VEC>
__device__ __forceinline__ void store8(__nv_bfloat16 *row, int col, int n, const float (&v)[8]) {
    if constexpr (VEC) {
        if (col < n) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t *>(&p);
            }
            *reinterpret_cast<uint4 *>(row + col) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (col + i < n) row[col + i] = __float2bfloat16_rn(v[i]);
    }
}

template <bool VEC>
__device__ __forceinline__ void load_w8(const void *w, bool f32, int col, int n, float (&v)[8]) {
    if (f32) {
        const float *p = static_cast<const float *>(w);
        if (VEC && col < n) {
            const float4 a = __ldg(reinterpret_cast<const float4 *>(p + col));
            const float4 b = __ldg(reinterpret_cast<const float4 *>(p + col) + 1);
            v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = col + i < n ? __ldg(p + col + i) : 0.0f;
        }
    } else {
        load8<VEC>(static_cast<const __nv_bfloat16 *>(w), col, n, v);
    }
}

// Sum / maximum over the blockDim.x threads of one row (threadIdx.y counts the rows of the block).
// `slot`: shared floats, one per warp of the block; each reduction of a loop uses other ones in turn.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, float *slot) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float x = __shfl_xor_sync(0xffffffffu, v, o);
        v = MAX ? max_nan(v, x) : v + x;
    }
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    float *mine = slot + threadIdx.y * warps;
    if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = mine[0];
    for (int i = 1; i < warps; ++i) r = MAX ? max_nan(r, mine[i]) : r + mine[i];
    return r;
}

// h = s * rstd * w as s * pre * w * post: where h becomes e4m3, pre is 7/8 of the power of two below rstd and post (in two
// floats) the rest.  A block's quotients h / (max |h| / 448) are those of u = s * pre * w, which has a rounding less than h,
// and with its factor of 7 max |u| / 448 is a division by 64: with a bf16 w both are exact as long as s has 13 bits.
// 16384 x 8192 with the residual: 6 of 134 million values are other than from 64 bits, 866 from h.
// (|u| < |h|, so u is finite where h is.  rstd zero, infinite or NaN: u is as the product with rstd.)
template <bool E4M3>
struct RowFactors {
    float pre, post, post_rest;
    __device__ __forceinline__ explicit RowFactors(float rstd) : pre(rstd), post(1.0f), post_rest(0.0f) {
        if constexpr (E4M3) {
            constexpr float kHi = (float)(8.0 / 7.0), kLo = (float)(8.0 / 7.0 - (double)kHi);
            const uint32_t bits = __float_as_uint(rstd);
            if (rstd == rstd) pre = 0.875f * __uint_as_float(bits & 0x7f800000u);
            const float f = __uint_as_float((bits & 0x007fffffu) | 0x3f800000u);
            post = f * kHi;
            post_rest = fmaf(f, kLo, fmaf(f, kHi, -post));
        }
    }
};

// The scale of a block of h whose largest |u| is `top`, and what turns its u into quotients.
struct NormScale {
    float scale, back, inv;
};
__device__ __forceinline__ NormScale norm_scale(float top, const RowFactors<true> &row) {
    const float d = top / 448.0f;
    NormScale r;
    r.back = remainder_scale(d);
    r.scale = fmaf(d, row.post, r.back * row.post_rest);
    r.inv = 1.0f / d;
    if (r.scale < FLT_MIN) {  // no normal number: 1, and values that are all below half of e4m3's smallest
        r.scale = 1.0f;
        r.back = r.inv = 0.0f;
    }
    return r;
}

// Eight values of a block to e4m3.
__device__ __forceinline__ uint2 quant8(const float (&v)[8], const NormScale &s) {
    uint32_t q[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e >> 1] |= quant2(make_float2(v[2 * e], v[2 * e + 1]), s.back, s.inv) << (16 * (e & 1));
    return make_uint2(q[0], q[1]);
}

struct FwdParams {
    long long T;
    int N;
    const __nv_bfloat16 *X, *R;
    __nv_bfloat16 *S;
    long long ldx, ldr, lds, ldy, ldscales;
    const void *W;
    void *Y;
    float *scales, *rstd;
    float eps;
    double inv_n;  // 1 / N
    int w_f32, row_scale;
};

// 1 / sqrt(mean of squares + eps) of a row's sum of squares, rounded once.
__device__ __forceinline__ float rstd_of(float sum, const FwdParams &p) { return (float)rsqrt(fma((double)sum, p.inv_n, (double)p.eps)); }

// Columns of thread t: (i * blockDim.x + t) * 8 .. + 7 for i < NV, so that 16 neighbouring threads hold
// one scale block of 128.
template <int NV, bool VEC, bool E4M3>
__global__ void __launch_bounds__(kNormMaxThreads) norm_forward_kernel(const FwdParams p) {
    __shared__ float slots[2][16];
    const long long row = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    const bool live = row < p.T;  // every thread takes part in the reductions
    const int n = live ? p.N : 0;
    const __nv_bfloat16 *x = p.X + (live ? row * p.ldx : 0);
    const __nv_bfloat16 *r = p.R ? p.R + (live ? row * p.ldr : 0) : nullptr;
    float v[NV][8];
    float sq = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) load8<VEC>(x, (i * blockDim.x + threadIdx.x) * 8, n, v[i]);
    if (r) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float a[8];
            load8<VEC>(r, (i * blockDim.x + threadIdx.x) * 8, n, a);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] += a[e];
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) sq = fmaf(v[i][e], v[i][e], sq);
    if (p.S) {
#pragma unroll
        for (int i = 0; i < NV; ++i) store8<VEC>(p.S + (live ? row * p.lds : 0), (i * blockDim.x + threadIdx.x) * 8, n, v[i]);
    }
    const float rstd = rstd_of(row_reduce<false>(sq, slots[0]), p);
    if (p.rstd && live && threadIdx.x == 0) p.rstd[row] = rstd;
    const RowFactors<E4M3> factors(rstd);
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        float w[8];
        load_w8<VEC>(p.W, p.w_f32, (i * blockDim.x + threadIdx.x) * 8, p.N, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[i][e] = v[i][e] * factors.pre * w[e];
            // past the row's end there is 0 * pre, which may be NaN: not part of any maximum
            if (E4M3 && p.row_scale && (i * blockDim.x + threadIdx.x) * 8 + e < n) top = max_nan(top, fabsf(v[i][e]));
        }
    }
    if constexpr (!E4M3) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
            store8<VEC>(static_cast<__nv_bfloat16 *>(p.Y) + (live ? row * p.ldy : 0), (i * blockDim.x + threadIdx.x) * 8, n, v[i]);
    } else {
        NormScale scale;
        if (p.row_scale) {
            scale = norm_scale(row_reduce<true>(top, slots[1]), factors);
            if (live && threadIdx.x == 0) p.scales[row * p.ldscales] = scale.scale;
        }
        uint8_t *y = static_cast<uint8_t *>(p.Y) + (live ? row * p.ldy : 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            if (!p.row_scale) {
                float m = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col + e < n) m = max_nan(m, fabsf(v[i][e]));
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                scale = norm_scale(m, factors);
                if (col < n && (threadIdx.x & 15) == 0) p.scales[row * p.ldscales + col / 128] = scale.scale;
            }
            const uint2 q2 = quant8(v[i], scale);
            const uint32_t q[2] = {q2.x, q2.y};
            if constexpr (VEC) {
                if (col < n) *reinterpret_cast<uint2 *>(y + col) = q2;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col + e < n) y[col + e] = (uint8_t)(q[e >> 2] >> (8 * (e & 3)));
            }
        }
    }
}

struct BwdParams {
    long long T;
    int N;
    const __nv_bfloat16 *dY, *S, *dR;
    __nv_bfloat16 *dX;
    long long lddy, lds, lddr, lddx;
    const void *W;
    const float *rstd;
    float *partial;  // [gridDim.x * blockDim.y][N], or NULL
    int w_f32;
};

// Each thread group walks the rows grid-stride and keeps its columns' share of dW in registers.
template <int NV, bool VEC>
__global__ void __launch_bounds__(kNormMaxThreads) norm_backward_kernel(const BwdParams p) {
    __shared__ float slots[2][16];
    float dw[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = 0.0f;
    const long long group = (long long)blockIdx.x * blockDim.y + threadIdx.y;
    const long long groups = (long long)gridDim.x * blockDim.y;
    int turn = 0;
    // all rows of a block's groups go through the same number of rounds (the reductions synchronise the block)
    for (long long row = group; row - threadIdx.y < p.T; row += groups, turn ^= 1) {
        const bool live = row < p.T;
        const int n = live ? p.N : 0;
        const long long at = live ? row : 0;
        const float rstd = p.rstd[at];
        float g[NV][8], nn[NV][8];
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            load8<VEC>(p.dY + at * p.lddy, col, n, g[i]);
            load8<VEC>(p.S + at * p.lds, col, n, nn[i]);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            float w[8];
            load_w8<VEC>(p.W, p.w_f32, col, p.N, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                nn[i][e] = col + e < n ? nn[i][e] * rstd : 0.0f;
                dw[i][e] = fmaf(g[i][e], nn[i][e], dw[i][e]);
                g[i][e] *= w[e];
                dot = fmaf(g[i][e], nn[i][e], dot);
            }
        }
        const float mean = row_reduce<false>(dot, slots[turn]) / (float)p.N;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            float out[8], dr[8];
            if (p.dR) load8<VEC>(p.dR + at * p.lddr, col, n, dr);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                out[e] = rstd * (g[i][e] - nn[i][e] * mean);
                if (p.dR) out[e] += dr[e];
            }
            store8<VEC>(p.dX + at * p.lddx, col, n, out);
        }
    }
    if (p.partial) {
        float *dst = p.partial + group * p.N;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int col = (i * blockDim.x + threadIdx.x) * 8 + e;
                if (col < p.N) dst[col] = dw[i][e];
            }
    }
}

// ---- many rows: a ring of bulk copies -------------------------------------------------------------
constexpr int kNormWait = 0x801;
constexpr int kNormMaxStages = 3;
constexpr int kRingMaxThreads = 1024;  // a row's; 64 registers
constexpr int kRingNv = 2;             // vectors of eight columns a thread, in the ring kernels

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}

// Eight values of a row in shared memory.
__device__ __forceinline__ void smem8(const uint8_t *at, float (&v)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4 *>(at);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

// The sum of the warps' values, for every thread.
__device__ __forceinline__ float block_sum(const float *slot) {
    float v = (threadIdx.x & 31) < (blockDim.x >> 5) ? slot[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// In both kernels a copy that does not arrive within the budget is reported and its rows are undefined; every
// thread still walks to the end (the flag ends the remaining waits at once).
template <bool E4M3>
__global__ void __launch_bounds__(kRingMaxThreads) norm_forward_ring_kernel(const FwdParams p, int stages, int *status, unsigned long long wait_ns) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float slots[2][32];
    __shared__ __align__(8) uint64_t bars[kNormMaxStages];
    __shared__ int abort_word;
    const int n = p.N;
    const uint32_t row_bytes = (uint32_t)n * 2, pitch = (row_bytes + 127) & ~127u;
    const int operands = p.R ? 2 : 1;
    const uint32_t stage_bytes = pitch * operands;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(smem_u32(&bars[s]), 1);
        abort_word = 0;
        fence_mbar_init();
    }
    __syncthreads();
    auto load = [&](long long row, int s) {
        const uint32_t bar = smem_u32(&bars[s]), dst = smem_u32(smem) + s * stage_bytes;
        mbar_arrive_expect_tx(bar, row_bytes * operands);
        bulk_load(dst, p.X + row * p.ldx, row_bytes, bar);
        if (p.R) bulk_load(dst + pitch, p.R + row * p.ldr, row_bytes, bar);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; ++s) {
            const long long row = blockIdx.x + (long long)s * gridDim.x;
            if (row < p.T) load(row, s);
        }
    float w[kRingNv][8];
#pragma unroll
    for (int i = 0; i < kRingNv; ++i) load_w8<true>(p.W, p.w_f32, (i * blockDim.x + threadIdx.x) * 8, n, w[i]);
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    for (long long row = blockIdx.x; row < p.T; row += gridDim.x, turn ^= 1) {
        mbar_wait_bounded(smem_u32(&bars[stage]), phase, &abort_word, status, kNormWait, wait_ns);
        const uint8_t *at = smem + stage * stage_bytes;
        float v[kRingNv][8];
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.0f;
            if (col < n) {
                smem8(at + col * 2, v[i]);
                if (p.R) {
                    float a[8];
                    smem8(at + pitch + col * 2, a);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] += a[e];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) sq = fmaf(v[i][e], v[i][e], sq);
            }
        }
        // the block's sum; behind the barrier in it the stage's values are in registers and it is loaded again
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        if ((threadIdx.x & 31) == 0) slots[turn][threadIdx.x >> 5] = sq;
        __syncthreads();
        if (threadIdx.x == 0 && row + (long long)stages * gridDim.x < p.T) {
            fence_proxy_async_smem();
            load(row + (long long)stages * gridDim.x, stage);
        }
        const float sum = block_sum(slots[turn]);
        const float rstd = rstd_of(sum, p);
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
        const RowFactors<E4M3> factors(rstd);
        if (p.S) {
#pragma unroll
            for (int i = 0; i < kRingNv; ++i) store8<true>(p.S + row * p.lds, (i * blockDim.x + threadIdx.x) * 8, n, v[i]);
        }
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * factors.pre * w[i][e];
            if constexpr (!E4M3) {
                store8<true>(static_cast<__nv_bfloat16 *>(p.Y) + row * p.ldy, col, n, v[i]);
            } else {
                float m = 0.0f;
                if (col < n) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) m = max_nan(m, fabsf(v[i][e]));
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                const NormScale scale = norm_scale(m, factors);
                if (col < n) {
                    if ((threadIdx.x & 15) == 0) p.scales[row * p.ldscales + col / 128] = scale.scale;
                    *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p.Y) + row * p.ldy + col) = quant8(v[i], scale);
                }
            }
        }
        if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    if (abort_word) {  // copies may still be in flight
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
}

// Rows that start anywhere (odd N, odd pitches): the same ring of the 16-byte chunks that hold any of a row's bytes
// (an aligned chunk with one byte of an allocation lies inside it), read from shared memory at the row's own offset;
// results go back through shared memory too, so that a warp's stores are contiguous.  Two bytes at a time straight from
// and to global memory, 10000 rows of 5003 with the residual took 248 us to e4m3 and 286 us backward;
// 120 us and 164 us this way.
struct OddRow {
    const __nv_bfloat16 *row;
    __device__ __forceinline__ uint32_t shift() const { return (uint32_t)(reinterpret_cast<uintptr_t>(row) & 15u); }
    __device__ __forceinline__ uint32_t bytes(int n) const { return (shift() + (uint32_t)n * 2 + 15u) & ~15u; }
    __device__ __forceinline__ const void *chunks() const { return reinterpret_cast<const uint8_t *>(row) - shift(); }
};
__host__ __device__ constexpr uint32_t odd_pitch(int64_t n) { return (uint32_t)((n * 2 + 16 + 127) / 128 * 128); }

// n two-byte (or one-byte) values from shared memory to a row that starts anywhere, by the whole block.
template <typename T>
__device__ __forceinline__ void copy_out(T *dst, const T *src, int n) {
    constexpr int kWord = 4 / sizeof(T);
    const int head = min((int)((4u - (reinterpret_cast<uintptr_t>(dst) & 3u)) & 3u) / (int)sizeof(T), n);
    const int words = (n - head) / kWord;
    for (int k = threadIdx.x; k < words; k += blockDim.x) {
        uint32_t w = 0;
#pragma unroll
        for (int e = 0; e < kWord; ++e) w |= (uint32_t)src[head + k * kWord + e] << (8 * sizeof(T) * e);
        *reinterpret_cast<uint32_t *>(dst + head + k * kWord) = w;
    }
    const int rest = head + words * kWord;
    if ((int)threadIdx.x < head) dst[threadIdx.x] = src[threadIdx.x];
    if ((int)threadIdx.x < n - rest) dst[rest + threadIdx.x] = src[rest + threadIdx.x];
}

template <bool E4M3>
__global__ void __launch_bounds__(kRingMaxThreads) norm_forward_odd_kernel(const FwdParams p, int stages, int *status, unsigned long long wait_ns) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float slots[2][32];
    __shared__ __align__(8) uint64_t bars[kNormMaxStages];
    __shared__ int abort_word;
    const int n = p.N;
    const uint32_t pitch = odd_pitch(n);
    const uint32_t stage_bytes = pitch * (p.R ? 2 : 1);
    uint8_t *s_out = smem + stages * stage_bytes, *y_out = s_out + pitch;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(smem_u32(&bars[s]), 1);
        abort_word = 0;
        fence_mbar_init();
    }
    __syncthreads();
    auto load = [&](long long row, int s) {
        const uint32_t bar = smem_u32(&bars[s]), dst = smem_u32(smem) + s * stage_bytes;
        const OddRow x{p.X + row * p.ldx}, r{p.R ? p.R + row * p.ldr : nullptr};
        mbar_arrive_expect_tx(bar, x.bytes(n) + (p.R ? r.bytes(n) : 0));
        bulk_load(dst, x.chunks(), x.bytes(n), bar);
        if (p.R) bulk_load(dst + pitch, r.chunks(), r.bytes(n), bar);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; ++s) {
            const long long row = blockIdx.x + (long long)s * gridDim.x;
            if (row < p.T) load(row, s);
        }
    float w[kRingNv][8];
#pragma unroll
    for (int i = 0; i < kRingNv; ++i) load_w8<false>(p.W, p.w_f32, (i * blockDim.x + threadIdx.x) * 8, n, w[i]);
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    for (long long row = blockIdx.x; row < p.T; row += gridDim.x, turn ^= 1) {
        mbar_wait_bounded(smem_u32(&bars[stage]), phase, &abort_word, status, kNormWait, wait_ns);
        const uint8_t *at = smem + stage * stage_bytes;
        const __nv_bfloat16 *x = reinterpret_cast<const __nv_bfloat16 *>(at + OddRow{p.X + row * p.ldx}.shift());
        const __nv_bfloat16 *r = p.R ? reinterpret_cast<const __nv_bfloat16 *>(at + pitch + OddRow{p.R + row * p.ldr}.shift()) : nullptr;
        float v[kRingNv][8];
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[i][e] = 0.0f;
                if (col + e < n) {
                    v[i][e] = __bfloat162float(x[col + e]);
                    if (r) v[i][e] += __bfloat162float(r[col + e]);
                    sq = fmaf(v[i][e], v[i][e], sq);
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
        if ((threadIdx.x & 31) == 0) slots[turn][threadIdx.x >> 5] = sq;
        __syncthreads();  // the stage is in registers, the last row's results have left
        if (threadIdx.x == 0 && row + (long long)stages * gridDim.x < p.T) {
            fence_proxy_async_smem();
            load(row + (long long)stages * gridDim.x, stage);
        }
        const float rstd = rstd_of(block_sum(slots[turn]), p);
        if (p.rstd && threadIdx.x == 0) p.rstd[row] = rstd;
        const RowFactors<E4M3> factors(rstd);
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            // (whole vectors: the buffers have room behind the row)
            if (p.S && col < n) store8<true>(reinterpret_cast<__nv_bfloat16 *>(s_out), col, n, v[i]);
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[i][e] = v[i][e] * factors.pre * w[i][e];
                if (E4M3 && col + e < n) m = max_nan(m, fabsf(v[i][e]));
            }
            if constexpr (!E4M3) {
                if (col < n) store8<true>(reinterpret_cast<__nv_bfloat16 *>(y_out), col, n, v[i]);
            } else {
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
                const NormScale scale = norm_scale(m, factors);
                if (col < n) {
                    if ((threadIdx.x & 15) == 0) p.scales[row * p.ldscales + col / 128] = scale.scale;
                    *reinterpret_cast<uint2 *>(y_out + col) = quant8(v[i], scale);
                }
            }
        }
        __syncthreads();
        if (p.S) copy_out(reinterpret_cast<uint16_t *>(p.S + row * p.lds), reinterpret_cast<const uint16_t *>(s_out), n);
        if constexpr (E4M3)
            copy_out(static_cast<uint8_t *>(p.Y) + row * p.ldy, y_out, n);
        else
            copy_out(static_cast<uint16_t *>(p.Y) + row * p.ldy, reinterpret_cast<const uint16_t *>(y_out), n);
        if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    if (abort_word) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
}

__global__ void __launch_bounds__(kRingMaxThreads) norm_backward_odd_kernel(const BwdParams p, int stages, int *status, unsigned long long wait_ns) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float slots[2][32];
    __shared__ __align__(8) uint64_t bars[kNormMaxStages];
    __shared__ int abort_word;
    const int n = p.N;
    const uint32_t pitch = odd_pitch(n);
    const uint32_t stage_bytes = pitch * (p.dR ? 3 : 2);
    uint8_t *dx_out = smem + stages * stage_bytes;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(smem_u32(&bars[s]), 1);
        abort_word = 0;
        fence_mbar_init();
    }
    __syncthreads();
    auto load = [&](long long row, int s) {
        const uint32_t bar = smem_u32(&bars[s]), dst = smem_u32(smem) + s * stage_bytes;
        const OddRow y{p.dY + row * p.lddy}, z{p.S + row * p.lds}, r{p.dR ? p.dR + row * p.lddr : nullptr};
        mbar_arrive_expect_tx(bar, y.bytes(n) + z.bytes(n) + (p.dR ? r.bytes(n) : 0));
        bulk_load(dst, y.chunks(), y.bytes(n), bar);
        bulk_load(dst + pitch, z.chunks(), z.bytes(n), bar);
        if (p.dR) bulk_load(dst + 2 * pitch, r.chunks(), r.bytes(n), bar);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; ++s) {
            const long long row = blockIdx.x + (long long)s * gridDim.x;
            if (row < p.T) load(row, s);
        }
    float dw[kRingNv][8], w[kRingNv][8];
#pragma unroll
    for (int i = 0; i < kRingNv; ++i) {
        load_w8<false>(p.W, p.w_f32, (i * blockDim.x + threadIdx.x) * 8, n, w[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) dw[i][e] = 0.0f;
    }
    int stage = 0, turn = 0;
    uint32_t phase = 0;
    for (long long row = blockIdx.x; row < p.T; row += gridDim.x, turn ^= 1) {
        const float rstd = p.rstd[row];
        mbar_wait_bounded(smem_u32(&bars[stage]), phase, &abort_word, status, kNormWait, wait_ns);
        const uint8_t *at = smem + stage * stage_bytes;
        const __nv_bfloat16 *dy = reinterpret_cast<const __nv_bfloat16 *>(at + OddRow{p.dY + row * p.lddy}.shift());
        const __nv_bfloat16 *z = reinterpret_cast<const __nv_bfloat16 *>(at + pitch + OddRow{p.S + row * p.lds}.shift());
        const __nv_bfloat16 *dr = p.dR ? reinterpret_cast<const __nv_bfloat16 *>(at + 2 * pitch + OddRow{p.dR + row * p.lddr}.shift()) : nullptr;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col + e < n) {
                    const float g = __bfloat162float(dy[col + e]), x = __bfloat162float(z[col + e]) * rstd;
                    dw[i][e] = fmaf(g, x, dw[i][e]);
                    dot = fmaf(g * w[i][e], x, dot);
                }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if ((threadIdx.x & 31) == 0) slots[turn][threadIdx.x >> 5] = dot;
        __syncthreads();  // (the last row's results have left, too)
        const float mean = block_sum(slots[turn]) / (float)n;
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            float out[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                out[e] = 0.0f;
                if (col + e < n) {
                    out[e] = rstd * (__bfloat162float(dy[col + e]) * w[i][e] - __bfloat162float(z[col + e]) * rstd * mean);
                    if (dr) out[e] += __bfloat162float(dr[col + e]);
                }
            }
            if (col < n) store8<true>(reinterpret_cast<__nv_bfloat16 *>(dx_out), col, n, out);
        }
        __syncthreads();
        if (threadIdx.x == 0 && row + (long long)stages * gridDim.x < p.T) {
            fence_proxy_async_smem();
            load(row + (long long)stages * gridDim.x, stage);
        }
        copy_out(reinterpret_cast<uint16_t *>(p.dX + row * p.lddx), reinterpret_cast<const uint16_t *>(dx_out), n);
        if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    griddep_launch_dependents();
    if (p.partial) {
        float *dst = p.partial + (long long)blockIdx.x * n;
#pragma unroll
        for (int i = 0; i < kRingNv; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int col = (i * blockDim.x + threadIdx.x) * 8 + e;
                if (col < n) dst[col] = dw[i][e];
            }
    }
    if (abort_word) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
}

__global__ void __launch_bounds__(kRingMaxThreads) norm_backward_ring_kernel(const BwdParams p, int stages, int w_in_smem, int *status, unsigned long long wait_ns) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float slots[2][32];
    __shared__ __align__(8) uint64_t bars[kNormMaxStages];
    __shared__ int abort_word;
    const int n = p.N;
    const uint32_t row_bytes = (uint32_t)n * 2, pitch = (row_bytes + 127) & ~127u;
    const int operands = p.dR ? 3 : 2;
    const uint32_t stage_bytes = pitch * operands;
    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) mbar_init(smem_u32(&bars[s]), 1);
        abort_word = 0;
        fence_mbar_init();
    }
    __syncthreads();
    auto load = [&](long long row, int s) {
        const uint32_t bar = smem_u32(&bars[s]), dst = smem_u32(smem) + s * stage_bytes;
        mbar_arrive_expect_tx(bar, row_bytes * operands);
        bulk_load(dst, p.dY + row * p.lddy, row_bytes, bar);
        bulk_load(dst + pitch, p.S + row * p.lds, row_bytes, bar);
        if (p.dR) bulk_load(dst + 2 * pitch, p.dR + row * p.lddr, row_bytes, bar);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; ++s) {
            const long long row = blockIdx.x + (long long)s * gridDim.x;
            if (row < p.T) load(row, s);
        }
    float dw[kRingNv][8];
#pragma unroll
    for (int i = 0; i < kRingNv; ++i) {
        const int col = (i * blockDim.x + threadIdx.x) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dw[i][e] = 0.0f;
        }
    }
    // a thread's columns of w lie behind the ring as they came (wide rows leave no room for them); nobody else reads them
    uint8_t *w_smem = smem + stages * stage_bytes;
    const int w_elem = p.w_f32 ? 4 : 2;
    if (w_in_smem) {
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            if (col < n) {
                const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint8_t *>(p.W) + (size_t)col * w_elem);
                uint4 *dst = reinterpret_cast<uint4 *>(w_smem + (size_t)col * w_elem);
                dst[0] = __ldg(src);
                if (p.w_f32) dst[1] = __ldg(src + 1);
            }
        }
    }
    auto weight8 = [&](int col, float (&w)[8]) __attribute__((always_inline)) {
        if (!w_in_smem) {
            load_w8<true>(p.W, p.w_f32, col, n, w);
        } else if (p.w_f32) {
            *reinterpret_cast<float4 *>(w) = *reinterpret_cast<const float4 *>(w_smem + col * 4);
            *reinterpret_cast<float4 *>(w + 4) = *reinterpret_cast<const float4 *>(w_smem + col * 4 + 16);
        } else {
            smem8(w_smem + col * 2, w);
        }
    };
    int stage = 0, turn = 0, before = 0;
    uint32_t phase = 0;
    for (long long row = blockIdx.x; row < p.T; row += gridDim.x, turn ^= 1) {
        const float rstd = p.rstd[row];
        mbar_wait_bounded(smem_u32(&bars[stage]), phase, &abort_word, status, kNormWait, wait_ns);
        const uint8_t *at = smem + stage * stage_bytes;
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            if (col < n) {
                float g[8], nn[8], w[8];
                smem8(at + col * 2, g);
                smem8(at + pitch + col * 2, nn);
                weight8(col, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = nn[e] * rstd;
                    dw[i][e] = fmaf(g[e], x, dw[i][e]);
                    dot = fmaf(g[e] * w[e], x, dot);
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if ((threadIdx.x & 31) == 0) slots[turn][threadIdx.x >> 5] = dot;
        __syncthreads();
        // everyone is past the row before: its stage is free
        if (threadIdx.x == 0 && row != blockIdx.x && row + (long long)(stages - 1) * gridDim.x < p.T) {
            fence_proxy_async_smem();
            load(row + (long long)(stages - 1) * gridDim.x, before);
        }
        const float mean = block_sum(slots[turn]) / (float)n;
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            if (col < n) {
                float g[8], nn[8], w[8], out[8], dr[8];
                smem8(at + col * 2, g);
                smem8(at + pitch + col * 2, nn);
                if (p.dR) smem8(at + 2 * pitch + col * 2, dr);
                weight8(col, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    out[e] = rstd * (g[e] * w[e] - nn[e] * rstd * mean);
                    if (p.dR) out[e] += dr[e];
                }
                store8<true>(p.dX + row * p.lddx, col, n, out);
            }
        }
        before = stage;
        if (++stage == stages) {
            stage = 0;
            phase ^= 1u;
        }
    }
    griddep_launch_dependents();
    if (p.partial) {
        float *dst = p.partial + (long long)blockIdx.x * n;
#pragma unroll
        for (int i = 0; i < kRingNv; ++i) {
            const int col = (i * blockDim.x + threadIdx.x) * 8;
            if (col < n) {
                *reinterpret_cast<float4 *>(dst + col) = make_float4(dw[i][0], dw[i][1], dw[i][2], dw[i][3]);
                *reinterpret_cast<float4 *>(dst + col + 4) = make_float4(dw[i][4], dw[i][5], dw[i][6], dw[i][7]);
            }
        }
    }
    if (abort_word) {
        const uint64_t t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
}

// dW[j] = sum over the partial rows: eight columns (one sector of each row) per block, THREADS / 8 down the rows.
// Launched so that its set-up overlaps the kernel that writes them.
template <int THREADS>
__global__ void __launch_bounds__(THREADS) norm_dw_kernel(const float *partial, int rows, int N, float *dW) {
    __shared__ float part[THREADS / 32][8];
    const int c = threadIdx.x & 7, col = blockIdx.x * 8 + c;
    griddep_wait();
    float s = 0.0f;
    if (col < N) {
#pragma unroll 8
        for (int r = threadIdx.x >> 3; r < rows; r += THREADS / 8) s += partial[(long long)r * N + col];
    }
    s += __shfl_xor_sync(0xffffffffu, s, 8);
    s += __shfl_xor_sync(0xffffffffu, s, 16);
    if ((threadIdx.x & 31) < 8) part[threadIdx.x >> 5][c] = s;
    __syncthreads();
    if (threadIdx.x < 256) {  // warp w adds column w
        const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
        s = lane < THREADS / 32 ? part[lane][w] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0 && blockIdx.x * 8 + w < N) dW[blockIdx.x * 8 + w] = s;
    }
}

bool vec8(const void *p, int64_t ld) { return !p || ((reinterpret_cast<uintptr_t>(p) & 15u) == 0 && ld % 8 == 0); }

// Threads per row (a multiple of 32) for NV vectors of eight columns a thread.
int threads_for(int64_t N, int nv) { return (int)((((N + 7) / 8 + nv - 1) / nv + 31) / 32 * 32); }

// The largest number of columns a thread may have decides between few and many threads per row: few rows
// want the row spread thin (latency), many rows want loads in flight per thread.
int pick_nv(int64_t N, int smallest) {
    int nv = smallest;
    while (threads_for(N, nv) > kNormMaxThreads) nv *= 2;
    return nv;
}

template <int NV, bool VEC>
int launch_forward(const FwdParams &p, bool e4m3, dim3 grid, dim3 block, cudaStream_t s) {
    if (e4m3)
        norm_forward_kernel<NV, VEC, true><<<grid, block, 0, s>>>(p);
    else
        norm_forward_kernel<NV, VEC, false><<<grid, block, 0, s>>>(p);
    return cudaGetLastError() == cudaSuccess ? O64_OK : O64_ERR_CUDA;
}

// Blocks that stay on an SM for rows of N columns with `operands` of them on their way, and the depth of their
// rings: 1024 threads and all shared memory of an SM, at most three rows ahead.  Two vectors a thread: with four, 8191
// rows of 5000 ran backward in 75 us instead of 70 and 6247 rows of 9984 to e4m3 in 92 us instead of 71.
struct RingShape {
    int threads, blocks_per_sm, stages;
    size_t smem;
};
// The rings are for two rows a resident block and more: 592 rows of 1024 to e4m3 4.3 us on a block per row, 3.7 on the ring, 296
// rows 2.8 and 3.5; 1184 x 4096 9.6 and 7.5, 296 x 4096 3.7 and 4.2.  (Backward the ring is ahead from one row a block on: 592 x 4096
// 15.4 and 10.7, 1184 x 4096 19.2 and 12.9.)
bool ring_shape(int64_t N, int operands, int extra_bytes_per_col, RingShape *r, bool odd = false) {
    r->threads = threads_for(N, kRingNv);
    if (r->threads > kRingMaxThreads) return false;
    const size_t row = odd ? (size_t)odd_pitch(N) * operands : (size_t)((N * 2 + 127) / 128 * 128) * operands;
    const size_t extra = odd ? (size_t)odd_pitch(N) * 2 : (size_t)N * extra_bytes_per_col;  // odd: two rows of results
    const int most = std::min(16, 1024 / r->threads);
    for (int b = most; b >= 1; --b)
        for (int s = 3; s >= 2; --s)
            if ((row * s + extra + 1536) * b <= 227 * 1024 && row * s + extra <= 220 * 1024) {
                r->blocks_per_sm = b, r->stages = s, r->smem = row * s + extra;
                return true;
            }
    return false;
}

template <typename F>
int allow_smem(F kern, KernelSetup &ks) {
    return ks.once([&](int *) { return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024) == cudaSuccess ? (int)O64_OK : (int)O64_ERR_CUDA; },
                   nullptr);
}

template <bool E4M3>
int launch_forward_ring(const FwdParams &p, const RingShape &r, const NormCall &c, int num_sms) {
    static KernelSetup ks;
    auto kern = norm_forward_ring_kernel<E4M3>;
    const int rc = allow_smem(kern, ks);
    if (rc) return rc;
    kern<<<r.blocks_per_sm * num_sms, r.threads, r.smem, c.stream>>>(p, r.stages, c.status, c.wait_ns);
    return cudaGetLastError() == cudaSuccess ? O64_OK : O64_ERR_CUDA;
}

template <bool E4M3>
int launch_forward_odd(const FwdParams &p, const RingShape &r, const NormCall &c, int num_sms) {
    static KernelSetup ks;
    auto kern = norm_forward_odd_kernel<E4M3>;
    const int rc = allow_smem(kern, ks);
    if (rc) return rc;
    kern<<<r.blocks_per_sm * num_sms, r.threads, r.smem, c.stream>>>(p, r.stages, c.status, c.wait_ns);
    return cudaGetLastError() == cudaSuccess ? O64_OK : O64_ERR_CUDA;
}

int launch_backward_odd(const BwdParams &p, const RingShape &r, const NormBackwardCall &c, int grid) {
    static KernelSetup ks;
    auto kern = norm_backward_odd_kernel;
    const int rc = allow_smem(kern, ks);
    if (rc) return rc;
    kern<<<grid, r.threads, r.smem, c.stream>>>(p, r.stages, c.status, c.wait_ns);
    return cudaGetLastError() == cudaSuccess ? O64_OK : O64_ERR_CUDA;
}

int launch_backward_ring(const BwdParams &p, const RingShape &r, const NormBackwardCall &c, int grid, int w_in_smem) {
    static KernelSetup ks;
    auto kern = norm_backward_ring_kernel;
    const int rc = allow_smem(kern, ks);
    if (rc) return rc;
    kern<<<grid, r.threads, r.smem, c.stream>>>(p, r.stages, w_in_smem, c.status, c.wait_ns);
    return cudaGetLastError() == cudaSuccess ? O64_OK : O64_ERR_CUDA;
}

}  // namespace

int norm_forward(const NormCall &c, int num_sms) {
    const bool e4m3 = c.out_kind == O64_OUT_E4M3;
    const bool y_ok = e4m3 ? (reinterpret_cast<uintptr_t>(c.Y) & 7u) == 0 && c.ldy % 8 == 0 : vec8(c.Y, c.ldy);
    const bool vec = c.N % 8 == 0 && vec8(c.X, c.ldx) && vec8(c.R, c.ldr) && vec8(c.S, c.lds) && y_ok && vec8(c.W, 8);
    FwdParams p;
    p.T = c.T, p.N = (int)c.N;
    p.X = static_cast<const __nv_bfloat16 *>(c.X), p.ldx = c.ldx;
    p.R = static_cast<const __nv_bfloat16 *>(c.R), p.ldr = c.ldr;
    p.S = static_cast<__nv_bfloat16 *>(c.S), p.lds = c.lds;
    p.W = c.W, p.w_f32 = c.w_f32, p.eps = c.eps, p.inv_n = 1.0 / (double)c.N;
    p.Y = c.Y, p.ldy = c.ldy, p.scales = c.scales, p.ldscales = c.ldscales, p.rstd = c.rstd, p.row_scale = c.row_scale;
    RingShape r;
    if (vec && !(e4m3 && c.row_scale) && c.N >= kRingCols && ring_shape(c.N, c.R ? 2 : 1, 0, &r) && c.T >= (int64_t)2 * r.blocks_per_sm * num_sms) {
        return e4m3 ? launch_forward_ring<true>(p, r, c, num_sms) : launch_forward_ring<false>(p, r, c, num_sms);
    }
    if (!vec && !(e4m3 && c.row_scale) && c.N >= kRingCols && ring_shape(c.N, c.R ? 2 : 1, 0, &r, true) && c.T >= (int64_t)2 * r.blocks_per_sm * num_sms)
        return e4m3 ? launch_forward_odd<true>(p, r, c, num_sms) : launch_forward_odd<false>(p, r, c, num_sms);
    const int nv = pick_nv(c.N, c.T <= 2 * num_sms ? 1 : 4);
    const int tpr = threads_for(c.N, nv);
    const int rows = tpr >= 128 ? 1 : 128 / tpr;
    const dim3 block(tpr, rows), grid((unsigned)((c.T + rows - 1) / rows));
    switch (nv) {
    case 1: return vec ? launch_forward<1, true>(p, e4m3, grid, block, c.stream) : launch_forward<1, false>(p, e4m3, grid, block, c.stream);
    case 2: return vec ? launch_forward<2, true>(p, e4m3, grid, block, c.stream) : launch_forward<2, false>(p, e4m3, grid, block, c.stream);
    case 4: return vec ? launch_forward<4, true>(p, e4m3, grid, block, c.stream) : launch_forward<4, false>(p, e4m3, grid, block, c.stream);
    default: return vec ? launch_forward<8, true>(p, e4m3, grid, block, c.stream) : launch_forward<8, false>(p, e4m3, grid, block, c.stream);
    }
}

static void backward_shape(int64_t T, int64_t N, int *nv, dim3 *block, int64_t *blocks) {
    *nv = pick_nv(N, 2);
    const int tpr = threads_for(N, *nv);
    const int rows = tpr >= 128 ? 1 : 128 / tpr;
    *block = dim3(tpr, rows);
    const int64_t want = (T + rows - 1) / rows;
    // three blocks per SM, and more of narrow rows: the partial rows then stay under 10 MB
    const int64_t most = std::min<int64_t>(2368, std::max<int64_t>(444, (int64_t)2400000 / N / rows / 148 * 148));
    *blocks = want < most ? want : most;
}

int64_t norm_backward_partials(int64_t T, int64_t N) {
    int nv;
    dim3 block;
    int64_t blocks;
    backward_shape(T, N, &nv, &block, &blocks);
    return blocks * block.y;
}

static int add_partials(const NormBackwardCall &c, int64_t rows) {
    cudaLaunchConfig_t cfg = {};
    const bool many = rows > 800;
    cfg.gridDim = dim3((unsigned)((c.N + 7) / 8));
    cfg.blockDim = dim3(many ? 1024 : 256);
    cfg.stream = c.stream;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    const float *partial = c.workspace;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, many ? norm_dw_kernel<1024> : norm_dw_kernel<256>, partial, (int)rows, (int)c.N, c.dW);
    if (e != cudaSuccess) (void)cudaGetLastError();
    return e == cudaSuccess ? O64_OK : O64_ERR_CUDA;
}

int norm_backward(const NormBackwardCall &c, int num_sms) {
    int nv;
    dim3 block;
    int64_t blocks;
    backward_shape(c.T, c.N, &nv, &block, &blocks);
    const bool vec = c.N % 8 == 0 && vec8(c.dY, c.lddy) && vec8(c.S, c.lds) && vec8(c.dR, c.lddr) && vec8(c.dX, c.lddx) && vec8(c.W, 8);
    BwdParams p;
    p.T = c.T, p.N = (int)c.N;
    p.dY = static_cast<const __nv_bfloat16 *>(c.dY), p.lddy = c.lddy;
    p.S = static_cast<const __nv_bfloat16 *>(c.S), p.lds = c.lds;
    p.dR = static_cast<const __nv_bfloat16 *>(c.dR), p.lddr = c.lddr;
    p.dX = static_cast<__nv_bfloat16 *>(c.dX), p.lddx = c.lddx;
    p.W = c.W, p.w_f32 = c.w_f32, p.rstd = c.rstd;
    p.partial = c.dW ? c.workspace : nullptr;
    RingShape r;
    // w stays in shared memory (4096 columns: 53 us with it and three blocks an SM, 59 without and four) unless only
    // one block fits then (8192 rows of 8192, fp32 w: 119 us with it, 99 from L2 and two blocks)
    RingShape with_w;
    bool fits = vec && c.N >= kRingCols && (reinterpret_cast<uintptr_t>(c.workspace) & 15u) == 0 && ring_shape(c.N, c.dR ? 3 : 2, 0, &r);
    const int w_in_smem = fits && ring_shape(c.N, c.dR ? 3 : 2, c.w_f32 ? 4 : 2, &with_w) && (with_w.blocks_per_sm > 1 || r.blocks_per_sm == 1);
    if (w_in_smem) r = with_w;
    if (fits && c.T >= (int64_t)2 * r.blocks_per_sm * num_sms) {
        const int grid = (int)std::min<int64_t>((int64_t)r.blocks_per_sm * num_sms, blocks * block.y);  // no more partial rows than the workspace has
        const int rc = launch_backward_ring(p, r, c, grid, w_in_smem);
        if (rc) return rc;
        return c.dW ? add_partials(c, grid) : O64_OK;
    }
    if (!vec && c.N >= kRingCols && ring_shape(c.N, c.dR ? 3 : 2, 0, &r, true) && c.T >= (int64_t)2 * r.blocks_per_sm * num_sms) {
        const int odd_grid = (int)std::min<int64_t>((int64_t)r.blocks_per_sm * num_sms, blocks * block.y);
        const int rc = launch_backward_odd(p, r, c, odd_grid);
        if (rc) return rc;
        return c.dW ? add_partials(c, odd_grid) : O64_OK;
    }
    const unsigned grid = (unsigned)blocks;
    switch (nv) {
    case 2: vec ? norm_backward_kernel<2, true><<<grid, block, 0, c.stream>>>(p) : norm_backward_kernel<2, false><<<grid, block, 0, c.stream>>>(p); break;
    case 4: vec ? norm_backward_kernel<4, true><<<grid, block, 0, c.stream>>>(p) : norm_backward_kernel<4, false><<<grid, block, 0, c.stream>>>(p); break;
    default: vec ? norm_backward_kernel<8, true><<<grid, block, 0, c.stream>>>(p) : norm_backward_kernel<8, false><<<grid, block, 0, c.stream>>>(p); break;
    }
    if (cudaGetLastError() != cudaSuccess) return O64_ERR_CUDA;
    return c.dW ? add_partials(c, blocks * block.y) : O64_OK;
}

}  // namespace o64
