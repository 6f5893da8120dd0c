// Products grouped by expert, and the e4m3 product with a scale for each block of 128: host-side
// interface and the pieces the kernels share (umma_grouped.cu: CTA pairs on 256 x 256 tiles;
// umma_grouped_rows.cu: few rows an expert).
#pragma once
#include <cuda.h>

#include "e4m3.cuh"
#include "umma_common.cuh"

namespace o64 {

// What is left in the accumulators becomes ...
enum : int {
    GEPI_BF16 = 0,         // bf16
    GEPI_F32 = 1,          // fp32 as it is
    GEPI_SWIGLU_BF16 = 2,  // silu(gate) * up, bf16
    GEPI_SWIGLU_E4M3 = 3   // silu(gate) * up, e4m3 with a scale for each 128 columns of a row
};
__host__ __device__ constexpr bool gepi_swiglu(int e) { return e >= GEPI_SWIGLU_BF16; }
__host__ __device__ constexpr int gepi_bytes(int e) { return e == GEPI_F32 ? 4 : (e == GEPI_SWIGLU_E4M3 ? 1 : 2); }

// Status-word codes.  0x6..: the group offsets in device memory are not ascending within 0 .. T.
constexpr int kBadOffsets = 0x601;
constexpr int kWaitGroupProducer = 0x701, kWaitGroupFull = 0x702, kWaitGroupAccEmpty = 0x703, kWaitGroupAccFull = 0x704,
              kWaitGroupTail = 0x705, kWaitGroupHalf = 0x706, kWaitGroupScales = 0x707;

// One call.  Rows T of A are sorted by group; offsets (device, G + 1 ints) bound the groups; NULL: one
// group of T rows.  B is [G][N][K] (or [G][K][N]: b_kn), C is [T][N].  wgrad: A is dC [T][N], B is the
// forward's A [T][K], C is [G][N][K] and the sum runs over a group's rows.  swiglu: N counts the result's
// columns, B has 2 N rows.  Leading dimensions in elements.
struct GroupedCall {
    int kind = O64_KIND_BF16;  // O64_KIND_BF16, or O64_KIND_FP8 with block scales
    bool b_kn = false, wgrad = false;
    int epi = GEPI_BF16;
    int64_t G = 1, T = 0, N = 0, K = 0;
    const void *A = nullptr, *B = nullptr;
    void *C = nullptr;
    int64_t lda = 0, ldb = 0, stride_b = 0, ldc = 0, stride_c = 0;
    const float *scale_a = nullptr, *scale_b = nullptr;  // [T][K/128]; [G][B rows/128][B columns/128]
    int64_t ldsa = 0, ldsb = 0, stride_sb = 0;
    float *scale_c = nullptr;
    int64_t ldsc = 0;
    const int *offsets = nullptr;
    int *status_word = nullptr;
    int num_sms = 148;
    unsigned long long wait_ns = 0;
    cudaStream_t stream = nullptr;
};

struct GroupedParams {
    int G, T, N, K;  // N: columns of C
    int rows_m;      // wgrad: rows of one C
    int num_m_tiles, num_n_tiles;
    int num_k_blocks;
    void *C;
    long long ldc, stride_c;
    const float *scale_a, *scale_b;
    long long ldsa, ldsb, stride_sb;
    float *scale_c;
    long long ldsc;
    const int *offsets;
    int vec_ok, tma_store;
    int a_groups, b_groups;  // wgrad: the operands' columns are mapped in groups of 64
    int split;   // few rows: CTAs that share a tile's K blocks
    int sa_vec;  // the rows of scale_a are 16-byte aligned
    int *status;
    unsigned long long wait_ns;
};

// A group's rows, kept inside [top, T) whatever the offsets say; *bad: they are not ascending within 0 .. T.  A walk
// over the groups passes the end of those before: offsets that overlap then make no more tiles than others, which is
// what the grids and the one tile of a cluster that divides K are sized for.  WRITTEN: the kernel may exist while the one
// before it still writes the offsets (see umma_grouped_rows.cu); else they come by the read-only path, which the compiler
// moves freely.
template <bool WRITTEN>
__device__ __forceinline__ void group_rows(const GroupedParams &p, int g, int top, int &begin, int &end, bool *bad = nullptr) {
    if (!p.offsets) {
        begin = 0;
        end = p.T;
        return;
    }
    const int a = WRITTEN ? p.offsets[g] : __ldg(p.offsets + g), b = WRITTEN ? p.offsets[g + 1] : __ldg(p.offsets + g + 1);
    begin = min(max(a, top), p.T);
    end = min(max(b, begin), p.T);
    if (bad) *bad = a < 0 || b < a || b > p.T;
}

int grouped_launch(const GroupedCall &c);
// Few rows a group: the kernel that reads every weight once for them.
// grouped_rows_tile: the rows of A of its tiles (16 ... 128), or 0 where CTA pairs are the faster choice.
int grouped_rows_tile(const GroupedCall &c);
int grouped_rows_launch(const GroupedCall &c, const GroupedParams &p, int tok);
// Sets the rows of the groups (wgrad: every C) to the empty sum: K == 0, or a weight gradient over no rows.
int grouped_zero_launch(const GroupedCall &c);

int encode_3d(CUtensorMap *tm, int elem, const void *base, int64_t cols, int64_t rows, int64_t depth, int64_t ld, int64_t stride,
              int box_cols, int box_rows, bool promote, int box_depth = 1);

__device__ __forceinline__ void tma_load_3d_pair(uint32_t smem_dst, const void *tmap, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const void *tmap, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_store_3d(const void *tmap, uint32_t smem_src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(tmap), "r"(smem_src),
                 "r"(x), "r"(y), "r"(z)
                 : "memory");
}

__device__ __forceinline__ float ex2_approx(float x) {  // 2 ulp; below 2^-126 zero
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {  // 1 ulp; below 2^-126 zero
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// silu(g) * u = g / (1 + exp(-g)) * u, within 2^-20 of the value.  With x = -g (between -104 and 104) and x log2(e) = hi + lo in two
// floats, exp(x) = 2^hi (1 + lo ln 2): in one float, its rounding alone is 2^-20 of the result at g = -20 and four times that at
// -80.  The correction goes to the quotient r = 1 / (1 + 2^hi), where it is -r (1 - r) lo ln 2 and 2^hi may be infinite: r is
// zero then and the result, below 1e-35 of u, too.  The power is within 2^-22, the reciprocal 2^-23, six roundings 2^-24 each.
// Two values at a time, by packed arithmetic (8 experts' 2 x 14336 x 4096: 1142 us, 1143 with the fast exp alone).
__device__ __forceinline__ float2 silu_mul2(float2 g, float2 u) {
    constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147181f;
    const float2 x = make_float2(fminf(fmaxf(-g.x, -104.0f), 104.0f), fminf(fmaxf(-g.y, -104.0f), 104.0f));
    const float2 hi = __fmul2_rn(x, make_float2(kLog2e, kLog2e));
    float2 lo = __ffma2_rn(x, make_float2(kLog2e, kLog2e), make_float2(-hi.x, -hi.y));
    lo = __ffma2_rn(x, make_float2(kLog2eRest, kLog2eRest), lo);
    const float2 d = __fadd2_rn(make_float2(ex2_approx(hi.x), ex2_approx(hi.y)), make_float2(1.0f, 1.0f));
    float2 r = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    const float2 rest = __fmul2_rn(__ffma2_rn(r, r, make_float2(-r.x, -r.y)), make_float2(kLn2, kLn2));  // -r (1 - r) ln 2
    r = __ffma2_rn(rest, lo, r);
    return __fmul2_rn(__fmul2_rn(g, r), u);
}

}  // namespace o64
