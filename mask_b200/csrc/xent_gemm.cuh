// The matrix products of the classifier head (xent.cu) on the tensor cores: logits = H W with the statistics of the
// softmax or its gradient as epilogue, and the two products of that gradient G with W and with H.
//
// One persistent block per SM: a producer thread feeds a ring of stages by TMA, one thread issues the MMAs into two
// accumulators of tensor memory (of each group of epilogue warps), eight warps, or sixteen where every logit costs an exponential
// or tiles are narrow, take the finished accumulator apart while the next one is computed.
// Operands are 16-bit "planes": one for bf16 and fp16 input.  FP32 input is scaled by a power of two that brings the
// operand's largest magnitude to 2^14..2^15 and split into two fp16 planes, x = hi + lo + e with |e| <= 2^-22 |x|, or 2^-40
// of the largest where that is more; a product is hi hi + hi lo + lo hi (the dropped lo lo is 2^-22 of it at most).
// The MMA cuts its sum off toward zero after every 16 products: 2e-7 of it at most, which adds up where the terms have one sign
// (16384 steps in a row left 1.7e-3 of dW; 2730 with terms of both signs 2e-5).  For FP32 input an accumulator therefore
// takes kXentSegment blocks of the contraction, and the segments are added in registers, rounded to nearest.  For 16-bit input the
// products with G, whose contraction has no bound, leave an accumulator after kXentLongSegment blocks and are added up in the parts
// (1e-7 times 1024 steps in fp16, 4096 in bf16: a fifth or a tenth of the results' own rounding; half as long cost the two products
// of 16384 x 512 x 16384 fp16 202 us each instead of 192); logits take all of theirs.
// All three products have the layouts TMA and the MMA take as they are, whichever axis is contracted:
//     logits[r,v] = sum_d H[r,d] W[v,d]     both operands K-major
//     dH[r,d]     = sum_v G[r,v] W[v,d]     G K-major, W MN-major
//     dW[v,d]     = sum_r G[r,v] H[r,d]     both MN-major
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "launch.cuh"
#include "umma_ptx.cuh"

namespace mask {

constexpr int kXentTileM = 128, kXentTileK = 64;
constexpr int kXentSegment = 2;                     // blocks of the contraction that an accumulator takes (FP32 input)
constexpr int kXentLongSegmentF16 = 256, kXentLongSegmentBf16 = 1024;      // the same for products with G of 16-bit input
enum XentMode {
    kXentStats,      // logits -> running maximum and sum of each row over a range of classes
    kXentGrad,       // logits -> G of a piece of the classes, with the rows' log sums known
    kXentGradOne,    // the same where one tile holds all classes: log sum, loss and G in one pass
    kXentDHidden,    // G W
    kXentDWeight     // G^T H
};

enum XentStore { kXentFinal, kXentPartial, kXentAccumulate };

struct XentArgs {
    const int32_t* count;      // labelled rows (device)
    int32_t classes, dim;
    int32_t v0, vc;            // piece of the classes
    int32_t splits;            // stats: parts of the classes' tiles; products: parts of the contraction
    int32_t rows_pad;
    int32_t half_type;         // planes hold fp16, not bf16
    const int32_t* label;      // [labelled row]
    const int32_t* row_of;     // [labelled row] -> row of the caller's arrays
    float2* stats;             // [splits * epilogue parts][rows_pad]: maximum, sum of exp(logit - maximum)
    float* label_logit;        // [labelled row]
    float* shift;              // [labelled row]: 16-bit input: log2 of the row's sum of exponentials, rounded up (no probability above 1); FP32: what the sum's
    float* factor;             //   exponents were taken less, and 2^15 over the sum (a log sum rounded to 32 bits would put 1e-6 on a whole row)
    float* row_loss;           // caller's, or NULL
    float* warp_loss;          // [rows_pad / 32]: sums of 32 rows' losses
    float* part;               // [splits][m_pad][n_pad]
    int64_t part_rows;         // m_pad
    int32_t part_ld;           // n_pad
    int32_t store;             // XentStore of a tile's first segment; the others are added to it
    int32_t segment;           // 16-bit input, products with G: blocks of the contraction that an accumulator takes
    void* out;                 // final store: element (m, n) at m * out_m + n * out_n
    int64_t out_m, out_n;
    int32_t out_type;          // MASK_F32 / MASK_BF16 / MASK_F16
    int32_t out_vec;           // rows of 32 values may be written as 32-byte (FP32) or 16-byte vectors
    float scale;
    int32_t mean;              // scale / count
    const uint32_t* range;     // bits of the largest finite magnitudes of hidden and weight, or NULL: planes are the operands themselves
    int32_t* status;
};

// Power of two of an operand's planes: planes = 2^(14 - e) operand.  Below 2^-100 everything is scaled alike.
__device__ __forceinline__ int plane_exponent(uint32_t largest) { return max((int)(largest >> 23) - 127, -100); }
// fp16 planes of G, one or two, hold 2^15 G: without it the probabilities of a head of 2^14 classes are subnormal, those below
// 2^-25 are 0 (a column of dW that is nobody's label was off by up to 2 % where most are), and a scaled loss, which comes behind the products,
// brings none of them back.  bf16 has float32's range.
constexpr int kGradExponent = 15;
// A plane of bf16 operands holds G itself, in 8 bits, as the products behind it take them: rounded once, by 2^-9 of each value at most,
// of the size of the results' own rounding; a second plane would double the two products of it, half of the head's work.

__device__ __forceinline__ float xent_scale(float scale, bool mean, int count) { return mean ? (count > 0 ? scale / (float)count : 0.f) : scale; }
// The same for a product of G's planes with those of an operand: two factors, since the power of two alone may be too small
// for a float.
struct ProductScale {
    float a, b;
    __device__ __forceinline__ float operator()(float x) const { return a * x * b; }
};
__device__ __forceinline__ ProductScale product_scale(float scale, bool mean, int count, const uint32_t* range, int operand, bool half_type) {
    scale = xent_scale(scale, mean, count);
    if (!range) return {half_type ? 1.f / (float)(1 << kGradExponent) : 1.f, scale};
    const int e = plane_exponent(range[operand]) - 14 - kGradExponent;
    return {ldexpf(scale, e / 2), ldexpf(1.f, e - e / 2)};
}

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// Power of two of a product of the planes of hidden and weight.
__device__ __forceinline__ int logit_exponent(const uint32_t* range) { return plane_exponent(range[0]) + plane_exponent(range[1]) - 28; }
// What such a product is multiplied with to become a logit in units of log 2.  Neither infinite (0 stays 0) nor 0 or subnormal
// (-inf, a row's maximum before its first logit, stays -inf): products that are smaller still vanish beside 1 anyway, and larger
// ones are beyond kLogitBound unless they are 0.
__device__ __forceinline__ float logit_factor(const uint32_t* range) { return range ? ldexpf(kLog2e, max(-126, min(logit_exponent(range), 126))) : kLog2e; }
// What the factor leaves out above, for a label's logit, which may be as far below the largest as it likes.
__device__ __forceinline__ float logit_rest(const uint32_t* range) { return range ? ldexpf(1.f, max(logit_exponent(range) - 126, 0)) : 1.f; }
// A row's largest logit, in bits, up to which there is a softmax.  Exponents are taken less the rounded number of bits, off by 64
// at most here; from twice that on they pass what an exponential takes, and the sum would be any number.  The row's sum is NaN
// instead.  (Tiny heads subtract the logits themselves.)
constexpr float kLogitBound = 2147483648.f;
__device__ __forceinline__ float bounded_sum(float sum, float base) { return fabsf(base) < kLogitBound ? sum : NAN; }

// CG: blocks that share a tile.  2: a cluster of two takes 256 rows, each block 128 of them and half of the columns' operand,
// and the first issues the MMAs for both.
// Parts of a tile's columns that different epilogue warps take.  Where every logit costs an exponential, four (16 warps): with
// two, a warp's waits for tensor memory and the special-function unit left the SM idle.
constexpr int xent_parts(int bn, int planes, bool logits) { return bn == 64 ? 1 : (planes == 1 && logits ? 4 : 2); }
// Columns that a warp writes of G at a time.
constexpr int xent_box(int bn, int planes) { return planes == 1 && bn / xent_parts(bn, planes, true) >= 64 ? 64 : 32; }

template <int BN, int P, int MODE, int CG>
struct XentLayout {
    // Epilogue warps: 4 quarters of 32 rows, each for so many parts of the columns -- and for narrow tiles groups of such warps
    // that take tiles in turn, since one such tile is all waiting (products with G of 300000 x 64 x 40, bf16: 23 and
    // 17 us, 32 and 23 with one group).
    static constexpr int kParts = xent_parts(BN, P, MODE <= kXentGradOne);
    static constexpr int kGroups = BN == 64 ? (P == 1 ? 4 : 2) : 1;
    static constexpr int kWarps = 4 * kParts * kGroups;
    static constexpr int kBuffers = 2 * kGroups;                          // accumulators, two a group
    // + producer + MMA issuer; where segments are summed in registers (P == 2) two warps more make three whole warpgroups, whose
    // 168 registers a thread are dealt again: 216 to the two that take accumulators apart, 72 to the third (3 x 168 in all).
    static constexpr int kThreads = 32 * (kWarps + (P == 2 ? 4 : 2));
    static constexpr bool kWritesG = MODE == kXentGrad || MODE == kXentGradOne;
    static constexpr int kTileA = kXentTileM * kXentTileK * 2, kTileB = BN / CG * kXentTileK * 2;
    static constexpr int kStage = P * (kTileA + kTileB);
    // G leaves through a warp's staging buffer of 4 KB: 32 rows of 64 columns where the warp has as many, else of 32, for both
    // planes or two in turn.
    static constexpr int kBox = xent_box(BN, P);
    static constexpr int kStagingBuffer = 4096;
    static constexpr int kStaging = kWritesG ? kWarps * kStagingBuffer : 0;
    static constexpr int kExchangeBytes = MODE == kXentGradOne ? 2 * kParts * 128 * 12 : 0;   // one-pass mode: [2 turns][parts][128 rows]
    static constexpr int kMost = 227 * 1024 - 1024 - 256 - kStaging - kExchangeBytes;
    static constexpr int S = kMost / kStage < 8 ? kMost / kStage : 8;
    static constexpr int kTmemCols = kBuffers * BN;
    static constexpr int kStagingAt = S * kStage;
    static constexpr int kExchange = kStagingAt + kStaging;
    static constexpr int kBars = kExchange + kExchangeBytes;
    static constexpr int kNumBars = 2 * S + 2 * kBuffers + 1 + 4;
    static constexpr int kTmemSlot = kBars + kNumBars * 8;
    static constexpr int kAbort = kTmemSlot + 8;
    static constexpr int kBytes = kAbort + 8;
    static constexpr int kDynamicBytes = kBytes + 1024;                    // room to align the base
    static_assert(S >= 2 && kDynamicBytes <= 227 * 1024 && kTmemCols <= 512, "tile does not fit");
};

// Descriptors as their two halves: stepping through an operand is one 32-bit addition.
template <int CG>
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}"
            ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, p;\n\t}"
            ::"r"(d_tmem), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate)
            : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// Bounded wait of a whole warp: a probe first, which is enough where the phase is over already.
__device__ __forceinline__ bool wait_all_lanes(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
    if (__all_sync(0xffffffffu, mbar_probe(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
}
// Arrives on `bar`, of both blocks of a pair, when the MMAs issued so far are done.
template <int CG>
__device__ __forceinline__ void xent_commit(uint32_t bar) {
    if constexpr (CG == 1) umma_commit(bar);
    else
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((uint16_t)3)
                     : "memory");
}
// The address of the same shared memory in the first block of the pair.
template <int CG>
__device__ __forceinline__ uint32_t in_leader(uint32_t at) {
    if constexpr (CG == 1) return at;
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(at));
    return r;
}
template <int CG>
__device__ __forceinline__ void arrive_at_leader(uint32_t bar) {
    if constexpr (CG == 1) mbar_arrive(bar);
    else asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(in_leader<CG>(bar)) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
// Completes on `bar`, which with CG == 2 is the first block's.
template <int CG>
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
    if constexpr (CG == 1)
        asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
                     : "memory");
    else
        asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                     ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
                     : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void xent_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ void st_shared_u16(uint32_t at, uint16_t v) {
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(v) : "memory");
}
// A whole 32-byte sector by one thread: pieces of 16 bytes of 32 different rows cost the L2 twice the requests.
__device__ __forceinline__ void st_global_v8(float* at, const float* v) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(at), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                 : "memory");
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b, bool half_type) {
    if (half_type) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// What a row's exponents are taken less: its maximum in bits, rounded.  Going from one to another multiplies the sum by
// exp2 of the difference of the two rounded numbers -- exactly 1 where they are the same; with an exact product on one side
// the sum drifts by a rounding with every 32 logits.
__device__ __forceinline__ float exponent_base(float top, float f) { return top == -INFINITY ? 0.f : __fmul_rn(top, f); }    // a row that has seen only -inf
__device__ __forceinline__ float rebase(float top, float f, float base) { return fast_exp2(__fsub_rn(__fmul_rn(top, f), base)); }

// Adds 32 logits of a row, in units of 1 / f bits, to its running maximum and sum.
__device__ __forceinline__ void online_softmax(const float (&v)[32], float f, float& top, float& sum) {
    float t[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int i = 4; i < 32; i++) t[i & 3] = fmaxf(t[i & 3], v[i]);
    const float now = fmaxf(top, fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
    const float base = exponent_base(now, f);
    float s[4] = {sum * rebase(top, f, base), 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 32; i++) s[i & 3] += fast_exp2(fmaf(v[i], f, -base));
    sum = (s[0] + s[1]) + (s[2] + s[3]);
    top = now;
}

// v[i] for an index of the thread's own, 0 <= i < 32: 31 selections.
__device__ __forceinline__ float pick(const float (&v)[32], int i) {
    float t[16];
#pragma unroll
    for (int j = 0; j < 16; j++) t[j] = i & 1 ? v[2 * j + 1] : v[2 * j];
#pragma unroll
    for (int j = 0; j < 8; j++) t[j] = i & 2 ? t[2 * j + 1] : t[2 * j];
#pragma unroll
    for (int j = 0; j < 4; j++) t[j] = i & 4 ? t[2 * j + 1] : t[2 * j];
    t[0] = i & 8 ? t[1] : t[0];
    t[1] = i & 8 ? t[3] : t[2];
    return i & 16 ? t[1] : t[0];
}

template <int BN, int P, int MODE, int CG>
__global__ void __launch_bounds__((XentLayout<BN, P, MODE, CG>::kThreads), 1)
xent_gemm_kernel(const XentArgs p, const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                 const __grid_constant__ CUtensorMap map_g) {
    using L = XentLayout<BN, P, MODE, CG>;
    constexpr int S = L::S;
    constexpr bool kLogits = MODE == kXentStats || MODE == kXentGrad || MODE == kXentGradOne;
    constexpr bool kAmn = MODE == kXentDWeight, kBmn = !kLogits;
    extern __shared__ unsigned char xent_smem_raw[];
    const uint32_t raw = (uint32_t)__cvta_generic_to_shared(xent_smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    unsigned char* gbase = xent_smem_raw + (base - raw);
    const uint32_t bars = base + L::kBars;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    auto accf_bar = [&](int b) { return bars + 8u * (2 * S + b); };
    auto acce_bar = [&](int b) { return bars + 8u * (2 * S + L::kBuffers + b); };
    const uint32_t drain_bar = bars + 8u * (2 * S + 2 * L::kBuffers);
    auto exchange_bar = [&](int q) { return bars + 8u * (2 * S + 2 * L::kBuffers + 1 + q); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gbase + L::kAbort);
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + L::kTmemSlot);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    uint32_t rank = 0;                                  // within the pair
    if constexpr (CG == 2) asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const int64_t group = blockIdx.x / CG, groups = gridDim.x / CG;

    if (tid == 0) {
        *abort_flag = 0;
        for (int s = 0; s < S; s++) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < L::kBuffers; b++) {
            mbar_init(accf_bar(b), 1);
            mbar_init(acce_bar(b), CG * L::kWarps / L::kGroups);
        }
        for (int q = 0; q < 4; q++) mbar_init(exchange_bar(q), L::kParts);
        mbar_init(drain_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == L::kWarps + 1) {
        if constexpr (CG == 1) {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::kTmemSlot), "r"(L::kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::kTmemSlot), "r"(L::kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (CG == 2) cluster_sync();             // both blocks' barriers and tensor memory are there
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_slot;

    wait_for_previous_kernel();
    let_next_kernel_start();

    // ---- work: an item is a tile of rows with a range of column tiles and a range of blocks of the contraction ----------
    const int count = *p.count;
    const int m_extent = MODE == kXentDWeight ? p.vc : count;
    const int n_extent = kLogits ? p.vc : p.dim;
    const int k_extent = kLogits ? p.dim : (MODE == kXentDHidden ? p.vc : count);
    const int m_tiles = (m_extent + CG * kXentTileM - 1) / (CG * kXentTileM), n_tiles = (n_extent + BN - 1) / BN;
    const int k_blocks = (k_extent + kXentTileK - 1) / kXentTileK;
    // stats: parts of the column tiles; G: every tile an item; products: every tile once for each part of the contraction
    const int64_t items = (int64_t)m_tiles * (MODE == kXentStats ? p.splits : (kLogits ? n_tiles : n_tiles * p.splits));
    struct Item { int m, split, n0, n1, k0, k1; };
    auto item_of = [&](int64_t i) {
        Item t;
        if constexpr (kLogits) {          // row tiles fastest: blocks that run together read the same tile of W
            const int q = (int)(i / m_tiles);
            t.m = (int)(i - (int64_t)q * m_tiles);
            t.split = MODE == kXentStats ? q : 0;
            t.n0 = MODE == kXentStats ? (int)((int64_t)n_tiles * q / p.splits) : q;
            t.n1 = MODE == kXentStats ? (int)((int64_t)n_tiles * (q + 1) / p.splits) : q + 1;
            t.k0 = 0;
            t.k1 = k_blocks;
        } else {                          // column tiles fastest: they share the tile of G
            const int64_t q = i / n_tiles;
            t.n0 = (int)(i - q * n_tiles);
            t.n1 = t.n0 + 1;
            t.split = (int)(q / m_tiles);
            t.m = (int)(q - (int64_t)t.split * m_tiles);
            t.k0 = (int)((int64_t)k_blocks * t.split / p.splits);
            t.k1 = (int)((int64_t)k_blocks * (t.split + 1) / p.splits);
        }
        return t;
    };

    if (warp >= L::kWarps) {
        if constexpr (P == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == L::kWarps) {
            // ------------------------------ producer -----------------------------------------------------------------------
            if (lane == 0) {
                int s = 0;
                uint32_t round = 0;
                bool ok = true;
                for (int64_t i = group; i < items && ok; i += groups) {
                    const Item t = item_of(i);
                    for (int n = t.n0; n < t.n1 && ok; n++) {
                        for (int k = t.k0; k < t.k1; k++) {
                            if (round > 0 && !mbar_wait(empty_bar(s), (round - 1) & 1, abort_flag)) { ok = false; break; }
                            const uint32_t bar = in_leader<CG>(full_bar(s)), at = base + s * L::kStage;
                            if (rank == 0) xent_expect_tx(full_bar(s), CG * L::kStage);
                            const int am = (t.m * CG + (int)rank) * kXentTileM, bn = n * BN + (int)rank * (BN / CG);
#pragma unroll
                            for (int z = 0; z < P; z++) {
                                const uint32_t a = at + z * L::kTileA, b = at + P * L::kTileA + z * L::kTileB;
                                if constexpr (kAmn) {
#pragma unroll
                                    for (int j = 0; j < kXentTileM / 64; j++)
                                        tma_load_3d<CG>(a + j * 8192, &map_a, bar, am + j * 64, k * kXentTileK, z);
                                } else {
                                    tma_load_3d<CG>(a, &map_a, bar, k * kXentTileK, am, z);
                                }
                                if constexpr (kBmn) {
#pragma unroll
                                    for (int j = 0; j < BN / CG / 64; j++)
                                        tma_load_3d<CG>(b + j * 8192, &map_b, bar, bn + j * 64, (MODE == kXentDHidden ? p.v0 : 0) + k * kXentTileK, z);
                                } else {
                                    tma_load_3d<CG>(b, &map_b, bar, k * kXentTileK, p.v0 + bn, z);
                                }
                            }
                            if (++s == S) { s = 0; round++; }
                        }
                    }
                }
            }
            __syncwarp();
        } else if (warp == L::kWarps + 1) {
            // ------------------------------ MMA issuer, of the pair's first block ----------------------------------------------
            // The whole warp goes through the loop and one elected lane issues, so that descriptors live in uniform registers:
            // from within a branch of one lane, four MMAs of 512 clocks took 790 to issue.
            if (rank == 0) {
                const bool elected = elect_one();
                const uint32_t fmt = p.half_type ? 0u : 1u;
                // instruction descriptor: D = F32, A and B bf16 or fp16, M = 128 a block
                const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (kAmn ? 1u << 15 : 0u) | (kBmn ? 1u << 16 : 0u) |
                                       ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(CG * kXentTileM >> 4) << 24);
                // 128-byte swizzle; K-major: groups of 8 rows 1024 bytes apart; MN-major: 64-wide atoms 8192 bytes apart, groups of 8 k 1024
                const uint64_t a0 = umma_smem_desc(base, kAmn ? 512 : 1, 64, 2);
                const uint64_t b0 = umma_smem_desc(base + P * L::kTileA, kBmn ? 512 : 1, 64, 2);
                const uint32_t a_hi = (uint32_t)(a0 >> 32), b_hi = (uint32_t)(b0 >> 32);
                constexpr uint32_t kStepA = kAmn ? 128 : 2, kStepB = kBmn ? 128 : 2;   // 16 of the contraction, in 16 bytes
                uint32_t a_lo = (uint32_t)a0, b_lo = (uint32_t)b0;                     // of stage s
                int s = 0;
                uint32_t round = 0, turn = 0;
                uint32_t uses[L::kGroups];                                             // of the groups' accumulators
#pragma unroll
                for (int g = 0; g < L::kGroups; g++) uses[g] = 0;
                bool ok = true;
                for (int64_t i = group; i < items && ok; i += groups, turn++) {
                    const Item t = item_of(i);
                    if (t.k0 >= t.k1) continue;
                    const uint32_t g = turn % L::kGroups;
                    uint32_t acc_it = uses[0];
#pragma unroll
                    for (int q = 1; q < L::kGroups; q++) acc_it = g == q ? uses[q] : acc_it;
                    for (int n = t.n0; n < t.n1 && ok; n++) {
                        uint32_t buf = 0, acc = 0, open = 0;
                        int left = 0;                        // blocks that the open accumulator still takes
                        for (int k = t.k0; k < t.k1; k++) {
                            if (!open) {
                                buf = 2 * g + (acc_it & 1);
                                acc = tmem_base + buf * BN;
                                left = P == 2 ? min(kXentSegment, t.k1 - k) : (kLogits ? t.k1 - k : min(p.segment, t.k1 - k));
                                if (acc_it >= 2 && !wait_all_lanes(acce_bar(buf), ((acc_it >> 1) - 1) & 1, abort_flag)) { ok = false; break; }
                            }
                            if (!wait_all_lanes(full_bar(s), round & 1, abort_flag)) { ok = false; break; }
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            if (elected) {
#pragma unroll
                                for (int c = 0; c < (P == 2 ? 3 : 1); c++) {     // hi hi, hi lo, lo hi
#pragma unroll
                                    for (int j = 0; j < kXentTileK / 16; j++)
                                        umma_f16<CG>(acc, a_lo + (c == 2 ? L::kTileA >> 4 : 0) + j * kStepA, a_hi, b_lo + (c == 1 ? L::kTileB >> 4 : 0) + j * kStepB,
                                                     b_hi, idesc, c + j ? 1u : open);
                                }
                                xent_commit<CG>(empty_bar(s));
                                if (left == 1) xent_commit<CG>(accf_bar(buf));
                            }
                            __syncwarp();
                            open = --left > 0;
                            if (left == 0) acc_it++;
                            a_lo += L::kStage >> 4;
                            b_lo += L::kStage >> 4;
                            if (++s == S) {
                                s = 0; round++;
                                a_lo = (uint32_t)a0; b_lo = (uint32_t)b0;
                            }
                        }
                    }
#pragma unroll
                    for (int q = 0; q < L::kGroups; q++) uses[q] = g == q ? acc_it : uses[q];
                }
                // whatever was issued must have finished before shared and tensor memory go away
                if (elected) xent_commit<CG>(drain_bar);
                __syncwarp();
                const long long start = clock64();
                while (!mbar_test(drain_bar, 0)) {
                    if (clock64() - start > kUmmaWaitCycles) { *abort_flag = 1; break; }
                }
            }
            __syncwarp();
        }
    } else {
        // ------------------------------ epilogue -----------------------------------------------------------------------
        if constexpr (P == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        constexpr int kWidth = BN / L::kParts;             // columns of a warp
        constexpr int kChunks = kWidth / 32, kUnroll = P == 2 ? kChunks : 1;
        const int quarter = warp & 3, part = (warp >> 2) % L::kParts;
        const uint32_t mine = (warp >> 2) / L::kParts;       // the group
        uint32_t acc_it = 0;
        bool ok = true;
        const bool half_type = p.half_type != 0;
        [[maybe_unused]] const uint32_t staging = base + L::kStagingAt + warp * L::kStagingBuffer;
        [[maybe_unused]] uint32_t stage_it = 0;
        uint32_t acc = 0;                                // the tile's accumulator in tensor memory (P == 1)
        [[maybe_unused]] float total[P == 2 ? kWidth : 1];   // or its sum so far
        auto release = [&]() {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) arrive_at_leader<CG>(acce_bar(2 * mine + (acc_it & 1)));
            acc_it++;
        };
        auto next_accumulator = [&]() -> bool {
            const uint32_t buf = 2 * mine + (acc_it & 1);
            if (!__all_sync(0xffffffffu, mbar_wait(accf_bar(buf), (acc_it >> 1) & 1, abort_flag))) return false;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            acc = tmem_base + ((uint32_t)(32 * quarter) << 16) + buf * BN + part * kWidth;
            return true;
        };
        // The tile's columns of this warp: left in tensor memory, or summed up from its segments.
        auto acquire = [&](int k0, int k1) -> bool {
            if constexpr (P == 1) return next_accumulator();
            for (int k = k0; k < k1; k += kXentSegment) {
                if (!next_accumulator()) return false;
                if (k == k0) {
#pragma unroll
                    for (int j = 0; j < (P == 2 ? kWidth : 0); j++) total[j] = 0.f;
                }
#pragma unroll
                for (int c = 0; c < 2 * kChunks; c++) {
                    uint32_t u[16];
                    tmem_ld16(acc + 16 * c, u);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 16; j++) total[P == 2 ? 16 * c + j : 0] += __uint_as_float(u[j]);
                }
                release();
            }
            return true;
        };
        auto done = [&]() {
            if constexpr (P == 1) release();
        };
        auto values = [&](int c, float (&v)[32]) {
            if constexpr (P == 1) {
                uint32_t u[32];
                tmem_ld32(acc + 32 * c, u);
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = __uint_as_float(u[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = total[32 * c + j];
            }
        };
        // G of the warp's 32 columns number c to global memory, through its staging buffer
        [[maybe_unused]] auto write_g = [&](const float (&g)[32], int row0, int col, int c, int y, float at_label) {
            if constexpr (L::kWritesG) {
                if (row0 >= p.rows_pad) return;            // a pair's second tile may lie behind the last row
                constexpr bool kWide = L::kBox == 64;
                const bool begins = !kWide || (c & 1) == 0, ends = !kWide || (c & 1) == 1;
                // what the buffer held must have been read, but for the other one of two in turn
                if (begins) {
                    if (lane == 0) {
                        if constexpr (P == 1 && !kWide) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                        else asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                    }
                    __syncwarp();
                }
                const uint32_t row = staging + lane * (kWide ? 128 : 64), x = kWide ? lane & 7 : (lane >> 1) & 3;
                const uint32_t first = P == 1 && !kWide ? (stage_it & 1) * 2048 : 0, chunk0 = kWide ? (c & 1) * 4 : 0;
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float u = g[8 * i + 2 * j], w = g[8 * i + 2 * j + 1];
                        h[j] = pack_half2(u, w, half_type);
                        if constexpr (P == 2) {
                            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
                            l[j] = pack_half2(u - f.x, w - f.y, true);
                        }
                    }
                    st_shared_v4(row + first + (((chunk0 + i) ^ x) << 4), h[0], h[1], h[2], h[3]);
                    if constexpr (P == 2) st_shared_v4(row + 2048 + ((i ^ x) << 4), l[0], l[1], l[2], l[3]);
                }
                if ((uint32_t)(y - col) < 32u) {           // this row's label is among the columns
                    const uint32_t i = y - col;
                    const uint16_t h = (uint16_t)pack_half2(at_label, 0.f, half_type);
                    st_shared_u16(row + first + (((chunk0 + (i >> 3)) ^ x) << 4) + 2 * (i & 7), h);
                    if constexpr (P == 2)
                        st_shared_u16(row + 2048 + (((i >> 3) ^ x) << 4) + 2 * (i & 7), (uint16_t)pack_half2(at_label - __half2float(__ushort_as_half(h)), 0.f, true));
                }
                if (ends) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
#pragma unroll
                        for (int z = 0; z < P; z++) tma_store_3d(&map_g, staging + first + z * 2048, kWide ? col - 32 : col, row0, z);
                        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                    }
                    stage_it++;
                }
            }
        };

        [[maybe_unused]] uint32_t turn = 0, count_of_items = 0;
        // 32 values of row r of a product, from column col, to the parts or to the caller
        [[maybe_unused]] auto write_out = [&](const float (&v)[32], const ProductScale& scale, int store, int split, int r, int col) {
            if (store != kXentFinal) {
                float* to = p.part + ((int64_t)split * p.part_rows + r) * p.part_ld + col;
                if (store == kXentAccumulate) {
                    float sum[32];
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float4 w = reinterpret_cast<const float4*>(to)[j];
                        sum[4 * j] = v[4 * j] + w.x; sum[4 * j + 1] = v[4 * j + 1] + w.y; sum[4 * j + 2] = v[4 * j + 2] + w.z; sum[4 * j + 3] = v[4 * j + 3] + w.w;
                    }
#pragma unroll
                    for (int j = 0; j < 4; j++) st_global_v8(to + 8 * j, sum + 8 * j);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) st_global_v8(to + 8 * j, v + 8 * j);
                }
                return;
            }
            const int64_t row = MODE == kXentDHidden ? (int64_t)p.row_of[r] : (int64_t)p.v0 + r;
            const int64_t at = row * p.out_m + (int64_t)col * p.out_n;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int left = n_extent - col - 8 * j;      // eight values at a time
                const int64_t to = at + 8 * j * p.out_n;
                if (p.out_vec && left >= 8) {
                    if (p.out_type == MASK_F32) {
                        float x[8];
#pragma unroll
                        for (int i = 0; i < 8; i++) x[i] = scale(v[8 * j + i]);
                        st_global_v8(static_cast<float*>(p.out) + to, x);
                    } else {
                        uint32_t h[4];
#pragma unroll
                        for (int q = 0; q < 4; q++) h[q] = pack_half2(scale(v[8 * j + 2 * q]), scale(v[8 * j + 2 * q + 1]), p.out_type == MASK_F16);
                        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + to) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (i >= left) continue;
                    const float x = scale(v[8 * j + i]);
                    if (p.out_type == MASK_F32) static_cast<float*>(p.out)[to + i * p.out_n] = x;
                    else if (p.out_type == MASK_F16) static_cast<__half*>(p.out)[to + i * p.out_n] = __float2half_rn(x);
                    else static_cast<__nv_bfloat16*>(p.out)[to + i * p.out_n] = __float2bfloat16_rn(x);
                }
            }
        };
        const float f = kLogits ? logit_factor(p.range) : 0.f;
        // exp(logit) over the row's sum, for fp16 planes times 2^15 (one plane: `shift` is less by that, rounded up so that nothing
        // passes 2^15); 0 outside the classes and the rows, whatever the weight made of a row of zeros (infinities: NaN)
        const float one = half_type ? (float)(1 << kGradExponent) : 1.f;
        auto row_shift = [&](float shift) { return P == 1 && half_type ? __fadd_ru(shift, -(float)kGradExponent) : shift; };
        [[maybe_unused]] auto gradient = [&](float (&v)[32], int col, int classes, bool live, float shift, float factor) {
#pragma unroll
            for (int j = 0; j < 32; j++) v[j] = fast_exp2(fmaf(v[j], f, -shift)) * (P == 2 ? factor : 1.f);
            if (__any_sync(0xffffffffu, !live)) {
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = live ? v[j] : 0.f;
            }
            if (col + 32 > classes) {
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (col + j >= classes) v[j] = 0.f;
            }
        };
        // the same less 1 at the row's label, whose logit is `picked`
        [[maybe_unused]] auto label_gradient = [&](float picked, float shift, float factor) {
            const float e = fast_exp2(fmaf(picked, f, -shift));
            return P == 2 ? e * factor - one : e - one;
        };
        for (int64_t i = group; i < items && ok; i += groups) {
            if (L::kGroups > 1 && count_of_items++ % L::kGroups != mine) continue;
            const Item t = item_of(i);
            const int r = (t.m * CG + (int)rank) * kXentTileM + 32 * quarter + lane;     // row of the tile that this thread holds
            if constexpr (MODE == kXentStats) {
                const int y = r < count ? p.label[r] : -1;
                float top = -INFINITY, sum = 0.f, picked = 0.f;
                bool have = false;
                for (int n = t.n0; n < t.n1; n++) {
                    if (!acquire(t.k0, t.k1)) { ok = false; break; }
#pragma unroll(kUnroll)
                    for (int c = 0; c < kChunks; c++) {
                        const int col = n * BN + part * kWidth + 32 * c;
                        if (col >= p.classes) break;
                        float v[32];
                        values(c, v);
                        if (col + 32 > p.classes) {
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (col + j >= p.classes) v[j] = -INFINITY;
                        }
                        online_softmax(v, f, top, sum);
                        if (__any_sync(0xffffffffu, (uint32_t)(y - col) < 32u)) {
                            const float x = pick(v, y - col);
                            if ((uint32_t)(y - col) < 32u) { picked = x; have = true; }
                        }
                    }
                    done();
                }
                if (ok && r < count) {
                    p.stats[(int64_t)(L::kParts * t.split + part) * p.rows_pad + r] = make_float2(top, sum);
                    if (have) p.label_logit[r] = picked;
                }
            } else if constexpr (MODE == kXentGrad) {
                const bool live = r < count;
                const int label = live ? p.label[r] - p.v0 : -1, y = label < p.vc ? label : -1;       // within the piece
                const float shift = live ? row_shift(p.shift[r]) : 0.f, factor = P == 2 && live ? p.factor[r] : 0.f;
                const float at_label = y >= 0 ? label_gradient(p.label_logit[r], shift, factor) : 0.f;
                if (!acquire(t.k0, t.k1)) { ok = false; break; }
#pragma unroll(kUnroll)
                for (int c = 0; c < kChunks; c++) {
                    const int col = t.n0 * BN + part * kWidth + 32 * c;     // within the piece
                    float v[32];
                    values(c, v);
                    gradient(v, col, p.vc, live, shift, factor);
                    write_g(v, r - lane, col, c, y, at_label);
                }
                done();
            } else if constexpr (MODE == kXentGradOne) {
                const bool live = r < count;
                const int y = live ? p.label[r] : -1;
                if (!acquire(t.k0, t.k1)) { ok = false; break; }
                float top = -INFINITY, sum = 0.f, picked = 0.f;
#pragma unroll(kUnroll)
                for (int c = 0; c < kChunks; c++) {
                    const int col = part * kWidth + 32 * c;
                    if (col >= p.classes) break;
                    float v[32];
                    values(c, v);
                    if (col + 32 > p.classes) {
#pragma unroll
                        for (int j = 0; j < 32; j++)
                            if (col + j >= p.classes) v[j] = -INFINITY;
                    }
                    online_softmax(v, f, top, sum);
                    const float x = pick(v, y - col);
                    if ((uint32_t)(y - col) < 32u) picked = x;
                }
                // The warps that hold parts of the same rows tell one another.  Two turns' worth of room: a warp writes turn i + 2
                // after all others have arrived at turn i + 1, hence read turn i.
                float* ex = reinterpret_cast<float*>(gbase + L::kExchange) + (turn & 1) * L::kParts * 128 * 3 + (32 * quarter + lane) * 3;
                if constexpr (L::kParts > 1) {
                    ex[part * 128 * 3] = top;
                    ex[part * 128 * 3 + 1] = sum;
                    ex[part * 128 * 3 + 2] = picked;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(exchange_bar(quarter));
                    if (!__all_sync(0xffffffffu, mbar_wait(exchange_bar(quarter), turn & 1, abort_flag))) { ok = false; break; }
                    turn++;
                }
                // all parts in the same order everywhere, so that everybody gets the same bits
                float most = top, all = sum, at_label = picked;
                if constexpr (L::kParts > 1) {
                    most = ex[0];
#pragma unroll
                    for (int i = 1; i < L::kParts; i++) most = fmaxf(most, ex[i * 128 * 3]);
                    all = at_label = 0.f;
                }
                const float bs = exponent_base(most, f);
                if constexpr (L::kParts > 1) {
#pragma unroll
                    for (int i = 0; i < L::kParts; i++) {
                        all += ex[i * 128 * 3 + 1] * rebase(ex[i * 128 * 3], f, bs);
                        at_label += ex[i * 128 * 3 + 2];
                    }
                }
                all = bounded_sum(all, bs);
                const float log_sum = log2f(all), shift = P == 2 ? bs : row_shift(__fadd_ru(bs, log_sum));
                const float factor = P == 2 && live ? (float)(1 << kGradExponent) / all : 0.f;
                const float own = live ? label_gradient(at_label, shift, factor) : 0.f;
                if (part == 0) {
                    const float loss = live ? kLn2 * (fmaf(-at_label * logit_rest(p.range), f, bs) + log_sum) : 0.f;
                    if (live && p.row_loss) p.row_loss[p.row_of[r]] = loss;
                    float w = loss;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
                    if (lane == 0 && r < p.rows_pad) p.warp_loss[r >> 5] = w;
                }
#pragma unroll(kUnroll)
                for (int c = 0; c < kChunks; c++) {
                    const int col = part * kWidth + 32 * c;
                    float v[32];
                    values(c, v);
                    gradient(v, col, p.classes, live, shift, factor);
                    write_g(v, r - lane, col, c, y, own);
                }
                done();
            } else {
                const bool empty = t.k0 >= t.k1;      // nothing to contract: the sum is zero
                const ProductScale scale = product_scale(p.scale, p.mean, count, p.range, MODE == kXentDHidden ? 1 : 0, half_type);
                const bool live = r < m_extent;
                int store = p.store, k = t.k0;
                do {                                  // segment by segment
                    if (!empty && !acquire(t.k0, t.k1)) { ok = false; break; }
#pragma unroll(kUnroll)
                    for (int c = 0; c < kChunks; c++) {
                        const int col = t.n0 * BN + part * kWidth + 32 * c;
                        if (col >= n_extent) break;
                        float v[32];
                        if (!empty) {
                            __syncwarp();
                            values(c, v);
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; j++) v[j] = 0.f;
                        }
                        if (live) write_out(v, scale, store, t.split, r, col);
                    }
                    if (!empty) done();
                    store = kXentAccumulate;
                    k += p.segment;
                } while (P == 1 && k < t.k1);
            }
        }
        if constexpr (L::kWritesG) {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
            __syncwarp();
        }
    }

    // ---- teardown: everybody gets here, aborting or not ---------------------------------------------------------------
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    // The pair's first block has waited for all its MMAs; the other one may still be reading or signalling this one.
    if constexpr (CG == 2) cluster_sync();
    if (*abort_flag) {
        // copies that were issued but never consumed may still be landing in this block's shared memory
        const long long start = clock64();
        while (clock64() - start < 2000000LL) {
        }
        __syncthreads();
    }
    if (warp == L::kWarps + 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(L::kTmemCols) : "memory");
    }
    if (tid == 0 && *abort_flag) atomicExch(p.status, 1);
}

}  // namespace mask
