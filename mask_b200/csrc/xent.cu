// Classifier head: softmax cross entropy of hidden * weight over the labelled rows and its gradients, without the
// logits in memory and with at most 2 GB (or 256 classes) of their gradient at a time (mask_linear_xent).
//
// With L the labelled rows, l = H W, s_r = log sum_v exp l_rv and G_rv = exp(l_rv - s_r) - [v = y_r]:
//     loss_r = s_r - l_{r,y_r},   dH = scale G W^T,   dW = scale H^T G.
// Steps (matrix products in xent_gemm.cuh):
//   1. the labelled rows are numbered (their order kept) and packed, with the weight, into zero-padded 16-bit planes that
//      TMA can fetch: every later step costs what the labelled rows cost, and nothing an unlabelled row holds goes on;
//   2. logits tile by tile, each row's running maximum and sum kept; parts of the classes are joined in a fixed order;
//   3. for a piece of the classes at a time: the logits' tiles again, now turned into G (in 16-bit planes, in scratch), then
//      dH += G W and that piece of dW = G^T H.
// Few classes (up to 256, FP32 128) fit one tile, and steps 2 and 3 share one product.  Contractions that leave SMs idle are split and
// their parts summed in a fixed order.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "tensor_map.h"
#include "xent_gemm.cuh"

namespace mask {

constexpr int kXentCountThreads = 1024;
// Rows and values (of hidden and of a weight that has to be packed) up to which one block prepares them, three launches fewer:
// 50 x 16 x 64, loss alone, 13.4 us and 17.3 without; 3000 x 20 x 40 58 us and 41.
constexpr int kXentSmallRows = 4096;
constexpr int64_t kXentSmallValues = 8192;
// What a piece of G may take.  Few pieces fill the SMs better and add dH up less often: 16384 x 512 x 131072 bf16 takes 7.2 ms
// with 2 GB, 7.6 with 1, 7.8 with 512 MB (which stays no more in the L2), 9.2 with 128; 200000 x 512 x 1000 float32 2.3, 2.4,
// 3.0 and 3.3.
constexpr size_t kXentPieceBytes = (size_t)2 << 30;

// ---- numbering of the labelled rows ------------------------------------------------------------------
__device__ __forceinline__ bool labelled(int64_t y, int32_t classes) { return y >= 0 && y < classes; }

struct XentNumberArgs {
    const int64_t* labels;
    int64_t rows, chunk;
    int32_t classes;
    const int32_t* counts;
    int32_t* row_of;
    int32_t* label;
    int32_t* total;
    int32_t* status;
    uint32_t* range;
    const uint2* ranges;       // what the scan's blocks found, or NULL: to be found later
    int32_t n_ranges;
    float* row_loss;
};

// The largest of all threads' values, for thread 0.
__device__ __forceinline__ void block_max(uint32_t (&most)[2]) {
    __shared__ uint32_t room[2];
    if (threadIdx.x < 2) room[threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, most[k]);
        if ((threadIdx.x & 31) == 0 && m) atomicMax(room + k, m);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        most[0] = room[0];
        most[1] = room[1];
    }
}

// Writes row_of and label of the block's chunk of rows behind those of the chunks before it; the last block leaves the
// total.  Losses of rows without a label are set to 0 here.
__device__ __forceinline__ void number_rows(const XentNumberArgs& p) {
    __shared__ int sums[32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int at = 0;
    for (int b = threadIdx.x; b < (int)blockIdx.x; b += kXentCountThreads) at += p.counts[b];
    at = __reduce_add_sync(0xffffffffu, at);
    if (lane == 0) sums[warp] = at;
    __syncthreads();
    at = __reduce_add_sync(0xffffffffu, sums[lane]);
    const int64_t r0 = blockIdx.x * p.chunk, r1 = min(p.rows, r0 + p.chunk);
    for (int64_t rb = r0; rb < r1; rb += kXentCountThreads) {
        const int64_t r = rb + threadIdx.x;
        const int64_t y = r < r1 ? p.labels[r] : -1;
        const bool mine = labelled(y, p.classes);
        const unsigned ballot = __ballot_sync(0xffffffffu, mine);
        __syncthreads();
        if (lane == 0) sums[warp] = __popc(ballot);
        __syncthreads();
        const int in_warp = sums[lane];
        const int before = __reduce_add_sync(0xffffffffu, lane < warp ? in_warp : 0);
        if (mine) {
            const int to = at + before + __popc(ballot & ((1u << lane) - 1));
            p.row_of[to] = (int32_t)r;
            p.label[to] = (int32_t)y;
        } else if (r < r1 && p.row_loss) {
            p.row_loss[r] = 0.f;
        }
        at += __reduce_add_sync(0xffffffffu, in_warp);
    }
    if (blockIdx.x < gridDim.x - 1) return;
    uint32_t most[2] = {0, 0};
    if (p.ranges) {
        for (int i = threadIdx.x; i < p.n_ranges; i += kXentCountThreads) {
            const uint2 m = p.ranges[i];
            most[0] = max(most[0], m.x);
            most[1] = max(most[1], m.y);
        }
        block_max(most);
    }
    if (threadIdx.x == 0) {
        *p.total = at;
        *p.status = 0;
        p.range[0] = most[0];
        p.range[1] = most[1];
    }
}
__global__ void __launch_bounds__(kXentCountThreads) xent_number_kernel(const XentNumberArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    number_rows(p);
}

// ---- planes ----------------------------------------------------------------------------------------------
struct XentPackArgs {
    int32_t dim, dim_pad, classes;
    int64_t rows;
    const int32_t* count;
    const int32_t* row_of;
    const int64_t* labels;
    const void* hidden;
    int64_t hidden_stride;
    uint16_t* h_planes;        // [P][rows_pad][dim_pad]
    int64_t h_plane;
    const void* weight;        // NULL: the weight is used where it lies
    int64_t w_dim_stride, w_class_stride;
    uint16_t* w_planes;        // [P][classes][dim_pad]
    int64_t w_plane;
    void* dhidden;             // rows without a label are set to 0
    int64_t dhidden_stride;
    bool cleared;
    uint32_t* range;           // FP32: bits of the largest finite magnitude of the labelled rows of hidden, and of weight
};

// Bits of |x|; 0 for infinities, NaN and what counts as infinite: from 2^110 on a factor of 2^-80 is enough for a logit beyond
// kLogitBound, and the one use of such a weight is to take a class out.  It must not set the scale of all others.
__device__ __forceinline__ uint32_t finite_magnitude(float x) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    return b < ((110u + 127u) << 23) ? b : 0u;
}

// Lanes for a row of n values, four to a lane: a power of two, so that a warp takes several short rows at a time.
__device__ __forceinline__ int lanes_for(int n) {
    int g = 1;
    while (g < 32 && 4 * g < n) g *= 2;
    return g;
}

// Rows base(i) of n values, `stride` apart: the largest finite magnitude.  A thread has four rows in flight.
template <typename Base>
__device__ __forceinline__ void scan_rows(int64_t rows, int64_t n, int64_t stride, int lanes, int64_t w0, int64_t warps, Base base, uint32_t& m) {
    const int lane = threadIdx.x & 31, sub = lane & (lanes - 1), side = 32 / lanes;
    const int64_t step = warps * side;
    for (int64_t i = w0 * side + lane / lanes; i < rows; i += 4 * step) {
        const float* row[4];
        bool vec = stride == 1;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            row[k] = base(min(i + k * step, rows - 1));
            vec = vec && (reinterpret_cast<uintptr_t>(row[k]) & 15) == 0;
        }
        if (vec) {
            int64_t d = 4 * sub;
            for (; d + 4 <= n; d += 4 * lanes) {
                float4 v[4];
#pragma unroll
                for (int k = 0; k < 4; k++) v[k] = __ldg(reinterpret_cast<const float4*>(row[k] + d));
#pragma unroll
                for (int k = 0; k < 4; k++) m = max(m, max(max(finite_magnitude(v[k].x), finite_magnitude(v[k].y)), max(finite_magnitude(v[k].z), finite_magnitude(v[k].w))));
            }
            for (; d < n; d++)
#pragma unroll
                for (int k = 0; k < 4; k++) m = max(m, finite_magnitude(__ldg(row[k] + d)));
        } else {
#pragma unroll 2
            for (int64_t d = sub; d < n; d += lanes)
#pragma unroll
                for (int k = 0; k < 4; k++) m = max(m, finite_magnitude(__ldg(row[k] + d * stride)));
        }
    }
}
__device__ __forceinline__ void scan_weight(const XentPackArgs& p, int64_t w0, int64_t warps, uint32_t& m) {
    const float* weight = static_cast<const float*>(p.weight);
    if (p.w_class_stride == 1) {
        // stretches of 4096 of each row, the last one beginning so that it ends with the row
        const int64_t n = min((int64_t)p.classes, (int64_t)4096), parts = (p.classes + n - 1) / n;
        scan_rows(p.dim * parts, n, 1, 32, w0, warps, [&](int64_t i) {
            const int64_t d = i / parts;
            return weight + d * p.w_dim_stride + min((i - d * parts) * n, p.classes - n);
        }, m);
    } else {
        scan_rows(p.classes, p.dim, p.w_dim_stride, lanes_for(p.dim), w0, warps, [&](int64_t v) { return weight + v * p.w_class_stride; }, m);
    }
}

// The largest finite magnitudes of both operands (FP32 input) to p.range.  A maximum does not depend on the order.
__device__ __forceinline__ void find_range(const XentPackArgs& p, int64_t w0, int64_t warps) {
    const float* hidden = static_cast<const float*>(p.hidden);
    uint32_t most[2] = {0, 0};
    scan_rows(*p.count, p.dim, 1, lanes_for(p.dim), w0, warps, [&](int64_t i) { return hidden + p.row_of[i] * p.hidden_stride; }, most[0]);
    scan_weight(p, w0, warps, most[1]);
    block_max(most);
    if (threadIdx.x == 0) {
        if (most[0]) atomicMax(p.range, most[0]);
        if (most[1]) atomicMax(p.range + 1, most[1]);
    }
}
__global__ void __launch_bounds__(256) xent_range_kernel(const XentPackArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    find_range(p, grid_warp(), (int64_t)gridDim.x * 8);
}

// Zeros to the rows of dhidden, among the 32 from r0, that `clear` has a bit for; by a warp.
template <bool kFloat>
__device__ __forceinline__ void clear_rows(const XentPackArgs& p, int64_t r0, unsigned clear) {
    constexpr int kBytes = kFloat ? 4 : 2;
    if (!clear) return;
    const int lane = threadIdx.x & 31, bytes = p.dim * kBytes;
    const bool vec = (reinterpret_cast<uintptr_t>(p.dhidden) & 15) == 0 && p.dhidden_stride * kBytes % 16 == 0 && bytes % 16 == 0;
    char* to = static_cast<char*>(p.dhidden) + r0 * p.dhidden_stride * kBytes;
    const int pieces = vec ? bytes / 16 : p.dim;       // of a row
    int row = lane / pieces, piece = lane % pieces;    // lanes go through the rows' pieces one after the other
    const int rows_on = 32 / pieces, pieces_on = 32 % pieces;
    while (row < 32) {
        if (clear >> row & 1) {
            char* at = to + row * p.dhidden_stride * kBytes;
            if (vec) *reinterpret_cast<uint4*>(at + 16 * piece) = make_uint4(0u, 0u, 0u, 0u);
            else if constexpr (kFloat) reinterpret_cast<float*>(at)[piece] = 0.f;
            else reinterpret_cast<uint16_t*>(at)[piece] = 0;
        }
        row += rows_on;
        piece += pieces_on;
        if (piece >= pieces) { piece -= pieces; row++; }
    }
}

// What of many rows needs no numbers yet, in one pass: a block per chunk counts its labelled rows, takes their largest
// magnitude (FP32) and clears the other rows of dhidden; the blocks behind those take the weight's.
template <bool kFloat>
__global__ void __launch_bounds__(kXentCountThreads) xent_scan_kernel(const XentPackArgs p, int64_t chunk, int n_chunks, int32_t* __restrict__ counts,
                                                                      uint2* __restrict__ ranges) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t most[2] = {0, 0};
    if ((int)blockIdx.x < n_chunks) {
        __shared__ int sums[32];
        const float* hidden = static_cast<const float*>(p.hidden);
        const int64_t r1 = min(p.rows, (blockIdx.x + 1) * chunk);
        __shared__ uint8_t numbers[32][32];        // of a warp's labelled rows
        const int lanes = lanes_for(p.dim);
        int n = 0;
        for (int64_t rb = blockIdx.x * chunk + 32 * warp; rb < r1; rb += kXentCountThreads) {
            const int64_t r = rb + lane;
            const bool real = r < r1, mine = real && labelled(p.labels[r], p.classes);
            const unsigned have = __ballot_sync(0xffffffffu, mine), clear = __ballot_sync(0xffffffffu, real && !mine);
            n += __popc(have);
            if constexpr (kFloat) {
                if (mine) numbers[warp][__popc(have & ((1u << lane) - 1))] = (uint8_t)lane;
                __syncwarp();
                scan_rows(__popc(have), p.dim, 1, lanes, 0, 1, [&](int64_t i) { return hidden + (rb + numbers[warp][i]) * p.hidden_stride; }, most[0]);
                __syncwarp();
            }
            if (p.dhidden) clear_rows<kFloat>(p, rb, clear);
        }
        if (lane == 0) sums[warp] = n;
        __syncthreads();
        if (threadIdx.x < 32) {
            n = __reduce_add_sync(0xffffffffu, sums[threadIdx.x]);
            if (threadIdx.x == 0) counts[blockIdx.x] = n;
        }
    } else if constexpr (kFloat) {
        scan_weight(p, (int64_t)(blockIdx.x - n_chunks) * 32 + warp, (int64_t)(gridDim.x - n_chunks) * 32, most[1]);
    }
    if constexpr (kFloat) {
        block_max(most);
        if (threadIdx.x == 0) ranges[blockIdx.x] = make_uint2(most[0], most[1]);
    }
}

// hi and lo of a scaled float.  What is beyond the scale (2^15 and more: all that finite_magnitude leaves out) is infinite, and
// an infinity is all lo: of the three products of parts only the one with the other operand's hi is infinite then, none is 0 times
// infinity.  NaN is all hi.
__device__ __forceinline__ void split_half(float x, uint32_t& hi, uint32_t& lo) {
    const bool beyond = fabsf(x) >= 32768.f;
    const __half h = __float2half_rn(beyond ? 0.f : x);
    hi = __half_as_ushort(h);
    lo = __half_as_ushort(__float2half_rn(beyond ? copysignf(INFINITY, x) : (isnan(x) ? 0.f : x - __half2float(h))));
}

// One row of `dim` elements `stride` apart to the planes, by `lanes` lanes of which this is number `lane`; `src` NULL writes zeros.
template <bool kFloat>
__device__ __forceinline__ void pack_row(const void* src, int64_t stride, int dim, int dim_pad, uint16_t* to, int64_t plane, float scale, int lane, int lanes) {
    const bool vec = stride == 1 && (reinterpret_cast<uintptr_t>(src) & (kFloat ? 15 : 7)) == 0;
#pragma unroll 4
    for (int d = 4 * lane; d < dim_pad; d += 4 * lanes) {
        if constexpr (kFloat) {
            float x[4] = {0.f, 0.f, 0.f, 0.f};
            const float* f = static_cast<const float*>(src);
            if (src && vec && d + 4 <= dim) {
                const float4 v = __ldg(reinterpret_cast<const float4*>(f + d));
                x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
            } else if (src) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (d + j < dim) x[j] = __ldg(f + (d + j) * stride);
            }
            uint32_t h[4], l[4];
#pragma unroll
            for (int j = 0; j < 4; j++) split_half(scale * x[j], h[j], l[j]);
            *reinterpret_cast<uint2*>(to + d) = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
            *reinterpret_cast<uint2*>(to + plane + d) = make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16);
        } else {
            uint2 v = make_uint2(0u, 0u);
            const uint16_t* f = static_cast<const uint16_t*>(src);
            if (src && vec && d + 4 <= dim) {
                v = __ldg(reinterpret_cast<const uint2*>(f + d));
            } else if (src) {
                uint32_t x[4] = {0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (d + j < dim) x[j] = __ldg(f + (d + j) * stride);
                v = make_uint2(x[0] | x[1] << 16, x[2] | x[3] << 16);
            }
            *reinterpret_cast<uint2*>(to + d) = v;
        }
    }
}

template <bool kFloat>
__device__ __forceinline__ float plane_scale(const XentPackArgs& p, int operand) { return kFloat ? exp2f((float)(14 - plane_exponent(__ldcg(p.range + operand)))) : 1.f; }

// The labelled rows to their planes; zeros to dhidden's other rows, unless they have been cleared.
template <bool kFloat>
__device__ __forceinline__ void pack_hidden(const XentPackArgs& p, int64_t w0, int64_t warps) {
    constexpr int kBytes = kFloat ? 4 : 2;
    const int lane = threadIdx.x & 31, count = *p.count;
    const float h_scale = plane_scale<kFloat>(p, 0);
    // labelled rows, and zeros up to a whole tile
    const int64_t end = ((int64_t)count + kXentTileM - 1) / kXentTileM * kXentTileM;
    const int lanes = lanes_for(p.dim_pad), rows = 32 / lanes;
    const int64_t step = warps * rows;
    auto source = [&](int64_t i) -> const void* {
        return i < count ? static_cast<const char*>(p.hidden) + (int64_t)p.row_of[i] * p.hidden_stride * kBytes : nullptr;
    };
    if (!kFloat && p.dim % 8 == 0 && p.hidden_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(p.hidden) & 15) == 0 && end * (p.dim / 8) < ((int64_t)1 << 30)) {
        // nothing but a copy, in vectors of 16 bytes, four of a thread's in flight
        const int per_row = p.dim / 8, total = (int)end * per_row, threads = (int)warps * 32;
        for (int i0 = (int)w0 * 32 + lane; i0 < total; i0 += 4 * threads) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int i = min(i0 + k * threads, total - 1), row = i / per_row;
                const uint4* from = static_cast<const uint4*>(source(row));
                v[k] = from ? __ldg(from + (i - row * per_row)) : make_uint4(0u, 0u, 0u, 0u);
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i0 + k * threads < total) reinterpret_cast<uint4*>(p.h_planes)[i0 + k * threads] = v[k];
        }
    } else {
        for (int64_t i = w0 * rows + lane / lanes; i < end; i += 2 * step) {
            const void* a = source(i);
            const void* b = i + step < end ? source(i + step) : nullptr;
            pack_row<kFloat>(a, 1, p.dim, p.dim_pad, p.h_planes + i * p.dim_pad, p.h_plane, h_scale, lane & (lanes - 1), lanes);
            if (i + step < end)
                pack_row<kFloat>(b, 1, p.dim, p.dim_pad, p.h_planes + (i + step) * p.dim_pad, p.h_plane, h_scale, lane & (lanes - 1), lanes);
        }
    }
    if (p.dhidden && !p.cleared && count < p.rows) {
        for (int64_t r0 = 32 * w0; r0 < p.rows; r0 += 32 * warps) {
            const int64_t r = r0 + lane;
            clear_rows<kFloat>(p, r0, __ballot_sync(0xffffffffu, r < p.rows && !labelled(p.labels[min(r, p.rows - 1)], p.classes)));
        }
    }
}

// The weight to its planes, class by class.
template <bool kFloat>
__device__ __forceinline__ void pack_weight(const XentPackArgs& p, int64_t w0, int64_t warps) {
    const float w_scale = plane_scale<kFloat>(p, 1);
    const int lane = threadIdx.x & 31, lanes = lanes_for(p.dim_pad), rows = 32 / lanes;
    for (int64_t v = w0 * rows + lane / lanes; v < p.classes; v += warps * rows)
        pack_row<kFloat>(static_cast<const char*>(p.weight) + v * p.w_class_stride * (kFloat ? 4 : 2), p.w_dim_stride, p.dim, p.dim_pad,
                         p.w_planes + v * p.dim_pad, p.w_plane, w_scale, lane & (lanes - 1), lanes);
}

constexpr int kXentPackThreads = 256;

template <bool kFloat>
__global__ void __launch_bounds__(kXentPackThreads) xent_pack_kernel(const XentPackArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (kXentPackThreads / 32), w0 = grid_warp();
    pack_hidden<kFloat>(p, w0, warps);
    if (!p.weight) return;
    if (p.w_dim_stride == 1 || p.w_class_stride != 1) {
        pack_weight<kFloat>(p, w0, warps);
        return;
    }
    const float w_scale = plane_scale<kFloat>(p, 1);
    // classes are contiguous: tiles of 32 x 32 turned over in shared memory
    __shared__ uint32_t tile[kXentPackThreads / 32][32][33];
    uint32_t(*t)[33] = tile[threadIdx.x >> 5];
    const int64_t vt = (p.classes + 31) / 32, dt = (p.dim_pad + 31) / 32;
    for (int64_t i = w0; i < vt * dt; i += warps) {
        const int64_t v0 = i % vt * 32, d0 = i / vt * 32;
#pragma unroll 8
        for (int j = 0; j < 32; j++) {
            uint32_t x = 0;
            if (d0 + j < p.dim && v0 + lane < p.classes) {
                const int64_t at = (d0 + j) * p.w_dim_stride + v0 + lane;
                if constexpr (kFloat) x = __ldg(static_cast<const uint32_t*>(p.weight) + at);
                else x = __ldg(static_cast<const uint16_t*>(p.weight) + at);
            }
            t[j][lane] = x;
        }
        __syncwarp();
        // two classes at a time, two features a lane (dim_pad is even)
        const int d = 2 * (lane & 15);
#pragma unroll 4
        for (int j = lane >> 4; j < 32; j += 2) {
            if (v0 + j < p.classes && d0 + d < p.dim_pad) {
                uint16_t* to = p.w_planes + (v0 + j) * p.dim_pad + d0 + d;
                const uint32_t x = t[d][j], y = t[d + 1][j];
                if constexpr (kFloat) {
                    uint32_t h[2], l[2];
                    split_half(w_scale * __uint_as_float(x), h[0], l[0]);
                    split_half(w_scale * __uint_as_float(y), h[1], l[1]);
                    *reinterpret_cast<uint32_t*>(to) = h[0] | h[1] << 16;
                    *reinterpret_cast<uint32_t*>(to + p.w_plane) = l[0] | l[1] << 16;
                } else {
                    *reinterpret_cast<uint32_t*>(to) = x | y << 16;
                }
            }
        }
        __syncwarp();
    }
}

// All of the above by one block, for heads so small that launches count (kXentSmallRows, kXentSmallValues).
template <bool kFloat>
__global__ void __launch_bounds__(kXentCountThreads) xent_prepare_kernel(const XentNumberArgs n, const XentPackArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    number_rows(n);
    __syncthreads();
    const int64_t w0 = threadIdx.x >> 5, warps = kXentCountThreads / 32;
    if constexpr (kFloat) {
        find_range(p, w0, warps);
        __syncthreads();
    }
    pack_hidden<kFloat>(p, w0, warps);
    if (p.weight) pack_weight<kFloat>(p, w0, warps);
}

// ---- tiny heads --------------------------------------------------------------------------------------------
// The whole head by one cluster of eight blocks and without tensor cores, in one launch, for problems that are smaller than
// their launches.  A block takes an eighth of the rows: a warp several labelled rows at a time, its lanes along the classes
// for the logits and along the features for dH; then its share of dW, with the rows of a product dealt to 1024 / (dim
// classes) threads.  Labelled rows and G stay in shared memory; the first block adds up the others' dW and losses in their
// order.  2708 x 16 x 7 with one row in twenty labelled or all of them: 9.2 and 17.6 us, 33 and 36 by the
// general way; 512 x 32 x 32 18 and 34; where one lane would go through long rows (100 x 1000 x 1) 140 and 54.
struct XentTinyArgs {
    const void* hidden;
    int64_t hidden_stride;
    const void* weight;
    int64_t w_dim_stride, w_class_stride;
    void* dhidden;             // or NULL
    int64_t dhidden_stride;
    void* dweight;             // or NULL
    int64_t dw_dim_stride, dw_class_stride;
    int32_t dim;
    float* loss;
    int32_t reduction;
    float scale;
};
constexpr int kXentTinyBlocks = 8;
constexpr int kXentTinyProduct = 1024;                  // dim * classes, at most
constexpr int kXentTinyDim = 256, kXentTinyClasses = 4; // at most, at least: a lane takes a feature or a class at a time
constexpr int64_t kXentTinyWork = (int64_t)1 << 19;     // rows * dim * classes
constexpr int kXentTinyRows = kXentSmallRows / kXentTinyBlocks, kXentTinyFeatures = 32768, kXentTinyGrads = 8192;     // of a block
constexpr int kXentTinyBytes = 4 * (kXentTinyRows + kXentTinyFeatures + kXentTinyGrads + 2 * kXentTinyProduct + kXentCountThreads);

// Rows (of hidden, of the weight) apart by an odd number of values, so that lanes with different rows use different banks.
__host__ __device__ constexpr int tiny_pitch(int dim) { return dim | 1; }

template <typename T> __device__ __forceinline__ float load_float(const void* p, int64_t i) {
    if constexpr (std::is_same<T, float>::value) return static_cast<const float*>(p)[i];
    else if constexpr (std::is_same<T, __half>::value) return __half2float(static_cast<const __half*>(p)[i]);
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
template <typename T> __device__ __forceinline__ void store_float(void* p, int64_t i, float v) {
    if constexpr (std::is_same<T, float>::value) static_cast<float*>(p)[i] = v;
    else if constexpr (std::is_same<T, __half>::value) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float load_of_block(const float* own, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
                 : "=f"(v)
                 : "r"((uint32_t)__cvta_generic_to_shared(own)), "r"(rank)
                 : "memory");
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kXentCountThreads) __cluster_dims__(kXentTinyBlocks, 1, 1) xent_tiny_kernel(const XentNumberArgs n, const XentTinyArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    extern __shared__ float tiny_smem[];
    uint32_t* info = reinterpret_cast<uint32_t*>(tiny_smem);          // [labelled row of the block]: row of the block, label << 16
    float* h = tiny_smem + kXentTinyRows;
    float* g_all = h + kXentTinyFeatures;
    float* w = g_all + kXentTinyGrads;                                // [dim][classes]
    float* room = w + 2 * kXentTinyProduct;
    __shared__ int sums[32];
    __shared__ uint32_t have[kXentTinyRows / 32];                     // a bit for each of the block's rows: labelled
    __shared__ double losses_of[32];
    __shared__ float result[kXentTinyProduct + 2];                    // the block's dW, then its loss as the sum of two floats
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = p.dim, V = n.classes, rows = (int)n.rows, pitch = tiny_pitch(D), w_pitch = tiny_pitch(V);
    const int share = (rows + kXentTinyBlocks - 1) / kXentTinyBlocks, r0 = min(rows, (int)blockIdx.x * share), mine = min(share, rows - r0);

    // labels: how many there are, and the block's own
    int count_all = 0;
    for (int r = threadIdx.x; r < (rows + kXentCountThreads - 1) / kXentCountThreads * kXentCountThreads; r += kXentCountThreads)
        count_all += __syncthreads_count(r < rows && labelled(n.labels[min(r, rows - 1)], V));
    const int64_t label_of = (int)threadIdx.x < mine ? n.labels[r0 + threadIdx.x] : -1;
    const bool have_label = labelled(label_of, V);
    const unsigned ballot = __ballot_sync(0xffffffffu, have_label);
    if (lane == 0) {
        sums[warp] = __popc(ballot);
        if (warp < kXentTinyRows / 32) have[warp] = ballot;
    }
    for (int i = threadIdx.x; i < D * V; i += kXentCountThreads) {
        const int d = i / V, v = i - d * V;
        w[d * w_pitch + v] = load_float<T>(p.weight, d * p.w_dim_stride + v * p.w_class_stride);
    }
    __syncthreads();
    const int in_warp = sums[lane], count = __reduce_add_sync(0xffffffffu, in_warp);
    const int before = __reduce_add_sync(0xffffffffu, lane < warp ? in_warp : 0);
    if (have_label) info[before + __popc(ballot & ((1u << lane) - 1))] = threadIdx.x | (uint32_t)label_of << 16;
    else if ((int)threadIdx.x < mine && n.row_loss) n.row_loss[r0 + threadIdx.x] = 0.f;
    __syncthreads();
    if (p.dhidden) {
        // rows without a label, neighbouring threads at neighbouring addresses
        constexpr int kWide = 16 / (int)sizeof(T);
        const bool vec = (reinterpret_cast<uintptr_t>(p.dhidden) & 15) == 0 && p.dhidden_stride % kWide == 0 && D % kWide == 0;
        const int pieces = vec ? D / kWide : D;
        for (int i = threadIdx.x; i < mine * pieces; i += kXentCountThreads) {
            const int r = i / pieces, piece = i - r * pieces;
            if (have[r >> 5] >> (r & 31) & 1) continue;
            T* to = static_cast<T*>(p.dhidden) + (r0 + r) * p.dhidden_stride;
            if (vec) reinterpret_cast<uint4*>(to)[piece] = make_uint4(0u, 0u, 0u, 0u);
            else store_float<T>(to, piece, 0.f);
        }
    }
    for (int i = threadIdx.x; i < count * D; i += kXentCountThreads) {
        const int at = i / D, d = i - at * D;
        h[at * pitch + d] = load_float<T>(p.hidden, (int64_t)(r0 + (int)(info[at] & 0xffff)) * p.hidden_stride + d);
    }
    __syncthreads();

    // a warp takes as many rows at a time as have room for their classes side by side
    const float scale = xent_scale(p.scale, p.reduction == MASK_REDUCE_MEAN, count_all);
    int width = 1;
    while (width < 32 && width < V) width *= 2;
    const int sub = lane & (width - 1), at_once = 32 / width;
    double losses = 0.0;
    for (int i0 = warp * at_once; i0 < count; i0 += 32 * at_once) {
        const int i = i0 + lane / width;
        const bool live = i < count;
        const int row = live ? i : 0, label = (int)(info[row] >> 16);
        const float* x = h + row * pitch;
        float* g = g_all + row * V;
        float top = -INFINITY, picked = 0.f;
        for (int v = sub; v < V; v += width) {
            float s = 0.f;
#pragma unroll 8
            for (int d = 0; d < D; d++) s = fmaf(x[d], w[d * w_pitch + v], s);
            if (live) g[v] = s;
            top = fmaxf(top, s);
            if (v == label) picked = s;
        }
        for (int o = width / 2; o > 0; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            picked += __shfl_xor_sync(0xffffffffu, picked, o);
        }
        float sum = 0.f;
        for (int v = sub; v < V; v += width) sum += live ? fast_exp2((g[v] - top) * kLog2e) : 0.f;
        for (int o = width / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        const float loss = live ? kLn2 * fmaf(top - picked, kLog2e, log2f(sum)) : 0.f;
        if (sub == 0 && live) {
            losses += loss;
            if (n.row_loss) n.row_loss[r0 + (int)(info[row] & 0xffff)] = loss;
        }
        if (!p.dhidden && !p.dweight) continue;
        const float inv = 1.f / sum;
        for (int v = sub; v < V; v += width) {
            if (!live) continue;
            const float e = fast_exp2((g[v] - top) * kLog2e) * inv;
            g[v] = v == label ? e - 1.f : e;
        }
        __syncwarp();
        if (p.dhidden && live) {
            const int64_t to = (int64_t)(r0 + (int)(info[row] & 0xffff)) * p.dhidden_stride;
            for (int d = sub; d < D; d += width) {
                float s = 0.f;
#pragma unroll 8
                for (int v = 0; v < V; v++) s = fmaf(g[v], w[d * w_pitch + v], s);
                store_float<T>(p.dhidden, to + d, scale * s);
            }
        }
        __syncwarp();
    }
    for (int o = 16; o > 0; o >>= 1) losses += __shfl_xor_sync(0xffffffffu, losses, o);
    if (lane == 0) losses_of[warp] = losses;
    __syncthreads();
    if (threadIdx.x == 0) {
        double s = 0.0;
        for (int i = 0; i < 32; i++) s += losses_of[i];
        result[kXentTinyProduct] = (float)s;
        result[kXentTinyProduct + 1] = (float)(s - (double)(float)s);
    }
    const int shares = kXentCountThreads / (D * V), part = threadIdx.x / (D * V), pair = threadIdx.x - part * (D * V);
    if (p.dweight) {
        const int d = pair / V, v = pair - d * V;
        float s = 0.f;
        if (part < shares) {
#pragma unroll 4
            for (int i = part; i < count; i += shares) s = fmaf(g_all[i * V + v], h[i * pitch + d], s);
        }
        room[threadIdx.x] = s;
        __syncthreads();
        if (part == 0) {
            for (int i = 1; i < shares; i++) s += room[i * D * V + pair];
            result[pair] = s;
        }
    }
    cluster_sync();
    if (blockIdx.x == 0) {
        if (p.dweight && part == 0) {
            float s = 0.f;
#pragma unroll
            for (uint32_t r = 0; r < kXentTinyBlocks; r++) s += load_of_block(result + pair, r);
            const int d = pair / V, v = pair - d * V;
            store_float<T>(p.dweight, d * p.dw_dim_stride + v * p.dw_class_stride, scale * s);
        }
        if (threadIdx.x == 0 && !n.row_loss) {
            double s = 0.0;
            for (uint32_t r = 0; r < kXentTinyBlocks; r++)
                s += (double)load_of_block(result + kXentTinyProduct, r) + (double)load_of_block(result + kXentTinyProduct + 1, r);
            *p.loss = count_all == 0 ? 0.f : (float)(p.reduction == MASK_REDUCE_MEAN ? s / count_all : s);
        }
    }
    cluster_sync();                   // the blocks' results have been read
}

template <typename T>
static int launch_xent_tiny(const XentNumberArgs& n, const XentTinyArgs& t, cudaStream_t st) {
    static std::atomic<uint64_t> done{0};
    const int rc = opt_in_shared_memory(reinterpret_cast<const void*>(xent_tiny_kernel<T>), kXentTinyBytes, done);
    if (rc != MASK_OK) return rc;
    return launch_overlapped(xent_tiny_kernel<T>, dim3(kXentTinyBlocks), kXentCountThreads, kXentTinyBytes, st, n, t);
}

// ---- joining -----------------------------------------------------------------------------------------------
// Log sums and losses of the rows from the parts of the classes: a block takes 1024 / shares rows, a warp 32 of them, and
// `shares` (a power of two) threads a row, whose shares of the parts are joined in their order.
__global__ void __launch_bounds__(1024) xent_join_kernel(const XentArgs p, int parts, int shares) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    __shared__ float2 room[1024];
    const int count = *p.count, rows = 1024 / shares, share = threadIdx.x / rows, at = threadIdx.x & (rows - 1);
    const float f = logit_factor(p.range), rest = logit_rest(p.range);
    const bool lost = *p.status != 0;
    for (int64_t r0 = rows * (int64_t)blockIdx.x; r0 < count; r0 += rows * (int64_t)gridDim.x) {
        const int64_t r = r0 + at;
        float top = -INFINITY, sum = 0.f;
        auto join = [&](float2 s) {
            const float now = fmaxf(top, s.x), base = exponent_base(now, f);
            sum = sum * rebase(top, f, base) + s.y * rebase(s.x, f, base);
            top = now;
        };
        if (r < count) {
#pragma unroll 4
            for (int i = share; i < parts; i += shares) join(p.stats[(int64_t)i * p.rows_pad + r]);
        }
        if (shares > 1) {
            __syncthreads();
            room[threadIdx.x] = make_float2(top, sum);
            __syncthreads();
        }
        if (share > 0) continue;
        for (int i = 1; i < shares; i++) join(room[i * rows + at]);
        float loss = 0.f;
        if (r < count) {
            const float base = exponent_base(top, f);
            sum = bounded_sum(sum, base);
            const float log_sum = log2f(sum);
            p.shift[r] = p.range ? base : __fadd_ru(base, log_sum);
            p.factor[r] = (float)(1 << kGradExponent) / sum;
            loss = lost ? NAN : kLn2 * (fmaf(-p.label_logit[r] * rest, f, base) + log_sum);
            if (p.row_loss) p.row_loss[p.row_of[r]] = loss;
        }
        const bool any = __any_sync(0xffffffffu, r < count);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) loss += __shfl_xor_sync(0xffffffffu, loss, o);
        if ((threadIdx.x & 31) == 0 && any) p.warp_loss[r >> 5] = loss;
    }
}

// Parts of a product summed up, scaled and written where the caller wants them.  A block takes 256 / shares vectors of four
// values, neighbouring threads along the axis that is contiguous in the output, and `shares` threads a vector (many parts of
// a small product), whose sums are added in their order.
struct XentReduceArgs {
    const float* part;
    int64_t part_rows;
    int32_t part_ld, splits, shares;
    int32_t m, n;
    const int32_t* count;      // labelled rows (for the scale)
    int32_t m_is_count;        // as many rows as are labelled, each to row_of[m]
    const int32_t* row_of;
    void* out;
    int64_t out_m, out_n, m0;
    int32_t out_type;
    float scale;
    int32_t mean, operand;
    const uint32_t* range;
};

__device__ __forceinline__ void reduce_parts(const XentReduceArgs& p) {
    const int count = *p.count;
    const int64_t m_end = p.m_is_count ? count : p.m, n_vec = (p.n + 3) / 4;
    const ProductScale scale = product_scale(p.scale, p.mean, count, p.range, p.operand, p.out_type == MASK_F16);
    const bool m_fast = p.out_m == 1 && p.out_n != 1;
    __shared__ float4 room[256];
    const int per_block = 256 / p.shares, share = threadIdx.x / per_block;
    const int64_t most = m_end * n_vec;
    for (int64_t i0 = (int64_t)blockIdx.x * per_block; i0 < most; i0 += (int64_t)gridDim.x * per_block) {
        const int64_t i = i0 + threadIdx.x % per_block;
        const int64_t m = m_fast ? i % m_end : i / n_vec, n = 4 * (m_fast ? i / m_end : i % n_vec);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < most) {
#pragma unroll 4
            for (int s = share; s < p.splits; s += p.shares) {
                const float4 v = *reinterpret_cast<const float4*>(p.part + (s * p.part_rows + m) * p.part_ld + n);
                a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
            }
        }
        if (p.shares > 1) {
            __syncthreads();
            room[threadIdx.x] = a;
            __syncthreads();
            if (share == 0) {
                for (int s = 1; s < p.shares; s++) {
                    const float4 v = room[s * per_block + threadIdx.x];
                    a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
                }
            }
        }
        if (share > 0 || i >= most) continue;
        const float v[4] = {scale(a.x), scale(a.y), scale(a.z), scale(a.w)};
        const int64_t at = (p.m_is_count ? (int64_t)p.row_of[m] : p.m0 + m) * p.out_m + n * p.out_n;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (n + j >= p.n) break;
            if (p.out_type == MASK_F32) static_cast<float*>(p.out)[at + j * p.out_n] = v[j];
            else if (p.out_type == MASK_F16) static_cast<__half*>(p.out)[at + j * p.out_n] = __float2half_rn(v[j]);
            else static_cast<__nv_bfloat16*>(p.out)[at + j * p.out_n] = __float2bfloat16_rn(v[j]);
        }
    }
}

struct XentLossArgs {
    const int32_t* count;
    const float* warp_loss;
    const int32_t* status;
    float* loss;               // NULL: not now
    int64_t rows;
    int32_t reduction;
};

// The loss of all rows, in a fixed order and 64 bits; NaN where a kernel gave up on a wait.
__device__ __forceinline__ void sum_losses(const XentLossArgs& p) {
    const int count = *p.count;
    if (*p.status) {
        const int64_t n = p.reduction == MASK_REDUCE_NONE ? p.rows : 1;
        for (int64_t r = threadIdx.x; r < n; r += 256) p.loss[r] = NAN;
        return;
    }
    if (p.reduction == MASK_REDUCE_NONE) return;
    __shared__ double sums[8];
    double sum = 0.0;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < ((int64_t)count + 31) / 32; i += 256) sum += p.warp_loss[i];
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0;
        for (int i = 0; i < 8; i++) sum += sums[i];
        *p.loss = count == 0 ? 0.f : (float)(p.reduction == MASK_REDUCE_MEAN ? sum / count : sum);
    }
}

// What is left of a call (grid.y: dweight's parts, dhidden's); a block that has no other part of it sums the losses.
__global__ void __launch_bounds__(256) xent_finish_kernel(const XentReduceArgs dw, const XentReduceArgs dh, const XentLossArgs loss) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    if (blockIdx.y == 2) {
        if (blockIdx.x == 0 && loss.loss) sum_losses(loss);
        return;
    }
    if (blockIdx.y == 0 ? dw.part != nullptr : dh.part != nullptr) {
        if (blockIdx.y == 0) reduce_parts(dw);
        else reduce_parts(dh);
    }
}

// ---- plan of a call ---------------------------------------------------------------------------------------
static int64_t round_up(int64_t x, int64_t m) { return (x + m - 1) / m * m; }

struct XentPlan {
    int planes, dim_pad;
    int64_t rows_pad, chunk;
    int n_chunks, weight_blocks;
    bool grads, one_pass, pack_weight, small, tiny;
    int bn_logits, bn_dim;
    int stats_splits, stats_parts;       // parts of the classes' tiles, and numbers a row gets from them
    int piece, n_pieces;                 // classes of a piece (a multiple of 256 unless one tile holds all), pieces
    int g_ld;
    int dh_splits, dw_splits;
    int segment;                         // blocks of their contraction that an accumulator takes (16-bit operands)
    bool dh_parts, dw_parts;
    int64_t part_dh_rows, part_dw_rows;
    int part_ld;
    // byte offsets into the scratch
    size_t counts, ranges, row_of, label, total, stats, label_logit, shift, factor, warp_loss, h_planes, w_planes, g, part_dh, part_dw, bytes;
};

// Blocks that share a tile of `bn` columns of a product with so many rows.  Pairs load a third less (dH of 16384 x 16384 x 512:
// 171 us instead of 195), but wait for one another's epilogue: logits, whose epilogue takes as long as contracting 500
// (16384 x 256 x 16384: 110 and 139 us a block alone, 144 and 182 in pairs; over 512 they take the same), are left to pairs only
// where more than that is contracted.
static int tile_blocks(int bn, int64_t rows, int contracted = 1 << 30) { return bn == 256 && rows > kXentTileM && contracted > 512 ? 2 : 1; }

// Parts to cut each tile's `units` of work into (tiles: those of `rows` rows, `others` of them side by side), so that they
// fill the SMs: the fewest rounds of the longest part, `rounds` at most.  A part costs two units beside its own (the
// accumulator's way out).
static int best_splits(int64_t rows, int cg, int64_t others, int64_t units, int rounds) {
    const int64_t sms = sm_count() / cg, tiles = (rows + cg * kXentTileM - 1) / (cg * kXentTileM) * others;
    int64_t best = 1, best_cost = INT64_MAX;
    const int64_t most = std::min<int64_t>(units, std::max<int64_t>(1, rounds * sms / std::max<int64_t>(tiles, 1)));
    for (int64_t s = 1; s <= most; s++) {
        const int64_t cost = (tiles * s + sms - 1) / sms * ((units + s - 1) / s + 2);
        if (cost < best_cost) { best_cost = cost; best = s; }
    }
    return (int)best;
}

static int tile_width(int n) {
    if (n <= 64) return 64;
    return n <= 128 || round_up(n, 128) < round_up(n, 256) ? 128 : 256;
}

// Whether rows of a result may be written in vectors of eight values (32 bytes of FP32, 16 of the others).  A product whose
// rows may not be leaves its tiles in parts, in scratch, which are then written by neighbouring threads: a thread per row
// costs a request for every value.
static bool vector_rows(const void* data, int64_t stride, int dtype) {
    return stride % 8 == 0 && (reinterpret_cast<uintptr_t>(data) & (dtype == MASK_F32 ? 31 : 15)) == 0;
}

static XentPlan plan_xent(const mask_head& h) {
    XentPlan p = {};
    p.planes = h.dtype == MASK_F32 ? 2 : 1;
    p.dim_pad = (int)round_up(h.dim, 8);
    p.rows_pad = round_up(std::max<int64_t>(h.rows, 1), kXentTileM);
    p.chunk = std::max<int64_t>(kXentCountThreads, round_up((h.rows + 2047) / 2048, kXentCountThreads));
    p.n_chunks = (int)std::max<int64_t>(1, (h.rows + p.chunk - 1) / p.chunk);
    p.grads = h.d_dhidden || h.d_dweight;
    p.pack_weight = p.planes == 2 || h.weight_dim_stride != 1 || h.weight_class_stride % 8 || h.weight_class_stride < h.dim ||
                    (reinterpret_cast<uintptr_t>(h.d_weight) & 15);
    p.small = h.rows <= kXentSmallRows && h.rows * h.dim + (p.pack_weight ? (int64_t)h.dim * h.classes : 0) <= kXentSmallValues;
    if (p.small) p.chunk = kXentSmallRows, p.n_chunks = 1;
    p.bn_logits = h.classes <= 64 ? 64 : (h.classes <= 128 ? 128 : 256);
    p.bn_dim = tile_width(h.dim);
    // one tile of all classes: 256 columns, with two planes of G in shared memory 128
    p.one_pass = p.grads && h.classes <= (p.planes == 2 ? 128 : 256);
    p.stats_splits = p.one_pass ? 1 : best_splits(p.rows_pad, tile_blocks(p.bn_logits, p.rows_pad, h.dim), 1, (h.classes + p.bn_logits - 1) / p.bn_logits, 16);
    p.stats_parts = p.stats_splits * xent_parts(p.bn_logits, p.planes, true);
    if (p.grads) {
        if (p.one_pass) {
            p.piece = h.classes;
            p.g_ld = p.bn_logits;
        } else {
            const int64_t fit = (int64_t)(kXentPieceBytes / (size_t)(2 * p.planes * p.rows_pad)) / 256 * 256;
            // as few pieces as fit, of equal length
            const int64_t pieces = (h.classes + std::max<int64_t>(fit, 256) - 1) / std::max<int64_t>(fit, 256);
            p.piece = p.g_ld = (int)round_up((h.classes + pieces - 1) / pieces, 256);
        }
        p.n_pieces = (int)((h.classes + (int64_t)p.piece - 1) / p.piece);
        const int64_t n_tiles = (h.dim + p.bn_dim - 1) / p.bn_dim;
        p.part_ld = (int)(n_tiles * p.bn_dim);
        p.segment = h.dtype == MASK_F16 ? kXentLongSegmentF16 : kXentLongSegmentBf16;
        // contractions of several segments are added up in the parts
        auto segmented = [&](int64_t contracted, int splits) {
            const int64_t units = (contracted + kXentTileK - 1) / kXentTileK;
            return p.planes == 1 && (units + splits - 1) / splits > p.segment;
        };
        if (h.d_dhidden) {
            p.dh_splits = best_splits(p.rows_pad, tile_blocks(p.bn_dim, p.rows_pad), n_tiles, (p.piece + kXentTileK - 1) / kXentTileK, 4);
            p.dh_parts = p.dh_splits > 1 || p.n_pieces > 1 || segmented(p.piece, p.dh_splits) || !vector_rows(h.d_dhidden, h.dhidden_stride, h.dtype);
            p.part_dh_rows = p.rows_pad;
        }
        if (h.d_dweight) {
            p.dw_splits = best_splits(p.piece, tile_blocks(p.bn_dim, p.piece), n_tiles, (p.rows_pad + kXentTileK - 1) / kXentTileK, 4);
            p.dw_parts = p.dw_splits > 1 || segmented(p.rows_pad, p.dw_splits) || (h.dweight_dim_stride == 1 && h.dweight_class_stride != 1 && !vector_rows(h.d_dweight, h.dweight_class_stride, h.dtype));
            p.part_dw_rows = round_up(p.piece, kXentTileM);
        }
    }
    const int64_t share = (h.rows + kXentTinyBlocks - 1) / kXentTinyBlocks;
    p.tiny = h.rows <= kXentSmallRows && h.dim <= kXentTinyDim && h.classes >= kXentTinyClasses && (int64_t)h.dim * h.classes <= kXentTinyProduct && h.rows * h.dim * h.classes <= kXentTinyWork &&
             share * tiny_pitch(h.dim) <= kXentTinyFeatures && share * h.classes <= kXentTinyGrads;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    const size_t rp = (size_t)p.rows_pad;
    p.total = take(256);
    p.counts = take(4 * (size_t)p.n_chunks);
    p.weight_blocks = (int)std::min<int64_t>(sm_count(), ((int64_t)h.dim * h.classes + 32767) / 32768);
    p.ranges = take(8 * (size_t)(p.n_chunks + p.weight_blocks));
    p.row_of = take(4 * rp);
    p.label = take(4 * rp);
    if (p.tiny) {
        p.chunk = kXentSmallRows;
        p.n_chunks = 1;
        p.bytes = at;
        return p;
    }
    p.stats = p.one_pass ? 0 : take(8 * rp * p.stats_parts);
    p.label_logit = take(4 * rp);
    p.shift = take(4 * rp);
    p.factor = take(4 * rp);
    p.warp_loss = take(rp / 8);
    p.h_planes = take(2 * (size_t)p.planes * rp * p.dim_pad);
    p.w_planes = p.pack_weight ? take(2 * (size_t)p.planes * h.classes * p.dim_pad) : 0;
    if (p.grads) {
        p.g = take(2 * (size_t)p.planes * rp * p.g_ld);
        if (p.dh_parts) p.part_dh = take(4 * (size_t)p.dh_splits * p.part_dh_rows * p.part_ld);
        if (p.dw_parts) p.part_dw = take(4 * (size_t)p.dw_splits * p.part_dw_rows * p.part_ld);
    }
    p.bytes = at;
    return p;
}

// Planes of 16-bit values as a tensor [planes][rows][columns], `ld` elements from row to row.
static int plane_map(CUtensorMap* map, const void* data, int64_t cols, int64_t rows, int planes, int64_t ld, int64_t plane, int box_cols, int box_rows) {
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return fail(MASK_ERR_CUDA, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, (cuuint64_t)plane * 2};
    const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(data), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           box_cols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with code %d (%lld x %lld, pitch %lld)", (int)r, (long long)rows, (long long)cols, (long long)ld);
        return MASK_ERR_CUDA;
    }
    return MASK_OK;
}

template <int BN, int P, int MODE, int CG>
static int launch_xent_gemm_as(const XentArgs& a, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mg, int64_t items, cudaStream_t st) {
    using L = XentLayout<BN, P, MODE, CG>;
    static std::atomic<uint64_t> done{0};
    const int rc = opt_in_shared_memory(reinterpret_cast<const void*>(xent_gemm_kernel<BN, P, MODE, CG>), L::kDynamicBytes, done);
    if (rc != MASK_OK) return rc;
    const unsigned grid = CG * (unsigned)std::max<int64_t>(1, std::min<int64_t>(items, sm_count() / CG));
    return launch_overlapped_clusters(CG, xent_gemm_kernel<BN, P, MODE, CG>, dim3(grid), L::kThreads, L::kDynamicBytes, st, a, ma, mb, mg);
}

template <int MODE, int P>
static int launch_xent_gemm_planes(int bn, int cg, const XentArgs& a, const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mg, int64_t items,
                                   cudaStream_t st) {
    if (bn == 64) return launch_xent_gemm_as<64, P, MODE, 1>(a, ma, mb, mg, items, st);
    if (bn == 128) return launch_xent_gemm_as<128, P, MODE, 1>(a, ma, mb, mg, items, st);
    if constexpr (P == 2 && MODE == kXentGradOne) return fail(MASK_ERR_INVALID_ARGUMENT, "no such kernel");
    else if (cg == 1) return launch_xent_gemm_as<256, P, MODE, 1>(a, ma, mb, mg, items, st);
    else return launch_xent_gemm_as<256, P, MODE, 2>(a, ma, mb, mg, items, st);
}

template <int MODE>
static int launch_xent_gemm(int bn, int planes, const XentArgs& a, int64_t rows, int64_t parts, const CUtensorMap& ma, const CUtensorMap& mb,
                            const CUtensorMap& mg, cudaStream_t st) {
    const int cg = MODE <= kXentGradOne ? tile_blocks(bn, rows, a.dim) : tile_blocks(bn, rows);
    const int64_t items = (rows + cg * kXentTileM - 1) / (cg * kXentTileM) * parts;
    return planes == 1 ? launch_xent_gemm_planes<MODE, 1>(bn, cg, a, ma, mb, mg, items, st) : launch_xent_gemm_planes<MODE, 2>(bn, cg, a, ma, mb, mg, items, st);
}

// Blocks for a product's parts (0: it has none), `rows` of them at most, and the threads that share a vector.
static int64_t share_parts(XentReduceArgs& r, int64_t rows) {
    if (!r.part) return 0;
    const int64_t vectors = rows * ((r.n + 3) / 4);
    // 16 parts or more and not enough vectors for two blocks an SM: up to 32 threads a vector
    r.shares = 1;
    while (r.shares < 32 && 8 * r.shares < r.splits && vectors * r.shares < 512 * (int64_t)sm_count()) r.shares *= 2;
    return std::min<int64_t>((vectors * r.shares + 255) / 256, 8 * (int64_t)sm_count());
}
static int launch_xent_finish(XentReduceArgs dw, int64_t dw_rows, XentReduceArgs dh, int64_t dh_rows, const XentLossArgs& loss, cudaStream_t st) {
    const int64_t blocks = std::max<int64_t>(1, std::max(share_parts(dw, dw_rows), share_parts(dh, dh_rows)));
    return launch_overlapped(xent_finish_kernel, dim3((unsigned)blocks, 3), 256, 0, st, dw, dh, loss);
}

static const char* refuse_head(const mask_head* h) {
    if (!h) return "head is NULL";
    if (h->dtype < MASK_F32 || h->dtype > MASK_F16) return "dtype must be MASK_F32, MASK_BF16 or MASK_F16";
    if (h->reduction < MASK_REDUCE_NONE || h->reduction > MASK_REDUCE_SUM) return "reduction must be MASK_REDUCE_NONE, _MEAN or _SUM";
    constexpr int64_t most = ((int64_t)1 << 31) - 256;
    if (h->rows < 0 || h->rows >= most) return "rows out of range";
    if (h->dim < 1 || h->dim > (1 << 20)) return "dim must be 1 to 2^20";
    if (h->classes < 1 || h->classes >= most) return "classes must be at least 1 and below 2^31 - 256";
    if (h->hidden_stride < 0 || h->weight_dim_stride < 0 || h->weight_class_stride < 0 || h->dhidden_stride < 0 || h->dweight_dim_stride < 0 ||
        h->dweight_class_stride < 0)
        return "strides must not be negative";
    if (!h->d_weight || (h->rows > 0 && (!h->d_hidden || !h->d_labels))) return "an operand is NULL";
    if (!h->d_loss && (h->reduction != MASK_REDUCE_NONE || h->rows > 0)) return "loss is NULL";
    const uintptr_t element = h->dtype == MASK_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(h->d_hidden) | reinterpret_cast<uintptr_t>(h->d_weight) | reinterpret_cast<uintptr_t>(h->d_dhidden) |
         reinterpret_cast<uintptr_t>(h->d_dweight)) & element)
        return "an operand is not aligned to its type";
    if ((reinterpret_cast<uintptr_t>(h->d_loss) & 3) || (reinterpret_cast<uintptr_t>(h->d_labels) & 7)) return "loss or labels are not aligned to their type";
    if (h->d_dhidden && h->rows > 1 && h->dhidden_stride < h->dim) return "rows of dhidden overlap";
    return nullptr;
}

static int run_xent(const mask_head& h, const XentPlan& plan, char* scratch, cudaStream_t st) {
    auto at = [&](size_t offset) { return scratch + offset; };
    int32_t* total = reinterpret_cast<int32_t*>(at(plan.total));
    int32_t* row_of = reinterpret_cast<int32_t*>(at(plan.row_of));
    int32_t* label = reinterpret_cast<int32_t*>(at(plan.label));
    int32_t* counts = reinterpret_cast<int32_t*>(at(plan.counts));
    uint32_t* range = reinterpret_cast<uint32_t*>(total + 2);
    float* row_loss = h.reduction == MASK_REDUCE_NONE ? h.d_loss : nullptr;
    const int P = plan.planes;
    const int64_t rp = plan.rows_pad;

    int rc = MASK_OK;
    XentNumberArgs number = {h.d_labels, h.rows, plan.chunk, h.classes, counts, row_of, label, total, total + 1, range, nullptr, 0, row_loss};
    if (plan.tiny) {
        const XentTinyArgs t = {h.d_hidden, h.hidden_stride, h.d_weight, h.weight_dim_stride, h.weight_class_stride, h.d_dhidden, h.dhidden_stride, h.d_dweight,
                                h.dweight_dim_stride, h.dweight_class_stride, h.dim, h.d_loss, h.reduction, h.grad_scale};
        if (h.dtype == MASK_F32) return launch_xent_tiny<float>(number, t, st);
        if (h.dtype == MASK_F16) return launch_xent_tiny<__half>(number, t, st);
        return launch_xent_tiny<__nv_bfloat16>(number, t, st);
    }

    XentPackArgs pk = {};
    pk.dim = h.dim; pk.dim_pad = plan.dim_pad; pk.classes = h.classes; pk.rows = h.rows;
    pk.count = total; pk.row_of = row_of; pk.labels = h.d_labels;
    pk.hidden = h.d_hidden; pk.hidden_stride = h.hidden_stride;
    pk.h_planes = reinterpret_cast<uint16_t*>(at(plan.h_planes)); pk.h_plane = rp * plan.dim_pad;
    pk.dhidden = h.d_dhidden; pk.dhidden_stride = h.dhidden_stride;
    if (plan.pack_weight) {
        pk.weight = h.d_weight; pk.w_dim_stride = h.weight_dim_stride; pk.w_class_stride = h.weight_class_stride;
        pk.w_planes = reinterpret_cast<uint16_t*>(at(plan.w_planes)); pk.w_plane = (int64_t)h.classes * plan.dim_pad;
    }
    pk.range = range;
    if (plan.small) {
        if (h.dtype == MASK_F32) rc = launch_overlapped(xent_prepare_kernel<true>, dim3(1), kXentCountThreads, 0, st, number, pk);
        else rc = launch_overlapped(xent_prepare_kernel<false>, dim3(1), kXentCountThreads, 0, st, number, pk);
        if (rc) return rc;
    } else {
        const dim3 chunks((unsigned)plan.n_chunks);
        if (plan.n_chunks > 1) {
            // a block per chunk, and for the weight at most one an SM
            const int blocks = plan.n_chunks + (P == 2 ? plan.weight_blocks : 0);
            uint2* ranges = reinterpret_cast<uint2*>(at(plan.ranges));
            if (P == 2) rc = launch_overlapped(xent_scan_kernel<true>, dim3((unsigned)blocks), kXentCountThreads, 0, st, pk, plan.chunk, plan.n_chunks, counts, ranges);
            else rc = launch_overlapped(xent_scan_kernel<false>, dim3((unsigned)blocks), kXentCountThreads, 0, st, pk, plan.chunk, plan.n_chunks, counts, ranges);
            if (rc) return rc;
            pk.cleared = true;
            if (P == 2) number.ranges = ranges, number.n_ranges = blocks;
        }
        if ((rc = launch_overlapped(xent_number_kernel, chunks, kXentCountThreads, 0, st, number))) return rc;
        const int64_t pack_rows = rp + (plan.pack_weight ? h.classes : 0);
        const dim3 pack_grid((unsigned)std::min<int64_t>((pack_rows + 7) / 8, 8 * (int64_t)sm_count()));
        if (P == 2) {
            if (plan.n_chunks == 1 && (rc = launch_overlapped(xent_range_kernel, pack_grid, 256, 0, st, pk))) return rc;
            rc = launch_overlapped(xent_pack_kernel<true>, pack_grid, kXentPackThreads, 0, st, pk);
        } else {
            rc = launch_overlapped(xent_pack_kernel<false>, pack_grid, kXentPackThreads, 0, st, pk);
        }
        if (rc) return rc;
    }

    const void* w_data = plan.pack_weight ? (const void*)pk.w_planes : h.d_weight;
    const int64_t w_ld = plan.pack_weight ? plan.dim_pad : h.weight_class_stride, w_plane = plan.pack_weight ? pk.w_plane : w_ld * h.classes;
    const int w_cols = plan.pack_weight ? plan.dim_pad : h.dim;
    CUtensorMap h_k, w_k, none = {};     // K-major, contracted over dim
    if ((rc = plane_map(&h_k, pk.h_planes, plan.dim_pad, rp, P, plan.dim_pad, pk.h_plane, 64, kXentTileM))) return rc;
    if ((rc = plane_map(&w_k, w_data, w_cols, h.classes, P, w_ld, w_plane, 64, plan.bn_logits / tile_blocks(plan.bn_logits, rp, h.dim)))) return rc;

    XentArgs a = {};
    a.count = total; a.status = total + 1;
    a.classes = h.classes; a.dim = h.dim; a.v0 = 0; a.vc = h.classes;
    a.rows_pad = (int32_t)rp; a.half_type = h.dtype != MASK_BF16; a.range = P == 2 ? range : nullptr;
    a.label = label; a.row_of = row_of; a.row_loss = row_loss;
    a.stats = reinterpret_cast<float2*>(at(plan.stats));
    a.label_logit = reinterpret_cast<float*>(at(plan.label_logit));
    a.shift = reinterpret_cast<float*>(at(plan.shift));
    a.factor = reinterpret_cast<float*>(at(plan.factor));
    a.warp_loss = reinterpret_cast<float*>(at(plan.warp_loss));
    a.segment = plan.segment; a.scale = h.grad_scale; a.mean = h.reduction == MASK_REDUCE_MEAN;
    a.out_type = h.dtype;

    if (!plan.one_pass) {
        a.splits = plan.stats_splits;
        if ((rc = launch_xent_gemm<kXentStats>(plan.bn_logits, P, a, rp, a.splits, h_k, w_k, none, st))) return rc;
        int shares = 1;
        while (shares < 32 && 8 * shares < plan.stats_parts) shares *= 2;
        const int64_t blocks = std::min<int64_t>((rp * shares + 1023) / 1024, 2 * (int64_t)sm_count());
        if ((rc = launch_overlapped(xent_join_kernel, dim3((unsigned)blocks), 1024, 0, st, a, plan.stats_parts, shares))) return rc;
    }
    XentReduceArgs dw = {}, dh = {};
    if (plan.grads) {
        char* g = at(plan.g);
        const int64_t g_plane = rp * plan.g_ld;
        CUtensorMap g_st, g_k, g_mn, w_mn, h_mn;
        if ((rc = plane_map(&g_st, g, plan.g_ld, rp, P, plan.g_ld, g_plane, xent_box(plan.bn_logits, P), 32))) return rc;
        if ((rc = plane_map(&g_k, g, plan.g_ld, rp, P, plan.g_ld, g_plane, 64, kXentTileM))) return rc;
        if ((rc = plane_map(&g_mn, g, plan.g_ld, rp, P, plan.g_ld, g_plane, 64, 64))) return rc;
        if ((rc = plane_map(&w_mn, w_data, w_cols, h.classes, P, w_ld, w_plane, 64, 64))) return rc;
        if ((rc = plane_map(&h_mn, pk.h_planes, plan.dim_pad, rp, P, plan.dim_pad, pk.h_plane, 64, 64))) return rc;
        const int64_t n_tiles = plan.part_ld / plan.bn_dim;
        XentReduceArgs r = {};
        r.part_ld = plan.part_ld; r.n = h.dim; r.count = total; r.row_of = row_of; r.out_type = h.dtype; r.scale = a.scale; r.mean = a.mean; r.range = a.range;
        for (int piece = 0; piece < plan.n_pieces; piece++) {
            a.v0 = piece * plan.piece;
            a.vc = std::min(plan.piece, h.classes - a.v0);
            const int64_t v_tiles = (a.vc + plan.bn_logits - 1) / plan.bn_logits;
            if (plan.one_pass) rc = launch_xent_gemm<kXentGradOne>(plan.bn_logits, P, a, rp, 1, h_k, w_k, g_st, st);
            else rc = launch_xent_gemm<kXentGrad>(plan.bn_logits, P, a, rp, v_tiles, h_k, w_k, g_st, st);
            if (rc) return rc;
            if (h.d_dhidden) {
                XentArgs b = a;
                b.splits = plan.dh_splits;
                b.store = !plan.dh_parts ? kXentFinal : (piece == 0 ? kXentPartial : kXentAccumulate);
                b.part = reinterpret_cast<float*>(at(plan.part_dh)); b.part_rows = plan.part_dh_rows; b.part_ld = plan.part_ld;
                b.out = h.d_dhidden; b.out_m = h.dhidden_stride; b.out_n = 1;
                b.out_vec = vector_rows(h.d_dhidden, h.dhidden_stride, h.dtype);
                if ((rc = launch_xent_gemm<kXentDHidden>(plan.bn_dim, P, b, rp, n_tiles * b.splits, g_k, w_mn, none, st))) return rc;
            }
            if (h.d_dweight) {
                XentArgs b = a;
                b.splits = plan.dw_splits;
                b.store = plan.dw_parts ? kXentPartial : kXentFinal;
                b.part = reinterpret_cast<float*>(at(plan.part_dw)); b.part_rows = plan.part_dw_rows; b.part_ld = plan.part_ld;
                b.out = h.d_dweight; b.out_m = h.dweight_class_stride; b.out_n = h.dweight_dim_stride;
                b.out_vec = b.out_n == 1 && vector_rows(h.d_dweight, b.out_m, h.dtype);
                if ((rc = launch_xent_gemm<kXentDWeight>(plan.bn_dim, P, b, a.vc, n_tiles * b.splits, g_mn, h_mn, none, st))) return rc;
                if (plan.dw_parts) {
                    XentReduceArgs w = r;
                    w.part = b.part; w.part_rows = b.part_rows; w.splits = b.splits; w.m = a.vc; w.m0 = a.v0;
                    w.out = b.out; w.out_m = b.out_m; w.out_n = b.out_n;
                    if (plan.n_pieces == 1) dw = w;
                    else if ((rc = launch_xent_finish(w, w.m, {}, 0, {}, st))) return rc;
                }
            }
        }
        if (h.d_dhidden && plan.dh_parts) {
            r.part = reinterpret_cast<float*>(at(plan.part_dh)); r.part_rows = plan.part_dh_rows; r.splits = plan.dh_splits;
            r.m_is_count = 1; r.operand = 1;
            r.out = h.d_dhidden; r.out_m = h.dhidden_stride; r.out_n = 1;
            dh = r;
        }
    }
    if (!plan.grads && h.reduction == MASK_REDUCE_NONE) return MASK_OK;      // the join has written every loss
    const XentLossArgs loss = {total, a.warp_loss, total + 1, h.d_loss, h.rows, h.reduction};
    return launch_xent_finish(dw, dw.m, dh, rp, loss, st);
}

}  // namespace mask

extern "C" size_t mask_linear_xent_scratch_bytes(const mask_head* head) {
    if (const char* why = mask::refuse_head(head)) {
        mask::set_error("%s", why);
        return 0;
    }
    return mask::plan_xent(*head).bytes;
}

extern "C" int mask_linear_xent(const mask_head* head, void* d_scratch, size_t scratch_bytes, void* stream) {
    using namespace mask;
    if (const char* why = refuse_head(head)) return fail(MASK_ERR_INVALID_ARGUMENT, why);
    const XentPlan plan = plan_xent(*head);
    MASK_REQUIRE(d_scratch != nullptr && (reinterpret_cast<uintptr_t>(d_scratch) & 255) == 0, "scratch must be 256-byte aligned");
    if (scratch_bytes < plan.bytes) return fail(MASK_ERR_SCRATCH_TOO_SMALL, "scratch is smaller than mask_linear_xent_scratch_bytes");
    return run_xent(*head, plan, static_cast<char*>(d_scratch), static_cast<cudaStream_t>(stream));
}
