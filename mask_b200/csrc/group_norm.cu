// Group norm with an activation over the node features of one graph or a batch of graphs, channels last, and its
// gradients (mask_group_norm, mask_group_norm_backward).
//
// For graph b (rows off[b] .. off[b+1]) and group g (C / G neighbouring channels), over their n values:
//     mean = sum x / n,  rstd = 1 / sqrt(sum (x - mean)^2 / n + eps),  u = (x - mean) (rstd gamma) + beta,  y = act(u)
//     du = dy act'(u),  xhat = (x - mean) rstd,  dbeta_c = sum du,  dgamma_c = sum du xhat   (over all rows),
//     dx = rstd (du gamma - m1 - xhat m2),  m1 = sum du gamma / n,  m2 = sum du gamma xhat / n   (over graph and group).
// Both directions are a pass of sums over the features, a join of the sums and a pass that writes.  Rows are dealt out in
// chunks of one graph; a block takes a chunk and up to 32 vectors of 16 bytes of channels, so that its loads are whole
// 512-byte stretches whatever the groups are, and leaves two numbers per channel.  They are joined in a fixed order: the
// same call gives the same bits.  The variance is never taken as a difference of squares: 8 values at a time are centred on
// their own mean, and (count, mean, sum of squares) triples are joined.  A batch's chunks need no table: chunk j of graph b
// has number off[b] / chunk + b + j, which leaves room for every graph's last, shorter chunk.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.cuh"

namespace mask {

constexpr int kNormThreads = 256;
constexpr int kNormBatch = 8;       // rows a thread has in flight

struct NormArgs {
    int64_t rows;
    int32_t channels, groups, per_group, graphs, activation;
    float eps;
    int32_t chunk;              // rows
    int32_t tx;                 // threads along the channels (a power of two), 256 / tx along the rows
    const int32_t* offsets;     // or NULL: one graph
    const void* x;
    int64_t x_stride;
    const float* weight;        // or NULL
    const float* bias;          // or NULL
    void* y;
    int64_t y_stride;
    float* mean;
    float* rstd;
    const void* grad;
    int64_t grad_stride;
    float* dweight;             // or NULL
    float* dbias;               // or NULL
    float2* part;               // [chunks][channels]: mean and sum of squares around it; backward: sums of du, du xhat
    float2* sums;               // [graphs][channels], backward
};

template <typename T> __device__ __forceinline__ float to_float(T x);
template <> __device__ __forceinline__ float to_float(float x) { return x; }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_float(float x);
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }

template <typename T, int VEC>
struct Vec {
    uint4 raw;
    __device__ __forceinline__ void load(const T* from) {
        if constexpr (VEC == 1) *reinterpret_cast<T*>(&raw) = *from;
        else raw = *reinterpret_cast<const uint4*>(from);
    }
    __device__ __forceinline__ void store(T* to) const {
        if constexpr (VEC == 1) *to = *reinterpret_cast<const T*>(&raw);
        else *reinterpret_cast<uint4*>(to) = raw;
    }
    __device__ __forceinline__ float get(int i) const { return to_float(reinterpret_cast<const T*>(&raw)[i]); }
    __device__ __forceinline__ void set(int i, float v) { reinterpret_cast<T*>(&raw)[i] = from_float<T>(v); }
};

__device__ __forceinline__ float sigmoid(float u) { return __fdividef(1.f, 1.f + __expf(-u)); }   // exp overflows to inf: 0
__device__ __forceinline__ float activate(float u, int activation) {
    if (activation == MASK_ACT_RELU) return u < 0.f ? 0.f : u;      // NaN stays
    if (activation == MASK_ACT_SILU) return u == -INFINITY ? 0.f : u * sigmoid(u);
    return u;
}
__device__ __forceinline__ float activate_slope(float u, int activation) {
    if (activation == MASK_ACT_RELU) return u > 0.f ? 1.f : (u <= 0.f ? 0.f : u);
    if (activation == MASK_ACT_SILU) {
        const float s = sigmoid(u);
        return s == 0.f ? 0.f : s * (1.f + u * (1.f - s));
    }
    return 1.f;
}

// ---- chunks ------------------------------------------------------------------------------------------------
struct Graph {
    int64_t begin, end;     // rows, inside the array whatever the offsets hold
    int64_t first;          // its first chunk
};
__device__ __forceinline__ Graph graph_of(const NormArgs& p, int b) {
    if (!p.offsets) return {0, p.rows, 0};
    const int64_t begin = min(max((int64_t)p.offsets[b], (int64_t)0), p.rows), end = min(max((int64_t)p.offsets[b + 1], begin), p.rows);
    return {begin, end, begin / p.chunk + b};
}
struct Chunk {
    int graph;
    int64_t row;
    int n;                  // rows, 0: no such chunk
};
// All lanes of a warp: 32 graphs are looked at at a time.
__device__ __forceinline__ Chunk chunk_of(const NormArgs& p, int64_t number) {
    int lo = 0, n = p.graphs;       // the last graph of [lo, lo + n) whose first chunk is not behind `number`
    const int lane = threadIdx.x & 31;
    while (n > 1) {
        const int step = (n + 31) / 32, at = lo + min(lane * step, n - 1);
        const bool reached = lane == 0 || (lane * step < n && graph_of(p, at).first <= number);
        const int last = 31 - __clz(__ballot_sync(0xffffffffu, reached));
        n = min(step, n - last * step);
        lo += last * step;
    }
    const Graph g = graph_of(p, lo);
    const int64_t row = g.begin + (number - g.first) * p.chunk;
    const bool real = number >= g.first && row < g.end;
    return {lo, row, real ? (int)min((int64_t)p.chunk, g.end - row) : 0};
}

// ---- forward -------------------------------------------------------------------------------------------------
struct Moments {
    float n, mean, m2;
};
__device__ __forceinline__ void join(Moments& a, const Moments& b) {
    const float n = a.n + b.n;
    if (n == 0.f) return;
    const float share = b.n / n, d = b.mean - a.mean;
    a.mean += d * share;
    a.m2 += b.m2 + d * d * a.n * share;
    a.n = n;
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) group_norm_moments_kernel(const NormArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    const Chunk chunk = chunk_of(p, blockIdx.x);
    if (chunk.n == 0) return;
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, rows = kNormThreads / p.tx;
    const int c = (blockIdx.y * p.tx + tx) * VEC;
    const T* x = static_cast<const T*>(p.x) + chunk.row * p.x_stride + c;
    float mean[VEC], m2[VEC], n = 0.f;
#pragma unroll
    for (int i = 0; i < VEC; i++) mean[i] = m2[i] = 0.f;
    if (c < p.channels) {
        for (int r = ty; r < chunk.n; r += kNormBatch * rows) {
            Vec<T, VEC> v[kNormBatch];
            const int have = min(kNormBatch, (chunk.n - r + rows - 1) / rows);
#pragma unroll
            for (int k = 0; k < kNormBatch; k++)
                if (k < have) v[k].load(x + (int64_t)(r + k * rows) * p.x_stride);
            const float inv = 1.f / (float)have, share = (float)have / (n + (float)have);
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                float s = 0.f, q = 0.f;
#pragma unroll
                for (int k = 0; k < kNormBatch; k++)
                    if (k < have) s += v[k].get(i);
                s *= inv;
#pragma unroll
                for (int k = 0; k < kNormBatch; k++)
                    if (k < have) {
                        const float d = v[k].get(i) - s;
                        q += d * d;
                    }
                const float d = s - mean[i];
                mean[i] += d * share;
                m2[i] += q + d * d * n * share;
            }
            n += (float)have;
        }
    }
    __shared__ float all[2][VEC][kNormThreads];
    __shared__ float counts[kNormThreads];
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        all[0][i][threadIdx.x] = mean[i];
        all[1][i][threadIdx.x] = m2[i];
    }
    counts[threadIdx.x] = n;
    for (int s = rows / 2; s > 0; s >>= 1) {
        __syncthreads();
        if (ty < s) {
            const int other = threadIdx.x + s * p.tx;
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                Moments a{n, mean[i], m2[i]};
                join(a, {counts[other], all[0][i][other], all[1][i][other]});
                all[0][i][threadIdx.x] = mean[i] = a.mean;
                all[1][i][threadIdx.x] = m2[i] = a.m2;
            }
            counts[threadIdx.x] = n = n + counts[other];
        }
    }
    if (ty == 0 && c < p.channels) {
        float2* to = p.part + (int64_t)blockIdx.x * p.channels + c;
#pragma unroll
        for (int i = 0; i < VEC; i++) to[i] = make_float2(mean[i], m2[i]);
    }
}

__device__ __forceinline__ double block_sum(double v, double* room) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < kNormThreads / 32; w++) v += room[w];
    return v;
}

// One block per graph and group: mean and rstd from the chunks' channels.
__global__ void __launch_bounds__(kNormThreads) group_norm_join_kernel(const NormArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    __shared__ double room[kNormThreads / 32];
    const int b = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
    const Graph graph = graph_of(p, b);
    const int64_t n = graph.end - graph.begin, chunks = (n + p.chunk - 1) / p.chunk, values = chunks * p.per_group;
    const float2* part = p.part + graph.first * p.channels + g * p.per_group;
    auto count = [&](int64_t j) { return (double)min((int64_t)p.chunk, n - j * p.chunk); };
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < values; i += kNormThreads) {
        const int64_t j = i / p.per_group;
        sum += count(j) * part[j * p.channels + (i - j * p.per_group)].x;
    }
    const double total = (double)n * p.per_group, mean = n ? block_sum(sum, room) / total : 0.0;
    double m2 = 0.0;
    for (int64_t i = threadIdx.x; i < values; i += kNormThreads) {
        const int64_t j = i / p.per_group;
        const float2 v = part[j * p.channels + (i - j * p.per_group)];
        const double d = v.x - mean;
        m2 += v.y + count(j) * d * d;
    }
    m2 = block_sum(m2, room);
    if (threadIdx.x == 0) {
        p.mean[blockIdx.x] = (float)mean;
        p.rstd[blockIdx.x] = (float)rsqrt((n ? m2 / total : 0.0) + (double)p.eps);
    }
}

// What a thread keeps of its channels.
template <int VEC>
struct Channels {
    float mean[VEC], rstd[VEC], gain[VEC], bias[VEC];      // gain = rstd gamma
    __device__ __forceinline__ void load(const NormArgs& p, int graph, int c) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const int64_t at = (int64_t)graph * p.groups + (c + i) / p.per_group;
            mean[i] = p.mean[at];
            rstd[i] = p.rstd[at];
            gain[i] = rstd[i] * (p.weight ? p.weight[c + i] : 1.f);
            bias[i] = p.bias ? p.bias[c + i] : 0.f;
        }
    }
    __device__ __forceinline__ float centred(float x, int i) const { return x - mean[i]; }
    __device__ __forceinline__ float linear(float centred, int i) const { return fmaf(centred, gain[i], bias[i]); }
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) group_norm_apply_kernel(const NormArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    // the last chunks first: the L2 still has them from the pass before
    const Chunk chunk = chunk_of(p, gridDim.x - 1 - blockIdx.x);
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, rows = kNormThreads / p.tx;
    const int c = (blockIdx.y * p.tx + tx) * VEC;
    if (chunk.n == 0 || c >= p.channels) return;
    Channels<VEC> ch;
    ch.load(p, chunk.graph, c);
    const T* x = static_cast<const T*>(p.x) + chunk.row * p.x_stride + c;
    T* y = static_cast<T*>(p.y) + chunk.row * p.y_stride + c;
    constexpr int kBatch = kNormBatch / 2;
    for (int r = ty; r < chunk.n; r += kBatch * rows) {
        Vec<T, VEC> v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++)
            if (r + k * rows < chunk.n) v[k].load(x + (int64_t)(r + k * rows) * p.x_stride);
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            if (r + k * rows >= chunk.n) break;
#pragma unroll
            for (int i = 0; i < VEC; i++) v[k].set(i, activate(ch.linear(ch.centred(v[k].get(i), i), i), p.activation));
            v[k].store(y + (int64_t)(r + k * rows) * p.y_stride);
        }
    }
}

// ---- backward ------------------------------------------------------------------------------------------------
template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) group_norm_grad_sums_kernel(const NormArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    const Chunk chunk = chunk_of(p, blockIdx.x);
    if (chunk.n == 0) return;
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, rows = kNormThreads / p.tx;
    const int c = (blockIdx.y * p.tx + tx) * VEC;
    float s1[VEC], s2[VEC];
#pragma unroll
    for (int i = 0; i < VEC; i++) s1[i] = s2[i] = 0.f;
    if (c < p.channels) {
        Channels<VEC> ch;
        ch.load(p, chunk.graph, c);
        const T* x = static_cast<const T*>(p.x) + chunk.row * p.x_stride + c;
        const T* dy = static_cast<const T*>(p.grad) + chunk.row * p.grad_stride + c;
        constexpr int kBatch = kNormBatch / 2;
        for (int r = ty; r < chunk.n; r += kBatch * rows) {
            Vec<T, VEC> v[kBatch], w[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; k++)
                if (r + k * rows < chunk.n) {
                    v[k].load(x + (int64_t)(r + k * rows) * p.x_stride);
                    w[k].load(dy + (int64_t)(r + k * rows) * p.grad_stride);
                }
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                if (r + k * rows >= chunk.n) break;
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const float d = ch.centred(v[k].get(i), i), du = w[k].get(i) * activate_slope(ch.linear(d, i), p.activation);
                    s1[i] += du;
                    s2[i] += du * (d * ch.rstd[i]);
                }
            }
        }
    }
    __shared__ float all[2][VEC][kNormThreads];
    for (int s = rows / 2; s > 0; s >>= 1) {
        if (ty >= s && ty < 2 * s) {
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                all[0][i][threadIdx.x] = s1[i];
                all[1][i][threadIdx.x] = s2[i];
            }
        }
        __syncthreads();
        if (ty < s) {
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                s1[i] += all[0][i][threadIdx.x + s * p.tx];
                s2[i] += all[1][i][threadIdx.x + s * p.tx];
            }
        }
    }
    if (ty == 0 && c < p.channels) {
        float2* to = p.part + (int64_t)blockIdx.x * p.channels + c;
#pragma unroll
        for (int i = 0; i < VEC; i++) to[i] = make_float2(s1[i], s2[i]);
    }
}

// sums[graph][channel] over the graph's chunks: a block per graph and 32 channels, 8 threads a channel.
__device__ __forceinline__ float2 sum_rows(const float2* from, int64_t n, int64_t stride, bool live, float2 (*room)[32]) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    double a = 0.0, b = 0.0;
    if (live)
        for (int64_t j = w; j < n; j += kNormThreads / 32) {
            const float2 v = from[j * stride];
            a += v.x;
            b += v.y;
        }
    __syncthreads();
    room[w][lane] = make_float2((float)a, (float)b);
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kNormThreads / 32; i++) {
        s.x += room[i][lane].x;
        s.y += room[i][lane].y;
    }
    return s;
}
__global__ void __launch_bounds__(kNormThreads) group_norm_grad_join_kernel(const NormArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    __shared__ float2 room[kNormThreads / 32][32];
    const int c = blockIdx.y * 32 + (threadIdx.x & 31);
    const Graph graph = graph_of(p, blockIdx.x);
    const int64_t chunks = (graph.end - graph.begin + p.chunk - 1) / p.chunk;
    const float2 s = sum_rows(p.part + graph.first * p.channels + c, chunks, p.channels, c < p.channels, room);
    if (threadIdx.x < 32 && c < p.channels) p.sums[(int64_t)blockIdx.x * p.channels + c] = s;
}

// Writes dx; the last blocks along x sum the graphs' channels up to dgamma and dbeta.
template <typename T, int VEC>
__global__ void __launch_bounds__(kNormThreads) group_norm_grad_apply_kernel(const NormArgs p, int64_t chunks) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    __shared__ float2 room[kNormThreads / 32][32];
    if (blockIdx.x >= chunks) {
        const int64_t block = (blockIdx.x - chunks) * gridDim.y + blockIdx.y;
        const int64_t c = block * 32 + (threadIdx.x & 31);
        if (block * 32 >= p.channels) return;
        const float2 s = sum_rows(p.sums + c, p.graphs, p.channels, c < p.channels, room);
        if (threadIdx.x < 32 && c < p.channels) {
            if (p.dbias) p.dbias[c] = s.x;
            if (p.dweight) p.dweight[c] = s.y;
        }
        return;
    }
    if (!p.y) return;
    const Chunk chunk = chunk_of(p, chunks - 1 - blockIdx.x);
    if (chunk.n == 0) return;
    // the block's groups' means of du gamma and du gamma xhat
    __shared__ float2 means[32 * 8];
    const int width = p.tx * VEC, first = (int)(blockIdx.y * width) / p.per_group;
    const int last = min((int)(blockIdx.y * width) + width, p.channels) - 1;
    const Graph graph = graph_of(p, chunk.graph);
    const float inv = 1.f / ((float)(graph.end - graph.begin) * (float)p.per_group);
    for (int g = first + (threadIdx.x >> 5); g <= last / p.per_group; g += kNormThreads / 32) {
        float a = 0.f, b = 0.f;
        for (int i = threadIdx.x & 31; i < p.per_group; i += 32) {
            const int c = g * p.per_group + i;
            const float2 s = p.sums[(int64_t)chunk.graph * p.channels + c];
            const float w = p.weight ? p.weight[c] : 1.f;
            a += w * s.x;
            b += w * s.y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        if ((threadIdx.x & 31) == 0) means[g - first] = make_float2(a * inv, b * inv);
    }
    __syncthreads();
    const int tx = threadIdx.x & (p.tx - 1), ty = threadIdx.x / p.tx, rows = kNormThreads / p.tx;
    const int c = (blockIdx.y * p.tx + tx) * VEC;
    if (c >= p.channels) return;
    Channels<VEC> ch;
    ch.load(p, chunk.graph, c);
    float m1[VEC], m2[VEC];      // times rstd
#pragma unroll
    for (int i = 0; i < VEC; i++) {
        const float2 m = means[(c + i) / p.per_group - first];
        m1[i] = m.x * ch.rstd[i];
        m2[i] = m.y * ch.rstd[i] * ch.rstd[i];
    }
    const T* x = static_cast<const T*>(p.x) + chunk.row * p.x_stride + c;
    const T* dy = static_cast<const T*>(p.grad) + chunk.row * p.grad_stride + c;
    T* dx = static_cast<T*>(p.y) + chunk.row * p.y_stride + c;
    constexpr int kBatch = kNormBatch / 2;
    for (int r = ty; r < chunk.n; r += kBatch * rows) {
        Vec<T, VEC> v[kBatch], w[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++)
            if (r + k * rows < chunk.n) {
                v[k].load(x + (int64_t)(r + k * rows) * p.x_stride);
                w[k].load(dy + (int64_t)(r + k * rows) * p.grad_stride);
            }
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            if (r + k * rows >= chunk.n) break;
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const float d = ch.centred(v[k].get(i), i), du = w[k].get(i) * activate_slope(ch.linear(d, i), p.activation);
                v[k].set(i, fmaf(du, ch.gain[i], -fmaf(d, m2[i], m1[i])));
            }
            v[k].store(dx + (int64_t)(r + k * rows) * p.y_stride);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------
struct NormPlan {
    int vec, tx, slabs, chunk;
    int64_t chunks;
    size_t part, sums, bytes;
};

static NormPlan plan_norm(const mask_norm& n, bool backward) {
    NormPlan p = {};
    const int element = n.dtype == MASK_F32 ? 4 : 2, wide = 16 / element;
    auto fits = [&](const void* data, int64_t stride) { return stride % wide == 0 && (reinterpret_cast<uintptr_t>(data) & 15) == 0; };
    const bool vec = n.channels % wide == 0 && fits(n.d_x, n.x_stride) && (!n.d_y || fits(n.d_y, n.y_stride)) && (!backward || fits(n.d_grad, n.grad_stride));
    p.vec = vec ? wide : 1;
    const int vectors = n.channels / p.vec;
    p.tx = 1;
    while (p.tx < 32 && p.tx < vectors) p.tx *= 2;
    p.slabs = (vectors + p.tx - 1) / p.tx;
    // six blocks an SM, chunks of 8 rows a thread to 1024 rows
    const int64_t want = 6 * (int64_t)sm_count(), least = std::max<int64_t>(16, std::min<int64_t>(8 * (kNormThreads / p.tx), 256));
    p.chunk = (int)std::min<int64_t>(std::max<int64_t>(n.rows * p.slabs / want, least), 1024);
    p.chunks = n.rows / p.chunk + n.graphs;
    auto take = [&](size_t bytes) {
        const size_t at = p.bytes;
        p.bytes += (bytes + 255) / 256 * 256;
        return at;
    };
    p.part = take((size_t)p.chunks * n.channels * sizeof(float2));
    if (backward) p.sums = take((size_t)n.graphs * n.channels * sizeof(float2));
    return p;
}

static const char* refuse_norm(const mask_norm* n, bool backward) {
    if (!n) return "norm is NULL";
    if (n->dtype < MASK_F32 || n->dtype > MASK_F16) return "dtype must be MASK_F32, MASK_BF16 or MASK_F16";
    if (n->activation < MASK_ACT_NONE || n->activation > MASK_ACT_SILU) return "activation must be MASK_ACT_NONE, _RELU or _SILU";
    constexpr int64_t most = (int64_t)1 << 31;
    if (n->rows < 0 || n->rows >= most) return "rows out of range";
    if (n->channels < 1 || n->channels > (1 << 20)) return "channels must be 1 to 2^20";
    if (n->groups < 1 || n->channels % n->groups) return "channels must be a multiple of groups";
    if (n->graphs < 1 || n->graphs >= (1 << 24) || (int64_t)n->graphs * n->groups >= most) return "graphs out of range";
    if (!n->d_offsets && n->graphs != 1) return "several graphs need offsets";
    if (!(n->eps >= 0.f)) return "eps must not be negative";
    if (n->rows > 0 && (!n->d_x || (!n->d_y && !backward))) return "an operand is NULL";
    if (!n->d_mean || !n->d_rstd) return "mean or rstd is NULL";
    if (backward && n->rows > 0 && !n->d_grad) return "grad is NULL";
    if (n->x_stride < 0 || n->y_stride < 0 || n->grad_stride < 0) return "strides must not be negative";
    if (n->d_y && n->rows > 1 && n->y_stride < n->channels) return "rows of the result overlap";
    const uintptr_t element = n->dtype == MASK_F32 ? 3 : 1;
    if ((reinterpret_cast<uintptr_t>(n->d_x) | reinterpret_cast<uintptr_t>(n->d_y) | (backward ? reinterpret_cast<uintptr_t>(n->d_grad) : 0)) & element)
        return "an operand is not aligned to its type";
    if ((reinterpret_cast<uintptr_t>(n->d_mean) | reinterpret_cast<uintptr_t>(n->d_rstd) | reinterpret_cast<uintptr_t>(n->d_weight) |
         reinterpret_cast<uintptr_t>(n->d_bias) | reinterpret_cast<uintptr_t>(n->d_offsets) | reinterpret_cast<uintptr_t>(n->d_dweight) |
         reinterpret_cast<uintptr_t>(n->d_dbias)) & 3)
        return "a float32 or int32 array is not aligned to its type";
    return nullptr;
}

template <typename T, int VEC>
static int launch_norm(const NormArgs& a, const NormPlan& p, bool backward, cudaStream_t st) {
    const dim3 grid((unsigned)p.chunks, (unsigned)p.slabs);
    int rc;
    if (!backward) {
        if ((rc = launch_overlapped(group_norm_moments_kernel<T, VEC>, grid, kNormThreads, 0, st, a))) return rc;
        if ((rc = launch_overlapped(group_norm_join_kernel, dim3((unsigned)(a.graphs * a.groups)), kNormThreads, 0, st, a))) return rc;
        return launch_overlapped(group_norm_apply_kernel<T, VEC>, grid, kNormThreads, 0, st, a);
    }
    const int32_t parts = (a.channels + 31) / 32;
    if ((rc = launch_overlapped(group_norm_grad_sums_kernel<T, VEC>, grid, kNormThreads, 0, st, a))) return rc;
    if ((rc = launch_overlapped(group_norm_grad_join_kernel, dim3((unsigned)a.graphs, (unsigned)parts), kNormThreads, 0, st, a))) return rc;
    const unsigned more = a.dweight || a.dbias ? (unsigned)((parts + p.slabs - 1) / p.slabs) : 0;
    return launch_overlapped(group_norm_grad_apply_kernel<T, VEC>, dim3(grid.x + more, grid.y), kNormThreads, 0, st, a, p.chunks);
}

template <typename T, int WIDE>
static int launch_norm_as(const NormArgs& a, const NormPlan& p, bool backward, cudaStream_t st) {
    return p.vec == 1 ? launch_norm<T, 1>(a, p, backward, st) : launch_norm<T, WIDE>(a, p, backward, st);
}

static int run_norm(const mask_norm* n, bool backward, void* d_scratch, size_t scratch_bytes, cudaStream_t st) {
    if (const char* why = refuse_norm(n, backward)) return fail(MASK_ERR_INVALID_ARGUMENT, why);
    const NormPlan p = plan_norm(*n, backward);
    MASK_REQUIRE(d_scratch != nullptr && (reinterpret_cast<uintptr_t>(d_scratch) & 255) == 0, "scratch must be 256-byte aligned");
    if (scratch_bytes < p.bytes) return fail(MASK_ERR_SCRATCH_TOO_SMALL, "scratch is smaller than mask_group_norm_scratch_bytes");
    NormArgs a = {};
    a.rows = n->rows; a.channels = n->channels; a.groups = n->groups; a.per_group = n->channels / n->groups; a.graphs = n->graphs;
    a.activation = n->activation; a.eps = n->eps; a.chunk = p.chunk; a.tx = p.tx;
    a.offsets = n->d_offsets; a.x = n->d_x; a.x_stride = n->x_stride; a.weight = n->d_weight; a.bias = n->d_bias;
    a.y = n->d_y; a.y_stride = n->y_stride; a.mean = n->d_mean; a.rstd = n->d_rstd;
    a.grad = n->d_grad; a.grad_stride = n->grad_stride; a.dweight = n->d_dweight; a.dbias = n->d_dbias;
    a.part = reinterpret_cast<float2*>(static_cast<char*>(d_scratch) + p.part);
    a.sums = reinterpret_cast<float2*>(static_cast<char*>(d_scratch) + p.sums);
    if (n->dtype == MASK_F32) return launch_norm_as<float, 4>(a, p, backward, st);
    if (n->dtype == MASK_BF16) return launch_norm_as<__nv_bfloat16, 8>(a, p, backward, st);
    return launch_norm_as<__half, 8>(a, p, backward, st);
}

}  // namespace mask

extern "C" size_t mask_group_norm_scratch_bytes(const mask_norm* norm, int backward) {
    if (const char* why = mask::refuse_norm(norm, backward != 0)) {
        mask::set_error("%s", why);
        return 0;
    }
    return mask::plan_norm(*norm, backward != 0).bytes;
}

extern "C" int mask_group_norm(const mask_norm* norm, void* d_scratch, size_t scratch_bytes, void* stream) {
    return mask::run_norm(norm, false, d_scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
}

extern "C" int mask_group_norm_backward(const mask_norm* norm, void* d_scratch, size_t scratch_bytes, void* stream) {
    return mask::run_norm(norm, true, d_scratch, scratch_bytes, static_cast<cudaStream_t>(stream));
}
