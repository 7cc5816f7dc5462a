// Group norm with an activation over the node features of one graph or a batch of graphs, channels last, and its
// gradients (mask_group_norm, mask_group_norm_backward).
//
// For graph b (rows off[b] .. off[b+1]) and group g (C / G neighbouring channels), over their n values:
//     mean = sum x / n,  rstd = 1 / sqrt(sum (x - mean)^2 / n + eps),  u = (x - mean) (rstd gamma) + beta,  y = act(u)
//     du = dy act'(u),  xhat = (x - mean) rstd,  dbeta_c = sum du,  dgamma_c = sum du xhat   (over all rows),
//     dx = rstd (du gamma - m1 - xhat m2),  m1 = sum du gamma / n,  m2 = sum du gamma xhat / n   (over graph and group).
// Both directions are a pass of sums over the features, a join of the sums and a pass that writes.  Rows are dealt out in
// chunks of one graph; a block takes a chunk and a slab of up to 32 x 4 channels, so that its loads are whole stretches of
// 256 or 512 bytes whatever the groups are, and leaves two numbers per channel.  A graph that is one chunk is finished by its
// block at once (where slabs hold whole groups): small graphs are read from memory once.  Sums are joined in a fixed order:
// the same call gives the same bits.  The variance is never taken as a difference of squares: 8 values at a time are centred
// on their own mean, and (count, mean, sum of squares) triples are joined.  A batch's chunks need no table: chunk j of graph b
// has number off[b] / chunk + b + j, which leaves room for every graph's last, shorter chunk.
//
// Bound by memory where nothing but sums is computed; SiLU costs two special-function operations a value, 8 values a clock
// and SM.  Channels go in pairs through the packed float instructions, which halves what else is issued (9 instead of 26
// instructions a value in the backward sums).
#include <algorithm>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.cuh"

namespace mask {

constexpr int kNormThreads = 256;
constexpr int kNormVec = 4;         // channels of a thread

struct NormArgs {
    int64_t rows;
    int32_t channels, groups, per_group, graphs;
    float eps;
    int32_t chunk;              // rows
    uint64_t chunk_inverse;     // 2^64 / chunk, rounded up: the high half of a product with it is a quotient (rows < 2^31)
    int32_t tx;                 // threads along the channels, 256 / tx along the rows
    int64_t handled;            // graphs of up to so many rows are finished by the first kernel (slabs hold whole groups)
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
    float2* sums;               // [graphs][channels], backward, graphs of several chunks
};

// ---- pairs -------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t bits(float2 a) { return *reinterpret_cast<uint64_t*>(&a); }
__device__ __forceinline__ float2 pair(uint64_t a) { return *reinterpret_cast<float2*>(&a); }
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return pair(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return pair(r);
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 1 / (1 + exp(-u)); exp's overflow gives 0
__device__ __forceinline__ float2 sigmoid2(float2 u) {
    const float2 t = mul2(u, both(-1.4426950408889634f));
    const float2 d = add2(make_float2(exp2_approx(t.x), exp2_approx(t.y)), both(1.f));
    return make_float2(rcp_approx(d.x), rcp_approx(d.y));
}
template <int ACT>
__device__ __forceinline__ float2 activate2(float2 u) {
    if constexpr (ACT == MASK_ACT_RELU) {     // NaN stays NaN
        float2 r;
        asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r.x) : "f"(u.x));
        asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r.y) : "f"(u.y));
        return r;
    }
    if constexpr (ACT == MASK_ACT_SILU) return mul2(u, sigmoid2(u));
    return u;
}
// dy act'(u)
template <int ACT>
__device__ __forceinline__ float2 through_activation2(float2 dy, float2 u) {
    if constexpr (ACT == MASK_ACT_RELU) {     // u of NaN: NaN
        return make_float2(u.x > 0.f ? dy.x : (u.x <= 0.f ? 0.f : u.x), u.y > 0.f ? dy.y : (u.y <= 0.f ? 0.f : u.y));
    }
    if constexpr (ACT == MASK_ACT_SILU) {     // s + u s (1 - s)
        const float2 s = sigmoid2(u);
        return mul2(dy, fma2(mul2(u, s), fma2(s, both(-1.f), both(1.f)), s));
    }
    return dy;
}

// Four channels of a row, or one (VEC == 1, where the addresses or the channel count rule out vectors).
template <typename T, int VEC>
struct Row {
    uint32_t raw[VEC == 1 ? 1 : (sizeof(T) == 4 ? 4 : 2)];
    // kLast: nobody reads it again, so that the cache may give its room to others first
    template <bool kLast = false>
    __device__ __forceinline__ void load(const T* from) {
        if constexpr (VEC == 1) {
            if constexpr (sizeof(T) == 4) raw[0] = *reinterpret_cast<const uint32_t*>(from);
            else raw[0] = *reinterpret_cast<const uint16_t*>(from);
        } else if constexpr (sizeof(T) == 4) {
            const uint4* at = reinterpret_cast<const uint4*>(from);
            const uint4 v = kLast ? __ldcs(at) : *at;
            raw[0] = v.x; raw[1] = v.y; raw[2] = v.z; raw[3] = v.w;
        } else {
            const uint2* at = reinterpret_cast<const uint2*>(from);
            const uint2 v = kLast ? __ldcs(at) : *at;
            raw[0] = v.x; raw[1] = v.y;
        }
    }
    __device__ __forceinline__ void store(T* to) const {
        if constexpr (VEC == 1) {
            if constexpr (sizeof(T) == 4) *reinterpret_cast<uint32_t*>(to) = raw[0];
            else *reinterpret_cast<uint16_t*>(to) = (uint16_t)raw[0];
        } else if constexpr (sizeof(T) == 4) {
            __stcs(reinterpret_cast<uint4*>(to), make_uint4(raw[0], raw[1], raw[2], raw[3]));
        } else {
            __stcs(reinterpret_cast<uint2*>(to), make_uint2(raw[0], raw[1]));
        }
    }
    // channels 2i and 2i + 1; VEC == 1: the second is 0
    __device__ __forceinline__ float2 get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return make_float2(__uint_as_float(raw[2 * i]), VEC == 1 ? 0.f : __uint_as_float(raw[VEC == 1 ? 0 : 2 * i + 1]));
        } else if constexpr (std::is_same<T, __half>::value) {
            return __half22float2(*reinterpret_cast<const __half2*>(&raw[i]));
        } else {
            return make_float2(__uint_as_float(raw[i] << 16), __uint_as_float(raw[i] & 0xffff0000u));
        }
    }
    __device__ __forceinline__ void set(int i, float2 v) {
        if constexpr (sizeof(T) == 4) {
            raw[2 * i] = __float_as_uint(v.x);
            if constexpr (VEC > 1) raw[2 * i + 1] = __float_as_uint(v.y);
        } else if constexpr (std::is_same<T, __half>::value) {
            const __half2 h = __float22half2_rn(v);
            raw[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __float22bfloat162_rn(v);
            raw[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
};

// ---- chunks ------------------------------------------------------------------------------------------------
struct Graph {
    int64_t begin, end;     // rows, inside the array whatever the offsets hold
    int64_t first;          // its first chunk
};
__device__ __forceinline__ Graph graph_of(const NormArgs& p, int b) {
    if (!p.offsets) return {0, p.rows, 0};
    const int64_t begin = min(max((int64_t)p.offsets[b], (int64_t)0), p.rows), end = min(max((int64_t)p.offsets[b + 1], begin), p.rows);
    return {begin, end, (int64_t)__umul64hi((uint64_t)begin, p.chunk_inverse) + b};
}
__device__ __forceinline__ int chunks_of(const NormArgs& p, const Graph& g) { return (int)__umul64hi((uint64_t)(g.end - g.begin + p.chunk - 1), p.chunk_inverse); }
struct Chunk {
    int graph;
    int64_t row;
    int n;                  // rows, 0: no such chunk
    bool handled;           // the graph is one that the first kernel finishes
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
    return {lo, row, real ? (int)min((int64_t)p.chunk, g.end - row) : 0, g.end - g.begin <= p.handled};
}

struct Place {
    int tx, ty, rows, c;        // threads along the rows; first channel
    bool live;
};
template <int VEC>
__device__ __forceinline__ Place place_of(const NormArgs& p) {
    Place at;
    at.ty = threadIdx.x / p.tx;
    at.tx = threadIdx.x - at.ty * p.tx;
    at.rows = kNormThreads / p.tx;
    at.c = (blockIdx.y * p.tx + at.tx) * VEC;
    at.live = at.c < p.channels && at.ty < at.rows;
    return at;
}

// What a thread keeps of its channels, in pairs: -mean, rstd gamma, beta.
template <int VEC>
struct Channels {
    static constexpr int kPairs = (VEC + 1) / 2;
    float2 minus_mean[kPairs], gain[kPairs], bias[kPairs];
    template <typename Mean, typename Rstd>
    __device__ __forceinline__ void load(const NormArgs& p, int c, Mean mean, Rstd rstd) {
        float* to[3] = {&minus_mean[0].x, &gain[0].x, &bias[0].x};
#pragma unroll
        for (int i = 0; i < 2 * kPairs; i++) {
            const bool real = i < VEC;
            to[0][i] = real ? -mean(c + i) : 0.f;
            to[1][i] = real ? rstd(c + i) * (p.weight ? p.weight[c + i] : 1.f) : 0.f;
            to[2][i] = real && p.bias ? p.bias[c + i] : 0.f;
        }
    }
    __device__ __forceinline__ void load(const NormArgs& p, int graph, int c) {
        const int64_t at = (int64_t)graph * p.groups;
        load(p, c, [&](int k) { return p.mean[at + k / p.per_group]; }, [&](int k) { return p.rstd[at + k / p.per_group]; });
    }
    __device__ __forceinline__ float2 centred(float2 x, int i) const { return add2(x, minus_mean[i]); }
    __device__ __forceinline__ float2 linear(float2 centred, int i) const { return fma2(centred, gain[i], bias[i]); }
};

// ---- forward -------------------------------------------------------------------------------------------------
template <typename T, int VEC, int ACT>
__device__ __forceinline__ void write_rows(const NormArgs& p, const Chunk& chunk, const Place& at, const Channels<VEC>& ch) {
    constexpr int kBatch = 4;
    const T* x = static_cast<const T*>(p.x) + chunk.row * p.x_stride + at.c;
    T* y = static_cast<T*>(p.y) + chunk.row * p.y_stride + at.c;
    for (int r = at.ty; r < chunk.n; r += kBatch * at.rows) {
        Row<T, VEC> v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++)
            if (r + k * at.rows < chunk.n) v[k].template load<true>(x + (int64_t)(r + k * at.rows) * p.x_stride);
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            if (r + k * at.rows >= chunk.n) break;
#pragma unroll
            for (int i = 0; i < Channels<VEC>::kPairs; i++) v[k].set(i, activate2<ACT>(ch.linear(ch.centred(v[k].get(i), i), i)));
            v[k].store(y + (int64_t)(r + k * at.rows) * p.y_stride);
        }
    }
}

// Joins `n2` values of mean `mean2` and squares `q2` to a pair of channels' first `n`; share = n2 / (n + n2).
__device__ __forceinline__ void join2(float2& mean, float2& m2, float n, float2 mean2, float2 q2, float share) {
    const float2 d = add2(mean2, mul2(mean, both(-1.f)));
    mean = fma2(d, both(share), mean);
    m2 = add2(m2, fma2(mul2(d, d), both(n * share), q2));
}

// The power of two below n, from which a tree over n goes down (0 for 1).
__device__ __forceinline__ int half_of(int n) { return n > 1 ? 1 << (31 - __clz(n - 1)) : 0; }

// Mean and squares around it of the chunk's channels; all of the block's rows end up with the threads of ty == 0.
template <typename T, int VEC>
__device__ __forceinline__ void chunk_moments(const NormArgs& p, const Chunk& chunk, const Place& at, float2 (&mean)[Channels<VEC>::kPairs],
                                              float2 (&m2)[Channels<VEC>::kPairs]) {
    constexpr int kPairs = Channels<VEC>::kPairs, kBatch = 8;
    const T* x = static_cast<const T*>(p.x) + chunk.row * p.x_stride + at.c;
    float n = 0.f;
#pragma unroll
    for (int i = 0; i < kPairs; i++) mean[i] = m2[i] = both(0.f);
    if (at.live) {
        for (int r = at.ty; r < chunk.n; r += kBatch * at.rows) {
            Row<T, VEC> v[kBatch];
            const int have = min(kBatch, (chunk.n - r + at.rows - 1) / at.rows);
#pragma unroll
            for (int k = 0; k < kBatch; k++)
                if (k < have) v[k].load(x + (int64_t)(r + k * at.rows) * p.x_stride);
            const float share = __fdividef((float)have, n + (float)have);
            if (have == kBatch) {
#pragma unroll
                for (int i = 0; i < kPairs; i++) {
                    float2 s = both(0.f), q = both(0.f);
#pragma unroll
                    for (int k = 0; k < kBatch; k++) s = add2(s, v[k].get(i));
                    const float2 minus = mul2(s, both(-1.f / kBatch));
#pragma unroll
                    for (int k = 0; k < kBatch; k++) {
                        const float2 d = add2(v[k].get(i), minus);
                        q = fma2(d, d, q);
                    }
                    join2(mean[i], m2[i], n, mul2(s, both(1.f / kBatch)), q, share);
                }
            } else {
                const float inv = 1.f / (float)have;
#pragma unroll
                for (int i = 0; i < kPairs; i++) {
                    float2 s = both(0.f), q = both(0.f);
#pragma unroll
                    for (int k = 0; k < kBatch; k++)
                        if (k < have) s = add2(s, v[k].get(i));
                    s = mul2(s, both(inv));
                    const float2 minus = mul2(s, both(-1.f));
#pragma unroll
                    for (int k = 0; k < kBatch; k++)
                        if (k < have) {
                            const float2 d = add2(v[k].get(i), minus);
                            q = fma2(d, d, q);
                        }
                    join2(mean[i], m2[i], n, s, q, share);
                }
            }
            n += (float)have;
        }
    }
    __shared__ float2 all[2][kPairs][kNormThreads];
    __shared__ float counts[kNormThreads];
    for (int s = half_of(at.rows); s > 0; s >>= 1) {
        if (at.ty >= s && at.ty < min(2 * s, at.rows)) {
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                all[0][i][threadIdx.x] = mean[i];
                all[1][i][threadIdx.x] = m2[i];
            }
            counts[threadIdx.x] = n;
        }
        __syncthreads();
        if (at.ty < s && at.ty + s < at.rows) {
            const int other = threadIdx.x + s * p.tx;
            const float more = counts[other], share = n + more > 0.f ? more / (n + more) : 0.f;
#pragma unroll
            for (int i = 0; i < kPairs; i++) join2(mean[i], m2[i], n, all[0][i][other], all[1][i][other], share);
            n += more;
        }
    }
}
template <int VEC>
__device__ __forceinline__ void put_channels(float2* to, const float2 (&a)[Channels<VEC>::kPairs], const float2 (&b)[Channels<VEC>::kPairs]) {
#pragma unroll
    for (int i = 0; i < Channels<VEC>::kPairs; i++) {
        to[2 * i] = make_float2(a[i].x, b[i].x);
        if (VEC > 1) to[2 * i + 1] = make_float2(a[i].y, b[i].y);
    }
}

// The rest of a graph whose `rows` rows the slab's channels' moments (`channel`, complete and the block's own) are of: its
// groups' statistics, then this block's rows once more (they are in the L1 or L2).
template <typename T, int VEC, int ACT>
__device__ __forceinline__ void finish_graph(const NormArgs& p, const Chunk& chunk, float rows, const Place& at, float2* channel, bool writes_stats) {
    const int width = p.tx * VEC, base = blockIdx.y * width, c = base + threadIdx.x;
    float2 stats = make_float2(0.f, 0.f);
    if ((int)threadIdx.x < width && c < p.channels) {
        const int g0 = threadIdx.x / p.per_group * p.per_group;      // groups begin with the slab
        float sum = 0.f, squares = 0.f;
        for (int i = 0; i < p.per_group; i++) sum += channel[g0 + i].x;
        const float m = sum / (float)p.per_group;
        for (int i = 0; i < p.per_group; i++) {
            const float d = channel[g0 + i].x - m;
            squares += channel[g0 + i].y + rows * d * d;
        }
        stats = make_float2(m, rsqrtf(squares / (rows * (float)p.per_group) + p.eps));
        if ((int)threadIdx.x == g0 && writes_stats) {
            const int64_t to = (int64_t)chunk.graph * p.groups + c / p.per_group;
            p.mean[to] = stats.x;
            p.rstd[to] = stats.y;
        }
    }
    __syncthreads();
    if ((int)threadIdx.x < width) channel[threadIdx.x] = stats;
    __syncthreads();
    if (!at.live) return;
    Channels<VEC> ch;
    ch.load(p, at.c, [&](int k) { return channel[k - base].x; }, [&](int k) { return channel[k - base].y; });
    write_rows<T, VEC, ACT>(p, chunk, at, ch);
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kNormThreads, 4) group_norm_moments_kernel(const NormArgs p) {
    constexpr int kPairs = Channels<VEC>::kPairs;
    wait_for_previous_kernel();
    let_next_kernel_start();
    const Chunk chunk = chunk_of(p, blockIdx.x);
    if (chunk.n == 0) return;
    const Place at = place_of<VEC>(p);
    float2 mean[kPairs], m2[kPairs];
    chunk_moments<T, VEC>(p, chunk, at, mean, m2);
    if (!chunk.handled) {
        if (at.ty == 0 && at.live) put_channels<VEC>(p.part + (int64_t)blockIdx.x * p.channels + at.c, mean, m2);
        return;
    }
    __shared__ float2 channel[32 * kNormVec];
    if (at.ty == 0) put_channels<VEC>(channel + at.tx * VEC, mean, m2);
    __syncthreads();
    finish_graph<T, VEC, ACT>(p, chunk, (float)chunk.n, at, channel, true);
}

// ---- clusters --------------------------------------------------------------------------------------------------
// One graph of middling size by a cluster of eight blocks for each slab of its channels, which take an eighth of the rows
// each and read one another's sums from shared memory: one launch, whose second pass over the rows finds them in the L2.
constexpr int kNormCluster = 8;
// Rows of a thread up to which that is faster than three launches over all SMs.  Forward 2708 x 64 (21 rows): 9.3 us, streamed
// 12.5; 8000 x 64 (62): 19.3 and 18.4; backward 1000 x 64 (8): 9.9 and 14.2; 2708 x 64: 18.8 and 14.5.  (Of batches of such
// graphs none gained: 16 of about 1000 x 128 took 23.8 us and 14.4 streamed.)
constexpr int kNormClusterForward = 28, kNormClusterBackward = 12;

__device__ __forceinline__ void norm_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 load_of_rank(const float2* own, uint32_t rank) {
    float2 v;
    asm volatile("{\n\t.reg .u32 a;\n\tmapa.shared::cluster.u32 a, %2, %3;\n\tld.shared::cluster.v2.f32 {%0, %1}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y)
                 : "r"((uint32_t)__cvta_generic_to_shared(own)), "r"(rank)
                 : "memory");
    return v;
}
// This block's share of the only graph's rows (0 behind the last); n: the graph's.
__device__ __forceinline__ Chunk share_of_cluster(const NormArgs& p, int64_t& n) {
    const Graph g = graph_of(p, 0);
    n = g.end - g.begin;
    const int64_t share = (n + kNormCluster - 1) / kNormCluster, row = g.begin + blockIdx.x * share;
    return {0, row, row < g.end ? (int)min(share, g.end - row) : 0, true};
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kNormThreads, 4) __cluster_dims__(kNormCluster, 1, 1) group_norm_cluster_kernel(const NormArgs p) {
    constexpr int kPairs = Channels<VEC>::kPairs;
    wait_for_previous_kernel();
    let_next_kernel_start();
    int64_t n;
    const Chunk chunk = share_of_cluster(p, n);
    const Place at = place_of<VEC>(p);
    float2 mean[kPairs], m2[kPairs];
    chunk_moments<T, VEC>(p, chunk, at, mean, m2);
    __shared__ float2 mine[32 * kNormVec], channel[32 * kNormVec];
    if (at.ty == 0) put_channels<VEC>(mine + at.tx * VEC, mean, m2);
    norm_cluster_sync();
    if ((int)threadIdx.x < p.tx * VEC) {
        const int64_t share = (n + kNormCluster - 1) / kNormCluster;
        float count = 0.f, mu = 0.f, squares = 0.f;
#pragma unroll
        for (uint32_t r = 0; r < kNormCluster; r++) {
            const float2 v = load_of_rank(mine + threadIdx.x, r);
            const float more = (float)max((int64_t)0, min(share, n - (int64_t)r * share));
            if (more > 0.f) {
                const float part = more / (count + more), d = v.x - mu;
                mu += d * part;
                squares += v.y + d * d * count * part;
                count += more;
            }
        }
        channel[threadIdx.x] = make_float2(mu, squares);
    }
    norm_cluster_sync();                     // nobody reads this block's sums any more; and the block's own barrier
    if (n == 0) {
        const int width = p.tx * VEC, c = blockIdx.y * width + threadIdx.x;
        if (blockIdx.x == 0 && (int)threadIdx.x < width && c < p.channels && c % p.per_group == 0) {
            p.mean[c / p.per_group] = 0.f;
            p.rstd[c / p.per_group] = rsqrtf(p.eps);
        }
        return;
    }
    finish_graph<T, VEC, ACT>(p, chunk, (float)n, at, channel, blockIdx.x == 0);
}

// Which of the graphs [b0, end), 256 at most, the first kernel has not finished (`empty`: those without rows, too), in their
// order; every thread looks at one.  Returns how many.
__device__ __forceinline__ int open_graphs(const NormArgs& p, int b0, int end, bool empty, int* list) {
    __shared__ int before[kNormThreads / 32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, b = b0 + threadIdx.x;
    bool open = false;
    if (b < end) {
        const Graph g = graph_of(p, b);
        open = g.end - g.begin > p.handled || (empty && g.end == g.begin);
    }
    const unsigned ballot = __ballot_sync(0xffffffffu, open);
    __syncthreads();                  // the list and the counts of the last call have been read
    if (lane == 0) before[warp] = __popc(ballot);
    __syncthreads();
    int at = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kNormThreads / 32; w++) {
        if (w < warp) at += before[w];
        all += before[w];
    }
    if (open) list[at + __popc(ballot & ((1u << lane) - 1))] = b;
    __syncthreads();
    return all;
}

// Mean and rstd of a graph and group from the chunks' channels, by a block.
__device__ __forceinline__ void join_group(const NormArgs& p, int b, int g) {
    const Graph graph = graph_of(p, b);
    const int64_t n = graph.end - graph.begin;
    const int chunks = chunks_of(p, graph), last = (int)(n - (int64_t)(chunks - 1) * p.chunk);
    // threads along the group's channels, the rest along the chunks; four chunks in flight
    int across = 1;
    while (across < p.per_group && across < kNormThreads) across *= 2;
    const int tx = threadIdx.x & (across - 1), ty = threadIdx.x / across, step = kNormThreads / across;
    const float2* part = p.part + graph.first * p.channels + g * p.per_group;
    float count = 0.f, mean = 0.f, m2 = 0.f;
    auto join = [&](float n2, float mean2, float q2) {
        if (n2 == 0.f) return;
        const float share = n2 / (count + n2), d = mean2 - mean;
        mean += d * share;
        m2 += q2 + d * d * count * share;
        count += n2;
    };
    for (int c = tx; c < p.per_group; c += across)
        for (int j = ty; j < chunks; j += 4 * step) {
            float2 v[4];
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (j + k * step < chunks) v[k] = part[(int64_t)(j + k * step) * p.channels + c];
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (j + k * step < chunks) join((float)(j + k * step == chunks - 1 ? last : p.chunk), v[k].x, v[k].y);
        }
    __shared__ float room[3][kNormThreads / 32];
    auto join_lanes = [&](int from) {
#pragma unroll
        for (int o = from; o > 0; o >>= 1) {
            const float n2 = __shfl_down_sync(0xffffffffu, count, o), mean_b = __shfl_down_sync(0xffffffffu, mean, o), q2 = __shfl_down_sync(0xffffffffu, m2, o);
            join(n2, mean_b, q2);
        }
    };
    join_lanes(16);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) {
        room[0][warp] = count;
        room[1][warp] = mean;
        room[2][warp] = m2;
    }
    __syncthreads();
    if (warp == 0) {
        count = lane < kNormThreads / 32 ? room[0][lane] : 0.f;
        mean = lane < kNormThreads / 32 ? room[1][lane] : 0.f;
        m2 = lane < kNormThreads / 32 ? room[2][lane] : 0.f;
        join_lanes(4);
        if (lane == 0) {
            p.mean[(int64_t)b * p.groups + g] = mean;
            p.rstd[(int64_t)b * p.groups + g] = rsqrtf((n ? m2 / ((float)n * (float)p.per_group) : 0.f) + p.eps);
        }
    }
    __syncthreads();
}
// A block per group and `per` graphs.
__global__ void __launch_bounds__(kNormThreads) group_norm_join_kernel(const NormArgs p, int per) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    __shared__ int list[kNormThreads];
    const int g = blockIdx.x % p.groups, begin = blockIdx.x / p.groups * per, end = min(begin + per, p.graphs);
    for (int b0 = begin; b0 < end; b0 += kNormThreads) {
        const int n = open_graphs(p, b0, end, true, list);
        for (int i = 0; i < n; i++) join_group(p, list[i], g);
    }
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kNormThreads, 4) group_norm_apply_kernel(const NormArgs p) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    const Chunk chunk = chunk_of(p, blockIdx.x);
    const Place at = place_of<VEC>(p);
    if (chunk.n == 0 || chunk.handled || !at.live) return;
    Channels<VEC> ch;
    ch.load(p, chunk.graph, at.c);
    write_rows<T, VEC, ACT>(p, chunk, at, ch);
}

// ---- backward ------------------------------------------------------------------------------------------------
// Sums over a group's channels, of a graph's sums per channel: means of du gamma (times -rstd) and of du gamma xhat (times
// -rstd^2), by all lanes of a warp.
__device__ __forceinline__ float2 group_means(const NormArgs& p, const float2* sums, int g, int64_t graph, int64_t rows) {
    float a = 0.f, b = 0.f;
    for (int i = threadIdx.x & 31; i < p.per_group; i += 32) {
        const int c = g * p.per_group + i;
        const float2 s = sums[c];
        const float w = p.weight ? p.weight[c] : 1.f;
        a += w * s.x;
        b += w * s.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffu, a, o);
        b += __shfl_xor_sync(0xffffffffu, b, o);
    }
    const float r = p.rstd[graph * p.groups + g], inv = -r / ((float)rows * (float)p.per_group);
    return make_float2(a * inv, b * inv * r);
}

template <typename T, int VEC, int ACT>
__device__ __forceinline__ void write_grads(const NormArgs& p, const Chunk& chunk, const Place& at, const Channels<VEC>& ch, const float2* means, int first) {
    constexpr int kPairs = Channels<VEC>::kPairs, kBatch = 4;
    float2 m1[kPairs], m2[kPairs];
#pragma unroll
    for (int i = 0; i < kPairs; i++) {
        const float2 a = means[(at.c + 2 * i) / p.per_group - first], b = VEC > 1 ? means[(at.c + 2 * i + 1) / p.per_group - first] : a;
        m1[i] = make_float2(a.x, b.x);
        m2[i] = make_float2(a.y, b.y);
    }
    const T* x = static_cast<const T*>(p.x) + chunk.row * p.x_stride + at.c;
    const T* dy = static_cast<const T*>(p.grad) + chunk.row * p.grad_stride + at.c;
    T* dx = static_cast<T*>(p.y) + chunk.row * p.y_stride + at.c;
    for (int r = at.ty; r < chunk.n; r += kBatch * at.rows) {
        Row<T, VEC> v[kBatch], w[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++)
            if (r + k * at.rows < chunk.n) {
                v[k].template load<true>(x + (int64_t)(r + k * at.rows) * p.x_stride);
                w[k].template load<true>(dy + (int64_t)(r + k * at.rows) * p.grad_stride);
            }
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            if (r + k * at.rows >= chunk.n) break;
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                const float2 d = ch.centred(v[k].get(i), i), du = through_activation2<ACT>(w[k].get(i), ch.linear(d, i));
                v[k].set(i, fma2(du, ch.gain[i], fma2(d, m2[i], m1[i])));
            }
            v[k].store(dx + (int64_t)(r + k * at.rows) * p.y_stride);
        }
    }
}

// Sums of du and du xhat of the chunk's channels; all of the block's rows end up with the threads of ty == 0.
template <typename T, int VEC, int ACT>
__device__ __forceinline__ void chunk_grad_sums(const NormArgs& p, const Chunk& chunk, const Place& at, Channels<VEC>& ch, float2 (&s1)[Channels<VEC>::kPairs],
                                                float2 (&s2)[Channels<VEC>::kPairs]) {
    constexpr int kPairs = Channels<VEC>::kPairs, kBatch = 4;
#pragma unroll
    for (int i = 0; i < kPairs; i++) s1[i] = s2[i] = both(0.f);
    if (at.live) {
        ch.load(p, chunk.graph, at.c);
        const T* x = static_cast<const T*>(p.x) + chunk.row * p.x_stride + at.c;
        const T* dy = static_cast<const T*>(p.grad) + chunk.row * p.grad_stride + at.c;
        for (int r = at.ty; r < chunk.n; r += kBatch * at.rows) {
            Row<T, VEC> v[kBatch], w[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; k++)
                if (r + k * at.rows < chunk.n) {
                    v[k].load(x + (int64_t)(r + k * at.rows) * p.x_stride);
                    w[k].load(dy + (int64_t)(r + k * at.rows) * p.grad_stride);
                }
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                if (r + k * at.rows >= chunk.n) break;
#pragma unroll
                for (int i = 0; i < kPairs; i++) {
                    const float2 d = ch.centred(v[k].get(i), i), du = through_activation2<ACT>(w[k].get(i), ch.linear(d, i));
                    s1[i] = add2(s1[i], du);
                    s2[i] = fma2(du, d, s2[i]);
                }
            }
        }
    }
    __shared__ float2 all[2][kPairs][kNormThreads];
    for (int s = half_of(at.rows); s > 0; s >>= 1) {
        if (at.ty >= s && at.ty < min(2 * s, at.rows)) {
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                all[0][i][threadIdx.x] = s1[i];
                all[1][i][threadIdx.x] = s2[i];
            }
        }
        __syncthreads();
        if (at.ty < s && at.ty + s < at.rows) {
#pragma unroll
            for (int i = 0; i < kPairs; i++) {
                s1[i] = add2(s1[i], all[0][i][threadIdx.x + s * p.tx]);
                s2[i] = add2(s2[i], all[1][i][threadIdx.x + s * p.tx]);
            }
        }
    }
    if (at.ty == 0 && at.live) {
        const float* rstd = p.rstd + (int64_t)chunk.graph * p.groups;
#pragma unroll
        for (int i = 0; i < kPairs; i++) {
            const int c = at.c + 2 * i;
            s2[i].x *= rstd[c / p.per_group];
            if (VEC > 1) s2[i].y *= rstd[(c + 1) / p.per_group];
        }
    }
}

// dx of this block's rows of a graph of `rows` rows, from the graph's sums of the slab's channels (`sums`, from the slab's first).
template <typename T, int VEC, int ACT>
__device__ __forceinline__ void finish_grads(const NormArgs& p, const Chunk& chunk, int64_t rows, const Place& at, const Channels<VEC>& ch, const float2* sums) {
    if (!p.y) return;
    __shared__ float2 means[32 * kNormVec];
    const int width = p.tx * VEC, base = blockIdx.y * width, first = base / p.per_group, end = min(base + width, p.channels);
    for (int g = first + (threadIdx.x >> 5); g * p.per_group < end; g += kNormThreads / 32) {
        const float2 m = group_means(p, sums - base, g, chunk.graph, rows);
        if ((threadIdx.x & 31) == 0) means[g - first] = m;
    }
    __syncthreads();
    if (at.live) write_grads<T, VEC, ACT>(p, chunk, at, ch, means, first);
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kNormThreads, 4) group_norm_grad_sums_kernel(const NormArgs p) {
    constexpr int kPairs = Channels<VEC>::kPairs;
    wait_for_previous_kernel();
    let_next_kernel_start();
    const Chunk chunk = chunk_of(p, blockIdx.x);
    if (chunk.n == 0) return;
    const Place at = place_of<VEC>(p);
    float2 s1[kPairs], s2[kPairs];
    Channels<VEC> ch;
    chunk_grad_sums<T, VEC, ACT>(p, chunk, at, ch, s1, s2);
    if (!chunk.handled) {
        if (at.ty == 0 && at.live) put_channels<VEC>(p.part + (int64_t)blockIdx.x * p.channels + at.c, s1, s2);
        return;
    }
    // the whole graph
    __shared__ float2 channel[32 * kNormVec];
    if (at.ty == 0) {
        put_channels<VEC>(channel + at.tx * VEC, s1, s2);
        if (at.live) put_channels<VEC>(p.sums + (int64_t)chunk.graph * p.channels + at.c, s1, s2);
    }
    __syncthreads();
    finish_grads<T, VEC, ACT>(p, chunk, chunk.n, at, ch, channel);
}

template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kNormThreads, 4) __cluster_dims__(kNormCluster, 1, 1) group_norm_grad_cluster_kernel(const NormArgs p) {
    constexpr int kPairs = Channels<VEC>::kPairs;
    wait_for_previous_kernel();
    let_next_kernel_start();
    int64_t n;
    const Chunk chunk = share_of_cluster(p, n);
    const Place at = place_of<VEC>(p);
    float2 s1[kPairs], s2[kPairs];
    Channels<VEC> ch;
    chunk_grad_sums<T, VEC, ACT>(p, chunk, at, ch, s1, s2);
    __shared__ float2 mine[32 * kNormVec], channel[32 * kNormVec];
    if (at.ty == 0) put_channels<VEC>(mine + at.tx * VEC, s1, s2);
    norm_cluster_sync();
    const int width = p.tx * VEC, c = blockIdx.y * width + threadIdx.x;
    if ((int)threadIdx.x < width) {
        float2 s = make_float2(0.f, 0.f);
#pragma unroll
        for (uint32_t r = 0; r < kNormCluster; r++) s = add2(s, load_of_rank(mine + threadIdx.x, r));
        channel[threadIdx.x] = s;
        if (c < p.channels && blockIdx.x == 0) {          // the only graph's sums are the result
            if (p.dbias) p.dbias[c] = s.x;
            if (p.dweight) p.dweight[c] = s.y;
        }
    }
    norm_cluster_sync();                     // nobody reads this block's sums any more; and the block's own barrier
    if (n > 0) finish_grads<T, VEC, ACT>(p, chunk, n, at, ch, channel);
}

// Sums of 8 channels by a block, 32 threads a channel, four values in flight each; every thread gets its channel's.
template <typename Value>
__device__ __forceinline__ float2 sum_of_channel(int n, Value value, float2 (*room)[8]) {
    const int c = threadIdx.x & 7, w = threadIdx.x >> 3;
    double a = 0.0, b = 0.0;
    for (int j = w; j < n; j += 4 * 32) {
        float2 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = j + 32 * k < n ? value(j + 32 * k) : make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            a += v[k].x;
            b += v[k].y;
        }
    }
    __syncthreads();
    room[w][c] = make_float2((float)a, (float)b);
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < 32; i++) s = add2(s, room[i][c]);
    return s;
}
// The graphs' sums from their chunks': a block per 8 channels and `per` graphs.
__global__ void __launch_bounds__(kNormThreads) group_norm_grad_join_kernel(const NormArgs p, int per) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    __shared__ float2 room[32][8];
    __shared__ int list[kNormThreads];
    const int c = blockIdx.x * 8 + (threadIdx.x & 7), begin = blockIdx.y * per, end = min(begin + per, p.graphs);
    for (int b0 = begin; b0 < end; b0 += kNormThreads) {
        const int n = open_graphs(p, b0, end, false, list);
        for (int i = 0; i < n; i++) {
            const Graph graph = graph_of(p, list[i]);
            const float2* part = p.part + graph.first * p.channels + c;
            const float2 s = sum_of_channel(chunks_of(p, graph), [&](int j) { return c < p.channels ? part[(int64_t)j * p.channels] : make_float2(0.f, 0.f); }, room);
            if (threadIdx.x < 8 && c < p.channels) p.sums[(int64_t)list[i] * p.channels + c] = s;
        }
    }
}

// Writes dx; the last blocks along x sum the graphs' channels up to dgamma and dbeta.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(kNormThreads, 4) group_norm_grad_apply_kernel(const NormArgs p, int64_t chunks) {
    wait_for_previous_kernel();
    let_next_kernel_start();
    if (blockIdx.x >= chunks) {
        __shared__ float2 room[32][8];
        const int64_t c0 = ((blockIdx.x - chunks) * gridDim.y + blockIdx.y) * 8, c = c0 + (threadIdx.x & 7);
        if (c0 >= p.channels) return;
        const float2 s = sum_of_channel(p.graphs, [&](int b) {
            // graphs without rows have no sums: what is read for them is dropped, so that no load waits for another
            const float2 v = p.sums[(int64_t)b * p.channels + min(c, (int64_t)p.channels - 1)];
            const Graph g = graph_of(p, b);
            return c < p.channels && g.end > g.begin ? v : make_float2(0.f, 0.f);
        }, room);
        if (threadIdx.x < 8 && c < p.channels) {
            if (p.dbias) p.dbias[c] = s.x;
            if (p.dweight) p.dweight[c] = s.y;
        }
        return;
    }
    const Chunk chunk = chunk_of(p, blockIdx.x);
    if (chunk.n == 0 || !p.y || chunk.handled) return;
    const Place at = place_of<VEC>(p);
    Channels<VEC> ch;
    if (at.live) ch.load(p, chunk.graph, at.c);
    const Graph graph = graph_of(p, chunk.graph);
    finish_grads<T, VEC, ACT>(p, chunk, graph.end - graph.begin, at, ch, p.sums + (int64_t)chunk.graph * p.channels + blockIdx.y * p.tx * VEC);
}

// ---- host ------------------------------------------------------------------------------------------------------
struct NormPlan {
    int vec, tx, slabs, chunk;
    int64_t handled;
    bool clusters;
    int64_t chunks;
    size_t part, sums, bytes;
};

static NormPlan plan_norm(const mask_norm& n, bool backward) {
    NormPlan p = {};
    const int bytes = (n.dtype == MASK_F32 ? 4 : 2) * kNormVec;
    auto fits = [&](const void* data, int64_t stride) { return stride % kNormVec == 0 && reinterpret_cast<uintptr_t>(data) % bytes == 0; };
    const bool vec = n.channels % kNormVec == 0 && fits(n.d_x, n.x_stride) && (!n.d_y || fits(n.d_y, n.y_stride)) && (!backward || fits(n.d_grad, n.grad_stride));
    p.vec = vec ? kNormVec : 1;
    const int vectors = n.channels / p.vec;
    // Threads along the channels: up to 32, of those that make slabs of whole groups (where there are any) the ones that leave
    // fewest idle; more where that is even.
    const int per_group = n.channels / n.groups;
    int unit = per_group;                       // vectors that hold whole groups
    while (unit % p.vec) unit += per_group;
    unit /= p.vec;
    const bool whole = vectors <= 32 || unit <= 32;
    if (vectors <= 32) unit = vectors;
    else if (unit > 32) unit = 16;
    int64_t least_cost = INT64_MAX;
    for (int tx = unit; tx <= 32; tx += unit) {
        const int64_t slabs = (vectors + tx - 1) / tx, cost = slabs * 256 / (kNormThreads / tx);     // threads' time for a row
        // 128 bytes of a row, or what there is: threads behind the row's end would have nothing to do (2^20 x 16 bf16: 25 us
        // forward and 38 backward, 61 and 97 with 16 threads for the row's four vectors)
        const bool wide = tx * (p.vec == 1 ? bytes / kNormVec : bytes) >= 128 || tx >= vectors || tx + unit > 32;
        if (wide && cost <= least_cost) { least_cost = cost; p.tx = tx; }
    }
    p.slabs = (vectors + p.tx - 1) / p.tx;
    // Four blocks an SM are resident: as many chunks as that, in whole batches of rows.  (300007 x 256 bf16 backward: 159 us;
    // twice as many 164, four times 199, since every chunk leaves sums to join and blocks have a start and an end.)  Four blocks
    // leave 64 registers a thread, of which the float32 backward kernels of four channels spill 56 to 120 bytes, the 16-bit ones
    // 4 to 16 (2^18 x 512 float32, ReLU, backward: 501 us, five passes over the features 410).
    const int64_t want = 4 * (int64_t)sm_count(), batch = 8 * (kNormThreads / p.tx), most = std::max<int64_t>(4096 / batch, 1) * batch;
    p.chunk = (int)std::min(std::max((n.rows * p.slabs + want * batch - 1) / (want * batch) * batch, std::min<int64_t>(batch, 256)), most);
    // Graphs of a chunk are finished by its block, one that is not much longer by clusters.
    p.handled = whole ? p.chunk : 0;
    const int64_t share = (int64_t)kNormCluster * (kNormThreads / p.tx) * (backward ? kNormClusterBackward : kNormClusterForward);
    p.clusters = whole && n.graphs == 1 && n.rows > p.chunk && n.rows <= share;
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

// Graphs a block, so that there are at most so many blocks for them (one at least).
static int share_of(int graphs, int blocks) { return (graphs + std::max(blocks, 1) - 1) / std::max(blocks, 1); }

template <typename T, int VEC, int ACT>
static int launch_norm(const NormArgs& a, const NormPlan& p, bool backward, cudaStream_t st) {
    const dim3 grid((unsigned)p.chunks, (unsigned)p.slabs);
    const dim3 clusters(kNormCluster, (unsigned)p.slabs);
    const bool all_handled = a.rows > 0 && a.rows <= p.handled;        // none can be longer
    int rc;
    if (!backward) {
        if (p.clusters) return launch_overlapped(group_norm_cluster_kernel<T, VEC, ACT>, clusters, kNormThreads, 0, st, a);
        if ((rc = launch_overlapped(group_norm_moments_kernel<T, VEC, ACT>, grid, kNormThreads, 0, st, a)) || (all_handled && !a.offsets)) return rc;
        const int per = share_of(a.graphs, 4096 / a.groups);
        if ((rc = launch_overlapped(group_norm_join_kernel, dim3((unsigned)((a.graphs + per - 1) / per * a.groups)), kNormThreads, 0, st, a, per))) return rc;
        return launch_overlapped(group_norm_apply_kernel<T, VEC, ACT>, grid, kNormThreads, 0, st, a);
    }
    if (p.clusters) return launch_overlapped(group_norm_grad_cluster_kernel<T, VEC, ACT>, clusters, kNormThreads, 0, st, a);
    const int32_t parts = (a.channels + 7) / 8;
    if ((rc = launch_overlapped(group_norm_grad_sums_kernel<T, VEC, ACT>, grid, kNormThreads, 0, st, a))) return rc;
    if (!all_handled) {
        const int per = share_of(a.graphs, 4 * sm_count() / parts);
        if ((rc = launch_overlapped(group_norm_grad_join_kernel, dim3((unsigned)parts, (unsigned)((a.graphs + per - 1) / per)), kNormThreads, 0, st, a, per))) return rc;
    }
    const unsigned more = a.dweight || a.dbias ? (unsigned)((parts + p.slabs - 1) / p.slabs) : 0;
    return launch_overlapped(group_norm_grad_apply_kernel<T, VEC, ACT>, dim3(grid.x + more, grid.y), kNormThreads, 0, st, a, p.chunks);
}

template <typename T, int VEC>
static int launch_norm_act(const NormArgs& a, const NormPlan& p, int activation, bool backward, cudaStream_t st) {
    if (activation == MASK_ACT_RELU) return launch_norm<T, VEC, MASK_ACT_RELU>(a, p, backward, st);
    if (activation == MASK_ACT_SILU) return launch_norm<T, VEC, MASK_ACT_SILU>(a, p, backward, st);
    return launch_norm<T, VEC, MASK_ACT_NONE>(a, p, backward, st);
}

template <typename T>
static int launch_norm_as(const NormArgs& a, const NormPlan& p, int activation, bool backward, cudaStream_t st) {
    return p.vec == 1 ? launch_norm_act<T, 1>(a, p, activation, backward, st) : launch_norm_act<T, kNormVec>(a, p, activation, backward, st);
}

static int run_norm(const mask_norm* n, bool backward, void* d_scratch, size_t scratch_bytes, cudaStream_t st) {
    if (const char* why = refuse_norm(n, backward)) return fail(MASK_ERR_INVALID_ARGUMENT, why);
    const NormPlan p = plan_norm(*n, backward);
    MASK_REQUIRE(d_scratch != nullptr && (reinterpret_cast<uintptr_t>(d_scratch) & 255) == 0, "scratch must be 256-byte aligned");
    if (scratch_bytes < p.bytes) return fail(MASK_ERR_SCRATCH_TOO_SMALL, "scratch is smaller than mask_group_norm_scratch_bytes");
    NormArgs a = {};
    a.rows = n->rows; a.channels = n->channels; a.groups = n->groups; a.per_group = n->channels / n->groups; a.graphs = n->graphs;
    a.eps = n->eps; a.chunk = p.chunk; a.chunk_inverse = ~(uint64_t)0 / (uint64_t)p.chunk + 1; a.tx = p.tx; a.handled = p.handled;
    a.offsets = n->d_offsets; a.x = n->d_x; a.x_stride = n->x_stride; a.weight = n->d_weight; a.bias = n->d_bias;
    a.y = n->d_y; a.y_stride = n->y_stride; a.mean = n->d_mean; a.rstd = n->d_rstd;
    a.grad = n->d_grad; a.grad_stride = n->grad_stride; a.dweight = n->d_dweight; a.dbias = n->d_dbias;
    a.part = reinterpret_cast<float2*>(static_cast<char*>(d_scratch) + p.part);
    a.sums = reinterpret_cast<float2*>(static_cast<char*>(d_scratch) + p.sums);
    if (n->dtype == MASK_F32) return launch_norm_as<float>(a, p, n->activation, backward, st);
    if (n->dtype == MASK_BF16) return launch_norm_as<__nv_bfloat16>(a, p, n->activation, backward, st);
    return launch_norm_as<__half>(a, p, n->activation, backward, st);
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
