// The gradients of group norm with activation over [N, T, C] (channels last).
//
// With xhat = (x - mean) rstd, z = weight xhat + bias, dz = dout act'(z):
//   dbias = sum dz, dweight = sum dz xhat (over every valid frame of the batch),
//   dx = rstd (weight dz - (s1 + xhat s2) / (M Cg)),
//   s1 = sum weight dz, s2 = sum weight dz xhat (over the group's M Cg values).
//
// Every sum is one over a channel's column first: dbias and dweight of this utterance, of which
// s1 and s2 are sums weighted by `weight`. A block's column sums go to the workspace, a row for
// each block, whose rows are added up in an order that the launch fixes.
//
// Two ways, chosen by size (shape_of):
// - Rows on chip: a block keeps its rows of x, and dz in fp32 in the place of dout, so x and dout
//   are read once and the slope is evaluated once; that takes 48 bytes for 8 values of a 16-bit
//   type. (32, with dout as it came and the slope evaluated again as the streams do, would let
//   one block hold half as much again; it has not been measured.) A cluster adds up (s1, s2)
//   where one block cannot hold an utterance's slab. A second launch adds the parameters'
//   gradients.
// - Streams: one launch for the sums, and one for dx and the parameters' gradients, which
//   evaluates the slope again. It reads x and dout twice, but none of its blocks waits for
//   another or holds 72 KB while it does.
//
// Measured: 256 x 375 x 1024 f16 ragged in 32 groups, SiLU, on chip, 126 us (52 % of a plain
// copy's rate for reading x and dout and writing dx once); 256 x 750 x 192 bf16 ragged in 6
// groups, Swoosh-R, streams, 51.3 us (48 %, and 79 % with what is read twice counted twice); 16 x
// 3000 x 1024 f16 in one group, SiLU, streams, 65 us (50 % and 83 %). Issue is 54 to 65 % busy (65
// instructions a pair of values on chip, 45 and 42 in the two streams) and the rest is a block's
// own latency: its parameters, its first rows and its sums across threads.
#include <type_traits>

#include "fga_kernels.h"
#include "group_norm.cuh"

namespace fga {
namespace {

using namespace group_norm;

constexpr int kTileBytes = 72 << 10;
constexpr int kGatherBytes = kMaxCluster * kMaxSlabGroups * static_cast<int>(sizeof(float2));

// dz as fp32 planes of 16 bytes of each vector, the first of which held dout.
template <typename T> constexpr int kPlanes = kVec<T> / 4;
template <typename T> constexpr int kVectorBytes = 16 + 16 * kPlanes<T>;
// The most that add_up takes.
template <typename T>
constexpr int kSumBytes = 2 * kThreads * kVec<T> * static_cast<int>(sizeof(float2));

template <typename T> struct Tensors {
    const T* dout;
    const T* x;
    const int32_t* lengths;
    const T* weight;
    const T* bias;
    const float* mean;  // [N, G]
    const float* rstd;
    T* dx;
};

// A column's shift, which stops short of where it would leave fp32: the slopes there are what they
// are further on, and silu's would be inf * 0. (2^126 log2 e of weight xhat still fit on top.)
// Infinities and NaN stay what they are. (No finite bias of fp16 gets there.)
template <typename T>
__device__ __forceinline__ float2 bounded_shift_of(float2 bias, int act) {
    constexpr float kMost = 2.1e38f;
    const float2 s = shift_of(bias, act);
    if (std::is_same_v<T, __half> || act == FGA_ACTIVATION_NONE) return s;
    return make_float2(isfinite(bias.x) ? fminf(fmaxf(s.x, -kMost), kMost) : s.x,
                       isfinite(bias.y) ? fminf(fmaxf(s.y, -kMost), kMost) : s.y);
}

// A column's parameters: d = x - mean, z = d scale + shift (both in the activation's units), xhat
// = d rstd. What `through` makes of dout is dz / unit: the sums make up for it at their end, dx
// in its product with scale.
template <typename T, bool kWhole> struct Column {
    static constexpr int kStats = kWhole ? 1 : kPairs<T>;
    float2 scale[kPairs<T>], shift[kPairs<T>], rstd[kStats], minus[kStats];  // minus the mean
    template <bool kAligned>
    __device__ __forceinline__ void read(const Tensors<T>& t, const Place<T>& p, const Geometry& g,
                                         int act) {
        const float2 unit = splat2(unit_of(act));
        unpack<T>(load<T, kAligned>(t.weight + p.channel(), p.count), scale);
        unpack<T>(load<T, kAligned>(t.bias + p.channel(), p.count), shift);
        const int64_t group = static_cast<int64_t>(p.n) * g.groups + p.first_group;
#pragma unroll
        for (int k = 0; k < kStats; ++k) {
            const int64_t i = group + p.group_of(2 * k, g);
            const int64_t j = kWhole ? i : group + p.group_of(2 * k + 1, g);
            rstd[k] = make_float2(t.rstd[i], t.rstd[j]);
            minus[k] = make_float2(-t.mean[i], -t.mean[j]);
        }
#pragma unroll
        for (int e = 0; e < kPairs<T>; ++e) {
            shift[e] = bounded_shift_of<T>(shift[e], act);
            scale[e] = mul2(mul2(scale[e], unit), rstd[kWhole ? 0 : e]);
        }
    }
    // x to x - mean.
    __device__ __forceinline__ void centre(float2 (&x)[kPairs<T>]) const {
#pragma unroll
        for (int e = 0; e < kPairs<T>; ++e) x[e] = add2(x[e], minus[kWhole ? 0 : e]);
    }
    // dout to dz / unit; x is centred.
    __device__ __forceinline__ void through(float2 (&d)[kPairs<T>], const float2 (&x)[kPairs<T>],
                                            int act) const {
        if (act == FGA_ACTIVATION_SILU) {
#pragma unroll
            for (int e = 0; e < kPairs<T>; ++e)
                d[e] = mul2(d[e], slope<FGA_ACTIVATION_SILU>(fma2(x[e], scale[e], shift[e])));
        } else if (act == FGA_ACTIVATION_SWOOSH_R) {
#pragma unroll
            for (int e = 0; e < kPairs<T>; ++e)
                d[e] = mul2(d[e], slope<FGA_ACTIVATION_SWOOSH_R>(fma2(x[e], scale[e], shift[e])));
        }
    }
    // The sums of dz and dz xhat, without their factors: unit, and (the second) rstd.
    __device__ __forceinline__ void add(float2 (&db)[kPairs<T>], float2 (&dw)[kPairs<T>],
                                        const float2 (&d)[kPairs<T>],
                                        const float2 (&x)[kPairs<T>]) const {
#pragma unroll
        for (int e = 0; e < kPairs<T>; ++e) {
            db[e] = add2(db[e], d[e]);
            dw[e] = fma2(d[e], x[e], dw[e]);
        }
    }
    // This vector's part of (s1, s2), from those sums: scale is weight unit rstd.
    __device__ __forceinline__ float2 weigh(const float2 (&db)[kPairs<T>],
                                            const float2 (&dw)[kPairs<T>]) const {
        float2 s1 = mul2(scale[0], db[0]), s2 = mul2(scale[0], dw[0]);
#pragma unroll
        for (int e = 1; e < kPairs<T>; ++e) {
            s1 = fma2(scale[e], db[e], s1);
            s2 = fma2(scale[e], dw[e], s2);
        }
        // (rstd is 0 where the variance overflowed: then dx is 0 whatever s1 is.)
        const float s = (s1.x + s1.y) * reciprocal_approx(rstd[0].x);
        return make_float2(rstd[0].x > 0.0f ? s : 0.0f, s2.x + s2.y);
    }
    // The sums with their factors.
    __device__ __forceinline__ void finish(float2 (&db)[kPairs<T>], float2 (&dw)[kPairs<T>],
                                           int act) const {
        const float2 unit = splat2(unit_of(act));
#pragma unroll
        for (int e = 0; e < kPairs<T>; ++e) {
            db[e] = mul2(db[e], unit);
            dw[e] = mul2(dw[e], mul2(unit, rstd[kWhole ? 0 : e]));
        }
    }
};

// dx = dz rstd weight + (x - mean) slope + offset, with the group's means m1 = s1 / (M Cg), m2 =
// s2 / (M Cg): slope = -rstd^2 m2, offset = -rstd m1.
template <typename T, bool kWhole> struct Final {
    static constexpr int kStats = kWhole ? 1 : kPairs<T>;
    float2 slope[kStats], offset[kStats];
    __device__ __forceinline__ void make(const Column<T, kWhole>& column, const float2* sums,
                                         float inv, const Place<T>& p, const Geometry& g) {
#pragma unroll
        for (int k = 0; k < kStats; ++k) {
            const float2 a = sums[p.group_of(2 * k, g)];
            const float2 b = kWhole ? a : sums[p.group_of(2 * k + 1, g)];
            const float2 r = mul2(column.rstd[k], splat2(-inv));
            offset[k] = mul2(r, make_float2(a.x, b.x));
            slope[k] = mul2(mul2(r, column.rstd[k]), make_float2(a.y, b.y));
        }
    }
    __device__ __forceinline__ float2 operator()(float2 dz, float2 x, float2 scale, int e) const {
        return fma2(dz, scale, fma2(x, slope[kWhole ? 0 : e], offset[kWhole ? 0 : e]));
    }
};

// The weight of the channel whose column this thread adds up, asked for early (not kWhole).
template <typename T>
__device__ __forceinline__ float own_weight(const T* weight, const Place<T>& p, const Geometry& g) {
    const int e = g.by_lanes.quotient(threadIdx.x), c = (threadIdx.x - e * g.lanes) * kVec<T> + e;
    return e < kVec<T> && c < p.channels ? to_f32<T>(weight[p.first_channel + c]) : 0.0f;
}

// What the threads of a block add up at their end, in shared memory: (dbias, dweight) of each
// column, [row][vector's channel][lane] so that neither side of the barrier meets a bank twice,
// and behind them for the groups' (s1, s2) what each vector contributes, [row][lane] (if not
// kWhole, the columns' weighted sums).
template <typename T, bool kWhole>
__device__ __forceinline__ void add_up(float2 (&db)[kPairs<T>], float2 (&dw)[kPairs<T>],
                                       float2 weighed, float w, float2* part, float2* group_sums,
                                       float2* __restrict__ sums, const T* __restrict__ weight,
                                       const Place<T>& p, const Geometry& g) {
    const int columns = g.lanes * kVec<T>;
    int rows = g.step, row = p.row;
    if (kWarp % g.lanes == 0) {
        // Whole rows of threads in a warp: the warp's own sum first.
        for (int o = g.lanes; o < kWarp; o *= 2) {
#pragma unroll
            for (int e = 0; e < kPairs<T>; ++e) {
                db[e] = add2(db[e], make_float2(__shfl_xor_sync(0xffffffffu, db[e].x, o),
                                                __shfl_xor_sync(0xffffffffu, db[e].y, o)));
                dw[e] = add2(dw[e], make_float2(__shfl_xor_sync(0xffffffffu, dw[e].x, o),
                                                __shfl_xor_sync(0xffffffffu, dw[e].y, o)));
            }
            if (kWhole)
                weighed = add2(weighed, make_float2(__shfl_xor_sync(0xffffffffu, weighed.x, o),
                                                    __shfl_xor_sync(0xffffffffu, weighed.y, o)));
        }
        rows = kBlockWarps;
        row = threadIdx.x % kWarp < g.lanes ? threadIdx.x / kWarp : rows;
    }
    float2* behind = part + rows * columns;
    if (row < rows) {
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e)
            part[row * columns + e * g.lanes + p.lane] =
                make_float2(channel_of(db, e), channel_of(dw, e));
        if (kWhole) behind[row * g.lanes + p.lane] = weighed;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < columns; i += kThreads) {
        float2 s = part[i];
#pragma unroll 4
        for (int r = 1; r < rows; ++r) s = add2(s, part[r * columns + i]);
        sums[i] = s;
        if (!kWhole) {
            const int e = g.by_lanes.quotient(i), c = (i - e * g.lanes) * kVec<T> + e;
            if (i >= kThreads)
                w = c < p.channels ? to_f32<T>(weight[p.first_channel + c]) : 0.0f;
            behind[c] = mul2(s, splat2(w));
        }
    }
    if (!kWhole) __syncthreads();
    const int width = kWhole ? p.width / kVec<T> : p.width;
    const Items first(width, g);
    for (int j = threadIdx.x / kWarp; j < p.groups; j += kBlockWarps) {
        float2 s = splat2(0.0f);
        for (Items i = first; i.row < (kWhole ? rows : 1); i.next())
            s = add2(s, behind[i.row * g.lanes + j * width + i.column]);
        s = make_float2(warp_sum(s.x), warp_sum(s.y));
        if (threadIdx.x % kWarp == 0) group_sums[j] = s;
    }
    __syncthreads();
}
// Shared memory of it, in float2.
template <typename T, bool kWhole> int sum_values(const Geometry& g) {
    const int columns = g.lanes * kVec<T>;
    const int rows = kWarp % g.lanes == 0 ? kBlockWarps : g.step;
    return columns * rows + (kWhole ? rows * g.lanes : columns);
}

// A row of column sums in the workspace: the slabs' columns in the order of add_up.
template <typename T> __host__ __device__ __forceinline__ int64_t sum_pitch(const Geometry& g) {
    return static_cast<int64_t>(g.slabs) * g.lanes * kVec<T>;
}
// The channel of column i of a row, -1 for the padding of a slab's last vector.
template <typename T> __device__ __forceinline__ int channel_at(const Geometry& g, int i) {
    const int columns = g.lanes * kVec<T>, slab = i / columns, at = i - slab * columns;
    const int c = at % g.lanes * kVec<T> + at / g.lanes;  // in the slab
    if (g.parts > 1) {
        const int group = slab / g.parts, from = (slab - group * g.parts) * g.part_channels;
        return c < min(g.part_channels, g.group_channels - from)
                   ? group * g.group_channels + from + c
                   : -1;
    }
    const int slab_channels = g.slab_groups * g.group_channels, from = slab * slab_channels;
    return c < min(slab_channels, g.channels - from) ? from + c : -1;
}

// Adds the rows of column sums, in an order that the launch fixes: kSumColumns columns a block, a
// thread every kSumRows-th row of one of them. (Unsigned: there may be INT32_MAX rows, and the
// last step goes past them.)
constexpr int kSumColumns = 8, kSumRows = kThreads / kSumColumns;
template <typename T>
__device__ __forceinline__ void sum_parameters(const float2* sums, T* __restrict__ dweight,
                                               T* __restrict__ dbias, uint32_t rows,
                                               const Geometry& g, int block, float2* part) {
    const uint32_t row = threadIdx.x / kSumColumns;
    const int i = block * kSumColumns + threadIdx.x % kSumColumns;
    const int64_t pitch = sum_pitch<T>(g);
    float2 s = splat2(0.0f);
    if (i < pitch) {
#pragma unroll 8
        for (uint32_t r = row; r < rows; r += kSumRows) s = add2(s, sums[r * pitch + i]);
    }
    part[threadIdx.x] = s;
#pragma unroll
    for (uint32_t half = kSumRows / 2; half > 0; half /= 2) {
        __syncthreads();
        if (row < half) {
            s = add2(s, part[threadIdx.x + half * kSumColumns]);
            part[threadIdx.x] = s;
        }
    }
    if (row == 0 && i < pitch) {
        const int c = channel_at<T>(g, i);
        if (c >= 0) {
            dbias[c] = from_f32<T>(s.x);
            dweight[c] = from_f32<T>(s.y);
        }
    }
}

// The place of a block's columns in its row of the workspace, a row for each block of each
// utterance.
template <typename T>
__device__ __forceinline__ float2* sums_of(float2* sums, const Place<T>& p, const Geometry& g) {
    return sums + (static_cast<int64_t>(p.n) * g.blocks + p.block) * sum_pitch<T>(g) +
           static_cast<int64_t>(p.slab) * g.lanes * kVec<T>;
}

template <typename T> struct Parameters {
    const float2* sums;
    T* dweight;
    T* dbias;
    uint32_t rows;
};

// `sums`: a row of column sums for each block of each utterance.
template <typename T, bool kAligned, bool kWhole>
__global__ void __launch_bounds__(kThreads, 3)
    group_norm_backward_kernel(Tensors<T> t, float2* __restrict__ sums, Geometry g, int act) {
    extern __shared__ __align__(16) uint4 shared[];
    __shared__ float2 means[kMaxSlabGroups];
    cudaTriggerProgrammaticLaunchCompletion();
    const Place<T> p = Place<T>::make(g, t.lengths, blockIdx.x);
    const int vectors = g.rows * g.lanes;
    uint4* xs = shared;
    uint4* ds = shared + vectors;
    float2* part = reinterpret_cast<float2*>(shared + (1 + kPlanes<T>) * vectors);
    const int mine = p.own_rows(), pitch = g.step * g.lanes, at = p.row * g.lanes + p.lane;
    const int64_t stride = static_cast<int64_t>(g.step) * g.channels;
    const int64_t first = p.at(g, p.begin + p.row);
    if (mine > 0) {
        const T *x = t.x + first, *d = t.dout + first;
#pragma unroll 4
        for (int i = 0; i < mine; ++i, x += stride, d += stride) {
            const bool inner = p.inner(g, p.begin + p.row + i * g.step);
            stage<T, kAligned>(xs + at + i * pitch, x, p.count, inner);
            stage<T, kAligned>(ds + at + i * pitch, d, p.count, inner);
        }
    }
    const float w = kWhole ? 0.0f : own_weight(t.weight, p, g);
    Column<T, kWhole> column;
    float2 db[kPairs<T>], dw[kPairs<T>];
#pragma unroll
    for (int e = 0; e < kPairs<T>; ++e) db[e] = dw[e] = splat2(0.0f);
    if (mine > 0) column.template read<kAligned>(t, p, g, act);
    arrived();
#pragma unroll 2
    for (int i = 0; i < mine; ++i) {
        float2 x[kPairs<T>], d[kPairs<T>];
        unpack<T>(xs[at + i * pitch], x);
        unpack<T>(ds[at + i * pitch], d);
        column.centre(x);
        column.through(d, x, act);
        column.add(db, dw, d, x);
#pragma unroll
        for (int q = 0; q < kPlanes<T>; ++q)
            ds[q * vectors + at + i * pitch] =
                make_uint4(__float_as_uint(d[2 * q].x), __float_as_uint(d[2 * q].y),
                           __float_as_uint(d[2 * q + 1].x), __float_as_uint(d[2 * q + 1].y));
    }
    float2 weighed = splat2(0.0f);
    if (mine > 0) {
        if (kWhole) weighed = column.weigh(db, dw);
        column.finish(db, dw, act);
    }
    add_up<T, kWhole>(db, dw, weighed, w, part, means, sums_of(sums, p, g), t.weight, p, g);
    if (g.blocks > 1) {
        float2* gathered = part;  // [block][group]
        auto cluster = cg::this_cluster();
        cluster.sync();  // every block runs, and has its sums
        for (int q = threadIdx.x / kWarp; q < g.blocks; q += kBlockWarps)
            for (int j = threadIdx.x % kWarp; j < p.groups; j += kWarp)
                *cluster.map_shared_rank(gathered + p.block * g.slab_groups + j, q) = means[j];
        cluster.sync();
        if (threadIdx.x < p.groups) {
            float2 s = make_float2(0.0f, 0.0f);
            for (int q = 0; q < g.blocks; ++q) {
                const float2 v = gathered[q * g.slab_groups + threadIdx.x];
                s.x += v.x;
                s.y += v.y;
            }
            means[threadIdx.x] = s;
        }
        __syncthreads();
    }
    if (mine > 0) {
        const float inv = 1.0f / (static_cast<float>(p.m) * static_cast<float>(g.group_channels));
        Final<T, kWhole> final_;
        final_.make(column, means, inv, p, g);
        T* to = t.dx + first;
#pragma unroll 2
        for (int i = 0; i < mine; ++i, to += stride) {
            float2 x[kPairs<T>], v[kPairs<T>];
            unpack<T>(xs[at + i * pitch], x);
            column.centre(x);
#pragma unroll
            for (int q = 0; q < kPlanes<T>; ++q) {
                float2 d[2];
                unpack<float>(ds[q * vectors + at + i * pitch], d);
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    v[2 * q + e] = final_(d[e], x[2 * q + e], column.scale[2 * q + e], 2 * q + e);
            }
            store<T, kAligned>(to, pack<T>(v), p.count);
        }
    }
    zero_padding<T, kAligned>(t.dx, p, g);
}

// The two launches of a stream. The first leaves each block's (s1, s2) in `partial` [N, G, parts *
// blocks]; the second goes through the rows against the order of the first, so that it begins
// with those that are still in L2, and its first blocks add up the parameters' gradients. It is
// launched early (programmatic dependent launch): its rows are on their way by the time the
// first has ended.
template <typename T, bool kAligned, bool kWhole>
__global__ void __launch_bounds__(kThreads, 3)
    group_norm_sums_kernel(Tensors<T> t, float2* __restrict__ sums, float2* __restrict__ partial,
                           Geometry g, int act) {
    extern __shared__ __align__(16) uint4 shared[];
    __shared__ float2 group_sums[kMaxSlabGroups];
    cudaTriggerProgrammaticLaunchCompletion();
    const Place<T> p = Place<T>::make(g, t.lengths, blockIdx.x);
    const int mine = p.own_rows();
    const int64_t from = p.at(g, p.begin + p.row);
    Stream<T, kAligned, 2> rows;
    rows.from[0] = t.x + from;
    rows.from[1] = t.dout + from;
    rows.start(shared, p, g);
    const float w = kWhole ? 0.0f : own_weight(t.weight, p, g);
    float2 db[kPairs<T>], dw[kPairs<T>], weighed = splat2(0.0f);
#pragma unroll
    for (int e = 0; e < kPairs<T>; ++e) db[e] = dw[e] = splat2(0.0f);
    if (mine > 0) {
        Column<T, kWhole> column;
        column.template read<kAligned>(t, p, g, act);
        rows.each([&](const uint4(&v)[2]) {
            float2 x[kPairs<T>], d[kPairs<T>];
            unpack<T>(v[0], x);
            unpack<T>(v[1], d);
            column.centre(x);
            column.through(d, x, act);
            column.add(db, dw, d, x);
        });
        if (kWhole) weighed = column.weigh(db, dw);
        column.finish(db, dw, act);
    }
    __syncthreads();  // the slots become the threads' sums
    add_up<T, kWhole>(db, dw, weighed, w, reinterpret_cast<float2*>(shared), group_sums,
                      sums_of(sums, p, g), t.weight, p, g);
    if (threadIdx.x < p.groups)
        partial[(static_cast<int64_t>(p.n) * g.groups + p.first_group + threadIdx.x) * g.parts *
                    g.blocks +
                p.slab % g.parts * g.blocks + p.block] = group_sums[threadIdx.x];
}

template <typename T, bool kAligned, bool kWhole>
__global__ void __launch_bounds__(kThreads, 3)
    group_norm_gradient_kernel(Tensors<T> t, const float2* partial, Parameters<T> out, int adders,
                               Geometry g, int act) {
    extern __shared__ __align__(16) uint4 shared[];
    if (blockIdx.x < adders) {
        cudaGridDependencySynchronize();
        __shared__ float2 part[kThreads];
        sum_parameters(out.sums, out.dweight, out.dbias, out.rows, g, blockIdx.x, part);
        return;
    }
    __shared__ float2 means[kMaxSlabGroups];
    const Place<T> p = Place<T>::make(g, t.lengths, gridDim.x - 1 - blockIdx.x);
    const int mine = p.own_rows();
    const int64_t stride = static_cast<int64_t>(g.step) * g.channels;
    const int64_t from = p.at(g, p.begin + p.row);
    Stream<T, kAligned, 2> rows;
    rows.from[0] = t.x + from;
    rows.from[1] = t.dout + from;
    rows.start(shared, p, g);
    Column<T, kWhole> column;
    if (mine > 0) column.template read<kAligned>(t, p, g, act);
    const int count = g.parts * g.blocks;
    cudaGridDependencySynchronize();
    for (int j = threadIdx.x / kWarp; j < p.groups; j += kBlockWarps) {
        const float2* add =
            partial + (static_cast<int64_t>(p.n) * g.groups + p.first_group + j) * count;
        float s1 = 0.0f, s2 = 0.0f;
        for (int i = threadIdx.x % kWarp; i < count; i += kWarp) {
            s1 += add[i].x;
            s2 += add[i].y;
        }
        s1 = warp_sum(s1);
        s2 = warp_sum(s2);
        if (threadIdx.x % kWarp == 0) means[j] = make_float2(s1, s2);
    }
    __syncthreads();
    if (mine > 0) {
        const float inv = 1.0f / (static_cast<float>(p.m) * static_cast<float>(g.group_channels));
        Final<T, kWhole> final_;
        final_.make(column, means, inv, p, g);
        T* to = t.dx + from;
        rows.each([&](const uint4(&v)[2]) {
            float2 x[kPairs<T>], d[kPairs<T>];
            unpack<T>(v[0], x);
            unpack<T>(v[1], d);
            column.centre(x);
            column.through(d, x, act);
#pragma unroll
            for (int e = 0; e < kPairs<T>; ++e) d[e] = final_(d[e], x[e], column.scale[e], e);
            store<T, kAligned>(to, pack<T>(d), p.count);
            to += stride;
        });
    }
    zero_padding<T, kAligned>(t.dx, p, g);
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    group_norm_parameters_kernel(Parameters<T> out, Geometry g) {
    __shared__ float2 part[kThreads];
    cudaGridDependencySynchronize();
    sum_parameters(out.sums, out.dweight, out.dbias, out.rows, g, blockIdx.x, part);
}

// Rows on chip where one block holds a slab's whole length. Where it takes a cluster, that still
// wins for small batches (x and dout of 18 MB bf16: 13.9 us against 17.5 in two streams) and in
// fp32, whose streams move twice the bytes for each slope they evaluate again (64 x 375 x 1024:
// 73 us against 87); larger ones of 16 bits stream (256 x 750 x 192 bf16 ragged: 52 against 65),
// and in fp32 those whose rows start anywhere (64 x 375 x 1001: 92 against 163). Between the 18
// and the 147 MB that were measured in 16 bits the switch is a guess, and it goes by the padded
// batch, since the host does not know the lengths.
constexpr int64_t kClusterBytes = 64 << 20;
Shape shape_of(const GroupNormBackwardProblem& p, bool aligned) {
    const int element = p.dtype == FGA_FLOAT ? 4 : 2;
    const Problem q{p.batch, p.length, p.channels, p.groups, element, aligned};
    const Shape s = resident_shape(q, element == 4 ? kVectorBytes<float> : kVectorBytes<__half>,
                                   kTileBytes);
    const int64_t bytes = 2LL * p.batch * p.length * p.channels * element;
    const bool resident =
        s.geo.blocks == 1 || (s.geo.blocks > 1 &&
                               ((element == 4 && s.aligned) || bytes <= kClusterBytes));
    return resident ? s : stream_shape(q);
}

int64_t sum_rows(const Shape& s, int batch) { return static_cast<int64_t>(batch) * s.geo.blocks; }

template <typename T, bool kAligned, bool kWhole>
cudaError_t run(const GroupNormBackwardProblem& p, const Shape& s, cudaStream_t stream) {
    static SmemAttr resident, first, second;
    const Tensors<T> t{static_cast<const T*>(p.grad_output), static_cast<const T*>(p.x),
                       p.valid_lengths, static_cast<const T*>(p.weight),
                       static_cast<const T*>(p.bias), p.mean, p.rstd, static_cast<T*>(p.grad_x)};
    const Geometry& g = s.geo;
    float2* sums = static_cast<float2*>(p.workspace);
    const int64_t rows = sum_rows(s, p.batch);
    // What a cluster gathers takes the place of the sums.
    const int part = static_cast<int>(sizeof(float2)) *
                     std::max(sum_values<T, kWhole>(g), s.split ? 0 : g.blocks * g.slab_groups);
    const Parameters<T> out{sums, static_cast<T*>(p.grad_weight), static_cast<T*>(p.grad_bias),
                            static_cast<uint32_t>(rows)};
    const int adders = static_cast<int>((sum_pitch<T>(g) + kSumColumns - 1) / kSumColumns);
    const int64_t blocks = s.units * g.blocks;
    cudaError_t e;
    if (!s.split) {
        e = launch(resident, group_norm_backward_kernel<T, kAligned, kWhole>,
                   {blocks, g.blocks, false, g.rows * g.lanes * kVectorBytes<T> + part,
                    kTileBytes + kThreads * kVectorBytes<T> + kSumBytes<T> + kGatherBytes},
                   stream, t, sums, g, p.activation);
        if (e != cudaSuccess) return e;
        return launch(second, group_norm_parameters_kernel<T>, {adders, 1, true, 0, 0}, stream,
                      out, g);
    }
    constexpr int kSlots = Stream<T, kAligned, 2>::kBytes, kMost = std::max(kSlots, kSumBytes<T>);
    float2* partial = sums + rows * sum_pitch<T>(g);
    e = launch(first, group_norm_sums_kernel<T, kAligned, kWhole>,
               {blocks, 1, false, std::max(kSlots, part), kMost}, stream, t, sums, partial, g,
               p.activation);
    if (e != cudaSuccess) return e;
    return launch(second, group_norm_gradient_kernel<T, kAligned, kWhole>,
                  {blocks + adders, 1, true, kSlots, kSlots}, stream, t,
                  static_cast<const float2*>(partial), out, adders, g,
                  p.activation);
}

template <typename T> cudaError_t run(const GroupNormBackwardProblem& p, cudaStream_t stream) {
    const Shape s = shape_of(p, aligned16({p.grad_output, p.x, p.weight, p.bias, p.grad_x}));
    if (!s.aligned) return run<T, false, false>(p, s, stream);
    return s.whole ? run<T, true, true>(p, s, stream) : run<T, true, false>(p, s, stream);
}

}  // namespace

size_t group_norm_backward_workspace(const GroupNormBackwardProblem& p) {
    size_t most = 0;
    for (bool aligned : {true, false}) {
        const Shape s = shape_of(p, aligned);
        size_t values = static_cast<size_t>(sum_rows(s, p.batch)) *
                        (p.dtype == FGA_FLOAT ? sum_pitch<float>(s.geo) : sum_pitch<__half>(s.geo));
        if (s.split)
            values += static_cast<size_t>(p.batch) * p.groups * s.geo.parts * s.geo.blocks;
        most = std::max(most, values * sizeof(float2));
    }
    return most;
}

cudaError_t launch_group_norm_backward(const GroupNormBackwardProblem& p, cudaStream_t s,
                                       const char** variant) {
    *variant = "group-norm-backward";
    if (p.dtype == FGA_FLOAT) return run<float>(p, s);
    if (p.dtype == FGA_HALF) return run<__half>(p, s);
    return run<__nv_bfloat16>(p, s);
}

}  // namespace fga
