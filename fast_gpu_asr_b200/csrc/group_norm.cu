// Group norm with activation over [N, T, C] (channels last).
//
// Over the M valid frames of an utterance and the Cg channels of a group:
//   mean = sum x / (M Cg), var = sum (x - mean)^2 / (M Cg), rstd = (var + eps)^-1/2,
//   out = act((x - mean) rstd weight + bias).
//
// The rows of an utterance's slab stay on chip between the statistics and the output: a block
// keeps them in shared memory, a cluster of up to 16 blocks where one is not enough. Every
// thread reads only vectors that it copied itself, so the tile needs no barrier. A thread
// takes the mean and the sum of squares about it over its own values, in one pass about a pivot
// (block_moments says what that costs in rounding), and pairs of (mean, squares) merge exactly
// as the two-pass formula would have it:
//   mean = sum n_i mean_i / sum n_i, squares = sum (squares_i + n_i (mean_i - mean)^2),
// without a difference of large sums. What no cluster holds is done in two launches, the first
// of which leaves each block's (mean, squares) in the workspace.
//
// So x is read once and out written once: 256 x 375 x 1024 f16 ragged, 32 groups, SiLU, takes
// 59 us, 81 % of a plain copy's rate for those bytes (fp32, 64 x 375 x 1024: 29.4 us, 81 %). In
// the way of the rest are instruction issue (56 % busy, 32 instructions a pair of values) and
// that a block loads, reduces and stores in turn; four on a multiprocessor cover for one another,
// which is what 48 KB of tile and 64 registers are chosen for.
#include <type_traits>

#include "fga_kernels.h"
#include "group_norm.cuh"

namespace fga {
namespace {

using namespace group_norm;

constexpr int kTileBytes = 48 << 10;
constexpr int kGatherBytes = kMaxCluster * kMaxSlabGroups * static_cast<int>(sizeof(float2));

// Merges (mean, squares) pairs: visit(add) calls add(count, pair) for each of this lane's, and
// is called twice. Every lane returns the whole's.
template <typename Visit> __device__ __forceinline__ float2 merge(float total, Visit visit) {
    float sum = 0.0f;
    visit([&](float count, float2 v) { sum = fmaf(count, v.x, sum); });
    const float mean = total > 0.0f ? warp_sum(sum) / total : 0.0f;
    float squares = 0.0f;
    visit([&](float count, float2 v) {
        const float d = v.x - mean;
        squares += fmaf(count * d, d, v.y);
    });
    return make_float2(mean, warp_sum(squares));
}

// (mean, squares) of every group of the slab over this block's rows to moments[group]; each(work)
// calls work(vector) for every row of this thread, `first` is that of its first. `part` holds an
// entry per thread (and channel, if not kWhole).
//
// A thread takes both in one pass, about a pivot: the mean of its own first vector (the first
// value of each channel). With n values and the first q of them in the pivot, squares about
// the mean are at least q (pivot - mean)^2, so the n (pivot - mean)^2 taken off the squares
// about the pivot is at most n / q times what is left, a factor on its rounding error. n / q is
// the thread's rows: 12 of a tile where all threads work, 23 at most (129 vectors a row leave
// 127 of the 256 threads idle), 64 of a stream; and it takes a first vector that is an outlier
// itself for the factor to be near that.
template <typename T, bool kWhole, typename Each>
__device__ __forceinline__ void block_moments(const uint4& first, Each each, float2* part,
                                              float2* moments, const Place<T>& p,
                                              const Geometry& g) {
    constexpr int kValues = kWhole ? 1 : kVec<T>, kSums = kWhole ? 1 : kPairs<T>;
    const int mine = p.own_rows(), columns = g.lanes * kValues;
    if (mine > 0) {
        float2 pivot[kSums], sum[kSums], squares[kSums], v[kPairs<T>];
        unpack<T>(first, v);
        if constexpr (kWhole) {
            float2 s = v[0];
#pragma unroll
            for (int i = 1; i < kPairs<T>; ++i) s = add2(s, v[i]);
            pivot[0] = splat2((s.x + s.y) * (-1.0f / kVec<T>));  // negative
        } else {
#pragma unroll
            for (int i = 0; i < kPairs<T>; ++i) pivot[i] = make_float2(-v[i].x, -v[i].y);
        }
#pragma unroll
        for (int k = 0; k < kSums; ++k) sum[k] = squares[k] = splat2(0.0f);
        each([&](const uint4& r) {
            unpack<T>(r, v);
#pragma unroll
            for (int e = 0; e < kPairs<T>; ++e) {
                constexpr bool kOne = kWhole;
                const int k = kOne ? 0 : e;
                const float2 d = add2(v[e], pivot[k]);
                sum[k] = add2(sum[k], d);
                squares[k] = fma2(d, d, squares[k]);
            }
        });
        const float inv = 1.0f / static_cast<float>(mine * (kWhole ? kVec<T> : 1));
#pragma unroll
        for (int e = 0; e < kValues; ++e) {
            float s = channel_of(sum, e), q = channel_of(squares, e);
            if constexpr (kWhole) {
                s += sum[0].y;
                q += squares[0].y;
            }
            const float off = s * inv;  // mean - pivot
            part[p.row * columns + p.lane * kValues + e] =
                make_float2(off - channel_of(pivot, e), fmaxf(fmaf(-s, off, q), 0.0f));
        }
    }
    __syncthreads();
    // A warp per group: its columns of every row of threads.
    const int width = kWhole ? p.width / kVec<T> : p.width;
    const Items first_item(width, g);
    const int used = min(g.step, p.rows);
    const float total = static_cast<float>(p.rows) * static_cast<float>(p.width);
    for (int j = threadIdx.x / kWarp; j < p.groups; j += kBlockWarps) {
        const float2 r = merge(total, [&](auto add) {
            for (Items i = first_item; i.row < used; i.next())
                add(static_cast<float>(p.rows_of(i.row) * (kWhole ? kVec<T> : 1)),
                    part[i.row * columns + j * width + i.column]);
        });
        if (threadIdx.x % kWarp == 0) moments[j] = r;
    }
}

// A column's parameters: z = (x - mean) scale + shift, scale = rstd weight, shift = bias (scale
// and shift in the activation's units). The mean is taken off first, not as part of shift: that
// would round mean * scale, which is hundreds in a group of small variance, and saves an
// instruction of about 16 a pair.
template <typename T, bool kWhole> struct Column {
    static constexpr int kMeans = kWhole ? 1 : kPairs<T>;
    float2 scale[kPairs<T>], shift[kPairs<T>], minus[kMeans];  // minus the mean
    uint4 weight, bias;
    // Asked for before the statistics are there.
    template <bool kAligned>
    __device__ __forceinline__ void read(const T* w, const T* b, const Place<T>& p) {
        weight = load<T, kAligned>(w + p.channel(), p.count);
        bias = load<T, kAligned>(b + p.channel(), p.count);
    }
    // Whether a bias is too far out for its shift (none of fp16 is, but infinities, which stay).
    __device__ __forceinline__ bool far(int act) const {
        if (std::is_same_v<T, __half> || act == FGA_ACTIVATION_NONE) return false;
        float2 v[kPairs<T>];
        unpack<T>(bias, v);
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < kPairs<T>; ++i) most = fmaxf(most, fmaxf(fabsf(v[i].x), fabsf(v[i].y)));
        return most >= kFarBias;
    }
    // `stats`: (mean, rstd) of the slab's groups.
    __device__ __forceinline__ void make(const float2* stats, const Place<T>& p, const Geometry& g,
                                         int act) {
        const float2 unit = splat2(unit_of(act));
        unpack<T>(weight, scale);
        unpack<T>(bias, shift);
#pragma unroll
        for (int i = 0; i < kPairs<T>; ++i) {
            const float2 s = stats[p.group_of(kWhole ? 0 : 2 * i, g)];
            const float2 t = kWhole ? s : stats[p.group_of(2 * i + 1, g)];
            scale[i] = mul2(mul2(scale[i], unit), make_float2(s.y, t.y));
            shift[i] = shift_of(shift[i], act);
            minus[kWhole ? 0 : i] = make_float2(-s.x, -t.x);
        }
    }
    __device__ __forceinline__ uint4 apply(const uint4& r, int act) const {
        float2 v[kPairs<T>];
        unpack<T>(r, v);
#pragma unroll
        for (int i = 0; i < kPairs<T>; ++i)
            v[i] = fma2(add2(v[i], minus[kWhole ? 0 : i]), scale[i], shift[i]);
        activate(v, act);
        return pack<T>(v);
    }
};

__device__ __forceinline__ float2 to_stats(float2 moments, float total, float eps) {
    return make_float2(moments.x, 1.0f / sqrtf((total > 0.0f ? moments.y / total : 0.0f) + eps));
}

template <typename T> struct Tensors {
    const T* x;
    const int32_t* lengths;
    const T* weight;
    const T* bias;
    T* out;
    float* mean;  // [N, G] or null
    float* rstd;
};

// This thread's values where a bias is too far out for its shift, from the formulas in z itself.
// It stands in place of the rows' loop and finds its place anew, from an index and a thread that
// the compiler cannot know to be the same, so that nothing is kept for it through the kernel (256
// x 375 x 1024 bf16 ragged, silu, without such a bias: 57.7 us, 57.9 without this branch, 59.7
// with the values put right after the loop). `stats`: (mean, rstd) of the slab's groups; `index`
// as for Place.
template <typename T>
__device__ __forceinline__ void far_biases(const Tensors<T>& t, const Geometry& g,
                                           const float2* stats, int index, int act) {
    int thread = threadIdx.x;
    asm volatile("" : "+r"(index), "+r"(thread));
    const Place<T> p = Place<T>::make(g, t.lengths, index, thread);
#pragma unroll 1
    for (int e = 0; e < p.count; ++e) {
        const int c = p.channel() + e;
        const float bias = to_f32<T>(t.bias[c]), weight = to_f32<T>(t.weight[c]);
        const float2 s = stats[p.group_of(e, g)];
#pragma unroll 1
        for (int i = 0; i < p.own_rows(); ++i) {
            const int64_t at = p.at(g, p.begin + p.row + i * g.step) + e;
            const float z = fmaf((to_f32<T>(t.x[at]) - s.x) * s.y, weight, bias), v = z - 1.0f;
            const float y = act == FGA_ACTIVATION_SILU
                                ? z / (1.0f + expf(-z))
                                : fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v))) - 0.08f * z -
                                      0.313261687f;
            t.out[at] = from_f32<T>(y);
        }
    }
}

template <typename T, bool kAligned, bool kWhole>
__global__ void __launch_bounds__(kThreads, 4)
    group_norm_kernel(Tensors<T> t, Geometry g, float eps, int act) {
    extern __shared__ __align__(16) uint4 tile[];
    __shared__ float2 part[kWhole ? kThreads : kThreads * kVec<T>];
    __shared__ float2 moments[kMaxSlabGroups];
    const Place<T> p = Place<T>::make(g, t.lengths, blockIdx.x);
    const int mine = p.own_rows(), pitch = g.step * g.lanes;
    uint4* at = tile + p.row * g.lanes + p.lane;
    const int64_t stride = static_cast<int64_t>(g.step) * g.channels;
    {
        const T* from = t.x + p.at(g, p.begin + p.row);
#pragma unroll 4
        for (int i = 0; i < mine; ++i, from += stride)
            stage<T, kAligned>(at + i * pitch, from, p.count,
                               p.inner(g, p.begin + p.row + i * g.step));
    }
    Column<T, kWhole> column;
    if (mine > 0) column.template read<kAligned>(t.weight, t.bias, p);
    arrived();
    block_moments<T, kWhole>(mine > 0 ? at[0] : uint4{}, [&](auto work) {
#pragma unroll 4
        for (int i = 0; i < mine; ++i) work(at[i * pitch]);
    }, part, moments, p, g);
    __syncthreads();
    const float width = static_cast<float>(g.group_channels);
    const float total = static_cast<float>(p.m) * width;
    if (g.blocks > 1) {
        // Behind the tile: [block][group].
        float2* gathered = reinterpret_cast<float2*>(tile + g.rows * g.lanes);
        auto cluster = cg::this_cluster();
        cluster.sync();  // every block runs, and may be written to
        for (int q = threadIdx.x / kWarp; q < g.blocks; q += kBlockWarps)
            for (int j = threadIdx.x % kWarp; j < p.groups; j += kWarp)
                *cluster.map_shared_rank(gathered + p.block * g.slab_groups + j, q) = moments[j];
        cluster.sync();
        for (int j = threadIdx.x / kWarp; j < p.groups; j += kBlockWarps) {
            const float2 r = merge(total, [&](auto add) {
                for (int i = threadIdx.x % kWarp; i < g.blocks; i += kWarp)
                    add(static_cast<float>(p.rows_of_block(i)) * width,
                        gathered[i * g.slab_groups + j]);
            });
            if (threadIdx.x % kWarp == 0) moments[j] = r;
        }
        __syncthreads();
    }
    if (threadIdx.x < p.groups) {
        const float2 s = to_stats(moments[threadIdx.x], total, eps);
        moments[threadIdx.x] = s;
        if (p.block == 0) {
            const int64_t i = static_cast<int64_t>(p.n) * g.groups + p.first_group + threadIdx.x;
            if (t.mean != nullptr) t.mean[i] = s.x;
            if (t.rstd != nullptr) t.rstd[i] = s.y;
        }
    }
    __syncthreads();
    if (mine > 0) {
        if (column.far(act)) {
            far_biases(t, g, moments, blockIdx.x, act);
        } else {
            column.make(moments, p, g, act);
            T* to = t.out + p.at(g, p.begin + p.row);
#pragma unroll 2
            for (int i = 0; i < mine; ++i, to += stride)
                store<T, kAligned>(to, column.apply(at[i * pitch], act), p.count);
        }
    }
    zero_padding<T, kAligned>(t.out, p, g);
}

// The two launches of a stream. The first leaves each block's moments in `partial` [N, G, parts *
// blocks], the second merges and applies them. It goes through the rows against the order of
// the first, so that it begins with those that are still in L2, and is launched early
// (programmatic dependent launch): its rows are on their way by the time the first has ended.
template <typename T, bool kAligned, bool kWhole>
__global__ void __launch_bounds__(kThreads, 4)
    group_norm_moments_kernel(Tensors<T> t, float2* __restrict__ partial, Geometry g) {
    extern __shared__ __align__(16) uint4 slots[];
    __shared__ float2 part[kWhole ? kThreads : kThreads * kVec<T>];
    __shared__ float2 moments[kMaxSlabGroups];
    cudaTriggerProgrammaticLaunchCompletion();
    const Place<T> p = Place<T>::make(g, t.lengths, blockIdx.x);
    Stream<T, kAligned, 1> rows;
    rows.from[0] = t.x + p.at(g, p.begin + p.row);
    const uint4 first = p.own_rows() > 0 ? load<T, kAligned>(rows.from[0], p.count) : uint4{};
    rows.start(slots, p, g);
    block_moments<T, kWhole>(first, [&](auto work) {
        rows.each([&](const uint4(&v)[1]) { work(v[0]); });
    }, part, moments, p, g);
    __syncthreads();
    if (threadIdx.x < p.groups)
        partial[(static_cast<int64_t>(p.n) * g.groups + p.first_group + threadIdx.x) * g.parts *
                    g.blocks +
                p.slab % g.parts * g.blocks + p.block] = moments[threadIdx.x];
}

template <typename T, bool kAligned, bool kWhole>
__global__ void __launch_bounds__(kThreads, 4)
    group_norm_apply_kernel(Tensors<T> t, const float2* partial, Geometry g, float eps,
                            int act) {
    extern __shared__ __align__(16) uint4 slots[];
    __shared__ float2 stats[kMaxSlabGroups];
    const Place<T> p = Place<T>::make(g, t.lengths, gridDim.x - 1 - blockIdx.x);
    const int mine = p.own_rows();
    const int64_t stride = static_cast<int64_t>(g.step) * g.channels;
    const int64_t from = p.at(g, p.begin + p.row);
    Stream<T, kAligned, 1> rows;
    rows.from[0] = t.x + from;
    rows.start(slots, p, g);
    Column<T, kWhole> column;
    if (mine > 0) column.template read<kAligned>(t.weight, t.bias, p);
    const int count = g.parts * g.blocks;
    const float width = static_cast<float>(g.group_channels);
    const float total = static_cast<float>(p.m) * width;
    constexpr int kHeld = 4;  // blocks a lane
    cudaGridDependencySynchronize();
    for (int j = threadIdx.x / kWarp; j < p.groups; j += kBlockWarps) {
        const int64_t group = static_cast<int64_t>(p.n) * g.groups + p.first_group + j;
        const float2* moments = partial + group * count;
        float2 r;
        if (g.parts == 1 && count <= kHeld * kWarp) {
            // Read once, all on their way together (14 x 4611 x 598 bf16 ragged in 46 groups, 85
            // blocks an utterance: 73 us, 83 by reading them for each sum).
            float2 held[kHeld];
#pragma unroll
            for (int k = 0; k < kHeld; ++k) {
                const int i = k * kWarp + threadIdx.x % kWarp;
                held[k] = i < count ? moments[i] : make_float2(0.0f, 0.0f);
            }
            r = merge(total, [&](auto add) {
#pragma unroll
                for (int k = 0; k < kHeld; ++k)
                    add(static_cast<float>(p.rows_of_block(k * kWarp + threadIdx.x % kWarp)) * width,
                        held[k]);
            });
        } else {
            r = merge(total, [&](auto add) {
                for (int i = threadIdx.x % kWarp; i < count; i += kWarp) {
                    const int q = g.by_blocks.quotient(i);
                    const int wide = min(g.part_channels, g.group_channels - q * g.part_channels);
                    add(static_cast<float>(p.rows_of_block(i - q * g.blocks)) *
                            static_cast<float>(wide),
                        moments[i]);
                }
            });
        }
        if (threadIdx.x % kWarp == 0) {
            const float2 s = to_stats(r, total, eps);
            stats[j] = s;
            if (p.block == 0 && p.slab % g.parts == 0) {
                if (t.mean != nullptr) t.mean[group] = s.x;
                if (t.rstd != nullptr) t.rstd[group] = s.y;
            }
        }
    }
    __syncthreads();
    if (mine > 0) {
        if (column.far(act)) {
            arrived();
            far_biases(t, g, stats, gridDim.x - 1 - blockIdx.x, act);
        } else {
            column.make(stats, p, g, act);
            T* to = t.out + from;
            rows.each([&](const uint4(&v)[1]) {
                store<T, kAligned>(to, column.apply(v[0], act), p.count);
                to += stride;
            });
        }
    }
    zero_padding<T, kAligned>(t.out, p, g);
}

template <typename T, bool kAligned, bool kWhole>
cudaError_t run(const GroupNormProblem& p, const Shape& s, cudaStream_t stream) {
    static SmemAttr resident, partial, apply;
    const Tensors<T> t{static_cast<const T*>(p.x), p.valid_lengths, static_cast<const T*>(p.weight),
                       static_cast<const T*>(p.bias), static_cast<T*>(p.output), p.mean, p.rstd};
    const Geometry& g = s.geo;
    const int gather = g.blocks > 1 ? g.blocks * g.slab_groups * static_cast<int>(sizeof(float2)) : 0;
    const int most = kTileBytes + kThreads * 16 + kGatherBytes;
    float2* ws = static_cast<float2*>(p.workspace);
    const int64_t blocks = s.units * g.blocks;
    if (!s.split)
        return launch(resident, group_norm_kernel<T, kAligned, kWhole>,
                      {blocks, g.blocks, false, g.rows * g.lanes * 16 + gather, most}, stream, t, g,
                      p.eps, p.activation);
    constexpr int kSlots = Stream<T, kAligned, 1>::kBytes;
    const cudaError_t e = launch(partial, group_norm_moments_kernel<T, kAligned, kWhole>,
                                 {blocks, 1, false, kSlots, kSlots}, stream, t, ws, g);
    if (e != cudaSuccess) return e;
    return launch(apply, group_norm_apply_kernel<T, kAligned, kWhole>,
                  {blocks, 1, true, kSlots, kSlots}, stream, t, static_cast<const float2*>(ws), g,
                  p.eps, p.activation);
}

// Rows on chip wherever a cluster holds them: as fast as two streams for large batches (256 x 375
// x 1024 f16 in one group: 105 us against 106), faster for small ones (1 x 3000 x 512: 8 against
// 14), where the streams' second launch shows. Rows that start anywhere are cut into as few
// slabs as can be, since a slab's ends share their words with its neighbours': streams where it
// would take a cluster and x is not small (x of 24 MB f16 in 7 groups of 143: 41 us on chip, 32
// in streams; of 12 MB 22.8 and 23.4, in one group of 514 19.5 and 25.9).
constexpr int64_t kAnywhereBytes = 16 << 20;
Shape shape_of(const GroupNormProblem& p, bool aligned) {
    const Problem q{p.batch, p.length, p.channels, p.groups, p.dtype == FGA_FLOAT ? 4 : 2, aligned};
    const Shape s = resident_shape(q, 16, kTileBytes);
    const int64_t bytes = static_cast<int64_t>(p.batch) * p.length * p.channels * q.element;
    const bool resident =
        s.geo.blocks == 1 || (s.geo.blocks > 1 && (s.aligned || bytes <= kAnywhereBytes));
    return resident ? s : stream_shape(q);
}

template <typename T> cudaError_t run(const GroupNormProblem& p, cudaStream_t stream) {
    const Shape s = shape_of(p, aligned16({p.x, p.weight, p.bias, p.output}));
    if (!s.aligned) return run<T, false, false>(p, s, stream);
    return s.whole ? run<T, true, true>(p, s, stream) : run<T, true, false>(p, s, stream);
}

}  // namespace

size_t group_norm_workspace(const GroupNormProblem& p) {
    size_t most = 0;
    for (bool aligned : {true, false}) {
        const Shape s = shape_of(p, aligned);
        if (s.split)
            most = std::max(most, sizeof(float2) * p.batch * p.groups * s.geo.parts * s.geo.blocks);
    }
    return most;
}

cudaError_t launch_group_norm(const GroupNormProblem& p, cudaStream_t s, const char** variant) {
    *variant = "group-norm";
    if (p.dtype == FGA_FLOAT) return run<float>(p, s);
    if (p.dtype == FGA_HALF) return run<__half>(p, s);
    return run<__nv_bfloat16>(p, s);
}

}  // namespace fga
