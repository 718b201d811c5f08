// What the forward and backward kernels of group norm with activation share: how [N, T, C] is
// cut into slabs of whole groups, a thread's vectors, the activations, and the launch shape.
//
// A block works on some rows of one utterance's slab: the channels of whole groups, at least
// 128 bytes a row where there are so many (or, for a group wider than a block's threads, a part
// of one). Its threads stand in `rows` x `lanes`, a lane one 16-byte vector of channels, and
// keep their column from row to row, so that a column's parameters stay in registers.
#pragma once

#include <cooperative_groups.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <numeric>

#include "../../include/fga_convolution.h"
#include "f32x2.cuh"
#include "fga_common.cuh"
#include "host_util.h"

namespace fga {
namespace group_norm {

namespace cg = cooperative_groups;

constexpr int kThreads = 256, kBlockWarps = kThreads / kWarp;
constexpr int kMaxCluster = 16;
constexpr int kMaxSlabGroups = 64;

template <typename T> constexpr int kVec = 16 / static_cast<int>(sizeof(T));

template <typename T> constexpr int kPairs = kVec<T> / 2;

// ---- vectors -------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void unpack(const uint4& r, float2 (&v)[kPairs<T>]) {
    if constexpr (sizeof(T) == 4) {
        v[0] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
        v[1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
    } else {
        v[0] = unpack2<T>(r.x);
        v[1] = unpack2<T>(r.y);
        v[2] = unpack2<T>(r.z);
        v[3] = unpack2<T>(r.w);
    }
}
template <typename T> __device__ __forceinline__ uint4 pack(const float2 (&v)[kPairs<T>]) {
    if constexpr (sizeof(T) == 4)
        return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x),
                          __float_as_uint(v[1].y));
    else
        return make_uint4(pack2<T>(v[0]), pack2<T>(v[1]), pack2<T>(v[2]), pack2<T>(v[3]));
}
// Channel e of a vector.
template <int kCount> __device__ __forceinline__ float& channel_of(float2 (&v)[kCount], int e) {
    return e % 2 == 0 ? v[e / 2].x : v[e / 2].y;
}

// `count` channels at p, which need only be aligned to their type unless kAligned; the others
// are zero.
template <typename T, bool kAligned>
__device__ __forceinline__ uint4 load(const T* p, int count) {
    if constexpr (kAligned) {
        return *reinterpret_cast<const uint4*>(p);
    } else {
        uint4 r = make_uint4(0, 0, 0, 0);
        T* v = reinterpret_cast<T*>(&r);
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e)
            if (e < count) v[e] = p[e];
        return r;
    }
}
template <typename T, bool kAligned>
__device__ __forceinline__ void store(T* p, const uint4& r, int count) {
    if constexpr (kAligned) {
        *reinterpret_cast<uint4*>(p) = r;
    } else if (sizeof(T) == 2 && count == kVec<T>) {
        // In words, between two halves at an odd element.
        uint32_t* words = reinterpret_cast<uint32_t*>(p);
        if (reinterpret_cast<uintptr_t>(p) & 2u) {
            uint16_t* halves = reinterpret_cast<uint16_t*>(p);
            words = reinterpret_cast<uint32_t*>(halves + 1);
            halves[0] = static_cast<uint16_t>(r.x);
            words[0] = __funnelshift_r(r.x, r.y, 16);
            words[1] = __funnelshift_r(r.y, r.z, 16);
            words[2] = __funnelshift_r(r.z, r.w, 16);
            halves[7] = static_cast<uint16_t>(r.w >> 16);
        } else {
            words[0] = r.x;
            words[1] = r.y;
            words[2] = r.z;
            words[3] = r.w;
        }
    } else {
        const T* v = reinterpret_cast<const T*>(&r);
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e)
            if (e < count) p[e] = v[e];
    }
}

// A vector that starts anywhere, from the one or two aligned words that hold it: 16 bytes an
// access where its elements one by one would take 8, which is what bounds a kernel then (14 x
// 4611 x 598 bf16 ragged in 46 groups, on chip: 239 us by elements, 130 so).
__device__ __forceinline__ uint32_t start_of(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p)) & 15u;
}
// `count` channels from byte `start` of the words; the others are zero.
template <typename T>
__device__ __forceinline__ uint4 vector_of(const uint4& a, const uint4& b, uint32_t start,
                                           int count) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = start & 8u ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = start & 4u ? w[i + 1] : w[i];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __funnelshift_r(w[i], w[i + 1], 8 * (start & 2u));
    }
    if (count < kVec<T>) {
        T* v = reinterpret_cast<T*>(w);
#pragma unroll
        for (int e = 0; e < kVec<T>; ++e)
            if (e >= count) v[e] = T(0.0f);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// Of these two, the second only if the vector reaches into it.
template <typename T> __device__ __forceinline__ bool in_two(uint32_t start, int count) {
    return start + static_cast<uint32_t>(count) * sizeof(T) > 16u;
}
template <typename T> __device__ __forceinline__ uint4 load_words(const T* p, int count) {
    const uint32_t start = start_of(p);
    const uint4* words = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p) - start);
    return vector_of<T>(words[0], in_two<T>(start, count) ? words[1] : uint4{}, start, count);
}

__device__ __forceinline__ void copy16(uint4* to, const void* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                 "l"(from)
                 : "memory");
}
// A vector into shared memory, to be read by the same thread after `arrived`. `inner`: its words
// are the tensor's own.
template <typename T, bool kAligned>
__device__ __forceinline__ void stage(uint4* to, const T* p, int count, bool inner) {
    if constexpr (kAligned)
        copy16(to, p);
    else
        *to = inner ? load_words<T>(p, count) : load<T, false>(p, count);
}
__device__ __forceinline__ void arrived() {
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// ---- activations ---------------------------------------------------------------------------
// The exponentials are base 2, so what the columns' parameters give for x is already in units of
// their exponent: y = unit (z - origin), which saves a multiplication, and for
// Swoosh-R an addition, of every value.
constexpr float kLn2 = 0.69314718f;
__device__ __forceinline__ float unit_of(int act) {
    return act == FGA_ACTIVATION_SILU ? -kLog2e : act == FGA_ACTIVATION_SWOOSH_R ? kLog2e : 1.0f;
}
__device__ __forceinline__ float origin_of(int act) {
    return act == FGA_ACTIVATION_SWOOSH_R ? 1.0f : 0.0f;
}
// A column's shift from its bias, which has to be below kFarBias for it to stay within fp32 in the
// exponent's units (with 2^126 log2 e of weight xhat on top).
constexpr float kFarBias = 1.5e38f;
__device__ __forceinline__ float2 shift_of(float2 bias, int act) {
    return mul2(add2(bias, splat2(-origin_of(act))), splat2(unit_of(act)));
}
__device__ __forceinline__ float2 exp2_of(float2 y) {
    return make_float2(exp2_approx(y.x), exp2_approx(y.y));
}
__device__ __forceinline__ float2 reciprocal_of(float2 y) {
    return make_float2(reciprocal_approx(y.x), reciprocal_approx(y.y));
}

// y to act(z).
template <int kCount> __device__ __forceinline__ void activate(float2 (&y)[kCount], int act) {
    if (act == FGA_ACTIVATION_SILU) {
        // z / (1 + exp(-z)) = y / (unit (1 + 2^y))
#pragma unroll
        for (int i = 0; i < kCount; ++i)
            y[i] = mul2(y[i], reciprocal_of(fma2(exp2_of(y[i]), splat2(-kLog2e), splat2(-kLog2e))));
    } else if (act == FGA_ACTIVATION_SWOOSH_R) {
        // softplus(v) = ln 2 (max(y, 0) + log2(1 + 2^-|y|)) with v = z - 1; the logarithm's
        // argument is in [1, 2], where an absolute error of 2^-22 is as good as log1p next to
        // the sum. -0.08 z - 0.313261687 = -0.08 v - 0.393261687.
#pragma unroll
        for (int i = 0; i < kCount; ++i) {
            const float2 d = add2(make_float2(exp2_approx(-fabsf(y[i].x)), exp2_approx(-fabsf(y[i].y))),
                                  splat2(1.0f));
            const float2 l = make_float2(log2_approx(d.x), log2_approx(d.y));
            const float2 soft = add2(l, make_float2(fmaxf(y[i].x, 0.0f), fmaxf(y[i].y, 0.0f)));
            y[i] = fma2(soft, splat2(kLn2),
                        fma2(y[i], splat2(-0.08f * kLn2), splat2(-0.393261687f)));
        }
    }
}

// y to act'(z) / unit.
template <int kAct> __device__ __forceinline__ float2 slope(float2 y) {
    if constexpr (kAct == FGA_ACTIVATION_SILU) {
        // s (1 + z (1 - s)) with z = -ln2 y, all times -ln2.
        const float2 s = reciprocal_of(add2(exp2_of(y), splat2(1.0f)));
        const float2 rest = fma2(s, splat2(-kLn2 * kLn2), splat2(kLn2 * kLn2));
        return mul2(s, fma2(y, rest, splat2(-kLn2)));
    } else {
        // sigmoid(v) - 0.08 = 0.92 - 1 / (1 + 2^y), times ln2.
        const float2 s = reciprocal_of(add2(exp2_of(y), splat2(1.0f)));
        return fma2(s, splat2(-kLn2), splat2(0.92f * kLn2));
    }
}

// ---- geometry ------------------------------------------------------------------------------
// Division by a number that the host knows, for dividends below 2^31: a block of a few
// microseconds would otherwise spend a third of its instructions on dividing indexes.
struct Divisor {
    uint32_t d, multiplier, shift;
    Divisor() = default;
    explicit Divisor(uint32_t divisor) : d(divisor), multiplier(0), shift(0) {
        if (d == 1) return;
        while ((1ull << shift) < d) ++shift;  // ceil(log2 d)
        multiplier = static_cast<uint32_t>(((1ull << (31 + shift)) + d - 1) / d);
        --shift;
    }
    __device__ __forceinline__ int quotient(int n) const {
        return d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), multiplier) >> shift);
    }
};

struct Geometry {
    int length, channels, groups, group_channels;
    int slab_groups;  // whole groups of a slab
    int parts;        // slabs of a group that is wider than one (then slab_groups is 1)
    int part_channels;
    int slabs;        // of a row
    int blocks;       // that divide the valid rows of an utterance's slab evenly
    int rows;         // most rows of a block
    int lanes, step;  // threads of a row, rows of a block's threads
    int edge;         // rows at either end of an utterance whose words may be partly another's
    int item_width, item_rows;  // of Items: a group's columns, and rows of 32 of them
    Divisor by_blocks, by_slabs, by_lanes, by_step, by_group, by_item;
};

template <typename T> struct Place {
    int n, m, slab, block;
    int first_group, groups;      // of the slab
    int first_channel, channels;  // of the slab
    int lane, row;                // of this thread
    int count;                    // valid channels of this thread's vector; below 1: no work
    int width;                    // channels of a group in the slab
    int begin, rows, each;        // rows of the block; of a block of this utterance
    int passes, extra;            // rows of a thread: passes, and one more in the first `extra`

    // `index`: of the block in the launch, or against it.
    __device__ static Place make(const Geometry& g, const int32_t* lengths, int index,
                                 int thread = threadIdx.x) {
        Place p;
        const int unit = g.by_blocks.quotient(index);
        p.block = index - unit * g.blocks;
        p.n = g.by_slabs.quotient(unit);
        p.slab = unit - p.n * g.slabs;
        p.m = min(max(lengths[p.n], 0), g.length);
        if (g.parts > 1) {
            p.first_group = p.slab / g.parts;
            p.groups = 1;
            const int at = p.slab % g.parts * g.part_channels;
            p.first_channel = p.first_group * g.group_channels + at;
            p.channels = p.width = min(g.part_channels, g.group_channels - at);
        } else {
            p.first_group = p.slab * g.slab_groups;
            p.groups = min(g.slab_groups, g.groups - p.first_group);
            p.first_channel = p.first_group * g.group_channels;
            p.width = g.group_channels;
            p.channels = p.groups * p.width;
        }
        p.row = g.by_lanes.quotient(thread);
        p.lane = thread - p.row * g.lanes;
        p.count = p.row < g.step ? min(kVec<T>, p.channels - p.lane * kVec<T>) : 0;
        p.each = g.by_blocks.quotient(p.m + g.blocks - 1);
        p.begin = min(p.m, p.block * p.each);
        p.rows = min(p.m - p.begin, p.each);
        p.passes = g.by_step.quotient(p.rows);
        p.extra = p.rows - p.passes * g.step;
        return p;
    }
    __device__ __forceinline__ int rows_of_block(int b) const {
        return max(0, min(each, m - b * each));
    }
    // Rows of the block in the threads of row r.
    __device__ __forceinline__ int rows_of(int r) const { return passes + (r < extra ? 1 : 0); }
    __device__ __forceinline__ int own_rows() const { return count > 0 ? rows_of(row) : 0; }
    // The group, within the slab, of this thread's channel e.
    __device__ __forceinline__ int group_of(int e, const Geometry& g) const {
        return g.parts > 1 ? 0 : min(g.by_group.quotient(lane * kVec<T> + e), groups - 1);
    }
    // Whether the words that hold row t are this utterance's.
    __device__ __forceinline__ static bool inner(const Geometry& g, int t) {
        return t >= g.edge && t < g.length - g.edge;
    }
    __device__ __forceinline__ int channel() const { return first_channel + lane * kVec<T>; }
    // Element offset of this thread's vector in row t.
    __device__ __forceinline__ int64_t at(const Geometry& g, int t) const {
        return (static_cast<int64_t>(n) * g.length + t) * g.channels + channel();
    }
};

// The items of one group in a matrix of `columns` columns, `width` of them the group's: a warp
// takes 32 at a time, row by row.
struct Items {
    int row, column, rows_by, columns_by, width;
    __device__ __forceinline__ Items(int width_, const Geometry& g) : width(width_) {
        const int lane = threadIdx.x % kWarp;
        // (A last part is narrower than the others.)
        row = width == g.item_width ? g.by_item.quotient(lane) : lane / width;
        rows_by = width == g.item_width ? g.item_rows : kWarp / width;
        column = lane - row * width;
        columns_by = kWarp - rows_by * width;
    }
    __device__ __forceinline__ void next() {
        row += rows_by;
        column += columns_by;
        if (column >= width) {
            column -= width;
            ++row;
        }
    }
};

// A thread's vectors of its rows, in order, from kSources tensors at once: kDepth - 1 of them are
// on their way through the thread's own slots of shared memory while it works on one, whatever
// the compiler makes of the loop's registers.
constexpr int kDepth = 4;
template <typename T, bool kAligned, int kSources> struct Stream {
    const T* from[kSources];
    uint4* slots;  // [kDepth][kSources][kWords][kThreads]
    int64_t stride;
    int rows, count;
    // Not kAligned: the next row to request, and where the next to work on starts in its words.
    int t, t_step, t_low, t_high;
    uint32_t begins[kSources];

    static constexpr int kWords = kAligned ? 1 : 2;
    static constexpr int kBytes = kDepth * kSources * kWords * kThreads * 16;

    __device__ __forceinline__ uint4* slot_of(int slot, int k) const {
        return slots + (slot * kSources + k) * kWords * kThreads;
    }
    __device__ __forceinline__ void request(bool wanted, int slot) {
        if (wanted) {
#pragma unroll
            for (int k = 0; k < kSources; ++k) {
                uint4* to = slot_of(slot, k);
                if constexpr (kAligned) {
                    copy16(to, from[k]);
                } else {
                    const uint32_t start = start_of(from[k]);
                    const char* words = reinterpret_cast<const char*>(from[k]) - start;
                    if (t >= t_low && t < t_high) {
                        copy16(to, words);
                        if (in_two<T>(start, count)) copy16(to + kThreads, words + 16);
                    } else {
                        for (int e = 0; e < count; ++e) {
                            const uint32_t at = start + e * static_cast<uint32_t>(sizeof(T));
                            char* word = reinterpret_cast<char*>(to + at / 16 * kThreads);
                            *reinterpret_cast<T*>(word + at % 16) = from[k][e];
                        }
                    }
                }
                from[k] += stride;
            }
            t += t_step;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ __forceinline__ void start(uint4* shared, const Place<T>& p, const Geometry& g) {
        slots = shared + threadIdx.x;
        rows = p.own_rows();
        stride = static_cast<int64_t>(g.step) * g.channels;
        count = p.count;
        t = p.begin + p.row;
        t_step = g.step;
        t_low = g.edge;
        t_high = g.length - g.edge;
#pragma unroll
        for (int k = 0; k < kSources; ++k) begins[k] = start_of(from[k]);
#pragma unroll
        for (int i = 0; i < kDepth - 1; ++i) request(i < rows, i);
    }
    // work(vectors) for every row.
    template <typename Work> __device__ __forceinline__ void each(Work work) {
        for (int i = 0; i < rows; i += kDepth) {
#pragma unroll
            for (int s = 0; s < kDepth; ++s) {
                if (i + s >= rows) break;
                uint4 v[kSources];
                request(i + s + kDepth - 1 < rows, (s + kDepth - 1) % kDepth);
                asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
#pragma unroll
                for (int k = 0; k < kSources; ++k) {
                    const uint4* at = slot_of(s, k);
                    if constexpr (kAligned) {
                        v[k] = at[0];
                    } else {
                        v[k] = vector_of<T>(at[0], at[kThreads], begins[k], count);
                        begins[k] = (begins[k] + static_cast<uint32_t>(stride) *
                                                     static_cast<uint32_t>(sizeof(T))) & 15u;
                    }
                }
                work(v);
            }
        }
    }
};

// Zeros in the rows past the valid ones, of which the unit's blocks take turns.
template <typename T, bool kAligned>
__device__ __forceinline__ void zero_padding(T* out, const Place<T>& p, const Geometry& g) {
    if (p.count <= 0) return;
    const int by = g.blocks * g.step;
    const int64_t stride = static_cast<int64_t>(by) * g.channels;
    int t = p.m + p.block * g.step + p.row;
    T* to = out + p.at(g, t);
    for (; t < g.length; t += by, to += stride)
        store<T, kAligned>(to, make_uint4(0, 0, 0, 0), p.count);
}

// ---- launch shape --------------------------------------------------------------------------
struct Problem {
    int batch, length, channels, groups, element;  // element: bytes
    bool aligned;                                  // the buffers, to 16 bytes
};

struct Shape {
    Geometry geo;
    bool aligned;  // vectors are 16-byte aligned in global memory, and full
    bool whole;    // a vector's channels are of one group
    bool split;    // several launches with a workspace between them
    int64_t units; // utterances x slabs
};

// Slabs of about slab_bytes a row.
inline Shape slabs_of(const Problem& p, int64_t slab_bytes) {
    Shape s{};
    const int vec = 16 / p.element, width = p.channels / p.groups;
    Geometry& g = s.geo;
    g.length = p.length;
    g.channels = p.channels;
    g.groups = p.groups;
    g.group_channels = width;
    g.parts = 1;
    g.part_channels = kThreads * vec;
    const int64_t group_bytes = static_cast<int64_t>(width) * p.element;
    // Slabs that start at a multiple of 16 bytes, if that takes no more than the threads.
    int64_t step = 16 / std::gcd<int64_t>(group_bytes, 16);
    if (step > p.groups) step = p.groups;  // one slab: the row
    s.aligned = p.aligned && p.channels % vec == 0 &&
                (step == 1 || step * group_bytes <= kThreads * 16);
    if (!s.aligned) step = 1;
    slab_bytes = std::min<int64_t>(slab_bytes, kThreads * 16);
    const int64_t most = std::min<int64_t>(p.groups, kMaxSlabGroups);
    g.slab_groups = static_cast<int>(
        std::min(step * std::max<int64_t>(1, slab_bytes / (step * group_bytes)),
                 std::max(step, most / step * step)));
    g.slabs = (p.groups + g.slab_groups - 1) / g.slab_groups;
    if (width > g.part_channels) {
        // (A group this wide has a step of 1, so parts of full vectors if aligned at all.)
        g.slab_groups = 1;
        g.parts = (width + g.part_channels - 1) / g.part_channels;
        g.slabs = p.groups * g.parts;
    }
    s.whole = s.aligned && width % vec == 0;
    s.units = static_cast<int64_t>(p.batch) * g.slabs;
    g.item_width = std::min(width, g.part_channels) / (s.whole ? vec : 1);
    g.lanes = (std::min(width * g.slab_groups, g.part_channels) + vec - 1) / vec;
    g.step = kThreads / g.lanes;
    const int64_t row_bytes = static_cast<int64_t>(p.channels) * p.element;
    g.edge = static_cast<int>((15 + row_bytes - 1) / row_bytes);
    return s;
}

inline void set_blocks(Shape& s, int64_t blocks) {
    Geometry& g = s.geo;
    g.blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(blocks, g.length)));
    g.rows = (g.length + g.blocks - 1) / g.blocks;
    g.by_blocks = Divisor(g.blocks);
    g.by_slabs = Divisor(g.slabs);
    g.by_lanes = Divisor(g.lanes);
    g.by_step = Divisor(g.step);
    g.by_group = Divisor(g.group_channels);
    g.by_item = Divisor(g.item_width);
    g.item_rows = kWarp / g.item_width;
}

// One launch that keeps its rows on chip, with bytes_per_vector of shared memory for a vector
// of them and at most tile_bytes a block. Slabs are as wide as that allows for the whole
// length, since a cluster costs two barriers, but at least 64 bytes a row, and no wider than
// 128 where that would leave multiprocessors without work. blocks is 0 where no cluster holds
// the rows.
inline Shape resident_shape(const Problem& p, int bytes_per_vector, int tile_bytes) {
    const int64_t row_fit = 16LL * tile_bytes / (static_cast<int64_t>(p.length) * bytes_per_vector);
    const int64_t wanted = (2LL * sm_count() + p.batch - 1) / p.batch;  // slabs for every processor
    const int64_t spread = std::max<int64_t>(
        128, static_cast<int64_t>(p.channels) * p.element / std::max<int64_t>(1, wanted));
    Shape s = slabs_of(p, std::max<int64_t>(64, std::min(row_fit, spread)));
    const Geometry& g = s.geo;
    const int64_t row_bytes = static_cast<int64_t>(g.lanes) * bytes_per_vector;
    const int64_t fit = std::max<int64_t>(1, tile_bytes / row_bytes);  // rows of a block
    const int64_t needed = (p.length + fit - 1) / fit;
    if (g.parts > 1 || needed > kMaxCluster) return s;
    // Enough blocks for two on every multiprocessor, as long as each has rows for its threads.
    const int64_t fill = std::min<int64_t>((2LL * sm_count() + s.units - 1) / s.units,
                                           (p.length + 2 * g.step - 1) / (2 * g.step));
    set_blocks(s, std::min<int64_t>(std::max(needed, fill), kMaxCluster));
    return s;
}

// Several launches that stream the rows: slabs as wide as the threads, and kStreamBlocks blocks
// for every multiprocessor, of at least 4 rows a thread (a block's sums cost as much as some
// rows) and at most 64.
constexpr int kStreamBlocks = 8;
inline Shape stream_shape(const Problem& p) {
    Shape s = slabs_of(p, kThreads * 16);
    s.split = true;
    const int64_t step = s.geo.step, most = (p.length + 4 * step - 1) / (4 * step);
    const int64_t least = (p.length + 64 * step - 1) / (64 * step);
    const int64_t share = (kStreamBlocks * std::max(1, sm_count()) + s.units - 1) / s.units;
    set_blocks(s, std::max(least, std::min(most, share)));
    return s;
}

inline bool aligned16(std::initializer_list<const void*> buffers) {
    uintptr_t all = 0;
    for (const void* b : buffers) all |= reinterpret_cast<uintptr_t>(b);
    return all % 16 == 0;
}

struct Launch {
    int64_t blocks;
    int cluster;  // blocks of a cluster
    bool early;   // may start before the launch before it ends: the kernel waits for that itself
    int smem, most_smem;
};

template <typename... Params, typename... Args>
cudaError_t launch(SmemAttr& attribute, void (*kernel)(Params...), const Launch& l,
                   cudaStream_t stream, Args... args) {
    const void* entry = reinterpret_cast<const void*>(kernel);
    cudaError_t e = cudaSuccess;
    if (l.most_smem > 0) e = attribute.ensure(entry, l.most_smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(l.blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(l.smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (l.cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(l.cluster);
        attr[cfg.numAttrs].val.clusterDim.y = attr[cfg.numAttrs].val.clusterDim.z = 1;
        ++cfg.numAttrs;
        if (l.cluster > 8)
            e = cudaFuncSetAttribute(entry, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    if (l.early) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++cfg.numAttrs;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace group_norm
}  // namespace fga
