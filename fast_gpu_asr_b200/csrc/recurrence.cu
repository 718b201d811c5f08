// Gated linear recurrence over [N, T, C], forward and backward:
//   f = sigmoid(gate), p = 1 - f, h[t] = f[t] h[t-1] + p[t] x[t];
//   G[t] = dout[t] + f[t+1] G[t+1] (+ dfinal at the last valid frame),
//   dx[t] = p[t] G[t], dgate[t] = f[t] p[t] (h[t-1] - x[t]) G[t], dinitial = f[0] G[0].
//
// A run of frames takes h to A h + B, with A the product of its f and B what it makes of
// h = 0, and runs compose: that is the scan. A warp takes kFrames consecutive frames of one
// 128-byte row's channels (a lane one value of f32, two of a 16-bit type), finds its (A, B),
// learns the state before its first frame from the warps before it through shared memory, and
// walks its frames again from there, so that no element is read twice. A block's warps cover
// one tile; a block walks the tiles of its utterance and channels in turn, with the next
// tile's rows on their way to shared memory meanwhile. The backward pass runs the same scan
// from the last tile to the first for the carry c[t] = f[t] G[t], and recomputes h from the
// states that the forward pass saved every 64 frames.
//
// Where utterances and channels are too few to fill the GPU, a cluster of blocks divides the
// frames: each block first finds the (A, B) of its whole range, reading it once more (the
// second time from L2), the blocks exchange them through distributed shared memory, and each
// walks its tiles from the state that it now knows.
#include <cooperative_groups.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "../../include/fga_convolution.h"
#include "fga_common.cuh"
#include "fga_kernels.h"
#include "host_util.h"

namespace fga {
namespace {

namespace cg = cooperative_groups;

constexpr int kChunk = FGA_RECURRENCE_STATE_FRAMES;
constexpr int kMaxCluster = 16;
constexpr int kRow = 128;  // bytes of a row that a warp takes
constexpr int kFrames = 8, kWarps = 8;
constexpr int kTile = kFrames * kWarps;
constexpr int kForwardBlocks = 4, kBackwardBlocks = 3;  // on a multiprocessor
static_assert(kTile == kChunk, "a tile starts at a saved state");

// ---- a lane's four bytes of a row ----------------------------------------------------------
template <typename T> struct Lane {
    static constexpr int kVec = 2;
    using Raw = uint32_t;
    static __device__ __forceinline__ void unpack(Raw r, float* v) {
        float2 f;
        if constexpr (std::is_same_v<T, __half>) f = __half22float2(*reinterpret_cast<__half2*>(&r));
        else f = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&r));
        v[0] = f.x;
        v[1] = f.y;
    }
    static __device__ __forceinline__ Raw pack(const float* v) {
        if constexpr (std::is_same_v<T, __half>) {
            const __half2 h = __floats2half2_rn(v[0], v[1]);
            return *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[0], v[1]);
            return *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    static constexpr uint32_t kInfinity = std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
};
template <> struct Lane<float> {
    static constexpr int kVec = 1;
    using Raw = float;
    static __device__ __forceinline__ void unpack(Raw r, float* v) { v[0] = r; }
    static __device__ __forceinline__ Raw pack(const float* v) { return v[0]; }
    static constexpr uint32_t kInfinity = 0x7f800000u;
};

// f and p = 1 - f, both with all their bits: e = exp(-gate), f = 1 / (1 + e), p = e f. The
// exponent stops at 126, where f is the smallest normal number and p is 1; a NaN stays one. The
// special functions flush subnormals: otherwise each costs three more instructions.
__device__ __forceinline__ void gates(float g, float& f, float& p) {
    float e;
    asm("min.NaN.f32 %0, %1, 0f42fc0000;" : "=f"(e) : "f"(g * -kLog2e));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(f) : "f"(1.0f + e));
    p = e * f;
}

// ---- rows between global and shared memory -------------------------------------------------
// A warp moves kFrames rows in units of kUnit bytes, which every row's address is a multiple
// of. `from` and `to` are the first row's slab.
struct Rows {
    uint32_t pitch;
    int bytes;  // of the slab's row: less than kRow in the last slab
};

template <int kUnit> __device__ __forceinline__ void copy_unit(char* to, const char* from) {
    if constexpr (kUnit == 2) {
        *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
    } else {
        const uint32_t s = static_cast<uint32_t>(__cvta_generic_to_shared(to));
        if constexpr (kUnit == 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(s), "l"(from) : "memory");
        else
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(s), "l"(from) : "memory");
    }
}

// The first `rows` rows; the others hold `fill`.
template <int kUnit>
__device__ __forceinline__ void fetch(char* to, const void* from, const Rows& at, int rows,
                                      uint32_t fill, int lane) {
    constexpr int kPerRow = kRow / kUnit;
#pragma unroll 2
    for (int j = 0; j < kFrames * kPerRow / kWarp; ++j) {
        const int u = j * kWarp + lane, row = u / kPerRow, byte = u % kPerRow * kUnit;
        if (row < rows) {
            if (byte < at.bytes)
                copy_unit<kUnit>(to + u * kUnit,
                                 static_cast<const char*>(from) + (row * at.pitch + byte));
        } else if constexpr (kUnit == 16) {
            *reinterpret_cast<uint4*>(to + u * kUnit) = make_uint4(fill, fill, fill, fill);
        } else if constexpr (kUnit == 4) {
            *reinterpret_cast<uint32_t*>(to + u * kUnit) = fill;
        } else {
            *reinterpret_cast<uint16_t*>(to + u * kUnit) = static_cast<uint16_t>(fill);
        }
    }
}

template <int kUnit>
__device__ __forceinline__ void store(void* to, const char* from, const Rows& at, int rows,
                                      int lane) {
    constexpr int kPerRow = kRow / kUnit;
    using Unit = std::conditional_t<kUnit == 16, uint4,
                                    std::conditional_t<kUnit == 4, uint32_t, uint16_t>>;
#pragma unroll 2
    for (int j = 0; j < kFrames * kPerRow / kWarp; ++j) {
        const int u = j * kWarp + lane, row = u / kPerRow, byte = u % kPerRow * kUnit;
        if (row < rows && byte < at.bytes)
            *reinterpret_cast<Unit*>(static_cast<char*>(to) + (row * at.pitch + byte)) =
                *reinterpret_cast<const Unit*>(from + u * kUnit);
    }
}

// Zeros in rows [from, to) of an utterance, of which this warp takes every `by`-th run of rows
// that one access of the warp covers.
template <int kUnit>
__device__ __forceinline__ void zero_rows(void* utterance, const Rows& at, int from, int to,
                                          int warp, int by, int lane) {
    constexpr int kPerRow = kRow / kUnit, kRun = kPerRow < kWarp ? kWarp / kPerRow : 1;
    using Unit = std::conditional_t<kUnit == 16, uint4,
                                    std::conditional_t<kUnit == 4, uint32_t, uint16_t>>;
    for (int t = from + warp * kRun; t < to; t += by * kRun) {
#pragma unroll
        for (int u = lane; u < kRun * kPerRow; u += kWarp) {
            const int row = t + u / kPerRow, byte = u % kPerRow * kUnit;
            if (row < to && byte < at.bytes)
                *reinterpret_cast<Unit*>(static_cast<char*>(utterance) +
                                         row * static_cast<int64_t>(at.pitch) + byte) = Unit{};
        }
    }
}

__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest group have arrived, for every lane of the warp.
__device__ __forceinline__ void arrived() {
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
}

struct Geometry {
    int length, channels, chunks;
    int slabs;    // of kRow bytes
    int cluster;  // blocks that share an utterance's slab
    int tiles;    // consecutive tiles of a block in a round of the cluster
};

// What a thread works on.
template <typename T> struct Place {
    int n, m, channel, rank, warp, lane;
    int64_t first;  // the utterance's first row at the slab, in elements
    Rows rows;
    __device__ Place(const Geometry& g, const int32_t* lengths) {
        warp = threadIdx.x / kWarp;
        lane = threadIdx.x % kWarp;
        rank = blockIdx.x % g.cluster;
        const int unit = blockIdx.x / g.cluster;
        n = unit / g.slabs;
        const int slab = unit % g.slabs * (kRow / static_cast<int>(sizeof(T)));
        channel = slab + lane * Lane<T>::kVec;
        m = min(max(lengths[n], 0), g.length);
        rows.pitch = static_cast<uint32_t>(g.channels) * sizeof(T);
        first = static_cast<int64_t>(n) * g.length * g.channels + slab;
        rows.bytes = min(kRow, (g.channels - slab) * static_cast<int>(sizeof(T)));
    }
};

// A lane's values of an [.., C] f32 row at the slab; channels past the last are skipped.
template <int kVec>
__device__ __forceinline__ void read_state(float* v, const float* row, int channel, int channels) {
#pragma unroll
    for (int i = 0; i < kVec; ++i) v[i] = row != nullptr && channel + i < channels ? row[channel + i] : 0.0f;
}
template <int kVec>
__device__ __forceinline__ void write_state(float* row, const float* v, int channel, int channels) {
#pragma unroll
    for (int i = 0; i < kVec; ++i)
        if (channel + i < channels) row[channel + i] = v[i];
}

// What the warps of a block and the blocks of a cluster tell one another. Two of each in turn,
// so that one barrier a tile (or a round) is enough.
struct Runs {
    float2 warp[2][kWarps][2 * kWarp];  // (A, B)
    float back[2][kWarps][2 * kWarp];   // B of the carry (backward)
    float behind[2][2 * kWarp];         // the state (forward) or carry (backward) after the tile
};
struct ClusterRuns {
    float2 block[2][kMaxCluster][2 * kWarp];
};

// Dynamic shared memory: each warp's stages of rows, Runs, and in a cluster ClusterRuns.
constexpr int kForwardStage = 2 * kFrames * kRow, kBackwardStage = 3 * kFrames * kRow;
constexpr int smem_bytes(int stage, bool cluster) {
    return 2 * kWarps * stage + static_cast<int>(sizeof(Runs)) +
           (cluster ? static_cast<int>(sizeof(ClusterRuns)) : 0);
}

// This block's share of a round of the cluster, in frames.
struct Range {
    int begin, end;
    __device__ Range(const Geometry& g, int m, int rank, int round_start) {
        if (g.cluster == 1) {
            begin = 0;
            end = m;
        } else {
            begin = round_start + rank * g.tiles * kTile;
            end = max(begin, min(m, begin + g.tiles * kTile));
        }
    }
};

// (A, B) of this block's frames to every block of the cluster, from those of its warps'
// consecutive parts in runs.warp[turn]: in the order of time, or against it. Returns once all
// have arrived in others.block[which].
template <int kVec, bool kBack>
__device__ __forceinline__ void exchange(const Runs& runs, ClusterRuns& others, int turn,
                                         int which, int rank, int warp, int state,
                                         int cluster_size) {
    auto cluster = cg::this_cluster();
    __syncthreads();
    float a[kVec], b[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) a[v] = 1.0f, b[v] = 0.0f;
    for (int i = 0; i < kWarps; ++i)
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            const float2 r = runs.warp[turn][kBack ? kWarps - 1 - i : i][state + v];
            b[v] = fmaf(r.x, b[v], r.y);
            a[v] *= r.x;
        }
    for (int q = warp; q < cluster_size; q += kWarps) {
        float2* there = cluster.map_shared_rank(&others.block[which][rank][0], q);
#pragma unroll
        for (int v = 0; v < kVec; ++v) there[state + v] = make_float2(a[v], b[v]);
    }
    cluster.sync();
}

template <typename T, int kUnit>
__global__ void __launch_bounds__(kWarps* kWarp, kForwardBlocks) recurrence_kernel(
    const T* __restrict__ x, const T* __restrict__ gate, const int32_t* __restrict__ lengths,
    const float* initial, T* __restrict__ out, float* final_state, float* __restrict__ states,
    Geometry geo) {
    using L = Lane<T>;
    using Raw = typename L::Raw;
    constexpr int kVec = L::kVec;
    extern __shared__ __align__(16) char smem[];
    Runs& runs = *reinterpret_cast<Runs*>(smem + 2 * kWarps * kForwardStage);
    ClusterRuns& others = *reinterpret_cast<ClusterRuns*>(&runs + 1);

    const Place<T> at(geo, lengths);
    char* stage = smem + at.warp * 2 * kForwardStage;
    const int last_warp = blockDim.x / kWarp - 1, state = at.lane * kVec;
    const int64_t state_row = static_cast<int64_t>(at.n) * geo.channels;
    float* saved = states == nullptr
                       ? nullptr
                       : states + static_cast<int64_t>(at.n) * geo.chunks * geo.channels;

    // Rows [t, end) to a stage.
    auto fetch_rows = [&](int t, int end, int which) {
        const int64_t here = at.first + t * static_cast<int64_t>(geo.channels);
        char* to = stage + which * kForwardStage;
        fetch<kUnit>(to, x + here, at.rows, end - t, 0u, at.lane);
        // An infinite gate keeps the state.
        fetch<kUnit>(to + kFrames * kRow, gate + here, at.rows, end - t, L::kInfinity, at.lane);
    };
    float carry[kVec];  // before the round
    read_state<kVec>(carry, initial == nullptr ? nullptr : initial + state_row, at.channel,
                     geo.channels);
    // Every block of the cluster runs, and has read its state, before any writes to another.
    if (geo.cluster > 1) cg::this_cluster().sync();

    int turn = 0, which = 0;
    const int round = geo.cluster == 1 ? geo.length : geo.cluster * geo.tiles * kTile;
    for (int round_start = 0; round_start < at.m; round_start += round, which ^= 1) {
        const Range range(geo, at.m, at.rank, round_start);
        float h[kVec];
        if (geo.cluster > 1) {
            // This warp's part of the range, for its (A, B) alone.
            const int part = geo.tiles * kFrames, from = range.begin + at.warp * part;
            const int to = min(range.end, from + part);
            float a[kVec], b[kVec];
#pragma unroll
            for (int v = 0; v < kVec; ++v) a[v] = 1.0f, b[v] = 0.0f;
            if (from < to) fetch_rows(from, to, 0);
            commit();
            for (int t = from, s = 0; t < to; t += kFrames, s ^= 1) {
                if (t + kFrames < to) fetch_rows(t + kFrames, to, s ^ 1);
                commit();
                arrived();
                const char* rows = stage + s * kForwardStage;
#pragma unroll
                for (int i = 0; i < kFrames; ++i) {
                    float xv[kVec], gv[kVec];
                    L::unpack(reinterpret_cast<const Raw*>(rows + i * kRow)[at.lane], xv);
                    L::unpack(reinterpret_cast<const Raw*>(rows + (kFrames + i) * kRow)[at.lane], gv);
#pragma unroll
                    for (int v = 0; v < kVec; ++v) {
                        float f, p;
                        gates(gv[v], f, p);
                        a[v] *= f;
                        b[v] = fmaf(f, b[v], p * xv[v]);
                    }
                }
                __syncwarp();
            }
#pragma unroll
            for (int v = 0; v < kVec; ++v)
                runs.warp[turn][at.warp][state + v] = make_float2(a[v], b[v]);
            exchange<kVec, false>(runs, others, turn, which, at.rank, at.warp, state, geo.cluster);
            for (int q = 0; q < geo.cluster; ++q)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = others.block[which][q][state + v];
                    if (q == at.rank) h[v] = carry[v];
                    carry[v] = fmaf(r.x, carry[v], r.y);
                }
        } else {
#pragma unroll
            for (int v = 0; v < kVec; ++v) h[v] = carry[v];
        }
        if (at.warp == 0)
#pragma unroll
            for (int v = 0; v < kVec; ++v) runs.behind[turn ^ 1][state + v] = h[v];

        const int mine = range.begin + at.warp * kFrames;
        if (mine < range.end) fetch_rows(mine, range.end, turn);
        else fetch_rows(0, 0, turn);
        commit();
        for (int start = range.begin; start < range.end; start += kTile, turn ^= 1) {
            const int t0 = start + at.warp * kFrames;
            if (start + kTile < range.end) fetch_rows(t0 + kTile, range.end, turn ^ 1);
            commit();
            arrived();
            char* rows = stage + turn * kForwardStage;
            // After each frame: the product of f, and h from 0.
            float a[kFrames][kVec], b[kFrames][kVec];
#pragma unroll
            for (int i = 0; i < kFrames; ++i) {
                float xv[kVec], gv[kVec];
                L::unpack(reinterpret_cast<const Raw*>(rows + i * kRow)[at.lane], xv);
                L::unpack(reinterpret_cast<const Raw*>(rows + (kFrames + i) * kRow)[at.lane], gv);
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    float f, p;
                    gates(gv[v], f, p);
                    a[i][v] = i == 0 ? f : a[i - 1][v] * f;
                    b[i][v] = i == 0 ? p * xv[v] : fmaf(f, b[i - 1][v], p * xv[v]);
                }
            }
#pragma unroll
            for (int v = 0; v < kVec; ++v)
                runs.warp[turn][at.warp][state + v] =
                    make_float2(a[kFrames - 1][v], b[kFrames - 1][v]);
            __syncthreads();
#pragma unroll
            for (int v = 0; v < kVec; ++v) h[v] = runs.behind[turn ^ 1][state + v];
            // The tile starts at a saved state.
            if (saved != nullptr && at.warp == 0)
                write_state<kVec>(saved + start / kChunk * static_cast<int64_t>(geo.channels), h,
                                  at.channel, geo.channels);
            for (int w = 0; w < at.warp; ++w)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = runs.warp[turn][w][state + v];
                    h[v] = fmaf(r.x, h[v], r.y);
                }
            // The outputs take the place of x.
            float hv[kVec];
#pragma unroll
            for (int i = 0; i < kFrames; ++i) {
#pragma unroll
                for (int v = 0; v < kVec; ++v) hv[v] = fmaf(a[i][v], h[v], b[i][v]);
                reinterpret_cast<Raw*>(rows + i * kRow)[at.lane] = L::pack(hv);
            }
            if (at.warp == last_warp) {
#pragma unroll
                for (int v = 0; v < kVec; ++v) runs.behind[turn][state + v] = hv[v];
                if (geo.cluster == 1)
#pragma unroll
                    for (int v = 0; v < kVec; ++v) carry[v] = hv[v];
            }
            __syncwarp();
            store<kUnit>(out + at.first + t0 * static_cast<int64_t>(geo.channels), rows, at.rows,
                         range.end - t0, at.lane);
            __syncwarp();
        }
    }
    if (at.rank == 0 && at.warp == last_warp)
        write_state<kVec>(final_state + state_row, carry, at.channel, geo.channels);
    const int index = at.rank * (last_warp + 1) + at.warp, by = geo.cluster * (last_warp + 1);
    zero_rows<kUnit>(out + at.first, at.rows, at.m, geo.length, index, by, at.lane);
    if (saved != nullptr) {
        const float zero[2] = {0.0f, 0.0f};
        for (int j = (at.m + kChunk - 1) / kChunk + index; j < geo.chunks; j += by)
            write_state<kVec>(saved + j * static_cast<int64_t>(geo.channels), zero, at.channel,
                              geo.channels);
    }
}

template <typename T, int kUnit>
__global__ void __launch_bounds__(kWarps* kWarp, kBackwardBlocks) recurrence_backward_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const T* __restrict__ gate,
    const int32_t* __restrict__ lengths, const float* __restrict__ states,
    const float* __restrict__ dfinal, T* __restrict__ dx, T* __restrict__ dgate,
    float* __restrict__ dinitial, Geometry geo) {
    using L = Lane<T>;
    using Raw = typename L::Raw;
    constexpr int kVec = L::kVec;
    extern __shared__ __align__(16) char smem[];
    Runs& runs = *reinterpret_cast<Runs*>(smem + 2 * kWarps * kBackwardStage);
    ClusterRuns& others = *reinterpret_cast<ClusterRuns*>(&runs + 1);

    const Place<T> at(geo, lengths);
    char* stage = smem + at.warp * 2 * kBackwardStage;
    const int last_warp = blockDim.x / kWarp - 1, state = at.lane * kVec;
    const int64_t state_row = static_cast<int64_t>(at.n) * geo.channels;
    const float* saved = states + static_cast<int64_t>(at.n) * geo.chunks * geo.channels;

    // Rows [t, end) to a stage: x, gate, dout; the scan for (A, B) alone needs no x.
    auto fetch_rows = [&](int t, int end, int which, bool with_x) {
        const int64_t here = at.first + t * static_cast<int64_t>(geo.channels);
        char* to = stage + which * kBackwardStage;
        if (with_x) fetch<kUnit>(to, x + here, at.rows, end - t, 0u, at.lane);
        fetch<kUnit>(to + kFrames * kRow, gate + here, at.rows, end - t, L::kInfinity, at.lane);
        fetch<kUnit>(to + 2 * kFrames * kRow, dout + here, at.rows, end - t, 0u, at.lane);
    };
    float carry[kVec];  // behind the round
    read_state<kVec>(carry, dfinal == nullptr ? nullptr : dfinal + state_row, at.channel,
                     geo.channels);
    if (geo.cluster > 1) cg::this_cluster().sync();

    int turn = 0, which = 0;
    const int round = geo.cluster == 1 ? geo.length : geo.cluster * geo.tiles * kTile;
    for (int round_start = at.m > 0 ? (at.m - 1) / round * round : -1; round_start >= 0;
         round_start -= round, which ^= 1) {
        const Range range(geo, at.m, at.rank, round_start);
        float c[kVec];
        if (geo.cluster > 1) {
            const int part = geo.tiles * kFrames, from = range.begin + at.warp * part;
            const int to = min(range.end, from + part);
            float a[kVec], b[kVec];
#pragma unroll
            for (int v = 0; v < kVec; ++v) a[v] = 1.0f, b[v] = 0.0f;
            const int last = from + (to - from - 1) / kFrames * kFrames;
            if (from < to) fetch_rows(last, to, 0, false);
            commit();
            for (int t = from < to ? last : from - 1, s = 0; t >= from; t -= kFrames, s ^= 1) {
                if (t > from) fetch_rows(t - kFrames, to, s ^ 1, false);
                commit();
                arrived();
                const char* rows = stage + s * kBackwardStage;
#pragma unroll
                for (int i = kFrames - 1; i >= 0; --i) {
                    float gv[kVec], dv[kVec];
                    L::unpack(reinterpret_cast<const Raw*>(rows + (kFrames + i) * kRow)[at.lane], gv);
                    L::unpack(reinterpret_cast<const Raw*>(rows + (2 * kFrames + i) * kRow)[at.lane],
                              dv);
#pragma unroll
                    for (int v = 0; v < kVec; ++v) {
                        float f, p;
                        gates(gv[v], f, p);
                        a[v] *= f;
                        b[v] = f * (dv[v] + b[v]);
                    }
                }
                __syncwarp();
            }
#pragma unroll
            for (int v = 0; v < kVec; ++v)
                runs.warp[turn][at.warp][state + v] = make_float2(a[v], b[v]);
            exchange<kVec, true>(runs, others, turn, which, at.rank, at.warp, state, geo.cluster);
            for (int q = geo.cluster - 1; q >= 0; --q)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = others.block[which][q][state + v];
                    if (q == at.rank) c[v] = carry[v];
                    carry[v] = fmaf(r.x, carry[v], r.y);
                }
        } else {
#pragma unroll
            for (int v = 0; v < kVec; ++v) c[v] = carry[v];
        }
        if (at.warp == 0)
#pragma unroll
            for (int v = 0; v < kVec; ++v) runs.behind[turn ^ 1][state + v] = c[v];

        const int tiles = (range.end - range.begin + kTile - 1) / kTile;
        const int last = range.begin + (tiles - 1) * kTile;
        if (tiles > 0 && last + at.warp * kFrames < range.end)
            fetch_rows(last + at.warp * kFrames, range.end, turn, true);
        else
            fetch_rows(0, 0, turn, true);
        commit();
        for (int i = 0, start = last; i < tiles; ++i, start -= kTile, turn ^= 1) {
            const int t0 = start + at.warp * kFrames;
            float h[kVec];  // the saved state before the tile
            read_state<kVec>(h, saved + start / kChunk * static_cast<int64_t>(geo.channels),
                             at.channel, geo.channels);
            if (i + 1 < tiles) fetch_rows(t0 - kTile, range.end, turn ^ 1, true);
            commit();
            arrived();
            char* rows = stage + turn * kBackwardStage;
            float f[kFrames][kVec], p[kFrames][kVec];
            float a[kVec], b[kVec], back[kVec];
#pragma unroll
            for (int v = 0; v < kVec; ++v) a[v] = 1.0f, b[v] = 0.0f, back[v] = 0.0f;
#pragma unroll
            for (int i = 0; i < kFrames; ++i) {
                float xv[kVec], gv[kVec];
                L::unpack(reinterpret_cast<const Raw*>(rows + i * kRow)[at.lane], xv);
                L::unpack(reinterpret_cast<const Raw*>(rows + (kFrames + i) * kRow)[at.lane], gv);
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    gates(gv[v], f[i][v], p[i][v]);
                    a[v] *= f[i][v];
                    b[v] = fmaf(f[i][v], b[v], p[i][v] * xv[v]);
                }
            }
#pragma unroll
            for (int i = kFrames - 1; i >= 0; --i) {
                float dv[kVec];
                L::unpack(reinterpret_cast<const Raw*>(rows + (2 * kFrames + i) * kRow)[at.lane], dv);
#pragma unroll
                for (int v = 0; v < kVec; ++v) back[v] = f[i][v] * (dv[v] + back[v]);
            }
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                runs.warp[turn][at.warp][state + v] = make_float2(a[v], b[v]);
                runs.back[turn][at.warp][state + v] = back[v];
            }
            __syncthreads();
            for (int w = 0; w < at.warp; ++w)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = runs.warp[turn][w][state + v];
                    h[v] = fmaf(r.x, h[v], r.y);
                }
#pragma unroll
            for (int v = 0; v < kVec; ++v) c[v] = runs.behind[turn ^ 1][state + v];
            for (int w = last_warp; w > at.warp; --w)
#pragma unroll
                for (int v = 0; v < kVec; ++v)
                    c[v] = fmaf(runs.warp[turn][w][state + v].x, c[v],
                                runs.back[turn][w][state + v]);
            float away[kFrames][kVec];  // h[t-1] - x[t]
#pragma unroll
            for (int i = 0; i < kFrames; ++i) {
                float xv[kVec];
                L::unpack(reinterpret_cast<const Raw*>(rows + i * kRow)[at.lane], xv);
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    away[i][v] = h[v] - xv[v];
                    h[v] = fmaf(f[i][v], h[v], p[i][v] * xv[v]);
                }
            }
            // dx takes the place of x, dgate that of gate.
#pragma unroll
            for (int i = kFrames - 1; i >= 0; --i) {
                float gx[kVec], gg[kVec];
                L::unpack(reinterpret_cast<const Raw*>(rows + (2 * kFrames + i) * kRow)[at.lane], gx);
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float total = gx[v] + c[v];
                    gx[v] = p[i][v] * total;
                    gg[v] = f[i][v] * gx[v] * away[i][v];
                    c[v] = f[i][v] * total;
                }
                reinterpret_cast<Raw*>(rows + i * kRow)[at.lane] = L::pack(gx);
                reinterpret_cast<Raw*>(rows + (kFrames + i) * kRow)[at.lane] = L::pack(gg);
            }
            if (at.warp == 0) {
#pragma unroll
                for (int v = 0; v < kVec; ++v) runs.behind[turn][state + v] = c[v];
                if (geo.cluster == 1)
#pragma unroll
                    for (int v = 0; v < kVec; ++v) carry[v] = c[v];
            }
            __syncwarp();
            const int64_t here = at.first + t0 * static_cast<int64_t>(geo.channels);
            store<kUnit>(dx + here, rows, at.rows, range.end - t0, at.lane);
            store<kUnit>(dgate + here, rows + kFrames * kRow, at.rows, range.end - t0, at.lane);
            __syncwarp();
        }
    }
    if (at.rank == 0 && at.warp == 0)
        write_state<kVec>(dinitial + state_row, carry, at.channel, geo.channels);
    const int index = at.rank * (last_warp + 1) + at.warp, by = geo.cluster * (last_warp + 1);
    for (T* grad : {dx, dgate})
        zero_rows<kUnit>(grad + at.first, at.rows, at.m, geo.length, index, by, at.lane);
}

// ---- launch --------------------------------------------------------------------------------

constexpr int64_t kClusterBlocks = 1, kRoundBytes = 32 << 20;

struct Shape {
    Geometry geo;
    int blocks, threads;
};

Shape shape_of(int batch, int length, int channels, int chunks, int row_channels) {
    Shape s{};
    const int slabs = (channels + row_channels - 1) / row_channels;
    const int64_t units = static_cast<int64_t>(batch) * slabs;
    const int64_t wanted = (kClusterBlocks * sm_count() + units - 1) / units;
    int cluster = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>(wanted, std::min(chunks, kMaxCluster))));
    // Rounds whose rows stay in L2 from the first reading to the second.
    const int64_t most = std::max<int64_t>(1, kRoundBytes / (units * cluster * kTile * kRow));
    const int64_t each = (chunks + cluster - 1) / cluster, rounds = (each + most - 1) / most;
    const int tiles = static_cast<int>((each + rounds - 1) / rounds);
    s.geo = {length, channels, chunks, slabs, cluster, tiles};
    s.blocks = static_cast<int>(units * cluster);
    s.threads = std::min(kWarps, (length + kFrames - 1) / kFrames) * kWarp;
    return s;
}

template <typename... Params, typename... Args>
cudaError_t launch(SmemAttr& attribute, void (*kernel)(Params...), const Shape& s, int stage,
                   cudaStream_t stream, Args... args) {
    const void* entry = reinterpret_cast<const void*>(kernel);
    cudaError_t e = attribute.ensure(entry, smem_bytes(stage, true));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(s.blocks));
    cfg.blockDim = dim3(static_cast<unsigned>(s.threads));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem_bytes(stage, s.geo.cluster > 1));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(s.geo.cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = s.geo.cluster > 1 ? 1 : 0;
    if (s.geo.cluster > 8) {
        e = cudaFuncSetAttribute(entry, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The widest unit that divides every row's address: 16 bytes, 4, or an element.
int unit_of(int64_t pitch, std::initializer_list<const void*> buffers) {
    uintptr_t all = static_cast<uintptr_t>(pitch);
    for (const void* b : buffers) all |= reinterpret_cast<uintptr_t>(b);
    return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
}

template <typename T, int kUnit> cudaError_t forward(const RecurrenceProblem& p, cudaStream_t s) {
    static SmemAttr attribute;
    const Shape shape = shape_of(p.batch, p.length, p.channels, p.chunks, kRow / sizeof(T));
    return launch(attribute, recurrence_kernel<T, kUnit>, shape, kForwardStage, s,
                  static_cast<const T*>(p.x), static_cast<const T*>(p.gate), p.valid_lengths,
                  p.initial_state, static_cast<T*>(p.output), p.final_state, p.states, shape.geo);
}

template <typename T, int kUnit>
cudaError_t backward(const RecurrenceBackwardProblem& p, cudaStream_t s) {
    static SmemAttr attribute;
    const Shape shape = shape_of(p.batch, p.length, p.channels, p.chunks, kRow / sizeof(T));
    return launch(attribute, recurrence_backward_kernel<T, kUnit>, shape, kBackwardStage, s,
                  static_cast<const T*>(p.grad_output), static_cast<const T*>(p.x),
                  static_cast<const T*>(p.gate), p.valid_lengths, p.states, p.grad_final_state,
                  static_cast<T*>(p.grad_x), static_cast<T*>(p.grad_gate), p.grad_initial_state,
                  shape.geo);
}

template <typename T> cudaError_t forward(const RecurrenceProblem& p, cudaStream_t s) {
    const int unit = unit_of(p.channels * static_cast<int64_t>(sizeof(T)), {p.x, p.gate, p.output});
    if (unit == 16) return forward<T, 16>(p, s);
    if constexpr (sizeof(T) == 2)
        if (unit == 2) return forward<T, 2>(p, s);
    return forward<T, 4>(p, s);
}

template <typename T> cudaError_t backward(const RecurrenceBackwardProblem& p, cudaStream_t s) {
    const int unit = unit_of(p.channels * static_cast<int64_t>(sizeof(T)),
                             {p.grad_output, p.x, p.gate, p.grad_x, p.grad_gate});
    if (unit == 16) return backward<T, 16>(p, s);
    if constexpr (sizeof(T) == 2)
        if (unit == 2) return backward<T, 2>(p, s);
    return backward<T, 4>(p, s);
}

}  // namespace

cudaError_t launch_recurrence(const RecurrenceProblem& p, cudaStream_t s, const char** variant) {
    *variant = "recurrence";
    if (p.dtype == FGA_FLOAT) return forward<float>(p, s);
    if (p.dtype == FGA_HALF) return forward<__half>(p, s);
    return forward<__nv_bfloat16>(p, s);
}

cudaError_t launch_recurrence_backward(const RecurrenceBackwardProblem& p, cudaStream_t s,
                                       const char** variant) {
    *variant = "recurrence-backward";
    if (p.dtype == FGA_FLOAT) return backward<float>(p, s);
    if (p.dtype == FGA_HALF) return backward<__half>(p, s);
    return backward<__nv_bfloat16>(p, s);
}

}  // namespace fga
