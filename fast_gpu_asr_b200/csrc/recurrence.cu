// Gated linear recurrence over [N, T, C], forward and backward:
//   f = sigmoid(gate), p = 1 - f, h[t] = f[t] h[t-1] + p[t] x[t];
//   G[t] = dout[t] + f[t+1] G[t+1] (+ dfinal at the last valid frame),
//   dx[t] = p[t] G[t], dgate[t] = f[t] p[t] (h[t-1] - x[t]) G[t], dinitial = f[0] G[0].
//
// A run of frames takes h to A h + B, with A the product of its f and B what it makes of
// h = 0, and runs compose: that is the scan, and the backward pass is the same scan against
// time for the carry c[t] = f[t] G[t]. A warp works on consecutive frames of a 128-byte row's
// channels (a lane one value of f32, two of a 16-bit type).
//
// A block walks the tiles of one utterance's slab of channels; its warps take kFrames frames of
// the tile each, find their (A, B), learn the state before their first frame from the warps
// before them, and finish from registers, so that no element is read twice. The next tile's
// rows are on their way to shared memory meanwhile. The backward pass recomputes h from the
// states that the forward pass saved every 64 frames.
//
// Bound by HBM where there are walks enough: 256 x 375 x 1024 ragged, forward bf16 72.7 us (90 %
// of a plain copy's rate for the bytes it cannot do without), backward f16 130 us (87 %). What
// is next is instruction issue (68 and 63 % busy, 48 instructions a pair of values forward and 82
// backward), which is why pairs go through the f32x2 instructions.
//
// Where utterances and channels are too few to fill the GPU, several blocks divide an
// utterance's tiles: a first launch leaves the (A, B) of each block's frames in the workspace,
// and a block of the second starts from what those before it make of the state. That reads the
// inputs twice, the second time from L2 where they fit: 2 x 12000 x 512, 24000 frames in 16
// walks: forward f16 with saved states 26.8 us, backward bf16 35.5 us; 168 and 284
// undivided.
#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "../../include/fga_convolution.h"
#include "f32x2.cuh"
#include "fga_common.cuh"
#include "fga_kernels.h"
#include "host_util.h"

namespace fga {
namespace {

constexpr int kChunk = FGA_RECURRENCE_STATE_FRAMES;
constexpr int kRow = 128;   // bytes of a row that a warp takes
constexpr int kFrames = 8;  // rows that a warp moves at a time
// In shared memory a row has room for where it starts in its first 16 bytes, unless all rows
// start at a multiple of 16.
template <int kUnit> constexpr int kPitch = kUnit == 16 ? kRow : kRow + 16;
template <int kUnit> constexpr int kRows = kFrames * kPitch<kUnit>;

// ---- a lane's four bytes of a row ----------------------------------------------------------
using fga::add2;
using fga::fma2;
using fga::mul2;
__device__ __forceinline__ float fma2(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float mul2(float a, float b) { return a * b; }
__device__ __forceinline__ float add2(float a, float b) { return a + b; }

template <typename T> struct Lane {
    static constexpr int kVec = 2;
    using Value = float2;
    using Raw = uint32_t;
    static __device__ __forceinline__ Value unpack(Raw r) { return unpack2<T>(r); }
    static __device__ __forceinline__ Raw pack(Value v) { return pack2<T>(v); }
    static __device__ __forceinline__ Value all(float v) { return splat2(v); }
    static constexpr uint32_t kInfinity = std::is_same_v<T, __half> ? 0x7c007c00u : 0x7f807f80u;
};
template <> struct Lane<float> {
    static constexpr int kVec = 1;
    using Value = float;
    using Raw = float;
    static __device__ __forceinline__ Value unpack(Raw r) { return r; }
    static __device__ __forceinline__ Raw pack(Value v) { return v; }
    static __device__ __forceinline__ Value all(float v) { return v; }
    static constexpr uint32_t kInfinity = 0x7f800000u;
};

// f and p = 1 - f: e = exp(-gate), f = 1 / (1 + e), p = e f, so that neither is a difference of
// numbers next to 1. What is off is e: the product with log2 e rounds, which makes e, and with it
// the smaller of f and p, relatively off by up to |gate| 2^-24, besides some steps of the
// exponential and the reciprocal. That is 6 bits of an fp32 p at |gate| = 60, and nothing that
// 16 bits show. The exponent stops at 126, where f is the smallest normal number and p is 1; a
// NaN stays one.
__device__ __forceinline__ float stop(float exponent) {
    float e;
    asm("min.NaN.f32 %0, %1, 0f42fc0000;" : "=f"(e) : "f"(exponent));
    return e;
}
__device__ __forceinline__ void gates(float g, float& f, float& p) {
    const float e = exp2_approx(stop(g * -kLog2e));
    f = reciprocal_approx(1.0f + e);
    p = e * f;
}
__device__ __forceinline__ void gates(float2 g, float2& f, float2& p) {
    const float2 t = mul2(g, splat2(-kLog2e));
    const float2 e = make_float2(exp2_approx(stop(t.x)), exp2_approx(stop(t.y)));
    const float2 d = add2(e, splat2(1.0f));
    f = make_float2(reciprocal_approx(d.x), reciprocal_approx(d.y));
    p = mul2(e, f);
}

// ---- rows between global and shared memory -------------------------------------------------
// A warp moves kFrames rows of a slab at a time, 16 bytes an access. kUnit bytes, which every
// row's address is a multiple of, is 16, 4 or an element. Below 16 a row is fetched as the
// aligned words that hold it, and its values are read from where it starts in the first: the 32
// and 64 accesses a row that units of 4 and 2 bytes would take are what bounds a kernel then (30
// x 2223 x 589 bf16 ragged, backward: 709 us by elements, 173 so; 15 x 9490 x 275 f32, forward:
// 289 and 156).
struct Rows {
    uint32_t pitch;
    int bytes;            // of the slab's row: less than kRow in the last slab
    uint32_t lane_bytes;  // of this lane's first 16-byte unit, where there are four rows a warp
    bool lane_present;    // whether it lies within the row
    // The words of a block of rows that this lane fetches where rows start anywhere: from row 0,
    // kOutside if there is none. Only if all inputs start alike (`alike`).
    int word[3];
    bool alike;
    int length;  // frames of the utterance
};
constexpr int kOutside = INT32_MIN;
constexpr int kHalf = kFrames / 2;
static_assert(kHalf * kRow == kWarp * 16, "a warp's 16-byte units cover half of its rows");

template <int kUnit>
using Unit = std::conditional_t<kUnit == 16, uint4,
                                std::conditional_t<kUnit == 4, uint32_t, uint16_t>>;

// A tensor's rows of one utterance at the slab.
struct Source {
    const char* first;       // row 0's slab
    const char *begin, *end; // the utterance's bytes: nothing outside is read
    // Where row i of any kFrames rows that start at a multiple of kFrames begins in its first
    // aligned word.
    __device__ __forceinline__ uint32_t offset(const Rows& at, int i) const {
        return (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(first)) + i * at.pitch) & 15u;
    }
};
static_assert(kFrames * sizeof(uint16_t) % 16 == 0, "every kFrames rows start alike");

__device__ __forceinline__ void copy16(char* to, const char* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                     static_cast<uint32_t>(__cvta_generic_to_shared(to))),
                 "l"(from)
                 : "memory");
}

// Rows t and up, `rows` of them at most; the others hold `fill`.
template <int kUnit>
__device__ __forceinline__ void fetch(char* to, const Source& source, int t, const Rows& at,
                                      int rows, uint32_t fill, int lane) {
    const char* from = source.first + t * static_cast<int64_t>(at.pitch);
    if constexpr (kUnit == 16) {
        if (rows >= kFrames) {  // all but an utterance's last rows
            if (at.lane_present) {
                const char* p = from + at.lane_bytes;
                copy16(to + lane * 16, p);
                copy16(to + kHalf * kRow + lane * 16, p + kHalf * at.pitch);
            }
            return;
        }
    }
    if constexpr (kUnit < 16) {
        // All but the first and last rows, which may share a word with other memory.
        if (at.alike && rows >= kFrames && t > 0 && t + 2 * kFrames <= at.length) {
#pragma unroll
            for (int j = 0; j < 3; ++j)
                if (at.word[j] != kOutside)
                    copy16(to + (j * kWarp + lane) * 16, from + at.word[j]);
            return;
        }
    }
    constexpr int kWords = kPitch<kUnit> / 16;  // of a row
#pragma unroll
    for (int j = 0; j < (kFrames * kWords + kWarp - 1) / kWarp; ++j) {
        const int u = j * kWarp + lane, row = u / kWords, k = u % kWords;
        if (u >= kFrames * kWords) break;
        char* word = to + u * 16;
        if (row < rows) {
            const char* p = from + row * at.pitch;
            const char* w = p + k * 16;
            if constexpr (kUnit < 16) w -= reinterpret_cast<uintptr_t>(p) & 15u;
            if (w < p + at.bytes) {
                if (kUnit == 16 || (w >= source.begin && w + 16 <= source.end)) {
                    copy16(word, w);
                } else {
                    for (int b = 0; b < 16; b += kUnit)
                        if (w + b >= source.begin && w + b < source.end)
                            *reinterpret_cast<Unit<kUnit>*>(word + b) =
                                *reinterpret_cast<const Unit<kUnit>*>(w + b);
                }
            }
        } else {
            *reinterpret_cast<uint4*>(word) = make_uint4(fill, fill, fill, fill);
        }
    }
}

// The same rows back, where they start at a multiple of 16 bytes.
__device__ __forceinline__ void store(char* to, const char* from, const Rows& at, int rows,
                                      int lane) {
    if (rows >= kFrames) {
        if (at.lane_present) {
            char* p = to + at.lane_bytes;
            *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(from + lane * 16);
            *reinterpret_cast<uint4*>(p + kHalf * at.pitch) =
                *reinterpret_cast<const uint4*>(from + kHalf * kRow + lane * 16);
        }
        return;
    }
    constexpr int kWords = kRow / 16;
#pragma unroll
    for (int j = 0; j < kFrames * kWords / kWarp; ++j) {
        const int u = j * kWarp + lane, row = u / kWords, byte = u % kWords * 16;
        if (row < rows && byte < at.bytes)
            *reinterpret_cast<uint4*>(to + (row * at.pitch + byte)) =
                *reinterpret_cast<const uint4*>(from + u * 16);
    }
}

// Zeros in rows [from, to) of an utterance, of which this warp takes every `by`-th run of rows
// that one access of the warp covers.
template <int kUnit>
__device__ __forceinline__ void zero_rows(void* utterance, const Rows& at, int from, int to,
                                          int warp, int by, int lane) {
    constexpr int kPerRow = kRow / kUnit, kRun = kPerRow < kWarp ? kWarp / kPerRow : 1;
    for (int t = from + warp * kRun; t < to; t += by * kRun) {
#pragma unroll
        for (int u = lane; u < kRun * kPerRow; u += kWarp) {
            const int row = t + u / kPerRow, byte = u % kPerRow * kUnit;
            if (row < to && byte < at.bytes)
                *reinterpret_cast<Unit<kUnit>*>(static_cast<char*>(utterance) +
                                                row * static_cast<int64_t>(at.pitch) + byte) =
                    Unit<kUnit>{};
        }
    }
}

__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest kNewer groups have arrived, for every lane of the warp.
template <int kNewer> __device__ __forceinline__ void arrived() {
    asm volatile("cp.async.wait_group %0;" ::"n"(kNewer) : "memory");
    __syncwarp();
}

struct Geometry {
    int length, channels, chunks;
    int slabs;   // of kRow bytes
    int blocks;  // that divide an utterance's slab
    int span;    // frames of a block, whole tiles
};

// What a thread works on.
template <typename T> struct Place {
    int n, m, channel, unit, block, warp, lane, warps;
    int begin, end;  // the block's frames
    int64_t first;  // the utterance's first row at the slab, in elements
    int64_t state;  // of [N, C] at this lane's channel
    Rows rows;
    int present;    // how many of the lane's channels exist
    __device__ Place(const Geometry& g, const int32_t* lengths) {
        warp = threadIdx.x / kWarp;
        lane = threadIdx.x % kWarp;
        warps = blockDim.x / kWarp;
        unit = blockIdx.x / g.blocks;
        block = blockIdx.x - unit * g.blocks;
        n = unit / g.slabs;
        const int slab = (unit - n * g.slabs) * (kRow / static_cast<int>(sizeof(T)));
        channel = slab + lane * Lane<T>::kVec;
        present = g.channels - channel;
        m = min(max(lengths[n], 0), g.length);
        begin = block * g.span;
        end = max(begin, min(m, begin + g.span));
        rows.pitch = static_cast<uint32_t>(g.channels) * sizeof(T);
        rows.length = g.length;
        first = static_cast<int64_t>(n) * g.length * g.channels + slab;
        state = static_cast<int64_t>(n) * g.channels + channel;
        rows.bytes = min(kRow, (g.channels - slab) * static_cast<int>(sizeof(T)));
        rows.lane_bytes = lane / (kRow / 16) * rows.pitch + lane % (kRow / 16) * 16;
        rows.lane_present = lane % (kRow / 16) * 16 < rows.bytes;
    }
    // The block of the last valid frame, or the first where there is none.
    __device__ bool last_valid(const Geometry& g) const {
        return begin < m ? m <= begin + g.span : m == 0 && block == 0;
    }
    // Of [N, chunks, C] at this lane's channel.
    __device__ int64_t saved(const Geometry& g, int chunk) const {
        return (static_cast<int64_t>(n) * g.chunks + chunk) * g.channels + channel;
    }
};

__device__ __forceinline__ void read_state(float2& v, const float* at, int present) {
    v.x = at != nullptr && present > 0 ? at[0] : 0.0f;
    v.y = at != nullptr && present > 1 ? at[1] : 0.0f;
}
__device__ __forceinline__ void read_state(float& v, const float* at, int present) {
    v = at != nullptr && present > 0 ? at[0] : 0.0f;
}
__device__ __forceinline__ void write_state(float* at, float2 v, int present) {
    if (present > 0) at[0] = v.x;
    if (present > 1) at[1] = v.y;
}
__device__ __forceinline__ void write_state(float* at, float v, int present) {
    if (present > 0) at[0] = v;
}

template <typename V> struct alignas(2 * sizeof(V)) Run {
    V a, b;  // takes h to a h + b
    __device__ __forceinline__ V operator()(V h) const { return fma2(a, h, b); }
    // This one, and then the next.
    __device__ __forceinline__ void then(const Run& next) {
        b = next(b);
        a = mul2(a, next.a);
    }
};

template <typename T> struct Forward {
    const T* x;
    const T* gate;
    const int32_t* lengths;
    const float* initial;  // or null
    T* out;
    float* final_state;    // may be `initial`
    float* states;         // or null
    void* runs;            // [units, blocks, 32] Run; null for one block
    float* first;          // the initial state's copy, behind them
};

template <typename T> struct Backward {
    const T* dout;
    const T* x;
    const T* gate;
    const int32_t* lengths;
    const float* states;
    const float* dfinal;  // or null
    T* dx;
    T* dgate;
    float* dinitial;
    void* runs;
};

template <typename T>
__device__ __forceinline__ Source source_of(const T* tensor, const Place<T>& at,
                                            const Geometry& g) {
    const T* utterance = tensor + static_cast<int64_t>(at.n) * g.length * g.channels;
    return {reinterpret_cast<const char*>(tensor + at.first),
            reinterpret_cast<const char*>(utterance),
            reinterpret_cast<const char*>(utterance + static_cast<int64_t>(g.length) * g.channels)};
}
// The lane's words, if all of `sources` start alike.
template <int kUnit>
__device__ __forceinline__ void plan(Rows& at, std::initializer_list<Source> sources, int lane) {
    if constexpr (kUnit < 16) {
        at.alike = true;
        const Source& one = *sources.begin();
        for (const Source& s : sources) at.alike = at.alike && s.offset(at, 0) == one.offset(at, 0);
        constexpr int kWords = kPitch<kUnit> / 16;
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            const int u = j * kWarp + lane, row = u / kWords;
            const int in_row = u % kWords * 16 - static_cast<int>(one.offset(at, row));
            at.word[j] = row < kFrames && in_row < at.bytes
                             ? static_cast<int>(row * at.pitch) + in_row
                             : kOutside;
        }
    }
}
// The lane's values of row i of those that `source` was fetched from.
template <typename T, int kUnit>
__device__ __forceinline__ typename Lane<T>::Value value(const char* rows, int i,
                                                         const Source& source,
                                                         const Place<T>& at) {
    using Raw = typename Lane<T>::Raw;
    rows += i * kPitch<kUnit> + at.lane * 4;
    if constexpr (kUnit < 16) rows += source.offset(at.rows, i);
    if constexpr (kUnit == 2) {
        // Two aligned words hold them.
        const uint32_t odd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(rows)) & 2u;
        const uint32_t* words = reinterpret_cast<const uint32_t*>(rows - odd);
        return Lane<T>::unpack(__funnelshift_r(words[0], words[1], 8 * odd));
    } else {
        return Lane<T>::unpack(*reinterpret_cast<const Raw*>(rows));
    }
}
// Row i's values of an output: to `rows`, which `store` moves, or from here. `frame`: row 0's.
template <typename T, int kUnit>
__device__ __forceinline__ void put(T* tensor, char* rows, int frame, int i, const Place<T>& at,
                                    const Geometry& g, typename Lane<T>::Value v) {
    using Raw = typename Lane<T>::Raw;
    const Raw raw = Lane<T>::pack(v);
    if constexpr (kUnit == 16) {
        reinterpret_cast<Raw*>(rows + i * kRow)[at.lane] = raw;
    } else if (frame + i < at.end && at.present > 0) {
        T* to = tensor + at.first + (frame + i) * static_cast<int64_t>(g.channels) +
                at.lane * Lane<T>::kVec;
        if constexpr (kUnit == 2) {
            uint16_t* halves = reinterpret_cast<uint16_t*>(to);
            halves[0] = static_cast<uint16_t>(raw);
            if (at.present > 1) halves[1] = static_cast<uint16_t>(raw >> 16);
        } else {
            *reinterpret_cast<Raw*>(to) = raw;
        }
    }
}
template <typename T, int kUnit>
__device__ __forceinline__ void store_rows(T* tensor, const char* rows, int frame,
                                           const Place<T>& at) {
    if constexpr (kUnit == 16)
        store(reinterpret_cast<char*>(tensor + at.first) +
                  frame * static_cast<int64_t>(at.rows.pitch),
              rows, at.rows, at.end - frame, at.lane);
}

// The padding of an output and of the saved states; `index` and `by` number all warps that work
// on the slab.
template <int kUnit, typename T>
__device__ __forceinline__ void finish(const Forward<T>& f, const Place<T>& at, const Geometry& g) {
    const int index = at.block * at.warps + at.warp, by = g.blocks * at.warps;
    zero_rows<kUnit>(f.out + at.first, at.rows, at.m, g.length, index, by, at.lane);
    if (f.states != nullptr)
        for (int j = (at.m + kChunk - 1) / kChunk + index; j < g.chunks; j += by)
            write_state(f.states + at.saved(g, j), Lane<T>::all(0.0f), at.present);
}
template <int kUnit, typename T>
__device__ __forceinline__ void finish(const Backward<T>& f, const Place<T>& at, const Geometry& g) {
    const int index = at.block * at.warps + at.warp, by = g.blocks * at.warps;
    for (T* grad : {f.dx, f.dgate})
        zero_rows<kUnit>(grad + at.first, at.rows, at.m, g.length, index, by, at.lane);
}

// ---- the walk ------------------------------------------------------------------------------
// A tile is 64 frames: 8 warps of 8. More frames a warp need more registers than an SM has for
// the blocks that hide the memory's latency (16 measured 167 us where 8 take 79, 256 x 375 x
// 1024 bf16 ragged); fewer spend more on the scan across warps.
constexpr int kWarps = 8, kTile = kFrames * kWarps;
constexpr int kForwardBlocks = 4, kBackwardBlocks = 3;  // on a multiprocessor
static_assert(kTile == kChunk, "a tile starts at a saved state");

// What the warps tell one another, two of each in turn, so that one barrier a tile is enough. It
// starts a block's shared memory and ends with the last warp that the block has.
template <typename V> struct Tile {
    V behind[2][kWarp];  // the state (forward) or carry (backward) after the tile
    struct Warp {
        Run<V> run[2][kWarp];
        V back[2][kWarp];  // B of the carry (backward)
    } warp[kWarps];
    static constexpr int bytes(int warps) {
        return static_cast<int>(sizeof(behind) + warps * sizeof(Warp));
    }
};
template <int kUnit> constexpr int kForwardStage = 2 * kRows<kUnit>;
template <int kUnit> constexpr int kBackwardStage = 3 * kRows<kUnit>;
// Shared memory of a walk: no more than its warps and tiles need, since a streaming step's blocks
// are one warp each, and as many as a multiprocessor takes have to fit (20000 x 1 x 512 f16: 97
// us, 422 with room for eight warps and two tiles; 256 x 16 x 1024: 7 and 11).
template <typename V> constexpr int tile_smem(int stage, int warps, bool one_tile) {
    return Tile<V>::bytes(warps) + (one_tile ? 1 : 2) * warps * stage;
}

// What the blocks before this one make of `v`, or (kBack) those behind it: each warp composes a
// share of their runs, which the warps then compose.
template <bool kBack, typename V, typename T>
__device__ __forceinline__ V through_blocks(V v, const void* runs, Tile<V>& tile,
                                            const Place<T>& at, const Geometry& g) {
    const Run<V>* all =
        static_cast<const Run<V>*>(runs) + static_cast<int64_t>(at.unit) * g.blocks * kWarp + at.lane;
    const int count = kBack ? g.blocks - 1 - at.block : at.block;
    const int each = (count + kWarps - 1) / kWarps, from = at.warp * each;
    Run<V> run{Lane<T>::all(1.0f), Lane<T>::all(0.0f)};
#pragma unroll 4
    for (int i = from; i < min(count, from + each); ++i)
        run.then(all[(kBack ? g.blocks - 1 - i : i) * kWarp]);
    tile.warp[at.warp].run[1][at.lane] = run;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) v = tile.warp[w].run[1][at.lane](v);
    return v;
}

template <typename T, int kUnit>
__global__ void __launch_bounds__(kWarps* kWarp, kForwardBlocks)
    recurrence_kernel(Forward<T> f, Geometry geo) {
    using L = Lane<T>;
    using V = typename L::Value;
    extern __shared__ __align__(16) char smem[];
    constexpr int kStage = kForwardStage<kUnit>, kGate = kRows<kUnit>;
    Place<T> at(geo, f.lengths);
    const Source x = source_of(f.x, at, geo), gate = source_of(f.gate, at, geo);
    plan<kUnit>(at.rows, {x, gate}, at.lane);
    const int buffers = geo.length > kTile ? 2 : 1;
    Tile<V>& tile = *reinterpret_cast<Tile<V>*>(smem);
    char* stage = smem + Tile<V>::bytes(at.warps) + at.warp * buffers * kStage;
    const int last = at.warps - 1;

    auto fetch_tile = [&](int start, int which) {
        const int t = start + at.warp * kFrames;
        char* to = stage + which * kStage;
        fetch<kUnit>(to, x, t, at.rows, at.end - t, 0u, at.lane);
        // An infinite gate keeps the state.
        fetch<kUnit>(to + kGate, gate, t, at.rows, at.end - t, L::kInfinity, at.lane);
    };
    if (at.begin < at.end) fetch_tile(at.begin, 0);
    commit();
    V h;
    if (geo.blocks > 1) {
        cudaGridDependencySynchronize();
        read_state(h, f.first + at.state, at.present);
        h = through_blocks<false>(h, f.runs, tile, at, geo);
    } else {
        read_state(h, f.initial == nullptr ? nullptr : f.initial + at.state, at.present);
    }
    if (at.warp == 0) tile.behind[1][at.lane] = h;

    int turn = 0;
    for (int start = at.begin; start < at.end; start += kTile, turn ^= 1) {
        if (start + kTile < at.end) fetch_tile(start + kTile, turn ^ 1);
        commit();
        arrived<1>();
        char* rows = stage + turn * kStage;
        const int frame = start + at.warp * kFrames;
        Run<V> run[kFrames];  // from the warp's first frame to each of them
#pragma unroll
        for (int i = 0; i < kFrames; ++i) {
            V keep, take;
            gates(value<T, kUnit>(rows + kGate, i, gate, at), keep, take);
            const V add = mul2(take, value<T, kUnit>(rows, i, x, at));
            run[i].a = i == 0 ? keep : mul2(run[i - 1].a, keep);
            run[i].b = i == 0 ? add : fma2(keep, run[i - 1].b, add);
        }
        tile.warp[at.warp].run[turn][at.lane] = run[kFrames - 1];
        __syncthreads();
        h = tile.behind[turn ^ 1][at.lane];
        if (f.states != nullptr && at.warp == 0)
            write_state(f.states + at.saved(geo, start / kChunk), h, at.present);
        for (int w = 0; w < at.warp; ++w) h = tile.warp[w].run[turn][at.lane](h);
        // The outputs take the place of x.
        V after;
#pragma unroll
        for (int i = 0; i < kFrames; ++i) {
            after = run[i](h);
            put<T, kUnit>(f.out, rows, frame, i, at, geo, after);
        }
        h = after;
        if (at.warp == last) tile.behind[turn][at.lane] = h;
        __syncwarp();
        store_rows<T, kUnit>(f.out, rows, frame, at);
        __syncwarp();
    }
    if (at.warp == last && at.last_valid(geo)) write_state(f.final_state + at.state, h, at.present);
    finish<kUnit>(f, at, geo);
}

// (Two blocks a multiprocessor with units of 2 bytes: three would spill registers, 173 us against
// 196 in the case above.)
template <typename T, int kUnit>
__global__ void __launch_bounds__(kWarps* kWarp, kUnit == 2 ? 2 : kBackwardBlocks)
    recurrence_backward_kernel(Backward<T> f, Geometry geo) {
    using L = Lane<T>;
    using V = typename L::Value;
    extern __shared__ __align__(16) char smem[];
    constexpr int kStage = kBackwardStage<kUnit>, kGate = kRows<kUnit>, kDout = 2 * kRows<kUnit>;
    Place<T> at(geo, f.lengths);
    const Source x = source_of(f.x, at, geo), gate = source_of(f.gate, at, geo),
                 dout = source_of(f.dout, at, geo);
    plan<kUnit>(at.rows, {x, gate, dout}, at.lane);
    const int buffers = geo.length > kTile ? 2 : 1;
    Tile<V>& tile = *reinterpret_cast<Tile<V>*>(smem);
    char* stage = smem + Tile<V>::bytes(at.warps) + at.warp * buffers * kStage;
    const int last = at.warps - 1;

    auto fetch_tile = [&](int start, int which) {
        const int t = start + at.warp * kFrames;
        char* to = stage + which * kStage;
        fetch<kUnit>(to, x, t, at.rows, at.end - t, 0u, at.lane);
        fetch<kUnit>(to + kGate, gate, t, at.rows, at.end - t, L::kInfinity, at.lane);
        fetch<kUnit>(to + kDout, dout, t, at.rows, at.end - t, 0u, at.lane);
    };
    const int top = at.begin < at.end ? (at.end - 1) / kTile * kTile : -1;  // the last tile
    if (top >= 0) fetch_tile(top, 0);
    commit();
    V carry;
    read_state(carry, f.dfinal == nullptr ? nullptr : f.dfinal + at.state, at.present);
    if (geo.blocks > 1) {
        cudaGridDependencySynchronize();
        carry = through_blocks<true>(carry, f.runs, tile, at, geo);
    }
    if (at.warp == 0) tile.behind[1][at.lane] = carry;

    int turn = 0;
    for (int start = top; start >= at.begin; start -= kTile, turn ^= 1) {
        V h;
        read_state(h, f.states + at.saved(geo, start / kChunk), at.present);
        if (start > at.begin) fetch_tile(start - kTile, turn ^ 1);
        commit();
        arrived<1>();
        char* rows = stage + turn * kStage;
        const int frame = start + at.warp * kFrames;
        V keep[kFrames], take[kFrames], back = L::all(0.0f);
        Run<V> run{L::all(1.0f), L::all(0.0f)};
#pragma unroll
        for (int i = 0; i < kFrames; ++i) {
            gates(value<T, kUnit>(rows + kGate, i, gate, at), keep[i], take[i]);
            run.a = mul2(run.a, keep[i]);
            run.b = fma2(keep[i], run.b, mul2(take[i], value<T, kUnit>(rows, i, x, at)));
            back = fma2(run.a, value<T, kUnit>(rows + kDout, i, dout, at), back);
        }
        tile.warp[at.warp].run[turn][at.lane] = run;
        tile.warp[at.warp].back[turn][at.lane] = back;
        __syncthreads();
        for (int w = 0; w < at.warp; ++w) h = tile.warp[w].run[turn][at.lane](h);
        carry = tile.behind[turn ^ 1][at.lane];
        for (int w = last; w > at.warp; --w)
            carry = fma2(tile.warp[w].run[turn][at.lane].a, carry, tile.warp[w].back[turn][at.lane]);
        V away[kFrames];  // h[t-1] - x[t]
#pragma unroll
        for (int i = 0; i < kFrames; ++i) {
            const V v = value<T, kUnit>(rows, i, x, at);
            away[i] = fma2(v, L::all(-1.0f), h);
            h = fma2(keep[i], h, mul2(take[i], v));
        }
        // dx takes the place of x, dgate that of the gates.
#pragma unroll
        for (int i = kFrames - 1; i >= 0; --i) {
            const V total = add2(value<T, kUnit>(rows + kDout, i, dout, at), carry);
            const V gx = mul2(take[i], total);
            carry = mul2(keep[i], total);
            put<T, kUnit>(f.dx, rows, frame, i, at, geo, gx);
            put<T, kUnit>(f.dgate, rows + kGate, frame, i, at, geo,
                          mul2(mul2(keep[i], gx), away[i]));
        }
        if (at.warp == 0) tile.behind[turn][at.lane] = carry;
        __syncwarp();
        store_rows<T, kUnit>(f.dx, rows, frame, at);
        store_rows<T, kUnit>(f.dgate, rows + kGate, frame, at);
        __syncwarp();
    }
    if (at.warp == 0 && at.block == 0) write_state(f.dinitial + at.state, carry, at.present);
    finish<kUnit>(f, at, geo);
}

// ---- the first launch of a divided walk ----------------------------------------------------
// Each warp streams an eighth of the block's frames, kFrames at a time through a ring of stages,
// for their run alone: (A, B) of the state from x and gate, or (kBack) of the carry from dout
// and gate: c[first] = A c + sum over t of (f[first] .. f[t]) dout[t]. Three stages let four
// blocks stand on a multiprocessor (2 x 12000 x 512 f16, both launches: 26.8 us; four stages
// 30.0).
constexpr int kDepth = 3;
template <int kUnit> constexpr int kRing = kDepth * 2 * kRows<kUnit>;
template <typename V, int kUnit> constexpr int runs_smem() {
    return kWarps * (kRing<kUnit> + kWarp * static_cast<int>(sizeof(Run<V>)));
}

template <typename T, int kUnit, bool kBack>
__global__ void __launch_bounds__(kWarps* kWarp, 4)
    recurrence_runs_kernel(const T* __restrict__ input, const T* __restrict__ gate,
                           const int32_t* __restrict__ lengths, const float* initial, void* runs,
                           float* first, Geometry geo) {
    using L = Lane<T>;
    using V = typename L::Value;
    extern __shared__ __align__(16) char smem[];
    cudaTriggerProgrammaticLaunchCompletion();
    Place<T> at(geo, lengths);
    const Source from = source_of(input, at, geo), gate_from = source_of(gate, at, geo);
    plan<kUnit>(at.rows, {from, gate_from}, at.lane);
    constexpr int kGate = kRows<kUnit>;
    char* ring = smem + at.warp * kRing<kUnit>;
    Run<V>* warps = reinterpret_cast<Run<V>*>(smem + kWarps * kRing<kUnit>);
    const int part = geo.span / kWarps, begin = at.begin + at.warp * part;
    const int end = min(at.end, begin + part);
    const int steps = begin < end ? (end - begin + kFrames - 1) / kFrames : 0;
    auto request = [&](int i) {
        if (i < steps) {
            char* to = ring + i % kDepth * 2 * kGate;
            const int t = begin + i * kFrames;
            fetch<kUnit>(to, from, t, at.rows, end - t, 0u, at.lane);
            fetch<kUnit>(to + kGate, gate_from, t, at.rows, end - t, L::kInfinity, at.lane);
        }
        commit();
    };
#pragma unroll
    for (int i = 0; i < kDepth - 1; ++i) request(i);
    Run<V> run{L::all(1.0f), L::all(0.0f)};
    for (int i = 0; i < steps; ++i) {
        request(i + kDepth - 1);
        arrived<kDepth - 1>();
        const char* rows = ring + i % kDepth * 2 * kGate;
#pragma unroll
        for (int k = 0; k < kFrames; ++k) {
            V keep, take;
            gates(value<T, kUnit>(rows + kGate, k, gate_from, at), keep, take);
            const V v = value<T, kUnit>(rows, k, from, at);
            run.a = mul2(run.a, keep);
            run.b = kBack ? fma2(run.a, v, run.b) : fma2(keep, run.b, mul2(take, v));
        }
        __syncwarp();
    }
    warps[at.warp * kWarp + at.lane] = run;
    __syncthreads();
    if (at.warp == 0) {
        run = warps[(kBack ? kWarps - 1 : 0) * kWarp + at.lane];
        for (int w = 1; w < kWarps; ++w)
            run.then(warps[(kBack ? kWarps - 1 - w : w) * kWarp + at.lane]);
        static_cast<Run<V>*>(runs)[(static_cast<int64_t>(at.unit) * geo.blocks + at.block) * kWarp +
                                   at.lane] = run;
    }
    // The second launch may write the final state on top of the initial one.
    if (!kBack && at.warp == 1 && at.block == 0) {
        V h;
        read_state(h, initial == nullptr ? nullptr : initial + at.state, at.present);
        write_state(first + at.state, h, at.present);
    }
}

// ---- launch --------------------------------------------------------------------------------

struct Shape {
    Geometry geo;
    int64_t units;
    int warps;
    size_t runs_bytes, workspace;
};

// A walk of more than two tiles is divided below three blocks of it for every four
// multiprocessors: into as many as `resident` blocks on each of them take. (T = 3000, C = 1024,
// bf16, forward: 4 utterances, 64 walks, 26 us divided and 45 not; 8 utterances, 128 walks, 52
// and 46; backward 38 and 73, 71 and 75. C = 512 f16, one utterance: two tiles 4.8 divided and
// 3.9 not, three 4.8 and 5.0; backward 5.0 and 5.0, 5.2 and 6.6.)
Shape shape_of(int batch, int length, int channels, int chunks, int element, int resident) {
    const int slab = kRow / element;
    Shape s{};
    s.geo = {length, channels, chunks, (channels + slab - 1) / slab, 1, 0};
    s.units = static_cast<int64_t>(batch) * s.geo.slabs;
    int each = chunks;
    if (chunks > 2 && 4 * s.units < 3 * sm_count()) {
        const int64_t blocks = std::min<int64_t>(chunks, resident * sm_count() / s.units);
        each = static_cast<int>((chunks + blocks - 1) / blocks);
        s.geo.blocks = (chunks + each - 1) / each;
    }
    s.geo.span = each * kTile;
    s.warps = s.geo.blocks > 1 ? kWarps : std::min(kWarps, (length + kFrames - 1) / kFrames);
    if (s.geo.blocks > 1) {
        s.runs_bytes = static_cast<size_t>(s.units) * s.geo.blocks * kWarp *
                       (element == 4 ? sizeof(Run<float>) : sizeof(Run<float2>));
        s.workspace = s.runs_bytes + sizeof(float) * batch * channels;
    }
    return s;
}

template <typename... Params, typename... Args>
cudaError_t launch(SmemAttr& attribute, void (*kernel)(Params...), const Shape& s, int smem,
                   int most_smem, bool early, cudaStream_t stream, Args... args) {
    const cudaError_t e = attribute.ensure(reinterpret_cast<const void*>(kernel), most_smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(s.units * s.geo.blocks));
    cfg.blockDim = dim3(static_cast<unsigned>(s.warps * kWarp));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    // The kernel waits for the launch before it itself, after its first rows are on their way.
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = early ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The widest unit that divides every row's address: 16 bytes, 4, or an element.
int unit_of(int64_t pitch, std::initializer_list<const void*> buffers) {
    uintptr_t all = static_cast<uintptr_t>(pitch);
    for (const void* b : buffers) all |= reinterpret_cast<uintptr_t>(b);
    return all % 16 == 0 ? 16 : all % 4 == 0 ? 4 : 2;
}

Shape shape_of(const RecurrenceProblem& p) {
    return shape_of(p.batch, p.length, p.channels, p.chunks, p.dtype == FGA_FLOAT ? 4 : 2,
                    kForwardBlocks);
}
Shape shape_of(const RecurrenceBackwardProblem& p) {
    return shape_of(p.batch, p.length, p.channels, p.chunks, p.dtype == FGA_FLOAT ? 4 : 2,
                    kBackwardBlocks);
}

template <typename T, int kUnit> cudaError_t forward(const RecurrenceProblem& p, cudaStream_t s) {
    using V = typename Lane<T>::Value;
    static SmemAttr walk, runs;
    const Shape shape = shape_of(p);
    Forward<T> f{static_cast<const T*>(p.x), static_cast<const T*>(p.gate), p.valid_lengths,
                 p.initial_state, static_cast<T*>(p.output), p.final_state, p.states, nullptr,
                 nullptr};
    const bool divided = shape.geo.blocks > 1;
    if (divided) {
        f.runs = p.workspace;
        f.first = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + shape.runs_bytes);
        const cudaError_t e =
            launch(runs, recurrence_runs_kernel<T, kUnit, false>, shape, runs_smem<V, kUnit>(),
                   runs_smem<V, kUnit>(), false, s, f.x, f.gate, f.lengths, f.initial, f.runs,
                   f.first, shape.geo);
        if (e != cudaSuccess) return e;
    }
    constexpr int kStage = kForwardStage<kUnit>;
    return launch(walk, recurrence_kernel<T, kUnit>, shape,
                  tile_smem<V>(kStage, shape.warps, p.length <= kTile),
                  tile_smem<V>(kStage, kWarps, false), divided, s, f, shape.geo);
}

template <typename T, int kUnit>
cudaError_t backward(const RecurrenceBackwardProblem& p, cudaStream_t s) {
    using V = typename Lane<T>::Value;
    static SmemAttr walk, runs;
    const Shape shape = shape_of(p);
    const bool divided = shape.geo.blocks > 1;
    const Backward<T> f{static_cast<const T*>(p.grad_output), static_cast<const T*>(p.x),
                        static_cast<const T*>(p.gate), p.valid_lengths, p.states,
                        p.grad_final_state, static_cast<T*>(p.grad_x),
                        static_cast<T*>(p.grad_gate), p.grad_initial_state,
                        divided ? p.workspace : nullptr};
    if (divided) {
        const cudaError_t e =
            launch(runs, recurrence_runs_kernel<T, kUnit, true>, shape, runs_smem<V, kUnit>(),
                   runs_smem<V, kUnit>(), false, s, f.dout, f.gate, f.lengths,
                   static_cast<const float*>(nullptr), f.runs, static_cast<float*>(nullptr),
                   shape.geo);
        if (e != cudaSuccess) return e;
    }
    constexpr int kStage = kBackwardStage<kUnit>;
    return launch(walk, recurrence_backward_kernel<T, kUnit>, shape,
                  tile_smem<V>(kStage, shape.warps, p.length <= kTile),
                  tile_smem<V>(kStage, kWarps, false), divided, s, f, shape.geo);
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

size_t recurrence_workspace(const RecurrenceProblem& p) { return shape_of(p).workspace; }
size_t recurrence_backward_workspace(const RecurrenceBackwardProblem& p) {
    return shape_of(p).workspace;
}

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
