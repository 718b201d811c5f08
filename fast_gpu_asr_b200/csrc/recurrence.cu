// Gated linear recurrence over [N, T, C], forward and backward:
//   f = sigmoid(gate), p = 1 - f, h[t] = f[t] h[t-1] + p[t] x[t];
//   G[t] = dout[t] + f[t+1] G[t+1] (+ dfinal at the last valid frame),
//   dx[t] = p[t] G[t], dgate[t] = f[t] p[t] (h[t-1] - x[t]) G[t], dinitial = f[0] G[0].
//
// A run of frames takes h to A h + B, with A the product of its f and B what it makes of
// h = 0, and runs compose: that is the scan. A warp holds kFrames consecutive frames of 32
// lanes' channels (one 128-byte row a frame) in registers, finds its (A, B), learns the state
// before its first frame from the warps before it through shared memory, and walks its frames
// a second time from there; no element is read twice. A block's warps cover one tile, a block
// walks the tiles of its utterance and channels in turn. Where utterances and channels are too
// few to fill the GPU, a cluster of blocks takes consecutive tiles and passes (A, B) on
// through distributed shared memory. The backward pass runs the same scan from the last tile
// to the first for the carry c[t] = f[t] G[t], and recomputes h within 64 frames of the states
// that the forward pass saved.
//
// Both are bound by HBM; arithmetic is fp32, of which the sigmoid's two special functions and
// about 20 instructions an element leave the issue slots about half free.
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

// ---- a lane's channels: a pair of a 16-bit type in one register, or one value --------------
template <typename T, int kVec> struct Lane;
template <typename T> struct Lane<T, 1> {
    using Raw = T;
    static __device__ __forceinline__ void unpack(Raw r, float* v) { v[0] = to_f32<T>(r); }
    static __device__ __forceinline__ Raw pack(const float* v) { return from_f32<T>(v[0]); }
    static __device__ __forceinline__ void keep_packed(Raw&) {}
};
template <typename T> struct Lane<T, 2> {
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
    // Hides from the compiler that a pair was unpacked before: it would keep the two floats
    // from one pass over the frames to the next, at twice the registers.
    static __device__ __forceinline__ void keep_packed(Raw& r) { asm("" : "+r"(r)); }
};
template <typename T, int kVec> __device__ __forceinline__ typename Lane<T, kVec>::Raw splat(float v) {
    const float two[2] = {v, v};
    return Lane<T, kVec>::pack(two);
}

// ---- the step ------------------------------------------------------------------------------
// Of f and p, the one below 1/2 has all its bits and the other is one minus it. `signed_gate`
// holds the small one, with its sign for which it is: f >= 0, or -p (so -0 keeps the state
// exactly and +0 takes x exactly).
__device__ __forceinline__ float signed_gate(float g) {
    const float e = __expf(-fabsf(g));
    const float small = e * __fdividef(1.0f, 1.0f + e);
    return __uint_as_float(__float_as_uint(small) | (~__float_as_uint(g) & 0x80000000u));
}
__device__ __forceinline__ bool keeps(float s) { return __float_as_int(s) < 0; }  // s is -p
// f h + p x, from the larger of the two: h + p (x - h) or x + f (h - x); d = h - x.
__device__ __forceinline__ float step(float s, float d, float h, float x) {
    return fmaf(s, d, keeps(s) ? h : x);
}
__device__ __forceinline__ float forget(float s) { return keeps(s) ? 1.0f + s : s; }  // f
__device__ __forceinline__ float take(float s) { return keeps(s) ? -s : 1.0f - s; }   // p
// f a
__device__ __forceinline__ float fade(float s, float a) {
    return fmaf(s, a, keeps(s) ? a : 0.0f);
}

struct Geometry {
    int length, channels, chunks;
    int slabs;    // channel slabs of 32 lanes
    int cluster;  // blocks that share an utterance's slab
};

// What a block works on.
template <int kVec> struct Place {
    int n, m, channel, rank, warp, lane, warps;
    bool active;
    __device__ Place(const Geometry& g, const int32_t* lengths) {
        warp = threadIdx.x / kWarp;
        lane = threadIdx.x % kWarp;
        warps = blockDim.x / kWarp;
        rank = blockIdx.x % g.cluster;
        const int unit = blockIdx.x / g.cluster;
        n = unit / g.slabs;
        channel = (unit % g.slabs * kWarp + lane) * kVec;
        active = channel < g.channels;
        m = min(max(lengths[n], 0), g.length);
    }
};

// kFrames rows from frame t0 on; rows at or past `limit` are `fill`.
template <typename Raw, int kFrames>
__device__ __forceinline__ void load_rows(Raw (&r)[kFrames], const Raw* p, int64_t stride, int t0,
                                          int limit, Raw fill) {
    if (t0 + kFrames <= limit) {
#pragma unroll
        for (int i = 0; i < kFrames; ++i, p += stride) r[i] = *p;
    } else {
#pragma unroll
        for (int i = 0; i < kFrames; ++i, p += stride) r[i] = t0 + i < limit ? *p : fill;
    }
}

template <typename Raw>
__device__ __forceinline__ void zero_rows(Raw* p, int64_t stride, int from, int to, int by,
                                          Raw zero) {
    for (int t = from; t < to; t += by) p[t * stride] = zero;
}

template <typename T, int kVec, int kFrames, int kWarps>
__global__ void __launch_bounds__(kWarps* kWarp, 3) recurrence_kernel(
    const T* __restrict__ x, const T* __restrict__ gate, const int32_t* __restrict__ lengths,
    const float* initial, T* __restrict__ out, float* final_state, float* __restrict__ states,
    Geometry geo) {
    using L = Lane<T, kVec>;
    using Raw = typename L::Raw;
    // Of each warp of the block and of each block of the cluster; two of them in turn, so that
    // one barrier a tile is enough.
    __shared__ float2 warp_run[2][kWarps][kWarp * kVec];
    __shared__ float2 block_run[2][kMaxCluster][kWarp * kVec];

    const Place<kVec> at(geo, lengths);
    const int limit = at.active ? at.m : 0;
    const int64_t stride = geo.channels / kVec;  // in Raw
    const int64_t base =
        static_cast<int64_t>(at.n) * geo.length * geo.channels + at.channel;
    const int64_t state_at = static_cast<int64_t>(at.n) * geo.channels + at.channel;
    float* saved = states == nullptr
                       ? nullptr
                       : states + static_cast<int64_t>(at.n) * geo.chunks * geo.channels + at.channel;

    float carry[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v)
        carry[v] = at.active && initial != nullptr ? initial[state_at + v] : 0.0f;
    // Every block of the cluster runs, and has read its state, before any writes to another.
    if (geo.cluster > 1) cg::this_cluster().sync();

    const int tile = at.warps * kFrames;
    int turn = 0;
    for (int start = 0; start < at.m; start += tile * geo.cluster, turn ^= 1) {
        const int t0 = start + at.rank * tile + at.warp * kFrames;
        const int64_t row = base + t0 * static_cast<int64_t>(geo.channels);
        Raw xr[kFrames];
        float s[kFrames][kVec];
        float a[kVec], b[kVec];
        {
            Raw gr[kFrames];
            load_rows(xr, reinterpret_cast<const Raw*>(x + row), stride, t0, limit,
                      splat<T, kVec>(0.0f));
            // An infinite gate keeps the state.
            load_rows(gr, reinterpret_cast<const Raw*>(gate + row), stride, t0, limit,
                      splat<T, kVec>(__int_as_float(0x7f800000)));
#pragma unroll
            for (int v = 0; v < kVec; ++v) a[v] = 1.0f, b[v] = 0.0f;
#pragma unroll
            for (int i = 0; i < kFrames; ++i) {
                float xv[kVec];
                L::unpack(gr[i], s[i]);
                L::unpack(xr[i], xv);
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    s[i][v] = signed_gate(s[i][v]);
                    a[v] = fade(s[i][v], a[v]);
                    b[v] = step(s[i][v], b[v] - xv[v], b[v], xv[v]);
                }
            }
        }
#pragma unroll
        for (int v = 0; v < kVec; ++v)
            warp_run[turn][at.warp][at.lane * kVec + v] = make_float2(a[v], b[v]);
        __syncthreads();
        if (geo.cluster > 1) {
            // Every warp finds the block's run; it tells its share of the cluster.
            auto cluster = cg::this_cluster();
#pragma unroll
            for (int v = 0; v < kVec; ++v) a[v] = 1.0f, b[v] = 0.0f;
            for (int w = 0; w < at.warps; ++w)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = warp_run[turn][w][at.lane * kVec + v];
                    b[v] = fmaf(r.x, b[v], r.y);
                    a[v] *= r.x;
                }
            for (int q = at.warp; q < geo.cluster; q += at.warps) {
                float2* there = cluster.map_shared_rank(&block_run[turn][at.rank][0], q);
#pragma unroll
                for (int v = 0; v < kVec; ++v)
                    there[at.lane * kVec + v] = make_float2(a[v], b[v]);
            }
            cluster.sync();
        }
        float h[kVec];
#pragma unroll
        for (int v = 0; v < kVec; ++v) h[v] = carry[v];
        if (geo.cluster > 1) {
            for (int q = 0; q < geo.cluster; ++q)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = block_run[turn][q][at.lane * kVec + v];
                    if (q == at.rank) h[v] = carry[v];
                    carry[v] = fmaf(r.x, carry[v], r.y);
                }
            for (int w = 0; w < at.warp; ++w)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = warp_run[turn][w][at.lane * kVec + v];
                    h[v] = fmaf(r.x, h[v], r.y);
                }
        } else {
            for (int w = 0; w < at.warps; ++w)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = warp_run[turn][w][at.lane * kVec + v];
                    if (w == at.warp) h[v] = carry[v];
                    carry[v] = fmaf(r.x, carry[v], r.y);
                }
        }
        if (saved != nullptr && t0 % kChunk == 0 && t0 < limit) {
#pragma unroll
            for (int v = 0; v < kVec; ++v)
                saved[static_cast<int64_t>(t0 / kChunk) * geo.channels + v] = h[v];
        }
        Raw* to = reinterpret_cast<Raw*>(out + row);
#pragma unroll
        for (int i = 0; i < kFrames; ++i, to += stride) {
            float xv[kVec];
            L::keep_packed(xr[i]);
            L::unpack(xr[i], xv);
#pragma unroll
            for (int v = 0; v < kVec; ++v) h[v] = step(s[i][v], h[v] - xv[v], h[v], xv[v]);
            if (t0 + i < limit) *to = L::pack(h);
        }
    }
    if (!at.active) return;
    if (at.rank == 0 && at.warp == 0) {
#pragma unroll
        for (int v = 0; v < kVec; ++v) final_state[state_at + v] = carry[v];
    }
    const int first = at.rank * at.warps + at.warp, by = geo.cluster * at.warps;
    zero_rows(reinterpret_cast<Raw*>(out + base), stride, at.m + first, geo.length, by,
              splat<T, kVec>(0.0f));
    if (saved != nullptr)
        for (int j = (at.m + kChunk - 1) / kChunk + first; j < geo.chunks; j += by)
#pragma unroll
            for (int v = 0; v < kVec; ++v)
                saved[static_cast<int64_t>(j) * geo.channels + v] = 0.0f;
}

template <typename T, int kVec, int kFrames, int kWarps>
__global__ void __launch_bounds__(kWarps* kWarp, 2) recurrence_backward_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const T* __restrict__ gate,
    const int32_t* __restrict__ lengths, const float* __restrict__ states,
    const float* __restrict__ dfinal, T* __restrict__ dx, T* __restrict__ dgate,
    float* __restrict__ dinitial, Geometry geo) {
    using L = Lane<T, kVec>;
    using Raw = typename L::Raw;
    // (A, B of h) of a warp; B of the carry; (A, B of the carry) of a block.
    __shared__ float2 warp_run[2][kWarps][kWarp * kVec];
    __shared__ float warp_back[2][kWarps][kWarp * kVec];
    __shared__ float2 block_run[2][kMaxCluster][kWarp * kVec];

    const Place<kVec> at(geo, lengths);
    const int limit = at.active ? at.m : 0;
    const int64_t stride = geo.channels / kVec;
    const int64_t base =
        static_cast<int64_t>(at.n) * geo.length * geo.channels + at.channel;
    const int64_t state_at = static_cast<int64_t>(at.n) * geo.channels + at.channel;
    const float* saved =
        states + static_cast<int64_t>(at.n) * geo.chunks * geo.channels + at.channel;

    float carry[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v)
        carry[v] = at.active && dfinal != nullptr ? dfinal[state_at + v] : 0.0f;
    if (geo.cluster > 1) cg::this_cluster().sync();

    const int tile = at.warps * kFrames, round = tile * geo.cluster;
    int turn = 0;
    for (int start = (at.m + round - 1) / round * round - round; start >= 0;
         start -= round, turn ^= 1) {
        const int t0 = start + at.rank * tile + at.warp * kFrames;
        const int64_t row = base + t0 * static_cast<int64_t>(geo.channels);
        Raw xr[kFrames], dr[kFrames];
        float s[kFrames][kVec];
        float a[kVec], b[kVec], c[kVec], h[kVec];
        {
            Raw gr[kFrames];
            load_rows(xr, reinterpret_cast<const Raw*>(x + row), stride, t0, limit,
                      splat<T, kVec>(0.0f));
            load_rows(gr, reinterpret_cast<const Raw*>(gate + row), stride, t0, limit,
                      splat<T, kVec>(__int_as_float(0x7f800000)));
            load_rows(dr, reinterpret_cast<const Raw*>(dout + row), stride, t0, limit,
                      splat<T, kVec>(0.0f));
            // The saved state at or before this warp's frames.
            const int64_t chunk = static_cast<int64_t>(t0 / kChunk) * geo.channels;
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                h[v] = t0 < limit ? saved[chunk + v] : 0.0f;
                a[v] = 1.0f, b[v] = 0.0f, c[v] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < kFrames; ++i) {
                float xv[kVec];
                L::unpack(gr[i], s[i]);
                L::unpack(xr[i], xv);
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    s[i][v] = signed_gate(s[i][v]);
                    a[v] = fade(s[i][v], a[v]);
                    b[v] = step(s[i][v], b[v] - xv[v], b[v], xv[v]);
                }
            }
#pragma unroll
            for (int i = kFrames - 1; i >= 0; --i) {
                float dv[kVec];
                L::unpack(dr[i], dv);
#pragma unroll
                for (int v = 0; v < kVec; ++v) c[v] = fade(s[i][v], dv[v] + c[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < kVec; ++v) {
            warp_run[turn][at.warp][at.lane * kVec + v] = make_float2(a[v], b[v]);
            warp_back[turn][at.warp][at.lane * kVec + v] = c[v];
        }
        __syncthreads();
        // h before this warp's frames: the saved state through the warps since.
        for (int w = at.warp - t0 % kChunk / kFrames; w < at.warp; ++w)
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                const float2 r = warp_run[turn][w][at.lane * kVec + v];
                h[v] = fmaf(r.x, h[v], r.y);
            }
        // The carry behind them.
        if (geo.cluster > 1) {
            auto cluster = cg::this_cluster();
#pragma unroll
            for (int v = 0; v < kVec; ++v) a[v] = 1.0f, c[v] = 0.0f;
            for (int w = at.warps - 1; w >= 0; --w)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float r = warp_run[turn][w][at.lane * kVec + v].x;
                    c[v] = fmaf(r, c[v], warp_back[turn][w][at.lane * kVec + v]);
                    a[v] *= r;
                }
            for (int q = at.warp; q < geo.cluster; q += at.warps) {
                float2* there = cluster.map_shared_rank(&block_run[turn][at.rank][0], q);
#pragma unroll
                for (int v = 0; v < kVec; ++v)
                    there[at.lane * kVec + v] = make_float2(a[v], c[v]);
            }
            cluster.sync();
            for (int q = geo.cluster - 1; q >= 0; --q)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    const float2 r = block_run[turn][q][at.lane * kVec + v];
                    if (q == at.rank) c[v] = carry[v];
                    carry[v] = fmaf(r.x, carry[v], r.y);
                }
            for (int w = at.warps - 1; w > at.warp; --w)
#pragma unroll
                for (int v = 0; v < kVec; ++v)
                    c[v] = fmaf(warp_run[turn][w][at.lane * kVec + v].x, c[v],
                                warp_back[turn][w][at.lane * kVec + v]);
        } else {
            for (int w = at.warps - 1; w >= 0; --w)
#pragma unroll
                for (int v = 0; v < kVec; ++v) {
                    if (w == at.warp) c[v] = carry[v];
                    carry[v] = fmaf(warp_run[turn][w][at.lane * kVec + v].x, carry[v],
                                    warp_back[turn][w][at.lane * kVec + v]);
                }
        }
        float away[kFrames][kVec];  // h[t-1] - x[t]
#pragma unroll
        for (int i = 0; i < kFrames; ++i) {
            float xv[kVec];
            L::keep_packed(xr[i]);
            L::unpack(xr[i], xv);
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                away[i][v] = h[v] - xv[v];
                h[v] = step(s[i][v], away[i][v], h[v], xv[v]);
            }
        }
        const int64_t end = row + (kFrames - 1) * static_cast<int64_t>(geo.channels);
        Raw* to_x = reinterpret_cast<Raw*>(dx + end);
        Raw* to_g = reinterpret_cast<Raw*>(dgate + end);
#pragma unroll
        for (int i = kFrames - 1; i >= 0; --i, to_x -= stride, to_g -= stride) {
            float gx[kVec], gg[kVec];
            L::keep_packed(dr[i]);
            L::unpack(dr[i], gx);
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                const float total = gx[v] + c[v], f = forget(s[i][v]);
                gx[v] = take(s[i][v]) * total;
                gg[v] = f * gx[v] * away[i][v];
                c[v] = f * total;
            }
            if (t0 + i < limit) {
                *to_x = L::pack(gx);
                *to_g = L::pack(gg);
            }
        }
    }
    if (!at.active) return;
    if (at.rank == 0 && at.warp == 0) {
#pragma unroll
        for (int v = 0; v < kVec; ++v) dinitial[state_at + v] = carry[v];
    }
    const int first = at.m + at.rank * at.warps + at.warp, by = geo.cluster * at.warps;
    const Raw zero = splat<T, kVec>(0.0f);
    zero_rows(reinterpret_cast<Raw*>(dx + base), stride, first, geo.length, by, zero);
    zero_rows(reinterpret_cast<Raw*>(dgate + base), stride, first, geo.length, by, zero);
}

// ---- launch --------------------------------------------------------------------------------

constexpr int kFrames = 16, kWarps = 8;

struct Shape {
    Geometry geo;
    int blocks, threads;
};

template <int kVec> Shape shape_of(int batch, int length, int channels, int chunks) {
    Shape s{};
    const int slabs = (channels + kWarp * kVec - 1) / (kWarp * kVec);
    const int warps = std::min(kWarps, (length + kFrames - 1) / kFrames);
    const int64_t units = static_cast<int64_t>(batch) * slabs;
    const int tiles = (length + kWarps * kFrames - 1) / (kWarps * kFrames);
    // Blocks for three on every multiprocessor, in rounds of the same number of tiles.
    const int64_t wanted = (3LL * sm_count() + units - 1) / units;
    int cluster = static_cast<int>(std::max<int64_t>(
        1, std::min<int64_t>(wanted, std::min(tiles, kMaxCluster))));
    const int rounds = (tiles + cluster - 1) / cluster;
    cluster = (tiles + rounds - 1) / rounds;
    s.geo = {length, channels, chunks, slabs, cluster};
    s.blocks = static_cast<int>(units * cluster);
    s.threads = warps * kWarp;
    return s;
}

template <typename... Params, typename... Args>
cudaError_t launch(void (*kernel)(Params...), const Shape& s, cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(s.blocks));
    cfg.blockDim = dim3(static_cast<unsigned>(s.threads));
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(s.geo.cluster);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = s.geo.cluster > 1 ? 1 : 0;
    if (s.geo.cluster > 8) {
        const cudaError_t e = cudaFuncSetAttribute(
            reinterpret_cast<const void*>(kernel),
            cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

bool pairs(int channels, std::initializer_list<const void*> buffers) {
    if (channels % 2 != 0) return false;
    for (const void* b : buffers)
        if (reinterpret_cast<uintptr_t>(b) % 4 != 0) return false;
    return true;
}

template <typename T, int kVec> cudaError_t forward(const RecurrenceProblem& p, cudaStream_t s) {
    const Shape shape = shape_of<kVec>(p.batch, p.length, p.channels, p.chunks);
    return launch(recurrence_kernel<T, kVec, kFrames, kWarps>, shape, s,
                  static_cast<const T*>(p.x), static_cast<const T*>(p.gate), p.valid_lengths,
                  p.initial_state, static_cast<T*>(p.output), p.final_state, p.states, shape.geo);
}

template <typename T, int kVec>
cudaError_t backward(const RecurrenceBackwardProblem& p, cudaStream_t s) {
    const Shape shape = shape_of<kVec>(p.batch, p.length, p.channels, p.chunks);
    return launch(recurrence_backward_kernel<T, kVec, kFrames, kWarps>, shape, s,
                  static_cast<const T*>(p.grad_output), static_cast<const T*>(p.x),
                  static_cast<const T*>(p.gate), p.valid_lengths, p.states, p.grad_final_state,
                  static_cast<T*>(p.grad_x), static_cast<T*>(p.grad_gate), p.grad_initial_state,
                  shape.geo);
}

}  // namespace

cudaError_t launch_recurrence(const RecurrenceProblem& p, cudaStream_t s, const char** variant) {
    *variant = "recurrence";
    const bool two = pairs(p.channels, {p.x, p.gate, p.output});
    if (p.dtype == FGA_FLOAT) return forward<float, 1>(p, s);
    if (p.dtype == FGA_HALF) return two ? forward<__half, 2>(p, s) : forward<__half, 1>(p, s);
    return two ? forward<__nv_bfloat16, 2>(p, s) : forward<__nv_bfloat16, 1>(p, s);
}

cudaError_t launch_recurrence_backward(const RecurrenceBackwardProblem& p, cudaStream_t s,
                                       const char** variant) {
    *variant = "recurrence-backward";
    const bool two = pairs(p.channels, {p.grad_output, p.x, p.gate, p.grad_x, p.grad_gate});
    if (p.dtype == FGA_FLOAT) return backward<float, 1>(p, s);
    if (p.dtype == FGA_HALF) return two ? backward<__half, 2>(p, s) : backward<__half, 1>(p, s);
    return two ? backward<__nv_bfloat16, 2>(p, s) : backward<__nv_bfloat16, 1>(p, s);
}

}  // namespace fga
