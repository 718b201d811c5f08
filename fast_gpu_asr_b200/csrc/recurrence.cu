// Gated linear recurrence over [N, T, C], forward and backward:
//   f = sigmoid(gate), p = 1 - f = sigmoid(-gate), h[t] = f[t] h[t-1] + p[t] x[t];
//   G[t] = dout[t] + f[t+1] G[t+1] (+ dfinal at the last valid frame),
//   dx[t] = p[t] G[t], dgate[t] = f[t] p[t] (h[t-1] - x[t]) G[t], dinitial = f[0] G[0].
//
// One thread per utterance and channel walks the frames. The backward walk goes through the
// saved states' 64-frame chunks from the last to the first and recomputes h within each.
#include <cstdint>

#include "../../include/fga_convolution.h"
#include "fga_common.cuh"
#include "fga_kernels.h"

namespace fga {
namespace {

constexpr int kThreads = 128;
constexpr int kChunk = FGA_RECURRENCE_STATE_FRAMES;

// f and p = 1 - f, each from the exponential that keeps its small values exact.
__device__ __forceinline__ void gates(float g, float& f, float& p) {
    const float e = __expf(-fabsf(g)), big = 1.0f / (1.0f + e), small = e * big;
    f = g < 0.0f ? small : big;
    p = g < 0.0f ? big : small;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) recurrence_kernel(
    const T* __restrict__ x, const T* __restrict__ gate, const int32_t* __restrict__ lengths,
    const float* initial, T* __restrict__ out, float* final_state, float* __restrict__ states,
    int rows, int length, int channels, int chunks) {
    const int row = blockIdx.x * kThreads + threadIdx.x;
    if (row >= rows) return;
    const int n = row / channels, c = row % channels;
    const int m = min(max(lengths[n], 0), length);
    float h = initial != nullptr ? initial[row] : 0.0f;
    for (int t = 0; t < length; ++t) {
        const int64_t at = (static_cast<int64_t>(n) * length + t) * channels + c;
        if (states != nullptr && t % kChunk == 0)
            states[(static_cast<int64_t>(n) * chunks + t / kChunk) * channels + c] =
                t < m ? h : 0.0f;
        if (t < m) {
            float f, p;
            gates(to_f32<T>(gate[at]), f, p);
            h = f * h + p * to_f32<T>(x[at]);
        }
        out[at] = from_f32<T>(t < m ? h : 0.0f);
    }
    final_state[row] = h;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) recurrence_backward_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const T* __restrict__ gate,
    const int32_t* __restrict__ lengths, const float* __restrict__ states,
    const float* __restrict__ dfinal, T* __restrict__ dx, T* __restrict__ dgate,
    float* __restrict__ dinitial, int rows, int length, int channels, int chunks) {
    const int row = blockIdx.x * kThreads + threadIdx.x;
    if (row >= rows) return;
    const int n = row / channels, c = row % channels;
    const int m = min(max(lengths[n], 0), length);
    float carry = dfinal != nullptr ? dfinal[row] : 0.0f;  // f[t+1] G[t+1]
    for (int j = chunks - 1; j >= 0; --j) {
        const int first = j * kChunk;
        float before[kChunk];
        float h = states[(static_cast<int64_t>(n) * chunks + j) * channels + c];
        for (int i = 0; i < kChunk; ++i) {
            before[i] = h;
            if (first + i < m) {
                const int64_t at = (static_cast<int64_t>(n) * length + first + i) * channels + c;
                float f, p;
                gates(to_f32<T>(gate[at]), f, p);
                h = f * h + p * to_f32<T>(x[at]);
            }
        }
        for (int i = kChunk - 1; i >= 0; --i) {
            const int t = first + i;
            if (t >= length) continue;
            const int64_t at = (static_cast<int64_t>(n) * length + t) * channels + c;
            float gx = 0.0f, gg = 0.0f;
            if (t < m) {
                float f, p;
                gates(to_f32<T>(gate[at]), f, p);
                const float total = to_f32<T>(dout[at]) + carry;
                gx = p * total;
                gg = f * gx * (before[i] - to_f32<T>(x[at]));
                carry = f * total;
            }
            dx[at] = from_f32<T>(gx);
            dgate[at] = from_f32<T>(gg);
        }
    }
    dinitial[row] = carry;
}

int blocks(int rows) { return (rows + kThreads - 1) / kThreads; }

template <typename T> cudaError_t forward(const RecurrenceProblem& p, cudaStream_t s) {
    const int rows = p.batch * p.channels;
    recurrence_kernel<T><<<blocks(rows), kThreads, 0, s>>>(
        static_cast<const T*>(p.x), static_cast<const T*>(p.gate), p.valid_lengths,
        p.initial_state, static_cast<T*>(p.output), p.final_state, p.states, rows, p.length,
        p.channels, p.chunks);
    return cudaGetLastError();
}

template <typename T> cudaError_t backward(const RecurrenceBackwardProblem& p, cudaStream_t s) {
    const int rows = p.batch * p.channels;
    recurrence_backward_kernel<T><<<blocks(rows), kThreads, 0, s>>>(
        static_cast<const T*>(p.grad_output), static_cast<const T*>(p.x),
        static_cast<const T*>(p.gate), p.valid_lengths, p.states, p.grad_final_state,
        static_cast<T*>(p.grad_x), static_cast<T*>(p.grad_gate), p.grad_initial_state, rows,
        p.length, p.channels, p.chunks);
    return cudaGetLastError();
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
