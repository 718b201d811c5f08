// The gradients of group norm with activation over [N, T, C] (channels last).
//
// Over the M valid frames of an utterance and the Cg channels of a group:
//   mean = sum x / (M Cg), var = sum (x - mean)^2 / (M Cg), rstd = (var + eps)^-1/2,
//   xhat = (x - mean) rstd, z = weight xhat + bias, out = act(z);
//   dz = dout act'(z), dbias = sum dz, dweight = sum dz xhat (over every valid frame),
//   dx = rstd (weight dz - (s1 + xhat s2) / (M Cg)),
//   s1 = sum weight dz, s2 = sum weight dz xhat (over the group).
//
// One block per utterance and group, one thread per element in turn; the parameters'
// gradients by one block per channel.
#include <cstdint>

#include "../../include/fga_convolution.h"
#include "fga_common.cuh"
#include "fga_kernels.h"

namespace fga {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float sigmoid(float v) { return 1.0f / (1.0f + __expf(-v)); }

__device__ __forceinline__ float slope(float z, int act) {
    if (act == FGA_ACTIVATION_SILU) {
        const float s = sigmoid(z);
        return s * (1.0f + z * (1.0f - s));
    }
    if (act == FGA_ACTIVATION_SWOOSH_R) return sigmoid(z - 1.0f) - 0.08f;
    return 1.0f;
}

// Sum over the block, the same value in every thread; `red` holds one float per warp.
__device__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    __syncthreads();
    if (threadIdx.x % kWarp == 0) red[threadIdx.x / kWarp] = v;
    __syncthreads();
    float total = 0.0f;
    for (int i = 0; i < kThreads / kWarp; ++i) total += red[i];
    return total;
}

__device__ __forceinline__ int valid_frames(const int32_t* lengths, int n, int length) {
    return min(max(lengths[n], 0), length);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) group_norm_backward_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const int32_t* __restrict__ lengths,
    const T* __restrict__ weight, const T* __restrict__ bias, const float* __restrict__ mean_in,
    const float* __restrict__ rstd_in, T* __restrict__ dx, int length, int channels, int groups,
    int act) {
    __shared__ float red[kThreads / kWarp];
    const int n = blockIdx.x / groups, g = blockIdx.x % groups, cg = channels / groups;
    const int m = valid_frames(lengths, n, length);
    const int64_t base = static_cast<int64_t>(n) * length * channels + g * cg;
    const int64_t count = static_cast<int64_t>(m) * cg, all = static_cast<int64_t>(length) * cg;
    const float inv = count > 0 ? 1.0f / static_cast<float>(count) : 0.0f;
    const float mean = mean_in[blockIdx.x], rstd = rstd_in[blockIdx.x];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t i = threadIdx.x; i < count; i += kThreads) {
        const int64_t at = base + i / cg * channels + i % cg;
        const int c = g * cg + static_cast<int>(i % cg);
        const float w = to_f32<T>(weight[c]), xhat = (to_f32<T>(x[at]) - mean) * rstd;
        const float d = w * to_f32<T>(dout[at]) * slope(xhat * w + to_f32<T>(bias[c]), act);
        s1 += d;
        s2 += d * xhat;
    }
    s1 = block_sum(s1, red) * inv;
    s2 = block_sum(s2, red) * inv;
    for (int64_t i = threadIdx.x; i < all; i += kThreads) {
        const int64_t at = base + i / cg * channels + i % cg;
        const int c = g * cg + static_cast<int>(i % cg);
        float v = 0.0f;
        if (i < count) {
            const float w = to_f32<T>(weight[c]), xhat = (to_f32<T>(x[at]) - mean) * rstd;
            const float d = w * to_f32<T>(dout[at]) * slope(xhat * w + to_f32<T>(bias[c]), act);
            v = rstd * (d - s1 - xhat * s2);
        }
        dx[at] = from_f32<T>(v);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) group_norm_parameters_kernel(
    const T* __restrict__ dout, const T* __restrict__ x, const int32_t* __restrict__ lengths,
    const T* __restrict__ weight, const T* __restrict__ bias, const float* __restrict__ mean,
    const float* __restrict__ rstd, T* __restrict__ dweight, T* __restrict__ dbias, int batch,
    int length, int channels, int groups, int act) {
    __shared__ float red[kThreads / kWarp];
    const int c = blockIdx.x, g = c / (channels / groups);
    const float w = to_f32<T>(weight[c]), b = to_f32<T>(bias[c]);
    float sw = 0.0f, sb = 0.0f;
    for (int n = 0; n < batch; ++n) {
        const int m = valid_frames(lengths, n, length);
        const float mu = mean[static_cast<int64_t>(n) * groups + g];
        const float r = rstd[static_cast<int64_t>(n) * groups + g];
        for (int t = threadIdx.x; t < m; t += kThreads) {
            const int64_t at = (static_cast<int64_t>(n) * length + t) * channels + c;
            const float xhat = (to_f32<T>(x[at]) - mu) * r;
            const float d = to_f32<T>(dout[at]) * slope(xhat * w + b, act);
            sb += d;
            sw += d * xhat;
        }
    }
    sw = block_sum(sw, red);
    sb = block_sum(sb, red);
    if (threadIdx.x == 0) {
        dweight[c] = from_f32<T>(sw);
        dbias[c] = from_f32<T>(sb);
    }
}

template <typename T>
cudaError_t backward(const GroupNormBackwardProblem& p, cudaStream_t s) {
    const T *dout = static_cast<const T*>(p.grad_output), *x = static_cast<const T*>(p.x),
            *w = static_cast<const T*>(p.weight), *b = static_cast<const T*>(p.bias);
    group_norm_backward_kernel<T><<<p.batch * p.groups, kThreads, 0, s>>>(
        dout, x, p.valid_lengths, w, b, p.mean, p.rstd, static_cast<T*>(p.grad_x), p.length,
        p.channels, p.groups, p.activation);
    group_norm_parameters_kernel<T><<<p.channels, kThreads, 0, s>>>(
        dout, x, p.valid_lengths, w, b, p.mean, p.rstd, static_cast<T*>(p.grad_weight),
        static_cast<T*>(p.grad_bias), p.batch, p.length, p.channels, p.groups, p.activation);
    return cudaGetLastError();
}

}  // namespace

size_t group_norm_backward_workspace(const GroupNormBackwardProblem&) { return 0; }

cudaError_t launch_group_norm_backward(const GroupNormBackwardProblem& p, cudaStream_t s,
                                       const char** variant) {
    *variant = "group-norm-backward";
    if (p.dtype == FGA_FLOAT) return backward<float>(p, s);
    if (p.dtype == FGA_HALF) return backward<__half>(p, s);
    return backward<__nv_bfloat16>(p, s);
}

}  // namespace fga
