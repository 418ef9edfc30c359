// y = x W^T + bias with 4-bit weights, a scale per group of K values and activations in floating point,
// optionally rotated by Hadamard blocks: the plainest kernel that is right for every case. A workgroup
// keeps one row of x in LDS in fp32 (rotated there) and each of its wavefronts sums one output column.
#include "mq_device.h"
#include "mq_internal.h"

namespace mq {
namespace {

__global__ void __launch_bounds__(256) w4a16_kernel(W4A16Args a) {
    extern __shared__ float xs[];
    const int64_t m = blockIdx.y;
    const int K = static_cast<int>(a.K);
    for (int k = threadIdx.x; k < K; k += 256) xs[k] = load_as_f32(a.x, a.x_dtype, m * a.ldx + k);
    __syncthreads();
    for (int st = 1; st < a.hblock; st *= 4) {
        for (int i = threadIdx.x; i < K / 4; i += 256) {
            const int k = (i / st) * 4 * st + i % st;
            const float x0 = xs[k], x1 = xs[k + st], x2 = xs[k + 2 * st], x3 = xs[k + 3 * st];
            const float t = 0.5f * (((x0 + x1) + x2) + x3);
            xs[k] = t - x3;
            xs[k + st] = t - x2;
            xs[k + 2 * st] = t - x1;
            xs[k + 3 * st] = t - x0;
        }
        __syncthreads();
    }
    const int lane = threadIdx.x & 63;
    const int64_t n = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (n >= a.N) return;
    float acc = 0.0f;
    for (int k = 2 * lane; k < K; k += 128) {
        const int g = k / a.group;
        const uint32_t w = a.qw[n * a.ldw + k / 2];
        const float s = load_as_f32(a.ws, a.s_dtype, n * a.ldws + g);
        float c0 = static_cast<float>(w & 15), c1 = static_cast<float>(w >> 4), z = 0.0f;
        if (a.zero == W4Zero::Signed) {
            c0 -= c0 > 7.0f ? 16.0f : 0.0f;
            c1 -= c1 > 7.0f ? 16.0f : 0.0f;
        } else if (a.zero == W4Zero::U4) {
            const float u = static_cast<float>((static_cast<const uint8_t*>(a.wz)[n * a.ldwz + g / 2] >> (4 * (g & 1))) & 15);
            c0 -= u;
            c1 -= u;
        } else {
            z = load_as_f32(a.wz, a.z_dtype, n * a.ldwz + g);
        }
        acc = __builtin_fmaf(xs[k], __builtin_fmaf(c0, s, z), acc);
        acc = __builtin_fmaf(xs[k + 1], __builtin_fmaf(c1, s, z), acc);
    }
    for (int x = 1; x < 64; x <<= 1) acc += __shfl_xor(acc, x);
    if (lane == 0) {
        if (a.bias) acc += load_as_f32(a.bias, a.bias_dtype, n);
        store_from_f32(a.y, a.y_dtype, m * a.ldy + n, acc);
    }
}

}  // namespace

int launch_w4a16(const W4A16Args& a, hipStream_t stream) {
    const size_t lds = a.K * 4;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(w4a16_kernel),
                                           hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(lds)) != hipSuccess) {
        set_error("w4a16: cannot reserve %zu bytes of LDS", lds);
        return -3;
    }
    hipLaunchKernelGGL(w4a16_kernel, dim3(static_cast<unsigned>((a.N + 3) / 4), static_cast<unsigned>(a.M)), dim3(256),
                       lds, stream, a);
    return launch_status("w4a16");
}

}  // namespace mq
