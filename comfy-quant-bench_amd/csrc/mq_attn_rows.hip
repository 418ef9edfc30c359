// Attention over a paged key-value cache, one wavefront per (new token, query head): the plainest kernel
// that is right for every case. Lane l holds values l, l + 64, ... of the head; the keys are taken one by
// one with a running maximum and sum of the softmax in fp32, both in base 2.
#include "mq_device.h"
#include "mq_internal.h"

namespace mq {
namespace {

constexpr int kMaxPer = 4;   // head width at most 256

__device__ __forceinline__ float load_kv(const void* p, int64_t i, int dt, bool i8, float s) {
    return i8 ? static_cast<float>(static_cast<const int8_t*>(p)[i]) * s : load_as_f32(p, dt, i);
}

__global__ void __launch_bounds__(256) attn_rows_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63;
    const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (item >= a.T * a.Hq) return;
    const int64_t t = item / a.Hq;
    const int hq = static_cast<int>(item - t * a.Hq), h = hq / (a.Hq / a.H);
    int64_t b = t, len, pos = -1;
    if (a.cu_q) {
        int64_t lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (a.cu_q[mid] <= t) lo = mid; else hi = mid;
        }
        b = lo;
        len = a.lens[b];
        if (t >= a.cu_q[b] && t < a.cu_q[b + 1]) pos = len - a.cu_q[b + 1] + t;
    } else {
        len = a.lens[b];
        pos = len - 1;
    }
    const int64_t mask = (int64_t(1) << a.page_shift) - 1;
    const int64_t cap = a.width << a.page_shift;
    const bool i8 = a.k_scale != nullptr;
    const int64_t qo = t * a.q_token + static_cast<int64_t>(hq) * a.q_head;
    float q[kMaxPer], o[kMaxPer];
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) {
        const int d = lane + 64 * i;
        q[i] = d < a.D ? load_as_f32(a.q, a.dtype, qo + d) * (a.scale * 1.4426950408889634f) : 0.0f;
        o[i] = 0.0f;
    }
    float m = -__builtin_inff(), l = 0.0f;
    bool any = false;
    for (int64_t j = 0; j <= pos && j < cap; ++j) {
        if (a.window > 0 && j <= pos - a.window && j >= a.sinks) {
            j = pos - a.window;
            continue;
        }
        const int page = a.table[b * a.ld_table + (j >> a.page_shift)];
        if (page < 0 || page >= a.pages) continue;
        any = true;
        const int64_t at = page * a.c_page + h * a.c_head + (j & mask) * a.c_token;
        const int64_t sc = page * a.s_page + h * a.s_head + (j & mask) * a.s_token;
        const float ks = i8 ? a.k_scale[sc] : 1.0f, vs = i8 ? a.v_scale[sc] : 1.0f;
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < kMaxPer; ++i) {
            const int d = lane + 64 * i;
            if (d < a.D) s = __builtin_fmaf(q[i], load_kv(a.kc, at + d, a.dtype, i8, ks), s);
        }
        for (int x = 1; x < 64; x <<= 1) s += __shfl_xor(s, x);
        const float mn = __builtin_fmaxf(m, s);
        const float base = mn == -__builtin_inff() ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(s - base);
        l = l * f + p;
#pragma unroll
        for (int i = 0; i < kMaxPer; ++i) {
            const int d = lane + 64 * i;
            if (d < a.D) o[i] = __builtin_fmaf(p, load_kv(a.vc, at + d, a.dtype, i8, vs), o[i] * f);
        }
        m = mn;
    }
    const int64_t oo = t * a.o_token + static_cast<int64_t>(hq) * a.o_head;
#pragma unroll
    for (int i = 0; i < kMaxPer; ++i) {
        const int d = lane + 64 * i;
        if (d < a.D) store_from_f32(a.o, a.dtype, oo + d, any ? o[i] / l : 0.0f);
    }
}

}  // namespace

int64_t attention_workspace_bytes(int64_t, int Hq, int H, int D, int64_t, bool ragged) {
    return ragged ? 0 : attn_decode_workspace_bytes(Hq, H, D);
}

int launch_attention(const AttnArgs& a, hipStream_t stream) {
    if (!a.cu_q) return launch_attn_decode(a, stream);
    const int64_t items = a.T * a.Hq;
    hipLaunchKernelGGL(attn_rows_kernel, dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0, stream, a);
    return launch_status("paged_attention");
}

}  // namespace mq
