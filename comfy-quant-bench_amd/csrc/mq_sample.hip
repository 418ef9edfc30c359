// The next token of every row of logits for a given random number.
//
//   w_i = exp((l_i - max l) / T), in the order of l (descending, ties by index): kept are the first k, of those the
//   shortest leading part whose mass reaches p of theirs, and of those w_i >= min_p; the token is the first i, in
//   the order of i, whose kept mass up to it exceeds u times all kept mass. T <= 0: the first largest.
//
// Weights are taken in fp64 (a polynomial of degree 12 on [-1/2, 1/2] octaves, 1e-16) and summed as integers, in
// units of 2^-B of the largest with B = 62 - log2(V): sums are exact and the same in every order, so the result does
// not depend on how a row is split or on which atomic comes first. (In fp32 the sum of a hundred thousand
// weights would be off by more than the share of a single token.)
#include "mq_device.h"
#include "mq_internal.h"

namespace mq {
namespace {

constexpr int kThreads = 1024, kWavesOf = kThreads / 64;
constexpr uint32_t kKeyInf = 0xff800000u;       // key of +infinity
constexpr uint32_t kKeyNone = 0x007fffffu;      // key of -infinity (and of NaN, which is never chosen)

// Logits as unsigned integers in their order; both zeros alike.
template <int DT>
__device__ __forceinline__ float logit(const void* row, int64_t i) {
    const float x = load_as_f32(row, DT, i) + 0.0f;
    return x == x ? x : -__builtin_inff();
}
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct Weights {
    double scale, unit;     // log2(e) / T; 2^(52 - B)
    float best;
    __device__ __forceinline__ double at(float x) const {
        if (x == best) return 1.0;
        const double y = (static_cast<double>(x) - static_cast<double>(best)) * scale;
        if (!(y > -64.0)) return 0.0;
        const double n = __builtin_rint(y), f = (y - n) * 0.69314718055994530942;
        double p = 1.0 / 479001600.0;
        p = __builtin_fma(p, f, 1.0 / 39916800.0);
        p = __builtin_fma(p, f, 1.0 / 3628800.0);
        p = __builtin_fma(p, f, 1.0 / 362880.0);
        p = __builtin_fma(p, f, 1.0 / 40320.0);
        p = __builtin_fma(p, f, 1.0 / 5040.0);
        p = __builtin_fma(p, f, 1.0 / 720.0);
        p = __builtin_fma(p, f, 1.0 / 120.0);
        p = __builtin_fma(p, f, 1.0 / 24.0);
        p = __builtin_fma(p, f, 1.0 / 6.0);
        p = __builtin_fma(p, f, 0.5);
        p = __builtin_fma(p, f, 1.0);
        p = __builtin_fma(p, f, 1.0);
        return __builtin_ldexp(p, static_cast<int>(n));
    }
    // In units: the mantissa of unit + w.
    __device__ __forceinline__ uint64_t whole(double w) const {
        return __builtin_bit_cast(uint64_t, unit + w) - __builtin_bit_cast(uint64_t, unit);
    }
};

// What is kept: keys above `key`, and those equal to it up to index `last`.
struct Limit {
    uint32_t key;
    int last;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

struct Shared {
    uint64_t wave[kWavesOf];
    uint64_t best;
    uint64_t mass[256];
    uint32_t count[256];
    int digit;
    uint64_t left;
    int found;
};

template <typename T>
__device__ __forceinline__ T wave_incl(T v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const T y = __shfl_up(v, s);
        if (lane >= s) v += y;
    }
    return v;
}

// The first i of the row, in its order, up to which more than `t` of weight(i) has been seen.
template <typename F>
__device__ int walk(int V, uint64_t t, F weight, Shared& sh) {
    const int tid = threadIdx.x, wave = tid >> 6;
    if (tid == 0) sh.found = V;
    uint64_t before = 0;
    for (int i0 = 0; i0 < V; i0 += kThreads) {
        const uint64_t w = i0 + tid < V ? weight(i0 + tid) : 0;
        uint64_t x = wave_incl(w);
        __syncthreads();
        if ((tid & 63) == 63) sh.wave[wave] = x;
        __syncthreads();
        uint64_t all = 0;
        for (int y = 0; y < kWavesOf; ++y) {
            if (y < wave) x += sh.wave[y];
            all += sh.wave[y];
        }
        if (before + all > t) {
            if (before + x > t) atomicMin(&sh.found, i0 + tid);
            break;
        }
        before += all;
    }
    __syncthreads();
    const int found = sh.found;
    __syncthreads();
    return found;
}

template <typename F>
__device__ uint64_t total_of(int V, F weight, Shared& sh) {
    uint64_t s = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) s += weight(i);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0;
    for (int y = 0; y < kWavesOf; ++y) s += sh.wave[y];
    return s;
}

// The tighter limit that leaves, of what `now` keeps, the shortest leading part with `need` (>= 1) elements, or (MASS)
// units: the key's digits from the top, eight bits at a time, then the index among equal keys.
template <bool MASS, typename K, typename W>
__device__ Limit tighten(int V, Limit now, uint64_t need, K key, W units, Shared& sh) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) { sh.count[tid] = 0; sh.mass[tid] = 0; }
        __syncthreads();
        for (int i = tid; i < V; i += kThreads) {
            const uint32_t k = key(i);
            if (!now.keeps(k, i) || (shift < 24 && k >> (shift + 8) != prefix >> (shift + 8))) continue;
            const int d = k >> shift & 255;
            if constexpr (MASS) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[d]), static_cast<unsigned long long>(units(k)));
            else atomicAdd(&sh.count[d], 1u);
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255;
            for (; d > 0; --d) {
                const uint64_t n = MASS ? sh.mass[d] : sh.count[d];
                if (n >= need) break;
                need -= n;
            }
            sh.digit = d;
            sh.left = need;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(sh.digit) << shift;
        need = sh.left;
    }
    if constexpr (MASS) {
        const uint64_t one = units(prefix);
        need = one ? (need + one - 1) / one : 1;
    }
    const int last = walk(V, need - 1, [&](int i) { return static_cast<uint64_t>(key(i) == prefix && now.keeps(prefix, i)); }, sh);
    return Limit{prefix, last};
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, V = static_cast<int>(a.V);
    const int64_t r = blockIdx.x;
    const void* row = static_cast<const char*>(a.x) + r * a.ld * (DT == kDtF32 ? 4 : 2);
    const float T = a.temperature ? a.temperature[r] : a.temperature1;
    const float p = a.top_p ? a.top_p[r] : a.top_p1, least = a.min_p ? a.min_p[r] : a.min_p1;
    const int64_t k = a.top_k ? a.top_k[r] : a.top_k1;
    auto key = [&](int i) { return key_of(logit<DT>(row, i)); };

    // the first largest
    uint64_t best = 0;
    for (int i = tid; i < V; i += kThreads) {
        const uint64_t x = static_cast<uint64_t>(key(i)) << 32 | static_cast<uint32_t>(~i);
        best = best > x ? best : x;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = __shfl_xor(best, d);
        best = best > y ? best : y;
    }
    if ((tid & 63) == 0) sh.wave[tid >> 6] = best;
    __syncthreads();
    for (int y = 0; y < kWavesOf; ++y) best = best > sh.wave[y] ? best : sh.wave[y];
    const uint32_t top = static_cast<uint32_t>(best >> 32);
    if (top == kKeyNone || !(T > 0.0f)) {
        if (tid == 0) a.token[r] = top == kKeyNone ? -1 : static_cast<int>(~static_cast<uint32_t>(best));
        return;
    }
    Weights w;
    w.best = value_of(top);
    w.scale = 1.4426950408889634074 / static_cast<double>(T);
    int bits = 62;
    for (int64_t n = 1; n < V; n <<= 1) --bits;
    bits = bits < 51 ? bits : 51;
    w.unit = __builtin_ldexp(1.0, 52 - bits);
    auto units = [&](uint32_t k_) { return w.whole(w.at(value_of(k_))); };

    Limit keep{0, V};
    if (k > 0 && k < V) keep = tighten<false>(V, keep, static_cast<uint64_t>(k), key, units, sh);
    if (p < 1.0f) {
        const uint64_t all = total_of(V, [&](int i) { const uint32_t x = key(i); return keep.keeps(x, i) ? units(x) : 0; }, sh);
        const double need = __builtin_ceil(static_cast<double>(p) * static_cast<double>(all));
        keep = tighten<true>(V, keep, need > 1.0 ? static_cast<uint64_t>(need) : 1, key, units, sh);
    }
    auto kept = [&](int i) {
        const float x = logit<DT>(row, i);
        if (!keep.keeps(key_of(x), i)) return uint64_t{0};
        const double v = w.at(x);
        return v < static_cast<double>(least) && x != w.best ? uint64_t{0} : w.whole(v);
    };
    const uint64_t all = total_of(V, kept, sh);
    const double u = a.u[r];
    const double at = u > 0.0 ? u * static_cast<double>(all) : 0.0;
    uint64_t t = at < static_cast<double>(all) ? static_cast<uint64_t>(at) : all - 1;
    t = t < all ? t : all - 1;
    const int token = walk(V, t, kept, sh);
    if (tid == 0) a.token[r] = token;
}

}  // namespace

int launch_sample(const SampleArgs& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(a.rows)), block(kThreads);
    if (a.dtype == kDtF32) hipLaunchKernelGGL((sample_kernel<kDtF32>), grid, block, 0, stream, a);
    else if (a.dtype == kDtF16) hipLaunchKernelGGL((sample_kernel<kDtF16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((sample_kernel<kDtBf16>), grid, block, 0, stream, a);
    return launch_status("sample");
}

}  // namespace mq
