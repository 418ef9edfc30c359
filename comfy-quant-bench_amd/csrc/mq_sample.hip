// The next token of every row of logits for a given random number.
//
//   w_i = exp((l_i - max l) / T), in the order of l (descending, ties by index): kept are the first k, of those the
//   shortest leading part whose mass reaches p of theirs, and of those w_i >= min_p; the token is the first i, in
//   the order of i, whose kept mass up to it exceeds u times all kept mass. T <= 0: the first largest.
//
// Weights are summed as integers, in units of 2^-B of the largest with B = 62 - log2(V): sums are exact and the same
// in every order, so the result does not depend on how a row is split or on which atomic comes first. (With fp32 weights the
// sum of a hundred thousand of them would be off by more than the share of a single token; a fp64 exponential for every
// value takes four times as long as all of the rest.) A weight is a table's entry (fp64, 1e-15) for the nearest multiple of a
// power of two, `step`, of which 4096 reach as far down as anything weighs ((B + 1) ln 2 T: 32 T for V = 2^17, 36 T for short
// rows), times 1 + e for the rest of l: that is exact in fp32, below T / 110, and its series takes four fp32 products. A weight is off
// by 2e-9 of itself and a unit at most.
//
// First reading: the largest value, and numbers and masses of the 4096 bins around those multiples below it, in LDS. The
// bins are places n modulo 4096, so that they stay where they are as the largest value seen rises; those that fall out of
// reach are cleared. A bin is one 64-bit sum: a value adds 1 in the upper bits and 2^fine (e + 1/32) in the lower ones; the bin's
// mass is its centre's weight times (number + sum of e). Sums over the bins from the top say which bin the limit cuts. (2^fine
// leaves room for V values: 2^33 up to V = 2^17. What a value adds is rounded to fp32 and to a whole number, so masses are off by 4e-9
// of themselves up to V = 2^19, beyond that by 2^(2 log2(V) - 68), 1e-6 at 2^24.)
//
// Second reading: where k limits a row (few values), those of the cut bin and above, into LDS, where everything else is decided;
// where p does, those of the cut bin alone and the masses of what is above it by blocks of 8192; without either, the masses of
// the blocks. A limit inside a bin, a value and an index among equal ones, is found by sums over ranges of values (then of
// indexes), narrowed by 4096 at a time; so is the token, in LDS or in the block that u is in, which is read once more.
//
// A workgroup of 1024 takes a row. Where there are fewer rows than compute units, long rows are cut into parts: a launch for the
// first reading, one for the second, and the part that ends last has all to choose from. What fits neither (a limit k of
// thousands, a cut bin of thousands, temperatures beyond 2^+-20 times what logits are like) is done by one workgroup that reads
// the row again as often as it takes.
#include "mq_device.h"
#include "mq_internal.h"

namespace mq {
namespace {

constexpr int kThreads = 1024, kWavesOf = kThreads / 64;
constexpr int kPer = 8, kBlock = kThreads * kPer;   // consecutive values of a thread; of the workgroup
constexpr int kBins = 4096, kMask = kBins - 1;
constexpr int kEach = kBins / kThreads;             // bins, and values of the list, of a thread
constexpr int kList = 4096;                         // values that are held in LDS
constexpr int kFew = 256;
constexpr int kMostBlocks = (1 << 24) / kBlock;
constexpr int kMostParts = 8;
constexpr float kNone = -__builtin_inff();          // of NaN too, which is never chosen
constexpr float kLeastT = 0x1p-100f;                // below it the first largest is taken
constexpr float kBias = 1.0f / 32.0f;               // what makes e positive in a bin's sum
static_assert(kMostBlocks <= kBins && kList == kBins);

// Values as unsigned integers in their order, both zeros alike.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// --- reading a row

struct __attribute__((packed, aligned(2))) Sixteen {
    uint32_t w[4];
};
// Eight values as they lie in memory.
template <int DT>
struct Raw8 {
    Sixteen a[DT == kDtF32 ? 2 : 1];
};
// Values i .. i + 7 of a row; what is at `end` and behind it as -infinity.
template <int DT>
__device__ __forceinline__ Raw8<DT> load_raw8(const void* row, int i, int end) {
    constexpr int kParts = DT == kDtF32 ? 2 : 1;
    Raw8<DT> r;
    if (i + kPer <= end) {
        const char* p = static_cast<const char*>(row) + static_cast<int64_t>(i) * (DT == kDtF32 ? 4 : 2);
#pragma unroll
        for (int h = 0; h < kParts; ++h) r.a[h] = *reinterpret_cast<const Sixteen*>(p + 16 * h);
        return r;
    }
    constexpr uint32_t kLow = DT == kDtF16 ? 0xfc00u : 0xff80u;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if constexpr (DT == kDtF32) {
            r.a[e / 4].w[e % 4] = i + e < end ? static_cast<const uint32_t*>(row)[i + e] : 0xff800000u;
        } else {
            const uint32_t x = i + e < end ? static_cast<const uint16_t*>(row)[i + e] : kLow;
            r.a[0].w[e / 2] = e & 1 ? r.a[0].w[e / 2] | x << 16 : x;
        }
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void unpack8(const Raw8<DT>& r, float (&v)[kPer]) {
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if constexpr (DT == kDtF32) {
            v[e] = __uint_as_float(r.a[e / 4].w[e % 4]);
        } else {
            const uint32_t w = r.a[0].w[e / 2];
            v[e] = DT == kDtF16 ? f16_bits_to_f32(static_cast<uint16_t>(e & 1 ? w >> 16 : w & 0xffffu)) : e & 1 ? bf16hi(w) : bf16lo(w);
        }
        v[e] = v[e] > kNone ? v[e] : kNone;         // NaN
    }
}

// f(i, values i .. i + 7) for this thread's of values b .. e - 1, 32 or 64 bytes a thread in flight. All threads make all calls;
// values behind the end are -infinity.
template <int DT, typename F>
__device__ __forceinline__ void scan(const void* row, int b, int e, F f) {
    constexpr int kAhead = DT == kDtF32 ? 2 : 4;
    const int mine = kPer * threadIdx.x;
    Raw8<DT> raw[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x)
        if (b + x * kBlock < e) raw[x] = load_raw8<DT>(row, b + x * kBlock + mine, e);
    for (int i0 = b; i0 < e; i0 += kAhead * kBlock) {
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            const int i = i0 + x * kBlock;
            if (i >= e) break;
            float v[kPer];
            unpack8<DT>(raw[x], v);
            if (i + kAhead * kBlock < e) raw[x] = load_raw8<DT>(row, i + kAhead * kBlock + mine, e);
            f(i + mine, v);
        }
    }
}

// What makes a number of units an fp64 whose last place is 1 (below 2^51.02 they are), and the number back.
constexpr double kUnits = 0x1p52;
__device__ __forceinline__ uint64_t units_of(double x) { return __builtin_bit_cast(uint64_t, x) & 0xfffffffffffffull; }

struct Lds {
    double weight[kBins];           // of the bins' centres in units, from the best's down, each kUnits more
    uint64_t bins[kBins + 64];      // first by place (n modulo 4096, and a place for each lane's values that are in none), then
                                    // masses from the best's down; blocks' masses
    alignas(16) uint64_t work[kBins];   // sums over ranges; a few values side by side
    uint64_t list[kList];           // index << 32 | key, in any order
    uint64_t wave[2 * kWavesOf];
    int found, n;
    uint64_t left;
};

// --- the workgroup together; every thread calls these

// (Lane exchanges through LDS take ten times as long.)
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0u, static_cast<uint32_t>(v), CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0u, static_cast<uint32_t>(v >> 32), CTRL, ROWS, 0xf, false);
    return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ __forceinline__ uint64_t lane64(uint64_t v, int lane) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane))) << 32 |
           static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane));
}
// The sum over the lanes up to and including this one.
__device__ __forceinline__ uint64_t wave_incl(uint64_t v) {
    v += dpp64<0x111, 0xf>(v);      // from 1, 2, 4, 8 lanes before, within 16
    v += dpp64<0x112, 0xf>(v);
    v += dpp64<0x114, 0xf>(v);
    v += dpp64<0x118, 0xf>(v);
    v += dpp64<0x142, 0xa>(v);      // lane 15 to the next 16, lane 31 to the upper 32
    v += dpp64<0x143, 0xc>(v);
    return v;
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp32(uint32_t v) { return __builtin_amdgcn_update_dpp(0u, v, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ uint32_t wave_incl(uint32_t v) {
    v += dpp32<0x111, 0xf>(v);
    v += dpp32<0x112, 0xf>(v);
    v += dpp32<0x114, 0xf>(v);
    v += dpp32<0x118, 0xf>(v);
    v += dpp32<0x142, 0xa>(v);
    v += dpp32<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) { return lane64(v, lane); }
__device__ __forceinline__ uint64_t wave_sum(uint64_t v) { return lane64(wave_incl(v), 63); }
__device__ __forceinline__ uint32_t wave_max(uint32_t b) {
    b = __builtin_elementwise_max(b, dpp_mov_u<kQuadXor1>(b));
    b = __builtin_elementwise_max(b, dpp_mov_u<kQuadXor2>(b));
    b = __builtin_elementwise_max(b, dpp_mov_u<kRowRor4>(b));
    b = __builtin_elementwise_max(b, dpp_mov_u<kRowRor8>(b));
    const uint32_t r0 = __builtin_amdgcn_readlane(b, 0), r1 = __builtin_amdgcn_readlane(b, 16);
    const uint32_t r2 = __builtin_amdgcn_readlane(b, 32), r3 = __builtin_amdgcn_readlane(b, 48);
    return __builtin_elementwise_max(__builtin_elementwise_max(r0, r1), __builtin_elementwise_max(r2, r3));
}

// The sum up to and including this thread's; *all = everybody's.
__device__ __forceinline__ uint64_t block_incl(uint64_t v, uint64_t* all, Lds& sh) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_incl(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.wave[wave] = v;
    __syncthreads();
    const uint64_t to = wave_incl(sh.wave[threadIdx.x & 15]);          // (each 16 lanes the same; the first 16's are read)
    *all = lane64(to, 15);
    return v + (wave ? lane64(to, wave - 1) : 0);
}

__device__ __forceinline__ uint64_t block_sum(uint64_t s, Lds& sh) {
    s = wave_sum(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = s;
    __syncthreads();
    return lane64(wave_incl(sh.wave[threadIdx.x & 15]), 15);
}
__device__ __forceinline__ uint32_t block_max(uint32_t s, Lds& sh) {
    s = wave_max(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = s;
    __syncthreads();
    return wave_max(static_cast<uint32_t>(sh.wave[threadIdx.x & 15]));
}

// Where the sum of x(0), x(1), ... x(4095), of type T, reaches `need` (> 0): the place (4096: nowhere), what is missing in front of
// it, and (*all, not null) the sum. Every wave sums 256 of them; the one where it is looks at its own again.
template <typename T, typename F>
__device__ __forceinline__ int cut(F x, T need, T* left, T* all, Lds& sh) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    T v[kEach], sum = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        v[e] = x(256 * wave + 64 * e + lane);
        sum += v[e];
    }
    sum = lane_of(wave_incl(sum), 63);
    __syncthreads();
    if (lane == 0) sh.wave[wave] = sum;
    __syncthreads();
    const T to = wave_incl(static_cast<T>(sh.wave[lane & 15])), upto = lane_of(to, wave), before = upto - sum, total = lane_of(to, 15);
    if (all) *all = total;
    if (wave == 0 && total < need && lane == 0) sh.found = kBins;
    if (before < need && upto >= need) {
        T at = before;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const T y = at + wave_incl(v[e]);
            if (y - v[e] < need && y >= need) {
                sh.found = 256 * wave + 64 * e + lane;
                sh.left = need - (y - v[e]);
            }
            at = lane_of(y, 63);
        }
    }
    __syncthreads();
    const int found = __builtin_amdgcn_readfirstlane(sh.found);
    *left = static_cast<T>(sh.left);
    __syncthreads();
    return found;
}

// The place, from 0 to `most`, where the sum of the values' x, in the order of their places `at`, reaches *need (> 0, reached):
// over 4096 ranges of places, then over the parts of the one where it does. *need: what is missing in front of the place.
// n: none of a thread's places from n on (of 1024 e + thread) has an x. Few: each against all.
__device__ __forceinline__ uint32_t narrow(int n, const uint32_t (&at)[kEach], uint64_t (&x)[kEach], uint32_t most, uint64_t* need, Lds& sh) {
    if (n <= kFew) {
        uint32_t* places = reinterpret_cast<uint32_t*>(sh.work + kFew);
        __syncthreads();
        if (threadIdx.x < kFew) {
            sh.work[threadIdx.x] = x[0];
            places[threadIdx.x] = at[0];
        }
        __syncthreads();
        const int i = threadIdx.x >> 2;
        const uint32_t mine = places[i];
        uint64_t before = 0, same = 0;
        for (int j = threadIdx.x & 3; j < n; j += 4) {
            const uint64_t y = sh.work[j];
            const uint32_t p = places[j];
            before += p < mine ? y : 0;
            same += p == mine ? y : 0;
        }
        before += dpp64<kQuadXor1, 0xf>(before);
        before += dpp64<kQuadXor2, 0xf>(before);
        same += dpp64<kQuadXor1, 0xf>(same);
        same += dpp64<kQuadXor2, 0xf>(same);
        if (i < n && before < *need && before + same >= *need) {
            sh.found = static_cast<int>(mine);
            sh.left = *need - before;
        }
        __syncthreads();
        *need = sh.left;
        return static_cast<uint32_t>(sh.found);
    }
    int shift = 0;
    uint32_t from = 0;
    while (most >> shift >= kBins) ++shift;
    for (;;) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) sh.work[kThreads * e + threadIdx.x] = 0;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (x[e]) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.work[(at[e] - from) >> shift]), static_cast<unsigned long long>(x[e]));
        __syncthreads();
        const int range = cut<uint64_t>([&](int i) { return sh.work[i]; }, *need, need, nullptr, sh);
        from += static_cast<uint32_t>(range < kBins ? range : kBins - 1) << shift;
        if (shift == 0) return from;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (at[e] < from || (at[e] - from) >> shift) x[e] = 0;
        shift = shift > 12 ? shift - 12 : 0;
    }
}

// --- a row

// What is kept: keys above `key`, and those equal to it up to index `last`.
struct Limit {
    uint32_t key;
    int last;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};

struct Row {
    const void* x;
    int V;
    float T, p, least, u;
    int64_t k;
    float best;             // the largest value
    int first;              // its first index
    int bits, fine, number; // B; fractional bits of a bin's sum of e; where its number begins
    float step, per_step;   // distance of the bins' centres, a power of two; its inverse
    float top;              // the best's bin, as a multiple of the step
    float inv, inv_rest;    // 1 / T in two parts
    float floor;            // the smallest value that min_p keeps

    // How many bins below the best's; 4096 or more (or NaN, for -infinity): out of reach.
    __device__ __forceinline__ float depth(float v) const { return top - __builtin_rintf(v * per_step); }
    // A value's weight over its bin's, less 1.
    __device__ __forceinline__ float excess(float v) const {
        const float rest = __builtin_fmaf(-__builtin_rintf(v * per_step), step, v);      // exact
        const float x = __builtin_fmaf(rest, inv, rest * inv_rest);
        const float e = __builtin_fmaf(x, 1.0f / 6.0f, 0.5f);
        return __builtin_fmaf(e, x, 1.0f) * x;
    }
    // A value's weight in units, from the table (0 out of reach): the bin's c and e c, added where an fp64's last place is a unit, so
    // that the sum's rounding is the only one. (c's upper 30 bits times e in integers, the rest of c left out, put weights of 2^-22
    // of the largest off by 1e-5 and those of 2^-32 by 4e-3; with the rest 256 rows of 131072 took 81 us instead of 76.)
    __device__ __forceinline__ uint64_t units(float v, const Lds& sh) const {
        const float d = depth(v), e = excess(v);
        const bool in = d < static_cast<float>(kBins);
        const double c = sh.weight[in ? static_cast<int>(d) : kMask];
        return in ? units_of(__builtin_fma(static_cast<double>(e), c - kUnits, c)) : 0;
    }
    // The same from its own exponential.
    __device__ __forceinline__ uint64_t units(float v) const {
        const double x = exp2((static_cast<double>(v) - static_cast<double>(best)) * (1.4426950408889634074 / static_cast<double>(T)));
        return static_cast<uint64_t>(__builtin_rint(x * __builtin_ldexp(1.0, bits)));
    }
    __device__ __forceinline__ bool k_limits() const { return k > 0 && k < V; }
    __device__ __forceinline__ bool p_limits() const { return p < 1.0f; }
    __device__ __forceinline__ uint64_t place(uint64_t all) const {     // u's in all kept units
        const double x = u, at = x > 0.0 ? x * static_cast<double>(all) : 0.0;
        const uint64_t t = at < static_cast<double>(all) ? static_cast<uint64_t>(at) : all - 1;
        return t < all ? t : all - 1;
    }
    // The least number or mass that reaches p of `all`.
    __device__ __forceinline__ uint64_t part(uint64_t all) const {
        const double need = __builtin_ceil(static_cast<double>(p) * static_cast<double>(all));
        const uint64_t n = need > 1.0 ? static_cast<uint64_t>(need) : 1;
        return n < all ? n : all;
    }
};

// What is the same in all lanes, in scalar registers.
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }

// Centres 2^at apart, for a temperature T.
__device__ __forceinline__ void set_step(Row& w, int at) {
    w.step = uniform(__builtin_ldexpf(1.0f, at));
    w.per_step = uniform(__builtin_ldexpf(1.0f, -at));
    const double inv = 1.0 / static_cast<double>(w.T);
    w.inv = uniform(static_cast<float>(inv));
    w.inv_rest = uniform(static_cast<float>(inv - static_cast<double>(w.inv)));
}

// The exponent of the smallest power of two of which 4094 reach as far as anything weighs: 2^-(B + 1) is half a unit.
__device__ __forceinline__ int step_of(const Row& w) {
    int at;
    (void)__builtin_frexpf(static_cast<float>((w.bits + 1.01) * 0.69314718055994531 / (kBins - 2) * static_cast<double>(w.T)), &at);
    return at;
}
__device__ __forceinline__ bool usual(float T) { return T >= 0x1p-20f && T <= 0x1p20f; }

template <int DT>
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t r) {
    Row w;
    w.x = static_cast<const char*>(a.x) + r * a.ld * (DT == kDtF32 ? 4 : 2);
    w.V = static_cast<int>(a.V);
    // (Read at once, not one behind the other. What is not given is read from u and not used.)
    const float u = a.u[r], t = (a.temperature ? a.temperature : a.u)[r], p = (a.top_p ? a.top_p : a.u)[r],
                least = (a.min_p ? a.min_p : a.u)[r];
    const int k = (a.top_k ? a.top_k : reinterpret_cast<const int*>(a.u))[r];
    w.T = uniform(a.temperature ? t : a.temperature1);
    w.T = w.T < 0x1p120f ? w.T : w.T >= 0x1p120f ? 0x1p120f : 0.0f;     // (NaN: 0)
    w.p = uniform(a.top_p ? p : a.top_p1);
    w.least = uniform(a.min_p ? least : a.min_p1);
    w.k = a.top_k ? __builtin_amdgcn_readfirstlane(k) : a.top_k1;
    w.u = uniform(u);
    int log2 = 0;
    while ((1 << log2) < w.V) ++log2;
    w.bits = 62 - log2 < 51 ? 62 - log2 : 51;
    w.number = 63 - log2;                           // V values at most, each below 2^(fine - 4)
    w.fine = 67 - 2 * log2 < 33 ? 67 - 2 * log2 : 33;
    if (usual(w.T)) set_step(w, step_of(w));
    return w;
}

// The first largest of values b .. e - 1: w.best, w.first.
template <int DT>
__device__ __forceinline__ void largest(Row& w, int b, int e, Lds& sh) {
    float top = kNone;
    int at = b;
    scan<DT>(w.x, b, e, [&](int i, const float (&v)[kPer]) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < kPer; ++x)
            if (v[x] > top) { top = v[x]; at = i + x; }
    });
    const uint32_t best = block_max(key_of(top), sh);
    w.best = uniform(value_of(best));
    w.first = __builtin_amdgcn_readfirstlane(~block_max(key_of(top) == best ? ~static_cast<uint32_t>(at) : 0u, sh));
}

// The first reading of values b .. e - 1 with their bins (numbers, MASSES: and sums of e). known: w.top says where the best's bin
// is; else it is found on the way, with w.best. *base: the place of the best's bin in sh.bins.
template <int DT, bool MASSES>
__device__ __forceinline__ void bins_of(Row& w, int b, int e, bool known, int* base, Lds& sh) {
    constexpr int kDepth = DT == kDtF32 ? 2 : 4;    // blocks in hand; as many are on their way
    const int mine = kPer * threadIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kBins + 64; i += kThreads) sh.bins[i] = 0;
    const uint64_t one = uint64_t{1} << w.number;
    const float scale = uniform(__builtin_ldexpf(1.0f, w.fine)), bias = uniform(kBias * scale + 0.5f);    // (rounded, where fp32 has halves)
    int at = 0, parity = 0;
    float top = known ? w.top : kNone;
    uint32_t best = key_of(kNone);
    Raw8<DT> raw[2][kDepth];
    auto load = [&](int h, int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < kDepth; ++x) raw[h][x] = load_raw8<DT>(w.x, i0 + x * kBlock + mine, e);
    };
    auto take = [&](int h) __attribute__((always_inline)) {
        if (!known) {
            // the best so far; places that have fallen out of reach are empty again
            float most = kNone;
#pragma unroll
            for (int x = 0; x < kDepth; ++x) {
                float v[kPer];
                unpack8<DT>(raw[h][x], v);
#pragma unroll
                for (int y = 0; y < kPer; ++y) most = v[y] > most ? v[y] : most;
            }
            const uint32_t k = wave_max(key_of(most));
            if (lane == 0) sh.wave[kWavesOf * parity + wave] = k;
            __syncthreads();
            uint32_t now = best;
#pragma unroll
            for (int y = 0; y < kWavesOf; ++y) {
                const uint32_t z = static_cast<uint32_t>(sh.wave[kWavesOf * parity + y]);
                now = now > z ? now : z;
            }
            parity ^= 1;
            now = __builtin_amdgcn_readfirstlane(now);
            if (now > best) {
                best = now;
                const float next = uniform(__builtin_rintf(value_of(best) * w.per_step));
                if (next > top) {
                    const float far = next - top;
                    const int up = far < static_cast<float>(kBins) ? static_cast<int>(far) : kBins;
                    at = (at - up) & kMask;
                    for (int i = threadIdx.x; i < up; i += kThreads) sh.bins[(at + i) & kMask] = 0;
                    top = next;
                }
                __syncthreads();
            }
        } else {
            __syncthreads();
        }
        w.top = top;
#pragma unroll
        for (int x = 0; x < kDepth; ++x) {
            float v[kPer];
            unpack8<DT>(raw[h][x], v);
#pragma unroll
            for (int y = 0; y < kPer; ++y) {
                const float d = w.depth(v[y]);
                const int to = d < static_cast<float>(kBins) ? (at + static_cast<int>(d)) & kMask : kBins + lane;
                uint64_t add = one;
                if constexpr (MASSES) add |= static_cast<uint32_t>(__builtin_fmaf(w.excess(v[y]), scale, bias));
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[to]), static_cast<unsigned long long>(add));
            }
        }
    };
    __syncthreads();
    constexpr int kStep = kDepth * kBlock;
    load(0, b);
    for (int i0 = b; i0 < e; i0 += 2 * kStep) {
        if (i0 + kStep < e) load(1, i0 + kStep);
        take(0);
        if (i0 + kStep >= e) break;
        if (i0 + 2 * kStep < e) load(0, i0 + 2 * kStep);
        take(1);
    }
    if (!known) w.best = uniform(value_of(best));
    *base = at;
    __syncthreads();
}

// The weights of the bins' centres: the best's times a power of the step's, from 64 and 64 of them.
__device__ __forceinline__ void weigh_bins(const Row& w, Lds& sh) {
    double* small = reinterpret_cast<double*>(sh.work);
    const double scale = 1.4426950408889634074 / static_cast<double>(w.T) * static_cast<double>(w.step);
    if (threadIdx.x < 128) {
        const int i = threadIdx.x & 63;
        small[threadIdx.x] = threadIdx.x < 64 ? exp2(-i * scale) : exp2(-64 * i * scale);
    }
    if (threadIdx.x == 128)
        small[128] = exp2((static_cast<double>(w.top) * static_cast<double>(w.step) - static_cast<double>(w.best)) * (1.4426950408889634074 / static_cast<double>(w.T)) + w.bits);
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) sh.weight[b] = __builtin_rint(small[128] * small[64 + (b >> 6)] * small[b & 63]) + kUnits;
    __syncthreads();
}

// sh.bins from places and sums to masses, the best's first.
__device__ __forceinline__ void masses_of(const Row& w, int base, Lds& sh) {
    uint64_t x[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int d = kThreads * e + threadIdx.x;
        const uint64_t s = sh.bins[(base + d) & kMask], part = s & ((uint64_t{1} << w.number) - 1);
        const double n = static_cast<double>(s >> w.number);
        const double sum = static_cast<double>(part) * __builtin_ldexp(1.0, -w.fine) - n * static_cast<double>(kBias);
        x[e] = static_cast<uint64_t>(__builtin_rint((sh.weight[d] - kUnits) * (n + sum)));
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) sh.bins[kThreads * e + threadIdx.x] = x[e];
    __syncthreads();
}

// The values of the list: f(value, index) in each of a thread's four places below n.
template <typename F>
__device__ __forceinline__ void listed(int n, const Lds& sh, F f) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = kThreads * e + threadIdx.x;
        if (i < n) {
            const uint64_t x = sh.list[i];
            f(e, value_of(static_cast<uint32_t>(x)), static_cast<int>(x >> 32));
        }
    }
}

// Values b .. e - 1 whose bins are between `least` and `most` to sh.list, as far as there is room, behind the sh.n there are.
template <int DT>
__device__ __forceinline__ void collect(const Row& w, int b, int e, int least, int most, Lds& sh) {
    scan<DT>(w.x, b, e, [&](int i, const float (&v)[kPer]) __attribute__((always_inline)) {
        bool take[kPer], any = false;
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            const float d = w.depth(v[x]);
            take[x] = d <= static_cast<float>(most) && d >= static_cast<float>(least);
            any |= take[x];
        }
        if (!any) return;
#pragma unroll
        for (int x = 0; x < kPer; ++x)
            if (take[x]) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < kList) sh.list[at] = static_cast<uint64_t>(i + x) << 32 | key_of(v[x]);
            }
    });
    __syncthreads();
}
__device__ __forceinline__ void empty_list(Lds& sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
}

// Kept masses of the blocks of values b .. e - 1 to sh.bins[block]: of values in bins above `cut` (and, cut < 4096, those in it
// to sh.list), or within a limit.
template <int DT, bool LIMIT>
__device__ __forceinline__ void block_masses(const Row& w, int b, int e, int cut, Limit limit, Lds& sh) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    scan<DT>(w.x, b, e, [&](int i, const float (&v)[kPer]) __attribute__((always_inline)) {
        uint64_t s = 0;
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            const float d = w.depth(v[x]);
            const bool ok = (LIMIT ? d < static_cast<float>(kBins) && limit.keeps(key_of(v[x]), i + x) : d < static_cast<float>(cut)) && v[x] >= w.floor;
            const uint64_t units = w.units(v[x], sh);
            s += ok ? units : 0;
            if (!LIMIT && cut < kBins && d == static_cast<float>(cut)) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < kList) sh.list[at] = static_cast<uint64_t>(i + x) << 32 | key_of(v[x]);
            }
        }
        s = wave_sum(s);
        if ((threadIdx.x & 63) == 0 && s)
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[i / kBlock]), static_cast<unsigned long long>(s));
    });
    __syncthreads();
}

// The token of a row whose blocks' masses are in sh.bins: in bins above `cut` or within the limit.
template <int DT>
__device__ __forceinline__ int choose_block(const Row& w, Limit limit, Lds& sh) {
    uint64_t s = 0, left, all;
#pragma unroll
    for (int e = 0; e < kEach; ++e) s += sh.bins[kThreads * e + threadIdx.x];
    all = block_sum(s, sh);
    const int i0 = cut<uint64_t>([&](int i) { return sh.bins[i]; }, w.place(all) + 1, &left, nullptr, sh) * kBlock, i = i0 + kPer * threadIdx.x;
    float v[kPer];
    uint64_t x[kPer], sum = 0;
    unpack8<DT>(load_raw8<DT>(w.x, i, w.V), v);
#pragma unroll
    for (int y = 0; y < kPer; ++y) {
        x[y] = v[y] >= w.floor && limit.keeps(key_of(v[y]), i + y) ? w.units(v[y], sh) : 0;
        sum += x[y];
    }
    uint64_t to = block_incl(sum, &all, sh) - sum;
#pragma unroll
    for (int y = 0; y < kPer; ++y) {
        if (to < left && to + x[y] >= left) sh.found = i + y;
        to += x[y];
    }
    __syncthreads();
    return sh.found;
}

// The limit among n values of the list: the shortest leading part, of those of one bin that `now` keeps, with `need` (> 0) of them,
// or (MASS) units.
template <bool MASS, typename W>
__device__ __forceinline__ Limit limit_in(const Row& w, int n, int bin, Limit now, uint64_t need, W units, Lds& sh) {
    uint32_t at[kEach], high = 0, low = 0xffffffffu, key[kEach];
    int index[kEach];
    uint64_t x[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) x[e] = 0;
    listed(n, sh, [&](int e, float v, int i) {
        key[e] = key_of(v);
        index[e] = i;
        if (w.depth(v) != static_cast<float>(bin) || !now.keeps(key[e], i)) return;
        x[e] = MASS ? units(v) : 1;
        if (MASS && x[e] == 0) x[e] = 1;            // (less than half a unit; there is nothing below to choose from)
        high = high > key[e] ? high : key[e];
        low = low < key[e] ? low : key[e];
    });
    high = block_max(high, sh);
    low = ~block_max(~low, sh);
    uint64_t y[kEach], all = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        at[e] = x[e] ? high - key[e] : 0;
        y[e] = x[e];
        all += x[e];
    }
    all = block_sum(all, sh);
    need = need < all ? need : all;
    Limit limit{high - narrow(n, at, y, high - low, &need, sh), w.V};
    // among equal ones
    uint64_t same = 0, of = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        y[e] = x[e] != 0 && key[e] == limit.key;
        at[e] = y[e] ? index[e] : 0;
        same += y[e];
        of = y[e] ? x[e] : of;
    }
    same = block_sum(same, sh);
    if (MASS) {
        // (all of them weigh the same)
        const uint32_t high_of = block_max(static_cast<uint32_t>(of >> 32), sh), low_of = block_max(static_cast<uint32_t>(of), sh);
        of = static_cast<uint64_t>(high_of) << 32 | low_of;
        need = (need + of - 1) / of;
    }
    if (need < same) limit.last = static_cast<int>(narrow(n, at, y, static_cast<uint32_t>(w.V - 1), &need, sh));
    else if (limit.key == now.key) limit.last = now.last;
    return limit;
}

// The same from the row, where the bin's values do not fit the list: digit by digit of the values' bits.
template <int DT, bool MASS>
__device__ __forceinline__ Limit limit_by_digits(const Row& w, int bin, Limit now, uint64_t need, Lds& sh) {
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.work[i] = 0;
        __syncthreads();
        scan<DT>(w.x, 0, w.V, [&](int i, const float (&v)[kPer]) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < kPer; ++x) {
                const uint32_t k = key_of(v[x]);
                if (w.depth(v[x]) != static_cast<float>(bin) || !now.keeps(k, i + x) || (shift < 24 && k >> (shift + 8) != prefix >> (shift + 8)))
                    continue;
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.work[255 - (k >> shift & 255)]),
                          MASS ? static_cast<unsigned long long>(w.units(v[x], sh)) : 1ull);
            }
        });
        __syncthreads();
        if (shift == 24) {
            // no more than there is: `need` may come from the bin's mass, which these units' sum misses by a few
            uint64_t all = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) all += sh.work[kThreads * e + threadIdx.x];
            all = block_sum(all, sh);
            need = need < all ? need : all;
        }
        const int d = cut<uint64_t>([&](int i) { return sh.work[i]; }, need, &need, nullptr, sh);
        prefix |= static_cast<uint32_t>(255 - (d < 256 ? d : 255)) << shift;
        if (d >= 256) need = 1;
    }
    if (MASS) {
        const uint64_t of = w.units(value_of(prefix), sh);
        need = of ? (need + of - 1) / of : 1;
    }
    // the need-th of the values that are equal to it
    uint64_t before = 0, all;
    __syncthreads();
    if (threadIdx.x == 0) sh.found = w.V;
    for (int i0 = 0; i0 < w.V && before < need; i0 += kBlock) {
        const int i = i0 + kPer * threadIdx.x;
        float v[kPer];
        unpack8<DT>(load_raw8<DT>(w.x, i, w.V), v);
        uint64_t n = 0;
#pragma unroll
        for (int x = 0; x < kPer; ++x) n += i + x < w.V && key_of(v[x]) == prefix;
        uint64_t to = before + block_incl(n, &all, sh) - n;
#pragma unroll
        for (int x = 0; x < kPer; ++x)
            if (i + x < w.V && key_of(v[x]) == prefix && ++to == need) sh.found = i + x;
        before += all;
    }
    __syncthreads();
    const int last = sh.found;
    __syncthreads();
    return Limit{prefix, prefix == now.key && now.last < last ? now.last : last};
}

// The limit in a bin of the row.
template <int DT, bool MASS>
__device__ __forceinline__ Limit limit_in_row(const Row& w, int bin, Limit now, uint64_t need, Lds& sh) {
    empty_list(sh);
    collect<DT>(w, 0, w.V, bin, bin, sh);
    const int n = sh.n;
    if (n > kList) return limit_by_digits<DT, MASS>(w, bin, now, need, sh);
    return limit_in<MASS>(w, n, bin, now, need, [&](float v) { return w.units(v, sh); }, sh);
}

// Few values in LDS (n <= kFew), one a thread: how many of them come before thread i's in the order, and their units.
struct Few {
    uint64_t code, units, before;   // code: larger comes first
    int rank;
};
struct alignas(16) Pair {
    uint64_t a, b;
};
__device__ __forceinline__ Pair* pairs_of(Lds& sh) { return reinterpret_cast<Pair*>(sh.work); }
__device__ __forceinline__ Few rank_few(int n, uint64_t units, Lds& sh) {
    Few f{0, units, 0, 0};
    const int i = threadIdx.x;
    if (i < n) {
        const uint64_t x = sh.list[i];
        f.code = x << 32 | static_cast<uint32_t>(~static_cast<uint32_t>(x >> 32));
    }
    if (i < kFew) pairs_of(sh)[i] = Pair{f.code, units};
    __syncthreads();
    if (i < n)
#pragma unroll 8
        for (int j = 0; j < (n + 7) / 8 * 8; ++j) {
            const Pair y = pairs_of(sh)[j];
            const bool ahead = y.a > f.code;        // (places behind n are 0)
            f.rank += ahead;
            f.before += ahead ? y.b : 0;
        }
    return f;
}
// The sum over the first four waves, of which only these are left.
__device__ __forceinline__ uint64_t four_sum(uint64_t s, Lds& sh) {
    s = wave_sum(s);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = s;
    __syncthreads();
    return sh.wave[0] + sh.wave[1] + sh.wave[2] + sh.wave[3];
}

// choose_listed for n <= kFew: the last thing that a workgroup does, by its first four waves.
__device__ __forceinline__ void choose_few(const Row& w, int n, int64_t* token, Lds& sh) {
    if (threadIdx.x >= kFew) return;
    const int i = threadIdx.x;
    const float v = i < n ? value_of(static_cast<uint32_t>(sh.list[i])) : kNone;
    Few f = rank_few(n, i < n ? w.units(v) : 0, sh);
    bool in = i < n && (!w.k_limits() || f.rank < w.k);
    if (w.p_limits()) {
        const uint64_t need = w.part(four_sum(in ? f.units : 0, sh));
        in = in && f.before < need;
    }
    const uint64_t x = in && v >= w.floor ? f.units : 0, t = w.place(four_sum(x, sh));
    const uint32_t mine = static_cast<uint32_t>(sh.list[i] >> 32);
    pairs_of(sh)[i] = Pair{mine, x};
    __syncthreads();
    uint64_t to = 0;
    if (x)
#pragma unroll 8
        for (int j = 0; j < (n + 7) / 8 * 8; ++j) {
            const Pair y = pairs_of(sh)[j];         // (behind n: nothing)
            to += static_cast<uint32_t>(y.a) < mine ? y.b : 0;
        }
    if (x && to <= t && to + x > t) *token = mine;
}

// The token of n values in LDS, all that k (the bin that it cuts and what it keeps of that; 4096: none) may keep.
__device__ __forceinline__ int choose_listed(const Row& w, int n, int k_bin, uint64_t k_left, Lds& sh) {
    Limit limit{0, w.V};
    auto units = [&](float v) { return w.units(v); };
    if (k_bin < kBins) limit = limit_in<false>(w, n, k_bin, limit, k_left, units, sh);
    uint64_t x[kEach], y[kEach];
    uint32_t at[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        x[e] = y[e] = 0;
        at[e] = 0;
    }
    if (w.p_limits()) {
        uint64_t s = 0, left;
        __syncthreads();
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.work[i] = 0;
        __syncthreads();
        listed(n, sh, [&](int e, float v, int i) {
            if (!limit.keeps(key_of(v), i)) return;
            const uint64_t z = units(v);
            s += z;
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.work[static_cast<int>(w.depth(v))]), static_cast<unsigned long long>(z));
        });
        s = block_sum(s, sh);
        const int bin = cut<uint64_t>([&](int i) { return sh.work[i]; }, w.part(s), &left, nullptr, sh);
        limit = limit_in<true>(w, n, bin, limit, left, units, sh);
    }
    uint64_t s = 0;
    listed(n, sh, [&](int e, float v, int i) {
        at[e] = i;
        x[e] = v >= w.floor && limit.keeps(key_of(v), i) ? w.units(v) : 0;
        s += x[e];
    });
    uint64_t need = w.place(block_sum(s, sh)) + 1;
    return static_cast<int>(narrow(n, at, x, static_cast<uint32_t>(w.V - 1), &need, sh));
}

// The token of a row that p alone limits, from the cut bin's n values in LDS and the masses of the blocks above it in sh.bins.
template <int DT>
__device__ __forceinline__ int choose_cut(const Row& w, int n, int bin, uint64_t left, Lds& sh) {
    auto units = [&](float v) { return w.units(v, sh); };
    Limit limit{0, w.V};
    if (n <= kList) {
        if (n <= kFew) {
            // the limit is the last one in front of which less than `left` lies
            const float v = static_cast<int>(threadIdx.x) < n ? value_of(static_cast<uint32_t>(sh.list[threadIdx.x])) : kNone;
            const Few f = rank_few(n, static_cast<int>(threadIdx.x) < n ? units(v) : 0, sh);
            const bool in = static_cast<int>(threadIdx.x) < n && (f.before < left || f.rank == 0);
            const uint32_t last = block_max(in ? static_cast<uint32_t>(f.rank) + 1 : 0u, sh);
            if (in && f.rank + 1 == static_cast<int>(last)) sh.left = f.code;
            __syncthreads();
            limit = Limit{static_cast<uint32_t>(sh.left >> 32), static_cast<int>(~static_cast<uint32_t>(sh.left))};
            __syncthreads();
        } else {
            limit = limit_in<true>(w, n, bin, limit, left, units, sh);
        }
        listed(n, sh, [&](int e, float v, int i) {
            if (v >= w.floor && limit.keeps(key_of(v), i))
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[i / kBlock]), static_cast<unsigned long long>(units(v)));
        });
        __syncthreads();
    } else {
        limit = limit_by_digits<DT, true>(w, bin, limit, left, sh);
        block_masses<DT, true>(w, 0, w.V, kBins, limit, sh);
    }
    return choose_block<DT>(w, limit, sh);
}

// The token of a row with +infinities: all of them weigh the same, and nothing else does.
template <int DT>
__device__ __forceinline__ int among_infinities(const Row& w, Lds& sh) {
    uint64_t n = 0, before = 0;
    scan<DT>(w.x, 0, w.V, [&](int, const float (&v)[kPer]) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < kPer; ++x) n += v[x] == __builtin_inff();
    });
    n = block_sum(n, sh);
    if (w.k > 0 && static_cast<uint64_t>(w.k) < n) n = static_cast<uint64_t>(w.k);
    if (w.p_limits()) n = w.part(n);
    const uint64_t t = w.place(n);
    for (int i0 = 0; before <= t; i0 += kBlock) {
        float v[kPer];
        unpack8<DT>(load_raw8<DT>(w.x, i0 + kPer * threadIdx.x, w.V), v);
        uint64_t mine = 0, all;
#pragma unroll
        for (int x = 0; x < kPer; ++x) mine += v[x] == __builtin_inff();
        uint64_t to = before + block_incl(mine, &all, sh) - mine;
#pragma unroll
        for (int x = 0; x < kPer; ++x)
            if (v[x] == __builtin_inff() && to++ == t) sh.found = i0 + kPer * threadIdx.x + x;
        before += all;
    }
    __syncthreads();
    return sh.found;
}

// w.floor from the best: w >= min_p is l >= best + T log(min_p), rounded up to fp32 (the best is kept in any case).
__device__ __forceinline__ void set_floor(Row& w) {
    w.floor = kNone;
    if (!(w.least > 0.0f)) return;
    const double x = static_cast<double>(w.best) + static_cast<double>(w.T) * log(static_cast<double>(w.least));
    float f = static_cast<float>(x);
    if (static_cast<double>(f) < x) f = value_of(key_of(f) + 1);
    w.floor = uniform(f < w.best ? f : w.best);
}

// Whether the best's bin is far from what fp32 loses places in; else the step is chosen anew, from the best: none is needed below a
// 2^25th of it (a value within reach that is no multiple of that is at least a quarter of the best away).
__device__ __forceinline__ bool well_placed(const Row& w) { return usual(w.T) && __builtin_fabsf(w.best * w.per_step) < 0x1p60f; }
__device__ __forceinline__ void place_again(Row& w) {
    int of_best = -120, at = step_of(w);
    if (w.best != 0.0f) (void)__builtin_frexpf(w.best, &of_best);
    at = at > of_best - 25 ? at : of_best - 25;
    set_step(w, at > -120 ? at < 120 ? at : 120 : -120);
    w.top = uniform(__builtin_rintf(w.best * w.per_step));
}

// Where numbers of the bins (by place) cut k: the bin (4096: nowhere), what it keeps, and how many values that bin and those above
// it have.
__device__ __forceinline__ int cut_number(const Row& w, int base, uint64_t* left, uint64_t* held, Lds& sh) {
    auto number = [&](int d) { return static_cast<uint32_t>(sh.bins[(base + d) & kMask] >> w.number); };
    uint32_t rest, all;
    const uint32_t k = static_cast<uint32_t>(w.k);
    const int bin = cut<uint32_t>(number, k, &rest, &all, sh);
    *left = rest;
    *held = bin < kBins ? k - rest + number(bin) : all;
    return bin;
}

// The token of a whole row with known best, one workgroup, as many readings as it takes (k of thousands, odd temperatures).
template <int DT>
__device__ __attribute__((noinline)) int by_readings(Row w, Lds& sh) {
    if (!well_placed(w)) place_again(w);
    else w.top = uniform(__builtin_rintf(w.best * w.per_step));
    weigh_bins(w, sh);
    Limit limit{0, w.V};
    uint64_t left, held, mass = 0;
    int base, bin = kBins;
    if (w.k_limits()) {
        bins_of<DT, false>(w, 0, w.V, true, &base, sh);
        bin = cut_number(w, base, &left, &held, sh);
        if (bin < kBins) limit = limit_in_row<DT, false>(w, bin, limit, left, sh);
    }
    if (w.p_limits()) {
        if (bin < kBins) {
            // what k keeps of its bin
            uint64_t s = 0;
            scan<DT>(w.x, 0, w.V, [&](int i, const float (&v)[kPer]) __attribute__((always_inline)) {
#pragma unroll
                for (int x = 0; x < kPer; ++x)
                    if (w.depth(v[x]) == static_cast<float>(bin) && limit.keeps(key_of(v[x]), i + x)) s += w.units(v[x], sh);
            });
            mass = block_sum(s, sh);
        }
        bins_of<DT, true>(w, 0, w.V, true, &base, sh);
        masses_of(w, base, sh);
        uint64_t s = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) s += kThreads * e + threadIdx.x < bin ? sh.bins[kThreads * e + threadIdx.x] : 0;
        const uint64_t above = block_sum(s, sh), need = w.part(above + mass);
        left = need - above;
        if (need <= above) bin = cut<uint64_t>([&](int i) { return sh.bins[i]; }, need, &left, nullptr, sh);
        if (bin < kBins) limit = limit_in_row<DT, true>(w, bin, limit, left, sh);
    }
    block_masses<DT, true>(w, 0, w.V, kBins, limit, sh);
    return choose_block<DT>(w, limit, sh);
}

// What the first reading of values b .. e - 1 leaves in w.best and w.first, or (limited, usual temperatures) w.best and the bins.
template <int DT>
__device__ __forceinline__ void first_reading(Row& w, int b, int e, int* base, Lds& sh) {
    if (w.T < kLeastT || !usual(w.T) || !(w.k_limits() || w.p_limits())) largest<DT>(w, b, e, sh);
    else if (w.k_limits()) bins_of<DT, false>(w, b, e, false, base, sh);
    else bins_of<DT, true>(w, b, e, false, base, sh);
}

// Rows whose token needs no second reading of parts: true, and the token.
template <int DT>
__device__ __forceinline__ bool known(Row& w, int* token) {
    if (w.best != kNone && w.T >= kLeastT) return false;
    *token = w.best == kNone ? -1 : w.first;
    return true;
}

// The bin that p cuts, from the masses in sh.bins.
__device__ __forceinline__ int cut_mass(const Row& w, uint64_t* left, Lds& sh) {
    uint64_t s = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) s += sh.bins[kThreads * e + threadIdx.x];
    return cut<uint64_t>([&](int i) { return sh.bins[i]; }, w.part(block_sum(s, sh)), left, nullptr, sh);
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
    __shared__ Lds sh;
    const int64_t r = blockIdx.x;
    Row w = row_of<DT>(a, r);
    int base = 0, token;
    first_reading<DT>(w, 0, w.V, &base, sh);
    if (!known<DT>(w, &token)) {
        set_floor(w);
        uint64_t left, held;
        if (w.best == __builtin_inff()) {
            token = among_infinities<DT>(w, sh);
        } else if (!well_placed(w)) {
            token = by_readings<DT>(w, sh);
        } else if (w.k_limits()) {
            const int bin = cut_number(w, base, &left, &held, sh);
            if (held <= kList) {
                empty_list(sh);
                collect<DT>(w, 0, w.V, 0, bin < kBins ? bin : kBins - 1, sh);
                if (sh.n <= kFew) {
                    choose_few(w, sh.n, a.token + r, sh);
                    return;
                }
                token = choose_listed(w, sh.n, bin, left, sh);
            } else {
                token = by_readings<DT>(w, sh);
            }
        } else {
            w.top = uniform(__builtin_rintf(w.best * w.per_step));
            weigh_bins(w, sh);
            int bin = kBins;
            if (w.p_limits()) {
                masses_of(w, base, sh);
                bin = cut_mass(w, &left, sh);
            }
            empty_list(sh);
            block_masses<DT, false>(w, 0, w.V, bin, Limit{0, w.V}, sh);
            token = bin < kBins ? choose_cut<DT>(w, sh.n, bin, left, sh) : choose_block<DT>(w, Limit{0, w.V}, sh);
        }
    }
    if (threadIdx.x == 0) a.token[r] = token;
}

// --- rows in parts: a row's share of the workspace

struct Share {
    uint32_t *best, *first;     // [kMostParts], of the parts
    int *n, *done;              // values in the list; parts that have ended
    uint64_t *bins, *list, *blocks;
};
constexpr int64_t kShareHead = 8 * kMostParts + 64;
__host__ __device__ constexpr int64_t share_bytes(int64_t V, int parts) {
    return kShareHead + 8 * (static_cast<int64_t>(parts) * kBins + kList + (V + kBlock - 1) / kBlock);
}
__device__ __forceinline__ Share share_of(const SampleArgs& a, int64_t r, int parts) {
    char* p = static_cast<char*>(a.work) + r * share_bytes(a.V, parts);
    Share s;
    s.best = reinterpret_cast<uint32_t*>(p);
    s.first = s.best + kMostParts;
    s.n = reinterpret_cast<int*>(s.first + kMostParts);
    s.done = s.n + 1;
    s.bins = reinterpret_cast<uint64_t*>(p + kShareHead);
    s.list = s.bins + static_cast<int64_t>(parts) * kBins;
    s.blocks = s.list + kList;
    return s;
}
// Between workgroups of one launch: past the caches that are not common to all of them.
__device__ __forceinline__ void send(uint64_t* p, uint64_t x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t receive(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

struct Part {
    int b, e;
};
__device__ __forceinline__ Part part_of(int V, int part, int parts) {
    const int blocks = (V + kBlock - 1) / kBlock, b = blocks * part / parts * kBlock, e = blocks * (part + 1) / parts * kBlock;
    return Part{b, e < V ? e : V};
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_first_kernel(SampleArgs a) {
    __shared__ Lds sh;
    const int parts = gridDim.x, part = blockIdx.x;
    const Share s = share_of(a, blockIdx.y, parts);
    Row w = row_of<DT>(a, blockIdx.y);
    const Part p = part_of(w.V, part, parts);
    int base = 0;
    w.first = p.b;
    first_reading<DT>(w, p.b, p.e, &base, sh);
    if (threadIdx.x == 0) {
        s.best[part] = key_of(w.best);
        s.first[part] = static_cast<uint32_t>(w.first);
        if (part == 0) { *s.n = 0; *s.done = 0; }
    }
    if (w.T >= kLeastT && usual(w.T) && (w.k_limits() || w.p_limits()))
        for (int d = threadIdx.x; d < kBins; d += kThreads) s.bins[part * kBins + d] = sh.bins[(base + d) & kMask];
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_second_kernel(SampleArgs a) {
    __shared__ Lds sh;
    const int parts = gridDim.x, part = blockIdx.x;
    const Share s = share_of(a, blockIdx.y, parts);
    Row w = row_of<DT>(a, blockIdx.y);
    uint32_t best = 0, bests[kMostParts];               // (all read at once)
    int of = 0, token;
#pragma unroll
    for (int y = 0; y < kMostParts; ++y) bests[y] = s.best[y < parts ? y : 0];
#pragma unroll
    for (int y = 0; y < kMostParts; ++y)
        if (y < parts && bests[y] > best) { best = bests[y]; of = y; }
    w.best = uniform(value_of(__builtin_amdgcn_readfirstlane(best)));
    w.first = static_cast<int>(s.first[of]);
    // what one workgroup does alone
    bool alone = known<DT>(w, &token);
    set_floor(w);
    if (!alone && (w.best == __builtin_inff() || !well_placed(w))) {
        if (part != 0) return;
        alone = true;
        token = w.best == __builtin_inff() ? among_infinities<DT>(w, sh) : by_readings<DT>(w, sh);
    }
    if (alone) {
        if (part == 0 && threadIdx.x == 0) a.token[blockIdx.y] = token;
        return;
    }
    w.top = uniform(__builtin_rintf(w.best * w.per_step));
    const Part p = part_of(w.V, part, parts);
    uint64_t left = 0, held;
    int bin = kBins;
    if (w.k_limits() || w.p_limits()) {
        // the parts' bins together, those of a lower best further down
        uint64_t x[kEach] = {0, 0, 0, 0};
#pragma unroll
        for (int y0 = 0; y0 < kMostParts; y0 += 4) {    // (four parts' at once)
            if (y0 >= parts) break;
            uint64_t z[4][kEach];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int y = y0 + j;
                const float far = w.top - __builtin_rintf(value_of(bests[y]) * w.per_step);
                const int up = y < parts && far < static_cast<float>(kBins) ? static_cast<int>(far) : kBins;
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int d = kThreads * e + static_cast<int>(threadIdx.x) - up;
                    z[j][e] = s.bins[(y < parts ? y : 0) * kBins + (d < 0 ? 0 : d)];
                    if (d < 0) z[j][e] = 0;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < kEach; ++e) x[e] += z[j][e];
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) sh.bins[kThreads * e + threadIdx.x] = x[e];
        __syncthreads();
    }
    empty_list(sh);
    if (w.k_limits()) {
        bin = cut_number(w, 0, &left, &held, sh);
        if (held > kList) {
            if (part != 0) return;
            token = by_readings<DT>(w, sh);
            if (threadIdx.x == 0) a.token[blockIdx.y] = token;
            return;
        }
        collect<DT>(w, p.b, p.e, 0, bin < kBins ? bin : kBins - 1, sh);
    } else {
        weigh_bins(w, sh);
        if (w.p_limits()) {
            masses_of(w, 0, sh);
            bin = cut_mass(w, &left, sh);
        }
        block_masses<DT, false>(w, p.b, p.e, bin, Limit{0, w.V}, sh);
        for (int i = p.b / kBlock + threadIdx.x; i * kBlock < p.e; i += kThreads) send(s.blocks + i, sh.bins[i]);
    }
    // the part's values to the row's list; the last part takes them all
    if (threadIdx.x == 0) sh.found = sh.n ? __hip_atomic_fetch_add(s.n, sh.n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    __syncthreads();
    const int mine = sh.n < kList ? sh.n : kList, to = sh.found;
    for (int i = threadIdx.x; i < mine && to + i < kList; i += kThreads) send(s.list + to + i, sh.list[i]);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) sh.found = __hip_atomic_fetch_add(s.done, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (sh.found != parts - 1) return;
    const int n = __hip_atomic_load(s.n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int i = threadIdx.x; i < n && i < kList; i += kThreads) sh.list[i] = receive(s.list + i);
    if (!w.k_limits())
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = static_cast<int64_t>(i) * kBlock < w.V ? receive(s.blocks + i) : 0;
    __syncthreads();
    if (w.k_limits() && n <= kFew) {
        choose_few(w, n, a.token + blockIdx.y, sh);
        return;
    }
    if (w.k_limits()) token = choose_listed(w, n, bin, left, sh);
    else token = bin < kBins ? choose_cut<DT>(w, n, bin, left, sh) : choose_block<DT>(w, Limit{0, w.V}, sh);
    if (threadIdx.x == 0) a.token[blockIdx.y] = token;
}

// Parts of a row: as many as fill the device, of at least a block each.
int parts_of(int64_t rows, int64_t V) {
    const int cus = device_cu_count();
    const int64_t blocks = (V + kBlock - 1) / kBlock, room = (cus > 0 ? cus : 256) / (rows > 0 ? rows : 1);
    const int64_t n = blocks < room ? blocks : room;
    return static_cast<int>(n < 1 ? 1 : n < kMostParts ? n : kMostParts);
}

template <int DT>
int launch_type(const SampleArgs& a, hipStream_t stream) {
    const int parts = parts_of(a.rows, a.V);
    if (parts == 1) {
        constexpr int64_t most = kMostThreads / kThreads;
        for (int64_t r = 0; r < a.rows; r += most) {
            SampleArgs b = a;
            b.x = static_cast<const char*>(a.x) + r * a.ld * (DT == kDtF32 ? 4 : 2);
            b.u = a.u + r;
            b.temperature = a.temperature ? a.temperature + r : nullptr;
            b.top_p = a.top_p ? a.top_p + r : nullptr;
            b.min_p = a.min_p ? a.min_p + r : nullptr;
            b.top_k = a.top_k ? a.top_k + r : nullptr;
            b.token = a.token + r;
            b.rows = a.rows - r < most ? a.rows - r : most;
            hipLaunchKernelGGL((sample_kernel<DT>), dim3(static_cast<unsigned>(b.rows)), dim3(kThreads), 0, stream, b);
        }
    } else {
        const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(a.rows));
        hipLaunchKernelGGL((sample_first_kernel<DT>), grid, dim3(kThreads), 0, stream, a);
        hipLaunchKernelGGL((sample_second_kernel<DT>), grid, dim3(kThreads), 0, stream, a);
    }
    return launch_status("sample");
}

}  // namespace

int64_t sample_workspace_bytes(int64_t rows, int64_t V) {
    const int parts = parts_of(rows, V);
    return parts == 1 ? 0 : rows * share_bytes(V, parts);
}

int launch_sample(const SampleArgs& a, hipStream_t stream) {
    if (a.dtype == kDtF32) return launch_type<kDtF32>(a, stream);
    return a.dtype == kDtF16 ? launch_type<kDtF16>(a, stream) : launch_type<kDtBf16>(a, stream);
}

}  // namespace mq
