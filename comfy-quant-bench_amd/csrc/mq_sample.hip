// The next token of every row of logits for a given random number.
//
//   w_i = exp((l_i - max l) / T), in the order of l (descending, ties by index): kept are the first k, of those the
//   shortest leading part whose mass reaches p of theirs, and of those w_i >= min_p; the token is the first i, in
//   the order of i, whose kept mass up to it exceeds u times all kept mass. T <= 0: the first largest.
//
// Weights are summed as integers, in units of 2^-B of the largest with B = 62 - log2(V): sums are exact and the same
// in every order, so the result does not depend on how a row is split or on which atomic comes first. A weight
// is a table's entry (fp64, 1e-16) for the nearest multiple of a power of two that cuts the row's reach into some 2048 bins, times
// 1 + e for the rest of l, which is exact in fp32, is below 0.018 T and takes five fp32 products: 1e-9 at most, of random signs.
// (With fp32 weights the sum of a hundred thousand of them would be off by more than the share of a single token; a fp64
// exponential for every value takes four times as long as all of the rest.)
//
// A row is read three times, from memory and then from the caches: for its largest and smallest value; for a histogram,
// numbers and masses, over 2048 bins of equal width in l, whose sums from the top say which bins the limits k and p cut;
// and for the values of those bins and above, in the order of i, into LDS. There the cut bin is sorted and the
// limits become one value and one index. Where more is kept than fits there (a flat row), only the cut bin is collected and
// the row is read once more for the kept masses of its blocks of 8192, and the block that the token is in; where
// even the cut bin does not fit (values alike by the thousand), its limit is found digit by digit of the values' bits.
//
// A workgroup of 1024 takes a row, where there are enough of them or they are short; else every row is cut into parts, for
// which the three readings are three launches, and the part that ends last has all to choose from.
#include "mq_device.h"
#include "mq_internal.h"

namespace mq {
namespace {

constexpr int kThreads = 1024, kWavesOf = kThreads / 64;
constexpr int kPer = 8, kBlock = kThreads * kPer;   // consecutive values of a thread; of the workgroup
constexpr int kBins = 2048;
constexpr int kList = 4096;                         // values that are held in LDS
constexpr int kMostBlocks = (1 << 24) / kBlock;
constexpr double kLog2e64 = 1.4426950408889634074;
constexpr float kNone = -__builtin_inff();          // of NaN too, which is never chosen

__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct __attribute__((packed, aligned(2))) Eight16 {
    uint32_t w[4];
};
struct __attribute__((packed, aligned(4))) Eight32 {
    float f[4];
};

// Values i .. i + 7 of a row; NaN and what is behind the end as -infinity, both zeros alike.
template <int DT>
__device__ __forceinline__ void load8(const void* row, int i, int end, float (&v)[kPer]) {
    if (i + kPer <= end) {
        if constexpr (DT == kDtF32) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const Eight32 x = *reinterpret_cast<const Eight32*>(static_cast<const float*>(row) + i + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * h + e] = x.f[e];
            }
        } else {
            const Eight16 x = *reinterpret_cast<const Eight16*>(static_cast<const uint16_t*>(row) + i);
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const uint32_t w = x.w[e / 2];
                v[e] = DT == kDtF16 ? f16_bits_to_f32(static_cast<uint16_t>(e & 1 ? w >> 16 : w & 0xffffu)) : e & 1 ? bf16hi(w) : bf16lo(w);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < kPer; ++e) v[e] = i + e < end ? load_as_f32(row, DT, i + e) : kNone;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) v[e] = v[e] == v[e] ? v[e] + 0.0f : kNone;
}

// What is kept: keys above `key`, and those equal to it up to index `last`.
struct Limit {
    uint32_t key;
    int last;
    __device__ __forceinline__ bool keeps(uint32_t k, int i) const { return k > key || (k == key && i <= last); }
};
__device__ __forceinline__ uint64_t code_of(uint32_t key, int i) {
    return static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(~i);        // larger: earlier in the order
}

struct Lds {
    double weight[kBins];           // of the bins' centres
    uint64_t mass[kBins];           // of the bins; of the blocks of a row
    uint32_t count[kBins];
    uint64_t list[kList];           // index << 32 | key
    uint64_t sort[kList];           // codes
    uint64_t wave[2 * kWavesOf];
    int found, n;
    uint64_t left;
};
static_assert(kMostBlocks <= kBins);

// --- sums over the workgroup; every thread calls them

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

// The sum up to and including this thread's; *all = everybody's.
__device__ __forceinline__ uint64_t block_incl(uint64_t v, uint64_t* all, Lds& sh) {
    const int wave = threadIdx.x >> 6;
    v = wave_incl(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sh.wave[wave] = v;
    __syncthreads();
    uint64_t sum = 0;
#pragma unroll
    for (int y = 0; y < kWavesOf; ++y) {
        if (y < wave) v += sh.wave[y];
        sum += sh.wave[y];
    }
    *all = sum;
    return v;
}

__device__ __forceinline__ uint64_t block_sum(uint64_t s, Lds& sh) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0;
#pragma unroll
    for (int y = 0; y < kWavesOf; ++y) s += sh.wave[y];
    return s;
}

// x[0 .. n) ascending or (DOWN) descending (n <= kList).
template <bool DOWN>
__device__ void sort_list(uint64_t* x, int n) {
    int size = 2;
    while (size < n) size *= 2;
    __syncthreads();
    for (int i = n + threadIdx.x; i < size; i += kThreads) x[i] = DOWN ? 0 : ~uint64_t{0};
    for (int k = 2; k <= size; k *= 2)
        for (int j = k / 2; j > 0; j /= 2) {
            __syncthreads();
            for (int t = threadIdx.x; t < size / 2; t += kThreads) {
                const int a = 2 * t - (t & (j - 1)), b = a + j;
                const uint64_t u = x[a], v = x[b];
                if ((u < v) == (((a & k) == 0) == DOWN)) { x[a] = v; x[b] = u; }
            }
        }
    __syncthreads();
}

// --- a row

struct Row {
    const void* x;
    int V;
    float T, p, least;
    int64_t k;
    float best;             // the largest value (rows with +infinities: 0, and these 0, all others -infinity)
    int first;              // its first index
    bool infinite;
    double scale, unit;     // log2(e) / T; 2^(52 - B)
    float half, reach;      // half of the best; of how far below it a value may be and weigh anything (halves: no overflow)
    float step, per_step;   // width of a bin, a power of two; its inverse
    float top;              // the best's multiple of it
    float inv, inv_rest;    // 1 / T in two parts
    const double* weights;  // of the bins

    __device__ __forceinline__ float seen(float v) const { return infinite ? v == __builtin_inff() ? 0.0f : kNone : v; }
    __device__ __forceinline__ bool heavy(float v) const { return __builtin_fmaf(v, -0.5f, half) < reach; }
    __device__ __forceinline__ int bin(float v) const {
        const int b = static_cast<int>(top - __builtin_rintf(v * per_step));
        return b < kBins - 1 ? b : kBins - 1;
    }
    // The weight of a value that is heavy.
    __device__ __forceinline__ double weight(float v) const {
        const float n = __builtin_rintf(v * per_step), rest = __builtin_fmaf(-n, step, v);      // exact
        const int b = static_cast<int>(top - n);
        const float x = __builtin_fmaf(rest, inv, rest * inv_rest);
        float e = __builtin_fmaf(x, 1.0f / 24.0f, 1.0f / 6.0f);
        e = __builtin_fmaf(e, x, 0.5f);
        e = __builtin_fmaf(e, x, 1.0f) * x;
        const double w = weights[b < kBins - 1 ? b : kBins - 1];
        return __builtin_fma(w, static_cast<double>(e), w);
    }
    // In units: the mantissa of unit + w.
    __device__ __forceinline__ uint64_t whole(double w) const {
        return __builtin_bit_cast(uint64_t, unit + w) - __builtin_bit_cast(uint64_t, unit);
    }
    __device__ __forceinline__ uint64_t units(float v) const { return whole(weight(v)); }
    __device__ __forceinline__ uint64_t kept_units(float v) const {
        const double w = weight(v);
        return w < static_cast<double>(least) && v != best ? uint64_t{0} : whole(w);
    }
    __device__ __forceinline__ bool limited() const { return (k > 0 && k < V) || p < 1.0f; }
};

template <int DT>
__device__ __forceinline__ Row row_of(const SampleArgs& a, int64_t r) {
    Row w;
    w.x = static_cast<const char*>(a.x) + r * a.ld * (DT == kDtF32 ? 4 : 2);
    w.V = static_cast<int>(a.V);
    w.T = a.temperature ? a.temperature[r] : a.temperature1;
    w.p = a.top_p ? a.top_p[r] : a.top_p1;
    w.least = a.min_p ? a.min_p[r] : a.min_p1;
    w.k = a.top_k ? a.top_k[r] : a.top_k1;
    return w;
}

// The first reading, of values b .. e - 1: the code of the first largest, the smallest above -infinity.
template <int DT>
__device__ __forceinline__ void extremes(const Row& w, int b, int e, uint64_t* best, float* low, Lds& sh) {
    float top = kNone, least = __builtin_inff();
    int at = b;
    for (int i0 = b; i0 < e; i0 += kBlock) {
        const int i = i0 + kPer * threadIdx.x;
        if (i >= e) break;
        float v[kPer];
        load8<DT>(w.x, i, e, v);
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            if (v[x] > top) { top = v[x]; at = i + x; }
            least = v[x] > kNone ? __builtin_fminf(least, v[x]) : least;
        }
    }
    uint64_t code = code_of(key_of(top), at);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t y = __shfl_xor(code, d);
        code = code > y ? code : y;
        least = __builtin_fminf(least, __shfl_xor(least, d));
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
        sh.wave[threadIdx.x >> 6] = code;
        sh.wave[kWavesOf + (threadIdx.x >> 6)] = __float_as_uint(least);
    }
    __syncthreads();
    for (int y = 0; y < kWavesOf; ++y) {
        code = code > sh.wave[y] ? code : sh.wave[y];
        least = __builtin_fminf(least, __uint_as_float(static_cast<uint32_t>(sh.wave[kWavesOf + y])));
    }
    *best = code;
    *low = least;
}

// What follows from the extremes; true: the token is known (*token).
__device__ __forceinline__ bool settle(Row& w, uint64_t best, float low, int64_t* token) {
    w.best = value_of(static_cast<uint32_t>(best >> 32));
    w.first = static_cast<int>(~static_cast<uint32_t>(best));
    if (w.best == kNone) {
        *token = -1;
        return true;
    }
    if (!(w.T > 0.0f)) {
        *token = w.first;
        return true;
    }
    w.infinite = w.best == __builtin_inff();
    if (w.infinite) { w.best = 0.0f; low = 0.0f; }
    w.scale = 1.4426950408889634074 / static_cast<double>(w.T);
    int bits = 62;
    for (int64_t n = 1; n < w.V; n <<= 1) --bits;
    bits = bits < 51 ? bits : 51;
    w.unit = __builtin_ldexp(1.0, 52 - bits);
    // 2^-(bits + 1) is half a unit: 0 once rounded (a tie to even; the reach ends a little beyond it)
    w.reach = static_cast<float>(0.5 * (bits + 1.01) / w.scale);
    w.half = 0.5f * w.best;
    const float range = w.half - 0.5f * low, span = range < w.reach ? range : w.reach;
    // the smallest power of two that is at least span / 1023; none is needed below a 2^25th of the best (a value within
    // reach that is no multiple of that is at least a quarter of the best away from it)
    int at = 0, of_best = 0;
    const float part = __builtin_frexpf(span * (2.0f / (kBins - 2)), &at);      // in [2^(at - 1), 2^at)
    at -= part == 0.5f;
    (void)__builtin_frexpf(w.best, &of_best);
    at = span > 0.0f && at > of_best - 25 ? at : of_best - 25;
    at = at > -120 ? at < 120 ? at : 120 : -120;
    w.step = __builtin_ldexpf(1.0f, at);
    w.per_step = __builtin_ldexpf(1.0f, -at);
    w.top = __builtin_rintf(w.best * w.per_step);
    const double inv = 1.0 / static_cast<double>(w.T);
    w.inv = static_cast<float>(inv);
    w.inv_rest = static_cast<float>(inv - static_cast<double>(w.inv));
    return false;
}

// The weights of the bins' centres.
__device__ __forceinline__ void weigh_bins(Row& w, Lds& sh) {
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
        const double d = (static_cast<double>(w.top) - b) * static_cast<double>(w.step) - static_cast<double>(w.best);
        sh.weight[b] = exp2(d * w.scale);
    }
    w.weights = sh.weight;
    __syncthreads();
}

// The second reading: numbers and (p) masses of the bins, added to count and mass.
template <int DT>
__device__ __forceinline__ void histogram(const Row& w, int b, int e, Lds& sh) {
    const bool masses = w.p < 1.0f;
    for (int i0 = b; i0 < e; i0 += kBlock) {
        const int i = i0 + kPer * threadIdx.x;
        if (i >= e) break;
        float v[kPer];
        load8<DT>(w.x, i, e, v);
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            const float y = w.seen(v[x]);
            if (!w.heavy(y)) continue;
            const int at = w.bin(y);
            atomicAdd(&sh.count[at], 1u);
            if (masses) atomicAdd(reinterpret_cast<unsigned long long*>(&sh.mass[at]), static_cast<unsigned long long>(w.units(y)));
        }
    }
}

// Where a sum over the bins from the top reaches `need` (> 0): the bin (kBins: nowhere) and what is missing in front of it.
template <typename T>
__device__ __forceinline__ int cut_bin(const T* bins, uint64_t need, uint64_t* left, Lds& sh) {
    const uint64_t a = bins[2 * threadIdx.x], b = bins[2 * threadIdx.x + 1];
    uint64_t all;
    const uint64_t to = block_incl(a + b, &all, sh), from = to - a - b;
    if (threadIdx.x == 0) sh.found = kBins;
    __syncthreads();
    if (from < need && to >= need) {
        const bool second = from + a < need;
        sh.found = 2 * threadIdx.x + second;
        sh.left = need - from - (second ? a : 0);
    }
    __syncthreads();
    const int found = sh.found;
    *left = sh.left;
    __syncthreads();
    return found;
}

// What there is to choose from: values in LDS (n >= 0), or the row.
template <int DT, typename F>
__device__ __forceinline__ void each(const Row& w, int n, const Lds& sh, F f) {
    if (n >= 0) {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const uint64_t x = sh.list[i];
            f(value_of(static_cast<uint32_t>(x)), static_cast<int>(x >> 32));
        }
        return;
    }
    for (int i0 = 0; i0 < w.V; i0 += kBlock) {
        const int i = i0 + kPer * threadIdx.x;
        if (i >= w.V) break;
        float v[kPer];
        load8<DT>(w.x, i, w.V, v);
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            const float y = w.seen(v[x]);
            if (w.heavy(y)) f(y, i + x);
        }
    }
}

// The last resort of `resolve`: the limit's value digit by digit, eight bits at a time, then the index among equal ones.
template <int DT, bool MASS>
__device__ Limit by_digits(const Row& w, int bin, Limit now, uint64_t need, Lds& sh) {
    const int tid = threadIdx.x;
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (tid < 256) sh.sort[tid] = 0;
        __syncthreads();
        each<DT>(w, -1, sh, [&](float v, int i) {
            const uint32_t k = key_of(v);
            if (w.bin(v) != bin || !now.keeps(k, i) || (shift < 24 && k >> (shift + 8) != prefix >> (shift + 8))) return;
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.sort[k >> shift & 255]), MASS ? static_cast<unsigned long long>(w.units(v)) : 1ull);
        });
        __syncthreads();
        if (tid == 0) {
            int d = 255;
            for (; d > 0 && sh.sort[d] < need; --d) need -= sh.sort[d];
            sh.found = d;
            sh.left = need;
        }
        __syncthreads();
        prefix |= static_cast<uint32_t>(sh.found) << shift;
        need = sh.left;
    }
    if (MASS) {
        const uint64_t one = w.units(value_of(prefix));
        need = one ? (need + one - 1) / one : 1;
    }
    // the need-th of the values that are equal to it
    uint64_t before = 0;
    __syncthreads();
    if (tid == 0) sh.found = w.V;
    for (int i0 = 0; i0 < w.V; i0 += kBlock) {
        const int i = i0 + kPer * tid;
        float v[kPer];
        int n = 0;
        if (i < w.V) {
            load8<DT>(w.x, i, w.V, v);
#pragma unroll
            for (int x = 0; x < kPer; ++x) n += key_of(w.seen(v[x])) == prefix;
        }
        uint64_t all;
        uint64_t to = before + block_incl(n, &all, sh) - n;
        if (n)
#pragma unroll
            for (int x = 0; x < kPer; ++x)
                if (key_of(w.seen(v[x])) == prefix && ++to == need) sh.found = i + x;
        before += all;
        if (before >= need) break;
    }
    __syncthreads();
    const int last = sh.found;
    return Limit{prefix, last < now.last || prefix != now.key ? last : now.last};
}

// The limit inside a bin: the shortest leading part, of what `now` keeps of it, with `need` (> 0) elements, or (MASS) units.
// *mass: the units of that part (numbers only, and only where the bin fits LDS or `masses` asks for them).
template <int DT, bool MASS>
__device__ Limit resolve(const Row& w, int n, int bin, Limit now, uint64_t need, bool masses, uint64_t* mass, Lds& sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    each<DT>(w, n, sh, [&](float v, int i) {
        const uint32_t k = key_of(v);
        if (w.bin(v) != bin || !now.keeps(k, i)) return;
        const int at = atomicAdd(&sh.n, 1);
        if (at < kList) sh.sort[at] = code_of(k, i);
    });
    __syncthreads();
    const int held = sh.n;
    Limit limit;
    if (held > kList) {
        limit = by_digits<DT, MASS>(w, bin, now, need, sh);
        if (!MASS && masses) {
            uint64_t s = 0;
            each<DT>(w, n, sh, [&](float v, int i) { s += w.bin(v) == bin && limit.keeps(key_of(v), i) ? w.units(v) : 0; });
            *mass = block_sum(s, sh);
        }
        return limit;
    }
    sort_list<true>(sh.sort, held);
    // four codes a thread, in order
    constexpr int kEach = kList / kThreads;
    uint64_t x[kEach], sum = 0;
    const bool weigh = MASS || masses;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = kEach * threadIdx.x + e;
        x[e] = i >= held || (!MASS && static_cast<uint64_t>(i) >= need) ? 0 : weigh ? w.units(value_of(static_cast<uint32_t>(sh.sort[i] >> 32))) : 0;
        sum += x[e];
    }
    uint64_t all = 0;
    if (weigh) {
        uint64_t to = block_incl(sum, &all, sh) - sum;
        if (MASS) {
            if (threadIdx.x == 0) sh.found = held - 1;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                if (to < need && to + x[e] >= need) sh.found = kEach * threadIdx.x + e;
                to += x[e];
            }
            __syncthreads();
        }
    }
    *mass = all;
    const int last = MASS ? sh.found : static_cast<int>(need) - 1;
    const uint64_t c = sh.sort[last < held ? last : held - 1];
    __syncthreads();
    return Limit{static_cast<uint32_t>(c >> 32), static_cast<int>(~static_cast<uint32_t>(c))};
}

// u's place in all kept units.
__device__ __forceinline__ uint64_t place(float u, uint64_t all) {
    const double x = u, at = x > 0.0 ? x * static_cast<double>(all) : 0.0;
    const uint64_t t = at < static_cast<double>(all) ? static_cast<uint64_t>(at) : all - 1;
    return t < all ? t : all - 1;
}

// The token of a value list in LDS.
__device__ __forceinline__ int choose(const Row& w, int n, Limit limit, float u, Lds& sh) {
    sort_list<false>(sh.list, n);
    constexpr int kEach = kList / kThreads;
    uint64_t x[kEach], sum = 0, all;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = kEach * threadIdx.x + e;
        x[e] = 0;
        if (i < n) {
            const uint64_t y = sh.list[i];
            const uint32_t k = static_cast<uint32_t>(y);
            if (limit.keeps(k, static_cast<int>(y >> 32))) x[e] = w.kept_units(value_of(k));
        }
        sum += x[e];
    }
    uint64_t to = block_incl(sum, &all, sh) - sum;
    const uint64_t t = place(u, all);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        if (to <= t && to + x[e] > t) sh.found = static_cast<int>(sh.list[kEach * threadIdx.x + e] >> 32);
        to += x[e];
    }
    __syncthreads();
    return sh.found;
}

// Kept units of values i0 .. i0 + 8191 of a row, this thread's eight.
template <int DT>
__device__ __forceinline__ uint64_t block_units(const Row& w, int i0, int e, Limit limit, uint64_t (&x)[kPer]) {
    const int i = i0 + kPer * threadIdx.x;
    uint64_t sum = 0;
    float v[kPer];
    if (i < e) load8<DT>(w.x, i, e, v);
#pragma unroll
    for (int y = 0; y < kPer; ++y) {
        x[y] = 0;
        if (i < e) {
            const float z = w.seen(v[y]);
            if (w.heavy(z) && limit.keeps(key_of(z), i + y)) x[y] = w.kept_units(z);
        }
        sum += x[y];
    }
    return sum;
}

// The masses of blocks b / 8192 ... of a row, to mass[block].
template <int DT>
__device__ __forceinline__ void block_masses(const Row& w, int b, int e, Limit limit, uint64_t* mass, Lds& sh) {
    for (int i0 = b; i0 < e; i0 += kBlock) {
        uint64_t x[kPer];
        const uint64_t s = block_sum(block_units<DT>(w, i0, e, limit, x), sh);
        if (threadIdx.x == 0) mass[i0 / kBlock] = s;
    }
}

// The token of a row whose blocks' masses are in sh.mass.
template <int DT>
__device__ __forceinline__ int choose_block(const Row& w, Limit limit, float u, Lds& sh) {
    __syncthreads();
    const int blocks = (w.V + kBlock - 1) / kBlock;
    for (int i = blocks + threadIdx.x; i < kBins; i += kThreads) sh.mass[i] = 0;
    __syncthreads();
    uint64_t s = 0;
    for (int i = threadIdx.x; i < blocks; i += kThreads) s += sh.mass[i];
    const uint64_t all = block_sum(s, sh);
    uint64_t left;
    const int at = cut_bin(sh.mass, place(u, all) + 1, &left, sh);
    uint64_t x[kPer], sum;
    const int i0 = at * kBlock;
    const uint64_t mine = block_units<DT>(w, i0, w.V, limit, x);
    uint64_t to = block_incl(mine, &sum, sh) - mine;
#pragma unroll
    for (int y = 0; y < kPer; ++y) {
        if (to < left && to + x[y] >= left) sh.found = i0 + kPer * threadIdx.x + y;
        to += x[y];
    }
    __syncthreads();
    return sh.found;
}

// What the histogram says: how far down values are to be collected.
struct Cuts {
    int k_bin, p_bin;           // the bins that the limits cut (kBins: none)
    uint64_t k_left, p_left;    // what of them is kept
    int most;                   // collect bins 0 .. most
    uint64_t held;              // how many values those are (no limits: not known)
};

__device__ __forceinline__ Cuts cuts_of(const Row& w, Lds& sh) {
    Cuts c{kBins, kBins, 0, 0, kBins - 1, 0};
    if (w.k > 0 && w.k < w.V) c.k_bin = cut_bin(sh.count, static_cast<uint64_t>(w.k), &c.k_left, sh);
    if (w.p < 1.0f && c.k_bin == kBins) {
        const uint64_t all = block_sum(sh.mass[2 * threadIdx.x] + sh.mass[2 * threadIdx.x + 1], sh);
        const double need = __builtin_ceil(static_cast<double>(w.p) * static_cast<double>(all));
        c.p_bin = cut_bin(sh.mass, need > 1.0 ? static_cast<uint64_t>(need) : 1, &c.p_left, sh);
    }
    c.most = c.k_bin < kBins ? c.k_bin : c.p_bin < kBins ? c.p_bin : kBins - 1;
    const int b = 2 * threadIdx.x;
    c.held = block_sum((b <= c.most ? sh.count[b] : 0) + (b + 1 <= c.most ? sh.count[b + 1] : 0), sh);
    return c;
}

// The one limit of both, from n values in LDS (or the row).
template <int DT>
__device__ Limit limit_of(const Row& w, int n, Cuts c, Lds& sh) {
    Limit limit{0, w.V};
    uint64_t mass = 0;
    if (c.k_bin < kBins) {
        limit = resolve<DT, false>(w, n, c.k_bin, limit, c.k_left, w.p < 1.0f, &mass, sh);
        if (w.p < 1.0f) {
            // the mass of what k keeps, and where p of it ends: in a bin above the cut one or in that
            const int b = 2 * threadIdx.x;
            const uint64_t above = block_sum((b < c.k_bin ? sh.mass[b] : 0) + (b + 1 < c.k_bin ? sh.mass[b + 1] : 0), sh);
            double need = __builtin_ceil(static_cast<double>(w.p) * static_cast<double>(above + mass));
            need = need > 1.0 ? need : 1.0;
            const uint64_t units = static_cast<uint64_t>(need) < above + mass ? static_cast<uint64_t>(need) : above + mass;
            c.p_bin = c.k_bin;
            c.p_left = units - above;
            if (units <= above) c.p_bin = cut_bin(sh.mass, units, &c.p_left, sh);
        }
    }
    if (c.p_bin < kBins) limit = resolve<DT, true>(w, n, c.p_bin, limit, c.p_left, false, &mass, sh);
    return limit;
}

// The third reading, of values b .. e - 1: those in bins 0 .. most to sh.list, in any order, as far as there is room; how many
// there are.
template <int DT>
__device__ __forceinline__ int collect(const Row& w, int b, int e, int most, Lds& sh) {
    __syncthreads();
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
    for (int i0 = b; i0 < e; i0 += kBlock) {
        const int i = i0 + kPer * threadIdx.x;
        if (i >= e) break;
        float v[kPer];
        load8<DT>(w.x, i, e, v);
#pragma unroll
        for (int x = 0; x < kPer; ++x) {
            v[x] = w.seen(v[x]);
            if (w.heavy(v[x]) && w.bin(v[x]) <= most) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < kList) sh.list[at] = static_cast<uint64_t>(i + x) << 32 | key_of(v[x]);
            }
        }
    }
    __syncthreads();
    const int n = sh.n;
    __syncthreads();
    return n;
}

// The last bin that w >= min_p can be in (min_p alone limits the row).
__device__ __forceinline__ int least_bin(const Row& w) {
    const double d = -log(static_cast<double>(w.least < 1.0f ? w.least : 1.0f)) * static_cast<double>(w.T) * 1.000001;
    const double b = d * w.per_step + 2.0;
    return b < kBins - 1 ? static_cast<int>(b) : kBins - 1;
}

// The token once what the histogram says is in LDS: from n values in sh.list, or (n > kList) from the row.
template <int DT>
__device__ int finish(const Row& w, const Cuts& c, int n, float u, Lds& sh) {
    const bool in_lds = n <= kList;
    const Limit limit = limit_of<DT>(w, in_lds ? n : -1, c, sh);
    if (in_lds) return choose(w, n, limit, u, sh);
    block_masses<DT>(w, 0, w.V, limit, sh.mass, sh);
    return choose_block<DT>(w, limit, u, sh);
}

__device__ __forceinline__ void clear_bins(Lds& sh) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) { sh.mass[i] = 0; sh.count[i] = 0; }
    __syncthreads();
}

template <int DT>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
    __shared__ Lds sh;
    const int64_t r = blockIdx.x;
    Row w = row_of<DT>(a, r);
    uint64_t best;
    float low;
    extremes<DT>(w, 0, w.V, &best, &low, sh);
    int64_t token;
    if (!settle(w, best, low, &token)) {
        weigh_bins(w, sh);
        Cuts c{kBins, kBins, 0, 0, kBins - 1, 0};
        if (w.limited()) {
            clear_bins(sh);
            histogram<DT>(w, 0, w.V, sh);
            __syncthreads();
            c = cuts_of(w, sh);
        } else if (w.least > 0.0f) {
            c.most = least_bin(w);
        }
        int n = kList + 1;
        if ((w.limited() && c.held <= kList) || (!w.limited() && w.least > 0.0f) || w.V <= kList)
            n = collect<DT>(w, 0, w.V, c.most, sh);
        token = finish<DT>(w, c, n, a.u[r], sh);
    }
    if (threadIdx.x == 0) a.token[r] = token;
}

}  // namespace

int64_t sample_workspace_bytes(int64_t, int64_t) { return 0; }

int launch_sample(const SampleArgs& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(a.rows)), block(kThreads);
    if (a.dtype == kDtF32) hipLaunchKernelGGL((sample_kernel<kDtF32>), grid, block, 0, stream, a);
    else if (a.dtype == kDtF16) hipLaunchKernelGGL((sample_kernel<kDtF16>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((sample_kernel<kDtBf16>), grid, block, 0, stream, a);
    return launch_status("sample");
}

}  // namespace mq
