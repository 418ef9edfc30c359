// y = x W^T + bias with 4-bit weights, a scale per group of K values and activations in floating point,
// optionally rotated by Hadamard blocks: for few rows, so bound by reading the weights once, and next to that by
// unpacking them: at 8 TB/s a SIMD has some 78 VALU operations for the 1 KB of a wave's step.
//
// The codes go through MFMA as 16-bit floats without being scaled first (a scaled weight would be rounded):
// bits of a code are or-ed into the mantissa of a constant, which makes 16 + c in bf16 (1024 + c in fp16), eight
// operations for the eight codes of a dword. What is too much is taken off exactly: in fp16 by a packed
// subtraction (which takes the zero-point with it), in bf16 behind the product, where acc - (16 + z) sum(x)
// needs the group's sum of x, a product with ones. Both sums are rounded to fp32 at up to 31 |x| a value, so 16, the
// least that has mantissa bits for a code, loses the least: 1.5e-7 of an fp32 output, 4096 normal values a row (128 + c,
// one operation less, 0.2 us of the 13.9 below: 7e-7). Each group's fp32 sum is then scaled into the output's.
// Rows of x that have more bits than the 16-bit type are split into as many rows as hold them (fp32: three
// bf16 rows, exactly), which the 16 rows of a product have room for, and the rows' outputs are added at the end.
//
// A workgroup owns 16 CT output columns; its W waves share the K values, 128 at a time: lane (c, g) reads the
// 16 bytes of column c that hold values 32 g .. 32 g + 31 (64 bytes of each of 16 rows a load), and two exchanges
// of lane and register index bits leave in register j the dword of values 32 j + 8 g. A wave keeps KB steps'
// loads in flight in a ring of registers (in which order: mq_w4a16_runs.h). x is staged in LDS, as much of it as fits, in the order of the unpacked
// codes (0 4 1 5 2 6 3 7); the waves' sums are added there at the end. Row 4 e + g of x is row 4 g + e of
// a product, so that up to 4 rows come out in one register of every lane, up to 16 in four.
//
// Sums that are not finite are added again weight by weight (plain): the shifts would make NaN of an infinity.
//
// Measured: 4096 x 4096, one row: 6.0 us (the launch and one round of loads); 3072 -> 18432, one rotated row: 13.9 us,
// 2.2 TB/s, bound by unpacking and the latency of the few rounds that each workgroup has.
#include <type_traits>

#include "mq_device.h"
#include "mq_internal.h"
#include "mq_rotate.h"
#include "mq_w4a16_runs.h"

namespace mq {
namespace {

typedef __bf16 w4_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 w4_f16x8 __attribute__((ext_vector_type(8)));
typedef float w4_f32x4 __attribute__((ext_vector_type(4)));
struct W4Frag { uint32_t w[4]; };

template <bool F16>
__device__ __forceinline__ w4_f32x4 w4_mfma(const W4Frag& a, const W4Frag& b, w4_f32x4 c) {
    if constexpr (F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(w4_f16x8, a), __builtin_bit_cast(w4_f16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(w4_bf16x8, a), __builtin_bit_cast(w4_bf16x8, b), c, 0, 0, 0);
}

constexpr int kBlk = 128;      // K values per wave step
constexpr int kPad = 8;        // 16-bit values between two staged rows' ends (16 bytes: rows start on other banks)

// How a call is cut up (chosen on the host).
struct W4Plan {
    int parts;      // rows that a row of x becomes
    int rows_m;     // rows of x per workgroup (blockIdx.y)
    int chunk;      // K values staged at a time
    int pitch;      // pairs of scale and zero-point a column in LDS
    int pair_bufs;  // tiles' worth of them
    // divisions as products: n / d = n m / 2^32 for n d < 2^32 with m = 2^32 / d rounded up (a thread divides for
    // every piece and pair, which took 2 us of 16 rows' 20)
    uint32_t by_pieces;   // pieces a staged row
    uint32_t by_halves;   // pairs of groups a column
};

__host__ __device__ __forceinline__ uint32_t w4_inverse(int64_t d) {   // d = 1 wraps to 0
    return static_cast<uint32_t>(((int64_t(1) << 32) + d - 1) / d);
}
__device__ __forceinline__ int w4_div(int n, uint32_t inverse) {
    return inverse ? static_cast<int>(__umulhi(static_cast<uint32_t>(n), inverse)) : n;
}

// A stored value of type dt from its bits.
__device__ __forceinline__ float as_float(uint32_t b, int dt) {
    return dt == kDtF32 ? __uint_as_float(b) : dt == kDtF16 ? f16_bits_to_f32(static_cast<uint16_t>(b)) : __uint_as_float(b << 16);
}

// Eight values as a row's 16 bytes, in the order of a dword's codes: 0 4 1 5 2 6 3 7.
__device__ __forceinline__ uint4 w4_order(const uint32_t (&h)[8]) {
    return make_uint4(h[0] | h[4] << 16, h[1] | h[5] << 16, h[2] | h[6] << 16, h[3] | h[7] << 16);
}

// Part p of v: what bf16 holds of it after the parts before (truncated: the parts add up to v exactly).
__device__ __forceinline__ uint32_t w4_part(float* v) {
    // (a NaN keeps a mantissa: its own may be all in the bits that are cut off)
    const uint32_t h = *v != *v ? 0x7fc00000u : __float_as_uint(*v) & 0xffff0000u;
    *v = __builtin_isfinite(*v) ? *v - __uint_as_float(h) : 0.0f;
    return h >> 16;
}

// A piece of x on its way into LDS: 8 values of a row, a piece a thread; rotated rows: 16 values a lane in the
// rotate+quantize kernel's layout of 1024 columns, a piece a wave.
struct W4Piece {
    uint4 raw[4];
    int m, kk;
    bool ok;        // values of x (else zeros, past K)

    __device__ __forceinline__ void load(const W4A16Args& a, const W4Plan& pl, int64_t m0, int e, int all, int k0) {
        const int lane = threadIdx.x & 63;
        const int width = a.hblock ? 1024 : 8, per = pl.chunk / width;
        const int at = e < all ? e : 0;
        m = w4_div(at, pl.by_pieces);
        kk = width * (at - m * per) + (a.hblock ? 16 * ((lane >> 2) + 16 * (lane & 3)) : 0);
        const int k = k0 + kk;
        ok = e < all && k < a.K;
        const int size = a.x_dtype == kDtF32 ? 4 : 2;
        const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(a.x) + ((m0 + m) * a.ldx + (ok ? k : 0)) * size);
        raw[0] = p[0];
        if (a.hblock || size == 4) raw[1] = p[1];
        if (a.hblock && size == 4) {
            raw[2] = p[2];
            raw[3] = p[3];
        }
    }
    template <int XT, bool ROT>
    __device__ __forceinline__ void put(const W4A16Args& a, const W4Plan& pl, uint16_t* to, int stride) {
        constexpr int kValues = ROT ? 16 : 8;
        constexpr int kLoads = kValues * (XT == kDtF32 ? 4 : 2) / 16;
        if (!ok) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) raw[i] = make_uint4(0, 0, 0, 0);
        }
        if constexpr (!ROT && XT != kDtF32) {
            const uint4 x = raw[0];                     // 16-bit rows go as they are
            *reinterpret_cast<uint4*>(to) =
                make_uint4(__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                           __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u));
        } else {
            float v[kValues];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (XT == kDtF32) {
                        v[4 * i + j] = __uint_as_float(w[j]);
                    } else {
                        v[8 * i + 2 * j] = XT == kDtF16 ? f16lo(w[j]) : bf16lo(w[j]);
                        v[8 * i + 2 * j + 1] = XT == kDtF16 ? f16hi(w[j]) : bf16hi(w[j]);
                    }
                }
            }
            if constexpr (ROT) {
                // rotated in fp32, in the pinned order, and brought back into the layout of the load
                const int lane = threadIdx.x & 63;
                if (a.hblock == 16) {
                    rotate_chunk<16>(v, lane);
                } else if (a.hblock == 64) {
                    rotate_chunk<64>(v, lane);
                    swap_lane_reg<3, 3>(v, lane);
                    swap_lane_reg<2, 2>(v, lane);
                } else {
                    rotate_chunk<256>(v, lane);
                    swap_lane_reg<5, 3>(v, lane);
                    swap_lane_reg<4, 2>(v, lane);
                    swap_lane_reg<3, 3>(v, lane);
                    swap_lane_reg<2, 2>(v, lane);
                }
            }
#pragma unroll 1
            for (int p = 0; p < pl.parts; ++p)
#pragma unroll
                for (int j = 0; j < kValues / 8; ++j) {
                    uint32_t h[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) h[i] = w4_part(v + 8 * j + i);
                    *reinterpret_cast<uint4*>(to + p * stride + 8 * j) = w4_order(h);
                }
        }
    }
    template <bool F16>
    __device__ __forceinline__ void store(const W4A16Args& a, const W4Plan& pl, uint16_t* xs, int stride) {
        uint16_t* to = xs + m * pl.parts * stride + kk;
        if (F16) {
            put<kDtF16, false>(a, pl, to, stride);
        } else if (a.hblock) {
            if (a.x_dtype == kDtF32) put<kDtF32, true>(a, pl, to, stride);
            else if (a.x_dtype == kDtF16) put<kDtF16, true>(a, pl, to, stride);
            else put<kDtBf16, true>(a, pl, to, stride);
        } else {
            if (a.x_dtype == kDtF32) put<kDtF32, false>(a, pl, to, stride);
            else put<kDtBf16, false>(a, pl, to, stride);
        }
    }
};

// Scale and zero-point of a group as LDS holds them: two fp16 in a dword, or two floats.
template <bool ANY>
struct W4Pair;
template <>
struct W4Pair<false> {
    uint32_t v;
    __device__ __forceinline__ float scale() const { return f16_bits_to_f32(static_cast<uint16_t>(v & 0xffffu)); }
    __device__ __forceinline__ float zero() const { return f16_bits_to_f32(static_cast<uint16_t>(v >> 16)); }
};
template <>
struct W4Pair<true> {
    float s, z;
    __device__ __forceinline__ float scale() const { return s; }
    __device__ __forceinline__ float zero() const { return z; }
};

// F16: fp16 rows and products, else bf16; Z: zero-points; G: groups of 64 or 128 with fp16 scales and zero-points,
// or 0: any group and type; CT: 16-column tiles; NE: registers of a product that hold rows (1: up to 4 rows, 4: up to
// 16); KB: 128-value steps in flight; W: waves.
template <bool F16, W4Zero Z, int G, int CT, int NE, int KB, int W>
__global__ void __launch_bounds__(64 * W, W == 8 ? 2 : CT == 2 ? 3 : 4)
w4a16_kernel(W4A16Args a, W4Plan pl) {
    constexpr bool ANY = G == 0;
    constexpr int kScales = ANY ? 4 : kBlk / G;         // scales that a step uses (any: the same ones again for larger groups)
    constexpr bool kSum = !F16 || Z == W4Zero::Float;   // the sum of x is needed
    constexpr int kCols = 16 * CT;
    constexpr bool kThrough = W == 8;                   // a workgroup goes through several tiles
    using Pair = W4Pair<ANY>;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int K = static_cast<int>(a.K);
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * pl.rows_m;
    const int rows = static_cast<int>(a.M - m0 < pl.rows_m ? a.M - m0 : pl.rows_m);
    const int all = rows * pl.parts;                    // staged rows
    const int stride = pl.chunk + kPad;
    const int gshift = a.group == 32 ? 5 : a.group == 64 ? 6 : 7;
    const int groups = K >> gshift, pitch = pl.pitch;
    uint16_t* xs = reinterpret_cast<uint16_t*>(lds);
    Pair* pairs = reinterpret_cast<Pair*>(xs + pl.rows_m * pl.parts * stride);          // [pair_bufs][column][pitch]
    float* red = reinterpret_cast<float*>(pairs + pl.pair_bufs * kCols * pitch);                // [wave][row][column]

    // loads complete in the order of their issue: the first piece of x ahead of the weights, so that x is
    // staged while the weights are on their way
    const int pieces = rows * (pl.chunk / (a.hblock ? 1024 : 8));
    const int mine = a.hblock ? wave : static_cast<int>(threadIdx.x), step = a.hblock ? W : 64 * W;
    // pieces a thread has in flight: as many as registers are free for (bf16 ones may be rotated or fp32 and take 16
    // each: 16 rows of 4096 into 4096 12.1 us, with four 12.7; fp16 ones into 12288 17.9 us, with two 18.2)
    constexpr int PB = !kThrough ? 1 : F16 ? 4 : 2;
    W4Piece piece[PB];
#pragma unroll
    for (int i = 0; i < PB; ++i) piece[i].load(a, pl, m0, mine + i * step, pieces, 0);
    __builtin_amdgcn_sched_barrier(0);

    const int tiles = static_cast<int>((a.N + kCols - 1) / kCols);
    const uint32_t last = static_cast<uint32_t>(K / 2 - 16);
    uint4 w[KB][CT];
    // step `blk` (128 values) of tile `tile` into ring place i; past the end of K the last values
    auto fetch = [&](int i, int tile, int blk) __attribute__((always_inline)) {
        const int64_t n0 = static_cast<int64_t>(tile) * kCols;
        // the address as a scalar base and a 32-bit offset of the lane: its column's, within the tile
        const char* base = reinterpret_cast<const char*>(a.qw) + n0 * a.ldw;
        const uint32_t at = static_cast<uint32_t>(blk) * (kBlk / 2) + 16 * g;
        const uint32_t kk = at < last ? at : last;
        const int left = static_cast<int>(a.N - 1 - n0 < kCols ? a.N - 1 - n0 : kCols);
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            const uint32_t col = 16 * t + c < left ? 16 * t + c : left;   // columns past N read the last one's weights
            w[i][t] = *reinterpret_cast<const uint4*>(base + (col * static_cast<uint32_t>(a.ldw) + kk));
        }
    };
    // each wave a run of consecutive steps of every chunk, so that it reads whole cache lines of a column; a tile's
    // last step is followed by the next tile's first
    const int blocks = (K + kBlk - 1) / kBlk, chunk_steps = pl.chunk / kBlk;
    const int per = w4_share<W>(chunk_steps), run = w4_run<KB>(per);
    W4Fetch<kThrough> ahead(blockIdx.x, wave, per);
    auto fetch_next = [&](int i) __attribute__((always_inline)) {
        if (ahead.any(per, blocks, tiles)) fetch(i, ahead.tile, ahead.blk);
        ahead.next(wave, per, run, chunk_steps, blocks, gridDim.x);
    };
#pragma unroll
    for (int i = 0; i < KB; ++i) fetch_next(i);

    // A tile's scales and zero-points are read along the columns' rows, a pair of groups a load (one by one through the
    // products' lanes they would cost as many cache lines as the weights do), and go to LDS: kAhead loads a thread
    // ahead of the work before them, the rest (many groups) when they are stored.
    constexpr int kAhead = CT == 2 ? 3 : 2;
    const int halves = (groups + 1) / 2, items = kCols * halves;
    uint32_t sb[kAhead], zb[kAhead];
    auto load_item = [&](int tile, int e, uint32_t* s, uint32_t* z) __attribute__((always_inline)) {
        const int64_t n0 = static_cast<int64_t>(tile) * kCols;
        const int at = e < items ? e : 0, col = w4_div(at, pl.by_halves), gi = 2 * (at - col * halves);
        const int64_t n = n0 + col < a.N ? n0 + col : a.N - 1;
        const int g0 = gi + 1 < groups ? gi : groups - 2;   // an odd last group behind the one before it (there are two)
        __builtin_memcpy(s, static_cast<const uint16_t*>(a.ws) + n * a.ldws + g0, 4);
        if constexpr (Z == W4Zero::U4) *z = static_cast<const uint8_t*>(a.wz)[n * a.ldwz + (gi >> 1)];
        if constexpr (Z == W4Zero::Float) __builtin_memcpy(z, static_cast<const uint16_t*>(a.wz) + n * a.ldwz + g0, 4);
    };
    auto store_item = [&](int e, uint32_t s, uint32_t z, Pair* to) __attribute__((always_inline)) {
        if constexpr (!ANY) {
            if (e >= items) return;
            const int col = w4_div(e, pl.by_halves), gi = 2 * (e - col * halves);
            uint32_t z0 = 0, z1 = 0;
            const bool odd = gi + 1 >= groups;
            if (odd) s >>= 16;
            if constexpr (Z == W4Zero::U4) {
                z0 = __builtin_bit_cast(uint16_t, static_cast<_Float16>(z & 15));
                z1 = __builtin_bit_cast(uint16_t, static_cast<_Float16>(z >> 4));
            } else if constexpr (Z == W4Zero::Float) {
                if (odd) z >>= 16;
                z0 = z & 0xffffu;
                z1 = z >> 16;
            }
            *reinterpret_cast<uint2*>(to + col * pitch + gi) = make_uint2((s & 0xffffu) | z0 << 16, s >> 16 | z1 << 16);
        }
    };
    auto load_pairs = [&](int tile) __attribute__((always_inline)) {
        if constexpr (!ANY)
#pragma unroll
            for (int i = 0; i < kAhead; ++i) load_item(tile, threadIdx.x + i * 64 * W, sb + i, zb + i);
    };
    auto store_pairs = [&](int tile, Pair* to) __attribute__((always_inline)) {
        if constexpr (!ANY) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) store_item(threadIdx.x + i * 64 * W, sb[i], zb[i], to);
            for (int e = threadIdx.x + kAhead * 64 * W; e < items; e += 64 * W) {
                uint32_t s, z = 0;
                load_item(tile, e, &s, &z);
                store_item(e, s, z, to);
            }
        } else {
            const int64_t n0 = static_cast<int64_t>(tile) * kCols;
            for (int e = threadIdx.x; e < kCols * groups; e += 64 * W) {
                const int col = e / groups, gi = e - col * groups;
                const int64_t n = n0 + col < a.N ? n0 + col : a.N - 1;
                Pair p;
                p.s = load_as_f32(a.ws, a.s_dtype, n * a.ldws + gi);
                p.z = Z == W4Zero::U4 ? static_cast<float>((static_cast<const uint8_t*>(a.wz)[n * a.ldwz + (gi >> 1)] >> (4 * (gi & 1))) & 15)
                      : Z == W4Zero::Float ? load_as_f32(a.wz, a.z_dtype, n * a.ldwz + gi) : 0.0f;
                to[col * pitch + gi] = p;
            }
        }
    };
    load_pairs(blockIdx.x);
    __builtin_amdgcn_sched_barrier(0);

    // and-or takes one constant from a scalar register and one from a vector register, none from the instruction
    uint32_t magic = F16 ? 0x64006400u : 0x41804180u, low = F16 ? 0x000f000fu : 0x00780078u;
    asm volatile("" : "+v"(magic));
    asm volatile("" : "+s"(low));
    constexpr uint32_t kOne = F16 ? 0x3c003c00u : 0x3f803f80u;
    const W4Frag ones{{kOne, kOne, kOne, kOne}};

    w4_f32x4 y[CT];
    // row c of a product is row 4 (c % 4) + c / 4 of the tile
    const int row_c = 4 * (c & 3) + (c >> 2);
    const uint16_t* xrow = xs + (row_c < all ? row_c : 0) * stride + 8 * g;   // a row that is not there: not stored either

    auto compute = [&](int i, int blk, int k0, const Pair* pr) __attribute__((always_inline)) {
        const int gb = blk * kBlk;
        uint32_t v[CT][4];
#pragma unroll
        for (int t = 0; t < CT; ++t) {
            v[t][0] = w[i][t].x; v[t][1] = w[i][t].y; v[t][2] = w[i][t].z; v[t][3] = w[i][t].w;
            swap_lane_reg<4, 0>(v[t], lane);
            swap_lane_reg<5, 1>(v[t], lane);
            if constexpr (Z == W4Zero::Signed)          // a signed code with its top bit turned is c + 8
#pragma unroll
                for (int j = 0; j < 4; ++j) v[t][j] ^= 0x88888888u;
        }
        const int xo = gb - k0;
#pragma unroll
        for (int s = 0; s < kScales; ++s) {
            float sc[CT], zp[CT];
            // a step that K ends in: its missing group's pair is not there, any will do (its x is zeros)
            const int ks = gb + s * (kBlk / kScales), gi = (ks < K ? ks : K - 1) >> gshift;
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const Pair p = pr[(16 * t + c) * pitch + gi];
                sc[t] = p.scale();
                zp[t] = Z == W4Zero::Signed ? 8.0f : p.zero();
            }
            w4_f32x4 acc[CT], sum = w4_f32x4{0, 0, 0, 0};
#pragma unroll
            for (int t = 0; t < CT; ++t) acc[t] = w4_f32x4{0, 0, 0, 0};
#pragma unroll
            for (int jj = 0; jj < 4 / kScales; ++jj) {
                const int j = s * (4 / kScales) + jj;
                const uint4 q = *reinterpret_cast<const uint4*>(xrow + xo + 32 * j);
                const W4Frag x{{q.x, q.y, q.z, q.w}};
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    W4Frag f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // nibbles e and e + 4: to the lowest mantissa bits (fp16), or three above them
                        const uint32_t n = F16 ? v[t][j] >> (4 * e) : e == 0 ? v[t][j] << 3 : v[t][j] >> (4 * e - 3);
                        f.w[e] = (n & low) | magic;
                    }
                    if constexpr (F16) {
                        // 1024 + c - (1024 + z): exact
                        const _Float16 off = static_cast<_Float16>(-1024.0f - (Z == W4Zero::Float ? 0.0f : zp[t]));
                        const mq_f16x2 off2 = {off, off};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            f.w[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(mq_f16x2, f.w[e]) + off2);
                    }
                    acc[t] = w4_mfma<F16>(x, f, acc[t]);
                }
                if constexpr (kSum) sum = w4_mfma<F16>(x, ones, sum);
            }
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const float off = -16.0f - (Z == W4Zero::Float ? 0.0f : zp[t]);
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    const float d = F16 ? acc[t][e] : __builtin_fmaf(off, sum[e], acc[t][e]);
                    y[t][e] = __builtin_fmaf(sc[t], d, y[t][e]);
                    if constexpr (Z == W4Zero::Float) y[t][e] = __builtin_fmaf(zp[t], sum[e], y[t][e]);
                }
            }
        }
    };

    // The wave's steps b0 .. b2 - 1 of a chunk as the formula stands, weight by weight in fp32, for the sums that are not
    // finite: a shifted code's infinity less the shift's is NaN where the weight's alone is an infinity (or, for values
    // near the end of the range, finite).
    auto plain = [&](int tile, int b0, int b2, int k0, const Pair* pr, const w4_f32x4 (&before)[CT]) {
#pragma unroll 1
        for (int t = 0; t < CT; ++t) {
            const int64_t n = static_cast<int64_t>(tile) * kCols + 16 * t + c;
            const uint8_t* col = a.qw + (n < a.N ? n : a.N - 1) * a.ldw;
            w4_f32x4 s = before[t];
#pragma unroll 1
            for (int k = b0 * kBlk; k < b2 * kBlk && k < K; k += 8) {
                const uint32_t codes = *reinterpret_cast<const uint32_t*>(col + k / 2);
                const Pair p = pr[(16 * t + c) * pitch + (k >> gshift)];
#pragma unroll 1
                for (int i = 0; i < 8; ++i) {
                    int code = codes >> (4 * i) & 15;
                    if constexpr (Z == W4Zero::Signed) code = (code ^ 8) - 8;
                    const float w = Z == W4Zero::Signed ? p.scale() * static_cast<float>(code)
                                    : Z == W4Zero::U4   ? p.scale() * (static_cast<float>(code) - p.zero())
                                                        : __builtin_fmaf(p.scale(), static_cast<float>(code), p.zero());
                    const uint16_t* x = xs + (k - k0) + (i < 4 ? 2 * i : 2 * i - 7);    // in the order of the codes
#pragma unroll
                    for (int e = 0; e < NE; ++e) {
                        const uint32_t h = x[(4 * e + g < all ? 4 * e + g : 0) * stride];
                        s[e] = __builtin_fmaf(as_float(h, F16 ? kDtF16 : kDtBf16), w, s[e]);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < CT; ++u)
#pragma unroll
                for (int e = 0; e < NE; ++e)
                    if (u == t && !__builtin_isfinite(y[u][e])) y[u][e] = s[e];
        }
    };

    // A workgroup of eight waves takes every gridDim.x-th tile; x is staged once if it fits (one chunk), else for every tile anew.
    store_pairs(blockIdx.x, pairs);
    bool staged = false;
    int buf = 0;
    int tile = blockIdx.x;
    do {
        const Pair* pr = pairs + buf * kCols * pitch;
        const bool more = kThrough && tile + static_cast<int>(gridDim.x) < tiles;
        if (more) load_pairs(tile + gridDim.x);
#pragma unroll
        for (int t = 0; t < CT; ++t) y[t] = w4_f32x4{0, 0, 0, 0};
        for (int k0 = 0; k0 < K; k0 += pl.chunk) {
            if (!staged) {
                if (k0 > 0 || (kThrough && tile != static_cast<int>(blockIdx.x))) {
                    __syncthreads();                    // the last chunk has been read
#pragma unroll
                    for (int i = 0; i < PB; ++i) piece[i].load(a, pl, m0, mine + i * step, pieces, k0);
                }
                for (int e = mine; e < pieces; e += PB * step) {
                    if (e != mine)
#pragma unroll
                        for (int i = 0; i < PB; ++i) piece[i].load(a, pl, m0, e + i * step, pieces, k0);
#pragma unroll
                    for (int i = 0; i < PB; ++i)
                        if (e + i * step < pieces) piece[i].template store<F16>(a, pl, xs, stride);
                }
                __syncthreads();
                staged = pl.chunk >= K;
            }
            const int b0 = k0 / kBlk + wave * per, chunk_end = (k0 + pl.chunk) / kBlk;
            const int b1 = b0 + per < chunk_end ? b0 + per : chunk_end, b2 = b1 < blocks ? b1 : blocks;
            w4_f32x4 before[CT];
#pragma unroll
            for (int t = 0; t < CT; ++t) before[t] = y[t];
            for (int b = b0; b < b0 + run; b += KB) {
#pragma unroll
                for (int i = 0; i < KB; ++i) {
                    if (b + i < b2) compute(i, b + i, k0, pr);
                    fetch_next(i);
                }
            }
            bool wild = false;
#pragma unroll
            for (int t = 0; t < CT; ++t)
#pragma unroll
                for (int e = 0; e < NE; ++e) wild |= !__builtin_isfinite(y[t][e]);
            if (__ballot(wild)) plain(tile, b0, b2, k0, pr, before);
        }
        if (more) store_pairs(tile + gridDim.x, pairs + (buf ^ 1) * kCols * pitch);
        // the waves' sums, once the last tile's have been read
        __syncthreads();
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int e = 0; e < NE; ++e)
                if (4 * e + g < all) red[(wave * all + 4 * e + g) * kCols + 16 * t + c] = y[t][e];
        __syncthreads();
        for (int e = threadIdx.x; e < rows * kCols; e += 64 * W) {
            const int m = e / kCols, cc = e % kCols;
            const int64_t n = static_cast<int64_t>(tile) * kCols + cc;
            if (n >= a.N) continue;
            float s = 0.0f;
            for (int p = 0; p < pl.parts; ++p)
#pragma unroll
                for (int wv = 0; wv < W; ++wv) s += red[(wv * all + m * pl.parts + p) * kCols + cc];
            if (a.bias) s += load_as_f32(a.bias, a.bias_dtype, n);
            store_from_f32(a.y, a.y_dtype, (m0 + m) * a.ldy + n, s);
        }
        tile += gridDim.x;
        buf ^= 1;
    } while (kThrough && tile < tiles);
}

template <bool F16, W4Zero Z, int G, int CT, int NE, int W>
int launch_tiles(const W4A16Args& a, W4Plan pl, hipStream_t stream) {
    constexpr int KB = CT == 2 ? 3 : 4;
    constexpr int64_t kLds = 163840;                    // of a compute unit
    const int unit = a.hblock ? 1024 : kBlk;
    const int64_t tiles = (a.N + 16 * CT - 1) / (16 * CT);
    const int cus = device_cu_count();
    pl.pitch = static_cast<int>((a.K / a.group + 1) / 4 * 4 + 2);   // even, and 16 columns on different banks
    pl.by_halves = w4_inverse((a.K / a.group + 1) / 2);             // at most 32 columns x 512 halves
    const bool through = W == 8 && tiles > cus && cus > 0 && 2 * 16 * CT * pl.pitch * sizeof(W4Pair<G == 0>) < kLds / 2;
    const int64_t groups = through ? cus : tiles;
    pl.pair_bufs = groups < tiles ? 2 : 1;
    const int64_t pairs = static_cast<int64_t>(pl.pair_bufs) * 16 * CT * pl.pitch * sizeof(W4Pair<G == 0>);
    int step = W * KB * kBlk;                           // x a chunk at a time: whole rounds of the rings and whole pieces
    while (step % unit) step += W * KB * kBlk;
    const int64_t all = (a.K + unit - 1) / unit * unit;
    int64_t lds = 0;
    for (;; pl.rows_m = (pl.rows_m + 1) / 2) {
        const int64_t rows = pl.rows_m * pl.parts, red = W * rows * 16 * CT * 4;
        // all of K if the workgroup's share of LDS holds it (W = 8: one workgroup a compute unit; else four)
        int64_t room = W == 8 ? kLds : 40960;
        if (room > kLds - pairs - red) room = kLds - pairs - red;
        int64_t chunk = all;
        if (rows * (chunk + kPad) * 2 > room) {
            chunk = (room / (2 * rows) - kPad) / step * step;
            if (chunk < step) chunk = step;
            if (chunk > all) chunk = all;
        }
        pl.chunk = static_cast<int>(chunk);
        pl.by_pieces = w4_inverse(chunk / (a.hblock ? 1024 : 8));   // at most 16 rows x 4096 pieces
        lds = rows * (chunk + kPad) * 2 + pairs + red;
        if (lds <= kLds) break;
        if (pl.rows_m == 1) {
            set_error("w4a16: %lld bytes of LDS for K=%lld", (long long)lds, (long long)a.K);
            return -2;
        }
    }
    auto kern = w4a16_kernel<F16, Z, G, CT, NE, KB, W>;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(lds)) != hipSuccess) {
        (void)hipGetLastError();
        set_error("w4a16: cannot reserve %lld bytes of LDS", (long long)lds);
        return -3;
    }
    const dim3 grid(static_cast<unsigned>(groups), static_cast<unsigned>((a.M + pl.rows_m - 1) / pl.rows_m));
    hipLaunchKernelGGL(kern, grid, dim3(64 * W), lds, stream, a, pl);
    return launch_status("w4a16");
}

template <bool F16, W4Zero Z, int G>
int launch_rows(const W4A16Args& a, hipStream_t stream) {
    W4Plan pl{};
    // fp32 rows (and rotated rows for an fp32 output) need three bf16 parts; rotated 16-bit rows that are rounded
    // to 16 bits again two: 16 bits of every rotated value, an error of 2^-16 of it against the output's 2^-8
    pl.parts = a.x_dtype == kDtF32 || (a.hblock && a.y_dtype == kDtF32) ? 3 : a.hblock ? 2 : 1;
    const int most = 16 / pl.parts;                     // a product's rows; more go to another blockIdx.y
    pl.rows_m = static_cast<int>(a.M < most ? a.M : most);
    const int cus = device_cu_count();
    if (pl.rows_m * pl.parts <= 4) {
        // two column tiles a workgroup stage x half as often (a rotated row of 3072 into 18432: 13.9 us, with one 14.9);
        // one where that would leave units idle (4096 x 4096: 6.0 us, with two 8.3)
        if constexpr (G != 0)
            if ((a.N + 31) / 32 >= 2 * (cus > 0 ? cus : 256)) return launch_tiles<F16, Z, G, 2, 1, 4>(a, pl, stream);
        // a workgroup a compute unit at most: eight waves, where four would need more than two rounds of their rings (a
        // rotated row of 12288 into 3072: 15.4 us, with four 25.0; 4096 x 4096: 6.5, with four 6.0) or the pairs are
        // loaded one by one (groups of 32 there: 7.7 to 8.8 us, with four 9.2)
        if ((a.N + 15) / 16 <= (cus > 0 ? cus : 256) && (G == 0 || a.K > 2 * 4 * 4 * kBlk))
            return launch_tiles<F16, Z, G, 1, 1, 8>(a, pl, stream);
        return launch_tiles<F16, Z, G, 1, 1, 4>(a, pl, stream);
    }
    // more rows: one workgroup a compute unit keeps all of x in LDS and goes through the tiles (16 rows of 4096 into
    // 12288: 17.9 us, 30.9 a tile a workgroup; one rotated row of 3072 into 18432 that way: 20.4 against 13.9 us)
    return launch_tiles<F16, Z, G, 1, 4, 8>(a, pl, stream);
}

template <bool F16>
int launch_kind(const W4A16Args& a, hipStream_t stream) {
    const bool any = a.group == 32 || a.s_dtype != kDtF16 || (a.zero == W4Zero::Float && a.z_dtype != kDtF16);
    const int g = any || a.K < 2 * a.group ? 0 : a.group;   // pairs of groups are read together
    auto go = [&](auto z) {
        constexpr W4Zero Z = decltype(z)::value;
        return g == 0 ? launch_rows<F16, Z, 0>(a, stream) : g == 64 ? launch_rows<F16, Z, 64>(a, stream)
                                                                    : launch_rows<F16, Z, 128>(a, stream);
    };
    switch (a.zero) {
        case W4Zero::Signed: return go(std::integral_constant<W4Zero, W4Zero::Signed>{});
        case W4Zero::U4: return go(std::integral_constant<W4Zero, W4Zero::U4>{});
        default: return go(std::integral_constant<W4Zero, W4Zero::Float>{});
    }
}

}  // namespace

int launch_w4a16(const W4A16Args& a, hipStream_t stream) {
    return a.x_dtype == kDtF16 && a.hblock == 0 ? launch_kind<true>(a, stream) : launch_kind<false>(a, stream);
}

}  // namespace mq
