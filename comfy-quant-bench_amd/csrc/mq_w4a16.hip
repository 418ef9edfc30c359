// y = x W^T + bias with 4-bit weights, a scale per group of K values and activations in floating point,
// optionally rotated by Hadamard blocks: for few rows, so bound by reading the weights once, and next to that by
// unpacking them: at 8 TB/s a SIMD has some 78 VALU operations for the 1 KB of a wave's step.
//
// The codes go through MFMA as 16-bit floats without being scaled first (a scaled weight would be rounded):
// bits of a code are or-ed into the mantissa of a constant, which makes 128 + c in bf16 (1024 + c in fp16), seven
// operations for the eight codes of a dword. What is too much is taken off exactly: in fp16 by a packed
// subtraction (which takes the zero-point with it), in bf16 behind the product, where acc - (128 + z) sum(x)
// needs the group's sum of x, a product with ones. Each group's fp32 sum is then scaled into the output's.
// Rows of x that have more bits than the 16-bit type are split into as many rows as hold them (fp32: three
// bf16 rows, exactly), which the 16 rows of a product have room for, and the rows' outputs are added at the end.
//
// A workgroup owns 16 CT output columns; its four waves share the K values, 128 at a time: lane (c, g) reads the
// 16 bytes of column c that hold values 32 g .. 32 g + 31 (64 bytes of each of 16 rows a load), and two exchanges
// of lane and register index bits leave in register j the dword of values 32 j + 8 g. A wave keeps KB steps'
// loads in flight in a ring of registers. x is staged in LDS, as much of it as fits, in the order of the unpacked
// codes (0 4 1 5 2 6 3 7); the waves' sums are added there at the end. Row 4 e + g of x is row 4 g + e of
// a product, so that up to 4 rows come out in one register of every lane, up to 8 in two.
#include <type_traits>

#include "mq_device.h"
#include "mq_internal.h"
#include "mq_rotate.h"

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
};

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
        m = at / per;
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
    __device__ __forceinline__ void store(const W4A16Args& a, const W4Plan& pl, uint16_t* xs, int stride) {
        uint16_t* to = xs + m * pl.parts * stride + kk;
        if (a.hblock) {
            if (a.x_dtype == kDtF32) put<kDtF32, true>(a, pl, to, stride);
            else if (a.x_dtype == kDtF16) put<kDtF16, true>(a, pl, to, stride);
            else put<kDtBf16, true>(a, pl, to, stride);
        } else {
            if (a.x_dtype == kDtF32) put<kDtF32, false>(a, pl, to, stride);
            else put<kDtBf16, false>(a, pl, to, stride);
        }
    }
};

constexpr int kWaves = 4;

// F16: fp16 rows and products, else bf16; Z: zero-points; G: groups of 64 or 128 with fp16 scales and zero-points,
// or 0: any group and type; RT: 16-row tiles; CT: 16-column tiles; NE: registers of a product that
// hold rows; KB: 128-value steps in flight.
template <bool F16, W4Zero Z, int G, int RT, int CT, int NE, int KB>
__global__ void __launch_bounds__(64 * kWaves, RT * CT >= 4 ? 2 : RT * CT >= 2 ? 3 : 4) w4a16_kernel(W4A16Args a, W4Plan pl) {
    static_assert(RT == 1 || NE == 4, "more rows than a product has fill all its registers");
    constexpr bool ANY = G == 0;
    constexpr int kScales = ANY ? 4 : kBlk / G;         // scales that a step uses (any: the same ones again for larger groups)
    constexpr int kHeld = ANY ? 4 : 1;                  // registers that hold them: two fp16 scales in one
    constexpr bool kSum = !F16 || Z == W4Zero::Float;   // the sum of x is needed
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int K = static_cast<int>(a.K);
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * pl.rows_m;
    const int rows = static_cast<int>(a.M - m0 < pl.rows_m ? a.M - m0 : pl.rows_m);
    const int all = rows * pl.parts;                    // staged rows
    const int stride = pl.chunk + kPad;
    uint16_t* xs = reinterpret_cast<uint16_t*>(lds);
    uint16_t* zero = xs + pl.rows_m * pl.parts * stride;   // 16 bytes of zeros: the rows of a product that are not there
    if (threadIdx.x < 8) zero[threadIdx.x] = 0;

    // loads complete in the order of their issue: the first piece of x ahead of the weights, so that x is
    // staged while the weights are on their way
    const int pieces = rows * (pl.chunk / (a.hblock ? 1024 : 8));
    const int mine = a.hblock ? wave : static_cast<int>(threadIdx.x), step = a.hblock ? kWaves : 64 * kWaves;
    W4Piece piece;
    piece.load(a, pl, m0, mine, pieces, 0);
    __builtin_amdgcn_sched_barrier(0);

    const int64_t n0 = static_cast<int64_t>(blockIdx.x) * 16 * CT;
    // addresses as a scalar base and a 32-bit offset of the lane: its column's, within the workgroup's
    const char* wbase = reinterpret_cast<const char*>(a.qw) + n0 * a.ldw;
    const char* sbase = static_cast<const char*>(a.ws) + n0 * a.ldws * (ANY && a.s_dtype == kDtF32 ? 4 : 2);
    const char* zbase = static_cast<const char*>(a.wz) +
                        n0 * a.ldwz * (Z == W4Zero::U4 ? 1 : ANY && a.z_dtype == kDtF32 ? 4 : 2);
    uint32_t wo[CT], so[CT], zo[CT];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
        const int left = static_cast<int>(a.N - 1 - n0 < 16 * CT ? a.N - 1 - n0 : 16 * CT);
        const uint32_t col = 16 * t + c < left ? 16 * t + c : left;       // columns past N read the last one's weights
        wo[t] = col * static_cast<uint32_t>(a.ldw);
        so[t] = col * static_cast<uint32_t>(a.ldws);
        zo[t] = col * static_cast<uint32_t>(a.ldwz);
    }
    const int gshift = a.group == 32 ? 5 : a.group == 64 ? 6 : 7;
    const uint32_t last = static_cast<uint32_t>(K / 2 - 16);
    uint4 w[KB][CT];
    uint32_t sb[KB][CT][kHeld], zb[KB][CT][kHeld];      // scales and zero-points as they are stored
    const int groups = K >> gshift;
    // step `blk` (128 values) into ring place i; past the end of K the last values
    auto fetch = [&](int i, int blk) __attribute__((always_inline)) {
        const uint32_t at = static_cast<uint32_t>(blk) * (kBlk / 2) + 16 * g;
        const uint32_t kk = at < last ? at : last;
#pragma unroll
        for (int t = 0; t < CT; ++t) w[i][t] = *reinterpret_cast<const uint4*>(wbase + (wo[t] + kk));
        auto half = [](const char* base, int64_t at, uint32_t o) __attribute__((always_inline)) {
            return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(base + 2 * at + 2 * o));
        };
        if constexpr (ANY) {
            // one branch on a type around all its loads: inside a branch each, they would be waited for one by one
            auto each = [&](auto&& f) __attribute__((always_inline)) {
#pragma unroll
                for (int s = 0; s < kScales; ++s) {
                    const int ks = blk * kBlk + s * (kBlk / kScales);
                    const int gi = (ks < K ? ks : K - 1) >> gshift;
#pragma unroll
                    for (int t = 0; t < CT; ++t) f(t, s, gi);
                }
            };
            auto word = [](const char* base, int64_t at, uint32_t o) __attribute__((always_inline)) {
                return *reinterpret_cast<const uint32_t*>(base + 4 * at + 4 * o);
            };
            if (a.s_dtype != kDtF32) each([&](int t, int s, int gi) { sb[i][t][s] = half(sbase, gi, so[t]); });
            else each([&](int t, int s, int gi) { sb[i][t][s] = word(sbase, gi, so[t]); });
            if constexpr (Z == W4Zero::U4) {
                each([&](int t, int s, int gi) { zb[i][t][s] = *reinterpret_cast<const uint8_t*>(zbase + (gi >> 1) + zo[t]); });
            } else if constexpr (Z == W4Zero::Float) {
                if (a.z_dtype != kDtF32) each([&](int t, int s, int gi) { zb[i][t][s] = half(zbase, gi, zo[t]); });
                else each([&](int t, int s, int gi) { zb[i][t][s] = word(zbase, gi, zo[t]); });
            }
        } else {
            // both scales of a step in one dword (an odd last group's alone); its uint4 zero-points are one byte
            const int gi = blk * kScales < groups ? blk * kScales : groups - 1;
            auto pair = [&](const char* base, uint32_t o) __attribute__((always_inline)) {
                if (kScales == 1 || gi + 1 >= groups) return half(base, gi, o);
                uint32_t v;
                __builtin_memcpy(&v, base + 2 * static_cast<int64_t>(gi) + 2 * o, 4);
                return v;
            };
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                sb[i][t][0] = pair(sbase, so[t]);
                if constexpr (Z == W4Zero::U4) zb[i][t][0] = *reinterpret_cast<const uint8_t*>(zbase + (gi >> 1) + zo[t]);
                else if constexpr (Z == W4Zero::Float) zb[i][t][0] = pair(zbase, zo[t]);
            }
        }
    };
    const int blocks = (K + kBlk - 1) / kBlk;
#pragma unroll
    for (int i = 0; i < KB; ++i) fetch(i, wave + i * kWaves);
    __builtin_amdgcn_sched_barrier(0);

    // and-or takes one constant from a scalar register and one from a vector register, none from the instruction
    uint32_t magic = F16 ? 0x64006400u : 0x43004300u, low = 0x000f000fu;
    asm volatile("" : "+v"(magic));
    asm volatile("" : "+s"(low));
    constexpr uint32_t kOne = F16 ? 0x3c003c00u : 0x3f803f80u;
    const W4Frag ones{{kOne, kOne, kOne, kOne}};

    w4_f32x4 y[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t) y[r][t] = w4_f32x4{0, 0, 0, 0};
    // row c of a product is row 4 (c % 4) + c / 4 of the tile
    const uint16_t* xrow[RT];
    bool there[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int row = 16 * r + 4 * (c & 3) + (c >> 2);
        there[r] = row < all;
        xrow[r] = there[r] ? xs + row * stride + 8 * g : zero;
    }

    auto compute = [&](int i, int blk, int k0) __attribute__((always_inline)) {
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
            const int gi = (gb + s * (kBlk / kScales)) >> gshift;
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                if constexpr (ANY) {
                    sc[t] = as_float(sb[i][t][s], a.s_dtype);
                    if constexpr (Z == W4Zero::Float) zp[t] = as_float(zb[i][t][s], a.z_dtype);
                } else {
                    sc[t] = as_float(sb[i][t][0] >> (16 * s), kDtF16);
                    if constexpr (Z == W4Zero::Float) zp[t] = as_float(zb[i][t][0] >> (16 * s), kDtF16);
                }
                if constexpr (Z == W4Zero::Signed) zp[t] = 8.0f;
                else if constexpr (Z == W4Zero::U4) zp[t] = static_cast<float>((zb[i][t][ANY ? s : 0] >> (4 * (gi & 1))) & 15);
            }
            w4_f32x4 acc[RT][CT], sum[RT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                sum[r] = w4_f32x4{0, 0, 0, 0};
#pragma unroll
                for (int t = 0; t < CT; ++t) acc[r][t] = w4_f32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int jj = 0; jj < 4 / kScales; ++jj) {
                const int j = s * (4 / kScales) + jj;
                W4Frag x[RT];
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const uint4 q = *reinterpret_cast<const uint4*>(xrow[r] + (there[r] ? xo + 32 * j : 0));
                    x[r] = W4Frag{{q.x, q.y, q.z, q.w}};
                }
#pragma unroll
                for (int t = 0; t < CT; ++t) {
                    W4Frag f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) f.w[e] = ((v[t][j] >> (4 * e)) & low) | magic;
                    if constexpr (F16) {
                        // 1024 + c - (1024 + z): exact
                        const _Float16 off = static_cast<_Float16>(-1024.0f - (Z == W4Zero::Float ? 0.0f : zp[t]));
                        const mq_f16x2 off2 = {off, off};
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            f.w[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(mq_f16x2, f.w[e]) + off2);
                    }
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[r][t] = w4_mfma<F16>(x[r], f, acc[r][t]);
                }
                if constexpr (kSum)
#pragma unroll
                    for (int r = 0; r < RT; ++r) sum[r] = w4_mfma<F16>(x[r], ones, sum[r]);
            }
#pragma unroll
            for (int t = 0; t < CT; ++t) {
                const float off = -128.0f - (Z == W4Zero::Float ? 0.0f : zp[t]);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int e = 0; e < NE; ++e) {
                        const float d = F16 ? acc[r][t][e] : __builtin_fmaf(off, sum[r][e], acc[r][t][e]);
                        y[r][t][e] = __builtin_fmaf(sc[t], d, y[r][t][e]);
                        if constexpr (Z == W4Zero::Float) y[r][t][e] = __builtin_fmaf(zp[t], sum[r][e], y[r][t][e]);
                    }
            }
        }
    };

    for (int k0 = 0; k0 < K; k0 += pl.chunk) {
        if (k0 > 0) {
            __syncthreads();                            // the last chunk has been read
            piece.load(a, pl, m0, mine, pieces, k0);
        }
        for (int e = mine; e < pieces; e += step) {
            if (e != mine) piece.load(a, pl, m0, e, pieces, k0);
            piece.store(a, pl, xs, stride);
        }
        __syncthreads();
        const int b0 = k0 / kBlk, b1 = b0 + pl.chunk / kBlk < blocks ? b0 + pl.chunk / kBlk : blocks;
        for (int b = b0; b < b1; b += kWaves * KB) {
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                const int blk = b + wave + i * kWaves;
                if (blk < b1) compute(i, blk, k0);
                if (blk + kWaves * KB < blocks) fetch(i, blk + kWaves * KB);
            }
        }
    }
    // the waves' sums: [wave][row][column]
    __syncthreads();
    float* red = reinterpret_cast<float*>(lds);
    constexpr int kCols = 16 * CT;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                const int row = 16 * r + 4 * e + g;
                if (row < all) red[(wave * all + row) * kCols + 16 * t + c] = y[r][t][e];
            }
    __syncthreads();
    for (int e = threadIdx.x; e < rows * kCols; e += 64 * kWaves) {
        const int m = e / kCols, cc = e % kCols;
        const int64_t n = n0 + cc;
        if (n >= a.N) continue;
        float s = 0.0f;
        for (int p = 0; p < pl.parts; ++p)
#pragma unroll
            for (int wv = 0; wv < kWaves; ++wv) s += red[(wv * all + m * pl.parts + p) * kCols + cc];
        if (a.bias) s += load_as_f32(a.bias, a.bias_dtype, n);
        store_from_f32(a.y, a.y_dtype, (m0 + m) * a.ldy + n, s);
    }
}

template <bool F16, W4Zero Z, int G, int RT, int CT, int NE>
int launch_tiles(const W4A16Args& a, W4Plan pl, hipStream_t stream) {
    constexpr int KB = RT == 1 && NE == 1 ? (G == 0 ? 3 : 4) : RT == 1 ? 2 : 1;
    constexpr int round = kWaves * KB * kBlk;           // values of K that the waves' rings cover
    const int unit = a.hblock ? 1024 : kBlk;
    const int rows = pl.rows_m * pl.parts;
    // all of K if 40 KB hold it (four workgroups a compute unit), else whole rounds of the rings
    const int64_t all = (a.K + unit - 1) / unit * unit;
    int64_t chunk = all;
    if (2 * rows * chunk > 40960) {
        int step = round;                               // whole rounds and whole pieces of x
        while (step % unit) step += round;
        chunk = 40960 / (2 * rows) / step * step;
        if (chunk < step) chunk = step;
        if (chunk > all) chunk = all;
    }
    pl.chunk = static_cast<int>(chunk);
    const size_t stage = static_cast<size_t>(rows) * (chunk + kPad) * 2 + 16;
    const size_t red = static_cast<size_t>(kWaves) * rows * 16 * CT * 4;
    const size_t lds = stage > red ? stage : red;
    auto kern = w4a16_kernel<F16, Z, G, RT, CT, NE, KB>;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(lds)) != hipSuccess) {
        set_error("w4a16: cannot reserve %zu bytes of LDS", lds);
        return -3;
    }
    const dim3 grid(static_cast<unsigned>((a.N + 16 * CT - 1) / (16 * CT)),
                    static_cast<unsigned>((a.M + pl.rows_m - 1) / pl.rows_m));
    hipLaunchKernelGGL(kern, grid, dim3(64 * kWaves), lds, stream, a, pl);
    return launch_status("w4a16");
}

template <bool F16, W4Zero Z, int G>
int launch_rows(const W4A16Args& a, hipStream_t stream) {
    W4Plan pl{};
    // fp32 rows (and rotated rows for an fp32 output) need three bf16 parts; rotated 16-bit rows that are rounded
    // to 16 bits again two: 16 bits of every rotated value, an error of 2^-16 of it against the output's 2^-8
    pl.parts = a.x_dtype == kDtF32 || (a.hblock && a.y_dtype == kDtF32) ? 3 : a.hblock ? 2 : 1;
    const int most = 64 / pl.parts;
    pl.rows_m = static_cast<int>(a.M < most ? a.M : most);
    const int rows = pl.rows_m * pl.parts, rt = (rows + 15) / 16;
    const int cus = device_cu_count();
    // two column tiles a workgroup read the staged rows half as often; one where that would leave units idle
    const bool two = G != 0 && (a.N + 31) / 32 >= 2 * (cus > 0 ? cus : 256);
    if (rows <= 4) return launch_tiles<F16, Z, G, 1, 1, 1>(a, pl, stream);
    if (rt <= 1) return launch_tiles<F16, Z, G, 1, 1, 4>(a, pl, stream);
    if constexpr (G != 0) {
        if (rt == 2 && two) return launch_tiles<F16, Z, G, 2, 2, 4>(a, pl, stream);
        if (rt > 2 && two) return launch_tiles<F16, Z, G, 4, 2, 4>(a, pl, stream);
    }
    return rt == 2 ? launch_tiles<F16, Z, G, 2, 1, 4>(a, pl, stream) : launch_tiles<F16, Z, G, 4, 1, 4>(a, pl, stream);
}

template <bool F16>
int launch_kind(const W4A16Args& a, hipStream_t stream) {
    const bool any = a.group == 32 || a.s_dtype != kDtF16 || (a.zero == W4Zero::Float && a.z_dtype != kDtF16);
    const int g = any ? 0 : a.group;
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
