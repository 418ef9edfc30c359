// Root-mean-square norm of rows, with the residual's addition in front of it and, behind it, an output in the rows' own
// type or as int8 codes with a scale per row, rotated by Hadamard blocks where the linear that reads them asks for it.
//
//   h = T(x + r)                       T: the rows' type; what the residual stream holds, so the norm is taken of it
//   y = h * w / sqrt(mean(h^2) + eps)  in fp32
//   out = T(y), or z = y (H y per block), s = max(max |z| / 127, 1e-10), q = rne(z / s)
//
// Memory-bound: a row is read once, kept in fp32 registers and written once. y is not rounded to T in front of the
// quantizer: that would move one code in twenty of a 16-bit row by a step.
//
// A row is `waves` wavefronts, each with UNITS pieces of 64 lanes x V values in registers (V = 8; rotated rows 16,
// in the order of columns that the rotation's stages want). The sum of squares, and of codes the largest value, meet in LDS.
// As many waves as have a piece: 10 for 5120 values (16, a power of two, 6 of them idle: 65 us instead of 61 rotated).
//
// 8192 rows of 4096 bf16 values with a residual, 268 MB: 43 us, 6.2 TB/s (a copy 5.1). 8192 of 5120 fp16 to codes
// rotated by 256, 294 MB: 63 us, 4.7 TB/s, three stages of the rotation on the VALU and two barriers between the reads and the
// writes. One row of 2048: 2.3 us, the launch.
#include "mq_internal.h"
#include "mq_rotate.h"

#pragma clang fp contract(off)

namespace mq {
namespace {

// Pieces of a row at any address that its type allows: the hardware takes wide accesses of any alignment, and at
// multiples of 16 bytes they cost what aligned ones do.
struct __attribute__((packed, aligned(2))) Piece16 {
    uint32_t w[4];
};
struct __attribute__((packed, aligned(4))) Piece32 {
    float f[4];
};
struct __attribute__((packed, aligned(1))) Codes {
    uint32_t w[4];
};
struct __attribute__((packed, aligned(1))) Codes8 {
    uint32_t w[2];
};

template <int DT>
constexpr int words_of(int n) { return DT == kDtF32 ? n : n / 2; }

// n <= V values of row p from column c on (elements); the others 0.
template <int DT, int V>
__device__ __forceinline__ void load_piece(const void* p, int64_t c, int n, uint32_t (&w)[words_of<DT>(V)]) {
    constexpr int kWords = words_of<DT>(V);
    if (n == V) {
        if constexpr (DT == kDtF32) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                const Piece32 x = *reinterpret_cast<const Piece32*>(static_cast<const float*>(p) + c + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * i + e] = __float_as_uint(x.f[e]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V / 8; ++i) {
                const Piece16 x = *reinterpret_cast<const Piece16*>(static_cast<const uint16_t*>(p) + c + 8 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * i + e] = x.w[e];
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n) {
            if constexpr (DT == kDtF32) w[i] = __float_as_uint(static_cast<const float*>(p)[c + i]);
            else w[i / 2] |= static_cast<uint32_t>(static_cast<const uint16_t*>(p)[c + i]) << (16 * (i & 1));
        }
}

template <int DT, int V>
__device__ __forceinline__ void store_piece(void* p, int64_t c, int n, const uint32_t (&w)[words_of<DT>(V)]) {
    if (n == V) {
        if constexpr (DT == kDtF32) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i)
                *reinterpret_cast<Piece32*>(static_cast<float*>(p) + c + 4 * i) =
                    Piece32{{__uint_as_float(w[4 * i]), __uint_as_float(w[4 * i + 1]), __uint_as_float(w[4 * i + 2]),
                             __uint_as_float(w[4 * i + 3])}};
        } else {
#pragma unroll
            for (int i = 0; i < V / 8; ++i)
                *reinterpret_cast<Piece16*>(static_cast<uint16_t*>(p) + c + 8 * i) =
                    Piece16{{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]}};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < n) {
            if constexpr (DT == kDtF32) static_cast<float*>(p)[c + i] = __uint_as_float(w[i]);
            else static_cast<uint16_t*>(p)[c + i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
        }
}

template <int DT, int V>
__device__ __forceinline__ void unpack(const uint32_t (&w)[words_of<DT>(V)], float* v) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (DT == kDtF32) v[i] = __uint_as_float(w[i]);
        else if constexpr (DT == kDtF16) v[i] = f16_bits_to_f32(static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1))));
        else v[i] = i & 1 ? bf16hi(w[i / 2]) : bf16lo(w[i / 2]);
    }
}

template <int DT, int V>
__device__ __forceinline__ void pack(const float* v, uint32_t (&w)[words_of<DT>(V)]) {
#pragma unroll
    for (int i = 0; i < words_of<DT>(V); ++i) {
        if constexpr (DT == kDtF32) w[i] = __float_as_uint(v[i]);
        else w[i] = pack_16x2(v[2 * i], v[2 * i + 1], DT);
    }
}

__device__ __forceinline__ float wave_sum(float v) {
    v += dpp_mov<kQuadXor1>(v);
    v += dpp_mov<kQuadXor2>(v);
    v += dpp_mov<kRowRor4>(v);
    v += dpp_mov<kRowRor8>(v);
    const float r0 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 0));
    const float r1 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 16));
    const float r2 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 32));
    const float r3 = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 48));
    return (r0 + r1) + (r2 + r3);
}

constexpr int kMostWaves = 16;
constexpr int kManyRows = 1024;

// BLK: -1 floating output, 0 codes, 16 / 64 / 256 codes of rotated rows.
template <int DT, int BLK, int UNITS>
__global__ void __launch_bounds__(1024) norm_kernel(NormArgs a, int waves) {
    constexpr bool kCodes = BLK >= 0, kRotate = BLK > 0;
    constexpr int V = kRotate ? 16 : 8, kWords = words_of<DT>(V);
    __shared__ float part[2][kMostWaves];
    extern __shared__ float turn[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int of_row = wave % waves, slot0 = wave - of_row;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / 64 / waves) + wave / waves;
    const bool here = row < a.M;
    // the lane's first column of a piece: 16 values of segment s = (L >> 2) + 16 (L & 3) where stages follow
    const int first = kRotate ? 16 * ((lane >> 2) + 16 * (lane & 3)) : 8 * lane;
    const int es = DT == kDtF32 ? 4 : 2;
    const char* x = static_cast<const char*>(a.x) + row * a.ldx * es;
    const char* r = a.r ? static_cast<const char*>(a.r) + row * a.ldr * es : nullptr;

    int col[UNITS], have[UNITS];
    float v[UNITS][V];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        col[u] = (u * waves + of_row) * 64 * V + first;
        const int left = here ? static_cast<int>(a.K) - col[u] : 0;
        have[u] = left < 0 ? 0 : left < V ? left : V;
    }
    uint32_t xw[UNITS][kWords], rw[UNITS][kWords];
#pragma unroll
    for (int u = 0; u < UNITS; ++u) load_piece<DT, V>(x, col[u], have[u], xw[u]);
    if (r)
#pragma unroll
        for (int u = 0; u < UNITS; ++u) load_piece<DT, V>(r, col[u], have[u], rw[u]);
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
        unpack<DT, V>(xw[u], v[u]);
        if (r) {
            float b[V];
            unpack<DT, V>(rw[u], b);
#pragma unroll
            for (int i = 0; i < V; ++i) v[u][i] += b[i];
            pack<DT, V>(v[u], xw[u]);
            unpack<DT, V>(xw[u], v[u]);
            store_piece<DT, V>(static_cast<char*>(a.h) + row * a.ldh * es, col[u], have[u], xw[u]);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sum = __builtin_fmaf(v[u][i], v[u][i], sum);
    }
    sum = wave_sum(sum);
    if (waves > 1) {
        if (lane == 0) part[0][wave] = sum;
        __syncthreads();
        sum = 0.0f;
        for (int i = 0; i < waves; ++i) sum += part[0][slot0 + i];
    }
    const float inv = 1.0f / __builtin_sqrtf(sum / static_cast<float>(a.K) + a.eps);
    float most = 0.0f;
    bool nan = false;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[u][i] *= inv;
        if (a.w) {
            float w[V];
            if (a.w_dtype == kDtF32) {
                uint32_t ww[V];
                load_piece<kDtF32, V>(a.w, col[u], have[u], ww);
                unpack<kDtF32, V>(ww, w);
            } else {
                uint32_t ww[V / 2];
                load_piece<kDtBf16, V>(a.w, col[u], have[u], ww);
                if (a.w_dtype == kDtF16) unpack<kDtF16, V>(ww, w);
                else unpack<kDtBf16, V>(ww, w);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) v[u][i] *= w[i];
        }
        if constexpr (!kCodes) {
            uint32_t o[kWords];
            pack<DT, V>(v[u], o);
            store_piece<DT, V>(static_cast<char*>(a.y) + row * a.ldy * es, col[u], have[u], o);
        } else {
            if constexpr (kRotate) {
                const LdsTranspose tr{turn + wave * kTrWave + (lane & 3) * kTrG + (lane >> 2),
                                      turn + wave * kTrWave + (lane & 3) * kTrG + (lane >> 2) * kTrS};
                rotate_chunk_lds<BLK>(v[u], tr);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float m = __builtin_fabsf(v[u][i]);
                nan |= !(m == m);
                most = __builtin_fmaxf(most, m);
            }
        }
    }
    if constexpr (kCodes) {
        // a row that holds a NaN or an infinity has no scale: codes 0, scale NaN, so it reads back as NaN
        most = nan || most == __builtin_inff() ? __builtin_inff() : most;
        most = wave_max_nonneg(most);
        if (waves > 1) {
            if (lane == 0) part[1][wave] = most;
            __syncthreads();
            most = 0.0f;
            for (int i = 0; i < waves; ++i) most = __builtin_fmaxf(most, part[1][slot0 + i]);
        }
        const bool fine = most < __builtin_inff();
        const float s = __builtin_fmaxf(div_limit<127>(most), 1e-10f), rs = recip_row(s);
        if (here && lane == 0 && of_row == 0) a.s[row] = fine ? s : __builtin_nanf("");
        uint8_t* q = static_cast<uint8_t*>(a.y) + row * a.ldy;
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            uint32_t c[V / 4];
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                if (!fine)
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[u][4 * i + e] = 0.0f;
                c[i] = quant4_word<127, false>(&v[u][4 * i], 1.0f, rs, s);
            }
            if (have[u] == V) {
                if constexpr (V == 16) *reinterpret_cast<Codes*>(q + col[u]) = Codes{{c[0], c[1], c[2], c[3]}};
                else *reinterpret_cast<Codes8*>(q + col[u]) = Codes8{{c[0], c[1]}};
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i < have[u]) q[col[u] + i] = static_cast<uint8_t>(c[i / 4] >> (8 * (i & 3)));
            }
        }
    }
}

template <int DT, int BLK, int UNITS>
int launch_units(const NormArgs& a, int waves, hipStream_t stream) {
    // rows of a few waves share a workgroup of four
    const int rows = waves < 4 ? 4 / waves : 1;
    const size_t lds = BLK > 0 ? sizeof(float) * kTrWave * waves * rows : 0;
    const int64_t most = kMostThreads / (64 * waves * rows) * rows;         // rows of a launch
    const int64_t es = DT == kDtF32 ? 4 : 2;
    auto kern = norm_kernel<DT, BLK, UNITS>;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(lds)) != hipSuccess) {
        (void)hipGetLastError();
        set_error("rms_norm: cannot reserve %zu bytes of LDS", lds);
        return -3;
    }
    for (int64_t m = 0; m < a.M; m += most) {
        NormArgs b = a;
        b.x = static_cast<const char*>(a.x) + m * a.ldx * es;
        b.r = a.r ? static_cast<const char*>(a.r) + m * a.ldr * es : nullptr;
        b.h = a.h ? static_cast<char*>(a.h) + m * a.ldh * es : nullptr;
        b.y = static_cast<char*>(a.y) + m * a.ldy * (BLK >= 0 ? 1 : es);
        b.s = a.s ? a.s + m : nullptr;
        b.M = a.M - m < most ? a.M - m : most;
        hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>((b.M + rows - 1) / rows)), dim3(64 * waves * rows), lds, stream, b, waves);
    }
    return launch_status("rms_norm");
}

template <int DT, int BLK>
int launch_block(const NormArgs& a, hipStream_t stream) {
    const int64_t pieces = (a.K + (BLK > 0 ? 1024 : 512) - 1) / (BLK > 0 ? 1024 : 512);
    auto waves_for = [&](int units) { return static_cast<int>((pieces + units - 1) / units); };
    // One piece a wave, so that few rows have many waves and all of a row is on its way at once; of many rows, and of long ones,
    // which have waves enough, a wave has two, and half as many waves meet at a row's barriers. (bf16, one against two, us:
    // 64 x 4096 2.9 / 3.2, 512 x 4096 4.4 / 4.6, 2048 x 4096 12.3 / 11.5, 512 x 8192 6.7 / 6.5, 8192 x 5120 to codes 67 / 53;
    // rotated 64 x 4096 4.7 / 6.4, 2048 x 4096 14.4 / 15.7; fp32, twice the registers, 8192 x 2560 68 / 74.)
    const bool two = BLK <= 0 && DT != kDtF32 && (pieces >= 16 || (a.M >= kManyRows && pieces > 1));
    if (waves_for(1) <= kMostWaves && !two) return launch_units<DT, BLK, 1>(a, waves_for(1), stream);
    // (rotated pieces are twice as long: two a wave are enough for every row)
    if constexpr (BLK <= 0)
        if (waves_for(2) > kMostWaves) return launch_units<DT, BLK, 4>(a, waves_for(4), stream);
    return launch_units<DT, BLK, 2>(a, waves_for(2), stream);
}

template <int DT>
int launch_type(const NormArgs& a, hipStream_t stream) {
    switch (a.hblock) {
        case -1: return launch_block<DT, -1>(a, stream);
        case 0: return launch_block<DT, 0>(a, stream);
        case 16: return launch_block<DT, 16>(a, stream);
        case 64: return launch_block<DT, 64>(a, stream);
        default: return launch_block<DT, 256>(a, stream);
    }
}

}  // namespace

int launch_norm(const NormArgs& a, hipStream_t stream) {
    if (a.dtype == kDtF32) return launch_type<kDtF32>(a, stream);
    return a.dtype == kDtF16 ? launch_type<kDtF16>(a, stream) : launch_type<kDtBf16>(a, stream);
}

}  // namespace mq
