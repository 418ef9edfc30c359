// New tokens into a paged cache with their positions turned into them on the way: queries to an output, keys and values
// to their sequences' pages (16 bits, or int8 with a scale per token and head).
//
// Pair i of a head, at position p, is turned by the angle p f_i: (a c - b s, a s + b c) with c and s its cosine and sine
// times `size`. Pairs are (i, i + n) for the first 2 n values of a head, or neighbours (2 i, 2 i + 1); values behind
// them stay as they are.
//
// Angles: f_i is given as a 64-bit fraction of a turn, so p f_i modulo a turn is the integer product p f_i modulo 2^64,
// exact for every position (in fp32 a position of 60000 would already be off by 4e-3); its cosine and sine are
// taken in fp64 and rounded to fp32 once. A workgroup takes a token, of few tokens a part of one's heads: it computes the angles, a
// thread a pair, and they serve all its heads from LDS.
//
// Memory-bound: each value is read once and written once. 17.5 k tokens of 48 heads of 128 in bf16, 429 MB: 85 us, 5.0 TB/s (a copy
// 5.1; under the profiler 89). 8.5 k tokens of 24 heads of 128 into int8, 96 MB: 28 us, 3.4 TB/s beside the angles in fp64 and eight
// divisions a lane (a row's values loaded in front of the angles, the next row's in front of a row's work: 32 us; into 16 bits, both
// under the profiler, 93 instead of 89). 64 single tokens: 3.7 us, chains of dependent loads (length, table, row) and the angles.
//
// A row is 8 values a lane on the 2^k lanes that hold it; a lane of a turned row of halves holds four values of each half, so
// that it has both of a pair.
#include "mq_device.h"
#include "mq_internal.h"

namespace mq {
namespace {

constexpr int kMostPairs = 128;

__device__ __forceinline__ float elem(uint32_t w, int hi, bool f16) {
    return f16 ? f16_bits_to_f32(static_cast<uint16_t>(hi ? w >> 16 : w & 0xffffu)) : hi ? bf16hi(w) : bf16lo(w);
}

template <int DT, bool I8>
__global__ void __launch_bounds__(256) kv_append_kernel(KvAppendArgs a) {
    constexpr bool kF16 = DT == kDtF16;
    __shared__ float2 turn[kMostPairs];
    const KvWriteArgs& w = a.w;
    const int lanes = 1 << w.row_shift;                     // lanes per row
    const int64_t t = a.first + blockIdx.x;
    int64_t b = t, pos;
    if (w.cu_q) {
        // the sequence of token t: cu_q[b] <= t < cu_q[b + 1]
        int64_t lo = 0, hi = w.B;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (w.cu_q[mid] <= t) lo = mid; else hi = mid;
        }
        b = lo;
        if (t < w.cu_q[b] || t >= w.cu_q[b + 1]) return;    // behind the last sequence's tokens
        pos = static_cast<int64_t>(w.lens[b]) - w.cu_q[b + 1] + t;
    } else {
        pos = static_cast<int64_t>(w.lens[b]) - 1;
    }
    const bool turned = pos >= 0;                           // a token without a position stays as it is
    const int pairs = a.turn / 2;
    for (int i = threadIdx.x; i < pairs; i += 256) {
        float2 cs = make_float2(1.0f, 0.0f);
        if (turned) {
            const uint64_t part = static_cast<uint64_t>(pos) * a.freq[i];
            double s, c;
            sincospi(static_cast<double>(static_cast<int64_t>(part)) * 0x1p-63, &s, &c);
            cs = make_float2(static_cast<float>(c * a.size), static_cast<float>(s * a.size));
        }
        turn[i] = cs;
    }
    // where its keys and values go
    const int64_t at = pos >> w.page_shift;
    int page = -1;
    if (turned && at < w.width) page = w.table[b * w.ld_table + at];
    const bool held = page >= 0 && page < w.pages;
    const int64_t slot = pos & ((int64_t(1) << w.page_shift) - 1);
    __syncthreads();

    const int64_t rows = a.Hq + 2 * w.H;
    const int c = static_cast<int>(threadIdx.x) & (lanes - 1);
    const int64_t step = static_cast<int64_t>(gridDim.y) * (256 >> w.row_shift);
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * (256 >> w.row_shift) + (threadIdx.x >> w.row_shift); r < rows; r += step) {
        const int kind = r < a.Hq ? 0 : r < a.Hq + w.H ? 1 : 2;         // query, key, value
        const int64_t h = kind == 0 ? r : kind == 1 ? r - a.Hq : r - a.Hq - w.H;
        if (kind > 0 && !held) continue;                                // no place for it: nothing is written
        const bool ok = 8 * c < w.D;
        const uint16_t* src = static_cast<const uint16_t*>(kind == 0 ? a.q : kind == 1 ? w.k : w.v) +
                              t * (kind == 0 ? a.q_token : kind == 1 ? w.k_token : w.v_token) +
                              h * (kind == 0 ? a.q_head : kind == 1 ? w.k_head : w.v_head);
        const bool mine = kind < 2 && 8 * c < a.turn;                   // values that are turned
        const bool halves = mine && !a.interleaved;
        const int d0 = halves ? 4 * c : 8 * c, d1 = halves ? pairs + 4 * c : 8 * c + 4;
        uint2 x0 = make_uint2(0, 0), x1 = make_uint2(0, 0);
        if (ok) {
            x0 = *reinterpret_cast<const uint2*>(src + d0);
            x1 = *reinterpret_cast<const uint2*>(src + d1);
        }
        float f[8] = {elem(x0.x, 0, kF16), elem(x0.x, 1, kF16), elem(x0.y, 0, kF16), elem(x0.y, 1, kF16),
                      elem(x1.x, 0, kF16), elem(x1.x, 1, kF16), elem(x1.y, 0, kF16), elem(x1.y, 1, kF16)};
        if (mine && turned) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 cs = turn[4 * c + i];
                const float u = halves ? f[i] : f[2 * i], v = halves ? f[i + 4] : f[2 * i + 1];
                const float y0 = u * cs.x - v * cs.y, y1 = u * cs.y + v * cs.x;
                if (halves) { f[i] = y0; f[i + 4] = y1; }
                else { f[2 * i] = y0; f[2 * i + 1] = y1; }
            }
            x0 = make_uint2(pack_16x2(f[0], f[1], DT), pack_16x2(f[2], f[3], DT));
            x1 = make_uint2(pack_16x2(f[4], f[5], DT), pack_16x2(f[6], f[7], DT));
        }
        if (kind == 0) {
            uint16_t* to = static_cast<uint16_t*>(a.o) + t * a.o_token + h * a.o_head;
            if (ok) {
                *reinterpret_cast<uint2*>(to + d0) = x0;
                *reinterpret_cast<uint2*>(to + d1) = x1;
            }
            continue;
        }
        const int64_t off = page * w.c_page + h * w.c_head + slot * w.c_token;
        if constexpr (!I8) {
            if (ok) {
                uint16_t* to = static_cast<uint16_t*>(kind == 2 ? w.vc : w.kc) + off;
                *reinterpret_cast<uint2*>(to + d0) = x0;
                *reinterpret_cast<uint2*>(to + d1) = x1;
            }
        } else {
            // the bits of |x| order as unsigned integers, NaN and infinity above every finite value
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = __builtin_elementwise_max(m, __float_as_uint(f[j]) & 0x7fffffffu);
            for (int s = 1; s < lanes; s <<= 1) m = __builtin_elementwise_max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), s)));
            const bool finite = m < 0x7f800000u;
            const float s = finite ? __builtin_fmaxf(__uint_as_float(m) / 127.0f, 1e-10f) : __uint_as_float(0x7fc00000u);
            uint32_t q[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float n = finite ? __builtin_rintf(f[j] / s) : 0.0f;
                q[j >> 2] |= (static_cast<uint32_t>(static_cast<int>(n)) & 0xffu) << (8 * (j & 3));
            }
            if (ok) {
                int8_t* to = static_cast<int8_t*>(kind == 2 ? w.vc : w.kc) + off;
                *reinterpret_cast<uint32_t*>(to + d0) = q[0];
                *reinterpret_cast<uint32_t*>(to + d1) = q[1];
            }
            if (c == 0) (kind == 2 ? w.v_scale : w.k_scale)[page * w.s_page + h * w.s_head + slot * w.s_token] = s;
        }
    }
}

template <int DT>
int launch_type(const KvAppendArgs& a, bool i8, hipStream_t stream) {
    // workgroups: one a token, and for few tokens as many as have rows for all their lanes
    const int64_t rows = a.Hq + 2 * a.w.H, per = 256 >> a.w.row_shift;
    const int64_t steps = (rows + per - 1) / per, want = (1024 + a.w.T - 1) / a.w.T, most = kMostThreads / 256;
    for (int64_t t = 0; t < a.w.T; t += most) {
        KvAppendArgs b = a;
        b.first = t;
        const dim3 grid(static_cast<unsigned>(a.w.T - t < most ? a.w.T - t : most), static_cast<unsigned>(steps < want ? steps : want));
        if (i8) hipLaunchKernelGGL((kv_append_kernel<DT, true>), grid, dim3(256), 0, stream, b);
        else hipLaunchKernelGGL((kv_append_kernel<DT, false>), grid, dim3(256), 0, stream, b);
    }
    return launch_status("kv_append");
}

}  // namespace

int launch_kv_append(const KvAppendArgs& a, int dtype, bool i8, hipStream_t stream) {
    KvAppendArgs b = a;
    b.w.row_shift = 0;
    while ((8 << b.w.row_shift) < b.w.D) ++b.w.row_shift;
    return dtype == kDtF16 ? launch_type<kDtF16>(b, i8, stream) : launch_type<kDtBf16>(b, i8, stream);
}

}  // namespace mq
