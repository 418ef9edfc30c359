// Attention of one new token per sequence over a paged key-value cache.
//
// HBM-bound: every visible key and value is read once for the query heads that share them (up to 16 on one
// MFMA tile) and used for 2 products each; the MFMAs are a few percent of that time. So the kernel is
// built around loads: straight from the pages into registers, whole rows, with the next tile's loads issued before
// this one is worked on, and nothing goes through LDS until the end.
//
//   S^T = K Q^T       A: 16 keys x 32 values, lane (c, g) = (l & 15, l >> 4) holds key c, values 8 g .. 8 g + 7 of
//                     each 32; B: the query heads' rows. Lane (c, g) gets query row c, keys 4 g + r (r < 4).
//   softmax           in base 2 over the running maximum of query row c: 8 scores a lane, joined over the four
//                     lanes that hold the row.
//   O^T = V^T P^T     a lane's 8 probabilities, rounded to 16 bits, are the B operand (the keys of a product may come in any
//                     order, so slot (g, j) is key 16 (j / 4) + 4 g + j % 4); for A a lane loads the same 8 keys'
//                     values VE c .. VE c + VE - 1 (VE = width / 16, so 16 lanes read a whole row) and pairs the
//                     keys' 16-bit values with v_perm. Product i gives values VE m + i of row m. The rounding is
//                     relative 2^-9 (bf16) or 2^-12 each, of random signs, in sums of thousands: 131071 bf16
//                     tokens come out 2.2e-3 from the exact result, 1.7e-3 if only the output were rounded; the sum
//                     that divides is of the unrounded ones. fp16 rows over an int8 cache, whose products are bf16,
//                     take what is rounded off in a second product.
//
// A workgroup's eight waves (four for heads of more than 128 values, whose operands take twice the registers) take
// 32 keys each of a tile, one workgroup a compute unit. The tiles of all sequences and cache heads are
// one line, cut into equal pieces for the resident workgroups (lengths are known on the device only, and a
// ragged batch is balanced this way). A piece may end inside a sequence: its maxima, sums and unnormalised outputs
// (fp32) then go to the workspace, and the workgroup that brings a sequence's last piece (a count per sequence
// and cache head tells, which it sets back to zero) joins them in the order of the pieces, so the result is the
// same every time.
//
// Measured: 131071 tokens of 8 heads of 128, bf16: 87 us, 6.2 TB/s (a fill of memory reaches 6.7, a copy 5.1); 64 ragged
// int8 sequences of up to 8000: 55 us, 3.4 TB/s, bound by unpacking and by the sequences' ends; one sequence of
// 260 visible tokens: 10 us, a chain of dependent loads (length, table, rows) and the launch.
#include "mq_attn.h"

namespace mq {
namespace {

constexpr int kKeys = 32;      // keys per wave and step
constexpr int waves_of(int dp) { return dp == 256 ? 4 : 8; }

// What the query at position pos sees, as tiles of TILE keys: tiles 0 .. ns - 1 (first tokens), then w0 ... (Positions
// and counts of tiles fit 32 bits: the host refuses tables that could hold more.)
struct Visible {
    int pos, last, lo, sinks;   // last key that is held; first key of the window; first tokens that stay visible
    int ns, nt, w0;
};

template <int TILE>
__device__ __forceinline__ Visible visible(const AttnArgs& a, int len) {
    Visible v;
    const int cap = static_cast<int>(a.width) << a.page_shift;
    v.pos = len - 1;
    v.last = v.pos < cap ? v.pos : cap - 1;
    const int window = static_cast<int>(a.window), sinks = static_cast<int>(a.sinks);
    v.lo = window > 0 && window <= v.pos ? v.pos - window + 1 : 0;
    v.sinks = sinks < v.lo ? sinks : v.lo;
    v.ns = 0;
    v.nt = 0;
    v.w0 = v.lo / TILE;
    if (v.last < 0) return v;
    const int first = v.sinks < v.last + 1 ? v.sinks : v.last + 1;
    int nw = 0;
    v.ns = (first + TILE - 1) / TILE;
    if (v.last >= v.lo) {
        nw = v.last / TILE - v.w0 + 1;
        v.ns = v.ns < v.w0 ? v.ns : v.w0;       // the window's first tile may hold first tokens too
    }
    v.nt = v.ns + nw;
    return v;
}

// A word that the kernel does not write, at an address that all lanes share: through the scalar unit.
__device__ __forceinline__ int scalar_word(const int* p) {
    return *reinterpret_cast<const __attribute__((address_space(4))) int*>(reinterpret_cast<uintptr_t>(p));
}

// The line of tiles: sequence b takes up `extra` places and its nt(b) tiles for each of `per` (cache head, row tile)
// pairs; the places stand for what a workgroup pays to begin and end a sequence, so that those with many short ones
// get fewer tiles. total: places; and the sequence that holds place t of it, with the places before it. Every wave
// of a workgroup computes them for itself, 64 sequences at a time.
template <int TILE>
__device__ __forceinline__ int places(const AttnArgs& a, int len, int extra) {
    const int nt = visible<TILE>(a, len).nt;
    return nt ? nt + extra : 0;
}

template <int TILE>
__device__ __forceinline__ int line_total(const AttnArgs& a, int per, int extra) {
    if (a.B == 1) return places<TILE>(a, scalar_word(a.lens), extra) * per;
    int n = 0;
    for (int b = threadIdx.x & 63; b < a.B; b += 64) n += places<TILE>(a, a.lens[b], extra);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) n += __shfl_xor(n, s);
    return __builtin_amdgcn_readfirstlane(n) * per;
}

template <int TILE>
__device__ __forceinline__ void find_seq(const AttnArgs& a, int per, int extra, int t, int* seq, int* before) {
    const int lane = threadIdx.x & 63;
    int base = 0;
    *seq = 0;
    *before = 0;
    if (a.B == 1) return;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int n = b0 + lane < a.B ? places<TILE>(a, a.lens[b0 + lane], extra) * per : 0;
        int x = n;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int y = __shfl_up(x, s);
            if (lane >= s) x += y;
        }
        const uint64_t past = __ballot(base + x > t);
        if (past) {
            const int first = __builtin_ctzll(past);
            *seq = b0 + first;
            *before = base + __builtin_amdgcn_readlane(x - n, first);
            return;
        }
        base += __builtin_amdgcn_readlane(x, 63);
    }
}

// A split sequence's pieces: [slot][row][D] outputs, then [slot][row][2] maxima and sums. The segment of a sequence
// that began before workgroup w's piece has slot 2 w, one that goes on behind it 2 w + 1.
__device__ __forceinline__ float* part_out(const AttnArgs& a, int rows, int64_t slot) {
    return static_cast<float*>(a.work) + slot * rows * a.D;
}
__device__ __forceinline__ float* part_stat(const AttnArgs& a, int rows, int64_t slots, int64_t slot) {
    return static_cast<float*>(a.work) + slots * rows * a.D + slot * rows * 2;
}

// Pieces go from one workgroup to another, maybe on another die: stores and loads that are coherent on the
// whole device (relaxed atomics of 8 bytes), so that no second level cache has to be written back for them.
__device__ __forceinline__ void send(float* p, float x, float y) {
    const uint64_t v = static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 receive(const float* p) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Keys and values are read once: past the caches' replacement (non-temporal), 10 % faster on a cache that does not
// fit them.
template <int BYTES>
struct Raw;   // BYTES bytes of a row
template <> struct Raw<4> { uint32_t w[1]; };
template <> struct Raw<8> { uint32_t w[2]; };
template <> struct Raw<16> { uint32_t w[4]; };
template <> struct Raw<32> { uint32_t w[8]; };   // 16-bit heads of more than 128 values

template <int BYTES>
__device__ __forceinline__ Raw<BYTES> load_raw(const char* p) {
    Raw<BYTES> r;
    if constexpr (BYTES == 4) {
        r.w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
    } else if constexpr (BYTES == 8) {
        const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(p));
        r.w[0] = x[0]; r.w[1] = x[1];
    } else {
        static_assert(BYTES == 16);
        const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = x[i];
    }
    return r;
}

// BYTES of a value row from value d on (at `off`), its head D wide: a piece of 16 bytes that begins behind the
// width reads the one before it instead (its products are never stored).
template <int BYTES, int E>
__device__ __forceinline__ Raw<BYTES> load_row(const char* row, uint32_t off, int d, int D) {
    if constexpr (BYTES == 32) {
        Raw<32> r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const u32x4 x = __builtin_nontemporal_load(
                reinterpret_cast<const u32x4*>(row + (off + (d + i * 16 / E < D ? 16 * i : 0))));
#pragma unroll
            for (int e = 0; e < 4; ++e) r.w[4 * i + e] = x[e];
        }
        return r;
    } else {
        return load_raw<BYTES>(row + off);
    }
}

// A split sequence's pieces p0 .. p1 together, for the query rows of one tile: groups of threads take every
// parts-th piece with a running maximum, four pieces' loads at a time, and are then added in LDS (buf).
template <int DP, int DT>
__device__ __forceinline__ void join_pieces(const AttnArgs& a, int rows, int rows_most, int slots, int s0, int piece, int p0,
                                            int p1, int b, int hq0, float* buf) {
    constexpr int kQuads = DP / 4;                      // float4 of a row
    constexpr int kThreads = 64 * waves_of(DP);
    const int items = rows * kQuads, parts = items >= kThreads ? 1 : kThreads / items;
    constexpr int kAhead = 4;
    for (int base = 0; base < items; base += kThreads) {
        const int part = parts == 1 ? 0 : static_cast<int>(threadIdx.x) / items;
        const int item = parts == 1 ? base + static_cast<int>(threadIdx.x) : static_cast<int>(threadIdx.x) % items;
        const int row = item / kQuads, d = 4 * (item % kQuads);
        const bool mine = item < items && part < parts && d < a.D;
        float m = kNegInf, l = 0.0f, x[4] = {0, 0, 0, 0};
        bool some = false;
        if (mine) {
            for (int p = p0 + part; p <= p1; p += kAhead * parts) {
                float pm[kAhead], pl[kAhead];
                float4 px[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int w = p + i * parts < p1 ? p + i * parts : p1;
                    const int slot = 2 * w + (w * piece < s0);
                    const float2 st = receive(part_stat(a, rows_most, slots, slot) + 2 * row);
                    const float* x = part_out(a, rows_most, slot) + row * a.D + d;
                    const float2 x0 = receive(x), x1 = receive(x + 2);
                    pm[i] = st.x;
                    pl[i] = p + i * parts <= p1 ? st.y : -1.0f;
                    px[i] = make_float4(x0.x, x0.y, x1.x, x1.y);
                }
                float top = m;
#pragma unroll
                for (int i = 0; i < kAhead; ++i) top = pl[i] < 0.0f ? top : __builtin_fmaxf(top, pm[i]);
                const float ref = top == kNegInf ? 0.0f : top;
                const float f = __builtin_amdgcn_exp2f(m - ref);
                m = top;
                l *= f;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] *= f;
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (pl[i] < 0.0f) continue;         // nothing seen there
                    some = true;
                    const float fi = __builtin_amdgcn_exp2f(pm[i] - ref);
                    l = __builtin_fmaf(fi, pl[i], l);
                    x[0] = __builtin_fmaf(fi, px[i].x, x[0]);
                    x[1] = __builtin_fmaf(fi, px[i].y, x[1]);
                    x[2] = __builtin_fmaf(fi, px[i].z, x[2]);
                    x[3] = __builtin_fmaf(fi, px[i].w, x[3]);
                }
            }
        }
        if (parts > 1) {
            __syncthreads();
            float* at = buf + 8 * threadIdx.x;
            at[0] = m; at[1] = some ? l : -1.0f; at[2] = x[0]; at[3] = x[1]; at[4] = x[2]; at[5] = x[3];
            __syncthreads();
            if (part == 0 && mine) {
                for (int o = 1; o < parts; ++o) {
                    const float* y = buf + 8 * (o * items + item);
                    if (y[1] < 0.0f) continue;
                    some = true;
                    const float top = __builtin_fmaxf(m, y[0]), ref = top == kNegInf ? 0.0f : top;
                    const float f = __builtin_amdgcn_exp2f(m - ref), fo = __builtin_amdgcn_exp2f(y[0] - ref);
                    m = top;
                    l = l * f + y[1] * fo;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = x[e] * f + y[2 + e] * fo;
                }
            }
        }
        if (mine && part == 0) {
            const float inv = some ? 1.0f / l : 0.0f;
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.o) + b * a.o_token + (hq0 + row) * a.o_head + d) =
                make_uint2(pack_16x2(x[0] * inv, x[1] * inv, DT), pack_16x2(x[2] * inv, x[3] * inv, DT));
        }
    }
    __syncthreads();
}

// DP: head width rounded up to 64, 128 or 256; DT: type of the tokens; I8: int8 cache; SMALL: pages of less than
// 16 tokens (a 16-key group may span pages, and every lane looks up its own keys).
template <int DP, int DT, bool I8, bool SMALL>
__global__ void __launch_bounds__(64 * waves_of(DP), waves_of(DP) / 4) attn_decode_kernel(AttnArgs a, int row_tiles, bool quads) {
    constexpr int kWaves = waves_of(DP), kTile = kWaves * kKeys;
    constexpr int E = I8 ? 1 : 2;                       // bytes per cached value
    constexpr int VE = DP / 16;                         // values a lane holds of a value row
    constexpr int kSteps = DP / 32;                     // products over the width
    constexpr int KB = 16;                              // bytes of a key load: 16 values (int8) or 8
    constexpr int KL = DP * E / 4 / KB;                 // key loads per row and lane
    constexpr bool kSplit = I8 && DT == kDtF16;         // fp16 rows against int8 keys: bf16 products of hi + lo
    constexpr int MT = I8 ? kDtBf16 : DT;               // type of the products
    // beginning and ending a sequence takes about as long as 128 KB of keys and values: counted where there are more
    // of them than workgroups (64 ragged int8 sequences of 8 heads: 66 -> 58 us); else every piece is a part of one
    // anyway (16 sequences of 2000: 30 us, 33 if counted)
    constexpr int kExtra = (131072 + kTile * DP * E) / (2 * kTile * DP * E);
    // the next segment's first tile is loaded ahead of this one's end where the registers for it are free
    constexpr bool kAcross = DP != 256 && !kSplit;
    // fp16 probabilities are held 2^14 times as large: they stay normal down to 2^-28 of the largest
    constexpr float kLift = MT == kDtF16 ? 14.0f : 0.0f;
    __shared__ float sm_out[kWaves][16][DP + 4];
    __shared__ float sm_m[kWaves][16], sm_l[kWaves][16];
    __shared__ int sm_any[kWaves];
    __shared__ int sm_last;

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int group = a.Hq / a.H;
    const int rows_most = group < 16 ? group : 16;
    const int per = a.H * row_tiles, extra = a.B * per > gridDim.x ? kExtra : 0;
    // sequences that see nothing have no tiles: zeros
    for (int e = blockIdx.x; e < a.B; e += gridDim.x) {
        if (visible<kTile>(a, scalar_word(a.lens + e)).nt != 0) continue;
        for (int x = threadIdx.x; x < a.Hq * (a.D / 8); x += 64 * kWaves) {
            const int row = x / (a.D / 8), d = 8 * (x % (a.D / 8));
            *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.o) + e * a.o_token + row * a.o_head + d) = make_uint4(0, 0, 0, 0);
        }
    }
    const int total = line_total<kTile>(a, per, extra);
    const int piece = (total + gridDim.x - 1) / gridDim.x;
    const int t0 = blockIdx.x * piece;
    const int t1 = t0 + piece < total ? t0 + piece : total;
    if (t0 >= t1) return;
    int b, before;
    find_seq<kTile>(a, per, extra, t0, &b, &before);
    const int mask = (1 << a.page_shift) - 1;
    const int last_page = static_cast<int>(a.pages) - 1;

    // the lane's places within 16 keys (bytes): key c, chunks 4 x + g; keys 4 g + r, values VE c ..
    const uint32_t tok = static_cast<uint32_t>(a.c_token) * E;
    uint32_t ko[KL], vo[4];
#pragma unroll
    for (int x = 0; x < KL; ++x) ko[x] = (SMALL ? 0 : c * tok) + (KB / E * (4 * x + g) < a.D ? KB * (4 * x + g) : 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) vo[r] = (SMALL ? 0 : (4 * g + r) * tok) + (VE * c < a.D ? VE * E * c : 0);

    // the segment in hand: tiles i0 .. i1 - 1 of a sequence's cache head and row tile, whose tile 0 is place s0
    Visible v;
    int pair, s0, i0, i1;
    const int* table;
    const char *kbase, *vbase;
    const float *ksb = nullptr, *vsb = nullptr;
    // the next one at or behind place t; false: none in this workgroup's piece
    auto open = [&](int t) __attribute__((always_inline)) {
        while (t < t1) {
            v = visible<kTile>(a, scalar_word(a.lens + b));
            const int size = v.nt + extra;
            if (v.nt == 0 || t - before >= size * per) {
                before += v.nt ? size * per : 0;
                ++b;
                continue;
            }
            pair = (t - before) / size;
            s0 = before + pair * size + extra;
            i0 = t > s0 ? t - s0 : 0;
            i1 = t1 - s0 < v.nt ? t1 - s0 : v.nt;
            if (i0 < i1) break;
            t = s0 + v.nt;                              // its extra places only
        }
        if (t >= t1) return false;
        const int h = pair / row_tiles;
        table = a.table + static_cast<int64_t>(b) * a.ld_table;
        kbase = static_cast<const char*>(a.kc) + static_cast<int64_t>(h) * a.c_head * E;
        vbase = static_cast<const char*>(a.vc) + static_cast<int64_t>(h) * a.c_head * E;
        if constexpr (I8) {
            ksb = a.k_scale + h * a.s_head;
            vsb = a.v_scale + h * a.s_head;
        }
        return true;
    };

    // the query rows: B operand, lane (c, g) = row c, the values that the key loads' slots stand for
    Frag q[kSteps], q2[kSplit ? kSteps : 1];
    auto load_q = [&]() __attribute__((always_inline)) {
        const int rt = pair % row_tiles, left = group - 16 * rt;
        const uint16_t* row = static_cast<const uint16_t*>(a.q) + b * a.q_token +
                              (pair / row_tiles * group + 16 * rt + (c < left ? c : 0)) * a.q_head;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int d = I8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
            const uint4 x = *reinterpret_cast<const uint4*>(row + (d < a.D ? d : 0));
            q[s] = Frag{{x.x, x.y, x.z, x.w}};
        }
    };
    Raw<KB> kr[2][2][KL];       // [buffer][16-key group][load]
    Raw<VE * E> vr[2][8];       // [buffer][key]
    float ksc[2][2][4], vsc[2][2][4];   // int8: scales of the lane's 8 keys
    uint32_t held[2];           // bit 16 u + x: key x of group u is in a page of the cache

    auto first_key = [&](int i) { return (i < v.ns ? i : v.w0 + (i - v.ns)) * kTile + wave * kKeys; };
    // the 32 keys from j on: every address is inside the cache (a key that is not held reads page 0)
    auto load = [&](int buf, int j) __attribute__((always_inline)) {
        held[buf] = 0;
        const int ne = static_cast<int>(a.width) - 1;
        if constexpr (!SMALL) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int at = (j + 16 * u) >> a.page_shift;
                const int p = scalar_word(table + (at < ne ? at : ne));
                const bool ok = p >= 0 && p <= last_page && at <= ne;
                held[buf] |= ok ? 0xffffu << (16 * u) : 0u;
                const int pg = ok ? p : 0, slot = (j + 16 * u) & mask;
                const int64_t off = (pg * a.c_page + slot * a.c_token) * E;
                const char* kp = kbase + off;
                const char* vp = vbase + off;
#pragma unroll
                for (int x = 0; x < KL; ++x) kr[buf][u][x] = load_raw<KB>(kp + ko[x]);
#pragma unroll
                for (int r = 0; r < 4; ++r) vr[buf][4 * u + r] = load_row<VE * E, E>(vp, vo[r], VE * c, a.D);
                if constexpr (I8) {
                    const int64_t so = pg * a.s_page + slot * a.s_token;
                    if (quads) {                    // four keys' scales are one aligned 16 bytes
                        const float4 x = *reinterpret_cast<const float4*>(ksb + so + 4 * g);
                        const float4 y = *reinterpret_cast<const float4*>(vsb + so + 4 * g);
                        ksc[buf][u][0] = x.x; ksc[buf][u][1] = x.y; ksc[buf][u][2] = x.z; ksc[buf][u][3] = x.w;
                        vsc[buf][u][0] = y.x; vsc[buf][u][1] = y.y; vsc[buf][u][2] = y.z; vsc[buf][u][3] = y.w;
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            ksc[buf][u][r] = ksb[so + (4 * g + r) * a.s_token];
                            vsc[buf][u][r] = vsb[so + (4 * g + r) * a.s_token];
                        }
                    }
                }
            }
        } else {
            // lane x (and x + 32) looks up key x of the 32: its row as page << page_shift | slot, or -1
            const int mine = j + (lane & 31), at = mine >> a.page_shift;
            const int p = table[at < ne ? at : ne];
            const bool ok = p >= 0 && p <= last_page && at <= ne;
            held[buf] = static_cast<uint32_t>(__ballot(ok));
            const int code = ok ? (p << a.page_shift) | (mine & mask) : 0;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int ck = __shfl(code, 16 * u + c);
                const char* kp = kbase + (static_cast<int64_t>(ck >> a.page_shift) * a.c_page + (ck & mask) * a.c_token) * E;
#pragma unroll
                for (int x = 0; x < KL; ++x) kr[buf][u][x] = load_raw<KB>(kp + ko[x]);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int cv = __shfl(code, 16 * u + 4 * g + r);
                    const int64_t pg = cv >> a.page_shift, slot = cv & mask;
                    vr[buf][4 * u + r] = load_row<VE * E, E>(vbase + (pg * a.c_page + slot * a.c_token) * E, vo[r], VE * c, a.D);
                    if constexpr (I8) {
                        ksc[buf][u][r] = ksb[pg * a.s_page + slot * a.s_token];
                        vsc[buf][u][r] = vsb[pg * a.s_page + slot * a.s_token];
                    }
                }
            }
        }
    };
    if (!open(t0)) return;
    load_q();
    load(0, first_key(i0));
    for (bool more = true; more;) {
        const int rt = pair % row_tiles, hq0 = pair / row_tiles * group + 16 * rt;
        const int rows = group - 16 * rt < 16 ? group - 16 * rt : 16;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int d = I8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
            if (c >= rows || d >= a.D) q[s] = Frag{{0, 0, 0, 0}};
            if constexpr (kSplit) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t hi, lo;
                    split_f16(q[s].w[j], &hi, &lo);
                    q[s].w[j] = hi;
                    q2[s].w[j] = lo;
                }
            }
        }
        f32x4 o[VE];
#pragma unroll
        for (int i = 0; i < VE; ++i) o[i] = f32x4{0, 0, 0, 0};
        float m = kNegInf, l = 0.0f;
        bool any = false;           // a key that the query sees (the same for all rows: it is one query's position)
        const float scale = a.scale * kLog2e;
        auto work = [&](int buf, int j) __attribute__((always_inline)) {
            // scores
            f32x4 s[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int st = 0; st < kSteps; ++st) {
                    Frag k;
                    if constexpr (I8) {
                        float f[8];
                        float f0[4], f1[4];
                        i8x4(kr[buf][u][st >> 1].w[2 * (st & 1)], f0);
                        i8x4(kr[buf][u][st >> 1].w[2 * (st & 1) + 1], f1);
#pragma unroll
                        for (int e = 0; e < 4; ++e) { f[e] = f0[e]; f[4 + e] = f1[e]; }
#pragma unroll
                        for (int e = 0; e < 4; ++e) k.w[e] = bf16_exact2(f[2 * e], f[2 * e + 1]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) k.w[e] = kr[buf][u][st].w[e];
                    }
                    // values past the width: the query's zeros would not stop an infinity there
                    const int d = I8 ? 64 * (st >> 1) + 16 * g + 8 * (st & 1) : 32 * st + 8 * g;
                    if (d >= a.D) k = Frag{{0, 0, 0, 0}};
                    s[u] = mfma16<MT>(k, q[st], s[u]);
                    if constexpr (kSplit) s[u] = mfma16<MT>(k, q2[st], s[u]);
                }
            }
            float p[8];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) p[4 * u + r] = s[u][r] * scale * (I8 ? ksc[buf][u][r] : 1.0f);
            // keys that the query sees; all of them in most tiles
            const bool whole = held[buf] == 0xffffffffu && j + kKeys - 1 <= v.last && (j >= v.lo || j + kKeys <= v.sinks);
            uint32_t see = 0xffu;
            any = any || whole;
            if (!whole) {
                see = 0;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const int at = 16 * (x >> 2) + 4 * g + (x & 3);
                    const int key = j + at;
                    const bool ok = ((held[buf] >> at) & 1) && key <= v.last && (key >= v.lo || key < v.sinks);
                    see |= ok ? 1u << x : 0u;
                    p[x] = ok ? p[x] : kNegInf;
                }
                any = any || __ballot(see != 0) != 0;
            }
            float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(p[0], p[1]), __builtin_fmaxf(p[2], p[3])),
                                        __builtin_fmaxf(__builtin_fmaxf(p[4], p[5]), __builtin_fmaxf(p[6], p[7])));
            top = max4(top);
            const float mn = __builtin_fmaxf(m, top);
            const float base = mn == kNegInf ? 0.0f : mn;
            const float f = __builtin_amdgcn_exp2f(m - base);
            m = mn;
#pragma unroll
            for (int x = 0; x < 8; ++x) p[x] = __builtin_amdgcn_exp2f(p[x] - base + kLift);
            float sum = ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
            l = l * f + sum;            // the lane's own keys; the four lanes of a row are added at the end
            Frag pf, pf2;
            if constexpr (I8) {
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    // a key that is not seen has weight 0 whatever its scale holds
                    p[x] = (see >> x) & 1 ? p[x] * vsc[buf][x >> 2][x & 3] : 0.0f;
                }
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                pf.w[x] = pack_16x2(p[2 * x], p[2 * x + 1], MT);
                if constexpr (kSplit)
                    pf2.w[x] = pack_16x2(p[2 * x] - bf16lo(pf.w[x]), p[2 * x + 1] - bf16hi(pf.w[x]), MT);
            }
#pragma unroll
            for (int i = 0; i < VE; ++i) o[i] *= f;
            if (!I8 && !whole) {        // 0 times an infinity or NaN: values that are not seen become 0
#pragma unroll
                for (int x = 0; x < 8; ++x)
#pragma unroll
                    for (int e = 0; e < VE * E / 4; ++e) vr[buf][x].w[e] = (see >> x) & 1 ? vr[buf][x].w[e] : 0u;
            }
            if constexpr (I8) {
#pragma unroll
                for (int w = 0; w < VE / 4; ++w) {
                    float f8[8][4];
#pragma unroll
                    for (int x = 0; x < 8; ++x) i8x4(vr[buf][x].w[w], f8[x]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        Frag k;
#pragma unroll
                        for (int x = 0; x < 4; ++x) k.w[x] = bf16_exact2(f8[2 * x][i], f8[2 * x + 1][i]);
                        o[4 * w + i] = mfma16<MT>(k, pf, o[4 * w + i]);
                        if constexpr (kSplit) o[4 * w + i] = mfma16<MT>(k, pf2, o[4 * w + i]);
                    }
                }
            } else {
#pragma unroll
                for (int w = 0; w < VE / 2; ++w) {
                    Frag k0, k1;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        k0.w[x] = pair16<0>(vr[buf][2 * x].w[w], vr[buf][2 * x + 1].w[w]);
                        k1.w[x] = pair16<1>(vr[buf][2 * x].w[w], vr[buf][2 * x + 1].w[w]);
                    }
                    o[2 * w] = mfma16<MT>(k0, pf, o[2 * w]);
                    o[2 * w + 1] = mfma16<MT>(k1, pf, o[2 * w + 1]);
                }
            }
        };

        int i = i0;
        for (; i + 1 < i1; i += 2) {
            load(1, first_key(i + 1));
            work(0, first_key(i));
            if (i + 2 < i1) load(0, first_key(i + 2));
            work(1, first_key(i + 1));
        }
        if (i < i1) work(0, first_key(i));
        l = sum4(l);
        // the next segment's first tile and query rows are on their way while this one is written
        const int cur_b = b, cur_pair = pair, cur_s0 = s0, nt = v.nt;
        const bool whole = i0 == 0 && i1 == nt;
        more = open(s0 + i1);
        if (kAcross && more) {
            load_q();
            load(0, first_key(i0));
        }

        // the waves' parts together: rows c, values VE (4 g + r) + i
        __syncthreads();
        if (lane == 0) sm_any[wave] = any;
        if (c < rows) {
            if (g == 0) {
                sm_m[wave][c] = m;
                sm_l[wave][c] = l;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < VE; ++e) sm_out[wave][c][VE * (4 * g + r) + e] = o[e][r];
        }
        __syncthreads();
        int some = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) some |= sm_any[w];
        const int slots = 2 * gridDim.x, slot = 2 * blockIdx.x + (t0 < cur_s0);
        for (int e = threadIdx.x; e < rows * DP / 4; e += 64 * kWaves) {
            const int row = e / (DP / 4), d = 4 * (e % (DP / 4));
            if (d >= a.D) continue;
            float top = kNegInf;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = __builtin_fmaxf(top, sm_m[w][row]);
            const float base = top == kNegInf ? 0.0f : top;
            float sum = 0.0f, x[4] = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(sm_m[w][row] - base);
                sum += f * sm_l[w][row];
                const float4 y = *reinterpret_cast<const float4*>(&sm_out[w][row][d]);
                x[0] = __builtin_fmaf(f, y.x, x[0]);
                x[1] = __builtin_fmaf(f, y.y, x[1]);
                x[2] = __builtin_fmaf(f, y.z, x[2]);
                x[3] = __builtin_fmaf(f, y.w, x[3]);
            }
            if (whole) {
                const float inv = some ? 1.0f / sum : 0.0f;     // nothing seen: zeros
                uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + cur_b * a.o_token +
                                                            (hq0 + row) * a.o_head + d);
                *reinterpret_cast<uint2*>(out) = make_uint2(pack_16x2(x[0] * inv, x[1] * inv, DT),
                                                            pack_16x2(x[2] * inv, x[3] * inv, DT));
            } else {
                float* to = part_out(a, rows_most, slot) + row * a.D + d;
                send(to, x[0], x[1]);
                send(to + 2, x[2], x[3]);
                if (d == 0) send(part_stat(a, rows_most, slots, slot) + 2 * row, top, some ? sum : -1.0f);   // -1: nothing seen
            }
        }
        if (!whole) {
            // the sequence's pieces: workgroups p0 .. p1 of the line
            const int p0 = cur_s0 / piece, p1 = (cur_s0 + nt - 1) / piece;
            // every thread's stores have arrived (they are written through to where the device is coherent) before
            // the workgroup is counted; the count's value says that the others' have too
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            if (threadIdx.x == 0) {
                int* count = a.counters + static_cast<int64_t>(cur_b) * per + cur_pair;
                const int old = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                // the last one: zero again for the next call
                if (old == p1 - p0) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                sm_last = old == p1 - p0;
            }
            __syncthreads();
            if (sm_last) {
                join_pieces<DP, DT>(a, rows, rows_most, slots, cur_s0, piece, p0, p1, cur_b, hq0, &sm_out[0][0][0]);
            }
        }
        if (!kAcross && more) {
            load_q();
            load(0, first_key(i0));
        }
    }
}

// Workgroups: as many as are resident at once, one a compute unit.
int decode_groups() {
    const int cus = device_cu_count();
    return cus > 0 ? cus : 256;
}

template <int DP, int DT, bool I8>
int launch_width(const AttnArgs& a, int row_tiles, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(decode_groups()));
    // int8 scales of 4 keys as 16 bytes: consecutive and aligned
    const bool quads = I8 && a.s_token == 1 && a.s_page % 4 == 0 && a.s_head % 4 == 0 &&
                       (reinterpret_cast<uintptr_t>(a.k_scale) | reinterpret_cast<uintptr_t>(a.v_scale)) % 16 == 0;
    if (a.page_shift >= 4)
        hipLaunchKernelGGL((attn_decode_kernel<DP, DT, I8, false>), grid, dim3(64 * waves_of(DP)), 0, stream, a, row_tiles, quads);
    else
        hipLaunchKernelGGL((attn_decode_kernel<DP, DT, I8, true>), grid, dim3(64 * waves_of(DP)), 0, stream, a, row_tiles, quads);
    return launch_status("paged_attention");
}

template <int DT, bool I8>
int launch_type(const AttnArgs& a, int row_tiles, hipStream_t stream) {
    if (a.D <= 64) return launch_width<64, DT, I8>(a, row_tiles, stream);
    if (a.D <= 128) return launch_width<128, DT, I8>(a, row_tiles, stream);
    return launch_width<256, DT, I8>(a, row_tiles, stream);
}

}  // namespace

int64_t attn_decode_workspace_bytes(int Hq, int H, int D) {
    const int group = Hq / H, rows = group < 16 ? group : 16;
    return 2 * static_cast<int64_t>(decode_groups()) * rows * (D + 2) * 4;
}

int launch_attn_decode(const AttnArgs& a, hipStream_t stream) {
    const int row_tiles = (a.Hq / a.H + 15) / 16;
    const bool i8 = a.k_scale != nullptr;
    if (a.dtype == kDtF16)
        return i8 ? launch_type<kDtF16, true>(a, row_tiles, stream) : launch_type<kDtF16, false>(a, row_tiles, stream);
    return i8 ? launch_type<kDtBf16, true>(a, row_tiles, stream) : launch_type<kDtBf16, false>(a, row_tiles, stream);
}

int64_t attn_decode_counters(int Hq, int H, int64_t B) { return B * H * ((Hq / H + 15) / 16); }

}  // namespace mq
