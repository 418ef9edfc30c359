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
//   O^T = V^T P^T     a lane's 8 probabilities are the B operand as they are (the keys of a product may come in any
//                     order, so slot (g, j) is key 16 (j / 4) + 4 g + j % 4); for A a lane loads the same 8 keys'
//                     values VE c .. VE c + VE - 1 (VE = width / 16, so 16 lanes read a whole row) and pairs the
//                     keys' 16-bit values with v_perm. Product i gives values VE m + i of row m.
//
// A workgroup's four waves take 32 keys each of a 128-key tile. The tiles of all sequences and cache heads are
// one line, cut into equal pieces for the resident workgroups (lengths are known on the device only, and a
// ragged batch is balanced this way); a piece may end inside a sequence, which is then joined from its pieces'
// maxima, sums and unnormalised outputs (fp32) by a second kernel in the order of the pieces, so the result is
// the same every time.
#include "mq_attn.h"

namespace mq {
namespace {

constexpr int kTile = 128;     // keys per workgroup step
constexpr int kKeys = 32;      // keys per wave and step
constexpr int kWaves = 4;

// What the query at position pos sees, as 128-key tiles: tiles 0 .. ns - 1 (first tokens), then w0 ...
struct Visible {
    int64_t pos, last, lo, sinks;   // last key that is held; first key of the window; first tokens that stay visible
    int ns, nt;
    int64_t w0;
};

__device__ __forceinline__ Visible visible(const AttnArgs& a, int len) {
    Visible v;
    const int64_t cap = a.width << a.page_shift;
    v.pos = static_cast<int64_t>(len) - 1;
    v.last = v.pos < cap ? v.pos : cap - 1;
    v.lo = a.window > 0 && a.window <= v.pos ? v.pos - a.window + 1 : 0;
    v.sinks = a.sinks < v.lo ? a.sinks : v.lo;
    v.ns = 0;
    v.nt = 0;
    v.w0 = v.lo / kTile;
    if (v.last < 0) return v;
    const int64_t first = v.sinks < v.last + 1 ? v.sinks : v.last + 1;
    int64_t ns = (first + kTile - 1) / kTile, nw = 0;
    if (v.last >= v.lo) {
        nw = v.last / kTile - v.w0 + 1;
        ns = ns < v.w0 ? ns : v.w0;      // the window's first tile may hold first tokens too
    }
    v.ns = static_cast<int>(ns);
    v.nt = static_cast<int>(ns + nw);
    return v;
}

// The line of tiles: sequence b has nt(b) tiles for each of `per` (cache head, row tile) pairs.
struct Line {
    int64_t total;     // tiles
    int64_t piece;     // per workgroup
};

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) v += __shfl_xor(v, s);
    return v;
}

// Sum of nt over sequences (every wave of the workgroup computes it for itself).
__device__ __forceinline__ int64_t count_tiles(const AttnArgs& a, int64_t b0, int64_t b1) {
    int64_t n = 0;
    for (int64_t b = b0 + (threadIdx.x & 63); b < b1; b += 64) n += visible(a, a.lens[b]).nt;
    return wave_sum(n);
}

// A value that all lanes hold, as the scalar unit sees it.
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

__device__ __forceinline__ Line line_of(const AttnArgs& a, int64_t per, int64_t groups) {
    Line l;
    l.total = uniform(count_tiles(a, 0, a.B)) * per;
    l.piece = (l.total + groups - 1) / groups;
    return l;
}

// The sequence that holds tile t of the line, and the line's tiles before it (t < total).
__device__ __forceinline__ void find_seq(const AttnArgs& a, int64_t per, int64_t t, int64_t* seq, int64_t* before) {
    const int lane = threadIdx.x & 63;
    int64_t base = 0;
    for (int64_t b0 = 0; b0 < a.B; b0 += 64) {
        int64_t n = b0 + lane < a.B ? visible(a, a.lens[b0 + lane]).nt * per : 0;
        int64_t x = n;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int64_t y = __shfl_up(x, s);
            if (lane >= s) x += y;
        }
        const uint64_t past = __ballot(base + x > t);
        if (past) {
            const int first = __builtin_ctzll(past);
            *seq = b0 + first;
            *before = base + __shfl(x - n, first);
            return;
        }
        base += __shfl(x, 63);
    }
    *seq = a.B;
    *before = base;
}

// A split sequence's pieces: [slot][row][D] outputs, then [slot][row][2] maxima and sums. A workgroup's first
// segment has slot 2 w, a last one that began inside its piece 2 w + 1.
__device__ __forceinline__ float* part_out(const AttnArgs& a, int rows, int64_t slot) {
    return static_cast<float*>(a.work) + slot * rows * a.D;
}
__device__ __forceinline__ float* part_stat(const AttnArgs& a, int rows, int64_t slots, int64_t slot) {
    return static_cast<float*>(a.work) + slots * rows * a.D + slot * rows * 2;
}

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
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (BYTES == 8) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        r.w[0] = x.x; r.w[1] = x.y;
    } else {
        static_assert(BYTES == 16);
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        r.w[0] = x.x; r.w[1] = x.y; r.w[2] = x.z; r.w[3] = x.w;
    }
    return r;
}

// BYTES of a value row from value d on, its head D wide: a piece of 16 bytes that begins behind the width reads
// the row's first one instead (its products are never stored).
template <int BYTES, int E>
__device__ __forceinline__ Raw<BYTES> load_row(const char* row, int d, int D) {
    if constexpr (BYTES == 32) {
        Raw<32> r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = d + i * 16 / E;
            const uint4 x = *reinterpret_cast<const uint4*>(row + (at < D ? at : 0) * E);
            r.w[4 * i] = x.x; r.w[4 * i + 1] = x.y; r.w[4 * i + 2] = x.z; r.w[4 * i + 3] = x.w;
        }
        return r;
    } else {
        return load_raw<BYTES>(row + (d < D ? d : 0) * E);
    }
}

// DP: head width rounded up to 64, 128 or 256; DT: type of the tokens; I8: int8 cache; SMALL: pages of less than
// 16 tokens (a 16-key group may span pages, and every lane looks up its own keys).
template <int DP, int DT, bool I8, bool SMALL>
__global__ void __launch_bounds__(64 * kWaves, DP == 256 ? 1 : 2) attn_decode_kernel(AttnArgs a, int row_tiles) {
    constexpr int E = I8 ? 1 : 2;                       // bytes per cached value
    constexpr int VE = DP / 16;                         // values a lane holds of a value row
    constexpr int kSteps = DP / 32;                     // products over the width
    constexpr int KB = 16;                              // bytes of a key load: 16 values (int8) or 8
    constexpr int KL = DP * E / 4 / KB;                 // key loads per row and lane
    constexpr bool kSplit = I8 && DT == kDtF16;         // fp16 rows against int8 keys: bf16 products of hi + lo
    constexpr int MT = I8 ? kDtBf16 : DT;               // type of the products
    // fp16 probabilities are held 2^14 times as large: they stay normal down to 2^-28 of the largest
    constexpr float kLift = MT == kDtF16 ? 14.0f : 0.0f;
    __shared__ float sm_out[kWaves][16][DP + 4];
    __shared__ float sm_m[kWaves][16], sm_l[kWaves][16];
    __shared__ int sm_any[kWaves];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int group = a.Hq / a.H;
    const int rows_most = group < 16 ? group : 16;
    const int64_t per = static_cast<int64_t>(a.H) * row_tiles;
    const Line line = line_of(a, per, gridDim.x);
    const int64_t t0 = blockIdx.x * line.piece;
    const int64_t t1 = t0 + line.piece < line.total ? t0 + line.piece : line.total;
    if (t0 >= t1) return;
    int64_t b, before;
    find_seq(a, per, t0, &b, &before);
    b = uniform(b);
    before = uniform(before);
    const int mask = (1 << a.page_shift) - 1;
    const int last_page = static_cast<int>(a.pages) - 1;

    for (int64_t t = t0; t < t1;) {
        Visible v = visible(a, a.lens[b]);
        while (v.nt == 0 || t - before >= v.nt * per) {   // on to the next sequence that has tiles
            before += v.nt * per;
            ++b;
            v = visible(a, a.lens[b]);
        }
        const int pair = static_cast<int>((t - before) / v.nt);
        const int i0 = static_cast<int>((t - before) - static_cast<int64_t>(pair) * v.nt);
        const int64_t left = t1 - t;
        const int i1 = i0 + (left < v.nt - i0 ? static_cast<int>(left) : v.nt - i0);   // this segment: tiles i0 .. i1 - 1
        const int h = pair / row_tiles, rt = pair % row_tiles;
        const int rows = group - 16 * rt < 16 ? group - 16 * rt : 16;
        const int hq0 = h * group + 16 * rt;
        const int* table = a.table + b * a.ld_table;

        // the query rows: B operand, lane (c, g) = row c, the values that the key loads' slots stand for
        Frag q[kSteps], q2[kSplit ? kSteps : 1];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int d = I8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (c < rows && d < a.D)
                x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + b * a.q_token +
                                                    (hq0 + c) * a.q_head + d);
            q[s] = Frag{{x.x, x.y, x.z, x.w}};
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
        const char* kbase = static_cast<const char*>(a.kc) + static_cast<int64_t>(h) * a.c_head * E;
        const char* vbase = static_cast<const char*>(a.vc) + static_cast<int64_t>(h) * a.c_head * E;

        Raw<KB> kr[2][2][KL];       // [buffer][16-key group][load]
        Raw<VE * E> vr[2][8];       // [buffer][key]
        float ksc[2][2][4], vsc[2][2][4];   // int8: scales of the lane's 8 keys
        uint32_t held[2];           // bit 16 u + x: key x of group u is in a page of the cache

        auto first_key = [&](int i) -> int64_t {
            const int64_t tile = i < v.ns ? i : v.w0 + (i - v.ns);
            return tile * kTile + wave * kKeys;
        };
        // the 32 keys from j on: every address is inside the cache (a key that is not held reads page 0)
        auto load = [&](int buf, int64_t j) __attribute__((always_inline)) {
            held[buf] = 0;
            const int64_t ne = a.width - 1;
            if constexpr (!SMALL) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int64_t at = (j + 16 * u) >> a.page_shift;
                    const int p = table[at < ne ? at : ne];
                    const bool ok = p >= 0 && p <= last_page && at <= ne;
                    held[buf] |= ok ? 0xffffu << (16 * u) : 0u;
                    const int pg = ok ? p : 0;
                    const int slot = static_cast<int>(j + 16 * u) & mask;
                    const int64_t off = (pg * a.c_page + slot * a.c_token) * E;
                    const int64_t tok = a.c_token * E;
#pragma unroll
                    for (int x = 0; x < KL; ++x) {
                        const int d = KB / E * (4 * x + g);
                        kr[buf][u][x] = load_raw<KB>(kbase + off + c * tok + (d < a.D ? d : 0) * E);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        vr[buf][4 * u + r] = load_row<VE * E, E>(vbase + off + (4 * g + r) * tok, VE * c, a.D);
                        if constexpr (I8) {
                            const int64_t so = pg * a.s_page + h * a.s_head + (slot + 4 * g + r) * a.s_token;
                            ksc[buf][u][r] = a.k_scale[so];
                            vsc[buf][u][r] = a.v_scale[so];
                        }
                    }
                }
            } else {
                // lane x (and x + 32) looks up key x of the 32: its row as page << page_shift | slot, or -1
                const int64_t mine = j + (lane & 31);
                const int64_t at = mine >> a.page_shift;
                const int p = table[at < ne ? at : ne];
                const bool ok = p >= 0 && p <= last_page && at <= ne;
                held[buf] = static_cast<uint32_t>(__ballot(ok));
                const int code = ok ? (p << a.page_shift) | (static_cast<int>(mine) & mask) : 0;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int ck = __shfl(code, 16 * u + c);
                    const char* kp = kbase + (static_cast<int64_t>(ck >> a.page_shift) * a.c_page + (ck & mask) * a.c_token) * E;
#pragma unroll
                    for (int x = 0; x < KL; ++x) {
                        const int d = KB / E * (4 * x + g);
                        kr[buf][u][x] = load_raw<KB>(kp + (d < a.D ? d : 0) * E);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int cv = __shfl(code, 16 * u + 4 * g + r);
                        const int64_t pg = cv >> a.page_shift, slot = cv & mask;
                        vr[buf][4 * u + r] = load_row<VE * E, E>(vbase + (pg * a.c_page + slot * a.c_token) * E, VE * c, a.D);
                        if constexpr (I8) {
                            const int64_t so = pg * a.s_page + h * a.s_head + slot * a.s_token;
                            ksc[buf][u][r] = a.k_scale[so];
                            vsc[buf][u][r] = a.v_scale[so];
                        }
                    }
                }
            }
        };
        auto work = [&](int buf, int64_t j) __attribute__((always_inline)) {
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
                    const int64_t key = j + at;
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

        load(0, first_key(i0));
        int i = i0;
        for (; i + 1 < i1; i += 2) {
            load(1, first_key(i + 1));
            work(0, first_key(i));
            if (i + 2 < i1) load(0, first_key(i + 2));
            work(1, first_key(i + 1));
        }
        if (i < i1) work(0, first_key(i));
        l = sum4(l);

        // the four waves' parts together: rows c, values VE (4 g + r) + i
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
        const bool whole = i0 == 0 && i1 == v.nt;
        const bool some = (sm_any[0] | sm_any[1] | sm_any[2] | sm_any[3]) != 0;
        const int64_t slots = 2 * static_cast<int64_t>(gridDim.x);
        const int64_t slot = 2 * static_cast<int64_t>(blockIdx.x) + (t != t0);
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
                uint32_t* out = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.o) + b * a.o_token +
                                                            (hq0 + row) * a.o_head + d);
                *reinterpret_cast<uint2*>(out) = make_uint2(pack_16x2(x[0] * inv, x[1] * inv, DT),
                                                            pack_16x2(x[2] * inv, x[3] * inv, DT));
            } else {
                *reinterpret_cast<float4*>(part_out(a, rows_most, slot) + row * a.D + d) = make_float4(x[0], x[1], x[2], x[3]);
                if (d == 0) {
                    float* st = part_stat(a, rows_most, slots, slot) + 2 * row;
                    st[0] = top;
                    st[1] = some ? sum : -1.0f;                 // -1: nothing seen
                }
            }
        }
        t += i1 - i0;
    }
}

// One workgroup per (sequence, query head): joins a split sequence's pieces in their order; zeros for a
// sequence that sees nothing. groups: the workgroups of the kernel before.
__global__ void __launch_bounds__(64) attn_join_kernel(AttnArgs a, int row_tiles, int groups) {
    const int64_t b = blockIdx.x / a.Hq;
    const int hq = static_cast<int>(blockIdx.x % a.Hq);
    const int group = a.Hq / a.H, rows_most = group < 16 ? group : 16;
    const int64_t per = static_cast<int64_t>(a.H) * row_tiles;
    const Visible v = visible(a, a.lens[b]);
    uint16_t* out = static_cast<uint16_t*>(a.o) + b * a.o_token + hq * a.o_head;
    const int d = 4 * static_cast<int>(threadIdx.x);
    if (v.nt == 0) {
        if (d < a.D) *reinterpret_cast<uint2*>(out + d) = make_uint2(0, 0);
        return;
    }
    const Line line = line_of(a, per, groups);
    const int pair = hq / group * row_tiles + hq % group / 16, row = hq % group % 16;
    const int64_t t0 = count_tiles(a, 0, b) * per + static_cast<int64_t>(pair) * v.nt, t1 = t0 + v.nt;
    const int64_t w0 = t0 / line.piece, w1 = (t1 - 1) / line.piece;
    if (w0 == w1 || d >= a.D) return;
    const int64_t slots = 2 * static_cast<int64_t>(groups);
    auto slot_of = [&](int64_t w) { return 2 * w + (w * line.piece < t0); };
    float top = kNegInf;
    for (int64_t w = w0; w <= w1; ++w) top = __builtin_fmaxf(top, part_stat(a, rows_most, slots, slot_of(w))[2 * row]);
    const float base = top == kNegInf ? 0.0f : top;
    float sum = 0.0f, x[4] = {0, 0, 0, 0};
    bool some = false;
#pragma unroll 4
    for (int64_t w = w0; w <= w1; ++w) {
        const int64_t slot = slot_of(w);
        const float* st = part_stat(a, rows_most, slots, slot) + 2 * row;
        if (st[1] < 0.0f) continue;
        some = true;
        const float f = __builtin_amdgcn_exp2f(st[0] - base);
        sum = __builtin_fmaf(f, st[1], sum);
        const float4 y = *reinterpret_cast<const float4*>(part_out(a, rows_most, slot) + row * a.D + d);
        x[0] = __builtin_fmaf(f, y.x, x[0]);
        x[1] = __builtin_fmaf(f, y.y, x[1]);
        x[2] = __builtin_fmaf(f, y.z, x[2]);
        x[3] = __builtin_fmaf(f, y.w, x[3]);
    }
    const float inv = some ? 1.0f / sum : 0.0f;
    *reinterpret_cast<uint2*>(out + d) =
        make_uint2(pack_16x2(x[0] * inv, x[1] * inv, a.dtype), pack_16x2(x[2] * inv, x[3] * inv, a.dtype));
}

int decode_groups() {
    const int cus = device_cu_count();
    return (cus > 0 ? cus : 256) * 2;
}

template <int DP, int DT, bool I8>
int launch_width(const AttnArgs& a, int row_tiles, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(decode_groups()));
    if (a.page_shift >= 4)
        hipLaunchKernelGGL((attn_decode_kernel<DP, DT, I8, false>), grid, dim3(64 * kWaves), 0, stream, a, row_tiles);
    else
        hipLaunchKernelGGL((attn_decode_kernel<DP, DT, I8, true>), grid, dim3(64 * kWaves), 0, stream, a, row_tiles);
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
    int rc;
    if (a.dtype == kDtF16)
        rc = i8 ? launch_type<kDtF16, true>(a, row_tiles, stream) : launch_type<kDtF16, false>(a, row_tiles, stream);
    else
        rc = i8 ? launch_type<kDtBf16, true>(a, row_tiles, stream) : launch_type<kDtBf16, false>(a, row_tiles, stream);
    if (rc) return rc;
    hipLaunchKernelGGL(attn_join_kernel, dim3(static_cast<unsigned>(a.B * a.Hq)), dim3(64), 0, stream, a, row_tiles,
                       decode_groups());
    return launch_status("paged_attention");
}

}  // namespace mq
