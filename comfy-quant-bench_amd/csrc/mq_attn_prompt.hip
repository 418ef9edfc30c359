// Attention of ragged prompt chunks over a paged key-value cache (causal, sliding window, first tokens).
//
// Bound by MFMA and VALU together, which barely run side by side on this part: a wave's 64 keys of 32 rows are 32
// products of 32 cycles (D = 128) and about 1000 cycles of softmax, of which the exponentials are half (two
// waves' softmax beside each other's products, interleaved by hand, was slower). Long prompts: 840 to 880
// TFLOP/s from card to card (8192 tokens, 32 heads of 128: 624 to 654 us; a large library matrix product reaches 1190).
//
// A workgroup of four waves takes 128 rows of one cache head: row = (new token, query head of the group),
// token-major, so the heads that share keys and values share their tiles too and a short prompt fills a tile.
// Each wave keeps 32 rows; tiles of 64 keys go through LDS, double-buffered, one barrier a tile: the next tile's
// loads go there by themselves (16-bit caches; through registers: 795 us, half of that for stores and their
// addresses) while this one is worked on. Two workgroups a compute unit.
//
//   S^T = K Q^T      32x32x16 products. A: 32 keys, from LDS rows of 16-byte chunks (chunk x of key k at
//                    x ^ (k & 7): eight lanes read all banks). B: 32 query rows, kept in registers. Lane (q, h)
//                    = (l & 31, l >> 5) gets row q, keys 8 (r / 4) + 4 h + r % 4, r < 16.
//   softmax          in base 2 and fp32, row by row in one lane and its partner l ^ 32. The reference maximum is only
//                    moved (and the sums rescaled) when a row's maximum exceeds it by 2^8: any reference gives
//                    the same quotient, and fp32 sums have the range.
//   O^T = V^T P^T    B: a lane's 8 probabilities of keys 16 t + 4 h + {0 .. 3, 8 .. 11}, rounded to the products'
//                    16 bits: relative 2^-9 (bf16) or 2^-12 each, of random signs, so less than the output's own
//                    rounding (8192 tokens of bf16: 2.0e-3 from the exact result, 1.5e-3 if only the output were
//                    rounded; a second product of what is rounded off would double the MFMA work of this half). The
//                    sum that divides is of the unrounded ones. fp16 ones are held 2^7 times as large; A: V^T from
//                    LDS in just that order: 16-bit caches lie there as in the pages and are transposed by the
//                    LDS reads (16 lanes exchange 4 keys x 16 values); int8 ones are transposed by v_perm on the
//                    way in, where they become bf16.
//
// Few rows over many keys would leave the chip idle: their tiles are split over several workgroups (the host gives
// room for as many as fill it, the kernel takes as many as have tiles enough), whose sums meet in memory; of each
// wave's pieces the last one to arrive adds all in their order. 5 tokens behind 32768: 845 -> 75 us.
//
// Rows of one tile may differ in what they see: hidden scores become -infinity, and their weight 0 leaves the sum
// alone unless V holds an infinity or NaN there (0 times that is NaN). Tiles at an edge are looked through for
// such values while they are stored; if there are any, the products run on V with them zeroed, and products of
// ones count which rows see which kind, and add it.
#include "mq_attn.h"

namespace mq {
namespace {

constexpr int kRows = 128;     // rows per workgroup
constexpr int kTile = 64;      // keys per step
// Tiles that a piece of a split sequence has at least: a piece costs its first loads and its way through memory, some
// three tiles' time (2000 tokens of 8 heads: 16 tiles 68 us, 8 43, 4 41; 64 tokens behind 1500: 54, 33, 29).
constexpr int kLeast = 4;

// Whether either 16-bit value of w is an infinity or NaN; w with such values zeroed.
template <int DT>
__device__ __forceinline__ bool has_wild(uint32_t w) {
    constexpr uint32_t e = DT == kDtF16 ? 0x7c00u : 0x7f80u;
    return (w & e) == e || (w >> 16 & e) == e;
}
template <int DT>
__device__ __forceinline__ uint32_t tame(uint32_t w) {
    constexpr uint32_t e = DT == kDtF16 ? 0x7c00u : 0x7f80u;
    return ((w & e) == e ? 0u : w & 0xffffu) | ((w >> 16 & e) == e ? 0u : w & 0xffff0000u);
}

// 0: +infinity, 1: -infinity, 2: NaN, 3: a finite value.
template <int DT>
__device__ __forceinline__ int wild_kind(uint32_t w) {
    constexpr uint32_t e = DT == kDtF16 ? 0x7c00u : 0x7f80u;
    if ((w & 0x7fffu) < e) return 3;
    return (w & 0x7fffu) > e ? 2 : static_cast<int>(w >> 15);
}

template <int DP>
struct __attribute__((aligned(16))) Lds {
    uint16_t k[2][kTile * DP];
    uint16_t v[2][DP * kTile];
    float ks[2][kTile], vs[2][kTile];
    int64_t at[3][kTile];      // 16-bit caches: where a key's row begins (bytes; of a key that is not held: 0)
    int code[3][kTile];        // int8 caches: page << page_shift | slot, or -1
    uint64_t held[3];          // bit x: key x is in a page of the cache
    int wild;                  // an edge tile's values hold an infinity or NaN
};

// Between workgroups of one launch: past the caches that are not common to all of them.
__device__ __forceinline__ void send1(float* p, float x) {
    __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float receive1(const float* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// DP: head width rounded up to 64, 128 or 256; DT: type of the tokens; I8: int8 cache.
template <int DP, int DT, bool I8>
__global__ void __launch_bounds__(256, DP == 256 ? 1 : 2) attn_prompt_kernel(AttnArgs a) {
    constexpr int E = I8 ? 1 : 2;
    constexpr bool kSplit = I8 && DT == kDtF16;         // fp16 rows against int8 keys: bf16 products of hi + lo
    constexpr int MT = I8 ? kDtBf16 : DT;               // type of the products
    constexpr float kSlack = 8.0f;                      // how far a row's maximum may pass its reference (log2)
    constexpr float kLift = MT == kDtF16 ? 7.0f : 0.0f; // fp16 probabilities are held 2^7 times as large
    constexpr int kSteps = DP / 16;                     // products over the width
    constexpr int kBlocks = DP / 32;                    // value blocks of the output
    constexpr int KC = DP / 32;                         // key chunks (8 values) a thread stages
    constexpr int kPerKey = DP / 8;                     // chunks per key
    constexpr int VE = DP / 16;                         // values of a row that a thread stages, of 4 keys
    constexpr int VW = VE * E / 4;                      // dwords of them
    extern __shared__ char lds_raw[];
    Lds<DP>& sm = *reinterpret_cast<Lds<DP>*>(lds_raw);

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane & 31, hf = lane >> 5;
    const int group = a.Hq / a.H;
    const int h = static_cast<int>(blockIdx.x % a.H);
    // this workgroup's sequence and 128 rows of it; the last tiles, which see the most keys, come first
    int64_t want = static_cast<int64_t>(gridDim.x) / a.H - 1 - blockIdx.x / a.H, b = -1, tile = 0;
    for (int64_t b0 = 0; b0 < a.B; b0 += 64) {
        int64_t n = 0;
        if (b0 + lane < a.B) {
            const int64_t tok = static_cast<int64_t>(a.cu_q[b0 + lane + 1]) - a.cu_q[b0 + lane];
            n = tok > 0 ? (tok * group + kRows - 1) / kRows : 0;
        }
        int64_t x = n;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int64_t y = __shfl_up(x, s);
            if (lane >= s) x += y;
        }
        const uint64_t past = __ballot(x > want);
        if (past) {
            const int first = __builtin_ctzll(past);
            b = b0 + first;
            tile = want - __shfl(x - n, first);
            break;
        }
        want -= __shfl(x, 63);
    }
    b = __builtin_amdgcn_readfirstlane(static_cast<int>(b));
    tile = __builtin_amdgcn_readfirstlane(static_cast<int>(tile));
    if (b < 0) return;
    const int64_t tok0 = a.cu_q[b];
    int64_t tok1 = a.cu_q[b + 1];
    tok1 = tok1 < a.T ? tok1 : a.T;                     // nothing behind the rows of q, whatever cu_q says
    if (tok0 < 0 || tok0 >= tok1) return;
    const int64_t tokens = tok1 - tok0, rows = tokens * group;
    const int64_t pos0 = static_cast<int64_t>(a.lens[b]) - (static_cast<int64_t>(a.cu_q[b + 1]) - tok0);
    const int64_t row0 = tile * kRows;
    if (row0 >= rows) return;
    const int64_t cap = a.width << a.page_shift;
    const int64_t most = rows - 1;

    // positions: of this lane's row (rows past the end take the last one's), of the wave's and the workgroup's ends
    const int64_t wrow = row0 + wave * 32;
    const int64_t myrow = wrow + q < most ? wrow + q : most;
    const int64_t tok = myrow / group;
    const int64_t pos = pos0 + tok;
    const int64_t wpos_lo = pos0 + (wrow < most ? wrow : most) / group;
    const int64_t wpos_hi = pos0 + (wrow + 31 < most ? wrow + 31 : most) / group;
    const int64_t pos_lo = pos0 + row0 / group;
    const int64_t pos_hi = pos0 + (row0 + kRows - 1 < most ? row0 + kRows - 1 : most) / group;
    auto first_of = [&](int64_t p) { return a.window > 0 && a.window <= p ? p - a.window + 1 : int64_t(0); };
    const int64_t lo = first_of(pos), wlo_hi = first_of(wpos_hi), wlo_lo = first_of(wpos_lo);
    const int64_t sinks = a.sinks;

    // the tiles that some row sees: 0 .. ns - 1 (first tokens), then w0 ...
    const int64_t last = pos_hi < cap ? pos_hi : cap - 1;
    int ns = 0, nt = 0;
    int64_t w0 = 0;
    if (last >= 0 && a.pages > 0) {
        const int64_t start = first_of(pos_lo);
        w0 = start / kTile;
        const int64_t first = sinks < last + 1 ? sinks : last + 1;
        int64_t s = start > 0 ? (first + kTile - 1) / kTile : 0;
        int64_t nw = 0;
        if (last >= start) {
            nw = last / kTile - w0 + 1;
            s = s < w0 ? s : w0;
        }
        ns = static_cast<int>(s);
        nt = static_cast<int>(s + nw);
    }
    // few rows over many tiles: this workgroup takes pieces' share `piece` of them, and the last to end joins them
    const int piece = blockIdx.y, room = nt / kLeast;
    const int pieces = room < 2 ? 1 : room < static_cast<int>(gridDim.y) ? room : static_cast<int>(gridDim.y);
    if (piece >= pieces) return;
    const int i0 = static_cast<int>(static_cast<int64_t>(nt) * piece / pieces);
    const int i1 = static_cast<int>(static_cast<int64_t>(nt) * (piece + 1) / pieces);
    auto key_of = [&](int i) { return (i < ns ? static_cast<int64_t>(i) : w0 + (i - ns)) * kTile; };

    // the query rows
    Frag qf[kSteps], qf2[kSplit ? kSteps : 1];
    const int64_t qrow = (tok0 + tok) * a.q_token + (h * group + myrow % group) * a.q_head;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int d = 16 * s + 8 * hf;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (d < a.D) x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + qrow + d);
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
        qf[s] = Frag{{x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign}};
        if constexpr (kSplit) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t hi, low;
                split_f16(qf[s].w[j], &hi, &low);
                qf[s].w[j] = hi;
                qf2[s].w[j] = low;
            }
        }
    }
    f32x16 o[kBlocks];
#pragma unroll
    for (int i = 0; i < kBlocks; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;
    float m = kNegInf, l = 0.0f;                        // reference maximum (of the scaled scores), sum of the lane's keys
    bool any = false;
    // the scores' scale, its sign moved into the query rows; a scale of 0 as one too small to tell, so that a
    // hidden score's -infinity stays one (a NaN stays a NaN)
    const float size = __builtin_fabsf(a.scale * kLog2e), scale = size < 0x1p-100f ? 0x1p-100f : size;

    const int* table = a.table + b * a.ld_table;
    const char* kbase = static_cast<const char*>(a.kc) + static_cast<int64_t>(h) * a.c_head * E;
    const char* vbase = static_cast<const char*>(a.vc) + static_cast<int64_t>(h) * a.c_head * E;
    const int mask = (1 << a.page_shift) - 1;
    const int vg = tid >> 4, vc = tid & 15;             // V staging (int8): keys 4 vg .. 4 vg + 3, values VE vc ..

    // the table's entry for key x = lane of tile i (wave 0), as it is: a wait for it here would stop the wave
    auto look_up = [&](int i) -> int {
        const int64_t at = (key_of(i) + lane) >> a.page_shift;
        return table[at < a.width ? at : a.width - 1];
    };
    auto put_codes = [&](int ring, int i, int p) {
        const int64_t key = key_of(i) + lane;
        const bool ok = i < i1 && key <= last && key >> a.page_shift < a.width && p >= 0 && p < a.pages;
        const int code = ok ? (p << a.page_shift) | (static_cast<int>(key) & mask) : -1;
        const uint64_t held = __ballot(code >= 0);
        if constexpr (I8)
            sm.code[ring][lane] = code;
        else
            sm.at[ring][lane] = code < 0 ? 0 : 2 * (static_cast<int64_t>(code >> a.page_shift) * a.c_page + (code & mask) * a.c_token);
        if (lane == 0) sm.held[ring] = held;
    };

    uint4 kr[I8 ? KC : 1];
    uint32_t vr[I8 ? 4 : 1][VW];
    float sc = 0.0f;
    // 16-bit caches: keys and values of the tile in sm.at[ring] straight into half `buf`, rows as they are, 16-byte
    // chunk c of key k at c ^ kswap(k) and c ^ vswap(k). What is wider than the heads is not written (zeros stay there).
    const int slot = tid % kPerKey;
    auto kswap = [](int key) { return key & 7; };
    auto vswap = [](int key) { return DP == 64 ? 4 * (key >> 1 & 1) : 4 * (key & 3); };
    const uint32_t lds_k = __builtin_amdgcn_readfirstlane(lds_offset(sm.k[0]) + wave * 1024);
    const uint32_t lds_v = __builtin_amdgcn_readfirstlane(lds_offset(sm.v[0]) + wave * 1024);
    auto fetch = [&](int ring, int buf) __attribute__((always_inline)) {
        const int key = tid / kPerKey, kc = slot ^ kswap(key), vc = slot ^ vswap(key);   // the swaps are alike in all x
        if (8 * kc < a.D) {
            int64_t at[KC];
#pragma unroll
            for (int x = 0; x < KC; ++x) at[x] = sm.at[ring][key + kTile / KC * x];
#pragma unroll
            for (int x = 0; x < KC; ++x) load_lds16(kbase + at[x] + 16 * kc, lds_k + buf * kTile * DP * 2 + 4096 * x);
        }
        if (8 * vc < a.D) {
            int64_t at[KC];
#pragma unroll
            for (int x = 0; x < KC; ++x) at[x] = sm.at[ring][key + kTile / KC * x];
#pragma unroll
            for (int x = 0; x < KC; ++x) load_lds16(vbase + at[x] + 16 * vc, lds_v + buf * kTile * DP * 2 + 4096 * x);
        }
    };
    // this thread's own values of half `buf`: infinities and NaN become 0 and are noted
    auto tame_own = [&](int buf) {
#pragma unroll
        for (int x = 0; x < KC; ++x) {
            uint4* p = reinterpret_cast<uint4*>(sm.v[buf]) + tid + 256 * x;
            const uint4 y = *p;
            bool bad = has_wild<DT>(y.x);
            bad |= has_wild<DT>(y.y);
            bad |= has_wild<DT>(y.z);
            bad |= has_wild<DT>(y.w);
            if (bad) {
                sm.wild = 1;
                *p = make_uint4(tame<DT>(y.x), tame<DT>(y.y), tame<DT>(y.z), tame<DT>(y.w));
            }
        }
    };
    // int8 caches: the tile whose codes are in sm.code[ring] into registers (a key that is not held: zeros)
    auto load = [&](int ring) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < KC; ++x) {
            const int e = tid + 256 * x, key = e / kPerKey, d = 8 * (e % kPerKey);
            const int code = sm.code[ring][key];
            kr[x] = make_uint4(0, 0, 0, 0);
            if (code >= 0 && d < a.D) {
                const uint2 y = *reinterpret_cast<const uint2*>(
                    kbase + static_cast<int64_t>(code >> a.page_shift) * a.c_page + (code & mask) * a.c_token + d);
                kr[x].x = y.x;
                kr[x].y = y.y;
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int code = sm.code[ring][4 * vg + r];
            const char* p = vbase + static_cast<int64_t>(code >> a.page_shift) * a.c_page + (code & mask) * a.c_token + VE * vc;
#pragma unroll
            for (int w = 0; w < VW; ++w) vr[r][w] = 0;
            if (code >= 0 && VE * vc < a.D) {
                if constexpr (VW == 1) {
                    vr[r][0] = *reinterpret_cast<const uint32_t*>(p);
                } else if constexpr (VW == 2) {
                    const uint2 y = *reinterpret_cast<const uint2*>(p);
                    vr[r][0] = y.x;
                    vr[r][1] = y.y;
                } else {
                    const uint4 y = *reinterpret_cast<const uint4*>(p);
                    vr[r][0] = y.x;
                    vr[r][1] = y.y;
                    vr[r][2] = y.z;
                    vr[r][3] = y.w;
                }
            }
        }
        if (tid < 128) {
            const int code = sm.code[ring][tid & 63];
            sc = code < 0 ? 0.0f
                          : (tid < 64 ? a.k_scale : a.v_scale)[static_cast<int64_t>(code >> a.page_shift) * a.s_page +
                                                               h * a.s_head + (code & mask) * a.s_token];
        }
    };
    // the registers into half `buf`, keys as above, values transposed: value d of keys 4 vg .. 4 vg + 3 is 8 bytes in
    // chunk 2 (vg / 4) + vg % 2, half vg / 2 % 2
    auto store = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < KC; ++x) {
            const int e = tid + 256 * x, key = e / kPerKey, chunk = e % kPerKey;
            float f0[4], f1[4];
            i8x4(kr[x].x, f0);
            i8x4(kr[x].y, f1);
            *reinterpret_cast<uint4*>(&sm.k[buf][key * DP + 8 * (chunk ^ kswap(key))]) =
                make_uint4(bf16_exact2(f0[0], f0[1]), bf16_exact2(f0[2], f0[3]), bf16_exact2(f1[0], f1[1]),
                           bf16_exact2(f1[2], f1[3]));
        }
        const int chunk = 2 * (vg >> 2) + (vg & 1), half = (vg >> 1) & 1;
#pragma unroll
        for (int w = 0; w < VW; ++w) {
            float f[4][4];
#pragma unroll
            for (int r = 0; r < 4; ++r) i8x4(vr[r][w], f[r]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = VE * vc + 4 * w + e;
                *reinterpret_cast<uint2*>(&sm.v[buf][d * kTile + 8 * (chunk ^ ((d ^ (d >> 3)) & 7)) + 4 * half]) =
                    make_uint2(bf16_exact2(f[0][e], f[1][e]), bf16_exact2(f[2][e], f[3][e]));
            }
        }
        if (tid < 64) sm.ks[buf][tid] = sc;
        else if (tid < 128) sm.vs[buf][tid - 64] = sc;
    };
    // whether some row of the workgroup sees a part of tile i only
    auto edge_of = [&](int i) {
        const int64_t j = key_of(i);
        return !(j + kTile - 1 <= pos_lo && (j >= first_of(pos_hi) || j + kTile <= sinks));
    };

    // a lane's places in the LDS rows: chunk 2 s + h of key 32 u + q is at (2 s) ^ (h ^ (q & 7)), so four bases serve
    // all steps; int8: V^T's chunk 2 t + h of row 32 i + q at (2 t) ^ 4 (i % 2) ^ (h ^ (q ^ q / 8) % 8) likewise
    const int kx = hf ^ (q & 7), vx = hf ^ ((q ^ (q >> 3)) & 7);
    // 16-bit: 16 lanes together read four keys of 16 values and get a value of four keys each; lane n reads key n / 4,
    // values 4 (n % 4) .. of them
    const int vn = lane & 15;
    auto v_frag = [&](int buf, int i, int t) __attribute__((always_inline)) {
        if constexpr (I8) {
            const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(sm.v[buf]) + q * kTile * 2 +
                                                            16 * ((2 * t) ^ (4 * (i & 1)) ^ vx) + i * 32 * kTile * 2);
            return Frag{{x.x, x.y, x.z, x.w}};
        } else {
            const int row = 4 * hf + (vn >> 2);
            const uint32_t base = lds_offset(sm.v[0]) + buf * kTile * DP * 2 + row * DP * 2 +
                                  16 * ((4 * (i & 3)) ^ vswap(row)) + 32 * (lane >> 4 & 1) + 8 * (vn & 3);
            const LdsShort4 p = (LdsShort4)(base) + (256 * (i >> 2) + 16 * t * DP * 2) / 8;
            const auto x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
            const auto y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p + DP * 2);
            const uint2 xw = __builtin_bit_cast(uint2, x), yw = __builtin_bit_cast(uint2, y);
            return Frag{{xw.x, xw.y, yw.x, yw.y}};
        }
    };
    auto below = [](int64_t n) { return n >= 64 ? ~uint64_t(0) : n <= 0 ? uint64_t(0) : (uint64_t(1) << n) - 1; };

    // the row's visible keys of the tile at j: bit 8 (r / 4) + r % 4 of each half
    auto visible = [&](uint64_t held, int64_t j) {
        return (held & below(pos - j + 1) & (~below(lo - j) | below(sinks - j))) >> (4 * hf);
    };

    auto work = [&](int buf, int i, int ring) __attribute__((always_inline)) {
        const int64_t j = key_of(i);
        if (wrow > most) return;                                                   // no rows in this wave
        if (j > wpos_hi || (j + kTile <= wlo_lo && j >= sinks)) return;            // no row of the wave sees it
        const char* kp[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) kp[x] = reinterpret_cast<const char*>(sm.k[buf]) + q * DP * 2 + 16 * ((2 * x) ^ kx);
        f32x16 s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][r] = 0.0f;
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                const uint4 x = *reinterpret_cast<const uint4*>(kp[st & 3] + (st >> 2) * 128 + u * 32 * DP * 2);
                const Frag k{{x.x, x.y, x.z, x.w}};
                s[u] = mfma32<MT>(k, qf[st], s[u]);
                if constexpr (kSplit) s[u] = mfma32<MT>(k, qf2[st], s[u]);
            }
        }
        if constexpr (I8) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const float4 x = *reinterpret_cast<const float4*>(&sm.ks[buf][32 * u + 8 * r4 + 4 * hf]);
                    s[u][4 * r4] *= x.x;
                    s[u][4 * r4 + 1] *= x.y;
                    s[u][4 * r4 + 2] *= x.z;
                    s[u][4 * r4 + 3] *= x.w;
                }
        }
        const uint64_t held = sm.held[ring];
        const bool whole = held == ~uint64_t(0) && j + kTile - 1 <= wpos_lo && (j >= wlo_hi || j + kTile <= sinks);
        // bit 8 (r / 4) + r % 4 of see[u]: the row sees that key
        uint32_t see[2] = {0xffffffffu, 0xffffffffu};
        if (!whole) {
            const uint64_t vis = visible(held, j);
            see[0] = static_cast<uint32_t>(vis);
            see[1] = static_cast<uint32_t>(vis >> 32);
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[u][r] = (see[u] >> (8 * (r >> 2) + (r & 3))) & 1 ? s[u][r] : kNegInf;
        }
        any = any || ((see[0] | see[1]) & 0x0f0f0f0fu) != 0;
        float top = kNegInf;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, s[u][r]);
        top = max2(top) * scale;
        const bool move = top > m + kSlack;             // of this row: what other rows hold does not change it
        if (__ballot(move)) {
            const float f = move ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
            m = move ? top : m;
            l *= f;
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[i][r] *= f;
        }
        const float base = kLift - (m == kNegInf ? 0.0f : m);
        float sum[4] = {0, 0, 0, 0};
        Frag p[4], p2[kSplit ? 4 : 1];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                float e[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    e[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][4 * r4 + r], scale, base));
                    sum[r] += e[r];
                }
                if constexpr (I8) {
                    const float4 x = *reinterpret_cast<const float4*>(&sm.vs[buf][32 * u + 8 * r4 + 4 * hf]);
                    const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int r = 0; r < 4; ++r)         // a hidden key has weight 0 whatever its scale holds
                        e[r] = (see[u] >> (8 * r4 + r)) & 1 ? e[r] * xs[r] : 0.0f;
                }
                const int t = 2 * u + (r4 >> 1), w = 2 * (r4 & 1);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    p[t].w[w + x] = pack_16x2(e[2 * x], e[2 * x + 1], MT);
                    if constexpr (kSplit)
                        p2[t].w[w + x] = pack_16x2(e[2 * x] - bf16lo(p[t].w[w + x]), e[2 * x + 1] - bf16hi(p[t].w[w + x]), MT);
                }
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const Frag v = v_frag(buf, i, t);
                o[i] = mfma32<MT>(v, p[t], o[i]);
                if constexpr (kSplit) o[i] = mfma32<MT>(v, p2[t], o[i]);
            }
    };

    // tile i is worked on from half i % 2 while tile i + 1 is loaded, and tile i + 2's rows are looked up; what says
    // where a tile's keys are goes round three places, so one barrier a tile is enough
    if (i1 > i0) {
        if (wave == 0) {
            put_codes(0, i0, look_up(i0));
            put_codes(1, i0 + 1, look_up(i0 + 1));
        }
        if (tid == 0) sm.wild = 0;
        if constexpr (!I8) {                            // what no load writes: keys and values beyond the heads' width
            if (8 * kPerKey > a.D)
                for (int e = tid; e < 2 * kTile * kPerKey; e += 256) {
                    reinterpret_cast<uint4*>(sm.k[0])[e] = make_uint4(0, 0, 0, 0);
                    reinterpret_cast<uint4*>(sm.v[0])[e] = make_uint4(0, 0, 0, 0);
                }
        }
        __syncthreads();
        // a tile that some row sees in part, or with keys that are not held
        auto part = [&](int i, int ring) { return edge_of(i) || sm.held[ring] != ~uint64_t(0); };
        auto arrive = [&](int i, int ring, int buf) __attribute__((always_inline)) {
            if constexpr (I8) {
                store(buf);
            } else {
                wait_loads();
                if (part(i, ring)) tame_own(buf);
            }
        };
        if constexpr (I8) load(0);
        else fetch(0, 0);
        arrive(i0, 0, 0);
        __syncthreads();
        int r0 = 0, r1 = 1, r2 = 2;
        for (int i = i0; i < i1; ++i) {
            const int cur = (i - i0) & 1, nxt = cur ^ 1;
            const bool more = i + 1 < i1;
            int ahead = 0;
            if (wave == 0) ahead = look_up(i + 2);
            if (more) {
                if constexpr (I8) load(r1);
                else fetch(r1, nxt);
            }
            work(cur, i, r0);
            if (wave == 0) put_codes(r2, i + 2, ahead);
            if (more) arrive(i + 1, r1, nxt);
            __syncthreads();
            const int r = r0;
            r0 = r1;
            r1 = r2;
            r2 = r;
        }
        if constexpr (!I8) {
            if (sm.wild) {
                // values that are infinite or NaN at an edge: products of ones count, for every row and value, which
                // kinds its keys hold, and they are added
                for (int i = i0; i < i1; ++i) {
                    __syncthreads();
                    if (wave == 0) put_codes(0, i, look_up(i));
                    __syncthreads();
                    if (!part(i, 0)) continue;
                    fetch(0, 0);
                    wait_loads();
                    __syncthreads();
                    const uint64_t vis = visible(sm.held[0], key_of(i));
                    constexpr uint32_t kOne = MT == kDtF16 ? 0x3c00u : 0x3f80u;
                    Frag one[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int bit = 16 * t + 8 * (x >> 1) + 2 * (x & 1);
                            one[t].w[x] = ((vis >> bit) & 1 ? kOne : 0u) | ((vis >> (bit + 1)) & 1 ? kOne << 16 : 0u);
                        }
#pragma unroll
                    for (int e = 0; e < kBlocks; ++e)
#pragma unroll 1
                        for (int kind = 0; kind < 3; ++kind) {
                            f32x16 n;
#pragma unroll
                            for (int r = 0; r < 16; ++r) n[r] = 0.0f;
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const Frag w = v_frag(0, e, t);
                                Frag v;
#pragma unroll
                                for (int y = 0; y < 4; ++y)
                                    v.w[y] = (wild_kind<MT>(w.w[y] & 0xffffu) == kind ? kOne : 0u) |
                                             (wild_kind<MT>(w.w[y] >> 16) == kind ? kOne << 16 : 0u);
                                n = mfma32<MT>(v, one[t], n);
                            }
                            const float w = kind == 0 ? __builtin_inff() : kind == 1 ? -__builtin_inff() : __builtin_nanf("");
#pragma unroll
                            for (int r = 0; r < 16; ++r) o[e][r] += n[r] > 0.0f ? w : 0.0f;
                        }
                }
            }
        }
    }
    l = sum2(l);
    any = (static_cast<int>(any) | __shfl_xor(static_cast<int>(any), 32)) != 0;
    if (pieces > 1 && wrow <= most) {
        // a wave's pieces meet in memory; the last one adds all of them in their order, so the order of arrival
        // changes nothing
        constexpr int kPart = (16 * kBlocks + 2) * 64;
        const int64_t slot = static_cast<int64_t>(blockIdx.x) * 4 + wave;
        float* parts = static_cast<float*>(a.work) + slot * gridDim.y * kPart + lane;
        float* to = parts + static_cast<int64_t>(piece) * kPart;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) send1(to + 64 * (16 * i + r), o[i][r]);
        send1(to + 64 * 16 * kBlocks, m);
        send1(to + 64 * (16 * kBlocks + 1), any ? l : -1.0f);
        __builtin_amdgcn_s_waitcnt(0);                  // all lanes' values are where other workgroups see them
        int before = 0;
        if (lane == 0) before = __hip_atomic_fetch_add(a.counters + slot, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (__builtin_amdgcn_readfirstlane(before) != pieces - 1) return;
        if (lane == 0) __hip_atomic_store(a.counters + slot, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        m = kNegInf;
        for (int x = 0; x < pieces; ++x)
            m = __builtin_fmaxf(m, receive1(parts + static_cast<int64_t>(x) * kPart + 64 * 16 * kBlocks));
        l = 0.0f;
        any = false;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[i][r] = 0.0f;
#pragma unroll 1
        for (int x = 0; x < pieces; ++x) {
            const float* from = parts + static_cast<int64_t>(x) * kPart;
            const float mx = receive1(from + 64 * 16 * kBlocks), lx = receive1(from + 64 * (16 * kBlocks + 1));
            const float f = mx == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mx - m);
            const bool some = !(lx == -1.0f);           // -1: the row sees nothing of this piece
            any = any || some;
            l += some ? lx * f : 0.0f;
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float y = receive1(from + 64 * (16 * i + r));
                    o[i][r] += some ? y * f : 0.0f;
                }
        }
    }
    if (wrow + q <= most && wrow <= most) {
        const float inv = 1.0f / l;
        uint16_t* out = static_cast<uint16_t*>(a.o) + (tok0 + tok) * a.o_token + (h * group + myrow % group) * a.o_head;
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int d = 32 * i + 8 * r4 + 4 * hf;
                // nothing seen: zeros (hidden scores leave o as it was, but a scale that is NaN makes NaN of them too)
                if (d < a.D)
                    *reinterpret_cast<uint2*>(out + d) =
                        make_uint2(any ? pack_16x2(o[i][4 * r4] * inv, o[i][4 * r4 + 1] * inv, DT) : 0u,
                                   any ? pack_16x2(o[i][4 * r4 + 2] * inv, o[i][4 * r4 + 3] * inv, DT) : 0u);
            }
    }
}

// Workgroups for whole sequences: at least as many as there are row tiles.
int64_t row_tiles(int64_t T, int Hq, int H, int64_t B) { return (T * (Hq / H) / kRows + B) * H; }

// Pieces that a sequence may be split in: as many as give every compute unit two workgroups (what fits beside each
// other), 32 at most, and none for fewer than 2 x kLeast tiles.
int64_t most_pieces(int64_t T, int Hq, int H, int64_t B) {
    const int cus = device_cu_count();
    const int64_t n = 2 * (cus > 0 ? cus : 256) / row_tiles(T, Hq, H, B);
    return n < 2 ? 1 : n < 32 ? n : 32;
}

template <int DP, int DT, bool I8>
int launch_width(const AttnArgs& a, hipStream_t stream) {
    const int64_t tiles = row_tiles(a.T, a.Hq, a.H, a.B);
    int64_t pieces = most_pieces(a.T, a.Hq, a.H, a.B);
    const int64_t room = (a.width << a.page_shift) / (kTile * kLeast);
    pieces = room < 2 ? 1 : pieces < room ? pieces : room;
    const size_t lds = sizeof(Lds<DP>);
    auto kern = attn_prompt_kernel<DP, DT, I8>;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(lds)) != hipSuccess) {
        (void)hipGetLastError();
        set_error("paged_attention: cannot reserve %zu bytes of LDS", lds);
        return -3;
    }
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(pieces)), dim3(256), lds, stream, a);
    return launch_status("paged_attention");
}

template <int DT, bool I8>
int launch_type(const AttnArgs& a, hipStream_t stream) {
    if (a.D <= 64) return launch_width<64, DT, I8>(a, stream);
    if (a.D <= 128) return launch_width<128, DT, I8>(a, stream);
    return launch_width<256, DT, I8>(a, stream);
}

}  // namespace

int64_t attn_prompt_workspace_bytes(int64_t T, int Hq, int H, int D, int64_t B) {
    const int64_t pieces = most_pieces(T, Hq, H, B), wide = D <= 64 ? 64 : D <= 128 ? 128 : 256;
    return pieces < 2 ? 0 : row_tiles(T, Hq, H, B) * pieces * 4 * (wide / 2 + 2) * 64 * 4;
}

int64_t attn_prompt_counters(int64_t T, int Hq, int H, int64_t B) {
    return most_pieces(T, Hq, H, B) < 2 ? 0 : 4 * row_tiles(T, Hq, H, B);
}

int launch_attn_prompt(const AttnArgs& a, hipStream_t stream) {
    const bool i8 = a.k_scale != nullptr;
    if (a.dtype == kDtF16) return i8 ? launch_type<kDtF16, true>(a, stream) : launch_type<kDtF16, false>(a, stream);
    return i8 ? launch_type<kDtBf16, true>(a, stream) : launch_type<kDtBf16, false>(a, stream);
}

}  // namespace mq
