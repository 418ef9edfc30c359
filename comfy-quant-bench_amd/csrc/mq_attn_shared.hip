// Attention of one new token per sequence where groups of sequences hold the same first pages (alternatives of a prompt,
// questions about one document): the keys and values that a group shares are read once for all of its rows.
//
//   softmax over [shared keys, own keys] = both parts' unnormalised outputs over a common maximum, divided by both sums
//
// The plan (once for all layers of a step) finds the groups. The first kernel takes the rows of a group (its sequences' query
// heads of one cache head) as tiles of 128 rows over the shared keys, cut into as many pieces as there are compute units. The
// second is the single-token kernel over each sequence's own keys; where it divides a row by its sum it adds the row's pieces of
// the first. (In a launch of their own the pieces cost 7 to 10 us a layer instead of 4 to 8. The workgroup that brings a
// tile's last piece, as in the single-token kernel, would have 128 rows of up to 17 pieces by itself.)
//
//   S^T = K Q^T, O^T = V^T P^T   products of 32 x 32 x 16. A wave has 32 rows, one a lane (and its partner), as B and P^T's
//                                operand straight from S^T's registers, as in mq_attn_prompt.hip
//   softmax                      base 2, fp32, against a row's running maximum; its sums are rescaled where it moves. The
//                                probabilities are rounded to the products' 16 bits as in the single-token kernel, the largest
//                                exact. (Moving only when the maximum passes its reference by 2^8, with fp16 probabilities held
//                                2^8 smaller for it: 2 % faster, but the output is off by 2.09e-3 instead of 1.85e-3 in bf16, where
//                                rounding it alone is 1.65e-3, and by 2.58e-4 instead of 2.32e-4 in fp16, and fp16
//                                probabilities below 2^-20 of the largest lose bits.)
//
// All rows of a group see all of its shared keys, so what is hidden (behind the shared length, in pages that are none) is
// hidden from every row.
//
// What bounds the first kernel: HBM, as it reads a tile of keys once for 128 rows, if enough is on its way (a compute unit's
// share of 5 TB/s over 2 us is 40 KB) and nothing else takes a tile's time (64 keys of 128 values, 32 KB: 1.6 us). So:
//   loads      go to LDS by themselves into a ring of tiles, three ahead of the one that is worked on, with the table's entries
//              of the tiles behind those among them: the loop has no other loads, and its one wait leaves those of the later
//              tiles on their way (in registers, one tile ahead: 8 us more)
//   LDS reads  of a tile's keys are all sent for before the first product, and its values before the softmax (each in front of
//              its product: 11 us more)
//   waves      eight at 128 values a head, so that a matrix unit has one wave's products while another's softmax runs; each
//              takes 32 of the 64 keys, or with up to 64 rows four do. 64 values: four, as a tile is half as long; 256: four,
//              whose sums need the registers of two
//   int8       16 bytes of a row by each thread, in 16 bits for all waves' products once
// 32 sequences of 32 heads over 32000 shared tokens of 8 cache heads, 131 MB: 49 us, 2.7 TB/s and 346 TFLOP/s (16 rows a
// wave with keys straight to registers, read again for every 64 rows: 22 us more).
#include "mq_attn_decode_kernel.h"

namespace mq {
namespace {

constexpr int kPlanThreads = 1024;

// ---------------------------------------------------------------------------------------- the plan
//
// Sequences belong together if their first pages are the same; what a group shares is the shortest run of equal pages
// of a member and the group's first sequence, no longer than any member. (So one member that has only a common beginning with
// the others leaves them only that to share, and of beginnings inside beginnings the outermost is shared.) Integers of a few hundred sequences: latency, of
// one workgroup (64 sequences of 9000 tokens in pages of 16: 12 us, a wave's tables one behind the other 14; 704 sequences that
// share nothing: 30 us, with a wave for each sequence's look at all the others 104).
// ON_CHIP: working space in LDS (up to kPlanRows sequences), else behind the plan.
constexpr int kPlanRows = 2048;

// (What atomics have changed is read past the first level cache.)
__device__ __forceinline__ int latest(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

template <bool ON_CHIP>
__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(const int* table, int64_t ld, int B, int width,
                                                                    const int* lens, int page_shift, int least_kib, int* plan) {
    __shared__ unsigned long long saved;
    __shared__ int wave_sum[2][kPlanThreads / 64];
    __shared__ int space[ON_CHIP ? 6 * kPlanRows : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* start = plan + SharedPlan::start();
    int* members = plan + SharedPlan::members(B);
    int* groups = plan + SharedPlan::groups(B);
    int* work = plan + SharedPlan::work(B);
    int* key = ON_CHIP ? space : work;                                  // first page
    int* lead = ON_CHIP ? space + kPlanRows : work + B;                 // first sequence with it
    int* tokens = ON_CHIP ? space + 2 * kPlanRows : work + 2 * static_cast<int64_t>(B);    // of a lead: what its group shares
    int* count = ON_CHIP ? space + 3 * kPlanRows : work + 3 * static_cast<int64_t>(B);     // of a lead: members
    int* rank = ON_CHIP ? space + 5 * kPlanRows : work + 4 * static_cast<int64_t>(B);      // members in front of it
    int* held_by = ON_CHIP ? space + 4 * kPlanRows : start;             // tokens of a sequence
    if (tid == 0) saved = 0;
    for (int b = tid; b < B; b += kPlanThreads) {
        const int n = lens[b], k = width > 0 ? table[b * ld] : -1;
        key[b] = n > 0 ? k : -1;
        tokens[b] = 0x7fffffff;
        held_by[b] = n;
    }
    if (ON_CHIP && tid < 8 && B + tid < ((B + 7) & ~7)) key[B + tid] = -2;
    __syncthreads();
    // a lane a sequence: the first with its first page, how many in front of it have that, how many all in all (from the last
    // sequence down; on chip the list goes on to a multiple of 8 with what no page is)
    for (int b0 = 64 * wave; b0 < B; b0 += kPlanThreads) {
        const int b = b0 + lane, k = b < B ? key[b] : -1;
        int l = -1, in_front = 0, in_wave = 0, behind = 0;
        auto look = [&](int from, int end, int& n, bool own) __attribute__((always_inline)) {
            for (int x0 = end - 8; x0 >= from; x0 -= 8) {
                int other[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) other[x] = key[ON_CHIP || x0 + x < B ? x0 + x : B - 1];
#pragma unroll
                for (int x = 7; x >= 0; --x) {
                    const bool same = other[x] == k && (ON_CHIP || x0 + x < B);
                    n += same;
                    if (own) in_wave += same && x0 + x < b;
                    l = same ? x0 + x : l;
                }
            }
        };
        const int end = (B + 7) & ~7, own_end = b0 + 64 < end ? b0 + 64 : end;
        look(own_end, end, behind, false);
        look(b0, own_end, behind, true);
        look(0, b0, in_front, false);
        if (b < B) {
            lead[b] = k < 0 ? -1 : l;
            rank[b] = in_front + in_wave;
            if (k >= 0 && l == b) count[b] = in_front + behind;
        }
    }
    __syncthreads();
    // a wave four sequences: entries that each has in common with its lead, 256 at a time
    constexpr int kFour = 4;
    for (int b0 = wave; b0 < B; b0 += kFour * (kPlanThreads / 64)) {
        int l[kFour], most[kFour], n[kFour], same[kFour], longest = 0;
        const int* mine[kFour];
        const int* first_of[kFour];
        bool open[kFour];
#pragma unroll
        for (int s = 0; s < kFour; ++s) {
            const int b = b0 + s * (kPlanThreads / 64), at = b < B ? b : b0;
            l[s] = __builtin_amdgcn_readfirstlane(lead[at]);
            open[s] = b < B && l[s] >= 0 && l[s] != b;
            const int of = open[s] ? l[s] : at, x = held_by[at], y = held_by[of];
            most[s] = __builtin_amdgcn_readfirstlane(x < y ? x : y);
            const int64_t entries = (static_cast<int64_t>(most[s]) + (1 << page_shift) - 1) >> page_shift;
            n[s] = !open[s] ? 0 : entries < width ? static_cast<int>(entries) : width;
            same[s] = n[s];
            mine[s] = table + at * ld;
            first_of[s] = table + of * ld;
            longest = longest > n[s] ? longest : n[s];
        }
        for (int i0 = 0; i0 < longest; i0 += 256) {
            int x[kFour][4], y[kFour][4];
#pragma unroll
            for (int s = 0; s < kFour; ++s)
                if (i0 < same[s])                       // (no difference yet)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = i0 + 64 * e + lane < n[s] ? i0 + 64 * e + lane : n[s] - 1;
                        x[s][e] = mine[s][i];
                        y[s][e] = first_of[s][i];
                    }
                else
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[s][e] = y[s][e] = 0;
#pragma unroll
            for (int s = 0; s < kFour; ++s)
#pragma unroll
                for (int e = 3; e >= 0; --e) {
                    const uint64_t any = __ballot(x[s][e] < 0 || x[s][e] != y[s][e]);
                    if (any) same[s] = i0 + 64 * e + __builtin_ctzll(any);
                }
        }
#pragma unroll
        for (int s = 0; s < kFour; ++s) {
            const int64_t held = static_cast<int64_t>(same[s]) << page_shift;
            if (lane == 0 && open[s]) atomicMin(&tokens[l[s]], held < most[s] ? static_cast<int>(held) : most[s]);
        }
    }
    __syncthreads();
    // groups in the order of their first sequences, members in their own
    int group0 = 0, member0 = 0;
    for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
        const int b = b0 + tid;
        const int held = b < B && lead[b] == b ? latest(count + b) : 0, keys = held >= 2 ? latest(tokens + b) : 0;
        const bool is = keys > 0;
        const int n = is ? held : 0;
        int g = is, m = n;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int y = __shfl_up(g, s), z = __shfl_up(m, s);
            if (lane >= s) { g += y; m += z; }
        }
        if (lane == 63) { wave_sum[0][wave] = g; wave_sum[1][wave] = m; }
        __syncthreads();
        int all_g = 0, all_m = 0;
        for (int w = 0; w < kPlanThreads / 64; ++w) {
            if (w < wave) { g += wave_sum[0][w]; m += wave_sum[1][w]; }
            all_g += wave_sum[0][w];
            all_m += wave_sum[1][w];
        }
        if (is) {
            int* to = groups + SharedPlan::kGroup * (group0 + g - 1);
            to[0] = keys;
            to[1] = b;
            to[2] = member0 + m - n;
            to[3] = n;
            atomicAdd(&saved, static_cast<unsigned long long>(n - 1) * keys);
            count[b] = -(member0 + m - n) - 1;      // a group: where its members begin
        }
        group0 += all_g;
        member0 += all_m;
        __syncthreads();
    }
    for (int b = tid; b < B; b += kPlanThreads) {
        const int l = lead[b], begin = l < 0 ? 0 : latest(count + l);
        const bool in = begin < 0;
        if (in) members[-begin - 1 + rank[b]] = b;
        start[b] = in ? latest(tokens + l) : 0;
    }
    if (tid == 0) {
        plan[0] = group0;
        plan[1] = saved < 0x7fffffff ? static_cast<int>(saved) : 0x7fffffff;
        plan[2] = least_kib;
        plan[3] = page_shift;
    }
}

// ---------------------------------------------------------------------------------------- the shared keys

constexpr int kSharedRows = 128;            // rows of a tile, 32 a wave
constexpr int tile_keys(int dp) { return dp == 256 ? 32 : 64; }     // keys and values of 16 or 32 KB
// Tiles of a workgroup at least: a piece more is one more to add for every row. (16 rows over 2000 tokens of 4 heads, both
// kernels: 1 tile 27.5 us, 2 27.3, 4 28.6)
constexpr int kLeastTiles = 2;
constexpr int tile_waves(int dp) { return dp == 128 ? 8 : 4; }
constexpr int tiles_ahead(int dp) { return dp == 64 ? 7 : 3; }      // on their way while one is worked on

struct Group {
    int tokens, lead, first, count;
};

// Group g of the plan, within bounds whatever it holds.
__device__ __forceinline__ Group group_of(const AttnArgs& a, int g) {
    const int* p = a.plan + SharedPlan::groups(a.B) + SharedPlan::kGroup * g;
    const int B = static_cast<int>(a.B), cap = static_cast<int>(a.width) << a.page_shift;
    Group r{p[0], p[1], p[2], p[3]};
    const bool ok = r.lead >= 0 && r.lead < B && r.first >= 0 && r.count > 0 && r.first < B && r.count <= B - r.first && r.tokens > 0;
    r.tokens = !ok ? 0 : r.tokens < cap ? r.tokens : cap;
    return r;
}

__device__ __forceinline__ int groups_of(const AttnArgs& a) {
    const int n = a.plan[0], most = static_cast<int>(a.B) / 2;
    return n < 0 || !worth_sharing(a) ? 0 : n < most ? n : most;
}

// The line of tiles (of `tile` keys): a group takes up its tiles for each (cache head, row tile) pair. (Its places fit 32 bits:
// the host refuses tables that could hold more.)
__device__ __forceinline__ int tiles_of(const Group& r, int tile) { return static_cast<int>((static_cast<uint32_t>(r.tokens) + tile - 1) / tile); }
__device__ __forceinline__ int row_tiles_of(const AttnArgs& a, const Group& r) {
    return (r.count * (a.Hq / a.H) + kSharedRows - 1) / kSharedRows;
}
__device__ __forceinline__ int places_of(const AttnArgs& a, const Group& r, int tile) { return tiles_of(r, tile) * row_tiles_of(a, r) * a.H; }

// Lane x: group g0 + x.
__device__ __forceinline__ Group groups_from(const AttnArgs& a, int g0) {
    const int at = g0 + (threadIdx.x & 63), most = static_cast<int>(a.B) / 2;
    Group r = group_of(a, at < most ? at : 0);          // (a group is read with their number: one wait less)
    if (at >= groups_of(a)) r.tokens = 0;
    return r;
}
__device__ __forceinline__ Group group_from(const Group& mine, int x) {
    return Group{__builtin_amdgcn_readlane(mine.tokens, x), __builtin_amdgcn_readlane(mine.lead, x),
                 __builtin_amdgcn_readlane(mine.first, x), __builtin_amdgcn_readlane(mine.count, x)};
}
// All places. mine: groups_from(a, 0).
__device__ __forceinline__ int line_of(const AttnArgs& a, const Group& mine, int n_groups, int tile) {
    int all = 0;
    for (int g0 = 0; g0 < n_groups; g0 += 64) all += places_of(a, g0 ? groups_from(a, g0) : mine, tile);
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) all += __shfl_xor(all, s);
    return __builtin_amdgcn_readfirstlane(all);
}
// The group that has place t of the line, and the places in front of it.
__device__ __forceinline__ Group group_at_place(const AttnArgs& a, const Group& mine, int n_groups, int t, int tile, int* before) {
    int front = 0;
    for (int g0 = 0; g0 < n_groups; g0 += 64) {
        const Group r = g0 ? groups_from(a, g0) : mine;
        const int n = places_of(a, r, tile);
        int sum = n;
#pragma unroll
        for (int s = 1; s < 64; s <<= 1) {
            const int y = __shfl_up(sum, s);
            sum += (threadIdx.x & 63) >= s ? y : 0;
        }
        const uint64_t behind = __ballot(front + sum > t);
        if (behind) {
            const int x = __builtin_ctzll(behind);
            *before = front + __builtin_amdgcn_readlane(sum - n, x);
            return group_from(r, x);
        }
        front += __builtin_amdgcn_readlane(sum, 63);
    }
    *before = front;
    return Group{0, 0, 0, 0};
}

template <int DP, bool I8>
struct __attribute__((aligned(16))) SharedLds {
    static constexpr int kTile = tile_keys(DP), kRing = tiles_ahead(DP) + 1, kWide = I8 ? 2 : kRing, kPages = DP == 64 ? 16 : 8;
    uint16_t k[kWide][kTile * DP], v[kWide][kTile * DP];    // tiles of 16 bits, chunks of 8 values in the order kswap and vswap
    int8_t kr[I8 ? kRing : 1][I8 ? kTile * DP : 16], vr[I8 ? kRing : 1][I8 ? kTile * DP : 16];  // int8 caches: as they come
    float scale[I8 ? kRing : 1][2][64];
    int page[tile_waves(DP)][kPages][64];    // a wave's own: where a tile's keys are
};

// 4 bytes per active lane from `src` to LDS bytes dst + 4 lane; loads on their way, up to N of a wave's newest
__device__ __forceinline__ void load_lds4(const void* src, uint32_t dst) {
    uint32_t m0;
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %1, off\n\ts_mov_b32 m0, %0"
                 : "=&s"(m0) : "v"(src), "s"(dst) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_but() {
    static_assert(N >= 0 && N < 64);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// (__syncthreads without a wait for loads that are meant to be on their way)
__device__ __forceinline__ void barrier_lds() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// DP: head width rounded up to 64, 128 or 256; DT: type of the tokens; I8: int8 cache.
template <int DP, int DT, bool I8>
__global__ void __launch_bounds__(64 * tile_waves(DP), 1) attn_shared_kernel(AttnArgs a) {
    using Lds = SharedLds<DP, I8>;
    constexpr int E = I8 ? 1 : 2, kTile = Lds::kTile, kRing = Lds::kRing, kAhead = kRing - 1, kPages = Lds::kPages, kThreads = 64 * tile_waves(DP);
    static_assert(kPages >= 2 * kRing - 1);
    constexpr bool kSplit = I8 && DT == kDtF16;         // fp16 rows against int8 keys: bf16 products of hi + lo
    constexpr int MT = I8 ? kDtBf16 : DT;               // type of the products
    // fp16 probabilities are held 2^14 times as large, as in the single-token kernel, which adds these
    constexpr float kLift = MT == kDtF16 ? 14.0f : 0.0f;
    constexpr int kSteps = DP / 16;                     // products over the width
    constexpr int kBlocks = DP / 32;                    // value blocks of the output
    constexpr int kV = 16 / E;                          // values of a 16-byte chunk in the cache
    constexpr int kPerKey = DP / kV;                    // chunks per key
    constexpr int KC = kTile * kPerKey / kThreads;           // chunks of keys (and of values) that a thread brings
    static_assert(KC > 0);
    constexpr int kLoads = 2 * KC + (I8 ? 1 : 0) + 1;   // a wave's loads for a tile: chunks, scales, pages of a later one
    extern __shared__ char lds_raw[];
    Lds& sm = *reinterpret_cast<Lds*>(lds_raw);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int q = lane & 31, hf = lane >> 5;
    const int group = a.Hq / a.H, B = static_cast<int>(a.B);
    const Group first = groups_from(a, 0);
    const int n_groups = groups_of(a);
    const int total = line_of(a, first, n_groups, kTile);
    const int even = (total + gridDim.x - 1) / gridDim.x, piece = even > kLeastTiles ? even : kLeastTiles;
    const int t0 = blockIdx.x * piece, t1 = t0 + piece < total ? t0 + piece : total;
    if (t0 >= t1) return;
    const int mask = (1 << a.page_shift) - 1;
    auto kswap = [](int key) { return key & 7; };
    auto vswap = [](int key) { return DP == 64 ? 4 * (key >> 1 & 1) : 4 * (key & 3); };
    const uint32_t lds_k = __builtin_amdgcn_readfirstlane(lds_offset(I8 ? (const void*)sm.kr : (const void*)sm.k) + wave * 1024);
    const uint32_t lds_v = __builtin_amdgcn_readfirstlane(lds_offset(I8 ? (const void*)sm.vr : (const void*)sm.v) + wave * 1024);
    const uint32_t lds_scale = __builtin_amdgcn_readfirstlane(lds_offset(sm.scale) + (wave & 1) * 256);
    const uint32_t lds_page = __builtin_amdgcn_readfirstlane(lds_offset(sm.page[wave]));
    const float size = __builtin_fabsf(a.scale * kLog2e), scale = size < 0x1p-100f ? 0x1p-100f : size;   // (0 times -infinity)
    const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
    // What no load writes, keys and values beyond the heads' width. (The zeros go over all of the ring: every wave's are there
    // before any wave's loads into it are sent for.)
    auto clear = [&] {
        if (!I8 && DP > a.D) {
            for (int e = tid; e < Lds::kWide * kTile * DP / 8; e += kThreads) {
                reinterpret_cast<uint4*>(sm.k)[e] = make_uint4(0, 0, 0, 0);
                reinterpret_cast<uint4*>(sm.v)[e] = make_uint4(0, 0, 0, 0);
            }
            __syncthreads();
        }
    };
    clear();

    for (int t = t0; t < t1;) {
        // the segment: tiles i0 .. i1 - 1 of a group's cache head and row tile, whose tile 0 is place s0
        int before;
        const Group r = group_at_place(a, first, n_groups, t, kTile, &before);
        const int nt = tiles_of(r, kTile);
        if (nt == 0) return;                            // (of a plan that is none)
        const int pair = (t - before) / nt;
        const int s0 = before + pair * nt;
        const int i0 = t - s0, i1 = t1 - s0 < nt ? t1 - s0 : nt;
        const int rtiles = row_tiles_of(a, r);
        const int h = pair / rtiles, row0 = pair % rtiles * kSharedRows;
        const int rows = r.count * group - row0 < kSharedRows ? r.count * group - row0 : kSharedRows;
        const int* table = a.table + static_cast<int64_t>(r.lead) * a.ld_table;
        const char* kbase = static_cast<const char*>(a.kc) + static_cast<int64_t>(h) * a.c_head * E;
        const char* vbase = static_cast<const char*>(a.vc) + static_cast<int64_t>(h) * a.c_head * E;
        const float* sbase = (wave & 1 ? a.v_scale : a.k_scale) + static_cast<int64_t>(h) * a.s_head;
        const uint32_t last = static_cast<uint32_t>(r.tokens) - 1;   // (no further than the table: group_of)

        const uint32_t pages = static_cast<uint32_t>(a.pages);

        // Where tile i's keys are, into the wave's own list
        auto look_up = [&](int i) __attribute__((always_inline)) {
            const uint32_t at = (static_cast<uint32_t>(i) * kTile + lane) >> a.page_shift, most = static_cast<uint32_t>(a.width) - 1;
            load_lds4(table + (at < most ? at : most), lds_page + (i & (kPages - 1)) * 256);
        };
        // key x of tile i: its page, or -1
        auto page_of = [&](int i, int x) __attribute__((always_inline)) {
            const int p = sm.page[wave][i & (kPages - 1)][x];
            return (i < i1) & (static_cast<uint32_t>(i) * kTile + x <= last) & (static_cast<uint32_t>(p) < pages) ? p : -1;
        };
        // Tile i on its way to ring place i % kRing (a key that is not held: the cache's first). 16-bit caches: 16-byte chunk c of
        // key x at c ^ kswap(x) and c ^ vswap(x)
        auto fetch = [&](int i) __attribute__((always_inline)) {
            const uint32_t place = static_cast<uint32_t>(i & (kRing - 1)) * kTile * DP * E;
            int64_t at[KC];
#pragma unroll
            for (int x = 0; x < KC; ++x) {
                const int key = tid / kPerKey + kThreads / kPerKey * x, p = page_of(i, key);
                at[x] = p < 0 ? 0 : static_cast<int64_t>(p) * a.c_page + ((static_cast<uint32_t>(i) * kTile + key) & mask) * a.c_token;
            }
            const int slot = tid % kPerKey, key0 = tid / kPerKey;       // (the order is the same for all of a thread's keys)
            const int kc = I8 ? slot : slot ^ kswap(key0), vc = I8 ? slot : slot ^ vswap(key0);
            if (kV * kc < a.D)
#pragma unroll
                for (int x = 0; x < KC; ++x) load_lds16(kbase + at[x] * E + 16 * kc, lds_k + place + 16 * kThreads * x);
            if (kV * vc < a.D)
#pragma unroll
                for (int x = 0; x < KC; ++x) load_lds16(vbase + at[x] * E + 16 * vc, lds_v + place + 16 * kThreads * x);
            if constexpr (I8) {
                if (lane < kTile) {
                    const int p = page_of(i, lane);
                    load_lds4(sbase + (p < 0 ? 0 : static_cast<int64_t>(p) * a.s_page + ((static_cast<uint32_t>(i) * kTile + lane) & mask) * a.s_token),
                              lds_scale + (i & (kRing - 1)) * 512);
                }
            }
            look_up(i + kAhead);
        };
#pragma unroll
        for (int x = 0; x < kAhead; ++x) look_up(i0 + x);

        // a wave's rows, and the 32 keys of a tile that it takes: eight waves take one half each, and so do four for few rows
        const bool few = kTile == 64 && rows <= kSharedRows / 2, split = kTile == 64 && (few || kThreads == 512);
        const int blocks = few ? 2 : 4, block = wave & (blocks - 1), part = wave / blocks;
        const int u0 = split ? part : 0, u1 = split ? part + 1 : kTile / 32, row = block * 32 + q;
        const bool active = block * 32 < rows && part < 2;
        // this lane's row: its sequence (-1: none) and query head
        int seq = -1, hq = 0;
        if (row < rows) {
            const int at = row0 + row;
            seq = a.plan[SharedPlan::members(a.B) + r.first + at / group];
            seq = seq >= 0 && seq < B ? seq : -1;
            hq = h * group + at % group;
        }
        Frag qf[kSteps], qf2[kSplit ? kSteps : 1];
        const uint16_t* qrow = static_cast<const uint16_t*>(a.q) + (seq < 0 ? 0 : seq) * a.q_token + hq * a.q_head;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int d = 16 * s + 8 * hf;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (seq >= 0 && d < a.D) x = *reinterpret_cast<const uint4*>(qrow + d);
            qf[s] = Frag{{x.x ^ sign, x.y ^ sign, x.z ^ sign, x.w ^ sign}};
            if constexpr (kSplit) {
#pragma unroll
                for (int j = 0; j < 4; ++j) split_f16(qf[s].w[j], &qf[s].w[j], &qf2[s].w[j]);
            }
        }
        // (The rows are here before the first tiles are sent for: a wait for them behind that would be one for all of those.)
#pragma unroll
        for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(qf[s].w[0]), "+v"(qf[s].w[1]), "+v"(qf[s].w[2]), "+v"(qf[s].w[3]));
        f32x16 o[kBlocks];
#pragma unroll
        for (int i = 0; i < kBlocks; ++i)
#pragma unroll
            for (int x = 0; x < 16; ++x) o[i][x] = 0.0f;
        float m = kNegInf, l = 0.0f;                    // reference maximum (of the scaled scores), sum of the lane's keys
        bool any = false;

        // 16-bit caches: this thread's own values of tile i whose keys are hidden: 0 (what is there may be an infinity)
        auto hide_own = [&](int i, uint64_t held) {
#pragma unroll
            for (int x = 0; x < KC; ++x)
                if (!(held >> (tid / kPerKey + kThreads / kPerKey * x) & 1))
                    reinterpret_cast<uint4*>(sm.v[i & (kRing - 1)])[tid + kThreads * x] = make_uint4(0, 0, 0, 0);
        };
        // int8 caches: this thread's own chunks of tile i in 16 bits
        auto widen = [&](int i) __attribute__((always_inline)) {
#pragma unroll
            for (int x = 0; x < KC; ++x) {
                const int e = tid + kThreads * x, key = e / kPerKey, c = e % kPerKey;
                uint4 y[2] = {reinterpret_cast<const uint4*>(sm.kr[I8 ? i & (kRing - 1) : 0])[e],
                              reinterpret_cast<const uint4*>(sm.vr[I8 ? i & (kRing - 1) : 0])[e]};
                if (kV * c >= a.D) y[0] = y[1] = make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int z = 0; z < 2; ++z) {
                    float f[4][4];
                    i8x4(y[z].x, f[0]);
                    i8x4(y[z].y, f[1]);
                    i8x4(y[z].z, f[2]);
                    i8x4(y[z].w, f[3]);
                    uint16_t* to = (z ? sm.v[i & 1] : sm.k[i & 1]) + key * DP;
                    const int swap = z ? vswap(key) : kswap(key);
#pragma unroll
                    for (int w = 0; w < 2; ++w)
                        *reinterpret_cast<uint4*>(to + 8 * ((2 * c + w) ^ swap)) =
                            make_uint4(bf16_exact2(f[2 * w][0], f[2 * w][1]), bf16_exact2(f[2 * w][2], f[2 * w][3]),
                                       bf16_exact2(f[2 * w + 1][0], f[2 * w + 1][1]), bf16_exact2(f[2 * w + 1][2], f[2 * w + 1][3]));
                }
            }
        };
        // a lane's places in the LDS rows (as in mq_attn_prompt.hip)
        const int kx = hf ^ (q & 7), vn = lane & 15;
        auto v_frag = [&](int buf, int u, int i, int x) __attribute__((always_inline)) {
            const int at = 4 * hf + (vn >> 2);
            const uint32_t base = lds_offset(sm.v[0]) + buf * kTile * DP * 2 + (32 * u + at) * DP * 2 +
                                  16 * ((4 * (i & 3)) ^ vswap(at)) + 32 * (lane >> 4 & 1) + 8 * (vn & 3);
            const LdsShort4 p = (LdsShort4)(base) + (256 * (i >> 2) + 16 * x * DP * 2) / 8;
            const auto y = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
            const auto z = __builtin_amdgcn_ds_read_tr16_b64_v4i16(p + DP * 2);
            const uint2 yw = __builtin_bit_cast(uint2, y), zw = __builtin_bit_cast(uint2, z);
            return Frag{{yw.x, yw.y, zw.x, zw.y}};
        };
        // keys 32 u .. 32 u + 31 of the tile
        auto work = [&](int buf, int ring, uint64_t held_all, int u) __attribute__((always_inline)) {
            const uint32_t held = static_cast<uint32_t>(held_all >> (32 * u));
            if (held == 0) return;
            any = true;
            // (All of the keys are sent for before the first product, and the values before the softmax: an LDS read takes as long
            // as four products, and a wave has only one other beside it.)
            const char* krow = reinterpret_cast<const char*>(sm.k[buf]) + (32 * u + q) * DP * 2;
            Frag k[kSteps];
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                const uint4 x = *reinterpret_cast<const uint4*>(krow + 16 * ((2 * (st & 3)) ^ kx) + (st >> 2) * 128);
                k[st] = Frag{{x.x, x.y, x.z, x.w}};
            }
            __builtin_amdgcn_sched_barrier(0);
            f32x16 s;
#pragma unroll
            for (int x = 0; x < 16; ++x) s[x] = 0.0f;
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
                s = mfma32<MT>(k[st], qf[st], s);
                if constexpr (kSplit) s = mfma32<MT>(k[st], qf2[st], s);
            }
            Frag v[kBlocks][2];
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                for (int x = 0; x < 2; ++x) v[i][x] = v_frag(buf, u, i, x);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (I8) {
#pragma unroll
                for (int r4 = 0; r4 < 4; ++r4) {
                    const float4 x = *reinterpret_cast<const float4*>(&sm.scale[ring][0][32 * u + 8 * r4 + 4 * hf]);
                    s[4 * r4] *= x.x;
                    s[4 * r4 + 1] *= x.y;
                    s[4 * r4 + 2] *= x.z;
                    s[4 * r4 + 3] *= x.w;
                }
            }
            const uint32_t see = held >> (4 * hf);          // bit 8 (x / 4) + x % 4: that key is seen (by every row)
            if (held != 0xffffffffu) {
#pragma unroll
                for (int x = 0; x < 16; ++x) s[x] = (see >> (8 * (x >> 2) + (x & 3))) & 1 ? s[x] : kNegInf;
            }
            float top = kNegInf;
#pragma unroll
            for (int x = 0; x < 16; ++x) top = __builtin_fmaxf(top, s[x]);
            top = max2(top) * scale;
            const bool move = top > m;
            if (__ballot(move)) {
                const float f = move ? __builtin_amdgcn_exp2f(m - top) : 1.0f;
                m = move ? top : m;
                l *= f;
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int x = 0; x < 16; ++x) o[i][x] *= f;
            }
            const float base = kLift - (m == kNegInf ? 0.0f : m);
            float sum[4] = {0, 0, 0, 0};
            Frag p[2], p2[kSplit ? 2 : 1];
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                float e[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    e[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * r4 + x], scale, base));
                    sum[x] += e[x];
                }
                if constexpr (I8) {
                    const float4 x = *reinterpret_cast<const float4*>(&sm.scale[ring][1][32 * u + 8 * r4 + 4 * hf]);
                    const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int y = 0; y < 4; ++y) e[y] *= xs[y];
                    if (held != 0xffffffffu)            // (0 times whatever a hidden key's scale is)
#pragma unroll
                        for (int y = 0; y < 4; ++y) e[y] = (see >> (8 * r4 + y)) & 1 ? e[y] : 0.0f;
                }
                const int x = r4 >> 1, w = 2 * (r4 & 1);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    p[x].w[w + y] = pack_16x2(e[2 * y], e[2 * y + 1], MT);
                    if constexpr (kSplit)
                        p2[x].w[w + y] = pack_16x2(e[2 * y] - bf16lo(p[x].w[w + y]), e[2 * y + 1] - bf16hi(p[x].w[w + y]), MT);
                }
            }
            l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
            for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    o[i] = mfma32<MT>(v[i][x], p[x], o[i]);
                    if constexpr (kSplit) o[i] = mfma32<MT>(v[i][x], p2[x], o[i]);
                }
        };

        // kAhead tiles are on their way while one is worked on. A tile's place in the ring is loaded again behind the barrier that
        // every wave reaches only when it is through with it, and each wave waits for its own loads in front of the barrier that the
        // others read them behind.
        wait_but<0>();
#pragma unroll
        for (int x = 0; x < kAhead; ++x) fetch(i0 + x);
        for (int i = i0; i < i1; ++i) {
            wait_but<(kAhead - 1) * kLoads>();
            const uint64_t held = __ballot(page_of(i, lane) >= 0) & (~uint64_t(0) >> (64 - kTile));
            if constexpr (I8) widen(i);
            else if (held != ~uint64_t(0) >> (64 - kTile)) hide_own(i, held);
            barrier_lds();
            fetch(i + kAhead);
            if (active)
#pragma unroll 1
                for (int u = u0; u < u1; ++u) work(I8 ? i & 1 : i & (kRing - 1), i & (kRing - 1), held, u);
        }
        wait_but<0>();
        barrier_lds();
        l = sum2(l);
        // a row's two parts together, the second's through LDS where the tiles were
        if (split) {
            constexpr int kRow = DP + 4;                // (rows begin 4 banks apart)
            float* sm_o = reinterpret_cast<float*>(lds_raw) + row * kRow;
            float2* sm_m = reinterpret_cast<float2*>(reinterpret_cast<float*>(lds_raw) + kSharedRows * kRow) + row;
            if (part == 1) {
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4)
                        *reinterpret_cast<float4*>(sm_o + 32 * i + 8 * r4 + 4 * hf) =
                            make_float4(o[i][4 * r4], o[i][4 * r4 + 1], o[i][4 * r4 + 2], o[i][4 * r4 + 3]);
                if (hf == 0) *sm_m = make_float2(m, any ? l : -1.0f);
            }
            __syncthreads();
            if (part == 0) {
                const float2 other = *sm_m;
                if (!(other.y == -1.0f)) {              // (of a part that saw nothing: sums of 0, a maximum of -infinity)
                    const float top = __builtin_fmaxf(m, other.x), ref = top == kNegInf ? 0.0f : top;
                    const float f = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(other.x - ref);
                    m = top;
                    l = l * f + other.y * f1;
#pragma unroll
                    for (int i = 0; i < kBlocks; ++i) {
                        float4 y[4];
#pragma unroll
                        for (int r4 = 0; r4 < 4; ++r4) y[r4] = *reinterpret_cast<const float4*>(sm_o + 32 * i + 8 * r4 + 4 * hf);
#pragma unroll
                        for (int r4 = 0; r4 < 4; ++r4) {
                            o[i][4 * r4] = o[i][4 * r4] * f + y[r4].x * f1;
                            o[i][4 * r4 + 1] = o[i][4 * r4 + 1] * f + y[r4].y * f1;
                            o[i][4 * r4 + 2] = o[i][4 * r4 + 2] * f + y[r4].z * f1;
                            o[i][4 * r4 + 3] = o[i][4 * r4 + 3] * f + y[r4].w * f1;
                        }
                    }
                    any = true;
                }
            }
        }
        // a tile's rows that one workgroup has seen all keys of are complete, others' pieces are in one of its two slots
        if (part == 0 && row < rows) {
            const bool complete = i0 == 0 && i1 == nt;
            const int64_t slots = 2 * gridDim.x, slot = 2 * blockIdx.x + (t0 < s0), place = slot * a.shared_most + row;
            const int64_t at = static_cast<int64_t>(seq < 0 ? 0 : seq) * a.Hq + hq;
            float* to = complete ? a.shared_out + at * a.D : a.shared_parts + place * a.D;
            float* stat = complete ? a.shared_stat + 2 * at : a.shared_parts + slots * a.shared_most * a.D + 2 * place;
            if (seq >= 0 || !complete) {
#pragma unroll
                for (int i = 0; i < kBlocks; ++i)
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) {
                        const int d = 32 * i + 8 * r4 + 4 * hf;
                        if (d < a.D)
                            *reinterpret_cast<float4*>(to + d) = make_float4(o[i][4 * r4], o[i][4 * r4 + 1], o[i][4 * r4 + 2], o[i][4 * r4 + 3]);
                    }
                if (hf == 0) *reinterpret_cast<float2*>(stat) = make_float2(m, any ? l : -1.0f);
            }
            if (hf == 0 && seq >= 0 && i0 == 0)
                reinterpret_cast<int4*>(a.shared_rows)[at] = make_int4(static_cast<int>(slot), complete ? -1 : (s0 + nt - 1) / piece, row, 0);
        }
        t = s0 + i1;
        if (t < t1) {
            __syncthreads();                            // what is in LDS has been read
            if (split) clear();                           // (over the part that was there)
        }
    }
}

template <int DP, int DT, bool I8>
int shared_width(const AttnArgs& a, hipStream_t stream) {
        const size_t lds = sizeof(SharedLds<DP, I8>);
    static_assert(sizeof(SharedLds<DP, I8>) <= 160 * 1024 && sizeof(SharedLds<DP, I8>) >= sizeof(float) * kSharedRows * (DP + 6));
    auto kern = attn_shared_kernel<DP, DT, I8>;
    if (lds > 65536 && hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize,
                                           static_cast<int>(lds)) != hipSuccess) {
        (void)hipGetLastError();
        set_error("paged_attention_shared: cannot reserve %zu bytes of LDS", lds);
        return -3;
    }
    hipLaunchKernelGGL(kern, dim3(static_cast<unsigned>(decode_groups())), dim3(64 * tile_waves(DP)), lds, stream, a);
    return launch_status("paged_attention_shared");
}

template <int DT, bool I8>
int shared_type(const AttnArgs& a, hipStream_t stream) {
    if (a.D <= 64) return shared_width<64, DT, I8>(a, stream);
    if (a.D <= 128) return shared_width<128, DT, I8>(a, stream);
    return shared_width<256, DT, I8>(a, stream);
}

// Rows of a slot: no tile has more.
int rows_most_of(int Hq, int H, int64_t B) {
    const int64_t rows = B * (Hq / H);
    return static_cast<int>(rows < kSharedRows ? rows : kSharedRows);
}
int64_t parts_bytes(int Hq, int H, int D, int64_t B) { return 2 * static_cast<int64_t>(decode_groups()) * rows_most_of(Hq, H, B) * (D + 2) * 4; }

}  // namespace

int64_t attn_shared_workspace_bytes(int Hq, int H, int D, int64_t B) {
    // the single-token kernel's pieces, the shared keys' pieces, their whole parts, where a row's are
    return attn_decode_workspace_bytes(Hq, H, D) + parts_bytes(Hq, H, D, B) + B * Hq * (D + 2 + 4) * 4;
}

int64_t attn_shared_counters(int Hq, int H, int64_t B) { return attn_decode_counters(Hq, H, B); }

int launch_attn_shared(const AttnArgs& args, hipStream_t stream) {
    AttnArgs a = args;
    // (each of them a multiple of 16 bytes: heads are of 8 values at least, slots and the slots' rows come in pairs of two floats)
    a.shared_most = rows_most_of(a.Hq, a.H, a.B);
    a.shared_parts = reinterpret_cast<float*>(static_cast<char*>(a.work) + attn_decode_workspace_bytes(a.Hq, a.H, a.D));
    a.shared_out = a.shared_parts + parts_bytes(a.Hq, a.H, a.D, a.B) / 4;
    a.shared_rows = reinterpret_cast<int*>(a.shared_out + a.B * a.Hq * a.D);
    a.shared_stat = reinterpret_cast<float*>(a.shared_rows + a.B * a.Hq * 4);
    a.start = a.plan + SharedPlan::start();
    const bool i8 = a.k_scale != nullptr;
    int rc;
    if (a.dtype == kDtF16) rc = i8 ? shared_type<kDtF16, true>(a, stream) : shared_type<kDtF16, false>(a, stream);
    else rc = i8 ? shared_type<kDtBf16, true>(a, stream) : shared_type<kDtBf16, false>(a, stream);
    return rc ? rc : decode<true>(a, stream);
}

int launch_kv_shared(const int* table, int64_t ld_table, int64_t rows, int64_t width, const int* lens, int page_shift,
                     int least_kib, int* plan, hipStream_t stream) {
    hipLaunchKernelGGL(rows <= kPlanRows ? shared_plan_kernel<true> : shared_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0,
                       stream, table, ld_table, static_cast<int>(rows), static_cast<int>(width), lens, page_shift, least_kib, plan);
    return launch_status("kv_shared");
}

}  // namespace mq
