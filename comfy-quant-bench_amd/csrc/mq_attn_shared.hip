// Attention of one new token per sequence where groups of sequences hold the same first pages (alternatives of a prompt,
// questions about one document): the keys and values that a group shares are read once for all of its rows.
//
//   softmax over [shared keys, own keys] = both parts' unnormalised outputs over a common maximum, divided by both sums
//
// The plan (once for all layers of a step) finds the groups. The first kernel takes the rows of a group (its sequences' query
// heads of one cache head) as tiles of 16 RT rows over the shared keys, cut into as many pieces as there are compute units;
// the second joins the pieces of every row; the third is the single-token kernel over each sequence's own keys, which adds that
// part before it divides. (Pieces joined by the workgroup that brings the last one, as the single-token kernel does it:
// 32 sequences over 32000 tokens 160 us instead of XX, most of it one workgroup's waiting for 17 x 64 rows.)
//
// The first kernel is the single-token kernel's plan with more rows: HBM-bound where a group has few of them, keys and
// values go straight from the pages into registers, each wave with 32 keys of a tile and all rows. At 64 rows (RT = 4) a
// wave's 32 keys of 128 values cost 64 products of 16 cycles and some 1500 cycles of softmax against the 16 KB that it
// waits for, a fifth of what HBM brings a compute unit in that time, so larger groups, whose tiles read the keys again from
// the caches, are still served at that rate.
//
//   S^T = K Q^T, O^T = V^T P^T   operands and lanes as in mq_attn_decode_kernel.h, once per 16 rows; keys are unpacked
//                                and values paired once for all of them
//   softmax                      base 2, fp32; the reference maximum of a row moves (and its sums are rescaled) only when
//                                the row's maximum passes it by 2^8
//
// All rows of a group see all of its shared keys, so what is hidden (behind the shared length, in pages that are none) is
// hidden from every row.
#include "mq_attn_decode_kernel.h"

namespace mq {
namespace {

constexpr int kPlanThreads = 1024;

// ---------------------------------------------------------------------------------------- the plan
//
// Sequences belong together if their first pages are the same; what a group shares is the shortest run of equal pages
// of a member and the group's first sequence, no longer than any member. Integers of a few hundred sequences: latency.
// ON_CHIP: working space in LDS (up to kPlanRows sequences), else behind the plan.
constexpr int kPlanRows = 2048;

// (What atomics have changed is read past the first level cache.)
__device__ __forceinline__ int latest(const int* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

template <bool ON_CHIP>
__global__ void __launch_bounds__(kPlanThreads) shared_plan_kernel(const int* table, int64_t ld, int B, int width,
                                                                    const int* lens, int page_shift, int* plan) {
    __shared__ int wave_sum[2][kPlanThreads / 64];
    __shared__ int space[ON_CHIP ? 4 * kPlanRows : 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int* start = plan + SharedPlan::start();
    int* members = plan + SharedPlan::members(B);
    int* groups = plan + SharedPlan::groups(B);
    int* group_at = plan + SharedPlan::group_at(B);
    int* rank_at = plan + SharedPlan::rank_at(B);
    int* work = plan + SharedPlan::work(B);
    int* key = ON_CHIP ? space : work;                                  // first page
    int* lead = ON_CHIP ? space + kPlanRows : work + B;                 // first sequence with it
    int* tokens = ON_CHIP ? space + 2 * kPlanRows : work + 2 * static_cast<int64_t>(B);    // of a lead: what its group shares
    int* count = ON_CHIP ? space + 3 * kPlanRows : work + 3 * static_cast<int64_t>(B);     // of a lead: members
    for (int b = tid; b < B; b += kPlanThreads) {
        key[b] = lens[b] > 0 && width > 0 ? table[b * ld] : -1;
        tokens[b] = 0x7fffffff;
        count[b] = 0;
    }
    __syncthreads();
    for (int b = tid; b < B; b += kPlanThreads) {
        const int k = key[b];
        int l = -1;
        if (k >= 0) {
            l = 0;
            while (key[l] != k) ++l;
            atomicAdd(&count[l], 1);
        }
        lead[b] = l;
    }
    __syncthreads();
    // a wave a sequence: entries that it has in common with its lead, 256 at a time
    for (int b = wave; b < B; b += kPlanThreads / 64) {
        const int l = lead[b];
        if (l < 0 || l == b || latest(count + l) < 2) continue;
        const int most = lens[b] < lens[l] ? lens[b] : lens[l];
        const int entries = static_cast<int>((static_cast<int64_t>(most) + (1 << page_shift) - 1) >> page_shift);
        const int n = entries < width ? entries : width;
        int same = n;
        for (int i0 = 0; i0 < n; i0 += 256) {
            int x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = i0 + 64 * e + lane < n ? i0 + 64 * e + lane : n - 1;
                x[e] = table[b * ld + i];
                y[e] = table[l * ld + i];
            }
            int first = n;
#pragma unroll
            for (int e = 3; e >= 0; --e) {
                const uint64_t any = __ballot(x[e] < 0 || x[e] != y[e]);
                if (any) first = i0 + 64 * e + __builtin_ctzll(any);
            }
            if (first < n) {
                same = first;
                break;
            }
        }
        const int64_t held = static_cast<int64_t>(same) << page_shift;
        if (lane == 0) atomicMin(&tokens[l], held < most ? static_cast<int>(held) : most);
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
            key[b] = group0 + g - 1;                // a group: its number, where its members begin
            count[b] = -(member0 + m - n) - 1;
        }
        group0 += all_g;
        member0 += all_m;
        __syncthreads();
    }
    for (int b = tid; b < B; b += kPlanThreads) {
        const int l = lead[b], begin = l < 0 ? 0 : latest(count + l);
        const bool in = begin < 0;
        int before = 0;
        if (in) {
            for (int x = l; x < b; ++x) before += lead[x] == l;
            members[-begin - 1 + before] = b;
        }
        start[b] = in ? latest(tokens + l) : 0;
        group_at[b] = in ? key[l] : -1;
        rank_at[b] = before;
    }
    if (tid == 0) {
        plan[0] = group0;
        plan[1] = plan[2] = plan[3] = 0;
    }
}

// ---------------------------------------------------------------------------------------- the shared keys

constexpr int kSharedWaves = 4;
constexpr int rows16_of(int dp) { return dp == 256 ? 2 : 4; }     // 16-row tiles that a wave holds

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

constexpr int kSharedTile = kSharedWaves * kKeys;

__device__ __forceinline__ int groups_of(const AttnArgs& a) {
    const int n = a.plan[0], most = static_cast<int>(a.B) / 2;
    return n < 0 ? 0 : n < most ? n : most;
}

// The line of tiles: a group takes up its tiles for each (cache head, row tile) pair.
__device__ __forceinline__ int tiles_of(const Group& r) { return (r.tokens + kSharedTile - 1) / kSharedTile; }
template <int ROWS>
__device__ __forceinline__ int row_tiles_of(const AttnArgs& a, const Group& r) { return (r.count * (a.Hq / a.H) + ROWS - 1) / ROWS; }
// Its places (they fit 32 bits: the host refuses tables that could hold more), and those of the groups in front of group g.
template <int ROWS>
__device__ __forceinline__ int line_of(const AttnArgs& a, int n_groups, int g, int* before) {
    int all = 0, front = 0;
    for (int x = threadIdx.x & 63; x < n_groups; x += 64) {
        const Group r = group_of(a, x);
        const int n = tiles_of(r) * row_tiles_of<ROWS>(a, r) * a.H;
        all += n;
        front += x < g ? n : 0;
    }
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        all += __shfl_xor(all, s);
        front += __shfl_xor(front, s);
    }
    *before = __builtin_amdgcn_readfirstlane(front);
    return __builtin_amdgcn_readfirstlane(all);
}

// The pieces of every row together, in their order: a wave a row (of a sequence and query head).
template <int DP, int ROWS>
__global__ void __launch_bounds__(256) attn_shared_join_kernel(AttnArgs a, int pieces_most) {
    const int64_t at = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * 4 + (threadIdx.x >> 6)));
    if (at >= a.B * a.Hq) return;
    const int b = static_cast<int>(at / a.Hq), hq = static_cast<int>(at % a.Hq), lane = threadIdx.x & 63;
    const int g = a.plan[SharedPlan::group_at(a.B) + b], rank = a.plan[SharedPlan::rank_at(a.B) + b], n_groups = groups_of(a);
    if (g < 0 || g >= n_groups || rank < 0) return;
    const Group r = group_of(a, g);
    if (r.tokens == 0 || rank >= r.count) return;
    int before;
    const int total = line_of<ROWS>(a, n_groups, g, &before), piece = (total + pieces_most - 1) / pieces_most;
    const int group = a.Hq / a.H, h = hq / group, of = rank * group + hq % group, nt = tiles_of(r);
    const int s0 = before + (h * row_tiles_of<ROWS>(a, r) + of / ROWS) * nt, row = of % ROWS;
    const int p0 = s0 / piece, p1 = (s0 + nt - 1) / piece, slots = 2 * pieces_most;
    constexpr int V = DP == 256 ? 4 : DP == 128 ? 2 : 1, kAhead = 8;
    const int d = V * lane;
    float top = kNegInf, sum = 0.0f, y[V];
#pragma unroll
    for (int e = 0; e < V; ++e) y[e] = 0.0f;
    bool some = false;
    for (int p = p0; p <= p1; p += kAhead) {
        float2 st[kAhead];
        float z[kAhead][V];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const int x = p + i < p1 ? p + i : p1, slot = 2 * x + (x * piece < s0);
            st[i] = *reinterpret_cast<const float2*>(part_stat(a, ROWS, slots, slot) + 2 * row);
            const float* from = part_out(a, ROWS, slot) + row * a.D + (d < a.D ? d : 0);
#pragma unroll
            for (int e = 0; e < V; ++e) z[i][e] = from[e];
        }
        float most = top;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) most = p + i <= p1 && st[i].y >= 0.0f ? __builtin_fmaxf(most, st[i].x) : most;
        const float ref = most == kNegInf ? 0.0f : most, f = __builtin_amdgcn_exp2f(top - ref);
        top = most;
        sum *= f;
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] *= f;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (p + i > p1 || st[i].y < 0.0f) continue;                 // nothing seen there
            some = true;
            const float fz = __builtin_amdgcn_exp2f(st[i].x - ref);
            sum += st[i].y * fz;
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] += z[i][e] * fz;
        }
    }
    if (d < a.D)
#pragma unroll
        for (int e = 0; e < V; ++e) a.shared_out[at * a.D + d + e] = y[e];
    if (lane == 0) reinterpret_cast<float2*>(a.shared_stat)[at] = make_float2(top, some ? sum : -1.0f);
}

template <int DP, int DT, bool I8, bool SMALL>
__global__ void __launch_bounds__(64 * kSharedWaves, 1) attn_shared_kernel(AttnArgs a, bool quads) {
    constexpr int RT = rows16_of(DP), kTileRows = 16 * RT;
    constexpr int kWaves = kSharedWaves, kTile = kSharedTile;
    constexpr int E = I8 ? 1 : 2;
    constexpr int VE = DP / 16;
    constexpr int kSteps = DP / 32;
    constexpr int KB = 16;
    constexpr int KL = DP * E / 4 / KB;
    constexpr bool kSplit = I8 && DT == kDtF16;
    constexpr int MT = I8 ? kDtBf16 : DT;
    constexpr float kLift = MT == kDtF16 ? 14.0f - 8.0f : 0.0f;     // of fp16 probabilities; kSlack below what they may reach
    constexpr float kShift = MT == kDtF16 ? 8.0f : 0.0f;            // what the single-token kernel lifts them by beyond that
    constexpr float kSlack = 8.0f;
    __shared__ float sm_out[kWaves][16][DP + 4];
    __shared__ float sm_m[kWaves][kTileRows], sm_l[kWaves][kTileRows];
    __shared__ int sm_any[kWaves];
    // the query rows, as the products take them: [row tile][step][lane]
    __shared__ Frag sm_q[RT][kSteps][64], sm_q2[kSplit ? RT : 1][kSplit ? kSteps : 1][64];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int group = a.Hq / a.H;
    const int B = static_cast<int>(a.B);
    const int n_groups = groups_of(a);
    int front;
    const int total = line_of<kTileRows>(a, n_groups, 0, &front);
    const int piece = (total + gridDim.x - 1) / gridDim.x;
    const int t0 = blockIdx.x * piece, t1 = t0 + piece < total ? t0 + piece : total;
    if (t0 >= t1) return;

    const int mask = (1 << a.page_shift) - 1;
    const int last_page = static_cast<int>(a.pages) - 1;
    const uint32_t tok = static_cast<uint32_t>(a.c_token) * E;
    uint32_t ko[KL], vo[4];
#pragma unroll
    for (int x = 0; x < KL; ++x) ko[x] = (SMALL ? 0 : c * tok) + (KB / E * (4 * x + g) < a.D ? KB * (4 * x + g) : 0);
#pragma unroll
    for (int r = 0; r < 4; ++r) vo[r] = (SMALL ? 0 : (4 * g + r) * tok) + (VE * c < a.D ? VE * E * c : 0);
    const float scale = a.scale * kLog2e;

    int gi = 0, before = 0;
    for (int t = t0; t < t1;) {
        // the segment: tiles i0 .. i1 - 1 of group gi's cache head and row tile, whose tile 0 is place s0
        Group r = group_of(a, gi);      // (uniform: the plan is read at the same place by all lanes)
        while (t - before >= tiles_of(r) * row_tiles_of<kTileRows>(a, r) * a.H) {
            before += tiles_of(r) * row_tiles_of<kTileRows>(a, r) * a.H;
            ++gi;
            r = group_of(a, gi);
        }
        const int nt = tiles_of(r), pair = (t - before) / nt;
        const int s0 = before + pair * nt;
        const int i0 = t - s0, i1 = t1 - s0 < nt ? t1 - s0 : nt;
        const int rtiles = row_tiles_of<kTileRows>(a, r);
        const int h = pair / rtiles, row0 = pair % rtiles * kTileRows;
        const int rows = r.count * group - row0 < kTileRows ? r.count * group - row0 : kTileRows;
        const int* table = a.table + static_cast<int64_t>(r.lead) * a.ld_table;
        const char* kbase = static_cast<const char*>(a.kc) + static_cast<int64_t>(h) * a.c_head * E;
        const char* vbase = static_cast<const char*>(a.vc) + static_cast<int64_t>(h) * a.c_head * E;
        const float* ksb = I8 ? a.k_scale + h * a.s_head : nullptr;
        const float* vsb = I8 ? a.v_scale + h * a.s_head : nullptr;
        const int last = r.tokens - 1;
        // row x of the tile: its sequence (-1: none of the batch) and query head
        auto row_of = [&](int x, int* seq, int* hq) {
            const int at = row0 + x;
            const int s = a.plan[SharedPlan::members(a.B) + r.first + at / group];
            *seq = s >= 0 && s < B ? s : -1;
            *hq = h * group + at % group;
        };

        for (int x = wave; x < RT; x += kWaves) {
            int seq = -1, hq = 0;
            if (16 * x + c < rows) row_of(16 * x + c, &seq, &hq);
            const uint16_t* row = static_cast<const uint16_t*>(a.q) + (seq < 0 ? 0 : seq) * a.q_token + hq * a.q_head;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const int d = I8 ? 64 * (s >> 1) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
                uint4 y = make_uint4(0, 0, 0, 0);
                if (seq >= 0 && d < a.D) y = *reinterpret_cast<const uint4*>(row + d);
                Frag q{{y.x, y.y, y.z, y.w}};
                if constexpr (kSplit) {
                    Frag q2;
#pragma unroll
                    for (int j = 0; j < 4; ++j) split_f16(q.w[j], &q.w[j], &q2.w[j]);
                    sm_q2[x][s][lane] = q2;
                }
                sm_q[x][s][lane] = q;
            }
        }
        __syncthreads();

        Raw<KB> kr[2][2][KL];
        Raw<VE * E> vr[2][8];
        float ksc[2][2][4], vsc[2][2][4];
        uint32_t held[2];
        auto first_key = [&](int i) { return i * kTile + wave * kKeys; };
        // the 32 keys from j on: every address is inside the cache (a key that is not held reads page 0)
        auto load = [&](int buf, int j) __attribute__((always_inline)) {
            held[buf] = 0;
            const int ne = static_cast<int>(a.width) - 1;
            if constexpr (!SMALL) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int at = (j + 16 * u) >> a.page_shift;
                    const int p = scalar_word(table + __builtin_amdgcn_readfirstlane(at < ne ? at : ne));
                    const bool ok = p >= 0 && p <= last_page && at <= ne;
                    held[buf] |= ok ? 0xffffu << (16 * u) : 0u;
                    const int pg = ok ? p : 0, slot = (j + 16 * u) & mask;
                    const int64_t off = (pg * a.c_page + slot * a.c_token) * E;
                    const char* kp = kbase + off;
                    const char* vp = vbase + off;
#pragma unroll
                    for (int x = 0; x < KL; ++x) kr[buf][u][x] = load_raw<KB>(kp + ko[x]);
#pragma unroll
                    for (int y = 0; y < 4; ++y) vr[buf][4 * u + y] = load_row<VE * E, E>(vp, vo[y], VE * c, a.D);
                    if constexpr (I8) {
                        const int64_t so = pg * a.s_page + slot * a.s_token;
                        if (quads) {
                            const float4 x = *reinterpret_cast<const float4*>(ksb + so + 4 * g);
                            const float4 y = *reinterpret_cast<const float4*>(vsb + so + 4 * g);
                            ksc[buf][u][0] = x.x; ksc[buf][u][1] = x.y; ksc[buf][u][2] = x.z; ksc[buf][u][3] = x.w;
                            vsc[buf][u][0] = y.x; vsc[buf][u][1] = y.y; vsc[buf][u][2] = y.z; vsc[buf][u][3] = y.w;
                        } else {
#pragma unroll
                            for (int y = 0; y < 4; ++y) {
                                ksc[buf][u][y] = ksb[so + (4 * g + y) * a.s_token];
                                vsc[buf][u][y] = vsb[so + (4 * g + y) * a.s_token];
                            }
                        }
                    }
                }
            } else {
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
                    for (int y = 0; y < 4; ++y) {
                        const int cv = __shfl(code, 16 * u + 4 * g + y);
                        const int64_t pg = cv >> a.page_shift, slot = cv & mask;
                        vr[buf][4 * u + y] = load_row<VE * E, E>(vbase + (pg * a.c_page + slot * a.c_token) * E, vo[y], VE * c, a.D);
                        if constexpr (I8) {
                            ksc[buf][u][y] = ksb[pg * a.s_page + slot * a.s_token];
                            vsc[buf][u][y] = vsb[pg * a.s_page + slot * a.s_token];
                        }
                    }
                }
            }
        };
        f32x4 o[RT][VE];
        float m[RT], l[RT];
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            m[x] = kNegInf;
            l[x] = 0.0f;
#pragma unroll
            for (int i = 0; i < VE; ++i) o[x][i] = f32x4{0, 0, 0, 0};
        }
        bool any = false;           // a key that is held (the same for all rows)
        auto work = [&](int buf, int j) __attribute__((always_inline)) {
            const bool whole = held[buf] == 0xffffffffu && j + kKeys - 1 <= last;
            uint32_t see = 0xffu;
            if (!whole) {
                see = 0;
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    const int at = 16 * (x >> 2) + 4 * g + (x & 3);
                    see |= ((held[buf] >> at) & 1) && j + at <= last ? 1u << x : 0u;
                }
            }
            any = any || whole || __ballot(see != 0) != 0;
            Frag k[2][kSteps];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int st = 0; st < kSteps; ++st) {
                    if constexpr (I8) {
                        float f0[4], f1[4];
                        i8x4(kr[buf][u][st >> 1].w[2 * (st & 1)], f0);
                        i8x4(kr[buf][u][st >> 1].w[2 * (st & 1) + 1], f1);
                        k[u][st] = Frag{{bf16_exact2(f0[0], f0[1]), bf16_exact2(f0[2], f0[3]), bf16_exact2(f1[0], f1[1]),
                                         bf16_exact2(f1[2], f1[3])}};
                    } else {
                        k[u][st] = Frag{{kr[buf][u][st].w[0], kr[buf][u][st].w[1], kr[buf][u][st].w[2], kr[buf][u][st].w[3]}};
                    }
                    const int d = I8 ? 64 * (st >> 1) + 16 * g + 8 * (st & 1) : 32 * st + 8 * g;
                    if (d >= a.D) k[u][st] = Frag{{0, 0, 0, 0}};
                }
            Frag pf[RT], pf2[kSplit ? RT : 1];
#pragma unroll
            for (int x = 0; x < RT; ++x) {
                float p[8];
                // (read here every time: kept from tile to tile, all rows' would push others out of the registers)
                asm volatile("" ::: "memory");
                Frag q[kSteps], q2[kSplit ? kSteps : 1];
#pragma unroll
                for (int st = 0; st < kSteps; ++st) {
                    q[st] = sm_q[x][st][lane];
                    if constexpr (kSplit) q2[st] = sm_q2[x][st][lane];
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    f32x4 s = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int st = 0; st < kSteps; ++st) {
                        s = mfma16<MT>(k[u][st], q[st], s);
                        if constexpr (kSplit) s = mfma16<MT>(k[u][st], q2[st], s);
                    }
#pragma unroll
                    for (int y = 0; y < 4; ++y) p[4 * u + y] = s[y] * scale * (I8 ? ksc[buf][u][y] : 1.0f);
                }
                if (!whole)
#pragma unroll
                    for (int y = 0; y < 8; ++y) p[y] = (see >> y) & 1 ? p[y] : kNegInf;
                float top = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(p[0], p[1]), __builtin_fmaxf(p[2], p[3])),
                                            __builtin_fmaxf(__builtin_fmaxf(p[4], p[5]), __builtin_fmaxf(p[6], p[7])));
                top = max4(top);
                const bool move = top > m[x] + kSlack;
                if (__ballot(move)) {
                    const float f = move ? __builtin_amdgcn_exp2f(m[x] - top) : 1.0f;
                    m[x] = move ? top : m[x];
                    l[x] *= f;
#pragma unroll
                    for (int i = 0; i < VE; ++i) o[x][i] *= f;
                }
                const float base = m[x] == kNegInf ? 0.0f : m[x];
#pragma unroll
                for (int y = 0; y < 8; ++y) p[y] = __builtin_amdgcn_exp2f(p[y] - base + kLift);
                l[x] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                if constexpr (I8) {
#pragma unroll
                    for (int y = 0; y < 8; ++y)         // a key that is not seen has weight 0 whatever its scale holds
                        p[y] = (see >> y) & 1 ? p[y] * vsc[buf][y >> 2][y & 3] : 0.0f;
                }
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    pf[x].w[y] = pack_16x2(p[2 * y], p[2 * y + 1], MT);
                    if constexpr (kSplit)
                        pf2[x].w[y] = pack_16x2(p[2 * y] - bf16lo(pf[x].w[y]), p[2 * y + 1] - bf16hi(pf[x].w[y]), MT);
                }
            }
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
                        Frag v;
#pragma unroll
                        for (int x = 0; x < 4; ++x) v.w[x] = bf16_exact2(f8[2 * x][i], f8[2 * x + 1][i]);
#pragma unroll
                        for (int x = 0; x < RT; ++x) {
                            o[x][4 * w + i] = mfma16<MT>(v, pf[x], o[x][4 * w + i]);
                            if constexpr (kSplit) o[x][4 * w + i] = mfma16<MT>(v, pf2[x], o[x][4 * w + i]);
                        }
                    }
                }
            } else {
#pragma unroll
                for (int w = 0; w < VE / 2; ++w) {
                    Frag v0, v1;
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        v0.w[x] = pair16<0>(vr[buf][2 * x].w[w], vr[buf][2 * x + 1].w[w]);
                        v1.w[x] = pair16<1>(vr[buf][2 * x].w[w], vr[buf][2 * x + 1].w[w]);
                    }
#pragma unroll
                    for (int x = 0; x < RT; ++x) {
                        o[x][2 * w] = mfma16<MT>(v0, pf[x], o[x][2 * w]);
                        o[x][2 * w + 1] = mfma16<MT>(v1, pf[x], o[x][2 * w + 1]);
                    }
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

        // the waves' parts together, 16 rows at a time: rows c, values VE (4 g + y) + e
        const int slots = 2 * gridDim.x, slot = 2 * blockIdx.x + (t0 < s0);
        if (lane == 0) sm_any[wave] = any;
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            const float sum = sum4(l[x]);
            if (g == 0) {
                sm_m[wave][16 * x + c] = m[x];
                sm_l[wave][16 * x + c] = sum;
            }
        }
#pragma unroll
        for (int x = 0; x < RT; ++x) {
            __syncthreads();
#pragma unroll
            for (int y = 0; y < 4; ++y)
#pragma unroll
                for (int e = 0; e < VE; ++e) sm_out[wave][c][VE * (4 * g + y) + e] = o[x][e][y];
            __syncthreads();
            int some = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) some |= sm_any[w];
            for (int e = threadIdx.x; e < 16 * DP / 4; e += 64 * kWaves) {
                const int row = 16 * x + e / (DP / 4), d = 4 * (e % (DP / 4));
                if (row >= rows || d >= a.D) continue;
                float top = kNegInf;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) top = __builtin_fmaxf(top, sm_m[w][row]);
                const float base = top == kNegInf ? 0.0f : top;
                float sum = 0.0f, y[4] = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const float f = __builtin_amdgcn_exp2f(sm_m[w][row] - base);
                    sum += f * sm_l[w][row];
                    const float4 z = *reinterpret_cast<const float4*>(&sm_out[w][row & 15][d]);
                    y[0] = __builtin_fmaf(f, z.x, y[0]);
                    y[1] = __builtin_fmaf(f, z.y, y[1]);
                    y[2] = __builtin_fmaf(f, z.z, y[2]);
                    y[3] = __builtin_fmaf(f, z.w, y[3]);
                }
                float* to = part_out(a, kTileRows, slot) + row * a.D + d;
                *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
                if (d == 0)
                    *reinterpret_cast<float2*>(part_stat(a, kTileRows, slots, slot) + 2 * row) = make_float2(top + kShift, some ? sum : -1.0f);
            }
        }
        __syncthreads();                                // what is in LDS has been read
        t = s0 + i1;
    }
}

template <int DP, int DT, bool I8>
int shared_width(const AttnArgs& a, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(decode_groups()));
    const bool quads = I8 && a.s_token == 1 && a.s_page % 4 == 0 && a.s_head % 4 == 0 &&
                       (reinterpret_cast<uintptr_t>(a.k_scale) | reinterpret_cast<uintptr_t>(a.v_scale)) % 16 == 0;
    if (a.page_shift >= 4)
        hipLaunchKernelGGL((attn_shared_kernel<DP, DT, I8, false>), grid, dim3(64 * kSharedWaves), 0, stream, a, quads);
    else
        hipLaunchKernelGGL((attn_shared_kernel<DP, DT, I8, true>), grid, dim3(64 * kSharedWaves), 0, stream, a, quads);
    const int64_t rows = a.B * a.Hq;
    hipLaunchKernelGGL((attn_shared_join_kernel<DP, 16 * rows16_of(DP)>), dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, stream,
                       a, static_cast<int>(grid.x));
    return launch_status("paged_attention_shared");
}

template <int DT, bool I8>
int shared_type(const AttnArgs& a, hipStream_t stream) {
    if (a.D <= 64) return shared_width<64, DT, I8>(a, stream);
    if (a.D <= 128) return shared_width<128, DT, I8>(a, stream);
    return shared_width<256, DT, I8>(a, stream);
}

int rows_of(int D) { return 16 * rows16_of(D <= 64 ? 64 : D <= 128 ? 128 : 256); }

int64_t parts_bytes(int D) { return 2 * static_cast<int64_t>(decode_groups()) * rows_of(D) * (D + 2) * 4; }

}  // namespace

int64_t attn_shared_workspace_bytes(int Hq, int H, int D, int64_t B) {
    // both kernels' pieces (one behind the other in time), then the shared parts
    const int64_t single = attn_decode_workspace_bytes(Hq, H, D), parts = parts_bytes(D);
    return (single > parts ? single : parts) + B * Hq * (D + 2) * 4;
}

int64_t attn_shared_counters(int Hq, int H, int64_t B) { return attn_decode_counters(Hq, H, B); }

int launch_attn_shared(const AttnArgs& args, hipStream_t stream) {
    AttnArgs a = args;
    const int64_t single = attn_decode_workspace_bytes(a.Hq, a.H, a.D), parts = parts_bytes(a.D);
    a.shared_out = reinterpret_cast<float*>(static_cast<char*>(a.work) + (single > parts ? single : parts));
    a.shared_stat = a.shared_out + a.B * a.Hq * a.D;
    a.start = a.plan + SharedPlan::start();
    const bool i8 = a.k_scale != nullptr;
    int rc;
    if (a.dtype == kDtF16) rc = i8 ? shared_type<kDtF16, true>(a, stream) : shared_type<kDtF16, false>(a, stream);
    else rc = i8 ? shared_type<kDtBf16, true>(a, stream) : shared_type<kDtBf16, false>(a, stream);
    return rc ? rc : decode<true>(a, stream);
}

int launch_kv_shared(const int* table, int64_t ld_table, int64_t rows, int64_t width, const int* lens, int page_shift,
                     int* plan, hipStream_t stream) {
    hipLaunchKernelGGL(rows <= kPlanRows ? shared_plan_kernel<true> : shared_plan_kernel<false>, dim3(1), dim3(kPlanThreads), 0,
                       stream, table, ld_table, static_cast<int>(rows), static_cast<int>(width), lens, page_shift, plan);
    return launch_status("kv_shared");
}

}  // namespace mq
