// Upkeep of a paged key-value cache: new tokens' keys and values into their pages (kv_write), and the
// pages' bookkeeping and copies (fork, grow, free, compact).
//
// The cache of one layer is K and V [pages, kv_heads, page_size, head_dim] (any strides, unit inner one).
// Sequence b holds lens[b] tokens; token j lies in slot j % page_size of page table[b, j / page_size].
// refs[p] counts the sequences that hold page p. Everything here is exact: bytes are copied, integers
// counted. Pages are handed out lowest first, so the same calls give the same tables.
#include "mq_device.h"
#include "mq_internal.h"

namespace mq {
namespace {

// ---------------------------------------------------------------------------------------- kv_write
//
// Memory-bound: each new row of head_dim values is read once and stored once (16-bit cache: as it is;
// int8: codes and one fp32 scale, s = max(absmax / 127, 1e-10), q = rne(x / s), the rule of the linears'
// activation quantizer; a row that holds an infinity or NaN gets codes 0 and scale NaN, so it reads back
// as NaN). A row is 8 values a lane on the 2^k lanes that hold it, K and V by the same lanes. 16700 tokens
// of 8 heads of 128: 33 us, 4.1 TB/s (a plain copy: 5.1); 64 tokens: 3 us, the launch.

template <int DT, bool I8>
__global__ void __launch_bounds__(256) kv_write_kernel(KvWriteArgs a) {
    const int lanes = 1 << a.row_shift;                     // lanes per row
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> a.row_shift;
    const int c = static_cast<int>(threadIdx.x) & (lanes - 1);
    if (row >= a.T * a.H) return;
    const int64_t t = row / a.H, h = row - t * a.H;
    int64_t b, pos;
    if (a.cu_q) {
        // the sequence of token t: cu_q[b] <= t < cu_q[b + 1]
        int64_t lo = 0, hi = a.B;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (a.cu_q[mid] <= t) lo = mid; else hi = mid;
        }
        b = lo;
        if (t < a.cu_q[b] || t >= a.cu_q[b + 1]) return;    // behind the last sequence's tokens
        pos = static_cast<int64_t>(a.lens[b]) - a.cu_q[b + 1] + t;
    } else {
        b = t;
        pos = static_cast<int64_t>(a.lens[b]) - 1;
    }
    const int64_t at = pos >> a.page_shift;
    if (pos < 0 || at >= a.width) return;                   // no place for it: nothing is written
    const int page = a.table[b * a.ld_table + at];
    if (page < 0 || page >= a.pages) return;
    const int64_t slot = pos & ((int64_t(1) << a.page_shift) - 1);
    const bool ok = 8 * c < a.D;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const uint16_t* src = static_cast<const uint16_t*>(kv ? a.v : a.k) + t * (kv ? a.v_token : a.k_token) +
                              h * (kv ? a.v_head : a.k_head) + 8 * c;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (ok) x = *reinterpret_cast<const uint4*>(src);
        const int64_t off = page * a.c_page + h * a.c_head + slot * a.c_token + 8 * c;
        if constexpr (!I8) {
            if (ok) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(kv ? a.vc : a.kc) + off) = x;
        } else {
            float f[8];
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[2 * j] = DT == kDtF16 ? f16_bits_to_f32(static_cast<uint16_t>(w[j] & 0xffffu)) : bf16lo(w[j]);
                f[2 * j + 1] = DT == kDtF16 ? f16_bits_to_f32(static_cast<uint16_t>(w[j] >> 16)) : bf16hi(w[j]);
            }
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
                const float r = finite ? __builtin_rintf(f[j] / s) : 0.0f;
                q[j >> 2] |= (static_cast<uint32_t>(static_cast<int>(r)) & 0xffu) << (8 * (j & 3));
            }
            if (ok) *reinterpret_cast<uint2*>(static_cast<int8_t*>(kv ? a.vc : a.kc) + off) = make_uint2(q[0], q[1]);
            if (c == 0) (kv ? a.v_scale : a.k_scale)[page * a.s_page + h * a.s_head + slot * a.s_token] = s;
        }
    }
}

// ---------------------------------------------------------------------------------------- bookkeeping
//
// One workgroup decides (integers of a few thousand sequences and pages: microseconds of latency, no
// bandwidth: 7 us for 48 forks, a chain of dependent loads); the pages' contents are then copied by the whole device. Every decision is checked before
// anything is changed: a call that cannot be done whole leaves tables, lengths and counts as they were
// and says so in *status (0 done, > 0 pages missing, -1 an argument out of range).

constexpr int kPlan = 1024;

constexpr int kSeenRows = 1 << 16;   // rows per window of the bitmap below

struct PlanShared {
    int64_t wave[kPlan / 64];
    int bad;
    uint32_t seen[kSeenRows / 32];
};

__device__ __forceinline__ bool row_ok(int r, int64_t rows) { return r >= 0 && r < rows; }

// sh.bad is set if a valid row is in `rows` twice, or (others given) in both lists: a bitmap of the rows,
// a window of them at a time.
__device__ void check_distinct(const int* rows, const int* others, int n, int64_t all, PlanShared& sh) {
    for (int64_t r0 = 0; r0 < all; r0 += kSeenRows) {
        for (int i = threadIdx.x; i < kSeenRows / 32; i += kPlan) sh.seen[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kPlan) {
            const int64_t r = rows[i] - r0;
            if (r < 0 || r >= kSeenRows || !row_ok(rows[i], all)) continue;
            const uint32_t bit = 1u << (r & 31);
            if (atomicOr(&sh.seen[r >> 5], bit) & bit) sh.bad = 1;
        }
        __syncthreads();
        if (others)
            for (int i = threadIdx.x; i < n; i += kPlan) {
                const int64_t r = others[i] - r0;
                if (r < 0 || r >= kSeenRows || !row_ok(others[i], all)) continue;
                if ((sh.seen[r >> 5] >> (r & 31)) & 1) sh.bad = 1;
            }
        __syncthreads();
    }
}

// Exclusive prefix sum over the workgroup; *total = the sum (T: int, or int64_t where it may pass 32 bits).
template <typename T>
__device__ __forceinline__ T block_scan(T v, PlanShared& sh, T* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T x = v;
#pragma unroll
    for (int s = 1; s < 64; s <<= 1) {
        const T y = __shfl_up(x, s);
        if (lane >= s) x += y;
    }
    if (lane == 63) sh.wave[wave] = x;
    __syncthreads();
    T before = 0, all = 0;
    for (int w = 0; w < kPlan / 64; ++w) {
        const T y = static_cast<T>(sh.wave[w]);
        if (w < wave) before += y;
        all += y;
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// The lowest `need` pages without a holder, ascending, to list; returns how many there are (at most need).
__device__ int find_free(const int* refs, int64_t pages, int need, int* list, PlanShared& sh) {
    constexpr int kPer = 8;
    int found = 0;
    for (int64_t p0 = 0; p0 < pages && found < need; p0 += kPlan * kPer) {
        const int64_t p = p0 + static_cast<int64_t>(threadIdx.x) * kPer;
        uint32_t free = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (p + j < pages && refs[p + j] == 0) free |= 1u << j;
        int total;
        int at = found + block_scan<int>(__popc(free), sh, &total);
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if ((free >> j) & 1) {
                if (at < need) list[at] = static_cast<int>(p + j);
                ++at;
            }
        found += total;
    }
    return found < need ? found : need;
}

__device__ __forceinline__ int pages_of(int len, int shift) {
    return static_cast<int>((static_cast<int64_t>(len) + (1 << shift) - 1) >> shift);
}

// Child i takes sequence src[i]'s full pages (one holder more each) and a copy of its partly filled last
// page, if it has one; moves[2 i] -> moves[2 i + 1] (-1: none) is copied by the kernel behind this one.
__global__ void __launch_bounds__(kPlan) fork_plan_kernel(KvTables a, const int* src, const int* dst, int n, int* moves,
                                                           int* list, int* status) {
    __shared__ PlanShared sh;
    const int tid = threadIdx.x;
    if (tid == 0) sh.bad = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kPlan) {
        const int s = src[i], d = dst[i];
        bool bad = !row_ok(s, a.rows) || !row_ok(d, a.rows);
        if (!bad) {
            const int len = a.lens[s];
            bad = len < 0 || pages_of(len, a.page_shift) > a.width || a.lens[d] != 0;
        }
        if (bad) sh.bad = 1;
    }
    // a row that is forked to twice, or forked from while it is forked to
    check_distinct(dst, src, n, a.rows, sh);
    __syncthreads();
    if (!sh.bad) {
        bool bad = false;
        for (int i = tid >> 6; i < n; i += kPlan / 64) {
            const int s = src[i], held = pages_of(a.lens[s], a.page_shift);
            for (int j = tid & 63; j < held; j += 64) {
                const int p = a.table[s * a.ld_table + j];
                bad = bad || p < 0 || p >= a.pages;
            }
        }
        if (bad) sh.bad = 1;
    }
    __syncthreads();
    const bool bad = sh.bad != 0;
    int need = 0;
    if (!bad) {
        for (int i0 = 0; i0 < n; i0 += kPlan) {
            const int i = i0 + tid;
            const int part = i < n && (a.lens[src[i]] & ((1 << a.page_shift) - 1)) != 0;
            int total;
            const int at = need + block_scan(part, sh, &total);
            if (i < n) moves[2 * i + 1] = part ? at : -1;   // which of the free pages, for now
            need += total;
        }
    }
    const int found = need > 0 ? find_free(a.refs, a.pages, need, list, sh) : 0;
    if (bad || found < need) {
        for (int i = tid; i < n; i += kPlan) moves[2 * i] = moves[2 * i + 1] = -1;
        if (tid == 0 && status) *status = bad ? -1 : need - found;
        return;
    }
    __syncthreads();   // the list is whole
    for (int i = tid; i < n; i += kPlan) {
        const int s = src[i], d = dst[i], len = a.lens[s], full = len >> a.page_shift;
        const int k = moves[2 * i + 1];
        moves[2 * i] = -1;
        if (k >= 0) {
            const int p = list[k];
            moves[2 * i] = a.table[s * a.ld_table + full];
            moves[2 * i + 1] = p;
            a.refs[p] = 1;
        }
        a.lens[d] = len;
    }
    __syncthreads();   // the moves are whole
    for (int i = tid >> 6; i < n; i += kPlan / 64) {       // a wave a child
        const int s = src[i], d = dst[i], full = a.lens[s] >> a.page_shift, part = moves[2 * i + 1];
        for (int64_t j = tid & 63; j < a.width; j += 64) {
            int p = j == full ? part : -1;
            if (j < full) {
                p = a.table[s * a.ld_table + j];
                atomicAdd(a.refs + p, 1);                   // integer: any order gives the same count
            }
            a.table[d * a.ld_table + j] = p;
        }
    }
    if (tid == 0 && status) *status = 0;
}

// counts[i] tokens more for sequence rows[i]: its table gets the lowest free pages that they need.
__global__ void __launch_bounds__(kPlan) grow_plan_kernel(KvTables a, const int* rows, const int* counts, int n, int* first,
                                                           int* list, int* status) {
    __shared__ PlanShared sh;
    const int tid = threadIdx.x;
    if (tid == 0) sh.bad = 0;
    __syncthreads();
    int64_t need = 0;
    for (int i0 = 0; i0 < n; i0 += kPlan) {
        const int i = i0 + tid;
        int more = 0;
        if (i < n) {
            const int r = rows[i], c = counts[i];
            bool bad = !row_ok(r, a.rows) || c < 0;
            if (!bad) {
                const int len = a.lens[r];
                bad = len < 0 || static_cast<int64_t>(len) + c > (a.width << a.page_shift) ||
                      static_cast<int64_t>(len) + c > 0x7fffffff;
                if (!bad) more = pages_of(len + c, a.page_shift) - pages_of(len, a.page_shift);
            }
            if (bad) { sh.bad = 1; more = 0; }
        }
        // 1024 sequences of 2^21 pages each pass 32 bits; places past `pages` are not used (nothing is changed then)
        int64_t total;
        const int64_t at = need + block_scan<int64_t>(more, sh, &total);
        if (i < n) first[i] = at < a.pages ? static_cast<int>(at) : 0;
        need += total;
    }
    check_distinct(rows, nullptr, n, a.rows, sh);
    __syncthreads();
    const bool bad = sh.bad != 0;
    const int want = static_cast<int>(need < a.pages ? need : a.pages);
    const int found = bad || want == 0 ? 0 : find_free(a.refs, a.pages, want, list, sh);
    if (bad || found < need) {
        if (tid == 0 && status) *status = bad ? -1 : static_cast<int>(need - found < 0x7fffffff ? need - found : 0x7fffffff);
        return;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kPlan) {
        const int r = rows[i], len = a.lens[r], now = len + counts[i];
        const int have = pages_of(len, a.page_shift), more = pages_of(now, a.page_shift) - have;
        for (int j = 0; j < more; ++j) {
            const int p = list[first[i] + j];
            a.table[r * a.ld_table + have + j] = p;
            a.refs[p] = 1;
        }
        a.lens[r] = now;
    }
    if (tid == 0 && status) *status = 0;
}

// Sequence rows[blockIdx.x] gives its pages back. The exchange lets one holder of a table entry count it
// off, so a row that is given twice is freed once.
__global__ void __launch_bounds__(256) free_kernel(KvTables a, const int* rows) {
    const int r = rows[blockIdx.x];
    if (!row_ok(r, a.rows)) return;
    for (int64_t j = threadIdx.x; j < a.width; j += 256) {
        const int p = atomicExch(a.table + r * a.ld_table + j, -1);
        if (p >= 0 && p < a.pages) atomicSub(a.refs + p, 1);
    }
    if (threadIdx.x == 0) a.lens[r] = 0;
}

// With n pages held, the held pages at n and above move to the free ones below n, both ascending: the
// fewest moves that leave pages 0 .. n - 1 held. moves: the pairs, 2 * n ints at most; place[p]: where
// page p is afterwards; *live = n, *count = the number of moves.
__global__ void __launch_bounds__(kPlan) compact_plan_kernel(int* refs, int64_t pages, int* moves, int* place, int* live,
                                                              int* count) {
    __shared__ PlanShared sh;
    constexpr int kPer = 8;
    const int tid = threadIdx.x;
    int mine = 0;
    for (int64_t p = tid; p < pages; p += kPlan) mine += refs[p] > 0;
    int n;
    block_scan(mine, sh, &n);
    int holes = 0, movers = 0;
    for (int64_t p0 = 0; p0 < pages; p0 += kPlan * kPer) {
        const int64_t p = p0 + static_cast<int64_t>(tid) * kPer;
        uint32_t hole = 0, mover = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (p + j < pages) {
                const bool held = refs[p + j] > 0;
                if (p + j < n && !held) hole |= 1u << j;
                if (p + j >= n && held) mover |= 1u << j;
                place[p + j] = static_cast<int>(p + j);
            }
        int th, tm;
        int ah = holes + block_scan<int>(__popc(hole), sh, &th), am = movers + block_scan<int>(__popc(mover), sh, &tm);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if ((hole >> j) & 1) moves[2 * ah++ + 1] = static_cast<int>(p + j);
            if ((mover >> j) & 1) moves[2 * am++] = static_cast<int>(p + j);
        }
        holes += th;
        movers += tm;
    }
    __syncthreads();
    for (int i = tid; i < movers; i += kPlan) {
        const int s = moves[2 * i], d = moves[2 * i + 1];
        place[s] = d;
        refs[d] = refs[s];
        refs[s] = 0;
    }
    if (tid == 0) {
        *live = n;
        *count = movers;
    }
}

// ---------------------------------------------------------------------------------------- page copies
//
// Pages moves[2 i] -> moves[2 i + 1] of every layer of K and V, then of their scales. No page is both
// read and written, so the copies need no order. HBM-bound: 16-byte loads and stores, a unit of 16 KB
// per workgroup and step, with all its loads in flight before the first store; K and V in turns, so that
// both fill the chip together. Half of 2048 pages of 16 layers (820 MB): 165 us, 5.0 TB/s; 48 pages (59 MB): 25 us.
template <typename T>
__global__ void __launch_bounds__(256) copy_pages_kernel(KvCopyArgs a) {
    const int count = a.count ? *a.count : a.n;
    const uint32_t step = gridDim.x;
    // compaction: the tables' entries to their pages' new places, a workgroup a row
    if (a.place)
        for (int64_t r = blockIdx.x; r < a.tb.rows; r += step)
            for (int64_t j = threadIdx.x; j < a.tb.width; j += 256) {
                int* cell = a.tb.table + r * a.tb.ld_table + j;
                const int p = *cell;
                if (p >= 0 && p < a.tb.pages) *cell = a.place[p];
            }
    constexpr int kUnit = 256 * 4;                          // elements of T per unit
    for (int w = 0; w < a.tensors; w += 2) {                // K and V, then their scales: alike in pairs
        const uint32_t per = static_cast<uint32_t>(a.t[w].page_bytes / static_cast<int64_t>(sizeof(T)));
        const uint32_t units = (per + kUnit - 1) / kUnit, layers = static_cast<uint32_t>(a.layers);
        const uint32_t blocks = 2 * layers * units;         // of a move: below 2^31, as the entry points see to
        uint32_t u = blockIdx.x % blocks;
        for (int64_t i = blockIdx.x / blocks; i < count;) {
            const int s = a.moves[2 * i], d = a.moves[2 * i + 1];
            if (s >= 0) {
                const uint32_t unit = u % units, rest = u / units, layer = rest >> 1;
                const KvCopyTensor& t = a.t[w + (rest & 1)];
                char* base = static_cast<char*>(t.base) + layer * t.layer_bytes;
                const T* from = reinterpret_cast<const T*>(base + s * t.page_pitch);
                T* to = reinterpret_cast<T*>(base + d * t.page_pitch);
                const uint32_t e0 = unit * kUnit + threadIdx.x;
                T x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (e0 + j * 256 < per) x[j] = from[e0 + j * 256];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (e0 + j * 256 < per) to[e0 + j * 256] = x[j];
            }
            const uint64_t next = static_cast<uint64_t>(u) + step;
            i += static_cast<int64_t>(next < blocks ? 0 : next < 2ull * blocks ? 1 : next / blocks);
            u = static_cast<uint32_t>(next < blocks ? next : next < 2ull * blocks ? next - blocks : next % blocks);
        }
    }
}

int launch_copies(const KvCopyArgs& a, hipStream_t stream) {
    bool wide = true;
    for (int w = 0; w < a.tensors; ++w)
        wide = wide && a.t[w].page_bytes % 16 == 0 && a.t[w].page_pitch % 16 == 0 && a.t[w].layer_bytes % 16 == 0 &&
               reinterpret_cast<uintptr_t>(a.t[w].base) % 16 == 0;
    int64_t units = 0;
    for (int w = 0; w < a.tensors; w += 2) {
        const int64_t blocks = 2 * a.layers * ((a.t[w].page_bytes / (wide ? 16 : 4) + 1023) / 1024);
        const int64_t n = static_cast<int64_t>(a.n) * blocks;
        units = units > n ? units : n;
    }
    const int cus = device_cu_count();
    const int64_t most = static_cast<int64_t>(cus > 0 ? cus : 256) * 8;
    const int64_t grid = units < most ? (units > 0 ? units : 1) : most;
    if (wide)
        hipLaunchKernelGGL(copy_pages_kernel<uint4>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL(copy_pages_kernel<uint32_t>, dim3(static_cast<unsigned>(grid)), dim3(256), 0, stream, a);
    return launch_status("kv_copy");
}

}  // namespace

int launch_kv_write(const KvWriteArgs& in, int dtype, bool i8, hipStream_t stream) {
    KvWriteArgs a = in;
    a.row_shift = 0;
    while ((8 << a.row_shift) < a.D) ++a.row_shift;
    const int64_t threads = (a.T * a.H) << a.row_shift;
    const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
    if (!i8)
        hipLaunchKernelGGL((kv_write_kernel<kDtBf16, false>), grid, dim3(256), 0, stream, a);
    else if (dtype == kDtF16)
        hipLaunchKernelGGL((kv_write_kernel<kDtF16, true>), grid, dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((kv_write_kernel<kDtBf16, true>), grid, dim3(256), 0, stream, a);
    return launch_status("kv_write");
}

int launch_kv_fork(const KvTables& tb, const KvCopyArgs& copies, const int* src, const int* dst, int n, int* work,
                   int* status, hipStream_t stream) {
    KvCopyArgs c = copies;
    c.moves = work;
    c.n = n;
    hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlan), 0, stream, tb, src, dst, n, work, work + 2 * n, status);
    const int rc = launch_status("kv_fork");
    return rc ? rc : launch_copies(c, stream);
}

int launch_kv_grow(const KvTables& tb, const int* rows, const int* counts, int n, int* work, int* status,
                   hipStream_t stream) {
    hipLaunchKernelGGL(grow_plan_kernel, dim3(1), dim3(kPlan), 0, stream, tb, rows, counts, n, work, work + n, status);
    return launch_status("kv_grow");
}

int launch_kv_free(const KvTables& tb, const int* rows, int n, hipStream_t stream) {
    hipLaunchKernelGGL(free_kernel, dim3(static_cast<unsigned>(n)), dim3(256), 0, stream, tb, rows);
    return launch_status("kv_free");
}

int launch_kv_compact(const KvTables& tb, const KvCopyArgs& copies, int* work, int* live, hipStream_t stream) {
    KvCopyArgs c = copies;
    c.tb = tb;
    c.moves = work;                       // at most pages / 2 moves: a mover and a hole each
    c.place = work + tb.pages + 1;
    c.count = work + 2 * tb.pages + 1;
    c.n = static_cast<int>(tb.pages / 2);
    hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlan), 0, stream, tb.refs, tb.pages, work, work + tb.pages + 1,
                       live, work + 2 * tb.pages + 1);
    const int rc = launch_status("kv_compact");
    return rc ? rc : launch_copies(c, stream);
}

}  // namespace mq
