// Internal declarations shared by the libmq translation units (not part of the C ABI).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>
#include <string>

namespace mq {

// Thread-local error message behind mq_last_error().
void set_error(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
void clear_error();

// Translates the HIP launch status into the ABI status and message.
int launch_status(const char* what);

// Compute units of the current device (0 if the runtime cannot say). The attribute query runs
// once per device; later calls read the cached value, so the launchers can size their grids on
// every call without a runtime query.
int device_cu_count();

// --- rotate + quantize (mq_rotquant*.hip), one launcher per input type
int launch_rotquant_bf16(const uint16_t* x, int64_t M, int64_t K, int64_t ldx, int hblock, int bits,
                         int packed, void* q, int64_t ldq, float* scale, hipStream_t stream);
int launch_rotquant_f16(const uint16_t* x, int64_t M, int64_t K, int64_t ldx, int hblock, int bits,
                        int packed, void* q, int64_t ldq, float* scale, hipStream_t stream);
int launch_rotquant_f32(const float* x, int64_t M, int64_t K, int64_t ldx, int hblock, int bits,
                        int packed, void* q, int64_t ldq, float* scale, hipStream_t stream);

// --- SwiGLU prologue + rotate + quantize (mq_swiglu*.hip); h holds gate | up, K columns each.
// The fused activation T(silu(g) * u) rounds once; the eager one T(T(silu(g)) * u) twice.
int launch_swiglu_rotquant_bf16(const uint16_t* h, int64_t M, int64_t K, int64_t ldh, int hblock, int bits,
                                int packed, void* q, int64_t ldq, float* scale, hipStream_t stream);
int launch_swiglu_rotquant_f16(const uint16_t* h, int64_t M, int64_t K, int64_t ldh, int hblock, int bits,
                               int packed, void* q, int64_t ldq, float* scale, hipStream_t stream);
int launch_swiglu_eager_rotquant_bf16(const uint16_t* h, int64_t M, int64_t K, int64_t ldh, int hblock, int bits,
                                      int packed, void* q, int64_t ldq, float* scale, hipStream_t stream);
int launch_swiglu_eager_rotquant_f16(const uint16_t* h, int64_t M, int64_t K, int64_t ldh, int hblock, int bits,
                                     int packed, void* q, int64_t ldq, float* scale, hipStream_t stream);

// --- load-time decode of the shipped asym_w4a8_int8 codebook weights (mq_codebook.hip), to rows or
// (tile) to the 16-row tiles of GemmArgs::wtile
int launch_decode_w4a8_codebook(const uint8_t* qdata, int64_t ldq, const uint8_t* s_rel, int64_t lds,
                                const float* s_channel, const float* codebook, int group_size, int64_t N,
                                int64_t K, int8_t* q8, int64_t ldq8, float* row_scale, bool tile,
                                hipStream_t stream);

// --- offline weight quantizer (mq_wquant.hip); dtype / format are MQ_DT_* / MQ_WFMT_*
int launch_quantize_weight(const void* w, int dtype, int64_t N, int64_t K, int64_t ldw, int hblock, int format,
                           void* q, int64_t ldq, void* scale, int64_t ld_scale, void* zero, int64_t ld_zero,
                           int* nonfinite, hipStream_t stream);

// int8 weights [N, K] into the 16-row tile layout of GemmArgs::wtile (mq_wquant.hip)
int launch_tile_weight_i8(const uint8_t* w, int64_t ldw, int64_t N, int64_t K, uint8_t* out, hipStream_t stream);

// packed 4-bit weights into int8 16-row tiles (mq_expand_weight_w4's layouts; mq_wquant.hip)
// dwords per [g][c] row of the scale pairs that expanded 4-bit weights carry (MQ_SCALE_PAIR_LD)
__host__ __device__ inline int64_t scale_pair_ld(int64_t N) { return ((N + 15) / 16 + 17) / 2; }
int launch_expand_scales_w4(const uint16_t* ws, int64_t ldws, int64_t N, int64_t K, uint32_t* out,
                            hipStream_t stream);
int launch_expand_weight_w4(const uint8_t* qw, int64_t ldw, const uint8_t* wz, int64_t ldwz, int64_t N, int64_t K,
                            int layout, uint8_t* out, hipStream_t stream);

// --- GEMMs (mq_gemm.hip)
enum class WKind : int { U4Asym = 0, I4Sym = 1, I8 = 2 };
enum class Epi : int { GroupScale = 0, GroupPartials = 1, RowScale = 2, RowAcc = 3 };

struct GemmArgs {
    const int8_t* qa;
    int64_t lda;
    const float* sa;
    const uint8_t* qw;
    int64_t ldw;
    const uint16_t* ws16;   // per-group fp16 scales [N, ldws]
    int64_t ldws;
    const float* ws32;      // per-row fp32 scales [N]
    const uint8_t* wz;      // packed u4 zero-points [N, ldwz]
    int64_t ldwz;
    const void* bias;       // [N] of type bias_dtype, or null
    void* y;                // [M, ldy] of type y_dtype
    int64_t ldy;
    int bias_dtype;         // MQ_DT_BF16 / MQ_DT_F16 / MQ_DT_F32
    int y_dtype;
    int32_t* part;          // int32 partials / accumulators
    int64_t M, N, K;
    int act_mode;           // group-scale GEMMs: MQ_ACT_* layout of qa (include/mq.h)
    // split-K (wide kernel, GroupScale / RowScale only): ksplit slices of kgroups K groups each
    // (a multiple of 4) write fp32 (GroupScale) or int32 (RowScale) partial outputs [ksplit][M][N]
    // to work, which a reduction kernel sums and finishes; ksplit 1 = no split
    int ksplit = 1;
    int kgroups = 0;
    void* work = nullptr;
    int64_t work_bytes = 0;   // capacity of work offered by the caller
    // output tile of the wide kernel: 256 (256 x 256), 192 (256 x 192) or 128 (128 x 128); 0:
    // choose_tile decides
    int tile = 0;
    // int8 weights (WKind::I8) in 16-row tiles: [ceil(N / 16)][K / 64][16][64] bytes, so that a
    // 1 KB block holds one K group of 16 consecutive rows (ldw = K); 0: rows of ldw bytes. With a
    // 4-bit kind (group scales): the weights expanded to int8 in those tiles (mq_expand_weight_w4),
    // read by the wide kernel only; wz then only tells uint4 asymmetric (non-null) from signed
    int wtile = 0;
    // activation codes (qa) in the same 16-row tiles, [ceil(M / 16)][K / 64][16][64] (lda = K): written
    // so by the whole-linear entries when the wide or few-row kernel runs their product. The last band
    // is 16 rows whatever M is: the few-row kernel reads its rows past M (and drops what they give)
    int atile = 0;
    // One-row whole linears (gemv_quantizes_row): the GEMV rotates and quantizes the activation
    // row x (x_dtype, Hadamard block hblock, x_bits-bit codes) itself instead of reading qa / sa
    const void* x = nullptr;
    int x_dtype = 0;
    int hblock = 0;
    int x_bits = 8;
};

// Output tile of the wide kernel for an M x N product (a tile code as above): 128 when 256 x 256
// tiles would occupy at most half of the compute units; else 192 when its rounds of resident
// workgroups take less time than 256 x 256 tiles (with their trailing rows, tail_rows) would
// (N = 3072 at M = 4096: 256 tiles in one round instead of 192); else 256.
int choose_tile(int64_t M, int64_t N);

// K slices for a GEMM of this shape with a workspace of work_bytes (1 = no split): used when the
// tiles of choose_tile leave most compute units idle (small M). int_sums: the row-scale epilogue
// (int32 sums), which splits only over a long K.
int choose_ksplit(int64_t M, int64_t N, int64_t K, int64_t work_bytes, int* kgroups, bool int_sums);

// Rows at the end of an M x N product that run as a separate GEMM (0: none): when the 256 x 256
// tiles leave a last wave of whole tile rows that would occupy at most a quarter of the compute
// units (M = 4352 = 4096 + 256 tokens against N = 12288: 816 tiles on 256 units), those rows run
// on their own, on the tile and K split that choose_tile and choose_ksplit give them, so they take
// a fraction of a 256 tile's time.
int64_t tail_rows(int64_t M, int64_t N, int64_t K);

// Workspace bytes the split-K of an M x N x K product uses with the group-scale (int_sums false)
// or row-scale epilogue (0: none).
int64_t workspace_bytes(int64_t M, int64_t N, int64_t K, bool int_sums);

// Power-of-two factor by which a group GEMM's MFMA result exceeds the true partial, per
// activation layout and weight kind (see mq_gemm_wide.hip).
__host__ __device__ inline int group_shift(int act_mode, WKind wk) {
    if (act_mode == 1) return 4;
    if (act_mode == 2) return wk == WKind::I4Sym ? 8 : 4;
    return 0;
}

int launch_gemm(const GemmArgs& a, WKind wk, Epi epi, hipStream_t stream);
// whether launch_gemm runs these arguments' product on the wide kernel (it and the few-row one read atile)
bool gemm_runs_wide(const GemmArgs& a, WKind wk, Epi epi);

// M <= 4 rows, GroupScale / RowScale only (mq_gemv.hip).
int launch_gemv(const GemmArgs& a, WKind wk, Epi epi, hipStream_t stream);
// Whether a whole linear of these operands can hand its activation row to the GEMV (one row,
// K <= 4096, a scaled epilogue): the GEMV then rotates and quantizes the row in its prologue with
// the rotate+quantize kernel's arithmetic, in the same launch.
bool gemv_quantizes_row(const GemmArgs& a, WKind wk, Epi epi);

// Up to 128 rows that the GEMV does not take (M >= 5, or M * K > 131072), GroupScale / RowScale
// (mq_gemm_few.hip); whether launch_gemm runs these arguments' product there (it reads qa in rows or in
// 16-row tiles).
int launch_gemm_few(const GemmArgs& a, WKind wk, Epi epi, hipStream_t stream);
bool gemm_runs_few(const GemmArgs& a, WKind wk, Epi epi);

// 256 x 256-tile kernel for large M (mq_gemm_wide.hip).
int launch_gemm_wide(const GemmArgs& a, WKind wk, Epi epi, hipStream_t stream);

// --- paged key-value cache (mq_kv.hip); strides in elements
struct KvWriteArgs {
    const void* k;            // [T, H, D], strides k_token / k_head
    const void* v;
    int64_t k_token, k_head, v_token, v_head;
    int64_t T, H, D;
    void* kc;                 // [pages, H, page size, D], K and V alike
    void* vc;
    int64_t c_page, c_head, c_token;
    float* k_scale;           // [pages, H, page size] (int8 cache)
    float* v_scale;
    int64_t s_page, s_head, s_token;
    int64_t pages;
    int page_shift;
    int row_shift;            // log2 of the lanes that hold a row
    const int* table;         // [B, width]
    int64_t ld_table, B, width;
    const int* lens;
    const int* cu_q;          // [B + 1], or null: one token per sequence
};
int launch_kv_write(const KvWriteArgs& a, int dtype, bool i8, hipStream_t stream);

// Threads of a launch along x at most: the runtime counts them in 32 bits, and with more leaves workgroups out without an error.
// Calls of more rows than that go in several launches.
constexpr int64_t kMostThreads = int64_t(1) << 31;

// --- new tokens turned by their positions and written (mq_append.hip)
struct KvAppendArgs {
    KvWriteArgs w;
    const void* q;            // [T, Hq, D], strides q_token / q_head
    int64_t q_token, q_head;
    void* o;                  // [T, Hq, D], the turned queries
    int64_t o_token, o_head;
    int64_t Hq;
    const uint64_t* freq;     // [turn / 2], turns a position as 64-bit fractions
    int turn;                 // values of a head that are turned
    int interleaved;          // pairs are neighbours, else halves
    float size;               // what cosines and sines are multiplied by
    int64_t first;            // the first token of a launch
};
int launch_kv_append(const KvAppendArgs& a, int dtype, bool i8, hipStream_t stream);

struct KvTables {
    int* table;               // [rows, width]
    int64_t ld_table, rows, width;
    int* lens;                // [rows]
    int* refs;                // [pages]
    int64_t pages;
    int page_shift;
};
struct KvCopyTensor {
    void* base;
    int64_t layer_bytes, page_pitch, page_bytes;
};
struct KvCopyArgs {
    KvCopyTensor t[4];        // K, V and their scales
    int tensors;
    int64_t layers;
    const int* moves;         // pairs (from, to); from < 0: none
    int n;                    // moves, or the most there can be
    const int* count;         // device count of the moves (null: n)
    const int* place;         // compaction: new place of every page, applied to tb.table (null: none)
    KvTables tb;
};
int launch_kv_fork(const KvTables& tb, const KvCopyArgs& copies, const int* src, const int* dst, int n, int* work,
                   int* status, hipStream_t stream);
int launch_kv_grow(const KvTables& tb, const int* rows, const int* counts, int n, int* work, int* status,
                   hipStream_t stream);
int launch_kv_free(const KvTables& tb, const int* rows, int n, hipStream_t stream);
int launch_kv_compact(const KvTables& tb, const KvCopyArgs& copies, int* work, int* live, hipStream_t stream);

// --- attention over the paged cache (mq_attn_*.hip)
struct AttnArgs {
    const void* q;            // [T, Hq, D]
    int64_t q_token, q_head;
    void* o;                  // [T, Hq, D]
    int64_t o_token, o_head;
    int64_t T;
    int Hq, H, D;             // query heads, cache heads, head width
    const void* kc;           // [pages, H, page size, D], K and V alike
    const void* vc;
    int64_t c_page, c_head, c_token;
    const float* k_scale;     // int8 cache: [pages, H, page size]; else null
    const float* v_scale;
    int64_t s_page, s_head, s_token;
    int64_t pages;
    int page_shift;
    const int* table;         // [B, width]
    int64_t ld_table, B, width;
    const int* lens;
    const int* cu_q;          // [B + 1], or null: one token per sequence
    float scale;              // of the scores
    int64_t window;           // keys that a query sees, its own among them; 0: all
    int64_t sinks;            // first keys that stay visible behind the window
    int dtype;                // of q and o
    void* work;
    int64_t work_bytes;
    int* counters;            // zeros before and after a call
    // sequences that share beginnings (mq_attn_shared.hip), else null
    const int* plan;          // groups (mq_kv_shared)
    const int* start;         // [B], keys of a sequence that its group's part covers
    float* shared_out;        // [B, Hq, D], the part over those keys, unnormalised
    float* shared_stat;       // [B, Hq, 2], its maximum (base 2) and sum; sum -1: nothing seen
    float* shared_parts;      // of rows whose part is in pieces: those, [slots, shared_most, D], and their maxima and sums
    int* shared_rows;         // [B, Hq, 4], first slot, last piece (-1: not in pieces), row in them
    int shared_most;
};
int launch_attn_prompt(const AttnArgs& a, hipStream_t stream);
int launch_attn_decode(const AttnArgs& a, hipStream_t stream);
int64_t attn_decode_workspace_bytes(int Hq, int H, int D);
int64_t attn_decode_counters(int Hq, int H, int64_t B);
int64_t attn_prompt_workspace_bytes(int64_t T, int Hq, int H, int D, int64_t B);
int64_t attn_prompt_counters(int64_t T, int Hq, int H, int64_t B);
int launch_attn_shared(const AttnArgs& a, hipStream_t stream);
int64_t attn_shared_workspace_bytes(int Hq, int H, int D, int64_t B);
int64_t attn_shared_counters(int Hq, int H, int64_t B);
int launch_kv_shared(const int* table, int64_t ld_table, int64_t rows, int64_t width, const int* lens, int page_shift,
                     int least_kib, int* plan, hipStream_t stream);

// The groups of sequences that hold the same first pages, as int32: their number; the tokens that reading each group's
// once saves; the least of their bytes, in KiB, that is worth it (kNever: no number of them); log2 of the page size; start[b],
// the tokens of sequence b that its group shares (0: none); the groups' members behind each other; for each group the tokens
// shared, the sequence whose pages are read, its first member's place and their number; working space.
struct SharedPlan {
    static constexpr int kHead = 4, kGroup = 4, kNever = 0x7fffffff;
    static int64_t ints(int64_t B) { return kHead + 9 * B; }
    __host__ __device__ static int64_t start() { return kHead; }
    __host__ __device__ static int64_t members(int64_t B) { return kHead + B; }
    __host__ __device__ static int64_t groups(int64_t B) { return kHead + 2 * B; }
    __host__ __device__ static int64_t work(int64_t B) { return kHead + 4 * B; }
};

// --- 4-bit weights, floating activations (mq_w4a16.hip)
enum class W4Zero : int { Signed = 0, U4 = 1, Float = 2 };
struct W4A16Args {
    const void* x;            // [M, K] of type x_dtype
    int x_dtype;
    int64_t ldx;
    int hblock;
    const uint8_t* qw;        // [N, K / 2]
    int64_t ldw;
    const void* ws;           // [N, K / group] of type s_dtype
    int s_dtype;
    int64_t ldws;
    const void* wz;           // packed uint4 [N, ceil(K / group / 2)] or [N, K / group] of type z_dtype
    int z_dtype;
    int64_t ldwz;
    W4Zero zero;
    int group;
    const void* bias;
    int bias_dtype;
    void* y;
    int y_dtype;
    int64_t ldy;
    int64_t M, N, K;
};
int launch_w4a16(const W4A16Args& a, hipStream_t stream);


// --- norms (mq_norm.hip)
struct NormArgs {
    const void* x;            // [M, K] of type dtype
    int64_t ldx;
    const void* r;            // residual, or null
    int64_t ldr;
    const void* w;            // [K] of type w_dtype, or null
    int w_dtype;
    float eps;
    void* h;                  // x + r (with a residual)
    int64_t ldh;
    void* y;                  // [M, K] of type dtype, or int8 codes
    int64_t ldy;
    float* s;                 // [M], the codes' scales
    int dtype;
    int hblock;               // -1: floating output; 0: codes; 16, 64, 256: codes of rotated rows
    int64_t M, K;
};
int launch_norm(const NormArgs& a, hipStream_t stream);

// --- the next token of rows of logits (mq_sample.hip)
struct SampleArgs {
    const void* x;            // [rows, V] of type dtype, row stride ld
    int dtype;
    int64_t ld, rows, V;
    const float* u;           // [rows]
    const float *temperature, *top_p, *min_p;   // [rows], or null: the values below
    const int* top_k;
    float temperature1, top_p1, min_p1;
    int64_t top_k1;
    int64_t* token;           // [rows]
    void* work;
};
int launch_sample(const SampleArgs& a, hipStream_t stream);
int64_t sample_workspace_bytes(int64_t rows, int64_t V);

}  // namespace mq
