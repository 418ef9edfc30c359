// extern "C" entry points of token generation (declared in include/mq.h): argument validation, error
// reporting and dispatch of the paged cache's upkeep, the attention over it and the linears with 4-bit
// weights and floating-point activations. Nothing here allocates device memory.
#include "../../include/mq.h"

#include "mq_check.h"
#include "mq_internal.h"

namespace mq {
namespace {

constexpr int64_t kMost = int64_t(1) << 31;

int log2_of(int64_t v) {
    int s = 0;
    while ((int64_t(1) << s) < v) ++s;
    return s;
}

// A cache of one layer and the sequences' tables (the arguments that mq_kv_write and
// mq_paged_attention share).
int check_cache(const char* what, int dtype, int64_t T, int64_t H, int64_t D, const void* kc, const void* vc,
                int cache_dtype, int64_t c_page, int64_t c_head, int64_t c_token, const float* ks, const float* vs,
                int64_t s_page, int64_t s_head, int64_t s_token, int64_t pages, int page_size, const int32_t* table,
                int64_t ld_table, int64_t B, int64_t width, const int32_t* lens, const int32_t* cu_q) {
    MQ_REQUIRE(dtype == MQ_DT_BF16 || dtype == MQ_DT_F16, "%s: the tokens' type must be bf16 (%d) or fp16 (%d), got %d",
               what, MQ_DT_BF16, MQ_DT_F16, dtype);
    const bool i8 = cache_dtype == MQ_DT_I8;
    MQ_REQUIRE(i8 || cache_dtype == dtype, "%s: the cache must have the tokens' type (%d) or int8 (%d), got %d", what,
               dtype, MQ_DT_I8, cache_dtype);
    MQ_REQUIRE(T >= 0 && H > 0 && D > 0 && B >= 0 && width >= 0 && pages >= 0,
               "%s: bad shape T=%lld H=%lld D=%lld B=%lld width=%lld pages=%lld", what, (long long)T, (long long)H,
               (long long)D, (long long)B, (long long)width, (long long)pages);
    MQ_REQUIRE(D <= 256 && D % (i8 ? 16 : 8) == 0, "%s: the head width must be a multiple of %d and <= 256 (got %lld)",
               what, i8 ? 16 : 8, (long long)D);
    MQ_REQUIRE(T < kMost && H < kMost && B < kMost && pages < kMost && width < kMost, "%s: shape too large", what);
    MQ_REQUIRE(page_size > 0 && (page_size & (page_size - 1)) == 0, "%s: page_size must be a power of two (got %d)",
               what, page_size);
    MQ_REQUIRE(width <= (kMost >> 1) / page_size, "%s: the tables hold too many tokens", what);
    MQ_REQUIRE(pages * page_size < kMost, "%s: the cache holds too many tokens", what);
    MQ_REQUIRE(cu_q || T == B, "%s: without cu_q every sequence has one token (T=%lld, B=%lld)", what, (long long)T,
               (long long)B);
    if (T == 0 || B == 0) return MQ_OK;
    MQ_REQUIRE(lens && aligned(lens, 4) && aligned(cu_q, 4), "%s: lens must be non-null, lens and cu_q 4-byte aligned", what);
    MQ_REQUIRE(width == 0 || (table && aligned(table, 4) && ld_table >= width),
               "%s: page_table must be non-null and 4-byte aligned with ld_table >= width", what);
    if (pages == 0) return MQ_OK;
    const int64_t per16 = i8 ? 16 : 8;
    MQ_REQUIRE(kc && vc && aligned(kc, 16) && aligned(vc, 16) && c_page % per16 == 0 && c_head % per16 == 0 &&
                   c_token % per16 == 0,
               "%s: the caches need 16-byte aligned bases and strides that are multiples of 16 bytes", what);
    MQ_REQUIRE(c_token < (1 << 25), "%s: token strides must be below 2^25 elements", what);
    MQ_REQUIRE(c_page >= 0 && c_head >= 0 && c_token >= 0 && s_page >= 0 && s_head >= 0 && s_token >= 0,
               "%s: negative stride", what);
    MQ_REQUIRE(!i8 || (ks && vs && aligned(ks, 4) && aligned(vs, 4)), "%s: an int8 cache needs its scales", what);
    return MQ_OK;
}

}  // namespace
}  // namespace mq

using namespace mq;

extern "C" {

int mq_kv_write(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                int dtype, int64_t T, int64_t H, int64_t D, void* k_cache, void* v_cache, int cache_dtype,
                int64_t c_page, int64_t c_head, int64_t c_token, float* k_scale, float* v_scale, int64_t s_page,
                int64_t s_head, int64_t s_token, int64_t pages, int page_size, const int32_t* page_table,
                int64_t ld_table, int64_t B, int64_t width, const int32_t* lens, const int32_t* cu_q, void* stream) {
    clear_error();
    const int rc = check_cache("kv_write", dtype, T, H, D, k_cache, v_cache, cache_dtype, c_page, c_head, c_token,
                               k_scale, v_scale, s_page, s_head, s_token, pages, page_size, page_table, ld_table, B,
                               width, lens, cu_q);
    if (rc != MQ_OK || T == 0 || B == 0 || pages == 0 || width == 0) return rc;
    MQ_REQUIRE(k && v && aligned(k, 16) && aligned(v, 16) && k_token % 8 == 0 && k_head % 8 == 0 && v_token % 8 == 0 &&
                   v_head % 8 == 0,
               "kv_write: k and v need 16-byte aligned bases and rows that start at multiples of 16 bytes");
    MQ_REQUIRE(T * H < (int64_t(1) << 33), "kv_write: too many rows");
    KvWriteArgs a{};
    a.k = k; a.v = v; a.k_token = k_token; a.k_head = k_head; a.v_token = v_token; a.v_head = v_head;
    a.T = T; a.H = H; a.D = D; a.kc = k_cache; a.vc = v_cache; a.c_page = c_page; a.c_head = c_head; a.c_token = c_token;
    a.k_scale = k_scale; a.v_scale = v_scale; a.s_page = s_page; a.s_head = s_head; a.s_token = s_token;
    a.pages = pages; a.page_shift = log2_of(page_size); a.table = page_table; a.ld_table = ld_table; a.B = B;
    a.width = width; a.lens = lens; a.cu_q = cu_q;
    return launch_kv_write(a, dtype, cache_dtype == MQ_DT_I8, static_cast<hipStream_t>(stream));
}

int64_t mq_paged_attention_counters(int64_t T, int64_t Hq, int64_t H, int64_t B, int ragged) {
    if (T <= 0 || Hq <= 0 || H <= 0 || B <= 0 || Hq >= 65536 || H > Hq || T * Hq >= kMost || B >= kMost) return 0;
    if (ragged) return attn_prompt_counters(T, static_cast<int>(Hq), static_cast<int>(H), B);
    return attn_decode_counters(static_cast<int>(Hq), static_cast<int>(H), B);
}

int64_t mq_paged_attention_workspace_bytes(int64_t T, int64_t Hq, int64_t H, int64_t D, int64_t B, int ragged) {
    if (T <= 0 || Hq <= 0 || H <= 0 || D <= 0 || B <= 0 || Hq >= 65536 || H > Hq || D > 256 || T * Hq >= kMost || B >= kMost)
        return 0;
    if (ragged) return attn_prompt_workspace_bytes(T, static_cast<int>(Hq), static_cast<int>(H), static_cast<int>(D), B);
    return attn_decode_workspace_bytes(static_cast<int>(Hq), static_cast<int>(H), static_cast<int>(D));
}

int mq_paged_attention(const void* q, int64_t q_token, int64_t q_head, int dtype, int64_t T, int64_t Hq, int64_t H,
                       int64_t D, const void* k_cache, const void* v_cache, int cache_dtype, int64_t c_page,
                       int64_t c_head, int64_t c_token, const float* k_scale, const float* v_scale, int64_t s_page,
                       int64_t s_head, int64_t s_token, int64_t pages, int page_size, const int32_t* page_table,
                       int64_t ld_table, int64_t B, int64_t width, const int32_t* lens, const int32_t* cu_q, float scale,
                       int64_t window, int64_t sinks, void* out, int64_t out_token, int64_t out_head, void* workspace,
                       int64_t workspace_bytes, int32_t* counters, void* stream) {
    clear_error();
    const int rc = check_cache("paged_attention", dtype, T, H, D, k_cache, v_cache, cache_dtype, c_page, c_head, c_token,
                               k_scale, v_scale, s_page, s_head, s_token, pages, page_size, page_table, ld_table, B,
                               width, lens, cu_q);
    if (rc != MQ_OK) return rc;
    MQ_REQUIRE(Hq > 0 && Hq % H == 0 && Hq < 65536 && H > 0, "paged_attention: %lld query heads for %lld cache heads (a multiple, < 65536)",
               (long long)Hq, (long long)H);
    // the kernels count tiles of at least 64 keys for every sequence, cache head and 16 query heads in 32 bits
    MQ_REQUIRE((B + 1) * H * ((Hq / H + 15) / 16) < (int64_t(1) << 36) / (width * page_size + 256),
               "paged_attention: the tables hold too many tokens");
    MQ_REQUIRE(window >= 0 && sinks >= 0, "paged_attention: window and sinks must be >= 0 (got %lld, %lld)",
               (long long)window, (long long)sinks);
    if (T == 0) return MQ_OK;
    MQ_REQUIRE(q && out && aligned(q, 16) && aligned(out, 16) && q_token % 8 == 0 && q_head % 8 == 0 &&
                   out_token % 8 == 0 && out_head % 8 == 0,
               "paged_attention: q and out need 16-byte aligned bases and rows that start at multiples of 16 bytes");
    MQ_REQUIRE(T * Hq < kMost, "paged_attention: too many rows");
    MQ_REQUIRE(B > 0 || cu_q == nullptr, "paged_attention: tokens without a sequence (B=0)");
    const int64_t need = mq_paged_attention_workspace_bytes(T, Hq, H, D, B, cu_q != nullptr);
    MQ_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need),
               "paged_attention: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    MQ_REQUIRE(mq_paged_attention_counters(T, Hq, H, B, cu_q != nullptr) == 0 || (counters && aligned(counters, 4)),
               "paged_attention: needs its counters (zeros)");
    AttnArgs a{};
    a.counters = counters;
    a.q = q; a.q_token = q_token; a.q_head = q_head; a.o = out; a.o_token = out_token; a.o_head = out_head; a.T = T;
    a.Hq = static_cast<int>(Hq); a.H = static_cast<int>(H); a.D = static_cast<int>(D);
    a.kc = k_cache; a.vc = v_cache; a.c_page = c_page; a.c_head = c_head; a.c_token = c_token;
    if (cache_dtype == MQ_DT_I8) { a.k_scale = k_scale; a.v_scale = v_scale; }
    a.s_page = s_page; a.s_head = s_head; a.s_token = s_token; a.pages = pages; a.page_shift = log2_of(page_size);
    a.table = page_table; a.ld_table = ld_table; a.B = B; a.width = pages > 0 ? width : 0; a.lens = lens; a.cu_q = cu_q;
    a.scale = scale; a.window = window < kMost ? window : 0; a.sinks = sinks < kMost ? sinks : kMost - 1; a.dtype = dtype; a.work = workspace; a.work_bytes = workspace_bytes;
    return cu_q ? launch_attn_prompt(a, static_cast<hipStream_t>(stream)) : launch_attn_decode(a, static_cast<hipStream_t>(stream));
}

}  // extern "C"

namespace {

int check_tables(const char* what, const int32_t* table, int64_t ld_table, int64_t rows, int64_t width,
                 const int32_t* lens, const int32_t* refs, int64_t pages, int page_size, int64_t n) {
    MQ_REQUIRE(rows >= 0 && width >= 0 && pages >= 0 && n >= 0 && rows < kMost && width < kMost && pages < (kMost >> 1) &&
                   n < (int64_t(1) << 24),
               "%s: bad shape rows=%lld width=%lld pages=%lld n=%lld", what, (long long)rows, (long long)width,
               (long long)pages, (long long)n);
    MQ_REQUIRE(page_size > 0 && (page_size & (page_size - 1)) == 0, "%s: page_size must be a power of two (got %d)",
               what, page_size);
    MQ_REQUIRE(width < kMost / page_size, "%s: the tables hold too many tokens", what);
    MQ_REQUIRE(rows == 0 || width == 0 || (table && aligned(table, 4) && ld_table >= width),
               "%s: page_table must be non-null and 4-byte aligned with ld_table >= width", what);
    MQ_REQUIRE((rows == 0 || (lens && aligned(lens, 4))) && (pages == 0 || (refs && aligned(refs, 4))),
               "%s: lens and refs must be non-null and 4-byte aligned", what);
    return MQ_OK;
}

int check_work(const char* what, const void* workspace, int64_t workspace_bytes, int64_t pages, int64_t n) {
    const int64_t need = mq_kv_workspace_bytes(pages, n);
    MQ_REQUIRE(workspace && aligned(workspace, 16) && workspace_bytes >= need,
               "%s: needs a 16-byte aligned workspace of %lld bytes", what, (long long)need);
    return MQ_OK;
}

KvTables tables_of(int32_t* table, int64_t ld_table, int64_t rows, int64_t width, int32_t* lens, int32_t* refs,
                   int64_t pages, int page_size) {
    KvTables t{};
    t.table = table; t.ld_table = ld_table; t.rows = rows; t.width = width; t.lens = lens; t.refs = refs;
    t.pages = pages; t.page_shift = log2_of(page_size);
    return t;
}

// A fork or growth of no sequence: done, which *status says in the order of the stream.
int empty_plan(int32_t* status, void* stream) {
    MQ_REQUIRE(aligned(status, 4), "status must be 4-byte aligned");
    return status ? launch_kv_grow(KvTables{}, nullptr, nullptr, 0, nullptr, status, static_cast<hipStream_t>(stream)) : MQ_OK;
}

// The caches that a fork or a compaction copies pages of.
int copies_of(const char* what, void* k, void* v, int64_t layers, int64_t layer_bytes, int64_t pitch, int64_t bytes,
              float* ks, float* vs, int64_t s_layer, int64_t s_pitch, int64_t s_bytes, int64_t pages, KvCopyArgs* out) {
    KvCopyArgs c{};
    MQ_REQUIRE(layers >= 0 && layers < kMost, "%s: bad number of layers %lld", what, (long long)layers);
    c.layers = layers;
    if (pages > 0 && layers > 0) {
        MQ_REQUIRE(k && v && aligned(k, 16) && aligned(v, 16), "%s: the caches must be non-null and 16-byte aligned", what);
        MQ_REQUIRE(bytes > 0 && bytes % 4 == 0 && pitch >= bytes && pitch % 4 == 0 && layer_bytes >= 0 && layer_bytes % 4 == 0,
                   "%s: pages of %lld bytes, %lld apart: multiples of 4, not overlapping", what, (long long)bytes,
                   (long long)pitch);
        // the copies count blocks of at least 4 KB of a page's layers in 32 bits
        MQ_REQUIRE(bytes < kMost && 2 * layers * (bytes / 4096 + 1) < kMost && s_bytes <= bytes,
                   "%s: a page of %lld bytes in %lld layers is too large", what, (long long)bytes, (long long)layers);
        c.t[c.tensors++] = {k, layer_bytes, pitch, bytes};
        c.t[c.tensors++] = {v, layer_bytes, pitch, bytes};
        MQ_REQUIRE((ks == nullptr) == (vs == nullptr), "%s: scales for both caches or none", what);
        if (ks) {
            MQ_REQUIRE(aligned(ks, 4) && aligned(vs, 4) && s_bytes > 0 && s_bytes % 4 == 0 && s_pitch >= s_bytes &&
                           s_pitch % 4 == 0 && s_layer >= 0 && s_layer % 4 == 0,
                       "%s: scales of %lld bytes a page, %lld apart: multiples of 4, not overlapping", what,
                       (long long)s_bytes, (long long)s_pitch);
            c.t[c.tensors++] = {ks, s_layer, s_pitch, s_bytes};
            c.t[c.tensors++] = {vs, s_layer, s_pitch, s_bytes};
        }
    }
    *out = c;
    return MQ_OK;
}

}  // namespace

extern "C" {

int64_t mq_kv_workspace_bytes(int64_t pages, int64_t n) {
    if (pages < 0 || n < 0) return 0;
    return 4 * (2 * pages + 3 * n + 4);
}

int mq_kv_fork(void* k, void* v, int64_t layers, int64_t layer_bytes, int64_t page_pitch, int64_t page_bytes,
               float* k_scale, float* v_scale, int64_t s_layer_bytes, int64_t s_page_pitch, int64_t s_page_bytes,
               int32_t* page_table, int64_t ld_table, int64_t rows, int64_t width, int32_t* lens, int32_t* refs,
               int64_t pages, int page_size, const int32_t* src, const int32_t* dst, int64_t n, int32_t* status,
               void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    int rc = check_tables("kv_fork", page_table, ld_table, rows, width, lens, refs, pages, page_size, n);
    if (rc) return rc;
    KvCopyArgs c;
    rc = copies_of("kv_fork", k, v, layers, layer_bytes, page_pitch, page_bytes, k_scale, v_scale, s_layer_bytes,
                   s_page_pitch, s_page_bytes, pages, &c);
    if (rc) return rc;
    if (n == 0) return empty_plan(status, stream);
    MQ_REQUIRE(src && dst && aligned(src, 4) && aligned(dst, 4) && aligned(status, 4), "kv_fork: src and dst must be non-null and 4-byte aligned");
    rc = check_work("kv_fork", workspace, workspace_bytes, pages, n);
    if (rc) return rc;
    return launch_kv_fork(tables_of(page_table, ld_table, rows, width, lens, refs, pages, page_size), c, src, dst,
                          static_cast<int>(n), static_cast<int*>(workspace), status, static_cast<hipStream_t>(stream));
}

int mq_kv_grow(int32_t* page_table, int64_t ld_table, int64_t rows, int64_t width, int32_t* lens, int32_t* refs,
               int64_t pages, int page_size, const int32_t* seqs, const int32_t* counts, int64_t n, int32_t* status,
               void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    int rc = check_tables("kv_grow", page_table, ld_table, rows, width, lens, refs, pages, page_size, n);
    if (rc) return rc;
    if (n == 0) return empty_plan(status, stream);
    MQ_REQUIRE(seqs && counts && aligned(seqs, 4) && aligned(counts, 4) && aligned(status, 4),
               "kv_grow: the sequences and counts must be non-null and 4-byte aligned");
    rc = check_work("kv_grow", workspace, workspace_bytes, pages, n);
    if (rc) return rc;
    return launch_kv_grow(tables_of(page_table, ld_table, rows, width, lens, refs, pages, page_size), seqs, counts,
                          static_cast<int>(n), static_cast<int*>(workspace), status, static_cast<hipStream_t>(stream));
}

int mq_kv_free(int32_t* page_table, int64_t ld_table, int64_t rows, int64_t width, int32_t* lens, int32_t* refs,
               int64_t pages, const int32_t* seqs, int64_t n, void* stream) {
    clear_error();
    const int rc = check_tables("kv_free", page_table, ld_table, rows, width, lens, refs, pages, 1, n);
    if (rc || n == 0) return rc;
    MQ_REQUIRE(seqs && aligned(seqs, 4), "kv_free: the sequences must be non-null and 4-byte aligned");
    return launch_kv_free(tables_of(page_table, ld_table, rows, width, lens, refs, pages, 1), seqs, static_cast<int>(n),
                          static_cast<hipStream_t>(stream));
}

int mq_kv_compact(void* k, void* v, int64_t layers, int64_t layer_bytes, int64_t page_pitch, int64_t page_bytes,
                  float* k_scale, float* v_scale, int64_t s_layer_bytes, int64_t s_page_pitch, int64_t s_page_bytes,
                  int32_t* page_table, int64_t ld_table, int64_t rows, int64_t width, int32_t* refs, int64_t pages,
                  int32_t* live, void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    MQ_REQUIRE(rows == 0 || page_table, "kv_compact: page_table must be non-null");
    int rc = check_tables("kv_compact", page_table, ld_table, rows, width, page_table, refs, pages, 1, 0);
    if (rc) return rc;
    KvCopyArgs c;
    rc = copies_of("kv_compact", k, v, layers, layer_bytes, page_pitch, page_bytes, k_scale, v_scale, s_layer_bytes,
                   s_page_pitch, s_page_bytes, pages, &c);
    if (rc) return rc;
    MQ_REQUIRE(live && aligned(live, 4), "kv_compact: live must be non-null and 4-byte aligned");
    rc = check_work("kv_compact", workspace, workspace_bytes, pages, 0);
    if (rc) return rc;
    return launch_kv_compact(tables_of(page_table, ld_table, rows, width, nullptr, refs, pages, 1), c,
                             static_cast<int*>(workspace), live, static_cast<hipStream_t>(stream));
}

int mq_linear_w4a16(const void* x, int x_dtype, int64_t ldx, int hblock, const uint8_t* qw, int64_t ldw, const void* ws,
                    int s_dtype, int64_t ldws, const void* wz, int zero, int z_dtype, int64_t ldwz, int group,
                    const void* bias, int bias_dtype, void* y, int y_dtype, int64_t ldy, int64_t M, int64_t N, int64_t K,
                    void* stream) {
    clear_error();
    auto float_type = [](int dt) { return dt >= MQ_DT_BF16 && dt <= MQ_DT_F32; };
    MQ_REQUIRE(float_type(x_dtype), "linear_w4a16: unknown input type %d", x_dtype);
    MQ_REQUIRE(float_type(s_dtype), "linear_w4a16: unknown scale type %d", s_dtype);
    MQ_REQUIRE(float_type(y_dtype), "linear_w4a16: unknown output type %d", y_dtype);
    MQ_REQUIRE(zero >= MQ_W4Z_SIGNED && zero <= MQ_W4Z_FLOAT, "linear_w4a16: unknown zero-point rule %d", zero);
    MQ_REQUIRE(zero != MQ_W4Z_FLOAT || float_type(z_dtype), "linear_w4a16: unknown zero-point type %d", z_dtype);
    MQ_REQUIRE(!bias || float_type(bias_dtype), "linear_w4a16: unknown bias type %d", bias_dtype);
    MQ_REQUIRE(group == 32 || group == 64 || group == 128, "linear_w4a16: group size must be 32, 64 or 128 (got %d)", group);
    MQ_REQUIRE(hblock == 0 || hblock == 16 || hblock == 64 || hblock == 256,
               "linear_w4a16: convrot group size must be 16, 64 or 256 (got %d)", hblock);
    MQ_REQUIRE(M >= 0 && N >= 0 && K > 0 && M < kMost && N < kMost - 256, "linear_w4a16: bad shape M=%lld N=%lld K=%lld",
               (long long)M, (long long)N, (long long)K);
    MQ_REQUIRE(K % group == 0, "linear_w4a16: K=%lld is not a multiple of the group size %d", (long long)K, group);
    MQ_REQUIRE(hblock == 0 || K % hblock == 0, "linear_w4a16: K=%lld is not a multiple of the convrot group size %d",
               (long long)K, hblock);
    if (K > 32768) {
        set_error("linear_w4a16: K=%lld exceeds 32768", (long long)K);
        return MQ_EUNSUPPORTED;
    }
    if (M == 0 || N == 0) return MQ_OK;
    MQ_REQUIRE(x && qw && ws && y && (zero == MQ_W4Z_SIGNED || wz), "linear_w4a16: null operand");
    const int64_t per16 = x_dtype == MQ_DT_F32 ? 4 : 8;
    MQ_REQUIRE(ldx >= K && ldx % per16 == 0 && aligned(x, 16),
               "linear_w4a16: x needs ldx >= K, ldx %% %lld == 0 and a 16-byte aligned base", (long long)per16);
    MQ_REQUIRE(ldw >= K / 2 && ldw % 16 == 0 && aligned(qw, 16),
               "linear_w4a16: qw needs ldw >= K/2 bytes, ldw %% 16 == 0 and a 16-byte aligned base");
    MQ_REQUIRE(ldw < (1 << 25) && ldws < (1 << 25) && ldwz < (1 << 25), "linear_w4a16: row strides must be below 2^25");
    MQ_REQUIRE(ldws >= K / group && aligned(ws, dtype_bytes(s_dtype)), "linear_w4a16: ws needs ldws >= K/group and an aligned base");
    MQ_REQUIRE(zero != MQ_W4Z_U4 || ldwz >= (K / group + 1) / 2, "linear_w4a16: ldwz < ceil(K/group/2)");
    MQ_REQUIRE(zero != MQ_W4Z_FLOAT || (ldwz >= K / group && aligned(wz, dtype_bytes(z_dtype))),
               "linear_w4a16: wz needs ldwz >= K/group and an aligned base");
    MQ_REQUIRE(aligned(y, dtype_bytes(y_dtype)) && ldy >= N && (!bias || aligned(bias, dtype_bytes(bias_dtype))),
               "linear_w4a16: y and bias must be aligned to their element size, ldy >= N");
    W4A16Args a{};
    a.x = x; a.x_dtype = x_dtype; a.ldx = ldx; a.hblock = hblock; a.qw = qw; a.ldw = ldw; a.ws = ws; a.s_dtype = s_dtype;
    a.ldws = ldws; a.wz = zero == MQ_W4Z_SIGNED ? nullptr : wz; a.z_dtype = z_dtype; a.ldwz = ldwz;
    a.zero = static_cast<W4Zero>(zero); a.group = group; a.bias = bias; a.bias_dtype = bias_dtype; a.y = y;
    a.y_dtype = y_dtype; a.ldy = ldy; a.M = M; a.N = N; a.K = K;
    return launch_w4a16(a, static_cast<hipStream_t>(stream));
}

}  // extern "C"
