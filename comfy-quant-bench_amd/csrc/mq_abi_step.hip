// extern "C" entry points of what a step of token generation does between its linears and behind them (declared in
// include/mq.h): argument validation, error reporting and dispatch of the norms and of the choice of the next token.
#include "../../include/mq.h"

#include "mq_check.h"
#include "mq_internal.h"

namespace mq {
namespace {

constexpr int64_t kMost = int64_t(1) << 31;

bool float_type(int dt) { return dt >= MQ_DT_BF16 && dt <= MQ_DT_F32; }

// What both norms ask of their input; out_ld: the output's row stride in elements of out_bytes.
int check_norm(const char* what, const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
               int w_dtype, const void* h, int64_t ldh, const void* out, int64_t ldo, int out_bytes, int64_t M, int64_t K) {
    MQ_REQUIRE(float_type(dtype), "%s: unknown input type %d", what, dtype);
    MQ_REQUIRE(!weight || float_type(w_dtype), "%s: unknown weight type %d", what, w_dtype);
    MQ_REQUIRE(M >= 0 && K > 0 && M < kMost, "%s: bad shape M=%lld K=%lld", what, (long long)M, (long long)K);
    if (K > 32768) {
        set_error("%s: K=%lld exceeds 32768", what, (long long)K);
        return MQ_EUNSUPPORTED;
    }
    if (M == 0) return MQ_OK;
    MQ_REQUIRE(x && out && (!residual || h), "%s: null operand", what);
    MQ_REQUIRE((M == 1 || (ldx >= K && ldo >= K)) && (!residual || M == 1 || (ldr >= K && ldh >= K)),
               "%s: row strides must be at least K", what);
    const int e = dtype_bytes(dtype);
    MQ_REQUIRE(aligned(x, e) && aligned(residual, e) && aligned(h, e) && aligned(out, out_bytes) &&
                   (!weight || aligned(weight, dtype_bytes(w_dtype))),
               "%s: operands must be aligned to their element size", what);
    return MQ_OK;
}

NormArgs norm_args(const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int w_dtype,
                   float eps, void* h, int64_t ldh, void* y, int64_t ldy, int64_t M, int64_t K) {
    NormArgs a{};
    a.x = x; a.ldx = ldx; a.r = residual; a.ldr = ldr; a.w = weight; a.w_dtype = w_dtype; a.eps = eps; a.h = h; a.ldh = ldh;
    a.y = y; a.ldy = ldy; a.dtype = dtype; a.M = M; a.K = K;
    return a;
}

}  // namespace
}  // namespace mq

using namespace mq;

extern "C" {

int mq_rms_norm(const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr, const void* weight, int w_dtype,
                float eps, void* h, int64_t ldh, void* y, int64_t ldy, int64_t M, int64_t K, void* stream) {
    clear_error();
    const int rc = check_norm("rms_norm", x, dtype, ldx, residual, ldr, weight, w_dtype, h, ldh, y, ldy, dtype_bytes(dtype), M, K);
    if (rc != MQ_OK || M == 0) return rc;
    NormArgs a = norm_args(x, dtype, ldx, residual, ldr, weight, w_dtype, eps, h, ldh, y, ldy, M, K);
    a.hblock = -1;
    return launch_norm(a, static_cast<hipStream_t>(stream));
}

int mq_rms_norm_quant(const void* x, int dtype, int64_t ldx, const void* residual, int64_t ldr, const void* weight,
                      int w_dtype, float eps, int hblock, void* h, int64_t ldh, int8_t* q, int64_t ldq, float* scale, int64_t M,
                      int64_t K, void* stream) {
    clear_error();
    MQ_REQUIRE(hblock == 0 || hblock == 16 || hblock == 64 || hblock == 256,
               "rms_norm_quant: convrot group size must be 16, 64 or 256 (got %d)", hblock);
    const int rc = check_norm("rms_norm_quant", x, dtype, ldx, residual, ldr, weight, w_dtype, h, ldh, q, ldq, 1, M, K);
    if (rc != MQ_OK) return rc;
    MQ_REQUIRE(hblock == 0 || K % hblock == 0, "rms_norm_quant: K=%lld is not a multiple of the convrot group size %d",
               (long long)K, hblock);
    if (M == 0) return MQ_OK;
    MQ_REQUIRE(scale && aligned(scale, 4), "rms_norm_quant: scale must be non-null and 4-byte aligned");
    NormArgs a = norm_args(x, dtype, ldx, residual, ldr, weight, w_dtype, eps, h, ldh, q, ldq, M, K);
    a.hblock = hblock;
    a.s = scale;
    return launch_norm(a, static_cast<hipStream_t>(stream));
}

int64_t mq_sample_workspace_bytes(int64_t rows, int64_t V) {
    return rows <= 0 || V <= 0 || rows >= kMost || V > (int64_t(1) << 24) ? 0 : sample_workspace_bytes(rows, V);
}

int mq_sample(const void* logits, int dtype, int64_t ld, int64_t rows, int64_t V, const float* u, const float* temperature,
              float temperature_all, const int32_t* top_k, int64_t top_k_all, const float* top_p, float top_p_all,
              const float* min_p, float min_p_all, int64_t* token, void* workspace, int64_t workspace_bytes, void* stream) {
    clear_error();
    MQ_REQUIRE(float_type(dtype), "sample: unknown type %d", dtype);
    MQ_REQUIRE(rows >= 0 && rows < kMost && V > 0, "sample: bad shape rows=%lld V=%lld", (long long)rows, (long long)V);
    if (V > (int64_t(1) << 24)) {
        set_error("sample: V=%lld exceeds 2^24", (long long)V);
        return MQ_EUNSUPPORTED;
    }
    if (rows == 0) return MQ_OK;
    MQ_REQUIRE(logits && u && token, "sample: null operand");
    MQ_REQUIRE(rows == 1 || ld >= V, "sample: the row stride must be at least V");
    MQ_REQUIRE(aligned(logits, dtype_bytes(dtype)) && aligned(u, 4) && aligned(temperature, 4) && aligned(top_k, 4) &&
                   aligned(top_p, 4) && aligned(min_p, 4) && aligned(token, 8),
               "sample: operands must be aligned to their element size");
    const int64_t need = mq_sample_workspace_bytes(rows, V);
    MQ_REQUIRE(need == 0 || (workspace && aligned(workspace, 16) && workspace_bytes >= need),
               "sample: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
    SampleArgs a{};
    a.work = workspace;
    a.x = logits; a.dtype = dtype; a.ld = ld; a.rows = rows; a.V = V; a.u = u; a.temperature = temperature; a.top_p = top_p;
    a.min_p = min_p; a.top_k = top_k; a.temperature1 = temperature_all; a.top_p1 = top_p_all; a.min_p1 = min_p_all;
    a.top_k1 = top_k_all; a.token = token;
    return launch_sample(a, static_cast<hipStream_t>(stream));
}

}  // extern "C"
