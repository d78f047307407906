// Root-mean-square norm to the rows' own type, and the entry points of all its forms (rms_norm.hpp).
#include "rms_norm.hpp"

namespace tsx {

int rms_norm_rows(const RmsNormParams &p, int type, hipStream_t stream) { return rms_norm_of<NORM_ROWS>(p, type, stream); }

namespace {

int check(const tsx_rms_norm *g, const char *what) {
    TSX_REQUIRE(g, "%s: null argument", what);
    TSX_REQUIRE(g->rows >= 0 && g->cols > 0 && g->cols <= 1 << 30, "%s: %lld rows of %d columns", what, (long long)g->rows, g->cols);
    TSX_REQUIRE(is_float_type(g->type), "%s: element type %d (fp32, fp16 or bf16)", what, g->type);
    TSX_REQUIRE(g->epsilon >= 0.f && g->epsilon < __builtin_inff(), "%s: epsilon %g", what, double(g->epsilon));
    TSX_REQUIRE(g->rows <= 1 || (g->x_stride >= g->cols && (!g->residual_dev || g->residual_stride >= g->cols) && (!g->sum_dev || g->sum_stride >= g->cols)),
                "%s: rows of %d columns overlap", what, g->cols);
    if (g->rows == 0) return 0;
    TSX_REQUIRE(g->x_dev, "%s: null pointer", what);
    TSX_REQUIRE(!g->residual_dev || g->sum_dev, "%s: a residual needs a place for the sum", what);
    const uintptr_t size = element_bytes(g->type);
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(g->x_dev) % size == 0 && reinterpret_cast<uintptr_t>(g->residual_dev) % size == 0 &&
                    reinterpret_cast<uintptr_t>(g->sum_dev) % size == 0 && reinterpret_cast<uintptr_t>(g->weight_dev) % 4 == 0,
                "%s: pointer is no multiple of its elements", what);
    return 0;
}

RmsNormParams params(const tsx_rms_norm *g, void *out, int64_t out_stride, void *scales, int64_t scales_stride) {
    return RmsNormParams{g->x_dev, g->residual_dev, g->sum_dev, g->weight_dev, out, scales, g->rows, g->x_stride, g->residual_stride, g->sum_stride,
                         out_stride, scales_stride, g->cols, 1.f / float(g->cols), g->epsilon};
}

}  // namespace
}  // namespace tsx

extern "C" {

int tsx_rms_norm_rows(const tsx_rms_norm *g, void *out_dev, int64_t out_stride, void *stream) {
    if (const int rc = tsx::check(g, "rms_norm")) return rc;
    TSX_REQUIRE(g->rows <= 1 || out_stride >= g->cols, "rms_norm: rows of %d columns overlap at stride %lld", g->cols, (long long)out_stride);
    if (g->rows == 0) return 0;
    TSX_REQUIRE(out_dev, "rms_norm: null pointer");
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(out_dev) % tsx::element_bytes(g->type) == 0, "rms_norm: pointer is no multiple of its elements");
    return tsx::rms_norm_rows(tsx::params(g, out_dev, out_stride, nullptr, 0), g->type, tsx::as_stream(stream));
}

int tsx_rms_norm_tokens(const tsx_rms_norm *g, int8_t *q_dev, float *scales_dev, void *stream) {
    if (const int rc = tsx::check(g, "rms_norm_tokens")) return rc;
    if (g->rows == 0) return 0;
    TSX_REQUIRE(q_dev && scales_dev, "rms_norm_tokens: null pointer");
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(scales_dev) % 4 == 0, "rms_norm_tokens: pointer is no multiple of its elements");
    return tsx::rms_norm_tokens(tsx::params(g, q_dev, g->cols, scales_dev, 0), g->type, tsx::as_stream(stream));
}

int tsx_rms_norm_mxfp4(const tsx_rms_norm *g, uint8_t *codes_dev, uint8_t *scales_dev, void *stream) {
    if (const int rc = tsx::check(g, "rms_norm_mxfp4")) return rc;
    if (g->rows == 0) return 0;
    TSX_REQUIRE(codes_dev && scales_dev, "rms_norm_mxfp4: null pointer");
    return tsx::rms_norm_mxfp4(tsx::params(g, codes_dev, (int64_t(g->cols) + 1) / 2, scales_dev, (int64_t(g->cols) + 31) / 32), g->type, tsx::as_stream(stream));
}

}  // extern "C"
