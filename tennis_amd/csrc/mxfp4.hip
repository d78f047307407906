// Rows of fp32, fp16 or bf16 values to MXFP4 and back, and int8 tokens to values.
//
// Bound: HBM, the values' bytes and 17 / 32 of a byte each.  A lane holds pieces of eight values; four neighbouring lanes hold a block, find
// its largest magnitude by two lane exchanges, and each leaves four bytes of codes.  Pieces of all rows are numbered through, so that short
// rows and long ones fill the card alike; nothing but the four lanes of a block has to meet.  One piece a lane: two, four and eight are no faster (bf16
// to codes, us: 8192 x 8192 30.1, 30.0, 31.3, 32.9; 4096 x 4096 8.1, 8.3, 8.8, 9.0).  8192 x 8192 is 5.6 TB/s, a copy of 1 GiB 5.1.
#include <algorithm>

#include "mxfp4.hpp"

namespace tsx {
namespace {

constexpr int PIECE = 8, THREADS = 256;

struct ToMxParams {
    const void *x;
    MxRows to;
    Divider pieces;               // of a row, a multiple of LANES
    int64_t x_stride;
    unsigned total;               // pieces of all rows
    int cols, cols_out;
};

// TAILS: rows end inside a piece, or pieces behind their ends are written; LANES: of a block, one where rows are one piece
template <int TYPE, bool TAILS, int LANES>
__global__ __launch_bounds__(THREADS) void quantize_mxfp4_kernel(ToMxParams p) {
    constexpr int SIZE = TYPE == TSX_TYPE_F32 ? 4 : 2;
    typedef Run<TYPE, PIECE> Values;
    const unsigned id = blockIdx.x * THREADS + threadIdx.x, at = min(id, p.total - 1), r = p.pieces.quotient(at);      // a block's lanes agree on whether they are there
    const int64_t row = r;
    const int piece = int(at - r * p.pieces.d);
    const char *const x = static_cast<const char *>(p.x) + row * p.x_stride * SIZE;
    Values v;
    if (!TAILS) {
        v.load(x + int64_t(piece) * (PIECE * SIZE));
    } else if (p.cols >= PIECE) {      // uniform
        load_piece<TYPE>(v, x, piece * PIECE, p.cols);
        settle_piece<TYPE>(v, piece * PIECE, p.cols);
    } else {
        v.clear();
        if (piece == 0) v.load_some(x, p.cols);
    }
    const unsigned top = over_lanes(v.top(0), lg_of(LANES), [](unsigned a, unsigned b) { return Values::template larger<TYPE>(a, b); });
    const unsigned scale = mx_scale(top_value<TYPE>(top)), codes = mx_codes<TYPE>(v, scale);
    if (id >= p.total) return;
    const int left = p.cols_out - piece * PIECE;
    if (!TAILS || left > 0) store_codes(p.to.codes + row * p.to.codes_stride + int64_t(piece) * (PIECE / 2), codes, TAILS ? left : PIECE);
    const int block = piece / 4;
    if (piece % LANES == 0) p.to.scales[row * p.to.scale_row + (block >> 2) * p.to.scale_group + (block & 3)] = uint8_t(scale);
}

struct FromParams {
    const uint8_t *codes, *scales;       // int8 tokens: q, and fp32 scales
    void *out;
    Divider pieces;
    int64_t codes_stride, scales_stride, out_stride;
    unsigned total;
    int cols;
};

// MX: MXFP4 rows, otherwise int8 tokens
template <int TYPE, bool MX>
__global__ __launch_bounds__(THREADS) void dequantize_kernel(FromParams p) {
    constexpr int SIZE = TYPE == TSX_TYPE_F32 ? 4 : 2, BYTES = MX ? PIECE / 2 : PIECE;
    const unsigned id = blockIdx.x * THREADS + threadIdx.x;
    if (id >= p.total) return;
    const unsigned r = p.pieces.quotient(id);
    const int64_t row = r;
    const int piece = int(id - r * p.pieces.d);
    const uint8_t *const codes = p.codes + row * p.codes_stride + int64_t(piece) * BYTES;
    const int bytes = (MX ? (p.cols + 1) / 2 : p.cols) - piece * BYTES;
    unsigned scale;
    if constexpr (MX) scale = p.scales[row * p.scales_stride + piece / 4];
    else scale = reinterpret_cast<const unsigned *>(p.scales)[row];
    v2u word = {0, 0};
    if (bytes >= BYTES) {
        if constexpr (MX) word[0] = *reinterpret_cast<const u_any *>(codes);
        else word = *reinterpret_cast<const v2u_any *>(codes);
    } else {
        static_for<0, BYTES - 1>([&](auto bc) {
            constexpr int b = decltype(bc)::value;
            if (b < bytes) word[b / 4] |= unsigned(codes[b]) << (8 * (b % 4));
        });
    }
    Run<TYPE, PIECE> v;
    if constexpr (MX) {
        v = mx_values<TYPE>(word[0], scale);
    } else {
        float f[PIECE];
        static_for<0, PIECE>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            unsigned product = __builtin_bit_cast(unsigned, __fmul_rn(float(int(word[e / 4] << (24 - 8 * (e % 4))) >> 24), __builtin_bit_cast(float, scale)));
            if constexpr (TYPE == TSX_TYPE_F16) renew(product);      // else the product and its conversion become one instruction with one rounding
            f[e] = __builtin_bit_cast(float, product);
        });
        v.set(f);
    }
    char *const out = static_cast<char *>(p.out) + (row * p.out_stride + int64_t(piece) * PIECE) * SIZE;
    const int left = p.cols - piece * PIECE;
    if (left >= PIECE) v.store(out);
    else v.store_some(out, left);
}

// Pieces are counted in 31 bits: rows in runs of as many as that holds.  launch(first row, rows)
template <class F>
int in_runs(int64_t rows, int64_t pieces, F &&launch) {
    const int64_t most = ((int64_t(1) << 31) - 1) / pieces;
    for (int64_t at = 0; at < rows; at += most)
        if (const int rc = launch(at, std::min(most, rows - at))) return rc;
    return 0;
}

template <int TYPE>
int to_mx(int64_t rows, int cols, int cols_out, const void *x, int64_t x_stride, const MxRows &to, hipStream_t stream) {
    const bool alone = cols_out <= PIECE;      // 16.8 million rows of one bf16 value 85 us, four lanes each 190
    const int64_t pieces = alone ? 1 : ceil_div(cols_out, MX_BLOCK) * (MX_BLOCK / PIECE);
    return in_runs(rows, pieces, [&](int64_t at, int64_t count) {
        const int64_t total = count * pieces;
        MxRows part = to;
        part.codes += at * to.codes_stride;
        part.scales += at * to.scale_row;
        const ToMxParams p{static_cast<const char *>(x) + at * x_stride * int64_t(element_bytes(TYPE)), part, Divider(pieces), x_stride, unsigned(total), cols, cols_out};
        const bool tails = cols % MX_BLOCK != 0 || cols_out != cols;
        hipLaunchKernelGGL((alone ? quantize_mxfp4_kernel<TYPE, true, 1> : tails ? quantize_mxfp4_kernel<TYPE, true, 4> : quantize_mxfp4_kernel<TYPE, false, 4>), dim3(unsigned(ceil_div(total, THREADS))), dim3(THREADS), 0, stream, p);
        TSX_LAUNCH_CHECK("quantize_mxfp4_kernel");
        return 0;
    });
}

template <int TYPE, bool MX>
int from(int64_t rows, int cols, const void *codes, int64_t codes_stride, const void *scales, int64_t scales_stride, void *out, int64_t out_stride,
         hipStream_t stream) {
    const int64_t pieces = ceil_div(cols, PIECE);
    return in_runs(rows, pieces, [&](int64_t at, int64_t count) {
        const int64_t total = count * pieces;
        const FromParams p{static_cast<const uint8_t *>(codes) + at * codes_stride, static_cast<const uint8_t *>(scales) + at * (MX ? scales_stride : 4),
                           static_cast<char *>(out) + at * out_stride * int64_t(element_bytes(TYPE)), Divider(pieces), codes_stride, scales_stride, out_stride,
                           unsigned(total), cols};
        hipLaunchKernelGGL((dequantize_kernel<TYPE, MX>), dim3(unsigned(ceil_div(total, THREADS))), dim3(THREADS), 0, stream, p);
        TSX_LAUNCH_CHECK("dequantize_kernel");
        return 0;
    });
}

template <bool MX, class... A>
int from_type(int type, A... a) {
    return type == TSX_TYPE_F32 ? from<TSX_TYPE_F32, MX>(a...) : type == TSX_TYPE_F16 ? from<TSX_TYPE_F16, MX>(a...) : from<TSX_TYPE_BF16, MX>(a...);
}

bool is_multiple(const void *at, size_t bytes) { return reinterpret_cast<uintptr_t>(at) % bytes == 0; }

}  // namespace

int quantize_mxfp4_rows(int64_t rows, int cols, int cols_out, const void *x, int type, int64_t x_stride, const MxRows &to, hipStream_t stream) {
    if (rows == 0) return 0;
    return type == TSX_TYPE_F32   ? to_mx<TSX_TYPE_F32>(rows, cols, cols_out, x, x_stride, to, stream)
           : type == TSX_TYPE_F16 ? to_mx<TSX_TYPE_F16>(rows, cols, cols_out, x, x_stride, to, stream)
                                  : to_mx<TSX_TYPE_BF16>(rows, cols, cols_out, x, x_stride, to, stream);
}

}  // namespace tsx

extern "C" {

int tsx_quantize_mxfp4(int64_t rows, int32_t cols, const void *x_dev, int32_t x_type, int64_t x_stride, uint8_t *codes_dev, int64_t codes_stride,
                       uint8_t *scales_dev, int64_t scales_stride, void *stream) {
    TSX_REQUIRE(rows >= 0 && cols > 0 && cols <= 1 << 30, "quantize_mxfp4: %lld rows of %d columns", (long long)rows, cols);
    TSX_REQUIRE(tsx::is_float_type(x_type), "quantize_mxfp4: element type %d (fp32, fp16 or bf16)", x_type);
    TSX_REQUIRE(rows <= 1 || (x_stride >= cols && codes_stride >= (cols + 1) / 2 && scales_stride >= (cols + 31) / 32),
                "quantize_mxfp4: rows of %d columns overlap at strides %lld, %lld and %lld", cols, (long long)x_stride, (long long)codes_stride, (long long)scales_stride);
    TSX_REQUIRE(rows == 0 || (x_dev && codes_dev && scales_dev), "quantize_mxfp4: null pointer");
    TSX_REQUIRE(tsx::is_multiple(x_dev, tsx::element_bytes(x_type)), "quantize_mxfp4: pointer is no multiple of its elements");
    return tsx::quantize_mxfp4_rows(rows, cols, cols, x_dev, x_type, x_stride, tsx::MxRows{codes_dev, scales_dev, codes_stride, scales_stride, 4}, tsx::as_stream(stream));
}

int tsx_dequantize_mxfp4(int64_t rows, int32_t cols, const uint8_t *codes_dev, int64_t codes_stride, const uint8_t *scales_dev, int64_t scales_stride,
                         void *out_dev, int32_t out_type, int64_t out_stride, void *stream) {
    TSX_REQUIRE(rows >= 0 && cols > 0 && cols <= 1 << 30, "dequantize_mxfp4: %lld rows of %d columns", (long long)rows, cols);
    TSX_REQUIRE(tsx::is_float_type(out_type), "dequantize_mxfp4: element type %d (fp32, fp16 or bf16)", out_type);
    TSX_REQUIRE(rows <= 1 || (out_stride >= cols && codes_stride >= (cols + 1) / 2 && scales_stride >= (cols + 31) / 32),
                "dequantize_mxfp4: rows of %d columns overlap at strides %lld, %lld and %lld", cols, (long long)codes_stride, (long long)scales_stride, (long long)out_stride);
    TSX_REQUIRE(rows == 0 || (codes_dev && scales_dev && out_dev), "dequantize_mxfp4: null pointer");
    TSX_REQUIRE(tsx::is_multiple(out_dev, tsx::element_bytes(out_type)), "dequantize_mxfp4: pointer is no multiple of its elements");
    return tsx::from_type<true>(out_type, rows, cols, codes_dev, codes_stride, scales_dev, scales_stride, out_dev, out_stride, tsx::as_stream(stream));
}

int tsx_dequantize_tokens(int64_t rows, int32_t cols, const int8_t *q_dev, int64_t q_stride, const float *scales_dev, void *out_dev, int32_t out_type,
                          int64_t out_stride, void *stream) {
    TSX_REQUIRE(rows >= 0 && cols > 0 && cols <= 1 << 30, "dequantize_tokens: %lld rows of %d columns", (long long)rows, cols);
    TSX_REQUIRE(tsx::is_float_type(out_type), "dequantize_tokens: element type %d (fp32, fp16 or bf16)", out_type);
    TSX_REQUIRE(rows <= 1 || (out_stride >= cols && q_stride >= cols), "dequantize_tokens: rows of %d columns overlap at strides %lld and %lld", cols,
                (long long)q_stride, (long long)out_stride);
    TSX_REQUIRE(rows == 0 || (q_dev && scales_dev && out_dev), "dequantize_tokens: null pointer");
    TSX_REQUIRE(tsx::is_multiple(out_dev, tsx::element_bytes(out_type)) && tsx::is_multiple(scales_dev, 4), "dequantize_tokens: pointer is no multiple of its elements");
    return tsx::from_type<false>(out_type, rows, cols, q_dev, q_stride, scales_dev, int64_t(0), out_dev, out_stride, tsx::as_stream(stream));
}

}  // extern "C"
