// Rows of fp32, fp16 or bf16 values to int8, each by its own largest magnitude.
//
// Bound: HBM, element size + 1 bytes a value: 8192 rows of 4096 bf16 19 us (5.3 TB/s, what a copy of that size takes), 4096 of them, which
// the caches hold, 16 us for 8192 values each (6 TB/s), 4 million rows of 8 19 us; one row of 4096 2 us in the kernel, the launch.  A row is read once: its values stay in registers, eight to a piece, while the
// threads that share it find its largest magnitude, and leave as eight bytes a piece.  That maximum is one of the values, whatever
// the order it is looked for in, and the rest is rounded as TokenScale says: results are the same on every path.
#include "tokens_i8.hpp"

namespace tsx {
namespace {

constexpr int PIECE = 8;

struct TokenParams {
    const void *x;
    int8_t *q;
    float *scales;
    int64_t rows, x_stride, q_stride;
    int cols, cols_out;       // columns from cols on, up to cols_out, become zeros
};

// T threads share a row and hold P pieces of it each; HELD: that is all of it, otherwise the row is read in turns, twice.
template <int TYPE, int T, int P, bool HELD>
__global__ __launch_bounds__(T < 256 ? 256 : T) void quantize_tokens_kernel(TokenParams p) {
    constexpr int THREADS = T < 256 ? 256 : T, ROWS = THREADS / T, SIZE = TYPE == TSX_TYPE_F32 ? 4 : 2;
    typedef Run<TYPE, PIECE> Values;
    __shared__ unsigned tops[T > 64 ? T / 64 : 1];
    const int tid = threadIdx.x, t = tid % T;
    const int pieces = (p.cols + PIECE - 1) / PIECE, pieces_out = (p.cols_out + PIECE - 1) / PIECE;
    for (int64_t row0 = int64_t(blockIdx.x) * ROWS; row0 < p.rows; row0 += int64_t(gridDim.x) * ROWS) {
        const int64_t row = row0 + tid / T;
        const bool there = row < p.rows;      // a row's threads agree; only T <= 64 has rows beyond the last one
        const char *x = static_cast<const char *>(p.x) + (there ? row : p.rows - 1) * p.x_stride * SIZE;
        Values v[P];
        unsigned top = 0;
        // All requests at once, none behind a branch, where it would be waited for: what lies behind the last whole piece is that piece
        // again, and then zeros, or the values that are left there.
        const int whole = p.cols / PIECE;
        auto fetch = [&](int first) __attribute__((always_inline)) {
            if (whole)       // uniform
                static_for<0, P>([&](auto ic) { v[decltype(ic)::value].load(x + int64_t(min(first + t + decltype(ic)::value * T, whole - 1)) * (PIECE * SIZE)); });
            Values last;
            last.clear();
            if (whole != pieces) last.load_some(x + int64_t(whole) * (PIECE * SIZE), p.cols - whole * PIECE);       // uniform
            static_for<0, P>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int piece = first + t + i * T;
                if (piece >= whole) v[i].clear();
                if (piece == whole) v[i] = last;
            });
        };
        const int turns = HELD ? 1 : (pieces_out + T * P - 1) / (T * P);
        for (int turn = 0; turn < turns; ++turn) {
            fetch(turn * T * P);
            static_for<0, P>([&](auto ic) { top = v[decltype(ic)::value].top(top); });
        }
        top = over_lanes(top, lg_of(T < 64 ? T : 64), [](unsigned a, unsigned b) { return Values::template larger<TYPE>(a, b); });
        if constexpr (T > 64) {
            if (tid % 64 == 0) tops[tid / 64] = top;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < T / 64; ++w) top = Values::template larger<TYPE>(top, tops[w]);
            __syncthreads();      // the next row writes them
        }
        const TokenScale s(top_value<TYPE>(top));
        if (there && t == 0) p.scales[row] = s.scale;
        int8_t *const q = p.q + (there ? row : 0) * p.q_stride;
        for (int turn = 0; turn < turns; ++turn) {
            if (!HELD) fetch(turn * T * P);
            static_for<0, P>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int piece = turn * T * P + t + i * T;
                if (piece >= pieces_out || !there) return;
                unsigned b[PIECE];
                static_for<0, PIECE>([&](auto ec) { constexpr int e = decltype(ec)::value; b[e] = s.bits(__fmul_rn(v[i].template get<e>(), s.lift)); });
                v2u out = {low_bytes(b[0], b[1], b[2], b[3]), low_bytes(b[4], b[5], b[6], b[7])};
                if (s.reciprocal == 0.f) out = v2u{0, 0};       // infinities times 0 among them
                int8_t *const at = q + int64_t(piece) * PIECE;
                if ((piece + 1) * PIECE <= p.cols_out) {
                    *reinterpret_cast<v2u_any *>(at) = out;
                } else {
                    static_for<0, PIECE>([&](auto ec) {
                        constexpr int e = decltype(ec)::value;
                        if (piece * PIECE + e < p.cols_out) at[e] = int8_t(out[e / 4] >> (8 * (e % 4)));
                    });
                }
            });
        }
    }
}

template <int TYPE, int T, int P, bool HELD>
int launch(const TokenParams &p, hipStream_t stream) {
    constexpr int THREADS = T < 256 ? 256 : T, ROWS = THREADS / T;
    const int64_t blocks = ceil_div(p.rows, ROWS), most = int64_t(1) << 20;       // beyond that a workgroup takes several rows
    hipLaunchKernelGGL((quantize_tokens_kernel<TYPE, T, P, HELD>), dim3(unsigned(blocks < most ? blocks : most)), dim3(THREADS), 0, stream, p);
    TSX_LAUNCH_CHECK("quantize_tokens_kernel");
    return 0;
}

template <int TYPE>
int launch_type(const TokenParams &p, hipStream_t stream) {
    // Several rows a wavefront where they are short (33 million rows of one value 130 us, a wavefront each 1400); a wavefront a row, with no
    // barrier, while there are rows for all CUs (8192 x 4096 bf16 19.4 us, 256 threads a row 21.6); more threads a row where there are few
    // rows or it is long.
    const int64_t pieces = ceil_div(p.cols_out, PIECE);
    if (pieces <= 1) return launch<TYPE, 1, 1, true>(p, stream);
    if (pieces <= 4) return launch<TYPE, 4, 1, true>(p, stream);
    if (pieces <= 16) return launch<TYPE, 16, 1, true>(p, stream);
    if (pieces <= 64) return launch<TYPE, 64, 1, true>(p, stream);
    if (p.rows >= 512 || pieces <= 128) {
        if (pieces <= 128) return launch<TYPE, 64, 2, true>(p, stream);
        if (pieces <= 256) return launch<TYPE, 64, 4, true>(p, stream);
        if (pieces <= 512) return launch<TYPE, 64, 8, true>(p, stream);
    }
    if (pieces <= 256) return launch<TYPE, 256, 1, true>(p, stream);
    if (pieces <= 512) return launch<TYPE, 256, 2, true>(p, stream);
    if (pieces <= 1024) return launch<TYPE, 256, 4, true>(p, stream);
    if (pieces <= 4096) return launch<TYPE, 1024, 4, true>(p, stream);
    return launch<TYPE, 1024, 4, false>(p, stream);
}

}  // namespace

int quantize_rows(int64_t rows, int cols, int cols_out, const void *x, int type, int64_t x_stride, int8_t *q, int64_t q_stride, float *scales,
                  hipStream_t stream) {
    if (rows == 0) return 0;
    const TokenParams p{x, q, scales, rows, x_stride, q_stride, cols, cols_out};
    return type == TSX_TYPE_F32 ? launch_type<TSX_TYPE_F32>(p, stream) : type == TSX_TYPE_F16 ? launch_type<TSX_TYPE_F16>(p, stream)
                                                                                              : launch_type<TSX_TYPE_BF16>(p, stream);
}

}  // namespace tsx

extern "C" int tsx_quantize_tokens(int64_t rows, int32_t cols, const void *x_dev, int32_t x_type, int64_t x_stride, int8_t *q_dev, int64_t q_stride,
                                   float *scales_dev, void *stream) {
    TSX_REQUIRE(rows >= 0 && cols > 0 && cols <= 1 << 30, "quantize_tokens: %lld rows of %d columns", (long long)rows, cols);
    TSX_REQUIRE(tsx::is_float_type(x_type), "quantize_tokens: element type %d (fp32, fp16 or bf16)", x_type);
    TSX_REQUIRE(rows <= 1 || (x_stride >= cols && q_stride >= cols), "quantize_tokens: rows of %d columns overlap at strides %lld and %lld", cols,
                (long long)x_stride, (long long)q_stride);
    TSX_REQUIRE(rows == 0 || (x_dev && q_dev && scales_dev), "quantize_tokens: null pointer");
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(x_dev) % tsx::element_bytes(x_type) == 0 && reinterpret_cast<uintptr_t>(scales_dev) % 4 == 0,
                "quantize_tokens: pointer is no multiple of its elements");
    return tsx::quantize_rows(rows, cols, cols, x_dev, x_type, x_stride, q_dev, q_stride, scales_dev, tsx::as_stream(stream));
}
