// int8 product with a scale for each token and each channel, on rows of fp32, fp16, bf16 or int8 values.
//
//     out[i][j] = act(float(sum_k q[i][k] w[k][j]) * w_scale[j] * x_scale[i] + bias[j]),  rounded once to the output's type
//
// Rows of floats become int8 first (tokens_i8.hip), in the workspace, padded with zeros to whole chunks of K.  int32 sums are
// exact, so every kernel here gives the same bits.
#include <algorithm>

#include "igemm_i8.hpp"
#include "tokens_i8.hpp"

namespace tsx {
namespace {

constexpr int CHUNK = 128;             // K bytes of a row per chunk: two packed K-steps

struct TokenGemmParams {
    const int8_t *q;                   // [m][pitch], 16-byte aligned, pitch a multiple of CHUNK... or k itself where that is one
    const float *x_scales;
    const int8_t *wp;                  // as tsx_gemm_i8_pack_weights lays them out
    const float *w_scales, *bias;
    void *out;
    int64_t pitch, out_stride;
    int m, n, frags, chunks;
    int act;
    float slope;
    int row_tiles, col_tiles, tiles_per_xcd;
};

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// 64 lanes x 16 bytes, from an address for each lane to consecutive bytes of LDS.  Complete when vmcnt says so.
__device__ __forceinline__ void to_lds(const int8_t *at, int8_t *lds) {
    __builtin_amdgcn_global_load_lds((global_void *)at, (lds_void *)lds, 16, 0, 0);
}

// What leaves a fragment of 32 output columns x 32 tokens: accumulator r of lane l is column 8 (r / 4) + 4 (l / 32) + r % 4 of token
// l % 32; swaps between the half-waves leave a lane with 16 consecutive columns, the lower ones with 0 .. 15, the upper ones with 16 .. 31.
template <int OUT>
__device__ __forceinline__ void store_fragment(const TokenGemmParams &p, const v16i &acc, const float (&ws)[16], const float (&bias)[16], float xs,
                                               int row, int col0) {
    const int lane = threadIdx.x % 64;
    float v[16];
    static_for<0, 16>([&](auto rc) { constexpr int r = decltype(rc)::value; v[r] = __fmul_rn(__fmul_rn(float(acc[r]), ws[r]), xs); });
    if (p.bias) static_for<0, 16>([&](auto rc) { constexpr int r = decltype(rc)::value; v[r] = __fadd_rn(v[r], bias[r]); });
    activate_tokens(v, p.act, p.slope);
    Run<OUT, 16> out, own;
    own.set(v);
    constexpr int W = Run<OUT, 4>::WORDS;      // words of four values
    static_for<0, 2>([&](auto pc) {
        constexpr int a = decltype(pc)::value;
        static_for<0, W>([&](auto wc) {
            constexpr int w = decltype(wc)::value;
            const auto s = __builtin_amdgcn_permlane32_swap(own.word[a * W + w], own.word[(a + 2) * W + w], false, false);
            out.word[2 * a * W + w] = s[0];
            out.word[(2 * a + 1) * W + w] = s[1];
        });
    });
    const int col = col0 + 16 * (lane / 32), left = p.n - col;
    if (row < p.m && left > 0) {
        char *const at = static_cast<char *>(p.out) + (int64_t(row) * p.out_stride + col) * (OUT == TSX_TYPE_F32 ? 4 : 2);
        if (left >= 16) out.store(at);
        else out.store_some(at, left);
    }
}

// the scales and biases of a lane's 16 accumulators
__device__ __forceinline__ void load_columns(const TokenGemmParams &p, int col0, float (&ws)[16], float (&bias)[16]) {
    const int half = (threadIdx.x % 64) / 32;
    static_for<0, 16>([&](auto rc) {
        constexpr int r = decltype(rc)::value;
        const int col = min(col0 + 8 * (r / 4) + 4 * half + r % 4, p.n - 1);
        ws[r] = p.w_scales[col];
        bias[r] = p.bias ? p.bias[col] : 0.f;
    });
}

// WR x WC wavefronts, each with FR x FC fragments of 32 tokens x 32 columns.
template <int WR, int WC, int FR, int FC, int OUT>
__global__ __launch_bounds__(WR *WC * 64) void gemm_i8_tokens_kernel(TokenGemmParams p) {
    constexpr int WAVES = WR * WC, ROWS = 32 * WR * FR, COLS = 32 * WC * FC;
    constexpr int A_BYTES = ROWS * CHUNK, B_BYTES = COLS * CHUNK, A_LOADS = A_BYTES / 1024 / WAVES, B_LOADS = B_BYTES / 1024 / WAVES;
    __shared__ __attribute__((aligned(16))) int8_t lds[2][A_BYTES + B_BYTES];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wave_r = wave / WC, wave_c = wave % WC;
    // blockIdx % 8 is the XCD: each takes a run of consecutive tiles, which walk four row tiles before the next column tile
    const int tiles = p.row_tiles * p.col_tiles;
    const int t = int(blockIdx.x % 8) * p.tiles_per_xcd + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= p.tiles_per_xcd || t >= tiles) return;      // uniform, ahead of every barrier
    const int group = t / (4 * p.col_tiles), in_group = t - group * 4 * p.col_tiles;
    const int group_rows = min(4, p.row_tiles - 4 * group);
    const int tile_c = in_group / group_rows, tile_r = 4 * group + in_group - tile_c * group_rows;
    const int row0 = tile_r * ROWS, frag0 = tile_c * (COLS / 32);

    // Rows in LDS are 128 bytes, their pieces of 16 XORed with bits 1 .. 3 of the row: 16 rows cover all banks for one piece.
    // A load instruction fills 8 rows; rows beyond m are the last one again, never stored.
    const int8_t *a_src[A_LOADS], *b_src[B_LOADS];
    static_for<0, A_LOADS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const int r = (wave * A_LOADS + i) * 8 + lane / 8;
        a_src[i] = p.q + int64_t(min(row0 + r, p.m - 1)) * p.pitch + ((lane % 8) ^ ((r >> 1) & 7)) * 16;
    });
    // weights: packed[K-step][fragment][half][lane][16], in LDS [K-step of the chunk][fragment][half][lane][16]
    static_for<0, B_LOADS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const int unit = wave * B_LOADS + i, step = unit / (2 * COLS / 32), in_step = unit % (2 * COLS / 32);
        const int frag = min(frag0 + in_step / 2, p.frags - 1);
        b_src[i] = p.wp + (int64_t(step) * p.frags + frag) * 2048 + (in_step % 2) * 1024 + lane * 16;
    });
    const int64_t b_step = int64_t(p.frags) * 4096;
    auto fetch = [&](int c, int buf) __attribute__((always_inline)) {
        static_for<0, A_LOADS>([&](auto ic) { constexpr int i = decltype(ic)::value; to_lds(a_src[i] + int64_t(c) * CHUNK, &lds[buf][(wave * A_LOADS + i) * 1024]); });
        static_for<0, B_LOADS>([&](auto ic) { constexpr int i = decltype(ic)::value; to_lds(b_src[i] + c * b_step, &lds[buf][A_BYTES + (wave * B_LOADS + i) * 1024]); });
    };

    v16i acc[FR][FC];
    static_for<0, FR * FC>([&](auto fc) {
        constexpr int f = decltype(fc)::value;
        static_for<0, 16>([&](auto rc) { acc[f / FC][f % FC][decltype(rc)::value] = 0; });
    });
    const int a_row = (wave_r * FR * 32 + lane % 32) * CHUNK, a_key = (lane >> 1) & 7;
    fetch(0, 0);
    for (int c = 0; c < p.chunks; ++c) {
        const int buf = c & 1;
        // chunk c is in LDS, for every wavefront, and the other buffer is read
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        if (c + 1 < p.chunks) fetch(c + 1, buf ^ 1);
        static_for<0, CHUNK / 32>([&](auto hc) {
            constexpr int h = decltype(hc)::value;
            v4i a[FR], b[FC];
            static_for<0, FR>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                a[i] = *reinterpret_cast<const v4i *>(&lds[buf][a_row + i * 32 * CHUNK + ((2 * h + lane / 32) ^ a_key) * 16]);
            });
            static_for<0, FC>([&](auto fc) {
                constexpr int f = decltype(fc)::value;
                b[f] = *reinterpret_cast<const v4i *>(&lds[buf][A_BYTES + (((h / 2) * (COLS / 32) + wave_c * FC + f) * 2 + h % 2) * 1024 + lane * 16]);
            });
            static_for<0, FR * FC>([&](auto fc) {
                constexpr int i = decltype(fc)::value / FC, f = decltype(fc)::value % FC;
                acc[i][f] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[f], a[i], acc[i][f], 0, 0, 0);
            });
        });
    }
    static_for<0, FC>([&](auto fc) {
        constexpr int f = decltype(fc)::value;
        const int col0 = (frag0 + wave_c * FC + f) * 32;
        if (col0 < p.n) {                                    // uniform
            float ws[16], bias[16];
            load_columns(p, col0, ws, bias);
            static_for<0, FR>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int row = row0 + (wave_r * FR + i) * 32 + lane % 32;
                store_fragment<OUT>(p, acc[i][f], ws, bias, p.x_scales[min(row, p.m - 1)], row, col0);
            });
        }
    });
}

template <int WR, int WC, int FR, int FC, int OUT>
int launch_tile(TokenGemmParams p, hipStream_t stream) {
    p.row_tiles = int(ceil_div(p.m, 32 * WR * FR));
    p.col_tiles = int(ceil_div(p.n, 32 * WC * FC));
    p.tiles_per_xcd = int(ceil_div(int64_t(p.row_tiles) * p.col_tiles, 8));
    hipLaunchKernelGGL((gemm_i8_tokens_kernel<WR, WC, FR, FC, OUT>), dim3(unsigned(8 * p.tiles_per_xcd)), dim3(WR * WC * 64), 0, stream, p);
    TSX_LAUNCH_CHECK("gemm_i8_tokens_kernel");
    return 0;
}

template <int OUT>
int launch(const TokenGemmParams &p, hipStream_t stream) {
    return launch_tile<2, 2, 2, 2, OUT>(p, stream);
}

// rows of int8 tokens of another length, stride or alignment than the kernels read, copied to whole chunks
__global__ __launch_bounds__(256) void copy_tokens_kernel(const int8_t *x, int64_t x_stride, int k, int8_t *q, int pitch, int64_t rows) {
    const int pieces = pitch / 16;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < rows * pieces; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / pieces;
        const int at = int(i - row * pieces) * 16;
        v4i v = {0, 0, 0, 0};
        const int8_t *const from = x + row * x_stride + at;
        if (at + 16 <= k) v = __builtin_bit_cast(v4i, v4u(*reinterpret_cast<const v4u_any *>(from)));
        else
            for (int b = 0; b < 16 && at + b < k; ++b) v[b / 4] |= int((unsigned(from[b]) & 255u) << (8 * (b % 4)));
        *reinterpret_cast<v4i *>(q + row * pitch + at) = v;
    }
}

int check(const tsx_token_gemm *g) {
    TSX_REQUIRE(g, "gemm_i8_tokens: null argument");
    TSX_REQUIRE(g->m >= 0 && g->n > 0 && g->k > 0, "gemm_i8_tokens: bad extents");
    TSX_REQUIRE(g->k < 1 << 17, "gemm_i8_tokens: K = %d (below 2^17: longer sums leave 32 bits)", g->k);
    TSX_REQUIRE(g->m < (1 << 30) && g->n < (1 << 30), "gemm_i8_tokens: extents of 2^30 and more");
    TSX_REQUIRE(is_float_type(g->x_type) || g->x_type == TSX_TYPE_I8, "gemm_i8_tokens: element type %d", g->x_type);
    TSX_REQUIRE(is_float_type(g->out_type), "gemm_i8_tokens: output type %d (fp32, fp16 or bf16)", g->out_type);
    TSX_REQUIRE(is_token_act(g->act), "gemm_i8_tokens: activation %d", g->act);
    TSX_REQUIRE(g->m <= 1 || (g->x_stride >= g->k && g->out_stride >= g->n), "gemm_i8_tokens: rows of %d and %d columns overlap at strides %lld and %lld",
                g->k, g->n, (long long)g->x_stride, (long long)g->out_stride);
    return 0;
}

int padded(int k) { return int(round_up(k, CHUNK)); }

bool reads_in_place(const tsx_token_gemm *g) {
    return g->x_type == TSX_TYPE_I8 && g->k % CHUNK == 0 && (g->m <= 1 || g->x_stride % 16 == 0) && reinterpret_cast<uintptr_t>(g->x_dev) % 16 == 0;
}

size_t scales_offset(const tsx_token_gemm *g) { return size_t(g->m) * padded(g->k); }

size_t workspace_bytes(const tsx_token_gemm *g) {
    if (g->m == 0 || reads_in_place(g)) return 0;
    return scales_offset(g) + (g->x_type == TSX_TYPE_I8 ? 0 : size_t(g->m) * 4);
}

}  // namespace
}  // namespace tsx

extern "C" {

size_t tsx_gemm_i8_tokens_workspace_bytes(const tsx_token_gemm *g) {
    if (tsx::check(g)) return 0;
    return tsx::workspace_bytes(g);
}

int tsx_gemm_i8_tokens(const tsx_token_gemm *g, void *workspace_dev, size_t workspace_bytes, void *stream_) {
    int rc = tsx::check(g);
    if (rc || g->m == 0) return rc;
    TSX_REQUIRE(g->x_dev && g->packed_w_dev && g->w_scales_dev && g->out_dev, "gemm_i8_tokens: null pointer");
    TSX_REQUIRE(g->x_type != TSX_TYPE_I8 || g->x_scales_dev, "gemm_i8_tokens: int8 rows need their scales");
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(g->packed_w_dev) % 16 == 0, "gemm_i8_tokens: packed weights must be 16-byte aligned");
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(g->x_dev) % tsx::element_bytes(g->x_type) == 0 &&
                    reinterpret_cast<uintptr_t>(g->out_dev) % tsx::element_bytes(g->out_type) == 0, "gemm_i8_tokens: pointer is no multiple of its elements");
    const size_t need = tsx::workspace_bytes(g);
    if (need) {
        if (!workspace_dev || workspace_bytes < need)
            return tsx::fail(TSX_E_WORKSPACE, "gemm_i8_tokens: workspace %zu < %zu bytes", workspace_dev ? workspace_bytes : size_t(0), need);
        TSX_REQUIRE(reinterpret_cast<uintptr_t>(workspace_dev) % 16 == 0, "gemm_i8_tokens: workspace must be 16-byte aligned");
    }
    hipStream_t stream = tsx::as_stream(stream_);
    tsx::TokenGemmParams p{};
    const int kp = tsx::padded(g->k);
    p.q = static_cast<const int8_t *>(need ? workspace_dev : g->x_dev);
    p.pitch = need ? kp : g->x_stride;
    p.x_scales = g->x_scales_dev;
    if (g->x_type != TSX_TYPE_I8) {
        float *const scales = reinterpret_cast<float *>(static_cast<char *>(workspace_dev) + tsx::scales_offset(g));
        rc = tsx::quantize_rows(g->m, g->k, kp, g->x_dev, g->x_type, g->x_stride, static_cast<int8_t *>(workspace_dev), kp, scales, stream);
        if (rc) return rc;
        p.x_scales = scales;
    } else if (need) {
        const int64_t pieces = int64_t(g->m) * (kp / 16), blocks = tsx::ceil_div(pieces, 256);
        hipLaunchKernelGGL(tsx::copy_tokens_kernel, dim3(unsigned(std::min<int64_t>(blocks, 1 << 16))), dim3(256), 0, stream,
                           static_cast<const int8_t *>(g->x_dev), g->x_stride, g->k, static_cast<int8_t *>(workspace_dev), kp, int64_t(g->m));
        TSX_LAUNCH_CHECK("copy_tokens_kernel");
    }
    p.wp = static_cast<const int8_t *>(g->packed_w_dev);
    p.w_scales = g->w_scales_dev;
    p.bias = g->bias_dev;
    p.out = g->out_dev;
    p.out_stride = g->out_stride;
    p.m = g->m;
    p.n = g->n;
    p.frags = int(tsx::round_up(g->n, 128) / 32);
    p.chunks = kp / tsx::CHUNK;
    p.act = g->act;
    p.slope = g->slope;
    return g->out_type == TSX_TYPE_F32 ? tsx::launch<TSX_TYPE_F32>(p, stream) : g->out_type == TSX_TYPE_F16 ? tsx::launch<TSX_TYPE_F16>(p, stream)
                                                                                                          : tsx::launch<TSX_TYPE_BF16>(p, stream);
}

}  // extern "C"
