// Group norm with an activation on channels-last tensors, to the tensor's own type or to int8 tokens.
//
// A group is `d` consecutive channels of all pixels of one image: mean and variance over them, then
// y = act((x - mean) / sqrt(variance + epsilon) * weight[c] + bias[c]).  Bound: HBM, one read and one write of the tensor.
//
// Pixels are taken `rows` at a time: S pixels whose S * c values are whole pieces of 16 bytes (S = 1 where c is a multiple of a
// piece), so that a thread that steps by whole rows keeps the channels of its piece, whatever c is, and a wavefront reads consecutive
// bytes.  Sums of a channel are taken around the channel's first value that the thread sees: the difference of two large sums that
// would cancel never forms, since the value itself is part of the variance that the error is measured by.  Partial results are
// merged as (count, mean, squares around the mean), in an order that the sizes fix.
#include <algorithm>

#include "elements.hpp"

namespace tsx {
namespace {

constexpr int MOST_CHANNELS = 8192;

struct NormParams {
    const void *x;
    void *out;
    int8_t *q;
    float *scales;
    const float *weight, *bias;
    float2 *partial;                   // [n][chunks][groups]: mean, squares around it
    int64_t pixels, image_stride, pixel_stride;
    int64_t rows;                      // whole rows of S pixels
    int c, groups, d;
    int S, pieces;                     // pixels of a row; pieces of a row
    int lanes;                         // rows that a workgroup's threads take side by side (0: pieces in turns)
    int chunks;                        // of an image's rows, for the statistics
    int64_t chunk_rows;
    float epsilon, slope;
    int act;
};

template <int TYPE>
struct Kind {
    static constexpr int SIZE = TYPE == TSX_TYPE_F32 ? 4 : 2;
};

// One piece of V values: whole, or of the image's last, incomplete row.  `at`: values from the image's first.
template <int TYPE, int V>
struct Piece {
    float v[V];
    __device__ __forceinline__ void load(const char *image, int64_t at) {
        constexpr int SIZE = Kind<TYPE>::SIZE;
        if constexpr (V == 1) {
            if constexpr (TYPE == TSX_TYPE_F32) v[0] = *reinterpret_cast<const float *>(image + at * SIZE);
            else v[0] = half_value<TYPE>(*reinterpret_cast<const unsigned short *>(image + at * SIZE));
        } else {
            Run<TYPE, V> r;
            r.load(image + at * SIZE);
            static_for<0, V>([&](auto ec) { v[decltype(ec)::value] = r.template get<decltype(ec)::value>(); });
        }
    }
    __device__ __forceinline__ void load_some(const char *image, int64_t at, int left) {
        constexpr int SIZE = Kind<TYPE>::SIZE;
        if constexpr (V == 1) {
            load(image, at);
        } else {
            Run<TYPE, V> r;
            r.load_some(image + at * SIZE, left);
            static_for<0, V>([&](auto ec) { v[decltype(ec)::value] = r.template get<decltype(ec)::value>(); });
        }
    }
    template <int KIND>
    static __device__ __forceinline__ float half_value(unsigned short bits) {
        if constexpr (KIND == TSX_TYPE_BF16) return __builtin_bit_cast(float, unsigned(bits) << 16);
        else return float(__builtin_bit_cast(_Float16, bits));
    }
    __device__ __forceinline__ void store(char *out, int64_t at, int left) const {
        constexpr int SIZE = Kind<TYPE>::SIZE;
        if constexpr (V == 1) {
            if constexpr (TYPE == TSX_TYPE_F32) *reinterpret_cast<float *>(out + at * SIZE) = v[0];
            else if constexpr (TYPE == TSX_TYPE_BF16) *reinterpret_cast<__bf16 *>(out + at * SIZE) = __bf16(v[0]);
            else *reinterpret_cast<_Float16 *>(out + at * SIZE) = _Float16(v[0]);
        } else {
            Run<TYPE, V> r;
            r.set(v);
            if (left >= V) r.store(out + at * SIZE);
            else r.store_some(out + at * SIZE, left);
        }
    }
};

// Sum over a wavefront's lanes, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int far = 1; far < 64; far *= 2) v += __shfl_xor(v, far);
    return v;
}

// ---- statistics of a chunk of rows of one image

template <int TYPE, int V>
__global__ __launch_bounds__(512) void group_norm_statistics_kernel(NormParams p) {
    extern __shared__ float entries[];                       // [lanes][S * c] means, then squares, then counts
    const int threads = blockDim.x, t = threadIdx.x;
    const int lanes = p.lanes ? p.lanes : 1, row_values = p.S * p.c;
    float *const means = entries, *const squares = means + lanes * row_values, *const counts = squares + lanes * row_values;
    const int64_t image = blockIdx.y;
    const int chunk = blockIdx.x;
    const char *const x = static_cast<const char *>(p.x) + image * p.image_stride * Kind<TYPE>::SIZE;
    const int64_t row_stride = p.S * p.pixel_stride, values = p.pixels * p.c;
    const int64_t first = chunk * p.chunk_rows, end = min(first + p.chunk_rows, p.rows);
    // the incomplete row, with the last chunk
    const bool with_tail = chunk == p.chunks - 1 && p.rows * p.S < p.pixels;
    for (int j0 = 0; j0 < p.pieces; j0 += threads) {         // one turn where the threads cover a row
        const int j = p.lanes ? t % p.pieces : j0 + t, lane = p.lanes ? t / p.pieces : 0;
        if (lane < lanes && j < p.pieces) {
            float base[V], sum[V], square[V], count = 0.f;
            static_for<0, V>([&](auto ec) { base[decltype(ec)::value] = sum[decltype(ec)::value] = square[decltype(ec)::value] = 0.f; });
            auto take = [&](const Piece<TYPE, V> &a) __attribute__((always_inline)) {
                static_for<0, V>([&](auto ec) {
                    constexpr int e = decltype(ec)::value;
                    const float d = a.v[e] - base[e];
                    sum[e] += d;
                    square[e] = __builtin_fmaf(d, d, square[e]);
                });
            };
            int64_t row = first + lane;
            if (row < end) {
                Piece<TYPE, V> a;
                a.load(x, row * row_stride + j * V);
                static_for<0, V>([&](auto ec) { base[decltype(ec)::value] = a.v[decltype(ec)::value]; });
                count = 1.f;
                row += lanes;
            }
            for (; row + 3 * lanes < end; row += 4 * lanes) {
                Piece<TYPE, V> a[4];
                static_for<0, 4>([&](auto uc) { a[decltype(uc)::value].load(x, (row + decltype(uc)::value * lanes) * row_stride + j * V); });
                static_for<0, 4>([&](auto uc) { take(a[decltype(uc)::value]); });
                count += 4.f;
            }
            for (; row < end; row += lanes) {
                Piece<TYPE, V> a;
                a.load(x, row * row_stride + j * V);
                take(a);
                count += 1.f;
            }
            float n[V];
            static_for<0, V>([&](auto ec) { n[decltype(ec)::value] = count; });
            if (with_tail && lane == 0) {
                const int64_t at = p.rows * row_values + j * V;
                const int left = int(min(values - at, int64_t(V)));
                if (left > 0) {
                    Piece<TYPE, V> a;
                    a.load_some(x, at, left);
                    static_for<0, V>([&](auto ec) {
                        constexpr int e = decltype(ec)::value;
                        if (e < left) {
                            if (count == 0.f) base[e] = a.v[e];
                            const float d = a.v[e] - base[e];
                            sum[e] += d;
                            square[e] = __builtin_fmaf(d, d, square[e]);
                            n[e] += 1.f;
                        }
                    });
                }
            }
            static_for<0, V>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                const int at = lane * row_values + j * V + e;
                const float m = n[e] > 0.f ? sum[e] / n[e] : 0.f;
                means[at] = base[e] + m;
                squares[at] = fmaxf(__builtin_fmaf(-m, sum[e], square[e]), 0.f);
                counts[at] = n[e];
            });
        }
        if (p.lanes) break;
    }
    __syncthreads();
    // a wavefront a group: entries [lane][pixel of the row][channel of the group]
    const int own = lanes * p.S * p.d;
    for (int g = t / 64; g < p.groups; g += threads / 64) {
        float n = 0.f, s = 0.f;
        const float about = means[g * p.d];
        for (int i = t % 64; i < own; i += 64) {
            const int q = i / p.d, at = q * p.c + g * p.d + (i - q * p.d);
            n += counts[at];
            s = __builtin_fmaf(counts[at], means[at] - about, s);
        }
        n = wave_sum(n);
        s = wave_sum(s);
        const float mean = about + (n > 0.f ? s / n : 0.f);
        float m2 = 0.f;
        for (int i = t % 64; i < own; i += 64) {
            const int q = i / p.d, at = q * p.c + g * p.d + (i - q * p.d);
            const float d = means[at] - mean;
            m2 += __builtin_fmaf(counts[at] * d, d, squares[at]);
        }
        m2 = wave_sum(m2);
        if (t % 64 == 0) p.partial[(image * p.chunks + chunk) * p.groups + g] = float2{mean, m2};
    }
}

// Mean and 1 / sqrt(variance + epsilon) of the groups of one image, into LDS: T = 16 threads a group.
__device__ __forceinline__ float sixteen_sum(float v) {
#pragma unroll
    for (int far = 1; far < 16; far *= 2) v += __shfl_xor(v, far);
    return v;
}
__device__ __forceinline__ void merge_chunks(const NormParams &p, int64_t image, float2 *group) {
    const float2 *const partial = p.partial + image * p.chunks * p.groups;
    const float whole = float(p.chunk_rows) * float(p.S) * float(p.d);
    const float last = float(p.pixels - (p.chunks - 1) * p.chunk_rows * p.S) * float(p.d);
    const float total = float(p.pixels) * float(p.d);
    for (int g = threadIdx.x / 16; g < p.groups; g += blockDim.x / 16) {
        const float about = partial[g].x;
        float s = 0.f, m2 = 0.f;
        for (int k = threadIdx.x % 16; k < p.chunks; k += 16) s = __builtin_fmaf(k == p.chunks - 1 ? last : whole, partial[int64_t(k) * p.groups + g].x - about, s);
        const float mean = about + sixteen_sum(s) / total;
        for (int k = threadIdx.x % 16; k < p.chunks; k += 16) {
            const float2 part = partial[int64_t(k) * p.groups + g];
            const float d = part.x - mean;
            m2 += __builtin_fmaf((k == p.chunks - 1 ? last : whole) * d, d, part.y);
        }
        m2 = sixteen_sum(m2);
        if (threadIdx.x % 16 == 0) group[g] = float2{mean, 1.f / sqrtf(m2 / total + p.epsilon)};
    }
}

// ---- the norm itself on rows of one image

template <int TYPE, int V>
__global__ __launch_bounds__(512) void group_norm_apply_kernel(NormParams p) {
    extern __shared__ float2 group[];
    const int threads = blockDim.x, t = threadIdx.x;
    const int lanes = p.lanes ? p.lanes : 1, row_values = p.S * p.c;
    const int64_t image = blockIdx.y;
    merge_chunks(p, image, group);
    __syncthreads();
    const char *const x = static_cast<const char *>(p.x) + image * p.image_stride * Kind<TYPE>::SIZE;
    char *const out = static_cast<char *>(p.out) + image * p.pixels * p.c * Kind<TYPE>::SIZE;
    const int64_t row_stride = p.S * p.pixel_stride, values = p.pixels * p.c;
    for (int j0 = 0; j0 < p.pieces; j0 += threads) {
        const int j = p.lanes ? t % p.pieces : j0 + t, lane = p.lanes ? t / p.pieces : 0;
        if (lane < lanes && j < p.pieces) {
            float mean[V], scale[V], shift[V];
            static_for<0, V>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                const int ch = (j * V + e) % p.c;
                const float2 g = group[ch / p.d];
                mean[e] = g.x;
                scale[e] = p.weight ? g.y * p.weight[ch] : g.y;
                shift[e] = p.bias ? p.bias[ch] : 0.f;
            });
            auto apply = [&](Piece<TYPE, V> &a) __attribute__((always_inline)) {
                static_for<0, V>([&](auto ec) { constexpr int e = decltype(ec)::value; a.v[e] = __builtin_fmaf(a.v[e] - mean[e], scale[e], shift[e]); });
                activate_tokens(a.v, p.act, p.slope);
            };
            const int64_t step = int64_t(gridDim.x) * lanes;
            int64_t row = int64_t(blockIdx.x) * lanes + lane;
            for (; row + step < p.rows; row += 2 * step) {
                Piece<TYPE, V> a[2];
                static_for<0, 2>([&](auto uc) { a[decltype(uc)::value].load(x, (row + decltype(uc)::value * step) * row_stride + j * V); });
                static_for<0, 2>([&](auto uc) {
                    apply(a[decltype(uc)::value]);
                    a[decltype(uc)::value].store(out, (row + decltype(uc)::value * step) * row_values + j * V, V);
                });
            }
            if (row < p.rows) {
                Piece<TYPE, V> a;
                a.load(x, row * row_stride + j * V);
                apply(a);
                a.store(out, row * row_values + j * V, V);
            }
            if (p.rows * p.S < p.pixels && blockIdx.x == 0 && lane == 0) {
                const int64_t at = p.rows * row_values + j * V;
                const int left = int(min(values - at, int64_t(V)));
                if (left > 0) {
                    Piece<TYPE, V> a;
                    a.load_some(x, at, left);
                    apply(a);
                    a.store(out, at, left);
                }
            }
        }
        if (p.lanes) break;
    }
}

// ---- the norm's values as int8 tokens: a wavefront a pixel, whose values it works out twice, for the largest and to round them
template <int TYPE>
__global__ __launch_bounds__(256) void group_norm_tokens_kernel(NormParams p) {
    extern __shared__ float2 group[];
    const int64_t image = blockIdx.y;
    merge_chunks(p, image, group);
    __syncthreads();
    const int lane = threadIdx.x % 64;
    for (int64_t pixel = int64_t(blockIdx.x) * 4 + threadIdx.x / 64; pixel < p.pixels; pixel += int64_t(gridDim.x) * 4) {
        const char *const x = static_cast<const char *>(p.x) + (image * p.image_stride + pixel * p.pixel_stride) * Kind<TYPE>::SIZE;
        auto value = [&](int ch) __attribute__((always_inline)) {
            Piece<TYPE, 1> a;
            a.load(x, ch);
            const float2 g = group[ch / p.d];
            float v[1] = {__builtin_fmaf(a.v[0] - g.x, p.weight ? g.y * p.weight[ch] : g.y, p.bias ? p.bias[ch] : 0.f)};
            activate_tokens(v, p.act, p.slope);
            return v[0];
        };
        unsigned top = 0;
        for (int ch = lane; ch < p.c; ch += 64) top = max(top, __builtin_bit_cast(unsigned, value(ch)) & 0x7fffffffu);
#pragma unroll
        for (int far = 1; far < 64; far *= 2) top = max(top, unsigned(__shfl_xor(int(top), far)));
        const TokenScale s(__builtin_bit_cast(float, top));
        const int64_t token = image * p.pixels + pixel;
        if (lane == 0) p.scales[token] = s.scale;
        for (int ch = lane; ch < p.c; ch += 64) p.q[token * p.c + ch] = s.reciprocal == 0.f ? int8_t(0) : int8_t(s.bits(__fmul_rn(value(ch), s.lift)));
    }
}

// ---- host side

constexpr int MOST_CHUNKS = 64;

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// Rows, threads and chunks of a call; V: values of a piece (1: a channel a thread, for pixels apart that are no whole pieces).
struct NormPlan {
    NormParams p;
    int V, threads;
};

NormPlan plan_of(const tsx_group_norm *g) {
    NormPlan pl{};
    NormParams &p = pl.p;
    const int whole = g->type == TSX_TYPE_F32 ? 4 : 8;
    const bool dense = g->pixel_stride == g->c || g->pixels <= 1;
    const int S = whole / gcd(g->c, whole);
    pl.V = S == 1 || (dense && S * g->c <= MOST_CHANNELS) ? whole : 1;
    p.S = pl.V == 1 ? 1 : S;
    p.x = g->x_dev;
    p.weight = g->weight_dev;
    p.bias = g->bias_dev;
    p.pixels = g->pixels;
    p.image_stride = g->image_stride;
    p.pixel_stride = g->pixels <= 1 ? g->c : g->pixel_stride;
    p.c = g->c;
    p.groups = g->groups;
    p.d = g->c / g->groups;
    p.epsilon = g->epsilon;
    p.slope = g->slope;
    p.act = g->act;
    p.rows = g->pixels / p.S;
    p.pieces = p.S * p.c / pl.V;
    pl.threads = p.pieces <= 256 ? 256 : 512;
    p.lanes = p.pieces <= pl.threads ? pl.threads / p.pieces : 0;
    const int side = p.lanes ? p.lanes : 1;
    const int64_t wanted = ceil_div(1024, g->n > 0 ? g->n : 1);
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>({wanted, int64_t(MOST_CHUNKS), p.rows / (4 * side)}));
    p.chunk_rows = std::max<int64_t>(1, ceil_div(p.rows, chunks));
    p.chunks = int(std::max<int64_t>(1, ceil_div(p.rows, p.chunk_rows)));
    return pl;
}

int check(const tsx_group_norm *g, const char *what) {
    TSX_REQUIRE(g, "%s: null argument", what);
    TSX_REQUIRE(g->n >= 0 && g->pixels >= 0 && g->c > 0 && g->groups > 0, "%s: bad extents", what);
    TSX_REQUIRE(g->c % g->groups == 0, "%s: %d channels are no %d groups", what, g->c, g->groups);
    TSX_REQUIRE(g->c <= MOST_CHANNELS, "%s: %d channels (at most %d)", what, g->c, MOST_CHANNELS);
    TSX_REQUIRE(is_float_type(g->type), "%s: element type %d (fp32, fp16 or bf16)", what, g->type);
    TSX_REQUIRE(g->n < 65536 && g->pixels <= int64_t(1) << 40, "%s: %d images of %lld pixels", what, g->n, (long long)g->pixels);
    TSX_REQUIRE(g->pixels <= 1 || g->pixel_stride >= g->c, "%s: pixels of %d channels overlap at a stride of %lld", what, g->c, (long long)g->pixel_stride);
    TSX_REQUIRE(g->n <= 1 || g->image_stride >= 0, "%s: negative image stride", what);
    TSX_REQUIRE(is_token_act(g->act), "%s: activation %d", what, g->act);
    TSX_REQUIRE(g->epsilon >= 0.f, "%s: epsilon is negative or NaN", what);
    TSX_REQUIRE(g->n == 0 || g->pixels == 0 || g->x_dev, "%s: null input", what);
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(g->x_dev) % element_bytes(g->type) == 0, "%s: pointer is no multiple of its elements", what);
    return 0;
}

size_t workspace_bytes(const tsx_group_norm *g) {
    const NormPlan pl = plan_of(g);
    return size_t(g->n) * pl.p.chunks * g->groups * sizeof(float2);
}

template <int TYPE, int V>
int launch_statistics(const NormPlan &pl, int n, hipStream_t stream) {
    const NormParams &p = pl.p;
    const size_t lds = size_t(p.lanes ? p.lanes : 1) * p.S * p.c * 3 * sizeof(float);
    if (lds > 64 * 1024)
        TSX_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(group_norm_statistics_kernel<TYPE, V>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    hipLaunchKernelGGL((group_norm_statistics_kernel<TYPE, V>), dim3(unsigned(p.chunks), unsigned(n)), dim3(pl.threads), lds, stream, p);
    TSX_LAUNCH_CHECK("group_norm_statistics_kernel");
    return 0;
}

template <int TYPE, int V>
int launch_apply(const NormPlan &pl, int n, hipStream_t stream) {
    const NormParams &p = pl.p;
    const int64_t side = p.lanes ? p.lanes : 1, most = ceil_div(2048, n);
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(ceil_div(p.rows, 2 * side), most));
    hipLaunchKernelGGL((group_norm_apply_kernel<TYPE, V>), dim3(unsigned(blocks), unsigned(n)), dim3(pl.threads), size_t(p.groups) * sizeof(float2), stream, p);
    TSX_LAUNCH_CHECK("group_norm_apply_kernel");
    return 0;
}

template <int TYPE>
int run(const tsx_group_norm *g, NormPlan pl, hipStream_t stream) {
    constexpr int V = TYPE == TSX_TYPE_F32 ? 4 : 8;
    int rc = pl.V == 1 ? launch_statistics<TYPE, 1>(pl, g->n, stream) : launch_statistics<TYPE, V>(pl, g->n, stream);
    if (rc) return rc;
    if (!pl.p.q) return pl.V == 1 ? launch_apply<TYPE, 1>(pl, g->n, stream) : launch_apply<TYPE, V>(pl, g->n, stream);
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>(ceil_div(g->pixels, 4), ceil_div(4096, g->n)));
    hipLaunchKernelGGL((group_norm_tokens_kernel<TYPE>), dim3(unsigned(blocks), unsigned(g->n)), dim3(256), size_t(g->groups) * sizeof(float2), stream, pl.p);
    TSX_LAUNCH_CHECK("group_norm_tokens_kernel");
    return 0;
}

int run_any(const tsx_group_norm *g, void *out, int8_t *q, float *scales, void *workspace, size_t bytes, const char *what, hipStream_t stream) {
    int rc = check(g, what);
    if (rc) return rc;
    if (g->n == 0 || g->pixels == 0) return 0;
    TSX_REQUIRE(q ? scales != nullptr : out != nullptr, "%s: null output", what);
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(out) % element_bytes(g->type) == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                "%s: pointer is no multiple of its elements", what);
    const size_t need = workspace_bytes(g);
    if (!workspace || bytes < need) return fail(TSX_E_WORKSPACE, "%s: workspace %zu < %zu bytes", what, workspace ? bytes : size_t(0), need);
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "%s: workspace must be 8-byte aligned", what);
    NormPlan pl = plan_of(g);
    pl.p.out = out;
    pl.p.q = q;
    pl.p.scales = scales;
    pl.p.partial = static_cast<float2 *>(workspace);
    return g->type == TSX_TYPE_F32 ? run<TSX_TYPE_F32>(g, pl, stream) : g->type == TSX_TYPE_F16 ? run<TSX_TYPE_F16>(g, pl, stream)
                                                                                                : run<TSX_TYPE_BF16>(g, pl, stream);
}

}  // namespace
}  // namespace tsx

extern "C" {

size_t tsx_group_norm_workspace_bytes(const tsx_group_norm *g) {
    if (tsx::check(g, "group_norm") || g->n == 0 || g->pixels == 0) return 0;
    return tsx::workspace_bytes(g);
}

int tsx_group_norm_nhwc(const tsx_group_norm *g, void *out_dev, void *workspace_dev, size_t workspace_bytes, void *stream) {
    return tsx::run_any(g, out_dev, nullptr, nullptr, workspace_dev, workspace_bytes, "group_norm", tsx::as_stream(stream));
}

int tsx_group_norm_tokens_nhwc(const tsx_group_norm *g, int8_t *q_dev, float *scales_dev, void *workspace_dev, size_t workspace_bytes, void *stream) {
    if (g && g->n > 0 && g->pixels > 0) TSX_REQUIRE(q_dev && scales_dev, "group_norm_tokens: null output");
    return tsx::run_any(g, nullptr, q_dev, scales_dev, workspace_dev, workspace_bytes, "group_norm_tokens", tsx::as_stream(stream));
}

}  // extern "C"
