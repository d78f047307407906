// Group norm with an activation on channels-last tensors, to the tensor's own type or to int8 tokens.
//
// A group is `d` consecutive channels of all pixels of one image: mean and variance over them, then
// y = act((x - mean) / sqrt(variance + epsilon) * weight[c] + bias[c]).  Bound: HBM, one read and one write of the tensor.
//
// Two kernels, the statistics of chunks and the norm, the least of 24 launches: 512 x 512 x 128 bf16 on 4 images, 268 MB, 45 and 81 us (6.0 and
// 6.6 TB/s: the second finds part of its input in the caches); 64 x 64 x 320 fp16 on 8, 21 MB, 7.4 and 9.8 us, of which each has 2 of launch and about 2 of
// prologue and reductions.
//
// Pixels are taken `rows` at a time: S pixels whose S * c values are whole pieces of 16 bytes (S = 1 where c is a multiple of a
// piece), so that a thread that steps by whole rows keeps the channels of its piece, whatever c is, and a wavefront reads consecutive
// bytes.  Sums of a channel are taken around its mean so far, which is brought up to date after 8, 16, 32, 64 rows and every 64 from there on:
// a batch is no longer than what came before it, so at most half of its squares cancels (of the first eight, around the first value, seven
// eighths).  Sums around one value for all n rows of a thread leave 1 / n of the squares where that value is far from the rest: with 1000 ahead
// of 1000 small ones the norm was off by a hundredth.  Of a mean's update what its rounding drops is kept, since it would add up where an image
// grows along its rows.  This takes 0.4 us (64 x 64 x 320).  Partial results are merged as (count, mean, squares around the mean), in an order
// that the sizes fix.
#include <algorithm>

#include "group_norm.hpp"

namespace tsx {
namespace {

// ---- statistics of a chunk of rows of one image

template <int TYPE, int V>
__global__ __launch_bounds__(NORM_MOST_THREADS) void group_norm_statistics_kernel(NormParams p) {
    extern __shared__ float entries[];                       // [lanes + 1][pitch] means, then squares
    __shared__ float waves[NORM_MOST_THREADS / 64];
    constexpr int SIZE = Kind<TYPE>::SIZE;
    const int threads = blockDim.x, t = threadIdx.x, chunk = blockIdx.x, image = blockIdx.y;
    const int lanes = p.lanes ? p.lanes : 1, pixel_entries = p.c >> p.lg_run, run = 1 << p.lg_run;
    const int pitch = (p.S * pixel_entries) | 1;             // odd: the lanes of one place lie in different banks
    float *const means = entries, *const squares = means + (lanes + 1) * pitch;
    const int first = chunk * p.chunk_rows, rows = min(p.chunk_rows, p.rows - first);
    const char *const x = static_cast<const char *>(p.x) + image * p.image_bytes;
    // the incomplete row, with the last chunk: entries of its own behind the lanes'
    const int tail = chunk == p.chunks - 1 ? p.tail : 0;
    const int full = lanes == 1 ? rows : udiv(rows, lanes, p.lanes_magic), over = rows - full * lanes;      // rows of a lane: one more for the first `over`
    auto leave = [&](int lane, int j, const float (&mean)[V], const float (&square)[V]) __attribute__((always_inline)) {
        int at = lane * pitch + (j * V >> p.lg_run);
        static_for<0, V>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            if ((e & (run - 1)) == 0) {
                means[at] = mean[e];
                squares[at++] = square[e];
            }
        });
    };
    // runs of values of one count become one entry: the mean of their means, their squares and n / 2 of the squared difference
    auto join = [&](float (&mean)[V], float (&square)[V], float count) __attribute__((always_inline)) {
        join_runs<V>(run, [&](auto ac, auto fc) {
            constexpr int a = decltype(ac)::value, b = a + decltype(fc)::value;
            const float d = mean[b] - mean[a];
            square[a] = square[a] + square[b] + (0.5f * decltype(fc)::value * count) * (d * d);
            mean[a] = __builtin_fmaf(d, 0.5f, mean[a]);
        });
    };
    for (int j0 = 0; j0 < p.pieces; j0 += threads) {         // one turn where the threads cover a row
        const int lane = p.lanes ? udiv(t, p.pieces, p.pieces_magic) : 0, j = p.lanes ? t - lane * p.pieces : j0 + t;
        if (lane < lanes && j < p.pieces) {
            const char *at = x + int64_t(first + lane) * p.row_bytes + j * (V * SIZE);
            const int count = full + (lane < over ? 1 : 0);
            // Requests of eight rows leave together; in the place of those that are none the last one is read again.
            constexpr int AHEAD = 8, LONGEST = 64;
            Run<TYPE, V> v[AHEAD];
            auto fetch = [&](int left) __attribute__((always_inline)) {
                static_for<0, AHEAD>([&](auto uc) { v[decltype(uc)::value].load(at + min(decltype(uc)::value, left - 1) * p.step_bytes); });
            };
            // mean + low and the squares around it of the `closed` rows so far; sums and squares of the differences from `mean` since
            float mean[V], low[V], square[V], sum[V], around[V];
            auto take = [&](auto uc) __attribute__((always_inline)) {
                static_for<0, V>([&](auto ec) {
                    constexpr int e = decltype(ec)::value;
                    const float d = v[decltype(uc)::value].template get<e>() - mean[e];
                    sum[e] += d;
                    around[e] = __builtin_fmaf(d, d, around[e]);
                });
            };
            auto close = [&](int closed, int rows) __attribute__((always_inline)) {
                const float n = float(closed), of_rows = __builtin_amdgcn_rcpf(float(rows));      // within a step: moves the mean by that much of its step
                static_for<0, V>([&](auto ec) {
                    constexpr int e = decltype(ec)::value;
                    const float nl = n * low[e], s = sum[e] + nl, step = s * of_rows, moved = mean[e] + step;
                    square[e] += __builtin_fmaf(-step, s, __builtin_fmaf(nl, low[e], around[e]));
                    low[e] = step - (moved - mean[e]);
                    mean[e] = moved;
                    sum[e] = around[e] = 0.f;
                });
            };
            int left = count;
            if (left > 0) fetch(left);
            static_for<0, V>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                mean[e] = left > 0 ? v[0].template get<e>() : 0.f;
                low[e] = square[e] = sum[e] = around[e] = 0.f;
            });
            int closed = 0, end = AHEAD;                     // the next batch's: as many rows as all before, at most LONGEST
            for (int rows = AHEAD; left > AHEAD; rows += AHEAD) {
                static_for<0, AHEAD>(take);
                at += AHEAD * p.step_bytes;
                left -= AHEAD;
                fetch(left);
                if (rows == end) {                           // uniform
                    close(closed, rows);
                    closed = rows;
                    end += min(rows, LONGEST);
                }
            }
            static_for<0, AHEAD>([&](auto uc) { if (decltype(uc)::value < left) take(uc); });
            if (count > 0) close(closed, count);
            join(mean, square, float(count));
            leave(lane, j, mean, square);
            if (lane == 0 && tail) {
                Piece<TYPE, V> a;
                static_for<0, V>([&](auto ec) { a.v[decltype(ec)::value] = square[decltype(ec)::value] = 0.f; });
                if (tail > j * V) a.load_some(x, int64_t(p.rows) * (p.S * p.c) + j * V, tail - j * V);
                join(a.v, square, 1.f);
                leave(lanes, j, a.v, square);
            }
        }
        if (p.lanes) break;
    }
    __syncthreads();
    // T threads a group, TL of them on lanes of their own, which share the lane's entries of the group
    const int group_entries = p.d >> p.lg_run, sides = lanes + (tail ? 1 : 0);
    const int T = 1 << p.lg_T, TL = 1 << p.lg_TL, TE = T >> p.lg_TL;
    const int tl = t & (TL - 1), te = (t & (T - 1)) >> p.lg_TL, tail_pixels = p.pixels - p.rows * p.S;
    auto each = [&](int g, auto &&body) __attribute__((always_inline)) {
        for (int lane = tl; lane < sides; lane += TL) {
            const float n = float(run * (lane == lanes ? 1 : full + (lane < over ? 1 : 0)));
            const int pixels = n == 0.f ? 0 : lane == lanes ? tail_pixels : p.S;
            for (int pixel = 0; pixel < pixels; ++pixel)
                for (int k = te; k < group_entries; k += TE) body(lane * pitch + pixel * pixel_entries + g * group_entries + k, n);
        }
    };
    const float of_values = __builtin_amdgcn_rcpf(chunk == p.chunks - 1 ? p.of_last : p.of_chunk);
    // Over the T threads of a group: of one wavefront, or of several, then through LDS
    auto sum_group = [&](float v) __attribute__((always_inline)) {
        v = sum_over_lanes(v, p.lg_T);
        if (T <= 64) return v;                             // uniform
        __syncthreads();
        if (t % 64 == 0) waves[t / 64] = v;
        __syncthreads();
        v = 0.f;
        for (int w = 0; w < T / 64; ++w) v += waves[(t >> p.lg_T) * (T / 64) + w];
        return v;
    };
    for (int g0 = 0; g0 < p.groups; g0 += threads >> p.lg_T) {
        const int g = min(g0 + (t >> p.lg_T), p.groups - 1); // T threads agree; behind the last group: that one again, not stored
        float s = 0.f, n2 = 0.f, m2 = 0.f;
        const float about = means[(rows ? 0 : lanes * pitch) + g * group_entries];
        each(g, [&](int at, float ni) __attribute__((always_inline)) { s = __builtin_fmaf(ni, means[at] - about, s); });
        s = sum_group(s);
        const float mean = about + s * of_values;
        // around that mean, and what the values are off it on the whole (its rounding)
        each(g, [&](int at, float ni) __attribute__((always_inline)) {
            const float d = means[at] - mean;
            n2 = __builtin_fmaf(ni, d, n2);
            m2 += __builtin_fmaf(ni * d, d, squares[at]);
        });
        n2 = sum_group(n2);
        m2 = sum_group(m2);
        const float shift = n2 * of_values;
        if ((t & (T - 1)) == 0 && g == g0 + (t >> p.lg_T)) p.partial[int64_t(image * p.groups + g) * p.chunks + chunk] = float2{mean + shift, __builtin_fmaf(-shift, n2, m2)};
    }
}

// ---- the norm itself: a part of a chunk's rows

// STREAMS: the output goes past the caches, which then keep more of what the statistics read (four images of 512 x 512 x 128 bf16, 268 MB:
// 156 us without, 132 with; one of them, 67 MB: 42 and 40).
template <int TYPE, int V, int ACT, bool STREAMS>
__global__ __launch_bounds__(NORM_MOST_THREADS) void group_norm_apply_kernel(NormParams p) {
    extern __shared__ float2 group[];
    constexpr int SIZE = Kind<TYPE>::SIZE, AHEAD = 4;
    typedef Run<TYPE, V> Values;
    const int threads = blockDim.x, t = threadIdx.x, lanes = p.lanes ? p.lanes : 1;
    // The last chunks first, since the statistics ended with them: what they read is still in the caches.  Each on the XCD that
    // read it: workgroups go to the XCDs in turn.
    const bool turned = p.chunks % 8 == 0;
    const int chunk = turned ? p.chunks - 8 - (blockIdx.x & ~7u) + (blockIdx.x & 7) : blockIdx.x, image = turned ? p.images - 1 - blockIdx.y : blockIdx.y;
    const int in_chunk = blockIdx.z * p.part_rows, first = chunk * p.chunk_rows + in_chunk;
    const int rows = min(min(p.part_rows, p.chunk_rows - in_chunk), p.rows - first);      // may be none
    const int tail = chunk == p.chunks - 1 && blockIdx.z == 0 ? p.tail : 0;
    const char *const x = static_cast<const char *>(p.x) + image * p.image_bytes;
    char *const out = static_cast<char *>(p.out) + image * p.out_image_bytes;
    for (int j0 = 0; j0 < p.pieces; j0 += threads) {
        const int lane = p.lanes ? udiv(t, p.pieces, p.pieces_magic) : 0, j = p.lanes ? t - lane * p.pieces : j0 + t;
        const bool mine = lane < lanes && j < p.pieces;
        const char *from = x + int64_t(first + lane) * p.row_bytes + j * (V * SIZE);
        char *to = out + int64_t(first + lane) * p.out_row_bytes + j * (V * SIZE);
        const int out_step = lanes * p.out_row_bytes, out_steps = AHEAD * out_step;
        // Requests of a batch leave together, the first ahead of the statistics; in the place of rows that are none the last one again.
        const int most = lanes == 1 ? rows - lane : udiv(max(rows - lane, 0) + lanes - 1, lanes, p.lanes_magic);
        int left = mine ? most : 0;
        Values v[AHEAD];
        auto fetch = [&] { static_for<0, AHEAD>([&](auto uc) { v[decltype(uc)::value].load(from + min(decltype(uc)::value, left - 1) * p.step_bytes); }); };
        if (left > 0) fetch();
        int ch = mine ? j * V : 0;
        if (p.S > 1) ch -= udiv(ch, p.c, p.c_magic) * p.c;
        Affine<V> affine(ch, p.c, p.weight, p.bias);
        if (j0 == 0) {
            merge_chunks(p, image, group);
            __syncthreads();
        }
        affine.take(group, ch, p.c, p.d, p.d_magic);
        auto apply = [&](auto uc) __attribute__((always_inline)) {
            constexpr int u = decltype(uc)::value;
            Piece<TYPE, V> a;
            static_for<0, V>([&](auto ec) { a.v[decltype(ec)::value] = v[u].template get<decltype(ec)::value>(); });
            affine.template apply<ACT>(p.act, p.slope, a);
            a.template store<STREAMS>(to + u * out_step, 0, V);
        };
        while (left > AHEAD) {
            static_for<0, AHEAD>(apply);
            from += AHEAD * p.step_bytes;
            to += out_steps;
            left -= AHEAD;
            fetch();
        }
        static_for<0, AHEAD>([&](auto uc) { if (decltype(uc)::value < left) apply(uc); });
        if (mine && lane == 0 && j * V < tail) {
            Piece<TYPE, V> a;
            const int64_t at = int64_t(p.rows) * (p.S * p.c) + j * V;
            a.load_some(x, at, tail - j * V);
            affine.template apply<ACT>(p.act, p.slope, a);
            a.store(out, at, tail - j * V);
        }
        if (p.lanes) break;
    }
}

// ---- host side

// One workgroup of 512 threads a CU: with more, each has its prologue and its reductions, and the caches hold more streams.  us (bf16) at
// 256, 512 and 2048 workgroups: 16384 pixels x 128 channels on 4 images 15.8, 17.4 and 17.4, 65536 x 64 on 2 16.4, 18.9 and 18.7, 262144 x
// 128 on 4 132, 137 and 140; 256 workgroups of 1024 threads: 16.3, 16.9, 144, and 16384 x 128 on 1 13.6 where 512 threads take 11.0.
constexpr int NORM_THREADS = 512, NORM_WORKGROUPS = 256, MOST_CHUNKS = 256;

// Rows, threads and chunks of a call; V: values of a piece (1: a channel a thread, for pixels apart that are no whole pieces).
struct NormPlan {
    NormParams p;
    int V, threads;
};

NormPlan plan_of(const tsx_group_norm *g) {
    NormPlan pl{};
    NormParams &p = pl.p;
    const int whole = g->type == TSX_TYPE_F32 ? 4 : 8, size = int(element_bytes(g->type));
    const bool dense = g->pixel_stride == g->c || g->pixels <= 1;
    const int S = whole / gcd(g->c, whole), n = std::max(g->n, 1), d = g->c / g->groups;
    const int64_t pixel_stride = g->pixels <= 1 ? g->c : g->pixel_stride;
    pl.V = S == 1 || (dense && S * g->c <= NORM_MOST_CHANNELS) ? whole : 1;
    p.S = pl.V == 1 ? 1 : S;
    p.x = g->x_dev;
    p.weight = g->weight_dev;
    p.bias = g->bias_dev;
    p.c = g->c;
    p.groups = g->groups;
    p.d = d;
    p.pixels = int(g->pixels);
    p.epsilon = g->epsilon;
    p.slope = g->slope;
    p.act = g->act;
    p.images = n;
    p.rows = p.pixels / p.S;
    p.tail = (p.pixels - p.rows * p.S) * p.c;
    p.pieces = p.S * p.c / pl.V;
    p.image_bytes = g->image_stride * size;
    p.out_image_bytes = g->pixels * g->c * size;
    p.row_bytes = int(p.S * pixel_stride * size);
    p.out_row_bytes = p.S * p.c * size;
    p.pixel_bytes = int(pixel_stride * size);
    pl.threads = p.pieces <= NORM_THREADS ? NORM_THREADS : NORM_MOST_THREADS;
    p.lanes = p.pieces <= pl.threads ? pl.threads / p.pieces : 0;
    const int side = p.lanes ? p.lanes : 1;
    p.step_bytes = int64_t(side) * p.row_bytes;
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>({ceil_div(NORM_WORKGROUPS, n), int64_t(MOST_CHUNKS), p.rows / (4 * side)}));
    p.chunk_rows = int(std::max<int64_t>(1, ceil_div(p.rows, chunks)));
    p.chunks = int(std::max<int64_t>(1, ceil_div(p.rows, p.chunk_rows)));
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(ceil_div(NORM_WORKGROUPS, int64_t(n) * p.chunks), p.chunk_rows / (4 * side)));
    p.part_rows = int(std::max<int64_t>(1, ceil_div(p.chunk_rows, parts)));
    p.parts = int(std::max<int64_t>(1, ceil_div(p.chunk_rows, p.part_rows)));
    p.of_chunk = float(int64_t(p.chunk_rows) * p.S * d);
    p.of_last = float((g->pixels - int64_t(p.chunks - 1) * p.chunk_rows * p.S) * d);
    p.of_image = float(1.0 / (double(g->pixels) * d));
    p.lg_run = lg_of(gcd(d, pl.V));
    p.pieces_magic = div_magic(p.pieces, NORM_MOST_THREADS);
    p.lanes_magic = div_magic(side, int64_t(p.chunk_rows) + side);
    p.c_magic = div_magic(p.c, NORM_MOST_CHANNELS);
    p.d_magic = div_magic(d, NORM_MOST_CHANNELS);
    // as far as a group's threads have eight entries each (9 pixels x 809 channels in one group: a call 14 us, with 64 threads 22)
    p.lg_T = lg_threads(pl.threads, p.groups, (side + 1) * p.S * (d >> p.lg_run) / 8, 9);
    if (p.lg_T < 6) p.lg_T = lg_threads(pl.threads, p.groups, (side + 1) * p.S * (d >> p.lg_run));
    p.lg_TL = lg_threads(1 << p.lg_T, 1, side);
    p.lg_merge = lg_threads(pl.threads, p.groups, p.chunks);
    return pl;
}

int check(const tsx_group_norm *g, const char *what) {
    TSX_REQUIRE(g, "%s: null argument", what);
    TSX_REQUIRE(g->n >= 0 && g->pixels >= 0 && g->c > 0 && g->groups > 0, "%s: bad extents", what);
    TSX_REQUIRE(g->c % g->groups == 0, "%s: %d channels are no %d groups", what, g->c, g->groups);
    TSX_REQUIRE(g->c <= NORM_MOST_CHANNELS, "%s: %d channels (at most %d)", what, g->c, NORM_MOST_CHANNELS);
    TSX_REQUIRE(is_float_type(g->type), "%s: element type %d (fp32, fp16 or bf16)", what, g->type);
    TSX_REQUIRE(g->n < 65536 && g->pixels < int64_t(1) << 30, "%s: %d images of %lld pixels", what, g->n, (long long)g->pixels);
    TSX_REQUIRE(g->pixels <= 1 || g->pixel_stride >= g->c, "%s: pixels of %d channels overlap at a stride of %lld", what, g->c, (long long)g->pixel_stride);
    TSX_REQUIRE(g->pixels <= 1 || g->pixel_stride <= 1 << 26, "%s: pixels at a stride of %lld (at most 2^26)", what, (long long)g->pixel_stride);
    TSX_REQUIRE(g->n <= 1 || g->image_stride >= 0, "%s: negative image stride", what);
    TSX_REQUIRE(is_token_act(g->act), "%s: activation %d", what, g->act);
    TSX_REQUIRE(g->epsilon >= 0.f, "%s: epsilon is negative or NaN", what);
    TSX_REQUIRE(g->n == 0 || g->pixels == 0 || g->x_dev, "%s: null input", what);
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(g->x_dev) % element_bytes(g->type) == 0, "%s: pointer is no multiple of its elements", what);
    return 0;
}

size_t workspace_bytes(const tsx_group_norm *g) {
    return size_t(g->n) * plan_of(g).p.chunks * g->groups * sizeof(float2);
}

template <int TYPE, int V>
int launch_statistics(const NormPlan &pl, hipStream_t stream) {
    const NormParams &p = pl.p;
    const size_t lds = size_t((p.lanes ? p.lanes : 1) + 1) * ((p.S * (p.c >> p.lg_run)) | 1) * 2 * sizeof(float);
    if (lds > 64 * 1024) {
        const int rc = grant_lds(reinterpret_cast<const void *>(group_norm_statistics_kernel<TYPE, V>), 136 * 1024);
        if (rc) return rc;
    }
    hipLaunchKernelGGL((group_norm_statistics_kernel<TYPE, V>), dim3(unsigned(p.chunks), unsigned(p.images)), dim3(pl.threads), lds, stream, p);
    TSX_LAUNCH_CHECK("group_norm_statistics_kernel");
    return 0;
}

template <int TYPE, int V>
int launch_apply(const NormPlan &pl, hipStream_t stream) {
    const NormParams &p = pl.p;
    // what a consumer would find in the caches is worth more where they hold it all (256 MB, of input and output)
    const bool streams = p.images * p.out_image_bytes >= int64_t(96) << 20;
    with_act(p.act, [&](auto act) {
        const auto kernel = streams ? group_norm_apply_kernel<TYPE, V, decltype(act)::value, V != 1> : group_norm_apply_kernel<TYPE, V, decltype(act)::value, false>;
        hipLaunchKernelGGL(kernel, dim3(unsigned(p.chunks), unsigned(p.images), unsigned(p.parts)), dim3(pl.threads), size_t(p.groups) * sizeof(float2), stream, p);
    });
    TSX_LAUNCH_CHECK("group_norm_apply_kernel");
    return 0;
}

template <int TYPE>
int run(const NormPlan &pl, hipStream_t stream) {
    constexpr int V = TYPE == TSX_TYPE_F32 ? 4 : 8;
    int rc = pl.V == 1 ? launch_statistics<TYPE, 1>(pl, stream) : launch_statistics<TYPE, V>(pl, stream);
    if (rc) return rc;
    if (pl.p.q) return group_norm_tokens(pl.p, TYPE, stream);
    return pl.V == 1 ? launch_apply<TYPE, 1>(pl, stream) : launch_apply<TYPE, V>(pl, stream);
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
    if (!q) {
        bool taken = false;
        rc = group_norm_held(g, pl.p, stream, &taken);
        if (taken) return rc;
    }
    return g->type == TSX_TYPE_F32 ? run<TSX_TYPE_F32>(pl, stream) : g->type == TSX_TYPE_F16 ? run<TSX_TYPE_F16>(pl, stream) : run<TSX_TYPE_BF16>(pl, stream);
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
