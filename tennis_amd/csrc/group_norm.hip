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
    int run;                           // neighbours of a piece that lie in one group, whichever piece
    int chunks;                        // of an image's rows: a workgroup's share of the statistics
    int places, parts;                 // n * chunks; workgroups that share a chunk of the norm itself
    int64_t chunk_rows, part_rows, part_pixels;
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

// The sum over T consecutive lanes, T a power of two, in every one of them.
__device__ __forceinline__ float sum_of(float v, int T) {
    for (int far = 1; far < T; far *= 2) v += __shfl_xor(v, far);
    return v;
}
// Threads that work on one group where `threads` share `groups` of `entries` each.
__device__ __forceinline__ int threads_a_group(int threads, int groups, int entries) {
    int T = 1;
    while (T < 64 && T * groups < threads && T < entries) T *= 2;
    return T;
}

// One piece's V values as V / run entries: neighbours of one group, `run` of them, become one.
template <int V, class Join>
__device__ __forceinline__ void join_runs(int run, Join &&join) {
    if constexpr (V >= 2) { if (run % 2 == 0) static_for<0, V / 2>([&](auto ic) { join(std::integral_constant<int, 2 * decltype(ic)::value>{}, std::integral_constant<int, 1>{}); }); }
    if constexpr (V >= 4) { if (run % 4 == 0) static_for<0, V / 4>([&](auto ic) { join(std::integral_constant<int, 4 * decltype(ic)::value>{}, std::integral_constant<int, 2>{}); }); }
    if constexpr (V >= 8) { if (run % 8 == 0) static_for<0, V / 8>([&](auto ic) { join(std::integral_constant<int, 8 * decltype(ic)::value>{}, std::integral_constant<int, 4>{}); }); }
}

// Where a workgroup of the two kernels below works: `of` = n * chunks places, consecutive ones on consecutive XCDs.
struct Place {
    int64_t image;
    int chunk;
    __device__ __forceinline__ Place(const NormParams &p, int at) : image(at / p.chunks), chunk(at % p.chunks) {}
};

// ---- statistics of a chunk of rows of one image

template <int TYPE, int V>
__global__ __launch_bounds__(512) void group_norm_statistics_kernel(NormParams p) {
    extern __shared__ float entries[];                       // [lanes + 1][S * c / run] means, then squares
    const int threads = blockDim.x, t = threadIdx.x;
    const int lanes = p.lanes ? p.lanes : 1, row_values = p.S * p.c, row_entries = row_values / p.run;
    float *const means = entries, *const squares = means + (lanes + 1) * row_entries;
    const Place place(p, blockIdx.x);
    const char *const x = static_cast<const char *>(p.x) + place.image * p.image_stride * Kind<TYPE>::SIZE;
    const int64_t row_stride = p.S * p.pixel_stride;
    const int64_t first = place.chunk * p.chunk_rows, end = min(first + p.chunk_rows, p.rows);
    // the incomplete row, with the last chunk: entries of its own behind the lanes'
    const int tail = place.chunk == p.chunks - 1 ? int(p.pixels - p.rows * p.S) * p.c : 0;
    auto leave = [&](int lane, int j, const float (&mean)[V], const float (&square)[V]) __attribute__((always_inline)) {
        static_for<0, V>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            if (e % p.run == 0) {
                const int at = lane * row_entries + (j * V + e) / p.run;
                means[at] = mean[e];
                squares[at] = square[e];
            }
        });
    };
    // runs of values of one count become one entry: the mean of their means, their squares and n / 2 of the squared difference
    auto join = [&](float (&mean)[V], float (&square)[V], float count) __attribute__((always_inline)) {
        join_runs<V>(p.run, [&](auto ac, auto fc) {
            constexpr int a = decltype(ac)::value, b = a + decltype(fc)::value;
            const float d = mean[b] - mean[a];
            square[a] = square[a] + square[b] + (0.5f * decltype(fc)::value * count) * (d * d);
            mean[a] = __builtin_fmaf(d, 0.5f, mean[a]);
        });
    };
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
            constexpr int AHEAD = 8;
            for (; row + (AHEAD - 1) * lanes < end; row += AHEAD * lanes) {
                Piece<TYPE, V> a[AHEAD];
                static_for<0, AHEAD>([&](auto uc) { a[decltype(uc)::value].load(x, (row + decltype(uc)::value * lanes) * row_stride + j * V); });
                static_for<0, AHEAD>([&](auto uc) { take(a[decltype(uc)::value]); });
                count += AHEAD;
            }
            for (; row < end; row += lanes) {
                Piece<TYPE, V> a;
                a.load(x, row * row_stride + j * V);
                take(a);
                count += 1.f;
            }
            const float of_count = count > 0.f ? 1.f / count : 0.f;
            static_for<0, V>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                const float m = sum[e] * of_count;
                square[e] = fmaxf(__builtin_fmaf(-m, sum[e], square[e]), 0.f);
                base[e] += m;
            });
            join(base, square, count);
            leave(lane, j, base, square);
            if (lane == 0) {
                const int left = tail - j * V;
                Piece<TYPE, V> a;
                static_for<0, V>([&](auto ec) { a.v[decltype(ec)::value] = square[decltype(ec)::value] = 0.f; });
                if (left > 0) a.load_some(x, p.rows * row_values + j * V, left);
                join(a.v, square, 1.f);
                leave(lanes, j, a.v, square);
            }
        }
        if (p.lanes) break;
    }
    __syncthreads();
    // T threads a group: its entries [lane][pixel of the row][run of the group's channels], whose counts follow from their places
    const int group_entries = p.d / p.run, lane_entries = p.S * group_entries, own = (lanes + (tail ? 1 : 0)) * lane_entries;
    const int T = threads_a_group(threads, p.groups, own), tail_entries = tail / p.run;
    const int64_t rows_here = end > first ? end - first : 0;
    for (int g0 = 0; g0 < p.groups; g0 += threads / T) {
        const int g = g0 + t / T;
        if (g >= p.groups) continue;                         // T threads agree
        auto at_of = [&](int i, float &n) __attribute__((always_inline)) {
            const int lane = i / lane_entries, in_lane = i - lane * lane_entries, pixel = in_lane / group_entries;
            const int in_row = pixel * (p.c / p.run) + g * group_entries + (in_lane - pixel * group_entries);
            n = float(p.run) * (lane < lanes ? float(rows_here > lane ? (rows_here - lane - 1) / lanes + 1 : 0) : in_row < tail_entries ? 1.f : 0.f);
            return lane * row_entries + in_row;
        };
        float n = 0.f, s = 0.f;
        const float about = rows_here ? means[g * group_entries] : means[lanes * row_entries + g * group_entries];
        for (int i = t % T; i < own; i += T) {
            float ni;
            const int at = at_of(i, ni);
            n += ni;
            s = __builtin_fmaf(ni, means[at] - about, s);
        }
        n = sum_of(n, T);
        s = sum_of(s, T);
        const float mean = about + (n > 0.f ? s / n : 0.f);
        float m2 = 0.f;
        for (int i = t % T; i < own; i += T) {
            float ni;
            const int at = at_of(i, ni);
            const float d = means[at] - mean;
            m2 += ni > 0.f ? __builtin_fmaf(ni * d, d, squares[at]) : 0.f;
        }
        m2 = sum_of(m2, T);
        if (t % T == 0) p.partial[int64_t(blockIdx.x) * p.groups + g] = float2{mean, m2};
    }
}

// Mean and 1 / sqrt(variance + epsilon) of the groups of one image, into LDS, from the chunks' means and squares, in one pass around
// the first chunk's mean: n_k (mean_k - mean_0)^2 is part of the variance, so what cancels is at most `chunks` times it.
__device__ __forceinline__ void merge_chunks(const NormParams &p, int64_t image, float2 *group) {
    const float2 *const partial = p.partial + image * p.chunks * p.groups;
    const float whole = float(p.chunk_rows) * float(p.S) * float(p.d);
    const float last = float(p.pixels - (p.chunks - 1) * p.chunk_rows * p.S) * float(p.d);
    const float of_total = 1.f / (float(p.pixels) * float(p.d));
    const int T = threads_a_group(blockDim.x, p.groups, p.chunks);
    for (int g0 = 0; g0 < p.groups; g0 += blockDim.x / T) {
        const int g = g0 + threadIdx.x / T;
        if (g >= p.groups) continue;                         // T threads agree
        const float about = partial[g].x;
        float s = 0.f, m2 = 0.f;
        for (int k = threadIdx.x % T; k < p.chunks; k += T) {
            const float2 part = partial[int64_t(k) * p.groups + g];
            const float n = k == p.chunks - 1 ? last : whole, d = part.x - about;
            s = __builtin_fmaf(n, d, s);
            m2 += __builtin_fmaf(n * d, d, part.y);
        }
        s = sum_of(s, T);
        m2 = sum_of(m2, T);
        const float shift = s * of_total, variance = fmaxf(__builtin_fmaf(-shift, s, m2), 0.f) * of_total;
        // a NaN among the squares stays one (fmaxf drops it)
        if (threadIdx.x % T == 0) group[g] = float2{about + shift, 1.f / sqrtf((m2 == m2 ? variance : m2) + p.epsilon)};
    }
}

// ---- the norm itself: a part of a chunk's rows

template <int TYPE, int V>
__global__ __launch_bounds__(512) void group_norm_apply_kernel(NormParams p) {
    extern __shared__ float2 group[];
    const int threads = blockDim.x, t = threadIdx.x;
    const int lanes = p.lanes ? p.lanes : 1, row_values = p.S * p.c;
    const int at = blockIdx.x % p.places, part = blockIdx.x / p.places;
    // The last chunks first, since the statistics ended with them: what they read is still in the caches.  Each on the XCD that
    // read it.
    const Place place(p, p.places % 8 == 0 ? p.places - 8 - at / 8 * 8 + at % 8 : at);
    merge_chunks(p, place.image, group);
    __syncthreads();
    const char *const x = static_cast<const char *>(p.x) + place.image * p.image_stride * Kind<TYPE>::SIZE;
    char *const out = static_cast<char *>(p.out) + place.image * p.pixels * p.c * Kind<TYPE>::SIZE;
    const int64_t row_stride = p.S * p.pixel_stride;
    const int64_t chunk_end = min((place.chunk + 1) * p.chunk_rows, p.rows);
    const int64_t first = place.chunk * p.chunk_rows + part * p.part_rows, end = min(first + p.part_rows, chunk_end);
    const int tail = place.chunk == p.chunks - 1 && part == 0 ? int(p.pixels - p.rows * p.S) * p.c : 0;
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
            int64_t row = first + lane;
            constexpr int AHEAD = 4;
            for (; row + (AHEAD - 1) * lanes < end; row += AHEAD * lanes) {
                Piece<TYPE, V> a[AHEAD];
                static_for<0, AHEAD>([&](auto uc) { a[decltype(uc)::value].load(x, (row + decltype(uc)::value * lanes) * row_stride + j * V); });
                static_for<0, AHEAD>([&](auto uc) {
                    apply(a[decltype(uc)::value]);
                    a[decltype(uc)::value].store(out, (row + decltype(uc)::value * lanes) * row_values + j * V, V);
                });
            }
            for (; row < end; row += lanes) {
                Piece<TYPE, V> a;
                a.load(x, row * row_stride + j * V);
                apply(a);
                a.store(out, row * row_values + j * V, V);
            }
            if (lane == 0 && j * V < tail) {
                Piece<TYPE, V> a;
                a.load_some(x, p.rows * row_values + j * V, tail - j * V);
                apply(a);
                a.store(out, p.rows * row_values + j * V, tail - j * V);
            }
        }
        if (p.lanes) break;
    }
}

// ---- the norm's values as int8 tokens
//
// L lanes of a wavefront share a pixel, each with P pieces of eight of its channels, which they hold from the load to the store.
// Mean, scale and bias of the channels lie in LDS: 12 bytes a value read from there at HBM's pace are a third of what LDS gives.
template <int TYPE, int L, int P>
__global__ __launch_bounds__(256) void group_norm_tokens_kernel(NormParams p) {
    extern __shared__ float2 group[];                        // [groups], behind them [3][channels in whole pieces]
    constexpr int V = 8, SIZE = Kind<TYPE>::SIZE;
    const int pieces = (p.c + V - 1) / V, width = pieces * V;
    float *const means = reinterpret_cast<float *>(group + (p.groups + 1) / 2 * 2), *const scales = means + width, *const shifts = scales + width;
    const int at = blockIdx.x % p.places, part = blockIdx.x / p.places;
    const Place place(p, p.places % 8 == 0 ? p.places - 8 - at / 8 * 8 + at % 8 : at);
    merge_chunks(p, place.image, group);
    __syncthreads();
    for (int ch = threadIdx.x; ch < width; ch += 256) {
        const float2 g = ch < p.c ? group[ch / p.d] : float2{0.f, 0.f};
        means[ch] = g.x;
        scales[ch] = ch < p.c && p.weight ? g.y * p.weight[ch] : g.y;
        shifts[ch] = ch < p.c && p.bias ? p.bias[ch] : 0.f;
    }
    __syncthreads();
    const int64_t chunk_pixels = p.chunk_rows * p.S, chunk_end = place.chunk == p.chunks - 1 ? p.pixels : (place.chunk + 1) * chunk_pixels;
    const int64_t first = place.chunk * chunk_pixels + part * p.part_pixels, end = part == p.parts - 1 ? chunk_end : min(first + p.part_pixels, chunk_end);
    const int l = threadIdx.x % L;
    const char *const x = static_cast<const char *>(p.x) + place.image * p.image_stride * SIZE;
    for (int64_t base = first; base < end; base += 256 / L) {
        const int64_t pixel = base + threadIdx.x / L;
        const bool there = pixel < end;                      // a pixel's lanes agree
        const char *const from = x + (there ? pixel : end - 1) * p.pixel_stride * SIZE;
        Run<TYPE, V> in[P];
        static_for<0, P>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            const int j = l + i * L;
            in[i].clear();
            if ((j + 1) * V <= p.c) in[i].load(from + j * (V * SIZE));
            else if (j < pieces) in[i].load_some(from + j * (V * SIZE), p.c - j * V);
        });
        float y[P][V];
        unsigned top = 0;
        static_for<0, P>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            const int j = min(l + i * L, pieces - 1);
            static_for<0, 2>([&](auto hc) {
                constexpr int h = 4 * decltype(hc)::value;
                typedef float v4f __attribute__((ext_vector_type(4)));
                const v4f m = *reinterpret_cast<const v4f *>(means + j * V + h), a = *reinterpret_cast<const v4f *>(scales + j * V + h),
                          b = *reinterpret_cast<const v4f *>(shifts + j * V + h);
                static_for<0, 4>([&](auto ec) { constexpr int e = decltype(ec)::value; y[i][h + e] = __builtin_fmaf(in[i].template get<h + e>() - m[e], a[e], b[e]); });
            });
            activate_tokens(y[i], p.act, p.slope);
            if (l + i * L < pieces - 1 || (l + i * L == pieces - 1 && width == p.c))
                static_for<0, V>([&](auto ec) { top = max(top, __builtin_bit_cast(unsigned, y[i][decltype(ec)::value]) & 0x7fffffffu); });
            else if (l + i * L < pieces)
                static_for<0, V>([&](auto ec) {
                    constexpr int e = decltype(ec)::value;
                    if ((pieces - 1) * V + e < p.c) top = max(top, __builtin_bit_cast(unsigned, y[i][e]) & 0x7fffffffu);
                });
        });
#pragma unroll
        for (int far = 1; far < L; far *= 2) top = max(top, unsigned(__shfl_xor(int(top), far)));
        const TokenScale s(__builtin_bit_cast(float, top));
        const int64_t token = place.image * p.pixels + pixel;
        if (there && l == 0) p.scales[token] = s.scale;
        if (there)
            static_for<0, P>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                const int j = l + i * L;
                if (j >= pieces) return;
                unsigned b[V];
                static_for<0, V>([&](auto ec) { constexpr int e = decltype(ec)::value; b[e] = s.bits(__fmul_rn(y[i][e], s.lift)); });
                v2u word = {low_bytes(b[0], b[1], b[2], b[3]), low_bytes(b[4], b[5], b[6], b[7])};
                if (s.reciprocal == 0.f) word = v2u{0, 0};
                int8_t *const to = p.q + token * p.c + j * V;
                if ((j + 1) * V <= p.c) *reinterpret_cast<v2u_any *>(to) = word;
                else static_for<0, V>([&](auto ec) { constexpr int e = decltype(ec)::value; if (j * V + e < p.c) to[e] = int8_t(word[e / 4] >> (8 * (e % 4))); });
            });
    }
}

// ---- host side

constexpr int MOST_CHUNKS = 256;

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
    p.run = gcd(p.d, pl.V);
    pl.threads = p.pieces <= 256 ? 256 : 512;
    p.lanes = p.pieces <= pl.threads ? pl.threads / p.pieces : 0;
    // Statistics: two workgroups a CU, of eight rows a thread at least.  The norm: four.
    const int side = p.lanes ? p.lanes : 1, n = std::max(g->n, 1);
    const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>({ceil_div(512, n), int64_t(MOST_CHUNKS), p.rows / (8 * side)}));
    p.chunk_rows = std::max<int64_t>(1, ceil_div(p.rows, chunks));
    p.chunks = int(std::max<int64_t>(1, ceil_div(p.rows, p.chunk_rows)));
    p.places = n * p.chunks;
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(ceil_div(1024, p.places), p.chunk_rows / (4 * side)));
    p.part_rows = std::max<int64_t>(1, ceil_div(p.chunk_rows, parts));
    p.parts = int(std::max<int64_t>(1, ceil_div(p.chunk_rows, p.part_rows)));
    p.part_pixels = p.part_rows * p.S;
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
int launch_statistics(const NormPlan &pl, hipStream_t stream) {
    const NormParams &p = pl.p;
    const size_t lds = size_t((p.lanes ? p.lanes : 1) + 1) * (p.S * p.c / p.run) * 2 * sizeof(float);
    if (lds > 64 * 1024)
        TSX_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(group_norm_statistics_kernel<TYPE, V>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    hipLaunchKernelGGL((group_norm_statistics_kernel<TYPE, V>), dim3(unsigned(p.places)), dim3(pl.threads), lds, stream, p);
    TSX_LAUNCH_CHECK("group_norm_statistics_kernel");
    return 0;
}

template <int TYPE, int V>
int launch_apply(const NormPlan &pl, hipStream_t stream) {
    const NormParams &p = pl.p;
    hipLaunchKernelGGL((group_norm_apply_kernel<TYPE, V>), dim3(unsigned(p.places) * unsigned(p.parts)), dim3(pl.threads), size_t(p.groups) * sizeof(float2), stream, p);
    TSX_LAUNCH_CHECK("group_norm_apply_kernel");
    return 0;
}

template <int TYPE, int L, int P>
int launch_tokens(const NormParams &p, hipStream_t stream) {
    const size_t lds = size_t(round_up(p.groups, 2)) * sizeof(float2) + size_t(round_up(p.c, 8)) * 3 * sizeof(float);
    if (lds > 64 * 1024)
        TSX_HIP(hipFuncSetAttribute(reinterpret_cast<const void *>(group_norm_tokens_kernel<TYPE, L, P>), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    hipLaunchKernelGGL((group_norm_tokens_kernel<TYPE, L, P>), dim3(unsigned(p.places) * unsigned(p.parts)), dim3(256), lds, stream, p);
    TSX_LAUNCH_CHECK("group_norm_tokens_kernel");
    return 0;
}

template <int TYPE>
int tokens(const NormParams &p, hipStream_t stream) {
    // the fewest lanes that hold a pixel in at most five pieces each
    const int pieces = int(ceil_div(p.c, 8));
    if (pieces <= 4) return launch_tokens<TYPE, 4, 1>(p, stream);
    if (pieces <= 8) return launch_tokens<TYPE, 4, 2>(p, stream);
    if (pieces <= 16) return launch_tokens<TYPE, 8, 2>(p, stream);
    if (pieces <= 24) return launch_tokens<TYPE, 8, 3>(p, stream);
    if (pieces <= 40) return launch_tokens<TYPE, 8, 5>(p, stream);
    if (pieces <= 48) return launch_tokens<TYPE, 16, 3>(p, stream);
    if (pieces <= 80) return launch_tokens<TYPE, 16, 5>(p, stream);
    if (pieces <= 96) return launch_tokens<TYPE, 32, 3>(p, stream);
    if (pieces <= 160) return launch_tokens<TYPE, 32, 5>(p, stream);
    if (pieces <= 192) return launch_tokens<TYPE, 64, 3>(p, stream);
    if (pieces <= 320) return launch_tokens<TYPE, 64, 5>(p, stream);
    if (pieces <= 512) return launch_tokens<TYPE, 64, 8>(p, stream);
    return launch_tokens<TYPE, 64, 16>(p, stream);
}

template <int TYPE>
int run(const NormPlan &pl, hipStream_t stream) {
    constexpr int V = TYPE == TSX_TYPE_F32 ? 4 : 8;
    int rc = pl.V == 1 ? launch_statistics<TYPE, 1>(pl, stream) : launch_statistics<TYPE, V>(pl, stream);
    if (rc) return rc;
    if (pl.p.q) return tokens<TYPE>(pl.p, stream);
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
    return g->type == TSX_TYPE_F32 ? run<TSX_TYPE_F32>(pl, stream) : g->type == TSX_TYPE_F16 ? run<TSX_TYPE_F16>(pl, stream)
                                                                                                : run<TSX_TYPE_BF16>(pl, stream);
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
