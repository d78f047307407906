// What the kernels of the group norm share (group_norm.hip, group_norm_tokens.hip): how an image's pixels are dealt out, and its
// statistics from those of its chunks.
#pragma once
#include "elements.hpp"
#include "igemm_i8.hpp"

namespace tsx {

constexpr int NORM_MOST_CHANNELS = 8192, NORM_MOST_THREADS = 1024;

struct NormParams {
    const void *x;
    void *out;
    int8_t *q;
    float *scales;
    const float *weight, *bias;
    float2 *partial;                   // [n][groups][chunks]: mean, squares around it (a group's chunks are read together)
    int64_t pixels, image_stride, pixel_stride;
    int64_t rows;                      // whole rows of S pixels
    int c, groups, d;
    int S, pieces;                     // pixels of a row; pieces of a row
    int lanes;                         // rows that a workgroup's threads take side by side (0: pieces in turns)
    int run, lg_run;                   // neighbours of a piece that lie in one group, whichever piece: a power of two
    int chunks;                        // of an image's rows: a workgroup's share of the statistics
    int places, parts;                 // n * chunks; workgroups that share a chunk of the norm itself
    int64_t chunk_rows, part_rows, part_pixels;
    float epsilon, slope;
    int act;
    unsigned pieces_magic, chunks_magic, places_magic, d_magic;      // udiv
    int lg_T, lg_TL;                   // threads that sum up one group's entries, of them on lanes of their own
    int lg_merge;                      // threads that sum up one group's chunks
};

// the norm's values as int8 tokens, from the statistics in p.partial
int group_norm_tokens(const NormParams &p, int type, hipStream_t stream);

// the norm in one launch, where that serves the call: *taken says whether
int group_norm_held(const tsx_group_norm *g, const NormParams &p, hipStream_t stream, bool *taken);

// Threads, as a power of two, that work on one group where `threads` share `groups` of `entries` each.
inline int lg_threads(int threads, int groups, int entries) {
    int lg = 0;
    while (lg < 6 && (groups << lg) < threads && (1 << lg) < entries) ++lg;
    return lg;
}

inline int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

#ifdef __HIPCC__

constexpr int ANY_ACT = -1;            // an activation that is looked up for each piece

template <int TYPE>
struct Kind {
    static constexpr int SIZE = TYPE == TSX_TYPE_F32 ? 4 : 2;
};

// Where a workgroup of the two kernels below works: `of` = n * chunks places, consecutive ones on consecutive XCDs.
struct Place {
    int64_t image;
    int chunk;
    __device__ __forceinline__ Place(const NormParams &p, int at) {
        const int i = udiv(at, p.chunks, p.chunks_magic);
        image = i;
        chunk = at - i * p.chunks;
    }
};

// Mean and 1 / sqrt(variance + epsilon) of the groups of one image, into LDS, from the chunks' means and squares, in one pass around
// the first chunk's mean: n_k (mean_k - mean_0)^2 is part of the variance, so what cancels is at most `chunks` times it.
__device__ __forceinline__ void merge_chunks(const NormParams &p, int64_t image, float2 *group) {
    const float whole = float(p.chunk_rows) * float(p.S) * float(p.d);
    const float last = float(p.pixels - (p.chunks - 1) * p.chunk_rows * p.S) * float(p.d);
    const float of_total = 1.f / (float(p.pixels) * float(p.d));
    const int lg = p.lg_merge, T = 1 << lg;
    for (int g0 = 0; g0 < p.groups; g0 += blockDim.x >> lg) {
        const int g = g0 + (threadIdx.x >> lg);
        if (g >= p.groups) continue;                         // T threads agree
        const float2 *const partial = p.partial + (image * p.groups + g) * p.chunks;
        const float about = partial[0].x;
        float s = 0.f, m2 = 0.f;
        constexpr int AHEAD = 8;                             // requests that leave together
        for (int k = threadIdx.x & (T - 1); k < p.chunks; k += AHEAD * T) {
            float2 part[AHEAD];
            static_for<0, AHEAD>([&](auto uc) { part[decltype(uc)::value] = partial[min(k + decltype(uc)::value * T, p.chunks - 1)]; });
            static_for<0, AHEAD>([&](auto uc) {
                constexpr int u = decltype(uc)::value;
                const int at = k + u * T;
                const float n = at < p.chunks - 1 ? whole : last, d = part[u].x - about;
                if (at < p.chunks) {
                    s = __builtin_fmaf(n, d, s);
                    m2 += __builtin_fmaf(n * d, d, part[u].y);
                }
            });
        }
        s = sum_over_lanes(s, lg);
        m2 = sum_over_lanes(m2, lg);
        const float shift = s * of_total, variance = fmaxf(__builtin_fmaf(-shift, s, m2), 0.f) * of_total;
        // a NaN among the squares stays one (fmaxf drops it)
        if ((threadIdx.x & (T - 1)) == 0) group[g] = float2{about + shift, 1.f / sqrtf((m2 == m2 ? variance : m2) + p.epsilon)};
    }
}

// One piece of V values: whole, or of the image's last, incomplete row.  `at`: values from the image's first.
template <int TYPE, int V>
struct Piece {
    float v[V];
    __device__ __forceinline__ void load(const char *image, int64_t at) {
        Run<TYPE, V> r;
        r.load(image + at * Kind<TYPE>::SIZE);
        static_for<0, V>([&](auto ec) { v[decltype(ec)::value] = r.template get<decltype(ec)::value>(); });
    }
    __device__ __forceinline__ void load_some(const char *image, int64_t at, int left) {
        Run<TYPE, V> r;
        r.load_some(image + at * Kind<TYPE>::SIZE, left);
        static_for<0, V>([&](auto ec) { v[decltype(ec)::value] = r.template get<decltype(ec)::value>(); });
    }
    __device__ __forceinline__ void store(char *out, int64_t at, int left) const {
        Run<TYPE, V> r;
        r.set(v);
        if (left >= V) r.store(out + at * Kind<TYPE>::SIZE);
        else r.store_some(out + at * Kind<TYPE>::SIZE, left);
    }
};

// One piece's V values as V / run entries: neighbours of one group, `run` of them, become one.
template <int V, class Join>
__device__ __forceinline__ void join_runs(int run, Join &&join) {
    if constexpr (V >= 2) { if (run % 2 == 0) static_for<0, V / 2>([&](auto ic) { join(std::integral_constant<int, 2 * decltype(ic)::value>{}, std::integral_constant<int, 1>{}); }); }
    if constexpr (V >= 4) { if (run % 4 == 0) static_for<0, V / 4>([&](auto ic) { join(std::integral_constant<int, 4 * decltype(ic)::value>{}, std::integral_constant<int, 2>{}); }); }
    if constexpr (V >= 8) { if (run % 8 == 0) static_for<0, V / 8>([&](auto ic) { join(std::integral_constant<int, 8 * decltype(ic)::value>{}, std::integral_constant<int, 4>{}); }); }
}

// Mean, scale and bias of V channels in a row, from channel ch on, of c that follow one another (behind the last one: the first) and
// begin with a group's first one.  weight and bias: of those channels, or null.  The vectors are requested by the constructor, ahead of
// the statistics, all behind one branch each: behind branches of their own they would wait for one another.
template <int V>
struct Affine {
    float mean[V], scale[V], shift[V];
    __device__ __forceinline__ Affine(int ch, int c, const float *weight, const float *bias) {
        int at[V];
        static_for<0, V>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            at[e] = ch++;
            if (ch == c) ch = 0;
            scale[e] = 1.f;
            shift[e] = 0.f;
        });
        if (bias) static_for<0, V>([&](auto ec) { shift[decltype(ec)::value] = bias[at[decltype(ec)::value]]; });
        if (weight) static_for<0, V>([&](auto ec) { scale[decltype(ec)::value] = weight[at[decltype(ec)::value]]; });
    }
    // group[0]: the statistics of the first of the c channels
    __device__ __forceinline__ void take(const float2 *group, int ch, int c, int d, unsigned d_magic) {
        int g = udiv(ch, d, d_magic), left = (g + 1) * d - ch;             // channels left in the group
        static_for<0, V>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            const float2 stat = group[g];
            mean[e] = stat.x;
            scale[e] *= stat.y;
            ++ch;
            if (--left == 0) {
                left = d;
                ++g;
                if (ch == c) g = ch = 0;
            }
        });
    }
    template <int ACT, int TYPE>
    __device__ __forceinline__ void apply(int act, float slope, Piece<TYPE, V> &a) const {
        static_for<0, V>([&](auto ec) { constexpr int e = decltype(ec)::value; a.v[e] = __builtin_fmaf(a.v[e] - mean[e], scale[e], shift[e]); });
        if constexpr (ACT == ANY_ACT) activate_tokens(a.v, act, slope);
        else activate_as<ACT>(a.v, slope);
    }
};

#endif  // __HIPCC__

}  // namespace tsx
