// What the kernels of the group norm share (group_norm.hip, group_norm_held.hip, group_norm_tokens.hip): how an image's pixels are dealt out, and its
// statistics from those of its chunks.
#pragma once
#include "elements.hpp"
#include "igemm_i8.hpp"

namespace tsx {

constexpr int NORM_MOST_CHANNELS = 8192, NORM_MOST_THREADS = 1024;

// Everything a kernel would otherwise work out from the sizes: sixteen wavefronts share a CU's scalar unit, and a prologue of 600
// instructions, most of them 64-bit products of strides, kept the last of them waiting for 8 us.
struct NormParams {
    const void *x;
    void *out;
    int8_t *q;
    float *scales;
    const float *weight, *bias;
    float2 *partial;                   // [n][groups][chunks]: mean, squares around it (a group's chunks are read together)
    int64_t image_bytes, out_image_bytes, step_bytes;      // from image to image; from a thread's row to its next one
    int c, groups, d, pixels;
    int S, pieces, rows;               // pixels of a row; pieces of a row; whole rows of an image
    int row_bytes, out_row_bytes, pixel_bytes;
    int lanes;                         // rows that a workgroup's threads take side by side (0: pieces in turns)
    int lg_run;                        // neighbours of a piece that lie in one group, whichever piece: 2^lg_run
    int images, chunks, parts;         // chunks of an image's rows: a workgroup's share of the statistics; parts of them: of the norm
    int chunk_rows, part_rows, part_pixels;
    int tail;                          // values of an image behind its last whole row
    int act;
    float epsilon, slope;
    float of_chunk, of_last, of_image; // values of a group in a chunk, in the last one; 1 / those in an image
    unsigned pieces_magic, lanes_magic, c_magic, d_magic;  // udiv
    int lg_T, lg_TL;                   // threads that sum up one group's entries, of them on lanes of their own
    int lg_merge;                      // threads that sum up one group's chunks
};

// the norm's values as int8 tokens, from the statistics in p.partial
int group_norm_tokens(const NormParams &p, int type, hipStream_t stream);

// the norm in one launch, where that serves the call: *taken says whether
int group_norm_held(const tsx_group_norm *g, const NormParams &p, hipStream_t stream, bool *taken);

// Threads, as a power of two and at most 2^most, that work on one group where `threads` share `groups` of `entries` each.
inline int lg_threads(int threads, int groups, int entries, int most = 6) {
    int lg = 0;
    while (lg < most && (groups << lg) < threads && (1 << lg) < entries) ++lg;
    return lg;
}

inline int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

#ifdef __HIPCC__

constexpr int ANY_ACT = -1;            // an activation that is looked up for each piece

template <int TYPE>
struct Kind {
    static constexpr int SIZE = TYPE == TSX_TYPE_F32 ? 4 : 2;
};

// 1 / sqrt(v) by the hardware's, within a step; its argument is no denormal
__device__ __forceinline__ float reciprocal_root(float v) {
    const bool tiny = v < 0x1p-100f;
    return __fmul_rn(__builtin_amdgcn_rsqf(tiny ? __fmul_rn(v, 0x1p100f) : v), tiny ? 0x1p50f : 1.f);
}

// 1 / sqrt(variance + epsilon) of an image's group.  Squares that left fp32, of which an infinity or a NaN is left, make it NaN: 1 / infinity
// would make the group its bias.
__device__ __forceinline__ float root_of(float squares, const NormParams &p) {
    const float r = reciprocal_root(__builtin_fmaf(fmaxf(squares, 0.f), p.of_image, p.epsilon));
    return squares < __builtin_inff() ? r : __builtin_nanf("");
}

// Mean and 1 / sqrt(variance + epsilon) of the groups of one image, into LDS, from the chunks' means and squares, in one pass around
// the average of the means that a group's threads request first, 4 T of them or all.  n_k (mean_k - average)^2 is part of the variance but for
// the average's own distance from the mean, of which a chunk far from the rest makes a (4 T)-th of its distance at most: what cancels is within
// chunks / (4 T)^2 times the variance, 16 for one thread a group and at most one from four threads on.  (Around one chunk's mean it is `chunks`
// times the variance where that chunk is the far one.  A second pass instead, around the mean, takes 0.2 us more.)
__device__ __forceinline__ void merge_chunks(const NormParams &p, int image, float2 *group) {
    const int lg = p.lg_merge, T = 1 << lg, t = threadIdx.x & (T - 1);
    const float2 *const partials = p.partial + int64_t(image * p.groups) * p.chunks;
    const float of_near = __builtin_amdgcn_rcpf(float(min(4 * T, p.chunks)));
    for (int g = threadIdx.x >> lg; g < p.groups; g += blockDim.x >> lg) {      // T threads agree
        const float2 *const partial = partials + g * p.chunks;
        float2 part[4];
        auto fetch = [&](int k) __attribute__((always_inline)) {               // four requests that leave together
            static_for<0, 4>([&](auto uc) { part[decltype(uc)::value] = partial[min(k + decltype(uc)::value * T, p.chunks - 1)]; });
        };
        float about = partial[0].x, off = 0.f, s = 0.f, m2 = 0.f;
        fetch(t);
        static_for<0, 4>([&](auto uc) { if (t + decltype(uc)::value * T < p.chunks) off += part[decltype(uc)::value].x - about; });
        about += sum_over_lanes(off * of_near, lg);
        for (int k = t; k < p.chunks; k += 4 * T) {
            if (k != t) fetch(k);
            static_for<0, 4>([&](auto uc) {
                constexpr int u = decltype(uc)::value;
                const int at = k + u * T;
                const float n = at < p.chunks - 1 ? p.of_chunk : p.of_last, d = part[u].x - about;
                if (at < p.chunks) {
                    s = __builtin_fmaf(n, d, s);
                    m2 += __builtin_fmaf(n * d, d, part[u].y);
                }
            });
        }
        s = sum_over_lanes(s, lg);
        m2 = sum_over_lanes(m2, lg);
        const float shift = s * p.of_image;
        if (t == 0) group[g] = float2{about + shift, root_of(__builtin_fmaf(-shift, s, m2), p)};
    }
}

// One piece of V values: whole, or of the image's last, incomplete row.  `at`: values from the image's first.
template <int TYPE, int V>
struct Piece {
    float v[V];
    __device__ __forceinline__ void load_some(const char *image, int64_t at, int left) {
        Run<TYPE, V> r;
        r.load_some(image + at * Kind<TYPE>::SIZE, left);
        static_for<0, V>([&](auto ec) { v[decltype(ec)::value] = r.template get<decltype(ec)::value>(); });
    }
    template <bool STREAMS = false>
    __device__ __forceinline__ void store(char *out, int64_t at, int left) const {
        Run<TYPE, V> r;
        r.set(v);
        if (left >= V) r.template store<STREAMS>(out + at * Kind<TYPE>::SIZE);
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
        static_for<0, V>([&](auto ec) {
            scale[decltype(ec)::value] = 1.f;
            shift[decltype(ec)::value] = 0.f;
        });
        const bool wraps = ch + V > c;
        auto load = [&](const float *from, float (&to)[V]) __attribute__((always_inline)) {
            if (wraps) {
                static_for<0, V>([&](auto ec) { const int at = ch + decltype(ec)::value; to[decltype(ec)::value] = from[at - (at >= c ? at / c * c : 0)]; });
            } else if constexpr (V % 4 == 0) {
                typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
                static_for<0, V / 4>([&](auto gc) {
                    constexpr int g = decltype(gc)::value;
                    const v4f v = *reinterpret_cast<const v4f_any *>(from + ch + 4 * g);
                    static_for<0, 4>([&](auto jc) { to[4 * g + decltype(jc)::value] = v[decltype(jc)::value]; });
                });
            } else {
                static_for<0, V>([&](auto ec) { to[decltype(ec)::value] = from[ch + decltype(ec)::value]; });
            }
        };
        if (bias) load(bias, shift);
        if (weight) load(weight, scale);
    }
    // group[0]: the statistics of the first of the c channels
    __device__ __forceinline__ void take(const float2 *group, int ch, int c, int d, unsigned d_magic) {
        int g = udiv(ch, d, d_magic), left = (g + 1) * d - ch;             // channels left in the group
        if (d % V == 0) {                                    // uniform: a piece lies in one group
            const float2 stat = group[g];
            static_for<0, V>([&](auto ec) {
                mean[decltype(ec)::value] = stat.x;
                scale[decltype(ec)::value] *= stat.y;
            });
            return;
        }
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
        if constexpr (ACT == ANY_ACT) activate_tokens<TYPE>(a.v, act, slope);
        else activate_as<TYPE, ACT>(a.v, slope);
    }
};

#endif  // __HIPCC__

}  // namespace tsx
