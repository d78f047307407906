// What the kernels of the group norm share (group_norm.hip, group_norm_tokens.hip): how an image's pixels are dealt out, and its
// statistics from those of its chunks.
#pragma once
#include "elements.hpp"

namespace tsx {

constexpr int NORM_MOST_CHANNELS = 8192, NORM_MOST_THREADS = 1024;

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

// the norm's values as int8 tokens, from the statistics in p.partial
int group_norm_tokens(const NormParams &p, int type, hipStream_t stream);

// the norm in one launch, where that serves the call: *taken says whether
int group_norm_held(const tsx_group_norm *g, const NormParams &p, hipStream_t stream, bool *taken);

inline int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

#ifdef __HIPCC__

constexpr int ANY_ACT = -1;            // an activation that is looked up for each piece

template <int TYPE>
struct Kind {
    static constexpr int SIZE = TYPE == TSX_TYPE_F32 ? 4 : 2;
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

// Where a workgroup of the two kernels below works: `of` = n * chunks places, consecutive ones on consecutive XCDs.
struct Place {
    int64_t image;
    int chunk;
    __device__ __forceinline__ Place(const NormParams &p, int at) : image(at / p.chunks), chunk(at % p.chunks) {}
};

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

// One piece's V values as V / run entries: neighbours of one group, `run` of them, become one.
template <int V, class Join>
__device__ __forceinline__ void join_runs(int run, Join &&join) {
    if constexpr (V >= 2) { if (run % 2 == 0) static_for<0, V / 2>([&](auto ic) { join(std::integral_constant<int, 2 * decltype(ic)::value>{}, std::integral_constant<int, 1>{}); }); }
    if constexpr (V >= 4) { if (run % 4 == 0) static_for<0, V / 4>([&](auto ic) { join(std::integral_constant<int, 4 * decltype(ic)::value>{}, std::integral_constant<int, 2>{}); }); }
    if constexpr (V >= 8) { if (run % 8 == 0) static_for<0, V / 8>([&](auto ic) { join(std::integral_constant<int, 8 * decltype(ic)::value>{}, std::integral_constant<int, 4>{}); }); }
}

// Mean, scale and bias of the V channels of piece j of a row
template <int V>
struct Affine {
    float mean[V], scale[V], shift[V];
    // from channel ch on, of c that follow one another and begin with a group's first one; group[0]: that group
    __device__ __forceinline__ Affine(const NormParams &p, const float2 *group, int ch, int c, const float *weight, const float *bias) {
        int g = ch / p.d, left = (g + 1) * p.d - ch;         // channels left in the group
        int at[V];
        static_for<0, V>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            const float2 stat = group[g];
            mean[e] = stat.x;
            scale[e] = stat.y;
            at[e] = ch++;
            if (--left == 0) {
                left = p.d;
                ++g;
                if (ch == c) g = ch = 0;
            }
        });
        // all requests behind one branch each: behind branches of their own they would wait for one another
        static_for<0, V>([&](auto ec) { shift[decltype(ec)::value] = 0.f; });
        if (bias) static_for<0, V>([&](auto ec) { shift[decltype(ec)::value] = bias[at[decltype(ec)::value]]; });
        if (weight) {
            float w[V];
            static_for<0, V>([&](auto ec) { w[decltype(ec)::value] = weight[at[decltype(ec)::value]]; });
            static_for<0, V>([&](auto ec) { scale[decltype(ec)::value] *= w[decltype(ec)::value]; });
        }
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
