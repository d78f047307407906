// The group norm's values as int8 tokens: a pixel's largest value decides its scale, so a pixel stays with one wavefront.
//
// Bound: HBM, one read and half of a write behind the statistics' read: 64 x 64 x 320 bf16 on 8 images 10.2 us behind 7.6 at the least, as much by the
// prologue (the vectors into LDS, the chunks' statistics) as by its 31 MB.
//
// L lanes of a wavefront share a pixel, each with P pieces of eight of its channels, which they hold from the load to the store.
// Mean, scale and bias of the channels lie in LDS: 12 bytes a value read from there at HBM's pace are a third of what LDS gives.
#include <algorithm>

#include "group_norm.hpp"

namespace tsx {
namespace {

// us (bf16) at 512, 1024 and 2048: 262144 pixels x 128 channels on 2 images 82.7, 73.2 and 75.0, 1024 x 640 on 32 27.7, 26.3 and 28.7, 4096 x 320
// on 8 18.4, 18.3 and 18.4
constexpr int TOKENS_WORKGROUPS = 1024;

template <int TYPE, int L, int P, int ACT>
__global__ __launch_bounds__(256) void group_norm_tokens_kernel(NormParams p) {
    extern __shared__ float2 group[];                        // [groups], behind them [3][channels in whole pieces]
    constexpr int V = 8, SIZE = Kind<TYPE>::SIZE;
    const int pieces = (p.c + V - 1) / V, width = pieces * V;
    float *const means = reinterpret_cast<float *>(group + (p.groups + 1) / 2 * 2), *const scales = means + width, *const shifts = scales + width;
    const bool turned = p.chunks % 8 == 0;      // as in the norm to its own type
    const int chunk = turned ? p.chunks - 8 - (blockIdx.x & ~7u) + (blockIdx.x & 7) : blockIdx.x, image = turned ? p.images - 1 - blockIdx.y : blockIdx.y;
    const int chunk_pixels = p.chunk_rows * p.S, chunk_first = chunk * chunk_pixels, chunk_end = chunk == p.chunks - 1 ? p.pixels : chunk_first + chunk_pixels;
    const int first = chunk_first + int(blockIdx.z) * p.part_pixels, end = int(blockIdx.z) == p.parts - 1 ? chunk_end : min(first + p.part_pixels, chunk_end);
    const int l = threadIdx.x % L, whole = p.c / V;
    const char *const x = static_cast<const char *>(p.x) + image * p.image_bytes;
    // All requests at once, none behind a branch, where it would be waited for; the first pixels' ahead of the statistics, and the
    // vectors' of the first 1024 channels.
    Run<TYPE, V> in[P];
    auto fetch = [&](int base) __attribute__((always_inline)) {
        const char *const from = x + int64_t(min(base + int(threadIdx.x / L), end - 1)) * p.pixel_bytes;
        if (whole)       // uniform
            static_for<0, P>([&](auto ic) { in[decltype(ic)::value].load(from + min(l + decltype(ic)::value * L, whole - 1) * (V * SIZE)); });
        if (whole != pieces) {   // uniform: the pixel's last, incomplete piece
            Run<TYPE, V> last;
            last.load_some(from + whole * (V * SIZE), p.c - whole * V);
            static_for<0, P>([&](auto ic) { if (l + decltype(ic)::value * L == whole) in[decltype(ic)::value] = last; });
        }
    };
    float w[4], b[4];
    auto fetch_vectors = [&](int ch) __attribute__((always_inline)) {
        static_for<0, 4>([&](auto uc) { w[decltype(uc)::value] = 1.f, b[decltype(uc)::value] = 0.f; });
        if (p.weight) static_for<0, 4>([&](auto uc) { w[decltype(uc)::value] = p.weight[min(ch + 256 * decltype(uc)::value, p.c - 1)]; });
        if (p.bias) static_for<0, 4>([&](auto uc) { b[decltype(uc)::value] = p.bias[min(ch + 256 * decltype(uc)::value, p.c - 1)]; });
    };
    if (first < end) fetch(first);
    fetch_vectors(threadIdx.x);
    merge_chunks(p, image, group);
    __syncthreads();
    for (int ch0 = threadIdx.x; ch0 < width; ch0 += 1024) {
        if (ch0 >= 1024) fetch_vectors(ch0);
        static_for<0, 4>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            const int ch = ch0 + 256 * u;
            if (ch < width) {
                const float2 g = group[udiv(min(ch, p.c - 1), p.d, p.d_magic)];
                means[ch] = g.x;
                scales[ch] = g.y * w[u];
                shifts[ch] = b[u];
            }
        });
    }
    __syncthreads();
    for (int base = first; base < end; base += 256 / L) {
        const int pixel = base + threadIdx.x / L;
        const bool there = pixel < end;                      // a pixel's lanes agree
        if (base != first) fetch(base);
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
            if constexpr (ACT == ANY_ACT) activate_tokens<TSX_TYPE_I8>(y[i], p.act, p.slope);
            else activate_as<TSX_TYPE_I8, ACT>(y[i], p.slope);
            if (l + i * L < pieces - 1 || (l + i * L == pieces - 1 && width == p.c))
                static_for<0, V>([&](auto ec) { top = max(top, __builtin_bit_cast(unsigned, y[i][decltype(ec)::value]) & 0x7fffffffu); });
            else if (l + i * L < pieces)
                static_for<0, V>([&](auto ec) {
                    constexpr int e = decltype(ec)::value;
                    if ((pieces - 1) * V + e < p.c) top = max(top, __builtin_bit_cast(unsigned, y[i][e]) & 0x7fffffffu);
                });
            __builtin_amdgcn_sched_barrier(0);               // a piece at a time: all at once they take twice the registers
        });
        top = over_lanes(top, lg_of(L), [](unsigned a, unsigned b) { return max(a, b); });
        const TokenScale s(__builtin_bit_cast(float, top));
        const int64_t token = int64_t(image) * p.pixels + pixel;
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

template <int TYPE, int L, int P>
int launch_tokens(NormParams p, hipStream_t stream) {
    const int chunk_pixels = p.chunk_rows * p.S, parts = int(std::max<int64_t>(1, std::min<int64_t>(ceil_div(TOKENS_WORKGROUPS, int64_t(p.images) * p.chunks), ceil_div(chunk_pixels, 256 / L))));
    p.part_pixels = int(ceil_div(chunk_pixels, parts));
    p.parts = int(ceil_div(chunk_pixels, p.part_pixels));
    p.lg_merge = lg_threads(256, p.groups, p.chunks);
    const size_t lds = size_t(round_up(p.groups, 2)) * sizeof(float2) + size_t(round_up(p.c, 8)) * 3 * sizeof(float);
    const auto kernel = p.act == TSX_ACT_SILU ? group_norm_tokens_kernel<TYPE, L, P, TSX_ACT_SILU> : group_norm_tokens_kernel<TYPE, L, P, ANY_ACT>;
    if (lds > 64 * 1024) {
        const int rc = grant_lds(reinterpret_cast<const void *>(kernel), 160 * 1024);
        if (rc) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(unsigned(p.chunks), unsigned(p.images), unsigned(p.parts)), dim3(256), lds, stream, p);
    TSX_LAUNCH_CHECK("group_norm_tokens_kernel");
    return 0;
}

template <int TYPE>
int launch(const NormParams &p, hipStream_t stream) {
    // the fewest lanes that hold a pixel in at most five pieces each
    const int pieces = int(ceil_div(p.c, 8));
    if (pieces <= 8) return launch_tokens<TYPE, 4, 2>(p, stream);
    if (pieces <= 16) return launch_tokens<TYPE, 8, 2>(p, stream);
    if (pieces <= 24) return launch_tokens<TYPE, 8, 3>(p, stream);
    if (pieces <= 32) return launch_tokens<TYPE, 8, 4>(p, stream);
    if (pieces <= 40) return launch_tokens<TYPE, 8, 5>(p, stream);
    if (pieces <= 64) return launch_tokens<TYPE, 16, 4>(p, stream);
    if (pieces <= 80) return launch_tokens<TYPE, 16, 5>(p, stream);
    if (pieces <= 128) return launch_tokens<TYPE, 32, 4>(p, stream);
    if (pieces <= 160) return launch_tokens<TYPE, 32, 5>(p, stream);
    if (pieces <= 320) return launch_tokens<TYPE, 64, 5>(p, stream);
    return launch_tokens<TYPE, 64, 16>(p, stream);
}

}  // namespace

int group_norm_tokens(const NormParams &p, int type, hipStream_t stream) {
    return type == TSX_TYPE_F32 ? launch<TSX_TYPE_F32>(p, stream) : type == TSX_TYPE_F16 ? launch<TSX_TYPE_F16>(p, stream) : launch<TSX_TYPE_BF16>(p, stream);
}

}  // namespace tsx
