// Group norm in one launch, where the pixels of a few groups are what one workgroup's registers hold.
//
// A workgroup takes B groups of one image, B * d channels of every pixel: whole pieces of V values.  Its threads hold them from the one
// read to the one write; in between the mean, as the sum over all of them, and then the sums of x - mean and of its square, whose first
// corrects the mean's rounding.  Two kernels read the tensor twice and wait for each other: 8 x 8 x 1280 on 2 images 9.8 us there, 5.2 here.
#include <algorithm>

#include "group_norm.hpp"

namespace tsx {
namespace {

struct HeldParams : NormParams {
    int B, a_image, pieces_a_pixel, held_lanes, bundles, per_xcd;      // a_image: bundles of an image
    int lg_TG;                         // threads that sum up one group's entries; lg_TL of them on lanes of their own
    unsigned pixel_magic, image_magic; // udiv by pieces_a_pixel, by groups / B
};

template <int TYPE, int V, int NP, int ACT>
__global__ __launch_bounds__(NORM_MOST_THREADS) void group_norm_held_kernel(HeldParams p) {
    extern __shared__ float entries[];                       // [2][lanes][pitch]
    __shared__ float2 group[NORM_MOST_THREADS];
    __shared__ float2 waves[NORM_MOST_THREADS / 64];
    constexpr int SIZE = Kind<TYPE>::SIZE;
    const int t = threadIdx.x, lanes = p.held_lanes, channels = p.B * p.d, row_entries = channels >> p.lg_run, pitch = row_entries | 1;
    // consecutive bundles of an image on one XCD: they share cache lines
    const int id = int(blockIdx.x % 8) * p.per_xcd + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= p.per_xcd || id >= p.bundles) return;       // uniform
    const int a_image = p.a_image, image = udiv(id, a_image, p.image_magic), ch0 = (id - image * a_image) * channels, pixels = p.pixels;
    const int lane = udiv(t, p.pieces_a_pixel, p.pixel_magic), j = t - lane * p.pieces_a_pixel;
    const bool mine = lane < lanes;
    // All requests at once, none behind a branch, where it would be waited for: threads without a pixel read another one again.
    const int j_in = mine ? j : 0, lane_in = mine ? lane : 0;
    const char *const x = static_cast<const char *>(p.x) + image * p.image_bytes + (ch0 + j_in * V) * SIZE;
    Run<TYPE, V> v[NP];
    static_for<0, NP>([&](auto ic) { v[decltype(ic)::value].load(x + int64_t(min(lane_in + decltype(ic)::value * lanes, pixels - 1)) * p.pixel_bytes); });
    Affine<V> affine(mine ? j * V : 0, channels, p.weight ? p.weight + ch0 : nullptr, p.bias ? p.bias + ch0 : nullptr);
    // The packed words anew for each pass over them: unpacked once for all three they would be twice as many registers.
    auto again = [&] { static_for<0, NP>([&](auto ic) { v[decltype(ic)::value].renew_words(); }); };
    // `leave`: a thread's V sums into LDS, neighbours of one group added up
    auto leave = [&](float *to, float (&s)[V]) __attribute__((always_inline)) {
        join_runs<V>(1 << p.lg_run, [&](auto ac, auto fc) { constexpr int a = decltype(ac)::value; s[a] += s[a + decltype(fc)::value]; });
        if (!mine) return;
        int at = lane * pitch + (j * V >> p.lg_run);
        static_for<0, V>([&](auto ec) { if ((decltype(ec)::value & ((1 << p.lg_run) - 1)) == 0) to[at++] = s[decltype(ec)::value]; });
    };
    // The sums of both arrays over a group's entries, for the TG threads of that group
    const int TG = 1 << p.lg_TG, TL = 1 << p.lg_TL, TE = TG >> p.lg_TL, group_entries = p.d >> p.lg_run;
    const int g = t >> p.lg_TG, tg = t & (TG - 1), tl = tg & (TL - 1), te = tg >> p.lg_TL;
    const float *const second = entries + lanes * pitch;
    auto gather = [&](bool both) __attribute__((always_inline)) {
        float2 s = {0.f, 0.f};
        if (g < p.B)
            for (int l = tl; l < lanes; l += TL)
                for (int k = te; k < group_entries; k += TE) {
                    const int at = l * pitch + g * group_entries + k;
                    s.x += entries[at];
                    if (both) s.y += second[at];
                }
        s.x = sum_over_lanes(s.x, p.lg_TG);
        if (both) s.y = sum_over_lanes(s.y, p.lg_TG);
        if (TG > 64) {                                     // uniform
            if (t % 64 == 0) waves[t / 64] = s;
            __syncthreads();
            s = float2{0.f, 0.f};
            for (int w = 0; w < TG / 64; ++w) {
                const float2 part = waves[g * (TG / 64) + w];
                s.x += part.x;
                s.y += part.y;
            }
        }
        return s;
    };
    const float of_count = p.of_image;
    float sum[V];
    static_for<0, V>([&](auto ec) { sum[decltype(ec)::value] = 0.f; });
    static_for<0, NP>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if (lane + i * lanes < pixels) static_for<0, V>([&](auto ec) { constexpr int e = decltype(ec)::value; sum[e] += v[i].template get<e>(); });
    });
    leave(entries, sum);
    __syncthreads();
    const float rough = gather(false).x * of_count;
    if (tg == 0 && g < p.B) group[g] = float2{rough, 0.f};
    __syncthreads();
    again();
    float square[V], mean[V];
    {
        int gi = mine ? udiv(j * V, p.d, p.d_magic) : 0, left = (gi + 1) * p.d - j * V;
        static_for<0, V>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            mean[e] = group[gi].x;
            if (--left == 0) left = p.d, gi = min(gi + 1, p.B - 1);
            sum[e] = square[e] = 0.f;
        });
    }
    static_for<0, NP>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if (lane + i * lanes < pixels)
            static_for<0, V>([&](auto ec) {
                constexpr int e = decltype(ec)::value;
                const float d = v[i].template get<e>() - mean[e];
                sum[e] += d;
                square[e] = __builtin_fmaf(d, d, square[e]);
            });
    });
    leave(entries, sum);
    leave(entries + lanes * pitch, square);
    __syncthreads();
    const float2 total = gather(true);
    if (tg == 0 && g < p.B) {
        const float shift = total.x * of_count;
        group[g] = float2{rough + shift, root_of(__builtin_fmaf(-shift, total.x, total.y), p)};
    }
    __syncthreads();
    if (!mine) return;
    again();
    affine.take(group, j * V, channels, p.d, p.d_magic);
    char *const out = static_cast<char *>(p.out) + image * p.out_image_bytes + (ch0 + j * V) * SIZE;
    static_for<0, NP>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if (lane + i * lanes < pixels) {
            Piece<TYPE, V> a;
            static_for<0, V>([&](auto ec) { a.v[decltype(ec)::value] = v[i].template get<decltype(ec)::value>(); });
            affine.template apply<ACT>(p.act, p.slope, a);
            a.store(out, int64_t(lane + i * lanes) * p.c, V);
        }
    });
}

int power_of_two(int v) {      // the next one up
    int p = 1;
    while (p < v) p *= 2;
    return p;
}

// Whether the one-launch kernel takes the call, on which pieces and threads (V = 0: it does not), by estimates of the times in us, fitted
// to bf16 with SiLU.  Here a workgroup's own values take their time, and all workgroups' that of the cache lines they share with one
// another (runs of less than 40 bytes at a pixel cost as much as 40).  Two kernels: two starts and the tensor's bytes.  Measured, one launch
// and two: 64 pixels x 1280 channels on 2 images 5.2 and 9.8, on 32 images 6.9 and 10.8; 1024 x 640 on 8 10.5 and 13.0, on 32 26.6 and 26.3;
// 4096 x 320 (groups of 10: runs of 20 bytes) on 1 21.5 and 11.4, on 8 21.2 and 17.7; 4096 x 128 on 1 9.4 and 10.0, on 16 18.1 and 15.7.
struct HeldPlan {
    HeldParams p;
    int V, NP, threads;
};

HeldPlan held_plan(const tsx_group_norm *g, const NormParams &rows) {
    HeldPlan best{};
    const float size = float(element_bytes(g->type));
    float best_cost = 10.f + 0.28e-6f * float(g->n) * float(g->pixels) * float(g->c) * size;
    if (g->pixels > 16384) return best;
    const int pixels = int(g->pixels), d = g->c / g->groups, whole = g->type == TSX_TYPE_F32 ? 4 : 8;
    // The divisors of the groups in ascending order, looked for up to their root: each B up to 8192 for itself was 10 .. 50 us of the call.
    int divisors[64], count = 0, root = 1;                   // no number up to NORM_MOST_CHANNELS has more than 64
    for (; root * root <= g->groups; ++root)
        if (g->groups % root == 0) divisors[count++] = root;
    for (int i = count - 1; i >= 0; --i)
        if (divisors[i] * divisors[i] != g->groups) divisors[count++] = g->groups / divisors[i];
    for (int V = whole; V >= 2; V /= 2)
        for (int i = 0; i < count; ++i) {
            const int B = divisors[i];
            if (B * d % V) continue;
            const int a_pixel = B * d / V;
            if (a_pixel > NORM_MOST_THREADS) break;
            const int most = V == 8 ? 12 : g->type == TSX_TYPE_F32 && V == 4 ? 16 : 24;      // what 128 registers hold beside the rest
            int threads = 256;
            while (threads < NORM_MOST_THREADS && (threads < a_pixel || ceil_div(pixels, threads / a_pixel) > 4)) threads *= 2;
            const int lanes = threads / a_pixel, need = int(ceil_div(pixels, lanes));
            if (need > most) break;
            if (power_of_two(B) > threads) continue;
            const int64_t bundles = int64_t(g->n) * (g->groups / B);
            if (bundles > 1 << 21) continue;      // with 1024 threads each, half of what a launch holds
            const float run = float(B * d) * size, pixel = float(pixels) / 20480.f;
            const float cost = 5.f + std::max(1.7f * pixel * run, 2.6f * float(bundles) / 256.f * pixel * std::max(run, 40.f)) * (V == 2 ? 2.f : 1.f);
            if (cost >= best_cost) continue;
            best_cost = cost;
            best.V = V;
            best.NP = need;
            best.threads = threads;
            HeldParams &p = best.p;
            static_cast<NormParams &>(p) = rows;
            p.B = B;
            p.pieces_a_pixel = a_pixel;
            p.held_lanes = lanes;
            p.bundles = int(bundles);
            p.per_xcd = int(ceil_div(bundles, 8));
            p.a_image = g->groups / B;
            p.lg_run = lg_of(gcd(d, V));
            p.lg_TG = lg_of(threads / power_of_two(B));
            p.lg_TL = std::min(p.lg_TG, lg_of(power_of_two(lanes)));
            p.pixel_magic = div_magic(a_pixel, NORM_MOST_THREADS);
            p.image_magic = div_magic(p.a_image, bundles);
        }
    return best;
}

template <int TYPE, int V, int NP>
int launch_held(const HeldPlan &h, hipStream_t stream) {
    const HeldParams &p = h.p;
    const size_t lds = size_t(p.held_lanes) * ((p.B * p.d >> p.lg_run) | 1) * 2 * sizeof(float);
    const auto kernel = p.act == TSX_ACT_SILU ? group_norm_held_kernel<TYPE, V, NP, TSX_ACT_SILU> : group_norm_held_kernel<TYPE, V, NP, ANY_ACT>;
    if (lds > 48 * 1024) {      // 9 KiB beside them are the kernel's own
        const int rc = grant_lds(reinterpret_cast<const void *>(kernel), 128 * 1024);
        if (rc) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(unsigned(8 * p.per_xcd)), dim3(h.threads), lds, stream, p);
    TSX_LAUNCH_CHECK("group_norm_held_kernel");
    return 0;
}

template <int TYPE, int V>
int held(const HeldPlan &h, hipStream_t stream) {
    if (h.NP <= 2) return launch_held<TYPE, V, 2>(h, stream);
    if (h.NP <= 4) return launch_held<TYPE, V, 4>(h, stream);
    if (h.NP <= 8) return launch_held<TYPE, V, 8>(h, stream);
    if constexpr (V == 8) {
        if (h.NP <= 12) return launch_held<TYPE, V, 12>(h, stream);
    } else {
        if (h.NP <= 16) return launch_held<TYPE, V, 16>(h, stream);
        if constexpr (TYPE != TSX_TYPE_F32 || V == 2) return launch_held<TYPE, V, 24>(h, stream);
    }
    return fail(TSX_E_INVALID, "group_norm: %d pieces a thread", h.NP);
}

template <int TYPE>
int run_held(const HeldPlan &h, hipStream_t stream) {
    if constexpr (TYPE != TSX_TYPE_F32) {
        if (h.V == 8) return held<TYPE, 8>(h, stream);
    }
    return h.V == 4 ? held<TYPE, 4>(h, stream) : held<TYPE, 2>(h, stream);
}

}  // namespace

int group_norm_held(const tsx_group_norm *g, const NormParams &p, hipStream_t stream, bool *taken) {
    const HeldPlan h = held_plan(g, p);
    *taken = h.V != 0;
    if (!*taken) return 0;
    return g->type == TSX_TYPE_F32 ? run_held<TSX_TYPE_F32>(h, stream) : g->type == TSX_TYPE_F16 ? run_held<TSX_TYPE_F16>(h, stream)
                                                                                                : run_held<TSX_TYPE_BF16>(h, stream);
}

}  // namespace tsx
