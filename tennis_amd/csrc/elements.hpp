// Tensors of fp32, fp16 and bf16 values: runs of them to and from registers, their magnitudes, and their rows as int8 tokens.
// All arithmetic on them is in fp32; a result is rounded once, to nearest even, when it is stored.
#pragma once
#include <atomic>

#include "tsx_common.hpp"

namespace tsx {

inline size_t element_bytes(int type) { return type == TSX_TYPE_F32 ? 4 : type == TSX_TYPE_I8 ? 1 : 2; }
inline bool is_float_type(int type) { return type == TSX_TYPE_F32 || type == TSX_TYPE_F16 || type == TSX_TYPE_BF16; }
inline bool is_token_act(int act) {      // the exact Mish is the host's bits for a given fp32 number, which no sum here has
    return act == TSX_ACT_NONE || act == TSX_ACT_RELU || act == TSX_ACT_LEAKY_RELU || act == TSX_ACT_MISH_FAST || act == TSX_ACT_SILU;
}

// Dynamic LDS beyond 64 KiB is granted per kernel and device: once for each, of a kernel always the same bytes.
inline int grant_lds(const void *kernel, int bytes) {
    struct Granted { std::atomic<const void *> kernel; std::atomic<uint64_t> devices; };
    constexpr unsigned PLACES = 256;       // more than there are kernels that ask
    static Granted table[PLACES];
    int dev = 0;
    TSX_HIP(hipGetDevice(&dev));
    const unsigned first = unsigned(reinterpret_cast<uintptr_t>(kernel) >> 4);
    for (unsigned i = 0; i < PLACES; ++i) {
        Granted &g = table[(first + i) % PLACES];
        const void *none = nullptr;
        if (g.kernel.load() != kernel && !g.kernel.compare_exchange_strong(none, kernel) && none != kernel) continue;
        if (dev < 64 && g.devices.load() >> dev & 1) return 0;
        TSX_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        if (dev < 64) g.devices.fetch_or(uint64_t(1) << dev);
        return 0;
    }
    return fail(TSX_E_INVALID, "no place for another kernel's LDS");
}

// f(the activation as a constant)
template <class F>
auto with_act(int act, F &&f) {
    switch (act) {
        case TSX_ACT_RELU: return f(std::integral_constant<int, TSX_ACT_RELU>{});
        case TSX_ACT_LEAKY_RELU: return f(std::integral_constant<int, TSX_ACT_LEAKY_RELU>{});
        case TSX_ACT_MISH_FAST: return f(std::integral_constant<int, TSX_ACT_MISH_FAST>{});
        case TSX_ACT_SILU: return f(std::integral_constant<int, TSX_ACT_SILU>{});
        default: return f(std::integral_constant<int, TSX_ACT_NONE>{});
    }
}

#ifdef __HIPCC__

typedef unsigned v2u __attribute__((ext_vector_type(2)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));
// at any address: global memory takes 16 bytes wherever they begin
typedef unsigned u_any __attribute__((aligned(1)));
typedef unsigned v2u_any __attribute__((ext_vector_type(2), aligned(1)));
typedef unsigned v4u_any __attribute__((ext_vector_type(4), aligned(1)));

// A value from the lane that is 2^K away (K < 6), for sums and maxima: up to there lanes hold one value, so a mirrored lane does for
// an exchanged one.  Vector instructions all the way: a shuffle through LDS takes some hundred cycles, and six of them a reduction.
template <int K>
__device__ __forceinline__ unsigned partner(unsigned v) {
    if constexpr (K < 4) {
        constexpr int CTRL = K == 0 ? 0xb1 : K == 1 ? 0x4e : K == 2 ? 0x141 : 0x140;      // quads [1,0,3,2] and [2,3,0,1], mirrors of 8 and of 16
        return unsigned(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xf, 0xf, true));
    } else {
        // both results together hold a lane's own value and its partner's
        const auto s = K == 4 ? __builtin_amdgcn_permlane16_swap(v, v, false, false) : __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (threadIdx.x >> K) & 1 ? s[0] : s[1];
    }
}
// f over 2^lg consecutive lanes (lg uniform), in every one of them
template <class F>
__device__ __forceinline__ unsigned over_lanes(unsigned v, int lg, F &&f) {
    static_for<0, 6>([&](auto kc) {
        constexpr int K = decltype(kc)::value;
        if (lg > K) v = f(v, partner<K>(v));
    });
    return v;
}
__device__ __forceinline__ float sum_over_lanes(float v, int lg) {
    return __builtin_bit_cast(float, over_lanes(__builtin_bit_cast(unsigned, v), lg, [](unsigned a, unsigned b) {
        return __builtin_bit_cast(unsigned, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
    }));
}
constexpr int lg_of(int power) { return power <= 1 ? 0 : 1 + lg_of(power / 2); }

// a value the compiler knows nothing of: not what it was computed from, nor that it is the same one later
__device__ __forceinline__ void renew(unsigned &word) { asm volatile("" : "+v"(word)); }

// N consecutive values as they lie in memory
template <int TYPE, int N>
struct Run {
    static constexpr int BYTES = N * (TYPE == TSX_TYPE_F32 ? 4 : 2), WORDS = (BYTES + 3) / 4, PER_WORD = TYPE == TSX_TYPE_F32 ? 1 : 2;
    static_assert(BYTES <= 4 || BYTES % 8 == 0, "a word or whole pairs of words");
    unsigned word[WORDS];

    __device__ __forceinline__ void renew_words() {
        static_for<0, WORDS>([&](auto wc) { renew(word[decltype(wc)::value]); });
    }
    __device__ __forceinline__ void clear() {
        static_for<0, WORDS>([&](auto wc) { word[decltype(wc)::value] = 0; });
    }
    __device__ __forceinline__ void load(const void *at) {
        if constexpr (BYTES == 2)
            word[0] = *reinterpret_cast<const unsigned short *>(at);
        else if constexpr (BYTES == 4)
            word[0] = *reinterpret_cast<const u_any *>(at);
        else if constexpr (BYTES % 16 == 0)
            static_for<0, BYTES / 16>([&](auto wc) {
                constexpr int w = decltype(wc)::value;
                const v4u v = reinterpret_cast<const v4u_any *>(at)[w];
                static_for<0, 4>([&](auto jc) { word[4 * w + decltype(jc)::value] = v[decltype(jc)::value]; });
            });
        else
            static_for<0, BYTES / 8>([&](auto wc) {
                constexpr int w = decltype(wc)::value;
                const v2u v = reinterpret_cast<const v2u_any *>(at)[w];
                static_for<0, 2>([&](auto jc) { word[2 * w + decltype(jc)::value] = v[decltype(jc)::value]; });
            });
    }
    // the first `left` values, one at least, behind them zeros; all requested at once, the last one again in the place of those
    __device__ __forceinline__ void load_some(const void *at, int left) {
        static_for<0, WORDS>([&](auto wc) {
            constexpr int w = decltype(wc)::value;
            if constexpr (TYPE == TSX_TYPE_F32) {
                const unsigned v = reinterpret_cast<const unsigned *>(at)[min(w, left - 1)];
                word[w] = w < left ? v : 0u;
            } else {
                const unsigned short *h = reinterpret_cast<const unsigned short *>(at);
                const unsigned lo = h[min(2 * w, left - 1)], hi = h[min(2 * w + 1, left - 1)];
                word[w] = (2 * w < left ? lo : 0u) | (2 * w + 1 < left ? hi << 16 : 0u);
            }
        });
    }
    // STREAMS: not to be kept in the caches
    template <bool STREAMS = false>
    __device__ __forceinline__ void store(void *at) const {
        if constexpr (BYTES == 2)
            *reinterpret_cast<unsigned short *>(at) = (unsigned short)word[0];
        else if constexpr (BYTES == 4)
            *reinterpret_cast<u_any *>(at) = word[0];
        else if constexpr (BYTES % 16 == 0)
            static_for<0, BYTES / 16>([&](auto wc) {
                constexpr int w = decltype(wc)::value;
                const v4u_any v = v4u{word[4 * w], word[4 * w + 1], word[4 * w + 2], word[4 * w + 3]};
                if constexpr (STREAMS) __builtin_nontemporal_store(v, reinterpret_cast<v4u_any *>(at) + w);
                else reinterpret_cast<v4u_any *>(at)[w] = v;
            });
        else
            static_for<0, BYTES / 8>([&](auto wc) {
                constexpr int w = decltype(wc)::value;
                reinterpret_cast<v2u_any *>(at)[w] = v2u{word[2 * w], word[2 * w + 1]};
            });
    }
    __device__ __forceinline__ void store_some(void *at, int left) const {
        static_for<0, N>([&](auto ec) {
            constexpr int e = decltype(ec)::value;
            if (e < left) {
                if constexpr (TYPE == TSX_TYPE_F32) reinterpret_cast<unsigned *>(at)[e] = word[e];
                else reinterpret_cast<unsigned short *>(at)[e] = (unsigned short)(word[e / 2] >> (16 * (e % 2)));
            }
        });
    }
    template <int E>
    __device__ __forceinline__ float get() const {
        if constexpr (TYPE == TSX_TYPE_F32) return __builtin_bit_cast(float, word[E]);
        else if constexpr (TYPE == TSX_TYPE_BF16) return __builtin_bit_cast(float, E % 2 ? word[E / 2] & 0xffff0000u : word[E / 2] << 16);
        else return float(__builtin_bit_cast(_Float16, (unsigned short)(word[E / 2] >> (16 * (E % 2)))));
    }
    __device__ __forceinline__ void set(const float (&v)[N]) {
        static_for<0, WORDS>([&](auto wc) {
            constexpr int w = decltype(wc)::value;
            if constexpr (TYPE == TSX_TYPE_F32) {
                word[w] = __builtin_bit_cast(unsigned, v[w]);
            } else if constexpr (TYPE == TSX_TYPE_BF16) {
                typedef __bf16 pair __attribute__((ext_vector_type(2)));
                typedef float two __attribute__((ext_vector_type(2)));
                word[w] = __builtin_bit_cast(unsigned, __builtin_convertvector((two{v[2 * w], 2 * w + 1 < N ? v[(2 * w + 1) % N] : 0.f}), pair));
            } else {
                typedef _Float16 pair __attribute__((ext_vector_type(2)));
                word[w] = __builtin_bit_cast(unsigned, pair{_Float16(v[2 * w]), _Float16(2 * w + 1 < N ? v[(2 * w + 1) % N] : 0.f)});
            }
        });
    }
    // The largest magnitude as the bits of that magnitude, which sort as whole numbers do: two 16-bit ones a word, or one of 32.
    // Infinities and NaN are the largest.
    __device__ __forceinline__ unsigned top(unsigned so_far) const {
        static_for<0, WORDS>([&](auto wc) { so_far = larger<TYPE>(so_far, word[decltype(wc)::value] & (PER_WORD == 1 ? 0x7fffffffu : 0x7fff7fffu)); });
        return so_far;
    }
    template <int KIND>
    static __device__ __forceinline__ unsigned larger(unsigned a, unsigned b) {
        if constexpr (KIND == TSX_TYPE_F32) return a > b ? a : b;
        typedef unsigned short pair __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(pair, a), __builtin_bit_cast(pair, b)));
    }
};

// the magnitude that Run::top found, as an fp32 number
template <int TYPE>
__device__ __forceinline__ float top_value(unsigned top) {
    if constexpr (TYPE == TSX_TYPE_F32) return __builtin_bit_cast(float, top);
    const unsigned lo = top & 0xffffu, hi = top >> 16, most = lo > hi ? lo : hi;
    if constexpr (TYPE == TSX_TYPE_BF16) return __builtin_bit_cast(float, most << 16);
    return float(__builtin_bit_cast(_Float16, (unsigned short)most));
}

// A token's way to int8: the largest magnitude a of a row becomes 127.
//   scale = fp32(a / 127),  q = round to nearest even of x * fp32(127 / a), the product exact.
// Rows below 2^-64, where 127 / a would leave fp32, are lifted by 2^64 first; a row with an infinity or NaN has zeros and the scale NaN.
struct TokenScale {
    float lift, reciprocal, scale;
    __device__ __forceinline__ explicit TokenScale(float top) {
        const bool finite = top < __builtin_inff();      // false for NaN
        lift = top < 0x1p-64f ? 0x1p64f : 1.f;
        reciprocal = finite && top > 0.f ? __fdiv_rn(127.f, __fmul_rn(top, lift)) : 0.f;
        scale = finite ? __fdiv_rn(top, 127.f) : __builtin_nanf("");
    }
    // One fused multiply-add: behind 1.5 * 2^23 the sum's last bit is 1, so its rounding, half to even, is that of the exact
    // product, and its low byte is the product in two's complement.  0 * infinity never gets here: then `reciprocal` is 0 and
    // the caller takes zeros (an infinity in the row), or x is finite.
    __device__ __forceinline__ unsigned bits(float x) const { return __builtin_bit_cast(unsigned, __builtin_fmaf(x, reciprocal, 0x1.8p23f)); }
};
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
    return __builtin_amdgcn_perm(b, a, 0x0c0c0400u) | __builtin_amdgcn_perm(d, c, 0x04000c0cu);
}

// silu and the activations of the epilogues on results of fp32 arithmetic.  OUT: the type that the result is rounded to.
//
// exp(-x) = 2^t (1 + r): t is -x log2(e) in fp32, r = -x - t ln 2 what that rounding dropped, |x| 2^-24 at most.  With it the result is within 8 2^-24
// of itself; without, which only fp32 shows, up to (8 + |x|) 2^-24 (64 x 64 x 320 fp16 on 8 images 18.1 us, with r 19.5).  The clamp keeps r finite.
template <int OUT>
__device__ __forceinline__ float silu(float x) {
    float e;
    if constexpr (OUT == TSX_TYPE_F32) {
        const float c = __builtin_amdgcn_fmed3f(x, -200.f, 200.f), t = __fmul_rn(c, -1.4426950216293335f);
        const float r = __builtin_fmaf(t, 1.904654299e-9f, __builtin_fmaf(t, -0.693147182464599609375f, -c));
        e = __fmul_rn(__builtin_amdgcn_exp2f(t), __fadd_rn(1.f, r));
    } else {
        e = __builtin_amdgcn_exp2f(__fmul_rn(x, -1.4426950216293335f));
    }
    return __fmul_rn(x, __builtin_amdgcn_rcpf(__fadd_rn(1.f, e)));
}
// The activation as a constant of the code: kernels bound by their arithmetic have a path for each, since five of them in turn
// behind each other's branches put every one an instruction-cache miss apart.
template <int OUT, int ACT, int N>
__device__ __forceinline__ void activate_as(float (&v)[N], float slope) {
    static_for<0, N>([&](auto rc) {
        constexpr int r = decltype(rc)::value;
        if constexpr (ACT == TSX_ACT_RELU) v[r] = max_zero(v[r]);
        if constexpr (ACT == TSX_ACT_LEAKY_RELU) v[r] = __builtin_fmaf(slope, min_zero(v[r]), max_zero(v[r]));
        if constexpr (ACT == TSX_ACT_MISH_FAST) v[r] = mish_short(v[r]);
        if constexpr (ACT == TSX_ACT_SILU) v[r] = silu<OUT>(v[r]);
    });
}
template <int OUT, int N>
__device__ __forceinline__ void activate_tokens(float (&v)[N], int act, float slope) {
    if (act == TSX_ACT_SILU) {
        asm volatile("; silu");
        static_for<0, N>([&](auto rc) { constexpr int r = decltype(rc)::value; v[r] = silu<OUT>(v[r]); });
    } else {
        activate_results(v, act, slope);
    }
}

#endif  // __HIPCC__

}  // namespace tsx
