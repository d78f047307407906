// Rows in microscaled 4-bit floating point: a block's scale from its largest magnitude, and values to codes and back by the
// conversion instructions, which multiply or divide by 2^(the exponent bits of their fp32 scale - 127) exactly, also by 2^-127, and
// round once, to nearest, ties to even codes, beyond 6 to 6 (every scale against the definition, tests/test_gpu_mxfp4.py).
#pragma once
#include "elements.hpp"

namespace tsx {

constexpr int MX_BLOCK = 32;           // values of a block
constexpr int MX_STEP = 128;           // values of a K-step of the products: four blocks, 64 bytes of codes, a word of scales

// Where rows in MXFP4 are written: codes at a stride in bytes, the scale of block b of a row at (b / 4) scale_group + b % 4 + row scale_row.
// Rows of scales: scale_group 4.  Words of four blocks, a K-step's of all rows side by side, as the products read them: scale_row 4.
struct MxRows {
    uint8_t *codes, *scales;
    int64_t codes_stride, scale_row, scale_group;
};

// tsx_quantize_mxfp4 without its checks; columns from cols up to cols_out, a multiple of 32 or cols itself, are zeros (their scales' bytes 0)
int quantize_mxfp4_rows(int64_t rows, int cols, int cols_out, const void *x, int type, int64_t x_stride, const MxRows &to, hipStream_t stream);

// n / d for n below 2^31 by a multiplication: m = ceil(2^(31 + l) / d) with 2^l >= d is off by less than d / 2^(31 + l) of a quotient
struct Divider {
    uint32_t d, m;
    int shift;
    explicit Divider(int64_t divisor) : d(uint32_t(divisor)) {
        int l = 0;
        while (int64_t(1) << l < divisor) ++l;
        shift = 31 + l;
        m = uint32_t(((uint64_t(1) << shift) + d - 1) / d);
    }
#ifdef __HIPCC__
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return uint32_t((uint64_t(n) * m) >> shift); }
#endif
};

#ifdef __HIPCC__

// The scale's byte of a block whose largest magnitude is `top`: 6 = 1.5 * 2^2 is the largest value, so that magnitude's exponent less 2.
__device__ __forceinline__ unsigned mx_scale(float top) {
    const unsigned e = __builtin_bit_cast(unsigned, top) >> 23;
    return e == 255 ? 255 : e < 2 ? 0 : e - 2;
}
__device__ __forceinline__ float mx_factor(unsigned scale) { return __builtin_bit_cast(float, scale << 23); }

// The piece of eight values that begins at value `at` of a row of at least eight: what is left of the row, behind it zeros.  load: the eight values
// there, or the row's last eight, a request like any other; then, where all requests are out, settle.
template <int TYPE>
__device__ __forceinline__ void load_piece(Run<TYPE, 8> &v, const char *row, int at, int cols) {
    v.load(row + int64_t(min(at, cols - 8)) * (TYPE == TSX_TYPE_F32 ? 4 : 2));
}
template <int TYPE>
__device__ __forceinline__ void settle_piece(Run<TYPE, 8> &v, int at, int cols) {
    const int over = at + 8 - cols;                // of the row's last eight, those that come first belong to the piece before
    if (over <= 0) return;
    if (over >= 8) {
        v.clear();
        return;
    }
    constexpr int W = Run<TYPE, 8>::WORDS, PER = 8 / W;
    static_for<0, 3>([&](auto bc) {
        constexpr int by = 4 >> decltype(bc)::value, words = by / PER;
        if (over & by) {
            if constexpr (words > 0) static_for<0, W>([&](auto wc) { constexpr int w = decltype(wc)::value; v.word[w] = w + words < W ? v.word[(w + words) % W] : 0u; });
            else static_for<0, W>([&](auto wc) { constexpr int w = decltype(wc)::value; v.word[w] = __builtin_amdgcn_alignbit(w + 1 < W ? v.word[(w + 1) % W] : 0u, v.word[w], 16); });
        }
    });
}

// eight values to four bytes of codes
template <int TYPE>
__device__ __forceinline__ unsigned mx_codes(const Run<TYPE, 8> &v, unsigned scale) {
    const float by = mx_factor(scale);
    unsigned codes = 0;
    static_for<0, 4>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (TYPE == TSX_TYPE_F32) {
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, v.template get<2 * i>(), v.template get<2 * i + 1>(), by, i);
        } else if constexpr (TYPE == TSX_TYPE_BF16) {
            typedef __bf16 pair __attribute__((ext_vector_type(2)));
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(pair, v.word[i]), by, i);
        } else {
            typedef _Float16 pair __attribute__((ext_vector_type(2)));
            codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(pair, v.word[i]), by, i);
        }
    });
    return scale == 255 ? 0 : codes;
}
// ... and back
template <int TYPE>
__device__ __forceinline__ Run<TYPE, 8> mx_values(unsigned codes, unsigned scale) {
    const float by = mx_factor(scale);
    Run<TYPE, 8> v;
    static_for<0, 4>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        if constexpr (TYPE == TSX_TYPE_F32) {      // exact in bf16, whose exponents are fp32's
            const unsigned two = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, by, i));
            v.word[2 * i] = two << 16;
            v.word[2 * i + 1] = two & 0xffff0000u;
        } else if constexpr (TYPE == TSX_TYPE_BF16) {
            v.word[i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, by, i));
        } else {
            v.word[i] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, by, i));
        }
    });
    return v;
}
// the codes of a piece of eight values, `left` of which, one at least, belong to the row
__device__ __forceinline__ void store_codes(uint8_t *at, unsigned codes, int left) {
    if (left >= 7) {
        *reinterpret_cast<u_any *>(at) = codes;
    } else {
        static_for<0, 3>([&](auto bc) {
            constexpr int b = decltype(bc)::value;
            if (2 * b < left) at[b] = uint8_t(codes >> (8 * b));
        });
    }
}

#endif  // __HIPCC__

}  // namespace tsx
