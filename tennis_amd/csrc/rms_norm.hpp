// Root-mean-square norm of rows, with the residual's addition in front of it; the result in the rows' type, as int8 tokens or as MXFP4.
//
//     h = x + residual, rounded to their type;  y = h r w,  r = 1 / sqrt(mean(h^2) + epsilon)
//
// Bound: HBM, four times the element size a value with a residual: 8192 x 4096 bf16 42 us, 6.4 TB/s with half of the input from the
// caches (a copy of 1 GiB 5.1); one row of 4096 2.5 - 2.9 us, the launch.  A row of up to 16384 values is read once (a longer one again for its results, and
// for each search on it scaled): T threads share it and hold h and the weight in registers, eight values to a piece, while they find the sum of its squares, and a
// workgroup requests its next row before it does.  As int8 tokens a row's codes do not know r: with A the largest |h w|, y's largest magnitude is A r, and
// y 127 / (A r) = h w 127 / A; so the search for A shares the one exchange between the threads with the sum, and only the scale, A r / 127, waits for r.
#pragma once
#include "mxfp4.hpp"

namespace tsx {

constexpr int NORM_ROWS = 0, NORM_TOKENS = 1, NORM_MXFP4 = 2;      // what leaves

struct RmsNormParams {
    const void *x, *residual;
    void *sum;
    const float *weight;
    void *out;                    // rows of x's type, int8 or codes
    void *scales;                 // fp32, or a byte a block
    int64_t rows, x_stride, residual_stride, sum_stride, out_stride, scales_stride;
    int cols;
    float inv_cols, epsilon;
};

int rms_norm_rows(const RmsNormParams &p, int type, hipStream_t stream);
int rms_norm_tokens(const RmsNormParams &p, int type, hipStream_t stream);
int rms_norm_mxfp4(const RmsNormParams &p, int type, hipStream_t stream);

#ifdef __HIPCC__

// A row whose mean square (with epsilon) leaves [2^-120, infinity) in fp32 is taken times a power of two instead; inside, what squares below 2^-126
// lose is 2^-30 of the mean.  Above: by 2^-80, so that 2^30 squares of the largest number stay below 2^126.  Below: by 2^105; the largest
// number that can be there, 2^-45 alone among 2^30 columns, becomes 2^60, and the mean with the least one, 2^-149 alone among them, 2^-118.
constexpr float NORM_LEAST = 0x1p-120f;
constexpr int NORM_DOWN = -80, NORM_UP = 105;

template <int TYPE, int TO, int T, int P, bool HELD>
__global__ __launch_bounds__(T <= 64 ? 256 : T, P == 3 && TYPE != TSX_TYPE_F32 ? 4 : 1) void rms_norm_kernel(RmsNormParams p) {
    constexpr int PIECE = 8, THREADS = T <= 64 ? 256 : T, ROWS = THREADS / T, SIZE = TYPE == TSX_TYPE_F32 ? 4 : 2, WAVES = T / 64;
    constexpr int LG = lg_of(T < 64 ? T : 64);
    typedef Run<TYPE, PIECE> Values;
    typedef Run<TSX_TYPE_F32, PIECE> Weights;
    __shared__ float sums[T > 64 ? WAVES : 1], tops[T > 64 ? WAVES : 1];
    const int tid = threadIdx.x, t = tid % T;
    const int pieces = (p.cols + PIECE - 1) / PIECE, whole = p.cols / PIECE, in_last = p.cols - whole * PIECE;
    const int turns = HELD ? 1 : (pieces + T * P - 1) / (T * P);
    Values h[P];
    Weights w[P];
    // P pieces of a row of values: all requests of a turn first, none behind a branch, where it would be waited for; then what lies behind the row's end
    // becomes zeros
    auto load = [&](auto &v, const char *from, int first) __attribute__((always_inline)) {
        static_for<0, P>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            const int piece = first + t + i * T;
            if (whole) {       // uniform
                load_piece(v[i], from, piece * PIECE, p.cols);
            } else {
                v[i].clear();
                if (piece == 0) v[i].load_some(from, p.cols);
            }
        });
    };
    auto settle = [&](auto &v, int first) __attribute__((always_inline)) {
        if (whole)
            static_for<0, P>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                if (first + (i + 1) * T > whole) settle_piece(v[i], (first + t + i * T) * PIECE, p.cols);       // uniform: where the row's end can be
            });
    };
    // HELD: the weights once, and a row's values while the one before is at work
    Values next_x[P], next_r[P];
    auto request = [&](int64_t row) __attribute__((always_inline)) {
        const int64_t at = min(row, p.rows - 1);
        load(next_x, static_cast<const char *>(p.x) + at * p.x_stride * SIZE, 0);
        if (p.residual) load(next_r, static_cast<const char *>(p.residual) + at * p.residual_stride * SIZE, 0);
    };
    auto weights = [&](int first) __attribute__((always_inline)) {
        if (p.weight) load(w, reinterpret_cast<const char *>(p.weight), first);
        else static_for<0, P>([&](auto ic) { static_for<0, PIECE>([&](auto ec) { w[decltype(ic)::value].word[decltype(ec)::value] = 0x3f800000u; }); });
    };
    auto add = [&](auto &r) __attribute__((always_inline)) {
        static_for<0, P>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            float v[PIECE];
            static_for<0, PIECE>([&](auto ec) { constexpr int e = decltype(ec)::value; v[e] = __fadd_rn(h[i].template get<e>(), r[i].template get<e>()); });
            h[i].set(v);
        });
    };
    if constexpr (HELD) {
        request(int64_t(blockIdx.x) * ROWS + tid / T);
        weights(0);
        if (p.weight) settle(w, 0);
    }
    for (int64_t row0 = int64_t(blockIdx.x) * ROWS; row0 < p.rows; row0 += int64_t(gridDim.x) * ROWS) {
        const int64_t row = row0 + tid / T;
        const bool there = row < p.rows;      // a row's threads agree; only T <= 64 has several rows, and some beyond the last one, which are that one again
        const int64_t at = there ? row : p.rows - 1;
        char *const sum = static_cast<char *>(p.sum) + at * p.sum_stride * SIZE;
        auto store = [&](const Values &v, char *to, int piece) __attribute__((always_inline)) {
            if (!there || piece >= pieces) return;
            if (piece < whole) v.store(to + int64_t(piece) * (PIECE * SIZE));
            else v.store_some(to + int64_t(piece) * (PIECE * SIZE), in_last);
        };
        // h of a row; the next row's values are requested ahead of any store, so that nobody waits for these with them
        auto take = [&]() __attribute__((always_inline)) {
            static_for<0, P>([&](auto ic) { h[decltype(ic)::value] = next_x[decltype(ic)::value]; });
            settle(h, 0);
            if (p.residual) {
                settle(next_r, 0);
                add(next_r);
            }
            if (row0 + int64_t(gridDim.x) * ROWS < p.rows) request(row + int64_t(gridDim.x) * ROWS);       // uniform
            if (p.sum) static_for<0, P>([&](auto ic) { store(h[decltype(ic)::value], sum, t + decltype(ic)::value * T); });
        };
        // not HELD: h of a turn, and the weights where they are wanted; again: h as it was kept
        auto fetch = [&](int first, bool again, bool weighted) __attribute__((always_inline)) {
            const bool adds = p.residual && !(again && p.sum);       // uniform, as all conditions here
            Values r[P];
            load(h, again && p.sum ? sum : static_cast<const char *>(p.x) + at * p.x_stride * SIZE, first);
            if (adds) load(r, static_cast<const char *>(p.residual) + at * p.residual_stride * SIZE, first);
            if (weighted) weights(first);
            settle(h, first);
            if (adds) {
                settle(r, first);
                add(r);
            }
            if (p.sum && !again) static_for<0, P>([&](auto ic) { store(h[decltype(ic)::value], sum, first + t + decltype(ic)::value * T); });
            if (weighted && p.weight) settle(w, first);
        };
        // the sum of (h 2^up)^2 and the largest |h 2^up w| over the row, in all its threads
        float squares, top;
        auto statistics = [&](auto lifted, int up, bool again) __attribute__((always_inline)) {
            constexpr bool LIFTED = decltype(lifted)::value;
            double long_sum = 0;                  // over turns
            unsigned most = 0;                    // magnitudes' bits sort as they do, infinities and NaN last
            for (int turn = 0; turn < turns; ++turn) {
                if (!HELD) fetch(turn * T * P, again, TO == NORM_TOKENS);
                else if (!again) take();
                float s[2] = {0.f, 0.f};
                static_for<0, P>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    static_for<0, PIECE>([&](auto ec) {
                        constexpr int e = decltype(ec)::value;
                        float v = h[i].template get<e>();
                        if (LIFTED) v = __builtin_ldexpf(v, up);
                        s[e % 2] = __builtin_fmaf(v, v, s[e % 2]);
                        if constexpr (TO == NORM_TOKENS) most = max(most, __builtin_bit_cast(unsigned, __fmul_rn(v, w[i].template get<e>())) & 0x7fffffffu);
                    });
                });
                if (HELD) squares = s[0] + s[1];
                else long_sum += double(s[0]) + double(s[1]);
            }
            if (!HELD) squares = float(long_sum);
            squares = sum_over_lanes(squares, LG);
            if constexpr (TO == NORM_TOKENS) most = over_lanes(most, LG, [](unsigned a, unsigned b) { return max(a, b); });
            if constexpr (T > 64) {
                if (tid % 64 == 0) sums[tid / 64] = squares, tops[tid / 64] = __builtin_bit_cast(float, most);
                __syncthreads();
                squares = 0.f;
#pragma unroll
                for (int i = 0; i < WAVES; ++i) squares += sums[i], most = max(most, __builtin_bit_cast(unsigned, tops[i]));
                __syncthreads();                  // the next row writes them
            }
            top = __builtin_bit_cast(float, most);
        };
        char *const out = static_cast<char *>(p.out) + at * p.out_stride * (TO == NORM_ROWS ? SIZE : 1);
        // the results of a row: y = (h 2^up) r w; up is 0 unless LIFTED
        auto leave = [&](auto lifted, int up, float r) __attribute__((always_inline)) {
            constexpr bool LIFTED = decltype(lifted)::value;
            const float largest = __fmul_rn(top, r);                      // |y|
            const bool finite = largest < __builtin_inff();               // false for NaN
            const TokenScale token(finite ? top : __builtin_inff());      // of y / r: zeros where y leaves fp32
            if (TO == NORM_TOKENS && there && t == 0) static_cast<float *>(p.scales)[row] = finite ? __fdiv_rn(largest, 127.f) : __builtin_nanf("");
            for (int turn = 0; turn < turns; ++turn) {
                if (!HELD) fetch(turn * T * P, true, true);
                static_for<0, P>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    const int piece = turn * T * P + t + i * T;
                    float y[PIECE];                   // of int8 tokens: y / r
                    static_for<0, PIECE>([&](auto ec) {
                        constexpr int e = decltype(ec)::value;
                        y[e] = h[i].template get<e>();
                        if (LIFTED) y[e] = __builtin_ldexpf(y[e], up);
                        if constexpr (TO != NORM_TOKENS) y[e] = __fmul_rn(y[e], r);      // ahead of the weight: h w may leave fp32 where y does not
                        y[e] = __fmul_rn(y[e], w[i].template get<e>());
                    });
                    if constexpr (TO == NORM_ROWS) {
                        Values v;
                        v.set(y);
                        store(v, out, piece);
                    } else if constexpr (TO == NORM_TOKENS) {
                        if (!there || piece >= pieces) return;
                        unsigned b[PIECE];
                        static_for<0, PIECE>([&](auto ec) { constexpr int e = decltype(ec)::value; b[e] = token.bits(__fmul_rn(y[e], token.lift)); });
                        v2u q = {low_bytes(b[0], b[1], b[2], b[3]), low_bytes(b[4], b[5], b[6], b[7])};
                        if (token.reciprocal == 0.f) q = v2u{0, 0};
                        char *const to = out + int64_t(piece) * PIECE;
                        if (piece < whole) {
                            *reinterpret_cast<v2u_any *>(to) = q;
                        } else {
                            static_for<0, PIECE - 1>([&](auto ec) {
                                constexpr int e = decltype(ec)::value;
                                if (e < in_last) to[e] = char(q[e / 4] >> (8 * (e % 4)));
                            });
                        }
                    } else {
                        Weights v;
                        v.set(y);
                        // a block's four lanes: pieces behind the row's end are zeros, but for r: NaN and infinities have to come from the row itself
                        const unsigned own = piece < pieces ? v.top(0) : 0u;
                        const unsigned scale = mx_scale(__builtin_bit_cast(float, over_lanes(own, T < 4 ? 0 : 2, [](unsigned a, unsigned b) { return max(a, b); })));
                        const unsigned codes = mx_codes<TSX_TYPE_F32>(v, scale);
                        if (!there || piece >= pieces) return;
                        store_codes(reinterpret_cast<uint8_t *>(out) + int64_t(piece) * (PIECE / 2), codes, piece < whole ? PIECE : in_last);
                        if (piece % 4 == 0) static_cast<uint8_t *>(p.scales)[at * p.scales_stride + piece / 4] = uint8_t(scale);
                    }
                });
            }
        };
        statistics(std::false_type{}, 0, false);
        float mean = __builtin_fmaf(squares, p.inv_cols, p.epsilon);
        int up = 0;
        if (!(mean >= NORM_LEAST && mean < __builtin_inff())) {       // a row's threads agree
            up = mean < NORM_LEAST ? NORM_UP : NORM_DOWN;
            statistics(std::true_type{}, up, true);
            mean = __builtin_fmaf(squares, p.inv_cols, __builtin_ldexpf(p.epsilon, 2 * up));
        }
        const float r = __builtin_amdgcn_rsqf(mean);
        // The least largest |h w| of whose row all products that do not become 0, from 1 / 254 of it on, are normal numbers.
        constexpr float LEAST_TOP = 0x1p-118f;
        if (TO == NORM_TOKENS && HELD) static_for<0, P>([&](auto ic) { w[decltype(ic)::value].renew_words(); });      // no product is kept from the search: registers
        if (TO == NORM_TOKENS && (up != 0 || top < LEAST_TOP)) {
            // With r in [1, 2) no |h 2^up w| is more than that |y|, nor less than half of it: such a row's products stay where y itself stays.
            // It has code of its own: in one path for both, ordinary rows (5000 x 2050) took 5 % longer.
            const int e = __builtin_amdgcn_frexp_expf(r) - 1;
            statistics(std::true_type{}, up + e, true);
            leave(std::true_type{}, up + e, __builtin_ldexpf(r, -e));
        } else {
            leave(std::bool_constant<TO != NORM_TOKENS>{}, up, r);
        }
    }
}

template <int TYPE, int TO, int T, int P, bool HELD>
int launch_rms_norm(const RmsNormParams &p, hipStream_t stream) {
    constexpr int THREADS = T <= 64 ? 256 : T, ROWS = THREADS / T;
    const int64_t blocks = ceil_div(p.rows, ROWS);
    // A workgroup takes one row after the other, the weights once, where rows are more than twice what the CUs hold at a time: 4096 threads each, 2048 with
    // the registers of longer rows.  As many rows each, one or all (bf16, us): 400000 x 64 31 and 21, 5000 x 2048 9.4 and 8.3, 20000 x 1000 as int8 22.9 and 22.5;
    // fewer threads than that: 8192 x 4096 with a residual 43.3 for 40.8.
    constexpr int AT_ONCE = P == 3 || T * P >= 1024 ? 2048 : 4096;
    const int64_t slots = 256 * AT_ONCE / THREADS;
    const int64_t grid = ceil_div(blocks, ceil_div(blocks, slots));
    hipLaunchKernelGGL((rms_norm_kernel<TYPE, TO, T, P, HELD>), dim3(unsigned(grid)), dim3(THREADS), 0, stream, p);
    TSX_LAUNCH_CHECK("rms_norm_kernel");
    return 0;
}

template <int TYPE, int TO>
int rms_norm_type(const RmsNormParams &p, hipStream_t stream) {
    // One piece of eight values a thread where that makes a workgroup, two or three of a longer row: more of them leave a CU too few threads (a row a workgroup, bf16
    // with a residual, us: 2048 x 2048 256 threads a row 7.5, 128 7.9, 64 8.9; 5000 x 2050 128 threads with three pieces each 16.7, 64 with five 18.4, 256 with two
    // 16.9; 8192 x 4096 256 threads 48, 64 55; 2000 x 8192 512 threads 27, 256 28).  Rows of two pieces a lane stay in a wavefront, with no barrier (8192 x
    // 1000: 11.7, 256 threads 15.9), several short ones to each, with lanes for their pieces and few more
    // (16.8 million rows of one value 137 us, four lanes each 389; 2 million of 8 25, 34; 419430 of 40 as int8 on eight lanes 22, on sixteen 34; 83886 of 200 on 32
    // lanes 20, on 64 31).  512 threads for rows of up to 4096 while there are few (1 x 4096 3.0, 256 threads 3.2).
    const int64_t pieces = ceil_div(p.cols, 8);
    if (pieces <= 1) return launch_rms_norm<TYPE, TO, 1, 1, true>(p, stream);
    if (pieces <= 4) return launch_rms_norm<TYPE, TO, 4, 1, true>(p, stream);
    if (pieces <= 8) return launch_rms_norm<TYPE, TO, 8, 1, true>(p, stream);
    if (pieces <= 16) return launch_rms_norm<TYPE, TO, 16, 1, true>(p, stream);
    if (pieces <= 32) return launch_rms_norm<TYPE, TO, 32, 1, true>(p, stream);
    if (pieces <= 64) return launch_rms_norm<TYPE, TO, 64, 1, true>(p, stream);
    if (pieces <= 128) return launch_rms_norm<TYPE, TO, 64, 2, true>(p, stream);
    if (pieces <= 256) return launch_rms_norm<TYPE, TO, 256, 1, true>(p, stream);
    if (pieces <= 384) return launch_rms_norm<TYPE, TO, 128, 3, true>(p, stream);
    if (pieces <= 512 && p.rows < 2048) return launch_rms_norm<TYPE, TO, 512, 1, true>(p, stream);
    if (pieces <= 512) return launch_rms_norm<TYPE, TO, 256, 2, true>(p, stream);
    if (pieces <= 1024) return launch_rms_norm<TYPE, TO, 512, 2, true>(p, stream);
    if (pieces <= 2048) return launch_rms_norm<TYPE, TO, 1024, 2, true>(p, stream);
    return launch_rms_norm<TYPE, TO, 1024, 2, false>(p, stream);
}
template <int TO>
int rms_norm_of(const RmsNormParams &p, int type, hipStream_t stream) {
    return type == TSX_TYPE_F32 ? rms_norm_type<TSX_TYPE_F32, TO>(p, stream) : type == TSX_TYPE_F16 ? rms_norm_type<TSX_TYPE_F16, TO>(p, stream)
                                                                                                    : rms_norm_type<TSX_TYPE_BF16, TO>(p, stream);
}

#endif  // __HIPCC__

}  // namespace tsx
