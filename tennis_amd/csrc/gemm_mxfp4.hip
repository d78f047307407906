// Product of MXFP4 rows (mxfp4.hpp) with MXFP4 weights, on rows of fp32, fp16, bf16 or MXFP4.
//
//     out[i][j] = act(sum over blocks b of 2^(s_x[i][b] + s_w[j][b] - 254) sum_k x[i][k] w[j][k] + bias[j]),  rounded once to the output's type
//
// The scaled matrix instructions take both scales with the codes: v_mfma_scale_f32_32x32x64_f8f6f4, where a lane supplies row l % 32 of block
// l / 32 of two, its 16 bytes of codes and its scale, and v_mfma_scale_f32_16x16x128_f8f6f4, row l % 16 of block l / 16 of four.  Sums are fp32.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "mxfp4.hpp"
#include "token_tiles.hpp"

namespace tsx {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));

constexpr int KSTEP = MX_STEP / 2;     // bytes of codes
constexpr int FP4 = 4;                 // the instructions' number for this type

// Packed weights: codes [K-step][fragment of 32 columns][half of the K-step][lane][16], as the 32x32x64 instruction takes them, behind
// them scales [K-step][column][4].  Columns in whole groups of 128, K-steps in whole chunks of every kernel, fours; zeros behind n and k, whose scales are 2^-127.
int frags_of(int n) { return int(round_up(n, 128) / 32); }
int ksteps_of(int k) { return int(round_up(ceil_div(k, MX_STEP), 4)); }
int64_t packed_codes(int k, int n) { return int64_t(ksteps_of(k)) * frags_of(n) * 2048; }

struct MxGemmParams {
    const uint8_t *x, *x_scales;       // codes [m] at x_pitch, a multiple of 16; scales: a K-step's word of a row at row scale_row + step scale_step
    const int8_t *w, *w_scales;
    const float *bias;
    void *out;
    int64_t x_pitch, scale_row, scale_step, out_stride;
    int m, n, k, frags, ksteps;        // k: bytes of codes of a row that are there, a multiple of 16; ksteps: of the weights
    int x_steps;                       // K-steps of x's scales
    float slope;
    int act;
    int row_tiles, col_tiles, tiles_per_xcd;
    bool streams;                      // outputs go past the caches
};

__device__ __forceinline__ v8i operand(v4i v) { return __builtin_shufflevector(v, v, 0, 1, 2, 3, -1, -1, -1, -1); }

// A fragment's values of 32 output columns x 32 tokens in the output's type: accumulator r of lane l is column 8 (r / 4) + 4 (l / 32) +
// r % 4 of token l % 32; swaps between the half-waves leave a lane with 16 consecutive columns, the lower ones with 0 .. 15, the upper
// ones with 16 .. 31.
template <int OUT>
__device__ __forceinline__ Run<OUT, 16> fragment_values(const float (&v)[16]) {
    Run<OUT, 16> to, own;
    own.set(v);
    constexpr int W = Run<OUT, 4>::WORDS;      // words of four values
    static_for<0, 2>([&](auto pc) {
        constexpr int a = decltype(pc)::value;
        static_for<0, W>([&](auto wc) {
            constexpr int w = decltype(wc)::value;
            const auto s = __builtin_amdgcn_permlane32_swap(own.word[a * W + w], own.word[(a + 2) * W + w], false, false);
            to.word[2 * a * W + w] = s[0];
            to.word[(2 * a + 1) * W + w] = s[1];
        });
    });
    return to;
}

__device__ __forceinline__ void word_to_lds(const uint8_t *at, int8_t *lds) {
    __builtin_amdgcn_global_load_lds((global_void *)at, (lds_void *)lds, 4, 0, 0);
}

// A wavefront's reads of LDS are done and its requests but the last N here, then those of all wavefronts.  In one piece: in front of a barrier of its
// own the compiler waits for every request.
template <int N>
__device__ __forceinline__ void barrier_but_for() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// WR x WC wavefronts, each with FR x FC fragments of 32 tokens x 32 columns; S chunks of KS K-steps in LDS, scales behind their codes; KG such groups of
// wavefronts, each with its part of every chunk's K-steps.
//
// Bound: 8192^3 260 us (median of calls on codes one behind the other), 4.2 P operations/s: waiting.  The matrix cores are busy for 61 - 65 % of the cycles at
// 1.7 GHz; the same instructions on random operands from registers, nothing else, make 6.5 P at 1.55 GHz, the clock that the card's power leaves them, so
// power is 9 % of the difference.  By products of K = 512 .. 8192 a tile takes 6.8 us for 1024 of K (5.0 P) and 9 - 10 of its 65 us for its first chunk and
// its epilogue, with nothing beside them.  4 x 4 fragments on four wavefronts read a third less LDS and take 268 us, one wavefront a SIMD hides less.
// Few tiles with a long K wait for one K-step after the other, 0.19 us each in tiles of 64; two groups of wavefronts halve that.
template <int WR, int WC, int FR, int FC, int KS, int S, int KG, int OUT>
__global__ __launch_bounds__(WR *WC *KG * 64, WR * FR == 4 && KG == 1 ? 3 : 1) void gemm_mxfp4_kernel(MxGemmParams p) {
    constexpr int CHUNK = KS * KSTEP, PIECES = CHUNK / 16, WAVES = WR * WC * KG, ROWS = 32 * WR * FR, COLS = 32 * WC * FC, HALVES = 2 * KS / KG;
    constexpr int A_BYTES = ROWS * CHUNK, B_BYTES = COLS * CHUNK, A_LOADS = A_BYTES / 1024 / WAVES, B_LOADS = B_BYTES / 1024 / WAVES;
    constexpr int A_WORDS = KS * ROWS / 64, WORDS = KS * (ROWS + COLS) / 64, S_LOADS = (WORDS + WAVES - 1) / WAVES;      // scales: by 64 words
    constexpr int SCALES = A_BYTES + B_BYTES, BUFFER = SCALES + KS * (ROWS + COLS) * 4, LOADS = A_LOADS + B_LOADS + S_LOADS;
    static_assert(4 % KS == 0 && S % 2 == 1, "the weights hold whole chunks; an even number of chunks in front of the last S of an odd number");
    static_assert(A_LOADS * 1024 * WAVES == A_BYTES && B_LOADS * 1024 * WAVES == B_BYTES && S >= 3 && (S - 1) * LOADS < 64,
                  "whole loads, counted in six bits");
    extern __shared__ __attribute__((aligned(16))) int8_t lds[];      // [S][BUFFER]
    __shared__ __attribute__((aligned(16))) float of_cols[COLS];      // biases, requested ahead of everything
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int in_group = wave % (WR * WC), k_group = wave / (WR * WC), wave_r = in_group / WC, wave_c = in_group % WC;
    // blockIdx % 8 is the XCD: each takes a run of consecutive tiles, which walk four row tiles before the next column tile
    const int tiles = p.row_tiles * p.col_tiles;
    const int t = int(blockIdx.x % 8) * p.tiles_per_xcd + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= p.tiles_per_xcd || t >= tiles) return;      // uniform, ahead of every barrier
    const int group = t / (4 * p.col_tiles), in_four = t - group * 4 * p.col_tiles;
    const int group_rows = min(4, p.row_tiles - 4 * group);
    const int tile_c = in_four / group_rows, tile_r = 4 * group + in_four - tile_c * group_rows;
    const int row0 = tile_r * ROWS, frag0 = tile_c * (COLS / 32);
    static_assert(COLS / 64 <= WAVES, "biases in one request a wavefront");
    if (wave < COLS / 64) {                                  // uniform, as the next
        const int first = wave * 64;
        if (p.bias) word_to_lds(reinterpret_cast<const uint8_t *>(p.bias + min(frag0 * 32 + first + lane, p.n - 1)), reinterpret_cast<int8_t *>(of_cols + first));
        else of_cols[first + lane] = -0.f;                   // changes no sum
    }

    // A row in LDS is its CHUNK bytes, its pieces of 16 XORed with bits of the row that make 16 rows cover all banks for one piece.  A
    // load instruction fills 1 KiB of such rows; rows beyond m are the last one again, never stored.  Pieces behind the end of a row are
    // its first one, against weights that are zero.  Scalar bases and 32-bit lane offsets.
    const auto key_of = [](int row) { return (row >> (KS == 1 ? 2 : KS == 2 ? 1 : 0)) & (PIECES - 1); };
    const int chunks = (p.x_steps + KS - 1) / KS;
    const uint8_t *const a_base = p.x + int64_t(row0) * p.x_pitch;
    unsigned a_off[A_LOADS], b_off[B_LOADS], s_off[S_LOADS];
    int a_piece[A_LOADS];
    static_for<0, A_LOADS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const int r = (wave * A_LOADS + i) * (64 / PIECES) + lane / PIECES;
        a_piece[i] = ((lane % PIECES) ^ key_of(r)) * 16;
        a_off[i] = unsigned(min(r, p.m - 1 - row0)) * unsigned(p.x_pitch);
    });
    static_for<0, B_LOADS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const int unit = wave * B_LOADS + i, step = unit / (2 * COLS / 32), in_step = unit % (2 * COLS / 32);
        const int frag = min(frag0 + in_step / 2, p.frags - 1);
        b_off[i] = unsigned(step * p.frags + frag) * 2048u + (in_step % 2) * 1024 + lane * 16;
    });
    // Scales in LDS: [K-step of the chunk][row], then [K-step of the chunk][column].  A request's K-steps lie s_stride apart, the last of them is
    // s_last; selects, no branches: all requests of a chunk are one run of instructions.
    const uint8_t *s_base[S_LOADS];
    int64_t s_stride[S_LOADS];
    int s_step[S_LOADS], s_last[S_LOADS];
    static_for<0, S_LOADS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const int unit = min(wave * S_LOADS + i, WORDS - 1), of_w = unit - A_WORDS;      // more wavefronts than requests: the last one again
        const bool is_x = unit < A_WORDS;
        s_step[i] = is_x ? unit / (ROWS / 64) : of_w / (COLS / 64);
        s_base[i] = is_x ? p.x_scales + int64_t(row0) * p.scale_row : reinterpret_cast<const uint8_t *>(p.w_scales) + frag0 * 128;
        s_stride[i] = is_x ? p.scale_step : int64_t(p.frags) * 128;
        s_last[i] = is_x ? p.x_steps - 1 : p.ksteps - 1;
        s_off[i] = is_x ? unsigned(min(unit % (ROWS / 64) * 64 + lane, p.m - 1 - row0)) * unsigned(p.scale_row)
                        : unsigned(min(of_w % (COLS / 64) * 64 + lane, (p.frags - frag0) * 32 - 1)) * 4u;
    });
    const int64_t b_step = int64_t(p.frags) * (KS * 2048);
    // request i of LOADS of a chunk
    auto request = [&](auto ic, int chunk, int buf) __attribute__((always_inline)) {
        constexpr int i = decltype(ic)::value;
        const int c = min(chunk, chunks - 1);                // behind the last chunk: that one again, not read from LDS
        int8_t *const at = lds + buf * BUFFER;
        if constexpr (i < A_LOADS) {
            const int k = c * CHUNK + a_piece[i];
            to_lds(reinterpret_cast<const int8_t *>(a_base) + (a_off[i] + unsigned(k < p.k ? k : 0)), at + (wave * A_LOADS + i) * 1024);
        } else if constexpr (i < A_LOADS + B_LOADS) {
            constexpr int j = i - A_LOADS;
            to_lds(p.w + c * b_step + b_off[j], at + A_BYTES + (wave * B_LOADS + j) * 1024);
        } else {
            constexpr int j = i - A_LOADS - B_LOADS;
            word_to_lds(s_base[j] + min(c * KS + s_step[j], s_last[j]) * s_stride[j] + s_off[j], at + SCALES + min(wave * S_LOADS + j, WORDS - 1) * 256);
        }
    };

    v16f acc[FR][FC];
    static_for<0, FR * FC>([&](auto fc) {
        constexpr int f = decltype(fc)::value;
        static_for<0, 16>([&](auto rc) { acc[f / FC][f % FC][decltype(rc)::value] = 0.f; });
    });
    const int a_row = (wave_r * FR * 32 + lane % 32) * CHUNK, a_key = key_of(lane % 32), upper = 8 * (lane / 32);
    int buf = 0, c = 0;
    // Few fragments: a chunk's operands are read all at once, a chunk ahead of its multiplications, so that these wait for nothing else in between (1024 x
    // 4096, K = 8192 in tiles of 128, the kernel alone on scales by K-steps, 31 -> 25 us).  Many: half a K-step ahead, which the registers hold without moving sums (8192^3 255 us, a chunk ahead 278).
    if constexpr (FR * FC <= 4) {
        constexpr int STEPS = KS / KG;                           // K-steps of a chunk that are this wavefront's; they lie together
        v4i a[2][HALVES][FR], b[2][HALVES][FC];
        int a_scale[2][STEPS][FR], b_scale[2][STEPS][FC];        // of a K-step: blocks l / 32 and 2 + l / 32 in bytes 0 and 2, once shifted
        constexpr int PER_HALF = FR + FC, READS = HALVES * PER_HALF + STEPS * PER_HALF;
        auto read = [&](auto sc, auto ic, int buf) __attribute__((always_inline)) {
            constexpr int set = decltype(sc)::value, n = decltype(ic)::value;
            const int8_t *const at = lds + buf * BUFFER;
            if constexpr (n < HALVES * PER_HALF) {
                constexpr int h = n / PER_HALF, i = n % PER_HALF;
                const int step = k_group * STEPS + h / 2;
                if constexpr (i < FC) b[set][h][i] = *reinterpret_cast<const v4i *>(at + A_BYTES + ((step * (COLS / 32) + wave_c * FC + i) * 2 + h % 2) * 1024 + lane * 16);
                else a[set][h][i - FC] = *reinterpret_cast<const v4i *>(at + a_row + (i - FC) * 32 * CHUNK + ((4 * step + 2 * (h % 2) + lane / 32) ^ a_key) * 16);
            } else {
                constexpr int u = (n - HALVES * PER_HALF) / PER_HALF, i = n % PER_HALF;
                const int step = k_group * STEPS + u;
                if constexpr (i < FC) b_scale[set][u][i] = *reinterpret_cast<const int *>(at + SCALES + (KS * ROWS + step * COLS + (wave_c * FC + i) * 32 + lane % 32) * 4);
                else a_scale[set][u][i - FC] = *reinterpret_cast<const int *>(at + SCALES + (step * ROWS + (wave_r * FR + i - FC) * 32 + lane % 32) * 4);
            }
        };
        static_for<0, S>([&](auto sc) { static_for<0, LOADS>([&](auto ic) { request(ic, decltype(sc)::value, decltype(sc)::value); }); });
        barrier_but_for<(S - 1) * LOADS>();
        // Which registers a chunk has goes by how many are left, so that the last ones are known to the code.
        if (chunks % 2) static_for<0, READS>([&](auto ic) { read(std::integral_constant<int, 0>{}, ic, 0); });
        else static_for<0, READS>([&](auto ic) { read(std::integral_constant<int, 1>{}, ic, 0); });
        // Between the multiplications of a chunk, one after each: the reads of the next chunk's operands, and the requests of the chunk S further on, into the
        // buffer that this chunk's operands came from.  Spread so, none of them keeps the matrix cores waiting for its turn to be issued.
        auto multiply = [&](auto sc, auto left) __attribute__((always_inline)) {
            constexpr int set = decltype(sc)::value, LEFT = decltype(left)::value, SLOTS = HALVES * FR * FC;      // LEFT: chunks from this one on; above S, more than S
            constexpr bool FETCHES = LEFT > S;
            const int after = buf + 1 == S ? 0 : buf + 1;
            // The next chunk is there for all behind the barrier, and every wavefront has this chunk's operands.
            if constexpr (LEFT > 1) barrier_but_for<(LEFT > S ? S - 2 : LEFT - 2) * LOADS>();
            int as[STEPS][FR], bs[STEPS][FC];
            static_for<0, STEPS>([&](auto uc) {
                constexpr int u = decltype(uc)::value;
                static_for<0, FR>([&](auto ic) { as[u][decltype(ic)::value] = int(unsigned(a_scale[set][u][decltype(ic)::value]) >> upper); });
                static_for<0, FC>([&](auto fc) { bs[u][decltype(fc)::value] = int(unsigned(b_scale[set][u][decltype(fc)::value]) >> upper); });
            });
            static_for<0, SLOTS>([&](auto fc) {
                constexpr int f = decltype(fc)::value, h = f / (FR * FC), i = f / FC % FR, j = f % FC;
                constexpr int R0 = READS * f / SLOTS, R1 = READS * (f + 1) / SLOTS, L0 = LOADS * f / SLOTS, L1 = LOADS * (f + 1) / SLOTS;
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(b[set][h][j]), operand(a[set][h][i]), acc[i][j], FP4, FP4, 2 * (h % 2), bs[h / 2][j],
                                                                            2 * (h % 2), as[h / 2][i]);
                if constexpr (LEFT > 1) static_for<R0, R1>([&](auto rc) { read(std::integral_constant<int, 1 - set>{}, rc, after); });
                if constexpr (FETCHES) static_for<L0, L1>([&](auto lc) { request(lc, c + S, buf); });
                __builtin_amdgcn_sched_barrier(0);
            });
            buf = after;
            ++c;
        };
        const std::integral_constant<int, 0> first;
        const std::integral_constant<int, 1> second;
        const std::integral_constant<int, S + 1> more;
        if (chunks > S && chunks % 2 == 0) multiply(second, more);
        while (chunks - c > S + 1) {
            multiply(first, more);
            multiply(second, more);
        }
        static_for<0, S>([&](auto rc) {                          // the last S chunks are all on their way
            constexpr int LEFT = S - decltype(rc)::value;
            if (chunks - c >= LEFT) multiply(std::integral_constant<int, (LEFT - 1) % 2>{}, std::integral_constant<int, LEFT>{});
        });
    } else {
        v4i a[2][FR], b[2][FC];
        int a_scale[2][FR], b_scale[2][FC];      // of a K-step: blocks l / 32 and 2 + l / 32 in bytes 0 and 2
        // read i of a half's operands; the scales of a K-step come with its first half
        constexpr int READS = 2 * (FR + FC);
        auto read = [&](auto hc, auto ic, int buf) __attribute__((always_inline)) {
            constexpr int h = decltype(hc)::value, i = decltype(ic)::value, set = h % 2;
            const int step = k_group * (KS / KG) + h / 2;      // a K group's K-steps of a chunk lie together
            const int8_t *const at = lds + buf * BUFFER;
            if constexpr (i < FC) {
                b[set][i] = *reinterpret_cast<const v4i *>(at + A_BYTES + ((step * (COLS / 32) + wave_c * FC + i) * 2 + h % 2) * 1024 + lane * 16);
            } else if constexpr (i < FC + FR) {
                constexpr int f = i - FC;
                a[set][f] = *reinterpret_cast<const v4i *>(at + a_row + f * 32 * CHUNK + ((4 * step + 2 * (h % 2) + lane / 32) ^ a_key) * 16);
            } else if constexpr (h % 2 == 0 && i < 2 * FC + FR) {
                constexpr int f = i - FC - FR;
                b_scale[h / 2 % 2][f] = *reinterpret_cast<const int *>(at + SCALES + (KS * ROWS + step * COLS + (wave_c * FC + f) * 32 + lane % 32) * 4);
            } else if constexpr (h % 2 == 0 && i < READS) {
                constexpr int f = i - 2 * FC - FR;
                a_scale[h / 2 % 2][f] = *reinterpret_cast<const int *>(at + SCALES + (step * ROWS + (wave_r * FR + f) * 32 + lane % 32) * 4);
            }
        };
        static_for<0, S - 1>([&](auto sc) { static_for<0, LOADS>([&](auto ic) { request(ic, decltype(sc)::value, decltype(sc)::value); }); });
        wait_for_all_but<(S - 2) * LOADS>();
        lds_barrier();
        static_for<0, READS>([&](auto ic) { read(std::integral_constant<int, 0>{}, ic, 0); });
        // A chunk.  Between its multiplications, one after each: the reads of the next half's operands, and the requests of the chunk S - 1 further on,
        // into the buffer that the barrier of the chunk before freed.  Spread so, none of them keeps the matrix cores waiting for its turn to be issued.
        auto multiply = [&](auto fetching) __attribute__((always_inline)) {
            constexpr bool FETCHES = decltype(fetching)::value;
            const int after = buf + 1 == S ? 0 : buf + 1, before = buf == 0 ? S - 1 : buf - 1;
            static_for<0, HALVES>([&](auto hc) {
                constexpr int h = decltype(hc)::value, SLOTS = FR * FC, FIRST = LOADS * h / HALVES, COUNT = LOADS * (h + 1) / HALVES - FIRST;
                int as[FR], bs[FC];
                static_for<0, FR>([&](auto ic) { as[decltype(ic)::value] = int(unsigned(a_scale[h / 2 % 2][decltype(ic)::value]) >> upper); });
                static_for<0, FC>([&](auto fc) { bs[decltype(fc)::value] = int(unsigned(b_scale[h / 2 % 2][decltype(fc)::value]) >> upper); });
                if constexpr (h + 1 == HALVES) {
                    // Every wavefront has its operands of this chunk in registers: its buffer is free behind the barrier, and the next
                    // chunk is there for all.  The rest of this chunk's arithmetic covers the first reads behind it.
                    barrier_but_for<FETCHES ? (S - 3) * LOADS + FIRST : 0>();
                }
                static_for<0, SLOTS>([&](auto fc) {
                    constexpr int f = decltype(fc)::value, i = f / FC, j = f % FC;
                    constexpr int R0 = READS * f / SLOTS, R1 = READS * (f + 1) / SLOTS, L0 = COUNT * f / SLOTS, L1 = COUNT * (f + 1) / SLOTS;
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(b[h % 2][j]), operand(a[h % 2][i]), acc[i][j], FP4, FP4, 2 * (h % 2), bs[j],
                                                                                2 * (h % 2), as[i]);
                    static_for<R0, R1>([&](auto rc) {
                        if constexpr (h + 1 == HALVES) read(std::integral_constant<int, 0>{}, rc, after);
                        else read(std::integral_constant<int, h + 1>{}, rc, buf);
                    });
                    if constexpr (FETCHES) static_for<FIRST + L0, FIRST + L1>([&](auto lc) { request(lc, c + S - 1, before); });
                    __builtin_amdgcn_sched_barrier(0);
                });
            });
            buf = after;
        };
        for (; c + S - 1 < chunks; ++c) multiply(std::true_type{});
        for (; c < chunks; ++c) multiply(std::false_type{});      // the last S - 1 chunks are all on their way
    }
    // The chunks' LDS is free: nothing is on its way into it, and behind this barrier nobody reads it.
    wait_for_all_but<0>();
    lds_barrier();
    constexpr int SUMS = FR * FC * 4096;                     // of a wavefront's fragments
    if constexpr (KG > 1) {                                  // the first group adds up all groups' sums, in their order
        float *const sums = reinterpret_cast<float *>(lds) + lane;
        const int mine = in_group * (SUMS / 4);
        if (k_group > 0)
            static_for<0, FR * FC>([&](auto fc) {
                constexpr int f = decltype(fc)::value;
                static_for<0, 16>([&](auto rc) { sums[(k_group - 1) * (WR * WC * SUMS / 4) + mine + f * 1024 + decltype(rc)::value * 64] = acc[f / FC][f % FC][decltype(rc)::value]; });
            });
        lds_barrier();
        if (k_group > 0) return;
        static_for<1, KG>([&](auto gc) {
            static_for<0, FR * FC>([&](auto fc) {
                constexpr int f = decltype(fc)::value;
                static_for<0, 16>([&](auto rc) { acc[f / FC][f % FC][decltype(rc)::value] += sums[(decltype(gc)::value - 1) * (WR * WC * SUMS / 4) + mine + f * 1024 + decltype(rc)::value * 64]; });
            });
        });
    }
    // A wavefront's 32 tokens x 32 FC columns go through LDS, so that a store instruction writes whole cache lines (straight from the registers it would
    // write 16 bytes of each of 64 runs).
    constexpr int SIZE = OUT == TSX_TYPE_F32 ? 4 : 2, ROW = FC * 32 * SIZE, PITCH = ROW + 16, IN_ROW = ROW / 16, AT_ONCE = 64 / IN_ROW, EACH = 16 / SIZE;
    constexpr int BEHIND = (KG - 1) * WR * WC * SUMS, AREAS = FR > 1 && BEHIND + WR * WC * 64 * PITCH <= S * BUFFER ? 2 : 1;      // 32 tokens on their way out while the next are computed, where there is room
    static_assert(BEHIND + WR * WC * AREAS * 32 * PITCH <= S * BUFFER, "room for all wavefronts");
    int8_t *const mine = lds + BEHIND + in_group * (AREAS * 32 * PITCH);
    const int col = (frag0 + wave_c * FC) * 32 + lane % IN_ROW * EACH, left = p.n - col;      // where a lane stores
    const bool inside = row0 + ROWS <= p.m && frag0 * 32 + COLS <= p.n;      // no test of rows and columns then: 4096 x 4096, K = 256 11.3 -> 9.9 us
    by_act(p.act, [&](auto act) __attribute__((always_inline)) {
        static_for<0, FR>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            const int in_tile = (wave_r * FR + i) * 32;
            int8_t *const area = mine + i % AREAS * (32 * PITCH);
            static_for<0, FC>([&](auto fc) {
                constexpr int f = decltype(fc)::value;
                float v[16];
                static_for<0, 4>([&](auto gc) {
                    constexpr int g = decltype(gc)::value;
                    const v4f bias = *reinterpret_cast<const v4f *>(of_cols + (wave_c * FC + f) * 32 + 8 * g + 4 * (lane / 32));
                    static_for<0, 4>([&](auto jc) { constexpr int j = decltype(jc)::value; v[4 * g + j] = __fadd_rn(acc[i][f][4 * g + j], bias[j]); });
                });
                activate_as<OUT, decltype(act)::value>(v, p.slope);
                const Run<OUT, 16> to = fragment_values<OUT>(v);
                v4u *const at = reinterpret_cast<v4u *>(area + lane % 32 * PITCH + (f * 32 + 16 * (lane / 32)) * SIZE);
                static_for<0, SIZE>([&](auto wc) { constexpr int w = 4 * decltype(wc)::value; at[w / 4] = v4u{to.word[w], to.word[w + 1], to.word[w + 2], to.word[w + 3]}; });
            });
            static_for<0, 32 / AT_ONCE>([&](auto kc) {
                const int r = decltype(kc)::value * AT_ONCE + lane / IN_ROW, row = row0 + in_tile + r;
                Run<OUT, EACH> to;
                const v4u got = *reinterpret_cast<const v4u *>(area + r * PITCH + lane % IN_ROW * 16);
                static_for<0, 4>([&](auto wc) { to.word[decltype(wc)::value] = got[decltype(wc)::value]; });
                char *const out = static_cast<char *>(p.out) + (int64_t(row) * p.out_stride + col) * SIZE;
                if (inside && p.streams) {                   // uniform
                    asm volatile("; past the caches");       // keeps the two stores from becoming one
                    to.template store<true>(out);
                } else if (inside) {
                    to.store(out);
                } else if (row < p.m) {
                    if (left >= EACH) to.store(out);
                    else if (left > 0) to.store_some(out, left);
                }
            });
        });
    });
}

// ---- few tokens: a stream over the weights
//
// There the product reads 17 / 32 n k bytes of weights and does little with each.  A workgroup owns 16 output columns of 16 tokens and its wavefronts split K,
// every WAVES-th K-step each; a K-step of 16 columns is one 16-byte load a lane and a word of scales, AHEAD of them in flight from the first instruction
// on.  X, the type of the rows: MXFP4, or floats, which a wavefront quantizes where it needs them: a K-step of 16 rows is four requests of whole cache lines,
// eight values a lane, four lanes a block, and its codes change lanes through the wavefront's own LDS.  Nothing there has to meet another wavefront, so
// there is no launch ahead of the product and no barrier in it before the partial sums meet.  16x16x128 instruction: accumulator r of lane l is
// column 4 (l / 16) + r of token l % 16.  4096 columns, K = 4096: one bf16 token 4.1 us, 16 MXFP4 tokens 5.1, of which the weights' bytes are 1.1 and the
// rest the launch, the first loads' way and the sums through LDS.
constexpr int FEW = 16, FEW_MOST = 1 << 14;      // rows up to which the stream is taken: its estimate is fitted to 8192 (a launch's second axis holds groups of 16 up to 2^20)

struct FewTokens : MxGemmParams {
    const void *values;                // rows of floats
    int64_t x_stride;
    int cols;                          // values of such a row
};

// What a wavefront writes to its own LDS it reads in that order, without a wait: the compiler is not to change it.
__device__ __forceinline__ void wavefront_order() { __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local"); }
template <int N>
__device__ __forceinline__ void put(const Run<N, 8> &v, char *at) {
    static_for<0, Run<N, 8>::WORDS / 4>([&](auto wc) { constexpr int w = 4 * decltype(wc)::value; reinterpret_cast<v4u *>(at)[w / 4] = v4u{v.word[w], v.word[w + 1], v.word[w + 2], v.word[w + 3]}; });
}
template <int N>
__device__ __forceinline__ void get(Run<N, 8> &v, const char *at) {
    static_for<0, Run<N, 8>::WORDS / 4>([&](auto wc) {
        constexpr int w = 4 * decltype(wc)::value;
        const v4u q = reinterpret_cast<const v4u *>(at)[w / 4];
        static_for<0, 4>([&](auto jc) { v.word[w + decltype(jc)::value] = q[decltype(jc)::value]; });
    });
}

// G: of a workgroup's rows of floats, in fours, those that are there: one, or all
template <int X, int G, int WAVES, int AHEAD, int OUT>
__global__ __launch_bounds__(WAVES * 64) void gemm_mxfp4_few_kernel(FewTokens p) {
    constexpr bool FLOATS = X != TSX_TYPE_MXFP4;
    // of a wavefront in LDS: a K-step, codes and scales of four rows or values of 16; then its sums [4][64]
    constexpr int OWN = !FLOATS || G == 1 ? 1024 : 16 * MX_STEP * (X == TSX_TYPE_F32 ? 4 : 2);
    __shared__ __attribute__((aligned(16))) char lds[WAVES * OWN];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), block = lane / 16, row = lane % 16;
    // blockIdx % 8 is the XCD: each takes a run of columns, so that no two L2s have parts of an output's cache line
    const int col16 = int(blockIdx.x % 8) * p.tiles_per_xcd + int(blockIdx.x / 8), row0 = int(blockIdx.y) * FEW;      // in columns of 16
    if (16 * col16 >= p.n) return;                           // uniform, ahead of the barriers
    const int8_t *const w = p.w + int64_t(col16 >> 1) * 2048 + (block >> 1) * 1024 + (16 * (col16 & 1) + row + 32 * (block & 1)) * 16;
    const int8_t *const ws = p.w_scales + (col16 * 16 + row) * 4;
    const int64_t w_step = int64_t(p.frags) * 2048, ws_step = int64_t(p.frags) * 128;
    v4i a[AHEAD];
    unsigned as[AHEAD];
    auto fetch = [&](int first) __attribute__((always_inline)) {
        static_for<0, AHEAD>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            const int step = min(first + WAVES * u, p.x_steps - 1);
            a[u] = *reinterpret_cast<const v4i *>(w + step * w_step);
            as[u] = *reinterpret_cast<const unsigned *>(ws + step * ws_step);
        });
    };
    fetch(wave);
    char *const mine = lds + wave * OWN;
    v4f acc = {0.f, 0.f, 0.f, 0.f};
    for (int first = wave; first < p.x_steps; first += WAVES * AHEAD) {
        v4i b[AHEAD];
        unsigned bs[AHEAD];
        if constexpr (FLOATS) {
            constexpr int SIZE = X == TSX_TYPE_F32 ? 4 : 2;
            typedef Run<X, 8> Values;
            Values v[G][AHEAD];
            static_for<0, G * AHEAD>([&](auto ic) {          // all requests at once; here `row` counts a K-step's pieces, `block` rows
                constexpr int i = decltype(ic)::value / AHEAD, u = decltype(ic)::value % AHEAD;
                const char *const x = static_cast<const char *>(p.values) + min(row0 + 4 * i + block, p.m - 1) * p.x_stride * SIZE;
                const int k = min(first + WAVES * u, p.x_steps - 1) * MX_STEP + 8 * row;
                if (p.cols >= 8) {                           // uniform
                    load_piece<X>(v[i][u], x, k, p.cols);
                } else {
                    v[i][u].clear();
                    if (k == 0) v[i][u].load_some(x, p.cols);
                }
            });
            const auto larger = [](unsigned one, unsigned other) { return Values::template larger<X>(one, other); };
            static_for<0, AHEAD>([&](auto uc) {
                constexpr int u = decltype(uc)::value;
                const int step = first + WAVES * u;
                if (u > 0 && step >= p.x_steps) return;      // uniform
                if ((step + 1) * MX_STEP > p.cols && p.cols >= 8) static_for<0, G>([&](auto ic) { settle_piece<X>(v[decltype(ic)::value][u], step * MX_STEP + 8 * row, p.cols); });
                if constexpr (G == 1) {                      // four lanes a block, before its codes change lanes
                    const unsigned scale = mx_scale(top_value<X>(over_lanes(v[0][u].top(0), 2, larger)));
                    *reinterpret_cast<unsigned *>(mine + block * KSTEP + 4 * row) = mx_codes<X>(v[0][u], scale);
                    if (row % 4 == 0) mine[4 * KSTEP + block * 4 + row / 4] = char(scale);
                    wavefront_order();
                    b[u] = *reinterpret_cast<const v4i *>(mine + row % 4 * KSTEP + block * 16);
                    bs[u] = static_cast<unsigned char>(mine[4 * KSTEP + row % 4 * 4 + block]);
                } else {                                     // values change lanes; a piece's place is XORed with its row, so that 16 rows cover all banks
                    constexpr int PIECE = 8 * SIZE;
                    static_for<0, 4>([&](auto ic) {
                        constexpr int i = decltype(ic)::value;
                        put(v[i][u], mine + ((4 * i + block) * 16 + (row ^ (4 * i + block))) * PIECE);
                    });
                    wavefront_order();
                    Values own[4];
                    unsigned top = 0;
                    static_for<0, 4>([&](auto qc) { constexpr int q = decltype(qc)::value; get(own[q], mine + (row * 16 + ((4 * block + q) ^ row)) * PIECE); });
                    static_for<0, 4>([&](auto qc) { top = own[decltype(qc)::value].top(top); });
                    bs[u] = mx_scale(top_value<X>(top));
                    static_for<0, 4>([&](auto qc) { constexpr int q = decltype(qc)::value; b[u][q] = int(mx_codes<X>(own[q], bs[u])); });
                }
                wavefront_order();
            });
        } else {
            const int token = min(row0 + row, p.m - 1);
            static_for<0, AHEAD>([&](auto uc) {
                constexpr int u = decltype(uc)::value;
                const int step = min(first + WAVES * u, p.x_steps - 1);
                b[u] = *reinterpret_cast<const v4i *>(p.x + token * p.x_pitch + (step * KSTEP + block * 16));
                bs[u] = p.x_scales[token * p.scale_row + step * p.scale_step + block];
            });
        }
        static_for<0, AHEAD>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            if (first + WAVES * u < p.x_steps)               // uniform
                acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(a[u]), operand(b[u]), acc, FP4, FP4, 0, int(as[u] >> (8 * block)), 0, int(bs[u]));
        });
        if (first + WAVES * AHEAD < p.x_steps) fetch(first + WAVES * AHEAD);
    }
    static_for<0, 4>([&](auto rc) { reinterpret_cast<float *>(mine)[decltype(rc)::value * 64 + lane] = acc[decltype(rc)::value]; });
    __syncthreads();
    const int in = threadIdx.x % 16, col = col16 * 16 + in, to = threadIdx.x / 16;
    if (to >= FEW || row0 + to >= p.m || col >= p.n) return;
    float v[1] = {0.f};
#pragma unroll
    for (int i = 0; i < WAVES; ++i) v[0] = __fadd_rn(v[0], reinterpret_cast<const float *>(lds + i * OWN)[in % 4 * 64 + to + 16 * (in / 4)]);
    if (p.bias) v[0] = __fadd_rn(v[0], p.bias[col]);
    activate_tokens<OUT>(v, p.act, p.slope);
    Run<OUT, 1> out;
    out.set(v);
    out.store(static_cast<char *>(p.out) + ((row0 + to) * p.out_stride + col) * (OUT == TSX_TYPE_F32 ? 4 : 2));
}

// 16 bytes of a row's codes from byte `at` on, zeros behind its end, and for what stands behind an odd number of values in its last byte
__device__ __forceinline__ v4i row_codes(const uint8_t *row, int64_t at, int k) {
    const int left = int(min(k - 2 * at, int64_t(32)));      // values
    if (left == 32) return __builtin_bit_cast(v4i, v4u(*reinterpret_cast<const v4u_any *>(row + at)));
    unsigned word[4];
    static_for<0, 4>([&](auto wc) {
        constexpr int w = decltype(wc)::value;
        word[w] = 0;
        static_for<0, 4>([&](auto bc) {
            constexpr int b = 4 * w + decltype(bc)::value;
            if (2 * b < left) word[w] |= unsigned(row[at + b] & (2 * b + 1 < left ? 0xff : 0x0f)) << (8 * (b % 4));
        });
    });
    return v4i{int(word[0]), int(word[1]), int(word[2]), int(word[3])};
}

// codes and scales of weights [n][k] to the layout above
__global__ __launch_bounds__(256) void pack_mxfp4_kernel(const uint8_t *codes, int64_t codes_stride, const uint8_t *scales, int64_t scales_stride, int n,
                                                         int k, int blocks, int frags, int64_t pieces, int64_t words, int8_t *packed) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < pieces + words; i += int64_t(gridDim.x) * 256) {
        if (i < pieces) {
            const int lane = int(i % 64);
            const int64_t unit = i / 64, step = unit / 2 / frags;
            const int half = int(unit % 2), frag = int(unit / 2 - step * frags);
            const int col = frag * 32 + lane % 32;
            const int64_t at = step * KSTEP + (2 * half + lane / 32) * 16;
            v4i v = {0, 0, 0, 0};
            if (col < n) v = row_codes(codes + col * codes_stride, at, k);
            reinterpret_cast<v4i *>(packed)[i] = v;
        } else {
            const int64_t word = i - pieces, step = word / (frags * 32);
            const int col = int(word - step * (frags * 32));
            unsigned v = 0;
            for (int b = 0; b < 4; ++b)
                if (col < n && step * 4 + b < blocks) v |= unsigned(scales[col * scales_stride + step * 4 + b]) << (8 * b);
            reinterpret_cast<unsigned *>(packed + pieces * 16)[word] = v;
        }
    }
}

// MXFP4 rows of another length, stride or alignment than the kernels read: codes to whole K-steps, scales to words of K-steps
__global__ __launch_bounds__(256) void copy_mxfp4_kernel(const uint8_t *codes, int64_t codes_stride, const uint8_t *scales, int64_t scales_stride, int k,
                                                         int blocks, int64_t rows, int steps, uint8_t *to, uint8_t *to_scales) {
    const int64_t pitch = int64_t(steps) * KSTEP, pieces = rows * steps * 4, words = rows * steps;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < pieces + words; i += int64_t(gridDim.x) * 256) {
        if (i < pieces) {
            const int64_t row = i / (steps * 4);
            const int at = int(i - row * (steps * 4)) * 16;
            *reinterpret_cast<v4i *>(to + row * pitch + at) = row_codes(codes + row * codes_stride, at, k);
        } else {
            const int64_t word = i - pieces, step = word / rows, row = word - step * rows;
            unsigned v = 0;
            for (int b = 0; b < 4; ++b)
                if (step * 4 + b < blocks) v |= unsigned(scales[row * scales_stride + step * 4 + b]) << (8 * b);
            reinterpret_cast<unsigned *>(to_scales)[word] = v;
        }
    }
}

// Rows of scales, whole words at multiples of 4, to words of K-steps: a lane has four words of a row
__global__ __launch_bounds__(256) void turn_scales_kernel(const uint8_t *scales, int64_t stride, int64_t rows, int steps, unsigned *to) {
    const int64_t row = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int first = int(blockIdx.y) * 4;
    if (row >= rows) return;
    const unsigned *const from = reinterpret_cast<const unsigned *>(scales + row * stride) + first;
    unsigned word[4];
    static_for<0, 4>([&](auto uc) { constexpr int u = decltype(uc)::value; word[u] = from[min(u, steps - 1 - first)]; });
    static_for<0, 4>([&](auto uc) {
        constexpr int u = decltype(uc)::value;
        if (first + u < steps) to[int64_t(first + u) * rows + row] = word[u];
    });
}

template <int WR, int WC, int FR, int FC, int KS, int S, int KG, int OUT>
int launch_tile(MxGemmParams p, hipStream_t stream) {
    p.row_tiles = int(ceil_div(p.m, 32 * WR * FR));
    p.col_tiles = int(ceil_div(p.n, 32 * WC * FC));
    const int64_t per_xcd = ceil_div(int64_t(p.row_tiles) * p.col_tiles, 8);
    TSX_REQUIRE(8 * per_xcd * WR * WC * KG * 64 < int64_t(1) << 32, "gemm_mxfp4: %d x %d outputs are more than a launch holds", p.m, p.n);
    p.tiles_per_xcd = int(per_xcd);
    // Outputs of more than 64 MiB go past the caches: what reads them next finds little there, and the product ends sooner.  The product and a norm of its
    // outputs, with and without (us): 33 MB 32.8 and 31.1, 67 MB 51.7 and 51.2, 134 MB 336 and 357.
    p.streams = int64_t(p.m) * p.n * int64_t(element_bytes(OUT)) > 64 << 20;
    constexpr int LDS = S * 32 * (WR * FR + WC * FC) * KS * (KSTEP + 4);
    const auto kernel = gemm_mxfp4_kernel<WR, WC, FR, FC, KS, S, KG, OUT>;
    if (LDS > 64 * 1024) {
        const int rc = grant_lds(reinterpret_cast<const void *>(kernel), LDS);
        if (rc) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(unsigned(8 * p.tiles_per_xcd)), dim3(WR * WC * KG * 64), LDS, stream, p);
    TSX_LAUNCH_CHECK("gemm_mxfp4_kernel");
    return 0;
}

template <int X, int G, int WAVES, int AHEAD, int OUT>
int launch_few(FewTokens p, hipStream_t stream) {
    p.tiles_per_xcd = int(ceil_div(p.n, 128));
    hipLaunchKernelGGL((gemm_mxfp4_few_kernel<X, G, WAVES, AHEAD, OUT>), dim3(unsigned(8 * p.tiles_per_xcd), unsigned(ceil_div(p.m, FEW))), dim3(WAVES * 64), 0, stream, p);
    TSX_LAUNCH_CHECK("gemm_mxfp4_few_kernel");
    return 0;
}
template <int X, int OUT>
int few_of(const FewTokens &p, hipStream_t stream) {
    // 16 wavefronts where K is long and the registers allow it: each has four K-steps up to K = 8192, all of them on their way at once
    if constexpr (X != TSX_TYPE_MXFP4)
        if (p.m > 4) return launch_few<X, 4, 8, X == TSX_TYPE_F32 ? 2 : 4, OUT>(p, stream);
    return p.x_steps > 32 ? launch_few<X, 1, 16, 4, OUT>(p, stream) : launch_few<X, 1, 8, 4, OUT>(p, stream);
}
template <int OUT>
int few_tokens(const tsx_mxfp4_gemm *g, const MxGemmParams &q, hipStream_t stream) {
    FewTokens p{};
    static_cast<MxGemmParams &>(p) = q;
    p.values = g->x_dev;
    p.x_stride = g->m <= 1 ? 0 : g->x_stride;
    p.cols = g->k;
    return g->x_type == TSX_TYPE_F32    ? few_of<TSX_TYPE_F32, OUT>(p, stream)
           : g->x_type == TSX_TYPE_F16  ? few_of<TSX_TYPE_F16, OUT>(p, stream)
           : g->x_type == TSX_TYPE_BF16 ? few_of<TSX_TYPE_BF16, OUT>(p, stream) : few_of<TSX_TYPE_MXFP4, OUT>(p, stream);
}

// The kernel a call takes, by an estimate of its time in us, fitted to products of 16 .. 8192 rows on 256 .. 8192 columns and K of 256 .. 8192 (bf16).
// r: workgroups or tiles a CU, ks: K / 1024.  MXFP4 rows: up to 16 the stream over the weights, else tiles.  Those of 64 with K split over two groups of
// wavefronts take a CU each, so they are for up to 256; those of 64 and 128 share CUs, so that their times go by r once they fill the card and by the length
// of K before; those of 256 columns come in whole turns, which a card half full goes through faster.  Measured (us), tiles of 64 by K, of 64, 128, 128 x
// 256 and 256: 64 x 4096, K = 4096 6.4, 6.8, 11, 16, 24; 256 x 4096, K = 4096 6.9, 6.9, 11, 17, 24; 512 x 4096, K = 4096 13, 10.5, 13, 17, 26; 512 x 8192, K =
// 1024 14, 8, 6.9, 8, 11; 1024 x 1024, K = 8192 10.4, 11.6, 22, 29, 43; 1024 x 4096, K = 4096 25, 21, 17, 19, 28; 2048 x 4096, K = 4096 46, 36, 28, 25, 30; 4096^3
// 94, 70, 47, 46, 41; 8192^3 580, 530, 325, 303, 265.
// Rows of floats: the stream, which quantizes them itself, against tiles behind a launch that does, 3 us and the rows' bytes.  The stream is a workgroup a CU
// at a time (of up to four rows, several, and always it); the stream and what tiles took with their launch: 64 x 1024, K = 1024 4.3 and 7.4, 128 x 1024 7.0
// and 7.5; 256 x 256, K = 256 4.0 and 7.2; 128 x 300, K = 4096 5.8 and 9.2; 32 x 4096, K = 300 6.5 and 7.7; 16 x 8192, K = 8192 15.7 and 12.4.
enum class Kernel { few, tile_64_by_k, tile_64, tile_128, tile_256, tile_128_256 };

Kernel choose(const tsx_mxfp4_gemm *g) {
    const int m = g->m, n = g->n, k = g->k;
    const bool floats = g->x_type != TSX_TYPE_MXFP4;
    if (m <= (floats ? 4 : FEW)) return Kernel::few;
    const float ks = float(k) / 1024.f;
    const auto rounds = [&](int rows, int cols) { return float(ceil_div(m, rows) * ceil_div(n, cols)) / 256.f; };
    const float r16 = rounds(FEW, 16), r64 = rounds(64, 64), r128 = rounds(128, 128), r256 = rounds(256, 256), r128_256 = rounds(128, 256);
    const float cost[] = {r64 <= 1.f ? 3.6f + ks * (0.72f + 0.15f * r64) : INFINITY, std::max(3.4f + 0.88f * ks, 2.8f + r64 * (0.42f + 0.97f * ks)),
                          std::max(3.7f + 1.82f * ks, 3.f + 0.4f * ks + r128 * (0.75f + 2.75f * ks)),
                          3.f + std::ceil(r256) * (7.7f + 7.65f * ks) * (0.5f + 0.5f * std::min(r256, 1.f)),
                          3.f + std::ceil(r128_256) * (3.2f + 4.65f * ks) * (0.54f + 0.46f * std::min(r128_256, 1.f))};
    int best = 0;
    for (int i = 1; i < 5; ++i)
        if (cost[i] < cost[best]) best = i;
    if (floats && m <= FEW_MOST) {
        const float few = 1.2f + std::ceil(r16) * (2.4f + 0.55f * ks);
        if (few < cost[best] + 3.f + float(m) * float(k) * 5e-7f) return Kernel::few;
    }
    return Kernel(best + 1);
}

template <int OUT>
int launch(Kernel kernel, const tsx_mxfp4_gemm *g, const MxGemmParams &p, hipStream_t stream) {
    switch (kernel) {
        case Kernel::few: return few_tokens<OUT>(g, p, stream);
        case Kernel::tile_64_by_k: return launch_tile<2, 2, 1, 1, 4, 3, 2, OUT>(p, stream);
        case Kernel::tile_64: return launch_tile<2, 2, 1, 1, 2, 3, 1, OUT>(p, stream);
        case Kernel::tile_128: return launch_tile<2, 2, 2, 2, 1, 3, 1, OUT>(p, stream);
        case Kernel::tile_128_256: return launch_tile<2, 4, 2, 2, 1, 3, 1, OUT>(p, stream);
        default: return launch_tile<2, 4, 4, 2, 1, 3, 1, OUT>(p, stream);
    }
}

int check(const tsx_mxfp4_gemm *g) {
    TSX_REQUIRE(g, "gemm_mxfp4: null argument");
    TSX_REQUIRE(g->m >= 0 && g->n > 0 && g->k > 0, "gemm_mxfp4: bad extents");
    TSX_REQUIRE(g->m < 1 << 28 && g->n < 1 << 24 && g->k < 1 << 21, "gemm_mxfp4: %d rows, %d columns, K = %d (below 2^28, 2^24 and 2^21)", g->m, g->n, g->k);
    TSX_REQUIRE(is_float_type(g->x_type) || g->x_type == TSX_TYPE_MXFP4, "gemm_mxfp4: element type %d", g->x_type);
    TSX_REQUIRE(is_float_type(g->out_type), "gemm_mxfp4: output type %d (fp32, fp16 or bf16)", g->out_type);
    TSX_REQUIRE(is_token_act(g->act), "gemm_mxfp4: activation %d", g->act);
    const bool codes = g->x_type == TSX_TYPE_MXFP4;
    TSX_REQUIRE(g->m <= 1 || (g->x_stride >= (codes ? (g->k + 1) / 2 : g->k) && g->out_stride >= g->n && (!codes || g->x_scales_stride >= (g->k + 31) / 32)),
                "gemm_mxfp4: rows of %d and %d columns overlap at strides %lld, %lld and %lld", g->k, g->n, (long long)g->x_stride, (long long)g->x_scales_stride,
                (long long)g->out_stride);
    return 0;
}

bool is_multiple(const void *at, size_t bytes) { return reinterpret_cast<uintptr_t>(at) % bytes == 0; }

// A tile's rows are reached by 32-bit offsets: 256 of them at 2^23.
bool reads_in_place(const tsx_mxfp4_gemm *g) {
    return g->x_type == TSX_TYPE_MXFP4 && g->k % MX_STEP == 0 && is_multiple(g->x_dev, 16) && is_multiple(g->x_scales_dev, 4) &&
           (g->m <= 1 || (g->x_stride % 16 == 0 && g->x_stride <= 1 << 23 && g->x_scales_stride % 4 == 0 && g->x_scales_stride <= 1 << 23));
}

// What a call does: its kernel, and whether the workspace holds its rows, codes [m][steps][64] and scales [steps][m][4], or such scales alone.
struct Plan {
    Kernel kernel;
    bool copies, turns;
    int64_t steps, code_bytes, word_bytes;      // word_bytes: of a K-step's scales
    explicit Plan(const tsx_mxfp4_gemm *g) {
        kernel = choose(g);
        // TSX_MXFP4_KERNEL: that kernel, by its place in the list above, for any call it can take (tests, measurements)
        const char *e = std::getenv("TSX_MXFP4_KERNEL");
        if (e && e[0] >= (g->m <= FEW_MOST ? '0' : '1') && e[0] <= '5') kernel = Kernel(e[0] - '0');
        steps = ceil_div(g->k, MX_STEP);
        copies = g->m > 0 && !reads_in_place(g) && (kernel != Kernel::few || g->x_type == TSX_TYPE_MXFP4);
        // Rows of scales cost a tile a request of 64 cache lines where words of K-steps are four: 0.09 us a K-step in tiles of 128, 0.15 in those of 256.
        // A launch that turns them is worth 4 us of that (us, without and with: 8192^3 291 and 267, 1024 x 4096, K = 8192 34.5 and 30.5, 2048 17 and 18).
        // Tiles of 128 x 256 have half the rows to a multiplication, and no second tile beside them that waits too: 34 and 36 at 2048 x 4096, K = 6144.
        const int side = kernel == Kernel::tile_256 ? 256 : 128;
        const float tiles = std::max(1.f, float(ceil_div(g->m, side) * ceil_div(g->n, side)) / 256.f);
        turns = g->m > 0 && !copies && (kernel == Kernel::tile_128 || kernel == Kernel::tile_256) && float(steps) * tiles * (side == 256 ? 0.15f : 0.09f) > 4.f;
        code_bytes = copies ? g->m * steps * KSTEP : 0;
        word_bytes = int64_t(g->m) * 4;
    }
    size_t workspace_bytes() const { return copies || turns ? size_t(code_bytes + word_bytes * steps) : 0; }
};

int check_weights(int32_t k, int32_t n) {
    TSX_REQUIRE(k > 0 && n > 0 && k < 1 << 21 && n < 1 << 24, "gemm_mxfp4: weights of %d columns, K = %d (below 2^24 and 2^21)", n, k);
    return 0;
}

}  // namespace
}  // namespace tsx

extern "C" {

size_t tsx_gemm_mxfp4_packed_weight_bytes(int32_t k, int32_t n) {
    if (tsx::check_weights(k, n)) return 0;
    return size_t(tsx::packed_codes(k, n)) + size_t(tsx::ksteps_of(k)) * tsx::frags_of(n) * 128;
}

int tsx_gemm_mxfp4_pack_weights(int32_t k, int32_t n, const uint8_t *codes_dev, int64_t codes_stride, const uint8_t *scales_dev, int64_t scales_stride,
                                void *packed_dev, void *stream) {
    if (const int rc = tsx::check_weights(k, n)) return rc;
    TSX_REQUIRE(n <= 1 || (codes_stride >= (k + 1) / 2 && scales_stride >= (k + 31) / 32), "gemm_mxfp4: rows of K = %d overlap at strides %lld and %lld", k,
                (long long)codes_stride, (long long)scales_stride);
    TSX_REQUIRE(codes_dev && scales_dev && packed_dev, "gemm_mxfp4: null pointer");
    TSX_REQUIRE(tsx::is_multiple(packed_dev, 16), "gemm_mxfp4: packed weights must be 16-byte aligned");
    const int64_t pieces = tsx::packed_codes(k, n) / 16, words = int64_t(tsx::ksteps_of(k)) * tsx::frags_of(n) * 32;
    const int64_t blocks = std::min<int64_t>(tsx::ceil_div(pieces + words, 256), 1 << 16);
    hipLaunchKernelGGL(tsx::pack_mxfp4_kernel, dim3(unsigned(blocks)), dim3(256), 0, tsx::as_stream(stream), codes_dev, codes_stride, scales_dev, scales_stride,
                       n, k, (k + 31) / 32, tsx::frags_of(n), pieces, words, static_cast<int8_t *>(packed_dev));
    TSX_LAUNCH_CHECK("pack_mxfp4_kernel");
    return 0;
}

size_t tsx_gemm_mxfp4_workspace_bytes(const tsx_mxfp4_gemm *g) {
    if (tsx::check(g)) return 0;
    return tsx::Plan(g).workspace_bytes();
}

int tsx_gemm_mxfp4(const tsx_mxfp4_gemm *g, void *workspace_dev, size_t workspace_bytes, void *stream_) {
    int rc = tsx::check(g);
    if (rc || g->m == 0) return rc;
    const bool codes = g->x_type == TSX_TYPE_MXFP4;
    TSX_REQUIRE(g->x_dev && g->packed_w_dev && g->out_dev, "gemm_mxfp4: null pointer");
    TSX_REQUIRE(!codes || g->x_scales_dev, "gemm_mxfp4: MXFP4 rows need their scales");
    TSX_REQUIRE(tsx::is_multiple(g->packed_w_dev, 16), "gemm_mxfp4: packed weights must be 16-byte aligned");
    TSX_REQUIRE((codes || tsx::is_multiple(g->x_dev, tsx::element_bytes(g->x_type))) && tsx::is_multiple(g->out_dev, tsx::element_bytes(g->out_type)) &&
                    tsx::is_multiple(g->bias_dev, 4), "gemm_mxfp4: pointer is no multiple of its elements");
    const tsx::Plan plan(g);
    const size_t need = plan.workspace_bytes();
    if (need) {
        if (!workspace_dev || workspace_bytes < need)
            return tsx::fail(TSX_E_WORKSPACE, "gemm_mxfp4: workspace %zu < %zu bytes", workspace_dev ? workspace_bytes : size_t(0), need);
        TSX_REQUIRE(tsx::is_multiple(workspace_dev, 16), "gemm_mxfp4: workspace must be 16-byte aligned");
    }
    hipStream_t stream = tsx::as_stream(stream_);
    tsx::MxGemmParams p{};
    const int steps = int(plan.steps);
    p.x_steps = steps;
    p.k = steps * tsx::KSTEP;
    if (plan.copies) {
        uint8_t *const to = static_cast<uint8_t *>(workspace_dev), *const to_scales = to + plan.code_bytes;
        p.x = to;
        p.x_scales = to_scales;
        p.x_pitch = p.k;
        p.scale_row = 4;
        p.scale_step = plan.word_bytes;
        if (codes) {
            const int64_t units = int64_t(g->m) * steps * 5, blocks = tsx::ceil_div(units, 256);
            hipLaunchKernelGGL(tsx::copy_mxfp4_kernel, dim3(unsigned(std::min<int64_t>(blocks, 1 << 16))), dim3(256), 0, stream, static_cast<const uint8_t *>(g->x_dev),
                               g->x_stride, g->x_scales_dev, g->x_scales_stride, g->k, (g->k + 31) / 32, int64_t(g->m), steps, to, to_scales);
            TSX_LAUNCH_CHECK("copy_mxfp4_kernel");
        } else {
            rc = tsx::quantize_mxfp4_rows(g->m, g->k, steps * tsx::MX_STEP, g->x_dev, g->x_type, g->x_stride,
                                          tsx::MxRows{to, to_scales, p.x_pitch, p.scale_row, p.scale_step}, stream);
            if (rc) return rc;
        }
    } else if (codes) {
        p.x = static_cast<const uint8_t *>(g->x_dev);
        p.x_scales = g->x_scales_dev;
        p.x_pitch = g->m <= 1 ? 0 : g->x_stride;
        p.scale_row = g->m <= 1 ? 0 : g->x_scales_stride;
        p.scale_step = 4;
        if (plan.turns) {
            hipLaunchKernelGGL(tsx::turn_scales_kernel, dim3(unsigned(tsx::ceil_div(g->m, 256)), unsigned(tsx::ceil_div(steps, 4))), dim3(256), 0, stream,
                               g->x_scales_dev, p.scale_row, int64_t(g->m), steps, static_cast<unsigned *>(workspace_dev));
            TSX_LAUNCH_CHECK("turn_scales_kernel");
            p.x_scales = static_cast<const uint8_t *>(workspace_dev);
            p.scale_row = 4;
            p.scale_step = plan.word_bytes;
        }
    }
    p.w = static_cast<const int8_t *>(g->packed_w_dev);
    p.w_scales = p.w + tsx::packed_codes(g->k, g->n);
    p.bias = g->bias_dev;
    p.out = g->out_dev;
    p.out_stride = g->out_stride;
    p.m = g->m;
    p.n = g->n;
    p.frags = tsx::frags_of(g->n);
    p.ksteps = tsx::ksteps_of(g->k);
    p.act = g->act;
    p.slope = g->slope;
    return g->out_type == TSX_TYPE_F32 ? tsx::launch<TSX_TYPE_F32>(plan.kernel, g, p, stream) : g->out_type == TSX_TYPE_F16 ? tsx::launch<TSX_TYPE_F16>(plan.kernel, g, p, stream)
                                                                                                          : tsx::launch<TSX_TYPE_BF16>(plan.kernel, g, p, stream);
}

}  // extern "C"
