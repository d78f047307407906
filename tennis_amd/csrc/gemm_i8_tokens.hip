// int8 product with a scale for each token and each channel, on rows of fp32, fp16, bf16 or int8 values.
//
//     out[i][j] = act(float(sum_k q[i][k] w[k][j]) * w_scale[j] * x_scale[i] + bias[j]),  rounded once to the output's type
//
// Rows of floats become int8 first (tokens_i8.hip), in the workspace, padded with zeros to whole chunks of K.  int32 sums are
// exact, so every kernel here gives the same bits.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "igemm_i8.hpp"
#include "tokens_i8.hpp"

namespace tsx {
namespace {

constexpr int KSTEP = 64;              // K bytes of a packed K-step

struct TokenGemmParams {
    const int8_t *q;                   // [m][pitch], rows and their length multiples of 16 bytes
    const float *x_scales;
    const int8_t *wp;                  // as tsx_gemm_i8_pack_weights lays them out
    const float *w_scales, *bias;
    void *out;
    int64_t pitch, out_stride;
    int m, n, k, frags, ksteps;        // k: bytes of a row that are read, a multiple of 16
    int act;
    float slope;
    int row_tiles, col_tiles, tiles_per_xcd;
};

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(1))) void global_void;

// 64 lanes x 16 bytes, from an address for each lane to consecutive bytes of LDS.  Complete when vmcnt says so.
__device__ __forceinline__ void to_lds(const int8_t *at, int8_t *lds) {
    __builtin_amdgcn_global_load_lds((global_void *)at, (lds_void *)lds, 16, 0, 0);
}

// A fragment's values of 32 output columns x 32 tokens in the output's type: accumulator r of lane l is column 8 (r / 4) + 4 (l / 32) +
// r % 4 of token l % 32; swaps between the half-waves leave a lane with 16 consecutive columns, the lower ones with 0 .. 15, the upper
// ones with 16 .. 31.  xs: the token's scale.
struct OfColumns {                     // scales and biases of a lane's columns of a fragment
    v4f scale[4], bias[4];
    __device__ __forceinline__ void read(const float *scales, const float *biases) {      // the fragment's, in LDS
        const int half = 4 * ((threadIdx.x % 64) / 32);
        static_for<0, 4>([&](auto gc) {
            constexpr int g = decltype(gc)::value;
            scale[g] = *reinterpret_cast<const v4f *>(scales + 8 * g + half);
            bias[g] = *reinterpret_cast<const v4f *>(biases + 8 * g + half);
        });
    }
};
template <int OUT, int ACT>
__device__ __forceinline__ Run<OUT, 16> fragment_values(const TokenGemmParams &p, const v16i &acc, const OfColumns &of, float xs) {
    float v[16];
    static_for<0, 4>([&](auto gc) {
        constexpr int g = decltype(gc)::value;
        static_for<0, 4>([&](auto jc) { constexpr int j = decltype(jc)::value; v[4 * g + j] = __fadd_rn(__fmul_rn(__fmul_rn(float(acc[4 * g + j]), of.scale[g][j]), xs), of.bias[g][j]); });
    });
    activate_as<OUT, ACT>(v, p.slope);
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

// f(the activation as a constant): one branch around all of a wavefront's values
template <class F>
__device__ __forceinline__ void by_act(int act, F &&f) {
    switch (act) {
        case TSX_ACT_RELU: f(std::integral_constant<int, TSX_ACT_RELU>{}); break;
        case TSX_ACT_LEAKY_RELU: f(std::integral_constant<int, TSX_ACT_LEAKY_RELU>{}); break;
        case TSX_ACT_MISH_FAST: f(std::integral_constant<int, TSX_ACT_MISH_FAST>{}); break;
        case TSX_ACT_SILU: f(std::integral_constant<int, TSX_ACT_SILU>{}); break;
        default: f(std::integral_constant<int, TSX_ACT_NONE>{}); break;
    }
}

// LDS is this workgroup's own: what was read from it is read, and what the wavefronts wrote is there, behind the barrier.  Requests to
// memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
template <int N>
__device__ __forceinline__ void wait_for_all_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// WR x WC wavefronts, each with FR x FC fragments of 32 tokens x 32 columns; S chunks of KS K-steps in LDS.
//
// Bound: the matrix cores where K is long.  256 x 256, K in chunks of 64, four of them on their way: a chunk's 64 multiplications of a
// wavefront take 2048 cycles of its SIMD and 24 LDS reads.  On int8 tokens, 20 calls in a row, the means of ten such rows: 4096^3 59 .. 67 us,
// 8192^3 422 .. 432 (2.3 and 2.6 P operations/s; the library's plain int8 product 63 .. 69 and 422), where the card holds its power by a clock of
// 1.5 .. 1.7 GHz; in a trace, each behind rows that become int8, 65 and 498 (440 at the least).  Where K is short, its start and its outputs,
// which wait for no other tile's arithmetic on the same CU: 32768 x 960, K = 320 25 us, of which 12 are the two turns' epilogues.  Tiles
// of 128: three of them a CU in 168 registers, which fill each other's waits (two of them: 29 us for 25, 131072 x 512, K = 128 37 for 29).
// Requests to memory fill LDS past the registers, and a wavefront waits for all but the newest chunks' of them.
template <int WR, int WC, int FR, int FC, int KS, int S, int OUT>
__global__ __launch_bounds__(WR *WC * 64, WR * FR == 4 ? 3 : 1) void gemm_i8_tokens_kernel(TokenGemmParams p) {
    constexpr int CHUNK = KS * KSTEP, PIECES = CHUNK / 16, WAVES = WR * WC, ROWS = 32 * WR * FR, COLS = 32 * WC * FC, HALVES = 2 * KS;
    constexpr int A_BYTES = ROWS * CHUNK, B_BYTES = COLS * CHUNK, A_LOADS = A_BYTES / 1024 / WAVES, B_LOADS = B_BYTES / 1024 / WAVES;
    static_assert(A_LOADS * 1024 * WAVES == A_BYTES && B_LOADS * 1024 * WAVES == B_BYTES && (S - 1) * (A_LOADS + B_LOADS) < 64, "whole loads, counted in six bits");
    extern __shared__ __attribute__((aligned(16))) int8_t lds[];      // [S][A_BYTES + B_BYTES]
    // The tile's scales and biases, requested ahead of everything and here by the time the first chunk is: in the epilogue each request
    // would be waited for.
    __shared__ __attribute__((aligned(16))) float of_cols[2][COLS], of_rows[ROWS];
    constexpr int THREADS = WAVES * 64;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int wave_r = wave / WC, wave_c = wave % WC;
    // blockIdx % 8 is the XCD: each takes a run of consecutive tiles, which walk four row tiles before the next column tile
    const int tiles = p.row_tiles * p.col_tiles;
    const int t = int(blockIdx.x % 8) * p.tiles_per_xcd + int(blockIdx.x / 8);
    if (int(blockIdx.x / 8) >= p.tiles_per_xcd || t >= tiles) return;      // uniform, ahead of every barrier
    const int group = t / (4 * p.col_tiles), in_group = t - group * 4 * p.col_tiles;
    const int group_rows = min(4, p.row_tiles - 4 * group);
    const int tile_c = in_group / group_rows, tile_r = 4 * group + in_group - tile_c * group_rows;
    const int row0 = tile_r * ROWS, frag0 = tile_c * (COLS / 32);
    constexpr int COL_TURNS = (COLS + THREADS - 1) / THREADS, ROW_TURNS = (ROWS + THREADS - 1) / THREADS;
    float col_scale[COL_TURNS], col_bias[COL_TURNS], row_scale[ROW_TURNS];
    static_for<0, COL_TURNS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        col_scale[i] = p.w_scales[min(frag0 * 32 + int(threadIdx.x) + i * THREADS, p.n - 1)];
        col_bias[i] = -0.f;                                  // changes no sum
    });
    if (p.bias) static_for<0, COL_TURNS>([&](auto ic) { col_bias[decltype(ic)::value] = p.bias[min(frag0 * 32 + int(threadIdx.x) + decltype(ic)::value * THREADS, p.n - 1)]; });
    static_for<0, ROW_TURNS>([&](auto ic) { row_scale[decltype(ic)::value] = p.x_scales[min(row0 + int(threadIdx.x) + decltype(ic)::value * THREADS, p.m - 1)]; });

    // A row in LDS is its CHUNK bytes, its pieces of 16 XORed with bits of the row that make 16 rows cover all banks for one piece.  A
    // load instruction fills 1 KiB of such rows; rows beyond m are the last one again, never stored.  Pieces behind the end of a row are
    // its first one, against weights that are zero.  Scalar bases and 32-bit lane offsets.
    const auto key_of = [](int row) { return (row >> (KS == 1 ? 2 : 1)) & (PIECES - 1); };
    const int chunks = (p.ksteps + KS - 1) / KS;
    const int8_t *const a_base = p.q + int64_t(row0) * p.pitch;
    unsigned a_off[A_LOADS], b_off[B_LOADS];
    int a_piece[A_LOADS];
    static_for<0, A_LOADS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const int r = (wave * A_LOADS + i) * (64 / PIECES) + lane / PIECES;
        a_piece[i] = ((lane % PIECES) ^ key_of(r)) * 16;
        a_off[i] = unsigned(min(r, p.m - 1 - row0)) * unsigned(p.pitch);
    });
    // weights: packed[K-step][fragment][half][lane][16], in LDS [K-step of the chunk][fragment][half][lane][16]
    static_for<0, B_LOADS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const int unit = wave * B_LOADS + i, step = unit / (2 * COLS / 32), in_step = unit % (2 * COLS / 32);
        const int frag = min(frag0 + in_step / 2, p.frags - 1);
        b_off[i] = unsigned(step * p.frags + frag) * 2048u + (in_step % 2) * 1024 + lane * 16;
    });
    const int64_t b_step = int64_t(p.frags) * (KS * 2048);
    auto fetch = [&](int chunk, int buf) __attribute__((always_inline)) {
        const int c = min(chunk, chunks - 1);                // behind the last chunk: that one again, not read from LDS
        int8_t *const at = lds + buf * (A_BYTES + B_BYTES);
        const int8_t *const b = p.wp + c * b_step;
        static_for<0, A_LOADS>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            const int k = c * CHUNK + a_piece[i];
            to_lds(a_base + (a_off[i] + unsigned(k < p.k ? k : 0)), at + (wave * A_LOADS + i) * 1024);
        });
        static_for<0, B_LOADS>([&](auto ic) { constexpr int i = decltype(ic)::value; to_lds(b + b_off[i], at + A_BYTES + (wave * B_LOADS + i) * 1024); });
    };

    v16i acc[FR][FC];
    static_for<0, FR * FC>([&](auto fc) {
        constexpr int f = decltype(fc)::value;
        static_for<0, 16>([&](auto rc) { acc[f / FC][f % FC][decltype(rc)::value] = 0; });
    });
    const int a_row = (wave_r * FR * 32 + lane % 32) * CHUNK, a_key = key_of(lane % 32);
    v4i a[2][FR], b[2][FC];
    auto read = [&](auto hc, int buf) __attribute__((always_inline)) {
        constexpr int h = decltype(hc)::value, set = h % 2;
        const int8_t *const at = lds + buf * (A_BYTES + B_BYTES);
        static_for<0, FC>([&](auto fc) {
            constexpr int f = decltype(fc)::value;
            b[set][f] = *reinterpret_cast<const v4i *>(at + A_BYTES + (((h / 2) * (COLS / 32) + wave_c * FC + f) * 2 + h % 2) * 1024 + lane * 16);
        });
        static_for<0, FR>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            a[set][i] = *reinterpret_cast<const v4i *>(at + a_row + i * 32 * CHUNK + ((2 * h + lane / 32) ^ a_key) * 16);
        });
    };
    static_for<0, S>([&](auto sc) { fetch(decltype(sc)::value, decltype(sc)::value); });     // behind the last chunk: that one again
    wait_for_all_but<(S - 1) * (A_LOADS + B_LOADS)>();
    static_for<0, COL_TURNS>([&](auto ic) {
        constexpr int i = decltype(ic)::value;
        const int at = threadIdx.x + i * THREADS;
        if (COLS % THREADS == 0 || at < COLS) of_cols[0][at] = col_scale[i], of_cols[1][at] = col_bias[i];
    });
    static_for<0, ROW_TURNS>([&](auto ic) {
        const int at = threadIdx.x + decltype(ic)::value * THREADS;
        if (ROWS % THREADS == 0 || at < ROWS) of_rows[at] = row_scale[decltype(ic)::value];
    });
    lds_barrier();
    read(std::integral_constant<int, 0>{}, 0);
    int buf = 0, c = 0;
    auto multiply = [&](auto fetching) __attribute__((always_inline)) {
        constexpr bool FETCHES = decltype(fetching)::value;
        const int after = buf + 1 == S ? 0 : buf + 1;
        static_for<0, HALVES>([&](auto hc) {
            constexpr int h = decltype(hc)::value;
            if constexpr (h + 1 < HALVES) {
                read(std::integral_constant<int, h + 1>{}, buf);
            } else {
                // Every wavefront has its operands of this chunk in registers: its buffer is free behind the barrier, and the next
                // chunk is there for all.  The rest of this chunk's arithmetic covers the first reads behind it.
                wait_for_all_but<FETCHES ? (S - 2) * (A_LOADS + B_LOADS) : 0>();
                lds_barrier();
                read(std::integral_constant<int, 0>{}, after);
                if constexpr (FETCHES) fetch(c + S, buf);
            }
            static_for<0, FR * FC>([&](auto fc) {
                constexpr int i = decltype(fc)::value / FC, f = decltype(fc)::value % FC;
                acc[i][f] = __builtin_amdgcn_mfma_i32_32x32x32_i8(b[h % 2][f], a[h % 2][i], acc[i][f], 0, 0, 0);
            });
            // reads and requests between the multiplications
            static_for<0, FR * FC>([&](auto fc) {
                if constexpr (FETCHES && h + 1 == HALVES) __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        buf = after;
    };
    for (; c + S < chunks; ++c) multiply(std::true_type{});
    for (; c < chunks; ++c) multiply(std::false_type{});      // the last S chunks are all on their way
    // The chunks' LDS is free: nothing is on its way into it, and behind this barrier nobody reads it.  A wavefront's 32 tokens x 32 FC
    // columns go through it, so that a store instruction writes whole cache lines (straight from the registers it would write 16 bytes of
    // each of 64 runs).
    wait_for_all_but<0>();
    lds_barrier();
    by_act(p.act, [&](auto act) __attribute__((always_inline)) {
        constexpr int SIZE = OUT == TSX_TYPE_F32 ? 4 : 2, ROW = FC * 32 * SIZE, PITCH = ROW + 16, IN_ROW = ROW / 16, AT_ONCE = 64 / IN_ROW, EACH = 16 / SIZE;
        static_assert(WAVES * 32 * PITCH <= S * (A_BYTES + B_BYTES), "room for all wavefronts");
        int8_t *const mine = lds + wave * (32 * PITCH);
        const int col = (frag0 + wave_c * FC) * 32 + lane % IN_ROW * EACH, left = p.n - col;      // where a lane stores
        // Read once where the registers hold them: each time they are as many LDS cycles as the values take.
        constexpr bool ONCE = FR > 2 || OUT == TSX_TYPE_BF16;
        OfColumns of[ONCE ? FC : 1];
        auto read_columns = [&](auto fc) {
            constexpr int f = decltype(fc)::value;
            of[ONCE ? f : 0].read(of_cols[0] + (wave_c * FC + f) * 32, of_cols[1] + (wave_c * FC + f) * 32);
        };
        if constexpr (ONCE) static_for<0, FC>(read_columns);
        static_for<0, FR>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            const int in_tile = (wave_r * FR + i) * 32;
            const float xs = of_rows[in_tile + lane % 32];
            static_for<0, FC>([&](auto fc) {
                constexpr int f = decltype(fc)::value;
                if constexpr (!ONCE) read_columns(fc);
                const Run<OUT, 16> v = fragment_values<OUT, decltype(act)::value>(p, acc[i][f], of[ONCE ? f : 0], xs);
                v4u *const to = reinterpret_cast<v4u *>(mine + lane % 32 * PITCH + (f * 32 + 16 * (lane / 32)) * SIZE);
                static_for<0, SIZE>([&](auto wc) { constexpr int w = 4 * decltype(wc)::value; to[w / 4] = v4u{v.word[w], v.word[w + 1], v.word[w + 2], v.word[w + 3]}; });
            });
            static_for<0, 32 / AT_ONCE>([&](auto kc) {
                const int r = decltype(kc)::value * AT_ONCE + lane / IN_ROW, row = row0 + in_tile + r;
                Run<OUT, EACH> v;
                const v4u got = *reinterpret_cast<const v4u *>(mine + r * PITCH + lane % IN_ROW * 16);
                static_for<0, 4>([&](auto wc) { v.word[decltype(wc)::value] = got[decltype(wc)::value]; });
                char *const out = static_cast<char *>(p.out) + (int64_t(row) * p.out_stride + col) * SIZE;
                if (row < p.m) {
                    if (left >= EACH) v.store(out);
                    else if (left > 0) v.store_some(out, left);
                }
            });
            __builtin_amdgcn_sched_barrier(0);               // 32 tokens at a time: their values would fill the registers
        });
    });
}

// ---- few tokens: a stream over the weights
//
// There the product reads n k bytes of weights and does little with each.  A workgroup owns 16 NC output columns (4096 columns: one
// workgroup a CU) and its 8 wavefronts split K, every eighth K-step each; a K-step of 16 columns is one 16-byte load a lane, AHEAD of them
// in flight from the first instruction on (4096 columns, K = 4096, one row of bf16: 5.1 .. 6.8 us in the kernel, 16.8 MB, of which 2 are the
// launch and 1 the first load's way; a call 6.3, which took 24 on tiles).  X, the type of the rows: TSX_TYPE_I8, or floats that the workgroup
// quantizes itself while its weights are on their way (all of them do, out of the L2: one launch and its start less).  MT: groups of 16
// tokens.  v_mfma_i32_16x16x64_i8: lane l supplies row (token or column) l % 16, K bytes 16 (l / 16) ..; accumulator r of lane l is
// column 4 (l / 16) + r of token l % 16.  The eight partial sums meet in LDS.
constexpr int FEW_THREADS = 512, FEW_WAVES = FEW_THREADS / 64;

struct FewTokens : TokenGemmParams {
    const void *x;
    int64_t x_stride;
    int lg_threads;                    // of a row that the workgroup quantizes
    int cols;                          // values of a row; k: of its int8 row, as the K-steps are
};

template <int X, int MT, int NC, int AHEAD, int OUT>
__global__ __launch_bounds__(FEW_THREADS) void gemm_i8_few_tokens_kernel(FewTokens p) {
    extern __shared__ __attribute__((aligned(16))) int8_t lds[];      // [8][MT][NC][4][64] partial sums, then the rows
    __shared__ float scales[16 * MT];
    __shared__ unsigned tops[FEW_WAVES];
    int *const sums = reinterpret_cast<int *>(lds);
    int8_t *const rows = lds + FEW_WAVES * MT * NC * 1024;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), piece = lane / 16, row = lane % 16;
    const int row0 = X == TSX_TYPE_I8 ? int(blockIdx.y) * 16 * MT : 0;
    const int col16 = blockIdx.x * NC;                       // in columns of 16
    const int8_t *w[NC];
    static_for<0, NC>([&](auto nc) {
        const int c = col16 + decltype(nc)::value;
        w[decltype(nc)::value] = p.wp + int64_t(c >> 1) * 2048 + (piece >> 1) * 1024 + (16 * (c & 1) + row + 32 * (piece & 1)) * 16;
    });
    const int64_t w_step = int64_t(p.frags) * 2048;
    v4i a[AHEAD][NC];
    auto fetch = [&](int first) __attribute__((always_inline)) {
        static_for<0, AHEAD>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            static_for<0, NC>([&](auto nc) { a[u][decltype(nc)::value] = *reinterpret_cast<const v4i *>(w[decltype(nc)::value] + min(first + FEW_WAVES * u, p.ksteps - 1) * w_step); });
        });
    };
    fetch(wave);
    const int pitch = p.ksteps * KSTEP + 16;                 // of a row in LDS: the 16 put the rows' pieces into different banks
    if constexpr (X != TSX_TYPE_I8) {
        constexpr int PIECE = 8, SIZE = X == TSX_TYPE_F32 ? 4 : 2, HELD = 4;
        typedef Run<X, PIECE> Values;
        const int lg = p.lg_threads, T = 1 << lg, whole = p.cols / PIECE, pieces = (p.cols + PIECE - 1) / PIECE;
        const int t = threadIdx.x & (T - 1), side = FEW_THREADS >> lg, turns = (pieces + HELD * T - 1) / (HELD * T);
        for (int r0 = 0; r0 < p.m; r0 += side) {
            const int r = r0 + (threadIdx.x >> lg);
            const char *const x = static_cast<const char *>(p.x) + min(r, p.m - 1) * p.x_stride * SIZE;
            Values v[HELD];
            auto load = [&](int first) __attribute__((always_inline)) {
                if (whole)           // uniform
                    static_for<0, HELD>([&](auto ic) { v[decltype(ic)::value].load(x + int64_t(min(first + t + decltype(ic)::value * T, whole - 1)) * (PIECE * SIZE)); });
                Values last;
                last.clear();
                if (whole != pieces) last.load_some(x + int64_t(whole) * (PIECE * SIZE), p.cols - whole * PIECE);       // uniform
                static_for<0, HELD>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    const int at = first + t + i * T;
                    if (at >= whole) v[i].clear();
                    if (at == whole) v[i] = last;
                });
            };
            unsigned top = 0;
            for (int turn = 0; turn < turns; ++turn) {
                load(turn * HELD * T);
                static_for<0, HELD>([&](auto ic) { top = v[decltype(ic)::value].top(top); });
            }
            top = over_lanes(top, lg, [](unsigned one, unsigned other) { return Values::template larger<X>(one, other); });
            if (lg > 6) {            // uniform: wavefronts share a row, all rows are this turn's
                if (lane == 0) tops[wave] = top;
                __syncthreads();
                for (int i = 0; i < T / 64; ++i) top = Values::template larger<X>(top, tops[(wave & ~(T / 64 - 1)) + i]);
            }
            const TokenScale s(top_value<X>(top));
            if (t == 0 && r < p.m) scales[r] = s.scale;
            for (int turn = 0; turn < turns; ++turn) {
                if (turns > 1) load(turn * HELD * T);
                static_for<0, HELD>([&](auto ic) {
                    constexpr int i = decltype(ic)::value;
                    const int at = turn * HELD * T + t + i * T;
                    if (at >= pieces || r >= p.m) return;
                    unsigned b[PIECE];
                    static_for<0, PIECE>([&](auto ec) { constexpr int e = decltype(ec)::value; b[e] = s.bits(__fmul_rn(v[i].template get<e>(), s.lift)); });
                    v2u out = {low_bytes(b[0], b[1], b[2], b[3]), low_bytes(b[4], b[5], b[6], b[7])};
                    if (s.reciprocal == 0.f) out = v2u{0, 0};
                    *reinterpret_cast<v2u *>(rows + r * pitch + at * PIECE) = out;       // behind the row's end: against weights that are zero
                });
            }
        }
        __syncthreads();
    } else {
        if (threadIdx.x < 16 * MT) scales[threadIdx.x] = p.x_scales[min(row0 + int(threadIdx.x), p.m - 1)];
    }
    v4i acc[MT][NC];
    static_for<0, MT * NC>([&](auto mc) { acc[decltype(mc)::value / NC][decltype(mc)::value % NC] = v4i{0, 0, 0, 0}; });
    for (int first = wave; first < p.ksteps; first += FEW_WAVES * AHEAD) {
        v4i b[AHEAD][MT];
        static_for<0, AHEAD>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            const int k = min(first + FEW_WAVES * u, p.ksteps - 1) * KSTEP + piece * 16;
            static_for<0, MT>([&](auto mc) {
                constexpr int i = decltype(mc)::value;
                const int token = min(row0 + 16 * i + row, p.m - 1);
                if constexpr (X == TSX_TYPE_I8) b[u][i] = *reinterpret_cast<const v4i *>(p.q + token * p.pitch + (k < p.k ? k : 0));
                else b[u][i] = *reinterpret_cast<const v4i *>(rows + token * pitch + k);
            });
        });
        static_for<0, AHEAD>([&](auto uc) {
            constexpr int u = decltype(uc)::value;
            if (first + FEW_WAVES * u < p.ksteps)            // uniform
                static_for<0, MT * NC>([&](auto mc) {
                    constexpr int i = decltype(mc)::value / NC, c = decltype(mc)::value % NC;
                    acc[i][c] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][c], b[u][i], acc[i][c], 0, 0, 0);
                });
        });
        if (first + FEW_WAVES * AHEAD < p.ksteps) fetch(first + FEW_WAVES * AHEAD);
    }
    static_for<0, MT * NC>([&](auto mc) {
        constexpr int i = decltype(mc)::value / NC, c = decltype(mc)::value % NC;
        static_for<0, 4>([&](auto rc) { sums[((wave * MT * NC + i * NC + c) * 4 + decltype(rc)::value) * 64 + lane] = acc[i][c][decltype(rc)::value]; });
    });
    __syncthreads();
    for (int at = threadIdx.x; at < 256 * MT * NC; at += FEW_THREADS) {
        const int in = at % (16 * NC), col = col16 * 16 + in, token = at / (16 * NC);
        if (col >= p.n || row0 + token >= p.m) continue;
        int sum = 0;
#pragma unroll
        for (int i = 0; i < FEW_WAVES; ++i) sum += sums[((i * MT * NC + token / 16 * NC + in / 16) * 4 + in % 4) * 64 + token % 16 + 16 * (in % 16 / 4)];
        float v[1] = {__fmul_rn(__fmul_rn(float(sum), p.w_scales[col]), scales[token])};
        if (p.bias) v[0] = __fadd_rn(v[0], p.bias[col]);
        activate_tokens<OUT>(v, p.act, p.slope);
        Run<OUT, 1> out;
        out.set(v);
        out.store(static_cast<char *>(p.out) + ((row0 + token) * p.out_stride + col) * (OUT == TSX_TYPE_F32 ? 4 : 2));
    }
}

template <int WR, int WC, int FR, int FC, int KS, int S, int OUT>
int launch_tile(TokenGemmParams p, hipStream_t stream) {
    p.row_tiles = int(ceil_div(p.m, 32 * WR * FR));
    p.col_tiles = int(ceil_div(p.n, 32 * WC * FC));
    const int64_t per_xcd = ceil_div(int64_t(p.row_tiles) * p.col_tiles, 8);
    TSX_REQUIRE(8 * per_xcd * WR * WC * 64 < int64_t(1) << 32, "gemm_i8_tokens: %d x %d outputs are more than a launch holds", p.m, p.n);
    p.tiles_per_xcd = int(per_xcd);
    constexpr int LDS = S * 32 * (WR * FR + WC * FC) * KS * KSTEP;
    const auto kernel = gemm_i8_tokens_kernel<WR, WC, FR, FC, KS, S, OUT>;
    if (LDS > 64 * 1024) {
        const int rc = grant_lds(reinterpret_cast<const void *>(kernel), LDS);
        if (rc) return rc;
    }
    hipLaunchKernelGGL(kernel, dim3(unsigned(8 * p.tiles_per_xcd)), dim3(WR * WC * 64), LDS, stream, p);
    TSX_LAUNCH_CHECK("gemm_i8_tokens_kernel");
    return 0;
}

// rows of LDS that the tokens of a call take where the product quantizes them
constexpr int FEW_LDS = 152 * 1024;
int64_t few_lds(int m, int k) { return int64_t(m) * (round_up(k, KSTEP) + 16); }

template <int X, int MT, int NC, int AHEAD, int OUT>
int launch_few_tokens(const FewTokens &p, hipStream_t stream) {
    const int lds = FEW_WAVES * MT * NC * 1024 + (X == TSX_TYPE_I8 ? 0 : int(few_lds(p.m, p.cols)));
    const auto kernel = gemm_i8_few_tokens_kernel<X, MT, NC, AHEAD, OUT>;
    if (lds > 64 * 1024) {
        const int rc = grant_lds(reinterpret_cast<const void *>(kernel), FEW_LDS);
        if (rc) return rc;
    }
    const dim3 grid(unsigned(ceil_div(p.n, 16 * NC)), X == TSX_TYPE_I8 ? unsigned(ceil_div(p.m, 16 * MT)) : 1);
    hipLaunchKernelGGL(kernel, grid, dim3(FEW_THREADS), lds, stream, p);
    TSX_LAUNCH_CHECK("gemm_i8_few_tokens_kernel");
    return 0;
}

template <int X, int OUT>
int few_tokens_of(const FewTokens &p, hipStream_t stream) {
    const bool deep = p.ksteps > 4 * FEW_WAVES;
    if (p.m <= 16) return deep ? launch_few_tokens<X, 1, 1, 8, OUT>(p, stream) : launch_few_tokens<X, 1, 1, 4, OUT>(p, stream);
    return deep ? launch_few_tokens<X, 2, 1, 8, OUT>(p, stream) : launch_few_tokens<X, 2, 1, 4, OUT>(p, stream);
}

template <int OUT>
int few_tokens(const tsx_token_gemm *g, const TokenGemmParams &q, bool quantizes, bool wide, hipStream_t stream) {
    FewTokens p{};
    static_cast<TokenGemmParams &>(p) = q;
    p.x = g->x_dev;
    p.x_stride = g->x_stride;
    p.cols = g->k;
    p.lg_threads = g->m <= 1 ? 9 : g->m <= 2 ? 8 : g->m <= 4 ? 7 : 6;
    if (quantizes)
        return g->x_type == TSX_TYPE_F32 ? few_tokens_of<TSX_TYPE_F32, OUT>(p, stream)
               : g->x_type == TSX_TYPE_F16 ? few_tokens_of<TSX_TYPE_F16, OUT>(p, stream) : few_tokens_of<TSX_TYPE_BF16, OUT>(p, stream);
    return wide ? launch_few_tokens<TSX_TYPE_I8, 2, 2, 4, OUT>(p, stream) : few_tokens_of<TSX_TYPE_I8, OUT>(p, stream);
}

// The kernel a call takes, by an estimate of its time in us, fitted to products of 16 .. 32768 rows on K of 128 .. 8192 (bf16 output):
// what a launch takes whatever its size, and for each 256 workgroups, one a CU, a fixed part and one for each 1024 of K (tiles of 256: a
// CU's only workgroup, in whole turns).  Measured, few tokens 16 x 32 and 32 x 32, tiles of 64, 128 and 256 (us): 32 x 1000, K = 2048: 4.4,
// 5.9, 7.3, 11.2, 22.6; 64 x 4096, K = 4096: 12.6, 9.9, 12.1, 19.6, 40; 197 x 777, K = 1500: 5.0, 5.3, 6.8, 11, 25; 512 x 3840, K = 1280:
// 33, 26, 7.2, 9.1, 17.7; tiles alone: 2048^3 17.3, 13.8, 24.7; 8192 x 1280, K = 640 18.1, 14.5, 15.5; 32768 x 960, K = 320 41, 24.7, 25.4;
// 131072 x 512, K = 128 58, 29.4, 33.7; 4096^3 107, 77, 62.
enum class TokenKernel { few_16, few_32, tile_64, tile_128, tile_256 };

constexpr int FEW_MOST = 1 << 14;      // rows of the kernels for few tokens: with more their groups of rows leave a launch's second axis

TokenKernel choose(int m, int n, int k) {
    if (m <= 16) return TokenKernel::few_16;
    const float ks = float(k) / 1024.f;
    const auto rounds = [&](int rows, int cols) { return float(ceil_div(m, rows) * ceil_div(n, cols)) / 256.f; };
    const float few = rounds(32, 16), few_wide = rounds(32, 32), r64 = rounds(64, 64), r128 = rounds(128, 128), r256 = rounds(256, 256);
    const float cost[] = {few <= 1.f ? 3.6f + ks * (k <= 2048 ? 0.5f : 1.25f * std::max(few, 0.5f)) : 3.6f + few * (0.25f + 1.1f * ks),
                          4.2f + std::max(few_wide, 1.f) * (0.2f + 1.35f * ks), 3.f + std::max(r64, 1.f) * (0.5f + 1.75f * ks),
                          4.6f + std::max(r128, 1.f) * (1.3f + 4.2f * ks), 3.f + std::ceil(r256) * (7.4f + 13.f * ks * (0.75f + 0.25f * std::min(r256, 1.f)))};
    int best = m <= FEW_MOST ? 0 : 2;
    for (int i = best + 1; i < 5; ++i)
        if (cost[i] < cost[best]) best = i;
    return TokenKernel(best);
}

template <int OUT>
int launch(const tsx_token_gemm *g, const TokenGemmParams &p, bool quantizes, hipStream_t stream) {
    if (quantizes) return few_tokens<OUT>(g, p, true, false, stream);
    // TSX_TOKENS_KERNEL: that kernel, by its place in the list above, for any call it can take (tests, measurements)
    const char *e = std::getenv("TSX_TOKENS_KERNEL");
    const bool named = e && e[0] >= (p.m <= FEW_MOST ? '0' : '2') && e[0] <= '4';
    switch (named ? TokenKernel(e[0] - '0') : choose(p.m, p.n, p.k)) {
        case TokenKernel::few_16: return few_tokens<OUT>(g, p, false, false, stream);
        case TokenKernel::few_32: return few_tokens<OUT>(g, p, false, true, stream);
        case TokenKernel::tile_64: return launch_tile<2, 2, 1, 1, 2, 3, OUT>(p, stream);
        case TokenKernel::tile_128: return launch_tile<2, 2, 2, 2, 1, 3, OUT>(p, stream);
        default: return launch_tile<2, 4, 4, 2, 1, 4, OUT>(p, stream);
    }
}

// rows of int8 tokens of another length, stride or alignment than the kernels read, copied to whole pieces of 16
__global__ __launch_bounds__(256) void copy_tokens_kernel(const int8_t *x, int64_t x_stride, int k, int8_t *q, int pitch, int64_t rows) {
    const int pieces = pitch / 16;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < rows * pieces; i += int64_t(gridDim.x) * 256) {
        const int64_t row = i / pieces;
        const int at = int(i - row * pieces) * 16;
        v4i v = {0, 0, 0, 0};
        const int8_t *const from = x + row * x_stride + at;
        if (at + 16 <= k) v = __builtin_bit_cast(v4i, v4u(*reinterpret_cast<const v4u_any *>(from)));
        else
            for (int b = 0; b < 16 && at + b < k; ++b) v[b / 4] |= int((unsigned(from[b]) & 255u) << (8 * (b % 4)));
        *reinterpret_cast<v4i *>(q + row * pitch + at) = v;
    }
}

int check(const tsx_token_gemm *g) {
    TSX_REQUIRE(g, "gemm_i8_tokens: null argument");
    TSX_REQUIRE(g->m >= 0 && g->n > 0 && g->k > 0, "gemm_i8_tokens: bad extents");
    TSX_REQUIRE(g->k < 1 << 17, "gemm_i8_tokens: K = %d (below 2^17: longer sums leave 32 bits)", g->k);
    TSX_REQUIRE(g->m < 1 << 28 && g->n < 1 << 24, "gemm_i8_tokens: %d rows and %d columns (below 2^28 and 2^24)", g->m, g->n);
    TSX_REQUIRE(is_float_type(g->x_type) || g->x_type == TSX_TYPE_I8, "gemm_i8_tokens: element type %d", g->x_type);
    TSX_REQUIRE(is_float_type(g->out_type), "gemm_i8_tokens: output type %d (fp32, fp16 or bf16)", g->out_type);
    TSX_REQUIRE(is_token_act(g->act), "gemm_i8_tokens: activation %d", g->act);
    TSX_REQUIRE(g->m <= 1 || (g->x_stride >= g->k && g->out_stride >= g->n), "gemm_i8_tokens: rows of %d and %d columns overlap at strides %lld and %lld",
                g->k, g->n, (long long)g->x_stride, (long long)g->out_stride);
    return 0;
}

int padded(int k) { return int(round_up(k, 16)); }

// Whether the product's workgroups quantize the rows themselves, each all of them: the launch that this saves is 2 us, and up to some
// 40 K values its work hides behind the weights (us with and without, 4096 columns, K = 4096: 1 row 6.0 and 7.9, 8 rows 7.4 and 8.9, 16
// rows 9.9 and 9.7; 1000 columns, K = 2048, 16 rows: 5.5 and 7.2).
bool quantizes_itself(const tsx_token_gemm *g) {
    return g->x_type != TSX_TYPE_I8 && g->m <= 32 && int64_t(g->m) * g->k <= 40960 && few_lds(g->m, g->k) + FEW_WAVES * 2048 <= FEW_LDS;
}

// A tile's rows are reached by 32-bit offsets: 256 of them at 2^23.
bool reads_in_place(const tsx_token_gemm *g) {
    return g->x_type == TSX_TYPE_I8 && g->k % 16 == 0 && (g->m <= 1 || (g->x_stride % 16 == 0 && g->x_stride <= 1 << 23)) && reinterpret_cast<uintptr_t>(g->x_dev) % 16 == 0;
}

size_t scales_offset(const tsx_token_gemm *g) { return size_t(g->m) * padded(g->k); }

size_t workspace_bytes(const tsx_token_gemm *g) {
    if (g->m == 0 || reads_in_place(g) || quantizes_itself(g)) return 0;
    return scales_offset(g) + (g->x_type == TSX_TYPE_I8 ? 0 : size_t(g->m) * 4);
}

}  // namespace
}  // namespace tsx

extern "C" {

size_t tsx_gemm_i8_tokens_workspace_bytes(const tsx_token_gemm *g) {
    if (tsx::check(g)) return 0;
    return tsx::workspace_bytes(g);
}

int tsx_gemm_i8_tokens(const tsx_token_gemm *g, void *workspace_dev, size_t workspace_bytes, void *stream_) {
    int rc = tsx::check(g);
    if (rc || g->m == 0) return rc;
    TSX_REQUIRE(g->x_dev && g->packed_w_dev && g->w_scales_dev && g->out_dev, "gemm_i8_tokens: null pointer");
    TSX_REQUIRE(g->x_type != TSX_TYPE_I8 || g->x_scales_dev, "gemm_i8_tokens: int8 rows need their scales");
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(g->packed_w_dev) % 16 == 0, "gemm_i8_tokens: packed weights must be 16-byte aligned");
    TSX_REQUIRE(reinterpret_cast<uintptr_t>(g->x_dev) % tsx::element_bytes(g->x_type) == 0 &&
                    reinterpret_cast<uintptr_t>(g->out_dev) % tsx::element_bytes(g->out_type) == 0, "gemm_i8_tokens: pointer is no multiple of its elements");
    const size_t need = tsx::workspace_bytes(g);
    if (need) {
        if (!workspace_dev || workspace_bytes < need)
            return tsx::fail(TSX_E_WORKSPACE, "gemm_i8_tokens: workspace %zu < %zu bytes", workspace_dev ? workspace_bytes : size_t(0), need);
        TSX_REQUIRE(reinterpret_cast<uintptr_t>(workspace_dev) % 16 == 0, "gemm_i8_tokens: workspace must be 16-byte aligned");
    }
    hipStream_t stream = tsx::as_stream(stream_);
    tsx::TokenGemmParams p{};
    const int kp = tsx::padded(g->k);
    p.q = static_cast<const int8_t *>(need ? workspace_dev : g->x_dev);
    p.pitch = need ? kp : g->m <= 1 ? 0 : g->x_stride;
    p.x_scales = g->x_scales_dev;
    const bool quantizes = tsx::quantizes_itself(g);
    if (quantizes) {
        // nothing ahead of the product
    } else if (g->x_type != TSX_TYPE_I8) {
        float *const scales = reinterpret_cast<float *>(static_cast<char *>(workspace_dev) + tsx::scales_offset(g));
        rc = tsx::quantize_rows(g->m, g->k, kp, g->x_dev, g->x_type, g->x_stride, static_cast<int8_t *>(workspace_dev), kp, scales, stream);
        if (rc) return rc;
        p.x_scales = scales;
    } else if (need) {
        const int64_t pieces = int64_t(g->m) * (kp / 16), blocks = tsx::ceil_div(pieces, 256);
        hipLaunchKernelGGL(tsx::copy_tokens_kernel, dim3(unsigned(std::min<int64_t>(blocks, 1 << 16))), dim3(256), 0, stream,
                           static_cast<const int8_t *>(g->x_dev), g->x_stride, g->k, static_cast<int8_t *>(workspace_dev), kp, int64_t(g->m));
        TSX_LAUNCH_CHECK("copy_tokens_kernel");
    }
    p.wp = static_cast<const int8_t *>(g->packed_w_dev);
    p.w_scales = g->w_scales_dev;
    p.bias = g->bias_dev;
    p.out = g->out_dev;
    p.out_stride = g->out_stride;
    p.m = g->m;
    p.n = g->n;
    p.frags = int(tsx::round_up(g->n, 128) / 32);
    p.k = kp;
    p.ksteps = int(tsx::ceil_div(kp, tsx::KSTEP));
    p.act = g->act;
    p.slope = g->slope;
    return g->out_type == TSX_TYPE_F32 ? tsx::launch<TSX_TYPE_F32>(g, p, quantizes, stream) : g->out_type == TSX_TYPE_F16 ? tsx::launch<TSX_TYPE_F16>(g, p, quantizes, stream)
                                                                                                          : tsx::launch<TSX_TYPE_BF16>(g, p, quantizes, stream);
}

}  // extern "C"
