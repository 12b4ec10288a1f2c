// The gated linear layer: out = act(x Wg + bg) * (x Wu + bu), and its gradient.  x [M, K], [Wg | Wu] the columns of W [K, 2 N].
//
//   gate = x Wg + bg, up = x Wu + bu;   dgate = dout up act'(gate), dup = dout act(gate);
//   dx = dgate Wg^T + dup Wu^T,   dW = x^T [dgate | dup],   db = column sums of [dgate | dup].
// gate and up are worked out again for the gradient: that is a third of its products, and keeping them would be 8 N bytes per row written and
// read, more time than the products take.
//
// Products run on the bf16 matrix cores with fp32 sums.  bf16 values are operands as they are.  An fp32 value is three bf16 pieces
// (mlp_split.hpp) and a product of two the six largest of nine, 2^-24 of it off.  In bf16 [dgate | dup], which is never rounded to
// bf16, goes into dx as two (16 bits: 2^-17 of a term, where storing dx costs 2^-8 of it) and into dW, which is fp32, as three.
//
// Operands lie in the workspace as fragments: 16 rows and 32 of the contracted index, a KiB in the order in which the 64 lanes of
// v_mfma_f32_16x16x32_bf16 hold them (lane 16 g + n: row n, elements 8 g .. 8 g + 7), the pieces of a fragment next to each other, all rows'
// fragments of 32 of the contracted index one behind the other, zeros past the ends.  Whoever makes an operand writes it so; reading is whole and in
// order, from memory to LDS past the registers and from there without conflicts.  The 2 N columns of gate and up alternate by 16.
#include "mlp_split.hpp"
#include "mrl_host.hpp"
#include "gate.hpp"

namespace mrl {
namespace glu {
namespace {

struct bf16_t { unsigned short bits; };
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4w __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));

constexpr int KIB = 512;   // elements of a fragment's piece

MRL_DEV float value_of(float x) { return x; }
MRL_DEV float value_of(bf16_t x) { return __uint_as_float((unsigned)x.bits << 16); }
MRL_DEV void give(float *p, float x) { *p = x; }
MRL_DEV void give(bf16_t *p, float x) { p->bits = __builtin_bit_cast(unsigned short, (__bf16)x); }

// eight neighbouring values, zeros from `n` on
MRL_DEV f32x8 load8(const float *p, int n) {
    f32x8 x = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (n >= 8) {
        const f32x4u a = *reinterpret_cast<const f32x4u *>(p), b = *reinterpret_cast<const f32x4u *>(p + 4);
        x = f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < n) x[i] = p[i];
    }
    return x;
}
MRL_DEV f32x8 load8(const bf16_t *p, int n) {
    f32x8 x = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
    if (n >= 8) {
        const u16x8u v = *reinterpret_cast<const u16x8u *>(p);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float((unsigned)v[i] << 16);
    } else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < n) x[i] = value_of(p[i]);
    }
    return x;
}

// the first P pieces of eight values
template <int P>
MRL_DEV void put_pieces(const f32x8 x, __bf16 *fragment, int lane) {
    if constexpr (P == 3) {
        bf16x8 p[SPLIT];
        split8(x, p);
#pragma unroll
        for (int i = 0; i < P; ++i) *reinterpret_cast<bf16x8 *>(fragment + i * KIB + lane * 8) = p[i];
    } else {
        *reinterpret_cast<bf16x8 *>(fragment + lane * 8) = __builtin_convertvector(x, bf16x8);
    }
}

// ---------------------------------------------------------------- operands from rows
// A matrix [rows, columns] of E, `ld` apart, whose columns may be gate and up side by side.
struct Source {
    const void *at;
    long ld;
    int rows, columns;   // columns: of gate and up each where they alternate
};
// Fragments of its rows, contracted along its columns; PAIRED: gate and up alternate by 16 columns.  A wavefront a fragment, number `at` of
// row_fragments * blocks.
template <class E, int P, bool PAIRED>
MRL_DEV void along_rows(const Source &s, __bf16 *to, int row_fragments, int blocks, long at) {
    const long fragment = at * 4 + (threadIdx.x >> 6);
    if (fragment >= (long)row_fragments * blocks) return;
    const int lane = threadIdx.x & 63, block = (int)(fragment / row_fragments), row = (int)(fragment - (long)block * row_fragments) * 16 + (lane & 15), g = lane >> 4;
    const int column = PAIRED ? block * 16 + (g & 1) * 8 : block * 32 + g * 8;
    const E *p = (const E *)s.at + row * s.ld + column + (PAIRED && g >= 2 ? s.columns : 0);
    put_pieces<P>(load8(p, row < s.rows ? s.columns - column : 0), to + fragment * P * KIB, lane);
}
// Fragments of its columns, contracted along its rows.  A workgroup 32 rows and 64 columns, turned in LDS.
template <class E, int P, bool PAIRED>
MRL_DEV void along_columns(const Source &s, __bf16 *to, int column_fragments, long at, float (&tile)[64][33]) {
    const int groups = (column_fragments + 3) / 4, block = (int)(at / groups), group = (int)(at - (long)block * groups), first = group * (PAIRED ? 32 : 64);   // (PAIRED: 32 of each)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (threadIdx.x >> 6), c = threadIdx.x & 63, row = block * 32 + r;
        // fragments in order: PAIRED has gate 0 .. 15, up 0 .. 15, gate 16 .. 31, up 16 .. 31
        const int column = PAIRED ? first + (c >> 5) * 16 + (c & 15) : first + c;
        const bool there = row < s.rows && column < s.columns;
        const float x = value_of(((const E *)s.at)[there ? row * s.ld + column + (PAIRED && (c & 16) ? s.columns : 0) : 0]);
        tile[c][r] = there ? x : 0.0f;
    }
    __syncthreads();
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, fragment = group * 4 + w;
    if (fragment >= column_fragments) return;
    f32x8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = tile[w * 16 + (lane & 15)][(lane >> 4) * 8 + i];
    put_pieces<P>(x, to + ((long)block * column_fragments + fragment) * P * KIB, lane);
}
// All operands that a call takes from its inputs, one launch for up to MOST_WORKGROUPS: the rows and columns of x, the columns and rows of W, those that are wanted.
struct Operands {
    Source x, w;
    __bf16 *x_rows, *x_columns, *w_columns, *w_rows;
    int x_row_fragments, x_column_fragments, w_column_fragments, w_row_fragments;
    unsigned end[4];   // workgroups up to and with each
    unsigned first;    // of this launch
};
constexpr unsigned MOST_WORKGROUPS = 1u << 23;   // of a launch, whose threads are counted in 32 bits
template <class E, int P>
__global__ __launch_bounds__(256) void operands_kernel(Operands o) {
    __shared__ float tile[64][33];
    const unsigned b = o.first + blockIdx.x;
    if (b < o.end[0]) along_columns<E, P, true>(o.w, o.w_columns, o.w_column_fragments, b, tile);
    else if (b < o.end[1]) along_rows<E, P, false>(o.x, o.x_rows, o.x_row_fragments, (o.x_column_fragments + 1) / 2, b - o.end[0]);
    else if (b < o.end[2]) along_columns<E, P, false>(o.x, o.x_columns, o.x_column_fragments, b - o.end[1], tile);
    else along_rows<E, P, true>(o.w, o.w_rows, o.w_row_fragments, o.w_column_fragments / 2, b - o.end[2]);
}

// ---------------------------------------------------------------- products
struct Operand {
    const __bf16 *at;
    int fragments;   // of 16 rows
    int rows;        // of a matrix of bf16 that is read as it is, `ld` apart
    long ld;
};

// a wavefront's KiB from memory to LDS
MRL_DEV void bring(const __bf16 *from, __bf16 *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
// Waits until at most LOADS of the wavefront's loads are under way and none of its LDS reads, then for the workgroup.
template <int LOADS>
MRL_DEV void meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((LOADS & 15) | (LOADS >> 4) << 14 | 7 << 4);   // (vmcnt; lgkmcnt 0)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// The tile of a product: A's fragments times B's, PA and PB pieces each, by WR wavefronts along A and WC along B, FA x FB fragments each.
// A stage is 32 of the contracted index; BUFFERS of them are in LDS or on their way.
template <int PA_, int PB_, int WR_, int WC_, int FA_, int FB_, int BUFFERS_>
struct Shape {
    static constexpr int PA = PA_, PB = PB_, WR = WR_, WC = WC_, WAVES = WR * WC, THREADS = 64 * WAVES, FA = FA_, FB = FB_, BUFFERS = BUFFERS_;
    static constexpr int ROWS = WR * FA, COLUMNS = WC * FB;   // fragments of the tile
    static constexpr int STAGE = (ROWS * PA + COLUMNS * PB), LOADS = STAGE / WAVES;   // KiB, and those that a wavefront brings
    static constexpr size_t LDS = sizeof(__bf16) * KIB * STAGE * BUFFERS;
    static_assert(STAGE % WAVES == 0 && LDS <= 160 * 1024, "whole loads that fit");
};

// A product's tiles in order, a share of neighbouring ones to each of the eight XCDs, which workgroups are dealt to in turn.  ACROSS tiles of a row
// are neighbours, then the same of the next row: the 64 tiles that an XCD works on together share few operands, which its L2 holds (all
// columns of a row first: 4 MB of W go through the L2 for every row of tiles, and 32768 rows of 512 x 2048 in bf16 take a tenth longer).
constexpr int ACROSS = 4;
struct Tiles {
    int down, across, parts;   // parts: of the contracted index
    int blocks;                // 32 of it each
    __host__ __device__ int count() const { return down * across * parts; }
    MRL_DEV void place(int &bi, int &bj, int &part, int &from, int &to) const {
        const int xcd = blockIdx.x & 7, share = count() >> 3, rest = count() & 7, number = xcd * share + min(xcd, rest) + (int)(blockIdx.x >> 3);
        part = number / (down * across);
        const int tile = number - part * down * across, group = tile / (down * ACROSS), in = tile - group * down * ACROSS, width = min(ACROSS, across - group * ACROSS);
        bi = in / width;
        bj = group * ACROSS + in - bi * width;
        const int per = (blocks + parts - 1) / parts;
        from = min(blocks, part * per);
        to = min(blocks, from + per);
    }
};

// The sums of a tile.  Operands arrive BUFFERS - 1 stages ahead.  AS_IS: A is a matrix of bf16 whose rows are whole 32 elements and start at
// 16 bytes: lanes read their eight elements where they are.
// What bounds it: LDS.  A stage of 128 x 256 in bf16 is 64 KiB read and 24 written, 700 cycles of LDS for 512 of the matrix cores; two
// workgroups a CU have one finish a tile while the other multiplies.  32768 rows of 512 x 2048 in bf16 take 175 us, of which 16 stages'
// loop is 100, the activation 19 and writing the outputs 27 at least (this card's library takes 161 us for the product alone); 256 x 256 by
// eight wavefronts, one workgroup a CU, 228, or 208 with the next tile's operands asked for ahead of a tile's end, which is slower (188) at 128 x 256;
// four wavefronts of 64 x 128 each 215.
template <class S, bool AS_IS>
MRL_DEV void multiply(const Operand &a, const Operand &b, int bi, int bj, int from, int to, __bf16 *lds, f32x4 (&acc)[S::FA][S::FB]) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = wave / S::WC, column = wave % S::WC;
    // which KiB of a stage this wavefront brings: A's first, then B's; a tile at the edge reads the last fragments again
    const __bf16 *src[S::LOADS];
    long step[S::LOADS];
#pragma unroll
    for (int l = 0; l < S::LOADS; ++l) {
        const int k = wave * S::LOADS + l;
        const bool of_a = k < S::ROWS * S::PA;
        const int in = of_a ? k : k - S::ROWS * S::PA, pieces = of_a ? S::PA : S::PB;
        const Operand &o = of_a ? a : b;
        const int fragment = min((of_a ? bi * S::ROWS : bj * S::COLUMNS) + in / pieces, o.fragments - 1);
        if (AS_IS && of_a) {
            step[l] = 32;
            src[l] = a.at + min(fragment * 16 + (lane & 15), a.rows - 1) * a.ld + from * 32 + (lane >> 4) * 8;
        } else {
            step[l] = (long)o.fragments * pieces * KIB;
            src[l] = o.at + ((long)fragment * pieces + in % pieces) * KIB + from * step[l] + lane * 8;
        }
    }
    const auto ask = [&](int stage) {
        __bf16 *const base = lds + (stage % S::BUFFERS * S::STAGE + wave * S::LOADS) * KIB;
#pragma unroll
        for (int l = 0; l < S::LOADS; ++l) {
            bring(src[l], base + l * KIB);
            src[l] += step[l];
        }
    };
    const int stages = to - from;
    constexpr bool PIECES = S::PA + S::PB > 2;
    f32x4 small[PIECES ? S::FA : 1][PIECES ? S::FB : 1] = {};   // all products but those of first pieces, which alone say what an infinity makes (split_sum)
#pragma unroll
    for (int s = 0; s < S::BUFFERS - 1; ++s)
        if (s < stages) ask(s);
    for (int s = 0; s < stages; ++s) {
        if (s + S::BUFFERS - 2 < stages) meet<(S::BUFFERS - 2) * S::LOADS>();
        else meet<0>();
        if (s + S::BUFFERS - 1 < stages) ask(s + S::BUFFERS - 1);   // into the buffer that everybody has left
        const __bf16 *const base = lds + s % S::BUFFERS * S::STAGE * KIB + lane * 8;
        const __bf16 *const pa = base + row * S::FA * S::PA * KIB, *const pb = base + (S::ROWS * S::PA + column * S::FB * S::PB) * KIB;
        bf16x8 y[S::FB][S::PB];
#pragma unroll
        for (int j = 0; j < S::FB; ++j)
#pragma unroll
            for (int p = 0; p < S::PB; ++p) y[j][p] = *reinterpret_cast<const bf16x8 *>(pb + (j * S::PB + p) * KIB);
#pragma unroll
        for (int i = 0; i < S::FA; ++i) {
            bf16x8 x[S::PA];
#pragma unroll
            for (int p = 0; p < S::PA; ++p) x[p] = *reinterpret_cast<const bf16x8 *>(pa + (i * S::PA + p) * KIB);
            constexpr int MOST = (S::PA > S::PB ? S::PA : S::PB) - 1;   // pieces' numbers add up to this at most; the smallest products first
#pragma unroll
            for (int sum = MOST; sum >= 0; --sum)
#pragma unroll
                for (int p = 0; p <= sum; ++p)
                    if (p < S::PA && sum - p < S::PB) {
#pragma unroll
                        for (int j = 0; j < S::FB; ++j) {
                            f32x4 &to = PIECES && sum > 0 ? small[PIECES ? i : 0][PIECES ? j : 0] : acc[i][j];
                            to = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[p], y[j][sum - p], to, 0, 0, 0);
                        }
                    }
        }
    }
    if constexpr (PIECES) {
#pragma unroll
        for (int i = 0; i < S::FA; ++i)
#pragma unroll
            for (int j = 0; j < S::FB; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[i][j][r] = split_sum(acc[i][j][r], small[i][j][r]);
    }
}

// 4 x 4 halves of four neighbouring lanes, transposed: element c of lane s becomes element s of lane c.  Pairs change places two
// lanes away, then halves one lane away.
MRL_DEV bf16x4 quad_transpose(bf16x4 v) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    u32x2 d = __builtin_bit_cast(u32x2, v);
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    const unsigned away = __builtin_amdgcn_mov_dpp(high ? d[0] : d[1], 0x4E, 0xF, 0xF, true);
    if (high) d[0] = away;
    else d[1] = away;
    const unsigned pick = odd ? 0x03020706u : 0x05040100u;   // bytes: 0 .. 3 of the own word, 4 .. 7 of the neighbour's
#pragma unroll
    for (int i = 0; i < 2; ++i) d[i] = __builtin_amdgcn_perm(__builtin_amdgcn_mov_dpp(d[i], 0xB1, 0xF, 0xF, true), d[i], pick);
    return __builtin_bit_cast(bf16x4, d);
}

enum { SIGMOID = MRL_GATE_SIGMOID, SILU = MRL_GATE_SILU, GELU = MRL_GATE_GELU, TANH = MRL_GATE_TANH };

MRL_DEV float activation(int act, float g) {
    float a, rest;
    if (act == GELU) return 0.5f * g * (1.0f + erff(g * 0.70710678f));
    if (act == TANH) return tanhf(g);
    sigmoid_pair(g, a, rest);
    return act == SILU ? g * a : a;
}
// and its slope
MRL_DEV void activation(int act, float g, float &value, float &slope) {
    if (act == GELU) {
        const float phi = 0.5f * (1.0f + erff(g * 0.70710678f));
        value = g * phi;
        slope = fmaf(g * 0.39894228f, expf(-0.5f * g * g), phi);
    } else if (act == TANH) {
        value = tanhf(g);
        slope = fmaf(-value, value, 1.0f);
    } else {
        float a, rest;
        sigmoid_pair(g, a, rest);
        value = act == SILU ? g * a : a;
        slope = act == SILU ? a * fmaf(g, rest, 1.0f) : a * rest;
    }
}

// sigmoid_pair holds sigmoid(g) from exp(-87) down; what is to have it as a factor (value or slope) goes on to 0 here, so that g sigmoid(g) does for the
// largest gates.  By four gates and in a branch, which hardly any takes: for every value it costs 32768 rows of 512 -> 2048 in bf16 5 us of 165.
MRL_DEV void fade(int act, const f32x4 g, f32x4 &x) {
    if ((act != SIGMOID && act != SILU) || fminf(fminf(g[0], g[1]), fminf(g[2], g[3])) >= -87.0f) return;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] *= __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g[r] + 87.0f, 0.0f) * 1.44269504f);
}

// 16 x 16 of a matrix [rows, columns] from a result's registers (row 4 g + r, column c) and into them, 0 where it has none.  bf16 goes by
// four neighbouring columns of a row, which four lanes turn among them.
MRL_DEV void store_tile(float *p, long ld, const f32x4 v, int row, int column, int rows, int columns, int g, int c) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (row + 4 * g + r < rows && column + c < columns) p[(row + 4 * g + r) * ld + column + c] = v[r];
}
MRL_DEV void store_tile(bf16_t *p, long ld, const f32x4 v, int row, int column, int rows, int columns, int g, int c) {
    const u16x4u x = __builtin_bit_cast(u16x4u, quad_transpose(__builtin_convertvector(v, bf16x4)));
    row += 4 * g + (c & 3);
    column += c & 12;
    if (row >= rows) return;
    bf16_t *const to = p + row * ld + column;
    if (column + 4 <= columns) *reinterpret_cast<u16x4u *>(to) = x;
    else {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (column + i < columns) to[i].bits = x[i];
    }
}
MRL_DEV f32x4 load_tile(const float *p, long ld, int row, int column, int rows, int columns, int g, int c) {
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const bool there = row + 4 * g + r < rows && column + c < columns;
        const float x = p[there ? (row + 4 * g + r) * ld + column + c : 0];
        v[r] = there ? x : 0.0f;
    }
    return v;
}
MRL_DEV f32x4 load_tile(const bf16_t *p, long ld, int row, int column, int rows, int columns, int g, int c) {
    row += 4 * g + (c & 3);
    column += c & 12;
    u16x4u x = {0, 0, 0, 0};
    if (row < rows) {
        const bf16_t *const from = p + row * ld + column;
        if (column + 4 <= columns) x = *reinterpret_cast<const u16x4u *>(from);
        else {
#pragma unroll
            for (int i = 0; i < 3; ++i)
                if (column + i < columns) x[i] = from[i].bits;
        }
    }
    return __builtin_convertvector(quad_transpose(__builtin_bit_cast(bf16x4, x)), f32x4);
}

struct Layer {
    int M, K, N, act;
    const void *x, *params, *grad_out;
    long x_ld, grad_out_ld;
    void *out, *grad_x;
    long out_ld, grad_x_ld;
    float *grads;
};

// Pieces of [dgate | dup].  For dW three, 22 bits and more, as fp32 has them: in bf16 two (16 bits) would be 2.5e-6 off in the 2-norm, where fp32 sums of
// products that are not split come to 1.1e-7 for 8 rows, 8e-7 for 2048 and 2e-6 for 32768, three pieces to 1.1e-7, 2e-7 and 5e-7.  16384 rows of
// 512 -> 1024 take 295 us; two took 38 less.
constexpr int COLUMN_PIECES = 3;

// FORWARD: the layer's outputs.  Otherwise [dgate | dup] as fragments, contracted along the columns (PR pieces, for dx) and along the rows
// (COLUMN_PIECES, for dW), and the sums of its columns over the wavefront's rows.
template <class E, class S, bool FORWARD, bool AS_IS, int PR>
__global__ __launch_bounds__(S::THREADS) void pre_kernel(Layer y, Operand a, Operand b, Tiles all, __bf16 *rows, __bf16 *columns, float *sums) {
    extern __shared__ __bf16 lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / S::WC, wc = wave % S::WC, g = lane >> 4, c = lane & 15;
    const E *const bias = (const E *)y.params + (long)y.K * 2 * y.N;
    const int fragments = b.fragments;   // of gate and up
    int bi, bj, part, from, to;
    all.place(bi, bj, part, from, to);
    f32x4 acc[S::FA][S::FB] = {};
    multiply<S, AS_IS>(a, b, bi, bj, from, to, lds, acc);
#pragma unroll
    for (int j = 0; j < S::FB; j += 2) {
        const int pair = (bj * S::COLUMNS + wc * S::FB + j) / 2, column = pair * 16 + c;
        const bool there = column < y.N;
        if (pair * 2 >= fragments) continue;
        const float bg = there ? value_of(bias[column]) : 0.0f, bu = there ? value_of(bias[y.N + column]) : 0.0f;
        float gate_sum = 0.0f, up_sum = 0.0f;
#pragma unroll
        for (int i = 0; i < S::FA; ++i) {
            const int fragment = bi * S::ROWS + wr * S::FA + i, row = fragment * 16 + 4 * g;
            if (fragment >= a.fragments) continue;
            if constexpr (FORWARD) {
                const f32x4 gate = acc[i][j] + bg;
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = activation(y.act, gate[r]);
                fade(y.act, gate, v);
                v *= acc[i][j + 1] + bu;
                store_tile((E *)y.out, y.out_ld, v, fragment * 16, pair * 16, y.M, y.N, g, c);
            } else {
                f32x4 dg, du, values, slopes;
                const f32x4 gate = acc[i][j] + bg;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float value, slope;
                    activation(y.act, gate[r], value, slope);
                    values[r] = value;
                    slopes[r] = slope;
                }
                fade(y.act, gate, values);
                fade(y.act, gate, slopes);
                const f32x4 grads = load_tile((const E *)y.grad_out, y.grad_out_ld, fragment * 16, pair * 16, y.M, y.N, g, c);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool inside = there && row + r < y.M;
                    const float grad = grads[r];
                    dg[r] = inside ? grad * (acc[i][j + 1][r] + bu) * slopes[r] : 0.0f;
                    du[r] = inside ? grad * values[r] : 0.0f;
                    gate_sum += dg[r];
                    up_sum += du[r];
                }
                // by columns: a fragment of 16 columns and 32 rows; this lane has rows 4 g .. 4 g + 3 of 16 of them, next to each other
                const auto put = [&](const f32x4 v, int f) {
                    bf16x4 p[SPLIT];
                    split4(v, p);
                    __bf16 *to = columns + ((long)(fragment >> 1) * fragments + f) * COLUMN_PIECES * KIB + (16 * ((fragment & 1) * 2 + (g >> 1)) + c) * 8 + (g & 1) * 4;
#pragma unroll
                    for (int k = 0; k < COLUMN_PIECES; ++k) *reinterpret_cast<bf16x4 *>(to + k * KIB) = p[k];
                    // by rows: a fragment of 16 rows and 32 columns, 16 of the gate and 16 of up
                    __bf16 *at = rows + ((long)(f >> 1) * a.fragments + fragment) * PR * KIB + (16 * ((f & 1) * 2 + (c >> 3)) + 4 * g + (c & 3)) * 8 + (c & 4);
#pragma unroll
                    for (int k = 0; k < PR; ++k) *reinterpret_cast<bf16x4 *>(at + k * KIB) = quad_transpose(p[k]);
                };
                put(dg, 2 * pair);
                put(du, 2 * pair + 1);
            }
        }
        if constexpr (!FORWARD) {
            gate_sum += __shfl_xor(gate_sum, 16);
            up_sum += __shfl_xor(up_sum, 16);
            gate_sum += __shfl_xor(gate_sum, 32);
            up_sum += __shfl_xor(up_sum, 32);
            if (g == 0) {
                float *to = sums + ((long)(bi * S::WR + wr) * fragments + 2 * pair) * 16 + c;
                to[0] = gate_sum;
                to[16] = up_sum;
            }
        }
    }
}

// dx: rows times the matrix' rows; where `all` has parts, their sums to partial [part][M, K]
template <class E, class S>
__global__ __launch_bounds__(S::THREADS) void grad_x_kernel(Layer y, Operand a, Operand b, Tiles all, float *partial) {
    extern __shared__ __bf16 lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / S::WC, wc = wave % S::WC, g = lane >> 4, c = lane & 15;
    int bi, bj, part, from, to;
    all.place(bi, bj, part, from, to);
    f32x4 acc[S::FA][S::FB] = {};
    multiply<S, false>(a, b, bi, bj, from, to, lds, acc);
#pragma unroll
    for (int i = 0; i < S::FA; ++i)
#pragma unroll
        for (int j = 0; j < S::FB; ++j) {
            const int row = (bi * S::ROWS + wr * S::FA + i) * 16, column = (bj * S::COLUMNS + wc * S::FB + j) * 16;
            if (partial != nullptr) store_tile(partial + (long)part * y.M * y.K, y.K, acc[i][j], row, column, y.M, y.K, g, c);
            else store_tile((E *)y.grad_x, y.grad_x_ld, acc[i][j], row, column, y.M, y.K, g, c);
        }
}

// dW, a share of the rows per workgroup where `parts` is more than 1: [part][K, 2 N]
template <class S>
__global__ __launch_bounds__(S::THREADS) void grad_w_kernel(int K, int N, Operand a, Operand b, Tiles all, float *out) {
    extern __shared__ __bf16 lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = wave / S::WC, wc = wave % S::WC, g = lane >> 4, c = lane & 15;
    int bi, bj, part, from, to;
    all.place(bi, bj, part, from, to);
    f32x4 acc[S::FA][S::FB] = {};
    multiply<S, false>(a, b, bi, bj, from, to, lds, acc);
    float *const here = out + (long)part * K * 2 * N;
#pragma unroll
    for (int i = 0; i < S::FA; ++i)
#pragma unroll
        for (int j = 0; j < S::FB; ++j) {
            const int fragment = bj * S::COLUMNS + wc * S::FB + j;
            store_tile(here + (fragment & 1) * N, 2L * N, acc[i][j], (bi * S::ROWS + wr * S::FA + i) * 16, (fragment >> 1) * 16, K, N, g, c);
        }
}

// The biases' gradients from the sums of rows of wavefronts, by the first workgroups, 64 columns each; the parts of dW added up, in order, by the next
// w_blocks, those of dx by the others, 1024 values each.
struct XParts {
    const float *at;
    int count;
};
template <class E>
__global__ __launch_bounds__(256) void finish_kernel(const float *parts, int count, long values, const float *sums, int rows, int columns, int w_blocks, XParts x, Layer y) {
    __shared__ float shared[4][64];
    const int bias_blocks = (columns + 63) / 64, N = y.N;
    float *const grads = y.grads;
    if ((int)blockIdx.x >= bias_blocks + w_blocks) {
        const int all = y.M * y.K;   // (parts come with few tiles)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = ((int)blockIdx.x - bias_blocks - w_blocks) * 1024 + j * 256 + (int)threadIdx.x;
            if (i >= all) break;
            float sum = x.at[i];
            for (int p = 1; p < x.count; ++p) sum += x.at[(long)p * all + i];
            give((E *)y.grad_x + i / y.K * y.grad_x_ld + i % y.K, sum);
        }
        return;
    }
    if ((int)blockIdx.x < bias_blocks) {
        const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, at = blockIdx.x * 64 + lane;
        float sum = 0.0f;
        if (at < columns) {
            float some[16] = {};
            for (int r = w; r < rows; r += 64)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float x = sums[(long)min(r + 4 * i, rows - 1) * columns + at];
                    some[i] += r + 4 * i < rows ? x : 0.0f;
                }
#pragma unroll
            for (int i = 0; i < 16; ++i) sum += some[i];
        }
        shared[w][lane] = sum;
        __syncthreads();
        const int column = (at >> 5) * 16 + (at & 15);
        if (w == 0 && at < columns && column < N)
            grads[values + (at & 16 ? N : 0) + column] = (shared[0][lane] + shared[1][lane]) + (shared[2][lane] + shared[3][lane]);
        return;
    }
    const long i = ((long)(blockIdx.x - bias_blocks) * 256 + threadIdx.x) * 4;
    if (i + 4 <= values) {
        f32x4 sum = *reinterpret_cast<const f32x4u *>(parts + i);
#pragma unroll 4
        for (int p = 1; p < count; ++p) sum += *reinterpret_cast<const f32x4u *>(parts + p * values + i);
        *reinterpret_cast<f32x4u *>(grads + i) = sum;
    } else {
        for (long j = i; j < values; ++j) {
            float sum = parts[j];
            for (int p = 1; p < count; ++p) sum += parts[p * values + j];
            grads[j] = sum;
        }
    }
}

// ---------------------------------------------------------------- few rows
// 16 rows at a time and 16 columns of gate and up by a workgroup, whose wavefronts take shares of K: straight from memory to
// v_mfma_f32_16x16x4_f32.  Reading the matrix is the work.
constexpr int FEW_WAVES = 8;
template <class E>
__global__ __launch_bounds__(64 * FEW_WAVES) void few_rows_kernel(Layer y) {
    __shared__ f32x4 sums[FEW_WAVES][2][64];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int column = blockIdx.x * 16 + c, row = blockIdx.y * 16 + c;
    const bool there = column < y.N;
    const E *const W = (const E *)y.params + (there ? column : 0);
    f32x4 gate = {0.0f, 0.0f, 0.0f, 0.0f}, up = gate;
    const int blocks = (y.K + 15) / 16;
    for (int block = w; block < blocks; block += FEW_WAVES) {
        const int k = block * 16 + 4 * g;
        float x[4], wg[4], wu[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const bool inside = k + r < y.K;
            const E *const from = W + (long)(inside ? k + r : 0) * 2 * y.N;
            x[r] = inside && row < y.M ? value_of(((const E *)y.x)[row * y.x_ld + k + r]) : 0.0f;
            wg[r] = inside ? value_of(from[0]) : 0.0f;
            wu[r] = inside ? value_of(from[y.N]) : 0.0f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            gate = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], wg[r], gate, 0, 0, 0);
            up = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], wu[r], up, 0, 0, 0);
        }
    }
    sums[w][0][lane] = gate;
    sums[w][1][lane] = up;
    __syncthreads();
    if (w != 0 || !there) return;
    for (int i = 1; i < FEW_WAVES; ++i) {
        gate += sums[i][0][lane];
        up += sums[i][1][lane];
    }
    const E *const bias = (const E *)y.params + (long)y.K * 2 * y.N;
    gate += value_of(bias[column]);
    up += value_of(bias[y.N + column]);
    f32x4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] = activation(y.act, gate[r]);
    fade(y.act, gate, v);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int at = blockIdx.y * 16 + 4 * g + r;
        if (at < y.M) give((E *)y.out + at * y.out_ld + column, v[r] * up[r]);
    }
}

// no row at all: zeros
__global__ __launch_bounds__(256) void zero_kernel(float *p, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) p[i] = 0.0f;
}

// ---------------------------------------------------------------- host
// Where the matrix cores' fp32 keep up with one launch that reads the matrix, no operands are made.  Its time grows with the products of its
// workgroups, and it reads a long K with too few loads in flight; the tiles' is 14 us for anything small, two launches.  256 -> 1024: 64 rows 7 us
// (tiles 14), 128 rows 7.6 (14), 256 rows 11.2 (14) in fp32; 256 -> 4096: 64 rows 11.3 (16.3), 12.5 in bf16 (13.6), 128 rows 19.3 (16.8); 2048 -> 512: 64 rows
// 19.6 (40.8) in fp32, 26.6 (19.3) in bf16; 2048 -> 4096: 32 rows 42.5 (59) in fp32, 52 (33.7) in bf16, 64 rows 84 (59).
inline bool few(const mrl_ctx *ctx, int dtype, int rows, int K, int N) {
    const long groups = (long)((rows + 15) / 16) * ((N + 15) / 16);
    return rows <= 256 && (dtype == MRL_F32 ? rows <= 32 || groups <= ctx->n_cus || groups * K <= 1 << 18 : K <= 512 && groups * K <= 1 << 18);
}
inline long up_to(long n, long unit) { return (n + unit - 1) / unit * unit; }

// Where things lie in the workspace, in bytes.
struct Plan {
    int M16, K16, N16;   // fragments of the rows, of the matrix' rows and (pairs) of its columns, an even number of the first two
    int pieces, row_pieces, parts, x_parts;
    size_t x_rows, w_columns, x_columns, w_rows, pre_rows, pre_columns, sums, partial, x_partial, bytes;
};
template <class S>
int tiles(long a, long b) { return (int)(((a + S::ROWS - 1) / S::ROWS) * ((b + S::COLUMNS - 1) / S::COLUMNS)); }

// 128 x 256 and 128 x 128 where there are as many tiles as CUs, 64 x 64 elsewhere.  256 -> 683, the gradient: 512 rows in fp32 take 43 us with small
// tiles and 60 with large ones, 32768 rows 683 and 602; in bf16 35 and 54, 407 and 348.
// Two pieces for dx cost 16384 rows of 512 -> 1024 35 us (tiles of 128 x 128: 48).
typedef Shape<1, 1, 2, 4, 4, 4, 3> Bf16Shape;
typedef Shape<1, 1, 4, 2, 1, 2, 4> Bf16Small;
typedef Shape<2, 1, 2, 4, 4, 4, 3> Bf16X;            // dx: 128 x 256, two pieces of [dgate | dup]
typedef Shape<2, 1, 4, 1, 1, 4, 4> Bf16XSmall;       // and 64 x 64
typedef Shape<1, 3, 2, 4, 4, 2, 4> Bf16W;            // dW: 128 x 128, three pieces of [dgate | dup]
typedef Shape<3, 3, 2, 4, 4, 2, 3> F32Shape;
typedef Shape<3, 3, 4, 2, 1, 2, 3> F32Small;
constexpr int WR_MOST = 4;
constexpr int X_STAGES = 8;   // of 32 of the contracted index, for a part of dx at least

Plan plan_of(const mrl_ctx *ctx, int dtype, int M, int K, int N, bool backward) {
    Plan p = {};
    p.M16 = (int)up_to((M + 15) / 16, 2);
    p.K16 = (int)up_to((K + 15) / 16, 2);
    p.N16 = (N + 15) / 16;
    const bool f32 = dtype == MRL_F32;
    p.pieces = f32 ? 3 : 1;
    p.row_pieces = f32 ? 3 : 2;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t was = at;
        at += up_to((long)bytes, 256);
        return was;
    };
    const auto fragments = [&](long rows16, long contracted16, int pieces) { return take(sizeof(__bf16) * KIB * (size_t)rows16 * (contracted16 / 2) * pieces); };
    if (!backward && few(ctx, dtype, M, K, N)) return p;
    p.x_rows = fragments(p.M16, p.K16, p.pieces);
    p.w_columns = fragments(2L * p.N16, p.K16, p.pieces);
    if (backward) {
        p.x_columns = fragments(p.K16, p.M16, p.pieces);
        p.w_rows = fragments(p.K16, 2L * p.N16, p.pieces);
        p.pre_rows = fragments(p.M16, 2L * p.N16, p.row_pieces);
        p.pre_columns = fragments(2L * p.N16, p.M16, COLUMN_PIECES);
        p.sums = take(sizeof(float) * ((size_t)p.M16 + WR_MOST) * 2 * p.N16 * 16);   // (a wavefront has a fragment of rows at least)
        const int all = f32 ? tiles<F32Shape>(p.K16, 2L * p.N16) : tiles<Bf16W>(p.K16, 2L * p.N16);
        const int blocks = p.M16 / 2;
        // dW's tiles are few, its contracted index is long: 2048 rows of 256 -> 683 in fp32 take 56 us, 111 with whole columns; 32768 rows 602 and 1485
        p.parts = (int)std::max<long>(1, std::min<long>((blocks + 7) / 8, (ctx->n_cus + all - 1) / all));
        if (p.parts > 1) p.partial = take(sizeof(float) * (size_t)p.parts * K * 2 * N);
        // so are dx's where there are few rows: 2048 rows of 256 -> 683 in fp32 take 56 us, 63 whole; 512 rows 43 and 53, in bf16 35 and 39
        const int large = f32 ? tiles<F32Shape>(p.M16, p.K16) : tiles<Bf16X>(p.M16, p.K16), small = f32 ? tiles<F32Small>(p.M16, p.K16) : tiles<Bf16XSmall>(p.M16, p.K16);
        p.x_parts = large >= ctx->n_cus ? 1 : std::max(1, std::min(p.N16 / X_STAGES, ctx->n_cus / small));
        if (p.x_parts > 1) p.x_partial = take(sizeof(float) * (size_t)p.x_parts * M * K);
    }
    p.bytes = at;
    return p;
}

template <class S>
Tiles tiles_in(long a, long b, int blocks, int parts = 1) { return {(int)((a + S::ROWS - 1) / S::ROWS), (int)((b + S::COLUMNS - 1) / S::COLUMNS), parts, blocks}; }
template <class E, class S, int P, int PR>
struct Launch {
    template <bool FORWARD>
    static void pre(const mrl_ctx *ctx, const Layer &y, const Plan &p, const Operand &x, const Operand &w, bool as_is, __bf16 *rows = nullptr, __bf16 *columns = nullptr,
                    float *sums = nullptr) {
        constexpr int ROW_PIECES = FORWARD ? 1 : PR;   // (not written forwards)
        const Tiles t = tiles_in<S>(p.M16, 2L * p.N16, p.K16 / 2);
        if constexpr (P == 1) {
            if (as_is) {
                hipLaunchKernelGGL((pre_kernel<E, S, FORWARD, true, ROW_PIECES>), dim3(t.count()), dim3(S::THREADS), S::LDS, ctx->stream, y, x, w, t, rows, columns, sums);
                return;
            }
        }
        hipLaunchKernelGGL((pre_kernel<E, S, FORWARD, false, ROW_PIECES>), dim3(t.count()), dim3(S::THREADS), S::LDS, ctx->stream, y, x, w, t, rows, columns, sums);
    }
    static int sum_rows(const Plan &p) { return tiles_in<S>(p.M16, 1, 1).down * S::WR; }
};

template <class E, class S>
void launch_grad_x(const mrl_ctx *ctx, const Layer &y, const Plan &p, const Operand &pre, const Operand &w, float *partial) {
    const Tiles t = tiles_in<S>(p.M16, p.K16, p.N16, p.x_parts);
    hipLaunchKernelGGL((grad_x_kernel<E, S>), dim3(t.count()), dim3(S::THREADS), S::LDS, ctx->stream, y, pre, w, t, partial);
}

template <class E, class S, class SMALL, class SX, class SXSMALL, class SW, int P, int PR>
void launch(const mrl_ctx *ctx, const Layer &y, const Plan &p, char *ws, bool backward) {
    typedef Launch<E, S, P, PR> Large;
    typedef Launch<E, SMALL, P, PR> Small;
    const bool as_is = P == 1 && y.K % 32 == 0 && y.x_ld % 8 == 0 && reinterpret_cast<uintptr_t>(y.x) % 16 == 0;
    const Operand x_rows = {as_is ? (const __bf16 *)y.x : (const __bf16 *)(ws + p.x_rows), p.M16, y.M, y.x_ld}, w_columns = {(const __bf16 *)(ws + p.w_columns), 2 * p.N16};
    Operands o = {};
    o.x = {y.x, y.x_ld, y.M, y.K};
    o.w = {y.params, 2L * y.N, y.K, y.N};
    o.x_rows = (__bf16 *)(ws + p.x_rows); o.w_columns = (__bf16 *)(ws + p.w_columns);
    o.x_columns = (__bf16 *)(ws + p.x_columns); o.w_rows = (__bf16 *)(ws + p.w_rows);
    o.x_row_fragments = p.M16; o.x_column_fragments = p.K16; o.w_column_fragments = 2 * p.N16; o.w_row_fragments = p.K16;
    const auto column_blocks = [](long fragments, long blocks) { return (unsigned)((fragments + 3) / 4 * blocks); };
    const auto row_blocks = [](long fragments, long blocks) { return (unsigned)((fragments * blocks + 3) / 4); };
    o.end[0] = column_blocks(2L * p.N16, p.K16 / 2);
    o.end[1] = o.end[0] + (as_is ? 0 : row_blocks(p.M16, p.K16 / 2));
    o.end[2] = o.end[1] + (backward ? column_blocks(p.K16, p.M16 / 2) : 0);
    o.end[3] = o.end[2] + (backward && y.grad_x ? row_blocks(p.K16, p.N16) : 0);
    for (; o.first < o.end[3]; o.first += MOST_WORKGROUPS)
        hipLaunchKernelGGL((operands_kernel<E, P>), dim3(std::min(MOST_WORKGROUPS, o.end[3] - o.first)), dim3(256), 0, ctx->stream, o);
    const bool pre_small = tiles<S>(p.M16, 2L * p.N16) < ctx->n_cus;
    if (!backward) {
        if (pre_small) Small::template pre<true>(ctx, y, p, x_rows, w_columns, as_is);
        else Large::template pre<true>(ctx, y, p, x_rows, w_columns, as_is);
        return;
    }
    __bf16 *const rows = (__bf16 *)(ws + p.pre_rows), *const columns = (__bf16 *)(ws + p.pre_columns);
    float *const sums = (float *)(ws + p.sums);
    if (pre_small) Small::template pre<false>(ctx, y, p, x_rows, w_columns, as_is, rows, columns, sums);
    else Large::template pre<false>(ctx, y, p, x_rows, w_columns, as_is, rows, columns, sums);
    const int sum_rows = pre_small ? Small::sum_rows(p) : Large::sum_rows(p);
    const Operand pre_rows = {rows, p.M16}, pre_columns = {columns, 2 * p.N16}, x_columns = {(const __bf16 *)(ws + p.x_columns), p.K16}, w_rows = {(const __bf16 *)(ws + p.w_rows), p.K16};
    if (y.grad_x != nullptr) {
        float *const partial = p.x_parts > 1 ? (float *)(ws + p.x_partial) : nullptr;
        if (tiles<SX>(p.M16, p.K16) < ctx->n_cus) launch_grad_x<E, SXSMALL>(ctx, y, p, pre_rows, w_rows, partial);
        else launch_grad_x<E, SX>(ctx, y, p, pre_rows, w_rows, partial);
    }
    const Tiles t = tiles_in<SW>(p.K16, 2L * p.N16, p.M16 / 2, p.parts);
    const long values = (long)y.K * 2 * y.N;
    float *const to = p.parts > 1 ? (float *)(ws + p.partial) : y.grads;
    hipLaunchKernelGGL((grad_w_kernel<SW>), dim3(t.count()), dim3(SW::THREADS), SW::LDS, ctx->stream, y.K, y.N, x_columns, pre_columns, t, to);
    const int bias_blocks = (2 * p.N16 * 16 + 63) / 64;
    const long w_blocks = p.parts > 1 ? (values + 1023) / 1024 : 0, x_blocks = y.grad_x != nullptr && p.x_parts > 1 ? ((long)y.M * y.K + 1023) / 1024 : 0;
    const XParts x = {(const float *)(ws + p.x_partial), p.x_parts};
    hipLaunchKernelGGL(finish_kernel<E>, dim3((unsigned)(bias_blocks + w_blocks + x_blocks)), dim3(256), 0, ctx->stream, to, p.parts, values, sums, sum_rows, 2 * p.N16 * 16,
                       (int)w_blocks, x, y);
}

int check_sizes(const char *who, int dtype, int act, int64_t rows, int in_dim, int out_dim) {
    MRL_CHECK_ARG(dtype == MRL_F32 || dtype == MRL_BF16, "%s: unknown element type %d", who, dtype);
    MRL_CHECK_ARG(act >= MRL_GATE_SIGMOID && act <= MRL_GATE_TANH, "%s: unknown activation %d", who, act);
    MRL_CHECK_ARG(rows >= 0 && rows < 1 << 26, "%s: %lld rows: 0 to 2^26 - 1 expected", who, (long long)rows);
    MRL_CHECK_ARG(in_dim >= 1 && in_dim <= 1 << 16 && out_dim >= 1 && out_dim <= 1 << 16, "%s: dims %d and %d: 1 to 65536 expected", who, in_dim, out_dim);
    return MRL_OK;
}
int check_workspace(const char *who, size_t need, void *workspace, uint64_t bytes) {
    MRL_CHECK_ARG(bytes >= need && (need == 0 || workspace != nullptr), "%s: the workspace holds %llu bytes, need %llu", who,
                  (unsigned long long)(workspace ? bytes : 0), (unsigned long long)need);
    MRL_CHECK_ARG(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: the workspace must be 16-byte aligned", who);
    return MRL_OK;
}

}  // namespace
}  // namespace glu
}  // namespace mrl

extern "C" {

int mrl_gated_linear_workspace(mrl_ctx *ctx, int dtype, int rows, int in_dim, int out_dim, int backward, uint64_t *bytes) {
    using namespace mrl;
    MRL_CHECK_ARG(ctx && bytes, "mrl_gated_linear_workspace: NULL ctx or result");
    const int rc = glu::check_sizes("mrl_gated_linear_workspace", dtype, MRL_GATE_SIGMOID, rows, in_dim, out_dim);
    if (rc != MRL_OK) return rc;
    *bytes = rows == 0 ? 0 : glu::plan_of(ctx, dtype, rows, in_dim, out_dim, backward != 0).bytes;
    return MRL_OK;
}

int mrl_gated_linear_forward(mrl_ctx *ctx, int dtype, int act, int rows, int in_dim, int out_dim, const void *in, int64_t in_ld, const void *params,
                             void *out, int64_t out_ld, void *workspace, uint64_t workspace_bytes) {
    using namespace mrl;
    using namespace mrl::glu;
    const char *who = "mrl_gated_linear_forward";
    MRL_CHECK_ARG(ctx, "%s: ctx is NULL", who);
    int rc = check_sizes(who, dtype, act, rows, in_dim, out_dim);
    if (rc != MRL_OK || rows == 0) return rc;
    MRL_CHECK_ARG(in && params && out, "%s: NULL buffer", who);
    MRL_CHECK_ARG(in_ld >= in_dim && out_ld >= out_dim, "%s: a row stride is smaller than the row", who);
    const Plan p = plan_of(ctx, dtype, rows, in_dim, out_dim, false);
    rc = check_workspace(who, p.bytes, workspace, workspace_bytes);
    if (rc != MRL_OK) return rc;
    const int64_t size = dtype == MRL_F32 ? 4 : 2;
    rc = check_apart(who, {Region("out", out, rows, size * out_dim, size * out_ld), Region("the workspace", p.bytes ? workspace : nullptr, (int64_t)p.bytes)},
                     {Region("in", in, rows, size * in_dim, size * in_ld), Region("params", params, size * 2 * out_dim * ((int64_t)in_dim + 1))});
    if (rc != MRL_OK) return rc;
    OnDevice on(ctx);
    Layer y = {};
    y.M = rows; y.K = in_dim; y.N = out_dim; y.act = act;
    y.x = in; y.x_ld = in_ld; y.params = params; y.out = out; y.out_ld = out_ld;
    if (few(ctx, dtype, rows, in_dim, out_dim)) {
        const dim3 grid((out_dim + 15) / 16, (rows + 15) / 16);
        if (dtype == MRL_F32) hipLaunchKernelGGL(few_rows_kernel<float>, grid, dim3(64 * FEW_WAVES), 0, ctx->stream, y);
        else hipLaunchKernelGGL(few_rows_kernel<bf16_t>, grid, dim3(64 * FEW_WAVES), 0, ctx->stream, y);
    } else if (dtype == MRL_F32) launch<float, F32Shape, F32Small, F32Shape, F32Small, F32Shape, 3, 3>(ctx, y, p, (char *)workspace, false);
    else launch<bf16_t, Bf16Shape, Bf16Small, Bf16X, Bf16XSmall, Bf16W, 1, 2>(ctx, y, p, (char *)workspace, false);
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}

int mrl_gated_linear_backward(mrl_ctx *ctx, int dtype, int act, int rows, int in_dim, int out_dim, const void *grad_out, int64_t grad_out_ld, const void *in,
                              int64_t in_ld, const void *params, void *grad_in, int64_t grad_in_ld, float *grads, void *workspace, uint64_t workspace_bytes) {
    using namespace mrl;
    using namespace mrl::glu;
    const char *who = "mrl_gated_linear_backward";
    MRL_CHECK_ARG(ctx, "%s: ctx is NULL", who);
    int rc = check_sizes(who, dtype, act, rows, in_dim, out_dim);
    if (rc != MRL_OK) return rc;
    MRL_CHECK_ARG(grads, "%s: NULL gradients", who);
    const int64_t values = 2LL * out_dim * (in_dim + 1), size = dtype == MRL_F32 ? 4 : 2;
    OnDevice on(ctx);
    if (rows == 0) {
        hipLaunchKernelGGL(zero_kernel, dim3((unsigned)std::min<int64_t>((values + 255) / 256, 4096)), dim3(256), 0, ctx->stream, grads, (long)values);
        MRL_CHECK_LAUNCH();
        return MRL_OK;
    }
    MRL_CHECK_ARG(grad_out && in && params, "%s: NULL buffer", who);
    MRL_CHECK_ARG(in_ld >= in_dim && grad_out_ld >= out_dim && (!grad_in || grad_in_ld >= in_dim), "%s: a row stride is smaller than the row", who);
    const Plan p = plan_of(ctx, dtype, rows, in_dim, out_dim, true);
    rc = check_workspace(who, p.bytes, workspace, workspace_bytes);
    if (rc != MRL_OK) return rc;
    rc = check_apart(who, {Region("grad_in", grad_in, rows, size * in_dim, size * grad_in_ld), Region("grads", grads, 4 * values), Region("the workspace", workspace, (int64_t)p.bytes)},
                     {Region("in", in, rows, size * in_dim, size * in_ld), Region("params", params, size * values), Region("grad_out", grad_out, rows, size * out_dim, size * grad_out_ld)});
    if (rc != MRL_OK) return rc;
    Layer y = {};
    y.M = rows; y.K = in_dim; y.N = out_dim; y.act = act;
    y.x = in; y.x_ld = in_ld; y.params = params; y.grad_out = grad_out; y.grad_out_ld = grad_out_ld;
    y.grad_x = grad_in; y.grad_x_ld = grad_in_ld; y.grads = grads;
    if (dtype == MRL_F32) launch<float, F32Shape, F32Small, F32Shape, F32Small, F32Shape, 3, 3>(ctx, y, p, (char *)workspace, true);
    else launch<bf16_t, Bf16Shape, Bf16Small, Bf16X, Bf16XSmall, Bf16W, 1, 2>(ctx, y, p, (char *)workspace, true);
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}

}  // extern "C"
