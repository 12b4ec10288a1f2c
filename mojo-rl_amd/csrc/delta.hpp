// What the kernels of the gated delta rule share (mrl_delta.hip, mrl_delta_back.hip).
//
// Per environment and head, with a = sigmoid(gate), b = sigmoid(rate), k = key / |key|, q = query / (|query| sqrt(dk)):
//   S' = a[t] S[t-1] (0 where the step before ended an episode),  u[t] = b[t] (v[t] - S'^T k[t]),  S[t] = S' + k[t] u[t]^T,
//   out[t] = S[t]^T q[t].
// TILE steps together, from the state S0 ahead of them: with G[i][j] = a[j+1] .. a[i] (1 for i = j, 0 for j > i, and 0 across a cut, whose
// a counts as 0), F[i] = a[0] .. a[i] and L[j] = G[TILE - 1][j],
//   A[i][j] = b[i] (k[i] k[j]) G[i][j] for j < i,   (1 + A) U = X,   X[i] = b[i] (v[i] - F[i] S0^T k[i]),
//   out[i] = F[i] S0^T q[i] + sum_j P[i][j] U[j],   P[i][j] = (q[i] k[j]) G[i][j],
//   S1 = F[TILE - 1] S0 + sum_j L[j] k[j] U[j]^T.
// The decays are products of the a themselves, not exponentials of differences of sums: they keep their relative accuracy
// whatever the a ahead of them were.
//
// Operands of v_mfma_f32_16x16x4_f32, lane = 16 g + n: A[row n][k = g], B[k = g][column n] -> D[row 4 g + r][column n], r = 0 .. 3.
// Four of them contract 16 values of an index; the r-th takes 4 g + r from lane group g.  So a result [16 x 16] as it stands in
// its registers is the B operand of a product that contracts its rows, and the A operand of such a product is four neighbouring
// values of a row.
#pragma once
#include <limits.h>
#include <cmath>
#include "mrl_host.hpp"
#include "mrl_device.hpp"
#include "gate.hpp"

namespace mrl {
namespace delta {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));

struct bf16_t { unsigned short bits; };

constexpr int TILE = 16;
constexpr int MOST_DIM = 128;
constexpr float EPS = 1e-6f;
// Beyond these, or NaN: blocks go one step to a tile, so that what overflows or is not finite does not meet the 0 of another step.  Below
// them no product of states, values and their gradients with each other or with keys and queries comes to 2^127: sums of a block's values and states
// by lane stay below LARGE, squared lengths below LARGE^2.
constexpr float LARGE = 1e15f, LARGE_SQUARE = 1e30f;

struct Delta {
    int T, N, H, HK, dk, dv;
    const void *query, *key, *value, *gate, *rate;
    long query_ld, key_ld, value_ld, gate_ld, rate_ld;
    const float *dones, *prev_dones, *state_in;
    void *out;
    long out_ld;
    float *state_out;
};

MRL_DEV float value_of(float x) { return x; }
MRL_DEV float value_of(bf16_t x) { return __uint_as_float((unsigned)x.bits << 16); }
MRL_DEV void give(float *p, float x) { *p = x; }
MRL_DEV void give(bf16_t *p, float x) { p->bits = __builtin_bit_cast(unsigned short, (__bf16)x); }

// four neighbouring values as they lie
template <class E> struct Four;
template <> struct Four<float> { typedef f32x4u type; };
template <> struct Four<bf16_t> { typedef u16x4u type; };
MRL_DEV f32x4 values_of(const f32x4u x) { return x; }
MRL_DEV f32x4 values_of(const u16x4u v) {
    f32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float((unsigned)v[i] << 16);
    return x;
}
// up to four neighbouring values, zeros from `n` on
MRL_DEV f32x4 load4(const float *p, int n) {
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n >= 4) x = *reinterpret_cast<const f32x4u *>(p);
    else {
        if (n > 0) x[0] = p[0];
        if (n > 1) x[1] = p[1];
        if (n > 2) x[2] = p[2];
    }
    return x;
}
MRL_DEV f32x4 load4(const bf16_t *p, int n) {
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n >= 4) {
        x = values_of(*reinterpret_cast<const u16x4u *>(p));
    } else {
        if (n > 0) x[0] = value_of(p[0]);
        if (n > 1) x[1] = value_of(p[1]);
        if (n > 2) x[2] = value_of(p[2]);
    }
    return x;
}
MRL_DEV void store4(float *p, f32x4 x, int n) {
    if (n >= 4) *reinterpret_cast<f32x4u *>(p) = x;
    else {
        if (n > 0) p[0] = x[0];
        if (n > 1) p[1] = x[1];
        if (n > 2) p[2] = x[2];
    }
}
MRL_DEV void store4(bf16_t *p, f32x4 x, int n) {
    const u16x4u v = __builtin_bit_cast(u16x4u, __builtin_convertvector(x, bf16x4));
    if (n >= 4) *reinterpret_cast<u16x4u *>(p) = v;
    else {
        if (n > 0) p[0].bits = v[0];
        if (n > 1) p[1].bits = v[1];
        if (n > 2) p[2].bits = v[2];
    }
}

MRL_DEV bool is_cut(const Delta &d, int t, int n) {
    const float *row = t > 0 ? d.dones : d.prev_dones;
    return row != nullptr && (t > 0 ? row[(long)(t - 1) * d.N + n] : row[n]) > 0.5f;
}

// This workgroup's number among all, so that neighbours, whose rows share cache lines, are on one of the eight XCDs (workgroups are dealt to them in
// turn).
MRL_DEV int group_number() {
    const int xcd = blockIdx.x & 7, share = gridDim.x >> 3, rest = gridDim.x & 7;
    return xcd * share + min(xcd, rest) + (int)(blockIdx.x >> 3);
}

// The last (or the first) step of [begin, end) that a cut is ahead of, -1 where there is none; by a whole workgroup.  `found`: an int in LDS.
template <bool LAST>
MRL_DEV int find_cut(const Delta &d, int begin, int end, int n, int *found) {
    if (d.dones == nullptr && d.prev_dones == nullptr) return -1;
    if (threadIdx.x == 0) *found = LAST ? -1 : INT_MAX;
    __syncthreads();
    int mine = LAST ? -1 : INT_MAX;
    for (int t = begin + (int)threadIdx.x; t < end; t += blockDim.x)
        if (is_cut(d, t, n)) mine = LAST ? max(mine, t) : min(mine, t);
    if (LAST && mine >= 0) atomicMax(found, mine);
    if (!LAST && mine < INT_MAX) atomicMin(found, mine);
    __syncthreads();
    const int at = *found;
    __syncthreads();
    return at == INT_MAX ? -1 : at;
}

// What is worked out from these is worked out here and not ahead of the loop around: kept there, the addresses and comparisons of all of a
// block's phases take more registers than the state.
MRL_DEV void anew(int &x) { asm volatile("" : "+v"(x)); }
MRL_DEV void anew(int &x, int &y) {
    anew(x);
    anew(y);
}

// Results of the matrix cores are not read for the ten instructions behind this.  The compiler sees to that within a block and mostly across
// branches, but in the backward kernels, of many blocks, it has been seen to read a result one instruction behind a branch: products whose next
// reader may be behind one end with it.  (Only the last needs the wait, whichever it is: one wait behind all of them.)
MRL_DEV void settle(f32x4 &x) { asm volatile("s_nop 9" : "+v"(x)); }
template <int N>
MRL_DEV void settle(f32x4 (&x)[N]) {
    if constexpr (N == 1) settle(x[0]);
    else if constexpr (N == 2) asm volatile("s_nop 9" : "+v"(x[0]), "+v"(x[1]));
    else if constexpr (N == 4) asm volatile("s_nop 9" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
    else asm volatile("s_nop 9" : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7]));
    static_assert(N == 1 || N == 2 || N == 4 || N == 8, "the row tiles of a state");
}

MRL_DEV f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// c + A B over 16 values of the contracted index
MRL_DEV f32x4 mfma16(const f32x4 a, const f32x4 b, f32x4 c) {
#pragma unroll
    for (int r = 0; r < 4; ++r) c = mfma(a[r], b[r], c);
    return c;
}

// Tiles that a workgroup prepares together, a block: as many as leave a CU's LDS room for two workgroups and more.
constexpr int tiles_forward(int DK) { return DK >= 64 ? 2 : 4; }
constexpr int tiles_backward(int DK) { return DK >= 64 ? 2 : 4; }
constexpr int SIDE = TILE + 4;        // floats from a row of a 16 x 16 matrix in LDS to the next

// From one lane to another of a row of 16, `missing` where there is none.
template <int CONTROL>
MRL_DEV float moved(float x, float missing) { return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(missing), __float_as_int(x), CONTROL, 0xF, 0xF, false)); }
// the sum over LANES neighbouring lanes, in all of them
template <int LANES>
MRL_DEV float sum_lanes(float x) {
    x += moved<0xB1>(x, 0.0f);
    x += moved<0x4E>(x, 0.0f);
    if (LANES >= 8) x += moved<0x141>(x, 0.0f);
    if (LANES >= 16) x += moved<0x140>(x, 0.0f);
    if (LANES >= 32) {
        const auto row = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(row[0]) + __uint_as_float(row[1]);
    }
    return x;
}

// G[4 g + r][n], 0 above the diagonal: in the row of 16 lanes g the products of the a behind n and ahead of 4 g, and from there on those of the group's own.
MRL_DEV f32x4 between(const float *a, int g, int n) {
    float mine = n < 4 * g ? a[n] : 1.0f;
    float run = moved<0x101>(mine, 1.0f);
    run *= moved<0x101>(run, 1.0f);
    run *= moved<0x102>(run, 1.0f);
    run *= moved<0x104>(run, 1.0f);
    run *= moved<0x108>(run, 1.0f);
    const f32x4 own = *reinterpret_cast<const f32x4 *>(a + 4 * g);
    f32x4 out;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        run *= 4 * g + r > n ? own[r] : 1.0f;
        out[r] = 4 * g + r >= n ? run : 0.0f;
    }
    return out;
}

// 1 / sqrt(x): the hardware's, a step off at most, and one of Newton's steps (0 for an infinity, like the division)
MRL_DEV float one_over_root(float x) {
    const float y = __builtin_amdgcn_rsqf(x);
    return x < 0x1p127f ? fmaf(0.5f * y, fmaf(-x * y, y, 1.0f), y) : y;
}

// The power of two to take out of a key or a query whose largest element is `most`, where products of it as it is may overflow: what is left is shorter
// than 1, and its length, sqrt(EPS) of it included, no less than 2^-5.  (Products of lengths with it undo it: |k| and EPS are in the same units.)
MRL_DEV int unit_of(float most) { return most > 0.0f ? max(-6, __builtin_amdgcn_frexp_expf(most) + 4) : -6; }
MRL_DEV float in_units(float x, int unit) { return __builtin_amdgcn_ldexpf(x, -unit); }

// the sum over the four lane groups, in all of them
MRL_DEV float sum_groups(float x) {
    const auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(half[0]) + __uint_as_float(half[1]);
    const auto row = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(row[0]) + __uint_as_float(row[1]);
}

// of two values, at little more than the price of one: their halves trade places first
MRL_DEV void sum_groups(float &x, float &y) {
    const auto half = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
    const float both = __uint_as_float(half[0]) + __uint_as_float(half[1]);   // x's in the lower half of the lanes, y's in the upper
    const auto row = __builtin_amdgcn_permlane16_swap(__float_as_uint(both), __float_as_uint(both), false, false);
    const float sum = __uint_as_float(row[0]) + __uint_as_float(row[1]);
    const auto back = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    x = __uint_as_float(back[0]);
    y = __uint_as_float(back[1]);
}

// Rows 4 g + r of column n of (1 + A)^-1, A [16][SIDE] strictly lower triangular: forward substitution, which is as exact as its terms allow
// where powers of A would grow (keys that are alike).  Four rows at a time: a lane group adds up what its own rows contribute, and all
// solve the four rows' triangle.
MRL_DEV f32x4 invert(const float *A, int g, int n) {
    f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        f32x4 own[4];
        float sum[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float *row = A + (4 * p + r) * SIDE;
            own[r] = *reinterpret_cast<const f32x4 *>(row + 4 * p);
            const f32x4 v = *reinterpret_cast<const f32x4 *>(row + 4 * g);   // (x is 0 for rows not solved yet)
            if (p > 0) sum[r] = fmaf(v[0], x[0], fmaf(v[1], x[1], fmaf(v[2], x[2], v[3] * x[3])));
        }
        if (p > 0) {
            sum_groups(sum[0], sum[1]);
            sum_groups(sum[2], sum[3]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) sum[r] = (4 * p + r == n ? 1.0f : 0.0f) - (p > 0 ? sum[r] : 0.0f);
#pragma unroll
        for (int r = 1; r < 4; ++r)
#pragma unroll
            for (int k = 0; k < r; ++k) sum[r] = fmaf(-own[r][k], sum[k], sum[r]);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = g == p ? sum[r] : x[r];
    }
    return x;
}

// A state (or its gradient) as an operand: fp32 as it is; next to rows of bf16 in three bf16 pieces (mlp_split.hpp), with which products of
// fp32 accuracy take a fifth of the matrix cores' time: v_mfma_f32_16x16x32_bf16 does in 16 cycles what eight v_mfma_f32_16x16x4_f32 do in 256.  Of
// two row tiles, lane group g has rows 4 g .. 4 g + 3 of each.
template <class E, int DK>
struct Pieces;
template <int DK>
struct Pieces<float, DK> {
    const f32x4 (&S)[DK / TILE];
    MRL_DEV explicit Pieces(const f32x4 (&s)[DK / TILE]) : S(s) {}
};
template <class V, class F>
MRL_DEV void split(const F x, V (&p)[3]) {
    F rest = x;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        p[i] = __builtin_convertvector(rest, V);
        if (i < 2) rest -= __builtin_convertvector(p[i], F);
    }
}
template <int DK>
struct Pieces<bf16_t, DK> {
    bf16x8 p[DK / 32][3];
    MRL_DEV explicit Pieces(const f32x4 (&S)[DK / TILE]) {
#pragma unroll
        for (int i = 0; i < DK / 32; ++i) split(__builtin_shufflevector(S[2 * i], S[2 * i + 1], 0, 1, 2, 3, 4, 5, 6, 7), p[i]);
    }
};
template <>
struct Pieces<bf16_t, 16> {
    bf16x4 p[3];
    MRL_DEV explicit Pieces(const f32x4 (&S)[1]) { split(S[0], p); }
};
// (Sixteen of the contracted index go as 32, half of them zeros or other pieces: a result of v_mfma_f32_16x16x16_bf16 that is another product's
// addend has been seen to come too late here, by a part in 2^18 of the sum.)
MRL_DEV f32x4 mfma_pieces(const bf16x8 a, const bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
MRL_DEV bf16x8 beside(const bf16x4 a, const bf16x4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
MRL_DEV bf16x8 alone(const bf16x4 a) { return beside(a, bf16x4{(__bf16)0.0f, (__bf16)0.0f, (__bf16)0.0f, (__bf16)0.0f}); }

// A block's keys or queries in LDS: rows of fp32; of bf16 rows and columns.
template <class E, int DK, int STEPS>
struct Rows;
template <int DK, int STEPS>
struct Rows<float, DK, STEPS> {
    static constexpr int ROW = DK + 4;
    static constexpr size_t FLOATS = (size_t)STEPS * ROW;
    float *at;
    MRL_DEV void put(int slot, int column, const f32x4 x) { *reinterpret_cast<f32x4 *>(at + slot * ROW + column) = x; }
    // rows 4 g + r of a tile, element c of a column tile
    MRL_DEV f32x4 column(int tile, int i, int g, int c) const {
        f32x4 k;
#pragma unroll
        for (int r = 0; r < 4; ++r) k[r] = at[(tile * TILE + 4 * g + r) * ROW + i * TILE + c];
        return k;
    }
    // products of a tile's rows with another's: [row of this][row of that]
    MRL_DEV f32x4 with(const Rows &that, int tile, int g, int c) const {
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < DK / TILE; ++i)
            x = mfma16(*reinterpret_cast<const f32x4 *>(at + (tile * TILE + c) * ROW + i * TILE + 4 * g),
                       *reinterpret_cast<const f32x4 *>(that.at + (tile * TILE + c) * ROW + i * TILE + 4 * g), x);
        return x;
    }
    // S^T k of a tile's 16 rows k: [row of the tile][column of S]
    MRL_DEV f32x4 ask(int tile, int g, int c, const Pieces<float, DK> &S) const {
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < DK / TILE; ++i) x = mfma16(*reinterpret_cast<const f32x4 *>(at + (tile * TILE + c) * ROW + i * TILE + 4 * g), S.S[i], x);
        return x;
    }
    // S + sum_i k[i] x[i]^T over a tile's rows k
    MRL_DEV void add(int tile, int g, int c, const f32x4 x, f32x4 (&S)[DK / TILE]) const {
#pragma unroll
        for (int i = 0; i < DK / TILE; ++i) S[i] = mfma16(column(tile, i, g, c), x, S[i]);
        settle(S);
    }
};
template <int DK, int STEPS>
struct Rows<bf16_t, DK, STEPS> {
    static constexpr int ROW = DK + 8, TURNED = STEPS + 4;   // elements from a row to the next, and from a column
    static constexpr size_t FLOATS = ((size_t)STEPS * ROW + (size_t)DK * TURNED) / 2;
    float *at;
    MRL_DEV __bf16 *rows() const { return reinterpret_cast<__bf16 *>(at); }
    MRL_DEV __bf16 *columns() const { return rows() + STEPS * ROW; }
    MRL_DEV void put(int slot, int column, const f32x4 x) {
        const bf16x4 v = __builtin_convertvector(x, bf16x4);
        *reinterpret_cast<bf16x4 *>(rows() + slot * ROW + column) = v;
#pragma unroll
        for (int i = 0; i < 4; ++i) columns()[(column + i) * TURNED + slot] = v[i];
    }
    MRL_DEV bf16x4 row4(int tile, int i, int g, int c) const { return *reinterpret_cast<const bf16x4 *>(rows() + (tile * TILE + c) * ROW + i * TILE + 4 * g); }
    MRL_DEV bf16x4 column4(int tile, int i, int g, int c) const { return *reinterpret_cast<const bf16x4 *>(columns() + (i * TILE + c) * TURNED + tile * TILE + 4 * g); }
    MRL_DEV f32x4 column(int tile, int i, int g, int c) const { return __builtin_convertvector(column4(tile, i, g, c), f32x4); }
    MRL_DEV f32x4 with(const Rows &that, int tile, int g, int c) const {
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (DK == 16) return mfma_pieces(alone(row4(tile, 0, g, c)), alone(that.row4(tile, 0, g, c)), x);
#pragma unroll
        for (int i = 0; i < DK / 32; ++i)
            x = mfma_pieces(beside(row4(tile, 2 * i, g, c), row4(tile, 2 * i + 1, g, c)), beside(that.row4(tile, 2 * i, g, c), that.row4(tile, 2 * i + 1, g, c)), x);
        return x;
    }
    MRL_DEV f32x4 ask(int tile, int g, int c, const Pieces<bf16_t, DK> &S) const {
        f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f}, small = x;
        if constexpr (DK == 16) {
            const bf16x4 k = row4(tile, 0, g, c);
            return mfma_pieces(beside(k, k), alone(S.p[0]), x) + mfma_pieces(beside(k, k), beside(S.p[1], S.p[2]), small);
        } else {
#pragma unroll
            for (int i = 0; i < DK / 32; ++i) {
                const bf16x8 k = beside(row4(tile, 2 * i, g, c), row4(tile, 2 * i + 1, g, c));
                small = mfma_pieces(k, S.p[i][2], small);
                x = mfma_pieces(k, S.p[i][0], x);
                small = mfma_pieces(k, S.p[i][1], small);
            }
            return x + small;
        }
    }
    // (two pieces of x side by side are 32 of the contracted index, with each key twice)
    MRL_DEV void add(int tile, int g, int c, const f32x4 x, f32x4 (&S)[DK / TILE]) const {
        bf16x4 p[3];
        split(x, p);
        const bf16x8 upper = beside(p[0], p[1]), lower = alone(p[2]);
#pragma unroll
        for (int i = 0; i < DK / TILE; ++i) {
            const bf16x4 k = column4(tile, i, g, c);
            S[i] = mfma_pieces(beside(k, k), upper, mfma_pieces(beside(k, k), lower, S[i]));
        }
        settle(S);
    }
};
template <class E>
constexpr size_t rows_floats(int DK, int tiles, bool keeps) {
    const size_t steps = (size_t)TILE * tiles, rows = sizeof(E) == 4 ? steps * (DK + 4) : (steps * (DK + 8) + DK * (steps + 4)) / 2;
    return 2 * rows + (keeps ? 3 : 2) * tiles * TILE * SIDE + 15 * steps + 4;
}

// What the wavefronts of a workgroup keep in LDS of a block's rows, from `lds` on.  KEEPS: A beside its inverse.
template <class E, int DK, int TILES_, bool KEEPS>
struct Block {
    static constexpr int TILES = TILES_, STEPS = TILE * TILES, LANES = DK / 4;
    Rows<E, DK, STEPS> keys, queries;
    float *As, *Ts, *Ps;
    // of every step: a, 1 - a (0 at a cut), b, 1 - b, 1 / |k|, 1 / (|q| sqrt(dk)), the squared lengths of key and query, F, L, b F / |k|, F / (|q| sqrt(dk)), L / |k|; of every tile F[15]
    float *as, *rests, *bs, *rate_rests, *key_lengths, *query_lengths, *kscale, *qscale, *from, *to, *key_reads, *query_reads, *key_takes, *wholes;
    int *key_units, *query_units;   // where span is 1: the powers of two that the key and the query, and all lengths of them here, are without
    int t0, span;   // the first step; steps of a tile: 1 where a value is not finite, so that it goes where the formulas send it and nowhere else
    MRL_DEV explicit Block(float *lds) {
        keys.at = lds;
        queries.at = lds + keys.FLOATS;
        As = queries.at + queries.FLOATS;
        Ts = KEEPS ? As + TILES * TILE * SIDE : As;
        Ps = Ts + TILES * TILE * SIDE;
        as = Ps + TILES * TILE * SIDE;
        rests = as + STEPS;
        bs = rests + STEPS;
        rate_rests = bs + STEPS;
        key_lengths = rate_rests + STEPS;
        query_lengths = key_lengths + STEPS;
        kscale = query_lengths + STEPS;
        qscale = kscale + STEPS;
        from = qscale + STEPS;
        to = from + STEPS;
        key_reads = to + STEPS;
        query_reads = key_reads + STEPS;
        key_takes = query_reads + STEPS;
        key_units = reinterpret_cast<int *>(key_takes + STEPS);
        query_units = key_units + STEPS;
        wholes = key_takes + 3 * STEPS;
    }
    MRL_DEV int time_of(int slot) const { return t0 + (slot >> 4) * span + (slot & 15); }
    MRL_DEV bool there(const Delta &d, int slot) const { return ((slot & 15) < span) & (time_of(slot) < d.T); }
    MRL_DEV bool full(const Delta &d) const { return span == TILE && t0 + STEPS <= d.T; }
    MRL_DEV f32x4 four(const float *scalars, int tile, int g) const { return *reinterpret_cast<const f32x4 *>(scalars + tile * TILE + 4 * g); }

    // a row by LANES lanes of four, and EPS beside its squares, without the row's power of two, which it returns
    MRL_DEV static int in_row_units(f32x4 &x, float &eps) {
        float most = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
#pragma unroll
        for (int s = 1; s < LANES; s *= 2) most = fmaxf(most, __shfl_xor(most, s));
        const int unit = unit_of(most);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = in_units(x[j], unit);
        eps = in_units(EPS, 2 * unit);
        return unit;
    }

    // Keys, queries (QUERIES), their lengths, gates and rates; rows behind the last step are zeros that change nothing (a = 1, b = 0).
    // Whether a value is too large for products with 0, or none.  All loads are asked for ahead of the first use of any: one wait for them, not
    // five.  They read a row that is there in place of one that is not, so that they stand together without a branch among them.
    template <bool QUERIES>
    MRL_DEV bool load(const Delta &d, int n, int h, int hk, int thread) {
        constexpr int ASKED = STEPS * LANES > 256 ? STEPS * LANES / 256 : 1;   // rows of a thread at a time: all of them where there are four wavefronts
        bool odd = false;
        const int part = (thread & 63) % LANES, count = d.dk - 4 * part, first = count > 0 ? 4 * part : 0, rows = (int)blockDim.x / LANES;
        const E *const key = (const E *)d.key + n * d.key_ld + (long)hk * d.dk + first, *const query = (const E *)d.query + n * d.query_ld + (long)hk * d.dk + first;
        const long key_step = (long)d.N * d.key_ld, query_step = (long)d.N * d.query_ld;
        const bool whole = (d.dk & 3) == 0, all = full(d) && d.dk == DK;
        E gate = {}, rate = {};   // (a workgroup has as many threads as a block has steps, or more)
        bool cut = false;
        if (thread < STEPS) {
            const int t = min(time_of(thread), d.T - 1);
            const long row = (long)t * d.N + n;
            gate = ((const E *)d.gate)[row * d.gate_ld + h];
            rate = ((const E *)d.rate)[row * d.rate_ld + h];
            cut = is_cut(d, t, n);
        }
        const auto take = [&](int slot, f32x4 k, f32x4 q) {
            if (!all) {
                const bool here = there(d, slot) & (count > 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    k[j] = here ? k[j] : 0.0f;
                    q[j] = here ? q[j] : 0.0f;
                }
            }
            float k_eps = EPS, q_eps = EPS;
            if (span == 1) {
                const int k_unit = in_row_units(k, k_eps), q_unit = in_row_units(q, q_eps);
                if (part == 0) {
                    key_units[slot] = k_unit;
                    query_units[slot] = q_unit;
                }
            }
            keys.put(slot, 4 * part, k);
            const float kk = sum_lanes<LANES>(fmaf(k[0], k[0], fmaf(k[1], k[1], fmaf(k[2], k[2], k[3] * k[3]))));
            float qq = 0.0f;
            if (QUERIES) {
                queries.put(slot, 4 * part, q);
                qq = sum_lanes<LANES>(fmaf(q[0], q[0], fmaf(q[1], q[1], fmaf(q[2], q[2], q[3] * q[3]))));
            }
            odd |= !(kk + qq < LARGE_SQUARE);
            if (part == 0) {   // (squares for now: prepare() makes lengths of them)
                kscale[slot] = kk + k_eps;
                qscale[slot] = qq + q_eps;
            }
        };
        const f32x4 none = {0.0f, 0.0f, 0.0f, 0.0f};
        if (whole) {
            for (int ahead = thread / LANES; ahead < STEPS; ahead += ASKED * rows) {
                typename Four<E>::type k[ASKED], q[ASKED];
#pragma unroll
                for (int i = 0; i < ASKED; ++i) {
                    const long t = min(time_of(ahead + i * rows), d.T - 1);
                    k[i] = *reinterpret_cast<const typename Four<E>::type *>(key + t * key_step);
                    if (QUERIES) q[i] = *reinterpret_cast<const typename Four<E>::type *>(query + t * query_step);
                }
#pragma unroll
                for (int i = 0; i < ASKED; ++i)
                    if (ahead + i * rows < STEPS) take(ahead + i * rows, values_of(k[i]), QUERIES ? values_of(q[i]) : none);
            }
        } else {
            for (int slot = thread / LANES; slot < STEPS; slot += rows) {
                const long t = min(time_of(slot), d.T - 1);
                take(slot, load4(key + t * key_step, count), QUERIES ? load4(query + t * query_step, count) : none);
            }
        }
        if (thread < STEPS) {
            float a = 1.0f, rest = 0.0f, b = 0.0f, other = 0.0f;
            if (there(d, thread)) {
                sigmoid_pair(value_of(gate), a, rest);
                sigmoid_pair(value_of(rate), b, other);
                odd |= !(a + b < LARGE);
                if (cut) a = rest = 0.0f;
            }
            as[thread] = a;
            rests[thread] = rest;
            bs[thread] = b;
            rate_rests[thread] = other;
        }
        return odd;
    }

    // What does not depend on the state, by halves of a tile, a wavefront each: A and (1 + A)^-1; P (QUERIES) and the decays.  Each half makes the
    // lengths that it needs.
    static constexpr int HALVES = 2 * TILES;
    template <bool QUERIES>
    MRL_DEV void prepare(const Delta &d, int half, int g, int c) {
        const int tile = half >> 1;
        const float kc = one_over_root(kscale[tile * TILE + c]);
        const f32x4 decay = between(as + tile * TILE, g, c);
        f32x4 products;
        if (half & 1) {
            const int slot = tile * TILE + c;
            const float qs = one_over_root(qscale[slot] * (float)d.dk), a = as[slot], b = bs[slot];
            if (QUERIES) products = queries.with(keys, tile, g, c);
            float ahead = a, behind = moved<0x101>(a, 1.0f);   // products up to here, and of those behind
            ahead *= moved<0x111>(ahead, 1.0f);
            behind *= moved<0x101>(behind, 1.0f);
            ahead *= moved<0x112>(ahead, 1.0f);
            behind *= moved<0x102>(behind, 1.0f);
            ahead *= moved<0x114>(ahead, 1.0f);
            behind *= moved<0x104>(behind, 1.0f);
            ahead *= moved<0x118>(ahead, 1.0f);
            behind *= moved<0x108>(behind, 1.0f);
            if (g == 0) {
                from[slot] = ahead;
                to[slot] = behind;
                key_lengths[slot] = kc;
                query_lengths[slot] = qs;
                key_reads[slot] = b * ahead * kc;
                query_reads[slot] = ahead * qs;
                key_takes[slot] = behind * kc;
                if (c == TILE - 1) wholes[tile] = ahead;
            }
            if (QUERIES) {
                const f32x4 squares = four(qscale, tile, g);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float qi = one_over_root(squares[r] * (float)d.dk);
                    Ps[(tile * TILE + 4 * g + r) * SIDE + c] = 4 * g + r >= c ? qi * (kc * products[r]) * decay[r] : 0.0f;
                }
            }
        } else {
            products = keys.with(keys, tile, g, c);
            const f32x4 b = four(bs, tile, g), squares = four(kscale, tile, g);
            float *A = As + tile * TILE * SIDE;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float ki = one_over_root(squares[r]);
                A[(4 * g + r) * SIDE + c] = 4 * g + r > c ? b[r] * ki * (kc * products[r]) * decay[r] : 0.0f;
            }
            __builtin_amdgcn_wave_barrier();
            const f32x4 x = invert(A, g, c);
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r = 0; r < 4; ++r) Ts[(tile * TILE + 4 * g + r) * SIDE + c] = x[r];
        }
    }
    MRL_DEV bool cut_ahead(int tile) const { return span == 1 && as[tile * TILE] == 0.0f; }   // hides whatever the state holds
};

// A value tile as a result's registers: row 4 g + r, column c.  `rows` points at the column (at one that is there) of the environment's row of
// step 0, `step` elements from a step to the next.  First the loads, later what is made of them.
template <class E, class B, int TILES>
MRL_DEV void ask_values(const Delta &d, const B &block, const E *rows, long step, int g, E (&V)[TILES][4]) {
    if (block.full(d)) {
        const E *const first = rows + 4 * g * step;
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile)
#pragma unroll
            for (int r = 0; r < 4; ++r) V[tile][r] = first[(long)(block.t0 + tile * TILE + r) * step];
    } else {
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile)
#pragma unroll
            for (int r = 0; r < 4; ++r) V[tile][r] = rows[min(block.time_of(tile * TILE + 4 * g + r), d.T - 1) * step];
    }
}
template <class E, class B, int TILES>
MRL_DEV bool take_values(const Delta &d, const B &block, const E (&asked)[TILES][4], bool live, int g, f32x4 (&V)[TILES]) {
    float size = 0.0f;
    const bool full = block.full(d);
#pragma unroll
    for (int tile = 0; tile < TILES; ++tile)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            V[tile][r] = live & (full | block.there(d, tile * TILE + 4 * g + r)) ? value_of(asked[tile][r]) : 0.0f;   // (no branches: the registers may be others' in one of them)
            size += fabsf(V[tile][r]);
        }
    return !(size < LARGE);
}
// and back: one tile
template <class E, class B>
MRL_DEV void store_values(const Delta &d, const B &block, E *rows, long step, bool live, int tile, int g, const f32x4 x) {
    if (block.full(d)) {
        E *const first = rows + 4 * g * step;
        if (live) {
#pragma unroll
            for (int r = 0; r < 4; ++r) give(first + (long)(block.t0 + tile * TILE + r) * step, x[r]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int slot = tile * TILE + 4 * g + r;
            if (live && block.there(d, slot)) give(rows + block.time_of(slot) * step, x[r]);
        }
    }
}
template <int B>
MRL_DEV bool is_odd(const f32x4 (&S)[B]) {
    float size = 0.0f;
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) size += fabsf(S[i][r]);
    return !(size < LARGE);
}

// U[4 g + r][c] of a tile; sk: S0^T k
template <class E, int DK, int TILES, bool KEEPS>
MRL_DEV f32x4 solve(const Block<E, DK, TILES, KEEPS> &block, int tile, int g, int c, const f32x4 v, const f32x4 sk) {
    const f32x4 b = block.four(block.bs, tile, g), reads = block.four(block.key_reads, tile, g);
    f32x4 x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = fmaf(b[r], v[r], -reads[r] * sk[r]);
    const f32x4 inverse = *reinterpret_cast<const f32x4 *>(block.Ts + tile * TILE * SIDE + c * SIDE + 4 * g);
    f32x4 u = mfma16(inverse, x, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
    settle(u);
    return u;
}
// S0 becomes S1
template <class E, int DK, int TILES, bool KEEPS>
MRL_DEV void go_on(const Block<E, DK, TILES, KEEPS> &block, int tile, int g, int c, f32x4 u, f32x4 (&S)[DK / TILE]) {
    u *= block.four(block.key_takes, tile, g);
    const float whole = block.wholes[tile];
#pragma unroll
    for (int i = 0; i < DK / TILE; ++i) S[i] *= whole;
    block.keys.add(tile, g, c, u, S);
}

// ---------------------------------------------------------------- a long rollout of a few environments, in parts
// Where heads and environments leave CUs without work the steps are cut into parts of `per` blocks.  A part takes the state S ahead of it to
// M S + B, a product of the steps' contractions and what it makes of a zero state; M and B of all parts come side by side (M as the part's result for
// the columns of the identity, without values), a second launch goes through them, M S + B, and then every part has its first state.  The
// same, from the last part to the first and with M^T, for the gradient of the state.  A part with a cut has M = 0, and says so; its B comes from the
// steps from the last cut on alone, and the gradient of the state ahead of it from those up to the first cut.
// States are kept as lanes hold them: [environment and head][part][tile of 16 columns][tile of 16 rows][lane][4].
struct Parts {
    int count, per;      // count 1: no parts
    float *ends;         // B of every part, then M: column_tiles(dv) + dk / 16 tiles
    float *starts;       // S ahead of every part
    int *cuts;           // whether a part has a cut
};
inline int padded(int dk) { return dk <= 16 ? 16 : dk <= 32 ? 32 : dk <= 64 ? 64 : 128; }
inline int column_tiles(int dv) { return (dv + TILE - 1) / TILE; }
inline int blocks_of(int T, int tiles) { return (T + TILE * tiles - 1) / (TILE * tiles); }
constexpr int floats_of(int DK) { return DK * TILE; }   // of a column tile

// How many parts: as many as give every CU PART_GROUPS workgroups, but no more than sqrt(20 blocks).  A part takes 13 to 16 us for each of its
// blocks of 128 x 128, twice, and the way through the parts 0.6 us for each of them, which is least at sqrt(50 blocks), but flat: 10 to 40 make no
// difference that is not lost between two runs.  8192 steps of 2 environments of 8 heads of 128 x 128 in bf16 take 265 us with two a CU,
// 274 to 322 with one, 312 with three; the gradient of 1001 steps of 7 environments of 3 heads of 40 x 24 130, 144 and 130.
constexpr int PART_GROUPS = 2, MOST_PARTS = 1024;
inline Parts parts_of(const mrl_ctx *ctx, const mrl_delta *r, int tiles) {
    Parts p = {};
    const int blocks = blocks_of(r->T, tiles), tile_columns = column_tiles(r->value_dim);
    const long groups = (long)r->N * r->heads * ((tile_columns + 7) / 8);
    const long want = std::min<long>({(long)blocks, (long)PART_GROUPS * ctx->n_cus / groups, (long)std::sqrt(20.0 * blocks), (long)MOST_PARTS});
    p.count = 1;
    p.per = blocks;
    if (want < 4) return p;
    p.per = (int)((blocks + want - 1) / want);
    p.count = (blocks + p.per - 1) / p.per;
    return p;
}
inline size_t ends_floats(const mrl_delta *r, const Parts &p) {
    const int DK = padded(r->key_dim);
    return p.count > 1 ? (size_t)r->N * r->heads * p.count * (column_tiles(r->value_dim) + DK / TILE) * floats_of(DK) : 0;
}
inline size_t starts_floats(const mrl_delta *r, const Parts &p) {
    return p.count > 1 ? (size_t)r->N * r->heads * p.count * column_tiles(r->value_dim) * floats_of(padded(r->key_dim)) : 0;
}
inline size_t cuts_floats(const mrl_delta *r, const Parts &p) { return p.count > 1 ? ((size_t)r->N * r->heads * p.count + 63) / 64 * 64 : 0; }

// M, B and the first states of all parts of blocks of the backward pass
int launch_starts(const mrl_ctx *ctx, int dtype, const Delta &d, const Parts &p);
// S ahead of every such block, to states [N * H][blocks][column tiles][DK / 16][64][4]
int launch_states(const mrl_ctx *ctx, int dtype, const Delta &d, const Parts &p, float *states, int blocks);
// the gradients of the states behind all parts, to p.starts, from those of parts with none behind them in `local`, laid out alike
int launch_grad_ends(const mrl_ctx *ctx, const Delta &d, const Parts &p, const float *grad_state_out, const float *local);

size_t forward_bytes(const mrl_ctx *ctx, const mrl_delta *r);
int check_sizes(const char *who, const mrl_delta *r);
int check(const char *who, const mrl_ctx *ctx, const mrl_delta *r);
Delta describe(const mrl_delta *r);
__global__ void pass_state_kernel(const float *from, float *to, long n);

}  // namespace delta
}  // namespace mrl
