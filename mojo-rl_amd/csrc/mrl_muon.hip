// Orthogonalised updates of weight matrices: Newton-Schulz products, and the optimiser's step around them.
//
// X = G / (|G| + eps) (Frobenius norm), then `steps` times  A = X X^T,  B = b A + c A A,  X <- a X + B X, on the side with fewer
// rows (m <= n): the quintic a s + b s^3 + c s^5 takes every singular value s of X into about [0.7, 1.2].
//
// Products.  Every operand is kept as two fp16 pieces of its fp32 value times a power of two, hi = fp16(x) and
// lo = fp16(x - hi): 22 significant bits.  A product is hi hi + hi lo + lo hi on the fp16 matrix cores with fp32 sums, a third of
// their rate and 2.4 times that of the fp32 instructions.  What is left out, lo lo and the pieces' rounding, is at most 2^-21 of
// a product, about what rounding the sum of a few hundred fp32 products costs (against 64 bits the results are closer than those
// of fp32 products).  The powers of two: X has norm at most sqrt(m) 1.2 and entries around 1 / sqrt(m n) .. 1 / sqrt(n), A and B
// entries below 3; times about sqrt(m n) (at most 2^14) and m (at most 2^13) they use fp16's range from the top, and a piece that
// ends among the subnormals is off by 2^-25 of a typical entry.
//
// Layout.  "Rows times rows": all three products contract the index that runs along the rows of both operands (A and B are
// symmetric, X is kept both ways), so every operand is read the same way.  A plane pair holds, for 16 rows and 32 of the
// contracted index, the 64 lanes' operands of v_mfma_f32_16x16x32_f16 in lane order, 1 KiB of hi and 1 KiB of lo next to
// each other: loads are whole and in order.  Element (row r, index k): lane 16 ((k % 32) / 8) + r % 16, k % 8.
// The sides are padded to multiples of 64 with zeros, which the products keep zero.
#include <limits.h>
#include <cmath>
#include "mrl_host.hpp"
#include "mrl_device.hpp"

namespace mrl {
namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float QA = 3.4445f, QB = -4.7750f, QC = 2.0315f;
constexpr int MOST = 16;        // matrices of a launch, where they differ
constexpr size_t BATCH_BYTES = 256 << 20, GROUP_ROOM = 1 << 30;   // of workspace from which on a launch takes no more matrices, alike or not
constexpr int LOAD = 32;        // sides of what a workgroup of the second launch takes
constexpr int CHUNK = 1024;     // elements that a workgroup of the first launch takes at a time
constexpr int MOST_SUMS = 1024;  // partial sums of squares per matrix

struct bf16_t { unsigned short bits; };

struct Mat {
    const void *in;
    void *out;
    float *momentum;
    int rows, cols, m, n, mp, np;   // the caller's sides; the shorter and the longer one, and both padded
    int tall;                       // rows > cols: X is the transpose
    int sums;                       // partial sums of squares
    float sx;                       // what X is stored times; A and B: sa
    float gram, square, update, result;   // sums to A, A A to B, B X to X, X to the caller: sa / sx^2, c / sa, 1 / sa, 1 / sx
    float factor;                   // of the update
    size_t x, xt, xt1, a, b, partial; // planes and partial sums: bytes from the workspace's start
};
struct Rest { float *p; const float *g; float2 *state; long n; };   // parameters that Adam updates
struct Group {
    int count, rests;
    int sym_tile, update_tile;   // sides of the products' tiles
    int begin_sym[MOST], begin_update[MOST];   // a matrix's first tile among all; none: INT_MAX
    size_t alike_in, alike_kept;               // mrl_orthogonalize: bytes from a matrix to the next, all described by the first
    int alike_sym, alike_update;               // and its tiles
    Mat mat[MOST];
    Rest rest[MOST + 1];
    double eps;
    float mu, keep;         // momentum; 1 - lr weight_decay
    int nesterov;
    float lr, beta1, beta2, omb1, omb2, adam_eps, bc1, bc2;
};
static_assert(sizeof(Group) <= 3584 && sizeof(Group) % 4 == 0, "kernel arguments");
constexpr size_t GROUP_BYTES = (sizeof(Group) + 63) / 64 * 64;

// what is there, for pointers that come out of memory
template <class T>
MRL_DEV auto in_memory(T *p) { return (__attribute__((address_space(1))) T *)p; }
template <class T>
MRL_DEV T *in_workspace(const Group *kept, size_t bytes) { return (T *)((char *)kept + bytes); }
MRL_DEV _Float16 *planes(const Group *kept, size_t bytes) { return in_workspace<_Float16>(kept, bytes); }

// a description out of memory, all at once
MRL_DEV Mat described(const Mat &m) {
    Mat own;
    __builtin_memcpy(&own, (const __attribute__((address_space(4))) Mat *)&m, sizeof(Mat));
    return own;
}

enum { F32 = 0, BF16 = 1, MUON = 2 };   // what a matrix is read from and written to
// Matrix k of the group, from the one that describes it; those of mrl_orthogonalize are alike, any number of them in a launch.
template <int KIND>
MRL_DEV int describes(int k) { return KIND == MUON ? k : 0; }
template <int KIND>
MRL_DEV Mat matrix(const Group &g, Mat m, int k) {
    if (KIND != MUON) {
        m.in = (const char *)m.in + k * g.alike_in;
        m.out = (char *)m.out + k * g.alike_in;
        const size_t kept = k * g.alike_kept;
        m.x += kept;
        m.xt += kept;
        m.xt1 += kept;
        m.a += kept;
        m.b += kept;
        m.partial += kept;
    }
    return m;
}

// What is orthogonalised, element i; FIRST: with MUON its momentum is brought up to date.
template <int KIND, bool FIRST = false>
MRL_DEV float source(const Group &g, const Mat &m, size_t i) {
    if (KIND == BF16) return __uint_as_float((unsigned)in_memory((const unsigned short *)m.in)[i] << 16);
    const float x = in_memory((const float *)m.in)[i];
    if (KIND == F32) return x;
    const auto at = in_memory(m.momentum) + i;
    float v = *at;
    if (FIRST) {
        v = fmaf(g.mu, v, x);
        *at = v;
    }
    return g.nesterov ? fmaf(g.mu, v, x) : v;
}
template <int KIND>
MRL_DEV double square_of(const Group &g, const Mat &m, size_t i) {
    const double x = source<KIND, true>(g, m, i);
    return x * x;
}
// Adam on the parameters between the matrices, by workgroup `block` of `blocks`
MRL_DEV void adam_rest(const Group &g, int block, int blocks) {
    for (int k = 0; k < g.rests; ++k) {
        const Rest &r = g.rest[k];
        for (long i = (long)block * blockDim.x + threadIdx.x; i < r.n; i += (long)blocks * blockDim.x)
            adam_one(r.p[i], r.g[i], r.state[i], g.lr, g.beta1, g.beta2, g.omb1, g.omb2, g.adam_eps, g.bc1, g.bc2);
    }
}
// Sums of squares of every matrix, in 64 bits and a fixed order, and Adam (3.6 us for 256 x 256, 8 for 2048 x 2048, 2 TB/s).  The group's description, 3 KiB of arguments that cost the
// host 1.5 us a launch, goes to the workspace, where the launches behind this one find it.
template <int KIND>
__global__ __launch_bounds__(256) void sums_kernel(Group g, Group *kept) {
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = threadIdx.x; i < (int)(sizeof(Group) / 4); i += 256) reinterpret_cast<int *>(kept)[i] = reinterpret_cast<const int *>(&g)[i];
    if (KIND == MUON && (int)blockIdx.y == g.count) {
        adam_rest(g, blockIdx.x, gridDim.x);
        return;
    }
    const Mat m = matrix<KIND>(g, g.mat[describes<KIND>(blockIdx.y)], blockIdx.y);
    const int block = blockIdx.x;
    if (block >= m.sums) return;
    const size_t size = (size_t)m.rows * m.cols;
    double sum = 0.0;
#pragma unroll 4
    for (size_t i = (size_t)block * 256 + threadIdx.x; i < size; i += (size_t)m.sums * 256) sum += square_of<KIND>(g, m, i);
    __shared__ double part[256];
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) part[threadIdx.x] += part[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) in_workspace<double>(kept, m.partial)[block] = part[0];
}

// Four neighbours along the contracted index (k a multiple of 4) of a row, in pieces
struct Piece {
    f16x4 hi, lo;
    Piece() = default;
    MRL_DEV explicit Piece(const f32x4 x) {
        hi = __builtin_convertvector(x, f16x4);
        lo = __builtin_convertvector(x - __builtin_convertvector(hi, f32x4), f16x4);
    }
    MRL_DEV f32x4 value() const { return __builtin_convertvector(hi, f32x4) + __builtin_convertvector(lo, f32x4); }
    MRL_DEV void load(const _Float16 *p) {
        hi = *reinterpret_cast<const f16x4 *>(p);
        lo = *reinterpret_cast<const f16x4 *>(p + 512);
    }
    MRL_DEV void store(_Float16 *p) const {
        *reinterpret_cast<f16x4 *>(p) = hi;
        *reinterpret_cast<f16x4 *>(p + 512) = lo;
    }
};
// where it is: of the 16 x 16 that start at (row, k), multiples of 16, and in them that of row r (below 16) and k = 4 quarter
MRL_DEV size_t square_at(int rows, int row, int k) { return ((size_t)(k >> 5) * (rows >> 4) + (row >> 4)) * 1024 + (k & 16) * 16; }
MRL_DEV int piece_in(int r, int quarter) { return (quarter >> 1) * 128 + r * 8 + (quarter & 1) * 4; }

// What X is multiplied by as it is read: the norm from the partial sums, in a fixed order.
MRL_DEV double scale_of(const Group &g, const Mat &m, double *part) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < m.sums; i += 256) sum += in_workspace<double>(&g, m.partial)[i];
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) part[threadIdx.x] += part[threadIdx.x + w];
        __syncthreads();
    }
    return (double)m.sx / (sqrt(part[0]) + g.eps);
}
// A square of X and of its transpose in pieces, through LDS: read along the caller's rows, written along both sides.
template <int KIND>
MRL_DEV void load_square(const Group &g, const Mat &m, int block, double scale, float (&tile)[LOAD][LOAD + 1]) {
    const int across = m.np / LOAD, i0 = block / across * LOAD, j0 = block % across * LOAD;
    for (int e = threadIdx.x; e < LOAD * LOAD; e += 256) {
        const int slow = e / LOAD, fast = e % LOAD;                            // fast runs along the caller's rows
        const int i = m.tall ? fast : slow, j = m.tall ? slow : fast;
        float x = 0.0f;
        if (i0 + i < m.m && j0 + j < m.n) {
            const size_t at = m.tall ? (size_t)(j0 + j) * m.m + (i0 + i) : (size_t)(i0 + i) * m.n + (j0 + j);
            x = (float)((double)source<KIND>(g, m, at) * scale);
        }
        tile[i][j] = x;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < LOAD * LOAD / 4; e += 256) {
        const int r = e % LOAD, c = e / LOAD * 4;
        const int in = (c & 16) * 16 + piece_in(r & 15, (c & 15) >> 2);
        Piece(f32x4{tile[r][c], tile[r][c + 1], tile[r][c + 2], tile[r][c + 3]}).store(planes(&g, m.x) + square_at(m.mp, i0 + r, j0) + in);
        Piece(f32x4{tile[c][r], tile[c + 1][r], tile[c + 2][r], tile[c + 3][r]}).store(planes(&g, m.xt) + square_at(m.np, j0 + r, i0) + in);
    }
}
// 5 us for 256 x 256, 16 for 2048 x 2048, a thirtieth of the whole: 3 TB/s.  Up to eight workgroups a CU, so that the norm is taken less
// often (a workgroup per square: 18 us, four of 1024 x 1024 19 for 15).
template <int KIND>
__global__ __launch_bounds__(256) void load_kernel(const Group *__restrict__ group) {
    const Group &g = *group;
    __shared__ double part[256];
    __shared__ float tile[LOAD][LOAD + 1];
    const Mat m = matrix<KIND>(g, described(g.mat[describes<KIND>(blockIdx.y)]), blockIdx.y);
    const int squares = m.mp / LOAD * (m.np / LOAD);
    if ((int)blockIdx.x >= squares) return;
    const double scale = scale_of(g, m, part);
    for (int block = blockIdx.x; block < squares; block += gridDim.x) {
        load_square<KIND>(g, m, block, scale, tile);
        __syncthreads();
    }
}

// 4 x 4 halves of four neighbouring lanes, transposed: element c of lane s becomes element s of lane c.  Pairs change places two
// lanes away, then halves one lane away.
MRL_DEV f16x4 quad_transpose(f16x4 v) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    u32x2 d = __builtin_bit_cast(u32x2, v);
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    const unsigned away = __builtin_amdgcn_mov_dpp(high ? d[0] : d[1], 0x4E, 0xF, 0xF, true);
    if (high) d[0] = away;
    else d[1] = away;
    const unsigned pick = odd ? 0x03020706u : 0x05040100u;   // bytes: 0 .. 3 of the own word, 4 .. 7 of the neighbour's
#pragma unroll
    for (int i = 0; i < 2; ++i) d[i] = __builtin_amdgcn_perm(__builtin_amdgcn_mov_dpp(d[i], 0xB1, 0xF, 0xF, true), d[i], pick);
    return __builtin_bit_cast(f16x4, d);
}

enum { GRAM = 0, SQUARE = 1, UPDATE = 2 };

// tile number `tile` on and above the diagonal: column bj has tiles 0 .. bj
MRL_DEV void above_diagonal(int tile, int &bi, int &bj) {
    bj = __builtin_amdgcn_readfirstlane((int)((sqrtf(8.0f * tile + 1.0f) - 1.0f) * 0.5f));
    while (bj * (bj + 1) / 2 > tile) --bj;
    while ((bj + 1) * (bj + 2) / 2 <= tile) ++bj;
    bi = tile - bj * (bj + 1) / 2;
}

// Which of `tiles` tiles, of which matrix, a workgroup works on.  Workgroups go to the eight XCDs in turn; each XCD gets a run of
// tiles that share operands, so that its L2 is read more often than what is behind it (every matrix on every XCD instead: eight of
// 777 x 333 212 us for 177).  All first tiles are looked at, from one scalar load, not one after the other.
template <int STAGE, int KIND, int TILE>
MRL_DEV Mat find_tile(const Group &g, int count, int tiles, int &bi, int &bj) {
    const int xcd = blockIdx.x & 7, each = tiles >> 3, more = tiles & 7;
    int id = xcd * each + min(xcd, more) + (blockIdx.x >> 3), k = 0;
    if (KIND != MUON && count > 1) {
        const int each_has = STAGE == UPDATE ? g.alike_update : g.alike_sym;
        k = __builtin_amdgcn_readfirstlane(id / each_has);
        id -= k * each_has;
    } else if (count > 1) {
        const int(&begin)[MOST] = STAGE == UPDATE ? g.begin_update : g.begin_sym;
#pragma unroll
        for (int i = 1; i < MOST; ++i) k += id >= begin[i];
        id -= begin[k];
    }
    const Mat m = matrix<KIND>(g, described(g.mat[describes<KIND>(k)]), k);
    if (STAGE == UPDATE) {
        const int rows = (m.mp + TILE - 1) / TILE, panel = __builtin_amdgcn_readfirstlane(id / (4 * rows)), in = id - panel * 4 * rows;
        const int width = min(4, (m.np + TILE - 1) / TILE - 4 * panel);   // panels of four columns, row by row
        bi = __builtin_amdgcn_readfirstlane(in / width);
        bj = 4 * panel + in - bi * width;
    } else {
        above_diagonal(id, bi, bj);
    }
    return m;
}

// Fragments of 16 x 16 sums: a lane has rows i .. i + 3, i = 4 (lane / 16), of column j = lane % 16.  `fi`, `fj`: of the fragment.
template <int STAGE>
MRL_DEV bool inside(const Mat &m, int fi, int fj) { return fi < m.mp && fj < (STAGE == UPDATE ? m.np : m.mp); }
// What the sums are added to, X or A there: asked for early, all at once.
template <int STAGE>
MRL_DEV void ask(const Group &g, const Mat &m, int from, int fi, int fj, Piece &piece) {
    const int lane = threadIdx.x & 63;
    if (STAGE == GRAM || !inside<STAGE>(m, fi, fj)) return;
    const _Float16 *of = planes(&g, STAGE == UPDATE ? (from ? m.xt1 : m.xt) : m.a);
    piece.load(of + square_at(STAGE == UPDATE ? m.np : m.mp, fj, fi) + piece_in(lane & 15, lane >> 4));
}
// A square's sums in pieces, as columns (row j, k = i) and as rows (row i, k = j)
MRL_DEV void store_both(_Float16 *columns, int column_rows, _Float16 *rows, int row_rows, int fi, int fj, const f32x4 v) {
    const int lane = threadIdx.x & 63, quarter = lane >> 4, column = lane & 15;
    Piece piece(v);
    piece.store(columns + square_at(column_rows, fj, fi) + piece_in(column, quarter));
    if (rows == nullptr) return;
    piece.hi = quad_transpose(piece.hi);
    piece.lo = quad_transpose(piece.lo);
    piece.store(rows + square_at(row_rows, fi, fj) + piece_in(4 * quarter + (column & 3), column >> 2));
}
// A square of the last X to the caller.
template <int KIND>
MRL_DEV void give(const Group &g, const Mat &m, int fi, int fj, const f32x4 v) {
    const int lane = threadIdx.x & 63, i = fi + 4 * (lane >> 4), j = fj + (lane & 15);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (i + e >= m.m || j >= m.n) continue;
        const size_t at = m.tall ? (size_t)j * m.m + (i + e) : (size_t)(i + e) * m.n + j;
        const float o = v[e] * m.result;
        if (KIND == BF16) {
            in_memory((unsigned short *)m.out)[at] = __builtin_bit_cast(unsigned short, (__bf16)o);
        } else if (KIND == F32) {
            in_memory((float *)m.out)[at] = o;
        } else {
            const auto w = in_memory((float *)m.out) + at;
            *w = fmaf(-m.factor, o, *w * g.keep);
        }
    }
}
// What becomes of the sums.
template <int STAGE, int KIND>
MRL_DEV void finish(const Group &g, const Mat &m, int from, int last, bool diagonal, int fi, int fj, f32x4 v, const Piece &piece) {
    if (!inside<STAGE>(m, fi, fj)) return;
    if (STAGE == UPDATE) {
        v = QA * piece.value() + v * m.update;
        if (last) give<KIND>(g, m, fi, fj, v);
        else store_both(planes(&g, (from ? m.xt : m.xt1)), m.np, planes(&g, m.x), m.mp, fi, fj, v);
    } else {
        _Float16 *to = planes(&g, STAGE == GRAM ? m.a : m.b);
        if (STAGE == GRAM) v = v * m.gram;
        else v = QB * piece.value() + v * m.square;
        store_both(to, m.mp, diagonal ? nullptr : to, m.mp, fi, fj, v);
    }
}

// Products of up to FEW rows on the fp32 matrix cores, which round every sum to nearest.  The fp16 ones add eight products at a time and
// cut off what is below 2^-23 of the largest, so their errors go towards 0, and with few rows the same way in every entry.  Off from 64
// bits, fp16 / fp32 / plain fp32: 8 x 64 1.7e-6, 0.8e-6, 0.8e-6; 1 x 500 1.1e-6, 0.4e-6, 0.4e-6; 8 x 721 1.6e-6, 1.1e-6, 0.9e-6.  On the fp16
// ones matrices of 17 to 48 rows are 0.4 to 1.4 times as far off as plain fp32 products, of 64 and more 0.3 to 1.1 times.  (16 x 16: 18 us
// for 14.)
constexpr int FEW = 16;
// 16 x 16 sums over 32 of the contracted index, four at a time
MRL_DEV void multiply_few(const f16x8 &ph, const f16x8 &pl, const f16x8 &qh, const f16x8 &ql, f32x4 &acc) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float p = (float)ph[i] + (float)pl[i], q = (float)qh[i] + (float)ql[i];
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(p, q, acc, 0, 0, 0);
    }
}
template <int F>
MRL_DEV void multiply(const f16x8 (&p)[F], const f16x8 (&q)[F], f32x4 (&acc)[F][F]) {
#pragma unroll
    for (int fi = 0; fi < F; ++fi)
#pragma unroll
        for (int fj = 0; fj < F; ++fj) acc[fi][fj] = __builtin_amdgcn_mfma_f32_16x16x32_f16(p[fi], q[fj], acc[fi][fj], 0, 0, 0);
}

template <int STAGE>
MRL_DEV void operands(const Group &g, const Mat &m, int from, const _Float16 *&P, const _Float16 *&Q, int &blocks) {
    P = planes(&g, STAGE == GRAM ? m.x : STAGE == SQUARE ? m.a : m.b);
    Q = planes(&g, STAGE == GRAM ? m.x : STAGE == SQUARE ? m.a : (from ? m.xt1 : m.xt));
    blocks = (STAGE == GRAM ? m.np : m.mp) / 32;
}

// A tile of 32 x 32 by four wavefronts that share the contracted index, operands straight to registers.  `there`: whether these four have
// a tile, or only come to the barrier.
// LONG: every STRETCH blocks of 32 of the contracted index begin sums of their own, so that rounding costs as much at 32768 as at 4096
// (64 rows: 1.6e-6 off 64 bits at 4096, at 32768 2.9e-6 in one sum, 1.5e-6 in stretches).  The registers that it takes cost shorter
// sums 0.2 us a launch, 256 x 256 69 us for 66.
constexpr int STRETCH = 128;
typedef f32x4 SmallSums[4][4][64];   // [fragment][wavefront][lane]
template <int STAGE, int KIND, bool LONG>
MRL_DEV void small_product(const Group &g, const Mat &m, int bi, int bj, int from, int last, SmallSums &sums, bool there = true) {
    const _Float16 *P, *Q;
    int blocks;
    operands<STAGE>(g, m, from, P, Q, blocks);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
    const int p_fragments = m.mp / 16, q_fragments = (STAGE == UPDATE ? m.np : m.mp) / 16;
    const _Float16 *p = P + bi * 2 * 1024 + lane * 8, *q = Q + bj * 2 * 1024 + lane * 8;
    f32x4 acc[2][2] = {};
    const int fi = (bi * 2 + (wave >> 1)) * 16, fj = (bj * 2 + (wave & 1)) * 16;
    Piece piece;
    if (there) ask<STAGE>(g, m, from, fi, fj, piece);
    struct Operands { f16x8 ph[2], pl[2], qh[2], ql[2]; };
    auto load = [&](int kb, Operands &o) {
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const _Float16 *pf = p + ((size_t)kb * p_fragments + f) * 1024, *qf = q + ((size_t)kb * q_fragments + f) * 1024;
            o.ph[f] = *reinterpret_cast<const f16x8 *>(pf);
            o.pl[f] = *reinterpret_cast<const f16x8 *>(pf + 512);
            o.qh[f] = *reinterpret_cast<const f16x8 *>(qf);
            o.ql[f] = *reinterpret_cast<const f16x8 *>(qf + 512);
        }
    };
    const bool few = m.m <= FEW;   // then the other squares are of zeros
    if (!there || (few && (bi > 0 || (STAGE != UPDATE && bj > 0)))) blocks = 0;
    auto work = [&](const Operands &o) {
        if (few) {
            multiply_few(o.ph[0], o.pl[0], o.qh[0], o.ql[0], acc[0][0]);
            if (STAGE == UPDATE) {
                multiply_few(o.ph[0], o.pl[0], o.qh[1], o.ql[1], acc[0][1]);
                // the compiler has been seen to read these 8 instructions later where blocks join, not the 10 that it leaves within one
                asm volatile("s_nop 9" : "+v"(acc[0][0]), "+v"(acc[0][1]));
            }
            return;
        }
        multiply<2>(o.pl, o.qh, acc);
        multiply<2>(o.ph, o.ql, acc);
        multiply<2>(o.ph, o.qh, acc);
    };
    auto stretch = [&](int start, int end) {
        // two steps' operands under way together (more bring nothing)
        int kb = start + wave;
        for (; kb + 4 < end; kb += 8) {
            Operands one, two;
            load(kb, one);
            load(kb + 4, two);
            work(one);
            work(two);
        }
        if (kb < end) {
            Operands one;
            load(kb, one);
            work(one);
        }
    };
    if (LONG) {
        f32x4 total[2][2] = {};
        for (int start = 0; start < blocks; start += STRETCH) {
            stretch(start, min(blocks, start + STRETCH));
#pragma unroll
            for (int f = 0; f < 4; ++f) {
                total[f >> 1][f & 1] = total[f >> 1][f & 1] + acc[f >> 1][f & 1];
                acc[f >> 1][f & 1] = f32x4{};
            }
        }
#pragma unroll
        for (int f = 0; f < 4; ++f) acc[f >> 1][f & 1] = total[f >> 1][f & 1];
    } else {
        stretch(0, blocks);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) sums[f][wave][lane] = acc[f >> 1][f & 1];
    __syncthreads();
    const f32x4 v = (sums[wave][0][lane] + sums[wave][1][lane]) + (sums[wave][2][lane] + sums[wave][3][lane]);
    if (there) finish<STAGE, KIND>(g, m, from, last, bi == bj, fi, fj, v, piece);
}
// Tile (bi, bj) of a side of 32 F of a matrix with few rows, whose neighbours in the launch have more: in squares of 32 x 32, one behind the
// other for each 256 lanes, so that such a matrix comes out as in launches of its own, bit by bit.  (8-1024-1024-1024-4 takes 301 us
// with the fp16 cores for its first layer too: the squares are done before the other layers' tiles are.)
template <int STAGE, int KIND, int F>
MRL_DEV void few_squares(const Group &g, const Mat &m, int bi, int bj, int from, int last, SmallSums *sums) {
    const int teams = blockDim.x / 256, team = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
    const int rows = min(F, m.mp / 32 - bi * F), columns = min(F, (STAGE == UPDATE ? m.np : m.mp) / 32 - bj * F);
    for (int k0 = 0; k0 < rows * columns; k0 += teams) {
        const int k = k0 + team, i = bi * F + k % rows, j = bj * F + k / rows;
        small_product<STAGE, KIND, STAGE == GRAM>(g, m, i, j, from, last, sums[team], k < rows * columns && (STAGE == UPDATE || i <= j));
        __syncthreads();
    }
}

// a wavefront's KiB of hi (0) or lo (1) from memory to LDS (the offset counts on both sides)
template <int PIECE>
MRL_DEV void bring(const _Float16 *from, _Float16 *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from, (__attribute__((address_space(3))) void *)to, 16, PIECE * 1024, 0);
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

// One product, a tile of 32 F x 32 F per workgroup.  GRAM: A = X X^T; SQUARE: B = b A + c A A; both symmetric, so only tiles on and
// above the diagonal are worked out and written to both sides.  UPDATE: X <- a X + B X, `last` to the caller.
// A set of four wavefronts shares the tile, 16 F x 16 F each, that of 128 of eight, 64 x 32 each.  At 96 two sets take turns at the
// contracted index and add up at the end.  Either way there are two wavefronts on a SIMD, one of which hands over its requests while the
// other multiplies (five steps of 2048 x 2048 564 us; 598 with one set at 96, 627 with four wavefronts at 128 too; 1536 x 1536 352
// for 386).  At 64, where two workgroups fit a CU, two sets do so only if there are no more tiles than CUs and more than 1024 to contract:
// 1400 x 1400 271 us for 289, 1000 x 4000 350 for 366, but 1024 x 1024 174 for 172 (a launch that takes all of a CU's LDS starts later).
// Operands go from memory to LDS past the registers, a stage of 32 of the contracted index at a time and BUFFERS stages ahead, because
// a stage is multiplied in less time than memory takes to answer.
// Bound by the matrix cores where there are tiles for all CUs: 2048 x 2048 in tiles of 128, an update takes 53 us, 0.97 PFLOP/s in fp16
// (a large fp16 product of this card's library: 1.1); a symmetric product in tiles of 96 34, 0.8 PFLOP/s.  Fewer tiles are bound by the
// stages' way through LDS, 0.2 to 0.35 us each at 64.
// A tile at the edge reads the last rows' operands again where it has none of its own, and leaves what comes of them.
template <int F> constexpr int BUFFERS = F == 3 ? 3 : 4;
constexpr int TWO_SETS = 1024;   // what is contracted by two sets at 64 is longer
template <int F> constexpr int STAGE_HALVES = 2 * 2 * F * 1024;   // [operand][fragment of 16 rows][hi, lo][512]
template <int F> constexpr int WAVES = F == 4 ? 8 : 4;
template <int F, int SETS> constexpr size_t RING_BYTES = sizeof(_Float16) * SETS * BUFFERS<F> * STAGE_HALVES<F>;
template <int STAGE, int KIND, int F, int SETS>
__global__ __launch_bounds__(64 * WAVES<F> * SETS) void product_kernel(const Group *__restrict__ group, int count, int tiles, int from, int last) {
    const Group &g = *group;
    constexpr int SIDE = 2 * F, AHEAD = BUFFERS<F>, ACROSS = WAVES<F> / 2, FP = F, FQ = SIDE / ACROSS, OWN = FQ, LOADS = 2 * OWN;
    extern __shared__ _Float16 lds[];
    int bi, bj;
    const Mat m = find_tile<STAGE, KIND, 32 * F>(g, count, tiles, bi, bj);
    static_assert(RING_BYTES<F, SETS> >= sizeof(SmallSums) * WAVES<F> * SETS / 4, "sums of every four wavefronts");
    if (KIND == MUON && m.m <= FEW) {   // (matrices that are alike go to tiles of 32 in this case)
        few_squares<STAGE, KIND, F>(g, m, bi, bj, from, last, reinterpret_cast<SmallSums *>(lds));
        return;
    }
    const _Float16 *P, *Q;
    int blocks;
    operands<STAGE>(g, m, from, P, Q, blocks);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % WAVES<F>;
    const int set = SETS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / WAVES<F>;
    _Float16 *const ring = lds + set * AHEAD * STAGE_HALVES<F>;
    blocks /= SETS;
    // the first half of the wavefronts brings in P, the other Q, OWN fragments each
    const int row = wave / ACROSS, column = wave % ACROSS, operand = row, fragments = ((operand && STAGE == UPDATE) ? m.np : m.mp) / 16;
    const _Float16 *src[OWN];
#pragma unroll
    for (int f = 0; f < OWN; ++f)
        src[f] = (operand ? Q : P) + min((operand ? bj : bi) * SIDE + column * OWN + f, fragments - 1) * 1024 + lane * 8 + set * fragments * 1024;
    int in_at = wave * OWN * 1024;   // where in LDS the next stage goes
    auto brought = [&]() {
#pragma unroll
        for (int f = 0; f < OWN; ++f) src[f] += SETS * fragments * 1024;
        in_at = in_at >= (AHEAD - 1) * STAGE_HALVES<F> ? in_at - (AHEAD - 1) * STAGE_HALVES<F> : in_at + STAGE_HALVES<F>;
    };
    const int p = row * FP * 1024 + lane * 8, q = (SIDE + column * FQ) * 1024 + lane * 8;
    int at = 0;   // of the stage that is worked on
    auto read = [&](int where) { return *reinterpret_cast<const f16x8 *>(ring + at + where); };
    f32x4 acc[FP][FQ] = {};
    // A stage's 3 FP FQ products in three groups.  The meeting behind which the next stage is there, and this one's buffer free, stands
    // ahead of the last group.  Requests to LDS and memory go out among the products, at most one ahead of each: a wavefront takes 16
    // cycles or more to hand over either, in which the matrix cores would wait if they stood together.  A buffer that the meeting
    // freed is asked for from there to the next meeting: EARLY loads in the last group, the others in the next stage's first two.
    constexpr int N = FP * FQ, READS = FP + FQ, EARLY = F == 4 ? 1 : F == 3 ? 1 : 0;
    auto request = [&](int load) {
        if (load % 2 == 0) bring<0>(src[load / 2], ring + in_at + load / 2 * 1024);
        else bring<1>(src[load / 2], ring + in_at + load / 2 * 1024);
    };
    auto product = [&](int k, const f16x8 (&x)[FP], const f16x8 (&y)[FQ]) {
        acc[k / FQ][k % FQ] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[k / FQ], y[k % FQ], acc[k / FQ][k % FQ], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto first_groups = [&](f16x8 (&ph)[FP], f16x8 (&pl)[FP], f16x8 (&qh)[FQ], bool more) {
        constexpr int STEP = (2 * N - READS) / (LOADS - EARLY);
        f16x8 ql[FQ];
#pragma unroll
        for (int k = 0; k < 2 * N; ++k) {
            if (k < FQ) ql[k] = read(q + 512 + k * 1024);
            else if (k < READS) ph[k - FQ] = read(p + (k - FQ) * 1024);
            else if ((k - READS) % STEP == 0 && (k - READS) / STEP < LOADS - EARLY && more) request(EARLY + (k - READS) / STEP);
            if (k < N) product(k, pl, qh);
            else product(k - N, ph, ql);
        }
        if (more) brought();
    };
    auto last_group = [&](f16x8 (&ph)[FP], f16x8 (&pl)[FP], f16x8 (&qh)[FQ], f16x8 (&next)[FQ], bool more) {
        at = at == (AHEAD - 1) * STAGE_HALVES<F> ? 0 : at + STAGE_HALVES<F>;
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (k < FQ) next[k] = read(q + k * 1024);
            else if (k < READS) pl[k - FQ] = read(p + 512 + (k - FQ) * 1024);
            else if ((k - READS) % 3 == 1 && (k - READS) / 3 < EARLY && more) request((k - READS) / 3);
            product(k, ph, qh);
        }
    };
    f16x8 ph[FP], pl[FP], qa[FQ], qb[FQ];
    for (int s = 0; s < AHEAD - 1 && s < blocks; ++s) {
#pragma unroll
        for (int load = 0; load < LOADS; ++load) request(load);
        brought();
    }
    if (AHEAD - 1 < blocks) {
#pragma unroll
        for (int load = 0; load < EARLY; ++load) request(load);
        meet<(AHEAD - 2) * LOADS + EARLY>();
    } else {
        meet<0>();
    }
#pragma unroll
    for (int f = 0; f < FQ; ++f) qa[f] = read(q + f * 1024);
#pragma unroll
    for (int f = 0; f < FP; ++f) pl[f] = read(p + 512 + f * 1024);
    int s = 0;
    for (; s + 1 + AHEAD < blocks; s += 2) {
        first_groups(ph, pl, qa, true);
        meet<(AHEAD - 2) * LOADS>();   // stages s + 2 .. s + AHEAD - 1 may be on their way
        last_group(ph, pl, qa, qb, true);
        first_groups(ph, pl, qb, true);
        meet<(AHEAD - 2) * LOADS>();
        last_group(ph, pl, qb, qa, true);
    }
    auto end_group = [&](f16x8 (&qh)[FQ]) {
#pragma unroll
        for (int k = 0; k < N; ++k) product(k, ph, qh);
    };
    for (; s < blocks; s += 2) {
        first_groups(ph, pl, qa, s - 1 + AHEAD < blocks);
        if (SETS > 1 && s + 1 == blocks) {
            end_group(qa);
            break;
        }
        meet<0>();
        last_group(ph, pl, qa, qb, s + AHEAD < blocks);
        first_groups(ph, pl, qb, s + AHEAD < blocks);
        if (s + 2 == blocks) {
            end_group(qb);
            break;
        }
        meet<0>();
        last_group(ph, pl, qb, qa, false);
    }
    // sums of the other set: a set finishes every second fragment
    auto mine = [&](int f) { return SETS == 1 || f % SETS == set; };
    if (SETS > 1) {
        f32x4 *sums = reinterpret_cast<f32x4 *>(lds) + wave * N * 64 + lane;
        meet<0>();
#pragma unroll
        for (int f = 0; f < N; ++f)
            if (!mine(f)) sums[f * 64] = acc[f / FQ][f % FQ];
        meet<0>();
#pragma unroll
        for (int f = 0; f < N; ++f)
            if (mine(f)) acc[f / FQ][f % FQ] = acc[f / FQ][f % FQ] + sums[f * 64];
    }
    const int fi = (bi * SIDE + row * FP) * 16, fj = (bj * SIDE + column * FQ) * 16;
    Piece pieces[N];
#pragma unroll
    for (int f = 0; f < N; ++f)
        if (mine(f)) ask<STAGE>(g, m, from, fi + 16 * (f / FQ), fj + 16 * (f % FQ), pieces[f]);
#pragma unroll
    for (int f = 0; f < N; ++f)
        if (mine(f)) finish<STAGE, KIND>(g, m, from, last, bi == bj, fi + 16 * (f / FQ), fj + 16 * (f % FQ), acc[f / FQ][f % FQ], pieces[f]);
}

// The same for small matrices, where a product is shorter than the way of a stage through memory and LDS and back: a tile of
// 32 x 32 per workgroup, straight to registers.  256 x 256: 4.2, 4.3 and 4.6 us for the three, most of it the launch and the trips to
// memory one behind the other (description, operands, sums).
template <int STAGE, int KIND, bool LONG>
__global__ __launch_bounds__(256) void small_product_kernel(const Group *__restrict__ group, int count, int tiles, int from, int last) {
    const Group &g = *group;
    __shared__ SmallSums sums;
    int bi, bj;
    const Mat m = find_tile<STAGE, KIND, 32>(g, count, tiles, bi, bj);
    small_product<STAGE, KIND, LONG>(g, m, bi, bj, from, last, sums);
}

// A small matrix by one workgroup in one launch, the optimiser's part included: all operands stay in LDS, sixteen wavefronts take
// 16 x 16 sums each and meet behind every product.  Five steps of 64 x 64: 20 us instead of 75 in launches of their own, 64 x 128 25
// instead of 78, 64 x 256 37 instead of 82, eleven of 216 x 10 25 instead of 116.  (Operands out of the caches instead: 28, 43 and 30
// us for the first, second and last, bound by what a CU's L1 gives, and from 96 x 128 on longer than the launches.)
constexpr int WHOLE_LDS = 160 * 1024, WHOLE_MOST = 5;   // squares of 16 x 16 of X per wavefront
constexpr size_t whole_lds(int mp, int np) { return sizeof(_Float16) * 4 * mp * (size_t)(np + mp); }   // X, its transpose, A, B
// sums of square (bi, bj) over `blocks` times 32, of those every `step`th from number `first`
MRL_DEV f32x4 square_sum(bool few, const _Float16 *P, int p_rows, int bi, const _Float16 *Q, int q_rows, int bj, int blocks, int first = 0, int step = 1) {
    const int lane = threadIdx.x & 63;
    const _Float16 *p = P + bi * 1024 + lane * 8 + first * p_rows * 64, *q = Q + bj * 1024 + lane * 8 + first * q_rows * 64;
    f32x4 acc = {};
    if (few) {
        for (int kb = first; kb < blocks; kb += step, p += step * p_rows * 64, q += step * q_rows * 64)
            multiply_few(*reinterpret_cast<const f16x8 *>(p), *reinterpret_cast<const f16x8 *>(p + 512), *reinterpret_cast<const f16x8 *>(q),
                         *reinterpret_cast<const f16x8 *>(q + 512), acc);
        return acc;
    }
#pragma unroll 2
    for (int kb = 0; kb < blocks; ++kb, p += p_rows * 64, q += q_rows * 64) {
        const f16x8 ph = *reinterpret_cast<const f16x8 *>(p), pl = *reinterpret_cast<const f16x8 *>(p + 512);
        const f16x8 qh = *reinterpret_cast<const f16x8 *>(q), ql = *reinterpret_cast<const f16x8 *>(q + 512);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, qh, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, ql, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, qh, acc, 0, 0, 0);
    }
    return acc;
}
template <int KIND, bool SOME_FEW>
__global__ __launch_bounds__(1024) void whole_kernel(Group g, int steps) {
    extern __shared__ _Float16 lds[];
    if (KIND == MUON && (int)blockIdx.x >= g.count) {
        adam_rest(g, blockIdx.x - g.count, gridDim.x - g.count);
        return;
    }
    const Mat m = matrix<KIND>(g, g.mat[describes<KIND>(blockIdx.x)], blockIdx.x);
    const int size = m.rows * m.cols, mp = m.mp, np = m.np;
    double *part = reinterpret_cast<double *>(lds);
    double sum = 0.0;
#pragma unroll 4
    for (int i = threadIdx.x; i < size; i += 1024) sum += square_of<KIND>(g, m, i);
    for (int w = 32; w > 0; w >>= 1) sum += __shfl_xor(sum, w);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
    __syncthreads();
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < 16; ++w) sum += part[w];
    __syncthreads();
    const double scale = (double)m.sx / (sqrt(sum) + g.eps);
    _Float16 *X = lds, *XT = X + 2 * mp * np, *A = XT + 2 * mp * np, *B = A + 2 * mp * mp;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rows = mp / 16, columns = np / 16;
    // an element at a time, along the caller's rows
    const int slow = m.tall ? np : mp, fast = m.tall ? mp : np;
    for (int f = lane; f < fast; f += 64) {
#pragma unroll 4
        for (int r = wave; r < slow; r += 16) {
            const int i = m.tall ? f : r, j = m.tall ? r : f;
            const float x = i < m.m && j < m.n ? (float)((double)source<KIND>(g, m, r * m.cols + f) * scale) : 0.0f;
            const _Float16 hi = (_Float16)x, lo = (_Float16)(x - (float)hi);
            _Float16 *p = X + square_at(mp, i, j) + piece_in(i & 15, (j & 15) >> 2) + (j & 3);
            p[0] = hi;
            p[512] = lo;
            p = XT + square_at(np, j, i) + piece_in(j & 15, (i & 15) >> 2) + (i & 3);
            p[0] = hi;
            p[512] = lo;
        }
    }
    __syncthreads();
    const int at = piece_in(lane & 15, lane >> 4);
    const bool few = SOME_FEW && m.m <= FEW;
    const int high = few ? 1 : rows;   // squares of X that are not of zeros
    for (int s = 0; s < steps; ++s) {
        if (few) {   // one square, shared by four wavefronts over B's 4 KiB; the others are zeros
            f32x4 *sums = reinterpret_cast<f32x4 *>(B);
            if (wave < 4) sums[wave * 64 + lane] = square_sum(true, X, mp, 0, X, mp, 0, np / 32, wave, 4);
            __syncthreads();
            if (wave < 3) {
                const f32x4 sum = (sums[lane] + sums[64 + lane]) + (sums[128 + lane] + sums[192 + lane]);
                store_both(A, mp, wave == 1 ? A : nullptr, mp, wave > 1 ? 16 : 0, wave > 0 ? 16 : 0, wave == 0 ? sum * m.gram : f32x4{});
            }
        } else {
            for (int t = wave; t < rows * (rows + 1) / 2; t += 16) {
                int bi, bj;
                above_diagonal(t, bi, bj);
                store_both(A, mp, bi == bj ? nullptr : A, mp, bi * 16, bj * 16, square_sum(false, X, mp, bi, X, mp, bj, np / 32) * m.gram);
            }
        }
        __syncthreads();
        for (int t = wave; t < rows * (rows + 1) / 2; t += 16) {
            int bi, bj;
            above_diagonal(t, bi, bj);
            Piece a;
            a.load(A + square_at(mp, bj * 16, bi * 16) + at);
            store_both(B, mp, bi == bj ? nullptr : B, mp, bi * 16, bj * 16, QB * a.value() + square_sum(few, A, mp, bi, A, mp, bj, mp / 32) * m.square);
        }
        __syncthreads();
        f32x4 v[WHOLE_MOST];
#pragma unroll
        for (int i = 0; i < WHOLE_MOST; ++i) {
            const int t = wave + 16 * i, bi = t % high, bj = t / high;
            if (t >= high * columns) continue;
            Piece x;
            x.load(XT + square_at(np, bj * 16, bi * 16) + at);
            v[i] = QA * x.value() + square_sum(few, B, mp, bi, XT, np, bj, mp / 32) * m.update;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WHOLE_MOST; ++i) {
            const int t = wave + 16 * i, bi = t % high, bj = t / high;
            if (t >= high * columns) continue;
            if (s == steps - 1) give<KIND>(g, m, bi * 16, bj * 16, v[i]);
            else store_both(XT, np, X, mp, bi * 16, bj * 16, v[i]);
        }
        __syncthreads();
    }
}

inline int pad(int x, int to = 64) { return (x + to - 1) / to * to; }

// Whether one workgroup takes every matrix of a group, and the LDS for it.
template <class S>
bool is_whole(const S *matrices, int count, size_t &lds) {
    lds = 128;   // (the partial sums of squares)
    for (int k = 0; k < count; ++k) {
        const int mp = pad(std::min(matrices[k].rows, matrices[k].cols), 32), np = pad(std::max(matrices[k].rows, matrices[k].cols), 32);
        lds = std::max(lds, whole_lds(mp, np));
        if (whole_lds(mp, np) > WHOLE_LDS || mp / 16 * (np / 16) > 16 * WHOLE_MOST) return false;
    }
    return true;
}

// bytes of one matrix's planes and sums
size_t matrix_bytes(int rows, int cols) {
    const size_t mp = pad(std::min(rows, cols)), np = pad(std::max(rows, cols));
    return sizeof(_Float16) * (6 * mp * np + 4 * mp * mp) + sizeof(double) * MOST_SUMS;
}

template <class S>
size_t group_bytes(const S *matrices, int count) {
    size_t lds, bytes = GROUP_BYTES;
    if (is_whole(matrices, count, lds)) return 0;
    for (int k = 0; k < count; ++k) bytes += matrix_bytes(matrices[k].rows, matrices[k].cols);
    return bytes;
}
// How many of these a launch takes.
template <class S>
int group_of(const S *matrices, int left) {
    size_t bytes = 0;
    int k = 0;
    for (; k < std::min(MOST, left); ++k) {
        bytes += matrix_bytes(matrices[k].rows, matrices[k].cols);
        if (k > 0 && bytes > GROUP_ROOM) break;
    }
    return k;
}
// Of `count` alike: how many a launch takes, and their workspace.  256 of 64 x 64 in one launch 21 us, sixteen at a time 319; 64 of
// 256 x 256 255 and 397.
int batch_of(int count, int rows, int cols) {
    Mat m = {};
    size_t lds;
    m.rows = rows;
    m.cols = cols;
    const size_t room = is_whole(&m, 1, lds) ? 1 << 20 : std::max<size_t>(1, BATCH_BYTES / matrix_bytes(rows, cols));
    return (int)std::min<size_t>(count, room);
}
size_t batch_bytes(int count, int rows, int cols) {
    Mat m = {};
    size_t lds;
    m.rows = rows;
    m.cols = cols;
    return is_whole(&m, 1, lds) ? 0 : GROUP_BYTES + batch_of(count, rows, cols) * matrix_bytes(rows, cols);
}

// Sides of the tiles of a group's symmetric products, or of its updates: those of the least time by what products of one to sixteen
// matrices of 256 to 2048 took, in us, K of the contracted index long (256 CUs; one workgroup per CU at 96 and 128):
//   32: 4.5 + 11.5e-6 tiles K    64: 5.5 + 0.0072 K rounds, with two sets 5.5 + K (0.0036 + 0.0036 share)
//   96: 7 + K (0.007 + 0.0062 share), 7 + 0.0155 K rounds in more than one    128: 7 + K rounds (0.012 + 0.0095 share)
// where share of the CUs have one; more of them get in each other's way at the caches.  Symmetric / update at 32, 64, 96, 128:
//   256: 4 / 5, 6 / 7, 7 / 10, 9 / 11    1024: 10 / 16, 10 / 13, 14 / 17, 19 / 21    2048: 66 / 96, 48 / 66, 34 / 70, 42 / 50
int tile_of(const mrl_ctx *ctx, const Group &g, int described, int copies, bool symmetric) {
    int best = 0;
    double least = 0.0;
    for (int tile : {32, 64, 96, 128}) {
        double tiles = 0.0, work = 0.0;
        for (int k = 0; k < described; ++k) {
            const double a = (g.mat[k].mp + tile - 1) / tile, b = (g.mat[k].np + tile - 1) / tile;
            const double own = copies * (symmetric ? a * (a + 1) / 2 : a * b);
            tiles += own;
            work += own * (symmetric ? 0.5 * (g.mat[k].mp + g.mat[k].np) : g.mat[k].mp);
        }
        const double K = work / tiles, per_cu = tiles / ctx->n_cus, rounds = std::ceil(per_cu), share = std::min(1.0, per_cu);
        const double time = tile == 32   ? 4.5 + 11.5e-6 * 256 * per_cu * K
                            : tile == 64 ? 5.5 + K * (rounds > 1.0 || K <= TWO_SETS ? 0.0072 * rounds : 0.0036 + 0.0036 * share)
                            : tile == 96 ? 7.0 + K * (rounds > 1.0 ? 0.0155 * rounds : 0.007 + 0.0062 * share)
                                         : 7.0 + K * rounds * (0.012 + 0.0095 * share);
        if (best == 0 || time < least) {
            least = time;
            best = tile;
        }
    }
    return best;
}

// sides, scales and a share of the workspace
void set_up(Mat &m, int to, size_t &used) {
    m.mp = pad(m.m, to);
    m.np = pad(m.n, to);
    m.sums = (int)std::min<long>(MOST_SUMS, ((long)m.m * m.n + CHUNK - 1) / CHUNK);
    m.sx = (float)std::ldexp(1.0, std::min(14, (int)std::lround(0.5 * std::log2((double)m.m * m.n))));
    const float sa = (float)std::ldexp(1.0, std::min(13, (int)std::lround(std::log2((double)m.m))));
    m.gram = sa / (m.sx * m.sx);
    m.square = QC / sa;
    m.update = 1.0f / sa;
    m.result = 1.0f / m.sx;
    auto take = [&](size_t bytes) {
        const size_t at = used;
        used += bytes;
        return at;
    };
    const size_t X = sizeof(_Float16) * 2 * m.mp * (size_t)m.np, A = sizeof(_Float16) * 2 * m.mp * (size_t)m.mp;
    m.partial = take(sizeof(double) * MOST_SUMS);
    m.x = take(X);
    m.xt = take(X);
    m.xt1 = take(X);
    m.a = take(A);
    m.b = take(A);
}
void sides(Mat &m, int rows, int cols) {
    m.rows = rows;
    m.cols = cols;
    m.tall = rows > cols;
    m.m = std::min(rows, cols);
    m.n = std::max(rows, cols);
}

template <int STAGE, int KIND>
void product(const mrl_ctx *ctx, const Group &g, const Group *kept, int tiles, int from, int last) {
    const int tile = STAGE == UPDATE ? g.update_tile : g.sym_tile;
    int K = 0;   // the longest contracted index
    for (int k = 0; k < (KIND == MUON ? g.count : 1); ++k) K = std::max(K, STAGE == GRAM ? g.mat[k].np : g.mat[k].mp);
    auto launch = [&](auto kernel, size_t lds, int threads = 256) {
        hipLaunchKernelGGL(kernel, dim3(tiles), dim3(threads), lds, ctx->stream, kept, g.count, tiles, from, last);
    };
    if (tile == 128) launch(product_kernel<STAGE, KIND, 4, 1>, RING_BYTES<4, 1>, 64 * WAVES<4>);
    else if (tile == 96) launch(product_kernel<STAGE, KIND, 3, 2>, RING_BYTES<3, 2>, 512);
    else if (tile == 64 && tiles <= ctx->n_cus && K > TWO_SETS) launch(product_kernel<STAGE, KIND, 2, 2>, RING_BYTES<2, 2>, 512);
    else if (tile == 64) launch(product_kernel<STAGE, KIND, 2, 1>, RING_BYTES<2, 1>);
    else if (STAGE == GRAM && K > 32 * STRETCH) launch(small_product_kernel<STAGE, KIND, STAGE == GRAM>, 0);   // (what the others contract is short in tiles of 32)
    else launch(small_product_kernel<STAGE, KIND, false>, 0);
}

template <int KIND>
void run(const mrl_ctx *ctx, Group &g, int steps, void *workspace) {
    size_t used = GROUP_BYTES;
    Group *kept = (Group *)workspace;
    size_t lds;
    const int described = KIND == MUON ? g.count : 1, copies = KIND == MUON ? 1 : g.count;
    const bool whole = is_whole(g.mat, described, lds);
    const int threads = whole ? 1024 : 256;
    int sums = 1;
    for (int k = 0; k < described; ++k) {
        set_up(g.mat[k], whole ? 32 : 64, used);   // (a whole group's planes are in LDS: there is no workspace)
        sums = std::max(sums, g.mat[k].sums);
    }
    long rest = 0;
    for (int k = 0; k < g.rests; ++k) rest += g.rest[k].n;
    rest = std::min<long>(2048, (rest + threads - 1) / threads);
    if (whole) {
        bool some_few = false;
        for (int k = 0; k < described; ++k) some_few |= g.mat[k].m <= FEW;
        auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(g.count + rest), dim3(threads), lds, ctx->stream, g, steps); };
        if (some_few) launch(whole_kernel<KIND, true>);
        else launch(whole_kernel<KIND, false>);   // (a twentieth faster)
        return;
    }
    const bool few = KIND != MUON && g.mat[0].m <= FEW;   // (worked out in squares of 32 whatever the tile)
    g.sym_tile = few ? 32 : tile_of(ctx, g, described, copies, true);
    g.update_tile = few ? 32 : tile_of(ctx, g, described, copies, false);
    std::fill(g.begin_sym, g.begin_sym + MOST, INT_MAX);
    std::fill(g.begin_update, g.begin_update + MOST, INT_MAX);
    int load = 0, sym = 0, update = 0;   // squares of the largest matrix, tiles of all
    for (int k = 0; k < described; ++k) {
        const Mat &m = g.mat[k];
        const int a = (m.mp + g.sym_tile - 1) / g.sym_tile;
        load = std::max(load, m.mp / LOAD * (m.np / LOAD));
        g.begin_sym[k] = sym;
        sym += a * (a + 1) / 2;
        g.begin_update[k] = update;
        update += ((m.mp + g.update_tile - 1) / g.update_tile) * ((m.np + g.update_tile - 1) / g.update_tile);
    }
    g.alike_kept = used - GROUP_BYTES;
    g.alike_sym = sym;
    g.alike_update = update;
    sym *= copies;
    update *= copies;
    hipLaunchKernelGGL(sums_kernel<KIND>, dim3(std::max<long>(sums, rest), g.count + (rest > 0)), dim3(threads), 0, ctx->stream, g, kept);
    load = std::min(load, std::max(1, 8 * ctx->n_cus / g.count));
    hipLaunchKernelGGL(load_kernel<KIND>, dim3(load, g.count), dim3(256), 0, ctx->stream, kept);
    for (int s = 0; s < steps; ++s) {
        product<GRAM, KIND>(ctx, g, kept, sym, s & 1, 0);
        product<SQUARE, KIND>(ctx, g, kept, sym, s & 1, 0);
        product<UPDATE, KIND>(ctx, g, kept, update, s & 1, s == steps - 1);
    }
}

constexpr int MOST_SIDE = 1 << 15;   // rows and columns: tiles and elements are counted in 32 bits, entries of X stay in fp16's range

int check_matrix(const char *who, int rows, int cols) {
    MRL_CHECK_ARG(rows >= 1 && cols >= 1 && rows <= MOST_SIDE && cols <= MOST_SIDE, "%s: a matrix of %d x %d: sides of 1 to %d expected", who,
                  rows, cols, MOST_SIDE);
    return MRL_OK;
}

// matrices 0 .. count - 1 are in order and apart, inside n parameters
int check_matrices(const char *who, int count, const mrl_matrix *matrices, int64_t n) {
    MRL_CHECK_ARG(count >= 0 && (count == 0 || matrices), "%s: %d matrices at NULL", who, count);
    int64_t at = 0;
    for (int k = 0; k < count; ++k) {
        const mrl_matrix &m = matrices[k];
        const int rc = check_matrix(who, m.rows, m.cols);
        if (rc != MRL_OK) return rc;
        MRL_CHECK_ARG(m.offset >= at && m.offset <= n && (int64_t)m.rows * m.cols <= n - m.offset,
                      "%s: matrix %d (%d x %d at %lld) overlaps the one before or ends behind the %lld parameters", who, k, m.rows, m.cols,
                      (long long)m.offset, (long long)n);
        at = m.offset + (int64_t)m.rows * m.cols;
    }
    return MRL_OK;
}

// eps where zeros have a quotient in 64 bits.  A norm that is not 0 is 2^-149 or more: what is added here is far below its last bit.
double norm_eps(double eps) { return eps > 0.0 ? std::max(eps, 0x1p-900) : eps; }

int check_workspace(const char *who, const void *ws, uint64_t have, uint64_t need) {
    MRL_CHECK_ARG(need == 0 || (ws && have >= need), "%s: the workspace holds %llu bytes, need %llu", who, (unsigned long long)(ws ? have : 0),
                  (unsigned long long)need);
    MRL_CHECK_ARG(reinterpret_cast<uintptr_t>(ws) % 16 == 0, "%s: the workspace must be 16-byte aligned", who);
    return MRL_OK;
}

}  // namespace
}  // namespace mrl

extern "C" {

int mrl_orthogonalize_workspace(int count, int rows, int cols, uint64_t *bytes) {
    const char *who = "mrl_orthogonalize_workspace";
    MRL_CHECK_ARG(bytes && count >= 0, "%s: bad arguments", who);
    const int rc = mrl::check_matrix(who, rows, cols);
    if (rc != MRL_OK) return rc;
    *bytes = mrl::batch_bytes(count, rows, cols);
    return MRL_OK;
}

int mrl_orthogonalize(mrl_ctx *ctx, int dtype, int count, int rows, int cols, const void *in, void *out, int steps, double eps,
                      void *workspace, uint64_t workspace_bytes) {
    const char *who = "mrl_orthogonalize";
    MRL_CHECK_ARG(ctx, "%s: ctx is NULL", who);
    MRL_CHECK_ARG(dtype == MRL_F32 || dtype == MRL_BF16, "%s: unknown element type %d", who, dtype);
    MRL_CHECK_ARG(count >= 0, "%s: negative count", who);
    MRL_CHECK_ARG(steps >= 1 && steps <= 64 && eps >= 0.0, "%s: 1 to 64 steps and eps >= 0 expected", who);
    int rc = mrl::check_matrix(who, rows, cols);
    if (rc != MRL_OK || count == 0) return rc;
    MRL_CHECK_ARG(in && out, "%s: NULL buffer", who);
    const uint64_t need = mrl::batch_bytes(count, rows, cols);
    rc = mrl::check_workspace(who, workspace, workspace_bytes, need);
    if (rc != MRL_OK) return rc;
    const size_t one = (size_t)rows * cols * (dtype == MRL_F32 ? 4 : 2);
    rc = mrl::check_apart(who, {{"out", out, (int64_t)(count * one)}, {"the workspace", workspace, (int64_t)need}}, {{"in", in == out ? nullptr : in, (int64_t)(count * one)}});
    if (rc != MRL_OK) return rc;
    mrl::OnDevice on(ctx);
    const int most = mrl::batch_of(count, rows, cols);
    for (long done = 0; done < count; done += most) {
        mrl::Group g = {};
        g.eps = mrl::norm_eps(eps);
        g.count = (int)std::min<long>(most, count - done);
        g.alike_in = one;
        mrl::sides(g.mat[0], rows, cols);
        g.mat[0].in = (const char *)in + done * one;
        g.mat[0].out = (char *)out + done * one;
        if (dtype == MRL_F32) mrl::run<mrl::F32>(ctx, g, steps, workspace);
        else mrl::run<mrl::BF16>(ctx, g, steps, workspace);
        MRL_CHECK_LAUNCH();
    }
    return MRL_OK;
}

int mrl_muon_workspace(int n_matrices, const mrl_matrix *matrices, uint64_t *bytes) {
    const char *who = "mrl_muon_workspace";
    MRL_CHECK_ARG(bytes, "%s: NULL result", who);
    const int rc = mrl::check_matrices(who, n_matrices, matrices, INT64_MAX);
    if (rc != MRL_OK) return rc;
    *bytes = 0;
    for (int done = 0, group; done < n_matrices; done += group) {
        group = mrl::group_of(matrices + done, n_matrices - done);
        *bytes = std::max<uint64_t>(*bytes, mrl::group_bytes(matrices + done, group));
    }
    return MRL_OK;
}

int mrl_muon_step(mrl_ctx *ctx, float *params, const float *grads, float *state, int64_t n, int n_matrices, const mrl_matrix *matrices,
                  int t, double lr, double momentum, int nesterov, double weight_decay, int steps, double eps, double adam_lr,
                  double beta1, double beta2, double adam_eps, void *workspace, uint64_t workspace_bytes) {
    const char *who = "mrl_muon_step";
    MRL_CHECK_ARG(ctx, "%s: ctx is NULL", who);
    MRL_CHECK_ARG(n >= 0 && n < 1LL << 38 && t >= 1, "%s: need 0 <= n < 2^38 and step count t >= 1", who);
    MRL_CHECK_ARG(steps >= 1 && steps <= 64 && eps >= 0.0, "%s: 1 to 64 steps and eps >= 0 expected", who);
    int rc = mrl::check_matrices(who, n_matrices, matrices, n);
    if (rc != MRL_OK || n == 0) return rc;
    MRL_CHECK_ARG(params && grads && state, "%s: NULL buffer", who);
    MRL_CHECK_ARG(reinterpret_cast<uintptr_t>(state) % 8 == 0, "%s: the state must be 8-byte aligned", who);
    uint64_t need = 0;
    rc = mrl_muon_workspace(n_matrices, matrices, &need);
    if (rc == MRL_OK) rc = mrl::check_workspace(who, workspace, workspace_bytes, need);
    if (rc == MRL_OK)
        rc = mrl::check_apart(who, {{"params", params, 4 * n}, {"state", state, 8 * n}, {"the workspace", workspace, (int64_t)need}}, {{"grads", grads, 4 * n}});
    if (rc != MRL_OK) return rc;
    mrl::OnDevice on(ctx);
    int64_t at = 0;
    int done = 0;
    do {
        mrl::Group g = {};
        g.eps = mrl::norm_eps(eps);
        g.mu = (float)momentum;
        g.nesterov = nesterov != 0;
        g.keep = (float)(1.0 - lr * weight_decay);
        g.lr = (float)adam_lr;
        g.beta1 = (float)beta1; g.beta2 = (float)beta2; g.omb1 = (float)(1.0 - beta1); g.omb2 = (float)(1.0 - beta2);
        g.adam_eps = (float)adam_eps;
        g.bc1 = (float)(1.0 - pow(beta1, (double)t)); g.bc2 = (float)(1.0 - pow(beta2, (double)t));
        g.count = mrl::group_of(matrices + done, n_matrices - done);
        auto rest = [&](int64_t to) {
            if (to > at) g.rest[g.rests++] = {params + at, grads + at, reinterpret_cast<float2 *>(state) + at, (long)(to - at)};
        };
        for (int k = 0; k < g.count; ++k) {
            const mrl_matrix &x = matrices[done + k];
            mrl::Mat &m = g.mat[k];
            rest(x.offset);
            mrl::sides(m, x.rows, x.cols);
            m.in = grads + x.offset;
            m.out = params + x.offset;
            m.momentum = state + 2 * x.offset;
            m.factor = (float)(lr * std::sqrt(std::max(1.0, (double)x.cols / x.rows)));
            at = x.offset + (int64_t)x.rows * x.cols;
        }
        done += g.count;
        if (done >= n_matrices) rest(n);
        mrl::run<mrl::MUON>(ctx, g, steps, workspace);
        MRL_CHECK_LAUNCH();
    } while (done < n_matrices);
    return MRL_OK;
}

}  // extern "C"
