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
// The sides are padded with zeros to whole tiles, which the products keep zero.
#include <cmath>
#include "mrl_host.hpp"
#include "mrl_device.hpp"

namespace mrl {
namespace {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float QA = 3.4445f, QB = -4.7750f, QC = 2.0315f;
constexpr int MOST = 16;        // matrices of a launch
constexpr int LOAD = 32;        // sides of what a workgroup of the second launch takes
constexpr int CHUNK = 4096;     // elements that a workgroup of the first launch takes at a time
constexpr int MOST_SUMS = 256;  // partial sums of squares per matrix

struct bf16_t { unsigned short bits; };

struct Mat {
    const void *in;
    void *out;
    float *momentum;
    int rows, cols, m, n, mp, np;   // the caller's sides; the shorter and the longer one, and both padded
    int tall;                       // rows > cols: X is the transpose
    int sums, begin_sums, begin_load, begin_sym, begin_update;   // workgroups of each launch
    float sx, sa;                   // what X and what A, B are stored times
    float factor;                   // of the update
    _Float16 *x, *xt[2], *a, *b;
    double *partial;
};
struct Rest { float *p; const float *g; float2 *state; long n; int begin; };   // parameters that Adam updates
struct Group {
    int count, rests;
    int tile;               // sides of the products' tiles; every matrix's sides are padded to it
    int total_sums;
    Mat mat[MOST];
    Rest rest[MOST + 1];
    double eps;
    float mu, keep;         // momentum; 1 - lr weight_decay
    int nesterov;
    float lr, beta1, beta2, omb1, omb2, adam_eps, bc1, bc2;
};
static_assert(sizeof(Group) <= 3584, "kernel arguments");

enum { F32 = 0, BF16 = 1, MUON = 2 };   // what a matrix is read from and written to

template <int KIND>
MRL_DEV float source(const Group &g, const Mat &m, size_t i) {
    if (KIND == BF16) return __uint_as_float((unsigned)((const unsigned short *)m.in)[i] << 16);
    const float x = ((const float *)m.in)[i];
    if (KIND == F32) return x;
    const float v = m.momentum[i];   // (already this step's)
    return g.nesterov ? fmaf(g.mu, v, x) : v;
}

// Sums of squares of every matrix, in 64 bits and a fixed order; with MUON also the new momentum, and Adam on the other parameters.
template <int KIND>
__global__ __launch_bounds__(256) void sums_kernel(Group g) {
    if (KIND == MUON && (int)blockIdx.x >= g.total_sums) {
        const int block = blockIdx.x - g.total_sums;
        int k = 0;
        while (k + 1 < g.rests && block >= g.rest[k + 1].begin) ++k;
        const Rest &r = g.rest[k];
        const long i = (long)(block - r.begin) * 256 + threadIdx.x;
        if (i < r.n) adam_one(r.p[i], r.g[i], r.state[i], g.lr, g.beta1, g.beta2, g.omb1, g.omb2, g.adam_eps, g.bc1, g.bc2);
        return;
    }
    int k = 0;
    while (k + 1 < g.count && (int)blockIdx.x >= g.mat[k + 1].begin_sums) ++k;
    const Mat &m = g.mat[k];
    const int block = blockIdx.x - m.begin_sums;
    const size_t size = (size_t)m.rows * m.cols;
    double sum = 0.0;
    for (size_t i = (size_t)block * 256 + threadIdx.x; i < size; i += (size_t)m.sums * 256) {
        if (KIND == MUON) m.momentum[i] = fmaf(g.mu, m.momentum[i], ((const float *)m.in)[i]);
        const float x = source<KIND>(g, m, i);
        sum += (double)x * (double)x;
    }
    __shared__ double part[256];
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) part[threadIdx.x] += part[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) m.partial[block] = part[0];
}

// hi and lo pieces of four neighbours along the contracted index k (a multiple of 4) of row `row`
MRL_DEV size_t piece_at(int blocks, int row, int k) {
    return ((size_t)(row >> 4) * blocks + (k >> 5)) * 1024 + (16 * ((k & 31) >> 3) + (row & 15)) * 8 + (k & 7);
}
MRL_DEV void put_piece(_Float16 *planes, int blocks, int row, int k, const f32x4 x) {
    const f16x4 hi = __builtin_convertvector(x, f16x4);
    const f16x4 lo = __builtin_convertvector(x - __builtin_convertvector(hi, f32x4), f16x4);
    _Float16 *p = planes + piece_at(blocks, row, k);
    *reinterpret_cast<f16x4 *>(p) = hi;
    *reinterpret_cast<f16x4 *>(p + 512) = lo;
}
MRL_DEV f32x4 get_piece(const _Float16 *planes, int blocks, int row, int k) {
    const _Float16 *p = planes + piece_at(blocks, row, k);
    return __builtin_convertvector(*reinterpret_cast<const f16x4 *>(p), f32x4) +
           __builtin_convertvector(*reinterpret_cast<const f16x4 *>(p + 512), f32x4);
}

// X and its transpose in pieces, a tile per workgroup, through LDS: read along the caller's rows, written along both sides.
template <int KIND>
__global__ __launch_bounds__(256) void load_kernel(Group g) {
    __shared__ double part[256];
    __shared__ float tile[LOAD][LOAD + 1];
    int k = 0;
    while (k + 1 < g.count && (int)blockIdx.x >= g.mat[k + 1].begin_load) ++k;
    const Mat &m = g.mat[k];
    const int block = blockIdx.x - m.begin_load, across = m.np / LOAD, i0 = block / across * LOAD, j0 = block % across * LOAD;
    part[threadIdx.x] = (int)threadIdx.x < m.sums ? m.partial[threadIdx.x] : 0.0;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if ((int)threadIdx.x < w) part[threadIdx.x] += part[threadIdx.x + w];
        __syncthreads();
    }
    const double scale = (double)m.sx / (sqrt(part[0]) + g.eps);
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
        put_piece(m.x, m.np / 32, i0 + r, j0 + c, f32x4{tile[r][c], tile[r][c + 1], tile[r][c + 2], tile[r][c + 3]});
        put_piece(m.xt[0], m.mp / 32, j0 + r, i0 + c, f32x4{tile[c][r], tile[c + 1][r], tile[c + 2][r], tile[c + 3][r]});
    }
}

// 4 x 4 values of four neighbouring lanes, transposed: v[c] of lane s becomes v[s] of lane c.
MRL_DEV f32x4 quad_transpose(f32x4 v) {
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
    auto swap1 = [](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0xB1, 0xF, 0xF, true)); };
    auto swap2 = [](float x) { return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), 0x4E, 0xF, 0xF, true)); };
#pragma unroll
    for (int p = 0; p < 4; p += 2) {
        const float other = swap1(odd ? v[p] : v[p + 1]);
        v[p] = odd ? other : v[p];
        v[p + 1] = odd ? v[p + 1] : other;
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const float other = swap2(high ? v[p] : v[p + 2]);
        v[p] = high ? other : v[p];
        v[p + 2] = high ? v[p + 2] : other;
    }
    return v;
}

enum { GRAM = 0, SQUARE = 1, UPDATE = 2 };

// Which tile of which matrix a workgroup works on.  Workgroups go to the eight XCDs in turn; each XCD gets a run of tiles that
// share operands, so that its L2 is read more often than what is behind it.
template <int STAGE>
MRL_DEV const Mat &find_tile(const Group &g, int total, int &bi, int &bj) {
    const int xcd = blockIdx.x & 7, each = total >> 3, more = total & 7;
    const int id = xcd * each + min(xcd, more) + (blockIdx.x >> 3);
    int k = 0;
    if (STAGE == UPDATE) {
        while (k + 1 < g.count && id >= g.mat[k + 1].begin_update) ++k;
        const Mat &m = g.mat[k];
        const int block = id - m.begin_update, rows = m.mp / g.tile, panel = block / (4 * rows), in = block - panel * 4 * rows;
        const int width = min(4, m.np / g.tile - 4 * panel);   // panels of four columns, row by row
        bi = in / width;
        bj = 4 * panel + in - bi * width;
        return m;
    }
    while (k + 1 < g.count && id >= g.mat[k + 1].begin_sym) ++k;
    const Mat &m = g.mat[k];
    int block = id - m.begin_sym;
    bj = (int)((sqrtf(8.0f * block + 1.0f) - 1.0f) * 0.5f);   // column bj has tiles 0 .. bj
    while (bj * (bj + 1) / 2 > block) --bj;
    while ((bj + 1) * (bj + 2) / 2 <= block) ++bj;
    bi = block - bj * (bj + 1) / 2;
    return m;
}

// What becomes of four sums: rows i .. i + 3 of column j, of a lane with column j % 16.
template <int STAGE, int KIND>
MRL_DEV void finish(const Group &g, const Mat &m, int from, int last, bool diagonal, int i, int j, f32x4 v) {
    const int it = i + (j & 3), jt = j & ~3;   // transposed: row it, columns jt .. jt + 3
    if (STAGE == UPDATE) {
        const f32x4 x = get_piece(m.xt[from], m.mp / 32, j, i);
        v = QA * x + v * (1.0f / m.sa);
        if (!last) {
            put_piece(m.xt[from ^ 1], m.mp / 32, j, i, v);
            put_piece(m.x, m.np / 32, it, jt, quad_transpose(v));
            return;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (i + e >= m.m || j >= m.n) continue;
            const size_t at = m.tall ? (size_t)j * m.m + (i + e) : (size_t)(i + e) * m.n + j;
            const float o = v[e] * (1.0f / m.sx);
            if (KIND == BF16) {
                ((unsigned short *)m.out)[at] = __builtin_bit_cast(unsigned short, (__bf16)o);
            } else if (KIND == F32) {
                ((float *)m.out)[at] = o;
            } else {
                float *w = (float *)m.out + at;
                *w = fmaf(-m.factor, o, *w * g.keep);
            }
        }
    } else {
        _Float16 *to = STAGE == GRAM ? m.a : m.b;
        if (STAGE == GRAM) v = v * (m.sa / (m.sx * m.sx));
        else v = QB * get_piece(m.a, m.mp / 32, j, i) + v * (QC / m.sa);
        put_piece(to, m.mp / 32, j, i, v);
        if (!diagonal) put_piece(to, m.mp / 32, it, jt, quad_transpose(v));
    }
}

template <int F>
MRL_DEV void multiply(const f16x8 (&ph)[F], const f16x8 (&pl)[F], const f16x8 (&qh)[F], const f16x8 (&ql)[F], f32x4 (&acc)[F][F]) {
#pragma unroll
    for (int fi = 0; fi < F; ++fi)
#pragma unroll
        for (int fj = 0; fj < F; ++fj) acc[fi][fj] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl[fi], qh[fj], acc[fi][fj], 0, 0, 0);
#pragma unroll
    for (int fi = 0; fi < F; ++fi)
#pragma unroll
        for (int fj = 0; fj < F; ++fj) acc[fi][fj] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[fi], ql[fj], acc[fi][fj], 0, 0, 0);
#pragma unroll
    for (int fi = 0; fi < F; ++fi)
#pragma unroll
        for (int fj = 0; fj < F; ++fj) acc[fi][fj] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[fi], qh[fj], acc[fi][fj], 0, 0, 0);
}

template <int STAGE>
MRL_DEV void operands(const Mat &m, int from, const _Float16 *&P, const _Float16 *&Q, int &blocks) {
    P = STAGE == GRAM ? m.x : STAGE == SQUARE ? m.a : m.b;
    Q = STAGE == GRAM ? m.x : STAGE == SQUARE ? m.a : m.xt[from];
    blocks = (STAGE == GRAM ? m.np : m.mp) / 32;
}

// One product, a tile of 32 F x 32 F per workgroup.  GRAM: A = X X^T; SQUARE: B = b A + c A A; both symmetric, so only tiles on and
// above the diagonal are worked out and written to both sides.  UPDATE: X <- a X + B X, `last` to the caller.
// Four wavefronts share the tile, 16 F x 16 F each, and KG such sets share the contracted index, 32 of it each at a time, so that
// a SIMD has KG wavefronts to take turns.  Operands go from memory to LDS past the registers, the next 32 KG while these are
// multiplied.  In the end the sets exchange sums through LDS and each finishes a part of the tile.
template <int STAGE, int KIND, int F, int KG>
__global__ __launch_bounds__(256 * KG) __attribute__((amdgpu_waves_per_eu(F == 4 ? 2 : 4))) void product_kernel(Group g, int total, int from, int last) {
    constexpr int SIDE = 2 * F;                        // fragments of 16 along a side
    constexpr int OPERAND = SIDE * KG * 1024;          // halves of one operand of a stage: [fragment][set][hi, lo][512]
    extern __shared__ _Float16 lds[];
    int bi, bj;
    const Mat &m = find_tile<STAGE>(g, total, bi, bj);
    const _Float16 *P, *Q;
    int blocks;
    operands<STAGE>(m, from, P, Q, blocks);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), set = wave >> 2, part = wave & 3;
    const int stages = blocks / KG;   // (whole: the sides are padded to the tile)
    // A stage of a fragment, KG times hi and lo, is one run of memory and of LDS; a wavefront brings in EACH fragments of an operand.
    constexpr int EACH = SIDE / (2 * KG);
    const int operand = wave / (2 * KG), first = wave % (2 * KG) * EACH;
    const _Float16 *src = (operand ? Q + (size_t)(bj * SIDE + first) * blocks * 1024 : P + (size_t)(bi * SIDE + first) * blocks * 1024) + lane * 8;
    _Float16 *to = lds + operand * OPERAND + first * KG * 1024;
    auto stage_in = [&](int stage) {
#pragma unroll
        for (int e = 0; e < EACH * 2 * KG; ++e)
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)(src + ((size_t)(e / (2 * KG)) * blocks + (size_t)stage * KG) * 1024 + e % (2 * KG) * 512),
                (__attribute__((address_space(3))) void *)(to + (stage & 1) * 2 * OPERAND + e * 512), 16, 0, 0);
    };
    f32x4 acc[F][F] = {};
    stage_in(0);
    for (int s = 0; s < stages; ++s) {
        __syncthreads();   // this stage is in LDS, and nobody reads the buffer of the next one any more
        if (s + 1 < stages) stage_in(s + 1);
        const _Float16 *p = lds + (s & 1) * 2 * OPERAND + ((part >> 1) * F * KG + set) * 1024 + lane * 8;
        const _Float16 *q = lds + (s & 1) * 2 * OPERAND + OPERAND + ((part & 1) * F * KG + set) * 1024 + lane * 8;
        f16x8 ph[F], pl[F], qh[F], ql[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {
            pl[f] = *reinterpret_cast<const f16x8 *>(p + f * KG * 1024 + 512);
            qh[f] = *reinterpret_cast<const f16x8 *>(q + f * KG * 1024);
        }
#pragma unroll
        for (int f = 0; f < F; ++f) {
            ph[f] = *reinterpret_cast<const f16x8 *>(p + f * KG * 1024);
            ql[f] = *reinterpret_cast<const f16x8 *>(q + f * KG * 1024 + 512);
        }
        multiply<F>(ph, pl, qh, ql, acc);
    }
    const int i0 = (bi * SIDE + (part >> 1) * F) * 16 + 4 * (lane >> 4), j0 = (bj * SIDE + (part & 1) * F) * 16 + (lane & 15);
    // set s finishes the fragments whose number is s modulo KG
    {
        f32x4 *sums = reinterpret_cast<f32x4 *>(lds);   // [set that finishes][set that has them][part][fragment / KG][lane]
        constexpr int SHARE = F * F / KG;
        __syncthreads();
#pragma unroll
        for (int f = 0; f < F * F; ++f)
            if (f % KG != set) sums[(((f % KG) * KG + set) * 4 + part) * SHARE * 64 + (f / KG) * 64 + lane] = acc[f / F][f % F];
        __syncthreads();
#pragma unroll
        for (int f = 0; f < F * F; ++f) {
            if (f % KG != set) continue;
            f32x4 v = acc[f / F][f % F];
#pragma unroll
            for (int other = 1; other < KG; ++other)
                v += sums[((set * KG + (set + other) % KG) * 4 + part) * SHARE * 64 + (f / KG) * 64 + lane];
            finish<STAGE, KIND>(g, m, from, last, bi == bj, i0 + 16 * (f / F), j0 + 16 * (f % F), v);
        }
    }
}

// The same for small matrices, where a launch is shorter than the way of a stage through memory and LDS and back: a tile of 32 x 32
// per workgroup, the contracted index shared by its four wavefronts, operands straight to registers.
template <int STAGE, int KIND>
__global__ __launch_bounds__(256) void small_product_kernel(Group g, int total, int from, int last) {
    __shared__ f32x4 sums[4][4][64];   // [fragment][wavefront][lane]
    int bi, bj;
    const Mat &m = find_tile<STAGE>(g, total, bi, bj);
    const _Float16 *P, *Q;
    int blocks;
    operands<STAGE>(m, from, P, Q, blocks);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const _Float16 *p = P + (size_t)bi * 2 * blocks * 1024 + lane * 8, *q = Q + (size_t)bj * 2 * blocks * 1024 + lane * 8;
    f32x4 acc[2][2] = {};
#pragma unroll 2
    for (int kb = wave; kb < blocks; kb += 4) {
        f16x8 ph[2], pl[2], qh[2], ql[2];
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const _Float16 *pf = p + ((size_t)f * blocks + kb) * 1024, *qf = q + ((size_t)f * blocks + kb) * 1024;
            ph[f] = *reinterpret_cast<const f16x8 *>(pf);
            pl[f] = *reinterpret_cast<const f16x8 *>(pf + 512);
            qh[f] = *reinterpret_cast<const f16x8 *>(qf);
            ql[f] = *reinterpret_cast<const f16x8 *>(qf + 512);
        }
        multiply<2>(ph, pl, qh, ql, acc);
    }
#pragma unroll
    for (int f = 0; f < 4; ++f) sums[f][wave][lane] = acc[f >> 1][f & 1];
    __syncthreads();
    const f32x4 v = (sums[wave][0][lane] + sums[wave][1][lane]) + (sums[wave][2][lane] + sums[wave][3][lane]);
    finish<STAGE, KIND>(g, m, from, last, bi == bj, (bi * 2 + (wave >> 1)) * 16 + 4 * (lane >> 4), (bj * 2 + (wave & 1)) * 16 + (lane & 15), v);
}

inline int pad(int x, int tile) { return (x + tile - 1) / tile * tile; }

// bytes of one matrix's planes and sums
size_t matrix_bytes(int rows, int cols, int tile) {
    const size_t mp = pad(std::min(rows, cols), tile), np = pad(std::max(rows, cols), tile);
    return sizeof(_Float16) * (6 * mp * np + 4 * mp * mp) + sizeof(double) * MOST_SUMS;
}

// The tiles of a launch: the largest of which the products have enough to go round.
struct Sides { int rows, cols; };
template <class S>
int tile_of(const S *matrices, int count) {
    for (int tile : {128, 64}) {
        long tiles = 0;
        for (int k = 0; k < count; ++k) tiles += (long)(pad(matrices[k].rows, tile) / tile) * (pad(matrices[k].cols, tile) / tile);
        if (tiles >= (tile == 128 ? 128 : 64)) return tile;
    }
    return 32;
}
template <class S>
size_t group_bytes(const S *matrices, int count) {
    const int tile = tile_of(matrices, count);
    size_t bytes = 0;
    for (int k = 0; k < count; ++k) bytes += matrix_bytes(matrices[k].rows, matrices[k].cols, tile);
    return bytes;
}

// of `count` alike, in launches of MOST; the last launch's tiles may be smaller, and so their padding
size_t batch_bytes(int count, int rows, int cols) {
    Sides sides[MOST];
    std::fill(sides, sides + MOST, Sides{rows, cols});
    const size_t whole = count >= MOST ? group_bytes(sides, MOST) : 0;
    return std::max(whole, count % MOST ? group_bytes(sides, count % MOST) : (size_t)0);
}

// sides, scales and a share of the workspace
void set_up(Mat &m, int rows, int cols, int tile, char *&ws) {
    m.rows = rows;
    m.cols = cols;
    m.tall = rows > cols;
    m.m = std::min(rows, cols);
    m.n = std::max(rows, cols);
    m.mp = pad(m.m, tile);
    m.np = pad(m.n, tile);
    m.sums = (int)std::min<long>(MOST_SUMS, ((long)rows * cols + CHUNK - 1) / CHUNK);
    m.sx = (float)std::ldexp(1.0, std::min(14, (int)std::lround(0.5 * std::log2((double)m.m * m.n))));
    m.sa = (float)std::ldexp(1.0, std::min(13, (int)std::lround(std::log2((double)m.m))));
    auto planes = [&](size_t elements) {
        _Float16 *p = reinterpret_cast<_Float16 *>(ws);
        ws += sizeof(_Float16) * 2 * elements;
        return p;
    };
    m.partial = reinterpret_cast<double *>(ws);
    ws += sizeof(double) * MOST_SUMS;
    m.x = planes((size_t)m.mp * m.np);
    m.xt[0] = planes((size_t)m.mp * m.np);
    m.xt[1] = planes((size_t)m.mp * m.np);
    m.a = planes((size_t)m.mp * m.mp);
    m.b = planes((size_t)m.mp * m.mp);
}

template <int STAGE, int KIND>
void product(const mrl_ctx *ctx, const Group &g, int total, int from, int last) {
    auto launch = [&](auto kernel, int threads, size_t lds) {
        hipLaunchKernelGGL(kernel, dim3(total), dim3(threads), lds, ctx->stream, g, total, from, last);
    };
    if (g.tile == 128) launch(product_kernel<STAGE, KIND, 4, 2>, 512, 2 * 2 * 8 * 2 * 2048);
    else if (g.tile == 64) launch(product_kernel<STAGE, KIND, 2, 2>, 512, 2 * 2 * 4 * 2 * 2048);
    else launch(small_product_kernel<STAGE, KIND>, 256, 0);
}

template <int KIND>
void run(const mrl_ctx *ctx, Group &g, int steps) {
    int sums = 0, load = 0, sym = 0, update = 0;
    for (int k = 0; k < g.count; ++k) {
        Mat &m = g.mat[k];
        const int a = m.mp / g.tile, b = m.np / g.tile;
        m.begin_sums = sums; sums += m.sums;
        m.begin_load = load; load += (m.mp / LOAD) * (m.np / LOAD);
        m.begin_sym = sym; sym += a * (a + 1) / 2;
        m.begin_update = update; update += a * b;
    }
    g.total_sums = sums;
    int rest = 0;
    for (int k = 0; k < g.rests; ++k) {
        g.rest[k].begin = rest;
        rest += grid_for(g.rest[k].n, 256);
    }
    if (sums + rest > 0) hipLaunchKernelGGL(sums_kernel<KIND>, dim3(sums + rest), dim3(256), 0, ctx->stream, g);
    if (g.count == 0) return;
    hipLaunchKernelGGL(load_kernel<KIND>, dim3(load), dim3(256), 0, ctx->stream, g);
    for (int s = 0; s < steps; ++s) {
        product<GRAM, KIND>(ctx, g, sym, s & 1, 0);
        product<SQUARE, KIND>(ctx, g, sym, s & 1, 0);
        product<UPDATE, KIND>(ctx, g, update, s & 1, s == steps - 1);
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
    rc = mrl::check_workspace(who, workspace, workspace_bytes, mrl::batch_bytes(count, rows, cols));
    if (rc != MRL_OK) return rc;
    mrl::OnDevice on(ctx);
    const size_t one = (size_t)rows * cols * (dtype == MRL_F32 ? 4 : 2);
    for (int done = 0; done < count; done += mrl::MOST) {
        mrl::Group g = {};
        g.eps = eps;
        g.count = std::min(mrl::MOST, count - done);
        char *ws = (char *)workspace;
        mrl::Sides sides[mrl::MOST];
        std::fill(sides, sides + mrl::MOST, mrl::Sides{rows, cols});
        g.tile = mrl::tile_of(sides, g.count);
        for (int k = 0; k < g.count; ++k) {
            mrl::set_up(g.mat[k], rows, cols, g.tile, ws);
            g.mat[k].in = (const char *)in + (done + k) * one;
            g.mat[k].out = (char *)out + (done + k) * one;
        }
        if (dtype == MRL_F32) mrl::run<mrl::F32>(ctx, g, steps);
        else mrl::run<mrl::BF16>(ctx, g, steps);
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
    for (int done = 0; done < n_matrices; done += mrl::MOST) {
        *bytes = std::max<uint64_t>(*bytes, mrl::group_bytes(matrices + done, std::min(mrl::MOST, n_matrices - done)));
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
    if (rc != MRL_OK) return rc;
    mrl::OnDevice on(ctx);
    int64_t at = 0;
    int done = 0;
    do {
        mrl::Group g = {};
        g.eps = eps;
        g.mu = (float)momentum;
        g.nesterov = nesterov != 0;
        g.keep = (float)(1.0 - lr * weight_decay);
        g.lr = (float)adam_lr;
        g.beta1 = (float)beta1; g.beta2 = (float)beta2; g.omb1 = (float)(1.0 - beta1); g.omb2 = (float)(1.0 - beta2);
        g.adam_eps = (float)adam_eps;
        g.bc1 = (float)(1.0 - pow(beta1, (double)t)); g.bc2 = (float)(1.0 - pow(beta2, (double)t));
        g.count = std::min(mrl::MOST, n_matrices - done);
        g.tile = mrl::tile_of(matrices + done, g.count);
        char *ws = (char *)workspace;
        auto rest = [&](int64_t to) {
            if (to > at) g.rest[g.rests++] = {params + at, grads + at, reinterpret_cast<float2 *>(state) + at, (long)(to - at), 0};
        };
        for (int k = 0; k < g.count; ++k) {
            const mrl_matrix &x = matrices[done + k];
            mrl::Mat &m = g.mat[k];
            rest(x.offset);
            mrl::set_up(m, x.rows, x.cols, g.tile, ws);
            m.in = grads + x.offset;
            m.out = params + x.offset;
            m.momentum = state + 2 * x.offset;
            m.factor = (float)(lr * std::sqrt(std::max(1.0, (double)x.cols / x.rows)));
            at = x.offset + (int64_t)x.rows * x.cols;
        }
        done += g.count;
        if (done >= n_matrices) rest(n);
        mrl::run<mrl::MUON>(ctx, g, steps);
        MRL_CHECK_LAUNCH();
    } while (done < n_matrices);
    return MRL_OK;
}

}  // extern "C"
