// The gated delta rule backwards.  With the names of delta.hpp, dS1 the gradient of the state behind a tile, dO that of its outputs:
//   dU = P^T dO + L k dS1,   dX = (1 + A)^-T dU,   dv = b dX,
//   dA[i][j] = -dX[i] U[j] (j < i),   dP[i][j] = dO[i] U[j] (j <= i),
//   dq[i] = F[i] S0 dO[i] + sum_j dP[i][j] G[i][j] k[j],
//   dk[i] = -b[i] F[i] S0 dX[i] + sum_j b[i] dA[i][j] G[i][j] k[j]                                    (as the one that reads)
//         + L[i] dS1 U[i] + sum_j b[j] dA[j][i] G[j][i] k[j] + sum_j dP[j][i] G[j][i] q[j]            (as the one that is read),
//   dS0 = F[15] dS1 + sum_i F[i] (q[i] dO[i]^T - b[i] k[i] dX[i]^T),   drate[i] = (1 - b[i]) dX[i] U[i].
// The gradient of log a[t] is the sum of everything that a[t] scales: with M[i][j] = dA A + dP P, e[i] = q[i] dq[i] + k[i] dk[i] of the terms with
// S0, f[j] = k[j] dk[j] of that with dS1,
//   sum_{i >= t > j} M[i][j] + sum_{i >= t} e[i] + sum_{j < t} f[j] + F[15] S0 dS1,
// added up as it stands: every term has a[t] in it.  (Sums of row and column dots, of which this is a difference, lose it where a is small.)
// dgate = (1 - a) times that, 0 at a cut.
//
// The dots that the lengths need are those of the terms: of a row's pairs they are sums over M's parts,
//   q[i] dq[i] = q[i] (F[i] S0 dO[i]) + sum_j dP[i][j] P[i][j],   k[i] dk[i] = e's share + f[i] + sum_j dA[i][j] A[i][j] + sum_j (dA[j][i] A[j][i] + dP[j][i] P[j][i]),
// and drate's is -dA's diagonal.
//
// A first launch leaves the state ahead of every block of tiles in the workspace (mrl_delta.hip).  In the last a workgroup goes through the blocks
// of one head of one environment from the last to the first: it repeats a block's tiles forwards, keeping each tile's S0 and U in registers,
// and takes the tiles backwards.  A wavefront holds 16 columns of S0 and dS1; what contracts over the columns (dq, dk, dA, dP) is done by 16
// rows of the states per wavefront, which they pass through LDS.  A rollout in parts has the gradients of the states behind the parts worked out
// ahead of that (chain_kernel, and the launch that goes through the parts).
//
// 128 steps of 512 environments of 4 heads of 64 x 64 in fp32 take 503 us, 82 of them the first launch (reading and writing the rows once takes 105, the
// formulas' products at the rate of a large fp32 one 140).  Bound by what a tile's phases wait for each other: the matrix cores are busy a third of the time,
// other instructions a quarter; LDS has room for two workgroups of four wavefronts a CU (78 KB; one takes 755 us).  Memory is no part of it: 489
// with all rows in the L2.  The pairs' sums by two wavefronts instead of one: 5 us; the lengths' dots from terms that are there: 13.
#include <type_traits>
#include "delta.hpp"

namespace mrl {
namespace delta {
namespace {

constexpr int MOST_WAVES = 8;

struct Back {
    Delta d;
    Parts parts;
    const void *grad_out;
    long grad_out_ld;
    const float *grad_state_out;
    void *query, *key, *value, *gate, *rate;   // gradients
    int per_head;   // those of query and key are float [rows][H][dk], to be summed over groups of heads
    long query_ld, key_ld, value_ld, gate_ld, rate_ld;
    float *state;
    const float *states;
    const float *grad_ends;   // of the states behind the parts
    float *local;             // the same of parts with none behind them
    int blocks;
};

MRL_DEV float sum16(float x) { return sum_lanes<16>(x); }
// of a row's 16 lanes, the sum of those from this one on, and of those ahead of it
MRL_DEV float sum_from(float x) {
    x += moved<0x101>(x, 0.0f);
    x += moved<0x102>(x, 0.0f);
    x += moved<0x104>(x, 0.0f);
    return x + moved<0x108>(x, 0.0f);
}
MRL_DEV float sum_ahead(float x) {
    x = moved<0x111>(x, 0.0f);
    x += moved<0x111>(x, 0.0f);
    x += moved<0x112>(x, 0.0f);
    x += moved<0x114>(x, 0.0f);
    return x + moved<0x118>(x, 0.0f);
}

// What a tile's columns make of dO and dS1: dX, and dS1 becomes dS0.
template <class E, int DK, int TILES, bool KEEPS>
MRL_DEV void pull(const Block<E, DK, TILES, KEEPS> &block, int tile, int g, int c, const f32x4 dO, f32x4 (&dS)[DK / TILE], f32x4 &dX) {
    const f32x4 read = block.keys.ask(tile, g, c, Pieces<E, DK>(dS)) * block.four(block.key_takes, tile, g);
    f32x4 p_column, t_column;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        p_column[r] = block.Ps[(tile * TILE + 4 * g + r) * SIDE + c];
        t_column[r] = block.Ts[(tile * TILE + 4 * g + r) * SIDE + c];
    }
    dX = mfma16(t_column, mfma16(p_column, dO, read), f32x4{0.0f, 0.0f, 0.0f, 0.0f});
    settle(dX);
    const float whole = block.wholes[tile];
#pragma unroll
    for (int i = 0; i < DK / TILE; ++i) dS[i] *= whole;
    block.queries.add(tile, g, c, dO * block.four(block.query_reads, tile, g), dS);
    block.keys.add(tile, g, c, -dX * block.four(block.key_reads, tile, g), dS);
    if (block.cut_ahead(tile)) {
#pragma unroll
        for (int i = 0; i < DK / TILE; ++i) dS[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
}

template <int B>
MRL_DEV void first_gradient(const Back &p, int at_part, int nh, int column_tile, int tiles, bool behind, int g, int c, f32x4 (&dS)[B]) {
    const Delta &d = p.d;
    const int column = column_tile * TILE + c, lane = threadIdx.x & 63;
    if (p.parts.count > 1) {
        const float *from = p.grad_ends + (((long)at_part * tiles + min(column_tile, tiles - 1)) * B * 64 + lane) * 4;
#pragma unroll
        for (int i = 0; i < B; ++i) dS[i] = behind ? *reinterpret_cast<const f32x4 *>(from + i * 256) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    } else {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = i * TILE + 4 * g + r;
                dS[i][r] = p.grad_state_out != nullptr && column < d.dv && row < d.dk ? p.grad_state_out[((long)nh * d.dk + row) * d.dv + column] : 0.0f;
            }
    }
}

// The gradient of the state ahead of a part with none behind it: the chain of the states' gradients alone.
template <class E, int DK>
__global__ __launch_bounds__(256, 2) void chain_kernel(Back p, int column_groups) {
    extern __shared__ float lds[];
    constexpr int B = DK / TILE, TILES = tiles_backward(DK), STEPS = TILE * TILES;
    const Delta &d = p.d;
    Block<E, DK, TILES, false> block(lds);
    const int W = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int g = lane >> 4, c = lane & 15, thread = threadIdx.x;
    const int at = group_number(), group = at % column_groups, at_part = at / column_groups, part = at_part % p.parts.count, nh = at_part / p.parts.count;
    const int n = nh / d.H, h = nh - n * d.H, hk = h / (d.H / d.HK), tiles = (d.dv + TILE - 1) / TILE, column_tile = group * W + w, column = column_tile * TILE + c;
    const bool live = column < d.dv;
    const E *const grads = (const E *)p.grad_out + n * p.grad_out_ld + (long)h * d.dv + min(column, d.dv - 1);
    f32x4 dS[B], dO[TILES];
#pragma unroll
    for (int i = 0; i < B; ++i) dS[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int first_block = part * p.parts.per, last_block = min(p.blocks, first_block + p.parts.per) - 1;
    const int cut = find_cut<false>(d, first_block * STEPS, min(d.T, (last_block + 1) * STEPS), n, (int *)lds);
    for (int number = cut >= 0 ? cut / STEPS : last_block; number >= first_block; --number) {
        const int begin = number * STEPS, end = min(begin + STEPS, d.T);
        block.t0 = begin;
        block.span = TILE;
        int rounds = 1;
        for (int round = 0; round < rounds;) {
            anew(g, c);
            anew(thread);
            E asked[TILES][4];
            ask_values(d, block, grads, (long)d.N * p.grad_out_ld, g, asked);
            bool odd = block.template load<true>(d, n, h, hk, thread);
            odd |= take_values(d, block, asked, live, g, dO) | is_odd(dS);
            if (__syncthreads_or(odd) && block.span == TILE) {   // one step to a tile, TILES of them at a time, from the last
                block.span = 1;
                rounds = (end - begin + TILES - 1) / TILES;
                block.t0 = begin + (rounds - 1) * TILES;
                continue;
            }
            anew(g, c);
            for (int half = w; half < block.HALVES; half += W) block.template prepare<true>(d, half, g, c);
            __syncthreads();
#pragma unroll
            for (int tile = TILES - 1; tile >= 0; --tile) {
                if (block.t0 + tile * block.span >= d.T) continue;
                anew(g, c);
                f32x4 dX;
                pull(block, tile, g, c, dO[tile], dS, dX);
            }
            block.t0 -= TILES;
            ++round;
            __syncthreads();
        }
    }
    if (column_tile >= tiles) return;
    float *to = p.local + (((long)at_part * tiles + column_tile) * B * 64 + lane) * 4;
#pragma unroll
    for (int i = 0; i < B; ++i) *reinterpret_cast<f32x4 *>(to + i * 256) = dS[i];
}

constexpr bool both_states(int DK) { return DK < 128; }   // S0 and dS1 in LDS side by side
inline int waves_of(int DK, int dv) { return std::max(column_tiles(dv), std::min(4, DK / TILE)); }
enum { Q_READS, K_READS, K_TAKES, DOTS };                            // q dq and k dk of the terms with S0, k dk of that with dS1: of a wavefront's rows
enum { OF_A, OF_P = 3, U_DX = 6, OF_PAIRS };                            // of the pairs, per step: of dA and of dP the next three,
enum { CROSSING, ROW, COLUMN };                                        // sums over what crosses the step, over its row and over its column
template <class E>
size_t back_floats(int DK, int dv) {
    const int columns = TILE * column_tiles(dv) + 4, W = waves_of(DK, dv);
    return rows_floats<E>(DK, tiles_backward(DK), true) + (size_t)(both_states(DK) ? 2 : 1) * DK * columns + 3 * TILE * columns + 2 * TILE * SIDE + (OF_PAIRS + DOTS * W) * TILE + 2 * W;
}

// EK: the type of the gradients of query and key (float where a group's are summed later)
template <class E, class EK, int DK>
__global__ __launch_bounds__(64 * MOST_WAVES, 2) void back_kernel(Back p) {
    extern __shared__ float lds[];
    constexpr int B = DK / TILE, TILES = tiles_backward(DK), STEPS = TILE * TILES, OWN = B <= 4 ? 1 : 2;   // OWN: row tiles of a wavefront
    constexpr bool BOTH = both_states(DK);
    const Delta &d = p.d;
    Block<E, DK, TILES, true> block(lds);
    const int W = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, tiles = (d.dv + TILE - 1) / TILE;
    int g = lane >> 4, c = lane & 15, thread = threadIdx.x;
    const int stride = TILE * tiles + 4;
    float *const states = lds + rows_floats<E>(DK, TILES, true), *const behind = BOTH ? states + DK * stride : states, *const dOs = behind + DK * stride;
    float *const dXs = dOs + TILE * stride, *const Us = dXs + TILE * stride, *const dAs = Us + TILE * stride, *const dPs = dAs + TILE * SIDE;
    float *const of_pairs = dPs + TILE * SIDE, *const dots = of_pairs + OF_PAIRS * TILE, *const wholes = dots + DOTS * TILE * W;   // [OF_PAIRS][16], [DOTS][W][16], [2][W]: two tiles' in turn
    const int at_part = group_number(), part = at_part % p.parts.count, nh = at_part / p.parts.count, n = nh / d.H, h = nh - n * d.H, hk = h / (d.H / d.HK);
    const bool owns = w < tiles;   // columns; the other wavefronts have rows only
    const int column = w * TILE + c;
    const bool live = column < d.dv;
    const long state_at = (long)nh * d.dk * d.dv + column;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int key_at = (p.per_head ? h : hk) * d.dk;
    const E *const values = (const E *)d.value + n * d.value_ld + (long)h * d.dv + min(column, d.dv - 1);
    const E *const grads = (const E *)p.grad_out + n * p.grad_out_ld + (long)h * d.dv + min(column, d.dv - 1);

    f32x4 dS[B], S[B], V[TILES], dO[TILES], kept[TILES][B], U[TILES];
    first_gradient(p, at_part, nh, w, tiles, owns, g, c, dS);
    const auto first_state = [&](int number) {
        if (number > 0) {
            const float *from = p.states + ((((long)nh * p.blocks + number) * tiles + min(w, tiles - 1)) * B * 64 + lane) * 4;
#pragma unroll
            for (int i = 0; i < B; ++i) S[i] = owns ? *reinterpret_cast<const f32x4 *>(from + i * 256) : zero;
        } else {
#pragma unroll
            for (int i = 0; i < B; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = i * TILE + 4 * g + r;
                    S[i][r] = d.state_in != nullptr && live && row < d.dk ? d.state_in[state_at + (long)row * d.dv] : 0.0f;
                }
        }
    };
    // the tiles that the block holds, forwards; keep: S0 and U of each stay
    const auto forwards = [&](auto keep) {
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile) {
            anew(g, c);
            if (block.cut_ahead(tile)) {
#pragma unroll
                for (int i = 0; i < B; ++i) S[i] = zero;
            }
            const f32x4 u = solve(block, tile, g, c, V[tile], block.keys.ask(tile, g, c, Pieces<E, DK>(S)));
            if constexpr (decltype(keep)::value) {
#pragma unroll
                for (int i = 0; i < B; ++i) kept[tile][i] = S[i];
                U[tile] = u;
            }
            if (!decltype(keep)::value || tile + 1 < TILES) go_on(block, tile, g, c, u, S);
        }
    };
    const auto load = [&]() {
        anew(g, c);
        anew(thread);
        E asked_values[TILES][4], asked_grads[TILES][4];
        ask_values(d, block, values, (long)d.N * d.value_ld, g, asked_values);
        ask_values(d, block, grads, (long)d.N * p.grad_out_ld, g, asked_grads);
        bool odd = block.template load<true>(d, n, h, hk, thread);
        odd |= take_values(d, block, asked_values, live, g, V);
        return odd | take_values(d, block, asked_grads, live, g, dO);
    };
    const auto spread = [&](float *to, const f32x4 (&x)[B]) {   // a wavefront's columns of a state
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) to[(i * TILE + 4 * g + r) * stride + w * TILE + c] = x[i][r];
    };

    for (int number = min(p.blocks, (part + 1) * p.parts.per) - 1; number >= part * p.parts.per; --number) {
        const int begin = number * STEPS, end = min(begin + STEPS, d.T);
        first_state(number);
        block.t0 = begin;
        block.span = TILE;
        bool odd = load();
        odd |= is_odd(S) | is_odd(dS);
        int rounds = 1;
        if (__syncthreads_or(odd)) {   // one step to a tile, TILES of them at a time
            block.span = 1;
            rounds = (end - begin + TILES - 1) / TILES;
        }
        for (int round = rounds - 1; round >= 0; --round) {
            if (block.span == 1) {
                first_state(number);
                for (int ahead = 0; ahead <= round; ++ahead) {   // up to this round's, every time: only where a value is not finite
                    block.t0 = begin + ahead * TILES;
                    __syncthreads();
                    load();
                    __syncthreads();
                    if (ahead == round) break;
                    for (int half = w; half < block.HALVES; half += W) block.template prepare<false>(d, half, g, c);
                    __syncthreads();
                    forwards(std::false_type{});
                }
            }
            anew(g, c);
            for (int half = w; half < block.HALVES; half += W) block.template prepare<true>(d, half, g, c);
            __syncthreads();
            if (owns) forwards(std::true_type{});
#pragma unroll
            for (int tile = TILES - 1; tile >= 0; --tile) {
                if (block.t0 + tile * block.span >= d.T) continue;
                anew(g, c);
                const int turn = tile & 1, has_a = W > B ? W - 1 : 2 * tile % W, has_p = W > B + 1 ? W - 2 : (2 * tile + 1) % W;   // the wavefronts that have dA and dP
                const f32x4 b = block.four(block.bs, tile, g);
                const f32x4 from = block.four(block.from, tile, g), to = block.four(block.to, tile, g), ks = block.four(block.key_lengths, tile, g), qs = block.four(block.query_lengths, tile, g);
                f32x4 q[OWN], k[OWN], dq[OWN], dk[OWN], sums[DOTS] = {zero, zero, zero};   // (this wavefront's rows)
                const auto read_by_rows = [&]() {   // L dS1 U of this wavefront's rows
#pragma unroll
                    for (int o = 0; o < OWN; ++o) {
                        const int i = w + o * W;
                        dk[o] = zero;
                        if (i >= B) continue;
                        for (int t = 0; t < tiles; ++t)
                            dk[o] = mfma16(*reinterpret_cast<const f32x4 *>(Us + c * stride + t * TILE + 4 * g),
                                           *reinterpret_cast<const f32x4 *>(behind + (i * TILE + c) * stride + t * TILE + 4 * g), dk[o]);
                        settle(dk[o]);
                        dk[o] *= to;
                        k[o] = block.keys.column(tile, i, g, c) * ks;
                        sums[K_TAKES] += k[o] * dk[o];
                    }
                };
                if (owns) {
                    spread(behind, dS);
#pragma unroll
                    for (int r = 0; r < 4; ++r) Us[(4 * g + r) * stride + column] = U[tile][r];
                }
                if constexpr (!BOTH) {   // S0 comes in dS1's place
                    __syncthreads();
                    read_by_rows();
                    __syncthreads();
                }
                // ---- by columns
                if (owns) {
                    float s_ds = 0.0f;
#pragma unroll
                    for (int i = 0; i < B; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s_ds = fmaf(kept[tile][i][r], dS[i][r], s_ds);
                    s_ds = sum_groups(sum16(s_ds));
                    if (lane == 0) wholes[turn * W + w] = s_ds;
                    spread(states, kept[tile]);
                    f32x4 dX;
                    pull(block, tile, g, c, dO[tile], dS, dX);
                    store_values(d, block, (E *)p.value + n * p.value_ld + (long)h * d.dv + column, (long)d.N * p.value_ld, live, tile, g, b * dX);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int at = (4 * g + r) * stride + column;
                        dOs[at] = dO[tile][r];
                        dXs[at] = dX[r];
                    }
                }
                __syncthreads();
                // ---- by rows of the states, their terms of dq and dk; by a wavefront each, dA and dP
                if constexpr (BOTH) read_by_rows();
#pragma unroll
                for (int o = 0; o < OWN; ++o) {
                    const int i = w + o * W;
                    dq[o] = zero;
                    if (i >= B) continue;
                    f32x4 reads_by = zero;
                    for (int t = 0; t < tiles; ++t) {
                        const f32x4 s = *reinterpret_cast<const f32x4 *>(states + (i * TILE + c) * stride + t * TILE + 4 * g);
                        dq[o] = mfma16(*reinterpret_cast<const f32x4 *>(dOs + c * stride + t * TILE + 4 * g), s, dq[o]);
                        reads_by = mfma16(*reinterpret_cast<const f32x4 *>(dXs + c * stride + t * TILE + 4 * g), s, reads_by);
                    }
                    settle(dq[o]);
                    settle(reads_by);
                    dq[o] *= from;
                    reads_by *= -from * b;
                    q[o] = block.queries.column(tile, i, g, c) * qs;
                    sums[Q_READS] += q[o] * dq[o];
                    sums[K_READS] += k[o] * reads_by;
                    dk[o] += reads_by;
                }
                if (w < B) {
#pragma unroll
                    for (int s = 0; s < DOTS; ++s)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float sum = sum16(sums[s][r]);
                            if (c == 0) dots[(s * W + w) * TILE + 4 * g + r] = sum;
                        }
                }
                const auto pairs = [&](auto of_a) {
                    constexpr bool A = decltype(of_a)::value;
                    float *const sums_of = of_pairs + (A ? OF_A : OF_P) * TILE, *const rows = A ? dXs : dOs, *const factors = A ? block.As : block.Ps, *const to = A ? dAs : dPs;
                    f32x4 d = zero;
                    for (int t = 0; t < tiles; ++t)
                        d = mfma16(*reinterpret_cast<const f32x4 *>(rows + c * stride + t * TILE + 4 * g), *reinterpret_cast<const f32x4 *>(Us + c * stride + t * TILE + 4 * g), d);
                    settle(d);
                    const f32x4 apart = between(block.as + tile * TILE, g, c);
                    f32x4 m;   // dA A or dP P
                    float diagonal = 0.0f;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = 4 * g + r;
                        const float x = A ? (i > c ? -d[r] : 0.0f) : (i >= c ? d[r] : 0.0f);
                        m[r] = x * factors[(tile * TILE + i) * SIDE + c];
                        to[i * SIDE + c] = x * apart[r] * (A ? b[r] : 1.0f);
                        const float row = sum16(m[r]);
                        if (c == 0) sums_of[ROW * TILE + i] = row;
                        diagonal = i == c ? d[r] : diagonal;
                    }
                    if (A && c >> 2 == g) of_pairs[U_DX * TILE + c] = diagonal;
                    // sums over the rows from 4 g + r on, and of these over the columns ahead
                    const float mine = (m[0] + m[1]) + (m[2] + m[3]);
                    const float of1 = __shfl(mine, 16 + c), of2 = __shfl(mine, 32 + c), of3 = __shfl(mine, 48 + c);
                    if (g == 0) sums_of[COLUMN * TILE + c] = (mine + of1) + (of2 + of3);
                    float run = (g < 3 ? of3 : 0.0f) + (g < 2 ? of2 : 0.0f) + (g < 1 ? of1 : 0.0f);
#pragma unroll
                    for (int r = 3; r >= 0; --r) {
                        run += m[r];
                        const float sum = sum16(c < 4 * g + r ? run : 0.0f);
                        if (c == 0) sums_of[CROSSING * TILE + 4 * g + r] = sum;
                    }
                };
                if (w == has_a) pairs(std::true_type{});
                if (w == has_p) pairs(std::false_type{});
                __syncthreads();
                // ---- the tile's own pairs, the lengths, gates and rates
                const auto of_pair = [&](int which) { return *reinterpret_cast<const f32x4 *>(of_pairs + which * TILE + 4 * g); };
                const int row_waves = min(W, B);
                f32x4 q_dot = of_pair(OF_P + ROW), k_dot = of_pair(OF_A + ROW) + (of_pair(OF_A + COLUMN) + of_pair(OF_P + COLUMN));
                for (int t = 0; t < row_waves; ++t) {
                    q_dot += *reinterpret_cast<const f32x4 *>(dots + (Q_READS * W + t) * TILE + 4 * g);
                    k_dot += *reinterpret_cast<const f32x4 *>(dots + (K_READS * W + t) * TILE + 4 * g) + *reinterpret_cast<const f32x4 *>(dots + (K_TAKES * W + t) * TILE + 4 * g);
                }
#pragma unroll
                for (int o = 0; o < OWN; ++o) {
                    const int i = w + o * W;
                    if (i >= B) continue;
                    f32x4 a_column, p_column;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        a_column[r] = dAs[(4 * g + r) * SIDE + c];
                        p_column[r] = dPs[(4 * g + r) * SIDE + c];
                    }
                    dq[o] = mfma16(*reinterpret_cast<const f32x4 *>(dPs + c * SIDE + 4 * g), k[o], dq[o]);
                    dk[o] = mfma16(*reinterpret_cast<const f32x4 *>(dAs + c * SIDE + 4 * g), k[o], dk[o]);
                    dk[o] = mfma16(p_column, q[o], mfma16(a_column, k[o], dk[o]));
                    settle(dq[o]);
                    settle(dk[o]);
                    const int at = i * TILE + c;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        q[o][r] = qs[r] * fmaf(-(float)d.dk * q[o][r], q_dot[r], dq[o][r]);
                        k[o][r] = ks[r] * fmaf(-k[o][r], k_dot[r], dk[o][r]);
                    }
                    if (block.span == 1) {   // lengths are without the rows' powers of two
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            q[o][r] = in_units(q[o][r], block.query_units[tile * TILE + 4 * g + r]);
                            k[o][r] = in_units(k[o][r], block.key_units[tile * TILE + 4 * g + r]);
                        }
                    }
                    store_values(d, block, (EK *)p.query + n * p.query_ld + key_at + at, (long)d.N * p.query_ld, at < d.dk, tile, g, q[o]);
                    store_values(d, block, (EK *)p.key + n * p.key_ld + key_at + at, (long)d.N * p.key_ld, at < d.dk, tile, g, k[o]);
                }
                if (w == has_a && g == 0) {
                    float e = 0.0f, f = 0.0f, all = 0.0f;
                    for (int t = 0; t < row_waves; ++t) {
                        e += dots[(Q_READS * W + t) * TILE + c] + dots[(K_READS * W + t) * TILE + c];
                        f += dots[(K_TAKES * W + t) * TILE + c];
                    }
                    for (int t = 0; t < tiles; ++t) all += wholes[turn * W + t];
                    const float sum = fmaf(block.wholes[tile], all, (of_pairs[(OF_A + CROSSING) * TILE + c] + of_pairs[(OF_P + CROSSING) * TILE + c]) + (sum_from(e) + sum_ahead(f)));
                    const int slot = tile * TILE + c;
                    if (block.there(d, slot)) {
                        const long row = (long)block.time_of(slot) * d.N + n;
                        give((E *)p.gate + row * p.gate_ld + h, block.as[slot] == 0.0f ? 0.0f : block.rests[slot] * sum);
                        give((E *)p.rate + row * p.rate_ld + h, block.rate_rests[slot] * of_pairs[U_DX * TILE + c]);
                    }
                }
                if constexpr (!BOTH) __syncthreads();
            }
            __syncthreads();
        }
    }
    if (p.state == nullptr || !live || part != 0) return;
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = i * TILE + 4 * g + r;
            if (row < d.dk) p.state[state_at + (long)row * d.dv] = dS[i][r];
        }
}

// gradients of a key head's query and key: those of its heads, [rows][H][dk], in order
template <class E>
__global__ __launch_bounds__(256) void sum_heads_kernel(const float *from, int64_t rows, int HK, int per, int dk, E *to, long ld) {
    const int64_t all = rows * HK * dk;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / (HK * dk);
        const int at = (int)(i - row * HK * dk), hk = at / dk, x = at - hk * dk;
        const float *p = from + (row * HK + hk) * per * dk + x;
        float sum = p[0];
        for (int j = 1; j < per; ++j) sum += p[(long)j * dk];
        give(to + row * ld + at, sum);
    }
}

struct Plan {
    Parts parts;
    int blocks;
    size_t states, partial, ends, starts, grads, cuts, bytes;   // bytes: of the states ahead of the blocks, the groups' gradients, what the parts take, all
};
Plan plan_of(const mrl_ctx *ctx, const mrl_delta *r) {
    Plan p = {};
    if (r->T == 0 || r->N == 0) return p;
    const int tiles = tiles_backward(padded(r->key_dim));
    p.parts = parts_of(ctx, r, tiles);
    p.blocks = blocks_of(r->T, tiles);
    if (p.blocks > 1) p.states = sizeof(float) * (size_t)r->N * r->heads * p.blocks * column_tiles(r->value_dim) * floats_of(padded(r->key_dim));
    if (r->heads != r->key_heads) p.partial = (sizeof(float) * (size_t)r->T * r->N * r->heads * r->key_dim + 15) / 16 * 16;
    p.ends = sizeof(float) * ends_floats(r, p.parts);
    p.starts = p.grads = sizeof(float) * starts_floats(r, p.parts);
    p.cuts = sizeof(float) * cuts_floats(r, p.parts);
    p.bytes = p.states + 2 * p.partial + p.ends + 2 * p.starts + p.grads + p.cuts;
    return p;
}

template <class E, class EK, int DK>
void launch(const mrl_ctx *ctx, const Back &p) {
    hipLaunchKernelGGL((back_kernel<E, EK, DK>), dim3(p.d.N * p.d.H * p.parts.count), dim3(64 * waves_of(DK, p.d.dv)), sizeof(float) * back_floats<E>(DK, p.d.dv), ctx->stream, p);
}
template <class E, int DK>
void launch_chain(const mrl_ctx *ctx, const Back &p) {
    const int tiles = column_tiles(p.d.dv), waves = std::min(4, tiles), groups = (tiles + waves - 1) / waves;
    hipLaunchKernelGGL((chain_kernel<E, DK>), dim3(p.d.N * p.d.H * p.parts.count * groups), dim3(64 * waves), sizeof(float) * rows_floats<E>(DK, tiles_backward(DK), false), ctx->stream, p, groups);
}
template <class E>
void launch_chain(const mrl_ctx *ctx, const Back &p) {
    switch (padded(p.d.dk)) {
        case 16: return launch_chain<E, 16>(ctx, p);
        case 32: return launch_chain<E, 32>(ctx, p);
        case 64: return launch_chain<E, 64>(ctx, p);
        default: return launch_chain<E, 128>(ctx, p);
    }
}
template <class E, class EK>
void launch(const mrl_ctx *ctx, const Back &p) {
    switch (padded(p.d.dk)) {
        case 16: return launch<E, EK, 16>(ctx, p);
        case 32: return launch<E, EK, 32>(ctx, p);
        case 64: return launch<E, EK, 64>(ctx, p);
        default: return launch<E, EK, 128>(ctx, p);
    }
}
template <class E>
void launch(const mrl_ctx *ctx, Back p, float *partial, size_t partial_bytes) {
    if (partial == nullptr) return launch<E, E>(ctx, p);
    E *const query = (E *)p.query, *const key = (E *)p.key;
    const long query_ld = p.query_ld, key_ld = p.key_ld;
    const Delta &d = p.d;
    p.query = partial;
    p.key = (char *)partial + partial_bytes;
    p.query_ld = p.key_ld = (long)d.H * d.dk;
    p.per_head = 1;
    launch<E, float>(ctx, p);
    const int64_t rows = (int64_t)d.T * d.N;
    const dim3 grid((unsigned)std::min<int64_t>((rows * d.HK * d.dk + 255) / 256, 8192));
    hipLaunchKernelGGL((sum_heads_kernel<E>), grid, dim3(256), 0, ctx->stream, (const float *)p.query, rows, d.HK, d.H / d.HK, d.dk, query, query_ld);
    hipLaunchKernelGGL((sum_heads_kernel<E>), grid, dim3(256), 0, ctx->stream, (const float *)p.key, rows, d.HK, d.H / d.HK, d.dk, key, key_ld);
}

}  // namespace
}  // namespace delta
}  // namespace mrl

extern "C" {

int mrl_delta_workspace(mrl_ctx *ctx, const mrl_delta *r, int backward, uint64_t *bytes) {
    using namespace mrl;
    MRL_CHECK_ARG(ctx && r && bytes, "mrl_delta_workspace: NULL ctx, description or result");
    const int rc = delta::check_sizes("mrl_delta_workspace", r);
    if (rc != MRL_OK) return rc;
    *bytes = backward ? delta::plan_of(ctx, r).bytes : delta::forward_bytes(ctx, r);
    return MRL_OK;
}

int mrl_delta_backward(mrl_ctx *ctx, const mrl_delta *r, const void *grad_out, int64_t grad_out_ld, const float *grad_state_out,
                       const mrl_delta_grads *grads, void *workspace, uint64_t workspace_bytes) {
    using namespace mrl;
    using namespace mrl::delta;
    const char *who = "mrl_delta_backward";
    const int rc = check(who, ctx, r);
    if (rc != MRL_OK) return rc;
    MRL_CHECK_ARG(grads, "%s: NULL gradients", who);
    if (r->N == 0) return MRL_OK;
    const mrl_delta_grads &to = *grads;
    const long states = (long)r->N * r->heads * r->key_dim * r->value_dim, k_width = (long)r->key_heads * r->key_dim, v_width = (long)r->heads * r->value_dim;
    const Plan plan = plan_of(ctx, r);
    const size_t need = plan.bytes;
    if (r->T > 0) {
        MRL_CHECK_ARG(grad_out && to.query && to.key && to.value && to.gate && to.rate, "%s: NULL buffer", who);
        MRL_CHECK_ARG(grad_out_ld >= v_width && to.query_ld >= k_width && to.key_ld >= k_width && to.value_ld >= v_width && to.gate_ld >= r->heads && to.rate_ld >= r->heads,
                      "%s: a row stride is smaller than the row", who);
        MRL_CHECK_ARG(workspace_bytes >= need && (need == 0 || workspace != nullptr), "%s: the workspace holds %llu bytes, need %llu", who,
                      (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)need);
        MRL_CHECK_ARG(need == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: the workspace must be 16-byte aligned", who);
    }
    const int64_t size = r->dtype == MRL_F32 ? 4 : 2, rows = (int64_t)r->T * r->N;
    const auto of = [&](const char *name, const void *at, long width, long ld) { return Region(name, at, rows, size * width, size * ld); };
    const int apart = check_apart(who, {of("grad_query", to.query, k_width, to.query_ld), of("grad_key", to.key, k_width, to.key_ld), of("grad_value", to.value, v_width, to.value_ld),
                                        of("grad_gate", to.gate, r->heads, to.gate_ld), of("grad_rate", to.rate, r->heads, to.rate_ld), Region("grad_state_in", to.state, 4 * states),
                                        Region("the workspace", need ? workspace : nullptr, (int64_t)need)},
                                  {of("query", r->query, k_width, r->query_ld), of("key", r->key, k_width, r->key_ld), of("value", r->value, v_width, r->value_ld),
                                   of("gate", r->gate, r->heads, r->gate_ld), of("rate", r->rate, r->heads, r->rate_ld), of("grad_out", grad_out, v_width, grad_out_ld),
                                   Region("dones", r->dones, 4 * rows), Region("prev_dones", r->prev_dones, 4LL * r->N), Region("state_in", r->state_in, 4 * states),
                                   Region("grad_state_out", grad_state_out == to.state ? nullptr : grad_state_out, 4 * states)});
    if (apart != MRL_OK) return apart;
    OnDevice on(ctx);
    if (r->T == 0) {
        if (to.state != nullptr && to.state != grad_state_out)
            hipLaunchKernelGGL(pass_state_kernel, dim3((int)std::min<long>((states + 255) / 256, 4096)), dim3(256), 0, ctx->stream, grad_state_out, to.state, states);
        MRL_CHECK_LAUNCH();
        return MRL_OK;
    }
    Back p = {};
    p.d = describe(r);
    p.grad_out = grad_out; p.grad_out_ld = grad_out_ld;
    p.grad_state_out = grad_state_out;
    p.query = to.query; p.key = to.key; p.value = to.value; p.gate = to.gate; p.rate = to.rate;
    p.query_ld = to.query_ld; p.key_ld = to.key_ld; p.value_ld = to.value_ld; p.gate_ld = to.gate_ld; p.rate_ld = to.rate_ld;
    p.state = to.state;
    p.blocks = plan.blocks;
    p.parts = plan.parts;
    char *at = (char *)workspace;
    const auto take = [&](size_t bytes) {
        char *const was = bytes ? at : nullptr;
        at += bytes;
        return (float *)was;
    };
    float *const ahead = take(plan.states), *const partial = take(2 * plan.partial), *const grad_ends = take(plan.grads);
    p.parts.ends = take(plan.ends);
    p.parts.starts = take(plan.starts);
    p.local = take(plan.grads);
    p.parts.cuts = (int *)take(plan.cuts);
    p.states = ahead;
    p.grad_ends = grad_ends;
    int launched = MRL_OK;
    if (plan.parts.count > 1) {
        launched = launch_starts(ctx, r->dtype, p.d, p.parts);
        if (launched != MRL_OK) return launched;
        if (r->dtype == MRL_F32) launch_chain<float>(ctx, p);
        else launch_chain<bf16_t>(ctx, p);
        Parts ends = p.parts;
        ends.starts = grad_ends;
        launched = launch_grad_ends(ctx, p.d, ends, grad_state_out, p.local);
        if (launched != MRL_OK) return launched;
    }
    if (plan.blocks > 1) launched = launch_states(ctx, r->dtype, p.d, p.parts, ahead, plan.blocks);
    if (launched != MRL_OK) return launched;
    if (r->dtype == MRL_F32) launch<float>(ctx, p, partial, plan.partial);
    else launch<bf16_t>(ctx, p, partial, plan.partial);
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}

}  // extern "C"
