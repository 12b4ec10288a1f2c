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
// A first launch leaves the state ahead of every block of tiles in the workspace (mrl_delta.hip).  In the second a workgroup goes through the blocks
// of one head of one environment from the last to the first: it repeats a block's tiles forwards, keeping each tile's S0 and U in registers,
// and takes the tiles backwards.  A wavefront holds 16 columns of S0 and dS1; what contracts over the columns (dq, dk, dA, dP) is done by 16
// rows of the states per wavefront, which they pass through LDS, S0 first and dS1 after it in the same place.
#include <type_traits>
#include "delta.hpp"

namespace mrl {
namespace delta {
namespace {

constexpr int MOST_WAVES = 8;

struct Back {
    Delta d;
    const void *grad_out;
    long grad_out_ld;
    const float *grad_state_out;
    void *query, *key, *value, *gate, *rate;   // gradients
    int per_head;   // those of query and key are float [rows][H][dk], to be summed over groups of heads
    long query_ld, key_ld, value_ld, gate_ld, rate_ld;
    float *state;
    const float *states;
    int blocks;
};

constexpr size_t back_floats(int DK, int W) {
    const int columns = TILE * W + 4;
    return rows_floats(DK) + (size_t)DK * columns + 3 * TILE * columns + 2 * TILE * SIDE + 3 * TILE * MOST_WAVES + MOST_WAVES;
}

MRL_DEV float sum16(float x) {   // over the 16 lanes of a group
#pragma unroll
    for (int s = 1; s < 16; s *= 2) x += __shfl_xor(x, s);
    return x;
}
// EK: the type of the gradients of query and key (float where a group's are summed later)
template <class E, class EK, int DK>
__global__ __launch_bounds__(64 * MOST_WAVES) void back_kernel(Back p) {
    extern __shared__ float lds[];
    constexpr int B = DK / TILE, TILES = Block<DK>::TILES, STEPS = Block<DK>::STEPS, ROW = Block<DK>::ROW;
    const Delta &d = p.d;
    Block<DK> block(lds);
    const int W = blockDim.x >> 6, w = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
    const int columns = TILE * W + 4;
    float *state = lds + rows_floats(DK), *dOs = state + DK * columns, *dXs = dOs + TILE * columns, *Us = dXs + TILE * columns;
    float *dAs = Us + TILE * columns, *dPs = dAs + TILE * SIDE, *dots = dPs + TILE * SIDE, *whole = dots + 3 * TILE * MOST_WAVES;
    const int nh = blockIdx.x, n = nh / d.H, h = nh - n * d.H, hk = h / (d.H / d.HK);
    const int column = w * TILE + c;
    const bool live = column < d.dv;
    const long state_at = (long)nh * d.dk * d.dv + column;
    const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    const int key_at = (p.per_head ? h : hk) * d.dk;

    f32x4 dS[B];
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = i * TILE + 4 * g + r;
            dS[i][r] = p.grad_state_out != nullptr && live && row < d.dk ? p.grad_state_out[state_at + (long)row * d.dv] : 0.0f;
        }

    const auto first_state = [&](int number, f32x4 (&S)[B]) {
        if (number > 0) {
            const float *from = p.states + ((((long)nh * p.blocks + number) * W + w) * B * 64 + lane) * 4;
#pragma unroll
            for (int i = 0; i < B; ++i) S[i] = *reinterpret_cast<const f32x4 *>(from + i * 256);
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
    f32x4 S[B], V[TILES], dO[TILES], kept[TILES][B], U[TILES];
    // the tiles that the block holds, forwards; keep: S0 and U of each stay
    const auto forwards = [&](auto keep) {
#pragma unroll
        for (int tile = 0; tile < TILES; ++tile) {
            Decays decay;
            decay.load(block.as + tile * TILE, g);
            if (block.cut_ahead(tile)) {
#pragma unroll
                for (int i = 0; i < B; ++i) S[i] = zero;
            }
            f32x4 sk = zero;
#pragma unroll
            for (int i = 0; i < B; ++i) sk = mfma16(*reinterpret_cast<const f32x4 *>(block.K + (tile * TILE + c) * ROW + i * TILE + 4 * g), S[i], sk);
            const f32x4 u = solve(block, decay, tile, g, c, V[tile], sk);
            if constexpr (decltype(keep)::value) {
#pragma unroll
                for (int i = 0; i < B; ++i) kept[tile][i] = S[i];
                U[tile] = u;
            }
            if (!decltype(keep)::value || tile + 1 < TILES) go_on(block, decay, tile, g, c, u, S);
        }
    };
    const E *const values = (const E *)d.value + n * d.value_ld + (long)h * d.dv + min(column, d.dv - 1);
    const E *const grads = (const E *)p.grad_out + n * p.grad_out_ld + (long)h * d.dv + min(column, d.dv - 1);
    const auto load = [&]() {
        bool odd = load_values<E, DK>(d, block, values, (long)d.N * d.value_ld, live, g, V);
        odd |= load_values<E, DK>(d, block, grads, (long)d.N * p.grad_out_ld, live, g, dO);
        odd |= block.template load<E, true>(d, n, h, hk, threadIdx.x);
        return odd;
    };

    for (int number = p.blocks - 1; number >= 0; --number) {
        const int begin = number * STEPS, end = min(begin + STEPS, d.T);
        first_state(number, S);
        block.t0 = begin;
        block.span = TILE;
        bool odd = is_odd(S) | is_odd(dS);
        odd |= load();
        int parts = 1;
        if (__syncthreads_or(odd)) {   // one step to a tile, TILES of them at a time
            block.span = 1;
            parts = (end - begin + TILES - 1) / TILES;
        }
        for (int part = parts - 1; part >= 0; --part) {
            if (block.span == 1) {
                first_state(number, S);
                for (int ahead = 0; ahead <= part; ++ahead) {   // up to this part, every time: only where a value is not finite
                    block.t0 = begin + ahead * TILES;
                    load();
                    __syncthreads();
                    if (ahead == part) break;
                    for (int tile = w; tile < TILES; tile += W) block.template prepare<false>(tile, g, c);
                    __syncthreads();
                    forwards(std::false_type{});
                    __syncthreads();
                }
            }
            for (int tile = w; tile < TILES; tile += W) block.template prepare<true>(tile, g, c);
            __syncthreads();
            forwards(std::true_type{});
#pragma unroll
            for (int tile = TILES - 1; tile >= 0; --tile) {
                if (block.t0 + tile * block.span >= d.T) continue;
                const float *k_tile = block.K + tile * TILE * ROW, *q_tile = block.Q + tile * TILE * ROW;
                const float *T = block.Ts + tile * TILE * SIDE, *P = block.Ps + tile * TILE * SIDE;
                Decays decay;
                decay.load(block.as + tile * TILE, g);
                const f32x4 b = block.four(block.bs, tile, g), ks = block.four(block.kscale, tile, g), qs = block.four(block.qscale, tile, g);
                const bool cut = block.cut_ahead(tile);
                // ---- by columns
                f32x4 dU = zero;
#pragma unroll
                for (int i = 0; i < B; ++i) dU = mfma16(*reinterpret_cast<const f32x4 *>(k_tile + c * ROW + i * TILE + 4 * g), dS[i], dU);
                f32x4 p_column, t_column;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    dU[r] *= decay.to[r] * ks[r];
                    p_column[r] = P[(4 * g + r) * SIDE + c];
                    t_column[r] = T[(4 * g + r) * SIDE + c];
                }
                dU = mfma16(p_column, dO[tile], dU);
                const f32x4 dX = mfma16(t_column, dU, zero);
                float s_ds = 0.0f;
#pragma unroll
                for (int i = 0; i < B; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s_ds = fmaf(kept[tile][i][r], dS[i][r], s_ds);
                        state[(i * TILE + 4 * g + r) * columns + column] = kept[tile][i][r];
                    }
                s_ds = sum_groups(sum16(s_ds));
                if (lane == 0) whole[w] = s_ds;
                f32x4 q_part, k_part;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int slot = tile * TILE + 4 * g + r, at = (4 * g + r) * columns + column;
                    dOs[at] = dO[tile][r];
                    dXs[at] = dX[r];
                    Us[at] = U[tile][r];
                    if (live && block.there(d, slot)) give((E *)p.value + ((long)block.time_of(slot) * d.N + n) * p.value_ld + h * d.dv + column, b[r] * dX[r]);
                    q_part[r] = decay.from[r] * qs[r] * dO[tile][r];
                    k_part[r] = -decay.from[r] * ks[r] * b[r] * dX[r];
                }
                f32x4 dS0[B];
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    f32x4 q, k;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        q[r] = q_tile[(4 * g + r) * ROW + i * TILE + c];
                        k[r] = k_tile[(4 * g + r) * ROW + i * TILE + c];
                    }
                    dS0[i] = mfma16(k, k_part, mfma16(q, q_part, dS[i] * decay.whole));
                    if (cut) dS0[i] = zero;
                }
                __syncthreads();
                // ---- by rows of S0: the terms of dq and dk with it; by the first wavefront, dA and dP
                f32x4 dq[B], dk_reads[B], dk_read[B];   // of which this wavefront has every W-th
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    dq[i] = dk_reads[i] = dk_read[i] = zero;
                    if (i % W != w) continue;
                    for (int t = 0; t < W; ++t) {
                        const f32x4 s = *reinterpret_cast<const f32x4 *>(state + (i * TILE + c) * columns + t * TILE + 4 * g);
                        dq[i] = mfma16(*reinterpret_cast<const f32x4 *>(dOs + c * columns + t * TILE + 4 * g), s, dq[i]);
                        dk_reads[i] = mfma16(*reinterpret_cast<const f32x4 *>(dXs + c * columns + t * TILE + 4 * g), s, dk_reads[i]);
                    }
                }
                f32x4 eq = zero, ek = zero, fk = zero;
#pragma unroll
                for (int i = 0; i < B; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        dq[i][r] *= decay.from[r];
                        dk_reads[i][r] *= -decay.from[r] * b[r];
                        if (i % W != w) continue;
                        eq[r] = fmaf(q_tile[(4 * g + r) * ROW + i * TILE + c] * qs[r], dq[i][r], eq[r]);
                        ek[r] = fmaf(k_tile[(4 * g + r) * ROW + i * TILE + c] * ks[r], dk_reads[i][r], ek[r]);
                    }
                f32x4 a_terms = zero, p_terms = zero;   // dA A and dP P
                if (w == 0) {
                    f32x4 dA = zero, dP = zero;
                    for (int t = 0; t < W; ++t) {
                        const f32x4 u = *reinterpret_cast<const f32x4 *>(Us + c * columns + t * TILE + 4 * g);
                        dA = mfma16(*reinterpret_cast<const f32x4 *>(dXs + c * columns + t * TILE + 4 * g), u, dA);
                        dP = mfma16(*reinterpret_cast<const f32x4 *>(dOs + c * columns + t * TILE + 4 * g), u, dP);
                    }
                    const f32x4 apart = between(block.as + tile * TILE, g, c);
                    f32x4 kk = zero, qk = zero;
#pragma unroll
                    for (int i = 0; i < B; ++i) {
                        const f32x4 k = *reinterpret_cast<const f32x4 *>(k_tile + c * ROW + i * TILE + 4 * g), q = *reinterpret_cast<const f32x4 *>(q_tile + c * ROW + i * TILE + 4 * g);
                        kk = mfma16(k, k, kk);
                        qk = mfma16(q, k, qk);
                    }
                    const float kc = block.kscale[tile * TILE + c];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int i = 4 * g + r, slot = tile * TILE + i;
                        if (i == c && block.there(d, slot))
                            give((E *)p.rate + ((long)block.time_of(slot) * d.N + n) * p.rate_ld + h, block.rate_rests[slot] * dA[r]);
                        const float a_times = i > c ? -dA[r] * b[r] * apart[r] : 0.0f, p_times = i >= c ? dP[r] * apart[r] : 0.0f;
                        a_terms[r] = i > c ? a_times * (ks[r] * kc * kk[r]) : 0.0f;
                        p_terms[r] = i >= c ? p_times * (qs[r] * kc * qk[r]) : 0.0f;
                        dAs[i * SIDE + c] = a_times;
                        dPs[i * SIDE + c] = p_times;
                    }
                }
                __syncthreads();
                // ---- dS1 in S0's place
#pragma unroll
                for (int i = 0; i < B; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) state[(i * TILE + 4 * g + r) * columns + column] = dS[i][r];
                __syncthreads();
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    dS[i] = dS0[i];
                    if (i % W != w) continue;
                    for (int t = 0; t < W; ++t)
                        dk_read[i] = mfma16(*reinterpret_cast<const f32x4 *>(Us + c * columns + t * TILE + 4 * g),
                                            *reinterpret_cast<const f32x4 *>(state + (i * TILE + c) * columns + t * TILE + 4 * g), dk_read[i]);
                    f32x4 k, q, a_column, p_column;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        dk_read[i][r] *= decay.to[r];
                        k[r] = k_tile[(4 * g + r) * ROW + i * TILE + c] * ks[r];
                        q[r] = q_tile[(4 * g + r) * ROW + i * TILE + c] * qs[r];
                        fk[r] = fmaf(k[r], dk_read[i][r], fk[r]);
                        a_column[r] = dAs[(4 * g + r) * SIDE + c];
                        p_column[r] = dPs[(4 * g + r) * SIDE + c];
                    }
                    dq[i] = mfma16(*reinterpret_cast<const f32x4 *>(dPs + c * SIDE + 4 * g), k, dq[i]);
                    dk_reads[i] = mfma16(*reinterpret_cast<const f32x4 *>(dAs + c * SIDE + 4 * g), k, dk_reads[i]);
                    dk_read[i] = mfma16(p_column, q, mfma16(a_column, k, dk_read[i]));
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float x = sum16(eq[r]), y = sum16(ek[r]), z = sum16(fk[r]);
                    if (c == 0) {
                        dots[(0 * MOST_WAVES + w) * TILE + 4 * g + r] = x;
                        dots[(1 * MOST_WAVES + w) * TILE + 4 * g + r] = y;
                        dots[(2 * MOST_WAVES + w) * TILE + 4 * g + r] = z;
                    }
                }
                float *sums = dAs;   // row i: what the dots of q and k take from the tile's own pairs
                __syncthreads();
                if (w == 0) {
                    f32x4 both = a_terms + p_terms;
                    float below = both[0] + both[1] + both[2] + both[3];   // rows of this column below the group's own
                    const float from1 = __shfl(below, 16 + c), from2 = __shfl(below, 32 + c), from3 = __shfl(below, 48 + c), from0 = __shfl(below, c);
                    const float read = from0 + from1 + from2 + from3;
                    f32x4 crossing;
                    float run = (g < 3 ? from3 : 0.0f) + (g < 2 ? from2 : 0.0f) + (g < 1 ? from1 : 0.0f);
                    f32x4 a_row, p_row;
#pragma unroll
                    for (int r = 3; r >= 0; --r) {
                        run += both[r];
                        crossing[r] = sum16(c < 4 * g + r ? run : 0.0f);
                        a_row[r] = sum16(a_terms[r]);
                        p_row[r] = sum16(p_terms[r]);
                    }
                    if (c == 0) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            sums[0 * TILE + 4 * g + r] = p_row[r];
                            sums[1 * TILE + 4 * g + r] = a_row[r];
                            sums[3 * TILE + 4 * g + r] = crossing[r];
                        }
                    }
                    if (g == 0) sums[2 * TILE + c] = read;
                }
                __syncthreads();
                f32x4 q_dot = *reinterpret_cast<const f32x4 *>(sums + 4 * g), k_dot = *reinterpret_cast<const f32x4 *>(sums + TILE + 4 * g) + *reinterpret_cast<const f32x4 *>(sums + 2 * TILE + 4 * g);
                for (int t = 0; t < W; ++t) {
                    q_dot += *reinterpret_cast<const f32x4 *>(dots + (0 * MOST_WAVES + t) * TILE + 4 * g);
                    k_dot += *reinterpret_cast<const f32x4 *>(dots + (1 * MOST_WAVES + t) * TILE + 4 * g) + *reinterpret_cast<const f32x4 *>(dots + (2 * MOST_WAVES + t) * TILE + 4 * g);
                }
#pragma unroll
                for (int i = 0; i < B; ++i) {
                    if (i % W != w) continue;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int slot = tile * TILE + 4 * g + r, at = i * TILE + c;
                        if (at >= d.dk || !block.there(d, slot)) continue;
                        const long row = (long)block.time_of(slot) * d.N + n;
                        const float q = q_tile[(4 * g + r) * ROW + at] * qs[r], k = k_tile[(4 * g + r) * ROW + at] * ks[r];
                        give((EK *)p.query + row * p.query_ld + key_at + at, qs[r] * fmaf(-(float)d.dk * q, q_dot[r], dq[i][r]));
                        give((EK *)p.key + row * p.key_ld + key_at + at, ks[r] * fmaf(-k, k_dot[r], dk_reads[i][r] + dk_read[i][r]));
                    }
                }
                if (w == 0 && lane < TILE && block.there(d, tile * TILE + lane)) {
                    float sum = sums[3 * TILE + lane], all = 0.0f;
                    for (int t = 0; t < W; ++t) {
                        for (int j = 0; j < TILE; ++j)
                            sum += j < lane ? dots[(2 * MOST_WAVES + t) * TILE + j] : dots[t * TILE + j] + dots[(1 * MOST_WAVES + t) * TILE + j];
                        all += whole[t];
                    }
                    sum = fmaf(decay.whole, all, sum);
                    const int slot = tile * TILE + lane;
                    give((E *)p.gate + ((long)block.time_of(slot) * d.N + n) * p.gate_ld + h, block.as[slot] == 0.0f ? 0.0f : block.rests[slot] * sum);
                }
                __syncthreads();
            }
        }
        __syncthreads();
    }
    if (p.state == nullptr || !live) return;
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
    int blocks;
    size_t states, partial;   // bytes
};
Plan plan_of(const mrl_delta *r) {
    Plan p = {};
    if (r->T == 0 || r->N == 0) return p;
    p.blocks = blocks_of(r->T, r->key_dim);
    if (p.blocks > 1) p.states = sizeof(float) * (size_t)r->N * r->heads * p.blocks * column_tiles(r->value_dim) * TILE * padded(r->key_dim);
    if (r->heads != r->key_heads) p.partial = (sizeof(float) * (size_t)r->T * r->N * r->heads * r->key_dim + 15) / 16 * 16;
    return p;
}

template <class E, class EK, int DK>
void launch(const mrl_ctx *ctx, const Back &p) {
    const int W = column_tiles(p.d.dv);
    hipLaunchKernelGGL((back_kernel<E, EK, DK>), dim3(p.d.N * p.d.H), dim3(64 * W), sizeof(float) * back_floats(DK, W), ctx->stream, p);
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
    const delta::Plan p = backward ? delta::plan_of(r) : delta::Plan{};
    *bytes = p.states + 2 * p.partial;
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
    const Plan plan = plan_of(r);
    const size_t need = plan.states + 2 * plan.partial;
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
    p.states = plan.states ? (const float *)workspace : nullptr;
    if (plan.blocks > 1) {
        const int launched = launch_states(ctx, r->dtype, p.d, (float *)workspace, plan.blocks);
        if (launched != MRL_OK) return launched;
    }
    float *const partial = plan.partial ? (float *)((char *)workspace + plan.states) : nullptr;
    if (r->dtype == MRL_F32) launch<float>(ctx, p, partial, plan.partial);
    else launch<bf16_t>(ctx, p, partial, plan.partial);
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}

}  // extern "C"
