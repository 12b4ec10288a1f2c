// The gated delta rule over a time-major rollout, forwards: whole rollouts in tiles of 16 steps, and single steps.  The formulas are in
// delta.hpp.
#include "delta.hpp"

namespace mrl {
namespace delta {
namespace {

// ---------------------------------------------------------------- a few steps
// A wavefront holds 4 L columns of a head's state in registers: lane l columns 4 (l % L) on, rows l / L, l / L + 64 / L, ..., at most
// R of them.  S^T k and S^T q are summed in one pass, out = a S^T q + (q k) u follows from them, and the state is read and written once.  Sums with the
// key and the query as they come, their lengths afterwards; where one overflows, again with their powers of two taken out first.
// Bound by that: a step of 8192 environments of 4 heads of 64 x 64 takes 202 us, 5.5 TB/s, what a copy of 256 MiB gets.
template <class E, int L, int R>
__global__ __launch_bounds__(256) void steps_kernel(Delta d, int units, int column_blocks) {
    constexpr int G = 64 / L;
    const int unit = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (unit >= units) return;
    const int block = unit % column_blocks, nh = unit / column_blocks, n = nh / d.H, h = nh - n * d.H, hk = h / (d.H / d.HK);
    const int c = block * 4 * L + 4 * (lane % L), mine = d.dv - c, rg = lane / L;
    const long at = (long)nh * d.dk * d.dv + c;
    f32x4 S[R];
#pragma unroll
    for (int i = 0; i < R; ++i) S[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (d.state_in != nullptr && !is_cut(d, 0, n)) {
#pragma unroll
        for (int i = 0; i < R; ++i) S[i] = load4(d.state_in + at + (long)(rg + i * G) * d.dv, rg + i * G < d.dk ? mine : 0);
    }
    for (int t = 0; t < d.T; ++t) {
        const long row = (long)t * d.N + n;
        if (t > 0 && is_cut(d, t, n)) {
#pragma unroll
            for (int i = 0; i < R; ++i) S[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const E *q_row = (const E *)d.query + row * d.query_ld + hk * d.dk, *k_row = (const E *)d.key + row * d.key_ld + hk * d.dk;
        const f32x4 v = load4((const E *)d.value + row * d.value_ld + (long)h * d.dv + c, mine);
        float a, b, rest;
        sigmoid_pair(value_of(((const E *)d.gate)[row * d.gate_ld + h]), a, rest);
        sigmoid_pair(value_of(((const E *)d.rate)[row * d.rate_ld + h]), b, rest);
        float k[R], q[R], kk, qq, qk, k_eps = EPS, q_eps = EPS;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool there = rg + i * G < d.dk;
            k[i] = there ? value_of(k_row[rg + i * G]) : 0.0f;
            q[i] = there ? value_of(q_row[rg + i * G]) : 0.0f;
        }
        f32x4 sk, sq;
        const auto sums = [&]() {
            kk = qq = qk = 0.0f;
            sk = sq = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < R; ++i) {
                kk = fmaf(k[i], k[i], kk);
                qq = fmaf(q[i], q[i], qq);
                qk = fmaf(q[i], k[i], qk);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sk[j] = fmaf(k[i], S[i][j], sk[j]);
                    sq[j] = fmaf(q[i], S[i][j], sq[j]);
                }
            }
#pragma unroll
            for (int s = L; s < 64; s *= 2) {
                kk += __shfl_xor(kk, s);
                qq += __shfl_xor(qq, s);
                qk += __shfl_xor(qk, s);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    sk[j] += __shfl_xor(sk[j], s);
                    sq[j] += __shfl_xor(sq[j], s);
                }
            }
        };
        sums();
        // 0 where all are finite; where they are not, or no longer, once more without the rows' powers of two
        float finite = 0.0f * (kk + (qq + q_eps) * (float)d.dk + qk);
#pragma unroll
        for (int j = 0; j < 4; ++j) finite = fmaf(0.0f, sk[j], fmaf(0.0f, sq[j], finite));
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(finite != 0.0f) != 0, 0)) {
            float most_k = 0.0f, most_q = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                most_k = fmaxf(most_k, fabsf(k[i]));
                most_q = fmaxf(most_q, fabsf(q[i]));
            }
#pragma unroll
            for (int s = L; s < 64; s *= 2) {
                most_k = fmaxf(most_k, __shfl_xor(most_k, s));
                most_q = fmaxf(most_q, __shfl_xor(most_q, s));
            }
            const int k_unit = unit_of(most_k), q_unit = unit_of(most_q);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                k[i] = in_units(k[i], k_unit);
                q[i] = in_units(q[i], q_unit);
            }
            k_eps = in_units(EPS, 2 * k_unit);
            q_eps = in_units(EPS, 2 * q_unit);
            sums();
        }
        const float ks = one_over_root(kk + k_eps), qs = one_over_root((qq + q_eps) * (float)d.dk);
        f32x4 u, o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u[j] = b * fmaf(-a * ks, sk[j], v[j]);
            o[j] = qs * fmaf(ks * qk, u[j], a * sq[j]);
        }
        if (rg == 0) store4((E *)d.out + row * d.out_ld + (long)h * d.dv + c, o, mine);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float ki = ks * k[i];
#pragma unroll
            for (int j = 0; j < 4; ++j) S[i][j] = fmaf(ki, u[j], a * S[i][j]);
        }
    }
    if (d.state_out == nullptr) return;
#pragma unroll
    for (int i = 0; i < R; ++i)
        if (rg + i * G < d.dk) store4(d.state_out + at + (long)(rg + i * G) * d.dv, S[i], mine);
}

// ---------------------------------------------------------------- rollouts
// All columns of a head in a workgroup, up to 128, so that its keys are prepared once: 128 steps of 512 environments of 4 heads of 128 x 128 take 255 us in
// bf16 and 384 in fp32, 285 and 392 with four wavefronts at most (of 64 x 80 163 and 155, the other way around), 8192 steps of 2 environments 265 and 280
// (on one card; others take 260 to 286).
constexpr int MOST_WAVES = 8;
enum { OUTPUTS, STATES, ENDS };   // of all steps; ahead of every block; M and B of every part

// A workgroup goes through a part's steps of one head of one environment; each of its wavefronts keeps 16 columns of the state in registers,
// all rows of them.  What does not depend on the state (A, its inverse and P) the wavefronts prepare by halves of a tile.
// 128 steps of 1024 environments of 4 heads of 64 x 64 in fp32 take 225 us (reading and writing the rows once takes 124): the fp32 matrix cores are busy
// half of that, 213 us pass with all rows in the L2, and the rest is what a block's phases wait for each other.
template <class E, int DK, int TILES, int WHAT>
__global__ __launch_bounds__(64 * MOST_WAVES, 4) void tiles_kernel(Delta d, Parts parts, int column_groups, float *states, int blocks) {
    extern __shared__ float lds[];
    constexpr int B = DK / TILE, STEPS = TILE * TILES;
    Block<E, DK, TILES, false> block(lds);
    const int W = blockDim.x >> 6, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int g = lane >> 4, c = lane & 15, thread = threadIdx.x;
    const int number = group_number(), group = number % column_groups, at_part = number / column_groups, part = at_part % parts.count, nh = at_part / parts.count;
    const int n = nh / d.H, h = nh - n * d.H, hk = h / (d.H / d.HK), tiles = (d.dv + TILE - 1) / TILE;
    const int column_tile = group * W + w, column = column_tile * TILE + c;
    const bool live = column < d.dv;
    const long state_at = (long)nh * d.dk * d.dv + column;

    f32x4 S[B];
    if (WHAT != ENDS && parts.count > 1) {
        const float *from = parts.starts + (((long)at_part * tiles + min(column_tile, tiles - 1)) * B * 64 + lane) * 4;
#pragma unroll
        for (int i = 0; i < B; ++i) S[i] = *reinterpret_cast<const f32x4 *>(from + i * 256);
    } else {
#pragma unroll
        for (int i = 0; i < B; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int row = i * TILE + 4 * g + r;
                if (WHAT == ENDS) S[i][r] = column - tiles * TILE == row ? 1.0f : 0.0f;   // the identity's columns come behind the values'
                else S[i][r] = d.state_in != nullptr && live && row < d.dk ? d.state_in[state_at + (long)row * d.dv] : 0.0f;
            }
    }

    const E *const values = (const E *)d.value + n * d.value_ld + (long)h * d.dv + min(column, d.dv - 1);
    E *const outs = (E *)d.out + n * d.out_ld + (long)h * d.dv + column;
    int begin = part * parts.per * STEPS;   // of the block
    const int end = min(d.T, begin + parts.per * STEPS);
    if (WHAT == ENDS) {
        const int last = find_cut<true>(d, begin, end, n, (int *)lds);
        if (threadIdx.x == 0 && group == 0) parts.cuts[at_part] = last >= 0;
        if (last >= 0) {
            if (group * W >= tiles) return;   // nobody asks for M
            begin = last / STEPS * STEPS;
        }
    }
    block.span = TILE;
    for (block.t0 = begin; block.t0 < end;) {
        if (WHAT == STATES && block.t0 == begin) {
            if (column_tile < tiles) {
                float *to = states + ((((long)nh * blocks + begin / STEPS) * tiles + column_tile) * B * 64 + lane) * 4;
#pragma unroll
                for (int i = 0; i < B; ++i) *reinterpret_cast<f32x4 *>(to + i * 256) = S[i];
            }
            if (begin + STEPS >= end) return;
        }
        f32x4 V[TILES];
        anew(g, c);
        anew(thread);
        E asked[TILES][4];
        ask_values(d, block, values, (long)d.N * d.value_ld, g, asked);
        bool odd = block.template load<WHAT == OUTPUTS>(d, n, h, hk, thread);
        odd |= take_values(d, block, asked, live, g, V) | is_odd(S);
        if (__syncthreads_or(odd) && block.span == TILE) {
            block.span = 1;
            continue;   // the same block again, one step to a tile
        }
        anew(g, c);
        for (int half = w; half < block.HALVES; half += W) block.template prepare<WHAT == OUTPUTS>(d, half, g, c);
        __syncthreads();
#pragma unroll 1
        for (int tile = 0; tile < TILES; ++tile) {
            if (block.t0 + tile * block.span >= d.T) break;
            anew(g, c);
            if (block.cut_ahead(tile)) {
#pragma unroll
                for (int i = 0; i < B; ++i) S[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            f32x4 v = V[0], o;
#pragma unroll
            for (int i = 1; i < TILES; ++i) v = tile == i ? V[i] : v;
            const Pieces<E, DK> pieces(S);
            const f32x4 sk = block.keys.ask(tile, g, c, pieces);
            if (WHAT == OUTPUTS) o = block.queries.ask(tile, g, c, pieces);
            const f32x4 u = solve(block, tile, g, c, v, sk);
            if (WHAT == OUTPUTS) {
                o *= block.four(block.query_reads, tile, g);
                o = mfma16(*reinterpret_cast<const f32x4 *>(block.Ps + tile * TILE * SIDE + c * SIDE + 4 * g), u, o);
                settle(o);
            }
            go_on(block, tile, g, c, u, S);
            if (WHAT == OUTPUTS) store_values(d, block, outs, (long)d.N * d.out_ld, live, tile, g, o);
        }
        block.t0 += TILES * block.span;
        if (block.t0 >= begin + STEPS) {
            begin = block.t0;
            block.span = TILE;
        }
        __syncthreads();
    }
    if (WHAT == ENDS) {
        if (column_tile >= tiles + B) return;
        float *to = parts.ends + (((long)at_part * (tiles + B) + column_tile) * B * 64 + lane) * 4;
#pragma unroll
        for (int i = 0; i < B; ++i) *reinterpret_cast<f32x4 *>(to + i * 256) = S[i];
    }
    if (WHAT != OUTPUTS || d.state_out == nullptr || !live || part != parts.count - 1) return;
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = i * TILE + 4 * g + r;
            if (row < d.dk) d.state_out[state_at + (long)row * d.dv] = S[i][r];
        }
}

// Through the parts: S <- M S + B, from the first to the last, S ahead of each to parts.starts; BACK: S <- M^T S + B from the last to the first, B in
// `local`, S behind each to parts.starts.  A workgroup 16 columns, a wavefront 16 rows of them; S changes hands through LDS.
template <int DK, bool BACK>
__global__ __launch_bounds__(DK * 4) void parts_kernel(Delta d, Parts parts, const float *first, const float *local) {
    __shared__ f32x4 S[2][DK / TILE][64];
    __shared__ int cuts[MOST_PARTS];
    constexpr int B = DK / TILE;
    const int tiles = (d.dv + TILE - 1) / TILE, column_tile = blockIdx.x % tiles, nh = blockIdx.x / tiles;
    const int i = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15, column = column_tile * TILE + c;
    for (int part = threadIdx.x; part < parts.count; part += DK * 4) cuts[part] = parts.cuts[(long)nh * parts.count + part];
    f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f}, next, m[B];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = i * TILE + 4 * g + r;
        if (first != nullptr && column < d.dv && row < d.dk) s[r] = first[((long)nh * d.dk + row) * d.dv + column];
    }
    __syncthreads();
    const auto part_of = [&](int step) { return BACK ? parts.count - 1 - step : step; };
    const auto ask = [&](int step) {   // B and M of a step, while the one ahead of it is worked out
        if (step >= parts.count - 1) return;
        const int part = part_of(step);
        const long at = (long)nh * parts.count + part;
        const float *const ends = parts.ends + at * (tiles + B) * B * 256, *const M = ends + (long)tiles * B * 256;   // M: [column tile][row tile][lane][4]
        next = *reinterpret_cast<const f32x4 *>(BACK ? local + (((at * tiles + column_tile) * B + i) * 64 + lane) * 4 : ends + ((column_tile * B + i) * 64 + lane) * 4);
        if (cuts[part]) return;
#pragma unroll
        for (int k = 0; k < B; ++k) {
            // the operand's row c and contracted 4 g .. 4 g + 3: of M^T four neighbouring rows of a column of M, as they lie; of M a row's columns
            if (BACK) m[k] = *reinterpret_cast<const f32x4 *>(M + ((i * B + k) * 64 + lane) * 4);
            else
#pragma unroll
                for (int r = 0; r < 4; ++r) m[k][r] = M[((k * B + i) * 64 + 16 * (c >> 2) + 4 * g + r) * 4 + (c & 3)];
        }
    };
    ask(0);
    const auto put = [&](int step) { *reinterpret_cast<f32x4 *>(parts.starts + ((((long)nh * parts.count + part_of(step)) * tiles + column_tile) * B + i) * 256 + lane * 4) = s; };
    for (int step = 0; step < parts.count - 1; ++step) {
        put(step);
        f32x4 after = next, mine[B];
#pragma unroll
        for (int k = 0; k < B; ++k) mine[k] = m[k];
        ask(step + 1);
        const bool goes_on = !cuts[part_of(step)];
        f32x4 (&here)[B][64] = S[step & 1];
        if (goes_on) here[i][lane] = s;
        __syncthreads();   // in every step, also where a cut leaves the buffer as it was: who writes it again is behind the next step's, and all have read it by then
        if (goes_on) {
#pragma unroll
            for (int k = 0; k < B; ++k) after = mfma16(mine[k], here[k][lane], after);
            settle(after);
        }
        s = after;
    }
    put(parts.count - 1);
}

// Up to here the state's own pass is ahead of the tiles: 4 steps of 2048 environments take 72 us (108 by tiles), 2 of 4096 112 (195); 16 of 1024 take 58 by
// tiles, four times the former's work.
constexpr int FEW_STEPS = 4;
template <class E, int L>
void launch_steps(const mrl_ctx *ctx, const Delta &d) {
    const int blocks = (d.dv + 4 * L - 1) / (4 * L), units = d.N * d.H * blocks, rows = (d.dk + 64 / L - 1) / (64 / L);
    const dim3 grid((units + 3) / 4), block(256);
    if (rows <= 4) hipLaunchKernelGGL((steps_kernel<E, L, 4>), grid, block, 0, ctx->stream, d, units, blocks);
    else if (rows <= 8) hipLaunchKernelGGL((steps_kernel<E, L, 8>), grid, block, 0, ctx->stream, d, units, blocks);
    else if (rows <= 16) hipLaunchKernelGGL((steps_kernel<E, L, 16>), grid, block, 0, ctx->stream, d, units, blocks);
    else hipLaunchKernelGGL((steps_kernel<E, L, 32>), grid, block, 0, ctx->stream, d, units, blocks);
}
template <class E, int DK, int TILES, int WHAT>
void launch_tiles(const mrl_ctx *ctx, const Delta &d, const Parts &p, float *states = nullptr, int blocks = 0) {
    const int tiles = column_tiles(d.dv) + (WHAT == ENDS ? DK / TILE : 0), waves = std::min(MOST_WAVES, tiles), groups = (tiles + waves - 1) / waves;
    hipLaunchKernelGGL((tiles_kernel<E, DK, TILES, WHAT>), dim3(d.N * d.H * p.count * groups), dim3(64 * waves), sizeof(float) * rows_floats<E>(DK, TILES, false), ctx->stream, d, p,
                       groups, states, blocks);
}
template <class E, int DK, int TILES>
void launch_starts(const mrl_ctx *ctx, const Delta &d, const Parts &p) {
    launch_tiles<E, DK, TILES, ENDS>(ctx, d, p);
    hipLaunchKernelGGL((parts_kernel<DK, false>), dim3(d.N * d.H * column_tiles(d.dv)), dim3(DK * 4), 0, ctx->stream, d, p, d.state_in, nullptr);
}
template <class E, int DK>
void launch_rollout(const mrl_ctx *ctx, const Delta &d, const Parts &p) {
    if (p.count > 1) launch_starts<E, DK, tiles_forward(DK)>(ctx, d, p);
    launch_tiles<E, DK, tiles_forward(DK), OUTPUTS>(ctx, d, p);
}
template <class E>
void launch(const mrl_ctx *ctx, const Delta &d, const Parts &p) {
    if (d.T <= FEW_STEPS) return d.dv <= 32 ? launch_steps<E, 8>(ctx, d) : launch_steps<E, 16>(ctx, d);
    switch (padded(d.dk)) {
        case 16: return launch_rollout<E, 16>(ctx, d, p);
        case 32: return launch_rollout<E, 32>(ctx, d, p);
        case 64: return launch_rollout<E, 64>(ctx, d, p);
        default: return launch_rollout<E, 128>(ctx, d, p);
    }
}

struct Plan {
    Parts parts;
    size_t bytes;
};
Plan plan_of(const mrl_ctx *ctx, const mrl_delta *r) {
    Plan p = {};
    if (r->T <= FEW_STEPS || r->N == 0) return p;
    p.parts = parts_of(ctx, r, tiles_forward(padded(r->key_dim)));
    p.bytes = sizeof(float) * (ends_floats(r, p.parts) + starts_floats(r, p.parts) + cuts_floats(r, p.parts));
    return p;
}

}  // namespace

size_t forward_bytes(const mrl_ctx *ctx, const mrl_delta *r) { return plan_of(ctx, r).bytes; }

// no step at all: the state goes through as it is
__global__ __launch_bounds__(256) void pass_state_kernel(const float *from, float *to, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) to[i] = from ? from[i] : 0.0f;
}

namespace {
template <class E, int DK>
void backward_starts(const mrl_ctx *ctx, const Delta &d, const Parts &p) { launch_starts<E, DK, tiles_backward(DK)>(ctx, d, p); }
template <class E, int DK>
void backward_states(const mrl_ctx *ctx, const Delta &d, const Parts &p, float *states, int blocks) {
    launch_tiles<E, DK, tiles_backward(DK), STATES>(ctx, d, p, states, blocks);
}
template <class E>
void backward_starts(const mrl_ctx *ctx, const Delta &d, const Parts &p) {
    switch (padded(d.dk)) {
        case 16: return backward_starts<E, 16>(ctx, d, p);
        case 32: return backward_starts<E, 32>(ctx, d, p);
        case 64: return backward_starts<E, 64>(ctx, d, p);
        default: return backward_starts<E, 128>(ctx, d, p);
    }
}
template <class E>
void backward_states(const mrl_ctx *ctx, const Delta &d, const Parts &p, float *states, int blocks) {
    switch (padded(d.dk)) {
        case 16: return backward_states<E, 16>(ctx, d, p, states, blocks);
        case 32: return backward_states<E, 32>(ctx, d, p, states, blocks);
        case 64: return backward_states<E, 64>(ctx, d, p, states, blocks);
        default: return backward_states<E, 128>(ctx, d, p, states, blocks);
    }
}
template <int DK>
void grad_ends(const mrl_ctx *ctx, const Delta &d, const Parts &p, const float *grad_state_out, const float *local) {
    hipLaunchKernelGGL((parts_kernel<DK, true>), dim3(d.N * d.H * column_tiles(d.dv)), dim3(DK * 4), 0, ctx->stream, d, p, grad_state_out, local);
}
}  // namespace

int launch_starts(const mrl_ctx *ctx, int dtype, const Delta &d, const Parts &p) {
    if (dtype == MRL_F32) backward_starts<float>(ctx, d, p);
    else backward_starts<bf16_t>(ctx, d, p);
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}
int launch_states(const mrl_ctx *ctx, int dtype, const Delta &d, const Parts &p, float *states, int blocks) {
    if (dtype == MRL_F32) backward_states<float>(ctx, d, p, states, blocks);
    else backward_states<bf16_t>(ctx, d, p, states, blocks);
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}
int launch_grad_ends(const mrl_ctx *ctx, const Delta &d, const Parts &p, const float *grad_state_out, const float *local) {
    switch (padded(d.dk)) {
        case 16: grad_ends<16>(ctx, d, p, grad_state_out, local); break;
        case 32: grad_ends<32>(ctx, d, p, grad_state_out, local); break;
        case 64: grad_ends<64>(ctx, d, p, grad_state_out, local); break;
        default: grad_ends<128>(ctx, d, p, grad_state_out, local); break;
    }
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}

int check_sizes(const char *who, const mrl_delta *r) {
    MRL_CHECK_ARG(r->dtype == MRL_F32 || r->dtype == MRL_BF16, "%s: unknown element type %d", who, r->dtype);
    MRL_CHECK_ARG(r->T >= 0 && r->N >= 0, "%s: negative size", who);
    MRL_CHECK_ARG(r->T < 1 << 30, "%s: %d steps are 2^30 or more", who, r->T);
    MRL_CHECK_ARG(r->heads >= 1 && r->key_heads >= 1 && r->heads % r->key_heads == 0, "%s: %d heads on %d key heads", who, r->heads, r->key_heads);
    MRL_CHECK_ARG(r->key_dim >= 1 && r->key_dim <= MOST_DIM && r->value_dim >= 1 && r->value_dim <= MOST_DIM,
                  "%s: key_dim %d and value_dim %d: 1 to %d expected", who, r->key_dim, r->value_dim, MOST_DIM);
    MRL_CHECK_ARG((long)r->N * r->heads < 1L << 22, "%s: %d environments of %d heads are 2^22 states or more", who, r->N, r->heads);
    MRL_CHECK_ARG(r->heads < 1 << 22, "%s: %d heads are 2^22 or more", who, r->heads);
    return MRL_OK;
}
int check(const char *who, const mrl_ctx *ctx, const mrl_delta *r) {
    MRL_CHECK_ARG(ctx && r, "%s: NULL ctx or description", who);
    const int rc = check_sizes(who, r);
    if (rc != MRL_OK) return rc;
    if (r->T == 0 || r->N == 0) return MRL_OK;
    MRL_CHECK_ARG(r->query && r->key && r->value && r->gate && r->rate, "%s: NULL buffer", who);
    const long k_width = (long)r->key_heads * r->key_dim, v_width = (long)r->heads * r->value_dim;
    MRL_CHECK_ARG(r->query_ld >= k_width && r->key_ld >= k_width && r->value_ld >= v_width && r->gate_ld >= r->heads && r->rate_ld >= r->heads,
                  "%s: a row stride is smaller than the row", who);
    return MRL_OK;
}

Delta describe(const mrl_delta *r) {
    Delta d = {};
    d.T = r->T; d.N = r->N; d.H = r->heads; d.HK = r->key_heads; d.dk = r->key_dim; d.dv = r->value_dim;
    d.query = r->query; d.key = r->key; d.value = r->value; d.gate = r->gate; d.rate = r->rate;
    d.query_ld = r->query_ld; d.key_ld = r->key_ld; d.value_ld = r->value_ld; d.gate_ld = r->gate_ld; d.rate_ld = r->rate_ld;
    d.dones = r->dones; d.prev_dones = r->prev_dones; d.state_in = r->state_in;
    return d;
}

}  // namespace delta
}  // namespace mrl

extern "C" {

int mrl_delta_forward(mrl_ctx *ctx, const mrl_delta *r, void *out, int64_t out_ld, float *state_out, void *workspace,
                      uint64_t workspace_bytes) {
    using namespace mrl;
    using namespace mrl::delta;
    const char *who = "mrl_delta_forward";
    const int rc = check(who, ctx, r);
    if (rc != MRL_OK) return rc;
    if (r->N == 0) return MRL_OK;
    const long states = (long)r->N * r->heads * r->key_dim * r->value_dim;
    MRL_CHECK_ARG(r->T == 0 || out, "%s: NULL buffer", who);
    MRL_CHECK_ARG(r->T == 0 || out_ld >= (long)r->heads * r->value_dim, "%s: a row stride is smaller than the row", who);
    const int64_t size = r->dtype == MRL_F32 ? 4 : 2, rows = (int64_t)r->T * r->N;
    const auto of = [&](const char *name, const void *at, long width, long ld) { return Region(name, at, rows, size * width, size * ld); };
    const long k_width = (long)r->key_heads * r->key_dim, v_width = (long)r->heads * r->value_dim;
    const Plan plan = plan_of(ctx, r);
    MRL_CHECK_ARG(workspace_bytes >= plan.bytes && (plan.bytes == 0 || workspace != nullptr), "%s: the workspace holds %llu bytes, need %llu", who,
                  (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)plan.bytes);
    MRL_CHECK_ARG(plan.bytes == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: the workspace must be 16-byte aligned", who);
    const int apart = check_apart(who, {of("out", out, v_width, out_ld), Region("state_out", state_out, 4 * states), Region("the workspace", plan.bytes ? workspace : nullptr, (int64_t)plan.bytes)},
                                  {of("query", r->query, k_width, r->query_ld), of("key", r->key, k_width, r->key_ld), of("value", r->value, v_width, r->value_ld),
                                   of("gate", r->gate, r->heads, r->gate_ld), of("rate", r->rate, r->heads, r->rate_ld), Region("dones", r->dones, 4 * rows),
                                   Region("prev_dones", r->prev_dones, 4LL * r->N), Region("state_in", r->state_in == state_out ? nullptr : r->state_in, 4 * states)});
    if (apart != MRL_OK) return apart;
    OnDevice on(ctx);
    if (r->T == 0) {
        if (state_out != nullptr && state_out != r->state_in)
            hipLaunchKernelGGL(pass_state_kernel, dim3((int)std::min<long>((states + 255) / 256, 4096)), dim3(256), 0, ctx->stream, r->state_in, state_out, states);
        MRL_CHECK_LAUNCH();
        return MRL_OK;
    }
    Delta d = describe(r);
    d.out = out; d.out_ld = out_ld; d.state_out = state_out;
    Parts p = plan.parts;
    p.ends = (float *)workspace;
    p.starts = p.ends + ends_floats(r, p);
    p.cuts = (int *)(p.starts + starts_floats(r, p));
    if (r->dtype == MRL_F32) launch<float>(ctx, d, p);
    else launch<bf16_t>(ctx, d, p);
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}

}  // extern "C"
