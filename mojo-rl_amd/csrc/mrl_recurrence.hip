// Gated linear recurrence over a time-major rollout, cut where episodes end, and its gradient:
//
//   a = sigmoid(gate),  h[t] = a[t] h'[t-1] + (1 - a[t]) x[t],   h'[t-1] = 0 where the step before ended an episode, h[t-1] elsewhere
//   d[t] = dh[t] + G[t+1],  G[t] = a[t] d[t] (0 where h' is cut),   dx = (1 - a) d,   dgate = a (1 - a) (h' - x) d
//
// Both are first-order linear recurrences per channel, s <- A s + B, one forwards and one backwards in time, and both are bound by
// memory: forward 3 values per element (12 bytes in fp32), backward 6.  What the kernels do about it is have enough loads in
// flight at every shape.  A lane holds V = 4 neighbouring channels of one environment, a wavefront 256 of them.  Where that alone
// fills the card (a rollout of many environments), a wavefront goes through the steps by itself, L steps' loads at a time.  With
// fewer channels a workgroup's W wavefronts take L consecutive steps each of a tile of W L: a wavefront's steps compose to one
// (A, B), these are exchanged through LDS, and each wavefront then repeats its steps from its own first state, so every state is
// the result of the formula above on the state before it and the inputs are read once.  With a few channels only, the time axis
// is also split into S segments over workgroups: a first launch leaves every segment's (A, B) in a workspace, the second starts each
// segment from those before it.  That reads gate and value twice, the second time out of the caches where they fit.
//
// A cut is a selection, never a product with 0: an infinity or NaN behind it goes nowhere.  In the composed coefficients A = 0
// says so; a product of gates that underflows stays at the smallest subnormal instead.
// States and sums are fp32 whatever the type; in bf16 only gate, value, output and their gradients are rounded, once, when stored.
#include "mrl_host.hpp"
#include "mrl_device.hpp"

namespace mrl {
namespace {

constexpr float TINY = 0x1p-149f;
constexpr int MAX_WAVES = 16;

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned short u16x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef __bf16 v4bf __attribute__((ext_vector_type(4)));

struct bf16_t { unsigned short bits; };

MRL_DEV void load_n(const float *p, float (&x)[4]) {
    const f32x4u v = *reinterpret_cast<const f32x4u *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = v[i];
}
MRL_DEV void load_n(const bf16_t *p, float (&x)[4]) {
    const u16x4u v = *reinterpret_cast<const u16x4u *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float((unsigned)v[i] << 16);
}
MRL_DEV void load_n(const float *p, float (&x)[1]) { x[0] = *p; }
MRL_DEV void load_n(const bf16_t *p, float (&x)[1]) { x[0] = __uint_as_float((unsigned)p->bits << 16); }

// the elements from `skip` on (the ones before belong to the neighbouring lane)
template <int V>
MRL_DEV void store_n(float *p, const float (&x)[V], int skip) {
    if (V == 4 && skip == 0) {
        *reinterpret_cast<f32x4u *>(p) = f32x4u{x[0], x[1], x[V - 2], x[V - 1]};
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i >= skip) p[i] = x[i];
    }
}
template <int V>
MRL_DEV void store_n(bf16_t *p, const float (&x)[V], int skip) {
    if (V == 4) {
        const v4bf h = __builtin_convertvector((v4f{x[0], x[V > 1 ? 1 : 0], x[V > 2 ? 2 : 0], x[V - 1]}), v4bf);
        const u16x4u v = __builtin_bit_cast(u16x4u, h);
        if (skip == 0) {
            *reinterpret_cast<u16x4u *>(p) = v;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i >= skip) p[i].bits = v[i];
        }
    } else {
        p->bits = __builtin_bit_cast(unsigned short, (__bf16)x[0]);
    }
}

// a = sigmoid(g) and rest = 1 - a, both to a few roundings of their own value.  exp(-|g|) = 2^y (1 + r ln 2) with r what rounding
// y = -|g| / ln 2 left; beyond 128 both ends are 0 and 1 in fp32 (and the difference of infinities would be NaN).
MRL_DEV void gates(float g, float &a, float &rest) {
    float m = fabsf(g);
    m = m > 128.0f ? 128.0f : m;   // (NaN stays)
    const float y = -m * 1.44269502f;
    const float r = fmaf(-m, 1.44269502f, -y) - m * 1.92596299e-8f;
    float e = __builtin_amdgcn_exp2f(y);
    e = fmaf(e, r * 0.693147182f, e);
    const float inv = __builtin_amdgcn_rcpf(1.0f + e), low = e * inv;
    a = g >= 0.0f ? inv : low;
    rest = g >= 0.0f ? low : inv;
}

struct Scan {
    int T, N, D, lanes_per_row, W, segments, segment_steps;
    int groups;              // of 64 lanes
    long lanes;              // N * lanes_per_row
    const void *gate, *value, *out, *grad_out;
    long gate_ld, value_ld, out_ld, grad_out_ld, grad_gate_ld, grad_value_ld;
    const float *dones, *prev_dones;
    const float *first;      // forward: state_in; backward: grad_state_out
    const float *state_in;   // backward
    float *last;             // forward: state_out; backward: grad_state_in
    void *dst, *dst2;        // forward: out; backward: grad_gate, grad_value
    float *ws;               // [segments][2][lanes * V] (A, B), then [lanes * V]: the first state
};

// What a lane works on: V channels from column d of environment n.  The last lane of a row whose width is no multiple of V starts
// early enough to read V channels, and stores (and owns) those from `skip` on only.
struct Place {
    long q;
    int n, d, skip;
    bool live;
};
template <int V>
MRL_DEV Place place(const Scan &s, int group) {
    Place p;
    p.q = (long)group * 64 + threadIdx.x;
    p.live = p.q < s.lanes;
    if (!p.live) p.q = s.lanes - 1;
    p.n = (int)(p.q / s.lanes_per_row);
    p.d = (int)(p.q - (long)p.n * s.lanes_per_row) * V;
    p.skip = 0;
    if (p.d + V > s.D) {
        p.skip = p.d + V - s.D;
        p.d = s.D - V;
    }
    return p;
}

// The flag of the step before t for environment n, 0 where the caller gave none: the load itself is from memory that is there
// whatever t is, so that a tile's loads stand together without a branch or a wait among them.
MRL_DEV float flag_ahead(const Scan &s, long t, int n) {
    const float *row = t > 0 ? (s.dones ? s.dones + (t - 1) * s.N : s.prev_dones) : (s.prev_dones ? s.prev_dones : s.dones);
    return row[n];
}
MRL_DEV bool is_cut(const Scan &s, long t, float flag) { return (t > 0 ? s.dones : s.prev_dones) != nullptr && flag > 0.5f; }

template <int V>
MRL_DEV void compose(float (&state)[V], const float *A, const float *B) {
#pragma unroll
    for (int i = 0; i < V; ++i) state[i] = A[i] == 0.0f ? B[i] : fmaf(A[i], state[i], B[i]);
}

template <int V>
MRL_DEV void put(float *p, const float (&x)[V]) {
    if (V == 4) *reinterpret_cast<v4f *>(p) = v4f{x[0], x[V > 1 ? 1 : 0], x[V > 2 ? 2 : 0], x[V - 1]};
    else p[0] = x[0];
}
template <int V>
MRL_DEV void get(const float *p, float (&x)[V]) {
    if (V == 4) {
        const v4f v = *reinterpret_cast<const v4f *>(p);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = v[i];
    } else {
        x[0] = p[0];
    }
}

// The state ahead of wavefront w's share, from the state ahead of the workgroup's and the shares' (A, B) in LDS; `carry` becomes
// the state behind all of them.
template <int V>
MRL_DEV void through_waves(const float *lds, int W, int w, float (&carry)[V], float (&mine)[V]) {
    for (int i = 0; i < W; ++i) {
        if (i == w) {
#pragma unroll
            for (int k = 0; k < V; ++k) mine[k] = carry[k];
        }
        float A[V], B[V];
        get(lds + ((size_t)i * 2 * 64 + threadIdx.x) * V, A);
        get(lds + (((size_t)i * 2 + 1) * 64 + threadIdx.x) * V, B);
        compose(carry, A, B);
    }
}
template <int V>
MRL_DEV void leave(float *lds, int w, const float (&A)[V], const float (&B)[V]) {
    put(lds + ((size_t)w * 2 * 64 + threadIdx.x) * V, A);
    put(lds + (((size_t)w * 2 + 1) * 64 + threadIdx.x) * V, B);
}

// step number p of the scan: time p forwards, T - 1 - p backwards
template <bool BACK>
MRL_DEV long time_of(const Scan &s, long p) { return BACK ? s.T - 1 - p : p; }

// One step's (A, B) on top of those before it.  The backward scan's state is G[t+1], what goes into step t from behind it.
template <bool BACK, int V>
MRL_DEV void add_step(float (&A)[V], float (&B)[V], float &low, bool cut, const float (&g)[V], const float (&x)[V]) {
    low = cut ? 0.0f : low;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float a, rest;
        gates(g[i], a, rest);
        const float after = BACK ? a * (B[i] + x[i]) : fmaf(a, B[i], rest * x[i]);
        B[i] = cut ? (BACK ? 0.0f : rest * x[i]) : after;
        A[i] = cut ? 0.0f : fmaxf(A[i] * a, low);
    }
}

// A segment's (A, B): every wavefront composes the steps of its own share, the first one the shares.
template <class E, int V, int L, bool BACK>
__global__ __launch_bounds__(64 * MAX_WAVES) void scan_segments_kernel(Scan s) {
    extern __shared__ float lds[];
    const Place at = place<V>(s, blockIdx.x);
    const int w = threadIdx.y, seg = blockIdx.y;
    const long begin = (long)seg * s.segment_steps, end = min((long)s.T, begin + s.segment_steps);
    const long share = (end - begin + s.W - 1) / s.W, from = min(end, begin + w * share), to = min(end, from + share);
    const E *gate = (const E *)s.gate + (long)at.n * s.gate_ld + at.d;
    const E *value = BACK ? (const E *)s.grad_out + (long)at.n * s.grad_out_ld + at.d : (const E *)s.value + (long)at.n * s.value_ld + at.d;
    const long gate_step = (long)s.N * s.gate_ld, value_step = (long)s.N * (BACK ? s.grad_out_ld : s.value_ld);
    const bool flagged = s.dones != nullptr || s.prev_dones != nullptr;
    float A[V], B[V], low = TINY;
#pragma unroll
    for (int i = 0; i < V; ++i) { A[i] = 1.0f; B[i] = 0.0f; }
    for (long p0 = from; p0 < to; p0 += L) {
        float g[L][V], x[L][V], flag[L] = {};
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const long t = time_of<BACK>(s, min(p0 + j, to - 1));
            load_n(gate + t * gate_step, g[j]);
            load_n(value + t * value_step, x[j]);
        }
        if (flagged) {
#pragma unroll
            for (int j = 0; j < L; ++j) flag[j] = flag_ahead(s, time_of<BACK>(s, min(p0 + j, to - 1)), at.n);
        }
#pragma unroll
        for (int j = 0; j < L; ++j)
            if (p0 + j < to) add_step<BACK>(A, B, low, is_cut(s, time_of<BACK>(s, p0 + j), flag[j]), g[j], x[j]);
    }
    if (s.W > 1) leave(lds, w, A, B);
    __syncthreads();
    if (w != 0 || !at.live) return;
    float total[V];
    for (int i = 1; i < s.W; ++i) {
        float A1[V], B1[V];
        get(lds + ((size_t)i * 2 * 64 + threadIdx.x) * V, A1);
        get(lds + (((size_t)i * 2 + 1) * 64 + threadIdx.x) * V, B1);
        compose(B, A1, B1);
#pragma unroll
        for (int k = 0; k < V; ++k) A[k] = A1[k] == 0.0f || A[k] == 0.0f ? 0.0f : fmaxf(A[k] * A1[k], TINY);
    }
    const long row = s.lanes * V;
    put(s.ws + ((long)seg * 2) * row + at.q * V, A);
    put(s.ws + ((long)seg * 2 + 1) * row + at.q * V, B);
    if (seg == 0) {   // the first state, which `last` may overwrite while segments still start
#pragma unroll
        for (int k = 0; k < V; ++k) total[k] = 0.0f;
        if (s.first != nullptr) load_n(s.first + (long)at.n * s.D + at.d, total);
        put(s.ws + (long)s.segments * 2 * row + at.q * V, total);
    }
}

// The scan itself.  PART: a workgroup's W wavefronts share the steps of one group of lanes; otherwise every wavefront has a
// group of its own.
template <class E, int V, int L, bool BACK, bool PART>
__global__ __launch_bounds__(PART ? 64 * MAX_WAVES : 256) void scan_kernel(Scan s) {
    extern __shared__ float lds[];
    const int w = PART ? threadIdx.y : 0, W = PART ? s.W : 1, seg = PART ? blockIdx.y : 0;
    const int group = PART ? blockIdx.x : blockIdx.x * blockDim.y + threadIdx.y;
    if (!PART && group >= s.groups) return;
    const Place at = place<V>(s, group);
    const long begin = PART ? (long)seg * s.segment_steps : 0, end = PART ? min((long)s.T, begin + s.segment_steps) : s.T;
    const int half = W * 2 * 64 * V;
    const bool flagged = s.dones != nullptr || s.prev_dones != nullptr;
    int buffer = 0;
    float carry[V], mine[V];
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = mine[i] = 0.0f;
    if (PART && s.segments > 1) {
        // each wavefront composes its share of the segments ahead of this one
        const long row = s.lanes * V;
        get(s.ws + (long)s.segments * 2 * row + at.q * V, carry);
        const int share = (seg + W - 1) / W, from = min(seg, w * share), to = min(seg, from + share);
        float A[V], B[V];
#pragma unroll
        for (int i = 0; i < V; ++i) { A[i] = 1.0f; B[i] = 0.0f; }
        for (int k = from; k < to; ++k) {
            float A1[V], B1[V];
            get(s.ws + (long)k * 2 * row + at.q * V, A1);
            get(s.ws + ((long)k * 2 + 1) * row + at.q * V, B1);
            compose(B, A1, B1);
#pragma unroll
            for (int i = 0; i < V; ++i) A[i] = A1[i] == 0.0f || A[i] == 0.0f ? 0.0f : fmaxf(A[i] * A1[i], TINY);
        }
        leave(lds, w, A, B);
        __syncthreads();
        through_waves(lds, W, w, carry, mine);
        buffer = 1;
    } else if (s.first != nullptr) {
        load_n(s.first + (long)at.n * s.D + at.d, carry);
    }
    const E *gate = (const E *)s.gate + (long)at.n * s.gate_ld + at.d;
    const E *value = (const E *)s.value + (long)at.n * s.value_ld + at.d;
    const long gate_step = (long)s.N * s.gate_ld, value_step = (long)s.N * s.value_ld, out_step = (long)s.N * s.out_ld;
    const E *out = (const E *)s.out + (long)at.n * s.out_ld + at.d;
    const E *grad = (const E *)s.grad_out + (long)at.n * s.grad_out_ld + at.d;
    const long grad_step = (long)s.N * s.grad_out_ld, dgate_step = (long)s.N * s.grad_gate_ld, dvalue_step = (long)s.N * s.grad_value_ld;
    E *dst = (E *)s.dst + (long)at.n * (BACK ? s.grad_gate_ld : s.out_ld) + at.d;
    E *dst2 = (E *)s.dst2 + (long)at.n * s.grad_value_ld + at.d;
    for (long tile = begin; tile < end; tile += (long)W * L) {
        const long p0 = tile + w * L;
        float g[L][V], x[L][V], dh[BACK ? L : 1][V], h1[BACK ? L : 1][V];
        float flag[L] = {};
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const long t = time_of<BACK>(s, min(p0 + j, end - 1));
            load_n(gate + t * gate_step, g[j]);
            load_n(value + t * value_step, x[j]);
            if (BACK) {
                load_n(grad + t * grad_step, dh[j]);
                load_n(out + max(t - 1, 0L) * out_step, h1[j]);
            }
        }
        if (flagged) {
#pragma unroll
            for (int j = 0; j < L; ++j) flag[j] = flag_ahead(s, time_of<BACK>(s, min(p0 + j, end - 1)), at.n);
        }
        if (BACK && time_of<BACK>(s, min(p0 + L, end) - 1) == 0) {   // the tile's last step is the first of the rollout
#pragma unroll
            for (int j = 0; j < L; ++j) {
                if (p0 + j != end - 1) continue;
#pragma unroll
                for (int i = 0; i < V; ++i) h1[BACK ? j : 0][i] = 0.0f;
                if (s.state_in != nullptr) load_n(s.state_in + (long)at.n * s.D + at.d, h1[BACK ? j : 0]);
            }
        }
        if (PART) {
            float A[V], B[V], low = TINY;
#pragma unroll
            for (int i = 0; i < V; ++i) { A[i] = 1.0f; B[i] = 0.0f; }
#pragma unroll
            for (int j = 0; j < L; ++j)
                if (p0 + j < end)
                    add_step<BACK>(A, B, low, is_cut(s, time_of<BACK>(s, p0 + j), flag[j]), g[j], BACK ? dh[BACK ? j : 0] : x[j]);
            leave(lds + buffer * half, w, A, B);
            __syncthreads();   // (the buffers alternate: the next tile's values go where nobody reads any more)
            through_waves(lds + buffer * half, W, w, carry, mine);
            buffer ^= 1;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) mine[i] = carry[i];
        }
#pragma unroll
        for (int j = 0; j < L; ++j) {
            if (p0 + j >= end) break;
            const long t = time_of<BACK>(s, p0 + j);
            const bool cut = is_cut(s, t, flag[j]);
            float y[V], y2[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float a, rest;
                gates(g[j][i], a, rest);
                if (BACK) {
                    const float d = dh[BACK ? j : 0][i] + mine[i];
                    y2[i] = rest * d;
                    y[i] = a * rest * ((cut ? 0.0f : h1[BACK ? j : 0][i]) - x[j][i]) * d;
                    mine[i] = cut ? 0.0f : a * d;
                } else {
                    const float b = rest * x[j][i];
                    mine[i] = y[i] = cut ? b : fmaf(a, mine[i], b);
                }
            }
            if (at.live) {
                store_n(dst + t * (BACK ? dgate_step : out_step), y, at.skip);
                if (BACK) store_n(dst2 + t * dvalue_step, y2, at.skip);
                if (p0 + j == s.T - 1 && s.last != nullptr) store_n(s.last + (long)at.n * s.D + at.d, mine, at.skip);
            }
        }
        if (!PART) {
#pragma unroll
            for (int i = 0; i < V; ++i) carry[i] = mine[i];
        }
    }
}

// no step at all: the state goes through as it is
__global__ __launch_bounds__(256) void pass_state_kernel(const float *from, float *to, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) to[i] = from ? from[i] : 0.0f;
}

// How a scan is laid out over the card.
struct Plan {
    int V, lanes_per_row, W, segments, segment_steps, groups;
    long lanes;
    size_t bytes;
};
constexpr int STEPS = 4;   // L of the kernels with more than one step
Plan plan_of(const mrl_ctx *ctx, int T, int N, int D) {
    Plan p;
    p.V = D >= 4 ? 4 : 1;
    p.lanes_per_row = (D + p.V - 1) / p.V;
    p.lanes = (long)N * p.lanes_per_row;
    p.groups = (int)((p.lanes + 63) / 64);
    p.W = 1;
    p.segments = 1;
    const long want = 8L * ctx->n_cus;   // wavefronts
    while (p.W < MAX_WAVES && (long)p.groups * p.W < want && (long)p.W * STEPS < T) p.W *= 2;
    const long tile = (long)p.W * STEPS, tiles = (T + tile - 1) / tile;
    if (p.W == MAX_WAVES && (long)p.groups * p.W < want && tiles >= 4) {
        const long most = std::min<long>(tiles / 2, want / ((long)p.groups * p.W));
        const long per = (tiles + most - 1) / most;
        p.segments = (int)((tiles + per - 1) / per);
        p.segment_steps = (int)(per * tile);
    }
    if (p.segments == 1) p.segment_steps = T;
    p.bytes = p.segments > 1 ? sizeof(float) * (size_t)p.lanes * p.V * (2 * (size_t)p.segments + 1) : 0;
    return p;
}

template <class E, int V, bool BACK>
void launch(const mrl_ctx *ctx, const Scan &s) {
    if (s.W == 1) {
        const int per = s.groups >= 4 * ctx->n_cus ? 4 : 1;
        const dim3 grid((s.groups + per - 1) / per), block(64, per);
        if (s.T == 1) hipLaunchKernelGGL((scan_kernel<E, V, 1, BACK, false>), grid, block, 0, ctx->stream, s);
        else hipLaunchKernelGGL((scan_kernel<E, V, STEPS, BACK, false>), grid, block, 0, ctx->stream, s);
        return;
    }
    const dim3 grid(s.groups, s.segments), block(64, s.W);
    const size_t half = sizeof(float) * s.W * 2 * 64 * V;
    if (s.segments > 1) hipLaunchKernelGGL((scan_segments_kernel<E, V, STEPS, BACK>), grid, block, half, ctx->stream, s);
    hipLaunchKernelGGL((scan_kernel<E, V, STEPS, BACK, true>), grid, block, 2 * half, ctx->stream, s);
}

template <bool BACK>
int scan(mrl_ctx *ctx, const char *who, int dtype, Scan &s, void *workspace, uint64_t workspace_bytes) {
    OnDevice on(ctx);
    if (s.T == 0) {
        const long n = (long)s.N * s.D;
        if (s.last != nullptr && s.last != s.first)
            hipLaunchKernelGGL(pass_state_kernel, dim3((int)std::min<long>((n + 255) / 256, 4096)), dim3(256), 0, ctx->stream, s.first, s.last, n);
        MRL_CHECK_LAUNCH();
        return MRL_OK;
    }
    const Plan p = plan_of(ctx, s.T, s.N, s.D);
    MRL_CHECK_ARG(workspace_bytes >= p.bytes && (p.bytes == 0 || workspace != nullptr),
                  "%s: the workspace holds %llu bytes, need %llu", who, (unsigned long long)(workspace ? workspace_bytes : 0),
                  (unsigned long long)p.bytes);
    MRL_CHECK_ARG(p.bytes == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: the workspace must be 16-byte aligned", who);
    s.lanes_per_row = p.lanes_per_row; s.lanes = p.lanes; s.groups = p.groups;
    s.W = p.W; s.segments = p.segments; s.segment_steps = p.segment_steps;
    s.ws = (float *)workspace;
    if (dtype == MRL_F32) {
        if (p.V == 4) launch<float, 4, BACK>(ctx, s);
        else launch<float, 1, BACK>(ctx, s);
    } else {
        if (p.V == 4) launch<bf16_t, 4, BACK>(ctx, s);
        else launch<bf16_t, 1, BACK>(ctx, s);
    }
    MRL_CHECK_LAUNCH();
    return MRL_OK;
}

// the sizes that every entry point takes
int check_sizes(const char *who, const mrl_ctx *ctx, int dtype, int T, int N, int D) {
    MRL_CHECK_ARG(ctx, "%s: ctx is NULL", who);
    MRL_CHECK_ARG(dtype == MRL_F32 || dtype == MRL_BF16, "%s: unknown element type %d", who, dtype);
    MRL_CHECK_ARG(T >= 0 && N >= 0 && D >= 0, "%s: negative size", who);
    MRL_CHECK_ARG((long)N * D < 1L << 31, "%s: %d environments of width %d are 2^31 states or more", who, N, D);
    return MRL_OK;
}

}  // namespace
}  // namespace mrl

extern "C" {

int mrl_recurrence_workspace(mrl_ctx *ctx, int T, int N, int D, uint64_t *bytes) {
    const int rc = mrl::check_sizes("mrl_recurrence_workspace", ctx, MRL_F32, T, N, D);
    if (rc != MRL_OK) return rc;
    MRL_CHECK_ARG(bytes, "mrl_recurrence_workspace: NULL result");
    *bytes = T == 0 || N == 0 || D == 0 ? 0 : mrl::plan_of(ctx, T, N, D).bytes;
    return MRL_OK;
}

int mrl_recurrence_forward(mrl_ctx *ctx, int dtype, int T, int N, int D, const void *gate, int64_t gate_ld, const void *value,
                           int64_t value_ld, const float *dones, const float *prev_dones, const float *state_in, void *out,
                           int64_t out_ld, float *state_out, void *workspace, uint64_t workspace_bytes) {
    const char *who = "mrl_recurrence_forward";
    const int rc = mrl::check_sizes(who, ctx, dtype, T, N, D);
    if (rc != MRL_OK) return rc;
    if (N == 0 || D == 0) return MRL_OK;
    MRL_CHECK_ARG(T == 0 || (gate && value && out), "%s: NULL buffer", who);
    MRL_CHECK_ARG(T == 0 || (gate_ld >= D && value_ld >= D && out_ld >= D), "%s: a row stride is smaller than the width %d", who, D);
    mrl::Scan s = {};
    s.T = T; s.N = N; s.D = D;
    s.gate = gate; s.gate_ld = gate_ld;
    s.value = value; s.value_ld = value_ld;
    s.dones = dones; s.prev_dones = prev_dones;
    s.first = state_in; s.last = state_out;
    s.dst = out; s.out_ld = out_ld;
    return mrl::scan<false>(ctx, who, dtype, s, workspace, workspace_bytes);
}

int mrl_recurrence_backward(mrl_ctx *ctx, int dtype, int T, int N, int D, const void *gate, int64_t gate_ld, const void *value,
                            int64_t value_ld, const void *out, int64_t out_ld, const float *dones, const float *prev_dones,
                            const float *state_in, const void *grad_out, int64_t grad_out_ld, const float *grad_state_out,
                            void *grad_gate, int64_t grad_gate_ld, void *grad_value, int64_t grad_value_ld, float *grad_state_in,
                            void *workspace, uint64_t workspace_bytes) {
    const char *who = "mrl_recurrence_backward";
    const int rc = mrl::check_sizes(who, ctx, dtype, T, N, D);
    if (rc != MRL_OK) return rc;
    if (N == 0 || D == 0) return MRL_OK;
    MRL_CHECK_ARG(T == 0 || (gate && value && out && grad_out && grad_gate && grad_value), "%s: NULL buffer", who);
    MRL_CHECK_ARG(T == 0 || (gate_ld >= D && value_ld >= D && out_ld >= D && grad_out_ld >= D && grad_gate_ld >= D && grad_value_ld >= D),
                  "%s: a row stride is smaller than the width %d", who, D);
    mrl::Scan s = {};
    s.T = T; s.N = N; s.D = D;
    s.gate = gate; s.gate_ld = gate_ld;
    s.value = value; s.value_ld = value_ld;
    s.out = out; s.out_ld = out_ld;
    s.dones = dones; s.prev_dones = prev_dones;
    s.state_in = state_in;
    s.grad_out = grad_out; s.grad_out_ld = grad_out_ld;
    s.first = grad_state_out; s.last = grad_state_in;
    s.dst = grad_gate; s.grad_gate_ld = grad_gate_ld;
    s.dst2 = grad_value; s.grad_value_ld = grad_value_ld;
    return mrl::scan<true>(ctx, who, dtype, s, workspace, workspace_bytes);
}

}  // extern "C"
