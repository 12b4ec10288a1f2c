// Gated linear recurrence over a time-major rollout, cut where episodes end, and its gradient:
//
//   a = sigmoid(gate),  h[t] = a[t] h'[t-1] + (1 - a[t]) x[t],   h'[t-1] = 0 where the step before ended an episode, h[t-1] elsewhere
//   d[t] = dh[t] + G[t+1],  G[t] = a[t] d[t] (0 where h' is cut),   dx = (1 - a) d,   dgate = a (1 - a) (h' - x) d
//
// Both are first-order linear recurrences per channel, s <- A s + B, one forwards and one backwards in time, and both are bound by
// memory: forward 3 values per element (12 bytes in fp32), backward 6.  What the kernels do about it is have enough loads in
// flight at every shape.  A lane holds V = 4, 2 or 1 neighbouring channels of one environment, a wavefront 64 V of them.  Three forms:
// - alone: where the channels fill the card, a wavefront goes through the steps by itself, L steps' loads at a time.  128 steps of
//   2048 environments of width 256 in fp32: 150 us, 5.4 TB/s, more than a large copy gets (4.9); backward, 1024 of them: 151 us, 5.3.
// - tiles: with fewer channels a workgroup's W wavefronts take L consecutive steps each of a tile of W L.  A wavefront's steps compose
//   to one (A, B), these are exchanged through LDS, and each wavefront then repeats its steps from its own first state, so every state
//   is the result of the formula above on the state before it and the inputs are read once.  1000 steps of 64 in fp32: 55 us.
// - segments: with a few channels and many steps the time axis is also split over workgroups.  A first launch leaves every segment's
//   (A, B) in a workspace, the second starts each segment from those before it.  Gate and value are read twice, the second time
//   out of the caches where they fit: 16384 steps of 2 of width 512 in bf16 44 us, 18 and 25, 3.7 and 4.0 TB/s.  Part of the 25 are trips
//   to memory one behind the other: a wavefront waits for each of up to eight segments' coefficients, then for each of those
//   of up to seven wavefronts ahead.  (One launch in which a segment waits for those ahead would save the second reading, but a wait
//   among XCDs takes 5 us and more here.)
//
// A cut is a selection, never a product with 0: an infinity or NaN behind it goes nowhere.  In the composed coefficients A = 0
// says so; a product of gates that underflows stays at the smallest subnormal instead.
// States and sums are fp32 whatever the type; in bf16 only gate, value, output and their gradients are rounded, once, when stored.
// The backward pass reads h' from the output, in bf16 as it was rounded: that moves dgate by at most half a step of h', 2^-8 of
// a (1 - a) h' d, about what rounding dgate itself costs where h' and x are alike in size.  States kept in fp32 for it would be 4 more bytes
// written forward and 2 more read backward for each value, of 6 and 12.
#include "mrl_host.hpp"
#include "mrl_device.hpp"

namespace mrl {
namespace {

constexpr float TINY = 0x1p-149f;
constexpr int MAX_WAVES = 8;   // of a workgroup with more than one channel per lane, for the registers; twice that with one

struct bf16_t { unsigned short bits; };

// V neighbouring values as they are in memory
template <class E, int V> struct Raw;
template <int V> struct Raw<float, V> {
    typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
    vec v;
    MRL_DEV void load(const float *p) { v = *reinterpret_cast<const vec *>(p); }
    MRL_DEV float operator[](int i) const { return v[i]; }
};
template <int V> struct Raw<bf16_t, V> {
    typedef unsigned short vec __attribute__((ext_vector_type(V), aligned(2)));
    vec v;
    MRL_DEV void load(const bf16_t *p) { v = *reinterpret_cast<const vec *>(p); }
    MRL_DEV float operator[](int i) const { return __uint_as_float((unsigned)v[i] << 16); }
};

template <int V>
MRL_DEV void load_state(const float *p, float (&x)[V]) {
    Raw<float, V> r;
    r.load(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = r[i];
}

// The elements from `skip` on (the ones before belong to the neighbouring lane); `whole`: no lane has any to skip.
template <int V>
MRL_DEV void store_n(float *p, const float (&x)[V], int skip, bool whole) {
    typename Raw<float, V>::vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = x[i];
    if (whole || skip == 0) {
        *reinterpret_cast<typename Raw<float, V>::vec *>(p) = v;
    } else {
#pragma unroll
        for (int i = 1; i < V; ++i)
            if (i >= skip) p[i] = x[i];
    }
}
template <int V>
MRL_DEV void store_n(bf16_t *p, const float (&x)[V], int skip, bool whole) {
    typedef float floats __attribute__((ext_vector_type(V)));
    typedef __bf16 halves __attribute__((ext_vector_type(V)));
    floats f;
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = x[i];
    const typename Raw<bf16_t, V>::vec v = __builtin_bit_cast(typename Raw<bf16_t, V>::vec, __builtin_convertvector(f, halves));
    if (whole || skip == 0) {
        *reinterpret_cast<typename Raw<bf16_t, V>::vec *>(p) = v;
    } else {
#pragma unroll
        for (int i = 1; i < V; ++i)
            if (i >= skip) p[i].bits = v[i];
    }
}

// a = sigmoid(g) and rest = 1 - a, both relative to their own value: with e = exp(-g), a = 1 / (1 + e) and rest = e a.  The argument is
// held where e stays finite (a below 2^-126 counts as 2^-126).  The reciprocal is off by a step, always to one side, and takes one of
// Newton's: without it states are 1.7 and their gradients 2.6 times as far from 64 bits as a sequence of plain fp32 steps, with it
// as far (bf16: 44 us for 43 at 16384 steps of 2 of width 512, which these instructions bound).  e is 2^y with y = -g / ln 2; in fp32,
// where memory leaves the time for it, what rounding y left of the argument, -g - y ln 2, is taken back (in bf16 that is 4 % slower and
// its states come no closer).
// (minimum and maximum, unlike fmin and fmax, keep NaN.)
MRL_DEV void sigmoid(float e, float &a, float &rest) {
    const float u = 1.0f + e;
    a = __builtin_amdgcn_rcpf(u);
    a = fmaf(a, fmaf(-u, a, 1.0f), a);
    rest = e * a;
}
MRL_DEV void gates(const float *, float g, float &a, float &rest) {
    g = __builtin_elementwise_minimum(__builtin_elementwise_maximum(g, -87.0f), 200.0f);
    const float y = g * -1.44269502f, e = __builtin_amdgcn_exp2f(y);
    sigmoid(fmaf(e, fmaf(y, -0.693147182f, -g), e), a, rest);
}
MRL_DEV void gates(const bf16_t *, float g, float &a, float &rest) {
    sigmoid(__builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g * -1.44269502f, 125.0f)), a, rest);
}

struct Scan {
    int T, N, D, lanes_per_row, W, segments, segment_steps, share;   // share: of a segment's steps, a wavefront's
    int groups;              // of 64 lanes
    int whole;               // no lane has elements to skip
    long lanes;              // N * lanes_per_row
    const void *gate, *value, *out, *grad_out;
    long gate_ld, value_ld, out_ld, grad_out_ld, grad_gate_ld, grad_value_ld;
    const float *dones, *prev_dones;
    const float *first;      // forward: state_in; backward: grad_state_out
    const float *state_in;   // backward
    float *last;             // forward: state_out; backward: grad_state_in
    void *dst, *dst2;        // forward: out; backward: grad_gate, grad_value
    float *ws;               // rows of lanes * V: (A, B) of every segment, (A, B) of every wavefront's share, the first state
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

// step number p of the scan: time p forwards, T - 1 - p backwards
template <bool BACK>
MRL_DEV long time_of(const Scan &s, long p) { return BACK ? s.T - 1 - p : p; }

// L steps' inputs of a lane
template <class E, int V, int L, bool BACK>
struct Steps {
    Raw<E, V> g[L], x[L];
    Raw<E, V> dh[BACK ? L : 1], before[BACK ? L : 1];
    float flag[L];   // of the step before: above 0.5 where it ended an episode
    bool full;       // all L steps are there, none is the rollout's first going backwards
};
// and their gates
template <int V, int L>
struct Gates {
    float a[L][V], rest[L][V];
    template <class E, bool BACK>
    MRL_DEV explicit Gates(const Steps<E, V, L, BACK> &k) {
#pragma unroll
        for (int j = 0; j < L; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) gates((const E *)nullptr, k.g[j][i], a[j][i], rest[j][i]);
    }
};
template <class E, int V, bool BACK>
struct Rows {   // where a lane's columns of step 0 are, and from a step to the next
    const E *gate, *value, *out, *grad;
    long gate_step, value_step, out_step, grad_step;
    bool flagged, whole;
    MRL_DEV Rows(const Scan &s, const Place &at) {
        gate = (const E *)s.gate + (long)at.n * s.gate_ld + at.d;
        value = (const E *)s.value + (long)at.n * s.value_ld + at.d;
        out = (const E *)s.out + (long)at.n * s.out_ld + at.d;
        grad = (const E *)s.grad_out + (long)at.n * s.grad_out_ld + at.d;
        gate_step = (long)s.N * s.gate_ld;
        value_step = (long)s.N * s.value_ld;
        out_step = (long)s.N * s.out_ld;
        grad_step = (long)s.N * s.grad_out_ld;
        flagged = s.dones != nullptr || s.prev_dones != nullptr;
        whole = s.whole != 0;
    }
};

// Steps p0 .. p0 + L - 1; those from `to` on are step to - 1 again, so that all loads stand together without a branch or a wait
// among them.  COEFFICIENTS: only what (A, B) take.
template <class E, int V, int L, bool BACK, bool COEFFICIENTS = false>
MRL_DEV void load_steps(const Scan &s, const Place &at, const Rows<E, V, BACK> &r, long p0, long to, Steps<E, V, L, BACK> &k) {
    const bool full = p0 + L <= to && (!BACK || p0 + L < s.T);
    if (full) {
        long t = time_of<BACK>(s, p0);
#pragma unroll
        for (int j = 0; j < L; ++j) {
            k.g[j].load(r.gate + t * r.gate_step);
            if (!(BACK && COEFFICIENTS)) k.x[j].load(r.value + t * r.value_step);
            if constexpr (BACK) {
                k.dh[j].load(r.grad + t * r.grad_step);
                if (!COEFFICIENTS) k.before[j].load(r.out + (t - 1) * r.out_step);
            }
            t += BACK ? -1 : 1;
        }
    } else {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const long t = time_of<BACK>(s, min(p0 + j, to - 1));
            k.g[j].load(r.gate + t * r.gate_step);
            if (!(BACK && COEFFICIENTS)) k.x[j].load(r.value + t * r.value_step);
            if constexpr (BACK) {
                k.dh[j].load(r.grad + t * r.grad_step);
                if (!COEFFICIENTS) k.before[j].load(r.out + max(t - 1, 0L) * r.out_step);
            }
        }
    }
    k.full = full;
    if (r.flagged) {
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const long t = time_of<BACK>(s, min(p0 + j, to - 1));
            const float *row = t > 0 ? s.dones + (t - 1) * s.N : s.prev_dones;
            k.flag[j] = (t > 0 ? s.dones : s.prev_dones) != nullptr ? row[at.n] : 0.0f;
        }
    }
}
// full, and no lane has a cut among the steps
template <class E, int V, int L, bool BACK>
MRL_DEV bool is_plain(const Rows<E, V, BACK> &r, const Steps<E, V, L, BACK> &k) {
    if (!r.flagged) return k.full;
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j < L; ++j) most = fmaxf(most, k.flag[j]);
    return k.full && __ballot(most > 0.5f) == 0;
}

template <int V>
MRL_DEV void compose(float (&state)[V], const float (&A)[V], const float (&B)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) state[i] = A[i] == 0.0f ? B[i] : fmaf(A[i], state[i], B[i]);
}
// (A, B) <- (A1, B1) after (A, B)
template <int V>
MRL_DEV void compose(float (&A)[V], float (&B)[V], const float (&A1)[V], const float (&B1)[V]) {
    compose(B, A1, B1);
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = A1[i] == 0.0f || A[i] == 0.0f ? 0.0f : fmaxf(A[i] * A1[i], TINY);
}

template <int V>
MRL_DEV void put(float *p, const float (&x)[V]) {
    typedef float vec __attribute__((ext_vector_type(V)));
    vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = x[i];
    *reinterpret_cast<vec *>(p) = v;
}
template <int V>
MRL_DEV void get(const float *p, float (&x)[V]) {
    typedef float vec __attribute__((ext_vector_type(V)));
    const vec v = *reinterpret_cast<const vec *>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = v[i];
}
template <int V>
MRL_DEV void identity(float (&A)[V], float (&B)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) { A[i] = 1.0f; B[i] = 0.0f; }
}

// The state ahead of wavefront w's share, from the state ahead of the workgroup's and the shares' (A, B), `apart` floats from
// one coefficient's row to the next; `carry` becomes the state behind all of them.
template <int V>
MRL_DEV void through_waves(const float *shares, long apart, int W, int w, float (&carry)[V], float (&mine)[V]) {
#pragma unroll 4
    for (int i = 0; i < W; ++i) {
        float A[V], B[V];
        get(shares + (long)i * 2 * apart, A);
        get(shares + ((long)i * 2 + 1) * apart, B);
#pragma unroll
        for (int k = 0; k < V; ++k) mine[k] = i == w ? carry[k] : mine[k];
        compose(carry, A, B);
    }
}

// (A, B) of these steps on top of those before them; `cuts`: whether a lane has seen a cut.  The backward scan's state is G[t+1],
// what goes into step t from behind it.
template <bool PLAIN, class E, int V, int L, bool BACK>
MRL_DEV void add_steps(const Rows<E, V, BACK> &r, const Steps<E, V, L, BACK> &k, const Gates<V, L> &gate, long p0, long to, float (&A)[V], float (&B)[V], bool &cuts) {
#pragma unroll
    for (int j = 0; j < L; ++j) {
        if (!PLAIN && p0 + j >= to) break;
        const bool cut = !PLAIN && r.flagged && k.flag[j] > 0.5f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (BACK) {
                B[i] = gate.a[j][i] * (B[i] + k.dh[j][i]);
                if (!PLAIN) B[i] = cut ? 0.0f : B[i];
            } else {
                if (!PLAIN) B[i] = cut ? 0.0f : B[i];
                B[i] = fmaf(gate.a[j][i], B[i], gate.rest[j][i] * k.x[j][i]);
            }
            A[i] *= gate.a[j][i];
        }
        if (!PLAIN) cuts |= cut;
    }
}
// A of a chain that has a cut is 0, that of one without never
template <int V>
MRL_DEV void settle(float (&A)[V], bool cuts) {
#pragma unroll
    for (int i = 0; i < V; ++i) A[i] = cuts ? 0.0f : fmaxf(A[i], TINY);
}

// These steps from the state ahead of them: results out, `mine` the state behind them.
template <bool PLAIN, class E, int V, int L, bool BACK>
MRL_DEV void do_steps(const Scan &s, const Place &at, const Rows<E, V, BACK> &r, const Steps<E, V, L, BACK> &k, const Gates<V, L> &gate, long p0,
                      long to, float (&mine)[V]) {
    E *dst = (E *)s.dst + (long)at.n * (BACK ? s.grad_gate_ld : s.out_ld) + at.d;
    E *dst2 = (E *)s.dst2 + (long)at.n * s.grad_value_ld + at.d;
    const long dst_step = (long)s.N * (BACK ? s.grad_gate_ld : s.out_ld), dst2_step = (long)s.N * s.grad_value_ld;
    long t = time_of<BACK>(s, p0);
#pragma unroll
    for (int j = 0; j < L; ++j, t += BACK ? -1 : 1) {
        if (!PLAIN && p0 + j >= to) break;
        const bool cut = !PLAIN && r.flagged && k.flag[j] > 0.5f;
        float y[V];
        if constexpr (BACK) {
            float y2[V], before[V];
#pragma unroll
            for (int i = 0; i < V; ++i) before[i] = k.before[j][i];
            if (!PLAIN) {
                if (t == 0) {
#pragma unroll
                    for (int i = 0; i < V; ++i) before[i] = 0.0f;
                    if (s.state_in != nullptr) load_state(s.state_in + (long)at.n * s.D + at.d, before);
                }
#pragma unroll
                for (int i = 0; i < V; ++i) before[i] = cut ? 0.0f : before[i];
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = k.dh[j][i] + mine[i];
                y2[i] = gate.rest[j][i] * d;
                mine[i] = gate.a[j][i] * d;
                y[i] = gate.rest[j][i] * mine[i] * (before[i] - k.x[j][i]);
                if (!PLAIN) mine[i] = cut ? 0.0f : mine[i];
            }
            if (at.live) store_n(dst2 + t * dst2_step, y2, at.skip, r.whole);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (!PLAIN) mine[i] = cut ? 0.0f : mine[i];
                y[i] = mine[i] = fmaf(gate.a[j][i], mine[i], gate.rest[j][i] * k.x[j][i]);
            }
        }
        if (at.live) store_n(dst + t * dst_step, y, at.skip, r.whole);
        if (j == L - 1 || !PLAIN) {
            if (p0 + j == s.T - 1 && at.live && s.last != nullptr) store_n(s.last + (long)at.n * s.D + at.d, mine, at.skip, r.whole);
        }
    }
}

// All steps from `from` to `to` in a row, the first L of them loaded.
template <class E, int V, int L, bool BACK>
MRL_DEV void stream_steps(const Scan &s, const Place &at, const Rows<E, V, BACK> &rows, long from, long to, Steps<E, V, L, BACK> &k, float (&mine)[V]) {
    for (long p0 = from; p0 < to; p0 += L) {
        if (p0 != from) load_steps(s, at, rows, p0, to, k);
        const Gates<V, L> gate(k);
        if (is_plain(rows, k)) do_steps<true>(s, at, rows, k, gate, p0, to, mine);
        else do_steps<false>(s, at, rows, k, gate, p0, to, mine);
    }
}

// A wavefront per group of lanes, all steps.
template <class E, int V, int L, bool BACK>
__global__ __launch_bounds__(256) void scan_alone_kernel(Scan s) {
    const int group = blockIdx.x * blockDim.y + threadIdx.y;
    if (group >= s.groups) return;
    const Place at = place<V>(s, group);
    const Rows<E, V, BACK> rows(s, at);
    Steps<E, V, L, BACK> k;
    load_steps(s, at, rows, 0, s.T, k);
    float mine[V];
#pragma unroll
    for (int i = 0; i < V; ++i) mine[i] = 0.0f;
    if (s.first != nullptr) load_state(s.first + (long)at.n * s.D + at.d, mine);
    stream_steps(s, at, rows, 0, s.T, k, mine);
}

// A workgroup per group of lanes, its wavefronts L steps each of a tile of W L.
template <class E, int V, int L, bool BACK>
__global__ __launch_bounds__(64 * MAX_WAVES * (V == 1 ? 2 : 1)) void scan_tiles_kernel(Scan s) {
    extern __shared__ float lds[];
    const Place at = place<V>(s, blockIdx.x);
    const Rows<E, V, BACK> rows(s, at);
    const int w = threadIdx.y, W = s.W;
    const int half = W * 2 * 64 * V;
    float carry[V], mine[V];
#pragma unroll
    for (int i = 0; i < V; ++i) carry[i] = mine[i] = 0.0f;
    if (s.first != nullptr) load_state(s.first + (long)at.n * s.D + at.d, carry);
    int buffer = 0;
    for (long t0 = 0; t0 < s.T; t0 += (long)W * L) {
        const long p0 = t0 + w * L;
        Steps<E, V, L, BACK> k;
        load_steps(s, at, rows, p0, s.T, k);
        const Gates<V, L> gate(k);
        const bool plain = is_plain(rows, k);
        float A[V], B[V];
        bool cuts = false;
        identity(A, B);
        if (plain) add_steps<true>(rows, k, gate, p0, s.T, A, B, cuts);
        else add_steps<false>(rows, k, gate, p0, s.T, A, B, cuts);
        settle(A, cuts);
        float *shares = lds + buffer * half + threadIdx.x * V;
        put(shares + (w * 2) * 64 * V, A);
        put(shares + (w * 2 + 1) * 64 * V, B);
        __syncthreads();   // (the buffers alternate: the next tile's values go where nobody reads any more)
        through_waves(shares, 64 * V, W, w, carry, mine);
        buffer ^= 1;
        if (plain) do_steps<true>(s, at, rows, k, gate, p0, s.T, mine);
        else do_steps<false>(s, at, rows, k, gate, p0, s.T, mine);
    }
}

MRL_DEV void share_of(const Scan &s, int seg, int w, long &from, long &to) {
    const long end = min((long)s.T, (long)(seg + 1) * s.segment_steps);
    from = min(end, (long)seg * s.segment_steps + (long)w * s.share);
    to = min(end, from + s.share);
}

// First launch of a scan in segments: every wavefront's (A, B), and the segment's.
template <class E, int V, int L, bool BACK>
__global__ __launch_bounds__(64 * MAX_WAVES) void scan_coefficients_kernel(Scan s) {
    extern __shared__ float lds[];
    const Place at = place<V>(s, blockIdx.x);
    const Rows<E, V, BACK> rows(s, at);
    const int w = threadIdx.y, seg = blockIdx.y;
    long from, to;
    share_of(s, seg, w, from, to);
    float A[V], B[V];
    bool cuts = false;
    identity(A, B);
    for (long p0 = from; p0 < to; p0 += L) {
        Steps<E, V, L, BACK> k;
        load_steps<E, V, L, BACK, true>(s, at, rows, p0, to, k);
        const Gates<V, L> gate(k);
        if (is_plain(rows, k)) add_steps<true>(rows, k, gate, p0, to, A, B, cuts);
        else add_steps<false>(rows, k, gate, p0, to, A, B, cuts);
    }
    settle(A, cuts);
    const long row = s.lanes * V;
    float *segments = s.ws + at.q * V, *shares = segments + (long)s.segments * 2 * row;
    if (at.live) {
        put(shares + ((long)seg * s.W + w) * 2 * row, A);
        put(shares + (((long)seg * s.W + w) * 2 + 1) * row, B);
    }
    float *mine = lds + threadIdx.x * V;
    put(mine + (w * 2) * 64 * V, A);
    put(mine + (w * 2 + 1) * 64 * V, B);
    __syncthreads();
    if (w != 0 || !at.live) return;
    for (int i = 1; i < s.W; ++i) {
        float A1[V], B1[V];
        get(mine + (i * 2) * 64 * V, A1);
        get(mine + (i * 2 + 1) * 64 * V, B1);
        compose(A, B, A1, B1);
    }
    put(segments + (long)seg * 2 * row, A);
    put(segments + ((long)seg * 2 + 1) * row, B);
    if (seg == 0) {   // the first state, which `last` may overwrite while segments still start
        float first[V];
#pragma unroll
        for (int i = 0; i < V; ++i) first[i] = 0.0f;
        if (s.first != nullptr) load_state(s.first + (long)at.n * s.D + at.d, first);
        put(shares + (long)s.segments * s.W * 2 * row, first);
    }
}

// Second launch: a wavefront starts from the segments ahead (its share of them, exchanged through LDS) and the wavefronts ahead.
template <class E, int V, int L, bool BACK>
__global__ __launch_bounds__(64 * MAX_WAVES) void scan_segments_kernel(Scan s) {
    extern __shared__ float lds[];
    const Place at = place<V>(s, blockIdx.x);
    const Rows<E, V, BACK> rows(s, at);
    const int w = threadIdx.y, seg = blockIdx.y;
    long from, to;
    share_of(s, seg, w, from, to);
    Steps<E, V, L, BACK> k;
    load_steps(s, at, rows, from, max(to, from + 1 - (from == s.T)), k);
    const long row = s.lanes * V;
    const float *segments = s.ws + at.q * V, *shares = segments + (long)s.segments * 2 * row;
    const int per = (seg + s.W - 1) / s.W, first = min(seg, w * per), last = min(seg, first + per);
    float A[V], B[V];
    identity(A, B);
    for (int i = first; i < last; ++i) {
        float A1[V], B1[V];
        get(segments + (long)i * 2 * row, A1);
        get(segments + ((long)i * 2 + 1) * row, B1);
        compose(A, B, A1, B1);
    }
    float *exchange = lds + threadIdx.x * V;
    put(exchange + (w * 2) * 64 * V, A);
    put(exchange + (w * 2 + 1) * 64 * V, B);
    float carry[V], mine[V];
    get(shares + (long)s.segments * s.W * 2 * row, carry);
    __syncthreads();
    through_waves(exchange, 64 * V, s.W, -1, carry, mine);
    for (int i = 0; i < w; ++i) {
        get(shares + ((long)seg * s.W + i) * 2 * row, A);
        get(shares + (((long)seg * s.W + i) * 2 + 1) * row, B);
        compose(carry, A, B);
    }
    stream_steps(s, at, rows, from, to, k, carry);
}

// no step at all: the state goes through as it is
__global__ __launch_bounds__(256) void pass_state_kernel(const float *from, float *to, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) to[i] = from ? from[i] : 0.0f;
}

constexpr int tile_steps(int V) { return V == 4 ? 4 : 8; }   // of a wavefront, for the registers

// How a scan is laid out over the card.
struct Plan {
    int V, lanes_per_row, W, segments, segment_steps, share, groups;
    long lanes;
    size_t bytes;
};
void channels(Plan &p, int V, int N, int D) {
    p.V = V = D >= V ? V : D >= 2 ? std::min(V, 2) : 1;
    p.lanes_per_row = (D + V - 1) / V;
    p.lanes = (long)N * p.lanes_per_row;
    p.groups = (int)((p.lanes + 63) / 64);
}
// Eight wavefronts per CU keep the memory busy.  Where one per group of 64 lanes with V = 4 channels gives fewer, workgroups of up to
// 8 share a group's steps; with fewer groups than CUs lanes have 2 channels, then 1 (and up to 16 wavefronts): the exchange
// between a tile's wavefronts costs as much whatever a lane holds.  us on 256 CUs, fp32, 1000 steps of width 256, V = 4 / 2 / 1:
//   N = 16: 90 / 56 / 36   64: 115 / 71 / 55   128: 127 / 83 / 94   256: 153 / 165 / 178
// Segments read gate and value twice but go through the time side by side.  Tiles / segments, 1000 steps, fp32 and bf16:
//   N = 1: 34 / 18, 34 / 18   16: 36 / 23   32: 39 / 39, 37 / 25   64: 55 / 72, 46 / 42   128: 83 / 134, 61 / 78
// (256 steps: N = 1 12 / 18, 32: 13 / 19; backward: 1000 steps, N = 32 66 / 58, 57 / 36, 64 90 / 108, 74 / 64).
// Where a few channels leave lanes without any, lanes have fewer.  65536 steps of width 64, V = 4 / 2 / 1: fp32 47 / 41 / 35, bf16
// 43 / 36 / 31, backward 59 / 53 / 49, 53 / 42 / 38.
Plan plan_of(const mrl_ctx *ctx, int T, int N, int D, int size) {
    Plan p = {};
    const long want = 8L * ctx->n_cus;   // wavefronts
    constexpr long SHARE = 16;            // steps that a wavefront of a segment has at least
    channels(p, 4, N, D);
    p.W = 1;
    p.segments = 1;
    if (T >= 512 && (long)p.groups * size * 2 < ctx->n_cus) {
        if ((long)p.groups * T < SHARE * want || p.lanes <= 32) channels(p, 2, N, D);
        if (p.lanes <= 32) channels(p, 1, N, D);
        const long shares = std::min<long>(((long)T + SHARE - 1) / SHARE, std::max<long>(2 * MAX_WAVES, want / p.groups));
        p.W = MAX_WAVES;
        p.share = (int)((T + shares - 1) / shares);
        p.segment_steps = p.share * p.W;
        p.segments = (int)(((long)T + p.segment_steps - 1) / p.segment_steps);
        p.bytes = sizeof(float) * (size_t)p.lanes * p.V * (2 * (size_t)p.segments * (p.W + 1) + 1);
        return p;
    }
    if (T == 1) return p;
    for (int V = 2; V >= 1 && p.groups <= ctx->n_cus / 2; --V) channels(p, V, N, D);
    const int most = MAX_WAVES * (p.V == 1 ? 2 : 1);
    while (p.W < most && (long)p.groups * p.W < want && (long)p.W * tile_steps(p.V) < T) p.W *= 2;
    return p;
}

template <class E, int V, bool BACK>
void launch(const mrl_ctx *ctx, const Scan &s) {
    constexpr int L = 4;   // steps whose loads are under way together
    if (s.segments > 1) {
        const dim3 grid(s.groups, s.segments), block(64, s.W);
        const size_t lds = sizeof(float) * s.W * 2 * 64 * V;
        hipLaunchKernelGGL((scan_coefficients_kernel<E, V, L, BACK>), grid, block, lds, ctx->stream, s);
        hipLaunchKernelGGL((scan_segments_kernel<E, V, L, BACK>), grid, block, lds, ctx->stream, s);
    } else if (s.W > 1) {
        hipLaunchKernelGGL((scan_tiles_kernel<E, V, tile_steps(V), BACK>), dim3(s.groups), dim3(64, s.W), sizeof(float) * 2 * s.W * 2 * 64 * V, ctx->stream, s);
    } else {
        const int per = s.groups >= 4 * ctx->n_cus ? 4 : 1;
        const dim3 grid((s.groups + per - 1) / per), block(64, per);
        if (s.T == 1) hipLaunchKernelGGL((scan_alone_kernel<E, V, 1, BACK>), grid, block, 0, ctx->stream, s);
        else hipLaunchKernelGGL((scan_alone_kernel<E, V, L, BACK>), grid, block, 0, ctx->stream, s);
    }
}
template <class E, bool BACK>
void launch(const mrl_ctx *ctx, const Scan &s, int V) {
    if (V == 4) launch<E, 4, BACK>(ctx, s);
    else if (V == 2) launch<E, 2, BACK>(ctx, s);
    else launch<E, 1, BACK>(ctx, s);
}

// No output has an element of an input or of another output; the last state may be the first.
template <bool BACK>
int check_buffers(const char *who, int dtype, const Scan &s, void *workspace, size_t workspace_bytes) {
    const int64_t size = dtype == MRL_F32 ? 4 : 2, rows = (int64_t)s.T * s.N, states = 4LL * s.N * s.D;
    auto of = [&](const char *name, const void *at, long ld) { return Region(name, at, rows, size * s.D, size * ld); };
    const Region ahead(BACK ? "grad_state_out" : "state_in", s.first == s.last ? nullptr : s.first, states), behind(BACK ? "grad_state_in" : "state_out", s.last, states);
    const Region gate = of("gate", s.gate, s.gate_ld), value = of("value", s.value, s.value_ld), scratch("the workspace", workspace, (int64_t)workspace_bytes);
    const Region dones("dones", s.dones, 4 * rows), prev_dones("prev_dones", s.prev_dones, 4LL * s.N);
    if (BACK)
        return check_apart(who, {of("grad_gate", s.dst, s.grad_gate_ld), of("grad_value", s.dst2, s.grad_value_ld), behind, scratch},
                           {gate, value, of("out", s.out, s.out_ld), of("grad_out", s.grad_out, s.grad_out_ld), dones, prev_dones, Region("state_in", s.state_in, states), ahead});
    return check_apart(who, {of("out", s.dst, s.out_ld), behind, scratch}, {gate, value, dones, prev_dones, ahead});
}

template <bool BACK>
int scan(mrl_ctx *ctx, const char *who, int dtype, Scan &s, void *workspace, uint64_t workspace_bytes) {
    OnDevice on(ctx);
    if (s.T == 0) {
        const long n = (long)s.N * s.D;
        const int rc = check_buffers<BACK>(who, dtype, s, nullptr, 0);
        if (rc != MRL_OK) return rc;
        if (s.last != nullptr && s.last != s.first)
            hipLaunchKernelGGL(pass_state_kernel, dim3((int)std::min<long>((n + 255) / 256, 4096)), dim3(256), 0, ctx->stream, s.first, s.last, n);
        MRL_CHECK_LAUNCH();
        return MRL_OK;
    }
    const Plan p = plan_of(ctx, s.T, s.N, s.D, dtype == MRL_F32 ? 4 : 2);
    MRL_CHECK_ARG(workspace_bytes >= p.bytes && (p.bytes == 0 || workspace != nullptr),
                  "%s: the workspace holds %llu bytes, need %llu", who, (unsigned long long)(workspace ? workspace_bytes : 0),
                  (unsigned long long)p.bytes);
    MRL_CHECK_ARG(p.bytes == 0 || reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: the workspace must be 16-byte aligned", who);
    const int rc = check_buffers<BACK>(who, dtype, s, workspace, p.bytes);
    if (rc != MRL_OK) return rc;
    s.lanes_per_row = p.lanes_per_row; s.lanes = p.lanes; s.groups = p.groups;
    s.W = p.W; s.segments = p.segments; s.segment_steps = p.segment_steps; s.share = p.share;
    s.whole = s.D % p.V == 0;
    s.ws = (float *)workspace;
    if (dtype == MRL_F32) launch<float, BACK>(ctx, s, p.V);
    else launch<bf16_t, BACK>(ctx, s, p.V);
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
    *bytes = T == 0 || N == 0 || D == 0 ? 0 : std::max(mrl::plan_of(ctx, T, N, D, 4).bytes, mrl::plan_of(ctx, T, N, D, 2).bytes);
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
