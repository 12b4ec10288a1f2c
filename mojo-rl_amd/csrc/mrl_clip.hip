// Clipping by the norm of all values of many tensors: out = x * (norm > max_norm ? max_norm / (norm + 1e-8) : 1).
//
// Two launches, each over all tensors in pieces of PIECE values: partial sums of squares, then every workgroup adds up the partial sums
// (the same order everywhere) and scales its pieces.  Squares and sums are Float64: no value's square overflows or vanishes, and the order of a
// few thousand partial sums does not show in fp32.  Bound by memory: every value is read twice, the second time out of the last-level
// cache where the tensors fit, and written once.  107 MB in 20 tensors take 19 us to sum (5.6 TB/s) and 36 to scale (5.9 TB/s), what this
// card copies 256 MiB with; 12 small tensors take 4 us twice, and the host 22 to make the two calls.
#include "mrl_host.hpp"
#include "mrl_device.hpp"

namespace mrl {
namespace {

constexpr int THREADS = 256, PIECE = 8 * THREADS;   // values
constexpr int MOST = 96;          // tensors of a launch: the table travels with the launch's arguments
constexpr int MOST_SUMS = 2048;   // partial sums of all launches

struct bf16_t { unsigned short bits; };

struct Table {
    int count, blocks, first_block;   // workgroups of this launch; partial sums of the launches ahead
    int64_t per;                      // pieces of a workgroup
    int64_t begin[MOST + 1];          // a tensor's first piece
    const void *in[MOST];
    void *out[MOST];
    int64_t n[MOST];
    int bf16[MOST];
};

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

MRL_DEV f32x8 load8(const float *p) {
    const f32x4u a = *reinterpret_cast<const f32x4u *>(p), b = *reinterpret_cast<const f32x4u *>(p + 4);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
MRL_DEV f32x8 load8(const bf16_t *p) {
    const u16x8u v = *reinterpret_cast<const u16x8u *>(p);
    f32x8 x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float((unsigned)v[i] << 16);
    return x;
}
MRL_DEV void store8(float *p, f32x8 x) {
    *reinterpret_cast<f32x4u *>(p) = f32x4u{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4u *>(p + 4) = f32x4u{x[4], x[5], x[6], x[7]};
}
MRL_DEV void store8(bf16_t *p, f32x8 x) { *reinterpret_cast<u16x8u *>(p) = __builtin_bit_cast(u16x8u, __builtin_convertvector(x, bf16x8)); }
MRL_DEV float value_of(float x) { return x; }
MRL_DEV float value_of(bf16_t x) { return __uint_as_float((unsigned)x.bits << 16); }
MRL_DEV void give(float *p, float x) { *p = x; }
MRL_DEV void give(bf16_t *p, float x) { p->bits = __builtin_bit_cast(unsigned short, (__bf16)x); }

template <class E>
MRL_DEV void squares(const E *p, int64_t n, int64_t at, double &sum) {
    const int64_t i = at + threadIdx.x * 8;
    if (i + 8 <= n) {
        const f32x8 x = load8(p + i);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fma((double)x[j], (double)x[j], sum);
    } else {
        for (int64_t j = i; j < n; ++j) sum = fma((double)value_of(p[j]), (double)value_of(p[j]), sum);
    }
}
template <class E>
MRL_DEV void scaled(const E *p, E *out, int64_t n, int64_t at, float scale, float unit) {
    const int64_t i = at + threadIdx.x * 8;
    if (i + 8 <= n) store8(out + i, load8(p + i) * scale * unit);
    else
        for (int64_t j = i; j < n; ++j) give(out + j, value_of(p[j]) * scale * unit);
}

MRL_DEV double block_sum(double x, double *shared) {
#pragma unroll
    for (int s = 32; s > 0; s /= 2) x += __shfl_xor(x, s);
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
    __syncthreads();
    return (shared[0] + shared[1]) + (shared[2] + shared[3]);
}

__global__ __launch_bounds__(THREADS) void squares_kernel(Table t, double *sums) {
    __shared__ double shared[4];
    double sum = 0.0;
    const int64_t from = blockIdx.x * t.per, to = min(from + t.per, t.begin[t.count]);
    int k = 0;
    for (int64_t piece = from; piece < to; ++piece) {
        while (piece >= t.begin[k + 1]) ++k;
        const int64_t at = (piece - t.begin[k]) * PIECE;
        if (t.bf16[k]) squares((const bf16_t *)t.in[k], t.n[k], at, sum);
        else squares((const float *)t.in[k], t.n[k], at, sum);
    }
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) sums[t.first_block + blockIdx.x] = sum;
}

__global__ __launch_bounds__(THREADS) void scale_kernel(Table t, const double *sums, int all, double max_norm, float *norm_out) {
    __shared__ double shared[4];
    double sum = 0.0;
    for (int i = threadIdx.x; i < all; i += THREADS) sum += sums[i];
    const double norm = sqrt(block_sum(sum, shared));
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) *norm_out = (float)norm;
    const bool clips = norm > max_norm;
    // a factor among fp32's subnormals, which would have few bits, is taken in two steps, the second a power of two
    const double factor = clips ? max_norm / (norm + 1e-8) : 1.0;
    const bool tiny = factor < 0x1p-100;
    const float scale = (float)(tiny ? factor * 0x1p100 : factor), unit = tiny ? 0x1p-100f : 1.0f;
    const int64_t from = blockIdx.x * t.per, to = min(from + t.per, t.begin[t.count]);
    int k = 0;
    for (int64_t piece = from; piece < to; ++piece) {
        while (piece >= t.begin[k + 1]) ++k;
        if (!clips && t.in[k] == t.out[k]) continue;
        const int64_t at = (piece - t.begin[k]) * PIECE;
        if (t.bf16[k]) scaled((const bf16_t *)t.in[k], (bf16_t *)t.out[k], t.n[k], at, scale, unit);
        else scaled((const float *)t.in[k], (float *)t.out[k], t.n[k], at, scale, unit);
    }
}

// No output has a byte of another tensor, but for its own input, which it may be.
int check_tensors(const char *who, int count, const mrl_tensor *tensors) {
    struct Span { uintptr_t from, to; bool written; };
    std::vector<Span> spans;
    spans.reserve(2 * (size_t)count);
    for (int i = 0; i < count; ++i) {
        const mrl_tensor &t = tensors[i];
        MRL_CHECK_ARG(t.dtype == MRL_F32 || t.dtype == MRL_BF16, "%s: unknown element type %d", who, t.dtype);
        MRL_CHECK_ARG(t.n >= 0 && t.n < (int64_t)1 << 48, "%s: tensor %d has %lld values", who, i, (long long)t.n);
        if (t.n == 0) continue;
        MRL_CHECK_ARG(t.in && t.out, "%s: NULL tensor %d", who, i);
        const uintptr_t bytes = (uintptr_t)t.n * (t.dtype == MRL_F32 ? 4 : 2), in = (uintptr_t)t.in, out = (uintptr_t)t.out;
        spans.push_back({out, out + bytes, true});
        if (in != out) spans.push_back({in, in + bytes, false});
    }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.from < b.from; });
    uintptr_t written = 0, any = 0;   // where those so far end
    for (const Span &s : spans) {
        MRL_CHECK_ARG(s.from >= (s.written ? any : written), "%s: an output overlaps another tensor", who);
        any = std::max(any, s.to);
        if (s.written) written = std::max(written, s.to);
    }
    return MRL_OK;
}

}  // namespace
}  // namespace mrl

extern "C" {

int mrl_clip_tensors(mrl_ctx *ctx, int count, const mrl_tensor *tensors, double max_norm, float *norm, void *workspace, uint64_t workspace_bytes) {
    using namespace mrl;
    const char *who = "mrl_clip_tensors";
    MRL_CHECK_ARG(ctx, "%s: ctx is NULL", who);
    MRL_CHECK_ARG(count >= 0 && (count == 0 || tensors), "%s: %d tensors", who, count);
    MRL_CHECK_ARG(max_norm >= 0.0, "%s: max_norm %g is below 0", who, max_norm);
    MRL_CHECK_ARG(workspace && workspace_bytes >= MRL_CLIP_TENSORS_WORKSPACE, "%s: the workspace holds %llu bytes, need %d", who,
                  (unsigned long long)(workspace ? workspace_bytes : 0), MRL_CLIP_TENSORS_WORKSPACE);
    MRL_CHECK_ARG(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: the workspace must be 16-byte aligned", who);
    static_assert(MRL_CLIP_TENSORS_WORKSPACE == sizeof(double) * MOST_SUMS, "the partial sums");
    try {
        const int rc = check_tensors(who, count, tensors);
        if (rc != MRL_OK) return rc;
        for (int i = 0; i < count; ++i) {
            const int64_t bytes = tensors[i].n * (tensors[i].dtype == MRL_F32 ? 4 : 2);
            const int apart = check_apart(who, {Region("norm", norm, 4), Region("the workspace", workspace, MRL_CLIP_TENSORS_WORKSPACE)},
                                          {Region("a tensor", tensors[i].in, bytes), Region("a tensor", tensors[i].out, bytes)});
            if (apart != MRL_OK) return apart;
        }
        std::vector<Table> tables;
        int64_t pieces = 0;
        for (int i = 0, k = MOST; i < count; ++i) {
            if (tensors[i].n == 0) continue;
            if (k == MOST) {
                tables.emplace_back();
                tables.back().count = k = 0;
                tables.back().begin[0] = 0;
            }
            Table &t = tables.back();
            t.in[k] = tensors[i].in;
            t.out[k] = tensors[i].out;
            t.n[k] = tensors[i].n;
            t.bf16[k] = tensors[i].dtype == MRL_BF16;
            const int64_t own = (tensors[i].n + PIECE - 1) / PIECE;
            t.begin[k + 1] = t.begin[k] + own;
            t.count = ++k;
            pieces += own;
        }
        if (tables.empty()) tables.emplace_back(), tables.back().count = 0, tables.back().begin[0] = 0;
        MRL_CHECK_ARG(tables.size() <= MOST_SUMS / 2, "%s: %d tensors are more than %d", who, count, MOST * MOST_SUMS / 2);
        // every launch has a workgroup at least, all together no more than partial sums
        const int64_t room = MOST_SUMS - (int64_t)tables.size(), per = std::max<int64_t>(1, (pieces + room - 1) / room);
        int blocks = 0;
        for (Table &t : tables) {
            t.per = per;
            t.blocks = (int)std::max<int64_t>(1, (t.begin[t.count] + per - 1) / per);
            t.first_block = blocks;
            blocks += t.blocks;
        }
        OnDevice on(ctx);
        double *sums = (double *)workspace;
        for (const Table &t : tables) hipLaunchKernelGGL(squares_kernel, dim3(t.blocks), dim3(THREADS), 0, ctx->stream, t, sums);
        for (const Table &t : tables)
            hipLaunchKernelGGL(scale_kernel, dim3(t.blocks), dim3(THREADS), 0, ctx->stream, t, sums, blocks, max_norm, &t == &tables[0] ? norm : nullptr);
        MRL_CHECK_LAUNCH();
    } catch (const std::bad_alloc &) {
        return set_error(MRL_E_ARG, "%s: no host memory for the description of %d tensors", who, count);
    }
    return MRL_OK;
}

}  // extern "C"
