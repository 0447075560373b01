// rotary_axes: rotary positions with several axes.
//   angle(t, j) = positions[axis(j), t] * inv_freq[j];   (a, b) -> (a cos - b sin, b cos + a sin);   gradient: -angle
// Every element is read once and written once: bound by HBM.  A workgroup takes a few tokens: it forms their R/2 sines and
// cosines once in LDS (the angle in 64 bits, reduced to a fraction of a turn before the fp32 sine, since positions run to
// millions), then streams the rows of all heads of q and k past them, 16 bytes per load.  Measured: 32768 tokens, 32 + 8 heads of
// 128, half of the channels turned, bf16: 130 us for 670 MB = 5.2 TB/s, the rate of a copy; 256 tokens: 4.8 us.
#include "common.h"
#include "device_utils.h"

namespace fla {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxPairs = 128;
constexpr int kMaxTokens = 4;   // tokens per workgroup

struct Rows {   // one of q, k
    const void *x;
    void *y;
    int64_t xb, xt, xh, yb, yt, yh;
};

struct RotaryParams {
    Rows q, k;
    const void *positions;
    int64_t pos_a, pos_b, pos_t;
    bool pos64, adjacent, inverse;
    const float *inv_freq;
    int64_t tokens;    // B * T
    int t_len, q_heads, heads, dim, pairs, tokens_per_wg;
    uint8_t axis[kMaxPairs];
};

template <typename T, int V> struct Piece { typedef T type __attribute__((ext_vector_type(V))); };

template <typename T, int V, bool ADJ>
__global__ void __launch_bounds__(kThreads) rotary_axes_kernel(const RotaryParams p) {
    typedef typename Piece<T, V>::type TV;
    __shared__ f32x2 turn[kMaxTokens * kMaxPairs];
    const int tid = threadIdx.x;
    const int64_t t0 = (int64_t)blockIdx.x * p.tokens_per_wg;
    const int count = (int)min((int64_t)p.tokens_per_wg, p.tokens - t0);
    for (int i = tid; i < count * p.pairs; i += kThreads) {
        const int t = i / p.pairs, j = i - t * p.pairs;
        const int64_t row = t0 + t, b = row / p.t_len, at = p.axis[j] * p.pos_a + b * p.pos_b + (row - b * p.t_len) * p.pos_t;
        const double pos = p.pos64 ? (double)static_cast<const int64_t *>(p.positions)[at] : (double)static_cast<const int32_t *>(p.positions)[at];
        const double turns = pos * (double)p.inv_freq[j] * 0.15915494309189533577;   // 1 / (2 pi)
        float s, c;
        sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
        turn[t * p.pairs + j] = f32x2{c, p.inverse ? -s : s};
    }
    __syncthreads();
    // a unit is two pieces of V channels of one row: the two halves of V pairs, or (adjacent pairs, channels that are
    // copied) two pieces half a row apart
    const int units = p.dim / (2 * V), rot = p.pairs / V, rest = (p.dim - 2 * p.pairs) / (2 * V);
    const int total = count * p.heads * units;
    for (int i = tid; i < total; i += kThreads) {
        const int row = i / units, u = i - row * units, t = row / p.heads, head = row - t * p.heads;
        const int64_t token = t0 + t, b = token / p.t_len, at = token - b * p.t_len;
        const bool is_q = head < p.q_heads;
        const Rows &r = is_q ? p.q : p.k;
        const int h = is_q ? head : head - p.q_heads;
        const T *x = static_cast<const T *>(r.x) + b * r.xb + at * r.xt + h * r.xh;
        T *y = static_cast<T *>(r.y) + b * r.yb + at * r.yt + h * r.yh;
        const f32x2 *tr = turn + t * p.pairs;
        if (!ADJ) {
            const int c0 = u < rot ? u * V : 2 * p.pairs + (u - rot) * V, c1 = u < rot ? c0 + p.pairs : c0 + rest * V;
            TV a = *reinterpret_cast<const TV *>(x + c0), d = *reinterpret_cast<const TV *>(x + c1);
            if (u < rot) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const f32x2 cs = tr[c0 + e];
                    const float fa = to_f32(a[e]), fd = to_f32(d[e]);
                    a[e] = from_f32<T>(fa * cs[0] - fd * cs[1]);
                    d[e] = from_f32<T>(fd * cs[0] + fa * cs[1]);
                }
            }
            *reinterpret_cast<TV *>(y + c0) = a;
            *reinterpret_cast<TV *>(y + c1) = d;
        } else if (V == 1) {   // one pair
            T a = x[2 * u], d = x[2 * u + 1];
            if (u < p.pairs) {
                const f32x2 cs = tr[u];
                const float fa = to_f32(a), fd = to_f32(d);
                a = from_f32<T>(fa * cs[0] - fd * cs[1]);
                d = from_f32<T>(fd * cs[0] + fa * cs[1]);
            }
            y[2 * u] = a;
            y[2 * u + 1] = d;
        } else {
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const int c0 = (u + part * units) * V;
                TV a = *reinterpret_cast<const TV *>(x + c0);
                if (c0 < 2 * p.pairs) {
#pragma unroll
                    for (int e = 0; e + 1 < V; e += 2) {
                        const f32x2 cs = tr[(c0 + e) / 2];
                        const float fa = to_f32(a[e]), fd = to_f32(a[e + 1]);
                        a[e] = from_f32<T>(fa * cs[0] - fd * cs[1]);
                        a[e + 1] = from_f32<T>(fd * cs[0] + fa * cs[1]);
                    }
                }
                *reinterpret_cast<TV *>(y + c0) = a;
            }
        }
    }
}

inline bool present(const fla_tensor *t) { return t != nullptr && t->data != nullptr; }

// strides of x and y ([B,T,H,D] or [T,H,D]) and the largest piece (a power of two of at most 16 bytes) that divides them
int rows_of(const char *op, const char *name, const fla_tensor *x, const fla_tensor *y, const fla_tensor *like, Rows &r, int &piece) {
    int rc;
    const int types = dt_bit(FLA_BF16) | dt_bit(FLA_F16) | dt_bit(FLA_F32);
    if ((rc = check_tensor(x, op, name, -1, like ? dt_bit(like->dtype) : types))) return rc;
    if ((rc = check_tensor(y, op, "output", -1, dt_bit(x->dtype)))) return rc;
    FLA_REQUIRE(x->ndim == 3 || x->ndim == 4, FLA_ERR_SHAPE, "%s: %s must be [B,T,H,D] or [T,H,D].", op, name);
    FLA_REQUIRE(same_shape(x, y), FLA_ERR_SHAPE, "%s: the output of %s has another shape.", op, name);
    if (like) {
        bool same = like->ndim == x->ndim;
        for (int i = 0; same && i < x->ndim; ++i) same = i == x->ndim - 2 || x->shape[i] == like->shape[i];
        FLA_REQUIRE(same, FLA_ERR_SHAPE, "%s: q and k may differ in their number of heads only.", op);
    }
    FLA_REQUIRE(inner_unit(x) && inner_unit(y), FLA_ERR_SHAPE, "%s: %s and its output must have unit innermost stride.", op, name);
    const int o = x->ndim - 3, size = (int)dtype_size(x->dtype);
    r.x = x->data;
    r.y = y->data;
    r.xb = o ? x->stride[0] : 0;
    r.yb = o ? y->stride[0] : 0;
    r.xt = x->stride[o];
    r.yt = y->stride[o];
    r.xh = x->stride[o + 1];
    r.yh = y->stride[o + 1];
    int64_t all = (int64_t)(reinterpret_cast<uintptr_t>(x->data) | reinterpret_cast<uintptr_t>(y->data));
    for (int i = 0; i < x->ndim - 1; ++i) {
        FLA_REQUIRE(x->stride[i] >= 0 && y->stride[i] >= 0, FLA_ERR_SHAPE, "%s: negative strides are not supported.", op);
        if (x->shape[i] > 1) all |= x->stride[i] * size;
        if (y->shape[i] > 1) all |= y->stride[i] * size;
    }
    FLA_REQUIRE(separate(y), FLA_ERR_SHAPE, "%s: rows of an output overlap.", op);
    while (piece > 1 && all % (piece * size)) piece >>= 1;
    return FLA_OK;
}

template <typename T> void launch(const RotaryParams &p, int piece, dim3 grid, hipStream_t stream) {
#define FLA_ROT(VV)                                                                                                              \
    do {                                                                                                                         \
        if (p.adjacent) FLA_LAUNCH("rotary_axes", stream, (rotary_axes_kernel<T, VV, true>), grid, dim3(kThreads), 0, stream, p);  \
        else FLA_LAUNCH("rotary_axes", stream, (rotary_axes_kernel<T, VV, false>), grid, dim3(kThreads), 0, stream, p);            \
    } while (0)
    if constexpr (sizeof(T) == 2) {
        if (piece == 8) { FLA_ROT(8); return; }
    }
    if (piece >= 4) FLA_ROT(4);
    else if (piece == 2) FLA_ROT(2);
    else FLA_ROT(1);
#undef FLA_ROT
}

int rotary_impl(const fla_tensor *q, const fla_tensor *k, const fla_tensor *positions, const fla_tensor *inv_freq,
                const fla_int_array *axis_of_freq, bool adjacent, bool inverse, const fla_tensor *q_out, const fla_tensor *k_out,
                hipStream_t stream) {
    const char *op = "rotary_axes";
    int rc;
    RotaryParams p{};
    int piece = 8;
    if ((rc = rows_of(op, "q", q, q_out, nullptr, p.q, piece))) return rc;
    FLA_REQUIRE(present(k) == present(k_out), FLA_ERR_NULL, "%s: k and k_out go together.", op);
    if (present(k) && (rc = rows_of(op, "k", k, k_out, q, p.k, piece))) return rc;
    if (q->dtype == FLA_F32 && piece > 4) piece = 4;
    const int o = q->ndim - 3;
    const int64_t B = o ? q->shape[0] : 1, T = q->shape[o], dim = q->shape[o + 2];
    if ((rc = check_tensor(positions, op, "positions", q->ndim - 1, dt_bit(FLA_I32) | dt_bit(FLA_I64)))) return rc;
    const int64_t axes = positions->shape[0];
    FLA_REQUIRE((!o || positions->shape[1] == B) && positions->shape[o + 1] == T, FLA_ERR_SHAPE, "%s: positions must be [axes,B,T] (or [axes,T]) for q.", op);
    if ((rc = check_tensor(inv_freq, op, "inv_freq", 1, dt_bit(FLA_F32)))) return rc;
    const int64_t pairs = inv_freq->shape[0];
    FLA_REQUIRE(is_contiguous(inv_freq), FLA_ERR_SHAPE, "%s: inv_freq must be contiguous.", op);
    FLA_REQUIRE(pairs >= 1 && 2 * pairs <= dim && pairs <= kMaxPairs, FLA_ERR_SHAPE,
                "%s: inv_freq must hold 1 .. %d frequencies and at most half as many as there are channels (%lld), got %lld.", op,
                kMaxPairs, (long long)dim, (long long)pairs);
    FLA_REQUIRE(dim % 2 == 0 && dim <= 4096, FLA_ERR_SHAPE, "%s: the number of channels must be even and at most 4096, got %lld.", op, (long long)dim);
    FLA_REQUIRE(axis_of_freq && axis_of_freq->data && (int64_t)axis_of_freq->size == pairs, FLA_ERR_SHAPE, "%s: axis_of_freq must have one entry for each frequency.", op);
    for (int64_t j = 0; j < pairs; ++j) {
        const int64_t a = axis_of_freq->data[j];
        FLA_REQUIRE(a >= 0 && a < axes && a < 256, FLA_ERR_SHAPE, "%s: axis_of_freq names axis %lld of %lld.", op, (long long)a, (long long)axes);
        p.axis[j] = (uint8_t)a;
    }
    const int64_t heads = q->shape[o + 1] + (present(k) ? k->shape[o + 1] : 0);
    const int64_t tokens = B * T;
    if (tokens == 0 || heads == 0) return FLA_OK;
    FLA_REQUIRE(heads <= 65536 && T < ((int64_t)1 << 31), FLA_ERR_SHAPE, "%s: sizes exceed the supported range.", op);
    // pieces divide the rotated half and, together, the rest (adjacent pairs: the rotated part and half a row)
    while (piece > 1 && (adjacent ? (2 * pairs % piece || dim % (2 * piece)) : (pairs % piece || (dim - 2 * pairs) % (2 * piece)))) piece >>= 1;
    p.positions = positions->data;
    p.pos64 = positions->dtype == FLA_I64;
    p.pos_a = positions->stride[0];
    p.pos_b = o ? positions->stride[1] : 0;
    p.pos_t = positions->stride[o + 1];
    p.adjacent = adjacent;
    p.inverse = inverse;
    p.inv_freq = static_cast<const float *>(inv_freq->data);
    p.tokens = tokens;
    p.t_len = (int)T;
    p.q_heads = (int)q->shape[o + 1];
    p.heads = (int)heads;
    p.dim = (int)dim;
    p.pairs = (int)pairs;
    // Four tokens a workgroup from 4096 on (32 + 8 heads of 128, all channels, bf16: 256 tokens 4.4 us with one and 6.1 with four,
    // 2048 9.8 and 10.4, 4096 16.7 and 16.0, 8192 34.4 and 34.3; at 32768 one is ahead again, 117 and 125).
    p.tokens_per_wg = tokens >= 4096 ? kMaxTokens : 1;
    const int64_t groups = (tokens + p.tokens_per_wg - 1) / p.tokens_per_wg;
    FLA_REQUIRE(groups * kThreads < ((int64_t)1 << 32), FLA_ERR_SHAPE, "%s: too many tokens.", op);
    const dim3 grid((unsigned)groups);
    if (q->dtype == FLA_BF16) launch<bf16>(p, piece, grid, stream);
    else if (q->dtype == FLA_F16) launch<f16>(p, piece, grid, stream);
    else launch<float>(p, piece, grid, stream);
    FLA_HIP_CHECK(hipGetLastError());
    return FLA_OK;
}

}  // namespace
}  // namespace fla

extern "C" int fla_rotary_axes(const fla_tensor *q, const fla_tensor *k, const fla_tensor *positions, const fla_tensor *inv_freq,
                               const fla_int_array *axis_of_freq, bool adjacent, bool inverse, const fla_tensor *q_out,
                               const fla_tensor *k_out, void *stream) {
    return fla::guarded([&] {
        return fla::rotary_impl(q, k, positions, inv_freq, axis_of_freq, adjacent, inverse, q_out, k_out, static_cast<hipStream_t>(stream));
    });
}
