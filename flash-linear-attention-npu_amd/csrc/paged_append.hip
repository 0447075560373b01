// paged_kv_append: new tokens' rows into the pages of a cache held in 8 bits, one scale for each page and head.
//   s = smallest power of two with max|x| / s <= 448 (e4m3) or 127 (int8) over what the page and head hold so far
//   code = round_to_nearest_even(x / s)
// Scales are powers of two so that x / s is exact and only the rounding to the code loses anything: an e4m3 code keeps
// its relative precision whatever the scale's mantissa would be, int8 codes lose at most one bit of range, and converting
// the codes of a page whose scale grows is exact for e4m3 (down to its subnormals) and one rounding for int8, so that a
// page filled token by token does not drift.
// Bound by HBM for a prefill, by latency for a decode step.  The rows of one page (a run: ascending slots) and one head
// of k or v are a unit of W waves: the rows pass through registers once (maximum, then codes), 16 bytes per load.  A
// workgroup looks for the first rows of runs among a few tokens; a run belongs to the workgroup of its first row.
#include "common.h"
#include "paged_cache.h"

namespace fla {
namespace {

struct AppendSide {   // k or v
    const void *x;
    void *cache;
    float *scales;
    int64_t x_t, x_h, c_p, c_h, c_t, s_p, s_h;
};

struct AppendParams {
    AppendSide side[2];
    const int64_t *slots;
    int64_t tokens, pool;
    int shift, heads, dim, tokens_per_wg;
};

// smallest power of two s >= 2^-126 with a / s <= most; 0 for a = 0.  a >= 0 and finite.
template <int CODE> __device__ __forceinline__ float step_for(float a) {
    // a = m 2^e, 1 <= m < 2; the largest code is M 2^E: 1.75 * 2^8 (448) or 1.984375 * 2^6 (127)
    constexpr unsigned kM = CODE == FLA_I8 ? 0x7e0000u : 0x600000u;
    constexpr int kE = CODE == FLA_I8 ? 6 : 8;
    const unsigned bits = __builtin_bit_cast(unsigned, a);
    const int e = (int)(bits >> 23) - kE + ((bits & 0x7fffffu) > kM ? 1 : 0);   // biased exponent of s
    return a == 0.f ? 0.f : __builtin_bit_cast(float, (unsigned)max(e, 1) << 23);
}

// four values (already divided by the scale) as four codes
template <int CODE> __device__ __forceinline__ unsigned encode4(float a, float b, float c, float d) {
    float v[4] = {a, b, c, d};
    if constexpr (CODE == FLA_I8) {
        unsigned r = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float t = v[e] == v[e] ? __builtin_amdgcn_fmed3f(v[e], -127.f, 127.f) : 0.f;
            r |= ((unsigned)(int)rintf(t) & 255u) << (8 * e);
        }
        return r;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = v[e] == v[e] ? __builtin_amdgcn_fmed3f(v[e], -448.f, 448.f) : v[e];
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
    }
}
template <int CODE> __device__ __forceinline__ void decode4(unsigned x, float (&v)[4]) {
    if constexpr (CODE == FLA_I8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)(signed char)(x >> (8 * e));
    } else {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)x, true);
        v[0] = lo[0];
        v[1] = lo[1];
        v[2] = hi[0];
        v[3] = hi[1];
    }
}

// division by a scale: a power of two (every scale this operator writes) takes an exact product
struct Divide {
    float by, inv;
    bool exact;
    __device__ __forceinline__ explicit Divide(float s)
        : by(s), inv(s > 0.f ? 1.f / s : 0.f), exact((__builtin_bit_cast(unsigned, s) & 0x7fffffu) == 0) {}
    __device__ __forceinline__ float operator()(float x) const { return exact || by == 0.f ? x * inv : x / by; }
};

constexpr int kPieces = 8;   // 8-element pieces a thread holds

template <typename T, int CODE, int W>
__global__ void __launch_bounds__(W * 64) paged_kv_append_kernel(const AppendParams p) {
    constexpr int kThreads = W * 64;
    typedef T T8 __attribute__((ext_vector_type(8)));
    __shared__ float wave_max[W];
    __shared__ int run_end;
    const int tid = threadIdx.x, lane = tid & 63;
    const AppendSide s = p.side[blockIdx.z];
    const int head = blockIdx.y, page = 1 << p.shift, ppr = p.dim >> 3;   // 8-element pieces per row
    const int64_t first = (int64_t)blockIdx.x * p.tokens_per_wg, last = min(first + p.tokens_per_wg, p.tokens);
    for (int64_t t = first; t < last; ++t) {
        const int64_t slot = p.slots[t], block = slot >> p.shift;
        if (slot < 0 || block >= p.pool) continue;
        const int off = (int)(slot & (page - 1));
        if (off > 0 && t > 0 && p.slots[t - 1] == slot - 1) continue;   // not the first row of its run
        // rows of the run: while the slots ascend one by one inside the page
        if (tid == 0) run_end = page - off;
        __syncthreads();
        for (int i = tid + 1; i < page - off; i += kThreads)
            if (t + i >= p.tokens || p.slots[t + i] != slot + i) atomicMin(&run_end, i);
        __syncthreads();
        const int rows = run_end, pieces = rows * ppr;
        const T *x = static_cast<const T *>(s.x) + t * s.x_t + head * s.x_h;
        T8 held[kPieces];
        float most = 0.f;
#pragma unroll
        for (int m = 0; m < kPieces; ++m) {
            const int i = tid + m * kThreads;
            if (i < pieces) {
                const int row = i / ppr;
                held[m] = *reinterpret_cast<const T8 *>(x + row * s.x_t + (i - row * ppr) * 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float a = fabsf(to_f32(held[m][e]));
                    most = fmaxf(most, a < INFINITY ? a : 0.f);
                }
            }
        }
#pragma unroll
        for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d, kWave));
        if (W > 1) {
            if (lane == 0) wave_max[tid >> 6] = most;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < W; ++w) most = fmaxf(most, wave_max[w]);
        }
        float *scale = s.scales + block * s.s_p + head * s.s_h;
        const float before = off > 0 ? *scale : 0.f, after = fmaxf(before, step_for<CODE>(most));
        uint8_t *cache = static_cast<uint8_t *>(s.cache) + block * s.c_p + head * s.c_h;
        if (after > before) {
            const float ratio = before / after;
            for (int i = tid; i < off * ppr; i += kThreads) {   // earlier codes to the new scale
                const int row = i / ppr;
                u32x2 *at = reinterpret_cast<u32x2 *>(cache + row * s.c_t + (i - row * ppr) * 8);
                u32x2 code = *at;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    float v[4];
                    decode4<CODE>(code[w], v);
                    code[w] = encode4<CODE>(v[0] * ratio, v[1] * ratio, v[2] * ratio, v[3] * ratio);
                }
                *at = code;
            }
        }
        const Divide div(after);
#pragma unroll
        for (int m = 0; m < kPieces; ++m) {
            const int i = tid + m * kThreads;
            if (i < pieces) {
                const int row = i / ppr;
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = div(to_f32(held[m][e]));
                const u32x2 code = {encode4<CODE>(v[0], v[1], v[2], v[3]), encode4<CODE>(v[4], v[5], v[6], v[7])};
                *reinterpret_cast<u32x2 *>(cache + (off + row) * s.c_t + (i - row * ppr) * 8) = code;
            }
        }
        __syncthreads();   // every thread has read the old scale and run_end
        if (tid == 0) *scale = after;
    }
}

template <typename T, int CODE> int launch(const AppendParams &p, hipStream_t stream) {
    const int64_t unit = ((int64_t)p.dim << p.shift) / 8;   // pieces of a full page
    const dim3 grid((unsigned)((p.tokens + p.tokens_per_wg - 1) / p.tokens_per_wg), (unsigned)p.heads, 2);
#define FLA_APPEND(W) FLA_LAUNCH("paged_kv_append", stream, (paged_kv_append_kernel<T, CODE, W>), grid, dim3(W * 64), 0, stream, p)
    if (unit <= 64 * kPieces) FLA_APPEND(1);
    else if (unit <= 256 * kPieces) FLA_APPEND(4);
    else FLA_APPEND(16);
#undef FLA_APPEND
    FLA_HIP_CHECK(hipGetLastError());
    return FLA_OK;
}

int append_impl(const fla_tensor *key, const fla_tensor *value, const fla_tensor *key_cache, const fla_tensor *value_cache,
                const fla_tensor *key_scales, const fla_tensor *value_scales, const fla_tensor *slots, hipStream_t stream) {
    const char *op = "paged_kv_append";
    int rc;
    CacheShape shape;
    AppendParams p{};
    const fla_tensor *x[2] = {key, value}, *cache[2] = {key_cache, value_cache}, *scales[2] = {key_scales, value_scales};
    for (int i = 0; i < 2; ++i) {
        if ((rc = check_cache(op, i ? "value_cache" : "key_cache", cache[i], i ? "value_scales" : "key_scales", scales[i], i ? &shape : nullptr, shape))) return rc;
        if ((rc = check_tensor(x[i], op, i ? "value" : "key", 3, i ? dt_bit(key->dtype) : dt_bit(FLA_BF16) | dt_bit(FLA_F16) | dt_bit(FLA_F32)))) return rc;
        FLA_REQUIRE(x[i]->shape[1] == shape.heads && x[i]->shape[2] == shape.dim && x[i]->shape[0] == key->shape[0], FLA_ERR_SHAPE,
                    "%s: %s must be [T,%lld,%lld] as the cache.", op, i ? "value" : "key", (long long)shape.heads, (long long)shape.dim);
        FLA_REQUIRE(inner_unit(x[i]) && x[i]->stride[0] >= 0 && x[i]->stride[1] >= 0 && x[i]->stride[0] % 8 == 0 && x[i]->stride[1] % 8 == 0 &&
                        reinterpret_cast<uintptr_t>(x[i]->data) % 16 == 0,
                    FLA_ERR_SHAPE, "%s: rows of %s must be contiguous and 16-byte aligned.", op, i ? "value" : "key");
        AppendSide &s = p.side[i];
        s.x = x[i]->data;
        s.x_t = x[i]->stride[0];
        s.x_h = x[i]->stride[1];
        s.cache = cache[i]->data;
        s.c_p = cache[i]->stride[0];
        s.c_h = cache[i]->stride[1];
        s.c_t = cache[i]->stride[2];
        s.scales = static_cast<float *>(scales[i]->data);
        s.s_p = scales[i]->stride[0];
        s.s_h = scales[i]->stride[1];
    }
    if ((rc = check_tensor(slots, op, "slot_mapping", 1, dt_bit(FLA_I64)))) return rc;
    FLA_REQUIRE(slots->shape[0] == key->shape[0] && is_contiguous(slots), FLA_ERR_SHAPE, "%s: slot_mapping must be a contiguous tensor with one slot for each row.", op);
    p.slots = static_cast<const int64_t *>(slots->data);
    p.tokens = key->shape[0];
    p.pool = shape.pool;
    p.shift = shape.shift;
    p.heads = (int)shape.heads;
    p.dim = (int)shape.dim;
    if (p.tokens == 0) return FLA_OK;
    FLA_REQUIRE(p.tokens < ((int64_t)1 << 31), FLA_ERR_SHAPE, "%s: too many tokens.", op);
    p.tokens_per_wg = 16;
#define FLA_BY_TYPE(CODE)                                                                \
    (key->dtype == FLA_BF16 ? launch<bf16, CODE>(p, stream) : key->dtype == FLA_F16 ? launch<f16, CODE>(p, stream) : launch<float, CODE>(p, stream))
    return shape.code == FLA_I8 ? FLA_BY_TYPE(FLA_I8) : FLA_BY_TYPE(FLA_F8E4M3);
#undef FLA_BY_TYPE
}

}  // namespace
}  // namespace fla

extern "C" int fla_paged_kv_append(const fla_tensor *key, const fla_tensor *value, const fla_tensor *key_cache, const fla_tensor *value_cache,
                                   const fla_tensor *key_scales, const fla_tensor *value_scales, const fla_tensor *slot_mapping, void *stream) {
    return fla::guarded([&] {
        return fla::append_impl(key, value, key_cache, value_cache, key_scales, value_scales, slot_mapping, static_cast<hipStream_t>(stream));
    });
}
