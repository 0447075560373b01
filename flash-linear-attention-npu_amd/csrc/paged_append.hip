// paged_kv_append: new tokens' rows into the pages of a cache held in 8 bits, one scale for each page and head.
//   s = smallest power of two with max|x| / s <= 448 (e4m3) or 127 (int8) over what the page and head hold so far
//   code = round_to_nearest_even(x / s)
// Scales are powers of two so that x / s is exact and only the rounding to the code loses anything: an e4m3 code keeps
// its relative precision whatever the scale's mantissa would be, int8 codes lose at most one bit of range, and converting
// the codes of a page whose scale grows is exact for e4m3 (down to its subnormals) and one rounding for int8, so that a
// page filled token by token does not drift.
// Bound by HBM for a prefill, by latency for a decode step.  The rows of one page (a run: ascending slots) and one head
// of k or v are a unit of W waves: the rows pass through registers once (maximum, then codes), 16 bytes per load.  A
// workgroup looks for the first rows of runs among a few tokens (slots in lanes, runs as bit masks); a run belongs to the
// workgroup of its first row.  Maxima are taken on the bit patterns, two 16-bit elements an instruction.
// Measured: 110 k tokens of 8 heads of 128, pages of 64: 134 us for 679 MB = 5.1 TB/s, the rate of a copy; 256 single
// rows: 5.7 us.
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
    int shift, heads, dim, row_shift, tokens_per_wg;   // row_shift: log2 of the 8-element pieces of a row
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

// Codes as numbers.
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

// Four values, already divided by the scale and inside the range of the codes, as four codes, rounded to nearest even.
template <int CODE> __device__ __forceinline__ unsigned encode4(const float (&v)[4]) {
    if constexpr (CODE == FLA_I8) {
        // 1.5 * 2^23 + v: the sum rounds v to an integer, whose two's complement is the low byte
        unsigned u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) u[e] = __builtin_bit_cast(unsigned, v[e] + 12582912.f);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400u), __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), 0x05040100u);
    } else {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
    }
}
// Infinities to the largest code; NaN stays (e4m3) or turns into 0 (int8).
template <int CODE> __device__ __forceinline__ float into_range(float v) {
    constexpr float kMost = CODE == FLA_I8 ? 127.f : 448.f;
    return v == v ? __builtin_amdgcn_fmed3f(v, -kMost, kMost) : CODE == FLA_I8 ? 0.f : v;
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// Running maximum of magnitudes as bit patterns (magnitudes order like them): two 16-bit values to a dword, or one fp32.
template <typename T> __device__ __forceinline__ unsigned max_bits(unsigned a, unsigned x) {
    if constexpr (sizeof(T) == 2)
        return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, x & 0x7fff7fffu)));
    else
        return max(a, x & 0x7fffffffu);
}
// fp32 magnitude of the larger half (or of the fp32 pattern); infinite or NaN if any element was
template <typename T> __device__ __forceinline__ float magnitude(unsigned bits) {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, bits);
    else return to_f32(__builtin_bit_cast(T, (unsigned short)max(bits & 0xffffu, bits >> 16)));
}

template <typename T> struct Piece8 {                 // eight elements
    static constexpr int kWords = sizeof(T) * 2;
    unsigned w[kWords];
    __device__ __forceinline__ void load(const T *p) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const u32x4 v = reinterpret_cast<const u32x4 *>(p)[i];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * i + e] = v[e];
        }
    }
    __device__ __forceinline__ float get(int e) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[e]);
        else if constexpr (__is_same(T, bf16)) return __builtin_bit_cast(float, (e & 1) ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
        else return to_f32(__builtin_bit_cast(T, (unsigned short)((e & 1) ? w[e >> 1] >> 16 : w[e >> 1])));
    }
};

template <int CODE, typename F> __device__ __forceinline__ void store_piece(uint8_t *at, F &&value) {
    u32x2 code;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = value(4 * half + e);
        code[half] = encode4<CODE>(v);
    }
    *reinterpret_cast<u32x2 *>(at) = code;
}

__device__ __forceinline__ int ones(uint64_t x) { return ~x ? (int)__ffsll((unsigned long long)~x) - 1 : 64; }   // trailing ones

__device__ __forceinline__ int64_t lane_value(int64_t v, int lane) {   // of a wave-uniform lane, into scalar registers
    const unsigned lo = __builtin_amdgcn_readlane((unsigned)v, lane), hi = __builtin_amdgcn_readlane((unsigned)(v >> 32), lane);
    return (int64_t)(((uint64_t)hi << 32) | lo);
}

// pieces of eight elements that a thread holds
template <typename T> constexpr int pieces_held() { return sizeof(T) == 2 ? 16 : 8; }

template <typename T, int CODE, int W>
__global__ void __launch_bounds__(W * 64) paged_kv_append_kernel(const AppendParams p) {
    constexpr int kThreads = W * 64, kHeld = pieces_held<T>();
    __shared__ float wave_max[W];
    const int tid = threadIdx.x, lane = tid & 63;
    const AppendSide s = p.side[blockIdx.z];
    const int head = blockIdx.y, page = 1 << p.shift, row_shift = p.row_shift, row_mask = (1 << row_shift) - 1;
    const int64_t first = (int64_t)blockIdx.x * p.tokens_per_wg;
    const int count = (int)min((int64_t)p.tokens_per_wg, p.tokens - first);
    // the slots of tokens first - 1 + lane and first + 63 + lane: the runs that begin here (at most 32 tokens) and nearly
    // always their ends.  Bit w of (lo, hi): token first - 1 + w continues the run of the one before it.
    const int64_t at = first - 1 + lane;
    const int64_t mine = at >= 0 && at < p.tokens ? p.slots[at] : -2, more = at + 64 < p.tokens ? p.slots[at + 64] : -2;
    const int64_t prev = __shfl_up(mine, 1, kWave), last = __shfl(mine, 63, kWave), up = __shfl_up(more, 1, kWave);
    const int64_t prev_more = lane ? up : last;
    const bool follows = lane >= 1 && prev >= 0 && mine == prev + 1 && (mine & (page - 1)) != 0;
    const uint64_t lo = __ballot(follows), hi = __ballot(prev_more >= 0 && more == prev_more + 1 && (more & (page - 1)) != 0);
    uint64_t starts = __ballot(lane >= 1 && lane <= count && mine >= 0 && (mine >> p.shift) < p.pool && !follows);
    while (starts) {
        const int l = __ffsll((unsigned long long)starts) - 1;
        starts &= starts - 1;
        const int64_t t = first + l - 1, slot = lane_value(mine, l), block = slot >> p.shift;
        const int off = (int)(slot & (page - 1));
        int rows = 1 + ones(lo >> (l + 1));                                       // zeros shift in behind bit 63
        if (rows == 64 - l) {
            rows += ones(hi);
            while (rows >= 128 - l && off + rows < page) {                        // pages of 128 or 256
                const int64_t u = t + rows + lane;
                const int n = ones(__ballot(u < p.tokens && p.slots[min(u, p.tokens - 1)] == slot + rows + lane));
                rows += n;
                if (n < 64) break;
            }
            rows = min(rows, page - off);
        }
        const int pieces = rows << row_shift;
        const T *x = static_cast<const T *>(s.x) + t * s.x_t + head * s.x_h;
        const unsigned x_t = (unsigned)s.x_t, c_t = (unsigned)s.c_t;              // rows of a page: 32-bit offsets
        float *scale = s.scales + block * s.s_p + head * s.s_h;
        const float before = off > 0 ? *scale : 0.f;
        Piece8<T> held[kHeld];
        unsigned bits = 0;
#pragma unroll
        for (int m = 0; m < kHeld; ++m) {
            const int i = tid + m * kThreads;
            if (m == 0 || m * kThreads < pieces) {
                const int j = min(i, pieces - 1);                                 // a piece too many is read twice
                held[m].load(x + ((unsigned)(j >> row_shift) * x_t + (j & row_mask) * 8));
            }
        }
#pragma unroll
        for (int m = 0; m < kHeld; ++m)
            if (m == 0 || m * kThreads < pieces) {
#pragma unroll
                for (int w = 0; w < Piece8<T>::kWords; ++w) bits = max_bits<T>(bits, held[m].w[w]);
            }
        float most = magnitude<T>(bits);
        bool odd = !(most < INFINITY);
        if (__any(odd)) {                                                         // infinities or NaN: the maximum of the others
            most = 0.f;
#pragma unroll
            for (int m = 0; m < kHeld; ++m)
                if (m * kThreads < pieces) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float a = fabsf(held[m].get(e));
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
        const float after = fmaxf(fabsf(before), step_for<CODE>(most));           // a negative scale comes from outside
        uint8_t *cache = static_cast<uint8_t *>(s.cache) + block * s.c_p + head * s.c_h;
        if (after > before) {
            const float ratio = before / after;
            for (int i = tid; i < off << row_shift; i += kThreads) {              // earlier codes to the new scale
                u32x2 *to = reinterpret_cast<u32x2 *>(cache + ((unsigned)(i >> row_shift) * c_t + (i & row_mask) * 8));
                u32x2 code = *to;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    float v[4];
                    decode4<CODE>(code[w], v);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = CODE == FLA_I8 ? fminf(v[e] * ratio, 127.f) : v[e] * ratio;   // -128 times -1
                    code[w] = encode4<CODE>(v);
                }
                *to = code;
            }
        }
        // a power of two (every scale this operator writes): an exact product; another scale from outside: a division
        const bool exact = (__builtin_bit_cast(unsigned, after) & 0x7fffffu) == 0;
        const float inv = after > 0.f ? 1.f / after : 1.f;                        // scale 0: zeros, and what is not finite as it is
        const bool plain = exact && !__any(odd);
#pragma unroll
        for (int m = 0; m < kHeld; ++m) {
            const int i = tid + m * kThreads;
            if (i < pieces) {
                uint8_t *to = cache + ((unsigned)(off + (i >> row_shift)) * c_t + (i & row_mask) * 8);
                if (plain) store_piece<CODE>(to, [&](int e) { return held[m].get(e) * inv; });
                else store_piece<CODE>(to, [&](int e) { return into_range<CODE>(exact ? held[m].get(e) * inv : held[m].get(e) / after); });
            }
        }
        if (W > 1) __syncthreads();                                               // every wave has read the old scale
        if (tid == 0) *scale = after;
    }
}

template <typename T, int CODE> int launch(AppendParams &p, hipStream_t stream) {
    const int64_t unit = ((int64_t)p.dim << p.shift) / 8 / pieces_held<T>();      // threads that hold a full page
    // Tokens per workgroup: as many as leave about 8192 workgroups, so that a decode step gets one for each row and a
    // prefill few that find no first row (110 k tokens, 8 heads of 128, pages of 64: 1 token 491 us, 4 195 us, 16 or 32
    // 135 us; 256 single rows: 1 to 8 tokens alike, 32 tokens twice the time).
    p.tokens_per_wg = 1;
    while (p.tokens_per_wg < 32 && p.tokens * p.heads * 2 >= (int64_t)8192 * 2 * p.tokens_per_wg) p.tokens_per_wg *= 2;
    const dim3 grid((unsigned)((p.tokens + p.tokens_per_wg - 1) / p.tokens_per_wg), (unsigned)p.heads, 2);
#define FLA_APPEND(W) FLA_LAUNCH("paged_kv_append", stream, (paged_kv_append_kernel<T, CODE, W>), grid, dim3(W * 64), 0, stream, p)
    if (unit <= 64) FLA_APPEND(1);
    else if (unit <= 256) FLA_APPEND(4);
    else FLA_APPEND((sizeof(T) == 2 ? 8 : 16));
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
    const Folded rows[2] = {Folded(key), Folded(value)}, codes[2] = {Folded(key_cache), Folded(value_cache)}, steps[2] = {Folded(key_scales), Folded(value_scales)};
    const fla_tensor *x[2] = {rows[0], rows[1]}, *cache[2] = {codes[0], codes[1]}, *scales[2] = {steps[0], steps[1]};
    for (int i = 0; i < 2; ++i) {
        if ((rc = check_cache(op, i ? "value_cache" : "key_cache", cache[i], i ? "value_scales" : "key_scales", scales[i], i ? &shape : nullptr, shape))) return rc;
        if ((rc = check_tensor(x[i], op, i ? "value" : "key", 3, i ? dt_bit(key->dtype) : dt_bit(FLA_BF16) | dt_bit(FLA_F16) | dt_bit(FLA_F32)))) return rc;
        FLA_REQUIRE(x[i]->shape[1] == shape.heads && x[i]->shape[2] == shape.dim && x[i]->shape[0] == key->shape[0], FLA_ERR_SHAPE,
                    "%s: %s must be [T,%lld,%lld] as the cache.", op, i ? "value" : "key", (long long)shape.heads, (long long)shape.dim);
        FLA_REQUIRE(inner_unit(x[i]) && x[i]->stride[0] >= 0 && x[i]->stride[1] >= 0 && x[i]->stride[0] % 8 == 0 && x[i]->stride[1] % 8 == 0 &&
                        reinterpret_cast<uintptr_t>(x[i]->data) % 16 == 0,
                    FLA_ERR_SHAPE, "%s: rows of %s must be contiguous and 16-byte aligned.", op, i ? "value" : "key");
        FLA_REQUIRE(separate(cache[i]), FLA_ERR_SHAPE, "%s: rows of %s overlap.", op, i ? "value_cache" : "key_cache");
        FLA_REQUIRE(separate(scales[i]), FLA_ERR_SHAPE, "%s: elements of %s overlap.", op, i ? "value_scales" : "key_scales");
        // rows of a page are addressed with 32-bit offsets
        FLA_REQUIRE(x[i]->stride[0] < ((int64_t)1 << 21) && cache[i]->stride[2] < ((int64_t)1 << 23), FLA_ERR_UNSUPPORTED,
                    "%s: tokens of %s or its cache lie too far apart.", op, i ? "value" : "key");
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
    FLA_REQUIRE(p.tokens < ((int64_t)1 << 26), FLA_ERR_SHAPE, "%s: too many tokens.", op);
    FLA_REQUIRE(key_cache->data != value_cache->data && key_scales->data != value_scales->data, FLA_ERR_SHAPE,
                "%s: keys and values need caches and scales of their own.", op);
    p.row_shift = __builtin_ctz((unsigned)p.dim / 8);
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
