// paged_kv_attention: softmax attention of a few query rows over a paged cache held in 8 bits (decode, checking of
// speculated tokens), the join of split key axes, and the entry point.
//   s_t = scale * ks_page (q . k8_t),  o = sum_t e^{s_t - m} vs_page v8_t / sum_t e^{s_t - m}
// Bound by HBM: each code is read once.  The waves of a workgroup take 32-token steps of a chunk in turn, each with its own
// running maximum, sum and accumulators (the walk of paged_attention.h: no LDS, no barrier), and are joined once at the end.
#include "paged_attention.h"

namespace fla {
namespace {

template <typename T, int CODE, int D, int NC, int W, bool WIDE>
__global__ void __launch_bounds__(W * 64) paged_decode_kernel(const AttnParams p) {
    constexpr int kRows = 16 * NC;
    __shared__ float lds_ml[W][kRows][2];
    extern __shared__ float lds_o[];                       // [W/2][kRows][D]
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, i = lane & 15;
    const int head = blockIdx.x % p.heads, item = blockIdx.x / p.heads;
    if (p.clear_tail && blockIdx.x >= gridDim.x - p.heads) clear_tail<T, W * 64>(p, head, D);
    int base;
    const Item it = find_item<kRows>(p, item, false, base);
    if (!it.found) return;
    const Request rq = request_of(p, it.r);
    Walk<T, CODE, D, NC, WIDE> walk;
    walk.start(p, rq, head, it.tile * kRows);
    const int64_t from = (int64_t)it.chunk * it.units * kUnit;
    const int end = it.chunks == 1 ? walk.most : (int)min((int64_t)walk.most, from + (int64_t)it.units * kUnit);
    if (from < end) walk.run(p, p.table + it.r * p.table_s, head, (int)from + 32 * wave, 32 * W, end);
    walk.finish();
    // join the waves: statistics first, then the accumulators pairwise through LDS
#pragma unroll
    for (int c = 0; c < NC; ++c)
        if (g == 0) {
            lds_ml[wave][16 * c + i][0] = walk.m[c];
            lds_ml[wave][16 * c + i][1] = walk.l[c];
        }
    __syncthreads();
    float m[NC], l[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        m[c] = kNegInf;
        l[c] = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) m[c] = fmaxf(m[c], lds_ml[w][16 * c + i][0]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float lw = lds_ml[w][16 * c + i][1];      // 0: the wave saw no token (its maximum is -inf)
            l[c] += lw == 0.f ? 0.f : lw * exp2f(lds_ml[w][16 * c + i][0] - m[c]);
        }
        const float by = walk.l[c] == 0.f ? 0.f : exp2f(walk.m[c] - m[c]) * walk.r;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) walk.o[c][j] *= by;
    }
#pragma unroll
    for (int half = W / 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
            f32x4 *dst = reinterpret_cast<f32x4 *>(lds_o + (size_t)(wave - half) * kRows * D);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < D / 16; ++j) dst[(c * (D / 16) + j) * 64 + lane] = walk.o[c][j];
        }
        __syncthreads();
        if (wave < half) {
            const f32x4 *src = reinterpret_cast<const f32x4 *>(lds_o + (size_t)wave * kRows * D);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < D / 16; ++j) walk.o[c][j] += src[(c * (D / 16) + j) * 64 + lane];
        }
        if (half > 1) __syncthreads();
    }
    if (wave == 0) walk.store(p, rq, it, item, head, kRows, 0, m, l);
}

// Joins the chunks of a tile: one workgroup for each (tile, cache head, query row), whose waves take the chunks in turn.
constexpr int kJoinWaves = 4;
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(64 * kJoinWaves) paged_join_kernel(const AttnParams p) {
    constexpr int V = D / 64;
    __shared__ float lds_m[kJoinWaves], lds_l[kJoinWaves], lds_o[kJoinWaves][D];
    int base;
    const int head = blockIdx.x % p.heads;
    const Item it = find_item<ROWS>(p, blockIdx.x / p.heads, true, base);
    if (!it.found || it.chunks == 1) return;
    const Request rq = request_of(p, it.r);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = min(ROWS, rq.rows - it.tile * ROWS);
    for (int in_tile = blockIdx.y; in_tile < rows; in_tile += gridDim.y) {
        const int r = it.tile * ROWS + in_tile;
        const int64_t first = ((int64_t)base * p.heads + head) * ROWS + in_tile, step = (int64_t)p.heads * ROWS;
        float m = kNegInf, l = 0.f, o[V];
#pragma unroll
        for (int x = 0; x < V; ++x) o[x] = 0.f;
        for (int c0 = wave; c0 < it.chunks; c0 += 4 * kJoinWaves) {      // four chunks in flight
            float mc[4], lc[4], oc[4][V], best = m;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int c = c0 + u * kJoinWaves;
                const int64_t slot = first + min(c, it.chunks - 1) * step;
                mc[u] = p.part_ml[slot * 2];
                lc[u] = c < it.chunks ? p.part_ml[slot * 2 + 1] : 0.f;
#pragma unroll
                for (int x = 0; x < V; ++x) oc[u][x] = p.part_o[slot * D + lane * V + x];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) best = fmaxf(best, mc[u]);
            const float old = l == 0.f ? 0.f : exp2f(m - best);
            l *= old;
#pragma unroll
            for (int x = 0; x < V; ++x) o[x] *= old;
            m = best;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float by = lc[u] == 0.f ? 0.f : exp2f(mc[u] - best);        // a sum of 0: the chunk has no token that the row sees
                l += by * lc[u];
#pragma unroll
                for (int x = 0; x < V; ++x) o[x] += lc[u] == 0.f ? 0.f : by * oc[u][x];
            }
        }
        if (lane == 0) {
            lds_m[wave] = m;
            lds_l[wave] = l;
        }
#pragma unroll
        for (int x = 0; x < V; ++x) lds_o[wave][lane * V + x] = o[x];
        __syncthreads();
        if (wave == 0) {
            float best = kNegInf, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kJoinWaves; ++w) best = fmaxf(best, lds_m[w]);
#pragma unroll
            for (int x = 0; x < V; ++x) o[x] = 0.f;
#pragma unroll
            for (int w = 0; w < kJoinWaves; ++w) {
                const float lw = lds_l[w], by = lw == 0.f ? 0.f : exp2f(lds_m[w] - best);
                sum += by * lw;
#pragma unroll
                for (int x = 0; x < V; ++x) o[x] += lw == 0.f ? 0.f : by * lds_o[w][lane * V + x];
            }
            const int tok = r / p.group, h = head * p.group + r - tok * p.group;
            const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
            T *dst = static_cast<T *>(p.out) + (int64_t)(rq.first + tok) * p.o_t + (int64_t)h * p.o_h;
#pragma unroll
            for (int x = 0; x < V; ++x) dst[lane * V + x] = (T)(o[x] * by);
            if (p.lse && lane == 0) p.lse[(int64_t)(rq.first + tok) * p.lse_t + (int64_t)h * p.lse_h] = (best + log2f(sum)) * (1.f / kLog2e);
        }
        __syncthreads();
    }
}

template <typename T, int CODE, int D, int NC, bool WIDE> int launch_decode(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    constexpr int W = NC * D <= 128 ? 8 : 4;
    const dim3 grid((unsigned)(plan.items * p.heads));
    const size_t lds = (size_t)(W / 2) * 16 * NC * D * 4;
    const auto kernel = paged_decode_kernel<T, CODE, D, NC, W, WIDE>;
    if (lds > 48 * 1024) FLA_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    FLA_LAUNCH("paged_kv_attention", stream, kernel, grid, dim3(W * 64), lds, stream, p);
    FLA_HIP_CHECK(hipGetLastError());
    return FLA_OK;
}

template <typename T, int ROWS> int launch_join(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    const dim3 grid((unsigned)(plan.tiles * p.heads), (unsigned)(plan.longest_rows < ROWS ? plan.longest_rows : ROWS)), block(64 * kJoinWaves);
    if (plan.dim == 64) FLA_LAUNCH("paged_kv_attention_join", stream, (paged_join_kernel<T, 64, ROWS>), grid, block, 0, stream, p);
    else if (plan.dim == 128) FLA_LAUNCH("paged_kv_attention_join", stream, (paged_join_kernel<T, 128, ROWS>), grid, block, 0, stream, p);
    else FLA_LAUNCH("paged_kv_attention_join", stream, (paged_join_kernel<T, 256, ROWS>), grid, block, 0, stream, p);
    FLA_HIP_CHECK(hipGetLastError());
    return FLA_OK;
}

template <typename T, int CODE> int launch_dim(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    const bool wide = p.shift >= 5;
#define FLA_NC(DD, NN) return wide ? launch_decode<T, CODE, DD, NN, true>(p, plan, stream) : launch_decode<T, CODE, DD, NN, false>(p, plan, stream)
    if (plan.dim == 64) {
        if (plan.nc == 1) FLA_NC(64, 1);
        FLA_NC(64, 2);
    } else if (plan.dim == 128) {
        if (plan.nc == 1) FLA_NC(128, 1);
        FLA_NC(128, 2);
    } else {
        if (plan.nc == 1) FLA_NC(256, 1);
        FLA_NC(256, 2);
    }
#undef FLA_NC
}

inline bool present(const fla_tensor *t) { return t != nullptr && t->data != nullptr; }

int attention_impl(const fla_tensor *q, const fla_tensor *kc, const fla_tensor *vc, const fla_tensor *ks, const fla_tensor *vs,
                   const fla_tensor *table, const fla_tensor *lens, const fla_tensor *cu, double scale, int64_t max_query_len,
                   bool clear_tail, const fla_tensor *out, const fla_tensor *lse, void *workspace, uint64_t size, hipStream_t stream,
                   uint64_t *query) {
    const char *op = "paged_kv_attention";
    int rc;
    CacheShape shape;
    if ((rc = check_cache(op, "key_cache", kc, "key_scales", ks, nullptr, shape))) return rc;
    if ((rc = check_cache(op, "value_cache", vc, "value_scales", vs, &shape, shape))) return rc;
    if ((rc = check_tensor(q, op, "query", 3, dt_bit(FLA_BF16) | dt_bit(FLA_F16)))) return rc;
    if ((rc = check_tensor(out, op, "out", 3, dt_bit(q->dtype)))) return rc;
    FLA_REQUIRE(same_shape(q, out), FLA_ERR_SHAPE, "%s: out must have the shape of query.", op);
    const int64_t T = q->shape[0], heads = q->shape[1], dim = q->shape[2];
    FLA_REQUIRE(dim == shape.dim, FLA_ERR_SHAPE, "%s: query has %lld channels, the cache %lld.", op, (long long)dim, (long long)shape.dim);
    FLA_REQUIRE(heads >= 1 && heads % shape.heads == 0, FLA_ERR_SHAPE, "%s: %lld query heads are not a multiple of the cache's %lld.", op,
                (long long)heads, (long long)shape.heads);
    for (const fla_tensor *t : {q, out}) {
        FLA_REQUIRE(inner_unit(t) && t->stride[0] >= 0 && t->stride[1] >= 0 && t->stride[0] % 8 == 0 && t->stride[1] % 8 == 0 &&
                        reinterpret_cast<uintptr_t>(t->data) % 16 == 0,
                    FLA_ERR_SHAPE, "%s: rows of %s must be contiguous and 16-byte aligned.", op, t == q ? "query" : "out");
    }
    FLA_REQUIRE((out->stride[0] > 0 || T <= 1) && (out->stride[1] > 0 || heads <= 1), FLA_ERR_SHAPE, "%s: rows of out overlap.", op);
    if ((rc = check_tensor(table, op, "block_table", 2, dt_bit(FLA_I32)))) return rc;
    if ((rc = check_tensor(lens, op, "seq_lens", 1, dt_bit(FLA_I32)))) return rc;
    const int64_t n = table->shape[0];
    FLA_REQUIRE(lens->shape[0] == n && is_contiguous(lens), FLA_ERR_SHAPE, "%s: seq_lens must be a contiguous tensor of %lld elements.", op, (long long)n);
    FLA_REQUIRE(inner_unit(table) && table->stride[0] >= 0, FLA_ERR_SHAPE, "%s: block_table must have unit innermost stride.", op);
    if (present(cu)) {
        if ((rc = check_tensor(cu, op, "cu_seqlens", 1, dt_bit(FLA_I32)))) return rc;
        FLA_REQUIRE(cu->shape[0] == n + 1 && is_contiguous(cu), FLA_ERR_SHAPE, "%s: cu_seqlens must be a contiguous tensor of %lld elements.", op, (long long)(n + 1));
    } else {
        FLA_REQUIRE(T == n, FLA_ERR_SHAPE, "%s: without cu_seqlens query must have one row for each of the %lld requests, got %lld.", op, (long long)n, (long long)T);
    }
    if (present(lse)) {
        if ((rc = check_tensor(lse, op, "lse", 2, dt_bit(FLA_F32)))) return rc;
        FLA_REQUIRE(lse->shape[0] == T && lse->shape[1] == heads && lse->stride[0] >= 0 && lse->stride[1] >= 0, FLA_ERR_SHAPE, "%s: lse must be [T,Hq].", op);
    }
    const int64_t group = heads / shape.heads;
    FLA_REQUIRE(T * group < ((int64_t)1 << 31) && n < ((int64_t)1 << 24) && table->shape[1] < ((int64_t)1 << 31), FLA_ERR_SHAPE, "%s: sizes exceed the supported range.", op);
    FLA_REQUIRE(max_query_len >= 0, FLA_ERR_SHAPE, "%s: max_query_len must not be negative.", op);

    for (const fla_tensor *t : {kc, vc})    // rows of a page are addressed with 32-bit offsets
        FLA_REQUIRE(t->stride[2] < ((int64_t)1 << 23), FLA_ERR_UNSUPPORTED, "%s: tokens of the cache lie too far apart.", op);
    AttnLaunch plan{};
    AttnParams p{};
    const int64_t longest = !present(cu) ? 1 : max_query_len ? (max_query_len < T ? max_query_len : T) : T;
    plan.longest_rows = (int)(longest * group < 4096 ? longest * group : 4096);
    const bool prefill = longest * group > 32;
    plan.nc = prefill ? (dim == 256 ? 2 : 4) : longest * group > 16 ? 2 : 1;
    plan.dim = (int)dim;
    plan.code = shape.code;
    plan.dtype = q->dtype;
    const int64_t rows = 16 * plan.nc;
    plan.tiles = present(cu) ? T * group / rows + n : n * ((group + rows - 1) / rows);
    p.tiles_each = (int)((group + rows - 1) / rows);
    p.target = (int)((1024 + shape.heads - 1) / shape.heads);
    p.min_units = 8;
    const int64_t capacity = table->shape[1] << shape.shift;
    if (prefill ? plan.tiles * shape.heads >= 1024 : capacity <= 2048) p.target = 0;
    plan.items = plan.tiles + p.target;
    FLA_REQUIRE(capacity <= INT32_MAX - 65536, FLA_ERR_SHAPE, "%s: a row of block_table names more than 2^31 - 2^16 tokens.", op);
    FLA_REQUIRE(plan.items * shape.heads < ((int64_t)1 << 31), FLA_ERR_SHAPE, "%s: too many query rows.", op);
    plan.o_bytes = p.target ? (uint64_t)plan.items * shape.heads * rows * dim * 4 : 0;
    plan.bytes = p.target ? plan.o_bytes + (uint64_t)plan.items * shape.heads * rows * 8 : 0;
    if (query) {
        *query = T && n ? plan.bytes : 0;
        return FLA_OK;
    }
    if (T == 0 || n == 0) return FLA_OK;
    FLA_REQUIRE(plan.bytes == 0 || (workspace && size >= plan.bytes), FLA_ERR_WORKSPACE, "%s: workspace of %llu bytes required, got %llu.", op,
                (unsigned long long)plan.bytes, (unsigned long long)size);
    p.part_o = static_cast<float *>(workspace);
    p.part_ml = reinterpret_cast<float *>(static_cast<char *>(workspace) + plan.o_bytes);
    p.q = q->data;
    p.q_t = q->stride[0];
    p.q_h = q->stride[1];
    p.out = out->data;
    p.o_t = out->stride[0];
    p.o_h = out->stride[1];
    p.lse = present(lse) ? static_cast<float *>(lse->data) : nullptr;
    p.lse_t = p.lse ? lse->stride[0] : 0;
    p.lse_h = p.lse ? lse->stride[1] : 0;
    p.kc = static_cast<const uint8_t *>(kc->data);
    p.vc = static_cast<const uint8_t *>(vc->data);
    p.ks = static_cast<const float *>(ks->data);
    p.vs = static_cast<const float *>(vs->data);
    p.kc_p = kc->stride[0];
    p.kc_h = kc->stride[1];
    p.kc_t = kc->stride[2];
    p.vc_p = vc->stride[0];
    p.vc_h = vc->stride[1];
    p.vc_t = vc->stride[2];
    p.ks_p = ks->stride[0];
    p.ks_h = ks->stride[1];
    p.vs_p = vs->stride[0];
    p.vs_h = vs->stride[1];
    p.table = static_cast<const int32_t *>(table->data);
    p.table_s = table->stride[0];
    p.lens = static_cast<const int32_t *>(lens->data);
    p.cu = present(cu) ? static_cast<const int32_t *>(cu->data) : nullptr;
    p.tokens = (int)T;
    p.n = (int)n;
    p.width = (int)table->shape[1];
    p.shift = shape.shift;
    p.group = (int)group;
    p.heads = (int)shape.heads;
    p.pool = (uint32_t)shape.pool;
    p.scale2 = (float)(scale * 1.44269504088896340736);
    p.clear_tail = clear_tail && p.cu;
    if (prefill) rc = launch_paged_prefill(p, plan, stream);
    else if (q->dtype == FLA_BF16) rc = shape.code == FLA_I8 ? launch_dim<bf16, FLA_I8>(p, plan, stream) : launch_dim<bf16, FLA_F8E4M3>(p, plan, stream);
    else rc = shape.code == FLA_I8 ? launch_dim<f16, FLA_I8>(p, plan, stream) : launch_dim<f16, FLA_F8E4M3>(p, plan, stream);
    if (rc || !p.target) return rc;
#define FLA_JOIN(T) (plan.nc == 1 ? launch_join<T, 16>(p, plan, stream) : plan.nc == 2 ? launch_join<T, 32>(p, plan, stream) : launch_join<T, 64>(p, plan, stream))
    return q->dtype == FLA_BF16 ? FLA_JOIN(bf16) : FLA_JOIN(f16);
#undef FLA_JOIN
}

}  // namespace
}  // namespace fla

extern "C" int fla_paged_kv_attention_get_workspace_size(
    const fla_tensor *query, const fla_tensor *key_cache, const fla_tensor *value_cache, const fla_tensor *key_scales,
    const fla_tensor *value_scales, const fla_tensor *block_table, const fla_tensor *seq_lens, const fla_tensor *cu_seqlens, double scale,
    int64_t max_query_len, bool clear_tail, const fla_tensor *out, const fla_tensor *lse, uint64_t *workspace_size) {
    if (!workspace_size) return fla::fail(FLA_ERR_NULL, "paged_kv_attention: workspace_size must not be null.");
    return fla::guarded([&] {
        return fla::attention_impl(query, key_cache, value_cache, key_scales, value_scales, block_table, seq_lens, cu_seqlens, scale,
                                   max_query_len, clear_tail, out, lse, nullptr, 0, nullptr, workspace_size);
    });
}
extern "C" int fla_paged_kv_attention(
    const fla_tensor *query, const fla_tensor *key_cache, const fla_tensor *value_cache, const fla_tensor *key_scales,
    const fla_tensor *value_scales, const fla_tensor *block_table, const fla_tensor *seq_lens, const fla_tensor *cu_seqlens, double scale,
    int64_t max_query_len, bool clear_tail, const fla_tensor *out, const fla_tensor *lse, void *workspace, uint64_t workspace_size,
    void *stream) {
    return fla::guarded([&] {
        return fla::attention_impl(query, key_cache, value_cache, key_scales, value_scales, block_table, seq_lens, cu_seqlens, scale,
                                   max_query_len, clear_tail, out, lse, workspace, workspace_size, static_cast<hipStream_t>(stream), nullptr);
    });
}
