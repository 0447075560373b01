// Entry point of paged_kv_attention: checks, the choice of kernel and split, and the launches.
#include "paged_attention.h"

namespace fla {
namespace {

inline bool present(const fla_tensor *t) { return t != nullptr && t->data != nullptr; }

int attention_impl(const fla_tensor *q_, const fla_tensor *kc_, const fla_tensor *vc_, const fla_tensor *ks_, const fla_tensor *vs_,
                   const fla_tensor *table, const fla_tensor *lens, const fla_tensor *cu, double scale, int64_t max_query_len,
                   bool clear_tail, const fla_tensor *out_, const fla_tensor *lse_, void *workspace, uint64_t size, hipStream_t stream,
                   uint64_t *query) {
    const char *op = "paged_kv_attention";
    int rc;
    const Folded fq(q_), fkc(kc_), fvc(vc_), fks(ks_), fvs(vs_), fout(out_), flse(lse_);
    const fla_tensor *q = fq, *kc = fkc, *vc = fvc, *ks = fks, *vs = fvs, *out = fout, *lse = flse;
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
    FLA_REQUIRE(separate(out), FLA_ERR_SHAPE, "%s: rows of out overlap.", op);
    if ((rc = check_table(op, table))) return rc;
    if ((rc = check_tensor(lens, op, "seq_lens", 1, dt_bit(FLA_I32)))) return rc;
    const int64_t n = table->shape[0];
    FLA_REQUIRE(lens->shape[0] == n && is_contiguous(lens), FLA_ERR_SHAPE, "%s: seq_lens must be a contiguous tensor of %lld elements.", op, (long long)n);
    FLA_REQUIRE(table->shape[1] == 0 || (inner_unit(table) && table->stride[0] >= 0), FLA_ERR_SHAPE, "%s: block_table must have unit innermost stride.", op);
    if (present(cu)) {
        if ((rc = check_tensor(cu, op, "cu_seqlens", 1, dt_bit(FLA_I32)))) return rc;
        FLA_REQUIRE(cu->shape[0] == n + 1 && is_contiguous(cu), FLA_ERR_SHAPE, "%s: cu_seqlens must be a contiguous tensor of %lld elements.", op, (long long)(n + 1));
    } else {
        FLA_REQUIRE(T == n, FLA_ERR_SHAPE, "%s: without cu_seqlens query must have one row for each of the %lld requests, got %lld.", op, (long long)n, (long long)T);
    }
    if (present(lse)) {
        if ((rc = check_tensor(lse, op, "lse", 2, dt_bit(FLA_F32)))) return rc;
        FLA_REQUIRE(lse->shape[0] == T && lse->shape[1] == heads && lse->stride[0] >= 0 && lse->stride[1] >= 0, FLA_ERR_SHAPE, "%s: lse must be [T,Hq].", op);
        FLA_REQUIRE(separate(lse), FLA_ERR_SHAPE, "%s: elements of lse overlap.", op);
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
    // Up to 64 rows of a request go to the decode kernel, in tiles of 16 or 32: it splits the keys among the waves of a
    // workgroup (48 requests of 1 to 7 rows times 6 heads, contexts to 5 k, when measured: tiles of 32 rows 42 us, one of 64
    // rows 66 us; since then 29 us in tiles of 32).
    const int64_t rows_most = longest * group;
    const bool prefill = rows_most > 64;
    plan.nc = !prefill ? (rows_most <= 16 ? 1 : 2) : dim == 256 ? 2 : 4;
    plan.dim = (int)dim;
    plan.code = shape.code;
    const int64_t rows = 16 * plan.nc;
    plan.tiles = present(cu) ? T * group / rows + n : n * ((group + rows - 1) / rows);
    p.tiles_each = (int)((group + rows - 1) / rows);
    // The split of the key axis.  Lengths are on the device; the host knows the most that a row of the table can name.
    //  - decode: about 512 workgroups (of chunks of at least 256 tokens) where there are few tiles; up to 2048, of chunks of at
    //    least 1024 tokens, where tiles alone fill the chip, since ragged requests balance better (32 heads on 8 of 128,
    //    e4m3: one request of 262 k tokens 102 us with 512 and 115 us with 2048 workgroups; 128 requests of up to 8 k 239
    //    and 211 us);
    //  - tables of at most 2048 tokens: one chunk and one launch, of eight waves (four requests of 1100: 11.6 us against 10.2
    //    to 12.3 us with two launches on the GPU, and one launch less on the host);
    //  - prefill: only where tiles, of one wave each, would leave compute units idle: below 2048 (rows behind 4096 tokens, 32
    //    heads on 8 of 128: 1024 rows split 125 us, whole 247; 2048 rows split 238, whole 297; 4096 rows split 458, whole 431);
    //  - chunks of at least 256 tokens (one prompt of 256 rows behind 1024: 128 tokens 43 us, 256 40, 512 47; one decode of 2100
    //    tokens 12.0, 12.1, 13.9; 64 rows behind 1024 would take 40 us with 128 and 44 with 256).
    const int64_t capacity = table->shape[1] << shape.shift, tiles_all = plan.tiles * shape.heads;
    plan.waves = 4;
    p.min_units = 4;
    p.target = (int)(((!prefill && tiles_all < 256 ? 512 : 2048) + shape.heads - 1) / shape.heads);
    p.few = prefill ? p.target : (int)((512 + shape.heads - 1) / shape.heads);
    if (prefill ? tiles_all >= 2048 : capacity <= 2048) {
        p.target = 0;
        if (plan.nc == 1 && tiles_all < 512) plan.waves = 8;
    }
    plan.items = plan.tiles + p.target;
    FLA_REQUIRE(capacity <= INT32_MAX - 65536, FLA_ERR_SHAPE, "%s: a row of block_table names more than 2^31 - 2^16 tokens.", op);
    FLA_REQUIRE(plan.items * shape.heads * 64 * (prefill ? 1 : plan.waves) < ((int64_t)1 << 32), FLA_ERR_SHAPE, "%s: too many query rows.", op);
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
    p.items = (int)plan.items;
    p.clear_tail = clear_tail && p.cu;
    const bool f16_rows = q->dtype == FLA_F16;
    if (prefill) rc = f16_rows ? launch_paged_prefill_f16(p, plan, stream) : launch_paged_prefill(p, plan, stream);
    else rc = f16_rows ? launch_paged_decode_f16(p, plan, stream) : launch_paged_decode(p, plan, stream);
    if (rc || !p.target) return rc;
    return f16_rows ? launch_paged_join_f16(p, plan, stream) : launch_paged_join(p, plan, stream);
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
