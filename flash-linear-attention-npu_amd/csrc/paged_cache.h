// Host-side checks shared by the operators on the paged 8-bit cache: codes [P,H,block,D], scales [P,H].
#pragma once

#include "common.h"
#include "device_utils.h"

namespace fla {

struct CacheShape {
    int64_t pool = 0, heads = 0, block = 0, dim = 0;
    int shift = 0, code = 0;
};

// A descriptor whose extents of one have stride 0: theirs leads nowhere and may be anything.
struct Folded {
    fla_tensor t;
    const fla_tensor *from;
    explicit Folded(const fla_tensor *x) : t(x ? *x : fla_tensor{}), from(x) {
        for (int i = 0; i < t.ndim && i < FLA_MAX_DIMS; ++i)
            if (t.shape[i] == 1) t.stride[i] = 0;
    }
    operator const fla_tensor *() const { return from ? &t : nullptr; }
};

// The pages of each request, i32 [N,M]; a table without columns has no data.
inline int check_table(const char *op, const fla_tensor *table) {
    const bool empty = table != nullptr && table->ndim == 2 && table->dtype == FLA_I32 && table->shape[0] >= 0 && table->shape[1] == 0;
    return empty ? FLA_OK : check_tensor(table, op, "block_table", 2, dt_bit(FLA_I32));
}

// `like`: the shape the cache must have (the value cache against the key cache), or NULL
inline int check_cache(const char *op, const char *name, const fla_tensor *cache, const char *scales_name, const fla_tensor *scales,
                       const CacheShape *like, CacheShape &shape) {
    int rc;
    if ((rc = check_tensor(cache, op, name, 4, dt_bit(FLA_I8) | dt_bit(FLA_F8E4M3)))) return rc;
    if ((rc = check_tensor(scales, op, scales_name, 2, dt_bit(FLA_F32)))) return rc;
    CacheShape s;
    s.pool = cache->shape[0];
    s.heads = cache->shape[1];
    s.block = cache->shape[2];
    s.dim = cache->shape[3];
    s.code = cache->dtype;
    FLA_REQUIRE(like == nullptr || (like->pool == s.pool && like->heads == s.heads && like->block == s.block && like->dim == s.dim && like->code == s.code),
                FLA_ERR_SHAPE, "%s: key_cache and value_cache must have the same shape and type.", op);
    FLA_REQUIRE(s.block >= 16 && s.block <= 256 && (s.block & (s.block - 1)) == 0, FLA_ERR_UNSUPPORTED,
                "%s: a page of %s must hold a power of two from 16 to 256 tokens, got %lld.", op, name, (long long)s.block);
    FLA_REQUIRE(s.dim == 64 || s.dim == 128 || s.dim == 256, FLA_ERR_UNSUPPORTED, "%s: head size must be 64, 128 or 256, got %lld.", op, (long long)s.dim);
    FLA_REQUIRE(s.pool >= 1 && s.pool < ((int64_t)1 << 31) && s.heads >= 1 && s.heads <= 65535, FLA_ERR_SHAPE, "%s: %s needs at least one page and 1 .. 65535 heads.", op, name);
    bool aligned = inner_unit(cache) && reinterpret_cast<uintptr_t>(cache->data) % 16 == 0;
    for (int i = 0; i < 3; ++i) aligned = aligned && cache->stride[i] >= 0 && cache->stride[i] % 16 == 0;
    FLA_REQUIRE(aligned, FLA_ERR_SHAPE, "%s: rows of %s must be contiguous and 16-byte aligned.", op, name);
    FLA_REQUIRE(scales->shape[0] == s.pool && scales->shape[1] == s.heads && scales->stride[0] >= 0 && scales->stride[1] >= 0, FLA_ERR_SHAPE,
                "%s: %s must be [%lld,%lld].", op, scales_name, (long long)s.pool, (long long)s.heads);
    s.shift = __builtin_ctzll((unsigned long long)s.block);
    shape = s;
    return FLA_OK;
}

}  // namespace fla
