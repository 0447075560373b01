// paged_kv_plan: where the new tokens of a step go in a paged cache.
//   need_r = min(ceil((c_r + q_r) / P), M) - min(ceil(c_r / P), M),   base_r = sum_{i<r} need_i,   cu_r = sum_{i<r} q_i
//   table[r, old_r + j] = free[base_r + j];  token t of request r: position c_r + t - cu_r, slot = page * P + offset
// A few kilobytes for a decode step: bound by latency, so the whole plan is ONE launch.  Every workgroup scans all
// lengths for itself (two prefix sums over tiles of 1024 requests in LDS) instead of waiting for another one's sums, then
// fills the pieces of 256 tokens and of 256 new pages that fall to it; a token finds its request by
// bisection in the tile's sums.  A slot in a page that this step opens is computed from the free list, never read back
// from the table, so no workgroup depends on another's writes.  Measured: 256 requests of one token 5.6 us, 64 requests of 110 k
// tokens in pages of 16 6.4 us (a launch alone: 1.8 us); four tokens a thread: 9.7 us.
#include "common.h"
#include "device_utils.h"
#include "paged_cache.h"

namespace fla {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 4;                       // requests per thread and tile
constexpr int kTile = kThreads * kPer;
constexpr int kPiece = kThreads;              // tokens or new pages a workgroup takes at a time: one for each thread

struct PlanParams {
    const int32_t *context, *query, *free_blocks, *state_rows;
    int32_t *table;
    int64_t table_s;
    int n, width, nfree, tokens, shift;
    int64_t *slots;
    int32_t *positions, *cu, *seq, *used, *state_indices;
};

__device__ __forceinline__ int64_t shfl_up64(int64_t v, int d) {
    const int lo = __shfl_up((int)(v & 0xffffffff), d, kWave), hi = __shfl_up((int)(v >> 32), d, kWave);
    return ((int64_t)hi << 32) | (uint32_t)lo;
}

// exclusive prefix sum of v over the workgroup; total: the sum.  Uses sums[kThreads / 64], ends with a barrier pending
// on the caller's next one.
__device__ __forceinline__ int64_t block_exclusive(int64_t v, int64_t *sums, int64_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t inc = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const int64_t up = shfl_up64(inc, d);
        if (lane >= d) inc += up;
    }
    if (lane == 63) sums[wave] = inc;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) {
        if (w < wave) before += sums[w];
        total += sums[w];
    }
    return before + inc - v;
}

// largest i in [0, n) with sums[i] <= x (sums ascending, sums[0] <= x)
__device__ __forceinline__ int bisect(const int64_t *sums, int n, int64_t x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kThreads) paged_kv_plan_kernel(const PlanParams p) {
    __shared__ int64_t first_token[kTile], first_page[kTile];
    __shared__ int32_t lds_context[kTile], lds_old[kTile];
    __shared__ int64_t wave_sums[2][kThreads / kWave];
    const int tid = threadIdx.x;
    const int64_t wg = blockIdx.x, groups = gridDim.x;
    int64_t tokens = 0, pages = 0;                         // sums over the tiles before this one
    for (int r0 = 0; r0 < p.n; r0 += kTile) {
        int64_t q[kPer], need[kPer], sum_q = 0, sum_need = 0;
        int c[kPer], old[kPer];
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int r = r0 + tid * kPer + e;
            c[e] = r < p.n ? max(p.context[r], 0) : 0;
            q[e] = r < p.n ? max(p.query[r], 0) : 0;
            const int64_t round = ((int64_t)1 << p.shift) - 1;
            old[e] = (int)min((c[e] + round) >> p.shift, (int64_t)p.width);
            need[e] = min((c[e] + q[e] + round) >> p.shift, (int64_t)p.width) - old[e];
            sum_q += q[e];
            sum_need += need[e];
        }
        int64_t tile_q, tile_need;
        int64_t at_q = tokens + block_exclusive(sum_q, wave_sums[0], tile_q);
        int64_t at_need = pages + block_exclusive(sum_need, wave_sums[1], tile_need);
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            const int i = tid * kPer + e, r = r0 + i;
            first_token[i] = at_q;
            first_page[i] = at_need;
            lds_context[i] = c[e];
            lds_old[i] = old[e];
            if (wg == 0 && r < p.n) {
                p.cu[r] = (int32_t)min(at_q, (int64_t)INT32_MAX);
                p.seq[r] = (int32_t)min(c[e] + q[e], (int64_t)INT32_MAX);
            }
            at_q += q[e];
            at_need += need[e];
        }
        __syncthreads();
        const int count = min(kTile, p.n - r0);
        // new pages of this tile: entries [pages, pages + tile_need) in pieces dealt to the workgroups in turn
        const int64_t page_end = pages + tile_need;
        for (int64_t piece = pages / kPiece + (wg - pages / kPiece % groups + groups) % groups; piece * kPiece < page_end; piece += groups) {
            const int64_t end = min(page_end, (piece + 1) * kPiece);
            for (int64_t j = max(pages, piece * kPiece) + tid; j < end; j += kThreads) {
                const int i = bisect(first_page, count, j);
                p.table[(r0 + i) * p.table_s + lds_old[i] + (j - first_page[i])] = j < p.nfree ? p.free_blocks[j] : -1;
            }
        }
        const int64_t token_end = min(tokens + tile_q, (int64_t)p.tokens);
        for (int64_t piece = tokens / kPiece + (wg - tokens / kPiece % groups + groups) % groups; piece * kPiece < token_end; piece += groups) {
            const int64_t end = min(token_end, (piece + 1) * kPiece);
            for (int64_t t = max(tokens, piece * kPiece) + tid; t < end; t += kThreads) {
                const int i = bisect(first_token, count, t);
                const int64_t pos = lds_context[i] + (t - first_token[i]), page = pos >> p.shift;
                int64_t slot = -1;
                if (page < p.width) {
                    const int64_t j = first_page[i] + page - lds_old[i];
                    const int block = page < lds_old[i] ? p.table[(r0 + i) * p.table_s + page] : j < p.nfree ? p.free_blocks[j] : -1;
                    if (block >= 0) slot = ((int64_t)block << p.shift) + (pos & ((1 << p.shift) - 1));
                }
                p.slots[t] = slot;
                p.positions[t] = (int32_t)min(pos, (int64_t)INT32_MAX);
                if (p.state_indices) p.state_indices[t] = p.state_rows[r0 + i];
            }
        }
        tokens += tile_q;
        pages += tile_need;
        __syncthreads();
    }
    if (wg == 0 && tid == 0) {
        p.cu[p.n] = (int32_t)min(tokens, (int64_t)INT32_MAX);
        p.used[0] = (int32_t)min(pages, (int64_t)INT32_MAX);
    }
    for (int64_t t = min(tokens, (int64_t)p.tokens) + wg * kThreads + tid; t < p.tokens; t += groups * kThreads) {   // padding
        p.slots[t] = -1;
        p.positions[t] = 0;
        if (p.state_indices) p.state_indices[t] = -1;
    }
}

inline bool present(const fla_tensor *t) { return t != nullptr && t->data != nullptr; }

int vec(const char *op, const fla_tensor *t, const char *name, int dtype, int64_t count) {
    const bool empty = t != nullptr && t->ndim == 1 && t->shape[0] == 0 && t->dtype == dtype;   // may have no data
    const int rc = empty ? FLA_OK : check_tensor(t, op, name, 1, dt_bit(dtype));
    if (rc) return rc;
    FLA_REQUIRE(t->shape[0] == count, FLA_ERR_SHAPE, "%s: %s must have %lld elements, got %lld.", op, name, (long long)count, (long long)t->shape[0]);
    FLA_REQUIRE(is_contiguous(t), FLA_ERR_SHAPE, "%s: %s must be contiguous.", op, name);
    return FLA_OK;
}

int plan_impl(const fla_tensor *context, const fla_tensor *query, const fla_tensor *table, const fla_tensor *free_blocks,
              const fla_tensor *state_rows, int64_t block_size, const fla_tensor *slots, const fla_tensor *positions,
              const fla_tensor *cu, const fla_tensor *seq, const fla_tensor *used, const fla_tensor *state_indices,
              hipStream_t stream) {
    const char *op = "paged_kv_plan";
    int rc;
    if ((rc = check_table(op, table))) return rc;
    const int64_t n = table->shape[0], width = table->shape[1];
    FLA_REQUIRE(width == 0 || (inner_unit(table) && table->stride[0] >= 0 && (n <= 1 || table->stride[0] >= width)), FLA_ERR_SHAPE,
                "%s: block_table must have unit innermost stride and rows that do not overlap.", op);
    FLA_REQUIRE(block_size >= 16 && block_size <= 256 && (block_size & (block_size - 1)) == 0, FLA_ERR_UNSUPPORTED,
                "%s: block_size must be a power of two from 16 to 256, got %lld.", op, (long long)block_size);
    FLA_REQUIRE(n < ((int64_t)1 << 30) && width < ((int64_t)1 << 30), FLA_ERR_SHAPE, "%s: block_table is too large.", op);
    if ((rc = vec(op, context, "context_lens", FLA_I32, n))) return rc;
    if ((rc = vec(op, query, "query_lens", FLA_I32, n))) return rc;
    FLA_REQUIRE(free_blocks && slots, FLA_ERR_NULL, "%s: free_blocks and slot_mapping must not be null.", op);
    if ((rc = vec(op, free_blocks, "free_blocks", FLA_I32, free_blocks->shape[0]))) return rc;
    const int64_t tokens = slots->shape[0];
    FLA_REQUIRE(tokens < ((int64_t)1 << 31) && free_blocks->shape[0] < ((int64_t)1 << 31), FLA_ERR_SHAPE, "%s: sizes exceed int32.", op);
    if ((rc = vec(op, slots, "slot_mapping", FLA_I64, tokens))) return rc;
    if ((rc = vec(op, positions, "positions", FLA_I32, tokens))) return rc;
    if ((rc = vec(op, cu, "cu_seqlens", FLA_I32, n + 1))) return rc;
    if ((rc = vec(op, seq, "seq_lens", FLA_I32, n))) return rc;
    if ((rc = vec(op, used, "blocks_used", FLA_I32, 1))) return rc;
    FLA_REQUIRE(tokens == 0 || present(state_rows) == present(state_indices), FLA_ERR_NULL, "%s: state_rows and state_indices go together.", op);
    if (tokens && present(state_rows)) {
        if ((rc = vec(op, state_rows, "state_rows", FLA_I32, n))) return rc;
        if ((rc = vec(op, state_indices, "state_indices", FLA_I32, tokens))) return rc;
    }
    PlanParams p{};
    p.context = static_cast<const int32_t *>(context->data);
    p.query = static_cast<const int32_t *>(query->data);
    p.free_blocks = static_cast<const int32_t *>(free_blocks->data);
    p.state_rows = present(state_rows) ? static_cast<const int32_t *>(state_rows->data) : nullptr;
    p.table = static_cast<int32_t *>(table->data);
    p.table_s = table->stride[0];
    p.n = (int)n;
    p.width = (int)width;
    p.nfree = (int)free_blocks->shape[0];
    p.tokens = (int)tokens;
    p.shift = __builtin_ctzll((unsigned long long)block_size);
    p.slots = static_cast<int64_t *>(slots->data);
    p.positions = static_cast<int32_t *>(positions->data);
    p.cu = static_cast<int32_t *>(cu->data);
    p.seq = static_cast<int32_t *>(seq->data);
    p.used = static_cast<int32_t *>(used->data);
    p.state_indices = present(state_indices) ? static_cast<int32_t *>(state_indices->data) : nullptr;
    const int64_t pieces = (tokens + kPiece - 1) / kPiece;
    const dim3 grid((unsigned)(pieces < 1 ? 1 : pieces > 1024 ? 1024 : pieces));
    FLA_LAUNCH(op, stream, paged_kv_plan_kernel, grid, dim3(kThreads), 0, stream, p);
    FLA_HIP_CHECK(hipGetLastError());
    return FLA_OK;
}

}  // namespace
}  // namespace fla

extern "C" int fla_paged_kv_plan(const fla_tensor *context_lens, const fla_tensor *query_lens, const fla_tensor *block_table,
                                 const fla_tensor *free_blocks, const fla_tensor *state_rows, int64_t block_size,
                                 const fla_tensor *slot_mapping, const fla_tensor *positions, const fla_tensor *cu_seqlens,
                                 const fla_tensor *seq_lens, const fla_tensor *blocks_used, const fla_tensor *state_indices,
                                 void *stream) {
    return fla::guarded([&] {
        return fla::plan_impl(context_lens, query_lens, block_table, free_blocks, state_rows, block_size, slot_mapping, positions,
                              cu_seqlens, seq_lens, blocks_used, state_indices, static_cast<hipStream_t>(stream));
    });
}
