// paged_kv_attention for many query rows (chunked prefill): a wave takes 64 of them (32 for D = 256) over all their keys.
// Bound by the vector and matrix units together.  For a 32-token step and D = 128 a wave issues 64 matrix instructions
// (1024 clocks of the matrix pipe) and about 230 vector ones, 32 of them exponentials; codes are widened once for 64 rows,
// straight from the loads of the wave, with no LDS (but for the queries, which would take registers) and no barrier: with a
// multiple of 8 cache heads the tiles of a head run on one XCD, whose L2 holds its keys.  32 rows a wave took 1150 us where 64
// took 852 (before the priorities of paged_attention.h).
// Measured: 2 x 4096 tokens behind 4096, 32 heads on 8 of 128, e4m3: 784 to 807 us by card in replays and calls back to back, 1020 to
// 1050 TFLOP/s, 73 to 75 % of what a library product of 8192^3 reaches; int8 886 to 904 us; D = 64 524 to 540 us; D = 256 1771 to 1815 us.
#include "paged_attention.h"

namespace fla {
namespace {

template <int CODE, int D, int NC, bool WIDE>
__global__ void __launch_bounds__(64, 2) paged_prefill_kernel(const AttnParams p) {
    constexpr int kRows = 16 * NC;
    __shared__ u32x4 lds_q[NC * (D / 32) * 64];
    const int head = blockIdx.x % p.heads;
    int base;
    const int item = (gridDim.x - 1 - blockIdx.x) / p.heads;      // long rows of a request first
    if (p.clear_tail) clear_tail<64>(p, head, D, item, gridDim.x / p.heads);
    const Item it = find_item<kRows>(p, item, false, base);
    if (!it.found) return;
    const int64_t from = (int64_t)it.chunk * it.units * kUnit;
    const int t0 = (int)min(from, (int64_t)INT32_MAX - 65536);
    const int32_t *row = p.table + it.r * p.table_s;
    PageWindow<WIDE> pages;
    pages.fill(p, row, t0, 32);
    const Request rq = request_of(p, it.r);
    Walk<CODE, D, NC, WIDE, kLate> walk;
    walk.start(p, rq, row, head, it.tile * kRows, lds_q);
    const int end = it.chunks == 1 ? walk.most : (int)min((int64_t)walk.most, from + (int64_t)it.units * kUnit);
    walk.run(p, row, pages, head, t0, 32, end);
    walk.finish();
    walk.store(p, rq, it, item, head, kRows, 0, walk.m, walk.l);
}

template <int CODE> int launch_dim(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    const dim3 grid((unsigned)(plan.items * p.heads));
#define FLA_PREFILL(DD, NN)                                                                                                                     \
    do {                                                                                                                                        \
        if (p.shift >= 5) FLA_LAUNCH("paged_kv_attention", stream, (paged_prefill_kernel<CODE, DD, NN, true>), grid, dim3(64), 0, stream, p);  \
        else FLA_LAUNCH("paged_kv_attention", stream, (paged_prefill_kernel<CODE, DD, NN, false>), grid, dim3(64), 0, stream, p);              \
    } while (0)
    if (plan.dim == 64) FLA_PREFILL(64, 4);
    else if (plan.dim == 128) FLA_PREFILL(128, 4);
    else FLA_PREFILL(256, 2);
#undef FLA_PREFILL
    FLA_HIP_CHECK(hipGetLastError());
    return FLA_OK;
}

}  // namespace

int FLA_PAGED(launch_paged_prefill)(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    return plan.code == FLA_I8 ? launch_dim<FLA_I8>(p, plan, stream) : launch_dim<FLA_F8E4M3>(p, plan, stream);
}

}  // namespace fla
