// paged_kv_attention for few query rows (decode, checking of speculated tokens), and the join of split key axes.
//   s_t = scale * ks_page (q . k8_t),  o = sum_t e^{s_t - m} vs_page v8_t / sum_t e^{s_t - m}
// Bound by HBM: each code is read once, with loads that leave the caches alone (a code is not read again in this call).  The
// waves of a workgroup take 32-token steps of a chunk in turn, each with its own running maximum, sum and accumulators (the
// walk of paged_attention.h: no LDS, no barrier), and are joined once at the end.
// Measured, 32 heads on 8 of 128: 128 ragged requests to 8192 tokens 187 us + 5.7 us of join for 1.04 GB, one of 262 k tokens
// 89 + 5.4 us for 537 MB (both with a part of the codes in the Infinity Cache); four to 1100 tokens 12.0 us (32 workgroups: 56 %
// of the waves' time is waiting for lengths, table and codes, 18 % for a turn to issue, 27 % issues); 24 heads on 4 of 64, 48
// requests of 1 to 7 rows 24 + 6.8 us.
#include "paged_attention.h"

namespace fla {
namespace {

template <int CODE, int D, int NC, int W, bool WIDE, Loads L>
__global__ void __launch_bounds__(W * 64, NC == 2 && D == 128 ? 3 : 2) paged_decode_kernel(const AttnParams p) {
    constexpr int kRows = 16 * NC;
    __shared__ float lds_ml[W][kRows][2];
    __shared__ u32x4 lds_q[NC > 1 ? NC * (D / 32) * 64 : 1];
    __shared__ f32x4 lds_o[W / 2][D / 16 * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), g = lane >> 4, i = lane & 15;
    const int head = blockIdx.x % p.heads, item = blockIdx.x / p.heads;
    if (p.clear_tail) clear_tail<W * 64>(p, head, D, item, gridDim.x / p.heads);
    int base;
    const Item it = find_item<kRows>(p, item, false, base);
    if (!it.found) return;
    const int64_t from = (int64_t)it.chunk * it.units * kUnit;
    const int t0 = (int)min(from, (int64_t)INT32_MAX - 65536) + 32 * wave;
    const int32_t *row = p.table + it.r * p.table_s;
    PageWindow<WIDE> pages;
    pages.fill(p, row, t0, 32 * W);
    const Request rq = request_of(p, it.r);
    Walk<CODE, D, NC, WIDE, L> walk;
    walk.start(p, rq, row, head, it.tile * kRows, lds_q);
    const int end = it.chunks == 1 ? walk.most : (int)min((int64_t)walk.most, from + (int64_t)it.units * kUnit);
    walk.run(p, row, pages, head, t0, 32 * W, end);
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
        const float by = walk.l[c] == 0.f ? 0.f : exp2f(walk.m[c] - m[c]);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) walk.o[c][j] *= by;
    }
    // one column tile at a time, so that the room does not keep other workgroups off the compute unit
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int half = W / 2; half >= 1; half >>= 1) {
            if (wave >= half && wave < 2 * half) {
#pragma unroll
                for (int j = 0; j < D / 16; ++j) lds_o[wave - half][j * 64 + lane] = walk.o[c][j];
            }
            __syncthreads();
            if (wave < half) {
#pragma unroll
                for (int j = 0; j < D / 16; ++j) walk.o[c][j] += lds_o[wave][j * 64 + lane];
            }
            if (half > 1 || c + 1 < NC) __syncthreads();
        }
    if (wave == 0) walk.store(p, rq, it, item, head, kRows, 0, m, l);
}

// Joins the chunks of a tile, a query row of it at a time: by one wave (WAVES = 1, a workgroup of four takes four rows), or
// by all WAVES of a workgroup, which take the chunks in turn (few rows with many chunks each).
template <int V> struct Joined {
    float m = kNegInf, l = 0.f, o[V] = {};
    // chunks from, from + by, ...; four in flight
    __device__ __forceinline__ void walk(const AttnParams &p, int64_t first, int64_t step, int from, int by, int chunks, int D, int lane) {
        for (int c0 = from; c0 < chunks; c0 += 4 * by) {
            float mc[4], lc[4], oc[4][V], best = m;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int c = c0 + u * by;
                const int64_t slot = first + min(c, chunks - 1) * step;
                const f32x2 ml = *reinterpret_cast<const f32x2 *>(p.part_ml + slot * 2);
                mc[u] = ml[0];
                lc[u] = c < chunks ? ml[1] : 0.f;
#pragma unroll
                for (int x = 0; x < V; ++x) oc[u][x] = p.part_o[slot * D + lane * V + x];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) best = fmaxf(best, mc[u]);
            scale_to(best);
#pragma unroll
            for (int u = 0; u < 4; ++u) add(mc[u], lc[u], oc[u]);
        }
    }
    __device__ __forceinline__ void scale_to(float best) {
        const float by = l == 0.f ? 0.f : exp2f(m - best);
        l *= by;
#pragma unroll
        for (int x = 0; x < V; ++x) o[x] *= by;
        m = best;
    }
    __device__ __forceinline__ void add(float mc, float lc, const float (&oc)[V]) {   // mc <= m
        if (lc == 0.f) return;                                                         // a chunk with no token that the row sees
        const float by = exp2f(mc - m);
        l += by * lc;
#pragma unroll
        for (int x = 0; x < V; ++x) o[x] += by * oc[x];
    }
};

template <int D, int ROWS, int WAVES>
__global__ void __launch_bounds__(64 * (WAVES > 4 ? WAVES : 4)) paged_join_kernel(const AttnParams p) {
    constexpr int V = D / 64;
    __shared__ float lds_m[WAVES], lds_l[WAVES], lds_o[WAVES][D];
    int base;
    const int head = blockIdx.x % p.heads;
    const Item it = find_item<ROWS>(p, blockIdx.x / p.heads, true, base);
    if (!it.found || it.chunks == 1 || base < 0 || base > p.items - it.chunks) return;    // the last two: cu_seqlens that descend
    const Request rq = request_of(p, it.r);
    const float unit = scale_unit(p, p.table + it.r * p.table_s, head);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), rows = min(ROWS, rq.rows - it.tile * ROWS);
    for (int in_tile = WAVES == 1 ? blockIdx.y * 4 + wave : blockIdx.y; in_tile < rows; in_tile += gridDim.y * (WAVES == 1 ? 4 : 1)) {
        const int r = it.tile * ROWS + in_tile;
        Joined<V> sum;
        sum.walk(p, ((int64_t)base * p.heads + head) * ROWS + in_tile, (int64_t)p.heads * ROWS, WAVES == 1 ? 0 : wave, WAVES, it.chunks, D, lane);
        if (WAVES > 1) {
            if (lane == 0) {
                lds_m[wave] = sum.m;
                lds_l[wave] = sum.l;
            }
#pragma unroll
            for (int x = 0; x < V; ++x) lds_o[wave][lane * V + x] = sum.o[x];
            __syncthreads();
            if (wave == 0) {
                float best = sum.m;
                for (int w = 1; w < WAVES; ++w) best = fmaxf(best, lds_m[w]);
                sum.scale_to(best);
                for (int w = 1; w < WAVES; ++w) {
                    float o[V];
#pragma unroll
                    for (int x = 0; x < V; ++x) o[x] = lds_o[w][lane * V + x];
                    sum.add(lds_m[w], lds_l[w], o);
                }
            }
        }
        if (WAVES == 1 || wave == 0) {
            const int tok = r / p.group, h = head * p.group + r - tok * p.group;
            const float by = sum.l > 0.f || sum.l != sum.l ? unit / sum.l : 0.f;
            elem *dst = static_cast<elem *>(p.out) + (int64_t)(rq.first + tok) * p.o_t + (int64_t)h * p.o_h;
#pragma unroll
            for (int x = 0; x < V; ++x) dst[lane * V + x] = (elem)(sum.o[x] * by);
            if (p.lse && lane == 0) p.lse[(int64_t)(rq.first + tok) * p.lse_t + (int64_t)h * p.lse_h] = log_sum(sum.m, sum.l);
        }
        if (WAVES > 1) __syncthreads();
    }
}

template <int CODE, int D, int NC, int W, bool WIDE, Loads L> int launch(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    const dim3 grid((unsigned)(plan.items * p.heads));
    FLA_LAUNCH("paged_kv_attention", stream, (paged_decode_kernel<CODE, D, NC, W, WIDE, L>), grid, dim3(W * 64), 0, stream, p);
    FLA_HIP_CHECK(hipGetLastError());
    return FLA_OK;
}

template <int CODE, int D, bool WIDE> int launch_rows(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    if (plan.nc == 1) {
        if (plan.waves == 8) return launch<CODE, D, 1, 8, WIDE, kAhead>(p, plan, stream);
        return launch<CODE, D, 1, 4, WIDE, kAheadOnce>(p, plan, stream);
    }
    return launch<CODE, D, 2, 4, WIDE, kAheadOnce>(p, plan, stream);
}

template <int CODE, int D> int launch_page(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    return p.shift >= 5 ? launch_rows<CODE, D, true>(p, plan, stream) : launch_rows<CODE, D, false>(p, plan, stream);
}

template <int CODE> int launch_dim(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    return plan.dim == 64 ? launch_page<CODE, 64>(p, plan, stream) : plan.dim == 128 ? launch_page<CODE, 128>(p, plan, stream) : launch_page<CODE, 256>(p, plan, stream);
}

template <int ROWS> int launch_join(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    constexpr int kMany = 16;
    const int rows = plan.longest_rows < ROWS ? plan.longest_rows : ROWS;
    // 16 waves on a row from 16 chunks of a tile on (decode of 1 x 262 k tokens 93 us, 99 with one wave a row; 1 x 32 k 22 and 28;
    // 4 x 32 k, 16 chunks, 52.4 and 51.9; 16 x 8 k, 4 chunks, 52.9 and 50.4)
    const bool many = p.target >= 16 * plan.tiles;
    const dim3 grid((unsigned)(plan.tiles * p.heads), (unsigned)(many ? rows : (rows + 3) / 4));
#define FLA_JOIN(DD)                                                                                                                           \
    do {                                                                                                                                       \
        if (many) FLA_LAUNCH("paged_kv_attention_join", stream, (paged_join_kernel<DD, ROWS, kMany>), grid, dim3(64 * kMany), 0, stream, p);  \
        else FLA_LAUNCH("paged_kv_attention_join", stream, (paged_join_kernel<DD, ROWS, 1>), grid, dim3(256), 0, stream, p);                  \
    } while (0)
    if (plan.dim == 64) FLA_JOIN(64);
    else if (plan.dim == 128) FLA_JOIN(128);
    else FLA_JOIN(256);
#undef FLA_JOIN
    FLA_HIP_CHECK(hipGetLastError());
    return FLA_OK;
}

}  // namespace

int FLA_PAGED(launch_paged_decode)(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    return plan.code == FLA_I8 ? launch_dim<FLA_I8>(p, plan, stream) : launch_dim<FLA_F8E4M3>(p, plan, stream);
}

int FLA_PAGED(launch_paged_join)(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream) {
    return plan.nc == 1 ? launch_join<16>(p, plan, stream) : plan.nc == 2 ? launch_join<32>(p, plan, stream) : launch_join<64>(p, plan, stream);
}

}  // namespace fla
