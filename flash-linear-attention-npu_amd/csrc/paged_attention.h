// Shared by the kernels of paged_kv_attention: parameters, the split of the work among workgroups, code conversion.
//
// Work.  The query rows of request r and one cache head are the q_r * G pairs (token, head of the group), taken as one
// list of rows; a tile is kRows of them.  The key axis of a tile is cut into chunks; an item is (request, tile, chunk) and
// a workgroup takes one item of one cache head.  The lengths live on the device, so the chunk length does too: every
// workgroup sums the work over all requests, derives the chunk length that gives about `target` items, and finds its own
// item by a prefix sum.  The host only bounds the number of items: sum over tiles of ceil(len / chunk) <= target + tiles.
// Items of a tile that has several leave (unnormalised o, max, sum) in the workspace; a second launch joins them.
#pragma once

#include "paged_cache.h"

namespace fla {

constexpr int kUnit = 64;          // tokens: chunks are multiples of this
constexpr float kLog2e = 1.44269504088896340736f;

struct AttnParams {
    const void *q;
    const uint8_t *kc, *vc;
    const float *ks, *vs;
    const int32_t *table, *lens, *cu;
    void *out;
    float *lse;
    float *part_o, *part_ml;       // [items][heads][kRows][D], [items][heads][kRows][2]
    int64_t q_t, q_h, o_t, o_h, lse_t, lse_h, kc_p, kc_h, kc_t, vc_p, vc_h, vc_t, ks_p, ks_h, vs_p, vs_h, table_s;
    int tokens, n, width, shift, group, heads;
    uint32_t pool;
    int target, min_units;         // items wanted; shortest chunk in units; target 0: one chunk for each tile
    float scale2;                  // scale * log2(e)
    bool clear_tail;
};

struct Request {
    int first, rows, units;        // first query token, query rows (tokens * group), key units
    int len, new_tokens;           // cached tokens that the table can name, query tokens
};

__device__ __forceinline__ Request request_of(const AttnParams &p, int r) {
    Request q;
    int a = r, b = r + 1;
    if (p.cu) {
        a = min(max(p.cu[r], 0), p.tokens);
        b = min(max(p.cu[r + 1], a), p.tokens);
    }
    q.first = a;
    q.new_tokens = b - a;
    q.rows = (b - a) * p.group;
    const int64_t most = (int64_t)p.width << p.shift;
    q.len = max(p.lens[r], 0);
    q.units = (int)((min((int64_t)q.len, most) + kUnit - 1) / kUnit);
    return q;
}

struct Item {
    int r, tile, chunk, chunks, units;   // units: of a chunk
    bool found;
};

template <int THREADS> __device__ __forceinline__ int64_t block_sum64(int64_t v, int64_t *sums) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const int lo = __shfl_xor((int)(v & 0xffffffff), d, kWave), hi = __shfl_xor((int)(v >> 32), d, kWave);
        v += ((int64_t)hi << 32) | (uint32_t)lo;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) total += sums[w];
    return total;
}

// Scratch of find_item in LDS.
template <int THREADS> struct ScheduleLds {
    int64_t sums[THREADS / kWave];
    int wave_items[THREADS / kWave];
    Item item;
    int64_t base;
};

// chunk length in units
template <int THREADS, int ROWS> __device__ __forceinline__ int chunk_units(const AttnParams &p, ScheduleLds<THREADS> &lds) {
    if (p.target == 0) return INT32_MAX;
    int64_t work = 0;
    for (int r = threadIdx.x; r < p.n; r += THREADS) {
        const Request q = request_of(p, r);
        work += (int64_t)((q.rows + ROWS - 1) / ROWS) * q.units;
    }
    work = block_sum64<THREADS>(work, lds.sums);
    const int64_t c = (work + p.target - 1) / p.target;
    return (int)min(max(c, (int64_t)p.min_units), (int64_t)INT32_MAX);
}

// The item with number `want`, or (by_tile) the first item of the tile with number `want` and, in base, its number.
template <int THREADS, int ROWS>
__device__ __forceinline__ Item find_item(const AttnParams &p, int64_t want, bool by_tile, ScheduleLds<THREADS> &lds, int64_t &base) {
    const int units = chunk_units<THREADS, ROWS>(p, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x == 0) lds.item.found = false;
    int64_t items_before = 0, tiles_before = 0;
    for (int r0 = 0; r0 < p.n; r0 += THREADS) {
        const int r = r0 + threadIdx.x;
        int tiles = 0, chunks = 0;
        if (r < p.n) {
            const Request q = request_of(p, r);
            tiles = (q.rows + ROWS - 1) / ROWS;
            chunks = q.units <= units ? 1 : (q.units + units - 1) / units;
        }
        const int items = tiles * chunks;
        int inc = items, inc_t = tiles;
#pragma unroll
        for (int d = 1; d < kWave; d <<= 1) {
            const int up = __shfl_up(inc, d, kWave), up_t = __shfl_up(inc_t, d, kWave);
            if (lane >= d) {
                inc += up;
                inc_t += up_t;
            }
        }
        __syncthreads();
        if (lane == 63) {
            lds.wave_items[wave] = inc;
            lds.sums[wave] = inc_t;
        }
        __syncthreads();
        int64_t at = items_before + inc - items, at_t = tiles_before + inc_t - tiles;
#pragma unroll
        for (int w = 0; w < THREADS / kWave; ++w) {
            if (w < wave) {
                at += lds.wave_items[w];
                at_t += lds.sums[w];
            }
            items_before += lds.wave_items[w];
            tiles_before += lds.sums[w];
        }
        const int64_t mine = by_tile ? at_t : at, count = by_tile ? tiles : items;
        if (want >= mine && want < mine + count) {
            const int64_t k = want - mine;
            Item it;
            it.r = r;
            it.tile = (int)(by_tile ? k : k / chunks);
            it.chunk = by_tile ? 0 : (int)(k - (int64_t)it.tile * chunks);
            it.chunks = chunks;
            it.units = units;
            it.found = true;
            lds.item = it;
            lds.base = at + (int64_t)it.tile * chunks;
        }
        if (want < (by_tile ? tiles_before : items_before)) break;
    }
    __syncthreads();
    base = lds.base;
    return lds.item;
}

// ---- codes to 16-bit operands ------------------------------------------------------------------------------------
typedef f16 f16x2v __attribute__((ext_vector_type(2)));

// codes 2*PAIR and 2*PAIR + 1 of a dword as two bf16 or f16, both exact
template <int CODE, typename T, int PAIR> __device__ __forceinline__ unsigned widen2(unsigned x) {
    if constexpr (CODE == FLA_F8E4M3) {
        if constexpr (sizeof(T) == 2 && __is_same(T, bf16)) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, PAIR == 1));
        else return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, PAIR == 1));
    } else {
        const float a = (float)(signed char)(x >> (16 * PAIR)), b = (float)(signed char)(x >> (16 * PAIR + 8));
        if constexpr (__is_same(T, bf16)) return pack_bf16(a, b);
        else {
            const f32x2 v = {a, b};
            return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2v));
        }
    }
}

}  // namespace fla
