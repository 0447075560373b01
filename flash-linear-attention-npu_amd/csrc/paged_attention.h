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
    // Chunk length: long enough for about `few` items, or shorter where chunks of 16 units and about `target` items allow it;
    // at least min_units.  target 0: one chunk for each tile.
    int target, few, min_units;
    int tiles_each;                // tiles of a request without cu
    int items;                     // that the grid and the workspace have room for
    float scale2;                  // scale * log2(e)
    bool clear_tail;
};

struct Request {
    int first, rows, units;        // first query token, query rows (tokens * group), key units
    int len, new_tokens;           // cached tokens, query tokens from `first` on: also those behind the last row of q
};

__device__ __forceinline__ Request request_of(const AttnParams &p, int r) {
    Request q;
    int a = r, b = r + 1, all = r + 1;
    if (p.cu) {
        a = min(max(p.cu[r], 0), p.tokens);
        all = max(p.cu[r + 1], a);
        b = min(all, p.tokens);
    }
    q.first = a;
    // Row j of a request is token len - (query tokens) + j also where q ends inside the request: the rows that q lacks count.
    q.new_tokens = all - a;
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

// Inclusive prefix sum over the 64 lanes of a wave, as wave_inclusive_scan.
__device__ __forceinline__ int wave_scan(int v) {
#define FLA_DPP_IADD(ctrl, row_mask) v += __builtin_amdgcn_update_dpp(0, v, (ctrl), (row_mask), 0xf, true)
    FLA_DPP_IADD(0x111, 0xf);
    FLA_DPP_IADD(0x112, 0xf);
    FLA_DPP_IADD(0x114, 0xf);
    FLA_DPP_IADD(0x118, 0xf);
    FLA_DPP_IADD(0x142, 0xa);
    FLA_DPP_IADD(0x143, 0xc);
#undef FLA_DPP_IADD
    return v;
}

// The item with number `want`, or (by_tile) the first item of the tile with number `want` and, in base, its number.  Every
// wave finds it for itself, 64 requests at a time, with no LDS and no barrier: this stands before the first load of codes.
template <int ROWS> __device__ __forceinline__ Item find_item(const AttnParams &p, int want, bool by_tile, int &base) {
    Item it;
    it.chunk = 0;
    it.chunks = 1;
    it.units = INT32_MAX;
    if (p.target == 0 && p.cu == nullptr) {            // decode, one chunk for each request
        it.r = want / p.tiles_each;
        it.tile = want - it.r * p.tiles_each;
        it.found = it.r < p.n;
        base = want;
        return it;
    }
    const int lane = threadIdx.x & 63;
    int tiles0 = 0, units0 = 0;                         // of request `lane`
    if (lane < p.n) {
        const Request q = request_of(p, lane);
        tiles0 = (q.rows + ROWS - 1) / ROWS;
        units0 = q.units;
    }
    if (p.target) {
        int64_t work = (int64_t)tiles0 * units0;
        for (int r = lane + kWave; r < p.n; r += kWave) {
            const Request q = request_of(p, r);
            work += (int64_t)((q.rows + ROWS - 1) / ROWS) * q.units;
        }
        // sum over the lanes in two halves; one more than the quotient, so that rounding cannot make more items than the grid
        const int lo = __builtin_amdgcn_readlane(wave_scan((int)(work & 0xffff)), 63), hi = __builtin_amdgcn_readlane(wave_scan((int)(work >> 16)), 63);
        const float all = (float)hi * 65536.f + (float)lo;
        const int most = (int)fminf(all / (float)p.few, 1e9f) + 1, least = (int)fminf(all / (float)p.target, 1e9f) + 1;
        it.units = max(min(most, max(least, 16)), p.min_units);
    }
    int items_before = 0, tiles_before = 0;
    for (int r0 = 0; r0 < p.n; r0 += kWave) {
        int tiles = tiles0, units = units0;
        if (r0) {
            tiles = units = 0;
            if (r0 + lane < p.n) {
                const Request q = request_of(p, r0 + lane);
                tiles = (q.rows + ROWS - 1) / ROWS;
                units = q.units;
            }
        }
        const int chunks = units <= it.units ? 1 : (units + it.units - 1) / it.units, items = tiles * chunks;
        const int end_i = items_before + wave_scan(items), end_t = tiles_before + wave_scan(tiles);
        const uint64_t past = __ballot((by_tile ? end_t : end_i) > want);        // the sums ascend: its request is the first one past it
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            it.r = r0 + l;
            it.chunks = __builtin_amdgcn_readlane(chunks, l);
            const int first_i = __builtin_amdgcn_readlane(end_i - items, l), first_t = __builtin_amdgcn_readlane(end_t - tiles, l);
            if (by_tile) {
                it.tile = want - first_t;
            } else {
                it.tile = (want - first_i) / it.chunks;
                it.chunk = want - first_i - it.tile * it.chunks;
            }
            base = first_i + it.tile * it.chunks;
            it.found = it.tile >= 0 && it.tile < __builtin_amdgcn_readlane(tiles, l);   // false only where meaningless lengths overflowed the sums
            return it;
        }
        items_before = __builtin_amdgcn_readlane(end_i, 63);
        tiles_before = __builtin_amdgcn_readlane(end_t, 63);
    }
    it.found = false;
    return it;
}

// ---- codes to 16-bit operands ------------------------------------------------------------------------------------
typedef f16 f16x2v __attribute__((ext_vector_type(2)));
constexpr float kNegInf = -__builtin_inff();

// codes 2*PAIR and 2*PAIR + 1 of a dword as two bf16 or f16, both exact
template <int CODE, typename T, int PAIR> __device__ __forceinline__ unsigned widen2(unsigned x) {
    if constexpr (CODE == FLA_F8E4M3) {
        if constexpr (__is_same(T, bf16)) return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.f, PAIR == 1));
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
template <int CODE> __device__ __forceinline__ bool has_nan4(unsigned x) {   // e4m3 NaN: 0x7f or 0xff in a byte
    return CODE == FLA_F8E4M3 && ((((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0);
}

// ---- one wave's walk over the keys ------------------------------------------------------------------------------
// Where the 32 tokens of a step lie.  WIDE: pages hold at least 32 tokens, so a step has one page and everything about it
// is uniform; else a lane knows the page of its eight tokens t0 + 8 g .. + 7.
template <bool WIDE> struct Place {
    int page;        // in the pool, whether held or not
    bool held;       // false: nothing to see
};

// The table's entries for the next 64 (32 where a step has two pages) steps, one in each lane: a step reads its own with
// no memory access, which would wait for every load issued before it.
template <bool WIDE> struct PageWindow {
    int entries;
    __device__ __forceinline__ void fill(const AttnParams &p, const int32_t *row, int t0, int stride) {
        const int lane = threadIdx.x & 63;
        const int64_t tok = WIDE ? (int64_t)t0 + (int64_t)lane * stride : (int64_t)t0 + (int64_t)(lane >> 1) * stride + 16 * (lane & 1);
        const int64_t at = tok >> p.shift;
        entries = at < p.width ? row[at] : -1;
    }
    __device__ __forceinline__ Place<WIDE> get(const AttnParams &p, const int32_t *row, int t0, int stride, int step, int most) {
        if (__builtin_expect(step && (step & (WIDE ? 63 : 31)) == 0, 0)) {
            fill(p, row, t0, stride);
            asm volatile("" : "+v"(entries));      // waited for here: behind the branch every step would wait for all its loads
        }
        const int k = step & (WIDE ? 63 : 31);
        int page;
        if (WIDE) page = __builtin_amdgcn_readlane(entries, k);
        else {                            // a page behind the last token may be anything
            const int a = __builtin_amdgcn_readlane(entries, 2 * k), b = __builtin_amdgcn_readlane(entries, 2 * k + 1);
            page = !(threadIdx.x & 32) ? a : t0 + 16 < most ? b : -1;
        }
        Place<WIDE> pl;
        pl.held = (uint32_t)page < p.pool;
        pl.page = pl.held ? page : 0;
        return pl;
    }
};

// lane offsets inside a page that hold for the whole walk (WIDE), in bytes
struct LaneOffsets {
    unsigned k, v;
};

// How a walk loads codes: kAhead (decode, memory far away): the next step's keys as soon as this step's are consumed, its
// values likewise; kAheadOnce: the same past the caches, for codes that nobody reads again.  kLate (prefill, keys in L2):
// values ahead of the first product and keys ahead of the second, which leaves 32 registers more.
enum Loads { kLate, kAhead, kAheadOnce };

template <Loads L, typename V> __device__ __forceinline__ V load_codes(const uint8_t *p) {
    if constexpr (L == kAheadOnce) return __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
    else return *reinterpret_cast<const V *>(p);
}

template <int D, bool WIDE, Loads L> struct KeyCodes {
    u32x4 c[2][D / 64];
    float scale;
    __device__ __forceinline__ void load(const AttnParams &p, int head, int t0, const Place<WIDE> &pl, const LaneOffsets &off) {
        const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15, in_page = (1 << p.shift) - 1;
        scale = p.ks[(int64_t)pl.page * p.ks_p + head * p.ks_h];
        const uint8_t *at;
        if (WIDE) {
            at = p.kc + (int64_t)pl.page * p.kc_p + (int64_t)head * p.kc_h + (int64_t)(t0 & in_page) * p.kc_t;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int h = 0; h < D / 64; ++h) c[t][h] = load_codes<L, u32x4>(at + (int64_t)(4 * t) * p.kc_t + 64 * h + off.k);
        } else {
            // the rows of this lane are those of lane group i / 4, whose page sits in lane 16 (i / 4)
            const int kg = i >> 2, page = __shfl(pl.page, kg * 16, kWave);
            at = p.kc + (int64_t)page * p.kc_p + (int64_t)head * p.kc_h + (int64_t)(((t0 + 8 * kg) & in_page) + (i & 3)) * p.kc_t + g * 16;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int h = 0; h < D / 64; ++h) c[t][h] = load_codes<L, u32x4>(at + 4 * t * p.kc_t + 64 * h);
        }
    }
};

template <int D, bool WIDE, Loads L> struct ValueCodes {
    static constexpr bool kRaw = L == kLate || D == 64;
    unsigned c[8][D / 64];
    float scale;           // kRaw: of page 0 where nothing is held
    __device__ __forceinline__ void load(const AttnParams &p, int head, int t0, const Place<WIDE> &pl, const LaneOffsets &off) {
        typedef unsigned VV __attribute__((ext_vector_type(D / 64)));
        const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15, in_page = (1 << p.shift) - 1;
        // The use of the scale here makes the loads below wait for those before them.  That holds a prefill up (2 x 4096: 760 us
        // with it, 745 us without; D = 256 1958 and 1800) and decode with D = 64, but larger heads decode faster with it (48
        // requests of 1 to 7 rows, D = 128: 47.5 and 51 us; 256 of 2500 tokens 155 and 159 us).
        const float s = p.vs[(int64_t)pl.page * p.vs_p + head * p.vs_h];
        scale = kRaw || pl.held ? s : 0.f;
        const uint8_t *at = p.vc + (int64_t)pl.page * p.vc_p + (int64_t)head * p.vc_h;
        if (WIDE) at += (int64_t)(t0 & in_page) * p.vc_t;
        else at += (int64_t)((t0 + 8 * g) & in_page) * p.vc_t + i * (D / 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint8_t *from = WIDE ? at + (int64_t)e * p.vc_t + off.v : at + e * p.vc_t;
            if constexpr (D == 64) c[e][0] = load_codes<L, unsigned>(from);
            else {
                const VV x = load_codes<L, VV>(from);
#pragma unroll
                for (int w = 0; w < D / 64; ++w) c[e][w] = x[w];
            }
        }
    }
};

// The power of two that the v scales of a request and head are measured in: that of its first page, if it has one.
__device__ __forceinline__ float scale_unit(const AttnParams &p, const int32_t *table_row, int head) {
    const int page = p.width ? table_row[0] : -1;
    const float s = (uint32_t)page < p.pool ? fabsf(p.vs[(int64_t)page * p.vs_p + head * p.vs_h]) : 0.f;
    if (!(s > 0.f && s < INFINITY)) return 0x1p-40f;
    return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, fminf(fmaxf(s, 0x1p-60f), 0x1p60f)) & 0x7f800000u);
}

// Natural logarithm of 2^m l.  The exponent of l joins m first: beside pages with a scale of 0 both are far from 0 (m counts their
// value scale as 2^-60 u, l takes it out again), and a logarithm of l rounded there would cost what their sum keeps.
__device__ __forceinline__ float log_sum(float m, float l) {
    return ((m + (float)__builtin_amdgcn_frexp_expf(l)) + log2f(__builtin_amdgcn_frexp_mantf(l))) * (1.f / kLog2e);
}

// One wave: 16 NC query rows against the tokens it is led over, 32 at a time.
//   S^T = K Q^T: tokens are the rows of the accumulators, query rows their columns; O^T += V^T P^T with P^T straight from
//   the accumulator layout.
//  - K: lane 16 g + i holds row i of a 16-token tile; it loads 16 bytes at 64 h + 16 g of its row, so a load touches whole
//    64-byte pieces.  The contraction index is permuted by that; q is loaded with the same permutation.
//  - rows are given to tokens so that the accumulators of lane group g are tokens 8 g .. 8 g + 7 of the step: the
//    contraction order of O^T.  V: lane 16 g + i loads D/16 neighbouring channels of those eight tokens, and a byte
//    transpose inside the lane gives the operands of D/16 tiles whose row i is channel D/16 i + j of tile j.
//  - scales of pages multiply S after the product (exact codes enter the matrix unit).  The v scale enters the weight of a
//    token as an addend of its exponent, w = 2^(s + log2(vs / u) - m), which costs nothing for each element; m is 10 below the
//    largest s + log2(vs / u), so weights are measured against the largest contribution, whatever the scales of other
//    pages are.  The sum of the softmax is that of w u / vs.  u, the scale of the request's first page as a power of two,
//    only keeps these numbers inside fp32.  A scale below 2^-60 u (0 above all) counts as 2^-60 u in the exponent and
//    multiplies the weight by the rest; of a negative one the magnitude is in the exponent.
//    (Where nearly all weight lies on such pages, the others' share is off by at most 2^-95 u of a code for each token.)
//  - weights are rounded to fp16 with 11 bits: a bf16 weight would add an error as large as the rounding of the result.  (bf16
//    results are as far from exact as with fp32 weights, 1.7e-3; fp16 ones 2.6e-4 where their own rounding leaves 2.1e-4.)  The
//    largest contribution stands at 2^10 or more, near the top of fp16, because the sum of the softmax counts light weights in
//    full: they keep 11 bits down to 2^-24 of the largest contribution and are off by at most 2^-35 of it below that, which
//    shows only where a heavy token has values of (nearly) 0.
//  - the maximum moves only when the eight weights of a lane sum to more than fp16 holds, which the sum that is needed anyway
//    tells, so most steps take no maximum, exchange nothing between lanes and rescale nothing.  (Prefill of 2 x 4096 tokens: 788
//    us with the largest contribution at 2^0 and sums to 2^11, 792 at 2^8 and 2^15, 804 at 2^10 and 2^15, 793 so.)
// Sums and statistics are fp32.
template <int CODE, int D, int NC, bool WIDE, Loads L> struct Walk {
    typedef elemx8 T8;
    static constexpr float kMost = 65504.f, kTop = 10.f;   // what sums may grow to, log2 of the weight of the largest contribution
    f32x4 o[NC][D / 16];   // o[c][j][e] of lane (g, i): channel D/16 (4 g + e) + j of query row 16 c + i, in units of u 2^m
    float m[NC], l[NC];    // the largest s + log2(vs / u) less kTop when it last moved (the same in all lanes of a column), this lane's share of the sum
    float unit, log_unit;  // u, log2 u
    unsigned seen;         // bit c: the column has seen a token
    bool fresh;
    static constexpr bool kQueriesInLds = NC > 1;
    u32x4 q[kQueriesInLds ? 1 : NC][D / 32];
    u32x4 *lds_q;          // [NC][D / 32][64]: every lane's own pieces; all waves of a workgroup hold the same rows
    int limit[NC];         // tokens that the column sees
    int least, most;       // the smallest and largest limit of the wave's real columns

    __device__ __forceinline__ void start(const AttnParams &p, const Request &rq, const int32_t *table_row, int head, int first_row, u32x4 *room) {
        lds_q = room;
        const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
        const int cap = (int)min((int64_t)rq.len, (int64_t)p.width << p.shift);
        least = INT32_MAX;
        most = 0;
        unit = scale_unit(p, table_row, head);
        log_unit = __builtin_amdgcn_logf(unit);
        seen = 0;
        fresh = true;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int row = first_row + 16 * c + i, tok = row / p.group, h = head * p.group + row - tok * p.group;
            const bool real = row < rq.rows;
            limit[c] = real ? min(max(rq.len - rq.new_tokens + tok + 1, 0), cap) : 0;
            const elem *src = static_cast<const elem *>(p.q) + (int64_t)(rq.first + (real ? tok : 0)) * p.q_t + (int64_t)(real ? h : 0) * p.q_h;
#pragma unroll
            for (int s = 0; s < D / 32; ++s) {
                const u32x4 x = *reinterpret_cast<const u32x4 *>(src + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
                const u32x4 y = real ? x : u32x4{0u, 0u, 0u, 0u};
                if (kQueriesInLds) lds_q[(c * (D / 32) + s) * 64 + lane] = y;
                else q[c][s] = y;
            }
            int lo = real ? limit[c] : INT32_MAX, hi = limit[c];
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) {
                lo = min(lo, __shfl_xor(lo, d, kWave));
                hi = max(hi, __shfl_xor(hi, d, kWave));
            }
            least = min(least, lo);
            most = max(most, hi);
            m[c] = l[c] = 0.f;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) o[c][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        least = __builtin_amdgcn_readfirstlane(least);
        most = __builtin_amdgcn_readfirstlane(most);
    }

    // tokens t0, t0 + stride, ... (32 each) below end <= most; pages: filled for t0 (before start, which waits for lengths)
    __device__ __forceinline__ void run(const AttnParams &p, const int32_t *row, PageWindow<WIDE> &pages, int head, int t0, int stride, int end) {
        if (t0 >= end) return;
        const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
        LaneOffsets off;
        off.k = (unsigned)(8 * (i >> 2) + (i & 3)) * (unsigned)p.kc_t + 16 * g;
        off.v = (unsigned)(8 * g) * (unsigned)p.vc_t + i * (D / 16);
        if constexpr (L != kLate) {
            KeyCodes<D, WIDE, L> k;
            ValueCodes<D, WIDE, L> v;
            Place<WIDE> at = pages.get(p, row, t0, stride, 0, most);
            k.load(p, head, t0, at, off);
            v.load(p, head, t0, at, off);
            for (int step = 1;; ++step) {
                const int t1 = t0 + stride;
                const bool go = t1 < end;
                f32x4 s[NC][2];
                scores(k, s);
                const float f = k.scale * p.scale2;
                // D = 64: not behind a branch, or the values of this step would wait for these loads too; after the last step all
                // lanes load one piece seen already (48 requests of 1 to 7 rows 31.0 us behind a branch, 29.6 us so; one row each
                // 25.2 and 23.6).  For larger heads the last loads cost more than the wait (48 requests of 1 to 7 rows, D = 128:
                // 47.4 and 49.6 us; 256 of 2500 tokens 154 and 157 us).
                Place<WIDE> next = at;
                if (D == 64 || go) {
                    const Place<WIDE> behind = pages.get(p, row, t1, stride, step, most);
                    if (go) next = behind;
                    k.load(p, head, go ? t1 : t0, next, {go ? off.k : 0u, off.v});
                }
                f16x8 w[NC];
                weigh(s, f, v, at.held, t0, w);
                accumulate(v, w);
                if (!go) break;
                v.load(p, head, t1, next, off);
                at = next;
                t0 = t1;
            }
        } else {
            KeyCodes<D, WIDE, L> k;
            ValueCodes<D, WIDE, L> v;
            Place<WIDE> at = pages.get(p, row, t0, stride, 0, most);
            k.load(p, head, t0, at, off);
            // Steps that every column sees whole, and that move no maximum, have a loop of their own: with the code for the
            // others in it, the compiler keeps the accumulators in memory for part of it.  The products go before the other
            // wave's vector instructions (s_setprio): the matrix unit is asked first while there is something for it, and the
            // two waves of a SIMD fall out of step (prefill of 2 x 4096 tokens, 32 heads on 8: D = 128 849 us without, 770 us with
            // it, int8 970 and 870; D = 64 571 and 533; D = 256 1815 and 1793).
            for (int step = 1; t0 < end;) {
                while (t0 < end && t0 + 32 <= least && !fresh) {
                    v.load(p, head, t0, at, off);
                    f32x4 s[NC][2];
                    __builtin_amdgcn_s_setprio(1);
                    scores(k, s);
                    __builtin_amdgcn_s_setprio(0);
                    const float f = k.scale * p.scale2, floor = unit * 0x1p-60f;
                    const float add = __builtin_amdgcn_logf(v.scale) - log_unit, back = unit * __builtin_amdgcn_rcpf(v.scale);
                    f16x8 w[NC];
                    float sum[NC], top = 0.f;
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        w[c] = exponentials(s[c], f, add - m[c], sum[c]);
                        top = fmaxf(top, sum[c]);
                    }
                    if (__builtin_expect(__any(top > kMost || !at.held || !(v.scale >= floor)), 0)) break;
#pragma unroll
                    for (int c = 0; c < NC; ++c) l[c] = fmaf(sum[c], back, l[c]);
                    advance(p, row, pages, head, t0, stride, end, step, at, k, off);
                    __builtin_amdgcn_s_setprio(1);
                    accumulate(v, w);
                    __builtin_amdgcn_s_setprio(0);
                }
                if (t0 >= end) break;
                v.load(p, head, t0, at, off);
                f32x4 s[NC][2];
                scores(k, s);
                f16x8 w[NC];
                fresh = true;                  // every maximum settles
                weigh(s, k.scale * p.scale2, v, at.held, t0, w);
                advance(p, row, pages, head, t0, stride, end, step, at, k, off);
                accumulate(v, w);
            }
        }
    }

    // to the next step, whose keys are loaded if there is one
    __device__ __forceinline__ void advance(const AttnParams &p, const int32_t *row, PageWindow<WIDE> &pages, int head, int &t0, int stride, int end,
                                            int &step, Place<WIDE> &at, KeyCodes<D, WIDE, L> &k, const LaneOffsets &off) {
        t0 += stride;
        if (t0 < end) {
            at = pages.get(p, row, t0, stride, step, most);
            k.load(p, head, t0, at, off);
        }
        ++step;
    }

    __device__ __forceinline__ void scores(const KeyCodes<D, WIDE, L> &k, f32x4 (&s)[NC][2]) {
#pragma unroll
        for (int c = 0; c < NC; ++c) s[c][0] = s[c][1] = f32x4{0.f, 0.f, 0.f, 0.f};
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));        // the reads below stay in the loop: hoisted, the queries would take registers again
        u32x4 b[2][NC];                                  // the next queries are read while these are used
#pragma unroll
        for (int c = 0; c < NC; ++c) b[0][c] = kQueriesInLds ? lds_q[c * (D / 32) * 64 + lane] : q[kQueriesInLds ? 0 : c][0];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            if (i + 1 < D / 32) {
#pragma unroll
                for (int c = 0; c < NC; ++c) b[(i + 1) & 1][c] = kQueriesInLds ? lds_q[(c * (D / 32) + i + 1) * 64 + lane] : q[kQueriesInLds ? 0 : c][i + 1];
            }
            if (kQueriesInLds) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const u32x4 a = {widen2<CODE, elem, 0>(k.c[t][i >> 1][2 * (i & 1)]), widen2<CODE, elem, 1>(k.c[t][i >> 1][2 * (i & 1)]),
                                 widen2<CODE, elem, 0>(k.c[t][i >> 1][2 * (i & 1) + 1]), widen2<CODE, elem, 1>(k.c[t][i >> 1][2 * (i & 1) + 1])};
#pragma unroll
                for (int c = 0; c < NC; ++c) s[c][t] = mfma16x32(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, b[i & 1][c]), s[c][t]);
            }
        }
    }

    // Moves the maximum of a column to its largest s + log2(vs / u) so far, less kTop; `by`: what its sum and accumulators are to be
    // multiplied by.  A column that has seen nothing keeps a maximum of 0 (its scores are -inf, its weights 0).
    __device__ __forceinline__ void settle(const f32x4 (&s)[2], float f, float add, int c, float &by) {
        float best = kNegInf;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) best = fmaxf(best, s[t][e] * f);
        best += add;
        best = fmaxf(best, __shfl_xor(best, 16, kWave));
        best = fmaxf(best, __shfl_xor(best, 32, kWave)) - kTop;
        const bool any = best > kNegInf, first = !(seen & (1u << c));
        const float top = !any ? m[c] : first ? best : fmaxf(best, m[c]);
        by = first ? 1.f : by * __builtin_amdgcn_exp2f(m[c] - top);                     // first: sum and accumulators are 0
        m[c] = top;
        seen |= any ? 1u << c : 0u;
    }

    // Eight weights of a column in the operand's order and their sum (before `ratio`).
    __device__ __forceinline__ f16x8 exponentials(const f32x4 (&s)[2], float f, float bias, float &sum, float ratio = 1.f) {
        u32x4 packed;
        f32x2 part[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const f32x2 x = {__builtin_amdgcn_exp2f(fmaf(s[t][e], f, bias)), __builtin_amdgcn_exp2f(fmaf(s[t][e + 1], f, bias))};
                part[2 * t + e / 2] = x;
                packed[2 * t + e / 2] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{x[0] * ratio, x[1] * ratio}, f16x2v));
            }
        sum = ((part[0][0] + part[0][1]) + (part[1][0] + part[1][1])) + ((part[2][0] + part[2][1]) + (part[3][0] + part[3][1]));
        return __builtin_bit_cast(f16x8, packed);
    }

    __device__ __forceinline__ void weigh(f32x4 (&s)[NC][2], float f, ValueCodes<D, WIDE, L> &v, bool held, int t0, f16x8 (&w)[NC]) {
        const int tok = t0 + 8 * (int)((threadIdx.x & 63) >> 4);
        const bool masked = t0 + 32 > least || __any(!held);      // some column does not see all of the step
        bool nan = false;
        if (__builtin_expect(masked, 0)) {
            bool mine = false;
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int x = 0; x < D / 64; ++x) {
                    // tokens that no column sees must not enter the second product: 0 times a NaN is a NaN
                    v.c[e][x] = tok + e < most && held ? v.c[e][x] : 0u;
                    mine = mine || has_nan4<CODE>(v.c[e][x]);
                }
            nan = __any(mine);
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[c][t][e] = tok + 4 * t + e < limit[c] && held ? s[c][t][e] * f : kNegInf;
            f = 1.f;
        }
        float by[NC];                      // what sums and accumulators are multiplied by
#pragma unroll
        for (int c = 0; c < NC; ++c) by[c] = 1.f;
        const float floor = unit * 0x1p-60f, page_scale = !ValueCodes<D, WIDE, L>::kRaw || held ? v.scale : 0.f, scale = fmaxf(fabsf(page_scale), floor), add = __builtin_amdgcn_logf(scale) - log_unit, back = unit * __builtin_amdgcn_rcpf(scale);
        const bool tiny = __any(!(page_scale >= floor)), early = masked || fresh;
        bool moved = early;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float sum;
            if (__builtin_expect(early, 0)) settle(s[c], f, add, c, by[c]);
            w[c] = exponentials(s[c], f, add - m[c], sum);
            if (__builtin_expect(__any(sum > kMost), 0)) {
                settle(s[c], f, add, c, by[c]);
                moved = true;
                w[c] = exponentials(s[c], f, add - m[c], sum);
            }
            if (__builtin_expect(tiny, 0)) w[c] = exponentials(s[c], f, add - m[c], sum, page_scale >= floor ? 1.f : page_scale / scale);
            l[c] = fmaf(sum, back, l[c] * by[c]);
        }
        if (__builtin_expect(fresh, 0)) {
            bool none = false;
#pragma unroll
            for (int c = 0; c < NC; ++c) none = none || (limit[c] > 0 && !(seen & (1u << c)));
            fresh = __any(none);
        }
        if (__builtin_expect(moved, 0)) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < D / 16; ++j) o[c][j] *= by[c];
        }
        if (__builtin_expect(nan, 0)) spread_nan(v, tok, held);
    }

    // A NaN in a token that some columns see and others do not: put into the columns that see it, taken out of the codes.
    __device__ __forceinline__ void spread_nan(ValueCodes<D, WIDE, L> &v, int tok, bool held) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            u32x4 sees = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (tok + e < limit[c] && held) sees[e >> 1] |= (e & 1) ? 0x3c000000u : 0x00003c00u;
#pragma unroll
            for (int x = 0; x < D / 64; ++x)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u32x4 bad = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (((v.c[e][x] >> (8 * j)) & 0x7fu) == 0x7fu) bad[e >> 1] |= (e & 1) ? 0x3c000000u : 0x00003c00u;
                    const f32x4 hit = mfma16x32(__builtin_bit_cast(f16x8, bad), __builtin_bit_cast(f16x8, sees), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (hit[e] > 0.f) o[c][4 * x + j][e] = __builtin_nanf("");
                    __builtin_amdgcn_sched_barrier(0);                 // one at a time: this path must not cost registers
                }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int x = 0; x < D / 64; ++x) {
                unsigned is = (v.c[e][x] & 0x7f7f7f7fu) + 0x01010101u;   // 0x80 in the bytes that hold a NaN
                is &= 0x80808080u;
                v.c[e][x] &= ~((is << 1) - (is >> 7));
            }
    }

    __device__ __forceinline__ void accumulate(const ValueCodes<D, WIDE, L> &v, const f16x8 (&w)[NC]) {   // O^T += V^T P^T
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
            unsigned pair[4][2];                      // bytes of two tokens side by side, channel by channel
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pair[e][0] = __builtin_amdgcn_perm(v.c[2 * e + 1][x], v.c[2 * e][x], 0x05010400u);
                pair[e][1] = __builtin_amdgcn_perm(v.c[2 * e + 1][x], v.c[2 * e][x], 0x07030602u);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                u32x4 a;
#pragma unroll
                for (int e = 0; e < 4; ++e) a[e] = (j & 1) ? widen2<CODE, f16, 1>(pair[e][j >> 1]) : widen2<CODE, f16, 0>(pair[e][j >> 1]);
#pragma unroll
                for (int c = 0; c < NC; ++c) o[c][4 * x + j] = mfma16x32(__builtin_bit_cast(f16x8, a), w[c], o[c][4 * x + j]);
            }
        }
    }

    // the sum over all lanes of each column; after the walk
    __device__ __forceinline__ void finish() {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            l[c] += __shfl_xor(l[c], 16, kWave);
            l[c] += __shfl_xor(l[c], 32, kWave);
            if (l[c] == 0.f) m[c] = kNegInf;
        }
    }

    // accumulators (joined with other waves', maximum mm, sum ll) to the result or the workspace
    __device__ __forceinline__ void store(const AttnParams &p, const Request &rq, const Item &it, int64_t item, int head, int rows_per_tile,
                                          int first_in_tile, const float (&mm)[NC], const float (&ll)[NC]) {
        const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int in_tile = first_in_tile + 16 * c + i, row = it.tile * rows_per_tile + in_tile;
            if (row >= rq.rows) continue;
            if (it.chunks == 1) {
                const int tok = row / p.group, h = head * p.group + row - tok * p.group;
                const float by = ll[c] > 0.f || ll[c] != ll[c] ? unit / ll[c] : 0.f;
                elem *dst = static_cast<elem *>(p.out) + (int64_t)(rq.first + tok) * p.o_t + (int64_t)h * p.o_h;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (D == 64) {
                        elemx4 y;
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = (elem)(o[c][j][e] * by);
                        *reinterpret_cast<elemx4 *>(dst + 4 * (4 * g + e)) = y;
                    } else {
#pragma unroll
                        for (int x = 0; x < D / 128; ++x) {
                            T8 y;
#pragma unroll
                            for (int j = 0; j < 8; ++j) y[j] = (elem)(o[c][8 * x + j][e] * by);
                            *reinterpret_cast<T8 *>(dst + D / 16 * (4 * g + e) + 8 * x) = y;
                        }
                    }
                }
                if (p.lse && g == 0) p.lse[(int64_t)(rq.first + tok) * p.lse_t + (int64_t)h * p.lse_h] = log_sum(mm[c], ll[c]);
            } else {
                const int64_t slot = (item * p.heads + head) * rows_per_tile + in_tile;
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int j = 0; j < D / 16; j += 4)
                        *reinterpret_cast<f32x4 *>(p.part_o + slot * D + D / 16 * (4 * g + e) + j) = f32x4{o[c][j][e], o[c][j + 1][e], o[c][j + 2][e], o[c][j + 3][e]};
                if (g == 0) {
                    p.part_ml[slot * 2] = mm[c];
                    p.part_ml[slot * 2 + 1] = ll[c];
                }
            }
        }
    }
};

// Rows behind the last request (and before the first, should cu not begin at 0): 0, lse -inf.  Workgroup `part` of `parts`
// takes every parts-th row.
template <int THREADS> __device__ __forceinline__ void clear_tail(const AttnParams &p, int head, int D, int part, int parts) {
    const int64_t first = min(max(p.cu[0], 0), p.tokens), last = min(max(p.cu[p.n], (int)first), p.tokens);
    for (int64_t row = part; row < first + p.tokens - last; row += parts) {
        const int64_t t = row < first ? row : row - first + last;
        for (int x = threadIdx.x; x < p.group * D; x += THREADS) {
            const int h = head * p.group + x / D, d = x % D;
            static_cast<elem *>(p.out)[t * p.o_t + h * p.o_h + d] = (elem)0.f;
            if (p.lse && d == 0) p.lse[t * p.lse_t + h * p.lse_h] = kNegInf;
        }
    }
}

struct AttnLaunch {
    int nc, dim, code, waves, longest_rows;
    int64_t tiles, items;      // bounds
    uint64_t o_bytes, bytes;
};

// The kernels are built once for each query type (the bf16 and the f16 object of their sources).
int launch_paged_decode(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream);
int launch_paged_decode_f16(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream);
int launch_paged_prefill(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream);
int launch_paged_prefill_f16(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream);
int launch_paged_join(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream);
int launch_paged_join_f16(const AttnParams &p, const AttnLaunch &plan, hipStream_t stream);
#ifdef FLA_ELEM_F16
#define FLA_PAGED(name) name##_f16
#else
#define FLA_PAGED(name) name
#endif

}  // namespace fla
