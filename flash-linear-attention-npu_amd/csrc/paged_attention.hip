// paged_kv_attention: softmax attention of a few query rows over a paged cache held in 8 bits (decode, checking of
// speculated tokens), the join of split key axes, and the entry point.
//   s_t = scale * ks_page (q . k8_t),  o = sum_t e^{s_t - m} vs_page v8_t / sum_t e^{s_t - m}
// Bound by HBM: each code is read once, and a wave needs about 220 vector instructions for the 8 KB of a 32-token step.
//
// Every wave of a workgroup walks 32-token steps of its chunk with no LDS and no barrier: S^T = K Q^T (tokens are the rows
// of the accumulator, query rows its columns), running maximum and sum per column, O^T += V^T P^T with P^T straight from
// the accumulator layout.
//  - K: lane 16g + i holds row i; it loads 16 bytes at 64 h + 16 g of its row, so a load touches whole 64-byte pieces.
//    The contraction index is permuted by that; q is loaded with the same permutation.
//  - rows are given to tokens so that the accumulators of lane group g are tokens 8g .. 8g+7 of the step: the contraction
//    order of O^T.  V: lane 16g + i loads D/16 neighbouring channels of those eight tokens, and a byte transpose within
//    the lane gives the operands of D/16 tiles whose row i is channel D/16 * i + j of tile j.
//  - scales of pages multiply S after the product (exact codes enter the matrix unit) and P: the weight of a token is
//    p * vs / R with R the largest v scale so far (the accumulators are kept in units of R), rounded to fp16 with 11 bits:
//    a bf16 weight would add an error as large as the rounding of the result.
//  - the maximum moves only when a score passes it by 2^8 (weights then stay below 2^8, far inside fp16), so most steps
//    need no exchange between lanes and no rescaling.
// The next step's codes are loaded while this one is computed.  Sums and statistics are fp32.
#include "paged_attention.h"

namespace fla {


namespace {

constexpr float kMoveMax = 8.f;
constexpr float kNegInf = -__builtin_inff();

template <int CODE> __device__ __forceinline__ bool has_nan4(unsigned x) {
    // e4m3 NaN: 0x7f or 0xff in a byte
    const unsigned y = x & 0x7f7f7f7fu;
    return CODE == FLA_F8E4M3 && (((y + 0x01010101u) & 0x80808080u) != 0);
}

template <int D> struct KvStep {
    u32x4 k[2][D / 64];
    unsigned v[8][D / 64];
    float ks, vs;
    bool held;       // the page is in the pool and holds tokens that some column sees
};

// page of this lane's eight tokens t0 + 8 g .. + 7 (all in one page); -1 outside the table or the pool
__device__ __forceinline__ int lane_page(const AttnParams &p, const int32_t *row, int t0) {
    const int64_t at = (int64_t)(t0 + 8 * (int)((threadIdx.x & 63) >> 4)) >> p.shift;
    return at < p.width ? row[at] : -1;
}

template <int D> __device__ __forceinline__ void load_step(const AttnParams &p, int head, int t0, int page, int most, KvStep<D> &st) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    st.held = (uint32_t)page < p.pool && t0 + 8 * g < most;   // a page behind the last token may be anything
    const int64_t pg = st.held ? page : 0;
    st.ks = p.ks[pg * p.ks_p + head * p.ks_h];
    st.vs = st.held ? p.vs[pg * p.vs_p + head * p.vs_h] : 0.f;
    const int in_page = (1 << p.shift) - 1, base = (t0 + 8 * g) & in_page;
    const uint8_t *v = p.vc + pg * p.vc_p + head * p.vc_h + base * p.vc_t + i * (D / 16);
    // K rows of this lane are those of lane group i / 4, whose page sits in lane 16 (i / 4)
    const int kg = i >> 2;
    const int kp = __shfl(st.held ? page : 0, kg * 16, kWave);
    const int kbase = (t0 + 8 * kg) & in_page;
    const uint8_t *k = p.kc + (int64_t)kp * p.kc_p + head * p.kc_h + (kbase + (i & 3)) * p.kc_t + g * 16;
#pragma unroll
    for (int h = 0; h < D / 64; ++h) {
        st.k[0][h] = *reinterpret_cast<const u32x4 *>(k + 64 * h);
        st.k[1][h] = *reinterpret_cast<const u32x4 *>(k + 4 * p.kc_t + 64 * h);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        typedef unsigned VV __attribute__((ext_vector_type(D / 64)));
        if constexpr (D == 64) st.v[e][0] = *reinterpret_cast<const unsigned *>(v + e * p.vc_t);
        else {
            const VV x = *reinterpret_cast<const VV *>(v + e * p.vc_t);
#pragma unroll
            for (int w = 0; w < D / 64; ++w) st.v[e][w] = x[w];
        }
    }
}

// state of a wave: column i = lane % 16 of tile c is query row 16 c + i
template <int D, int NC> struct Softmax {
    f32x4 o[NC][D / 16];   // o[c][j][e] of lane (g, i): channel D/16 (4 g + e) + j of column i, in units of r
    float m[NC], l[NC];    // maximum (the same in all lanes of a column), this lane's share of the sum
    float r;
};

template <typename T, int CODE, int D, int NC>
__device__ __forceinline__ void attend_step(const AttnParams &p, KvStep<D> &st, const u32x4 (&q)[NC][D / 32], const int (&limit)[NC],
                                            int least, int most, int t0, Softmax<D, NC> &sm) {
    const int g = (threadIdx.x & 63) >> 4, tok = t0 + 8 * g;
    typedef typename Vec8<T>::type T8;
    f32x4 s[NC][2];
#pragma unroll
    for (int c = 0; c < NC; ++c) s[c][0] = s[c][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int h = 0; h < D / 64; ++h)
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const u32x4 a = {widen2<CODE, T, 0>(st.k[t][h][2 * half]), widen2<CODE, T, 1>(st.k[t][h][2 * half]),
                                 widen2<CODE, T, 0>(st.k[t][h][2 * half + 1]), widen2<CODE, T, 1>(st.k[t][h][2 * half + 1])};
#pragma unroll
                for (int c = 0; c < NC; ++c)
                    s[c][t] = mfma16x32(__builtin_bit_cast(T8, a), __builtin_bit_cast(T8, q[c][2 * h + half]), s[c][t]);
            }
    const float f = st.ks * p.scale2;
    const bool masked = t0 + 32 > least || __any(!st.held);   // some column does not see all of the step
    if (masked) {
        // tokens that no column sees must not enter the second product: 0 times a NaN is a NaN
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int w = 0; w < D / 64; ++w) st.v[e][w] = tok + e < most && st.held ? st.v[e][w] : 0u;
    }
    // scores in units of log2
    bool move = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        float best = kNegInf;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = s[c][t][e] * f;
                if (masked && !(tok + 4 * t + e < limit[c] && st.held)) x = kNegInf;
                s[c][t][e] = x;
                best = fmaxf(best, x);
            }
        move = move || best > sm.m[c] + kMoveMax;
    }
    if (__any(move)) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            float best = sm.m[c];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) best = fmaxf(best, s[c][t][e]);
            best = fmaxf(best, __shfl_xor(best, 16, kWave));
            best = fmaxf(best, __shfl_xor(best, 32, kWave));
            const float by = best == kNegInf ? 1.f : exp2f(sm.m[c] - best);   // m = -inf before the first token: 0
            sm.m[c] = best;
            sm.l[c] *= by;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) sm.o[c][j] *= by;
        }
    }
    if (__any(st.vs > sm.r)) {
        float r = fmaxf(sm.r, st.vs);
        r = fmaxf(r, __shfl_xor(r, 16, kWave));
        r = fmaxf(r, __shfl_xor(r, 32, kWave));
        const float by = sm.r / r;
        sm.r = r;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int j = 0; j < D / 16; ++j) sm.o[c][j] *= by;
    }
    const float ratio = sm.r > 0.f ? st.vs / sm.r : 0.f;
    f16x8 w[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        u32x4 packed;
        const float m = sm.m[c] == kNegInf ? 0.f : sm.m[c];   // nothing seen yet: every weight is exp2(-inf) = 0
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float a = __builtin_amdgcn_exp2f(s[c][t][e] - m), b = __builtin_amdgcn_exp2f(s[c][t][e + 1] - m);
                sm.l[c] += a + b;
                const f32x2 v = {a * ratio, b * ratio};
                packed[2 * t + e / 2] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2v));
            }
        w[c] = __builtin_bit_cast(f16x8, packed);
    }
    bool slow = false;
    if (CODE == FLA_F8E4M3 && masked && t0 < most) {
        // a NaN in a token that some columns see and others do not: taken out of the product and put into the columns
        // that see it
        bool mine = false;
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int x = 0; x < D / 64; ++x) mine = mine || has_nan4<CODE>(st.v[e][x]);
        slow = __any(mine);
    }
    // operands of the second product: 8 tokens x D/16 channels, transposed in pairs of tokens
#pragma unroll
    for (int x = 0; x < D / 64; ++x) {
        unsigned wide[8][2];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            wide[e][0] = widen2<CODE, f16, 0>(st.v[e][x]);
            wide[e][1] = widen2<CODE, f16, 1>(st.v[e][x]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            u32x4 a;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                a[e] = __builtin_amdgcn_perm(wide[2 * e + 1][j >> 1], wide[2 * e][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
            if (slow) {
                u32x4 nan = {0u, 0u, 0u, 0u};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const bool is = ((st.v[e][x] >> (8 * j)) & 0x7fu) == 0x7fu;
                    const unsigned keep = (e & 1) ? 0x0000ffffu : 0xffff0000u, one = (e & 1) ? 0x3c000000u : 0x00003c00u;
                    if (is) {
                        a[e >> 1] &= keep;
                        nan[e >> 1] |= one;
                    }
                }
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    u32x4 sees = {0u, 0u, 0u, 0u};
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (tok + e < limit[c] && st.held) sees[e >> 1] |= (e & 1) ? 0x3c000000u : 0x00003c00u;
                    const f32x4 hit = mfma16x32(__builtin_bit_cast(f16x8, nan), __builtin_bit_cast(f16x8, sees), f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (hit[e] > 0.f) sm.o[c][4 * x + j][e] = __builtin_nanf("");
                }
            }
#pragma unroll
            for (int c = 0; c < NC; ++c) sm.o[c][4 * x + j] = mfma16x32(__builtin_bit_cast(f16x8, a), w[c], sm.o[c][4 * x + j]);
        }
    }
}

template <typename T, int CODE, int D, int NC, int W>
__global__ void __launch_bounds__(W * 64) paged_decode_kernel(const AttnParams p) {
    constexpr int kRows = 16 * NC, kThreads = W * 64;
    __shared__ ScheduleLds<kThreads> sched;
    __shared__ float lds_ml[W][kRows][2], lds_r[W];
    extern __shared__ float lds_o[];                       // [W/2][kRows][D]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, i = lane & 15;
    const int head = blockIdx.y;
    if (p.clear_tail && blockIdx.x == gridDim.x - 1) {     // the last workgroups also clear the rows behind the last request
        const int from = p.n ? min(max(p.cu[p.n], 0), p.tokens) : 0;
        for (int64_t t = from; t < p.tokens; ++t)
            for (int x = tid; x < p.group * D; x += kThreads) {
                const int h = head * p.group + x / D;
                static_cast<T *>(p.out)[t * p.o_t + h * p.o_h + x % D] = (T)0.f;
                if (p.lse && x % D == 0) p.lse[t * p.lse_t + h * p.lse_h] = kNegInf;
            }
    }
    int64_t base;
    const Item it = find_item<kThreads, kRows>(p, blockIdx.x, false, sched, base);
    if (!it.found) return;
    const Request rq = request_of(p, it.r);
    // queries: column i of tile c is row kRows * tile + 16 c + i of the request's list
    u32x4 q[NC][D / 32];
    int limit[NC], least = INT32_MAX, most = 0;
    const int64_t table_most = (int64_t)p.width << p.shift;
    const int cap = (int)min((int64_t)rq.len, table_most);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int row = it.tile * kRows + 16 * c + i, tok = row / p.group, h = head * p.group + row % p.group;
        const bool real = row < rq.rows;
        limit[c] = real ? min(max(rq.len - rq.new_tokens + tok + 1, 0), cap) : 0;
        const T *src = static_cast<const T *>(p.q) + (int64_t)(rq.first + (real ? tok : 0)) * p.q_t + (real ? h : 0) * p.q_h;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const u32x4 x = *reinterpret_cast<const u32x4 *>(src + 64 * (s >> 1) + 16 * g + 8 * (s & 1));
            q[c][s] = real ? x : u32x4{0u, 0u, 0u, 0u};
        }
        int lo = real ? limit[c] : INT32_MAX, hi = limit[c];
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            lo = min(lo, __shfl_xor(lo, d, kWave));
            hi = max(hi, __shfl_xor(hi, d, kWave));
        }
        least = min(least, lo);
        most = max(most, hi);
    }
    Softmax<D, NC> sm;
    sm.r = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        sm.m[c] = kNegInf;
        sm.l[c] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) sm.o[c][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const int64_t from = (int64_t)it.chunk * it.units * kUnit;
    const int end = (int)min((int64_t)most, it.chunks == 1 ? (int64_t)most : from + (int64_t)it.units * kUnit);
    const int32_t *row = p.table + it.r * p.table_s;
    int t0 = (int)min(from, (int64_t)INT32_MAX - 65536) + 32 * wave;
    if (t0 < end) {
        KvStep<D> cur;
        load_step<D>(p, head, t0, lane_page(p, row, t0), most, cur);
        int page = t0 + 32 * W < end ? lane_page(p, row, t0 + 32 * W) : -1;
        while (true) {
            const int next = t0 + 32 * W;
            KvStep<D> nxt;
            if (next < end) {
                load_step<D>(p, head, next, page, most, nxt);
                page = next + 32 * W < end ? lane_page(p, row, next + 32 * W) : -1;
            }
            attend_step<T, CODE, D, NC>(p, cur, q, limit, least, most, t0, sm);
            if (next >= end) break;
            cur = nxt;
            t0 = next;
        }
    }
    // join the waves: statistics first, then the accumulators pairwise through LDS
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        sm.l[c] += __shfl_xor(sm.l[c], 16, kWave);
        sm.l[c] += __shfl_xor(sm.l[c], 32, kWave);
        if (g == 0) {
            lds_ml[wave][16 * c + i][0] = sm.m[c];
            lds_ml[wave][16 * c + i][1] = sm.l[c];
        }
    }
    if (lane == 0) lds_r[wave] = sm.r;
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
        const float by = sm.l[c] == 0.f ? 0.f : exp2f(sm.m[c] - m[c]) * sm.r;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) sm.o[c][j] *= by;
    }
#pragma unroll
    for (int half = W / 2; half >= 1; half >>= 1) {
        if (wave >= half && wave < 2 * half) {
            float *dst = lds_o + (size_t)(wave - half) * kRows * D;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) dst[((c * (D / 16) + j) * 4 + e) * 64 + lane] = sm.o[c][j][e];
        }
        __syncthreads();
        if (wave < half) {
            const float *src = lds_o + (size_t)wave * kRows * D;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sm.o[c][j][e] += src[((c * (D / 16) + j) * 4 + e) * 64 + lane];
        }
        __syncthreads();
    }
    if (wave != 0) return;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int r = it.tile * kRows + 16 * c + i;
        if (r >= rq.rows) continue;
        if (it.chunks == 1) {
            const int64_t tok = rq.first + r / p.group;
            const int h = head * p.group + r % p.group;
            const float by = l[c] > 0.f || l[c] != l[c] ? 1.f / l[c] : 0.f;
            T *dst = static_cast<T *>(p.out) + tok * p.o_t + h * p.o_h;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < D / 16; ++j) dst[D / 16 * (4 * g + e) + j] = (T)(sm.o[c][j][e] * by);
            if (p.lse && g == 0) p.lse[tok * p.lse_t + h * p.lse_h] = (m[c] + log2f(l[c])) * (1.f / kLog2e);
        } else {
            const int64_t slot = ((int64_t)blockIdx.x * p.heads + head) * kRows + 16 * c + i;
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int j = 0; j < D / 16; ++j) p.part_o[slot * D + D / 16 * (4 * g + e) + j] = sm.o[c][j][e];
            if (g == 0) {
                p.part_ml[slot * 2] = m[c];
                p.part_ml[slot * 2 + 1] = l[c];
            }
        }
    }
}

// Joins the chunks of a tile: one workgroup of 64 threads for each (tile, cache head, query row).
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(64) paged_join_kernel(const AttnParams p) {
    __shared__ ScheduleLds<64> sched;
    int64_t base;
    const Item it = find_item<64, ROWS>(p, blockIdx.x, true, sched, base);
    if (!it.found || it.chunks == 1) return;
    const Request rq = request_of(p, it.r);
    const int head = blockIdx.y, r = it.tile * ROWS + blockIdx.z, lane = threadIdx.x;
    if (r >= rq.rows) return;
    const int64_t first = (base * p.heads + head) * ROWS + blockIdx.z, step = (int64_t)p.heads * ROWS;
    float m = kNegInf;
    for (int c = lane; c < it.chunks; c += 64) m = fmaxf(m, p.part_ml[(first + c * step) * 2]);
#pragma unroll
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, kWave));
    float l = 0.f, o[D / 64];
#pragma unroll
    for (int x = 0; x < D / 64; ++x) o[x] = 0.f;
#pragma unroll 4
    for (int c = 0; c < it.chunks; ++c) {
        const int64_t slot = first + c * step;
        const float lc = p.part_ml[slot * 2 + 1], by = lc == 0.f ? 0.f : exp2f(p.part_ml[slot * 2] - m);
        l += by * lc;
#pragma unroll
        for (int x = 0; x < D / 64; ++x) o[x] += by * p.part_o[slot * D + x * 64 + lane];
    }
    const int64_t tok = rq.first + r / p.group;
    const int h = head * p.group + r % p.group;
    const float by = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
    for (int x = 0; x < D / 64; ++x) static_cast<T *>(p.out)[tok * p.o_t + h * p.o_h + x * 64 + lane] = (T)(o[x] * by);
    if (p.lse && lane == 0) p.lse[tok * p.lse_t + h * p.lse_h] = (m + log2f(l)) * (1.f / kLog2e);
}

struct Plan {
    int nc, waves;
    int64_t tiles, items;      // bounds
    uint64_t o_bytes, bytes;
};

template <typename T, int CODE, int D, int NC> int launch_decode(const AttnParams &p, const Plan &plan, hipStream_t stream) {
    constexpr int W = 4;
    const dim3 grid((unsigned)plan.items, (unsigned)p.heads);
    const size_t lds = (size_t)(W / 2) * 16 * NC * D * 4;
    FLA_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(paged_decode_kernel<T, CODE, D, NC, W>),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds));
    FLA_LAUNCH("paged_kv_attention", stream, (paged_decode_kernel<T, CODE, D, NC, W>), grid, dim3(W * 64), lds, stream, p);
    FLA_HIP_CHECK(hipGetLastError());
    if (p.target) {
        FLA_LAUNCH("paged_kv_attention_join", stream, (paged_join_kernel<T, D, 16 * NC>), dim3((unsigned)plan.tiles, (unsigned)p.heads, 16 * NC), dim3(64), 0, stream, p);
        FLA_HIP_CHECK(hipGetLastError());
    }
    return FLA_OK;
}

template <typename T, int CODE> int launch_dim(const AttnParams &p, const Plan &plan, int dim, hipStream_t stream) {
#define FLA_NC(DD)                                                                   \
    do {                                                                             \
        if (plan.nc == 1) return launch_decode<T, CODE, DD, 1>(p, plan, stream);     \
        if (plan.nc == 2) return launch_decode<T, CODE, DD, 2>(p, plan, stream);     \
    } while (0)
    if (dim == 64) FLA_NC(64);
    else if (dim == 128) FLA_NC(128);
    else FLA_NC(256);
#undef FLA_NC
    return fail(FLA_ERR_UNSUPPORTED, "paged_kv_attention: no kernel for this shape.");
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

    Plan plan{};
    const int64_t longest = !present(cu) ? 1 : max_query_len ? (max_query_len < T ? max_query_len : T) : T;
    plan.nc = longest * group > 16 ? 2 : 1;
    const int64_t rows = 16 * plan.nc;
    plan.tiles = T * group / rows + n;
    AttnParams p{};
    p.target = (int)((1024 + shape.heads - 1) / shape.heads);
    p.min_units = 4;
    plan.items = plan.tiles + p.target;
    FLA_REQUIRE(plan.items < ((int64_t)1 << 31), FLA_ERR_SHAPE, "%s: too many query rows.", op);
    plan.o_bytes = (uint64_t)plan.items * shape.heads * rows * dim * 4;
    plan.bytes = plan.o_bytes + (uint64_t)plan.items * shape.heads * rows * 8;
    if (query) {
        *query = T && n ? plan.bytes : 0;
        return FLA_OK;
    }
    if (T == 0 || n == 0) return FLA_OK;
    FLA_REQUIRE(workspace && size >= plan.bytes, FLA_ERR_WORKSPACE, "%s: workspace of %llu bytes required, got %llu.", op,
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
#define FLA_CODE(T) (shape.code == FLA_I8 ? launch_dim<T, FLA_I8>(p, plan, (int)dim, stream) : launch_dim<T, FLA_F8E4M3>(p, plan, (int)dim, stream))
    return q->dtype == FLA_BF16 ? FLA_CODE(bf16) : FLA_CODE(f16);
#undef FLA_CODE
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
