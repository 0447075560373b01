"""Paged 8-bit cache operators against their 64-bit restatement.

Bounds (eps = torch.finfo(type).eps; a rounding is off by at most eps / 2 of the value):
* plan, append: equal.  Scales are powers of two, so x / scale is exact and the code is one rounding of it.
* rotary: one rounding to the output type, plus fp32 arithmetic on (a, b): the sine and cosine are within 2^-22 (an fp32
  fraction of a turn, 2^-24 of at most pi, and the function's own 2^-23), two products and a sum add 3 * 2^-24 of
  |a| + |b| <= 2^-21 (|a| + |b|) in all.
* attention: one rounding to the output type.  Every weight carries 2^-12 (fp16) and the error of its score: a sum of D
  products in fp32, at most (D + 8) * 2^-24 of sum |q||k| * scale, twice (weight and normalisation).  These are relative
  errors of weights, so they count for sum p|v| ("spread").  A weight below 2^-14 is off by at most 2^-25 of the
  row's largest p * value scale ("peak") times the largest code, for each token.  lse: the score error, and 2^-21 of its value.
"""
import math
import random

import pytest
import torch

from oracle import paged_kv as ref

pytestmark = pytest.mark.gpu
E4M3, INT8 = torch.float8_e4m3fn, torch.int8
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


# ---- plan ------------------------------------------------------------------------------------------------------------

def make_plan(n, page, seed, most_context, most_query, spare=3, width_cut=0):
    rng = random.Random(seed)
    context = [rng.choice([0, 1, page - 1, page, page + 1, rng.randint(0, most_context)]) for _ in range(n)]
    query = [rng.choice([0, 1, 1, rng.randint(0, most_query)]) for _ in range(n)]
    width = max(1, max(-(-(c + q) // page) for c, q in zip(context, query)) - width_cut)
    ids = list(range(100000))
    rng.shuffle(ids)
    table = []
    for c in context:
        held = min(-(-c // page), width)
        table.append([ids.pop() for _ in range(held)] + [-7] * (width - held))
    need = sum(min(-(-(c + q) // page), width) - min(-(-c // page), width) for c, q in zip(context, query))
    free = [ids.pop() for _ in range(max(0, need + spare))]
    return context, query, table, free


@pytest.mark.parametrize("n,page,most_context,most_query,pad,spare,cut", [
    (1, 16, 40, 1, 0, 3, 0), (3, 64, 300, 5, 4, 0, 0), (7, 32, 0, 200, 0, 1, 0), (257, 16, 90, 3, 31, 9, 0),
    (1030, 16, 40, 4, 0, 0, 0), (2500, 64, 100, 3, 1000, 2, 0), (5, 256, 1000, 3000, 7, 0, 0),
    (9, 16, 200, 60, -50, 0, 0), (40, 16, 100, 40, 3, -5, 0), (12, 32, 300, 100, 0, 2, 2)])
def test_plan(dev, n, page, most_context, most_query, pad, spare, cut):
    from fla_hip import ops
    context, query, table, free = make_plan(n, page, 7 * n + page, most_context, most_query, spare, cut)
    tokens = max(0, sum(query) + pad)
    rows = random.Random(n).sample(range(5000), n)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    wide = torch.full((n, len(table[0]) + 3), -9, dtype=torch.int32, device=dev)     # rows that are not adjacent
    wide[:, :-3] = i32(table)
    view = wide[:, :-3]
    got = ops.paged_kv_plan(i32(context), i32(query), view, i32(free), page, tokens, state_rows=i32(rows))
    want = ref.plan(context, query, table, free, page, tokens, rows)
    for name, g in zip(("slots", "positions", "cu", "seq", "used", "states"), got):
        assert g.dtype == want[name].dtype and torch.equal(g.cpu(), want[name]), name
    assert torch.equal(view.cpu(), want["table"])
    assert bool((wide[:, -3:] == -9).all())
    assert ops.paged_kv_plan(i32(context), i32(query), view, i32(free), page, tokens)[5] is None


def test_plan_negative_lengths_count_as_zero_and_nothing_to_do(dev):
    from fla_hip import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    table = torch.full((3, 2), -1, dtype=torch.int32, device=dev)
    slots, pos, cu, seq, used, _ = ops.paged_kv_plan(i32([-4, 3, 0]), i32([2, -1, 0]), table, i32([5]), 16, 3)
    assert slots.tolist() == [80, 81, -1] and cu.tolist() == [0, 2, 2, 2] and seq.tolist() == [2, 3, 0] and used.tolist() == [1]
    assert table.tolist() == [[5, -1], [-1, -1], [-1, -1]]
    empty = torch.empty(0, dtype=torch.int32, device=dev)
    slots, pos, cu, seq, used, _ = ops.paged_kv_plan(i32([4]), i32([0]), table[:1], empty, 16, 0)
    assert slots.numel() == 0 and cu.tolist() == [0, 0] and used.tolist() == [0]
    slots, pos, cu, seq, used, st = ops.paged_kv_plan(empty, empty, table[:0], empty, 16, 2, state_rows=empty)
    assert slots.tolist() == [-1, -1] and cu.tolist() == [0] and st.tolist() == [-1, -1] and used.tolist() == [0]


# ---- rotary ----------------------------------------------------------------------------------------------------------

def rotary_bound(x, want, rotated, pairing, dtype):
    """Elementwise bound of the module's docstring."""
    half = rotated // 2
    a = x.double().abs()
    first, second = (slice(0, rotated, 2), slice(1, rotated, 2)) if pairing == "adjacent" else (slice(0, half), slice(half, rotated))
    pair = torch.zeros_like(a)
    pair[..., first] = pair[..., second] = a[..., first] + a[..., second]
    return want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + pair * 2.0 ** -21 + torch.finfo(dtype).tiny


ROTARY = [
    # batch, tokens, q heads, k heads, dim, rotated, sections, order, pairing, dtype
    ((), 1, 4, 1, 128, 128, (64,), "blocked", "half", BF),
    ((), 33, 5, 2, 64, 64, (12, 10, 10), "interleaved", "half", F16),
    ((2,), 65, 32, 8, 128, 64, (16, 8, 8), "blocked", "half", BF),
    ((2,), 9, 3, 3, 256, 64, (11, 11, 10), "interleaved", "adjacent", BF),
    ((), 4100, 2, 1, 64, 32, (8, 8), "blocked", "adjacent", F32),
    ((), 17, 3, 0, 80, 40, (20,), "blocked", "half", BF),            # pieces of 4
    ((3,), 5, 2, 1, 34, 18, (4, 3, 2), "interleaved", "half", F16),   # single elements
    ((), 7, 2, 1, 6, 6, (3,), "blocked", "adjacent", F32),
    ((), 21, 2, 2, 256, 256, (64, 32, 32), "blocked", "half", F32),
]


@pytest.mark.parametrize("batch,T,hq,hk,dim,rotated,sections,order,pairing,dtype", ROTARY)
@pytest.mark.parametrize("head_first", [False, True])
def test_rotary_forward_and_gradient(dev, batch, T, hq, hk, dim, rotated, sections, order, pairing, dtype, head_first):
    from fla_hip import ops
    gen = torch.Generator().manual_seed(T * dim)

    def new(h):
        x = torch.randn(*batch, T, h, dim, generator=gen).to(dtype).to(dev)
        return x.transpose(-2, -3).contiguous().transpose(-2, -3) if head_first else x

    q, k = new(hq), new(hk) if hk else None
    pos = torch.randint(0, 1 << 20, (len(sections), *batch, T), generator=gen)
    pos.flatten()[0] = 1 << 30
    inv = (10000.0 ** (-torch.arange(rotated // 2, dtype=torch.float64) / (rotated // 2))).float()
    args = (pos.to(dev) if T % 2 else pos.int().to(dev), inv.to(dev), sections)
    how = dict(axis_order=order, pairing=pairing)
    xs = [x for x in (q, k) if x is not None]
    for x in xs:
        x.requires_grad_()
    got = ops.rotary_axes(q, k, *args, **how)
    grads = [torch.randn(x.shape, generator=gen).to(dtype).to(dev) for x in xs]
    back = torch.autograd.grad([g for g in got if g is not None], xs, grads)
    assert (got[1] is None) == (k is None)
    for x, y, dy, dx in zip(xs, got, grads, back):
        assert y.dtype == dtype and y.stride() == x.stride()
        for source, result, inverse in ((x, y, False), (dy, dx, True)):
            want = ref.rotary(source.detach().cpu(), pos, inv, sections, order, pairing, inverse)
            error = (result.detach().cpu().double() - want).abs()
            bound = rotary_bound(source.detach().cpu(), want, rotated, pairing, dtype)
            assert bool((error <= bound).all()), float((error / bound).max())
        assert torch.equal(y[..., rotated:], x.detach()[..., rotated:])


def test_rotary_gradient_against_differences(dev):
    """The operator is linear in x: central differences in fp32 with a step of 1 are exact up to rounding (2^-21 of the pair,
    twice, each way)."""
    from fla_hip import ops
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(3, 2, 16, generator=gen).to(dev).requires_grad_()
    pos, inv, dy = torch.randint(0, 999, (2, 3), generator=gen).to(dev), torch.rand(4, generator=gen).to(dev), torch.randn(3, 2, 16, generator=gen).to(dev)
    y, _ = ops.rotary_axes(x, None, pos, inv, (2, 2), pairing="adjacent")
    (dx,) = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        for i in (0, 1, 6, 7, 8, 15):
            step = torch.zeros_like(x)
            step[1, 1, i] = 1
            plus, minus = (ops.rotary_axes(x + s * step, None, pos, inv, (2, 2), pairing="adjacent")[0] for s in (1, -1))
            num = ((plus - minus).double() * dy.double()).sum() / 2
            assert abs(float(num) - float(dx[1, 1, i])) <= 16 * 2.0 ** -21 * float(dy[1, 1].abs().sum()), i


def test_rotary_one_gradient_only_and_expanded_gradient(dev):
    from fla_hip import ops
    q, k = torch.randn(5, 2, 64, device=dev, requires_grad=True), torch.randn(5, 1, 64, device=dev, requires_grad=True)
    pos, inv = torch.arange(5, device=dev)[None], torch.rand(32, device=dev)
    a, b = ops.rotary_axes(q, k, pos, inv, (32,))
    (dk,) = torch.autograd.grad(b.sum(), k, retain_graph=True)      # an expanded gradient, and none for q
    want = ref.rotary(torch.ones(5, 1, 64), pos.cpu(), inv.cpu(), (32,), "blocked", "half", True)
    assert torch.allclose(dk.cpu().double(), want, atol=2.0 ** -19, rtol=0)
    (dq,) = torch.autograd.grad(a.sum(), q)
    assert torch.allclose(dq.cpu().double(), want.expand(5, 2, 64), atol=2.0 ** -19, rtol=0)


# ---- append ----------------------------------------------------------------------------------------------------------

def codes_of(cache):
    return cache.cpu().double() if cache.dtype == INT8 else cache.cpu().float().double()


def random_cache(gen, pool, heads, page, dim, code, dev, token_major=False):
    x = torch.randn(pool, heads, page, dim, generator=gen)
    c = (x * 31).round().clamp(-127, 127).to(INT8) if code == INT8 else (x * 100).clamp(-448, 448).to(E4M3)
    s = 2.0 ** torch.randint(-9, -4, (pool, heads), generator=gen).float()
    c = c.to(dev)
    if token_major:
        c = c.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(code)
    return c, s.to(dev)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("page,dim,heads,token_major", [(16, 64, 3, False), (64, 128, 2, True), (256, 256, 1, False), (32, 256, 2, True)])
def test_append(dev, dtype, code, page, dim, heads, token_major):
    from fla_hip import ops
    gen = torch.Generator().manual_seed(page + dim)
    pool = 9
    kc, ks = random_cache(gen, pool, heads, page, dim, code, dev, token_major)
    vc, vs = random_cache(gen, pool, heads, page, dim, code, dev, token_major)
    # runs: inside a page, up to its end, from its start, one row, a full page, skipped rows between, past the pool
    runs = [(3, 5, 7), (5, page - 4, 4), (2, 0, 3), (-1, 0, 2), (7, page - 1, 1), (0, 0, page), (pool, 0, 3), (1, 1, 1), (8, 0, 1), (8, 1, page - 1)]
    slots = [s for b, o, n in runs for s in ([-1] * n if b < 0 else range(b * page + o, b * page + o + n))]
    T = len(slots)
    size = torch.exp(torch.randn(T, 1, 1, generator=gen) * 2)
    make = lambda: (torch.randn(T, heads, dim, generator=gen) * size).to(dtype)
    k, v = make(), make()
    k[0, 0] = 0
    k[0, 0, 1] = 1e-7                    # scale stays, code rounds to 0
    v[runs[0][2] + 4 + 1] = 0            # rows of zeros
    k[slots.index(3 * page + 7), 1 % heads, 3:6] = torch.tensor([math.inf, -math.inf, math.nan])
    kc2, vc2, ks2, vs2 = clone_strided(kc), clone_strided(vc), ks.clone(), vs.clone()
    ops.paged_kv_append(k.to(dev), v.to(dev), kc2, vc2, ks2, vs2, torch.tensor(slots, device=dev))
    for x, c, s, c2, s2, name in ((k, kc, ks, kc2, ks2, "key"), (v, vc, vs, vc2, vs2, "value")):
        want, scale = codes_of(c), s.cpu().double()
        ref.append(x, want, scale, slots, code)
        assert torch.equal(s2.cpu().double(), scale), name
        got = codes_of(c2)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num()), name


def clone_strided(c):
    raw = torch.empty_strided(c.shape, c.stride(), dtype=torch.uint8, device=c.device)
    raw.copy_(c.view(torch.uint8))
    return raw.view(c.dtype)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_extremes_of_scale(dev, code):
    """All zeros (scale 0, then the first larger row), the smallest and largest fp32 magnitudes, exact powers of two times the
    largest code and its neighbours."""
    from fla_hip import ops
    most = ref.LARGEST[code]
    up = lambda x: float(torch.nextafter(torch.tensor(x), torch.tensor(math.inf)))
    tops = [0.0, 1e-45, 2.0 ** -126, most * 2.0 ** -126, most, up(most), most * 2.0 ** 30, up(most * 2.0 ** 30), 3.4e38, 2.0, 1.0, 1.75, up(1.75), 1.984375, up(1.984375)]
    T, page = len(tops), 16
    x = torch.zeros(T, 1, 64)
    x[:, 0, 0] = torch.tensor(tops)
    x[:, 0, 1] = -torch.tensor(tops) / 3
    slots = [t * page for t in range(T)]
    new = lambda: torch.zeros(T, 1, page, 64, dtype=torch.uint8, device=dev).view(code)
    kc, vc, ks, vs = new(), new(), torch.full((T, 1), 77.0, device=dev), torch.full((T, 1), 77.0, device=dev)
    for step in range(2):                # the second row of each page comes after the first, ten times as large
        rows = (x * 10 ** step).clamp(-3.4e38, 3.4e38)
        ops.paged_kv_append(rows.to(dev), (-rows).to(dev), kc, vc, ks, vs, torch.tensor([s + step for s in slots], device=dev))
        if step == 0:
            want, scale = torch.zeros(T, 1, page, 64, dtype=torch.float64), torch.full((T, 1), 77.0, dtype=torch.float64)
        ref.append(rows, want, scale, [s + step for s in slots], code)
        assert torch.equal(ks.cpu().double(), scale) and torch.equal(vs.cpu().double(), scale)
        assert torch.equal(codes_of(kc), want) and torch.equal(codes_of(vc), -want)


# ---- attention -------------------------------------------------------------------------------------------------------

def make_table(rng, lens, page, width, pool):
    ids = list(range(pool))
    rng.shuffle(ids)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for r, n in enumerate(lens):
        for j in range(min(-(-n // page), width)):
            table[r, j] = ids.pop()
    return table


def check_attention(dev, q, caches, table, lens, cu, scale, *, got=None, **kw):
    from fla_hip import ops
    kc, vc, ks, vs = caches
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    if got is None:
        got = ops.paged_kv_attention(q.to(dev), kc, vc, ks, vs, table.to(dev), i32(lens), None if cu is None else i32(cu), scale=scale, return_lse=True, **kw)
    out, lse = (t.cpu().double() for t in got)
    want, want_lse, spread, reach, peak = ref.attention(q, codes_of(kc), codes_of(vc), ks.cpu(), vs.cpu(), table, lens, cu, scale)
    d = q.shape[-1]
    score = (d + 8) * 2.0 ** -24 * reach
    top = peak[..., None] * ref.LARGEST[kc.dtype]
    bound = want.abs() * torch.finfo(q.dtype).eps / 2 * 1.01 + spread * (2.0 ** -12 * 1.01 + 2 * score[..., None]) + max(lens) * 2.0 ** -25 * top + torch.finfo(q.dtype).tiny
    assert torch.equal(out.isnan(), want.isnan())
    error = torch.where(want.isnan(), 0.0, (out - want).abs())
    assert bool((error <= torch.where(bound.isnan(), math.inf, bound)).all()), float((error / bound).nan_to_num().max())
    seen = want_lse > -math.inf
    assert torch.equal(lse > -math.inf, seen)
    lse_error = (lse - want_lse)[seen].abs()
    assert bool((lse_error <= score[seen] + 2.0 ** -21 * (1 + want_lse[seen].abs())).all()), float(lse_error.max())
    return out, lse


DECODE = [
    # page, heads, kv heads, dim, query type, code
    (64, 8, 2, 128, BF, E4M3), (16, 6, 1, 64, F16, INT8), (32, 4, 4, 256, BF, INT8), (128, 20, 1, 128, F16, E4M3),
    (256, 5, 1, 64, BF, E4M3), (16, 40, 2, 256, F16, E4M3), (64, 7, 7, 128, BF, INT8)]


@pytest.mark.parametrize("page,heads,kv_heads,dim,dtype,code", DECODE)
def test_decode(dev, page, heads, kv_heads, dim, dtype, code):
    rng, gen = random.Random(page + heads), torch.Generator().manual_seed(heads * dim)
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 256, 257, 700, 3, 1029, 8]
    width = max(-(-n // page) for n in lens) + 2
    pool = sum(-(-n // page) for n in lens) + 5
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, code, dev, token_major=page == 32)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, code, dev, token_major=page == 32)
    q = torch.randn(len(lens), heads, dim, generator=gen).to(dtype)
    out, lse = check_attention(dev, q, (kc, vc, ks, vs), make_table(rng, lens, page, width, pool), lens, None, dim ** -0.5)
    assert bool((out[1] == 0).all()) and bool((lse[1] == -math.inf).all())


@pytest.mark.parametrize("page,heads,kv_heads,dim,dtype,code", DECODE)
def test_several_query_rows(dev, page, heads, kv_heads, dim, dtype, code):
    """Ragged numbers of query rows, causal inside them; a request without any, one whose query is its whole text."""
    rng, gen = random.Random(page), torch.Generator().manual_seed(page * dim)
    new = [1, 4, 0, 7, 33, 70, 2, 5]
    lens = [50, 4, 30, 300, 40, 70, 1 + 2 * page, 260]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    width = max(-(-n // page) for n in lens)
    pool = sum(-(-n // page) for n in lens) + 2
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, code, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, code, dev)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(dtype)
    table = make_table(rng, lens, page, width, pool)
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, cu, dim ** -0.5, max_query_len=70)
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, cu, 0.2)
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, cu, dim ** -0.5, max_query_len=1)     # a hint that is wrong only costs time


@pytest.mark.parametrize("lens", [[20011], [9000, 1, 0, 300], [2049, 4097, 64]])
@pytest.mark.parametrize("code", [E4M3, INT8])
def test_long_contexts_are_split_and_joined(dev, lens, code):
    rng, gen = random.Random(1), torch.Generator().manual_seed(len(lens))
    page, heads, kv_heads, dim = 64, 8, 2, 128
    pool = sum(-(-n // page) for n in lens) + 2
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, code, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, code, dev)
    table = make_table(rng, lens, page, max(-(-n // page) for n in lens), pool)
    q = torch.randn(len(lens), heads, dim, generator=gen).to(BF)
    check_attention(dev, q * 3, (kc, vc, ks, vs), table, lens, None, dim ** -0.5)
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + min(n, 3))
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(BF)
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, cu, dim ** -0.5, max_query_len=3)


@pytest.mark.parametrize("new", [1, 5, 80])
@pytest.mark.parametrize("page", [16, 64])
def test_what_is_not_seen_may_hold_anything(dev, new, page):
    """NaN codes behind the last token, in pages of nobody, in tokens that only later rows see; scales of pages of nobody
    NaN and infinite; table entries behind the last page that name them."""
    rng, gen = random.Random(3), torch.Generator().manual_seed(page)
    heads, kv_heads, dim, lens = 8, 2, 128, [new + 5, new + page, new, new + 3 * page + 7]
    pool = sum(-(-n // page) for n in lens) + 6
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    width = max(-(-n // page) for n in lens) + 3
    table = make_table(rng, lens, page, width, pool)
    owned = set(table[table >= 0].tolist())
    nobody = [b for b in range(pool) if b not in owned]
    nan = 0x7f
    for c in (kc, vc):
        raw = c.view(torch.uint8)
        raw[nobody] = nan
        for r, n in enumerate(lens):
            if n % page:
                raw[int(table[r, (n - 1) // page]), :, n % page:] = nan
    for s, bad in ((ks, math.nan), (vs, math.inf), (vs, math.nan)):
        s[nobody[::2] if bad == math.inf else nobody[1::2]] = bad
    for r in range(len(lens)):
        table[r, -(-lens[r] // page):] = torch.tensor([nobody[(r + j) % len(nobody)] for j in range(width - -(-lens[r] // page))])
    cu = [new * r for r in range(len(lens) + 1)]
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(BF)
    safe_ks, safe_vs = ks.clone(), vs.clone()
    safe_ks[nobody] = 0
    safe_vs[nobody] = 0
    from fla_hip import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    got = ops.paged_kv_attention(q.to(dev), kc, vc, ks, vs, table.to(dev), i32(lens), i32(cu), return_lse=True)
    check_attention(dev, q, (kc, vc, safe_ks, safe_vs), table, lens, cu, dim ** -0.5, got=got)
    if new > 1:                            # the last token of request 0: its row sees a NaN, the others must not
        where = int(table[0, (lens[0] - 1) // page]), (lens[0] - 1) % page
        kc.view(torch.uint8)[where[0], :, where[1]] = nan
        vc.view(torch.uint8)[where[0], 0, where[1], 5] = nan
        got = ops.paged_kv_attention(q.to(dev), kc, vc, ks, vs, table.to(dev), i32(lens), i32(cu), return_lse=True)
        out = got[0].cpu()
        assert bool(out[new - 1].isnan().all()) and bool(out[:new - 1].isfinite().all()) and bool(out[new:].isfinite().all())
        kc.view(torch.uint8)[where[0], :, where[1]] = 0x38
        got = ops.paged_kv_attention(q.to(dev), kc, vc, ks, vs, table.to(dev), i32(lens), i32(cu), return_lse=True)
        check_attention(dev, q, (kc, vc, safe_ks, safe_vs), table, lens, cu, dim ** -0.5, got=got)
        assert bool(got[0][new - 1, :heads // kv_heads, 5].isnan().all()) and int(got[0].isnan().sum()) == heads // kv_heads


def test_pages_outside_the_pool_are_not_seen(dev):
    rng, gen = random.Random(4), torch.Generator().manual_seed(4)
    page, heads, kv_heads, dim = 16, 4, 1, 64
    lens = [100, 70, 40, 33]
    kc, ks = random_cache(gen, 30, kv_heads, page, dim, INT8, dev)
    vc, vs = random_cache(gen, 30, kv_heads, page, dim, INT8, dev)
    table = make_table(rng, lens, page, 5, 30)                  # request 0 is longer than its row of the table
    table[0, 1], table[1, 0], table[1, 3] = -1, 30, 2 ** 31 - 1
    table[2] = -5                                                # sees nothing
    q = torch.randn(4, heads, dim, generator=gen).to(BF)
    out, lse = check_attention(dev, q, (kc, vc, ks, vs), table, lens, None, dim ** -0.5)
    assert bool((out[2] == 0).all()) and bool((lse[2] == -math.inf).all())


@pytest.mark.parametrize("new", [1, 40])
def test_scales_of_very_different_sizes(dev, new):
    """Pages of zeros (scale 0), of tiny and of large values side by side."""
    rng, gen = random.Random(6), torch.Generator().manual_seed(6)
    page, heads, kv_heads, dim, lens = 16, 8, 2, 128, [333, 250]
    pool = 60
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    vs.copy_(torch.tensor([0.0, 2.0 ** -126, 1e-30, 1e-3, 1.0, 37.0])[torch.randint(0, 6, (pool, kv_heads), generator=gen)])
    ks[::3] = 0
    table = make_table(rng, lens, page, 21, pool)
    q = torch.randn(2 * new, heads, dim, generator=gen).to(BF)
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, [0, new, 2 * new], dim ** -0.5)
    # one request whose rows look at pages with tiny values next to pages with large ones that they all but ignore
    kc.copy_(torch.where(torch.rand(pool, 1, 1, 1, generator=gen) < 0.5, 1.0, -1.0).expand(pool, kv_heads, page, dim).to(E4M3))
    ks.fill_(1.0)
    vs.copy_(torch.where(codes_of(kc)[:, 0, 0, :1] > 0, 2.0 ** -30, 2.0 ** 10).expand(pool, kv_heads).float())
    check_attention(dev, torch.full((2 * new, heads, dim), 0.5).to(BF), (kc, vc, ks, vs), table, lens, [0, new, 2 * new], 0.5)
    vs.fill_(2.0 ** -120)                  # fp32 holds it, the result type bf16 as well
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, [0, new, 2 * new], dim ** -0.5)
    vs.zero_()
    out, _ = check_attention(dev, q, (kc, vc, ks, vs), table, lens, [0, new, 2 * new], dim ** -0.5)
    assert bool((out == 0).all())


def test_peaked_and_far_scores(dev):
    """Scores of a few hundred with the largest at the end, at the start, and all equal."""
    rng, gen = random.Random(8), torch.Generator().manual_seed(8)
    page, heads, kv_heads, dim, lens = 64, 4, 1, 64, [500, 500, 500]
    kc, ks = random_cache(gen, 30, kv_heads, page, dim, INT8, dev)
    vc, vs = random_cache(gen, 30, kv_heads, page, dim, INT8, dev)
    table = make_table(rng, lens, page, 8, 30)
    ks.fill_(2.0 ** -5)
    first, last = int(table[0, 0]), int(table[1, 7])
    kc[first, :, 0] = 127
    kc[last, :, 499 % page] = 127
    kc[table[2].long()] = 1
    q = torch.full((3, heads, dim), 8.0).to(BF)
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, None, 1.0)
    check_attention(dev, -q, (kc, vc, ks, vs), table, lens, None, 1.0)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("new", [1, 20, 90])
def test_scores_that_jump_up_along_the_text(dev, new, wide):
    """Scores rise by 2 to 400 (in log2) from one step to the next, in steps that every row sees whole: maxima move by little
    (weights still fit fp16) and by much (they do not)."""
    rng, gen = random.Random(10), torch.Generator().manual_seed(10)
    page, heads, kv_heads, dim, n = 32, 4, 1, 64, 700
    kc, ks = random_cache(gen, 60, kv_heads, page, dim, INT8, dev)
    vc, vs = random_cache(gen, 60, kv_heads, page, dim, INT8, dev)
    lens = [n + new, n + new - 100]
    table = make_table(rng, lens, page, -(-max(lens) // page), 60)
    ks.fill_(2.0 ** -4)
    level = [1, 2, 3, 8, 9, 20, 21, 22, 50, 51, 52, 53, 100, 101, 126, 127]
    for r in range(2):
        for t in range(lens[r]):
            kc[int(table[r, t // page]), 0, t % page, 0] = level[min(t // 40, 15)] if t % 40 >= 33 else 0
    for weight in (2.0, 40.0, -40.0):                      # channel 0 of the queries: log2 of the weights rises by up to 400
        q = torch.randn(2 * new, heads, dim, generator=gen) * 0.1
        q[:, :, 0] = weight
        check_attention(dev, q.to(BF), (kc, vc, ks, vs), widen(table, page) if wide else table, lens, [0, new, 2 * new], 1.0, max_query_len=new)


def test_given_out_keeps_the_rows_behind_the_last_request(dev):
    from fla_hip import ops
    rng, gen = random.Random(9), torch.Generator().manual_seed(9)
    page, heads, kv_heads, dim, lens, cu = 16, 4, 2, 64, [20, 33], [0, 2, 5]
    kc, ks = random_cache(gen, 9, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, 9, kv_heads, page, dim, E4M3, dev)
    table = make_table(rng, lens, page, 3, 9)
    q = torch.randn(9, heads, dim, generator=gen).to(BF)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    args = (q.to(dev), kc, vc, ks, vs, table.to(dev), i32(lens), i32(cu))
    wide = torch.full((9, heads + 1, 2 * dim), 3.0, dtype=BF, device=dev)
    out = wide[:, 1:, :dim]
    version = wide._version
    assert ops.paged_kv_attention(*args, out=out) is out and wide._version > version
    new, lse = ops.paged_kv_attention(*args, return_lse=True)
    assert torch.equal(out[:5], new[:5]) and bool((out[5:] == 3).all()) and bool((wide[:, 0] == 3).all()) and bool((wide[:, :, dim:] == 3).all())
    assert bool((new[5:] == 0).all()) and bool((lse[5:] == -math.inf).all()) and bool(lse[:5].isfinite().all())
    check_attention(dev, q[:5], (kc, vc, ks, vs), table, lens, cu, dim ** -0.5, got=(new[:5], lse[:5]))


def test_cache_beyond_32_bit_offsets(dev):
    """Pages whose codes lie past 2^32 bytes."""
    from fla_hip import ops
    page, heads, kv_heads, dim = 64, 4, 8, 128
    pool = (1 << 32) // (page * kv_heads * dim) + 40
    caches = [torch.empty(pool, kv_heads, page, dim, dtype=torch.uint8, device=dev).view(E4M3) for _ in range(2)]
    scales = [torch.zeros(pool, kv_heads, device=dev) for _ in range(2)]
    gen = torch.Generator().manual_seed(1)
    lens, n = [150], 150
    table = torch.tensor([[pool - 1, 3, pool - 7]], dtype=torch.int32)
    slots = torch.tensor([int(table[0, t // page]) * page + t % page for t in range(n)], device=dev)
    k, v = torch.randn(n, kv_heads, dim, generator=gen).to(BF), torch.randn(n, kv_heads, dim, generator=gen).to(BF)
    ops.paged_kv_append(k.to(dev), v.to(dev), *caches, *scales, slots)
    q = torch.randn(1, 8 * 4, dim, generator=gen).to(BF)
    got = ops.paged_kv_attention(q.to(dev), *caches, *scales, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), return_lse=True)
    used = table[0].long()
    small = [c.view(torch.uint8)[used.to(dev)].view(E4M3) for c in caches] + [s[used.to(dev)] for s in scales]
    check_attention(dev, q, small, torch.tensor([[0, 1, 2]], dtype=torch.int32), lens, None, dim ** -0.5, got=got)


# Tables that name more than 2048 tokens split the keys over workgroups, whatever the lengths are.
WIDE = 5000


def widen(table, page):
    more = torch.full((table.shape[0], -(-WIDE // page)), -1, dtype=torch.int32)
    return torch.cat([table, more], 1)


@pytest.mark.parametrize("page,heads,kv_heads,dim,dtype,code", DECODE + [(32, 80, 1, 64, BF, E4M3)])
def test_wide_tables(dev, page, heads, kv_heads, dim, dtype, code):
    rng, gen = random.Random(page + heads), torch.Generator().manual_seed(heads * dim + 1)
    lens = [1, 0, 17, 700, 33, 1300, 2, 511, 513]
    pool = sum(-(-n // page) for n in lens) + 5
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, code, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, code, dev)
    table = widen(make_table(rng, lens, page, max(-(-n // page) for n in lens), pool), page)
    table[5, 3] = pool + 4                                      # a page that is not there
    q = torch.randn(len(lens), heads, dim, generator=gen).to(dtype)
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, None, dim ** -0.5)
    cu = [0, 1, 1, 8, 11, 11, 20, 22, 23, 40]
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(dtype)
    for hint in (17, 3, None):
        check_attention(dev, q, (kc, vc, ks, vs), table, lens, cu, dim ** -0.5, max_query_len=hint)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("n,most,new", [(150, 90, 1), (200, 400, 3), (130, 60, 25)])
def test_many_requests(dev, n, most, new, wide):
    """More requests than a wave has lanes; requests without rows and without tokens among them."""
    rng, gen = random.Random(n), torch.Generator().manual_seed(n)
    page, heads, kv_heads, dim = 16, 6, 2, 64
    rows = [rng.choice([0, 1, rng.randint(1, new)]) if new > 1 else 1 for _ in range(n)]
    lens = [rng.choice([r, r + rng.randint(0, most)]) for r in rows]
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    pool = sum(-(-m // page) for m in lens) + 3
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    table = make_table(rng, lens, page, max(-(-m // page) for m in lens), pool)
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(F16)
    check_attention(dev, q, (kc, vc, ks, vs), widen(table, page) if wide else table, lens, None if new == 1 else cu, dim ** -0.5, max_query_len=new)


@pytest.mark.parametrize("new", [1, 5, 80])
def test_what_is_not_seen_may_hold_anything_in_wide_tables(dev, new):
    rng, gen = random.Random(5), torch.Generator().manual_seed(5)
    page, heads, kv_heads, dim, lens = 16, 8, 2, 128, [new + 5, new + 900, new, new + 300]
    pool = sum(-(-n // page) for n in lens) + 4
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    table = widen(make_table(rng, lens, page, max(-(-n // page) for n in lens), pool), page)
    nobody = sorted(set(range(pool)) - set(table[table >= 0].tolist()))
    safe = [c.view(torch.uint8).clone().view(E4M3) for c in (kc, vc)] + [ks.clone(), vs.clone()]
    for c in (kc, vc):
        c.view(torch.uint8)[nobody] = 0x7f
        for r, n in enumerate(lens):
            if n % page:
                c.view(torch.uint8)[int(table[r, (n - 1) // page]), :, n % page:] = 0xff
    ks[nobody], vs[nobody] = math.nan, math.inf
    bad = table.clone()
    bad[table < 0] = nobody[0]
    cu = [new * r for r in range(len(lens) + 1)]
    q = torch.randn(cu[-1], heads, dim, generator=gen).to(BF)
    from fla_hip import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    got = ops.paged_kv_attention(q.to(dev), kc, vc, ks, vs, bad.to(dev), i32(lens), i32(cu), max_query_len=new, return_lse=True)
    check_attention(dev, q, safe, table, lens, cu, dim ** -0.5, got=got)


@pytest.mark.parametrize("code,dtype,page", [(E4M3, BF, 64), (INT8, F16, 16)])
def test_prefill_that_fills_the_chip(dev, code, dtype, page):
    """Enough tiles that keys are not split; against the formula in float64 on the GPU, a head at a time.  Padded rows."""
    from fla_hip import ops
    gen, rng = torch.Generator().manual_seed(3), random.Random(3)
    heads, kv_heads, dim, lens, rows, pad = 64, 64, 64, [2100, 700], [2000, 333], 30
    cu = [0, 2000, 2333]
    pool = sum(-(-n // page) for n in lens) + 2
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, code, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, code, dev)
    table = make_table(rng, lens, page, -(-lens[0] // page), pool).to(dev)
    q = torch.randn(cu[-1] + pad, heads, dim, generator=gen).to(dtype).to(dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    out, lse = ops.paged_kv_attention(q, kc, vc, ks, vs, table, i32(lens), i32(cu), max_query_len=2000, return_lse=True)
    assert bool((out[cu[-1]:] == 0).all()) and bool((lse[cu[-1]:] == -math.inf).all())
    values = lambda c, s, blocks, h: ((c[blocks, h].double() if code == INT8 else c.view(torch.uint8)[blocks, h].view(E4M3).float().double()) * s[blocks, h].double()[:, None, None]).flatten(0, 1)
    for r, n in enumerate(lens):
        blocks = table[r, :-(-n // page)].long()
        seen = torch.arange(n, device=dev) <= torch.arange(n - rows[r], n, device=dev)[:, None]
        for h in range(0, heads, 5):
            k, v = (values(c, s, blocks, h)[:n] for c, s in ((kc, ks), (vc, vs)))
            x = q[cu[r]:cu[r + 1], h].double()
            score = torch.where(seen, (x @ k.t()) * dim ** -0.5, -math.inf)
            p = torch.softmax(score, -1)
            want, spread = p @ v, p @ v.abs()
            err = (dim + 8) * 2.0 ** -24 * ((x.abs() @ k.abs().t()) * dim ** -0.5).amax(-1)
            peak = (p * vs[blocks, h].double().repeat_interleave(page)[:n]).amax(-1)[:, None] * ref.LARGEST[code]
            bound = want.abs() * torch.finfo(dtype).eps / 2 * 1.01 + spread * (2.0 ** -12 * 1.01 + 2 * err[:, None]) + n * 2.0 ** -25 * peak + torch.finfo(dtype).tiny
            assert bool(((out[cu[r]:cu[r + 1], h].double() - want).abs() <= bound).all()), (r, h)
            assert bool(((lse[cu[r]:cu[r + 1], h].double() - score.logsumexp(-1)).abs() <= err + 2.0 ** -21 * (1 + score.logsumexp(-1).abs())).all()), (r, h)


def test_split_attention_replays_from_a_graph(dev):
    """Lengths, tables and rows change between replays; eager calls with other sizes use workspaces in between."""
    from fla_hip import ops
    gen, rng = torch.Generator().manual_seed(8), random.Random(8)
    page, heads, kv_heads, dim, n, T = 64, 8, 2, 128, 3, 7
    pool, width = 200, -(-WIDE // page)
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    buf = dict(q=torch.zeros(T, heads, dim, dtype=BF, device=dev), table=torch.zeros(n, width, dtype=torch.int32, device=dev),
               lens=torch.ones(n, dtype=torch.int32, device=dev), cu=torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=dev))
    call = lambda: ops.paged_kv_attention(buf["q"], kc, vc, ks, vs, buf["table"], buf["lens"], buf["cu"], max_query_len=4, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:                                             # two graphs of the same call, replayed in turn
        with torch.cuda.graph(g):
            outs.append(call())
    for trial in range(4):
        lens = [rng.choice([1, 70, 3000, 4900]) for _ in range(n)]
        cu = [0, 1, 1 + trial, 4 + trial - (trial > 2)]
        table = make_table(rng, lens, page, width, pool)
        lens = [max(m, b - a) for m, a, b in zip(lens, cu, cu[1:])]
        q = torch.randn(T, heads, dim, generator=gen).to(BF)
        for name, v in (("q", q), ("table", table), ("lens", torch.tensor(lens)), ("cu", torch.tensor(cu))):
            buf[name].copy_(v)
        eager = [t.clone() for t in call()]
        ops.paged_kv_attention(buf["q"][:n], kc, vc, ks, vs, buf["table"], buf["lens"])
        torch.cuda.synchronize()
        for g, out in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1]), trial
        check_attention(dev, q[:cu[-1]], (kc, vc, ks, vs), table, lens, cu, dim ** -0.5, got=tuple(t[:cu[-1]] for t in eager))


def test_append_of_many_rows(dev):
    """Workgroups that look for first rows among 32: runs that begin and end anywhere, pages longer than what a wave sees at
    once, skipped rows, a run as long as its page, the last row alone."""
    from fla_hip import ops
    rng, gen = random.Random(2), torch.Generator().manual_seed(2)
    page, heads, dim, pool = 128, 8, 64, 700
    ids, slots = list(range(pool)), []
    rng.shuffle(ids)
    while len(slots) < 33000 and ids:
        if rng.random() < 0.1:
            slots += [-1] * rng.randint(1, 40)
            continue
        off = rng.choice([0, 0, 1, rng.randint(0, page - 1)])
        n = rng.choice([1, 2, page - off, page - off, rng.randint(1, page - off)])
        slots += range(ids[-1] * page + off, ids.pop() * page + off + n)
    assert len(slots) * heads * 2 >= 8192 * 32
    kc, ks = random_cache(gen, pool, heads, page, dim, INT8, dev)
    vc, vs = random_cache(gen, pool, heads, page, dim, INT8, dev)
    x = torch.randn(len(slots), heads, dim, generator=gen).to(BF)
    want, scale = codes_of(kc), ks.cpu().double()
    ops.paged_kv_append(x.to(dev), x.flip(0).to(dev), kc, vc, ks, vs, torch.tensor(slots, device=dev))
    ref.append(x, want, scale, slots, INT8)
    assert torch.equal(ks.cpu().double(), scale) and torch.equal(codes_of(kc), want)


# ---- together --------------------------------------------------------------------------------------------------------

def serve(dev, steps, code, capture, side_stream=False):
    """A batch served for several steps: plan, rotary, append, attention; every step against the restatement."""
    from fla_hip import ops
    gen, rng = torch.Generator().manual_seed(11), random.Random(11)
    page, heads, kv_heads, dim, pool, n, width, T = 16, 8, 2, 64, 64, 4, 10, steps[0][1]
    new = lambda: torch.zeros(pool, kv_heads, page, dim, dtype=torch.uint8, device=dev).view(code)
    kc, vc, ks, vs = new(), new(), torch.zeros(pool, kv_heads, device=dev), torch.zeros(pool, kv_heads, device=dev)
    table = torch.full((n, width), -1, dtype=torch.int32, device=dev)
    ids = list(range(pool))
    rng.shuffle(ids)
    inv = (10000.0 ** (-torch.arange(16) / 16)).to(dev)
    buf = dict(context=torch.zeros(n, dtype=torch.int32, device=dev), query=torch.zeros(n, dtype=torch.int32, device=dev),
               free=torch.zeros(16, dtype=torch.int32, device=dev), q=torch.zeros(T, heads, dim, dtype=BF, device=dev),
               k=torch.zeros(T, kv_heads, dim, dtype=BF, device=dev), v=torch.zeros(T, kv_heads, dim, dtype=BF, device=dev))

    def step():
        slots, pos, cu, seq, used, _ = ops.paged_kv_plan(buf["context"], buf["query"], table, buf["free"], page, T)
        q, k = ops.rotary_axes(buf["q"], buf["k"], pos[None].expand(2, -1), inv, (8, 8), axis_order="interleaved")
        ops.paged_kv_append(k, buf["v"], kc, vc, ks, vs, slots)
        return q, k, slots, cu, seq, used, ops.paged_kv_attention(q, kc, vc, ks, vs, table, seq, cu, max_query_len=T, return_lse=True)

    graph = None
    if capture:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static = step()
        for t in (kc, vc):
            t.view(torch.uint8).zero_()
        ks.zero_()
        vs.zero_()
        table.fill_(-1)
    context, at = [0] * n, 0
    ref_table = [[-1] * width for _ in range(n)]
    state = [torch.zeros(pool, kv_heads, page, dim, dtype=torch.float64) for _ in range(2)] + [torch.zeros(pool, kv_heads, dtype=torch.float64) for _ in range(2)]
    for query, tokens in steps:
        assert tokens == T
        free = ids[at:at + 16]
        buf["context"].copy_(torch.tensor(context))
        buf["query"].copy_(torch.tensor(query))
        buf["free"][:len(free)] = torch.tensor(free, dtype=torch.int32, device=dev)
        for name in "qkv":
            buf[name].copy_(torch.randn(buf[name].shape, generator=gen) * (1 + sum(context)))
        if side_stream:
            stream = torch.cuda.Stream()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                q, k, slots, cu, seq, used, got = step()
            torch.cuda.current_stream().wait_stream(stream)
        elif graph is not None:
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            q, k, slots, cu, seq, used, got = static
        else:
            q, k, slots, cu, seq, used, got = step()
        want = ref.plan(context, query, ref_table, free, page, T)
        assert torch.equal(slots.cpu(), want["slots"]) and torch.equal(table.cpu(), want["table"]) and torch.equal(used.cpu(), want["used"])
        total = sum(query)
        ref.append(k.cpu(), state[0], state[2], want["slots"], code)
        ref.append(buf["v"].cpu(), state[1], state[3], want["slots"], code)
        assert torch.equal(ks.cpu().double(), state[2]) and torch.equal(vs.cpu().double(), state[3])
        assert torch.equal(codes_of(kc), state[0]) and torch.equal(codes_of(vc), state[1])
        out, lse = (t[:total] for t in got)
        assert bool((got[0][total:] == 0).all())
        check_attention(dev, q[:total].cpu(), (kc, vc, ks, vs), table.cpu(), seq.tolist(), cu.tolist(), dim ** -0.5, got=(out, lse))
        context = [c + m for c, m in zip(context, query)]
        at += int(used)


PREFILL = [([17, 5, 0, 10], 32)]
STEPS = [([3, 1, 20, 1], 32), ([1, 1, 1, 1], 32), ([0, 16, 1, 2], 32), ([1, 0, 1, 30], 32)]


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("way", ["eager", "graph", "stream"])
def test_plan_rotary_append_attention_together(dev, code, way):
    serve(dev, PREFILL + STEPS, code, way == "graph", way == "stream")


def test_plan_feeds_the_recurrent_operator(dev):
    """The plan's state rows and lengths drive recurrent_gated_delta_rule on its state pool, as one step of a hybrid stack."""
    from fla_hip import ops
    import torch.nn.functional as F
    gen = torch.Generator().manual_seed(2)
    lens, D, H, rows = [2, 1, 3], 64, 2, [4, 0, 6]
    T = sum(lens)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    with_lead = i32([0] + lens)                 # the recurrent operator's lengths; the plan takes the same buffer without the lead
    *_, states = ops.paged_kv_plan(i32([5, 0, 9]), with_lead[1:], torch.full((3, 2), -1, dtype=torch.int32, device=dev), i32([1, 2, 3, 4]), 16, T, state_rows=i32(rows))
    assert states.tolist() == [r for r, n in zip(rows, lens) for _ in range(n)]
    rn = lambda *s: torch.randn(*s, generator=gen)
    q, k, v = (F.normalize(rn(T, H, D), dim=-1).to(BF).to(dev) for _ in range(3))
    beta, g = torch.sigmoid(rn(T, H)).to(BF).to(dev), F.logsigmoid(rn(T, H)).to(dev)
    pool = (rn(8, H, D, D) * 0.01).to(dev)
    expect_pool = pool.clone()
    kw = dict(beta=beta, scale=D ** -0.5, actual_seq_lengths=with_lead, g=g)
    o = ops.recurrent_gated_delta_rule(q, k, v, pool, ssm_state_indices=states, **kw)
    e = ops.recurrent_gated_delta_rule(q, k, v, expect_pool, ssm_state_indices=i32([4, 4, 0, 6, 6, 6]), **kw)
    assert torch.equal(o, e) and torch.equal(pool, expect_pool)


def test_refusals_of_gradients_and_cpu_tensors(dev):
    from fla_hip import ops
    gen = torch.Generator().manual_seed(0)
    kc, ks = random_cache(gen, 4, 1, 16, 64, E4M3, dev)
    q = torch.randn(1, 2, 64, device=dev, dtype=BF, requires_grad=True)
    table, lens = torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    with pytest.raises(NotImplementedError, match="no gradient is bound for query"):
        ops.paged_kv_attention(q, kc, kc, ks, ks, table, lens)
    with torch.no_grad():
        ops.paged_kv_attention(q, kc, kc, ks, ks, table, lens)
    with torch.inference_mode():
        ops.paged_kv_attention(q, kc, kc, ks, ks, table, lens, out=torch.empty(1, 2, 64, device=dev, dtype=BF))
    with pytest.raises(TypeError, match="key_cache must be a ROCm GPU tensor"):
        ops.paged_kv_attention(q.detach(), kc.cpu(), kc, ks, ks, table, lens)


def test_plan_without_tokens_keeps_its_state_rows_apart(dev):
    from fla_hip import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    table = torch.full((2, 2), -1, dtype=torch.int32, device=dev)
    slots, pos, cu, seq, used, states = ops.paged_kv_plan(i32([4, 0]), i32([0, 3]), table, i32([7]), 16, 0, state_rows=i32([1, 0]))
    assert slots.numel() == pos.numel() == states.numel() == 0 and states.dtype == torch.int32
    assert cu.tolist() == [0, 0, 3] and seq.tolist() == [4, 3] and used.tolist() == [1] and table.tolist() == [[-1, -1], [7, -1]]


@pytest.mark.parametrize("new", [2, 40])
def test_rows_before_the_first_request(dev, new):
    from fla_hip import ops
    rng, gen = random.Random(3), torch.Generator().manual_seed(3)
    page, heads, kv_heads, dim, lens = 16, 4, 2, 64, [50, 43]
    cu = [3, 3 + new, 3 + 2 * new]
    kc, ks = random_cache(gen, 9, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, 9, kv_heads, page, dim, E4M3, dev)
    table = make_table(rng, lens, page, 4, 9)
    q = torch.randn(cu[-1] + 2, heads, dim, generator=gen).to(BF)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    args = (q.to(dev), kc, vc, ks, vs, table.to(dev), i32(lens), i32(cu))
    torch.empty(1 << 20, dtype=BF, device=dev).fill_(7.0)             # what a new result may find in its memory
    out, lse = ops.paged_kv_attention(*args, max_query_len=new, return_lse=True)
    for rows in (slice(0, 3), slice(cu[-1], None)):
        assert bool((out[rows] == 0).all()) and bool((lse[rows] == -math.inf).all())
    mine = slice(3, cu[-1])
    check_attention(dev, q[mine], (kc, vc, ks, vs), table, lens, [c - 3 for c in cu], dim ** -0.5, got=(out[mine], lse[mine]))
    given = torch.full_like(q, 3.0).to(dev)
    ops.paged_kv_attention(*args, out=given, max_query_len=new)
    assert torch.equal(given[mine], out[mine]) and bool((given[:3] == 3).all()) and bool((given[cu[-1]:] == 3).all())


@pytest.mark.parametrize("adjacent", [False, True])
def test_rotary_gradient_has_a_gradient(dev, adjacent):
    """The operator is linear, so the gradient of <u, dq(w)> in w is the operator itself applied to u: the same kernel on the
    same numbers, equal to the bit."""
    from fla_hip import ops
    gen = torch.Generator().manual_seed(8)
    q, w, u = (torch.randn(9, 3, 16, generator=gen).to(dev) for _ in range(3))
    k, wk, uk = (torch.randn(9, 1, 16, generator=gen).to(dev) for _ in range(3))
    pos, freq = torch.arange(9, device=dev)[None], torch.rand(6, generator=gen).to(dev)
    how = dict(pairing="adjacent" if adjacent else "half")
    q.requires_grad_(), k.requires_grad_(), w.requires_grad_(), wk.requires_grad_()
    grads = torch.autograd.grad(ops.rotary_axes(q, k, pos, freq, (6,), **how), (q, k), (w, wk), create_graph=True)
    again = torch.autograd.grad(grads, (w, wk), (u, uk))
    with torch.no_grad():
        want = ops.rotary_axes(u, uk, pos, freq, (6,), **how)
        back = ops.rotary_axes_bwd(w, wk, pos, freq, (6,), **how)
    assert all(torch.equal(a, b) for a, b in zip(grads, back)) and all(torch.equal(a, b) for a, b in zip(again, want))
    only = torch.autograd.grad(ops.rotary_axes(q, k, pos, freq, (6,), **how)[1], k, wk, create_graph=True)[0]
    assert torch.equal(torch.autograd.grad(only, wk, uk)[0], want[1])


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("new,kept", [(4, 2), (7, 9), (70, 33), (90, 100)])
def test_requests_that_the_batch_cuts_off(dev, new, kept, wide):
    """cu_seqlens past the rows of the query: a row keeps its place in its request, so it is as if the request were shorter by
    the rows that are not there."""
    from fla_hip import ops
    rng, gen = random.Random(new), torch.Generator().manual_seed(new)
    page, heads, kv_heads, dim, lens = 16, 8, 2, 64, [new + 40, new + 6, new + 300, new]
    cu, rows = [new * r for r in range(5)], new + kept
    kc, ks = random_cache(gen, 80, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, 80, kv_heads, page, dim, E4M3, dev)
    table = make_table(rng, lens, page, max(-(-n // page) for n in lens), 80)
    q = torch.randn(rows, heads, dim, generator=gen).to(BF)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    given = (widen(table, page) if wide else table).to(dev)
    got = ops.paged_kv_attention(q.to(dev), kc, vc, ks, vs, given, i32(lens), i32(cu), max_query_len=new, return_lse=True)
    cut = [min(c, rows) for c in cu]
    short = [n - (new - (b - a)) for n, a, b in zip(lens, cut, cut[1:])]
    check_attention(dev, q, (kc, vc, ks, vs), table, short, cut, dim ** -0.5, got=got)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("new,tokens", [(4, 6), (60, 100)])
def test_a_step_with_fewer_rows_than_tokens(dev, new, tokens, wide):
    """Plan, append and attention of a step whose batch ends inside a request: what is not appended (NaN here) is not seen."""
    from fla_hip import ops
    gen = torch.Generator().manual_seed(tokens)
    page, heads, kv_heads, dim, n = 16, 4, 1, 64, 3
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    kc, vc = (torch.full((40, kv_heads, page, dim), 0x7f, dtype=torch.uint8, device=dev).view(E4M3) for _ in range(2))
    ks, vs = torch.zeros(40, kv_heads, device=dev), torch.zeros(40, kv_heads, device=dev)
    table = torch.full((n, 400 if wide else 12), -1, dtype=torch.int32, device=dev)
    slots, _, cu, seq, _, _ = ops.paged_kv_plan(i32([0] * n), i32([new] * n), table, i32(list(range(39, 9, -1))), page, tokens)
    q, k, v = (torch.randn(tokens, h, dim, generator=gen).to(BF) for h in (heads, kv_heads, kv_heads))
    ops.paged_kv_append(k.to(dev), v.to(dev), kc, vc, ks, vs, slots)
    got = ops.paged_kv_attention(q.to(dev), kc, vc, ks, vs, table, seq, cu, max_query_len=new, return_lse=True)
    cut = [min(c, tokens) for c in cu.tolist()]
    check_attention(dev, q, (kc, vc, ks, vs), table.cpu(), [b - a for a, b in zip(cut, cut[1:])], cut, dim ** -0.5, got=got)


@pytest.mark.parametrize("gap", [14.0, 17.0, 18.0, 20.0])
@pytest.mark.parametrize("rows,heads,n", [(2340, 64, 4096), (40, 4, 250), (1, 4, 1500)])
def test_a_first_token_that_draws_the_weight_and_holds_no_values(dev, rows, heads, n, gap):
    """The first key of a text stands ``gap`` nats above the others and its values are 0, so the result is what the light weights
    add up to.  A weight is fp16 with the largest contribution at 2^10 or more: one below 2^-14 is off by at most 2^-25, so
    2^-35 of the largest contribution, times its code.  In float64 on the GPU, some heads."""
    from fla_hip import ops
    gen = torch.Generator().manual_seed(int(gap))
    page, dim = 64, 64
    pool = -(-n // page)
    k = torch.randn(pool, heads, page, dim, generator=gen) * 0.25
    k[..., 0] = 0
    k[0, :, 0] = 0
    k[0, :, 0, 0] = 16.0
    v = torch.rand(pool, heads, page, dim, generator=gen) * 3 + 1
    v[0, :, 0] = 0
    kc, vc = k.to(E4M3).to(dev), v.to(E4M3).to(dev)
    ones = torch.ones(pool, heads, device=dev)
    q = torch.randn(rows, heads, dim, generator=gen) * 0.5
    scale = 0.125
    q[..., 0] = gap / 16 / scale
    q = q.to(BF).to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    out, lse = ops.paged_kv_attention(q, kc, vc, ones, ones, torch.arange(pool, device=dev, dtype=torch.int32)[None], i32([n]), i32([0, rows]),
                                      scale=scale, max_query_len=rows, return_lse=True)
    seen = torch.arange(n, device=dev) <= torch.arange(n - rows, n, device=dev)[:, None]
    for h in range(0, heads, max(1, heads // 4)):
        kd, vd = (c.view(torch.uint8)[:, h].view(E4M3).float().double().flatten(0, 1)[:n] for c in (kc, vc))
        x = q[:, h].double()
        score = torch.where(seen, (x @ kd.t()) * scale, -math.inf)
        p = torch.softmax(score, -1)
        want = p @ vd
        err = (dim + 8) * 2.0 ** -24 * ((x.abs() @ kd.abs().t()) * scale).amax(-1)[:, None]
        peak = p.amax(-1)[:, None]
        # the result's rounding (8 significant bits: 2^-8 of its value), the weights' (11: 2^-11) and the scores'; codes are at most 4
        bound = want * (torch.finfo(BF).eps / 2 * 1.01 + torch.finfo(F16).eps / 2 * 1.01 + 2 * err) + n * 2.0 ** -35 * peak * 4 + torch.finfo(BF).tiny
        error = (out[:, h].double() - want).abs()
        assert bool((error <= bound).all()), (h, float((error / bound).max()), float((error / want).max()))
        want_lse = score.logsumexp(-1)
        assert bool(((lse[:, h].double() - want_lse).abs() <= err[:, 0] + 2.0 ** -21 * (1 + want_lse.abs())).all())


@pytest.mark.parametrize("code", [E4M3, INT8])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_of_infinities_without_a_finite_value(dev, code, dtype):
    """Pages whose scale is 0: infinities store the largest code all the same, NaN stores NaN (e4m3) or 0 (int8)."""
    from fla_hip import ops
    page, dim, heads = 16, 64, 2
    x = torch.zeros(6, heads, dim, dtype=dtype)
    x[0, 0, 3], x[0, 0, 5], x[1, 1, 7], x[2, 0, 9] = math.inf, -math.inf, math.nan, math.inf
    x[4, 0, 0], x[5, 0, 0] = math.inf, 1.0                               # a finite row later on
    slots = [0, 1, page, 2 * page + 15, 3 * page, 3 * page + 1]
    new = lambda: torch.zeros(5, heads, page, dim, dtype=torch.uint8, device=dev).view(code)
    kc, vc, ks, vs = new(), new(), torch.full((5, heads), 3.0, device=dev), torch.full((5, heads), 3.0, device=dev)
    want, scale = torch.zeros(5, heads, page, dim, dtype=torch.float64), torch.full((5, heads), 3.0, dtype=torch.float64)
    ks[2], scale[2] = 0, 0
    vs[2] = 0
    for part in (slice(0, 5), slice(5, 6)):
        ops.paged_kv_append(x[part].to(dev), -x[part].to(dev), kc, vc, ks, vs, torch.tensor(slots[part], device=dev))
        ref.append(x[part], want, scale, slots[part], code)
        assert torch.equal(ks.cpu().double(), scale) and torch.equal(vs.cpu().double(), scale)
        for cache, sign in ((kc, 1), (vc, -1)):
            got = codes_of(cache) * sign
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


def test_rotary_has_a_tangent(dev):
    """The same kernel on the tangents: equal to the bit, in the gradient as well; expanded tangents among them."""
    from fla_hip import ops
    from torch.autograd import forward_ad as ad
    gen = torch.Generator().manual_seed(4)
    q, tq, w = (torch.randn(9, 3, 16, generator=gen).to(dev) for _ in range(3))
    k, tk = torch.randn(9, 1, 16, generator=gen).to(dev), torch.randn(9, 1, 1, generator=gen).to(dev).expand(9, 1, 16)
    how = torch.arange(9, device=dev)[None], torch.rand(6, generator=gen).to(dev), (6,)
    want = ops.rotary_axes(q, k, *how) + ops.rotary_axes(tq, tk.contiguous(), *how)
    with ad.dual_level():
        leaf = q.clone().requires_grad_()
        for x in (q, leaf):
            y = ops.rotary_axes(ad.make_dual(x, tq), ad.make_dual(k, tk), *how)
            got = [ad.unpack_dual(a) for a in y]
            assert all(torch.equal(a, b) for a, b in zip([g.primal for g in got] + [g.tangent for g in got], want))
        dq = ad.unpack_dual(torch.autograd.grad(y[0], leaf, ad.make_dual(w, tq))[0])
        assert torch.equal(dq.primal, ops.rotary_axes_bwd(w, None, *how)[0]) and torch.equal(dq.tangent, ops.rotary_axes_bwd(tq, None, *how)[0])


@pytest.mark.parametrize("new", [1, 5, 80])
@pytest.mark.parametrize("dim", [64, 128])
def test_negative_scales(dev, new, dim):
    """A stored value is code times scale, whatever the scale's sign; the first page's is negative too."""
    rng, gen = random.Random(new), torch.Generator().manual_seed(new)
    page, heads, kv_heads, lens = 16, 8, 2, [new + 333, new + 40]
    kc, ks = random_cache(gen, 60, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, 60, kv_heads, page, dim, E4M3, dev)
    table = make_table(rng, lens, page, -(-max(lens) // page), 60)
    ks *= torch.where(torch.rand(60, kv_heads, generator=gen) < 0.5, -1.0, 1.0).to(dev)
    vs *= torch.where(torch.rand(60, kv_heads, generator=gen) < 0.5, -1.0, 1.0).to(dev)
    vs[int(table[0, 0])] = -2.0 ** -5
    q = torch.randn(2 * new, heads, dim, generator=gen).to(BF)
    for t in (table, widen(table, page)):
        check_attention(dev, q, (kc, vc, ks, vs), t, lens, [0, new, 2 * new], dim ** -0.5, max_query_len=new)
    vs.fill_(-0.25)
    check_attention(dev, q, (kc, vc, ks, vs), table, lens, [0, new, 2 * new], dim ** -0.5, max_query_len=new)


@pytest.mark.parametrize("code", [E4M3, INT8])
def test_append_behind_a_negative_scale(dev, code):
    """A page written elsewhere with a negative scale: its scale turns positive, its values stay (to one rounding)."""
    from fla_hip import ops
    gen = torch.Generator().manual_seed(1)
    kc, _ = random_cache(gen, 3, 1, 16, 64, code, dev)
    vc, _ = random_cache(gen, 3, 1, 16, 64, code, dev)
    ks, vs = (torch.tensor([[-2.0 ** -5], [-1.0], [-2.0 ** -9]], device=dev) for _ in range(2))
    before = [codes_of(c) * s.cpu().double()[..., None, None] for c, s in ((kc, ks), (vc, vs))]
    x = torch.randn(3, 1, 64, generator=gen).to(BF)
    x[0, 0, 0] = 100.0
    ops.paged_kv_append(x.to(dev), x.to(dev), kc, vc, ks, vs, torch.tensor([7, 16 + 7, 32 + 7], device=dev))
    for c, s, had in ((kc, ks, before[0]), (vc, vs, before[1])):
        assert bool((s > 0).all())
        now = codes_of(c) * s.cpu().double()[..., None, None]
        step = s.cpu().double()[..., None, None] * (0.5 if code == INT8 else 2.0 ** -10)
        assert bool(((now - had)[:, :, :7].abs() <= (step if code == INT8 else torch.maximum(step, had[:, :, :7].abs() * 2.0 ** -4))).all())
        assert bool(((now[:, :, 7] - x.double()).abs() <= torch.maximum(s.cpu().double()[..., None] * (0.5 if code == INT8 else 2.0 ** -10), x.double().abs() * (0 if code == INT8 else 2.0 ** -4))).all())


def test_tables_without_columns(dev):
    """Requests that cannot hold a page: no token has a slot, no row sees anything."""
    from fla_hip import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    gen = torch.Generator().manual_seed(0)
    table = torch.empty(2, 0, dtype=torch.int32, device=dev)
    slots, pos, cu, seq, used, _ = ops.paged_kv_plan(i32([0, 4]), i32([2, 1]), table, i32([5]), 16, 4)
    assert slots.tolist() == [-1] * 4 and pos.tolist() == [0, 1, 4, 0] and cu.tolist() == [0, 2, 3] and seq.tolist() == [2, 5] and used.tolist() == [0]
    kc, ks = random_cache(gen, 4, 1, 16, 64, E4M3, dev)
    for rows in (2, 300):
        q = torch.randn(rows, 4, 64, device=dev).to(BF)
        out, lse = ops.paged_kv_attention(q, kc, kc, ks, ks, table, i32([3, 500]), i32([0, 1, rows]), return_lse=True)
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_strides_of_extents_of_one(dev):
    """One token taken out of a long buffer, one head, one page: the stride of an extent of one leads nowhere and may be anything."""
    from fla_hip import ops
    gen = torch.Generator().manual_seed(0)
    page, heads, dim = 16, 4, 64
    one = lambda x, at: x.as_strided(x.shape, at)
    long = torch.randn(1, (1 << 21) // (heads * dim) + 5, heads, dim, generator=gen).to(BF).to(dev)
    kv = long[:, 7]                                           # [1, heads, dim], 2^21 elements to the next batch entry
    assert kv.stride(0) >= 1 << 21
    kc, ks = random_cache(gen, 1, heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, 1, heads, page, dim, E4M3, dev)
    q = torch.randn(1, heads * 2, dim, generator=gen).to(BF).to(dev)
    slots, table, lens = torch.tensor([3], device=dev), torch.zeros(1, 1, dtype=torch.int32, device=dev), torch.tensor([4], dtype=torch.int32, device=dev)
    plain = [clone_strided(kc), clone_strided(vc), ks.clone(), vs.clone()]
    ops.paged_kv_append(kv.contiguous(), kv.contiguous(), *plain, slots)
    want = ops.paged_kv_attention(q, *plain, table, lens)
    odd = [one(c, (7, page * dim, dim, 1)) for c in (kc, vc)]
    odd += [one(s, (0, 1)) for s in (ks, vs)]
    ops.paged_kv_append(kv, kv, *odd, slots)
    got = ops.paged_kv_attention(one(q, (3, dim, 1)), *odd, table, lens, out=one(torch.empty_like(q), (5, dim, 1)))
    assert torch.equal(got, want) and torch.equal(codes_of(kc), codes_of(plain[0])) and torch.equal(ks, plain[2])
    flat = torch.randn(page, dim, generator=gen)
    single = torch.zeros(6, 1, page, dim, dtype=torch.uint8, device=dev).view(E4M3)
    s1 = torch.ones(6, 1, device=dev)
    single.view(torch.uint8).copy_(flat.to(E4M3).view(torch.uint8).to(dev))
    a = ops.paged_kv_attention(q, single, single, s1, s1, table + 2, lens)
    b = ops.paged_kv_attention(q, one(single, (page * dim, 1, dim, 1)), one(single, (page * dim, 3, dim, 1)), s1, s1, table + 2, lens)
    assert torch.equal(a, b)


def test_rotary_gradient_replays_from_a_graph(dev):
    """Forward and gradient captured together; inputs, positions and gradients change between replays, eager calls run in between."""
    from fla_hip import ops
    gen = torch.Generator().manual_seed(6)
    rn = lambda *s: torch.randn(*s, generator=gen).to(BF)
    q, k = rn(40, 4, 64).to(dev).requires_grad_(), rn(40, 2, 64).to(dev).requires_grad_()
    dq, dk, pos = rn(40, 4, 64).to(dev), rn(40, 2, 64).to(dev), torch.arange(40, device=dev)[None].contiguous()
    freq = torch.rand(32, generator=gen).to(dev)

    def both(a, b):
        y = ops.rotary_axes(a, b, pos, freq, (32,))
        return [t.detach() for t in y] + list(torch.autograd.grad(y, (a, b), (dq, dk)))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both(q, k)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = both(q, k)
    for _ in range(4):
        with torch.no_grad():
            for t in (q, k, dq, dk):
                t.copy_(rn(*t.shape))
            pos.copy_(torch.randint(0, 1 << 20, pos.shape, generator=gen))
        eager = both(q.detach().clone().requires_grad_(), k.detach().clone().requires_grad_())
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, eager))


def test_split_attention_on_two_streams_at_once(dev):
    """Calls that are joined through workspaces run side by side; each has its own."""
    from fla_hip import ops
    rng, gen = random.Random(2), torch.Generator().manual_seed(2)
    page, heads, kv_heads, dim, lens = 64, 8, 2, 128, [4000, 2500, 70]
    kc, ks = random_cache(gen, 120, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, 120, kv_heads, page, dim, E4M3, dev)
    table, seq = make_table(rng, lens, page, 80, 120).to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)
    qs = [torch.randn(3, heads, dim, generator=gen).to(BF).to(dev) for _ in range(2)]
    want = [ops.paged_kv_attention(q, kc, vc, ks, vs, table, seq, return_lse=True) for q in qs]
    streams, got = [torch.cuda.Stream() for _ in qs], []
    torch.cuda.synchronize()
    for _ in range(8):
        for q, s in zip(qs, streams):
            with torch.cuda.stream(s):
                got.append(ops.paged_kv_attention(q, kc, vc, ks, vs, table, seq, return_lse=True))
    torch.cuda.synchronize()
    for i, (out, lse) in enumerate(got):
        assert torch.equal(out, want[i % 2][0]) and torch.equal(lse, want[i % 2][1])


@pytest.mark.parametrize("new", [1, 3, 80])
def test_log_sums_beside_pages_with_a_scale_of_zero(dev, new):
    """Values of 0 do not enter the sum of the softmax.  Many small texts.  Bound: the scores' error, (D + 8) * 2^-24 of sum |q||k| * scale,
    and 2^-21 of 1 + |lse| (exponents up to 16 are rounded by 2^-21, times ln 2; the sums and the logarithm by less)."""
    from fla_hip import ops
    rng, gen = random.Random(new), torch.Generator().manual_seed(new)
    page, heads, kv_heads, dim, n = 16, 12, 3, 64, 60 if new < 80 else 6
    lens = [new + rng.choice([0, 1, 2, 9, 40]) for _ in range(n)]
    pool = sum(-(-m // page) for m in lens) + 2
    kc, ks = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    vc, vs = random_cache(gen, pool, kv_heads, page, dim, E4M3, dev)
    table = make_table(rng, lens, page, -(-max(lens) // page), pool)
    q = torch.randn(n * new, heads, dim, generator=gen).to(F16)
    cu = [new * r for r in range(n + 1)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    _, want, _, reach, _ = ref.attention(q, codes_of(kc), codes_of(vc), ks.cpu(), vs.cpu(), table, lens, cu, -0.1)
    for zero in (slice(0, None, 2), slice(None)):
        vs[zero] = 0
        for t in (table, widen(table, page)):
            _, lse = ops.paged_kv_attention(q.to(dev), kc, vc, ks, vs, t.to(dev), i32(lens), i32(cu), scale=-0.1, max_query_len=new, return_lse=True)
            error, bound = (lse.cpu().double() - want).abs(), (dim + 8) * 2.0 ** -24 * reach + 2.0 ** -21 * (1 + want.abs())
            assert bool((error <= bound).all()), (float((error / bound).max()), float(error.max()))
