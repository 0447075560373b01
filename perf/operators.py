"""Serving path of the softmax-attention layers that stand between linear-attention layers: page plan, rotary
positions, 8-bit cache append and the attention that reads the cache.

``listed()`` names the measured cases, ``draw()`` makes more of the same ranges, ``run()`` is one pass in plain torch
operations (``own`` false) or through ``fla_hip.ops`` (``own`` true), ``exact()`` the same outputs in 64 bits.
"""
import math
import os
import random
import sys

import torch

own = False

E4M3_MOST, INT8_MOST = 448.0, 127.0
SMALLEST = 2.0 ** -126  # smallest normal fp32: the lowest scale of a page that holds anything but zeros


def _ops():
    root = os.path.join(os.getcwd(), "flash-linear-attention-npu_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from fla_hip import ops

    return ops


def listed():
    return [
        # one decode step of a full serving batch: every request adds one token, few need a new page
        dict(name="plan_decode_256", op="plan", requests=256, most_context=8192, most_query=1, lens=1, page=64),
        # a packed prefill batch (64 requests, about 142 k tokens, as the varlen prefill benchmark), small pages
        dict(name="plan_prefill_64", op="plan", requests=64, most_context=0, most_query=4400, lens=2, page=16),
        # one decode step of the batch: every token of q and k gets its (time, height, width) angle
        dict(name="rotary_decode_256", op="rotary", tokens=256, heads=32, kv_heads=8, dim=128, rotated=128, axes=3,
             interleaved=True, adjacent=False, dtype="bfloat16", train=False, far=1 << 20),
        # training forward and gradient of an image / text batch at 4 x 8192 tokens, rotation of half of the channels
        dict(name="rotary_train_32768", op="rotary", tokens=32768, heads=32, kv_heads=8, dim=128, rotated=64, axes=3,
             interleaved=False, adjacent=False, dtype="bfloat16", train=True, far=32768),
        # one decode step of the batch: one row for each request and head into pages that are partly full
        dict(name="append_decode_256", op="append", requests=256, most_context=8192, most_query=1, lens=1, page=64,
             kv_heads=8, dim=128, dtype="bfloat16", cache="e4m3"),
        # packed prefill: whole pages written at once
        dict(name="append_prefill_64", op="append", requests=64, most_context=0, most_query=4400, lens=2, page=64,
             kv_heads=8, dim=128, dtype="bfloat16", cache="e4m3"),
        # second chunk of a chunked prefill with odd lengths: pages that begin and end inside a chunk, int8 codes
        dict(name="append_chunk_odd", op="append", requests=9, most_context=700, most_query=1501, lens=3, page=16,
             kv_heads=4, dim=64, dtype="float16", cache="int8"),
        # a few interactive requests: latency counts
        dict(name="decode_small", op="attention", requests=4, most_context=1100, most_query=1, lens=4, page=64, heads=32,
             kv_heads=8, dim=128, dtype="bfloat16", cache="e4m3"),
        # a serving batch of ragged contexts
        dict(name="decode_ragged_128", op="attention", requests=128, most_context=8192, most_query=1, lens=5, page=64,
             heads=32, kv_heads=8, dim=128, dtype="bfloat16", cache="e4m3"),
        # one request with a very long document
        dict(name="decode_long", op="attention", requests=1, most_context=262147, most_query=1, lens=0, page=64, heads=32,
             kv_heads=8, dim=128, dtype="bfloat16", cache="int8"),
        # checking speculated tokens: one to seven query tokens for each request, small pages and heads
        dict(name="verify_ragged_48", op="attention", requests=48, most_context=5003, most_query=7, lens=6, page=16, heads=24,
             kv_heads=4, dim=64, dtype="float16", cache="e4m3"),
        # chunked prefill: a chunk of 4096 tokens for each of two requests behind what is cached already
        dict(name="prefill_chunk_2x4096", op="attention", requests=2, most_context=4096, most_query=4096, lens=0, page=64,
             heads=32, kv_heads=8, dim=128, dtype="bfloat16", cache="e4m3"),
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["plan", "rotary", "append", "attention", "attention"])
    page = rng.choice([16, 32, 64, 128])
    lens = rng.randrange(1, 1 << 20)
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    cache = rng.choice(["e4m3", "e4m3", "int8"])
    if op == "rotary":
        rotated = rng.choice([32, 64, 128])
        dim, kind = rng.choice([d for d in (64, 128, 256) if d >= rotated]), rng.choice(["bfloat16", "float16", "float32"])
        most = 32768 * 128 // max(dim, 128) // (2 if kind == "float32" else 1)
        return dict(op=op, tokens=_spread(rng, 1, most), heads=rng.choice([4, 14, 16, 32]), kv_heads=rng.choice([1, 2, 4, 8]), dim=dim,
                    rotated=rotated, axes=rng.choice([1, 2, 3]), interleaved=rng.random() < 0.5, adjacent=rng.random() < 0.5,
                    dtype=kind, train=rng.random() < 0.5, far=_spread(rng, 100, 1 << 20))
    if op in ("plan", "append"):
        long = rng.random() < 0.6  # prefill rather than decode
        requests = _spread(rng, 1, 64) if long else _spread(rng, 1, 256)
        case = dict(op=op, requests=requests, most_context=_spread(rng, 1, 8192) if not long else rng.choice([0, _spread(rng, 1, 2000)]),
                    most_query=_spread(rng, 2, 4400) if long else 1, lens=lens, page=page)
        if op == "append":
            case |= dict(kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128, 256]) if requests <= 32 else 64, dtype=dtype, cache=cache)
        return case
    kind = rng.choice(["decode", "decode", "verify", "prefill"])
    dim = rng.choice([64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8] if dim < 256 else [1, 2, 4])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 6, 8] if dim < 256 else [2, 4, 8])
    if kind == "prefill":
        requests = rng.choice([1, 2, 3])
        return dict(op=op, requests=requests, most_context=_spread(rng, 1, 4096 if requests < 3 else 1500),
                    most_query=_spread(rng, 64, 4096 if requests < 3 else 1500),
                    lens=rng.choice([0, lens]), page=page, heads=min(heads, 32 if dim < 256 else 16), kv_heads=kv_heads, dim=dim, dtype=dtype, cache=cache)
    if rng.random() < 0.3:
        requests, context = rng.choice([1, 2]), _spread(rng, 4096, 65536)
    else:
        requests, context = _spread(rng, 1, 64), _spread(rng, 1, 8192)
    return dict(op=op, requests=requests, most_context=context, most_query=1 if kind == "decode" else rng.choice([2, 3, 4, 6, 8]),
                lens=lens, page=page, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, cache=cache)


def _lengths(case):
    """(cached tokens, new tokens) of each request: the largest for all where ``lens`` is 0, else ragged, the first ones
    of the smallest and largest lengths."""
    n, c, q = case["requests"], case["most_context"], case["most_query"]
    if case["lens"] == 0:
        return [c] * n, [q] * n
    rng = random.Random(case["lens"])
    context = [rng.randint(0, c) for _ in range(n)]
    query = [rng.randint(1, q) if q < 64 else rng.randint(q // 64, q) for _ in range(n)]
    context[0] = c
    return context, query


def _sections(case):
    half, axes = case["rotated"] // 2, case["axes"]
    rest = half // axes if axes > 1 else 0
    return [half - rest * (axes - 1)] + [rest] * (axes - 1)


def _axis_of(case):
    """Which axis each frequency turns with: contiguous sections, or the axes in turn while they have any left."""
    left = _sections(case)
    if not case["interleaved"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    got = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                left[a] -= 1
                got.append(a)
    return got


def _dtype(case):
    return getattr(torch, case["dtype"])


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _pages(total, page):
    return -(-total // page)


def _table(case, lens, g):
    """Block table over a pool in random order; entries past a request's pages are -1."""
    counts = [_pages(n, case["page"]) for n in lens]
    width = max(max(counts), 1)
    order = torch.randperm(sum(counts) + 3, generator=g, device="cuda").int()
    count = torch.tensor(counts, device="cuda")
    base = count.cumsum(0) - count
    col = torch.arange(width, device="cuda")
    table = torch.where(col < count[:, None], order[(base[:, None] + col).clamp(max=order.numel() - 1)], -1)
    return table.int(), order, sum(counts)


def _codes(shape, cache, g):
    x = torch.empty(shape, device="cuda", dtype=torch.float16).normal_(generator=g)
    if cache == "int8":
        return (x * 31).round_().clamp_(-127, 127).to(torch.int8)
    return (x * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "rotary":
        t, d, dt = case["tokens"], case["dim"], _dtype(case)
        new = lambda h: torch.randn(t, h, d, generator=g, device="cuda").to(dt)  # noqa: E731
        half = case["rotated"] // 2
        s = dict(case=case, q=new(case["heads"]), k=new(case["kv_heads"]),
                 positions=torch.randint(0, case["far"], (case["axes"], t), generator=g, device="cuda"),
                 inv_freq=(10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda(),
                 sections=_sections(case), axis_of=torch.tensor(_axis_of(case), device="cuda"))
        if case["train"]:
            s |= dict(dq=new(case["heads"]), dk=new(case["kv_heads"]))
            s["q"].requires_grad_()
            s["k"].requires_grad_()
        return s
    context, query = _lengths(case)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = dict(case=case, page=case["page"])
    total = [a + b for a, b in zip(context, query)]
    tokens = sum(query)
    if op == "plan":
        table, order, used = _table(case, context, g)
        width = max(max(_pages(n, case["page"]) for n in total), 1)
        full = torch.full((len(total), width), -1, dtype=torch.int32, device="cuda")
        full[:, :min(width, table.shape[1])] = table[:, :width]
        extra = sum(_pages(n, case["page"]) for n in total) - used + 16
        free = (torch.randperm(extra, generator=g, device="cuda") + order.numel()).int()
        return s | dict(context=ints(context), query=ints(query), table=full, free=free, tokens=tokens + 5,
                        rows=torch.randperm(len(total), generator=g, device="cuda").int())
    table, order, _ = _table(case, total, g)
    pool, h, d = order.numel(), case["kv_heads"], case["dim"]
    cu = ints([0] + torch.tensor(query).cumsum(0).tolist())
    s |= dict(kc=_codes((pool, h, case["page"], d), case["cache"], g), vc=_codes((pool, h, case["page"], d), case["cache"], g))
    steps = torch.tensor([2.0 ** -8, 2.0 ** -7, 2.0 ** -6] if case["cache"] == "e4m3" else [2.0 ** -6, 2.0 ** -5, 2.0 ** -4], device="cuda")
    pick = lambda: steps[torch.randint(0, 3, (pool, h), generator=g, device="cuda")]  # noqa: E731
    s |= dict(ks=pick(), vs=pick())
    dt = _dtype(case)
    if op == "append":
        rows = torch.repeat_interleave(torch.arange(len(total), device="cuda"), cu.diff().long())
        pos = torch.arange(tokens, device="cuda") - cu[rows].long() + torch.tensor(context, device="cuda")[rows]
        slots = table[rows, pos // case["page"]].long() * case["page"] + pos % case["page"]
        # a row's size changes along the text, so that some pages need a larger scale than they have
        size = torch.exp(torch.randn(tokens, 1, 1, generator=g, device="cuda") * 0.7)
        new = lambda: (torch.randn(tokens, h, d, generator=g, device="cuda") * size).to(dt)  # noqa: E731
        return s | dict(k=new(), v=new(), slots=slots, runs=min(tokens, tokens // case["page"] + 2 * len(total)))
    q = torch.randn(tokens, case["heads"], d, generator=g, device="cuda").to(dt)
    return s | dict(q=q, table=table, lens=ints(total), cu=None if case["most_query"] == 1 else cu, cu_plain=cu, scale=d ** -0.5,
                    most_query=max(query), most_len=max(total))


# ---- plain forms --------------------------------------------------------------------------------------------------

def _plan(s):
    page, table, free = s["page"], s["table"], s["free"]
    ctx, new = s["context"].long(), s["query"].long()
    n, width = table.shape
    total, end = ctx + new, new.cumsum(0)
    start = end - new
    old = ((ctx + page - 1) // page).clamp(max=width)
    need = ((total + page - 1) // page).clamp(max=width) - old
    base = need.cumsum(0) - need
    col = torch.arange(width, device="cuda")
    at = base[:, None] + col - old[:, None]
    given = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where((col >= old[:, None]) & (col < (old + need)[:, None]), given, table))
    t = torch.arange(s["tokens"], device="cuda")
    row = torch.searchsorted(end, t, right=True).clamp(max=n - 1)
    held = t < end[-1]
    pos = torch.where(held, ctx[row] + t - start[row], 0)
    block = table[row, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where(held & (block >= 0) & (pos < width * page), block * page + pos % page, -1)
    cu = torch.cat([end.new_zeros(1), end]).int()
    return slots, pos.int(), cu, total.int(), need.sum(0, keepdim=True).int(), torch.where(held, s["rows"][row], -1).int(), table


def _turn(x, cos, sin, adjacent):
    half = cos.shape[-1]
    y = x.float()
    if adjacent:
        a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = y[..., :half], y[..., half:2 * half]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1).to(x.dtype)


def _rotary(s):
    angle = s["positions"].double()[s["axis_of"]].t() * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    adjacent = s["case"]["adjacent"]
    got = _turn(s["q"].detach(), cos, sin, adjacent), _turn(s["k"].detach(), cos, sin, adjacent)
    if s["case"]["train"]:
        got += _turn(s["dq"], cos, -sin, adjacent), _turn(s["dk"], cos, -sin, adjacent)
    return got


def _append_one(x, cache, scales, slots, runs):
    """The tokens of one page follow each other: a run. ``runs`` is the most there can be."""
    h, page, d = cache.shape[1:]
    most = INT8_MOST if cache.dtype == torch.int8 else E4M3_MOST
    block, off = slots // page, slots % page
    run = torch.cat((block.new_zeros(1), (block[1:] != block[:-1]).long())).cumsum(0)
    which = torch.arange(runs, device="cuda")
    which = torch.where(which <= run[-1], which, 0)  # entries behind the last run repeat the first
    y = x.float()
    finite = torch.where(y.isfinite(), y.abs(), 0)
    largest = torch.zeros(runs, h, device="cuda").scatter_reduce_(0, run[:, None].expand(-1, h), finite.amax(-1), "amax")
    first = torch.full((runs,), page, device="cuda").scatter_reduce_(0, run, off, "amin")
    blocks = block.new_zeros(runs).scatter_(0, run, block)
    # smallest power of two s with largest / s <= most
    mant, exp = torch.frexp(largest.double() / most)
    step = torch.ldexp(torch.ones_like(mant), torch.where(mant == 0.5, exp - 1, exp)).clamp(min=SMALLEST).float()
    step = torch.where(largest > 0, step, 0)
    before = torch.where((first > 0)[:, None], scales[blocks], 0)
    after = torch.maximum(before, step)
    held = (torch.arange(page, device="cuda") < first[:, None])[:, None, :, None]
    code = lambda v: v.round().clamp(-most, most).to(torch.int8) if cache.dtype == torch.int8 else v.clamp(-most, most).to(cache.dtype)  # noqa: E731
    raw = cache.view(torch.uint8)
    values = raw[blocks].view(cache.dtype).float()
    ratio = torch.where(after > before, before / after, 1)[..., None, None]
    again = torch.where(held, code(values * ratio).float(), values)
    divisor = after[run][..., None]
    rows = torch.where(divisor > 0, y / divisor, 0)
    rows = rows.nan_to_num(nan=0.0, posinf=most, neginf=-most) if cache.dtype == torch.int8 else torch.where(y.isinf(), y.sign() * most, rows)
    again[run, :, off] = code(rows).float()
    raw[blocks[which]] = again[which].to(cache.dtype).view(torch.uint8)
    scales[blocks[which]] = after[which]


def _append(s):
    _append_one(s["k"], s["kc"], s["ks"], s["slots"], s["runs"])
    _append_one(s["v"], s["vc"], s["vs"], s["slots"], s["runs"])
    return s["kc"], s["vc"], s["ks"], s["vs"]


def _gathered(cache, scales, blocks):
    raw = cache.view(torch.uint8)[blocks].view(cache.dtype).float() * scales[blocks][..., None, None]
    n, b, h, p, d = raw.shape
    return raw.transpose(1, 2).reshape(n, h, b * p, d)


def _attention(s):
    q, cu, lens = s["q"], s["cu_plain"].long(), s["lens"].long()
    tokens, heads, d = q.shape
    blocks = s["table"][:, :_pages(s["most_len"], s["page"])].clamp(min=0).long()
    k = _gathered(s["kc"], s["ks"], blocks)
    n, h, length, _ = k.shape
    new, j = cu.diff(), torch.arange(s["most_query"], device="cuda")
    held = j < new[:, None]
    at = torch.where(held, cu[:-1, None] + j, 0)
    rows = q[at].float().reshape(n, j.numel(), h, heads // h, d).permute(0, 2, 3, 1, 4).reshape(n, h, -1, d)
    score = (rows @ k.transpose(-1, -2)).reshape(n, h, heads // h, j.numel(), length) * s["scale"]
    del k
    last = (lens - new)[:, None] + j
    seen = torch.arange(length, device="cuda") <= last[:, :, None]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    most = score.amax(-1, keepdim=True)
    score = score.sub_(most).exp_()
    total = score.sum(-1, keepdim=True)
    o = (score.reshape(n, h, -1, length) @ _gathered(s["vc"], s["vs"], blocks)).reshape(n, h, heads // h, j.numel(), d) / total
    lse = (most + total.log()).squeeze(-1)
    to = torch.where(held, at, tokens)
    out = torch.zeros(tokens + 1, heads, d, device="cuda", dtype=q.dtype)
    out[to] = o.permute(0, 3, 1, 2, 4).reshape(n, j.numel(), heads, d).to(q.dtype)
    back = torch.zeros(tokens + 1, heads, device="cuda")
    back[to] = lse.permute(0, 3, 1, 2).reshape(n, j.numel(), heads)
    return out[:tokens], back[:tokens]


# ---- the framework's operators -------------------------------------------------------------------------------------

def _own(s):
    ops, case = _ops(), s["case"]
    if case["op"] == "plan":
        return *ops.paged_kv_plan(s["context"], s["query"], s["table"], s["free"], s["page"], s["tokens"], state_rows=s["rows"]), s["table"]
    if case["op"] == "rotary":
        how = dict(axis_order="interleaved" if case["interleaved"] else "blocked", pairing="adjacent" if case["adjacent"] else "half")
        q, k = ops.rotary_axes(s["q"], s["k"], s["positions"], s["inv_freq"], s["sections"], **how)
        if not case["train"]:
            return q, k
        return q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
    if case["op"] == "append":
        ops.paged_kv_append(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
        return s["kc"], s["vc"], s["ks"], s["vs"]
    return ops.paged_kv_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], s["table"], s["lens"], s["cu"], scale=s["scale"],
                                  max_query_len=s["most_query"], return_lse=True)


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "rotary": _rotary, "append": _append, "attention": _attention}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "rotary":
        count = case["tokens"] * (case["heads"] + case["kv_heads"])
        turns, size = 2 if case["train"] else 1, 4 if case["dtype"] == "float32" else 2
        return {"bytes": turns * (2 * count * case["dim"] * size + 8 * case["axes"] * case["tokens"]), "flops": turns * count * case["rotated"] * 3}
    context, query = _lengths(case)
    tokens, n, page = sum(query), case["requests"], case["page"]
    if case["op"] == "plan":
        new = sum(_pages(a + b, page) - _pages(a, page) for a, b in zip(context, query))
        return {"bytes": 8 * n + 8 * new + 16 * (tokens + 5) + 8 * n, "flops": 0}
    h, d = case["kv_heads"], case["dim"]
    if case["op"] == "append":
        pages = sum(_pages(a + b, page) - a // page for a, b in zip(context, query))
        return {"bytes": 2 * tokens * h * d * 3 + 8 * tokens + 8 * pages * h, "flops": 2 * tokens * h * d * 2}
    pairs = sum(b * a + b * (b + 1) // 2 for a, b in zip(context, query))
    pages = sum(_pages(a + b, page) for a, b in zip(context, query))
    cached = 2 * sum(context[i] + query[i] for i in range(n)) * h * d
    return {"bytes": cached + pages * (8 * h + 4) + tokens * case["heads"] * (4 * d + 4), "flops": 4 * case["heads"] * d * pairs}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _exact_rotary(s, case):
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       torch.stack([s["positions"][a].double() * s["inv_freq"][j].double() for j, a in enumerate(_axis_of(case))], -1))
    half = case["rotated"] // 2

    def one(x, by):
        x = x.detach().double()
        pairs = x[..., :2 * half]
        z = torch.view_as_complex(pairs.reshape(*pairs.shape[:-1], half, 2)) if case["adjacent"] else torch.complex(*pairs.chunk(2, -1))
        z = torch.view_as_real(z * by[:, None])
        y = x.clone()
        y[..., :2 * half] = z.flatten(-2) if case["adjacent"] else z.transpose(-1, -2).flatten(-2)
        return y

    got = [one(s["q"], turn), one(s["k"], turn)]
    if case["train"]:
        got += [one(s["dq"], turn.conj()), one(s["dk"], turn.conj())]
    return got


def _exact_append(s, case):
    """Page by page, in the tokens' order; the codes as numbers."""
    import numpy as np

    page, most = case["page"], INT8_MOST if case["cache"] == "int8" else E4M3_MOST
    slots = s["slots"].cpu().numpy()
    blocks = slots // page
    begins = np.flatnonzero(np.r_[True, blocks[1:] != blocks[:-1]])
    ends = np.r_[begins[1:], len(slots)]
    begin, end = (torch.from_numpy(v).cuda() for v in (begins, ends))
    touched = torch.from_numpy(blocks[begins]).cuda()
    first = torch.from_numpy(slots[begins] % page).cuda()
    put = torch.arange(page, device="cuda")
    source = begin[:, None] + put - first[:, None]
    fresh = (put >= first[:, None]) & (source < end[:, None])

    def one(x, cache, scales):
        codes, steps = cache.double(), scales.double()
        for part in torch.arange(len(begins), device="cuda").split(4096):
            rows = x[source[part].clamp(0, x.shape[0] - 1)].double().transpose(1, 2)  # [pages, heads, page, dim]
            rows = torch.where(fresh[part][:, None, :, None], rows, 0)
            largest = rows.abs().amax((-1, -2))
            step = torch.exp2(torch.ceil(torch.log2(largest / most)))
            step = torch.where(largest > most * step, step * 2, torch.where(largest <= most * step / 2, step / 2, step))
            step = torch.where(largest > 0, step.clamp(min=SMALLEST), 0)
            had = torch.where(first[part][:, None] > 0, steps[touched[part]], 0)
            now = torch.maximum(had, step)
            kept = codes[touched[part]] * torch.where(now > had, had / now, 1)[..., None, None]
            old = (put < first[part][:, None])[:, None, :, None]
            to = (lambda v: v.round()) if case["cache"] == "int8" else (lambda v: v.float().to(torch.float8_e4m3fn).double())
            scaled = torch.where(now[..., None, None] > 0, rows / now[..., None, None], 0)
            codes[touched[part]] = torch.where(old, to(kept), torch.where(fresh[part][:, None, :, None], to(scaled), codes[touched[part]]))
            steps[touched[part]] = now
        return codes, steps

    (kc, ks), (vc, vs) = one(s["k"], s["kc"], s["ks"]), one(s["v"], s["vc"], s["vs"])
    return [kc, vc, ks, vs]


def _exact_attention(s, case):
    context, query = _lengths(case)
    group, page, outs, lses, at = case["heads"] // case["kv_heads"], case["page"], [], [], 0
    for r, (had, new) in enumerate(zip(context, query)):
        total = had + new
        blocks = s["table"][r, :_pages(total, page)].long()
        q = s["q"][at:at + new].double()
        o = torch.empty_like(q)
        lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
        seen = torch.arange(total, device="cuda") <= torch.arange(had, total, device="cuda")[:, None]
        for h in range(case["kv_heads"]):
            k = (s["kc"][:, h].view(torch.uint8)[blocks].view(s["kc"].dtype).double() * s["ks"][blocks, h].double()[:, None, None]).flatten(0, 1)[:total]
            v = (s["vc"][:, h].view(torch.uint8)[blocks].view(s["vc"].dtype).double() * s["vs"][blocks, h].double()[:, None, None]).flatten(0, 1)[:total]
            for head in range(h * group, (h + 1) * group):
                score = torch.where(seen, (q[:, head] @ k.t()) * s["scale"], -math.inf)
                lse[:, head] = torch.logsumexp(score, -1)
                o[:, head] = torch.softmax(score, -1) @ v
        outs.append(o)
        lses.append(lse)
        at += new
    return torch.cat(outs), torch.cat(lses)


def exact(case, seed):
    if case["op"] == "plan":  # whole numbers only
        return None
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(s, case)
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["requests"] * case["heads"] > 8192:
        return None
    return _exact_attention(s, case)
