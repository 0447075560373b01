"""Paged 8-bit cache: plan, rotary positions, append and attention, restated in 64 bits, one request, page and row at a time."""
import math

import torch

LARGEST = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def plan(context, query, table, free, page, num_tokens, state_rows=None):
    """Lists in, dict of tensors out; ``table`` is a list of lists and is changed in place."""
    width = len(table[0]) if table else 0
    pages = lambda n: min(-(-n // page), width)
    slots, positions, states, cu, seq, used = [], [], [], [0], [], 0
    for r, (c, q) in enumerate(zip(context, query)):
        c, q = max(c, 0), max(q, 0)
        for j in range(pages(c), pages(c + q)):
            table[r][j] = free[used] if used < len(free) else -1
            used += 1
        for pos in range(c, c + q):
            block = table[r][pos // page] if pos // page < width else -1
            slots.append(block * page + pos % page if block >= 0 else -1)
            positions.append(pos)
            states.append(-1 if state_rows is None else state_rows[r])
        cu.append(cu[-1] + q)
        seq.append(c + q)
    fit = lambda v, pad: (v + [pad] * num_tokens)[:num_tokens]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    return dict(slots=torch.tensor(fit(slots, -1), dtype=torch.int64), positions=i32(fit(positions, 0)), cu=i32(cu), seq=i32(seq),
                used=i32([used]), states=i32(fit(states, -1)), table=i32(table))


def axis_of(sections, order):
    if order == "blocked":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [a for i in range(max(sections)) for a, n in enumerate(sections) if i < n]


def rotary(x, positions, inv_freq, sections, order, pairing, inverse=False):
    """x [..., T, H, D] in any float type; returns float64."""
    x = x.double()
    half = inv_freq.numel()
    angle = torch.stack([positions[a].double() * inv_freq[j].double() for j, a in enumerate(axis_of(sections, order))], -1)
    if inverse:
        angle = -angle
    cos, sin = angle.cos()[..., None, :], angle.sin()[..., None, :]
    first = slice(0, 2 * half, 2) if pairing == "adjacent" else slice(0, half)
    second = slice(1, 2 * half, 2) if pairing == "adjacent" else slice(half, 2 * half)
    y = x.clone()
    a, b = x[..., first], x[..., second]
    y[..., first] = a * cos - b * sin
    y[..., second] = b * cos + a * sin
    return y


def encode(v, dtype):
    """float64 values (already divided by the scale) to codes as numbers, round to nearest even."""
    most = LARGEST[dtype]
    if dtype == torch.int8:
        return torch.where(v.isnan(), 0.0, v).clamp(-most, most).round()
    v = v.clamp(-most, most)                                                       # NaN stays
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)   # 3 fraction bits; subnormals below 2^-6
    return torch.where(v.isnan(), v, (v / step).round() * step)


def step_for(most_abs, dtype):
    if most_abs == 0:
        return 0.0
    s = 2.0 ** -126
    while most_abs / s > LARGEST[dtype]:
        s *= 2
    while s > 2.0 ** -126 and most_abs / (s / 2) <= LARGEST[dtype]:
        s /= 2
    return s


def append(x, codes, scales, slots, dtype):
    """codes float64 [P,H,page,D] and scales float64 [P,H] are changed in place."""
    pool, heads, page, _ = codes.shape
    t, slots = 0, [int(s) for s in slots]
    while t < len(slots):
        if slots[t] < 0 or slots[t] // page >= pool:
            t += 1
            continue
        block, off, n = slots[t] // page, slots[t] % page, 1
        while off + n < page and t + n < len(slots) and slots[t + n] == slots[t] + n:
            n += 1
        for h in range(heads):
            rows = x[t:t + n, h].double()
            finite = rows.abs()[rows.isfinite()]
            before = float(scales[block, h]) if off else 0.0
            after = max(before, step_for(float(finite.max()) if finite.numel() else 0.0, dtype))
            if off and after > before:
                codes[block, h, :off] = encode(codes[block, h, :off] * (before / after), dtype)
            codes[block, h, off:off + n] = encode(rows / after if after else torch.where(rows.isfinite(), 0.0, rows), dtype)
            scales[block, h] = after
        t += n


def attention(q, key_codes, value_codes, key_scales, value_scales, table, lens, cu, scale):
    """float64 (out, lse, spread, reach, peak) for codes given as float64 [P,H,page,D].  ``spread``: the weighted mean of |v|,
    ``reach``: the largest scale * sum |q||k| of a row, and ``peak``: the largest p * value scale of a row: they bound the
    effect of relative errors of the weights, of the scores, and of absolute errors of the weights.  ``cu`` None: one row
    for each request."""
    tokens, heads, d = q.shape
    pool, kv_heads, page, _ = key_codes.shape
    group = heads // kv_heads
    out, spread = torch.zeros(tokens, heads, d, dtype=torch.float64), torch.zeros(tokens, heads, d, dtype=torch.float64)
    lse, reach = torch.full((tokens, heads), -math.inf, dtype=torch.float64), torch.zeros(tokens, heads, dtype=torch.float64)
    peak = torch.zeros(tokens, heads, dtype=torch.float64)
    cu = list(range(len(lens) + 1)) if cu is None else [int(c) for c in cu]
    for r, length in enumerate(int(n) for n in lens):
        blocks = [int(b) for b in table[r]]
        held = [t for t in range(min(length, len(blocks) * page)) if 0 <= blocks[t // page] < pool]
        new = cu[r + 1] - cu[r]
        if not held or not new:
            continue
        at = torch.tensor(held)
        block = torch.tensor([blocks[t // page] for t in held])
        off = at % page
        for h in range(kv_heads):
            k = key_codes[block, h, off].double() * key_scales[block, h].double()[:, None]
            v = value_codes[block, h, off].double() * value_scales[block, h].double()[:, None]
            for j in range(new):
                n = int((at <= length - new + j).sum())
                if n == 0:
                    continue
                qs = q[cu[r] + j, h * group:(h + 1) * group].double()
                s = (qs @ k[:n].t()) * scale
                p = torch.softmax(s, -1)
                sl = (cu[r] + j, slice(h * group, (h + 1) * group))
                out[sl], spread[sl] = p @ v[:n], p @ v[:n].abs()
                lse[sl] = torch.logsumexp(s, -1)
                peak[sl] = (p * value_scales[block[:n], h].double().abs()).amax(-1)
                reach[sl] = (qs.abs() @ k[:n].abs().t()).amax(-1) * abs(scale)
    return out, lse, spread, reach, peak
