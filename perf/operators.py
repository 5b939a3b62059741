"""Workloads of the operators around a quantised cache of keys and values.

The cache holds keys and values in pages, in the OCP MX block formats that the quantising norms
write: elements of 4 bits (e2m1, two to a byte, the even one in the low nibble) or 8 bits (e4m3),
and one power-of-two scale (E8M0) for 32 elements of a head vector.  It is a tuple

    (k_codes, k_scales, v_codes, v_scales)
    codes   [pages, kv_heads, page, head_dim / 2]  float4_e2m1fn_x2, or
            [pages, kv_heads, page, head_dim]      float8_e4m3fn
    scales  [pages, kv_heads, head_dim / 32, page] float8_e8m0fnu

and a token's place in it is its slot, page_index * page + place in the page.

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs and the cache on the GPU
    run(state)          one pass: its outputs
    work(case)          bytes and operations a pass cannot do without
    exact(case, seed)   the same outputs from the definition, in 64 bits

Operators:
    write       rope_mx_cache_write (rope true) or mx_cache_write of new tokens' keys and values, which
                come as slices of one projection's output; the values they became are read back by
                mx_cache_read
    read        mx_cache_read of whole sequences
    attention   mx_cache_attention of new tokens over everything their sequence holds
"""

import math

import torch

own = False  # the framework's kernels instead of the plain forms

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
BLOCK = 32
EMAX = {"e2m1": 2, "e4m3": 8}


def listed():
    return [
        # one decode step of a few sequences, rotated and written: latency
        dict(name="write_step_8", op="write", fmt="e2m1", dtype="bf16", heads=32, kv_heads=8, dim=128,
             page=16, batch=8, shortest=700, longest=4000, new=1, new_min=1, pad=0, rope=True),
        # a prefill chunk of one sequence that starts inside a page
        dict(name="write_chunk_8191", op="write", fmt="e2m1", dtype="bf16", heads=32, kv_heads=8,
             dim=128, page=64, batch=1, shortest=12301, longest=12301, new=8191, new_min=8191, pad=1,
             rope=True),
        # ragged chunks of several sequences in fp32, already rotated, with padding rows
        dict(name="write_ragged_fp32", op="write", fmt="e4m3", dtype="fp32", heads=0, kv_heads=4,
             dim=64, page=16, batch=9, shortest=90, longest=1500, new=700, new_min=3, pad=37, rope=False),
        # sequences read back whole, to be moved or attended to elsewhere
        dict(name="read_64k_tokens", op="read", fmt="e2m1", dtype="bf16", kv_heads=8, dim=128, page=64,
             batch=4, shortest=16000, longest=17000),
        dict(name="read_ragged_fp16", op="read", fmt="e4m3", dtype="fp16", kv_heads=2, dim=256, page=16,
             batch=7, shortest=1, longest=2001),
        # the smallest decode step: one sequence of ordinary length
        dict(name="step_1x2000", op="attention", fmt="e2m1", dtype="bf16", heads=32, kv_heads=8, dim=128,
             page=16, batch=1, shortest=2000, longest=2000, new=1, new_min=1, pad=0, empty=0),
        # a serving batch's decode step, sequences of very different lengths
        dict(name="step_64_ragged", op="attention", fmt="e2m1", dtype="bf16", heads=32, kv_heads=8,
             dim=128, page=64, batch=64, shortest=300, longest=12001, new=1, new_min=1, pad=0, empty=0),
        # long contexts, few sequences
        dict(name="step_2x131072", op="attention", fmt="e2m1", dtype="bf16", heads=64, kv_heads=8,
             dim=128, page=128, batch=2, shortest=131001, longest=131072, new=1, new_min=1, pad=0,
             empty=0),
        # 8-bit elements, wide heads, a padded batch with an empty sequence
        dict(name="step_24_e4m3_fp16", op="attention", fmt="e4m3", dtype="fp16", heads=16, kv_heads=2,
             dim=256, page=16, batch=24, shortest=1, longest=9000, new=1, new_min=1, pad=3, empty=1),
        # several drafted tokens a sequence, checked at once; fp32 queries
        dict(name="draft_16x5_fp32", op="attention", fmt="e4m3", dtype="fp32", heads=16, kv_heads=4,
             dim=64, page=16, batch=16, shortest=900, longest=5003, new=5, new_min=5, pad=0, empty=0),
        # chunks of prefill and single tokens in one batch
        dict(name="mixed_24_ragged", op="attention", fmt="e2m1", dtype="bf16", heads=32, kv_heads=8,
             dim=64, page=32, batch=24, shortest=600, longest=4100, new=517, new_min=1, pad=11,
             empty=1),
        # a prefill chunk on a long prefix: the matrix products
        dict(name="chunk_4096_of_16383", op="attention", fmt="e2m1", dtype="bf16", heads=32, kv_heads=8,
             dim=128, page=64, batch=1, shortest=16383, longest=16383, new=4096, new_min=4096, pad=0,
             empty=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["write", "read", "attention", "attention"])
    c = dict(op=op, fmt=rng.choice(["e2m1", "e2m1", "e4m3"]), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]),
             kv_heads=rng.choice([1, 2, 3, 4, 8]), dim=rng.choice([64, 128, 128, 256]),
             page=rng.choice([16, 32, 64, 128, 256]))
    if op == "read":
        batch, longest = _log(rng, 1, 16), _log(rng, 20, 6000)
        return dict(c, batch=batch, shortest=rng.randint(1, longest), longest=longest)
    c["heads"] = c["kv_heads"] * rng.choice([g for g in (1, 2, 4, 5, 8, 16) if g * c["kv_heads"] <= 64])
    if op == "write":
        batch, new = _log(rng, 1, 64), rng.choice([1, _log(rng, 2, 1000)])
        longest = new + _log(rng, 1, 8000)
        rope = rng.random() < 0.7
        return dict(c, heads=c["heads"] if rope else 0, batch=batch, new=new, new_min=rng.randint(1, new),
                    longest=longest, shortest=rng.randint(new, longest),
                    pad=rng.choice([0, rng.randint(1, 40)]), rope=rope)
    kind = rng.choice(["step", "step", "draft", "chunk"])
    if kind == "step":
        batch, new, longest = _log(rng, 1, 100), 1, _log(rng, 30, 16000)
        new_min = 1
    elif kind == "draft":
        batch, new, longest = _log(rng, 1, 32), rng.randint(2, 12), _log(rng, 60, 8000)
        new_min = rng.randint(1, new)
    else:
        batch, new, longest = _log(rng, 1, 8), _log(rng, 20, 1200), _log(rng, 1300, 6000)
        new_min = rng.randint(1, new)
    return dict(c, batch=batch, shortest=rng.randint(min(new, longest), longest), longest=longest, new=new,
                new_min=new_min, pad=rng.choice([0, rng.randint(1, 9)]), empty=rng.choice([0, 0, 1]))


def _spread(low, high, n):
    return [low + (high - low) * i // max(1, n - 1) for i in range(n - 1)] + [high]


def _plan(case):
    """(tokens held, new tokens) of each sequence."""
    held = _spread(case["shortest"], case["longest"], case["batch"])
    new = _spread(case.get("new_min", 0), case.get("new", 0), case["batch"])
    for i in range(case.get("empty", 0)):
        held[i] = 0
    return held, new


def _encode(x, fmt):
    """MX codes (bytes) of x [..., dim] and scale bytes [..., dim / 32]."""
    blocks = x.float().unflatten(-1, (-1, BLOCK))
    top = blocks.abs().amax(-1, keepdim=True)
    s = (torch.frexp(top)[1] - 1 - EMAX[fmt]).clamp(-127, 127)
    s = torch.where(top == 0, -127, s)
    scaled = torch.ldexp(blocks, -s).flatten(-2)
    if fmt == "e4m3":
        codes = scaled.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        a = scaled.abs().clamp(max=6.0)  # 0, 0.5 .. 2, then 3, 4, 6: steps of 0.5, 1 and 2
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        a = ((a / step).round() * step).clamp(max=6.0)
        codes = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)) + 8 * torch.signbit(scaled)
        codes = codes.to(torch.uint8)
        codes = codes[..., 0::2] + codes[..., 1::2] * 16
    return codes, (s + 127).to(torch.uint8).squeeze(-1)


def _decode(codes, scales, fmt):
    """Values of codes [..., bytes] with scale bytes [..., dim / 32], in 32 bits."""
    if fmt == "e4m3":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
        a = (n & 7).float()
        a = torch.where(a < 4, 0.5 * a, torch.where(a < 6, a - 2, 2 * a - 8))
        v = torch.where(n > 7, -a, a)
    s = scales.int()
    f = torch.where(s == 0, 1 << 22, s << 23).view(torch.float32)
    f = torch.where(s == 255, float("nan"), f)
    return (v.unflatten(-1, (-1, BLOCK)) * f[..., None]).flatten(-2)


def _bytes(cache):
    return [t.view(torch.uint8) for t in cache]


def _make(case, gen, pages):
    """A cache full of tokens' keys (some channels larger, as keys have them) and values."""
    fmt, heads, dim, page = case["fmt"], case["kv_heads"], case["dim"], case["page"]
    size = dim // 2 if fmt == "e2m1" else dim
    channels = torch.exp(0.5 * torch.randn(heads, 1, dim, device="cuda", generator=gen))
    out = []
    for scale in (channels, 1.0):
        codes = torch.empty(pages, heads, page, size, device="cuda", dtype=torch.uint8)
        scales = torch.empty(pages, heads, dim // BLOCK, page, device="cuda", dtype=torch.uint8)
        step = max(1, (1 << 26) // (heads * page * dim))
        for at in range(0, pages, step):
            n = min(step, pages - at)
            x = torch.randn(n, heads, page, dim, device="cuda", generator=gen) * scale
            c, s = _encode(x, fmt)
            codes[at:at + n], scales[at:at + n] = c, s.transpose(-1, -2)
        out += [codes.view(torch.float4_e2m1fn_x2 if fmt == "e2m1" else torch.float8_e4m3fn),
                scales.view(torch.float8_e8m0fnu)]
    return tuple(out)


def _slots(table, first, last, page):
    """Slots of each sequence's tokens first .. last - 1, one after the other."""
    got = []
    for i, (a, b) in enumerate(zip(first, last)):
        t = torch.arange(a, b, device="cuda")
        got.append(table[i, t // page].long() * page + t % page)
    return torch.cat(got)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    held, new = _plan(case)
    page = case["page"]
    need = [-(-h // page) for h in held]
    width = max(1, max(need))
    spare = 3
    order = torch.randperm(sum(need) + spare, device="cuda", generator=gen).int()
    table = torch.zeros(len(held), width, device="cuda", dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    dtype = DTYPES[case["dtype"]]
    s = {"case": dict(case), "cache": _make(case, gen, sum(need) + spare)}
    if case["op"] == "read":
        s["slots"] = _slots(table, [0] * len(held), held, page)
    elif case["op"] == "write":
        q_heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        slots = _slots(table, [h - n for h, n in zip(held, new)], held, page)
        total = slots.numel() + case["pad"]
        x = torch.randn(total, q_heads + 2 * kv_heads, dim, device="cuda", generator=gen)
        x[:, q_heads:q_heads + kv_heads] *= torch.exp(0.5 * torch.randn(dim, device="cuda", generator=gen))
        x = x.to(dtype)
        s["q"], s["k"], s["v"] = x.split([q_heads, kv_heads, kv_heads], dim=1)
        s["slots"] = torch.cat((slots, slots.new_full((case["pad"],), -1)))
        if case["rope"]:
            where = torch.cat([torch.arange(h - n, h, device="cuda") for h, n in zip(held, new)])
            s["positions"] = torch.cat((where, where.new_zeros(case["pad"])))
            j = torch.arange(dim // 2, device="cuda", dtype=torch.float64)
            angle = torch.arange(max(held), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (-2 * j / dim)
            s["cos_sin"] = torch.cat((angle.cos(), angle.sin()), -1).float()
    else:
        total = sum(new) + case["pad"]
        s["q"] = torch.randn(total, case["heads"], case["dim"], device="cuda", generator=gen).to(dtype)
        s["table"] = table
        s["lengths"] = torch.tensor(held, device="cuda", dtype=torch.int32)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        one_each = case["new"] == 1 and not case["pad"]
        s["starts"] = None if one_each else torch.tensor(starts, device="cuda", dtype=torch.int32)
        s["most"] = max(new)
    return s


def run(state):
    op = state["case"]["op"]
    return _write(state) if op == "write" else _read(state) if op == "read" else _attention(state)


def _write(s):
    case = s["case"]
    if own:
        from velograd_amd import kernels as vk
        q = None
        if case["rope"]:
            q = vk.rope_mx_cache_write(s["q"], s["k"], s["v"], s["cos_sin"], s["positions"], s["cache"], s["slots"])
        else:
            vk.mx_cache_write(s["k"], s["v"], s["cache"], s["slots"])
        k, v = vk.mx_cache_read(s["cache"], s["slots"], s["k"].dtype)
        return {"k": k, "v": v} if q is None else {"q": q, "k": k, "v": v}
    out, k = {}, s["k"]
    if case["rope"]:
        c, d = s["cos_sin"][s["positions"]][:, None].chunk(2, -1)
        out["q"], k = _rotate(s["q"], c, d), _rotate(k, c, d)
    n = k.shape[0] - case["pad"]
    slots = s["slots"][:n]
    page, place = slots // case["page"], slots % case["page"]
    kc, ks, vc, vs = _bytes(s["cache"])
    kc[page, :, place], ks[page, :, :, place] = _encode(k[:n], case["fmt"])
    vc[page, :, place], vs[page, :, :, place] = _encode(s["v"][:n], case["fmt"])
    out["k"] = _held(kc, ks, page, place, case)
    out["v"] = _held(vc, vs, page, place, case)
    return out


def _held(codes, scales, page, place, case):
    x = _decode(codes[page, :, place], scales[page, :, :, place], case["fmt"]).to(DTYPES[case["dtype"]])
    return torch.cat((x, x.new_zeros((case.get("pad", 0),) + x.shape[1:])))


def _rotate(x, c, s):
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * c - b * s, a * s + b * c), -1).to(x.dtype)


def _read(s):
    case = s["case"]
    dtype = DTYPES[case["dtype"]]
    if own:
        from velograd_amd import kernels as vk
        k, v = vk.mx_cache_read(s["cache"], s["slots"], dtype)
        return {"k": k, "v": v}
    page, place = s["slots"] // case["page"], s["slots"] % case["page"]
    kc, ks, vc, vs = _bytes(s["cache"])
    return {"k": _held(kc, ks, page, place, case), "v": _held(vc, vs, page, place, case)}


def _attention(s):
    if own:
        from velograd_amd import kernels as vk
        out, lse = vk.mx_cache_attention(s["q"], s["cache"], s["table"], s["lengths"], s["starts"], return_lse=True)
        return {"out": out, "lse": lse}
    case, q, lengths, most = s["case"], s["q"], s["lengths"].long(), s["most"]
    total, heads, dim = q.shape
    batch, group = lengths.numel(), heads // case["kv_heads"]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(batch + 1, device=q.device)
    new = starts[1:] - starts[:-1]
    i = torch.arange(most, device=q.device)
    rows = (starts[:-1, None] + i).clamp(max=total - 1)
    x = q[rows].float() * dim ** -0.5
    x = x.view(batch, most, -1, group, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    kc, ks, vc, vs = _bytes(s["cache"])
    table = s["table"].long()
    k = _decode(kc[table], ks[table].transpose(-1, -2), case["fmt"]).transpose(1, 2).flatten(2, 3)
    scores = (x @ k.transpose(-1, -2)).unflatten(2, (group, most))
    del k
    j = torch.arange(scores.shape[-1], device=q.device)
    limit = torch.minimum(lengths[:, None], lengths[:, None] - new[:, None] + i + 1)
    hidden = j >= limit[..., None]
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(top.clamp(min=-1e30)).exp_()
    below = scores.sum(-1, keepdim=True)
    v = _decode(vc[table], vs[table].transpose(-1, -2), case["fmt"]).transpose(1, 2).flatten(2, 3)
    o = (scores.flatten(2, 3) @ v).unflatten(2, (group, most))
    o = torch.where(below > 0, o / below, 0.0)
    lse = (top + below.log()).squeeze(-1)
    flat = (torch.arange(total, device=q.device) - starts[:-1, None])
    inside = (flat >= 0) & (flat < new[:, None])
    which, at = inside.int().argmax(0), (flat * inside).sum(0)
    any_ = inside.any(0)
    o = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[which, at]
    lse = lse.permute(0, 3, 1, 2).flatten(2, 3)[which, at]
    return {"out": torch.where(any_[:, None, None], o, 0.0).to(q.dtype),
            "lse": torch.where(any_[:, None], lse, -math.inf)}


def work(case):
    held, new = _plan(case)
    kv, dim = case["kv_heads"], case["dim"]
    stored = 2 * kv * ((dim // 2 if case["fmt"] == "e2m1" else dim) + dim // BLOCK)  # of a token in the cache
    b = SIZES[case["dtype"]]
    if case["op"] == "read":
        n = sum(held)
        return {"bytes": float(n * (stored + 2 * kv * dim * b + 8)), "flops": float(2 * n * kv * dim)}
    if case["op"] == "write":
        n = sum(new)
        t = n + case["pad"]
        size = n * (2 * kv * dim * b + 2 * stored + 8) + t * 2 * kv * dim * b
        if case["rope"]:
            size += 2 * t * case["heads"] * dim * b + 8 * t + 4 * dim * min(t, max(held))
        return {"bytes": float(size), "flops": float(n * (8 * kv + 3 * case["heads"]) * dim)}
    t = sum(new) + case["pad"]
    seen = sum(sum(max(0, h - n + i + 1) for i in range(n)) for h, n in zip(held, new))
    size = sum(held) * stored + t * case["heads"] * (2 * dim * b + 4) + 4 * sum(-(-h // case["page"]) for h in held)
    return {"bytes": float(size), "flops": 4.0 * dim * case["heads"] * seen}


def exact(case, seed):
    s = prepare(case, seed)
    return {"write": _exact_write, "read": _exact_read, "attention": _exact_attention}[case["op"]](s, case)


def _exact_elements(codes, fmt):
    """What element codes stand for, in 64 bits, from their fields: sign, exponent, mantissa."""
    c = codes.int()
    if fmt == "e2m1":
        sign, e, m, width, bias = c // 8, (c // 2) % 4, c % 2, 2.0, 1
    else:
        sign, e, m, width, bias = c // 128, (c // 8) % 16, c % 8, 8.0, 7
    v = torch.where(e == 0, (m / width).double() * 2.0 ** (1 - bias),
                    (1 + m / width).double() * torch.exp2((e - bias).double()))
    return (1.0 - 2.0 * sign) * v


def _exact_values(codes, scales, fmt):
    """[tokens, heads, dim] in 64 bits."""
    if fmt == "e2m1":
        codes = torch.stack((codes % 16, codes // 16), -1).flatten(-2)
    f = torch.exp2(scales.double() - 127).masked_fill(scales == 255, math.nan)
    return _exact_elements(codes, fmt) * f.repeat_interleave(BLOCK, -1)


def _exact_rounded(x, fmt):
    """The nearest values, ties to the even code, that the format has for x [tokens, heads, dim]."""
    b = x.double().unflatten(-1, (-1, BLOCK))
    top = b.abs().amax(-1, keepdim=True)
    s = torch.floor(torch.log2(top))
    s = torch.where(torch.exp2(s) > top, s - 1, torch.where(torch.exp2(s + 1) <= top, s + 1, s))
    f = torch.exp2((s - EMAX[fmt]).clamp(-127, 127))
    grid = _exact_elements(torch.arange(8 if fmt == "e2m1" else 127, device=x.device), fmt)
    mid = (grid[1:] + grid[:-1]) / 2
    a = torch.where(top > 0, b.abs() / f, 0.0)
    at = torch.searchsorted(mid, a)  # a value at a midpoint gets the lower neighbour
    tie = (at < len(mid)) & (a == mid[at.clamp(max=len(mid) - 1)]) & (at % 2 == 1)
    return (torch.sign(b) * grid[at + tie] * f).flatten(-2)


def _exact_write(s, case):
    n = s["k"].shape[0] - case["pad"]
    k, v, out = s["k"].double(), s["v"].double(), {}
    if case["rope"]:
        c, d = s["cos_sin"].double()[s["positions"]][:, None].chunk(2, -1)

        def turned(x):
            a, b = x.double().chunk(2, -1)
            return torch.cat((a * c - b * d, b * c + a * d), -1)
        out["q"] = turned(s["q"])
        k = turned(k).to(s["k"].dtype)  # what is quantised is the rotated key as its type holds it
    for name, x in (("k", k), ("v", v)):
        x = _exact_rounded(x[:n], case["fmt"])
        out[name] = torch.cat((x, x.new_zeros((case["pad"],) + x.shape[1:])))
    return out


def _exact_read(s, case):
    page, place = s["slots"] // case["page"], s["slots"] % case["page"]
    kc, ks, vc, vs = _bytes(s["cache"])
    return {"k": _exact_values(kc[page, :, place], ks[page, :, :, place], case["fmt"]),
            "v": _exact_values(vc[page, :, place], vs[page, :, :, place], case["fmt"])}


def _exact_attention(s, case):
    held, new = _plan(case)
    q = s["q"].double()
    total, heads, dim = q.shape
    kv, page = case["kv_heads"], case["page"]
    kc, ks, vc, vs = _bytes(s["cache"])
    out, lse = torch.zeros_like(q), torch.full((total, heads), -math.inf, device=q.device, dtype=torch.float64)
    at = 0
    for i, (length, n) in enumerate(zip(held, new)):
        if length:
            t = torch.arange(length, device=q.device)
            p, r = s["table"][i, t // page].long(), t % page
            k = _exact_values(kc[p, :, r], ks[p, :, :, r], case["fmt"])
            v = _exact_values(vc[p, :, r], vs[p, :, :, r], case["fmt"])
            seen = t <= torch.arange(length - n, length, device=q.device)[:, None]
            for h in range(heads):
                w = (q[at:at + n, h] @ k[:, h // (heads // kv)].T) / math.sqrt(dim)
                w = w.masked_fill(~seen, -math.inf)
                lse[at:at + n, h] = torch.logsumexp(w, -1)
                out[at:at + n, h] = torch.softmax(w, -1) @ v[:, h // (heads // kv)]
        at += n
    return {"out": out, "lse": lse}
