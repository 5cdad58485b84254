"""Serving from a quantised paged KV cache, as cases that can be timed and checked.

What a layer of a model does to a step's new tokens and to its cache, where the cache is held in 4 or 8 bits:

* rotary: queries and keys rotated by their tokens' positions;
* append: new keys and values quantised into their slots, and read back the way a chunk of a prompt is for what
  comes after it in the layer;
* read: the values of any slots of a cache;
* attend: attention of each sequence's last tokens (one, or a few that are being verified) over its pages.

A row (one token's key or value of one KV head, D channels) is stored as codes c of 4 or 8 bits, a scale s and a
lowest value m, both bf16: its values are m + c s.  Of a row x, m is the least value, s the least bf16 whose last
multiple, 15 s or 255 s, reaches max(x) - m, and c the whole number next to (x - m) / s, the even one of two; both
differences are rounded to fp32.  A cache is bytes [num_blocks][Hkv][page * (8 + D bits / 4)]: for
each (page, KV head) first (s, m) of the key and (s, m) of the value of every token, then the tokens' rows of key
codes, then those of the value codes.  In 4 bits dword j of a row holds channels 8j + 2i in bits 4i and up and
channels 8j + 2i + 1 in bits 16 + 4i and up; in 8 bits every channel is a byte.

Queries, keys and values are N(0, 1) times a log-normal scale per channel, pages are handed out in a random order.
"""
import math

import torch

own = False


def listed():
    return [
        # One user's next token: the smallest call, nothing but latency.
        dict(name="rotary_t1", kind="rotary", tokens=1, padded=0, heads=32, kv_heads=8, dim=128, rotated=128,
             interleaved=False, base=500000.0, stretch=1.0, far=8000, type="bfloat16"),
        # A chunk of a few long prompts, positions stretched for a longer context.
        dict(name="rotary_t8000", kind="rotary", tokens=8000, padded=192, heads=32, kv_heads=8, dim=128, rotated=128,
             interleaved=False, base=500000.0, stretch=8.0, far=1000000, type="bfloat16"),
        # Neighbouring channels in pairs, half of each head left as it is.
        dict(name="rotary_part_t3001", kind="rotary", tokens=3001, padded=0, heads=16, kv_heads=16, dim=64, rotated=32,
             interleaved=True, base=10000.0, stretch=1.0, far=100000, type="float16"),
        # A decode step's new keys and values, as slices of the fused projection's output.
        dict(name="append_b32", kind="append", bits=4, batch=32, tokens=32, heads=32, kv_heads=8, dim=128, page=16,
             padded=0),
        # A prefill chunk of a few requests with ragged lengths, in a padded batch.
        dict(name="append_t8000", kind="append", bits=4, batch=5, tokens=8000, heads=32, kv_heads=8, dim=128, page=16,
             padded=192),
        # Small heads in large pages, 8 bits.
        dict(name="append_d64_t3001", kind="append", bits=8, batch=3, tokens=3001, heads=16, kv_heads=16, dim=64,
             page=128, padded=0),
        # A shared prompt of some hundred tokens taken out of the cache.
        dict(name="read_t700", kind="read", bits=8, batch=1, tokens=700, kv_heads=8, dim=128, page=16),
        # A batch's long contexts taken out to be kept elsewhere.
        dict(name="read_t60000", kind="read", bits=4, batch=7, tokens=60000, kv_heads=8, dim=128, page=16),
        # One user's next token after a long context: few rows, so latency and the spread over the chip.
        dict(name="attend_b1_t32k", kind="attend", bits=4, batch=1, new=1, tokens=32000, ragged=False, heads=32,
             kv_heads=8, dim=128, page=16),
        # A large serving batch: the cache's bytes from HBM.
        dict(name="attend_b64_t8k", kind="attend", bits=4, batch=64, new=1, tokens=8000, ragged=False, heads=64,
             kv_heads=8, dim=128, page=16),
        # Small heads without groups, ragged contexts, 8 bits.
        dict(name="attend_d64_mha_b20", kind="attend", bits=8, batch=20, new=1, tokens=5001, ragged=True, heads=16,
             kv_heads=16, dim=64, page=32),
        # Five proposed tokens of each request verified at once.
        dict(name="attend_new5_b16", kind="attend", bits=4, batch=16, new=5, tokens=12000, ragged=True, heads=64,
             kv_heads=8, dim=128, page=64),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "read", "attend"])
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (16, 16), (8, 1), (28, 4), (40, 8), (16, 2), (32, 2)])
    dim = rng.choice([128, 128, 64])
    if kind == "rotary":
        tokens = _spread(rng, 1, 8000 * 40 // max(40, heads + kv_heads))
        return dict(kind=kind, tokens=tokens, padded=rng.choice([0, 0, rng.randint(1, 100)]), heads=heads,
                    kv_heads=kv_heads, dim=dim, rotated=rng.choice([dim, dim, dim // 2, dim // 4]),
                    interleaved=rng.random() < 0.5, base=rng.choice([10000.0, 500000.0, 1000000.0]),
                    stretch=rng.choice([1.0, 1.0, 4.0, 8.0]), far=_spread(rng, 100, 1000000),
                    type=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
    bits = rng.choice([4, 4, 8])
    if kind == "append":
        tokens = _spread(rng, 1, 8000 * 8 // max(8, kv_heads))
        return dict(kind=kind, bits=bits, batch=min(tokens, _spread(rng, 1, 64)), tokens=tokens, heads=heads,
                    kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128]),
                    padded=rng.choice([0, 0, rng.randint(1, 100)]))
    if kind == "read":
        tokens = _spread(rng, 1, 60000 * 8 // max(8, kv_heads))
        return dict(kind=kind, bits=bits, batch=min(tokens, _spread(rng, 1, 64)), tokens=tokens, kv_heads=kv_heads,
                    dim=dim, page=rng.choice([16, 32, 64, 128]))
    batch, new = _spread(rng, 1, 64), rng.choice([1, 1, 1, rng.randint(2, 8)])
    # at most 2 M (token, head) rows a cache, 1 M in 8 bits, and 100 M scores
    most = min((8_000_000 // bits) // (batch * kv_heads), 100_000_000 // (batch * heads * new))
    return dict(kind=kind, bits=bits, batch=batch, new=new, tokens=_spread(rng, 8, max(40, min(130_000, most))),
                ragged=rng.random() < 0.5, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 16, 32, 64]))


# --------------------------------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _lengths(case):
    """Tokens of each sequence, the new ones among them: all, or spread evenly up to all."""
    b, t = case["batch"], case["tokens"]
    if not case["ragged"]:
        return [t] * b
    lens = [max(1, t * (i + 1) // b) for i in range(b)]
    return lens[::2] + lens[1::2][::-1]


def _parts(total, count, g):
    """`total` cut into `count` whole numbers of one or more."""
    cuts = torch.randperm(total - 1, device="cuda", generator=g)[: count - 1].sort().values + 1
    edge = torch.zeros(1, dtype=torch.int64, device="cuda")
    return torch.diff(torch.cat([edge, cuts, edge + total]))


def _table(pages, width, blocks, g):
    """A block table (rows of `width`) that gives row b its pages[b] of `blocks` pages in a random order."""
    order = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32)
    held = torch.arange(width, device="cuda") < torch.tensor(pages, device="cuda")[:, None]
    table = torch.zeros(len(pages), width, dtype=torch.int32, device="cuda")
    table[held] = order[:sum(pages)]
    return table


def _scale(shape, g):
    return torch.randn(shape, device="cuda", generator=g).exp_()


def _filled(blocks, case, g):
    """A cache whose every row is a quantised key and value."""
    page, kv, dim, bits = (case[n] for n in ("page", "kv_heads", "dim", "bits"))
    data = torch.empty(blocks, kv, page * (8 + dim * bits // 4), dtype=torch.uint8, device="cuda")
    scale = _scale((2, kv, 1, dim), g)
    step = max(1, 2 ** 26 // (kv * page * dim))
    for at in range(0, blocks, step):
        some = data[at: at + step]
        side = []
        for i, codes in enumerate(_codes(some, page)):
            x = torch.randn(len(some), kv, page, dim, device="cuda", generator=g).mul_(scale[i])
            c, s, m = _quantized(x.to(torch.bfloat16).float(), bits)
            codes.copy_(_packed(c, bits))
            side += [s, m]
        _side(some, page).copy_(torch.stack(side, -1).to(torch.bfloat16).view(torch.uint8))
    return data


def _side(data, page):
    """Scales and lowest values in a cache's bytes: (blocks, Hkv, page, 8)."""
    return data[..., : 8 * page].unflatten(-1, (page, 8))


def _codes(data, page):
    """The key and the value codes in a cache's bytes: (blocks, Hkv, page, D bits / 8) each."""
    half = (data.shape[-1] - 8 * page) // 2
    return [data[..., 8 * page + i * half: 8 * page + (i + 1) * half].unflatten(-1, (page, half // page))
            for i in range(2)]


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    state = dict(case=case)
    if kind == "rotary":
        heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
        n = case["tokens"] + case["padded"]
        type_ = getattr(torch, case["type"])
        qkv = torch.randn(n, (heads + 2 * kv) * dim, device="cuda", generator=g)
        qkv = qkv.mul_(_scale(qkv.shape[1], g)).to(type_)
        state["q"] = qkv[:, : heads * dim].view(n, heads, dim)
        state["k"] = qkv[:, heads * dim: (heads + kv) * dim].view(n, kv, dim)
        first = torch.randint(0, case["far"], (1,), device="cuda", generator=g)
        at = torch.arange(n, device="cuda")
        at = torch.where(at < case["tokens"], (first + at) % case["far"], -1)  # two prompts in a row, then padding
        state["positions"] = at.to(torch.int32)
        pair = torch.arange(case["rotated"] // 2, dtype=torch.float64, device="cuda")
        state["frequencies"] = case["base"] ** (-2 * pair / case["rotated"]) / case["stretch"]
        state["factor"] = 1.0 if case["stretch"] == 1.0 else 0.1 * math.log(case["stretch"]) + 1.0
        return state
    page, kv, dim = case["page"], case["kv_heads"], case["dim"]
    if kind == "attend":
        lens = _lengths(case)
        pages = [-(-n // page) for n in lens]
        blocks = sum(pages) + sum(pages) // 4 + 1
        state["table"] = _table(pages, max(pages), blocks, g)
        state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        q = torch.randn(case["batch"], case["new"], case["heads"], dim, device="cuda", generator=g)
        state["q"] = q.to(torch.bfloat16)
        state["data"] = _filled(blocks, case, g)
        return state
    new = _parts(case["tokens"], case["batch"], g)
    start = torch.randint(0, 8 * page if kind == "append" else 1, (case["batch"],), device="cuda", generator=g)
    pages = ((start + new + page - 1) // page).tolist()
    blocks = case["tokens"] // page + 10 * case["batch"]
    table = _table(pages, max(pages), blocks, g)
    row = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), new)
    at = torch.arange(case["tokens"], device="cuda") - (new.cumsum(0) - new)[row] + start[row]
    slots = (table[row, at // page].long() * page + at % page).to(torch.int32)
    state["data"] = _filled(blocks, case, g)
    if kind == "read":
        return dict(state, slots=slots)
    heads, n = case["heads"], case["tokens"] + case["padded"]
    state["slots"] = torch.cat([slots, torch.full((case["padded"],), -1, dtype=torch.int32, device="cuda")])
    scale = torch.ones((heads + 2 * kv) * dim, device="cuda")
    scale[heads * dim:] = _scale(2 * kv * dim, g)
    qkv = torch.randn(n, (heads + 2 * kv) * dim, device="cuda", generator=g).mul_(scale).to(torch.bfloat16)
    state["k"] = qkv[:, heads * dim: (heads + kv) * dim].view(n, kv, dim)
    state["v"] = qkv[:, (heads + kv) * dim:].view(n, kv, dim)
    return state


# --------------------------------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    kind = case["kind"]
    if own:
        from zipserv_asplos26_amd import attention, paged, rotary
        if kind == "rotary":
            q, k = rotary.apply_rotary(state["q"], state["k"], state["positions"], state["frequencies"],
                                       factor=state["factor"], interleaved=case["interleaved"])
            return dict(q=q, k=k)
        cache = paged.QuantizedKVCache(state["data"], case["page"], case["dim"], case["bits"])
        if kind == "attend":
            out, lse = attention.flash_attn_with_kvcache_quantized(state["q"], cache, state["table"], state["lens"],
                                                                   return_softmax_lse=True)
            return dict(out=out, lse=lse)
        if kind == "append":
            paged.append_paged_kv_quantized(state["k"], state["v"], cache, state["slots"])
        k, v = paged.read_paged_kv_quantized(cache, state["slots"])
        return dict(k=k, v=v)
    if kind == "rotary":
        return dict(q=_rotary(state, state["q"]), k=_rotary(state, state["k"]))
    if kind == "attend":
        return _attend(state)
    if kind == "append":
        _append(state)
    return _read(state)


def _rotary(state, x):
    case = state["case"]
    n, at = case["rotated"], state["positions"]
    angle = at.double()[:, None, None] * state["frequencies"]
    cos, sin = (angle.cos() * state["factor"]).float(), (angle.sin() * state["factor"]).float()
    y = x.float()
    part = y[..., :n]
    if case["interleaved"]:
        a, b = part[..., ::2], part[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = part[..., : n // 2], part[..., n // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    turned = torch.where(at[:, None, None] >= 0, turned, part)  # a token without a place stays as it is
    return torch.cat([turned, y[..., n:]], -1).to(x.dtype)


def _quantized(x, bits):
    """Codes, scales and lowest values of rows (float, D last).  The quotients in 64 bits: many are next to or on the
    border of two scales or two codes."""
    most = 2 ** bits - 1
    low = x.amin(-1)
    scale = (x.amax(-1) - low).double() / most
    scale = ((scale.view(torch.int64) + (1 << 45) - 1) & -1 << 45).view(torch.float64)  # up to 8 significant bits
    code = ((x - low[..., None]).double() / scale[..., None]).round()
    return torch.where(scale[..., None] == 0, 0, code).to(torch.int32), scale.float(), low


def _packed(code, bits):
    """Codes (int32, D last) as bytes."""
    if bits == 8:
        return code.to(torch.uint8)
    c = code.unflatten(-1, (-1, 4, 2))  # channel 8j + 2i + k
    even = c[..., 0, 0] | c[..., 1, 0] << 4 | c[..., 2, 0] << 8 | c[..., 3, 0] << 12
    odd = c[..., 0, 1] | c[..., 1, 1] << 4 | c[..., 2, 1] << 8 | c[..., 3, 1] << 12
    return (even | odd << 16).contiguous().view(torch.uint8)


def _values(codes, scale, low, bits):
    """Rows of code bytes, a scale and a lowest value each, as floats."""
    if bits == 4:
        word = codes.contiguous().view(torch.int32)
        codes = torch.stack([word >> s & 15 for s in (0, 16, 4, 20, 8, 24, 12, 28)], -1).flatten(-2)
    return codes.float() * scale.float()[..., None] + low.float()[..., None]


def _append(state):
    case, data, slots = state["case"], state["data"], state["slots"].long()
    page, bits = case["page"], case["bits"]
    # a padded token does what the first live one does, so that every row is written with one value
    live = slots >= 0
    token = torch.where(live, torch.arange(len(slots), device="cuda"), live.to(torch.int32).argmax())
    at = slots[token]
    block, off = at // page, at % page
    side = []
    for x, codes in zip((state["k"], state["v"]), _codes(data, page)):
        c, s, m = _quantized(x[token].float(), bits)
        codes[block, :, off] = _packed(c, bits)
        side += [s, m]
    _side(data, page)[block, :, off] = torch.stack(side, -1).to(torch.bfloat16).view(torch.uint8)


def _read(state):
    case, data, slots = state["case"], state["data"], state["slots"].long()
    page, live = case["page"], (slots >= 0)[:, None, None]
    at = slots.clamp(min=0)
    block, off = at // page, at % page
    side = _side(data, page)[block, :, off].contiguous().view(torch.bfloat16)
    k, v = (torch.where(live, _values(codes[block, :, off], side[..., 2 * i], side[..., 2 * i + 1], case["bits"]), 0)
            for i, codes in enumerate(_codes(data, page)))
    return dict(k=k.to(torch.bfloat16), v=v.to(torch.bfloat16))


def _attend(state):
    case, lens = state["case"], state["lens"]
    batch, new, heads, dim = state["q"].shape
    page, kv = case["page"], case["kv_heads"]
    data = state["data"][state["table"].long()].transpose(1, 2).contiguous()  # (batch, Hkv, pages, bytes)
    side = _side(data, page).contiguous().view(torch.bfloat16)
    k, v = (_values(codes, side[..., 2 * i], side[..., 2 * i + 1], case["bits"]).flatten(2, 3)
            for i, codes in enumerate(_codes(data, page)))
    q = state["q"].float().view(batch, new, kv, heads // kv, dim).transpose(1, 2).reshape(batch, kv, -1, dim)
    score = torch.matmul(k, q.transpose(2, 3).contiguous()) * (1 / math.sqrt(dim))  # (batch, Hkv, tokens, rows)
    last = lens[:, None] - new + torch.arange(new, device="cuda")  # what each new token sees, up to itself
    hidden = torch.arange(k.shape[2], device="cuda")[:, None] > last.repeat_interleave(heads // kv, 1)[:, None, None]
    score.masked_fill_(hidden, -math.inf)
    most = score.amax(2, keepdim=True)
    weight = (score - torch.where(most == -math.inf, 0, most)).exp()
    total = weight.sum(2, keepdim=True)
    out = torch.matmul(weight.transpose(2, 3).contiguous(), v)
    out = torch.where(total == 0, 0, out.transpose(2, 3) / total).transpose(2, 3)
    lse = (most + total.log())[:, :, 0]

    def rows(x):  # (batch, Hkv, new * group, ...) -> (batch, new, heads, ...)
        return x.view(batch, kv, new, -1, *x.shape[3:]).transpose(1, 2).reshape(batch, new, heads, *x.shape[3:])

    return dict(out=rows(out).to(torch.bfloat16), lse=rows(lse).transpose(1, 2).contiguous())


# --------------------------------------------------------------------------------------------------------------
# What a pass has to move and compute, and its result in 64 bits
# --------------------------------------------------------------------------------------------------------------
def work(case):
    kind, dim, kv = case["kind"], case["dim"], case["kv_heads"]
    if kind == "rotary":
        n, rows = case["tokens"] + case["padded"], case["heads"] + kv
        size = 4 if case["type"] == "float32" else 2
        return {"bytes": n * (4 + 2 * size * rows * dim) + 4 * case["rotated"],
                "flops": 3 * case["tokens"] * rows * case["rotated"]}
    row = 8 + dim * case["bits"] // 4  # a token's key and value of one head, as they are held
    if kind == "read":
        return {"bytes": case["tokens"] * (4 + kv * (row + 4 * dim)), "flops": 4 * case["tokens"] * kv * dim}
    if kind == "append":  # new rows in, held rows out, and what a reader gets of them
        return {"bytes": case["tokens"] * (4 + kv * (row + 8 * dim)) + case["padded"] * (4 + 4 * kv * dim),
                "flops": 12 * case["tokens"] * kv * dim}
    lens, heads, new, batch = _lengths(case), case["heads"], case["new"], case["batch"]
    return {"bytes": sum(lens) * kv * row + sum(4 * -(-n // case["page"]) for n in lens)
            + batch * (4 + new * heads * (4 * dim + 4)), "flops": 4 * sum(lens) * new * heads * dim}


def _exact_rows(data, page, block, off, dim, bits):
    """Keys and values of rows (block[i], off[i]) of all heads, (n, Hkv, D) in 64 bits, channel by channel."""
    width = dim * bits // 8
    if bits == 8:
        byte, shift = list(range(dim)), [0] * dim
    else:  # channel c: half c % 2 of dword c // 8, its nibble c % 8 // 2
        byte = [4 * (c // 8) + 2 * (c % 2) + c % 8 // 4 for c in range(dim)]
        shift = [4 * (c % 4 // 2) for c in range(dim)]
    byte, shift = torch.tensor(byte, device="cuda"), torch.tensor(shift, device="cuda")
    rows = data[block].transpose(0, 1)  # (Hkv, n, bytes)
    out = []
    for i in range(2):
        start = 8 * page + i * page * width + off * width
        code = torch.gather(rows, 2, (start[:, None] + byte).expand(len(rows), -1, -1)).int() >> shift & 2 ** bits - 1
        pair = torch.gather(rows, 2, (8 * off[:, None] + 4 * i + torch.arange(4, device="cuda")).expand(
            len(rows), -1, -1)).long()
        scale, low = ((pair[..., j] << 16 | pair[..., j + 1] << 24).to(torch.int32).view(torch.float32).double()
                      for j in (0, 2))
        out.append((low[..., None] + code.double() * scale[..., None]).transpose(0, 1))
    return out


def exact(case, seed):
    """In 64 bits, sequence by sequence."""
    kind = case["kind"]
    state = prepare(case, seed)
    if kind == "rotary":
        n = case["rotated"]
        turn = torch.polar(torch.full_like(state["positions"], 1.0, dtype=torch.float64)[:, None] * state["factor"],
                           state["positions"].double()[:, None] * state["frequencies"])[:, None]
        result = {}
        for name in ("q", "k"):
            x = state[name].double()
            z = x[..., :n].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
            z = z if case["interleaved"] else z.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
            z = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
            live = state["positions"] >= 0
            y = x.clone()
            y[live, :, :n] = z[live]
            result[name] = y
        return result
    page, dim, bits, kv = case["page"], case["dim"], case["bits"], case["kv_heads"]
    if kind == "read":
        slots = state["slots"].long()
        k, v = _exact_rows(state["data"], page, slots // page, slots % page, dim, bits)
        return dict(k=k, v=v)
    if kind == "append":
        result = {}
        for name in ("k", "v"):
            x = state[name].double()
            low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
            part, power = torch.frexp((high - low).float().double() / (2 ** bits - 1))
            scale = torch.ldexp((part * 256).ceil() / 256, power)
            code = torch.where(scale > 0, ((x - low).float().double() / scale).round(), 0)
            result[name] = torch.where((state["slots"] >= 0)[:, None, None], low + code * scale, 0)
        return result
    batch, new, heads = case["batch"], case["new"], case["heads"]
    group = heads // kv
    out = torch.zeros(batch, new, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((batch, heads, new), -math.inf, dtype=torch.float64, device="cuda")
    for b, length in enumerate(_lengths(case)):
        at = torch.arange(length, device="cuda")
        k, v = _exact_rows(state["data"], page, state["table"][b].long()[at // page], at % page, dim, bits)
        for i in range(new):
            seen = length - new + i + 1
            if seen <= 0:
                continue
            for h in range(kv):
                rows = slice(h * group, (h + 1) * group)
                score = state["q"][b, i, rows].double() @ k[:seen, h].t() / math.sqrt(dim)
                lse[b, rows, i] = torch.logsumexp(score, 1)
                out[b, i, rows] = torch.softmax(score, 1) @ v[:seen, h]
    return dict(out=out, lse=lse)
