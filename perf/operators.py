"""Serving from an appendable paged KV cache, as cases that can be timed and checked.

One decode or prefill step over a pool of pages, from the lengths of its requests to the attention's output, is
four operators:

* plan: block tables, slot maps, positions and lengths of a step from the requests' lengths;
* append: the step's keys and values into their slots, and each page's bounds (the smallest and the largest key of
  each channel) brought up to date;
* select: for each query and KV head, the pages whose bounds allow the largest score;
* attend: decode attention over the selected pages.

A "decode" case is select and attend in a row, the way a layer of a model with a long context uses them.  Keys and
values are N(0, 1) times a log-normal scale per channel, pages are handed out in a random order.
"""
import math

import torch

own = False


def listed():
    return [
        # One user's next token: the smallest call, nothing but latency.
        dict(name="plan_b1", kind="plan", batch=1, prefills=0, prefill_tokens=0, context=1000, page=16, padded=7),
        # A step of a large server: most requests decode, some bring a chunk of their prompt.
        dict(name="plan_b300_mixed", kind="plan", batch=300, prefills=24, prefill_tokens=1000, context=20000, page=16,
             padded=100),
        # A decode step's new keys and values, as slices of the fused projection's output.
        dict(name="append_b32", kind="append", batch=32, tokens=32, heads=32, kv_heads=8, dim=128, page=16, padded=0),
        # A prefill chunk of a few requests with ragged lengths, in a padded batch.
        dict(name="append_t8000", kind="append", batch=5, tokens=8000, heads=32, kv_heads=8, dim=128, page=16,
             padded=192),
        # Small heads in large pages.
        dict(name="append_d64_t3001", kind="append", batch=3, tokens=3001, heads=16, kv_heads=16, dim=64, page=128,
             padded=0),
        # One user with a long context: few rows, so latency and the spread over the chip.
        dict(name="select_b1_t32k", kind="select", batch=1, tokens=32000, ragged=False, heads=32, kv_heads=8, dim=128,
             page=16, top_k=128),
        # A batch of long ragged contexts: the bounds' bytes from HBM.
        dict(name="select_b32_t64k", kind="select", batch=32, tokens=64000, ragged=True, heads=64, kv_heads=8, dim=128,
             page=16, top_k=256),
        # One user's selected pages.
        dict(name="attend_b1_k128", kind="attend", batch=1, tokens=16000, ragged=False, heads=32, kv_heads=8, dim=128,
             page=16, top_k=128),
        # A large batch whose selected pages come from HBM.
        dict(name="attend_b64_k256", kind="attend", batch=64, tokens=8000, ragged=False, heads=64, kv_heads=8, dim=128,
             page=16, top_k=256),
        # Small heads without groups, ragged contexts, some shorter than what may be selected.
        dict(name="attend_d64_mha_b20", kind="attend", batch=20, tokens=5001, ragged=True, heads=16, kv_heads=16,
             dim=64, page=32, top_k=50),
        # One user with a very long context, both operators.
        dict(name="decode_b1_t128k", kind="decode", batch=1, tokens=131000, ragged=False, heads=32, kv_heads=8,
             dim=128, page=16, top_k=256),
        # A serving batch of ragged long contexts in larger pages, both operators.
        dict(name="decode_b16_t40k", kind="decode", batch=16, tokens=40000, ragged=True, heads=64, kv_heads=8, dim=128,
             page=64, top_k=64),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["plan", "append", "select", "attend", "decode"])
    if kind == "plan":
        batch = _spread(rng, 1, 600)
        prefills = rng.randint(0, min(batch, 24))
        return dict(kind=kind, batch=batch, prefills=prefills,
                    prefill_tokens=_spread(rng, 2, 1000) if prefills else 0, context=_spread(rng, 1, 20000),
                    page=rng.choice([16, 32, 64, 128]), padded=rng.randint(0, 100))
    heads, kv_heads = rng.choice([(32, 8), (64, 8), (16, 16), (8, 1), (28, 4), (40, 8), (16, 2), (32, 2)])
    dim = rng.choice([128, 128, 64])
    if kind == "append":
        tokens = _spread(rng, 1, 8000 * 8 // max(8, kv_heads))
        return dict(kind=kind, batch=min(tokens, _spread(rng, 1, 64)), tokens=tokens, heads=heads, kv_heads=kv_heads,
                    dim=dim, page=rng.choice([16, 32, 64, 128]), padded=rng.choice([0, 0, rng.randint(1, 100)]))
    page = rng.choice([16, 16, 32, 64])
    batch = _spread(rng, 1, 48)
    # at most 4 M (page, head) bounds and 1.5 M (token, head) rows a cache
    most = 400_000 // (batch * kv_heads) * page if kind == "select" else 2_000_000 // (batch * kv_heads)
    tokens = _spread(rng, 40, max(100, min(100_000, most)))
    top_k = _spread(rng, 2, max(3, min(512, 16_000_000 // (batch * heads * page), tokens // page)))
    return dict(kind=kind, batch=batch, tokens=tokens, ragged=rng.random() < 0.5, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, top_k=top_k)


# --------------------------------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lengths(case):
    """Cached tokens of each sequence: all, or spread evenly up to all."""
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


def _table(pages, width, g, pool=None):
    """A block table (rows of `width`) that gives row b its pages[b] pages in a random order, and the free ones:
    a quarter more than those in use, or what is left of `pool`."""
    total = sum(pages)
    order = torch.randperm(pool or total + total // 4 + 1, device="cuda", generator=g).to(torch.int32)
    held = torch.arange(width, device="cuda") < torch.tensor(pages, device="cuda")[:, None]
    table = torch.zeros(len(pages), width, dtype=torch.int32, device="cuda")
    table[held] = order[:total]
    return table, order[total:].contiguous()


def _cache(blocks, case, g):
    shape = (blocks, case["page"], case["kv_heads"], case["dim"])
    scale = torch.randn(shape[2:], device="cuda", generator=g).exp_().to(torch.bfloat16)
    return torch.randn(shape, device="cuda", generator=g, dtype=torch.bfloat16).mul_(scale)


def _bounds(k_cache):
    """(blocks, kv_heads, 2, dim): the smallest and the largest key of each page's channels."""
    return torch.stack([k_cache.amin(1), k_cache.amax(1)], 2)


def _plan_inputs(case, g):
    batch, page = case["batch"], case["page"]
    context = torch.randint(0, case["context"] + 1, (batch,), device="cuda", generator=g)
    new = torch.ones(batch, dtype=torch.int64, device="cuda")
    if case["prefills"]:
        who = torch.randperm(batch, device="cuda", generator=g)[: case["prefills"]]
        new[who] = torch.randint(1, case["prefill_tokens"] + 1, (case["prefills"],), device="cuda", generator=g)
    held = ((context + page - 1) // page).tolist()
    width = (case["context"] + max(1, case["prefill_tokens"])) // page + 2
    table, free = _table(held, width, g)
    need = sum(-(-(c + n) // page) for c, n in zip(context.tolist(), new.tolist())) - sum(held)
    more = torch.arange(need, device="cuda", dtype=torch.int32) + (sum(held) + len(free))  # never short of pages
    free = torch.cat([free, more])
    return dict(context=context.to(torch.int32), new=new.to(torch.int32), table=table, free=free,
                num_free=_ints([len(free)]),
                max_tokens=batch + case["prefills"] * case["prefill_tokens"] + case["padded"])


def _append_inputs(case, g):
    page, heads, kv, dim = case["page"], case["heads"], case["kv_heads"], case["dim"]
    new = _parts(case["tokens"], case["batch"], g)
    start = torch.randint(0, 8 * page, (case["batch"],), device="cuda", generator=g)
    pages = ((start + new + page - 1) // page).tolist()
    blocks = case["tokens"] // page + 10 * case["batch"]
    table, _ = _table(pages, max(pages), g, blocks)
    row = torch.repeat_interleave(torch.arange(case["batch"], device="cuda"), new)
    at = torch.arange(case["tokens"], device="cuda") - (new.cumsum(0) - new)[row] + start[row]
    slots = table[row, at // page].long() * page + at % page
    n = case["tokens"] + case["padded"]
    slots = torch.cat([slots, torch.full((case["padded"],), -1, device="cuda")]).to(torch.int32)
    scale = torch.ones((heads + 2 * kv) * dim, device="cuda")
    scale[heads * dim:] = torch.randn(2 * kv * dim, device="cuda", generator=g).exp_()
    qkv = torch.randn(n, (heads + 2 * kv) * dim, device="cuda", generator=g).mul_(scale).to(torch.bfloat16)
    k = qkv[:, heads * dim: (heads + kv) * dim].view(n, kv, dim)
    v = qkv[:, (heads + kv) * dim:].view(n, kv, dim)
    k_cache, v_cache = _cache(blocks, case, g), _cache(blocks, case, g)
    return dict(k=k, v=v, k_cache=k_cache, v_cache=v_cache, slots=slots, bounds=_bounds(k_cache))


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    state = dict(case=case)
    if kind == "plan":
        return dict(state, **_plan_inputs(case, g))
    if kind == "append":
        return dict(state, **_append_inputs(case, g))
    lens = _lengths(case)
    pages = [-(-n // case["page"]) for n in lens]
    state["table"], free = _table(pages, max(pages), g)
    blocks = sum(pages) + len(free)
    state["lens"] = _ints(lens)
    state["q"] = torch.randn(case["batch"], case["heads"], case["dim"], device="cuda", generator=g).to(torch.bfloat16)
    if kind == "select":  # the bounds of pages of 16 keys, without the keys
        shape = (blocks, case["kv_heads"], case["dim"])
        scale = torch.randn(shape[1:], device="cuda", generator=g).exp_()
        mid = torch.randn(shape, device="cuda", generator=g).mul_(0.5)
        half = torch.rand(shape, device="cuda", generator=g).add_(1.0)
        state["bounds"] = torch.stack([(mid - half) * scale, (mid + half) * scale], 2).to(torch.bfloat16)
        return state
    state["k_cache"], state["v_cache"] = _cache(blocks, case, g), _cache(blocks, case, g)
    if kind == "decode":
        state["bounds"] = _bounds(state["k_cache"])
        return state
    # any selection: a random choice of each sequence's pages, in ascending order, all where there are few
    width = max(pages)
    rank = torch.rand(case["batch"], case["kv_heads"], width, device="cuda", generator=g)
    rank.masked_fill_(torch.arange(width, device="cuda") >= torch.tensor(pages, device="cuda")[:, None, None], 2.0)
    value, index = rank.topk(min(case["top_k"], width), largest=False)
    index = index.masked_fill(value == 2.0, width).sort().values
    chosen = torch.full((case["batch"], case["kv_heads"], case["top_k"]), -1, dtype=torch.int32, device="cuda")
    chosen[..., : index.shape[-1]] = index.masked_fill(index == width, -1).to(torch.int32)
    state["pages"] = chosen
    return state


# --------------------------------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------------------------------
def run(state):
    kind, page = state["case"]["kind"], state["case"]["page"]
    if own:
        from zipserv_asplos26_amd import attention, paged
        if kind == "plan":
            p = paged.plan_paged_step(state["context"], state["new"], state["table"], state["free"],
                                      state["num_free"], page, state["max_tokens"])
            return dict(table=state["table"], slots=p.slots, sequences=p.sequences, positions=p.positions,
                        seqlens=p.seqlens, cu_new=p.cu_new, counts=p.counts)
        if kind == "append":
            paged.append_paged_kv(state["k"], state["v"], state["k_cache"], state["v_cache"], state["slots"],
                                  state["bounds"])
            return dict(k_cache=state["k_cache"], v_cache=state["v_cache"], bounds=state["bounds"])
        pages = state.get("pages")
        if pages is None:
            pages = paged.select_kv_pages(state["q"], state["bounds"], state["table"], state["lens"], page,
                                          state["case"]["top_k"])
        if kind == "select":
            return dict(pages=pages)
        out, lse = attention.flash_attn_with_kvcache_sparse(state["q"], state["k_cache"], state["v_cache"],
                                                            state["table"], pages, state["lens"],
                                                            return_softmax_lse=True)
        return dict(pages=pages, out=out, lse=lse)
    if kind == "plan":
        return _plan(state, page)
    if kind == "append":
        return _append(state, page)
    pages = state.get("pages")
    if pages is None:
        pages = _select(state, page, state["case"]["top_k"])
    if kind == "select":
        return dict(pages=pages)
    out, lse = _attend(state, pages, page)
    return dict(pages=pages, out=out, lse=lse)


def _plan(state, page):
    context, new, table, most = state["context"].long(), state["new"].long(), state["table"], state["max_tokens"]
    batch = len(context)
    ends = new.cumsum(0)
    asked = ends[-1:]
    ends = ends.clamp(max=most)
    first = torch.cat([torch.zeros_like(asked), ends[:-1]])
    new = ends - first
    held = (context + page - 1) // page
    more = (context + new + page - 1) // page - held
    given = more.cumsum(0)
    at = torch.arange(most, device="cuda")
    row = torch.searchsorted(ends, at, right=True)
    live = row < batch
    row = row.clamp(max=batch - 1)
    pos = torch.where(live, at - first[row] + context[row], 0)  # behind the last token: a place that exists
    fresh = pos // page - held[row]  # of the sequence's new pages the how-manieth; below 0: it had it already
    number = (given - more)[row] + fresh
    stack = state["free"][(state["num_free"] - 1 - number).clamp(min=0, max=len(state["free"]) - 1)]
    entry = torch.where(fresh >= 0, stack, table[row, pos // page])
    starts = live & (fresh >= 0) & (pos % page == 0)
    place = torch.where(starts, row * table.shape[1] + pos // page, table.numel())  # a new page's first token sets its entry
    table.copy_(torch.cat([table.view(-1), entry[:1]]).scatter(0, place, entry)[:-1].view_as(table))
    none = torch.full_like(at, -1)
    whole = lambda x: torch.where(live, x, none).to(torch.int32)  # noqa: E731
    taken = given[-1:]
    return dict(table=table, slots=whole(entry.long() * page + pos % page), sequences=whole(row),
                positions=whole(pos), seqlens=(context + new).to(torch.int32),
                cu_new=torch.cat([first, ends[-1:]]).to(torch.int32),
                counts=torch.cat([asked, taken, taken - taken, state["num_free"] - taken]).to(torch.int32))


def _append(state, page):
    slots, bounds = state["slots"].long(), state["bounds"]
    # a padded token does what the first live one does, so that every row is written with one value
    live = slots >= 0
    token = torch.where(live, torch.arange(len(slots), device="cuda"), live.to(torch.int32).argmax())
    at, k = slots[token], state["k"][token]
    state["k_cache"].view(-1, *k.shape[1:])[at] = k
    state["v_cache"].view(-1, *k.shape[1:])[at] = state["v"][token]
    low, high = bounds.float().unbind(2)
    opened = torch.zeros(len(bounds) * page, dtype=torch.bool, device="cuda").index_fill_(0, at, True)[::page]
    low = low.masked_fill(opened[:, None, None], math.inf)
    high = high.masked_fill(opened[:, None, None], -math.inf)
    index, k = (at // page)[:, None, None].expand(k.shape), k.float()
    bounds.copy_(torch.stack([low.scatter_reduce(0, index, k, "amin"), high.scatter_reduce(0, index, k, "amax")], 2))
    return dict(k_cache=state["k_cache"], v_cache=state["v_cache"], bounds=bounds)


def _select(state, page, top_k):
    q, table, lens = state["q"].double(), state["table"], state["lens"]
    batch, heads, dim = q.shape
    kv = state["bounds"].shape[1]
    width = table.shape[1]
    q = q.view(batch, kv, heads // kv, dim)
    sides = torch.cat([q.clamp(max=0.0), q.clamp(min=0.0)], 3)
    reach = state["bounds"][table.long()].view(batch, width, kv, 2 * dim).transpose(1, 2).double()
    score = torch.matmul(reach, sides.transpose(2, 3).contiguous()).amax(3)
    index = torch.arange(width, device="cuda")
    count = ((lens + page - 1) // page)[:, None, None]
    score.masked_fill_((index == 0) | (index == count - 1), math.inf)
    score.masked_fill_(index >= count, -math.inf)
    best = score.sort(descending=True, stable=True).indices[..., :top_k]
    best = best.masked_fill(best >= count, width).sort().values
    best = best.masked_fill(best == width, -1).to(torch.int32)
    rest = torch.full((batch, kv, top_k - best.shape[2]), -1, dtype=torch.int32, device="cuda")
    return torch.cat([best, rest], 2)


def _attend(state, pages, page):
    q, table, lens = state["q"].float(), state["table"], state["lens"]
    batch, heads, dim = q.shape
    kv, top_k = pages.shape[1:]
    at = pages.long().clamp(min=0)
    block = torch.gather(table.long()[:, None, :].expand(-1, kv, -1), 2, at)
    head = torch.arange(kv, device="cuda")[:, None]
    k = state["k_cache"][block, :, head].view(batch, kv, top_k * page, dim).float()
    token = at[..., None] * page + torch.arange(page, device="cuda")
    hidden = (token >= lens[:, None, None, None]) | (pages < 0)[..., None]
    score = torch.matmul(k, q.view(batch, kv, heads // kv, dim).transpose(2, 3).contiguous()) * (1 / math.sqrt(dim))
    score.masked_fill_(hidden.view(batch, kv, -1, 1), -math.inf)
    most = score.amax(2, keepdim=True)
    weight = (score - most).exp()
    total = weight.sum(2, keepdim=True)
    v = state["v_cache"][block, :, head].view(batch, kv, top_k * page, dim).float()
    out = torch.matmul(weight.transpose(2, 3).contiguous(), v) / total.transpose(2, 3)
    lse = (most + total.log()).view(batch, heads)
    return out.view(batch, heads, dim).to(torch.bfloat16), lse


# --------------------------------------------------------------------------------------------------------------
# What a pass has to move and compute, and its result in 64 bits
# --------------------------------------------------------------------------------------------------------------
def work(case):
    kind, page, batch = case["kind"], case["page"], case["batch"]
    if kind == "plan":
        tokens = batch + case["prefills"] * max(0, case["prefill_tokens"] - 1) // 2
        rows = batch + case["prefills"] * case["prefill_tokens"] + case["padded"]
        # lengths in and out, three values a row of the step, a free page into the table for each page of new tokens
        return {"bytes": 16 * batch + 12 * rows + 8 * tokens / page, "flops": 0}
    kv, dim = case["kv_heads"], case["dim"]
    if kind == "append":
        tokens = case["tokens"]
        touched = tokens / page + batch
        return {"bytes": tokens * (4 + 8 * kv * dim) + touched * 6 * kv * dim, "flops": 2 * tokens * kv * dim}
    heads, lens = case["heads"], _lengths(case)
    ends = 2 * batch * heads * dim
    pages = [-(-n // page) for n in lens]
    scan = sum(pages) * (4 * kv * dim + 4) + ends + 4 * batch * kv * case["top_k"]
    chosen = sum(min(n, p * page) for n, p in ((n, min(p, case["top_k"])) for n, p in zip(lens, pages)))
    read = 4 * chosen * kv * dim + 2 * ends + 4 * batch * heads + 4 * batch * kv * case["top_k"]
    bytes_ = (scan if kind != "attend" else 0) + (read if kind != "select" else 0)
    flops = (4 * sum(pages) * heads * dim if kind != "attend" else 0) + (4 * chosen * heads * dim if kind != "select" else 0)
    return {"bytes": bytes_, "flops": flops}


def exact(case, seed):
    """In 64 bits, sequence by sequence.  The plan's and the selection's whole numbers are left to the comparison."""
    kind, page = case["kind"], case["page"]
    if kind in ("plan", "select"):
        return None
    state = prepare(case, seed)
    if kind == "append":
        k, v, slots = state["k"].double(), state["v"].double(), state["slots"].tolist()
        k_cache, v_cache, bounds = state["k_cache"].double(), state["v_cache"].double(), state["bounds"].double()
        groups = {}
        for i, s in enumerate(slots):
            if s >= 0:
                groups.setdefault(s // page, []).append(i)
        for block, rows in groups.items():
            offsets = [slots[i] % page for i in rows]
            k_cache[block, offsets], v_cache[block, offsets] = k[rows], v[rows]
            fresh = k[rows]
            if 0 not in offsets:
                fresh = torch.cat([fresh, bounds[block].transpose(0, 1)])
            bounds[block, :, 0], bounds[block, :, 1] = fresh.min(0).values, fresh.max(0).values
        return dict(k_cache=k_cache, v_cache=v_cache, bounds=bounds)
    batch, heads, dim, kv = case["batch"], case["heads"], case["dim"], case["kv_heads"]
    group = heads // kv
    out = torch.zeros(batch, heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.zeros(batch, heads, dtype=torch.float64, device="cuda")
    chosen = state.get("pages")
    for b, length in enumerate(_lengths(case)):
        table = state["table"][b, : -(-length // page)].long()
        for h in range(kv):
            q = state["q"][b, h * group: (h + 1) * group].double()
            if chosen is None:
                low, high = state["bounds"][table, h].double().unbind(1)
                score = torch.maximum(q[:, None] * low, q[:, None] * high).sum(2).max(0).values
                score[0] = score[-1] = math.inf
                mine = score.sort(descending=True, stable=True).indices[: case["top_k"]].sort().values
            else:
                mine = chosen[b, h].long()
                mine = mine[mine >= 0]
            token = (mine[:, None] * page + torch.arange(page, device="cuda")).view(-1)
            seen = token < length
            k = state["k_cache"][table[mine], :, h].reshape(-1, dim)[seen].double()
            v = state["v_cache"][table[mine], :, h].reshape(-1, dim)[seen].double()
            score = q @ k.t() / math.sqrt(dim)
            rows = slice(h * group, (h + 1) * group)
            lse[b, rows] = torch.logsumexp(score, 1)
            out[b, rows] = torch.softmax(score, 1) @ v
    return dict(pages=None, out=out, lse=lse)
