"""Plan, append and selection over an appendable paged KV cache against plain
references: whole numbers and copies bit for bit."""
import random

import pytest

import paged_testutil as ref
from zipserv_asplos26_amd import attention, paged

pytestmark = pytest.mark.gpu


def ints(torch, x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------------------
# Plan
# ------------------------------------------------------------------------------------------------------------
def check_plan(torch, context, new, table, free, num_free, page, most, view=None):
    want = ref.plan(context, new, table, free, num_free, page, most)
    dev = ints(torch, table) if view is None else view
    p = paged.plan_paged_step(ints(torch, context), ints(torch, new), dev, ints(torch, free), ints(torch, [num_free]),
                              page, most)
    got = [dev, p.slots, p.sequences, p.positions, p.seqlens, p.cu_new, p.counts]
    for name, g, w in zip(("table", "slots", "sequences", "positions", "seqlens", "cu_new", "counts"), got, want):
        assert g.cpu().tolist() == w, name
    assert p.num_free.tolist() == [want[-1][3]]
    return want


@pytest.mark.parametrize("page,batch,most_new,context,extra", [
    (16, 1, 1, 0, 0), (16, 1, 1, 15, 3), (16, 1, 40, 16, 0), (32, 7, 70, 100, 9), (48, 64, 1, 500, 0),
    (16, 255, 3, 60, 1), (16, 256, 20, 60, 0), (128, 257, 300, 1000, 5), (16, 4096, 2, 40, 17)])
def test_plan(torch_cuda, page, batch, most_new, context, extra):
    rng = random.Random(page * batch + most_new)
    ctx = [rng.randint(0, context) for _ in range(batch)]
    new = [rng.choice([0, 1, rng.randint(0, most_new)]) for _ in range(batch)]
    width = (context + most_new) // page + 2
    held = [-(-c // page) for c in ctx]
    blocks = list(range(sum(held) + sum(new) + batch))
    rng.shuffle(blocks)
    table = [[0] * width for _ in range(batch)]
    for b, n in enumerate(held):
        for i in range(n):
            table[b][i] = blocks.pop()
    want = check_plan(torch_cuda, ctx, new, table, blocks, len(blocks), page, sum(new) + extra)
    assert want[-1][2] == 0


def test_plan_without_room(torch_cuda):
    # too few free pages, a full row, more tokens than the buffers hold, lengths below zero, a count of free
    # pages past the list's end or below zero, a missing page of the context
    T = torch_cuda
    table = [[1, 2, 0, 0], [3, 4, 5, 6], [0, 0, 0, 0], [7, -1, 0, 0]]
    check_plan(T, [20, 60, 0, 17], [50, 10, 100, 3], table, [20, 21, 22], 3, 16, 200)
    check_plan(T, [20, 60, 0, 17], [50, 10, 100, 3], table, [20, 21, 22, 23, 24, 25, 26, 27, 28], 9, 16, 55)
    check_plan(T, [20, 60, 0, 17], [50, 10, 100, 3], table, list(range(20, 60)), 99, 16, 0)
    check_plan(T, [-5, 64, 500, 0], [-3, 1, 20, -1], table, [20, 21], 5, 16, 30)
    check_plan(T, [5, 0, 0, 0], [20, 0, 0, 1], table, [20, 21], -4, 16, 30)
    check_plan(T, [5, 0, 0, 0], [20, 0, 0, 1], table, [], 0, 16, 30)
    check_plan(T, [5, 0, 0, 0], [0, 0, 0, 0], table, [9], 1, 16, 0)


def test_plan_lengths_past_32_bits(torch_cuda):
    # sums past 2^31 saturate or are cut; nothing is written outside the buffers
    T = torch_cuda
    big = 2 ** 31 - 1
    p = paged.plan_paged_step(ints(T, [0, big, 3]), ints(T, [big, big, big]), ints(T, [[0, 0]] * 3), ints(T, [4, 5]),
                              ints(T, [2]), 16, 40)
    assert p.counts.tolist() == [big, 2, 1, 0] and p.cu_new.tolist() == [0, 40, 40, 40]
    assert p.seqlens.tolist() == [32, big, 3]
    assert p.slots.tolist() == list(range(80, 96)) + list(range(64, 80)) + [-1] * 8
    assert p.positions.tolist() == list(range(40))


def test_plan_of_a_wider_table(torch_cuda):
    # rows of a larger table: what stands beside them stays
    T = torch_cuda
    whole = T.full((3, 9), -7, dtype=T.int32, device="cuda")
    whole[:, 2:6] = 0
    check_plan(T, [0, 0, 0], [20, 0, 33], [[0] * 4] * 3, [1, 2, 3, 4, 5, 6], 6, 16, 60, view=whole[:, 2:6])
    assert (whole[:, :2] == -7).all() and (whole[:, 6:] == -7).all()
    for bad in (T.zeros(4, 2, dtype=T.int32, device="cuda").t(), ints(T, [[1, 2]]).expand(2, 2)):
        with pytest.raises(ValueError, match="in place"):
            paged.plan_paged_step(ints(T, [0, 0]), ints(T, [0, 0]), bad, ints(T, [1]), ints(T, [1]), 16, 4)


def test_plan_refuses(torch_cuda):
    T = torch_cuda
    i2, t2 = ints(T, [1, 1]), ints(T, [[0, 0]] * 2)
    for bad in [dict(new=ints(T, [1])), dict(new=i2.long()), dict(table=ints(T, [[0, 0]])), dict(num=i2),
                dict(new=i2.cpu()), dict(most=-1), dict(context=T.zeros(4, dtype=T.int32, device="cuda")[::2])]:
        a = {**dict(context=i2, new=i2, table=t2, free=i2, num=ints(T, [2]), most=4), **bad}
        with pytest.raises(ValueError):
            paged.plan_paged_step(a["context"], a["new"], a["table"], a["free"], a["num"], 16, a["most"])


# ------------------------------------------------------------------------------------------------------------
# Append
# ------------------------------------------------------------------------------------------------------------
def bits(torch, x):
    return x.detach().cpu().view(torch.int16)


def same(torch, a, b):
    """Equal bits, or both not a number."""
    a, b = a.detach().cpu(), b.detach().cpu()
    return bool(((bits(torch, a) == bits(torch, b)) | (a.isnan() & b.isnan()) | ((a == 0) & (b == 0))).all())


def run_slots(rng, blocks, page, runs):
    """Slots of `runs` (offset, tokens) pieces, each in pages of its own."""
    order = list(range(blocks))
    rng.shuffle(order)
    slots = []
    for offset, tokens in runs:
        block = order.pop()
        for _ in range(tokens):
            slots.append(block * page + offset)
            offset += 1
            if offset == page:
                block, offset = order.pop(), 0
    return slots


@pytest.mark.parametrize("heads_k,dim,page,runs,tail", [
    (8, 128, 16, [(0, 1)], 0), (8, 128, 16, [(15, 1), (3, 1), (0, 1)], 2), (8, 128, 16, [(5, 40), (0, 16), (9, 7)], 0),
    (1, 64, 16, [(5, 40), (0, 33), (9, 7)], 70), (16, 64, 128, [(100, 300), (0, 128), (1, 1)], 0),
    (2, 128, 64, [(63, 130)], 1), (3, 128, 48, [(0, 48), (47, 1), (46, 2), (20, 60)], 0),
    (5, 64, 256, [(250, 520), (0, 1), (17, 239)], 5), (1, 128, 1040, [(1000, 2200), (3, 900)], 0),
    (8, 128, 16, [(i % 16, 1) for i in range(65)], 0)])
@pytest.mark.parametrize("with_bounds", [True, False])
def test_append(torch_cuda, heads_k, dim, page, runs, tail, with_bounds):
    T = torch_cuda
    rng = random.Random(dim + page)
    g = T.Generator().manual_seed(len(runs))
    blocks = sum(n // page + 3 for _, n in runs)
    slots = run_slots(rng, blocks, page, runs) + [-1] * tail
    n = len(slots)
    # k and v as slices of a fused projection
    qkv = T.randn(n, (4 + 2 * heads_k) * dim, generator=g).to(T.bfloat16).cuda()
    k = qkv[:, 4 * dim:(4 + heads_k) * dim].view(n, heads_k, dim)
    v = qkv[:, (4 + heads_k) * dim:].view(n, heads_k, dim)
    kc, vc = (T.randn(blocks, page, heads_k, dim, generator=g).to(T.bfloat16) for _ in range(2))
    bounds = T.stack([kc.amin(1), kc.amax(1)], 2) if with_bounds else None
    if with_bounds:  # a page that has never been written to may hold anything
        for i, s in enumerate(slots):
            if s >= 0 and s % page == 0:
                bounds[s // page] = float("nan")
    dev = [kc.cuda(), vc.cuda(), bounds.cuda() if with_bounds else None]
    paged.append_paged_kv(k, v, dev[0], dev[1], ints(T, slots), dev[2])
    ref.append(k.cpu(), v.cpu(), kc, vc, T.tensor(slots), bounds)
    assert T.equal(bits(T, dev[0]), bits(T, kc)) and T.equal(bits(T, dev[1]), bits(T, vc))
    if with_bounds:
        assert same(T, dev[2], bounds)


@pytest.mark.parametrize("dim", [64, 128])
def test_append_values_that_are_no_numbers(torch_cuda, dim):
    # NaNs are no bound, infinities are; every bit pattern is copied
    T = torch_cuda
    g = T.Generator().manual_seed(3)
    k, v = (T.randint(-32768, 32768, (50, 2, dim), generator=g, dtype=T.int16).view(T.bfloat16) for _ in range(2))
    k[20:30] = T.randn(10, 2, dim, generator=g).to(T.bfloat16)
    k[20:30, :, ::3] = float("nan")
    k[25, :, 1::3] = float("inf")
    kc, vc = (T.zeros(6, 16, 2, dim, dtype=T.bfloat16) for _ in range(2))
    bounds = T.zeros(6, 2, 2, dim, dtype=T.bfloat16)
    slots = list(range(16, 36)) + list(range(64, 74)) + list(range(2, 14)) + [90, 91, 92, 93, 94, 95, -1, 96]
    dev = [x.cuda() for x in (kc, vc, bounds)]
    paged.append_paged_kv(k.cuda(), v.cuda(), dev[0], dev[1], ints(T, slots), dev[2])
    ref.append(k, v, kc, vc, T.tensor(slots), bounds)
    assert T.equal(bits(T, dev[0]), bits(T, kc)) and T.equal(bits(T, dev[1]), bits(T, vc))
    assert same(T, dev[2], bounds)


def test_append_skips_slots_outside_the_pool(torch_cuda):
    T = torch_cuda
    kc, vc = (T.zeros(2, 16, 1, 64, dtype=T.bfloat16, device="cuda") for _ in range(2))
    bounds = T.zeros(2, 1, 2, 64, dtype=T.bfloat16, device="cuda")
    x = T.ones(5, 1, 64, dtype=T.bfloat16, device="cuda")
    paged.append_paged_kv(x, x, kc, vc, ints(T, [-1, 32, 2 ** 31 - 1, -2 ** 31, 31]), bounds)
    assert kc.sum() == 64 and (kc[1, 15] == 1).all() and vc.sum() == 64
    assert bounds[0].sum() == 0 and bounds[1, 0, 1].sum() == 64 and bounds[1, 0, 0].sum() == 0
    paged.append_paged_kv(x[:0], x[:0], kc, vc, ints(T, []), bounds)


@pytest.mark.parametrize("how", ["offset", "transposed", "last"])
def test_append_of_other_strides(torch_cuda, how):
    # rows that are not 16-byte pieces of contiguous heads
    T = torch_cuda
    x = T.randn(9, 2, 72, device="cuda").to(T.bfloat16)
    k = {"offset": x[..., 3:67], "transposed": x[..., :64].transpose(0, 1).contiguous().transpose(0, 1),
         "last": T.randn(9, 64, 2, device="cuda").to(T.bfloat16).transpose(1, 2)}[how]
    kc, vc = (T.zeros(2, 16, 2, 64, dtype=T.bfloat16, device="cuda") for _ in range(2))
    paged.append_paged_kv(k, k, kc, vc, ints(T, range(4, 13)))
    flat = kc.view(32, 2, 64)
    assert T.equal(flat[4:13], k) and T.equal(vc, kc) and flat[:4].abs().sum() + flat[13:].abs().sum() == 0


def test_append_refuses(torch_cuda):
    T = torch_cuda
    kc = T.zeros(2, 16, 2, 64, dtype=T.bfloat16, device="cuda")
    x, s = T.zeros(3, 2, 64, dtype=T.bfloat16, device="cuda"), ints(T, [0, 1, 2])
    b = T.zeros(2, 2, 2, 64, dtype=T.bfloat16, device="cuda")
    for args in [(x[:2], x, kc, kc, s), (x, x.float(), kc, kc, s), (x, x, kc, kc[:1], s), (x, x, kc[:, ::2], kc, s),
                 (x, x, kc, kc, s.long()), (x, x, kc, kc, s, b[:1]), (x, x, kc, kc, s, b.float()),
                 (x[..., :32], x, kc, kc, s), (x.cpu(), x, kc, kc, s)]:
        with pytest.raises(ValueError):
            paged.append_paged_kv(*args)


# ------------------------------------------------------------------------------------------------------------
# Selection
# ------------------------------------------------------------------------------------------------------------
def make_select(T, seed, batch, heads, heads_k, dim, page, width, spread=1.0):
    g = T.Generator().manual_seed(seed)
    blocks = batch * width + 3
    table = T.randperm(blocks, generator=g)[:batch * width].view(batch, width).to(T.int32)
    keys = T.randn(blocks, 4, heads_k, dim, generator=g).mul_(T.randn(heads_k, dim, generator=g).mul(spread).exp())
    keys = keys.to(T.bfloat16)
    bounds = T.stack([keys.amin(1), keys.amax(1)], 2)
    q = T.randn(batch, heads, dim, generator=g).to(T.bfloat16)
    return q, bounds, table


def check_select(T, q, bounds, table, lens, page, top_k, **kw):
    got = paged.select_kv_pages(q.cuda(), bounds.cuda(), table.cuda(), ints(T, lens), page, top_k, **kw)
    want = ref.select(q, bounds, table, lens, page, top_k, kw.get("sink_pages", 1), kw.get("local_pages", 1))
    assert T.equal(got.cpu(), want)
    return want


@pytest.mark.parametrize("heads,heads_k,dim,page,width,top_k,sink,local", [
    (8, 8, 128, 16, 40, 5, 1, 1), (32, 8, 128, 16, 300, 20, 1, 1), (64, 8, 64, 16, 70, 7, 0, 0),
    (16, 1, 128, 32, 33, 32, 4, 4), (28, 4, 64, 48, 90, 1, 0, 1), (5, 5, 128, 16, 20, 2, 2, 0),
    (40, 8, 128, 64, 257, 64, 1, 3), (2, 2, 64, 16, 3, 8, 1, 1), (30, 2, 128, 256, 65, 3, 0, 0), (16, 1, 64, 1040, 40, 6, 1, 2),
    (3, 3, 128, 16, 2100, 30, 1, 1), (4, 2, 64, 16, 4200, 9, 0, 1)])
def test_select(torch_cuda, heads, heads_k, dim, page, width, top_k, sink, local):
    T = torch_cuda
    most = width * page
    lens = [most, 0, 1, page, page + 1, (top_k + 1) * page, min(most, top_k * page), most - 1, most + 5 * page]
    q, bounds, table = make_select(T, width, len(lens), heads, heads_k, dim, page, width)
    check_select(T, q, bounds, table, lens, page, top_k, sink_pages=sink, local_pages=local)


@pytest.mark.parametrize("top_k", [1, 3, 64, 299])
def test_select_ties_go_to_the_lowest_page(torch_cuda, top_k):
    # equal bounds everywhere; a few distinct values; 0 and -0; values whose sums cancel
    T = torch_cuda
    q, bounds, table = make_select(T, 5, 4, 8, 2, 64, 16, 300)
    b = bounds.clone()
    b[table[0].long()] = bounds[0]
    few = T.randint(0, 3, (300,), generator=T.Generator().manual_seed(1))
    b[table[1].long()] = bounds[few]
    b[table[2].long()] = 0.0
    b[table[2, ::2].long()] = -0.0
    q[2] = q[2].abs()
    b[table[3].long(), :, 0] = -1.0
    b[table[3].long(), :, 1] = (1 + T.randint(0, 2, (300, 1, 1), generator=T.Generator().manual_seed(2))).to(T.bfloat16)
    for sink, local in ((0, 0), (1, 0)):
        check_select(T, q, b, table, [4800, 4790, 4800, 4700], 16, top_k, sink_pages=sink, local_pages=local)


def test_select_values_that_are_no_numbers(torch_cuda):
    T = torch_cuda
    q, bounds, table = make_select(T, 6, 4, 8, 2, 128, 16, 60)
    inf, nan = float("inf"), float("nan")
    bounds[table[0, 7].long(), :, 1, 3] = inf
    bounds[table[0, 40].long(), 0, 0, 9] = -inf
    bounds[table[0, 30].long(), 1] = nan
    q[1, 5, 2] = nan        # every page of one KV head is a tie
    q[2] = 0.0              # every score is 0
    q[1, 0, 5] = inf        # -inf for pages whose bounds are below 0 there
    bounds[table[1, ::2].long(), 0, :, 5] = -T.tensor([2.0, 1.0], dtype=T.bfloat16)
    q[3, 0] = T.full((128,), 3e38, dtype=T.bfloat16)
    bounds[table[3].long()] *= 1e38  # products past the range of 32 bits
    check_select(T, q, bounds, table, [950] * 4, 16, 9)


def test_select_entries_outside_the_pool_come_last(torch_cuda):
    T = torch_cuda
    q, bounds, table = make_select(T, 7, 2, 4, 2, 64, 16, 40)
    table[0, 3], table[0, 17], table[1, ::2] = -1, 2 ** 31 - 1, len(bounds)
    check_select(T, q, bounds, table, [640, 640], 16, 12, sink_pages=0, local_pages=0)
    check_select(T, q, bounds, table, [640, 640], 16, 39, sink_pages=2, local_pages=1)


def test_select_near_ties(torch_cuda):
    # scores that differ by less than an fp32 sum of their products is off by
    T = torch_cuda
    q, bounds, table = make_select(T, 8, 2, 4, 1, 128, 16, 200)
    q[..., 0], q[..., 1] = 256.0, 256.0
    low, high = bounds[:, :, 0], bounds[:, :, 1]
    low.zero_(), high.zero_()
    high[..., 0] = 254.0
    step = 2.0 ** -24 * T.randint(0, 4, (len(bounds), 1), generator=T.Generator().manual_seed(4))
    high[..., 1] = step.to(T.bfloat16)  # the sum moves by 2^-16 of 2^16: a bit of fp32 below its last
    check_select(T, q, bounds, table, [3200, 3111], 16, 50, sink_pages=0, local_pages=0)


def check_select_many(T, q, bounds, table, length, page, top_k, sink=1, local=1):
    """One sequence of many pages: the scores by torch, in 64 bits, sorted with ties to the lowest page."""
    got = paged.select_kv_pages(q, bounds, table, length, page, top_k, sink, local)
    n, heads_k = -(-length // page), bounds.shape[1]
    b = bounds[table[0, :n].long()].double()
    group = q.shape[1] // heads_k
    for h in range(heads_k):
        x = q[0, group * h:group * h + group].double()
        s = ((b[:, None, h, 1] * x.clamp(min=0)).sum(2) + (b[:, None, h, 0] * x.clamp(max=0)).sum(2)).amax(1)
        s = s.masked_fill(s.isnan(), float("inf"))
        index = T.arange(n, device="cuda")
        order = T.argsort(s, descending=True, stable=True)
        forced = (index < sink) | (index >= n - local)
        take = T.cat([index[forced], order[~forced[order]][: top_k - sink - local]]).sort().values
        assert T.equal(got[0, h].long(), take)


@pytest.mark.parametrize("width,top_k", [(2048, 100), (2049, 1000), (8192, 8191), (8200, 64), (40000, 700),
                                         (65536, 300), (70001, 5000), (140000, 64), (62500, 30000),
                                         (140000, 70000)])
def test_select_long_sequence(torch_cuda, width, top_k):
    # more pages than a workgroup holds in registers, and than one bit map of them
    T = torch_cuda
    g = T.Generator(device="cuda").manual_seed(width)
    q = T.randn(1, 8, 128, device="cuda", generator=g).to(T.bfloat16)
    bounds = T.randn(width, 2, 2, 128, device="cuda", generator=g).sort(2).values.to(T.bfloat16)
    table = T.randperm(width, device="cuda", generator=g).to(T.int32).view(1, width)
    for sink, local in ((1, 1), (0, 0), (3, 61)):
        check_select_many(T, q, bounds, table, width * 16 - 3, 16, top_k, sink, local)


@pytest.mark.parametrize("kind", ["equal", "few values", "crowd and one far", "two crowds", "one page far below",
                                  "large", "small queries", "nearly equal", "stranger"])
@pytest.mark.parametrize("width,top_k", [(1500, 400), (5000, 90), (70000, 9000)])
def test_select_score_distributions(torch_cuda, kind, width, top_k):
    # the scores themselves, as the first channel of bounds that are 0 elsewhere: crowds that a first look cannot
    # part, scores that fp32 cannot tell from each other, values past what its error is known for
    T = torch_cuda
    g = T.Generator(device="cuda").manual_seed(5)
    q = T.zeros(1, 2, 64, dtype=T.bfloat16, device="cuda")
    q[..., :4] = T.tensor([1.0, 1.0, 2.0 ** -20, 1.0])
    bounds = T.zeros(width, 1, 2, 64, dtype=T.bfloat16, device="cuda")
    x = T.rand(width, device="cuda", generator=g)
    if kind == "equal":
        x.fill_(0.5)
    elif kind == "few values":
        x = (4 * x).floor()
    elif kind == "crowd and one far":
        x[width // 2] = 300.0
    elif kind == "two crowds":
        x[:top_k - 7] += 1e6
    elif kind == "one page far below":
        x[width // 3] = -1e7
    elif kind == "large":
        x *= 1e30
    elif kind == "small queries":
        q *= 2.0 ** -130  # below the normal range, against bounds that make up for it
        x *= 2.0 ** 120
    elif kind == "nearly equal":
        bounds[:, 0, 1, 2] = x.to(T.bfloat16)  # 2^-20 of it counts
        x.fill_(0.75)
    bounds[:, 0, 1, 0] = x.to(T.bfloat16)
    bounds[:, 0, 1, 1] = (x - bounds[:, 0, 1, 0].float()).to(T.bfloat16)  # 16 bits of x in all
    if kind == "stranger":
        bounds[width // 2, 0, 1, 3] = float("nan")
    table = T.randperm(width, device="cuda", generator=g).to(T.int32).view(1, width)
    check_select_many(T, q, bounds, table, width * 16, 16, top_k)
    check_select_many(T, q, bounds, table, width * 16, 16, top_k, 0, 0)


def test_select_bounds_far_apart(torch_cuda):
    # a channel whose smallest key is 2^80 times its largest, and of the other sign of what is asked for
    T = torch_cuda
    q, bounds, table = make_select(T, 9, 2, 4, 2, 128, 16, 300)
    q.abs_()
    bounds[:, :, 0, 7] = -2.0 ** 80
    bounds[:, 1, 0, 9] = -2.0 ** 40
    bounds[::3, 0, 1] *= 2.0 ** 70
    check_select(T, q, bounds, table, [4800, 4000], 16, 31, sink_pages=0, local_pages=0)


def test_many_rows(torch_cuda):
    # more (sequence, KV head) rows than a dimension of a grid but the first holds
    T = torch_cuda
    g = T.Generator(device="cuda").manual_seed(3)
    batch, heads_k, dim, page, width, top_k = 4500, 16, 64, 16, 6, 3
    blocks = 400
    kc, vc = (T.randn(blocks, page, heads_k, dim, device="cuda", generator=g).to(T.bfloat16) for _ in range(2))
    bounds = T.stack([kc.amin(1), kc.amax(1)], 2)
    table = T.randint(0, blocks, (batch, width), device="cuda", generator=g, dtype=T.int32)
    lens = T.randint(0, width * page + 1, (batch,), device="cuda", generator=g, dtype=T.int32)
    q = T.randn(batch, heads_k, dim, device="cuda", generator=g).to(T.bfloat16)
    pages = paged.select_kv_pages(q, bounds, table, lens, page, top_k, 0, 0)
    b, x = bounds[table.long()].double(), q.double()[:, None]
    s = (b[:, :, :, 1] * x.clamp(min=0) + b[:, :, :, 0] * x.clamp(max=0)).sum(3).transpose(1, 2)  # (batch, heads, width)
    n = ((lens + page - 1) // page)[:, None, None]
    s = s.masked_fill(T.arange(width, device="cuda") >= n, -float("inf"))
    best = s.sort(descending=True, stable=True).indices[..., :top_k]
    best = best.masked_fill(best >= n, width).sort().values
    assert T.equal(pages.long(), best.masked_fill(best == width, -1))
    out, lse = attention.flash_attn_with_kvcache_sparse(q, kc, vc, table, pages, lens, return_softmax_lse=True)
    some = T.tensor([0, 1, 77, 2222, 4095, 4096, 4499])
    want, want_lse, tol, lse_tol = ref.attend(q[some].cpu(), kc.cpu(), vc.cpu(), table[some].cpu(), pages[some].cpu(),
                                              lens[some].tolist())
    assert ((out[some].cpu().double() - want).abs() <= tol).all()
    live = (lens[some] > 0).cpu()
    assert ((lse[some].cpu().double() - want_lse).abs() <= lse_tol)[live].all()


@pytest.mark.parametrize("how", ["row", "heads", "offset", "four"])
def test_select_of_other_strides(torch_cuda, how):
    T = torch_cuda
    q, bounds, table = make_select(T, 9, 3, 4, 2, 64, 16, 50)
    dev = q.cuda()
    if how == "row":
        dev = T.cat([dev.view(3, 256), T.zeros(3, 128, device="cuda", dtype=T.bfloat16)], 1)[:, :256].view(3, 4, 64)
    elif how == "heads":
        dev = dev.transpose(0, 1).contiguous().transpose(0, 1)
    elif how == "offset":
        dev = T.nn.functional.pad(dev, (1, 0))[..., 1:]
    else:
        dev = dev.view(3, 1, 4, 64)
    wide = T.zeros(3, 64, dtype=T.int32, device="cuda")
    wide[:, 5:55] = table.cuda()
    got = paged.select_kv_pages(dev, bounds.cuda(), wide[:, 5:55], ints(T, [800, 700, 30]), 16, 6)
    assert T.equal(got.cpu(), ref.select(q, bounds, table, [800, 700, 30], 16, 6))


def test_select_refuses(torch_cuda):
    T = torch_cuda
    q, bounds, table = (x.cuda() for x in make_select(T, 9, 3, 4, 2, 64, 16, 50))
    lens = ints(T, [1, 2, 3])
    for a in [dict(top_k=0), dict(top_k=1), dict(sink=-1), dict(q=q[:2]), dict(q=q.float()), dict(bounds=bounds[:, :, :1]),
              dict(table=table[:2]), dict(table=table.long()), dict(lens=lens[:2]), dict(lens=lens.long()), dict(q=q[:, :3]),
              dict(bounds=bounds.cpu())]:
        d = {**dict(q=q, bounds=bounds, table=table, lens=lens, top_k=4, sink=1), **a}
        with pytest.raises(ValueError):
            paged.select_kv_pages(d["q"], d["bounds"], d["table"], d["lens"], 16, d["top_k"], d["sink"])


# ------------------------------------------------------------------------------------------------------------
# All of them, as a server uses them
# ------------------------------------------------------------------------------------------------------------
class Server:
    """A few requests over one pool: prompts in ragged chunks, then single tokens."""

    def __init__(self, T, batch=4, heads=8, heads_k=2, dim=64, page=16, blocks=64, width=20, most=48):
        self.T, self.page, self.most, self.shape = T, page, most, (heads, heads_k, dim)
        self.k_cache, self.v_cache = (T.full((blocks, page, heads_k, dim), float("nan"), dtype=T.bfloat16, device="cuda")
                                      for _ in range(2))
        self.bounds = T.full((blocks, heads_k, 2, dim), float("nan"), dtype=T.bfloat16, device="cuda")
        self.table = T.zeros(batch, width, dtype=T.int32, device="cuda")
        self.free = T.randperm(blocks, generator=T.Generator().manual_seed(0)).to(T.int32).cuda()
        self.num_free = ints(T, [blocks])
        self.lens = T.zeros(batch, dtype=T.int32, device="cuda")
        self.new = T.zeros(batch, dtype=T.int32, device="cuda")
        self.qkv = T.zeros(most, (heads + 2 * heads_k) * dim, dtype=T.bfloat16, device="cuda")

    def step(self, top_k=4):
        T, (H, Hk, D), n = self.T, self.shape, self.most
        p = paged.plan_paged_step(self.lens, self.new, self.table, self.free, self.num_free, self.page, n)
        k = self.qkv[:, H * D:(H + Hk) * D].view(n, Hk, D)
        v = self.qkv[:, (H + Hk) * D:].view(n, Hk, D)
        paged.append_paged_kv(k, v, self.k_cache, self.v_cache, p.slots, self.bounds)
        last = (p.cu_new[1:].long() - 1).clamp(min=0)  # each sequence's last new token asks
        q = self.qkv[:, :H * D].view(n, H, D)[last]
        pages = paged.select_kv_pages(q, self.bounds, self.table, p.seqlens, self.page, top_k)
        out, lse = attention.flash_attn_with_kvcache_sparse(q, self.k_cache, self.v_cache, self.table, pages, p.seqlens,
                                                            return_softmax_lse=True)
        self.lens.copy_(p.seqlens)
        self.num_free.copy_(p.num_free)
        return p, q, pages, out, lse

    def feed(self, new, seed):
        T = self.T
        self.new.copy_(ints(T, new))
        self.qkv.copy_(T.randn(self.qkv.shape, generator=T.Generator().manual_seed(seed)).to(T.bfloat16))


STEPS = [[20, 1, 0, 7], [1, 30, 2, 15], [1, 1, 1, 1], [0, 1, 16, 1], [1, 1, 1, 1], [16, 1, 1, 30], [1, 1, 1, 1]]


def test_a_run_of_steps(torch_cuda):
    # the caches against what was fed, the selection and the attention against the references over it
    T = torch_cuda
    s = Server(T)
    H, Hk, D = s.shape
    fed = [[] for _ in range(4)]
    for i, new in enumerate(STEPS):
        s.feed(new, i)
        p, q, pages, out, lse = s.step()
        rows, at = s.qkv.cpu(), 0
        for b, n in enumerate(new):
            fed[b] += list(rows[at:at + n])
            at += n
        lens = [len(f) for f in fed]
        assert p.seqlens.tolist() == lens and s.lens.tolist() == lens
        table, kc, vc = s.table.cpu(), s.k_cache.cpu(), s.v_cache.cpu()
        used = [int(table[b, j]) for b in range(4) for j in range(-(-lens[b] // 16))]
        assert len(set(used)) == len(used) == 64 - s.num_free.item()
        for b, f in enumerate(fed):
            for t, r in enumerate(f):
                assert T.equal(kc[table[b, t // 16], t % 16].reshape(-1), r[H * D:(H + Hk) * D])
                assert T.equal(vc[table[b, t // 16], t % 16].reshape(-1), r[(H + Hk) * D:])
        bounds = s.bounds.cpu()
        for b in range(4):
            for j in range(-(-lens[b] // 16)):
                live = kc[table[b, j], : lens[b] - 16 * j]
                assert T.equal(bounds[table[b, j], :, 0], live.amin(0)) and T.equal(bounds[table[b, j], :, 1], live.amax(0))
        assert T.equal(pages.cpu(), ref.select(q.cpu(), bounds, table, lens, 16, 4))
        want, want_lse, tol, lse_tol = ref.attend(q.cpu(), kc, vc, table, pages.cpu(), lens)
        assert ((out.cpu().double() - want).abs() <= tol).all()
        live = T.tensor(lens) > 0
        assert ((lse.cpu().double() - want_lse).abs() <= lse_tol)[live].all()


def test_a_captured_step_replays(torch_cuda):
    # one graph holds a whole step; its replays, with eager work between them, equal an eager server's
    T = torch_cuda
    a, b = Server(T), Server(T)
    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(side):  # a step without new tokens changes nothing
        a.step()
    T.cuda.current_stream().wait_stream(side)
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        held = a.step()
    for i, new in enumerate(STEPS):
        a.feed(new, i)
        b.feed(new, i)
        graph.replay()
        want = b.step()
        T.cuda.synchronize()
        for x, y in zip((held[0].slots, held[0].seqlens, held[0].counts, *held[1:]),
                        (want[0].slots, want[0].seqlens, want[0].counts, *want[1:])):
            assert T.equal(x, y)
        assert T.equal(a.table, b.table) and same(T, a.bounds, b.bounds)


def test_two_streams_at_once(torch_cuda):
    # two servers' steps on streams of their own, nothing waited for in between
    T = torch_cuda
    a, b, alone = Server(T), Server(T), Server(T)
    streams = [T.cuda.Stream(), T.cuda.Stream()]
    for i, new in enumerate(STEPS):
        for s in (a, b, alone):
            s.feed(new, i)
        T.cuda.synchronize()
        got = []
        for s, stream in ((a, streams[0]), (b, streams[1])):
            with T.cuda.stream(stream):
                got.append(s.step())
        T.cuda.synchronize()
        want = alone.step()
        for g in got:
            for x, y in zip(g[1:], want[1:]):
                assert T.equal(x, y)


# ------------------------------------------------------------------------------------------------------------
# Numbers that a C int does not hold
# ------------------------------------------------------------------------------------------------------------
def test_numbers_past_32_bits_are_refused(torch_cuda):
    # each is a small, valid number modulo 2^32
    T, big = torch_cuda, 2 ** 32
    q, bounds, table = (x.cuda() for x in make_select(T, 9, 3, 4, 2, 64, 16, 5))
    kc = T.zeros(len(bounds), 16, 2, 64, dtype=T.bfloat16, device="cuda")
    i3, wide = ints(T, [1, 2, 3]), table[:, :1].expand(3, big + 1)
    pages = T.zeros(3, 2, 2, dtype=T.int32, device="cuda")
    plan = lambda page, most: paged.plan_paged_step(i3, i3, table, i3, i3[2:], page, most)  # noqa: E731
    select = lambda q, table, page, top_k: paged.select_kv_pages(q, bounds, table, i3, page, top_k)  # noqa: E731
    attend = lambda q, table, splits: attention.flash_attn_with_kvcache_sparse(  # noqa: E731
        q, kc, kc, table, pages, i3, num_splits=splits)
    many = q[:, :1].expand(3, big + 4, 64)
    for call in [lambda: plan(16, big + 4), lambda: plan(big + 16, 4), lambda: select(q, table, big + 16, 2),
                 lambda: select(q, table, 16, big + 2), lambda: select(q, wide, 16, 2), lambda: select(many, table, 16, 2),
                 lambda: attend(q, table, big + 1), lambda: attend(q, table, 1 - big), lambda: attend(q, wide, 1),
                 lambda: attend(many, table, 1),
                 lambda: paged.plan_paged_step(i3, i3, wide, i3, i3[2:], 16, 4)]:
        with pytest.raises(ValueError):
            call()


# ------------------------------------------------------------------------------------------------------------
# Heads of 64 in tables of 2049 to 4096 pages
# ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("width,top_k", [(2049, 2048), (2500, 60), (4096, 1500)])
def test_select_small_heads(torch_cuda, width, top_k):
    T = torch_cuda
    q, bounds, table = (x.cuda() for x in make_select(T, width, 1, 8, 2, 64, 16, width))
    for length in (width * 16, width * 16 - 900, (top_k + 1) * 16):
        if length <= top_k * 16:  # the row keeps all of its pages
            got = paged.select_kv_pages(q, bounds, table, length, 16, top_k)
            want = T.arange(top_k, device="cuda")
            assert T.equal(got.long(), want.masked_fill(want >= -(-length // 16), -1).expand(1, 2, top_k))
            continue
        for sink, local in ((1, 1), (0, 0)):
            check_select_many(T, q, bounds, table, length, 16, top_k, sink, local)


@pytest.mark.parametrize("kind", ["equal", "few values", "crowd and one far", "two crowds", "one page far below",
                                  "large", "small queries", "nearly equal", "stranger"])
def test_select_score_distributions_of_small_heads(torch_cuda, kind):
    test_select_score_distributions(torch_cuda, kind, 3000, 700)


def test_plan_of_a_context_that_is_not_in_the_table(torch_cuda):
    # what the documentation says of it: slot -1, in seqlens, not among the missing pages; the other sequences' places
    # are what they would be
    T = torch_cuda
    table = [[0, 0], [4, -1], [0, 0]]
    p = paged.plan_paged_step(ints(T, [100, 20, 0]), ints(T, [5, 3, 17]), ints(T, table), ints(T, [7, 8, 9]),
                              ints(T, [3]), 16, 30)
    assert p.slots.tolist() == [-1] * 8 + list(range(9 * 16, 10 * 16)) + [8 * 16] + [-1] * 5
    assert p.seqlens.tolist() == [105, 23, 17] and p.counts.tolist() == [25, 2, 0, 1]
    assert p.positions.tolist()[:8] == [100, 101, 102, 103, 104, 20, 21, 22]


def test_pages_of_finished_sequences_go_back(torch_cuda):
    # by torch operations that do not wait; more tokens pass through the pool than it holds, and every sequence's
    # are there when it attends
    T = torch_cuda
    s = Server(T, blocks=24)
    s.free = T.cat([s.free, s.free[:1]])  # one place more, for what is not given back
    H, Hk, D = s.shape
    fed, rng = [[] for _ in range(4)], random.Random(1)
    for i in range(40):
        done = T.tensor([len(f) > rng.randint(40, 90) for f in fed])
        for b in range(4):
            if done[b]:
                fed[b] = []
        dev = done.cuda()
        T.cuda.set_sync_debug_mode("error")
        held = (s.lens + s.page - 1) // s.page
        give = (dev[:, None] & (T.arange(s.table.shape[1], device="cuda") < held[:, None])).view(-1)
        at = give.cumsum(0)
        place = T.where(give, s.num_free + at - 1, s.free.numel() - 1)
        s.free.scatter_(0, place, s.table.view(-1))
        s.num_free.copy_(s.num_free + at[-1:].to(T.int32))
        s.lens.copy_(s.lens.masked_fill(dev, 0))
        T.cuda.set_sync_debug_mode("default")
        s.feed([rng.randint(0, 12) for _ in range(4)], i)
        p = s.step()[0]
        rows, lens = s.qkv.cpu(), p.cu_new.tolist()
        for b in range(4):
            fed[b] += list(rows[lens[b]:lens[b + 1]])
        assert p.counts[2] == 0 and p.seqlens.tolist() == [len(f) for f in fed]
        table, kc = s.table.cpu(), s.k_cache.cpu()
        used = [int(table[b, j]) for b in range(4) for j in range(-(-len(fed[b]) // 16))]
        left = s.free[:s.num_free.item()].tolist()
        assert sorted(used + left) == list(range(24))
        for b, f in enumerate(fed):
            for t, r in enumerate(f):
                assert T.equal(kc[table[b, t // 16], t % 16].reshape(-1), r[H * D:(H + Hk) * D])
