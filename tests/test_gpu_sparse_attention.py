"""Decode attention over chosen pages of a paged cache against attention in 64 bits
over the same tokens; what is masked holds NaNs and infinities."""
import random

import pytest

import paged_testutil as ref
from zipserv_asplos26_amd import attention, paged

pytestmark = pytest.mark.gpu


def make(T, seed, batch, heads, heads_k, dim, page, width, spread=1.0, spare=5):
    g = T.Generator().manual_seed(seed)
    blocks = batch * width + spare
    table = T.randperm(blocks, generator=g)[:batch * width].view(batch, width).to(T.int32)
    scale = T.randn(2, heads_k, dim, generator=g).mul(spread).exp()
    kc, vc = (T.randn(blocks, page, heads_k, dim, generator=g).mul_(scale[i]).to(T.bfloat16) for i in range(2))
    q = T.randn(batch, heads, dim, generator=g).to(T.bfloat16)
    return q, kc, vc, table


def poison(T, kc, vc, table, pages, lens):
    """NaNs and infinities into everything that the lists and lengths leave out (of pages that no KV head of
    another sequence reads: every table here gives a page to one sequence)."""
    blocks, page, heads_k, _ = kc.shape
    seen = T.zeros(blocks, page, heads_k, dtype=T.bool)
    for b in range(len(lens)):
        for h in range(heads_k):
            for lp in pages[b, h].tolist():
                if 0 <= lp < table.shape[1] and 0 <= int(table[b, lp]) < blocks:
                    live = min(max(int(lens[b]) - lp * page, 0), page)
                    seen[int(table[b, lp]), :live, h] = True
    for i, c in enumerate((kc, vc)):
        c[~seen] = float("nan")
        c[~seen & (T.arange(page) % 3 == i)[None, :, None]] = float("inf")


def some_pages(T, rng, lens, heads_k, page, top_k, width):
    """Lists in no order, with entries that are no page among them; every page once at most."""
    out = T.full((len(lens), heads_k, top_k), -1, dtype=T.int32)
    for b, n in enumerate(lens):
        have = min(-(-max(n, 0) // page), width)
        for h in range(heads_k):
            take = rng.sample(range(have), min(have, rng.randint(max(0, top_k - 2), top_k)))
            take += [rng.choice([-1, have, have + 1, width, 2 ** 31 - 1, -2 ** 31]) for _ in range(top_k - len(take))]
            rng.shuffle(take)
            out[b, h] = T.tensor(take, dtype=T.int32)
    return out


def check(T, q, kc, vc, table, pages, lens, scale=None, q_dev=None, **kw):
    want, want_lse, tol, lse_tol = ref.attend(q, kc, vc, table, pages, lens, scale)
    got, lse = attention.flash_attn_with_kvcache_sparse(
        q.cuda() if q_dev is None else q_dev, kc.cuda(), vc.cuda(), table.cuda(), pages.cuda(),
        T.tensor(lens, dtype=T.int32, device="cuda"), softmax_scale=scale, return_softmax_lse=True, **kw)
    o, l = got.cpu().double().view(want.shape), lse.cpu().double()
    empty = want_lse == -float("inf")
    assert (o[empty] == 0).all() and (l[empty] == -float("inf")).all()
    assert ((o - want).abs() <= tol).all(), float(((o - want).abs() / tol).max())
    assert ((l - want_lse).abs() <= lse_tol)[~empty].all(), float(((l - want_lse).abs() / lse_tol)[~empty].max())
    return got, lse


@pytest.mark.parametrize("splits", [1, 0, 3])
@pytest.mark.parametrize("heads,heads_k,dim,page,width,top_k", [
    (1, 1, 128, 16, 3, 1), (8, 8, 64, 16, 9, 4), (32, 8, 128, 16, 70, 60), (16, 1, 128, 32, 20, 18),
    (28, 4, 64, 48, 12, 12), (64, 8, 128, 64, 9, 7), (30, 2, 64, 256, 3, 3), (5, 5, 128, 128, 4, 3),
    (16, 1, 64, 1040, 2, 2)])
def test_sparse_attention(torch_cuda, heads, heads_k, dim, page, width, top_k, splits):
    T = torch_cuda
    rng = random.Random(width * page + splits)
    lens = [width * page, 0, 1, page - 1, page, page + 1, 15, 17, width * page - 1, 3 * page // 2 + 1]
    q, kc, vc, table = make(T, top_k, len(lens), heads, heads_k, dim, page, width)
    pages = some_pages(T, rng, lens, heads_k, page, top_k, width)
    poison(T, kc, vc, table, pages, lens)
    check(T, q, kc, vc, table, pages, lens, num_splits=splits)


@pytest.mark.parametrize("page,dim", [(16, 128), (64, 64)])
def test_every_length(torch_cuda, page, dim):
    # pages that end inside a tile, at every place of one
    T = torch_cuda
    lens = list(range(0, 2 * page + 18))
    width = 3 if page > 16 else 4
    q, kc, vc, table = make(T, 1, len(lens), 4, 2, dim, page, width)
    pages = T.arange(width, dtype=T.int32).flip(0).expand(len(lens), 2, width).contiguous()
    poison(T, kc, vc, table, pages, lens)
    check(T, q, kc, vc, table, pages, lens)


def test_lists_in_any_order_agree(torch_cuda):
    # the same pages in another order, and with holes between them, give the same within the bounds; a list that
    # leaves out nothing gives the dense paged attention's result
    T = torch_cuda
    lens, page, width = [600, 333, 1000], 16, 64
    q, kc, vc, table = make(T, 2, 3, 16, 2, 128, page, width)
    whole = T.arange(width, dtype=T.int32).expand(3, 2, width).contiguous()
    shuffled = whole[..., T.randperm(width)].contiguous()
    holes = T.full((3, 2, 2 * width), -1, dtype=T.int32)
    holes[..., ::2] = whole
    outs = [check(T, q, kc, vc, table, p, lens) for p in (whole, shuffled, holes)]
    dense = attention.flash_attn_with_kvcache_dense(
        q.cuda(), kc.cuda(), vc.cuda(), T.tensor(lens, dtype=T.int32, device="cuda"), block_table=table.cuda())
    _, _, tol, _ = ref.attend(q, kc, vc, table, whole, lens)
    # (the dense kernel rounds its weights to bf16: 2^-8 of the weighted sizes more)
    sizes = ref.attend(q, kc, vc.abs(), table, whole, lens)[0]
    assert ((dense.cpu().double() - outs[0][0].cpu().double()).abs() <= 2 * tol + 2.0 ** -8 * sizes).all()


def test_a_page_listed_twice_counts_twice(torch_cuda):
    T = torch_cuda
    q, kc, vc, table = make(T, 3, 1, 4, 2, 64, 16, 8)
    pages = T.tensor([[[1, 1, 3, 7], [5, 5, 5, 5]]], dtype=T.int32)
    check(T, q, kc, vc, table, pages, [128])


def test_nothing_to_attend_to(torch_cuda):
    # no list, no length, no page in the pool: zeros, whatever the pool holds
    T = torch_cuda
    q, kc, vc, table = make(T, 4, 4, 4, 2, 128, 16, 6)
    kc.fill_(float("nan")), vc.fill_(float("inf"))
    table[2], table[3, ::2], table[3, 1::2] = -1, len(kc), 2 ** 31 - 1
    pages = T.arange(6, dtype=T.int32).expand(4, 2, 6).contiguous()
    pages[0] = -1
    for splits in (1, 2, 0):
        check(T, q, kc, vc, table, pages, [96, -3, 96, 96], num_splits=splits)


def test_values_that_are_no_numbers_show(torch_cuda):
    # an infinite value that is attended to comes out, in its channel and heads alone; a key that is no number
    # makes its heads' rows no number
    T = torch_cuda
    q, kc, vc, table = make(T, 5, 3, 8, 2, 64, 16, 4, spread=0.3)
    q.mul_(0.2)
    lens = [50, 64, 61]
    vc[table[0, 1], 5, 0, 7] = float("inf")
    vc[table[1, 2], 0, 1, 3] = -float("inf")
    kc[table[2, 0], 9, 1, 11] = float("nan")
    pages = T.arange(4, dtype=T.int32).expand(3, 2, 4).contiguous()
    out = attention.flash_attn_with_kvcache_sparse(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), pages.cuda(),
                                                   T.tensor(lens, dtype=T.int32, device="cuda")).cpu()
    want = T.zeros_like(out, dtype=T.bool)
    want[0, :4, 7] = True
    assert (out[0].isinf() == want[0]).all() and (out[0, :4, 7] > 0).all()
    want[1, 4:, 3] = True
    assert (out[1].isinf() == want[1]).all() and (out[1, 4:, 3] < 0).all()
    assert out[2, 4:].isnan().all() and out[2, :4].isfinite().all()


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 30.0])
def test_scales(torch_cuda, scale):
    # equal weights, and softmax with a single winner
    T = torch_cuda
    q, kc, vc, table = make(T, 6, 2, 8, 4, 128, 16, 20)
    pages = some_pages(T, random.Random(1), [320, 171], 4, 16, 12, 20)
    check(T, q, kc, vc, table, pages, [320, 171], scale=scale)


def test_one_token_returns_its_value(torch_cuda):
    T = torch_cuda
    q, kc, vc, table = make(T, 7, 3, 8, 2, 128, 16, 2)
    pages = T.tensor([0, -1], dtype=T.int32).expand(3, 2, 2).contiguous()
    got, _ = check(T, q, kc, vc, table, pages, [1, 1, 1])
    want = vc[table[:, 0].long(), 0][:, :, None].expand(3, 2, 4, 128).reshape(3, 8, 128)
    assert T.equal(got.cpu().float(), want.float())


@pytest.mark.parametrize("splits", [0, 1, 2, 5, 64])
def test_splits(torch_cuda, splits):
    # long lists: more tiles a wave than its table of places holds, splits of all lengths, some empty
    T = torch_cuda
    lens = [9000, 40, 8000, 700]
    q, kc, vc, table = make(T, 8, 4, 4, 1, 64, 16, 563)
    pages = some_pages(T, random.Random(5), lens, 1, 16, 561, 563)
    poison(T, kc, vc, table, pages, lens)
    check(T, q, kc, vc, table, pages, lens, num_splits=splits)


@pytest.mark.parametrize("how", ["slice", "transposed", "shared"])
def test_tables_of_other_strides(torch_cuda, how):
    # a part of a wider table, one that is laid out by columns, one row for all; lengths past the table's pages
    T = torch_cuda
    q, kc, vc, table = make(T, 12, 3, 4, 2, 64, 16, 6)
    lens, dev = [96, 200, 50], table.cuda()
    if how == "slice":
        dev = T.full((3, 20), 10 ** 6, dtype=T.int32, device="cuda")
        dev[:, 4:10] = table.cuda()
        dev = dev[:, 4:10]
    elif how == "transposed":
        dev = dev.t().contiguous().t()
    else:
        table = table[:1].expand(3, 6)
        dev = dev[:1].expand(3, 6)
    pages = some_pages(T, random.Random(3), lens, 2, 16, 4, 6)
    want, want_lse, tol, lse_tol = ref.attend(q, kc, vc, table, pages, lens)
    got, lse = attention.flash_attn_with_kvcache_sparse(q.cuda(), kc.cuda(), vc.cuda(), dev, pages.cuda(),
                                                        T.tensor(lens, dtype=T.int32, device="cuda"),
                                                        return_softmax_lse=True)
    assert ((got.cpu().double() - want).abs() <= tol).all() and ((lse.cpu().double() - want_lse).abs() <= lse_tol).all()


@pytest.mark.parametrize("how", ["row", "heads", "offset", "four"])
def test_queries_of_other_strides(torch_cuda, how):
    T = torch_cuda
    q, kc, vc, table = make(T, 9, 3, 4, 2, 64, 16, 6)
    dev = q.cuda()
    if how == "row":
        dev = T.cat([dev.view(3, 256), T.ones(3, 128, device="cuda", dtype=T.bfloat16)], 1)[:, :256].view(3, 4, 64)
    elif how == "heads":
        dev = dev.transpose(0, 1).contiguous().transpose(0, 1)
    elif how == "offset":
        dev = T.nn.functional.pad(dev, (1, 0))[..., 1:]
    else:
        dev = dev.view(3, 1, 4, 64)
    pages = some_pages(T, random.Random(2), [96, 50, 3], 2, 16, 4, 6)
    got, _ = check(T, q, kc, vc, table, pages, [96, 50, 3], q_dev=dev)
    assert got.shape == dev.shape


def test_same_result_every_time(torch_cuda):
    T = torch_cuda
    q, kc, vc, table = (x.cuda() for x in make(T, 10, 4, 32, 8, 128, 16, 100))
    pages = T.arange(90, dtype=T.int32, device="cuda").expand(4, 8, 90).contiguous()
    lens = T.tensor([1600, 999, 1200, 3], dtype=T.int32, device="cuda")
    call = lambda: attention.flash_attn_with_kvcache_sparse(q, kc, vc, table, pages, lens)  # noqa: E731
    first = call()
    for _ in range(20):
        assert T.equal(call(), first)


def test_pool_past_32_bits(torch_cuda):
    # pages whose elements lie past 2^32: append and attention there equal those of a small pool
    from zipserv_asplos26_amd import paged
    T = torch_cuda
    page, heads_k, dim = 64, 8, 128
    blocks = (1 << 32) // (page * heads_k * dim) + 40
    g = T.Generator().manual_seed(11)
    k, v = (T.randn(300, heads_k, dim, generator=g).to(T.bfloat16).cuda() for _ in range(2))
    q = T.randn(1, 16, dim, generator=g).to(T.bfloat16).cuda()
    outs = []
    for n, first in ((40, 7), (blocks, blocks - 10)):
        kc, vc = (T.empty(n, page, heads_k, dim, dtype=T.bfloat16, device="cuda") for _ in range(2))
        bounds = T.empty(n, heads_k, 2, dim, dtype=T.bfloat16, device="cuda")
        table = T.arange(first, first + 5, dtype=T.int32, device="cuda").view(1, 5)
        slots = T.arange(first * page, first * page + 300, dtype=T.int32, device="cuda")
        paged.append_paged_kv(k, v, kc, vc, slots, bounds)
        assert T.equal(kc.view(-1, heads_k, dim)[first * page:first * page + 300], k)
        assert T.equal(vc.view(-1, heads_k, dim)[first * page:first * page + 300], v)
        pages = paged.select_kv_pages(q, bounds, table, 300, page, 3)
        outs.append((pages, attention.flash_attn_with_kvcache_sparse(q, kc, vc, table, pages, 300)))
        del kc, vc
    assert T.equal(outs[0][0], outs[1][0]) and T.equal(outs[0][1], outs[1][1])


def test_sparse_attention_refuses(torch_cuda):
    T = torch_cuda
    q, kc, vc, table = (x.cuda() for x in make(T, 9, 3, 4, 2, 64, 16, 6))
    pages = T.zeros(3, 2, 4, dtype=T.int32, device="cuda")
    lens = T.tensor([9, 9, 9], dtype=T.int32, device="cuda")
    for a in [dict(q=q[:2]), dict(q=q.float()), dict(kc=kc[:, :, :, :32]), dict(vc=vc[:4]), dict(kc=kc.cpu()),
              dict(table=table[:1]), dict(pages=pages[:, :1]), dict(pages=pages.long()), dict(lens=lens[:1]),
              dict(pages=pages[:, :, ::2]), dict(q=q[:, :3]), dict(q=q.view(3, 4, 8, 8))]:
        d = {**dict(q=q, kc=kc, vc=vc, table=table, pages=pages, lens=lens), **a}
        with pytest.raises(ValueError):
            attention.flash_attn_with_kvcache_sparse(d["q"], d["kc"], d["vc"], d["table"], d["pages"], d["lens"])


def one_channel(T, batch, heads_k, dim, score, v):
    """A page of tokens with given scores q.k, exact in fp32 (q is 1 in channel 0 alone): score (batch, heads_k,
    tokens), v (batch, heads_k, tokens, dim)."""
    n = score.shape[2]
    q = T.zeros(batch, heads_k, dim, dtype=T.bfloat16)
    q[..., 0] = 1
    kc = T.zeros(batch, 16, heads_k, dim, dtype=T.bfloat16)
    vc = T.zeros_like(kc)
    kc[:, :n, :, 0] = score.transpose(1, 2).to(T.bfloat16)
    vc[:, :n] = v.transpose(1, 2).to(T.bfloat16)
    table = T.arange(batch, dtype=T.int32).view(batch, 1)
    pages = T.zeros(batch, heads_k, 1, dtype=T.int32)
    return q, kc, vc, table, pages, [n] * batch


@pytest.mark.parametrize("dim", [64, 128])
def test_weights_enter_the_product_as_fp32(torch_cuda, dim):
    # four tokens whose weighted values cancel: each of the last three takes away what its forerunners leave, to 8
    # bits, so 2^-27 of them is left and the output's rounding hides nothing.  What may be left of the sizes: a
    # weight is off by 2^-24 for the scale, as much for its product with the score (below 1 in size) and 2^-23 for
    # the exponential, 4 in all; 12 additions (a weight is at most 3 bf16) by 2^-23 each, 24.  A weight of 16 bits
    # is off by up to 2^-16, half of that in relation to both sizes.
    T = torch_cuda
    g = T.Generator().manual_seed(dim)
    batch, heads_k = 16, 8
    score = -T.rand(batch, heads_k, 4, generator=g).to(T.bfloat16)
    score[..., 0] = 0
    w = score.double().exp()
    v = T.zeros(batch, heads_k, 4, dim, dtype=T.bfloat16)
    v[..., 1, :] = (1 + T.rand(batch, heads_k, dim, generator=g)).to(T.bfloat16)
    for t in (0, 2, 3):
        left = (w[..., None] * v.double()).sum(2)
        v[..., t, :] = (-left / w[..., t, None]).to(T.bfloat16)
    q, kc, vc, table, pages, lens = one_channel(T, batch, heads_k, dim, score, v)
    out = attention.flash_attn_with_kvcache_sparse(q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), pages.cuda(), 4,
                                                   softmax_scale=1.0).cpu().double()
    w = w / w.sum(2, keepdim=True)
    want = (w[..., None] * v.double()).sum(2)
    sizes = (w[..., None] * v.double().abs()).sum(2)
    far = (out - want).abs() - want.abs() * (2.0 ** -8 + 2.0 ** -20)
    assert (far <= 28 * 2.0 ** -24 * sizes).all(), float((far / sizes).max() * 2 ** 24)


@pytest.mark.parametrize("dim", [64, 128])
def test_weights_of_nothing(torch_cuda, dim):
    # a weight that underflows (e^-200) takes nothing of the largest value, and no other weight more than its part
    T = torch_cuda
    score = T.tensor([0.0, -200.0, -75.0]).expand(3, 2, 3)
    v = T.zeros(3, 2, 3, dim)
    v[..., 0, :] = 1.0
    v[..., 1, :] = 3.0e38
    v[1, :, 2] = 2.0e32  # e^-75 of it: 0.5
    v[2, :, 1] *= -1
    want, _, tol, _ = ref.attend(*(x := one_channel(T, 3, 2, dim, score, v)), scale=1.0)
    out = attention.flash_attn_with_kvcache_sparse(*(y.cuda() for y in x[:5]), 3, softmax_scale=1.0).cpu().double()
    assert ((out - want).abs() <= tol).all(), (out - want).abs().max()


@pytest.mark.parametrize("dim", [64, 128])
def test_infinite_values_with_small_weights_show(torch_cuda, dim):
    # weights of 2^-n, which one bf16 holds, and others, down to the smallest normal number
    T = torch_cuda
    for scale, scores in ((0.6931471805599453, [-1, -7, -30, -64, -100, -110, -120, -125]),
                          (1.0, [-0.5, -3.3, -40.0, -60.0, -70.0, -76.0, -82.0, -86.5])):
        score = T.zeros(8, 1, 2)
        score[:, 0, 1] = T.tensor(scores)
        v = T.ones(8, 1, 2, dim)
        v[:, :, 1, 1] = float("inf")
        v[:, :, 1, 5] = -float("inf")
        x = one_channel(T, 8, 1, dim, score, v)
        out = attention.flash_attn_with_kvcache_sparse(*(y.cuda() for y in x[:5]), 2, softmax_scale=scale).cpu()
        assert (out[..., 1] == float("inf")).all() and (out[..., 5] == -float("inf")).all(), out[..., 0, :8]
        rest = [i for i in range(dim) if i not in (1, 5)]
        assert (out[..., rest] == 1).all()


def splits_asked(batch, heads, heads_k, dim, tiles, splits=0):
    """The splits that a call is cut into, by the workspace that it asks for."""
    need = paged._bytes("zs_decode_attention_sparse_workspace_bytes", batch, heads, heads_k, dim, tiles, 16, splits)
    assert need % (batch * heads * (dim + 2) * 4) == 0
    return need // (batch * heads * (dim + 2) * 4)


def check_some(T, seed, batch, heads, heads_k, dim, tiles, alone, splits=0):
    """Lists of `tiles` pages of 16 for `batch` sequences.  The first `alone` have pages of their own, ragged lengths,
    lists in any order and NaNs and infinities in all that these leave out, and are compared with attention in 64
    bits; the others share a few pages, and the last is compared too."""
    rng = random.Random(seed)
    width = tiles + 3
    q, kc, vc, table = make(T, seed, alone + 1, heads, heads_k, dim, 16, width)
    lens = [width * 16, 16 * tiles // 2 + 5, 16 * tiles - 1, 33, 0, 1][:alone]
    assert len(lens) == alone
    lens.append(16 * tiles)
    pages = some_pages(T, rng, lens, heads_k, 16, tiles, width)
    pages[-1] = T.arange(tiles, dtype=T.int32)
    poison(T, kc, vc, table, pages, lens)
    more = batch - len(lens)  # copies of the last sequence, with queries of their own
    q = T.cat([q, T.randn(more, heads, dim, generator=T.Generator().manual_seed(seed)).to(T.bfloat16)])
    grow = lambda x: T.cat([x, x[-1:].expand(more, *x.shape[1:])])  # noqa: E731
    got, lse = attention.flash_attn_with_kvcache_sparse(
        q.cuda(), kc.cuda(), vc.cuda(), grow(table).cuda(), grow(pages).cuda(),
        T.tensor(lens + more * [lens[-1]], dtype=T.int32, device="cuda"), return_softmax_lse=True, num_splits=splits)
    some = list(range(alone)) + [batch - 1]
    want, want_lse, tol, lse_tol = ref.attend(q[some], kc, vc, table, pages, lens)
    o, l = got.cpu()[some].double(), lse.cpu()[some].double()
    empty = want_lse == -float("inf")
    assert (o[empty] == 0).all() and (l[empty] == -float("inf")).all()
    assert ((o - want).abs() <= tol).all(), float(((o - want).abs() / tol).max())
    assert ((l - want_lse).abs() <= lse_tol)[~empty].all()
    assert got.isfinite().all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,heads_k,group,tiles,splits", [
    (20, 16, 1, 25, 3), (20, 16, 2, 100, 3), (40, 8, 4, 200, 3), (16, 20, 1, 33, 3), (60, 7, 2, 61, 2),
    (105, 10, 1, 300, 1), (75, 14, 1, 140, 1), (300, 1, 16, 300, 3)])
def test_workgroups_of_two_waves(torch_cuda, dim, batch, heads_k, group, tiles, splits):
    # rows that fill the last round of the CUs badly: lists over more tiles than a wave's table of places holds
    # (128 for two waves), and splits that are merged.  (Four waves would take all of them in one split; they do
    # not show in what is asked for where two take one as well.)
    T = torch_cuda
    if T.cuda.get_device_properties(0).multi_processor_count == 256:
        assert splits_asked(batch, heads_k * group, heads_k, dim, tiles) == (splits if splits > 1 else 0)
    check_some(T, tiles, batch, heads_k * group, heads_k, dim, tiles, 4)


@pytest.mark.parametrize("splits,dim", [(257, 128), (300, 64), (600, 128)])
@pytest.mark.parametrize("most_in", ["first", "last", "middle", "none"])
def test_merge_of_hundreds_of_splits(torch_cuda, dim, most_in, splits):
    # more splits than the merge takes at once, the largest scores in its first chunk, its last or between
    T = torch_cuda
    tiles = 8 * splits
    assert splits_asked(2, 4, 2, dim, tiles, splits) == splits
    q, kc, vc, table = make(T, splits, 2, 4, 2, dim, 16, tiles, spread=0.3)
    lens = [16 * tiles, 16 * tiles - 16 * 8 * 20 - 3]  # (the second one's last splits are empty)
    for b in range(2):
        if most_in != "none":
            at = {"first": 3, "last": tiles - 170, "middle": 8 * 250}[most_in]
            kc[table[b, at].long(), 7] = 1.5 * q[b].view(2, 2, dim).mean(1)
        vc[table[b, :8 * 256].long()] += 1  # what the chunks hold differs
        vc[table[b, 8 * 256:].long()] -= 1
    pages = T.arange(tiles, dtype=T.int32).expand(2, 2, tiles).contiguous()
    poison(T, kc, vc, table, pages, lens)
    want, want_lse, tol, lse_tol = ref.attend(q, kc, vc, table, pages, lens)
    sizes = ref.attend(q, kc, vc.abs(), table, pages, lens)[0]
    # in place of 3 T 2^-24 for the sums, what these have: 32 tokens' 96 products by 2^-23 each (192), a rescaling and
    # an addition for each of 4 waves (8), for each of 150 splits of a merging wave and 4 of these (308), less
    # than 2^-15; the normaliser's 8 and 2 and 4 tokens, waves and lanes, 3 chunks, 64 lanes and 4 waves by 2^-24 or
    # two, less than 2^-18
    many = 3 * 2.0 ** -24 * T.tensor(lens, dtype=T.float64)
    tol = tol + sizes * (2.0 ** -15 + 2.0 ** -18 - many)[:, None, None]
    lse_tol = lse_tol + (2.0 ** -18 - many)[:, None]
    got, lse = attention.flash_attn_with_kvcache_sparse(
        q.cuda(), kc.cuda(), vc.cuda(), table.cuda(), pages.cuda(), T.tensor(lens, dtype=T.int32, device="cuda"),
        return_softmax_lse=True, num_splits=splits)
    off, lse_off = (got.cpu().double() - want).abs(), (lse.cpu().double() - want_lse).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert (lse_off <= lse_tol).all(), float((lse_off / lse_tol).max())
