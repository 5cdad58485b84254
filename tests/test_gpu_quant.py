"""The quantised paged cache on the GPU: appends byte for byte, reads value for
value, attention against attention in 64 bits over the same codes, and the operators
in a row as a server runs them."""
import random

import numpy as np
import pytest

import paged_testutil
import quant_testutil as ref
from zipserv_asplos26_amd import attention, paged, rotary

pytestmark = pytest.mark.gpu

NAN, INF = 0x7FC0, 0x7F80


def gpu_cache(T, data, page, dim, bits):
    return paged.QuantizedKVCache(T.from_numpy(data).cuda(), page, dim, bits)


def rows_of_all_kinds(T, g, n, heads_k, dim):
    """Rows where quantising can go wrong, among ordinary ones (n at least 24)."""
    x = T.randn(n, heads_k, dim, generator=g).mul_(T.randn(n, heads_k, 1, generator=g).exp())
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 3.25                                                       # no span
    x[3] = T.arange(dim).float() % 16                                 # steps of one: whole codes
    x[4] = (T.arange(dim).float() % 31) / 2                           # half codes: ties
    x[5] = T.randint(-8, 8, (heads_k, dim), generator=g).float()
    x[6, :, 1] = 1e4                                                  # one channel far out
    x[7, :, dim - 1] = -3e38
    x[8, :, 0], x[8, :, 1] = 3e38, -3e38                              # a span that no fp32 holds
    x[9] = float("inf")
    x[10, :, 3] = float("-inf")
    x[11, :, dim // 2] = float("nan")
    x[12] *= 2.0 ** -126                                              # subnormals
    x[13] = 2.0 ** -133 * (T.arange(dim).float() % 3)
    x[14] *= 1e30
    x[15] *= 1e-30
    x[16] = 1.0 + 2.0 ** -7 * (T.arange(dim).float() % 2)             # a span of one step
    x[17] = 2.0 ** (T.arange(dim).float() % 30 - 20)
    x[18, 0] = float("nan")                                           # one head of the token
    x[19] = -T.rand(heads_k, dim, generator=g)
    x[20] = 255.0 - T.arange(dim).float()
    x[21] = T.arange(dim).float() * 1.5
    x[22] *= 2.0 ** 60
    x[23] *= 2.0 ** -62
    return x.to(T.bfloat16)


POOLS = [(1, 64, 16, 4), (8, 128, 16, 4), (3, 64, 48, 8), (2, 128, 32, 8), (5, 128, 128, 4), (16, 64, 16, 8)]


@pytest.mark.parametrize("heads_k,dim,page,bits", POOLS)
def test_append_and_read(torch_cuda, heads_k, dim, page, bits):
    T = torch_cuda
    g = T.Generator().manual_seed(dim + bits)
    blocks, n = 9, 61
    data = ref.random_pool(g, blocks, heads_k, page, dim, bits)
    k, v = (rows_of_all_kinds(T, g, n, heads_k, dim) for _ in range(2))
    slots = T.randperm(blocks * page, generator=g)[:n].to(T.int32)
    slots[5], slots[30], slots[40], slots[60] = -1, blocks * page, -2 ** 31, 2 ** 31 - 1
    cache = gpu_cache(T, data, page, dim, bits)
    paged.append_paged_kv_quantized(k.cuda(), v.cuda(), cache, slots.cuda())
    want = data.copy()
    ref.append(k, v, want, slots, page, dim, bits)
    got = cache.data.cpu().numpy()
    np.testing.assert_array_equal(got[..., :8 * page], want[..., :8 * page])  # scales and lows
    np.testing.assert_array_equal(got, want)
    # and back: these slots in another order, some twice, some that are none
    back = T.cat([slots.flip(0), slots[:3], T.arange(0, blocks * page, 7, dtype=T.int32)])
    for x, y in zip(paged.read_paged_kv_quantized(cache, back.cuda()), ref.read(want, back, page, dim, bits)):
        x = x.cpu()
        assert T.equal(x.isnan(), y.isnan()) and T.equal(x.nan_to_num(), y.nan_to_num())


@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 300])
@pytest.mark.parametrize("bits", [4, 8])
def test_append_counts_and_strides(torch_cuda, n, bits):
    # k and v as slices of a fused projection, and heads that are not next to one another
    T = torch_cuda
    g = T.Generator().manual_seed(n)
    heads, heads_k, dim, page, blocks = 6, 2, 64, 16, 25
    qkv = T.randn(n, (heads + 2 * heads_k) * dim, generator=g).to(T.bfloat16)
    x = qkv.cuda()
    k, v = (x[:, (heads + i * heads_k) * dim:][:, :heads_k * dim].view(n, heads_k, dim) for i in range(2))
    data = ref.random_pool(g, blocks, heads_k, page, dim, bits)
    slots = T.randperm(blocks * page, generator=g)[:n].to(T.int32)
    want = data.copy()
    ref.append(k.cpu(), v.cpu(), want, slots, page, dim, bits)
    for a, b in ((k, v), (k.transpose(0, 1).contiguous().transpose(0, 1), v.contiguous()),
                 (k.transpose(1, 2).contiguous().transpose(1, 2), v)):
        cache = gpu_cache(T, data, page, dim, bits)
        paged.append_paged_kv_quantized(a, b, cache, slots.cuda())
        np.testing.assert_array_equal(cache.data.cpu().numpy(), want)
    for y, z in zip(paged.read_paged_kv_quantized(cache, slots.cuda()), ref.read(want, slots, page, dim, bits)):
        assert y.shape == (n, heads_k, dim) and T.equal(y.cpu(), z)


def test_pools_past_32_bits(torch_cuda):
    # 5.7 GB of pool: slots at both ends, and a sequence whose pages lie there
    T = torch_cuda
    heads_k, dim, page, bits = 8, 128, 64, 8
    blocks = 42000
    cache = paged.quantized_kv_cache(blocks, page, heads_k, dim, bits)
    assert cache.data.numel() > 5.6e9
    g = T.Generator().manual_seed(3)
    k, v = (T.randn(2 * page, heads_k, dim, generator=g).to(T.bfloat16) for _ in range(2))
    slots = T.cat([T.arange(page), T.arange(page) + (blocks - 1) * page]).to(T.int32)
    paged.append_paged_kv_quantized(k.cuda(), v.cuda(), cache, slots.cuda())
    small = np.zeros((2, heads_k, ref.record_bytes(page, dim, bits)), dtype=np.uint8)
    ref.append(k, v, small, T.arange(2 * page), page, dim, bits)
    for i, at in enumerate((0, blocks - 1)):
        np.testing.assert_array_equal(cache.data[at].cpu().numpy(), small[i])
    for x, y in zip(paged.read_paged_kv_quantized(cache, slots.cuda()),
                    ref.read(small, T.arange(2 * page), page, dim, bits)):
        assert T.equal(x.cpu(), y)
    q = T.randn(1, 32, dim, generator=g).to(T.bfloat16)
    want, want_lse, tol, lse_tol = ref.attend(q[:, None], small, T.tensor([[1, 0]], dtype=T.int32), [100], page, bits)
    out = attention.flash_attn_with_kvcache_quantized(q.cuda(), cache,
                                                      T.tensor([[blocks - 1, 0]], dtype=T.int32, device="cuda"), 100)
    assert ((out.cpu().double() - want[:, 0]).abs() <= tol[:, 0]).all()


def test_tokens_past_32_bits(torch_cuda):
    # more than 2^31 elements of keys: only the last tokens have slots, read back among many that have none
    T = torch_cuda
    n, heads_k, dim, page, bits = 2100000, 8, 128, 16, 4
    assert n * heads_k * dim > 2 ** 31
    cache = paged.quantized_kv_cache(2, page, heads_k, dim, bits)
    cache.data.zero_()
    g = T.Generator().manual_seed(4)
    last = T.randn(page, heads_k, dim, generator=g).to(T.bfloat16)
    k = T.zeros(n, heads_k, dim, dtype=T.bfloat16, device="cuda")
    k[-page:] = last.cuda()
    slots = T.full((n,), -1, dtype=T.int32, device="cuda")
    slots[-page:] = T.arange(page, dtype=T.int32, device="cuda") + page
    paged.append_paged_kv_quantized(k, k, cache, slots)
    mirror = np.zeros((2, heads_k, ref.record_bytes(page, dim, bits)), dtype=np.uint8)
    ref.append(last, last, mirror, T.arange(page) + page, page, dim, bits)
    np.testing.assert_array_equal(cache.data.cpu().numpy(), mirror)
    del k
    for x, y in zip(paged.read_paged_kv_quantized(cache, slots), ref.read(mirror, T.arange(page) + page, page, dim, bits)):
        assert T.equal(x[-page:].cpu(), y)
        assert not x[:5].any() and not x[n // 2:n // 2 + 5].any() and not x[-page - 5:-page].any()


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def make(T, seed, batch, new, heads, heads_k, dim, page, width, bits, spread=1.0, spare=5):
    g = T.Generator().manual_seed(seed)
    blocks = batch * width + spare
    table = T.randperm(blocks, generator=g)[:batch * width].view(batch, width).to(T.int32)
    data = ref.random_pool(g, blocks, heads_k, page, dim, bits, spread)
    q = T.randn(batch, new, heads, dim, generator=g).to(T.bfloat16)
    return q, data, table


def poison(T, data, table, lens, page):
    """NaN and infinite scales and lows wherever no sequence has a token (every table here gives a page to one)."""
    blocks, heads_k = data.shape[:2]
    seen = np.zeros((blocks, page), dtype=bool)
    for b, n in enumerate(lens):
        for lp, block in enumerate(table[b].tolist()):
            if 0 <= block < blocks:
                seen[block, :min(max(n - lp * page, 0), page)] = True
    side = data[..., :8 * page].view(np.uint16).reshape(blocks, heads_k, page, 4)
    for i in range(2):
        side[:, :, :, i::2][~np.broadcast_to(seen[:, None], side.shape[:3])] = (NAN, INF)[i]


def check(T, q, data, table, lens, page, bits, scale=None, q_dev=None, want=None, **kw):
    want, want_lse, tol, lse_tol = want or ref.attend(q, data, table, lens, page, bits, scale)
    got, lse = attention.flash_attn_with_kvcache_quantized(
        q.cuda() if q_dev is None else q_dev, gpu_cache(T, data, page, q.shape[-1], bits), table.cuda(),
        T.tensor(lens, dtype=T.int32, device="cuda"), softmax_scale=scale, return_softmax_lse=True, **kw)
    o, l = got.cpu().double().view(want.shape), lse.cpu().double().view(want_lse.shape)
    empty = want_lse == -float("inf")
    assert (o[empty.transpose(1, 2)] == 0).all() and (l[empty] == -float("inf")).all()
    assert ((o - want).abs() <= tol).all(), float(((o - want).abs() / tol.clamp(min=1e-300)).max())
    assert ((l - want_lse).abs() <= lse_tol)[~empty].all(), float(((l - want_lse).abs() / lse_tol)[~empty].max())
    return got, lse


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads,heads_k,dim,page,width,new", [
    (1, 1, 128, 16, 3, 1), (8, 8, 64, 16, 9, 1), (32, 8, 128, 16, 40, 1), (16, 1, 128, 32, 20, 3), (28, 4, 64, 48, 12, 5),
    (64, 8, 128, 64, 9, 2), (30, 2, 64, 256, 3, 4), (5, 5, 128, 128, 4, 1), (16, 1, 64, 1040, 2, 1), (40, 1, 128, 16, 12, 1),
    (6, 2, 64, 16, 20, 70)])
def test_attention(torch_cuda, heads, heads_k, dim, page, width, new, bits):
    T = torch_cuda
    lens = [width * page, 0, 1, page - 1, page, page + 1, 15, 17, width * page - 1, 3 * page // 2 + 1]
    q, data, table = make(T, width + new, len(lens), new, heads, heads_k, dim, page, width, bits)
    poison(T, data, table, lens, page)
    want = ref.attend(q, data, table, lens, page, bits)
    for splits in (1, 0, 3, 1000):
        check(T, q, data, table, lens, page, bits, want=want, num_splits=splits)


@pytest.mark.parametrize("dim,bits", [(128, 4), (128, 8), (64, 4), (64, 8)])
@pytest.mark.parametrize("group,new", [(8, 4), (1, 29), (4, 12), (8, 8), (5, 13), (3, 35), (2, 60)])
def test_columns_in_several_tiles(torch_cuda, group, new, dim, bits):
    # two to eight tiles of 16 columns, the last one whole or not, one or two to a workgroup; the new tokens
    # of short sequences before the first one see nothing, and scales differ enough for late maxima
    T = torch_cuda
    lens, page, width = [1090, 0, 1, 5, 30, 47, 333], 16, 70
    q, data, table = make(T, group + new, len(lens), new, 2 * group, 2, dim, page, width, bits)
    side = data[..., :8 * page].view(np.uint16).reshape(len(data), 2, page, 4)
    power = T.randint(-12, 12, side.shape[:3], generator=T.Generator().manual_seed(new)).float()
    side[..., 2] = ref.bf16_bits((2.0 ** power).to(T.bfloat16))
    side[..., 3] = ref.bf16_bits((-2.0 ** (power + bits - 1)).to(T.bfloat16))
    poison(T, data, table, lens, page)
    want = ref.attend(q, data, table, lens, page, bits)
    for splits in (1, 0, 3):
        check(T, q, data, table, lens, page, bits, want=want, num_splits=splits)


@pytest.mark.parametrize("dim,bits,new", [(128, 4, 1), (64, 4, 3), (128, 8, 2), (64, 8, 1)])
def test_every_length(torch_cuda, dim, bits, new):
    # sequences that end at every place of a tile and of a pair of tiles
    T = torch_cuda
    lens, page, width = list(range(0, 82)), 16, 6
    q, data, table = make(T, 1, len(lens), new, 4, 2, dim, page, width, bits)
    poison(T, data, table, lens, page)
    want = ref.attend(q, data, table, lens, page, bits)
    for splits in (1, 0):
        check(T, q, data, table, lens, page, bits, want=want, num_splits=splits)


@pytest.mark.parametrize("kind", ["ragged", "empty", "one", "edges", "even"])
@pytest.mark.parametrize("batch", [2, 64, 65, 200])
def test_batches_cut_by_their_lengths(torch_cuda, batch, kind):
    # parts that hold pieces of several sequences, sequences in several parts, and empty ones wherever they stand
    T = torch_cuda
    rng = random.Random(batch)
    page, width = 16, 80
    lens = {"ragged": [rng.choice([0, 0, 1, 5, 16, 17, 100, 333, 640, 1111]) for _ in range(batch)], "empty": [0] * batch,
            "one": [0] * (batch - 1) + [611], "edges": [0] * batch, "even": [320] * batch}[kind]
    if kind == "edges":  # the places around which sequences are looked through
        for b in (0, 1, 62, 63, 64, 65, 127, 128, batch - 2):
            lens[b % batch] = rng.choice([16, 512, 640])
    q, data, table = make(T, batch, batch, 1, 2, 1, 64, page, width, 4)
    poison(T, data, table, lens, page)
    want = ref.attend(q, data, table, lens, page, 4)
    for n in (lens, lens[::-1]):
        if n is not lens:
            q, table = q.flip(0).contiguous(), table.flip(0).contiguous()
            want = tuple(w.flip(0) for w in want)
        check(T, q, data, table, n, page, 4, want=want)


@pytest.mark.parametrize("bits", [4, 8])
def test_long_context(torch_cuda, bits):
    # one sequence over many splits, next to short ones in a wide table
    T = torch_cuda
    lens, page, width = [20011, 3, 700], 16, 1300
    q, data, table = make(T, 4, 3, 1, 8, 2, 128, page, width, bits)
    poison(T, data, table, lens, page)
    want = ref.attend(q, data, table, lens, page, bits)
    for splits in (0, 1, 300):
        check(T, q, data, table, lens, page, bits, want=want, num_splits=splits)


def test_queries_past_32_bits(torch_cuda):
    # more than 2^31 elements of q: the same few sequences again and again
    T = torch_cuda
    few, times, new, heads, page, width, bits = 4, 1030, 64, 64, 16, 5, 4
    lens = [80, 3, 0, 65]
    q, data, table = make(T, 31, few, new, heads, 8, 128, page, width, bits)
    assert q.numel() * times > 2 ** 31
    cache, many = gpu_cache(T, data, page, 128, bits), T.tensor(lens, dtype=T.int32).repeat(times).cuda()
    out, lse = attention.flash_attn_with_kvcache_quantized(
        q.cuda().repeat(times, 1, 1, 1), cache, table.repeat(times, 1).cuda(), many, return_softmax_lse=True)
    one, one_lse = check(T, q, data, table, lens, page, bits, num_splits=1)
    assert (out.view(times, few, new, heads, 128) == one).all() and (lse.view(times, few, heads, new) == one_lse).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_scores_far_apart(torch_cuda, bits):
    # scores of hundreds: weights that underflow, maxima that move late, lows far from 0
    T = torch_cuda
    lens, page, width = [333, 200, 64], 16, 21
    q, data, table = make(T, 11, 3, 2, 8, 2, 64, page, width, bits, spread=3.0)
    q = (q.float() * 8).to(T.bfloat16)
    check(T, q, data, table, lens, page, bits)
    check(T, q, data, table, lens, page, bits, scale=-0.7)
    check(T, q, data, table, lens, page, bits, scale=0.0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("which", ["apart", "small", "large", "flat", "zero", "mixed"])
def test_values_of_all_sizes(torch_cuda, which, bits):
    # value rows whose scales are far apart, all small, all large, or 0 (rows of one value)
    T = torch_cuda
    lens, page, width = [700, 333, 64], 16, 44
    q, data, table = make(T, 17, 3, 1, 8, 2, 64, page, width, bits)
    side = data[..., :8 * page].view(np.uint16).reshape(len(data), 2, page, 4)
    g = T.Generator().manual_seed(18)
    power = T.randint(-20, 20, side.shape[:3], generator=g).float() if which == "apart" else \
        T.full(side.shape[:3], {"small": -29.0, "large": 100.0}.get(which, 0.0))
    if which == "mixed":  # nearly nothing, then a few that are 2^150 times as large
        power = T.full(side.shape[:3], -60.0)
        power[int(table[0, 30])] = power[int(table[1, 2])] = 90.0
    scale = T.randn(side.shape[:3], generator=g).exp() * 2.0 ** power
    low = -scale * 2 ** (bits - 1)
    if which in ("flat", "zero"):
        flat = T.rand(side.shape[:3], generator=g) < (0.5 if which == "flat" else 2.0)
        scale[flat] = 0.0
    side[..., 2], side[..., 3] = ref.bf16_bits(scale.to(T.bfloat16)), ref.bf16_bits(low.to(T.bfloat16))
    want = ref.attend(q, data, table, lens, page, bits)
    for splits in (1, 0, 5):
        check(T, q, data, table, lens, page, bits, want=want, num_splits=splits)


@pytest.mark.parametrize("bits", [4, 8])
def test_pages_that_are_not_in_the_pool(torch_cuda, bits):
    T = torch_cuda
    lens, page, width = [150, 96, 40, 70], 16, 10
    q, data, table = make(T, 12, 4, 2, 8, 2, 64, page, width, bits)
    table[0, 2], table[0, 7], table[1, 0], table[1, 5] = -1, len(data), 2 ** 31 - 1, -2 ** 31
    table[2] = -1
    want = ref.attend(q, data, table, lens, page, bits)
    assert (want[1][2] == -float("inf")).all()
    for splits in (1, 0, 4):
        check(T, q, data, table, lens, page, bits, want=want, num_splits=splits)
    # lengths past the table's width, and below 0
    lens = [2 ** 31 - 1, 161, -5, -2 ** 31]
    some = [160, 160, 0, 0]
    q1 = q[:, :1].contiguous()
    check(T, q1, data, table, lens, page, bits, want=ref.attend(q1, data, table, some, page, bits))


def test_a_row_that_is_no_number_shows(torch_cuda):
    # a stored row of NaNs reaches the queries that see it, and no others
    T = torch_cuda
    page, width, new, bits = 16, 4, 3, 4
    for side in (0, 1):
        q, data, table = make(T, 13, 2, new, 8, 2, 128, page, width, bits)
        block = int(table[1, 2])
        data[block, 1, :8 * page].view(np.uint16).reshape(page, 4)[5, 2 * side:2 * side + 2] = NAN  # token 37, head 1
        lens = [50, 39]  # new tokens see 37, 38 and 39 tokens
        got, lse = attention.flash_attn_with_kvcache_quantized(
            q.cuda(), gpu_cache(T, data, page, 128, bits), table.cuda(), T.tensor(lens, dtype=T.int32).cuda(),
            return_softmax_lse=True)
        bad = got.isnan().any(-1).cpu()
        assert bad[1, 1:, 4:].all() and not bad[1, 0].any() and not bad[1, :, :4].any() and not bad[0].any()
        assert got[1, 1:, 4:].isnan().all() and lse.isnan().cpu().any() == (side == 0)


def test_query_layouts(torch_cuda):
    T = torch_cuda
    page, width, bits = 16, 8, 4
    q, data, table = make(T, 14, 3, 2, 8, 2, 64, page, width, bits)
    lens = T.tensor([128, 77, 5], dtype=T.int32, device="cuda")
    cache, tab = gpu_cache(T, data, page, 64, bits), table.cuda()

    def run(x, t=tab, n=lens, **kw):
        return attention.flash_attn_with_kvcache_quantized(x, cache, t, n, **kw)

    want = run(q.cuda())
    fused = T.zeros(3, 2, 12 * 64, dtype=T.bfloat16, device="cuda")
    fused[..., 64:9 * 64] = q.view(3, 2, -1).cuda()
    assert T.equal(run(fused[..., 64:9 * 64].view(3, 2, 8, 64)), want)
    shifted = T.zeros(3, 2, 8 * 64 + 1, dtype=T.bfloat16, device="cuda")  # off by one element: copied
    shifted[..., 1:] = q.view(3, 2, -1).cuda()
    assert T.equal(run(shifted[..., 1:].unflatten(-1, (8, 64))), want)
    assert T.equal(run(q.cuda().transpose(1, 2).contiguous().transpose(1, 2)), want)
    wide = T.full((3, 20), -7, dtype=T.int32, device="cuda")
    wide[:, :width] = tab
    assert T.equal(run(q.cuda(), wide[:, :width]), want)
    assert T.equal(run(q.cuda(), tab.t().contiguous().t()), want)
    one, lse = run(q[:, 1].cuda(), return_softmax_lse=True)
    assert one.shape == (3, 8, 64) and lse.shape == (3, 8)
    assert T.equal(one, run(q[:, 1:].cuda())[:, 0])
    assert T.equal(run(q[:, 1:].cuda(), n=60), run(q[:, 1:].cuda(), n=T.full_like(lens, 60)))


def test_python_refuses(torch_cuda):
    T = torch_cuda
    cache = paged.quantized_kv_cache(4, 16, 2, 64)
    q = T.zeros(2, 4, 64, dtype=T.bfloat16, device="cuda")
    table, lens = T.zeros(2, 2, dtype=T.int32, device="cuda"), T.ones(2, dtype=T.int32, device="cuda")
    slots = T.zeros(2, dtype=T.int32, device="cuda")
    kv = T.zeros(2, 2, 64, dtype=T.bfloat16, device="cuda")
    wrong = paged.QuantizedKVCache(cache.data[..., :-16].contiguous(), 16, 64, 4)
    cpu = paged.QuantizedKVCache(cache.data.cpu(), 16, 64, 4)
    run = attention.flash_attn_with_kvcache_quantized
    for args in ((q.half(), cache, table, lens), (q[0], cache, table, lens), (q[..., :32], cache, table, lens),
                 (q[:, :3], cache, table, lens), (q, cache.data, table, lens), (q, wrong, table, lens),
                 (q, cpu, table, lens), (q, cache, table[:1], lens), (q, cache, table.long(), lens),
                 (q, cache, table, lens.long()), (q, cache, table, lens[:1])):
        with pytest.raises(ValueError):
            run(*args)
    with pytest.raises(ValueError):
        run(q, cache, table, lens, num_splits=2 ** 31)
    for args in ((kv.float(), kv, cache, slots), (kv, kv[:1], cache, slots), (kv, kv, cache, slots.long()),
                 (kv[:, :1], kv, cache, slots), (kv, kv, wrong, slots), (kv, kv, cpu, slots)):
        with pytest.raises(ValueError):
            paged.append_paged_kv_quantized(*args)
    for args in ((wrong, slots), (cpu, slots), (cache, slots.long()), (cache, slots.view(1, 2))):
        with pytest.raises(ValueError):
            paged.read_paged_kv_quantized(*args)


# ---------------------------------------------------------------------------
# A server's steps
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("bits,dim", [(4, 128), (8, 64)])
def test_steps_of_a_server(torch_cuda, bits, dim):
    # prompts, decode steps and verified tokens: plan, rotary, append, attention, each against its definition
    T = torch_cuda
    g, rng = T.Generator().manual_seed(21), random.Random(21)
    batch, heads, heads_k, page, blocks, width = 3, 8, 2, 16, 40, 12
    cache = gpu_cache(T, ref.random_pool(g, blocks, heads_k, page, dim, bits), page, dim, bits)
    mirror = cache.data.cpu().numpy().copy()
    table = T.full((batch, width), -1, dtype=T.int32, device="cuda")
    free = T.randperm(blocks, generator=g).to(T.int32).cuda()
    num_free = T.tensor([blocks], dtype=T.int32, device="cuda")
    seqlens = T.zeros(batch, dtype=T.int32, device="cuda")
    f, factor = rotary.rotary_frequencies(dim, base=500000.0, scaling="ramp", stretch=4.0, trained=64)
    for step, new in enumerate([[40, 1, 17], [1, 1, 1], [3, 3, 3], [1, 1, 1]]):
        total = sum(new) + (5 if step == 0 else 0)  # a padded prefill
        plan = paged.plan_paged_step(seqlens, T.tensor(new, dtype=T.int32).cuda(), table, free, num_free, page, total)
        qkv = T.randn(total, (heads + 2 * heads_k) * dim, generator=g).to(T.bfloat16).cuda()
        q, k, v = (t.unflatten(-1, (-1, dim)) for t in qkv.split([heads * dim, heads_k * dim, heads_k * dim], 1))
        q, k = rotary.apply_rotary(q, k, plan.positions, f, factor=factor)
        paged.append_paged_kv_quantized(k, v, cache, plan.slots)
        ref.append(k.cpu(), v.cpu(), mirror, plan.slots.cpu(), page, dim, bits)
        assert plan.slots[:sum(new)].min() >= 0
        seqlens, num_free = plan.seqlens, plan.num_free
        if step == 0:  # the chunk as the rest of the layer sees it
            got = paged.read_paged_kv_quantized(cache, plan.slots)
            for x, y in zip(got, ref.read(mirror, plan.slots.cpu(), page, dim, bits)):
                assert T.equal(x.cpu(), y)
            continue
        np.testing.assert_array_equal(cache.data.cpu().numpy(), mirror)
        qs = q.view(batch, new[0], heads, dim)
        out, lse = attention.flash_attn_with_kvcache_quantized(qs, cache, table, seqlens, return_softmax_lse=True,
                                                               num_splits=rng.choice([0, 2]))
        want, want_lse, tol, lse_tol = ref.attend(qs.cpu(), mirror, table.cpu(), seqlens.tolist(), page, bits)
        assert ((out.cpu().double() - want).abs() <= tol).all()
        assert ((lse.cpu().double() - want_lse).abs() <= lse_tol).all()


def test_captured_steps_replay(torch_cuda):
    # two decode steps' graphs that are replayed in turn, each over its own caches, with eager work between
    T = torch_cuda
    g = T.Generator().manual_seed(22)
    graphs, states = [], []
    f = rotary.rotary_frequencies(128)[0]
    for i in range(2):
        batch, heads, heads_k, page, width, bits = 2 + i, 8, 2, 16, 80, (4, 8)[i]
        blocks = batch * width
        cache = gpu_cache(T, ref.random_pool(g, blocks, heads_k, page, 128, bits), page, 128, bits)
        table = T.randperm(blocks, generator=g).view(batch, width).to(T.int32).cuda()
        lens = T.tensor([1000, 37, 600][:batch], dtype=T.int32, device="cuda")
        slots = (table.gather(1, ((lens - 1) // page)[:, None].long())[:, 0] * page + (lens - 1) % page).to(T.int32)
        qkv = T.randn(batch, 12 * 128, generator=g).to(T.bfloat16).cuda()

        def step(qkv=qkv, cache=cache, table=table, lens=lens, slots=slots):
            q, k, v = (t.unflatten(-1, (-1, 128)) for t in qkv.split([8 * 128, 2 * 128, 2 * 128], 1))
            q, k = rotary.apply_rotary(q, k, lens - 1, f)
            paged.append_paged_kv_quantized(k, v, cache, slots)
            out = attention.flash_attn_with_kvcache_quantized(q, cache, table, lens)
            return out, paged.read_paged_kv_quantized(cache, slots)[0]

        step()
        T.cuda.synchronize()
        graph = T.cuda.CUDAGraph()
        with T.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
        states.append((qkv, step))
    for turn in range(4):
        for (graph, outs), (qkv, step) in zip(graphs, states):
            qkv.copy_(T.randn(qkv.shape, generator=g).to(T.bfloat16))
            graph.replay()
            got = [o.clone() for o in outs]
            for x, y in zip(got, step()):  # (the same tokens again: the cache stays the same)
                assert T.equal(x, y), turn
        T.cuda.synchronize()


@pytest.mark.parametrize("new,bits", [(1, 4), (1, 8), (5, 8), (8, 4)])
def test_captured_lengths_change(torch_cuda, new, bits):
    # one captured call, replayed as sequences grow, end, come back and share each other's pages
    T = torch_cuda
    page, width, batch, heads, heads_k, dim = 16, 100, 70, 16, 2, 64
    q, data, table = make(T, 40 + new, batch, new, heads, heads_k, dim, page, width, bits)
    cache, tab, qd = gpu_cache(T, data, page, dim, bits), table.cuda(), q.cuda()
    lens = T.full((batch,), 1600, dtype=T.int32, device="cuda")

    def call():
        return attention.flash_attn_with_kvcache_quantized(qd, cache, tab, lens, return_softmax_lse=True)

    call()
    T.cuda.synchronize()
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        out, lse = call()
    rng = random.Random(new)
    for turn in range(6):
        now = [[1600] * batch, [0] * batch, [0] * (batch - 1) + [1600], [rng.choice([0, 1, 17, 333]) for _ in range(batch)],
               [rng.randrange(1601) for _ in range(batch)], [1 + b for b in range(batch)]][turn]
        lens.copy_(T.tensor(now, dtype=T.int32))
        if turn == 4:
            table[1:5] = table[0]
            tab.copy_(table)
        graph.replay()
        want, want_lse = call()
        assert T.equal(out, want) and T.equal(lse, want_lse), turn
        if turn in (3, 4):
            few = slice(0, 6)
            o, l, tol, lse_tol = ref.attend(q[few], data, table[few], now[few], page, bits)
            seen = l > -float("inf")
            assert ((out[few].cpu().double() - o).abs() <= tol).all()
            assert T.equal(lse[few].cpu() > -float("inf"), seen)
            assert ((lse[few].cpu().double() - l).abs() <= lse_tol)[seen].all()


def test_two_streams_at_once(torch_cuda):
    # calls that overlap share no workspace
    T = torch_cuda
    page, width, bits = 16, 700, 4
    q, data, table = make(T, 30, 1, 1, 16, 2, 128, page, width, bits)
    cache, tab = gpu_cache(T, data, page, 128, bits), table.cuda()
    lens = T.tensor([11111], dtype=T.int32, device="cuda")
    qs = [q.cuda(), (q * 2).cuda()]
    want = [attention.flash_attn_with_kvcache_quantized(x, cache, tab, lens) for x in qs]
    streams = [T.cuda.Stream() for _ in range(2)]
    T.cuda.synchronize()
    got = []
    for _ in range(10):
        for x, s in zip(qs, streams):
            with T.cuda.stream(s):
                got.append(attention.flash_attn_with_kvcache_quantized(x, cache, tab, lens))
    T.cuda.synchronize()
    for i, x in enumerate(got):
        assert T.equal(x, want[i % 2])
