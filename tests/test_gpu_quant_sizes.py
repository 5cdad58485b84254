"""Attention over a quantised cache whose rows and queries are of unusual sizes: constant
rows, scales of any size a bf16 has, rows of zeros that take the weight, rows that are no
number; and the digits that weights keep."""
import math

import numpy as np
import pytest

import quant_testutil as ref
from zipserv_asplos26_amd import attention, paged

pytestmark = pytest.mark.gpu


def attend(q, data, table, lens, page, bits, scale=None):
    """(out, lse, allowed error of out, of lse) as `quant_testutil.attend`, float64, with less allowed.

    A score is s_k (q.c) + low_k sum(q) in fp32: D + 8 operations, each off by 2^-24 of the sum of the sizes
    |q| (s_k c + |low_k|) at most, which move a weight by twice that relatively at most, the normaliser included.
    T weights and T products of s_v c + |low_v|, their rescalings, a merge of splits and the exponentials: 3 T
    2^-24 of the weighted sizes (T counted from 64).  The output's rounding: 2^-8 of it, or half of the least
    subnormal, 2^-134.  Nothing is allowed for small or large values."""
    import torch
    B, new, H, D = q.shape
    blocks, heads_k = data.shape[:2]
    group = H // heads_k
    scale = 1 / math.sqrt(D) if scale is None else scale
    (kc, ks, km), (vc, vs, vm) = ref.parts(data, page, D, bits)
    out, tol = torch.zeros(B, new, H, D, dtype=torch.float64), torch.zeros(B, new, H, D, dtype=torch.float64)
    lse = torch.full((B, H, new), -math.inf, dtype=torch.float64)
    lse_tol = torch.zeros(B, H, new, dtype=torch.float64)
    for b in range(B):
        for i in range(new):
            at = torch.arange(max(0, min(int(lens[b]) - new + 1 + i, table.shape[1] * page)))
            block = table[b].long()[at // page]
            seen = (block >= 0) & (block < blocks)
            block, off = block[seen], at[seen] % page
            if not len(block):
                continue
            for h in range(heads_k):
                rows = slice(h * group, (h + 1) * group)
                c, s, m = kc[block, h, off], ks[block, h, off][:, None], km[block, h, off][:, None]
                k, k_size = c * s + m, c * s.abs() + m.abs()
                c, s, m = vc[block, h, off], vs[block, h, off][:, None], vm[block, h, off][:, None]
                v, v_size = c * s + m, c * s.abs() + m.abs()
                x = q[b, i, rows].double()
                score = x @ k.t() * scale
                w = torch.softmax(score, 1)
                o = w @ v
                ds = (x.abs() @ k_size.t()).amax(1, keepdim=True) * abs(scale) * (D + 8) * 2.0 ** -24
                many = 3 * max(len(block), 64) * 2.0 ** -24
                out[b, i, rows], lse[b, rows, i] = o, torch.logsumexp(score, 1)
                tol[b, i, rows] = 2.0 ** -8 * o.abs() + 2.0 ** -134 + (w @ v_size) * (2 * ds + many)
                lse_tol[b, rows, i] = ds[:, 0] + many + 2.0 ** -22 * lse[b, rows, i].abs()
    return out, lse, tol, lse_tol


def make(T, seed, batch, new, heads, heads_k, dim, page, width, bits):
    g = T.Generator().manual_seed(seed)
    blocks = batch * width + 3
    table = T.randperm(blocks, generator=g)[:batch * width].view(batch, width).to(T.int32)
    return T.randn(batch, new, heads, dim, generator=g).to(T.bfloat16), \
        ref.random_pool(g, blocks, heads_k, page, dim, bits), table, g


def sides(data, page):
    """(scale, low) of every key and value, bf16 bits that can be written to: (blocks, Hkv, page, 4)."""
    return data[..., :8 * page].view(np.uint16).reshape(*data.shape[:2], page, 4)


def run(T, q, data, table, lens, page, bits, **kw):
    cache = paged.QuantizedKVCache(T.from_numpy(data).cuda(), page, q.shape[-1], bits)
    out, lse = attention.flash_attn_with_kvcache_quantized(q.cuda(), cache, table.cuda(), T.tensor(
        lens, dtype=T.int32, device="cuda"), return_softmax_lse=True, **kw)
    return out.cpu().double(), lse.cpu().double()


def check(T, q, data, table, lens, page, bits, splits=(1, 0, 5), scale=None):
    want, want_lse, tol, lse_tol = attend(q, data, table, lens, page, bits, scale)
    for n in splits:
        out, lse = run(T, q, data, table, lens, page, bits, num_splits=n, softmax_scale=scale)
        seen = want_lse > -math.inf
        assert ((out - want).abs() <= tol).all(), (n, float(((out - want).abs() / tol.clamp(min=1e-300)).max()))
        assert ((lse - want_lse).abs() <= lse_tol)[seen].all(), n


SHAPES = [(2, 1, 64, 4), (8, 1, 128, 4), (8, 2, 128, 4), (8, 4, 64, 4), (8, 4, 128, 4),
          (1, 1, 128, 8), (8, 1, 64, 8), (4, 4, 128, 8), (8, 4, 64, 8), (8, 4, 128, 8)]  # a kernel each
# flat rows of +-2^n; scales of about 2^n; scales of all sizes a bf16 has
KINDS = ["flat80", "flat86", "flat100", "flat127", "2^-133", "2^-126", "2^-70", "2^-56", "2^-31", "2^17", "2^60", "2^118",
         "all"]


def values_of(T, kind, side, bits, g):
    """Scales and lows of the values of a pool, into side."""
    shape = side.shape[:3]
    sign = 1.0 - 2 * T.randint(0, 2, shape, generator=g).float()
    if kind.startswith("flat"):
        low = sign * T.rand(shape, generator=g).add(1).to(T.bfloat16).double().mul(2.0 ** (int(kind[4:]) - 1)).float()
        scale = T.zeros(shape)
    else:
        n = T.randint(-133, 119, shape, generator=g) if kind == "all" else T.full(shape, int(kind[2:]))
        scale = (T.rand(shape, generator=g).double() + 1).mul(2.0 ** n.double()).float()
        low = -scale * 2 ** (bits - 1)
    side[..., 2], side[..., 3] = ref.bf16_bits(scale.to(T.bfloat16)), ref.bf16_bits(low.to(T.bfloat16))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("group,new,dim,bits", SHAPES)
def test_value_rows_of_any_size(torch_cuda, group, new, dim, bits, kind):
    # alone, and among ordinary rows: one in eight, and a single one
    T = torch_cuda
    lens, page, width = [1100, 333, 64, 1], 16, 70
    q, data, table, g = make(T, 17 + new, 4, new, 2 * group, 2, dim, page, width, bits)
    ordinary = sides(data, page).copy()
    values_of(T, kind, sides(data, page), bits, g)
    unusual = sides(data, page).copy()
    check(T, q, data, table, lens, page, bits)
    keep = (T.rand(ordinary.shape[:3], generator=g) < 0.875).numpy()
    sides(data, page)[keep] = ordinary[keep]
    check(T, q, data, table, lens, page, bits)
    sides(data, page)[...] = ordinary
    sides(data, page)[int(table[0, 31]), :, 7] = unusual[int(table[0, 31]), :, 7]
    check(T, q, data, table, lens, page, bits, splits=(0, 5))


@pytest.mark.parametrize("group,new,dim,bits", SHAPES)
def test_weights_next_to_a_value_that_is_no_number(torch_cuda, group, new, dim, bits):
    # its head's outputs are NaN, but the log-sum-exp is of the keys alone, and other heads do not see it
    T = torch_cuda
    lens, page, width = [1100, 333], 16, 70
    q, data, table, _ = make(T, 23, 2, new, 2 * group, 2, dim, page, width, bits)
    want, want_lse, tol, lse_tol = attend(q, data, table, lens, page, bits)
    sides(data, page)[int(table[0, 3]), 1, 5, 2:] = 0x7FC0
    for n in (1, 0, 5):
        out, lse = run(T, q, data, table, lens, page, bits, num_splits=n)
        assert out[0, :, group:].isnan().all() and not out[0, :, :group].isnan().any()
        ok = ~out.isnan()
        assert ((out - want).abs() <= tol)[ok].all() and ok[1].all()
        assert ((lse - want_lse).abs() <= lse_tol).all(), n


@pytest.mark.parametrize("gap", [20, 50, 80, 110])
@pytest.mark.parametrize("group,new,dim,bits", SHAPES)
def test_rows_of_zeros_that_take_the_weight(torch_cuda, group, new, dim, bits, gap):
    # most tokens are rows of zeros with scores `gap` powers of two above the others', so the output is that much
    # smaller than a value; all keys are flat, so scores are 2 sum(q) times a key's low
    T = torch_cuda
    lens, page, width = [1100, 80], 16, 70
    q, data, table, g = make(T, 29, 2, new, 2 * group, 2, dim, page, width, bits)
    q[:] = 2.0 / dim
    side = sides(data, page)
    others = (T.rand(side.shape[:3], generator=g) < 0.2).numpy()
    side[~others] = 0
    side[..., 0] = 0
    low = T.where(T.from_numpy(others), -0.5 * gap, 0.25 * T.rand(others.shape, generator=g))
    side[..., 1] = ref.bf16_bits(low.to(T.bfloat16))
    check(T, q, data, table, lens, page, bits, scale=math.log(2))


@pytest.mark.parametrize("group,new,dim,bits", SHAPES)
def test_weights_keep_their_digits(torch_cuda, group, new, dim, bits):
    # Of three tokens the first is a row of zeros with a larger score; the other two have one key, so the same weight w
    # of 24 bits, and are a row of codes 1, scale 1 and low 0, and a flat row of -1: 1 w - w is 0.  w is exact in any
    # product with 1, so no rounding is needed; allowed is half of one of w, 2^-25 w, which the sum of the weights, 2 w
    # at least, halves.
    T = torch_cuda
    page, row = 16, dim * bits // 8
    q, data, table, g = make(T, 31, 1, new, 64 * group, 64, dim, page, 1, bits)
    q[:] = 2.0 / dim
    data[..., 8 * page:] = 0x11 if bits == 4 else 1
    data[..., (8 + row) * page:][..., :row] = 0
    side = sides(data, page)
    side[:, :, :, 0], side[:, :, 1:, 1] = 0, 0                 # flat keys: a score is 2 low
    side[:, :, 0, 1] = ref.bf16_bits((T.rand(side.shape[:2], generator=g) / 2).to(T.bfloat16))
    side[:, :, :2, 2], side[:, :, :2, 3] = 0x3F80, 0
    side[:, :, 2, 2], side[:, :, 2, 3] = 0, 0xBF80
    out, lse = run(T, q, data, table, [3], page, bits, num_splits=1, softmax_scale=math.log(2))
    assert lse[0, :, -1].isfinite().all()
    assert (out[:, -1].abs() <= 2.0 ** -26).all(), float(out[:, -1].abs().max()) * 2 ** 26


@pytest.mark.parametrize("kind", ["2^-50", "2^-48", "2^-47", "2^-46", "2^-44", "2^24", "2^26", "2^27", "2^28", "2^40", "flat106",
                                  "flat110", "flat112", "flat113", "flat114"])
@pytest.mark.parametrize("group,new,dim,bits", SHAPES)
def test_value_rows_at_the_borders_of_a_second_pass(torch_cuda, group, new, dim, bits, kind):
    # sums just within what one pass holds, and just past it; in some sequences, heads and parts only
    T = torch_cuda
    lens, page, width = [1100, 333, 64, 1], 16, 70
    q, data, table, g = make(T, 37 + new, 4, new, 2 * group, 2, dim, page, width, bits)
    ordinary = sides(data, page).copy()
    values_of(T, kind, sides(data, page), bits, g)
    keep = np.zeros(ordinary.shape[:3], dtype=bool)
    keep[table[1].numpy()] = True
    keep[:, 1] = True
    keep[table[0, 20:50].numpy()] = True
    sides(data, page)[keep] = ordinary[keep]
    check(T, q, data, table, lens, page, bits)


@pytest.mark.parametrize("group,new,dim,bits", SHAPES)
def test_pools_without_a_value(torch_cuda, group, new, dim, bits):
    # a pool of zeros, and one of rows without a scale
    T = torch_cuda
    lens, page, width = [1100, 333, 64, 0], 16, 70
    q, data, table, g = make(T, 41, 4, new, 2 * group, 2, dim, page, width, bits)
    side = sides(data, page)
    side[..., 2] = 0
    check(T, q, data, table, lens, page, bits)
    data[:] = 0
    for n in (1, 0, 5):
        out, lse = run(T, q, data, table, lens, page, bits, num_splits=n)
        assert (out == 0).all()
        for i in range(new):
            for b, length in enumerate(lens):
                want = math.log(length - new + 1 + i) if length - new + 1 + i > 0 else -math.inf
                assert (lse[b, :, i] == want).all() or (lse[b, :, i] - want).abs().max() <= 2.0 ** -22 * max(want, 1)


@pytest.mark.parametrize("group,new,dim,bits", SHAPES)
def test_captured_passes_over_changing_rows(torch_cuda, group, new, dim, bits):
    # one captured call, replayed as rows of a part become unusual and ordinary again, with two streams' calls between
    T = torch_cuda
    lens, page, width = [1100, 333, 64, 0], 16, 70
    q, data, table, g = make(T, 43, 4, new, 2 * group, 2, dim, page, width, bits)
    pools = [data.copy() for _ in range(4)]
    values_of(T, "2^60", sides(pools[1], page), bits, g)
    for block in table[0, 40:45].tolist():
        sides(pools[3], page)[block, :, ::2, 2:] = 0, 0x7180  # flat rows of 2^100
    wants = [attend(q, x, table, lens, page, bits) for x in pools]
    cache = paged.QuantizedKVCache(T.from_numpy(data).cuda(), page, dim, bits)
    qd, tab, n = q.cuda(), table.cuda(), T.tensor(lens, dtype=T.int32, device="cuda")

    def call():
        return attention.flash_attn_with_kvcache_quantized(qd, cache, tab, n, return_softmax_lse=True)

    call()
    T.cuda.synchronize()
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        out, lse = call()
    streams = [T.cuda.Stream() for _ in range(2)]
    for turn in (0, 1, 2, 3, 1, 0):
        cache.data.copy_(T.from_numpy(pools[turn]))
        graph.replay()
        T.cuda.synchronize()
        others = []
        for s in streams:
            with T.cuda.stream(s):
                others.append(call())
        T.cuda.synchronize()
        want, want_lse, tol, lse_tol = wants[turn]
        seen = want_lse > -math.inf
        assert ((out.cpu().double() - want).abs() <= tol).all(), turn
        assert ((lse.cpu().double() - want_lse).abs() <= lse_tol)[seen].all(), turn
        for o, l in others:
            assert T.equal(o, out) and T.equal(l, lse), turn
