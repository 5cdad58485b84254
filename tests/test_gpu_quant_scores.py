"""The digits of the quantised attention's scores: log-sum-exps against fp32 in elementary operations, and
queries whose channels are far apart."""
import math

import numpy as np
import pytest

import quant_testutil as ref
from test_gpu_quant_sizes import attend
from zipserv_asplos26_amd import attention, paged

pytestmark = pytest.mark.gpu


def log_sums(T, q, data, table, lens, page, bits, **kw):
    cache = paged.QuantizedKVCache(T.from_numpy(data).cuda(), page, q.shape[-1], bits)
    out, lse = attention.flash_attn_with_kvcache_quantized(q.cuda(), cache, table.cuda(), T.tensor(
        lens, dtype=T.int32, device="cuda"), return_softmax_lse=True, **kw)
    return out.cpu().double(), lse.cpu().double()


@pytest.mark.parametrize("group", [2, 8, 16, 32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bits", [4, 8])
def test_scores_have_the_digits_of_fp32(torch_cuda, bits, dim, group):
    # The root mean square error of 1024 log-sum-exps or more, against the same formula, s (q.c) + low sum(q), in fp32
    # operations whose long sums are made in two stages.  Both round products and sums alike, so both errors
    # are the same but for chance: the mean square of 1024 has a deviation of 1 / sqrt(512) if errors are normal, so
    # 1.25 in its root allows for more than ten of them, and for orders of summation.
    T = torch_cuda
    g = T.Generator().manual_seed(bits + dim + group)
    batch, heads_k, page, width = 1024 // (8 * group) or 4, 8, 16, 13
    data = ref.random_pool(g, batch * width, heads_k, page, dim, bits)
    table = T.arange(batch * width, dtype=T.int32).view(batch, width)
    n = 203
    q = T.randn(batch, heads_k * group, dim, generator=g).to(T.bfloat16)
    exact, plain = [], []
    (kc, ks, km), _ = ref.parts(data, page, dim, bits)
    for kind, to in ((T.float64, exact), (T.float32, plain)):
        c, s, m = (x.to(kind).view(batch, width, heads_k, page, *x.shape[3:]).transpose(1, 2).flatten(2, 3)[:, :, :n]
                   for x in (kc, ks, km))
        x = q.to(kind).view(batch, heads_k, group, 1, dim)

        def long_sum(y):
            return y.unflatten(-1, (-1, 8)).sum(-1).sum(-1)

        for b in range(batch):
            dot = long_sum(x[b] * c[b][:, None])
            score = (s[b][:, None] * dot + m[b][:, None] * long_sum(x[b])) * T.tensor(1 / math.sqrt(dim), dtype=kind)
            to.append(T.logsumexp(score, -1).flatten())
    exact, plain = T.stack(exact), T.stack(plain).double()
    _, lse = log_sums(T, q, data, table, [n] * batch, page, bits)
    off, fp32 = ((x - exact).square().mean().sqrt() for x in (lse.view_as(exact), plain))
    print(f"log-sum-exps {float(off):.2e} off, in fp32 {float(fp32):.2e}: {float(off / fp32):.2f}")
    assert off <= 1.25 * fp32


@pytest.mark.parametrize("group,new,dim,bits", [(2, 1, 64, 4), (8, 1, 128, 4), (8, 2, 128, 4), (8, 4, 64, 4), (8, 4, 128, 4),
                                                (1, 1, 128, 8), (8, 1, 64, 8), (4, 4, 128, 8), (8, 4, 128, 8)])
def test_channels_of_a_query_far_apart(torch_cuda, group, new, dim, bits):
    # Half of the channels of q are 2^45 as large as the others, and the keys' codes are 0 there, and their lows 0: what
    # is left of a score is the small channels' part, and the errors allowed are that part's alone.
    T = torch_cuda
    g = T.Generator().manual_seed(dim + new)
    batch, heads_k, page, width = 3, 2, 16, 20
    lens, heads = [320, 77, 16], heads_k * group
    data = ref.random_pool(g, batch * width, heads_k, page, dim, bits)
    table = T.randperm(batch * width, generator=g).view(batch, width).to(T.int32)
    side = data[..., :8 * page].view(np.uint16).reshape(*data.shape[:2], page, 4)
    side[..., 1] = 0
    row = dim * bits // 8
    codes = data[..., 8 * page:][..., :page * row].reshape(*data.shape[:2], page, row)
    where = ref.places(dim, bits)
    clear = np.full(row, 255, dtype=np.uint8)
    for byte, shift in where[::2]:
        clear[byte] &= ~((2 ** bits - 1) << shift) & 255
    data[..., 8 * page:][..., :page * row] = (codes & clear).reshape(*data.shape[:2], page * row)
    for large in (45, 60, 90):
        q = T.randn(batch, new, heads, dim, generator=g)
        q[..., ::2] *= 2.0 ** large
        q = q.to(T.bfloat16)
        want, want_lse, tol, lse_tol = attend(q, data, table, lens, page, bits)
        out, lse = log_sums(T, q, data, table, lens, page, bits)
        seen = want_lse > -math.inf
        assert ((lse - want_lse).abs() <= lse_tol)[seen].all() and ((out - want).abs() <= tol).all(), large
