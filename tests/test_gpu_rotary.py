"""Rotary positions against the rotation in 64 bits: types, layouts, strides, far
positions, tokens without one, in place, and captured into a graph."""
import math

import pytest

import quant_testutil as ref
from zipserv_asplos26_amd import rotary

pytestmark = pytest.mark.gpu


def within(got, want, tol):
    got = got.cpu().double().reshape(want.shape)
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol.clamp(min=1e-300)).max())


def inputs(T, seed, tokens, heads, heads_k, dim, dtype, lead=0):
    """q and k as slices of a fused projection's output, `lead` elements into its rows."""
    g = T.Generator().manual_seed(seed)
    x = T.randn(tokens, lead + (heads + 2 * heads_k) * dim, generator=g).mul(1.5).to(dtype)
    q = x[:, lead:lead + heads * dim].view(tokens, heads, dim)
    k = x[:, lead + heads * dim:lead + (heads + heads_k) * dim].view(tokens, heads_k, dim)
    return q, k, x


def on_gpu(q, k, x):
    y = x.cuda()
    return (y.as_strided(t.shape, t.stride(), t.storage_offset()) for t in (q, k))


SHAPES = [  # tokens, heads, heads_k, dim, rotated, lead
    (1, 32, 8, 128, 128, 0), (7, 8, 1, 64, 64, 0), (130, 5, 5, 128, 64, 8), (33, 28, 4, 128, 32, 0), (9, 3, 2, 64, 16, 0),
    (20, 4, 1, 80, 40, 0), (5, 2, 2, 96, 96, 3), (6, 3, 1, 33, 20, 1), (3, 1, 1, 2, 2, 0), (2, 2, 1, 1024, 1024, 0),
    (11, 1, 3, 256, 6, 0)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("tokens,heads,heads_k,dim,rotated,lead", SHAPES)
def test_rotary(torch_cuda, tokens, heads, heads_k, dim, rotated, lead, dtype, interleaved):
    T = torch_cuda
    q, k, x = inputs(T, dim + tokens, tokens, heads, heads_k, dim, getattr(T, dtype), lead)
    at = T.randint(0, 40000, (tokens,), generator=T.Generator().manual_seed(1), dtype=T.int32)
    at[::5] = -1
    f, _ = rotary.rotary_frequencies(rotated, base=10000.0, device="cpu")
    qd, kd = on_gpu(q, k, x)
    for factor in (1.0, 1.25):
        got = rotary.apply_rotary(qd, kd, at.cuda(), f.cuda(), factor=factor, interleaved=interleaved)
        for y, z in zip((q, k), got):
            assert z.dtype == y.dtype and z.shape == y.shape and z.is_contiguous()
            within(z, *ref.rotary(y, at, f, factor, interleaved))
    assert T.equal(qd.cpu(), q) and T.equal(kd.cpu(), k)  # the inputs stay


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(torch_cuda, interleaved):
    # every position of an int32 and frequencies of all sizes; positions that follow a quarter of a turn closely
    T = torch_cuda
    at = T.tensor([0, 1, 2, 1000003, 2 ** 24 + 1, 2 ** 30 + 12345, 2 ** 31 - 1, -1, -2 ** 31, 999999], dtype=T.int32)
    q, k, x = inputs(T, 5, len(at), 3, 1, 64, T.float32)
    f = T.cat([10000.0 ** (-T.arange(16, dtype=T.float64) / 16), T.arange(1, 9, dtype=T.float64) * math.pi / 4,
               T.tensor([0.0, 1e-30, -0.5, 3.0, -1e-3, 2 * math.pi, 1.0, 7.0], dtype=T.float64)])
    qd, kd = on_gpu(q, k, x)
    for y, z in zip((q, k), rotary.apply_rotary(qd, kd, at.cuda(), f.cuda(), interleaved=interleaved)):
        within(z, *ref.rotary(y, at, f, 1.0, interleaved))


def test_tokens_past_32_bits(torch_cuda):
    # more than 2^31 elements of q: the same few tokens again and again, into an output and in place
    T = torch_cuda
    q, _, _ = inputs(T, 10, 64, 32, 1, 128, T.bfloat16)
    at, f = T.arange(100, 164, dtype=T.int32, device="cuda"), rotary.rotary_frequencies(128)[0]
    want = rotary.apply_rotary(q.cuda(), None, at, f)[0]
    many = q.cuda().repeat(8200, 1, 1)
    assert many.numel() > 2 ** 31
    got = rotary.apply_rotary(many, None, at.repeat(8200), f)[0]
    assert (got.view(8200, 64, 32, 128) == want).all()
    del got
    rotary.apply_rotary(many, None, at.repeat(8200), f, inplace=True)
    assert (many.view(8200, 64, 32, 128) == want).all()


def test_turned_back(torch_cuda):
    # negated frequencies undo a rotation, whatever is left of it is the two roundings
    T = torch_cuda
    q, k, x = inputs(T, 6, 50, 4, 2, 128, T.float32)
    at = T.arange(1000, 1050, dtype=T.int32, device="cuda")
    f, _ = rotary.rotary_frequencies(128)
    qd, kd = on_gpu(q, k, x)
    back = rotary.apply_rotary(*rotary.apply_rotary(qd, kd, at, f), at, -f)
    for y, z in zip((q, k), back):
        size = y[..., :64].abs() + y[..., 64:].abs()  # (8 * 2^-24 of both channels: four roundings in each rotation)
        assert ((z.cpu() - y).abs() <= 8 * 2.0 ** -24 * size.repeat(1, 1, 2)).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rotated", [(128, 128), (128, 64), (64, 20)])
def test_in_place(torch_cuda, dim, rotated, interleaved):
    T = torch_cuda
    q, k, x = inputs(T, 7, 70, 6, 2, dim, T.bfloat16)
    at = T.arange(70, dtype=T.int32)
    at[60:] = -1
    f, _ = rotary.rotary_frequencies(rotated, device="cpu")
    y = x.cuda()
    qd, kd = (y.as_strided(t.shape, t.stride(), t.storage_offset()) for t in (q, k))
    want = rotary.apply_rotary(qd, kd, at.cuda(), f.cuda(), interleaved=interleaved)
    got = rotary.apply_rotary(qd, kd, at.cuda(), f.cuda(), interleaved=interleaved, inplace=True)
    assert got[0] is qd and got[1] is kd
    assert T.equal(want[0], qd) and T.equal(want[1], kd)
    assert T.equal(y[:, 8 * dim:].cpu(), x[:, 8 * dim:])  # what is neither stays


def test_shapes_that_callers_have(torch_cuda):
    T = torch_cuda
    q, k, x = inputs(T, 8, 24, 4, 2, 64, T.bfloat16)
    f, _ = rotary.rotary_frequencies(64)
    at = T.arange(24, dtype=T.int32, device="cuda")
    qd, kd = on_gpu(q, k, x)
    want = rotary.apply_rotary(qd, kd, at, f)
    only, none = rotary.apply_rotary(qd, None, at, f)
    assert none is None and T.equal(only, want[0])
    # (B, new, H, D), also where the tokens do not follow one stride
    four = rotary.apply_rotary(qd.view(8, 3, 4, 64), kd.view(8, 3, 2, 64), at.view(8, 3), f)
    assert four[0].shape == (8, 3, 4, 64) and T.equal(four[0].view(24, 4, 64), want[0])
    assert T.equal(four[1].view(24, 2, 64), want[1])
    turned = rotary.apply_rotary(qd.view(8, 3, 4, 64).transpose(0, 1), None, at.view(8, 3).t().contiguous(), f)[0]
    assert T.equal(turned.transpose(0, 1).reshape(24, 4, 64), want[0])
    # channels that do not stand next to one another
    odd = qd.transpose(1, 2).contiguous().transpose(1, 2)
    assert T.equal(rotary.apply_rotary(odd, None, at, f)[0], want[0])
    empty = rotary.apply_rotary(qd[:0], kd[:0], at[:0], f)
    assert empty[0].shape == (0, 4, 64) and empty[1].shape == (0, 2, 64)


def test_python_refuses(torch_cuda):
    T = torch_cuda
    q, k = T.zeros(4, 2, 64, device="cuda"), T.zeros(4, 1, 64, device="cuda")
    at, f = T.zeros(4, dtype=T.int32, device="cuda"), T.zeros(32, dtype=T.float64, device="cuda")
    for args in ((q.double(), k, at, f), (q, k.half(), at, f), (q, k[:3], at, f), (q, k[..., :32], at, f),
                 (q, k, at.long(), f), (q, k, at[:3], f), (q, k, at, f.float()), (q, k, at, f[:0]),
                 (q, k, at, T.zeros(33, dtype=T.float64, device="cuda")), (q[0], k, at, f), (q.cpu(), k, at, f)):
        with pytest.raises(ValueError):
            rotary.apply_rotary(*args)
    for wrong in (q[:1].expand(4, 2, 64), q.transpose(1, 2).contiguous().transpose(1, 2)):
        with pytest.raises(ValueError, match="in place"):
            rotary.apply_rotary(wrong, None, at, f, inplace=True)


def test_in_place_of_one_another(torch_cuda):
    # q and k of one buffer: rows that follow one another, heads that alternate, and places in common
    T = torch_cuda
    x = T.randn(10, 12, 64, device="cuda")
    f, at = rotary.rotary_frequencies(64)[0], T.arange(10, dtype=T.int32, device="cuda")
    for q, k in ((x[:, :8], x[:, 8:10]), (x[:, 4:], x[:, :2]), (x[:, ::3], x[:, 1::3]), (x[:, 2::3], x[:, ::3]),
                 (x[:4], x[4:8]), (x[:1, :3], x[:1, 3:]), (x[:1, ::2], x[:1, 1::2]), (x[2:6, :1], x[2:6, 5:6])):
        n = q.shape[0]
        want = rotary.apply_rotary(q, k, at[:n], f)
        got = rotary.apply_rotary(q, k, at[:n], f, inplace=True)
        assert T.equal(got[0], want[0]) and T.equal(got[1], want[1])
    for q, k in ((x, x), (x[:, :8], x[:, 7:]), (x[:, ::3], x[:, 3::3]), (x[:, 4:], x[:, :5]), (x[:6, :6], x[4:, :6]),
                 (x[:1], x[:1]), (x[:1, :4], x[:1, 3:]), (x[..., :32], x[..., 16:48])):
        before = x.clone()
        with pytest.raises(ValueError):
            rotary.apply_rotary(q, k, at[:q.shape[0]], f[:8], inplace=True)
        assert T.equal(x, before)


def test_in_a_graph_and_on_a_stream(torch_cuda):
    T = torch_cuda
    q, k, x = inputs(T, 9, 300, 8, 2, 128, T.bfloat16)
    qd, kd = on_gpu(q, k, x)
    at, f = T.arange(300, dtype=T.int32, device="cuda"), rotary.rotary_frequencies(128)[0]
    side = T.cuda.Stream()
    side.wait_stream(T.cuda.current_stream())
    with T.cuda.stream(side):
        warm = rotary.apply_rotary(qd, kd, at, f)
    T.cuda.current_stream().wait_stream(side)
    graph = T.cuda.CUDAGraph()
    with T.cuda.graph(graph):
        got = rotary.apply_rotary(qd, kd, at, f)
    for step in range(3):
        at += 1000 * step
        graph.replay()
        want = rotary.apply_rotary(qd, kd, at, f)
        T.cuda.synchronize()
        assert T.equal(got[0], want[0]) and T.equal(got[1], want[1])
        assert step or (T.equal(warm[0], want[0]) and T.equal(warm[1], want[1]))
