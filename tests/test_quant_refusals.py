"""Rotary positions and the quantised paged cache refuse what they do not take, before
any launch (no GPU: pointers are numbers that nothing reads); the frequencies are
their formulas; and the references that the GPU tests compare with hold what they
are said to."""
import math

import numpy as np
import pytest
import torch

import quant_testutil as ref
import zipserv_asplos26_amd as zs
from zipserv_asplos26_amd import _lib, attention, paged, rotary

P = 1 << 20  # an aligned address that no refused call reads
INVAL, UNSUPPORTED, OVERFLOW = _lib.ZS_E_INVAL, _lib.ZS_E_UNSUPPORTED, _lib.ZS_E_OVERFLOW


def call(fn, defaults, **changed):
    assert set(changed) <= set(defaults)
    return getattr(zs.lib(), fn)(0, *{**defaults, **changed}.values())


ROTARY = dict(q=P, qt=4096, qh=128, qo=P + 4096, qot=4096, qoh=128, heads=32, k=P, kt=1024, kh=128, ko=P, kot=1024, koh=128,
              heads_k=8, type=0, positions=P, tokens=4, dim=128, frequencies=P, pairs=64, factor=1.0, interleaved=0)


@pytest.mark.parametrize("changed,status", [
    *[({n: 0}, INVAL) for n in ("q", "qo", "k", "ko", "positions", "frequencies", "dim", "pairs")],
    *[({n: -1}, INVAL) for n in ("heads", "heads_k", "tokens", "type", "pairs")],
    *[({n: P + 1}, INVAL) for n in ("q", "qo", "k", "ko", "positions")],
    (dict(frequencies=P + 4), INVAL), (dict(type=3), INVAL), (dict(pairs=65), INVAL), (dict(type=2, q=P + 2), INVAL),
    (dict(dim=2048, pairs=513), UNSUPPORTED), (dict(dim=1 << 27), OVERFLOW),
    (dict(tokens=0, q=0, k=0, positions=0), _lib.ZS_OK), (dict(heads=0, heads_k=0), _lib.ZS_OK)])
def test_rotary_refuses(changed, status):
    assert call("zs_rotary", ROTARY, **changed) == status


APPEND = dict(k=P, v=P, kt=1024, kh=128, vt=1024, vh=128, slots=P, n=4, cache=P, blocks=8, page=16, heads=8, dim=128,
              bits=4)
READ = dict(cache=P, blocks=8, page=16, heads=8, dim=128, bits=4, slots=P, n=4, k=P, v=P)
POOL = [*[({n: 0}, INVAL) for n in ("cache", "blocks", "page", "heads")], (dict(cache=P + 8), INVAL),
        (dict(page=20), UNSUPPORTED), (dict(dim=96), UNSUPPORTED), (dict(dim=256), UNSUPPORTED),
        (dict(bits=2), UNSUPPORTED), (dict(bits=16), UNSUPPORTED), (dict(heads=65536), UNSUPPORTED),
        (dict(blocks=1 << 27), OVERFLOW), (dict(blocks=1, page=1 << 24), OVERFLOW)]


@pytest.mark.parametrize("changed,status", POOL + [
    *[({n: 0}, INVAL) for n in ("k", "v", "slots")], *[({n: P + 8}, INVAL) for n in ("k", "v")],
    *[({n: 1020}, INVAL) for n in ("kt", "kh", "vt", "vh")], (dict(n=-1), INVAL),
    (dict(n=1 << 20, heads=256), OVERFLOW), (dict(n=0, k=0, v=0, slots=0), _lib.ZS_OK)])
def test_append_refuses(changed, status):
    assert call("zs_paged_append_quant", APPEND, **changed) == status


@pytest.mark.parametrize("changed,status", POOL + [
    *[({n: 0}, INVAL) for n in ("k", "v", "slots")], *[({n: P + 8}, INVAL) for n in ("k", "v")], (dict(n=-1), INVAL),
    (dict(n=1 << 20, heads=256), OVERFLOW), (dict(n=0, k=0, v=0, slots=0), _lib.ZS_OK)])
def test_read_refuses(changed, status):
    assert call("zs_paged_read_quant", READ, **changed) == status


ATTEND = dict(q=P, qb=4096, qt=4096, qh=128, cache=P, blocks=8, page=16, bits=4, table=P, stride=64, width=64, lens=P,
              batch=2, new=1, heads=32, heads_k=8, dim=128, scale=0.1, out=P, lse=P, ws=0, ws_bytes=0, splits=1)


@pytest.mark.parametrize("changed,status", [
    *[({n: 0}, INVAL) for n in ("q", "cache", "table", "lens", "out", "batch", "new", "heads", "heads_k", "width",
                                "blocks", "page")],
    *[({n: P + 8}, INVAL) for n in ("q", "cache", "out", "ws")], (dict(qb=4), INVAL), (dict(qt=4), INVAL),
    (dict(qh=130), INVAL), (dict(stride=63), INVAL), (dict(heads=30), INVAL), (dict(splits=-1), INVAL),
    (dict(splits=2), INVAL), (dict(splits=2, ws=P, ws_bytes=64 * 2 * 130 * 4 - 1), INVAL), (dict(page=40), UNSUPPORTED),
    (dict(dim=80), UNSUPPORTED), (dict(bits=5), UNSUPPORTED), (dict(blocks=1 << 27), OVERFLOW),
    (dict(batch=1 << 20, new=1 << 10), OVERFLOW), (dict(batch=1 << 20, heads=64, heads_k=64), OVERFLOW),
    (dict(width=2 ** 31 - 1, stride=1 << 31, page=32), OVERFLOW),
    (dict(batch=65535, heads=65535, heads_k=65535), OVERFLOW),
    (dict(width=1 << 28, stride=1 << 28, splits=1 << 24, ws=P, ws_bytes=1 << 60), OVERFLOW)])
def test_attention_refuses(changed, status):
    assert call("zs_decode_attention_quant_paged", ATTEND, **changed) == status


def test_size_queries():
    L = zs.lib()
    assert L.zs_quant_record_bytes(16, 128, 4) == 16 * 136 and L.zs_quant_record_bytes(48, 64, 8) == 48 * 136
    assert [L.zs_quant_record_bytes(*a) for a in ((0, 128, 4), (16, 100, 4), (16, 128, 6))] == [-1, -1, -1]
    query = L.zs_decode_attention_quant_workspace_bytes
    assert query(1, 1, 32, 8, 128, 64, 16, 1) == 0 and query(0, 1, 32, 8, 128, 64, 16, 4) == 0
    assert query(1, 1, 32, 8, 128, 640, 16, 4) >= 32 * 4 * 130 * 4
    assert query(2, 3, 32, 8, 64, 640, 16, 4) >= 2 * 3 * 32 * 4 * 66 * 4
    # short tables are not cut, and no more splits are made than there are 128-token pieces
    assert query(1, 1, 32, 8, 128, 8, 16, 0) == 0 and query(1, 1, 32, 8, 128, 8, 16, 9) == 0


def test_python_takes_gpu_tensors_of_its_shapes_only():
    x = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    f = torch.zeros(64, dtype=torch.float64)
    cache = paged.quantized_kv_cache(4, 16, 8, 128, device="cpu")
    assert cache.data.shape == (4, 8, 16 * 136)
    assert paged.quantized_kv_cache(4, 16, 8, 64, bits=8, device="cpu").data.shape == (4, 8, 16 * 136)
    for wrong in (dict(bits=3), dict(head_dim=80), dict(page_block_size=24), dict(page_block_size=0)):
        with pytest.raises(ValueError):
            paged.quantized_kv_cache(**{**dict(num_blocks=4, page_block_size=16, num_heads_k=8, head_dim=128,
                                               device="cpu"), **wrong})
    for fn in (lambda: paged.append_paged_kv_quantized(x, x, cache, i), lambda: paged.read_paged_kv_quantized(cache, i),
               lambda: attention.flash_attn_with_kvcache_quantized(x, cache, i.view(2, 1), i),
               lambda: rotary.apply_rotary(x, x, i, f)):
        with pytest.raises(ValueError, match="CUDA"):
            fn()
    with pytest.raises(ValueError, match="QuantizedKVCache"):
        paged.read_paged_kv_quantized(cache.data, i)


def test_frequencies():
    none, one = rotary.rotary_frequencies(128, base=500000.0, device="cpu")
    assert none.dtype == torch.float64 and none.shape == (64,) and one == 1.0
    assert none[0] == 1.0 and abs(float(none[1]) - 500000.0 ** (-1 / 64)) < 1e-15
    linear, _ = rotary.rotary_frequencies(128, base=500000.0, scaling="linear", stretch=4.0, device="cpu")
    assert torch.equal(linear, none / 4)
    base, _ = rotary.rotary_frequencies(128, base=500000.0, scaling="base", stretch=4.0, device="cpu")
    assert base[0] == 1.0 and abs(float(base[-1] / none[-1]) - 0.25) < 1e-12
    turns = 8192 * none / (2 * math.pi)
    bands, _ = rotary.rotary_frequencies(128, base=500000.0, scaling="bands", stretch=8.0, trained=8192, device="cpu")
    assert torch.equal(bands[turns >= 4], none[turns >= 4])
    assert torch.allclose(bands[turns <= 1], none[turns <= 1] / 8, rtol=1e-15, atol=0)
    mid = (turns > 1) & (turns < 4)
    share = (turns[mid] - 1) / 3
    assert mid.any() and torch.allclose(bands[mid], none[mid] * share + none[mid] / 8 * (1 - share), rtol=1e-14, atol=0)
    ramp, factor = rotary.rotary_frequencies(128, scaling="ramp", stretch=16.0, trained=4096, device="cpu")
    plain, _ = rotary.rotary_frequencies(128, device="cpu")
    turns = 4096 * plain / (2 * math.pi)
    assert abs(factor - (0.1 * math.log(16.0) + 1)) < 1e-15
    assert torch.equal(ramp[turns >= 40], plain[turns >= 40]) and torch.allclose(ramp[turns <= 0.8],
                                                                                  plain[turns <= 0.8] / 16)
    assert (ramp.diff() < 0).all()
    for wrong in (dict(rotated=3), dict(rotated=0), dict(rotated=8, scaling="other"), dict(rotated=8, base=0.0),
                  dict(rotated=8, scaling="bands", stretch=2.0), dict(rotated=2, scaling="base", stretch=2.0)):
        with pytest.raises(ValueError):
            rotary.rotary_frequencies(**wrong, device="cpu")


@pytest.mark.parametrize("bits", [4, 8])
def test_reference_quantisation_is_half_a_step_off(bits):
    g = torch.Generator().manual_seed(bits)
    x = torch.randn(50, 64, generator=g).mul_(torch.randn(50, 1, generator=g).mul(20).exp()).to(torch.bfloat16)
    codes, scale, low = ref.quantize(x, bits)
    s, m = (torch.from_numpy((a.astype(np.uint32) << 16).view(np.float32)).double()[:, None] for a in (scale, low))
    off = (torch.from_numpy(codes) * s + m - x.double()).abs()
    assert codes.min() >= 0 and codes.max() == 2 ** bits - 1
    assert (off <= s / 2 + 2.0 ** -24 * (x.double() - m)).all()


@pytest.mark.parametrize("dim,bits", [(64, 4), (128, 4), (64, 8), (128, 8)])
def test_reference_layout_holds_every_code_once(dim, bits):
    where = ref.places(dim, bits)
    assert len(set(where)) == dim and {b for b, _ in where} == set(range(dim * bits // 8))
    # what was appended is read back
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(5, 2, dim, generator=g).to(torch.bfloat16) for _ in range(2))
    data = np.zeros((2, 2, ref.record_bytes(16, dim, bits)), dtype=np.uint8)
    slots = torch.tensor([3, 31, -1, 16, 0])
    ref.append(k, v, data, slots, 16, dim, bits)
    got = ref.read(data, slots, 16, dim, bits)
    step = 8.0 / (2 ** bits - 1)
    for x, y in zip((k, v), got):
        live = slots >= 0
        assert ((x - y).abs()[live] <= step).all() and (y[~live] == 0).all()
