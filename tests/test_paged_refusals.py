"""The paged-cache entry points refuse what they do not take, before any launch
(no GPU: pointers are numbers that nothing reads), and the references that the GPU
tests compare with hold what they are said to."""
import itertools

import pytest
import torch

import paged_testutil as ref
import zipserv_asplos26_amd as zs
from zipserv_asplos26_amd import _lib, paged

P = 1 << 20  # an aligned address that no refused call reads
INVAL, UNSUPPORTED, OVERFLOW = _lib.ZS_E_INVAL, _lib.ZS_E_UNSUPPORTED, _lib.ZS_E_OVERFLOW


def call(fn, defaults, **changed):
    assert set(changed) <= set(defaults)
    return getattr(zs.lib(), fn)(0, *{**defaults, **changed}.values())


PLAN = dict(context=P, new=P, batch=4, table=P, stride=8, width=8, free=P, capacity=16, num_free=P, page=16,
            most=64, slots=P, sequences=P, positions=P, seqlens=P, cu=P, counts=P)


@pytest.mark.parametrize("changed,status", [
    *[({n: 0}, INVAL) for n in ("context", "new", "table", "free", "num_free", "slots", "sequences", "positions",
                                "seqlens", "cu", "counts")],
    (dict(batch=0), INVAL), (dict(batch=-1), INVAL), (dict(batch=4097), UNSUPPORTED), (dict(width=0), INVAL),
    (dict(stride=7), INVAL), (dict(capacity=-1), INVAL), (dict(page=0), INVAL), (dict(page=-16), INVAL),
    (dict(page=8), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(most=-1), INVAL)])
def test_plan_refuses(changed, status):
    assert call("zs_paged_plan", PLAN, **changed) == status


APPEND = dict(k=P, v=P, kt=1024, kh=128, vt=1024, vh=128, slots=P, n=4, kc=P, vc=P, bounds=P, blocks=8, page=16,
              heads=8, dim=128)


@pytest.mark.parametrize("changed,status", [
    *[({n: 0}, INVAL) for n in ("k", "v", "slots", "kc", "vc", "blocks", "page", "heads")],
    *[({n: P + 8}, INVAL) for n in ("k", "v", "kc", "vc", "bounds")],
    *[({n: 1020}, INVAL) for n in ("kt", "kh", "vt", "vh")],
    (dict(n=-1), INVAL), (dict(page=20), UNSUPPORTED), (dict(dim=96), UNSUPPORTED), (dict(dim=256), UNSUPPORTED),
    (dict(heads=65536), UNSUPPORTED), (dict(blocks=1 << 27), OVERFLOW), (dict(n=0, k=0, v=0, slots=0), _lib.ZS_OK)])
def test_append_refuses(changed, status):
    assert call("zs_paged_append", APPEND, **changed) == status


SELECT = dict(q=P, qb=4096, qh=128, bounds=P, blocks=8, page=16, table=P, stride=8, width=8, lens=P, batch=2,
              heads=32, heads_k=8, dim=128, top_k=4, sink=1, local=1, pages=P, ws=P, ws_bytes=2 * 8 * 8 * 8)


@pytest.mark.parametrize("changed,status", [
    *[({n: 0}, INVAL) for n in ("q", "bounds", "table", "lens", "pages", "ws", "batch", "heads", "heads_k", "width",
                                "top_k", "blocks", "page")],
    (dict(q=P + 2), INVAL), (dict(bounds=P + 8), INVAL), (dict(ws=P + 4), INVAL), (dict(qb=4), INVAL),
    (dict(qh=130), INVAL), (dict(stride=7), INVAL), (dict(heads=30), INVAL), (dict(sink=-1), INVAL),
    (dict(local=-1), INVAL), (dict(sink=2, local=3), INVAL), (dict(sink=2147483647, local=2147483647), INVAL),
    (dict(ws_bytes=2 * 8 * 8 * 8 - 1), INVAL), (dict(page=40), UNSUPPORTED), (dict(dim=80), UNSUPPORTED),
    (dict(heads=136), UNSUPPORTED), (dict(batch=65536, ws_bytes=1 << 40), UNSUPPORTED),
    (dict(blocks=1 << 27), OVERFLOW), (dict(width=2 ** 31 - 1, stride=1 << 31, ws_bytes=1 << 50), OVERFLOW)])
def test_select_refuses(changed, status):
    assert call("zs_select_kv_pages", SELECT, **changed) == status


SPARSE = dict(q=P, qb=4096, qh=128, kc=P, vc=P, blocks=8, page=16, table=P, stride=8, width=8, pages=P, top_k=4,
              lens=P, batch=2, heads=32, heads_k=8, dim=128, scale=0.1, out=P, lse=P, ws=0, ws_bytes=0, splits=1)


@pytest.mark.parametrize("changed,status", [
    *[({n: 0}, INVAL) for n in ("q", "kc", "vc", "table", "pages", "lens", "out", "batch", "heads", "heads_k",
                                "width", "top_k", "blocks", "page")],
    *[({n: P + 8}, INVAL) for n in ("q", "kc", "vc", "out", "ws")],
    (dict(qb=4), INVAL), (dict(qh=130), INVAL), (dict(stride=7), INVAL), (dict(heads=30), INVAL),
    (dict(splits=-1), INVAL), (dict(top_k=64, splits=2), INVAL), (dict(page=40), UNSUPPORTED),
    (dict(dim=80), UNSUPPORTED), (dict(heads=136), UNSUPPORTED), (dict(batch=65536), UNSUPPORTED),
    (dict(blocks=1 << 27), OVERFLOW), (dict(top_k=1 << 30, page=48), OVERFLOW)])
def test_sparse_attention_refuses(changed, status):
    assert call("zs_decode_attention_sparse_paged", SPARSE, **changed) == status


def test_workspace_queries():
    L = zs.lib()
    assert L.zs_select_kv_pages_workspace_bytes(3, 8, 100) >= 3 * 8 * 100 * 8
    assert L.zs_select_kv_pages_workspace_bytes(0, 8, 100) == 0
    assert L.zs_decode_attention_sparse_workspace_bytes(1, 32, 8, 128, 64, 16, 1) == 0
    assert L.zs_decode_attention_sparse_workspace_bytes(1, 32, 8, 128, 64, 16, 4) >= 32 * 4 * 130 * 4
    # no more splits than there are 128-token pieces of the lists
    assert L.zs_decode_attention_sparse_workspace_bytes(1, 32, 8, 128, 4, 16, 4) == 0


def test_python_takes_gpu_tensors_only():
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    pool = torch.zeros(4, 16, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        paged.plan_paged_step(i, i, i.view(2, 1), i, i[:1], 16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        paged.append_paged_kv(x, x, pool, pool, i)
    with pytest.raises(ValueError, match="CUDA"):
        paged.select_kv_pages(x, torch.zeros(4, 8, 2, 128, dtype=torch.bfloat16), i.view(2, 1), i, 16, 2)


def test_reference_plan_gives_every_token_a_place_of_its_own():
    table, slots, seqs, poss, lens, cu, counts = ref.plan([5, 0, 16, 40], [30, 1, 0, 9], [[3, 0, 0], [0] * 3, [4, 0, 0],
                                                          [5, 6, 7]], [9, 8, 2, 1], 4, 16, 48)
    assert cu == [0, 30, 31, 31, 40] and lens == [35, 1, 16, 48 + 0] and counts == [40, 3, 1, 1]
    live = [s for s in slots if s >= 0]
    assert len(set(live)) == len(live) == 39 and slots[40:] == [-1] * 8
    assert table[0] == [3, 1, 2] and table[1][0] == 8 and poss[39] == 48 and slots[39] == -1


def test_reference_bound_is_a_bound():
    # no key of a page scores more than the page
    g = torch.Generator().manual_seed(1)
    q = torch.randn(1, 4, 64, generator=g).to(torch.bfloat16)
    keys = torch.randn(3, 16, 2, 64, generator=g).to(torch.bfloat16)
    bounds = torch.stack([keys.amin(1), keys.amax(1)], 2)
    s = ref.scores(q, bounds, torch.arange(3).view(1, 3), 48, 16, 2, 0)
    for h, p in itertools.product(range(2), range(3)):
        most = (q[0, 2 * h:2 * h + 2].double() @ keys[p, :, h].double().t()).max()
        assert most <= s[h, p]


def test_python_refuses_numbers_that_a_c_int_does_not_hold():
    assert [paged._whole(n, "n") for n in (0, -1, 2 ** 31 - 1, True, 7.0)] == [0, -1, 2 ** 31 - 1, 1, 7]
    for n in (2 ** 31, 2 ** 32 + 4, -2 ** 31, -2 ** 32 + 1):
        with pytest.raises(ValueError, match="2\\^31"):
            paged._whole(n, "n")


@pytest.mark.parametrize("fn,defaults,changed", [
    # 2^24 workgroups of 256 threads, 2^25
    ("zs_paged_append", APPEND, dict(n=1 << 20, heads=256)),
    ("zs_paged_append", APPEND, dict(n=1 << 30, dim=64, heads=1)),
    # 2^26 workgroups of one wave, and 2^22 rows of 1024 threads, 2^23 of 512, 2^24 of 256
    ("zs_select_kv_pages", SELECT, dict(width=1 << 27, stride=1 << 27, ws_bytes=1 << 50)),
    ("zs_select_kv_pages", SELECT, dict(batch=1 << 14, heads=256, heads_k=256, width=2049, stride=2049,
                                        ws_bytes=1 << 50)),
    ("zs_select_kv_pages", SELECT, dict(batch=1 << 14, heads=512, heads_k=512, width=1025, stride=1025,
                                        ws_bytes=1 << 50)),
    ("zs_select_kv_pages", SELECT, dict(batch=1 << 14, heads=1024, heads_k=1024, width=8, ws_bytes=1 << 50)),
    # 2^24 splits of 256 threads; 2^24 (sequence, head) rows of the merge
    ("zs_decode_attention_sparse_paged", SPARSE, dict(top_k=1 << 27, splits=1 << 24, ws=P, ws_bytes=1 << 50)),
    ("zs_decode_attention_sparse_paged", SPARSE, dict(batch=1 << 14, heads=1024, heads_k=1024, top_k=64, splits=2,
                                                      ws=P, ws_bytes=1 << 50))])
def test_grids_of_2_to_the_32_threads_are_refused(fn, defaults, changed):
    # (a launch refuses them too, after others of the same call, and with a code of its own)
    assert call(fn, defaults, **changed) == OVERFLOW
