"""Refusals of the paged-cache and sampling entry points on the host (nothing is launched), and the 64-bit forms that
the GPU tests go by, against hand-made cases."""

import ctypes
import math

import pytest
import torch

from axiomlm_amd import _lib
from oracle import serving

P = 4096  # an address that is never followed


def desc(**change):
    d = dict(k=P, v=2 * P, k_scales=P, v_scales=P, block_table=P, page_stride=2 * 16 * 128, scale_stride=2 * 16 * 2,
             kv_dtype=0, n_kv_head=2, head_dim=64, page_size=16, n_pages=3, n_seqs=2, max_pages=4)
    d.update(change)
    return _lib.PagedKv(**d)


BAD_DESC = [dict(k=None), dict(v=None), dict(block_table=None), dict(head_dim=96), dict(head_dim=0), dict(kv_dtype=3),
            dict(kv_dtype=-1), dict(kv_dtype=1, k_scales=None), dict(kv_dtype=2, v_scales=None), dict(page_size=12),
            dict(page_size=8), dict(page_size=2048), dict(n_kv_head=0), dict(n_pages=0), dict(n_seqs=0),
            dict(max_pages=0), dict(max_pages=1 << 28), dict(page_stride=4080), dict(page_stride=4097), dict(k=P + 8),
            dict(kv_dtype=1, page_stride=2048, scale_stride=60), dict(kv_dtype=1, k_scales=P + 2)]


def refused(rc, text=None):
    msg = _lib.lib().axm_last_error().decode()
    assert rc < 0 and msg
    assert text is None or text in msg, msg


@pytest.mark.parametrize("bad", BAD_DESC, ids=str)
def test_bad_caches_are_refused_by_every_entry(bad):
    L = _lib.lib()
    d = ctypes.byref(desc(**bad))
    refused(L.axm_paged_flash_decode(P, 512, d, P, P, 8, None, 0, P, 1 << 30, None))
    refused(L.axm_rope_paged_kv_write(P, 1024, 1, P, 10, P, None, None, None, d, 512, None))
    refused(L.axm_evict_paged_kv(d, 1, 0, 0, P, P, 64, 8, 2, P + 64, P, P, None))


def test_decode_refusals():
    L, d = _lib.lib(), ctypes.byref(desc())
    good = [P, 512, d, P, P, 8, None, 0, P, 1 << 30, None]
    for at, value, text in ((0, None, "null"), (3, None, "null"), (4, None, "null"), (5, 7, "n_head"), (5, 0, "n_head"),
                            (5, 1024, "n_head"), (1, 511, "aligned"), (1, 504, "aligned"), (0, P + 8, "aligned")):
        args = list(good)
        args[at] = value
        refused(L.axm_paged_flash_decode(*args), text)
    args = list(good)
    args[6], args[7] = P, 63  # an account shorter than the table
    refused(L.axm_paged_flash_decode(*args), "mass")
    need = L.axm_paged_decode_workspace_bytes(2, 8, 2, 64, 16, 4, 1)
    assert need > 0
    args[7], args[9] = 64, need - 1
    refused(L.axm_paged_flash_decode(*args), "workspace")


def test_write_refusals():
    L, d = _lib.lib(), ctypes.byref(desc())
    good = [P, 768, 1, P, 10, P, None, None, None, d, 512, None]
    for at, value in ((0, None), (3, None), (5, None), (2, 0), (2, 1 << 21), (4, 0), (10, 500), (10, 0), (1, 767), (1, 760),
                      (0, P + 2)):
        args = list(good)
        args[at] = value
        refused(L.axm_rope_paged_kv_write(*args))


def test_evict_refusals():
    L, d = _lib.lib(), ctypes.byref(desc())
    good = [d, 2, 1 << 20, 0, P, P, 64, 8, 2, 2 * P, P, P, None]
    for at, value in ((1, 0), (4, None), (5, None), (9, None), (10, None), (11, None), (9, P), (6, 63), (7, 0), (8, -1),
                      (8, 9), (2, 0), (2, 1000)):
        args = list(good)
        args[at] = value
        refused(L.axm_evict_paged_kv(*args))
    refused(L.axm_evict_paged_kv(ctypes.byref(desc(v=P)), *good[1:]), "same pages")


def test_sampling_refusals():
    L = _lib.lib()
    good = [P, 0, 100, 2, 100, P, None, None, None, None, 1.0, 0, 1.0, 0.0, P, None, None, 0, None]
    for at, value in ((0, None), (5, None), (14, None), (1, 3), (1, -1), (2, 99), (3, 0), (3, 1 << 22), (4, 0),
                      (4, (1 << 24) + 1)):
        args = list(good)
        args[at] = value
        if at == 4:
            args[2] = max(args[2], value)
        refused(L.axm_sample_rows(*args))


# ---- the 64-bit forms -----------------------------------------------------------------------------------------------
def test_oracle_formats():
    v = serving.e4m3_values()
    ref = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(v.nan_to_num(1e9), ref.nan_to_num(1e9))
    assert serving.code_values(torch.tensor([0x8F, 0x70], dtype=torch.uint8), "int4").tolist() == [-1, -8, 0, 7]


def test_oracle_decode_by_hand():
    k = torch.zeros(3, 1, 8, 64, dtype=torch.float16)
    v = torch.zeros_like(k)
    table = torch.tensor([[2, 0]])
    k[2, 0, 7, 0], k[0, 0, 0, 0] = 8 * math.log(3), 0.0  # slots 7 and 8; q = 1: scores log 3 and 0
    v[2, 0, 7], v[0, 0, 0] = 1.0, 2.0
    q = torch.zeros(1, 1, 64, dtype=torch.float16)
    q[0, 0, 0] = 1.0
    mass = torch.zeros(1, 1, 16)
    out, bound, mass, _ = serving.decode(q, k, v, table, [9], mass=mass)
    assert torch.allclose(out, torch.full_like(out, (3 + 2) / 11), atol=2e-3)  # seven more keys of score 0
    assert abs(mass.sum().item() - 1) < 1e-12 and mass[0, 0, 7].item() == pytest.approx(3 / 11, abs=1e-3)
    assert bool((bound > 0).all()) and bool((bound < 4e-3).all())


def test_oracle_eviction_by_hand():
    nan = float("nan")
    assert serving.evict_choice([5, 1, 5, 5, 0, 9], 6, 3, 1) == [0, 2, 5]
    assert serving.evict_choice([nan, -1.0, nan, 3.0, 0, 0], 6, 5, 2) == [0, 1, 3, 4, 5]
    assert serving.evict_choice([1, 2, 3], 3, 3, 0) == [0, 1, 2]
    assert serving.evict_choice([1, 2, 3, 4], 4, 2, 2) == [2, 3]


def test_oracle_sampling_by_hand():
    z = torch.log(torch.tensor([1.0, 4.0, 3.0, 2.0]))
    row = lambda *a: serving.sample_row(z, *a)  # noqa: E731
    assert row(0.05, 1.0, 0, 1.0, 0.0)[0] == 0 and row(0.45, 1.0, 0, 1.0, 0.0)[0] == 1
    assert row(0.99, 1.0, 2, 1.0, 0.0) == (2, pytest.approx(3 / 7))
    assert row(0.99, 1.0, 0, 0.39, 0.0) == (1, pytest.approx(1.0))   # 0.4 reaches 0.39
    assert row(0.99, 1.0, 0, 0.41, 0.0) == (2, pytest.approx(3 / 7))
    assert row(0.0, 1.0, 0, 1.0, 0.6) == (1, pytest.approx(4 / 7))
    assert row(0.3, 0.0, 0, 1.0, 0.0) == (1, 1.0)
    assert serving.sample_row(torch.full((5,), -math.inf), 0.5, 1.0, 0, 1.0, 0.0) == (-1, 0.0)
    assert serving.sample_row(torch.tensor([0.0, math.inf, 1.0, math.inf]), 0.6, 1.0, 0, 1.0, 0.0) == (3, 0.5)
