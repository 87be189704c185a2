"""The low-bit operators' refusals that need no GPU (arguments are checked before
any CUDA call), and the tests' own 64-bit forms."""
from __future__ import annotations

import ctypes as C

import pytest

from minimind_orangepi_b200._lib import Kv8Cache, lib

torch = pytest.importorskip("torch")

from lowbit_reference import block_scale, e4m3_round, e4m3_table  # noqa: E402

P = 1 << 20  # an aligned address that nothing reads: every call here is refused
INVALID = 1


def cache(**kw):
    f = dict(n_pages=4, layers=2, nkv=2, hd=64, max_seqs=3, max_pages=2, d_codes=P, d_scales=P, d_block_table=P,
             d_seq_pos=P, d_error=P)
    f.update(kw)
    return Kv8Cache(*f.values())


def append(c, layer=0, n_seqs=2, rows=2, max_new=1, slots=P, start=None, nq=4, qkv=P, qn=P, kn=P, cos=P, sin=P,
           max_pos=128, eps=1e-5, q=P):
    return lib().mmc_op_kv8_append(c, layer, n_seqs, rows, max_new, slots, start, nq, qkv, qn, kn, cos, sin, max_pos,
                                   eps, q, None)


def attend(c, layer=0, n_seqs=2, rows=2, max_new=1, slots=P, start=None, nq=4, q=P, max_ctx=128, out=P, ws=P,
           ws_bytes=1 << 30):
    return lib().mmc_op_kv8_attention(c, layer, n_seqs, rows, max_new, slots, start, nq, q, max_ctx, out, ws, ws_bytes,
                                      None)


BATCHES = [dict(layer=2), dict(layer=-1), dict(n_seqs=0), dict(n_seqs=65536, rows=65536), dict(rows=0),
           dict(rows=3), dict(max_new=2, rows=2), dict(max_new=0), dict(max_new=3, start=P), dict(slots=None),
           dict(nq=3), dict(nq=0), dict(nq=-2)]
CACHES = [dict(hd=48), dict(hd=0), dict(hd=256), dict(n_pages=0), dict(layers=0), dict(nkv=0), dict(max_seqs=0),
          dict(max_pages=0), dict(d_codes=None), dict(d_scales=None), dict(d_block_table=None), dict(d_seq_pos=None),
          dict(d_error=None), dict(d_codes=P + 8), dict(d_scales=P + 4), dict(n_pages=1 << 30)]


@pytest.mark.parametrize("kw", BATCHES + [dict(qkv=None), dict(qn=None), dict(kn=None), dict(cos=None),
                                          dict(sin=None), dict(q=None), dict(max_pos=0), dict(eps=-1.0),
                                          dict(eps=float("nan")), dict(qkv=P + 4), dict(q=P + 2)])
def test_append_refuses(kw):
    assert append(cache(), **kw) == INVALID and lib().mmc_last_error()


@pytest.mark.parametrize("kw", BATCHES + [dict(q=None), dict(out=None), dict(ws=None), dict(max_ctx=0),
                                          dict(q=P + 8), dict(out=P + 8), dict(ws=P + 4)])
def test_attention_refuses(kw):
    assert attend(cache(), **kw) == INVALID and lib().mmc_last_error()


@pytest.mark.parametrize("kw", CACHES)
def test_cache_refused(kw):
    assert append(cache(**kw)) == INVALID
    assert attend(cache(**kw)) == INVALID


def test_null_cache_refused():
    assert append(None) == INVALID and attend(None) == INVALID
    assert lib().mmc_op_kv8_status(None, None) == INVALID
    n = C.c_size_t()
    assert lib().mmc_op_kv8_attention_workspace_size(None, 1, 1, 1, 1, 1, C.byref(n)) == INVALID
    assert lib().mmc_op_kv8_attention_workspace_size(cache(), 1, 1, 1, 4, 1, None) == INVALID
    assert lib().mmc_op_kv8_attention_workspace_size(cache(), 1, 1, 1, 4, 0, C.byref(n)) == INVALID


@pytest.mark.parametrize("kw", [dict(batch=0), dict(batch=65536), dict(n=0), dict(k=0), dict(group=16),
                                dict(group=96), dict(k=96, group=64), dict(codes=None), dict(scales=None),
                                dict(x=None), dict(y=None), dict(codes=P + 8), dict(x=P + 8), dict(y=P + 8),
                                dict(scales=P + 1)])
def test_projection_refuses(kw):
    a = dict(batch=1, n=64, k=128, group=64, codes=P, scales=P, zeros=None, x=P, y=P)
    a.update(kw)
    assert lib().mmc_op_w4_projection(*a.values(), None) == INVALID and lib().mmc_last_error()


def test_reference_e4m3():
    """The tests' rounding against the format: every value is its own, halves go to the even code, and torch agrees."""
    t = e4m3_table()
    fine = t[~t.isnan()]
    assert torch.equal(e4m3_round(fine), fine)
    v = t[:127]
    even = torch.where(torch.arange(126) % 2 == 0, v[:-1], v[1:])
    assert torch.equal(e4m3_round((v[:-1] + v[1:]) / 2), even)
    x = torch.randn(4000, generator=torch.Generator().manual_seed(3)) * 40
    assert torch.equal(e4m3_round(x), x.to(torch.float8_e4m3fn).double())


def test_reference_scale():
    x = torch.tensor([448.0, 448.0000001, 449.0, 224.0, 1.75, 1.7500001, 0.0, 1e-45], dtype=torch.float64)
    assert block_scale(x).tolist() == [1.0, 2.0, 2.0, 0.5, 2.0 ** -8, 2.0 ** -7, 2.0 ** -126, 2.0 ** -126]


@pytest.mark.parametrize("kw", [dict(n_pages=2 ** 31 - 1, layers=2 ** 31 - 1), dict(n_pages=2 ** 31 - 1, nkv=4),
                                dict(layers=2 ** 31 - 1, nkv=4), dict(n_pages=2 ** 31 - 1, layers=2 ** 30, nkv=4),
                                dict(n_pages=1 << 30, layers=1 << 30, nkv=4)])
def test_cache_too_large_for_its_indexes_refused(kw):
    """Also where the product of the sizes passes 64 bits."""
    c, n = cache(**kw), C.c_size_t()
    assert append(c) == INVALID and b"too large" in lib().mmc_last_error()
    assert attend(c) == INVALID and b"too large" in lib().mmc_last_error()
    assert lib().mmc_op_kv8_attention_workspace_size(c, 2, 2, 1, 4, 128, C.byref(n)) == INVALID
