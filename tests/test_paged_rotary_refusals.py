"""Refusals of the rotation's entry points without a GPU: bad arguments before any launch."""

import ctypes

import pytest
import torch

from maskahead_amd import _native as N
from maskahead_amd.kernels.paged import rotary_table

E, U = N.MA_EINVAL, N.MA_EUNSUPPORTED


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from maskahead_amd.build import build

        build()
    return N.load()


def _pages(**kw):
    p = N.MaPages()
    p.pool = p.k_tail = p.v_tail = p.table = p.lengths = 4096
    p.num_pages, p.width, p.page_tokens, p.dtype = 8, 4, 64, N.MA_BF16
    p.s_pool[0], p.s_pool[1] = 2 * 10240, 10240
    for k, v in kw.items():
        setattr(p, k, v)
    return ctypes.byref(p)


def _t4(dtype=N.MA_BF16, ptr=4096):
    m = N.MaTensor4()
    m.ptr, m.dtype = ptr, dtype
    return m


def _rot(**kw):
    r = N.MaRotary()
    r.table, r.s_row, r.rows, r.dim = 4096, 64, 10, 64
    for k, v in kw.items():
        setattr(r, k, v)
    return ctypes.byref(r)


@pytest.mark.parametrize("kw", [dict(table=None), dict(rows=0), dict(rows=-1), dict(dim=0), dict(dim=24), dict(dim=80),
                                dict(dim=-16), dict(table=4104), dict(s_row=66)])
def test_a_bad_table_is_refused(lib, kw):
    r = _rot(**kw)
    assert lib.ma_rotate_block(_t4(), 4, _t4(), _t4(), 2, _t4(), 2, 1, 64, 4096, r, None) == E
    assert lib.ma_page_append_rotary(_pages(), _t4(), _t4(), 2, 2, 1, 64, 4096, 4096, r, _t4(), 4, _t4(), None) == E


def test_no_table_is_refused(lib):
    assert lib.ma_rotate_block(_t4(), 4, _t4(), _t4(), 2, _t4(), 2, 1, 64, 4096, None, None) == E
    assert lib.ma_page_append_rotary(_pages(), _t4(), _t4(), 2, 2, 1, 64, 4096, 4096, None, _t4(), 4, _t4(), None) == E


@pytest.mark.parametrize("rc,change", [
    (E, dict(q=_t4(ptr=None))), (E, dict(qo=_t4(ptr=None))), (E, dict(k=_t4(ptr=None))), (E, dict(ko=_t4(ptr=None))),
    (E, dict(hq=0)), (E, dict(hk=-1)), (E, dict(b=0)), (E, dict(t=0)), (U, dict(d=96)), (E, dict(lengths=None)),
    (U, dict(q=_t4(N.MA_F32))), (E, dict(qo=_t4(N.MA_F16))), (E, dict(k=_t4(N.MA_F16))), (E, dict(ko=_t4(N.MA_F32))),
    (U, dict(b=65536)), (U, dict(hq=4 * 65535)), (U, dict(hk=4 * 65535)), (U, dict(t=1 << 30))])
def test_bad_rows_are_refused(lib, rc, change):
    a = dict(q=_t4(), hq=4, qo=_t4(), k=_t4(), hk=2, ko=_t4(), b=2, t=1, d=64, lengths=4096)
    a.update(change)
    assert lib.ma_rotate_block(a["q"], a["hq"], a["qo"], a["k"], a["hk"], a["ko"], a["b"], a["t"], a["d"], a["lengths"],
                               _rot(), None) == rc


@pytest.mark.parametrize("rc,change", [
    (E, dict(k=_t4(ptr=None))), (E, dict(q=_t4(ptr=None))), (E, dict(qo=_t4(ptr=None))), (E, dict(hq=-1)),
    (E, dict(t=0)), (E, dict(q=_t4(N.MA_F16))), (E, dict(qo=_t4(N.MA_F16))), (E, dict(v=_t4(N.MA_F16))),
    (U, dict(d=96)), (U, dict(b=65536)), (U, dict(hq=4 * 65535)), (U, dict(t=(1 << 30) + 64)), (E, dict(p=dict(pool=4104))), (E, dict(p=dict(lengths=None)))])
def test_bad_appends_are_refused(lib, rc, change):
    a = dict(k=_t4(), v=_t4(), q=_t4(), hq=4, qo=_t4(), b=2, t=1, d=64, p={})
    a.update(change)
    assert lib.ma_page_append_rotary(_pages(**a["p"]), a["k"], a["v"], a["b"], 2, a["t"], a["d"], 4096, 4096, _rot(), a["q"],
                                     a["hq"], a["qo"], None) == rc


def test_tables_are_checked_and_built_on_the_cpu():
    for bad in (lambda: rotary_table(0, 128, device="cpu"), lambda: rotary_table(3, 128, rotary_dim=8, device="cpu"),
                lambda: rotary_table(3, 64, rotary_dim=80, device="cpu"),
                lambda: rotary_table(3, 64, inv_freq=torch.ones(31), device="cpu"), lambda: rotary_table(-1, 64, device="cpu")):
        with pytest.raises(ValueError):
            bad()
    t = rotary_table(5, 64, rotary_dim=32, base=100.0, device="cpu")
    assert t.shape == (5, 32) and t.dtype is torch.float32
    at = torch.arange(5, dtype=torch.float64)[:, None] * 100.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    assert torch.allclose(t[:, :16].double(), at.cos(), atol=2.0 ** -24) and torch.allclose(t[:, 16:].double(), at.sin(), atol=2.0 ** -24)
