"""Refusals of the block selection's entry point without a GPU: bad arguments before any launch."""

import ctypes

import pytest

from maskahead_amd import _native as N

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


@pytest.mark.parametrize("rc,change", [
    (E, dict(hq=5)), (E, dict(hq=0)), (E, dict(t=0)), (E, dict(run=-1)), (E, dict(per=0)), (E, dict(per=48)),
    (E, dict(per=-32)), (E, dict(count=0)), (E, dict(first=-1)), (E, dict(last=-1)), (E, dict(first=3, last=2)),
    (E, dict(first=2147483647, last=2147483647)), (E, dict(q=_t4(ptr=None))), (E, dict(blocks=None)),
    (E, dict(q=_t4(N.MA_F16))), (U, dict(d=96)), (E, dict(p=dict(pool=4104))), (E, dict(p=dict(table=None))),
    (E, dict(b=0)), (U, dict(p=dict(dtype=N.MA_F32))), (U, dict(b=1 << 20, t=4096, run=1)), (U, dict(b=1 << 12, t=512, run=1)), (U, dict(t=1 << 28)),
    (N.MA_EWORKSPACE, dict(ws=None)), (N.MA_EWORKSPACE, dict(ws=4100)), (N.MA_EWORKSPACE, dict(bytes=255))])
def test_bad_selections_are_refused(lib, rc, change):
    a = dict(q=_t4(), b=2, hq=4, t=2, d=64, p={}, h=2, run=0, per=64, count=4, first=1, last=1, blocks=4096, ws=4096,
             bytes=1 << 40)
    a.update(change)
    assert lib.ma_select_blocks(a["q"], a["b"], a["hq"], a["t"], a["d"], _pages(**a["p"]), a["h"], None, a["run"], a["per"],
                                a["count"], a["first"], a["last"], a["blocks"], None, a["ws"], a["bytes"], None) == rc


def test_workspace_sizes(lib):
    size = lib.ma_select_workspace_bytes
    assert size(2, 3, 4, 640) == -(-2 * 3 * 4 * 20 * 4 // 256) * 256
    for bad in ((0, 1, 1, 32), (1, 0, 1, 32), (1, 1, 0, 32), (1, 1, 1, 0), (1 << 16, 1 << 15, 1, 32), (1, 1, 1, 1 << 31)):
        assert size(*bad) == -1
