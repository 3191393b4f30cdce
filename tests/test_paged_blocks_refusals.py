"""Refusals of the attention over selected blocks without a GPU: bad arguments before any launch."""

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
    (E, dict(blocks=None)), (E, dict(count=0)), (E, dict(count=-1)), (E, dict(per=0)), (E, dict(per=33)), (E, dict(per=-32)),
    (E, dict(run=-1)), (E, dict(hq=5)), (E, dict(t=0)), (E, dict(causal=-1)), (E, dict(kc=_t4(ptr=None))),
    (E, dict(out=_t4(N.MA_F16))), (U, dict(d=96)), (E, dict(p=dict(pool=None))), (E, dict(q=_t4(ptr=None))),
    # (a head's rows, segments and items that the kernels do not count)
    (E, dict(t=1 << 28)), (U, dict(b=1 << 13, h=32, hq=32, t=64, run=1)), (E, dict(b=1 << 20, h=32, hq=32, t=64, run=1)),
    (N.MA_EWORKSPACE, dict(ws=None)), (N.MA_EWORKSPACE, dict(ws=4100)), (N.MA_EWORKSPACE, dict(bytes=256))])
def test_bad_lists_are_refused(lib, rc, change):
    a = dict(q=_t4(), b=2, hq=4, t=2, d=64, p={}, h=2, kc=_t4(), vc=_t4(), causal=0, out=_t4(), blocks=4096, count=4, per=64,
             run=0, ws=4096, bytes=1 << 50)
    a.update(change)
    assert lib.ma_paged_attention_blocks(a["q"], a["b"], a["hq"], a["t"], a["d"], _pages(**a["p"]), a["h"], a["kc"], a["vc"],
                                         None, a["causal"], 1.0, a["out"], a["blocks"], a["count"], a["per"], a["run"],
                                         a["ws"], a["bytes"], None) == rc


def test_workspace_sizes(lib):
    runs = lib.ma_paged_blocks_workspace_bytes
    for t in (1, 5, 40):
        assert runs(2, 4, 28, t, 128, 64, 32, 0) == runs(2, 4, 28, t, 128, 64, 32, t) == runs(2, 4, 28, t, 128, 64, 32, 99) > 0
    assert runs(2, 4, 28, 512, 128, 8, 32, 1) == 0             # a workgroup a segment: nothing to join
    for bad in ((2, 4, 28, 512, 128, 8, 32, -1), (2, 4, 28, 512, 128, 0, 32, 1), (2, 4, 28, 512, 128, 8, 33, 1),
                (2, 4, 28, 512, 128, 8, 0, 1), (1 << 16, 1 << 10, 1 << 10, 64, 128, 8, 32, 1), (2, 3, 4, 1, 64, 8, 32, 0)):
        assert runs(*bad) == -1
