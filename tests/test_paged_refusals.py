"""Refusals of the paged cache's entry points without a GPU: the C ABI rejects bad arguments
before any launch, and the Python layer refuses CPU tensors and shapes it has no kernel for."""

import ctypes

import pytest
import torch

from maskahead_amd import _native as N
from maskahead_amd.kernels.paged import PagedPrefix, plan_pages, record_bytes
from maskahead_amd.paged import PagedKVCache


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
    return p


def _t4(dtype=N.MA_BF16, ptr=4096):
    m = N.MaTensor4()
    m.ptr, m.dtype = ptr, dtype
    return m


def test_record_bytes():
    assert record_bytes(128) == 5120 and record_bytes(64) == 2560


@pytest.mark.parametrize("kw,d,rc", [
    (dict(), 96, N.MA_EUNSUPPORTED), (dict(dtype=N.MA_F32), 128, N.MA_EUNSUPPORTED), (dict(pool=None), 128, N.MA_EINVAL),
    (dict(lengths=None), 128, N.MA_EINVAL), (dict(page_tokens=48), 128, N.MA_EINVAL), (dict(page_tokens=0), 128, N.MA_EINVAL),
    (dict(num_pages=0), 128, N.MA_EINVAL), (dict(width=0), 128, N.MA_EINVAL), (dict(pool=4104), 128, N.MA_EINVAL),
    (dict(width=1 << 28), 128, N.MA_EUNSUPPORTED)])
def test_a_bad_store_is_refused_by_every_entry(lib, kw, d, rc):
    p = ctypes.byref(_pages(**kw))
    assert lib.ma_page_append(p, _t4(), _t4(), 2, 2, 1, d, 4096, 4096, None) == rc
    assert lib.ma_page_dequant(p, 2, 2, d, None, 1, _t4(), _t4(), None) == rc
    assert lib.ma_paged_attention(_t4(), 2, 4, 1, d, p, 2, _t4(), _t4(), None, 0, 1.0, _t4(), 4096, 1 << 40, None) == rc


def test_bad_calls_are_refused(lib):
    p = ctypes.byref(_pages())
    big = 1 << 40
    E = N.MA_EINVAL
    # append: no tokens, no slots, another dtype
    assert lib.ma_page_append(p, _t4(), _t4(), 2, 2, 0, 128, 4096, 4096, None) == E
    assert lib.ma_page_append(p, _t4(), _t4(), 2, 2, 1, 128, 4096, None, None) == E
    assert lib.ma_page_append(p, _t4(N.MA_F16), _t4(), 2, 2, 1, 128, 4096, 4096, None) == E
    assert lib.ma_page_append(p, _t4(), _t4(), 70000, 2, 1, 128, 4096, 4096, None) == N.MA_EUNSUPPORTED
    # read-back: a negative range, mixed types
    assert lib.ma_page_dequant(p, 2, 2, 128, None, -1, _t4(), _t4(), None) == E
    assert lib.ma_page_dequant(p, 2, 2, 128, None, 1, _t4(), _t4(N.MA_F32), None) == E
    assert lib.ma_page_dequant(p, 2, 2, 128, None, 0, _t4(), _t4(), None) == N.MA_OK
    # attention: heads, dtypes, half a block, workspace
    assert lib.ma_paged_attention(_t4(), 2, 5, 1, 128, p, 2, _t4(), _t4(), None, 0, 1.0, _t4(), 4096, big, None) == E
    assert lib.ma_paged_attention(_t4(), 2, 4, 1, 128, p, 2, _t4(), _t4(ptr=None), None, 0, 1.0, _t4(), 4096, big, None) == E
    assert lib.ma_paged_attention(_t4(N.MA_F16), 2, 4, 1, 128, p, 2, _t4(), _t4(), None, 0, 1.0, _t4(), 4096, big, None) == E
    assert lib.ma_paged_attention(_t4(), 2, 4, 1, 128, p, 2, _t4(), _t4(), None, -1, 1.0, _t4(), 4096, big, None) == E
    need = lib.ma_paged_workspace_bytes(2, 2, 4, 1, 128)
    W = N.MA_EWORKSPACE
    assert need > 0
    assert lib.ma_paged_attention(_t4(), 2, 4, 1, 128, p, 2, _t4(), _t4(), None, 0, 1.0, _t4(), 4096, need - 1, None) == W
    assert lib.ma_paged_attention(_t4(), 2, 4, 1, 128, p, 2, _t4(), _t4(), None, 0, 1.0, _t4(), 4100, need, None) == W
    assert lib.ma_paged_attention(_t4(), 2, 4, 1, 128, p, 2, _t4(), _t4(), None, 0, 1.0, _t4(), None, need, None) == W
    assert lib.ma_paged_workspace_bytes(2, 3, 4, 1, 128) == -1
    assert lib.ma_paged_workspace_bytes(2, 2, 4, 0, 128) == -1
    # plan
    ok = dict(lengths=4096, new=4096, B=2, T=1, page=64, table=4096, s=4, width=4, ring=4096, pages=8, state=4096,
              slots=4096, ends=4096)
    for kw, rc in ((dict(page=33), E), (dict(B=0), E), (dict(T=-1), E), (dict(width=0), E), (dict(pages=0), E),
                   (dict(ring=None), E), (dict(slots=None), E), (dict(width=1 << 26), N.MA_EUNSUPPORTED),
                   (dict(pages=1 << 30), N.MA_EUNSUPPORTED)):
        a = {**ok, **kw}
        assert lib.ma_page_plan(a["lengths"], a["new"], a["B"], a["T"], a["page"], a["table"], a["s"], a["width"], a["ring"],
                                a["pages"], a["state"], a["slots"], a["ends"], None) == rc, kw


def test_cpu_tensors_and_unbuilt_shapes_are_refused():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    with pytest.raises(N.KernelUnavailableError):
        plan_pages(i32(2), i32(2), i32(2, 3), i32(8), i32(4), page_tokens=64, tokens=1)
    tail = torch.zeros((2, 1, 32, 64), dtype=torch.bfloat16)
    pool = torch.zeros((4, 1, 2, 2560), dtype=torch.uint8)
    with pytest.raises(N.KernelUnavailableError):
        PagedPrefix(pool, tail, tail, i32(2, 3), i32(2))
    with pytest.raises(N.KernelUnavailableError):
        PagedPrefix(pool, tail.float(), tail.float(), i32(2, 3), i32(2))
    with pytest.raises(ValueError):
        PagedPrefix(pool, tail[:, :, :31], tail[:, :, :31], i32(2, 3), i32(2))
    with pytest.raises(ValueError):
        PagedPrefix(pool, tail, tail, i32(3, 3), i32(2))
    with pytest.raises(ValueError):
        PagedPrefix(pool[..., 1:], tail, tail, i32(2, 3), i32(2))
    kw = dict(num_layers=1, batch_size=1, num_kv_heads=1, head_dim=64, num_pages=4, max_tokens=64)
    for more, error in ((dict(device="cpu"), N.KernelUnavailableError), (dict(head_dim=96), N.KernelUnavailableError),
                        (dict(compute_dtype=torch.float32), N.KernelUnavailableError), (dict(page_tokens=40), ValueError),
                        (dict(num_pages=0), ValueError)):
        with pytest.raises(error):
            PagedKVCache(**{**kw, **more})


def test_overlapping_plan_arguments_are_refused(lib):
    """What one workgroup writes while another reads it: ends over lengths or new_lens, two
    requests' table rows in one place."""
    ok = dict(lengths=4096, new=8192, s=4, ends=16384)
    call = lambda a: lib.ma_page_plan(a["lengths"], a["new"], 2, 1, 64, 4096, a["s"], 4, 4096, 8, 4096, 4096,  # noqa: E731
                                      a["ends"], None)
    for kw in (dict(ends=4096), dict(ends=4100), dict(ends=4092), dict(ends=8192), dict(ends=8196), dict(s=0), dict(s=3)):
        assert call({**ok, **kw}) == N.MA_EINVAL, kw


def test_a_line_past_31_bits_is_refused(lib):
    """64 requests of up to 2^30 tokens and 2 heads are 2^32 groups of tokens."""
    p = ctypes.byref(_pages(width=1 << 24))
    assert lib.ma_paged_attention(_t4(), 64, 4, 1, 128, p, 2, _t4(), _t4(), None, 0, 1.0, _t4(), 4096, 1 << 40,
                                  None) == N.MA_EUNSUPPORTED
    # rows that no launch holds
    assert lib.ma_paged_workspace_bytes(1, 1, 1 << 16, 1 << 16, 128) == -1


@pytest.mark.parametrize("heads,t,segments", [(4, 1, 1 << 23), (4, 33, 1 << 24), (1, 300, 1 << 24)])
def test_more_segments_than_a_launch_holds_are_refused(lib, heads, t, segments):
    """Before the first launch: 2^32 threads of the merge in one dimension (512 a segment of few rows,
    256 of many; 300 rows are 2 row groups)."""
    b = segments // heads // (2 if t == 300 else 1)
    p = ctypes.byref(_pages(width=1, page_tokens=32))
    assert lib.ma_paged_attention(_t4(), b, heads, t, 128, p, heads, _t4(ptr=None), _t4(ptr=None), None, 0, 1.0, _t4(),
                                  4096, 1 << 60, None) == N.MA_EUNSUPPORTED
    assert b"segments" in lib.ma_last_error()


def test_the_plan_of_an_append_refuses_what_a_plan_does(lib):
    for page, b, ring, rc in ((33, 2, 4096, N.MA_EINVAL), (64, 0, 4096, N.MA_EINVAL), (64, 2, None, N.MA_EINVAL)):
        assert lib.ma_page_plan_append(4096, 8192, b, 1, page, 4096, 4, 4, ring, 8, 4096, 4096, 16384, None) == rc
    assert lib.ma_page_plan_append(4096, 8192, 2, 1, 64, 4096, 4, 4, 4096, 8, 4096, 4096, 4096, None) == N.MA_EINVAL
    assert b"ma_page_plan_append" in lib.ma_last_error()
