"""Sizes that the kernels over selected blocks do not count in 32 bits, refused without a GPU."""

import ctypes

import pytest

from maskahead_amd import _native as N


@pytest.fixture(scope="module")
def lib():
    if not N.LIB_PATH.exists():
        from maskahead_amd.build import build

        build()
    return N.load()


def _pages():
    p = N.MaPages()
    p.pool = p.k_tail = p.v_tail = p.table = p.lengths = 4096
    p.num_pages, p.width, p.page_tokens, p.dtype = 8, 4, 64, N.MA_BF16
    p.s_pool[0], p.s_pool[1] = 2 * 10240, 10240
    return ctypes.byref(p)


def _t4():
    m = N.MaTensor4()
    m.ptr, m.dtype = 4096, N.MA_BF16
    return m


@pytest.mark.parametrize("t,run", [(2 ** 31 - 1, 1024), (2 ** 31 - 1, 256), (2 ** 31 - 1, 1 << 26), (2 ** 31 - 1024, 1025),
                                   (2 ** 31 - 20, 1 << 10)])
def test_positions_whose_runs_end_past_32_bits(lib, t, run):
    assert lib.ma_paged_blocks_workspace_bytes(1, 1, 1, t, 64, 8, 32, run) == -1
    assert lib.ma_paged_attention_blocks(_t4(), 1, 1, t, 64, _pages(), 1, _t4(), _t4(), None, 0, 1.0, _t4(), 4096, 8, 32, run,
                                         4096, 1 << 50, None) == N.MA_EINVAL
    assert lib.ma_select_blocks(_t4(), 1, 1, t, 64, _pages(), 1, None, run, 32, 4, 0, 0, 4096, None, 4096, 1 << 50,
                                None) == N.MA_EUNSUPPORTED


def test_the_last_size_has_a_workspace(lib):
    assert lib.ma_paged_blocks_workspace_bytes(1, 1, 1, 2 ** 31 - 1 - 1024, 64, 8, 32, 1024) >= 0
