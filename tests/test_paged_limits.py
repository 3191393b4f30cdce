"""Refusals without a GPU: sizes that the kernels over selected blocks do not count in 32 bits, and outputs of
rotated rows that share memory."""

import ctypes
import itertools
from types import SimpleNamespace

import pytest
import torch

from maskahead_amd import _native as N
from maskahead_amd.kernels import paged as P


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


def _view(shape, strides, room=1 << 16):
    return torch.as_strided(torch.zeros(room, dtype=torch.bfloat16), shape, strides)


@pytest.mark.parametrize("shape,strides,shared", [
    ((2, 3, 4, 64), (768, 256, 64, 1), False), ((2, 3, 4, 64), (64, 512, 128, 1), False),      # contiguous; [H, T, B, D] rows
    ((2, 3, 4, 64), (768, 64, 192, 1), False), ((1, 3, 1, 64), (5, 64, 3, 1), False),         # [B, T, H, D]; strides of one
    ((1, 2, 3, 64), (0, 192, 128, 1), False),        # rows of one head between those of the other
    ((2, 3, 4, 64), (768, 256, 32, 1), True), ((2, 3, 4, 64), (768, 256, 63, 1), True),        # each row into the next
    ((2, 3, 4, 64), (256, 256, 64, 1), True), ((2, 3, 4, 64), (0, 256, 64, 1), True),
    ((1, 2, 3, 64), (0, 128, 128, 1), True), ((1, 2, 3, 64), (0, 256, 128, 1), True),         # two ways to one place
    ((1, 2, 3, 64), (0, 160, 128, 1), True)])        # half a row of one head over the other's
def test_outputs_whose_rows_share_memory(shape, strides, shared):
    """Every row is written, by threads in no order: rows in one place would hold either."""
    prefix = SimpleNamespace(batch=shape[0], head_dim=64, index=-1, dtype=torch.bfloat16, device="cpu")
    rows, out = torch.zeros(shape, dtype=torch.bfloat16), _view(shape, strides)
    starts = sorted(sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, shape[:3])))
    assert shared == any(y - x < 64 for x, y in zip(starts, starts[1:]))
    if shared:
        with pytest.raises(ValueError, match="share their memory"):
            P._check_rows("query", rows, prefix, out)
    else:
        assert P._check_rows("query", rows, prefix, out) is out


@pytest.mark.parametrize("kw,rc", [
    (dict(b=1 << 13, h=32, t=64, run=1), N.MA_EUNSUPPORTED), (dict(b=1 << 18, h=32, t=1, run=0), N.MA_EUNSUPPORTED),
    (dict(b=1 << 25, h=32, t=2, run=1), N.MA_EINVAL), (dict(b=1 << 26, h=32, t=1, run=0), N.MA_EINVAL),
    (dict(b=1, h=1, t=1 << 27, run=0), N.MA_EINVAL)])
def test_segments_that_are_not_built(lib, kw, rc):
    """2^23 segments or more are unsupported; what has no workspace is an invalid argument."""
    b, h, t, run = kw["b"], kw["h"], kw["t"], kw["run"]
    need = lib.ma_paged_blocks_workspace_bytes(b, h, h, t, 64, 8, 32, run)
    assert (need == -1) == (rc == N.MA_EINVAL)
    assert lib.ma_paged_attention_blocks(_t4(), b, h, t, 64, _pages(), h, _t4(), _t4(), None, 0, 1.0, _t4(), 4096, 8, 32, run,
                                         4096, 1 << 50, None) == rc
