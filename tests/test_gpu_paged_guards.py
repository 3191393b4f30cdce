"""What PagedKVCache refuses or reports of the calls between a layer's staging and the commit."""

import pytest
import torch

from maskahead_amd._native import KernelUnavailableError
from maskahead_amd.kernels.paged import append_pages, rotary_table, rotate_block

from _paged import Requests

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def test_a_staged_descriptor_needs_a_staged_layer(gpu):
    """Outside of an append it would describe the lengths of the last one, whose pages may be another's by now."""
    r = Requests(gpu, [40, 64], h=1, d=64, page=32, layers=2)
    c = r.cache

    def refused(layer):
        with pytest.raises(RuntimeError, match="not staged"):
            c.prefix(layer, staged=True)

    refused(0)
    k, v = (x.to(gpu) for x in r.block([1, 0], 1))
    c.begin_append(r.i32([1, 0]), 1)
    refused(0)
    c.stage_layer(0, k, v)
    assert c.prefix(0, staged=True).lengths.tolist() == [41, 64]
    refused(1)
    c.stage_layer(1, k, v)
    c.commit_append()
    refused(0)
    c.release(torch.tensor([True, False], device=gpu))
    refused(1)
    for layer in (-1, 2):
        with pytest.raises(IndexError):
            c.prefix(layer, staged=True)
    assert c.prefix(0).lengths.tolist() == [0, 64]


@pytest.mark.parametrize("t,new,rows,behind", [(3, [3, 0], 42, True), (3, [3, 0], 43, False), (3, [2, 0], 42, False),
                                               (1, [1, 0], 40, True), (70, [70, 3], 110, False), (70, [70, 3], 109, True),
                                               (70, [2, 60], 64, True)])
@pytest.mark.parametrize("way", ["staged", "rotated"])
def test_positions_behind_the_table_are_reported(gpu, t, new, rows, behind, way):
    """A new token whose position the rotary table does not hold takes its last row: check() says so."""
    lens = [40, 100 if new[1] == 0 else 5]       # (an idle request may lie behind the table)
    r = Requests(gpu, lens, h=2, d=64, page=32, room=128)
    c = r.cache
    table = rotary_table(rows, 64, device=gpu)
    k, v = (torch.nan_to_num(x).to(gpu) for x in r.block(new, t))
    q = torch.zeros((2, 4, t, 64), dtype=BF, device=gpu)
    first = c.lengths.clone()
    c.rotate(q, k, rotary=table)                 # (no append in progress: whose rows count is not known)
    c.check()
    c.begin_append(r.i32(new), t)
    c.rotate(q, k, rotary=table, positions=first)        # (the caller's own positions are the caller's)
    c.check()
    if way == "rotated":
        _, k = c.rotate(q, k, rotary=table)
        c.stage_layer(0, k, v)
    else:
        c.stage_layer(0, k, v, rotary=table, query=q)
    c.commit_append()
    if behind:
        with pytest.raises(RuntimeError, match="rotary table"):
            c.check()
    c.check()                                    # (reported once)


def test_a_captured_step_reports_too(gpu):
    r = Requests(gpu, [30], h=1, d=64, page=32, room=32)
    c = r.cache
    table = rotary_table(33, 64, device=gpu)
    k, v = (x.to(gpu) for x in r.block([1], 1))
    q = torch.zeros((1, 2, 1, 64), dtype=BF, device=gpu)
    news = r.i32([1])

    def step():
        c.begin_append(news, 1)
        c.stage_layer(0, k, v, rotary=table, query=q)
        c.commit_append()

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):                           # positions 31, 32, 33, 34 of a table of 33
        graph.replay()
        torch.cuda.synchronize()
        if i < 2:
            c.check()
        else:
            with pytest.raises(RuntimeError, match="rotary table"):
                c.check()
    assert c.lengths.tolist() == [35]


def test_a_plan_and_a_position_are_both_named(gpu):
    r = Requests(gpu, [40], h=1, d=64, page=32, room=30)
    c = r.cache
    table = rotary_table(41, 64, device=gpu)
    k, v = (x.to(gpu) for x in r.block([2], 2))
    c.begin_append(r.i32([2]), 2)
    c.stage_layer(0, k, v, rotary=table)
    c.commit_append()
    c.begin_append(r.i32([200]), 2)
    c.stage_layer(0, k, v)
    c.commit_append()
    with pytest.raises(RuntimeError, match="page plan refused.*more new tokens.*rotary table"):
        c.check()
    c.check()


def test_a_status_of_the_callers_own(gpu):
    """rotate_block and append_pages with a ring_state: positions of the caller's, below the table too."""
    r = Requests(gpu, [40, 3], h=2, d=128, page=32, room=32)
    p, table = r.cache.prefixes[0], rotary_table(20, 128, device=gpu)
    q = torch.zeros((2, 4, 3, 128), dtype=BF, device=gpu)
    k = torch.zeros((2, 2, 3, 128), dtype=BF, device=gpu)
    slots = torch.tensor([[0, 1, 2], [-1, -1, -1]], device=gpu)      # (request 1 stores nothing)
    state = r.i32([0, 0, 0, 0])

    def status(call, *first, new=(3, 3)):
        state.fill_(5)
        call(r.i32(list(first)), r.i32(list(new)))
        assert state[:3].tolist() == [5] * 3
        return int(state[3])

    def turn(first, new):
        rotate_block(p, q, k, rotary=table, positions=first, new_lens=new, ring_state=state)

    def keys_alone(first, new):
        rotate_block(p, q[:, :0], k, rotary=table, positions=first, new_lens=new, ring_state=state)

    def all_rows(first, new):
        rotate_block(p, q, rotary=table, positions=first, ring_state=state)

    def append(first, new):
        append_pages(p, k, k, new, slots, rotary=table, positions=first, query=q, ring_state=state)

    for call in (turn, keys_alone, all_rows, append):
        assert status(call, 17, 0) == 5
        for first in (18, -1, 20, 2 ** 31 - 1, -2 ** 31):
            assert status(call, first, 0) == 37
            assert status(call, 0, first) == (5 if call is append else 37)
        assert status(call, 18, 0, new=(2, 0)) == (37 if call is all_rows else 5)
        assert status(call, 99, 0, new=(0, 3)) == (37 if call is all_rows else 5)
        assert status(call, 99, 0, new=(-1, 3)) == (37 if call is all_rows else 5)
        assert status(call, 17, 0, new=(90, 0)) == 5
    for bad in (state.long(), state[:3], state.cpu()):
        with pytest.raises((ValueError, KernelUnavailableError)):
            rotate_block(p, q, rotary=table, ring_state=bad)
    with pytest.raises(ValueError):
        rotate_block(p, q, rotary=table, ring_state=state, new_lens=r.i32([1]))
    with pytest.raises(ValueError):
        append_pages(p, k, k, r.i32([1, 1]), slots, ring_state=state)
