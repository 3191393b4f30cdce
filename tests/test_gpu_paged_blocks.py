"""Attention over selected blocks: against 64 bits within the bound of its roundings, bit for bit
against itself, and a run of rotation, selection, attention and append together."""

import pytest
import torch

from maskahead_amd.kernels.paged import paged_attention, rotary_table, select_blocks
from maskahead_amd.paged import PagedKVCache

from _paged import Requests, attend64, check_attention, group_scores, rotated, select_rule

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


def _lists(gen, lens, h, runs, count, per, holes=False):
    """Random lists in ascending order, -1 behind them (holes: anywhere, and entries behind the last block)."""
    out = torch.full((len(lens), h, runs, count), -1, dtype=torch.int32)
    for b, x in enumerate(lens):
        nb = -(-(x // 32) // (per // 32))
        for kv in range(h):
            for r in range(runs):
                pick = torch.randperm(nb, generator=gen)[:count]
                if holes and len(pick) > 2:
                    pick[torch.randint(len(pick), (), generator=gen)] = -1
                    pick[torch.randint(len(pick), (), generator=gen)] = [nb, 2 ** 31 - 1, -2 ** 31, nb + 5][r % 4]
                    pick = pick[torch.randperm(len(pick), generator=gen)]
                else:
                    pick = pick.sort().values
                out[b, kv, r, :len(pick)] = pick.to(torch.int32)
    return out


def _check(r, q, ck, cv, out, lists, new, *, per, run, causal, mask=None, before=None):
    t, h, dtype = q.shape[2], r.h, r.dtype
    g = q.shape[1] // h
    run = run or t
    for b, n in enumerate(new):
        if before is not None:
            assert torch.equal(out[b, :, n:].cpu(), before[b, :, n:])
        if n == 0:
            continue
        k, v = r.kv64(b)
        x = k.shape[1]
        for i in range(-(-n // run)):
            lo, hi = i * run, min(n, (i + 1) * run)
            seen = torch.zeros((h, x), dtype=torch.bool)
            seen[:, x // 32 * 32:] = True
            nb = -(-(x // 32) // (per // 32))
            for kv in range(h):
                for e in lists[b, kv, i].tolist()[:nb]:
                    if 0 <= e < nb:
                        seen[kv, e * per:min((e + 1) * per, x // 32 * 32)] = True
            if mask is not None:
                live = torch.nn.functional.pad(mask[b], (0, max(0, x - mask.shape[2])))[:, :x] != 0
                seen &= live
            rows, keys = ck[b, :, :0], cv[b, :, :0]
            if ck.shape[2]:
                rows, keys = ck[b, :, :n], cv[b, :, :n]
            # (attend64's rows are the positions behind its length: those of this run alone are looked at)
            qq = q[b, :, :n] if rows.shape[1] else q[b, :, lo:hi]
            want, bound = attend64(qq, k, v, rows, keys, seen=seen, causal=causal)
            if rows.shape[1]:
                want, bound = want[:, lo:hi], bound[:, lo:hi]
            check_attention(out[b, :, lo:hi], want, bound, dtype)


@pytest.mark.parametrize("d,h,g,dtype,page,t,run,causal", [
    (128, 2, 7, BF, 64, 1, 0, 0), (64, 1, 4, F16, 32, 3, 0, 0), (128, 1, 1, F16, 96, 5, 1, 1), (64, 2, 8, BF, 128, 9, 4, 0),
    (128, 1, 7, BF, 64, 32, 0, 0), (128, 2, 4, BF, 32, 40, 32, 32), (64, 1, 4, F16, 64, 70, 33, 7), (64, 1, 20, BF, 64, 5, 2, 0),
    (128, 1, 7, F16, 64, 66, 32, 0), (128, 1, 16, BF, 64, 30, 0, 4)])
@pytest.mark.parametrize("count,per,dead", [(3, 32, False), (4, 96, True), (40, 64, False)])
def test_attention_over_blocks(gpu, d, h, g, dtype, page, t, run, causal, count, per, dead):
    lens = [0, 31, 32, 700, 1500, 1024, 97]
    new = [t, t, t, t, max(1, t - 1), 0, -(-t // 2)]
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=page)
    q = torch.randn((7, h * g, t, d), generator=r.gen).to(dtype)
    ck, cv = r.block(new, t)
    runs = -(-t // (run or t))
    lists = _lists(r.gen, lens, h, runs, count, per, holes=dead)
    mask = (torch.rand((7, h, 1400), generator=r.gen) < 0.6).to(torch.uint8) if dead else None
    prefix = r.cache.prefix(0, mask=mask.to(gpu) if dead else None)
    before = torch.randn((7, h * g, t, d), generator=r.gen).to(dtype)
    kw = dict(new_lens=r.i32(new), causal_block=causal, blocks=lists.to(gpu), block_tokens=per, query_block=run)
    out = paged_attention(q.to(gpu), prefix, ck.to(gpu), cv.to(gpu), out=before.to(gpu), **kw)
    _check(r, q, ck, cv, out, lists, new, per=per, run=run, causal=causal, mask=mask, before=before)
    again = paged_attention(q.to(gpu), prefix, ck.to(gpu), cv.to(gpu), out=before.to(gpu), **kw)
    assert torch.equal(out, again)
    # the stored tokens alone
    del kw["causal_block"]
    out = paged_attention(q.to(gpu), prefix, out=before.to(gpu), **kw)
    _check(r, q, ck[:, :, :0], cv[:, :, :0], out, lists, new, per=per, run=run, causal=0, mask=mask, before=before)


def test_all_blocks_are_the_whole_cache(gpu):
    """Lists of everything give the values of attention without lists."""
    r = Requests(gpu, [960, 333, 64], h=2, d=128)
    q = torch.randn((3, 8, 2, 128), generator=r.gen).to(BF).to(gpu)
    k, v = (x.to(gpu) for x in r.block([2, 2, 2], 2))
    full = paged_attention(q, r.cache.prefixes[0], k, v)
    lists = torch.arange(30, dtype=torch.int32, device=gpu).expand(3, 2, 1, 30).contiguous()
    got = paged_attention(q, r.cache.prefixes[0], k, v, blocks=lists)
    # (two results of the same softmax, summed in another order, each rounded once: at most a step apart)
    assert ((got.double() - full.double()).abs() <= 2 * torch.finfo(BF).eps * full.double().abs() + 2.0 ** -9).all()
    flip = paged_attention(q, r.cache.prefixes[0], k, v, blocks=lists.flip(-1).contiguous())
    short = flip[0].double() - full[0].double()
    assert (short.abs() <= 2 * torch.finfo(BF).eps * full[0].double().abs() + 2.0 ** -9).all()


def test_no_blocks_is_the_tail_and_the_block(gpu):
    lens, new = [40, 64, 7], [2, 2, 1]
    r = Requests(gpu, lens)
    q = torch.randn((3, 4, 2, 128), generator=r.gen).to(BF)
    ck, cv = r.block(new, 2)
    for lists in (torch.full((3, 2, 1, 5), -1, dtype=torch.int32), torch.empty((3, 2, 1, 0), dtype=torch.int32)):
        out = paged_attention(q.to(gpu), r.cache.prefixes[0], ck.to(gpu), cv.to(gpu), new_lens=r.i32(new), blocks=lists.to(gpu))
        _check(r, q, ck, cv, out, lists, new, per=32, run=0, causal=0)
        # a request of whole groups without a block of its own: nothing to see
        out = paged_attention(q.to(gpu), r.cache.prefixes[0], new_lens=r.i32(new), blocks=lists.to(gpu))
        assert (out[1] == 0).all()


def test_a_block_listed_twice_weighs_twice(gpu):
    r = Requests(gpu, [96], h=1)
    q = torch.randn((1, 1, 1, 128), generator=r.gen).to(BF)
    lists = torch.tensor([[[[1, 0, 1]]]], dtype=torch.int32)
    out = paged_attention(q.to(gpu), r.cache.prefixes[0], blocks=lists.to(gpu))
    k, v = r.kv64(0)
    twice = lambda x: torch.cat((x[:, :64], x[:, 32:64]), 1)  # noqa: E731
    none = torch.empty((1, 0, 128), dtype=BF)
    want, bound = attend64(q[0], twice(k), twice(v), none, none, seen=torch.ones((1, 96), dtype=torch.bool))
    check_attention(out[0], want, bound, BF)


def test_pages_of_no_pool_and_long_lists(gpu):
    r = Requests(gpu, [3000, 200], h=1, d=64, page=32)
    r.cache.block_table[0, 5], r.cache.block_table[0, 6] = -1, 12345
    q = torch.randn((2, 3, 1, 64), generator=r.gen).to(BF)
    lists = torch.arange(300, dtype=torch.int32).expand(2, 1, 1, 300).contiguous()      # (more than there are)
    mask = torch.ones((2, 1, 3000), dtype=torch.uint8)
    mask[0, :, 160:224] = 0
    out = paged_attention(q.to(gpu), r.cache.prefixes[0], blocks=lists.to(gpu))
    _check(r, q, *r.block([0, 0], 0), out, lists, [1, 1], per=32, run=0, causal=0, mask=mask)


def test_many_requests(gpu):
    """More than 64 requests: the line is found by the whole workgroup."""
    lens = [(61 * i) % 500 for i in range(130)]
    new = [i % 3 for i in range(130)]
    r = Requests(gpu, lens, h=1, d=64, page=32)
    q = torch.randn((130, 4, 2, 64), generator=r.gen).to(BF)
    ck, cv = r.block(new, 2)
    lists = _lists(r.gen, lens, 1, 2, 4, 64)
    out = paged_attention(q.to(gpu), r.cache.prefixes[0], ck.to(gpu), cv.to(gpu), new_lens=r.i32(new), blocks=lists.to(gpu),
                          block_tokens=64, query_block=1)
    _check(r, q, ck, cv, out, lists, new, per=64, run=1, causal=0)
    # and many rows of each
    q = torch.randn((130, 24, 2, 64), generator=r.gen).to(BF)
    lists = _lists(r.gen, lens, 1, 1, 4, 64)
    out = paged_attention(q.to(gpu), r.cache.prefixes[0], ck.to(gpu), cv.to(gpu), new_lens=r.i32(new), blocks=lists.to(gpu),
                          block_tokens=64)
    _check(r, q, ck, cv, out, lists, new, per=64, run=0, causal=0)


@pytest.mark.parametrize("t,run,dtype,d", [(1, 0, BF, 128), (33, 32, BF, 128), (5, 0, F16, 64)])
def test_positions_selection_attention_and_append_together(gpu, t, run, dtype, d):
    """Steps of a batch as a program runs them, captured and replayed: rotate, select, attend, stage."""
    lens, hq, h, count = [300, 30, 1000, 64], 8, 2, 5
    new = [t, t, 0, max(1, t - 2)]
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=32, room=6 * t + 32)
    c = r.cache
    table = rotary_table(1300, d, device=gpu)
    cpu = table.cpu()
    news = r.i32(new)
    k, v = (torch.zeros((4, h, t, d), dtype=dtype, device=gpu) for _ in range(2))
    q = torch.zeros((4, hq, t, d), dtype=dtype, device=gpu)
    out = torch.zeros_like(q)
    kw = dict(block_tokens=64, query_block=run)

    def step():
        c.begin_append(news, t)
        rq, rk = c.rotate(q, k, rotary=table)
        blocks = c.select(0, rq, count, keep_first=1, keep_last=1, **kw)
        c.attend(0, rq, rk, v, blocks=blocks, causal_block=32, out=out, **kw)
        c.stage_layer(0, k, v, rotary=table)
        c.commit_append()
        return blocks

    graph = blocks = None
    for i in range(5):
        hk, hv = r.block(new, t)
        hk, hv = torch.nan_to_num(hk), torch.nan_to_num(hv)
        h_q = torch.randn((4, hq, t, d), generator=r.gen).to(dtype)
        k.copy_(hk), v.copy_(hv), q.copy_(h_q)
        at = c.lengths.tolist()
        state = (c.pool, c.k_tail, c.v_tail, c.block_table, c.lengths, c.free_ring, c.ring_state)
        if i == 1:
            saved = [x.clone() for x in state]
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                blocks = step()
            for x, y in zip(state, saved):
                x.copy_(y)
        pool, rows = c.pool[0].cpu(), c.block_table.tolist()
        if graph:
            graph.replay()
        else:
            blocks = step()
        torch.cuda.synchronize()
        rq, rk = rotated(h_q, cpu, at, False), rotated(hk, cpu, at, False)
        got = blocks.cpu()
        for b, n in enumerate(new):
            for kv in range(h):
                for u in range(got.shape[2]):
                    part = rq[b, kv * 4:kv * 4 + 4, u * (run or t):min((u + 1) * (run or t), n)].flatten(0, 1)
                    s = group_scores(pool, rows[b], at[b] // 32, kv, part) if len(part) else []
                    took, _ = select_rule(s, 2, count, 1, 1)
                    assert got[b, kv, u].tolist() == took + [-1] * (count - len(took))
        _check(r, rq, rk, hv, out, got, new, per=64, run=run, causal=32)
        r.note(new, rk, hv)
        assert c.lengths.tolist() == [x + n for x, n in zip(at, new)]
    c.check()
    for b in range(4):
        kk, vv = c.dequantize_layer(0, 1200, dtype=torch.float32)
        k64, v64 = r.kv64(b)
        n = k64.shape[1]
        assert torch.equal(kk[b, :, :n].cpu().double(), k64) and torch.equal(vv[b, :, :n].cpu().double(), v64)


def test_select_and_attend_a_staged_layer(gpu):
    lens, new = [40, 95], [1, 1]
    r = Requests(gpu, lens, h=1, d=64, page=32)
    c = r.cache
    table = rotary_table(128, 64, device=gpu)
    k, v = r.block(new, 1)
    q = torch.randn((2, 4, 1, 64), generator=r.gen).to(BF)
    c.begin_append(r.i32(new), 1)
    with pytest.raises(RuntimeError):
        c.select(0, q.to(gpu), 2, staged=True)
    rq = c.stage_layer(0, k.to(gpu), v.to(gpu), rotary=table, query=q.to(gpu))
    with pytest.raises(RuntimeError):
        c.select(0, rq, 2)
    lists = c.select(0, rq, 2, staged=True)
    out = c.attend(0, rq, staged=True, blocks=lists)
    c.commit_append()
    r.note(new, rotated(k, table.cpu(), lens, False), v)
    rq, lists = rotated(q, table.cpu(), lens, False), lists.cpu()
    assert lists[0, 0, 0].tolist() == [0, -1] and -1 not in lists[1, 0, 0].tolist()
    _check(r, rq, *r.block([0, 0], 0), out, lists, new, per=32, run=0, causal=0)


def test_another_stream_and_two_at_once(gpu):
    r = Requests(gpu, [700, 96], h=2, d=64)
    q = torch.randn((2, 4, 1, 64), generator=r.gen).to(BF).to(gpu)
    lists = [_lists(r.gen, [700, 96], 2, 1, 4, 32) for _ in range(2)]
    dev = [x.to(gpu) for x in lists]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for s, x in zip(streams, dev):
        with torch.cuda.stream(s):
            outs.append(paged_attention(q, r.cache.prefixes[0], blocks=x))
    torch.cuda.synchronize()
    for x, out in zip(lists, outs):
        _check(r, q.cpu(), *r.block([0, 0], 0), out, x, [1, 1], per=32, run=0, causal=0)


def test_refused_lists(gpu):
    r = Requests(gpu, [100, 10], h=2)
    p, q = r.cache.prefixes[0], torch.zeros((2, 4, 3, 128), dtype=BF, device=gpu)
    ok = torch.zeros((2, 2, 1, 4), dtype=torch.int32, device=gpu)
    for kw in (dict(blocks=ok.long()), dict(blocks=ok[0]), dict(blocks=ok[:, :1]), dict(blocks=ok, query_block=1),
               dict(blocks=ok, block_tokens=33), dict(blocks=ok, block_tokens=0), dict(blocks=ok, query_block=-1),
               dict(blocks=ok.expand(2, 2, 1, 4)[..., ::2]), dict(query_block=2)):
        with pytest.raises(ValueError):
            paged_attention(q, p, **kw)
    from maskahead_amd._native import KernelUnavailableError
    with pytest.raises((ValueError, KernelUnavailableError)):
        paged_attention(q, p, blocks=ok.cpu())
    # lists of a call without positions
    assert paged_attention(q[:, :, :0], p, blocks=ok[:, :, :0]).shape == (2, 4, 0, 128)
    blocks = select_blocks(q, p, 4)
    assert paged_attention(q, p, blocks=blocks).shape == q.shape


@pytest.mark.parametrize("per", [2048, 2 ** 31 - 32])
def test_blocks_longer_than_requests(gpu, per):
    lens = [0, 40, 1000, 320]
    r = Requests(gpu, lens, h=1, d=64, page=32)
    q = torch.randn((4, 2, 1, 64), generator=r.gen).to(BF)
    lists, scores = select_blocks(q.to(gpu), r.cache.prefixes[0], 3, block_tokens=per, return_scores=True)
    assert lists[:, 0, 0].tolist() == [[-1] * 3] + [[0, -1, -1]] * 3 and scores.shape[3] == 1
    for b, x in enumerate(lens[1:], 1):
        s = group_scores(r.cache.pool[0].cpu(), r.cache.block_table[b].tolist(), x // 32, 0, q[b, :, 0])
        assert scores[b, 0, 0, 0] == torch.tensor(max(s), dtype=torch.float64).float()
    out = paged_attention(q.to(gpu), r.cache.prefixes[0], blocks=lists, block_tokens=per)
    assert torch.equal(out, paged_attention(q.to(gpu), r.cache.prefixes[0], blocks=lists[..., :1].contiguous(), block_tokens=per))
    full = paged_attention(q.to(gpu), r.cache.prefixes[0])
    assert ((out.double() - full.double()).abs() <= 2 * torch.finfo(BF).eps * full.double().abs() + 2.0 ** -9).all()


@pytest.mark.parametrize("d,h,g,t,dtype,causal", [(128, 2, 7, 1, BF, 0), (64, 2, 7, 3, F16, 1), (64, 4, 4, 8, BF, 2), (128, 4, 3, 6, F16, 0)])
@pytest.mark.parametrize("count,dead", [(3, False), (14, True)])
def test_a_workgroup_for_each_request(gpu, d, h, g, t, dtype, causal, count, dead):
    """About as many heads of requests as the card has CUs: the widest workgroups, and nothing to join."""
    b = 200 // h
    lens = [(97 * i) % 640 for i in range(b)]
    new = [(i * 5) % (t + 1) for i in range(b)]
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=32, room=0)
    q = torch.randn((b, h * g, t, d), generator=r.gen).to(dtype)
    ck, cv = r.block(new, t)
    if causal:
        for i, n in enumerate(new):
            if n > 1:
                cv[i, :, n - 1, 5::9] = float("inf") if i % 2 else float("nan")     # (the last position's alone see it)
    lists = _lists(r.gen, lens, h, 1, count, 32, holes=dead)
    mask = (torch.rand((b, h, 600), generator=r.gen) < 0.6).to(torch.uint8) if dead else None
    before = torch.randn((b, h * g, t, d), generator=r.gen).to(dtype)
    out = paged_attention(q.to(gpu), r.cache.prefix(0, mask=mask.to(gpu) if dead else None), ck.to(gpu), cv.to(gpu),
                          out=before.to(gpu), new_lens=r.i32(new), causal_block=causal, blocks=lists.to(gpu))
    if causal:
        for i, n in enumerate(new):
            # rows that see the last key: those of its causal block
            if n > 1:
                last = (lens[i] + n - 1) // causal
                rows = [x for x in range(n) if (lens[i] + x) // causal >= last]
                assert not torch.isfinite(out[i, :, rows][..., 5::9]).any()
                keep = torch.ones(d, dtype=torch.bool)
                keep[5::9] = False
                assert torch.isfinite(out[i, :, :n][..., keep.to(gpu)]).all()
                early = [x for x in range(n) if x not in rows]
                assert torch.isfinite(out[i, :, early]).all()
                cv[i, :, n - 1, 5::9] = 0.0
                out[i, :, rows] = torch.where(keep.to(gpu), out[i, :, rows], 0.0)
        again = paged_attention(q.to(gpu), r.cache.prefix(0, mask=mask.to(gpu) if dead else None), ck.to(gpu), cv.to(gpu),
                                out=before.to(gpu), new_lens=r.i32(new), causal_block=causal, blocks=lists.to(gpu))
        for i, n in enumerate(new):
            last = (lens[i] + n - 1) // causal
            for x in range(n):
                if n == 1 or (lens[i] + x) // causal < last:
                    assert torch.equal(again[i, :, x], out[i, :, x])
        out = again
    _check(r, q, ck, cv, out, lists, new, per=32, run=0, causal=causal, mask=mask, before=before)


@pytest.mark.parametrize("d,g,t,run,causal,dtype", [(128, 1, 9, 4, 3, BF), (64, 4, 7, 0, 2, F16), (128, 7, 70, 32, 32, BF),
                                                    (64, 7, 70, 33, 16, F16), (128, 7, 40, 0, 8, BF)])
def test_what_is_not_seen_may_hold_anything(gpu, d, g, t, run, causal, dtype):
    """Blocks that no list names and the block's keys behind a row's causal block: no number there changes a bit."""
    lens, h = [700, 96, 33], 2
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=32)
    q = torch.randn((3, h * g, t, d), generator=r.gen).to(dtype).to(gpu)
    ck, cv = (x.to(gpu) for x in r.block([t] * 3, t))
    runs = -(-t // (run or t))
    lists = torch.tensor([0, 2, -1], dtype=torch.int32, device=gpu).expand(3, h, runs, 3).contiguous()
    prefix = r.cache.prefixes[0]

    def call():
        return paged_attention(q, prefix, ck, cv, blocks=lists, query_block=run, causal_block=causal)

    want = call()
    assert want.isfinite().all()
    pages = r.cache.block_table
    for b, x in enumerate(lens):
        for i in range(x // 32):
            if i not in (0, 2):
                r.cache.pool[0, int(pages[b, i])] = 255
    assert torch.equal(call(), want)
    ck[:, :, -1], cv[:, :, -1, 3] = ck[:, :, -1] * 0 + float("nan"), float("inf")
    out = call()
    for b, x in enumerate(lens):
        at = (x + torch.arange(t)) // causal
        last = (at == at[-1]).to(gpu)
        assert torch.equal(out[b, :, ~last], want[b, :, ~last]) and out[b, :, last].isnan().all()
    ck[:, :, -1] = 0
    out = call()
    for b, x in enumerate(lens):
        at = (x + torch.arange(t)) // causal
        last = (at == at[-1]).to(gpu)
        assert torch.equal(out[b, :, ~last], want[b, :, ~last])
        assert not out[b, :, last][..., 3].isfinite().any() and out[b, :, last][..., 4:].isfinite().all()


def test_pages_beyond_32_bit_offsets(gpu):
    """Rotated appends, selections and reads of pages at byte offsets past 2^31 and 2^32: as of a small pool."""
    d, h, page = 128, 1, 128
    rec = 40 * d * page // 32
    total = (1 << 32) // rec + 40
    far = [total - 1, (1 << 31) // rec + 1, total - 9, 5, (1 << 32) // rec, 0, (1 << 31) // rec - 1, 9]
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn((2, h, 500, d), generator=gen).to(BF).to(gpu) for _ in range(2))
    new = torch.tensor([500, 400], dtype=torch.int32, device=gpu)
    table = rotary_table(600, d, device=gpu)
    got = []
    for pages in (total, 8):
        c = PagedKVCache(num_layers=1, batch_size=2, num_kv_heads=h, head_dim=d, num_pages=pages, max_tokens=1024,
                         page_tokens=page, device=gpu)
        if pages == total:
            c.free_ring[:8] = torch.tensor(far, dtype=torch.int32, device=gpu)
        c.begin_append(new, 500)
        c.stage_layer(0, k, v, rotary=table)
        c.commit_append()
        c.check()
        x = list(c.dequantize_layer(0, 500))
        for t in (1, 40):
            q = torch.randn((2, 4, t, d), generator=torch.Generator().manual_seed(t)).to(BF).to(gpu)
            rq, _ = c.rotate(q, rotary=table)
            lists = c.select(0, rq, 4)
            x += [rq, lists, c.attend(0, rq, blocks=lists)]
        got.append(x)
        if pages == total:
            assert c.block_table[0, :4].tolist() == far[:4]
    assert all(torch.equal(x, y) for x, y in zip(*got))
