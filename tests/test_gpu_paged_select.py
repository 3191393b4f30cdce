"""Block selection over the paged cache: scores and blocks equal to whole-number arithmetic."""

import math

import pytest
import torch

from maskahead_amd.kernels.paged import PagedPrefix, select_blocks

from _paged import Requests, group_scores, select_rule

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


def _check(cache_pool, table, lens, new, q, h, got, *, count, per=32, run=0, first=0, last=0, mask=None):
    """Blocks and scores of every request, head and run, against the rule."""
    blocks, scores = (x.cpu() for x in got)
    t, g, m = q.shape[2], q.shape[1] // h, per // 32
    run = run or t
    assert blocks.shape == (len(lens), h, -(-t // run), count) and blocks.dtype is torch.int32
    pool, table = cache_pool.cpu(), table.cpu().tolist()
    for b, (x, n) in enumerate(zip(lens, new)):
        for kv in range(h):
            for r in range(blocks.shape[2]):
                rows = q[b, kv * g:(kv + 1) * g, r * run:min((r + 1) * run, n)].flatten(0, 1)
                s = group_scores(pool, table[b], x // 32, kv, rows) if len(rows) else []
                if mask is not None:
                    live = mask[b, kv, :len(s) * 32]
                    live = torch.nn.functional.pad(live, (0, len(s) * 32 - len(live))).view(len(s), 32).any(1).tolist()
                    s = [v if ok else None for v, ok in zip(s, live)]
                took, block = select_rule(s, m, count, first, last)
                assert blocks[b, kv, r].tolist() == took + [-1] * (count - len(took)), (b, kv, r)
                want = torch.full(scores[b, kv, r].shape, -math.inf)
                want[:len(block)] = torch.tensor(block, dtype=torch.float64).float()
                assert torch.equal(scores[b, kv, r], want), (b, kv, r)


@pytest.mark.parametrize("d,h,g,dtype,page,t,run", [(128, 2, 7, BF, 64, 1, 0), (64, 1, 4, F16, 32, 5, 0),
                                                    (128, 1, 1, F16, 96, 3, 1), (64, 2, 8, BF, 128, 9, 4),
                                                    (128, 1, 3, BF, 32, 32, 0), (64, 1, 2, BF, 64, 40, 64)])
@pytest.mark.parametrize("count,per,first,last", [(4, 32, 0, 0), (5, 96, 1, 1), (3, 64, 0, 2), (200, 32, 1, 0)])
def test_selection_is_that_of_whole_numbers(gpu, d, h, g, dtype, page, t, run, count, per, first, last):
    lens = [0, 31, 32, 700, 3000, 1024, 97]
    new = [t, t, t, t, max(1, t - 1), 0, t // 2]
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=page)
    q = torch.randn((7, h * g, t, d), generator=r.gen).to(dtype)
    for b, n in enumerate(new):
        q[b, :, n:] = float("nan")
    kw = dict(block_tokens=per, query_block=run, keep_first=first, keep_last=last)
    got = select_blocks(q.to(gpu), r.cache.prefixes[0], count, new_lens=r.i32(new), return_scores=True, **kw)
    _check(r.cache.pool[0], r.cache.block_table, lens, new, q, h, got, count=count, per=per, run=run, first=first, last=last)
    again = select_blocks(q.to(gpu), r.cache.prefixes[0], count, new_lens=r.i32(new), **kw)
    assert torch.equal(again, got[0])


def _store(dev, lens, *, h=1, d=64, page=32, dtype=BF, seed=0, width=None):
    """A store of random records whose parameters are finite, pages in no order; and its table."""
    g = torch.Generator().manual_seed(seed)
    width = width or max(-(-max(lens) // page), 1)
    per = page // 32
    pages = sum(-(-x // page) for x in lens) + 2
    pool = torch.randint(0, 256, (pages, h, per, 40 * d), generator=g, dtype=torch.uint8)
    par = torch.randn((pages, h, per, 4 * d), generator=g)
    par[..., :d], par[..., 2 * d:3 * d] = par[..., :d].abs() / 15, par[..., 2 * d:3 * d].abs()
    pool[..., 32 * d:] = par.to(F16).view(torch.uint8)
    ids = torch.randperm(pages, generator=g).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, x in enumerate(lens):
        for j in range(-(-x // page)):
            table[b, j] = ids.pop()
    tail = torch.zeros((len(lens), h, 32, d), dtype=dtype, device=dev)
    return pool, table, lambda mask=None: PagedPrefix(pool.to(dev), tail, tail, table.to(dev), torch.tensor(
        lens, dtype=torch.int32, device=dev), mask=mask)


def _set_params(pool, page, h, gi, *, scale=None, zero=None):
    d = pool.shape[3] // 40
    for at, x in ((32 * d, scale), (34 * d, zero)):
        if x is not None:
            pool[page, h, gi, at:at + 2 * d] = torch.as_tensor(x, dtype=F16).expand(d).contiguous().view(torch.uint8)


def test_equal_scores_go_to_the_lowest_index(gpu):
    lens, d = [32 * 600, 32 * 37], 64
    pool, table, prefix = _store(gpu, lens, d=d)
    gen = torch.Generator().manual_seed(4)
    for b, x in enumerate(lens):           # only three kinds of groups
        kinds = [(torch.rand(d, generator=gen), torch.randn(d, generator=gen)) for _ in range(3)]
        for i in range(x // 32):
            s, z = kinds[(i * 7) % 3 if i % 5 else 1]
            _set_params(pool, table[b, i], 0, 0, scale=s, zero=z)
    q = torch.randn((2, 3, 1, d), generator=gen).to(BF)
    for count in (1, 7, 36, 37, 38, 200, 201, 599, 600, 700):
        got = select_blocks(q.to(gpu), prefix(), count, return_scores=True)
        _check(pool, table, lens, [1, 1], q, 1, got, count=count)
    _check(pool, table, lens, [1, 1], q, 1, select_blocks(q.to(gpu), prefix(), 9, block_tokens=96, keep_first=2, keep_last=3,
                                                          return_scores=True), count=9, per=96, first=2, last=3)


@pytest.mark.parametrize("dtype", [BF, F16])
def test_values_of_any_size(gpu, dtype):
    """Outlier channels, zeros, subnormal and largest parameters and queries, infinities and NaN."""
    d, lens = 64, [32 * 40] * 6
    pool, table, prefix = _store(gpu, lens, d=d, dtype=dtype, seed=3)
    gen = torch.Generator().manual_seed(5)
    par = torch.zeros(d, dtype=F16)
    for b in range(6):
        row = table[b].tolist()
        out = par.clone()
        out[3] = 40000.0
        _set_params(pool, row[1], 0, 0, zero=out)
        _set_params(pool, row[2], 0, 0, scale=0.0, zero=0.0)
        _set_params(pool, row[3], 0, 0, scale=6e-8, zero=-6e-8)
        _set_params(pool, row[4], 0, 0, scale=65504.0, zero=-65504.0)
        _set_params(pool, row[5], 0, 0, scale=0.0, zero=2.0 ** -14)
        if b % 2:
            out[3] = float("inf")
            _set_params(pool, row[6], 0, 0, zero=out)
            out[3] = float("nan")
            _set_params(pool, row[7], 0, 0, scale=out)
    q = torch.randn((6, 2, 2, d), generator=gen)
    q[0] *= 1e-4
    q[1] = 0.0
    q[2, :, :, 5] = 3e4 if dtype is F16 else 3e38
    q[3, 0, 1, 7] = float("nan")
    q[4, 1, 0, 9] = float("-inf")
    q[5] *= 1e-7 if dtype is F16 else 1e-39
    q = q.to(dtype)
    got = select_blocks(q.to(gpu), prefix(), 6, query_block=1, return_scores=True)
    _check(pool, table, lens, [2] * 6, q, 1, got, count=6, run=1)


def test_pages_that_are_none_and_dead_tokens(gpu):
    lens = [32 * 50, 33, 32 * 20 + 5]
    pool, table, prefix = _store(gpu, lens, h=2, page=64, seed=6, width=30)
    table[0, 3], table[0, 7], table[2, 1] = -1, 9999, -5
    q = torch.randn((3, 4, 2, 64)).to(BF)
    got = select_blocks(q.to(gpu), prefix(), 11, block_tokens=64, return_scores=True)
    _check(pool, table, lens, [2] * 3, q, 2, got, count=11, per=64)
    for tokens in (0, 3, 32 * 30, 32 * 60):
        mask = (torch.rand((3, 2, tokens)) < 0.03).to(torch.uint8)
        if tokens > 640:
            mask[0, 0, 32:640] = 0
        wide = torch.zeros((3, 2, tokens + 5), dtype=torch.uint8)
        wide[..., 2:tokens + 2] = mask
        got = select_blocks(q.to(gpu), prefix(wide.to(gpu)[..., 2:tokens + 2]), 11, keep_first=1, keep_last=1,
                            return_scores=True)
        _check(pool, table, lens, [2] * 3, q, 2, got, count=11, first=1, last=1, mask=mask)


@pytest.mark.parametrize("groups", [1023, 4096, 5000, 17000, 33000])
def test_long_requests(gpu, groups):
    """Every way in which a selection keeps its keys."""
    lens = [32 * groups + 3, 32]
    pool, table, prefix = _store(gpu, lens, page=128, seed=groups)
    q = torch.randn((2, 2, 1, 64), generator=torch.Generator().manual_seed(1)).to(BF)
    for count in (1, 200, groups // 2):
        blocks, scores = (x.cpu() for x in select_blocks(q.to(gpu), prefix(), count, return_scores=True, keep_last=1))
        s = scores[0, 0, 0, :groups]
        if count == 1:
            want = torch.tensor(group_scores(pool, table[0].tolist(), 40, 0, q[0, :, 0]), dtype=torch.float64).float()
            assert torch.equal(s[:40], want) and torch.isfinite(s).all()
        s = s.clone()
        s[-1] = math.inf
        order = torch.sort(s, descending=True, stable=True).indices[:count]
        assert torch.equal(blocks[0, 0, 0].long(), order.sort().values)
        assert blocks[1, 0, 0, 0] == 0 and (blocks[1, 0, 0, 1:] == -1).all()


def test_many_requests_and_rows(gpu):
    lens = [(37 * i) % 400 for i in range(150)]
    pool, table, prefix = _store(gpu, lens, seed=8)
    new = [i % 4 for i in range(150)]
    q = torch.randn((150, 2, 3, 64)).to(BF)
    got = select_blocks(q.to(gpu), prefix(), 3, new_lens=torch.tensor(new, dtype=torch.int32, device=gpu), query_block=2,
                        return_scores=True)
    _check(pool, table, lens, new, q, 1, got, count=3, run=2)
    q = torch.randn((1, 6, 50, 64)).to(BF)          # 300 rows
    pool, table, prefix = _store(gpu, [2000], seed=9)
    _check(pool, table, [2000], [50], q, 1, select_blocks(q.to(gpu), prefix(), 20, return_scores=True), count=20)


def test_captured_other_streams_and_strides(gpu):
    lens = [900, 50]
    pool, table, prefix = _store(gpu, lens, seed=10, h=2)
    p = prefix()
    q = torch.randn((2, 3, 4, 64)).to(BF).transpose(1, 2)[:, :, 1:]        # [B, T, H, D] rows
    buf = torch.zeros((2, 3, 4, 64), dtype=BF, device=gpu).transpose(1, 2)
    dq = buf[:, :, 1:]
    assert dq.shape == q.shape
    dq.copy_(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = select_blocks(dq, p, 6, return_scores=True)
    s.synchronize()
    _check(pool, table, lens, [2, 2], q, 2, a, count=6)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = select_blocks(dq, p, 6, return_scores=True)
    for i in range(4):
        q = torch.randn((2, 4, 2, 64)).to(BF)
        dq.copy_(q)
        eager = select_blocks(dq, p, 6, return_scores=True)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0]) and torch.equal(got[1], eager[1])
        _check(pool, table, lens, [2, 2], q, 2, got, count=6)


def test_nothing_to_select_from_and_refusals(gpu):
    pool, table, prefix = _store(gpu, [40, 0])
    p = prefix()
    q = torch.zeros((2, 2, 3, 64), dtype=BF, device=gpu)
    assert select_blocks(q[:, :, :0], p, 4).shape == (2, 1, 0, 4)
    assert (select_blocks(q, p, 4, new_lens=torch.zeros(2, dtype=torch.int32, device=gpu)) == -1).all()
    for bad in (dict(count=0), dict(count=2, keep_first=2, keep_last=1), dict(count=2, block_tokens=48),
                dict(count=2, block_tokens=0), dict(count=2, query_block=-1), dict(count=2, keep_first=-1),
                dict(count=1 << 31), dict(count=2, new_lens=torch.zeros(3, dtype=torch.int32, device=gpu))):
        with pytest.raises(ValueError):
            select_blocks(q, p, **bad)
    with pytest.raises(ValueError):
        select_blocks(q.half(), p, 2)
    with pytest.raises(ValueError):
        select_blocks(q[:1], p, 2)


def test_many_runs_of_many_rows(gpu):
    """Workgroups that share their rows' digits among 128 groups."""
    lens, h, t, run = [2100, 900, 4300, 32], 4, 200, 17
    pool, table, prefix = _store(gpu, lens, h=h, page=64, seed=12, width=300)
    new = [200, 45, 170, 0]
    q = torch.randn((4, h * 4, t, 64), generator=torch.Generator().manual_seed(3)).to(BF)
    got = select_blocks(q.to(gpu), prefix(), 7, new_lens=torch.tensor(new, dtype=torch.int32, device=gpu), query_block=run,
                        keep_first=1, return_scores=True)
    # (of 48 selections a request some are checked against whole numbers, all against a call of their own)
    blocks, scores = (x.cpu() for x in got)
    for b, kv, r in ((0, 0, 0), (0, 3, 11), (1, 2, 2), (2, 1, 9), (1, 0, 5)):
        rows = q[b, kv * 4:kv * 4 + 4, r * run:min((r + 1) * run, new[b])].flatten(0, 1)
        s = group_scores(pool, table[b].tolist(), lens[b] // 32, kv, rows) if len(rows) else []
        took, block = select_rule(s, 1, 7, 1, 0)
        assert blocks[b, kv, r].tolist() == took + [-1] * (7 - len(took))
        assert torch.equal(scores[b, kv, r, :len(block)], torch.tensor(block, dtype=torch.float64).float())
    for r in range(12):
        one = torch.tensor([min(max(n - r * run, 0), run) for n in new], dtype=torch.int32, device=gpu)
        part = torch.zeros((4, h * 4, run, 64), dtype=BF)
        x = q[:, :, r * run:(r + 1) * run]
        part[:, :, :x.shape[2]] = x
        alone = select_blocks(part.to(gpu), prefix(), 7, new_lens=one, keep_first=1, return_scores=True)
        assert torch.equal(alone[0][:, :, 0].cpu(), blocks[:, :, r]) and torch.equal(alone[1][:, :, 0].cpu(), scores[:, :, r])
