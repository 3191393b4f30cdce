"""Block selection where its kernels take further turns: more units of work than workgroups, rows of
several turns, and every way in which a selection keeps its keys, with blocks of several groups."""

import math

import pytest
import torch

from maskahead_amd.kernels.paged import PagedPrefix, select_blocks

from _paged import group_scores, group_scores_of

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


def _shared(dev, lens, *, h, d, page, dtype, pages=61, seed=0, width=None):
    """Requests of these lengths whose table rows name pages of one small pool, in no order."""
    g = torch.Generator().manual_seed(seed)
    pool = torch.randint(0, 256, (pages, h, page // 32, 40 * d), generator=g, dtype=torch.uint8)
    par = torch.randn((pages, h, page // 32, 4 * d), generator=g)
    par[..., :d], par[..., 2 * d:3 * d] = par[..., :d].abs() / 15, par[..., 2 * d:3 * d].abs()
    pool[..., 32 * d:] = par.to(F16).view(torch.uint8)
    width = width or -(-max(lens) // page)
    table = torch.randint(0, pages, (len(lens), width), generator=g, dtype=torch.int32)
    tail = torch.zeros((len(lens), h, 32, d), dtype=dtype, device=dev)
    return pool, table, PagedPrefix(pool.to(dev), tail, tail, table.to(dev),
                                    torch.tensor(lens, dtype=torch.int32, device=dev))


def _taken(scores, m, count, last):
    """The blocks of m groups that are taken (keep_last: last), and every block's score."""
    pad = torch.nn.functional.pad(scores, (0, -len(scores) % m), value=-math.inf).view(-1, m).amax(1)
    key = pad.clone()
    if last:
        key[len(key) - last:] = math.inf
    order = torch.sort(key, descending=True, stable=True).indices[:count]
    return order.sort().values, pad


def _check_row(got, scores, m, count, last):
    blocks, out = got
    want, block = _taken(scores, m, count, last)
    assert torch.equal(blocks[:len(want)].long(), want) and (blocks[len(want):] == -1).all()
    assert torch.equal(out[:len(block)], block) and (out[len(block):] == -math.inf).all()


def test_both_oracles_agree():
    g = torch.Generator().manual_seed(2)
    pool = torch.randint(0, 256, (5, 2, 2, 40 * 64), generator=g, dtype=torch.uint8)
    pool[..., 32 * 64:] = torch.randn((5, 2, 2, 4 * 64), generator=g).to(F16).view(torch.uint8)
    q = torch.randn((3, 64), generator=g).to(BF)
    row = [4, 0, 3, 3, 1]
    one = torch.tensor(group_scores(pool, row, 9, 1, q), dtype=torch.float64).float()
    assert torch.equal(one, group_scores_of(pool, row, 9, 1, q))


@pytest.mark.parametrize("d,dtype,b,h,g,t,run,most,waves", [
    (128, BF, 96, 8, 2, 1, 0, 16384, 4), (64, F16, 96, 8, 7, 7, 0, 12000, 4),      # a tile; four
    (64, BF, 12, 8, 7, 400, 20, 20000, 8), (128, F16, 8, 8, 5, 640, 20, 20000, 8)])  # nine and seven of 8 waves'
def test_more_units_than_workgroups(gpu, d, dtype, b, h, g, t, run, most, waves):
    gen = torch.Generator().manual_seed(b + t)
    lens = [int(x) for x in torch.randint(most // 2, most, (b,), generator=gen)]
    lens[1], lens[-1] = 31, most
    new = [t - (i % 3) * (t // 3) for i in range(b)]
    pool, table, prefix = _shared(gpu, lens, h=h, d=d, page=64, dtype=dtype, seed=t)
    run_ = run or t
    units = sum(-(-(x // 32) // (16 * waves)) * h * -(-n // run_) for x, n in zip(lens, new))
    assert units > 3 * 4 * torch.cuda.get_device_properties(gpu).multi_processor_count
    q = torch.randn((b, h * g, t, d), generator=gen) * torch.exp(torch.randn((b, h * g, t, 1), generator=gen))
    q = q.to(dtype)
    news = torch.tensor(new, dtype=torch.int32, device=gpu)
    kw = dict(new_lens=news, query_block=run, keep_last=1)
    blocks, scores = (x.cpu() for x in select_blocks(q.to(gpu), prefix, 20, return_scores=True, **kw))
    again = select_blocks(q.to(gpu), prefix, 20, **kw).cpu()
    assert torch.equal(again, blocks)
    runs = blocks.shape[2]
    for i, (x, n) in enumerate(zip(lens, new)):
        for kv in range(h):
            for r in range(runs):
                if runs > 1 and (i + kv + r) % 3:            # (a third of the many runs)
                    continue
                rows = q[i, kv * g:(kv + 1) * g, r * run_:min((r + 1) * run_, n)].flatten(0, 1)
                if len(rows) == 0:
                    assert (blocks[i, kv, r] == -1).all() and (scores[i, kv, r] == -math.inf).all()
                    continue
                if x < 32:
                    assert (blocks[i, kv, r] == -1).all()
                    continue
                _check_row((blocks[i, kv, r], scores[i, kv, r]), group_scores_of(pool, table[i], x // 32, kv, rows), 1, 20, 1)


@pytest.mark.parametrize("per,groups", [(32, 5000), (32, 33000), (64, 2050), (96, 3100), (64, 8195), (96, 12400), (64, 65600), (96, 98500)])
def test_keys_of_long_rows(gpu, per, groups):
    """Rows of up to 1 024, 4 096, 32 768 and more blocks of one to three groups; every group's score."""
    m = per // 32
    lens = [32 * groups + 3, 32 * (groups // 2) + 5, 70]
    pool, table, prefix = _shared(gpu, lens, h=1, d=64, page=128, dtype=BF, seed=groups)
    q = torch.randn((3, 2, 1, 64), generator=torch.Generator().manual_seed(1)).to(BF)
    score = [group_scores_of(pool, table[b], x // 32, 0, q[b, :, 0]) for b, x in enumerate(lens)]
    for count in (1, 200, groups // m // 2):
        kw = dict(block_tokens=per, keep_last=1)
        blocks, scores = (x.cpu() for x in select_blocks(q.to(gpu), prefix, count, return_scores=True, **kw))
        for b in range(3):
            _check_row((blocks[b, 0, 0], scores[b, 0, 0]), score[b], m, count, 1)
        assert torch.equal(select_blocks(q.to(gpu), prefix, count, **kw).cpu(), blocks)


@pytest.mark.parametrize("d,dtype", [(128, BF), (128, F16), (64, F16)])
def test_rows_shared_by_eight_waves(gpu, d, dtype):
    """Workgroups of 8 waves, of every width and type."""
    lens, h, g, t, run = [2100, 900, 4300, 32], 4, 4, 200, 17
    new = [200, 45, 170, 0]
    pool, table, prefix = _shared(gpu, lens, h=h, d=d, page=64, dtype=dtype, seed=12, width=300)
    q = torch.randn((4, h * g, t, d), generator=torch.Generator().manual_seed(3)).to(dtype)
    blocks, scores = (x.cpu() for x in select_blocks(
        q.to(gpu), prefix, 7, new_lens=torch.tensor(new, dtype=torch.int32, device=gpu), query_block=run, keep_last=1,
        block_tokens=64, return_scores=True))
    for b, (x, n) in enumerate(zip(lens, new)):
        for kv in range(h):
            for r in range(blocks.shape[2]):
                rows = q[b, kv * g:(kv + 1) * g, r * run:min((r + 1) * run, n)].flatten(0, 1)
                if len(rows) == 0:
                    assert (blocks[b, kv, r] == -1).all() and (scores[b, kv, r] == -math.inf).all()
                else:
                    _check_row((blocks[b, kv, r], scores[b, kv, r]), group_scores_of(pool, table[b], x // 32, kv, rows), 2, 7, 1)
