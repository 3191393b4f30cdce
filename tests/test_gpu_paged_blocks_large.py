"""Attention over lists of several hundred groups in one workgroup: a wave's records are looked up 64 at a
time, and a list's entries from the 65th on are read where they lie."""

import pytest
import torch

from maskahead_amd.kernels.paged import PagedPrefix, paged_attention

from _paged import Requests, attend64, check_attention

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("d,g,t,dtype,segments,count,causal", [
    # few rows: one workgroup of 4 waves a segment (more segments than CUs), of 8 (about as many)
    (128, 7, 1, BF, 1.2, 150, 0), (64, 3, 5, F16, 1.2, 150, 0), (128, 7, 4, F16, 1.2, 140, 0), (64, 8, 4, BF, 1.2, 150, 4),
    (128, 7, 1, BF, 0.8, 280, 0), (64, 4, 4, F16, 0.8, 280, 0), (128, 6, 5, BF, 0.8, 270, 0),
    # many: one of 4 (f16, D 128: 3) items a step
    (128, 4, 10, BF, 0.55, 150, 0), (128, 4, 10, F16, 0.55, 150, 0), (64, 7, 20, BF, 0.55, 150, 16), (64, 7, 10, F16, 0.55, 140, 0)])
@pytest.mark.parametrize("dead", [False, True])
def test_lists_of_hundreds_of_groups(gpu, d, g, t, dtype, segments, count, causal, dead):
    h, page, per = 2, 64, 64
    base = Requests(gpu, [20480], h=h, d=d, dtype=dtype, page=page, room=0, pieces=[20480])
    gen, cus = base.gen, torch.cuda.get_device_properties(gpu).multi_processor_count
    b = int(cus * segments) // h
    # every request's pages are the first one's in an order of its own
    ids, pages = base.cache.block_table[0].cpu(), 20480 // page
    order = torch.stack([torch.randperm(pages, generator=gen) for _ in range(b)])
    lens = [int(x) for x in torch.randint(count * per, 20480, (b,), generator=gen)]
    lens[0], lens[1], lens[2] = 20480, 300, 20447
    new = [t - (i % 2) * (t // 3) for i in range(b)]
    tails = [torch.randn((b, h, 32, d), generator=gen).to(dtype) for _ in range(2)]
    mask = (torch.rand((b, h, 20000), generator=gen) < 0.7).to(torch.uint8) if dead else None
    prefix = PagedPrefix(base.cache.pool[0], tails[0].to(gpu), tails[1].to(gpu), ids[order].to(torch.int32).to(gpu),
                         torch.tensor(lens, dtype=torch.int32, device=gpu), mask=mask.to(gpu) if dead else None)
    lists = torch.full((b, h, 1, count), -1, dtype=torch.int32)
    for i, x in enumerate(lens):
        for kv in range(h):
            nb = -(-(x // 32) // 2)
            pick = torch.randperm(nb, generator=gen)[:count]
            if i % 2:
                pick = pick.sort().values
            lists[i, kv, 0, :len(pick)] = pick.to(torch.int32)
            if i % 3 == 2 and len(pick) > 100:
                lists[i, kv, 0, 70], lists[i, kv, 0, 99] = -1, nb
    q = torch.randn((b, h * g, t, d), generator=gen).to(dtype)
    ck, cv = (torch.randn((b, h, t, d), generator=gen).to(dtype) for _ in range(2))
    news = torch.tensor(new, dtype=torch.int32, device=gpu)
    before = torch.randn((b, h * g, t, d), generator=gen).to(dtype)
    kw = dict(new_lens=news, blocks=lists.to(gpu), block_tokens=per, causal_block=causal)
    out = paged_attention(q.to(gpu), prefix, ck.to(gpu), cv.to(gpu), out=before.to(gpu), **kw)
    again = paged_attention(q.to(gpu), prefix, ck.to(gpu), cv.to(gpu), out=before.to(gpu), **kw)
    assert torch.equal(out, again)
    k64, v64 = base.kv64(0)
    out = out.cpu()
    for i in [*range(4), b // 2, b - 2, b - 1]:
        x, n = lens[i], new[i]
        assert torch.equal(out[i, :, n:], before[i, :, n:])
        token = (order[i][:, None] * page + torch.arange(page)).flatten()
        whole = x // 32 * 32
        for kv in range(h):
            seen = torch.zeros(whole, dtype=torch.bool)
            nb = -(-(x // 32) // 2)
            for e in lists[i, kv, 0].tolist()[:nb]:
                if 0 <= e < nb:
                    seen[e * per:(e + 1) * per] = True
            rest = torch.ones(x - whole, dtype=torch.bool)
            if dead:
                live = torch.nn.functional.pad(mask[i, kv], (0, max(0, x - mask.shape[2])))[:x] != 0
                seen, rest = seen & live[:whole], rest & live[whole:]
            at = token[:whole][seen]
            # (the tokens that count, and those before the block that do not: causal blocks are counted from token 0)
            k = torch.cat((k64[kv:kv + 1, at], tails[0][i, kv:kv + 1, :x - whole][:, rest].double()), 1)
            v = torch.cat((v64[kv:kv + 1, at], tails[1][i, kv:kv + 1, :x - whole][:, rest].double()), 1)
            gap = -(k.shape[1] - x) % causal if causal else 0
            none = torch.zeros((1, gap, d), dtype=torch.float64)
            k, v = torch.cat((none, k), 1), torch.cat((none, v), 1)
            see = torch.ones((1, k.shape[1]), dtype=torch.bool)
            see[:, :gap] = False
            want, bound = attend64(q[i, kv * g:(kv + 1) * g, :n], k, v, ck[i, kv:kv + 1, :n], cv[i, kv:kv + 1, :n], seen=see,
                                   causal=causal)
            check_attention(out[i, kv * g:(kv + 1) * g, :n], want, bound, dtype)
