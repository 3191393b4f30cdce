"""Positions over the paged cache: rotated rows bit for bit against the same f32 operations and
within half a step of 64 bits, rotated appends bit for bit against a rotation and an append."""

import pytest
import torch

from maskahead_amd.kernels.paged import PagedPrefix, append_pages, plan_pages, rotary_table, rotate_block
from maskahead_amd.paged import PagedKVCache

from _paged import Requests, attend64, check_attention, rotated

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


def _prefix(dev, lens, *, h=2, d=128, dtype=BF, page=32, width=64):
    b = len(lens)
    return PagedPrefix(torch.zeros((4, h, page // 32, 40 * d), dtype=torch.uint8, device=dev),
                       torch.zeros((b, h, 32, d), dtype=dtype, device=dev), torch.zeros((b, h, 32, d), dtype=dtype, device=dev),
                       torch.full((b, width), -1, dtype=torch.int32, device=dev),
                       torch.tensor(lens, dtype=torch.int32, device=dev))


def _check(got, x, table, first, interleaved):
    """Equal to the f32 operations; and within the roundings of 64 bits: a product and a sum in f32
    (2^-24 each, of |x c| + |y s|, three in all) and half a step of the type."""
    got = got.cpu()
    assert torch.equal(got, rotated(x, table, first, interleaved)), "other bits than the same operations"
    want = rotated(x.double(), table.double(), first, interleaved)
    size = rotated(x.double().abs(), table.double().abs(), first, interleaved, add=True)
    bound = 3 * 2.0 ** -24 * size * (1 + 2.0 ** -7) + torch.finfo(x.dtype).eps / 2 * want.abs() + \
        torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("d,dtype,rd,interleaved", [(128, BF, 128, False), (128, F16, 128, True), (64, BF, 64, True),
                                                    (64, F16, 64, False), (128, BF, 64, False), (128, F16, 16, False),
                                                    (64, BF, 48, True), (128, BF, 112, False)])
@pytest.mark.parametrize("t,hq,hk", [(1, 7, 1), (5, 4, 2), (33, 9, 5)])
def test_rotated_rows(gpu, d, dtype, rd, interleaved, t, hq, hk):
    g = torch.Generator().manual_seed(d + rd + t)
    lens = [0, 1, 40, 900]
    table = rotary_table(950, d, rotary_dim=rd, base=1e6, device="cpu")
    q, k = (torch.randn((4, h, t, d), generator=g).to(dtype) for h in (hq, hk))
    p = _prefix(gpu, lens, d=d, dtype=dtype)
    gq, gk = rotate_block(p, q.to(gpu), k.to(gpu), rotary=table.to(gpu), interleaved=interleaved)
    _check(gq, q, table, lens, interleaved)
    _check(gk, k, table, lens, interleaved)
    # positions of the caller's, one of them below and one behind the table
    first = [948, 3, -2, 2 ** 31 - 1]
    gq, none = rotate_block(p, q.to(gpu), rotary=table.to(gpu), interleaved=interleaved,
                            positions=torch.tensor(first, dtype=torch.int32, device=gpu))
    assert none is None
    _check(gq, q, table, first, interleaved)


def test_rotated_rows_of_other_strides_and_in_place(gpu):
    g = torch.Generator().manual_seed(1)
    lens, t, d, rd = [5, 77], 11, 128, 96
    wide = rotary_table(100, d, rotary_dim=d, device="cpu")
    table = wide[:, 16:16 + rd]                      # rows of a wider tensor, 16-byte aligned
    p = _prefix(gpu, lens, d=d)
    q = torch.randn((2, t, 6, d + 2), generator=g).to(BF)[..., :d].transpose(1, 2)      # [B, T, H, D + 2] rows
    k = torch.randn((2, 3, t, d), generator=g).to(BF)
    dq = torch.zeros((2, t, 6, d + 2), dtype=BF, device=gpu)
    dq[..., :d].transpose(1, 2).copy_(q)
    qv, dk = dq[..., :d].transpose(1, 2), k.to(gpu)
    dt = wide.to(gpu)[:, 16:16 + rd]
    oq, ok = rotate_block(p, qv, dk, rotary=dt, out_query=qv, out_key=dk)
    assert oq is qv and ok is dk
    _check(qv, q, table, lens, False)
    _check(dk, k, table, lens, False)
    assert (dq[..., d:] == 0).all()
    # no positions, no heads
    assert rotate_block(p, q[:, :, :0].to(gpu), rotary=dt)[0].shape == (2, 6, 0, d)
    oq, ok = rotate_block(p, q[:, :0].to(gpu), k.to(gpu), rotary=dt)
    assert oq.shape == (2, 0, t, d)
    _check(ok, k, table, lens, False)


def test_a_long_chunk_is_rotated(gpu):
    g = torch.Generator().manual_seed(2)
    lens, t = [30000, 7], 1025
    table = rotary_table(31100, 128, base=1e6, device=gpu)
    q, k = (torch.randn((2, h, t, 128), generator=g).to(BF) for h in (5, 2))
    gq, gk = rotate_block(_prefix(gpu, lens), q.to(gpu), k.to(gpu), rotary=table)
    _check(gq, q, table.cpu(), lens, False)
    _check(gk, k, table.cpu(), lens, False)


def test_the_table_holds_far_angles(gpu):
    """Row 1 000 000 of the table against angles reduced in whole turns of 64 bits."""
    import math
    t = rotary_table(1000001, 64, base=1e6, rotary_dim=16, device=gpu)[-1].double().cpu()
    for i in range(8):
        a = math.fmod(1e6 * 1e6 ** (-i / 8), 2 * math.pi)
        assert abs(t[i] - math.cos(a)) < 1e-7 and abs(t[8 + i] - math.sin(a)) < 1e-7
    inv = torch.tensor([0.5, 0.25] * 4)
    u = rotary_table(3, 64, rotary_dim=16, inv_freq=inv, device="cpu")
    assert torch.equal(u[2, :8], (2 * inv.double()).cos().float()) and torch.equal(u[0, 8:], torch.zeros(8))


@pytest.mark.parametrize("d,h,dtype,page,rd,interleaved", [(128, 2, BF, 64, 128, False), (128, 3, F16, 32, 64, False),
                                                           (64, 1, BF, 128, 64, True), (64, 4, F16, 64, 64, False),
                                                           (128, 1, BF, 96, 128, True), (64, 2, BF, 32, 32, False)])
@pytest.mark.parametrize("new,t", [([1, 1, 0, 1, 1], 1), ([40, 3, 0, 33, 100], 100), ([32, 31, 0, 1, 64], 70)])
def test_a_rotated_append_is_a_rotation_and_an_append(gpu, d, h, dtype, page, rd, interleaved, new, t):
    lens = [31, 0, 50, 64, 97]
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=page, room=200)
    c = r.cache
    table = rotary_table(400, d, rotary_dim=rd, device=gpu)
    k, v = (x.to(gpu) for x in r.block(new, t))
    q = torch.randn((5, 5, t, d), generator=r.gen).to(dtype).to(gpu)
    for positions in (None, torch.tensor([0, 299, 3, 17, 40], dtype=torch.int32, device=gpu)):
        news = r.i32(new)
        pool, kt, vt = c.pool.clone(), c.k_tail.clone(), c.v_tail.clone()
        slots, ends = plan_pages(c.lengths, news, c.block_table.clone(), c.free_ring.clone(), c.ring_state.clone(),
                                 page_tokens=page, tokens=t)
        p = c.prefixes[0]
        kw = dict(rotary=table, interleaved=interleaved, positions=positions)
        kept = k.clone()
        got = append_pages(p, k, v, news, slots, query=q, **kw)
        mine = (c.pool.clone(), c.k_tail.clone(), c.v_tail.clone())
        assert torch.equal(k.view(torch.int16), kept.view(torch.int16))
        c.pool.copy_(pool), c.k_tail.copy_(kt), c.v_tail.copy_(vt)
        gq, gk = rotate_block(p, q, k, **kw)
        assert append_pages(p, gk, v, news, slots) is None
        assert torch.equal(got, gq)
        for a, b in zip(mine, (c.pool, c.k_tail, c.v_tail)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        # into the queries themselves, and without any
        c.pool.copy_(pool), c.k_tail.copy_(kt), c.v_tail.copy_(vt)
        own = q.clone()
        assert append_pages(p, k, v, news, slots, query=own, out_query=own, **kw) is own
        assert torch.equal(own, gq)
        c.pool.copy_(pool), c.k_tail.copy_(kt), c.v_tail.copy_(vt)
        assert append_pages(p, k, v, news, slots, **kw) is None
        for a, b in zip(mine, (c.pool, c.k_tail, c.v_tail)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        c.pool.copy_(pool), c.k_tail.copy_(kt), c.v_tail.copy_(vt)


def test_a_refused_plan_stores_nothing_and_rotates(gpu):
    r = Requests(gpu, [40, 3], room=64)
    c, t = r.cache, 2
    table = rotary_table(200, 128, device=gpu)
    k, v = (x.to(gpu) for x in r.block([2, 2], t))
    q = torch.randn((2, 2, t, 128), generator=r.gen).to(BF)
    pool, kt = c.pool.clone(), c.k_tail.clone()
    slots = torch.full((2, t), -1, dtype=torch.int64, device=gpu)
    got = append_pages(c.prefixes[0], k, v, r.i32([2, 2]), slots, rotary=table, query=q.to(gpu))
    _check(got, q, table.cpu(), [40, 3], False)
    assert torch.equal(pool, c.pool) and torch.equal(kt.view(torch.int16), c.k_tail.view(torch.int16))


@pytest.mark.parametrize("dtype,d", [(BF, 128), (F16, 64)])
def test_tokens_rotated_staged_and_read(gpu, dtype, d):
    """A decoding step, five times, through a captured graph: rotated on the way, read while staged."""
    lens, hq, h = [0, 30, 100, 64], 4, 2
    table = rotary_table(300, d, device=gpu)
    cpu = table.cpu()
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=32)
    c = r.cache
    new = [1, 1, 0, 1]
    news, k, v = r.i32(new), *(x.to(gpu) for x in r.block(new, 1))
    q = torch.zeros((4, hq, 1, d), dtype=dtype, device=gpu)
    out = torch.zeros_like(q)

    def step():
        c.begin_append(news, 1)
        with pytest.raises(RuntimeError):
            c.attend(0, q, staged=True)
        rq = c.stage_layer(0, k, v, rotary=table, query=q)
        with pytest.raises(RuntimeError):
            c.attend(0, rq)
        with pytest.raises(ValueError):
            c.attend(0, rq, k, v, staged=True)
        with pytest.raises(ValueError):
            c.attend(0, rq, causal_block=1, staged=True)
        c.attend(0, rq, staged=True, out=out)
        c.commit_append()

    graph = None
    for i in range(6):
        hk, hv = r.block(new, 1)
        hq_ = torch.randn((4, hq, 1, d), generator=r.gen).to(dtype)
        k.copy_(hk), v.copy_(hv), q.copy_(hq_)
        at = c.lengths.tolist()
        if i == 1:
            graph = torch.cuda.CUDAGraph()
            saved = [x.clone() for x in (c.pool, c.k_tail, c.v_tail, c.block_table, c.lengths, c.free_ring, c.ring_state)]
            with torch.cuda.graph(graph):
                step()
            for x, y in zip((c.pool, c.k_tail, c.v_tail, c.block_table, c.lengths, c.free_ring, c.ring_state), saved):
                x.copy_(y)
        graph.replay() if graph else step()
        torch.cuda.synchronize()
        r.note(new, rotated(hk, cpu, at, False), hv)
        rq = rotated(hq_, cpu, at, False)
        assert c.lengths.tolist() == [x + n for x, n in zip(at, new)]
        for b in range(4):
            if not new[b]:
                assert (out[b] == 0).all()
                continue
            kk, vv = r.kv64(b)
            none = torch.empty((h, 0, d), dtype=dtype)
            want, bound = attend64(rq[b], kk, vv, none, none, seen=torch.ones((h, kk.shape[1]), dtype=torch.bool))
            check_attention(out[b], want, bound, dtype)


def test_rotation_on_another_stream(gpu):
    table = rotary_table(64, 128, device=gpu)
    p = _prefix(gpu, [3])
    q = torch.randn((1, 4, 9, 128)).to(BF)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = q.to(gpu)
        got, _ = rotate_block(p, x, rotary=table)
    s.synchronize()
    _check(got, q, table.cpu(), [3], False)


def test_refused_shapes(gpu):
    p = _prefix(gpu, [3, 4])
    table = rotary_table(16, 128, device=gpu)
    q = torch.zeros((2, 4, 3, 128), dtype=BF, device=gpu)
    k = torch.zeros((2, 2, 3, 128), dtype=BF, device=gpu)
    news, slots = torch.ones(2, dtype=torch.int32, device=gpu), torch.full((2, 3), -1, device=gpu)
    for bad in (table[:, :24], table.double(), table[0], table[:0], table.t()):
        with pytest.raises(ValueError):
            rotate_block(p, q, k, rotary=bad)
        with pytest.raises(ValueError):
            append_pages(p, k, k, news, slots, rotary=bad)
    off = torch.zeros(16 * 128 + 1, device=gpu)[1:].view(16, 128)
    for call in (lambda: rotate_block(p, q, rotary=off), lambda: rotate_block(p, q, k[:, :, :2], rotary=table),
                 lambda: rotate_block(p, q, rotary=table, positions=news.long()),
                 lambda: rotate_block(p, q, rotary=table, out_key=k),
                 lambda: rotate_block(p, q, k, rotary=table, out_query=q[:, :2]),
                 lambda: rotate_block(p, q.half(), k, rotary=table),
                 lambda: rotate_block(p, q, out_query=q[:, :1].expand(2, 4, 3, 128), rotary=table),
                 lambda: append_pages(p, k, k, news, slots, rotary=table, query=q, out_query=q[:1].expand(2, 4, 3, 128)),
                 lambda: append_pages(p, k, k, news, slots, query=q),
                 lambda: append_pages(p, k, k, news, slots, rotary=table, query=q[:, :, :1]),
                 lambda: append_pages(p, k, k, news, slots, rotary=table, out_query=q),
                 lambda: append_pages(p, k, k, news, slots, positions=news),
                 lambda: rotary_table(0, 128), lambda: rotary_table(4, 128, rotary_dim=24),
                 lambda: rotary_table(4, 64, rotary_dim=128), lambda: rotary_table(4, 64, inv_freq=table[0])):
        with pytest.raises(ValueError):
            call()
