"""The paged 4-bit cache: page plans against whole-number arithmetic, append and read-back bit
for bit against the oracle's quantizers, attention against 64 bits within the bound of its
roundings, and a run of the operators together against the contiguous cache's attention."""

import random

import pytest
import torch

from maskahead_amd.cache import PackedKVCache
from maskahead_amd.config import QuantizationConfig
from maskahead_amd.kernels.paged import (PagedPrefix, append_pages, check_plan, dequantize_pages, paged_attention,
                                         plan_pages)
from maskahead_amd.kernels.splitk import Prefix, splitk_attention
from maskahead_amd.paged import PagedKVCache

from _paged import Requests, attend64, check_attention, plan_rule, stored

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


# ------------------------------------------------------------------ plans
def _ring(dev, rng, b, width, total, page, lens):
    """A table, ring and state as after some use: pages of the lengths taken, the rest free."""
    ids = list(range(total))
    rng.shuffle(ids)
    table = [[-1] * width for _ in range(b)]
    for row, x in zip(table, lens):
        for j in range(-(-x // page)):
            row[j] = ids.pop()
    ring, head = [-7] * total, rng.randrange(total)
    for i, p in enumerate(ids):
        ring[(head + i) % total] = p
    return table, ring, [head, len(ids), 0, 0]


@pytest.mark.parametrize("b,tokens,page", [(1, 1, 32), (3, 40, 32), (64, 1, 64), (300, 7, 32), (5, 5000, 128),
                                           (1, 4097, 64), (2100, 1, 64), (17, 0, 96), (2049, 3, 32)])
def test_plans_follow_the_rule(gpu, b, tokens, page):
    rng = random.Random(b * 7 + tokens)
    most = 6 * page
    lens = [rng.choice([0, 1, page - 1, page, rng.randrange(most)]) for _ in range(b)]
    width = -(-(most + 6 * tokens) // page) + 1
    total = sum(-(-x // page) for x in lens) + b * (-(-6 * tokens // page) + 3)
    table, ring, state = _ring(gpu, rng, b, width, total, page, lens)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    # a table whose rows are part of a wider one
    wide = torch.full((b, width + 3), -9, dtype=torch.int32, device=gpu)
    wide[:, 1:width + 1] = i32(table)
    tg, rg, sg = wide[:, 1:width + 1], i32(ring), i32(state)
    for step in range(5):
        # growth, idle rows, part given back, everything given back (far below minus the length too)
        new = [rng.choice([tokens, 0, rng.randint(0, tokens), -rng.randint(0, x), -x, -2 ** 31 + 1]) if step else
               rng.choice([tokens, tokens // 2, 0]) for x in lens]
        slots, ends = plan_pages(i32(lens), i32(new), tg, rg, sg, page_tokens=page, tokens=tokens)
        want_slots, want_ends = plan_rule(lens, new, table, ring, state, page, tokens)
        assert ends.tolist() == want_ends
        assert torch.equal(slots.cpu(), torch.tensor(want_slots, dtype=torch.int64).reshape(b, tokens))
        assert torch.equal(tg.cpu(), torch.tensor(table, dtype=torch.int32))
        assert rg.tolist() == ring and sg.tolist() == state
        lens = want_ends
    assert (wide[:, 0] == -9).all() and (wide[:, width + 1:] == -9).all()
    check_plan(sg)


@pytest.mark.parametrize("what,bit", [("pages", 1), ("width", 2), ("tokens", 4), ("length", 8)])
def test_a_plan_that_cannot_be_met_changes_nothing(gpu, what, bit):
    rng = random.Random(3)
    lens, new, page, tokens, width = [40, 0, 100], [8, 33, -100], 32, 40, 4
    table, ring, state = _ring(gpu, rng, 3, width, 8, page, lens)      # 2 + 0 + 4 pages in use, 2 free
    if what == "pages":
        new = [40, 40, -100]
    elif what == "width":
        new = [8, 1, 40]
    elif what == "tokens":
        new = [41, 0, 0]
    else:
        lens[1] = -1
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    tg, rg, sg = i32(table), i32(ring), i32(state)
    slots, ends = plan_pages(i32(lens), i32(new), tg, rg, sg, page_tokens=page, tokens=tokens)
    assert (slots == -1).all() and ends.tolist() == lens
    assert tg.tolist() == table and rg.tolist() == ring and sg.tolist()[:3] == state[:3]
    assert sg.tolist()[3] & bit
    with pytest.raises(RuntimeError, match="page plan refused"):
        check_plan(sg)
    check_plan(sg)      # reported once
    lens = [40, 0, 100]
    # and the next plan goes through
    slots, ends = plan_pages(i32(lens), i32([8, 33, -100]), tg, rg, sg, page_tokens=page, tokens=tokens)
    want_slots, want_ends = plan_rule(lens, [8, 33, -100], table, ring, state, page, tokens)
    assert ends.tolist() == want_ends and slots.tolist() == want_slots and tg.tolist() == table


# ------------------------------------------------------------------ append and read-back
@pytest.mark.parametrize("d,h,dtype,page,pieces", [(128, 2, BF, 64, [1]), (128, 3, F16, 32, [33, 7]),
                                                   (64, 1, BF, 128, [200]), (64, 4, F16, 64, [31, 1, 32]),
                                                   (128, 8, BF, 96, [64])])
def test_append_stores_what_the_quantizers_store(gpu, d, h, dtype, page, pieces):
    lens = [0, 1, 31, 32, 33, 64, 97, 150]
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=page, pieces=pieces, layers=2)
    assert r.cache.lengths.tolist() == lens
    r.cache.check()
    for layer in range(2):
        for out in (torch.float32, dtype):
            k, v = r.cache.dequantize_layer(layer, 160, dtype=out)
            for b, n in enumerate(lens):
                for got, which, x in ((k, "k", r.k[b]), (v, "v", r.v[b])):
                    assert torch.equal(got[b, :, :n].cpu(), stored(x, which).to(torch.float32).to(out)), (b, which)
                    assert (got[b, :, n:] == 0).all()


def test_append_touches_only_what_it_names(gpu):
    r = Requests(gpu, [20, 70, 5, 0], page=32)
    c = r.cache
    for new, t in (([3, 40, 0, 0], 40), ([0, 0, 27, 64], 64)):
        pool, kt, vt = c.pool.clone(), c.k_tail.clone(), c.v_tail.clone()
        old = list(c.lengths.tolist())
        r.append(new, t)
        page_of = c.block_table.tolist()
        mine = set()
        for b, n in enumerate(new):
            for g in range(old[b] // 32, (old[b] + n) // 32):
                mine.add((page_of[b][g * 32 // 32], 0))
        changed = (c.pool != pool)[0].flatten(1).any(1).nonzero().flatten().tolist()
        assert set(changed) <= {p for p, _ in mine}
        for b, n in enumerate(new):
            x, y = old[b], old[b] + n
            for now, was in ((c.k_tail, kt), (c.v_tail, vt)):
                same = (now[0, b].view(torch.int16) == was[0, b].view(torch.int16)).all(-1).all(0).tolist()
                rows = set(range(32)) - set(range(x % 32 if x // 32 == y // 32 else 0, y % 32)) if n else set(range(32))
                assert all(same[i] for i in rows), (b, n)


def test_append_without_a_slot_stores_nothing(gpu):
    r = Requests(gpu, [20, 40], page=32, pages=4)
    c = r.cache
    before = [x.clone() for x in (c.pool, c.k_tail, c.v_tail, c.lengths, c.block_table)]
    k, v = r.block([30, 64], 64)
    slots = c.begin_append(r.i32([30, 64]), 64)          # 3 pages needed, 1 free
    assert (slots == -1).all()
    c.stage_layer(0, k.to(gpu), v.to(gpu))
    c.commit_append()
    for x, y in zip(before, (c.pool, c.k_tail, c.v_tail, c.lengths, c.block_table)):
        x, y = (t.view(torch.int16) if t.dtype == BF else t for t in (x, y))
        assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="free pages run out"):
        c.check()


@pytest.mark.parametrize("d", [64, 128])
def test_append_and_attention_take_any_strides(gpu, d):
    """New tokens and queries as views whose rows are not 16-byte aligned, heads innermost, and
    an output inside a wider tensor."""
    r = Requests(gpu, [45, 64], d=d, h=2)
    k, v = r.block([37, 30], 37)

    def odd(x):
        buf = torch.full((x.shape[0], x.shape[2], x.shape[1], d + 3), 7.0, dtype=x.dtype, device=gpu)
        y = buf.transpose(1, 2)[..., 1:d + 1]
        y.copy_(x)
        return y

    q = torch.randn((2, 6, 37, d), generator=r.gen).to(BF)
    new = r.i32([37, 30])
    wide = torch.full((2, 6, 37, d + 5), 3.0, dtype=BF, device=gpu)
    out = wide[..., 3:d + 3]
    got = r.cache.attend(0, odd(q), odd(k), odd(v), new_lens=new, out=out)
    assert got.data_ptr() == out.data_ptr()
    assert (wide[..., :3] == 3).all() and (wide[..., d + 3:] == 3).all()
    for b, n in enumerate([37, 30]):
        seen = torch.ones((2, r.lens[b]), dtype=torch.bool)
        want, bound = attend64(q[b, :, :n], *r.kv64(b), k[b, :, :n], v[b, :, :n], seen=seen)
        check_attention(got[b, :, :n], want, bound, BF)
    assert (got[1, :, 30:] == 3).all()
    slots = r.cache.begin_append(new, 37)
    append_pages(r.cache.prefixes[0], odd(k), odd(v), new, slots)
    r.cache._plan[3].add(0)
    r.cache.commit_append()
    r.note([37, 30], k, v)
    kk, vv = r.cache.dequantize_layer(0, 96, dtype=torch.float32)
    for b in range(2):
        n = r.k[b].shape[1]
        assert torch.equal(kk[b, :, :n].cpu().double(), stored(r.k[b], "k"))
        assert torch.equal(vv[b, :, :n].cpu().double(), stored(r.v[b], "v"))


@pytest.mark.parametrize("tokens", [1, 31, 32, 70, 300])
def test_read_back_of_a_range(gpu, tokens):
    lens = [0, 5, 64, 130, 200]
    r = Requests(gpu, lens, d=64, page=32, dtype=F16)
    starts = [0, 3, 33, 64, 199]
    k, v = r.cache.dequantize_layer(0, tokens, starts=r.i32(starts), dtype=torch.float32)
    for b, (n, s) in enumerate(zip(lens, starts)):
        for got, which, x in ((k, "k", r.k[b]), (v, "v", r.v[b])):
            want = torch.zeros((2, tokens, 64), dtype=torch.float64)
            part = stored(x, which)[:, s:s + tokens]
            want[:, :part.shape[1]] = part
            assert torch.equal(got[b].cpu().double(), want), (b, which)


def test_pages_that_the_pool_does_not_have_read_as_absent(gpu):
    r = Requests(gpu, [100, 100], page=32)
    c = r.cache
    q = torch.randn((2, 4, 1, 128), generator=r.gen).to(BF)
    c.block_table[0, 1] = -1
    c.block_table[1, 2] = c.num_pages
    k, _ = c.dequantize_layer(0, 100, dtype=torch.float32)
    got = c.attend(0, q.to(gpu))
    for b, lost in ((0, 1), (1, 2)):
        seen = torch.ones((2, 100), dtype=torch.bool)
        seen[:, 32 * lost:32 * lost + 32] = False
        want_k = stored(r.k[b], "k")
        want_k[:, 32 * lost:32 * lost + 32] = 0
        assert torch.equal(k[b].cpu().double(), want_k)
        none = torch.empty((2, 0, 128))
        want, bound = attend64(q[b], *r.kv64(b), none, none, seen=seen)
        check_attention(got[b], want, bound, BF)


# ------------------------------------------------------------------ attention
def _attend(gpu, *, lens, new, t, hq, h, d, dtype, page=64, causal=0, dead=0.0, current=True, scale=None, seed=0):
    r = Requests(gpu, lens, h=h, d=d, dtype=dtype, page=page, room=8, seed=seed)
    q = torch.randn((len(lens), hq, t, d), generator=r.gen).to(dtype)
    for b, n in enumerate(new):
        q[b, :, n:] = float("nan")
    k, v = r.block(new, t)
    mask = None
    if dead:
        mask = (torch.rand((len(lens), h, max(lens) + 1), generator=r.gen) >= dead).to(torch.uint8)
    out = torch.full((len(lens), hq, t, d), 5.0, dtype=dtype, device=gpu)
    r.cache.attend(0, q.to(gpu), k.to(gpu) if current else None, v.to(gpu) if current else None, new_lens=r.i32(new),
                   causal_block=causal, scaling=scale, mask=None if mask is None else mask.to(gpu), out=out)
    for b, n in enumerate(new):
        assert (out[b, :, n:] == 5.0).all(), "rows behind the new tokens changed"
        if n == 0:
            continue
        seen = torch.ones((h, lens[b]), dtype=torch.bool) if mask is None else mask[b, :, :lens[b]].bool()
        m = n if current else 0
        want, bound = attend64(q[b, :, :n], *r.kv64(b), k[b, :, :m], v[b, :, :m], seen=seen, causal=causal, scale=scale)
        check_attention(out[b, :, :n], want, bound, dtype)
    return r


@pytest.mark.parametrize("hq,h,t", [(1, 1, 1), (7, 1, 1), (16, 1, 1), (4, 2, 3), (17, 1, 1), (14, 2, 4), (7, 1, 8),
                                    (14, 2, 16), (8, 2, 32), (14, 2, 32), (16, 2, 33), (4, 4, 100)])
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, F16)])
def test_attention_over_ragged_requests(gpu, hq, h, t, d, dtype):
    """Row counts in and between the built tiles, head_dims and types, and lengths from none to
    several pages, part of them idle or padded."""
    _attend(gpu, lens=[0, 1, 31, 32, 100, 321], new=[t, t, max(1, t - 1), 0, t, (t + 1) // 2], t=t, hq=hq, h=h, d=d,
            dtype=dtype)


@pytest.mark.parametrize("d,dtype", [(64, BF), (128, F16)])
@pytest.mark.parametrize("causal", [1, 32, 40])
def test_attention_causal_by_blocks(gpu, d, dtype, causal):
    _attend(gpu, lens=[0, 7, 64, 95], new=[70, 70, 33, 64], t=70, hq=4, h=2, d=d, dtype=dtype, causal=causal, page=32)


@pytest.mark.parametrize("dead", [0.3, 0.97, 1.0])
@pytest.mark.parametrize("t,current", [(1, True), (1, False), (20, True), (20, False)])
def test_attention_skips_dead_entries(gpu, dead, t, current):
    """Entries the mask marks, up to all of them: a row that sees nothing is zero."""
    _attend(gpu, lens=[0, 40, 200, 333], new=[t] * 4, t=t, hq=8, h=2, d=128, dtype=BF, dead=dead, current=current, page=32)


def test_attention_with_nothing_to_see_is_zero(gpu):
    r = Requests(gpu, [0, 0], d=64)
    q = torch.randn((2, 2, 5, 64), generator=r.gen).to(BF).to(gpu)
    out = torch.full_like(q, 9.0)
    assert (r.cache.attend(0, q, out=out) == 0).all()


def test_dead_entries_may_hold_anything(gpu):
    """NaN and infinite parameters and tails behind a 0 of the mask change nothing."""
    r = Requests(gpu, [70, 45], page=32)
    c = r.cache
    q = torch.randn((2, 4, 2, 128), generator=r.gen).to(BF).to(gpu)
    mask = torch.ones((2, 2, 128), dtype=torch.uint8, device=gpu)
    mask[0, :, 32:64] = 0          # a whole group, one token of a group, one of the tail
    mask[1, :, 3] = 0
    mask[1, :, 40] = 0
    want = c.attend(0, q, mask=mask)
    page = c.block_table[0, 1].long()
    c.pool[0, page] = 0xff                                                 # f16 NaN parameters, codes 15
    other = c.block_table[1, 0].long()
    words = c.pool[0, other].view(torch.float16)             # [H, 1, 20 D] of the page's record
    for first in (18 * 128, 19 * 128):                       # value scales, value zeros: [4][32] of a token
        words[..., first + 3:first + 128:32] = float("inf")  # token 3 of every channel group
    c.pool[0, other] = words.view(torch.uint8)
    c.k_tail[0, 1, :, 8] = float("nan")
    c.v_tail[0, 1, :, 8] = float("nan")
    got = c.attend(0, q, mask=mask)
    assert torch.equal(got, want)


@pytest.mark.parametrize("scale_q,scale_k", [(3e4, 1e-4), (1e-5, 300.0), (1.0, 1e-6), (2e5, 1e-6)])
def test_attention_of_large_and_small_values(gpu, scale_q, scale_k):
    """Queries outside f16's range and keys near its ends: the scores stay ordinary."""
    r = Requests(gpu, [200], h=1)
    k = (r.k[0].float() * scale_k).to(BF)
    r2 = Requests(gpu, [0], h=1, room=256)
    r2.cache.begin_append(r2.i32([200]), 200)
    r2.cache.stage_layer(0, k[None].to(gpu), r.v[0][None].to(gpu))
    r2.cache.commit_append()
    q = (torch.randn((1, 2, 1, 128), generator=r.gen) * scale_q).to(BF)
    got = r2.cache.attend(0, q.to(gpu))
    none = torch.empty((1, 0, 128))
    want, bound = attend64(q[0], stored(k, "k"), stored(r.v[0], "v"), none, none, seen=torch.ones((1, 200), dtype=torch.bool))
    assert torch.isfinite(got).all()
    assert ((got[0].double().cpu() - want).abs() <= bound).all()


def test_attention_over_long_requests(gpu):
    """Requests cut between many workgroups beside short ones, with other heads' and rows' counts."""
    _attend(gpu, lens=[20000, 3, 777], new=[1, 1, 1], t=1, hq=7, h=1, d=128, dtype=BF, page=128)
    _attend(gpu, lens=[9000, 3, 777], new=[32, 32, 5], t=32, hq=7, h=1, d=128, dtype=BF, page=128)


def test_a_pool_beyond_32_bit_offsets(gpu):
    """Pages whose byte offsets pass 2^31 and 2^32."""
    d, h, page = 128, 1, 128
    rec = 40 * d * page // 32
    total = (1 << 32) // rec + 40
    c = PagedKVCache(num_layers=1, batch_size=2, num_kv_heads=h, head_dim=d, num_pages=total, max_tokens=1024,
                     page_tokens=page, device=gpu)
    far = [total - 1, (1 << 31) // rec + 1, total - 9, 5, (1 << 32) // rec, 0, (1 << 31) // rec - 1, 9]
    c.free_ring[:8] = torch.tensor(far, dtype=torch.int32, device=gpu)
    gen = torch.Generator().manual_seed(1)
    k, v = (torch.randn((2, h, 500, d), generator=gen).to(BF) for _ in range(2))
    new = torch.tensor([500, 400], dtype=torch.int32, device=gpu)
    c.begin_append(new, 500)
    c.stage_layer(0, k.to(gpu), v.to(gpu))
    c.commit_append()
    assert c.block_table[0, :4].tolist() == far[:4]
    kk, _ = c.dequantize_layer(0, 500, dtype=torch.float32)
    q = torch.randn((2, 4, 1, d), generator=gen).to(BF)
    got = c.attend(0, q.to(gpu))
    none = torch.empty((h, 0, d))
    for b, n in enumerate((500, 400)):
        want_k = stored(k[b, :, :n], "k")
        assert torch.equal(kk[b, :, :n].cpu().double(), want_k)
        want, bound = attend64(q[b], want_k, stored(v[b, :, :n], "v"), none, none, seen=torch.ones((h, n), dtype=torch.bool))
        check_attention(got[b], want, bound, BF)


# ------------------------------------------------------------------ together
def test_a_batch_decodes_as_contiguous_caches_do(gpu):
    """Prompts, then blocks and single tokens of a ragged batch over two layers, requests
    leaving and coming back: the same stored values as one contiguous cache per request, and
    the outputs of the contiguous attention over them (both within their roundings: half a
    step of the result each, and bf16 copies of K, V and P there)."""
    b, h, hq, d, layers = 3, 2, 8, 128, 2
    gen = torch.Generator().manual_seed(4)
    c = PagedKVCache(num_layers=layers, batch_size=b, num_kv_heads=h, head_dim=d, num_pages=30, max_tokens=320,
                     page_tokens=32, device=gpu)
    quant = QuantizationConfig(residual_tokens=0)
    one = lambda: PackedKVCache(num_layers=layers, batch_size=1, num_kv_heads=h, head_dim=d, max_tokens=512,  # noqa: E731
                                quant=quant, device=gpu)
    flat = [one() for _ in range(b)]
    steps = [([50, 96, 7], 96), ([32, 32, 32], 32), ([1, 1, 1], 1), ([1, 0, 1], 1), ([32, 5, 0], 32), "release",
             ([32, 32, 60], 60), ([1, 1, 1], 1)]
    for step in steps:
        if step == "release":
            c.release(torch.tensor([False, True, False], device=gpu))
            flat[1] = one()
            assert (c.block_table[1] == -1).all()
            continue
        new, t = step
        news = torch.tensor(new, dtype=torch.int32, device=gpu)
        c.begin_append(news, t)
        for i, f in enumerate(flat):
            if new[i]:
                f.begin_append(new[i])
        for layer in range(layers):
            q, k, v = (torch.randn((b, x, t, d), generator=gen).to(BF).to(gpu) for x in (hq, h, h))
            out = c.attend(layer, q, k, v)
            c.stage_layer(layer, k, v)
            for i, f in enumerate(flat):
                n = new[i]
                if n == 0:
                    continue
                want, _ = splitk_attention(q[i:i + 1, :, :n].contiguous(), Prefix.from_view(f.layer_view(layer)),
                                           k[i:i + 1, :, :n].contiguous(), v[i:i + 1, :, :n].contiguous())
                f.stage_layer(layer, k[i:i + 1, :, :n].contiguous(), v[i:i + 1, :, :n].contiguous())
                rel = float((out[i, :, :n].float() - want[0].float()).norm() / want.float().norm())
                assert rel <= 2 * 2.0 ** -8 + 3 * 2.0 ** -8, (step, layer, i, rel)
        c.commit_append()
        for i, f in enumerate(flat):
            if new[i]:
                f.commit_append()
        c.check()
        assert c.lengths.tolist() == [f.length for f in flat]
        for layer in range(layers):
            kk, vv = c.dequantize_layer(layer, 320, dtype=torch.float32)
            for i, f in enumerate(flat):
                wk, wv = f.dequantize_layer(layer, dtype=torch.float32)
                assert torch.equal(kk[i, :, :f.length], wk[0]) and torch.equal(vv[i, :, :f.length], wv[0])


def test_a_step_is_captured_and_replayed(gpu):
    """A whole step -- plan, attention, append, commit -- captured once and replayed while the
    requests grow over groups and pages; every replay against the eager calls on a twin, with
    eager work of other sizes in between."""
    b, h, d = 3, 2, 64
    gen = torch.Generator().manual_seed(9)
    caches = [PagedKVCache(num_layers=1, batch_size=b, num_kv_heads=h, head_dim=d, num_pages=24, max_tokens=256,
                           page_tokens=32, device=gpu) for _ in range(2)]
    draw = lambda heads, t: torch.randn((b, heads, t, d), generator=gen).to(BF).to(gpu)  # noqa: E731
    k0, v0 = draw(h, 40), draw(h, 40)
    first = torch.tensor([40, 25, 31], dtype=torch.int32, device=gpu)
    for c in caches:
        c.begin_append(first, 40)
        c.stage_layer(0, k0, v0)
        c.commit_append()
    q, k, v = draw(4, 1), draw(h, 1), draw(h, 1)
    new = torch.ones(b, dtype=torch.int32, device=gpu)
    out = torch.zeros((b, 4, 1, d), dtype=BF, device=gpu)

    def step(c, out):
        c.begin_append(new, 1)
        c.attend(0, q, k, v, out=out)
        c.stage_layer(0, k, v)
        c.commit_append()

    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(caches[0], out)
    twin = torch.zeros_like(out)
    for i in range(40):
        q.copy_(draw(4, 1))
        k.copy_(draw(h, 1))
        v.copy_(draw(h, 1))
        new.copy_(torch.tensor([1, i % 2, 1 if i > 3 else 0], dtype=torch.int32))
        graph.replay()
        step(caches[1], twin)
        caches[1].attend(0, draw(4, 20))          # eager work of another size
        torch.cuda.synchronize()
        assert torch.equal(out, twin), i
        assert caches[0].lengths.tolist() == caches[1].lengths.tolist()
    assert torch.equal(caches[0].block_table, caches[1].block_table)
    kk = [c.dequantize_layer(0, 100) for c in caches]
    assert torch.equal(kk[0][0], kk[1][0]) and torch.equal(kk[0][1], kk[1][1])


def test_calls_on_two_streams_do_not_meet(gpu):
    """Attention of two batches at once, on streams of their own, eager and as two graphs."""
    rs = [Requests(gpu, [3000, 40], seed=i) for i in range(2)]
    qs = [torch.randn((2, 4, 1, 128), generator=r.gen).to(BF).to(gpu) for r in rs]
    want = [r.cache.attend(0, q) for r, q in zip(rs, qs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in rs]
    outs = [torch.zeros_like(q) for q in qs]
    for _ in range(10):
        for s, r, q, o in zip(streams, rs, qs, outs):
            with torch.cuda.stream(s):
                r.cache.attend(0, q, out=o)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))
    graphs = []
    for r, q, o in zip(rs, qs, outs):
        o.zero_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r.cache.attend(0, q, out=o)
        graphs.append(g)
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_the_protocol_is_kept(gpu):
    c = PagedKVCache(num_layers=2, batch_size=2, num_kv_heads=1, head_dim=64, num_pages=6, max_tokens=128, page_tokens=32,
                     device=gpu)
    new = torch.tensor([40, 3], dtype=torch.int32, device=gpu)
    k = torch.randn((2, 1, 40, 64), device=gpu).to(BF)
    with pytest.raises(RuntimeError):
        c.stage_layer(0, k, k)
    with pytest.raises(RuntimeError):
        c.commit_append()
    ring, state = c.free_ring.tolist(), c.ring_state.tolist()
    c.begin_append(new, 40)
    with pytest.raises(RuntimeError):
        c.begin_append(new, 40)
    with pytest.raises(RuntimeError):
        c.release(torch.tensor([True, False], device=gpu))
    c.abort_append()
    assert (c.block_table == -1).all() and c.lengths.tolist() == [0, 0] and c.ring_state[1] == state[1]
    assert sorted(c.free_ring.tolist()) == sorted(ring)
    c.begin_append(new, 40)
    c.stage_layer(0, k, k)
    with pytest.raises(RuntimeError):
        c.stage_layer(0, k, k)
    with pytest.raises(RuntimeError):
        c.abort_append()
    with pytest.raises(RuntimeError):
        c.commit_append()
    with pytest.raises(ValueError):
        c.stage_layer(1, k[:, :, :39], k[:, :, :39])
    c.stage_layer(1, k, k)
    c.commit_append()
    assert c.lengths.tolist() == [40, 3]


def test_refusals_on_the_gpu(gpu):
    c = PagedKVCache(num_layers=1, batch_size=2, num_kv_heads=2, head_dim=64, num_pages=6, max_tokens=128, page_tokens=32,
                     device=gpu)
    p = c.prefixes[0]
    q = torch.zeros((2, 4, 3, 64), dtype=BF, device=gpu)
    kv = torch.zeros((2, 2, 3, 64), dtype=BF, device=gpu)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    bad = [lambda: paged_attention(q[:1], p), lambda: paged_attention(q[:, :3], p), lambda: paged_attention(q.half(), p),
           lambda: paged_attention(q, p, kv), lambda: paged_attention(q, p, kv[:, :, :2], kv[:, :, :2]),
           lambda: paged_attention(q, p, kv, kv, new_lens=i32([1])), lambda: paged_attention(q, p, causal_block=-1),
           lambda: paged_attention(q, p, new_lens=torch.zeros(2, dtype=torch.int64, device=gpu)),
           lambda: paged_attention(q, p, out=q[:, :, :2]), lambda: paged_attention(q.transpose(2, 3), p),
           lambda: append_pages(p, kv, kv, i32([1, 1]), torch.zeros((2, 2), dtype=torch.int64, device=gpu)),
           lambda: append_pages(p, kv.half(), kv.half(), i32([1, 1]), torch.zeros((2, 3), dtype=torch.int64, device=gpu)),
           lambda: dequantize_pages(p, -1), lambda: dequantize_pages(p, 3, starts=i32([0])),
           lambda: dequantize_pages(p, 3, dtype=torch.int8),
           lambda: plan_pages(c.lengths, i32([1, 1]), c.block_table, c.free_ring, c.ring_state, page_tokens=33, tokens=1),
           lambda: plan_pages(c.lengths, i32([1, 1]), c.block_table, c.free_ring, c.ring_state, page_tokens=32, tokens=-1),
           lambda: plan_pages(c.lengths, i32([1, 1]), c.block_table[:1], c.free_ring, c.ring_state, page_tokens=32, tokens=1),
           lambda: c.release(i32([1, 0])),
           lambda: PagedPrefix(c.pool[0], c.k_tail[0], c.v_tail[0], c.block_table, c.lengths.long()),
           lambda: PagedPrefix(c.pool[0], c.k_tail[0], c.v_tail[0].half(), c.block_table, c.lengths),
           lambda: PagedPrefix(c.pool[0], c.k_tail[0], c.v_tail[0], c.block_table, c.lengths,
                               mask=torch.zeros((2, 1, 64), dtype=torch.uint8, device=gpu))]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            raise AssertionError(f"call {i} was not refused")
    torch.cuda.synchronize()


# ------------------------------------------------------------------ what a server does besides
@pytest.mark.parametrize("b,t,hq", [(65, 1, 1), (300, 1, 2), (600, 3, 1), (70, 40, 1), (600, 34, 1)])
def test_attention_of_many_requests(gpu, b, t, hq):
    """More requests than lanes of a wave and than threads of a workgroup, part of them idle or
    empty, of few rows and of many."""
    rng = random.Random(b + t)
    lens = [rng.choice((0, 1, 20, 32, 33, 70)) for _ in range(b)]
    _attend(gpu, lens=lens, new=[rng.choice((0, t, t, max(1, t // 2))) for _ in lens], t=t, hq=hq, h=1, d=64, dtype=BF,
            page=32)


@pytest.mark.parametrize("b,t,hq,d,dtype", [(4, 1, 8, 64, BF), (4, 1, 16, 128, F16), (2, 8, 40, 128, BF), (2, 8, 40, 64, F16)])
def test_attention_over_a_table_of_repeated_pages(gpu, b, t, hq, d, dtype):
    """160 000 tokens of every request, the same 8 pages over and over, shared by all of them: a
    stretch of the line is longer than what a wave looks up at once.  A softmax over tokens that
    are repeated equally often is that over one of each; the longest chain of f32 additions is 32
    products of an instruction, some 80 items of a wave, its workgroup's 4 waves and fewer than 70
    partials, which the bound's 256 additions cover."""
    h, page = 8, 32
    r = Requests(gpu, [256], h=h, d=d, dtype=dtype, page=page)
    row = r.cache.block_table[0, :8].repeat(625)
    wide = torch.zeros((b, h, 32, d), dtype=dtype, device=gpu)
    p = PagedPrefix(r.cache.pool[0], wide, wide, row[None].expand(b, -1), r.i32([5000 * 32] * b))
    q = torch.randn((b, hq, t, d), generator=r.gen).to(dtype)
    got = paged_attention(q.to(gpu), p)
    none = torch.empty((h, 0, d))
    for i in range(b):
        want, bound = attend64(q[i], *r.kv64(0), none, none, seen=torch.ones((h, 256), dtype=torch.bool))
        check_attention(got[i], want, bound, dtype)
    assert torch.equal(paged_attention(q.to(gpu), p), got)      # (no atomics: the same bits)


@pytest.mark.parametrize("t,hq", [(1, 4), (40, 2)])
@pytest.mark.parametrize("tokens", [1, 5, 8, 33, 90])
def test_a_mask_shorter_than_the_requests(gpu, tokens, t, hq):
    """Positions past a mask's end are dead."""
    r = Requests(gpu, [20, 100, 77], h=2, page=32)
    q = torch.randn((3, hq, t, 128), generator=r.gen).to(BF)
    k, v = r.block([t] * 3, t)
    mask = (torch.rand((3, 2, tokens), generator=r.gen) >= 0.3).to(torch.uint8)
    got = r.cache.attend(0, q.to(gpu), k.to(gpu), v.to(gpu), mask=mask.to(gpu))
    for b, n in enumerate(r.lens):
        seen = torch.zeros((2, n), dtype=torch.bool)
        m = min(n, tokens)
        seen[:, :m] = mask[b, :, :m].bool()
        want, bound = attend64(q[b], *r.kv64(b), k[b], v[b], seen=seen)
        check_attention(got[b], want, bound, BF)


@pytest.mark.parametrize("causal", [1, 32, 250, 1000])
@pytest.mark.parametrize("t,hq", [(600, 1), (300, 2)])
def test_attention_causal_over_several_row_groups(gpu, causal, t, hq):
    """Row groups that end inside a head's positions or cross from one head into the next: what no
    row of a group sees is left out."""
    _attend(gpu, lens=[0, 45, 1000], new=[t, t - 77, t], t=t, hq=hq, h=1, d=128, dtype=BF, causal=causal)


def test_a_block_is_captured_and_replayed(gpu):
    """A captured call of many rows over growing requests, replayed with eager work between."""
    r = Requests(gpu, [50, 3, 200], h=2, d=128, room=300)
    c, t = r.cache, 40
    q = torch.randn((3, 4, t, 128), generator=r.gen).to(BF).to(gpu)
    k, v = (x.to(gpu) for x in r.block([t] * 3, t))
    out = torch.zeros_like(q)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        c.attend(0, q, k, v, causal_block=32, out=out)
    for i in range(6):
        graph.replay()
        want = c.attend(0, q, k, v, causal_block=32)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        r.append([30, i, 9 * i], 60)
        q.mul_(-0.75)


def test_read_back_far_behind_the_end_is_zero(gpu):
    r = Requests(gpu, [40, 70], d=64, page=32)
    k, v = r.cache.dequantize_layer(0, 50, starts=r.i32([(1 << 31) - 1, 69]))
    assert (k[0] == 0).all() and (v[0] == 0).all() and (k[1, :, 1:] == 0).all()
    assert torch.equal(k[1, :, 0].cpu(), r.k[1][:, 69]) and torch.equal(v[1, :, 0].cpu(), r.v[1][:, 69])


def test_sizes_past_32_bits_and_overlapping_arguments_are_refused(gpu):
    c = PagedKVCache(num_layers=1, batch_size=2, num_kv_heads=1, head_dim=64, num_pages=6, max_tokens=128, page_tokens=32,
                     device=gpu)
    q = torch.zeros((2, 2, 1, 64), dtype=BF, device=gpu)
    new = torch.ones(2, dtype=torch.int32, device=gpu)
    plan = lambda **kw: plan_pages(c.lengths, new, kw.pop("table", c.block_table), c.free_ring, c.ring_state,  # noqa: E731
                                   **{**dict(page_tokens=32, tokens=1), **kw})
    for call in (lambda: c.attend(0, q, causal_block=1 << 32), lambda: plan(page_tokens=(1 << 32) + 32),
                 lambda: plan(tokens=(1 << 32) + 1), lambda: c.dequantize_layer(0, 1 << 32), lambda: plan(ends=c.lengths),
                 lambda: plan(ends=new), lambda: plan(table=c.block_table[:1].expand(2, -1))):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: c.attend(1, q), lambda: c.attend(-1, q), lambda: c.dequantize_layer(-1, 1)):
        with pytest.raises(IndexError):
            call()
    assert c.ring_state.tolist() == [0, 6, 0, 0] and c.lengths.tolist() == [0, 0]


@pytest.mark.parametrize("t,hq", [(1, 4), (20, 8)])
def test_broadcast_queries_masks_and_tables(gpu, t, hq):
    """One tensor for all heads or requests (strides of 0) is read as its copies are, and requests
    that share their pages agree."""
    r = Requests(gpu, [150], h=2, page=32)
    c = r.cache
    rows = lambda x: x.expand(3, *x.shape[1:])  # noqa: E731
    lens = r.i32([150, 150, 150])
    q = torch.randn((1, hq, t, 128), generator=r.gen).to(BF).to(gpu)
    mask = (torch.rand((1, 1, 150), generator=r.gen) >= 0.4).to(torch.uint8).to(gpu)
    k, v = (x.to(gpu) for x in r.block([t], t))
    p = PagedPrefix(c.pool[0], rows(c.k_tail[0]), rows(c.v_tail[0]), c.block_table.expand(3, -1), lens,
                    mask=mask.expand(3, 2, -1))
    got = paged_attention(rows(q), p, rows(k), rows(v))
    copies = PagedPrefix(c.pool[0], rows(c.k_tail[0]).contiguous(), rows(c.v_tail[0]).contiguous(),
                         c.block_table.expand(3, -1).contiguous(), lens, mask=mask.expand(3, 2, -1).contiguous())
    assert torch.equal(paged_attention(rows(q).contiguous(), copies, rows(k).contiguous(), rows(v).contiguous()), got)
    seen = mask[0].expand(2, -1).bool().cpu()
    want, bound = attend64(q[0].cpu(), *r.kv64(0), k[0].cpu(), v[0].cpu(), seen=seen)
    for b in range(3):
        check_attention(got[b], want, bound, BF)
