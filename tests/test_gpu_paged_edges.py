"""The paged 4-bit cache where its rules are easily missed: masks without a position, layers that
were written but not committed, counts below zero, weights far below the largest,
values that a causal row does not see, and groups whose parameters are not ordinary numbers."""

import math

import pytest
import torch

from maskahead_amd.cache import PackedKVCache
from maskahead_amd.config import QuantizationConfig
from maskahead_amd.kernels.paged import PagedPrefix, paged_attention
from maskahead_amd.paged import PagedKVCache

from _paged import Requests, attend64, check_attention, stored

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


# ------------------------------------------------------------------ masks
@pytest.mark.parametrize("t,hq", [(1, 4), (40, 2)])
@pytest.mark.parametrize("sliced", [False, True])
def test_a_mask_without_positions_leaves_the_block_alone(gpu, t, hq, sliced):
    """Positions past a mask's end are dead: of a mask of no tokens (an empty tensor or an empty
    slice of one) every stored token is, the block's own keys are not."""
    r = Requests(gpu, [20, 100, 0], h=2, page=32)
    q = torch.randn((3, hq, t, 128), generator=r.gen).to(BF)
    k, v = r.block([t] * 3, t)
    mask = torch.ones((3, 2, 8 if sliced else 0), dtype=torch.uint8, device=gpu)[:, :, :0]
    got = r.cache.attend(0, q.to(gpu), k.to(gpu), v.to(gpu), mask=mask)
    for b, n in enumerate(r.lens):
        want, bound = attend64(q[b], *r.kv64(b), k[b], v[b], seen=torch.zeros((2, n), dtype=torch.bool))
        check_attention(got[b], want, bound, BF)
    assert (r.cache.attend(0, q.to(gpu), mask=mask, out=torch.full_like(got, 9.0)) == 0).all()


# ------------------------------------------------------------------ the step protocol
def test_a_staged_layer_is_not_read_before_the_commit(gpu):
    """Its tail is already the new one while its length is the old one."""
    r = Requests(gpu, [20, 70], layers=2, page=32)
    c = r.cache
    q = torch.randn((2, 4, 30, 128), generator=r.gen).to(BF).to(gpu)
    k, v = (x.to(gpu) for x in r.block([30, 5], 30))
    c.begin_append(r.i32([30, 5]), 30)
    want = c.attend(1, q, k, v).clone()
    c.stage_layer(0, k, v)
    for call in (lambda: c.attend(0, q, k, v), lambda: c.attend(0, q), lambda: c.dequantize_layer(0, 40),
                 lambda: c.attend(0, q, mask=torch.ones((2, 2, 9), dtype=torch.uint8, device=gpu))):
        with pytest.raises(RuntimeError, match="staged"):
            call()
    assert torch.equal(c.attend(1, q, k, v)[0], want[0])      # the other layer is as it was
    c.dequantize_layer(1, 40)
    c.stage_layer(1, k, v)
    c.commit_append()
    c.attend(0, q)
    kk, _ = c.dequantize_layer(0, 75)
    assert torch.equal(kk[1, :, 64:].cpu(), torch.cat((r.k[1][:, 64:], k[1, :, :5].cpu()), 1))


@pytest.mark.parametrize("new", [[-20, 5], [3, -1], [-40, -10]])
def test_an_append_of_fewer_than_no_tokens_is_refused(gpu, new):
    """Tokens of a packed group do not return to the tail, so only abort_append and release give
    tokens back."""
    r = Requests(gpu, [40, 10], page=32)
    c = r.cache
    before = [x.clone() for x in (c.pool, c.k_tail, c.v_tail, c.lengths, c.block_table, c.free_ring, c.ring_state[:3])]
    k, v = r.block([8, 8], 8)
    assert (c.begin_append(r.i32(new), 8) == -1).all()
    c.stage_layer(0, k.to(gpu), v.to(gpu))
    c.commit_append()
    for x, y in zip(before, (c.pool, c.k_tail, c.v_tail, c.lengths, c.block_table, c.free_ring, c.ring_state[:3])):
        x, y = (t.view(torch.int16) if t.dtype == BF else t for t in (x, y))
        assert torch.equal(x, y)
    with pytest.raises(RuntimeError, match="negative number of new tokens"):
        c.check()
    c.begin_append(r.i32([8, 8]), 8)
    c.abort_append()
    c.release(torch.tensor([True, False], device=gpu))
    c.check()
    assert c.lengths.tolist() == [0, 10]


def test_a_cache_without_heads_is_refused(gpu):
    i32 = lambda *x: torch.zeros(x, dtype=torch.int32, device=gpu)  # noqa: E731
    tail = torch.zeros((2, 0, 32, 64), dtype=BF, device=gpu)
    p = PagedPrefix(torch.zeros((4, 0, 2, 2560), dtype=torch.uint8, device=gpu), tail, tail, i32(2, 3), i32(2))
    for heads in (0, 4):
        with pytest.raises(ValueError, match="Hq"):
            paged_attention(torch.zeros((2, heads, 1, 64), dtype=BF, device=gpu), p)


# ------------------------------------------------------------------ weights
def _led(gen, h, n, d, lead, dtype, at):
    """Keys of whole numbers -8 .. 7 that every group of 32 stores exactly (each channel has both
    ends: step 1), values, and the direction u that key `at` has: a query lead * u / (7 sqrt(d)) scores
    it `lead`.  Its own value is 0."""
    k = torch.randint(-8, 8, (h, n, d), generator=gen).float()
    for g in range(n // 32):
        rows = 1 + torch.rand((h, 31, d), generator=gen).argsort(1)[:, :2] + 32 * g
        k.scatter_(1, rows[:, :1], -8.0)
        k.scatter_(1, rows[:, 1:], 7.0)
    v = torch.randn((h, n, d), generator=gen) * (1000.0 if dtype == F16 else 1.0)
    u = torch.randint(0, 2, (h, d), generator=gen).float() * 2 - 1
    if at is not None:
        k[:, at], v[:, at] = 7 * u, 0.0
    return k.to(dtype), v.to(dtype), u


@pytest.mark.parametrize("dtype,lead", [(BF, 12), (BF, 20), (BF, 29), (F16, 12), (F16, 17)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t,where", [(1, "first"), (1, "middle"), (1, "tail"), (1, "block"), (9, "first"),
                                     (40, "first"), (40, "middle"), (40, "tail"), (40, "block"), (130, "first")])
def test_a_leading_key_without_a_value_leaves_the_others_their_digits(gpu, t, where, d, dtype, lead):
    """One key takes nearly all of the weight and adds nothing (an attention sink): the result is
    that of the other keys, whose weights lie 2^-17 to 2^-42 below the largest.

    The bound.  Scores are exact up to f32's rounding of exponents below 2^7 (2^-16 of a weight, with
    the exponential's own).  A weight and a value are each rounded to f16: 2^-11 of them, or, where a
    weight is subnormal, half of f16's least step, 2^-25, at most the weight itself.  That is on a
    scale where the largest weight of the row among the item's 32 keys is at least 2^-8 (2^-17 of it);
    where the item holds the leading key, on the scale that this key or an item with smaller weights
    moved last, to 2^7 (2^-32 of the leading one: its 31 neighbours keep no digits once it leads by 22
    nats).  The sum of the weights is that of what is multiplied.  So |do| <= sum_j dp_j |v_j - o| +
    2^-11 sum_j p_j |v_j|, doubled for the higher orders, and the result's own rounding.  In the
    2-norm of a row the roundings are independent and of no sign: the result's half step, three of
    f16, and the absolute parts, which meet independent values, in quadrature (twice that)."""
    h, g, n = 2, 2, 1000 if where == "tail" else 992
    gen = torch.Generator().manual_seed(int(lead) + t + d)
    at = {"first": 0, "middle": 512, "tail": 995, "block": None}[where]
    k, v, u = _led(gen, h, n, d, lead, dtype, at)
    ck = torch.randint(-8, 8, (h, t, d), generator=gen).to(dtype)
    cv = (torch.randn((h, t, d), generator=gen) * (1000.0 if dtype == F16 else 1.0)).to(dtype)
    if where == "block":
        ck[:, 0], cv[:, 0] = (7 * u).to(dtype), 0.0
    alpha = round(lead / (7 * math.sqrt(d)) * 256) / 256
    q = alpha * u.repeat_interleave(g, 0)[:, None] + torch.round(torch.randn((h * g, t, d), generator=gen) * 4) / 64
    q = q.to(dtype)
    r = Requests(gpu, [0, 0], h=h, d=d, dtype=dtype, room=n, page=64)
    rows = lambda x: torch.stack((x, x)).to(gpu)  # noqa: E731
    r.cache.begin_append(r.i32([n, n]), n)
    r.cache.stage_layer(0, rows(k), rows(v))
    r.cache.commit_append()
    got = r.cache.attend(0, rows(q), rows(ck), rows(cv)).double().cpu()
    k64 = stored(k, "k")
    assert torch.equal(k64, k.double())
    kk = torch.cat((k64, ck.double()), 1).repeat_interleave(g, 0)
    vv = torch.cat((stored(v, "v"), cv.double()), 1).repeat_interleave(g, 0)
    p = torch.softmax(torch.matmul(q.double(), kk.transpose(1, 2)) * d ** -0.5, -1)
    want = torch.matmul(p, vv)
    # the largest weight among each key's item: 32 packed tokens, the tail, or 32 of the block's keys
    sizes = [32] * (n // 32) + [n % 32] * bool(n % 32) + [32] * (t // 32) + [t % 32] * bool(t % 32)
    top = torch.cat([x.amax(-1, keepdim=True).expand_as(x) for x in p.split(sizes, -1)], -1)
    step = 2.0 ** -11
    lead = p.argmax(-1, keepdim=True) == torch.arange(p.shape[-1])
    led = torch.cat([x.any(-1, keepdim=True).expand_as(x) for x in lead.split(sizes, -1)], -1)
    lost = torch.minimum(p, torch.where(led, 2.0 ** -32, 2.0 ** -17) * top)
    dp = (step + 2.0 ** -16) * p + lost
    bound = 2 * (torch.matmul(dp + step * p, vv.abs()) + dp.sum(-1, keepdim=True) * want.abs())
    fine = torch.finfo(dtype)
    bound += fine.eps / 2 * want.abs() + fine.smallest_normal * fine.eps
    over = ((got - want).abs() / bound).max()
    assert over <= 1, f"an element is {float(over):.2f} of its bound off"
    tiny = math.sqrt(d) * fine.smallest_normal * fine.eps / 2
    lost = torch.matmul(lost ** 2, vv.norm(dim=-1, keepdim=True) ** 2).sqrt()[..., 0]
    rel = ((got - want).norm(dim=-1) / (want.norm(dim=-1) * (fine.eps / 2 + 3 * step) + 2 * lost + tiny)).max()
    assert rel <= 1, f"a row is {float(rel):.2f} of its 2-norm's bound off"


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("t", [1, 9, 40, 130])
@pytest.mark.parametrize("offset", [-400, -90, -20, 20, 90, 400])
def test_scores_far_from_zero(gpu, offset, t, d, dtype):
    """All of a row's scores lie `offset` nats from zero (a channel that is 7 in every key): the weights
    are those without the offset.  An exponent of up to 2^10 is rounded to f32 in its product and in its
    difference to the reference: 2^-13 of a weight; otherwise as above, without a leading key."""
    h, g, n = 2, 2, 203
    gen = torch.Generator().manual_seed(t + d)
    k, v, _ = _led(gen, h, n, d, 0, dtype, None)
    ck = torch.randint(-8, 8, (h, t, d), generator=gen).to(dtype)
    cv = torch.randn((h, t, d), generator=gen).to(dtype)
    k[..., 0], ck[..., 0] = 7.0, 7.0
    if dtype == F16:
        v = v / 1000.0
    q = (torch.round(torch.randn((h * g, t, d), generator=gen) * 8) / 64).to(dtype)
    q[..., 0] = round(offset * math.sqrt(d) / 7)
    r = Requests(gpu, [0, 0], h=h, d=d, dtype=dtype, room=n, page=64)
    rows = lambda x: torch.stack((x, x)).to(gpu)  # noqa: E731
    r.cache.begin_append(r.i32([n, n]), n)
    r.cache.stage_layer(0, rows(k), rows(v))
    r.cache.commit_append()
    got = r.cache.attend(0, rows(q), rows(ck), rows(cv)).double().cpu()
    assert torch.equal(stored(k, "k"), k.double())
    kk = torch.cat((k.double(), ck.double()), 1).repeat_interleave(g, 0)
    vv = torch.cat((stored(v, "v"), cv.double()), 1).repeat_interleave(g, 0)
    p = torch.softmax(torch.matmul(q.double(), kk.transpose(1, 2)) * d ** -0.5, -1)
    want = torch.matmul(p, vv)
    step = 2.0 ** -11
    dp = (step + 2.0 ** -13) * p + 2.0 ** -17 * p.amax(-1, keepdim=True)
    bound = 2 * (torch.matmul(dp + step * p, vv.abs()) + dp.sum(-1, keepdim=True) * want.abs())
    bound += torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -24
    over = ((got - want).abs() / bound).max()
    assert over <= 1, f"an element is {float(over):.2f} of its bound off"
    rel = ((got - want).norm(dim=-1) / want.norm(dim=-1)).max()
    assert rel <= torch.finfo(dtype).eps / 2 + 3 * step + 2.0 ** -13


@pytest.mark.parametrize("t,hq,most", [(1, 4, 1.1), (1, 14, 1.1), (8, 8, 1.1), (12, 14, 1.5), (40, 8, 1.5), (130, 4, 1.5)])
@pytest.mark.parametrize("d", [64, 128])
def test_f16_results_have_f16s_digits(gpu, t, hq, most, d):
    """The error in the 2-norm, beside what rounding the exact result to f16 leaves.  Up to 32 rows keys,
    values and weights are products and sums of two f16 each, exact to 2^-18 of a weight or value:
    nothing beside the result's own rounding (a tenth is allowed).  More rows round each value
    once: as much again, independent of it, is a factor of 2^(1/2)."""
    lens = [0, 700, 333, 64]
    r = Requests(gpu, lens, h=2, d=d, dtype=F16, room=t)
    q = (1.5 * torch.randn((4, hq, t, d), generator=r.gen)).to(F16)
    k, v = r.block([t] * 4, t)
    got = r.cache.attend(0, q.to(gpu), k.to(gpu), v.to(gpu)).double().cpu()
    off = rounded = 0.0
    for b, n in enumerate(lens):
        want, _ = attend64(q[b], *r.kv64(b), k[b], v[b], seen=torch.ones((2, n), dtype=torch.bool))
        if n:
            off += float((got[b] - want).norm() ** 2)
            rounded += float((want.half().double() - want).norm() ** 2)
    assert off ** 0.5 <= most * rounded ** 0.5, (off / rounded) ** 0.5


@pytest.mark.parametrize("scale_k,scale_v", [(2e-5, 1.0), (1e-3, 1e-4), (30.0, 1000.0), (2000.0, 6000.0), (1.0, 3e-6)])
@pytest.mark.parametrize("t,hq,most", [(1, 8, 1.1), (40, 4, 1.5)])
@pytest.mark.parametrize("d", [64, 128])
def test_f16_digits_of_large_and_small_values(gpu, t, hq, most, d, scale_k, scale_v):
    """Keys and values from the subnormal ones to a range of f16's largest (beyond it the cache stores
    no numbers), the scores ordinary: as above, and half of f16's least step beside."""
    h, n = 2, 500
    gen = torch.Generator().manual_seed(d)
    k, ck = ((torch.randn((h, x, d), generator=gen) * scale_k).to(F16) for x in (n, t))
    v, cv = ((torch.randn((h, x, d), generator=gen) * scale_v).to(F16) for x in (n, t))
    q = torch.randn((hq, t, d), generator=gen).to(F16)
    r = Requests(gpu, [0], h=h, d=d, dtype=F16, room=n, page=64)
    one = lambda x: x[None].to(gpu)  # noqa: E731
    r.cache.begin_append(r.i32([n]), n)
    r.cache.stage_layer(0, one(k), one(v))
    r.cache.commit_append()
    scale = d ** -0.5 / scale_k
    got = r.cache.attend(0, one(q), one(ck), one(cv), scaling=scale)[0].double().cpu()
    want, _ = attend64(q, stored(k, "k"), stored(v, "v"), ck, cv, seen=torch.ones((h, n), dtype=torch.bool), scale=scale)
    assert torch.isfinite(got).all()
    least = math.sqrt(want.numel()) * 2.0 ** -25
    assert float((got - want).norm()) <= most * float((want.half().double() - want).norm()) + least


# ------------------------------------------------------------------ values that are not numbers
@pytest.mark.parametrize("d,dtype", [(128, BF), (64, F16), (64, BF), (128, F16)])
@pytest.mark.parametrize("t,hq,causal", [(8, 2, 4), (12, 4, 5), (70, 2, 32), (40, 8, 1), (300, 2, 100)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), float("-inf")])
def test_what_a_causal_row_does_not_see_may_be_no_number(gpu, t, hq, causal, what, d, dtype):
    """A key or value of a later causal block changes no row of an earlier one, whatever it holds;
    the rows that see it are no numbers either, and in the other channels what they are beside a
    number: fewer than 512 products summed in another order, 2^-24 of them each on both sides, may
    round to the next value of the type."""
    lens = [45, 3, 64]
    r = Requests(gpu, lens, h=2, d=d, dtype=dtype, page=32)
    q = torch.randn((3, hq, t, d), generator=r.gen).to(dtype).to(gpu)
    k, v = (x.to(gpu) for x in r.block([t, t - 1, t], t))
    new = r.i32([t, t - 1, t])
    want = r.cache.attend(0, q, k, v, new_lens=new, causal_block=causal)
    biggest = max(float(x.abs().nan_to_num().max()) for x in (v, *r.v))
    for place, part in (((t - 2, t - 3), "v"), ((t - 2,), "k"), ((t // 2, t - 2), "v")):
        kb, vb = k.clone(), v.clone()
        for j in place:
            (kb if part == "k" else vb)[:, 1, j, 3 if part == "k" else slice(0, 5)] = what
        got = r.cache.attend(0, q, kb, vb, new_lens=new, causal_block=causal)
        for b, n in enumerate([t, t - 1, t]):
            assert torch.equal(got[b, :hq // 2, :n], want[b, :hq // 2, :n])          # the other KV head's
            for i in range(n):
                sees = any((lens[b] + j) // causal <= (lens[b] + i) // causal for j in place)
                row, was = got[b, hq // 2:, i], want[b, hq // 2:, i]
                if not sees:
                    assert torch.equal(row, was), (b, i, part)
                elif part == "v":
                    assert not torch.isfinite(row[:, :5]).any(), (b, i)
                    off = (row[:, 5:].float() - was[:, 5:].float()).abs() - torch.finfo(dtype).eps * was[:, 5:].float().abs()
                    assert off.max() <= 1024 * 2.0 ** -24 * biggest, (b, i)


# ------------------------------------------------------------------ quantization
def _read_back(x, dtype):
    """Groups x [..., 32] as they are stored and read, NaN passed over (its code is 0), every operation
    rounded to dtype."""
    r = lambda y: y.to(dtype).float()  # noqa: E731
    x = x.float()
    lo = torch.where(x.isnan(), math.inf, x).amin(-1, keepdim=True)
    hi = torch.where(x.isnan(), -math.inf, x).amax(-1, keepdim=True)
    step = r(r(r(hi - lo) / 15).clamp_min(1e-8))
    code = torch.nan_to_num(r(r(x - lo) / step)).round().clamp(0, 15)
    return code * step.half().float() + lo.half().float()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("pieces", [[160], [31, 1, 70, 58]])
def test_groups_of_any_values_are_stored_as_the_packed_cache_stores_them(gpu, d, dtype, pieces):
    """Constant, zero and signed-zero groups, infinities, NaN, the type's largest and smallest
    values: the codes and parameters of the contiguous cache's quantizers, in the first group and
    in ones that a tail completes.  A signalling NaN is passed over like a quiet one (the contiguous
    cache's minimum loses numbers beside it): that group against the rule itself."""
    h, n = 2, 160
    gen = torch.Generator().manual_seed(d)
    fine = torch.finfo(dtype)
    signalling = torch.tensor([0x7F81 if dtype == BF else 0x7C01], dtype=torch.int16).view(dtype)[0]

    def special(x):      # x [..., 32] of ordinary values: one kind of group a row
        y = x.clone()
        y[0] = 1.5
        y[1] = 0.0
        y[2] = 0.0
        y[2, ..., ::3] = -0.0
        y[3, ..., 7] = float("inf")
        y[4, ..., 9] = float("-inf")
        y[5, ..., 0], y[5, ..., 31] = float("inf"), float("-inf")
        y[6, ..., 5] = float("nan")
        y[7] = float("nan")
        y[8, ..., 3], y[8, ..., 30] = fine.max, fine.min
        y[9] = fine.smallest_normal * fine.eps * torch.arange(32).to(dtype)
        y[10] = 1.0
        y[10, ..., 4] = 1.0 + fine.eps
        y[11] = float("inf")
        y[12, ..., 17] = signalling
        y[13] = 1e-4
        y[13, ..., 1] = 1e-4 + 1e-7
        return y

    k, v = (torch.randn((1, h, n, d), generator=gen).to(dtype) for _ in range(2))
    for g in (0, 32, 96):
        # keys: a group is 32 tokens of a channel; values: 32 channels of a token
        k[0, :, g:g + 32] = special(k[0, :, g:g + 32].permute(2, 0, 1).contiguous()).permute(1, 2, 0)
        x = v[0, :, g:g + 32].unflatten(-1, (d // 32, 32)).permute(1, 0, 2, 3).contiguous()
        v[0, :, g:g + 32] = special(x).permute(1, 0, 2, 3).flatten(-2)
    c = PagedKVCache(num_layers=1, batch_size=1, num_kv_heads=h, head_dim=d, num_pages=6, max_tokens=192, page_tokens=32,
                     device=gpu, compute_dtype=dtype)
    f = PackedKVCache(num_layers=1, batch_size=1, num_kv_heads=h, head_dim=d, max_tokens=192,
                      quant=QuantizationConfig(residual_tokens=0), device=gpu, compute_dtype=dtype)
    k, v = k.to(gpu), v.to(gpu)
    f.begin_append(n)
    f.stage_layer(0, k, v)
    f.commit_append()
    at = 0
    for t in pieces:
        c.begin_append(torch.tensor([t], dtype=torch.int32, device=gpu), t)
        c.stage_layer(0, k[:, :, at:at + t], v[:, :, at:at + t])
        c.commit_append()
        at += t
    got, want = c.dequantize_layer(0, n, dtype=torch.float32), f.dequantize_layer(0, dtype=torch.float32)
    for x, y, src, key in zip(got, want, (k, v), (True, False)):
        x, y = x.cpu(), y[:, :, :n].cpu()
        for g in (0, 32, 96):
            at = (0, slice(None), slice(g, g + 32), 12) if key else (0, slice(None), g + 12)
            y[at] = _read_back(src[at].cpu().unflatten(-1, (-1, 32)), dtype).flatten(-2)
        torch.testing.assert_close(x, y, rtol=0, atol=0, equal_nan=True)
