"""Positions and read sets over the paged 4-bit KV cache, as measured cases.

Four operators, each over requests whose lengths lie on the GPU:

  rotate  rotate_block: a block's queries and keys rotated at their requests' positions
  append  append_pages with a rotary table (then dequantize_pages of what it touched): keys
          rotated on the way into the pages, and the queries beside them
  select  select_blocks: the blocks of stored tokens that a run of queries should read, by a
          cheap score from the parameters that the 4-bit records hold; the scores come back too
          (a program adds them up for the eviction that comes later)
  attend  paged_attention over selected blocks, the tail and the block's own keys

The storage.  A page holds `page` tokens (a multiple of 32) of every KV head; per head, one
record of 40 D bytes for each group of 32 tokens: K codes (16 D), V codes (16 D), then f16
key scales and zeros (D each, one pair per channel) and value scales and zeros (one pair per
32 channels of a token, channel groups outermost).  A code word is 4 bytes with 8 codes,
elements 0 2 4 6 1 3 5 7 from its lowest nibble up; the words' order is that of the matrix
instruction's operands (`_k_words`, `_v_words`).  A value is code * scale + zero, and every
operation of the quantization is rounded to the type of the values.  The newest length % 32
tokens of a request stay at 16 bits in its tail.

The score of a group for a query row is the largest that q k could be for keys within the
group's channel ranges, sum of q_c zero_c + max(q_c, 0) 15 scale_c, with queries and parameters in
14 bits fixed point (`_fixed`): a whole number times a power of two, so that no order of sums
changes it, nor the blocks that it selects.
"""

import math

import torch

own = False

GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
BITS = 13             # a largest value lies in [2^13, 2^14) of its fixed point
LEAST_Q, LEAST_P = -100, -24
FLT_MAX = 3.4028234663852886e38


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the token that each of 64 requests decodes, queries and keys of one layer: latency
        dict(name="rotate_token", op="rotate", b=64, hq=28, hkv=4, d=128, t=1, lo=20, hi=32768, page=64, dtype="bf16",
             rd=128, pairs="half"),
        # a 4 096-token chunk of long prompts, before its attention
        dict(name="rotate_chunk", op="rotate", b=4, hq=32, hkv=8, d=128, t=4096, lo=9000, hi=60000, page=64, dtype="bf16",
             rd=128, pairs="half"),
        # the same decoded tokens stored on the way, one request idle: mostly the tail, now and then a group
        dict(name="append_token", op="append", b=64, hq=28, hkv=4, d=128, t=1, lo=20, hi=16000, page=64, dtype="bf16",
             rd=128, pairs="half", pad=1),
        # a finished block of 32 positions, head_dim 64, neighbouring channels paired in half of them
        dict(name="append_block", op="append", b=16, hq=16, hkv=4, d=64, t=32, lo=500, hi=9000, page=32, dtype="f16",
             rd=32, pairs="next", pad=1),
        # ragged prompts quantized into their pages (their queries were rotated for the attention)
        dict(name="append_prompts", op="append", b=8, hq=0, hkv=8, d=128, t=8192, lo=1, hi=500, page=64, dtype="bf16",
             rd=128, pairs="half", pad=1),
        # a decoding step of a ragged batch: 2 048 tokens a KV head to read
        dict(name="select_token", op="select", b=64, hq=28, hkv=4, d=128, t=1, lo=700, hi=16384, page=64, dtype="bf16",
             count=64, per=32, run=0, first=1, last=2, dead=0.0, pad=1),
        # single tokens over very long requests, blocks of 64 tokens
        dict(name="select_long", op="select", b=2, hq=32, hkv=8, d=128, t=1, lo=90000, hi=131072, page=128, dtype="bf16",
             count=64, per=64, run=0, first=1, last=1, dead=0.0, pad=0),
        # a 512-token chunk of long prompts, a read set for every 32 of its positions
        dict(name="select_chunk", op="select", b=2, hq=28, hkv=4, d=128, t=512, lo=6000, hi=16384, page=64, dtype="bf16",
             count=64, per=32, run=32, first=1, last=2, dead=0.0, pad=0),
        # attention over what select_token's step selects
        dict(name="attend_token", op="attend", b=64, hq=28, hkv=4, d=128, t=1, lo=700, hi=16384, page=64, dtype="bf16",
             count=64, per=32, run=0, dead=0.0, causal=0, pad=1),
        # 4 096 tokens a KV head of very long requests
        dict(name="attend_long", op="attend", b=2, hq=32, hkv=8, d=128, t=1, lo=90000, hi=131072, page=128, dtype="bf16",
             count=64, per=64, run=0, dead=0.0, causal=0, pad=0),
        # part of a block over caches that an eviction left with dead entries, head_dim 64, f16
        dict(name="attend_evicted", op="attend", b=6, hq=16, hkv=4, d=64, t=8, lo=500, hi=9000, page=32, dtype="f16",
             count=32, per=32, run=0, dead=0.2, causal=0, pad=1),
        # the chunk's attention: every 32 positions over their own read set, causal by blocks of 32
        dict(name="attend_chunk", op="attend", b=2, hq=28, hkv=4, d=128, t=512, lo=6000, hi=16384, page=64, dtype="bf16",
             count=64, per=32, run=32, dead=0.0, causal=32, pad=0),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, uniform over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "append", "select", "select", "attend", "attend", "attend"])
    hkv, d, dtype = rng.choice([4, 4, 8]), rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "f16"])
    g, page = rng.choice([1, 4, 7, 7, 8]), rng.choice([32, 64, 64, 128])
    case = dict(op=op, hkv=hkv, d=d, dtype=dtype, page=page)
    if op in ("rotate", "append"):
        t = rng.choice([1, 1, 8, 32, _spread(rng, 2, 4096)])
        hq = hkv * g if rng.random() < 0.75 else 0
        return dict(case, b=_spread(rng, 1, max(2, min(256, (8192 if hq else 32768) // t))), hq=hq, t=t,
                    lo=_spread(rng, 1, 64), hi=_spread(rng, 100, 32768 if op == "rotate" else 2000),
                    rd=rng.choice([d, d, d // 2, 16]), pairs=rng.choice(["half", "half", "next"]),
                    pad=rng.choice([0, 1]))
    t = rng.choice([1, 1, 1, 2, 5, 8, 16, 32, 32, _spread(rng, 33, 512)])
    hi = _spread(rng, 50, 131072 if t == 1 else 32768 if t <= 32 else 8192)
    per = rng.choice([32, 32, 64, 96, 128])
    b = min(96, max(1, 2048 // t), max(2, (500000 if t == 1 else 65536 if t <= 32 else 8192) // hi))
    case.update(b=_spread(rng, 1, b),
                hq=hkv * (g if t <= 32 else 4), t=t, lo=_spread(rng, 1, hi), hi=hi, per=per,
                count=_spread(rng, 2, max(2, 4096 // per)), run=rng.choice([0, 0, 1, 8, 32]) if t > 1 else 0,
                dead=rng.choice([0.0, 0.0, 0.0, 0.3]), pad=rng.choice([0, 1]))
    if op == "select":
        return dict(case, first=rng.choice([0, 1]), last=rng.choice([0, 1]))
    return dict(case, causal=rng.choice([0, 0, 1, 32]))


def _lengths(case):
    """The stored tokens of every request, spread over [lo, hi] (the longest is hi)."""
    b, lo, hi = case["b"], case["lo"], case["hi"]
    return [hi if i == 0 else int(round(lo * (hi / lo) ** ((i * 0.6180339887) % 1.0))) for i in range(b)]


def _new_lens(case):
    """The new tokens of every request: t, with `pad` one idle request last, and ragged where
    they are prompts."""
    b, t = case["b"], case["t"]
    n = [max(1, t - (t * 5 * i // (6 * b))) for i in range(b)] if case["op"] == "append" and t > 32 else [t] * b
    if case.get("pad") and b > 1:
        n[-1] = 0
    return n


def _up(x, unit):
    return -(-x // unit)


def _runs(case):
    """Runs of query positions that share a selection, and positions of a run."""
    run = case["run"] or case["t"]
    return _up(case["t"], run), run


# ------------------------------------------------------------------ what the storage holds
def _words(codes):
    """[..., 8] codes -> [..., 4] bytes of one code word."""
    return codes[..., [0, 4, 1, 5]] | (codes[..., [2, 6, 3, 7]] << 4)


def _unwords(b):
    """[..., 4] bytes -> [..., 8] codes."""
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)[..., [0, 4, 1, 5, 2, 6, 3, 7]]


def _k_words(codes):
    """[..., 32, D] key codes -> [..., 16 D] bytes: words of 8 channels, in the order of (half of the
    octets' tokens, quarter of the channels, octet, token of the half octet, word)."""
    d = codes.shape[-1]
    x = codes.unflatten(-1, (4, d // 32, 8)).unflatten(-4, (4, 2, 4))   # a, mt, q, h, cb, i
    lead = list(range(x.ndim - 6))
    n = len(lead)
    return _words(x.permute(*lead, n + 1, n + 3, n, n + 2, n + 4, n + 5)).flatten(-6)


def _k_codes(b, d):
    x = _unwords(b.unflatten(-1, (2, 4, 4, 4, d // 32, 4)))            # mt, h, a, q, cb, i
    lead = list(range(x.ndim - 6))
    n = len(lead)
    return x.permute(*lead, n + 2, n, n + 3, n + 1, n + 4, n + 5).flatten(-3).flatten(-4, -2)


def _v_words(codes):
    """[..., 32, D] value codes -> [..., 16 D] bytes: words of 8 tokens, in the order of (quad of a
    row's channels, octet, row of the D / 16 channels, channel of the quad)."""
    d = codes.shape[-1]
    x = codes.unflatten(-1, (16, d // 64, 4)).unflatten(-4, (4, 8))     # h, i, m, half, c
    lead = list(range(x.ndim - 5))
    n = len(lead)
    return _words(x.permute(*lead, n + 3, n, n + 2, n + 4, n + 1)).flatten(-5)


def _v_codes(b, d):
    x = _unwords(b.unflatten(-1, (d // 64, 4, 16, 4, 4)))              # half, h, m, c, i
    lead = list(range(x.ndim - 5))
    n = len(lead)
    return x.permute(*lead, n + 1, n + 4, n + 2, n, n + 3).flatten(-3).flatten(-3, -2)


def _f16_bytes(x):
    return x.to(torch.float16).contiguous().view(torch.uint8)


def _f16_values(x):
    return x.contiguous().view(torch.float16).float()


def _quantize(x, dim, dtype):
    """Codes, step and lowest value of x (f32 that holds values of dtype) over `dim`, every operation
    rounded to dtype: 32 bits hold twice a 16-bit significand and two bits, so rounding again is exact."""
    r = lambda v: v.to(dtype).float()  # noqa: E731
    lo, hi = x.amin(dim, keepdim=True), x.amax(dim, keepdim=True)
    step = r(r(r(hi - lo) / 15).clamp_min(1e-8))
    q = torch.nan_to_num(r(r(x - lo) / step)).round().clamp(0, 15)
    return q.to(torch.uint8), step, lo


def _records(k, v, dtype):
    """[..., 32, D] K and V (f32) of whole groups -> [..., 40 D] bytes."""
    d = k.shape[-1]
    kc, ks, kz = _quantize(k, -2, dtype)
    vc, vs, vz = _quantize(v.unflatten(-1, (d // 32, 32)), -1, dtype)
    turn = lambda p: _f16_bytes(p.squeeze(-1).transpose(-1, -2)).flatten(-2)  # noqa: E731
    return torch.cat((_k_words(kc), _v_words(vc.flatten(-2)), _f16_bytes(ks.squeeze(-2)), _f16_bytes(kz.squeeze(-2)),
                      turn(vs), turn(vz)), -1)


def _values(rec):
    """[..., 40 D] bytes -> K and V [..., 32, D] in 32 bits."""
    d = rec.shape[-1] // 40
    kb, vb, ks, kz, vs, vz = rec.split((16 * d, 16 * d, 2 * d, 2 * d, 2 * d, 2 * d), -1)
    wide = lambda x: _f16_values(x).unflatten(-1, (d // 32, 32)).transpose(-1, -2).repeat_interleave(32, -1)  # noqa: E731
    k = _k_codes(kb, d).float() * _f16_values(ks).unsqueeze(-2) + _f16_values(kz).unsqueeze(-2)
    v = _v_codes(vb, d).float() * wide(vs) + wide(vz)
    return k, v


# ------------------------------------------------------------------ what a program has in hand
def _rotary(positions, rd, dev):
    """cos and sin [positions, rd] of the angles position / 1e6^(2 i / rd), which are taken in 64 bits."""
    at = torch.arange(positions, dtype=torch.float64, device=dev)[:, None]
    angle = at * 1e6 ** (-torch.arange(0, rd, 2, dtype=torch.float64, device=dev) / rd)
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    b, t, page, op = case["b"], case["t"], case["page"], case["op"]
    hq, hkv, d, dt = case["hq"], case["hkv"], case["d"], DTYPES[case["dtype"]]
    lens, new = _lengths(case), _new_lens(case)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    lengths, news = i32(lens), i32(new)
    chan = torch.exp(0.5 * torch.randn((hkv, 1, d), generator=g, device=dev))
    state = dict(case=case, lengths=lengths, new=news, mask=None)
    state["k"] = (torch.randn((b, hkv, t, d), generator=g, device=dev) * chan).to(dt)
    state["v"] = torch.randn((b, hkv, t, d), generator=g, device=dev).to(dt)
    state["q"] = torch.randn((b, hq, t, d), generator=g, device=dev).to(dt) if hq else None
    grown = [x + n for x, n in zip(lens, new)]
    width = max(_up(max(lens) + t, page), 1)
    if op in ("rotate", "append"):
        state["rotary"] = _rotary(width * page, case["rd"], dev)
    # every page that the batch needs, some more, and one page that nothing names; in no order
    total = sum(_up(x, page) for x in grown) + 8
    if op == "rotate":
        total = 1
    ids = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    pages = i32([_up(x, page) for x in grown])
    at = torch.arange(width, device=dev)
    first = pages.cumsum(0) - pages
    table = torch.where(at[None] < pages[:, None], ids[(first[:, None] + at[None]).clamp_max(total - 1).long()], -1)
    state["table"] = table.to(torch.int32).contiguous()
    pool = torch.zeros((total + 1, hkv, page // GROUP, 40 * d), dtype=torch.uint8, device=dev)
    tails = torch.zeros((2, b, hkv, GROUP, d), dtype=dt, device=dev)
    for i in range(b if op != "rotate" else 0):   # request by request: the 16-bit tokens of one at a time are held
        n = lens[i]
        k = torch.randn((hkv, n, d), generator=g, device=dev) * chan
        # tokens that lie together are alike, and some passages are spoken of more than others
        k += torch.randn((hkv, _up(n, 64), d), generator=g, device=dev).repeat_interleave(64, 1)[:, :n] * chan
        v = torch.randn((hkv, n, d), generator=g, device=dev)
        k[:, :4] *= 4.0                                    # the tokens that every query attends to
        k, v = k.to(dt).float(), v.to(dt).float()
        m = n // GROUP
        if m:
            rec = _records(k[:, :m * GROUP].unflatten(1, (m, GROUP)), v[:, :m * GROUP].unflatten(1, (m, GROUP)), dt)
            w = torch.arange(m, device=dev)
            pool[state["table"][i, w * GROUP // page].long(), :, w % (page // GROUP)] = rec.transpose(0, 1)
        tails[0, i, :, :n - m * GROUP], tails[1, i, :, :n - m * GROUP] = k[:, m * GROUP:], v[:, m * GROUP:]
    state["pool"], state["k_tail"], state["v_tail"] = pool, tails[0], tails[1]
    if op == "append":
        pos = lengths[:, None] + torch.arange(t, device=dev)[None]
        slot = torch.gather(state["table"], 1, (pos // page).long()).long() * page + pos % page
        state["slots"] = torch.where(torch.arange(t, device=dev)[None] < news[:, None], slot, -1)
        state["ends"], state["starts"] = lengths + news, lengths // GROUP * GROUP
    if op in ("select", "attend") and case["dead"]:
        keep = torch.rand((b, hkv, width * page), generator=g, device=dev) >= case["dead"]
        # (and some blocks that nothing is left of)
        whole = torch.rand((b, hkv, _up(width * page, case["per"])), generator=g, device=dev) >= case["dead"] / 4
        state["mask"] = (keep & whole.repeat_interleave(case["per"], 2)[..., :width * page]).to(torch.uint8)
    if op == "attend":
        runs, _ = _runs(case)
        most = width * page // GROUP
        nb = i32([_up(x // GROUP, case["per"] // GROUP) for x in lens])[:, None, None, None]
        j = torch.arange(most, device=dev)
        u = torch.rand((b, hkv, runs, most), generator=g, device=dev)
        u = torch.where((j == 0) | (j == nb - 1), -1.0, torch.where(j < nb, u, 2.0))     # the first, the last, others
        pick = u.sort(-1).indices[..., :case["count"]]
        pick = torch.where(pick < nb, pick, most).sort(-1).values
        if pick.shape[-1] < case["count"]:
            pick = torch.nn.functional.pad(pick, (0, case["count"] - pick.shape[-1]), value=most)
        state["blocks"] = torch.where(pick < most, pick, -1).to(torch.int32)
        state["out"] = torch.zeros((b, hq, t, d), dtype=dt, device=dev)
    if own:   # the descriptors that a program keeps beside its cache
        from maskahead_amd.kernels.paged import PagedPrefix
        make = lambda n: PagedPrefix(state["pool"], state["k_tail"], state["v_tail"], state["table"], n,  # noqa: E731
                                     mask=state["mask"])
        state["prefix"] = make(lengths)
        if op == "append":
            state["after"] = make(state["ends"])
    return state


# ------------------------------------------------------------------ one pass
def _plain_rotate(state, x):
    """x [B, H, T, D] with its first rd channels rotated at the positions lengths[b] + t."""
    case, table = state["case"], state["rotary"]
    rd, t = case["rd"], case["t"]
    pos = state["lengths"][:, None] + torch.arange(t, device=x.device)[None]
    c, s = table[pos.long()][:, None].chunk(2, -1)
    f = x[..., :rd].float()
    a, b = (f[..., 0::2], f[..., 1::2]) if case["pairs"] == "next" else f.chunk(2, -1)
    a, b = a * c - b * s, b * c + a * s
    f = torch.stack((a, b), -1).flatten(-2) if case["pairs"] == "next" else torch.cat((a, b), -1)
    return torch.cat((f.to(x.dtype), x[..., rd:]), -1)


def _plain_read(state, lengths, starts, t):
    """K and V [B, H, t, D] in 32 bits of the tokens from `starts` on, zeros from `lengths` on."""
    pool, table, page = state["pool"], state["table"], state["case"]["page"]
    d, m, per = state["k_tail"].shape[3], -(-t // GROUP) + 1, state["case"]["page"] // GROUP
    g0 = starts.long() // GROUP
    grp = g0[:, None] + torch.arange(m, device=pool.device)[None]
    ids = torch.gather(table.long(), 1, (grp // per).clamp_max(table.shape[1] - 1)).clamp_min(0)
    k, v = _values(pool[ids, :, grp % per])                              # [B, m, H, 32, D]
    tail = (grp == (lengths.long() // GROUP)[:, None])[..., None, None, None]
    i = torch.arange(t, device=pool.device)[None]
    pick = (starts.long() % GROUP)[:, None] + i
    live = (starts.long()[:, None] + i < lengths[:, None])[:, None, :, None]
    out = []
    for x, end in ((k, state["k_tail"]), (v, state["v_tail"])):
        x = torch.where(tail, end.float()[:, None], x).transpose(1, 2).flatten(2, 3)
        x = torch.gather(x, 2, pick[:, None, :, None].expand(-1, x.shape[1], -1, d))
        out.append(torch.where(live, x, 0.0))
    return out


def _plain_append(state):
    case, pool, dt = state["case"], state["pool"], state["k"].dtype
    t, per = case["t"], case["page"] // GROUP
    m = (t + GROUP - 1 + GROUP - 1) // GROUP
    lengths, new = state["lengths"].long(), state["new"].long()
    r = (lengths % GROUP)[:, None]
    j = torch.arange(m * GROUP, device=pool.device)[None]
    window = []
    for tail, x in ((state["k_tail"], _plain_rotate(state, state["k"])), (state["v_tail"], state["v"])):
        h, d = x.shape[1], x.shape[3]
        both = torch.cat((tail, x), 2).float()
        at = torch.where(j < r, j, (GROUP + j - r).clamp_max(GROUP + t - 1))
        window.append(torch.gather(both, 2, at[:, None, :, None].expand(-1, h, -1, d)))
    k, v = (w.unflatten(2, (m, GROUP)) for w in window)
    rec = _records(k, v, dt).transpose(1, 2)                             # [B, m, H, 40 D]
    grp = torch.arange(m, device=pool.device)[None]
    whole = (grp + 1) * GROUP <= r + new[:, None]
    last = ((grp + 1) * GROUP - 1 - r).clamp(0, t - 1)
    base = torch.gather(state["slots"], 1, last) // GROUP
    whole = whole & (base >= 0)
    pool[torch.where(whole, base // per, pool.shape[0] - 1), :, torch.where(whole, base % per, 0)] = rec
    rest = (r + new[:, None]) // GROUP * GROUP
    i = torch.arange(GROUP, device=pool.device)[None]
    kept = (i < r + new[:, None] - rest) & (new[:, None] > 0)
    for tail, w in ((state["k_tail"], window[0]), (state["v_tail"], window[1])):
        x = torch.gather(w, 2, (rest + i).clamp_max(m * GROUP - 1)[:, None, :, None].expand_as(tail))
        tail.copy_(torch.where(kept[:, None, :, None], x.to(dt), tail))


def _pow2(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _fixed(x, top, least):
    """x as whole numbers (in 64 bits) of which `top` lies in [2^13, 2^14), and the exponents of that."""
    e = (torch.frexp(top).exponent - 1).clamp_min(least)
    return torch.nan_to_num(x.double() * _pow2(BITS - e)).round(), e


def _plain_select(state):
    case, q, table = state["case"], state["q"], state["table"]
    b, hq, hkv, d, t, page = case["b"], case["hq"], case["hkv"], case["d"], case["t"], case["page"]
    per, m, count = page // GROUP, case["per"] // GROUP, case["count"]
    runs, run = _runs(case)
    ng = state["lengths"].long() // GROUP
    nb = -(-ng // m)
    most = table.shape[1] * per // m * m + m
    grp = torch.arange(most, device=q.device)
    ids = table.long()[:, (grp // per).clamp_max(table.shape[1] - 1)].clamp_min(0)
    par = _f16_values(state["pool"][..., 32 * d:36 * d][ids, :, grp % per]).transpose(1, 2)  # [B, H, most, 2 D]
    span, zero = (15 * par[..., :d]), par[..., d:]
    top = torch.maximum(span, zero.abs()).amax(-1, keepdim=True)
    odd = ~(torch.isfinite(span) & torch.isfinite(zero)).all(-1)
    top = torch.where(odd[..., None], 0.0, top)
    (zero, f), (span, _) = _fixed(zero, top, LEAST_P), _fixed(span, top, LEAST_P)
    rows = torch.nn.functional.pad(q, (0, 0, 0, runs * run - t)).unflatten(2, (runs, run)).unflatten(1, (hkv, hq // hkv))
    rows = rows.permute(0, 1, 3, 2, 4, 5).flatten(3, 4).float()                              # [B, H, runs, G run, D]
    odd_row = ~torch.isfinite(rows).all(-1)
    fixed, e = _fixed(rows, torch.where(odd_row, 0.0, rows.abs().amax(-1))[..., None], LEAST_Q)
    both = torch.cat((fixed, fixed.clamp_min(0)), -1).flatten(2, 3)
    s = torch.matmul(both, torch.cat((zero, span), -1).transpose(2, 3).contiguous()).unflatten(2, (runs, -1))
    s = (s * _pow2(e - BITS) * _pow2(f - BITS).squeeze(-1)[:, :, None, None]).float().clamp_min(-FLT_MAX)
    s = torch.where(odd_row[..., None] | odd[:, :, None, None], math.inf, s)
    at = (torch.arange(runs, device=q.device)[:, None] * run + torch.arange(run, device=q.device)[None])
    real = (at[None] < state["new"][:, None, None]).repeat(1, 1, hq // hkv)                  # [B, runs, G run]
    s = torch.where(real[:, None, ..., None], s, -math.inf).amax(3)                          # [B, H, runs, most]
    there = (grp[None] < ng[:, None])[:, None].expand(b, hkv, most)
    if state["mask"] is not None:
        live = torch.nn.functional.pad(state["mask"], (0, max(0, most * GROUP - state["mask"].shape[2])))
        there = there & (live[..., :most * GROUP].unflatten(2, (most, GROUP)) != 0).any(-1)
    s = torch.where(there[:, :, None], s, -math.inf).unflatten(3, (most // m, m)).amax(-1).double()
    j = torch.arange(most // m, device=q.device)
    kept = ((j < case["first"]) | (j >= (nb - case["last"])[:, None]))[:, None, None]
    key = torch.where(s > -math.inf, torch.where(kept, 1e301, s.clamp_max(1e300)), -math.inf)
    if key.shape[-1] < count:
        key = torch.nn.functional.pad(key, (0, count - key.shape[-1]), value=-math.inf)
    best, at = key.sort(dim=-1, descending=True, stable=True)
    end = key.shape[-1]
    pick = torch.where(best[..., :count] > -math.inf, at[..., :count], end).sort(-1).values
    return torch.where(pick < end, pick, -1).to(torch.int32), s[..., :_up(table.shape[1] * per, m)].float()


def _plain_attend(state):
    case, q = state["case"], state["q"]
    b, hq, hkv, d, t, n = case["b"], case["hq"], case["hkv"], case["d"], case["t"], case["hi"]
    runs, run = _runs(case)
    lengths, new = state["lengths"], state["new"]
    k, v = _plain_read(state, lengths, torch.zeros_like(lengths), n)
    i, j = torch.arange(t, device=q.device), torch.arange(n, device=q.device)
    # a token is seen where its block is listed, or behind the last whole group
    most = _up(n, case["per"]) + 1
    listed = torch.zeros((b, hkv, runs, most), dtype=torch.bool, device=q.device)
    listed.scatter_(3, torch.where(state["blocks"] >= 0, state["blocks"], most - 1).long(), True)
    seen = listed[..., :-1].repeat_interleave(case["per"], 3)[..., :n]
    seen = seen | (j[None] >= (lengths // GROUP * GROUP)[:, None])[:, None, None]
    seen = seen & (j[None] < lengths[:, None])[:, None, None]            # [B, H, runs, n]
    if state["mask"] is not None:
        seen = seen & (state["mask"][:, :, None, :n] != 0)
    seen = seen[:, :, i // run]                                          # [B, H, t, n]
    block = (i[None, None] < new[:, None, None]).expand(b, t, t)         # [B, query, current key]
    if case["causal"]:
        at = (lengths[:, None] + i[None]) // case["causal"]
        block = block & (at[:, None, :] <= at[:, :, None])
    ck = torch.where((i[None] < new[:, None])[:, None, :, None], state["k"].float(), 0.0)
    cv = torch.where((i[None] < new[:, None])[:, None, :, None], state["v"].float(), 0.0)
    qf = q.float().unflatten(1, (hkv, hq // hkv)).flatten(2, 3)          # [B, H, G t, D]
    s = torch.matmul(qf, torch.cat((k, ck), 2).transpose(2, 3)) * d ** -0.5
    s = s.unflatten(2, (hq // hkv, t))
    see = torch.cat((seen, block[:, None].expand(b, hkv, t, t)), -1)[:, :, None]
    s = torch.where(see, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.flatten(2, 3), torch.cat((v, cv), 2)).unflatten(2, (hq // hkv, t))
    o = torch.where(total > 0, o / total, 0.0).flatten(1, 2)
    state["out"].copy_(torch.where((i[None] < new[:, None])[:, None, :, None], o.to(q.dtype), state["out"]))
    return state["out"]


def run(state):
    case = state["case"]
    op, t = case["op"], case["t"]
    if own:
        from maskahead_amd.kernels import paged as P
        if op == "rotate":
            return P.rotate_block(state["prefix"], state["q"] if case["hq"] else state["k"],
                                  state["k"] if case["hq"] else None, rotary=state["rotary"],
                                  interleaved=case["pairs"] == "next")
        if op == "append":
            q = P.append_pages(state["prefix"], state["k"], state["v"], state["new"], state["slots"],
                               rotary=state["rotary"], interleaved=case["pairs"] == "next", query=state["q"])
            span = (t + 2 * GROUP - 2) // GROUP * GROUP        # the groups that the new tokens touch
            return (q, *P.dequantize_pages(state["after"], span, starts=state["starts"], dtype=state["k"].dtype))
        if op == "select":
            return P.select_blocks(state["q"], state["prefix"], case["count"], new_lens=state["new"],
                                   block_tokens=case["per"], query_block=case["run"], keep_first=case["first"],
                                   keep_last=case["last"], return_scores=True)
        return P.paged_attention(state["q"], state["prefix"], state["k"], state["v"], new_lens=state["new"],
                                 causal_block=case["causal"], out=state["out"], blocks=state["blocks"],
                                 block_tokens=case["per"], query_block=case["run"])
    if op == "rotate":
        k = _plain_rotate(state, state["k"])
        return (_plain_rotate(state, state["q"]), k) if case["hq"] else (k, None)
    if op == "append":
        span = (t + 2 * GROUP - 2) // GROUP * GROUP
        q = _plain_rotate(state, state["q"]) if case["hq"] else None
        _plain_append(state)
        k, v = _plain_read(state, state["ends"], state["starts"], span)
        return q, k.to(state["k"].dtype), v.to(state["k"].dtype)
    return _plain_select(state) if op == "select" else _plain_attend(state)


# ------------------------------------------------------------------ what it cannot do without
def work(case):
    b, t, hq, h, d, op = case["b"], case["t"], case["hq"], case["hkv"], case["d"], case["op"]
    lens, new = _lengths(case), _new_lens(case)
    group, token = 40 * d * h, 4 * d * h            # bytes of a stored group, and of a 16-bit token's K and V
    if op == "rotate":
        return {"bytes": b * t * (4 * d * (hq + h) + 4 * case["rd"]), "flops": 3 * b * t * (hq + h) * case["rd"]}
    if op == "append":
        whole = [(x % GROUP + n) // GROUP for x, n in zip(lens, new)]
        kept = [(x % GROUP + n) % GROUP if n else 0 for x, n in zip(lens, new)]
        old = [x % GROUP if w else 0 for x, w in zip(lens, whole)]
        span = (t + 2 * GROUP - 2) // GROUP * GROUP
        # new tokens, their positions and replaced tails read, groups and tails written; all of it read and
        # written out; queries read and written
        return {"bytes": sum(new) * (token + 4 * case["rd"]) + sum(old) * token
                + 2 * (sum(whole) * group + sum(kept) * token) + b * span * token + 4 * d * hq * b * t,
                "flops": 12 * d * h * GROUP * sum(whole) + 3 * case["rd"] * (hq * b * t + h * sum(new))}
    live = [(x, n) for x, n in zip(lens, new) if n]
    runs, run = _runs(case)
    masks = h * sum(x for x, _ in live) if case["dead"] else 0
    if op == "select":
        groups = sum(x // GROUP for x, _ in live)
        return {"bytes": 4 * d * h * groups + masks + sum(2 * d * hq * n for _, n in live)
                + 4 * h * runs * (b * case["count"] + groups * GROUP // case["per"]),
                "flops": sum(4 * d * hq * n * (x // GROUP) for x, n in live)}
    read = lambda x: min(x // GROUP * GROUP, case["count"] * case["per"])  # noqa: E731
    keys = [read(x) + x % GROUP + (n if not case["causal"] else (n + min(n, case["causal"])) / 2) for x, n in live]
    # (what several runs of a request list is read once)
    cached = sum(min(x // GROUP, runs * read(x) // GROUP) * group + x % GROUP * token for x, _ in live)
    if case["dead"]:
        masks = h * sum(min(x, runs * read(x)) for x, _ in live)
    return {"bytes": cached + masks + 4 * b * h * runs * case["count"] + sum(n for _, n in live) * (token + 4 * d * hq),
            "flops": sum(4 * d * hq * n * x for (_, n), x in zip(live, keys))}


# ------------------------------------------------------------------ in 64 bits
def _exact_group(rec, d):
    """K and V [H, m, 32, D] in 64 bits of records [H, m, 40 D], each value looked up by its place."""
    dev = rec.device
    tok = torch.arange(GROUP, device=dev)[:, None]
    ch = torch.arange(d, device=dev)[None]
    nib = lambda e: torch.where(e % 2 == 0, e // 2, 4 + e // 2)  # noqa: E731
    quarter, per = d // 4, d // 16
    h, cb, i = ch // quarter, ch % quarter // 8, ch % 8
    row = 4 * (tok // 8) + tok % 4
    word = (((tok // 4 % 2) * 4 + h) * 16 + row) * (d // 32) + cb
    kbyte, kshift = word * 4 + nib(i) // 2, nib(i) % 2 * 4
    ct = ch % per
    word = ((ct // 4 * 4 + tok // 8) * 16 + ch // per) * 4 + ct % 4
    vbyte, vshift = 16 * d + word * 4 + nib(tok % 8) // 2, nib(tok % 8) % 2 * 4
    look = lambda at: rec[..., at.expand(GROUP, d)].long()  # noqa: E731
    ks, kz = (_exact_half(rec, at + 2 * ch.expand(GROUP, d)) for at in (32 * d, 34 * d))
    vs, vz = (_exact_half(rec, at + 2 * (ch // 32 * 32 + tok)) for at in (36 * d, 38 * d))
    return (look(kbyte) >> kshift & 15) * ks + kz, (look(vbyte) >> vshift & 15) * vs + vz


def _exact_half(rec, at):
    """The f16 numbers at the bytes `at` of records, in 64 bits."""
    two = torch.stack((rec[..., at], rec[..., at + 1]), -1)
    return two.contiguous().view(torch.float16).squeeze(-1).double()


def _exact_records(state, i, n):
    page = state["case"]["page"]
    g = torch.arange(n // GROUP, device=state["pool"].device)
    return state["pool"][state["table"][i, g * GROUP // page].long(), :, g % (page // GROUP)].transpose(0, 1)


def _exact_prefix(state, i, n):
    """K and V [H, n, D] in 64 bits of request i's first n tokens."""
    m, d = n // GROUP, state["k_tail"].shape[3]
    out = []
    for x, tail in zip(_exact_group(_exact_records(state, i, n), d), (state["k_tail"], state["v_tail"])):
        out.append(torch.cat((x.flatten(1, 2), tail[i, :, :n - m * GROUP].double()), 1))
    return out


def _exact_stored(x, dtype, dim):
    """The values that a group's x (64 bits) is stored as: quantized by the rule, each operation rounded."""
    r = lambda v: v.to(dtype).double()  # noqa: E731
    lo, hi = x.min(dim, keepdim=True).values, x.max(dim, keepdim=True).values
    step = r(torch.maximum(r(r(hi - lo) / 15.0), torch.full_like(lo, float(torch.tensor(1e-8)))))
    code = torch.nan_to_num(r(r(x - lo) / step)).round().clamp(0, 15)
    return code * step.to(torch.float16).double() + lo.to(torch.float16).double()


def _exact_rotate(state, i, x):
    """x [H, T, D] of request i turned as complex numbers, in 64 bits."""
    rd, n = state["case"]["rd"], x.shape[1]
    rows = state["rotary"].double()[int(state["lengths"][i]) + torch.arange(n, device=x.device)]
    turn = torch.complex(rows[:, :rd // 2], rows[:, rd // 2:])
    y = x.double().clone()
    even = torch.arange(rd // 2, device=x.device) * (2 if state["case"]["pairs"] == "next" else 1)
    odd = even + (1 if state["case"]["pairs"] == "next" else rd // 2)
    z = torch.complex(y[..., even], y[..., odd]) * turn
    y[..., even], y[..., odd] = z.real, z.imag
    return y


def _exact_select(case, state):
    dev, d, hkv, count = state["q"].device, case["d"], case["hkv"], case["count"]
    runs, run = _runs(case)
    g, m = case["hq"] // hkv, case["per"] // GROUP
    out = torch.full((case["b"], hkv, runs, count), -1, dtype=torch.int32, device=dev)
    scores = torch.full((case["b"], hkv, runs, _up(state["table"].shape[1] * case["page"], case["per"])), -math.inf,
                        dtype=torch.float64, device=dev)

    def whole(x, least):      # whole numbers [..., D], exponents [...]
        e = (torch.frexp(x.abs().amax(-1)).exponent - 1).clamp(min=least)
        return torch.round(x * _pow2(13 - e)[..., None]).long(), e

    for i, (x, n) in enumerate(zip(_lengths(case), _new_lens(case))):
        ng = x // GROUP
        if not n or not ng:
            continue
        rec = _exact_records(state, i, x)
        at = 2 * torch.arange(d, device=dev)
        z, span = _exact_half(rec, 34 * d + at), 15 * _exact_half(rec, 32 * d + at)
        par, f = whole(torch.cat((z, span), -1), LEAST_P)                # [H, ng, 2 D]
        nb = _up(ng, m)
        for kv in range(hkv):
            dead = None
            if state["mask"] is not None:
                dead = ~state["mask"][i, kv, :ng * GROUP].view(ng, GROUP).bool().any(1)
            for r in range(_up(n, run)):
                q, e = whole(state["q"][i, kv * g:(kv + 1) * g, r * run:min(n, (r + 1) * run)].double().flatten(0, 1), LEAST_Q)
                best = torch.full((ng,), -math.inf, dtype=torch.float64, device=dev)
                for row in range(q.shape[0]):
                    dot = (q[row] * par[kv, :, :d]).sum(-1) + (q[row].clamp_min(0) * par[kv, :, d:]).sum(-1)
                    best = torch.maximum(best, dot.double() * _pow2(e[row] + f[kv] - 26))
                if dead is not None:
                    best = best.masked_fill(dead, -math.inf)
                best = torch.nn.functional.pad(best, (0, nb * m - ng), value=-math.inf).view(nb, m).amax(1)
                scores[i, kv, r, :nb] = best
                score = best.float().tolist()           # (what is ranked is held in 32 bits)
                there = [j for j in range(nb) if score[j] > -math.inf]
                must = [j for j in there if j < case["first"] or j >= nb - case["last"]][:count]
                rest = sorted(set(there) - set(must), key=lambda j: (-score[j], j))
                took = sorted(must + rest[:count - len(must)])
                out[i, kv, r, :len(took)] = torch.tensor(took, dtype=torch.int32, device=dev)
    return out, scores


def exact(case, seed):
    lens, new, op, t = _lengths(case), _new_lens(case), case["op"], case["t"]
    if op == "select" and case["hq"] * sum(new) > 60000:
        return None           # (row by row: too long)
    state = prepare(case, seed)
    dt, hq, hkv, d = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]
    if op == "select":
        return _exact_select(case, state)
    if op in ("rotate", "append"):
        turned = [torch.stack([_exact_rotate(state, i, x[i]) for i in range(case["b"])])
                  for x in ((state["q"], state["k"]) if hq else (state["k"],))]
        if op == "rotate":
            return (turned[0], turned[1] if hq else None)
        span = (t + 2 * GROUP - 2) // GROUP * GROUP
        outs = [torch.zeros((case["b"], hkv, span, d), dtype=torch.float64, device="cuda") for _ in range(2)]
        for i, (x, n) in enumerate(zip(lens, new)):
            r = x % GROUP
            # (a key is rounded to its type when it is rotated: that is what is quantized)
            for which, (o, tail, fresh) in enumerate(zip(outs, (state["k_tail"], state["v_tail"]),
                                                         (turned[-1].to(dt), state["v"]))):
                w = torch.cat((tail[i, :, :r], fresh[i, :, :n]), 1).double()
                m = (r + n) // GROUP * GROUP
                y = w[:, :0]
                if m:
                    y = w[:, :m].unflatten(1, (m // GROUP, GROUP))
                    y = _exact_stored(y, dt, 2) if which == 0 else \
                        _exact_stored(y.unflatten(3, (d // 32, 32)), dt, 4).flatten(3)
                    y = y.flatten(1, 2)
                o[i, :, :r + n] = torch.cat((y, w[:, m:]), 1)
        return (turned[0] if hq else None, *outs)
    runs, run = _runs(case)
    out = torch.zeros((case["b"], hq, t, d), dtype=torch.float64, device="cuda")
    g = hq // hkv
    blocks = state["blocks"].tolist()
    for i, (x, n) in enumerate(zip(lens, new)):
        if not n:
            continue
        k, v = _exact_prefix(state, i, x)
        pos = x + torch.arange(n, device="cuda")
        blk = torch.ones((n, n), dtype=torch.bool, device="cuda")
        if case["causal"]:
            blk = pos[None] // case["causal"] <= pos[:, None] // case["causal"]
        for kv in range(hkv):
            keep = torch.zeros((_up(n, run), x), dtype=torch.bool, device="cuda")
            keep[:, x // GROUP * GROUP:] = True
            for r in range(keep.shape[0]):
                for j in blocks[i][kv][r]:
                    if j >= 0:
                        keep[r, j * case["per"]:min((j + 1) * case["per"], x // GROUP * GROUP)] = True
            if state["mask"] is not None:
                keep &= state["mask"][i, kv, None, :x].bool()
            see = torch.cat((keep.repeat_interleave(run, 0)[:n], blk), 1)
            kk = torch.cat((k[kv], state["k"][i, kv, :n].double()))
            vv = torch.cat((v[kv], state["v"][i, kv, :n].double()))
            for head in range(kv * g, (kv + 1) * g):
                s = state["q"][i, head, :n].double() @ kk.T / math.sqrt(d)
                out[i, head, :n] = torch.nan_to_num(torch.softmax(s.masked_fill(~see, -math.inf), -1)) @ vv
    return out
