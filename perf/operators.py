"""The paged 4-bit KV cache of a batch of requests, as measured cases.

Four operators, each over requests whose lengths lie on the GPU:

  pages   plan_pages: block tables, slot maps and the ring of free pages, from the lengths
  append  append_pages (then dequantize_pages of what it touched): new tokens into pages
  read    dequantize_pages: a range of every request's tokens at 16 bits
  attend  paged_attention: a block of queries over [pages | tail | current block]

The storage.  A page holds `page` tokens (a multiple of 32) of every KV head; per head, one
record of 40 D bytes for each group of 32 tokens: K codes (16 D), V codes (16 D), then f16
key scales and zeros (D each, one pair per channel) and value scales and zeros (one pair per
32 channels of a token, channel groups outermost).  A code word is 4 bytes with 8 codes,
elements 0 2 4 6 1 3 5 7 from its lowest nibble up.  K words run over 8 channels of a token,
V words over 8 tokens of a channel; their order is that of the matrix instruction's operands
(`_k_words`, `_v_words`).  A value is code * scale + zero.  The newest length % 32 tokens of a
request stay at 16 bits in its tail.

Quantization is the rule of the framework's other 4-bit caches: every operation rounded to the
type of the values, which is part of what is stored and so of the plain form.
"""

import math

import torch

own = False

GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # a decoding step of a full batch: one token each, a few requests need a page; taken back
        # as when the step is given up, all latency
        dict(name="pages_decode", op="pages", b=64, t=1, lo=20, hi=32768, page=64, pad=1),
        # prompts of up to 2 048 tokens admitted at once
        dict(name="pages_prompts", op="pages", b=256, t=2048, lo=1, hi=4096, page=32, pad=0),
        # the token that each of 64 requests decoded, one layer: mostly the tail, now and then a group
        dict(name="append_decode", op="append", b=64, hkv=4, d=128, t=1, lo=20, hi=16000, page=64, dtype="bf16", pad=1),
        # ragged prompts quantized into their pages
        dict(name="append_prompts", op="append", b=8, hkv=8, d=128, t=8192, lo=0, hi=500, page=64, dtype="bf16", pad=1),
        # the newest part of short requests read back at 16 bits, head_dim 64
        dict(name="read_recent", op="read", b=16, hkv=4, d=64, t=256, lo=40, hi=3000, page=32, dtype="f16"),
        # a long request's whole prefix read back, as before a step that needs it at 16 bits
        dict(name="read_prefix", op="read", b=2, hkv=8, d=128, t=65536, lo=50000, hi=65536, page=128, dtype="bf16"),
        # the first tokens after short prompts: latency
        dict(name="attend_first_tokens", op="attend", b=8, hq=32, hkv=8, d=128, t=1, lo=3, hi=700, page=64,
             dtype="bf16", dead=0.0, causal=0, pad=1),
        # a decoding step of a ragged batch, the ordinary case of a server
        dict(name="attend_decode", op="attend", b=64, hq=28, hkv=4, d=128, t=1, lo=700, hi=16384, page=64,
             dtype="bf16", dead=0.0, causal=0, pad=1),
        # single tokens over very long requests: few rows, one long axis
        dict(name="attend_decode_long", op="attend", b=2, hq=32, hkv=8, d=128, t=1, lo=90000, hi=131072, page=128,
             dtype="bf16", dead=0.0, causal=0, pad=0),
        # a block-diffusion step: 32 positions that see each other
        dict(name="attend_block", op="attend", b=8, hq=28, hkv=4, d=128, t=32, lo=2000, hi=16384, page=64,
             dtype="bf16", dead=0.0, causal=0, pad=0),
        # part of a block over caches that an eviction left with dead entries, head_dim 64, f16
        dict(name="attend_evicted", op="attend", b=6, hq=16, hkv=4, d=64, t=8, lo=500, hi=9000, page=32, dtype="f16",
             dead=0.2, causal=0, pad=1),
        # a 512-token chunk of a long prompt, causal by blocks of 32
        dict(name="attend_chunk", op="attend", b=2, hq=28, hkv=4, d=128, t=512, lo=6000, hi=16384, page=64,
             dtype="bf16", dead=0.0, causal=32, pad=0),
    ]


def _spread(rng, lo, hi):
    """A size between lo and hi, uniform over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["pages", "append", "append", "read", "attend", "attend", "attend", "attend"])
    page, pad = rng.choice([32, 64, 64, 128]), rng.choice([0, 1])
    if op == "pages":
        t = _spread(rng, 1, 2048)
        return dict(op=op, b=_spread(rng, 1, min(2048, 500000 // t)), t=t, lo=_spread(rng, 1, 50),
                    hi=_spread(rng, 100, 32768), page=page, pad=pad)
    hkv, d, dtype = rng.choice([4, 4, 8]), rng.choice([128, 128, 64]), rng.choice(["bf16", "bf16", "f16"])
    if op == "append":
        t = rng.choice([1, 1, 8, 32, _spread(rng, 2, 8192)])
        return dict(op=op, b=_spread(rng, 1, max(2, min(256, 65536 // t))), hkv=hkv, d=d, t=t, lo=_spread(rng, 1, 64),
                    hi=_spread(rng, 100, 2000), page=page, dtype=dtype, pad=pad)
    if op == "read":
        t = _spread(rng, 1, 65536)
        return dict(op=op, b=_spread(rng, 1, max(2, min(64, 131072 // t))), hkv=hkv, d=d, t=t, lo=_spread(rng, 1, t),
                    hi=_spread(rng, t, 2 * t) + 1, page=page, dtype=dtype)
    t = rng.choice([1, 1, 1, 2, 5, 8, 16, 32, 32, _spread(rng, 33, 512)])
    hi = _spread(rng, 50, 131072 if t == 1 else 32768 if t <= 32 else 8192)
    b = _spread(rng, 1, max(2, min(96, (500000 if t == 1 else 65536 if t <= 32 else 8192) // hi)))
    return dict(op=op, b=b, hq=hkv * rng.choice([1, 4, 7, 7, 8]) if t <= 32 else hkv * 4, hkv=hkv, d=d, t=t,
                lo=_spread(rng, 1, hi), hi=hi, page=page, dtype=dtype, dead=rng.choice([0.0, 0.0, 0.0, 0.3]),
                causal=rng.choice([0, 0, 1, 32]), pad=pad)


def _lengths(case):
    """The stored tokens of every request, spread over [lo, hi] (the longest is hi)."""
    b, lo, hi = case["b"], case["lo"], case["hi"]
    if lo < 1:
        return [lo + (hi - lo) * ((7 * i + 3) % b) // max(1, b - 1) if b > 1 else hi for i in range(b)]
    return [hi if i == 0 else int(round(lo * (hi / lo) ** ((i * 0.6180339887) % 1.0))) for i in range(b)]


def _new_lens(case):
    """The new tokens of every request: t, with `pad` one idle request last, and ragged where
    they are prompts."""
    b, t = case["b"], case["t"]
    if case["op"] in ("pages", "append") and t > 32:
        n = [max(1, t - (t * 5 * i // (6 * b))) for i in range(b)]
    else:
        n = [t] * b
    if case.get("pad") and b > 1:
        n[-1] = 0
    return n


def _pages(x, page):
    return -(-x // page)


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
    f = lambda x: x.contiguous().view(torch.float16).float()  # noqa: E731
    wide = lambda x: f(x).unflatten(-1, (d // 32, 32)).transpose(-1, -2).repeat_interleave(32, -1)  # noqa: E731
    k = _k_codes(kb, d).float() * f(ks).unsqueeze(-2) + f(kz).unsqueeze(-2)
    v = _v_codes(vb, d).float() * wide(vs) + wide(vz)
    return k, v


# ------------------------------------------------------------------ what a program has in hand
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    b, t, page = case["b"], case["t"], case["page"]
    lens, new = _lengths(case), _new_lens(case)
    grown = [x + n for x, n in zip(lens, new)]
    width = max(_pages(max(lens) + max(t, 1), page), 1)
    used = [_pages(x, page) for x in lens]
    # every page that the batch could need, some more, and one page that nothing names
    total = sum(_pages(x, page) for x in grown) + 8
    ids = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    lengths, news = i32(lens), i32(new)
    at = torch.arange(width, device=dev)
    first = torch.cat((i32([0]), i32(used).cumsum(0)[:-1]))
    mine = at[None] < i32(used)[:, None]
    table = torch.where(mine, ids[(first[:, None] + at[None]).clamp_max(total - 1).long()], -1).to(torch.int32)
    if case["op"] == "pages":
        # the free pages, oldest first, from the middle of the ring on
        free, head = total - sum(used), total // 2
        ring = torch.full((total,), -1, dtype=torch.int32, device=dev)
        ring[(head + torch.arange(free, device=dev)) % total] = ids[sum(used):]
        return dict(case=case, lengths=lengths, new=news, undo=-news, table=table, ring=ring,
                    ring_state=i32([head, free, 0, 0]))
    hkv, d, dt = case["hkv"], case["d"], DTYPES[case["dtype"]]
    pool = torch.zeros((total + 1, hkv, page // GROUP, 40 * d), dtype=torch.uint8, device=dev)
    chan = torch.exp(0.5 * torch.randn((hkv, 1, d), generator=g, device=dev))
    tails = []
    for i in range(b):   # request by request, so that the 16-bit tokens of one at a time are held
        n = lens[i]
        k = torch.randn((hkv, n, d), generator=g, device=dev) * chan
        v = torch.randn((hkv, n, d), generator=g, device=dev)
        k[:, :4] *= 4.0                                    # the tokens that every query attends to
        k, v = k.to(dt).float(), v.to(dt).float()
        m = n // GROUP
        if m:
            rec = _records(k[:, :m * GROUP].unflatten(1, (m, GROUP)), v[:, :m * GROUP].unflatten(1, (m, GROUP)), dt)
            w = torch.arange(m, device=dev)
            pool[table[i, w * GROUP // page].long(), :, w % (page // GROUP)] = rec.transpose(0, 1)
        tail = torch.zeros((2, hkv, GROUP, d), dtype=dt, device=dev)
        tail[0, :, :n - m * GROUP], tail[1, :, :n - m * GROUP] = k[:, m * GROUP:], v[:, m * GROUP:]
        tails.append(tail)
    tails = torch.stack(tails)
    state = dict(case=case, lengths=lengths, new=news, table=table, pool=pool, k_tail=tails[:, 0].contiguous(),
                 v_tail=tails[:, 1].contiguous(), mask=None)
    if case["op"] == "read":
        state["starts"] = (lengths - t).clamp_min(0)
    else:
        state["k"] = (torch.randn((b, hkv, t, d), generator=g, device=dev) * chan).to(dt)
        state["v"] = torch.randn((b, hkv, t, d), generator=g, device=dev).to(dt)
    if case["op"] == "append":
        gone = i32([_pages(x, page) for x in lens]).cumsum(0)[-1]
        more = [_pages(x, page) - u for x, u in zip(grown, used)]
        last = torch.cat((i32([0]), i32(more).cumsum(0)[:-1])) + gone - i32(used)
        fresh = (at[None] >= i32(used)[:, None]) & (at[None] < i32(used)[:, None] + i32(more)[:, None])
        table = torch.where(fresh, ids[(last[:, None] + at[None]).clamp(0, total - 1).long()], table).to(torch.int32)
        pos = lengths[:, None] + torch.arange(t, device=dev)[None]
        slot = torch.gather(table, 1, (pos // page).long()).long() * page + pos % page
        state["slots"] = torch.where(torch.arange(t, device=dev)[None] < news[:, None], slot, -1)
        state["table"], state["ends"], state["starts"] = table, lengths + news, lengths // GROUP * GROUP
    if case["op"] == "attend":
        state["q"] = torch.randn((b, case["hq"], t, d), generator=g, device=dev).to(dt)
        state["out"] = torch.zeros((b, case["hq"], t, d), dtype=dt, device=dev)
        if case["dead"]:
            state["mask"] = (torch.rand((b, hkv, width * page), generator=g, device=dev) >= case["dead"]).to(torch.uint8)
    if own:   # the descriptors that a program keeps beside its cache
        from maskahead_amd.kernels.paged import PagedPrefix
        make = lambda n: PagedPrefix(state["pool"], state["k_tail"], state["v_tail"], state["table"], n,  # noqa: E731
                                     mask=state["mask"])
        state["prefix"] = make(lengths)
        if case["op"] == "append":
            state["after"] = make(state["ends"])
    return state


# ------------------------------------------------------------------ one pass
def _plain_plan(state, lengths, new, t):
    """One plan in elementary operations on whole numbers; tables, ring and state change in place."""
    table, ring, rs, page = state["table"], state["ring"], state["ring_state"], state["case"]["page"]
    total, width = ring.numel(), table.shape[1]
    old = lengths.long()
    ends = (old + new).clamp_min(0)
    p0, p1 = (old + page - 1) // page, (ends + page - 1) // page
    grow, back = (p1 - p0).clamp_min(0), (p0 - p1).clamp_min(0)
    taken, given = grow.cumsum(0), back.cumsum(0)
    head, count = rs[0].long(), rs[1].long()
    refused = (taken[-1] > count).long() | ((p1 > width).any().long() << 1)
    ok = refused == 0
    at = torch.arange(width, device=table.device)[None]
    there = table.long()
    # the pages that go back, to the ring's end (one place behind it takes what is not given)
    gone = (at >= p1[:, None]) & (at < p0[:, None]) & ok
    to = (head + count + (given - back)[:, None] + at - p1[:, None]) % total
    longer = torch.cat((ring, ring[:1]))
    longer.scatter_(0, torch.where(gone, to, total).flatten(), table.flatten())
    come = (at >= p0[:, None]) & (at < p1[:, None]) & ok
    ids = ring.long()[(head + (taken - grow)[:, None] + at - p0[:, None]) % total]
    there = torch.where(come, ids, torch.where(gone, -1, there))
    table.copy_(there)
    ring.copy_(longer[:total])
    i = torch.arange(t, device=table.device)[None]
    pos = old[:, None] + i
    slots = torch.gather(there, 1, (pos // page).clamp_max(width - 1)) * page + pos % page
    slots = torch.where((i < new[:, None]) & ok, slots, -1)
    moved = torch.stack(((head + taken[-1]) % total, count - taken[-1] + given[-1], rs[2].long(), rs[3].long()))
    rs.copy_(torch.where(ok, moved, torch.stack((head, count, rs[2].long(), rs[3].long() | refused))))
    return slots, torch.where(ok, ends, old).to(torch.int32)


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
    for tail, x in ((state["k_tail"], state["k"]), (state["v_tail"], state["v"])):
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


def _plain_attend(state):
    case, q, t = state["case"], state["q"], state["case"]["t"]
    b, hq, hkv, d = case["b"], case["hq"], case["hkv"], case["d"]
    n = case["hi"]
    lengths, new = state["lengths"], state["new"]
    k, v = _plain_read(state, lengths, torch.zeros_like(lengths), n)
    i, j = torch.arange(t, device=q.device), torch.arange(n, device=q.device)
    seen = (j[None] < lengths[:, None])[:, None, None, None]             # [B, 1, 1, 1, n]
    if state["mask"] is not None:
        seen = seen & (state["mask"][:, :, None, None, :n] != 0)
    block = (i[None, None] < new[:, None, None]).expand(b, t, t)         # [B, query, current key]
    if case["causal"]:
        at = (lengths[:, None] + i[None]) // case["causal"]
        block = block & (at[:, None, :] <= at[:, :, None])
    ck = torch.where((i[None] < new[:, None])[:, None, :, None], state["k"].float(), 0.0)
    cv = torch.where((i[None] < new[:, None])[:, None, :, None], state["v"].float(), 0.0)
    qf = q.float().unflatten(1, (hkv, hq // hkv)).flatten(2, 3)          # [B, H, G t, D]
    s = torch.matmul(qf, torch.cat((k, ck), 2).transpose(2, 3)) * d ** -0.5
    s = s.unflatten(2, (hq // hkv, t))
    see = torch.cat((seen.expand(b, hkv, hq // hkv, t, n), block[:, None, None].expand(b, hkv, hq // hkv, t, t)), -1)
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
    if op == "pages":
        plan = (lambda n, x: P.plan_pages(n, x, state["table"], state["ring"], state["ring_state"],  # noqa: E731
                                          page_tokens=case["page"], tokens=t)) if own else \
            (lambda n, x: _plain_plan(state, n, x, t))
        slots, ends = plan(state["lengths"], state["new"])
        _, back = plan(ends, state["undo"])                # the step is given up: its pages go back
        return slots, ends, back, state["table"], state["ring"], state["ring_state"]
    if op == "append":
        span = (t + 2 * GROUP - 2) // GROUP * GROUP        # the groups that the new tokens touch
        if own:
            P.append_pages(state["prefix"], state["k"], state["v"], state["new"], state["slots"])
            return P.dequantize_pages(state["after"], span, starts=state["starts"], dtype=state["k"].dtype)
        _plain_append(state)
        k, v = _plain_read(state, state["ends"], state["starts"], span)
        return k.to(state["k"].dtype), v.to(state["k"].dtype)
    if op == "read":
        dt = state["k_tail"].dtype
        if own:
            return P.dequantize_pages(state["prefix"], t, starts=state["starts"], dtype=dt)
        k, v = _plain_read(state, state["lengths"], state["starts"], t)
        return k.to(dt), v.to(dt)
    if own:
        return P.paged_attention(state["q"], state["prefix"], state["k"], state["v"], new_lens=state["new"],
                                 causal_block=case["causal"], out=state["out"])
    return _plain_attend(state)


# ------------------------------------------------------------------ what it cannot do without
def work(case):
    b, t, page = case["b"], case["t"], case["page"]
    lens, new = _lengths(case), _new_lens(case)
    if case["op"] == "pages":
        more = sum(_pages(x + n, page) - _pages(x, page) for x, n in zip(lens, new))
        # lengths and counts read, ends and slots written; a page moves from ring to table and back
        return {"bytes": 2 * (12 * b + 8 * b * t) + 4 * 4 * more, "flops": 0}
    h, d = case["hkv"], case["d"]
    group, token = 40 * d * h, 4 * d * h            # bytes of a stored group, and of a 16-bit token's K and V
    if case["op"] == "read":
        live = [min(x, t) for x in lens]
        packed = [max(0, x // GROUP * GROUP - max(0, x - t)) for x in lens]
        return {"bytes": sum(p * group / GROUP + (n - p) * token for p, n in zip(packed, live)) + b * t * token,
                "flops": 4 * d * h * sum(packed)}
    if case["op"] == "append":
        whole = [(x % GROUP + n) // GROUP for x, n in zip(lens, new)]
        kept = [(x % GROUP + n) % GROUP if n else 0 for x, n in zip(lens, new)]
        old = [x % GROUP if w else 0 for x, w in zip(lens, whole)]
        span = (t + 2 * GROUP - 2) // GROUP * GROUP
        # new tokens and replaced tails read, groups and tails written; then all of it read and written out
        return {"bytes": sum(new) * token + sum(old) * token + 2 * (sum(whole) * group + sum(kept) * token)
                + b * span * token, "flops": 12 * d * h * GROUP * sum(whole)}
    hq = case["hq"]
    live = [(x, n) for x, n in zip(lens, new) if n]
    keys = [x + (n if not case["causal"] else (n + min(n, case["causal"])) / 2) for x, n in live]
    cached = sum(x // GROUP * group + x % GROUP * token for x, _ in live)
    if case["dead"]:
        cached += h * sum(x for x, _ in live)
    return {"bytes": cached + sum(n for _, n in live) * (token + 4 * d * hq),
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

    def par(first, index):
        at = first + 2 * index
        two = torch.stack((rec[..., at], rec[..., at + 1]), -1)
        return two.contiguous().view(torch.float16).squeeze(-1).double()

    ks, kz = par(32 * d, ch.expand(GROUP, d)), par(34 * d, ch.expand(GROUP, d))
    vs, vz = par(36 * d, ch // 32 * 32 + tok), par(38 * d, ch // 32 * 32 + tok)
    return (look(kbyte) >> kshift & 15) * ks + kz, (look(vbyte) >> vshift & 15) * vs + vz


def _exact_prefix(state, i, n):
    """K and V [H, n, D] in 64 bits of request i's first n tokens."""
    page, d = state["case"]["page"], state["k_tail"].shape[3]
    m = n // GROUP
    g = torch.arange(m, device=state["pool"].device)
    rec = state["pool"][state["table"][i, g * GROUP // page].long(), :, g % (page // GROUP)].transpose(0, 1)
    out = []
    for x, tail in zip(_exact_group(rec, d), (state["k_tail"], state["v_tail"])):
        out.append(torch.cat((x.flatten(1, 2), tail[i, :, :n - m * GROUP].double()), 1))
    return out


def _exact_stored(x, dtype, dim):
    """The values that a group's x (64 bits) is stored as: quantized by the rule, each operation rounded."""
    r = lambda v: v.to(dtype).double()  # noqa: E731
    lo, hi = x.min(dim, keepdim=True).values, x.max(dim, keepdim=True).values
    step = r(torch.maximum(r(r(hi - lo) / 15.0), torch.full_like(lo, float(torch.tensor(1e-8)))))
    code = torch.nan_to_num(r(r(x - lo) / step)).round().clamp(0, 15)
    return code * step.to(torch.float16).double() + lo.to(torch.float16).double()


def _exact_pages(case, state):
    page, t = case["page"], case["t"]
    table, ring = state["table"].tolist(), state["ring"].tolist()
    head, count, ticket, status = state["ring_state"].tolist()
    total = len(ring)
    lens, new = state["lengths"].tolist(), state["new"].tolist()
    slots = [[-1] * t for _ in lens]
    gone = []
    for b, (x, n) in enumerate(zip(lens, new)):
        for i in range(n):
            at, off = divmod(x + i, page)
            if off == 0:
                table[b][at] = ring[head]
                head, count = (head + 1) % total, count - 1
                gone.append((b, at))
            slots[b][i] = table[b][at] * page + off
    for b, at in gone:
        ring[(head + count) % total] = table[b][at]
        table[b][at] = -1
        count += 1
    dev = state["table"].device
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    return (torch.tensor(slots, dtype=torch.int64, device=dev), i32([x + n for x, n in zip(lens, new)]), i32(lens),
            i32(table), i32(ring), i32([head, count, ticket, status]))


def exact(case, seed):
    state = prepare(case, seed)
    op, t = case["op"], case["t"]
    if op == "pages":
        return _exact_pages(case, state)
    dt, lens, new = DTYPES[case["dtype"]], _lengths(case), _new_lens(case)
    if op in ("append", "read"):
        span = (t + 2 * GROUP - 2) // GROUP * GROUP if op == "append" else t
        outs = [torch.zeros((case["b"], case["hkv"], span, case["d"]), dtype=torch.float64, device="cuda")
                for _ in range(2)]
        for i, (x, n) in enumerate(zip(lens, new)):
            if op == "read":
                first = max(0, x - t)
                for o, y in zip(outs, _exact_prefix(state, i, x)):
                    o[i, :, :x - first] = y[:, first:]
                continue
            r = x % GROUP
            for which, (o, tail, fresh) in enumerate(zip(outs, (state["k_tail"], state["v_tail"]),
                                                         (state["k"], state["v"]))):
                w = torch.cat((tail[i, :, :r], fresh[i, :, :n]), 1).double()
                m = (r + n) // GROUP * GROUP
                y = w[:, :m].unflatten(1, (m // GROUP, GROUP)) if m else w[:, :0]
                if m:
                    y = _exact_stored(y, dt, 2) if which == 0 else \
                        _exact_stored(y.unflatten(3, (case["d"] // 32, 32)), dt, 4).flatten(3)
                    y = y.flatten(1, 2)
                o[i, :, :r + n] = torch.cat((y, w[:, m:]), 1)
        return tuple(outs)
    out = torch.zeros((case["b"], case["hq"], t, case["d"]), dtype=torch.float64, device="cuda")
    g = case["hq"] // case["hkv"]
    for i, (x, n) in enumerate(zip(lens, new)):
        if not n:
            continue
        k, v = _exact_prefix(state, i, x)
        keep = torch.ones((case["hkv"], 1, x), dtype=torch.bool, device="cuda")
        if state["mask"] is not None:
            keep = state["mask"][i, :, None, :x].bool()
        pos = x + torch.arange(n, device="cuda")
        blk = torch.ones((n, n), dtype=torch.bool, device="cuda")
        if case["causal"]:
            blk = pos[None] // case["causal"] <= pos[:, None] // case["causal"]
        for head in range(case["hq"]):
            kv = head // g
            kk = torch.cat((k[kv], state["k"][i, kv, :n].double()))
            vv = torch.cat((v[kv], state["v"][i, kv, :n].double()))
            s = state["q"][i, head, :n].double() @ kk.T / math.sqrt(case["d"])
            s = s.masked_fill(~torch.cat((keep[kv].expand(n, x), blk), 1), -math.inf)
            out[i, head, :n] = torch.nan_to_num(torch.softmax(s, -1)) @ vv
    return out
