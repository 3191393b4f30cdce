"""Shared helpers of the paged-cache tests: page plans in whole numbers, what a request's
stored tokens are read as (the oracle's quantizers and dequantization), and attention in 64
bits with the error that the kernels' roundings allow."""

from __future__ import annotations

import math

import torch

from oracle import attention as OA

G = 32


def plan_rule(lens, new, table, ring, state, page, tokens):
    """plan_pages in whole numbers: (slots, ends) and the table, ring and state changed in
    place (lists)."""
    head, count, _, status = state
    total, width = len(ring), len(table[0])
    ends = [max(0, x + n) for x, n in zip(lens, new)]
    up = lambda x: -(-x // page)  # noqa: E731
    need = sum(max(0, up(e) - up(x)) for x, e in zip(lens, ends))
    bad = (1 if need > count else 0) | (2 if any(max(up(e), up(x)) > width for x, e in zip(lens, ends)) else 0) | \
        (4 if any(n > tokens for n in new) else 0) | (8 if any(x < 0 for x in lens) else 0)
    slots = [[-1] * tokens for _ in lens]
    if bad:
        state[3] = status | bad
        return slots, list(lens)
    taken = 0
    for b, (x, e) in enumerate(zip(lens, ends)):
        for j in range(up(x), up(e)):
            table[b][j] = ring[(head + taken) % total]
            taken += 1
    given = 0
    for b, (x, e) in enumerate(zip(lens, ends)):
        for j in range(up(e), up(x)):
            ring[(head + count + given) % total] = table[b][j]
            table[b][j] = -1
            given += 1
    for b, (x, n) in enumerate(zip(lens, new)):
        for i in range(max(n, 0)):
            slots[b][i] = table[b][(x + i) // page] * page + (x + i) % page
    state[0], state[1] = (head + taken) % total, count - taken + given
    return slots, ends


def stored(x: torch.Tensor, which: str) -> torch.Tensor:
    """[H, n, D] tokens of one request as the cache reads them back, in float64: whole groups
    through the oracle's quantizer, the rest as they are."""
    m = x.shape[1] // G * G
    out = x.double().clone()
    if m:
        y = x[None, :, :m].contiguous()
        if which == "k":
            out[:, :m] = OA.dequantize_keys(*OA.quantize_keys(y))[0].double()
        else:
            out[:, :m] = OA.dequantize_values(*OA.quantize_values(y))[0].double()
    return out


def attend64(q, k, v, ck, cv, *, seen, causal=0, scale=None):
    """One request's attention in float64: q [Hq, n, D]; k, v [H, len, D]; ck, cv [H, n, D];
    seen [H, len] bool.  Returns (out, bound): bound is what the kernels' roundings may move an
    element by, by arithmetic.  With u = 2^-11 (half a step of f16, which bounds the bf16 pair
    too): a score is off by ds <= scale u sum |q||k| for packed keys (K rounded once), so p / sum
    p by a factor within exp(+-2 ds); p and v each carry one rounding: |do| <= (2 u + 2 ds + n 2^-24)
    sum p |v| + 2 ds |o| to first order (doubled for the higher ones), and the result is rounded
    once to its own type."""
    hq, n, d = q.shape
    h, length = k.shape[0], k.shape[1]
    g = hq // h
    scale = d ** -0.5 if scale is None else scale
    kk = torch.cat((k.double(), ck.double()), 1).repeat_interleave(g, 0)
    vv = torch.cat((v.double(), cv.double()), 1).repeat_interleave(g, 0)
    s = torch.matmul(q.double(), kk.transpose(1, 2)) * scale
    pos = length + torch.arange(ck.shape[1])
    blk = torch.ones((n, ck.shape[1]), dtype=torch.bool)
    if causal:
        blk = (pos[None] // causal) <= ((length + torch.arange(n))[:, None] // causal)
    see = torch.cat((seen.repeat_interleave(g, 0)[:, None].expand(hq, n, length), blk[None].expand(hq, -1, -1)), 2)
    s = s.masked_fill(~see, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1)) if s.shape[2] else s
    # keys and values that nobody sees may hold anything
    vv = torch.where(see.any(1)[..., None], vv, 0.0)
    out = torch.matmul(p, vv)
    u = 2.0 ** -11
    ds = scale * u * torch.matmul(q.double().abs(), torch.nan_to_num(kk.abs().transpose(1, 2)))
    ds = (ds.masked_fill(~see, 0.0).amax(-1, keepdim=True) if s.shape[2] else torch.zeros((hq, n, 1)))
    spread = torch.matmul(p, vv.abs())
    bound = 2 * ((2 * u + 2 * ds + s.shape[2] * 2.0 ** -24) * spread + 2 * ds * out.abs())
    return out, bound + torch.finfo(q.dtype).eps / 2 * out.abs() + 2.0 ** -24


def check_attention(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, dtype: torch.dtype) -> None:
    """Every element within its bound, and the whole within what independent roundings add up to
    in the 2-norm: half a step of the result and three of f16 (K, P, V)."""
    got, want = got.double().cpu(), want
    assert torch.isfinite(got).all()
    over = ((got - want).abs() / bound).max() if want.numel() else torch.tensor(0.0)
    assert over <= 1, f"an element is {float(over):.2f} of its bound off"
    norm = float(want.norm())
    if norm:
        rel = float((got - want).norm()) / norm
        assert rel <= torch.finfo(dtype).eps / 2 + 3 * 2.0 ** -11, f"2-norm {rel:.2e}"


class Requests:
    """Requests' tokens on the CPU and their paged cache on the GPU, filled by the cache's own
    plans and appends in the given pieces."""

    def __init__(self, dev, lens, *, h=2, d=128, dtype=torch.bfloat16, page=64, layers=1, room=64, pieces=None, seed=0,
                 pages=None):
        from maskahead_amd.paged import PagedKVCache

        self.dev, self.lens, self.h, self.d, self.dtype = dev, list(lens), h, d, dtype
        self.gen = torch.Generator().manual_seed(seed)
        width = max(self.lens) + room
        total = pages or sum(-(-(x + room) // page) for x in self.lens) + 3
        self.cache = PagedKVCache(num_layers=layers, batch_size=len(self.lens), num_kv_heads=h, head_dim=d,
                                  num_pages=total, max_tokens=width, page_tokens=page, device=dev, compute_dtype=dtype)
        # pages handed out in no order, and what was in them before
        self.cache.free_ring.copy_(torch.randperm(total, generator=self.gen).to(torch.int32))
        self.cache.pool.random_(0, 256, generator=None)
        self.cache.k_tail.fill_(float("nan"))
        self.cache.v_tail.fill_(float("nan"))
        self.k = [torch.empty((h, 0, d), dtype=dtype) for _ in self.lens]
        self.v = [torch.empty((h, 0, d), dtype=dtype) for _ in self.lens]
        left = list(self.lens)
        pieces = pieces or [max(left) or 1]
        i = 0
        while max(left) > 0:
            t = pieces[i % len(pieces)]
            new = [min(t, x) for x in left]
            self.append(new, t)
            left = [x - n for x, n in zip(left, new)]
            i += 1

    def tokens(self, n):
        x = torch.randn((self.h, n, self.d), generator=self.gen) * torch.exp(
            0.5 * torch.randn((self.h, 1, self.d), generator=self.gen))
        return x.to(self.dtype)

    def block(self, new, t):
        """k, v [B, H, t, D] of new[b] tokens each (NaN behind them)."""
        out = []
        for _ in range(2):
            x = torch.full((len(new), self.h, t, self.d), float("nan"), dtype=self.dtype)
            for b, n in enumerate(new):
                if n > 0:
                    x[b, :, :n] = self.tokens(n)
            out.append(x)
        return out

    def i32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.dev)

    def append(self, new, t):
        k, v = self.block(new, t)
        self.cache.begin_append(self.i32(new), t)
        for layer in range(self.cache.num_layers):
            self.cache.stage_layer(layer, k.to(self.dev), v.to(self.dev))
        self.cache.commit_append()
        self.note(new, k, v)

    def note(self, new, k, v):
        for b, n in enumerate(new):
            if n > 0:
                self.k[b] = torch.cat((self.k[b], k[b, :, :n]), 1)
                self.v[b] = torch.cat((self.v[b], v[b, :, :n]), 1)

    def kv64(self, b):
        return stored(self.k[b], "k"), stored(self.v[b], "v")
