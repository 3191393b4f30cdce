"""Pages of 4-bit K/V: one cache for a batch of requests whose lengths lie on the GPU.

    slots, ends = plan_pages(lengths, new_lens, table, ring, ring_state, page_tokens=64, tokens=T)
    out = paged_attention(q, prefix, k, v, new_lens=new_lens)          # per layer
    append_pages(prefix, k, v, new_lens, slots)                        # per layer

``rotate_block`` (and ``append_pages`` on the way) turns queries and keys at their requests'
positions, ``select_blocks`` lists the blocks of stored tokens that a run of queries should read, and
``paged_attention(blocks=...)`` reads those alone:

    q, k = rotate_block(prefix, q, k, rotary=table)                    # rotary_table, made once
    blocks = select_blocks(q, prefix, 64, new_lens=new_lens)
    out = paged_attention(q, prefix, k, v, new_lens=new_lens, blocks=blocks)

The reference's cache holds one scalar length for all its batch rows (cache.py:94-96), and
``splitk_attention`` follows it; here every request has its own, read by the kernels, so a
step of a ragged batch needs no padding, no host copy of a length and one launch per layer
and operator.  The codes, scales and zeros are those of the framework's other quantizers
(``quantize_key_groups_into``, ``quantize_values_into``), bit for bit (but beside a signalling
NaN, which is passed over like any other here); they are stored in
records of 32 tokens of one KV head in the order in which the matrix instructions read them
(``csrc/ma_pages.h``).  ``maskahead_amd.paged.PagedKVCache`` keeps the planes of every layer
and the step protocol; these functions are its kernels.

All calls run on the current stream of their tensors' device and return without waiting.
"""

from __future__ import annotations

import struct

import torch

from .. import _native as N

GROUP = 32   # tokens of a record


def record_bytes(head_dim: int) -> int:
    """Bytes of one record: 32 tokens of one KV head, K and V (codes, scales, zeros)."""
    return 40 * int(head_dim)


def _i32(t: torch.Tensor, name: str, shape: tuple, index: int) -> None:
    """A contiguous int32 tensor of this shape on GPU `index` (checked together; what is wrong
    is looked for only when something is)."""
    if t.is_cuda and t.dtype is torch.int32 and t.shape == shape and t.is_contiguous() and t.get_device() == index:
        return
    N.require_gpu(t, name)
    if t.dtype != torch.int32 or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 tensor of shape {shape}, got {t.dtype} {tuple(t.shape)}")
    raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")


def _check_table(t: torch.Tensor, b: int) -> None:
    if t.ndim != 2 or t.dtype is not torch.int32 or t.shape[0] != b or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"block_table must be an int32 [{b}, width] tensor with contiguous rows")


def _c_int(name: str, value: int) -> int:
    """A size that the C entry points take as 32 bits."""
    value = int(value)
    if not 0 <= value < 1 << 31:
        raise ValueError(f"{name} must lie in 0 .. 2^31 - 1, got {value}")
    return value


def _same_device(index: int, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")


def _call(index: int, name: str, *args) -> None:
    """Entry point `name` on GPU `index`'s current stream, which is its last argument."""
    fn = getattr(N.load(), name)
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        N.check(rc, name)


class PagedPrefix:
    """What the kernels read of one layer's pages (a descriptor over the caller's tensors).

    pool      uint8 [pages, Hkv, page_tokens / 32, 40 D], each head's records contiguous
    k_tail, v_tail   bf16 or f16 [B, Hkv, 32, D]: the newest lengths % 32 tokens, rows 0 ...
    block_table      int32 [B, width]: the pages of a request in order (rows may be strided)
    lengths   int32 [B]: stored tokens of each request
    mask      uint8 [B, Hkv, tokens] or None: 0 = dead (``paged_attention`` skips it, as it
              does positions past the mask's end)

    A page id outside the pool and a length past the table's width are read as if those
    tokens were not there.  Strides and addresses are taken when the descriptor is made."""

    __slots__ = ("pool", "k_tail", "v_tail", "block_table", "lengths", "mask", "batch", "heads", "head_dim",
                 "page_tokens", "dtype", "device", "index", "_nat")

    def __init__(self, pool: torch.Tensor, k_tail: torch.Tensor, v_tail: torch.Tensor, block_table: torch.Tensor,
                 lengths: torch.Tensor, mask: torch.Tensor | None = None):
        if pool.ndim != 4 or pool.dtype != torch.uint8 or pool.shape[3] % 40:
            raise ValueError("pool must be a uint8 [pages, Hkv, page_tokens / 32, 40 * D] tensor")
        pages, hkv, per, rec = pool.shape
        d = rec // 40
        if pages and hkv and per and (pool.stride(3) != 1 or (per > 1 and pool.stride(2) != rec)):
            raise ValueError("pool: the records of a page and head must be contiguous")
        if k_tail.ndim != 4 or tuple(k_tail.shape[1:]) != (hkv, GROUP, d) or k_tail.shape != v_tail.shape:
            raise ValueError(f"k_tail and v_tail must be [B, {hkv}, {GROUP}, {d}]")
        if k_tail.stride() != v_tail.stride() or k_tail.stride(3) != 1:
            raise ValueError("k_tail and v_tail must share their strides, channels contiguous")
        if k_tail.dtype != v_tail.dtype:
            raise ValueError("k_tail and v_tail dtypes differ")
        if k_tail.dtype not in (torch.bfloat16, torch.float16):
            raise N.KernelUnavailableError(f"tails of {k_tail.dtype} are not built (bf16, f16)")
        b = k_tail.shape[0]
        _check_table(block_table, b)
        if mask is not None and (mask.ndim != 3 or mask.dtype != torch.uint8 or tuple(mask.shape[:2]) != (b, hkv) or
                                 (mask.shape[2] > 1 and mask.stride(2) != 1)):
            raise ValueError(f"mask must be a uint8 [{b}, {hkv}, tokens] tensor with contiguous tokens")
        if mask is not None:
            _c_int("mask's tokens", mask.shape[2])
        N.require_gpu(pool, "pool")
        index = pool.get_device()
        _i32(lengths, "lengths", (b,), index)
        _same_device(index, k_tail=k_tail, v_tail=v_tail, block_table=block_table, lengths=lengths, mask=mask)
        self.pool, self.k_tail, self.v_tail = pool, k_tail, v_tail
        self.block_table, self.lengths, self.mask = block_table, lengths, mask
        self.batch, self.heads, self.head_dim, self.page_tokens = b, hkv, d, per * GROUP
        self.dtype, self.device, self.index = k_tail.dtype, pool.device, index
        p = N.MaPages()
        p.pool, p.k_tail, p.v_tail = pool.data_ptr(), k_tail.data_ptr(), v_tail.data_ptr()
        p.table, p.lengths = block_table.data_ptr(), lengths.data_ptr()
        p.s_pool[0], p.s_pool[1] = pool.stride(0), pool.stride(1)
        for i in range(3):
            p.s_tail[i] = k_tail.stride(i)
        p.s_table = block_table.stride(0)
        p.num_pages, p.width, p.page_tokens = pages, block_table.shape[1], per * GROUP
        if mask is not None:
            # (an empty tensor's address is 0, which is no mask: any other stands for one whose positions
            # are all behind its end, and is not read)
            p.mask, p.mask_tokens = mask.data_ptr() or lengths.data_ptr(), mask.shape[2]
            p.s_mask[0], p.s_mask[1] = mask.stride(0), mask.stride(1)
        p.dtype = N.dtype_code(k_tail.dtype)
        self._nat = p

    def native(self) -> N.MaPages:
        return self._nat


def plan_pages(lengths: torch.Tensor, new_lens: torch.Tensor, block_table: torch.Tensor, free_ring: torch.Tensor,
               ring_state: torch.Tensor, *, page_tokens: int, tokens: int, slots: torch.Tensor | None = None,
               ends: torch.Tensor | None = None, give_back: bool = True):
    """Pages for one step, planned on the GPU: request b goes from lengths[b] to ends[b] =
    max(0, lengths[b] + new_lens[b]) tokens.  Returns (slots int64 [B, tokens], ends int32
    [B]): slot = page id * page_tokens + offset of each new token, -1 behind new_lens[b].

    block_table [B, width] gets the pages that appear and -1 for those that go (its rows must
    not overlap, nor ends lengths or new_lens).  free_ring
    int32 [pages] holds the free pages' ids first in, first out; ring_state int32 [4] =
    (place of the oldest, free pages, 0, status).  Growing requests take the oldest pages, in
    request order; pages given back (new_lens[b] < 0: that many tokens, at most all) enter
    behind the newest and are free from the next plan on: for a step given up before its
    append, or a request that ends (tokens of a packed group do not return to the tail).  A step
    that stores tokens passes give_back=False: a negative count then refuses it.  lengths is not
    written.

    A plan that cannot be met changes nothing, returns slots of -1 and ends = lengths, and
    adds to the status, which stays until the caller clears it: 1 the pages run out, 2 a
    request outgrows its table row, 4 new_lens[b] > tokens, 8 a negative length, 16 a negative
    new_lens[b] without give_back (``check_plan`` reads it and raises)."""
    if lengths.ndim != 1:
        raise ValueError(f"lengths must be [B], got {tuple(lengths.shape)}")
    N.require_gpu(lengths, "lengths")
    shape, index = lengths.shape, lengths.get_device()
    b = shape[0]
    _i32(lengths, "lengths", shape, index)
    _i32(new_lens, "new_lens", shape, index)
    _check_table(block_table, b)
    _i32(free_ring, "free_ring", (free_ring.numel(),), index)
    _i32(ring_state, "ring_state", (4,), index)
    tokens, page_tokens = _c_int("tokens", tokens), _c_int("page_tokens", page_tokens)
    if slots is None:
        slots = torch.empty((b, tokens), device=lengths.device, dtype=torch.int64)
    elif slots.dtype is not torch.int64 or slots.shape != (b, tokens) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 [{b}, {tokens}] tensor")
    if ends is None:
        ends = torch.empty_like(lengths)
    else:
        _i32(ends, "ends", shape, index)
    if block_table.get_device() != index or slots.get_device() != index:
        _same_device(index, block_table=block_table, slots=slots)
    if b == 0:
        return slots, ends
    _call(index, "ma_page_plan" if give_back else "ma_page_plan_append", lengths.data_ptr(), new_lens.data_ptr(), b, tokens, page_tokens,
          block_table.data_ptr(), block_table.stride(0), block_table.shape[1], free_ring.data_ptr(), free_ring.numel(),
          ring_state.data_ptr(), slots.data_ptr() if tokens else None, ends.data_ptr())
    return slots, ends


_PLAN_ERRORS = ((1, "the free pages run out"), (2, "a request outgrows its block table row"),
                (4, "more new tokens than the plan's tokens"), (8, "a negative length"),
                (16, "a negative number of new tokens"))


_OUTSIDE = 32     # of the status: a new token's position that a rotary table does not hold


def check_plan(ring_state: torch.Tensor) -> None:
    """Raise RuntimeError for what plans since the last check could not meet, and for new tokens
    that were rotated outside of their table (waits for them, and clears the status)."""
    status = int(ring_state[3].item())
    if status:
        ring_state[3].zero_()
        what = ["page plan refused: " + ", ".join(text for bit, text in _PLAN_ERRORS if status & bit)] if status & ~_OUTSIDE else []
        if status & _OUTSIDE:
            what.append("new tokens at positions outside the rotary table were turned by its nearest row")
        raise RuntimeError("; ".join(what))


def _check_block(name: str, t: torch.Tensor, prefix: PagedPrefix, heads: int | None = None) -> torch.Size:
    """[B, heads, T, D] of the prefix's batch, head_dim, dtype and device; returns the shape."""
    s = t.shape
    if len(s) != 4 or s[0] != prefix.batch or s[3] != prefix.head_dim or (heads is not None and s[1] != heads):
        raise ValueError(f"{name} must be [{prefix.batch}, {'H' if heads is None else heads}, T, {prefix.head_dim}], "
                         f"got {tuple(s)}")
    if t.get_device() != prefix.index:
        N.require_gpu(t, name)
        raise ValueError(f"{name} is on {t.device}, expected {prefix.device}")
    if t.dtype is not prefix.dtype:
        raise ValueError(f"{name} is {t.dtype}, the prefix {prefix.dtype}")
    return s


def rotary_table(positions: int, head_dim: int, *, base: float = 10000.0, rotary_dim: int | None = None,
                 inv_freq: torch.Tensor | None = None, device: torch.device | str = "cuda") -> torch.Tensor:
    """The f32 [positions, rotary_dim] table of ``rotate_block`` and ``append_pages``: row p holds
    the cosines, then the sines, of p * inv_freq (default: base ** (-2 i / rotary_dim), i = 0 ..
    rotary_dim / 2 - 1), angles and functions in 64 bits.  rotary_dim: a multiple of 16 up to
    head_dim, its default.  Made once; a program keeps it for all layers and steps."""
    positions, dim = _c_int("positions", positions), int(head_dim if rotary_dim is None else rotary_dim)
    if positions == 0 or dim <= 0 or dim > head_dim or dim % 16:
        raise ValueError(f"a rotary table needs a position and a multiple of 16 up to {head_dim} channels, got "
                         f"{positions} and {dim}")
    if inv_freq is None:
        inv_freq = base ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    elif tuple(inv_freq.shape) != (dim // 2,):
        raise ValueError(f"inv_freq must be [{dim // 2}], got {tuple(inv_freq.shape)}")
    at = torch.arange(positions, dtype=torch.float64, device=device)
    angle = at[:, None] * inv_freq.to(device=device, dtype=torch.float64)[None]
    return torch.cat((angle.cos(), angle.sin()), 1).float()


_ROTARY_PACK = struct.Struct("=QQqiiiiQQ").pack


def _rotary(prefix: PagedPrefix, table: torch.Tensor, interleaved: bool, positions: torch.Tensor | None,
            ring_state: torch.Tensor | None, new_lens: torch.Tensor | None = None) -> N.MaRotary:
    """The kernels' descriptor of a rotary table (positions None: the prefix's lengths; ring_state: whose
    status is told of positions outside the table)."""
    s = table.shape
    if len(s) != 2 or table.dtype is not torch.float32 or not s[0] or not 0 < s[1] <= prefix.head_dim or s[1] % 16 or \
            table.stride(1) != 1:
        raise ValueError(f"rotary must be a float32 [positions, channels] tensor with contiguous rows of a multiple of 16 "
                         f"up to {prefix.head_dim} channels, got {table.dtype} {tuple(s)}")
    if table.get_device() != prefix.index:
        N.require_gpu(table, "rotary")
        raise ValueError(f"rotary is on {table.device}, expected {prefix.device}")
    if positions is not None:
        _i32(positions, "positions", (prefix.batch,), prefix.index)
    status = count = 0
    if ring_state is not None:
        _i32(ring_state, "ring_state", (4,), prefix.index)
        status = ring_state.data_ptr() + 12
        if new_lens is not None:
            _i32(new_lens, "new_lens", (prefix.batch,), prefix.index)
            count = new_lens.data_ptr()
    return N.MaRotary.from_buffer_copy(_ROTARY_PACK(
        table.data_ptr(), 0 if positions is None else positions.data_ptr(), table.stride(0) if s[0] > 1 else s[1],
        _c_int("rotary's positions", s[0]), s[1], bool(interleaved), 0, status, count))


def _rows_overlap(t: torch.Tensor) -> bool:
    """Two rows of [B, H, T, D] (channels contiguous) have bytes in common."""
    if t.is_contiguous():
        return False
    end = t.shape[3]
    dims = sorted((st, n) for st, n in zip(t.stride(), t.shape[:3]) if n > 1)
    for st, n in dims:
        if st < end:
            break
        end += st * (n - 1)
    else:
        return False         # (every step is longer than what the shorter ones span)
    starts = torch.zeros(1, dtype=torch.int64)
    for st, n in dims:       # (rows between rows: rare)
        starts = (starts[:, None] + st * torch.arange(n)).flatten()
    starts = starts.sort().values
    return bool((starts[1:] - starts[:-1] < t.shape[3]).any())


def _check_rows(name: str, t: torch.Tensor, prefix: PagedPrefix, out: torch.Tensor | None) -> torch.Tensor:
    """The output of rotated rows t [B, H, T, D]: `out`, or a new tensor."""
    shape = _check_block(name, t, prefix)
    if out is None:
        return torch.empty_like(t)        # (half the time of one by shape)
    if _check_block(f"out_{name}", out, prefix, shape[1]) != shape:
        raise ValueError(f"out_{name} must be {tuple(shape)}")
    if _rows_overlap(out):
        raise ValueError(f"out_{name} holds rows that share their memory")
    return out


def rotate_block(prefix: PagedPrefix, query: torch.Tensor, key: torch.Tensor | None = None, *, rotary: torch.Tensor,
                 interleaved: bool = False, positions: torch.Tensor | None = None,
                 out_query: torch.Tensor | None = None, out_key: torch.Tensor | None = None,
                 new_lens: torch.Tensor | None = None, ring_state: torch.Tensor | None = None):
    """query [B, Hq, T, D] and key [B, Hk, T, D] (or None) rotated at their positions: position t of
    request b is prefix.lengths[b] + t (positions int32 [B]: positions[b] + t).  Returns (query, key).

    rotary is a ``rotary_table``; channels i and i + rotary_dim / 2 are a pair (interleaved: 2 i
    and 2 i + 1), channels from rotary_dim on stay as they are.  x' = x cos - y sin, y' = y cos + x
    sin, each operation rounded to f32, the result once to its type.  Positions outside the table
    take its nearest row; with ring_state (``plan_pages``) such a position of a real new token (t <
    new_lens[b]; None: T) is noted in its status, for ``check_plan``.  All T rows are rotated.  out_query may
    be query, out_key key; otherwise they must not overlap them."""
    out_query = _check_rows("query", query, prefix, out_query)
    if key is None and out_key is not None:
        raise ValueError("out_key without a key")
    if key is not None:
        out_key = _check_rows("key", key, prefix, out_key)
        if key.shape[2] != query.shape[2]:
            raise ValueError(f"key must hold {query.shape[2]} positions like the queries")
    rot = _rotary(prefix, rotary, interleaved, positions, ring_state, new_lens)
    b, hq, t, d = query.shape
    hk = 0 if key is None else key.shape[1]
    if hq == 0 and hk:      # (the kernel wants rows in its first place)
        rotate_block(prefix, key, None, rotary=rotary, interleaved=interleaved, positions=positions, out_query=out_key,
                     new_lens=new_lens, ring_state=ring_state)
    elif b and t and hq:
        _call(prefix.index, "ma_rotate_block", N.t4(query), hq, N.t4(out_query), N.t4(key if hk else None), hk,
              N.t4(out_key if hk else None), b, t, d, prefix.lengths.data_ptr(), rot)
    return out_query, out_key


def append_pages(prefix: PagedPrefix, key: torch.Tensor, value: torch.Tensor, new_lens: torch.Tensor,
                 slots: torch.Tensor, *, rotary: torch.Tensor | None = None, interleaved: bool = False,
                 positions: torch.Tensor | None = None, query: torch.Tensor | None = None,
                 out_query: torch.Tensor | None = None, ring_state: torch.Tensor | None = None) -> torch.Tensor | None:
    """Store new_lens[b] (0 .. T) tokens of key, value [B, Hkv, T, D] behind request b's
    prefix.lengths[b] tokens: every 32-token group that they complete is quantized into the
    page that ``slots`` (``plan_pages``) names, the rest stays in the tail at 16 bits.
    prefix.lengths is not written: it is to become plan_pages' ends when every layer has been
    appended to.  Requests without new tokens, or whose slots are -1, are left as they are.

    rotary (a ``rotary_table``): the keys are rotated at their positions on the way; what is stored
    is what ``rotate_block`` and an append of its result would store, bit for bit, and key is not
    written.  interleaved, positions, ring_state: as there.  With query [B, Hq, T, D] the same launch rotates all
    its rows, and they are returned (in out_query, if given, which may be query and overlaps nothing
    else that the call reads)."""
    shape = _check_block("key", key, prefix, prefix.heads)
    if _check_block("value", value, prefix, prefix.heads) != shape:
        raise ValueError("key and value shapes differ")
    b, h, t, d = shape
    _i32(new_lens, "new_lens", (b,), prefix.index)
    if slots.dtype is not torch.int64 or slots.shape != (b, t) or not slots.is_contiguous():
        raise ValueError(f"slots must be a contiguous int64 [{b}, {t}] tensor")
    if slots.get_device() != prefix.index:
        raise ValueError(f"slots is on {slots.device}, expected {prefix.device}")
    if rotary is None:
        if query is not None or out_query is not None or positions is not None or ring_state is not None:
            raise ValueError("query, out_query, positions and ring_state need a rotary table")
        if b and t:
            _call(prefix.index, "ma_page_append", prefix._nat, N.t4(key), N.t4(value), b, h, t, d, new_lens.data_ptr(),
                  slots.data_ptr())
        return None
    rot, hq = _rotary(prefix, rotary, interleaved, positions, ring_state), 0
    if query is not None:
        out_query = _check_rows("query", query, prefix, out_query)
        hq = query.shape[1]
        if query.shape[2] != t:
            raise ValueError(f"query must hold {t} positions like the keys")
    elif out_query is not None:
        raise ValueError("out_query without a query")
    if b and t:
        _call(prefix.index, "ma_page_append_rotary", prefix._nat, N.t4(key), N.t4(value), b, h, t, d, new_lens.data_ptr(),
              slots.data_ptr(), rot, N.t4(query if hq else None), hq, N.t4(out_query if hq else None))
    return out_query


def dequantize_pages(prefix: PagedPrefix, tokens: int, *, starts: torch.Tensor | None = None,
                     dtype: torch.dtype | None = None, out_key: torch.Tensor | None = None,
                     out_value: torch.Tensor | None = None):
    """Tokens starts[b] .. starts[b] + tokens of every request (starts None: from 0) as K and V
    [B, Hkv, tokens, D] in dtype (default: the tails'), zero from the request's length on."""
    tokens = _c_int("tokens", tokens)
    shape = (prefix.batch, prefix.heads, tokens, prefix.head_dim)
    dtype = dtype or (out_key.dtype if out_key is not None else prefix.dtype)
    if out_key is None:
        out_key = torch.empty(shape, device=prefix.device, dtype=dtype)
        if out_value is None:
            out_value = torch.empty_like(out_key)     # (a third cheaper than by its shape)
    if out_value is None:
        out_value = torch.empty(shape, device=prefix.device, dtype=dtype)
    for name, t in (("out_key", out_key), ("out_value", out_value)):
        if t.shape != shape or t.dtype is not dtype or t.get_device() != prefix.index:
            raise ValueError(f"{name} must be {dtype} {shape} on {prefix.device}")
    if starts is not None:
        _i32(starts, "starts", (prefix.batch,), prefix.index)
    if prefix.batch == 0 or tokens == 0:
        return out_key, out_value
    _call(prefix.index, "ma_page_dequant", prefix._nat, prefix.batch, prefix.heads, prefix.head_dim, N.ptr(starts),
          tokens, N.t4(out_key), N.t4(out_value))
    return out_key, out_value


def select_blocks(query: torch.Tensor, prefix: PagedPrefix, count: int, *, new_lens: torch.Tensor | None = None,
                  block_tokens: int = GROUP, query_block: int = 0, keep_first: int = 0, keep_last: int = 0,
                  return_scores: bool = False):
    """The blocks of stored tokens that the queries [B, Hq, T, D] of every request should read:
    int32 [B, Hkv, runs, count], ascending, -1 behind the last.  A run is query_block positions
    (0: all T) of the Hq / Hkv query heads of a KV head, runs = ceil(T / query_block); positions t >=
    new_lens[b] (None: T) count for nothing.  Block i is the tokens i * block_tokens ... (a multiple of
    32) of a request's whole groups of 32; the newest lengths % 32 tokens are in no block
    (``paged_attention`` reads them always).

    A block's score is what q . k could be at most for its keys' channel ranges, which the 4-bit
    records hold: a tenth of the cache is read.  It is the largest over the run's rows and the block's
    groups, computed in whole numbers (14 bits of the row's and of the group's largest), so the
    same blocks are taken whatever the batch.  The count best are taken, ties to the lowest index;
    the keep_first oldest and keep_last newest blocks in any case.  Blocks without a live token
    (prefix.mask) are not.  A row or a group with NaN or infinities scores infinity.

    return_scores: also the scores, float32 [B, Hkv, runs, blocks that a table row can name], -inf
    where there is no block."""
    b, hq, t, d = _check_block("query", query, prefix)
    h, width = prefix.heads, prefix._nat.width
    if h == 0 or hq == 0 or hq % h:
        raise ValueError("Hq must be a positive multiple of Hkv")
    count, block_tokens, query_block = _c_int("count", count), _c_int("block_tokens", block_tokens), _c_int("query_block", query_block)
    keep_first, keep_last = _c_int("keep_first", keep_first), _c_int("keep_last", keep_last)
    if not block_tokens or block_tokens % GROUP:
        raise ValueError(f"block_tokens must be a positive multiple of {GROUP}, got {block_tokens}")
    if count < 1 or keep_first + keep_last > count:
        raise ValueError(f"count must be positive and hold keep_first and keep_last, got {count}, {keep_first} and {keep_last}")
    if new_lens is not None:
        _i32(new_lens, "new_lens", (b,), prefix.index)
    runs = -(-t // query_block) if query_block else min(t, 1)
    tokens = width * prefix.page_tokens
    blocks = query.new_empty((b, h, runs, count), dtype=torch.int32)
    scores = query.new_empty((b, h, runs, -(-tokens // block_tokens)), dtype=torch.float32) if return_scores else None
    if b and t:
        if tokens == 0 or prefix._nat.num_pages == 0:
            blocks.fill_(-1)
            if return_scores:
                scores.fill_(float("-inf"))
            return (blocks, scores) if return_scores else blocks
        need = N.size_query("ma_select_workspace_bytes", b, h, runs, tokens)
        if need < 0:
            raise N.KernelUnavailableError(f"{b * h * runs} selections over {tokens} tokens are not built")
        # (blocks of one group: their scores are the groups', and lie where they are returned)
        ws = scores if return_scores and block_tokens == GROUP else query.new_empty((need,), dtype=torch.uint8)
        _call(prefix.index, "ma_select_blocks", N.t4(query), b, hq, t, d, prefix._nat, h, N.ptr(new_lens), query_block,
              block_tokens, count, keep_first, keep_last, blocks.data_ptr(), N.ptr(scores), ws.data_ptr(), need)
    return (blocks, scores) if return_scores else blocks


def paged_attention(query: torch.Tensor, prefix: PagedPrefix, current_key: torch.Tensor | None = None,
                    current_value: torch.Tensor | None = None, *, new_lens: torch.Tensor | None = None,
                    scaling: float | None = None, causal_block: int = 0, out: torch.Tensor | None = None,
                    blocks: torch.Tensor | None = None, block_tokens: int = GROUP, query_block: int = 0):
    """softmax over [request b's stored tokens | the block's own keys] for every query row of
    query [B, Hq, T, D] (``splitk_attention`` with one length per request; Hq a multiple of
    Hkv, head_dim 64 or 128, one dtype of bf16 and f16 throughout).

    current_key, current_value [B, Hkv, T, D] (None: the stored tokens alone).  new_lens int32
    [B] (None: T each) counts each request's real positions: rows t >= new_lens[b] of out are
    left as they are, keys j >= new_lens[b] not seen.  causal_block > 0: key j is seen by query
    t only if (lengths[b] + j) // causal_block <= (lengths[b] + t) // causal_block.  A row that
    sees nothing is zero; what a row does not see may hold anything, NaN and infinities too.  A
    packed value is an f16 here (beyond 65504: infinite).  The same call gives the same bits.
    ``out`` [B, Hq, T, D] (not overlapping the inputs) receives the result; without it a new
    tensor does, whose rows t >= new_lens[b] are undefined.

    blocks int32 [B, Hkv, runs, count] (``select_blocks``, with the same block_tokens and query_block)
    names the stored tokens that each run of query_block positions (0: all T) reads, beside the tail and
    the block's own keys, in the place of all: entry i is tokens i * block_tokens ... of the request's
    whole groups of 32.  Entries that are no block (-1) read nothing, entries behind as many as the
    request has blocks are not looked at, one listed twice weighs twice."""
    shape = _check_block("query", query, prefix)
    b, hq, t, d = shape
    h = prefix.heads
    if h == 0 or hq == 0 or hq % h:
        raise ValueError("Hq must be a positive multiple of Hkv")
    if blocks is not None:
        block_tokens, query_block = _c_int("block_tokens", block_tokens), _c_int("query_block", query_block)
        if not block_tokens or block_tokens % GROUP:
            raise ValueError(f"block_tokens must be a positive multiple of {GROUP}, got {block_tokens}")
        runs = -(-t // query_block) if query_block else min(t, 1)
        if blocks.ndim != 4:
            raise ValueError(f"blocks must be [{b}, {h}, {runs}, count], got {tuple(blocks.shape)}")
        _i32(blocks, "blocks", (b, h, runs, blocks.shape[3]), prefix.index)
    elif query_block:
        raise ValueError("query_block without blocks")
    if (current_key is None) != (current_value is None):
        raise ValueError("current_key and current_value go together")
    if current_key is not None:
        if _check_block("current_key", current_key, prefix, h)[2] != t or \
                _check_block("current_value", current_value, prefix, h)[2] != t:
            raise ValueError(f"the block's keys and values must hold {t} positions like its queries")
    if new_lens is not None:
        _i32(new_lens, "new_lens", (b,), prefix.index)
    causal_block = _c_int("causal_block", causal_block)
    if out is None:
        out = torch.empty(shape, device=query.device, dtype=query.dtype)
    elif _check_block("out", out, prefix, hq) != shape:
        raise ValueError(f"out must be {tuple(shape)}")
    if b == 0 or t == 0:
        return out
    scale = float(scaling) if scaling is not None else d ** -0.5
    if blocks is not None:
        if blocks.shape[3] == 0:
            blocks = torch.full((b, h, runs, 1), -1, device=query.device, dtype=torch.int32)
        need = N.size_query("ma_paged_blocks_workspace_bytes", b, h, hq, t, d, blocks.shape[3], block_tokens, query_block)
    else:
        need = N.size_query("ma_paged_workspace_bytes", b, h, hq, t, d)
    if need < 0:
        raise N.KernelUnavailableError(f"{hq // h * t} rows for each of {b * h} KV heads are not built")
    ws = query.new_empty((need,), dtype=torch.uint8) if need else None
    if blocks is not None:
        _call(prefix.index, "ma_paged_attention_blocks", N.t4(query), b, hq, t, d, prefix._nat, h, N.t4(current_key),
              N.t4(current_value), N.ptr(new_lens), causal_block, scale, N.t4(out), blocks.data_ptr(), blocks.shape[3],
              block_tokens, query_block, N.ptr(ws), need)
        return out
    _call(prefix.index, "ma_paged_attention", N.t4(query), b, hq, t, d, prefix._nat, h, N.t4(current_key),
          N.t4(current_value), N.ptr(new_lens), causal_block, scale, N.t4(out), ws.data_ptr(), need)
    return out


__all__ = ["PagedPrefix", "append_pages", "check_plan", "dequantize_pages", "paged_attention", "plan_pages",
           "record_bytes", "rotary_table", "rotate_block", "select_blocks"]
