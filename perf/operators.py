"""The calls that the paged KV cache's operators are judged by.

A serving program keeps one pool of pages for the keys and values of all its
requests.  Each step it (1) builds the block tables and the slot map of the
new tokens from the requests' lengths, on the GPU (``paged_step``), (2) writes
the new keys and values into their pages in 8 bits (``paged_kv_write``), (3)
attends over the pages (``paged_attention``), and (4) takes pages back when
requests end or drafted tokens are rejected (``paged_trim``).

Cache: ``codes`` [P, NB, Hkv, 2, 64 D] e4m3 bytes and ``scales`` [P, NB, Hkv, 2]
E8M0 bytes (2^(b - 127)): a page is NB blocks of 64 tokens, and each block and
head has one scale for its keys (index 0) and one for its values (index 1).
The 64 D bytes of a block hold
  keys:   [4 tg][D/64 dg][4 q][16 c][16 j] = token 16 tg + c, dim 64 dg + 16 q + j
  values: [D/16 dt][4 q][16 c][4 w][4 j]   = token 16 w + 4 q + j, dim 16 dt + c

Sizes are generic ones of grouped-query attention (64 query heads on 8 KV
heads of 128, 16 on 16 of 64, 32 on 4 of 128), contexts of one token to 131072,
batches of 1 to 4096 requests.  The lengths of a case's requests follow from
the case alone, everything else from the seed.
"""
from __future__ import annotations

import math
from types import SimpleNamespace

import torch

own = False

BLOCK = 64
NAN_CODE = 0x7F


def listed() -> list:
    return [
        # block tables and slots of a small decode batch: the smallest call, latency alone
        dict(name="step_decode_r16", op="step", r=16, ctx=4096, n=1, every=1, page=64, pad=0, dry=False),
        # a large batch in which every 16th request brings a piece of its prompt, in a padded token buffer
        dict(name="step_mixed_r2048", op="step", r=2048, ctx=8192, n=512, every=16, page=64, pad=100, dry=False),
        # drafted tokens rejected and ended requests released in a decode batch
        dict(name="trim_r64", op="trim", r=64, ctx=8192, page=64, ended=8),
        # the same for a large batch, many of whose requests end at once
        dict(name="trim_r2048", op="trim", r=2048, ctx=16384, page=128, ended=2),
        # one token of each of 64 requests into the ends of their pages
        dict(name="write_decode_r64", op="write", r=64, ctx=2000, n=1, hkv=8, d=128, page=64),
        # prompts of several requests, written whole
        dict(name="write_prompts_r8", op="write", r=8, ctx=0, n=8192, hkv=8, d=128, page=64),
        # ragged pieces that begin and end inside blocks
        dict(name="write_pieces_r33", op="write", r=33, ctx=777, n=150, hkv=16, d=64, page=128),
        # one user's decode step with a short context: latency
        dict(name="attn_decode_r1_short", op="attn", r=1, ctx=516, n=1, hq=64, hkv=8, d=128, page=64, window=0,
             sink=False),
        # one user's decode step with a very long context: few rows over a long axis
        dict(name="attn_decode_r1_long", op="attn", r=1, ctx=131000, n=1, hq=64, hkv=8, d=128, page=64, window=0,
             sink=False),
        # a decode step of 64 requests of very unequal lengths
        dict(name="attn_decode_r64", op="attn", r=64, ctx=32768, n=1, hq=64, hkv=8, d=128, page=64, window=0,
             sink=True),
        # the prompt of one request
        dict(name="attn_prompt_s4096", op="attn", r=1, ctx=0, n=4096, hq=64, hkv=8, d=128, page=64, window=0,
             sink=False),
        # ragged pieces of prompts behind longer contexts, windowed, a key head for each query head
        dict(name="attn_pieces_r8", op="attn", r=8, ctx=2500, n=500, hq=16, hkv=16, d=64, page=128, window=1000,
             sink=True),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    op = rng.choice(["step", "trim", "write", "write", "attn_decode", "attn_decode", "attn_prompt", "attn_prompt"])
    page = rng.choice([64, 64, 128, 256])
    if op == "step":
        r = _log_int(rng, 1, 2048)
        every = rng.choice([1, 1, 4, 16])
        n = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, min(8192, 65536 * every // r)))
        return dict(op=op, r=r, ctx=_log_int(rng, 1, 8192), n=n, every=every, page=page, pad=rng.choice([0, 1, 77]),
                    dry=rng.random() < 0.2)
    if op == "trim":
        return dict(op=op, r=_log_int(rng, 1, 2048), ctx=_log_int(rng, 8, 16384), page=page,
                    ended=rng.choice([1, 2, 8, 1 << 20]))
    hkv, d = rng.choice([(8, 128), (8, 128), (16, 64), (4, 128), (1, 128), (2, 256), (5, 64)])
    if op == "write":
        n = 1 if rng.random() < 0.3 else _log_int(rng, 2, 8192)
        most = max(1, min(256, 8 * 8192 * 1024 // (n * hkv * d)))  # tokens of all requests, by their size
        return dict(op=op, r=_log_int(rng, 1, most), ctx=rng.choice([0, _log_int(rng, 1, 2000)]), n=n, hkv=hkv, d=d,
                    page=page)
    group = rng.choice([1, 4, 7, 8, 16]) if hkv * d < 2048 else rng.choice([4, 8])
    window, sink = rng.choice([0, 0, 128, 1000]), rng.random() < 0.5
    if op == "attn_decode":
        n = rng.choice([1, 1, 1, 2, 4])
        r = _log_int(rng, 1, 64)
        ctx = _log_int(rng, 1, max(1, min(131000, 2000000 // r)))
    else:
        r = rng.randint(1, 8)
        n = _log_int(rng, 16, 4096 // r)
        ctx = rng.choice([0, _log_int(rng, 1, 8192 // r)])
        room = 1 << 30  # scores of the plain form
        while r * n * group * hkv * (ctx + n) > room:
            n, ctx = max(1, n // 2), ctx // 2
    return dict(op="attn", r=r, ctx=ctx, n=n, hq=hkv * group, hkv=hkv, d=d, page=page, window=window, sink=sink)


# ----------------------------------------------------------------- lengths ---
def _spread(i: int, most: int) -> int:
    """Request i's share of `most`: spread evenly over 1..most, the first request's whole."""
    return max(1, math.ceil(most * (1.0 - (i * 0.6180339887498949) % 1.0)))


def _lengths(case) -> tuple:
    """(tokens held before, tokens of this call) of each request, from the case alone."""
    r, ctx = case["r"], case["ctx"]
    old = [_spread(i, ctx) if ctx else 0 for i in range(r)]
    if case["op"] == "trim":
        return old, [0] * r
    every = case.get("every", 1)
    decode = case["n"] <= 4  # decode steps and drafts bring as many tokens for each request
    new = [(case["n"] if decode else _spread(3 * i, case["n"])) if i % every == 0 else 1 for i in range(r)]
    return old, new


def _kept(case, old) -> list:
    """What each request keeps in a trim: the ended ones nothing, the others all but up to three drafted tokens."""
    return [0 if i % case["ended"] == 0 else max(0, x - i % 4) for i, x in enumerate(old)]


def _pages(x: int, page: int) -> int:
    return -(-x // page)


# ----------------------------------------------------------------- prepare ---
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    old, new = _lengths(case)
    page, r = case["page"], case["r"]
    both = [a + b for a, b in zip(old, new)]
    st = SimpleNamespace(op=case["op"], case=case, page=page)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    # the pool: the requests' pages lie in no order, as after hours of serving
    held = sum(_pages(x, page) for x in old)
    fresh = sum(_pages(b, page) - _pages(a, page) for a, b in zip(old, both))
    st.width = max(_pages(b, page) for b in both) + 3
    total = held + fresh + 5
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)

    def table(lengths, ids):
        n = torch.tensor([_pages(x, page) for x in lengths], device="cuda")
        at = torch.arange(st.width, device="cuda")[None, :]
        here = at < n[:, None]
        t = torch.full((r, st.width), -1, dtype=torch.int32, device="cuda")
        t[here] = ids[: int(n.sum())]
        return t

    def pool(hkv, d):
        """Codes of N(0, 1) values scaled to their block's largest, and scales that put them near 1."""
        nb = page // BLOCK
        codes = torch.empty(total, nb, hkv, 2, BLOCK * d, dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 27) // (nb * hkv * 2 * BLOCK * d))
        for i in range(0, total, step):
            part = codes[i:i + step]
            x = torch.randn(part.shape, generator=g, device="cuda").mul_(112.0).clamp_(-448.0, 448.0)
            part.copy_(x.to(torch.float8_e4m3fn).view(torch.uint8))
        scales = torch.randint(118, 122, (total, nb, hkv, 2), generator=g, device="cuda").to(torch.uint8)
        return codes, scales

    if st.op in ("step", "trim"):
        st.table = table(old, order)
        st.lengths = ints(old)
        st.free = torch.zeros(total, dtype=torch.int32, device="cuda")
        spare = order[held:]
        if case.get("dry"):
            spare = spare[: (2 * fresh) // 3]  # a pool that runs out
        st.free[: spare.numel()] = spare
        st.count = ints([spare.numel()])
        if st.op == "step":
            st.new = ints(new)
            st.tokens = sum(new) + case["pad"]
        else:
            st.keep = ints(_kept(case, old))
        return st
    starts = [0]
    for b in new:
        starts.append(starts[-1] + b)
    st.starts, st.seq = ints(starts), ints(both)
    st.most_new, st.most = max(new), max(both)
    st.table = table(both, order)
    hkv, d = case["hkv"], case["d"]
    st.codes, st.scales = pool(hkv, d)
    t = starts[-1]
    if st.op == "write":
        # keys and values as slices of one projection's output, channels of unequal size
        size = torch.exp(0.5 * torch.randn(2 * hkv * d, generator=g, device="cuda"))
        kv = (torch.randn(t, 2 * hkv * d, generator=g, device="cuda") * size).to(torch.bfloat16)
        st.k, st.v = kv[:, :hkv * d].view(t, hkv, d), kv[:, hkv * d:].view(t, hkv, d)
        return st
    st.q = torch.randn(t, case["hq"], d, generator=g, device="cuda").to(torch.bfloat16)
    st.sink = torch.randn(case["hq"], generator=g, device="cuda") if case["sink"] else None
    st.scale = d ** -0.5
    st.window = case["window"]
    return st


# --------------------------------------------------------------------- run ---
def run(st):
    if own:
        from mosaic_amd import ops

        if st.op == "step":
            s = ops.paged_step(st.lengths, st.new, st.table, st.tokens, st.page, st.free, st.count)
            return dict(table=st.table, starts=s.starts, lengths=s.lengths, seq_lens=s.seq_lens,
                        positions=s.positions, slots=s.slots, free_count=s.free_count)
        if st.op == "trim":
            lengths, count = ops.paged_trim(st.lengths, st.keep, st.table, st.page, st.free, st.count)
            return dict(lengths=lengths, free_count=count, free=st.free)
        if st.op == "write":
            ops.paged_kv_write(st.k, st.v, st.codes, st.scales, st.table, st.starts, st.seq)
            return dict(codes=st.codes.view(torch.float8_e4m3fn), scales=st.scales)
        return ops.paged_attention(st.q, st.codes, st.scales, st.table, st.starts, st.seq, st.scale, sink=st.sink,
                                   window=st.window, max_new=st.most_new)
    if st.op == "step":
        return _plain_step(st)
    if st.op == "trim":
        return _plain_trim(st)
    if st.op == "write":
        return _plain_write(st)
    return _plain_attention(st)


# ------------------------------------------------------------- plain forms ---
def _plain_step(st):
    page, tokens = st.page, st.tokens
    r, width = st.table.shape
    held, new = st.lengths.long().clamp(min=0), st.new.long().clamp(min=0)
    ends = torch.cumsum(new, 0)
    free = st.count.long().clamp(0, st.free.numel())
    fits = (ends <= tokens) & (held + new <= width * page)
    before, after = (held + page - 1) // page, (held + new + page - 1) // page
    need = torch.where(fits, after - before, 0)
    taken = torch.cumsum(need, 0)
    placed = fits & ((need == 0) | (taken <= free))
    lengths = torch.where(placed, held + new, held)
    seq = torch.where(placed, held + new, 0)
    left = free - torch.where(placed, need, 0).sum()
    # page j of a request's new ones is popped after those of the requests before it
    col = torch.arange(width, device=st.table.device)[None, :]
    j = col - before[:, None]
    mine = placed[:, None] & (j >= 0) & (col < after[:, None])
    pop = (free - 1 - (taken - need)[:, None] - j).clamp(0, st.free.numel() - 1)
    st.table.copy_(torch.where(mine, st.free[pop], st.table))
    # the request of a token row, its position and its slot
    t = torch.arange(tokens, device=st.table.device)
    row = torch.searchsorted(ends, t, right=True).clamp(max=r - 1)
    pos = held[row] + t - (ends - new)[row]
    real = placed[row] & (t < ends[-1])
    slot = st.table[row, (pos // page).clamp(max=width - 1)].long() * page + pos % page
    starts = torch.cat([ends.new_zeros(1), ends]).clamp(max=tokens)
    return dict(table=st.table, starts=starts.int(), lengths=lengths.int(), seq_lens=seq.int(),
                positions=torch.where(real, pos, -1).int(), slots=torch.where(real, slot, -1).int(),
                free_count=left.int())


def _plain_trim(st):
    page = st.page
    width = st.table.shape[1]
    held = st.lengths.long().clamp(0, width * page)
    keep = torch.minimum(st.keep.long().clamp(min=0), held)
    first, last = (keep + page - 1) // page, (held + page - 1) // page
    ends = torch.cumsum(last - first, 0)
    total = ends[-1]
    free = st.count.long()
    # the inverse of taking them: the last request's last page goes back first
    col = torch.arange(width, device=st.table.device)[None, :]
    back = (col >= first[:, None]) & (col < last[:, None])
    rank = (ends - (last - first))[:, None] + col - first[:, None]
    at = free + total - 1 - rank
    st.free[at[back]] = st.table[back]
    return dict(lengths=keep.int(), free_count=(free + total).int(), free=st.free)


def _to_tokens(codes, part: int, d: int):
    """Codes [..., 2, 64 D] of whole blocks -> values [..., 64, D] in 32 bits, without their scales."""
    x = codes[..., part, :].view(torch.float8_e4m3fn).float()
    lead = x.shape[:-1]
    n = len(lead)
    if part == 0:
        x = x.view(*lead, 4, d // 64, 4, 16, 16).permute(*range(n), n, n + 3, n + 1, n + 2, n + 4)
    else:
        x = x.view(*lead, d // 16, 4, 16, 4, 4).permute(*range(n), n + 3, n + 1, n + 4, n, n + 2)
    return x.reshape(*lead, BLOCK, d)


def _from_tokens(x, part: int, d: int):
    """The inverse, of e4m3 values: [..., 64, D] -> bytes [..., 64 D]."""
    lead = x.shape[:-2]
    n = len(lead)
    if part == 0:
        x = x.view(*lead, 4, 16, d // 64, 4, 16).permute(*range(n), n, n + 2, n + 3, n + 1, n + 4)
    else:
        x = x.view(*lead, 4, 4, 4, d // 16, 16).permute(*range(n), n + 3, n + 1, n + 4, n, n + 2)
    return x.reshape(*lead, BLOCK * d).to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_write(st):
    d, nb = st.case["d"], st.page // BLOCK
    starts, seq = st.starts.long(), st.seq.long()
    new = starts[1:] - starts[:-1]
    held = seq - new
    # the blocks of 64 tokens that take new tokens
    first, last = held // BLOCK, (seq + BLOCK - 1) // BLOCK
    most = _pages(st.most_new, BLOCK) + 1
    j = first[:, None] + torch.arange(most, device=seq.device)[None, :]
    row, col = torch.nonzero((j < last[:, None]) & (new > 0)[:, None], as_tuple=True)
    block = j[row, col]
    page, sub = st.table[row, block // nb].long(), block % nb
    pos = block[:, None] * BLOCK + torch.arange(BLOCK, device=seq.device)  # [U, 64]
    is_old = (pos < held[row][:, None])[:, None, :, None]
    is_new = (~is_old[:, 0, :, 0] & (pos < seq[row][:, None]))[:, None, :, None]
    src = (starts[row][:, None] + pos - held[row][:, None]).clamp(0, st.k.shape[0] - 1)
    any_old = is_old.any(2).any(2)  # [U, 1]
    codes, scales = st.codes[page, sub], st.scales[page, sub]  # [U, Hkv, 2, 64 D], [U, Hkv, 2]
    out, exps = [], []
    for part, x in enumerate((st.k, st.v)):
        x = x[src].transpose(1, 2).float()  # [U, Hkv, 64, D]
        size = torch.where(is_new & torch.isfinite(x), x.abs(), 0.0).amax((2, 3))
        mant, e = torch.frexp(size / 448.0)  # a power of two: 448 2^e holds the largest (the quotient rounds up or exactly)
        e = e - (torch.ldexp(torch.full_like(size, 448.0), e - 1) >= size).to(e.dtype)
        e = torch.where(size > 0, e, -126).clamp(-126, 127)
        was = scales[..., part].to(torch.int32) - 127
        e = torch.where(any_old, torch.maximum(e, was), e)
        # old tokens move to the larger scale, new ones are rounded once
        old = torch.ldexp(_to_tokens(codes, part, d), (was - e)[..., None, None])
        fresh = torch.where(torch.isnan(x), x, torch.ldexp(x, -e[..., None, None]).clamp(-448.0, 448.0))
        vals = torch.where(is_old, old, torch.where(is_new, fresh, 0.0))
        coded = _from_tokens(vals, part, d)
        # behind the last token of a block that held some before, bytes stay as they were
        keep = any_old[..., None, None] & ~is_old & ~is_new
        mask = _from_tokens(keep.float().expand_as(vals).contiguous(), part, d) != 0
        out.append(torch.where(mask, codes[..., part, :], coded))
        exps.append((e + 127).to(torch.uint8))
    st.codes[page, sub] = torch.stack(out, 2)
    st.scales[page, sub] = torch.stack(exps, 2)
    return dict(codes=st.codes.view(torch.float8_e4m3fn), scales=st.scales)


def _plain_attention(st):
    case = st.case
    d, hq, hkv, nb = case["d"], case["hq"], case["hkv"], st.page // BLOCK
    r, g = case["r"], hq // hkv
    starts, seq = st.starts.long(), st.seq.long()
    new = starts[1:] - starts[:-1]
    pages = st.table[:, : _pages(st.most, st.page)].clamp(min=0).long()
    codes, scales = st.codes[pages], st.scales[pages]  # [R, pages, NB, Hkv, 2, 64 D]
    size = torch.ldexp(torch.ones(scales.shape, device=codes.device), scales.to(torch.int32) - 127)
    kv = []
    for part in (0, 1):
        x = _to_tokens(codes, part, d).mul_(size[..., part, None, None])
        kv.append(x.permute(0, 3, 1, 2, 4, 5).reshape(r, hkv, -1, d))
    k, v = kv
    n = st.most_new
    i = torch.arange(n, device=codes.device)[None, :]
    src = (starts[:-1, None] + i).clamp(max=st.q.shape[0] - 1)
    q = st.q[src].float().view(r, n, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(r, hkv, g * n, d)
    s = torch.matmul(q, k.transpose(2, 3)).mul_(st.scale).view(r, hkv, g, n, -1)
    pos = (seq - new)[:, None] + i  # [R, n]
    at = torch.arange(k.shape[2], device=codes.device)
    seen = at <= pos[..., None]
    if st.window:
        seen = seen & (at > pos[..., None] - st.window)
    s = s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    if st.sink is not None:
        total = total + torch.exp(st.sink.view(1, hkv, g, 1, 1) - top)
    o = torch.matmul(p.view(r, hkv, g * n, -1), v).view(r, hkv, g, n, d) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(r, n, hq, d).to(torch.bfloat16)
    return o[i < new[:, None]]


# -------------------------------------------------------------------- work ---
def work(case) -> dict:
    old, new = _lengths(case)
    both = [a + b for a, b in zip(old, new)]
    page, r = case["page"], case["r"]
    if case["op"] == "step":
        tokens = sum(new) + case["pad"]
        fresh = sum(_pages(b, page) - _pages(a, page) for a, b in zip(old, both))
        # lengths and counts in, starts and both lengths out, pages popped and entered, two values a token
        return dict(bytes=4 * (2 * r + 3 * r + 2 + 2 * fresh + 2 * tokens), flops=0)
    if case["op"] == "trim":
        kept = _kept(case, old)
        back = sum(_pages(a, page) - _pages(b, page) for a, b in zip(old, kept))
        return dict(bytes=4 * (3 * r + 2 + 2 * back), flops=0)
    hkv, d = case["hkv"], case["d"]
    if case["op"] == "write":
        blocks = sum(_pages(b, BLOCK) - a // BLOCK for a, b in zip(old, both))
        values = 2 * sum(new) * hkv * d
        return dict(bytes=3 * values + 2 * 2 * blocks * hkv, flops=0)
    w = case["window"]
    pairs = read = 0
    for a, b in zip(old, both):
        lo = 0 if not w else max(0, a + 1 - w)
        read += b - lo
        n = b - a
        if not w:
            pairs += n * a + n * (n + 1) // 2
        else:  # position p sees min(p + 1, w) keys
            short = max(0, min(b, w) - a)
            pairs += sum(range(a + 1, a + short + 1)) + (n - short) * w
    return dict(bytes=2 * read * hkv * d + 4 * sum(new) * case["hq"] * d, flops=4 * pairs * case["hq"] * d)


# ------------------------------------------------------------------- exact ---
def exact(case, seed):
    if case["op"] in ("step", "trim"):
        return None  # whole numbers
    st = prepare(case, seed)
    d, hkv, nb = case["d"], case["hkv"], case["page"] // BLOCK
    old, new = _lengths(case)
    dev = "cuda"
    # the 256 values of e4m3: sign, 4 bits of exponent, 3 of fraction
    vals = []
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        v = f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7)
        v = math.nan if c & 127 == 127 else v
        vals.append(-v if c & 128 else v)
    grid = torch.tensor(vals, dtype=torch.float64, device=dev)
    t, c = torch.arange(BLOCK, device=dev)[:, None], torch.arange(d, device=dev)[None, :]
    at_k = (((t // 16) * (d // 64) + c // 64) * 64 + (c % 64) // 16 * 16 + t % 16) * 16 + c % 16
    at_v = ((c // 16) * 64 + (t % 16) // 4 * 16 + c % 16) * 16 + t // 16 * 4 + t % 4
    table = st.table.tolist()
    first = 0
    if case["op"] == "write":
        out = grid[st.codes.long()] if st.codes.numel() < 1 << 28 else None
        if out is None:
            return None
        scales = st.scales.cpu()
        for i in range(case["r"]):
            for b in range(old[i] // BLOCK, _pages(old[i] + new[i], BLOCK)):
                p, sub = table[i][b // nb], b % nb
                lo, hi = max(old[i], BLOCK * b), min(old[i] + new[i], BLOCK * (b + 1))
                had = max(0, min(old[i] - BLOCK * b, BLOCK))
                for part, (x, at) in enumerate(((st.k, at_k), (st.v, at_v))):
                    x = x[first + lo - old[i]:first + hi - old[i]].double().transpose(0, 1)  # [Hkv, m, D]
                    big = x.abs().amax((1, 2)).tolist()
                    e = [max(-126, math.ceil(math.log2(m / 448))) if m > 0 else -126 for m in big]
                    e = [z + 1 if m > 448 * 2.0 ** z else z - 1 if m <= 448 * 2.0 ** (z - 1) and z > -126 else z
                         for z, m in zip(e, big)]
                    was = [int(z) - 127 for z in scales[p, sub, :, part]]
                    e = [max(z, w) if had else z for z, w in zip(e, was)]
                    vs = torch.zeros(hkv, BLOCK, d, dtype=torch.float64, device=dev)
                    if had:
                        held = out[p, sub, :, part][:, at]
                        ratio = torch.tensor([2.0 ** (w - z) for z, w in zip(e, was)], dtype=torch.float64, device=dev)
                        vs = held.clone()
                        vs[:, :had] = held[:, :had] * ratio[:, None, None]
                    size = torch.tensor([2.0 ** z for z in e], dtype=torch.float64, device=dev)
                    vs[:, lo - BLOCK * b:hi - BLOCK * b] = x / size[:, None, None]
                    # the nearest value of the grid, ties to the even fraction
                    a = vs.abs().clamp(max=448.0)
                    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
                    vs = torch.where(torch.isnan(vs), vs, torch.round(a / step) * step * torch.sign(vs))
                    out[p, sub, :, part, :][:, at.reshape(-1)] = vs.reshape(hkv, -1)
            first += new[i]
        return dict(codes=out, scales=None)
    g = case["hq"] // hkv
    o = torch.zeros(st.q.shape, dtype=torch.float64, device=dev)
    for i in range(case["r"]):
        a, n = old[i], new[i]
        length = a + n
        ids = torch.tensor(table[i][: _pages(length, st.page)], device=dev)
        pos = a + torch.arange(n, device=dev)
        seen = torch.arange(length, device=dev)[None, :] <= pos[:, None]
        if st.window:
            seen &= torch.arange(length, device=dev)[None, :] > pos[:, None] - st.window
        for h in range(hkv):
            sc = torch.exp2(st.scales[ids][:, :, h].double() - 127)
            by = st.codes[ids][:, :, h] if ids.numel() * nb * hkv * d < 1 << 26 else torch.stack(
                [st.codes[j, :, h] for j in ids.tolist()])
            k = (grid[by[:, :, 0][:, :, at_k].long()] * sc[:, :, 0, None, None]).view(-1, d)[:length]
            v = (grid[by[:, :, 1][:, :, at_v].long()] * sc[:, :, 1, None, None]).view(-1, d)[:length]
            for m in range(h * g, (h + 1) * g):
                s = st.q[first:first + n, m].double() @ k.T * st.scale
                s = s.masked_fill(~seen, -math.inf)
                most = s.amax(1, keepdim=True)
                p = torch.exp(s - most)
                under = p.sum(1, keepdim=True)
                if st.sink is not None:
                    under = under + torch.exp(st.sink[m].double() - most)
                o[first:first + n, m] = p @ v / under
        first += n
    return o
