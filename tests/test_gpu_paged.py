"""The paged 8-bit KV cache on the GPU against the oracle: tables, slots, codes and scales bit for bit,
attention within the bound that ``oracle.paged.attention`` derives, and the parts together."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import codecs as C
from oracle import paged as P

pytestmark = pytest.mark.gpu


def _i32(a, dev):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)


def _bf16(rng, *shape):
    return C.round_bf16(rng.standard_normal(shape).astype(np.float32))


def _pool(rng, lengths, after, page, spare):
    """Tables [R, B] that hold `lengths` tokens of requests that grow to `after`, and a stack of free pages."""
    held = [-(-max(int(x), 0) // page) for x in lengths]
    fresh = sum(-(-max(int(b), 0) // page) for b in after) - sum(held)
    total = sum(held) + max(fresh, 0) + spare
    ids = rng.permutation(total).astype(np.int32)
    width = max(1, max(-(-max(int(b), 0) // page) for b in after)) + 1
    table = rng.integers(-5, 5, (len(lengths), width)).astype(np.int32)  # behind the last page: anything
    at = 0
    for i, n in enumerate(held):
        table[i, :n] = ids[at:at + n]
        at += n
    free = np.full(total, -9, np.int32)
    free[:total - at] = ids[at:]
    return table, free, total - at, total


# ----------------------------------------------------------- step, trim ----
@pytest.mark.parametrize("r,most,n,page,pad,dry,allocate", [
    (1, 1, 1, 64, 0, False, True), (1, 0, 1, 64, 3, False, True), (16, 500, 1, 64, 0, False, True),
    (7, 300, 200, 128, 5, False, True), (64, 1000, 3, 192, 0, True, True), (1024, 200, 2, 64, 1, False, True),
    (1025, 200, 5, 64, 0, True, True), (2500, 90, 20, 64, 77, False, True), (3, 5000, 4000, 64, 0, False, True),
    (300, 64, 130, 64, 0, True, True), (40, 400, 60, 256, 2, False, False), (5, 70, 0, 64, 4, False, True),
    (256, 300, 40, 64, 9, False, True), (257, 300, 40, 64, 0, True, True), (2048, 130, 3, 64, 0, False, True),
    (2049, 130, 3, 64, 2, True, True), (4500, 70, 2, 64, 1, False, True)])
def test_step(dev, r, most, n, page, pad, dry, allocate):
    from mosaic_amd import ops
    rng = np.random.default_rng(r + most + n)
    lengths = rng.integers(0, most + 1, r).astype(np.int32)
    new = rng.integers(0, n + 1, r).astype(np.int32)
    if r > 4:
        lengths[3], new[2] = -5, -2  # read as nothing
    after = np.maximum(lengths, 0) + np.maximum(new, 0)
    table, free, count, total = _pool(rng, lengths if allocate else after, after, page, 3)
    if dry:
        count = count // 2
    tokens = int(np.maximum(new, 0).sum()) + pad
    t = _i32(table, dev)
    args = dict(free_pages=_i32(free, dev), free_count=_i32([count], dev)) if allocate else {}
    lt, nt = _i32(lengths, dev), _i32(new, dev)
    s = ops.paged_step(lt, nt, t, tokens, page, **args)
    want = P.step(lengths, new, table, tokens, page, free if allocate else None, count if allocate else 0)
    for name, x in want.items():
        np.testing.assert_array_equal(getattr(s, name).cpu().numpy(), x, err_msg=name)
    np.testing.assert_array_equal(t.cpu().numpy(), table)
    np.testing.assert_array_equal(lt.cpu().numpy(), lengths)
    if dry:
        assert (want["seq_lens"] == 0).any() and int(want["free_count"][0]) >= 0


def test_step_rows_and_tables_that_do_not_suffice(dev):
    from mosaic_amd import ops
    rng = np.random.default_rng(5)
    lengths, new = np.array([10, 64, 100, 0, 3], np.int32), np.array([5, 200, 2 ** 30, 7, 1], np.int32)
    table, free, count, _ = _pool(rng, lengths, lengths + 70, 64, 9)
    for tokens in (0, 4, 5, 300, 205 + (1 << 20)):
        tb = table.copy()
        t = _i32(tb, dev)
        s = ops.paged_step(_i32(lengths, dev), _i32(new, dev), t, tokens, 64, _i32(free, dev), _i32([count], dev))
        want = P.step(lengths, new, tb, tokens, 64, free, count)
        for name, x in want.items():
            np.testing.assert_array_equal(getattr(s, name).cpu().numpy(), x, err_msg=f"{tokens} {name}")
        np.testing.assert_array_equal(t.cpu().numpy(), tb)


@pytest.mark.parametrize("r", [2048, 2100, 4096])
def test_step_counts_past_the_most_rows(dev, r):
    """The most rows there may be, and counts whose sum passes 32 bits: after the first that does not fit, none does."""
    from mosaic_amd import ops
    lengths, new = np.zeros(r, np.int32), np.full(r, 2 ** 30, np.int32)
    new[:3] = 5, 0, 7
    table, free, count, _ = _pool(np.random.default_rng(6), lengths, lengths + 1, 64, 9)
    tokens, t = 2 ** 21 - 1, _i32(table, dev)
    s = ops.paged_step(_i32(lengths, dev), _i32(new, dev), t, tokens, 64, _i32(free, dev), _i32([count], dev))
    want = P.step(lengths, new, table, tokens, 64, free, count)
    for name, x in want.items():
        np.testing.assert_array_equal(getattr(s, name).cpu().numpy(), x, err_msg=name)
    np.testing.assert_array_equal(t.cpu().numpy(), table)


def test_step_without_requests(dev):
    from mosaic_amd import ops
    s = ops.paged_step(_i32([], dev), _i32([], dev), torch.zeros(0, 3, dtype=torch.int32, device=dev), 5, 64,
                       _i32([4, 2], dev), _i32([2], dev))
    assert s.starts.tolist() == [0] and s.positions.tolist() == [-1] * 5 and s.free_count.tolist() == [2]


@pytest.mark.parametrize("r,most,page", [(1, 500, 64), (33, 2000, 64), (1024, 300, 128), (1030, 700, 64), (2100, 64, 64), (256, 900, 64), (257, 900, 64),
                                         (2048, 200, 64), (4100, 100, 64)])
def test_trim(dev, r, most, page):
    from mosaic_amd import ops
    rng = np.random.default_rng(r)
    lengths = rng.integers(0, most + 1, r).astype(np.int32)
    keep = np.where(rng.random(r) < 0.3, 0, lengths - rng.integers(-3, 70, r)).astype(np.int32)
    table, free, count, total = _pool(rng, lengths, lengths, page, 4)
    t, f = _i32(table, dev), _i32(free, dev)
    kept, left = ops.paged_trim(_i32(lengths, dev), _i32(keep, dev), t, page, f, _i32([count], dev))
    want, n = P.trim(lengths, keep, table, page, free, count)
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    np.testing.assert_array_equal(f.cpu().numpy(), free)
    assert left.tolist() == [n]
    np.testing.assert_array_equal(t.cpu().numpy(), table)


def test_trim_onto_a_full_stack_writes_nothing_past_it(dev):
    from mosaic_amd import ops
    f = torch.arange(6, dtype=torch.int32, device=dev)
    guard = f.clone()
    kept, left = ops.paged_trim(_i32([300], dev), _i32([0], dev), _i32([[1, 2, 3, 4, 5]], dev), 64, f[:3], _i32([2], dev))
    assert kept.tolist() == [0] and left.tolist() == [3]
    assert f.tolist() == guard[:2].tolist() + [5] + guard[3:].tolist()


# ---------------------------------------------------------------- write ----
def _cache(rng, total, nb, hkv, d):
    codes = rng.integers(0, 256, (total, nb, hkv, 2, 64 * d)).astype(np.uint8)
    codes[(codes & 0x7F) == 0x7F] = 0x30
    return codes, rng.integers(118, 124, (total, nb, hkv, 2)).astype(np.uint8)


def _batch(rng, held, new, page, spare=2):
    held, new = np.array(held), np.array(new)
    seq = held + new
    table, _, _, total = _pool(rng, seq, seq, page, spare)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    return table, total, starts, seq.astype(np.int32)


def _same_codes(got, want):
    """Equal bytes; a NaN's sign is free."""
    nan = (want & 0x7F) == 0x7F
    np.testing.assert_array_equal((got & 0x7F)[nan], want[nan] & 0x7F)
    np.testing.assert_array_equal(got[~nan], want[~nan])


@pytest.mark.parametrize("hkv,d,page,held,new", [
    (1, 64, 64, [0], [1]), (2, 128, 64, [0, 5, 63, 64, 65], [1, 1, 1, 1, 1]), (8, 128, 64, [0, 10], [64, 128]),
    (3, 64, 128, [7, 0, 100, 130], [150, 3, 28, 0]), (2, 256, 192, [190, 1], [5, 300]), (4, 128, 256, [0], [700]),
    (5, 64, 64, list(range(0, 300)), [2] * 300)])
def test_write(dev, hkv, d, page, held, new):
    from mosaic_amd import ops
    rng = np.random.default_rng(hkv * d + len(held))
    table, total, starts, seq = _batch(rng, held, new, page)
    codes, scales = _cache(rng, total, page // 64, hkv, d)
    t = int(starts[-1]) + 3  # rows behind the last request are not read
    k, v = _bf16(rng, t, hkv, d) * 2.0 ** rng.integers(-8, 5, (t, 1, 1)), _bf16(rng, t, hkv, d) * 0.01
    k[int(starts[-1]):] = np.nan
    kv = torch.from_numpy(np.concatenate([k, v], 1).astype(np.float32)).to(dev).to(torch.bfloat16)
    ct, st = torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev)
    ops.paged_kv_write(kv[:, :hkv], kv[:, hkv:], ct, st, _i32(table, dev), _i32(starts, dev), _i32(seq, dev))
    x = kv.double().cpu().numpy()  # the oracle gets the bf16 values that the call gets
    P.write(x[:, :hkv], x[:, hkv:], codes, scales, table, starts, seq)
    np.testing.assert_array_equal(st.cpu().numpy(), scales)
    _same_codes(ct.cpu().numpy(), codes)


def test_write_extremes(dev):
    """Zeros, bf16's smallest and largest, infinities and NaN; a scale that grows by one and by many powers."""
    from mosaic_amd import ops
    rng = np.random.default_rng(8)
    hkv, d = 6, 64
    table, total, starts, seq = _batch(rng, [0, 20, 40], [70, 9, 2], 64)
    codes, scales = _cache(rng, total, 1, hkv, d)
    t = int(starts[-1])
    k = _bf16(rng, t, hkv, d).astype(np.float64)
    k[:, 0] = 0.0
    k[:, 1] *= 2.0 ** -130
    k[:, 2] *= 2.0 ** 120
    k[::3, 3, ::5], k[1::3, 3, ::7], k[2::3, 3, ::9] = np.inf, -np.inf, np.nan
    k[:, 4] = np.inf
    k[:, 5, :] = 448.0 * 2.0 ** 3
    k = C.round_bf16(k.astype(np.float32)).astype(np.float64)
    scales[:, :, 0] = 1
    codes[:, 0, 3, 1, ::11] = 0xFF
    x = torch.from_numpy(k.astype(np.float32)).to(dev).to(torch.bfloat16)
    ct, st = torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev)
    ops.paged_kv_write(x, x, ct, st, _i32(table, dev), _i32(starts, dev), _i32(seq, dev))
    P.write(k, k, codes, scales, table, starts, seq)
    np.testing.assert_array_equal(st.cpu().numpy(), scales)
    _same_codes(ct.cpu().numpy(), codes)


def test_write_skips_what_is_not_placed(dev):
    """Requests with seq_lens 0, pages outside the pool and starts outside the rows change nothing."""
    from mosaic_amd import ops
    rng = np.random.default_rng(9)
    codes, scales = _cache(rng, 4, 1, 2, 64)
    x = torch.from_numpy(_bf16(rng, 30, 2, 64)).to(dev).to(torch.bfloat16)
    ct, st = torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev)
    table = _i32([[0, 1], [4, -1], [2, 3], [3, 3]], dev)
    ops.paged_kv_write(x, x, ct, st, table, _i32([0, 10, 20, 20, 20], dev), _i32([0, 10, 50, 7], dev))
    ops.paged_kv_write(x, x, ct, st, table, _i32([30, 40, 100, 2 ** 31 - 1, 2 ** 31 - 1], dev), _i32([64, 128, 128, 64], dev))
    np.testing.assert_array_equal(ct.cpu().numpy(), codes)
    np.testing.assert_array_equal(st.cpu().numpy(), scales)


# ------------------------------------------------------------ attention ----
def _attention_case(dev, rng, hq, hkv, d, page, held, new, window=0, sink=False, pad=0, max_new=None, codes=None,
                    change=None, scale=None):
    from mosaic_amd import ops
    table, total, starts, seq = _batch(rng, held, new, page)
    c, s = _cache(rng, total, page // 64, hkv, d)
    if change is not None:
        change(c, s, table, seq, starts)
    t = int(starts[-1]) + pad
    q = _bf16(rng, t, hq, d)
    snk = rng.standard_normal(hq).astype(np.float32) if sink else None
    scale = d ** -0.5 if scale is None else scale
    qt = torch.from_numpy(q).to(dev).to(torch.bfloat16)
    out = torch.full((t, hq, d), float("nan"), dtype=torch.bfloat16, device=dev)
    got = ops.paged_attention(qt, torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev), _i32(table, dev),
                              _i32(starts, dev), _i32(seq, dev), scale,
                              sink=None if snk is None else torch.from_numpy(snk).to(dev), window=window,
                              max_new=max_new, out=out)
    assert got.data_ptr() == out.data_ptr()
    want, tol = P.attention(q.astype(np.float64), c, s, table, starts, seq, scale, snk, window)
    o = out.float().cpu().numpy().astype(np.float64)
    np.testing.assert_array_equal(np.isnan(o), np.isnan(want))
    bad = ~(np.abs(o - want) <= tol) & ~np.isnan(want)
    assert not bad.any(), f"{bad.sum()} values off, worst {np.nanmax(np.abs(o - want) / np.maximum(tol, 1e-30))} of the bound"


@pytest.mark.parametrize("hq,hkv,d,page,held,new,window,sink", [
    (1, 1, 64, 64, [0], [1], 0, False),                       # one token alone
    (8, 1, 128, 64, [0, 1, 62, 63, 64, 500], [1] * 6, 0, False),
    (64, 8, 128, 64, [516], [1], 0, True),
    (16, 2, 128, 128, [2000, 3, 127, 128], [1] * 4, 0, True),
    (14, 2, 64, 64, [300, 20], [1, 1], 100, False),           # seven heads a key head
    (6, 6, 64, 192, [700, 10, 0], [1, 1, 1], 64, True),       # a key head each
    (32, 2, 256, 64, [130, 999], [1, 1], 0, False),           # sixteen heads a key head
    (40, 2, 128, 64, [150], [1], 0, False),                   # twenty: two tiles
    (16, 2, 128, 64, [100, 0, 37, 700], [4, 2, 0, 3], 0, True),      # drafts, a resting request
    (16, 2, 128, 64, [100, 0, 37], [4, 2, 3], 5, False),
    (8, 2, 64, 64, [0], [200], 0, False),                     # a prompt
    (8, 2, 128, 64, [0, 70, 5], [130, 1, 65], 0, True),       # pieces of prompts and a decode step
    (8, 1, 256, 128, [60], [150], 33, True),
    (4, 4, 64, 64, [0, 200], [129, 70], 128, False)])
def test_attention(dev, hq, hkv, d, page, held, new, window, sink):
    rng = np.random.default_rng(hq + d + len(held) + window)
    _attention_case(dev, rng, hq, hkv, d, page, held, new, window, sink, max_new=max(new))
    _attention_case(dev, rng, hq, hkv, d, page, held, new, window, sink, pad=3)


def test_attention_long_context(dev):
    """Few rows over a long axis: cut among all workgroups and joined."""
    rng = np.random.default_rng(11)
    _attention_case(dev, rng, 8, 1, 128, 64, [40000], [1], sink=True)
    _attention_case(dev, rng, 4, 2, 64, 256, [30001, 5, 12345], [1, 2, 1])


@pytest.mark.parametrize("hq,hkv,d,page,held,new,window", [
    (8, 1, 128, 64, [3000, 40, 0], [100, 1, 17], 0), (16, 2, 64, 128, [5000], [60], 0), (4, 4, 256, 64, [2000], [33], 0),
    (6, 2, 128, 64, [1500, 1500], [40, 90], 700), (16, 1, 64, 64, [4000], [2], 0), (4, 1, 64, 64, [4000], [260], 2000)])
def test_attention_pieces_behind_long_contexts(dev, hq, hkv, d, page, held, new, window):
    """Few tiles of many rows over a long axis: each is cut among workgroups and joined."""
    _attention_case(dev, np.random.default_rng(d + len(held)), hq, hkv, d, page, held, new, window, sink=True)


def test_attention_row_whose_piece_is_empty(dev):
    """A window that leaves whole pieces of a cut tile without keys for some of its rows."""
    _attention_case(dev, np.random.default_rng(30), 4, 1, 64, 64, [2500], [260], window=30)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_attention_scales(dev, scale):
    for new in ([1, 3], [90, 1]):
        _attention_case(dev, np.random.default_rng(31), 4, 2, 64, 64, [100, 20], new, scale=scale)


def test_attention_queries_of_unequal_size(dev):
    """Rows from 2^-60 to 2^20 of the others, dims within a row over 2^16, rows of zeros."""
    from mosaic_amd import ops
    rng = np.random.default_rng(32)
    table, total, starts, seq = _batch(rng, [70], [60], 64)
    c, s = _cache(rng, total, 1, 2, 64)
    q = _bf16(rng, 60, 4, 64) * np.exp2(rng.integers(-16, 1, (60, 4, 64)))
    q[::7] *= 2.0 ** -60
    q[3::7] *= 2.0 ** 20
    q[5, 1] = 0.0
    q = C.round_bf16(q.astype(np.float32))
    o = ops.paged_attention(torch.from_numpy(q).to(dev).to(torch.bfloat16), torch.from_numpy(c).to(dev),
                            torch.from_numpy(s).to(dev), _i32(table, dev), _i32(starts, dev), _i32(seq, dev), 2.0 ** -6)
    want, tol = P.attention(q.astype(np.float64), c, s, table, starts, seq, 2.0 ** -6)
    assert np.all(np.abs(o.float().cpu().numpy() - want) <= tol)


def test_attention_many_short_requests(dev):
    rng = np.random.default_rng(12)
    held = rng.integers(0, 200, 700)
    _attention_case(dev, rng, 4, 1, 64, 64, held, rng.integers(0, 3, 700), pad=2)


@pytest.mark.parametrize("hq,hkv,d,r,most,window", [(8, 8, 128, 40, 700, 0), (16, 8, 64, 70, 900, 100), (6, 6, 256, 50, 300, 0),
                                                     (16, 4, 128, 70, 1500, 0), (16, 4, 128, 30, 2500, 600)])
def test_attention_more_tiles_than_workgroups(dev, hq, hkv, d, r, most, window):
    """Whole and cut tiles, several of a workgroup's, of unequal lengths; resting requests and drafts among them."""
    rng = np.random.default_rng(36 + r)
    _attention_case(dev, rng, hq, hkv, d, 64, rng.integers(0, most, r), rng.integers(0, 4, r), window, sink=True, max_new=3, pad=2)


def test_attention_scale_bytes(dev):
    """The least and largest scales that the writer makes of bf16 values near its range's ends, mixed in one row."""
    def change(c, s, table, seq, starts):
        s[..., 0] = 100  # small keys: flat scores
        s[table[0, 0], :, :, 1] = 20
        s[table[0, 1], :, :, 1] = 200
        s[table[0, 2], :, :, 1] = 127
    _attention_case(dev, np.random.default_rng(13), 8, 2, 128, 64, [180], [3], change=change)


def test_attention_does_not_read_behind_a_request(dev):
    """NaN codes behind the last token and before a window, NaN scales and pages of no pool that no row sees."""
    def change(c, s, table, seq, starts):
        for i in range(len(seq)):
            at_k, at_v = P.block_maps(64)
            lo = max(0, int(seq[i]) - 1 - 99 - 64)
            for b in range(-(-int(seq[i]) // 64)):
                for tok in range(64):
                    p = 64 * b + tok
                    if p >= seq[i] or p < int(seq[i]) - (int(starts[i + 1]) - int(starts[i])) - 99:
                        c[table[i, b], 0, :, 0][:, at_k[tok]] = 0x7F
                        c[table[i, b], 0, :, 1][:, at_v[tok]] = 0xFF
            for b in range(lo // 64):
                s[table[i, b]] = 255
                table[i, b] = [-1, 1 << 30][b % 2]
    _attention_case(dev, np.random.default_rng(14), 8, 2, 64, 64, [300, 10, 700, 500], [1, 1, 3, 100], window=100,
                    sink=True, change=change)


def test_attention_nan_reaches_only_rows_that_see_it(dev):
    """NaN keys and values of tokens in the middle of the new ones: earlier rows stay numbers, each dim by itself."""
    def change(c, s, table, seq, starts):
        at_k, at_v = P.block_maps(64)
        c[table[0, 0], 0, 0, 1, at_v[40, 5:7]] = 0x7F
        c[table[0, 0], 0, 1, 0, at_k[50, 9]] = 0xFF
        s[table[0, 2], 0, 1, 1] = 255
        s[table[1, 0], 0, 0, 0] = 255
    _attention_case(dev, np.random.default_rng(15), 4, 2, 64, 64, [30, 20], [150, 30], change=change)


def test_attention_pages_outside_the_pool_hold_no_keys(dev):
    def change(c, s, table, seq, starts):
        table[0, 1], table[1, 0], table[2, :] = -1, c.shape[0], -7
    _attention_case(dev, np.random.default_rng(16), 8, 2, 128, 64, [200, 30, 100], [2, 40, 1], sink=True, change=change)


def test_attention_unplaced_requests_give_zeros(dev):
    from mosaic_amd import ops
    rng = np.random.default_rng(17)
    c, s = _cache(rng, 3, 1, 1, 64)
    q = torch.from_numpy(_bf16(rng, 6, 2, 64)).to(dev).to(torch.bfloat16)
    out = torch.full_like(q, float("nan"))
    o = ops.paged_attention(q, torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev), _i32([[0], [1], [2]], dev),
                            _i32([0, 2, 3, 4], dev), _i32([0, 9, 0], dev), 0.125,
                            sink=torch.zeros(2, device=dev), out=out)
    assert not o[[0, 1, 3, 4, 5]].any() and o[2].abs().max() > 0


@pytest.mark.parametrize("new", [[1, 2, 1], [90, 1, 40]])
def test_attention_of_requests_that_share_a_prefix(dev, new):
    def change(c, s, table, seq, starts):
        table[1:, :3] = table[0, :3]
    _attention_case(dev, np.random.default_rng(33), 8, 2, 128, 64, [200, 300, 192], new, change=change)


def test_calls_without_rows(dev):
    """A step in which every request rests: nothing is read or written."""
    from mosaic_amd import ops
    rng = np.random.default_rng(34)
    c, s = _cache(rng, 4, 1, 2, 64)
    ct, st = torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev)
    x = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=dev)
    for r in (0, 3):
        table, starts, seq = _i32(np.zeros((r, 2)), dev), _i32(np.zeros(r + 1), dev), _i32(np.full(r, 70), dev)
        ops.paged_kv_write(x, x, ct, st, table, starts, seq)
        assert ops.paged_attention(x, ct, st, table, starts, seq, 0.125).shape == (0, 2, 64)
    np.testing.assert_array_equal(ct.cpu().numpy(), c)
    np.testing.assert_array_equal(st.cpu().numpy(), s)


def test_tables_of_one_page(dev):
    """A column of a table turned on its side: the stride within a row of one entry does not matter."""
    from mosaic_amd import ops
    rng = np.random.default_rng(35)
    c, s = (torch.from_numpy(x).to(dev) for x in _cache(rng, 4, 1, 2, 64))
    q = torch.from_numpy(_bf16(rng, 3, 2, 64)).to(dev).to(torch.bfloat16)
    table, starts, seq = _i32([[2], [0], [3]], dev), _i32([0, 1, 2, 3], dev), _i32([5, 64, 1], dev)
    want = ops.paged_attention(q, c, s, table, starts, seq, 0.125)
    turned = _i32([[2, 0, 3]], dev).t()
    assert turned.stride() == (1, 3)
    assert torch.equal(ops.paged_attention(q, c, s, turned, starts, seq, 0.125), want)


def test_attention_without_requests_clears_its_rows(dev):
    from mosaic_amd import ops
    c, s = _cache(np.random.default_rng(33), 2, 1, 1, 64)
    for t, hq in ((1, 1), (3, 8), (300, 4)):
        q = torch.ones(t, hq, 64, dtype=torch.bfloat16, device=dev)
        out = torch.full_like(q, float("nan"))
        ops.paged_attention(q, torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev),
                            torch.zeros(0, 3, dtype=torch.int32, device=dev), _i32([0], dev), _i32([], dev), 1.0, out=out)
        assert not out.any()


@pytest.mark.parametrize("max_new", [1, 2, 500])
def test_attention_holds_with_a_wrong_max_new(dev, max_new):
    """max_new sizes the launches only: requests of more rows than it says are done all the same."""
    _attention_case(dev, np.random.default_rng(34), 8, 2, 64, 64, [1500, 40, 0], [3, 70, 12], max_new=max_new, pad=1)


@pytest.mark.parametrize("window", [1, 64, 2 ** 30 - 1, 2 ** 31 - 1])
def test_attention_windows(dev, window):
    _attention_case(dev, np.random.default_rng(35), 4, 2, 64, 64, [130, 0], [1, 90], window=window)


def test_attention_starts_outside_the_rows(dev):
    """Starts that pass the rows are cut: no row outside is read or written."""
    from mosaic_amd import ops
    rng = np.random.default_rng(18)
    c, s = _cache(rng, 3, 1, 1, 64)
    q = torch.from_numpy(_bf16(rng, 8, 2, 64)).to(dev).to(torch.bfloat16)
    buf = torch.full((10, 2, 64), 7.0, dtype=torch.bfloat16, device=dev)
    for starts in ([0, 100, 200, 300], [-5, 3, 1, 2 ** 31 - 1], [9, 9, 9, 9]):
        ops.paged_attention(q, torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev), _i32([[0], [1], [2]], dev),
                            _i32(starts, dev), _i32([64, 9, 2 ** 31 - 1], dev), 0.125, out=buf[1:9])
        assert (buf[0] == 7).all() and (buf[9] == 7).all()


def test_attention_strided_and_unaligned_q(dev):
    from mosaic_amd import ops
    rng = np.random.default_rng(19)
    table, total, starts, seq = _batch(rng, [70, 3], [1, 5], 64)
    c, s = (torch.from_numpy(x).to(dev) for x in _cache(rng, total, 1, 2, 64))
    qkv = torch.from_numpy(_bf16(rng, 6, 8 * 64 + 8)).to(dev).to(torch.bfloat16)
    args = (c, s, _i32(table, dev), _i32(starts, dev), _i32(seq, dev), 0.125)
    for q in (qkv[:, :256].view(6, 4, 64), qkv[:, 8:264].view(6, 4, 64), qkv[:, 3:259].view(6, 4, 64),
              qkv[:, :512].view(6, 8, 64)[:, ::2], qkv[:, :256].reshape(6, 64, 4).transpose(1, 2)):
        assert torch.equal(ops.paged_attention(q, *args), ops.paged_attention(q.clone(memory_format=torch.contiguous_format), *args))
    wide = torch.full((2, 50), -1, dtype=torch.int32, device=dev)
    wide[:, 3:3 + table.shape[1]] = _i32(table, dev)
    cut = wide[:, 3:3 + table.shape[1]]
    q = qkv[:, :256].view(6, 4, 64)
    assert torch.equal(ops.paged_attention(q, c, s, cut, *args[3:]), ops.paged_attention(q, *args))


def test_attention_repeats_its_bits(dev):
    from mosaic_amd import ops
    rng = np.random.default_rng(20)
    table, total, starts, seq = _batch(rng, [3000, 3, 900], [1, 2, 300], 64)
    c, s = (torch.from_numpy(x).to(dev) for x in _cache(rng, total, 1, 2, 128))
    q = torch.from_numpy(_bf16(rng, 303, 8, 128)).to(dev).to(torch.bfloat16)
    ws = ops.MoEWorkspace()
    args = (q, c, s, _i32(table, dev), _i32(starts, dev), _i32(seq, dev), 0.1)
    first = ops.paged_attention(*args)
    for _ in range(5):
        assert torch.equal(ops.paged_attention(*args, workspace=ws), first)


def test_codes_past_32_bits(dev):
    """A pool of more than 4 GiB: its last pages are written and read at their own place."""
    from mosaic_amd import ops
    rng = np.random.default_rng(21)
    hkv, d = 8, 256
    pages = (1 << 32) // (hkv * 2 * 64 * d) + 40
    codes = torch.zeros(pages, 1, hkv, 2, 64 * d, dtype=torch.uint8, device=dev)
    scales = torch.full((pages, 1, hkv, 2), 127, dtype=torch.uint8, device=dev)
    k, v = (torch.from_numpy(_bf16(rng, 90, hkv, d)).to(dev).to(torch.bfloat16) for _ in range(2))
    q = torch.from_numpy(_bf16(rng, 90, hkv, d)).to(dev).to(torch.bfloat16)
    outs = []
    for ids in ([pages - 1, pages - 30], [0, 1]):
        table = _i32([ids], dev)
        st, sq = _i32([0, 90], dev), _i32([90], dev)
        ops.paged_kv_write(k, v, codes, scales, table, st, sq)
        outs.append(ops.paged_attention(q, codes, scales, table, st, sq, d ** -0.5))
    assert torch.equal(*outs)
    assert torch.equal(codes[pages - 1], codes[0]) and torch.equal(codes[pages - 30], codes[1])
    assert not codes[2:pages - 30].any() and not codes[pages - 29:pages - 1].any()


# ------------------------------------------------------------- together ----
class _Model:
    """The cache's parts together, in the oracle."""

    def __init__(self, pages, hkv, d, r, most, page, layers):
        self.page = page
        self.codes = np.zeros((layers, pages, page // 64, hkv, 2, 64 * d), np.uint8)
        self.scales = np.full((layers, pages, page // 64, hkv, 2), 127, np.uint8)
        self.table = np.full((r, -(-most // page)), -1, np.int32)
        self.free, self.count = np.arange(pages - 1, -1, -1).astype(np.int32), pages
        self.lengths = np.zeros(r, np.int32)

    def step(self, new, tokens):
        s = P.step(self.lengths, new, self.table, tokens, self.page, self.free, self.count)
        self.lengths, self.count = s["lengths"], int(s["free_count"][0])
        return s

    def trim(self, keep):
        self.lengths, self.count = P.trim(self.lengths, keep, self.table, self.page, self.free, self.count)


def test_serving_run(dev):
    """Prompts, decode steps, drafts that are rejected, requests that end and begin, a pool that runs dry."""
    from mosaic_amd.kernels.paged import PagedKVCache
    rng = np.random.default_rng(22)
    r, hq, hkv, d, page, layers, pages, most = 5, 8, 2, 64, 64, 2, 14, 400
    cache = PagedKVCache(pages, hkv, d, r, most, page, layers, dev)
    model = _Model(pages, hkv, d, r, most, page, layers)
    sink = rng.standard_normal(hq).astype(np.float32)
    plan = [([130, 5, 0, 64, 1], None), ([1, 1, 70, 1, 1], None), ([4, 4, 4, 4, 4], [133, 8, 73, 66, 4]),
            ([1, 1, 1, 1, 1], [0, 9, 74, 67, 0]), ([200, 1, 1, 1, 33], None), ([1, 300, 1, 400, 90], None),
            ([1, 1, 1, 1, 1], [0, 0, 0, 0, 0]), ([63, 64, 65, 1, 2], None)]
    refused = 0
    for new, keep in plan:
        tokens = sum(new) + 2
        s = cache.step(_i32(new, dev), tokens)
        w = model.step(np.array(new), tokens)
        for name, x in w.items():
            np.testing.assert_array_equal(getattr(s, name).cpu().numpy(), x, err_msg=name)
        refused += int(((w["seq_lens"] == 0) & (np.array(new) > 0)).sum())
        for layer in range(layers):
            q, k, v = _bf16(rng, tokens, hq, d), _bf16(rng, tokens, hkv, d), _bf16(rng, tokens, hkv, d)
            t = [torch.from_numpy(x).to(dev).to(torch.bfloat16) for x in (q, k, v)]
            o = cache.update(s, *t, 0.125, sink=torch.from_numpy(sink).to(dev), layer=layer,
                             max_new=max(new)).float().cpu().numpy()
            P.write(k.astype(np.float64), v.astype(np.float64), model.codes[layer], model.scales[layer], model.table,
                    w["starts"], w["seq_lens"])
            np.testing.assert_array_equal(cache.scales[layer].cpu().numpy(), model.scales[layer])
            np.testing.assert_array_equal(cache.codes[layer].cpu().numpy(), model.codes[layer])
            want, tol = P.attention(q.astype(np.float64), model.codes[layer], model.scales[layer], model.table,
                                    w["starts"], w["seq_lens"], 0.125, sink)
            assert np.all(np.abs(o - want) <= tol)
        if keep is not None:
            cache.trim(_i32(keep, dev))
            model.trim(np.array(keep))
        np.testing.assert_array_equal(cache.lengths.cpu().numpy(), model.lengths)
        assert cache.free_count.tolist() == [model.count]
        np.testing.assert_array_equal(cache.free_pages.cpu().numpy()[:model.count], model.free[:model.count])
    assert refused


def test_decode_steps_in_a_graph(dev):
    """A captured decode step (tables, write, attention, commit), replayed beside the same steps run eagerly."""
    from mosaic_amd import ops
    from mosaic_amd.kernels.paged import PagedKVCache
    rng = np.random.default_rng(23)
    r, hq, hkv, d = 3, 8, 2, 64
    caches = [PagedKVCache(20, hkv, d, r, 300, device=dev) for _ in range(2)]
    first = _i32([60, 1, 127], dev)
    prompt = [torch.from_numpy(_bf16(rng, 188, h, d)).to(dev).to(torch.bfloat16) for h in (hq, hkv, hkv)]
    for c in caches:
        c.update(c.step(first, 188), *prompt, 0.125)
    one = torch.ones(r, dtype=torch.int32, device=dev)
    x = [torch.zeros(r, h, d, dtype=torch.bfloat16, device=dev) for h in (hq, hkv, hkv)]
    ws = ops.MoEWorkspace()
    out = ops.PagedStep.empty(r, r, dev)
    state = [t.clone() for t in (caches[0].codes, caches[0].scales, caches[0].block_table, caches[0].lengths, caches[0].free_count)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):  # the library and workspace are warm
        caches[0].update(caches[0].step(one, r, out), *x, 0.125, max_new=1, workspace=ws)
    stream.synchronize()
    for t, was in zip((caches[0].codes, caches[0].scales, caches[0].block_table, caches[0].lengths, caches[0].free_count), state):
        t.copy_(was)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = caches[0].update(caches[0].step(one, r, out), *x, 0.125, max_new=1, workspace=ws)
    for i in range(8):
        for t in x:
            t.copy_(torch.from_numpy(_bf16(rng, *t.shape)).to(dev))
        graph.replay()
        torch.cuda.synchronize()
        want = caches[1].update(caches[1].step(one, r), *x, 0.125, max_new=1)
        assert torch.equal(o, want), i
        assert torch.equal(caches[0].codes, caches[1].codes) and torch.equal(caches[0].lengths, caches[1].lengths)
        assert torch.equal(caches[0].block_table, caches[1].block_table)


def test_other_stream(dev):
    """The operators run on torch's current stream, behind what was put there before."""
    from mosaic_amd import ops
    rng = np.random.default_rng(24)
    table, total, starts, seq = _batch(rng, [500, 70], [1, 1], 64)
    c, s = (torch.from_numpy(x).to(dev) for x in _cache(rng, total, 1, 2, 128))
    args = (c, s, _i32(table, dev), _i32(starts, dev), _i32(seq, dev), 0.1)
    q = torch.from_numpy(_bf16(rng, 2, 8, 128)).to(dev).to(torch.bfloat16)
    want = ops.paged_attention(q, *args)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        late = torch.zeros_like(q)
        for _ in range(50):
            late = late + 0  # work in front
        late.copy_(q)
        got = ops.paged_attention(late, *args)
    stream.synchronize()
    assert torch.equal(got, want)


def test_refusals_of_the_wrappers(dev):
    from mosaic_amd import ops
    z = lambda *s, dt=torch.int32: torch.zeros(*s, dtype=dt, device=dev)  # noqa: E731
    q, codes, scales = z(2, 4, 64, dt=torch.bfloat16), z(3, 1, 2, 2, 64 * 64, dt=torch.uint8), z(3, 1, 2, 2, dt=torch.uint8)
    ok = dict(q=q, codes=codes, scales=scales, block_table=z(2, 3), starts=z(3), seq_lens=z(2), softmax_scale=1.0)
    ops.paged_attention(**ok)
    for kw in (dict(q=q.float()), dict(q=q[0]), dict(q=z(2, 3, 64, dt=torch.bfloat16)), dict(codes=codes[..., ::2]),
               dict(codes=codes.int()), dict(scales=scales[:2]), dict(block_table=z(2, 3).long()), dict(starts=z(2)),
               dict(seq_lens=z(2).long()), dict(seq_lens=z(4)[::2]), dict(sink=z(3, dt=torch.float32)), dict(window=-1),
               dict(max_new=0), dict(out=q[:1]), dict(block_table=z(3, 3)), dict(starts=z(3).cpu())):
        with pytest.raises((ValueError, TypeError)):
            ops.paged_attention(**{**ok, **kw})
    k = z(2, 2, 64, dt=torch.bfloat16)
    ok = dict(k=k, v=k, codes=codes, scales=scales, block_table=z(2, 3), starts=z(3), seq_lens=z(2))
    ops.paged_kv_write(**ok)
    for kw in (dict(k=k.half()), dict(v=k[:1]), dict(k=z(2, 1, 64, dt=torch.bfloat16)), dict(codes=codes[:, :, :1])):
        with pytest.raises((ValueError, TypeError)):
            ops.paged_kv_write(**{**ok, **kw})
    ok = dict(lengths=z(2), new=z(2), block_table=z(2, 3), tokens=2, page_size=64, free_pages=z(3), free_count=z(1))
    ops.paged_step(**ok)
    same = z(2)
    for kw in (dict(tokens=-1), dict(page_size=16), dict(new=z(3)), dict(free_count=None), dict(lengths=z(2).float()),
               dict(out=ops.PagedStep.empty(2, 3, dev)), dict(lengths=same, out=ops.PagedStep(z(3), same, z(1), z(2), z(2), z(2)))):
        with pytest.raises((ValueError, TypeError)):
            ops.paged_step(**{**ok, **kw})


# --------------------------------------------------- the ends of the range ----
def _attend(dev, q, c, s, table, starts, seq, scale, sink=None, window=0):
    from mosaic_amd import ops
    q = torch.from_numpy(np.asarray(q, np.float32)).to(dev).to(torch.bfloat16)
    snk = None if sink is None else torch.from_numpy(sink).to(dev)
    return ops.paged_attention(q, torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev), _i32(table, dev),
                               _i32(starts, dev), _i32(seq, dev), scale, sink=snk,
                               window=window).float().cpu().numpy().astype(np.float64)


# rows of a request that the few-row kernel finishes itself, cuts and joins, and the same of many rows
KINDS = [([150, 130], [3, 1]), ([3000, 140], [1, 2]), ([140], [40]), ([3000], [40])]


@pytest.mark.parametrize("sink", [False, True])
@pytest.mark.parametrize("held,new", KINDS)
def test_attention_scores_below_the_range(dev, held, new, sink):
    """Keys whose scores overflow to -inf weigh nothing beside later ones, however many blocks they fill."""
    rng = np.random.default_rng(40)
    table, total, starts, seq = _batch(rng, held, new, 64)
    c, s = _cache(rng, total, 1, 2, 64)
    c[:, :, :, 0] = 0  # scores of 0
    for i in range(len(held)):
        for b in table[i, :2]:  # the first 128 tokens: every dim at least 2^-6 2^60 below 0, times 2^100 and more
            c[b, :, :, 0] = 0x80 | rng.integers(8, 0x7F, c[b, :, :, 0].shape).astype(np.uint8)
            s[b, :, :, 0] = 127 + 60
    t = int(starts[-1])
    q = np.exp2(rng.integers(100, 110, (t, 4, 64)).astype(np.float64))
    snk = rng.standard_normal(4).astype(np.float32) if sink else None
    o = _attend(dev, q, c, s, table, starts, seq, 0.125, snk)
    # the same without these keys, and without what no longer matters, the size of the queries
    hidden = table.copy()
    hidden[:, :2] = -1
    want, tol = P.attention(np.zeros_like(q), c, s, hidden, starts, seq, 0.125, snk)
    assert np.isfinite(o).all() and np.all(np.abs(o - want) <= tol)


@pytest.mark.parametrize("held,new", KINDS)
def test_attention_rows_of_scores_all_minus_infinity(dev, held, new):
    """0 / 0 where there is no sink, and 0 beside one; rows that see no key are 0 in either case."""
    rng = np.random.default_rng(41)
    table, total, starts, seq = _batch(rng, held + [0, 0], new + [2, 20], 64)
    c, s = _cache(rng, total, 1, 2, 64)
    at_k = P.block_maps(64)[0]
    c[:, :, :, 0, at_k[:, 5]] = 0x80 | rng.integers(1, 0x7F, (total, 1, 2, 64)).astype(np.uint8)  # below 0
    table[-2:] = -1  # requests without pages
    q = _bf16(rng, int(starts[-1]), 4, 64).astype(np.float64)
    q[..., 5] = np.inf
    keyless = np.arange(int(starts[-1])) >= starts[-3]
    plain = _attend(dev, q, c, s, table, starts, seq, 0.125)
    assert np.isnan(plain[~keyless]).all() and not plain[keyless].any()
    assert not _attend(dev, q, c, s, table, starts, seq, 0.125, np.zeros(4, np.float32)).any()
    want, _ = P.attention(q, c, s, table, starts, seq, 0.125)
    np.testing.assert_array_equal(np.isnan(plain), np.isnan(want))


@pytest.mark.parametrize("scale", [0.0, 2.0 ** -130, 3e38, -3e38])
@pytest.mark.parametrize("held,new", KINDS)
def test_attention_scales_at_the_ends(dev, held, new, scale):
    """A scale of 0, or one that brings large scores back to where they do not count, gives means; so does the
    largest where every score is 0."""
    rng = np.random.default_rng(42)
    table, total, starts, seq = _batch(rng, held, new, 64)
    c, s = _cache(rng, total, 1, 2, 64)
    q = _bf16(rng, int(starts[-1]), 4, 64).astype(np.float64) * (2.0 ** 116 if abs(scale) < 1 else 0.0)
    want, tol = P.attention(q, c, s, table, starts, seq, scale)
    if abs(scale) < 1:  # the products are within fp32's range
        for i in range(len(held)):
            k = P.gather(c, s, table[i], int(seq[i]))[0]
            rows = q[starts[i]:starts[i + 1]]
            assert max(float((np.abs(k[h // 2]) @ np.abs(rows[:, h]).T).max()) for h in range(4)) < 2.0 ** 128
    o = _attend(dev, q, c, s, table, starts, seq, scale)
    assert np.all(np.abs(o - want) <= tol)


@pytest.mark.parametrize("n", [3, 40])
def test_values_near_the_largest_are_read_back(dev, n):
    """bf16's largest values, and infinities among them, are written so that what is read back is a number."""
    from mosaic_amd import ops
    rng = np.random.default_rng(43)
    hkv, d, t = 2, 64, n
    codes, scales = _cache(rng, 2, 1, hkv, d)
    x = np.exp2(127.0) * (1 + rng.integers(0, 128, (t, hkv, d)) / 128) * np.where(rng.random((t, hkv, d)) < 0.5, -1, 1)
    x[0] = 2.0 ** 127 * (2 - 2.0 ** -7)
    bad = rng.random((t, hkv, d)) < 0.1
    bad[0] = False
    xt = torch.from_numpy(np.where(bad, np.sign(x) * np.inf, x).astype(np.float32)).to(dev).to(torch.bfloat16)
    ct, st = torch.from_numpy(codes).to(dev), torch.from_numpy(scales).to(dev)
    table, starts, seq = _i32([[1]], dev), _i32([0, t], dev), _i32([t], dev)
    ops.paged_kv_write(xt, xt, ct, st, table, starts, seq)
    P.write(xt.double().cpu().numpy(), xt.double().cpu().numpy(), codes, scales, table.cpu().numpy(), [0, t], [t])
    np.testing.assert_array_equal(st.cpu().numpy(), scales)
    _same_codes(ct.cpu().numpy(), codes)
    # one key a row: the value itself
    q = torch.zeros(t, hkv, d, dtype=torch.bfloat16, device=dev)
    o = ops.paged_attention(q, ct, st, table, starts, seq, 0.125, window=1).float().cpu().numpy().astype(np.float64)
    assert np.isfinite(o).all()
    # at most 2^-4 off, half a step of e4m3; the codes above 240 are not used, 15/255 of the largest
    assert np.all(np.abs(o - x)[~bad] <= 2.0 ** -4 * np.abs(x)[~bad])
    np.testing.assert_array_equal(o[bad], np.sign(x)[bad] * 240.0 * 2.0 ** 120)


@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("byte", [0, 1, 2, 3, 100, 245, 246, 247, 248, 254])
def test_values_of_every_code_and_scale(dev, n, byte):
    """One key a row: the output is the code times 2^(byte - 127), rounded to bf16; 2^128 and more is not a
    number, for the rows that see it alone."""
    rng = np.random.default_rng(44)
    c, s = _cache(rng, 5, 1, 1, 64)
    all_codes = np.array([x for x in range(256) if x & 0x7F != 0x7F], np.uint8)
    at_v = P.block_maps(64)[1]
    held = 250 - n
    for b in range(4):
        c[b, 0, 0, 1, at_v] = np.resize(np.roll(all_codes, 37 * b), (64, 64))
    s[..., 1] = byte
    table = np.array([[0, 1, 2, 3]])
    starts, seq = np.array([0, n]), np.array([held + n])
    o = _attend(dev, np.zeros((n, 1, 64)), c, s, table, starts, seq, 0.125, window=1)
    b = np.arange(held, held + n) // 64
    v = C.e4m3_decode(c[table[0, b], 0, 0, 1]).astype(np.float64)[np.arange(n)[:, None], at_v[np.arange(held, held + n) % 64]]
    v *= 2.0 ** (byte - 127)
    fits = np.abs(v) < 2.0 ** 128
    assert (byte < 247) == fits.all()
    np.testing.assert_array_equal(np.isnan(o[:, 0]), ~fits)
    off = np.abs(o[:, 0] - v)[fits]
    # exact but below bf16's normal numbers, whose step is 2^-133
    assert np.all(off <= np.where(np.abs(v[fits]) < 2.0 ** -126, 2.0 ** -134, 0.0)), off.max()


@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("byte", [0, 1, 6, 246, 254])
def test_keys_of_the_ends_of_the_scales(dev, n, byte):
    """Scores of keys at the ends of the range, brought to ordinary size by the queries."""
    rng = np.random.default_rng(45)
    table, total, starts, seq = _batch(rng, [100], [n], 64)
    c, s = _cache(rng, total, 1, 2, 64)
    s[..., 0] = byte
    c[:, :, :, 0] = (c[:, :, :, 0] & 0xBF) | 0x20  # magnitudes of 2^-3 to 2^0.9: normal numbers in bf16 from byte 4 on
    size = 2.0 ** (120 if byte < 127 else -118)
    q = _bf16(rng, n, 4, 64).astype(np.float64) * size
    scale = 2.0 ** (127 - byte) / size if byte < 127 else 2.0 ** -8
    o = _attend(dev, q, c, s, table, starts, seq, scale)
    want, tol = P.attention(q, c, s, table, starts, seq, scale)
    assert np.all(np.abs(o - want) <= tol)


@pytest.mark.parametrize("held,new", KINDS)
@pytest.mark.parametrize("byte", [247, 250, 254])
def test_attention_values_past_the_range_reach_only_rows_that_see_them(dev, held, new, byte):
    """Values of 2^128 and more make the dim of every row that sees them no number, and of no other; keys of
    that size have infinite scores, which weigh nothing below and leave no number above."""
    rng = np.random.default_rng(46)
    table, total, starts, seq = _batch(rng, held, new, 64)
    c, s = _cache(rng, total, 1, 2, 64)
    at_k, at_v = P.block_maps(64)
    for i in range(len(held)):
        last = int(seq[i]) - 1
        for b, tok, dim, code in ((0, 3, 9, 0xFE), (last // 64, last % 64, 7, 0x7E)):  # all rows see it; one alone
            s[table[i, b], 0, 1, 1] = byte
            c[table[i, b], 0, 1, 1] = 0
            c[table[i, b], 0, 1, 1, at_v[tok, dim]] = code
        c[table[i, 1], 0, 0, 0] = 0
        c[table[i, 1], 0, 0, 0, at_k[20]] = 0x7E
        s[table[i, 1], 0, 0, 0] = byte
    q = _bf16(rng, int(starts[-1]), 4, 64).astype(np.float64)
    q[:, 0], q[:, 1] = np.abs(q[:, 0]) + 0.5, -np.abs(q[:, 1]) - 0.5
    o = _attend(dev, q, c, s, table, starts, seq, 0.125)
    assert np.isnan(o[:, 0]).all() and np.isfinite(o[:, 1]).all()
    want, tol = P.attention(q, c, s, table, starts, seq, 0.125)
    own = np.zeros(o[:, 2:].shape, bool)
    own[..., 9] = True
    own[starts[1:] - 1, :, 7] = True
    np.testing.assert_array_equal(np.isnan(want[:, 2:]), own)
    np.testing.assert_array_equal(np.isnan(o[:, 2:]), own)
    assert np.all((np.abs(o - want) <= tol)[:, 2:][~own])
    for i in range(len(held)):
        s[table[i, 1], 0, 0, 0] = 240  # the same key, its score far below but finite
    np.testing.assert_array_equal(_attend(dev, q, c, s, table, starts, seq, 0.125)[:, 1], o[:, 1])


# -------------------------------------------- the pool's edges and promises ----
def test_slots_of_pages_outside_the_pool(dev):
    """An id below 0, or whose slots would pass 31 bits, gives its rows none, from the stack as from a table."""
    from mosaic_amd import ops
    free = np.array([3, -1, 9, 1 << 30, 4], np.int32)
    table = np.zeros((3, 4), np.int32)
    lengths, new = np.array([0, 0, 0], np.int32), np.array([100, 130, 5], np.int32)
    count = 5
    t = _i32(table, dev)
    s = ops.paged_step(_i32(lengths, dev), _i32(new, dev), t, 235, 64, _i32(free, dev), _i32([count], dev))
    slots, pos = s.slots.cpu().numpy(), s.positions.cpu().numpy()
    assert pos[:100].tolist() == list(range(100))
    assert slots[:64].tolist() == list(range(4 * 64, 5 * 64)) and (slots[64:100] == -1).all()
    assert slots[100:164].tolist() == list(range(9 * 64, 10 * 64)) and (slots[164:228] == -1).all()
    assert slots[228:230].tolist() == [3 * 64, 3 * 64 + 1] and (slots[230:] == -1).all()
    given = _i32([[-7, 5, 1 << 26, 0]], dev)
    s = ops.paged_step(_i32([10], dev), _i32([200], dev), given, 200, 64)
    slots = s.slots.cpu().numpy()
    assert (slots[:54] == -1).all() and slots[54:118].tolist() == list(range(320, 384)) and (slots[118:182] == -1).all()
    assert slots[182:].tolist() == list(range(18))


def test_step_with_an_empty_pool(dev):
    """A pool of no pages places what needs none."""
    from mosaic_amd import ops
    s = ops.paged_step(_i32([3, 64], dev), _i32([2, 1], dev), _i32([[7, 7], [8, 8]], dev), 3, 64, _i32([], dev), _i32([0], dev))
    assert s.seq_lens.tolist() == [5, 0] and s.lengths.tolist() == [5, 64] and s.free_count.tolist() == [0]


def test_step_refuses_in_order(dev):
    """Pages are handed out in the order of the requests: one that gets too few keeps later ones from theirs, but
    not those that need none."""
    from mosaic_amd import ops
    lengths, new = [10, 60, 64, 64, 5], [1, 600, 1, 0, 2]  # pages needed: 0, 10, 1, 0, 0
    table = _i32(np.tile(np.arange(16), (5, 1)), dev)
    s = ops.paged_step(_i32(lengths, dev), _i32(new, dev), table, 604, 64, _i32([20, 21, 22], dev), _i32([3], dev))
    assert s.seq_lens.tolist() == [11, 0, 0, 64, 7]
    assert s.lengths.tolist() == [11, 60, 64, 64, 7] and s.free_count.tolist() == [3]


def test_trim_of_requests_that_share_a_prefix(dev):
    """Each is shortened to the shared pages, which only their last owner gives back: every page is freed once."""
    from mosaic_amd.kernels.paged import PagedKVCache
    cache = PagedKVCache(12, 1, 64, 3, 400, device=dev)
    cache.step(_i32([200, 0, 0], dev), 200)  # four pages, three of them full
    cache.block_table[1:, :3] = cache.block_table[0, :3]  # two more begin with the full ones
    cache.lengths[1:] = 192
    cache.step(_i32([1, 70, 5], dev), 76)
    assert cache.free_count.tolist() == [12 - 4 - 2 - 1]
    for keep in ([250, 192, 300], [300, 300, 192], [0, 300, 300]):  # behind the shared pages; the last owner: all
        cache.trim(_i32(keep, dev))
        cache.lengths[1:] *= (cache.lengths[1:] != 192)  # the shared ones stay in the pool: no longer this request's
    assert cache.lengths.tolist() == [0, 0, 0] and cache.free_count.tolist() == [12]
    assert sorted(cache.free_pages.tolist()) == list(range(12))


def _wide(rng, dev, r, pages, hkv, d, width):
    """A cache and tables so wide that tiles of few rows and of many are cut and joined."""
    c, s = _cache(rng, pages, 1, hkv, d)
    return torch.from_numpy(c).to(dev), torch.from_numpy(s).to(dev), _i32(rng.integers(0, pages, (r, width)), dev)


def test_cut_tiles_in_a_graph(dev):
    """Attention that cuts and joins tiles of both kinds, captured once and replayed while lengths and rows change."""
    from mosaic_amd import ops
    rng = np.random.default_rng(47)
    r, t, hq, hkv, d, width = 4, 60, 8, 2, 128, 80
    c, s, table = _wide(rng, dev, r, 100, hkv, d, width)
    q = torch.zeros(t, hq, d, dtype=torch.bfloat16, device=dev)
    starts, seq = _i32(np.zeros(r + 1), dev), _i32(np.zeros(r), dev)
    ws = ops.MoEWorkspace()
    args = (q, c, s, table, starts, seq, 0.1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.paged_attention(*args, workspace=ws)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops.paged_attention(*args, workspace=ws)
    for new, held in (([1, 1, 1, 1], [5000, 3, 1200, 0]), ([40, 1, 0, 2], [4900, 5000, 7, 64]), ([0, 0, 0, 0], [9, 9, 9, 9]),
                      ([4, 4, 4, 4], [100, 200, 5100, 5]), ([50, 1, 2, 3], [0, 4000, 4000, 4000]), ([1, 1, 1, 1], [64, 65, 63, 1])):
        q.copy_(torch.from_numpy(_bf16(rng, t, hq, d)).to(dev))
        starts.copy_(_i32(np.concatenate([[0], np.cumsum(new)]), dev))
        seq.copy_(_i32(np.array(new) + np.array(held), dev))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, ops.paged_attention(*args)), new


def test_two_streams_at_once(dev):
    """Calls on two streams, each with a workspace of its own, beside each other over one cache."""
    from mosaic_amd import ops
    rng = np.random.default_rng(48)
    c, s, table = _wide(rng, dev, 3, 60, 2, 64, 90)
    calls = []
    for new, held in (([1, 1, 1], [5500, 40, 3000]), ([70, 1, 30], [5000, 2000, 10])):
        q = torch.from_numpy(_bf16(rng, sum(new), 8, 64)).to(dev).to(torch.bfloat16)
        calls.append((q, c, s, table, _i32(np.concatenate([[0], np.cumsum(new)]), dev),
                      _i32(np.array(new) + np.array(held), dev), 0.125))
    want = [ops.paged_attention(*a) for a in calls]
    streams, ws = [torch.cuda.Stream() for _ in calls], [ops.MoEWorkspace() for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(ops.paged_attention(*calls[i], workspace=ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
