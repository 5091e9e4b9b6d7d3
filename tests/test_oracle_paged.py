"""The paged cache's oracle checked by properties it does not use itself, and the operators' refusals (CPU only)."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from mosaic_amd import _lib
from oracle import codecs as C
from oracle import paged as P


@pytest.mark.parametrize("d", [64, 128, 256])
def test_block_maps_are_permutations(d):
    for m in P.block_maps(d):
        assert np.array_equal(np.sort(m.ravel()), np.arange(64 * d))


def test_step_then_trim_restores_the_pool():
    rng = np.random.default_rng(0)
    lengths = rng.integers(0, 300, 40).astype(np.int32)
    new = rng.integers(0, 200, 40).astype(np.int32)
    pages = int(sum(-(-int(x) // 64) for x in lengths)) + 90
    ids = rng.permutation(pages).astype(np.int32)
    table = np.full((40, 9), -1, np.int32)
    at = 0
    for i, x in enumerate(lengths):
        n = -(-int(x) // 64)
        table[i, :n] = ids[at:at + n]
        at += n
    free = np.zeros(pages, np.int32)
    count = pages - at
    free[:count] = ids[at:]
    before = free.copy()
    s = P.step(lengths, new, table, int(new.sum()), 64, free, count)
    left = int(s["free_count"][0])
    assert left < count
    used = np.concatenate([table[i, :-(-int(x) // 64)] for i, x in enumerate(s["lengths"])] + [free[:left]])
    assert np.array_equal(np.sort(used), np.arange(pages))  # every page has one owner
    free[left:count] = -7  # what was popped is not read again
    kept, back = P.trim(s["lengths"], lengths, table, 64, free, left)
    assert back == count and np.array_equal(kept, lengths) and np.array_equal(free, before)


def test_scale_is_the_least_that_holds():
    rng = np.random.default_rng(1)
    for x in list(np.exp2(rng.uniform(-130, 120, 300))) + [448.0, 449.0, 447.0, 224.0, 2.0 ** -120 * 448]:
        e = P.scale_exp(float(x))
        assert x <= 448.0 * 2.0 ** e or e == 120
        assert e == -126 or x > 448.0 * 2.0 ** (e - 1)


def test_write_then_gather_is_within_half_a_step():
    rng = np.random.default_rng(2)
    codes, scales = np.zeros((5, 1, 2, 2, 64 * 64), np.uint8), np.full((5, 1, 2, 2), 127, np.uint8)
    k = rng.standard_normal((150, 2, 64)) * np.exp2(rng.integers(-6, 6, (150, 1, 1)))
    v = rng.standard_normal((150, 2, 64))
    table = np.array([[3, 0, 4]], np.int32)
    for a, b in ((0, 1), (1, 70), (70, 150)):  # scales grow as larger tokens come
        P.write(k[a:b], v[a:b], codes, scales, table, np.array([0, b - a]), np.array([b]))
    kk, vv = P.gather(codes, scales, table[0], 150)
    for got, x in ((kk, k), (vv, v)):
        for h in range(2):
            for b in range(3):
                part, have = x[64 * b:64 * b + 64, h], got[h, 64 * b:64 * b + 64]
                size = 2.0 ** P.scale_exp(float(np.abs(part).max()))
                # half a step of e4m3 (2^-4 relative, 2^-10 of the scale below 2^-6), twice where the scale moved
                assert np.all(np.abs(have - part) <= 2 * np.maximum(np.abs(part) * 2.0 ** -4, size * 2.0 ** -10))


def test_attention_of_one_key_is_its_value():
    rng = np.random.default_rng(3)
    codes, scales = np.zeros((2, 1, 1, 2, 64 * 64), np.uint8), np.full((2, 1, 1, 2), 127, np.uint8)
    v = C.e4m3_decode(rng.integers(0, 0x7F, (3, 1, 64)).astype(np.uint8)).astype(np.float64)
    P.write(v, v, codes, scales, np.array([[1]]), np.array([0, 3]), np.array([3]))
    o, _ = P.attention(rng.standard_normal((3, 2, 64)), codes, scales, np.array([[1]]), np.array([0, 3]), np.array([3]),
                       0.1, window=1)
    got = P.gather(codes, scales, np.array([1]), 3)[1][0]
    np.testing.assert_allclose(o, np.repeat(got[:, None], 2, 1), rtol=1e-12)


# ------------------------------------------------------------- refusals ----
PTR = ctypes.c_void_p(4096)  # never followed: the checks fail first


def _refused(name, args, text):
    rc = getattr(_lib.lib(), name)(*args)
    assert rc < 0
    assert text in _lib.lib().mosaic_last_error().decode()


def _step(**kw):
    a = dict(lengths=ctypes.c_void_p(1 << 12), add=ctypes.c_void_p(2 << 12), table=ctypes.c_void_p(3 << 12), stride=4,
             free=ctypes.c_void_p(4 << 12), count=ctypes.c_void_p(5 << 12), r=2, width=4, pages=8, tokens=2, page=64,
             starts=ctypes.c_void_p(6 << 12), out=ctypes.c_void_p(7 << 12), seq=ctypes.c_void_p(8 << 12),
             pos=ctypes.c_void_p(9 << 12), slots=ctypes.c_void_p(10 << 12), left=ctypes.c_void_p(11 << 12))
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,text", [
    (dict(page=32), "page size"), (dict(page=100), "page size"), (dict(page=8192), "page size"),
    (dict(tokens=1 << 21), "token rows"), (dict(tokens=-1), "token rows"), (dict(r=(1 << 20) + 1), "requests"),
    (dict(width=0), "tables"), (dict(stride=3), "tables"), (dict(width=1 << 24, stride=1 << 24), "tables"),
    (dict(pages=1 << 25), "slots"), (dict(count=None), "goes with"), (dict(starts=None), "null"),
    (dict(out=ctypes.c_void_p(1 << 12)), "overlaps"), (dict(left=ctypes.c_void_p(5 << 12)), "overlaps"),
    (dict(seq=ctypes.c_void_p((2 << 12) + 4)), "overlaps")])
def test_step_refusals(kw, text):
    _refused("mosaic_paged_step", _step(**kw), text)


def _trim(**kw):
    a = dict(lengths=ctypes.c_void_p(1 << 12), keep=ctypes.c_void_p(2 << 12), table=ctypes.c_void_p(3 << 12), stride=4,
             free=ctypes.c_void_p(4 << 12), count=ctypes.c_void_p(5 << 12), r=2, width=4, pages=8, page=64,
             out=ctypes.c_void_p(6 << 12), left=ctypes.c_void_p(7 << 12))
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,text", [
    (dict(page=65), "page size"), (dict(width=0), "tables"), (dict(pages=1 << 25), "pages"), (dict(r=-1), "requests"),
    (dict(out=None), "null"), (dict(out=ctypes.c_void_p(1 << 12)), "overlaps"),
    (dict(left=ctypes.c_void_p(5 << 12)), "overlaps"), (dict(free=ctypes.c_void_p(2 << 12)), "overlaps")])
def test_trim_refusals(kw, text):
    _refused("mosaic_paged_trim", _trim(**kw), text)


def _write(**kw):
    a = dict(k=PTR, v=PTR, kt=128, kh=128, vt=128, vh=128, tokens=3, codes=PTR, scales=PTR, pages=4, blocks=1, heads=1,
             d=128, table=PTR, stride=2, width=2, starts=PTR, seq=PTR, r=1)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,text", [
    (dict(d=96), "head dim"), (dict(heads=0), "heads"), (dict(blocks=65), "blocks"), (dict(tokens=1 << 21), "tokens"),
    (dict(kt=130), "16 bytes"), (dict(vh=4), "16 bytes"), (dict(k=ctypes.c_void_p(4104)), "16 bytes"),
    (dict(codes=ctypes.c_void_p(4100)), "16 bytes"), (dict(width=3), "tables"), (dict(seq=None), "null")])
def test_write_refusals(kw, text):
    _refused("mosaic_paged_kv_write", _write(**kw), text)


def _attn(**kw):
    a = dict(q=PTR, qt=256, qh=128, tokens=3, hq=2, codes=PTR, scales=PTR, pages=4, blocks=1, hkv=1, d=128, table=PTR,
             stride=2, width=2, starts=PTR, seq=PTR, r=1, sink=None, window=0, new=0, scale=0.1, out=PTR, ws=PTR,
             nws=1 << 40)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,text", [
    (dict(hq=3, hkv=2), "query heads"), (dict(hkv=0), "query heads"), (dict(d=32), "query heads"),
    (dict(tokens=1 << 21), "tokens"), (dict(blocks=0), "blocks"), (dict(pages=0), "pages"), (dict(window=-1), "window"), (dict(new=-1), "max_new"),
    (dict(scale=float("nan")), "finite"), (dict(scale=float("inf")), "finite"), (dict(qt=260), "16 bytes"),
    (dict(q=ctypes.c_void_p(4104)), "16 bytes"), (dict(out=ctypes.c_void_p(4104)), "16 bytes"),
    (dict(scales=ctypes.c_void_p(4097)), "16 bytes"), (dict(width=200, stride=200, nws=1000), "workspace"), (dict(width=200, stride=200, ws=None), "workspace"), (dict(out=None), "null"),
    (dict(stride=1), "tables"), (dict(), "overlaps"),
    (dict(tokens=1 << 20, r=1 << 20, hq=16, hkv=16), "too many")])
def test_attention_refusals(kw, text):
    _refused("mosaic_paged_attention", _attn(**kw), text)


def test_workspace_sizes():
    """A query for every kind of call, those without requests among them, and 0 for shapes that are refused."""
    size = _lib.lib().mosaic_paged_attention_workspace_bytes
    assert size(5, 0, 64, 8, 128, 1, 40, 0) > 0 and size(0, 0, 64, 8, 128, 1, 40, 0) > 0
    assert size(64, 64, 64, 8, 128, 1, 32, 1) == 0 < size(64, 64, 64, 8, 128, 1, 33, 1)  # narrow tables are not cut
    assert size(4096, 1, 64, 8, 128, 1, 64, 0) == 0  # many uncut tiles of one request need none
    assert size(512, 1, 64, 8, 128, 1, 480, 0) > 1 << 20
    for bad in ((1, 1, 3, 2, 128, 1, 1, 0), (1, 1, 8, 8, 96, 1, 1, 0), (1 << 21, 1, 8, 8, 64, 1, 1, 0),
                (1, 1, 8, 8, 64, 0, 1, 0), (1, 1, 8, 8, 64, 1, 0, 0), (1, 1, 8, 8, 64, 1, 1, -1)):
        assert size(*bad) == 0


def test_empty_calls_launch_nothing():
    before = _lib.lib().mosaic_launch_count()
    assert _lib.lib().mosaic_paged_kv_write(*_write(tokens=0)) == 0
    assert _lib.lib().mosaic_paged_attention(*_attn(tokens=0)) == 0
    assert _lib.lib().mosaic_launch_count() == before


def test_wrappers_refuse_cpu_tensors_and_bad_caches():
    from mosaic_amd import ops
    from mosaic_amd.kernels.paged import PagedKVCache
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.paged_step(i, i, torch.zeros(2, 3, dtype=torch.int32), 2, 64)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.paged_trim(i, i, torch.zeros(2, 3, dtype=torch.int32), 64, i, i[:1])
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.paged_kv_write(x, x, None, None, None, None, None)
    with pytest.raises(ValueError, match="GPU tensor"):
        ops.paged_attention(x, None, None, None, None, None, 1.0)
    for kw in (dict(page_size=32), dict(head_dim=96), dict(pages=0), dict(max_length=0)):
        with pytest.raises(ValueError):
            PagedKVCache(**{**dict(pages=4, kv_heads=1, head_dim=64, max_requests=1, max_length=64, device="cpu"), **kw})


@pytest.mark.parametrize("r,width", [(1 << 12, 1 << 19), (1 << 20, 1 << 11), (1 << 8, (1 << 24) - 1)])
def test_trim_refuses_tables_whose_pages_pass_32_bits(r, width):
    """Lengths that claim whole tables would make the count of freed pages wrap, and columns be read outside a row."""
    _refused("mosaic_paged_trim", _trim(r=r, width=width, stride=width), "entries")


def _at(page, word=0):
    return ctypes.c_void_p((page << 12) + 4 * word)


@pytest.mark.parametrize("kw,text", [
    (dict(out=_at(3, 1)), "overlaps the tables"), (dict(pos=_at(3, 7)), "overlaps the tables"),
    (dict(slots=_at(3, 999), stride=1000), "overlaps the tables"), (dict(left=_at(3, 1003), stride=1000), "overlaps the tables"),
    (dict(table=_at(1, 1)), "tables overlap"), (dict(table=_at(2, -1000), stride=1000), "tables overlap"),
    (dict(table=_at(4, -3)), "tables overlap"), (dict(table=_at(5)), "tables overlap"),
    (dict(seq=_at(7, 1)), "overlaps another"), (dict(slots=_at(9, -1)), "overlaps another"),
    (dict(left=_at(6, 2)), "overlaps another")])
def test_step_refuses_shared_memory(kw, text):
    _refused("mosaic_paged_step", _step(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(out=_at(3, 7)), "overlaps the tables"), (dict(free=_at(3, -7)), "overlaps the tables"),
    (dict(left=_at(3, 1001), stride=1000), "overlaps the tables"), (dict(left=_at(6, 1)), "overlaps another"),
    (dict(out=_at(4, 7)), "overlaps another")])
def test_trim_refuses_shared_memory(kw, text):
    _refused("mosaic_paged_trim", _trim(**kw), text)


@pytest.mark.parametrize("kw", [dict(out=_at(3, 4), stride=1000), dict(out=_at(3, 998), stride=1000), dict(pos=_at(3, 1004), stride=1000),
                                dict(table=_at(1, 2), free=None, count=None)])
def test_step_takes_what_lies_between_the_rows(kw):
    """Memory between a table's rows is another's, and one that nothing is written to may be an input too: these
    calls pass the checks (what fails is the launch, without a GPU)."""
    if torch.cuda.is_available():
        pytest.skip("the pointers are made up")
    assert _lib.lib().mosaic_paged_step(*_step(**kw)) > 0
