"""The C entries of the 4-bit cache refuse arguments on the host, before any
device work (null streams, no GPU)."""
import ctypes

import pytest

from slimkv_b200 import _lib, cache4
from test_tree_library import ALIGNMENT, INVALID, P, SHAPE, WORKSPACE, attention, fill, mass

FAR = 1 << 24


def rows(**kw):
    a = _lib.Cache4RowsArgs()
    a.batch, a.rows, a.kv_heads, a.dim_qk, a.dim_v, a.type = 2, 4, 2, 64, 64, 0
    a.k, a.v, a.cache.k, a.cache.v, a.cache.rows = FAR, 2 * FAR, 3 * FAR, 4 * FAR, 64
    for s in (a.k_stride, a.v_stride):
        s[0], s[1], s[2] = 4 * 2 * 64, 2 * 64, 64
    for s in (a.cache.k_stride, a.cache.v_stride):
        s[0], s[1], s[2] = 64 * 2 * 48, 2 * 48, 48
    return fill(a, kw)


def attention4(**kw):
    strides = {f'cache__{x}_stride__x{i}': s for x in 'kv' for i, s in enumerate((64 * 2 * 48, 2 * 48, 48))}
    return attention(**dict(strides, **kw))


def mass4(**kw):
    strides = {f'cache__k_stride__x{i}': s for i, s in enumerate((64 * 2 * 48, 2 * 48, 48))}
    return mass(**dict(strides, **kw))


BOTH = [
    (dict(batch=0), INVALID), (dict(batch=65536), INVALID), (dict(rows=0), INVALID), (dict(kv_heads=0), INVALID),
    (dict(type=2), INVALID), (dict(dim_qk=40), SHAPE), (dict(dim_v=352), SHAPE), (dict(dim_v=0), SHAPE), (dict(k=0), INVALID),
    (dict(v=0), INVALID), (dict(cache__k=0), INVALID), (dict(cache__v=0), INVALID), (dict(cache__rows=0), INVALID),
    (dict(k=FAR + 8), ALIGNMENT), (dict(v_stride__x1=132), ALIGNMENT), (dict(v_stride__x1=-128), ALIGNMENT),
    (dict(cache__k=3 * FAR + 8), ALIGNMENT), (dict(cache__v_stride__x1=100), ALIGNMENT), (dict(cache__table=P), INVALID),
    (dict(rows=1 << 30), SHAPE),
    (dict(k=3 * FAR), INVALID), (dict(v=4 * FAR + 64 * 2 * 48 - 16), INVALID), (dict(k=4 * FAR - 16), INVALID)]
CASES = [
    ('slimkv_cache4_write', rows, BOTH + [
        (dict(cache__k_stride__x0=0), INVALID), (dict(cache__v_stride__x1=0), INVALID), (dict(cache__k_stride__x1=32), INVALID),
        (dict(cache__v=3 * FAR), INVALID), (dict(cache__v=3 * FAR + 16), INVALID)]),
    ('slimkv_cache4_read', rows, BOTH + [
        (dict(k_stride__x0=0), INVALID), (dict(v_stride__x2=0), INVALID), (dict(v_stride__x2=32), INVALID), (dict(v=FAR), INVALID),
        (dict(v=FAR + 64), INVALID)]),
    ('slimkv_cache4_attention', attention4, [
        (dict(batch=0), INVALID), (dict(batch=4097), INVALID), (dict(nodes=0), INVALID), (dict(nodes=1025), INVALID),
        (dict(heads=7), INVALID), (dict(heads=258), SHAPE), (dict(dim_qk=40), SHAPE), (dict(dim_qk=352), SHAPE), (dict(dim_v=8), SHAPE),
        (dict(type=2), INVALID), (dict(q=0), INVALID), (dict(lengths=0), INVALID), (dict(lse=0), INVALID), (dict(out=0), INVALID),
        (dict(cache__k=0), INVALID), (dict(cache__v=0), INVALID), (dict(cache__rows=0), INVALID), (dict(scale=0.0), INVALID),
        (dict(scale=float('nan')), INVALID), (dict(scale=float('inf')), INVALID), (dict(q_stride__x1=4), ALIGNMENT),
        (dict(q=P + 8), ALIGNMENT), (dict(cache__k=P + 8), ALIGNMENT), (dict(cache__v_stride__x1=100), ALIGNMENT),
        (dict(cache__table=P), INVALID),
        (dict(cache__table=P, cache__table_pages=2, cache__num_pages=2, cache__table_stride=2, cache__rows=12), SHAPE),
        (dict(), WORKSPACE)]),
    ('slimkv_cache4_key_mass', mass4, [
        (dict(batch=0), INVALID), (dict(nodes=1025), INVALID), (dict(heads=7), INVALID), (dict(mass_rows=0), INVALID),
        (dict(heads=258), SHAPE), (dict(dim=40), SHAPE), (dict(dim=352), SHAPE), (dict(type=2), INVALID),
        (dict(scale=float('nan')), INVALID), (dict(decay=float('inf')), INVALID), (dict(q_stride__x0=4), ALIGNMENT),
        (dict(q=P + 2), ALIGNMENT), (dict(cache__k=0), INVALID), (dict(cache__k=P + 8), ALIGNMENT), (dict(mass=0), INVALID),
        (dict(cache__table=P, cache__table_pages=2, cache__num_pages=2, cache__table_stride=2, cache__rows=12), SHAPE)]),
]


def call(entry, a):
    extra = (None, 0) if entry.endswith('attention') else ()
    return getattr(_lib.load(), entry)(a, *extra, None)


@pytest.mark.parametrize('entry,make,change,code', [(e, m, c, k) for e, m, cases in CASES for c, k in cases])
def test_refusals(entry, make, change, code):
    assert call(entry, ctypes.byref(make(**change))) == code
    assert _lib.load().slimkv_last_error()


@pytest.mark.parametrize('entry', [c[0] for c in CASES])
def test_null_arguments(entry):
    assert call(entry, None) == INVALID


@pytest.mark.parametrize('entry', ['slimkv_cache4_write', 'slimkv_cache4_read'])
def test_k_and_v_by_turns_in_one_page_are_apart(entry):
    """K and V rows side by side under the same strides share no byte; a byte further they do."""
    pages = dict(cache__table=P, cache__table_pages=4, cache__num_pages=8, cache__table_stride=4, cache__rows=16)
    strides = {f'cache__{x}_stride__x{i}': s for x in 'kv' for i, s in enumerate((16 * 2 * 2 * 48, 2 * 2 * 48, 48))}
    a = dict(pages, cache__v=3 * FAR + 2 * 48, **strides)
    if entry.endswith('write'):         # refused for overlap if V starts 16 bytes earlier, which is checked before the launch
        assert call(entry, ctypes.byref(rows(**dict(a, cache__v=3 * FAR + 2 * 48 - 16)))) == INVALID
        assert b'K and V' in _lib.load().slimkv_last_error()
    a['type'] = 7                       # (the valid call would launch: stop it at another check)
    assert call(entry, ctypes.byref(rows(**a))) == INVALID
    assert b'bf16 or fp16' in _lib.load().slimkv_last_error()


def test_row_bytes():
    size = _lib.load().slimkv_row4_bytes
    for dim in range(32, 321, 32):
        assert size(dim) == cache4.row_bytes(dim) == -(-(dim // 2 + dim // 32 * 4) // 16) * 16
    assert [size(d) for d in (0, -32, 8, 40, 352)] == [0] * 5
    assert len(set(map(cache4.row_bytes, range(32, 321, 32)))) == 10      # a row's bytes name its dim
    with pytest.raises(RuntimeError):
        cache4.row_bytes(48)


def test_workspace_size():
    size = _lib.load().slimkv_cache4_attention_workspace_size
    assert size(ctypes.byref(attention4(dim_qk=40))) == 0 and size(None) == 0
