"""Keys and values held in 4 bits.

A cache of 16-bit rows takes 2 bytes a value; here a value is a 4-bit code, and
each group of 32 dims of a row has a scale and a least value in the rows' type
(0.625 bytes a value in all, rows filled up to multiples of 16 bytes):

* :func:`empty` — room for such rows;
* :func:`write` — rows quantised into the cache as a step makes them;
* :func:`read` — rows of the cache as 16-bit rows;
* :func:`attention` — ``tree.tree_attention`` over the cache;
* :func:`key_mass` — ``eviction.key_mass`` over its keys.

The caches are uint8 tensors ``[B, rows, Hkv, row_bytes(D)]`` or pages ``[n,
page, Hkv, row_bytes(D)]``; any dim that is a multiple of 32 up to 320 has rows
of its own length.  Their bytes move as they are: ``tree.tree_commit`` and
``eviction.evict`` take them like any other cache.

The reference holds every row in 16 bits; these entry points stand beside its
caches.  Torch wrappers over ``include/slimkv_b200.h`` (where the rows' layout
and rounding are defined); there is no CPU path.
"""
from ctypes import byref

import torch

from . import _lib
from .eviction import mass_args
from .tree import _TYPES, _check_rows, _i32, _refuse, _run, _run_in_workspace, attention_args, fill_cache

# Dims and the bytes of their rows, one to one.
_BYTES = {dim: (dim // 2 + dim // 8 + 15) // 16 * 16 for dim in range(32, 321, 32)}
_DIMS = {size: dim for dim, size in _BYTES.items()}


def row_bytes(dim):
    """Bytes of a row of ``dim`` values (a multiple of 32 up to 320)."""
    if dim not in _BYTES:
        _refuse('4-bit rows have a multiple of 32 up to 320 dims')
    return _BYTES[dim]


def empty(sequences, rows, kv_heads, dim, dim_v=None, device='cuda'):
    """K and V caches of ``rows`` rows for each of ``sequences`` (or of pages of
    ``rows`` rows): uint8 ``[sequences, rows, Hkv, bytes]``, a head's rows one
    behind the other."""
    return tuple(torch.empty((sequences, kv_heads, rows, row_bytes(d)), dtype=torch.uint8, device=device).transpose(1, 2)
                 for d in (dim, dim_v or dim))


def _dim_of(rows, what):
    dim = _DIMS.get(rows.shape[-1]) if rows.dtype == torch.uint8 else None
    if dim is None:
        _refuse('%s must be uint8 rows of row_bytes(dim) bytes', what)
    return dim


def _rows_args(k, v, k4, v4, starts, counts, block_tables, dim, dim_v):
    batch, rows, heads = k.shape[:3]
    dev = k.device
    if k4.device != dev or k4.shape[2] != heads:
        _refuse('rows and caches need the same heads and device')
    a = _lib.Cache4RowsArgs()
    fill_cache(a.cache, k4, v4, block_tables, batch)
    a.batch, a.rows, a.kv_heads, a.dim_qk, a.dim_v, a.type = batch, rows, heads, dim, dim_v, _TYPES[k.dtype]
    a.k, a.v = k.data_ptr(), v.data_ptr()
    x, y = a.k_stride, a.v_stride
    x[0], x[1], x[2] = k.stride()[:3]
    y[0], y[1], y[2] = v.stride()[:3]
    if starts is not None:
        a.starts = _i32(starts, (batch,), dev, 'starts')
    if counts is not None:
        a.counts = _i32(counts, (batch,), dev, 'counts')
    return a


def _caches(k4, v4):
    """Dims of 4-bit K and V caches that agree otherwise."""
    if not (k4.is_cuda and v4.is_cuda and k4.dim() == v4.dim() == 4 and k4.device == v4.device):
        _refuse('4-bit caches must be CUDA tensors [B, rows, Hkv, bytes] (or pages) on one device')
    return _dim_of(k4, 'k4'), _dim_of(v4, 'v4')


def write(k, v, k4, v4, starts=None, counts=None, block_tables=None):
    """Quantises rows into a 4-bit cache (``slimkv_cache4_write``).

    Row i of sequence b of ``k`` / ``v [B, n, Hkv, D / Dv]`` (bf16 or fp16),
    i < ``counts[b]`` (int32 ``[B]``; default: all n), becomes cache row
    ``starts[b] + i`` (int32 ``[B]``, the old lengths; default: 0) of ``k4`` /
    ``v4`` (dense, or pages with int32 ``block_tables [B, pages]``).  Other
    rows keep their bytes.  A group of 32 dims with an infinity or a NaN reads
    back as NaN.
    """
    _check_rows(k, v, 4)
    dim, dim_v = _caches(k4, v4)
    if k.dtype not in (torch.bfloat16, torch.float16) or k.shape[:3] != v.shape[:3] or k.stride(3) != 1 or v.stride(3) != 1:
        _refuse('rows must be bf16 or fp16 [B, n, Hkv, D] with a contiguous last dimension')
    if k.shape[3] != dim or v.shape[3] != dim_v:
        _refuse('caches need rows of row_bytes(D) and row_bytes(Dv) bytes')
    if k.numel() == 0:
        return
    a = _rows_args(k, v, k4, v4, starts, counts, block_tables, dim, dim_v)
    _run(k.device, _lib.load().slimkv_cache4_write, byref(a))


def read(k4, v4, counts, dtype, rows=None, starts=None, block_tables=None, out=None):
    """Rows of a 4-bit cache as 16-bit rows (``slimkv_cache4_read``).

    ``dtype``: bf16 or fp16, that of the rows written.  Row i of the results,
    i < ``counts[b]`` (int32 ``[B]``), is cache row ``starts[b] + i`` (default:
    i).  Returns new ``(k [B, rows, Hkv, D], v [B, rows, Hkv, Dv])`` with zeros
    past a sequence's count, or writes ``out = (k, v)``, whose other rows stay as
    they are (``rows`` is theirs then).
    """
    dim, dim_v = _caches(k4, v4)
    if dtype not in (torch.bfloat16, torch.float16) or counts.dim() != 1:
        _refuse('rows are read as bf16 or fp16, counts int32 [B]')
    batch, heads, dev = counts.shape[0], k4.shape[2], k4.device
    if out is None:
        if rows is None:
            if block_tables is not None:
                _refuse('rows: how many of each sequence')
            rows = k4.shape[1]
        k, v = (torch.empty_strided((batch, rows, heads, d), (rows * heads * d, heads * d, d, 1), dtype=dtype, device=dev)
                for d in (dim, dim_v))
    else:
        k, v = out
        _check_rows(k, v, 4)
        if not (k.dtype == dtype and k.shape[0] == batch and k.shape[:3] == v.shape[:3] and k.shape[3] == dim and
                v.shape[3] == dim_v and k.stride(3) == v.stride(3) == 1 and rows in (None, k.shape[1])):
            _refuse('out must be [B, rows, Hkv, D] and [B, rows, Hkv, Dv] of the type')
    if k.numel() == 0:
        return k, v
    a = _rows_args(k, v, k4, v4, starts, counts, block_tables, dim, dim_v)
    a.zero_rest = out is None
    _run(dev, _lib.load().slimkv_cache4_read, byref(a))
    return k, v


def attention(q, k4, v4, lengths, scale, mask=None, nodes=None, block_tables=None, context_only=False, out=None,
              lse=None, wait_limit_ns=0):
    """``tree.tree_attention`` over a 4-bit cache (``slimkv_cache4_attention``):
    the same arguments and results, ``k4`` / ``v4`` the caches that
    :func:`write` filled from rows of q's type.  The query rows of a KV head are
    taken 8, 16 or (of wide rows) 32 at a time, each time over all keys: made for
    single tokens and small trees.  For many (over long caches from about 17
    nodes of 4 heads, over latents from 4 of 32) :func:`read`, then
    ``tree.tree_attention`` is faster."""
    dim, dim_v = _caches(k4, v4)
    if q.dim() != 4 or q.shape[3] != dim:
        _refuse('q must be [B, T, H, D] with caches of row_bytes(D) bytes a row')
    a, out, lse = attention_args(q, k4, v4, lengths, scale, mask, nodes, block_tables, context_only, out, lse,
                                 wait_limit_ns, torch.uint8, k4.shape[3], dim_v)
    lib = _lib.load()
    _run_in_workspace(q.device, lib.slimkv_cache4_attention_workspace_size, lib.slimkv_cache4_attention, a)
    return out, lse


def key_mass(q, k4, lse, mass, lengths, scale, rows=None, counts=None, decay=1.0, block_tables=None,
             context_only=False, wait_limit_ns=0):
    """``eviction.key_mass`` over the keys of a 4-bit cache
    (``slimkv_cache4_key_mass``): the same arguments and results.  Over latents
    with many accepted rows, ``read`` and ``eviction.key_mass`` are faster."""
    if not (k4.is_cuda and k4.dim() == 4 and q.dim() == 4 and q.shape[3] == _dim_of(k4, 'k4')):
        _refuse('q must be [B, T, H, D], k4 a CUDA cache of row_bytes(D) bytes a row')
    a = mass_args(q, k4, lse, mass, lengths, scale, rows, counts, decay, block_tables, context_only, wait_limit_ns,
                  torch.uint8, k4.shape[3])
    _run(q.device, _lib.load().slimkv_cache4_key_mass, byref(a))
    return mass
