"""A cache kept within a budget by the attention its keys receive.

* :func:`key_mass` — adds the attention weights that the step's accepted rows
  gave each key to its running mass;
* :func:`evict` — keeps the sinks, the recent rows and the rows of the largest
  mass, in order, in a cache of ``keep`` rows.

Beacon latents carry no position, and raw keys are cached rotated, so a row
can leave without touching the others.  The reference never drops a cached
row.  Torch wrappers over ``include/slimkv_b200.h``; there is no CPU path.
"""
import ctypes

import torch

from . import _lib
from .kernels import _ptr, _require, _stream
from .tree import _TYPES, _i32, fill_cache


def _plane(t, dtype, batch, heads, what):
    _require(t.is_cuda and t.dtype == dtype and t.dim() == 3 and t.shape[:2] == (batch, heads) and t.stride(2) == 1,
             f'{what} must be {dtype} [B, Hkv, rows] on CUDA with contiguous rows')
    return t.data_ptr()


def key_mass(q, k, lse, mass, lengths, scale, rows=None, counts=None, decay=1.0, block_tables=None,
             context_only=False, wait_limit_ns=0):
    """Accumulates attention weights per key, in place (``slimkv_key_mass``).

    ``mass [B, Hkv, rows]`` (fp32): entry n becomes ``decay * mass[n] + sum_i
    sum_h exp(scale * q[b, r_i, h] . k[b, n] - lse[b, r_i, h])`` over the
    accepted rows ``r_i = rows[b, i]``, i < ``counts[b]`` (int32 ``[B, T]`` /
    ``[B]``: ``path`` and ``count`` of ``tree.tree_accept``; default: all rows)
    and the heads of the KV head's group, for the ``lengths[b]`` old rows and
    the accepted rows themselves, which follow them after ``tree.tree_commit``
    (row i sees n <= lengths[b] + i; a new row's mass starts from 0).
    ``context_only``: only the ``lengths[b]`` rows (Beacon latents).  ``q [B, T,
    H, D]`` and ``lse [B, T, H]`` as ``tree.tree_attention`` took and returned
    them; for a key set attended in parts, pass the merged lse.  Other entries
    of ``mass`` keep their values.  Returns ``mass``.
    """
    _require(q.is_cuda and q.dim() == 4 and q.stride(3) == 1 and q.dtype in (torch.bfloat16, torch.float16),
             'q must be bf16 or fp16 [B, T, H, D] on CUDA with a contiguous last dimension')
    _require(k.dtype == q.dtype and k.shape[-1] == q.shape[3] and k.device == q.device, 'a cache of q\'s type, dim and device')
    batch, t, heads, dim = q.shape
    _require(lse.is_cuda and lse.dtype == torch.float32 and lse.shape == (batch, t, heads) and lse.is_contiguous(),
             'lse must be contiguous fp32 [B, T, H] on CUDA')
    a = _lib.KeyMassArgs()
    fill_cache(a.cache, k, k, block_tables, batch)
    kv_heads = k.shape[2]
    a.batch, a.nodes, a.heads, a.kv_heads, a.dim, a.type = batch, t, heads, kv_heads, dim, _TYPES[q.dtype]
    a.q, a.lse, a.lengths = q.data_ptr(), lse.data_ptr(), _i32(lengths, (batch,), 'lengths')
    a.q_stride[:] = q.stride()[:3]
    if rows is not None:
        a.rows = _i32(rows, (batch, t), 'rows')
    if counts is not None:
        a.counts = _i32(counts, (batch,), 'counts')
    a.mass, a.mass_rows = _plane(mass, torch.float32, batch, kv_heads, 'mass'), mass.shape[2]
    a.mass_stride[:] = mass.stride()[:2]
    a.context_only, a.scale, a.decay, a.wait_limit_ns = int(bool(context_only)), float(scale), float(decay), int(wait_limit_ns)
    with torch.cuda.device(q.device):
        _lib.check(_lib.load().slimkv_key_mass(ctypes.byref(a), _stream()))
    return mass


def evict(k, v, mass, positions, lengths, keep, sinks=0, recent=0, block_tables=None, out=None):
    """Keeps ``min(lengths[b], keep)`` rows of each (sequence, KV head)
    (``slimkv_evict``).

    ``k`` / ``v [B, rows, Hkv, D]`` (or pages with ``block_tables``; any 1-, 2-
    or 4-byte type), ``mass [B, Hkv, rows]`` fp32, ``positions`` int32 of that
    shape or None.  The first ``sinks`` and the last ``recent`` rows stay, then
    those of the largest mass (ties: the lowest row), all in their order.
    Returns ``(k, v, mass, positions, lengths)`` of ``keep`` rows, zeros past a
    sequence's new length; ``out = (k, v, mass, positions)`` gives buffers (at
    least ``keep`` rows, not the inputs) to write instead of new ones.
    """
    _require(mass.dim() == 3 and k.dim() == 4, 'mass must be [B, Hkv, rows], caches [B, rows, Hkv, D]')
    batch, heads = mass.shape[0], k.shape[2]
    a = _lib.EvictArgs()
    fill_cache(a.src, k, v, block_tables, batch)
    keep = int(keep)
    if out is None:
        # Each (sequence, head) a contiguous run of rows.
        out_k = torch.empty((batch, heads, keep, k.shape[3]), dtype=k.dtype, device=k.device).transpose(1, 2)
        out_v = torch.empty((batch, heads, keep, v.shape[3]), dtype=v.dtype, device=k.device).transpose(1, 2)
        out_mass = torch.empty((batch, heads, keep), dtype=torch.float32, device=k.device)
        out_positions = None if positions is None else torch.empty((batch, heads, keep), dtype=torch.int32, device=k.device)
    else:
        out_k, out_v, out_mass, out_positions = out
        _require(out_k.shape[0] == batch and out_k.shape[2:] == k.shape[2:] and out_v.shape[2:] == v.shape[2:] and
                 out_k.dtype == k.dtype and out_k.shape[1] >= keep, 'out caches must be like the caches, with keep rows')
        _require((positions is None) == (out_positions is None), 'positions and their output go together')
        _require(out_mass.shape[2] >= keep and (out_positions is None or out_positions.shape[2] >= keep),
                 'out planes need keep rows')
    fill_cache(a.dst, out_k, out_v, None, batch)
    a.dst.k_stride[0], a.dst.v_stride[0] = out_k.stride(0), out_v.stride(0)
    a.batch, a.kv_heads, a.dim_qk, a.dim_v, a.elem_bytes = batch, heads, k.shape[3], v.shape[3], k.element_size()
    a.mass, a.mass_rows = _plane(mass, torch.float32, batch, heads, 'mass'), mass.shape[2]
    a.mass_stride[:] = mass.stride()[:2]
    a.out_mass = _plane(out_mass, torch.float32, batch, heads, 'out mass')
    a.out_mass_stride[:] = out_mass.stride()[:2]
    if positions is not None:
        _require(positions.shape == mass.shape, 'positions must be shaped like mass')
        a.positions = _plane(positions, torch.int32, batch, heads, 'positions')
        a.positions_stride[:] = positions.stride()[:2]
        a.out_positions = _plane(out_positions, torch.int32, batch, heads, 'out positions')
        a.out_positions_stride[:] = out_positions.stride()[:2]
    new_lengths = torch.empty(batch, dtype=torch.int32, device=k.device)
    a.lengths, a.new_lengths = _i32(lengths, (batch,), 'lengths'), new_lengths.data_ptr()
    a.keep, a.sinks, a.recent = keep, int(sinks), int(recent)
    lib = _lib.load()
    with torch.cuda.device(k.device):
        size = lib.slimkv_evict_workspace_size(ctypes.byref(a))
        ws = torch.empty(size, dtype=torch.uint8, device=k.device)
        _lib.check(lib.slimkv_evict(ctypes.byref(a), _ptr(ws), size, _stream()))
    return out_k, out_v, out_mass, out_positions, new_lengths
