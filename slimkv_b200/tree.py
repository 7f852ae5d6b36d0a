"""Verification of a drafted token tree over a cache.

A speculative step drafts a tree of tokens behind the last accepted one
(node 0), runs the model once over all its nodes, and keeps the longest path
from the root that the model itself would have taken:

* :func:`tree_masks` — which nodes each node sees, once per tree;
* :func:`tree_attention` — each layer's attention of the nodes over the
  context and their ancestors (dense caches, serving pages, or the Beacon
  latents with ``context_only``);
* :func:`tree_accept` — greedy acceptance from the step's logits;
* :func:`tree_commit` — the accepted nodes' K/V rows moved next to the
  context, in place.

The reference verifies no drafts (its decode takes one raw token and a
Beacon, slimkv/llama3/fa2_decode.py:77-166); these entry points stand beside
that decode.  Torch wrappers over ``include/slimkv_b200.h``: checks, current
stream, workspaces from PyTorch's allocator (calls can be captured in CUDA
graphs).  There is no CPU path.
"""
import ctypes

import torch

from . import _lib
from .kernels import _ptr, _require, _stream

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _i32(t, shape, what):
    _require(t.is_cuda and t.dtype == torch.int32 and t.is_contiguous() and t.shape == shape,
             f'{what} must be contiguous int32 {list(shape)} on CUDA')
    return t.data_ptr()


def fill_cache(c, k, v, block_tables, batch):
    """``slimkv_cache`` of k / v ``[B or 1, rows, Hkv, D]`` (dense; 1: shared by
    the batch) or ``[pages, page, Hkv, D]`` with int32 ``block_tables [B, n]``."""
    for x, stride in ((k, c.k_stride), (v, c.v_stride)):
        _require(x.is_cuda and x.dim() == 4 and x.stride(3) == 1 and x.dtype == k.dtype,
                 'caches must be [B, rows, Hkv, D] (or pages) on CUDA with a contiguous last dimension')
        stride[:] = x.stride()[:3]
    _require(k.shape[:3] == v.shape[:3] and k.device == v.device, 'K and V must agree in all but their last dimension')
    c.k, c.v, c.rows = k.data_ptr(), v.data_ptr(), k.shape[1]
    if block_tables is None:
        _require(k.shape[0] in (1, batch), 'one cache for each sequence, or one for all')
        if k.shape[0] == 1:
            c.k_stride[0] = c.v_stride[0] = 0
    else:
        _require(block_tables.is_cuda and block_tables.dtype == torch.int32 and block_tables.dim() == 2 and
                 block_tables.shape[0] == batch and block_tables.stride(1) == 1, 'block tables must be int32 [B, n] on CUDA')
        c.table, c.table_stride = block_tables.data_ptr(), block_tables.stride(0)
        c.table_pages, c.num_pages = block_tables.shape[1], k.shape[0]


def tree_masks(parents):
    """Ancestor words of drafted trees (``slimkv_tree_masks``): ``parents [B,
    T]`` int32 (a parent before its children; -1: a root) -> int32 ``[B, T,
    (T + 31) // 32]``, bit i of node t set when t sees i (its ancestors and
    itself)."""
    _require(parents.dim() == 2, 'parents must be [B, T]')
    p = _i32(parents, parents.shape, 'parents')
    batch, nodes = parents.shape
    out = torch.empty((batch, nodes, (nodes + 31) // 32), dtype=torch.int32, device=parents.device)
    with torch.cuda.device(parents.device):
        _lib.check(_lib.load().slimkv_tree_masks(p, batch, nodes, _ptr(out), _stream()))
    return out


def tree_attention(q, k, v, lengths, scale, mask=None, nodes=None, block_tables=None, context_only=False, out=None,
                   lse=None, wait_limit_ns=0):
    """Attention of drafted nodes over a cache (``slimkv_tree_attention``).

    ``q [B, T, H, D]`` (bf16 or fp16, rotated); ``k`` / ``v`` dense ``[B, rows,
    Hkv, D / Dv]`` (``[1, ...]``: shared) or pages ``[n, page, Hkv, ...]`` with
    int32 ``block_tables [B, pages]``.  Node t of sequence b sees the
    ``lengths[b]`` (int32) context rows and, of the rows ``lengths[b] + i``
    that hold the nodes' own K/V, those whose bit is set in ``mask`` (int32
    ``[B or 1, T, (T + 31) // 32]``, :func:`tree_masks`); without a mask the
    nodes are a chain (a single token: T = 1).  ``nodes`` (int32 ``[B]``)
    limits a sequence to its first nodes.  ``context_only``: the cache holds no
    rows of the nodes (Beacon latents: absorbed queries, one KV head).
    Returns ``(out [B, T, H, Dv], lse [B, T, H] fp32 natural log)``; a row that
    sees nothing gets zeros and -inf.  Dims: multiples of 8 up to 320.
    """
    _require(q.is_cuda and q.dim() == 4 and q.stride(3) == 1 and q.dtype in (torch.bfloat16, torch.float16),
             'q must be bf16 or fp16 [B, T, H, D] on CUDA with a contiguous last dimension')
    _require(k.dtype == q.dtype and k.shape[-1] == q.shape[3] and k.device == q.device, 'caches of q\'s type, dim and device')
    batch, t, heads, dim = q.shape
    a = _lib.TreeAttentionArgs()
    fill_cache(a.cache, k, v, block_tables, batch)
    dim_v = v.shape[3]
    if out is None:
        out = torch.empty((batch, t, heads, dim_v), dtype=q.dtype, device=q.device)
    if lse is None:
        lse = torch.empty((batch, t, heads), dtype=torch.float32, device=q.device)
    _require(out.shape == (batch, t, heads, dim_v) and out.dtype == q.dtype and out.is_cuda and out.stride(3) == 1,
             'out must be [B, T, H, Dv] of q\'s type')
    _require(lse.shape == (batch, t, heads) and lse.dtype == torch.float32 and lse.is_cuda and lse.is_contiguous(),
             'lse must be contiguous fp32 [B, T, H]')
    a.batch, a.nodes, a.heads, a.kv_heads, a.dim_qk, a.dim_v, a.type = (batch, t, heads, k.shape[2], dim, dim_v,
                                                                        _TYPES[q.dtype])
    a.q, a.out, a.lse, a.lengths = q.data_ptr(), out.data_ptr(), lse.data_ptr(), _i32(lengths, (batch,), 'lengths')
    a.q_stride[:] = q.stride()[:3]
    a.out_stride[:] = out.stride()[:3]
    if nodes is not None:
        a.nodes_len = _i32(nodes, (batch,), 'nodes')
    if mask is not None:
        _require(not context_only, 'the nodes\' own rows are not in a context_only cache: no mask')
        _require(mask.dim() == 3 and mask.shape[0] in (1, batch), 'mask must be [B or 1, T, words]')
        a.mask = _i32(mask, (mask.shape[0], t, (t + 31) // 32), 'mask')
        a.mask_stride = mask.stride(0) if mask.shape[0] > 1 else 0
    a.context_only, a.scale, a.wait_limit_ns = int(bool(context_only)), float(scale), int(wait_limit_ns)
    lib = _lib.load()
    with torch.cuda.device(q.device):
        size = lib.slimkv_tree_attention_workspace_size(ctypes.byref(a))
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        _lib.check(lib.slimkv_tree_attention(ctypes.byref(a), _ptr(ws), size, _stream()))
    return out, lse


def tree_accept(logits, tokens, parents, nodes=None):
    """Greedy acceptance of drafted trees (``slimkv_tree_accept``).

    ``logits [B, T, V]`` (bf16, fp16 or fp32, contiguous last dimension),
    ``tokens [B, T]`` int64 (the nodes' drafted tokens; node 0 holds the last
    accepted one), ``parents [B, T]`` int32.  Returns ``(path [B, T] int32,
    count [B] int32, next_token [B] int64)``: the accepted nodes from the root
    on (-1 past them), their number, and the model's token after the last.
    Ties of the largest logit go to the lowest token; a NaN counts above every
    number.
    """
    _require(logits.is_cuda and logits.dim() == 3 and logits.stride(2) == 1 and logits.dtype in _TYPES,
             'logits must be bf16, fp16 or fp32 [B, T, V] on CUDA with a contiguous last dimension')
    batch, t, vocab = logits.shape
    _require(tokens.is_cuda and tokens.dtype == torch.int64 and tokens.shape == (batch, t) and tokens.is_contiguous(),
             'tokens must be contiguous int64 [B, T] on CUDA')
    a = _lib.TreeAcceptArgs()
    a.batch, a.nodes, a.vocab, a.type = batch, t, vocab, _TYPES[logits.dtype]
    a.logits, a.tokens, a.parents = logits.data_ptr(), tokens.data_ptr(), _i32(parents, (batch, t), 'parents')
    a.logits_stride[:] = logits.stride()[:2]
    if nodes is not None:
        a.nodes_len = _i32(nodes, (batch,), 'nodes')
    dev = logits.device
    path = torch.empty((batch, t), dtype=torch.int32, device=dev)
    count = torch.empty(batch, dtype=torch.int32, device=dev)
    following = torch.empty(batch, dtype=torch.int64, device=dev)
    a.path, a.count, a.next = path.data_ptr(), count.data_ptr(), following.data_ptr()
    lib = _lib.load()
    with torch.cuda.device(dev):
        size = lib.slimkv_tree_accept_workspace_size(ctypes.byref(a))
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        _lib.check(lib.slimkv_tree_accept(ctypes.byref(a), _ptr(ws), size, _stream()))
    return path, count, following


def tree_commit(k, v, lengths, path, count, block_tables=None):
    """Moves the accepted nodes' rows next to the context, in place
    (``slimkv_tree_commit``): cache row ``lengths[b] + path[b, i]`` becomes row
    ``lengths[b] + i`` for ``i < count[b]``.

    ``k`` / ``v`` one layer ``[B, rows, Hkv, D]`` (or pages with
    ``block_tables``), or every layer at once with a leading layer dimension;
    any 1-, 2- or 4-byte type.  ``path`` / ``count`` as :func:`tree_accept`
    returns them.  Returns the new lengths (int32 ``[B]``).
    """
    _require(k.dim() == v.dim() and k.dim() in (4, 5) and k.dtype == v.dtype, 'k and v must be [(layers,) B, rows, Hkv, D]')
    if k.dim() == 4:
        k, v = k.unsqueeze(0), v.unsqueeze(0)
    _require(k.shape[0] == v.shape[0] and k.shape[0] > 0 and path.dim() == 2, 'K and V of the same layers; path [B, T]')
    batch, t = path.shape
    _require(block_tables is not None or k.shape[1] == batch, 'one cache for each sequence')
    a = _lib.TreeCommitArgs()
    fill_cache(a.cache, k[0], v[0], block_tables, batch)
    a.cache.k_stride[0], a.cache.v_stride[0] = k.stride(1), v.stride(1)
    a.layers, a.batch, a.nodes, a.kv_heads = k.shape[0], batch, t, k.shape[3]
    a.dim_qk, a.dim_v, a.elem_bytes = k.shape[4], v.shape[4], k.element_size()
    a.k_layer_stride, a.v_layer_stride = k.stride(0), v.stride(0)
    new_lengths = torch.empty(batch, dtype=torch.int32, device=k.device)
    a.lengths, a.path, a.count = (_i32(lengths, (batch,), 'lengths'), _i32(path, (batch, t), 'path'),
                                  _i32(count, (batch,), 'count'))
    a.new_lengths = new_lengths.data_ptr()
    with torch.cuda.device(k.device):
        _lib.check(_lib.load().slimkv_tree_commit(ctypes.byref(a), _stream()))
    return new_lengths
