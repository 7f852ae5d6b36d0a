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
from ctypes import byref

import torch

from . import _lib

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


# A decode step makes these calls once per layer, outside a graph with the
# launch itself as their only other cost: the checks build no text unless they
# fail, the device is only switched to when it is another one, and new tensors
# come from empty_strided (1.5 us; empty with a shape and a type 2.3).
def _refuse(msg, *args):
    raise RuntimeError(msg % args)


def _i32(t, shape, device, what):
    if not (t.device == device and t.dtype == torch.int32 and t.shape == shape and t.is_contiguous()):
        _refuse('%s must be contiguous int32 %s on %s', what, list(shape), device)
    return t.data_ptr()


def _run(device, call, *args):
    """``call(*args, stream)`` on ``device`` and its current stream; raises its error."""
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _run_in_workspace(device, size_of, call, a):
    """``call(a, workspace, bytes, stream)`` with a new workspace of ``size_of(a)``
    bytes (0: the call itself refuses its arguments)."""
    index = device.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(index):
            return _run_in_workspace(device, size_of, call, a)
    args = byref(a)
    size = size_of(args)
    workspace = torch.empty(size, dtype=torch.uint8, device=device)
    rc = call(args, workspace.data_ptr(), size, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc)


def _check_rows(k, v, dims):
    if not (k.is_cuda and v.is_cuda and k.dim() == v.dim() == dims and k.dtype == v.dtype and k.device == v.device):
        _refuse('caches must be CUDA tensors [B, rows, Hkv, D] (or pages) of one type on one device')


def fill_cache(c, k, v, block_tables, batch, first=0):
    """``slimkv_cache`` of k / v ``[B or 1, rows, Hkv, D]`` (dense; 1: shared by
    the batch) or ``[pages, page, Hkv, D]`` with int32 ``block_tables [B, n]``;
    ``first`` dimensions in front are the caller's."""
    ks, vs, shape, v_shape = k.stride(), v.stride(), k.shape, v.shape
    if ks[-1] != 1 or vs[-1] != 1 or shape[:-1] != v_shape[:-1]:
        _refuse('caches need a contiguous last dimension, and K and V must agree in all others')
    c.k, c.v, c.rows = k.data_ptr(), v.data_ptr(), shape[first + 1]
    sequences = shape[first]
    x, y = c.k_stride, c.v_stride
    x[0], x[1], x[2] = ks[first:first + 3]
    y[0], y[1], y[2] = vs[first:first + 3]
    if block_tables is None:
        if sequences != batch:
            if sequences != 1:
                _refuse('one cache for each sequence, or one for all')
            x[0] = y[0] = 0
    else:
        if not (block_tables.device == k.device and block_tables.dtype == torch.int32 and block_tables.dim() == 2 and
                block_tables.shape[0] == batch and block_tables.stride(1) == 1):
            _refuse('block tables must be int32 [B, n] on the caches\' device')
        c.table, c.table_stride = block_tables.data_ptr(), block_tables.stride(0)
        c.table_pages, c.num_pages = block_tables.shape[1], sequences


def tree_masks(parents):
    """Ancestor words of drafted trees (``slimkv_tree_masks``): ``parents [B,
    T]`` int32 (a parent before its children; -1: a root) -> int32 ``[B, T,
    (T + 31) // 32]``, bit i of node t set when t sees i (its ancestors and
    itself)."""
    if not (parents.is_cuda and parents.dim() == 2):
        _refuse('parents must be [B, T] on CUDA')
    p = _i32(parents, parents.shape, parents.device, 'parents')
    batch, nodes = parents.shape
    out = torch.empty((batch, nodes, (nodes + 31) // 32), dtype=torch.int32, device=parents.device)
    _run(parents.device, _lib.load().slimkv_tree_masks, p, batch, nodes, out.data_ptr())
    return out


def attention_args(q, k, v, lengths, scale, mask, nodes, block_tables, context_only, out, lse, wait_limit_ns,
                   cache_type=None, dim_qk=None, dim_v=None):
    """``slimkv_tree_attention_args`` of a call, with its outputs: ``(args, out,
    lse)``.  ``cache_type``: that of the caches' elements (default: q's), whose
    rows have ``dim_qk`` / ``dim_v`` elements (default: the queries' and V's)."""
    kind = q.dtype
    if not (q.is_cuda and q.dim() == 4 and kind in (torch.bfloat16, torch.float16)):
        _refuse('q must be bf16 or fp16 [B, T, H, D] on CUDA')
    batch, t, heads, dim = q.shape
    qs, dev = q.stride(), q.device
    _check_rows(k, v, 4)
    if qs[3] != 1 or k.dtype != (cache_type or kind) or k.shape[3] != (dim_qk or dim) or k.device != dev:
        _refuse('q needs a contiguous last dimension, and caches of its type, dim and device')
    a = _lib.TreeAttentionArgs()
    fill_cache(a.cache, k, v, block_tables, batch)
    dim_v = dim_v or v.shape[3]
    if out is None:
        out = torch.empty_strided((batch, t, heads, dim_v), (t * heads * dim_v, heads * dim_v, dim_v, 1), dtype=kind, device=dev)
    elif not (out.shape == (batch, t, heads, dim_v) and out.dtype == kind and out.device == dev and out.stride(3) == 1):
        _refuse('out must be [B, T, H, Dv] of q\'s type')
    if lse is None:
        lse = torch.empty_strided((batch, t, heads), (t * heads, heads, 1), dtype=torch.float32, device=dev)
    elif not (lse.shape == (batch, t, heads) and lse.dtype == torch.float32 and lse.device == dev and lse.is_contiguous()):
        _refuse('lse must be contiguous fp32 [B, T, H]')
    a.batch, a.nodes, a.heads, a.kv_heads = batch, t, heads, k.shape[2]
    a.dim_qk, a.dim_v, a.type = dim, dim_v, _TYPES[kind]
    a.q, a.out, a.lse, a.lengths = q.data_ptr(), out.data_ptr(), lse.data_ptr(), _i32(lengths, (batch,), dev, 'lengths')
    x, y = a.q_stride, a.out_stride
    x[0], x[1], x[2] = qs[:3]
    y[0], y[1], y[2] = out.stride()[:3]
    if nodes is not None:
        a.nodes_len = _i32(nodes, (batch,), dev, 'nodes')
    if mask is not None:
        if context_only:
            _refuse('the nodes\' own rows are not in a context_only cache: no mask')
        many = mask.shape[0] if mask.dim() == 3 else 0
        if many not in (1, batch):
            _refuse('mask must be [B or 1, T, words]')
        a.mask = _i32(mask, (many, t, (t + 31) // 32), dev, 'mask')
        a.mask_stride = mask.stride(0) if many > 1 else 0
    a.context_only, a.scale, a.wait_limit_ns = bool(context_only), scale, wait_limit_ns
    return a, out, lse


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
    a, out, lse = attention_args(q, k, v, lengths, scale, mask, nodes, block_tables, context_only, out, lse, wait_limit_ns)
    lib = _lib.load()
    _run_in_workspace(q.device, lib.slimkv_tree_attention_workspace_size, lib.slimkv_tree_attention, a)
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
    if not (logits.is_cuda and logits.dim() == 3 and logits.dtype in _TYPES and logits.stride(2) == 1):
        _refuse('logits must be bf16, fp16 or fp32 [B, T, V] on CUDA with a contiguous last dimension')
    batch, t, vocab = logits.shape
    dev = logits.device
    if not (tokens.dtype == torch.int64 and tokens.shape == (batch, t) and tokens.device == dev and tokens.is_contiguous()):
        _refuse('tokens must be contiguous int64 [B, T] on the logits\' device')
    a = _lib.TreeAcceptArgs()
    a.batch, a.nodes, a.vocab, a.type = batch, t, vocab, _TYPES[logits.dtype]
    a.logits, a.tokens, a.parents = logits.data_ptr(), tokens.data_ptr(), _i32(parents, (batch, t), dev, 'parents')
    a.logits_stride[0], a.logits_stride[1] = logits.stride()[:2]
    if nodes is not None:
        a.nodes_len = _i32(nodes, (batch,), dev, 'nodes')
    path = torch.empty_strided((batch, t), (t, 1), dtype=torch.int32, device=dev)
    count = torch.empty_strided((batch,), (1,), dtype=torch.int32, device=dev)
    following = torch.empty_strided((batch,), (1,), dtype=torch.int64, device=dev)
    a.path, a.count, a.next = path.data_ptr(), count.data_ptr(), following.data_ptr()
    lib = _lib.load()
    _run_in_workspace(dev, lib.slimkv_tree_accept_workspace_size, lib.slimkv_tree_accept, a)
    return path, count, following


def tree_commit(k, v, lengths, path, count, block_tables=None):
    """Moves the accepted nodes' rows next to the context, in place
    (``slimkv_tree_commit``): cache row ``lengths[b] + path[b, i]`` becomes row
    ``lengths[b] + i`` for ``i < count[b]``.

    ``k`` / ``v`` one layer ``[B, rows, Hkv, D]`` (or pages with
    ``block_tables``), or every layer at once with a leading layer dimension;
    any 1-, 2- or 4-byte type.  K and V may be (parts of) the same rows; each
    sequence has rows of its own.  ``path`` / ``count`` as :func:`tree_accept`
    returns them.  Returns the new lengths (int32 ``[B]``).
    """
    first = k.dim() - 4
    if first not in (0, 1) or path.dim() != 2:
        _refuse('k and v must be [(layers,) B, rows, Hkv, D], path [B, T]')
    _check_rows(k, v, 4 + first)
    batch, t = path.shape
    shape, v_dim, dev = k.shape, v.shape[-1], k.device
    if block_tables is None and shape[first] != batch:
        _refuse('one cache for each sequence')
    a = _lib.TreeCommitArgs()
    fill_cache(a.cache, k, v, block_tables, batch, first)
    a.layers, a.batch, a.nodes, a.kv_heads = shape[0] if first else 1, batch, t, shape[-2]
    a.dim_qk, a.dim_v, a.elem_bytes = shape[-1], v_dim, k.element_size()
    if first:
        a.k_layer_stride, a.v_layer_stride = k.stride(0), v.stride(0)
    new_lengths = torch.empty_strided((batch,), (1,), dtype=torch.int32, device=dev)
    a.lengths, a.path, a.count = (_i32(lengths, (batch,), dev, 'lengths'), _i32(path, (batch, t), dev, 'path'),
                                  _i32(count, (batch,), dev, 'count'))
    a.new_lengths = new_lengths.data_ptr()
    _run(dev, _lib.load().slimkv_tree_commit, byref(a))
    return new_lengths
