"""The C entries of tree attention, acceptance, commit, key mass and eviction
refuse arguments on the host, before any device work (null streams, no GPU)."""
import ctypes

import pytest

from slimkv_b200 import _lib

P = 4096        # an aligned address that nothing reads: each case is refused first


def cache(c, rows=64, dim=64, heads=2):
    c.k = c.v = P
    c.rows = rows
    for s in (c.k_stride, c.v_stride):
        s[0], s[1], s[2] = rows * heads * dim, heads * dim, dim


def attention(**kw):
    a = _lib.TreeAttentionArgs()
    a.batch, a.nodes, a.heads, a.kv_heads, a.dim_qk, a.dim_v, a.type, a.scale = 2, 4, 8, 2, 64, 64, 0, 0.1
    cache(a.cache)
    a.q = a.out = a.lse = a.lengths = P
    for s in (a.q_stride, a.out_stride):
        s[0], s[1], s[2] = 4 * 8 * 64, 8 * 64, 64
    return fill(a, kw)


def accept(**kw):
    a = _lib.TreeAcceptArgs()
    a.batch, a.nodes, a.vocab, a.type = 2, 4, 100, 2
    a.logits = a.tokens = a.parents = a.path = a.count = a.next = P
    a.logits_stride[0], a.logits_stride[1] = 400, 100
    return fill(a, kw)


def commit(**kw):
    a = _lib.TreeCommitArgs()
    a.layers, a.batch, a.nodes, a.kv_heads, a.dim_qk, a.dim_v, a.elem_bytes = 1, 2, 4, 2, 64, 64, 2
    cache(a.cache)
    a.lengths = a.path = a.count = a.new_lengths = P
    return fill(a, kw)


def mass(**kw):
    a = _lib.KeyMassArgs()
    a.batch, a.nodes, a.heads, a.kv_heads, a.dim, a.type, a.scale, a.decay = 2, 4, 8, 2, 64, 0, 0.1, 1.0
    cache(a.cache)
    a.q = a.lengths = a.lse = a.mass = P
    a.q_stride[0], a.q_stride[1], a.q_stride[2] = 4 * 8 * 64, 8 * 64, 64
    a.mass_stride[0], a.mass_stride[1], a.mass_rows = 128, 64, 64
    return fill(a, kw)


def evict(**kw):
    a = _lib.EvictArgs()
    a.batch, a.kv_heads, a.dim_qk, a.dim_v, a.elem_bytes = 2, 2, 64, 64, 2
    cache(a.src)
    cache(a.dst)
    a.dst.k = a.dst.v = 2 * P
    a.lengths = a.mass = a.new_lengths = P
    a.out_mass = 2 * P
    for s in (a.mass_stride, a.out_mass_stride):
        s[0], s[1] = 128, 64
    a.mass_rows, a.keep, a.sinks, a.recent = 64, 32, 4, 8
    return fill(a, kw)


def fill(a, kw):
    for name, value in kw.items():
        *path, last = name.split('__')
        at = a
        for p in path:
            at = getattr(at, p)
        if last.startswith('x'):                    # an entry of an array: name__x2
            at[int(last[1:])] = value
        else:
            setattr(at, last, value)
    return a


INVALID, SHAPE, ALIGNMENT, WORKSPACE = 1, 2, 3, 4

CASES = [
    ('slimkv_tree_attention', attention, [
        (dict(batch=0), INVALID), (dict(batch=4097), INVALID), (dict(nodes=0), INVALID), (dict(nodes=1025), INVALID),
        (dict(heads=7), INVALID), (dict(heads=258), SHAPE), (dict(dim_qk=60), SHAPE), (dict(dim_qk=328), SHAPE),
        (dict(dim_v=0), SHAPE), (dict(type=2), INVALID), (dict(q=0), INVALID), (dict(lengths=0), INVALID),
        (dict(lse=0), INVALID), (dict(cache__k=0), INVALID), (dict(cache__v=0), INVALID), (dict(cache__rows=0), INVALID),
        (dict(scale=0.0), INVALID), (dict(scale=float('nan')), INVALID), (dict(scale=float('inf')), INVALID),
        (dict(q_stride__x1=4), ALIGNMENT), (dict(q=P + 8), ALIGNMENT), (dict(cache__k=P + 2), ALIGNMENT),
        (dict(cache__v_stride__x1=65), ALIGNMENT), (dict(cache__table=P), INVALID),
        (dict(cache__table=P, cache__table_pages=2, cache__num_pages=2, cache__table_stride=2, cache__rows=12), SHAPE),
        (dict(), WORKSPACE)]),
    ('slimkv_tree_accept', accept, [
        (dict(batch=0), INVALID), (dict(nodes=0), INVALID), (dict(nodes=1025), INVALID), (dict(vocab=0), INVALID),
        (dict(type=3), INVALID), (dict(logits=0), INVALID), (dict(parents=0), INVALID), (dict(next=0), INVALID),
        (dict(logits_stride__x1=-1), INVALID), (dict(), WORKSPACE)]),
    ('slimkv_key_mass', mass, [
        (dict(batch=0), INVALID), (dict(nodes=1025), INVALID), (dict(heads=7), INVALID), (dict(mass_rows=0), INVALID),
        (dict(heads=258), SHAPE), (dict(dim=12), SHAPE), (dict(dim=328), SHAPE), (dict(type=2), INVALID),
        (dict(scale=float('nan')), INVALID), (dict(decay=float('inf')), INVALID), (dict(q_stride__x0=4), ALIGNMENT),
        (dict(q=P + 2), ALIGNMENT), (dict(cache__k=0), INVALID), (dict(cache__k=P + 2), ALIGNMENT), (dict(mass=0), INVALID)]),
    ('slimkv_evict', evict, [
        (dict(batch=0), INVALID), (dict(mass_rows=0), INVALID), (dict(keep=0), INVALID), (dict(sinks=30), INVALID),
        (dict(recent=-1), INVALID), (dict(elem_bytes=8), INVALID), (dict(lengths=0), INVALID), (dict(out_mass=P), INVALID),
        (dict(positions=P), INVALID), (dict(dst__rows=16), INVALID), (dict(dst__k=P), INVALID),
        (dict(src__k=P + 2), ALIGNMENT), (dict(src__v=0), INVALID), (dict(), WORKSPACE)]),
    ('slimkv_tree_commit', commit, [
        (dict(layers=0), INVALID), (dict(batch=0), INVALID), (dict(nodes=1025), INVALID), (dict(elem_bytes=3), INVALID),
        (dict(path=0), INVALID), (dict(new_lengths=0), INVALID), (dict(cache__k=0), INVALID),
        (dict(cache__k_stride__x1=65), ALIGNMENT), (dict(layers=2, k_layer_stride=4), ALIGNMENT)]),
]


@pytest.mark.parametrize('entry,make,change,code', [(e, m, c, k) for e, m, cases in CASES for c, k in cases])
def test_refusals(entry, make, change, code):
    a, call = make(**change), getattr(_lib.load(), entry)
    without = entry in ('slimkv_key_mass', 'slimkv_tree_commit')
    assert call(ctypes.byref(a), *(() if without else (None, 0)), None) == code
    assert _lib.load().slimkv_last_error()


@pytest.mark.parametrize('entry', [c[0] for c in CASES])
def test_null_arguments(entry):
    without = entry in ('slimkv_key_mass', 'slimkv_tree_commit')
    assert getattr(_lib.load(), entry)(None, *(() if without else (None, 0)), None) == INVALID


def test_workspace_sizes():
    """Refused arguments have none.  (Tree attention's is one share for each SM, so it needs a device.)"""
    lib = _lib.load()
    for size, make, bad in ((lib.slimkv_tree_accept_workspace_size, accept, dict(vocab=0)),
                            (lib.slimkv_evict_workspace_size, evict, dict(keep=0))):
        assert size(ctypes.byref(make())) > 0
        assert size(ctypes.byref(make(**bad))) == 0
    size = lib.slimkv_tree_attention_workspace_size
    assert size(ctypes.byref(attention(dim_qk=60))) == 0
    assert size(ctypes.byref(attention())) == size(ctypes.byref(attention(cache__rows=100000)))


def test_masks_refusals():
    lib = _lib.load()
    for args in ((None, 2, 4, P), (P, 2, 4, None), (P, 0, 4, P), (P, 2, 1025, P), (P, 2, 0, P)):
        assert lib.slimkv_tree_masks(*args, None) == INVALID


@pytest.mark.parametrize('entry,make,workspace', [('slimkv_tree_commit', commit, ()), ('slimkv_evict', evict, (P, 1 << 20))])
@pytest.mark.parametrize('apart', [0, 4, -4])
def test_new_lengths_are_not_the_lengths(entry, make, workspace, apart):
    """Two sequences' lengths: the arrays are the same, or share one entry."""
    assert getattr(_lib.load(), entry)(ctypes.byref(make(new_lengths=P + apart)), *workspace, None) == INVALID
    assert b'new_lengths' in _lib.load().slimkv_last_error()


@pytest.mark.parametrize('change', [
    dict(cache__v=P + 128),                                     # V a head of K's further on
    dict(cache__v=P + 2 * 64 * 2),                              # a row further on
    dict(cache__v=P + 64 * 2 * 64 * 2),                         # a sequence further on
    dict(cache__v_stride__x1=64),                               # the same place in another order
    dict(cache__v=P + 64, dim_v=96),                            # V past the end of K's head, into the next
    dict(layers=2, k_layer_stride=2 * 64 * 2 * 64, v_layer_stride=64 * 2 * 64)])
def test_commit_refuses_keys_and_values_that_share_rows_in_part(change):
    assert _lib.load().slimkv_tree_commit(ctypes.byref(commit(**dict(dict(new_lengths=2 * P), **change))), None) == INVALID
    assert b'K and V' in _lib.load().slimkv_last_error()


@pytest.mark.parametrize('which', ['k', 'v'])
def test_commit_refuses_a_cache_shared_by_the_batch(which):
    """Every sequence would move the same rows."""
    a = commit(new_lengths=2 * P, cache__v=64 * P, **{f'cache__{which}_stride__x0': 0})
    assert _lib.load().slimkv_tree_commit(ctypes.byref(a), None) == INVALID
    assert b'each sequence' in _lib.load().slimkv_last_error()


I = 16 * P      # where an input lies


@pytest.mark.parametrize('change', [
    dict(dst__k=I + 2 * 64 * 2 * 4),                            # the input from its fourth row on
    dict(dst__v=I + 2 * 64 * 2 * 63),                           # from its last row on
    dict(dst__k=I - 2 * 64 * 2 * 31),                           # up to its first row
    dict(dst__k=I + 64 * 2 * 64 * 2),                           # from its second sequence on
    dict(dst__k_stride__x1=64, dst__k_stride__x2=64 * 64, dst__k=I + 64 * 2 * 64 * 2),      # the same in another order
    dict(out_mass=I + 4 * 63), dict(out_mass=I - 4 * 31), dict(positions=I, out_positions=I + 4 * 32)])
def test_evict_refuses_an_output_over_its_input(change):
    far = dict(src__k=I, src__v=I, mass=I, dst__k=4 * I, dst__v=8 * I, out_mass=12 * I, new_lengths=16 * I)
    a = evict(**dict(far, **change))
    assert _lib.load().slimkv_evict(ctypes.byref(a), P, 1 << 20, None) == INVALID
    assert b'overlap' in _lib.load().slimkv_last_error()


@pytest.mark.parametrize('which', ['k', 'v'])
@pytest.mark.parametrize('dim', [0, 1, 2])
def test_evict_refuses_output_rows_in_one_place(which, dim):
    a = evict(src__k=I, src__v=I, mass=I, dst__k=4 * I, dst__v=8 * I, out_mass=12 * I, new_lengths=16 * I,
              **{f'dst__{which}_stride__x{dim}': 0})
    assert _lib.load().slimkv_evict(ctypes.byref(a), P, 1 << 20, None) == INVALID
    assert b'own place' in _lib.load().slimkv_last_error()


@pytest.mark.parametrize('batch,nodes,vocab,kind', [(1, 1024, 33001, 0), (4, 70, 64001, 2), (2, 256, 128256, 0), (8, 1024, 128256, 0)])
def test_long_paths_are_not_left_to_serial_steps(batch, nodes, vocab, kind):
    """Where every node may be accepted and walking them costs many scans of all, the call has room for the scan's argmaxes."""
    a = accept(batch=batch, nodes=nodes, vocab=vocab, type=kind)
    assert _lib.load().slimkv_tree_accept_workspace_size(ctypes.byref(a)) >= 8 * batch * nodes
