"""Accumulated attention weight and eviction (``slimkv_b200.eviction``)
against plain 64-bit forms."""
import ctypes
import math
import random

import pytest
import torch

import tree_oracle as oracle
from slimkv_b200 import _lib, eviction, kernels, tree

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(7)


def make(B, T, H, G, D, lengths, dtype=BF16, page=0, seed=0, spare=9):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    cap = max(lengths) + T + spare
    rand = lambda *s: torch.randn(*s, generator=gen, device='cuda', dtype=dtype)
    tables = None
    if page:
        per = -(-cap // page)
        k = rand(B * per, page, 2, G, D)[:, :, 0]
        tables = torch.randperm(B * per, generator=gen, device='cuda').view(B, per).to(torch.int32)
    else:
        k = rand(B, G, cap, D).transpose(1, 2)
    q = rand(B, T, H, D)
    mass = torch.rand(B, G, cap, generator=gen, device='cuda')
    return q, k, mass, torch.tensor(lengths, dtype=torch.int32, device='cuda'), tables


def check_mass(q, k, lse, mass, lens, scale, **kw):
    old = mass.clone()
    got = eviction.key_mass(q, k, lse, mass, lens, scale, **kw)
    torch.cuda.synchronize()
    assert got is mass and _lib.device_status() == 0
    tables = kw.pop('block_tables', None)
    rows, counts = kw.pop('rows', None), kw.pop('counts', None)
    want, tol = oracle.mass(q, k, lse, old, lens.tolist(), scale, None if rows is None else rows.tolist() and rows.cpu(),
                            None if counts is None else counts.tolist(), tables=tables, **kw)
    off = (mass.double().cpu() - want).abs() - 1.05 * tol
    # Entries past a sequence's rows have a bound of 0: they keep their bits.
    assert off.max() <= 0, f'off its bound by {off.max():.3e}'


@pytest.mark.parametrize('B,T,H,G,D,lengths,dtype,page', [
    (1, 1, 32, 8, 128, [1028], BF16, 0), (2, 3, 8, 2, 128, [0, 300], BF16, 16), (3, 8, 8, 8, 64, [127, 1, 128], FP16, 48),
    (2, 5, 6, 2, 96, [500, 77], BF16, 24), (1, 20, 16, 1, 64, [260], BF16, 0), (2, 70, 8, 1, 128, [129, 40], FP16, 0),
    (1, 2, 3, 1, 8, [50], BF16, 0)])
@pytest.mark.parametrize('decay', [1.0, 0.9])
def test_accepted_rows(B, T, H, G, D, lengths, dtype, page, decay):
    q, k, mass, lens, tables = make(B, T, H, G, D, lengths, dtype, page, seed=T)
    rng = random.Random(T)
    counts = [rng.randint(1, T) for _ in range(B)]
    rows = torch.tensor([sorted(rng.sample(range(T), c)) + [-1] * (T - c) for c in counts], dtype=torch.int32, device='cuda')
    counts = torch.tensor(counts, dtype=torch.int32, device='cuda')
    lse = 3 + torch.rand(B, T, H, device='cuda') * 4
    scale = D ** -0.5
    check_mass(q, k, lse, mass, lens, scale, rows=rows, counts=counts, decay=decay, block_tables=tables)
    check_mass(q, k, lse, mass, lens, scale, decay=decay, block_tables=tables)      # every row


@pytest.mark.parametrize('T,rank,lengths', [(1, 320, [700, 0]), (8, 320, [1000, 129]), (12, 160, [33, 500])])
def test_latents(T, rank, lengths):
    lat = torch.randn(2, 2, max(lengths) + 2, rank, device='cuda').to(BF16)
    for b, n in enumerate(lengths):
        lat[b, :, n:] = math.nan
    k = lat[:, 0].unsqueeze(2)
    q = torch.randn(2, T, 32, rank, device='cuda').to(BF16)
    lens = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    mass = torch.rand(2, 1, k.shape[1], device='cuda')
    lse = 5 + torch.rand(2, T, 32, device='cuda')
    counts = torch.tensor([T, 0], dtype=torch.int32, device='cuda')
    check_mass(q, k, lse, mass, lens, rank ** -0.5, context_only=True, decay=0.5)
    check_mass(q, k, lse, mass, lens, rank ** -0.5, context_only=True, counts=counts)


def test_masses_of_a_row_sum_to_its_heads():
    """With the lse that tree_attention returned, each accepted row gives G * group = H in all."""
    q, k, mass, lens, _ = make(2, 4, 8, 2, 64, [300, 5])
    _, lse = tree.tree_attention(q, k, k, lens, 0.125)
    eviction.key_mass(q, k, lse, mass.zero_(), lens, 0.125)
    assert torch.allclose(mass.sum((1, 2)), torch.full((2,), 32.0, device='cuda'), atol=1e-3)


def test_empty_rows_and_unseen_keys():
    """Rows with lse +inf give nothing, the lse -inf of a row infinite masses to the keys that it sees and no others;
    NaN keys past the end stay out."""
    q, k, mass, lens, _ = make(2, 3, 4, 2, 64, [100, 128])
    k[0, 103:], k[1, 131:] = math.nan, math.inf
    mass[:, :, 131:] = math.nan
    keep = mass.clone()
    lse = torch.full((2, 3, 4), 4.0, device='cuda')
    lse[0, 1], lse[1, 2, 0] = -math.inf, math.inf
    eviction.key_mass(q, k, lse, mass, lens, 0.125)
    want, tol = oracle.mass(q, k, lse, keep, [100, 128], 0.125)
    live = tol > 0
    got, infinite = mass.double().cpu(), want == math.inf
    assert torch.equal(got == math.inf, infinite)
    assert ((got - want).abs() <= 1.05 * tol)[live & ~infinite].all()
    assert torch.equal(mass.cpu()[~live].isnan(), keep.cpu()[~live].isnan())
    assert (mass[0, :, :102] == math.inf).all() and mass[0, :, 102].isfinite().all()


def test_mass_refusals():
    q, k, mass, lens, _ = make(2, 3, 4, 2, 64, [100, 128])
    lse = torch.zeros(2, 3, 4, device='cuda')
    for args in ((q.float(), k, lse, mass, lens, 0.1), (q, k, lse.half(), mass, lens, 0.1), (q, k, lse, mass.double(), lens, 0.1),
                 (q, k, lse, mass, lens.long(), 0.1), (q, k, lse, mass[:, :1], lens, 0.1), (q, k, lse, mass, lens, math.inf),
                 (q, k, lse, mass, lens[:1], 0.1)):
        with pytest.raises(RuntimeError):
            eviction.key_mass(*args)


def test_mass_rows_out_of_the_tree_are_reported():
    q, k, mass, lens, _ = make(1, 3, 4, 2, 64, [100])
    _lib.device_status(clear=True)
    eviction.key_mass(q, k, torch.zeros(1, 3, 4, device='cuda'), mass, lens, 0.1,
                      rows=torch.tensor([[0, 7, -1]], dtype=torch.int32, device='cuda'))
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH


# ------------------------------------------------------------------ evict --
def same(got, want):
    k, v, mass, positions, lengths = got
    for x, y in ((k, want[0]), (v, want[1])):
        assert torch.equal(x.cpu().double(), y)
    m = mass.cpu().double()
    assert torch.equal(m.nan_to_num(nan=-5.0), want[2].nan_to_num(nan=-5.0))
    if positions is not None:
        assert torch.equal(positions.cpu(), want[3])
    assert torch.equal(lengths.cpu(), want[4])
    assert _lib.device_status() == 0


@pytest.mark.parametrize('B,G,D,Dv,lengths,keep,sinks,recent,dtype,page', [
    (1, 1, 8, 8, [1], 1, 0, 0, BF16, 0), (2, 8, 128, 128, [300, 255], 200, 4, 32, BF16, 0), (3, 2, 64, 128, [0, 1000, 513], 512, 4, 0, FP16, 0),
    (2, 1, 320, 320, [3000, 2999], 700, 0, 257, BF16, 0), (1, 4, 16, 4, [70000], 50, 3, 40, torch.float32, 0),
    (2, 2, 64, 64, [400, 33], 256, 2, 2, BF16, 16), (2, 3, 32, 16, [90, 260], 300, 4, 4, torch.uint8, 5), (1, 2, 64, 64, [1025], 1, 0, 1, BF16, 0)])
@pytest.mark.parametrize('kind', ['spread', 'ties', 'odd'])
def test_evict(B, G, D, Dv, lengths, keep, sinks, recent, dtype, page, kind):
    gen = torch.Generator(device='cuda').manual_seed(keep)
    cap = max(lengths) + 3
    per = -(-cap // page) if page else 0
    shape = (B * per, page, G) if page else (B, cap, G)
    k, v = (torch.randint(0, 200, shape + (d,), generator=gen, device='cuda').to(dtype) for d in (D, Dv))
    tables = torch.randperm(B * per, generator=gen, device='cuda').view(B, per).to(torch.int32) if page else None
    mass = torch.randn(B, G, cap, generator=gen, device='cuda').mul_(2).exp_()
    if kind == 'ties':
        mass = (mass > 1).float() * 2
    elif kind == 'odd':
        pick = torch.randint(0, 8, mass.shape, generator=gen, device='cuda')
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, -1.0)):
            mass[pick == i] = x
    positions = torch.randint(0, 1 << 30, mass.shape, generator=gen, device='cuda', dtype=torch.int32)
    lens = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    want = oracle.evict(k, v, mass, positions, lengths, keep, sinks, recent, tables)
    same(eviction.evict(k, v, mass, positions, lens, keep, sinks, recent, block_tables=tables), want)
    same(eviction.evict(k, v, mass, None, lens, keep, sinks, recent, block_tables=tables), want)


@pytest.mark.parametrize('shift', [0, 8, 16, 23])
@pytest.mark.parametrize('n,keep', [(300, 57), (20000, 12345), (40000, 1)])
def test_evict_masses_that_differ_in_one_digit(shift, n, keep):
    """One, two or many equal rows per value; a threshold between values and within one."""
    for each in (1, 2, 300):
        values = (torch.randperm(n, device='cuda') // each) % (256 if shift < 23 else 200)
        mass = ((values.int() << shift) + (0x3f000000 if shift < 23 else 0x00800000)).view(torch.float32)
        mass = torch.stack([mass, -mass]).view(1, 2, n)
        k = torch.randint(0, 200, (1, n, 2, 16), device='cuda').to(BF16)
        lens = torch.tensor([n], dtype=torch.int32, device='cuda')
        same(eviction.evict(k, k, mass, None, lens, keep, 1 if keep > 1 else 0, 3 if keep > 4 else 0),
             oracle.evict(k, k, mass, None, [n], keep, 1 if keep > 1 else 0, 3 if keep > 4 else 0))


def test_evict_into_given_buffers():
    k = torch.randn(2, 500, 2, 64, device='cuda').to(BF16)
    mass = torch.rand(2, 2, 500, device='cuda')
    lens = torch.tensor([500, 90], dtype=torch.int32, device='cuda')
    ok, ov = torch.full((2, 140, 2, 72), 7.0, device='cuda', dtype=BF16), torch.full((2, 2, 140, 64), 7.0, device='cuda', dtype=BF16)
    om = torch.full((2, 2, 140), 7.0, device='cuda')
    got = eviction.evict(k, k, mass, None, lens, 128, sinks=4, recent=16, out=(ok[..., :64], ov.transpose(1, 2), om, None))
    want = oracle.evict(k, k, mass, None, [500, 90], 128, 4, 16)
    same((got[0][:, :128], got[1][:, :128], got[2][..., :128], None, got[4]), want)
    assert (ok[:, 128:] == 7).all() and (ok[..., 64:] == 7).all() and (ov[:, :, 128:] == 7).all() and (om[..., 128:] == 7).all()


def test_evict_refusals():
    k = torch.randn(2, 50, 2, 64, device='cuda').to(BF16)
    mass = torch.rand(2, 2, 50, device='cuda')
    lens = torch.tensor([50, 9], dtype=torch.int32, device='cuda')
    for kw in (dict(keep=0), dict(keep=10, sinks=6, recent=5), dict(keep=10, sinks=-1)):
        with pytest.raises(RuntimeError):
            eviction.evict(k, k, mass, None, lens, **kw)
    with pytest.raises(RuntimeError):
        eviction.evict(k, k, mass.double(), None, lens, 10)
    with pytest.raises(RuntimeError):
        eviction.evict(k, k, mass, mass, lens, 10)
    with pytest.raises(RuntimeError):                    # onto itself
        eviction.evict(k, k.clone(), mass, None, lens, 10, out=(k, k.clone(), mass.clone(), None))
    with pytest.raises(RuntimeError):                    # too small
        eviction.evict(k, k, mass, None, lens, 40, out=(k[:, :20].clone(), k[:, :20].clone(), mass.clone(), None))
    with pytest.raises(RuntimeError):                    # 12-byte rows
        eviction.evict(k[..., :6], k[..., :6], mass, None, lens, 10)


def test_a_bounded_cache_step():
    """Attention, acceptance, commit, mass and eviction, as a serving loop calls them."""
    B, T, H, G, D, V = 2, 6, 8, 2, 64, 97
    rng = random.Random(3)
    lengths = [60, 41]
    q, k, mass, lens, _ = make(B, T, H, G, D, lengths, spare=30)
    v = torch.randn_like(k)
    parents = torch.tensor([[-1, 0, 0, 1, 1, 3], [-1, 0, 1, 2, 0, 4]], dtype=torch.int32, device='cuda')
    _, lse = tree.tree_attention(q, k, v, lens, 0.125, mask=tree.tree_masks(parents))
    logits = torch.randn(B, T, V, device='cuda')
    tokens = torch.arange(B * T, device='cuda').view(B, T)      # all different
    logits[0, 0, tokens[0, 1]] = logits[0, 1, tokens[0, 4]] = 9.0
    path, count, _ = tree.tree_accept(logits, tokens, parents)
    assert path[0].tolist() == [0, 1, 4, -1, -1, -1]
    new = tree.tree_commit(k, v, lens, path, count)
    eviction.key_mass(q, k, lse, mass, lens, 0.125, rows=path, counts=count, decay=0.9)
    positions = torch.arange(k.shape[1], device='cuda', dtype=torch.int32).expand(B, G, -1).contiguous()
    got = eviction.evict(k, v, mass, positions, new, 40, sinks=4, recent=8)
    same(got, oracle.evict(k, v, mass, positions, new.tolist(), 40, 4, 8))
    assert got[4].tolist() == [40, 40] and (got[3][0, :, -8:].cpu() == torch.arange(55, 63)).all()


def test_refusals_of_tensors_elsewhere():
    """What lies on the CPU (or on another GPU) is refused before a launch."""
    q, k, mass, lens, _ = make(2, 3, 4, 2, 64, [30, 20])
    lse = torch.zeros(2, 3, 4, device='cuda')
    path = torch.zeros(2, 3, dtype=torch.int32, device='cuda')
    tables = torch.zeros(2, 4, dtype=torch.int32)
    pages = torch.zeros(8, 16, 2, 64, dtype=BF16, device='cuda')
    for call in (lambda: eviction.key_mass(q, k, lse, mass.cpu(), lens, 0.1), lambda: eviction.key_mass(q, k, lse, mass, lens.cpu(), 0.1),
                 lambda: eviction.key_mass(q, k, lse, mass, lens, 0.1, rows=path.cpu()),
                 lambda: eviction.key_mass(q, k, lse.cpu(), mass, lens, 0.1),
                 lambda: eviction.evict(k, k, mass.cpu(), None, lens, 8), lambda: eviction.evict(k, k, mass, None, lens.cpu(), 8),
                 lambda: eviction.evict(k, k, mass, mass.int().cpu(), lens, 8),
                 lambda: tree.tree_attention(q, k, k, lens.cpu(), 0.1), lambda: tree.tree_attention(q.cpu(), k, k, lens, 0.1),
                 lambda: tree.tree_attention(q, pages, pages, lens, 0.1, block_tables=tables),
                 lambda: tree.tree_commit(k, k.clone(), lens, path.cpu(), lens), lambda: tree.tree_commit(k, k.clone(), lens, path, lens.cpu()),
                 lambda: tree.tree_masks(path.cpu()), lambda: tree.tree_accept(lse, path.long(), path.cpu())):
        with pytest.raises(RuntimeError):
            call()


def test_evict_reads_a_clamped_page_for_one_outside_the_pool():
    """It is reported, and every row of the output is written."""
    pages = torch.randn(6, 16, 2, 64, device='cuda').to(BF16)
    tables = torch.tensor([[3, -7, 1], [99, 0, 5]], dtype=torch.int32, device='cuda')
    mass = torch.rand(2, 2, 48, device='cuda')
    lens = torch.tensor([40, 48], dtype=torch.int32, device='cuda')
    out = [torch.full((2, 20, 2, 64), 7.0, device='cuda', dtype=BF16) for _ in range(2)] + [torch.full((2, 2, 20), 7.0, device='cuda')]
    _lib.device_status(clear=True)
    got = eviction.evict(pages, pages, mass, None, lens, 20, sinks=2, recent=4, block_tables=tables, out=(*out, None))
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH
    same(got, oracle.evict(pages, pages, mass, None, [40, 48], 20, 2, 4, tables.clamp(0, 5)))


@pytest.mark.parametrize('form', ['planes', 'behind', 'sides', 'before'])
def test_evict_within_one_buffer(form):
    """Outputs between or behind the input's rows, none over them."""
    n, keep = 300, 100
    k, v, mass, out = {
        # Two caches of each sequence side by side, their masses too.
        'planes': lambda x, m: (x[:, 0], x[:, 1], m[:, 0], (x[:, 2], x[:, 3], m[:, 1], None)),
        # The rows behind the input's.
        'behind': lambda x, m: (x[:, 0, :n], x[:, 1, :n], m[:, 0, :, :n], (x[:, 0, n:], x[:, 1, n:], m[:, 0, :, n:], None)),
        # Input and output in the halves of each row.
        'sides': lambda x, m: (x[:, 0, ..., :32], x[:, 1, ..., :32], m[:, 0], (x[:, 0, ..., 32:], x[:, 1, ..., 32:], m[:, 1], None)),
        'before': lambda x, m: (x[1:, 0], x[1:, 1], m[1:, 0], (x[:1, 0], x[:1, 1], m[:1, 0], None))}[form](
            torch.randn(2, 4, 500, 3, 64, device='cuda').to(BF16), torch.rand(2, 2, 3, 500, device='cuda'))
    B = k.shape[0]
    lengths = [n, 250][:B]
    lens = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    want = oracle.evict(k.clone(), v.clone(), mass.clone(), None, lengths, keep, 4, 16)
    got = eviction.evict(k, v, mass, None, lens, keep, sinks=4, recent=16, out=out)
    same((got[0][:, :keep], got[1][:, :keep], got[2][..., :keep], None, got[4]), want)


def test_evict_refuses_outputs_over_their_inputs():
    k, v = (torch.randn(2, 300, 2, 64, device='cuda').to(BF16) for _ in range(2))
    mass, spare = torch.rand(2, 2, 300, device='cuda'), torch.rand(2, 2, 300, device='cuda')
    lens = torch.tensor([300, 250], dtype=torch.int32, device='cuda')
    for out in ((k[:, 4:], v.clone(), spare, None), (k.clone(), v[:, 299 - 100:], spare, None), (v[:, 7:], k.clone(), spare, None),
                (k.clone(), v.clone(), mass[..., 100:], None)):
        with pytest.raises(RuntimeError):
            eviction.evict(k, v, mass, None, lens, 100, out=out)


@pytest.mark.parametrize('T,H,D', [(4, 32, 320), (70, 8, 128)])
def test_waits_of_the_masses_that_run_out_are_reported(T, H, D):
    """With a limit of 1 ns the waits run out while the ring is full (one and several column blocks): the timeout is
    reported, and the next call, with the usual limit, gives what the one before gave."""
    q, k, mass, lens, _ = make(1, T, H, 1, D, [60000])
    lse = torch.full((1, T, H), 5.0, device='cuda')
    want = eviction.key_mass(q, k, lse, mass.clone(), lens, 0.1)
    assert _lib.device_status(clear=True) == 0
    eviction.key_mass(q, k, lse, mass.clone(), lens, 0.1, wait_limit_ns=1)
    assert _lib.device_status(clear=True) & _lib.DEVICE_TIMEOUT
    assert torch.equal(eviction.key_mass(q, k, lse, mass, lens, 0.1), want)
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize('T,page,rank', [(5, 48, 320), (3, 96, 160), (1, 16, 64)])
def test_masses_over_latent_pages(T, page, rank):
    """Only the context has masses; NaN rows past it and table entries of no page stay out."""
    q, k, mass, lens, tables = make(3, T, 32, 1, rank, [0, 700, 129], page=page)
    for b, n in enumerate(lens.tolist()):
        k[tables[b, n // page].long(), n % page:] = math.nan
        tables[b, -(-n // page):] = -7
    lse = torch.full((3, T, 32), 4.0, device='cuda')
    check_mass(q, k, lse, mass, lens, rank ** -0.5, block_tables=tables, context_only=True, decay=0.5)


def test_masses_over_a_cache_shared_by_the_batch():
    q, _, mass, lens, _ = make(3, 4, 8, 2, 128, [50, 60, 170])
    k = torch.randn(1, mass.shape[2], 2, 128, device='cuda').to(BF16)
    check_mass(q, k, torch.full((3, 4, 8), 4.0, device='cuda'), mass, lens, 0.1, decay=0.9)


def test_counts_leave_out_rows_that_saw_nothing():
    """A batch of smaller trees: rows past a sequence's nodes have lse -inf, and its count of nodes keeps them out."""
    q, k, mass, lens, _ = make(3, 4, 8, 2, 128, [50, 60, 170])
    nodes = torch.tensor([4, 0, 2], dtype=torch.int32, device='cuda')
    _, lse = tree.tree_attention(q, k, k, lens, 0.1, nodes=nodes)
    assert (lse[1] == -math.inf).all() and (lse[2, 2:] == -math.inf).all()
    check_mass(q, k, lse, mass, lens, 0.1, counts=nodes, decay=0.9)
    assert mass.isfinite().all()


@pytest.mark.parametrize('page', [16, 5])
def test_evict_from_pages_into_pages_without_masses(page):
    """The C entry alone: an output with block tables, and no output of masses or positions."""
    B, G, D, lengths, keep = 2, 2, 64, [90, 40], 64
    i32 = dict(dtype=torch.int32, device='cuda')
    pages = torch.randn(B * 20, page, G, D, device='cuda').to(BF16)
    tables = torch.randperm(B * 20, device='cuda')[:B * 20].view(B, 20).to(torch.int32)
    per = -(-keep // page)
    new = torch.full((B * per + 1, page, G, D), 7.0, device='cuda', dtype=BF16)
    new_v = new.clone()
    new_tables = torch.randperm(B * per + 1, device='cuda')[:B * per].view(B, per).to(torch.int32)
    mass, lens, after = torch.rand(B, G, 100, device='cuda'), torch.tensor(lengths, **i32), torch.zeros(B, **i32)
    a = _lib.EvictArgs()
    tree.fill_cache(a.src, pages, pages, tables, B)
    tree.fill_cache(a.dst, new, new_v, new_tables, B)
    a.batch, a.kv_heads, a.dim_qk, a.dim_v, a.elem_bytes, a.mass_rows = B, G, D, D, 2, 100
    a.mass, a.lengths, a.new_lengths = mass.data_ptr(), lens.data_ptr(), after.data_ptr()
    a.mass_stride[0], a.mass_stride[1] = mass.stride()[:2]
    a.keep, a.sinks, a.recent = keep, 4, 8
    lib = _lib.load()
    workspace = torch.empty(lib.slimkv_evict_workspace_size(ctypes.byref(a)), dtype=torch.uint8, device='cuda')
    _lib.check(lib.slimkv_evict(ctypes.byref(a), workspace.data_ptr(), workspace.numel(), torch.cuda.current_stream().cuda_stream))
    want = oracle.evict(pages, pages, mass, None, lengths, keep, 4, 8, tables)
    for x in (new, new_v):
        rows = x[new_tables.long()].flatten(1, 2)
        assert torch.equal(rows[:, :keep].double().cpu(), want[0]) and (rows[:, keep:] == 7).all()
        left = torch.ones(len(x), dtype=torch.bool, device='cuda').index_fill(0, new_tables.flatten().long(), False)
        assert (x[left] == 7).all()
    assert after.tolist() == [min(n, keep) for n in lengths] and _lib.device_status() == 0


def test_a_step_over_latents_and_raw_rows():
    """SlimKV's cache in its two parts: attention over each, merged, the accepted rows committed, and the masses of both
    as shares of one softmax."""
    B, T, H, G, D, R = 2, 6, 8, 2, 64, 160
    raw_n, lat_n, scale = [70, 33], [300, 129], 0.125
    q, raw_k, raw_mass, raw_lens, _ = make(B, T, H, G, D, raw_n)
    raw_v = torch.randn_like(raw_k)
    lat = torch.randn(B, 2, 310, R, device='cuda').to(BF16)
    lat_k, lat_v = lat[:, 0].unsqueeze(2), lat[:, 1].unsqueeze(2)
    up_k, up_v = (torch.randn(H, R, D, device='cuda').mul_(R ** -0.5).to(BF16) for _ in range(2))
    absorbed = torch.einsum('bthd,hrd->bthr', q.float(), up_k.float()).to(BF16)
    lat_lens = torch.tensor(lat_n, dtype=torch.int32, device='cuda')
    parents = torch.tensor([[-1, 0, 0, 1, 1, 3], [-1, 0, 1, 2, 0, 4]], dtype=torch.int32, device='cuda')
    seen = torch.stack([oracle.ancestors(p) for p in parents.tolist()])
    raw, raw_lse = tree.tree_attention(q, raw_k, raw_v, raw_lens, scale, mask=tree.tree_masks(parents))
    part, lat_lse = tree.tree_attention(absorbed, lat_k, lat_v, lat_lens, scale, context_only=True)
    up = torch.einsum('bthr,hrd->bthd', part.float(), up_v.float()).to(BF16)
    out = kernels.merge(raw.transpose(1, 2), raw_lse.transpose(1, 2), up.transpose(1, 2), lat_lse.transpose(1, 2)).transpose(1, 2)
    lse = torch.logaddexp(raw_lse, lat_lse)
    # In 64 bits, each part's bound weighted by its share; a share is off by the two lse's bounds, the up-projected part
    # and the output are rounded to bf16 once.
    ro, rl, rt, rlt = oracle.attention(q, raw_k, raw_v, raw_n, scale, seen)
    lo, ll, lt, llt = oracle.attention(absorbed, lat_k, lat_v, lat_n, scale, context_only=True)
    lo = torch.einsum('bthr,hrd->bthd', lo, up_v.double().cpu())
    lt = torch.einsum('bthr,hrd->bthd', lt, up_v.double().cpu().abs()) + 2.0 ** -8 * lo.abs() + 1e-5
    total = torch.logaddexp(rl, ll)
    wr, wl = (rl - total).exp()[..., None], (ll - total).exp()[..., None]
    want = wr * ro + wl * lo
    tol = wr * rt + wl * lt + (rlt + llt + 1e-5)[..., None] * (wr * ro.abs() + wl * lo.abs()) + 2.0 ** -8 * want.abs() + 1e-6
    assert ((out.double().cpu() - want).abs() <= 1.05 * tol).all()
    assert ((lse.double().cpu() - total).abs() <= 1.05 * (rlt + llt + 1e-6)).all()
    path = torch.tensor([[0, 1, 3, 5, -1, -1], [0, 4, -1, -1, -1, -1]], dtype=torch.int32, device='cuda')
    count = torch.tensor([4, 2], dtype=torch.int32, device='cuda')
    new = tree.tree_commit(raw_k, raw_v, raw_lens, path, count)
    assert new.tolist() == [74, 35]
    lat_mass = torch.rand(B, 1, 310, device='cuda')
    check_mass(absorbed, lat_k, lse, lat_mass.clone(), lat_lens, scale, rows=path, counts=count, context_only=True)
    check_mass(q, raw_k, lse, raw_mass.clone(), raw_lens, scale, rows=path, counts=count)
    # Every accepted row has given each head's weight once, over both parts.
    eviction.key_mass(absorbed, lat_k, lse, lat_mass.zero_(), lat_lens, scale, rows=path, counts=count, context_only=True)
    eviction.key_mass(q, raw_k, lse, raw_mass.zero_(), raw_lens, scale, rows=path, counts=count)
    given = lat_mass.double().sum((1, 2)) + raw_mass.double().sum((1, 2))
    assert (given - H * count).abs().max() < 1e-3
