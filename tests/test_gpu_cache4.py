"""The 4-bit cache (``slimkv_b200.cache4``) against plain 64-bit forms: rows
written and read back (bit for bit), attention, key mass, and the calls that
move its rows."""
import math
import random

import pytest
import torch

import cache4_oracle as rows4
import tree_oracle as oracle
from slimkv_b200 import _lib, cache4, eviction, tree

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(11)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device='cuda')


def make_rows(shape, dtype, seed=0):
    """Rows with channels of their own size and mean, as keys have them."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    d = shape[-1]
    x = torch.randn(shape, generator=gen, device='cuda')
    return (x * (0.2 + torch.rand(d, generator=gen, device='cuda')) + 2 * torch.randn(d, generator=gen, device='cuda')).to(dtype)


def caches(B, rows, G, D, Dv, page=0, layout='heads', fill=0xA5):
    """k4, v4 and block tables; every byte `fill` until written."""
    sizes = [cache4.row_bytes(d) for d in (D, Dv)]
    if page:
        per = -(-rows // page)
        n = B * per + 2
        if sizes[0] == sizes[1]:                # K and V by turns in one page, as a serving engine keeps them
            pages = torch.full((n, page, 2, G, sizes[0]), fill, dtype=torch.uint8, device='cuda')
            k4, v4 = pages[:, :, 0], pages[:, :, 1]
        else:
            k4, v4 = (torch.full((n, page, G, s), fill, dtype=torch.uint8, device='cuda') for s in sizes)
        gen = torch.Generator(device='cuda').manual_seed(rows)
        return k4, v4, torch.randperm(n, generator=gen, device='cuda')[:B * per].view(B, per).to(torch.int32)
    if layout == 'heads':
        k4, v4 = cache4.empty(B, rows, G, D, Dv)
        return k4.fill_(fill), v4.fill_(fill), None
    if layout == 'wide':                        # rows with room behind them
        return *(torch.full((B, rows, G, s + 32), fill, dtype=torch.uint8, device='cuda')[..., :s] for s in sizes), None
    return *(torch.full((B, rows, G, s), fill, dtype=torch.uint8, device='cuda') for s in sizes), None


def place(cache, tables, b, n):
    """Cache row n of sequence b."""
    if tables is None:
        return cache[b, n]
    page = cache.shape[1]
    return cache[int(tables[b, n // page]), n % page]


# ------------------------------------------------------------ write, read --
@pytest.mark.parametrize('B,n,G,D,Dv,dtype,page,layout', [
    (1, 1, 8, 128, 128, BF16, 0, 'heads'), (3, 5, 2, 128, 64, FP16, 0, 'rows'), (2, 37, 1, 320, 320, BF16, 0, 'heads'),
    (2, 19, 3, 96, 160, BF16, 8, ''), (4, 33, 2, 64, 64, FP16, 16, ''), (2, 70, 1, 32, 224, BF16, 24, ''),
    (1, 9, 5, 288, 256, FP16, 0, 'wide'), (2, 130, 8, 128, 128, BF16, 48, ''), (1, 3, 40, 192, 192, FP16, 0, 'rows')])
def test_written_rows_are_the_format(B, n, G, D, Dv, dtype, page, layout):
    """Bytes of the rows written, all others untouched, and what is read back."""
    k, v = make_rows((B, n, G, D), dtype), make_rows((B, n, G, Dv + 8), dtype, 1)[..., :Dv]
    starts = [3 * b for b in range(B)]
    counts = [max(0, n - 4 * b) for b in range(B)]
    k4, v4, tables = caches(B, n + 3 * B + 2, G, D, Dv, page, layout)
    cache4.write(k, v, k4, v4, i32(starts), i32(counts), tables)
    got = cache4.read(k4, v4, i32(counts), dtype, rows=n, starts=i32(starts), block_tables=tables)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    for x, x4, read, d in ((k, k4, got[0], D), (v, v4, got[1], Dv)):
        codes, scale, low = rows4.quantise(x.cpu())
        want, back = rows4.pack(codes, scale, low), rows4.values(codes, scale, low)
        used = d // 2 + d // 8
        expected = torch.full_like(x4, 0xA5).cpu()
        tab = None if tables is None else tables.cpu()
        for b in range(B):
            for i in range(counts[b]):
                place(expected, tab, b, starts[b] + i)[..., :used] = want[b, i][..., :used]
            assert rows4.same(read[b, :counts[b]].cpu(), back[b, :counts[b]])
            assert (read[b, counts[b]:] == 0).all()
        assert torch.equal(x4.cpu(), expected)
        assert rows4.same(rows4.unpack(want, d, dtype), back)


@pytest.mark.parametrize('dtype', [BF16, FP16])
def test_values_at_the_edges(dtype):
    """Ties, constant groups, the largest and smallest numbers, infinities and NaN."""
    big, tiny = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    least = 2.0 ** -133 if dtype == BF16 else 2.0 ** -24
    groups = [
        [0.0] * 32, [-1.5] * 32, [0.0, 15.0] + [i + 0.5 for i in range(15)] * 2,                   # ties of a scale of 1
        [-7.5, 7.5] + [i - 7.0 for i in range(15)] * 2, [0.0, 30.0] + [2 * i + 1.0 for i in range(15)] * 2,
        [big, -big] + [0.0] * 30, [0.0, big] + [big / 2] * 30, [big] * 32, [-big, 0.0] + [-big / 3] * 30,
        [tiny, 2 * tiny] + [1.5 * tiny] * 30, [0.0, least] * 16, [0.0, 22 * least, 9 * least, least] * 8, [0.0, 15 * tiny] + [tiny] * 30,
        [1.0, math.nan] + [0.5] * 30, [math.inf] + [2.0] * 31, [-math.inf, math.inf] + [0.0] * 30, [math.inf] * 32,
        [-0.0, 0.0] * 16, [1000.0] + [least * i for i in range(31)], [-7.5, 7.5] + [least, -least] * 15,
        [100.0] + [100.0 * (1 - 2.0 ** -8)] * 31, [-big, -big / 2] * 16]
    x = torch.tensor(groups, dtype=torch.float64).to(dtype)
    x = torch.cat([x, x.flip(-1)]).reshape(1, -1, 1, 64)
    k = x.cuda()
    k4, v4 = cache4.empty(1, k.shape[1], 1, 64)
    cache4.write(k, k, k4, v4)
    got, _ = cache4.read(k4, v4, i32([k.shape[1]]), dtype)
    codes, scale, low = rows4.quantise(x)
    back = rows4.values(codes, scale, low)
    assert rows4.same(got.cpu(), back)
    bad = ~x.unflatten(-1, (-1, 32)).isfinite().all(-1, keepdim=True).expand(*x.shape[:-1], 2, 32).flatten(-2)
    assert got.cpu()[bad].isnan().all() and got.cpu()[~bad].isfinite().all()
    same = torch.equal(k4.cpu()[..., :32], rows4.pack(codes, scale, low)[..., :32])
    assert same and torch.equal(k4[..., :40], v4[..., :40])       # (what fills a row up is never written)


@pytest.mark.parametrize('dtype', [BF16, FP16])
def test_values_next_to_borders(dtype):
    """Rows of few distinct numbers: many quotients at or a step from a half."""
    gen = torch.Generator().manual_seed(3)
    low = torch.randint(-40, 40, (1, 4000, 1, 2, 1), generator=gen).double() * 2.0 ** torch.randint(-6, 4, (1, 4000, 1, 2, 1), generator=gen)
    step = torch.randint(1, 64, (1, 4000, 1, 2, 1), generator=gen).double() * 2.0 ** torch.randint(-9, 4, (1, 4000, 1, 2, 1), generator=gen)
    x = (low + step * torch.randint(0, 31, (1, 4000, 1, 2, 32), generator=gen) / 2).flatten(-2).to(dtype)
    k4, v4 = cache4.empty(1, 4000, 1, 64)
    cache4.write(x.cuda(), x.cuda(), k4, v4)
    assert torch.equal(k4.cpu()[..., :40], rows4.pack(*rows4.quantise(x))[..., :40])


@pytest.mark.parametrize('dtype', [BF16, FP16])
def test_every_code_reads_back_as_the_format_says(dtype):
    """Rows with codes and pairs of any bits (finite): one rounding of code * scale + low."""
    gen = torch.Generator().manual_seed(5)
    D, n = 96, 600
    raw = torch.randint(0, 256, (1, n, 2, cache4.row_bytes(D)), generator=gen).to(torch.uint8)
    pairs = (torch.randn(1, n, 2, 3, 2, generator=gen) * 2.0 ** torch.randint(-8, 8, (1, n, 2, 3, 2), generator=gen)).to(dtype)
    raw[..., 48:60] = pairs.flatten(-2).view(torch.uint8)
    k4 = raw.cuda()
    got, v = cache4.read(k4, k4.clone(), i32([n]), dtype)
    want = rows4.unpack(raw, D, dtype)
    assert rows4.same(got.cpu(), want) and rows4.same(v.cpu(), want)


def test_read_into_buffers_leaves_the_rest():
    k = make_rows((2, 20, 2, 64), BF16)
    k4, v4, tables = caches(2, 32, 2, 64, 64, 16)
    cache4.write(k, k, k4, v4, block_tables=tables)
    wide = torch.full((2, 24, 2, 72), 7.0, device='cuda', dtype=BF16)
    out = wide[..., :64], torch.full((2, 24, 2, 64), 7.0, device='cuda', dtype=BF16)
    cache4.read(k4, v4, i32([0, 9]), BF16, starts=i32([1, 4]), block_tables=tables, out=out)
    want, _ = cache4.read(k4, v4, i32([0, 9]), BF16, rows=24, starts=i32([1, 4]), block_tables=tables)
    for x in out:
        assert torch.equal(x[1, :9], want[1, :9]) and (x[0] == 7).all() and (x[1, 9:] == 7).all()
    assert (wide[..., 64:] == 7).all()


def test_rows_of_very_different_lengths_in_a_large_call():
    """2^28 rows of 32 and 320 dims in one call: of blocks cut for the longer rows, those of the shorter lie past 2^31."""
    n = 1 << 28
    k, v = make_rows((1, 4, 1, 32), BF16), make_rows((1, 4, 1, 320), BF16, 1)
    guarded = [torch.full((1, 4096, 1, cache4.row_bytes(d)), 0xA5, dtype=torch.uint8, device='cuda') for d in (32, 320)]
    k4, v4 = (x[:, 2040:2050] for x in guarded)
    cache4.write(k[:, :1].expand(1, n, 1, 32), v[:, :1].expand(1, n, 1, 320), k4, v4, i32([2]), i32([3]))
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    got = cache4.read(k4, v4, i32([3]), BF16, rows=3, starts=i32([2]))
    for x, x4, back in ((k, guarded[0], got[0]), (v, guarded[1], got[1])):
        assert rows4.same(back.cpu(), rows4.values(*rows4.quantise(x[:, :1].expand(1, 3, 1, -1).cpu())))
        touched = (x4 != 0xA5).any(-1).nonzero()[:, 1].tolist()
        assert touched == [2042, 2043, 2044]


def test_sequences_that_share_pages_and_caches_read_the_same_rows():
    k = make_rows((1, 40, 2, 128), FP16)
    k4, v4, tables = caches(1, 40, 2, 128, 128, 8)
    cache4.write(k, k, k4, v4, block_tables=tables)
    got, _ = cache4.read(k4, v4, i32([40, 33, 0]), FP16, rows=40, block_tables=tables.expand(3, -1))
    d4, e4 = cache4.empty(1, 40, 2, 128)
    cache4.write(k, k, d4, e4)
    dense, _ = cache4.read(d4, e4, i32([40, 33, 0]), FP16)
    assert torch.equal(got, dense) and torch.equal(got[0, :33], got[1, :33]) and (got[1, 33:] == 0).all() and (got[2] == 0).all()


def test_rows_without_a_place_are_reported():
    k = make_rows((1, 6, 1, 32), BF16)
    k4, v4 = cache4.empty(1, 10, 1, 32)
    for start, count, kept in ((7, 6, [7, 8, 9]), (-1, 6, []), (0, 7, [0, 1, 2, 3, 4, 5]), (12, 1, []), (3, -2, [])):
        k4.fill_(0xA5)
        v4.fill_(0xA5)
        _lib.device_status(clear=True)
        cache4.write(k, k, k4, v4, i32([start]), i32([count]))
        assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH
        assert (k4[0, :, 0, :20] != 0xA5).any(-1).nonzero()[:, 0].tolist() == kept
        cache4.read(k4, v4, i32([count]), BF16, rows=6, starts=i32([start]))
        assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH
    p4, q4, tables = caches(1, 32, 1, 32, 32, 8)
    tables[0, 1] = p4.shape[0]
    kept = p4.clone()
    rows = make_rows((1, 24, 1, 32), BF16)
    cache4.write(rows, rows, p4, q4, block_tables=tables)
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH
    others = [p for p in range(p4.shape[0]) if p not in (int(tables[0, 0]), int(tables[0, 2]))]
    assert torch.equal(p4[others], kept[others])


# -------------------------------------------------------------- attention --
def make(B, T, H, G, D, lengths, Dv=None, dtype=BF16, page=0, layout='heads', context_only=False, seed=0, spare=5):
    """q, 4-bit caches, lengths, tables, and the caches' 16-bit rows (dense); what no row may read is NaN."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    Dv = Dv or D
    ends = [n + (0 if context_only else T) for n in lengths]
    cap = max(ends) + spare
    q = torch.randn(B, T, H, D, generator=gen, device='cuda', dtype=dtype)
    k4, v4, tables = caches(B if layout != 'shared' else 1, cap, G, D, Dv, page, layout, fill=0xFF)      # NaN pairs
    many = 1 if layout == 'shared' else B
    k, v = make_rows((many, max(ends), G, D), dtype, seed + 1), make_rows((many, max(ends), G, Dv), dtype, seed + 2)
    cache4.write(k, v, k4, v4, counts=i32(ends if many == B else [max(ends)]), block_tables=tables)
    if page:        # entries past the rows in use name no page
        for b in range(B):
            tables[b, -(-ends[b] // page):] = -7
    return q, k4, v4, i32(lengths), tables


def dense_rows(k4, v4, tables, dtype, dims, used):
    """The 16-bit rows of a cache, by the format alone."""
    out = []
    for x4, d in zip((k4, v4), dims):
        raw = x4.cpu()
        if tables is not None:
            raw = raw[tables.cpu().long().clamp(0, raw.shape[0] - 1)].flatten(1, 2)
        out.append(rows4.unpack(raw[:, :used].contiguous(), d, dtype))
    return out


def run(q, k4, v4, lens, tables=None, seen=None, nodes=None, context_only=False, scale=None, Dv=None):
    scale = scale or 0.5 * q.shape[3] ** -0.5
    mask = None if seen is None else oracle.words_of(seen).cuda()
    got = cache4.attention(q, k4, v4, lens, scale, mask=mask, nodes=nodes, block_tables=tables, context_only=context_only)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    used = int(lens.max()) + (0 if context_only else q.shape[1])
    k, v = dense_rows(k4, v4, tables, q.dtype, (q.shape[3], got[0].shape[3]), used)
    # K, V and q exact in the products; P and the output rounded to the type, as in tree attention.
    oracle.check_attention(got, oracle.attention(q, k, v, lens.tolist(), scale, seen, None if nodes is None else nodes.tolist(),
                                                 None, context_only))
    return got


def random_parents(rng, nodes):
    return [-1] + [rng.randrange(max(0, i - 4), i) for i in range(1, nodes)]


def trees(B, T, seed):
    rng = random.Random(seed)
    return torch.stack([oracle.ancestors(random_parents(rng, T)) for _ in range(B)])


@pytest.mark.parametrize('lengths', [[0], [1], [14], [15], [16], [17], [62], [63], [64], [65], [517], [3001]])
@pytest.mark.parametrize('dtype', [BF16, FP16])
def test_single_tokens(lengths, dtype):
    run(*make(1, 1, 32, 8, 128, lengths, dtype=dtype))


@pytest.mark.parametrize('D', list(range(32, 321, 32)))
@pytest.mark.parametrize('T', [1, 3])
def test_every_dim(D, T):
    run(*make(2, T, 8, 2, D, [77, 130], dtype=BF16 if D % 64 else FP16, seed=D))


@pytest.mark.parametrize('B,T,H,G,D,lengths,dtype,page,layout', [
    (3, 13, 8, 2, 128, [0, 300, 77], BF16, 0, 'heads'),
    (2, 7, 10, 2, 128, [1000, 5], BF16, 16, ''),
    (2, 33, 8, 8, 64, [130, 256], FP16, 48, ''),
    (2, 40, 8, 2, 64, [0, 129], BF16, 24, ''),
    (1, 70, 8, 2, 128, [385], BF16, 0, 'rows'),
    (2, 5, 40, 8, 128, [100, 300], BF16, 8, ''),
    (2, 9, 6, 2, 96, [64, 700], FP16, 128, ''),
    (4, 5, 3, 3, 32, [9, 0, 128, 1111], BF16, 0, 'wide'),
    (1, 2, 128, 1, 32, [200], FP16, 0, 'heads'),
    (2, 4, 12, 4, 160, [300, 31], BF16, 0, 'heads'),
    (1, 6, 5, 1, 320, [2000], FP16, 32, ''),
    (20, 2, 4, 2, 64, [50 * i for i in range(20)], BF16, 16, '')])
def test_trees(B, T, H, G, D, lengths, dtype, page, layout):
    run(*make(B, T, H, G, D, lengths, dtype=dtype, page=page, layout=layout, seed=T), seen=trees(B, T, T))


@pytest.mark.parametrize('D,Dv,T', [(128, 64, 9), (64, 128, 4), (320, 64, 3), (96, 320, 5), (256, 288, 1), (32, 320, 1), (320, 32, 1)])
def test_value_dims_of_their_own(D, Dv, T):
    run(*make(2, T, 8, 2, D, [200, 411], Dv=Dv), seen=trees(2, T, 3))


@pytest.mark.parametrize('T', [1, 4, 33, 70])
def test_a_chain_needs_no_mask(T):
    args = make(2, T, 8, 2, 128, [100, 260])
    got = run(*args)
    chain = torch.ones(1, T, T).tril().bool()
    same = cache4.attention(*args[:3], args[3], 0.5 * 128 ** -0.5, mask=oracle.words_of(chain).cuda())
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])


@pytest.mark.parametrize('rank,T,lengths', [(320, 1, [1000, 0, 77]), (160, 1, [1, 500, 128]), (320, 9, [4000, 129, 2]), (256, 2, [15, 16, 17])])
@pytest.mark.parametrize('page', [0, 48])
def test_latents(rank, T, lengths, page):
    """One latent head, no rows of the nodes."""
    run(*make(3, T, 32, 1, rank, lengths, context_only=True, page=page), context_only=True)


# Dims of 128 and of 256, whose rows (20 and more) the two kernels take.
@pytest.mark.parametrize('D', [128, 256])
@pytest.mark.parametrize('T', [5, 40])
def test_ragged_trees(T, D):
    """Sequences with fewer nodes (or none): the rows past them are empty."""
    q, k4, v4, lens, _ = make(4, T, 8, 2, D, [0, 140, 256, 0])
    run(q, k4, v4, lens, seen=trees(4, T, 1), nodes=i32([T, T - 3, 0, 1]))


# One tile of keys (a segment written by one block) and several (merged).
@pytest.mark.parametrize('lengths', [[0, 20, 100, 90], [0, 140, 2000, 700]])
@pytest.mark.parametrize('D', [128, 256, 320])
@pytest.mark.parametrize('context_only', [False, True])
def test_rows_past_the_nodes_are_empty_whatever_they_hold(lengths, D, context_only):
    """Queries of a padded batch hold anything, and a value of the context may be NaN."""
    T, nodes = 9, [9, 6, 0, 1]
    q, k4, v4, lens, _ = make(4, T, 8, 2, D, lengths, context_only=context_only)
    for b, (n, fill) in enumerate(zip(nodes, (0.0, math.nan, math.inf, -math.inf))):
        q[b, n:] = fill
    v4[3, 5, 1, D // 2:D // 2 + 4] = 0xFF                # a value of the context, in all rows of sequence 3
    out, lse = cache4.attention(q, k4, v4, lens, 0.5 * D ** -0.5, nodes=i32(nodes), context_only=context_only)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    for b, n in enumerate(nodes):
        assert (out[b, n:] == 0).all() and (lse[b, n:] == -math.inf).all()
    assert lse[0, :].isfinite().all() == (not context_only) and out[1, :6].isfinite().all() and lse[1, :6].isfinite().all()
    assert out[3, 0, 4:, :32].isnan().all() and out[3, 0, :4].isfinite().all() and out[3, 0, 4:, 32:].isfinite().all()


@pytest.mark.parametrize('D', [128, 256])
def test_empty_rows(D):
    """Mask rows without a bit: over an empty context nothing is seen."""
    q, k4, v4, lens, _ = make(2, 6, 8, 2, D, [0, 40])
    seen = trees(2, 6, 2)
    seen[:, 3] = False
    got = run(q, k4, v4, lens, seen=seen)
    assert (got[0][0, 3] == 0).all() and (got[1][0, 3] == -math.inf).all() and got[1][1, 3].isfinite().all()


@pytest.mark.parametrize('D', [128, 256])
@pytest.mark.parametrize('T,page', [(6, 0), (40, 0), (6, 16)])
def test_unseen_nans_do_not_spread(T, page, D):
    """A node's non-finite key or value reaches the rows that see it and no other."""
    q, k4, v4, lens, tables = make(2, T, 8, 2, D, [100, 133], page=page)
    seen = trees(2, T, 4)
    for b, n in enumerate([100, 133]):
        for node, x4, group in ((2, v4, 0), (3, v4, 3), (4, k4, 1), (1, v4, 2)):
            seen[b, :, node] = torch.arange(T) == node           # only the node itself sees it
            place(x4, tables, b, n + node)[1, D // 2 + 4 * group:D // 2 + 4 * group + 4] = 0xFF
    got = run(q, k4, v4, lens, tables, seen=seen)
    assert got[0][:, 0].isfinite().all() and got[0][:, 5:].isfinite().all() and got[0][:, 1:5].isnan().any()


@pytest.mark.parametrize('T,D', [(3, 128), (7, 256), (9, 320)])
@pytest.mark.parametrize('scale', [2.0, 0.5])
@pytest.mark.parametrize('dtype', [BF16, FP16])
def test_peaked_scores(scale, dtype, T, D):
    """Scores up to the hundreds: maxima that keep growing along the keys."""
    q, k4, v4, lens, _ = make(1, T, 8, 2, D, [700], dtype=dtype)
    k = torch.randn(1, 700 + T, 2, D, device='cuda') * torch.linspace(0.1, 3, 700 + T, device='cuda')[None, :, None, None]
    cache4.write(k.to(dtype), k.to(dtype), k4, v4)
    run(q, k4, v4, lens, scale=scale)


@pytest.mark.parametrize('H,D', [(1, 32), (17, 224)])
def test_small_probabilities_count_in_fp16(H, D):
    """One key far above 20,000 others: their share of the weight stays."""
    n = 20000
    k4, v4 = cache4.empty(1, n + 1, 1, D)
    k = torch.zeros(1, n + 1, 1, D, device='cuda', dtype=FP16)
    v = torch.ones_like(k)
    k[0, 5, 0, 0], v[0, 5] = 15.0, 0.0
    cache4.write(k, v, k4, v4)
    q = torch.zeros(1, 1, H, D, device='cuda', dtype=FP16)
    q[..., 0] = 1.0
    run(q, k4, v4, i32([n]), scale=1.0)


@pytest.mark.parametrize('H,D,dtype', [(4, 128, BF16), (12, 64, FP16), (40, 320, BF16), (20, 256, FP16)])
@pytest.mark.parametrize('n', [40, 20000])
def test_values_without_weight_that_are_nan(H, D, dtype, n):
    """A context's NaN value makes its group NaN whatever its weight (the formula's 0 x NaN), in one piece and in many."""
    k4, v4 = cache4.empty(1, n + 1, 1, D)
    k, v = torch.zeros(1, n + 1, 1, D, device='cuda', dtype=dtype), make_rows((1, n + 1, 1, D), dtype)
    k[..., 0] = -16.0                                       # e^-512 of the last row's weight
    k[:, n] = 0.0
    k[:, n, :, 0] = 16.0
    cache4.write(k, v, k4, v4)
    for row in (7, n // 2):
        v4[0, row, 0, D // 2 + 4:D // 2 + 8] = 0xFF
        q = torch.zeros(1, 1, H, D, device='cuda', dtype=dtype)
        q[..., 0] = 16.0
        got = run(q, k4, v4, i32([n]), scale=1.0)
        assert got[0][..., 32:64].isnan().all() and got[0][..., :32].isfinite().all() and got[0][..., 64:].isfinite().all()
        cache4.write(k, v, k4, v4)


def test_shared_cache_and_strided_outputs():
    q, k4, v4, lens, _ = make(3, 4, 8, 2, 128, [50, 60, 170], layout='shared')
    run(q, k4, v4, lens, seen=trees(3, 4, 5))
    wide = torch.zeros(3, 4, 8, 144, device='cuda', dtype=BF16)
    lse = torch.zeros(3, 4, 8, device='cuda')
    out, _ = cache4.attention(q, k4, v4, lens, 0.1, out=wide[..., 8:136], lse=lse)
    again, lse2 = cache4.attention(q, k4, v4, lens, 0.1)
    assert torch.equal(out, again) and torch.equal(lse, lse2) and (wide[..., :8] == 0).all() and (wide[..., 136:] == 0).all()


def test_strided_queries():
    q, k4, v4, lens, _ = make(2, 3, 8, 2, 64, [50, 61])
    want = run(q, k4, v4, lens)
    other = torch.randn(3, 8, 2, 72, device='cuda').to(BF16)[..., :64].permute(2, 0, 1, 3)
    other.copy_(q)
    got = cache4.attention(other, k4, v4, lens, 0.5 * 64 ** -0.5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize('B,H,G,D,lengths', [
    (40, 32, 8, 64, [(7 * b) % 30 for b in range(40)]), (1, 4, 1, 64, [70000]), (3, 8, 4, 64, [20000, 3, 9000]),
    (40, 40, 2, 224, [(11 * b) % 300 for b in range(40)]), (1, 40, 1, 320, [40000]), (3, 68, 2, 256, [9000, 3, 129])])
def test_many_and_long_segments(B, H, G, D, lengths):
    """Shares of many short segments, and segments over many shares; twice the same bits."""
    args = make(B, 1, H, G, D, lengths)
    got = run(*args)
    again = cache4.attention(*args[:3], args[3], 0.5 * D ** -0.5)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


# More than 16 query rows of 224 or 256 dims: two tiles' probabilities may be under way at a piece's end.
@pytest.mark.parametrize('H,D,Dv,dtype', [(24, 256, 256, BF16), (40, 224, 256, FP16), (40, 256, 64, BF16), (24, 64, 224, FP16)])
def test_pieces_end_with_all_their_products(H, D, Dv, dtype):
    """Pieces of 1 to 12 tiles, over and over beside other traffic: the exact result, and the same bits each time."""
    B = 150
    lengths = [128 * (1 + b % 12) - b % 7 for b in range(B)]
    q, k4, v4, lens, _ = make(B, 1, H, 1, D, lengths, Dv=Dv, dtype=dtype, layout='shared', context_only=True)
    want = run(q, k4, v4, lens, context_only=True)
    side, a = torch.cuda.Stream(), torch.zeros(1 << 28, dtype=torch.uint8, device='cuda')
    b = torch.empty_like(a)
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(side):
            for _ in range(4):
                b.copy_(a)
        for _ in range(10):
            got = cache4.attention(q, k4, v4, lens, 0.5 * D ** -0.5, context_only=True)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


def test_offsets_past_32_bits():
    """Sequence strides of more than 2^32 bytes."""
    big = torch.empty(2, (1 << 32) + (1 << 12), dtype=torch.uint8, device='cuda')
    k4 = big.as_strided((2, 400, 1, 80), (big.stride(0), 1 << 16, 80, 1))
    v4 = big.as_strided((2, 400, 1, 80), (big.stride(0), 1 << 16, 80, 1), 1 << 10)
    k = make_rows((2, 393, 1, 128), BF16)
    cache4.write(k, k, k4, v4)
    q = torch.randn(2, 3, 4, 128, device='cuda').to(BF16)
    run(q, k4, v4, i32([390, 111]))
    back, _ = cache4.read(k4, v4, i32([393, 393]), BF16, rows=393)
    codes = rows4.quantise(k.cpu())
    assert rows4.same(back.cpu(), rows4.values(*codes))


@pytest.mark.parametrize('D', [128, 256])
def test_another_stream_and_two_graphs(D):
    q, k4, v4, lens, _ = make(2, 8, 8, 2, D, [300, 10])
    mask = oracle.words_of(trees(2, 8, 7)).cuda()
    want = cache4.attention(q, k4, v4, lens, 0.09, mask=mask)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = cache4.attention(q, k4, v4, lens, 0.09, mask=mask)
        side.synchronize()
        graphs, held = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
        for graph in graphs:
            with torch.cuda.graph(graph, stream=side):
                held.append(cache4.attention(q, k4, v4, lens, 0.09, mask=mask))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    lens.copy_(torch.tensor([17, 9], dtype=torch.int32))
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    again = cache4.attention(q, k4, v4, lens, 0.09, mask=mask)
    for h in held:
        assert torch.equal(h[0], again[0]) and torch.equal(h[1], again[1])


def test_attention_is_that_over_the_rows_read_back():
    """The same call over the 16-bit rows: both are within the rounding of P and the output of the exact one."""
    q, k4, v4, lens, tables = make(3, 4, 32, 8, 128, [700, 33, 1900], page=16)
    k, v = cache4.read(k4, v4, lens + 4, BF16, rows=1904, block_tables=tables)
    got = cache4.attention(q, k4, v4, lens, 0.05, block_tables=tables)
    want = tree.tree_attention(q, k, v, lens, 0.05)
    norm = lambda x: x.double().norm()
    assert norm(got[0].double() - want[0].double()) <= 4 * 2.0 ** -8 * norm(want[0])
    assert (got[1] - want[1]).abs().max() <= 2e-5


@pytest.mark.parametrize('H,D', [(8, 128), (40, 320)])
def test_lengths_past_the_cache_are_reported(H, D):
    q, k4, v4, _, _ = make(1, 2, H, 2, D, [60], spare=0)
    _lib.device_status(clear=True)
    cache4.attention(q, k4, v4, i32([61]), 0.1)
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH
    cache4.attention(q, k4, v4, i32([-1]), 0.1)
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH


@pytest.mark.parametrize('H,D', [(8, 128), (40, 320)])
def test_pages_outside_the_pool_are_reported(H, D):
    q, k4, v4, lens, tables = make(1, 2, H, 2, D, [60], page=16)
    _lib.device_status(clear=True)
    tables[0, 2] = k4.shape[0]
    cache4.attention(q, k4, v4, lens, 0.1, block_tables=tables)
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH


@pytest.mark.parametrize('H,D,n', [(8, 128, 9000), (8, 64, 40), (40, 320, 9000), (40, 256, 300)])
def test_a_wait_that_runs_out_is_reported(H, D, n):
    """Every wait ends at its limit, the call returns, and the next one is right."""
    q, k4, v4, lens, _ = make(3, 2, H, 2, D, [n, n // 2, n])
    lse = torch.zeros(3, 2, H, device='cuda')
    for limit in (1, 1000):
        _lib.device_status(clear=True)
        cache4.attention(q, k4, v4, lens, 0.1, wait_limit_ns=limit)
        assert _lib.device_status(clear=True) in (0, _lib.DEVICE_TIMEOUT)
        cache4.key_mass(q, k4, lse, torch.zeros(3, 2, n + 10, device='cuda'), lens, 0.1, wait_limit_ns=limit)
        assert _lib.device_status(clear=True) in (0, _lib.DEVICE_TIMEOUT)
    run(q, k4, v4, lens)


@pytest.mark.parametrize('B,H,G,D,dtype', [(3, 8, 2, 128, BF16), (16, 4, 1, 64, FP16), (4, 12, 1, 192, BF16)])
def test_waits_that_run_out_end_the_narrow_pipeline(B, H, G, D, dtype):
    """With a limit of 1 ns a wait for the first keys runs out, since no warp has anything to do meanwhile and a copy
    takes a microsecond: reported each time, and the next call is right.  (12 rows of 192 dims have their Q in shared
    memory: the block loads it and meets at a barrier first, by which time the keys may have come.)"""
    q, k4, v4, lens, _ = make(B, 1, H, G, D, [9000 - 300 * b for b in range(B)], dtype=dtype)
    for _ in range(3):
        _lib.device_status(clear=True)
        cache4.attention(q, k4, v4, lens, 0.1, wait_limit_ns=1)
        assert _lib.device_status(clear=True) in ((0, _lib.DEVICE_TIMEOUT) if D == 192 else (_lib.DEVICE_TIMEOUT,))
    run(q[:2], k4[:2], v4[:2], lens[:2])


@pytest.mark.parametrize('B,H,G,D', [(3, 40, 2, 320), (3, 40, 2, 256), (20, 24, 1, 224)])
def test_waits_that_run_out_end_the_wide_pipeline(B, H, G, D):
    """With a limit of 1 ns the first products' waits run out while copies are under way (they take a microsecond):
    the call reports it and ends with nothing under way, again and again, and the next one is right."""
    q, k4, v4, lens, _ = make(B, 1, H, G, D, [9000 - 400 * b for b in range(B)])
    for _ in range(3):
        _lib.device_status(clear=True)
        cache4.attention(q, k4, v4, lens, 0.1, wait_limit_ns=1)
        assert _lib.device_status(clear=True) == _lib.DEVICE_TIMEOUT
    if B > 3:
        q, k4, v4, lens = q[:2], k4[:2], v4[:2], lens[:2]
    run(q, k4, v4, lens)


# ------------------------------------------------------------------- mass --
def run_mass(q, k4, lens, tables=None, rows=None, counts=None, decay=1.0, context_only=False, scale=None, cap=None):
    B, T, H, D = q.shape
    scale = scale or 0.5 * D ** -0.5
    used = int(lens.max()) + (0 if context_only else T)
    k, _ = dense_rows(k4, k4, tables, q.dtype, (D, D), used)
    lse = torch.rand(B, T, H, device='cuda') * 4 + 3
    old = torch.rand(B, k4.shape[2], cap or used + 3, device='cuda')
    mass = old.clone()
    got = cache4.key_mass(q, k4, lse, mass, lens, scale, rows=rows, counts=counts, decay=decay, block_tables=tables,
                          context_only=context_only)
    torch.cuda.synchronize()
    assert got is mass and _lib.device_status() == 0
    want, tol = oracle.mass(q, k, lse, old, lens.tolist(), scale, rows, counts, decay, None, context_only)
    assert ((mass.double().cpu() - want).abs() <= 1.05 * tol).all()
    return mass


@pytest.mark.parametrize('B,T,H,G,D,lengths,dtype,page,layout', [
    (1, 1, 32, 8, 128, [1028], BF16, 0, 'heads'),
    (3, 5, 8, 2, 128, [0, 300, 77], BF16, 0, 'rows'),
    (2, 7, 10, 2, 96, [100, 5], FP16, 16, ''),
    (2, 16, 8, 8, 64, [130, 256], FP16, 24, ''),
    (2, 40, 8, 2, 32, [0, 129], BF16, 8, ''),
    (20, 2, 4, 2, 64, [50 * i for i in range(20)], BF16, 48, ''),
    (2, 3, 12, 4, 160, [300, 31], BF16, 0, 'wide'),
    (1, 1, 4, 1, 256, [30000], FP16, 0, 'heads')])
def test_key_mass(B, T, H, G, D, lengths, dtype, page, layout):
    q, k4, _, lens, tables = make(B, T, H, G, D, lengths, dtype=dtype, page=page, layout=layout, seed=T)
    run_mass(q, k4, lens, tables)
    rng = random.Random(T)
    counts = [rng.randint(0, T) for _ in range(B)]
    rows = [sorted(rng.sample(range(T), c)) + [-1] * (T - c) for c in counts]
    run_mass(q, k4, lens, tables, i32(rows), i32(counts), decay=0.9)


@pytest.mark.parametrize('rank,T,lengths', [(320, 9, [1000, 0, 77]), (160, 1, [1, 500, 128]), (320, 2, [4000, 129, 2])])
def test_key_mass_of_latents(rank, T, lengths):
    q, k4, _, lens, _ = make(3, T, 32, 1, rank, lengths, context_only=True)
    first = run_mass(q, k4, lens, context_only=True, decay=0.5)
    assert first.isfinite().all()


def test_key_mass_of_rows_that_give_nothing():
    """An lse of +inf, and sequences without accepted rows: only the decay."""
    q, k4, _, lens, _ = make(2, 2, 8, 2, 64, [50, 61])
    mass = torch.rand(2, 2, 70, device='cuda')
    old = mass.clone()
    lse = torch.full((2, 2, 8), math.inf, device='cuda')
    cache4.key_mass(q, k4, lse, mass, lens, 0.1, counts=i32([2, 0]), decay=0.5)
    want = old.clone()
    want[0, :, :50] *= 0.5
    want[0, :, 50:52] = 0
    want[1, :, :61] *= 0.5
    assert torch.equal(mass, want)


# --------------------------------------------------- rows that move, a run --
@pytest.mark.parametrize('page', [0, 16])
def test_a_run_of_steps_over_the_cache(page):
    """Prompt written, a tree verified, its rows committed, masses, an eviction, and
    attention over what is left: each step as the 16-bit operators do it on the same rows."""
    B, T, H, G, D = 2, 6, 8, 2, 128
    lengths = [150, 97]
    q, k4, v4, lens, tables = make(B, T, H, G, D, lengths, page=page)
    dense = lambda n: cache4.read(k4, v4, i32(n), BF16, rows=max(n), block_tables=tables)
    k, v = dense([n + T for n in lengths])
    parents = [random_parents(random.Random(b), T) for b in range(B)]
    mask = tree.tree_masks(i32(parents))
    out, lse = cache4.attention(q, k4, v4, lens, 0.05, mask=mask, block_tables=tables)
    path, count = i32([[0, 2, 5, -1, -1, -1], [0, 1, -1, -1, -1, -1]]), i32([3, 2])
    kc, vc = k.clone(), v.clone()
    new = tree.tree_commit(k4, v4, lens, path, count, block_tables=tables)
    assert torch.equal(new, tree.tree_commit(kc, vc, lens, path, count))
    k, v = dense(new.tolist())
    for b, n in enumerate(new.tolist()):
        assert torch.equal(k[b, :n], kc[b, :n]) and torch.equal(v[b, :n], vc[b, :n])
    cap = 160
    mass, mass16 = torch.zeros(B, G, cap, device='cuda'), torch.zeros(B, G, cap, device='cuda')
    cache4.key_mass(q, k4, lse, mass, lens, 0.05, rows=path, counts=count, block_tables=tables)
    eviction.key_mass(q, kc, lse, mass16, lens, 0.05, rows=path, counts=count)
    assert torch.allclose(mass, mass16, rtol=1e-4, atol=0)
    e4, f4, m4, _, l4 = eviction.evict(k4, v4, mass, None, new, 64, sinks=4, recent=16, block_tables=tables)
    ek, ev, em, _, el = eviction.evict(kc, vc, mass, None, new, 64, sinks=4, recent=16)
    gk, gv = cache4.read(e4, f4, l4, BF16)
    assert torch.equal(l4, el) and torch.equal(m4, em) and torch.equal(gk, ek) and torch.equal(gv, ev)
    run(q[:, :1].contiguous(), e4, f4, l4, context_only=True)


def test_a_decode_loop_in_a_graph():
    """One captured step (write behind the lengths, attention, lengths + 1) replayed."""
    B, H, G, D, cap = 3, 8, 2, 64, 40
    k4, v4 = cache4.empty(B, cap, G, D)
    lens = i32([0, 3, 9])
    start = make_rows((B, 9, G, D), BF16, 3)
    cache4.write(start, start, k4, v4, counts=lens)
    q, k, v = (torch.empty(B, 1, h, D, device='cuda', dtype=BF16) for h in (H, G, G))

    def step():
        cache4.write(k, v, k4, v4, lens)
        got = cache4.attention(q, k4, v4, lens, 0.1)
        lens.add_(1)
        return got
    for x in (q, k, v):
        x.normal_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step()
    for i in range(12):
        for x in (q, k, v):
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        before = lens - 1
        kk, vv = dense_rows(k4, v4, None, BF16, (D, D), int(before.max()) + 1)
        oracle.check_attention(held, oracle.attention(q, kk, vv, before.tolist(), 0.1))
    assert lens.tolist() == [12, 15, 21] and _lib.device_status() == 0


# -------------------------------------------------------------- refusals --
def test_refusals():
    q, k4, v4, lens, _ = make(2, 4, 8, 2, 128, [50, 60])
    k = make_rows((2, 4, 2, 128), BF16)
    bad = lambda f, *a, **kw: pytest.raises(RuntimeError, f, *a, **kw)
    bad(cache4.row_bytes, 40)
    bad(cache4.empty, 1, 8, 1, 352)
    bad(cache4.write, k.float(), k.float(), k4, v4)
    bad(cache4.write, k, k[:, :3], k4, v4)
    bad(cache4.write, k[..., :64], k, k4, v4)
    bad(cache4.write, k, k, k4, v4, lens.long())
    bad(cache4.write, k, k, k4, k4)
    bad(cache4.write, k, k, k4[:1], v4[:1])                      # one cache for two sequences
    bad(cache4.write, k, k, k4.view(torch.int8), v4)
    bad(cache4.write, k.cpu(), k.cpu(), k4.cpu(), v4.cpu())
    bad(cache4.write, k.transpose(2, 3), k.transpose(2, 3), k4, v4)
    bad(cache4.write, k, k, k4[:, :, :1], v4[:, :, :1])
    bad(cache4.read, k4, v4, lens, torch.float32)
    bad(cache4.read, k4, v4, lens, BF16, out=(k, k))             # K and V into the same rows
    bad(cache4.read, k4, v4, lens, BF16, out=(k, k[:, :2]))
    bad(cache4.read, k4, v4, lens, BF16, block_tables=torch.zeros(2, 3, dtype=torch.int32, device='cuda'))
    bad(cache4.attention, q[..., :64], k4, v4, lens, 0.1)
    bad(cache4.attention, q.float(), k4, v4, lens, 0.1)
    bad(cache4.attention, q, k4, v4, lens, 0.0)
    bad(cache4.attention, q, k, k, lens, 0.1)
    bad(cache4.attention, q, k4, v4, lens.long(), 0.1)
    bad(cache4.attention, q[:, :, :7], k4, v4, lens, 0.1)
    pages = torch.zeros(20, 12, 2, 80, device='cuda', dtype=torch.uint8)
    bad(cache4.attention, q, pages, pages, lens, 0.1, block_tables=torch.zeros(2, 8, dtype=torch.int32, device='cuda'))
    mass = torch.zeros(2, 2, 70, device='cuda')
    lse = torch.zeros(2, 4, 8, device='cuda')
    bad(cache4.key_mass, q[..., :64], k4, lse, mass, lens, 0.1)
    bad(cache4.key_mass, q, k, lse, mass, lens, 0.1)
    bad(cache4.key_mass, q, k4, lse[:, :2], mass, lens, 0.1)
    assert _lib.device_status() == 0
