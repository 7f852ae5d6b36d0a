"""Verification of drafted trees (``slimkv_b200.tree``) against plain 64-bit
forms: attention over dense, paged and shared caches, acceptance, commit."""
import math
import random

import pytest
import torch

import tree_oracle as oracle
from slimkv_b200 import _lib, tree

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def seeded():
    torch.manual_seed(7)


def random_parents(rng, nodes):
    return [-1] + [rng.randrange(max(0, i - 4), i) for i in range(1, nodes)]


def make(B, T, H, G, D, lengths, Dv=None, dtype=BF16, page=0, layout='heads', context_only=False, seed=0, spare=5):
    """q, k, v, lengths, tables; what no row may read is NaN."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    Dv = Dv or D
    cap = max(lengths) + T + spare
    rand = lambda *s: torch.randn(*s, generator=gen, device='cuda', dtype=dtype)
    q = rand(B, T, H, D)
    tables = None
    if page:
        per = -(-cap // page)
        k, v = (rand(B * per + 3, page, 2, G, d)[:, :, 1] for d in (D, Dv))
        tables = torch.randperm(B * per + 3, generator=gen, device='cuda')[:B * per].view(B, per).to(torch.int32)
    elif layout == 'heads':
        k, v = (rand(B, G, cap, d).transpose(1, 2) for d in (D, Dv))
    elif layout == 'shared':
        k, v = (rand(1, cap, G, d) for d in (D, Dv))
    else:
        k, v = (rand(B, cap, G, d + 8)[..., :d] for d in (D, Dv))
    lens = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    for b in range(B):
        if layout == 'shared':
            break
        end = lengths[b] + (0 if context_only else T)
        for x in (k, v):
            if page:
                x[tables[b, end // page].long(), end % page:] = math.nan
                x[tables[b, end // page + 1:].long()] = math.nan
            else:
                x[b, end:] = math.nan
    if page:        # entries past the rows in use name no page
        for b in range(B):
            tables[b, -(-(lengths[b] + (0 if context_only else T)) // page):] = -7
    return q, k, v, lens, tables


def run(q, k, v, lens, tables=None, seen=None, nodes=None, context_only=False, scale=None):
    scale = scale or q.shape[3] ** -0.5
    mask = None if seen is None else oracle.words_of(seen).cuda()
    got = tree.tree_attention(q, k, v, lens, scale, mask=mask, nodes=nodes, block_tables=tables, context_only=context_only)
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    oracle.check_attention(got, oracle.attention(q, k, v, lens.tolist(), scale, seen, None if nodes is None else nodes.tolist(),
                                                 tables, context_only))
    return got


def trees(B, T, seed):
    rng = random.Random(seed)
    return torch.stack([oracle.ancestors(random_parents(rng, T)) for _ in range(B)])


@pytest.mark.parametrize('lengths', [[0], [1], [127], [128], [129], [517], [3000]])
def test_single_tokens(lengths):
    run(*make(1, 1, 32, 8, 128, lengths))


@pytest.mark.parametrize('B,T,H,G,D,lengths,dtype,page,layout', [
    (3, 13, 8, 2, 128, [0, 300, 77], BF16, 0, 'heads'),
    (2, 7, 10, 2, 128, [1000, 5], BF16, 16, ''),
    (2, 33, 8, 8, 64, [130, 256], FP16, 48, ''),
    (2, 40, 8, 2, 64, [0, 129], BF16, 24, ''),
    (1, 70, 8, 2, 128, [385], BF16, 0, 'rows'),
    (2, 129, 2, 1, 128, [100, 300], BF16, 0, 'rows'),
    (2, 90, 6, 2, 96, [64, 700], FP16, 128, ''),
    (4, 5, 3, 3, 40, [9, 0, 128, 1111], BF16, 0, 'rows'),
    (1, 3, 128, 1, 8, [200], FP16, 0, 'heads'),
    (2, 4, 12, 4, 160, [300, 31], BF16, 0, 'heads'),
    (1, 6, 5, 1, 320, [2000], FP16, 32, ''),
    (20, 2, 4, 2, 64, [50 * i for i in range(20)], BF16, 16, '')])
def test_trees(B, T, H, G, D, lengths, dtype, page, layout):
    run(*make(B, T, H, G, D, lengths, dtype=dtype, page=page, layout=layout, seed=T), seen=trees(B, T, T))


@pytest.mark.parametrize('D,Dv,T', [(128, 64, 9), (64, 128, 40), (320, 64, 3), (72, 320, 5)])
def test_value_dims_of_their_own(D, Dv, T):
    run(*make(2, T, 8, 2, D, [200, 411], Dv=Dv), seen=trees(2, T, 3))


@pytest.mark.parametrize('T', [1, 4, 33, 70])
def test_a_chain_needs_no_mask(T):
    args = make(2, T, 8, 2, 128, [100, 260])
    got = run(*args)
    chain = torch.ones(1, T, T).tril().bool()
    same = tree.tree_attention(*args[:3], args[3], 128 ** -0.5, mask=oracle.words_of(chain).cuda())
    assert torch.equal(got[0], same[0]) and torch.equal(got[1], same[1])


@pytest.mark.parametrize('rank,T,lengths', [(320, 4, [1000, 0, 77]), (160, 1, [1, 500, 128]), (320, 9, [4000, 129, 2])])
def test_latents(rank, T, lengths):
    """One latent head, planes of one buffer, no rows of the nodes."""
    lat = torch.randn(3, 2, max(lengths) + 3, rank, device='cuda').to(BF16)
    for b, n in enumerate(lengths):
        lat[b, :, n:] = math.nan
    q = torch.randn(3, T, 32, rank, device='cuda').to(BF16)
    run(q, lat[:, 0].unsqueeze(2), lat[:, 1].unsqueeze(2), torch.tensor(lengths, dtype=torch.int32, device='cuda'),
        context_only=True)


@pytest.mark.parametrize('T', [5, 40])
def test_ragged_trees(T):
    """Sequences with fewer nodes (or none): the rows past them are empty."""
    q, k, v, lens, _ = make(4, T, 8, 2, 128, [0, 140, 256, 0])
    nodes = torch.tensor([T, T - 3, 0, 1], dtype=torch.int32, device='cuda')
    run(q, k, v, lens, seen=trees(4, T, 1), nodes=nodes)


def test_empty_rows():
    """Mask rows without a bit: over an empty context nothing is seen."""
    q, k, v, lens, _ = make(2, 6, 8, 2, 128, [0, 40])
    seen = trees(2, 6, 2)
    seen[:, 3] = False
    got = run(q, k, v, lens, seen=seen)
    assert (got[0][0, 3] == 0).all() and (got[1][0, 3] == -math.inf).all() and got[1][1, 3].isfinite().all()


@pytest.mark.parametrize('T,page', [(6, 0), (40, 0), (6, 16)])
def test_unseen_infinities_do_not_spread(T, page):
    """A node's non-finite key or value reaches the rows that see it and no other."""
    q, k, v, lens, tables = make(2, T, 8, 2, 128, [100, 133], page=page)
    seen = trees(2, T, 4)
    for b, n in enumerate([100, 133]):
        for node, x, col, bad in ((2, v, 5, math.inf), (3, v, 70, math.nan), (4, k, 9, math.nan), (1, v, 127, -math.inf)):
            seen[b, :, node] = torch.arange(T) == node           # only the node itself sees it
            at = n + node
            if page:
                x[tables[b, at // page].long(), at % page, 1, col] = bad
            else:
                x[b, at, 1, col] = bad
    got = run(q, k, v, lens, tables, seen=seen)
    assert got[0][:, 0].isfinite().all() and got[0][:, 5:].isfinite().all()


@pytest.mark.parametrize('T,D', [(64, 64), (64, 128), (5, 64)])
def test_seen_infinities_in_many_short_pieces(T, D):
    """Shares of many segments of one or two key tiles, some of whose nodes hold
    infinities: they reach the rows that see them in every segment."""
    B, G = 40, 8
    lengths = [(7 * b) % 30 for b in range(B)]
    q, k, v, lens, _ = make(B, T, 32, G, D, lengths, seed=7)
    seen = trees(B, T, 8)
    for b, n in enumerate(lengths):
        v[b, n + (3 if b % 3 else T - 1), b % G, b % D] = math.inf
    want = torch.zeros(B, T, 32, D, dtype=torch.bool)
    for b in range(B):
        node = 3 if b % 3 else T - 1
        want[b, :, 4 * (b % G):4 * (b % G) + 4, b % D] = seen[b, :, node, None]
    for _ in range(20):
        out, _ = tree.tree_attention(q, k, v, lens, D ** -0.5, mask=oracle.words_of(seen).cuda())
        assert torch.equal(out.cpu() == math.inf, want) and not out.isnan().any()
    assert _lib.device_status(clear=True) == 0


@pytest.mark.parametrize('scale', [2.0, 0.5])
def test_peaked_scores(scale):
    """Scores up to the hundreds: maxima that keep growing along the keys."""
    q, k, v, lens, _ = make(1, 3, 8, 2, 128, [700])
    k.mul_(torch.linspace(0.1, 3, k.shape[1], device='cuda')[None, :, None, None])
    k[:, 703:] = math.nan
    run(q, k, v, lens, scale=scale)


def test_shared_cache_and_strided_outputs():
    q, k, v, lens, _ = make(3, 4, 8, 2, 128, [50, 60, 170], layout='shared')
    run(q, k, v, lens, seen=trees(3, 4, 5))
    wide = torch.zeros(3, 4, 8, 144, device='cuda', dtype=BF16)
    lse = torch.zeros(3, 4, 8, device='cuda')
    out, _ = tree.tree_attention(q, k, v, lens, 0.1, out=wide[..., 8:136], lse=lse)
    again, lse2 = tree.tree_attention(q, k, v, lens, 0.1)
    assert torch.equal(out, again) and torch.equal(lse, lse2) and (wide[..., :8] == 0).all() and (wide[..., 136:] == 0).all()


def test_offsets_past_32_bits():
    """Sequence strides of more than 2^32 bytes."""
    big = torch.empty(2, (1 << 24) + 64, 1, 128, device='cuda', dtype=BF16)      # 4.3 GB a sequence
    k = big.as_strided((2, 400, 1, 128), (big.stride(0), 1 << 15, 128, 1))
    v = big.as_strided((2, 400, 1, 128), (big.stride(0), 1 << 15, 128, 1), 256)
    k.normal_()
    v.normal_()
    q = torch.randn(2, 3, 4, 128, device='cuda').to(BF16)
    run(q, k, v, torch.tensor([390, 111], dtype=torch.int32, device='cuda'))


def test_another_stream_and_a_graph():
    q, k, v, lens, _ = make(2, 8, 8, 2, 128, [300, 10])
    mask = oracle.words_of(trees(2, 8, 7)).cuda()
    want = tree.tree_attention(q, k, v, lens, 0.09, mask=mask)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = tree.tree_attention(q, k, v, lens, 0.09, mask=mask)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = tree.tree_attention(q, k, v, lens, 0.09, mask=mask)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    lens.copy_(torch.tensor([17, 9], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    again = tree.tree_attention(q, k, v, lens, 0.09, mask=mask)
    assert torch.equal(held[0], again[0]) and torch.equal(held[1], again[1])


def test_lengths_past_the_cache_are_reported():
    q, k, v, _, _ = make(1, 2, 8, 2, 128, [60], spare=0)
    _lib.device_status(clear=True)
    tree.tree_attention(q, k, v, torch.tensor([61], dtype=torch.int32, device='cuda'), 0.1)
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH


def test_a_wait_that_runs_out_is_reported():
    q, k, v, lens, _ = make(1, 2, 8, 2, 128, [900])
    _lib.device_status(clear=True)
    tree.tree_attention(q, k, v, lens, 0.1, wait_limit_ns=1)
    assert _lib.device_status(clear=True) in (0, _lib.DEVICE_TIMEOUT)
    run(q, k, v, lens)


def test_attention_refusals():
    q, k, v, lens, _ = make(2, 4, 8, 2, 128, [50, 60])
    mask = torch.zeros(2, 4, 1, dtype=torch.int32, device='cuda')
    ok = dict(scale=0.1)
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan)):
        with pytest.raises(RuntimeError):
            tree.tree_attention(q, k, v, lens, **bad)
    with pytest.raises(RuntimeError):
        tree.tree_attention(q.float(), k, v, lens, **ok)
    with pytest.raises(RuntimeError):
        tree.tree_attention(q, k.to(FP16), v, lens, **ok)
    with pytest.raises(RuntimeError):
        tree.tree_attention(q, k, v, lens.long(), **ok)
    with pytest.raises(RuntimeError):
        tree.tree_attention(q, k, v, lens, mask=mask[:, :3], **ok)
    with pytest.raises(RuntimeError):
        tree.tree_attention(q, k, v, lens, mask=mask, context_only=True, **ok)
    with pytest.raises(RuntimeError):                    # 8 heads over 3
        tree.tree_attention(q, k[:, :, :1].expand(-1, -1, 3, -1).contiguous(), v[:, :, :1].expand(-1, -1, 3, -1).contiguous(), lens, **ok)
    with pytest.raises(RuntimeError):                    # rows not 16-byte aligned
        wide = torch.zeros(2, 70, 2, 132, device='cuda', dtype=BF16)
        tree.tree_attention(q, wide[..., :128], wide[..., :128], lens, **ok)
    with pytest.raises(RuntimeError):                    # pages of 12 rows
        pages = torch.zeros(20, 12, 2, 128, device='cuda', dtype=BF16)
        tree.tree_attention(q, pages, pages, lens, block_tables=torch.zeros(2, 8, dtype=torch.int32, device='cuda'), **ok)
    with pytest.raises(RuntimeError):
        tree.tree_attention(q.cpu(), k, v, lens, **ok)
    wide = torch.zeros(1, 8, 1, 328, device='cuda', dtype=BF16)
    with pytest.raises(RuntimeError):
        tree.tree_attention(wide, wide, wide, lens[:1], **ok)


# ------------------------------------------------------------------ masks --
@pytest.mark.parametrize('T', [1, 31, 32, 33, 64, 300, 1024])
def test_tree_masks(T):
    rng = random.Random(T)
    parents = [random_parents(rng, T), [-1] + list(range(T - 1)), [-1] * T]
    parents[2][T // 2] = T + 5                           # no node: a root
    got = tree.tree_masks(torch.tensor(parents, dtype=torch.int32, device='cuda')).cpu()
    assert torch.equal(got, oracle.words_of(torch.stack([oracle.ancestors(p) for p in parents])))


# ----------------------------------------------------------------- accept --
@pytest.mark.parametrize('B,T,V,dtype', [(1, 1, 7, torch.float32), (3, 9, 1000, BF16), (2, 40, 5003, FP16), (5, 5, 128256, torch.float32),
                                         (2, 70, 4097, BF16), (40, 3, 33, FP16), (16, 64, 32000, BF16)])
@pytest.mark.parametrize('offset', [0, 1])
def test_tree_accept(B, T, V, dtype, offset):
    rng = random.Random(V + offset)
    gen = torch.Generator(device='cuda').manual_seed(V)
    logits = torch.randn(B, T, V + 3, generator=gen, device='cuda').to(dtype)[..., offset:offset + V]   # rows off 16-byte boundaries
    parents = torch.tensor([random_parents(rng, T) for _ in range(B)], dtype=torch.int32)
    best = logits.float().argmax(-1).cpu()
    tokens = torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(1))
    for b in range(B):                                   # most nodes drafted what their parent's logits say
        for t in range(1, T):
            if rng.random() < 0.7:
                tokens[b, t] = best[b, parents[b, t]]
    got = tree.tree_accept(logits, tokens.cuda(), parents.cuda())
    for x, y in zip(got, oracle.accept(logits, tokens, parents)):
        assert torch.equal(x.cpu(), y)
    nodes = torch.tensor([rng.randint(0, T) for _ in range(B)], dtype=torch.int32)
    got = tree.tree_accept(logits, tokens.cuda(), parents.cuda(), nodes=nodes.cuda())
    for x, y in zip(got, oracle.accept(logits, tokens, parents, nodes.tolist())):
        assert torch.equal(x.cpu(), y)


@pytest.mark.parametrize('B,T,V,dtype', [(17, 64, 32003, BF16), (4, 70, 64001, torch.float32), (3, 90, 130003, FP16), (1, 1024, 33001, BF16),
                                         (70, 2, 240007, BF16)])
@pytest.mark.parametrize('offset', [0, 1])
def test_tree_accept_along_the_path(B, T, V, dtype, offset):
    """More than 64 MB of logits: argmaxes taken as the walk gets to them."""
    test_tree_accept(B, T, V, dtype, offset)


@pytest.mark.parametrize('dtype', [torch.float32, BF16, FP16])
def test_accept_ties_along_the_path(dtype):
    V = 3000005
    x = torch.full((6, 2, V), -math.inf, device='cuda', dtype=dtype)
    x[0, 0, [17, 375000, 375001, 2999999]] = 3.0         # a tie, within and across blocks
    x[1, 0, 2000005], x[1, 0, 4] = 0.0, -0.0
    x[2, 0, 3000004], x[2, 0, 3] = math.nan, math.inf
    x[3, 0, 1500000] = math.inf
    x[5, 0, [80000, 600000]] = math.nan
    x[5, 0, 600000] = -math.nan
    tokens = torch.tensor([[0, 17], [0, 4], [0, 3000004], [0, 1500000], [0, 0], [0, 80000]], device='cuda')
    parents = torch.tensor([[-1, 0]] * 6, dtype=torch.int32, device='cuda')
    path, count, _ = tree.tree_accept(x, tokens, parents)
    assert count.tolist() == [2] * 6 and path.tolist() == [[0, 1]] * 6


@pytest.mark.parametrize('dtype', [torch.float32, BF16, FP16])
def test_accept_ties_zeros_nan_and_infinities(dtype):
    V = 9000
    x = torch.full((6, 2, V), -math.inf, device='cuda', dtype=dtype)
    x[0, 0, [17, 4099, 8000]] = 3.0                      # a tie
    x[1, 0, 5], x[1, 0, 4] = 0.0, -0.0                   # the zeros are equal
    x[2, 0, 8999], x[2, 0, 3] = math.nan, math.inf       # a NaN is above infinity
    x[3, 0, 70] = math.inf
    x[5, 0, [8, 6000]] = math.nan
    x[5, 0, 6000] = -math.nan
    tokens = torch.tensor([[0, 17], [0, 4], [0, 8999], [0, 70], [0, 0], [0, 8]], device='cuda')
    parents = torch.tensor([[-1, 0]] * 6, dtype=torch.int32, device='cuda')
    path, count, _ = tree.tree_accept(x, tokens, parents)
    assert count.tolist() == [2] * 6 and path.tolist() == [[0, 1]] * 6


def test_accept_takes_the_first_of_equal_children_and_ignores_malformed_parents():
    x = torch.zeros(2, 5, 50, device='cuda')
    x[:, :, 9] = 1.0
    tokens = torch.full((2, 5), 9, device='cuda')
    parents = torch.tensor([[-1, 0, 0, 2, 1], [4, 3, 99, -5, 2]], dtype=torch.int32, device='cuda')
    path, count, after = tree.tree_accept(x, tokens, parents)
    assert path.tolist() == [[0, 1, 4, -1, -1], [0, -1, -1, -1, -1]] and count.tolist() == [3, 1] and after.tolist() == [9, 9]


def test_accept_refusals():
    x = torch.zeros(2, 3, 40, device='cuda')
    tokens, parents = torch.zeros(2, 3, dtype=torch.int64, device='cuda'), torch.zeros(2, 3, dtype=torch.int32, device='cuda')
    for args in ((x.double(), tokens, parents), (x, tokens.int(), parents), (x, tokens, parents.long()), (x, tokens[:1], parents),
                 (x.transpose(1, 2), tokens, parents), (x.cpu(), tokens, parents)):
        with pytest.raises(RuntimeError):
            tree.tree_accept(*args)


# ----------------------------------------------------------------- commit --
@pytest.mark.parametrize('L,B,T,G,D,Dv,dtype,page', [(1, 1, 1, 1, 8, 8, BF16, 0), (1, 3, 9, 2, 64, 128, BF16, 0),
                                                     (5, 2, 30, 8, 128, 128, BF16, 0), (2, 4, 20, 1, 320, 320, FP16, 0),
                                                     (1, 2, 13, 2, 64, 64, BF16, 16), (3, 2, 12, 2, 64, 64, torch.float32, 5),
                                                     (1, 2, 9, 4, 32, 16, torch.uint8, 0)])
def test_tree_commit(L, B, T, G, D, Dv, dtype, page):
    rng = random.Random(T)
    lengths = [rng.randint(0, 40) for _ in range(B)]
    paths = [[0] + sorted(rng.sample(range(1, T), rng.randint(0, T - 1))) for _ in range(B)]
    cap = max(lengths) + T
    per = -(-cap // page) if page else 0
    shape = (L, B * per, page, G) if page else (L, B, cap, G)
    k, v = (torch.randint(0, 100, shape + (d,), device='cuda').to(dtype) for d in (D, Dv))
    tables = torch.randperm(B * per)[:B * per].view(B, per).to(torch.int32).cuda() if page else None
    want = [k.clone(), v.clone()]
    for x in want:
        for b in range(B):
            rows = x[:, tables[b].long()].flatten(1, 2) if page else x[:, b].clone()
            new = rows.clone()
            for i, p in enumerate(paths[b]):
                new[:, lengths[b] + i] = rows[:, lengths[b] + p]
            if page:
                x[:, tables[b].long()] = new.unflatten(1, (per, page))
            else:
                x[:, b] = new
    if L == 1:
        k, v, want = k[0], v[0], [want[0][0], want[1][0]]
    i32 = dict(dtype=torch.int32, device='cuda')
    got = tree.tree_commit(k, v, torch.tensor(lengths, **i32), torch.tensor([p + [-1] * (T - len(p)) for p in paths], **i32),
                           torch.tensor([len(p) for p in paths], **i32), block_tables=tables)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    assert got.tolist() == [n + len(p) for n, p in zip(lengths, paths)]
    assert _lib.device_status() == 0


def test_commit_refusals_and_reports():
    k = torch.zeros(2, 10, 2, 64, device='cuda', dtype=BF16)
    i32 = dict(dtype=torch.int32, device='cuda')
    lens, path, count = torch.tensor([1, 2], **i32), torch.tensor([[0, 2], [0, 1]], **i32), torch.tensor([2, 2], **i32)
    with pytest.raises(RuntimeError):
        tree.tree_commit(k, k[..., :60], lens, path, count)
    with pytest.raises(RuntimeError):
        tree.tree_commit(k, k.float(), lens, path, count)
    with pytest.raises(RuntimeError):
        tree.tree_commit(k[:1], k[:1], lens, path, count)
    with pytest.raises(RuntimeError):
        tree.tree_commit(k, k, lens, path.long(), count)
    _lib.device_status(clear=True)
    before = k.clone()
    tree.tree_commit(k, k.clone(), lens, torch.tensor([[0, 9], [0, 1]], **i32), count)     # a node that the tree has not
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH and torch.equal(k, before)


def test_commit_reports_rows_without_a_place():
    """A destination in a page outside the pool, and accepted rows past the cache, moved or not."""
    i32 = dict(dtype=torch.int32, device='cuda')
    pages = torch.randn(6, 8, 2, 64, device='cuda').to(BF16)
    v, before = pages.clone(), pages.clone()
    _lib.device_status(clear=True)
    path = torch.tensor([[4, 5, 6, -1, -1, -1, -1]], **i32)
    new = tree.tree_commit(pages, v, torch.tensor([12], **i32), path, torch.tensor([2], **i32),
                           block_tables=torch.tensor([[0, 9, 2]], **i32))         # 16 and 17 to 12 and 13, in no page
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH and new.tolist() == [14]
    assert torch.equal(pages, before) and torch.equal(v, before)
    new = tree.tree_commit(pages, v, torch.tensor([12], **i32), torch.tensor([[0, 1, -1]], **i32), torch.tensor([2], **i32),
                           block_tables=torch.tensor([[0, -1, 2]], **i32))        # rows that stay, in no page
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH and new.tolist() == [14]
    k = pages[:1].contiguous()
    new = tree.tree_commit(k, k.clone(), torch.tensor([6], **i32), torch.tensor([[0, 1, 2, -1]], **i32), torch.tensor([3], **i32))
    assert _lib.device_status(clear=True) == _lib.DEVICE_BAD_LENGTH and new.tolist() == [8]
    new = tree.tree_commit(k, k.clone(), torch.tensor([6], **i32), torch.tensor([[0, 1, 2, -1]], **i32), torch.tensor([2], **i32))
    assert _lib.device_status(clear=True) == 0 and new.tolist() == [8]


@pytest.mark.parametrize('form', ['same', 'front', 'back', 'overlap', 'pages', 'planes', 'halves'])
def test_commit_of_keys_and_values_in_one_buffer(form):
    """K and V that are (parts of) the same rows move once; those that lie between each other's rows move each."""
    B, T, cap, G, D = 5, 40, 60, 2, 128
    rng = random.Random(11)
    lengths = [rng.randint(0, 20) for _ in range(B)]
    paths = [[0] + sorted(rng.sample(range(1, T), rng.randint(15, T - 1))) for _ in range(B)]
    tables = None
    if form == 'pages':
        x = torch.randn(B * 4, 15, 2, G, D, device='cuda').to(BF16)
        tables = torch.randperm(B * 4)[:B * 4].view(B, 4).to(torch.int32).cuda()
        k, v = x[:, :, 0], x[:, :, 1]
    elif form == 'planes':
        x = torch.randn(B, 2, cap, G, D, device='cuda').to(BF16)
        k, v = x[:, 0], x[:, 1]
    else:
        x = torch.randn(B, cap, G, D, device='cuda').to(BF16)
        k, v = {'same': (x, x), 'front': (x, x[..., :64]), 'back': (x, x[..., 64:]), 'overlap': (x[..., :96], x[..., 32:]),
                'halves': (x[..., :64], x[..., 64:])}[form]
    want = x.clone()
    for b in range(B):
        for i, p in enumerate(paths[b]):
            if form == 'pages':
                (pd, rd), (ps, rs) = (divmod(lengths[b] + j, 15) for j in (i, p))
                want[tables[b, pd].long(), rd] = x[tables[b, ps].long(), rs]
            elif form == 'planes':
                want[b, :, lengths[b] + i] = x[b, :, lengths[b] + p]
            else:
                want[b, lengths[b] + i] = x[b, lengths[b] + p]
    i32 = dict(dtype=torch.int32, device='cuda')
    tree.tree_commit(k, v, torch.tensor(lengths, **i32), torch.tensor([p + [-1] * (T - len(p)) for p in paths], **i32),
                     torch.tensor([len(p) for p in paths], **i32), block_tables=tables)
    assert torch.equal(x, want) and _lib.device_status() == 0


@pytest.mark.parametrize('T,G', [(1, 8), (5, 8), (40, 8)])
@pytest.mark.parametrize('dtype', [FP16, BF16])
def test_many_small_probabilities_behind_a_dominant_one(T, G, dtype):
    """One key 17.5 to 20 nats above thousands: their weight of some 2^-26 each does not get lost.  The values' bound is
    the oracle's with a probability's fp16 rounding below 2^-32 of the largest (not 2^-25)."""
    n, D, H, B = 4000, 64, 8, 16
    q = torch.zeros(B, T, H, D, device='cuda', dtype=dtype)
    q[..., 0] = 8
    k = torch.zeros(1, n, G, D, device='cuda', dtype=dtype)
    k[..., 0] = -torch.empty(1, n, G, device='cuda').uniform_(17.5, 20)
    k[:, 0] = 0
    v = torch.rand(1, n, G, D, device='cuda').to(dtype)
    v[:, 0] = 0
    lens = torch.full((B,), n, dtype=torch.int32, device='cuda')
    got = tree.tree_attention(q, k, v, lens, 0.125, context_only=True)
    out, lse, tol, tol_lse = oracle.attention(q[:1, :1], k, v, [n], 0.125, context_only=True)
    if dtype == FP16:
        tol = tol - n * (2.0 ** -25 - 2.0 ** -32) * v.double().cpu()[0].amax(0)[torch.arange(H) * G // H]
    for b in range(0, B, 5):
        for t in range(T):
            oracle.check_attention((got[0][b:b + 1, t:t + 1], got[1][b:b + 1, t:t + 1]), (out, lse, tol, tol_lse))


@pytest.mark.parametrize('step', [5.4, 5.6, 11.0])
@pytest.mark.parametrize('T', [3, 40])
def test_fp16_probabilities_above_the_running_maximum(T, step):
    """Maxima that grow by a little less and more than 2^8 and 2^15 from one key tile to the next."""
    q, k, v, lens, _ = make(1, T, 8, 2, 64, [700], dtype=FP16)
    q.zero_()
    q[..., 0] = 8
    k[:, :700 + T, :, 0] = (torch.arange(700 + T, device='cuda') // 64 * step - 30)[None, :, None].to(FP16)
    run(q, k, v, lens, scale=0.125)


@pytest.mark.parametrize('B,T,V,dtype', [(4, 70, 64001, torch.float32), (1, 1024, 33001, BF16), (20, 33, 60001, FP16), (16, 64, 33001, BF16)])
def test_accepted_chains_of_every_length(B, T, V, dtype):
    """Chains accepted up to each length around the number of steps after which a walk may stop, or whole."""
    gen = torch.Generator(device='cuda').manual_seed(V)
    logits = torch.randn(B, T, V, generator=gen, device='cuda').to(dtype)
    best = torch.stack([x.float().argmax(-1) for x in logits])
    parents = torch.arange(-1, T - 1, dtype=torch.int32, device='cuda').expand(B, T).contiguous()
    lengths = [1, 2, 6, 7, 8, 9, 10, 17, T - 1, T]
    for turn in range(0, len(lengths), B) if B < len(lengths) else range(1):
        tokens = torch.cat([best[:, :1], best[:, :-1]], 1)
        want = [lengths[(turn + b) % len(lengths)] for b in range(B)]
        for b, n in enumerate(want):
            if n < T:
                tokens[b, n] = (tokens[b, n] + 1) % V
        nodes = [T if b % 3 else max(1, T - 1 - b) for b in range(B)]
        for given in (None, torch.tensor(nodes, dtype=torch.int32, device='cuda')):
            path, count, after = tree.tree_accept(logits, tokens, parents, nodes=given)
            counts = [min(n, T if given is None else m) for n, m in zip(want, nodes)]
            assert count.tolist() == counts and after.tolist() == [int(best[b, c - 1]) for b, c in enumerate(counts)]
            assert path.tolist() == [list(range(c)) + [-1] * (T - c) for c in counts]


@pytest.mark.parametrize('T,H,G,D,n,context_only', [(2, 8, 2, 128, 60000, False), (20, 8, 1, 128, 60000, False), (4, 32, 1, 320, 60000, True)])
def test_waits_that_run_out_end_every_pipeline(T, H, G, D, n, context_only):
    """With a limit of 1 ns the waits run out while the rings are full (one and two row tiles, K slots of a row and of a
    chunk): the timeout is reported, and the next call, with the usual limit, gives what the one before gave."""
    q, k, v, lens, _ = make(1, T, H, G, D, [n], context_only=context_only)
    want = tree.tree_attention(q, k, v, lens, 0.1, context_only=context_only)
    assert _lib.device_status(clear=True) == 0
    tree.tree_attention(q, k, v, lens, 0.1, context_only=context_only, wait_limit_ns=1)
    assert _lib.device_status(clear=True) & _lib.DEVICE_TIMEOUT
    got = tree.tree_attention(q, k, v, lens, 0.1, context_only=context_only)
    assert _lib.device_status(clear=True) == 0
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize('T,page,rank', [(5, 48, 320), (3, 96, 160), (1, 16, 64)])
def test_latent_pages(T, page, rank):
    """Latents in pages, which hold no rows of the nodes."""
    q, k, v, lens, tables = make(3, T, 32, 1, rank, [0, 700, 129], page=page, context_only=True)
    run(q, k, v, lens, tables, context_only=True)
