"""Trees of drafted tokens on the paged 8-bit cache, on the GPU against 64-bit restatements (oracle/drafts.py): masks, attention, rotation at positions of several axes, kept rows, and all of them in turn."""
import random

import pytest
import torch

from moshi_b200.models import PagedBatch, PagedKVCache, PagedTree, PagePool, RotaryTable
from moshi_b200.models import paged
from oracle import drafts, paged as oracle

from .paged_util import Content, batch_of

pytestmark = pytest.mark.gpu
FORMS = [("int8", 128, 64), ("fp8_e4m3", 128, 16), ("int8", 64, 16), ("fp8_e4m3", 64, 128), ("int8", 128, 32)]


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).cuda()


def some_tree(n, seed, kind="mixed"):
    r = random.Random(seed)
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1) if n else []
    if kind == "roots":
        return [-1] * n
    return [-1 if i == 0 or r.random() < 0.1 else i - 1 if r.random() < 0.4 else r.randrange(i) for i in range(n)]


def check(lengths, trees, heads, form, window=0, sinks=0, scale=None, spread=1.0, total=None, q_size=1.0, seed=1, first=0):
    """lengths: tokens in front of the step; trees: of the sequences.  The step's own tokens are in the cache already."""
    dtype, dim, page = form
    hq, hkv = heads
    new = [len(t) for t in trees]
    c = Content([a + n for a, n in zip(lengths, new)], hkv, dim, page, dtype, seed=seed, spread=spread)
    cache = c.cache()
    T = first + sum(new) if total is None else total
    g = torch.Generator().manual_seed(seed + 1)
    wide = (torch.randn(T, hq + 3, dim, generator=g) * q_size).bfloat16().cuda()
    q = wide[:, 2:hq + 2]                                # rows lie apart
    out = torch.full((T, hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    rows = [first]
    for n in new:
        rows.append(rows[-1] + n)
    batch = PagedBatch(i32(c.table), i32(lengths), i32(rows), T, max(new))
    tree = PagedTree(batch, i32([0] * first + [x for t in trees for x in t] + [0] * (T - rows[-1])))
    got = cache.attend(batch, q, scale=scale, window=window, sinks=sinks, out=out, tree=tree)
    assert got is out and cache.error_flags() == 0 and tree.error_flags() == 0
    for s, (a, t) in enumerate(zip(lengths, trees)):
        if t:
            at = rows[s]
            want, tol = drafts.attend(q[at:at + len(t)].double().cpu(), *c.kvt(s), drafts.visible(t, a, window, sinks), dim ** -0.5 if scale is None else scale)
            off = (out[at:at + len(t)].double().cpu() - want).abs()
            assert bool((off <= tol).all()), (s, a, len(t), float((off - tol).max()), float((off / tol.clamp_min(1e-30)).max()))
    assert bool((out[:first] == 7.0).all()) and bool((out[rows[-1]:] == 7.0).all())      # rows of no sequence
    return out


# ---- the tree ----
@pytest.mark.parametrize("sizes", [[1, 0, 31, 32, 33], [64, 65, 100, 1], [1024, 700, 3], [1]], ids=str)
@pytest.mark.parametrize("kind", ["mixed", "chain", "star", "roots"])
def test_masks_and_positions(sizes, kind):
    trees = [some_tree(n, 7 + i, kind) for i, n in enumerate(sizes)]
    before = [5 + 1000 * i for i in range(len(sizes))]
    T = sum(sizes) + 4
    batch = batch_of(torch.zeros(len(sizes), 300, dtype=torch.int32), before, sizes, total=T)
    tree = PagedTree(batch, i32([x for t in trees for x in t] + [9] * 4))
    tree.seen[T - 4:], tree.positions[T - 4:] = 77, 78
    tree.update()
    assert tree.error_flags() == 0 and tree.seen.shape == (T, -(-max(sizes) // 32))
    seen, pos, at = tree.seen.cpu().long() & 0xffffffff, tree.positions.cpu(), 0
    for b, t in zip(before, trees):
        want = drafts.visible(t, 0)
        bits = ((seen[at:at + len(t)].repeat_interleave(32, 1) >> torch.arange(32).repeat(seen.shape[1])) & 1).bool()
        assert torch.equal(bits[:, :len(t)], want) and not bool(bits[:, len(t):].any())
        assert pos[at:at + len(t)].tolist() == [b + d for d in drafts.depths(t)]
        at += len(t)
    assert bool((tree.seen[T - 4:] == 77).all()) and bool((tree.positions[T - 4:] == 78).all())


def test_parents_that_are_not_in_front_count_as_the_last_cached_token():
    parents = [-1, 0, 2, 7, -2, 1000000, -2 ** 31, 4]
    batch = batch_of(torch.zeros(1, 4, dtype=torch.int32), [10], [8])
    tree = PagedTree(batch, i32(parents))
    assert tree.error_flags() == paged.BAD_TREE and tree.positions.tolist() == [10 + d for d in drafts.depths(parents)]
    tree.clear_error_flags()
    tree.parents.copy_(i32([-1, 0, 1, 2, 3, 4, 5, 6]))
    tree.update()
    assert tree.error_flags() == 0 and tree.positions.tolist() == list(range(10, 18))
    for rows, before in (([0, 9], [10]), ([-1, 7], [10]), ([5, 3], [10]), ([0, 8], [-1])):
        other = PagedTree(PagedBatch(i32(torch.zeros(1, 4)), i32(before), i32(rows), 8, 8), i32(parents))
        assert other.error_flags() == paged.BAD_BATCH and bool((other.positions == 0).all())


# ---- attention ----
@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("heads", [(4, 4), (8, 1), (6, 2), (15, 3), (40, 2)], ids=str)
def test_trees_of_a_few_tokens(form, heads):
    lengths = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 300, 40]
    check(lengths, [some_tree((i * 5) % 9, i) for i in range(12)], heads, form)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("heads", [(4, 4), (7, 1), (24, 2)], ids=str)
@pytest.mark.parametrize("sizes", [[12, 5, 1, 0, 9], [33, 0, 64, 1], [130, 257], [20]], ids=str)
def test_larger_trees(form, heads, sizes):
    check([0, 37, 100, 5, 64][:len(sizes)], [some_tree(n, 3 * n) for n in sizes], heads, form)


@pytest.mark.parametrize("size", [10, 14, 25])
@pytest.mark.parametrize("dim,page", [(128, 64), (64, 128)])
def test_one_unit_for_all_ctas(size, dim, page):
    """One head of the cache: 4, 12 and over 50 parts of a unit, of 32 to 128 columns."""
    for length in (3000, 9500, 40000):
        check([length], [some_tree(size, length)], (4, 1), ("int8", dim, page))
    check([14000, 20000], [some_tree(size, 1), some_tree(size - 1, 2)], (4, 1), ("fp8_e4m3", dim, page), window=12800, sinks=100)


@pytest.mark.parametrize("n", [1, 31, 32, 33, 512, 513])
def test_numbers_of_sequences(n):
    """A warp looks at 32 sequences, a block at 512."""
    r = random.Random(n)
    check([r.choice([0, 5, 30, 64]) for _ in range(n)], [some_tree(r.randint(0, 9) if i + 1 < n else 9, i) for i in range(n)], (8, 1), ("int8", 64, 32))
    check([r.choice([0, 300, 500]) for _ in range(n)], [some_tree(r.choice([0, 0, 0, 5]) if i + 1 < n else 5, i) for i in range(n)], (8, 1), ("int8", 128, 32))


@pytest.mark.parametrize("size", [2, 5, 18])
def test_many_sequences(size):
    """More than a block looks at in one go, most of them short, some empty."""
    r = random.Random(size)
    check([r.choice([0, 1, 17, 40]) for _ in range(1500)], [some_tree(r.randint(0, size), i) for i in range(1500)], (8, 1), ("int8", 64, 16))


@pytest.mark.parametrize("kind", ["chain", "star", "roots"])
@pytest.mark.parametrize("size", [5, 40])
def test_kinds_of_trees(kind, size):
    check([200, 64], [some_tree(size, 1, kind), some_tree(size - 2, 2, kind)], (8, 2), ("int8", 128, 64))
    check([200, 64], [some_tree(size, 1, kind), some_tree(size - 2, 2, kind)], (8, 2), ("fp8_e4m3", 64, 16), window=8, sinks=2)


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_units_that_are_cut(form):
    """Few sequences: their keys go to all CTAs, ends of runs among the places that are no tiles."""
    check([9000], [some_tree(20, 1)], (4, 1), form)
    check([5000, 257], [some_tree(3, 1), some_tree(2, 2)], (4, 2), form)
    check([3001, 0, 4000], [some_tree(70, 1), some_tree(1, 2), some_tree(9, 3)], (6, 2), form)


@pytest.mark.parametrize("window,sinks", [(1, 0), (2, 1), (16, 0), (17, 4), (100, 70), (64, 16), (1000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_windows_and_first_tokens(form, window, sinks):
    """Windows shorter than the trees are deep, too."""
    check([0, 3, 90, 400, 1500], [some_tree(4, s) for s in range(5)], (4, 2), form, window, sinks)
    check([0, 120, 700], [some_tree(50, 1, "chain"), some_tree(20, 2), some_tree(45, 3)], (6, 2), form, window, sinks)


@pytest.mark.parametrize("size", [2, 60])
def test_rows_of_no_sequence(size):
    check([50, 3], [some_tree(size, 1), some_tree(2, 2)], (8, 2), ("int8", 128, 64), total=size + 2 + 37)
    check([50, 3], [some_tree(size, 1), some_tree(2, 2)], (8, 2), ("int8", 128, 64), total=size + 2 + 37, first=11)


@pytest.mark.parametrize("size", [4, 50])
def test_scales_far_apart_and_large_queries(size):
    trees = [some_tree(size, 1), some_tree(size, 2)]
    check([400, 77], trees, (8, 2), ("int8", 128, 32), spread=30.0)
    check([400, 77], trees, (8, 2), ("fp8_e4m3", 128, 32), spread=1000.0)
    check([400, 77], trees, (8, 2), ("int8", 64, 64), q_size=300.0)
    check([400, 77], trees, (8, 2), ("int8", 64, 64), q_size=1e-30, scale=1e20)


@pytest.mark.parametrize("size", [3, 40])
def test_pages_of_zeros(size):
    t = some_tree(size, 5)
    c = Content([300 + size], 2, 128, 64, "int8")
    cache = c.cache()
    page = int(c.table[0, 1])
    for side, (pool, scale) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        pool[page], scale[page], c.codes[side][page], c.scales[side][page] = 0, 0, 0, 0
    q = torch.randn(size, 8, 128).bfloat16().cuda()
    want, tol = drafts.attend(q.double().cpu(), *c.kvt(0), drafts.visible(t, 300), 128 ** -0.5)
    batch = batch_of(c.table, [300], [size])
    assert bool(((cache.attend(batch, q, tree=PagedTree(batch, i32(t))).double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("size", [4, 40, 100])
def test_a_query_that_is_not_finite_spoils_its_own_results_only(size):
    c = Content([500 + size], 2, 128, 64, "int8")
    cache, q = c.cache(), torch.randn(size, 8, 128).bfloat16().cuda()
    batch = batch_of(c.table, [500], [size])
    tree = PagedTree(batch, i32(some_tree(size, 3)))
    want = cache.attend(batch, q, tree=tree)
    q[0, 3, 5], q[-1, 6, 0] = float("nan"), float("inf")
    got = cache.attend(batch, q, tree=tree)
    spoilt = torch.zeros(size, 8, dtype=torch.bool, device="cuda")
    spoilt[0, 3] = spoilt[-1, 6] = True
    assert bool(got[spoilt].isnan().all()) and torch.equal(got[~spoilt], want[~spoilt])


@pytest.mark.parametrize("size", [4, 60])
def test_what_does_not_fit_is_left_out_and_recorded(size):
    c = Content([100 + size, 200 + size], 2, 64, 16, "int8")
    cache, q, trees = c.cache(), torch.randn(2 * size, 8, 64).bfloat16().cuda(), [some_tree(size, 1), some_tree(size, 2)]
    parents = i32(trees[0] + trees[1])
    exact = [drafts.attend(q[size * s:size * (s + 1)].double().cpu(), *c.kvt(s), drafts.visible(trees[s], (100, 200)[s]), 0.125) for s in (0, 1)]

    def run(table, before, rows, max_rows=size):
        out = torch.full_like(q, 7.0)
        batch = PagedBatch(i32(table), i32(before), i32(rows), 2 * size, max_rows)
        cache.attend(batch, q, out=out, tree=PagedTree(batch, parents))
        flags = cache.error_flags()
        cache.clear_error_flags()
        return out.cpu(), flags

    def good(out, s):
        want, tol = exact[s]
        return bool(((out[size * s:size * (s + 1)].double() - want).abs() <= tol).all())
    rows = [0, size, 2 * size]
    for before, r in (([-1, 200], rows), ([2 ** 31 - 1, 200], rows), ([100000, 200], rows), ([100, 200], [-5, size, 2 * size]), ([100, 200], [2 * size, size, 2 * size])):
        out, flags = run(c.table, before, r)
        assert flags == paged.BAD_BATCH and good(out, 1) and bool((out[:size] == 7).all())
    out, flags = run(c.table, [100, 200], [0, size, 2 * size + 1])
    assert flags == paged.BAD_BATCH and good(out, 0) and bool((out[size:] == 7).all())
    out, flags = run(c.table, [100, 200], [0, 0, 2 * size])               # more than max_rows
    assert flags == paged.BAD_BATCH and bool((out == 7).all())
    for bad in (-1, c.pages, 2 ** 31 - 1, -2 ** 31):                      # tokens of a page that is not there are left out
        table = c.table.clone()
        table[0, 2] = bad
        out, flags = run(table, [100, 200], rows)
        assert flags == paged.BAD_PAGE and good(out, 1)
        seen = drafts.visible(trees[0], 100)
        seen[:, 32:48] = False
        want, tol = drafts.attend(q[:size].double().cpu(), *c.kvt(0), seen, 0.125)
        assert bool(((out[:size].double() - want).abs() <= tol).all())


@pytest.mark.parametrize("size", [4, 40])
def test_a_row_whose_own_page_is_missing_gets_zeros(size):
    """Nothing cached and no page: the mask leaves rows empty."""
    c = Content([size], 2, 128, 64, "int8")
    cache, q, out = c.cache(), torch.randn(size, 8, 128).bfloat16().cuda(), torch.full((size, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    batch = batch_of(torch.full_like(c.table, -1), [0], [size])
    cache.attend(batch, q, out=out, tree=PagedTree(batch, i32(some_tree(size, 1))))
    assert cache.error_flags() == paged.BAD_PAGE and bool((out == 0).all())


@pytest.mark.parametrize("size", [3, 30, 200])
def test_captured_steps(size):
    """Two graphs side by side; new trees, lengths and queries behind the same pointers."""
    c = Content([3000 + size], 2, 128, 64, "int8")
    cache, runs = c.cache(), []
    for i in range(2):
        q = torch.randn(size, 8, 128, generator=torch.Generator().manual_seed(i)).bfloat16().cuda()
        batch = batch_of(c.table, [3000], [size])
        tree = PagedTree(batch, i32(some_tree(size, i)))
        want = cache.attend(batch, q, tree=tree)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            tree.update()
            out = cache.attend(batch, q, tree=tree)
        runs.append((graph, stream, batch, tree, q, out, want))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for *_, out, want in runs:
        assert torch.equal(out, want)
    graph, stream, batch, tree, q, out, want = runs[0]
    q.copy_(runs[1][4])
    tree.parents.copy_(i32(some_tree(size, 9)))
    batch.before.fill_(1000)
    other = batch_of(c.table, [1000], [size])
    fresh = cache.attend(other, q, tree=PagedTree(other, i32(some_tree(size, 9))))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, fresh) and not torch.equal(out, want) and cache.error_flags() == 0


def test_another_stream_than_the_default():
    c = Content([700 + 30], 2, 128, 64, "int8")
    cache, q = c.cache(), torch.randn(30, 8, 128).bfloat16().cuda()
    batch = batch_of(c.table, [700], [30])
    tree = PagedTree(batch, i32(some_tree(30, 1)))
    want = cache.attend(batch, q, tree=tree)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [cache.attend(batch, q, tree=tree) for _ in range(30)]
    stream.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("size", [4, 40])
def test_far_positions_under_a_window(size):
    """Lengths of two billion: tables that are nearly all one page."""
    page, dim, before = 128, 64, 2 * 10 ** 9
    t = some_tree(size, 4)
    cache = PagedKVCache(3, 1, dim, page, "int8")
    table = torch.zeros(1, (before + size) // page + 1, dtype=torch.int32, device="cuda")
    table[0, -1], table[0, -2] = 1, 2
    batch = PagedBatch(table, i32([before]), i32([0, size]), size, size)
    k, v, q = (torch.randn(size, 1, dim).bfloat16().cuda() for _ in range(3))
    tree = PagedTree(batch, i32(t))
    cache.append(batch, k, v)
    out = cache.attend(batch, q, window=3, tree=tree)
    rows = [torch.zeros(0)]
    kv = []
    for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        blocks = [int(table[0, b]) for b in range((before - 2) // page, (before + size - 1) // page + 1)]
        x = torch.cat([pool[b].float().double().cpu().transpose(0, 1) * float(scale[b, 0]) for b in blocks])
        at = before - (before - 2) // page * page
        kv.append(x[at - 2:at + size])
    seen = drafts.visible(t, 2, 3)
    want, tol = drafts.attend(q.double().cpu(), kv[0], kv[1], torch.full((size + 2, 1), 10.0, dtype=torch.float64), seen, dim ** -0.5)
    assert cache.error_flags() == 0 and bool(((out.double().cpu() - want).abs() <= tol).all()) and rows


def test_offsets_past_32_bits():
    """A cache above 2^32 bytes a side: attention, keep and copies of its last pages."""
    page, dim, heads = 128, 128, 8
    pages = (1 << 32) // (page * dim * heads) + 20
    k, v = (torch.empty(pages, heads, page, dim, dtype=torch.int8, device="cuda") for _ in range(2))
    cache = PagedKVCache.from_tensors(k, v, *(torch.ones(pages, heads, device="cuda") for _ in range(2)))
    size, before = 40, 300
    c = Content([before + size], heads, dim, page, "int8", spare=0)
    used = torch.arange(pages - c.pages, pages)
    for pool, scale, codes, s in zip((k, v), (cache.k_scale, cache.v_scale), c.codes, c.scales):
        pool[used.cuda()], scale[used.cuda()] = codes.to(torch.int8).cuda(), s.cuda()
    batch = batch_of(c.table + (pages - c.pages), [before], [size])
    t, q = some_tree(size, 1), torch.randn(size, 16, dim).bfloat16().cuda()
    out = cache.attend(batch, q, tree=PagedTree(batch, i32(t)))
    want, tol = drafts.attend(q.double().cpu(), *c.kvt(0), drafts.visible(t, before), dim ** -0.5)
    assert bool(((out.double().cpu() - want).abs() <= tol).all())
    path = [0, 3, 4, 30]
    moved = k[used[c.table[0, 2].item()].item(), 0, (before + 3) % page].clone()
    cache.keep(batch, i32(path + [0] * (size - 4)), i32([4]))
    assert torch.equal(k[used[c.table[0, 2].item()].item(), 0, (before + 1) % page], moved) and cache.error_flags() == 0
    pool = PagePool([cache], 2, 4)
    pool.table[0, 0], pool.lengths[0], pool.held[0], pool.refs[:] = pages - 1, 5, 1, 1
    pool.refs[pages - 3] = 0
    pool.rearrange(i32([0, 0]))
    pool.reserve(i32([1, 1]))
    assert pool.error_flags() == 0 and pool.table[:, 0].tolist() == [pages - 3, pages - 1] and torch.equal(k[pages - 3], k[pages - 1]) and torch.equal(v[pages - 3], v[pages - 1])


# ---- rotation at positions of the rows' own ----
@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("pairing,part", [("adjacent", 1.0), ("halves", 1.0), ("halves", 0.5), ("adjacent", 0.25)])
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("new", [[1, 3, 0, 16], [70, 2, 17, 0]], ids=str)
def test_positions_of_several_axes(form, pairing, part, axes, new):
    dtype, dim, page = form
    before, hkv, hq, T, rot = [0, 17, 64, 30], 3, 6, sum(new) + 3, int(part * dim)
    r = random.Random(5)
    pair_axis = [r.randrange(axes) for _ in range(rot // 2)]
    pair_axis[-1] = axes - 1
    c = Content(before, hkv, dim, page, dtype, capacity=[b + n for b, n in zip(before, new)])
    cache = c.cache()
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(T, h, dim, generator=g).bfloat16().cuda() for h in (hq, hkv, hkv))
    positions = torch.randint(-2 ** 31, 2 ** 31, (axes, T), generator=g).int()
    positions[:, ::2] = torch.randint(-300, 5000, (axes, (T + 1) // 2), generator=g).int()
    wide = torch.zeros(axes, T + 6, dtype=torch.int32)
    wide[:, 2:T + 2] = positions
    rotary = RotaryTable(rot, pairing=pairing, axes=pair_axis)
    assert rotary.axes == axes
    q_out = torch.full((T, hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    batch = batch_of(c.table, before, new, total=T)
    cache.append(batch, k, v, q=q, rotary=rotary, q_out=q_out, positions=wide.cuda()[:, 2:T + 2])
    assert cache.error_flags() == 0
    at = 0
    for s, (b, n) in enumerate(zip(before, new)):
        here = positions[:, at:at + n].long()
        # the 64-bit angle itself is off by position * 2^-53 of a radian and by 2^-53 of the position's share
        exact = drafts.rotated(q[at:at + n].double().cpu(), here, pair_axis, rot, pairing=pairing)
        if n:
            assert bool(((q_out[at:at + n].double().cpu() - exact).abs() <= 2.0 ** -8 * exact.abs() + 2.0 ** -18 * exact.abs().amax(-1, keepdim=True)).all())
        rows = (drafts.rotated(k[at:at + n].double().cpu(), here, pair_axis, rot, pairing=pairing), v[at:at + n].double().cpu())
        for side, (x, pool, scale) in enumerate(zip(rows, (cache.k, cache.v), (cache.k_scale, cache.v_scale))):
            for p in range(b // page, -(-(b + n) // page)) if n else ():
                pg, o, e = int(c.table[s, p]), max(b - p * page, 0), min(b + n - p * page, page)
                for h in range(hkv):
                    y = x[p * page + o - b:p * page + e - b, h]
                    _, want_s = oracle.append(c.codes[side][pg, h], float(c.scales[side][pg, h]), o, y, dtype)
                    got_s = float(scale[pg, h])
                    assert abs(got_s - want_s) <= 2.0 ** -18 * want_s
                    half = 0.5 * got_s if dtype == "int8" else torch.maximum(2.0 ** -4 * y.abs(), torch.as_tensor(2.0 ** -10 * got_s))
                    # half a step, and 2^-18 of the page's largest (448 steps at most) for the rotation
                    assert bool(((pool[pg, h, o:e].float().double().cpu() * got_s - y).abs() <= half * (1 + 2.0 ** -9) + 2.0 ** -9 * got_s).all())
        at += n
    assert bool((q_out[at:] == 7.0).all())


@pytest.mark.parametrize("new", [[1, 5, 0], [40, 3, 100]], ids=str)
def test_positions_that_are_the_places_change_nothing(new):
    before, results = [0, 60, 1000], []
    c = Content(before, 2, 128, 64, "int8", capacity=[b + n for b, n in zip(before, new)])
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(sum(new), h, 128, generator=g).bfloat16().cuda() for h in (4, 2, 2))
    batch = batch_of(c.table, before, new)
    positions = i32([b + i for b, n in zip(before, new) for i in range(n)])
    for rotary, at in ((RotaryTable(128), None), (RotaryTable(128), positions), (RotaryTable(128), positions[None]), (RotaryTable(128, axes=[j % 3 for j in range(64)]), positions[None].expand(3, -1).contiguous())):
        cache = c.cache()
        q_out = cache.append(batch, k, v, q=q, rotary=rotary, positions=at)
        results.append([q_out, cache.k, cache.v, cache.k_scale.nan_to_num(-1), cache.v_scale.nan_to_num(-1)])
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(results[0], r))


# ---- kept rows ----
@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("spread", [1.0, 8.0])
@pytest.mark.parametrize("sizes", [[5, 1, 0, 16, 9], [40, 70, 1, 130, 3]], ids=str)
def test_kept_rows(form, spread, sizes):
    dtype, dim, page = form
    before, heads, r = [0, 15, 30, 64, 127], 3, random.Random(len(sizes) + sizes[0])
    caches, contents = [], []
    for layer in range(2):
        c = Content([b + n for b, n in zip(before, sizes)], heads, dim, page, dtype, seed=layer, spread=spread)
        c.table = contents[0].table if layer else c.table
        contents.append(c)
        caches.append(c.cache() if layer == 0 else None)
    # the second layer's pages lie where the first's do
    contents[1].codes = [x.clone() for x in contents[1].codes]
    caches[1] = contents[1].cache()
    paths = [sorted(r.sample(range(n), r.randint(0, n))) for n in sizes]
    paths[3] = list(range(sizes[3]))                     # all of them
    kept = [x for p, n in zip(paths, sizes) for x in p + [-7] * (n - len(p))]
    was = [[x.clone() for x in (c.k.view(torch.int8), c.v.view(torch.int8), c.k_scale, c.v_scale)] for c in caches]
    batch = batch_of(contents[0].table, before, sizes)
    PagePool(caches, 1, 1).keep(batch, i32(kept), i32([len(p) for p in paths]))
    assert all(c.error_flags() == 0 for c in caches)
    for c, cache, old in zip(contents, caches, was):
        touched = torch.zeros(c.pages, dtype=torch.bool)
        for s, (b, path) in enumerate(zip(before, paths)):
            moved = next((i for i, a in enumerate(path) if a != i), None)
            blocks = -(-(b + sizes[s]) // page)
            for side, (pool, scale) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
                for h in range(heads):
                    pages = [int(c.table[s, x]) for x in range(blocks)]
                    codes, scales = [c.codes[side][p, h] for p in pages], [float(c.scales[side][p, h]) for p in pages]
                    _, want_s, rows = drafts.keep(path, b, page, codes, scales, dtype)
                    for value, block, slot, far in rows:
                        got_s = float(scale[pages[block], h])
                        assert abs(got_s - want_s[block]) <= 2.0 ** -21 * want_s[block]
                        got = pool[pages[block], h, slot].float().double().cpu() * got_s
                        if not far and got_s == scales[block]:
                            assert torch.equal(got, value)
                        # half a step; value and quotient are off by 2^-22 of themselves
                        half = 0.5 * got_s if dtype == "int8" else torch.maximum(2.0 ** -4 * value.abs(), torch.as_tensor(2.0 ** -10 * got_s))
                        assert bool(((got - value).abs() <= half * (1 + 2.0 ** -9)).all())
                    for block in range(blocks):          # what lay there in front of the step
                        o = max(0, min(b - block * page, page))
                        got_s = float(scale[pages[block], h])
                        got, here = pool[pages[block], h, :o].float().double().cpu() * got_s, codes[block][:o] * scales[block]
                        if got_s == scales[block]:
                            assert torch.equal(got, here)
                        else:
                            assert bool(((got - here).abs() <= (0.5 if dtype == "int8" else 2.0 ** -10) * got_s * (1 + 1e-6)).all())
            if moved is not None:
                touched[[int(c.table[s, x]) for x in range((b + moved) // page, (b + len(path) - 1) // page + 1)]] = True
        for a, b in zip((cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale), old):
            x, y = a.cpu()[~touched], b.cpu()[~touched]
            assert torch.equal(x.nan_to_num(-1.0) if x.is_floating_point() else x, y.nan_to_num(-1.0) if y.is_floating_point() else y)


def test_kept_rows_of_one_scale_keep_their_codes():
    """Pages of one scale, the largest codes among the rows that change pages: nothing is rounded."""
    cache = PagedKVCache(4, 2, 64, 16, "int8")
    cache.k.random_(-127, 128), cache.v.random_(-127, 128), cache.k_scale.fill_(0.1), cache.v_scale.fill_(3.0)
    cache.k[:, :, :, 0] = 127
    k, v = cache.k.clone(), cache.v.clone()
    cache.keep(batch_of(torch.arange(4)[None], [3], [50]), i32([0, 20, 21, 40] + [0] * 46), i32([4]))
    assert cache.error_flags() == 0 and bool((cache.k_scale == cache.k_scale[0, 0]).all())
    for x, y in ((cache.k, k), (cache.v, v)):
        for i, a in enumerate((0, 20, 21, 40)):
            assert torch.equal(x[0, :, 3 + i], y[(3 + a) // 16, :, (3 + a) % 16])
        assert torch.equal(x[1:], y[1:]) and torch.equal(x[0, :, :3], y[0, :, :3])


def test_lists_that_do_not_rise_leave_their_sequence_out():
    c = Content([20, 20, 20], 2, 64, 16, "int8")
    for bad, n in (([2, 1, 3], 3), ([1, 1], 2), ([-1, 2], 2), ([1, 10], 2), ([2 ** 31 - 1], 1), ([0, 1], 11), ([0, 1], -1), ([0, 1], 2 ** 31 - 1)):
        cache = c.cache()
        k = cache.k.clone()
        cache.keep(batch_of(c.table, [10] * 3, [10] * 3), i32(bad + [0] * (10 - len(bad)) + [3, 5] + [0] * 8 + [0] * 10), i32([n, 2, 0]))
        assert cache.error_flags() == paged.BAD_BATCH
        used = [int(x) for x in c.table[0]] + [int(x) for x in c.table[2]]
        assert torch.equal(cache.k[used], k[used]) and not torch.equal(cache.k, k)


def test_pages_that_are_not_there_are_left_out():
    c = Content([40], 2, 64, 16, "int8")
    for block in (1, 2):                                 # where rows go, and where they come from
        cache = c.cache()
        table, k = c.table.clone(), cache.k.clone()
        table[0, block] = 10 ** 6
        cache.keep(batch_of(table, [14], [26]), i32([0, 5, 20] + [0] * 23), i32([3]))
        assert cache.error_flags() == paged.BAD_PAGE
        assert torch.equal(cache.k[int(c.table[0, 0]), :, 14], k[int(c.table[0, 0]), :, 14])
        assert torch.equal(cache.k[int(c.table[0, 2])], k[int(c.table[0, 2])])


def test_more_caches_than_a_launch_takes():
    caches = [PagedKVCache(2, 1, 64, 16, "int8") for _ in range(70)]
    for i, c in enumerate(caches):
        c.k.fill_(i), c.v.fill_(-i), c.k_scale.fill_(1.0), c.v_scale.fill_(1.0)
        c.k[1, 0, 7], c.v[1, 0, 7] = 100 - i, i - 100
    pool = PagePool(caches, 2, 2)
    batch = batch_of([[1, 0]], [2], [14])
    pool.keep(batch, i32([5] + [0] * 13), i32([1]))
    assert all(bool((c.k[1, 0, 2] == 100 - i).all()) and bool((c.v[1, 0, 2] == i - 100).all()) for i, c in enumerate(caches))
    pool.table[0, 0], pool.lengths[0], pool.held[0], pool.refs[1] = 1, 3, 1, 1
    pool.rearrange(i32([0, 0]))
    pool.reserve(i32([1, 0]))
    assert pool.table[:, 0].tolist() == [0, 1] and all(torch.equal(c.k[0], c.k[1]) for c in caches)


@pytest.mark.parametrize("seed", range(3))
def test_captured_keeps_follow_their_tensors(seed):
    """Two caches' keeps in graphs that are replayed side by side, with other paths each time."""
    graphs, cases = [], []
    for i in range(2):
        c = Content([70, 25, 90], 2, 64, 32, "int8", seed=seed + i)
        cache, kept, counts = c.cache(), i32([0] * 90), i32([0] * 3)
        batch = batch_of(c.table, [30, 5, 60], [40, 20, 30])
        cache.keep(batch, kept, counts)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.keep(batch, kept, counts)
        graphs.append(graph), cases.append((c, cache, kept, counts, batch, torch.cuda.Stream()))
    r = random.Random(seed)
    for _ in range(4):
        alone = []
        for c, cache, kept, counts, batch, _ in cases:
            paths = [sorted(r.sample(range(n), r.randint(0, n))) for n in (40, 20, 30)]
            kept.copy_(i32([x for p, n in zip(paths, (40, 20, 30)) for x in p + [0] * (n - len(p))])), counts.copy_(i32([len(p) for p in paths]))
            other = PagedKVCache(c.pages, 2, 64, 32, "int8")
            for a, b in ((other.k, cache.k), (other.v, cache.v), (other.k_scale, cache.k_scale), (other.v_scale, cache.v_scale)):
                a.copy_(b)
            other.keep(batch, kept, counts)
            alone.append(other)
        torch.cuda.synchronize()
        for graph, case in zip(graphs, cases):
            with torch.cuda.stream(case[-1]):
                graph.replay()
        torch.cuda.synchronize()
        for other, (_, cache, *_) in zip(alone, cases):
            assert all(torch.equal(getattr(other, n).nan_to_num(-1) if "scale" in n else getattr(other, n), getattr(cache, n).nan_to_num(-1) if "scale" in n else getattr(cache, n)) for n in ("k", "v", "k_scale", "v_scale"))
            assert cache.error_flags() == 0


# ---- refusals ----
def test_tensors_that_do_not_fit_are_refused():
    cache = PagedKVCache(8, 2, 64, 16, "int8")
    batch = batch_of(torch.arange(8)[None], [3], [5])
    parents, x = i32([-1, 0, 1, 0, 2]), torch.zeros(5, 2, 64, dtype=torch.bfloat16, device="cuda")
    tree = PagedTree(batch, parents)
    for bad in (parents.long(), parents[:4], parents.cpu(), parents.repeat_interleave(2)[::2], parents[None]):
        with pytest.raises(ValueError):
            PagedTree(batch, bad)
    with pytest.raises(ValueError, match="1024"):
        PagedTree(batch_of(torch.arange(8)[None], [3], [1025]), torch.zeros(1025, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="another batch"):
        cache.attend(batch_of(torch.arange(8)[None], [3], [5]), x, tree=tree)
    rotary, two = RotaryTable(64), RotaryTable(64, axes=[0, 1] * 16)
    for table, at in ((two, None), (two, tree.positions), (None, tree.positions), (rotary, tree.positions.long()), (rotary, tree.positions[:4]), (two, torch.zeros(5, 2, dtype=torch.int32, device="cuda").t()),
                      (rotary, tree.positions.cpu()), (rotary, torch.zeros(2, 5, dtype=torch.int32, device="cuda")), (two, torch.zeros(1, 5, dtype=torch.int32, device="cuda").expand(2, -1))):
        with pytest.raises(ValueError):
            cache.append(batch, x, x, rotary=table, positions=at)
    for axes in ([0] * 31, [0] * 31 + [4], [-1] + [0] * 31):
        with pytest.raises(ValueError):
            RotaryTable(64, axes=axes)
    for kept, counts in ((parents[:4], i32([1])), (parents, i32([1, 1])), (parents.long(), i32([1])), (parents.cpu(), i32([1]))):
        with pytest.raises(ValueError):
            cache.keep(batch, kept, counts)
    with pytest.raises(ValueError):
        cache.attend(batch, x.float(), tree=tree)
    with pytest.raises(ValueError, match="gradient"):
        cache.attend(batch, x.clone().requires_grad_(), tree=tree)
    for caches in ([], [cache, PagedKVCache(9, 2, 64, 16, "int8")], [cache, PagedKVCache(8, 2, 64, 16, "fp8_e4m3")], [cache, PagedKVCache(8, 1, 64, 16, "int8")]):
        with pytest.raises(ValueError):
            PagePool(caches, 2, 2)
    for n, w in ((0, 1), (4097, 1), (1, 0)):
        with pytest.raises(ValueError):
            PagePool([cache], n, w)
    pool = PagePool([cache], 3, 2)
    for bad in (i32([0, 1]), i32([0, 1, 2]).long(), torch.zeros(3, dtype=torch.int32), i32([0, 0, 1, 1, 2, 2])[::2]):
        for call in (pool.rearrange, pool.reserve):
            with pytest.raises(ValueError):
                call(bad)


def test_steps_without_rows():
    cache = PagedKVCache(8, 2, 64, 16, "int8")
    batch = batch_of(torch.arange(8)[None], [3], [0])
    tree = PagedTree(batch, torch.zeros(0, dtype=torch.int32, device="cuda"))
    x = torch.zeros(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    assert cache.append(batch, x, x, q=x, rotary=RotaryTable(64), positions=tree.positions).shape == x.shape
    assert cache.attend(batch, x, tree=tree).shape == x.shape
    cache.keep(batch, tree.parents, i32([0]))
    assert cache.error_flags() == 0 and tree.error_flags() == 0


# ---- all of it in turn ----
@pytest.mark.parametrize("dtype,dim,page,window,sinks", [("int8", 128, 32, 0, 0), ("fp8_e4m3", 64, 16, 40, 3), ("int8", 64, 64, 0, 0)])
def test_drafting_step_by_step(dtype, dim, page, window, sinks):
    """Prompts, then steps of drafted trees whose accepted path is kept, with pages from a pool; every attention is held against what the cache has, and the cache in the end against the tokens that were kept."""
    layers, S, hq, hkv, steps = 2, 3, 8, 2, 8
    caches = [PagedKVCache(60, hkv, dim, page, dtype) for _ in range(layers)]
    pool, rotary, r = PagePool(caches, S, 20), RotaryTable(dim), random.Random(dim + page)
    g = torch.Generator().manual_seed(1)
    truth = [[[torch.zeros(0, hkv, dim, dtype=torch.float64) for _ in range(2)] for _ in range(S)] for _ in range(layers)]
    for step in range(steps):
        sizes = [r.randint(10, 60) for _ in range(S)] if step == 0 else [r.randint(1, 24) for _ in range(S)]
        trees = [some_tree(n, step, "chain" if step == 0 else "mixed") for n in sizes]
        paths = []
        for t in trees:
            path = drafts.lines(t)[r.randrange(len(t))] if step else list(range(len(t)))
            paths.append(path)
        before = pool.lengths.tolist()
        pool.reserve(i32(sizes))
        rows, T = [0], sum(sizes)
        for n in sizes:
            rows.append(rows[-1] + n)
        batch = PagedBatch(pool.table, pool.lengths, i32(rows), T, max(sizes))
        tree = PagedTree(batch, i32([x for t in trees for x in t]))
        for layer, cache in enumerate(caches):
            q, k, v = (torch.randn(T, h, dim, generator=g).bfloat16().cuda() for h in (hq, hkv, hkv))
            turned = cache.append(batch, k, v, q=q, rotary=rotary, positions=tree.positions)
            out = cache.attend(batch, turned, window=window, sinks=sinks, tree=tree)
            for s, t in enumerate(trees):
                at, n = rows[s], before[s] + sizes[s]
                pages = pool.table[s, :-(-n // page)].long().cpu()
                kv = [(p.float().double().cpu()[pages] * sc.double().cpu()[pages][..., None, None]).transpose(1, 2).reshape(-1, hkv, dim)[:n] for p, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]
                top = (cache.v_scale.double().cpu()[pages] * oracle.Q_MAX[dtype])[:, None].expand(-1, page, -1).reshape(-1, hkv)[:n]
                want, tol = drafts.attend(turned[at:at + sizes[s]].double().cpu(), *kv, top, drafts.visible(t, before[s], window, sinks), dim ** -0.5)
                assert bool(((out[at:at + sizes[s]].double().cpu() - want).abs() <= tol).all()), (step, layer, s)
                pos = torch.tensor([before[s] + d for d in drafts.depths(t)])[None]
                new = (drafts.rotated(k[at:at + sizes[s]].double().cpu(), pos, [0] * (dim // 2), dim), v[at:at + sizes[s]].double().cpu())
                truth[layer][s] = [torch.cat((a, b[paths[s]])) for a, b in zip(truth[layer][s], new)]
        kept = [x for p, n in zip(paths, sizes) for x in p + [0] * (n - len(p))]
        counts = i32([len(p) for p in paths])
        pool.keep(batch, i32(kept), counts)
        pool.lengths += counts
        assert all(c.error_flags() == 0 for c in caches) and pool.error_flags() == 0 and tree.error_flags() == 0
    for layer, cache in enumerate(caches):
        for s in range(S):
            n = int(pool.lengths[s])
            pages = pool.table[s, :-(-n // page)].long().cpu()
            for side, (p, sc) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
                step_of = sc.double().cpu()[pages][:, None].expand(-1, page, -1).reshape(-1, hkv)[:n, :, None]
                got = (p.float().double().cpu()[pages] * sc.double().cpu()[pages][..., None, None]).transpose(1, 2).reshape(-1, hkv, dim)[:n]
                want = truth[layer][s][side]
                # a step from appending (half, and halves of it for each doubling) and half a step from the one move; e4m3: half steps of the value, twice, and of the subnormals
                tol = 1.5 * step_of if dtype == "int8" else 2 * 2.0 ** -4 * want.abs() * (1 + 2.0 ** -4) + 3 * 2.0 ** -10 * step_of
                assert want.shape == got.shape and bool(((got - want).abs() <= tol * (1 + 2.0 ** -9)).all())


# ---- pages that are missing ----
@pytest.mark.parametrize("dim,page", [(128, 64), (128, 128), (64, 64), (64, 128)])
@pytest.mark.parametrize("size", [1, 5, 10, 25])
def test_tiles_without_a_page_count_for_nothing(size, dim, page):
    """4, 20, 40 and 100 columns over tables that lack whole tiles: the first ones, single ones and runs of them, at the beginnings of cut units too.  What lay in shared memory, here bytes that are NaN in e4m3, must not be taken for their values."""
    r = random.Random(size + dim + page)
    for lengths, heads in (([700, 9000], (4, 1)), ([300, 0, 2000, 1100], (16, 4))):
        trees = [some_tree(size, 10 + s) for s in range(len(lengths))]
        c = Content([n + size for n in lengths], heads[1], dim, page, "fp8_e4m3", seed=size)
        q = torch.randn(size * len(lengths), heads[0], dim, generator=torch.Generator().manual_seed(size)).bfloat16().cuda()
        parents, batch = i32([x for t in trees for x in t]), batch_of(c.table, lengths, [size] * len(lengths))
        tree = PagedTree(batch, parents)
        odd = PagedKVCache(c.pages, heads[1], dim, page, "int8")
        odd.k.fill_(127), odd.v.fill_(-1), odd.k_scale.fill_(0.01), odd.v_scale.fill_(1.0)
        cache, table, seen = c.cache(), c.table.clone(), []
        for s, n in enumerate(lengths):
            missing = {b for b in range((n + size) // page) if b in (0, 8, 9) or b % 16 == 15 or r.random() < 0.15} - {(n + size - 1) // page}
            mask = drafts.visible(trees[s], n)
            for b in missing:
                table[s, b] = -1
                mask[:, b * page:(b + 1) * page] = False
            seen.append(mask)
        for _ in range(3):
            odd.attend(batch, q, tree=tree)
            batch.table.copy_(table)
            out = cache.attend(batch, q, tree=tree).double().cpu()
            batch.table.copy_(c.table)
            for s in range(len(lengths)):
                want, tol = drafts.attend(q[size * s:size * (s + 1)].double().cpu(), *c.kvt(s), seen[s], dim ** -0.5)
                assert bool(((out[size * s:size * (s + 1)] - want).abs() <= tol).all()), (lengths, s)
        assert cache.error_flags() == paged.BAD_PAGE and odd.error_flags() == 0


# ---- columns that end inside a warp ----
@pytest.mark.parametrize("dim,page", [(128, 64), (64, 32)])
@pytest.mark.parametrize("size", [17, 31, 33, 47, 65, 95, 97, 100, 127, 129, 161, 193])
def test_units_whose_last_warp_is_partly_filled(size, dim, page):
    """One head: as many columns as rows.  Units that a CTA has whole, cut ones, and the same again with another sequence's columns beside them."""
    check([100, 30], [some_tree(size, 1), some_tree(size - 9, 2)], (1, 1), ("int8", dim, page))
    first = check([7000], [some_tree(size, 3)], (1, 1), ("fp8_e4m3", dim, page))
    assert all(torch.equal(first, check([7000], [some_tree(size, 3)], (1, 1), ("fp8_e4m3", dim, page))) for _ in range(3))
    check([700, 50, 3000], [some_tree(size, 4), some_tree(1, 5), some_tree(size // 2, 6)], (3, 3), ("int8", dim, page), window=500, sinks=5)
