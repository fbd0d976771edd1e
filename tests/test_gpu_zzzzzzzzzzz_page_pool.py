"""Pages of a pool on the GPU against lists (oracle/drafts.py): forks, beams, copies before a shared page is written, moves to the front."""
import random

import pytest
import torch

from moshi_b200.models import PagedBatch, PagedKVCache, PagePool
from moshi_b200.models import paged
from oracle import drafts

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32).cuda()


class Both:
    """A pool and what it should be; the caches' content is theirs page by page."""

    def __init__(self, pages, page, sequences, width, dtype="int8", layers=2, heads=3, dim=64):
        g = torch.Generator(device="cuda").manual_seed(1)
        self.caches = [PagedKVCache(pages, heads, dim, page, dtype) for _ in range(layers)]
        for c in self.caches:
            for x in (c.k, c.v):
                x.view(torch.int8).copy_(torch.randint(-100, 100, x.shape, generator=g, device="cuda", dtype=torch.int8))
            for x in (c.k_scale, c.v_scale):
                x.copy_(torch.rand(x.shape, generator=g, device="cuda") + 0.5)
        self.tensors = [t for c in self.caches for t in (c.k.view(torch.int8), c.v.view(torch.int8), c.k_scale, c.v_scale)]
        self.pool, self.want, self.content = PagePool(self.caches, sequences, width), drafts.Pool(pages, page, sequences, width), [t.clone() for t in self.tensors]

    def moved(self, moves):
        for t in self.content:
            for a, b in moves:
                t[b] = t[a]

    def rearrange(self, source):
        self.pool.rearrange(i32(source))
        self.want.rearrange(source)

    def reserve(self, add, grow=True):
        self.pool.reserve(i32(add))
        moves = self.want.reserve(add)
        if moves is not None:
            self.moved(moves)
            if grow:
                for s, a in enumerate(add):
                    if a > 0 and self.want.lengths[s] + a <= self.want.width * self.want.page_tokens:
                        self.want.lengths[s] += a
                self.pool.lengths.copy_(i32(self.want.lengths))
        return moves

    def compact(self):
        self.pool.compact()
        self.moved(self.want.compact())

    def check(self, flags=0):
        w, p = self.want, self.pool
        assert p.error_flags() == flags
        p.clear_error_flags()
        assert p.lengths.tolist() == w.lengths and p.held.tolist() == [len(t) for t in w.table] and p.refs.tolist() == w.refs
        assert p.table.tolist() == [t + [-1] * (w.width - len(t)) for t in w.table]
        assert all(torch.equal(a, b) for a, b in zip(self.tensors, self.content))


@pytest.mark.parametrize("page,dtype", [(16, "int8"), (64, "fp8_e4m3"), (128, "int8")])
@pytest.mark.parametrize("seed", range(4))
def test_any_calls_in_any_order(page, dtype, seed):
    r = random.Random(seed)
    b = Both(90, page, 9, 12, dtype)
    for _ in range(60):
        kind = r.randrange(4)
        if kind == 0:
            b.rearrange([r.choice([-1, i, i, i, r.randrange(9)]) for i in range(9)])
        elif kind < 3:
            if b.reserve([r.choice([0, 0, 1, 5, page, 3 * page + 1]) for _ in range(9)]) is None:
                b.check(paged.NO_PAGES)
                b.rearrange([i if r.random() < 0.5 else -1 for i in range(9)])
        else:
            b.compact()
        flags = b.pool.error_flags()
        if flags == paged.BAD_BATCH:                     # a sequence asked for more than its table holds: it was left out
            b.check(paged.BAD_BATCH)
        b.check()


def test_one_into_many_and_beams():
    b = Both(64, 16, 8, 6)
    b.reserve([37] + [0] * 7)
    b.rearrange([0] * 8)
    b.check()
    assert b.pool.refs.max() == 8
    b.reserve([1] * 8)                                   # seven copies of the third page
    b.check()
    for source in ([1, 1, 2, 2, 3, 3, 0, 0], [7, 6, 5, 4, 3, 2, 1, 0], [4] * 8):
        b.rearrange(source)
        b.reserve([1] * 8)
        b.check()
    b.rearrange([-1] * 8)
    b.check()
    assert bool((b.pool.refs == 0).all()) and bool((b.pool.table == -1).all())


def test_a_full_page_is_shared_for_good():
    b = Both(32, 16, 4, 6)
    b.reserve([32, 0, 0, 0])
    b.rearrange([0, 0, 0, 0])
    assert b.reserve([5, 5, 0, 0]) == []                 # they go on in pages of their own
    b.check()


def test_the_last_sharer_keeps_the_page_unless_another_sequence_holds_it():
    b = Both(32, 16, 4, 6)
    b.reserve([20, 0, 0, 0])
    b.rearrange([0, 0, 0, 0])
    page = int(b.pool.table[0, 1])
    assert len(b.reserve([0, 1, 1, 0])) == 2 and int(b.pool.table[0, 1]) == int(b.pool.table[3, 1]) == page
    b.check()
    assert len(b.reserve([1, 0, 0, 1])) == 1 and int(b.pool.table[3, 1]) == page
    b.check()


def test_pages_held_in_reserve_are_given_back():
    b = Both(32, 16, 3, 8)
    b.reserve([50, 10, 0], grow=False)
    b.pool.lengths.copy_(i32([3, 10, 0]))
    b.want.lengths = [3, 10, 0]
    b.rearrange([0, 1, 0])
    b.check()
    assert b.pool.held.tolist() == [1, 1, 1]


def test_too_few_pages_change_nothing():
    b = Both(5, 16, 3, 5)
    b.reserve([30, 0, 0])
    b.rearrange([0, 0, -1])
    assert b.reserve([1, 1, 64]) is None
    b.check(paged.NO_PAGES)
    assert b.reserve([1, 1, 32]) is not None             # exactly as many as there are
    b.check()
    assert b.reserve([0, 0, 17]) is None
    b.check(paged.NO_PAGES)


def test_compacting_a_compact_pool_moves_nothing():
    b = Both(40, 16, 4, 8)
    b.reserve([100, 50, 0, 3])
    b.compact()
    b.check()
    b.rearrange([-1, 1, 2, 1])
    b.compact()
    b.check()
    assert sorted({p for t in b.want.table for p in t}) == list(range(4))


def test_what_does_not_fit_is_left_out_and_recorded():
    b = Both(40, 16, 4, 4)
    b.reserve([10, 20, 30, 40])
    before = b.pool.table.clone()
    b.pool.rearrange(i32([7, -9, 2 ** 31 - 1, -2 ** 31]))     # no sequences: all stay what they are
    assert torch.equal(b.pool.table, before) and b.pool.error_flags() == paged.BAD_BATCH
    b.pool.clear_error_flags()
    b.check()
    b.pool.reserve(i32([-1, 60, 2 ** 31 - 1, 1]))             # less than none, more than a table holds
    assert b.pool.error_flags() == paged.BAD_BATCH
    b.pool.clear_error_flags()
    b.want.reserve([0, 0, 0, 1])
    b.check()
    for lengths, held in (([-1, 20, 30, 40], None), ([1000, 20, 30, 40], None), (None, [-5, 2, 2, 3]), (None, [5, 2, 2, 3]), (None, [0, 2, 2, 3])):
        keep = [b.pool.lengths.clone(), b.pool.held.clone(), b.pool.table.clone(), b.pool.refs.clone()]
        if lengths:
            b.pool.lengths.copy_(i32(lengths))
        if held:
            b.pool.held.copy_(i32(held))
        b.pool.reserve(i32([1, 0, 0, 0]))
        assert b.pool.error_flags() & paged.BAD_BATCH and torch.equal(b.pool.table, keep[2]) and torch.equal(b.pool.refs, keep[3])
        b.pool.clear_error_flags()
        b.pool.rearrange(i32([0, 1, 2, 3]))
        assert b.pool.error_flags() & paged.BAD_BATCH and torch.equal(b.pool.table[1:], keep[2][1:]) and b.pool.held[0] == 0
        b.pool.clear_error_flags()
        for t, x in zip((b.pool.lengths, b.pool.held, b.pool.table, b.pool.refs), keep):
            t.copy_(x)
    for bad in (-1, 40, 2 ** 31 - 1):
        keep = [b.pool.table.clone(), b.pool.refs.clone()]
        b.pool.table[3, 0] = bad
        b.pool.compact()
        assert b.pool.error_flags() == paged.BAD_PAGE
        b.pool.clear_error_flags()
        b.pool.rearrange(i32([0, 1, 2, 3]))
        assert b.pool.error_flags() == paged.BAD_PAGE
        b.pool.clear_error_flags()
        for t, x in zip((b.pool.table, b.pool.refs), keep):
            t.copy_(x)


def test_many_sequences_and_many_pages():
    r = random.Random(3)
    b = Both(30000, 16, 4096, 7, layers=1, heads=1)
    b.reserve([r.randint(0, 100) for _ in range(4096)])
    b.check()
    b.rearrange([r.choice([-1, i, i, r.randrange(4096), i & ~7]) for i in range(4096)])
    b.reserve([r.choice([0, 1]) if b.want.lengths[i] < 112 else 0 for i in range(4096)])
    b.check()
    b.compact()
    b.check()


def test_captured_calls_follow_their_tensors():
    b = Both(80, 16, 6, 8)
    source, add = i32(list(range(6))), i32([0] * 6)
    b.pool.rearrange(source)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.pool.rearrange(source)
        b.pool.compact()
        b.pool.reserve(add)
    r = random.Random(4)
    for _ in range(25):
        s, a = [r.choice([-1, i, i, r.randrange(6)]) for i in range(6)], [r.choice([0, 1, 20]) for _ in range(6)]
        b.want.rearrange(s)
        a = [x if b.want.lengths[i] + x <= 128 else 0 for i, x in enumerate(a)]
        source.copy_(i32(s)), add.copy_(i32(a))
        graph.replay()
        b.moved(b.want.compact())
        moves = b.want.reserve(a)
        b.moved(moves)
        b.want.lengths = [n + x for n, x in zip(b.want.lengths, a)]
        b.pool.lengths += add
        b.check()


def test_another_stream_than_the_default():
    b = Both(200, 16, 16, 10)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        r = random.Random(6)
        b.reserve([33] * 4 + [0] * 12)
        for _ in range(10):
            b.rearrange([r.randrange(4) * 4 % 16 if i else 0 for i in range(16)])
            b.reserve([1] * 16)
            b.compact()
    stream.synchronize()
    b.check()


def test_forked_requests_read_what_they_share_and_write_on_their_own():
    """A prompt that is sampled three times: each sample appends another token behind the same page."""
    cache = PagedKVCache(20, 2, 64, 16, "int8")
    pool, g = PagePool([cache], 3, 4), torch.Generator().manual_seed(2)
    x = torch.randn(21, 2, 64, generator=g).bfloat16().cuda()
    pool.reserve(i32([20, 0, 0]))
    cache.append(PagedBatch(pool.table, pool.lengths, i32([0, 20, 20, 20]), 20, 20), x[:20], x[:20])
    pool.lengths += i32([20, 0, 0])
    pool.rearrange(i32([0, 0, 0]))
    pool.reserve(i32([1, 1, 1]))
    new = torch.randn(3, 2, 64, generator=g).bfloat16().cuda()
    cache.append(PagedBatch(pool.table, pool.lengths, i32([0, 1, 2, 3]), 3, 1), new, new)
    k, _ = cache.read(PagedBatch(pool.table, i32([0, 0, 0]), i32([0, 21, 42, 63]), 63, 21))
    alone = PagedKVCache(4, 2, 64, 16, "int8")
    for s in range(3):
        batch = PagedBatch(i32([[0, 1]]), i32([0]), i32([0, 20]), 20, 20)
        alone.append(batch, x[:20], x[:20])
        alone.append(PagedBatch(i32([[0, 1]]), i32([20]), i32([0, 1]), 1, 1), new[s:s + 1], new[s:s + 1])
        want, _ = alone.read(PagedBatch(i32([[0, 1]]), i32([0]), i32([0, 21]), 21, 21))
        assert torch.equal(k[21 * s:21 * s + 21], want)
    assert pool.error_flags() == 0 and cache.error_flags() == 0


def test_a_cache_is_in_a_pool_once():
    cache = PagedKVCache(8, 2, 64, 16, "int8")
    with pytest.raises(ValueError, match="memory of their own"):
        PagePool([cache, PagedKVCache(8, 2, 64, 16, "int8"), cache], 2, 2)


@pytest.mark.parametrize("shorter", [3, 16, 20, 32])
def test_a_sequence_that_was_made_shorter(shorter):
    """What lies behind its tokens may be another's: it gets pages once it has been rearranged, and none before."""
    b = Both(32, 16, 3, 6)
    b.reserve([70, 5, 0])
    b.rearrange([0, 1, 0])
    for x in (b.want.lengths, b.pool.lengths):
        x[0] = shorter
    assert b.reserve([1, 3, 0], grow=False) == []
    b.check(paged.BAD_BATCH)
    b.rearrange([0, 1, 2])
    b.check()
    assert len(b.reserve([1, 3, 1])) == (shorter % 16 > 0)      # the third's last page is its own now
    b.check()


def test_a_pool_s_tensors_stay():
    """The library has their addresses: another tensor in their place is refused, and the calls go on with the ones that there are."""
    b = Both(32, 16, 3, 6)
    b.reserve([20, 5, 0], grow=False)
    for name in ("table", "lengths", "held", "refs", "flags"):
        with pytest.raises(AttributeError, match=name):
            setattr(b.pool, name, getattr(b.pool, name) + 0)
    b.pool.lengths += i32([20, 5, 0])
    b.want.lengths = [20, 5, 0]
    b.rearrange([0, 0, 1])
    b.reserve([1, 1, 30])
    b.check()


def test_caches_that_share_memory_are_read_only():
    """Two layers with one tensor of values, or of scales, or keys a page apart in one allocation; keys that are the values too."""
    def cache(k, v, k_scale, v_scale):
        return PagedKVCache.from_tensors(k, v, k_scale, v_scale)
    k, v = (torch.zeros(17, 2, 16, 64, dtype=torch.int8, device="cuda") for _ in range(2))
    scales = [torch.ones(8, 2, device="cuda") for _ in range(4)]
    others = [torch.zeros(8, 2, 16, 64, dtype=torch.int8, device="cuda") for _ in range(3)]
    first = cache(k[:8], v[:8], *scales[:2])
    for second in (cache(others[0], v[:8], *scales[2:]), cache(others[0], others[1], scales[0], scales[3]), cache(others[0], others[1], scales[2], scales[1]), cache(k[7:15], others[1], *scales[2:]),
                   cache(others[0], k[1:9], *scales[2:]), cache(others[0], others[0], *scales[2:])):
        with pytest.raises(ValueError, match="memory of their own"):
            PagePool([first, second], 2, 2)
    PagePool([first, cache(k[8:16], v[8:16], *scales[2:])], 2, 2)            # side by side in one allocation
    both = cache(others[0], others[0], *scales[2:])
    batch, x = PagedBatch(i32([[0, 1]]), i32([0]), i32([0, 3]), 3, 3), torch.zeros(3, 2, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: both.append(batch, x, x), lambda: both.keep(batch, i32([1, 2, 0]), i32([2]))):
        with pytest.raises(ValueError, match="over one another"):
            call()
    assert bool((both.attend(batch, x) == 0).all()) and both.error_flags() == 0


@pytest.mark.parametrize("sequences,width", [(6, 8), (1100, 8)])
@pytest.mark.parametrize("source", ["itself", "others", "nobody"])
@pytest.mark.parametrize("wrong", [-1, -2 ** 31, 33, 2 ** 31 - 1])
def test_a_length_that_the_pages_do_not_take_loses_no_pages(sequences, width, source, wrong):
    """By the kernel of small tables and by that of large ones: the sequence becomes empty and its pages are free again."""
    b = Both(40, 16, sequences, width)
    rest = [0] * (sequences - 4)
    b.reserve([20, 32, 0, 5] + rest)
    b.rearrange([0, 1, 1, 3] + [-1] * (sequences - 4))
    b.reserve([1, 0, 1, 0] + rest)                       # the third goes on behind two shared pages
    b.check()
    for x in (b.want.lengths, b.pool.lengths):
        x[1] = wrong
    b.rearrange({"itself": [0, 1, 2, 3], "others": [1, 1, 2, 1], "nobody": [0, -1, 2, 3]}[source] + [-1] * (sequences - 4))
    b.check(paged.BAD_BATCH)
    assert b.pool.refs.sum() == b.pool.held.sum() and b.pool.held[1] == 0
    b.rearrange([-1] * sequences)
    b.check()
    assert bool((b.pool.refs == 0).all())
    assert b.reserve([7 * 16, 8 * 16, 8 * 16, 8 * 16] + [16] * min(9, sequences - 4) + [0] * (sequences - 4 - min(9, sequences - 4))) is not None
    b.check()


def test_lengths_raised_without_pages():
    """A step that got none, and whose lengths were raised all the same: what the sequence held goes back, the others are as they were."""
    b = Both(6, 16, 3, 6)
    b.reserve([40, 16, 0])
    assert b.reserve([20, 20, 20], grow=False) is None
    for s, n in enumerate((60, 36, 0)):
        b.want.lengths[s] = n
    b.pool.lengths += i32([20, 20, 0])
    b.check(paged.NO_PAGES)
    b.rearrange([0, 1, 2])
    b.check(paged.BAD_BATCH)
    assert b.reserve([96, 0, 0]) is not None
    b.check()
