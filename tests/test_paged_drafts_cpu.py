"""Drafted trees, kept rows and page pools without a GPU: which kernels a call launches and what it refuses (on the fake CUDA runtime), the oracle's own properties."""
import ctypes as C
import math
import random
import types

import pytest
import torch

from moshi_b200 import _lib
from moshi_b200.models import paged
from oracle import drafts, paged as oracle

from . import fake_cuda


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return fake_cuda.load(tmp_path_factory.mktemp("fake"))


class Call:
    """Arguments of calls that are taken; any of them can be replaced."""

    def __init__(self, **changed):
        self.memory = C.create_string_buffer(1 << 12)
        at = (C.addressof(self.memory) + 63) // 64 * 64
        self.cache = dict(k=at, v=at, k_scale=at, v_scale=at, flags=at, pages=100, page_tokens=64, kv_heads=8, dim=128, kv_dtype=_lib.B200_KV_INT8, device=0)
        self.batch = dict(table=at, before=at, rows=at, table_ld=64, sequences=4, table_width=64, total_rows=100, max_rows=30)
        self.tree = dict(seen=at, position=at, words=1)
        self.pool = dict(p_table=at, lengths=at, held=at, refs=at, p_flags=at, p_ld=64, p_sequences=16, p_width=64, p_pages=100, p_page_tokens=64, p_device=0)
        self.rotary = dict(turns=at, rot_dims=128, pairing=0)
        self.at = dict(positions=at, positions_ld=100, pair_axis=at, axes=3)
        self.args = dict(parents=at, tree_flags=at, q=at, q_ld=32 * 128, out=at, out_ld=32 * 128, q_heads=32, scale=0.1, window=0, sinks=0, work=at, work_bytes=1 << 40, kept=at, counts=at, n_caches=2, source=at, add=at)
        self.null = set()
        for name, x in changed.items():
            for d in (self.cache, self.batch, self.tree, self.pool, self.rotary, self.at, self.args):
                if name in d:
                    d[name] = x
                    break
            else:
                assert name in ("no_cache", "no_batch", "no_tree", "no_pool", "no_rotary", "no_at", "odd_cache"), name
                self.null.add(name)
        n = max(self.args["n_caches"], 1)
        self.c = (_lib.PagedCacheC * n)(*(_lib.PagedCacheC(**{**self.cache, **({"pages": 99} if i and "odd_cache" in self.null else {})}) for i in range(n)))
        self.b, self.t = _lib.PagedBatchC(**self.batch), _lib.PagedTreeC(**self.tree)
        self.p = _lib.PagePoolC(*(self.pool[k] for k in ("p_table", "lengths", "held", "refs", "p_flags", "p_ld", "p_sequences", "p_width", "p_pages", "p_page_tokens", "p_device")))
        self.r, self.a = _lib.RotaryC(**self.rotary), _lib.PagedPositionsC(self.at["positions"], self.at["positions_ld"], self.at["pair_axis"], self.at["axes"])

    def ref(self, name, x):
        return None if name in self.null else C.byref(x)

    def build(self, lib):
        return lib.b200_paged_tree_build(self.ref("no_batch", self.b), self.ref("no_tree", self.t), self.args["parents"], self.args["tree_flags"], self.cache["device"], None)

    def bytes(self, lib):
        a = self.args
        return lib.b200_paged_tree_attention_bytes(self.ref("no_cache", self.c), self.ref("no_batch", self.b), a["q_heads"], a["window"], a["sinks"])

    def attend(self, lib):
        a = self.args
        return lib.b200_paged_tree_attention(self.ref("no_cache", self.c), self.ref("no_batch", self.b), self.ref("no_tree", self.t), a["q"], a["q_ld"], a["out"], a["out_ld"], a["q_heads"], a["scale"], a["window"],
                                             a["sinks"], a["work"], a["work_bytes"], None)

    def append(self, lib):
        a, row = self.args, self.cache["kv_heads"] * self.cache["dim"]
        return lib.b200_paged_append_at(self.ref("no_cache", self.c), self.ref("no_batch", self.b), a["q"], row, a["q"], row, a["q"], a["q_ld"], a["out"], a["out_ld"], a["q_heads"], self.ref("no_rotary", self.r),
                                        self.ref("no_at", self.a), None)

    def keep(self, lib):
        return lib.b200_paged_keep(self.ref("no_cache", self.c), self.args["n_caches"], self.ref("no_batch", self.b), self.args["kept"], self.args["counts"], None)

    def rearrange(self, lib):
        return lib.b200_page_pool_rearrange(self.ref("no_pool", self.p), self.args["source"], self.args["work"], self.args["work_bytes"], None)

    def reserve(self, lib):
        return lib.b200_page_pool_reserve(self.ref("no_pool", self.p), self.ref("no_cache", self.c), self.args["n_caches"], self.args["add"], self.args["work"], self.args["work_bytes"], None)

    def compact(self, lib):
        return lib.b200_page_pool_compact(self.ref("no_pool", self.p), self.ref("no_cache", self.c), self.args["n_caches"], self.args["work"], self.args["work_bytes"], None)


NAMES = ("tree_join", "tree_kernel", "tree_build", "few_rows", "join_kernel", "append_few", "append_many", "keep_kernel", "rearrange_small", "rearrange_count", "rearrange_take", "reserve_kernel", "compact_kernel", "renumber", "copy_kernel")


def kernels(fake, call, what):
    fake_cuda.launches(fake)
    fake_cuda.check(fake, getattr(call, what)(fake))
    return [(d, next(k for k in NAMES if k in name)) for d, name in fake_cuda.launches(fake)]


@pytest.mark.parametrize("changed,names", [
    (dict(), ["tree_kernel", "tree_join"]),
    (dict(max_rows=4, total_rows=16), ["few_rows", "join_kernel"]),                               # 16 columns
    (dict(max_rows=5, total_rows=16), ["tree_kernel", "tree_join"]),                              # 20
    (dict(max_rows=1, total_rows=1, sequences=1, table_width=6), ["few_rows"]),
    (dict(dim=64, q_heads=32, q_ld=2048, out_ld=2048, max_rows=8), ["few_rows", "join_kernel"]),  # 32 columns of 64
    (dict(dim=64, q_heads=32, q_ld=2048, out_ld=2048, max_rows=9), ["tree_kernel", "tree_join"]),
    (dict(max_rows=1024, words=32, total_rows=4096, window=100, sinks=3), ["tree_kernel", "tree_join"]),
    (dict(total_rows=0, q=None), []), (dict(max_rows=0, out=None), []),
], ids=str)
@pytest.mark.parametrize("kv_dtype", [_lib.B200_KV_INT8, _lib.B200_KV_FP8_E4M3])
def test_which_kernels_attend(fake, changed, names, kv_dtype):
    assert kernels(fake, Call(kv_dtype=kv_dtype, **changed), "attend") == [(0, n) for n in names]


def test_which_kernels_the_others_launch(fake):
    assert kernels(fake, Call(), "build") == [(0, "tree_build")] and kernels(fake, Call(total_rows=0), "build") == []
    assert kernels(fake, Call(), "append") == [(0, "append_many")] and kernels(fake, Call(max_rows=16), "append") == [(0, "append_few")]
    assert kernels(fake, Call(axes=1, pair_axis=None), "append") == [(0, "append_many")]
    assert kernels(fake, Call(), "keep") == [(0, "keep_kernel")] and kernels(fake, Call(n_caches=64), "keep") == [(0, "keep_kernel")] and kernels(fake, Call(n_caches=65), "keep") == 2 * [(0, "keep_kernel")]
    assert kernels(fake, Call(total_rows=0), "keep") == []
    assert kernels(fake, Call(), "rearrange") == [(0, "rearrange_small")] and kernels(fake, Call(p_sequences=1025, p_width=4), "rearrange") == [(0, "rearrange_count"), (0, "rearrange_take")]
    assert kernels(fake, Call(p_sequences=129), "rearrange") == [(0, "rearrange_count"), (0, "rearrange_take")]
    assert kernels(fake, Call(), "reserve") == [(0, "reserve_kernel"), (0, "copy_kernel")] and kernels(fake, Call(n_caches=130), "reserve") == [(0, "reserve_kernel")] + 3 * [(0, "copy_kernel")]
    assert kernels(fake, Call(n_caches=0, no_cache=1), "reserve") == [(0, "reserve_kernel")]
    assert kernels(fake, Call(), "compact") == [(0, "compact_kernel"), (0, "copy_kernel")]
    assert kernels(fake, Call(p_sequences=129), "compact") == [(0, "compact_kernel"), (0, "renumber"), (0, "copy_kernel")]


def test_every_page_size_and_head_size(fake):
    for page in (16, 32, 64, 128):
        for dim in (64, 128):
            more = dict(page_tokens=page, p_page_tokens=page, dim=dim, q_ld=32 * dim, out_ld=32 * dim, rot_dims=dim)
            for what in ("attend", "append", "keep", "reserve", "compact"):
                assert kernels(fake, Call(**more), what)


def test_calls_run_on_the_cache_s_device(fake):
    for what in ("attend", "append", "keep", "build", "rearrange", "reserve", "compact"):
        assert {d for d, _ in kernels(fake, Call(device=1, p_device=1), what)} == {1}


def test_workspaces(fake):
    for changed in (dict(), dict(max_rows=4), dict(max_rows=1000, words=32)):
        n = Call(**changed).bytes(fake)
        assert n > 0
        assert Call(work_bytes=n, **changed).attend(fake) == 0
        assert Call(work_bytes=n - 1, **changed).attend(fake) == _lib.B200_ERR_INVALID and b"workspace" in fake.b200_last_error()
        assert Call(work=None, **changed).attend(fake) == _lib.B200_ERR_INVALID
    assert Call(max_rows=1, total_rows=1, sequences=1, table_width=6).bytes(fake) == 0
    for changed in (dict(no_cache=1), dict(no_batch=1), dict(q_heads=0), dict(q_heads=12), dict(window=-1), dict(sequences=0), dict(total_rows=0), dict(max_rows=0)):
        assert Call(**changed).bytes(fake) == 0
    n = fake.b200_page_pool_bytes(C.byref(Call().p))
    assert n > 0 and fake.b200_page_pool_bytes(None) == 0
    for what in ("rearrange", "reserve", "compact"):
        assert getattr(Call(work_bytes=n), what)(fake) == 0
        assert getattr(Call(work_bytes=n - 1), what)(fake) == _lib.B200_ERR_INVALID
        assert getattr(Call(work=None), what)(fake) == _lib.B200_ERR_INVALID
        assert getattr(Call(work=Call().args["work"] + 4), what)(fake) == _lib.B200_ERR_INVALID


BATCH = [dict(no_batch=1), *({n: None} for n in ("table", "before", "rows")), dict(sequences=0), dict(sequences=1 << 20), dict(total_rows=-1), dict(max_rows=-1), dict(table_width=0), dict(table_ld=63)]
CACHE = [dict(no_cache=1), *({n: None} for n in ("k", "v", "k_scale", "v_scale", "flags")), dict(kv_dtype=0), dict(dim=96), dict(page_tokens=48), dict(pages=0), dict(kv_heads=0)]


def refused(fake, call, what):
    fake_cuda.launches(fake)
    assert getattr(call, what)(fake) in (_lib.B200_ERR_INVALID, _lib.B200_ERR_SHAPE)
    assert fake_cuda.launches(fake) == [] and fake.b200_last_error()


@pytest.mark.parametrize("changed", BATCH + CACHE, ids=str)
def test_caches_and_batches_that_are_refused(fake, changed):
    for what in ("attend", "append", "keep"):
        refused(fake, Call(**changed), what)


@pytest.mark.parametrize("changed", [dict(no_tree=1), dict(seen=None), dict(position=None), dict(words=0), dict(words=33), dict(max_rows=33), dict(max_rows=1025, words=32), dict(max_rows=1025, words=33)], ids=str)
def test_trees_that_are_refused(fake, changed):
    refused(fake, Call(**changed), "attend")
    refused(fake, Call(**changed), "build")


@pytest.mark.parametrize("changed", [dict(parents=None), dict(tree_flags=None), dict(no_batch=1), dict(before=None), dict(rows=None), dict(sequences=0), dict(total_rows=-1), dict(max_rows=-1)], ids=str)
def test_builds_that_are_refused(fake, changed):
    refused(fake, Call(**changed), "build")


@pytest.mark.parametrize("changed", [dict(q=None), dict(out=None), dict(q_ld=4095), dict(out_ld=100), dict(q_heads=12), dict(q_heads=0), dict(q_heads=8 * 300), dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf),
                                     dict(window=-1), dict(sinks=-1)], ids=str)
def test_attention_calls_that_are_refused(fake, changed):
    refused(fake, Call(**changed), "attend")


@pytest.mark.parametrize("changed", [dict(no_at=1), dict(no_rotary=1), dict(positions=None), dict(axes=0), dict(axes=5), dict(pair_axis=None), dict(positions_ld=99), dict(turns=None), dict(rot_dims=24)], ids=str)
def test_positions_that_are_refused(fake, changed):
    refused(fake, Call(**changed), "append")
    refused(fake, Call(pair_axis=Call().at["pair_axis"] + 4), "append")


@pytest.mark.parametrize("changed", [dict(kept=None), dict(counts=None), dict(n_caches=0), dict(odd_cache=1)], ids=str)
def test_keeps_that_are_refused(fake, changed):
    refused(fake, Call(**changed), "keep")


@pytest.mark.parametrize("changed", [dict(no_pool=1), *({n: None} for n in ("p_table", "lengths", "held", "refs", "p_flags")), dict(p_sequences=0), dict(p_sequences=4097), dict(p_width=0), dict(p_ld=63), dict(p_pages=0),
                                     dict(p_page_tokens=20), dict(p_width=1 << 26, p_ld=1 << 26),
                                     dict(p_sequences=4096, p_width=1 << 19, p_ld=1 << 19, p_page_tokens=16)], ids=str)
def test_pools_that_are_refused(fake, changed):
    for what in ("rearrange", "reserve", "compact"):
        refused(fake, Call(**changed), what)


def test_pools_and_caches_that_do_not_fit_together(fake):
    for changed in (dict(p_pages=99), dict(p_page_tokens=32), dict(p_device=1), dict(odd_cache=1), dict(no_cache=1)):
        refused(fake, Call(**changed), "reserve")
        refused(fake, Call(**changed), "compact")
    refused(fake, Call(source=None), "rearrange")
    refused(fake, Call(add=None), "reserve")


# ---- attributes that the library has the addresses of ----
@pytest.mark.parametrize("kind,names", [(paged.RotaryTable, ("turns", "pair_axis")), (paged.PagedBatch, ("table", "before", "rows")), (paged.PagedTree, ("seen", "positions", "flags")),
                                        (paged.PagedKVCache, ("k", "v", "k_scale", "v_scale", "flags")), (paged.PagePool, ("table", "lengths", "held", "refs", "flags"))])
def test_tensors_are_written_into_and_not_replaced(kind, names):
    x = kind.__new__(kind)
    for name in names:
        t = torch.zeros(4, dtype=torch.int32)
        setattr(x, name, t)
        with pytest.raises(AttributeError, match=f"{name} stays"):
            setattr(x, name, t + 1)
        with pytest.raises(AttributeError, match=f"{name} stays"):
            setattr(x, name, t[:])
        setattr(x, name, t)
        assert getattr(x, name) is t
    x.other = 1
    x.other = 2


def test_lengths_are_raised_in_place():
    pool = paged.PagePool.__new__(paged.PagePool)
    pool.lengths = torch.zeros(3, dtype=torch.int32)
    at = pool.lengths.data_ptr()
    pool.lengths += torch.tensor([1, 2, 3], dtype=torch.int32)
    assert pool.lengths.tolist() == [1, 2, 3] and pool.lengths.data_ptr() == at
    with pytest.raises(AttributeError, match="PagePool.lengths stays"):
        pool.lengths = pool.lengths + 1
    assert pool.lengths.tolist() == [1, 2, 3]


def test_a_tree_s_parents_may_be_others_of_its_rows():
    tree = paged.PagedTree.__new__(paged.PagedTree)
    tree.batch = types.SimpleNamespace(total_rows=3, device=torch.device("cpu"))
    for good in (torch.zeros(3, dtype=torch.int32), torch.zeros(9, dtype=torch.int32)[3:6]):
        tree.parents = good
        assert tree.parents is good
    for bad in (torch.zeros(3), torch.zeros(4, dtype=torch.int32), torch.zeros(6, dtype=torch.int32)[::2], torch.zeros(3, 1, dtype=torch.int32), torch.zeros(3, dtype=torch.int32, device="meta")):
        with pytest.raises(ValueError, match="parents"):
            tree.parents = bad
    assert tree.parents is good
    with pytest.raises(AttributeError):
        tree.batch = types.SimpleNamespace(total_rows=9, device=torch.device("cpu"))


def test_memory_that_lies_over_itself_is_found():
    a, b, c = torch.zeros(100, dtype=torch.int8), torch.zeros(64), torch.zeros(10, dtype=torch.float64)
    assert paged._apart([a, b, c]) and paged._apart([a[:50], a[50:], b[10:20], b[:10], b[20:]]) and paged._apart([]) and paged._apart([b])
    for over in ([a, b, a], [a, c, a[99:]], [a[:51], b, a[50:]], [b[:11], b[10:].view(torch.int32)], [c, c[3:4], b]):
        assert not paged._apart(over)


# ---- the oracle's own properties ----
def test_lines_and_depths():
    parents = [-1, 0, 0, 2, -1, 4, 3, 9, -5]
    assert drafts.lines(parents) == [[0], [0, 1], [0, 2], [0, 2, 3], [4], [4, 5], [0, 2, 3, 6], [7], [8]]
    assert drafts.depths(parents) == [0, 1, 1, 2, 0, 1, 3, 0, 0]


def test_a_chain_sees_what_a_step_s_rows_see():
    for window, sinks in ((0, 0), (3, 0), (5, 2)):
        assert torch.equal(drafts.visible([-1, 0, 1, 2, 3], 7, window, sinks), oracle.visible(torch.arange(7, 12), 12, window, sinks))


def test_one_axis_is_the_usual_rotation():
    x = torch.randn(5, 2, 64, dtype=torch.float64)
    for pairing in ("adjacent", "halves"):
        assert torch.allclose(drafts.rotated(x, torch.arange(9, 14)[None], [0] * 16, 32, pairing=pairing), oracle.rotated(x, 9, 32, pairing=pairing), atol=1e-13)


@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
def test_kept_rows_stay_within_half_a_step_of_where_they_go(dtype):
    g, page = torch.Generator().manual_seed(0), 16
    for seed in range(20):
        r = random.Random(seed)
        before, n = r.randint(0, 40), r.randint(1, 30)
        blocks = -(-(before + n) // page)
        scales = [2.0 ** r.uniform(-4, 4) for _ in range(blocks)]
        codes = [oracle.nearest(torch.randn(page, 8, generator=g, dtype=torch.float64) * oracle.Q_MAX[dtype] / 3, dtype) for _ in range(blocks)]
        path = sorted(r.sample(range(n), r.randint(1, n)))
        after, now, rows = drafts.keep(path, before, page, codes, scales, dtype)
        assert len(rows) == len(path)
        for i, (value, block, slot, far) in enumerate(rows):
            assert block * page + slot == before + i
            off, s = (after[block][slot] * now[block] - value).abs(), now[block]
            half = 0.5 * s if dtype == "int8" else torch.maximum(2.0 ** -4 * value.abs(), torch.as_tensor(2.0 ** -10 * s))
            assert bool((off <= half * (1 + 1e-9)).all())
            if not far and now[block] == scales[block]:
                assert bool((off == 0).all())
        if path == list(range(n)):
            assert all(torch.equal(a, b) for a, b in zip(codes, after)) and now == scales


def test_equal_scales_never_double():
    """Rows that move between pages of one scale keep their codes, the largest code among them."""
    for dtype, top in (("int8", 127.0), ("fp8_e4m3", 448.0)):
        codes = [torch.full((16, 4), top, dtype=torch.float64) for _ in range(2)]
        after, now, _ = drafts.keep([0, 14], 2, 16, codes, [0.1, 0.1], dtype)
        assert now == [0.1, 0.1] and all(torch.equal(a, b) for a, b in zip(codes, after))


def test_pools_account_for_every_page():
    r = random.Random(1)
    pool = drafts.Pool(60, 16, 8, 10)
    for step in range(300):
        before = ([list(t) for t in pool.table], list(pool.refs))
        kind = r.randrange(4)
        if kind == 0:
            pool.rearrange([r.choice([-1, i, i, r.randrange(8)]) for i in range(8)])
        elif kind == 1:
            add = [r.choice([0, 1, 5, 40]) for _ in range(8)]
            moves = pool.reserve(add)
            if moves is None:
                assert (pool.table, pool.refs) == before
            else:
                pool.lengths = [min(n + a, 160) if n + a <= 160 else n for n, a in zip(pool.lengths, add)]
        elif kind == 2:
            pool.compact()
            assert all(x > 0 for x in pool.refs[:sum(x > 0 for x in pool.refs)])
        held = [p for t in pool.table for p in t]
        assert [held.count(p) for p in range(60)] == pool.refs and all(len(t) >= -(-n // 16) for t, n in zip(pool.table, pool.lengths))
