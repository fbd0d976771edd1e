"""Rare calls of the paged 8-bit cache on the GPU, against 64-bit restatements (oracle/paged.py)."""
import pytest
import torch

from moshi_b200 import _lib
from moshi_b200.models import PagedBatch, PagedKVCache, RotaryTable, paged
from oracle import paged as oracle

from .paged_util import Content, batch_of

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32).cuda()


@pytest.mark.parametrize("rows", [[0, 5, 1, 2], [0, 2, 0, 0], [0, 0, 9, 3], [0, 14, 14, 3]], ids=str)
@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
def test_rows_that_no_sequence_has_are_left_out(rows, dtype):
    """Rows out of order, under which a row is counted to a sequence that does not have it.  Lengths end where the tables do, and the table is a slice of a larger one whose other entries name a page of
    its own: it is not read, and queries, keys and values of such rows stay as they are."""
    T, S, width, page, dim = 14, 3, 2, 16, 64
    cache = PagedKVCache(8, 2, dim, page, dtype)
    for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        pool.view(torch.int8)[:6], scale[:6] = 8, 1.0
        pool.view(torch.int8)[6], scale[6] = 64, 4.0     # int8: 256; e4m3: 8
    wide = torch.full((S + 4, width + 3), 6, dtype=torch.int32, device="cuda")
    wide[:S, :width] = torch.arange(S * width, device="cuda").view(S, width)
    before = [width * page - max(b - a, 0) for a, b in zip(rows, rows[1:])]
    before[2] = width * page - 1 if rows[3] - rows[2] == 1 else width * page
    batch = PagedBatch(wide[:S, :width], i32(before), i32(rows), T)
    seen = [0] * T                                       # of rows that exactly one well-formed sequence has and is counted to
    for r in range(T):
        s = sum(x <= r for x in rows[1:])
        seen[r] = s < S and rows[s] <= r < rows[s + 1] and 0 <= rows[s] and rows[s + 1] <= T and before[s] + rows[s + 1] - rows[s] <= width * page
    k, v = (torch.full((T, 2, dim), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    _lib.check(_lib.lib().b200_paged_read(cache._ref, batch._ref, k.data_ptr(), v.data_ptr(), torch.cuda.current_stream().cuda_stream))
    one = 8.0 if dtype == "int8" else 2.0 ** -6
    for got in (k, v):
        assert [float(x) for x in got.float().amax((1, 2))] == [one if ok else 7.0 for ok in seen]
        assert torch.equal(got.float().amin((1, 2)), got.float().amax((1, 2)))
    assert cache.error_flags() == paged.BAD_BATCH
    cache.clear_error_flags()
    x, q = (torch.randn(T, h, dim).bfloat16().cuda() for h in (2, 4))
    q_out = torch.full_like(q, 7.0)
    cache.append(batch, x, x, q=q, q_out=q_out, rotary=RotaryTable(dim))
    assert [bool((y == 7).all()) for y in q_out] == [not ok for ok in seen] and cache.error_flags() == paged.BAD_BATCH
    assert bool((cache.k.view(torch.int8)[6] == 64).all())


@pytest.mark.parametrize("first", [1, 15, 16, 17, 40, 200])
@pytest.mark.parametrize("new", [(1, 2), (30, 17)], ids=str)
def test_any_number_of_rows_in_front_of_the_first_sequence(first, new):
    """They belong to nobody, like those behind the last: left as they are, and nothing is recorded."""
    c = Content([41, 52], 2, 128, 16, "int8", capacity=[41 + new[0], 52 + new[1]])
    cache, other, n = c.cache(), c.cache(), sum(new)
    x, q = torch.randn(first + n + 3, 2, 128).bfloat16().cuda(), torch.randn(first + n + 3, 4, 128).bfloat16().cuda()
    batch = PagedBatch(c.table.cuda(), i32([41, 52]), i32([first, first + new[0], first + n]), first + n + 3, max(new))
    rotary = RotaryTable(128)
    turned = cache.append(batch, x, x, q=q, rotary=rotary, q_out=torch.full_like(q, 7.0))
    out = cache.attend(batch, turned, out=torch.full_like(q, 7.0))
    k, v = cache.read(batch)
    assert cache.error_flags() == 0
    for t in (turned, out):
        assert bool((t[:first] == 7).all()) and bool((t[first + n:] == 7).all())
    mine = slice(first, first + n)
    batch = batch_of(c.table, [41, 52], new)
    q2 = other.append(batch, x[mine].clone(), x[mine].clone(), q=q[mine].clone(), rotary=rotary)
    k2, v2 = other.read(batch)
    assert torch.equal(q2, turned[mine]) and torch.equal(other.attend(batch, q2), out[mine]) and torch.equal(k2, k[mine]) and torch.equal(v2, v[mine])
    assert torch.equal(other.k, cache.k) and torch.equal(other.v, cache.v)


@pytest.mark.parametrize("rows,before", [([0, 40, 0, 0], [0, 0, 0]), ([5, 0, 0, 0], [0, 0, 0]), ([0, 2, 2, 4], [0, -1, 0]), ([0, 2, 2, 4], [0, 65, 0]), ([0, 0, 0, 41], [0, 0, 24]),
                                         ([0, 1, 2, 41], [0, 0, 0])], ids=str)
def test_every_call_records_every_sequence_that_does_not_fit(rows, before):
    """Also one without rows, or one that the others' rows hide."""
    cache = PagedKVCache(12, 2, 64, 16, "int8")
    x, q = torch.randn(41, 2, 64).bfloat16().cuda(), torch.randn(41, 4, 64).bfloat16().cuda()
    batch = PagedBatch(torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4), i32(before), i32(rows), 41, 40)
    fits = rows in ([0, 1, 2, 41],)
    for call in (lambda: cache.append(batch, x, x), lambda: cache.append(batch, x, x, q=q), lambda: cache.attend(batch, q), lambda: cache.read(batch)):
        call()
        assert cache.error_flags() == (0 if fits else paged.BAD_BATCH)
        cache.clear_error_flags()


@pytest.mark.parametrize("new", [1, 140])
@pytest.mark.parametrize("size", [1.0, 1e-6, 1e-9])
@pytest.mark.parametrize("dtype,dim,page", [("int8", 128, 64), ("fp8_e4m3", 64, 16)])
def test_pages_of_zero_values_beside_small_values(new, size, dtype, dim, page):
    """A page whose values are all 0 (its scale is 0) has its share of the weights and takes no bits from the others', however small their scales are; nor does it where its keys have the largest scores."""
    c = Content([300 + new], 2, dim, page, dtype)
    cache = c.cache()
    cache.v_scale.mul_(size)
    c.scales[1] = cache.v_scale.cpu()
    for block in (0, 2):
        pg = int(c.table[0, block])
        cache.v.view(torch.int8)[pg], cache.v_scale[pg], c.codes[1][pg], c.scales[1][pg] = 0, 0, 0, 0
    for grow in (1.0, 3.0):                              # of the zeros' keys
        pg = int(c.table[0, 2])
        cache.k_scale[pg] *= grow
        c.scales[0][pg] *= grow
        q = torch.randn(new, 4, dim, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
        want, tol = oracle.attend(q.double().cpu(), *c.kvt(0), 300, dim ** -0.5)
        off = (cache.attend(batch_of(c.table, [300], [new]), q).double().cpu() - want).abs()
        assert bool((off <= tol).all()), float((off / tol).max())


@pytest.mark.parametrize("new", [1, 140])
def test_nothing_but_zero_values(new):
    c = Content([300 + new], 2, 128, 64, "int8")
    cache = c.cache()
    cache.v.zero_(), cache.v_scale.zero_()
    out = cache.attend(batch_of(c.table, [300], [new]), torch.randn(new, 4, 128).bfloat16().cuda())
    assert bool((out == 0).all()) and cache.error_flags() == 0


@pytest.mark.parametrize("new", [1, 140])
@pytest.mark.parametrize("heads", [(8, 2), (6, 1)], ids=str)
@pytest.mark.parametrize("dim", [64, 128])
def test_a_large_query_leaves_its_neighbours_alone(new, heads, dim):
    """Rows and heads of very different size in one step: each has its own result, whatever lies beside it."""
    c = Content([500 + new], heads[1], dim, 64, "int8")
    cache, batch = c.cache(), batch_of(c.table, [500], [new])
    q = torch.randn(new, heads[0], dim, generator=torch.Generator().manual_seed(2)).bfloat16()
    want, tol = oracle.attend(q.double(), *c.kvt(0), 500, dim ** -0.5)
    small, tol_small = oracle.attend(q[:, 0].double()[:, None] * 2.0 ** -30, *(x[:, :1] for x in c.kvt(0)), 500, dim ** -0.5 * 2.0 ** 30)
    large = q.clone()
    large[:, 1] *= 2.0 ** 40
    large[new // 2, 3] *= 2.0 ** 100
    got = cache.attend(batch, large.cuda()).double().cpu()
    plain = torch.ones(new, heads[0], dtype=torch.bool)
    plain[:, 1] = plain[new // 2, 3] = False
    assert bool(((got - want).abs() <= tol)[plain].all())
    assert bool(got.isfinite().all())
    tiny = q.clone()
    tiny[:, 0] *= 2.0 ** -30
    got = cache.attend(batch, tiny.cuda(), scale=dim ** -0.5 * 2.0 ** 30).double().cpu()
    assert bool(((got[:, :1] - small).abs() <= tol_small).all())


@pytest.mark.parametrize("new,before", [(1, 0), (1, 3000), (140, 0), (140, 3000)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_queries_that_are_not_finite_give_nan_whatever_they_meet(new, before, value):
    """Also where every product with a key is minus infinity: one key alone, or keys of one sign."""
    c = Content([before + new], 2, 128, 64, "int8")
    c.codes[0][..., 5] = -c.codes[0][..., 5].abs() - 1
    cache, batch = c.cache(), batch_of(c.table, [before], [new])
    q = torch.randn(new, 8, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    want = cache.attend(batch, q)
    spoilt = torch.zeros(new, 8, dtype=torch.bool, device="cuda")
    for row, head in ((0, 2), (0, 7), (new // 2, 4), (new - 1, 0)):
        q[row, head, 5] = value
        spoilt[row, head] = True
    got = cache.attend(batch, q)
    assert bool(got[spoilt].isnan().all()) and torch.equal(got[~spoilt], want[~spoilt])
    table = torch.full_like(c.table, -1)                 # a row that sees nothing gets zeros, whatever it asks
    assert bool((cache.attend(batch_of(table, [before], [new]), q) == 0).all()) and cache.error_flags() == paged.BAD_PAGE


@pytest.mark.parametrize("new", [1, 140])
@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
@pytest.mark.parametrize("power", [18, 20, 21, 22, 23])
def test_scores_whose_last_bit_is_several_units(new, dtype, power):
    """Scores of 2^(power + 6) and more in base 2, which climb by their last bit from 128 tokens to the next.  `scale` is what makes scale * log2(e) round to 1, so that all scores are exact in 32 bits."""
    scale, dim, page = 0.6931471824645996, 64, 128
    c = Content([1000 + new], 2, dim, page, dtype)
    for b, pg in enumerate(c.table[0].tolist()):
        c.scales[0][pg] = 2.0 ** power * (1 + b * 2.0 ** -23)
    c.scales[1].fill_(1.0)
    c.codes[0] = torch.zeros_like(c.codes[0])
    c.codes[0][..., 0] = 64
    q = torch.zeros(new, 4, dim)
    q[..., 0] = 1.0
    got = c.cache().attend(batch_of(c.table, [1000], [new]), q.bfloat16().cuda(), scale=scale).double().cpu()
    k, v, top = c.kvt(0)
    want, _ = oracle.attend(q.double(), k, v, top, 1000, scale)
    # weights in f16 and the result's rounding; `scale` misses ln 2 by 2e-9 of it, and scores that count differ by 2^6 at most
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * v.abs().amax()).all()), float((got - want).abs().max())


@pytest.mark.parametrize("new", [1, 20, 140])
@pytest.mark.parametrize("before,far", [(200, 0), (200, 100), (3000, 0), (3000, 2990)])
@pytest.mark.parametrize("dtype,dim", [("int8", 128), ("fp8_e4m3", 64)])
def test_weights_far_under_the_largest(new, before, far, dtype, dim):
    """One token has nearly all of the weight and a value of 0, the others 2^-26 of it each: what they add is the result."""
    c = Content([before + new], 2, dim, 64, dtype)
    page, slot = int(c.table[0, far // 64]), far % 64
    top = oracle.Q_MAX[dtype]
    c.codes[0][..., 0] = 0
    c.codes[0][page, :, slot], c.codes[0][page, :, slot, 0] = 0, top
    c.codes[1] = c.codes[1].abs()
    c.codes[1][page, :, slot] = 0
    c.scales[0].fill_(1 / top), c.scales[1].fill_(1 / top)
    q = torch.randn(new, 4, dim, generator=torch.Generator().manual_seed(2))
    q[..., 0] = 26 * 0.6931 * dim ** 0.5
    q = q.bfloat16()
    k, v, most = c.kvt(0)
    scale = dim ** -0.5
    want, tol = oracle.attend(q.double(), k, v, most, before, scale)
    off = (c.cache().attend(batch_of(c.table, [before], [new]), q.cuda()).double().cpu() - want).abs()
    assert float((tol / want.clamp_min(1e-30)).median()) < 0.2
    assert bool((off <= tol).all()), (float((off / tol).max()), float((off / want.clamp_min(1e-30)).max()))


def test_error_flags_wait_for_every_stream():
    """What a kernel records on another stream than the current one counts, however late it comes."""
    cache = PagedKVCache(4, 2, 64, 16, "int8")
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    batch = batch_of(torch.zeros(1, 2, dtype=torch.int32), [-1], [1])
    cache.append(batch, x, x)                            # the kernel is loaded
    assert cache.error_flags() == paged.BAD_BATCH
    cache.clear_error_flags()
    assert cache.error_flags() == 0
    torch.cuda._sleep(1000)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        torch.cuda._sleep(400_000_000)                   # 0.2 s
        cache.append(batch, x, x)
    assert cache.error_flags() == paged.BAD_BATCH


@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
@pytest.mark.parametrize("new", [15, 24])
def test_codes_are_those_of_a_division(dtype, new):
    """x / scale in 32 bits, rounded once, and that to the nearest code: over all scales, values that end up between two codes among them."""
    page, dim, pages, heads = 32, 128, 238, 2
    top = oracle.Q_MAX[dtype]
    g = torch.Generator().manual_seed(4)
    cache = PagedKVCache(pages, heads, dim, page, dtype)
    # a page holds one row already, under a scale of any size from 2^-60 to 2^58
    scale = torch.ldexp(1 + torch.rand(pages, heads, generator=g) * (torch.arange(pages) % 2)[:, None], torch.arange(pages).div(2, rounding_mode="floor")[:, None] - 60).clamp_max(2.0 ** 58).float()
    cache.v_scale.copy_(scale), cache.k_scale.copy_(scale)
    y = (torch.rand(pages, new, heads, dim, generator=g) * 2 - 1) * top
    y[:, ::3] = y[:, ::3].round() + 0.5
    if dtype == "fp8_e4m3":
        y[:, 1::3] *= torch.exp2(-12 * torch.rand(pages, (new + 1) // 3, heads, 1, generator=g))[:, :y[:, 1::3].shape[1]]
    x = (y.clamp(-0.99 * top, 0.99 * top) * scale[:, None, :, None]).bfloat16()
    x = torch.where(x.float().abs() <= top * scale[:, None, :, None], x, torch.zeros_like(x)).clamp(-2.0 ** 64, 2.0 ** 64)
    batch = batch_of(torch.arange(pages, dtype=torch.int32)[:, None], [1] * pages, [new] * pages)
    cache.append(batch, *(x.flatten(0, 1).cuda() for _ in range(2)))
    assert cache.error_flags() == 0
    for pool, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        assert torch.equal(s.cpu(), scale)
        quotient = (x.float() / scale[:, None, :, None]).transpose(1, 2)
        want = quotient.round() if dtype == "int8" else quotient.to(torch.float8_e4m3fn).float()
        got = pool[:, :, 1:1 + new].float().cpu()
        assert torch.equal(got, want), (got - want).abs().max()


@pytest.mark.parametrize("new", [1, 5, 140])
@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
def test_far_positions_under_a_window(new, dtype):
    """Two billion tokens in, all of them on one page: what a session sees that is as far from a page's border and much younger."""
    page, near = 128, 1700
    far = near + page * 15_600_000
    cache = Content([page], 2, 128, page, dtype, spare=0).cache()
    q = torch.randn(new, 8, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    table = torch.zeros(1, -(-(far + new) // page), dtype=torch.int32, device="cuda")
    for window, sinks in ((500, 0), (333, 3), (1, 200), (1500, 130)):
        a, b = (cache.attend(PagedBatch(table, i32([before]), i32([0, new]), new), q, window=window, sinks=sinks).float() for before in (near, far))
        # each within half a step of bf16 and 2^-11 and less of what it sums up, which is 3 at most a value
        assert bool(((a - b).abs() <= 2.0 ** -7 * torch.maximum(a.abs(), b.abs()) + 2.0 ** -9 * 3).all())
    assert cache.error_flags() == 0


@pytest.mark.parametrize("dtype,dim,page", [("int8", 128, 64), ("fp8_e4m3", 64, 16)])
def test_a_step_in_two_batches_over_the_same_tensors(dtype, dim, page):
    """A portion of a prompt and single rows, each with a plan of its own: the other's rows belong to nobody, and are left as they are."""
    new, before = [150, 1, 1, 1, 0, 1], [700, 300, 64, 63, 5, 0]
    c = Content(before, 2, dim, page, dtype, capacity=[b + n for b, n in zip(before, new)])
    one, two = c.cache(), c.cache()
    q, k, v = (torch.randn(sum(new), h, dim).bfloat16().cuda() for h in (8, 2, 2))
    batch, rotary = batch_of(c.table, before, new), RotaryTable(dim)
    want_q = one.append(batch, k, v, q=q, rotary=rotary)
    assert torch.equal(one.append(batch, k, v, q=q, rotary=rotary), want_q)
    got_q, out, T = torch.full_like(q, 7.0), torch.full_like(q, 7.0), batch.total_rows
    parts = [PagedBatch(batch.table[:1], batch.before[:1], batch.rows[:2], T, 150), PagedBatch(batch.table[1:], batch.before[1:], batch.rows[1:], T, 1)]
    for b in parts:
        two.append(b, k, v, q=q, rotary=rotary, q_out=got_q)
    for b in parts:
        two.attend(b, got_q, out=out)
    assert torch.equal(got_q, want_q) and one.error_flags() == two.error_flags() == 0
    assert all(torch.equal(a.view(torch.int8), b.view(torch.int8)) for a, b in ((one.k, two.k), (one.v, two.v)))       # as bytes: unwritten places are NaN
    # the same rows cut into other ranges: 32-bit sums in another order, weights in f16, and half a step of bf16 each
    want = one.attend(batch, want_q).float()
    assert bool(((out.float() - want).abs() <= 2.0 ** -7 * torch.maximum(out.float().abs(), want.abs()) + 2.0 ** -9 * 3).all())


@pytest.mark.parametrize("dim,page", [(128, 16), (64, 64)])
def test_last_tiles_in_which_only_some_lanes_hide_tokens(dim, page):
    """Every number of tokens in the last tile; what lies behind them is NaN.  The same call gives the same bits."""
    lengths = list(range(1, 34)) + [95, 96, 97]
    c = Content(lengths, 2, dim, page, "fp8_e4m3")
    cache, q = c.cache(), torch.randn(len(lengths), 8, dim, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    batch = batch_of(c.table, [n - 1 for n in lengths], [1] * len(lengths))
    out = [cache.attend(batch, q) for _ in range(5)]
    assert all(torch.equal(x, out[0]) for x in out) and cache.error_flags() == 0
    for s, n in enumerate(lengths):
        want, tol = oracle.attend(q[s:s + 1].double().cpu(), *c.kvt(s), n - 1, dim ** -0.5)
        assert bool(((out[0][s:s + 1].double().cpu() - want).abs() <= tol).all()), n


@pytest.mark.parametrize("sequences", [1, 33, 500, 700])
def test_prompts_among_any_number_of_sequences(sequences):
    """The first block looks at all of them, 512 at a time: whole warps, parts of one, several turns."""
    lengths, new = [40] * sequences, [0] * sequences
    new[0] = new[-1] = 40
    c = Content(lengths, 1, 64, 64, "int8")
    cache, q = c.cache(), torch.randn(sum(new), 8, 64, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    batch = batch_of(c.table, [n - m for n, m in zip(lengths, new)], new)
    out = [cache.attend(batch, q) for _ in range(3)]
    assert all(torch.equal(x, out[0]) for x in out) and cache.error_flags() == 0
    for at, s in enumerate(sorted({0, sequences - 1})):
        want, tol = oracle.attend(q[40 * at:40 * at + 40].double().cpu(), *c.kvt(s), 0, 64 ** -0.5)
        assert bool(((out[0][40 * at:40 * at + 40].double().cpu() - want).abs() <= tol).all()), s
