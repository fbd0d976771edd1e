"""The paged 8-bit cache on the GPU against 64-bit restatements (oracle/paged.py)."""
import pytest
import torch

from moshi_b200.models import PagedBatch, PagedKVCache, RotaryTable
from moshi_b200.models import paged
from oracle import paged as oracle

from .paged_util import Content, batch_of

pytestmark = pytest.mark.gpu
FORMS = [("int8", 128, 64), ("fp8_e4m3", 128, 16), ("int8", 64, 16), ("fp8_e4m3", 64, 128), ("int8", 128, 32)]


def check_attention(lengths, new, heads, form, window=0, sinks=0, scale=None, spread=1.0, total=None, q_size=1.0, seed=1):
    """lengths: tokens in front of the step; rows `new`.  The step's own tokens are in the cache already."""
    dtype, dim, page = form
    hq, hkv = heads
    c = Content([a + n for a, n in zip(lengths, new)], hkv, dim, page, dtype, seed=seed, spread=spread)
    cache = c.cache()
    T = sum(new) if total is None else total
    g = torch.Generator().manual_seed(seed + 1)
    wide = (torch.randn(T, hq + 3, dim, generator=g) * q_size).bfloat16().cuda()
    q = wide[:, 2:hq + 2]                                # rows lie apart
    out = torch.full((T, hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    batch = batch_of(c.table, lengths, new, total=T)
    got = cache.attend(batch, q, scale=scale, window=window, sinks=sinks, out=out)
    assert got is out and cache.error_flags() == 0
    at = 0
    for s, (a, n) in enumerate(zip(lengths, new)):
        if n:
            want, tol = oracle.attend(q[at:at + n].double().cpu(), *c.kvt(s), a, dim ** -0.5 if scale is None else scale, window, sinks)
            off = (out[at:at + n].double().cpu() - want).abs()
            assert bool((off <= tol).all()), (s, a, n, float((off - tol).max()), float((off / tol.clamp_min(1e-30)).max()))
        at += n
    assert bool((out[at:] == 7.0).all())                 # rows behind the last sequence
    return out


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("heads", [(4, 4), (8, 1), (6, 2), (15, 3), (40, 2)], ids=str)
def test_single_tokens(form, heads):
    """Lengths around the borders of tiles and pages, an empty cache among them; a sequence without a row."""
    check_attention([0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 300, 40], [1] * 11 + [0], heads, form)


@pytest.mark.parametrize("form", FORMS, ids=str)
def test_ranges_of_the_keys(form):
    """Few sequences: the keys are cut into ranges, unevenly long ones and empty ones."""
    check_attention([5000, 257], [1, 1], (4, 2), form)
    check_attention([3001], [1], (3, 1), form)
    check_attention([2000, 0, 900], [3, 0, 2], (4, 2), form)


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("heads", [(4, 4), (7, 1), (24, 2)], ids=str)
@pytest.mark.parametrize("new", [[2, 5, 1, 0, 9], [33, 0, 64, 1], [130, 257]], ids=str)
def test_several_rows(form, heads, new):
    check_attention([0, 37, 100, 5, 64][:len(new)], new, heads, form)


@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 4), (100, 70), (64, 16), (1000, 3), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("form", FORMS, ids=str)
def test_windows_and_first_tokens(form, window, sinks):
    check_attention([0, 3, 90, 400, 1500], [1, 1, 1, 1, 1], (4, 2), form, window, sinks)
    check_attention([0, 120, 700], [70, 5, 200], (6, 2), form, window, sinks)


def test_pages_outside_the_window_are_not_looked_at():
    """Their entries may name pages that do not exist."""
    c = Content([1000], 2, 128, 16, "int8")
    cache, q = c.cache(), torch.randn(1, 4, 128).bfloat16().cuda()
    want = cache.attend(batch_of(c.table, [999], [1]), q, window=100, sinks=4)
    table = c.table.clone()
    table[0, 1:50] = 10 ** 9
    got = cache.attend(batch_of(table, [999], [1]), q, window=100, sinks=4)
    assert torch.equal(got, want) and cache.error_flags() == 0


@pytest.mark.parametrize("new", [1, 200])
def test_rows_behind_the_last_sequence(new):
    check_attention([50, 3], [new, 2], (8, 2), ("int8", 128, 64), total=new + 2 + 37)


@pytest.mark.parametrize("new", [1, 150])
def test_scales_far_apart_and_large_queries(new):
    """Pages whose scales differ by many powers of two; scores in the hundreds, so that one key takes all."""
    check_attention([400, 77], [new, new], (8, 2), ("int8", 128, 32), spread=30.0)
    check_attention([400, 77], [new, new], (8, 2), ("fp8_e4m3", 128, 32), spread=1000.0)
    check_attention([400, 77], [new, new], (8, 2), ("int8", 64, 64), q_size=300.0)
    check_attention([400, 77], [new, new], (8, 2), ("int8", 64, 64), q_size=1e-30, scale=1e20)


@pytest.mark.parametrize("new", [1, 140])
def test_pages_of_zeros(new):
    c = Content([300 + new], 2, 128, 64, "int8")
    cache = c.cache()
    page = int(c.table[0, 1])
    for side, (pool, scale) in enumerate(((cache.k, cache.k_scale), (cache.v, cache.v_scale))):
        pool[page], scale[page], c.codes[side][page], c.scales[side][page] = 0, 0, 0, 0
    q = torch.randn(new, 4, 128).bfloat16().cuda()
    want, tol = oracle.attend(q.double().cpu(), *c.kvt(0), 300, 128 ** -0.5)
    assert bool(((cache.attend(batch_of(c.table, [300], [new]), q).double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("new", [1, 140])
def test_a_query_that_is_not_finite_spoils_its_own_results_only(new):
    c = Content([500 + new], 2, 128, 64, "int8")
    cache, q = c.cache(), torch.randn(new, 8, 128).bfloat16().cuda()
    batch = batch_of(c.table, [500], [new])
    want = cache.attend(batch, q)
    q[0, 3, 5], q[-1, 6, 0] = float("nan"), float("inf")
    got = cache.attend(batch, q)
    spoilt = torch.zeros(new, 8, dtype=torch.bool, device="cuda")
    spoilt[0, 3] = spoilt[-1, 6] = True
    assert bool(got[spoilt].isnan().all()) and torch.equal(got[~spoilt], want[~spoilt])


@pytest.mark.parametrize("new", [1, 140])
def test_what_does_not_fit_is_left_out_and_recorded(new):
    c = Content([100 + new, 200 + new], 2, 64, 16, "int8")
    cache, q = c.cache(), torch.randn(2 * new, 2, 64).bfloat16().cuda()
    exact = [oracle.attend(q[new * s:new * (s + 1)].double().cpu(), *c.kvt(s), (100, 200)[s], 0.125) for s in (0, 1)]

    def good(out, s):
        want, tol = exact[s]
        return bool(((out[new * s:new * (s + 1)].double().cpu() - want).abs() <= tol).all())

    def untouched(out, s):
        return bool((out[new * s:new * (s + 1)] == 7).all())

    def run(table, before, rows, max_rows=None):
        out = torch.full_like(q, 7.0)
        cache.attend(PagedBatch(table.cuda(), *(torch.tensor(x, dtype=torch.int32).cuda() for x in (before, rows)), 2 * new, max_rows), q, out=out)
        flags = cache.error_flags()
        cache.clear_error_flags()
        return out, flags
    rows = [0, new, 2 * new]
    for before, r in (([-1, 200], rows), ([2 ** 31 - 1, 200], rows), ([100000, 200], rows), ([100, 200], [-5, new, 2 * new])):
        out, flags = run(c.table, before, r, new)
        assert flags == paged.BAD_BATCH and untouched(out, 0) and good(out, 1), before
    out, flags = run(c.table, [100, 200], [0, new, 2 * new + 1])
    assert flags == paged.BAD_BATCH and good(out, 0) and untouched(out, 1)
    if new > 1:
        out, flags = run(c.table, [100, 200], rows, new - 1)
        assert flags == paged.BAD_BATCH and untouched(out, 0) and untouched(out, 1)
    for bad in (-1, c.pages, 2 ** 31 - 1):
        table = c.table.clone()
        table[0, 2] = bad
        out, flags = run(table, [100, 200], rows)
        assert flags == paged.BAD_PAGE and good(out, 1)
        k, v, top = (torch.cat((x[:32], x[48:])) for x in c.kvt(0))
        if new == 1:                                     # its tokens are left out
            want, tol = oracle.attend(q[:1].double().cpu(), k, v, top, len(k), 0.125)
            assert bool(((out[:1].double().cpu() - want).abs() <= tol).all())


# ------------------------------------------------------------------------------------------------------------------------
# append and read
# ------------------------------------------------------------------------------------------------------------------------
def within(dtype, x, got, s):
    """Codes of x (f64) with the scale s: half a step and what 32-bit rotations are off by (2^-21 of the page's largest, 2^-13 of a step)."""
    half = 0.5 * s if dtype == "int8" else torch.maximum(2.0 ** -4 * x.abs(), torch.as_tensor(2.0 ** -10 * s))
    return (got - x).abs() <= half * (1 + 2.0 ** -9) + 2.0 ** -12 * s


@pytest.mark.parametrize("form", FORMS, ids=str)
@pytest.mark.parametrize("pairing,rot", [("adjacent", 1.0), ("halves", 1.0), ("halves", 0.5), ("adjacent", 0.25), (None, 0)])
@pytest.mark.parametrize("new", [[1] * 6, [3, 0, 4, 2, 1, 1], [16, 9, 0, 5, 13, 1], [17, 1, 2, 0, 3, 16], [70, 1, 0, 129, 16, 5]], ids=str)
def test_append(form, pairing, rot, new):
    dtype, dim, page = form
    before, hkv, hq, T = [0, 17, 63, 64, 1000, 100000], 3, 6, sum(new) + 5
    before = [min(b, 4 * page + b % page) if b == 100000 else b for b in before]
    c = Content(before, hkv, dim, page, dtype, capacity=[b + n for b, n in zip(before, new)])
    cache = c.cache()
    kept = [x.clone() for x in (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)]
    rot = int(rot * dim)
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(T, (hq + 2 * hkv) * dim, generator=g)
    wide *= torch.exp2(2 * torch.randn(T, 1, generator=g))                # so that scales grow
    wide = wide.bfloat16().cuda()
    q, k, v = (x.unflatten(1, (-1, dim)) for x in wide.split([hq * dim, hkv * dim, hkv * dim], 1))
    batch = batch_of(c.table, before, new, total=T)
    rotary = RotaryTable(rot, pairing=pairing) if pairing else None
    q_out = torch.full((T, hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    assert cache.append(batch, k, v, q=q, rotary=rotary, q_out=q_out) is q_out and cache.error_flags() == 0
    once = [x.clone() for x in (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)]
    cache.append(batch, k, v, q=q, rotary=rotary, q_out=q_out)            # the same rows again: nothing changes
    assert all(torch.equal(a, b) or bool((a.isnan() & b.isnan() | (a == b)).all()) for a, b in zip(once, (cache.k.view(torch.int8), cache.v.view(torch.int8), cache.k_scale, cache.v_scale)))
    rk, rv = cache.read(batch_of(c.table, [0] * 6, [b + n for b, n in zip(before, new)]))
    rk, rv = rk.double().cpu(), rv.double().cpu()
    at = back = 0
    touched = torch.zeros(c.pages, dtype=torch.bool)
    for s, (b, n) in enumerate(zip(before, new)):
        exact = oracle.rotated(q[at:at + n].double().cpu(), b, rot, pairing=pairing) if pairing else q[at:at + n].double().cpu()
        assert bool(((q_out[at:at + n].double().cpu() - exact).abs() <= 2.0 ** -8 * exact.abs() + 2.0 ** -20 * exact.abs().amax(-1, keepdim=True)).all()) if n else True
        for side, (rows, read, pool, scale) in enumerate(((k, rk, cache.k, cache.k_scale), (v, rv, cache.v, cache.v_scale))):
            x = rows[at:at + n].double().cpu()
            if side == 0 and pairing:
                x = oracle.rotated(x, b, rot, pairing=pairing)
            for p in range(b // page, -(-(b + n) // page)) if n else ():
                pg, o, e = int(c.table[s, p]), max(b - p * page, 0), min(b + n - p * page, page)
                touched[pg] = True
                for h in range(hkv):
                    new_x = x[p * page + o - b:p * page + e - b, h]
                    _, want_s = oracle.append(c.codes[side][pg, h], float(c.scales[side][pg, h]), o, new_x, dtype)
                    got_s = float(scale[pg, h])
                    assert abs(got_s - want_s) <= 2.0 ** -20 * want_s, (s, p, h, got_s, want_s)
                    codes = pool[pg, h].float().double().cpu()
                    assert bool(within(dtype, new_x, codes[o:e] * got_s, got_s).all())
                    old, was = codes[:o] * got_s, c.codes[side][pg, h, :o] * float(c.scales[side][pg, h])
                    assert bool(((old - was).abs() <= (0.5 if dtype == "int8" else 2.0 ** -10) * got_s * (1 + 1e-6)).all())
                    if got_s == float(c.scales[side][pg, h]):
                        assert torch.equal(codes[:o], c.codes[side][pg, h, :o])
                    here = codes[:e] * got_s
                    assert bool(((read[back + p * page:back + p * page + e, h] - here).abs() <= 2.0 ** -8 * here.abs()).all())
                    raw, was = pool.view(torch.int8)[pg, h, e:], kept[side][pg, h, e:]
                    assert torch.equal(raw, was)                          # behind the last row
        at += n
        back += b + n
    assert bool((q_out[at:] == 7.0).all())
    for a, b in zip(once, kept):                                          # pages that the step does not touch
        x, y = a.cpu()[~touched], b.cpu()[~touched]
        assert torch.equal(x.nan_to_num(-1.0) if x.is_floating_point() else x, y.nan_to_num(-1.0) if y.is_floating_point() else y)


@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
@pytest.mark.parametrize("growth", [1.001, 1.05, 1.7, 0.8])
def test_a_page_that_grows_token_by_token(dtype, growth):
    """Every code stays within one step of the page's last scale (half a step, a quarter and so on: at most a step; for e4m3 its half step and subnormals')."""
    page, n, dim = 128, 128, 64
    cache = PagedKVCache(2, 2, dim, page, dtype)
    g = torch.Generator().manual_seed(5)
    x = (torch.randn(n, 2, dim, generator=g) * growth ** torch.arange(n)[:, None, None]).bfloat16()
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    for i in range(n):
        cache.append(batch_of(table, [i], [1]), x[i:i + 1].cuda(), x[i:i + 1].cuda())
    k, v = cache.read(batch_of(table, [0], [n]))
    for read, pool, scale in ((k, cache.k, cache.k_scale), (v, cache.v, cache.v_scale)):
        s = scale[1].double().cpu()
        got = pool[1].float().double().cpu().transpose(0, 1) * s[:, None]
        want = torch.where(x.abs() <= oracle.MAGNITUDE, x, torch.zeros_like(x)).double()      # what is larger is stored as 0
        step = s[:, None] * torch.ones_like(want) if dtype == "int8" else 2.0 ** -4 * want.abs() * (1 + 2.0 ** -6) + 2.0 ** -9 * s[:, None]
        assert bool(((got - want).abs() <= step).all())
        assert bool(((read.double().cpu() - got).abs() <= 2.0 ** -8 * got.abs()).all())


def test_far_positions():
    """The angle of position 2 * 10^9, where an angle in 32 bits is hundreds of turns off."""
    page, before = 128, 2 * 10 ** 9
    blocks = before // page + 1
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda").expand(1, 1)
    wide = torch.zeros(1, blocks, dtype=torch.int32, device="cuda")
    cache = PagedKVCache(1, 1, 128, page, "int8")
    q = torch.randn(1, 2, 128).bfloat16().cuda()
    k = torch.randn(1, 1, 128).bfloat16().cuda()
    for pairing in ("adjacent", "halves"):
        got = cache.append(PagedBatch(wide, torch.tensor([before], dtype=torch.int32, device="cuda"), torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1), k, k, q=q,
                           rotary=RotaryTable(128, pairing=pairing))
        want = oracle.rotated(q.double().cpu(), before, 128, pairing=pairing)
        # the 64-bit angle itself is off by before * 2^-53 = 2.2e-7 of a radian
        assert bool(((got.double().cpu() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -19 * want.abs().amax()).all())
    assert cache.error_flags() == 0 and table.shape == (1, 1)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes a side."""
    pages, page, heads, dim = 4200, 128, 64, 128
    cache = PagedKVCache(pages, heads, dim, page, "int8")
    assert cache.k.numel() > 2 ** 32
    table = torch.tensor([[pages - 1, pages - 2], [0, 1]], dtype=torch.int32)
    g = torch.Generator().manual_seed(0)
    for new in ([150, 140], [1, 1]):
        before = [0, 0] if new[0] > 1 else [150, 140]
        k, v, q = (torch.randn(sum(new), heads, dim, generator=g).bfloat16().cuda() for _ in range(3))
        batch = batch_of(table, before, new)
        cache.append(batch, k, v)
        out = cache.attend(batch, q)
        rk, rv = cache.read(batch_of(table, [0, 0], [b + n for b, n in zip(before, new)]))
        at = back = 0
        for b, n in zip(before, new):
            # against what was read back; its rounding to bf16 moves scores by 2^-8 of a key's share at most, values by 2^-8
            kk, vv = (x[back:back + b + n].double().cpu() for x in (rk, rv))
            want, _ = oracle.attend(q[at:at + n].double().cpu(), kk, vv, vv.abs().amax(-1), b, dim ** -0.5)
            assert float((out[at:at + n].double().cpu() - want).norm() / want.norm()) < 2.0 ** -6
            at, back = at + n, back + b + n
    assert cache.error_flags() == 0


@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
def test_values_that_are_not_finite_are_stored_as_zero(dtype):
    cache = PagedKVCache(2, 2, 128, 16, dtype)
    table = torch.tensor([[0, 1]], dtype=torch.int32)
    k = torch.randn(20, 2, 128).bfloat16()
    bad = k.clone()
    bad[3, 1, 7], bad[4, 0, 100], bad[18, 1, 127], bad[18, 1, 0] = float("nan"), float("inf"), -float("inf"), 1e30
    clean = torch.where(bad.abs() <= 1.8e19, bad, torch.zeros_like(bad))
    cache.append(batch_of(table, [0], [20]), bad.cuda(), bad.cuda())
    assert cache.error_flags() == paged.NOT_FINITE
    other = PagedKVCache(2, 2, 128, 16, dtype)
    other.append(batch_of(table, [0], [20]), clean.cuda(), clean.cuda())
    assert other.error_flags() == 0
    for a, b in zip((cache.k.view(torch.int8), cache.v_scale, cache.k_scale), (other.k.view(torch.int8), other.v_scale, other.k_scale)):
        assert torch.equal(a, b)


def test_tiny_and_zero_rows():
    """Zeros have the scale 0 until something else comes; magnitudes under 2^-60 are stored in steps of 2^-60."""
    cache = PagedKVCache(1, 1, 64, 16, "int8")
    row = lambda x: torch.full((1, 1, 64), x).bfloat16().cuda()           # noqa: E731
    table = torch.tensor([[0]], dtype=torch.int32)
    seen = []
    for i, x in enumerate((0.0, 0.0, 1e-30, 2.0 ** -58, 1.0, 0.0)):
        cache.append(batch_of(table, [i], [1]), row(x), row(x))
        seen.append(float(cache.k_scale[0, 0]))
    assert seen[:4] == [0.0, 0.0, 2.0 ** -60, 2.0 ** -60] and seen[4] == seen[5] and 1 / 127 <= seen[4] < 2 / 127
    assert cache.k[0, 0, :6, 0].tolist()[:4] == [0, 0, 0, 0] and 63 < cache.k[0, 0, 4, 0] <= 127 and cache.error_flags() == 0


def test_append_leaves_out_what_does_not_fit():
    c = Content([20, 40], 2, 64, 16, "int8", capacity=[30, 50])
    x = torch.randn(4, 2, 64).bfloat16().cuda()
    for before, rows, max_rows, flag in (([-1, 40], [0, 2, 4], 2, paged.BAD_BATCH), ([63, 40], [0, 2, 4], 2, paged.BAD_BATCH), ([20, 40], [0, 3, 4], 2, paged.BAD_BATCH),
                                         ([2 ** 31 - 1, 40], [0, 2, 4], 2, paged.BAD_BATCH), ([20, 40], [0, 2, 4], 2, paged.BAD_PAGE)):
        cache = c.cache()
        table = c.table.clone()
        if flag == paged.BAD_PAGE:
            table[0, 1] = c.pages
        mine = c.table[0].clamp_min(0).unique()
        was = cache.k.view(torch.int8)[mine].clone()
        kw = [torch.tensor(t, dtype=torch.int32).cuda() for t in (before, rows)]
        q = x.clone()
        cache.append(PagedBatch(table.cuda(), *kw, 4, max_rows), x, x, q=q, q_out=q, rotary=RotaryTable(64))
        assert cache.error_flags() == flag, (before, rows)
        assert torch.equal(cache.k.view(torch.int8)[c.table[0][c.table[0] >= 0].long()], was[torch.searchsorted(mine, c.table[0][c.table[0] >= 0])])
        assert not torch.equal(q[rows[1]:], x[rows[1]:])                  # the other sequence has its rows
        if flag == paged.BAD_BATCH:
            assert torch.equal(q[:rows[1]], x[:rows[1]])


@pytest.mark.parametrize("rows", [[0, 10, 5, 12], [12, 4, 2, 0], [3, 3, 1, 9], [0, 2 ** 31 - 1, -2 ** 31, 4]])
def test_rows_out_of_order_stay_within_the_tensors(rows):
    """Recorded, and nothing else than the batch's own pages and rows is touched."""
    c = Content([40, 40, 40], 2, 64, 16, "int8", capacity=[60, 60, 60], spare=5)
    cache = c.cache()
    was = [x.clone() for x in (cache.k.view(torch.int8), cache.v.view(torch.int8))]
    x = torch.randn(14, 2, 64).bfloat16().cuda()
    wide = torch.full((34, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    q = wide[10:24]
    batch = PagedBatch(c.table.cuda(), torch.tensor([40] * 3, dtype=torch.int32).cuda(), torch.tensor(rows, dtype=torch.int32).cuda(), 14)
    for new in (x, x.repeat(1, 1, 1)):
        cache.append(batch, new, new, q=q, q_out=q, rotary=RotaryTable(64))
    cache.attend(batch, q.clone(), out=q)
    cache.read(batch)
    assert cache.error_flags() & paged.BAD_BATCH
    assert bool((wide[:10] == 7).all()) and bool((wide[24:] == 7).all())
    mine = c.table[c.table >= 0].long()
    others = torch.ones(c.pages, dtype=torch.bool)
    others[mine] = False
    for a, b in zip((cache.k.view(torch.int8), cache.v.view(torch.int8)), was):
        assert torch.equal(a.cpu()[others], b.cpu()[others])
        assert torch.equal(a.cpu()[c.table[:, :2].long()], b.cpu()[c.table[:, :2].long()])      # pages that are full already


def test_rows_in_front_of_the_first_sequence():
    c = Content([41, 52], 2, 128, 16, "int8", capacity=[45, 60])
    cache = c.cache()
    x, q = torch.randn(9, 2, 128).bfloat16().cuda(), torch.randn(9, 4, 128).bfloat16().cuda()
    args = [torch.tensor(t, dtype=torch.int32).cuda() for t in ([41, 52], [3, 4, 6])]
    batch = PagedBatch(c.table.cuda(), *args, 9, 2)
    turned = cache.append(batch, x, x, q=q, rotary=RotaryTable(128), q_out=torch.full_like(q, 7.0))
    out = cache.attend(batch, turned, out=torch.full_like(q, 7.0))
    for t in (turned, out):
        assert bool((t[:3] == 7).all()) and bool((t[6:] == 7).all()) and not bool((t[3:6] == 7).all())
    other = c.cache()
    batch = batch_of(c.table, [41, 52], [1, 2])
    turned = other.append(batch, x[3:6].clone(), x[3:6].clone(), q=q[3:6].clone(), rotary=RotaryTable(128))
    assert torch.equal(other.attend(batch, turned), out[3:6]) and torch.equal(other.k, cache.k) and cache.error_flags() == 0


def test_tensors_that_do_not_fit_are_refused():
    cache = PagedKVCache(8, 2, 128, 16, "int8")
    batch = batch_of(torch.zeros(2, 4, dtype=torch.int32), [0, 0], [1, 2])
    good, q = torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(3, 4, 128, dtype=torch.bfloat16, device="cuda")
    for k in (good.float(), good[:2], good[..., :64], good[:, :1], good.transpose(0, 1), good.cpu(), good[..., None], torch.zeros(3, 128, 2, dtype=torch.bfloat16, device="cuda").transpose(1, 2),
              torch.zeros(3, 2, 128, dtype=torch.bfloat16, device="cuda", requires_grad=True), torch.zeros(1, 2, 128, dtype=torch.bfloat16, device="cuda").expand(3, 2, 128),
              torch.zeros(3 * 260 + 4, dtype=torch.bfloat16, device="cuda")[4:784].view(3, 260)[:, :256].unflatten(1, (2, 128))):
        with pytest.raises((ValueError, AssertionError)):
            cache.append(batch, k, good)
        with pytest.raises((ValueError, AssertionError)):
            cache.append(batch, good, k)
    for bad in (q[..., :64], q.float(), q[:2], q.flatten(1), torch.zeros(3, 3, 128, dtype=torch.bfloat16, device="cuda"), q.clone().requires_grad_()):
        with pytest.raises((ValueError, AssertionError)):
            cache.attend(batch, bad)
        with pytest.raises((ValueError, AssertionError)):
            cache.attend(batch, q, out=bad)
    for kw in (dict(window=-1), dict(sinks=-1), dict(window=2 ** 31), dict(window=2 ** 32 + 5), dict(scale=0.0), dict(scale=float("nan"))):
        with pytest.raises(ValueError):
            cache.attend(batch, q, **kw)
    with pytest.raises(ValueError):
        cache.append(batch, good, good, q_out=q)
    with pytest.raises(ValueError):
        cache.append(batch, good, good, q=q, rotary=RotaryTable(256))
    i32 = dict(dtype=torch.int32, device="cuda")
    for args in ((torch.zeros(2, 4, **i32), torch.zeros(3, **i32), torch.zeros(3, **i32), 3), (torch.zeros(2, 4, **i32).long(), torch.zeros(2, **i32), torch.zeros(3, **i32), 3),
                 (torch.zeros(4, 2, **i32).t(), torch.zeros(2, **i32), torch.zeros(3, **i32), 3), (torch.zeros(2, 4, **i32), torch.zeros(2, **i32), torch.zeros(3, **i32), -1),
                 (torch.zeros(1, 4, **i32).expand(2, 4), torch.zeros(2, **i32), torch.zeros(3, **i32), 3), (torch.zeros(2, 4, **i32), torch.zeros(2, **i32).cpu(), torch.zeros(3, **i32), 3)):
        with pytest.raises(ValueError):
            PagedBatch(*args)
    with torch.no_grad():                                # a tensor that could have a gradient, where none is asked for
        cache.append(batch, good.clone().requires_grad_(), good)
    assert cache.error_flags() == 0


# ------------------------------------------------------------------------------------------------------------------------
# a run of them together
# ------------------------------------------------------------------------------------------------------------------------
def model_run(dtype, dim, page, window, sinks, portions, seed=0):
    """Three sequences through steps of a layer, pages handed out as they are needed; every step against 64 bits on what the cache holds."""
    hq, hkv, S = 6, 2, 3
    total = [sum(p[s] for p in portions) for s in range(S)]
    g = torch.Generator().manual_seed(seed)
    cache = PagedKVCache(sum(-(-x // page) for x in total), hkv, dim, page, dtype)
    free = torch.randperm(cache.pages, generator=g).tolist()
    width = max(-(-x // page) for x in total)
    table = torch.zeros(S, width, dtype=torch.int32)
    lengths, rotary = [0] * S, RotaryTable(dim, pairing="halves")
    for new in portions:
        for s in range(S):
            for b in range(-(-lengths[s] // page), -(-(lengths[s] + new[s]) // page)):
                table[s, b] = free.pop()
        T = sum(new)
        qkv = torch.randn(T, (hq + 2 * hkv) * dim, generator=g).bfloat16().cuda()
        q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([hq * dim, hkv * dim, hkv * dim], 1))
        batch = batch_of(table, lengths, new)
        turned = cache.append(batch, k, v, q=q, rotary=rotary)
        out = cache.attend(batch, turned, window=window, sinks=sinks)
        at = 0
        for s, n in enumerate(new):
            m = lengths[s] + n
            if n:
                pg = table[s, :-(-m // page)].long()
                kk, vv = ((pool.float()[pg.cuda()].double() * sc[pg.cuda()][..., None, None].double()).transpose(1, 2).reshape(-1, hkv, dim)[:m].cpu()
                          for pool, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
                top = (cache.v_scale[pg.cuda()].double().cpu() * oracle.Q_MAX[dtype])[:, None].expand(-1, page, -1).reshape(-1, hkv)[:m]
                want, tol = oracle.attend(turned[at:at + n].double().cpu(), kk, vv, top, lengths[s], dim ** -0.5, window, sinks)
                assert bool(((out[at:at + n].double().cpu() - want).abs() <= tol).all())
            at, lengths[s] = at + n, m
    assert cache.error_flags() == 0


@pytest.mark.parametrize("dtype,dim,page", [("int8", 128, 64), ("fp8_e4m3", 64, 16)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_prompts_and_tokens(dtype, dim, page, window, sinks):
    model_run(dtype, dim, page, window, sinks, [[150, 3, 0], [1, 1, 90], [1, 1, 1], [70, 0, 1], [1, 1, 1], [2, 4, 1], [1, 1, 1]])


def test_shared_pages_of_a_prefix():
    """Two sequences whose tables name the same pages in front; each appends to pages of its own."""
    page, dim = 16, 128
    c = Content([64], 2, dim, page, "int8", spare=6)
    cache = c.cache()
    free = [p for p in range(c.pages) if p not in c.table[0].tolist()]
    table = torch.cat((c.table.repeat(2, 1), torch.tensor([free[:2], free[2:4]], dtype=torch.int32)), 1)
    k, v, q = (torch.randn(40, h, dim).bfloat16().cuda() for h in (2, 2, 4))
    batch = batch_of(table, [64, 64], [20, 20])
    cache.append(batch, k, v)
    out = cache.attend(batch, q)
    codes = [x.float().double().cpu() for x in (cache.k, cache.v)]
    scales = [x.double().cpu() for x in (cache.k_scale, cache.v_scale)]
    assert torch.equal(codes[0][c.table[0].long()], c.codes[0][c.table[0].long()])
    for s in range(2):
        pg = table[s].long()
        kk, vv, top = (x.transpose(1, 2).reshape(-1, 2, x.shape[3])[:84] for x in (codes[0][pg] * scales[0][pg][..., None, None], codes[1][pg] * scales[1][pg][..., None, None],
                                                                                       (127 * scales[1][pg][..., None, None]).expand(-1, -1, page, 1)))
        want, tol = oracle.attend(q[20 * s:20 * s + 20].double().cpu(), kk, vv, top[..., 0], 64, dim ** -0.5)
        assert bool(((out[20 * s:20 * s + 20].double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("new", [1, 6, 200])
def test_captured_steps_on_two_streams(new):
    """Two graphs of the same cache's attention, replayed side by side and with new content behind the same pointers."""
    c = Content([3000 + new], 2, 128, 64, "int8")
    cache = c.cache()
    runs = []
    for i in range(2):
        q = torch.randn(new, 8, 128, generator=torch.Generator().manual_seed(i)).bfloat16().cuda()
        k, v = (torch.randn(new, 2, 128).bfloat16().cuda() for _ in range(2))
        batch = batch_of(c.table, [3000], [new])
        want = cache.attend(batch, q)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(graph, stream=stream):
            out = cache.attend(batch, q)
        runs.append((graph, stream, batch, q, out, want))
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, stream, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for *_, out, want in runs:
        assert torch.equal(out, want)
    graph, stream, batch, q, out, want = runs[0]
    q.copy_(runs[1][3])
    batch.before.fill_(1000)
    short = cache.attend(batch_of(c.table, [1000], [new]), q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, short) and not torch.equal(out, want)


def test_captured_append_and_attend():
    page, dim = 64, 128
    results = []
    for captured in (False, True):
        cache = PagedKVCache(8, 2, dim, page, "int8")
        table = torch.arange(8, dtype=torch.int32)[None]
        g = torch.Generator().manual_seed(11)
        rows = torch.randn(100, 1, 10 * dim, generator=g).bfloat16().cuda()
        qkv = torch.zeros(1, 10 * dim, dtype=torch.bfloat16, device="cuda")
        q, k, v = (x.unflatten(1, (-1, dim)) for x in qkv.split([6 * dim, 2 * dim, 2 * dim], 1))
        batch, rotary, outs = batch_of(table, [0], [1]), RotaryTable(dim), []

        def step():
            return cache.attend(batch, cache.append(batch, k, v, q=q, rotary=rotary), window=50, sinks=2)
        if captured:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
        for i in range(100):
            qkv.copy_(rows[i])
            batch.before.fill_(i)
            if captured:
                graph.replay()
            else:
                out = step()
            outs.append(out.clone())
        results.append(torch.cat(outs))
        assert cache.error_flags() == 0
    assert torch.equal(*results)


def test_calls_side_by_side_on_two_streams():
    """Steps of two batches over one cache at once, prompts beside single tokens, appends to pages of their own among them."""
    c = Content([900, 1400, 300], 2, 128, 64, "int8", capacity=[1200, 1500, 400])
    cache = c.cache()
    jobs = []
    for i, (s, new) in enumerate(((0, 250), (1, 1))):
        g = torch.Generator().manual_seed(i)
        kv, q = torch.randn(new, 2, 128, generator=g).bfloat16().cuda(), torch.randn(new, 8, 128, generator=g).bfloat16().cuda()
        jobs.append((batch_of(c.table[s:s + 1], [c.lengths[s]], [new]), kv, q, torch.cuda.Stream(), []))
    torch.cuda.synchronize()
    for _ in range(30):
        for batch, kv, q, stream, outs in jobs:
            with torch.cuda.stream(stream):
                cache.append(batch, kv, kv)
                outs.append(cache.attend(batch, q, window=700, sinks=5))
    torch.cuda.synchronize()
    other = c.cache()
    for batch, kv, q, _, outs in jobs:
        other.append(batch, kv, kv)
        want = other.attend(batch, q, window=700, sinks=5)
        assert all(torch.equal(x, want) for x in outs)
    assert cache.error_flags() == 0


@pytest.mark.parametrize("dim,new", [(64, 7), (64, 8), (64, 9), (128, 4), (128, 5)])
@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
def test_columns_around_the_border_between_the_kernels(dim, new, dtype):
    """Four heads a group: 28, 32 and 36 columns, 16 and 20; with a sequence of one row beside."""
    check_attention([300, 1000, 64], [new, 1, 2], (8, 2), (dtype, dim, 16))
    check_attention([300, 1000, 64], [new, 1, 2], (8, 2), (dtype, dim, 64), window=50, sinks=3)
    check_attention([777], [new], (4, 1), (dtype, dim, 32))


def test_another_stream_than_the_current_default():
    c = Content([700], 2, 128, 64, "int8")
    cache, q = c.cache(), torch.randn(1, 8, 128).bfloat16().cuda()
    batch = batch_of(c.table, [699], [1])
    want = cache.attend(batch, q)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [cache.attend(batch, q) for _ in range(50)]
    stream.synchronize()
    assert all(torch.equal(x, want) for x in got)
