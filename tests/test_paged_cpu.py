"""The paged 8-bit cache without a GPU: which kernels a call launches and what it refuses (on the fake CUDA runtime), the oracle's own properties, the rotation's fixed point."""
import ctypes as C
import decimal
import math

import pytest
import torch

from moshi_b200 import _lib
from moshi_b200.models import paged
from oracle import paged as oracle

from . import fake_cuda


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    return fake_cuda.load(tmp_path_factory.mktemp("fake"))


class Call:
    """Arguments of a call that is taken; any of them can be replaced."""

    def __init__(self, **changed):
        self.memory = C.create_string_buffer(1 << 12)
        at = (C.addressof(self.memory) + 63) // 64 * 64
        self.cache = dict(k=at, v=at, k_scale=at, v_scale=at, flags=at, pages=100, page_tokens=64, kv_heads=8, dim=128, kv_dtype=_lib.B200_KV_INT8, device=0)
        self.batch = dict(table=at, before=at, rows=at, table_ld=64, sequences=4, table_width=64, total_rows=4, max_rows=1)
        self.rotary = dict(turns=at, rot_dims=128, pairing=0)
        self.args = dict(k_ptr=at, k_row=8 * 128, v_ptr=at, v_row=8 * 128, q=at, q_ld=32 * 128, out=at, out_ld=32 * 128, q_heads=32, scale=0.1, window=0, sinks=0, work=at, work_bytes=1 << 40)
        self.null = set()
        for name, x in changed.items():
            for d in (self.cache, self.batch, self.rotary, self.args):
                if name in d:
                    d[name] = x
                    break
            else:
                assert name in ("no_cache", "no_batch", "no_rotary"), name
                self.null.add(name)
        self.c, self.b, self.r = _lib.PagedCacheC(**self.cache), _lib.PagedBatchC(**self.batch), _lib.RotaryC(**self.rotary)

    def refs(self):
        return (None if "no_cache" in self.null else C.byref(self.c)), (None if "no_batch" in self.null else C.byref(self.b))

    def append(self, lib):
        a = self.args
        return lib.b200_paged_append(*self.refs(), a["k_ptr"], a["k_row"], a["v_ptr"], a["v_row"], a["q"], a["q_ld"], a["out"], a["out_ld"], a["q_heads"], None if "no_rotary" in self.null else C.byref(self.r), None)

    def attend(self, lib):
        a = self.args
        return lib.b200_paged_attention(*self.refs(), a["q"], a["q_ld"], a["out"], a["out_ld"], a["q_heads"], a["scale"], a["window"], a["sinks"], a["work"], a["work_bytes"], None)

    def read(self, lib):
        return lib.b200_paged_read(*self.refs(), self.args["k_ptr"], self.args["v_ptr"], None)

    def bytes(self, lib):
        a = self.args
        return lib.b200_paged_attention_bytes(*self.refs(), a["q_heads"], a["window"], a["sinks"])


def kernels(fake, call, what):
    fake_cuda.launches(fake)
    fake_cuda.check(fake, getattr(call, what)(fake))
    return [(d, next(k for k in ("append_few", "append_many", "read_kernel", "few_rows", "prompt_join", "join_kernel", "prompt_kernel") if k in name)) for d, name in fake_cuda.launches(fake)]


@pytest.mark.parametrize("changed,names", [
    (dict(), ["few_rows", "join_kernel"]),                                                       # decoding
    (dict(sequences=1, total_rows=1, table_width=6), ["few_rows"]),                               # few short units: uncut
    (dict(sequences=64, total_rows=64, table_width=6), ["few_rows", "join_kernel"]),
    (dict(window=512, sinks=4), ["few_rows"]),
    (dict(total_rows=16, max_rows=4), ["few_rows", "join_kernel"]),                               # 16 columns
    (dict(total_rows=20, max_rows=5), ["prompt_kernel", "prompt_join", "few_rows", "join_kernel"]),
    (dict(sequences=1, total_rows=17, max_rows=17), ["prompt_kernel", "prompt_join"]),           # the only sequence goes there with all its rows
    (dict(sequences=1, total_rows=5000, max_rows=5000), ["prompt_kernel"]),
    (dict(sequences=8, total_rows=5000, max_rows=900), ["prompt_kernel", "few_rows", "join_kernel"]),
    (dict(dim=64, q_heads=8, q_ld=512, out_ld=512, total_rows=16, max_rows=16, sequences=1), ["few_rows", "join_kernel"]),
    (dict(total_rows=0), []), (dict(max_rows=0), []),
], ids=str)
@pytest.mark.parametrize("kv_dtype", [_lib.B200_KV_INT8, _lib.B200_KV_FP8_E4M3])
def test_which_kernels_attend(fake, changed, names, kv_dtype):
    assert kernels(fake, Call(kv_dtype=kv_dtype, **changed), "attend") == [(0, n) for n in names]


def test_which_kernels_append_and_read(fake):
    assert kernels(fake, Call(max_rows=16, total_rows=16), "append") == [(0, "append_few")]
    assert kernels(fake, Call(max_rows=17, total_rows=40), "append") == [(0, "append_many")]
    assert kernels(fake, Call(no_rotary=1, q=None, out=None, q_heads=0), "append") == [(0, "append_few")]
    assert kernels(fake, Call(total_rows=0, k_ptr=None), "append") == []
    assert kernels(fake, Call(), "read") == [(0, "read_kernel")]
    assert kernels(fake, Call(total_rows=0), "read") == []


def test_every_page_size_and_head_size_fits_its_blocks(fake):
    for page in (16, 32, 64, 128):
        for dim in (64, 128):
            more = dict(page_tokens=page, dim=dim, k_row=8 * dim, v_row=8 * dim, q_ld=32 * dim, out_ld=32 * dim, rot_dims=dim, total_rows=400, max_rows=100)
            for what in ("append", "attend", "read"):
                assert kernels(fake, Call(**more), what)


def test_the_call_runs_on_the_cache_s_device(fake):
    for what in ("append", "attend", "read"):
        assert {d for d, _ in kernels(fake, Call(device=1), what)} == {1}
    assert {d for d, _ in kernels(fake, Call(device=0), "attend")} == {0}


def test_workspaces(fake):
    """What attention asks for is what it insists on, and calls that need none take none."""
    for changed in (dict(), dict(total_rows=68, max_rows=17), dict(sequences=1, total_rows=17, max_rows=17)):
        n = Call(**changed).bytes(fake)
        assert n > 0
        assert Call(work_bytes=n, **changed).attend(fake) == 0
        assert Call(work_bytes=n - 1, **changed).attend(fake) == _lib.B200_ERR_INVALID and b"workspace" in fake.b200_last_error()
        assert Call(work=None, **changed).attend(fake) == _lib.B200_ERR_INVALID
    for changed in (dict(sequences=1, total_rows=1, table_width=6), dict(total_rows=0), dict(max_rows=0)):
        assert Call(**changed).bytes(fake) == 0 and Call(work=None, work_bytes=0, **changed).attend(fake) == 0
    for changed in (dict(no_cache=1), dict(no_batch=1), dict(q_heads=0), dict(q_heads=12), dict(window=-1), dict(sequences=0)):
        assert Call(**changed).bytes(fake) == 0


ODD = [dict(no_cache=1), dict(no_batch=1), *({n: None} for n in ("k", "v", "k_scale", "v_scale", "flags", "table", "before", "rows")), dict(kv_dtype=0), dict(kv_dtype=3), dict(dim=96), dict(dim=256),
       dict(page_tokens=8), dict(page_tokens=48), dict(page_tokens=256), dict(pages=0), dict(kv_heads=0), dict(kv_heads=2000), dict(pages=2 ** 31 - 1), dict(sequences=0), dict(sequences=1 << 20),
       dict(total_rows=-1), dict(total_rows=(1 << 24) + 1), dict(max_rows=-1), dict(table_width=0), dict(table_ld=63), dict(table_width=2 ** 31 - 1, table_ld=2 ** 40)]


@pytest.mark.parametrize("changed", ODD, ids=str)
def test_caches_and_batches_that_are_refused(fake, changed):
    for what in ("append", "attend", "read"):
        fake_cuda.launches(fake)
        assert getattr(Call(**changed), what)(fake) in (_lib.B200_ERR_INVALID, _lib.B200_ERR_SHAPE), (what, changed)
        assert fake_cuda.launches(fake) == [] and fake.b200_last_error()


@pytest.mark.parametrize("changed", [dict(q=None), dict(out=None), dict(q_ld=4095), dict(q_ld=4000), dict(out_ld=100), dict(out_ld=4100), dict(q_heads=12), dict(q_heads=4), dict(q_heads=0), dict(q_heads=8 * 300),
                                     dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(window=-1), dict(sinks=-1)], ids=str)
def test_attention_calls_that_are_refused(fake, changed):
    fake_cuda.launches(fake)
    assert Call(**changed).attend(fake) in (_lib.B200_ERR_INVALID, _lib.B200_ERR_SHAPE)
    assert fake_cuda.launches(fake) == []


@pytest.mark.parametrize("changed", [dict(k_ptr=None), dict(v_ptr=None), dict(k_row=1000), dict(v_row=1027), dict(out=None), dict(q_ld=4000), dict(q_heads=0), dict(q_heads=9000), dict(turns=None), dict(rot_dims=8),
                                     dict(rot_dims=24), dict(rot_dims=144), dict(pairing=2)], ids=str)
def test_append_calls_that_are_refused(fake, changed):
    fake_cuda.launches(fake)
    assert Call(**changed).append(fake) == _lib.B200_ERR_INVALID
    assert fake_cuda.launches(fake) == []


def test_pointers_off_a_16_byte_border_are_refused(fake):
    at = Call().args["q"]
    for name in ("k", "v"):
        for what in ("append", "attend", "read"):
            c = Call(**{name: at + 8})
            assert getattr(c, what)(fake) == _lib.B200_ERR_INVALID
    assert Call(q=at + 2).attend(fake) == _lib.B200_ERR_INVALID and Call(out=at + 8).attend(fake) == _lib.B200_ERR_INVALID and Call(work=at + 4).attend(fake) == _lib.B200_ERR_INVALID
    assert Call(k_ptr=at + 2).append(fake) == _lib.B200_ERR_INVALID and Call(v_ptr=at + 8).read(fake) == _lib.B200_ERR_INVALID


def test_python_refuses_what_is_not_on_a_gpu():
    i32 = dict(dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA device"):
        paged.PagedBatch(torch.zeros(1, 2, **i32), torch.zeros(1, **i32), torch.zeros(2, **i32), 1)
    with pytest.raises(RuntimeError, match="CUDA device only"):
        paged.PagedKVCache(4, 2, 128, device="cpu")
    with pytest.raises(ValueError, match="one CUDA device"):
        paged.PagedKVCache.from_tensors(torch.zeros(2, 2, 16, 64, dtype=torch.int8), torch.zeros(2, 2, 16, 64, dtype=torch.int8), torch.zeros(2, 2), torch.zeros(2, 2))
    with pytest.raises(ValueError, match="dtype"):
        paged.PagedKVCache(4, 2, 128, dtype="bf16")
    for args in (dict(rot_dims=8), dict(rot_dims=40), dict(rot_dims=64, pairing="thirds"), dict(rot_dims=64, freqs=[1.0])):
        with pytest.raises(ValueError):
            paged.RotaryTable(**args)


def test_turns_are_exact_to_64_bits():
    decimal.getcontext().prec = 80
    two_pi = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803482534211706798")
    for f in (1.0, 0.5, 10000.0 ** (-2 / 128), 1e-4, 1e-9, 3.0, 100.0):
        (turn,) = paged.turns_of([f])
        want = decimal.Decimal(f) / two_pi
        want -= int(want)
        assert abs(decimal.Decimal(turn) - want * 2 ** 64) <= 1, f


# ---- the oracle's own properties ----
@pytest.mark.parametrize("dtype", ["int8", "fp8_e4m3"])
@pytest.mark.parametrize("growth", [1.001, 1.1, 2.5])
def test_pages_that_only_double_their_scale_stay_within_a_step(dtype, growth):
    """Half a step from the first rounding, and after k doublings halves of older ones: 1/2 + 1/4 + ... of the last step."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 16, generator=g, dtype=torch.float64) * growth ** torch.arange(40.0)[:, None]
    codes, scale = torch.zeros(64, 16, dtype=torch.float64), 0.0
    for i in range(40):
        codes, scale = oracle.append(codes, scale, i, x[i:i + 1], dtype)
    off = (codes[:40] * scale - x).abs()
    assert bool((off <= (scale if dtype == "int8" else 2.0 ** -4 * x.abs() * (1 + 2.0 ** -6) + 2.0 ** -9 * scale)).all())
    again = oracle.append(codes, scale, 39, x[39:], dtype)
    assert torch.equal(again[0], codes) and again[1] == scale


def test_growing_to_the_exact_maximum_would_drift():
    """Why scales double: each time a little more, the roundings of a code all have the same sign."""
    top, codes, scale = 1.0, torch.tensor([127.0], dtype=torch.float64), 1.0 / 127
    for i in range(1, 64):
        now = 1.001 ** i / 127
        codes, scale = (codes * scale / now).round(), now
    assert float((codes * scale - top).abs()) > 6 * scale


def test_visible_tokens():
    pos = torch.tensor([0, 5, 9])
    assert oracle.visible(pos, 10, 3, 2).tolist() == [[j <= p and (p - j < 3 or j < 2) for j in range(10)] for p in (0, 5, 9)]
    assert oracle.visible(pos, 10, 0, 4).tolist() == [[j <= p for j in range(10)] for p in (0, 5, 9)]


def test_attention_of_the_oracle_against_softmax():
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, 64, generator=g, dtype=torch.float64) for n, h in ((3, 4), (20, 2), (20, 2)))
    out, tol = oracle.attend(q, k, v, v.abs().amax(-1), 17, 0.125, 6, 2)
    for i in range(3):
        for h in range(4):
            keep = [j for j in range(18 + i) if 17 + i - j < 6 or j < 2]
            w = torch.softmax(k[keep, h // 2] @ q[i, h] * 0.125, 0)
            assert torch.allclose(out[i, h], w @ v[keep, h // 2], atol=1e-12)
    assert bool((tol > 0).all())
