"""A paged cache of keys and values in 8 bits, with what reads and writes it (``b200_paged_*``).

``PagedKVCache`` owns the pages of one layer; ``PagedBatch`` describes a step, which all layers share: which rows belong to which sequence, how many tokens each has cached,
and its table of pages; ``RotaryTable`` holds the position rotation.  A layer's step is ``append`` (rotates and stores) and then ``attend``::

    batch = PagedBatch(table, before, rows, total_rows, max_rows)
    q = cache.append(batch, k, v, q=q, rotary=rotary)
    out = cache.attend(batch, q, window=4096, sinks=4)

Drafted tokens are checked as a tree (``PagedTree``): append at its positions, attend with its masks, and keep the accepted path; ``PagePool`` keeps account of who holds which pages, on the device, for
forks, beams and requests that come and go::

    pool = PagePool(caches, sequences, width)              # the caches of all layers
    pool.reserve(add)                                      # pages for the step's rows
    batch = PagedBatch(pool.table, pool.lengths, rows, total_rows, max_rows)
    tree = PagedTree(batch, parents)
    for cache in caches:
        q = cache.append(batch, k, v, q=q, rotary=rotary, positions=tree.positions)
        out = cache.attend(batch, q, tree=tree)
    pool.keep(batch, kept, counts)
    pool.lengths += counts

The calls enqueue on the current stream and wait for nothing, so that they may be captured into a graph.  They are for inference: there are no gradients, and inputs that ask for
one are refused.  Pages are handed out by the caller or a pool; a page that is written to must belong to one sequence of the batch only (pages that are only read may be shared).  A step
of prompts and single rows is quicker as two batches over the same tensors, ``PagedBatch(table[:n], before[:n], rows[:n + 1], ...)`` and ``PagedBatch(table[n:], before[n:], rows[n:],
...)``, each with its own ``max_rows``: the other's rows belong to nobody and are left as they are.
"""
from __future__ import annotations

import ctypes as C
import typing as tp

import torch

from .. import _lib
from ..config import ROT_PAIRINGS

_KV = {"int8": (torch.int8, _lib.B200_KV_INT8), "fp8_e4m3": (torch.float8_e4m3fn, _lib.B200_KV_FP8_E4M3)}
_NAMES = {dtype: name for name, (dtype, _) in _KV.items()}
# floor(2^192 / (2 pi))
_TURN = (1 << 192) * 10 ** 60 // (2 * 3141592653589793238462643383279502884197169399375105820974944)
BAD_BATCH, BAD_PAGE, NOT_FINITE, WAIT, BAD_TREE, NO_PAGES = 1, 2, 4, 8, 16, 32
MAX_NODES = 1024                                # of a tree
MAX_AXES = 4
_OVER = "the cache's keys, values and scales lie over one another: what is written to one would change another"


def _cuda(device: torch.device | str) -> torch.device:
    device = torch.device(device)
    if device.type != "cuda":
        raise RuntimeError("the paged cache lives on a CUDA device only (no CPU fallback)")
    return torch.device("cuda", torch.cuda.current_device()) if device.index is None else device


# the current stream's handle: a microsecond less without the object around it
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _entry(name: str):
    fn = getattr(_lib.lib(), name, None)
    if fn is None:
        raise RuntimeError(f"this build of the library has no {name}; build all of it with `python -m moshi_b200.build`")
    return fn


def _apart(tensors: tp.Iterable[torch.Tensor]) -> bool:
    """Whether no byte belongs to two of these contiguous tensors."""
    ranges = sorted((t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors)
    return all(a[1] <= b[0] for a, b in zip(ranges, ranges[1:]))


class _Fixed:
    """Attributes whose addresses the library has: once set, they take nothing but the same tensor back, as ``pool.lengths += counts`` gives it.  Another tensor would not be looked at, and the first one's memory
    would be somebody else's."""
    _fixed: tp.ClassVar[frozenset[str]] = frozenset()

    def __setattr__(self, name: str, value: tp.Any) -> None:
        if name in self._fixed and self.__dict__.get(name, value) is not value:
            raise AttributeError(f"{type(self).__name__}.{name} stays the tensor that it is: write into it (copy_, +=)")
        object.__setattr__(self, name, value)


def turns_of(freqs: tp.Iterable[float]) -> list[int]:
    """Turns per position, of frequencies in radians, as fractions of 2^64: the product with a position drops whole turns and nothing else."""
    return [((num * _TURN // den + (1 << 127)) >> 128) % (1 << 64) for num, den in (f.as_integer_ratio() for f in freqs)]


class RotaryTable(_Fixed):
    """Frequencies of a position rotation: ``base ** (-2 j / rot_dims)`` radians per position for the pair j, or ``freqs`` (rot_dims / 2 numbers).  ``pairing``: "adjacent" turns
    dimensions (2j, 2j + 1), "halves" (j, j + rot_dims / 2); dimensions from ``rot_dims`` on stay as they are.  ``axes``: for each pair the axis (0 .. 3) whose position turns it, where rows have positions of
    several (time, height, width); those are given to every ``append``."""
    _fixed = frozenset(("turns", "pair_axis"))

    def __init__(self, rot_dims: int, base: float = 10000.0, pairing: str = "adjacent", freqs: tp.Sequence[float] | None = None, device: torch.device | str = "cuda",
                 axes: tp.Sequence[int] | None = None):
        if rot_dims < 16 or rot_dims % 16:
            raise ValueError(f"rot_dims {rot_dims}: a multiple of 16")
        if pairing not in ROT_PAIRINGS:
            raise ValueError(f"pairing {pairing!r}: one of {sorted(ROT_PAIRINGS)}")
        freqs = [base ** (-2.0 * j / rot_dims) for j in range(rot_dims // 2)] if freqs is None else [float(f) for f in freqs]
        if len(freqs) != rot_dims // 2:
            raise ValueError(f"{len(freqs)} frequencies for {rot_dims} dimensions")
        axes = [0] * len(freqs) if axes is None else [int(a) for a in axes]
        if len(axes) != len(freqs) or min(axes) < 0 or max(axes) >= MAX_AXES:
            raise ValueError(f"axes {axes}: one of 0 .. {MAX_AXES - 1} for each of {len(freqs)} pairs")
        turns = turns_of(freqs)
        self.device = _cuda(device)
        self.rot_dims, self.pairing = rot_dims, pairing
        self.turns = torch.tensor([t - (1 << 64) if t >> 63 else t for t in turns], dtype=torch.int64, device=self.device)
        self._c = _lib.RotaryC(self.turns.data_ptr(), rot_dims, ROT_PAIRINGS[pairing])
        self._ref = C.addressof(self._c)
        self.axes = max(axes) + 1
        self.pair_axis = torch.tensor(axes, dtype=torch.uint8, device=self.device) if self.axes > 1 else None


class PagedBatch(_Fixed):
    """One step.  ``table`` i32 [sequences, pages]: where a sequence's tokens lie; ``before`` i32 [sequences]: tokens that it has cached in front of the step; ``rows`` i32
    [sequences + 1]: sequence s adds rows[s] .. rows[s + 1] - 1 (none, one or many) of the step's ``total_rows``.  ``max_rows``: the most that any of them adds.  The work is laid
    out by it, and a sequence with more is left out; without it (``total_rows``) a step of many sequences takes longer than it has to (48 of one row each: attention 1.4 times, append 2.5 to 3.7
    times as long).  The tensors stay where they are and may be refilled between steps of a captured graph."""
    _fixed = frozenset(("table", "before", "rows"))

    def __init__(self, table: torch.Tensor, before: torch.Tensor, rows: torch.Tensor, total_rows: int, max_rows: int | None = None):
        for name, t, dims in (("table", table, 2), ("before", before, 1), ("rows", rows, 1)):
            if t.dtype != torch.int32 or t.dim() != dims or t.device.type != "cuda" or t.device != table.device:
                raise ValueError(f"{name}: i32, {dims} dimension(s), on the table's CUDA device; got {t.dtype}, {tuple(t.shape)}, {t.device}")
        S = before.shape[0]
        if S < 1 or table.shape[0] != S or table.shape[1] < 1 or rows.shape[0] != S + 1:
            raise ValueError(f"table {tuple(table.shape)}, before {tuple(before.shape)}, rows {tuple(rows.shape)} do not describe the same sequences")
        if before.stride(0) != 1 and S > 1 or rows.stride(0) != 1 or table.stride(1) != 1 and table.shape[1] > 1 or table.stride(0) < table.shape[1] and S > 1:
            raise ValueError("table, before and rows have to be dense along their last dimension, tables apart from one another")
        total_rows = int(total_rows)
        max_rows = total_rows if max_rows is None else int(max_rows)
        if not 0 <= total_rows <= 1 << 24 or not 0 <= max_rows:
            raise ValueError(f"total_rows {total_rows}, max_rows {max_rows}")
        self.table, self.before, self.rows, self.total_rows, self.max_rows = table, before, rows, total_rows, min(max_rows, total_rows)
        self.device, self.sequences = table.device, S
        self._index, self._work = table.device.index, {}
        self._c = _lib.PagedBatchC(table.data_ptr(), before.data_ptr(), rows.data_ptr(), max(table.stride(0), table.shape[1]), S, table.shape[1], total_rows, self.max_rows)
        self._ref = C.addressof(self._c)


class PagedTree(_Fixed):
    """The rows of a batch as trees of drafted tokens.  ``parents`` i32 [total_rows]: row i of a sequence comes behind its row parents[rows[s] + i], which has a lower number, or, -1, behind the last cached token; a
    parent that is neither counts as -1 and is recorded.  At most 1024 rows of a sequence.  A row's position is before + depth (``positions`` i32 [total_rows], for ``append``); it sees what
    is cached, itself and those that it comes behind (``seen`` i32 [total_rows, words], bit i for the sequence's row i).  All layers of a step share a tree; once ``parents`` or the batch's tensors have been refilled,
    ``update`` fills it anew on the current stream."""
    _fixed = frozenset(("batch", "seen", "positions", "flags"))

    def __init__(self, batch: PagedBatch, parents: torch.Tensor):
        if batch.max_rows > MAX_NODES:
            raise ValueError(f"trees of up to {batch.max_rows} rows: {MAX_NODES} at most")
        words = max(1, -(-batch.max_rows // 32))
        self.batch, self.parents = batch, parents
        self.seen = torch.zeros(batch.total_rows, words, dtype=torch.int32, device=batch.device)
        self.positions = torch.zeros(batch.total_rows, dtype=torch.int32, device=batch.device)
        self.flags = torch.zeros(1, dtype=torch.int32, device=batch.device)
        self._c = _lib.PagedTreeC(self.seen.data_ptr(), self.positions.data_ptr(), words)
        self._ref = C.addressof(self._c)
        self._build = _entry("b200_paged_tree_build")
        self.update()

    @property
    def parents(self) -> torch.Tensor:
        return self._parents

    @parents.setter
    def parents(self, t: torch.Tensor) -> None:
        rows, device = self.batch.total_rows, self.batch.device
        if t.dtype != torch.int32 or t.shape != (rows,) or t.device != device or (t.numel() > 1 and t.stride(0) != 1):
            raise ValueError(f"parents: i32 [{rows}], dense, on {device}; got {t.dtype}, {tuple(t.shape)}, {t.device}")
        self._parents = t

    def update(self) -> None:
        rc = self._build(self.batch._ref, self._ref, self.parents.data_ptr(), self.flags.data_ptr(), self.batch._index, _stream(self.batch._index)) if self.batch.total_rows else 0
        if rc:
            _lib.check(rc)

    def error_flags(self) -> int:
        """BAD_BATCH, BAD_TREE of updates since the last ``clear_error_flags``.  Waits for all streams of the device."""
        torch.cuda.synchronize(self.batch.device)
        return int(self.flags.item())

    def clear_error_flags(self) -> None:
        """Behind what the current stream has been given, and before what it is given next."""
        self.flags.zero_()


class PagedKVCache(_Fixed):
    """The pages of one layer: ``k``, ``v`` [pages, kv_heads, page_tokens, head_dim] int8 or float8_e4m3fn, with ``k_scale``, ``v_scale`` f32 [pages, kv_heads]; a code stands for
    code * scale.  A new cache's content is arbitrary: what no append has written is never looked at."""
    _fixed = frozenset(("k", "v", "k_scale", "v_scale", "flags"))

    def __init__(self, pages: int, kv_heads: int, head_dim: int, page_tokens: int = 64, dtype: str = "int8", device: torch.device | str = "cuda"):
        if dtype not in _KV:
            raise ValueError(f"dtype {dtype!r}: one of {sorted(_KV)}")
        device = _cuda(device)
        if pages < 1 or kv_heads < 1:
            raise ValueError(f"{pages} pages, {kv_heads} heads")
        shape = (pages, kv_heads, page_tokens, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.int8, device=device).view(_KV[dtype][0]) for _ in range(2))
        self._take(k, v, *(torch.zeros(pages, kv_heads, dtype=torch.float32, device=device) for _ in range(2)))

    @classmethod
    def from_tensors(cls, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor) -> "PagedKVCache":
        """A cache in the caller's memory.  Scales of pages in use lie within 2^-60 .. 2^58; where one is 0, all codes of that page and head are 0.  Tensors that lie over one another can be read, and not written
        to (``append``, ``keep``, a pool)."""
        self = cls.__new__(cls)
        self._take(k, v, k_scale, v_scale)
        return self

    def _take(self, k, v, k_scale, v_scale) -> None:
        if k.dtype not in _NAMES or v.dtype != k.dtype or k.dim() != 4 or v.shape != k.shape or k_scale.shape != k.shape[:2] or v_scale.shape != k.shape[:2] or \
                k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise ValueError("k and v: int8 or float8_e4m3fn [pages, kv_heads, page_tokens, head_dim]; their scales: f32 [pages, kv_heads]")
        if k.shape[2] not in (16, 32, 64, 128) or k.shape[3] not in (64, 128):
            raise ValueError(f"pages of {k.shape[2]} tokens (16, 32, 64 or 128), head size {k.shape[3]} (64 or 128)")
        for t in (k, v, k_scale, v_scale):
            if t.device != k.device or t.device.type != "cuda" or not t.is_contiguous():
                raise ValueError("a cache's tensors are contiguous and on one CUDA device")
        self.k, self.v, self.k_scale, self.v_scale, self.device = k, v, k_scale, v_scale, k.device
        self.pages, self.kv_heads, self.page_tokens, self.head_dim = k.shape
        self.dtype = _NAMES[k.dtype]
        self._index, self._shape = self.device.index, (self.page_tokens, self.kv_heads, self.head_dim)
        self._own = _apart(self._tensors())
        self.flags = torch.zeros(1, dtype=torch.int32, device=self.device)
        self._c = _lib.PagedCacheC(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), self.flags.data_ptr(), self.pages, self.page_tokens, self.kv_heads, self.head_dim, _KV[self.dtype][1], self.device.index)
        self._ref = C.addressof(self._c)
        self._append, self._attend, self._bytes, self._read = (_entry(f"b200_paged_{n}") for n in ("append", "attention", "attention_bytes", "read"))
        self._append_at, self._attend_tree, self._tree_bytes, self._keep = (_entry(f"b200_paged_{n}") for n in ("append_at", "tree_attention", "tree_attention_bytes", "keep"))

    def _tensors(self) -> tuple[torch.Tensor, ...]:
        return self.k, self.v, self.k_scale, self.v_scale

    def _rows(self, name: str, t: torch.Tensor, batch: PagedBatch, heads: int) -> int:
        """Checks a step's tensor [total_rows, heads, head_dim]; its elements from row to row."""
        T, D = batch.total_rows, self.head_dim
        if t.dtype is not torch.bfloat16 or t.shape != (T, heads, D):
            raise ValueError(f"{name}: bf16 {[T, heads, D]}; got {t.dtype} {list(t.shape)}")
        if t.get_device() != self._index or batch._index != self._index:
            raise ValueError(f"{name} on {t.device}, the batch on {batch.device}, the cache on {self.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} asks for a gradient: the paged cache has none")
        ld, head, one = t.stride()
        if one != 1 or (head != D and heads > 1):
            raise ValueError(f"{name}: a row's heads have to lie side by side; strides {t.stride()}")
        return ld if T > 1 else heads * D

    def _heads(self, name: str, t: torch.Tensor) -> int:
        if t.dim() != 3:
            raise ValueError(f"{name}: [total_rows, heads, head_dim]; got {list(t.shape)}")
        return t.shape[1]

    def append(self, batch: PagedBatch, k: torch.Tensor, v: torch.Tensor, q: torch.Tensor | None = None, rotary: RotaryTable | None = None,
               q_out: torch.Tensor | None = None, positions: torch.Tensor | None = None) -> torch.Tensor | None:
        """Stores the step's keys and values, bf16 [total_rows, kv_heads, head_dim] (rows may lie apart, as in a projection of all three), keys rotated by their positions.  Returns
        the queries ``q`` [total_rows, q_heads, head_dim] rotated likewise, in ``q_out`` (which may be ``q``) or a new tensor.  ``positions`` i32 [total_rows] or [axes, total_rows]: positions of the rows' own
        for the rotation, as a tree's tokens have (``PagedTree.positions``) or an image's patches; where a row is stored does not go by them."""
        if not self._own:
            raise ValueError(_OVER)
        k_ld, v_ld = self._rows("k", k, batch, self.kv_heads), self._rows("v", v, batch, self.kv_heads)
        if rotary is not None and (rotary.device != self.device or rotary.rot_dims > self.head_dim):
            raise ValueError(f"{rotary.rot_dims} rotated dimensions on {rotary.device} for heads of {self.head_dim} on {self.device}")
        q_ptr = q_ld = o_ptr = o_ld = heads = 0
        if q is not None:
            heads = self._heads("q", q)
            q_ld = self._rows("q", q, batch, heads)
            if q_out is None:
                q_out, o_ld = q.new_empty(q.shape), heads * self.head_dim
            else:
                o_ld = self._rows("q_out", q_out, batch, heads)
            q_ptr, o_ptr = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        if positions is not None:
            at = self._positions(batch, rotary, positions)
            rc = self._append_at(self._ref, batch._ref, k.data_ptr(), k_ld, v.data_ptr(), v_ld, q_ptr, q_ld, o_ptr, o_ld, heads, rotary._ref, C.addressof(at), _stream(self._index))
        elif rotary is not None and rotary.axes > 1:
            raise ValueError(f"a rotation of {rotary.axes} axes needs the rows' positions")
        else:
            rc = self._append(self._ref, batch._ref, k.data_ptr(), k_ld, v.data_ptr(), v_ld, q_ptr, q_ld, o_ptr, o_ld, heads, rotary._ref if rotary is not None else None,
                              _stream(self._index))
        if rc:
            _lib.check(rc)
        return q_out

    def _positions(self, batch: PagedBatch, rotary: RotaryTable | None, t: torch.Tensor) -> _lib.PagedPositionsC:
        if rotary is None:
            raise ValueError("positions without a rotary table")
        if t.dim() == 1 and rotary.axes == 1:
            t = t[None]
        if t.dtype is not torch.int32 or t.shape != (rotary.axes, batch.total_rows) or t.get_device() != self._index or (t.shape[1] > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
            raise ValueError(f"positions: i32 {[rotary.axes, batch.total_rows]}, dense along the rows, on {self.device}; got {t.dtype} {list(t.shape)}, strides {t.stride()}, {t.device}")
        return _lib.PagedPositionsC(t.data_ptr(), max(t.stride(0), batch.total_rows), rotary.pair_axis.data_ptr() if rotary.pair_axis is not None else None, rotary.axes)

    def attend(self, batch: PagedBatch, q: torch.Tensor, scale: float | None = None, window: int = 0, sinks: int = 0, out: torch.Tensor | None = None,
               tree: PagedTree | None = None) -> torch.Tensor:
        """Attention of the step's rows over what their sequences have cached, the step's own rows included (``append`` comes first): the row at position p sees tokens j <= p
        and, with a ``window``, of these only p - j < window and the first ``sinks`` tokens.  q bf16 [total_rows, q_heads, head_dim], q_heads a multiple of kv_heads; scores are
        multiplied by ``scale`` > 0 (default head_dim ** -0.5).  With a ``tree`` of this batch a row sees what is cached in front of the step and, of the step's rows, itself and those that it comes behind; window and
        first tokens then go by the tree's positions.  Rows that belong to no sequence are left as they are in ``out``; a query that is not finite gives NaN in its own row and head."""
        heads = self._heads("q", q)
        q_ld = self._rows("q", q, batch, heads)
        if out is None:
            out, o_ld = q.new_empty(q.shape), heads * self.head_dim
        else:
            o_ld = self._rows("out", out, batch, heads)
        if not 0 <= window < 1 << 31 or not 0 <= sinks < 1 << 31:
            raise ValueError(f"window {window}, {sinks} first tokens")
        if tree is not None and tree.batch is not batch:
            raise ValueError("the tree is of another batch")
        of = (self._shape, heads, window, sinks, tree is None)
        n = batch._work.get(of)                       # a size, by sizes alone; the layers of a step ask for the same
        if n is None:
            n = batch._work[of] = (self._bytes if tree is None else self._tree_bytes)(self._ref, batch._ref, heads, window, sinks)
        work = q.new_empty((n + 1) // 2) if n else None
        if tree is not None:
            rc = self._attend_tree(self._ref, batch._ref, tree._ref, q.data_ptr(), q_ld, out.data_ptr(), o_ld, heads, self.head_dim ** -0.5 if scale is None else scale, window, sinks,
                                   work.data_ptr() if n else None, n, _stream(self._index))
            if rc:
                _lib.check(rc)
            return out
        rc = self._attend(self._ref, batch._ref, q.data_ptr(), q_ld, out.data_ptr(), o_ld, heads, self.head_dim ** -0.5 if scale is None else scale, window, sinks,
                          work.data_ptr() if n else None, n, _stream(self._index))
        if rc:
            _lib.check(rc)
        return out

    def read(self, batch: PagedBatch) -> tuple[torch.Tensor, torch.Tensor]:
        """What the cache holds at the batch's positions ``before[s] + i``: keys and values bf16 [total_rows, kv_heads, head_dim].  Rows that belong to no sequence hold anything."""
        if batch._index != self._index:
            raise ValueError(f"the batch on {batch.device}, the cache on {self.device}")
        k, v = (torch.empty(batch.total_rows, self.kv_heads, self.head_dim, dtype=torch.bfloat16, device=self.device) for _ in range(2))
        rc = self._read(self._ref, batch._ref, k.data_ptr(), v.data_ptr(), _stream(self._index))
        if rc:
            _lib.check(rc)
        return k, v

    def keep(self, batch: PagedBatch, kept: torch.Tensor, counts: torch.Tensor) -> None:
        """Of the step's rows sequence s keeps counts[s] (i32 [sequences]), those of the numbers kept[rows[s]], kept[rows[s] + 1], .. (i32 [total_rows]) among its own, which rise: the accepted path of a
        tree.  They move to the places from before[s] on, and what lies behind them is of no use any more.  Codes move as they are within a page; to another page's scale they are rounded once more."""
        if not self._own:
            raise ValueError(_OVER)
        _keep([self], self._ref, 1, batch, kept, counts)

    def error_flags(self) -> int:
        """What the kernels found wrong since the last ``clear_error_flags``: BAD_BATCH, BAD_PAGE, NOT_FINITE, WAIT.  Waits for all streams of the device."""
        torch.cuda.synchronize(self.device)
        return int(self.flags.item())

    def clear_error_flags(self) -> None:
        """Behind what the current stream has been given, and before what it is given next."""
        self.flags.zero_()


def _keep(caches: tp.Sequence[PagedKVCache], ref, n: int, batch: PagedBatch, kept: torch.Tensor, counts: torch.Tensor) -> None:
    cache = caches[0]
    for name, t, size in (("kept", kept, batch.total_rows), ("counts", counts, batch.sequences)):
        if t.dtype is not torch.int32 or t.shape != (size,) or t.get_device() != cache._index or (size > 1 and t.stride(0) != 1):
            raise ValueError(f"{name}: i32 [{size}], dense, on {cache.device}; got {t.dtype} {list(t.shape)}, {t.device}")
    if batch._index != cache._index:
        raise ValueError(f"the batch on {batch.device}, the cache on {cache.device}")
    rc = cache._keep(ref, n, batch._ref, kept.data_ptr(), counts.data_ptr(), _stream(cache._index))
    if rc:
        _lib.check(rc)


class PagePool(_Fixed):
    """Who holds which pages, on the device, for sequences whose tokens lie in ``caches`` (one per layer, alike).  ``table`` i32 [sequences, width], -1 behind what a sequence holds; ``lengths`` i32 [sequences]: tokens that
    it has (the caller's to raise in place, by what a step has left, or to lower, before a ``rearrange`` that gives back what lies behind); ``held``: pages that it holds, enough for them; ``refs`` i32 [pages]: sequences that hold a page.  A pool begins empty.  ``table`` and
    ``lengths`` are what a ``PagedBatch`` takes.  The calls may be captured; none waits."""
    _fixed = frozenset(("table", "lengths", "held", "refs", "flags", "caches"))

    def __init__(self, caches: tp.Sequence[PagedKVCache], sequences: int, width: int):
        caches = tuple(caches)
        if not caches or any((c.device, c.pages, c._shape, c.dtype) != (caches[0].device, caches[0].pages, caches[0]._shape, caches[0].dtype) for c in caches):
            raise ValueError("a pool's caches are alike: device, pages, sizes and type")
        if not _apart(t for c in caches for t in c._tensors()):
            raise ValueError("a pool's caches have memory of their own: what moves in one would move twice")
        if not 1 <= sequences <= 4096 or width < 1:
            raise ValueError(f"{sequences} sequences (1 .. 4096) of {width} pages")
        self.caches, self.device, self.sequences, self.width, self.pages = caches, caches[0].device, int(sequences), int(width), caches[0].pages
        i32 = dict(dtype=torch.int32, device=self.device)
        self.table = torch.full((sequences, width), -1, **i32)
        self.lengths, self.held, self.refs, self.flags = (torch.zeros(n, **i32) for n in (sequences, sequences, self.pages, 1))
        self._c = _lib.PagePoolC(self.table.data_ptr(), self.lengths.data_ptr(), self.held.data_ptr(), self.refs.data_ptr(), self.flags.data_ptr(), width, sequences, width, self.pages,
                                 caches[0].page_tokens, self.device.index)
        self._ref, self._index = C.addressof(self._c), self.device.index
        self._of = (_lib.PagedCacheC * len(caches))(*(c._c for c in caches))
        self._caches = C.addressof(self._of)
        self._rearrange, self._reserve, self._compact = (_entry(f"b200_page_pool_{n}") for n in ("rearrange", "reserve", "compact"))
        self._bytes = _entry("b200_page_pool_bytes")(self._ref)

    def _work(self) -> torch.Tensor:
        return torch.empty(self._bytes, dtype=torch.uint8, device=self.device)

    def _of_sequences(self, name: str, t: torch.Tensor) -> int:
        if t.dtype is not torch.int32 or t.shape != (self.sequences,) or t.get_device() != self._index or (self.sequences > 1 and t.stride(0) != 1):
            raise ValueError(f"{name}: i32 [{self.sequences}], dense, on {self.device}; got {t.dtype} {list(t.shape)}, {t.device}")
        return t.data_ptr()

    def rearrange(self, source: torch.Tensor) -> None:
        """All at once, sequence i becomes what sequence source[i] was (i32 [sequences]), -1: empty.  Forks requests (their pages are shared), moves beams, gives pages back; so are pages that were held in reserve.
        A sequence whose length is negative or more than its pages take counts as empty: it gives all of its pages back, and BAD_BATCH is recorded."""
        at, work = self._of_sequences("source", source), self._work()
        rc = self._rearrange(self._ref, at, work.data_ptr(), self._bytes, _stream(self._index))
        if rc:
            _lib.check(rc)

    def reserve(self, add: torch.Tensor) -> None:
        """Pages for add[s] tokens (i32 [sequences]) behind the lengths[s] that sequence s has: by rising numbers, to sequences by rising numbers.  Where the next token goes to a partly filled page that others hold too, the
        sequence gets a copy of it first, in all caches (of those in this call that share it, the last keeps it if nobody else holds it).  A sequence whose pages behind its tokens are shared (it was made shorter without a ``rearrange``)
        is left out, and BAD_BATCH is recorded.  With too few free pages nobody gets any, and NO_PAGES is recorded: what the step would write to may be shared still."""
        at, work = self._of_sequences("add", add), self._work()
        rc = self._reserve(self._ref, self._caches, len(self.caches), at, work.data_ptr(), self._bytes, _stream(self._index))
        if rc:
            _lib.check(rc)

    def compact(self) -> None:
        """Moves the pages in use to the lowest numbers, in all caches."""
        work = self._work()
        rc = self._compact(self._ref, self._caches, len(self.caches), work.data_ptr(), self._bytes, _stream(self._index))
        if rc:
            _lib.check(rc)

    def keep(self, batch: PagedBatch, kept: torch.Tensor, counts: torch.Tensor) -> None:
        """``PagedKVCache.keep`` in all caches at once; what is found wrong is recorded in the first one's flags.  ``lengths`` stay as they are."""
        _keep(self.caches, self._caches, len(self.caches), batch, kept, counts)

    def error_flags(self) -> int:
        """BAD_BATCH, BAD_PAGE, NO_PAGES of calls since the last ``clear_error_flags``.  Waits for all streams of the device."""
        torch.cuda.synchronize(self.device)
        return int(self.flags.item())

    def clear_error_flags(self) -> None:
        """Behind what the current stream has been given, and before what it is given next."""
        self.flags.zero_()
