"""Calls around drafted trees on the paged 8-bit cache: attention of trees of tokens, keys and queries turned by positions of their own on one or several axes, the accepted
path's move to the front, and the pages of a pool: forks with copies on write, beams that change places, requests that leave and the rest that moves together.

``listed()`` names cases over the range of uses, ``draw()`` gives more of them, ``run()`` makes one pass: the plain form in elementary torch operations, or, where ``own`` is
true, the calls of ``moshi_b200.models``: ``PagedKVCache``, ``PagedTree``, ``RotaryTable``, ``PagePool``.
"""
import math

import torch

own = False

SCALE_MIN = 2.0 ** -60
Q_MAX = {"int8": 127.0, "fp8_e4m3": 448.0}
CODES = {"int8": torch.int8, "fp8_e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------------------------------------------------------------
# cases.  kind: what is called; seqs: sequences; before_min .. before_max: tokens that they have cached (spread over the logarithm); new_min .. new_max: rows that each of
# them adds; q_heads / kv_heads / dim; page: tokens of a page; layers: caches that share the pages; axes: of the positions; group: sequences that are beams of one request
# ------------------------------------------------------------------------------------------------------------------------
def _case(kind, seqs, before, new, heads, dim, page, dtype, window=0, sinks=0, pairing="adjacent", layers=1, axes=1, group=1):
    return {"kind": kind, "seqs": seqs, "before_min": before[0], "before_max": before[1], "new_min": new[0], "new_max": new[1], "q_heads": heads[0], "kv_heads": heads[1],
            "dim": dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "pairing": pairing, "layers": layers, "axes": axes, "group": group}


def listed():
    return [
        # one young session checks a small tree, every head with keys of its own: the call's latency
        {"name": "tree, one young session", **_case("tree", 1, (374, 374), (8, 8), (32, 32), 128, 64, "int8")},
        # continuous batching with drafts: trees of about thirty tokens, grouped heads
        {"name": "tree, 16 requests", **_case("tree", 16, (1000, 6000), (25, 32), (32, 8), 128, 64, "int8")},
        # a box of dialogue sessions, a dozen drafted tokens each: the cache's bytes
        {"name": "tree, 48 sessions", **_case("tree", 48, (1000, 2980), (12, 12), (32, 32), 128, 64, "fp8_e4m3")},
        # one long document and a wide tree: little to share out but the length
        {"name": "tree, one long request", **_case("tree", 1, (131000, 131000), (64, 64), (32, 8), 128, 128, "int8")},
        # endless dialogues under a window, narrow heads, small pages, trees of very different size
        {"name": "tree, narrow heads, window", **_case("tree", 24, (100, 20000), (5, 48), (24, 4), 64, 16, "fp8_e4m3", window=1024, sinks=4)},
        # prompts with images: rows at (time, height, width), pairs dealt out in turn
        {"name": "positions, three axes", **_case("positions", 4, (0, 700), (900, 2500), (32, 8), 128, 64, "int8", pairing="halves", axes=3)},
        # a few rows of many requests at places of two axes
        {"name": "positions, 32 requests", **_case("positions", 32, (40, 3000), (8, 8), (24, 4), 64, 32, "fp8_e4m3", axes=2)},
        # the accepted path moves to the front in all layers at once
        {"name": "keep, 16 requests", **_case("keep", 16, (500, 4000), (16, 40), (32, 8), 128, 16, "int8", layers=8)},
        # a prompt is sampled eight times
        {"name": "fork, one into eight", **_case("fork", 8, (700, 700), (1, 1), (32, 8), 128, 64, "int8", group=8)},
        # beam search: the beams of every request change places and write on
        {"name": "fork, 64 beams", **_case("fork", 64, (200, 1500), (1, 1), (32, 8), 128, 64, "fp8_e4m3", layers=8, group=4)},
        # half of the requests leave, the others' pages move together, new ones come
        {"name": "pages, half leave", **_case("pages", 48, (300, 2500), (0, 0), (32, 8), 128, 64, "int8", layers=4)},
        # a layer's step with drafts: the tree, append at its positions, attention, the accepted path
        {"name": "step, 32 requests", **_case("step", 32, (500, 8000), (6, 20), (16, 4), 128, 32, "int8", pairing="halves")},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    while True:
        kind = rng.choice(("tree", "tree", "tree", "tree", "positions", "positions", "keep", "fork", "pages", "step"))
        dim, page, dtype = rng.choice((64, 128)), rng.choice((16, 32, 64, 128)), rng.choice(("int8", "fp8_e4m3"))
        kv = rng.choice((1, 2, 3, 4, 8, 16, 32))
        heads = kv * rng.choice((1, 1, 2, 3, 4, 6, 7, 8) if kv <= 8 else (1, 2))
        more = {"pairing": rng.choice(("adjacent", "halves"))}
        if kind in ("tree", "step"):
            seqs, new, before = _log_int(rng, 1, 48), _log_int(rng, 1, 200), rng.choice((rng.randint(0, 40), _log_int(rng, 30, 16000), _log_int(rng, 300, 16000), _log_int(rng, 300, 130000)))
            if rng.random() < 0.35:
                more.update(window=_log_int(rng, 1, 4096), sinks=rng.choice((0, 1, 4, 16, 70)))
        elif kind == "positions":
            seqs, new, before = _log_int(rng, 1, 48), _log_int(rng, 1, 2500), rng.choice((rng.randint(0, 40), _log_int(rng, 30, 4000)))
            more["axes"] = rng.randint(1, 4)
        elif kind == "keep":
            seqs, new, before = _log_int(rng, 1, 48), _log_int(rng, 2, 100), rng.choice((rng.randint(0, 40), _log_int(rng, 30, 4000)))
            more["layers"] = rng.randint(1, 8)
        else:
            more["group"] = rng.choice((2, 3, 4, 8)) if kind == "fork" else 1
            seqs, new, before = more["group"] * _log_int(rng, 1, 16) if kind == "fork" else rng.randint(2, 64), rng.randint(1, 20) if kind == "fork" else 0, _log_int(rng, 20, 4000)
            more["layers"] = rng.randint(1, 8)
        ragged = rng.random() < 0.6
        c = _case(kind, seqs, (int(before * rng.uniform(0.05, 1)) if ragged else before, before), (max(min(1, new), int(new * rng.uniform(0.3, 1))) if ragged else new, new),
                  (heads, kv), dim, page, dtype, **more)
        w, last = work(c), before + new
        # no dearer than the listed ones, for either form: bytes, operations, scores, keys and pages of the plain form
        if w["bytes"] > 8e8 or w["flops"] > 1.2e11 or (kind in ("tree", "step") and seqs * heads * new * last > 2.7e8) or seqs * kv * dim * last * c["layers"] > 1.9e8 or seqs * heads * dim * new > 4e7:
            continue
        return c


def _lengths(c):
    """Tokens before the step and new rows of every sequence: fixed by the case, odd and spread over their ranges."""
    def spread(lo, hi, step):
        if c["seqs"] == 1 or lo >= hi:
            return [hi] * c["seqs"]
        a = [(i * step % c["seqs"]) / (c["seqs"] - 1) for i in range(c["seqs"])]
        return [int(round((lo + 1) * ((hi + 1) / (lo + 1)) ** x)) - 1 for x in a]
    step = next(s for s in (7, 11, 13, 17) if math.gcd(s, c["seqs"]) == 1)
    return spread(c["before_min"], c["before_max"], step), spread(c["new_min"], c["new_max"], step)


def _path(n):
    """Tokens of a tree of n that are kept."""
    return max(1, n // 5)


def work(c):
    before, new = _lengths(c)
    rows, P, L, D, H = sum(new), c["page"], c["layers"], c["dim"], c["kv_heads"]
    row, q_row = 2 * H * D, c["q_heads"] * D                    # codes of a token's key and value
    page = P * row + 8 * H
    out = {"bytes": 0.0, "flops": 0.0}
    if c["kind"] in ("positions", "step"):
        # q, k and v and positions read, turned queries, codes and scales written
        out["bytes"] += rows * (4 * q_row + 3 * row + 4 * c["axes"])
        out["flops"] += 6 * rows * (q_row + row // 2)
    if c["kind"] == "positions":
        out["bytes"] += sum(n + b % P for b, n in zip(before, new)) * 3 * row        # the pages' values read back as bf16
    if c["kind"] in ("tree", "step"):
        cached = pairs = 0
        for b, n in zip(before, new):
            first = max(0, b + 1 - c["window"]) if c["window"] else 0
            seen = b - first + min(first, c["sinks"])
            cached += seen + n
            pairs += n * (seen + min(n, 4))                     # a token and a few in front of it
        out["bytes"] += cached * (row + 8 * H / P) + rows * (4 * q_row + 4 * ((max(new) + 31) // 32))
        out["flops"] += 4.0 * pairs * q_row
    if c["kind"] in ("keep", "step"):
        # the kept rows' codes from one place to the other, the touched pages' values read back as bf16
        out["bytes"] += L * sum(2 * _path(n) * row + (b % P + _path(n)) * 3 * row for b, n in zip(before, new))
        out["flops"] += L * sum((b % P + 2 * _path(n)) * row for b, n in zip(before, new))
    if c["kind"] == "fork":
        before = [before[i - i % c["group"]] for i in range(c["seqs"])]
        out["bytes"] += 12.0 * sum(-(-b // P) for b in before) + sum(2 * L * page for i, b in enumerate(before) if b % P and i % c["group"])
    if c["kind"] == "pages":
        held = [-(-b // P) for b in before]
        out["bytes"] += 16.0 * sum(held) + L * page * min(sum(held[:c["seqs"] // 2]), sum(held[c["seqs"] // 2:])) * 2
    return out


# ------------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------------
def _tree(n, rng):
    """Parents of n drafted tokens, chains that branch and begin anew at the last cached token now and then; and a path of them from its first one on."""
    u = torch.rand(n, 2, generator=rng)
    parents = [-1 if i == 0 or a < 0.03 else i - 1 if a < 0.3 else int(b * i) for i, (a, b) in enumerate(u.tolist())]
    path = [0] + sorted((torch.randperm(n - 1, generator=rng)[:_path(n) - 1] + 1).tolist())
    for i, j in zip(path, path[1:]):
        parents[j] = i
    return parents, path


def _pair_axes(c):
    """The axis of each pair of dimensions: dealt out in turn for halves, in sections for adjacent pairs."""
    n = c["dim"] // 2
    return [j % c["axes"] if c["pairing"] == "halves" else j * c["axes"] // n for j in range(n)]


def prepare(c, seed):
    dev = torch.device("cuda")
    g, rng = torch.Generator(device=dev).manual_seed(seed), torch.Generator().manual_seed(seed)
    before, new = _lengths(c)
    S, P, H, D, L, last = c["seqs"], c["page"], c["kv_heads"], c["dim"], c["layers"], [b + n for b, n in zip(before, new)]
    B = c["group"] if c["kind"] == "fork" else 1
    if c["kind"] == "fork":                     # one request that is to be sampled, or beams of several, which share their pages but for the last, unless that is full
        before = [before[i - i % B] if S > B or i == 0 else 0 for i in range(S)]
    held = [-(-x // P) for x in (before if c["kind"] in ("fork", "pages") else last)]
    width = max(-(-x // P) for x in last + [b + n for b, n in zip(before, new)])
    # every sequence's pages, from anywhere in the cache; what a table has behind them is never looked at
    pages = 3 + sum(held) + (S * (2 + -(-max(new) // P)) if c["kind"] == "fork" else max(held) * (S - S // 2) if c["kind"] == "pages" else 0)
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((S, width), -1, dtype=torch.int32, device=dev)
    at, refs = 0, torch.zeros(pages, dtype=torch.int32, device=dev)
    for s, n in enumerate(held):
        shared = before[s] // P if s % B else 0
        table[s, :shared] = table[s - s % B, :shared]
        table[s, shared:n] = order[at:at + n - shared]
        at += n - shared
        refs[table[s, :n].long()] += 1
    qm = Q_MAX[c["dtype"]]

    def codes():
        # as of normal values whose largest of a page meets the type's largest
        x = torch.randn(L, pages, H, P, D, generator=g, device=dev, dtype=torch.bfloat16) * (qm / 4.2)
        return (x.round_() if c["dtype"] == "int8" else x).clamp_(-qm, qm).to(CODES[c["dtype"]])

    def scales(size):
        return size * 4.2 / qm * (0.8 + 0.4 * torch.rand(L, pages, H, generator=g, device=dev))

    rows_at = [0]
    for n in new:
        rows_at.append(rows_at[-1] + n)
    total, i32 = rows_at[-1], dict(dtype=torch.int32, device=dev)
    st = {"c": c, "k_pool": codes(), "v_pool": codes(), "k_scale": scales(1.0), "v_scale": scales(0.5), "table": table, "before": torch.tensor(before, **i32), "rows": torch.tensor(rows_at, **i32)}
    if own:
        from moshi_b200.models import PagedBatch, PagedKVCache, PagedTree, PagePool, RotaryTable
        st["caches"] = [PagedKVCache.from_tensors(st["k_pool"][i], st["v_pool"][i], st["k_scale"][i], st["v_scale"][i]) for i in range(L)]
        st["pool"] = PagePool(st["caches"], S, width)
    if c["kind"] in ("fork", "pages"):
        st.update(lengths=st["before"], held=torch.tensor(held, **i32), refs=refs)
        if c["kind"] == "fork":
            source = [i - i % B + int(x * B) if S > B else 0 for i, x in enumerate(torch.rand(S, generator=rng).tolist())]
            add = new
        else:                                   # the first half leaves, the second takes its places, new ones of its lengths come
            source = [i + S - S // 2 if i + S - S // 2 < S else -1 for i in range(S)]
            add = [before[i] if source[i] < 0 else 0 for i in range(S)]
        st["source"], st["add"] = torch.tensor(source, **i32), torch.tensor(add, **i32)
        if own:
            for name in ("table", "lengths", "held", "refs"):
                getattr(st["pool"], name).copy_(st[name])
        return st
    # rows of a projection of q, k and v side by side, as the layer in front hands them on
    st["qkv"] = torch.randn(total, (c["q_heads"] + 2 * H) * D, generator=g, device=dev, dtype=torch.bfloat16)
    st["q"] = st["qkv"][:, :c["q_heads"] * D].unflatten(1, (c["q_heads"], D))
    st["k"] = st["qkv"][:, c["q_heads"] * D:(c["q_heads"] + H) * D].unflatten(1, (H, D))
    st["v"] = st["qkv"][:, (c["q_heads"] + H) * D:].unflatten(1, (H, D)).mul_(0.5)
    st["freq"] = 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64, device=dev) / (D // 2))
    st["axis"] = torch.tensor(_pair_axes(c), device=dev)
    # where every row lies: its sequence, its place among the sequence's rows, its slot
    seq = torch.repeat_interleave(torch.arange(S, device=dev), torch.tensor(new, device=dev))
    place = torch.arange(total, device=dev) - st["rows"][:-1].long()[seq]
    slot = st["before"].long()[seq] + place
    trees = [_tree(n, rng) for n in new]
    st.update(seq=seq, place=place, slot=slot, longest=max(new), parents=torch.tensor([x for t, _ in trees for x in t], **i32))
    kept = [path for _, path in trees]
    st["counts"], st["kept"] = torch.tensor([len(p) for p in kept], **i32), torch.zeros(total, **i32)
    flat = [x for p in kept for x in p]
    ks = torch.repeat_interleave(torch.arange(S, device=dev), st["counts"].long())
    ki = torch.arange(len(flat), device=dev) - (st["counts"].long().cumsum(0) - st["counts"].long())[ks]
    st["kept"][st["rows"][:-1].long()[ks] + ki] = torch.tensor(flat, **i32)
    if c["kind"] == "positions":                # patches of images, line after line and frame after frame, on top of what there is
        side = max(1, int(math.sqrt(max(new)) / 1.5))
        axes = [place // (side * side), place // side % side, place % side, place]
        st["positions"] = torch.stack([st["before"].long()[seq] + (place if c["axes"] == 1 else axes[i]) for i in range(c["axes"])]).to(torch.int32)
        end = last
    else:
        end = [b + n for b, n in zip(before, st["counts"].tolist())]
    # pages that the pass changes, read back from their beginning
    start = [b - b % P for b in before]
    count = [x - s for x, s in zip(end, start)]
    at = [0]
    for n in count:
        at.append(at[-1] + n)
    st["back_before"], st["back_rows"], st["back_total"] = torch.tensor(start, **i32), torch.tensor(at, **i32), at[-1]
    touched = [(s, b) for s in range(S) for b in range(start[s] // P, -(-last[s] // P))]
    of = {x: i for i, x in enumerate(touched)}
    t_seq, t_blk = (torch.tensor([x[i] for x in touched], device=dev) for i in (0, 1))
    first = torch.tensor([of[(s, start[s] // P)] for s in range(S)], device=dev)
    base = st["before"].long() // P
    st["t_page"] = table[t_seq, t_blk].long()
    st["t_old"] = (st["before"].long()[t_seq] - t_blk * P).clamp(0, P)                 # rows that the page has already
    st["t_end"] = (torch.tensor(last, device=dev)[t_seq] - t_blk * P).clamp(0, P)
    st["row_t"], st["row_slot"] = first[seq] + slot // P - base[seq], slot % P
    ka, kb = st["before"].long()[ks] + torch.tensor(flat, device=dev), st["before"].long()[ks] + ki
    st["from_t"], st["from_slot"], st["to_t"], st["to_slot"] = first[ks] + ka // P - base[ks], ka % P, first[ks] + kb // P - base[ks], kb % P
    bs = torch.repeat_interleave(torch.arange(S, device=dev), torch.tensor(count, device=dev))
    bp = torch.tensor(start, device=dev)[bs] + torch.arange(at[-1], device=dev) - st["back_rows"][:-1].long()[bs]
    st["back_t"], st["back_slot"] = first[bs] + bp // P - base[bs], bp % P
    if own:
        st["rotary"] = RotaryTable(D, base=10000.0, pairing=c["pairing"], axes=_pair_axes(c), device=dev)
        st["batch"] = PagedBatch(table, st["before"], st["rows"], total, max_rows=max(new))
        st["back"] = PagedBatch(table, st["back_before"], st["back_rows"], st["back_total"], max_rows=max(count))
        if c["kind"] in ("tree", "step"):
            st["tree"] = PagedTree(st["batch"], st["parents"])
    elif c["kind"] == "tree":                   # of a step, which has many layers
        st["seen"], st["depth"] = _ancestors(st)
    return st


# ------------------------------------------------------------------------------------------------------------------------
# the plain form
# ------------------------------------------------------------------------------------------------------------------------
def _rotated(st, x, pos):
    x = x.float()
    angle = pos.double()[st["axis"]].t() * st["freq"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if st["c"]["pairing"] == "adjacent":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _stored(st, x, pool, scale):
    """x f32 [rows, heads, dim] into the touched pages of a layer: the scales and codes of these pages afterwards."""
    c, (N, P) = st["c"], (st["t_page"].numel(), st["c"]["page"])
    qm = Q_MAX[c["dtype"]]
    new = torch.zeros(N, P, x.shape[1], x.shape[2], device=x.device)
    new[st["row_t"], st["row_slot"]] = x
    new = new.transpose(1, 2)
    top = new.abs().amax((2, 3))
    need = torch.where(top > 0, (top / qm).clamp_min(SCALE_MIN), torch.zeros_like(top))
    old = scale[st["t_page"]]
    had = (st["t_old"] > 0)[:, None] & (old > 0)
    one = torch.where(had, old, torch.ones_like(old))
    part, power = torch.frexp(torch.where(need > one, need / one, torch.ones_like(need)))
    power = torch.where(had & (need > one), power - (part == 0.5).int(), torch.zeros_like(power))          # doublings
    s = torch.where(had, torch.ldexp(old, power), need)
    was = pool[st["t_page"]].float()
    keep = torch.ldexp(was, -power[:, :, None, None]) * (old > 0)[:, :, None, None]
    put = new / torch.where(s > 0, s, torch.ones_like(s))[:, :, None, None]
    if c["dtype"] == "int8":
        keep, put = keep.round(), put.round()
    slot = torch.arange(P, device=x.device)
    is_old, is_new = (slot < st["t_old"][:, None])[:, None, :, None], (slot < st["t_end"][:, None])[:, None, :, None]
    codes = torch.where(is_old, keep, torch.where(is_new, put.clamp(-qm, qm), was)).to(pool.dtype)
    pool.view(torch.int8)[st["t_page"]] = codes.view(torch.int8)
    scale[st["t_page"]] = s


def _append(st, pos):
    q = _rotated(st, st["q"], pos).to(torch.bfloat16)
    _stored(st, _rotated(st, st["k"], pos), st["k_pool"][0], st["k_scale"][0])
    _stored(st, st["v"].float(), st["v_pool"][0], st["v_scale"][0])
    return q


def _ancestors(st):
    """[seqs, rows, rows]: whether a token is the other or comes behind it; and the tokens' depths."""
    S, n = st["c"]["seqs"], st["longest"]
    up = torch.zeros(S, n, n, device=st["q"].device)
    parent = st["parents"].long()
    up[st["seq"], st["place"], parent.clamp_min(0)] = (parent >= 0).float()
    one = torch.eye(n, device=up.device).expand(S, n, n)
    # 1 + up + up^2 + ..., whole numbers all along
    seen = torch.linalg.solve_triangular(one - up, one, upper=False, unitriangular=True).round() > 0
    return seen, seen.sum(2) - 1


def _attend(st, q, seen, depth):
    c = st["c"]
    S, H, D, n = c["seqs"], c["kv_heads"], c["dim"], st["longest"]
    G = c["q_heads"] // H
    page = st["table"].long().clamp_min(0)

    def values(pool, scale):
        x = pool[page].float() * scale[page][..., None, None]                  # [seqs, pages, heads, page, dim]
        return x.transpose(2, 3).reshape(S, -1, H, D).transpose(1, 2)

    row = (st["rows"][:-1].long()[:, None] + torch.arange(n, device=q.device)).clamp_max(q.shape[0] - 1)
    qs = q.float()[row].reshape(S, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, n * G, D)
    scores = torch.matmul(qs, values(st["k_pool"][0], st["k_scale"][0]).transpose(2, 3)) * D ** -0.5
    before, key = st["before"].long()[:, None], torch.arange(scores.shape[-1], device=q.device)
    drafted = key >= before                                                    # [seqs, keys]
    i = (key - before).clamp(0, n - 1)
    sees = ~drafted[:, None] | (seen.gather(2, i[:, None].expand(S, n, -1)) & (key < before + st["rows"].diff()[:, None])[:, None])
    if c["window"]:
        pos, key_pos = (before + depth)[..., None], torch.where(drafted, before + depth.gather(1, i), key)[:, None]
        sees = sees & ((pos - key_pos < c["window"]) | (key_pos < c["sinks"]))
    scores.masked_fill_(~sees.repeat_interleave(G, 1)[:, None], float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    v = values(st["v_pool"][0], st["v_scale"][0])
    v = v.masked_fill((key >= before + st["rows"].diff()[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(scores, v).div_(total).reshape(S, H, n, G, D).permute(0, 2, 1, 3, 4).reshape(S, n, H * G, D)
    return out[st["seq"], st["place"]].to(torch.bfloat16)


def _kept(st, pools, scales):
    """The kept rows to the front, in all layers: what is read back of one side."""
    c, (N, P) = st["c"], (st["t_page"].numel(), st["c"]["page"])
    qm, L, H = Q_MAX[c["dtype"]], c["layers"], c["kv_heads"]
    pages = pools[:, st["t_page"]].float()                                     # [layers, touched, heads, page, dim]
    old = scales[:, st["t_page"]]
    rows = pages.permute(1, 3, 0, 2, 4)[st["from_t"], st["from_slot"]]         # [kept, layers, heads, dim]
    far = st["from_t"] != st["to_t"]                                           # from another page
    size = rows.abs().amax(-1) * old.transpose(0, 1)[st["from_t"]] * far[:, None, None]
    top = torch.zeros(N, L, H, device=rows.device).index_reduce_(0, st["to_t"], size, "amax").transpose(0, 1)
    resident = torch.zeros(N, dtype=torch.int64, device=rows.device).index_add_(0, st["to_t"], (~far).long()) + st["t_old"] > 0
    arrives = torch.zeros(N, dtype=torch.int64, device=rows.device).index_add_(0, st["to_t"], far.long()) > 0
    need = torch.where(top > 0, (top / qm).clamp_min(SCALE_MIN), torch.zeros_like(top))
    had = resident[None, :, None] & (old > 0)                                  # codes that stay: their scale is doubled until the largest value has a code
    limit = torch.where(had, old * qm, torch.ones_like(old))
    part, power = torch.frexp(torch.where(top > limit, top / limit, torch.ones_like(top)))
    power = torch.where(had & (top > limit), power - (part == 0.5).int(), torch.zeros_like(power))
    s = torch.where(arrives[None, :, None], torch.where(had, torch.ldexp(old, power), need), old)
    stay = torch.ldexp(pages, -power[..., None, None]) * ((old > 0) | ~arrives[None, :, None])[..., None, None]
    by = torch.where(s > 0, s, torch.ones_like(s)).transpose(0, 1)[st["to_t"]][..., None]
    moved = (rows * old.transpose(0, 1)[st["from_t"]][..., None] / by).clamp(-qm, qm)
    if c["dtype"] == "int8":
        stay, moved = stay.round(), moved.round()
    put = torch.where(far[:, None, None, None], moved, stay.permute(1, 3, 0, 2, 4)[st["from_t"], st["from_slot"]])
    after = torch.where((torch.arange(P, device=rows.device) < st["t_old"][:, None])[None, :, None, :, None], stay, pages)
    after.permute(1, 3, 0, 2, 4)[st["to_t"], st["to_slot"]] = put
    codes = after.to(pools.dtype)
    pools.view(torch.int8)[:, st["t_page"]] = codes.view(torch.int8)
    scales[:, st["t_page"]] = s
    return _read(st, pools, scales)


def _read(st, pools, scales):
    """[layers, rows, heads, dim]: the changed pages' values."""
    page = st["t_page"][st["back_t"]]
    x = pools.permute(1, 3, 0, 2, 4)[page, st["back_slot"]].float() * scales.transpose(0, 1)[page][..., None]
    return x.transpose(0, 1).to(torch.bfloat16)


def _rearranged(st):
    P, n = st["c"]["page"], st["table"].shape[1]
    at = st["source"].long()
    st["lengths"] = torch.where(at >= 0, st["lengths"][at.clamp_min(0)], torch.zeros_like(st["lengths"]))
    st["held"] = (st["lengths"] + P - 1) // P
    has = torch.arange(n, device=at.device) < st["held"][:, None]
    st["table"] = torch.where(has, st["table"][at.clamp_min(0)], torch.full_like(st["table"], -1))
    st["refs"] = torch.zeros_like(st["refs"]).index_add_(0, st["table"].clamp_min(0).flatten().long(), has.flatten().int())


def _copied(st, dst, src):
    for name in ("k_pool", "v_pool", "k_scale", "v_scale"):
        x = st[name].view(torch.int8) if "pool" in name else st[name]
        x[:, dst] = x[:, src]


def _reserved(st):
    """Pages for `add` tokens behind what there is, the lowest free ones first; a shared page that tokens are added to is copied, but for the last of those that share it."""
    P, S, n = st["c"]["page"], st["c"]["seqs"], st["table"].shape[1]
    lengths, add, held = st["lengths"].long(), st["add"].long(), st["held"].long()
    want = torch.maximum(held, torch.where(add > 0, (lengths + add + P - 1) // P, held))
    block = (lengths // P).clamp_max(n - 1)
    page = st["table"].long().gather(1, block[:, None])[:, 0]
    begun = (lengths % P > 0) & (add > 0)
    rank = ((page[:, None] == page) & begun & begun[:, None]).tril(-1).sum(1)
    copies = begun & (st["refs"].long()[page.clamp_min(0)] - rank > 1)
    need = want - held + copies
    at = need.cumsum(0) - need
    free = torch.sort(st["refs"] > 0, stable=True).indices                     # free ones first, lowest first
    fits = need.sum() <= (st["refs"] == 0).sum()
    need, copies, want = need * fits, copies & fits, torch.where(fits, want, held)
    b = torch.arange(n, device=page.device)
    fresh = (b >= held[:, None]) & (b < want[:, None])
    new = free[(at[:, None] + copies[:, None] + b - held[:, None]).clamp(0, free.numel() - 1)]
    st["table"] = torch.where(fresh, new.int(), st["table"])
    copy_to = free[at.clamp_max(free.numel() - 1)]
    st["table"] = torch.where((b == block[:, None]) & copies[:, None], copy_to[:, None].int(), st["table"])
    refs = st["refs"].clone().index_add_(0, page.clamp_min(0), -copies.int()).index_add_(0, copy_to, copies.int())
    st["refs"] = refs.index_add_(0, st["table"].clamp_min(0).flatten().long(), fresh.flatten().int())
    st["held"] = want.int()
    _copied(st, copy_to[copies], page[copies])


def _compacted(st):
    used = st["refs"] > 0
    number = torch.arange(used.numel(), device=used.device)
    end = used.sum()
    src, dst = number[used & (number >= end)], number[~used & (number < end)]
    _copied(st, dst, src)
    to = number.clone()
    to[src] = dst
    st["table"] = torch.where(st["table"] >= 0, to[st["table"].long().clamp_min(0)].int(), st["table"])
    refs = st["refs"].clone()
    refs[dst], refs[src] = st["refs"][src], 0
    st["refs"] = refs


def _pages(st, of):
    return {**{n: getattr(of, n) if of else st[n] for n in ("table", "lengths", "held", "refs")}, "k": st["k_pool"].view(torch.int8), "v": st["v_pool"].view(torch.int8),
            "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _plain(st):
    c = st["c"]
    if c["kind"] == "fork":
        _rearranged(st)
        _reserved(st)
        return _pages(st, None)
    if c["kind"] == "pages":
        _rearranged(st)
        _compacted(st)
        _reserved(st)
        st["lengths"] = st["lengths"] + st["add"]
        return _pages(st, None)
    if c["kind"] == "positions":
        q = _append(st, st["positions"])
        return {"q": q, "k": _read(st, st["k_pool"], st["k_scale"]), "v": _read(st, st["v_pool"], st["v_scale"])}
    if c["kind"] == "keep":
        return {"k": _kept(st, st["k_pool"], st["k_scale"]), "v": _kept(st, st["v_pool"], st["v_scale"])}
    if c["kind"] == "tree":
        return {"out": _attend(st, st["q"], st["seen"], st["depth"])}
    seen, depth = _ancestors(st)
    q = _append(st, (st["before"].long()[st["seq"]] + depth[st["seq"], st["place"]])[None])
    out = _attend(st, q, seen, depth)
    return {"q": q, "out": out, "k": _kept(st, st["k_pool"], st["k_scale"]), "v": _kept(st, st["v_pool"], st["v_scale"])}


def _read_own(st):
    back = [cache.read(st["back"]) for cache in st["caches"]]
    return {n: torch.stack([x[i] for x in back]) if len(back) > 1 else back[0][i][None] for i, n in enumerate("kv")}


def run(st):
    if not own:
        return _plain(st)
    c = st["c"]
    if c["kind"] == "fork":
        st["pool"].rearrange(st["source"])
        st["pool"].reserve(st["add"])
        return _pages(st, st["pool"])
    if c["kind"] == "pages":
        st["pool"].rearrange(st["source"])
        st["pool"].compact()
        st["pool"].reserve(st["add"])
        st["pool"].lengths += st["add"]
        return _pages(st, st["pool"])
    batch = st["batch"]
    if c["kind"] == "positions":
        return {"q": st["caches"][0].append(batch, st["k"], st["v"], q=st["q"], rotary=st["rotary"], positions=st["positions"]), **_read_own(st)}
    if c["kind"] == "keep":
        st["pool"].keep(batch, st["kept"], st["counts"])
        return _read_own(st)
    tree, cache = st["tree"], st["caches"][0]
    if c["kind"] == "tree":
        return {"out": cache.attend(batch, st["q"], window=c["window"], sinks=c["sinks"], tree=tree)}
    tree.update()
    q = cache.append(batch, st["k"], st["v"], q=st["q"], rotary=st["rotary"], positions=tree.positions)
    out = cache.attend(batch, q, window=c["window"], sinks=c["sinks"], tree=tree)
    cache.keep(batch, st["kept"], st["counts"])
    return {"q": q, "out": out, **_read_own(st)}


# ------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ------------------------------------------------------------------------------------------------------------------------
def _exact_rotation(x, pos, axes, pairing):
    """x f64 [rows, heads, dim] at pos [axes, rows], as complex numbers turned."""
    d = x.shape[-1]
    i = torch.arange(d // 2, dtype=torch.float64, device=x.device)
    angle = torch.stack([pos[a].double() for a in axes], 1) * torch.exp(-i * (2.0 / d) * math.log(10000.0))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if pairing == "adjacent":
        return torch.view_as_real(torch.view_as_complex(x.unflatten(2, (d // 2, 2)).contiguous()) * turn).flatten(2)
    z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn
    return torch.cat((z.real, z.imag), 2)


def _nearest(y, dtype):
    y = y.clamp(-Q_MAX[dtype], Q_MAX[dtype])
    return y.round() if dtype == "int8" else y.to(torch.float32).to(torch.float8_e4m3fn).double()


def _exact_scale(top, old, resident, dtype, exactly):
    """What a page's scale [heads] becomes for rows of up to `top`, and its doublings; exactly: up to the last bit of top, whose rows have been codes before."""
    need = torch.where(top > 0, torch.clamp(top / Q_MAX[dtype], min=SCALE_MIN), torch.zeros_like(top))
    if not resident:
        return need, torch.zeros_like(need)
    limit = torch.where(old > 0, old, torch.ones_like(old))
    part, power = torch.frexp(top / (Q_MAX[dtype] * limit) if exactly else need / limit)
    doublings = torch.where((old > 0) & (top > 0), power - (part == 0.5).int(), torch.zeros_like(power)).clamp_min(0)
    return torch.where(old > 0, old * 2.0 ** doublings, need), doublings


def _exact_append(x, b, pages, scales, table, P, dtype):
    """Rows x f64 [n, heads, dim] behind the first b tokens of a sequence; pages {number: f64 [page, heads, dim]}, scales {number: f64 [heads]} change."""
    done = 0
    while done < x.shape[0]:
        o, m = (b + done) % P, min(x.shape[0] - done, P - (b + done) % P)
        page, y = table[(b + done) // P], x[done:done + m]
        old, codes = scales[page], pages[page]
        s, doublings = _exact_scale(y.abs().amax((0, 2)), old, o > 0, dtype, False)
        codes[:o] = torch.where(old[None, :, None] > 0, _nearest(codes[:o] * (2.0 ** -doublings)[None, :, None], dtype), torch.zeros_like(codes[:o]))
        codes[o:o + m] = _nearest(y / torch.where(s > 0, s, torch.ones_like(s))[None, :, None], dtype)
        scales[page] = s
        done += m


def _exact_keep(path, b, pages, scales, table, P, dtype):
    was, had = {p: x.clone() for p, x in pages.items()}, dict(scales)
    for block in range(b // P, (b + len(path) - 1) // P + 1):
        page, o = table[block], max(0, b - block * P)
        mine = [(b + i - block * P, (b + a) % P, table[(b + a) // P]) for i, a in enumerate(path) if (b + i) // P == block]
        far = [x for x in mine if x[2] != page]
        if far:
            top = torch.stack([was[p][slot].abs().amax(-1) * had[p] for _, slot, p in far]).amax(0)
            s, doublings = _exact_scale(top, had[page], o > 0 or len(far) < len(mine), dtype, True)
        else:
            s, doublings = had[page], torch.zeros_like(had[page])
        stay = _nearest(was[page] * (2.0 ** -doublings)[None, :, None], dtype)
        if far:
            stay = torch.where(had[page][None, :, None] > 0, stay, torch.zeros_like(stay))
        pages[page][:o] = stay[:o]
        for to, slot, p in mine:
            pages[page][to] = stay[slot] if p == page else _nearest(was[p][slot] * had[p][:, None] / torch.where(s > 0, s, torch.ones_like(s))[:, None], dtype)
        scales[page] = s


def _exact_pages(c, st):
    """Tables, references and moves with lists, one thing after the other."""
    P, S = c["page"], c["seqs"]
    lengths, refs = st["lengths"].tolist(), st["refs"].tolist()
    table = [row[:h] for row, h in zip(st["table"].tolist(), st["held"].tolist())]
    scale = [st["k_scale"].double().clone(), st["v_scale"].double().clone()]

    def move(src, dst):
        for x in scale:
            x[:, dst] = x[:, src]

    source, add = st["source"].tolist(), st["add"].tolist()
    old, old_lengths = [list(t) for t in table], list(lengths)
    lengths = [old_lengths[s] if s >= 0 else 0 for s in source]
    table = [old[s][:-(-n // P)] if s >= 0 else [] for s, n in zip(source, lengths)]
    refs = [0] * len(refs)
    for t in table:
        for p in t:
            refs[p] += 1
    if c["kind"] == "pages":
        end = sum(r > 0 for r in refs)
        holes = [p for p in range(end) if refs[p] == 0]
        for p, to in zip([p for p in range(end, len(refs)) if refs[p] > 0], holes):
            move(p, to)
            refs[to], refs[p] = refs[p], 0
            table = [[to if x == p else x for x in t] for t in table]
    free = [p for p, r in enumerate(refs) if r == 0]
    for i in range(S):
        if add[i] and lengths[i] % P and refs[table[i][lengths[i] // P]] > 1:
            p = table[i][lengths[i] // P]
            to = free.pop(0)
            move(p, to)
            refs[p], refs[to], table[i][lengths[i] // P] = refs[p] - 1, 1, to
        while add[i] and len(table[i]) < -(-(lengths[i] + add[i]) // P):
            refs[free[0]] = 1
            table[i].append(free.pop(0))
    if c["kind"] == "pages":
        lengths = [n + a for n, a in zip(lengths, add)]
    i32 = dict(dtype=torch.int32)
    width = st["table"].shape[1]
    return {"table": torch.tensor([t + [-1] * (width - len(t)) for t in table], **i32), "lengths": torch.tensor(lengths, **i32), "held": torch.tensor([len(t) for t in table], **i32),
            "refs": torch.tensor(refs, **i32), "k": None, "v": None, "k_scale": scale[0], "v_scale": scale[1]}


def exact(c, seed):
    st = prepare(c, seed)
    if c["kind"] in ("fork", "pages"):
        return _exact_pages(c, st)
    before, new = _lengths(c)
    P, H, D, L, dtype, dev = c["page"], c["kv_heads"], c["dim"], c["layers"], c["dtype"], st["q"].device
    G, table, at = c["q_heads"] // H, st["table"].tolist(), [0]
    for n in new:
        at.append(at[-1] + n)
    paths = [st["kept"][a:a + k].tolist() for a, k in zip(at, st["counts"].tolist())]
    q, parents, axes = st["q"].double(), st["parents"].tolist(), _pair_axes(c)
    answer, turned, back = torch.zeros_like(q), [], ([], [])
    for s, (b, n) in enumerate(zip(before, new)):
        rows = slice(at[s], at[s + 1])
        line = []                                          # of each drafted token: the tokens that it sees
        for i, p in enumerate(parents[rows]):
            line.append((line[p] if p >= 0 else []) + [i])
        depth = torch.tensor([len(x) - 1 for x in line], device=dev)
        place = st["positions"][:, rows] if c["kind"] == "positions" else (b + depth)[None]
        qs = q[rows]
        sides = []
        for side, (pool, scale) in enumerate(((st["k_pool"], st["k_scale"]), (st["v_pool"], st["v_scale"]))):
            for layer in range(L):
                touched = table[s][b // P:-(-(b + n) // P)]
                pages, scales = {p: pool[layer, p].float().double().transpose(0, 1) for p in touched}, {p: scale[layer, p].double() for p in touched}
                if c["kind"] in ("positions", "step"):
                    x = (st["v"] if side else st["k"])[rows].double()
                    _exact_append(x if side else _exact_rotation(x, place, axes, c["pairing"]), b, pages, scales, table[s], P, dtype)
                if c["kind"] in ("tree", "step"):
                    count = -(-(b + n) // P)
                    page = st["table"][s, :count].long()
                    x = pool[layer][page].float().double() * scale[layer][page].double()[..., None, None]
                    for j, p in enumerate(touched):
                        x[b // P + j] = (pages[p] * scales[p][None, :, None]).transpose(0, 1)
                    sides.append(x.transpose(0, 1).reshape(H, count * P, D)[:, :b + n])
                if c["kind"] in ("keep", "step"):
                    _exact_keep(paths[s], b, pages, scales, table[s], P, dtype)
                end = b + (n if c["kind"] == "positions" else len(paths[s]))
                back[side].append([(pages[p] * scales[p][None, :, None])[:min(P, end - i * P)] for i, p in enumerate(table[s]) if b // P <= i <= (end - 1) // P])
        if c["kind"] in ("positions", "step"):
            qs = _exact_rotation(qs, place, axes, c["pairing"])
            turned.append(qs)
        if c["kind"] in ("tree", "step"):
            sees = torch.zeros(n, b + n, dtype=torch.bool, device=dev)
            sees[:, :b] = True
            for i, x in enumerate(line):
                sees[i, [b + j for j in x]] = True
            if c["window"]:
                key = torch.cat((torch.arange(b, device=dev), b + depth))
                sees &= ((b + depth)[:, None] - key < c["window"]) | (key < c["sinks"])
            for h in range(c["q_heads"]):
                w = (qs[:, h] @ sides[0][h // G].t()) / math.sqrt(D)
                answer[rows, h] = torch.softmax(w.masked_fill(~sees, float("-inf")), -1) @ sides[1][h // G]
    out = {}
    if c["kind"] in ("tree", "step"):
        out["out"] = answer
    if c["kind"] in ("positions", "step"):
        out["q"] = torch.cat(turned)
    if c["kind"] != "tree":
        for side, name in enumerate("kv"):                 # sequence after sequence, layer after layer -> layers of all sequences
            out[name] = torch.stack([torch.cat([x for s in range(c["seqs"]) for x in back[side][s * L + layer]]) for layer in range(L)])
    return out
