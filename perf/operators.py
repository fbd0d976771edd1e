"""Calls of the paged 8-bit cache: appending rotated keys and values, attention over it with and without a window, a decoder step of both.

``listed()`` names cases over the range of uses, ``draw()`` gives more of them, ``run()`` makes one pass: the plain form in elementary torch
operations, or, where ``own`` is true, the calls of ``moshi_b200.models.PagedKVCache``.
"""
import math

import torch

own = False

SCALE_MIN = 2.0 ** -60
Q_MAX = {"int8": 127.0, "fp8_e4m3": 448.0}
CODES = {"int8": torch.int8, "fp8_e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------------------------------------------------------------
# cases.  kind: what is called; seqs: sequences of the batch; before_min .. before_max: tokens that they have cached (spread
# over the logarithm); new_min .. new_max: rows that each of them adds; q_heads / kv_heads / dim; page: tokens of a page
# ------------------------------------------------------------------------------------------------------------------------
def _case(kind, seqs, before, new, heads, dim, page, dtype, window=0, sinks=0, pairing="adjacent"):
    return {"kind": kind, "seqs": seqs, "before_min": before[0], "before_max": before[1], "new_min": new[0], "new_max": new[1], "q_heads": heads[0],
            "kv_heads": heads[1], "dim": dim, "page": page, "dtype": dtype, "window": window, "sinks": sinks, "pairing": pairing}


def listed():
    return [
        # a frame of 48 dialogue sessions of different age: each appends one row to its page, all heads have keys of their own
        {"name": "append, 48 sessions' frame", **_case("append", 48, (40, 3000), (1, 1), (32, 32), 128, 64, "fp8_e4m3")},
        # prompts of several requests in one step, grouped heads, ends inside pages
        {"name": "append, four prompts", **_case("append", 4, (0, 700), (1500, 2500), (32, 8), 128, 64, "int8", pairing="halves")},
        # one session, half a minute old, one token: the call's latency
        {"name": "attend, one young session", **_case("attend", 1, (374, 374), (1, 1), (32, 32), 128, 64, "int8")},
        # a full box of long sessions: the cache's bytes
        {"name": "attend, 48 full sessions", **_case("attend", 48, (2999, 2999), (1, 1), (32, 32), 128, 64, "fp8_e4m3")},
        # continuous batching: requests of very different length decode together, grouped heads
        {"name": "attend, 64 ragged requests", **_case("attend", 64, (100, 16000), (1, 1), (32, 8), 128, 64, "int8")},
        # one long document: little to share out but the length
        {"name": "attend, one long request", **_case("attend", 1, (131071, 131071), (1, 1), (32, 8), 128, 128, "int8")},
        # drafted tokens checked together, narrow heads, small pages
        {"name": "attend, drafts of five", **_case("attend", 16, (1000, 6000), (5, 5), (24, 4), 64, 16, "fp8_e4m3")},
        # a portion of a long prompt on top of what is cached
        {"name": "attend, prompt portion", **_case("attend", 1, (6100, 6100), (2048, 2048), (32, 8), 128, 64, "int8")},
        # several new prompts at once, every head with keys of its own
        {"name": "attend, eight prompts", **_case("attend", 8, (0, 0), (200, 900), (16, 16), 64, 32, "fp8_e4m3")},
        # endless dialogues: the first tokens and the last thousand
        {"name": "window, 128 sessions", **_case("window", 128, (300, 20000), (1, 1), (32, 8), 128, 64, "int8", window=1024, sinks=4)},
        # a long prompt under the same window
        {"name": "window, long prompt", **_case("window", 1, (100, 100), (6000, 6000), (16, 4), 128, 64, "fp8_e4m3", window=1024, sinks=4)},
        # a layer's step of a decoder: append, then attend
        {"name": "step, 32 requests", **_case("step", 32, (500, 8000), (1, 1), (16, 4), 128, 32, "int8", pairing="halves")},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    while True:
        kind = rng.choice(("append", "attend", "attend", "window", "window", "step"))
        dim, page, dtype = rng.choice((64, 128)), rng.choice((16, 32, 64, 128)), rng.choice(("int8", "fp8_e4m3"))
        kv = rng.choice((1, 2, 3, 4, 8, 16, 32))
        heads = kv * rng.choice((1, 1, 2, 3, 4, 6, 7, 8) if kv <= 8 else (1, 2))
        shape = rng.choice(("decode", "decode", "drafts", "prompt"))
        if shape == "decode":
            seqs, new, before = _log_int(rng, 1, 128), 1, _log_int(rng, 1, 130000)
        elif shape == "drafts":
            seqs, new, before = _log_int(rng, 1, 32), rng.randint(2, 12), _log_int(rng, 1, 16000)
        else:
            seqs, new, before = _log_int(rng, 1, 8), _log_int(rng, 16, 6000), rng.choice((0, _log_int(rng, 1, 8000)))
        ragged = rng.random() < 0.6
        c = _case(kind, seqs, (int(before * rng.uniform(0.05, 1)) if ragged else before, before), (max(1, int(new * rng.uniform(0.3, 1))) if ragged else new, new),
                  (heads, kv), dim, page, dtype, pairing=rng.choice(("adjacent", "halves")))
        if kind == "window" or (kind == "step" and rng.random() < 0.3):
            c["window"], c["sinks"] = _log_int(rng, 1, 4096), rng.choice((0, 1, 4, 16, 70))
        w, last = work(c), before + new
        # no dearer than the listed ones, for either form: bytes of the cache, operations, scores and keys of the plain form
        if w["bytes"] > 1.1e9 or w["flops"] > 2.2e11 or seqs * heads * new * last > 1.6e9 or seqs * kv * dim * last > 5.5e8:
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


def _seen(c, p):
    """Keys that the row at position p sees."""
    if not c["window"]:
        return p + 1
    first = max(0, p + 1 - c["window"])
    return p + 1 - first + min(first, c["sinks"])


def work(c):
    before, new = _lengths(c)
    rows, row = sum(new), 2 * c["kv_heads"] * c["dim"]          # codes of a token's key and value
    q_row = c["q_heads"] * c["dim"]
    out = {"bytes": 0.0, "flops": 0.0}
    if c["kind"] in ("append", "step"):
        # q, k and v read, rotated queries, codes and scales written; the pages' values read back as bf16
        heads = sum(n + b % c["page"] for b, n in zip(before, new))
        out["bytes"] += rows * (4 * q_row + 3 * row) + heads * 3 * row
        out["flops"] += 6 * rows * (q_row + row // 2)
    if c["kind"] != "append":
        cached = pairs = 0
        for b, n in zip(before, new):
            first = max(0, b + 1 - c["window"]) if c["window"] else 0
            cached += b + n - first + min(first, c["sinks"])
            pairs += sum(_seen(c, p) for p in range(b, b + n))
        out["bytes"] += cached * (row + 8 * c["kv_heads"] / c["page"]) + rows * 4 * q_row
        out["flops"] += 4.0 * pairs * q_row
    return out


# ------------------------------------------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------------------------------------------
def prepare(c, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    before, new = _lengths(c)
    S, P, H, D, last = c["seqs"], c["page"], c["kv_heads"], c["dim"], [b + n for b, n in zip(before, new)]
    width = max(-(-x // P) for x in last)
    pages = sum(-(-x // P) for x in last) + 3
    # every sequence's pages, from anywhere in the cache; what a table has behind a sequence's last page is never looked at
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(S, width, dtype=torch.int32, device=dev)
    at = 0
    for s, x in enumerate(last):
        n = -(-x // P)
        table[s, :n] = order[at:at + n]
        at += n
    qm = Q_MAX[c["dtype"]]

    def codes():
        # as of normal values whose largest of a page meets the type's largest
        x = torch.randn(pages, H, P, D, generator=g, device=dev, dtype=torch.bfloat16) * (qm / 4.2)
        return (x.round() if c["dtype"] == "int8" else x).clamp(-qm, qm).to(CODES[c["dtype"]])

    def scales(size):
        return size * 4.2 / qm * (0.8 + 0.4 * torch.rand(pages, H, generator=g, device=dev))

    rows_at = [0]
    for n in new:
        rows_at.append(rows_at[-1] + n)
    total = rows_at[-1]
    st = {"c": c, "k_pool": codes(), "v_pool": codes(), "k_scale": scales(1.0), "v_scale": scales(0.5), "table": table,
          "before": torch.tensor(before, dtype=torch.int32, device=dev), "rows": torch.tensor(rows_at, dtype=torch.int32, device=dev),
          "freq": 10000.0 ** (-torch.arange(D // 2, dtype=torch.float64, device=dev) / (D // 2)),
          # rows of a projection of q, k and v side by side, as the layer in front hands them on
          "qkv": torch.randn(total, (c["q_heads"] + 2 * H) * D, generator=g, device=dev, dtype=torch.bfloat16)}
    st["q"] = st["qkv"][:, :c["q_heads"] * D].unflatten(1, (c["q_heads"], D))
    st["k"] = st["qkv"][:, c["q_heads"] * D:(c["q_heads"] + H) * D].unflatten(1, (H, D))
    st["v"] = st["qkv"][:, (c["q_heads"] + H) * D:].unflatten(1, (H, D)).mul_(0.5)
    # where every row lies: its sequence, its place among the sequence's rows, its position, page and place in the page
    seq = torch.repeat_interleave(torch.arange(S, device=dev), torch.tensor(new, device=dev))
    place = torch.arange(total, device=dev) - st["rows"][:-1].long()[seq]
    pos = st["before"].long()[seq] + place
    st.update(seq=seq, place=place, pos=pos, longest=max(new))
    if c["kind"] in ("append", "step"):
        # pages that the step touches, read back from their beginning
        start = [b - b % P for b in before]
        count = [x - s for x, s in zip(last, start)]
        at = [0]
        for n in count:
            at.append(at[-1] + n)
        st["back_before"], st["back_rows"], st["back_total"] = torch.tensor(start, dtype=torch.int32, device=dev), torch.tensor(at, dtype=torch.int32, device=dev), at[-1]
        touched = [(s, b) for s in range(S) for b in range(start[s] // P, -(-last[s] // P))]
        of = {x: i for i, x in enumerate(touched)}
        t_seq, t_blk = (torch.tensor([x[i] for x in touched], device=dev) for i in (0, 1))
        first = torch.tensor([of[(s, start[s] // P)] for s in range(S)], device=dev)
        st["t_page"] = table[t_seq, t_blk].long()
        st["t_old"] = (st["before"].long()[t_seq] - t_blk * P).clamp(0, P)             # rows that the page has already
        st["t_end"] = (torch.tensor(last, device=dev)[t_seq] - t_blk * P).clamp(0, P)
        st["row_t"] = first[seq] + pos // P - st["before"].long()[seq] // P
        bs = torch.repeat_interleave(torch.arange(S, device=dev), torch.tensor(count, device=dev))
        bp = torch.tensor(start, device=dev)[bs] + torch.arange(at[-1], device=dev) - st["back_rows"][:-1].long()[bs]
        st["back_t"], st["back_slot"] = first[bs] + bp // P - st["before"].long()[bs] // P, bp % P
    if own:
        from moshi_b200.models import PagedBatch, PagedKVCache, RotaryTable
        st["cache"] = PagedKVCache.from_tensors(st["k_pool"], st["v_pool"], st["k_scale"], st["v_scale"])
        st["rotary"] = RotaryTable(D, base=10000.0, pairing=c["pairing"], device=dev)
        st["batch"] = PagedBatch(table, st["before"], st["rows"], total, max_rows=max(new))
        if "back_rows" in st:
            st["back"] = PagedBatch(table, st["back_before"], st["back_rows"], st["back_total"], max_rows=max(count))
    return st


# ------------------------------------------------------------------------------------------------------------------------
# the plain form
# ------------------------------------------------------------------------------------------------------------------------
def _rotated(x, pos, freq, pairing):
    x = x.float()
    angle = pos.double()[:, None] * freq[None]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if pairing == "adjacent":
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)


def _stored(st, x, pool, scale):
    """x f32 [rows, heads, dim] into the touched pages of a pool: the scales and codes of these pages afterwards."""
    c, (N, P) = st["c"], (st["t_page"].numel(), st["c"]["page"])
    qm = Q_MAX[c["dtype"]]
    new = torch.zeros(N, P, x.shape[1], x.shape[2], device=x.device)
    new[st["row_t"], st["pos"] % P] = x
    new = new.transpose(1, 2)
    top = new.abs().amax((2, 3))
    need = torch.where(top > 0, (top / qm).clamp_min(SCALE_MIN), torch.zeros_like(top))
    had = (st["t_old"] > 0)[:, None] & (scale[st["t_page"]] > 0)
    old = torch.where(had, scale[st["t_page"]], torch.ones_like(need))
    part, power = torch.frexp(torch.where(need > old, need / old, torch.ones_like(need)))
    power = torch.where(need > old, power - (part == 0.5).int(), torch.zeros_like(power))      # doublings
    s = torch.where(had, torch.ldexp(old, power), need)
    was = pool[st["t_page"]].float()
    keep = torch.ldexp(was, -power[:, :, None, None]) * (scale[st["t_page"]] > 0)[:, :, None, None]
    put = new / torch.where(s > 0, s, torch.ones_like(s))[:, :, None, None]
    if c["dtype"] == "int8":
        keep, put = keep.round(), put.round()
    slot = torch.arange(P, device=x.device)
    is_old, is_new = (slot < st["t_old"][:, None])[:, None, :, None], (slot < st["t_end"][:, None])[:, None, :, None]
    codes = torch.where(is_old, keep, torch.where(is_new, put.clamp(-qm, qm), was)).to(pool.dtype)
    pool.view(torch.int8)[st["t_page"]] = codes.view(torch.int8)
    scale[st["t_page"]] = s
    values = codes[st["back_t"], :, st["back_slot"]].float() * s[st["back_t"]][:, :, None]
    return values.to(torch.bfloat16)


def _append(st):
    c = st["c"]
    q = _rotated(st["q"], st["pos"], st["freq"], c["pairing"]).to(torch.bfloat16)
    k = _stored(st, _rotated(st["k"], st["pos"], st["freq"], c["pairing"]), st["k_pool"], st["k_scale"])
    v = _stored(st, st["v"].float(), st["v_pool"], st["v_scale"])
    return q, k, v


def _attend(st, q):
    c = st["c"]
    S, H, D, n = c["seqs"], c["kv_heads"], c["dim"], st["longest"]
    G = c["q_heads"] // H
    page = st["table"].long()

    def values(pool, scale):
        x = pool[page].float() * scale[page][..., None, None]                  # [seqs, pages, heads, page, dim]
        return x.transpose(2, 3).reshape(S, -1, H, D).transpose(1, 2)

    row = (st["rows"][:-1].long()[:, None] + torch.arange(n, device=q.device)).clamp_max(q.shape[0] - 1)
    qs = q.float()[row].reshape(S, n, H, G, D).permute(0, 2, 1, 3, 4).reshape(S, H, n * G, D)
    scores = torch.matmul(qs, values(st["k_pool"], st["k_scale"]).transpose(2, 3)) * D ** -0.5
    pos = (st["before"].long()[:, None] + torch.arange(n, device=q.device))[..., None]
    key = torch.arange(scores.shape[-1], device=q.device)
    seen = key <= pos
    if c["window"]:
        seen = seen & ((pos - key < c["window"]) | (key < c["sinks"]))
    hidden = ~seen.repeat_interleave(G, 1)[:, None]
    scores.masked_fill_(hidden, float("-inf"))
    scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = scores.sum(-1, keepdim=True)
    v = values(st["v_pool"], st["v_scale"])
    last = (st["before"] + st["rows"].diff()).long()
    v = v.masked_fill((key >= last[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(scores, v) / total
    out = out.reshape(S, H, n, G, D).transpose(1, 2).reshape(S, n, H * G, D)
    return out[st["seq"], st["place"]].to(torch.bfloat16)


def run(st):
    c = st["c"]
    if own:
        out = {}
        q = st["q"]
        if c["kind"] in ("append", "step"):
            q = st["cache"].append(st["batch"], st["k"], st["v"], q=q, rotary=st["rotary"])
            out["k"], out["v"] = st["cache"].read(st["back"])
            out.update(q=q, k_scale=st["k_scale"], v_scale=st["v_scale"])
        if c["kind"] != "append":
            out["out"] = st["cache"].attend(st["batch"], q, window=c["window"], sinks=c["sinks"])
        return out
    out = {}
    q = st["q"]
    if c["kind"] in ("append", "step"):
        q, out["k"], out["v"] = _append(st)
        out.update(q=q, k_scale=st["k_scale"], v_scale=st["v_scale"])
    if c["kind"] != "append":
        out["out"] = _attend(st, q)
    return out


# ------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ------------------------------------------------------------------------------------------------------------------------
def _exact_rotation(x, first, pairing):
    """x f64 [rows, heads, dim] of the positions from `first` on, as complex numbers turned."""
    n, _, d = x.shape
    i = torch.arange(d // 2, dtype=torch.float64, device=x.device)
    angle = torch.outer(torch.arange(first, first + n, dtype=torch.float64, device=x.device), torch.exp(-i * (2.0 / d) * math.log(10000.0)))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    if pairing == "adjacent":
        return torch.view_as_real(torch.view_as_complex(x.unflatten(2, (d // 2, 2)).contiguous()) * turn).flatten(2)
    z = torch.complex(x[..., :d // 2].contiguous(), x[..., d // 2:].contiguous()) * turn
    return torch.cat((z.real, z.imag), 2)


def _exact_page(x, o, codes, scale, dtype):
    """New rows x f64 [n, heads, dim] behind the first o of a page (codes f64 [page, heads, dim], scale f64 [heads]): codes and scale afterwards."""
    qm = Q_MAX[dtype]

    def nearest(y):
        return y.round() if dtype == "int8" else y.to(torch.float32).to(torch.float8_e4m3fn).double()
    codes, top = codes.clone(), x.abs().amax((0, 2))
    need = torch.where(top > 0, torch.clamp(top / qm, min=SCALE_MIN), torch.zeros_like(top))
    if o == 0:
        s = need
    else:
        doublings = torch.where((need > scale) & (scale > 0), torch.ceil(torch.log2(need / torch.where(scale > 0, scale, torch.ones_like(scale)))), torch.zeros_like(need))
        s = torch.where(scale > 0, scale * 2.0 ** doublings, need)
        codes[:o] = torch.where(scale[None, :, None] > 0, nearest(codes[:o] * (2.0 ** -doublings)[None, :, None]), torch.zeros_like(codes[:o]))
    codes[o:o + x.shape[0]] = nearest((x / torch.where(s > 0, s, torch.ones_like(s))[None, :, None]).clamp(-qm, qm))
    return codes, s


def exact(c, seed):
    st = prepare(c, seed)
    before, new = _lengths(c)
    P, H, D = c["page"], c["kv_heads"], c["dim"]
    G = c["q_heads"] // H
    q = st["q"].double()
    pools, scale = [st["k_pool"], st["v_pool"]], [st["k_scale"].double(), st["v_scale"].double()]
    out, changed = {}, [{}, {}]
    table = st["table"].tolist()
    if c["kind"] in ("append", "step"):
        at, turned, back = 0, [], ([], [])
        for s, (b, n) in enumerate(zip(before, new)):
            rows = slice(at, at + n)
            at += n
            turned.append(_exact_rotation(q[rows], b, c["pairing"]))
            for i, x in enumerate((_exact_rotation(st["k"][rows].double(), b, c["pairing"]), st["v"][rows].double())):
                done = 0
                while done < n:
                    p = b + done
                    o, m = p % P, min(n - done, P - p % P)
                    page = table[s][p // P]
                    codes, sc = _exact_page(x[done:done + m], o, pools[i][page].float().double().transpose(0, 1), scale[i][page], c["dtype"])
                    changed[i][page], scale[i][page] = codes, sc
                    back[i].append(codes[:o + m] * sc[None, :, None])
                    done += m
        q = torch.cat(turned)
        out.update(k=torch.cat(back[0]), v=torch.cat(back[1]), q=q, k_scale=scale[0], v_scale=scale[1])
    if c["kind"] != "append":
        answer, at = torch.zeros(q.shape, dtype=torch.float64, device=q.device), 0
        for s, (b, n) in enumerate(zip(before, new)):
            count = -(-(b + n) // P)
            page = st["table"][s, :count].long()
            kv = []
            for i in (0, 1):
                x = pools[i][page].float().double()
                for j, pg in enumerate(table[s][:count]):
                    if pg in changed[i]:
                        x[j] = changed[i][pg].transpose(0, 1)
                kv.append((x * scale[i][page][..., None, None]).transpose(0, 1).reshape(H, count * P, D)[:, :b + n])
            pos, key = torch.arange(b, b + n, device=q.device)[:, None], torch.arange(b + n, device=q.device)
            far = key > pos
            if c["window"]:
                far = far | ((key <= pos - c["window"]) & (key >= c["sinks"]))
            for h in range(c["q_heads"]):
                w = (q[at:at + n, h] @ kv[0][h // G].t()) / math.sqrt(D)
                answer[at:at + n, h] = torch.softmax(w.masked_fill(far, float("-inf")), -1) @ kv[1][h // G]
            at += n
        out["out"] = answer
    return out
