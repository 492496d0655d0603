"""The key-value cache in 4 bits and the eviction of cached tokens by the attention
they got, as measured cases: their plain form in elementary torch operations, the
same calls on the framework's kernels, and the 64-bit definition.

The text decoder served here has 16 query and 8 key-value heads of 128; its caches
hold up to 4096 tokens a request in a batch of 64, or 131072 tokens in a batch of 4.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DEV = "cuda"
_EPS = 1e-6


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one new token of a single request, written in 4 bits and read back: all latency
        _append("append_1x1", 1, 1, 16, 8, 128, 128, "bf16", 16, 1024, True, False),
        # the decode step of a full batch, one token each at ragged positions
        _append("append_64x1", 64, 1, 16, 8, 128, 128, "bf16", 16, 4096, True, False),
        # eight prompts of 2048 tokens brought into a fresh 4-bit cache
        _append("append_8x2048", 8, 2048, 16, 8, 128, 64, "bf16", 64, 2048, True, False),
        # a ragged chunk of a padded batch: odd sizes, a page of 24 rows, no norms
        _append("append_odd", 5, 77, 6, 2, 64, 64, "fp16", 24, 500, False, True),
        # one request in the middle of a chat: the smallest attention, all latency
        _attend("attend_1x1024", 1, 16, 8, 128, 128, "bf16", 16, 1024, 1024, False),
        # a full batch with ragged caches
        _attend("attend_64x4096", 64, 16, 8, 128, 128, "bf16", 16, 256, 4096, False),
        # four long documents
        _attend("attend_4x131072", 4, 16, 8, 128, 64, "bf16", 64, 131072, 131072, False),
        # odd sizes: empty and one-token caches among them, skipped first slots
        _attend("attend_odd", 17, 12, 2, 64, 64, "fp16", 24, 0, 2999, True),
        # what a step's attention gave to each cached token, a full batch on 16-bit pages
        _weigh("weigh_64x4096", 64, 1, 16, 8, 128, 0, "bf16", 16, 256, 4096, False),
        # the last 16 queries of long 4-bit caches, ahead of an eviction
        _weigh("weigh_window_4x16384", 4, 16, 16, 8, 128, 128, "bf16", 64, 9000, 16384, True),
        # a batch cut to 1024 tokens a request, 16-bit pages
        _evict("evict_32x4096", 32, 8, 128, 0, "bf16", 16, 800, 4096, 1024, 4, 256),
        # odd sizes on 4-bit pages: short and empty caches among them, many equal weights
        _evict("evict_odd", 7, 2, 64, 64, "fp16", 24, 0, 1501, 333, 3, 50),
    ]


def _append(name, batch, seq, hq, hkv, dim, group, dtype, page, cap, norm, ragged):
    return {"name": name, "op": "append", "batch": batch, "seq": seq, "hq": hq, "hkv": hkv, "dim": dim, "group": group,
            "dtype": dtype, "page": page, "cap": cap, "norm": norm, "ragged": ragged}


def _attend(name, batch, hq, hkv, dim, group, dtype, page, lo, hi, starts):
    return {"name": name, "op": "attend", "batch": batch, "hq": hq, "hkv": hkv, "dim": dim, "group": group,
            "dtype": dtype, "page": page, "lo": lo, "hi": hi, "starts": starts}


def _weigh(name, batch, seq, hq, hkv, dim, group, dtype, page, lo, hi, starts):
    """group 0: pages of the queries' own type."""
    return {"name": name, "op": "weigh", "batch": batch, "seq": seq, "hq": hq, "hkv": hkv, "dim": dim, "group": group,
            "dtype": dtype, "page": page, "lo": lo, "hi": hi, "starts": starts}


def _evict(name, batch, hkv, dim, group, dtype, page, lo, hi, keep, first, last):
    return {"name": name, "op": "evict", "batch": batch, "hkv": hkv, "dim": dim, "group": group, "dtype": dtype,
            "page": page, "lo": lo, "hi": hi, "keep": keep, "first": first, "last": last}


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["append", "attend", "weigh", "evict"])
    dtype = rng.choice(["bf16", "fp16"])
    hq, hkv = rng.choice([(16, 8), (8, 8), (12, 2), (32, 4), (20, 4), (6, 2), (16, 1)])
    dim = rng.choice([64, 128, 128])
    group = rng.choice([64, dim])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    flip = lambda: rng.random() < 0.5  # noqa: E731
    batch = _spread(rng, 1, 64)
    if op == "append":
        seq = 1 if flip() else _spread(rng, 2, 16384 // batch)
        case = _append("", batch, seq, hq, hkv, dim, group, dtype, page, seq + _spread(rng, 16, 2048), flip(), flip())
    elif op == "attend":
        hi = _spread(rng, 32, min(131072, 262144 // batch))
        case = _attend("", batch, hq, hkv, dim, group, dtype, page, rng.choice([0, 1, hi // 2, hi]), hi, flip())
    elif op == "weigh":
        seq = 1 if flip() else _spread(rng, 2, 32)
        hi = _spread(rng, 32, min(65536, 262144 // batch // seq))
        case = _weigh("", batch, seq, hq, hkv, dim, rng.choice([0, group]), dtype, page,
                      rng.choice([0, 1, hi // 2, hi]), hi, flip())
    else:
        hi = _spread(rng, 32, min(65536, 131072 // batch))
        keep = _spread(rng, 8, hi)
        first = rng.choice([0, 1, min(4, keep)])
        case = _evict("", batch, hkv, dim, rng.choice([0, group]), dtype, page, rng.choice([0, 1, hi // 2, hi]), hi,
                      keep, first, rng.choice([0, 1, (keep - first) // 3, keep - first]))
    return {k: v for k, v in case.items() if k != "name"}


def _lengths(case):
    """The cached lengths and first valid slots of a batch: spread evenly over
    the case's range in a shuffled order, the same for every seed."""
    lo, hi, n = case["lo"], case["hi"], case["batch"]
    lens = [lo + int((hi - lo) * ((0.6180339887 * i + 0.37) % 1.0) + 0.5) for i in range(n)]
    if n > 2 and lo == 0:
        lens[1], lens[2] = 0, 1  # an empty cache and a cache of one token
    if n > 1:
        lens[0] = hi
    starts = [int(length * 0.4 * ((0.7548776662 * i + 0.2) % 1.0)) for i, length in enumerate(lens)]
    return lens, starts if case.get("starts") else [0] * n


def _counts(case):
    """How many of a padded batch's tokens are real, a request each."""
    n, s = case["batch"], case["seq"]
    return [1 + int((s - 1) * ((0.6180339887 * i + 0.9) % 1.0) + 0.5) for i in range(n)] if case["ragged"] else [s] * n


# ------------------------------------------------------------------ the inputs


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    return {"append": _prepare_append, "attend": _prepare_attend, "weigh": _prepare_weigh,
            "evict": _prepare_evict}[case["op"]](case, g)


def _randn(g, dtype, *shape):
    return torch.randn(shape, generator=g, device=_DEV, dtype=torch.float32).to(dtype)


def _table(case, capacity, g):
    """How many pages there are, and each request's page numbers in the order of its tokens."""
    per = -(-capacity // case["page"])
    pages = case["batch"] * per + 3
    table = torch.randperm(pages, generator=g, device=_DEV)[: case["batch"] * per].to(torch.int32)
    return pages, table.view(case["batch"], per).contiguous()


def _pages(case, pages, g):
    """Pages of normal values: of the case's type, or (codes, scales) of 4 bits: codes
    [P, Hkv, page, D / 2] (even d in the low half of a byte) and (scale, least value)
    of each group of a row, as rounding such values leaves them."""
    shape, dt = (pages, case["hkv"], case["page"], case["dim"]), _DT[case["dtype"]]
    if not case["group"]:
        return torch.empty(shape, device=_DEV, dtype=dt).normal_(generator=g)
    q = torch.empty(shape, device=_DEV, dtype=torch.float16).normal_(7.5, 2.9, generator=g)
    q = q.round_().clamp_(0, 15).to(torch.uint8)
    scales = torch.empty(*shape[:3], case["dim"] // case["group"], 2, device=_DEV, dtype=torch.float32)
    scales[..., 0].uniform_(0.25, 0.45, generator=g)
    scales[..., 1].uniform_(-3.2, -2.0, generator=g)
    return q[..., 0::2] | (q[..., 1::2] << 4), scales.to(dt)


def _prepare_append(case, g):
    b, s, d, dt = case["batch"], case["seq"], case["dim"], _DT[case["dtype"]]
    pages, table = _table(case, case["cap"], g)
    shape = (pages, case["hkv"], case["page"])
    kv = [(torch.zeros(*shape, d // 2, device=_DEV, dtype=torch.uint8),
           torch.zeros(*shape, d // case["group"], 2, device=_DEV, dtype=dt)) for _ in range(2)]
    # projections come as [B, S, H, D] and are passed as [B, H, S, D] views
    q, k, v = (_randn(g, dt, b, s, h, d).transpose(1, 2) for h in (case["hq"], case["hkv"], case["hkv"]))
    pos = torch.randint(0, case["cap"] - s + 1, (b,), generator=g, device=_DEV, dtype=torch.int64)
    inv = 5e6 ** (-torch.arange(0, d, 2, device=_DEV, dtype=torch.float64) / d)
    ang = (pos[:, None] + torch.arange(s, device=_DEV))[..., None].double() * inv
    ang = torch.cat([ang, ang], -1)
    w = [1 + 0.2 * _randn(g, torch.float32, d) for _ in range(2)] if case["norm"] else [None, None]
    return {"case": case, "q": q, "k": k, "v": v, "cos": ang.cos().float(), "sin": ang.sin().float(), "kp": kv[0],
            "vp": kv[1], "table": table, "pos": pos.to(torch.int32),
            "new": torch.tensor(_counts(case), dtype=torch.int32, device=_DEV) if case["ragged"] else None,
            "lens": torch.zeros(b, dtype=torch.int32, device=_DEV),
            "qw": None if w[0] is None else w[0].to(dt), "kw": None if w[1] is None else w[1].to(dt)}


def _bounds(case):
    lens, starts = _lengths(case)
    return {"lens": torch.tensor(lens, dtype=torch.int32, device=_DEV),
            "starts": torch.tensor(starts, dtype=torch.int32, device=_DEV) if case.get("starts") else None}


def _prepare_attend(case, g):
    pages, table = _table(case, max(1, case["hi"]), g)
    return {"case": case, "q": _randn(g, _DT[case["dtype"]], case["batch"], case["hq"], 1, case["dim"]),
            "kp": _pages(case, pages, g), "vp": _pages(case, pages, g), "table": table} | _bounds(case)


def _prepare_weigh(case, g):
    b, hq, s = case["batch"], case["hq"], case["seq"]
    pages, table = _table(case, max(1, case["hi"]), g)
    st = {"case": case, "q": _randn(g, _DT[case["dtype"]], b, hq, s, case["dim"]), "kp": _pages(case, pages, g),
          "table": table} | _bounds(case)
    # the log-sum-exp that the queries' attention returned, and what a few earlier steps added up
    st["lse"] = (torch.logsumexp(_window_scores(st), -1) / math.log(2.0)).reshape(b, hq, s)
    st["weights"] = torch.rand(b, case["hkv"], table.shape[1] * case["page"], generator=g, device=_DEV) * (4 / case["hi"])
    return st


def _prepare_evict(case, g):
    pages, table = _table(case, max(1, case["hi"]), g)
    # sums of attention weights: a few large, most small; on odd pages many are equal
    w = torch.rand(case["batch"], case["hkv"], table.shape[1] * case["page"], generator=g, device=_DEV).pow(6)
    if case["page"] % 16:
        w = (w * 64).floor() / 64
    return {"case": case, "kp": _pages(case, pages, g), "vp": _pages(case, pages, g), "table": table, "weights": w,
            "new_weights": torch.zeros_like(w), "new_lens": torch.zeros(case["batch"], dtype=torch.int32, device=_DEV),
            "zero": torch.zeros(case["batch"], dtype=torch.int32, device=_DEV)} | _bounds(case)


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "weigh": _own_weigh, "evict": _own_evict}[op](state)
    return {"append": _plain_append, "attend": _plain_attend, "weigh": _plain_weigh, "evict": _plain_evict}[op](state)


def _own_append(st):
    import aicas_b200 as ab

    kp, vp = ab.Int4Pages(*st["kp"]), ab.Int4Pages(*st["vp"])
    q = ab.paged_rope_kv_append_int4(st["q"], st["k"], st["v"], st["cos"], st["sin"], kp, vp, st["table"], st["pos"],
                                     num_new=st["new"], kv_lens_out=st["lens"], q_norm_weight=st["qw"],
                                     k_norm_weight=st["kw"], eps=_EPS)
    k, v = ab.paged_kv_read_int4(kp, vp, st["table"], st["pos"], st["case"]["seq"], num_tokens=st["new"])
    return {"q": q, "k": k, "v": v, "lens": st["lens"]}


def _own_attend(st):
    import aicas_b200 as ab

    c = st["case"]
    out, lse = ab.paged_gqa_decode_attention_int4(
        st["q"], ab.Int4Pages(*st["kp"]), ab.Int4Pages(*st["vp"]), st["table"], sm_scale=c["dim"] ** -0.5,
        num_key_value_groups=c["hq"] // c["hkv"], kv_lens=st["lens"], kv_starts=st["starts"], return_lse=True)
    return {"out": out, "lse": lse}


def _own_weigh(st):
    import aicas_b200 as ab

    c = st["case"]
    return ab.paged_attention_weights(
        st["q"], ab.Int4Pages(*st["kp"]) if c["group"] else st["kp"], st["table"], st["lse"], st["weights"],
        sm_scale=c["dim"] ** -0.5, num_key_value_groups=c["hq"] // c["hkv"], kv_lens=st["lens"],
        kv_starts=st["starts"])


def _own_evict(st):
    import aicas_b200 as ab

    c = st["case"]
    kp, vp = (ab.Int4Pages(*p) if c["group"] else p for p in (st["kp"], st["vp"]))
    kept = ab.paged_kv_evict(kp, vp, st["table"], st["weights"], st["lens"], keep=c["keep"], keep_first=c["first"],
                             keep_last=c["last"], kv_lens_out=st["new_lens"], weights_out=st["new_weights"])
    if c["group"]:
        kp, vp = ab.paged_kv_read_int4(kp, vp, st["table"], st["zero"], c["keep"], num_tokens=st["new_lens"])
    return {"kept": kept, "lens": st["new_lens"], "weights": st["new_weights"], "k": kp, "v": vp}


def _rotated(x, w, cos, sin):
    """Norm (where there is a weight) and rotation of [B, H, S, D] in 32 bits."""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS) * w.float()
    h = y.shape[-1] // 2
    turned = torch.cat([-y[..., h:], y[..., :h]], -1)
    return y * cos[:, None] + turned * sin[:, None]


def _rounded(x, group, dtype):
    """(codes, scales) of rows [..., D] in 32 bits: the least value of a group and a
    fifteenth of its range in the cache's type, codes to the nearest level."""
    y = x.unflatten(-1, (-1, group))
    least = y.amin(-1).to(dtype)
    scale = ((y.amax(-1) - least.float()) / 15).to(dtype)
    step = scale.float()[..., None]
    q = torch.where(step > 0, (y - least.float()[..., None]) / torch.where(step > 0, step, 1.0), 0.0)
    q = q.round().clamp(0, 15).to(torch.uint8).flatten(-2)
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.stack([scale, least], -1)


def _widened(codes, scales):
    """The 32-bit values [..., D] that codes and scales stand for."""
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (scales.shape[-2], -1)).float()
    s = scales.float()
    return (q * s[..., :1] + s[..., 1:]).flatten(-2)


def _in_order(page_part, table):
    """Pages [P, Hkv, page, ...] as the requests' rows [B, Hkv, slots, ...]."""
    return page_part[table.long()].transpose(1, 2).flatten(2, 3)


def _cached(pages, table):
    """The 32-bit rows [B, Hkv, slots, D] of 16-bit or 4-bit pages."""
    if isinstance(pages, tuple):
        return _widened(*(_in_order(p, table) for p in pages))
    return _in_order(pages, table).float()


def _plain_append(st):
    c = st["case"]
    s, page, dt = c["seq"], c["page"], _DT[c["dtype"]]
    q = _rotated(st["q"], st["qw"], st["cos"], st["sin"]).to(dt)
    new = st["new"] if st["new"] is not None else torch.full_like(st["pos"], s)
    # padding writes the last real token of its request once more
    tok = torch.minimum(torch.arange(s, device=q.device)[None], new[:, None].long() - 1)
    slot = st["pos"][:, None].long() + tok
    page_no = torch.gather(st["table"].long(), 1, slot // page)
    row = slot % page
    request = torch.arange(c["batch"], device=q.device)[:, None]
    real = (torch.arange(s, device=q.device)[None] < new[:, None])[:, None, :, None]

    def through(pages, x):
        """Rows [B, Hkv, S, D] into the pages, and from there what they became."""
        codes, scales = (p.transpose(1, 2)[request, tok] for p in _rounded(x, c["group"], dt))
        pages[0][page_no, :, row] = codes
        pages[1][page_no, :, row] = scales
        back = _widened(pages[0][page_no, :, row], pages[1][page_no, :, row]).transpose(1, 2)
        return torch.where(real, back, 0.0).to(dt)

    k = through(st["kp"], _rotated(st["k"], st["kw"], st["cos"], st["sin"]))
    v = through(st["vp"], st["v"].float())
    st["lens"].copy_(st["pos"] + new)
    return {"q": q, "k": k, "v": v, "lens": st["lens"]}


def _plain_attend(st):
    c = st["case"]
    b, hq, hkv, d = c["batch"], c["hq"], c["hkv"], c["dim"]
    k, v = (_cached(p, st["table"]) for p in (st["kp"], st["vp"]))
    q = st["q"].float().view(b, hkv, hq // hkv, d)
    s = torch.matmul(q, k.transpose(2, 3)) * d ** -0.5
    at = torch.arange(s.shape[-1], device=s.device)[None]
    seen = at < st["lens"][:, None]
    if st["starts"] is not None:
        seen = seen & (at >= st["starts"][:, None])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = (m + torch.log(total)) / math.log(2.0)
    return {"out": o.reshape(b, hq, 1, d).to(st["q"].dtype), "lse": lse.reshape(b, hq)}


def _window_scores(st):
    """[B, Hkv, queries of the group, slots] in 32 bits, -inf where a query sees nothing:
    the window's query i is the token at slot len - S + i and sees those up to its own."""
    c = st["case"]
    b, hq, hkv, s, d = c["batch"], c["hq"], c["hkv"], c["seq"], c["dim"]
    k = _cached(st["kp"], st["table"])
    scores = torch.matmul(st["q"].float().reshape(b, hkv, hq // hkv * s, d), k.transpose(2, 3)) * d ** -0.5
    at = torch.arange(k.shape[2], device=k.device)
    end = st["lens"][:, None] - s + 1 + torch.arange(s, device=k.device)[None]
    seen = at < end[..., None]
    if st["starts"] is not None:
        seen = seen & (at >= st["starts"][:, None, None])
    seen = seen[:, None].expand(-1, hq // hkv, -1, -1).reshape(b, 1, hq // hkv * s, -1)
    return scores.masked_fill(~seen, -math.inf)


def _plain_weigh(st):
    c = st["case"]
    scores = _window_scores(st)
    lse = st["lse"].reshape(c["batch"], c["hkv"], -1, 1) * math.log(2.0)
    given = torch.exp(scores - torch.where(lse == -math.inf, 0.0, lse))
    st["weights"] += given.sum(2)
    return st["weights"]


def _plain_evict(st):
    c = st["case"]
    keep, w, page = c["keep"], st["weights"], c["page"]
    slots = w.shape[2]
    at = torch.arange(slots, device=w.device)
    lens = st["lens"].long()[:, None, None]
    # what must stay comes first, then by weight, then what is not there
    rank = torch.where(at < c["first"], math.inf, w)
    rank = torch.where(at >= lens - c["last"], math.inf, rank)
    rank = torch.where(at < lens, rank, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    order = order[..., : min(keep, slots)]
    order = torch.sort(torch.where(order < lens, order, slots), dim=-1).values
    kept = torch.full((*w.shape[:2], keep), -1, device=w.device, dtype=torch.int32)
    kept[..., : order.shape[-1]] = torch.where(order < slots, order, -1).to(torch.int32)
    cut = lens > keep
    # the kept rows to the front, in their order; shorter caches stay as they are
    src = torch.where(order < slots, order, 0)
    dst = torch.arange(src.shape[-1], device=w.device).expand_as(src)
    src = torch.where(cut, src, dst)
    request = torch.arange(c["batch"], device=w.device)[:, None, None]
    head = torch.arange(c["hkv"], device=w.device)[None, :, None]
    table = st["table"].long()
    new_w = torch.where(cut & (at >= keep), 0.0, w)
    new_w[..., : src.shape[-1]] = torch.gather(w, 2, src)
    st["new_weights"].copy_(torch.where(at < lens, new_w, st["new_weights"]))
    for_all = lambda p: p if isinstance(p, tuple) else (p,)  # noqa: E731

    def moved(part):
        part[table[request, dst // page], head, dst % page] = part[table[request, src // page], head, src % page]
        return part

    kp, vp = (tuple(map(moved, for_all(p))) for p in (st["kp"], st["vp"]))
    st["new_lens"].copy_(st["lens"].clamp(max=keep))
    if not c["group"]:
        return {"kept": kept, "lens": st["new_lens"], "weights": st["new_weights"], "k": kp[0], "v": vp[0]}
    live = (at[:keep] < st["new_lens"][:, None])[:, None, :, None]

    def front(pages):
        rows = _cached(pages, st["table"])[:, :, :keep]
        rows = torch.where(live, rows, 0.0).to(_DT[c["dtype"]])
        return torch.cat([rows, rows.new_zeros(*rows.shape[:2], keep - rows.shape[2], c["dim"])], 2)

    return {"kept": kept, "lens": st["new_lens"], "weights": st["new_weights"], "k": front(kp), "v": front(vp)}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    d, hkv, group = case["dim"], case["hkv"], case["group"]
    row = d // 2 + 4 * (d // group) if group else 2 * d  # bytes of a cached row of one head
    if case["op"] == "append":
        tokens, all_tokens = sum(_counts(case)), case["batch"] * case["seq"]
        hq = case["hq"]
        moved = 4 * d * hq * all_tokens + all_tokens * d * 8 + case["batch"] * 12
        # k and v in, their rows of 4 bits out, and what those stand for
        moved += 2 * hkv * (tokens * (2 * d + row) + all_tokens * 2 * d)
        return {"bytes": moved, "flops": d * (hq * all_tokens + hkv * tokens) * (7 if case["norm"] else 3)
                + 12 * d * hkv * tokens}
    lens, starts = _lengths(case)
    if case["op"] == "attend":
        slots, hq = sum(a - z for a, z in zip(lens, starts)), case["hq"]
        pages = sum(-(-a // case["page"]) for a in lens)
        return {"bytes": slots * hkv * 2 * row + case["batch"] * hq * (4 * d + 4) + 4 * pages,
                "flops": 4 * slots * hq * d}
    if case["op"] == "weigh":
        slots, s, hq = sum(a - z for a, z in zip(lens, starts)), case["seq"], case["hq"]
        pages = sum(-(-a // case["page"]) for a in lens)
        return {"bytes": slots * hkv * (row + 8) + case["batch"] * hq * s * (2 * d + 4) + 4 * pages,
                "flops": 2 * slots * hq * s * d}
    keep, first, last = case["keep"], case["first"], case["last"]
    moved = flops = 0
    for length in lens:
        n = min(length, keep)
        moved += hkv * (4 * n + 8 * length) + 8  # the kept slots' numbers, the weights in and out, the lengths
        if length > keep:  # rows move but for those that must stay in front
            moved += hkv * 2 * 2 * row * (keep - first)
            flops += hkv * (length - first - last)
        if group:  # the kept rows that do not move are read all the same
            moved += 2 * hkv * row * (first if length > keep else n)
    if group:
        moved += 2 * hkv * case["batch"] * keep * 2 * d  # and written as 16-bit values
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "weigh": _exact_weigh,
            "evict": _exact_evict}[case["op"]](st)


def _values(codes, scales):
    """Rows [..., D] of (codes, scales) in 64 bits."""
    out = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], device=codes.device, dtype=torch.float64)
    out[..., 0::2] = (codes % 16).double()
    out[..., 1::2] = (codes // 16).double()
    each = out.shape[-1] // scales.shape[-2]
    scale, least = (scales[..., i].double().repeat_interleave(each, -1) for i in (0, 1))
    return out * scale + least


def _exact_append(st):
    c, d = st["case"], st["case"]["dim"]
    half, dt, b, s = d // 2, _DT[c["dtype"]], c["batch"], c["seq"]
    cos, sin = st["cos"].double(), st["sin"].double()

    def turn(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + _EPS) * w.double()
        out = torch.empty_like(x)
        a, z = x[..., :half], x[..., half:]
        out[..., :half] = a * cos[:, None, :, :half] - z * sin[:, None, :, :half]
        out[..., half:] = z * cos[:, None, :, half:] + a * sin[:, None, :, half:]
        return out

    def held(x):
        """What a 4-bit row of x is worth, a group at a time."""
        out = torch.empty_like(x)
        for g0 in range(0, d, c["group"]):
            y = x[..., g0 : g0 + c["group"]]
            least = y.min(-1, keepdim=True).values.to(dt).double()
            step = ((y.max(-1, keepdim=True).values - least) / 15).to(dt).double()
            code = torch.clamp(torch.round((y - least) / step), 0, 15)
            out[..., g0 : g0 + c["group"]] = torch.where(step > 0, least + code * step, least)
        for i, n in enumerate(_counts(c)):
            out[i, :, n:] = 0
        return out

    lens = [p + n for p, n in zip(st["pos"].tolist(), _counts(c))]
    return {"q": turn(st["q"], st["qw"]), "k": held(turn(st["k"], st["kw"])), "v": held(st["v"].double()),
            "lens": torch.tensor(lens, dtype=torch.int32)}


def _exact_rows(pages, rows, head, d):
    """Every slot of one request and head, [slots, D] in 64 bits."""
    if isinstance(pages, tuple):
        return _values(*(p[rows, head].flatten(0, 1) for p in pages))
    return pages[rows, head].reshape(-1, d).double()


def _exact_attend(st):
    c = st["case"]
    lens, starts = _lengths(c)
    hq, hkv, d = c["hq"], c["hkv"], c["dim"]
    out = torch.zeros(c["batch"], hq, 1, d, dtype=torch.float64, device=_DEV)
    lse = torch.full((c["batch"], hq), -math.inf, dtype=torch.float64, device=_DEV)
    for b in range(c["batch"]):
        if lens[b] <= starts[b]:
            continue
        rows = st["table"][b].long()
        for h in range(hkv):
            k, v = (_exact_rows(st[p], rows, h, d)[starts[b] : lens[b]] for p in ("kp", "vp"))
            mine = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            s = st["q"][b, mine, 0].double() @ k.t() / math.sqrt(d)
            out[b, mine, 0] = torch.softmax(s, -1) @ v
            lse[b, mine] = torch.logsumexp(s, -1) / math.log(2.0)
    return {"out": out, "lse": lse}


def _exact_weigh(st):
    c = st["case"]
    lens, starts = _lengths(c)
    hq, hkv, d, s = c["hq"], c["hkv"], c["dim"], c["seq"]
    out = st["weights"].double()
    for b in range(c["batch"]):
        rows = st["table"][b].long()
        for h in range(hkv):
            k = _exact_rows(st["kp"], rows, h, d)
            for i in range(s):
                end = lens[b] - s + 1 + i
                if end <= starts[b]:
                    continue
                for j in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                    score = k[starts[b] : end] @ st["q"][b, j, i].double() / math.sqrt(d)
                    out[b, h, starts[b] : end] += torch.exp(score - st["lse"][b, j, i].double() * math.log(2.0))
    return out


def _exact_evict(st):
    c = st["case"]
    lens, page, keep = _lengths(c)[0], c["page"], c["keep"]
    weights = st["weights"].cpu().clone()
    new_weights = torch.zeros_like(weights)
    kept = torch.full((c["batch"], c["hkv"], keep), -1, dtype=torch.int32)
    wide = [p.double() for p in (st["kp"], st["vp"])] if not c["group"] else \
        [torch.zeros(c["batch"], c["hkv"], keep, c["dim"], dtype=torch.float64, device=_DEV) for _ in range(2)]
    for b, n in enumerate(lens):
        rows = st["table"][b].long()
        for h in range(c["hkv"]):
            if n > keep:
                w = weights[b, h, :n].clone()
                each = w.tolist()
                middle = sorted(range(c["first"], n - c["last"]), key=lambda t: (-each[t], t))
                mine = sorted([*range(c["first"]), *middle[: keep - c["first"] - c["last"]], *range(n - c["last"], n)])
                new_weights[b, h, :keep] = w[mine]
            else:
                mine = list(range(n))
                new_weights[b, h, :n] = weights[b, h, :n]
            kept[b, h, : len(mine)] = torch.tensor(mine, dtype=torch.int32)
            at = torch.tensor(mine, dtype=torch.long, device=_DEV)
            to = torch.arange(len(mine), device=_DEV)
            for out, p in zip(wide, (st["kp"], st["vp"])):
                if c["group"]:
                    out[b, h, : len(mine)] = _exact_rows(p, rows, h, c["dim"])[at]
                else:
                    out[rows[to // page], h, to % page] = p[rows[at // page], h, at % page].double()
    return {"kept": kept, "lens": torch.tensor([min(n, keep) for n in lens], dtype=torch.int32),
            "weights": new_weights.double(), "k": wide[0], "v": wide[1]}
