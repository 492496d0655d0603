"""The paged key-value cache and 4-bit weight operators as measured cases: their
plain form in elementary torch operations, the same calls on the framework's
kernels, and the 64-bit definition.

The text decoder served here has 16 query and 8 key-value heads of 128, a hidden
size of 2048, an MLP of 6144 and a vocabulary of 151936; its caches hold up to
4096 tokens a request in a batch of 64, or 131072 tokens in a batch of 4.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # one new token of a single request: the smallest append, all latency
        _append("append_1x1", 1, 1, 16, 8, 128, "bf16", 16, 1024, True, False),
        # the decode step of a full batch, one token each at ragged positions
        _append("append_64x1", 64, 1, 16, 8, 128, "bf16", 16, 4096, True, False),
        # eight prompts of 2048 tokens brought into a fresh paged cache
        _append("append_8x2048", 8, 2048, 16, 8, 128, "bf16", 64, 2048, True, False),
        # a ragged chunk of a padded batch: odd sizes, a page of 24 rows, no norms
        _append("append_odd", 5, 77, 6, 2, 64, "fp16", 24, 500, False, True),
        # one request in the middle of a chat: the smallest attention, all latency
        _attend("attend_1x1024", 1, 16, 8, 128, "bf16", 16, 1024, 1024, False),
        # a full batch with ragged caches
        _attend("attend_64x4096", 64, 16, 8, 128, "bf16", 16, 256, 4096, False),
        # four long documents
        _attend("attend_4x131072", 4, 16, 8, 128, "bf16", 64, 131072, 131072, False),
        # odd sizes: empty and one-token caches among them, skipped first slots
        _attend("attend_odd", 17, 12, 2, 64, "fp16", 24, 0, 2999, True),
        # q, k and v of one token, with the norm before them
        _linear("int4_qkv_1", 1, 2048, 4096, 128, "bf16", True, False, False, False),
        # gate and up of eight tokens, normalised, SiLU * up
        _linear("int4_gate_up_8", 8, 2048, 6144, 128, "bf16", True, False, True, True),
        # the down projection of 32 tokens added to the residual stream
        _linear("int4_down_32", 32, 6144, 2048, 64, "fp16", False, True, False, True),
        # the vocabulary product of one token, the largest weight of the model
        _linear("int4_head_1", 1, 2048, 151936, 128, "bf16", True, False, False, False),
    ]


def _append(name, batch, seq, hq, hkv, dim, dtype, page, cap, norm, ragged):
    return {"name": name, "op": "append", "batch": batch, "seq": seq, "hq": hq, "hkv": hkv, "dim": dim,
            "dtype": dtype, "page": page, "cap": cap, "norm": norm, "ragged": ragged}


def _attend(name, batch, hq, hkv, dim, dtype, page, lo, hi, starts):
    return {"name": name, "op": "attend", "batch": batch, "hq": hq, "hkv": hkv, "dim": dim, "dtype": dtype,
            "page": page, "lo": lo, "hi": hi, "starts": starts}


def _linear(name, rows, k, n, group, dtype, norm, residual, swiglu, zeros):
    return {"name": name, "op": "int4", "rows": rows, "k": k, "n": n, "group": group, "dtype": dtype,
            "norm": norm, "residual": residual, "swiglu": swiglu, "zeros": zeros}


def _spread(rng, lo, hi, multiple=1):
    """A whole number of [lo, hi], spread over its logarithm, of the given multiple."""
    while True:
        v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))
        v = max(lo, min(hi, v // multiple * multiple))
        if v != 3072:
            return v


def draw(rng):
    op = rng.choice(["append", "attend", "int4"])
    dtype = rng.choice(["bf16", "fp16"])
    heads = rng.choice([(16, 8), (8, 8), (12, 2), (32, 4), (20, 4), (6, 2), (16, 1)])
    dim = rng.choice([64, 128, 128])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    flip = lambda: rng.random() < 0.5  # noqa: E731
    if op == "append":
        batch = _spread(rng, 1, 64)
        seq = 1 if flip() else _spread(rng, 2, 16384 // batch)
        cap = seq + _spread(rng, 16, 2048)
        cap += cap == 3072
        return {k: v for k, v in _append("", batch, seq, *heads, dim, dtype, page, cap, flip(), flip()).items()
                if k != "name"}
    if op == "attend":
        batch = _spread(rng, 1, 64)
        hi = _spread(rng, 32, min(131072, 262144 // batch))
        lo = rng.choice([0, 1, hi // 2, hi])
        return {k: v for k, v in _attend("", batch, *heads, dim, dtype, page, lo, hi, flip()).items() if k != "name"}
    group = rng.choice([32, 64, 128, 128])
    swiglu = rng.random() < 0.3
    return {k: v for k, v in _linear("", _spread(rng, 1, 32), _spread(rng, 512, 8192, group),
                                     _spread(rng, 100, 24000), group, dtype, flip(), not swiglu and flip(), swiglu,
                                     flip()).items() if k != "name"}


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
    return lens, starts if case["starts"] else [0] * n


def _counts(case):
    """How many of a padded batch's tokens are real, a request each."""
    n, s = case["batch"], case["seq"]
    return [1 + int((s - 1) * ((0.6180339887 * i + 0.9) % 1.0) + 0.5) for i in range(n)] if case["ragged"] else [s] * n


# ------------------------------------------------------------------ the inputs


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    return {"append": _prepare_append, "attend": _prepare_attend, "int4": _prepare_int4}[case["op"]](case, g)


def _randn(g, dtype, *shape):
    return torch.randn(shape, generator=g, device=_DEV, dtype=torch.float32).to(dtype)


def _pool(case, capacity, g):
    """A pool of pages and each request's page numbers in the order of its tokens."""
    per = -(-capacity // case["page"])
    pages = case["batch"] * per + 3
    table = torch.randperm(pages, generator=g, device=_DEV)[: case["batch"] * per].to(torch.int32)
    shape = (pages, case["hkv"], case["page"], case["dim"])
    dt = _DT[case["dtype"]]
    return _pages(g, dt, shape), _pages(g, dt, shape), table.view(case["batch"], per).contiguous()


def _pages(g, dtype, shape):
    out = torch.empty(shape, device=_DEV, dtype=dtype)
    return out.normal_(generator=g)


def _prepare_append(case, g):
    b, s, d, dt = case["batch"], case["seq"], case["dim"], _DT[case["dtype"]]
    kp, vp, table = _pool(case, case["cap"], g)
    # projections come as [B, S, H, D] and are passed as [B, H, S, D] views
    q, k, v = (_randn(g, dt, b, s, h, d).transpose(1, 2) for h in (case["hq"], case["hkv"], case["hkv"]))
    pos = torch.randint(0, case["cap"] - s + 1, (b,), generator=g, device=_DEV, dtype=torch.int64)
    inv = 5e6 ** (-torch.arange(0, d, 2, device=_DEV, dtype=torch.float64) / d)
    ang = (pos[:, None] + torch.arange(s, device=_DEV))[..., None].double() * inv
    ang = torch.cat([ang, ang], -1)
    w = [1 + 0.2 * _randn(g, torch.float32, d) for _ in range(2)] if case["norm"] else [None, None]
    return {"case": case, "q": q, "k": k, "v": v, "cos": ang.cos().float(), "sin": ang.sin().float(), "kp": kp,
            "vp": vp, "table": table, "pos": pos.to(torch.int32),
            "new": torch.tensor(_counts(case), dtype=torch.int32, device=_DEV) if case["ragged"] else None,
            "lens": torch.zeros(b, dtype=torch.int32, device=_DEV),
            "qw": None if w[0] is None else w[0].to(dt), "kw": None if w[1] is None else w[1].to(dt)}


def _prepare_attend(case, g):
    lens, starts = _lengths(case)
    kp, vp, table = _pool(case, max(1, case["hi"]), g)
    return {"case": case, "q": _randn(g, _DT[case["dtype"]], case["batch"], case["hq"], 1, case["dim"]), "kp": kp,
            "vp": vp, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device=_DEV),
            "starts": torch.tensor(starts, dtype=torch.int32, device=_DEV) if case["starts"] else None}


def _int4_weight(case, g):
    """A weight of N rows in 4 bits: [N, K/2] bytes (even k in the low half),
    scales and, for the asymmetric kind, zero points of each group along K."""
    n, k, groups = case["n"], case["k"], case["k"] // case["group"]
    q = torch.empty(n, k, device=_DEV, dtype=torch.float16).normal_(8.0, 3.0, generator=g)
    q = q.round_().clamp_(0, 15).to(torch.uint8)
    scales = (0.5 + torch.rand(n, groups, generator=g, device=_DEV)) / (3 * math.sqrt(k))
    zeros = torch.randint(5, 12, (n, groups), generator=g, device=_DEV, dtype=torch.uint8) if case["zeros"] else None
    return q[:, 0::2] | (q[:, 1::2] << 4), scales.to(_DT[case["dtype"]]), zeros


def _prepare_int4(case, g):
    dt = _DT[case["dtype"]]
    weight = [_int4_weight(case, g) for _ in range(2)] if case["swiglu"] else _int4_weight(case, g)
    return {"case": case, "x": _randn(g, dt, case["rows"], case["k"]), "w": weight,
            "nw": (1 + 0.2 * _randn(g, torch.float32, case["k"])).to(dt) if case["norm"] else None,
            "res": _randn(g, dt, case["rows"], case["n"]) if case["residual"] else None}


# ------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "int4": _own_int4}[op](state)
    return {"append": _plain_append, "attend": _plain_attend, "int4": _plain_int4}[op](state)


def _own_append(st):
    import aicas_b200 as ab

    q = ab.paged_rope_kv_append(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["kp"], st["vp"], st["table"],
                                st["pos"], num_new=st["new"], kv_lens_out=st["lens"], q_norm_weight=st["qw"],
                                k_norm_weight=st["kw"], eps=1e-6)
    return {"q": q, "k_pages": st["kp"], "v_pages": st["vp"], "lens": st["lens"]}


def _own_attend(st):
    import aicas_b200 as ab

    c = st["case"]
    out, lse = ab.paged_gqa_decode_attention(st["q"], st["kp"], st["vp"], st["table"], sm_scale=c["dim"] ** -0.5,
                                             num_key_value_groups=c["hq"] // c["hkv"], kv_lens=st["lens"],
                                             kv_starts=st["starts"], return_lse=True)
    return {"out": out, "lse": lse}


def _own_int4(st):
    import aicas_b200 as ab

    c = st["case"]
    w = [ab.Int4Weight(*w) for w in st["w"]] if c["swiglu"] else ab.Int4Weight(*st["w"])
    return ab.decode_linear_int4(st["x"], w, norm_weight=st["nw"], eps=1e-6, residual=st["res"], swiglu=c["swiglu"])


def _rotated(x, w, cos, sin):
    """Norm (where there is a weight) and rotation of [B, H, S, D] in 32 bits."""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    h = y.shape[-1] // 2
    turned = torch.cat([-y[..., h:], y[..., :h]], -1)
    return (y * cos[:, None] + turned * sin[:, None]).to(x.dtype)


def _plain_append(st):
    c = st["case"]
    s, page = c["seq"], c["page"]
    q = _rotated(st["q"], st["qw"], st["cos"], st["sin"])
    k = _rotated(st["k"], st["kw"], st["cos"], st["sin"])
    new = st["new"] if st["new"] is not None else torch.full_like(st["pos"], s)
    # padding writes the last real token of its request once more
    tok = torch.minimum(torch.arange(s, device=q.device)[None], new[:, None].long() - 1)
    slot = st["pos"][:, None].long() + tok
    page_no = torch.gather(st["table"].long(), 1, slot // page)
    pick = tok[:, :, None, None]
    for_pages = lambda t: torch.gather(t.transpose(1, 2), 1, pick.expand(-1, -1, t.shape[1], t.shape[3]))  # noqa: E731
    st["kp"][page_no, :, slot % page] = for_pages(k)
    st["vp"][page_no, :, slot % page] = for_pages(st["v"])
    st["lens"].copy_(st["pos"] + new)
    return {"q": q, "k_pages": st["kp"], "v_pages": st["vp"], "lens": st["lens"]}


def _plain_attend(st):
    c = st["case"]
    b, hq, hkv, d = c["batch"], c["hq"], c["hkv"], c["dim"]
    k, v = (p[st["table"].long()].float().transpose(1, 2).reshape(b, hkv, -1, d) for p in (st["kp"], st["vp"]))
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


def _widened(weight):
    q, scales, zeros = weight
    n, groups = scales.shape
    q = torch.stack([q & 15, q >> 4], -1).view(n, groups, -1).float()
    z = 8.0 if zeros is None else zeros.float()[..., None]
    return ((q - z) * scales.float()[..., None]).view(n, -1)


def _plain_int4(st):
    c, x = st["case"], st["x"].float()
    if st["nw"] is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * st["nw"].float()
    if c["swiglu"]:
        gate, up = (torch.matmul(x, _widened(w).t()) for w in st["w"])
        y = gate / (1 + torch.exp(-gate)) * up
    else:
        y = torch.matmul(x, _widened(st["w"]).t())
    if st["res"] is not None:
        y = y + st["res"].float()
    return y.to(st["x"].dtype)


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    if case["op"] == "append":
        tokens, all_tokens = sum(_counts(case)), case["batch"] * case["seq"]
        d, hq, hkv = case["dim"], case["hq"], case["hkv"]
        moved = 2 * 2 * d * (hq * all_tokens + 2 * hkv * tokens) + all_tokens * d * 8 + case["batch"] * 12
        return {"bytes": moved, "flops": d * (hq * all_tokens + hkv * tokens) * (7 if case["norm"] else 3)}
    if case["op"] == "attend":
        lens, starts = _lengths(case)
        slots = sum(a - z for a, z in zip(lens, starts))
        pages = sum(-(-a // case["page"]) for a in lens)
        d, hq = case["dim"], case["hq"]
        return {"bytes": slots * case["hkv"] * d * 4 + case["batch"] * hq * (4 * d + 4) + 4 * pages,
                "flops": 4 * slots * hq * d}
    n, k, r = case["n"] * (2 if case["swiglu"] else 1), case["k"], case["rows"]
    groups = k // case["group"]
    moved = n * k // 2 + n * groups * (3 if case["zeros"] else 2) + 2 * r * (k + case["n"])
    moved += (2 * k if case["norm"] else 0) + (2 * r * case["n"] if case["residual"] else 0)
    return {"bytes": moved, "flops": 2 * r * n * k}


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "int4": _exact_int4}[case["op"]](st)


def _exact_append(st):
    c, half, page = st["case"], st["case"]["dim"] // 2, st["case"]["page"]
    cos, sin = st["cos"].double(), st["sin"].double()

    def turn(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6) * w.double()
        out = torch.empty_like(x)
        a, b = x[..., :half], x[..., half:]
        out[..., :half] = a * cos[:, None, :, :half] - b * sin[:, None, :, :half]
        out[..., half:] = b * cos[:, None, :, half:] + a * sin[:, None, :, half:]
        return out

    q, k = turn(st["q"], st["qw"]), turn(st["k"], st["kw"])
    kp, vp = st["kp"].double(), st["vp"].double()
    pos, table, ends = st["pos"].tolist(), st["table"].tolist(), []
    for b, n in enumerate(_counts(c)):
        ends.append(pos[b] + n)
        t = pos[b]
        while t < ends[b]:  # a page's worth at a time
            stop = min(ends[b], (t // page + 1) * page)
            rows, toks = slice(t % page, t % page + stop - t), slice(t - pos[b], stop - pos[b])
            kp[table[b][t // page], :, rows] = k[b, :, toks]
            vp[table[b][t // page], :, rows] = st["v"][b, :, toks].double()
            t = stop
    return {"q": q, "k_pages": kp, "v_pages": vp, "lens": torch.tensor(ends, dtype=torch.int32)}


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
            k = st["kp"][rows, h].reshape(-1, d)[starts[b] : lens[b]].double()
            v = st["vp"][rows, h].reshape(-1, d)[starts[b] : lens[b]].double()
            mine = slice(h * (hq // hkv), (h + 1) * (hq // hkv))
            s = st["q"][b, mine, 0].double() @ k.t() / math.sqrt(d)
            out[b, mine, 0] = torch.softmax(s, -1) @ v
            lse[b, mine] = torch.logsumexp(s, -1) / math.log(2.0)
    return {"out": out, "lse": lse}


def _exact_int4(st):
    c, x = st["case"], st["x"].double()
    if st["nw"] is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / c["k"] + 1e-6) * st["nw"].double()

    def product(weight):
        q, scales, zeros = weight
        y = torch.empty(c["rows"], c["n"], dtype=torch.float64, device=_DEV)
        for n0 in range(0, c["n"], 16384):
            part = q[n0 : n0 + 16384]
            w = torch.empty(part.shape[0], c["k"], dtype=torch.float64, device=_DEV)
            w[:, 0::2] = (part % 16).double()
            w[:, 1::2] = (part // 16).double()
            s = scales[n0 : n0 + 16384].double().repeat_interleave(c["group"], 1)
            z = 8 if zeros is None else zeros[n0 : n0 + 16384].double().repeat_interleave(c["group"], 1)
            y[:, n0 : n0 + 16384] = x @ ((w - z) * s).t()
        return y

    if c["swiglu"]:
        gate, up = product(st["w"][0]), product(st["w"][1])
        y = gate * torch.sigmoid(gate) * up
    else:
        y = product(st["w"])
    return y if st["res"] is None else y + st["res"].double()
