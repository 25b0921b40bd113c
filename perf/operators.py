"""The operators of a cache that holds its keys and values in 8 bits, as cases to time and to compare.

A row of the cache (one token's key or value in one KV head) is held as e4m3 codes and one power of two: entry = code *
2^(exponent - 127), the exponent the smallest that keeps the row's largest magnitude within 448.  Five calls deal with it:

* ``store``: a step's [q | k | v] rows; RMS norms of every query and key head (where the layer has them), the position
  rotation, q handed on, k and v written into the cache (8 bits, or the run's own type: the norms go with either cache);
* ``read``: the keys and values of requests back in the run's type;
* ``decode``: attention of one new token per request over the pages of its context;
* ``portions``: causal attention of prompt portions over the same pages;
* ``step``: what a layer does while it decodes: ``store``, then ``decode``.

A case: ``op``, the heads (``nh`` query heads, ``nkv`` KV heads of ``hd`` entries), ``page`` (tokens a page), ``dtype``,
``new`` (rows that each request brings) and ``behind`` (tokens that the cache already holds), both as lists in a text;
``rot`` (leading entries of a head that turn), ``norm`` (heads are normed), ``cache`` ("e4m3" or "plain"), ``window`` (0: all
keys), ``pad`` (rows of the batch that belong to no request).
"""

import math

import torch

own = False
DEV = "cuda:0"
EPS = 1e-6
BIGGEST = 1.875 * 2.0**127  # what a held number is bounded by: 240 * 2^120, the largest that rounds to a finite one


def _case(name, op, heads, new, behind, page=16, dtype="bfloat16", rot=None, norm=False, cache="e4m3", window=0, pad=0):
    nh, nkv, hd = heads
    case = dict(name=name, op=op, nh=nh, nkv=nkv, hd=hd, page=page, dtype=dtype, new=_list(new), behind=_list(behind),
                rot=hd if rot is None else rot, norm=norm, cache=cache, window=window, pad=pad)
    if not name:
        del case["name"]
    return case


SMALL, MIDDLE, LARGE = (12, 2, 128), (28, 4, 128), (40, 8, 128)  # the named shapes' heads: 1.5B, 7B, 32B


def listed():
    ragged = [1 + (7919 * i * i + 331 * i) % 8000 for i in range(64)]
    return [
        # the smallest call: eight requests' new tokens on their way into the cache, where the launch is what counts
        _case("store_8", "store", SMALL, [1] * 8, [1000 + 13 * i for i in range(8)]),
        # a prompt of ordinary length, heads normed
        _case("store_2048_norms", "store", MIDDLE, [2048], [0], norm=True),
        # the norms beside a float32 cache that is not quantised: two portions, half of a head turns, padding rows
        _case("store_plain_odd", "store", (6, 2, 96), [200, 131], [7, 2900], page=8, dtype="float32", rot=48, norm=True, cache="plain", pad=5),
        # three requests' contexts back in bfloat16, what a short prompt behind a long shared prefix has to do first
        _case("read_ragged", "read", SMALL, [0] * 3, [5000, 1, 777]),
        # the same for many long requests of a wide layer
        _case("read_long", "read", LARGE, [0] * 12, [9000 + 1009 * i for i in range(12)]),
        # a chat server's steady state at a small batch
        _case("decode_8", "decode", SMALL, [0] * 8, [1024] * 8),
        # a busy server: 64 requests of one token to 8,000, a wide layer
        _case("decode_64_ragged", "decode", MIDDLE, [0] * 64, ragged),
        # long documents: the largest call
        _case("decode_long", "decode", LARGE, [0] * 4, [131072, 100001, 65536, 120345]),
        # two prompts' portions, one at its start and one behind a context
        _case("portions_short", "portions", SMALL, [391, 130], [0, 5170]),
        # a late portion of a long document beside two that follow a shared prefix
        _case("portions_long", "portions", MIDDLE, [1003, 64, 200], [9001, 12000, 300]),
        # one layer of a decoding step for two requests: norms, rotation, cache write and attention, where latency counts
        _case("step_2", "step", SMALL, [1] * 2, [411, 96], norm=True),
        # the same for 32 requests behind a sliding window: as many KV heads as query heads, small pages
        _case("step_32_window", "step", (16, 16, 64), [1] * 32, [40 + 171 * i for i in range(32)], page=8, window=2000),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("store", "read", "decode", "decode", "portions", "step"))
    heads = rng.choice((SMALL, MIDDLE, LARGE, (16, 16, 64), (16, 1, 64), (9, 3, 32), (24, 2, 128), (8, 4, 256), (6, 2, 96)))
    page = rng.choice((8, 16, 16, 32, 64))
    wide = heads[1] * heads[2]
    if op == "store":
        n = rng.randint(1, 4)
        dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
        return _case("", op, heads, [log(1, 500) for _ in range(n)], [log(1, 30000) for _ in range(n)], page, dtype,
                     rot=rng.choice((heads[2], heads[2], heads[2] // 2)), norm=rng.random() < 0.6,
                     cache=rng.choice(("e4m3", "e4m3", "plain")), pad=rng.choice((0, 0, 3)))
    if op == "read":
        n = log(1, 24)
        return _case("", op, heads, [0] * n, [log(1, max(8, 60_000_000 // (wide * n * 4))) for _ in range(n)], page)
    if op == "portions":
        heads = rng.choice((SMALL, MIDDLE, (16, 16, 64), (6, 2, 128)))
        n = rng.randint(1, 3)
        return _case("", op, heads, [log(2, 900) for _ in range(n)], [rng.choice((0, log(1, 9000))) for _ in range(n)], page)
    n = log(1, 64)
    most = max(16, min(100_000, 200_000_000 // (wide * n)))
    behind = [log(1, most) for _ in range(n)]
    window = rng.choice((0, 0, 0, log(16, 4000)))
    if op == "decode":
        return _case("", op, heads, [0] * n, behind, page, window=window)
    return _case("", op, heads, [1] * n, behind, page, norm=rng.random() < 0.5, window=window)


def _list(numbers):
    return ",".join(str(n) for n in numbers)


def _numbers(text):
    return [int(n) for n in text.split(",")]


def _lengths(case):
    """(rows that each request brings, tokens of each in the cache when the call reads it)."""
    new, behind = _numbers(case["new"]), _numbers(case["behind"])
    return new, [a + b for a, b in zip(new, behind)]


# ---- the inputs -----------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    nh, nkv, hd, page, op = case["nh"], case["nkv"], case["hd"], case["page"], case["op"]
    dtype = getattr(torch, case["dtype"])
    new, ctx = _lengths(case)
    rows, count = sum(new), len(new)
    st = dict(case, g=None, dtype=dtype, status=torch.zeros(4, dtype=torch.int32, device=DEV), scale=hd**-0.5)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=DEV)

    # Pages in no order.  The store alone needs the pages that its rows land in; the others the whole contexts.
    first = [(c - n) // page if op == "store" else 0 for n, c in zip(new, ctx)]
    blocks = [-(-c // page) - f for c, f in zip(ctx, first)]
    pages = sum(blocks) + 2
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    tables = torch.full((count, max(blocks)), -1, dtype=torch.int32, device=DEV)
    at = 0
    for s, b in enumerate(blocks):
        tables[s, :b] = order[at : at + b]
        at += b
    st.update(pages=pages, tables=tables, ctx=ints(ctx), new_host=new, ctx_host=ctx,
              q_start=ints([sum(new[:i]) for i in range(count + 1)]))

    # Keys with a few loud channels, as trained models have them; values whose size differs from token to token.
    loud = 1.0 + 5.0 * (torch.rand(nkv, hd, generator=g, device=DEV) > 0.95)
    if case["cache"] == "plain":
        st["k"], st["v"] = (torch.zeros(pages, page, nkv, hd, dtype=dtype, device=DEV) for _ in range(2))
    else:
        for name, shape in (("k", loud), ("v", torch.ones_like(loud))):
            codes = torch.empty(pages, page, nkv, hd, dtype=torch.float8_e4m3fn, device=DEV)
            exps = torch.empty(pages, nkv, page, dtype=torch.uint8, device=DEV)
            for lo in range(0, pages, 2048):  # a slice at a time: the pool in 32 bits would be large
                n = min(2048, pages - lo)
                size = 1.0 if name == "k" else torch.exp(0.7 * randn(n, page, nkv, 1))
                c, e = _quantised(randn(n, page, nkv, hd) * shape * size)
                codes[lo : lo + n], exps[lo : lo + n] = c, e.transpose(1, 2)
            st[name], st[name + "_exp"] = codes, exps

    if op in ("store", "step"):
        total = rows + case["pad"]
        x = randn(total, nh + 2 * nkv, hd)
        x[:, nh : nh + nkv] *= loud
        st["qkv"] = x.reshape(total, -1).to(dtype)
        pos = [p for n, c in zip(new, ctx) for p in range(c - n, c)] + [0] * case["pad"]
        seq = [s for s, n in enumerate(new) for _ in range(n)]
        slots = torch.full((total,), -1, dtype=torch.int32, device=DEV)
        p, s = ints(pos[:rows]), ints(seq)
        block = p // page - ints(first)[s.long()]
        slots[:rows] = tables[s.long(), block.long()] * page + p % page
        st.update(positions=ints(pos), slots=slots, q_weight=None, k_weight=None)
        half = torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"]
        st["inv_freq"] = (1.0e6**-half).float()
        if case["norm"]:
            st["q_weight"], st["k_weight"] = 1.2 + 0.2 * randn(hd), 1.0 + 0.2 * randn(hd)
    if op in ("decode", "portions"):
        st["q"] = (1.5 * randn(count if op == "decode" else rows, nh * hd)).to(dtype)
    if op == "read":
        st["out_k"], st["out_v"] = (torch.zeros(pages, page, nkv, hd, dtype=dtype, device=DEV) for _ in range(2))
    return st


# ---- the plain form ---------------------------------------------------------------------------------------------------
def _pow2(e):
    """2^e in float32 for whole e in [-126, 127], by its bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantised(x):
    """(codes, exponents + 127) of float32 rows [..., entries]."""
    x = x.clamp(-BIGGEST, BIGGEST)
    big = x.abs().amax(-1)
    m, e = torch.frexp(big)  # big = m * 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-124)
    e = torch.where(big == 0, torch.zeros_like(e), e)
    codes = (x * _pow2(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes, (e + 127).to(torch.uint8)


def _held(codes, exps):
    """The numbers that pages stand for, float32 [..., page, nkv, hd]."""
    return codes.float() * _pow2(exps.to(torch.int32) - 127).transpose(-1, -2)[..., None]


def _normed(x, weight):
    return x if weight is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight


def _turned(x, angle, rot):
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _store(st):
    nh, nkv, hd = st["nh"], st["nkv"], st["hd"]
    x = st["qkv"].float().view(-1, nh + 2 * nkv, hd)
    angle = st["positions"].double()[:, None] * st["inv_freq"].double()
    q = _turned(_normed(x[:, :nh], st["q_weight"]), angle, st["rot"])
    k = _turned(_normed(x[:, nh : nh + nkv], st["k_weight"]), angle, st["rot"])
    v = x[:, nh + nkv :]
    keep = st["slots"] >= 0
    slots = st["slots"][keep].long()
    page, off = slots // st["page"], slots % st["page"]
    if st["cache"] == "plain":
        st["k"][page, off], st["v"][page, off] = k[keep].to(st["dtype"]), v[keep].to(st["dtype"])
        return q.reshape(q.shape[0], -1).to(st["dtype"]), (st["k"], st["v"])
    kc, ke = _quantised(k[keep])
    vc, ve = _quantised(v[keep])
    st["k"].view(torch.uint8)[page, off] = kc.view(torch.uint8)
    st["v"].view(torch.uint8)[page, off] = vc.view(torch.uint8)
    st["k_exp"][page, :, off], st["v_exp"][page, :, off] = ke, ve
    return q.reshape(q.shape[0], -1).to(st["dtype"]), _cache(st)


def _cache(st):
    return tuple(st[n] for n in ("k", "v")) + tuple(st[n + "_exp"].view(torch.float8_e8m0fnu) for n in ("k", "v"))


def _gathered(st):
    """Every request's keys and values, float32 [S, tokens, nkv, hd] (what lies behind a context: zeros)."""
    tables = st["tables"].long().clamp(min=0)
    held = [_held(st[n][tables], st[n + "_exp"][tables]).flatten(1, 2) for n in ("k", "v")]
    there = torch.arange(held[0].shape[1], device=DEV) < st["ctx"][:, None]
    return [torch.where(there[..., None, None], h, 0.0) for h in held]


def _attend(st, q, first):
    """``q`` float32 [S, rows, nh, hd], row r of request s at position ``first[s] + r``; [S, rows, nh, hd]."""
    k, v = _gathered(st)
    s, rows, nh, hd = q.shape
    group = q.view(s, rows, st["nkv"], nh // st["nkv"], hd)
    scores = torch.einsum("srhgd,sthd->srhgt", group, k) * st["scale"]
    at = torch.arange(k.shape[1], device=DEV)
    row = (first[:, None] + torch.arange(rows, device=DEV))[..., None]
    seen = (at <= row) & (at > row - (st["window"] or 1 << 30)) & (at < st["ctx"][:, None, None])
    scores = scores.masked_fill(~seen[:, :, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = weights.sum(-1, keepdim=True)
    out = torch.einsum("srhgt,sthd->srhgd", weights / torch.where(total == 0, 1.0, total), v)
    return out.reshape(s, rows, nh, hd)


def _decode(st, q):
    out = _attend(st, q.float().view(-1, 1, st["nh"], st["hd"]), st["ctx"] - 1)
    return out.reshape(q.shape).to(st["dtype"])


def _portions(st):
    count, most = len(st["new_host"]), max(st["new_host"])
    lens = st["q_start"][1:] - st["q_start"][:-1]
    row = torch.arange(most, device=DEV)
    there = row < lens[:, None]
    flat = (st["q_start"][:-1, None] + row).clamp(max=st["q"].shape[0] - 1).long()
    q = st["q"].float().view(-1, st["nh"], st["hd"])[flat]
    out = _attend(st, q, st["ctx"] - lens)
    return out[there].reshape(st["q"].shape).to(st["dtype"])


def _read(st):
    for name in ("k", "v"):
        held = _held(st[name], st[name + "_exp"])
        used = torch.zeros(st["pages"], st["page"], dtype=torch.bool, device=DEV)
        at = torch.arange(st["tables"].shape[1] * st["page"], device=DEV).view(-1, st["page"])
        there = at < st["ctx"][:, None, None]
        named = st["tables"] >= 0
        used[st["tables"][named].long()] = there[named]
        st["out_" + name][used] = held[used].to(st["dtype"])
    return st["out_k"], st["out_v"]


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(st):
    op = st["op"]
    if own:
        return _own(st)
    if op == "store":
        return _store(st)
    if op == "read":
        return _read(st)
    if op == "decode":
        return _decode(st, st["q"])
    if op == "portions":
        return _portions(st)
    q, cache = _store(st)
    return _decode(st, q), cache


def _own(st):
    from clockwork_b200.ops import quantised

    op, heads = st["op"], (st["nh"], st["nkv"], st["hd"])
    if st["cache"] == "plain":
        cache = quantised.PlainPages(st["k"], st["v"])
    else:
        cache = quantised.E4M3Pages(st["k"], st["v"], st["k_exp"], st["v_exp"])
    window = st["window"] or None
    if op == "store":
        q = quantised.norm_rotate_store(st["qkv"], st["positions"], st["slots"], st["inv_freq"], cache, *heads, st["status"],
                                        q_weight=st["q_weight"], k_weight=st["k_weight"], eps=EPS)
        return q, ((st["k"], st["v"]) if st["cache"] == "plain" else _cache(st))
    if op == "read":
        quantised.read_pages(cache, st["tables"], st["ctx"], st["out_k"], st["out_v"], st["status"])
        return st["out_k"], st["out_v"]
    if op == "decode":
        return quantised.attention_decode(st["q"], cache, st["tables"], st["ctx"], st["nh"], st["scale"], st["status"], window=window)
    if op == "portions":
        plan = st.get("plan")
        if plan is None:  # made once per step, shared by its layers
            plan = st["plan"] = quantised.plan_portions(st["new_host"], st["ctx_host"], *heads, st["page"], st["q"].device)
        return quantised.attention_portions(st["q"], cache, st["tables"], st["q_start"], st["ctx"], plan, st["nh"], st["scale"],
                                            st["status"], window=window)
    out = quantised.decode_step(st["qkv"], st["positions"], st["slots"], st["inv_freq"], cache, st["tables"], st["ctx"], *heads,
                                st["scale"], st["status"], q_weight=st["q_weight"], k_weight=st["k_weight"], eps=EPS, window=window)
    return out, _cache(st)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    nh, nkv, hd, page = case["nh"], case["nkv"], case["hd"], case["page"]
    size = 2 if case["dtype"] == "bfloat16" else 4
    new, ctx = _lengths(case)
    held = nkv * (hd + 1) * 2 if case["cache"] == "e4m3" else nkv * hd * 2 * size  # a token's key and value in the cache
    window = case["window"] or 1 << 60
    rows = sum(new) + case["pad"]
    store = rows * ((nh + 2 * nkv) * hd * size + 8) + sum(new) * held
    if case["op"] == "store":
        return {"bytes": store + rows * nh * hd * size + case["rot"] * 2, "flops": rows * (nh + nkv) * hd * (7 if case["norm"] else 3)}
    if case["op"] == "read":
        return {"bytes": sum(ctx) * (held + 2 * nkv * hd * size) + sum(-(-c // page) for c in ctx) * 4, "flops": sum(ctx) * nkv * hd * 2}
    if case["op"] == "portions":
        # (a row sees the tokens up to its own; the window, where there is one, bounds them)
        seen = sum(min(c - n + r + 1, window) for n, c in zip(new, ctx) for r in range(n))
        return {"bytes": 2 * rows * nh * hd * size + sum(ctx) * held, "flops": 4 * seen * nh * hd}
    read = sum(min(c, window) for c in ctx)
    total = read * held + len(ctx) * 2 * nh * hd * size + sum(-(-c // page) for c in ctx) * 4
    if case["op"] == "step":
        total += store - len(ctx) * (nh * hd * size + held)  # q does not leave the call; the new tokens are read where they are made
    return {"bytes": total, "flops": 4 * read * nh * hd}


# ---- the definition in 64 bits --------------------------------------------------------------------------------------------
def _round_e4m3(y):
    """The nearest number of the format (4 bits of significand, smallest step 2^-9), ties to the even one."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def _exact_row(x):
    """(codes, powers) of float64 rows: the smallest power of two 2^n, n >= -124, with the row within 448 * 2^n."""
    x = x.clamp(-BIGGEST, BIGGEST)
    top = x.abs().amax(-1, keepdim=True)
    n = torch.ceil(torch.log2(top / 448.0))
    two = torch.full_like(top, 2.0)
    n = torch.where(top > 448.0 * two**n, n + 1, n)
    n = torch.where(top <= 448.0 * two ** (n - 1), n - 1, n)
    n = torch.where(top == 0, torch.zeros_like(n), n.clamp(min=-124.0))
    return _round_e4m3(x / two**n), two**n


def _exact_values(codes, exps):
    return codes.double() * torch.exp2(exps.double() - 127.0).transpose(-1, -2)[..., None]


def _exact_heads(x, weight, positions, inv_freq, rot):
    if weight is not None:
        x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS) * weight.double()
    angle = torch.outer(positions.double(), inv_freq.double())[:, None, :]
    out = x.clone()
    h = rot // 2
    out[..., :h] = x[..., :h] * torch.cos(angle) - x[..., h:rot] * torch.sin(angle)
    out[..., h:rot] = x[..., :h] * torch.sin(angle) + x[..., h:rot] * torch.cos(angle)
    return out


def _exact_attention(q, k, v, first, window, scale):
    """One request: float64 q [rows, nh, hd], k and v [tokens, nkv, hd]; row r stands at position first + r."""
    rows, nh, hd = q.shape
    nkv = k.shape[1]
    out = torch.empty_like(q)
    seen = torch.arange(k.shape[0], device=DEV)[None] - (first + torch.arange(rows, device=DEV))[:, None]
    mask = (seen > 0) | (seen <= -(window or 1 << 40))
    for h in range(nh):
        kv = h // (nh // nkv)
        s = (q[:, h] @ k[:, kv].T * scale).masked_fill(mask, -math.inf)
        out[:, h] = torch.softmax(s, -1) @ v[:, kv]
    return out


def exact(case, seed):
    st = prepare(case, seed)
    nh, nkv, hd, page = st["nh"], st["nkv"], st["hd"], st["page"]
    op, q, stored = st["op"], None, None
    if op in ("store", "step"):
        x = st["qkv"].double().view(-1, nh + 2 * nkv, hd)
        args = (st["positions"], st["inv_freq"], st["rot"])
        q = _exact_heads(x[:, :nh], st["q_weight"], *args)
        rows = {"k": _exact_heads(x[:, nh : nh + nkv], st["k_weight"], *args), "v": x[:, nh + nkv :]}
        keep = torch.nonzero(st["slots"] >= 0)[:, 0]
        slots = st["slots"][keep].long()
        if st["cache"] == "plain":
            stored = tuple(st[n].double().flatten(0, 1).index_copy(0, slots, rows[n][keep]).view(st[n].shape) for n in ("k", "v"))
            return q.reshape(q.shape[0], -1), stored
        codes, powers = [], []
        for n in ("k", "v"):
            c, p = _exact_row(rows[n][keep])
            codes.append(st[n].double().flatten(0, 1).index_copy(0, slots, c).view(st[n].shape))
            held = torch.exp2(st[n + "_exp"].double() - 127.0).transpose(1, 2).flatten(0, 1).index_copy(0, slots, p[..., 0])
            powers.append(held.view(-1, page, nkv).transpose(1, 2).contiguous())
        stored = (*codes, *powers)
        if op == "store":
            return q.reshape(q.shape[0], -1), stored
        q = q.reshape(q.shape[0], -1).to(st["dtype"]).double()  # (q is handed on in the run's type)
    if op == "read":
        out = []
        for n in ("k", "v"):
            held = torch.zeros(st["pages"], page, nkv, hd, dtype=torch.float64, device=DEV)
            for s, c in enumerate(st["ctx_host"]):
                ids = st["tables"][s, : -(-c // page)].long()
                values = _exact_values(st[n][ids], st[n + "_exp"][ids]).flatten(0, 1)
                values[c:] = 0
                held[ids] = values.view(-1, page, nkv, hd)
            out.append(held)
        return tuple(out)
    q = st["q"].double() if q is None else q
    outs, at = [], 0
    for s, c in enumerate(st["ctx_host"]):
        ids = st["tables"][s, : -(-c // page)].long()
        if stored is None:
            k, v = (_exact_values(st[n][ids], st[n + "_exp"][ids]) for n in ("k", "v"))
        else:
            k, v = (stored[i][ids] * stored[i + 2][ids].transpose(1, 2)[..., None] for i in (0, 1))
        n = st["new_host"][s] if op == "portions" else 1
        rows = q[at : at + n].view(n, nh, hd)
        outs.append(_exact_attention(rows, k.flatten(0, 1)[:c], v.flatten(0, 1)[:c], c - n, st["window"], st["scale"]).reshape(n, -1))
        at += n
    out = torch.cat(outs)
    return out if op != "step" else (out, stored)
