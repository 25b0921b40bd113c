"""The 8-bit cache in float64, for the tests of its kernels: what the format holds, pages in no order with rubbish around what is
held, and attention over what pages hold."""

import torch

BIGGEST = 1.875 * 2.0**127
CODES = torch.float8_e4m3fn


def power_of(big: torch.Tensor) -> torch.Tensor:
    """E of rows with these largest magnitudes (float64): the smallest from 3 on with big <= 448 * 2^(E - 127); 127 for zeros."""
    m, e = torch.frexp(big)
    n = torch.where(m > 0.875, e - 8, e - 9).clamp(min=-124) + 127
    return torch.where(big == 0, torch.full_like(n, 127), n)


def nearest_codes(y: torch.Tensor) -> torch.Tensor:
    """The e4m3 numbers nearest to float64 y (ties to even), as float64."""
    _, e = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (e - 1).clamp(min=-6) - 3)
    return (torch.round(y / step) * step).clamp(-448.0, 448.0)


def held(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """[pages, page_size, nkv, hd] float64 values of codes and powers [pages, nkv, page_size]."""
    return codes.double() * torch.exp2(exps.double() - 127).transpose(-1, -2)[..., None]


def quantise(x: torch.Tensor):
    """(codes, powers) of float rows [..., entries], as tensors of the cache's types."""
    x = x.double().clamp(-BIGGEST, BIGGEST)
    n = power_of(x.abs().amax(-1))
    return nearest_codes(x / torch.exp2(n.double() - 127)[..., None]).float().to(CODES), n.to(torch.uint8)


def tables_for(ctx, page, g, spare=2):
    """(pages, block tables int32 [S, blocks] with -1 behind a request's last page): pages in no order, `spare` unused ones."""
    blocks = [-(-c // page) for c in ctx]
    pages = sum(blocks) + spare
    order = torch.randperm(pages, generator=g).to(torch.int32)
    tables = torch.full((len(ctx), max(max(blocks), 1)), -1, dtype=torch.int32)
    at = 0
    for s, b in enumerate(blocks):
        tables[s, :b] = order[at : at + b]
        at += b
    return pages, tables


def filled_pages(ctx, page, nkv, hd, g, spread=1.0, rubbish=True):
    """A cache that holds random keys and values for contexts of these lengths, on the CPU: ((k, v, k_exp, v_exp), tables).  Slots
    that no request owns hold NaN codes under the largest power, or zeros."""
    pages, tables = tables_for(ctx, page, g)
    out = []
    for _ in range(2):
        codes = torch.zeros(pages, page, nkv, hd, dtype=torch.uint8)
        exps = torch.zeros(pages, nkv, page, dtype=torch.uint8)
        if rubbish:
            codes.fill_(0x7F)
            exps.fill_(254)
        for s, c in enumerate(ctx):
            x = torch.randn(c, nkv, hd, generator=g) * torch.exp(spread * torch.randn(c, nkv, 1, generator=g))
            kc, ke = quantise(x)
            for b in range(-(-c // page)):
                n = min(page, c - b * page)
                codes[tables[s, b], :n] = kc[b * page : b * page + n].view(torch.uint8)
                exps[tables[s, b], :, :n] = ke[b * page : b * page + n].T
        out.append((codes.view(CODES), exps))
    return (out[0][0], out[1][0], out[0][1], out[1][1]), tables


def context(codes, exps, table, c, page):
    """The first c rows of a request, float64 [c, nkv, hd]."""
    ids = table[: -(-c // page)].long()
    return held(codes.view(torch.uint8)[ids].view(CODES), exps[ids]).flatten(0, 1)[:c]


def attention(q, k, v, first, window, scale):
    """float64 attention of q [rows, nh, hd] (row r at position first + r) over k, v [tokens, nkv, hd]: (out, weights' sum of |v|,
    the largest sum of |q| |k| of a score)."""
    rows, nh, hd = q.shape
    group = nh // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("rhd,thd->rht", q, k) * scale
    at, row = torch.arange(k.shape[0], device=q.device), first + torch.arange(rows, device=q.device)[:, None]
    s = s.masked_fill(((at > row) | (at <= row - (window or 1 << 40)))[:, None], float("-inf"))
    w = torch.softmax(s, -1)
    sizes = torch.einsum("rhd,thd->rht", q.abs(), k.abs()) * scale
    return torch.einsum("rht,thd->rhd", w, v), torch.einsum("rht,thd->rhd", w, v.abs()), sizes.amax(-1)[..., None]


def attention_bound(out, size, score, hd, dtype, weight_bits=24):
    """How far a kernel's output may be: half a step of its type; scores off by a chain of hd + 4 float32 roundings of their
    terms, an absolute error that changes numerator and denominator by as much relatively; weights held in `weight_bits` bits
    (at most half a step, 2^-weight_bits... of each), their exponentials and sums in float32 (2^-18 for long sums)."""
    step = torch.finfo(dtype).eps / 2
    return step * out.abs() + (2 * (hd + 4) * 2.0**-24 * score + 2.0**-weight_bits + 2.0**-18) * size + 1e-30
