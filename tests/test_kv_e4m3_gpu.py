"""Writing a cache behind norms and rotation, and reading an 8-bit cache back, against float64."""

import pytest
import torch

from clockwork_b200 import ops
from clockwork_b200.ops import quantised
from tests.e4m3_tools import BIGGEST, CODES, context, filled_pages, held, nearest_codes, power_of
from tests.gpu_tools import DEV

pytestmark = pytest.mark.gpu


def _exact_rows(x, weight, eps, pos, freq):
    """float64 norm and rotation of [N, heads, hd]; also a bound on what float32 makes of it."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight.double()
    half = 0 if freq is None else freq.shape[0]
    out, size = x.clone(), x.abs()
    if half:
        a = (pos.double()[:, None] * freq.double())[:, None]
        u, w = x[..., :half], x[..., half : 2 * half]
        out[..., :half], out[..., half : 2 * half] = u * a.cos() - w * a.sin(), w * a.cos() + u * a.sin()
        size[..., :half] = size[..., half : 2 * half] = u.abs() + w.abs()
    # the norm: a sum of squares of up to 256 terms in a few chains, rsqrt and two products (under 16 roundings); the turn: sine
    # and cosine within 4 roundings of 1, two products, one sum
    return out, 24 * 2.0**-24 * size


def _inputs(heads, n, dtype, rot, norm, g, page, pages, pos_top=40000):
    nh, nkv, hd = heads
    x = torch.randn(n, nh + 2 * nkv, hd, generator=g) * torch.exp(torch.randn(n, nh + 2 * nkv, 1, generator=g))
    qkv = x.reshape(n, -1).to(dtype)
    pos = torch.randint(0, pos_top, (n,), generator=g, dtype=torch.int32)
    slots = torch.randperm(pages * page, generator=g)[:n].to(torch.int32)
    freq = None if rot == 0 else (10000.0 ** -(torch.arange(0, rot, 2).double() / rot)).float()
    w = [1.0 + 0.3 * torch.randn(hd, generator=g) if norm else None for _ in range(2)]
    return qkv, pos, slots, freq, w


def _cache(kind, dtype, pages, page, nkv, hd):
    if kind == "plain":
        return quantised.PlainPages(*(torch.full((pages, page, nkv, hd), 7.0, dtype=dtype, device=DEV) for _ in range(2)))
    cache = quantised.allocate_pages(pages, page, nkv, hd, DEV)
    for t in cache[:2]:
        t.view(torch.uint8).fill_(0x2A)
    for t in cache[2:]:
        t.fill_(99)
    return cache


def _on(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


def _check_rows(cache, kind, slots, rows, slack, dtype, page, untouched):
    nkv = rows[0].shape[1]
    for i, (want, off) in enumerate(zip(rows, slack)):
        keep = (slots >= 0).nonzero()[:, 0]
        sl = slots[keep].long()
        if kind == "plain":
            got = cache[i].double().cpu().flatten(0, 1)
            bound = torch.finfo(dtype).eps / 2 * want[keep].abs() + off[keep] * 1.01
            assert ((got[sl] - want[keep]).abs() <= bound).all()
            rest = torch.ones(got.shape[0], dtype=torch.bool)
            rest[sl] = False
            assert (got[rest] == 7.0).all()
            continue
        codes, exps = cache[i].cpu(), cache[2 + i].cpu()
        e = exps.transpose(1, 2).reshape(-1, nkv)[sl].to(torch.int32)
        x, o = want[keep], off[keep]
        big = x.abs().amax(-1)
        err = torch.where(x.abs() == big[..., None], o, torch.zeros_like(o)).amax(-1)
        lo, hi = power_of((big - 2 * err).clamp(min=0)), power_of(big + 2 * err)
        assert ((e >= torch.minimum(lo, hi)) & (e <= torch.maximum(lo, hi))).all()
        unit = torch.exp2(e.double() - 127)[..., None]
        got = codes.double().flatten(0, 1)[sl] * unit
        # half a step of a code: 2^-4 of a normal number, 2^-10 of the row's power for a subnormal one
        assert ((got - x).abs() <= torch.maximum(2.0**-4 * x.abs(), 2.0**-10 * unit) + 1.1 * o).all()
        rest = torch.ones(codes.shape[0] * page, dtype=torch.bool)
        rest[sl] = False
        assert (codes.view(torch.uint8).flatten(0, 1)[rest] == 0x2A).all() and (exps.transpose(1, 2).reshape(-1, nkv)[rest] == 99).all()
    assert untouched


CASES = [  # heads, rows, rotary entries, norms, page size
    ((12, 2, 128), 1, 128, False, 16), ((28, 4, 128), 37, 128, True, 16), ((4, 4, 16), 5, 16, True, 8), ((6, 2, 96), 11, 48, True, 8),
    ((2, 1, 256), 9, 256, True, 4), ((3, 3, 80), 7, 80, False, 5), ((16, 16, 64), 300, 64, True, 32), ((5, 1, 32), 3, 0, True, 1),
    ((3, 1, 48), 6, 6, True, 16), ((2, 2, 112), 4, 50, False, 7), ((40, 8, 192), 2, 64, True, 16), ((70, 10, 16), 3, 16, False, 16)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kind", ["e4m3", "plain"])
@pytest.mark.parametrize("heads, n, rot, norm, page", CASES)
def test_norm_rotate_store(heads, n, rot, norm, page, kind, dtype):
    nh, nkv, hd = heads
    g = torch.Generator().manual_seed(n * hd + rot)
    pages = -(-n // page) + 3
    qkv, pos, slots, freq, (wq, wk) = _inputs(heads, n, dtype, rot, norm, g, page, pages)
    if n > 2:
        slots[1] = -1  # a padding row: q is worked out, nothing is stored
    cache = _cache(kind, dtype, pages, page, nkv, hd)
    status = ops.new_status(DEV)
    before, args = qkv.to(DEV), _on(pos, slots, freq)
    q = quantised.norm_rotate_store(before, *args, cache, nh, nkv, hd, status, q_weight=_on(wq)[0], k_weight=_on(wk)[0], eps=1e-6)
    ops.raise_on_status(status)
    x = qkv.view(n, nh + 2 * nkv, hd)
    want, off = _exact_rows(x[:, :nh], wq, 1e-6, pos, freq)
    assert ((q.double().cpu().view(n, nh, hd) - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + off * 1.01).all()
    k, k_off = _exact_rows(x[:, nh : nh + nkv], wk, 1e-6, pos, freq)
    v = x[:, nh + nkv :].double()
    _check_rows(cache, kind, slots, (k, v), (k_off, torch.zeros_like(v)), dtype, page, torch.equal(before.cpu(), qkv))


def test_only_one_of_the_norms_and_unaligned_rows():
    """q normed and k not, and weights that begin four bytes behind a multiple of 16 (the kernel that reads entry by entry)."""
    g = torch.Generator().manual_seed(3)
    nh, nkv, hd, n = 6, 2, 64, 9
    qkv, pos, slots, freq, (wq, wk) = _inputs((nh, nkv, hd), n, torch.bfloat16, hd, True, g, 16, 3)
    odd = torch.cat([torch.zeros(1), wq]).to(DEV)[1:]
    status, out = ops.new_status(DEV), []
    for weight in (odd, wq.to(DEV)):
        cache = _cache("e4m3", torch.bfloat16, 3, 16, nkv, hd)
        q = quantised.norm_rotate_store(qkv.to(DEV), *_on(pos, slots, freq), cache, nh, nkv, hd, status, q_weight=weight, eps=1e-5)
        want, off = _exact_rows(qkv.view(n, -1, hd)[:, :nh], wq, 1e-5, pos, freq)
        assert ((q.double().cpu().view(n, nh, hd) - want).abs() <= 2.0**-8 * want.abs() + off * 1.01).all()
        k, k_off = _exact_rows(qkv.view(n, -1, hd)[:, nh : nh + nkv], None, 1e-5, pos, freq)
        v = qkv.view(n, -1, hd)[:, nh + nkv :].double()
        _check_rows(cache, "e4m3", slots, (k, v), (k_off, torch.zeros_like(v)), torch.bfloat16, 16, True)
    ops.raise_on_status(status)


@pytest.mark.parametrize("top", [64, 1 << 20, (1 << 31) - 1])
def test_far_positions_are_turned_exactly(top):
    """Positions of a million and a billion: float32 angles would be off by hundredths of a radian, and by many turns."""
    g = torch.Generator().manual_seed(4)
    qkv, pos, slots, freq, _ = _inputs((4, 2, 128), 64, torch.float32, 128, False, g, 16, 5, pos_top=top)
    cache = _cache("plain", torch.float32, 5, 16, 2, 128)
    status = ops.new_status(DEV)
    q = quantised.norm_rotate_store(qkv.to(DEV), *_on(pos, slots, freq), cache, 4, 2, 128, status)
    want, off = _exact_rows(qkv.view(64, 8, 128)[:, :4], None, 0.0, pos, freq)
    # (both sides' angles are off by float64's last bit at most: 2^-53 of 2^31, 2^-22, here and there, for the farthest)
    far = 2.0**-21 if top > 1 << 20 else 2.0**-32
    assert ((q.double().cpu().view(64, 4, 128) - want).abs() <= 2.0**-24 * want.abs() + off + far * want.abs().amax(-1, keepdim=True)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_extreme_numbers(dtype):
    """Zeros, the smallest and the largest numbers, borders of the powers, infinities and NaN; v rows are held as they are given."""
    nkv, hd, page = 1, 32, 4
    tiny = 2.0**-133 if dtype == torch.bfloat16 else 2.0**-149
    top = torch.finfo(dtype).max
    rows = [torch.zeros(hd), torch.full((hd,), tiny), torch.full((hd,), top), torch.linspace(-448, 448, hd), torch.linspace(-449, 449, hd),
            torch.cat([torch.tensor([float("inf"), float("-inf"), 1.0]), torch.ones(hd - 3)]),
            torch.cat([torch.tensor([float("nan"), 2.0]), torch.ones(hd - 2)]), torch.full((hd,), float("nan")),
            torch.cat([torch.tensor([1.0]), torch.full((hd - 1,), 2.0**-18)]), torch.full((hd,), 2.0**-126)]
    x = torch.stack(rows).to(dtype)
    n = len(rows)
    qkv = torch.cat([torch.ones(n, 2 * hd, dtype=dtype), x], 1)
    cache = quantised.allocate_pages(4, page, nkv, hd, DEV)
    status = ops.new_status(DEV)
    ints = torch.arange(n, dtype=torch.int32, device=DEV)
    quantised.norm_rotate_store(qkv.to(DEV), ints, ints, None, cache, 1, nkv, hd, status)
    e = cache.v_exp.cpu().transpose(1, 2).reshape(-1)[:n].to(torch.int32)
    got = held(cache.v.cpu(), cache.v_exp.cpu()).flatten(0, 1)[:n, 0]
    y = x.double().clamp(-BIGGEST, BIGGEST)
    finite = ~y.isnan()
    big = torch.where(finite, y, 0.0).abs().amax(-1)
    assert torch.equal(e, power_of(big).to(torch.int32))
    want = nearest_codes(y / torch.exp2(e.double() - 127)[:, None]) * torch.exp2(e.double() - 127)[:, None]
    assert torch.equal(got[finite], want[finite]) and got[~finite].isnan().all()
    back = [torch.zeros(4, page, nkv, hd, dtype=dtype, device=DEV) for _ in range(2)]
    tables = torch.arange(4, dtype=torch.int32, device=DEV)[None]
    quantised.read_pages(cache, tables, torch.tensor([n], dtype=torch.int32, device=DEV), *back, status)
    ops.raise_on_status(status)
    rb = back[1].double().cpu().flatten(0, 1)[:n, 0]
    assert torch.equal(rb[finite], want[finite]) and rb[~finite].isnan().all()


def test_slots_outside_the_pool_are_reported():
    cache = _cache("e4m3", torch.bfloat16, 2, 4, 1, 32)
    status = ops.new_status(DEV)
    qkv = torch.ones(3, 3 * 32, dtype=torch.bfloat16, device=DEV)
    ints = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    quantised.norm_rotate_store(qkv, ints, torch.tensor([0, 8, 7], dtype=torch.int32, device=DEV), None, cache, 1, 1, 32, status)
    with pytest.raises(RuntimeError, match="slot"):
        ops.raise_on_status(status)
    e = cache.k_exp.cpu().reshape(-1)
    assert e[0] != 99 and e[7] != 99 and (e[1:7] == 99).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ctx, page, nkv, hd, window", [
    ([1], 16, 2, 128, None), ([0, 5, 33, 16], 16, 2, 128, None), ([700, 3, 129], 8, 4, 64, 50), ([40] * 70, 5, 1, 16, None),
    ([1000, 2000], 64, 3, 80, 1), ([17, 4099], 1, 1, 256, 4000)])
def test_read_pages(ctx, page, nkv, hd, window, dtype):
    g = torch.Generator().manual_seed(sum(ctx) + hd)
    cache, tables = filled_pages(ctx, page, nkv, hd, g)
    status = ops.new_status(DEV)
    out = [torch.full(cache[0].shape, 3.0, dtype=dtype, device=DEV) for _ in range(2)]
    quantised.read_pages(quantised.E4M3Pages(*_on(*cache)), *_on(tables, torch.tensor(ctx, dtype=torch.int32)), *out, status, window=window)
    ops.raise_on_status(status)
    for i in range(2):
        want = torch.full(cache[0].shape, 3.0, dtype=torch.float64)
        for s, c in enumerate(ctx):
            rows = context(cache[i], cache[2 + i], tables[s], c, page)
            for b in range(max(0, c - window) // page if window else 0, -(-c // page)):
                n = min(page, c - b * page)
                want[tables[s, b]] = 0.0
                want[tables[s, b], :n] = rows[b * page : b * page + n]
        assert torch.equal(out[i].double().cpu(), want if dtype == torch.float32 else want.to(dtype).double())
        assert dtype == torch.float32 or torch.equal(want.to(dtype).double(), want)  # bfloat16 holds every held number


@pytest.mark.parametrize("least", [1, 2, 11])
def test_read_pages_of_the_requests_that_bring_rows(least):
    """With q_start only requests of at least so many rows are read, from the page on that their first row's window reaches."""
    ctx, new, page, window = [100, 90, 64, 50], [10, 1, 0, 40], 8, 16
    g = torch.Generator().manual_seed(8)
    cache, tables = filled_pages(ctx, page, 2, 32, g)
    status = ops.new_status(DEV)
    out = [torch.full(cache[0].shape, 3.0, device=DEV) for _ in range(2)]
    starts = torch.tensor([0, 10, 11, 11, 51], dtype=torch.int32)
    quantised.read_pages(quantised.E4M3Pages(*_on(*cache)), *_on(tables, torch.tensor(ctx, dtype=torch.int32)), *out, status, window=window,
                         q_start=starts.to(DEV), least_rows=least)
    ops.raise_on_status(status)
    read = (out[0] != 3.0).flatten(1).any(1).cpu()
    want = torch.zeros_like(read)
    for s, (c, n) in enumerate(zip(ctx, new)):
        if n >= least:
            want[tables[s, max(0, c - n + 1 - window) // page : -(-c // page)].long()] = True
    assert torch.equal(read, want)


def test_pages_outside_the_pool_are_reported_on_reading():
    g = torch.Generator().manual_seed(9)
    cache, tables = filled_pages([40], 16, 1, 16, g)
    tables[0, 1] = 77
    status = ops.new_status(DEV)
    out = [torch.full(cache[0].shape, 3.0, device=DEV) for _ in range(2)]
    quantised.read_pages(quantised.E4M3Pages(*_on(*cache)), *_on(tables, torch.tensor([40], dtype=torch.int32)), *out, status)
    with pytest.raises(RuntimeError, match="page id"):
        ops.raise_on_status(status)
    assert (out[0][tables[0, 0].item()] != 3.0).any() and (out[0][tables[0, 2].item()] != 3.0).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ctx, page", [([1000, 1010, 1003], 16), ([30, 33, 1, 38], 8), ([70, 95, 66], 32)])
def test_requests_that_share_a_partly_filled_page(ctx, page, dtype):
    """Requests over one table, each with a context of its own, and one whose last page, filled in part, stands in its table a second time
    and there in full: every held row arrives, whichever request comes first; zeros are left where none holds anything."""
    g = torch.Generator().manual_seed(sum(ctx))
    longest = max(range(len(ctx)), key=lambda s: ctx[s])
    cache, tables = filled_pages([ctx[longest]], page, 2, 64, g)
    blocks = tables.shape[1]
    tables = tables.repeat(len(ctx) + 1, 1)
    last = (ctx[0] - 1) // page  # request 0's last page; the further request holds all of it as its first
    tables[-1, 0], ctx = tables[0, last], [*ctx, min(page + 1, ctx[longest])]
    full = min(page, ctx[longest] - last * page) == page
    if not full:
        ctx[-1] = ctx[longest] - last * page
    want = torch.zeros(cache[0].shape, dtype=torch.float64)
    touched = torch.zeros(cache[0].shape[:2], dtype=torch.bool)
    values = [held(cache[i], cache[2 + i]) for i in range(2)]
    rows = torch.zeros(cache[0].shape[:2], dtype=torch.bool)
    for s, c in enumerate(ctx):
        for b in range(-(-c // page)):
            touched[tables[s, b]] = True
            rows[tables[s, b], : min(page, c - b * page)] = True
    assert blocks > 1 and (touched & ~rows).any()
    on, lens, status = quantised.E4M3Pages(*_on(*cache)), torch.tensor(ctx, dtype=torch.int32, device=DEV), ops.new_status(DEV)
    tables = tables.to(DEV)
    for order in (list(range(len(ctx))), list(range(len(ctx)))[::-1]):
        for _ in range(20):
            out = [torch.full(cache[0].shape, 3.0, dtype=dtype, device=DEV) for _ in range(2)]
            quantised.read_pages(on, tables[order].contiguous(), lens[order].contiguous(), *out, status)
            for got, value in zip(out, values):
                want = torch.where(rows[..., None, None], value, torch.where(touched, 0.0, 3.0).double()[..., None, None])
                assert torch.equal(got.double().cpu(), want)
    ops.raise_on_status(status)
