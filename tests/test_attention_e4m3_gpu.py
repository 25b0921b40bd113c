"""Attention over an 8-bit cache, of single tokens and of prompt portions, against float64.  Slots that no request owns hold NaN."""

import pytest
import torch

from clockwork_b200 import ops
from clockwork_b200.ops import quantised
from tests.e4m3_tools import CODES, attention, attention_bound, context, filled_pages, quantise
from tests.gpu_tools import DEV

pytestmark = pytest.mark.gpu
WEIGHT_BITS = 11  # the least that a kernel here holds a weight in: half precision (half a step, 2^-11 of it)


def _on(*tensors):
    return [None if t is None else t.to(DEV) for t in tensors]


def _check(out, q, cache, tables, ctx, rows, page, window, scale, dtype, bits=WEIGHT_BITS):
    """``rows``: (request, first row, rows, position of the first) of what is looked at."""
    nh, hd = q.shape[1] // cache[0].shape[3], cache[0].shape[3]
    for s, at, n, first in rows:
        k, v = (context(cache[i], cache[2 + i], tables[s], ctx[s], page) for i in (0, 1))
        want, size, score = attention(q[at : at + n].double().view(n, nh, hd), k, v, first, window, scale)
        got = out[at : at + n].double().cpu().view(n, nh, hd)
        bound = attention_bound(want, size, score, hd, dtype, bits)
        finite, worst = bool(got.isfinite().all()), float(((got - want).abs() / bound).max())
        assert finite and worst <= 1.0, f"request {s}"


DECODE = [  # heads, contexts, page size, window
    ((12, 2, 128), [1], 16, None), ((12, 2, 128), [1024] * 8, 16, None), ((28, 4, 128), [1, 2, 31, 32, 33, 63, 64, 65, 500, 4000], 16, None),
    ((16, 16, 64), [5, 700, 128], 8, 100), ((9, 3, 32), [77, 3], 32, None), ((16, 1, 64), [900], 64, None), ((24, 2, 128), [300, 4], 16, 33),
    ((8, 4, 256), [129, 1000], 16, None), ((6, 2, 96), [200, 41], 8, None), ((4, 1, 16), [50, 51], 16, None), ((10, 2, 80), [333], 16, 7),
    ((3, 1, 160), [90], 5, None), ((48, 2, 64), [257, 12], 16, None), ((40, 1, 192), [260], 16, None), ((32, 2, 256), [70, 513], 16, None),
    ((2, 2, 112), [19], 3, 1), ((5, 5, 48), [64, 65], 1, None), ((12, 2, 128), [20000, 3, 9000], 16, None)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, ctx, page, window", DECODE)
def test_decode(heads, ctx, page, window, dtype):
    nh, nkv, hd = heads
    g = torch.Generator().manual_seed(sum(ctx) + nh * hd)
    cache, tables = filled_pages(ctx, page, nkv, hd, g)
    q = (torch.randn(len(ctx), nh * hd, generator=g) * torch.exp(0.5 * torch.randn(len(ctx), 1, generator=g))).to(dtype)
    status = ops.new_status(DEV)
    out = quantised.attention_decode(q.to(DEV), quantised.E4M3Pages(*_on(*cache)), *_on(tables, torch.tensor(ctx, dtype=torch.int32)), nh,
                                     hd**-0.5, status, window=window)
    ops.raise_on_status(status)
    assert out.dtype == dtype
    _check(out, q, cache, tables, ctx, [(s, s, 1, c - 1) for s, c in enumerate(ctx)], page, window, hd**-0.5, dtype)


def test_decode_of_empty_contexts_and_many_requests():
    """Padding rows (contexts of 0) give zeros, also between others and when they are all there is."""
    nh, nkv, hd, page = 6, 2, 64, 16
    g = torch.Generator().manual_seed(1)
    for ctx in ([0], [0, 70, 0, 0, 3, 0], [(i * 7) % 40 for i in range(700)]):
        cache, tables = filled_pages(ctx, page, nkv, hd, g)
        q = torch.randn(len(ctx), nh * hd, generator=g).bfloat16()
        status = ops.new_status(DEV)
        out = quantised.attention_decode(q.to(DEV), quantised.E4M3Pages(*_on(*cache)), *_on(tables, torch.tensor(ctx, dtype=torch.int32)),
                                         nh, 0.2, status)
        ops.raise_on_status(status)
        assert all((out[s] == 0).all() for s, c in enumerate(ctx) if c == 0)
        _check(out, q, cache, tables, ctx, [(s, s, 1, c - 1) for s, c in list(enumerate(ctx))[:60] if c], page, None, 0.2, torch.bfloat16)


def test_decode_beside_portions():
    """A flat batch: only requests of one row are served, other rows and rows behind the last request stay as they were; q is a
    column slice of a wider matrix."""
    nh, nkv, hd, page = 12, 2, 128, 16
    ctx, new = [50, 300, 20, 0, 41], [1, 17, 1, 0, 1]
    g = torch.Generator().manual_seed(2)
    cache, tables = filled_pages(ctx, page, nkv, hd, g)
    starts = [sum(new[:i]) for i in range(6)]
    wide = torch.randn(starts[-1] + 3, nh * hd + 64, generator=g).bfloat16()
    out = torch.full((wide.shape[0], nh * hd), 5.0, dtype=torch.bfloat16, device=DEV)
    status = ops.new_status(DEV)
    got = quantised.attention_decode(wide.to(DEV)[:, : nh * hd], quantised.E4M3Pages(*_on(*cache)),
                                     *_on(tables, torch.tensor(ctx, dtype=torch.int32)), nh, 0.1, status,
                                     q_start=torch.tensor(starts, dtype=torch.int32, device=DEV), out=out)
    ops.raise_on_status(status)
    assert got is out
    mine = [starts[s] for s in range(5) if new[s] == 1]
    rest = [r for r in range(out.shape[0]) if r not in mine]
    assert (out[rest] == 5.0).all()
    _check(out, wide[:, : nh * hd].contiguous(), cache, tables, ctx, [(s, starts[s], 1, ctx[s] - 1) for s in (0, 2, 4)], page, None, 0.1, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_decode_of_extreme_rows(dtype):
    """A sink (a large score on a value of zeros), values of very different sizes, scores that differ by hundreds, keys and values
    of all zeros, queries near the ends of the type."""
    nh, nkv, hd, page, c = 4, 1, 64, 16, 200
    g = torch.Generator().manual_seed(5)
    (k, v, ke, ve), tables = filled_pages([c] * 3, page, nkv, hd, g, spread=0.2)
    ids = tables[0].long()
    v.view(torch.uint8)[ids[0], 3] = 0
    ve[ids[0], 0, 3] = 127
    k.view(torch.uint8)[ids[0], 3] = torch.full((hd,), 448.0).to(k.dtype).view(torch.uint8)
    ke[ids[0], 0, 3] = 127 - 6                      # the sink's key: 7 in every entry
    ve[ids[2], 0, :] = 127 - 30                     # tiny values
    ve[ids[3], 0, 0] = 127 + 15                     # a huge one
    k.view(torch.uint8)[tables[1].long()] = 0       # request 1: all scores 0
    v.view(torch.uint8)[tables[2, 1].long()] = 0    # request 2: values of zeros among others
    q = torch.randn(3, nh * hd, generator=g)
    q[0, :hd] = 3.0
    q[0, hd : 2 * hd] = -3.0
    q[2] *= 2.0**-100
    q[1] *= 2.0**60
    q = q.to(dtype)
    cache, status = (k, v, ke, ve), ops.new_status(DEV)
    out = quantised.attention_decode(q.to(DEV), quantised.E4M3Pages(*_on(*cache)), *_on(tables, torch.full((3,), c, dtype=torch.int32)), nh,
                                     0.125, status)
    ops.raise_on_status(status)
    _check(out, q, cache, tables, [c] * 3, [(s, s, 1, c - 1) for s in range(3)], page, None, 0.125, dtype)


def test_decode_reports_pages_outside_the_pool():
    g = torch.Generator().manual_seed(6)
    cache, tables = filled_pages([100, 60], 16, 1, 64, g)
    tables[0, 2], tables[1, 1] = 1000, -1
    status = ops.new_status(DEV)
    out = quantised.attention_decode(torch.ones(2, 64, dtype=torch.bfloat16, device=DEV), quantised.E4M3Pages(*_on(*cache)),
                                     *_on(tables, torch.tensor([100, 60], dtype=torch.int32)), 1, 0.1, status)
    assert out.isfinite().all()  # (the tokens of such pages count for nothing)
    with pytest.raises(RuntimeError, match="page id"):
        ops.raise_on_status(status)


STEPS = [  # heads, contexts, page size, window, entries that turn, norms, type
    ((12, 2, 128), [1], 16, None, 128, False, torch.bfloat16), ((12, 2, 128), [1024] * 8, 16, None, 128, True, torch.bfloat16),
    ((28, 4, 128), [1, 2, 31, 32, 33, 0, 63, 64, 65, 500, 4000], 16, None, 128, False, torch.bfloat16),
    ((16, 16, 64), [5, 700, 128, 0], 8, 100, 64, True, torch.bfloat16), ((24, 1, 128), [300, 1], 5, None, 128, True, torch.bfloat16),
    ((48, 2, 64), [257, 12, 64, 65], 16, 1, 64, False, torch.bfloat16), ((32, 2, 256), [70, 1, 513, 16], 16, None, 256, True, torch.bfloat16),
    ((14, 2, 64), [1, 129], 1, None, 0, True, torch.bfloat16), ((4, 4, 128), [0, 0], 16, None, 128, False, torch.bfloat16),
    ((12, 2, 128), [20000, 3, 9000], 16, None, 128, True, torch.bfloat16), ((16, 16, 64), [200] * 900, 16, None, 64, False, torch.bfloat16),
    ((6, 2, 96), [200, 41, 0], 8, None, 96, True, torch.bfloat16), ((12, 2, 128), [77, 0], 16, None, 64, True, torch.bfloat16),
    ((12, 2, 128), [77, 64, 0], 16, 40, 128, True, torch.float32)]


def _turned(x, w, eps, at, freq):
    """Heads [n, heads, hd] normed and turned in float64, and the sums of the sizes of each result's terms."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    size = x.abs()
    if freq is not None:
        angle = at.double()[:, None] * freq.double()
        c, s, h = angle.cos()[:, None], angle.sin()[:, None], len(freq)
        a, b = x[..., :h], x[..., h : 2 * h]
        size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), x[..., 2 * h :].abs()], -1)
        x = torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * h :]], -1)
    return x, size


@pytest.mark.parametrize("early", [False, True])
@pytest.mark.parametrize("heads, ctx, page, window, rot, norm, dtype", STEPS)
def test_whole_step(heads, ctx, page, window, rot, norm, dtype, early):
    """One call of norms, rotation, store and attention: the rows that it stores (contexts of 0 too, whose output is 0), against the
    formulas; its output over the cache that it leaves; nothing else in the cache changes."""
    nh, nkv, hd = heads
    n, g = len(ctx), torch.Generator().manual_seed(sum(ctx) + nh * hd + rot)
    before, tables = filled_pages(ctx, page, nkv, hd, g)
    owned = sum(-(-c // page) for c in ctx)
    spare = [p for p in range(owned + 2) if p not in set(tables.flatten().tolist())]
    slots = torch.tensor([int(tables[s, (c - 1) // page]) * page + (c - 1) % page if c else spare[s % 2] * page + s // 2 % page
                          for s, c in enumerate(ctx)], dtype=torch.int32)
    at = (torch.tensor(ctx) - 1 + torch.randint(0, 50, (n,), generator=g)).clamp(min=0).to(torch.int32)
    qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g).to(dtype)
    freq = (10000.0 ** -(torch.arange(0, rot, 2).double() / max(rot, 1))).float() if rot else None
    w = [1.0 + 0.2 * torch.randn(hd, generator=g) if norm else None for _ in range(2)]
    w_on, scale, status = _on(*w), hd**-0.5, ops.new_status(DEV)
    lens = torch.tensor(ctx, dtype=torch.int32)

    def run(where, cache):
        out = quantised.decode_step(*_on(qkv, at, where, freq), cache, *_on(tables, lens), nh, nkv, hd, scale, status, q_weight=w_on[0],
                                    k_weight=w_on[1], eps=1e-6, window=window, early=early)
        ops.raise_on_status(status)
        return out

    cache = quantised.E4M3Pages(*_on(*before))
    out = run(slots, cache)
    after = tuple(t.cpu() for t in cache)
    rows = qkv.view(n, -1, hd)
    q, q_size = _turned(rows[:, :nh], w[0], 1e-6, at, freq)
    k, k_size = _turned(rows[:, nh : nh + nkv], w[1], 1e-6, at, freq)
    page_at, off = slots.long() // page, slots.long() % page
    off_by = (hd + 16) * 2.0**-24  # float32 roundings of sums of squares, a root, a quotient, a weight, an angle, two products
    for i, (want, size) in enumerate(((k, k_size), (rows[:, nh + nkv :].double(), 0.0))):
        codes, power = after[i].view(torch.uint8)[page_at, off].view(CODES).double(), after[2 + i][page_at, :, off].double()
        up = torch.exp2(power - 127)[..., None]
        # half a step of a code: 2^-4 of it, or 2^-10 of the power below the smallest whole one
        assert ((codes * up - want).abs() <= torch.maximum(want.abs() * 2.0**-4, up * 2.0**-10) * 1.0001 + off_by * size).all()
        big = want.abs().amax(-1)
        assert (big <= 448.001 * up[..., 0]).all() and (big >= 223.99 * up[..., 0]).all()
        for was, now in ((before[i].view(torch.uint8), after[i].view(torch.uint8)), (before[2 + i].transpose(1, 2), after[2 + i].transpose(1, 2))):
            was, now = was.clone(), now.clone()
            was[page_at, off] = now[page_at, off] = 0
            assert torch.equal(was, now)
    assert all((out[s] == 0).all() for s, c in enumerate(ctx) if c == 0)
    # queries are rounded to the run's type; where float32's errors leave open which way, by so much either way
    low, high = (q - off_by * q_size).to(dtype).double(), (q + off_by * q_size).to(dtype).double()
    q = q.to(dtype).double()
    for s in [s for s, c in enumerate(ctx) if c][:40]:
        keys, values = (context(after[i], after[2 + i], tables[s], ctx[s], page) for i in (0, 1))
        want, size, score = attention(q[s : s + 1], keys, values, ctx[s] - 1, window, scale)
        open_by = scale * ((high - low)[s] * keys.abs().amax(0).repeat_interleave(nh // nkv, 0)).sum(-1)[None, :, None]
        bound = attention_bound(want, size, score, hd, dtype, WEIGHT_BITS) + 2.5 * open_by * size
        got = out[s].double().cpu().view(1, nh, hd)
        assert got.isfinite().all() and float(((got - want).abs() / bound).max()) <= 1.0, f"request {s}"


def test_whole_step_reports_slots_outside_the_pool():
    """Such tokens are not stored."""
    g = torch.Generator().manual_seed(16)
    cache, tables = filled_pages([33, 5], 16, 1, 64, g)
    status, held = ops.new_status(DEV), quantised.E4M3Pages(*_on(*cache))
    slots = torch.tensor([cache[0].shape[0] * 16, 2**31 - 1], dtype=torch.int32, device=DEV)
    out = quantised.decode_step(torch.ones(2, 4 * 64, dtype=torch.bfloat16, device=DEV), *_on(torch.tensor([32, 4], dtype=torch.int32)), slots, None,
                                held, *_on(tables, torch.tensor([33, 5], dtype=torch.int32)), 2, 1, 64, 0.1, status)
    assert out.isfinite().all() and all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(held, cache))
    with pytest.raises(RuntimeError, match="slot"):
        ops.raise_on_status(status)


PORTIONS = [  # heads, rows of each request, tokens behind them, page size, window
    ((12, 2, 128), [130], [0], 16, None), ((12, 2, 128), [64, 1, 200], [300, 40, 0], 16, None), ((4, 4, 64), [150, 0, 7], [0, 9, 1000], 8, 60),
    ((4, 2, 16), [33], [12], 4, None), ((6, 2, 96), [20, 50], [5, 0], 16, None), ((2, 1, 256), [40], [77], 16, None),
    ((28, 4, 128), [5, 17, 2], [3000, 0, 64], 16, None), ((9, 3, 32), [11, 100], [70, 31], 7, 20), ((16, 16, 64), [2] * 40, [90] * 40, 16, None),
    ((70, 2, 64), [3, 40], [200, 1], 16, None), ((12, 2, 128), [300, 22], [3000, 9000], 16, None), ((14, 2, 64), [18, 19, 37], [1000, 0, 64], 8, 130), ((4, 1, 128), [60, 1, 61], [2000, 500, 4000], 64, 700), ((40, 8, 128), [16], [5000], 16, None)]


@pytest.mark.parametrize("dtype, most, packed", [(torch.bfloat16, None, None), (torch.bfloat16, 0, False), (torch.bfloat16, 0, True),
                                                 (torch.bfloat16, 10000, None), (torch.float32, None, None)])
@pytest.mark.parametrize("heads, new, behind, page, window", PORTIONS)
def test_portions(heads, new, behind, page, window, dtype, most, packed):
    """``most``: requests of up to so many rows straight from the codes (None: as the operator chooses); ``packed``: the heads of a KV
    head in the tiles of the others, or a head to a tile."""
    nh, nkv, hd = heads
    if most and hd not in quantised.SHORT_HEAD_DIMS:
        pytest.skip("this head size is read back")
    ctx = [a + b for a, b in zip(new, behind)]
    g = torch.Generator().manual_seed(sum(ctx) + hd)
    cache, tables = filled_pages(ctx, page, nkv, hd, g)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    q = torch.randn(starts[-1] + 2, nh * hd, generator=g).to(dtype)  # (two rows behind the last request's)
    status = ops.new_status(DEV)
    plan = quantised.plan_portions(new, ctx, nh, nkv, hd, page, torch.device(DEV), most_rows=most, packed=packed)
    out = quantised.attention_portions(q.to(DEV), quantised.E4M3Pages(*_on(*cache)),
                                       *_on(tables, torch.tensor(starts, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32)), plan, nh,
                                       hd**-0.5, status, window=window)
    ops.raise_on_status(status)
    # (the bfloat16 kernels over pages read back hold a weight in that type: half a step, 2^-8 of it)
    _check(out, q, cache, tables, ctx, [(s, starts[s], n, ctx[s] - n) for s, n in enumerate(new) if n], page, window, hd**-0.5, dtype,
           24 if dtype == torch.float32 else WEIGHT_BITS if most == 10000 else 8)


@pytest.mark.parametrize("norm", [False, True])
def test_a_request_from_its_prompt_on(norm):
    """The operators as a layer uses them: a prompt's portions stored and attended, then single tokens; every row against float64
    attention over what the cache holds by then."""
    nh, nkv, hd, page, dtype = 12, 2, 128, 16, torch.bfloat16
    g = torch.Generator().manual_seed(7)
    cache = quantised.allocate_pages(12, page, nkv, hd, DEV)
    status = ops.new_status(DEV)
    tables = torch.randperm(12, generator=g)[:8].to(torch.int32)[None]
    freq = (10000.0 ** -(torch.arange(0, hd, 2).double() / hd)).float().to(DEV)
    w = [1.0 + 0.2 * torch.randn(hd, generator=g).to(DEV) if norm else None for _ in range(2)]
    done = 0
    for n in (40, 37, 1, 1, 1, 1):
        qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g).to(dtype).to(DEV)
        at = torch.arange(done, done + n, dtype=torch.int32)
        slots = tables[0, (at // page).long()] * page + at % page
        done += n
        ctx = torch.tensor([done], dtype=torch.int32, device=DEV)
        args = dict(q_weight=w[0], k_weight=w[1], eps=1e-6)
        q = quantised.norm_rotate_store(qkv, at.to(DEV), slots.to(DEV), freq, cache, nh, nkv, hd, status, **args)
        if n > 1:
            plan = quantised.plan_portions([n], [done], nh, nkv, hd, page, torch.device(DEV))
            out = quantised.attention_portions(q, cache, tables.to(DEV), torch.tensor([0, n], dtype=torch.int32, device=DEV), ctx, plan, nh,
                                               0.09, status)
        else:
            out = quantised.decode_step(qkv, at.to(DEV), slots.to(DEV), freq, cache, tables.to(DEV), ctx, nh, nkv, hd, 0.09, status, **args)
        ops.raise_on_status(status)
        _check(out, q.cpu(), tuple(t.cpu() for t in cache), tables, [done], [(0, 0, n, done - n)], page, None, 0.09, dtype, 8 if n > 1 else WEIGHT_BITS)


@pytest.mark.parametrize("dtype, most", [(torch.bfloat16, 0), (torch.bfloat16, None), (torch.float32, None)])
@pytest.mark.parametrize("ctx, new, page", [([1000, 1010], [100, 60], 16), ([70, 95, 66], [30, 3, 40], 32)])
def test_portions_of_requests_over_one_table(ctx, new, page, dtype, most):
    """Portions whose contexts end in the same page, one before the other: what the shorter does not hold the longer one sees."""
    nh, nkv, hd = 12, 2, 128
    g = torch.Generator().manual_seed(sum(ctx))
    cache, tables = filled_pages([max(ctx)], page, nkv, hd, g)
    tables = tables.repeat(len(ctx), 1)
    starts = [sum(new[:i]) for i in range(len(new) + 1)]
    q = torch.randn(starts[-1], nh * hd, generator=g).to(dtype)
    status, on = ops.new_status(DEV), quantised.E4M3Pages(*_on(*cache))
    plan = quantised.plan_portions(new, ctx, nh, nkv, hd, page, torch.device(DEV), most_rows=most)
    lens = _on(tables, torch.tensor(starts, dtype=torch.int32), torch.tensor(ctx, dtype=torch.int32))
    outs = [quantised.attention_portions(q.to(DEV), on, *lens, plan, nh, hd**-0.5, status) for _ in range(10)]
    ops.raise_on_status(status)
    assert all(torch.equal(out, outs[0]) for out in outs)
    _check(outs[0], q, cache, tables, ctx, [(s, starts[s], n, ctx[s] - n) for s, n in enumerate(new)], page, None, hd**-0.5, dtype,
           24 if dtype == torch.float32 else 8)


def _stated_bound(q, k, v, first, scale, hd):
    """What the operator states, summed over the tokens: 2^-11 of each contribution, 2^-38 of a row's largest, 2^-90 (half a step of the smallest
    weights, 2^-25, of 448 times a power that counts as 2^-60 at least, over the 2^14 that weights are held times: 2^-90.1); scores in float32 from
    queries that count down to 2^-39 of their head's largest entry, which move every weight by as much relatively; sums in float32 (2^-18);
    half a step of the output."""
    rows, nh, _ = q.shape
    group = nh // k.shape[1]
    k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("rhd,thd->rht", q, k) * scale
    n = k.shape[0]
    s = s.masked_fill((torch.arange(n) > first + torch.arange(rows)[:, None])[:, None], float("-inf"))
    w = torch.softmax(s, -1)
    want, size = torch.einsum("rht,thd->rhd", w, v), torch.einsum("rht,thd->rhd", w, v.abs())
    largest = (w[..., None] * v.abs().transpose(0, 1)).flatten(2).amax(-1)[..., None]
    score = scale * (2 * (hd + 4) * 2.0**-24 * torch.einsum("rhd,thd->rht", q.abs(), k.abs()).amax(-1) +
                     hd * 2.0**-39 * q.abs().amax(-1) * k.abs().amax((0, 2)))[..., None]
    off = (2.0**-11 + 2.0**-18 + 2 * score) * size + n * (2.0**-38 * largest + 2.0**-90)
    return want, off + 2.0**-8 * (want.abs() + off)


SMALL = [("one zero row of weight 2^20", 20, 0), ("2^25", 25, 0), ("2^30", 30, 0), ("2^35", 35, 0), ("2^60", 60, 0), ("2^100", 100, 0),
         ("tiny values beside it", 0, -30), ("smaller ones", 3, -70), ("values at the format's end", 0, -118), ("no zero row", None, -80),
         ("large values beside it", 20, 35), ("a huge value of little weight", -150, 118)]


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("heads, ctx", [((4, 1, 64), 200), ((12, 2, 128), 3000), ((4, 1, 256), 70), ((6, 3, 32), 5000)])
@pytest.mark.parametrize("what, lead, power", SMALL)
def test_small_contributions(what, lead, power, heads, ctx, rows):
    """A token that has most of the weight and a value of zeros (its power says 2^0), or all values tiny, or one huge: the others'
    contributions keep their bits.  ``lead``: log2 of that token's weight over the others'; ``power``: of the others' values (of the one
    huge value, where there is such).  Portions of few rows go the same way."""
    nh, nkv, hd = heads
    page, scale = 16, hd**-0.5
    g = torch.Generator().manual_seed(ctx + hd + (lead or 0))
    (k, v, ke, ve), tables = filled_pages([ctx], page, nkv, hd, g, spread=0.1)
    ids, at = tables[0].long(), ctx // 3
    huge = lead is not None and lead < 0
    if not huge:
        ve[ids] = torch.where(ve[ids] == 254, ve[ids].int(), (ve[ids].int() + power).clamp(min=3, max=246)).to(torch.uint8)
    q = torch.randn(rows, nh, hd, generator=g).bfloat16()
    if lead is not None:
        q[:, :, 0] = 8.0  # (the token's key: as much in this entry as the lead takes, nothing elsewhere)
        k.view(torch.uint8)[ids[at // page], at % page] = 0
        size = lead / 1.4426950408889634 / (8.0 * scale)
        codes, e = quantise(torch.cat([torch.full((nkv, 1), size), torch.zeros(nkv, hd - 1)], 1))
        k.view(torch.uint8)[ids[at // page], at % page] = codes.view(torch.uint8)
        ke[ids[at // page], :, at % page] = e
        value = torch.zeros(nkv, hd) if not huge else 2.0**power * (1.0 + torch.rand(nkv, hd, generator=g))
        codes, e = quantise(value)
        v.view(torch.uint8)[ids[at // page], at % page] = codes.view(torch.uint8)
        ve[ids[at // page], :, at % page] = e
        assert huge or (e == 127).all()
    cache, status = (k, v, ke, ve), ops.new_status(DEV)
    on, lens = quantised.E4M3Pages(*_on(*cache)), torch.tensor([ctx], dtype=torch.int32)
    if rows == 1:
        out = quantised.attention_decode(q.flatten(1).to(DEV), on, *_on(tables, lens), nh, scale, status)
    elif hd in quantised.SHORT_HEAD_DIMS:
        plan = quantised.plan_portions([rows], [ctx], nh, nkv, hd, page, torch.device(DEV), most_rows=rows)
        assert plan.short == rows
        out = quantised.attention_portions(q.flatten(1).to(DEV), on, *_on(tables, torch.tensor([0, rows], dtype=torch.int32), lens), plan, nh, scale, status)
    else:
        pytest.skip("this head size is read back")
    ops.raise_on_status(status)
    keys, values = (context(cache[i], cache[2 + i], tables[0], ctx, page) for i in (0, 1))
    want, bound = _stated_bound(q.double(), keys, values, ctx - rows, scale, hd)
    got = out.double().cpu().view(rows, nh, hd)
    assert got.isfinite().all() and float(((got - want).abs() / bound).max()) <= 1.0
