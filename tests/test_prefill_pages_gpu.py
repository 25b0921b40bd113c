"""tcgen05 prefill attention: tiles reach over pages that a window has given back and past a request's last page; neither is looked
up, and what other requests' pages hold does not matter."""

import pytest
import torch

from clockwork_b200 import ops
from clockwork_b200.ops import attention_fast as fast
from tests.gpu_tools import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("window, page", [(None, 16), (40, 8), (40, 64), (200, 16)])
def test_pages_without_a_visible_key(hd, window, page):
    nh, nkv, n, ctx = 4, 2, 50, 330
    g = torch.Generator().manual_seed(hd + page)
    blocks = -(-ctx // page)
    pages = blocks + 2
    k, v = (torch.randn(pages, page, nkv, hd, generator=g).bfloat16() for _ in range(2))
    k[0], v[0] = float("nan"), float("nan")  # another request's page
    table = torch.arange(1, blocks + 1, dtype=torch.int32)
    first = 0 if window is None else max(0, ctx - n + 1 - window) // page
    given = table.clone()
    given[:first] = -1
    k[table[-1], ctx % page or page :] = 0
    v[table[-1], ctx % page or page :] = 0
    q = torch.randn(n, nh * hd, generator=g).bfloat16()
    status = ops.new_status(DEV)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    out = fast.attention_prefill(q.to(DEV), k.to(DEV), v.to(DEV), given[None].contiguous().to(DEV), ints([0, n]), ints([ctx]), ints([0]), ints([0]), 1, nh, nkv,
                                 hd, hd**-0.5, window, status)
    ops.raise_on_status(status)
    kk, vv = (t[table.long()].flatten(0, 1)[:ctx].double().repeat_interleave(nh // nkv, 1) for t in (k, v))
    s = torch.einsum("rhd,thd->rht", q.view(n, nh, hd).double(), kk) * hd**-0.5
    at, row = torch.arange(ctx), torch.arange(ctx - n, ctx)[:, None]
    s = s.masked_fill(((at > row) | (at <= row - (window or 1 << 30)))[:, None], float("-inf"))
    w = torch.softmax(s, -1)
    want, size = torch.einsum("rht,thd->rhd", w, vv), torch.einsum("rht,thd->rhd", w, vv.abs())
    got = out.double().cpu().view(n, nh, hd)
    # output and weights in bfloat16: half a step, 2^-8, of each; scores in float32
    assert ((got - want).abs() <= 2.0**-8 * want.abs() + (2.0**-8 + 2.0**-14) * size).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("each", [1, 2])
def test_contexts_shorter_than_their_rows(hd, each):
    """Rows before a request's first token see nothing and give zeros; no entry of the block table is looked up for them, the first
    request's least of all.  (``each``: query heads of a KV head to a tile.)"""
    nh, nkv, page, lens, new = 4, 2, 16, [0, 3, 200], [150, 10, 20]
    g = torch.Generator().manual_seed(hd + each)
    k, v = (torch.randn(16, page, nkv, hd, generator=g).bfloat16() for _ in range(2))
    k[0], v[0] = 0.0, 0.0
    tables = torch.full((3, 13), -1, dtype=torch.int32)
    tables[1, 0], tables[2] = 14, torch.arange(1, 14, dtype=torch.int32)
    q = torch.randn(sum(new), nh * hd, generator=g).bfloat16()
    status = ops.new_status(DEV)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    tile = 128 // each
    items = [(s, at) for s, n in enumerate(new) for at in range(0, n, tile)]
    out = torch.full((q.shape[0], nh * hd), 5.0, dtype=torch.bfloat16, device=DEV)
    fast.launch_prefill(q.to(DEV), k.to(DEV), v.to(DEV), tables.to(DEV), ints([0, 150, 160, 180]), ints(lens), ints([s for s, _ in items]),
                        ints([at for _, at in items]), len(items), nh, nkv, hd, hd**-0.5, None, status, True, None, out, each)
    ops.raise_on_status(status)
    at = 0
    for s, (c, n) in enumerate(zip(lens, new)):
        blind = max(0, n - c)
        got = out[at : at + n].double().cpu().view(n, nh, hd)
        assert (got[:blind] == 0).all()
        if c:
            kk, vv = (t[tables[s, : -(-c // page)].long()].flatten(0, 1)[:c].double().repeat_interleave(nh // nkv, 1) for t in (k, v))
            rows = n - blind
            sc = torch.einsum("rhd,thd->rht", q[at + blind : at + n].view(rows, nh, hd).double(), kk) * hd**-0.5
            sc = sc.masked_fill((torch.arange(c) > torch.arange(c - rows, c)[:, None])[:, None], float("-inf"))
            w = torch.softmax(sc, -1)
            want, size = torch.einsum("rht,thd->rhd", w, vv), torch.einsum("rht,thd->rhd", w, vv.abs())
            # output and weights in bfloat16: half a step, 2^-8, of each; scores in float32
            assert ((got[blind:] - want).abs() <= 2.0**-8 * want.abs() + (2.0**-8 + 2.0**-14) * size).all()
        at += n
