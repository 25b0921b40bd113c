"""The 8-bit cache's operators as programs use them: captured in graphs, on two streams at once, with and without a workspace of their
own, called again and again on one workspace, at the ends of their ranges."""

import ctypes

import pytest
import torch

from clockwork_b200 import ops
from clockwork_b200.ops import quantised
from tests import test_e4m3_refusals as refusals
from tests.e4m3_tools import filled_pages
from tests.gpu_tools import DEV

pytestmark = pytest.mark.gpu
NH, NKV, HD, PAGE = 12, 2, 128, 16


def _problem(ctx, seed, nh=NH, nkv=NKV, hd=HD):
    g = torch.Generator().manual_seed(seed)
    cache, tables = filled_pages(ctx, PAGE, nkv, hd, g)
    q = torch.randn(len(ctx), nh * hd, generator=g).bfloat16()
    return (q.to(DEV), quantised.E4M3Pages(*(t.to(DEV) for t in cache)), tables.to(DEV), torch.tensor(ctx, dtype=torch.int32, device=DEV))


def _run(problem, status, nh=NH, **kwargs):
    q, cache, tables, ctx = problem
    return quantised.attention_decode(q, cache, tables, ctx, nh, 0.09, status, **kwargs)


@pytest.mark.parametrize("own", [False, True])
def test_captured_calls_give_the_bits_of_plain_ones(own):
    """Replayed many times, with the lengths changed between replays, and two graphs one after the other."""
    status = ops.new_status(DEV)
    workspace = quantised.DecodeWorkspace(HD, DEV) if own else None
    problems = [_problem([700, 3, 2000, 64], 1), _problem([5000], 2)]
    want = [_run(p, status) for p in problems]
    graphs, outs = [], []
    for p in problems:
        _run(p, status, workspace=workspace)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_run(p, status, workspace=workspace))
        graphs.append(graph)
    for _ in range(3):
        for graph, out, w in zip(graphs, outs, want):
            out.zero_()
            graph.replay()
            assert torch.equal(out, w)
    lengths = problems[0][3]
    lengths.copy_(torch.tensor([1, 0, 1999, 33], dtype=torch.int32))
    shorter = _run(problems[0], status)
    graphs[0].replay()
    assert torch.equal(outs[0], shorter) and (shorter[1] == 0).all() and not torch.equal(shorter, want[0])
    ops.raise_on_status(status)


def test_two_streams_and_two_graphs_at_once():
    """Calls that bring no workspace may overlap on the GPU: every stream, and every captured call, has scratch of its own."""
    status = [ops.new_status(DEV), ops.new_status(DEV)]
    problems = [_problem([9000, 8000], 3), _problem([20000], 4)]
    want = [_run(p, s) for p, s in zip(problems, status)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(_run(problems[i], status[i]))
    graphs, outs = [], []
    torch.cuda.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_run(problems[i], status[i]))
        graphs.append(graph)
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    for i in range(2):
        ops.raise_on_status(status[i])
        assert all(torch.equal(x, want[i]) for x in got[i]) and torch.equal(outs[i], want[i])


def test_one_workspace_serves_calls_of_every_shape():
    """Counters are zero again after each call, whatever its heads, lengths and pieces."""
    workspace, status = quantised.DecodeWorkspace(HD, DEV), ops.new_status(DEV)
    shapes = [([100000], 12, 2, 128), ([5] * 300, 12, 2, 128), ([3000, 1], 16, 16, 64), ([40, 7000, 0, 900], 24, 2, 128), ([12345] * 3, 8, 4, 32)]
    problems = [(_problem(ctx, 5 + i, nh, nkv, hd), nh) for i, (ctx, nh, nkv, hd) in enumerate(shapes)]
    want = [_run(p, status, nh) for p, nh in problems]
    for _ in range(3):
        for (p, nh), w in zip(problems, want):
            assert torch.equal(_run(p, status, nh, workspace=workspace), w)
    assert (workspace.words == 0).all()
    with pytest.raises(ValueError, match="workspace"):
        _run(_problem([40], 9, 2, 1, 256), status, 2, workspace=workspace)
    ops.raise_on_status(status)


def test_portions_in_a_graph():
    status = ops.new_status(DEV)
    ctx, new = [300, 2000, 90], [7, 150, 1]
    g = torch.Generator().manual_seed(11)
    cache, tables = filled_pages(ctx, PAGE, NKV, HD, g)
    cache, tables = quantised.E4M3Pages(*(t.to(DEV) for t in cache)), tables.to(DEV)
    q = torch.randn(sum(new), NH * HD, generator=g).bfloat16().to(DEV)
    starts = torch.tensor([0, 7, 157, 158], dtype=torch.int32, device=DEV)
    lens = torch.tensor(ctx, dtype=torch.int32, device=DEV)
    plan = quantised.plan_portions(new, ctx, NH, NKV, HD, PAGE, torch.device(DEV), most_rows=quantised.short_rows(NH, NKV, HD))
    assert plan.short == 8 and plan.items > 0  # both kernels

    def run():
        return quantised.attention_portions(q, cache, tables, starts, lens, plan, NH, 0.09, status)

    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    ops.raise_on_status(status)


def test_the_same_page_in_two_requests_and_twice_in_one():
    """Block tables may name a page more than once (a shared prefix; a request that repeats a page)."""
    q, cache, tables, ctx = _problem([64, 64, 64], 12)
    tables[1, :2] = tables[0, :2]
    tables[2, 1] = tables[2, 0]
    status = ops.new_status(DEV)
    out = quantised.attention_decode(q, cache, tables, ctx, NH, 0.09, status)
    out_k, out_v = (torch.zeros(cache.k.shape, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    quantised.read_pages(cache, tables, ctx, out_k, out_v, status)
    ops.raise_on_status(status)
    from clockwork_b200.ops.attention_fast import attention_decode

    plain = attention_decode(q, out_k, out_v, tables, ctx, NH, NKV, HD, 0.09, None, 64, status)
    # two kernels over the same numbers: weights in 11 and 8 bits, outputs in 8
    size = out_v.float().abs().max()
    assert (out.float() - plain.float()).abs().max() <= (2.0**-8 + 2.0**-8 + 2.0**-10) * size


def test_queries_that_are_not_aligned_for_pairs():
    """Rows that begin at an odd entry go to the kernel that reads entry by entry."""
    q, cache, tables, ctx = _problem([200, 31], 13)
    wide = torch.zeros(2, NH * HD + 3, dtype=torch.bfloat16, device=DEV)
    wide[:, 1 : 1 + NH * HD] = q
    status = ops.new_status(DEV)
    a = quantised.attention_decode(wide[:, 1 : 1 + NH * HD], cache, tables, ctx, NH, 0.09, status)
    b = quantised.attention_decode(q, cache, tables, ctx, NH, 0.09, status)
    ops.raise_on_status(status)
    assert (a.float() - b.float()).abs().max() <= 2.0**-7 * b.float().abs().max()


def test_no_rows_at_all():
    status = ops.new_status(DEV)
    cache = quantised.allocate_pages(2, PAGE, NKV, HD, DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    q = quantised.norm_rotate_store(torch.zeros(0, (NH + 2 * NKV) * HD, dtype=torch.bfloat16, device=DEV), none, none, None, cache, NH, NKV, HD, status)
    assert q.shape == (0, NH * HD)
    out = quantised.attention_decode(q, cache, torch.zeros(0, 1, dtype=torch.int32, device=DEV), none, NH, 0.09, status)
    assert out.shape == (0, NH * HD)
    ops.raise_on_status(status)
    out = quantised.decode_step(torch.zeros(0, (NH + 2 * NKV) * HD, dtype=torch.bfloat16, device=DEV), none, none, None, cache,
                                torch.zeros(0, 1, dtype=torch.int32, device=DEV), none, NH, NKV, HD, 0.09, status)
    assert out.shape == (0, NH * HD)


def _steps(seed, start, steps, nh=NH, nkv=NKV, hd=HD):
    """Requests that grow by a token a step: (cache, tables, qkv [steps, requests, ..], slots and contexts [steps, requests])."""
    g = torch.Generator().manual_seed(seed)
    cache, tables = filled_pages([c + steps for c in start], PAGE, nkv, hd, g)
    ctx = torch.tensor(start, dtype=torch.int32) + 1 + torch.arange(steps, dtype=torch.int32)[:, None]
    slots = torch.stack([tables[s, (ctx[:, s].long() - 1) // PAGE] * PAGE + (ctx[:, s] - 1) % PAGE for s in range(len(start))], 1).to(torch.int32)
    qkv = torch.randn(steps, len(start), (nh + 2 * nkv) * hd, generator=g).bfloat16()
    return (lambda: quantised.E4M3Pages(*(t.to(DEV) for t in cache))), tables.to(DEV), qkv.to(DEV), slots.to(DEV), ctx.to(DEV)


@pytest.mark.parametrize("early", [False, True])
def test_captured_steps_give_the_bits_of_plain_ones(early):
    """Two layers' whole steps in one graph, replayed while the contexts grow over the ends of pages and tiles."""
    status, steps = ops.new_status(DEV), 40
    fresh, tables, qkv, slots, ctx = _steps(21, [1, 30, 1000, 0], steps)
    freq = (10000.0 ** -(torch.arange(0, HD, 2).double() / HD)).float().to(DEV)
    now = {"qkv": qkv[0].clone(), "slots": slots[0].clone(), "ctx": ctx[0].clone(), "at": ctx[0] - 1}

    def run(layers):
        return [quantised.decode_step(now["qkv"], now["at"], now["slots"], freq, layer, tables, now["ctx"], NH, NKV, HD, 0.09, status,
                                      early=early) for layer in layers]

    def bring(i):
        for name, t in (("qkv", qkv[i]), ("slots", slots[i]), ("ctx", ctx[i]), ("at", ctx[i] - 1)):
            now[name].copy_(t)

    plain, layers, want = [fresh(), fresh()], [fresh(), fresh()], []
    for i in range(steps):
        bring(i)
        want.append([out.clone() for out in run(plain)])
    bring(0)
    run([fresh()])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(layers)
    for i in range(steps):
        bring(i)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i])), i
    for a, b in zip(plain, layers):
        assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))
    ops.raise_on_status(status)


def test_whole_steps_on_two_streams():
    status = [ops.new_status(DEV), ops.new_status(DEV)]
    problems = [_steps(22, [9000, 8000], 10), _steps(23, [20000], 10)]

    def run(i, cache):
        _, tables, qkv, slots, ctx = problems[i]
        return [quantised.decode_step(qkv[j], ctx[j] - 1, slots[j], None, cache, tables, ctx[j], NH, NKV, HD, 0.09, status[i]) for j in range(10)]

    caches = [p[0]() for p in problems]
    want = [run(i, p[0]()) for i, p in enumerate(problems)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            got.append(run(i, caches[i]))
    torch.cuda.synchronize()
    for i in range(2):
        ops.raise_on_status(status[i])
        assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))


def test_steps_whose_rows_begin_at_an_odd_entry():
    """They go to the two kernels that read entry by entry, and hold the same rows."""
    status = ops.new_status(DEV)
    fresh, tables, qkv, slots, ctx = _steps(24, [200, 31], 1)
    odd = torch.zeros(qkv[0].numel() + 1, dtype=torch.bfloat16, device=DEV)[1:].view_as(qkv[0])
    odd.copy_(qkv[0])
    caches, outs = [fresh(), fresh()], []
    for rows, cache in zip((qkv[0], odd), caches):
        outs.append(quantised.decode_step(rows, ctx[0] - 1, slots[0], None, cache, tables, ctx[0], NH, NKV, HD, 0.09, status))
    ops.raise_on_status(status)
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(*caches))
    assert torch.equal(*outs)  # (their queries are the same bits: neither is normed nor turned)


def _moved(x):
    if isinstance(x, torch.Tensor):
        return x.to(DEV) if x.is_contiguous() else x.t().contiguous().to(DEV).t() if x.dim() == 2 and x.t().is_contiguous() else \
            torch.repeat_interleave(x.to(DEV), 2, -1)[..., ::2]
    return type(x)(*map(_moved, x)) if isinstance(x, tuple) else x


@pytest.fixture
def entry_points():
    """The module of common calls with entry points that only count how often they are reached (nothing is launched)."""
    module, reached = quantised._calls(), []
    entry = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_void_p)(lambda words: reached.append(words) or 0)
    address = ctypes.cast(entry, ctypes.c_void_p).value
    module.bind(*[address] * 5, quantised.E4M3Pages, quantised.PlainPages)
    yield module, reached
    quantised._calls_module = None  # (bound anew by the next call)


def test_common_calls_refuse_what_the_others_name(entry_points):
    """Every call that the checks in Python refuse, on the GPU's tensors, and mixtures of devices: the short way finds it too."""
    module, reached = entry_points
    base = {k: _moved(v) for k, v in refusals._args().items()}
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)  # noqa: E731
    scratch = quantised.DecodeWorkspace(128, DEV).pointers
    names = ("qkv", "positions", "slots", "inv_freq", "cache", "num_heads", "num_kv_heads", "head_dim", "status", "q_weight", "k_weight", "eps")
    store = {**base, "q_weight": None, "k_weight": None, "eps": 1e-6, "early": False}
    step = {**store, "block_tables": ints(3, 2), "ctx_lens": ints(3), "scale": 1.0, "window": None, "scratch": scratch, "sms": 148}
    decode = dict(q=torch.zeros(3, 128, dtype=torch.bfloat16, device=DEV), cache=base["cache"], block_tables=ints(3, 2), ctx_lens=ints(3), num_heads=4,
                  scale=1.0, status=base["status"], window=None, scratch=scratch, sms=148, early=False)
    plain = torch.zeros(4, 8, 2, 32, device=DEV)
    read = dict(cache=base["cache"], block_tables=ints(3, 2), ctx_lens=ints(3), out_k=plain, out_v=plain.clone(), status=base["status"], window=None, blocks=4)
    few = refusals._args(hd=64)
    pages = torch.zeros(4, 8, 2, 64, dtype=torch.bfloat16, device=DEV)
    portions = dict(q=torch.zeros(5, 256, dtype=torch.bfloat16, device=DEV), cache=_moved(few["cache"]), block_tables=ints(3, 2),
                    q_start=torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=DEV), ctx_lens=ints(3),
                    plan=quantised.plan_portions([2, 0, 3], [2, 0, 9], 4, 2, 64, 8, DEV, most_rows=2), num_heads=4, scale=1.0, status=base["status"],
                    window=None, scratch=scratch, sms=148, blocks=4, k=pages, v=pages.clone(), parts=(16, 32, 48))
    assert portions["plan"].items > 0 and portions["plan"].short == 2
    other_plans = [quantised.plan_portions([2, 0, 3], [2, 0, 9], *shape, DEV, most_rows=2) for shape in ((8, 2, 64, 8), (4, 4, 64, 8), (4, 2, 128, 8), (4, 2, 64, 16))]
    other_plans += [quantised.plan_portions([2, 3], [2, 9], 4, 2, 64, 8, DEV, most_rows=2), quantised.plan_portions([2, 1, 3], [2, 1, 9], 4, 2, 64, 8, DEV, most_rows=2)]
    plans = [({"plan": plan}, "") for plan in (*other_plans, tuple(portions["plan"])[:-1], "x", None)]
    forms = [(module.portions, portions, tuple(portions), [c for c in refusals.PORTIONS if not {"plan", "cache", "q", "q_start", "block_tables"} & set(c[0])] + plans),
             (module.store, store, (*names, "early"), refusals.STORE),
             (module.step, step, (*names, "early", "block_tables", "ctx_lens", "scale", "window", "scratch", "sms"), refusals.STEP),
             (module.decode, decode, tuple(decode), [c for c in refusals.DECODE if not {"q_start", "out"} & set(c[0])]),
             (module.read, read, tuple(read), [c for c in refusals.READ if "q_start" not in c[0]])]
    for call, good, order, refused in forms:
        assert call(*(good[name] for name in order)) is not None and len(reached) == {module.step: 2, module.portions: 3}.get(call, 1)
        reached.clear()
        cases = [{k: v if k == "plan" else _moved(v) for k, v in change.items()} for change, _ in refused if change]
        for name, value in good.items():  # a tensor elsewhere, of another type, of other sizes; what is no tensor at all
            if isinstance(value, torch.Tensor):
                cases += [{name: value.cpu()}, {name: value.to(torch.float16)}, {name: value[1:]}, {name: value[None]}, {name: "x"}, {name: None}]
            elif isinstance(value, tuple) and name == "cache":
                cases += [{name: value._replace(**{f: getattr(value, f).cpu()})} for f in value._fields]
                cases += [{name: value._replace(**{f: getattr(value, f)[:, 1:].contiguous()})} for f in value._fields]
                cases += [{name: tuple(value)}, {name: None}]
            elif name == "scratch":
                cases += [{name: (*value[:2], 16, 0)}, {name: (*value[:3], 1)}, {name: None}]
            elif isinstance(value, int) and name not in ("early", "sms", "blocks"):
                cases += [{name: value + 1}, {name: -value}, {name: 0}, {name: 1 << 40}, {name: 1 << 70}, {name: 1.5}]
        for case in cases:
            if (case.keys() & {"inv_freq", "q_weight", "k_weight"}) and list(case.values())[0] is None or case.keys() == {"inv_freq"} and \
                    isinstance(case["inv_freq"], torch.Tensor) and case["inv_freq"].shape == (15,):
                continue  # (those may be left out, and fewer entries may turn)
            if case.keys() == {"status"} and isinstance(case["status"], torch.Tensor) and case["status"].shape[:1] == (1,) and case["status"].is_cuda and \
                    case["status"].dtype == torch.int32:
                continue  # (four words of any shape)
            result = call(*({**good, **case}[name] for name in order))
            assert result is None and not reached, (call, case.keys(), [getattr(v, "shape", v) for v in case.values()])


@pytest.mark.parametrize("tile, nh, nkv, hd", [(64, 8, 2, 64), (32, NH, NKV, HD), (16, 4, 1, 256)])
def test_tokens_of_one_sequence_as_requests_of_a_step(tile, nh, nkv, hd):
    """Draft tokens: the rows of one call are neighbours in one sequence, so that each sees the rows that the call stores for those before
    it, in its last tile of keys or the one before that.  The same bits as a store that is complete before attention begins."""
    status, rows = ops.new_status(DEV), 5
    g = torch.Generator().manual_seed(31)
    for base in (tile - 2, 3 * tile - 3, 40 * tile - 4):
        cache, tables = filled_pages([base + rows], PAGE, nkv, hd, g)
        at = torch.arange(base, base + rows, dtype=torch.int32)
        slots = tables[0, at.long() // PAGE] * PAGE + at % PAGE
        tables, at, slots, ctx = tables.repeat(rows, 1).to(DEV), at.to(DEV), slots.to(torch.int32).to(DEV), (at + 1).to(DEV)
        for _ in range(10):
            qkv = torch.randn(rows, (nh + 2 * nkv) * hd, generator=g).bfloat16().to(DEV)
            one, two = (quantised.E4M3Pages(*(t.to(DEV) for t in cache)) for _ in range(2))
            q = quantised.norm_rotate_store(qkv, at, slots, None, one, nh, nkv, hd, status)
            torch.cuda.synchronize()
            want = quantised.attention_decode(q, one, tables, ctx, nh, 0.09, status)
            torch.cuda.synchronize()
            got = quantised.decode_step(qkv, at, slots, None, two, tables, ctx, nh, nkv, hd, 0.09, status)
            assert torch.equal(got, want) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(one, two))
    ops.raise_on_status(status)


@pytest.mark.parametrize("early", [False, True])
def test_rows_that_the_kernel_in_front_writes(early):
    """``qkv`` comes from a kernel that lets this call begin before it has finished, and is written anew each time."""
    status, steps = ops.new_status(DEV), 30
    fresh, tables, qkv, slots, ctx = _steps(25, [300, 31, 2000], steps)
    heads, cache, plain, want = NH + 2 * NKV, fresh(), fresh(), []
    for i in range(steps):
        want.append(quantised.decode_step(qkv[i], ctx[i] - 1, slots[i], None, plain, tables, ctx[i], NH, NKV, HD, 0.09, status))
        torch.cuda.synchronize()
    spare = quantised.allocate_pages(1, PAGE, 1, HD, DEV)
    wide = torch.zeros(steps, 3, (heads + 2) * HD, dtype=torch.bfloat16, device=DEV)
    wide[:, :, : heads * HD] = qkv
    nowhere = torch.full((3,), -1, dtype=torch.int32, device=DEV)
    at = ctx - 1
    torch.cuda.synchronize()
    got = []
    for i in range(steps):  # (rows that neither norm nor turn: the store hands them on as they are)
        torch.cuda.synchronize()  # (the rows of the steps before are complete)
        made = quantised.norm_rotate_store(wide[i], at[i], nowhere, None, spare, heads, 1, HD, status, early=True)
        got.append(quantised.decode_step(made, at[i], slots[i], None, cache, tables, ctx[i], NH, NKV, HD, 0.09, status, early=early))
    ops.raise_on_status(status)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def _portion_problem(new, behind, seed):
    ctx = [a + b for a, b in zip(new, behind)]
    g = torch.Generator().manual_seed(seed)
    cache, tables = filled_pages(ctx, PAGE, NKV, HD, g)
    q = torch.randn(sum(new), NH * HD, generator=g).bfloat16().to(DEV)
    starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    plan = quantised.plan_portions(new, ctx, NH, NKV, HD, PAGE, torch.device(DEV), most_rows=8)
    assert plan.items > 0 and plan.item_split is not None  # (parts, which meet through counters)
    return q, quantised.E4M3Pages(*(t.to(DEV) for t in cache)), tables.to(DEV), starts, torch.tensor(ctx, dtype=torch.int32, device=DEV), plan


def test_portions_on_two_streams_and_in_graphs_at_once():
    """Calls that bring nothing share nothing: two streams whose caches have the same shape, two graphs of them, and a graph beside plain
    calls, over and over."""
    status = [ops.new_status(DEV), ops.new_status(DEV)]
    problems = [_portion_problem([130, 5], [6000, 900], 41), _portion_problem([130, 7], [6000, 900], 42)]
    assert problems[0][1].k.shape == problems[1][1].k.shape

    def run(i, **kwargs):
        q, cache, tables, starts, ctx, plan = problems[i]
        return quantised.attention_portions(q, cache, tables, starts, ctx, plan, NH, 0.09, status[i], **kwargs)

    want = [run(0), run(1)]
    back = quantised.PlainPages(*(torch.full(problems[0][1].k.shape, float("nan"), dtype=torch.bfloat16, device=DEV) for _ in range(2)))
    workspace = quantised.DecodeWorkspace(HD, DEV)
    assert all(torch.equal(run(i, back=back, workspace=workspace), want[i]) for i in range(2))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(i))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(i))
        graphs.append(graph)
    for k in range(30):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay() if k % 2 == 0 or i == 0 else got[i].append(run(i))
    torch.cuda.synchronize()
    for i in range(2):
        ops.raise_on_status(status[i])
        assert torch.equal(outs[i], want[i]) and all(torch.equal(x, want[i]) for x in got[i])
    empty = quantised.DecodeWorkspace(HD, DEV)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before it is captured"):
        with torch.cuda.graph(graph):
            run(0, workspace=empty)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):  # (and with one that has room)
        out = run(0, workspace=workspace, back=back)
    graph.replay()
    assert torch.equal(out, want[0])
