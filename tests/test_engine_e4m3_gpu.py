"""A cache in 8 bits and normed heads inside the engine: the attention part over it, steps with and without captured graphs, forks,
shared prefixes, portions beside single tokens."""

import pytest
import torch

from clockwork_b200 import EngineConfig, ops
from clockwork_b200.cache import CacheManager
from clockwork_b200.config import PartSpec
from clockwork_b200.engine import LLMEngine
from clockwork_b200.engine.step import StepBuilder, StepEntry
from clockwork_b200.engine.trace import TraceSession
from clockwork_b200.ops import quantised
from clockwork_b200.parts import build_part
from clockwork_b200.sampling import SamplingParams
from clockwork_b200.weights import write_random_model
from tests.e4m3_tools import attention, attention_bound, context, quantise
from tests.gpu_tools import DEV
from tests.plain import qwen2_plain as plain
from tests.test_parts_gpu import load, weights
from tests.tiny_configs import TINY, tokens_for

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16]


class Untouched:
    """In an output projection's place: hands on what attention made."""

    def add_or_defer(self, x, stream):
        return x


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kv_dtype, norm", [("e4m3", None), ("e4m3", 1e-5), ("auto", 1e-5)])
@pytest.mark.parametrize("heads, window", [((6, 2, 48), None), ((8, 2, 64), None), ((8, 2, 64), 16), ((4, 1, 32), 20), ((2, 2, 128), 9), ((3, 3, 128), None), ((2, 1, 256), 33)])
def test_attention_part(heads, window, kv_dtype, norm, dtype):
    """Portions, single tokens and both in one step.  q and what the cache holds are checked in the kernels' own tests; here they are
    taken from the kernel and the cache, and attention of every row is worked out from them in float64."""
    nh, nkv, hd = heads
    part = build_part("mixer", PartSpec("attention", dict(hidden_size=80, num_heads=nh, num_kv_heads=nkv, head_dim=hd, qkv_bias=True, o_bias=False,
                                                          scale=hd**-0.5, window=window, qk_norm=norm,
                                                          position=PartSpec("rope_neox", {"theta": 5000.0, "rotary_dim": hd}))), "a", dtype, DEV)
    w = weights(part.tensor_decls(), dtype, seed=hd)
    load(part, w)
    assert ("a.q_norm.weight" in w) == (norm is not None)
    part.o = Untouched()
    cache = CacheManager({0: part.cache_need()}, num_pages=40, page_size=8, dtype=dtype, device=DEV, num_state_slots=4, kv_dtype=kv_dtype)
    builder = StepBuilder(cache, dtype, DEV, cache.status)
    g = torch.Generator().manual_seed(hd)
    seen = {}
    original, whole = ops.quantised.norm_rotate_store, ops.quantised.decode_step

    def noting(*args, **kwargs):
        seen["q"] = original(*args, **kwargs)
        return seen["q"]

    def noting_step(qkv, positions, slots, inv_freq, cache, tables, ctx, nh, nkv, hd, scale, status, **kwargs):
        norms = {name: kwargs[name] for name in ("q_weight", "k_weight", "eps")}
        seen["q"] = original(qkv, positions, torch.full_like(slots, -1), inv_freq, cache, nh, nkv, hd, status, **norms)  # (stored nowhere)
        return whole(qkv, positions, slots, inv_freq, cache, tables, ctx, nh, nkv, hd, scale, status, **kwargs)

    ops.quantised.norm_rotate_store, ops.quantised.decode_step = noting, noting_step
    try:
        for step in ({"a": 21}, {"b": 40, "a": 1}, {"a": 1, "b": 1}, {"c": 5, "a": 9, "b": 1}, {"a": 1, "b": 1, "c": 1}):
            entries = []
            for rid, n in step.items():
                if rid not in cache.requests:
                    cache.open(rid)
                entries.append(StepEntry(rid, [0] * n, []))
            prepared = builder.prepare(entries)
            view = prepared.ctx.views[0]
            assert (view.k_exp is not None) == (kv_dtype == "e4m3")
            x = torch.randn(sum(step.values()), 80, generator=g).to(dtype)
            out = part.forward(prepared.ctx, x.to(DEV), view, None).double().cpu()
            ops.raise_on_status(cache.status)
            at = 0
            for s, (rid, n) in enumerate(step.items()):
                table, c = view.block_tables[s].cpu(), prepared.ctx_lens[s]
                if kv_dtype == "e4m3":
                    k, v = (context(t.cpu(), e.cpu(), table, c, 8) for t, e in ((view.k_cache, view.k_exp), (view.v_cache, view.v_exp)))
                else:
                    k, v = (t.double().cpu()[table[: -(-c // 8)].long()].flatten(0, 1)[:c] for t in (view.k_cache, view.v_cache))
                q = seen["q"][at : at + n].double().cpu().view(n, nh, hd)
                want, size, score = attention(q, k, v, c - n, window, hd**-0.5)
                bound = attention_bound(want, size, score, hd, dtype, 8 if dtype == torch.bfloat16 else 24)
                worst = float(((out[at : at + n].view(n, nh, hd) - want).abs() / bound).max())
                assert worst <= 1.0, (step, rid)
                at += n
            builder.commit(prepared)
    finally:
        ops.quantised.norm_rotate_store, ops.quantised.decode_step = original, whole


@pytest.fixture(scope="module")
def oracles(sharp_dirs):
    """(exact, activations rounded to bfloat16, keys and values held in 8 bits) logits of a request at every place."""
    cache = {}
    original = plain.causal_attention

    def held(x):
        codes, e = quantise(x)
        return (codes.double() * torch.exp2(e.double() - 127)[..., None]).to(x.dtype)

    def in_8_bits(q, k, v, scale, **kwargs):
        return original(q, held(k), held(v), scale, **kwargs)

    def get(name, tokens):
        key = (name, tuple(tokens))
        if key not in cache:
            config, w = plain.read_model_dir(sharp_dirs[name])
            both = [plain.all_position_logits(config, w, tokens), plain.all_position_logits(config, w, tokens, rnd=plain.to_bfloat16_and_back)]
            plain.causal_attention = in_8_bits
            try:
                both.append(plain.all_position_logits(config, w, tokens))
            finally:
                plain.causal_attention = original
            cache[key] = both
        return cache[key]

    return get


@pytest.mark.parametrize("graphs", [True, False], ids=["graphs", "no-graphs"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", sorted(TINY))
def test_logits_of_prompts_portions_and_single_tokens(name, dtype, graphs, sharp_dirs, oracles):
    """Every place's logits against the plain model that holds keys and values in 8 bits ("eight"; its distance from the exact model
    is what 8 bits cost, "cost").  float32: the engine's activations differ by so little that a few codes in a million fall to the
    neighbour: at most half the cost at any place, a tenth on average.  bfloat16: rounding moves activations by up to 2^-9, which
    is a twentieth of a code's step, so that all along the request other codes are chosen, and the engine's 8-bit error is another
    draw of the same size: |engine - eight| <= |engine - exact| + |exact - eight|, the first at most what rounding costs (2.5
    and 2 times the yardstick, as in the trace tests) and its own 8-bit error, the second the cost: two costs in all."""
    raw, _seed, page = TINY[name]
    session = TraceSession(sharp_dirs[name], dtype, 640, page, graphs=graphs, kv_dtype="e4m3")
    assert session.cache.groups[0].kv.dtype == torch.float8_e4m3fn
    toks = {rid: tokens_for(name, n, salt=i) for i, (rid, n) in enumerate((("whole", 120), ("cut", 120), ("tail", 50)))}
    logits = {rid: [] for rid in toks}
    step = 0

    def run(**portions):
        nonlocal step
        entries, want = [], []
        for rid, n in portions.items():
            at = sum(x.shape[0] for x in logits[rid])
            entries.append({"id": rid, "tokens": toks[rid][at : at + n], "want": list(range(n))})
        out, _ = session.run_step({"step": step, "entries": entries})
        step, at = step + 1, 0
        for rid, n in portions.items():
            logits[rid].append(torch.from_numpy(out[at : at + n]))
            at += n

    run(whole=119)
    run(cut=37, tail=9)
    run(cut=2, tail=1)
    run(cut=60, tail=1, whole=1)
    for _ in range(8):
        run(cut=1, tail=1)
    run(cut=13)
    for rid, parts in logits.items():
        got = torch.cat(parts)
        exact, rounded, eight = (x[: got.shape[0]].float() for x in oracles(name, toks[rid]))
        yard, cost, diff = (rounded - exact).abs(), (eight - exact).abs(), (got - eight).abs()
        if dtype == "float32":
            most, mean = 1e-5 + 0.5 * cost.max(), 1e-5 + 0.1 * cost.mean()
        else:
            most, mean = 2.5 * yard.max() + 2 * cost.max(), 2 * yard.mean() + 2 * cost.mean()
        assert diff.max() <= most and diff.mean() <= mean, (rid, float(diff.max()), float(most), float(diff.mean()), float(mean))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_forks_and_shared_prefixes(dtype, sharp_dirs):
    """A fork goes on from shared pages (codes and powers of the page it writes into are copied), a prefix hit takes pages over:
    the logits are those of a request that shares nothing, bit for bit where it is in the same row of steps of the same lengths (how
    a context is cut over the GPU, and so the order of its sums, goes by the step's lengths and the request's place among them)."""
    name = "B"
    page = TINY[name][2]
    toks = tokens_for(name, 90)
    ends = {"a": tokens_for(name, 12, salt=1), "b": tokens_for(name, 12, salt=2)}
    together = TraceSession(sharp_dirs[name], dtype, 640, page, kv_dtype="e4m3")
    together.run_step({"step": 0, "entries": [{"id": "a", "tokens": toks, "want": [0]}]})
    got = {"a": [], "b": []}
    for i in range(12):
        record = {"step": i + 1, "entries": [{"id": r, "tokens": [ends[r][i]], "want": [0]} for r in ("a", "b")]}
        if i == 0:
            record["fork"] = [{"from": "a", "to": "b"}]
        out, _ = together.run_step(record)
        for r, row in zip(("a", "b"), out):
            got[r].append(row)
    for row, r in enumerate(("a", "b")):
        alone = TraceSession(sharp_dirs[name], dtype, 640, page, kv_dtype="e4m3")
        alone.run_step({"step": 0, "entries": [{"id": "x", "tokens": toks, "want": [0]}]})
        alone.run_step({"step": 0, "entries": [{"id": "y", "tokens": toks, "want": [0]}]})
        for i in range(12):
            out, _ = alone.run_step({"step": 1, "entries": [{"id": "x", "tokens": [ends[r][i]], "want": [0]}, {"id": "y", "tokens": [ends[r][i]], "want": [0]}]})
            assert (out[row] == got[r][i]).all(), (r, i)
    shared = TraceSession(sharp_dirs[name], dtype, 640, page, prefix_cache=True, kv_dtype="e4m3")
    first, _ = shared.run_step({"step": 0, "entries": [{"id": "p", "tokens": toks, "want": [89]}]})
    again, cached = shared.run_step({"step": 1, "entries": [{"id": "q", "tokens": toks, "want": [89]}]})
    assert cached["q"] == 89 // page * page
    assert abs(first - again).max() <= 2.0 * 2.0**-8 * abs(first).max() if dtype == "bfloat16" else abs(first - again).max() <= 1e-4


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", sorted(TINY))
def test_generation(name, dtype, tiny_dirs):
    """Requests of different lengths, admitted while others decode, with and without captured graphs: the same tokens; and a pool
    of half the bytes for as many tokens."""
    made = []
    for graphs in (True, False):
        cfg = EngineConfig.defaults(str(tiny_dirs[name]), dtype=dtype, num_blocks=96, block_size=8, max_num_seqs=3, max_model_len=200,
                                    kv_dtype="e4m3", cuda_graphs=graphs, enable_prefix_cache=False)
        engine = LLMEngine(cfg)
        prompts = [tokens_for(name, n, salt=n) for n in (3, 50, 17, 90, 1)]
        made.append([o.token_ids for o in engine.generate(prompts, SamplingParams(max_tokens=20, temperature=0.0))])
        plain_need = engine.model.cache_needs()[0]
        held = plain_need.num_kv_heads * (plain_need.head_dim + 1) * 2 * TINY[name][0]["num_hidden_layers"]
        assert engine.cache.bytes_per_token() == held
        engine.cache.check_invariants()
    assert made[0] == made[1] and all(len(t) == 20 for t in made[0])


@pytest.mark.parametrize("kv_dtype", ["auto", "e4m3"])
def test_a_model_of_normed_heads(tmp_path, kv_dtype):
    raw = dict(TINY["B"][0], qk_norm=True)
    folder = write_random_model(tmp_path, raw, seed=3)
    outs = []
    for graphs in (True, False):
        engine = LLMEngine(EngineConfig.defaults(str(folder), dtype="bfloat16", num_blocks=64, block_size=8, max_num_seqs=2, max_model_len=200,
                                                 kv_dtype=kv_dtype, cuda_graphs=graphs))
        outs.append([o.token_ids for o in engine.generate([tokens_for("B", 40), tokens_for("B", 5)], SamplingParams(max_tokens=12, temperature=0.0))])
    assert outs[0] == outs[1]


def test_models_whose_rows_cannot_be_held_in_8_bits_are_refused():
    from clockwork_b200.parts import PagedKVNeed, SlotStateNeed

    for needs in ({0: PagedKVNeed(1, 64, planes=1)}, {0: PagedKVNeed(1, 64, e4m3=True), 1: PagedKVNeed(2, 64)}, {0: SlotStateNeed((4,))}):
        with pytest.raises(ValueError, match="e4m3"):
            CacheManager(needs, num_pages=4, page_size=8, kv_dtype="e4m3")
    with pytest.raises(ValueError, match="kv_dtype"):
        CacheManager({0: PagedKVNeed(1, 64, e4m3=True)}, num_pages=4, page_size=8, kv_dtype="e5m2")


@pytest.mark.parametrize("dtype", DTYPES)
def test_what_prompts_are_read_back_to_is_allocated_with_the_pool(dtype):
    """A pool that fits when it is made still does when the first prompt comes: a step allocates nothing of the pool's size."""
    part = build_part("mixer", PartSpec("attention", dict(hidden_size=80, num_heads=4, num_kv_heads=2, head_dim=64, qkv_bias=True, o_bias=False,
                                                          scale=0.125, window=None, position=PartSpec("rope_neox", {"theta": 5000.0, "rotary_dim": 64}))), "a", dtype, DEV)
    load(part, weights(part.tensor_decls(), dtype, seed=4))
    part.o = Untouched()
    before = torch.cuda.memory_allocated()
    cache = CacheManager({0: part.cache_need()}, num_pages=8000, page_size=16, dtype=dtype, device=DEV, num_state_slots=4, kv_dtype="e4m3")
    tokens = 8000 * 16
    assert cache.shared_bytes() == tokens * 2 * 2 * 64 * torch.finfo(dtype).bits // 8
    assert torch.cuda.memory_allocated() - before >= cache.shared_bytes() + tokens * cache.bytes_per_token()
    builder = StepBuilder(cache, dtype, DEV, cache.status)
    for rid, n in (("a", 300), ("b", 40), ("a", 200)):
        if rid not in cache.requests:
            cache.open(rid)
        prepared = builder.prepare([StepEntry(rid, [0] * n, [])])
        x = torch.randn(n, 80, device=DEV).to(dtype)
        part.qkv(x)
        quantised.step_workspace(64, 0)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        part.forward(prepared.ctx, x, prepared.ctx.views[0], None)
        ops.raise_on_status(cache.status)
        assert torch.cuda.max_memory_allocated() - held < cache.shared_bytes() // 2
        builder.commit(prepared)


@pytest.mark.parametrize("kv_dtype", ["auto", "e4m3"])
@pytest.mark.parametrize("heads", [(6, 2, 48), (4, 1, 128)])
def test_normed_heads_from_the_layer_s_input_on(heads, kv_dtype):
    """float32, from x to the output in float64 by the tensors' names: the query heads' norm is ``q_norm.weight``'s, the key heads' ``k_norm.weight``'s,
    before the rotation.  (The other tests take q and k from the kernel.)"""
    nh, nkv, hd = heads
    eps, theta, n, dtype, scale = 1e-5, 5000.0, 30, torch.float32, heads[2] ** -0.5
    part = build_part("mixer", PartSpec("attention", dict(hidden_size=80, num_heads=nh, num_kv_heads=nkv, head_dim=hd, qkv_bias=True, o_bias=False,
                                                          scale=scale, window=None, qk_norm=eps,
                                                          position=PartSpec("rope_neox", {"theta": theta, "rotary_dim": hd}))), "a", dtype, DEV)
    w = weights(part.tensor_decls(), dtype, seed=hd)
    w["a.q_norm.weight"] = 1.0 + 0.5 * torch.rand(hd, generator=torch.Generator().manual_seed(1))
    w["a.k_norm.weight"] = 1.0 - 0.5 * torch.rand(hd, generator=torch.Generator().manual_seed(2))
    load(part, w)
    part.o = Untouched()
    cache = CacheManager({0: part.cache_need()}, num_pages=8, page_size=8, dtype=dtype, device=DEV, num_state_slots=4, kv_dtype=kv_dtype)
    builder = StepBuilder(cache, dtype, DEV, cache.status)
    cache.open("a")
    x = torch.randn(n, 80, generator=torch.Generator().manual_seed(3))
    angle = torch.arange(n).double()[:, None] * (theta ** -(torch.arange(0, hd, 2).double() / hd)).float().double()

    def exact(name, count, norm):
        """A projection's heads, normed and turned, and how far float32 may be off: a sum of 81 terms, its error divided by the heads' size as
        it is; 24 roundings of each result (as in the store's own tests)."""
        m, b = w[f"a.{name}.weight"].double(), w[f"a.{name}.bias"].double()
        y = (x.double() @ m.T + b).view(n, count, hd)
        off = (82 * 2.0**-24 * (x.double().abs() @ m.abs().T + b.abs())).view(n, count, hd)
        if norm is None:
            return y, off
        root = (y.square().mean(-1, keepdim=True) + eps).sqrt()
        weight = w[f"a.{norm}.weight"].double()
        off = (off + y.abs() * off.square().mean(-1, keepdim=True).sqrt() / root) / root * weight
        y = y / root * weight
        c, s, h = angle.cos()[:, None], angle.sin()[:, None], hd // 2
        turn = lambda t, c, s: torch.cat([t[..., :h] * c - t[..., h:] * s, t[..., h:] * c + t[..., :h] * s], -1)  # noqa: E731
        off = turn(off, c.abs(), -s.abs()).abs() + torch.cat([off[..., :h], off[..., :h]], -1) * s.abs().repeat(1, 1, 2)
        return turn(y, c, s), off + 24 * 2.0**-24 * (y.abs() + torch.cat([y[..., h:], y[..., :h]], -1).abs())

    q, q_off = exact("q_proj", nh, "q_norm")
    k, k_off = exact("k_proj", nkv, "k_norm")
    v, v_off = exact("v_proj", nkv, None)
    if kv_dtype == "e4m3":  # half a step of the codes, and the whole of one where float32's error decides between two
        k_off, v_off = (off + 2.0**-4 * t.abs() + 2.0**-10 * t.abs().amax(-1, keepdim=True) / 223.0 * 2 for t, off in ((k, k_off), (v, v_off)))
    outs, done = [], 0
    for m in (17, 12, 1):
        prepared = builder.prepare([StepEntry("a", [0] * m, [])])
        outs.append(part.forward(prepared.ctx, x[done : done + m].to(DEV), prepared.ctx.views[0], None).double().cpu())
        ops.raise_on_status(cache.status)
        builder.commit(prepared)
        done += m
    want, size, _ = attention(q, k, v, 0, None, scale)
    group = nh // nkv
    k, k_off, v_off = (t.repeat_interleave(group, 1) for t in (k, k_off, v_off))
    score_off = scale * (torch.einsum("rhd,thd->rht", q_off, k.abs() + k_off) + torch.einsum("rhd,thd->rht", q.abs(), k_off)).amax(-1)[..., None]
    bound = 1.05 * torch.expm1(2 * score_off) * (size + v_off.amax((0, 2))[:, None]) + v_off.amax(0) + 2.0**-18 * size
    got = torch.cat(outs).view(n, nh, hd)
    worst = float(((got - want).abs() / bound).max())
    assert worst <= 1.0
    other, _, _ = attention(q / w["a.q_norm.weight"].double() * w["a.k_norm.weight"].double(), k[:, ::group] , v, 0, None, scale)
    assert kv_dtype == "e4m3" or float(((got - other).abs() / bound).max()) > 100  # (a mistaken norm would be far outside)
