"""What the operators of the 8-bit cache refuse, on the CPU: everything is looked at before the device is."""

import pytest
import torch

from clockwork_b200.ops import quantised
from tests.e4m3_tools import CODES, filled_pages, nearest_codes, quantise


def _args(n=3, nh=4, nkv=2, hd=32, page=8, pages=4, dtype=torch.bfloat16):
    cache = quantised.E4M3Pages(torch.zeros(pages, page, nkv, hd).to(CODES), torch.zeros(pages, page, nkv, hd).to(CODES),
                                torch.zeros(pages, nkv, page, dtype=torch.uint8), torch.zeros(pages, nkv, page, dtype=torch.uint8))
    ints = torch.zeros(n, dtype=torch.int32)
    return dict(qkv=torch.zeros(n, (nh + 2 * nkv) * hd, dtype=dtype), positions=ints, slots=ints.clone(), inv_freq=torch.ones(hd // 2), cache=cache,
                num_heads=nh, num_kv_heads=nkv, head_dim=hd, status=torch.zeros(4, dtype=torch.int32))


STORE = [
    (dict(qkv=torch.zeros(3, 256, dtype=torch.float16)), "dtype"), (dict(qkv=torch.zeros(3, 250, dtype=torch.bfloat16)), "qkv"),
    (dict(qkv=torch.zeros(256, 3, dtype=torch.bfloat16).T), "qkv"), (dict(positions=torch.zeros(3)), "positions"),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), "positions"), (dict(slots=torch.zeros(3, dtype=torch.int64)), "slots"),
    (dict(inv_freq=torch.ones(17)), "turns"), (dict(inv_freq=torch.ones(16, dtype=torch.float64)), "inv_freq"),
    (dict(q_weight=torch.ones(31)), "q_weight"), (dict(k_weight=torch.ones(32, dtype=torch.bfloat16)), "k_weight"),
    (dict(num_kv_heads=1, num_heads=6), "KV heads"), (dict(status=torch.zeros(3, dtype=torch.int32)), "status"),
    (dict(cache=quantised.PlainPages(torch.zeros(4, 8, 2, 32), torch.zeros(4, 8, 2, 32))), "plain cache"),
    (dict(head_dim=512, num_kv_heads=0, num_heads=0, qkv=torch.zeros(3, 0, dtype=torch.bfloat16)), "head_dim"), ({}, "CUDA")]


@pytest.mark.parametrize("change, words", STORE)
def test_store_refuses(change, words):
    with pytest.raises(ValueError, match=words):
        quantised.norm_rotate_store(**{**_args(), **change})


def _bad_caches():
    c = _args()["cache"]
    yield c._replace(k=c.k.float()), "float8"
    yield c._replace(v_exp=c.v_exp.to(torch.int8)), "uint8"
    yield c._replace(k_exp=torch.zeros(4, 8, 2, dtype=torch.uint8)), "belong"
    yield c._replace(v=torch.zeros(4, 8, 2, 16).to(CODES)), "belong"
    yield c._replace(k=torch.zeros(4, 2, 8, 32).to(CODES).transpose(1, 2)), "contiguous"
    yield quantised.PlainPages(c.k, c.v), "8-bit cache"


@pytest.mark.parametrize("cache, words", list(_bad_caches()))
def test_caches_that_do_not_fit_together_are_refused(cache, words):
    with pytest.raises(ValueError, match=words):
        quantised.attention_decode(torch.zeros(3, 128, dtype=torch.bfloat16), cache, torch.zeros(3, 2, dtype=torch.int32),
                                   torch.zeros(3, dtype=torch.int32), 4, 1.0, torch.zeros(4, dtype=torch.int32))


DECODE = [(dict(q=torch.zeros(3, 100, dtype=torch.bfloat16)), "q must"), (dict(q=torch.zeros(4, 128, dtype=torch.bfloat16)), "rows"),
          (dict(num_heads=3), "multiple"), (dict(num_heads=0), "multiple"), (dict(window=0), "window"), (dict(ctx_lens=torch.zeros(2, dtype=torch.int32)), "ctx_lens"),
          (dict(block_tables=torch.zeros(3, 2, dtype=torch.int64)), "block_tables"), (dict(q_start=torch.zeros(4, dtype=torch.int32)), "output"),
          (dict(out=torch.zeros(3, 128)), "out"), (dict(q=torch.zeros(3, 256, dtype=torch.bfloat16)[:, ::2]), "stride"), ({}, "CUDA")]


@pytest.mark.parametrize("change, words", DECODE)
def test_decode_refuses(change, words):
    args = dict(q=torch.zeros(3, 128, dtype=torch.bfloat16), cache=_args()["cache"], block_tables=torch.zeros(3, 2, dtype=torch.int32),
                ctx_lens=torch.zeros(3, dtype=torch.int32), num_heads=4, scale=1.0, status=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match=words):
        quantised.attention_decode(**{**args, **change})


READ = [(dict(out_k=torch.zeros(4, 8, 2, 16)), "out_k"), (dict(out_v=torch.zeros(4, 8, 2, 32, dtype=torch.bfloat16)), "out_v"), (dict(window=-1), "window"),
        (dict(q_start=torch.zeros(3, dtype=torch.int32)), "q_start"), (dict(status=torch.zeros(4)), "status"), ({}, "CUDA")]


@pytest.mark.parametrize("change, words", READ)
def test_read_refuses(change, words):
    args = dict(cache=_args()["cache"], block_tables=torch.zeros(3, 2, dtype=torch.int32), ctx_lens=torch.zeros(3, dtype=torch.int32),
                out_k=torch.zeros(4, 8, 2, 32), out_v=torch.zeros(4, 8, 2, 32), status=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match=words):
        quantised.read_pages(**{**args, **change})


STEP = [*((change, words) for change, words in STORE if "cache" not in change), (dict(cache=quantised.PlainPages(torch.zeros(4, 8, 2, 32), torch.zeros(4, 8, 2, 32))), "8-bit cache"),
        (dict(block_tables=torch.zeros(2, 2, dtype=torch.int32)), "block_tables"), (dict(block_tables=torch.zeros(3, 2)), "block_tables"),
        (dict(ctx_lens=torch.zeros(3, dtype=torch.int64)), "ctx_lens"), (dict(window=0), "window"),
        (dict(num_heads=3, qkv=torch.zeros(3, 224, dtype=torch.bfloat16)), "multiple"),
        (dict(cache=_args(hd=24)["cache"], head_dim=24, qkv=torch.zeros(3, 192, dtype=torch.bfloat16), inv_freq=None), "multiple of 16")]


@pytest.mark.parametrize("change, words", STEP)
def test_step_refuses(change, words):
    args = dict(**_args(), block_tables=torch.zeros(3, 2, dtype=torch.int32), ctx_lens=torch.zeros(3, dtype=torch.int32), scale=1.0)
    for early in (False, True):
        with pytest.raises(ValueError, match=words):
            quantised.decode_step(**{**args, **change}, early=early)


PORTIONS = [(dict(q=torch.zeros(5, 100, dtype=torch.bfloat16)), "q must"), (dict(q=torch.zeros(5, 128, dtype=torch.float16)), "dtype"),
            (dict(q=torch.zeros(5, 256, dtype=torch.bfloat16)[:, ::2]), "stride"), (dict(num_heads=3), "multiple"), (dict(num_heads=0), "multiple"),
            (dict(num_heads=2), "plan is for"), (dict(q=torch.zeros(4, 128, dtype=torch.bfloat16)), "plan is for"),
            (dict(q_start=torch.zeros(3, dtype=torch.int32)), "q_start"), (dict(ctx_lens=torch.zeros(3)), "ctx_lens"),
            (dict(block_tables=torch.zeros(2, 2, dtype=torch.int32), ctx_lens=torch.zeros(2, dtype=torch.int32), q_start=torch.zeros(3, dtype=torch.int32)), "plan is for"),
            (dict(cache=_args(page=16)["cache"]), "plan is for"), (dict(window=-2), "window"), (dict(status=torch.zeros(4)), "status"), ({}, "CUDA")]


@pytest.mark.parametrize("change, words", PORTIONS)
def test_portions_refuse(change, words):
    args = dict(q=torch.zeros(5, 128, dtype=torch.bfloat16), cache=_args()["cache"], block_tables=torch.zeros(3, 2, dtype=torch.int32),
                q_start=torch.tensor([0, 2, 2, 5], dtype=torch.int32), ctx_lens=torch.tensor([2, 0, 9], dtype=torch.int32),
                plan=quantised.plan_portions([2, 0, 3], [2, 0, 9], 4, 2, 32, 8, "cpu"), num_heads=4, scale=1.0, status=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match=words):
        quantised.attention_portions(**{**args, **change})


def test_plans_of_impossible_portions_are_refused():
    with pytest.raises(ValueError, match="context"):
        quantised.plan_portions([3, 2], [5, 1], 4, 2, 32, 8, "cpu")
    with pytest.raises(ValueError, match="context"):
        quantised.plan_portions([3], [5, 1], 4, 2, 32, 8, "cpu")
    with pytest.raises(ValueError, match="KV heads"):
        quantised.plan_portions([3], [5], 5, 2, 32, 8, "cpu")


def test_requests_of_few_rows_go_with_the_others_where_they_have_little_behind_them():
    most = quantised.short_rows(12, 2, 128)
    assert most == 16 and quantised.plan_portions([7, 10], [7, 200], 12, 2, 128, 5, "cpu").short == 17  # there are no others
    assert quantised.plan_portions([7, 10, 200], [7, 200, 200], 12, 2, 128, 5, "cpu").short == 0
    edge = quantised.TOGETHER_ENTRIES // 256
    assert quantised.plan_portions([7, 200], [edge, 200], 12, 2, 128, 5, "cpu").short == 0
    assert quantised.plan_portions([7, 200], [edge + 1, 200], 12, 2, 128, 5, "cpu").short == 7
    assert quantised.plan_portions([7, 1, 200], [edge + 1, 9, 200], 12, 2, 128, 5, "cpu", least_rows=2).short == 7
    assert quantised.plan_portions([1, 7, 200], [10 * edge, 9, 200], 12, 2, 128, 5, "cpu", least_rows=2).short == 0  # (the one is served apart)


def test_the_oracle_rounds_as_the_type_does():
    x = torch.cat([torch.linspace(-448, 448, 4097).double(), torch.ldexp(torch.linspace(1, 2, 65).double(), torch.tensor(-9))])
    assert torch.equal(nearest_codes(x), x.float().to(CODES).double())


def test_the_oracle_holds_rows_within_half_a_step():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(200, 64, generator=g) * torch.exp(3 * torch.randn(200, 1, generator=g))
    codes, e = quantise(x)
    unit = torch.exp2(e.double() - 127)[:, None]
    assert ((codes.double() * unit - x.double()).abs() <= torch.maximum(2.0**-4 * x.double().abs(), 2.0**-10 * unit)).all()
    assert (codes.double().abs().amax(1) > 216).all()  # no power is larger than it has to be (224, rounded)
    cache, tables = filled_pages([9, 0, 3], 4, 2, 16, g)
    assert tables.shape == (3, 3) and (tables[1] == -1).all() and cache[0].dtype == CODES


@pytest.mark.parametrize("back", [torch.zeros(2, 4, 8, 2, 32, dtype=torch.bfloat16), quantised.PlainPages(torch.zeros(4, 8, 2, 32), torch.zeros(4, 8, 2, 32)),
                                  quantised.PlainPages(torch.zeros(4, 8, 2, 32, dtype=torch.bfloat16), torch.zeros(3, 8, 2, 32, dtype=torch.bfloat16)),
                                  quantised.PlainPages(*(torch.zeros(4, 2, 8, 32, dtype=torch.bfloat16).transpose(1, 2) for _ in range(2)))])
def test_pages_to_read_back_to_that_do_not_fit_are_refused(back):
    with pytest.raises(ValueError, match="back must be"):
        quantised._check_back(back, _args()["cache"], torch.zeros(5, 128, dtype=torch.bfloat16))


@pytest.mark.parametrize("new, most, start, width, refused", [([2, 0, 3], 0, 1, 160, "16 bytes"), ([2, 0, 3], 0, 0, 161, "16 bytes"), ([2, 0, 3], 5, 1, 160, "4 bytes"),
                                                              ([2, 0, 3], 5, 0, 161, "4 bytes"), ([2, 0, 3], 5, 2, 162, "CUDA"), ([2, 0, 3], 0, 8, 168, "CUDA")])
def test_portions_whose_rows_begin_where_no_kernel_reads_them_are_refused(new, most, start, width, refused):
    """Before anything is launched; rows that can be read get as far as the device's check."""
    args = dict(q=torch.zeros(5, width, dtype=torch.bfloat16)[:, start : start + 128], cache=_args()["cache"], block_tables=torch.zeros(3, 2, dtype=torch.int32),
                q_start=torch.tensor([0, 2, 2, 5], dtype=torch.int32), ctx_lens=torch.tensor([2, 0, 9], dtype=torch.int32),
                plan=quantised.plan_portions(new, [2, 0, 9], 4, 2, 32, 8, "cpu", most_rows=most), num_heads=4, scale=1.0, status=torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match=refused):
        quantised.attention_portions(**args)
