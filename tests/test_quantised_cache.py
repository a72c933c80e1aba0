"""The quantised cache on the CPU: its layout, what a group is held as, and what the entry points refuse."""

import math

import pytest
import torch

from cwm_amd import ops
from helpers import quantised as held


@pytest.mark.parametrize("bits", [4, 8])
def test_a_group_is_held_within_half_a_step(bits):
    g = torch.Generator().manual_seed(bits)
    x = torch.randn(400, 32, generator=g) * torch.exp(6 * torch.randn(400, 1, generator=g)) + 20 * torch.randn(400, 1, generator=g)
    c, s, z = held.hold(x, bits)
    assert int(c.min()) >= 0 and int(c.max()) < 2 ** bits
    assert ((held.stands_for(c, s, z, bits) - x.double()).abs() <= s[:, None] / 2 * (1 + 1e-12)).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_equal_values_are_held_as_they_are(bits):
    x = torch.tensor([0.0, -0.0, 3.140625, -1e30, 1e-30]).bfloat16()[:, None].expand(5, 32)
    c, s, z = held.hold(x, bits)
    assert torch.equal(held.stands_for(c, s, z, bits), x.double()) and not s.any()


@pytest.mark.parametrize("bits,dim,page", [(4, 32, 8), (4, 96, 24), (8, 64, 8), (8, 160, 16)])
def test_the_layout_at_once_is_the_layout_one_by_one(bits, dim, page):
    g = torch.Generator().manual_seed(1)
    shape = (2, *ops.quant_page_shape(2, dim, page, bits))
    one, all_ = torch.full(shape, 7, dtype=torch.uint8), torch.full(shape, 7, dtype=torch.uint8)
    k, v = torch.randn(9, 2, dim, generator=g), torch.randn(9, 2, dim, generator=g)
    v[2, 1, 3] = math.inf
    pages, slots = torch.arange(9) % 2, torch.arange(9) // 2 + 1
    for t in range(9):
        held.put(one, int(pages[t]), int(slots[t]), k[t], v[t], bits)
    held.put_tokens(all_, pages, slots, k, v, bits)
    assert torch.equal(one, all_)


def test_sizes_that_are_refused():
    assert ops.quant_cache_limits(128, 256, 4) is None and ops.quant_cache_limits(32, 8, 8) is None
    assert "4 or 8 bits" in ops.quant_cache_limits(128, 256, 3)
    assert "multiple of 32" in ops.quant_cache_limits(80, 256, 4)
    assert "multiple of 32" in ops.quant_cache_limits(288, 256, 4)
    assert "multiple of 8" in ops.quant_cache_limits(64, 12, 4)
    assert "2 GiB" in ops.quant_cache_limits(256, 1 << 23, 8)


def test_there_is_no_cpu_path():
    k = torch.zeros(1, 1, 32)
    cache = torch.zeros((1, *ops.quant_page_shape(1, 32, 8, 4)), dtype=torch.uint8)
    one, table = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    with pytest.raises(ops.KernelError, match="HIP device"):
        ops.quant_kv_write(k, k, one, None, cache, table, one, 4)
    with pytest.raises(ops.KernelError, match="HIP device"):
        ops.quant_kv_read(cache, table, one, one, 32, 4, torch.float32)
    step = held.Step([1], [1], 8)
    with pytest.raises(ops.KernelError, match="HIP device"):
        ops.quant_paged_attention(k, cache, table, step.batch("cpu"), None, 1.0, 4)



@pytest.fixture
def no_device(monkeypatch):
    from cwm_amd.ops import quantised

    monkeypatch.setattr(quantised, "_check_device", lambda *t: None)
    monkeypatch.setattr(quantised, "_entries", {})

    def refuse(*a, **k):
        raise AssertionError("a call that should have been refused went on to the kernel")

    monkeypatch.setattr(quantised._build, "load", refuse)


def _write_args(**changed):
    a = dict(
        k=torch.zeros(3, 2, 64), v=torch.zeros(3, 2, 64), positions=torch.zeros(3, dtype=torch.int32), inv_freq=torch.zeros(32),
        cache=torch.zeros((2, *ops.quant_page_shape(2, 64, 16, 4)), dtype=torch.uint8), block_table=torch.zeros(1, 2, dtype=torch.int32),
        seq_of_token=torch.zeros(3, dtype=torch.int32), bits=4,
    )
    return {**a, **changed}


@pytest.mark.parametrize("changed,why", [
    (dict(bits=5), "4 or 8 bits"),
    (dict(bits=8), "does not fit"),
    (dict(k=torch.zeros(3, 2, 48), v=torch.zeros(3, 2, 48)), "multiple of 32"),
    (dict(k=torch.zeros(3, 128)), "contiguous heads"),
    (dict(k=torch.zeros(3, 64, 2).transpose(1, 2)), "contiguous heads"),
    (dict(v=torch.zeros(3, 1, 64)), "contiguous heads"),
    (dict(v=torch.zeros(2, 2, 64)), "contiguous heads"),
    (dict(v=torch.zeros(3, 2, 64, dtype=torch.bfloat16)), "one type"),
    (dict(k=torch.zeros(3, 2, 64, dtype=torch.float16), v=torch.zeros(3, 2, 64, dtype=torch.float16)), "float32 and bfloat16"),
    (dict(cache=torch.zeros((2, *ops.quant_page_shape(3, 64, 16, 4)), dtype=torch.uint8)), "does not fit"),
    (dict(cache=torch.zeros((2, 2, 1235), dtype=torch.uint8)), "does not fit"),
    (dict(cache=torch.zeros((2, 2, 12 * 76), dtype=torch.uint8)), "multiple of 8"),
    (dict(cache=torch.zeros((2, *ops.quant_page_shape(2, 64, 16, 4)), dtype=torch.int8)), "does not fit"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), r"\[T\]"),
    (dict(seq_of_token=torch.zeros(4, dtype=torch.int32)), r"\[T\]"),
    (dict(inv_freq=torch.zeros(64)), "rotary table"),
    (dict(inv_freq=torch.zeros(32, dtype=torch.float64)), "rotary table"),
    (dict(block_table=torch.zeros(2, dtype=torch.int32)), "block_table"),
    (dict(q=torch.zeros(3, 4, 32)), "contiguous heads"),
    (dict(q=torch.zeros(1, 4, 64).expand(3, 4, 64)), "overlap"),
])
def test_writes_that_are_refused(no_device, changed, why):
    with pytest.raises(ops.KernelError, match=why):
        ops.quant_kv_write(**_write_args(**changed))


@pytest.mark.parametrize("changed,why", [
    (dict(bits=6), "4 or 8 bits"),
    (dict(head_dim=96), "does not fit"),
    (dict(positions=torch.zeros(3, dtype=torch.int64)), "int32"),
    (dict(seq_of_token=torch.zeros(2, dtype=torch.int32)), r"\[T\]"),
    (dict(dtype=torch.float16), "float32 and bfloat16"),
])
def test_reads_that_are_refused(no_device, changed, why):
    a = _write_args()
    args = dict(cache=a["cache"], block_table=a["block_table"], positions=a["positions"], seq_of_token=a["seq_of_token"], head_dim=64, bits=4, dtype=torch.float32)
    with pytest.raises(ops.KernelError, match=why):
        ops.quant_kv_read(**{**args, **changed})


@pytest.mark.parametrize("changed,why", [
    (dict(bits=16), "4 or 8 bits"),
    (dict(window=0), "window"),
    (dict(scale=0.0), "positive"),
    (dict(scale=math.nan), "positive"),
    (dict(q=torch.zeros(3, 3, 64)), "divide"),
    (dict(q=torch.zeros(3, 4, 32)), "does not fit|multiple"),
    (dict(q=torch.zeros(3, 4, 64, dtype=torch.float64)), "float32 and bfloat16"),
    (dict(q=torch.zeros(2, 4, 64)), "for its tokens"),
    (dict(q=torch.zeros(3, 4 * 64 + 2)[:, :256].unflatten(1, (4, 64))), "aligned"),
    (dict(block_table=torch.zeros(2, 2, dtype=torch.int32)), "for the batch"),
    (dict(block_table=torch.zeros(1, 2, dtype=torch.int64)), "int32"),
])
def test_attention_that_is_refused(no_device, changed, why):
    args = dict(q=torch.zeros(3, 4, 64), cache=_write_args()["cache"], block_table=torch.zeros(1, 2, dtype=torch.int32),
                batch=held.Step([3], [5], 16).batch("cpu"), window=None, scale=0.125, bits=4)
    with pytest.raises(ops.KernelError, match=why):
        ops.quant_paged_attention(**{**args, **changed})


def _product_args(**changed):
    a = dict(x=torch.zeros(3, 64), weight=torch.zeros(5, 64, dtype=torch.int8), weight_scale=torch.ones(5), bias=None, out_dtype=None)
    return {**a, **changed}


@pytest.mark.parametrize("changed,why", [
    (dict(x=torch.zeros(3, 48)), "do not fit"),
    (dict(x=torch.zeros(64)), "do not fit"),
    (dict(x=torch.zeros(3, 40), weight=torch.zeros(5, 40, dtype=torch.int8)), "multiple of 16"),
    (dict(x=torch.zeros(1, 131088), weight=torch.zeros(1, 131088, dtype=torch.int8), weight_scale=torch.ones(1)), "131072"),
    (dict(weight=torch.zeros(5, 64)), "int8"),
    (dict(weight=torch.zeros(64, 5, dtype=torch.int8).t()), "int8"),
    (dict(weight=torch.zeros(5, 72, dtype=torch.int8)[:, :64]), "aligned"),
    (dict(weight=torch.zeros(1, 64, dtype=torch.int8).expand(5, 64)), "aligned"),
    (dict(weight_scale=torch.ones(4)), "scales"),
    (dict(weight_scale=torch.ones(5, dtype=torch.bfloat16)), "scales"),
    (dict(bias=torch.ones(4)), "bias"),
    (dict(bias=torch.ones(5, dtype=torch.bfloat16)), "bias"),
    (dict(out_dtype=torch.float16), "float32 and bfloat16"),
    (dict(x=torch.zeros(3, 64, dtype=torch.float16), out_dtype=torch.float32), "float32 and bfloat16"),
    (dict(x=torch.zeros(64, 3).t()), "contiguous rows"),
])
def test_products_that_are_refused(no_device, changed, why):
    with pytest.raises(ops.KernelError, match=why):
        ops.linear_int8(**_product_args(**changed))


def test_the_product_has_no_cpu_path():
    with pytest.raises(ops.KernelError, match="HIP device"):
        ops.linear_int8(**_product_args())
    with pytest.raises(ops.KernelError, match="HIP device"):
        ops.quantize_rows(torch.zeros(2, 16))


def test_entry_points_are_those_of_their_build(monkeypatch):
    """A library's builds export the same names with other arguments: none gets another's, and one whose arguments are not known is refused."""
    from cwm_amd.ops import quantised

    class Library(dict):
        def __missing__(self, name):
            self[name] = type("Function", (), {})()
            return self[name]

    built = {}

    def load(library, defines=None):
        return built.setdefault((library, tuple(sorted((defines or {}).items()))), Library())

    monkeypatch.setattr(quantised, "_entries", {})
    monkeypatch.setattr(quantised._build, "load", load)
    half = quantised._entry("attention_mfma", "cwm_attention_mfma", 64, "HALF_INPUTS")
    assert half[0] is built["attention_mfma", (("HALF_INPUTS", 1), ("HEAD_DIM", 64))]["cwm_attention_mfma"] and len(half[0].argtypes) == 37
    assert quantised._entry("attention_mfma", "cwm_attention_mfma", 64, "HALF_INPUTS") is half
    assert quantised._entry("attention_mfma", "cwm_attention_mfma", 128, "HALF_INPUTS") is not half
    for switches in ((), ("KEPT_KEYS",)):
        with pytest.raises(KeyError):
            quantised._entry("attention_mfma", "cwm_attention_mfma", 64, *switches)
    assert quantised._entry("quant_cache", "cwm_quant_kv_read") is quantised._entry("quant_cache", "cwm_quant_kv_read")
