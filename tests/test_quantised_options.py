"""Options of fewer bits on the CPU: what is refused, and what a cache of bytes tells the manager and the storage."""

import pytest
import torch

from cwm_amd import ops
from cwm_amd.cache import CacheManager, CacheStorage
from cwm_amd.config.registry import parse_config
from cwm_amd.engine import Engine, GenArgs, pool_sizes
from cwm_amd.models.model import Model
from cwm_amd.parts.base import PagedKVSpec, QuantKVSpec, Runtime
from cwm_amd.parts.linear import LinearWeights
from helpers import configs, lapevik


def _plan(config):
    arch, typed = parse_config(config)
    return arch.build_plan(typed)


@pytest.mark.parametrize("options", [dict(cache_bits=16), dict(cache_bits=2), dict(weight_bits=4), dict(weight_bits=16)])
def test_bits_that_do_not_exist(options):
    with pytest.raises(ValueError, match="bits must be"):
        GenArgs(**options)


def test_a_cache_of_bytes():
    config = configs.get("tiny_d")
    model = Model(_plan(config), cache_bits=4)
    assert all(isinstance(s, QuantKVSpec) and s.bits == 4 for s in model.cache_specs)
    assert {s.window for s in model.cache_specs} == {s.window for s in Model(_plan(config)).cache_specs}
    spec = model.cache_specs[0]
    assert spec.page_shape(16) == (2, 16 * (64 + 12)) and spec.bytes_per_token(2) == spec.bytes_per_token(4) == 2 * 76
    manager = CacheManager(model.cache_specs, 16, 3, 2)
    storage = CacheStorage(manager, torch.device("cpu"), torch.bfloat16)
    assert all(t.dtype == torch.uint8 and t.shape == (3, 2, 16 * 76) for t in storage.paged.values())
    storage.fill_pages(0, [1], float("nan"))
    filled = storage.paged[manager.groups[0].cache_ids[0]]
    assert (filled[1] == 255).all() and not filled[0].any()
    with pytest.raises(ValueError, match="multiple of 8"):
        CacheStorage(CacheManager(model.cache_specs, 4, 3, 2), torch.device("cpu"), torch.bfloat16)


def test_the_storage_of_other_caches_is_as_it_was():
    model = Model(_plan(configs.get("tiny_d")))
    manager = CacheManager(model.cache_specs, 16, 3, 2)
    assert all(type(s) is PagedKVSpec for s in model.cache_specs)
    assert all(t.dtype == torch.bfloat16 for t in CacheStorage(manager, torch.device("cpu"), torch.bfloat16).paged.values())


def test_models_that_cannot():
    with pytest.raises(ValueError, match="multiple of 32"):
        Model(_plan(configs.get("tiny_a")), cache_bits=4)  # heads of 16
    other = _plan(lapevik.get("tiny_p"))
    with pytest.raises(ValueError, match="activations' type only"):
        Model(other, cache_bits=8)
    with pytest.raises(ValueError, match="activations' type only"):
        Model(other).bind({}, Runtime(torch.device("cpu"), torch.float32, weight_bits=8))
    with pytest.raises(ValueError, match="8 bits"):
        Model(_plan(configs.get("tiny_b"))).bind({}, Runtime(torch.device("cpu"), torch.float32, weight_bits=4))


def test_what_8_bits_are_refused():
    model = Model(_plan(configs.get("tiny_b")))
    model.blocks = [object()]
    with pytest.raises(ValueError, match="keeps its parts itself"):
        model.bind({}, Runtime(torch.device("cpu"), torch.float32, weight_bits=8))
    matrix = LinearWeights(torch.randn(32, 64))
    matrix.codes = torch.zeros(32, 64, dtype=torch.int8)
    with pytest.raises(ValueError, match="not divided"):
        matrix.rows(0, 16)


def test_an_engine_asks_for_what_its_model_has():
    model = Model(_plan(configs.get("tiny_b")))
    model.runtime = Runtime(torch.device("cpu"), torch.float32)
    with pytest.raises(ValueError, match="cache_bits=8 is asked for"):
        Engine(GenArgs(max_seq=64, cache_block=16, cache_bits=8), model)
    with pytest.raises(ValueError, match="weight_bits=8 is asked for"):
        Engine(GenArgs(max_seq=64, cache_block=16, weight_bits=8), model)


def test_what_portions_unpack_is_reserved():
    """Pools sized from free memory leave room for the keys and values, in 16 bits, of a request of the context's length in one layer, and for
    the partial results of its chunks."""
    config = dict(configs.get("tiny_d"), n_layers=2, n_heads=48, n_kv_heads=8, head_dim=128, max_seq_len=131072)
    config.pop("window_attn")

    def taken(cache_bits, dtype=torch.bfloat16, **changed):
        model = Model(_plan(dict(config, **changed)), cache_bits=cache_bits)
        model.runtime = Runtime(torch.device("cpu"), dtype)
        sizes = pool_sizes(model, GenArgs(max_seq=-1, cache_block=256, cache_bits=cache_bits), torch.device("cuda:0"), free_bytes=int(20e9))
        esize = 4 if dtype == torch.float32 else 2
        return sum(sizes[None] * 256 * spec.bytes_per_token(esize) for spec in model.cache_specs) / 0.9

    one = 131072 * 4 * 8 * 128
    work = ops.quant_attention_workspace(8, 128, 131072, 256)
    assert one < work < one + 200e6
    assert abs(taken(None) - 18e9) < 2e6 and abs(taken(4, torch.float32) - 18e9) < 2e6
    for bits in (4, 8):
        assert abs(taken(bits) - (18e9 - work)) < 2e6
    assert abs(taken(4, max_seq_len=1 << 20) - (18e9 - ops.quant_attention_workspace(8, 128, 1 << 20, 256))) < 2e6
    # a window's portions read no more than the window and the portion
    assert ops.quant_attention_workspace(8, 128, 8191 + 4096, 256) == ops.quantised.UNPACK_BYTES


def _step(new, kv):
    from helpers.quantised import Step

    return Step(new, kv, 256).batch("cpu")


def test_portions_take_turns(monkeypatch):
    """Sequences of many rows share a turn while what they unpack fits; every other one is in the first."""
    from cwm_amd.ops import quantised

    monkeypatch.setattr(quantised, "_units", lambda device: 256)
    monkeypatch.setattr(quantised, "UNPACK_BYTES", 20 << 20)  # 4 KiB a key of 8 heads of 128: 5,120 keys
    device = torch.device("cpu")
    new, kv = [1, 100, 100, 1, 100, 300, 0, 40], [9000, 2000, 1000, 50, 3000, 30000, 77, 500]
    batch = _step(new, kv)
    turns = quantised._turns(batch, 6, None, 8, 128, device)
    assert quantised._turns(batch, 6, None, 8, 128, device) is turns
    assert [[b for b, m in enumerate(t.q_lens) if m] for t in turns] == [[0, 1, 2, 3], [4], [5], [7]]
    assert all(t.kv_lens == kv and t.n_tokens == batch.n_tokens and t.cu_q is batch.cu_q for t in turns)
    assert [sum(t.q_lens[b] for t in turns) for b in range(len(new))] == new
    windowed = quantised._turns(batch, 6, 500, 8, 128, device)
    assert len(windowed) < len(turns)
    few = _step([1, 100], [9, 2000])
    assert quantised._turns(few, 6, None, 8, 128, device) == []
