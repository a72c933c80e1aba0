"""Options of fewer bits on the CPU: what is refused, and what a cache of bytes tells the manager and the storage."""

import pytest
import torch

from cwm_amd.cache import CacheManager, CacheStorage
from cwm_amd.config.registry import parse_config
from cwm_amd.engine import Engine, GenArgs
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
