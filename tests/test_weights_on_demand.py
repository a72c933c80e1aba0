"""Loading a model whose matrices are held in 8 bits: the originals of one layer at a time, on the CPU (the rows' quantiser, which has no CPU
path, replaced by its definition)."""

import gc
import weakref

import pytest
import torch

from cwm_amd import ops
from cwm_amd.config.registry import parse_config
from cwm_amd.engine import loading
from cwm_amd.models.model import Model
from cwm_amd.parts.base import Runtime
from cwm_amd.weights import TensorsOnDemand, load_tensors, open_tensors
from helpers import configs, models

CPU = torch.device("cpu")


def _rows(x):
    x = x.float()
    a = x.abs().amax(1) / torch.full((x.shape[0],), 127.0)
    return torch.where(a[:, None] > 0, torch.round(x / a[:, None]), torch.zeros_like(x)).to(torch.int8), a


def test_tensors_are_made_when_asked_for():
    asked = []

    def make(name):
        asked.append(name)
        return torch.zeros(1)

    tensors = TensorsOnDemand(["b", "a"], make)
    assert list(tensors) == ["b", "a"] and len(tensors) == 2 and "a" in tensors and "c" not in tensors and not asked
    assert tensors["a"] is not tensors["a"] and asked == ["a", "a"]
    with pytest.raises(KeyError):
        tensors["c"]
    assert list(dict(tensors)) == ["b", "a"] and asked == ["a", "a", "b", "a"]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_folder_read_on_demand_is_the_folder(tmp_path, dtype):
    folder = models.make_folder(tmp_path, "tiny_b", seed=3, dtype="float32")
    arch, config = parse_config(configs.get("tiny_b"))
    specs = Model(arch.build_plan(config)).tensor_specs()
    at_once, on_demand = load_tensors(folder, specs, dtype, CPU), open_tensors(folder, specs, dtype, CPU)
    assert type(at_once) is dict and list(at_once) == list(on_demand) and set(at_once) == set(specs)
    assert all(torch.equal(at_once[n], on_demand[n]) and at_once[n].dtype == on_demand[n].dtype for n in specs)


@pytest.mark.parametrize("from_folder", [True, False])
def test_the_originals_of_one_layer_at_a_time(tmp_path, monkeypatch, from_folder):
    monkeypatch.setattr(ops, "quantize_rows", _rows)
    most, alive = [0], [0]

    def counted(make):
        def get(self, name):
            t = make(self, name)
            if name.startswith("layers.") and t.dim() == 2:
                t = t.clone()
                alive[0] += t.numel()
                most[0] = max(most[0], alive[0])
                weakref.finalize(t, lambda n=t.numel(): alive.__setitem__(0, alive[0] - n))
            return t

        return get

    monkeypatch.setattr(TensorsOnDemand, "__getitem__", counted(TensorsOnDemand.__getitem__))
    if from_folder:
        model, _ = loading.load_model(models.make_folder(tmp_path, "tiny_b", seed=3), "float32", CPU, weight_bits=8)
    else:
        model, _ = loading.random_model(configs.get("tiny_b"), 3, "float32", CPU, weight_bits=8)
    gc.collect()
    matrices = [abs(s.shape[0] * s.shape[1]) for n, s in model.tensor_specs().items() if n.startswith("layers.") and len(s.shape) == 2]
    layers = len(model.blocks)
    assert layers > 1 and alive[0] == 0 and most[0] == sum(matrices) // layers
    held = [w for b in model.blocks for w in (b.mixer.qkv, b.mixer.wo, b.feed_forward.gate_up, b.feed_forward.down)]
    assert all(w.weight is None and w.codes.dtype == torch.int8 for w in held)


def test_every_tensor_is_asked_for_once():
    arch, config = parse_config(configs.get("tiny_b"))
    model = Model(arch.build_plan(config))
    specs = model.tensor_specs()
    asked = []

    def make(name):
        asked.append(name)
        return torch.zeros(specs[name].drawn_shape())

    model.bind(TensorsOnDemand(specs, make), Runtime(CPU, torch.float32))
    assert sorted(asked) == sorted(specs)
