"""What a model whose matrices are held in 8 bits takes of the device's memory: while it is loaded, and afterwards, as the pools' sizes see it."""

import gc

import pytest
import torch

from cwm_amd.engine import GenArgs, load_model
from cwm_amd.engine.engine import pool_sizes
from cwm_amd.engine.loading import random_model
from cwm_amd.weights import write_random_model
from helpers import configs

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


CONFIG = dict(
    configs.get("tiny_b"), dim=1024, n_layers=16, n_heads=16, n_kv_heads=16, head_dim=64, ffn_dim_multiplier=1.5, multiple_of=256,
)
CONFIG.pop("window_attn"), CONFIG.pop("layer_types")


def _matrix_bytes(model):
    layer = [abs(s.shape[0] * s.shape[1]) * 2 for n, s in model.tensor_specs().items() if n.startswith("layers.0.") and len(s.shape) == 2]
    return sum(layer), sum(layer) * len(model.blocks)


@pytest.mark.parametrize("from_folder", [True, False])
def test_memory_while_loading_and_after(tmp_path, from_folder):
    """bfloat16, sixteen layers.  Held in the end: a byte and a scale's share a value.  At most, while loading: beside that the originals of
    one layer, their joined copies, and a float32 drawing of one matrix, four layers' worth together."""
    if from_folder:
        write_random_model(str(tmp_path), CONFIG, 1, dtype="bfloat16")
    free, peak, sizes = {}, {}, {}
    for bits in (8, None):
        gc.collect()
        torch.cuda.empty_cache()
        before = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        if from_folder:
            model, _ = load_model(str(tmp_path), "bfloat16", DEV, stream_copies=False, weight_bits=bits)
        else:
            model, _ = random_model(CONFIG, 1, "bfloat16", DEV, stream_copies=False, weight_bits=bits)
        peak[bits] = torch.cuda.max_memory_allocated() - before
        free[bits] = torch.cuda.mem_get_info(DEV)[0]
        sizes[bits] = pool_sizes(model, GenArgs(max_batch=2, max_seq=-1, cache_block=64, weight_bits=bits), DEV)[None]
        layer, total = _matrix_bytes(model)
        page_bytes = sum(s.bytes_per_token(2) * 64 for s in model.cache_specs)
        del model
    assert total > 500e6
    assert peak[8] <= 0.51 * total + 4 * layer + 20e6
    # the pages that half the matrices' bytes make room for, less what the allocator rounds up
    assert sizes[8] - sizes[None] >= 0.9 * (0.45 * total - 64e6) / page_bytes
