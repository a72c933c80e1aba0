from .loader import TensorsOnDemand, WeightError, load_tensors, open_tensors, target_dtype, weight_files
from .random_init import random_tensor, random_tensors, write_random_model

__all__ = [
    "WeightError",
    "load_tensors",
    "target_dtype",
    "weight_files",
    "random_tensor",
    "random_tensors",
    "write_random_model",
]
