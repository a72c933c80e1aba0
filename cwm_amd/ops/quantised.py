"""Entry points of the kernels that serve in fewer bits: the paged cache of keys and values in 4 or 8 bits
(`csrc/quant_cache.hip`, `csrc/attention_quant.hip`; layout and formulas in `csrc/quant_cache.h`), and the product of 8-bit
integers with a scale for every token and output channel (`csrc/gemm_int8.hip`).  Shapes, types and devices are checked on the
host; there is no CPU path."""

from __future__ import annotations

import ctypes
import functools
from typing import Optional, Tuple

import torch

from . import build as _build

CACHE_BITS = (4, 8)
QUANT_MAX_DIM = 256  # csrc/quant_cache.h


@functools.cache  # an import statement costs a launch-bound step a microsecond and more a call
def _base():
    from . import KernelError, _check, _code, _i32, _need_gpu, _ptr, _stream  # the shared helpers of this package

    return KernelError, _check, _code, _i32, _need_gpu, _ptr, _stream


def _token_bytes(head_dim: int, bits: int) -> int:
    """Bytes of one token of one key/value head: codes of key and value, a word for every 32 elements of the key, one for the value."""
    return 2 * (head_dim * bits // 8) + head_dim // 32 * 4 + 4


def quant_cache_limits(head_dim: int, page_size: int, bits: int) -> Optional[str]:
    """Why a cache of `bits` bits cannot hold heads of this size in pages of this many tokens, or None if it can."""
    if bits not in CACHE_BITS:
        return f"a quantised cache holds 4 or 8 bits a value, not {bits}"
    if head_dim % 32 != 0 or not 32 <= head_dim <= QUANT_MAX_DIM:
        return f"a quantised cache takes head sizes of a multiple of 32 up to {QUANT_MAX_DIM}, not {head_dim}"
    if page_size < 1 or page_size % 8 != 0:
        return f"a quantised cache takes pages of a multiple of 8 tokens, not {page_size}"
    if page_size * _token_bytes(head_dim, bits) >= 2 ** 31:
        return f"a quantised cache takes pages whose heads have less than 2 GiB, not {page_size} tokens"
    return None


def quant_page_shape(n_kv_heads: int, head_dim: int, page_size: int, bits: int) -> Tuple[int, int]:
    """Shape of one page of a quantised cache (uint8): [key/value heads, bytes of a head]."""
    return (n_kv_heads, page_size * _token_bytes(head_dim, bits))


def _check_cache(cache: torch.Tensor, block_table: torch.Tensor, n_kv: Optional[int], head_dim: int, bits: int) -> int:
    """The tokens of a page of `cache`, a contiguous uint8 [pages, key/value heads, head bytes]."""
    KernelError, _, _, _i32, *_ = _base()
    if bits not in CACHE_BITS:
        raise KernelError(f"a quantised cache holds 4 or 8 bits a value, not {bits}")
    if head_dim % 32 != 0 or not 32 <= head_dim <= QUANT_MAX_DIM:
        raise KernelError(f"a quantised cache takes head sizes of a multiple of 32 up to {QUANT_MAX_DIM}, not {head_dim}")
    token = 2 * (head_dim * bits // 8) + head_dim // 32 * 4 + 4
    if (
        cache.dtype != torch.uint8 or cache.dim() != 3 or not cache.is_contiguous() or cache.shape[0] < 1 or cache.shape[1] < 1
        or (n_kv is not None and cache.shape[1] != n_kv) or cache.shape[2] < 1 or cache.shape[2] % token != 0
    ):
        raise KernelError(f"cache {tuple(cache.shape)} {cache.dtype} does not fit {n_kv or 'any'} heads of size {head_dim} in {bits} bits")
    page_size = cache.shape[2] // token
    why = quant_cache_limits(head_dim, page_size, bits)
    if why is not None:
        raise KernelError(why)
    _i32(block_table, "block_table")
    if block_table.dim() != 2 or block_table.shape[1] < 1:
        raise KernelError("block_table must be [B, W]")
    return page_size


def _check_device(*tensors: Optional[torch.Tensor]) -> None:
    """All on one device, and that the current one: kernels are launched on its stream."""
    KernelError, *_ = _base()
    current = torch._C._cuda_getDevice()
    for t in tensors:
        if t is not None and t.get_device() != current:
            raise KernelError(f"a tensor is on {t.device}, the current device is cuda:{current}")


def quant_kv_write(
    k: torch.Tensor,
    v: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: Optional[torch.Tensor],
    cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_of_token: torch.Tensor,
    bits: int,
    q: Optional[torch.Tensor] = None,
) -> None:
    """Rotate `k` [T, Hkv, hd] by positions * inv_freq (adjacent pairs; None: no rotation), round it to its type, and write it
    and `v` into the paged `cache` in 4 or 8 bits ([pages, Hkv, head bytes] of uint8, `quant_page_shape`) at the rows the block
    table gives; tokens whose page is not held are not written.  `k` and `v` (float32 or bfloat16) stay as they are; they may be
    views into one wider tensor (token stride free, heads contiguous).  `q` [T, Hq, hd], where given, is rotated in place by the
    same angles.  No two tokens of a call may have the same place.  A group of values with an infinity or a NaN is
    held as NaN."""
    KernelError, _check, _code, _i32, _need_gpu, _ptr, _stream = _base()
    _need_gpu(k, v, q, positions, inv_freq, cache, block_table, seq_of_token)
    _check_device(k, v, q, positions, inv_freq, cache, block_table, seq_of_token)
    if k.dim() != 3:
        raise KernelError("k must be [T, Hkv, hd] with contiguous heads")
    n_tokens, n_kv, hd = k.shape
    for name, t in (("k", k), ("v", v), ("q", q)):
        if t is None:
            continue
        if t.dim() != 3 or t.shape[0] != n_tokens or t.shape[2] != hd or t.stride(2) != 1 or t.stride(1) != hd or (name == "v" and t.shape[1] != n_kv):
            raise KernelError(f"{name} must be [T, {'Hq' if name == 'q' else 'Hkv'}, hd] with contiguous heads")
        if t.dtype != k.dtype:
            raise KernelError("q, k and v must have one type")
    code = _code(k.dtype)
    page_size = _check_cache(cache, block_table, n_kv, hd, bits)
    _i32(positions, "positions")
    _i32(seq_of_token, "seq_of_token")
    if positions.numel() != n_tokens or seq_of_token.numel() != n_tokens:
        raise KernelError("positions and seq_of_token must be [T]")
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or inv_freq.numel() != hd // 2 or not inv_freq.is_contiguous()):
        raise KernelError(f"the rotary table must be float32 [{hd // 2}]")
    if q is not None and n_tokens > 1 and q.stride(0) < q.shape[1] * hd:
        raise KernelError("q is rotated in place: its rows must not overlap")
    lib = _build.load("quant_cache")
    _check(
        lib,
        lib.cwm_quant_kv_write(
            _ptr(k), ctypes.c_long(k.stride(0)), _ptr(v), ctypes.c_long(v.stride(0)), _ptr(q), ctypes.c_long(q.stride(0) if q is not None else 0),
            code, _ptr(positions), _ptr(seq_of_token), _ptr(inv_freq), _ptr(cache), _ptr(block_table),
            block_table.shape[0], block_table.shape[1], page_size, cache.shape[0], n_tokens, n_kv, q.shape[1] if q is not None else 0, hd, bits,
            _stream(),
        ),
    )


def quant_kv_read(
    cache: torch.Tensor,
    block_table: torch.Tensor,
    positions: torch.Tensor,
    seq_of_token: torch.Tensor,
    head_dim: int,
    bits: int,
    dtype: torch.dtype,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values, each [T, Hkv, head_dim] of `dtype` (float32 or bfloat16), that a quantised `cache` holds of the
    tokens at `positions` [T] of the sequences `seq_of_token` [T] (rows of the block table); zeros where no page is held."""
    KernelError, _check, _code, _i32, _need_gpu, _ptr, _stream = _base()
    _need_gpu(cache, block_table, positions, seq_of_token)
    _check_device(cache, block_table, positions, seq_of_token)
    page_size = _check_cache(cache, block_table, None, head_dim, bits)
    _i32(positions, "positions")
    _i32(seq_of_token, "seq_of_token")
    n_tokens = positions.numel()
    if seq_of_token.numel() != n_tokens:
        raise KernelError("positions and seq_of_token must be [T]")
    code = _code(dtype)
    k = torch.empty((n_tokens, cache.shape[1], head_dim), dtype=dtype, device=cache.device)
    v = torch.empty_like(k)
    lib = _build.load("quant_cache")
    _check(
        lib,
        lib.cwm_quant_kv_read(
            _ptr(k), _ptr(v), code, _ptr(positions), _ptr(seq_of_token), _ptr(cache), _ptr(block_table), block_table.shape[0],
            block_table.shape[1], page_size, cache.shape[0], n_tokens, cache.shape[1], head_dim, bits, _stream(),
        ),
    )
    return k, v


def quant_paged_attention(
    q: torch.Tensor,
    cache: torch.Tensor,
    block_table: torch.Tensor,
    batch,
    window: Optional[int],
    scale: float,
    bits: int,
) -> torch.Tensor:
    """Attention of the step's tokens over a quantised cache (`quant_kv_write`), prompt portions and decoded tokens in one
    call: `q` [T, Hq, hd] (float32 or bfloat16, rotated), `batch` the step's `StepBatch`, `window` the keys a query reads, its
    own included (None: all).  Returns [T, Hq * hd] in q's type.  A query one of whose keys has no page gets NaN."""
    KernelError, _check, _code, _i32, _need_gpu, _ptr, _stream = _base()
    from . import _attention_plan, _check_mask

    _need_gpu(q, cache, block_table)
    _check_device(q, cache, block_table, batch.cu_q, batch.kv_len)
    _check_mask(window, None, None)
    if q.dim() != 3 or q.stride(2) != 1 or q.stride(1) != q.shape[2]:
        raise KernelError("q must be [T, Hq, hd] with contiguous heads")
    n_tokens, n_q, hd = q.shape
    page_size = _check_cache(cache, block_table, None, hd, bits)
    n_kv = cache.shape[1]
    if n_q % n_kv != 0 or n_q == 0:
        raise KernelError(f"{n_q} query heads do not divide into {n_kv} key/value heads")
    code = _code(q.dtype)
    if not scale > 0:
        raise KernelError("the scale of the scores must be positive")
    if block_table.shape[0] != batch.n_seqs or n_tokens != batch.n_tokens:
        raise KernelError("block_table must be [B, W] for the batch's sequences, q [T, ...] for its tokens")
    if (n_tokens > 1 and q.stride(0) % (16 // q.element_size()) != 0) or q.data_ptr() % 16 != 0:
        raise KernelError("q rows must be 16-byte aligned")
    out = torch.empty((n_tokens, n_q * hd), dtype=q.dtype, device=q.device)
    if n_tokens == 0:
        return out
    plan = _attention_plan(batch, n_q // n_kv, n_kv, hd, window, q.device)
    partial = None
    if plan.n_partials:
        partial = torch.empty(plan.n_partials * n_kv * 16 * (hd + 4), dtype=torch.float32, device=q.device)
    lib = _build.load("attention_quant", {"HEAD_DIM": hd})
    _check(
        lib,
        lib.cwm_attention_quant(
            _ptr(q), ctypes.c_long(q.stride(0) if n_tokens > 1 else n_q * hd), code, _ptr(out), ctypes.c_long(n_q * hd), _ptr(cache), _ptr(block_table), block_table.shape[1],
            _ptr(batch.cu_q), _ptr(batch.kv_len), _ptr(plan.work), plan.n_work, _ptr(plan.wide), plan.n_wide, plan.item_tiles,
            _ptr(plan.merge), plan.n_merge, _ptr(partial), n_q, n_kv, hd, page_size, cache.shape[0],
            -1 if window is None else window - 1, ctypes.c_float(scale), bits, _stream(),
        ),
    )
    return out


# --------------------------------------------------------------------------- #
INT8_MAX_K = 131072  # csrc/gemm_int8.hip: 127^2 K fits the 32 bits of a sum
INT8_FEW_ROWS = 64
_INT8_TILES = {1: (256, 128), 2: (128, 256), 3: (64, 128), 4: (128, 128)}


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """`x` [M, K] (float32 or bfloat16) as int8 [M, K] and a float32 scale a row [M]: the scale is the row's largest magnitude over
    127, the integers x / scale rounded, ties to even.  A row of zeros has a scale of 0; one with an infinity or a NaN has a NaN
    for its scale.  The integers are a view of rows padded with zeros to a multiple of 128, which `linear_int8` likes best for
    its weights."""
    KernelError, _check, _code, _i32, _need_gpu, _ptr, _stream = _base()
    _need_gpu(x)
    _check_device(x)
    if x.dim() != 2 or x.shape[1] < 1 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise KernelError("rows to quantise must be [M, K] with contiguous rows")
    code = _code(x.dtype)
    m, k = x.shape
    padded = -(-k // 128) * 128
    codes = torch.empty((m, padded), dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    lib = _build.load("gemm_int8")
    _check(lib, lib.cwm_quantize_rows(_ptr(x), ctypes.c_long(x.stride(0)), code, _ptr(codes), ctypes.c_long(padded), _ptr(scale), m, k, padded, _stream()))
    return codes[:, :k], scale


def int8_limits(n: int, k: int) -> Optional[str]:
    """Why a weight [n, k] cannot be one of `linear_int8`, or None if it can."""
    if n < 1 or k < 1 or k % 16 != 0 or k > INT8_MAX_K:
        return f"the product of 8-bit integers takes rows of a multiple of 16 columns up to {INT8_MAX_K}, not {k}"
    return None


def linear_int8(
    x: torch.Tensor,
    weight: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
    tile: Optional[int] = None,
) -> torch.Tensor:
    """y = x W^T (+ bias) in 8-bit integers: the rows of `x` [M, K] (float32 or bfloat16) are quantised as by `quantize_rows`,
    multiplied with the int8 `weight` [N, K] with exact 32-bit sums, and scaled by the rows' scales and the float32
    `weight_scale` [N] (`quantize_rows` of the weight); `bias` float32 [N].  K a multiple of 16, rows of the weight 16-byte
    aligned.  Returns [M, N] in `out_dtype` (default: x's).  `tile` (tests) names one of the kernels."""
    KernelError, _check, _code, _i32, _need_gpu, _ptr, _stream = _base()
    from . import _compute_units

    _need_gpu(x, weight, weight_scale, bias)
    _check_device(x, weight, weight_scale, bias)
    if x.dim() != 2 or weight.dim() != 2 or x.shape[1] != weight.shape[1]:
        raise KernelError(f"linear_int8: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not fit")
    m, k = x.shape
    n = weight.shape[0]
    why = int8_limits(n, k)
    if why is not None:
        raise KernelError(why)
    if weight.dtype != torch.int8 or weight.stride(1) != 1 or weight.data_ptr() % 16 != 0 or (n > 1 and (weight.stride(0) % 16 != 0 or weight.stride(0) < k)):
        raise KernelError(f"the weight must be int8 with 16-byte aligned rows, found {weight.dtype} with strides {weight.stride()}")
    if weight_scale.dtype != torch.float32 or weight_scale.shape != (n,) or not weight_scale.is_contiguous():
        raise KernelError(f"the weight's scales must be a contiguous float32 [{n}] tensor")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous()):
        raise KernelError(f"linear_int8: the bias must be a contiguous float32 [{n}] tensor")
    y = torch.empty((m, n), dtype=out_dtype or x.dtype, device=x.device)
    code = _code(y.dtype)
    if m == 0:
        _code(x.dtype)
        return y
    codes, scale = quantize_rows(x)
    if tile is None:
        tile = _int8_tile(m, n, k)
    lib = _build.load("gemm_int8")
    _check(
        lib,
        lib.cwm_gemm_int8(
            _ptr(codes), ctypes.c_long(codes.stride(0)), _ptr(scale), _ptr(weight), ctypes.c_long(weight.stride(0) if n > 1 else max(k, weight.stride(0))),
            _ptr(weight_scale), _ptr(bias), _ptr(y), code, ctypes.c_long(n), m, n, k, _compute_units(x.device), tile, _stream(),
        ),
    )
    return y


def _int8_tile(m: int, n: int, k: int) -> int:
    """The kernel for a product's sizes."""
    if m <= INT8_FEW_ROWS or k % 128 != 0:
        return 0
    return 1
