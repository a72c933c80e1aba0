"""Entry points of the kernels that serve in fewer bits: the paged cache of keys and values in 4 or 8 bits
(`csrc/quant_cache.hip`, `csrc/attention_quant.hip`; layout and formulas in `csrc/quant_cache.h`), and the product of 8-bit
integers with a scale for every token and output channel (`csrc/gemm_int8.hip`).  Shapes, types and devices are checked on the
host; there is no CPU path."""

from __future__ import annotations

import ctypes
import dataclasses
import functools
from typing import List, Optional, Tuple

import numpy as np
import torch

from . import build as _build

CACHE_BITS = (4, 8)
QUANT_MAX_DIM = 256  # csrc/quant_cache.h

_P, _L, _I, _F = ctypes.c_void_p, ctypes.c_long, ctypes.c_int, ctypes.c_float
# The C entry points with their arguments' types, by name and the switches of a build that change them: with these ctypes converts
# plain numbers by itself, which for twenty arguments is 3 us less a call than objects made one by one.
_ARGTYPES = {
    "cwm_quant_kv_write": (_P, _L, _P, _L, _P, _L, _I, _P, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P),
    "cwm_quant_kv_read": (_P, _P, _I, _P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _P),
    "cwm_attention_quant": (_P, _L, _I, _P, _L, _P, _P, _I, _P, _P, _P, _I, _P, _I, _I, _P, _I, _P, _I, _I, _I, _I, _I, _I, _F, _I, _P),
    "cwm_quant_unpack": (_P, _P, _I, _P, _I, _P, _P, _I, _I, _I, _P, _I, _I, _I, _P),
    ("cwm_attention_mfma", "HALF_INPUTS"): (
        _P, _L, _P, _L, _P, _P, _I, _P, _P, _P, _I, _I, _P, _I, _I, _I, _P, _I, _I, _I, _P, _I, _I, _I, _I, _I, _I, _I, _F, _F, _P, _P, _P, _P, _I, _P, _P,
    ),
    "cwm_quantize_rows": (_P, _L, _I, _P, _L, _P, _I, _I, _I, _P),
    "cwm_linear_int8": (_P, _L, _I, _P, _P, _P, _L, _P, _P, _P, _I, _L, _I, _I, _I, _I, _I, _I, _P, _P),
}
_entries: dict = {}


def _entry(library: str, name: str, head_dim: Optional[int] = None, *switches: str):
    """The entry point `name` of a library built for a head size with the named switches, and the library (for its error message)."""
    found = _entries.get((library, name, head_dim, switches))
    if found is None:
        lib = _build.load(library, None if head_dim is None else {"HEAD_DIM": head_dim, **dict.fromkeys(switches, 1)})
        function = lib[name]  # an object of its own: other callers of the library hand in objects of ctypes
        function.argtypes = _ARGTYPES[(name, *switches) if switches else name]
        found = _entries[(library, name, head_dim, switches)] = (function, lib)
    return found


@functools.cache  # an import statement costs a launch-bound step a microsecond and more a call
def _base():
    from . import KernelError, _check, _code  # the shared helpers of this package

    return KernelError, _check, _code


@functools.cache
def _planning():
    from . import _attention_plan, _check_mask, _half_blocks_built, _three_blocks_a_unit

    return _attention_plan, _check_mask, _half_blocks_built, _three_blocks_a_unit


@functools.cache
def _units(device: torch.device) -> int:
    from . import _compute_units

    return _compute_units(device)


# looked up once: the attributes of `torch` and `torch._C` cost a launch-bound call half a microsecond
_INT32, _FLOAT32, _UINT8 = torch.int32, torch.float32, torch.uint8
_current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _check_device(first: torch.Tensor, *tensors: Optional[torch.Tensor]) -> int:
    """That all are on one HIP device, and that the current one: kernels are launched on its stream.  Returns that stream's handle."""
    current = _current_device() if first.is_cuda else None
    if current is not None and first.get_device() == current:
        for t in tensors:
            if t is not None and t.get_device() != current:
                break
        else:
            return _current_stream(current)
    KernelError = _base()[0]
    for t in (first, *tensors):
        if t is not None and not t.is_cuda:
            raise KernelError(f"cwm_amd kernels run on a HIP device only; got a tensor on {t.device}. There is no CPU path.")
    raise KernelError(f"tensors are on {', '.join(sorted({str(t.device) for t in (first, *tensors) if t is not None}))}, the current device is cuda:{current}")


def _check_vector(t: torch.Tensor, n: int, what: str) -> None:
    if t.dtype is not _INT32 or t.numel() != n or not t.is_contiguous():
        raise _base()[0](f"{what} must be a contiguous int32 [T] tensor for {n} tokens, found {t.dtype} {tuple(t.shape)} with strides {t.stride()}")


def _token_bytes(head_dim: int, bits: int) -> int:
    """Bytes of one token of one key/value head: codes of key and value, a word for every 32 elements of the key, one for the value."""
    return 2 * (head_dim * bits // 8) + head_dim // 32 * 4 + 4


@functools.lru_cache(maxsize=1024)
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


@functools.lru_cache(maxsize=1024)
def _page_size(shape: Tuple[int, ...], n_kv: Optional[int], head_dim: int, bits: int) -> Tuple[int, Optional[str]]:
    """Tokens of a page of a cache of this shape, and why it is none."""
    why = quant_cache_limits(head_dim, 8, bits)
    if why is not None:
        return 0, why
    token = _token_bytes(head_dim, bits)
    if len(shape) != 3 or min(shape) < 1 or (n_kv is not None and shape[1] != n_kv) or shape[2] % token != 0:
        return 0, f"cache {tuple(shape)} does not fit {n_kv or 'any'} heads of size {head_dim} in {bits} bits"
    return shape[2] // token, quant_cache_limits(head_dim, shape[2] // token, bits)


def _check_cache(cache: torch.Tensor, block_table: torch.Tensor, n_kv: Optional[int], head_dim: int, bits: int) -> int:
    """The tokens of a page of `cache`, a contiguous uint8 [pages, key/value heads, head bytes]."""
    page_size, why = _page_size(cache.shape, n_kv, head_dim, bits)
    if why is None and (cache.dtype is not _UINT8 or not cache.is_contiguous()):
        why = f"the cache does not fit: it is contiguous and of bytes (uint8), found {cache.dtype} with strides {cache.stride()}"
    if why is None and (block_table.dtype is not _INT32 or block_table.dim() != 2 or block_table.shape[1] < 1 or not block_table.is_contiguous()):
        why = f"block_table must be a contiguous int32 [B, W] tensor, found {block_table.dtype} {tuple(block_table.shape)}"
    if why is not None:
        raise _base()[0](why)
    return page_size


def _bad_heads(name: str, t: torch.Tensor, n_tokens: int, heads: Optional[int], hd: int, dtype: torch.dtype) -> None:
    """Raise what is wrong with queries, keys or values that are not [T, heads, hd] of `dtype` with contiguous heads."""
    KernelError = _base()[0]
    if t.dim() == 3 and t.shape[0] == n_tokens and t.shape[2] == hd and (heads is None or t.shape[1] == heads) and t.dtype != dtype:
        raise KernelError("q, k and v must have one type")
    raise KernelError(f"{name} must be [T, {'Hq' if name == 'q' else 'Hkv'}, hd] with contiguous heads, found {tuple(t.shape)} with strides {t.stride()}")


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
    KernelError, _check, _code = _base()
    stream = _check_device(k, v, q, positions, inv_freq, cache, block_table, seq_of_token)
    if k.dim() != 3:
        raise KernelError("k must be [T, Hkv, hd] with contiguous heads")
    dtype = k.dtype
    n_tokens, n_kv, hd = shape = k.shape
    k_token, k_head, k_one = k.stride()
    if k_one != 1 or k_head != hd:
        _bad_heads("k", k, n_tokens, n_kv, hd, dtype)
    if v.shape != shape or v.dtype != dtype or v.stride()[1:] != (hd, 1):
        _bad_heads("v", v, n_tokens, n_kv, hd, dtype)
    n_q = q_token = 0
    if q is not None:
        if q.dim() != 3 or q.shape[0] != n_tokens or q.shape[2] != hd or q.dtype != dtype or q.stride()[1:] != (hd, 1):
            _bad_heads("q", q, n_tokens, None, hd, dtype)
        n_q, q_token = q.shape[1], q.stride(0)
        if n_tokens > 1 and q_token < n_q * hd:
            raise KernelError("q is rotated in place: its rows must not overlap")
    code = _code(dtype)
    page_size = _check_cache(cache, block_table, n_kv, hd, bits)
    _check_vector(positions, n_tokens, "positions")
    _check_vector(seq_of_token, n_tokens, "seq_of_token")
    if inv_freq is not None and (inv_freq.dtype is not _FLOAT32 or inv_freq.numel() != hd // 2 or not inv_freq.is_contiguous()):
        raise KernelError(f"the rotary table must be float32 [{hd // 2}]")
    function, lib = _entry("quant_cache", "cwm_quant_kv_write")
    n_seqs, width = block_table.shape
    status = function(
        k.data_ptr(), k_token, v.data_ptr(), v.stride(0), None if q is None else q.data_ptr(), q_token, code, positions.data_ptr(),
        seq_of_token.data_ptr(), None if inv_freq is None else inv_freq.data_ptr(), cache.data_ptr(), block_table.data_ptr(), n_seqs, width, page_size,
        cache.shape[0], n_tokens, n_kv, n_q, hd, bits, stream,
    )
    if status:
        _check(lib, status)


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
    _, _check, _code = _base()
    stream = _check_device(cache, block_table, positions, seq_of_token)
    page_size = _check_cache(cache, block_table, None, head_dim, bits)
    n_tokens = positions.numel()
    _check_vector(positions, n_tokens, "positions")
    _check_vector(seq_of_token, n_tokens, "seq_of_token")
    code = _code(dtype)
    pages, n_kv, _ = cache.shape
    both = torch.empty((2, n_tokens, n_kv, head_dim), dtype=dtype, device=cache.device)
    k, v = both.unbind(0)
    function, lib = _entry("quant_cache", "cwm_quant_kv_read")
    n_seqs, width = block_table.shape
    status = function(
        k.data_ptr(), v.data_ptr(), code, positions.data_ptr(), seq_of_token.data_ptr(), cache.data_ptr(), block_table.data_ptr(), n_seqs, width,
        page_size, pages, n_tokens, n_kv, head_dim, bits, stream,
    )
    if status:
        _check(lib, status)
    return k, v


UNPACK_KEYS = 64  # csrc/quant_cache.hip
UNPACK_PAGE = 256  # tokens of a page of the unpacked cache
# Bytes of unpacked keys and values and of partial results that the portions of a step take at a time: the sequences of a step take turns,
# one at least in a turn.  One of 131,072 keys and 8 heads of 128 has 512 MiB of keys and values, read in 5 ms: what two more launches cost is nothing.
UNPACK_BYTES = 1 << 29


def _portion_bytes(n_kv: int, head_dim: int, n_keys: int, n_slots: int) -> int:
    """Bytes of the unpacked keys and values of a sequence of which portions read `n_keys`, and of `n_slots` partial results of a row tile."""
    pages = -(-n_keys // UNPACK_PAGE) + 1  # a window need not begin with a page
    return n_kv * (pages * (UNPACK_PAGE * head_dim * 4 + UNPACK_PAGE // 32 * 8) + n_slots * 16 * (head_dim + 4) * 4)


def quant_attention_workspace(n_kv: int, head_dim: int, n_keys: int, units: int) -> int:
    """The most bytes that `quant_paged_attention` takes for the portions of a step whose sequences hold up to `n_keys` keys, on `units`
    compute units (bfloat16)."""
    from .attention_plan import PACKED_WIDE_BLOCKS, WIDE_TILES

    cut_below = -(-2 * units // n_kv)  # a sequence is cut if it has fewer blocks of WIDE_TILES row tiles, see `wide_chunk`
    return max(UNPACK_BYTES, _portion_bytes(n_kv, head_dim, n_keys, (PACKED_WIDE_BLOCKS + 1) * cut_below * WIDE_TILES))


def _turns(batch, group: int, window: Optional[int], n_kv: int, head_dim: int, device: torch.device) -> list:
    """Pieces of the step that have some of its portions each, and the others as if they had no new tokens, where all of them would unpack
    more than UNPACK_BYTES; none where they may go together.  Made once a step.  A row's result does not depend on what else is in its piece."""
    key = ("quant_turns", group, window, n_kv, head_dim)
    turns = batch.scratch.get(key)
    if turns is None:
        from .attention_plan import ROWS_PER_TILE, SPLIT_MAX_TILES, WIDE_TILES, first_keys, wide_chunk

        cut_below = -(-2 * _units(device) // n_kv)
        pieces: List[List[int]] = []
        room = 0
        for b, (m, n) in enumerate(zip(batch.q_lens, batch.kv_lens)):
            tiles = -(-m * group // ROWS_PER_TILE)
            if tiles <= SPLIT_MAX_TILES:
                continue
            n_wide = -(-tiles // WIDE_TILES)
            cut = wide_chunk(n_wide, m, n, window, cut_below, True)
            first = int(first_keys(n - m, window, None))
            chunks = (n - 1) // cut - first // cut + 1 if cut else 1  # at most, of a block
            needs = _portion_bytes(n_kv, head_dim, n - first, tiles * chunks if chunks > 1 else 0)
            if not pieces or needs > room:
                pieces.append([])
                room = UNPACK_BYTES
            pieces[-1].append(b)
            room -= needs
        turns = []
        if len(pieces) > 1:
            many = {b for piece in pieces for b in piece}
            for i, piece in enumerate(pieces):
                mine = set(piece) if i else set(piece) | set(range(len(batch.q_lens))) - many  # the first has the decoded tokens
                turns.append(dataclasses.replace(batch, q_lens=[m if b in mine else 0 for b, m in enumerate(batch.q_lens)], scratch={}))
        batch.scratch[key] = turns
    return turns


def _unpack_list(batch, group: int, window: Optional[int], device: torch.device):
    """The work of unpacking the sequences of a step that have blocks of many rows: the list of `cwm_quant_unpack` and the block table of
    the unpacked cache in one device vector, the items, the table's width and the pages; made once a step."""
    key = ("quant_unpack", group, window)
    held = batch.scratch.get(key)
    if held is None:
        from .attention_plan import ROWS_PER_TILE, SPLIT_MAX_TILES, first_keys

        width = max(-(-n // UNPACK_PAGE) for n in batch.kv_lens)
        table = np.full((len(batch.kv_lens), width), -1, dtype=np.int32)
        items, pages = [], 0
        for b, (m, n) in enumerate(zip(batch.q_lens, batch.kv_lens)):
            if -(-m * group // ROWS_PER_TILE) <= SPLIT_MAX_TILES:
                continue
            first = int(first_keys(n - m, window, None))
            lo = first // UNPACK_PAGE
            count = -(-n // UNPACK_PAGE) - lo
            table[b, lo : lo + count] = np.arange(pages, pages + count)
            keys = np.arange(first // UNPACK_KEYS * UNPACK_KEYS, n, UNPACK_KEYS)
            items.append(np.stack([np.full_like(keys, b), keys, pages + keys // UNPACK_PAGE - lo, np.full_like(keys, first)], axis=1))
            pages += count
        rows = np.concatenate(items).astype(np.int32)
        host = torch.from_numpy(np.concatenate([rows.reshape(-1), table.reshape(-1)]))
        dev = host.pin_memory().to(device, non_blocking=True)
        held = batch.scratch[key] = (dev, rows.shape[0], width, pages)
    return held


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
    own included (None: all).  Returns [T, Hq * hd] in q's type.  A query one of whose keys has no page gets NaN.
    bfloat16 portions of more than 128 rows (tokens times query heads of a key/value head) unpack what they read of the cache to 16 bits for
    the time of the call: 4 Hkv hd bytes a key, for as many sequences at a time as 512 MiB hold, and for one at least
    (`quant_attention_workspace`)."""
    KernelError, _check, _code = _base()
    _attention_plan, _check_mask, _half_blocks_built, _three_blocks_a_unit = _planning()
    stream = _check_device(q, cache, block_table, batch.cu_q, batch.kv_len)
    _check_mask(window, None, None)
    if q.dim() != 3 or q.stride(2) != 1 or q.stride(1) != q.shape[2]:
        raise KernelError("q must be [T, Hq, hd] with contiguous heads")
    n_tokens, n_q, hd = q.shape
    page_size = _check_cache(cache, block_table, None, hd, bits)
    pages, n_kv, _ = cache.shape
    if n_q % n_kv != 0 or n_q == 0:
        raise KernelError(f"{n_q} query heads do not divide into {n_kv} key/value heads")
    dtype = q.dtype
    code = _code(dtype)
    if not scale > 0:
        raise KernelError("the scale of the scores must be positive")
    if block_table.shape[0] != batch.n_seqs or n_tokens != batch.n_tokens:
        raise KernelError("block_table must be [B, W] for the batch's sequences, q [T, ...] for its tokens")
    token = q.stride(0) if n_tokens > 1 else n_q * hd
    if token % (4 if dtype == torch.float32 else 8) != 0 or q.data_ptr() % 16 != 0:
        raise KernelError("q rows must be 16-byte aligned")
    out = torch.empty((n_tokens, n_q * hd), dtype=dtype, device=q.device)
    if n_tokens == 0:
        return out
    group = n_q // n_kv
    # bfloat16 queries of many rows: their keys and values are unpacked once, to float16, and read by the attention over a cache of 16 bits
    halves = dtype == torch.bfloat16 and _half_blocks_built(n_kv, hd, UNPACK_PAGE)
    plan = _attention_plan(batch, group, n_kv, hd, window, q.device, None, halves, packed=True)
    unpacks = plan.n_wide > 0 and dtype == torch.bfloat16
    pieces = unpacks and _turns(batch, group, window, n_kv, hd, q.device)
    for piece in pieces or (batch,):
        if pieces:
            plan = _attention_plan(piece, group, n_kv, hd, window, q.device, None, halves, packed=True)
        partials = partial = unpacked = None  # a piece's memory is free for the next one
        if plan.n_partials:
            partials = torch.empty(plan.n_partials * n_kv * 16 * (hd + 4), dtype=torch.float32, device=q.device)  # held until the last launch
            partial = partials.data_ptr()
        table, width = block_table.data_ptr(), block_table.shape[1]
        first, lengths, work, wide, merge = batch.cu_q.data_ptr(), batch.kv_len.data_ptr(), plan.work.data_ptr(), plan.wide.data_ptr(), plan.merge.data_ptr()
        if plan.n_work or not unpacks:
            function, lib = _entry("attention_quant", "cwm_attention_quant", hd)
            status = function(
                q.data_ptr(), token, code, out.data_ptr(), n_q * hd, cache.data_ptr(), table, width, first, lengths, work, plan.n_work, wide,
                0 if unpacks else plan.n_wide, plan.item_tiles, merge, 0 if unpacks else plan.n_merge, partial, n_q, n_kv, hd, page_size, pages,
                -1 if window is None else window - 1, scale, bits, stream,
            )
            if status:
                _check(lib, status)
        if unpacks:
            listed, n_items, wide_width, n_pages = _unpack_list(piece, group, window, q.device)
            held = n_pages * 2 * n_kv * UNPACK_PAGE * hd * 2  # bytes; behind them two exponents for every 32 keys of a head
            unpacked = torch.empty(held + n_pages * n_kv * (UNPACK_PAGE // 32) * 8, dtype=torch.uint8, device=q.device)
            exponents = unpacked.data_ptr() + held
            function, lib = _entry("quant_cache", "cwm_quant_unpack")
            status = function(
                unpacked.data_ptr(), exponents, UNPACK_PAGE, listed.data_ptr(), n_items, cache.data_ptr(), table, width, page_size, pages, lengths, n_kv, hd, bits, stream,
            )
            if status:
                _check(lib, status)
            function, lib = _entry("attention_mfma", "cwm_attention_mfma", hd, "HALF_INPUTS")
            status = function(
                q.data_ptr(), token, out.data_ptr(), n_q * hd, unpacked.data_ptr(), listed.data_ptr() + 16 * n_items, wide_width, first, lengths,
                work, 0, 0, wide, plan.n_wide, plan.item_tiles, _three_blocks_a_unit(plan.n_wide * n_kv, plan.wide_shape, q.device),
                merge, plan.n_merge, plan.n_merge_mid, plan.n_merge_wide, partial, n_q, n_kv, hd, UNPACK_PAGE, n_pages,
                -1 if window is None else window - 1, 0, scale, 0.0, None, None, None, None, 0, exponents, stream,
            )
            if status:
                _check(lib, status)
    return out


# --------------------------------------------------------------------------- #
INT8_MAX_K = 131072  # csrc/gemm_int8.hip: 127^2 K fits the 32 bits of a sum
INT8_FEW_ROWS, INT8_FEW_WEIGHTS = 16, 50_400_000
INT8_FUSED_ROWS, INT8_FUSED_K = 4, 16384  # csrc/gemm_int8.hip: rows of x, and the columns of one row, that every block makes the integers of


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """`x` [M, K] (float32 or bfloat16) as int8 [M, K] and a float32 scale a row [M]: the scale is the row's largest magnitude over
    127, the integers x / scale rounded, ties to even, and limited to -127 .. 127 (which tells in rows below 2.3e-41, whose scale
    is a few of float32's smallest steps).  A row of zeros has a scale of 0; one with an infinity or a NaN has a NaN for its scale.
    The integers are a view of rows padded with zeros to a multiple of 128, which `linear_int8` likes best for its weights."""
    KernelError, _check, _code = _base()
    stream = _check_device(x)
    if x.dim() != 2 or x.shape[1] < 1 or (x.shape[1] > 1 and x.stride(1) != 1):
        raise KernelError("rows to quantise must be [M, K] with contiguous rows")
    code = _code(x.dtype)
    m, k = x.shape
    padded = -(-k // 128) * 128
    codes = torch.empty((m, padded), dtype=torch.int8, device=x.device)
    scale = torch.empty(m, dtype=torch.float32, device=x.device)
    function, lib = _entry("gemm_int8", "cwm_quantize_rows")
    status = function(x.data_ptr(), x.stride(0), code, codes.data_ptr(), padded, scale.data_ptr(), m, k, padded, stream)
    if status:
        _check(lib, status)
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
    parts: int = 1,
) -> torch.Tensor:
    """y = x W^T (+ bias) in 8-bit integers: the rows of `x` [M, K] (float32 or bfloat16) are quantised as by `quantize_rows`,
    multiplied with the int8 `weight` [N, K] with exact 32-bit sums, and scaled by the rows' scales and the float32
    `weight_scale` [N] (`quantize_rows` of the weight); `bias` float32 [N].  K a multiple of 16, rows of the weight 16-byte
    aligned.  Returns [M, N] in `out_dtype` (default: x's).  `tile` (tests) names one of the kernels and
    `parts` in how many pieces it takes K."""
    KernelError, _check, _code = _base()
    stream = _check_device(x, weight, weight_scale, bias)
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
    if k > 1 and x.stride(1) != 1:
        raise KernelError("linear_int8: x must have contiguous rows")
    x_code = _code(x.dtype)
    y = torch.empty((m, n), dtype=out_dtype or x.dtype, device=x.device)
    code = _code(y.dtype)
    if m == 0:
        return y
    if tile is None:
        tile, parts = _int8_tile(m, n, k, _units(x.device))
    codes = scale = sums = joined = None
    if tile >= 0:
        padded = -(-k // 128) * 128
        room = torch.empty(m * (padded + 4), dtype=torch.uint8, device=x.device)  # the integers of x, then their scales
        codes = room.data_ptr()
        scale = codes + m * padded
    if parts > 1:
        sums = torch.empty((parts, m, -(-n // 128) * 128), dtype=torch.int32, device=x.device)  # held until the last launch
        joined = sums.data_ptr()
    function, lib = _entry("gemm_int8", "cwm_linear_int8")
    status = function(
        x.data_ptr(), x.stride(0), x_code, codes, scale, weight.data_ptr(), weight.stride(0) if n > 1 else k,
        weight_scale.data_ptr(), None if bias is None else bias.data_ptr(), y.data_ptr(), code, n, m, n, k, _units(x.device), tile, parts, joined, stream,
    )
    if status:
        _check(lib, status)
    return y


# The tiles of many rows (number of the kernel's, rows, columns), and what each costs: us a round of tiles, and a step of 128 columns of K
# of a round.  Fitted to 2,048 x 43,008 with a K of 1,536, 3,200 and 6,144 (tiles of 256 x 128: 161, 281 and 509 us, 128 x 256 162, 290 and
# 495, 64 x 128 259, 465 and 820, 128 x 128 199, 346 and 590).
_INT8_TILES = ((1, 256, 128, 2.9, 0.98), (2, 128, 256, 5.6, 0.85), (3, 64, 128, 1.6, 0.38), (4, 128, 128, 3.2, 0.52))


_INT8_PARTS_US, _INT8_PARTS_BYTES = 5.0, 4e6  # of joining the parts of K: a launch, and the bytes of their sums a us


@functools.lru_cache(maxsize=1024)
def _int8_tile(m: int, n: int, k: int, units: int) -> Tuple[int, int]:
    """The kernel for a product's sizes, and the parts it takes K in.  Up to four rows one launch does all, while W is not so large that
    the tiles' loads, further ahead, are the faster ones (us in one launch, in two and by tiles: 1 x 6,144 x 6,144 12.5, 16.2, 19.6; 1 x
    10,240 x 8,192 21.0, 26.2, 23.4; 1 x 28,672 x 4,096 26.2, 31.7, 24.3; 1 x 43,008 x 6,144 58, 65, 48); up to 16 rows W is read straight
    into the matrix instruction, with half that limit (8 x 6,144 x 8,192 19.3, by tiles 20.1; 16 x 14,336 x 4,096 23.7 and 20.5; 8 x 28,672 x
    2,048 22.4 and 16.4).  More rows take the tile of least cost, and where its tiles are fewer than the compute units, K in parts (33 x
    6,144 x 6,144 29.3, in five parts 21.2; 64 x 4,096 x 14,336 64.0 and, in eight, 31.7; 64 x 8,192 x 1,024 15.3 and, in two, 20.3,
    which stays whole)."""
    if m <= INT8_FUSED_ROWS and k <= INT8_FUSED_K // (m if m <= 2 else 4) and n * k < 2 * INT8_FEW_WEIGHTS:
        return -1, 1
    if k < 128 or (m <= INT8_FEW_ROWS and n * k < INT8_FEW_WEIGHTS):
        return 0, 1
    steps, best = -(-k // 128), None
    for tile, rows, columns, start, step in _INT8_TILES:
        tiles = -(-m // rows) * -(-n // columns)
        for parts in range(1, max(1, min(units // tiles, steps)) + 1 if tile in (3, 4) else 2):
            cost = -(-tiles * parts // units) * (start + -(-steps // parts) * step)
            if parts > 1:
                cost += _INT8_PARTS_US + 8 * parts * m * n / _INT8_PARTS_BYTES
            if best is None or cost < best[0]:
                best = (cost, tile, parts)
    return best[1:]
