"""Work lists of steps whose cache holds 4 or 8 bits: chunks of their own, every key of every row once, homes of captured steps."""

import numpy as np
import pytest

from cwm_amd.ops.attention_plan import (
    PACKED_WIDE_BLOCKS, PACKED_WIDE_CHUNK, WIDE_TILES, build_plan, capacity_until, chunk_keys, pad_plan, wide_chunk, wide_chunks, wide_item_tiles,
)


def test_chunks():
    assert [int(chunk_keys(n, False, True)) for n in (1, 2048, 2049, 8192, 8193, 65537, 10 ** 6)] == [2048, 2048, 1024, 1024, 2048, 2048, 2048]
    assert [int(chunk_keys(n)) for n in (2048, 2049, 8193, 65537)] == [2048, 512, 1024, 2048]
    assert wide_chunks(True) == (PACKED_WIDE_CHUNK, PACKED_WIDE_CHUNK) and wide_chunks(False) == (8192, 2048)


@pytest.mark.parametrize("q,kv,group,window", [([1], [9000], 6, None), ([1, 30, 300], [5000, 30, 4000], 4, None), ([1, 200], [70000, 3000], 8, 2500)])
def test_every_key_of_a_tile_is_in_one_item(q, kv, group, window):
    plan = build_plan(q, kv, group, window, 64, packed=True)
    for items, tiles in ((plan.work, 1), (plan.work_wide, 8)):
        for b, row0 in {(int(w[0]), int(w[1])) for w in items}:
            parts = sorted((int(w[2]), int(w[3])) for w in items if w[0] == b and w[1] == row0)
            assert all(a[1] == b_[0] for a, b_ in zip(parts, parts[1:]))
            last = min(row0 + 16 * tiles, q[b] * group) - 1
            first_token = kv[b] - q[b] + row0 // group
            assert parts[0][0] == (0 if window is None else max(0, first_token - window + 1))
            assert parts[-1][1] == kv[b] - q[b] + last // group + 1
    slots = [int(w[4]) for w in plan.work if w[4] >= 0]
    assert len(set(slots)) == len(slots)


def test_a_captured_step_holds_its_packed_lists():
    q, kv = [1, 1, 1], [2000, 300, 8100]
    for window in (None, 3000):
        _, capacity = capacity_until(q, kv, 6, window, 64, 12000, packed=True)
        for t in range(0, 3900, 13):
            assert pad_plan(build_plan(q, [n + t for n in kv], 6, window, 64, packed=True), capacity) is not None, (window, t)


@pytest.mark.parametrize("new,kv,window", [(1300, 131072, None), (512, 131072, None), (22, 10 ** 6, None), (64, 30000, None), (1300, 131072, 8192), (700, 701, None)])
def test_partial_results_of_portions_do_not_grow_with_the_context(new, kv, window):
    """The blocks of a sequence that is cut are at most four times those with which every compute unit has two (64 a key/value head), and one more
    for each row of blocks, whose range need not begin at a cut."""
    group, cut_below = 6, 64
    n_wide = -(-new * group // (16 * WIDE_TILES))
    plan = build_plan([new], [kv], group, window, cut_below, packed=True)
    assert plan.work_wide.shape[0] <= PACKED_WIDE_BLOCKS * cut_below + n_wide
    assert plan.n_partials <= WIDE_TILES * plan.work_wide.shape[0]
    assert plan.n_partials * 8 * 16 * (128 + 4) * 4 <= 175e6  # bytes of eight heads of 128
    alone = build_plan([new], [kv], group, window, cut_below, packed=True).work_wide
    beside = build_plan([5, new, 300], [9, kv, 9000], group, window, cut_below, packed=True).work_wide
    ranges = lambda w, b: sorted(tuple(int(x) for x in r[1:4]) for r in w if r[0] == b)  # noqa: E731
    assert ranges(alone, 0) == ranges(beside, 1)


def test_chunks_of_portions():
    def cut(n_new, kv, window=None, group=4):
        return wide_chunk(-(-n_new * group // 128), n_new, kv, window, 64, True)

    assert [cut(64, 30000), cut(513, 3585, 2048), cut(300, 300), cut(64, 131072), cut(512, 131072), cut(1300, 131072)] == [1024, 1024, 1024, 1024, 8192, 32768]
    assert cut(2048, 4096) == 0 and wide_chunk(10, 300, 10 ** 6, None, 64, False) == 8192 and wide_chunk(3, 70, 10 ** 6, None, 64, False) == 2048
    assert cut(300, 131072, 2048) == 1024  # what a window reads counts, not what lies before it
    assert wide_item_tiles([300, 40], [300, 500], 4, 8, 128, 64, 256, True) == 4
    assert wide_item_tiles([300, 40], [300, 5000], 4, 8, 128, 64, 256, True) == WIDE_TILES
    # a portion in a window that is shorter than its chunk may be cut at a multiple of it all the same
    assert wide_item_tiles([300], [131072], 4, 8, 128, 64, 256, True, 700) == WIDE_TILES
