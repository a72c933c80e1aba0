"""Work lists of steps whose cache holds 4 or 8 bits: chunks of their own, every key of every row once, homes of captured steps."""

import numpy as np
import pytest

from cwm_amd.ops.attention_plan import PACKED_WIDE_CHUNK, build_plan, capacity_until, chunk_keys, pad_plan, wide_chunks


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
