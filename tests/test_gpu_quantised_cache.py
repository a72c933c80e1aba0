"""The quantised cache on the GPU: bytes as the layout says, what is read back, and attention over it."""

import math

import pytest
import torch

from cwm_amd import ops
from helpers import quantised as held

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _inv_freq(dim):
    return 1.0 / (500000.0 ** (torch.arange(0, dim, 2).float() / dim))


def _garbage(shape, seed):
    """Bytes of every kind: words that are NaN, infinite and subnormal among them."""
    return torch.randint(0, 256, shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(seed))


def _joined(tokens, q_heads, heads, dim, dtype, seed):
    """Keys and values as views of a joined projection's rows."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(tokens, (q_heads + 2 * heads) * dim, generator=g)
    x[:, q_heads * dim : (q_heads + heads) * dim] += 3 * torch.randn(heads * dim, generator=g) * (torch.rand(heads * dim, generator=g) < 0.1)
    x = x.to(dtype)
    return x, x[:, : q_heads * dim].unflatten(1, (q_heads, dim)), x[:, q_heads * dim : -heads * dim].unflatten(1, (heads, dim)), x[:, -heads * dim :].unflatten(1, (heads, dim))


def _views(x, q_heads, heads, dim):
    return x[:, : q_heads * dim].unflatten(1, (q_heads, dim)), x[:, q_heads * dim : -heads * dim].unflatten(1, (heads, dim)), x[:, -heads * dim :].unflatten(1, (heads, dim))


WRITES = [  # new tokens, lengths, page, heads
    ([1], [1], 8, 1),
    ([1, 1, 1], [9, 40, 17], 16, 2),
    ([8], [16], 8, 3),
    ([37], [37], 32, 8),
    ([5, 1, 30], [25, 40, 31], 24, 9),
    ([64, 3], [64, 70], 256, 17),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_written_bytes(dim, bits, dtype):
    for i, (new, kv, page, heads) in enumerate(WRITES):
        step = held.Step(new, kv, page, seed=i)
        x, _, k, v = _joined(sum(new), 2, heads, dim, dtype, seed=10 + i)
        before = _garbage((step.pool, *ops.quant_page_shape(heads, dim, page, bits)), i)
        turned = held.turn(k, step.positions, _inv_freq(dim))
        want = before.clone()
        at = step.positions.long()
        held.put_tokens(want, step.table[step.seq.long(), at // page].long(), at % page, turned, v, bits)
        cache, xd = before.to(DEV), x.to(DEV)
        q_d, k_d, v_d = _views(xd, 2, heads, dim)
        table, positions, seq = step.table.to(DEV), step.positions.to(DEV), step.seq.to(DEV)
        ops.quant_kv_write(k_d, v_d, positions, _inv_freq(dim).to(DEV), cache, table, seq, bits, q=q_d)
        off = int((cache.cpu() != want).sum())
        assert off == 0, (off, new, kv, page, heads)
        q_want = held.turn(x[:, : 2 * dim].unflatten(1, (2, dim)), step.positions, _inv_freq(dim))
        assert torch.equal(q_d.cpu(), q_want)
        assert torch.equal(xd[:, 2 * dim :].cpu(), x[:, 2 * dim :])  # keys and values stay as they are
        # what is held, read back token by token in another order
        order = torch.randperm(sum(new), generator=torch.Generator().manual_seed(i))
        for places in (torch.arange(sum(new)), order):
            k_r, v_r = ops.quant_kv_read(cache, table, positions[places.to(DEV)], seq[places.to(DEV)], dim, bits, dtype)
            kc = held.stands_for(*held.hold(turned.reshape(-1, heads, dim // 32, 32), bits), bits).flatten(2)
            vc = held.stands_for(*held.hold(v, bits), bits)
            # z + s (c - H) in one fused float32 rounding, then to the type: the float64 value rounded twice
            assert torch.equal(k_r.cpu(), kc[places].float().to(dtype))
            assert torch.equal(v_r.cpu(), vc[places].float().to(dtype))


@pytest.mark.parametrize("bits", [4, 8])
def test_writing_without_rotation_and_with_loose_rows(bits):
    """Rows that no vector load can take (an odd token stride, an odd first element), and no table of angles."""
    dim, heads, page, n = 64, 2, 16, 21
    step = held.Step([n], [n + 3], page)
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(n, 2 * heads * dim + 5, generator=g).bfloat16()
    for offset in (1, 2, 4):
        def views(t):
            return t[:, offset : offset + heads * dim].unflatten(1, (heads, dim)), t[:, offset + heads * dim : offset + 2 * heads * dim].unflatten(1, (heads, dim))

        (k, v), (kd, vd) = views(wide), views(wide.to(DEV))
        cache = torch.zeros((step.pool, *ops.quant_page_shape(heads, dim, page, bits)), dtype=torch.uint8)
        want, at = cache.clone(), step.positions.long()
        held.put_tokens(want, step.table[0, at // page].long(), at % page, k, v, bits)
        cache = cache.to(DEV)
        ops.quant_kv_write(kd, vd, step.positions.to(DEV), None, cache, step.table.to(DEV), step.seq.to(DEV), bits)
        assert torch.equal(cache.cpu(), want)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_writing_values_of_every_kind(bits, dtype):
    """Equal values, zeros, far ends of the range, subnormal numbers, infinities and NaN."""
    dim, heads, page, n = 64, 1, 16, 16
    step = held.Step([n], [n], page)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(n, heads, dim, generator=g)
    x[0] = 0.0
    x[1] = 3.7
    x[2] *= 1e36
    x[3] *= 1e-36
    x[4, 0, 5] = math.inf
    x[5, 0, 40] = -math.inf
    x[6, 0, 31] = math.nan
    x[7, 0, 32:] = 1e-40
    x[8, 0, 3] = 1e30
    x[9] = 100.0 + 1e-3 * torch.randn(heads, dim, generator=g)
    x[10] = torch.where(torch.rand(heads, dim, generator=g) < 0.5, 3.3e38, -3.3e38)
    x = x.to(dtype)
    want = torch.zeros((step.pool, *ops.quant_page_shape(heads, dim, page, bits)), dtype=torch.uint8)
    cache = want.to(DEV)
    at = step.positions.long()
    held.put_tokens(want, step.table[0, at // page].long(), at % page, x, x, bits)
    ops.quant_kv_write(x.to(DEV), x.to(DEV), step.positions.to(DEV), None, cache, step.table.to(DEV), step.seq.to(DEV), bits)
    assert torch.equal(cache.cpu(), want)
    k, v = ops.quant_kv_read(cache, step.table.to(DEV), step.positions.to(DEV), step.seq.to(DEV), dim, bits, torch.float32)
    assert torch.isnan(k[4, 0, :32]).all() and not torch.isnan(k[4, 0, 32:]).any() and torch.isnan(v[4]).all()
    assert torch.isnan(k[5, 0, 32:]).all() and torch.isnan(v[6]).all() and torch.isfinite(v[:4]).all()


def test_tokens_without_a_page():
    """A token whose page is not held, or lies outside the pool or the table, is not written, and reads as zeros."""
    dim, heads, page, bits = 32, 2, 8, 4
    g = torch.Generator().manual_seed(5)
    k, v = torch.randn(6, heads, dim, generator=g), torch.randn(6, heads, dim, generator=g)
    table = torch.tensor([[1, -1, 7]], dtype=torch.int32)  # a pool of three pages
    positions, seq = torch.tensor([0, 8, 16, 24, 7, 2], dtype=torch.int32), torch.tensor([0, 0, 0, 0, 0, 1], dtype=torch.int32)
    before = _garbage((3, *ops.quant_page_shape(heads, dim, page, bits)), 1)
    want = before.clone()
    held.put_tokens(want, torch.tensor([1, 1]), torch.tensor([0, 7]), k[[0, 4]], v[[0, 4]], bits)
    cache = before.to(DEV)
    args = positions.to(DEV), seq.to(DEV)
    ops.quant_kv_write(k.to(DEV), v.to(DEV), args[0], None, cache, table.to(DEV), args[1], bits)
    assert torch.equal(cache.cpu(), want)
    kr, vr = ops.quant_kv_read(cache, table.to(DEV), *args, dim, bits, torch.float32)
    assert not kr[[1, 2, 3, 5]].any() and not vr[[1, 2, 3, 5]].any()
    assert torch.equal(vr[[0, 4]].cpu(), held.stands_for(*held.hold(v[[0, 4]], bits), bits).float())


def test_no_tokens():
    cache = _garbage((1, *ops.quant_page_shape(1, 32, 8, 4)), 2).to(DEV)
    none, table = torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    before = cache.clone()
    ops.quant_kv_write(torch.zeros(0, 1, 32, device=DEV), torch.zeros(0, 1, 32, device=DEV), none, None, cache, table, none, 4)
    k, v = ops.quant_kv_read(cache, table, none, none, 32, 4, torch.bfloat16)
    assert torch.equal(cache, before) and k.shape == v.shape == (0, 1, 32)


def _case(new, kv, page, q_heads, heads, dim, bits, dtype, window, seed, sharpen=1.5):
    """The operands of an attention step over a cache that is garbage wherever no key is, and the float64 result."""
    step = held.Step(new, kv, page, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    centre = 3 * torch.randn(heads, dim, generator=g) * (torch.rand(heads, dim, generator=g) < 0.1)
    keys = [(torch.randn(n, heads, dim, generator=g) + centre).to(dtype) for n in kv]
    values = [(torch.randn(n, heads, dim, generator=g) + 0.5).to(dtype) for n in kv]
    cache = _garbage((step.pool, *ops.quant_page_shape(heads, dim, page, bits)), seed)
    held.put_all(cache, step.table, kv, keys, values, bits)
    q = (sharpen * torch.randn(sum(new), q_heads, dim, generator=g)).to(dtype)
    return step, cache, q, keys, values


def _attend(step, cache, q, bits, window, scale):
    return ops.quant_paged_attention(q.to(DEV), cache.to(DEV), step.table.to(DEV), step.batch(DEV), window, scale, bits)


def _close(got, step, q, keys, values, bits, window, scale):
    want, limit = held.attention(step, q, keys, values, bits, window, scale)
    off = (got.cpu().double() - want).abs()
    assert torch.isfinite(got).all()
    worst = float((off / limit).max())
    assert worst <= 1, f"{worst} of the limit, {float(off.max())} off"


STEPS = [  # new tokens, lengths, page, query heads, key/value heads, window
    ([1], [1], 8, 1, 1, None),
    ([1], [33], 32, 6, 1, None),
    ([1, 1, 1], [7, 100, 64], 16, 8, 2, None),
    ([1, 1], [300, 45], 24, 16, 1, 40),
    ([1, 9, 1, 20], [61, 9, 500, 33], 64, 6, 2, None),
    ([13], [200], 8, 3, 3, 17),
    ([1, 1], [2300, 2049], 256, 5, 1, None),  # longer than a block takes: cut and joined
    ([70], [70], 32, 8, 2, None),  # 280 rows: blocks of 128
    ([150, 1, 50], [190, 70, 50], 40, 3, 1, 64),
    ([1], [77], 96, 20, 1, 1),  # more than 16 query heads to a key/value head
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention(dim, bits, dtype):
    for i, (new, kv, page, q_heads, heads, window) in enumerate(STEPS):
        step, cache, q, keys, values = _case(new, kv, page, q_heads, heads, dim, bits, dtype, window, 100 + i)
        scale = dim ** -0.5
        got = _attend(step, cache, q, bits, window, scale)
        print(dim, bits, dtype, new, kv, page, q_heads, heads, window, flush=True)
        _close(got, step, q, keys, values, bits, window, scale)


@pytest.mark.parametrize("bits,dtype", [(4, torch.bfloat16), (8, torch.bfloat16), (4, torch.float32)])
def test_long_contexts(bits, dtype):
    for new, kv, heads, window in [([1], [9001], 2, None), ([1, 1], [70003, 12], 1, None), ([2], [20000], 1, 8195), ([60], [5003], 1, None)]:
        step, cache, q, keys, values = _case(new, kv, 64, 3 * heads, heads, 64, bits, dtype, window, 7)
        _close(_attend(step, cache, q, bits, window, 0.125), step, q, keys, values, bits, window, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
def test_scores_that_outgrow_their_reference(bits):
    """Scores that climb by far more than 256 from tile to tile, and fall again."""
    new, kv, dim = [1, 40], [700, 300], 64
    step, cache, q, keys, values = _case(new, kv, 32, 4, 1, dim, bits, torch.bfloat16, None, 9)
    for k in keys:
        n = k.shape[0]
        k *= (1 + 3 * torch.sin(torch.arange(n) * 6.0 / n))[:, None, None].to(k.dtype)
    held.put_all(cache, step.table, kv, keys, values, bits)
    q *= 8
    _close(_attend(step, cache, q, bits, None, 0.125), step, q, keys, values, bits, None, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 96, 192])
def test_portions_whose_numbers_do_not_fit_16_bits(dim, bits):
    """Queries, keys and values from 2^-60 to 2^60, by row and by some of the tokens."""
    new, kv, group = [80, 50], [333, 50], 4
    for i, (of_q, of_k, of_v) in enumerate([(0, 0, 40), (0, 0, -40), (-25, 25, 0), (25, -25, 12), (-60, 60, -30), (3, -14, 60)]):
        step, cache, q, keys, values = _case(new, kv, 32, group, 1, dim, bits, torch.bfloat16, None, 60 + i)
        for j, (k, v) in enumerate(zip(keys, values)):
            k *= 2.0 ** of_k
            some = torch.arange(v.shape[0]) // 40 % 3 == j
            v *= torch.where(some, 2.0 ** of_v, 2.0 ** (of_v // 2))[:, None, None].to(v.dtype)
        keys[0][70:90] *= 2.0 ** -9
        q *= 2.0 ** of_q
        q[3:60:7] *= 2.0 ** -8
        held.put_all(cache, step.table, kv, keys, values, bits)
        _close(_attend(step, cache, q, bits, None, dim ** -0.5), step, q, keys, values, bits, None, dim ** -0.5)


def test_a_key_that_is_not_finite_reaches_its_readers_only():
    new, kv, dim, bits = [12, 1], [60, 300], 64, 4
    step, cache, q, keys, values = _case(new, kv, 16, 4, 2, dim, bits, torch.bfloat16, 20, 11)
    values[0][55, 1, 3] = math.nan  # head 1: read by the queries at 55 .. 59 (tokens 7 .. 11)
    keys[1][100, 0, 0] = math.inf  # outside the window of the token at 299
    held.put_all(cache, step.table, kv, keys, values, bits)
    got = _attend(step, cache, q, bits, 20, 0.125).reshape(13, 4, dim)
    bad = torch.isnan(got).all(-1).cpu()
    want = torch.zeros(13, 4, dtype=torch.bool)
    want[7:12, 2:] = True
    assert torch.equal(bad, want) and torch.isfinite(got[~want.to(DEV)]).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_portions_of_many_rows_and_what_is_not_finite(bits):
    """Portions whose keys are unpacked first: a window that has passed pages, pages of 24 and of 512 tokens, a key and a value that are
    not finite, and a page that is missing, beside decoded tokens."""
    for page in (24, 512):
        dim, group, heads, window = 64, 4, 2, 300
        new, kv = [100, 1, 200], [1500, 40, 200]
        step, cache, q, keys, values = _case(new, kv, page, group * heads, heads, dim, bits, torch.bfloat16, window, 31 + page)
        for lp in range((1400 - window + 1) // page):
            step.table[0, lp] = -1  # given back: the window has passed them
        _close(_attend(step, cache, q, bits, window, 0.125), step, q, keys, values, bits, window, 0.125)
        keys[0][1440, 0, 40], values[2][150, 1, 7] = math.inf, math.nan
        for b, key in ((0, 1440), (2, 150)):
            place = step.table[b, key // page].long().reshape(1), torch.tensor([key % page])
            held.put_tokens(cache, *place, keys[b][key : key + 1], values[b][key : key + 1], bits)
        got = torch.isnan(_attend(step, cache, q, bits, window, 0.125)).reshape(301, 2, group, dim).all(-1).all(-1).cpu()
        want = torch.zeros(301, 2, dtype=torch.bool)
        want[40:100, 0] = True  # the tokens at 1440 .. 1499
        want[101 + 150 :, 1] = True
        assert torch.equal(got, want)
    step.table[2, 0] = 10 ** 6
    got = torch.isnan(_attend(step, cache, q, bits, window, 0.125)).all(-1)
    assert got[101:].all() and not got[:40].any()


def test_a_missing_page_is_seen():
    new, kv, dim, bits = [1, 1], [60, 60], 64, 4
    step, cache, q, keys, values = _case(new, kv, 16, 4, 2, dim, bits, torch.bfloat16, 20, 12)
    step.table[0, 0] = -1  # given back: the window has passed it
    step.table[1, 3] = 99
    got = _attend(step, cache, q, bits, 20, 0.125)
    assert torch.isfinite(got[0]).all() and torch.isnan(got[1]).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_row_does_not_depend_on_its_batch(dtype):
    dim, bits = 128, 4
    new, kv = [1, 1, 40, 1], [3000, 77, 40, 513]
    step, cache, q, keys, values = _case(new, kv, 32, 16, 2, dim, bits, dtype, None, 13)
    together = _attend(step, cache, q, bits, None, dim ** -0.5)
    t0 = 0
    for b, m in enumerate(new):
        alone = held.Step([m], [kv[b]], 32)
        alone.table = step.table[b : b + 1].contiguous()
        got = _attend(alone, cache, q[t0 : t0 + m], bits, None, dim ** -0.5)
        assert torch.equal(got, together[t0 : t0 + m])
        t0 += m
    assert torch.equal(together, _attend(step, cache, q, bits, None, dim ** -0.5))


def test_written_then_attended_in_one_stream_of_steps():
    """A prompt in portions and decoded tokens, as a model's layer runs them: each step writes, then reads."""
    dim, heads, q_heads, page, bits = 64, 2, 8, 16, 4
    total, cuts = 75, [0, 30, 31, 62, 63, 64, 75]
    g = torch.Generator().manual_seed(21)
    x = torch.randn(total, (q_heads + 2 * heads) * dim, generator=g).bfloat16()
    full = held.Step([total], [total], page)
    cache = _garbage((full.pool, *ops.quant_page_shape(heads, dim, page, bits)), 3).to(DEV)
    got = []
    for a, b in zip(cuts, cuts[1:]):
        step = held.Step([b - a], [b], page)
        step.table = full.table
        q, k, v = _views(x[a:b].to(DEV), q_heads, heads, dim)
        batch = step.batch(DEV)
        ops.quant_kv_write(k, v, batch.positions, _inv_freq(dim).to(DEV), cache, full.table.to(DEV), batch.seq_of_token, bits, q=q)
        got.append(ops.quant_paged_attention(q, cache, full.table.to(DEV), batch, None, 0.125, bits))
    q, k, v = _views(x, q_heads, heads, dim)
    turned = [held.turn(t, full.positions, _inv_freq(dim)) for t in (q, k)]
    _close(torch.cat(got), full, turned[0], [turned[1]], [v], bits, None, 0.125)


def test_on_a_stream_of_its_own_and_captured():
    dim, bits = 64, 4
    new, kv = [1, 1], [40, 300]
    step, cache, q, keys, values = _case(new, kv, 32, 8, 2, dim, bits, torch.bfloat16, None, 17)
    cache, table, batch = cache.to(DEV), step.table.to(DEV), step.batch(DEV)
    k, v = torch.randn(2, 2, dim, device=DEV).bfloat16(), torch.randn(2, 2, dim, device=DEV).bfloat16()
    k2, v2 = torch.randn(2, 2, dim, device=DEV).bfloat16(), torch.randn(2, 2, dim, device=DEV).bfloat16()
    qd = q.to(DEV)
    kin, vin = k.clone(), v.clone()

    def layer():
        ops.quant_kv_write(kin, vin, batch.positions, None, cache, table, batch.seq_of_token, bits)
        read = ops.quant_kv_read(cache, table, batch.positions, batch.seq_of_token, dim, bits, torch.bfloat16)
        return (ops.quant_paged_attention(qd, cache, table, batch, None, 0.125, bits), *read)

    want = [t.clone() for t in layer()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = layer()
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for kk, vv in ((k2, v2), (k, v), (k2, v2)):
        kin.copy_(kk), vin.copy_(vv)
        graph.replay()
        replayed = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(replayed, layer()))


@pytest.mark.parametrize("bits", [4, 8])
def test_sequences_without_new_tokens(bits):
    """Beside portions and decoded tokens: they have pages, and nothing to do."""
    new, kv, dim = [0, 80, 1, 0], [64, 80, 2300, 0], 64
    step, cache, q, keys, values = _case(new, kv, 32, 8, 2, dim, bits, torch.bfloat16, None, 18)
    _close(_attend(step, cache, q, bits, None, 0.125), step, q, keys, values, bits, None, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
def test_portions_of_many_rows_captured(bits):
    """A step whose lists are on the device already is captured, replayed with other queries and pages, with eager steps in between."""
    new, kv, dim = [70, 1, 200], [500, 2100, 200], 128
    step, cache, q, keys, values = _case(new, kv, 32, 12, 2, dim, bits, torch.bfloat16, None, 19)
    other = _case(new, kv, 32, 12, 2, dim, bits, torch.bfloat16, None, 20)
    cache, table, batch, qd = cache.to(DEV), step.table.to(DEV), step.batch(DEV), q.to(DEV)
    sets = [(cache.clone(), table.clone(), qd.clone()), (other[1].to(DEV), other[0].table.to(DEV), other[2].to(DEV))]
    run = lambda c, t, x: ops.quant_paged_attention(x, c, t, batch, None, dim ** -0.5, bits)  # noqa: E731
    want = [run(*s) for s in sets]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(cache, table, qd)
    for i in (1, 0, 1, 1, 0):
        for to, source in zip((cache, table, qd), sets[i]):
            to.copy_(source)
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(replayed, want[i]) and torch.equal(run(*sets[i]), want[i])


@pytest.mark.parametrize("portion", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bits", [4, 8])
def test_cut_rows_keep_what_is_not_finite(bits, dtype, portion):
    """Rows cut in chunks of 1,024 keys: a chunk whose keys are all not finite (the newest key, alone in the last one; a whole
    chunk in the middle) has no largest score, and is not a chunk without keys.  Its reader gets NaN, its neighbour nothing of it."""
    dim, group, heads = 64, 4, 2
    new, kv = [1, 1, 1] + [60] * portion, [4097, 4097, 3000] + [5003] * portion
    step, cache, q, keys, values = _case(new, kv, 64, group * heads, heads, dim, bits, dtype, None, 41)
    keys[0][4096, 0, 3] = math.inf
    keys[1][1024:2048, 1] = math.nan
    if portion:
        keys[3][1024:2048, 0, 40] = -math.inf
    held.put_all(cache, step.table, kv, keys, values, bits)
    got = _attend(step, cache, q, bits, None, 0.125).cpu().reshape(-1, heads, group * dim)
    want = torch.zeros(got.shape[:2], dtype=torch.bool)
    want[0, 0] = want[1, 1] = True
    want[3:, 0] = True
    assert torch.equal(torch.isnan(got).all(-1), want) and torch.isfinite(got[~want]).all()


@pytest.mark.parametrize("portion", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_missing_chunk_is_seen_whatever_is_read_in_its_place(dtype, portion):
    """All pages of a chunk missing, and the page that is read instead full of bytes of 255, whose words are NaN."""
    dim, group, heads, bits, page = 64, 4, 1, 4, 64
    new, kv = [1, 1] + [60] * portion, [4097, 3000] + [5003] * portion
    step, _, q, keys, values = _case(new, kv, page, group * heads, heads, dim, bits, dtype, None, 42)
    step.table[step.table == 0] = min(set(range(1, step.pool)) - set(step.table.reshape(-1).tolist()))
    cache = torch.full((step.pool, *ops.quant_page_shape(heads, dim, page, bits)), 255, dtype=torch.uint8)
    held.put_all(cache, step.table, kv, keys, values, bits)
    step.table[0, 64] = -1  # the last chunk: one key
    if portion:
        step.table[2, 16:32] = 10 ** 6
    got = _attend(step, cache, q, bits, None, 0.125).cpu()
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1]).all() and torch.isnan(got[2:]).all()


@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("bits", [4, 8])
def test_keys_that_a_window_has_passed_may_hold_anything(bits, page):
    """Portions: the pages before the window's first key belong to somebody else now, and hold numbers of 2^125."""
    new, kv, dim, group, window = [100, 3], [400, 300], 64, 4, 50
    step, cache, q, keys, values = _case(new, kv, page, group, 1, dim, bits, torch.bfloat16, window, 44)
    spare = next(p for p in range(step.pool) if p not in step.table)
    cache[spare] = 0x7E  # steps and offsets of 8.4e37
    step.table[0, : (300 - window + 1) // page] = spare
    _close(_attend(step, cache, q, bits, window, 0.125), step, q, keys, values, bits, window, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
def test_small_weights_of_portions_add_up(bits):
    """A portion over one key that takes nearly all of the softmax, with a value of zeros, and thousands of keys of e^-18 of it, with
    values of ones: the result is what the small weights make together.  A weight is off by 2^-32 of the row's largest at most, or by
    2^-12 of itself, in all n 2^-32 and 2^-12 of the result; its exponential and the sums by under 2^-16 of it, and the result is rounded."""
    new, kv, dim, group = [80], [4000], 64, 4
    step, cache, q, keys, values = _case(new, kv, 32, group, 1, dim, bits, torch.bfloat16, None, 43)
    keys[0][:], values[0][:], q[:] = 0.0, 1.0, 1.0
    keys[0][5], values[0][5] = 2.25, 0.0  # a score of 64 * 2.25 / 8 = 18
    held.put_all(cache, step.table, kv, keys, values, bits)
    got = _attend(step, cache, q, bits, None, 0.125).cpu().double()
    others = torch.arange(kv[0] - new[0], kv[0]).double()[:, None]  # a query at p reads p small ones
    want = others * math.exp(-18) / (1 + others * math.exp(-18))
    limit = others * 2.0 ** -32 + (2.0 ** -12 + 2.0 ** -16) * want
    limit = limit + 2.0 ** -8 * (want + limit)
    assert ((got - want).abs() <= limit).all(), float(((got - want).abs() / limit).max())


@pytest.mark.parametrize("bits", [4, 8])
def test_groups_whose_codes_are_nearly_all_the_lowest(bits):
    """The words of codes 0 and 2H - 1 side by side, at every place of a group."""
    dim, page, n = 64, 32, 32
    step = held.Step([n], [n], page)
    x = torch.full((n, 1, dim), -1.0)
    for t in range(n):
        x[t, 0, [t, 63 - t]] = 1.0
    want = torch.zeros((step.pool, *ops.quant_page_shape(1, dim, page, bits)), dtype=torch.uint8)
    cache, at = want.to(DEV), step.positions.long()
    held.put_tokens(want, step.table[0, at // page].long(), at % page, x, x, bits)
    ops.quant_kv_write(x.to(DEV), x.to(DEV), step.positions.to(DEV), None, cache, step.table.to(DEV), step.seq.to(DEV), bits)
    assert torch.equal(cache.cpu(), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_portions_whose_chunks_are_doubled(monkeypatch, dtype):
    """Short chunks, so that a short context has more of them than a step may leave partial results of."""
    from cwm_amd.ops import attention_plan

    monkeypatch.setattr(attention_plan, "PACKED_WIDE_CHUNK", 128)
    monkeypatch.setattr(attention_plan, "PACKED_WIDE_BLOCKS", 1)
    new, kv, dim, bits = [100, 1], [3001, 500], 64, 4
    for window in (None, 700):
        step, cache, q, keys, values = _case(new, kv, 32, 32, 8, dim, bits, dtype, window, 46)
        assert attention_plan.wide_chunk(4, 100, 3001, window, 64, True) == (256 if window is None else 128)
        _close(_attend(step, cache, q, bits, window, 0.125), step, q, keys, values, bits, window, 0.125)


@pytest.mark.parametrize("bits", [4, 8])
def test_portions_that_take_turns(monkeypatch, bits):
    """What a step unpacks is held for some of its sequences at a time: the rows are those of one piece, and the memory is bounded."""
    from cwm_amd.ops import quantised

    new, kv, dim, heads, group = [100, 1, 70, 200, 1, 90], [9000, 5000, 8200, 9300, 40, 90], 128, 2, 4
    step, cache, q, _, _ = _case(new, kv, 32, group * heads, heads, dim, bits, torch.bfloat16, None, 47)
    cache, table, qd = cache.to(DEV), step.table.to(DEV), q.to(DEV)
    for window in (None, 700):
        peaks, got = [], []
        for most in (1 << 29, 1):
            monkeypatch.setattr(quantised, "UNPACK_BYTES", most)
            batch = step.batch(DEV)
            run = lambda: ops.quant_paged_attention(qd, cache, table, batch, window, dim ** -0.5, bits)  # noqa: E731
            run()
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
            before = torch.cuda.memory_allocated()
            torch.cuda.reset_peak_memory_stats()
            got.append(run())
            peaks.append(torch.cuda.max_memory_allocated() - before)
            assert torch.equal(got[-1], run())
        assert torch.equal(*got) and torch.isfinite(got[0]).all()
        assert peaks[1] < 0.6 * peaks[0]


@pytest.mark.parametrize("bits", [4, 8])
def test_portions_over_values_far_apart(bits):
    """Sums of 2^64 that are brought to the exponent of a tile of values of 2^-70, the lowest there is, and back."""
    new, kv, dim, group = [80], [480], 64, 4
    step, cache, q, keys, values = _case(new, kv, 32, group, 1, dim, bits, torch.bfloat16, None, 48, sharpen=0.1)
    values[0][:320] = (1 + values[0][:320].abs()) * 2.0 ** 55
    values[0][320:448] *= 2.0 ** -70
    held.put_all(cache, step.table, kv, keys, values, bits)
    _close(_attend(step, cache, q, bits, None, 0.125), step, q, keys, values, bits, None, 0.125)


def test_portions_that_take_turns_captured(monkeypatch):
    """The pieces of a step in one graph, replayed with other queries, with eager steps in between."""
    from cwm_amd.ops import quantised

    monkeypatch.setattr(quantised, "UNPACK_BYTES", 1)
    new, kv, dim, bits = [70, 1, 100, 60], [500, 2100, 3000, 60], 64, 4
    step, cache, q, _, _ = _case(new, kv, 32, 12, 2, dim, bits, torch.bfloat16, None, 49)
    cache, table, batch = cache.to(DEV), step.table.to(DEV), step.batch(DEV)
    sets = [q.to(DEV), q.flip(0).to(DEV)]
    held_q = sets[0].clone()
    run = lambda x: ops.quant_paged_attention(x, cache, table, batch, None, dim ** -0.5, bits)  # noqa: E731
    want = [run(x) for x in sets]
    assert len(quantised._turns(batch, 6, None, 2, dim, held_q.device)) == 3
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(held_q)
    for i in (1, 0, 1, 1, 0):
        held_q.copy_(sets[i])
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(replayed, want[i]) and torch.equal(run(sets[i]), want[i])
