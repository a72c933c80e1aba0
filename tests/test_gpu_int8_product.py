"""The product of 8-bit integers: the integers of a row, every kernel at sizes that end inside its tiles, and the whole call."""

import math

import pytest
import torch

from cwm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rows(m, k, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, k, generator=g) * torch.exp(torch.randn(1, k, generator=g))).to(dtype)


def _quantised(x):
    """The definition: float32 scale, true quotients, ties to even."""
    x = x.float()
    top = x.abs().amax(1)
    a = top / torch.full_like(top, 127)
    c = torch.where(a[:, None] > 0, torch.round(x / a[:, None]), torch.zeros_like(x))
    return c.to(torch.int8), a


def _weight(n, k, seed, stride=None):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(-127, 128, (n, stride or k), generator=g).to(torch.int8)
    return w[:, :k], torch.rand(n, generator=g) * 0.01 + 1e-4


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 16), (3, 100), (7, 1), (2, 129), (5, 4096), (300, 2056)])
def test_integers_of_rows(m, k, dtype):
    x = _rows(m, k, dtype, m + k)
    x[0] *= 0
    codes, scale = ops.quantize_rows(x.to(DEV))
    want, a = _quantised(x)
    assert codes.shape == (m, k) and torch.equal(codes.cpu(), want) and torch.equal(scale.cpu(), a)
    assert codes.stride(0) % 128 == 0 and not codes._base[:, k:].any()
    wide = torch.cat([x, x[:, :3]], 1).to(DEV)[:, 1 : 1 + k] if k > 1 else x.to(DEV)  # rows that no vector load takes
    codes, scale = ops.quantize_rows(wide)
    want, a = _quantised(wide.cpu())
    assert torch.equal(codes.cpu(), want) and torch.equal(scale.cpu(), a)


@pytest.mark.parametrize("k", [8, 120, 4104, 8200, 16392, 32768, 32776])
def test_integers_of_long_rows_ties_and_the_ends_of_the_range(k):
    """Rows of which a thread keeps one to eight pieces, or none; quotients that are ties; scales whose reciprocal is no float32."""
    for dtype in (torch.bfloat16, torch.float32):
        x = _rows(5, k, dtype, k)
        x[1] = (torch.arange(k) % 255 - 127) / 2
        x[1, 3] = 127.0  # a scale of 1: every second quotient is a tie
        x[2] *= 1e-39
        x[3] = 0
        x[3, k // 2] = 3e38
        x[4, k - 1] = 1000.0
        codes, scale = ops.quantize_rows(x.to(DEV))
        want, a = _quantised(x)
        assert torch.equal(codes.cpu(), want) and torch.equal(scale.cpu(), a)
        assert not codes._base[:, k:].any()


def test_rows_that_are_not_finite():
    x = _rows(5, 64, torch.float32, 1)
    x[1, 3], x[2, 60], x[3, 0] = math.nan, math.inf, -math.inf
    codes, scale = ops.quantize_rows(x.to(DEV))
    assert torch.isnan(scale[1:4]).all() and torch.isfinite(scale[[0, 4]]).all() and not codes[1:4].any()
    w, s = _weight(40, 64, 2)
    y = ops.linear_int8(x.to(DEV), w.to(DEV), s.to(DEV))
    assert torch.isnan(y[1:4]).all() and torch.isfinite(y[[0, 4]]).all()


def _check(x, w, s, bias, out_dtype, tile=None):
    y = ops.linear_int8(x.to(DEV), w.to(DEV), s.to(DEV), None if bias is None else bias.to(DEV), out_dtype, tile)
    codes, a = _quantised(x)
    exact = (codes.double() @ w.double().t()) * a.double()[:, None] * s.double()
    # the sum's conversion, two products and the bias's sum, 2^-24 of themselves each, and the result's own rounding
    limit = 3.01 * 2.0 ** -24 * exact.abs()
    if bias is not None:
        exact = exact + bias.double()
        limit = limit + 2.0 ** -24 * (exact.abs() + limit)
    limit = limit + (2.0 ** -8 if out_dtype == torch.bfloat16 else 0) * (exact.abs() + limit) + 1e-44
    assert y.dtype == out_dtype and y.shape == exact.shape
    off = (y.cpu().double() - exact).abs()
    assert (off <= limit).all(), (x.shape, w.shape, tile, float((off / limit).max()))


SIZES = [  # rows, columns, K
    (1, 1, 16), (1, 100, 48), (3, 16, 128), (16, 33, 144), (17, 64, 256), (33, 31, 1040), (64, 130, 384), (70, 48, 112), (129, 70, 272),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products_of_few_rows(dtype):
    for i, (m, n, k) in enumerate(SIZES):
        x = _rows(m, k, dtype, i)
        w, s = _weight(n, k, i)
        _check(x, w, s, torch.randn(n) if i % 2 else None, dtype, 0)
        w, s = _weight(n, k, i, stride=k + 16)
        _check(x, w, s, None, torch.float32, 0)


@pytest.mark.parametrize("tile", [3, 4])
def test_products_with_k_in_parts(tile):
    """The parts' sums are whole numbers: whatever the parts, the result is the same."""
    for i, (m, n, k, parts) in enumerate([(1, 1, 256, 2), (5, 130, 272, 3), (17, 33, 1040, 4), (64, 129, 1168, 9), (65, 70, 2048, 16), (130, 260, 640, 3)]):
        for dtype in (torch.bfloat16, torch.float32):
            x = _rows(m, k, dtype, 40 + i)
            w, s = _weight(n, k, 40 + i, stride=k + 16 * (i % 2))
            bias = torch.randn(n) if i % 2 else None
            given = (x.to(DEV), w.to(DEV), s.to(DEV), None if bias is None else bias.to(DEV))
            for out in (torch.bfloat16, torch.float32):
                _check(x, w, s, bias, out, tile)
                assert torch.equal(ops.linear_int8(*given, out, tile, parts), ops.linear_int8(*given, out, tile))
                assert torch.equal(ops.linear_int8(*given, out), ops.linear_int8(*given, out, tile))
    with pytest.raises(ops.KernelError, match="parts"):
        ops.linear_int8(*given, tile=tile, parts=6)
    for other in (-1, 0, 1, 2):
        with pytest.raises(ops.KernelError, match="parts"):
            ops.linear_int8(given[0][:1], *given[1:], tile=other, parts=2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_products_of_one_launch(dtype):
    """Up to four rows, whose integers every block makes itself."""
    for i, (m, n, k) in enumerate([(1, 1, 16), (1, 100, 48), (2, 33, 2048), (3, 16, 144), (3, 9000, 256), (4, 70, 1040), (4, 130, 4096), (1, 20, 16384), (2, 20, 8176)]):
        x = _rows(m, k, dtype, i)
        w, s = _weight(n, k, i, stride=k + 16 * (i % 2))
        bias = torch.randn(n) if i % 2 else None
        for out in (torch.bfloat16, torch.float32):
            _check(x, w, s, bias, out, -1)
        y = ops.linear_int8(x.to(DEV), w.to(DEV), s.to(DEV), tile=-1)
        assert torch.equal(y, ops.linear_int8(x.to(DEV), w.to(DEV), s.to(DEV), tile=0))
        wide = torch.cat([x, x], 1).to(DEV)[:, 1 : 1 + k]  # rows that no vector load takes
        _check(wide.cpu(), w, s, bias, dtype, -1)
        assert torch.equal(ops.linear_int8(wide, w.to(DEV), s.to(DEV), tile=-1), ops.linear_int8(wide, w.to(DEV), s.to(DEV), tile=0))
    x = _rows(4, 64, dtype, 1)
    x[0] *= 0
    x[1, 3], x[2, 60] = math.nan, math.inf
    w, s = _weight(40, 64, 2)
    y = ops.linear_int8(x.to(DEV), w.to(DEV), s.to(DEV), tile=-1)
    assert torch.isnan(y[1:3]).all() and not y[0].any() and torch.isfinite(y[3]).all()


@pytest.mark.parametrize("tile", [1, 2, 3, 4])
def test_products_of_many_rows(tile):
    for i, (m, n, k) in enumerate([(1, 1, 128), (65, 100, 256), (300, 130, 384), (257, 513, 1024), (1000, 2000, 512), (513, 1027, 128), (70, 300, 144), (130, 131, 2032), (5, 17, 1104)]):
        x = _rows(m, k, torch.bfloat16, i)
        w, s = _weight(n, k, i, stride=k + 128 * (i % 2))
        _check(x, w, s, torch.randn(n) if i % 2 else None, torch.bfloat16 if i % 3 else torch.float32, tile)


def test_sums_at_the_end_of_their_range():
    """All integers 127 at the largest K: the sum is 32 bits to the last one."""
    k = ops.INT8_MAX_K
    for m, tile in ((2, 0), (70, 3)):
        x, w = torch.ones(m, k), torch.full((20, k), 127, dtype=torch.int8)
        _check(x, w, torch.ones(20), None, torch.float32, tile)
        _check(-x, w, torch.ones(20), None, torch.float32, tile)


def test_the_call_chooses_among_its_kernels():
    for m, n, k in [(1, 2048, 2048), (5, 512, 8192), (40, 4096, 512), (100, 1024, 1024), (600, 1536, 640), (200, 256, 2064), (17, 300, 112), (300, 9000, 4080)]:
        x = _rows(m, k, torch.bfloat16, m)
        w, s = _weight(n, k, m)
        _check(x, w, s, None, torch.bfloat16)


def test_no_rows_and_weights_of_its_own_making():
    w = torch.randn(48, 200, device=DEV)
    codes, scale = ops.quantize_rows(w)
    x = torch.randn(9, 208, device=DEV)
    with pytest.raises(ops.KernelError, match="multiple of 16"):
        ops.linear_int8(x[:, :200], codes, scale)
    codes, scale = ops.quantize_rows(torch.randn(48, 208, device=DEV))
    _check(x.cpu(), codes.cpu(), scale.cpu(), None, torch.float32)
    assert ops.linear_int8(x[:0], codes, scale).shape == (0, 48)
    assert torch.equal(ops.linear_int8(x, codes, scale), ops.linear_int8(x, codes.contiguous(), scale))


def test_a_row_does_not_depend_on_its_batch():
    x = _rows(500, 1024, torch.bfloat16, 3).to(DEV)
    w, s = (t.to(DEV) for t in _weight(700, 1024, 4))
    whole = ops.linear_int8(x, w, s)
    for a, b in ((0, 1), (3, 20), (100, 163), (7, 200), (0, 400)):
        assert torch.equal(ops.linear_int8(x[a:b], w, s), whole[a:b])


def test_on_a_stream_of_its_own_and_captured():
    x = [_rows(m, 512, torch.bfloat16, m).to(DEV) for m in (3, 200)]
    other = [t.flip(0) * 2 for t in x]
    w, s = (t.to(DEV) for t in _weight(300, 512, 5))
    want = [ops.linear_int8(t, w, s) for t in x]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = [ops.linear_int8(t, w, s) for t in x]
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    held = [t.clone() for t in x]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = [ops.linear_int8(t, w, s) for t in held]
    for source in (other, x, other):
        for h, t in zip(held, source):
            h.copy_(t)
        graph.replay()
        replayed = [t.clone() for t in out]
        torch.cuda.synchronize()
        assert all(torch.equal(a, ops.linear_int8(t, w, s)) for a, t in zip(replayed, source))


def test_k_in_parts_captured():
    w, s = (t.to(DEV) for t in _weight(300, 8192, 6))
    x = _rows(40, 8192, torch.bfloat16, 7).to(DEV)
    held, sources = x.clone(), (x, x.flip(0) * 3)
    want = [ops.linear_int8(t, w, s) for t in sources]
    assert torch.equal(want[0], ops.linear_int8(x, w, s, tile=1))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_int8(held, w, s)
    for i in (1, 0, 1):
        held.copy_(sources[i])
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(replayed, want[i]) and torch.equal(ops.linear_int8(sources[i], w, s), want[i])


@pytest.mark.parametrize("k", [16, 100, 4096])
def test_integers_end_at_127(k):
    """Rows whose largest is a few of float32's smallest steps: their scale is one such step, or two, and quotients pass 127."""
    step = 2.0 ** -149
    x = torch.zeros(6, k)
    for m, top in enumerate((190, 127, 100, 64, 63, 191)):
        x[m, 0], x[m, k - 1], x[m, 3] = top * step, -top * step, 7 * step
    want, a = _quantised(x.clone())
    steps = torch.where(a[:, None] > 0, torch.round(x.double() / a.double()[:, None]), torch.zeros_like(x, dtype=torch.float64)).clamp(-127, 127)
    assert a.tolist() == [step, step, step, step, 0.0, 2 * step] and float(steps[0, 0]) == 127
    codes, scale = ops.quantize_rows(x.to(DEV))
    assert torch.equal(scale.cpu(), a) and torch.equal(codes.cpu().double(), steps)
    if k % 16:
        return
    w, s = _weight(20, k, 8)
    s = s * 2.0 ** 120
    exact = (steps @ w.double().t()) * a.double()[:, None] * s.double()
    for rows, tile in ((4, -1), (1, -1), (6, 0), (6, 3), (6, None)):
        if tile == 3 and k < 128:
            continue
        y = ops.linear_int8(x[:rows].to(DEV), w.to(DEV), s.to(DEV), tile=tile)
        off = (y.cpu().double() - exact[:rows]).abs()
        assert (off <= 3.01 * 2.0 ** -24 * exact[:rows].abs()).all(), (rows, tile)


def test_a_single_column_with_any_stride():
    """One output channel: the stride between rows of the weight counts for nothing."""
    x = _rows(5, 64, torch.bfloat16, 4)
    for stride in (64, 72, 4099):
        w, s = _weight(1, 64, 9, stride=stride)
        assert w.stride(0) == stride
        for rows in (1, 5):
            _check(x[:rows], w.clone(), s, None, torch.float32)
            given = torch.zeros(1, stride, dtype=torch.int8, device=DEV)
            given[:, :64] = w.to(DEV)
            y = ops.linear_int8(x[:rows].to(DEV), given[:, :64], s.to(DEV), out_dtype=torch.float32)
            assert torch.equal(y, ops.linear_int8(x[:rows].to(DEV), w.to(DEV).clone(memory_format=torch.contiguous_format), s.to(DEV), out_dtype=torch.float32))


def test_scales_that_are_subnormal():
    """Around the scales whose reciprocal float32 just holds, 2^-128, and the smallest normal one."""
    for k in (64, 100):
        x = _rows(9, k, torch.float32, 21 + k)
        x = x / x.abs().amax(1, keepdim=True) * 127
        x = x * 2.0 ** torch.tensor([-125.0, -126, -126.9, -127, -127.5, -128, -129, -135, -140])[:, None]
        codes, scale = ops.quantize_rows(x.to(DEV))
        want, a = _quantised(x)
        assert torch.equal(scale.cpu(), a) and torch.equal(codes.cpu(), want) and int(want.abs().max()) == 127


@pytest.mark.parametrize("pieces", [1, 2, 3, 4, 5, 6, 7, 8, 9, 12, 13, 16])
def test_pieces_in_flight(pieces):
    """Every number of pieces a wavefront, at its smallest and largest K, with an end inside a piece: up to four rows in one launch, and in two."""
    for k in (1024 * (pieces - 1) + 128, 1024 * pieces - 112, 1024 * pieces):
        for m, tile in ((1, -1), (3, -1), (9, 0)):
            if tile < 0 and k > 16384 // (1 if m == 1 else 4):
                continue
            x = _rows(m, k, torch.bfloat16, k + m)
            w, s = _weight(40, k, k)
            _check(x, w, s, None, torch.bfloat16, tile)
