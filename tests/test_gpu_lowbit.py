"""The low-bit operators on the GPU against their definitions in 64 bits (lowbit_reference.py).

Tolerances. Packed forms: none, every byte is defined. Products: the factors are exact, so a sum of K products in 32 bits is off by
at most K * 2^-23 of the sum of the products' magnitudes (each of K additions rounds, or truncates, once), and the result is rounded to its type
once: half a last place. Functions of one value: a few roundings in 32 bits, each relative to the quantity it rounds, 2^-19 of
(1 + |x|) times the factor that is multiplied on, and the type's rounding."""
import numpy as np
import pytest
import torch

import lowbit_reference as ref
from cntk_amd import QuantizerLogicError, lowbit

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
KINDS = sorted(lowbit.ACTIVATIONS)
HALF_PLACE = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def make(seed, rows, cols, dtype, spread=1.0):
    """Normal values, every column of a size of its own."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(cols, generator=g))
    return x.to(dtype).cuda()


def np64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, slack, dtype):
    """Every element within `slack` (absolute) and the type's rounding; NaN where NaN is wanted and nowhere else."""
    got, want = np64(got), np.asarray(want)
    assert got.shape == want.shape
    assert (np.isnan(got) == np.isnan(want)).all()
    allowed = slack + HALF_PLACE[dtype] * (np.abs(want) + slack) + SMALLEST[dtype]
    off = np.abs(got - want) - allowed
    off = off[~np.isnan(off)]
    assert off.size == 0 or off.max() <= 0, "off by up to %g more than allowed" % off.max()


def check_mx4(q, x):
    codes, scales, values = ref.mx4(np64(x))
    rows, cols = x.shape
    got_codes, got_scales = ref.unpack_mx4(q.buffer.cpu().numpy(), rows, cols)
    np.testing.assert_array_equal(got_scales[:rows, :scales.shape[1]], scales)
    np.testing.assert_array_equal(got_codes[:rows, :codes.shape[1]], codes)
    # what is beyond the matrix is zero
    assert not got_codes[rows:].any() and not got_codes[:, codes.shape[1]:].any()
    assert not got_scales[rows:].any() and not got_scales[:, scales.shape[1]:].any()
    return values


SHAPES = [(1, 1), (1, 32), (3, 33), (16, 128), (17, 129), (64, 429), (65, 257), (130, 1000), (5, 2049)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_four_bits(rows, cols, dtype):
    x = make(rows * 31 + cols, rows, cols, dtype)
    q = lowbit.mx4_quantize(x)
    values = check_mx4(q, x)
    for out in (torch.float32, torch.bfloat16):
        np.testing.assert_array_equal(np64(lowbit.mx4_dequantize(q, out)), values)
    # the transposed view of the transposed matrix: the same bytes
    assert torch.equal(lowbit.mx4_quantize(x.t().contiguous().t()).buffer, q.buffer)
    # rows at any element of a wider matrix, and columns two apart
    wide = torch.full((rows, 2 * cols + 3), float("nan"), dtype=dtype, device="cuda")
    wide[:, 1:1 + cols] = x
    assert torch.equal(lowbit.mx4_quantize(wide[:, 1:1 + cols]).buffer, q.buffer)
    wide[:, 1:1 + 2 * cols:2] = x
    assert torch.equal(lowbit.mx4_quantize(wide[:, 1:1 + 2 * cols:2]).buffer, q.buffer)


def special_blocks(dtype):
    """Blocks whose largest magnitude is every power of two of the type and its neighbours, with values at the rounding's ties around it;
    zeros of both signs, subnormals, infinities, NaN."""
    low, high = (-24, 15) if dtype == torch.float16 else (-149 if dtype == torch.float32 else -133, 127)
    rows = []
    for e in range(low, high + 1):
        top = 2.0 ** e
        rows.append([top] + [top * m / 8.0 * s for s in (1, -1) for m in (0.5, 0.75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.5)] + [-0.0])
        rows.append([top * 1.5, -top * 1.25] + [top * (k / 16.0) * (-1) ** k for k in range(30)])
        rows.append([top * 1.9921875, top * 1.75] + [top * (k / 15.0) for k in range(30)])
    rows.append([0.0] * 32)
    rows.append([-0.0] * 32)
    rows.append([float("inf")] + [1.0] * 31)
    rows.append([1.0] * 31 + [float("-inf")])
    rows.append([1.0] * 17 + [float("nan")] + [0.0] * 14)
    t = torch.tensor(rows, dtype=torch.float64)
    limit = torch.finfo(dtype).max
    return torch.where(t.isfinite(), t.clamp(-limit, limit), t).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_four_and_eight_bits_of_special_values(dtype):
    x = special_blocks(dtype).cuda()
    values = check_mx4(lowbit.mx4_quantize(x), x)
    np.testing.assert_array_equal(np64(lowbit.mx4_dequantize(lowbit.mx4_quantize(x), torch.float32)), values)
    check_mx4(lowbit.mx4_quantize(x.t().contiguous().t()), x)
    check_save8(lowbit.save8(x), x)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_four_and_eight_bits_of_every_sixteen_bit_value(dtype):
    bits = torch.arange(65536, dtype=torch.int32)
    every = bits.to(torch.int16).view(dtype)
    every = every[every.isfinite()]
    # neighbours in size share blocks; then each with a larger one (both types have a multiple of 32 finite values)
    x = every[every.float().abs().argsort()].view(-1, 32).cuda()
    check_mx4(lowbit.mx4_quantize(x), x)
    check_save8(lowbit.save8(x), x)
    for times in (3.0, 11.0):
        y = x.float()
        y[:, 0] = (y.abs().amax(-1) * times).clamp(max=torch.finfo(dtype).max)
        y = y.to(dtype)
        check_mx4(lowbit.mx4_quantize(y), y)
        check_save8(lowbit.save8(y), y)


# ---- products -------------------------------------------------------------------------------------


def product(xv, wv, bias):
    want = xv @ wv.T
    sizes = np.abs(xv) @ np.abs(wv).T
    slack = (xv.shape[1] + 1) * 2.0 ** -23 * (sizes + (0 if bias is None else np.abs(np64(bias))))
    return (want if bias is None else want + np64(bias)), slack


PRODUCTS = [(1, 1, 1), (1, 33, 40), (2, 128, 17), (16, 300, 64), (17, 429, 65), (64, 129, 130), (65, 257, 129), (128, 1024, 257),
            (200, 429, 300), (300, 160, 500), (513, 97, 33)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", PRODUCTS)
def test_products(m, k, n, dtype):
    x, w = make(m + k, m, k, dtype), make(k + n, n, k, dtype)
    bias = make(n, 1, n, dtype).view(n) if (m + n) % 2 else None
    xq, wq = lowbit.mx4_quantize(x), lowbit.mx4_quantize(w)
    want, slack = product(ref.mx4(np64(x))[2], ref.mx4(np64(w))[2], bias)
    for out in DTYPES:
        if np.abs(want).max() < torch.finfo(out).max:
            close(lowbit.mx4_matmul(xq, wq, bias, dtype=out), want, slack, out)
    if np.abs(want).max() < torch.finfo(dtype).max:
        y = lowbit.mx4_linear(x, wq, bias)
        assert y.dtype == dtype
        close(y, want, slack, dtype)
        kept_y, kept = lowbit.mx4_linear(x, wq, bias, save=True)
        close(kept_y, want, slack, dtype)
        assert torch.equal(kept.buffer, lowbit.save8(x).buffer)


def on_gpu(xq, wq, bias, dy, kept):
    """The products and weight gradients of what is packed, and what they may be off by, in 64 bits on the GPU."""
    a, b = lowbit.mx4_dequantize(xq, torch.float32).double(), lowbit.mx4_dequantize(wq, torch.float32).double()
    slack = (a.shape[1] + 1) * 2.0 ** -23
    yield a @ b.t() + bias.double(), slack * (a.abs() @ b.abs().t() + bias.double().abs())
    if dy is not None:
        x8, d = kept.values(torch.float32).double(), dy.double()
        yield d.t() @ x8, (3 * d.shape[0] + 1) * 2.0 ** -23 * (d.abs().t() @ x8.abs())


def near(got, want, slack):
    half = HALF_PLACE[got.dtype]
    assert ((got.double() - want).abs() <= slack + half * (want.abs() + slack) + SMALLEST[got.dtype]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m", [1, 5, 16])
@pytest.mark.parametrize("k,n", [(200, 4099), (333, 8205), (4700, 8192), (4701, 1000)])
def test_few_rows_of_many_columns(m, k, n, dtype):
    x, w, bias = make(m + k, m, k, dtype, 0.2), make(n, n, k, dtype, 0.2), make(n + 1, 1, n, dtype).view(n)
    wq = lowbit.mx4_quantize(w)
    (want, slack), = on_gpu(lowbit.mx4_quantize(x), wq, bias, None, None)
    near(lowbit.mx4_linear(x, wq, bias), want, slack)
    near(lowbit.mx4_linear(x, wq, bias, dtype=torch.float32), want, slack)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(600, 200, 1900), (1100, 300, 2050), (2049, 333, 1999), (65, 2047, 9301), (9301, 129, 2047), (2100, 513, 4097)])
def test_blocks_of_every_size(m, k, n, dtype):
    """Results of some thousand rows and columns, ragged on every side, as the rules deal them to blocks."""
    x, w, bias = make(1, m, k, dtype, 0.2), make(2, n, k, dtype, 0.2), make(3, 1, n, dtype).view(n)
    xq, wq = lowbit.mx4_quantize(x), lowbit.mx4_quantize(w)
    dy, kept = make(4, k, m, dtype, 0.2), lowbit.save8(w.t())
    (want, slack), (dw, dw_slack) = on_gpu(xq, wq, bias, dy, kept)
    for out in DTYPES:
        near(lowbit.mx4_matmul(xq, wq, bias, dtype=out), want, slack)
    got = lowbit.weight_gradient(dy, kept)
    near(got, dw, dw_slack)
    lowbit.weight_gradient(dy, kept, out=got, accumulate=True)
    near(got, 2 * dw, 3 * dw_slack)


def test_a_large_product():
    """More than 256 blocks of output tiles, ragged on every side."""
    m, k, n = 4113, 333, 4121
    x, w = make(1, m, k, torch.bfloat16), make(2, n, k, torch.bfloat16)
    xq, wq = lowbit.mx4_quantize(x), lowbit.mx4_quantize(w)
    a = lowbit.mx4_dequantize(xq, torch.float32).double()
    b = lowbit.mx4_dequantize(wq, torch.float32).double()
    want, sizes = (a @ b.t()).cpu().numpy(), (a.abs() @ b.abs().t()).cpu().numpy()
    close(lowbit.mx4_matmul(xq, wq, dtype=torch.float32), want, (k + 1) * 2.0 ** -23 * sizes, torch.float32)
    # an output within a wider matrix, at an odd place
    wide = torch.zeros(m, n + 6, dtype=torch.bfloat16, device="cuda")
    lowbit.mx4_matmul(xq, wq, out=wide[:, 3:3 + n])
    close(wide[:, 3:3 + n], want, (k + 1) * 2.0 ** -23 * sizes, torch.bfloat16)
    assert not wide[:, :3].any() and not wide[:, 3 + n:].any()


@pytest.mark.parametrize("m,k,n", [(1, 4100, 100), (40, 4100, 100), (192, 4100, 384), (2048, 2048, 2048), (4096, 1500, 4096)])
def test_long_inner_sides(m, k, n):
    """Many stages of the tile kernels, every result, several times over: a stage that is read before it has arrived shows as a result of
    other values."""
    x, w, dy = make(1, m, k, torch.bfloat16, 0.3), make(2, n, k, torch.bfloat16, 0.3), make(3, k, m, torch.bfloat16, 0.3)
    kept = lowbit.save8(w.t())
    xq, wq = lowbit.mx4_quantize(x), lowbit.mx4_quantize(w)
    factors = [(lowbit.mx4_dequantize(xq, torch.float32).double(), lowbit.mx4_dequantize(wq, torch.float32).double()),
               (dy.t().double(), kept.values(torch.float32).t().double())]
    for _ in range(3):
        results = lowbit.mx4_matmul(xq, wq, dtype=torch.float32), lowbit.weight_gradient(dy, kept)
        for (a, b), got in zip(factors, results):
            off = (got.double() - a @ b.t()).abs() - (k + 1) * 2.0 ** -23 * (a.abs() @ b.abs().t())
            assert off.max() <= 0


@pytest.mark.parametrize("m", [3, 40, 200])
def test_a_row_that_is_not_finite_stays_in_its_row(m):
    x, w = make(3, m, 300, torch.bfloat16), make(4, 70, 300, torch.bfloat16)
    want, slack = product(ref.mx4(np64(x))[2], ref.mx4(np64(w))[2], None)
    x[1, 77], x[m - 1, 299] = float("inf"), float("nan")
    want[[1, m - 1]] = np.nan
    close(lowbit.mx4_linear(x, lowbit.mx4_quantize(w)), want, slack, torch.bfloat16)
    w[5, 0] = float("nan")
    want[:, 5] = np.nan
    close(lowbit.mx4_linear(x, lowbit.mx4_quantize(w)), want, slack, torch.bfloat16)


@pytest.mark.parametrize("m", [1, 20, 100])
def test_products_of_the_extremes(m):
    """The largest and smallest scales, one against the other."""
    x = torch.zeros(m, 64, device="cuda")
    w = torch.zeros(20, 64, device="cuda")
    x[:, 0], w[:, 0] = 1.5 * 2.0 ** 127, 2.0 ** -126
    x[:, 40], w[:, 40] = 2.0 ** -120, 2.0 ** 120
    want, slack = product(ref.mx4(np64(x))[2], ref.mx4(np64(w))[2], None)
    assert (want == 4.0).all()
    close(lowbit.mx4_linear(x, lowbit.mx4_quantize(w)), want, slack, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(17, 40, 33), (100, 129, 70), (200, 429, 2048), (33, 2048, 500), (300, 257, 1030), (1030, 65, 513), (2050, 100, 60), (64, 2047, 2049), (129, 2048, 2048)])
def test_small_products_of_rows_as_they_are(m, k, n, dtype):
    """Some hundred rows, put into 4 bits by every workgroup for itself or once: the product of the two packed matrices, whatever the
    rows' stride."""
    x, w, bias = make(1, m, k, dtype, 0.2), make(2, n, k, dtype, 0.2), make(3, 1, n, dtype).view(n)
    wq = lowbit.mx4_quantize(w)
    a, b = (lowbit.mx4_dequantize(q, torch.float32).double() for q in (lowbit.mx4_quantize(x), wq))
    want, sizes = a @ b.t() + bias.double(), a.abs() @ b.abs().t() + bias.double().abs()
    y = lowbit.mx4_linear(x, wq, bias, dtype=torch.float32)
    assert ((y.double() - want).abs() <= (k + 2) * 2.0 ** -23 * sizes).all()
    wide = torch.full((m, k + 3), float("nan"), dtype=dtype, device="cuda")
    wide[:, 1:1 + k].copy_(x)
    assert torch.equal(lowbit.mx4_linear(wide[:, 1:1 + k], wq, bias, dtype=torch.float32), y)
    kept_y, kept = lowbit.mx4_linear(x, wq, bias, save=True, dtype=torch.float32)
    assert ((kept_y.double() - want).abs() <= (k + 2) * 2.0 ** -23 * sizes).all()
    assert torch.equal(kept.buffer, lowbit.save8(x).buffer)


def test_products_without_an_inner_side_and_empty_ones():
    bias = make(1, 1, 9, torch.float32).view(9)
    for m in (2, 100):
        y = lowbit.mx4_linear(torch.zeros(m, 0, device="cuda"), lowbit.mx4_quantize(torch.zeros(9, 0, device="cuda")), bias)
        assert torch.equal(y, bias.expand(m, 9))
    w = lowbit.mx4_quantize(make(2, 9, 40, torch.float32))
    y, kept = lowbit.mx4_linear(torch.zeros(0, 40, device="cuda"), w, save=True)
    assert y.shape == (0, 9)
    assert torch.equal(lowbit.weight_gradient(torch.zeros(0, 9, device="cuda"), kept), torch.zeros(9, 40, device="cuda"))
    empty = lowbit.mx4_quantize(torch.zeros(0, 40, device="cuda"))
    assert lowbit.mx4_linear(torch.zeros(5, 40, device="cuda"), empty).shape == (5, 0)
    assert lowbit.mx4_dequantize(empty).shape == (0, 40)


def test_rows_of_more_dimensions():
    x, w = make(5, 6, 40, torch.bfloat16).view(2, 3, 40), make(6, 10, 40, torch.bfloat16)
    q = lowbit.mx4_quantize(w)
    y, kept = lowbit.mx4_linear(x, q, save=True)
    assert y.shape == (2, 3, 10) and kept.shape == (2, 3, 40)
    assert torch.equal(y.view(6, 10), lowbit.mx4_linear(x.view(6, 40), q))
    assert torch.equal(lowbit.mx4_linear(x[0, 0], q), y[0, 0])
    dy = make(7, 6, 10, torch.bfloat16).view(2, 3, 10)
    assert torch.equal(lowbit.weight_gradient(dy, kept), lowbit.weight_gradient(dy.view(6, 10), lowbit.save8(x.view(6, 40))))
    # a gradient that was broadcast
    ones = torch.ones(1, 1, 1, dtype=torch.bfloat16, device="cuda").expand(2, 3, 10)
    assert torch.equal(lowbit.weight_gradient(ones, kept), lowbit.weight_gradient(torch.ones_like(dy), kept))


# ---- 8 bits ---------------------------------------------------------------------------------------


def check_save8(kept, x):
    codes, scales, values = ref.save8(np64(x))
    got_codes, got_scales = ref.unpack_save8(kept.buffer.cpu().numpy(), *x.shape)
    np.testing.assert_array_equal(got_scales, scales)
    np.testing.assert_array_equal(got_codes, codes)
    return values


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols", SHAPES + [(700, 31), (3, 9304)])
def test_eight_bits(rows, cols, dtype):
    x = make(rows * 37 + cols, rows, cols, dtype)
    kept = lowbit.save8(x)
    values = check_save8(kept, x)
    for out in (torch.float32, torch.bfloat16):
        np.testing.assert_array_equal(np64(kept.values(out)), values)
    wide = torch.full((rows, 2 * cols + 3), float("nan"), dtype=dtype, device="cuda")
    wide[:, 1:1 + cols] = x
    assert torch.equal(lowbit.save8(wide[:, 1:1 + cols]).buffer, kept.buffer)
    assert torch.equal(lowbit.save8(x.t().contiguous().t()).buffer, kept.buffer)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("kind", KINDS)
def test_activations(kind, dtype):
    for rows, cols in [(1, 1), (7, 33), (130, 429), (3, 2049)]:
        x, dy = make(rows + cols, rows, cols, dtype, 0.7), make(rows * cols, rows, cols, dtype, 0.3)
        y, kept = lowbit.activation_forward(kind, x)
        x8 = check_save8(kept, x)
        f, _ = ref.activation(kind, np64(x))
        close(y, f, 2.0 ** -19 * (1 + np.abs(np64(x))) * (kind != "relu"), dtype)
        _, d = ref.activation(kind, x8)
        near = 2.0 ** -19 * (1 + np.abs(x8)) * (kind != "relu")
        close(lowbit.activation_backward(dy, kept), np64(dy) * d, np.abs(np64(dy)) * near, dtype)
        # gated
        gate = make(rows + 5 * cols, rows, cols, dtype, 0.7)
        y, kept = lowbit.activation_forward(kind, x, gate)
        check_save8(kept, x)
        g, x_, dy_ = np64(gate), np64(x), np64(dy)
        f, _ = ref.activation(kind, g)
        close(y, f * x_, np.abs(x_) * 2.0 ** -19 * (1 + np.abs(g)), dtype)
        _, g8 = kept.values(torch.float32)
        g8 = np64(g8)
        np.testing.assert_array_equal(g8, ref.save8(g)[2])
        f, d = ref.activation(kind, g8)
        dx, dgate = lowbit.activation_backward(dy, kept)
        near = 2.0 ** -19 * (1 + np.abs(g8))
        close(dx, dy_ * f, np.abs(dy_) * near, dtype)
        close(dgate, dy_ * x8 * d, np.abs(dy_ * x8) * near, dtype)


@pytest.mark.parametrize("kind", KINDS)
def test_activation_gradient_against_differences(kind):
    """A step of 2^-4 either way between values that the 8-bit form holds (multiples of 2^-5 below 4): the slope of the forward pass's own
    results is off by step^2 / 6 times the third derivative (2 at most for these functions) and by the results' rounding over the step."""
    x = (torch.arange(-96, 96, device="cuda") / 32.0 + 1.0 / 64.0).view(6, 32)
    step = 2.0 ** -4
    up, _ = lowbit.activation_forward(kind, x + step)
    down, _ = lowbit.activation_forward(kind, x - step)
    slope = (np64(up) - np64(down)) / (2 * step)
    x[:, 31] = 3.999  # every block's largest magnitude: its 8 bits are multiples of 2^-5, and x lies half a step off one
    _, kept = lowbit.activation_forward(kind, x)
    d = np64(lowbit.activation_backward(torch.ones_like(x), kept))
    away = np.abs(np64(kept.values()) - np64(x))
    allowed = step ** 2 / 6 * 2.0 + 2.0 ** -18 / step + away * 1.0  # (no second derivative is above 1)
    smooth = np.abs(np64(x)) > step + 2.0 ** -5 if kind == "relu" else np.ones(x.shape, bool)
    assert (np.abs(slope - d) <= allowed)[:, :31][smooth[:, :31]].all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(5, 8), (131, 40), (67, 2048), (3, 4104)])
def test_activations_of_whole_eights(rows, cols, kind, dtype):
    """Widths that are a multiple of eight take kernels of their own: a ragged last block, a row on all lanes of a workgroup, one on several; rows
    that leave a workgroup partly empty. Inputs as they lie and as columns of a wider matrix, at any element."""
    x, gate, dy = make(rows, rows, cols, dtype, 0.7), make(rows + 1, rows, cols, dtype, 0.7), make(rows + 2, rows, cols, dtype, 0.3)
    x64, g64, dy64 = np64(x), np64(gate), np64(dy)
    x8, g8 = ref.save8(x64)[2], ref.save8(g64)[2]
    smooth = 2.0 ** -19 * (kind != "relu")

    def inside(t):
        wide = torch.full((rows, cols + 5), float("nan"), dtype=dtype, device="cuda")
        wide[:, 3:3 + cols] = t
        return wide[:, 3:3 + cols]

    f, _ = ref.activation(kind, x64)
    _, d = ref.activation(kind, x8)
    for given, back in ((x, dy), (inside(x), inside(dy))):
        y, kept = lowbit.activation_forward(kind, given)
        check_save8(kept, x)
        close(y, f, smooth * (1 + np.abs(x64)), dtype)
        close(lowbit.activation_backward(back, kept), dy64 * d, np.abs(dy64) * smooth * (1 + np.abs(x8)), dtype)
    f, _ = ref.activation(kind, g64)
    f8, d8 = ref.activation(kind, g8)
    for given, by, back in ((x, gate, dy), (inside(x), inside(gate), inside(dy))):
        y, kept = lowbit.activation_forward(kind, given, by)
        check_save8(kept, x)
        codes, scales = ref.unpack_save8(kept.gate.cpu().numpy(), rows, cols)
        np.testing.assert_array_equal(codes, ref.save8(g64)[0])
        np.testing.assert_array_equal(scales, ref.save8(g64)[1])
        close(y, f * x64, np.abs(x64) * 2.0 ** -19 * (1 + np.abs(g64)), dtype)
        dx, dgate = lowbit.activation_backward(back, kept)
        near = 2.0 ** -19 * (1 + np.abs(g8))
        close(dx, dy64 * f8, np.abs(dy64) * near, dtype)
        close(dgate, dy64 * x8 * d8, np.abs(dy64 * x8) * near, dtype)


def test_exponentials_keep_their_places():
    """Sigmoid and SiLU far below zero in single precision, where an absolute bound asks for nothing. e^-x: its last place (2^-23) and half a place where the
    remainder is multiplied on; half a place each for the sum and the quotient: 2^-21.6 of the result. The slopes take that factor and one that is
    within 2^-21.7 of itself (sigmoid: 1 - f of f up to a half; SiLU: 1 + x (1 - f), whose terms cancel by a third at most below -3) and round their
    product: 2^-20.5. Each bound is taken at the next power of two."""
    x = -torch.linspace(3.0, 85.0, 32 * 4096, device="cuda").view(4096, 32)
    a = np64(x)
    for kind in ("sigmoid", "silu"):
        y, kept = lowbit.activation_forward(kind, x)
        f, _ = ref.activation(kind, a)
        assert (np.abs(np64(y) - f) <= 2.0 ** -21 * np.abs(f)).all()
        _, d = ref.activation(kind, np64(kept.values()))
        got = np64(lowbit.activation_backward(torch.ones_like(x), kept))
        assert (np.abs(got - d) <= 2.0 ** -20 * np.abs(d)).all()
        # gated, the function is a factor
        y, kept = lowbit.activation_forward(kind, torch.ones_like(x), x)
        assert (np.abs(np64(y) - f) <= 2.0 ** -21 * np.abs(f)).all()
    # where it is 0 or infinite
    far = torch.tensor([[-1e30, -3.4e38, -200.0, -89.0, 89.0, 200.0, 1e30, 3.4e38, float("inf"), float("-inf"), float("nan")]], device="cuda")
    y, _ = lowbit.activation_forward("sigmoid", far)
    assert torch.equal(y[0, 4:9], torch.ones(5, device="cuda")) and float(y[0, :4].abs().max()) < 1e-37 and y[0, 9] == 0.0 and torch.isnan(y[0, 10])
    y, _ = lowbit.activation_forward("silu", far)
    assert torch.equal(y[0, 4:9], far[0, 4:9]) and float(y[0, :4].abs().max()) < 1e-35
    _, kept = lowbit.activation_forward("sigmoid", far[:, :8].repeat_interleave(32, 1))
    assert float(lowbit.activation_backward(torch.ones(1, 256, device="cuda"), kept).abs().max()) < 1e-37


# ---- weight gradients -----------------------------------------------------------------------------


def check_weight_gradient(dw, db, dy, x8, dw0=0.0, db0=0.0):
    dy = np64(dy)
    m = dy.shape[0]
    slack = (3 * m + 1) * 2.0 ** -23
    close(dw, dy.T @ x8 + dw0, slack * (np.abs(dy).T @ np.abs(x8) + np.abs(dw0)), torch.float32)
    if db is not None:
        close(db, dy.sum(0) + db0, (m + 1) * 2.0 ** -23 * (np.abs(dy).sum(0) + np.abs(db0)), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 40, 33), (2, 33, 300), (31, 129, 65), (257, 429, 130), (300, 64, 257), (1030, 100, 40), (64, 2049, 5)])
def test_weight_gradients(m, k, n, dtype):
    x, dy = make(m + k, m, k, dtype), make(m + n, m, n, dtype)
    kept = lowbit.save8(x)
    x8 = ref.save8(np64(x))[2]
    dw, db = lowbit.weight_gradient(dy, kept, bias=True)
    check_weight_gradient(dw, db, dy, x8)
    assert torch.equal(lowbit.weight_gradient(dy, kept), dw)  # the same sums in the same order
    # added to what is there, within a wider matrix at an odd place
    wide = torch.zeros(n, k + 5, device="cuda")
    at = wide[:, 3:3 + k]
    at.copy_(make(9, n, k, torch.float32))
    dw0, db0 = np64(at), make(10, 1, n, torch.float32).view(n)
    db0_ = np64(db0)
    lowbit.weight_gradient(dy, kept, bias=True, out=(at, db0), accumulate=True)
    check_weight_gradient(at, db0, dy, x8, dw0, db0_)
    assert not wide[:, :3].any() and not wide[:, 3 + k:].any()
    # rows of a wider gradient
    if dy.shape[1] > 1:
        check_weight_gradient(lowbit.weight_gradient(dy[:, 1:], kept), None, dy[:, 1:], x8)


@pytest.mark.parametrize("m,k,n", [(1, 1000, 1288), (33, 264, 4104), (70, 1032, 1024), (257, 700, 2056), (300, 136, 9304), (64, 4100, 1000), (95, 2050, 5000)])
def test_weight_gradients_from_gradients_as_they_lie(m, k, n):
    """Many results of bfloat16 gradients, whose rows may be whole 16 bytes or not: the same sums in the same order. What lies around
    the gradient in memory does not matter."""
    x = make(1, m, k, torch.bfloat16)
    kept, x8 = lowbit.save8(x), ref.save8(np64(x))[2]
    near = make(2, m, n, torch.bfloat16)
    dw, db = lowbit.weight_gradient(near, kept, bias=True)
    check_weight_gradient(dw, db, near, x8)
    for before, after in ((8, 0), (0, 8), (16, 40), (4, 4), (1, 0)):
        wide = torch.full((m, before + n + after), float("nan"), dtype=torch.bfloat16, device="cuda")
        dy = wide[:, before:before + n]
        dy.copy_(near)
        got, got_db = lowbit.weight_gradient(dy, kept, bias=True)
        assert torch.equal(got, dw) and torch.equal(got_db, db)
    assert torch.equal(lowbit.weight_gradient(near, kept), dw)
    dw0, db0 = make(3, n, k, torch.float32), make(4, 1, n, torch.float32).view(n)
    at, at_db = dw0.clone(), db0.clone()
    lowbit.weight_gradient(near, kept, bias=True, out=(at, at_db), accumulate=True)
    check_weight_gradient(at, at_db, near, x8, np64(dw0), np64(db0))
    # one row for all, and an infinity and a NaN that reach their own rows of dw
    same = near[:1].expand(m, n)
    check_weight_gradient(lowbit.weight_gradient(same, kept), None, same, x8)
    near[m // 2, 9], near[0, n - 1] = float("inf"), float("nan")
    bad = ~torch.isfinite(lowbit.weight_gradient(near, kept))
    assert bad[n - 1].all() and int(bad.sum()) == k + int(bad[9].sum())


@pytest.mark.parametrize("m", [1, 31, 64, 70, 95, 257])
@pytest.mark.parametrize("k,n", [(1000, 1288), (264, 4104), (700, 2056), (136, 9304), (2050, 5000)])
def test_weight_gradients_do_not_see_the_rows_below(m, k, n):
    """The gradient's rows are the first ones of a taller matrix, whose other rows hold NaN and infinities: whole stages of the product end
    beyond the last row, and what lies there takes no part."""
    kept = lowbit.save8(make(1, m, k, torch.bfloat16))
    near = make(2, m, n, torch.bfloat16)
    dw, db = lowbit.weight_gradient(near, kept, bias=True)
    assert torch.isfinite(dw).all() and torch.isfinite(db).all()
    for beside in (0, 24):
        tall = torch.full((m + 160, n + beside), float("nan"), dtype=torch.bfloat16, device="cuda")
        tall[m + 1::2] = float("inf")
        tall[:m, :n] = near
        got, got_db = lowbit.weight_gradient(tall[:m, :n], kept, bias=True)
        assert torch.equal(got, dw) and torch.equal(got_db, db)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(1300, 2, 100001), (1300, 100001, 2), (1500, 16, 20000), (1025, 33, 9303), (1030, 64, 20001), (700, 30001, 60), (1100, 700, 900),
                                   (1024, 900, 900), (2000, 500, 500), (1200, 2000, 1000), (96, 1900, 1101), (300, 70000, 1), (65, 1, 70000)])
def test_weight_gradients_by_their_shape(m, k, n, dtype):
    """Few results and many, of few rows and many, narrow on either side: every way that one is made, each with its column sums."""
    x, dy = make(1, m, k, dtype, 0.3), make(2, m, n, dtype, 0.3)
    kept = lowbit.save8(x)
    a, b = dy.double(), kept.values(torch.float32).double()
    want, sizes, sums, sum_sizes = a.t() @ b, a.abs().t() @ b.abs(), a.sum(0), a.abs().sum(0)
    dw, db = lowbit.weight_gradient(dy, kept, bias=True)
    slack = (3 * m + 2) * 2.0 ** -23
    assert ((dw.double() - want).abs() <= slack * sizes).all()
    assert ((db.double() - sums).abs() <= slack * sum_sizes).all()
    assert torch.equal(lowbit.weight_gradient(dy, kept), dw)
    lowbit.weight_gradient(dy, kept, bias=True, out=(dw, db), accumulate=True)
    assert ((dw.double() - 2.0 * want).abs() <= 3.0 * slack * sizes).all()
    assert ((db.double() - 2.0 * sums).abs() <= 3.0 * slack * sum_sizes).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,n", [(40, 9), (1500, 5000), (3, 1), (33, 300000), (0, 7)])
def test_column_sums_of_a_layer_without_inputs(m, n, dtype):
    dy = make(1, max(m, 1), n, dtype)[:m]
    dw, db = lowbit.weight_gradient(dy, lowbit.save8(torch.zeros(m, 0, dtype=dtype, device="cuda")), bias=True)
    assert dw.shape == (n, 0)
    a = dy.double()
    assert ((db.double() - a.sum(0)).abs() <= (m + 1) * 2.0 ** -23 * a.abs().sum(0)).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m", [0, 1, 40, 1024, 1025, 5000])
def test_layers_without_results(m, dtype):
    """No columns of the gradient, of any number of rows; then no rows."""
    x = make(1, max(m, 1), 40, dtype)[:m]
    w = lowbit.mx4_quantize(torch.zeros(0, 40, dtype=dtype, device="cuda"))
    y, kept = lowbit.mx4_linear(x, w, save=True)
    assert y.shape == (m, 0) and lowbit.mx4_linear(x, w).shape == (m, 0)
    assert torch.equal(kept.buffer, lowbit.save8(x).buffer)
    dw, db = lowbit.weight_gradient(torch.zeros(m, 0, dtype=dtype, device="cuda"), kept, bias=True)
    assert dw.shape == (0, 40) and db.shape == (0,)
    assert lowbit.weight_gradient(torch.zeros(m, 0, dtype=dtype, device="cuda"), kept, out=dw, accumulate=True) is dw
    # the input gradient: a product without an inner side
    dx = lowbit.mx4_linear(torch.zeros(m, 0, dtype=dtype, device="cuda"), lowbit.mx4_quantize(torch.zeros(40, 0, dtype=dtype, device="cuda")))
    assert dx.shape == (m, 40) and not dx.any()


def test_a_large_weight_gradient():
    m, k, n = 70, 4100, 4200
    x, dy = make(1, m, k, torch.bfloat16), make(2, m, n, torch.bfloat16)
    kept = lowbit.save8(x)
    dw, db = lowbit.weight_gradient(dy, kept, bias=True)
    a, b = dy.double(), kept.values(torch.float32).double()
    want, sizes = (a.t() @ b).cpu().numpy(), (a.abs().t() @ b.abs()).cpu().numpy()
    close(dw, want, (m + 1) * 2.0 ** -23 * sizes, torch.float32)
    close(db, np64(dy).sum(0), (m + 1) * 2.0 ** -23 * np.abs(np64(dy)).sum(0), torch.float32)


def test_a_weight_gradient_of_more_rows_than_one_pair_of_launches_takes():
    m, k, n = (1 << 21) + 77, 40, 19
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(m, k, generator=g, device="cuda", dtype=torch.bfloat16)
    dy = torch.randn(m, n, generator=g, device="cuda", dtype=torch.bfloat16)
    kept = lowbit.save8(x)
    a, b = dy.double(), kept.values(torch.float32).double()
    for _ in range(2):
        dw, db = lowbit.weight_gradient(dy, kept, bias=True)
        # millions of rows: the products' roundings are taken as independent, four times the root of their number
        assert ((dw.double() - a.t() @ b).abs() <= 4 * 2.0 ** -23 * m ** 0.5 * (a.abs().t() @ b.abs()).max()).all()
        assert ((db.double() - a.sum(0)).abs() <= 4 * 2.0 ** -23 * m ** 0.5 * a.abs().sum(0).max()).all()


def whole_numbers(seed, rows, cols, most, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-most, most + 1, (rows, cols), generator=g, device="cuda", dtype=torch.int8).to(dtype)


@pytest.mark.parametrize("dtype,n", [(torch.bfloat16, 520), (torch.bfloat16, 521), (torch.float16, 520)], ids=["bf16 as it lies", "bf16 turned", "f16 turned"])
def test_a_weight_gradient_in_several_pairs_of_launches(dtype, n):
    """Many results of more than 2^21 rows: the second piece's rows, codes and scales, added to the first one's results. Whole numbers, so small that every
    product and sum in 32 bits is exact, whatever the order."""
    m, k = (1 << 21) + 77, 2024
    x, dy = whole_numbers(1, m, k, 3, torch.bfloat16), whole_numbers(2, m, n, 2, dtype)
    x[:, ::32] *= torch.where(torch.arange(m, device="cuda") % 3 == 0, 20.0, 1.0).to(torch.bfloat16)[:, None]  # scales that differ from row to row
    kept = lowbit.save8(x)
    want, sums = torch.zeros(n, k, device="cuda"), torch.zeros(n, device="cuda")
    for row in range(0, m, 1 << 18):
        a, b = dy[row:row + (1 << 18)].float(), x[row:row + (1 << 18)].float()
        want += a.t().contiguous() @ b
        sums += a.sum(0)
    assert float(want.abs().max()) < 2 ** 23
    dw, db = lowbit.weight_gradient(dy, kept, bias=True)
    assert torch.equal(dw, want) and torch.equal(db, sums)
    lowbit.weight_gradient(dy, kept, bias=True, out=(dw, db), accumulate=True)
    assert torch.equal(dw, 2.0 * want) and torch.equal(db, 2.0 * sums)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [24, 23])
def test_column_sums_in_several_pairs_of_launches(n, dtype):
    m = (1 << 22) + 1
    dy = whole_numbers(3, m, n, 2, dtype)
    sums = dy.double().sum(0).float()
    kept = lowbit.save8(torch.zeros(m, 0, dtype=dtype, device="cuda"))
    dw, db = lowbit.weight_gradient(dy, kept, bias=True)
    assert dw.shape == (n, 0) and torch.equal(db, sums)
    lowbit.weight_gradient(dy, kept, bias=True, out=(dw, db), accumulate=True)
    assert torch.equal(db, 2.0 * sums)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", [(40, 64, 50), (1100, 40, 30), (40, 1500, 1501)])
def test_weight_gradients_of_the_smallest_values(m, k, n, dtype):
    """Gradients and kept inputs down to the smallest number of the type, subnormal ones among them, against large factors. Of a single-precision gradient the
    bits below 2^-133 are not multiplied; everything else is."""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    low, high = (-24, 10) if dtype == torch.float16 else (-149, -99)
    dy = torch.randn(m, n, generator=g, device="cuda") * torch.exp2(torch.randint(low, high, (m, n), generator=g, device="cuda").float())
    dy = dy.to(dtype)
    assert torch.isfinite(dy).all()
    kept = lowbit.save8(torch.randn(m, k, generator=g, device="cuda") * 2.0 ** 30)
    a, b = dy.double(), kept.values(torch.float32).double()
    want, sizes = a.t() @ b, a.abs().t() @ b.abs()
    left_out = 2.0 ** -133 * b.abs().sum(0) if dtype == torch.float32 else 0.0
    got = lowbit.weight_gradient(dy, kept)
    assert ((got.double() - want).abs() <= (3 * m + 1) * 2.0 ** -23 * sizes + left_out + (3 * m + 1) * 2.0 ** -149).all()
    # the smallest kept inputs
    x = torch.randn(m, k, generator=g, device="cuda") * torch.exp2(torch.randint(-149, -100, (m, k // 2), generator=g, device="cuda").float()).repeat(1, 2)
    kept = lowbit.save8(x)
    dy = (torch.randn(m, n, generator=g, device="cuda") * 2.0 ** 14).to(dtype).clamp(-60000.0, 60000.0)
    a, b = dy.double(), kept.values(torch.float32).double()
    want, sizes = a.t() @ b, a.abs().t() @ b.abs()
    assert float(want.abs().max()) > 0.0
    assert ((lowbit.weight_gradient(dy, kept).double() - want).abs() <= (3 * m + 1) * 2.0 ** -23 * sizes + (3 * m + 1) * 2.0 ** -149).all()


def test_weight_gradients_of_what_is_not_finite():
    """An infinity or a NaN of dy reaches its own row of dw; one of x its block's columns."""
    for dtype in DTYPES:
        x, dy = make(1, 40, 100, dtype), make(2, 40, 50, dtype)
        dy[3, 7], dy[5, 8] = float("inf"), float("nan")
        dw, db = lowbit.weight_gradient(dy, lowbit.save8(x), bias=True)
        bad = ~torch.isfinite(dw)
        assert bad[7].all() and bad[8].all() and int(bad.sum()) == 200
        assert torch.isinf(db[7]) and torch.isnan(db[8]) and int((~torch.isfinite(db)).sum()) == 2
        dy, x = make(2, 40, 50, dtype), x.clone()
        x[4, 33] = float("inf")
        bad = torch.isnan(lowbit.weight_gradient(dy, lowbit.save8(x)))
        assert bad[:, 32:64].all() and int(bad.sum()) == 50 * 32
    big = torch.full((2, 4), 3.4e38, device="cuda")  # above the largest bfloat16, a finite number all the same
    dw = lowbit.weight_gradient(big, lowbit.save8(torch.full((2, 4), 2.0 ** -10, device="cuda")))
    np.testing.assert_allclose(np64(dw), np64(big)[:1].repeat(4, 0) * 2.0 ** -9, rtol=2.0 ** -22)


# ---- streams, graphs, offsets, refusals -----------------------------------------------------------


def step(x, dy, w, w_t, bias, dw, db):
    """The whole of a layer with a gated unit behind it."""
    y, kept = lowbit.mx4_linear(x, w, bias, save=True)
    z, kept_z = lowbit.activation_forward("silu", y, y)
    dz, dg = lowbit.activation_backward(dy, kept_z)
    dx = lowbit.mx4_linear(dz, w_t)
    lowbit.weight_gradient(dg, kept, bias=True, out=(dw, db))
    few = lowbit.mx4_linear(x[:4], w, bias)
    return [y, z, dz, dg, dx, dw, db, few, lowbit.mx4_dequantize(lowbit.mx4_quantize(x))]


def test_other_streams_and_graphs():
    m, k, n = 150, 200, 300
    x, dy, w = make(1, m, k, torch.bfloat16), make(2, m, n, torch.bfloat16), make(3, n, k, torch.bfloat16, 0.1)
    bias = make(4, 1, n, torch.bfloat16).view(n)
    dw, db = torch.empty(n, k, device="cuda"), torch.empty(n, device="cuda")
    q, q_t = lowbit.mx4_quantize(w), lowbit.mx4_quantize(w.t())
    want = [t.clone() for t in step(x, dy, q, q_t, bias, dw, db)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, dy, q, q_t, bias, dw, db)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, dy, q, q_t, bias, dw, db)
    for seed in (11, 12, 13):
        x.copy_(make(seed, m, k, torch.bfloat16))
        dy.copy_(make(seed + 50, m, n, torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        eager = step(x, dy, q, q_t, bias, dw, db)
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_offsets_beyond_32_bits():
    """Rows so far apart that their offsets pass 2^32 elements."""
    apart = (1 << 31) + 24
    store = torch.empty(2 * apart + 64, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(store, (3, 40), (apart, 1))
    x.copy_(make(1, 3, 40, torch.bfloat16))
    near = x.contiguous()
    q = lowbit.mx4_quantize(near)
    assert torch.equal(lowbit.mx4_quantize(x).buffer, q.buffer)
    assert torch.equal(lowbit.mx4_quantize(x.t()).buffer, lowbit.mx4_quantize(near.t()).buffer)
    assert torch.equal(lowbit.save8(x).buffer, lowbit.save8(near).buffer)
    w = lowbit.mx4_quantize(make(2, 33, 40, torch.bfloat16))
    want = lowbit.mx4_linear(near, w)
    assert torch.equal(lowbit.mx4_linear(x, w), want)
    kept = lowbit.save8(make(3, 3, 50, torch.bfloat16))
    assert torch.equal(lowbit.weight_gradient(x, kept), lowbit.weight_gradient(near, kept))
    y, kept = lowbit.activation_forward("gelu", x, x)
    y2, kept2 = lowbit.activation_forward("gelu", near, near)
    assert torch.equal(y, y2) and torch.equal(kept.gate, kept2.gate)
    assert torch.equal(lowbit.activation_backward(x, kept)[0], lowbit.activation_backward(near, kept2)[0])
    out = torch.as_strided(store, (3, 33), (apart, 1))
    lowbit.mx4_matmul(q, w, out=out)
    assert torch.equal(out, want)


def test_refusals():
    x, w = make(1, 20, 40, torch.bfloat16), make(2, 30, 40, torch.bfloat16)
    q = lowbit.mx4_quantize(w)
    kept = lowbit.save8(x)
    refused = [
        lambda: lowbit.mx4_quantize(x.cpu()),
        lambda: lowbit.mx4_quantize(x.double()),
        lambda: lowbit.mx4_quantize(torch.tensor(1.0, device="cuda")),
        lambda: lowbit.mx4_quantize(x, out=lowbit.Mx4Matrix(20, 41)),
        lambda: lowbit.Mx4Matrix(20, 40, torch.empty(7, dtype=torch.uint8, device="cuda")),
        lambda: lowbit.mx4_dequantize(q, torch.float64),
        lambda: lowbit.mx4_linear(x[:, :39], q),
        lambda: lowbit.mx4_linear(x, q, bias=x[0]),
        lambda: lowbit.mx4_linear(x, q, bias=torch.zeros(30)),
        lambda: lowbit.mx4_linear(x, q, dtype=torch.int8),
        lambda: lowbit.mx4_linear(x, q, out=torch.empty(20, 31, dtype=torch.bfloat16, device="cuda")),
        lambda: lowbit.mx4_matmul(q, lowbit.mx4_quantize(make(3, 5, 41, torch.bfloat16))),
        lambda: lowbit.mx4_matmul(q, q, out=torch.empty(30, 30, device="cuda")),
        lambda: lowbit.mx4_matmul(q, q, out=torch.empty(30, 30, dtype=torch.bfloat16, device="cuda").t()),
        lambda: lowbit.mx4_matmul(q, q, out=torch.empty(1, 30, dtype=torch.bfloat16, device="cuda").expand(30, 30)),
        lambda: lowbit.activation_forward("softplus", x),
        lambda: lowbit.activation_forward("relu", x, x.float()),
        lambda: lowbit.activation_forward("relu", x, x[:5]),
        lambda: lowbit.activation_backward(x, kept),
        lambda: lowbit.activation_backward(x.float(), lowbit.activation_forward("relu", x)[1]),
        lambda: lowbit.weight_gradient(x[:19], kept),
        lambda: lowbit.weight_gradient(x, lowbit.activation_forward("relu", x)[1]),
        lambda: lowbit.weight_gradient(x, kept, accumulate=True),
        lambda: lowbit.weight_gradient(x, kept, out=torch.empty(40, 41, device="cuda")),
        lambda: lowbit.LowBitActivation("swish"),
    ]
    for call in refused:
        with pytest.raises(QuantizerLogicError):
            call()


def writes(x, dy, q, kept):
    """(name, call with an out, a new out) of every function that writes into the caller's tensors."""
    def new(*sizes):
        return torch.zeros(*sizes, device="cuda")

    return [("dequantize", lambda out: lowbit.mx4_dequantize(q, torch.float32, out=out), lambda: new(30, 40)),
            ("matmul", lambda out: lowbit.mx4_matmul(q, q, dtype=torch.float32, out=out), lambda: new(30, 30)),
            ("linear", lambda out: lowbit.mx4_linear(x, q, out=out), lambda: new(20, 30)),
            ("linear that keeps x", lambda out: lowbit.mx4_linear(x, q, save=True, out=out), lambda: new(20, 30)),
            ("dw", lambda out: lowbit.weight_gradient(dy, kept, out=out), lambda: new(30, 40)),
            ("dw of a pair", lambda out: lowbit.weight_gradient(dy, kept, bias=True, out=(out, None)), lambda: new(30, 40)),
            ("db of a pair", lambda out: lowbit.weight_gradient(dy, kept, bias=True, out=(None, out)), lambda: new(30))]


def test_what_is_written_is_known_to_autograd():
    x, dy = make(1, 20, 40, torch.float32), make(2, 20, 30, torch.float32)
    q, kept = lowbit.mx4_quantize(make(3, 30, 40, torch.float32)), lowbit.save8(x)
    for name, call, new in writes(x, dy, q, kept):
        out = new()
        before = out._version
        call(out)
        assert out._version == before + 1, name
        # another operator saved it for its backward pass: that must not go on with other values
        factor = torch.ones_like(out, requires_grad=True)
        loss = (factor * out).sum()
        call(out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
        # part of a graph, as a leaf and as a view of one
        for leaf in (new().requires_grad_(), new().requires_grad_().view(out.shape)):
            with pytest.raises(QuantizerLogicError):
                call(leaf)
            assert not leaf.detach().any(), name
            with torch.no_grad():
                call(leaf)
            assert torch.equal(leaf.detach(), out)
        with torch.inference_mode():
            inner = new()
            call(inner)
        assert torch.equal(inner, out)
        with pytest.raises(QuantizerLogicError):
            call(inner)
    # a refused call has written nothing, and says nothing else
    out = torch.zeros(20, 31, device="cuda")
    with pytest.raises(QuantizerLogicError):
        lowbit.mx4_linear(x, q, out=out)
    assert out._version == 0
    matrix = lowbit.Mx4Matrix(20, 40)
    before = matrix.buffer._version
    lowbit.mx4_quantize(x, out=matrix)
    assert matrix.buffer._version == before + 1


def test_results_share_no_memory_with_the_rest_of_a_call():
    square = lowbit.mx4_quantize(make(1, 40, 40, torch.float32))
    x = make(2, 40, 40, torch.float32)
    kept = lowbit.save8(x)
    store = torch.zeros(1 << 16, device="cuda")

    def at(offset, rows, cols, stride):
        return store.as_strided((rows, cols), (stride, 1), offset)

    refused = [
        lambda: lowbit.mx4_linear(x, square, out=x),
        lambda: lowbit.mx4_linear(at(0, 40, 40, 40), square, out=at(1599, 40, 40, 40)),
        lambda: lowbit.mx4_linear(at(1600, 40, 40, 40), square, out=at(1, 40, 40, 40)),
        lambda: lowbit.mx4_linear(at(0, 40, 40, 100), square, out=at(39, 40, 40, 100)),  # one column
        lambda: lowbit.mx4_linear(at(0, 40, 40, 100), square, out=at(61, 40, 40, 100)),  # the next row's first one
        lambda: lowbit.mx4_linear(at(0, 40, 40, 100), square, out=at(40, 40, 40, 120)),  # rows that come nearer
        lambda: lowbit.mx4_linear(at(0, 1, 40, 40).expand(40, 40), square, out=at(0, 40, 40, 40)),
        lambda: lowbit.mx4_linear(x, square, at(0, 1, 40, 40)[0], out=at(0, 40, 40, 40)),
        lambda: lowbit.mx4_linear(x, lowbit.Mx4Matrix(40, 40, store.view(torch.uint8)[:square.buffer.numel()]), out=at(0, 40, 40, 40)),
        lambda: lowbit.mx4_matmul(square, lowbit.Mx4Matrix(40, 40, store.view(torch.uint8)[:square.buffer.numel()]), dtype=torch.float32, out=at(0, 40, 40, 40)),
        lambda: lowbit.mx4_matmul(square, square, at(0, 1, 40, 40)[0], dtype=torch.float32, out=at(0, 40, 40, 40)),
        lambda: lowbit.mx4_dequantize(lowbit.Mx4Matrix(40, 40, store.view(torch.uint8)[:square.buffer.numel()]), torch.float32, out=at(9, 40, 40, 40)),
        lambda: lowbit.mx4_quantize(at(0, 40, 40, 40), out=lowbit.Mx4Matrix(40, 40, store.view(torch.uint8)[:square.buffer.numel()])),
        lambda: lowbit.mx4_quantize(at(0, 40, 40, 40).t(), out=lowbit.Mx4Matrix(40, 40, store.view(torch.uint8)[:square.buffer.numel()])),
        lambda: lowbit.weight_gradient(at(0, 40, 40, 40), kept, out=at(40, 40, 40, 40)),
        lambda: lowbit.weight_gradient(at(0, 40, 40, 40), kept, bias=True, out=(None, store[1599:1639])),
        lambda: lowbit.weight_gradient(x, kept, bias=True, out=(at(0, 40, 40, 40), store[1599:1639])),
        lambda: lowbit.weight_gradient(x, lowbit.Saved8(x.shape, x.dtype, store.view(torch.uint8)[:kept.buffer.numel()]), out=at(0, 40, 40, 40)),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(QuantizerLogicError, match="shares memory"):
            call()
        assert not store.any(), i
    # side by side: rows of one between the rows of the other, at equal distances and at others, and end to end
    want = lowbit.mx4_linear(x, square)
    for (x_at, x_stride), (out_at, out_stride) in [((0, 80), (40, 80)), ((40, 80), (0, 80)), ((0, 80), (1000 * 40, 80)), ((0, 40), (1600, 40)), ((1600, 40), (0, 40)),
                                                   ((40, 160), (0, 80)), ((0, 80), (40, 160)), ((3, 91), (45, 91)), ((91, 91), (43, 91)), ((0, 1640), (40, 40))]:
        store.fill_(float("nan"))
        v, out = at(x_at, 40, 40, x_stride), at(out_at, 40, 40, out_stride)
        v.copy_(x)
        lowbit.mx4_linear(v, square, out=out)
        assert torch.equal(out, want) and torch.equal(v, x)
    store.zero_()
    dw, db = lowbit.weight_gradient(x, kept, bias=True, out=(at(0, 40, 40, 41), store[1639:1679]))
    assert torch.equal(dw, lowbit.weight_gradient(x, kept)) and torch.equal(db, lowbit.weight_gradient(x, kept, bias=True)[1])


def negated(t):
    """A view with t's values over memory that holds their negatives."""
    v = torch._neg_view(-t)
    assert v.is_neg() and torch.equal(v, t)
    return v


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_views_that_stand_for_their_negative(dtype):
    x, w, dy = make(1, 24, 40, dtype), make(2, 30, 40, dtype), make(3, 24, 30, dtype)
    bias = make(4, 1, 30, dtype).view(30)
    q = lowbit.mx4_quantize(w)
    for shape in ((24, 40), (2, 3, 4, 40)):
        v = x.view(shape)
        assert torch.equal(lowbit.mx4_quantize(negated(v)).buffer, lowbit.mx4_quantize(x).buffer)
        assert torch.equal(lowbit.save8(negated(v)).buffer, lowbit.save8(x).buffer)
        y, kept = lowbit.mx4_linear(v, q, bias, save=True)
        y_, kept_ = lowbit.mx4_linear(negated(v), q, negated(bias), save=True)
        assert torch.equal(y, y_) and torch.equal(kept.buffer, kept_.buffer)
        assert torch.equal(lowbit.mx4_linear(negated(v)[:1], q, negated(bias)), lowbit.mx4_linear(v[:1], q, bias))
        d = dy.view(shape[:-1] + (30,))
        for a, b in zip(lowbit.weight_gradient(negated(d), kept, bias=True), lowbit.weight_gradient(d, kept, bias=True)):
            assert torch.equal(a, b)
        z, held = lowbit.activation_forward("silu", v, v)
        z_, held_ = lowbit.activation_forward("silu", negated(v), negated(v))
        assert torch.equal(z, z_) and torch.equal(held.buffer, held_.buffer) and torch.equal(held.gate, held_.gate)
        for a, b in zip(lowbit.activation_backward(negated(v), held), lowbit.activation_backward(v, held)):
            assert torch.equal(a, b)
    assert torch.equal(lowbit.mx4_quantize(negated(w).t()).buffer, lowbit.mx4_quantize(w.t()).buffer)
    assert torch.equal(lowbit.mx4_matmul(lowbit.mx4_quantize(x), q, negated(bias)), lowbit.mx4_matmul(lowbit.mx4_quantize(x), q, bias))
    # the imaginary part of a conjugate is one
    z = torch.complex(make(5, 24, 40, torch.float32), make(6, 24, 40, torch.float32))
    assert z.conj().imag.is_neg()
    assert torch.equal(lowbit.mx4_quantize(z.conj().imag).buffer, lowbit.mx4_quantize(-z.imag).buffer)
    # nothing is written through one
    for call in (lambda: lowbit.mx4_linear(x, q, out=torch._neg_view(torch.zeros(24, 30, dtype=dtype, device="cuda"))),
                 lambda: lowbit.mx4_dequantize(q, torch.float32, out=torch._neg_view(torch.zeros(30, 40, device="cuda"))),
                 lambda: lowbit.weight_gradient(dy, kept, out=torch._neg_view(torch.zeros(30, 40, device="cuda"))),
                 lambda: lowbit.weight_gradient(dy, kept, bias=True, out=(None, torch._neg_view(torch.zeros(30, device="cuda"))))):
        with pytest.raises(QuantizerLogicError):
            call()


def test_adding_needs_every_result():
    """A result that is to be added to and is not given would be added to memory that nobody has written."""
    x, dy = make(1, 20, 40, torch.bfloat16), make(2, 20, 30, torch.bfloat16)
    kept = lowbit.save8(x)
    dw, db = torch.zeros(30, 40, device="cuda"), torch.zeros(30, device="cuda")
    for given in (None, (dw, None), (None, db), (None, None)):
        with pytest.raises(QuantizerLogicError):
            lowbit.weight_gradient(dy, kept, bias=True, out=given, accumulate=True)
    with pytest.raises(QuantizerLogicError):
        lowbit.weight_gradient(dy, kept, accumulate=True)
    assert not dw.any() and not db.any()
    want, want_db = lowbit.weight_gradient(dy, kept, bias=True)
    # one of two given, to write into
    for given in ((dw, None), (None, db)):
        got, got_db = lowbit.weight_gradient(dy, kept, bias=True, out=given)
        assert torch.equal(got, want) and torch.equal(got_db, want_db)
    lowbit.weight_gradient(dy, kept, bias=True, out=(dw, db), accumulate=True)
    assert torch.equal(dw, 2.0 * want) and torch.equal(db, 2.0 * want_db)
    lowbit.weight_gradient(dy, kept, out=dw, accumulate=True)
    assert torch.allclose(dw, 3.0 * want, rtol=2.0 ** -22, atol=0.0) and torch.equal(db, 2.0 * want_db)


# ---- modules --------------------------------------------------------------------------------------


def test_modules_give_the_formulas_gradients():
    """Two layers with an activation between: outputs and gradients are those of the operators' definitions, taken step by step."""
    torch.manual_seed(5)
    first, second = lowbit.LowBitLinear(70, 90, device="cuda"), lowbit.LowBitLinear(90, 33, bias=False, device="cuda")
    act = lowbit.LowBitActivation("tanh")
    x = make(1, 50, 70, torch.float32, 0.2).requires_grad_()
    h = first(x)
    h.retain_grad()
    a = act(h)
    a.retain_grad()
    y = second(a)
    dy = make(2, 50, 33, torch.float32, 0.2)
    y.backward(dy)
    q = lambda t: ref.mx4(np64(t))[2]  # noqa: E731
    check, slack = product(q(x), q(first.weight), first.bias)
    close(h, check, slack, torch.float32)
    check, slack = product(q(dy), q(second.weight.t()), None)
    close(a.grad, check, slack, torch.float32)
    check_weight_gradient(second.weight.grad, None, dy, ref.save8(np64(a))[2])
    slope = ref.activation("tanh", ref.save8(np64(h))[2])[1]
    close(h.grad, np64(a.grad) * slope, np.abs(np64(a.grad)) * 2.0 ** -19 * 5, torch.float32)
    check, slack = product(q(h.grad), q(first.weight.t()), None)
    close(x.grad, check, slack, torch.float32)
    check_weight_gradient(first.weight.grad, first.bias.grad, h.grad, ref.save8(np64(x))[2])
    frozen = first.freeze()(x)
    assert torch.equal(frozen, h) and not frozen.requires_grad


def test_modules_free_what_they_kept_and_refuse_second_derivatives():
    layer, act = lowbit.LowBitLinear(40, 24, device="cuda"), lowbit.LowBitActivation("silu")
    x = make(3, 9, 40, torch.float32, 0.2).requires_grad_()
    y = act(layer(x), layer(x)).sum()
    y.backward()
    with pytest.raises(RuntimeError):
        y.backward()
    dx, = torch.autograd.grad(act(layer(x)).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()
