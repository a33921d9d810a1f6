"""The readout operators against plain 64-bit implementations.

Tolerances are bounds on rounding: eps = 2^-24 is half a float32 unit in the
last place, 2^-8 the same for bfloat16 and 2^-11 for float16; a sum's error is
bounded by its number of additions times eps times the sum of magnitudes.
"""

from __future__ import annotations

import math

import pytest

torch = pytest.importorskip("torch")

from mdescriptor_b200 import readout  # noqa: E402

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
HALF_ULP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


@pytest.fixture(autouse=True)
def _cuda(cuda_device):
    yield


def generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def matrix(seed, rows, width, dtype=torch.float32, pad=0, offset=0, scale=1.0):
    """Random rows as a view: `pad` unused columns, the first element `offset` elements into the storage."""
    flat = torch.randn(offset + rows * (width + pad) + 8, generator=generator(seed), device="cuda") * scale
    return flat.to(dtype)[offset:offset + rows * (width + pad)].view(rows, width + pad)[:, :width]


def e4m3(v):
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.clamp(torch.round(v / step) * step, -448.0, 448.0)


def tops(z):
    rows, width = z.shape
    blocks = (width + 127) // 128
    full = torch.zeros(rows, blocks * 128, dtype=z.dtype, device=z.device)
    full[:, :width] = z
    return full.view(rows, blocks, 128).abs().amax(2)


def spread(blocks, width):
    return blocks.repeat_interleave(128, dim=1)[:, :width]


def assert_codes(values, scales, z, factor=None, top=None, scale_tolerance=6 * EPS32):
    """Codes are the nearest e4m3 values of 448 z / A up to a relative 2^-21 (three float32 roundings) at a tie."""
    rows, width = z.shape
    top = tops(z) if top is None else top
    expected = top / 448.0 if factor is None else top / 448.0 * factor
    expected = torch.where(top < 2.0 ** -100, torch.zeros_like(expected), expected)
    assert scales.shape == expected.shape
    assert torch.all((scales.double() - expected).abs() <= expected.abs() * scale_tolerance)
    v = torch.where(spread(top, width) < 2.0 ** -100, torch.zeros_like(z), 448.0 * z / spread(top, width))
    got, best = values.float().double(), e4m3(v)
    assert torch.all((got - v).abs() <= (best - v).abs() + v.abs() * 2.0 ** -21)


# ---------------------------------------------------------------- norm

NORM_SHAPES = [(1, 1), (1, 144), (3, 127), (5, 128), (2, 129), (4, 255), (7, 2325), (300, 144), (4700, 96), (2500, 1224),
               (3, 20011), (2, 210000), (2400, 61)]


@pytest.mark.parametrize("rows,width", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_forms(rows, width, dtype):
    for residual in (False, True):
        pad, offset = (0, 0) if residual else (3, 1)
        x = matrix(1, rows, width, dtype, pad, offset)
        x[rows // 2] = 0
        r = matrix(2, rows, width, dtype, pad + 1, 3) if residual else None
        w = 1.0 + 0.2 * torch.randn(width, generator=generator(3), device="cuda")
        s32 = x.float() + r.float() if residual else x.float()
        s = s32.double()
        rstd = 1.0 / torch.sqrt((s * s).mean(1) + 1e-6)
        # a lane adds width / 32 squares one after the other, five more levels join the lanes, eight warps
        rtol = (width / 32 + 24) * EPS32
        for output in (None, "float8"):
            got = readout.rms_norm(x, w, residual=r, output=output)
            assert torch.all((got.rstd.double() - rstd).abs() <= rtol * rstd)
            if residual:
                assert torch.equal(got.sum, s32.to(dtype))
            else:
                assert got.sum is x
            if output is None:
                y = s * rstd[:, None] * w.double()
                # float16 results below the normal range are rounded to its smallest step
                tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
                assert torch.all((got.output.double() - y).abs() <= y.abs() * (rtol + 4 * EPS32 + HALF_ULP[dtype]) + tiny)
            else:
                z = (s32 * w).double()
                assert_codes(got.output.values, got.output.scales, z, rstd[:, None], scale_tolerance=rtol + 8 * EPS32)


def test_norm_non_finite_and_extreme_rows():
    x = torch.ones(6, 300, device="cuda")
    x[0, 5] = float("nan")
    x[1, 200] = float("inf")
    x[2] = 0.0
    x[3] = 1e-30
    x[4] = 1e18
    w = torch.ones(300, device="cuda")
    got = readout.rms_norm(x, w, output="float8").output
    y = got.float()
    assert torch.isnan(y[0]).all()  # the row factor is NaN
    assert torch.isnan(y[1, 128:256]).all()
    assert (y[2] == 0).all() and (got.scales[2] == 0).all()
    assert torch.allclose(y[3], torch.full((300,), 1e-27, device="cuda"), rtol=1e-6)  # eps holds the row factor at 1000
    assert torch.allclose(y[4], torch.ones(300, device="cuda"), rtol=1e-6)
    assert torch.allclose(y[5], torch.ones(300, device="cuda"), rtol=1e-5)


def test_norm_rows_beyond_32_bit_offsets():
    stride = 2 ** 31 + 24
    flat = torch.empty(2 * stride + 200, dtype=torch.bfloat16, device="cuda")
    x = flat.as_strided((3, 200), (stride, 1))
    x.copy_(matrix(5, 3, 200, torch.bfloat16))
    w = torch.ones(200, device="cuda")
    a, b = readout.rms_norm(x, w, output="float8"), readout.rms_norm(x.contiguous(), w, output="float8")
    assert torch.equal(a.output.float(), b.output.float()) and torch.equal(a.rstd, b.rstd)
    q = readout.quantize(x, layout="both")
    assert torch.equal(q.columns.float(), readout.quantize(x.contiguous(), layout="both").columns.float())


BACKWARD_SHAPES = [(1, 1), (1, 144), (5, 129), (33, 250), (700, 500), (900, 1000), (300, 2325), (150, 4100), (70, 8200),
                   (20, 16000), (9, 33001)]


@pytest.mark.parametrize("rows,width", BACKWARD_SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm_gradient(rows, width, dtype):
    for with_dsum in (False, True):
        pad, offset = (0, 0) if with_dsum else (5, 3)
        s = matrix(1, rows, width, dtype, pad, offset)
        dy = matrix(2, rows, width, dtype, pad + 2, 1)
        dsum = matrix(3, rows, width, dtype, pad, 2) if with_dsum else None
        w = 1.0 + 0.2 * torch.randn(width, generator=generator(4), device="cuda")
        rstd = torch.rsqrt((s.float() ** 2).mean(1) + 1e-6)
        dx, dw = readout.rms_norm_backward(dy, s, rstd, w, dsum=dsum)
        S, D, W, R = s.double(), dy.double(), w.double(), rstd.double()[:, None]
        c = (D * W * S).sum(1, keepdim=True)
        near = R * W * D
        far = S * R ** 3 * c / width
        want = near - far + (dsum.double() if with_dsum else 0.0)
        # the sum c: width / 32 additions a lane, then the lanes and warps; ten roundings of the rest
        slack = (width / 32 + 32) * EPS32 * (S.abs() * R ** 3 * (D * W * S).abs().sum(1, keepdim=True) / width)
        slack = slack + 10 * EPS32 * (near.abs() + far.abs()) + HALF_ULP[dtype] * want.abs()
        if dtype == torch.float16:
            slack = slack + 2.0 ** -25
        if with_dsum:
            slack = slack + EPS32 * want.abs()
        assert torch.all((dx.double() - want).abs() <= slack)
        each = D * S * R
        assert torch.all((dw.double() - each.sum(0)).abs() <= (rows + 8) * EPS32 * each.abs().sum(0))
        again = readout.rms_norm_backward(dy, s, rstd, w, dsum=dsum)
        assert torch.equal(dx, again[0]) and torch.equal(dw, again[1])


def test_norm_gradient_against_differences():
    rows, width = 6, 150
    x, dy = matrix(1, rows, width), matrix(2, rows, width)
    w = 1.0 + 0.2 * torch.randn(width, generator=generator(3), device="cuda")
    norm = readout.rms_norm(x, w)
    dx, dw = readout.rms_norm_backward(dy, norm.sum, norm.rstd, w)

    def loss(x, w):
        return (x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-6) * w * dy.double()).sum()

    h = 1e-5  # truncation h^2 and cancellation 1e-16 / h, both near 1e-10
    for i, j in [(0, 0), (2, 77), (5, 149)]:
        e = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
        e[i, j] = h
        slope = (loss(x.double() + e, w.double()) - loss(x.double() - e, w.double())) / (2 * h)
        assert abs(slope.item() - dx[i, j].item()) <= 1e-5 * max(1.0, abs(slope.item()))
        e = torch.zeros(width, dtype=torch.float64, device="cuda")
        e[j] = h
        slope = (loss(x.double(), w.double() + e) - loss(x.double(), w.double() - e)) / (2 * h)
        assert abs(slope.item() - dw[j].item()) <= 1e-5 * max(1.0, abs(slope.item()))


# ---------------------------------------------------------------- blocks

BLOCK_SHAPES = [(1, 1), (1, 300), (300, 1), (127, 129), (128, 128), (129, 127), (257, 1000), (1000, 144), (2501, 333)]


@pytest.mark.parametrize("rows,width", BLOCK_SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1)])
def test_quantize_layouts(rows, width, dtype, pad, offset):
    x = matrix(1, rows, width, dtype, pad, offset)
    x[rows // 3] = 0
    f = torch.exp(0.5 * torch.randn(rows, generator=generator(2), device="cuda"))
    g = torch.randn(width, generator=generator(3), device="cuda")  # of both signs
    for factors in (False, True):
        kw = {"row_factor": f, "col_factor": g} if factors else {}
        along_rows = (x.float() * g if factors else x.float()).double()
        along_columns = (x.float() * f[:, None] if factors else x.float()).double().t().contiguous()
        results = {layout: readout.quantize(x, layout=layout, **kw) for layout in ("rows", "columns", "both")}
        for layout in ("rows", "both"):
            q = results[layout].rows
            assert_codes(q.values, q.scales, along_rows, f.double()[:, None] if factors else None)
        for layout in ("columns", "both"):
            q = results[layout].columns
            assert_codes(q.values, q.scales, along_columns, g.double()[:, None] if factors else None)
        assert results["rows"].columns is None and results["columns"].rows is None
    q = readout.quantize(x, layout="tiles")
    tile = tops(tops(x.double()).t().contiguous()).t()
    full = tile.repeat_interleave(128, dim=0)[:rows]
    assert q.rows.scales.shape == tile.shape
    assert_codes(q.rows.values, q.rows.scales.repeat_interleave(128, dim=0)[:rows], x.double(), top=full)
    assert torch.equal(q.columns.values.float(), q.rows.values.float().t())
    assert torch.equal(q.columns.scales, q.rows.scales.t())


def test_quantize_non_finite_blocks():
    x = torch.ones(256, 256, device="cuda")
    x[3, 5] = float("nan")
    x[200, 130] = float("inf")
    x[10, 128:] = 0.0
    q = readout.quantize(x, layout="both")
    rows, columns = q.rows.values.float(), q.columns.values.float()
    assert torch.isnan(rows[3, :128]).all() and (rows[3, 128:] == 448).all()
    assert torch.isnan(rows[200, 130]) and (rows[200, 131:] == 0).all() and torch.isinf(q.rows.scales[200, 1])
    assert (rows[10, 128:] == 0).all() and q.rows.scales[10, 1] == 0
    assert torch.isnan(columns[5, :128]).all() and (columns[5, 128:] == 448).all()
    assert torch.isnan(columns[130, 200]) and (columns[130, 128:200] == 0).all()


# ---------------------------------------------------------------- product


def blocks(seed, rows, k, tiles=False):
    x = matrix(seed, rows, k) * torch.exp(torch.randn(k, generator=generator(seed + 1), device="cuda"))
    q = readout.quantize(x, layout="tiles" if tiles else "rows").rows
    return readout.Blocks(q.values, q.scales), x


def assert_product(got, a, b, extra=None):
    A, B = a.float().double(), b.float().double()
    want, size = A @ B.t(), A.abs() @ B.abs().t()
    if extra is not None:
        want, size = want + extra, size + extra.abs()
    # scales (two roundings), four instructions a block whose sums keep 21 bits or more, one float32 addition a block
    k_blocks = (A.shape[1] + 127) // 128
    slack = (2.0 ** -19 + (k_blocks + 4) * EPS32) * size + HALF_ULP[got.dtype] * want.abs()
    assert torch.all((got.double() - want).abs() <= slack)


PRODUCT_SHAPES = [(1, 1, 1), (1, 1024, 3696), (1, 64, 144), (2, 130, 128), (7, 300, 129), (16, 257, 500), (64, 1000, 2100),
                  (65, 128, 127), (128, 128, 128), (129, 127, 1000), (300, 513, 2325), (1000, 1024, 144), (2048, 1536, 700),
                  (4097, 520, 333), (33, 4097, 64), (260, 100, 9000)]


@pytest.mark.parametrize("m,n,k", PRODUCT_SHAPES)
@pytest.mark.parametrize("tiles", [True, False])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_product(m, n, k, tiles, dtype):
    a, b = blocks(1, m, k)[0], blocks(5, n, k, tiles)[0]
    got = readout.matmul(a, b, dtype=dtype)
    assert_product(got, a, b)
    assert torch.equal(got, readout.matmul(a, b, dtype=dtype))
    readout.check()


@pytest.mark.parametrize("m,n,k", [(3, 130, 200), (300, 333, 1000), (256, 256, 20000)])
def test_product_into_a_view_and_accumulated(m, n, k):
    a, b = blocks(1, m, k)[0], blocks(5, n, k)[0]
    for dtype in (torch.float32, torch.bfloat16):
        held = torch.full((m + 1, n + 5), 7.0, dtype=dtype, device="cuda")
        out = held[1:, 3:3 + n]
        assert readout.matmul(a, b, out=out) is out
        assert_product(out, a, b)
        assert (held[0] == 7).all() and (held[:, :3] == 7).all() and (held[:, 3 + n:] == 7).all()
    out = matrix(9, m, n)
    before = out.double()
    readout.matmul(a, b, out=out, accumulate=True)
    assert_product(out, a, b, before)


def test_product_long_sums_and_strided_scales():
    a, b = blocks(1, 130, 65537)[0], blocks(5, 140, 65537)[0]
    assert_product(readout.matmul(a, b, dtype="float32"), a, b)
    wide = readout.Blocks(a.values, torch.cat([a.scales, a.scales], 1)[:, :a.scales.shape[1]])
    assert torch.equal(readout.matmul(wide, b, dtype="float32"), readout.matmul(a, b, dtype="float32"))
    half = readout.Blocks(a.values[::2], a.scales[::2])
    pitch = a.values.stride(0)
    copy = torch.zeros(65, pitch, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)[:, :65537]
    copy.copy_(half.values)  # the same rows, one after the other
    same = readout.Blocks(copy, half.scales.contiguous())
    assert torch.equal(readout.matmul(half, b, dtype="float32"), readout.matmul(same, b, dtype="float32"))
    assert_product(readout.matmul(half, b, dtype="float32"), half, b)


def test_product_non_finite_stays_in_its_row():
    a, b = blocks(1, 200, 400)[0], blocks(5, 150, 400, True)[0]
    clean = readout.matmul(a, b)
    a.scales[7, 1] = float("nan")
    got = readout.matmul(a, b)
    assert torch.isnan(got[7]).all()
    keep = torch.arange(200, device="cuda") != 7
    assert torch.equal(got[keep], clean[keep])


def test_empty_operands():
    w = torch.ones(5, device="cuda")
    empty = torch.empty(0, 5, device="cuda")
    assert readout.rms_norm(empty, w, output="float8").output.values.shape == (0, 5)
    dx, dw = readout.rms_norm_backward(empty, empty, torch.empty(0, device="cuda"), w)
    assert dx.shape == (0, 5) and (dw == 0).all()
    q = readout.quantize(empty, layout="both")
    assert q.rows.values.shape == (0, 5) and q.columns.values.shape == (5, 0)
    some = readout.quantize(torch.ones(3, 5, device="cuda")).rows
    assert readout.matmul(q.rows, some).shape == (0, 3)
    assert (readout.matmul(readout.quantize(torch.ones(4, 3, device="cuda")[:, :0]).rows,
                           readout.quantize(torch.ones(2, 3, device="cuda")[:, :0]).rows) == 0).all()


def test_layer_gradients_of_the_product():
    """dX and dW of y = X W^T through blocks, against the same products of what the blocks stand for."""
    rows, k, n = 517, 400, 300
    x, w, dy = matrix(1, rows, k), matrix(2, n, k, scale=0.05), matrix(3, rows, n, torch.bfloat16)
    weight = readout.quantize(w, layout="tiles")
    d, x8 = readout.quantize(dy, layout="both"), readout.quantize(x, layout="columns")
    assert_product(readout.matmul(d.rows, weight.columns, dtype="float32"), d.rows, weight.columns)
    dw = readout.matmul(d.columns, x8.columns, dtype="float32")
    assert_product(dw, d.columns, x8.columns)
    # against the formula without rounding to 8 bits: each factor is off by at most 1/16 of itself, or 2^-10 / 448 of its block
    want = dy.double().t() @ x.double()
    size = dy.double().abs().t() @ x.double().abs()
    assert torch.all((dw.double() - want).abs() <= 0.13 * size + 1e-3 * rows * 4.5 * 4.5 * 2.0 ** -9)


def test_operators_on_another_stream():
    x = matrix(1, 600, 700, torch.bfloat16)
    w = torch.ones(700, device="cuda")
    b = blocks(5, 300, 700, True)[0]
    want = readout.matmul(readout.rms_norm(x, w, output="float8").output, b)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            got = readout.matmul(readout.rms_norm(x, w, output="float8").output, b)
    side.synchronize()
    assert torch.equal(got, want)


def test_products_on_two_streams_at_once():
    """Both streams' kernels want whole SMs and their tensor memory; neither may disturb the other."""
    a, b = blocks(1, 700, 900)[0], blocks(5, 600, 900, True)[0]
    few = blocks(9, 5, 900)[0]
    want, want_few = readout.matmul(a, b), readout.matmul(few, b)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(10):
        with torch.cuda.stream(streams[0]):
            got.append((readout.matmul(a, b), want))
        with torch.cuda.stream(streams[1]):
            got.append((readout.matmul(few, b), want_few))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in got)


def test_products_beyond_32_bit_offsets():
    # codes: 1 100 000 rows of 4096 bytes
    codes = torch.randint(0, 256, (1100000, 4096), dtype=torch.uint8, device="cuda", generator=generator(1))
    codes[(codes & 127) == 127] = 0  # no NaN
    a = readout.Blocks(codes.view(torch.float8_e4m3fn), torch.rand(1100000, 32, generator=generator(2), device="cuda"))
    b = blocks(5, 72, 4096, True)[0]
    got = readout.matmul(a, b, dtype="float32")
    for rows in (slice(0, 300), slice(1048500, 1048700), slice(1099700, 1100000)):
        part = readout.Blocks(a.values[rows], a.scales[rows])
        assert_product(got[rows], part, b)
    # results: 2.3 G elements, through the copy engine and row by row
    a, w = blocks(1, 70000, 64)[0], blocks(5, 33000, 64, True)[0]
    for n in (33000, 32999):
        b = readout.Blocks(w.values[:n], w.scales)
        got = readout.matmul(a, b)
        for rows in (slice(0, 200), slice(69800, 70000)):
            assert_product(got[rows], readout.Blocks(a.values[rows], a.scales[rows]), b)
        del got


# ---------------------------------------------------------------- optimizer


def uniform(count, seed, step):
    low = 0xFFFFFFFF
    h = torch.arange(count, device="cuda", dtype=torch.int64) ^ ((seed * 0x6A09E667 + step * 0xBB67AE85) & low)
    h = ((h ^ (h >> 16)) * 0xA54FF53B) & low
    h = ((h ^ (h >> 15)) * 0x510E527F) & low
    h = h ^ (h >> 16)
    return (h >> 16).double() * 2.0 ** -16, (h & 0xFFFF).double() * 2.0 ** -16


def reference_update(p, g, m, v, step, lr, b1, b2, eps, decay):
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    update = m / (1 - b1 ** step) / (torch.sqrt(v / (1 - b2 ** step)) + eps)
    return p - lr * decay * p - lr * update, m, v, lr * update


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
def test_adamw_32(dtype, grad_dtype):
    sizes = [1, 5, 128, 129, 4096, 4097, 0, 10001] + [37] * 500  # more tensors than one launch takes
    flat = [matrix(i, 1, n + 3, dtype)[0] for i, n in enumerate(sizes)]
    params = [f[i % 3:i % 3 + n] for i, (f, n) in enumerate(zip(flat, sizes))]  # of every alignment
    decays = [0.01 * (i % 2) for i in range(len(sizes))]
    opt = readout.AdamW(params, lr=2e-3, weight_decay=decays, seed=3)
    P = [p.double() for p in params]
    M, V = [torch.zeros_like(p) for p in P], [torch.zeros_like(p) for p in P]
    for step in (1, 2, 3):
        grads = [matrix(1000 * step + i, 1, n + 1, grad_dtype, scale=0.1)[0][1:] for i, n in enumerate(sizes)]
        opt.step(grads, grad_scale=0.5)
        for i in range(len(sizes)):
            P[i], M[i], V[i], moved = reference_update(P[i], grads[i].double() * 0.5, M[i], V[i], step, 2e-3, 0.9, 0.999,
                                                       1e-8, decays[i])
            # a dozen float32 roundings of the update, three of m and v; the stored p is rounded once a step
            assert torch.all((opt.state["exp_avg"][i].double() - M[i]).abs() <= 4 * step * EPS32 * (M[i].abs() + 0.1))
            assert torch.all((opt.state["exp_avg_sq"][i].double() - V[i]).abs() <= 5 * step * EPS32 * V[i] + 1e-40)
            slack = HALF_ULP[dtype] * (P[i].abs() + 1e-2) + 4 * EPS32 * P[i].abs() + 1e-4 * moved.abs()
            assert torch.all((params[i].double() - P[i]).abs() <= slack)
            P[i] = params[i].double()  # each step from the stored value
            M[i], V[i] = opt.state["exp_avg"][i].double(), opt.state["exp_avg_sq"][i].double()
    assert opt.state["step"] == 3


def test_adamw_8():
    sizes = [1, 127, 128, 300, 5000, 12345]
    params = [matrix(i, 1, n)[0].clone() for i, n in enumerate(sizes)]
    opt = readout.AdamW(params, state_bits=8, seed=11)
    firsts = [sum((n + 127) // 128 * 128 for n in sizes[:i]) for i in range(len(sizes))]
    total = firsts[-1] + sizes[-1]
    for step in (1, 2, 3):
        P = [p.double() for p in params]
        held = {key: [readout.Blocks(q.view(1, -1), s.view(1, -1)).float().double()[0] for q, s in
                      zip(opt.state[key], opt.state[key + "_scale"])] for key in ("exp_avg", "exp_avg_sq")}
        grads = [matrix(1000 * step + i, 1, n, scale=0.1)[0] * torch.exp(torch.randn(n, generator=generator(i), device="cuda"))
                 for i, n in enumerate(sizes)]
        opt.step(grads)
        noise = uniform(total, 11, step)
        for i, n in enumerate(sizes):
            p, m, v, moved = reference_update(P[i], grads[i].double(), held["exp_avg"][i], held["exp_avg_sq"][i], step, 1e-3,
                                              0.9, 0.999, 1e-8, 0.01)
            assert torch.all((params[i].double() - p).abs() <= 4 * EPS32 * (p.abs() + moved.abs()) + 16 * EPS32 * moved.abs())
            # the states are defined on float32 products (with 0.9 and 0.1 as floats): m's two may cancel
            m = (held["exp_avg"][i].float() * 0.9).double() + (grads[i] * (1.0 - 0.9)).double()
            for key, x, u in (("exp_avg", m, noise[0]), ("exp_avg_sq", v, noise[1])):
                top = tops(x.view(1, -1))
                assert torch.all((opt.state[key + "_scale"][i].double() - top[0] / 448).abs() <= 8 * EPS32 * top[0] / 448 + 1e-37)
                a = 448 * x.abs() / spread(top, n)[0]
                unit = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
                at = a / unit + u[firsts[i]:firsts[i] + n]
                want = torch.clamp(torch.floor(at) * unit, max=448.0)
                if key == "exp_avg_sq":
                    want = torch.where((x > 0) & (want == 0), 2.0 ** -9, want)
                got = opt.state[key][i].float().double()
                # a is off by a few float32 roundings of itself (at most 16 steps): 2^-18 of a step, beside u's grid
                near = (at - torch.round(at)).abs() <= 2.0 ** -17
                assert torch.all((got.abs() == want) | (near & ((got.abs() - want).abs() <= unit)))
                assert torch.all((got == 0) | (torch.sign(got) == torch.sign(x)))
    again = readout.AdamW([p.clone() for p in params], state_bits=8, seed=11, state=opt.state)
    assert again.state["step"] == 3


def test_adamw_8_follows_a_slow_change():
    """v falls towards g^2 by a thousandth a step although its codes lie at least 1/16 apart."""
    n = 4096
    p = torch.zeros(n, device="cuda")
    g = torch.full((n,), 0.1, device="cuda")
    state = {"step": 10000, "exp_avg": [torch.full((n,), 448.0, device="cuda").to(torch.float8_e4m3fn)],
             "exp_avg_sq": [torch.full((n,), 224.0, device="cuda").to(torch.float8_e4m3fn)],
             "exp_avg_scale": [torch.full((n // 128,), 0.1 / 448, device="cuda")],
             "exp_avg_sq_scale": [torch.full((n // 128,), 0.04 / 224, device="cuda")]}
    state["exp_avg_sq"][0].view(torch.uint8)[::128] = 0x7E  # a larger value holds the block's scale
    opt = readout.AdamW([p], state_bits=8, state=state)
    for _ in range(1000):
        opt.step([g])
    v = readout.Blocks(opt.state["exp_avg_sq"][0].view(1, -1), opt.state["exp_avg_sq_scale"][0].view(1, -1)).float()[0]
    rest = torch.arange(n, device="cuda") % 128 != 0
    want = 0.01 + 0.03 * 0.999 ** 1000
    # 4064 values, each off by at most an eighth of itself in steps that dithering makes independent
    assert abs(v[rest].mean().item() / want - 1) < 0.02


# ---------------------------------------------------------------- refusals


def test_refusals():
    x, w = torch.ones(4, 8, device="cuda"), torch.ones(8, device="cuda")
    with pytest.raises(ValueError, match="two dimensions"):
        readout.rms_norm(x[0], w)
    with pytest.raises(ValueError, match="CUDA"):
        readout.rms_norm(x.cpu(), w)
    with pytest.raises(ValueError, match="column stride"):
        readout.rms_norm(x.t(), torch.ones(4, device="cuda"))
    with pytest.raises(ValueError, match="float32, bfloat16 or float16"):
        readout.rms_norm(x.double(), w)
    with pytest.raises(ValueError, match="weight"):
        readout.rms_norm(x, w[:7])
    with pytest.raises(ValueError, match="residual"):
        readout.rms_norm(x, w, residual=x.bfloat16())
    with pytest.raises(ValueError, match="eps"):
        readout.rms_norm(x, w, eps=0.0)
    with pytest.raises(ValueError, match="output"):
        readout.rms_norm(x, w, output="int8")
    with pytest.raises(ValueError, match="overlap"):
        readout.quantize(torch.ones(100, device="cuda").as_strided((4, 8), (2, 1)))
    with pytest.raises(ValueError, match="dy"):
        readout.rms_norm_backward(x[:3], x, torch.ones(4, device="cuda"), w)
    with pytest.raises(ValueError, match="layout"):
        readout.quantize(x, layout="diagonal")
    with pytest.raises(ValueError, match="factors"):
        readout.quantize(x, layout="tiles", col_factor=w)
    a, b = readout.quantize(x).rows, readout.quantize(torch.ones(3, 8, device="cuda")).rows
    with pytest.raises(ValueError, match="same width"):
        readout.matmul(a, readout.quantize(torch.ones(3, 9, device="cuda")).rows)
    with pytest.raises(ValueError, match="dtype"):
        readout.matmul(a, b, dtype="float16")
    with pytest.raises(ValueError, match="accumulate"):
        readout.matmul(a, b, accumulate=True)
    with pytest.raises(ValueError, match="accumulate"):
        readout.matmul(a, b, out=torch.empty(4, 3, device="cuda", dtype=torch.bfloat16), accumulate=True)
    with pytest.raises(ValueError, match="out"):
        readout.matmul(a, b, out=torch.empty(3, 4, device="cuda"))
    with pytest.raises(ValueError, match="multiple of 16"):
        readout.matmul(readout.Blocks(a.values.contiguous(), a.scales), b)
    with pytest.raises(ValueError, match="scales"):
        readout.matmul(readout.Blocks(a.values, a.scales[:2]), b)
    with pytest.raises(ValueError, match="float8"):
        readout.matmul(readout.Blocks(x, a.scales), b)
    p = torch.ones(10, device="cuda")
    with pytest.raises(ValueError, match="state_bits"):
        readout.AdamW([p], state_bits=16)
    with pytest.raises(ValueError, match="contiguous"):
        readout.AdamW([torch.ones(4, 4, device="cuda").t()[:, :2]])
    with pytest.raises(ValueError, match="at least one"):
        readout.AdamW([])
    with pytest.raises(ValueError, match="weight_decay"):
        readout.AdamW([p], weight_decay=[0.1, 0.2])
    with pytest.raises(ValueError, match="weight decay"):
        readout.AdamW([p], weight_decay=-1.0)
    with pytest.raises(ValueError, match="exp_avg"):
        readout.AdamW([p], state={"step": 0, "exp_avg": [], "exp_avg_sq": []})
    opt = readout.AdamW([p])
    with pytest.raises(ValueError, match="grads"):
        opt.step([])
    with pytest.raises(ValueError, match="grads"):
        opt.step([p[:5]])
    with pytest.raises(ValueError, match="grads"):
        opt.step([p.double()])
    with pytest.raises(ValueError, match="settings"):
        opt.step([p], lr=math.inf)
    assert opt.state["step"] == 0
