"""The readout operators where their launches, waits and checks change: many tiles
for each pair of CTAs, shapes past a limit, other tensors behind an optimizer.

Values are held to the bounds of test_gpu_readout.py.
"""

from __future__ import annotations

import ctypes
import threading
import time

import pytest

torch = pytest.importorskip("torch")

from mdescriptor_b200 import _lib, readout  # noqa: E402
from mdescriptor_b200._lib import lib, raise_for  # noqa: E402
from test_gpu_readout import (EPS32, HALF_ULP, assert_codes, assert_product, blocks, generator, matrix, spread, tops,
                              uniform)  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda(cuda_device):
    yield


# ---------------------------------------------------------------- products with scales of rows

# 256 tiles (or 120) for 74 pairs of CTAs: each pair goes from tile to tile.  Four blocks of K share a fill of the
# scales' buffer: 2, 4, 9 and 17 blocks are an odd number of fills, after which the next tile must not take up the
# same half of it; 1, 5 and 157 an odd or even one beside them.
MANY_TILES = [(4096, 4096, 128), (4096, 4096, 130), (4096, 4096, 400), (4096, 4096, 520), (4096, 4096, 1100),
              (4000, 4096, 2100), (3000, 2325, 20000)]


@pytest.mark.parametrize("m,n,k", MANY_TILES)
@pytest.mark.parametrize("tiles", [False, True])
def test_product_of_many_tiles_a_pair(m, n, k, tiles):
    a, b = blocks(1, m, k)[0], blocks(5, n, k, tiles)[0]
    for dtype in ("bfloat16", "float32"):
        got = readout.matmul(a, b, dtype=dtype)
        assert_product(got, a, b)
        for _ in range(4):
            assert torch.equal(got, readout.matmul(a, b, dtype=dtype))
    # row by row instead of through the copy engine, and added to what is there
    held = torch.zeros(m, n + 3, device="cuda")
    out = held[:, 1:1 + n]
    out.copy_(matrix(9, m, n))
    before = out.double()
    readout.matmul(a, b, out=out, accumulate=True)
    assert_product(out, a, b, before)
    readout.check()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_product_of_many_rows_in_parts(dtype):
    """Parts of K (one tile more than the pairs take in whole rounds) and more rows than a grid's second dimension holds."""
    m, n, k = 265472, 250, 40960
    codes = torch.randint(0, 126, (m, k), dtype=torch.uint8, device="cuda", generator=generator(1))
    a = readout.Blocks(codes.view(torch.float8_e4m3fn), torch.rand(m, k // 128, generator=generator(2), device="cuda"))
    b = blocks(5, n, k, True)[0]
    parts = ctypes.c_int64()
    raise_for(lib.mdsoap_matmul_bytes(m, n, k, 1, 0, ctypes.byref(parts)))
    assert parts.value > 0
    got = readout.matmul(a, b, dtype=dtype)
    for rows in (slice(0, 300), slice(262100, 262400), slice(m - 300, m)):
        assert_product(got[rows], readout.Blocks(a.values[rows], a.scales[rows]), b)


# ---------------------------------------------------------------- products whose copies stop


@pytest.fixture
def withheld():
    """Lets the copies of later products stop after so many blocks; all of them again afterwards."""
    yield lib.mdsoap_probe_matmul
    lib.mdsoap_probe_matmul(-1, -1)


@pytest.mark.parametrize("m,n,k,tiles,copied", [
    (700, 600, 1300, False, 3), (700, 600, 1300, True, 0), (1000, 1024, 9000, False, 7), (4096, 4096, 700, False, 8),
    (4096, 4096, 700, True, 8), (5, 300, 3696, True, 1), (100, 19000, 700, False, 2)])
def test_product_whose_copies_stop_ends(m, n, k, tiles, copied, withheld):
    """Each wait ends after its second, the warps that meet at barriers all come to them, and the next product is right."""
    a, b = blocks(1, m, k)[0], blocks(5, n, k, tiles)[0]
    readout.check()
    withheld(copied, copied)
    start = time.perf_counter()
    readout.matmul(a, b, dtype="float32")
    with pytest.raises(RuntimeError, match="did not complete in time"):
        readout.check()
    assert time.perf_counter() - start < 8.0  # waits one after the other: a copy, an accumulator, what is in flight
    readout.check()  # reported once
    withheld(-1, -1)
    assert_product(readout.matmul(a, b, dtype="float32"), a, b)
    readout.check()


@pytest.mark.parametrize("first,second", [(5, 3), (3, 5), (0, 2), (2, 0), (7, 6)])
@pytest.mark.parametrize("tiles", [False, True])
def test_product_whose_ctas_stop_at_different_blocks(first, second, tiles, withheld):
    """Neither CTA of a pair leaves before both CTAs' copies have landed, wherever each of them stopped."""
    a, b = blocks(1, 700, 1300)[0], blocks(5, 600, 1300, tiles)[0]
    readout.check()
    withheld(first, second)
    start = time.perf_counter()
    readout.matmul(a, b)
    with pytest.raises(RuntimeError, match="did not complete in time"):
        readout.check()
    # a second for the copies that never come, and none for those in flight, which all land
    assert time.perf_counter() - start < 1.9
    withheld(-1, -1)
    assert_product(readout.matmul(a, b), a, b)
    readout.check()


# ---------------------------------------------------------------- products into views


@pytest.mark.parametrize("m,n", [(700, 601), (700, 602), (300, 603), (4000, 4093), (1000, 257), (130, 127), (20, 61)])
@pytest.mark.parametrize("k", [200, 1300])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_product_into_a_view_of_whole_pieces(m, n, k, tiles, dtype):
    """Rows that begin on 16 bytes and end inside such a piece: what lies behind them stays."""
    a, b = blocks(1, m, k)[0], blocks(5, n, k, tiles)[0]
    held = torch.full((m + 2, (n // 16 + 2) * 16), 7.0, dtype=dtype, device="cuda")
    out = held[1:-1, :n]
    readout.matmul(a, b, out=out)
    assert_product(out, a, b)
    assert (held[0] == 7).all() and (held[-1] == 7).all() and (held[:, n:] == 7).all()

@pytest.mark.parametrize("m,n,k,tiles,first,second", [
    (700, 600, 1300, False, 3, 3), (700, 601, 1300, True, 5, 3), (1000, 1024, 9000, False, 7, 8), (300, 300, 2100, True, 2, 2),
    (4096, 4096, 700, False, 8, 8), (4000, 4096, 700, True, 9, 8), (4000, 4093, 700, True, 8, 8),
    (5, 300, 3696, True, 1, 1), (100, 700, 1300, False, 2, 2), (60, 19000, 700, False, 2, 2)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_results_that_could_not_be_had_are_nan(m, n, k, tiles, first, second, dtype, withheld):
    a, b = blocks(1, m, k)[0], blocks(5, n, k, tiles)[0]
    clean = readout.matmul(a, b, out=torch.zeros(m, n, dtype=dtype, device="cuda"))
    readout.check()
    held = torch.full((m + 1, n + 3), 7.0, dtype=dtype, device="cuda")
    for out in (torch.zeros(m, n, dtype=dtype, device="cuda"), held[1:, :n]):
        withheld(first, second)
        readout.matmul(a, b, out=out)
        with pytest.raises(RuntimeError, match="did not complete in time"):
            readout.check()
        withheld(-1, -1)
        missing = torch.isnan(out)
        assert missing.any()
        assert torch.equal(out[~missing], clean[~missing])
    assert (held[0] == 7).all() and (held[:, n:] == 7).all()


# ---------------------------------------------------------------- shared memory of wide rows


@pytest.mark.parametrize("blocks_", [12279, 12281, 12288, 12289])
def test_rows_around_the_shared_memory_that_every_launch_has(blocks_):
    """One float for each block of 128 beside the kernel's own few bytes: 48 KB at 12 280 blocks."""
    width = blocks_ * 128 - 5
    x, w = matrix(1, 2, width), torch.ones(width, device="cuda")
    q = readout.quantize(x).rows
    assert_codes(q.values, q.scales, x.double())
    n = readout.rms_norm(x, w, output="float8")
    assert torch.equal(n.output.values.view(torch.uint8), q.values.view(torch.uint8))


def on_two_threads(*calls):
    """Statuses of calls into the library that run side by side (ctypes lets go of the interpreter's lock)."""
    seen = []

    def repeat(call):
        for _ in range(400):
            seen.append(call())

    threads = [threading.Thread(target=repeat, args=(call,)) for call in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return seen


def test_wide_rows_from_two_threads():
    """Widths that share a kernel and need more shared memory than every launch has, at the same time."""
    def norm(width):
        x, w, rstd = torch.ones(1, width, device="cuda"), torch.ones(width, device="cuda"), torch.empty(1, device="cuda")
        values = torch.empty(1, width, dtype=torch.uint8, device="cuda")
        scales = torch.empty(1, width // 128, device="cuda")
        held = (x, w, rstd, values, scales)
        return lambda: held and lib.mdsoap_rms_norm(
            x.data_ptr(), 1, width, width, None, 0, _lib.FLOAT32, w.data_ptr(), 1e-6, None, 0, rstd.data_ptr(),
            values.data_ptr(), width, scales.data_ptr(), width // 128, 0, torch.cuda.current_stream().cuda_stream)

    assert set(on_two_threads(norm(12800 * 128), norm(40000 * 128))) == {_lib.OK}


def test_norm_gradients_from_two_threads():
    """Widths that share a kernel and take 48 and 144 KB of its ring, at the same time."""
    def gradient(width):
        t = [torch.ones(9, width, device="cuda", dtype=torch.bfloat16) for _ in range(3)]
        v = [torch.ones(n, device="cuda") for n in (9, width, width)]
        size = ctypes.c_int64()
        raise_for(lib.mdsoap_rms_norm_backward_bytes(9, width, _lib.BFLOAT16, 0, ctypes.byref(size)))
        space = torch.empty(size.value, dtype=torch.uint8, device="cuda")
        held = (t, v, space)
        return lambda: held and lib.mdsoap_rms_norm_backward(
            t[0].data_ptr(), 9, width, width, t[1].data_ptr(), width, v[0].data_ptr(), v[1].data_ptr(), None, 0,
            _lib.BFLOAT16, t[2].data_ptr(), width, v[2].data_ptr(), space.data_ptr(), size.value, 0,
            torch.cuda.current_stream().cuda_stream)

    assert set(on_two_threads(gradient(2400), gradient(8000))) == {_lib.OK}


@pytest.mark.parametrize("output", [None, "float8"])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_of_no_columns(output, with_residual):
    x, w = torch.empty(5, 0, device="cuda"), torch.empty(0, device="cuda")
    junk = [torch.full((5,), 7.0, device="cuda") for _ in range(8)]
    del junk  # what a result that nobody fills would hold
    n = readout.rms_norm(x, w, residual=x if with_residual else None, output=output)
    assert n.rstd.shape == (5,) and torch.isnan(n.rstd).all()
    assert n.sum.shape == (5, 0)
    assert (n.output if output is None else n.output.values).shape == (5, 0)
    dx, dw = readout.rms_norm_backward(x, n.sum, n.rstd, w)
    assert dx.shape == (5, 0) and dw.shape == (0,)


# ---------------------------------------------------------------- optimizer


@pytest.mark.parametrize("state_bits", [32, 8])
def test_adamw_gradients_of_every_size(state_bits):
    """The first step moves p by lr wherever the gradient's square is a float32, whatever the gradient's size."""
    sizes = torch.logspace(-18.5, 19, 76, dtype=torch.float64).tolist()
    params = [torch.zeros(1000, device="cuda") for _ in sizes]
    grads = [torch.full((1000,), size, device="cuda") for size in sizes]
    for p, g in zip(params, grads):
        g[::2].neg_()
    opt = readout.AdamW(params, lr=1e-3, eps=0.0, weight_decay=0.0, state_bits=state_bits)
    opt.step(grads)
    for p, g in zip(params, grads):
        # v = 0.001 g^2 is off by three roundings, and below the normal range by half of its smallest step too
        v = 1e-3 * g.double() ** 2
        slack = 16 * EPS32 + 0.5 * (2.0 ** -150 / v + 2.0 ** -22)
        assert torch.all((p.double() + 1e-3 * torch.sign(g).double()).abs() <= 1e-3 * slack)


def adamw_pair(state_bits, dtype=torch.float32):
    """Parameters and gradients of two like optimizers."""
    sizes = [300, 4097, 5]
    params = [matrix(i, 1, n, dtype)[0].clone() for i, n in enumerate(sizes)]
    grads = [matrix(10 + i, 1, n)[0].clone() for i, n in enumerate(sizes)]
    return params, [p.clone() for p in params], grads


def assert_like(a, b):
    for x, y in zip(a.params, b.params):
        assert torch.equal(x, y)
    for key in ("exp_avg", "exp_avg_sq"):
        for x, y in zip(a.state[key], b.state[key]):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("state_bits", [32, 8])
def test_adamw_takes_up_replaced_state(state_bits):
    params, others, grads = adamw_pair(state_bits)
    a, b = readout.AdamW(params, state_bits=state_bits), readout.AdamW(others, state_bits=state_bits)
    a.step(grads), b.step(grads)
    saved = {key: value if key == "step" else [t.clone() for t in value] for key, value in a.state.items()}
    a.step(grads)
    for x, y in zip(params, others):
        x.copy_(y)
    a.state = saved  # back to the first step
    a.step(grads), b.step(grads)
    assert_like(a, b)
    moments = a.state["exp_avg"]
    moments[2] = moments[2].clone()
    a.step(grads), b.step(grads)
    moments[1] = moments[1].clone()
    a.state["exp_avg_sq"] = tuple(a.state["exp_avg_sq"])
    before = a.state["exp_avg"][1].view(torch.uint8).clone()
    junk = [torch.full_like(params[1], 9.0) for _ in range(8)]  # takes memory that nobody holds any more
    a.step(grads), b.step(grads)
    assert_like(a, b)
    assert not torch.equal(a.state["exp_avg"][1].view(torch.uint8), before)
    assert all((j == 9.0).all() for j in junk)


@pytest.mark.parametrize("state_bits", [32, 8])
def test_adamw_follows_parameters_to_other_memory(state_bits):
    params, others, grads = adamw_pair(state_bits)
    a, b = readout.AdamW(params, state_bits=state_bits), readout.AdamW(others, state_bits=state_bits)
    a.step(grads), b.step(grads)
    params[1].data = params[1].data.clone()
    junk = [torch.full_like(params[1], 9.0) for _ in range(8)]
    a.step(grads), b.step(grads)
    assert_like(a, b)
    a.params[0] = params[0].clone()
    a.step(grads), b.step(grads)
    assert_like(a, b)
    assert all((j == 9.0).all() for j in junk)
    for p in a.params:
        p.data = p.data.bfloat16()
    for p in b.params:
        p.data = p.data.bfloat16()
    a.step(grads)
    again = readout.AdamW(b.params, state_bits=state_bits, state=b.state)
    again.step(grads)
    assert_like(a, again)


def test_adamw_refuses_replacements_that_do_not_fit():
    params, _, grads = adamw_pair(32)
    opt = readout.AdamW(params)
    opt.step(grads)
    held = opt.state["exp_avg"][1]
    opt.state["exp_avg"][1] = held[:-1].clone()
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step(grads)
    opt.state["exp_avg"][1] = held
    params[2].data = torch.ones(9, device="cuda")
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step(grads)
    assert opt.state["step"] == 1
    opt.params.pop()
    with pytest.raises(ValueError, match="params must hold 3"):
        opt.step(grads[:2])


def test_closed_adamw_refuses_its_step():
    params, _, grads = adamw_pair(32)
    opt = readout.AdamW(params)
    opt.step(grads)
    opt.close()
    opt.close()
    with pytest.raises(ValueError, match="closed"):
        opt.step(grads)
    assert opt.state["step"] == 1


def test_adamw_after_a_refused_replacement():
    """Put back, the refused tensor's predecessor goes on as if nothing had been."""
    params, others, grads = adamw_pair(32)
    a, b = readout.AdamW(params), readout.AdamW(others)
    a.step(grads), b.step(grads)
    held = params[2].data
    params[2].data = torch.ones(9, device="cuda")
    with pytest.raises(ValueError, match="exp_avg"):
        a.step(grads)
    params[2].data = held
    with pytest.raises(ValueError, match="grads"):
        a.step([*grads[:2], torch.ones(9, device="cuda")])
    a.step(grads), b.step(grads)
    assert_like(a, b)


@pytest.mark.parametrize("steps_before", [0, 2])
def test_adamw_refuses_to_be_captured(steps_before):
    """Replays would repeat one step's number; the first step could not be captured at all."""
    params, others, grads = adamw_pair(32)
    a, b = readout.AdamW(params), readout.AdamW(others)
    for _ in range(steps_before):
        a.step(grads), b.step(grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        doubled = grads[0] * 2.0
        with pytest.raises(ValueError, match="captured"):
            a.step(grads)
    graph.replay()  # what else was captured is whole
    assert torch.equal(doubled, grads[0] * 2.0)
    assert a.state["step"] == steps_before
    a.step(grads), b.step(grads)
    assert_like(a, b)


# More tiles of 4096 than three CTAs an SM take in two turns, full ones beside partial ones and tensors of no, one and a
# few elements between them: each CTA goes from tile to tile, reading half a tile ahead where the next one is full.
MANY_TILES_SIZES = [4096 * 300, 17, 4096 * 200 + 1, 0, 4095, 4096, 1, 4096 * 350 + 129, 300, 4096 * 300, 8192]


@pytest.mark.parametrize("state_bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("grad_dtype,offset", [(torch.float32, 0), (torch.bfloat16, 1)])
def test_adamw_of_many_tiles(state_bits, dtype, grad_dtype, offset):
    sizes, lr, b1, b2, eps, decay, seed = MANY_TILES_SIZES, 1e-3, 0.9, 0.999, 1e-8, 0.01, 7

    def tensors(like, kind, make):
        # `offset`: each tensor one element into its memory, so that no unit of four is aligned
        held = [make(n + offset).to(torch.float32) for n in like]
        if kind == torch.float8_e4m3fn:
            return [t.to(torch.uint8).view(kind)[offset:] for t in held]
        return [t.to(kind)[offset:] for t in held]

    g = generator(3)
    params = tensors(sizes, dtype, lambda n: 0.1 * torch.randn(n, generator=g, device="cuda"))
    blocks_ = [(n + 127) // 128 for n in sizes]
    kind = torch.float8_e4m3fn if state_bits == 8 else torch.float32
    state = {"step": 0}
    for key in ("exp_avg", "exp_avg_sq"):
        state[key] = tensors(sizes, kind, lambda n: torch.zeros(n, device="cuda"))
        if state_bits == 8:
            state[key + "_scale"] = tensors(blocks_, torch.float32, lambda n: torch.zeros(n, device="cuda"))
    opt = readout.AdamW(params, lr=lr, betas=(b1, b2), eps=eps, weight_decay=decay, state_bits=state_bits, seed=seed, state=state)
    firsts = [sum(blocks_[:i]) * 128 for i in range(len(sizes))]
    for step in (1, 2):
        P = [p.double() for p in params]
        held = {}
        for key in ("exp_avg", "exp_avg_sq"):
            held[key] = [t.float().clone() for t in opt.state[key]]
            if state_bits == 8:
                held[key] = [t * s.repeat_interleave(128)[:t.numel()] for t, s in zip(held[key], opt.state[key + "_scale"])]
        grads = tensors(sizes, grad_dtype, lambda n: 0.1 * torch.randn(n, generator=g, device="cuda"))
        opt.step(grads)
        noise = uniform(firsts[-1] + sizes[-1], seed, step)
        for i, n in enumerate(sizes):
            if n == 0:
                continue
            M, V, G = held["exp_avg"][i].double(), held["exp_avg_sq"][i].double(), grads[i].double()
            m, v = b1 * M + (1 - b1) * G, b2 * V + (1 - b2) * G * G
            size = b1 * M.abs() + (1 - b1) * G.abs()  # of m's two terms
            scale = lr / (1 - b1 ** step) / (torch.sqrt(v / (1 - b2 ** step)) + eps)
            want = P[i] * (1 - lr * decay) - scale * m
            # m: four roundings of its terms; v's five count half in the root; root, quotient and settings eight more
            slack = 16 * EPS32 * scale * size + 4 * EPS32 * P[i].abs() + HALF_ULP[dtype] * want.abs()
            if dtype == torch.float16:
                slack = slack + 2.0 ** -25  # half of its smallest step
            assert torch.all((params[i].double() - want).abs() <= slack)
            if state_bits == 32:
                assert torch.all((opt.state["exp_avg"][i].double() - m).abs() <= 4 * EPS32 * size)
                assert torch.all((opt.state["exp_avg_sq"][i].double() - v).abs() <= 5 * EPS32 * v)
                continue
            # the states are defined on float32 products (m's two may cancel)
            m = (held["exp_avg"][i] * b1).double() + (grads[i].float() * (1.0 - b1)).double()
            for key, x, u in (("exp_avg", m, noise[0]), ("exp_avg_sq", v, noise[1])):
                top = tops(x.view(1, -1))
                got_scale = opt.state[key + "_scale"][i].double()
                assert torch.all((got_scale - top[0] / 448).abs() <= 8 * EPS32 * top[0] / 448)
                a = 448 * x.abs() / spread(top, n)[0]
                unit = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3)
                at = a / unit + u[firsts[i]:firsts[i] + n]
                code = torch.clamp(torch.floor(at) * unit, max=448.0)
                if key == "exp_avg_sq":
                    code = torch.where((x > 0) & (code == 0), 2.0 ** -9, code)
                got = opt.state[key][i].float().double()
                # a is off by a few float32 roundings of itself (at most 16 steps): 2^-18 of a step, beside u's grid
                near = (at - torch.round(at)).abs() <= 2.0 ** -17
                assert torch.all((got.abs() == code) | (near & ((got.abs() - code).abs() <= unit)))
                assert torch.all((got == 0) | (torch.sign(got) == torch.sign(x)))


# ---------------------------------------------------------------- beside autograd


def test_writes_in_place_are_seen_by_autograd():
    """A graph that kept what a call has written over refuses its gradient, as with torch's own in-place operations."""
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    loss = (p * p).sum()
    readout.AdamW([p]).step([torch.ones(8, device="cuda")])
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    a, b = blocks(1, 200, 100)[0], blocks(5, 30, 100)[0]
    for accumulate in (False, True):
        out = torch.ones(200, 30, device="cuda")
        x = torch.ones(200, 30, device="cuda", requires_grad=True)
        loss = (out * x).sum()
        readout.matmul(a, b, out=out, accumulate=accumulate)
        with pytest.raises(RuntimeError, match="inplace operation"):
            loss.backward()
