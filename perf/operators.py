"""The operators of a readout trained on descriptor rows, as measured cases.

A readout maps SOAP rows [atoms, features] to per-atom answers: a residual
stream that is normalised and stored in 8 bits, 8-bit matrix products whose
scales belong to blocks of 128, their gradients, and the AdamW step over all of
its tensors.  ``run`` computes one pass in plain torch operations (``own``
false) or through ``mdescriptor_b200.readout`` (``own`` true).

Definitions.  e4(x) is the nearest e4m3 value (ties to even; beyond 448 it is
448).  A block of 128 entries z with A = max |z| is stored as codes
e4(448 z / A) and the scale A / 448; a block with A < 2^-100 as zeros with
scale 0.
"""

import math
import random

import torch

own = False

BLOCK = 128
TOP = 448.0
TINY = 2.0 ** -100
EPS = 1e-6
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}

# Feature counts F of this repository's benchmark configurations 1 to 5:
# 144, 3696, 1224, 2325, 2100.  Rows are atoms (or structures).


def listed():
    return [
        # The row of one structure (configuration 1, averaged over its atoms) on its way into the first product, where latency counts.
        {"name": "norm-one-row", "op": "norm", "rows": 1, "width": 144, "dtype": "float32", "residual": False},
        # The residual stream of 512 structures of configuration 5 (256 atoms each), at the width of its rows.
        {"name": "norm-stream", "op": "norm", "rows": 131072, "width": 2100, "dtype": "bfloat16", "residual": True},
        # The gradient through the norm of a shuffled minibatch of configuration-4 atoms: rows of an odd width.
        {"name": "norm-gradient-odd", "op": "norm_backward", "rows": 40001, "width": 2325, "dtype": "bfloat16", "residual": True},
        # The gradient of one layer's output, wanted along its rows (for the input's gradient) and along its columns (for the weight's).
        {"name": "blocks-both", "op": "quantize", "layout": "both", "rows": 32771, "width": 1024, "dtype": "bfloat16", "factors": False},
        # Normalised rows of configuration 2 rebuilt from the stored sum and row factors, along columns, for the weight's gradient.
        {"name": "blocks-columns-norm", "op": "quantize", "layout": "columns", "rows": 65536, "width": 3696, "dtype": "bfloat16", "factors": True},
        # A weight after its optimizer step, in tiles of 128 x 128, as it is and transposed.
        {"name": "blocks-tiles", "op": "quantize", "layout": "tiles", "rows": 1000, "width": 2100, "dtype": "float32", "factors": False},
        # One row against the first layer's weight: an answer inside a simulation's loop.
        {"name": "product-one-row", "op": "product", "m": 1, "n": 1024, "k": 3696, "scales": "tiles", "dtype": "bfloat16"},
        # Training rows of configuration 1 (64 cells of 64 atoms) against a layer as wide as configuration 5's rows.
        {"name": "product-batch", "op": "product", "m": 4096, "n": 1024, "k": 2100, "scales": "tiles", "dtype": "bfloat16"},
        # All atoms of configuration 2 (1024 cells of 128 atoms) against a wide first layer.
        {"name": "product-all-atoms", "op": "product", "m": 131072, "n": 4096, "k": 3696, "scales": "tiles", "dtype": "bfloat16"},
        # The weight's gradient of a layer: the contraction runs over an odd number of rows, both sides have a scale for each row's block.
        {"name": "product-weight-gradient", "op": "product", "m": 1024, "n": 2100, "k": 65537, "scales": "rows", "dtype": "float32"},
        # The parameters of a small readout for configuration 1: a dozen short tensors, where latency counts.
        {"name": "adamw-small", "op": "adamw", "tensors": 12, "elements": 50001, "state_bits": 32, "dtype": "float32", "grads": "float32"},
        # One readout per species, a stack of wide layers each: hundreds of tensors, states in 8 bits.
        {"name": "adamw-8-bit", "op": "adamw", "tensors": 211, "elements": 64000000, "state_bits": 8, "dtype": "float32", "grads": "bfloat16"},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_backward", "quantize", "quantize", "product", "product", "product", "product", "adamw", "adamw"])
    if op in ("norm", "norm_backward"):
        width = _log(rng, 64, 8192)
        rows = _log(rng, 1, min(262144, 131072 * 2100 // width))
        return {"op": op, "rows": rows, "width": width, "dtype": rng.choice(["float32", "bfloat16"]), "residual": rng.random() < 0.7}
    if op == "quantize":
        layout = rng.choice(["both", "columns", "tiles", "rows"])
        width = _log(rng, 64, 8192)
        rows = _log(rng, 64, 4096 if layout == "tiles" else min(131072, 65536 * 3696 // width))
        return {"op": op, "layout": layout, "rows": rows, "width": width, "dtype": "float32" if layout == "tiles" else rng.choice(["float32", "bfloat16"]),
                "factors": layout == "columns" and rng.random() < 0.5}
    if op == "product":
        kind = rng.choice(["few", "many", "gradient"])
        if kind == "few":
            return {"op": op, "m": _log(rng, 1, 128), "n": _log(rng, 64, 8192), "k": _log(rng, 64, 8192), "scales": "tiles", "dtype": rng.choice(["bfloat16", "float32"])}
        n, k = _log(rng, 64, 4096), _log(rng, 128, 4096)
        if kind == "many":
            return {"op": op, "m": _log(rng, 128, 131072), "n": n, "k": k, "scales": "tiles", "dtype": rng.choice(["bfloat16", "float32"])}
        return {"op": op, "m": n, "n": k, "k": _log(rng, 128, 131072), "scales": "rows", "dtype": "float32"}
    return {"op": op, "tensors": _log(rng, 1, 400), "elements": _log(rng, 30000, 60000000), "state_bits": rng.choice([8, 32]),
            "dtype": rng.choice(["float32", "float32", "bfloat16"]), "grads": rng.choice(["float32", "bfloat16"])}


# ---------------------------------------------------------------- inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _rows(g, rows, width, dtype):
    """Stream rows: channels of very different size, a few rows of padding atoms that are all zero."""
    x = _normal(g, rows, width) * torch.exp(_normal(g, width))
    if rows > 64:
        x[torch.randint(0, rows, (rows // 64,), generator=g, device="cuda")] = 0.0
    return x.to(dtype)


def _pitched(t, unit):
    """`t` as a view whose row pitch is a multiple of `unit` elements, as the quantiser lays its results out."""
    rows, cols = t.shape
    pitch = -(-cols // unit) * unit
    if pitch == cols:
        return t.contiguous()
    out = torch.zeros(rows, pitch, device=t.device, dtype=torch.uint8 if t.element_size() == 1 else t.dtype).view(t.dtype)
    out = out[:, :cols]
    out.copy_(t)
    return out


def _sizes(case):
    """Element counts of a readout's tensors: weights and short ones, log-normal, their sum near `elements`."""
    rng = random.Random(case["tensors"] * 1000003 + case["elements"])
    weights = [math.exp(rng.gauss(0.0, 1.5)) for _ in range(case["tensors"])]
    total = sum(weights)
    return [max(1, int(case["elements"] * w / total)) for w in weights]


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    state = {"case": dict(case)}
    if op in ("norm", "norm_backward"):
        rows, width, dtype = case["rows"], case["width"], DTYPES[case["dtype"]]
        state["x"] = _rows(g, rows, width, dtype)
        state["weight"] = 1.0 + 0.2 * _normal(g, width)
        if op == "norm":
            state["residual"] = _rows(g, rows, width, dtype) if case["residual"] else None
        else:
            x = state["x"].float()
            state["rstd"] = torch.rsqrt((x * x).mean(1) + EPS)
            state["dy"] = (_normal(g, rows, width) * 0.01).to(dtype)
            state["dsum"] = (_normal(g, rows, width) * 0.01).to(dtype) if case["residual"] else None
    elif op == "quantize":
        rows, width = case["rows"], case["width"]
        x = _normal(g, rows, width) * 0.02 if case["layout"] == "tiles" else _rows(g, rows, width, torch.float32)
        state["x"] = x.to(DTYPES[case["dtype"]])
        state["row_factor"] = state["col_factor"] = None
        if case["factors"]:
            state["row_factor"] = torch.exp(0.3 * _normal(g, rows))
            state["col_factor"] = 1.0 + 0.2 * _normal(g, width)
    elif op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        for key, rows in (("a", m), ("b", n)):
            x = _rows(g, rows, k, torch.float32) if key == "a" else _normal(g, rows, k) * 0.02
            if key == "b" and case["scales"] == "tiles":
                values, scales = _plain_tiles(x)
            else:
                values, scales = _plain_blocks(x)
            state[key] = (_pitched(values, 16), _pitched(scales, 4))
            del x, values, scales
    else:
        sizes = _sizes(case)
        starts, at = [], 0
        for size in sizes:
            starts.append(at)
            at += -(-size // BLOCK) * BLOCK  # each tensor begins on a block
        live = torch.zeros(at, device="cuda", dtype=torch.bool)
        for start, size in zip(starts, sizes):
            live[start:start + size] = True
        scale = torch.exp(1.5 * _normal(g, at // BLOCK)).repeat_interleave(BLOCK) * 1e-3 * live
        state["p"] = (0.02 * _normal(g, at) * live).to(DTYPES[case["dtype"]])
        state["g"] = (scale * _normal(g, at)).to(DTYPES[case["grads"]])
        m, v = 0.3 * scale * _normal(g, at), (scale * (0.5 + torch.rand(at, generator=g, device="cuda"))) ** 2
        if case["state_bits"] == 8:
            for key, x in (("m", m), ("v", v)):
                values, scales = _plain_blocks(x.view(-1, BLOCK))
                if key == "v":
                    values = torch.where((values.float() == 0) & (x.view(-1, BLOCK) > 0), 2.0 ** -9, values.float()).to(torch.float8_e4m3fn)
                state[key], state[key + "_scale"] = values.view(-1), scales.view(-1)
        else:
            state["m"], state["v"] = m, v
        state["step"] = 1000
        state["settings"] = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01, "seed": int(seed) & 0xFFFF}
        if own:
            from mdescriptor_b200 import readout

            def views(flat):
                return [flat[start:start + size] for start, size in zip(starts, sizes)]

            def scale_views(flat):
                return [flat[start // BLOCK:start // BLOCK + -(-size // BLOCK)] for start, size in zip(starts, sizes)]

            held = {"step": state["step"], "exp_avg": views(state["m"]), "exp_avg_sq": views(state["v"])}
            if case["state_bits"] == 8:
                held["exp_avg_scale"], held["exp_avg_sq_scale"] = scale_views(state["m_scale"]), scale_views(state["v_scale"])
            state["optimizer"] = readout.AdamW(views(state["p"]), state_bits=case["state_bits"], state=held, **state["settings"])
            state["grads"] = views(state["g"])
    return state


# ---------------------------------------------------------------- plain forms


def _codes(z, top):
    """e4(448 z / top) where `top` has z's shape; zeros where top < TINY."""
    q = torch.where(top < TINY, torch.zeros_like(z), z / (top / TOP)).clamp(-TOP, TOP)
    return q.to(torch.float8_e4m3fn)


def _spread(blocks, count):
    """A value for each block of the last dimension, for each of its `count` entries."""
    return blocks.repeat_interleave(BLOCK, dim=-1)[..., :count]


def _tops(z):
    rows, cols = z.shape
    pad = -cols % BLOCK
    z = torch.cat([z, z.new_zeros(rows, pad)], dim=1) if pad else z
    return z.abs().view(rows, -1, BLOCK).amax(dim=2)


def _scale(top):
    return torch.where(top < TINY, torch.zeros_like(top), top / TOP)


def _plain_blocks(z):
    top = _tops(z)
    return _codes(z, _spread(top, z.shape[1])), _scale(top)


def _plain_tiles(z):
    rows = z.shape[0]
    top = _tops(_tops(z).t().contiguous()).t().contiguous()
    return _codes(z, _spread(top, z.shape[1]).repeat_interleave(BLOCK, dim=0)[:rows]), _scale(top)


def _uniform(count, seed, step):
    """Two uniform numbers in [0, 1) (multiples of 2^-16) for each element and step, from a counter.

    The factors are the fractional parts of the square roots of 2, 3, 5, 7 and 11, made odd.
    """
    low = 0xFFFFFFFF
    key = (seed * 0x6A09E667 + step * 0xBB67AE85) & low
    h = torch.arange(count, device="cuda", dtype=torch.int64)
    h = (h ^ ((h >> 32) * 0x3C6EF373) ^ key) & low
    h = ((h ^ (h >> 16)) * 0xA54FF53B) & low
    h = ((h ^ (h >> 15)) * 0x510E527F) & low
    h = h ^ (h >> 16)
    return (h >> 16).float() * 2.0 ** -16, (h & 0xFFFF).float() * 2.0 ** -16


def _dithered(x, u, least):
    """|x| blocks of 128 as e4m3 codes by rounding down after adding u of a step, with `least` as the smallest non-zero code's floor."""
    top = x.abs().view(-1, BLOCK).amax(dim=1)
    scale = _scale(top)
    a = x.abs() / torch.where(scale == 0, torch.ones_like(scale), scale).repeat_interleave(BLOCK)
    unit = torch.exp2(torch.clamp(torch.frexp(a)[1] - 1, min=-6).float() - 3.0)
    q = torch.clamp(torch.floor(a / unit + u) * unit, max=TOP)
    q = torch.where((x > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q) if least else q
    q = torch.where(scale.repeat_interleave(BLOCK) == 0, torch.zeros_like(q), q)
    return (q * torch.sign(x)).to(torch.float8_e4m3fn), scale


def _plain(state):
    case, op = state["case"], state["case"]["op"]
    if op == "norm":
        s = state["x"].float()
        if state["residual"] is not None:
            s = s + state["residual"].float()
        rstd = torch.rsqrt((s * s).mean(1) + EPS)
        values, scales = _plain_blocks(s * state["weight"])
        out = {"values": values, "scales": scales * rstd[:, None], "rstd": rstd}
        if state["residual"] is not None:
            out["sum"] = s.to(state["x"].dtype)
        return out
    if op == "norm_backward":
        s, dy, rstd = state["x"].float(), state["dy"].float(), state["rstd"][:, None]
        wdy = dy * state["weight"]
        ds = rstd * wdy - s * (rstd ** 3 * (wdy * s).mean(1, keepdim=True))
        if state["dsum"] is not None:
            ds = ds + state["dsum"].float()
        return {"dx": ds.to(state["x"].dtype), "dweight": (dy * s * rstd).sum(0)}
    if op == "quantize":
        x = state["x"].float()
        if state["row_factor"] is not None:
            x = x * state["row_factor"][:, None] * state["col_factor"]
        if case["layout"] == "tiles":
            values, scales = _plain_tiles(x)
            return {"values": values, "scales": scales, "values_t": values.view(torch.uint8).t().contiguous().view(torch.float8_e4m3fn), "scales_t": scales.t().contiguous()}
        out = {}
        if case["layout"] in ("rows", "both"):
            out["values"], out["scales"] = _plain_blocks(x)
        if case["layout"] in ("columns", "both"):
            out["values_t"], out["scales_t"] = _plain_blocks(x.t().contiguous())
        return out
    if op == "product":
        k = case["k"]
        a = state["a"][0].float() * _spread(state["a"][1], k)
        b_scale = _spread(state["b"][1], k)
        if case["scales"] == "tiles":
            b_scale = b_scale.repeat_interleave(BLOCK, dim=0)[: case["n"]]
        return {"out": (a @ (state["b"][0].float() * b_scale).t()).to(DTYPES[case["dtype"]])}
    return _plain_adamw(state)


def _plain_adamw(state):
    case, settings = state["case"], state["settings"]
    state["step"] += 1
    t, (b1, b2), lr = state["step"], settings["betas"], settings["lr"]
    grad = state["g"].float()
    small = case["state_bits"] == 8
    m, v = state["m"].float(), state["v"].float()
    if small:
        m, v = m * state["m_scale"].repeat_interleave(BLOCK), v * state["v_scale"].repeat_interleave(BLOCK)
    m = b1 * m + (1.0 - b1) * grad
    v = b2 * v + (1.0 - b2) * grad * grad
    p = state["p"].float() * (1.0 - lr * settings["weight_decay"])
    p = p - (lr / (1.0 - b1 ** t)) * m / (torch.sqrt(v) * (1.0 / math.sqrt(1.0 - b2 ** t)) + settings["eps"])
    state["p"].copy_(p)
    if small:
        u, w = _uniform(m.numel(), settings["seed"], t)
        for key, x, noise in (("m", m, u), ("v", v, w)):
            values, scales = _dithered(x, noise, key == "v")
            state[key].view(torch.uint8).copy_(values.view(torch.uint8))
            state[key + "_scale"].copy_(scales)
    else:
        state["m"].copy_(m)
        state["v"].copy_(v)
    return _adamw_outputs(state)


def _adamw_outputs(state):
    return {key: state[key] for key in ("p", "m", "v", "m_scale", "v_scale") if key in state}


# ---------------------------------------------------------------- one pass


def run(state):
    if not own:
        return _plain(state)
    from mdescriptor_b200 import readout

    case, op = state["case"], state["case"]["op"]
    if op == "norm":
        r = readout.rms_norm(state["x"], state["weight"], residual=state["residual"], eps=EPS, output="float8")
        out = {"values": r.output.values, "scales": r.output.scales, "rstd": r.rstd}
        if state["residual"] is not None:
            out["sum"] = r.sum
        return out
    if op == "norm_backward":
        dx, dweight = readout.rms_norm_backward(state["dy"], state["x"], state["rstd"], state["weight"], dsum=state["dsum"])
        return {"dx": dx, "dweight": dweight}
    if op == "quantize":
        r = readout.quantize(state["x"], layout=case["layout"], row_factor=state["row_factor"], col_factor=state["col_factor"])
        out = {}
        if r.rows is not None:
            out["values"], out["scales"] = r.rows.values, r.rows.scales
        if r.columns is not None:
            out["values_t"], out["scales_t"] = r.columns.values, r.columns.scales
        return out
    if op == "product":
        return {"out": readout.matmul(readout.Blocks(*state["a"]), readout.Blocks(*state["b"]), dtype=case["dtype"])}
    state["optimizer"].step(state["grads"])
    return _adamw_outputs(state)


# ---------------------------------------------------------------- what a pass cannot do without


def work(case):
    op = case["op"]
    size = {"float32": 4, "bfloat16": 2}
    up = lambda a: -(-a // BLOCK)  # noqa: E731
    if op == "norm":
        t, d, b = case["rows"], case["width"], size[case["dtype"]]
        return {"bytes": t * d * (b * (3 if case["residual"] else 1) + 1) + 4 * t * (up(d) + 1) + 4 * d, "flops": 8 * t * d}
    if op == "norm_backward":
        t, d, b = case["rows"], case["width"], size[case["dtype"]]
        return {"bytes": t * d * b * (4 if case["residual"] else 3) + 4 * t + 8 * d, "flops": 12 * t * d}
    if op == "quantize":
        t, d, b = case["rows"], case["width"], size[case["dtype"]]
        ways = 1 if case["layout"] in ("rows", "columns") else 2
        scales = {"rows": t * up(d), "columns": d * up(t), "both": t * up(d) + d * up(t), "tiles": 2 * up(t) * up(d)}[case["layout"]]
        return {"bytes": t * d * (b + ways) + 4 * scales + (4 * (t + d) if case["factors"] else 0), "flops": 3 * t * d * ways}
    if op == "product":
        m, n, k = case["m"], case["n"], case["k"]
        scales = m * up(k) + (up(n) if case["scales"] == "tiles" else n) * up(k)
        return {"bytes": (m + n) * k + 4 * scales + m * n * size[case["dtype"]], "flops": 2 * m * n * k}
    count = sum(_sizes(case))
    state = 16 if case["state_bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": count * (2 * size[case["dtype"]] + size[case["grads"]] + state), "flops": 14 * count}


# ---------------------------------------------------------------- the definitions in 64 bits


def _e4m3(v):
    """The nearest e4m3 value of each double, ties to even, at most 448 in magnitude."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return torch.clamp(torch.round(v / step) * step, -TOP, TOP)


def _blocks64(z, tile_rows=1):
    """Codes and scales of blocks of `tile_rows` x 128 entries."""
    rows, cols = z.shape
    nr, nc = -(-rows // tile_rows), -(-cols // BLOCK)
    full = torch.zeros(nr * tile_rows, nc * BLOCK, dtype=torch.float64, device=z.device)
    full[:rows, :cols] = z
    top = full.view(nr, tile_rows, nc, BLOCK).abs().amax(dim=(1, 3))
    top = torch.where(top < TINY, torch.zeros_like(top), top)
    inverse = torch.where(top > 0, TOP / top, torch.zeros_like(top))
    codes = _e4m3(full.view(nr, tile_rows, nc, BLOCK) * inverse[:, None, :, None]).view(nr * tile_rows, nc * BLOCK)
    return codes[:rows, :cols], top / TOP


def _dithered64(x, u, least):
    full = x.abs().view(-1, BLOCK)
    top = full.amax(dim=1, keepdim=True)
    top = torch.where(top < TINY, torch.zeros_like(top), top)
    a = torch.where(top > 0, full * TOP / top, torch.zeros_like(full)).view(-1)
    step = torch.exp2(torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3.0)
    q = torch.clamp(torch.floor(a / step + u.double()) * step, max=TOP)
    if least:
        q = torch.where((a > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
    return torch.where(x < 0, -q, q), top.view(-1) / TOP


def exact(case, seed):
    state, op = prepare(case, seed), case["op"]
    d = {key: value.double() for key, value in state.items() if isinstance(value, torch.Tensor)}
    if op == "norm":
        s = d["x"] if state["residual"] is None else d["x"] + d["residual"]
        rstd = 1.0 / torch.sqrt(torch.sum(s ** 2, dim=1) / case["width"] + EPS)
        values, scales = _blocks64(s * d["weight"])
        out = {"values": values, "scales": scales * rstd[:, None], "rstd": rstd}
        if state["residual"] is not None:
            out["sum"] = s
        return out
    if op == "norm_backward":
        hat = d["x"] * d["rstd"][:, None]
        wdy = d["dy"] * d["weight"]
        ds = (wdy - hat * (torch.sum(wdy * hat, dim=1) / case["width"])[:, None]) * d["rstd"][:, None]
        if state["dsum"] is not None:
            ds = ds + d["dsum"]
        return {"dx": ds, "dweight": torch.sum(d["dy"] * hat, dim=0)}
    if op == "quantize":
        x = d["x"]
        if case["factors"]:
            x = d["row_factor"][:, None] * x * d["col_factor"][None, :]
        out = {}
        if case["layout"] == "tiles":
            out["values"], out["scales"] = _blocks64(x, BLOCK)
            out["values_t"], out["scales_t"] = out["values"].t(), out["scales"].t()
        if case["layout"] in ("rows", "both"):
            out["values"], out["scales"] = _blocks64(x)
        if case["layout"] in ("columns", "both"):
            out["values_t"], out["scales_t"] = _blocks64(x.t())
        return out
    if op == "product":
        sides = []
        for key, tall in (("a", 1), ("b", BLOCK if case["scales"] == "tiles" else 1)):
            values, scales = state[key]
            row = torch.arange(values.shape[0], device=values.device) // tall
            col = torch.arange(values.shape[1], device=values.device) // BLOCK
            sides.append(values.float().double() * scales.double()[row][:, col])
        return {"out": torch.matmul(sides[0], sides[1].t())}
    settings, t = state["settings"], state["step"] + 1
    b1, b2 = settings["betas"]
    m, v = d["m"], d["v"]
    if case["state_bits"] == 8:
        m, v = state["m"].float().double(), state["v"].float().double()
        m = (m.view(-1, BLOCK) * d["m_scale"][:, None]).view(-1)
        v = (v.view(-1, BLOCK) * d["v_scale"][:, None]).view(-1)
    m, v = m + (1.0 - b1) * (d["g"] - m), v + (1.0 - b2) * (d["g"] ** 2 - v)
    update = (m / (1.0 - b1 ** t)) / (torch.sqrt(v / (1.0 - b2 ** t)) + settings["eps"])
    out = {"p": d["p"] - settings["lr"] * (settings["weight_decay"] * d["p"] + update)}
    if case["state_bits"] == 32:
        return dict(out, m=m, v=v)
    u, w = _uniform(m.numel(), settings["seed"], t)
    out["m"], out["m_scale"] = _dithered64(m, u, False)
    out["v"], out["v_scale"] = _dithered64(v, w, True)
    return out
