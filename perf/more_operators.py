"""The calls that three operators around a box convolution are timed and compared on, all on channels-last data:

``norm``      ``residual_norm``: what lies between two blocks of a residual network. With rows x of C channels,
              ``s = residual + scale * gate * norm_after(x)``, ``h = norm_before(s)``; both norms are root-mean-square or
              layer norms over a row's channels with a weight (layer norms with a bias too). The gate is one value per channel,
              per batch item and channel, or per element.
``quantize``  ``quantize_blocks``: rows of values to 8-bit floating point (e4m3) with a power of two for each block of 128.
``product``   ``linear_act_float8``: ``act(x @ weight.T + bias + residual)`` of such rows; values are quantized in the call.
``serve``     the three together: the norm before a block hands its 8-bit rows to the block's first product.

Blocks of 128 hold ``code * 2**(exponent - 127)``: exponent - 127 is the least integer, not below -126, for which the block's largest magnitude is
at most 448 times its power of two (0 for a block of zeros), code is the value over that power, rounded to nearest, ties to even.
Rows of codes are padded to whole blocks with zeros, rows of exponents to multiples of four with 127.

``mode`` is "infer" for the forward call without autograd, "train" for the forward call and the gradients of everything that has one.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
BLOCK = 128


def _norm(mode, dtype, B, h, w, C, kind, gate, after=True, before=True, residual=True, half_params=False, name=None):
    case = {"op": "norm", "mode": mode, "dtype": dtype, "B": B, "h": h, "w": w, "C": C, "kind": kind, "gate": gate,
            "after": after, "before": before, "residual": residual, "half_params": half_params, "scale": 0.5}
    return case if name is None else {**case, "name": name}


def _quantize(dtype, rows, K, name=None):
    case = {"op": "quantize", "mode": "infer", "dtype": dtype, "rows": rows, "K": K}
    return case if name is None else {**case, "name": name}


def _product(dtype, rows, K, N, act, given="values", bias=True, residual=False, name=None):
    case = {"op": "product", "mode": "infer", "dtype": dtype, "rows": rows, "K": K, "N": N, "act": act, "given": given,
            "bias": bias, "residual": residual}
    return case if name is None else {**case, "name": name}


def _serve(dtype, rows, C, N, act, kind="rms", name=None):
    case = {"op": "serve", "mode": "infer", "dtype": dtype, "B": 1, "h": 1, "w": rows, "C": C, "rows": rows, "K": C, "N": N,
            "act": act, "kind": kind, "gate": "channel", "after": True, "before": True, "residual": True, "bias": True,
            "half_params": True, "scale": 0.5}
    return case if name is None else {**case, "name": name}


def listed():
    return [
        # one row between two blocks of a wide network: the smallest call, where latency counts
        _norm("infer", "bfloat16", 1, 1, 1, 4096, "rms", "channel", half_params=True, name="norm_infer_1_row"),
        # feature maps of an encoder at 1/4 resolution in training, each image with a gate of its own
        _norm("train", "bfloat16", 4, 128, 256, 128, "layer", "item", name="norm_train_bf16_128x256"),
        # rows of a wide residual stream in training, a layer scale per channel
        _norm("train", "bfloat16", 1, 64, 128, 4096, "rms", "channel", half_params=True, name="norm_train_bf16_wide"),
        # odd and ragged: 52 channels, an image that no tile divides, a gate per element
        _norm("train", "float16", 2, 301, 767, 52, "layer", "full", half_params=True, name="norm_train_ragged_301x767"),
        # the weights of a wide layer, once, from their float32 master copy
        _quantize("float32", 4096, 2048, name="quantize_weight_f32"),
        # rows that several products will read
        _quantize("bfloat16", 8192, 4096, name="quantize_rows_bf16"),
        # one row through a wide layer: the weights are all there is to read
        _product("bfloat16", 1, 1024, 4096, "silu", name="product_1_row"),
        # the 1 x 1 convolution that leads into a bottleneck: 4 x 128 x 256 pixels, 128 -> 32 channels
        _product("bfloat16", 4 * 128 * 256, 128, 32, "relu", name="product_bf16_128to32"),
        # a wide layer: the product itself is the work
        _product("bfloat16", 8192, 4096, 2048, "silu", residual=True, name="product_bf16_wide"),
        # odd and ragged: no size is a multiple of a tile or of a block
        _product("float16", 1501, 333, 517, "gelu", residual=True, name="product_ragged"),
        # sixteen rows between two blocks and through the next one's first layer
        _serve("bfloat16", 16, 1024, 4096, "silu", name="serve_16_rows"),
        # the same for many rows
        _serve("bfloat16", 8192, 2048, 4096, "gelu", name="serve_bf16_wide"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# most elements of a drawn tensor, and most multiplications of a drawn product: those of the largest listed cases
_MOST_ELEMENTS, _MOST_PRODUCTS = 8192 * 4096, 8192 * 4096 * 2048


def draw(rng):
    op = rng.choice(["norm", "norm", "quantize", "product", "product", "serve"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    act = rng.choice(["none", "relu", "silu", "gelu"])
    if op == "norm":
        if rng.random() < 0.5:                       # channels of feature maps
            C, h, w, B = _log_uniform(rng, 8, 512), _log_uniform(rng, 7, 1024), _log_uniform(rng, 7, 1024), _log_uniform(rng, 1, 32)
        else:                                        # rows of wide layers
            C, h, w, B = _log_uniform(rng, 256, 8192), 1, _log_uniform(rng, 1, 8192), _log_uniform(rng, 1, 8)
        if rng.random() < 0.6:
            C = max(8, C // 8 * 8)
        while B * C * h * w > _MOST_ELEMENTS // (2 if dtype == "float32" else 1):
            if B > 1:
                B //= 2
            elif h > w:
                h = (h + 1) // 2
            else:
                w = (w + 1) // 2
        after, before = rng.choice([(True, True), (True, True), (True, False), (False, True)])
        return _norm(rng.choice(["infer", "train"]), dtype, B, h, w, C, rng.choice(["rms", "layer"]),
                     rng.choice(["none", "channel", "item", "full"]), after, before, rng.random() < 0.8, rng.random() < 0.4)
    rows = _log_uniform(rng, 1, 64) if rng.random() < 0.3 else _log_uniform(rng, 64, 1 << 17)
    K, N = _log_uniform(rng, 32, 4096), _log_uniform(rng, 32, 4096)
    if rng.random() < 0.6:
        step = rng.choice([8, 128])
        K, N = max(step, K // step * step), max(step, N // step * step)
    while rows * max(K, N) > _MOST_ELEMENTS // (2 if dtype == "float32" else 1) or rows * K * N > _MOST_PRODUCTS:
        rows = (rows + 1) // 2
    if op == "quantize":
        return _quantize(dtype, rows, K)
    if op == "serve":
        return _serve(dtype, rows, K, N, act, rng.choice(["rms", "layer"]))
    return _product(dtype, rows, K, N, act, rng.choice(["values", "values", "codes"]), rng.random() < 0.8, rng.random() < 0.4)


# ---- blocks of 128 in 8 bits ------------------------------------------------------------------

def _pad(x, to):
    """Rows padded with zeros to a multiple of `to`."""
    more = -x.shape[-1] % to
    return torch.cat([x, x.new_zeros(*x.shape[:-1], more)], -1) if more else x


def _power(e):
    """2**e as float32, e of int32 in [-126, 127], exactly."""
    return ((e + 127) << 23).view(torch.float32)


def _to_blocks(x):
    """(codes as float8_e4m3fn, exponents as uint8) of rows of float32 values, in the layout described above."""
    x = _pad(x, BLOCK)
    parts = x.reshape(*x.shape[:-1], -1, BLOCK)
    mantissa, exponent = torch.frexp(parts.abs().amax(-1))            # mantissa in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp_min(-126)
    e = torch.where(mantissa == 0, torch.zeros_like(e), e)
    codes = (parts * _power(-e[..., None])).to(torch.float8_e4m3fn).reshape(x.shape)
    e = (e + 127).to(torch.uint8)
    more = -e.shape[-1] % 4
    return codes, torch.cat([e, e.new_full((*e.shape[:-1], more), 127)], -1).contiguous() if more else e


def _from_blocks(codes, exponents, K):
    """The float32 values that [rows, K] codes stand for."""
    parts = codes.float().reshape(codes.shape[0], -1, BLOCK)
    power = exponents[:, :parts.shape[1], None].int() - 127
    return (parts * _power(power)).reshape(codes.shape)[:, :K]


# ---- data -------------------------------------------------------------------------------------

def _data(case, seed):
    """The tensors of a case, on the GPU, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(to)

    d = {}
    if case["op"] in ("norm", "serve"):
        B, h, w, C = (case[k] for k in ("B", "h", "w", "C"))
        kind = dtype if case["half_params"] else torch.float32
        # channels of different mean and size, as behind an activation or a residual stream
        shift, spread = normal(C, scale=0.3, to=torch.float32), torch.rand(C, generator=gen, device="cuda") + 0.5

        def image(scale=1.0):
            x = torch.randn(B, h, w, C, generator=gen, device="cuda").mul_(spread).add_(shift).mul_(scale)
            return x.to(dtype).permute(0, 3, 1, 2)
        d["x"] = image()
        if case["residual"]:
            d["residual"] = image(2.0)
        if case["gate"] == "channel":
            d["gate"] = normal(C, scale=0.2, shift=0.5, to=kind)
        elif case["gate"] == "item":
            d["gate"] = normal(B, C, scale=0.5, shift=0.5)
        elif case["gate"] == "full":
            d["gate"] = torch.sigmoid(image().float()).to(dtype)
        for at in ("after", "before"):
            if case[at]:
                d[at + "_weight"] = normal(C, scale=0.2, shift=1.0, to=kind)
                if case["kind"] == "layer":
                    d[at + "_bias"] = normal(C, scale=0.2, to=kind)
        if case["mode"] == "train":
            d["grad_stream"] = image()
            if case["before"]:
                d["grad_normed"] = image()
    if case["op"] == "quantize":
        d["x"] = _rows(gen, case["rows"], case["K"]).to(dtype)
    if case["op"] in ("product", "serve"):
        rows, K, N = case["rows"], case["K"], case["N"]
        if case["op"] == "product":
            d["x"] = _rows(gen, rows, K).to(dtype)
            if case["given"] == "codes":
                d["x_codes"], d["x_exponents"] = _to_blocks(d.pop("x").float())
        d["weight_codes"], d["weight_exponents"] = _to_blocks(_rows(gen, N, K, K ** -0.5))
        d["linear_bias"] = normal(N, scale=0.2) if case["bias"] else None
        d["linear_residual"] = normal(rows, N) if case.get("residual") and case["op"] == "product" else None
    return d


def _rows(gen, rows, K, scale=1.0):
    """Activations or weights: normal, with a few channels that are many times larger than the rest."""
    channel = torch.exp(0.7 * torch.randn(K, generator=gen, device="cuda"))
    return torch.randn(rows, K, generator=gen, device="cuda") * (channel * scale)


_LEAVES = ("x", "residual", "gate", "after_weight", "after_bias", "before_weight", "before_bias")


def prepare(case, seed):
    state = _data(case, seed)
    if case["mode"] == "train":
        for name in _LEAVES:
            if name in state:
                state[name].requires_grad_(True)
    state["case"] = case
    return state


# ---- the plain form ---------------------------------------------------------------------------

def _act(z, act):
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    return z


def _unit(v, kind):
    """(v normalised over its last axis, one over its deviation)."""
    centred = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    rstd = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + 1e-6)
    return centred * rstd, rstd


def _unit_grad(g, unit, rstd, kind):
    """The gradient of v from that of the normalised v."""
    g = g - unit * (g * unit).mean(-1, keepdim=True) - (g.mean(-1, keepdim=True) if kind == "layer" else 0.0)
    return g * rstd


def _between(s):
    """What the plain norm computes of a state's rows: every piece in float32 as [B, h * w, C]."""
    case = s["case"]

    def rows(t):
        return t.permute(0, 2, 3, 1).reshape(case["B"], -1, case["C"]).float()
    p = {"x": rows(s["x"])}
    unit, p["rstd_x"] = _unit(p["x"], case["kind"]) if case["after"] else (p["x"], None)
    p["unit_x"] = unit
    if case["after"]:
        unit = unit * s["after_weight"].float()
        if "after_bias" in s:
            unit = unit + s["after_bias"].float()
    p["u"] = unit
    gate = s.get("gate")
    if gate is not None:
        gate = {"channel": lambda: gate.float(), "item": lambda: gate.float()[:, None, :], "full": lambda: rows(gate)}[case["gate"]]()
        unit = unit * gate
    p["gate"] = gate
    p["stream"] = unit * case["scale"]
    if case["residual"]:
        p["stream"] = rows(s["residual"]) + p["stream"]
    if case["before"]:
        p["unit_s"], p["rstd_s"] = _unit(p["stream"], case["kind"])
        p["normed"] = p["unit_s"] * s["before_weight"].float()
        if "before_bias" in s:
            p["normed"] = p["normed"] + s["before_bias"].float()
    return p, rows


def _plain_norm(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    kind = case["kind"]

    def image(t):
        return t.reshape(case["B"], case["h"], case["w"], case["C"]).to(dtype).permute(0, 3, 1, 2)
    p, rows = _between(s)
    out = {"stream": image(p["stream"])}
    if case["before"]:
        out["normed"] = image(p["normed"])
    if case["mode"] == "infer":
        return out
    ds, like = rows(s["grad_stream"]), {name: s[name].dtype for name in _LEAVES if name in s}
    if case["before"]:
        dh = rows(s["grad_normed"])
        out["before_weight"] = (dh * p["unit_s"]).sum((0, 1)).to(like["before_weight"])
        if kind == "layer":
            out["before_bias"] = dh.sum((0, 1)).to(like["before_bias"])
        ds = ds + _unit_grad(dh * s["before_weight"].float(), p["unit_s"], p["rstd_s"], kind)
    if case["residual"]:
        out["residual"] = image(ds)
    du = ds * case["scale"]
    if p["gate"] is not None:
        dg = du * p["u"]
        out["gate"] = image(dg) if case["gate"] == "full" else dg.sum(1 if case["gate"] == "item" else (0, 1)).to(like["gate"])
        du = du * p["gate"]
    if case["after"]:
        out["after_weight"] = (du * p["unit_x"]).sum((0, 1)).to(like["after_weight"])
        if kind == "layer":
            out["after_bias"] = du.sum((0, 1)).to(like["after_bias"])
        du = _unit_grad(du * s["after_weight"].float(), p["unit_x"], p["rstd_x"], kind)
    out["x"] = image(du)
    return out


def _plain_product(s, x):
    """x: float32 values on the grid of their blocks."""
    z = x @ _from_blocks(s["weight_codes"], s["weight_exponents"], s["case"]["K"]).t()
    if s["linear_bias"] is not None:
        z = z + s["linear_bias"].float()
    if s["linear_residual"] is not None:
        z = z + s["linear_residual"].float()
    return _act(z, s["case"]["act"]).to(DTYPES[s["case"]["dtype"]])


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        return _plain_norm(s)
    if case["op"] == "quantize":
        return list(_to_blocks(s["x"].float()))
    if case["op"] == "serve":
        p, _ = _between(s)
        stream = p["stream"].reshape(1, 1, -1, case["C"]).to(DTYPES[case["dtype"]]).permute(0, 3, 1, 2)
        blocks = _to_blocks(p["normed"][0])
        return {"stream": stream, "y": _plain_product(s, _from_blocks(*blocks, case["K"]))}
    given = (s["x_codes"], s["x_exponents"]) if case["given"] == "codes" else _to_blocks(s["x"].float())
    return [_plain_product(s, _from_blocks(*given, case["K"]))]


# ---- the framework's operators ----------------------------------------------------------------

def _package():
    path = os.path.join(os.getcwd(), "box-convolutions_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import box_convolution
    return box_convolution


def _own(s):
    case, package = s["case"], _package()
    op, train = case["op"], case["mode"] == "train"
    act = None if case.get("act") in (None, "none") else case["act"]
    with torch.set_grad_enabled(train):
        if op == "quantize":
            blocks = package.quantize_blocks(s["x"])
            return [blocks.codes, blocks.exponents]
        if op in ("norm", "serve"):
            after = (s["after_weight"], s.get("after_bias")) if case["after"] else None
            before = (s["before_weight"], s.get("before_bias")) if case["before"] else None
            out = package.residual_norm(s["x"], s.get("residual"), s.get("gate"), case["scale"], after=after, before=before,
                                        kind=case["kind"], eps=1e-6, quantize=op == "serve")
        if op in ("product", "serve"):
            weight = package.Float8Blocks(s["weight_codes"], s["weight_exponents"], case["K"])
            x = out[1] if op == "serve" else s["x"] if case["given"] == "values" else package.Float8Blocks(
                s["x_codes"], s["x_exponents"], case["K"])
            y = package.linear_act_float8(x, weight, s["linear_bias"], residual=s["linear_residual"], activation=act,
                                          dtype=DTYPES[case["dtype"]])
            return [y] if op == "product" else {"stream": out[0], "y": y.reshape(case["rows"], case["N"])}
    stream, normed = out if case["before"] else (out, None)
    found = {"stream": stream.detach()}
    if case["before"]:
        found["normed"] = normed.detach()
    if train:
        names = [name for name in _LEAVES if name in s]
        outputs, grads = ([stream, normed], [s["grad_stream"], s["grad_normed"]]) if case["before"] else ([stream], [s["grad_stream"]])
        found.update(zip(names, torch.autograd.grad(outputs, [s[name] for name in names], grads)))
    return found


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    """Each input read once, each output written once; two operations per multiply-add of a product, 12 per element and norm
    forward and 20 backward, 4 per quantized value."""
    size = DTYPES[case["dtype"]].itemsize
    nbytes = flops = 0
    if case["op"] in ("norm", "serve"):
        n = case["B"] * case["h"] * case["w"] * case["C"]
        r, full, norms = int(case["residual"]), int(case["gate"] == "full"), int(case["after"]) + int(case["before"])
        before = int(case["before"]) if case["op"] == "norm" else 0        # (serve: the normed rows stay in 8 bits between the two)
        nbytes = n * size * (2 + r + full + before)
        flops = 12 * norms * n
        if case["mode"] == "train":
            nbytes += n * size * (3 + 2 * r + 2 * full + before)           # x, grads, dx; residual's and gate's
            flops += 20 * norms * n
    if case["op"] == "quantize":
        n = case["rows"] * case["K"]
        return {"bytes": n * size + n + n // BLOCK, "flops": 4 * n}
    if case["op"] in ("product", "serve"):
        rows, K, N = case["rows"], case["K"], case["N"]
        if case["op"] == "product":
            nbytes += rows * K * (1 if case["given"] == "codes" else size) + (rows * N * size if case["residual"] else 0)
        nbytes += N * K + N * K // BLOCK + rows * N * size
        flops += 2 * rows * K * N
    return {"bytes": nbytes, "flops": flops}


# ---- the definition in 64 bits ----------------------------------------------------------------

def _two_to(e):
    """2**e of whole numbers in 64 bits; the general power may be a rounding off."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _grid(x):
    """([rows, K] values of the 8-bit format in units of each block's power, the powers' exponents per block), in 64 bits."""
    rows, K = x.shape
    full = torch.zeros(rows, -(-K // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :K] = x
    full = full.view(rows, -1, BLOCK)
    most = full.abs().max(-1).values
    e = torch.ceil(torch.log2((most / 448.0).clamp_min(2.0 ** -300)))
    e = torch.where(most > 448.0 * _two_to(e), e + 1, torch.where(most <= 448.0 * _two_to(e - 1), e - 1, e))    # (log2's rounding)
    e = torch.where(most > 0, e.clamp_min(-126.0), torch.zeros_like(e))
    units = full / _two_to(e)[..., None]
    step = _two_to(torch.floor(torch.log2(units.abs().clamp_min(2.0 ** -6))) - 3)       # three digits behind the leading one; subnormals below 2^-6
    step = torch.where(units.abs() >= 16 * step, 2 * step, step)                        # (log2's rounding)
    step = torch.where((units.abs() < 8 * step) & (step > 2.0 ** -9), step / 2, step)
    return torch.round(units / step) * step, e


def _grid_values(x):
    units, e = _grid(x)
    return (units * _two_to(e)[..., None]).reshape(x.shape[0], -1)[:, :x.shape[1]]


def _stored_values(codes, exponents, K):
    each = torch.repeat_interleave(_two_to(exponents.to(torch.int64) - 127), BLOCK, dim=1)
    return codes.double()[:, :K] * each[:, :K]


def _exact_product(case, d, x):
    z = torch.mm(x, _stored_values(d["weight_codes"], d["weight_exponents"], case["K"]).t().contiguous())
    for extra in (d["linear_bias"], d["linear_residual"]):
        if extra is not None:
            z += extra.double()
    if case["act"] == "relu":
        return z.clamp(min=0.0)
    if case["act"] == "silu":
        return z * (0.5 + 0.5 * torch.tanh(0.5 * z))
    if case["act"] == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    return z


def _exact_norms(case, d, leaves):
    """(stream, normed or None) as [B, C, h, w], from `leaves` in 64 bits."""
    def norm(v, at):
        if case["kind"] == "layer":
            v = v - v.sum(1, keepdim=True) / case["C"]
        v = v / torch.sqrt(v.square().sum(1, keepdim=True) / case["C"] + 1e-6)
        v = v * leaves[at + "_weight"].view(1, -1, 1, 1)
        return v + leaves[at + "_bias"].view(1, -1, 1, 1) if at + "_bias" in leaves else v
    t = norm(leaves["x"], "after") if case["after"] else leaves["x"]
    if "gate" in leaves:
        g = leaves["gate"]
        t = t * (g.view(1, -1, 1, 1) if case["gate"] == "channel" else g[:, :, None, None] if case["gate"] == "item" else g)
    t = case["scale"] * t
    if "residual" in leaves:
        t = leaves["residual"] + t
    return t, norm(t, "before") if case["before"] else None


def exact(case, seed):
    d = _data(case, seed)
    if case["op"] == "quantize":
        units, e = _grid(d["x"].double())
        more = torch.full((case["rows"], -e.shape[1] % 4), 127.0, dtype=torch.float64, device=e.device)
        return [units.reshape(case["rows"], -1), torch.cat([e + 127.0, more], 1).to(torch.uint8)]
    if case["op"] == "product":
        x = _stored_values(d["x_codes"], d["x_exponents"], case["K"]) if case["given"] == "codes" else _grid_values(d["x"].double())
        return [_exact_product(case, d, x)]
    train = case["mode"] == "train"
    leaves = {name: d[name].double().requires_grad_(train) for name in _LEAVES if name in d}
    with torch.set_grad_enabled(train):
        stream, normed = _exact_norms(case, d, leaves)
    if case["op"] == "serve":
        return {"stream": stream, "y": _exact_product(case, d, _grid_values(normed[0, :, 0, :].t().contiguous()))}
    out = {"stream": stream.detach()}
    if normed is not None:
        out["normed"] = normed.detach()
    if train:
        outputs, grads = ([stream, normed], ["grad_stream", "grad_normed"]) if normed is not None else ([stream], ["grad_stream"])
        out.update(zip(leaves, torch.autograd.grad(outputs, list(leaves.values()), [d[g].double() for g in grads])))
    return out
