"""The calls that the operators around a box convolution are timed and compared on: the pointwise (1 x 1)
matrix product with its epilogue, and group norm with an activation, both on channels-last data.

``op`` names the operator, ``mode`` how it is used:

* ``infer``  the forward call without autograd;
* ``train``  the forward call and the gradients of everything that has one.

``group_norm``: ``y = act(norm(x) * weight + bias + residual)``; x is [B, C, h, w] in channels-last memory, mean
and variance are taken over the h*w pixels and C/groups channels of a group.
``linear``: ``y = act(x @ weight.T + bias + residual)``; x is [rows, K], weight [N, K]. A 1 x 1 convolution over a
channels-last image of B x h x w pixels is this product with rows = B*h*w.

act is one of "none", "relu", "silu", "gelu" (the one with the error function). Parameters of group_norm are float32 unless
``half_params``; those of linear have the type of its input.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _norm(mode, dtype, B, C, groups, h, w, act, residual=False, half_params=False, name=None):
    case = {"op": "group_norm", "mode": mode, "dtype": dtype, "B": B, "C": C, "groups": groups, "h": h, "w": w,
            "act": act, "residual": residual, "half_params": half_params}
    if name is not None:
        case["name"] = name
    return case


def _linear(mode, dtype, rows, K, N, act, bias=True, residual=False, name=None):
    case = {"op": "linear", "mode": mode, "dtype": dtype, "rows": rows, "K": K, "N": N, "act": act, "bias": bias,
            "residual": residual}
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # one 28 x 28 image behind 40 box filters: the smallest call, where latency counts
        _norm("infer", "bfloat16", 1, 40, 8, 28, 28, "relu", name="norm_infer_28x28"),
        # an encoder's feature maps at 1/4 resolution in half precision, inference
        _norm("infer", "bfloat16", 8, 128, 32, 128, 256, "silu", name="norm_infer_bf16_128x256"),
        # the end of a bottleneck block in training: norm, residual add, ReLU
        _norm("train", "bfloat16", 4, 128, 32, 128, 256, "relu", residual=True, name="norm_train_bf16_128x256"),
        # full resolution: 2 x 16 planes of 8 box filters each, float32. The largest tensors
        _norm("train", "float32", 2, 128, 32, 512, 1024, "silu", name="norm_train_fullres_512x1024"),
        # odd and ragged: an image that no tile divides, six groups of eight channels, parameters in half precision
        _norm("train", "float16", 2, 48, 6, 301, 767, "gelu", residual=True, half_params=True,
              name="norm_train_ragged_301x767"),
        # one row through a wide layer: the weights are all there is to read
        _linear("infer", "bfloat16", 1, 1024, 4096, "silu", name="linear_infer_1_row"),
        # sixteen rows back from a wide layer into a residual stream
        _linear("infer", "float16", 16, 4096, 1024, "none", residual=True, name="linear_infer_16_rows"),
        # the 1 x 1 convolution that leads into a bottleneck: 4 x 128 x 256 pixels, 128 -> 32 channels
        _linear("train", "bfloat16", 4 * 128 * 256, 128, 32, "relu", bias=True, name="linear_train_bf16_128to32"),
        # a deep block at 1/8 resolution in float32: 8 x 64 x 128 pixels, 256 -> 64 channels
        _linear("train", "float32", 8 * 64 * 128, 256, 64, "relu", name="linear_train_f32_256to64"),
        # wide layers: the products themselves are the work
        _linear("infer", "bfloat16", 8192, 2048, 4096, "gelu", name="linear_infer_bf16_wide"),
        _linear("train", "bfloat16", 8192, 4096, 2048, "silu", residual=True, name="linear_train_bf16_wide"),
        # odd and ragged: no size is a multiple of a tile or of an aligned load
        _linear("train", "float16", 1501, 333, 517, "gelu", residual=True, name="linear_train_ragged"),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


# most elements of a drawn image, and most multiplications of a drawn product: those of the largest listed cases
_MOST_ELEMENTS, _MOST_PRODUCTS = 2 * 128 * 512 * 1024, 8192 * 4096 * 2048


def draw(rng):
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    mode = rng.choice(["infer", "train"])
    act = rng.choice(["none", "relu", "silu", "gelu"])
    residual = rng.random() < 0.4
    if rng.random() < 0.5:
        groups = rng.choice([1, 4, 6, 8, 16, 32])
        per_group = rng.choice([1, 2, 3, 4, 5, 8, 16]) if groups > 1 else _log_uniform(rng, 8, 256)
        C = groups * per_group
        h, w = _log_uniform(rng, 7, 1024), _log_uniform(rng, 7, 1024)
        if rng.random() < 0.4:                       # feature maps are often multiples of 8
            h, w = max(8, h // 8 * 8), max(8, w // 8 * 8)
        B = _log_uniform(rng, 1, 32)
        while B * C * h * w > _MOST_ELEMENTS:
            if B > 1:
                B //= 2
            else:
                h, w = (h + 1) // 2, w
        return _norm(mode, dtype, B, C, groups, h, w, act, residual, half_params=rng.random() < 0.3)
    if rng.random() < 0.5:                           # pixels of feature maps through narrow layers
        rows, K, N = _log_uniform(rng, 500, 1 << 20), _log_uniform(rng, 8, 512), _log_uniform(rng, 8, 512)
    else:                                            # rows through wide layers
        rows, K, N = _log_uniform(rng, 1, 8192), _log_uniform(rng, 64, 4096), _log_uniform(rng, 64, 4096)
    if rng.random() < 0.6:                           # channels are often multiples of 8 or 32
        step = rng.choice([8, 32])
        K, N = max(step, K // step * step), max(step, N // step * step)
    most = _MOST_PRODUCTS if dtype != "float32" else _MOST_PRODUCTS // 8
    while rows * K * N > most or rows * max(K, N) > _MOST_ELEMENTS:
        rows = (rows + 1) // 2
    return _linear(mode, dtype, rows, K, N, act, rng.random() < 0.8, residual)


def _data(case, seed):
    """The tensors of a case, on the GPU, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale + shift).to(to)

    d = {"residual": None, "weight": None, "bias": None}
    if case["op"] == "group_norm":
        B, C, h, w = case["B"], case["C"], case["h"], case["w"]
        kind = dtype if case["half_params"] else torch.float32
        # feature maps: every channel has a mean and a spread of its own
        shift = torch.randn(C, generator=gen, device="cuda")
        spread = torch.rand(C, generator=gen, device="cuda") + 0.5

        def image():
            return torch.randn(B, h, w, C, generator=gen, device="cuda")
        d["x"] = image().mul_(spread).add_(shift).to(dtype).permute(0, 3, 1, 2)
        d["weight"] = normal(C, scale=0.2, shift=1.0, to=kind)
        d["bias"] = normal(C, scale=0.2, to=kind)
        if case["residual"]:
            d["residual"] = image().to(dtype).permute(0, 3, 1, 2)
        if case["mode"] == "train":
            d["grad"] = image().to(dtype).permute(0, 3, 1, 2)
    else:
        rows, K, N = case["rows"], case["K"], case["N"]
        d["x"] = normal(rows, K)
        d["weight"] = normal(N, K, scale=K ** -0.5)
        if case["bias"]:
            d["bias"] = normal(N, scale=0.2)
        if case["residual"]:
            d["residual"] = normal(rows, N)
        if case["mode"] == "train":
            d["grad"] = normal(rows, N)
    return d


def prepare(case, seed):
    state = _data(case, seed)
    state["case"] = case
    if case["mode"] == "train":
        for name in ("x", "weight", "bias", "residual"):
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# ---- the plain form ---------------------------------------------------------------------------

def _act(z, act):
    """act(z) in the type of z."""
    if act == "relu":
        return z.clamp_min(0.0)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    return z


def _slope(z, act):
    """The derivative of act at z."""
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    return torch.ones_like(z)


def _plain_norm(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    B, C, G, h, w = case["B"], case["C"], case["groups"], case["h"], case["w"]

    def rows(t):
        return t.permute(0, 2, 3, 1).reshape(B, h * w, G, C // G).float()

    def image(t):
        return t.reshape(B, h, w, C).to(dtype).permute(0, 3, 1, 2)
    x, weight, bias = rows(s["x"]), s["weight"].float().view(G, C // G), s["bias"].float().view(G, C // G)
    mean = x.mean((1, 3), keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean((1, 3), keepdim=True) + 1e-5)
    unit = centred * rstd
    z = unit * weight + bias
    if case["residual"]:
        z = z + rows(s["residual"])
    y = image(_act(z, case["act"]))
    if case["mode"] == "infer":
        return [y]
    dz = rows(s["grad"]) * _slope(z, case["act"])
    dweight, dbias = (dz * unit).sum((0, 1)), dz.sum((0, 1))
    du = dz * weight
    dx = rstd * (du - du.mean((1, 3), keepdim=True) - unit * (du * unit).mean((1, 3), keepdim=True))
    out = [y, image(dx), dweight.reshape(C).to(s["weight"].dtype), dbias.reshape(C).to(s["bias"].dtype)]
    return out + [image(dz)] if case["residual"] else out


def _plain_linear(s):
    case, dtype = s["case"], DTYPES[s["case"]["dtype"]]
    x, weight = s["x"].float(), s["weight"].float()
    z = x @ weight.t()
    if case["bias"]:
        z = z + s["bias"].float()
    if case["residual"]:
        z = z + s["residual"].float()
    y = _act(z, case["act"]).to(dtype)
    if case["mode"] == "infer":
        return [y]
    dz = s["grad"].float() * _slope(z, case["act"])
    out = [y, (dz @ weight).to(dtype), (dz.t() @ x).to(dtype)]
    if case["bias"]:
        out.append(dz.sum(0).to(dtype))
    return out + [dz.to(dtype)] if case["residual"] else out


# ---- the framework's operators ----------------------------------------------------------------

def _package():
    path = os.path.join(os.getcwd(), "box-convolutions_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import box_convolution
    return box_convolution


def _own(s):
    case, package = s["case"], _package()
    act = None if case["act"] == "none" else case["act"]
    train = case["mode"] == "train"
    with torch.set_grad_enabled(train):
        if case["op"] == "group_norm":
            y = package.group_norm_act(s["x"], case["groups"], s["weight"], s["bias"], residual=s["residual"],
                                       activation=act, eps=1e-5)
        else:
            y = package.linear_act(s["x"], s["weight"], s["bias"], residual=s["residual"], activation=act)
    if not train:
        return [y]
    wanted = [s[name] for name in ("x", "weight", "bias", "residual") if s[name] is not None]
    return [y.detach()] + list(torch.autograd.grad(y, wanted, s["grad"]))


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_norm(state) if state["case"]["op"] == "group_norm" else _plain_linear(state)


def work(case):
    """Each input read once, each output written once; two operations per multiply-add of a product, ten
    per element of a norm in each direction."""
    size = DTYPES[case["dtype"]].itemsize
    train, residual = case["mode"] == "train", int(case["residual"])
    if case["op"] == "group_norm":
        n = case["B"] * case["C"] * case["h"] * case["w"]
        tensors = (4 + 2 * residual) if train else 2 + residual      # x, y (grad, dx) and residual (and its gradient)
        params = 2 * case["C"] * (size if case["half_params"] else 4)
        return {"bytes": n * size * tensors + params * (2 if train else 1), "flops": n * (20 if train else 10)}
    rows, K, N = case["rows"], case["K"], case["N"]
    elements = rows * K + N * K + rows * N + N * int(case["bias"]) + rows * N * residual
    products = 2 * rows * K * N
    return {"bytes": size * elements * (2 if train else 1), "flops": products * (3 if train else 1)}


# ---- the definition in 64 bits ----------------------------------------------------------------

def _phi(z):
    """The normal distribution's probability below z, by the complementary error function."""
    return 0.5 * torch.special.erfc(-z / math.sqrt(2.0))


def _exact_act(z, act):
    """(act(z), its derivative)."""
    if act == "relu":
        keep = z > 0
        return torch.where(keep, z, torch.zeros_like(z)), keep.double()
    if act == "silu":
        t = torch.tanh(0.5 * z)                      # sigmoid(z) = (1 + tanh(z/2)) / 2
        s = 0.5 + 0.5 * t
        return z * s, s + 0.25 * z * (1.0 - t * t)
    if act == "gelu":
        p = _phi(z)
        return z * p, p + z * torch.exp(-z * z / 2.0) / math.sqrt(2.0 * math.pi)
    return z, torch.ones_like(z)


def exact(case, seed):
    d = _data(case, seed)
    with torch.no_grad():
        if case["op"] == "group_norm":
            return _exact_norm(case, d)
        x, weight = d["x"].double(), d["weight"].double()
        z = torch.mm(x, weight.t().contiguous())
        for extra in (d["bias"], d["residual"]):
            if extra is not None:
                z += extra.double()
        y, slope = _exact_act(z, case["act"])
        if case["mode"] == "infer":
            return [y]
        dz = slope * d["grad"].double()
        out = [y, torch.mm(dz, weight), torch.mm(dz.t().contiguous(), x)]
        if case["bias"]:
            out.append(dz.sum(0))
        return out + [dz] if case["residual"] else out


def _exact_norm(case, d):
    """One image of the batch after the other; sums over the batch at the end."""
    G, C = case["groups"], case["C"]
    per = C // G
    weight, bias = d["weight"].double(), d["bias"].double()
    ys, dxs, dzs = [], [], []
    dweight, dbias = torch.zeros_like(weight), torch.zeros_like(bias)
    for b in range(case["B"]):
        x = d["x"][b].double().reshape(G, -1)                     # [group, channel * pixel]
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        scale = 1.0 / torch.sqrt(var + 1e-5)
        unit = ((x - mean) * scale).reshape(C, -1)
        z = unit * weight[:, None] + bias[:, None]
        if d["residual"] is not None:
            z += d["residual"][b].double().reshape(C, -1)
        y, slope = _exact_act(z, case["act"])
        ys.append(y.reshape(C, case["h"], case["w"]))
        if case["mode"] == "infer":
            continue
        dz = slope * d["grad"][b].double().reshape(C, -1)
        dweight += (dz * unit).sum(1)
        dbias += dz.sum(1)
        du = (dz * weight[:, None]).reshape(G, -1)
        u = unit.reshape(G, -1)
        n = per * case["h"] * case["w"]
        dx = scale / n * (n * du - du.sum(1, keepdim=True) - u * (du * u).sum(1, keepdim=True))
        dxs.append(dx.reshape(C, case["h"], case["w"]))
        dzs.append(dz.reshape(C, case["h"], case["w"]))
    if case["mode"] == "infer":
        return [torch.stack(ys)]
    out = [torch.stack(ys), torch.stack(dxs), dweight, dbias]
    return out + [torch.stack(dzs)] if d["residual"] is not None else out
