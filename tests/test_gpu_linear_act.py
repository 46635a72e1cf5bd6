"""``linear_act`` and ``PointwiseConv2d`` against the product in 64 bits (tests/operator_reference.py derives the
bounds), at sizes, strides, alignments and values where tiles, vectors and splits end."""
import pytest
import torch

import operator_reference as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "silu", "gelu"]


def make(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, dtype=torch.float64) * scale).to(dtype)


def run(x, weight, bias, residual, name, grad, like=None):
    """Host tensors in, {output: device tensor} out; `like` makes the device tensor of a host tensor (default: a copy)."""
    from box_convolution import linear_act
    like = like or (lambda t: t.cuda())
    dev = {k: like(t).detach().requires_grad_(grad is not None) for k, t in
           (("x", x), ("weight", weight), ("bias", bias), ("residual", residual)) if t is not None}
    y = linear_act(dev["x"], dev["weight"], dev.get("bias"), residual=dev.get("residual"), activation=name)
    out = {"y": y}
    if grad is not None:
        out.update(zip(dev, torch.autograd.grad(y, list(dev.values()), like(grad))))
    return out


def case(M, K, N, dtype, name, bias=True, residual=False, seed=0, train=True):
    gen = torch.Generator().manual_seed(seed + 7 * M + 11 * K + 13 * N)
    x, weight = make((M, K), gen, dtype), make((N, K), gen, dtype, max(K, 1) ** -0.5)
    b = make((N,), gen, dtype) if bias else None
    r = make((M, N), gen, dtype) if residual else None
    g = make((M, N), gen, dtype) if train else None
    return x, weight, b, r, name, g


def expected(x, weight, b, r, name, g, dtype):
    d = [None if t is None else t.double() for t in (x, weight, b, r)]
    return ref.linear(*d, name, None if g is None else g.double(), dtype)


SIZES = [(1, 1, 1), (1, 64, 64), (2, 8, 200), (3, 5, 7), (16, 128, 32), (17, 1000, 24), (63, 65, 64), (65, 63, 66), (128, 128, 128),
         (129, 130, 257), (200, 32, 128), (257, 100, 60), (1000, 40, 8), (1, 333, 517), (16, 2048, 256), (300, 8, 16), (4099, 33, 129),
         (5000, 128, 32), (2048, 16, 16), (700, 520, 264), (33, 24, 1030), (1, 4096, 40), (8, 72, 1024)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_sizes(hip, i, dtype):
    """Every size with one activation (another for each type) and every second with a residual, forward and backward."""
    M, K, N = SIZES[i]
    args = case(M, K, N, dtype, ACTS[(i + TYPES.index(dtype)) % 4], bias=i % 3 != 2, residual=i % 2 == 1)
    ref.check(run(*args), expected(*args, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, True)])
def test_epilogues(hip, name, bias, residual, dtype):
    for M, K, N in ((130, 72, 136), (7, 72, 136), (3000, 64, 48)):
        args = case(M, K, N, dtype, name, bias, residual, seed=5)
        ref.check(run(*args), expected(*args, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_products(hip, dtype):
    """Tiles of the wide kernels, whole ones and a rest on every side, and a long sum."""
    for M, K, N in ((640, 512, 768), (1030, 584, 1096), (264, 8200, 256)):
        args = case(M, K, N, dtype, "silu", residual=True)
        ref.check(run(*args), expected(*args, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(70, 40, 72), (3000, 64, 32), (520, 256, 512), (5, 136, 264)])
def test_rows_apart_and_any_address(hip, M, K, N, dtype):
    """Inputs inside larger tensors that hold NaN around them: nothing outside is used, at addresses of one element."""
    args = case(M, K, N, dtype, "gelu", residual=True, seed=3)
    for shift in (0, 1):
        def inside(t):
            if t.dim() == 1:
                big = torch.full((t.numel() + 2,), float("nan"), dtype=t.dtype, device="cuda")
                view = big[shift:shift + t.numel()]
            else:
                big = torch.full((t.size(0) + 2, t.size(1) + 8), float("nan"), dtype=t.dtype, device="cuda")
                view = big[1:1 + t.size(0), shift * 3:shift * 3 + t.size(1)]
            view.copy_(t)
            return view
        ref.check(run(*args, like=inside), expected(*args, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_that_are_copied_or_broadcast(hip, dtype):
    from box_convolution import linear_act
    gen = torch.Generator().manual_seed(1)
    x, w = make((48, 33), gen, dtype).cuda(), make((33, 20), gen, dtype).cuda()
    plain = linear_act(x, w.t().contiguous())
    assert torch.equal(linear_act(x.t().contiguous().t(), w.t()), plain)
    assert torch.equal(linear_act(x.view(4, 3, 4, 33), w.t()), plain.view(4, 3, 4, 20))
    row = x[:1].expand(300, 33).detach().requires_grad_(True)          # rows 0 elements apart
    one = x[:1].repeat(300, 1).requires_grad_(True)
    g = make((300, 20), gen, dtype).cuda()
    assert torch.equal(linear_act(row, w.t()), linear_act(one, w.t()))
    assert torch.equal(torch.autograd.grad(linear_act(row, w.t()), row, g)[0], torch.autograd.grad(linear_act(one, w.t()), one, g)[0])
    # a broadcast gradient (of a sum) and a single vector as input
    w2 = w.t().contiguous().requires_grad_(True)
    a = torch.autograd.grad(linear_act(x, w2, activation="silu").sum(), w2)[0]
    b = torch.autograd.grad(linear_act(x, w2, activation="silu"), w2, torch.ones(48, 20, dtype=dtype, device="cuda"))[0]
    assert torch.equal(a, b)
    assert torch.equal(linear_act(x[0], w2), linear_act(x[:1], w2)[0])


@pytest.mark.parametrize("dtype", TYPES)
def test_empty(hip, dtype):
    for M, K, N in ((0, 5, 7), (4, 0, 6), (4, 5, 0), (0, 0, 0)):
        args = case(M, K, N, dtype, "gelu", residual=True)
        ref.check(run(*args), expected(*args, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(40, 40, 40), (2000, 64, 32), (600, 264, 520), (4, 512, 96)])
def test_nan_and_infinity_stay_in_their_row_and_column(hip, M, K, N, dtype):
    x, w, b, _, _, g = case(M, K, N, dtype, None)
    x[1, 3], x[2, 0], w[5, 1] = float("nan"), float("inf"), float("-inf")
    with torch.no_grad():
        out = run(x, w, b, None, None, None)["y"].double().cpu()
    z = x.double() @ w.double().t() + b.double()
    assert torch.equal(out.isnan(), z.isnan()) and torch.equal(out.isinf(), z.isinf())
    # a NaN in the gradient stays in its row of dx and its row of dweight
    g[2, 4] = float("nan")
    out = run(*case(M, K, N, dtype, None)[:5], g)
    assert out["x"].isnan().any(1).nonzero().flatten().tolist() == [2]
    assert out["weight"].isnan().any(1).nonzero().flatten().tolist() == [4]
    assert out["bias"].isnan().nonzero().flatten().tolist() == [4]
    for name in ("relu", "silu", "gelu"):                              # and one in z reaches the gradients
        x, w, b, _, _, g = case(M, K, N, dtype, name)
        x[1, 3] = float("nan")
        out = run(x, w, b, None, name, g)
        assert out["y"][1].isnan().all() and not out["y"][0].isnan().any()
        if name != "relu":                                             # (no comparison with NaN is true: relu's derivative is 0 there)
            assert out["x"][1].isnan().all()


@pytest.mark.parametrize("name", [None, "silu", "gelu"])
def test_gradients_against_differences(hip, name):
    """Central differences of the operator itself along a random direction. Bounds: the forward's own error over the
    step, and the change of the 64-bit quotient when the step is doubled (three times a step's truncation error where the
    function is smooth: relu, whose kinks a step crosses, is held to its formula alone)."""
    M, K, N, h = 37, 45, 29, 2.0 ** -7
    x, w, b, r, _, g = case(M, K, N, torch.float32, name, residual=True, seed=9)
    grads = run(x, w, b, r, name, g)
    base = {"x": x, "weight": w, "bias": b, "residual": r}
    gen = torch.Generator().manual_seed(2)
    for which in base:
        v = torch.randn(base[which].shape, generator=gen)

        def loss(step, exact):
            t = dict(base)
            t[which] = t[which].double() + step * v.double() if exact else (t[which].double() + step * v.double()).float()
            if exact:
                y = ref.linear(*[t[k].double() for k in base], name, None, torch.float32)["y"][0]
            else:
                y = run(t["x"], t["weight"], t["bias"], t["residual"], name, None)["y"].double().cpu()
            return (y * g.double()).sum().item()
        quotient = (loss(h, False) - loss(-h, False)) / (2 * h)
        exact = [(loss(s, True) - loss(-s, True)) / (2 * s) for s in (h, 2 * h)]
        bound = (ref.linear(*[t.double() for t in base.values()], name, None, torch.float32)["y"][1] * g.double().abs()).sum().item()
        rounding = 2.0 ** -24 * (base[which].double().abs() * grads[which].double().cpu().abs()).sum().item()
        got = (grads[which].double().cpu() * v.double()).sum().item()
        assert abs(got - quotient) <= 2 * (bound + rounding) / h + 2 * abs(exact[1] - exact[0]) + 1e-6 * abs(got), which


def test_only_what_is_needed(hip):
    from box_convolution import linear_act
    gen = torch.Generator().manual_seed(4)
    x, w, b, r, g = (make(s, gen, torch.bfloat16).cuda() for s in ((50, 24), (40, 24), (40,), (50, 40), (50, 40)))
    for name in ACTS:
        full = [t.detach().requires_grad_(True) for t in (x, w, b, r)]
        whole = torch.autograd.grad(linear_act(full[0], full[1], full[2], full[3], name), full, g)
        for i in range(4):
            some = [t.detach().requires_grad_(i == k) for k, t in enumerate((x, w, b, r))]
            assert torch.equal(torch.autograd.grad(linear_act(*some, name), some[i], g)[0], whole[i])


def test_another_stream_and_same_bits(hip):
    """The same call on a stream of its own, twice: the same bits everywhere (no order of additions is left open)."""
    args = case(3000, 96, 72, torch.bfloat16, "silu", residual=True)
    first = run(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(*args)
    side.synchronize()
    for k in first:
        assert torch.equal(first[k], second[k]), k


def test_graph_replays(hip):
    x, w, b, r, _, g = (t.cuda() if torch.is_tensor(t) else t for t in case(600, 72, 40, torch.float16, "gelu", residual=True))

    def step():
        y, kept = hip.linear_forward(x, w, b, r, "gelu", True)
        return [y] + hip.linear_backward(x, w, kept, "gelu", g, (True,) * 4)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        x.copy_(x.roll(k + 1, 0))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        for a, e in zip(got, step()):
            assert torch.equal(a, e)


def test_pointwise_conv(hip):
    """The module is the 1 x 1 convolution of its parameters, on channels-last images and on others."""
    from box_convolution import PointwiseConv2d
    torch.manual_seed(3)
    module = PointwiseConv2d(24, 40, activation="relu").cuda()
    plain = torch.nn.Conv2d(24, 40, 1)
    plain.load_state_dict(module.state_dict())
    x, r = torch.randn(2, 24, 9, 13), torch.randn(2, 40, 9, 13)
    e = ref.linear(x.double().permute(0, 2, 3, 1).reshape(-1, 24), plain.weight.detach().double().flatten(1), plain.bias.detach().double(),
                   r.double().permute(0, 2, 3, 1).reshape(-1, 40), "relu", None, torch.float32)
    for layout in (torch.channels_last, torch.contiguous_format):
        y = module(x.cuda().to(memory_format=layout), r.cuda().to(memory_format=layout))
        assert y.shape == r.shape and y.is_contiguous(memory_format=torch.channels_last)
        ref.check({"y": y.permute(0, 2, 3, 1)}, e)


@pytest.fixture(params=["C++", "Python"])
def host_side(request, hip, monkeypatch):
    """Both host sides of the operators (the second one is what runs where the C++ extension was not built)."""
    if request.param == "Python":
        monkeypatch.setattr(hip, "_glue", False)
        assert hip.glue() is None
    elif hip.glue() is None:
        pytest.skip("the C++ extension was not built")
    return request.param


@pytest.mark.parametrize("dtype", TYPES)
def test_both_host_sides(host_side, dtype):
    for name in ACTS:
        args = case(70, 40, 24, dtype, name, bias=name != "relu", residual=name != "silu")
        ref.check(run(*args), expected(*args, dtype))
        args = case(0, 40, 24, dtype, name, residual=True)
        ref.check(run(*args), expected(*args, dtype))


def test_refusals(host_side):
    from box_convolution import PointwiseConv2d, linear_act
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    for bad, match in ((lambda: linear_act(x, w[:, :7]), "weight"), (lambda: linear_act(x, w[0]), "weight"),
                       (lambda: linear_act(x, w.half()), "weight"), (lambda: linear_act(x, w.cpu()), "weight"),
                       (lambda: linear_act(x, w, torch.zeros(5, device="cuda")), "bias"),
                       (lambda: linear_act(x, w, torch.zeros(6, device="cuda", dtype=torch.bfloat16)), "bias"),
                       (lambda: linear_act(x, w, residual=torch.zeros(1, 6, device="cuda")), "residual"),
                       (lambda: linear_act(x.double(), w.double()), "float32, float16 or bfloat16"),
                       (lambda: linear_act(x, w, activation="tanh"), "activation"),
                       (lambda: linear_act(x.cpu(), w), "AMD GPUs only"),
                       (lambda: PointwiseConv2d(3, 4, activation="tanh"), "activation"),
                       (lambda: PointwiseConv2d(3, 4).cuda()(torch.zeros(3, 5, 5, device="cuda")), "4 dimensions")):
        with pytest.raises(RuntimeError, match=match):
            bad()


def test_not_twice(host_side):
    """Gradients of gradients are refused, not taken for zero; asking for a graph alone changes no gradient."""
    from box_convolution import linear_act
    x, w = torch.randn(5, 8, device="cuda"), torch.randn(6, 8, device="cuda", requires_grad=True)
    r = torch.randn(5, 6, device="cuda", requires_grad=True)
    once = torch.autograd.grad(linear_act(x, w, residual=r, activation="silu").sum(), [w, r])
    again = torch.autograd.grad(linear_act(x, w, residual=r, activation="silu").sum(), [w, r], create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(once, again))
    for g in again:
        with pytest.raises(RuntimeError, match="not twice"):
            g.square().sum().backward()


@pytest.mark.parametrize("K,N", [(64, 64), (33, 64)])
def test_more_than_2_31_elements(hip, K, N):
    """Rows whose elements lie beyond 2^31 of each tensor, through few channels (whole chunks, and any alignment): the first and
    the last rows against the product of those rows alone, and the weight's gradient against the sum over halves."""
    from box_convolution import linear_act
    rows = (1 << 31) // 33 + 1000
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(rows, K, generator=gen, device="cuda", dtype=torch.bfloat16)
    w = torch.randn(N, K, generator=gen, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    g = torch.randn(rows, N, generator=gen, device="cuda", dtype=torch.bfloat16)
    assert x.numel() > 1 << 31 and g.numel() > 1 << 31
    x.requires_grad_(True)
    y = linear_act(x, w, activation="relu")
    dx, dw = torch.autograd.grad(y, (x, w), g)
    for part in (slice(0, 700), slice(rows - 700, rows)):
        xs = x.detach()[part].clone().requires_grad_(True)
        ys = linear_act(xs, w, activation="relu")
        assert torch.equal(ys, y[part])
        # (another kernel may take so few rows: one more rounding of dx)
        ds = torch.autograd.grad(ys, xs, g[part])[0]
        assert (ds.double() - dx[part].double()).abs().max() <= 2.0 ** -7 * ds.double().abs().max()
    half = rows // 2
    sums = torch.zeros(N, K, dtype=torch.float64, device="cuda")
    for part in (slice(0, half), slice(half, rows)):
        xs, ws = x.detach()[part], w.detach().clone().requires_grad_(True)
        sums += torch.autograd.grad(linear_act(xs, ws, activation="relu"), ws, g[part])[0].double()
    assert (sums - dw.double()).abs().max() <= 3 * 2.0 ** -8 * dw.double().abs().max()      # three bfloat16 roundings


@pytest.mark.parametrize("K", [4, 8, 12])
@pytest.mark.parametrize("N", [4, 8, 12])
def test_few_channels_on_both_sides(hip, K, N):
    """float32 layers whose tiles take less LDS than the bias sums of all 512 threads would: only the rows of a tile are kept there."""
    for M in (33, 70, 5000):
        args = case(M, K, N, torch.float32, "relu", residual=K == N)
        ref.check(run(*args), expected(*args, torch.float32))


@pytest.mark.parametrize("unpack", [lambda t: torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t),
                                    lambda t: t.t().contiguous().t()])
def test_saved_tensors_of_another_layout(host_side, unpack):
    """Hooks on saved tensors may give the values back in any memory order."""
    for M, K, N in ((70, 40, 24), (600, 264, 520)):
        for name in ACTS:
            args = case(M, K, N, torch.float16, name, residual=True)
            plain = run(*args)
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                hooked = run(*args)
            for k in plain:
                assert torch.equal(plain[k], hooked[k]), (k, name)


def test_forward_mode_is_refused(host_side):
    """A tangent on any input, or on the gradient, is refused and not dropped, whether or not gradients are recorded."""
    import torch.autograd.forward_ad as forward_ad
    from box_convolution import linear_act
    plain = [torch.randn(s, device="cuda") for s in ((5, 8), (6, 8), (6,), (5, 6))]
    with forward_ad.dual_level():
        for i in range(4):
            args = [forward_ad.make_dual(t, torch.ones_like(t)) if i == k else t for k, t in enumerate(plain)]
            for recorded in (False, True):
                with torch.set_grad_enabled(recorded), pytest.raises(RuntimeError, match="forward-mode"):
                    linear_act(*args, "silu")
        leaf = plain[0].clone().requires_grad_(True)
        y = linear_act(leaf, *plain[1:], "silu")
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
        assert torch.equal(linear_act(*plain, "silu"), y)


@pytest.mark.parametrize("dtype", TYPES)
def test_infinity_in_a_broadcast_row(hip, dtype):
    """Rows that lie on top of each other: beyond the last one the weight's gradient takes none of their values (0 times infinity is NaN)."""
    gen = torch.Generator().manual_seed(1)
    row, w, g = make((1, 64), gen, dtype), make((72, 64), gen, dtype), make((301, 72), gen, dtype).abs() + 1
    row[0, 3] = float("inf")
    w.requires_grad_(True)
    from box_convolution import linear_act
    wd = w.detach().cuda().requires_grad_(True)
    for x in (row.cuda().expand(301, 64), row.cuda().repeat(301, 1)):
        dw = torch.autograd.grad(linear_act(x, wd), wd, g.cuda())[0]
        assert not dw.isnan().any() and bool((dw[:, 3] == float("inf")).all()) and int(dw.isinf().sum()) == 72


@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_small_values_keep_their_digits(hip, name):
    """float32 values and derivatives far below zero against 64 bits, relatively: the exponential's argument a is a product rounded twice
    (3 * 2^-24 |a| with its constant), everything else a dozen roundings, and gelu's fit of the error function 2e-7."""
    lowest = {"silu": -80.0, "gelu": -12.0}[name]
    z = torch.linspace(lowest, -2.0, 4001, dtype=torch.float64).float().reshape(-1, 1)
    out = run(z, torch.ones(1, 1), None, torch.zeros_like(z), name, torch.ones_like(z))
    zd = z.double()
    a = zd.abs() if name == "silu" else 0.5 * zd.square()
    allowed = 3 * 2.0 ** -24 * a + 12 * 2.0 ** -23 + 2e-7
    for got, want, extra in ((out["y"], ref.act(zd, name), 1), (out["residual"], ref.slope(zd, name), 4)):
        off = ((got.double().cpu() - want) / want).abs() / (extra * allowed)
        assert off.max() <= 1, (off.max().item(), z[off.argmax()].item())


def _tail_values(name, dtype):
    """z from where the derivative of silu or gelu is some 1e-10 to where it is 1."""
    lowest = {"silu": -27.0, "gelu": -7.0}[name]
    z = torch.linspace(lowest, 8.0, 4001, dtype=torch.float64).to(dtype)
    return z.reshape(-1, 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_small_slopes_keep_their_digits(hip, name, dtype):
    """dz = act'(z) for a gradient of 1 and z = x: the kept 16-bit act' is off by at most 2^-16, and below 2^-5 by 2^-13.9 |act'|^(3/4) (a code of
    its fourth root in steps of 1/13100: 4 * 0.5 / 13100 * 2^(-5/4) |act'|^(3/4)), the float32 derivative by 4e-7 near its zero and, in
    the tail, by the exponential's argument's rounding, and the result is rounded once."""
    z = _tail_values(name, dtype)
    ones = torch.ones(z.size(0), 1, dtype=dtype)
    got = run(z, torch.ones(1, 1, dtype=dtype), None, torch.zeros_like(ones), name, ones)["residual"].double().cpu()
    d = ref.slope(z.double(), name)
    error = torch.where(d.abs() < 2.0 ** -5, 2.0 ** -13.9 * d.abs() ** 0.75, 2.0 ** -16) + 1e-6 * d.abs() * (1 + z.double().square()) + 4e-7 * (z.double().abs() < 3)
    assert bool(((got - d).abs() <= ref.rounded(d, error, dtype)).all())
    # and what that is: two roundings of float16 (little more than one of bfloat16) at most, wherever |act'| is at least 2^-12
    tail = (d.abs() >= 2.0 ** -12) & (z.double().abs() > 2)
    assert bool(((got - d).abs()[tail] <= 2.1 * ref.UNIT[dtype] * d.abs()[tail]).all())
    assert name == "silu" or bool((got[z.double() == 8] == 1).all())


def test_more_tiles_than_a_grid_takes(hip):
    """Rows in so many tiles that their workgroups have 2^32 threads together: the rows around the place where the second launch starts, the
    first and the last are those of the same rows alone."""
    from box_convolution import linear_act
    rows, base = (1 << 30) + 777, 1 << 20
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(base, 8, generator=gen, device="cuda", dtype=torch.bfloat16).repeat(rows // base + 1, 1)[:rows].requires_grad_(True)
    w = torch.randn(1, 8, generator=gen, device="cuda", dtype=torch.bfloat16)
    y = linear_act(x, w, activation="silu")
    g = torch.randn(base, 1, generator=gen, device="cuda", dtype=torch.bfloat16).repeat(rows // base + 1, 1)[:rows]
    dx = torch.autograd.grad(y, x, g)[0]
    for at in (0, (1 << 30) - 64 - 500, (1 << 30) - 500, rows - 1000):
        part = slice(at, at + 1000)
        xs = x.detach()[part].requires_grad_(True)
        ys = linear_act(xs, w, activation="silu")
        assert torch.equal(ys, y[part]) and torch.equal(torch.autograd.grad(ys, xs, g[part])[0], dx[part]), at


def test_nothing_to_sum_at_the_c_entry(hip):
    """Without rows the parameters' gradients are sums of nothing, without output features the input's: 0, written by the call."""
    lib, stream = hip.load(), torch.cuda.current_stream().cuda_stream
    for dtype, code in zip(TYPES, (0, 1, 2)):
        dx, dw, db = (torch.full(s, float("nan"), device="cuda", dtype=dtype) for s in ((5, 8), (6, 8), (6,)))
        assert lib.boxconv_linear_backward(None, 8, None, None, None, None, dw.data_ptr(), db.data_ptr(), None, code, 0, 8, 6, 0, None, 0, stream) == 0
        assert lib.boxconv_linear_backward(None, 8, None, None, None, dx.data_ptr(), None, None, None, code, 5, 8, 0, 0, None, 0, stream) == 0
        assert not dw.any() and not db.any() and not dx.any()
