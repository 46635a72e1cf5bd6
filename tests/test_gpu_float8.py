"""``quantize_blocks``, ``linear_act_float8`` and what hands its rows to them, against the 8-bit format and the product in 64 bits
(tests/block_reference.py), at sizes and values where blocks, tiles and the format end."""
import random

import pytest
import torch

import block_reference as ref
from operator_reference import check

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
ACTS = [None, "relu", "silu", "gelu"]


def rows(gen, M, K, dtype=torch.float32, scale=1.0):
    """Rows with channels of very different size."""
    return (torch.randn(M, K, generator=gen, dtype=torch.float64) * torch.exp(torch.randn(K, generator=gen, dtype=torch.float64)) * scale).to(dtype)


def same_blocks(blocks, x):
    """Codes and exponents equal the reference's, padding among them."""
    units, words = ref.quantize(x.double().reshape(-1, x.size(-1)))
    got = blocks.codes.float().cpu().double().reshape(units.shape)
    assert torch.equal(blocks.exponents.cpu().reshape(words.shape), words)
    assert torch.equal(got.isnan(), units.isnan()) and torch.equal(got.nan_to_num(0.0), units.nan_to_num(0.0))


# ---- quantize_blocks ----------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (3, 7), (2, 127), (2, 128), (5, 129), (1, 4096), (33, 333), (257, 512), (64, 640), (1000, 136), (7, 5000), (2, 32769)])
def test_quantize_sizes(hip, M, K, dtype):
    from box_convolution import quantize_blocks
    x = rows(torch.Generator().manual_seed(M + K), M, K, dtype)
    same_blocks(quantize_blocks(x.cuda()), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_every_value_of_the_format_and_every_tie(hip, dtype):
    """Blocks whose power is 1 (their largest value is 448): all code values, the midpoints between them and the values next to those."""
    from box_convolution import quantize_blocks
    v = ref.CODE_VALUES
    ties = (v[1:] + v[:-1]) / 2
    values = torch.cat([v, ties, ties * (1 + 2.0 ** -7), ties * (1 - 2.0 ** -7)])
    values = torch.cat([values, -values])
    values = values[(values.abs() <= 448)]
    full = torch.full((-(-values.numel() // 127), 128), 448.0, dtype=torch.float64)
    full[:, 1:].reshape(-1)
    flat = torch.zeros(full.size(0) * 127, dtype=torch.float64)
    flat[:values.numel()] = values
    full[:, 1:] = flat.view(-1, 127)
    x = full.to(dtype)
    blocks = quantize_blocks(x.cuda())
    same_blocks(blocks, x)
    assert (blocks.exponents[:, 0] == 127).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_powers(hip, dtype):
    """Largest values on both sides of 448 times a power of two, over the type's whole range; subnormal and zero blocks."""
    from box_convolution import quantize_blocks
    info = torch.finfo(dtype)
    most = []
    for e in range(-140, 120):
        for m in (448.0, 448.0 * (1 + info.eps), 448.0 * (1 - info.eps), 256.0):
            if float(torch.tensor(m * 2.0 ** e, dtype=torch.float64).to(dtype)) not in (0.0, float("inf")):
                most.append(m * 2.0 ** e)
    x = torch.zeros(len(most) + 1, 128, dtype=torch.float64)
    x[:-1, 5] = torch.tensor(most, dtype=torch.float64)
    x[:-1, 9] = -x[:-1, 5] * 0.3
    x = x.to(dtype)
    same_blocks(quantize_blocks(x.cuda()), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_nan_and_infinity(hip, dtype):
    from box_convolution import quantize_blocks
    x = rows(torch.Generator().manual_seed(0), 6, 300, dtype)
    x[0, 3], x[1, 130], x[2, 299], x[3] = float("nan"), float("inf"), float("-inf"), float("nan")
    same_blocks(quantize_blocks(x.cuda()), x)


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_layouts(hip, dtype):
    """Rows apart, at any element, inside a buffer of NaN; leading dimensions; transposed; no rows."""
    from box_convolution import quantize_blocks
    x = rows(torch.Generator().manual_seed(1), 12, 200, dtype)
    for shift in (0, 1, 3):
        big = torch.full((14, 211), float("nan"), dtype=dtype, device="cuda")
        view = big[1:13, shift:shift + 200]
        view.copy_(x)
        same_blocks(quantize_blocks(view), x)
    same_blocks(quantize_blocks(x.cuda().t().contiguous().t()), x)
    blocks = quantize_blocks(x.cuda().view(3, 4, 200))
    assert blocks.shape == (3, 4, 200) and blocks.codes.shape == (3, 4, 256) and blocks.exponents.shape == (3, 4, 4)
    assert (blocks.dequantize(torch.float64).cpu().view(12, 200) == ref.dequantize(x.double())).all()
    assert quantize_blocks(x.cuda()[:0]).codes.shape == (0, 256)
    assert torch.equal(quantize_blocks(x.cuda()[0]).codes.float(), blocks.codes[0, 0].float())
    expanded = x.cuda()[:1].expand(5, 200)
    same_blocks(quantize_blocks(expanded), x[:1].expand(5, 200))


# ---- the product --------------------------------------------------------------------------------

def case(M, K, N, dtype, name, bias=True, residual=False, seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * M + 11 * K + 13 * N)
    x, w = rows(gen, M, K, dtype), rows(gen, N, K, torch.float32, K ** -0.5)
    b = torch.randn(N, generator=gen).to(dtype) if bias else None
    r = torch.randn(M, N, generator=gen).to(dtype) if residual else None
    return x, w, b, r, name


def run(x, w, b, r, name, coded, like=None):
    from box_convolution import linear_act_float8, quantize_blocks
    like = like or (lambda t: None if t is None else t.cuda())
    given = quantize_blocks(x.cuda()) if coded else like(x)
    return {"y": linear_act_float8(given, quantize_blocks(w.cuda()), like(b), residual=like(r), activation=name, dtype=x.dtype)}


def expected(x, w, b, r, name):
    wide = [None if t is None else t.double() for t in (b, r)]
    return ref.product(ref.dequantize(x.double()), ref.dequantize(w.double()), *wide, name, x.dtype)


SIZES = [(1, 1, 1), (1, 128, 64), (2, 8, 200), (3, 130, 7), (15, 256, 33), (16, 1000, 24), (17, 512, 96), (31, 129, 130), (32, 384, 64), (33, 640, 96), (63, 65, 64),
         (65, 63, 66), (64, 256, 64), (128, 128, 128), (129, 130, 257), (200, 512, 128), (257, 1152, 260), (1000, 40, 8), (1, 333, 517), (16, 2048, 256), (5, 4096, 100),
         (300, 8, 16), (4099, 33, 129), (5000, 128, 32), (700, 520, 264), (33, 24, 1030), (100, 4224, 72), (32, 1024, 1024)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_sizes(hip, i, dtype):
    M, K, N = SIZES[i]
    args = case(M, K, N, dtype, ACTS[(i + TYPES.index(dtype)) % 4], bias=i % 3 != 2, residual=i % 2 == 1)
    for coded in (False, True):
        check(run(*args, coded), expected(*args))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("bias,residual", [(False, False), (True, True)])
def test_epilogues(hip, name, bias, residual, dtype):
    for M, K, N in ((130, 72, 136), (7, 272, 136), (24, 300, 50), (900, 640, 48)):
        args = case(M, K, N, dtype, name, bias, residual, seed=5)
        check(run(*args, M % 2 == 0), expected(*args))


@pytest.mark.parametrize("dtype", TYPES)
def test_large_products(hip, dtype):
    """Tiles of every size, whole ones and a rest on every side, and long sums."""
    for M, K, N in ((640, 512, 768), (1030, 584, 1096), (264, 8200, 256), (2048, 256, 2100), (48, 16500, 40)):
        args = case(M, K, N, dtype, "silu", residual=True)
        for coded in (False, True):
            check(run(*args, coded), expected(*args))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(65536, 128, 32), (65600, 100, 40), (70001, 256, 33), (65543, 8, 5), (66000, 300, 72), (65536, 512, 24), (65537, 130, 8)])
def test_many_rows_through_few_channels(hip, M, K, N, dtype):
    args = case(M, K, N, dtype, ACTS[(M + K) % 4], residual=K % 3 == 0)
    want = expected(*args)
    for coded in (False, True):
        check(run(*args, coded), want)
    x, w = args[:2]
    x[M - 1, 3], x[5, K - 1], w[N - 1, 0] = float("nan"), float("inf"), float("nan")
    bad = run(x, w, None, None, None, False)["y"].isnan().cpu()
    rows_, columns = bad.all(1).nonzero().flatten().tolist(), bad.all(0).nonzero().flatten().tolist()
    assert rows_ == [5, M - 1] and columns == [N - 1] and int(bad.sum()) == 2 * N + M - 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 256, 40), (20, 200, 72), (70, 40, 72), (520, 256, 512)])
def test_powers_of_all_sizes(hip, M, K, N, dtype):
    """Blocks whose powers differ by many orders within a row: each is multiplied by its own."""
    x, w, b, _, _ = case(M, K, N, dtype, None)
    gen = torch.Generator().manual_seed(1)
    for t in (x, w):
        for k in range(0, K, 128):
            t[:, k:k + 128] *= torch.pow(2.0, torch.randint(-6, 6, (t.size(0), 1), generator=gen).float()).to(t.dtype)
    for coded in (False, True):
        check(run(x, w, b, None, None, coded), expected(x, w, b, None, None))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 40, 72), (5, 136, 264), (32, 300, 40), (70, 40, 72), (520, 256, 512)])
def test_rows_apart_and_any_address(hip, M, K, N, dtype):
    """Inputs, bias and residual inside larger tensors that hold NaN around them, at addresses of one element."""
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
        check(run(*args, False, like=inside), expected(*args))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(4, 512, 96), (24, 130, 40), (40, 40, 40), (2000, 64, 32), (600, 264, 520)])
def test_nan_and_infinity_stay_in_their_row_and_column(hip, M, K, N, dtype):
    """Where the values have a NaN or an infinity, the row (or column of the result) is NaN, nothing else."""
    x, w, b, _, _ = case(M, K, N, dtype, None)
    x[1, 3], x[2, 0], w[5, 1] = float("nan"), float("inf"), float("-inf")
    for coded in (False, True):
        bad = run(x, w, b, None, None, coded)["y"].isnan().cpu()
        want = torch.zeros(M, N, dtype=torch.bool)
        want[1], want[2], want[:, 5] = True, True, True
        assert torch.equal(bad, want)


def test_every_row_count_up_to_a_tile(hip):
    """The rules that choose a kernel by the number of rows all give the same product, to float32's roundings."""
    from box_convolution import linear_act_float8, quantize_blocks
    x, w, _, _, _ = case(70, 520, 48, torch.float32, None)
    w8, whole = quantize_blocks(w.cuda()), ref.product(ref.dequantize(x.double()), ref.dequantize(w.double()), None, None, None, torch.float32)["y"]
    for M in list(range(1, 36)) + [48, 64, 65, 70]:
        y = linear_act_float8(x.cuda()[:M], w8).double().cpu()
        assert bool(((y - whole[0][:M]).abs() <= whole[1][:M]).all()), M


def test_shapes_and_empty(hip):
    from box_convolution import linear_act_float8, quantize_blocks
    x, w, _, _, _ = case(24, 40, 16, torch.bfloat16, None)
    w8 = quantize_blocks(w.cuda())
    plain = linear_act_float8(x.cuda(), w8)
    assert torch.equal(linear_act_float8(x.cuda().view(2, 3, 4, 40), w8), plain.view(2, 3, 4, 16))
    assert linear_act_float8(x.cuda()[:0], w8).shape == (0, 16)
    assert linear_act_float8(x.cuda(), quantize_blocks(w.cuda()[:0])).shape == (24, 0)
    assert linear_act_float8(quantize_blocks(x.cuda()), w8).dtype == torch.bfloat16
    got = linear_act_float8(quantize_blocks(x.cuda()), w8, dtype=torch.float32)
    assert got.dtype == torch.float32 and (got - plain.float()).abs().max() <= 2.0 ** -7 * got.abs().max()
    one = linear_act_float8(x.cuda()[0], w8)
    assert one.shape == (16,) and (one.float() - plain[0].float()).abs().max() <= 2.0 ** -7 * plain.abs().max()


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
    from box_convolution import linear_act_float8, quantize_blocks, residual_norm
    for M, K, N in ((5, 40, 24), (40, 200, 24)):
        args = case(M, K, N, dtype, "gelu", residual=True)
        for coded in (False, True):
            check(run(*args, coded), expected(*args))
        x, w8 = args[0].cuda(), quantize_blocks(args[1].cuda())
        same_blocks(quantize_blocks(x.view(1, M, K)), args[0])
        plain = linear_act_float8(x, w8)
        assert torch.equal(linear_act_float8(x.view(1, M, 1, K), w8), plain.view(1, M, 1, N)) and linear_act_float8(x[:0], w8).shape == (0, N)
        w = torch.ones(K, device="cuda")
        stream, blocks = residual_norm(x.view(1, M, K).movedim(-1, 1), before=(w, None), quantize=True)
        assert blocks.shape == (1, M, K) and stream.shape == (1, K, M)
        assert torch.equal(linear_act_float8(blocks, w8, dtype=dtype)[0], linear_act_float8(quantize_blocks(blocks.dequantize()[0]), w8, dtype=dtype))


def test_module_after_a_change_of_type(hip):
    """Codes stay codes when a module's floating-point buffers are converted."""
    from box_convolution import PointwiseConv2dFloat8
    torch.manual_seed(0)
    module = PointwiseConv2dFloat8(torch.nn.Conv2d(40, 24, 1).cuda(), activation="relu")
    x = torch.randn(2, 40, 3, 5, device="cuda")
    want = module(x)
    half = PointwiseConv2dFloat8(torch.nn.Conv2d(40, 24, 1).cuda())
    half.load_state_dict(module.state_dict())
    half.activation = "relu"
    half = half.to(torch.float16)
    got = half(x.half())
    assert got.dtype == torch.float16 and torch.equal(half.codes, module.codes)
    # another rounding of the input moves a code by at most a step, 2^-3 of its value, here in a few places
    assert (got.float() - want).norm() <= 2.0 ** -5 * want.norm()


def test_refusals(host_side):
    from box_convolution import Float8Blocks, PointwiseConv2dFloat8, linear_act_float8, quantize_blocks
    x, w = torch.randn(4, 40, device="cuda"), torch.randn(8, 40, device="cuda")
    w8, x8 = quantize_blocks(w), quantize_blocks(x)
    bias = torch.zeros(8, device="cuda")
    codes = torch.zeros(8 * 128 + 1, device="cuda", dtype=torch.uint8)
    for bad, match in ((lambda: quantize_blocks(x.cpu()), "AMD GPUs only"), (lambda: quantize_blocks(x.double()), "float32, float16 or bfloat16"),
                       (lambda: quantize_blocks(x[:, :0]), "at least one column"), (lambda: quantize_blocks(x[0, 0]), "at least one column"),
                       (lambda: quantize_blocks(x.clone().requires_grad_(True)), "no gradient"),
                       (lambda: linear_act_float8(x, w), "Float8Blocks"), (lambda: linear_act_float8(x.cpu(), w8), "AMD GPUs only"),
                       (lambda: linear_act_float8(x[:, :39], w8), r"\[N, K\]"), (lambda: linear_act_float8(x, w8, dtype=torch.float16), "result's type"),
                       (lambda: linear_act_float8(x8, w8, dtype=torch.float64), "result's type"), (lambda: linear_act_float8(x.double(), w8), "float32, float16"),
                       (lambda: linear_act_float8(x, w8, bias.half()), "bias"), (lambda: linear_act_float8(x, w8, bias[:7]), "bias"),
                       (lambda: linear_act_float8(x, w8, residual=x), "residual"), (lambda: linear_act_float8(x, w8, activation="tanh"), "activation"),
                       (lambda: linear_act_float8(x.clone().requires_grad_(True), w8), "no gradient"),
                       (lambda: linear_act_float8(x8, w8, bias.clone().requires_grad_(True), dtype=torch.float32), "no gradient"),
                       (lambda: Float8Blocks(w8.codes, w8.exponents, 129), "256"), (lambda: Float8Blocks(w8.codes.view(torch.uint8), w8.exponents, 40), "float8_e4m3fn"),
                       (lambda: Float8Blocks(w8.codes, w8.exponents.cpu(), 40), "one device"), (lambda: Float8Blocks(w8.codes, w8.exponents[:7], 40), "exponents"),
                       (lambda: Float8Blocks(codes[1:].view(torch.float8_e4m3fn).view(8, 128), w8.exponents, 40), "addresses"),
                       (lambda: Float8Blocks(w8.codes.t().contiguous().t(), w8.exponents, 40), "contiguous"),
                       (lambda: PointwiseConv2dFloat8(torch.nn.Conv2d(8, 8, 3).cuda()), "1 x 1"), (lambda: PointwiseConv2dFloat8(torch.nn.Conv2d(8, 8, 1, 2).cuda()), "1 x 1")):
        with pytest.raises(RuntimeError, match=match):
            bad()
    with torch.no_grad():
        assert torch.equal(linear_act_float8(x.clone().requires_grad_(True), w8), linear_act_float8(x, w8))


@pytest.mark.parametrize("M", [1, 24, 300, 66000])
def test_another_stream_and_graph_replays(hip, M):
    from box_convolution import linear_act_float8, quantize_blocks
    K = 1030 if M < 65536 else 128
    x, w, b, r, _ = (t.cuda() if torch.is_tensor(t) else t for t in case(M, K, 72, torch.bfloat16, "silu", residual=True))
    w8 = quantize_blocks(w)

    def step():
        return linear_act_float8(x, w8, b, r, "silu"), quantize_blocks(x).codes
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    assert torch.equal(first[0], second[0]) and torch.equal(first[1].view(torch.uint8), second[1].view(torch.uint8))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        x.copy_(x.roll(k + 1, 1))
        graph.replay()
        torch.cuda.synchronize()
        got = captured[0].clone()
        assert torch.equal(got, step()[0])


def test_codes_beyond_2_31(hip):
    """Rows of codes past 2^31 bytes, and rows of the result past 2^31 elements."""
    from box_convolution import linear_act_float8, quantize_blocks
    gen = torch.Generator(device="cuda").manual_seed(0)
    M, K, N = (1 << 24) + 70, 129, 136
    x = torch.randn(1 << 16, K, generator=gen, device="cuda", dtype=torch.bfloat16)
    w8 = quantize_blocks(torch.randn(N, K, generator=gen, device="cuda"))
    some = quantize_blocks(x)
    many = quantize_blocks(x.repeat(257, 1)[:M])
    assert many.codes.numel() > 1 << 31
    y, want = linear_act_float8(many, w8), linear_act_float8(some, w8)
    assert y.numel() > 1 << 31
    for k in (0, 255):
        part = slice(k << 16, (k + 1) << 16)
        assert torch.equal(many.codes[part].view(torch.uint8), some.codes.view(torch.uint8)) and torch.equal(y[part], want)
    assert torch.equal(y[256 << 16:], want[:70])
    del many, y, some, want
    # the same through tiles: rows of 640 codes
    M, K, N = (1 << 22) + 70, 600, 72
    x = torch.randn(1 << 16, K, generator=gen, device="cuda", dtype=torch.bfloat16)
    w8 = quantize_blocks(torch.randn(N, K, generator=gen, device="cuda"))
    r = torch.randn(1 << 16, N, generator=gen, device="cuda", dtype=torch.bfloat16)
    many = quantize_blocks(x.repeat(65, 1)[:M])
    assert many.codes.numel() > 1 << 31
    y, want = linear_act_float8(many, w8, residual=r.repeat(65, 1)[:M]), linear_act_float8(quantize_blocks(x), w8, residual=r)
    for k in (0, 63):
        assert torch.equal(y[k << 16:(k + 1) << 16], want)
    assert torch.equal(y[64 << 16:], want[:70])


# ---- together -----------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("C,rows_", [(8, 3), (52, 40), (64, 33), (128, 70), (136, 9), (512, 17), (1000, 5), (1024, 5), (1100, 3), (4096, 2), (4104, 2), (6001, 3), (8192, 2), (9000, 2), (17000, 2)])
def test_norm_writes_blocks(hip, C, rows_, kind, dtype):
    """The normed rows in 8 bits stand within their format's rounding of the formula, and are exactly the blocks of some float32 rows within the norm's
    own bound: every code is the rounding of the value or of a neighbour within the bound."""
    from box_convolution import residual_norm
    gen = torch.Generator().manual_seed(C)
    x, r = (torch.randn(rows_, C, generator=gen).to(dtype) for _ in range(2))
    w, b, g = torch.rand(C, generator=gen) + 0.5, torch.randn(C, generator=gen) if kind == "layer" else None, torch.randn(C, generator=gen)
    dev = [None if t is None else t.cuda() for t in (x, r, g, w, b)]
    stream, blocks = residual_norm(dev[0], dev[1], dev[2], 0.5, (dev[3], dev[4]), (dev[3], dev[4]), kind, quantize=True)
    plain, normed = residual_norm(dev[0], dev[1], dev[2], 0.5, (dev[3], dev[4]), (dev[3], dev[4]), kind)
    assert torch.equal(stream, plain) and blocks.shape == (rows_, C)
    wide = [None if t is None else t.double() for t in (w, b)]
    value, bound = ref.residual_norm(x.double()[:, None], r.double()[:, None], g.double(), 0.5, wide, wide, kind, 1e-6, None, None, torch.float32,
                                     torch.float32, torch.float32)["normed"]
    value, bound = value[:, 0], bound[:, 0]
    got = blocks.dequantize(torch.float64).cpu()
    power = ref.two_to(blocks.exponents.cpu().to(torch.int64) - 127).repeat_interleave(128, 1)[:, :C]
    assert bool(((got - value).abs() <= bound + 2.0 ** -4 * (value.abs() + bound) + 2.0 ** -10 * power).all())
    # the powers: least for the largest magnitude, give or take the bound
    blocks_of = blocks.codes.size(-1) // 128
    pad = torch.zeros(rows_, blocks_of * 128, dtype=torch.float64)
    pad[:, :C] = value.abs()
    most = pad.view(rows_, blocks_of, 128).amax(-1)
    slack = bound.max()
    p = ref.two_to(blocks.exponents[:, :blocks_of].cpu().to(torch.int64) - 127)
    assert bool((most - slack <= 448 * p).all()) and bool((most + slack > 224 * p).all())
    assert not blocks.codes.float()[:, C:].any() and bool((blocks.exponents[:, blocks_of:] == 127).all())
    if dtype == torch.float32:                                       # the same float32 rows, quantized afterwards
        same_blocks(blocks, normed.cpu())


def test_a_block_for_inference(hip):
    """As a network uses them: the boundary behind one block quantizes what the next block's two products read, against the same in
    64 bits. Tolerance: the first product's own bound, widened by what a neighbouring code in its input may change (2^-4 of a value in one place per
    thousand: below 2^-6 of the row's size together), and by bfloat16's rounding of the hidden rows."""
    from box_convolution import PointwiseConv2d, PointwiseConv2dFloat8, ResidualNorm
    torch.manual_seed(0)
    norm = ResidualNorm(64, kind="layer", scale=0.5).cuda()
    up, down = PointwiseConv2d(64, 160, activation="gelu").cuda().bfloat16(), PointwiseConv2d(160, 64).cuda().bfloat16()
    up8, down8 = PointwiseConv2dFloat8(up), PointwiseConv2dFloat8(down)
    assert up8.activation == "gelu" and not list(up8.parameters()) and "160" in repr(up8)
    x, r = (torch.randn(2, 64, 9, 11, device="cuda", dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last) for _ in range(2))
    with torch.no_grad():
        stream, blocks = norm(x, r, quantize=True)
        got = down8(up8(blocks), residual=stream)
        assert got.shape == (2, 64, 9, 11) and got.is_contiguous(memory_format=torch.channels_last)
        s, h = norm(x, r)
        want = down(up(h), residual=s)
        assert torch.equal(s, stream)
        # 8 bits move every value by at most 2^-4 of itself; of sums of random signs that is a twentieth at most
        assert (got.float() - want.float()).norm() <= 0.05 * want.float().norm()
        h8 = blocks.dequantize(torch.float64).cpu().reshape(-1, 64)
        hidden = ref.product(h8, ref.dequantize(up.weight.flatten(1).double().cpu()), up.bias.double().cpu(), None, "gelu", torch.bfloat16)["y"]
        first = up8(blocks).permute(0, 2, 3, 1).reshape(-1, 160)
        check({"y": first}, {"y": hidden})
        second = ref.product(ref.dequantize(first.double().cpu()), ref.dequantize(down.weight.flatten(1).double().cpu()), down.bias.double().cpu(),
                             stream.permute(0, 2, 3, 1).reshape(-1, 64).double().cpu(), None, torch.bfloat16)
        check({"y": got.permute(0, 2, 3, 1).reshape(-1, 64)}, second)


def test_random_sizes(hip):
    rng = random.Random(7)
    for i in range(40):
        M, K, N = (int(2 ** rng.uniform(0, top)) for top in (9.5, 10.5, 9.5))
        args = case(M, K, N, rng.choice(TYPES), rng.choice(ACTS), rng.random() < 0.7, rng.random() < 0.5, seed=i)
        check(run(*args, rng.random() < 0.5), expected(*args))
