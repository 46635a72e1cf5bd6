"""How far the sums of ``linear_act_float8`` may be off: float32 results have float32's sums of exact products; for 16-bit results the matrix instructions
cut every product down (towards zero) to a multiple of 2^-13 of the largest among 8 neighbouring ones. Data of one sign, whose cuts add up, products that
cancel, and powers over their whole range."""
import pytest
import torch

import block_reference as ref
from operator_reference import TINY, U32, UNIT

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# rows through every kernel: few rows, few columns of many rows, tiles
SHAPES = [(1, 256, 40), (16, 1024, 24), (20, 200, 72), (33, 640, 96), (130, 512, 136), (600, 264, 520), (65540, 128, 8)]


def values(codes, exponents, K):
    """The float64 values of blocks, [rows, K]."""
    power = ref.two_to(exponents.to(torch.int64) - 127).repeat_interleave(128, 1)
    return codes.double()[:, :K] * power[:, :K]


def bounds(x, w, dtype):
    """(x @ w.T, how far the result may be off) of float64 values on their grids: (K + 8) roundings of float32; for 16-bit types also what each product
    may lose, all of it or 2^-13 of the largest in its group of 8; one rounding to the type."""
    K = x.size(1)
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    error = (K + 8) * U32 * size
    if dtype != torch.float32:
        pad = torch.nn.functional.pad
        a, b = (pad(t.abs(), (0, -K % 8)).view(t.size(0), -1, 8) for t in (x, w))
        for m in range(0, x.size(0), 64):                                   # [64, N, K / 8, 8] at a time
            p = a[m:m + 64, None] * b[None]
            error[m:m + 64] += torch.minimum(p, 2.0 ** -13 * p.amax(-1, keepdim=True)).sum((-1, -2))
    return z, error + UNIT[dtype] * (z.abs() + error) + TINY[dtype]


def within(y, x, w, dtype):
    z, bound = bounds(x, w, dtype)
    y, most = y.double().cpu(), torch.finfo(dtype).max
    off = (y - z).abs()
    off[y.isinf() & (y.sign() == z.sign()) & (z.abs() + bound >= most)] = 0.0          # (rounds to an infinity, or may)
    worst = (off / bound).max().item()
    assert worst <= 1.0, "%.3g times the bound" % worst


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_values_of_one_sign(hip, M, K, N, dtype):
    """Rows behind a relu through weights of one sign, with channels of very different size: nothing cancels, every cut is a loss."""
    from box_convolution import linear_act_float8, quantize_blocks
    gen = torch.Generator().manual_seed(M + K)
    rows = min(M, 300)
    x = (torch.randn(rows, K, generator=gen).clamp_min(0) * torch.exp(torch.randn(K, generator=gen))).to(dtype)
    w = torch.randn(N, K, generator=gen).abs() * K ** -0.5
    w8, repeat = quantize_blocks(w.cuda()), -(-M // rows)
    x8, xs = ref.dequantize(x.double()), x.cuda().repeat(repeat, 1)[:M]
    for given in (xs, quantize_blocks(xs)):
        y = linear_act_float8(given, w8, dtype=dtype)
        within(y[:rows], x8, ref.dequantize(w.double()), dtype)
        assert torch.equal(y[M - M % rows:], y[:M % rows])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_products_that_cancel(hip, M, K, N, dtype):
    """Two large products of opposite sign in a group of 8 and six small ones: float32 results are what the small ones add up to, exactly."""
    from box_convolution import Float8Blocks, linear_act_float8, quantize_blocks
    gen = torch.Generator().manual_seed(M + K)
    x, w = (torch.randint(-8, 9, (n, K), generator=gen).float() / 8 for n in (min(M, 300), N))
    x[:, 0::8], x[:, 7::8], w[:, 0::8], w[:, 7::8] = 256.0, 256.0, 256.0, -256.0
    if K % 8:
        x[:, K // 8 * 8:] = 0.0
    w8, xs = quantize_blocks(w.cuda()), x.repeat(-(-M // x.size(0)), 1)[:M].cuda().to(dtype)
    assert torch.equal(w8.dequantize().cpu(), w)
    given = quantize_blocks(xs)
    assert isinstance(given, Float8Blocks) and torch.equal(given.dequantize()[:x.size(0)].cpu(), x)
    y = linear_act_float8(given, w8, dtype=dtype)[:x.size(0)]
    within(y, x.double(), w.double(), dtype)
    if dtype == torch.float32:
        assert torch.equal(y.cpu().double(), x.double() @ w.double().t())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_powers_over_their_whole_range(hip, M, K, N, dtype):
    """Codes of every size under powers from 2^-126 to 2^127 on one side and their inverses on the other: the products are of moderate size, whatever
    their factors are."""
    from box_convolution import Float8Blocks, linear_act_float8
    gen = torch.Generator().manual_seed(M + K)
    rows, blocks = min(M, 300), -(-K // 128)

    def some(n, exponents):
        codes = torch.randn(n, blocks * 128, generator=gen) * 100
        codes = (codes.clamp(-448, 448) * torch.exp2(-torch.randint(0, 16, codes.shape, generator=gen).float())).to(torch.float8_e4m3fn)
        codes.view(torch.uint8)[:, K:] = 0
        words = torch.full((n, -(-blocks // 4) * 4), 127, dtype=torch.uint8)
        words[:, :blocks] = exponents.to(torch.uint8)
        return codes, words
    for low in (1, 2, 4, 12, 60, 127, 200, 242, 247, 250, 253):
        e = torch.randint(low, min(low + 3, 254), (1, blocks), generator=gen)
        x, w = some(rows, e.expand(rows, blocks)), some(N, 254 - e.expand(N, blocks))
        many = [t.view(torch.uint8).repeat(-(-M // rows), 1)[:M].cuda() for t in x]
        y = linear_act_float8(Float8Blocks(many[0].view(torch.float8_e4m3fn), many[1], K), Float8Blocks(w[0].cuda(), w[1].cuda(), K), dtype=dtype)
        within(y[:rows], values(*x, K), values(*w, K), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_largest_and_smallest_values_of_the_type(hip, M, K, N, dtype):
    """Values next to the type's ends (a mask of its lowest value among them): their blocks have the format's last exponents, the results are
    of moderate size."""
    from box_convolution import linear_act_float8, quantize_blocks
    gen = torch.Generator().manual_seed(M + K)
    rows, info = min(M, 300), torch.finfo(dtype)
    for size in (info.max, info.smallest_normal):
        x = torch.rand(rows, K, generator=gen) * 2 - 1
        x[:, ::5], x[0, 1] = torch.sign(x[:, ::5]), -1.0
        x = (x.double() * size).to(dtype)
        scale = 1.0 / max(size, 2.0 ** -100)
        w = (torch.randn(N, K, generator=gen).double() * K ** -0.5 * scale).float()
        w8, xs = quantize_blocks(w.cuda()), x.cuda().repeat(-(-M // rows), 1)[:M]
        for given in (xs, quantize_blocks(xs)):
            y = linear_act_float8(given, w8, dtype=dtype)[:rows]
            assert bool(y.isfinite().all())
            within(y, ref.dequantize(x.double()), ref.dequantize(w.double()), dtype)
