"""``residual_norm`` with a gate per batch item, at numbers of items that the workgroups do not divide: the last workgroup has fewer than the others,
and reads no gate behind the last item's (tests/test_row_plan_host.py walks the plan itself)."""
import pytest
import torch

from operator_reference import check
from test_gpu_residual_norm import TYPES, case, expected, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,C,spatial", [(1025, 24, (1,)), (1300, 20, (3,)), (4099, 8, (1,)), (1025, 40, (1,)), (257, 700, (1,)), (1023, 513, (1,)), (2049, 700, (1,)), (257, 4096, (1,)),
                                         (513, 4095, (1,)), (257, 6000, (1,)), (130, 8200, (1,)), (257, 8200, (1,))])
def test_items_that_workgroups_do_not_divide(hip, B, C, spatial, dtype):
    c = case(B, C, spatial, dtype, ("layer", "rms")[C % 2], "item", params=("same", "float")[B % 2], float_gate=C % 16 == 0)
    check(run(c), expected(c))


def test_blocks_of_items_that_workgroups_do_not_divide(hip):
    from box_convolution import quantize_blocks, residual_norm
    for B, C in ((1025, 24), (2049, 700), (513, 4096), (257, 6000)):
        torch.manual_seed(B)
        x, gate, w = torch.randn(B, C, 2, device="cuda"), torch.randn(B, C, device="cuda"), torch.rand(C, device="cuda") + 0.5
        stream, blocks = residual_norm(x, None, gate, 0.5, (w, None), (w, None), quantize=True)
        same, normed = residual_norm(x, None, gate, 0.5, (w, None), (w, None))
        want = quantize_blocks(normed.movedim(1, -1))
        assert torch.equal(stream, same) and torch.equal(blocks.exponents, want.exponents)
        assert torch.equal(blocks.codes.view(torch.uint8), want.codes.view(torch.uint8))


@pytest.mark.parametrize("side", ["C++", "Python"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,C", [(1, 40), (5, 52), (1025, 24), (257, 700), (513, 4096), (9, 8200)])
def test_float32_gate_per_item_of_rows(hip, monkeypatch, B, C, dtype, side):
    """An input [B, C] has a row per item: a float32 gate [B, C] beside 16-bit rows is a gate per item like any other, with a float32 gradient."""
    if side == "Python":
        monkeypatch.setattr(hip, "_glue", False)
    c = case(B, C, (), dtype, ("layer", "rms")[C % 3 == 0], "item", params="float", float_gate=True)
    out = run(c)
    assert out["gate"].dtype == torch.float32
    check(out, expected(c))


@pytest.mark.parametrize("B,C,pixels,gate", [(1 << 21, 8, 1, "item"), (1 << 20, 12, 2, "item"), (300007, 40, 1, "item"), (1 << 17, 520, 1, "item"), (1 << 22, 8, 1, "channel")])
def test_sums_over_many_items(hip, B, C, pixels, gate):
    """Items of a row or two, as many as a tensor of a few dozen megabytes has: the parameters' gradients are no longer chains of additions for that. The same
    gradients everywhere, so that a chain's roundings would add up; 512 additions in a row are allowed, as everywhere."""
    from box_convolution import residual_norm
    g = torch.full((B, C, pixels), 1.1, device="cuda")
    x, r = (torch.randn(B, C, pixels, device="cuda") for _ in range(2))
    gate_, w, b = torch.ones(B, C, device="cuda") if gate == "item" else torch.ones(C, device="cuda"), torch.ones(C, device="cuda"), torch.zeros(C, device="cuda")
    leaves = [t.requires_grad_(True) for t in (w, b, w.detach().clone(), b.detach().clone())]
    s, h = residual_norm(x, r, gate_, 1.0, (leaves[0], leaves[1]), (leaves[2], leaves[3]), "layer")
    got = torch.autograd.grad([s, h], leaves[1::2], [g, torch.zeros_like(h)])[0], torch.autograd.grad(residual_norm(x, r, gate_, 1.0, (w, b), (leaves[2], leaves[3]), "layer")[1],
                                                                                                        leaves[3], g)[0]
    want = g[0, 0, 0].double().item() * B * pixels
    for k, sums in enumerate(got):
        assert (sums.double() - want).abs().max().item() <= 512 * 2.0 ** -24 * want, (k, (sums.double() / want - 1).abs().max().item() * 2 ** 24)
