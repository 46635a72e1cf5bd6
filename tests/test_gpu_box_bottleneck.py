"""The bottleneck block of box_bottleneck.py: the pointwise product, group norm and the box convolution together, as a
network uses them."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def _double_block(block, x, boxes_out):
    """The block in float64 on the CPU, with the box convolution's own output and input gradient taken from the GPU."""
    squeeze = torch.nn.functional.conv2d(x, block.squeeze.weight.detach().double().cpu())
    norm = block.norm_in
    inner = torch.relu(torch.nn.functional.group_norm(squeeze, norm.num_groups, norm.weight.detach().double().cpu(),
                                                      norm.bias.detach().double().cpu(), norm.eps))
    norm = block.norm_out
    return inner, torch.relu(torch.nn.functional.group_norm(boxes_out, norm.num_groups, norm.weight.detach().double().cpu(),
                                                            norm.bias.detach().double().cpu(), norm.eps) + x)


@pytest.mark.parametrize("size", [(2, 32, 4, 24, 40), (1, 24, 2, 33, 47)])
def test_block_is_its_parts(hip, size):
    """Forward and the gradients on both sides of the box convolution, against the same parts in 64 bits. Tolerance: 64 float32
    roundings of the largest value (a few dozen additions and products of each pixel's channels), as everywhere in
    units of the tensor's largest magnitude."""
    from box_bottleneck import BoxBottleneck
    B, C, F, h, w = size
    random.seed(1)
    torch.manual_seed(1)
    block = BoxBottleneck(C, F, h, w, groups=4).cuda()
    with torch.no_grad():
        for p in list(block.norm_in.parameters()) + list(block.norm_out.parameters()):
            p.add_(torch.randn_like(p) * 0.2)
    x = torch.randn(B, C, h, w).cuda().contiguous(memory_format=torch.channels_last).requires_grad_(True)
    seen = {}
    block.boxes.register_forward_hook(lambda m, i, o: seen.update(inner=i[0], out=o))
    y = block(x)
    g = torch.randn(B, C, h, w).cuda()
    inner_grad, out_grad, x_grad = torch.autograd.grad(y, (seen["inner"], seen["out"], x), g)
    xd = x.detach().double().cpu().requires_grad_(True)
    out = seen["out"].detach().double().cpu().requires_grad_(True)
    inner, yd = _double_block(block, xd, out)

    def close(a, b):
        a, b = a.detach().double().cpu(), b.detach()
        assert (a - b).abs().max() <= 64 * 2.0 ** -24 * b.abs().max()
    close(seen["inner"], inner)
    close(y, yd)
    through_norm, direct = torch.autograd.grad(yd, (out, xd), g.double().cpu())
    close(out_grad, through_norm)
    close(x_grad, direct + torch.autograd.grad(inner, xd, inner_grad.double().cpu())[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_training_learns(hip, dtype):
    """Twenty steps find the bright rectangle: the last losses are below the first."""
    from box_bottleneck import train
    random.seed(0)
    losses = train(20, dtype=dtype)
    assert all(loss == loss for loss in losses)
    assert sum(losses[-5:]) < 0.7 * sum(losses[:5])
