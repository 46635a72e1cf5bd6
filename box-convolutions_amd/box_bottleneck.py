"""A bottleneck block around a box convolution, with everything but the box convolution itself in two fused operators, and a
small training run of it on synthetic data:

    python box-convolutions_amd/box_bottleneck.py [--steps 20] [--dtype float32|bfloat16|float16]

The block follows the reference's BottleneckBoxConv (examples/Cityscapes/models/ENet.py:282-304): 1 x 1 convolution to a
quarter of the channels, norm, activation, box convolution back to all of them, norm, residual add, activation. Group norm stands
in for its batch norm: segmentation trains with one to a few images per GPU, too few for statistics over a batch.

Layouts: the pointwise product and group norm work on channels-last memory (a pixel's channels side by side), the box
convolution on planes; each change of layout is one copy.
"""
import argparse

import torch

from box_convolution import BoxConv2d, GroupNormAct, PointwiseConv2d


class BoxBottleneck(torch.nn.Module):
    """``[B, channels, h, w]`` -> the same shape. ``channels`` = ``num_filters`` times the squeezed channels."""

    def __init__(self, channels, num_filters, max_input_h, max_input_w, groups=8, activation="relu"):
        super().__init__()
        if channels % num_filters != 0:
            raise ValueError("channels must be a multiple of num_filters")
        squeezed = channels // num_filters
        self.squeeze = PointwiseConv2d(channels, squeezed, bias=False)
        self.norm_in = GroupNormAct(min(groups, squeezed), squeezed, activation=activation)
        self.boxes = BoxConv2d(squeezed, num_filters, max_input_h, max_input_w)
        self.norm_out = GroupNormAct(groups, channels, activation=activation)

    def forward(self, x):
        return self.norm_out(self.boxes(self.norm_in(self.squeeze(x))), residual=x)


class BoxSegmenter(torch.nn.Module):
    """Two blocks between a pointwise stem and a pointwise classifier: enough to train something end to end."""

    def __init__(self, in_channels, classes, channels=32, num_filters=4, h=64, w=128):
        super().__init__()
        self.stem = PointwiseConv2d(in_channels, channels, activation="relu")
        self.blocks = torch.nn.Sequential(*(BoxBottleneck(channels, num_filters, h, w) for _ in range(2)))
        self.classify = PointwiseConv2d(channels, classes)

    def forward(self, x):
        return self.classify(self.blocks(self.stem(x)))


def synthetic_batch(batch, h, w, gen, device):
    """Images with two channels of noise and one bright rectangle each; the label is whether a pixel is inside one."""
    image = torch.randn(batch, 3, h, w, generator=gen) * 0.5
    label = torch.zeros(batch, h, w, dtype=torch.long)
    for b in range(batch):
        i, j = (int(torch.randint(0, n // 2, (1,), generator=gen)) for n in (h, w))
        label[b, i:i + h // 3, j:j + w // 3] = 1
    image[:, 2] += label
    return image.to(device), label.to(device)


def train(steps=20, batch=4, h=64, w=128, dtype=torch.float32, device="cuda", seed=0):
    """Losses of `steps` training steps. Half precision trains with that type's parameters in the pointwise products and float32
    ones everywhere else."""
    torch.manual_seed(seed)
    gen = torch.Generator().manual_seed(seed)
    net = BoxSegmenter(3, 2, h=h, w=w).to(device)
    for module in net.modules():
        if isinstance(module, PointwiseConv2d):
            module.to(dtype)
    optimizer = torch.optim.SGD(net.parameters(), lr=0.05, momentum=0.9)
    losses = []
    for _ in range(steps):
        image, label = synthetic_batch(batch, h, w, gen, device)
        logits = net(image.to(dtype).contiguous(memory_format=torch.channels_last))
        loss = torch.nn.functional.cross_entropy(logits.float(), label)
        optimizer.zero_grad(set_to_none=True)
        loss.backward()
        optimizer.step()
        losses.append(float(loss.detach()))
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--dtype", default="float32", choices=("float32", "bfloat16", "float16"))
    args = ap.parse_args()
    for step, loss in enumerate(train(args.steps, dtype=getattr(torch, args.dtype))):
        print("step %3d  loss %.4f" % (step, loss))
