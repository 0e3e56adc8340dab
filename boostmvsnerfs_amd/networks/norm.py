"""Group normalisation in the networks' convolution blocks, in the place of batch normalisation.

A fine-tune step sees one target view: batch statistics are then one image's own, differ between training and inference (the
running averages), and have to be exchanged between ranks (nn.SyncBatchNorm, which the reference's trainer converts to under
DDP: lib/train/trainers/trainer.py:15-22).  A group's statistics belong to one sample: training, inference and any number of
ranks compute the same thing.  `convert_group_norm` is to that what nn.SyncBatchNorm.convert_sync_batchnorm is to exchanged
batch statistics.  The normalisation and the activation behind it are one operator (autograd.GroupNormAct,
csrc/group_norm.hip).  Statistics that depend on the input cannot be folded into convolution weights: a converted network
runs its convolution blocks module by module at inference too (same convolution engine, no fused frame).
"""
import torch.nn as nn

from .. import autograd as A


class GroupNorm(nn.Module):
    """act(group_norm(x)); `weight`, `bias` as nn.GroupNorm has them.  `relu`: the activation behind it (False, True, a leaky
    slope, "silu"), which a call may override."""

    def __init__(self, groups, weight, bias, eps=1e-5, relu=False):
        super().__init__()
        self.groups, self.eps, self.relu = int(groups), float(eps), relu
        self.weight, self.bias = weight, bias

    def forward(self, x, relu=None):
        return A.GroupNormAct.apply(x, self.groups, self.weight, self.bias, self.eps, self.relu if relu is None else relu)

    def extra_repr(self):
        return f"groups={self.groups}, channels={self.weight.numel()}, eps={self.eps}, relu={self.relu}"


def convert_group_norm(net, group_size=8, eps=1e-5):
    """Every batch norm of `net` -- a whole Network of this package -- becomes a group norm over `group_size` channels, in
    place; its weight and bias stay the parameters they are (same state-dict keys; the running statistics are dropped).
    Returns `net`."""
    from .enerf import cnn as enerf_cnn
    from .enerf.conv_train import Conv2d, Conv3d, ConvTranspose3d
    from .mvsnerf import network as mvsnerf
    engines = (enerf_cnn.FeatureNet, enerf_cnn._CostReg, mvsnerf.FeatureNet, mvsnerf.CostRegNet)
    if isinstance(net, engines) or not any(isinstance(m, engines) for m in net.modules()):
        raise TypeError(f"convert_group_norm: expected a whole Network, got {type(net).__name__}")
    norms = [(parent, name, m) for parent in net.modules() for name, m in parent.named_children()
             if isinstance(m, (nn.modules.batchnorm._BatchNorm, mvsnerf.ABN))]
    for _, name, m in norms:
        if m.weight is None or m.weight.numel() % group_size:
            raise ValueError(f"convert_group_norm: {name} has {0 if m.weight is None else m.weight.numel()} channels, "
                             f"groups of {group_size} do not divide them")
    for parent, name, m in norms:
        # (ABN carries its activation; ConvBnReLU's is handed over by the block)
        setattr(parent, name, GroupNorm(m.weight.numel() // group_size, m.weight, m.bias, eps,
                                        float(m.slope) if isinstance(m, mvsnerf.ABN) else False))
    for m in net.modules():
        if isinstance(m, engines):
            m.group_norm = True           # nothing to fold: see _engine_ok
        elif isinstance(m, (Conv2d, Conv3d, ConvTranspose3d)):
            m.engine_always = True        # ... so the single convolutions take the engine without autograd as well
    net._apply(lambda t: t)               # packed weights and captured frames of the old modules are stale
    return net
