"""Group normalisation with an activation on channels-last tensors: the norm + ReLU of RAFT's encoders
(core/extractor_origin.py:12-55,119-170: group norm with width // 8 groups, or instance norm = one channel a group), forward
and backward, backed by libraftcorr.so (C ABI in include/raftcorr.h).

PyTorch is used for device memory, streams and autograd bookkeeping only (csrc/glue.cpp); there is no fallback path.
"""
import torch

from . import _lib

__all__ = ["group_norm", "GroupNorm"]


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, activation="none"):
    """act(group_norm(x)) of a (N, C, *spatial) CUDA tensor in float32, float16 or bfloat16; differentiable in x, weight, bias.

    num_groups divides C; num_groups == C is instance norm.  weight, bias: (C,) or None.  activation: "none", "relu", "silu".
    The result has x's type and lies channels-last (for four dimensions: torch.channels_last).  x is read in place where its
    channels are neighbours and its positions evenly spaced (channels-last tensors, their channel or batch slices); any other
    layout is copied first, and so is the gradient that comes back.  Statistics are summed in float64,
    gradients in float32, whatever x's type.  An empty x gives an empty result.

    Forward and backward passes can be captured into a HIP graph; a leaf of which an eager graph is still alive is refused there."""
    act = _lib.ACTIVATIONS.get("none" if activation is None else activation)
    if act is None:
        raise RuntimeError(f"activation must be one of {sorted(_lib.ACTIVATIONS)}, got {activation!r}")
    return _lib.glue().group_norm(x, num_groups, weight, bias, eps, act)


class GroupNorm(torch.nn.Module):
    """nn.GroupNorm with an activation behind it (same arguments and parameter names, so its checkpoints load); with
    num_groups == num_channels and affine=False it stands for nn.InstanceNorm2d.  See group_norm."""

    def __init__(self, num_groups, num_channels, eps=1e-5, affine=True, activation="none", device=None, dtype=None):
        super().__init__()
        if num_groups < 1 or num_channels % num_groups:
            raise ValueError(f"num_groups = {num_groups} does not divide {num_channels} channels")
        if activation not in _lib.ACTIVATIONS:
            raise ValueError(f"activation must be one of {sorted(_lib.ACTIVATIONS)}, got {activation!r}")
        self.num_groups, self.num_channels, self.eps, self.affine, self.activation = num_groups, num_channels, eps, affine, activation
        for name, fill in (("weight", torch.ones), ("bias", torch.zeros)):
            self.register_parameter(name, torch.nn.Parameter(fill(num_channels, device=device, dtype=dtype)) if affine else None)

    def forward(self, x):
        return group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)

    def extra_repr(self):
        return f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.affine}, activation={self.activation!r}"
