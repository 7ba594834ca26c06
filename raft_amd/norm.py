"""Group normalisation with an activation on channels-last tensors: the norm + ReLU of RAFT's encoders
(core/extractor_origin.py:12-55,119-170: group norm with width // 8 groups, or instance norm = one channel a group), forward
and backward, backed by libraftcorr.so (C ABI in include/raftcorr.h).

PyTorch is used for device memory, streams and autograd bookkeeping only; there is no fallback path.
"""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .corr import _guard, _require_cuda, _stream

__all__ = ["group_norm", "GroupNorm"]


def _rows(t):
    """(tensor, batch stride, row stride) under which a (N, C, *spatial) tensor is N x P rows of C neighbouring values; a tensor
    of any other layout is copied to dense channels-last first."""
    C = t.shape[1]
    row, size = None, 1                                 # stride of the rows so far, positions they cover
    ok = C == 1 or t.stride(1) == 1
    for n, s in zip(reversed(t.shape[2:]), reversed(t.stride()[2:])):
        if n == 1:
            continue
        if row is None:
            row = s
            ok = ok and s >= C
        ok = ok and s == row * size
        size *= n
    if not ok:
        t = t.movedim(1, -1).contiguous().movedim(-1, 1)
        row = C
    batch = t.stride(0) if t.shape[0] > 1 else 0
    return t, batch, C if row is None else row


def _like_rows(x):
    """An uninitialised dense channels-last tensor of x's sizes and type."""
    return torch.empty((x.shape[0],) + tuple(x.shape[2:]) + (x.shape[1],), dtype=x.dtype, device=x.device).movedim(-1, 1)


def _forward(x, weight, bias, groups, eps, act):
    x, batch, row = _rows(x)
    N, C = x.shape[:2]
    y = _like_rows(x)
    stats = torch.empty(N, groups, 2, dtype=torch.float32, device=x.device)
    if x.numel():
        lib = _lib.load()
        wbytes = lib.raftcorr_group_norm_workspace_bytes(N, C, groups)
        work = torch.empty(wbytes, dtype=torch.uint8, device=x.device)
        with _guard(x):
            _lib.check(lib.raftcorr_group_norm_fwd(x.data_ptr(), batch, row, _lib.DTYPES[str(x.dtype)], N, x.numel() // (N * C), C, groups,
                                                   None if weight is None else weight.data_ptr(),
                                                   None if bias is None else bias.data_ptr(), eps, act, y.data_ptr(),
                                                   stats.data_ptr(), work.data_ptr(), wbytes, _stream(x)), "group_norm_fwd")
    return x, y, stats


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        x, y, stats = _forward(x, weight, bias, groups, eps, act)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups, ctx.act = groups, act
        ctx.set_materialize_grads(False)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        if dy is None:
            return None, None, None, None, None, None
        x, weight, bias, stats = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        N, C = x.shape[:2]
        dx = _like_rows(x) if need_x else None
        new = torch.empty if x.numel() else torch.zeros
        dw = new(C, dtype=torch.float32, device=x.device) if need_w else None
        db = new(C, dtype=torch.float32, device=x.device) if need_b else None
        if x.numel():
            _, batch, row = _rows(x)
            dy, dbatch, drow = _rows(dy if dy.dtype == x.dtype else dy.to(x.dtype))
            lib = _lib.load()
            wbytes = lib.raftcorr_group_norm_workspace_bytes(N, C, ctx.groups)
            work = torch.empty(wbytes, dtype=torch.uint8, device=x.device)

            def ptr(t):
                return None if t is None else t.data_ptr()

            with _guard(x):
                _lib.check(lib.raftcorr_group_norm_bwd(x.data_ptr(), batch, row, dy.data_ptr(), dbatch, drow, _lib.DTYPES[str(x.dtype)], N,
                                                       x.numel() // (N * C), C, ctx.groups, ptr(weight), ptr(bias), ctx.act,
                                                       stats.data_ptr(), ptr(dx), ptr(dw), ptr(db), work.data_ptr(), wbytes,
                                                       _stream(x)), "group_norm_bwd")
        return dx, dw, db, None, None, None


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, activation="none"):
    """act(group_norm(x)) of a (N, C, *spatial) CUDA tensor in float32, float16 or bfloat16; differentiable in x, weight, bias.

    num_groups divides C; num_groups == C is instance norm.  weight, bias: (C,) or None.  activation: "none", "relu", "silu".
    The result has x's type and lies channels-last (for four dimensions: torch.channels_last).  x is read in place where its
    channels are neighbours and its positions evenly spaced (channels-last tensors, their channel or batch slices); any other
    layout is copied first, and so is the gradient that comes back.  Statistics and sums are float32 whatever x's type.  An
    empty x gives an empty result."""
    _require_cuda(x=x, **{k: t for k, t in (("weight", weight), ("bias", bias)) if t is not None})
    if x.dim() < 2:
        raise RuntimeError(f"x must be (N, C, *spatial), got shape {tuple(x.shape)}")
    if str(x.dtype) not in _lib.DTYPES:
        raise RuntimeError(f"x must be float32, float16 or bfloat16, got {x.dtype}")
    C = x.shape[1]
    groups = int(num_groups)
    if groups < 1 or C % groups or C < 1:
        raise RuntimeError(f"num_groups = {num_groups} does not divide {C} channels")
    if not eps >= 0:
        raise RuntimeError(f"eps = {eps}")
    act = _lib.ACTIVATIONS.get("none" if activation is None else activation)
    if act is None:
        raise RuntimeError(f"activation must be one of {sorted(_lib.ACTIVATIONS)}, got {activation!r}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and (tuple(t.shape) != (C,) or not t.is_floating_point()):
            raise RuntimeError(f"{name} must be a floating-point tensor of shape ({C},), got {t.dtype} {tuple(t.shape)}")
    weight = None if weight is None else weight.float().contiguous()
    bias = None if bias is None else bias.float().contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _GroupNorm.apply(x, weight, bias, groups, float(eps), act)
    return _forward(x, weight, bias, groups, float(eps), act)[1]


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
