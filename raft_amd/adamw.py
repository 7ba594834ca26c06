"""The optimizer step of RAFT's training recipe -- AdamW behind clip_grad_norm_ (core/train_origin.py:84-95,210-216) -- over all
tensors of a model in a few launches, with moments in 32 or in 8 bits, backed by libraftcorr.so (C ABI in include/raftcorr.h).

PyTorch is used for device memory, streams and the optimizer's bookkeeping only (csrc/glue.cpp walks the parameters); there is no
fallback path.
"""
import torch

from . import _lib
from .corr import _guard, _stream

__all__ = ["AdamW"]

_DTYPES = (torch.float32, torch.bfloat16)


class _Bucket:
    """The parameters of one group that share device and type, and their state in flat buffers: parameter i's moments start at
    value offsets[i], a multiple of the tile, in the order of the parameter's own memory."""

    def __init__(self, params, bits, index):
        self.params, self.bits, self.index = params, bits, index
        self.device, self.dtype = params[0].device, params[0].dtype
        self.strides = [p.stride() for p in params]
        self.glue = _lib.glue().Bucket(params)
        self.numels, self.offsets, self.total = self.glue.numels, self.glue.offsets, self.glue.total
        total = self.total
        kind = torch.float32 if bits == 32 else torch.uint8
        self.m, self.v = (torch.zeros(total, dtype=kind, device=self.device) for _ in range(2))
        blocks = 0 if bits == 32 else total // _lib.ADAMW_BLOCK
        self.me, self.ve = (torch.zeros(blocks, dtype=torch.uint8, device=self.device) for _ in range(2))
        self.steps = torch.zeros(len(params), dtype=torch.float32, device=self.device)
        self.state = [self._views(i) for i in range(len(params))]        # what stands in the optimizer's state

    def holds(self, params):
        """Whether the bucket is that of these parameters as they are now."""
        return (len(params) == len(self.params) and all(p is q for p, q in zip(params, self.params)) and
                all(p.stride() == s and p.numel() == n for p, s, n in zip(params, self.strides, self.numels)))

    def _views(self, i):
        p, at = self.params[i], self.offsets[i]
        out = {"step": self.steps[i]}
        for name, flat in (("exp_avg", self.m), ("exp_avg_sq", self.v)):
            out[name] = flat.as_strided(p.shape, p.stride(), at)
        if self.bits == 8:
            first, last = at // _lib.ADAMW_BLOCK, (at + self.numels[i] + _lib.ADAMW_BLOCK - 1) // _lib.ADAMW_BLOCK
            out["exp_avg_exponent"], out["exp_avg_sq_exponent"] = self.me[first:last], self.ve[first:last]
        return out


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW (without amsgrad and maximize) with the clipping by the gradients' global norm inside the step.

    state_bits  32, or 8: each moment in one byte and one exponent byte for 64 of them (include/raftcorr.h); coded with
                stochastic rounding whose random bits come from (seed, step, position) alone, so a run repeats bit by bit.
    max_norm    None, or the bound on the 2-norm over all gradients of the optimizer.  The gradients themselves stay as they
                are; the norm of the last step is in `grad_norm` (a device tensor).
    lr          a number, or a float32 tensor on the parameters' device, which a captured step reads anew at each replay.

    Parameters: CUDA, float32 or bfloat16 (rounded stochastically; no 32-bit copy is kept), in one stretch of memory.
    Gradients: of the parameters' type; parameters without one are passed over.  A step can be captured into a HIP graph once
    one step has been taken; numbers among its options stay what they were.  `state` holds views ("step", "exp_avg", "exp_avg_sq",
    with 8 bits their codes and exponents) into one buffer a bucket of parameters: write into them, another tensor put in their
    place is not seen.  torch.optim.AdamW's state_dict can be loaded with state_bits=32, and the other way round.
    """

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, max_norm=None, seed=0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_norm is not None and not max_norm > 0:
            raise ValueError(f"max_norm must be positive or None, got {max_norm}")
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, max_norm=max_norm, seed=int(seed))
        self._buckets, self._stale, self._held = [], True, 0
        self.grad_norm = None
        super().__init__(params, defaults)

    def __setstate__(self, state):
        super().__setstate__(state)
        if "_buckets" not in self.__dict__:                   # unpickled or copied
            self._buckets, self._held, self.grad_norm = [], 0, None
        self._stale = True

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            _options(group)
            if group["state_bits"] != self.defaults["state_bits"] or group["max_norm"] != self.defaults["max_norm"]:
                raise ValueError("state_bits and max_norm hold for the whole optimizer")
            for p in group["params"]:
                if p.dtype not in _DTYPES:
                    raise ValueError(f"parameters must be float32 or bfloat16, got {p.dtype}")
        except ValueError:
            self.param_groups.pop()
            raise
        self._stale = True

    # -- state ------------------------------------------------------------------------------------------------------

    def _ready(self):
        """The buckets, one list a group: made on the first call, and made to hold what `state` says after it was loaded or
        emptied or a group was added.  Buffers of unchanged buckets stay where they are (a captured step may use them)."""
        if not self._stale and len(self.state) >= self._held and (not self._held or self.state.get(self._first[0]) is self._first[1]):
            return self._buckets
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: take one step before a step is captured (the state is made by the first one)")
        bits, made, known = self.defaults["state_bits"], [], [b for buckets in self._buckets for b in buckets]
        for group in self.param_groups:
            by_kind = {}
            for p in group["params"]:
                if not p.is_cuda:
                    raise RuntimeError("parameter must be a CUDA tensor")
                if p.dtype not in _DTYPES:
                    raise RuntimeError(f"parameters must be float32 or bfloat16, got {p.dtype}")
                if p.numel():
                    by_kind.setdefault((p.device, p.dtype), []).append(p)
            made.append([])
            for (device, dtype), params in by_kind.items():
                index = sum(map(len, made))
                old = [b for b in known if b.index == index and (b.device, b.dtype) == (device, dtype) and b.holds(params)]
                made[-1].append(old[0] if old else _Bucket(params, bits, index))
        buckets = [b for of in made for b in of]
        if _lib.glue().Bucket.overlap([p for b in buckets for p in b.params]):
            raise RuntimeError("two parameters share memory (or one is listed twice)")
        for b in buckets:
            for p, views in zip(b.params, b.state):
                old = self.state.get(p)
                if old is not views:
                    if old:
                        _adopt(views, old, bits)
                    else:
                        for t in views.values():
                            t.zero_()
                    self.state[p] = views
        self._buckets, self._stale, self._held = made, False, sum(len(b.params) for b in buckets)
        self._first = (buckets[0].params[0], buckets[0].state[0]) if buckets else None
        return made

    def load_state_dict(self, state_dict):
        """Takes the values as they are: the base class would cast them to the parameter's type."""
        for old in state_dict["state"].values():
            if old:
                _adopt(None, old, self.defaults["state_bits"])          # refused before anything is taken over
        for group in state_dict["param_groups"]:
            if group.get("amsgrad") or group.get("maximize"):
                raise RuntimeError("the loaded state is one of amsgrad or maximize")
        super().load_state_dict(state_dict)
        for group in self.param_groups:
            _options(group)
            group["state_bits"], group["max_norm"] = self.defaults["state_bits"], self.defaults["max_norm"]
            group.setdefault("seed", self.defaults["seed"])
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        params = [p for g in self.param_groups for p in g["params"]]
        for i, p in zip(ids, params):
            old = state_dict["state"].get(i)
            if old:
                self.state[p] = {k: v.detach().clone() if torch.is_tensor(v) else v for k, v in old.items()}
        self._stale = True
        if params and all(p.is_cuda for p in params):
            self._ready()

    def packed_moments(self, dtype=None):
        """[(first, second moments)] of each bucket (a group's parameters of one device and type) as flat tensors, laid out as
        packed_layout says.  32 bits: the state itself, or a copy in `dtype`.  8 bits: decoded to float32 or bfloat16 (which holds
        the codes' values exactly from 2^-126 up)."""
        out = []
        for b in (b for buckets in self._ready() for b in buckets):
            if b.bits == 32:
                out.append((b.m, b.v) if dtype is None else (b.m.to(dtype), b.v.to(dtype)))
                continue
            kind = torch.float32 if dtype is None else dtype
            if kind not in _DTYPES:
                raise RuntimeError(f"8-bit moments are decoded to float32 or bfloat16, not {kind}")
            m, v = (torch.empty(b.total, dtype=kind, device=b.device) for _ in range(2))
            with _guard(m):
                _lib.check(_lib.load().raftcorr_adamw_decode(b.m.data_ptr(), b.v.data_ptr(), b.me.data_ptr(), b.ve.data_ptr(), b.total,
                                                             _lib.DTYPES[str(kind)], m.data_ptr(), v.data_ptr(), _stream(m)), "adamw_decode")
            out.append((m, v))
        return out

    def packed_layout(self):
        """[[(parameter, offset)]] of each bucket: where a parameter's moments start in packed_moments (values, a multiple of 512;
        the gaps are zero).  They follow the order of the parameter's memory."""
        return [list(zip(b.params, b.offsets)) for buckets in self._ready() for b in buckets]

    # -- step -------------------------------------------------------------------------------------------------------

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        buckets = self._ready()
        work = [(group, b) for group, of in zip(self.param_groups, buckets) for b in of if b.glue.collect(b.params)]
        for group, b in work:               # options that went bad since, before anything is changed (one bucket's numbers: by the call itself)
            lr = group["lr"]
            if len(work) > 1 or torch.is_tensor(lr):
                _options(group)
                if torch.is_tensor(lr) and lr.is_cuda and lr.device != b.device:
                    raise RuntimeError(f"lr is on {lr.device}, expected {b.device}")
        max_norm, partial, self.grad_norm = self.defaults["max_norm"], None, None
        if max_norm is not None:
            device = work[0][1].device if work else None
            if any(b.device != device for _, b in work):
                raise RuntimeError("max_norm: the parameters are on more than one device")
            self.grad_norm = torch.empty((), dtype=torch.float32, device=device) if work else torch.zeros(())
            if work:
                pieces = [b.glue.partials() for _, b in work]
                partial, at = torch.empty(sum(pieces) + 1, dtype=torch.float64, device=device), 0      # the last one: the coefficient
                for (_, b), n in zip(work, pieces):
                    b.glue.norm(partial, at)
                    at += n
        for group, b in work:
            lr, (b1, b2) = group["lr"], group["betas"]
            on_device = lr if torch.is_tensor(lr) and lr.is_cuda else None
            b.glue.step(b.bits, b.m, b.v, b.me, b.ve, b.steps, on_device, 0.0 if on_device is not None else float(lr), b1, b2, group["eps"],
                        group["weight_decay"], (group["seed"] + 7919 * b.index) & 0xFFFFFFFF, partial, max_norm or 0.0, self.grad_norm)
        return loss


def _options(group):
    lr, betas, eps, decay = group["lr"], group["betas"], group["eps"], group["weight_decay"]
    if torch.is_tensor(lr):
        if lr.numel() != 1 or (lr.is_cuda and lr.dtype != torch.float32):
            raise ValueError(f"lr must be a number or one float32 value, got {lr.dtype} {tuple(lr.shape)}")
    elif not lr >= 0:
        raise ValueError(f"lr = {lr}")
    if not (len(betas) == 2 and all(0 <= b < 1 for b in betas)):
        raise ValueError(f"betas = {betas}")
    if not eps >= 0 or not decay >= 0:
        raise ValueError(f"eps = {eps}, weight_decay = {decay}")


def _adopt(views, old, bits):
    """The values of a parameter's loaded state into the buffers (views: a bucket's; None: only look whether they fit)."""
    names = ["exp_avg", "exp_avg_sq"] + (["exp_avg_exponent", "exp_avg_sq_exponent"] if bits == 8 else [])
    held = 8 if "exp_avg_exponent" in old else 32
    if held != bits or any(k not in old for k in names):
        raise RuntimeError(f"the loaded state holds {held}-bit moments, this optimizer keeps {bits}-bit ones")
    if views is None:
        return
    for name in names:
        if old[name].shape != views[name].shape:
            raise RuntimeError(f"the loaded {name} has shape {tuple(old[name].shape)}, expected {tuple(views[name].shape)}")
        if bits == 8 and not _lib.glue().same_order(old[name], views[name]):
            raise RuntimeError(f"the loaded {name} has another memory order than the parameter: its blocks of 8-bit values differ")
        views[name].copy_(old[name])
    views["step"].fill_(float(old["step"]))
