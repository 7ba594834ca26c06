"""CPU: what raft_amd.group_norm, GroupNorm and AdamW refuse before anything is launched, and what the C ABI refuses."""
import ctypes

import pytest
import torch


def test_group_norm_refuses():
    from raft_amd import GroupNorm, group_norm
    x = torch.zeros(1, 8, 4, 4)
    with pytest.raises(RuntimeError, match="x must be a CUDA tensor"):
        group_norm(x, 2)
    for bad in (dict(num_groups=3), dict(num_groups=0)):
        with pytest.raises(ValueError, match="does not divide"):
            GroupNorm(num_channels=8, **bad)
    with pytest.raises(ValueError, match="activation"):
        GroupNorm(2, 8, activation="gelu")
    with pytest.raises(RuntimeError, match="CUDA"):
        GroupNorm(2, 8)(x)


def test_group_norm_module_takes_stock_checkpoints():
    from raft_amd import GroupNorm
    stock = torch.nn.GroupNorm(4, 16)
    ours = GroupNorm(4, 16, activation="relu")
    assert ours.load_state_dict(stock.state_dict()) and "activation='relu'" in repr(ours)
    assert not list(GroupNorm(16, 16, affine=False).parameters())


def test_rows_are_found_without_copies():
    """Channels-last tensors and their slices are read in place, anything else is copied to dense rows."""
    from raft_amd import _lib
    _rows = _lib.glue().rows
    x = torch.arange(2 * 3 * 4 * 5.0).view(2, 4, 5, 3).movedim(-1, 1)
    t, batch, row = _rows(x)
    assert t.data_ptr() == x.data_ptr() and (batch, row) == (60, 3)
    big = torch.zeros(4, 4, 5, 7).movedim(-1, 1)
    t, batch, row = _rows(big[::2, 2:5])
    assert t.data_ptr() == big[::2, 2:5].data_ptr() and (batch, row) == (280, 7)
    for other in (torch.randn(2, 3, 4, 5), x[:, :, ::2], x[:, :, :, ::2], torch.ones(1, 1, 1, 1).expand(2, 3, 4, 5), x.flip(1), x.movedim(2, 3)):
        t, batch, row = _rows(other)
        assert torch.equal(t, other) and row >= 3
        flat = torch.as_strided(t, (2, t.shape[2] * t.shape[3], 3), (batch, row, 1))
        assert torch.equal(flat, other.movedim(1, -1).reshape(2, -1, 3))
    t, batch, row = _rows(torch.randn(2, 3, 1, 1))
    assert row == 3
    t, batch, row = _rows(torch.randn(5, 1, 4, 4)[:, :, ::2])           # one channel: positions need even steps only
    assert torch.equal(torch.as_strided(t, (5, 8, 1), (batch, row, 1)).view(5, 1, 2, 4), t)


def test_adamw_refuses():
    from raft_amd import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    for bad in (dict(state_bits=16), dict(max_norm=0.0), dict(max_norm=-1.0), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)),
                dict(eps=-1e-8), dict(weight_decay=-1.0), dict(lr=float("nan"))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.float64))])
    opt = AdamW([p])
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match="CUDA"):
        opt.step()
    with pytest.raises(ValueError, match="whole optimizer"):
        opt.add_param_group({"params": [torch.nn.Parameter(torch.zeros(2))], "state_bits": 8})
    assert len(opt.param_groups) == 1
    stock = torch.optim.AdamW([p])
    p.grad = torch.ones(4)
    stock.step()
    with pytest.raises(RuntimeError, match="32-bit moments"):
        AdamW([p], state_bits=8).load_state_dict(stock.state_dict())
    other = torch.optim.AdamW([p], amsgrad=True)
    with pytest.raises(RuntimeError, match="amsgrad"):
        AdamW([p]).load_state_dict(other.state_dict())


def test_c_abi_refuses_without_touching_the_gpu():
    from raft_amd import _lib
    lib = _lib.load()
    ws = lib.raftcorr_group_norm_workspace_bytes(2, 8, 2)
    assert ws > 0 and lib.raftcorr_group_norm_workspace_bytes(2, 8, 3) == 0

    def fwd(x=16, batch=0, row=8, dtype=0, N=2, P=4, C=8, G=2, eps=1e-5, act=0, y=16, stats=16, work=16, bytes_=ws):
        return lib.raftcorr_group_norm_fwd(x, batch, row, dtype, N, P, C, G, None, None, eps, act, y, stats, work, bytes_, None)

    for bad in (dict(x=None), dict(y=None), dict(stats=None), dict(work=None), dict(bytes_=ws - 1), dict(row=7), dict(dtype=3), dict(N=0), dict(P=0),
                dict(C=0), dict(G=3), dict(G=0), dict(act=3), dict(eps=-1.0), dict(eps=float("nan"))):
        assert fwd(**bad) == -1, bad
    assert lib.raftcorr_group_norm_fwd(16, 0, 1 << 21, 0, 1, 4, 1 << 21, 8, None, None, 1e-5, 0, 16, 16, 16, 1 << 62, None) == -2
    assert lib.raftcorr_group_norm_bwd(16, 0, 8, 16, 0, 7, 0, 2, 4, 8, 2, None, None, 0, 16, 16, None, None, 16, ws, None) == -1
    assert b"overlap" in lib.raftcorr_last_error()
    ptr, n = (ctypes.c_void_p * 1)(16), (ctypes.c_int64 * 1)(5)
    off, slot = (ctypes.c_int64 * 1)(0), (ctypes.c_int32 * 1)(0)
    assert lib.raftcorr_adamw_norm_partials(n, 1) == 1 and lib.raftcorr_adamw_norm_partials(None, 1) == 0
    assert lib.raftcorr_adamw_norm(ptr, n, 1, 1, 16, None) == -1 and lib.raftcorr_adamw_norm(ptr, n, 0, 0, 16, None) == -1

    def step(params=ptr, grads=ptr, numels=n, offsets=off, slots=slot, count=1, dtype=0, bits=32, m=16, v=16, me=None, ve=None, steps=16, scale=16,
             lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, partial=None, partials=0, max_norm=0.0, clip=None, norm=None):
        return lib.raftcorr_adamw_step(params, grads, numels, offsets, slots, count, dtype, bits, m, v, me, ve, steps, scale, lr, None, b1, b2, eps,
                                       wd, 0, partial, partials, max_norm, clip, norm, None)

    null, zero, odd = (ctypes.c_void_p * 1)(), (ctypes.c_int64 * 1)(0), (ctypes.c_int64 * 1)(64)
    for bad in (dict(params=null), dict(grads=null), dict(numels=zero), dict(offsets=odd), dict(count=0), dict(dtype=1), dict(bits=16), dict(bits=8),
                dict(m=None), dict(steps=None), dict(scale=None), dict(lr=-1.0), dict(lr=float("nan")), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0),
                dict(wd=-1.0), dict(partials=1), dict(partials=-1), dict(partials=1, partial=16, clip=16, norm=16)):
        assert step(**bad) == -1, bad
    huge = (ctypes.c_int64 * 1)(1 << 40)
    assert step(numels=huge) == -2
    assert lib.raftcorr_adamw_decode(16, 16, 16, 16, 500, 0, 16, 16, None) == -1
    assert lib.raftcorr_adamw_decode(16, 16, 16, 16, 512, 1, 16, 16, None) == -1


def test_constants_match_the_header():
    import os
    import re
    from conftest import ROOT
    from raft_amd import _lib
    text = open(os.path.join(ROOT, "include", "raftcorr.h")).read()
    named = dict(re.findall(r"#define RAFTCORR_(\w+)\s+(\d+)\s", text))
    assert {k: str(v) for k, v in (("ADAMW_TILE", _lib.ADAMW_TILE), ("ADAMW_BLOCK", _lib.ADAMW_BLOCK))}.items() <= named.items()
    assert {f"ACT_{k.upper()}": str(v) for k, v in _lib.ACTIVATIONS.items()}.items() <= named.items()
    assert _lib.DTYPES == {"torch.float32": int(named["DTYPE_FP32"]), "torch.float16": int(named["DTYPE_FP16"]), "torch.bfloat16": int(named["DTYPE_BF16"])}


def test_random_bits_are_even():
    """The position hash of the stochastic rounding (stated here in Python): bits balanced, neighbours and successive steps
    unrelated.  2^18 draws: a fair bit's count deviates by 5 standard deviations (1280) once in 10^6."""
    import numpy as np
    low = np.uint64(0xFFFFFFFF)

    def mix(x):
        x = x ^ (x >> np.uint64(16))
        x = (x * np.uint64(0x6A09E667)) & low
        x = x ^ (x >> np.uint64(15))
        x = (x * np.uint64(0xBB67AE85)) & low
        return x ^ (x >> np.uint64(16))

    def draw(step):
        pos = np.arange(1 << 18, dtype=np.uint64)
        key = mix(mix(np.uint64((0x9E3779B9 * step) & 0xFFFFFFFF)))
        return mix((pos * np.uint64(0x9E3779B9) + key) & low)

    a, b = draw(1), draw(2)
    for word in (a, b, a ^ b, a[1:] ^ a[:-1], a[512:] ^ a[:-512]):
        for bit in range(32):
            ones = int(((word >> np.uint64(bit)) & np.uint64(1)).sum())
            assert abs(ones - len(word) / 2) < 5 * 256
    for half in (a & np.uint64(0xFFFF), a >> np.uint64(16)):
        assert abs(half.astype(float).mean() / 32767.5 - 1) < 5 * 0.5774 / 512
    x, y = (a & np.uint64(0xFFFF)).astype(float), (a >> np.uint64(16)).astype(float)
    assert abs(np.corrcoef(x, y)[0, 1]) < 5 / 512
