"""raft_amd.group_norm against the formula in 64 bits, forward and backward.

Tolerances.  u = 2^-24.  A gradient's sum here is a tree: 4 rows in registers, at most 16 joins of a thread's own rounds at these
sizes, 10 levels over a workgroup's threads, at most 22 steps over row ranges and channels; with the roundings of the formula
itself no value passes through more than 64.  The statistics are sums in 64 bits that are rounded once.  So z is within 64 u times
(|xh| + |mean| rstd + 1) |w| + |b|, and a result of a 16-bit type is then rounded once (half a step, finfo.eps / 2).  ReLU's slope is
that of z in 64 bits and has no tolerance."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 64 * 2.0 ** -24
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def formula(x, w, b, groups, eps, act, dy):
    """float64 on the CPU: results with their bounds."""
    N, C = x.shape[:2]
    half = 0.0 if x.dtype == torch.float32 else torch.finfo(x.dtype).eps / 2
    tiny = 0.0 if x.dtype != torch.float16 else 2.0 ** -25                       # half of float16's smallest step
    xd = x.detach().cpu().double().reshape(N, groups, -1)
    per = [1, C] + [1] * (x.dim() - 2)
    wd = (torch.ones(C) if w is None else w.detach().cpu()).double().view(per)
    bd = (torch.zeros(C) if b is None else b.detach().cpu()).double().view(per)
    mean = xd.mean(2, keepdim=True)
    var = ((xd - mean) ** 2).mean(2, keepdim=True)
    rstd = (var + eps) ** -0.5
    xh = ((xd - mean) * rstd).view(x.shape)
    shift = (xd.abs().mean(2, keepdim=True) * rstd * torch.ones_like(xd)).view(x.shape)
    rs = (rstd * torch.ones_like(xd)).view(x.shape)
    z = xh * wd + bd
    # the statistics' error times the value: mean within U mean|x|, rstd within U (+ what the mean's error adds)
    zt = U * ((2 * xh.abs() + shift + 1) * wd.abs() + bd.abs())
    s = torch.sigmoid(z)
    y = {"none": z, "relu": z.clamp_min(0), "silu": z * s}[act]
    yt = 1.1 * zt + U * y.abs() + half * y.abs() + tiny
    if dy is None:
        return (y, yt)
    d = dy.detach().cpu().double()
    slope = {"none": torch.ones_like(z), "relu": (z > 0).double(), "silu": s * (1 + z * (1 - s))}[act]
    # an error of z moves the slope of silu by at most half of it
    st = {"none": torch.zeros_like(z), "relu": torch.zeros_like(z), "silu": 0.5 * zt + U * (1 + z.abs())}[act]
    xt = U * (2 * xh.abs() + shift + 1)
    g, gt = d * slope, d.abs() * st + U * (d * slope).abs()
    gw, gwt = g * wd, gt * wd.abs()

    def group_mean(t):
        m = t.reshape(N, groups, -1).mean(2, keepdim=True)
        return (m * torch.ones_like(xd)).view(x.shape)

    s1, s1t = group_mean(gw), group_mean(gwt + U * gw.abs())
    s2, s2t = group_mean(gw * xh), group_mean(gwt * xh.abs() + gw.abs() * xt + U * (gw * xh).abs())
    dx = rs * (gw - s1 - xh * s2)
    dxt = rs * (gwt + s1t + xh.abs() * s2t + xt * s2.abs() + U * (gw.abs() + s1.abs() + (xh * s2).abs()))
    dxt = dxt + U * dx.abs() + half * dx.abs() + tiny
    axes = [0] + list(range(2, x.dim()))
    dw, db = (g * xh).sum(axes), g.sum(axes)
    dwt = (gt * xh.abs() + g.abs() * xt + U * (g * xh).abs()).sum(axes)
    dbt = (gt + U * g.abs()).sum(axes)
    return (y, yt), (dx, dxt), (dw, dwt), (db, dbt)


def near(name, got, want):
    value, bound = want
    err = (got.detach().cpu().double() - value).abs()
    worst = (err - bound).max().item() if err.numel() else 0.0
    assert not err.isnan().any() and worst <= 0, f"{name}: {worst} beyond its bound, largest error {err.max().item()}"


def check(dev, shape, groups, act="relu", dtype="fp32", affine=True, layout="last", train=True, seed=0, eps=1e-5, shift=1.0):
    from raft_amd import group_norm
    g = torch.Generator().manual_seed(seed)
    N, C = shape[:2]
    per = [1, C] + [1] * (len(shape) - 2)
    x = torch.randn(shape, generator=g) * torch.exp(0.5 * torch.randn(per, generator=g)) + shift * torch.randn(per, generator=g)
    x = x.to(DTYPES[dtype]).to(dev)
    dy = torch.randn(shape, generator=g).to(DTYPES[dtype]).to(dev)

    def last(t):
        return t.movedim(1, -1).contiguous().movedim(-1, 1)

    if layout == "last":
        x, dy = last(x), last(dy)
    elif layout == "slice":                      # channels and samples out of a larger channels-last tensor
        big = torch.full((2 * N,) + shape[2:] + (C + 5,), float("nan"), dtype=x.dtype, device=dev)
        big[::2][..., 3:3 + C] = x.movedim(1, -1)
        x = big[::2][..., 3:3 + C].movedim(-1, 1)
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(dev).requires_grad_(train) if affine else None
    b = (0.3 * torch.randn(C, generator=g)).to(dev).requires_grad_(train) if affine else None
    if train:
        x.requires_grad_(True)
    y = group_norm(x, groups, w, b, eps=eps, activation=act)
    assert y.shape == x.shape and y.dtype == x.dtype and y.movedim(1, -1).is_contiguous()
    want = formula(x, w, b, groups, eps, act, dy if train else None)
    if not train:
        near("y", y, want)
        return
    near("y", y, want[0])
    leaves = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    for name, got, ref in zip(("dx", "dw", "db"), grads, want[1:]):
        near(name, got, ref)


SIZES = [((1, 1, 1, 1), 1), ((2, 4, 1, 1), 2), ((3, 6, 2, 1), 6), ((1, 3, 5, 7), 1), ((2, 3, 9, 31), 3), ((2, 8, 13, 17), 8), ((1, 42, 19, 23), 7),
         ((2, 96, 25, 40), 96), ((1, 64, 55, 128), 8), ((3, 33, 31, 33), 11), ((1, 257, 9, 11), 257), ((2, 260, 12, 7), 4), ((1, 1030, 5, 9), 2),
         ((2, 42, 61, 67), 7), ((1, 1030, 40, 41), 5), ((1, 2056, 43, 21), 257), ((5, 3, 71, 73), 1), ((1, 96, 111, 65), 96), ((9, 16, 64, 64), 2),
         ((3, 512, 1, 1), 1), ((70, 24, 8, 9), 24), ((2, 64, 32, 32), 64), ((1, 8200, 2, 3), 5), ((1, 2050, 3, 5), 41), ((1, 4104, 3, 5), 3), ((1, 8, 300, 301), 1), ((130, 16, 3, 3), 4), ((1300, 5, 2, 3), 5)]


@pytest.mark.parametrize("shape,groups", SIZES, ids=lambda v: "x".join(map(str, v)) if isinstance(v, tuple) else f"g{v}")
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_sizes(dev, shape, groups, dtype):
    check(dev, shape, groups, dtype=dtype)


@pytest.mark.parametrize("act", ["none", "relu", "silu"])
@pytest.mark.parametrize("affine", [True, False])
@pytest.mark.parametrize("layout", ["last", "first", "slice"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_activations_weights_and_layouts(dev, act, affine, layout, dtype):
    check(dev, (2, 24, 17, 29), 6, act, dtype, affine, layout, seed=1)
    check(dev, (2, 21, 17, 29), 3, act, dtype, affine, layout, seed=2)


@pytest.mark.parametrize("shape", [(4, 12), (2, 12, 37), (2, 12, 3, 5, 7)], ids=str)
def test_other_dimensions(dev, shape):
    check(dev, shape, 4, "silu", seed=3)


def test_inference_and_training_give_the_same_bits(dev):
    from raft_amd import group_norm
    x = torch.randn(2, 48, 41, 43, device=dev).contiguous(memory_format=torch.channels_last)
    with torch.no_grad():
        a = group_norm(x, 6, activation="relu")
    b = group_norm(x.clone().requires_grad_(True), 6, activation="relu")
    assert torch.equal(a, b) and a.is_contiguous(memory_format=torch.channels_last)
    assert torch.equal(a, group_norm(x, 6, activation="relu"))


def test_large_means_do_not_cancel(dev):
    """mean / width = 1000: with sums of squares in float32 the variance would have no digit left."""
    check(dev, (2, 16, 60, 61), 4, "none", shift=1000.0, seed=4)
    check(dev, (1, 64, 130, 131), 64, "none", affine=False, shift=1000.0, seed=5)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(2, 16, 6, 7), (1, 16, 90, 91)], ids=str)
def test_relu_takes_the_side_of_the_exact_value(dev, dtype, shape):
    """A bias that puts the zero of z a few units of 2^-24 from many of the values, above and below, for weights of both signs and of
    zero: what passes the gradient on is decided as in 64 bits."""
    from raft_amd import group_norm
    g = torch.Generator().manual_seed(11)
    x = torch.randn(shape, generator=g).to(DTYPES[dtype]).to(dev)
    x = x.contiguous(memory_format=torch.channels_last)
    xd = x.double().cpu()
    per = xd.reshape(shape[0], 4, -1)
    mean, var = per.mean(2), per.var(2, unbiased=False)
    rstd = ((var + 1e-5) ** -0.5).repeat_interleave(4, 1)
    mean = mean.repeat_interleave(4, 1)
    w = torch.randn(16, generator=g)
    w[3] = 0.0
    b = torch.empty(16)
    for c in range(16):                                   # the zero close to one of the channel's values
        b[c] = -(xd[0, c, 3, 4] - mean[0, c]) * rstd[0, c] * w[c]
    b = b * (1 + (torch.arange(16) % 5 - 2) * 2.0 ** -23)
    b[3] = 0.25
    z = (xd - mean[:, :, None, None]) * rstd[:, :, None, None] * w.double().view(1, -1, 1, 1) + b.double().view(1, -1, 1, 1)
    for whole in (False, True):                           # d(bias) counts the values that pass: the one at the border, and all of them
        dy = torch.ones_like(x) if whole else torch.zeros_like(x)
        dy[0, :, 3, 4] = 1.0
        leaf = b.to(dev).requires_grad_(True)
        y = group_norm(x, 4, w.to(dev), leaf, activation="relu")
        db, = torch.autograd.grad(y, leaf, dy)
        want = ((z > 0).double() * dy.double().cpu()).sum((0, 2, 3))
        assert torch.equal(db.double().cpu(), want), db.cpu() - want


def test_constant_groups(dev):
    from raft_amd import group_norm
    x = torch.full((2, 8, 9, 9), 3.25, device=dev).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    bias = torch.arange(8.0, device=dev)
    y = group_norm(x, 2, None, bias)
    assert torch.equal(y, bias.view(1, 8, 1, 1).expand_as(y))
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.equal(dx, torch.zeros_like(dx))


def test_values_that_are_not_finite_stay_in_their_group(dev):
    from raft_amd import group_norm
    x = torch.randn(2, 8, 6, 6, device=dev).contiguous(memory_format=torch.channels_last)
    clean = group_norm(x, 4, activation="relu")
    x[0, 2, 1, 1] = float("nan")
    x[1, 7, 0, 3] = float("inf")
    y = group_norm(x, 4, activation="relu")
    assert y[0, 2:4].isnan().all() and y[1, 6:8].isnan().all()
    keep = torch.ones(2, 8, dtype=torch.bool)
    keep[0, 2:4] = keep[1, 6:8] = False
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("shape", [(0, 8, 4, 4), (2, 8, 0, 4)], ids=str)
def test_empty(dev, shape):
    from raft_amd import group_norm
    x = torch.empty(shape, device=dev, requires_grad=True)
    w, b = torch.ones(8, device=dev, requires_grad=True), torch.ones(8, device=dev, requires_grad=True)
    y = group_norm(x, 2, w, b, activation="silu")
    assert y.shape == x.shape
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(shape, device=dev))
    assert dx.shape == x.shape and torch.equal(dw, torch.zeros(8, device=dev)) and torch.equal(db, torch.zeros(8, device=dev))


def test_broadcast_gradient_and_partial_leaves(dev):
    """d(y) of a sum is one value with strides of zero; leaves that need no gradient get none."""
    from raft_amd import group_norm
    x = torch.randn(2, 12, 7, 9, device=dev).contiguous(memory_format=torch.channels_last)
    w = torch.randn(12, device=dev).requires_grad_(True)
    y = group_norm(x, 3, w, None, activation="silu")
    dw, = torch.autograd.grad(y.sum(), w)
    near("dw", dw, formula(x, w, None, 3, 1e-5, "silu", torch.ones_like(x))[2])
    xg = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(group_norm(xg, 3, w.detach(), None, activation="silu").sum(), xg)
    near("dx", dx, formula(x, w, None, 3, 1e-5, "silu", torch.ones_like(x))[1])


def test_16bit_weights_get_16bit_gradients(dev):
    from raft_amd import GroupNorm
    m = GroupNorm(4, 16, activation="relu", device=dev, dtype=torch.bfloat16)
    x = torch.randn(2, 16, 11, 13, device=dev, dtype=torch.bfloat16).contiguous(memory_format=torch.channels_last)
    m(x).float().square().sum().backward()
    assert m.weight.grad.dtype == torch.bfloat16 and m.bias.grad.dtype == torch.bfloat16


def test_gradient_against_differences(dev):
    """Central differences of the kernels' own forward pass in float32 (activation silu, smooth): with h = 2^-7 the formula's error
    is h^2 / 6 times a third derivative of order 1, rounding gives 2^-24 sqrt(count) |loss terms| / h < 2e-4."""
    from raft_amd import group_norm
    g = torch.Generator().manual_seed(7)
    x = torch.randn(1, 6, 4, 5, generator=g).to(dev)
    w, b = torch.randn(6, generator=g).to(dev), torch.randn(6, generator=g).to(dev)
    r = torch.randn(1, 6, 4, 5, generator=g).to(dev)

    def loss(x, w, b):
        return (group_norm(x, 2, w, b, activation="silu").double() * r.double()).sum()

    args = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(loss(*args), args)
    h = 2.0 ** -7
    for k, t in enumerate((x, w, b)):
        for i in range(0, t.numel(), 3):
            up, down = [a.clone() for a in (x, w, b)], [a.clone() for a in (x, w, b)]
            up[k].view(-1)[i] += h
            down[k].view(-1)[i] -= h
            diff = (loss(*up) - loss(*down)).item() / (2 * h)
            assert abs(diff - grads[k].reshape(-1)[i].item()) < 2e-3, (k, i)


def test_captured_step_replays(dev):
    """Forward and backward in one captured graph, replayed with other inputs and eager work between the replays (no eager graph of
    the leaf is alive while the capture runs: torch's accumulation node would belong to the other stream)."""
    from raft_amd import group_norm
    shape = (2, 24, 33, 35)
    x = torch.randn(shape, device=dev).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    w, b = torch.randn(24, device=dev), torch.randn(24, device=dev)
    dy = torch.randn(shape, device=dev).contiguous(memory_format=torch.channels_last)

    def step():
        y = group_norm(x, 4, w, b, activation="relu")
        return y, torch.autograd.grad(y, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(shape, device=dev) * (k + 1))
        graph.replay()
        got = [t.clone() for t in out]
        torch.cuda.synchronize()
        for a, e in zip(got, step()):
            assert torch.equal(a, e), k


def test_another_stream(dev):
    from raft_amd import group_norm
    x = torch.randn(2, 32, 40, 41, device=dev).contiguous(memory_format=torch.channels_last)
    want = group_norm(x, 8, activation="relu")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = group_norm(x, 8, activation="relu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_offsets_beyond_32_bits(dev):
    """2.3 billion values: the second half of the last sample lies behind 2^31 elements."""
    from raft_amd import group_norm
    N, C, H, W = 3, 96, 2000, 4000
    x = torch.empty(N, H, W, C, dtype=torch.float16, device=dev).normal_().movedim(-1, 1)
    y = group_norm(x, 96, activation="none")
    for at in ((N - 1, H - 1, W - 3), (N - 1, 1000, 17), (0, 0, 5)):
        n = at[0]
        channel = 95
        col = x[n, channel].double()
        want = (x[n, channel, at[1], at[2]].double() - col.mean()) / (col.var(unbiased=False) + 1e-5).sqrt()
        assert abs(y[n, channel, at[1], at[2]].double() - want) <= 2.0 ** -11 * abs(want) + 1e-4


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_beyond_the_last_level_cache(dev, dtype):
    """More than 256 MB, where a pass streams most of its rows and the next begins at the end: every value of a few channels.  A
    value passes through 32 rounds of a thread at most here, 10 levels and 6 joins: within the 64 of all the other sizes."""
    from raft_amd import group_norm
    N, C, H, W = 3, 48 if dtype == "fp32" else 104, 750, 683
    g = torch.Generator(dev).manual_seed(3)
    x, dy = [torch.randn(N, H, W, C, generator=g, device=dev).to(DTYPES[dtype]).movedim(-1, 1) for _ in range(2)]
    w, b = [(1 + 0.3 * torch.randn(C, generator=g, device=dev)).requires_grad_(True) for _ in range(2)]
    x.requires_grad_(True)
    y = group_norm(x, C, w, b, activation="relu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    at = [0, 17, C - 1]
    want = formula(x[:, at], w[at], b[at], len(at), 1e-5, "relu", dy[:, at])
    for name, got, ref in zip(("y", "dx", "dw", "db"), (y[:, at], dx[:, at], dw[at], db[at]), want):
        near(name, got, ref)


def test_more_samples_than_a_launch_takes(dev):
    """2^24 + 100 samples of one row: a workgroup each would be 2^32 threads and more.  The channels' sums run over all samples: 64 u of
    the sum of sizes, and x's type is exact enough for d(y) = 1 to make d(bias) a count."""
    from raft_amd import group_norm
    N, C = (1 << 24) + 100, 8
    x = torch.empty(N, C, dtype=torch.float16, device=dev).normal_().requires_grad_(True)
    w, b = torch.ones(C, device=dev, requires_grad=True), torch.zeros(C, device=dev, requires_grad=True)
    y = group_norm(x, 2, w, b, activation="relu")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    for at in (slice(0, 1000), slice((1 << 24) - 500, (1 << 24) + 100)):
        want = formula(x[at].detach(), w, b, 2, 1e-5, "relu", torch.ones_like(x[at]))
        near("y", y[at], want[0])
        near("dx", dx[at], want[1])
    passed, xh = torch.zeros(C, dtype=torch.float64, device=dev), torch.zeros(C, dtype=torch.float64, device=dev)
    sizes = xh.clone()
    for part in x.detach().split(1 << 21):
        d = part.double().view(-1, 2, 4)
        d = d - d.mean(2, keepdim=True)
        z = (d / ((d * d).mean(2, keepdim=True) + 1e-5).sqrt()).view(-1, C)
        passed += (z > 0).sum(0)
        xh += (z * (z > 0)).sum(0)
        sizes += (z * (z > 0)).abs().sum(0)
    assert ((db.double() - passed).abs() <= U * passed).all()
    assert ((dw.double() - xh).abs() <= U * sizes).all()


def test_capture_with_a_live_eager_graph_is_refused(dev):
    from raft_amd import group_norm
    x = torch.randn(2, 8, 6, 7, device=dev).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    dy = torch.ones_like(x)
    eager = group_norm(x, 2)
    with pytest.raises(RuntimeError, match="eager graph of x is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            group_norm(x, 2)
    want, = torch.autograd.grad(eager, x, dy)
    del eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(group_norm(x, 2), x, dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_no_second_derivative(dev):
    from raft_amd import group_norm
    x = torch.randn(2, 8, 6, 7, device=dev, requires_grad=True)
    dx, = torch.autograd.grad(group_norm(x, 2).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiate twice"):
        dx.sum().backward()


def test_refusals(dev):
    from raft_amd import group_norm
    x = torch.randn(2, 8, 6, 7, device=dev)
    for args, words in (((x, 3), "does not divide"), ((x, 0), "does not divide"), ((x.double(), 2), "float32, float16 or bfloat16"), ((x[0, 0, 0], 1), "shape"),
                        ((x, 2, torch.ones(7, device=dev)), "weight must be"), ((x, 2, None, torch.ones(8)), "bias is on cpu"),
                        ((x, 2, torch.ones(8, device=dev).int()), "weight must be"), ((x, 2, None, None, -1.0), "eps")):
        with pytest.raises(RuntimeError, match=words):
            group_norm(*args)
    with pytest.raises(RuntimeError, match="activation"):
        group_norm(x, 2, activation="gelu")
