"""raft_amd.AdamW against its definition in 64 bits, one step at a time: the definition starts from the state that the kernel left.

Tolerances, u = 2^-24.  32-bit moments: the clipped gradient has two roundings (coefficient, product); the first moment adds
its factor's, a product and the sum: 5 u of the terms' sizes.  The second squares the clipped gradient (four), and adds its factor's,
two products and the sum: 8 u (float32's smallest step besides).  The update lr' m / (sqrt(v) r + eps) carries
the first moment's 5 u (of its terms: they may cancel) and half the second's 8 u; the root and the reciprocal are instructions within
a unit in the last place, 2 u each; r, its product, eps, the sum, the product with m, lr' and its product one u each: 4 + 2 + 2 + 7 = 15,
taken as 16 u of the update's size, and 6 u of lr' (|b1 m| + |(1 - b1) g|) / (sqrt(v) r + eps).  The difference and the decay: 3 u of the
parameter's.
bfloat16 parameters may be either neighbour of that.  8-bit moments are codes: those of the 64-bit
sums rounded to 32 bits, equal bit for bit (the kernel sums in 64 bits too)."""
import copy
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
LOW = 0xFFFFFFFF
U = 2.0 ** -24


def mix(x):
    x = x ^ (x >> np.uint64(16))
    x = (x * np.uint64(0x6A09E667)) & np.uint64(LOW)
    x = x ^ (x >> np.uint64(15))
    x = (x * np.uint64(0xBB67AE85)) & np.uint64(LOW)
    return x ^ (x >> np.uint64(16))


def random_bits(seed, step, start, n):
    pos = np.arange(start, start + n, dtype=np.uint64)
    key = mix((mix(np.uint64((seed + 0x9E3779B9 * step) & LOW)) + (pos >> np.uint64(32))) & np.uint64(LOW))
    return mix(((pos & np.uint64(LOW)) * np.uint64(0x9E3779B9) + key) & np.uint64(LOW))


def blocks(x):
    out = np.zeros((len(x) + 63) // 64 * 64, x.dtype)
    out[:len(x)] = x
    return out.reshape(-1, 64)


def exponents_of(x32):
    bits = blocks(np.abs(x32)).view(np.uint32)
    return (np.where((bits >> 23) == 255, np.uint32(0x7F800000), bits).max(1) >> 23).astype(np.int64)


def codes_of(x32, bits16, top):
    """Codes of |x| and the blocks' exponents, by sums and products."""
    E = exponents_of(x32)
    u = blocks(np.abs(x32)).astype(np.float64) * 2.0 ** (127.0 + top - E)[:, None]
    low = u < 8
    u = np.where(low, (u.astype(np.float32) + np.float32(8)).astype(np.float64) - 8, u)       # below 8 units: to 2^-20 of one
    with np.errstate(invalid="ignore"):
        e = np.where(low, 0, np.frexp(u)[1] - 4)
        whole = np.floor(u / 2.0 ** e + blocks(bits16.astype(np.float64)) / 65536)               # 0..8, or 8..16 half-open binades
        code = np.where(low, whole, whole + 8 * e)
    dead = (E == 0) | (E == 255)
    code = np.where(dead[:, None], 0, code)
    if top == 32:
        code = np.where(~dead[:, None] & (blocks(np.abs(x32)) > 0) & (code == 0), 1, code)
    return code.reshape(-1)[:len(x32)].astype(np.uint8), E.astype(np.uint8)


def values_of(codes, E, top):
    c = codes.astype(np.int64)
    v = np.where(c < 8, c, (8 + (c & 7)) * 2.0 ** ((c >> 3) - 1))
    e = np.repeat(E.astype(np.int64), 64)[:len(c)]
    return np.where(e == 255, np.nan, np.where(e == 0, 0.0, v * 2.0 ** (e - 127.0 - top)))


def flat(t):
    """The values in the order of the tensor's memory."""
    return t.detach().as_strided((t.numel(),), (1,)).float().cpu().numpy().astype(np.float64)


def read(opt):
    """Everything the next step starts from."""
    out = []
    for layout, b in zip(opt.packed_layout(), (b for g in opt._ready() for b in g)):
        for (p, at), slot in zip(layout, range(10 ** 6)):
            n = p.numel()
            s = dict(p=flat(p), step=float(b.steps[slot]), at=at, seed=b.index * 7919)
            if b.bits == 32:
                s["m"], s["v"] = (b.m[at:at + n].cpu().numpy().astype(np.float64), b.v[at:at + n].cpu().numpy().astype(np.float64))
            else:
                sl, ex = slice(at, at + n), slice(at // 64, (at + n + 63) // 64)
                mc, vc = b.m[sl].cpu().numpy(), b.v[sl].cpu().numpy()
                s["codes"] = (mc, vc, b.me[ex].cpu().numpy(), b.ve[ex].cpu().numpy())
                s["m"] = np.where(mc & 128, -1, 1) * values_of(mc & 127, s["codes"][2], 16)
                s["v"] = values_of(vc, s["codes"][3], 32)
            out.append((p, s))
    return out


def check_step(opt, group_of=None, bits=32):
    """One step of opt against the definition, from the state before it."""
    opt._ready()
    before = read(opt)
    grads = [None if p.grad is None else flat(torch.empty_like(p).copy_(p.grad)) for p, _ in before]
    max_norm, clip = opt.defaults["max_norm"], 1.0
    total = math.sqrt(sum(float((g * g).sum()) for g in grads if g is not None))
    if max_norm is not None:
        clip = min(1.0, max_norm / (total + 1e-6))
    opt.step()
    torch.cuda.synchronize()
    if max_norm is not None:
        assert abs(float(opt.grad_norm) - total) <= 2 * U * total
    groups = {id(p): g for g in opt.param_groups for p in g["params"]}
    for (p, old), (_, new), g in zip(before, read(opt), grads):
        if g is None:
            assert new["step"] == old["step"] and np.array_equal(new["p"], old["p"]) and np.array_equal(new["m"], old["m"], equal_nan=True)
            continue
        opts = groups[id(p)]
        t = old["step"] + 1
        assert new["step"] == t
        (b1, b2), lr = opts["betas"], float(opts["lr"])
        e = g * clip
        m, v = b1 * old["m"] + (1 - b1) * e, b2 * old["v"] + (1 - b2) * e * e
        if bits == 32:
            for name, value, size, k in (("m", m, np.abs(b1 * old["m"]) + np.abs((1 - b1) * e), 5), ("v", v, v, 8)):
                assert np.all(np.abs(new[name] - value) <= k * U * size + 2.0 ** -148), name
        else:
            bit = random_bits(opts["seed"] + old["seed"], int(t), old["at"], len(g))
            with np.errstate(over="ignore"):
                m32, v32 = m.astype(np.float32), v.astype(np.float32)
            want = codes_of(m32, bit & np.uint64(0xFFFF), 16), codes_of(v32, bit >> np.uint64(16), 32)
            sign = np.where((m32 < 0) & (np.repeat(want[0][1], 64)[:len(g)] % 255 != 0), 128, 0)
            assert np.array_equal(new["codes"][0], want[0][0] | sign) and np.array_equal(new["codes"][2], want[0][1])
            assert np.array_equal(new["codes"][1], want[1][0]) and np.array_equal(new["codes"][3], want[1][1])
            m, v = m32.astype(np.float64), v32.astype(np.float64)
        with np.errstate(invalid="ignore"):
            factor = lr / (1 - b1 ** t) / (np.sqrt(v) / math.sqrt(1 - b2 ** t) + opts["eps"])
            step, terms = factor * m, factor * (np.abs(b1 * old["m"]) + np.abs((1 - b1) * e))
            value = old["p"] * (1 - lr * opts["weight_decay"]) - step
            bound = 16 * U * np.abs(step) + 6 * U * terms + 3 * U * (np.abs(old["p"]) + np.abs(value)) + 2.0 ** -148
            if p.dtype == torch.bfloat16:
                bound = bound + np.abs(value) * 2.0 ** -7                    # one whole step: up or down
            off = np.abs(new["p"] - value)
        sound = np.isfinite(value)
        assert np.all(off[sound] <= bound[sound]), (off - bound)[sound].max()
        assert np.array_equal(np.isnan(value), np.isnan(new["p"]))


def tensors(dev, sizes, dtype=torch.float32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, n in enumerate(sizes):
        p = torch.nn.Parameter(torch.randn(n, generator=g).to(dtype).to(dev))
        p.grad = (scale * 10.0 ** (-(i % 7)) * torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g))).to(dtype).to(dev)
        out.append(p)
    return out


SIZES = [1, 2, 63, 64, 65, 511, 512, 513, 1000, 4097, 0, 30011]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("max_norm", [None, 0.5, 1e6])
def test_steps(dev, bits, dtype, max_norm):
    from raft_amd import AdamW
    ps = tensors(dev, SIZES, dtype)
    opt = AdamW(ps, lr=3e-3, weight_decay=0.1, state_bits=bits, max_norm=max_norm, seed=5)
    for k in range(4):
        check_step(opt, bits=bits)
        for p in ps:
            p.grad.mul_(0.3).add_(torch.randn_like(p) * 0.01)
        ps[5].grad.zero_()


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(dev, bits):
    """More tensors than one launch's arguments hold, for each of the three kernels (120, 240, 960)."""
    from raft_amd import AdamW
    ps = tensors(dev, [1 + (37 * i) % 700 for i in range(1100)])
    opt = AdamW(ps, state_bits=bits, max_norm=1.0)
    for _ in range(2):
        check_step(opt, bits=bits)


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_are_passed_over(dev, bits):
    from raft_amd import AdamW
    ps = tensors(dev, [700, 5, 64, 1300])
    opt = AdamW(ps, state_bits=bits, max_norm=1.0)
    grads = [p.grad for p in ps]
    for missing in ((), (1, 3), (0,), (0, 1, 2, 3), ()):
        for i, p in enumerate(ps):
            p.grad = None if i in missing else grads[i]
        check_step(opt, bits=bits)
    assert [float(opt.state[p]["step"]) for p in ps] == [3, 3, 4, 3]


@pytest.mark.parametrize("bits", [32, 8])
def test_layouts(dev, bits):
    """Odd addresses, channels-last and transposed parameters, gradients in another order than their parameter's, single values."""
    from raft_amd import AdamW
    g = torch.Generator().manual_seed(1)
    buf, gbuf = torch.randn(5000, generator=g).to(dev), torch.randn(5000, generator=g).to(dev)
    ps = [torch.nn.Parameter(buf[1:1002]), torch.nn.Parameter(buf[1003:4000].view(333, 9))]
    ps[0].grad, ps[1].grad = gbuf[7:1008], gbuf[1001:3998].view(333, 9)
    conv = torch.nn.Parameter(torch.randn(8, 6, 3, 3, generator=g).to(dev).contiguous(memory_format=torch.channels_last))
    conv.grad = torch.randn(8, 6, 3, 3, generator=g).to(dev)
    turned = torch.nn.Parameter(torch.randn(40, 30, generator=g).to(dev).t())
    turned.grad = torch.randn(30, 40, generator=g).to(dev)
    spread = torch.nn.Parameter(torch.randn(50, generator=g).to(dev))
    spread.grad = torch.ones(1, device=dev).expand(50)
    one = torch.nn.Parameter(torch.tensor(2.0, device=dev))
    one.grad = torch.tensor(0.25, device=dev)
    ps += [conv, turned, spread, one]
    opt = AdamW(ps, state_bits=bits, max_norm=1.0)
    rest = buf[1002].item(), buf[4000:].clone(), buf[0].item()
    for _ in range(2):
        check_step(opt, bits=bits)
    assert rest[0] == buf[1002].item() and torch.equal(rest[1], buf[4000:]) and rest[2] == buf[0].item()
    assert opt.state[conv]["exp_avg"].shape == conv.shape and opt.state[conv]["exp_avg"].stride() == conv.stride()
    with pytest.raises(RuntimeError, match="one stretch"):
        bad = torch.nn.Parameter(torch.zeros(4, 6, device=dev)[:, ::2])
        AdamW([bad])._ready()
    conv.data = conv.data.contiguous()
    with pytest.raises(RuntimeError, match="memory order"):
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_types_and_one_norm(dev, bits):
    from raft_amd import AdamW
    a, b, c = tensors(dev, [300, 77]), tensors(dev, [1000], torch.bfloat16, 3), tensors(dev, [65], seed=4)
    opt = AdamW([{"params": a + b, "lr": 1e-2}, {"params": c, "weight_decay": 0.5, "betas": (0.8, 0.95), "eps": 1e-3}], state_bits=bits, max_norm=0.1)
    for _ in range(3):
        check_step(opt, bits=bits)


def test_follows_the_stock_optimizer(dev):
    """24 steps beside torch.optim.AdamW + clip_grad_norm_ on the same gradients; float32 both, so the paths part by rounding alone:
    at most 24 steps of 32 u of lr-sized updates and of the parameter."""
    from raft_amd import AdamW
    ours = tensors(dev, [1000, 33, 4096])
    stock = [torch.nn.Parameter(p.detach().clone()) for p in ours]
    a = AdamW(ours, lr=1e-2, weight_decay=0.01, max_norm=1.0)
    b = torch.optim.AdamW(stock, lr=1e-2, weight_decay=0.01)
    g = torch.Generator().manual_seed(9)
    for k in range(24):
        for p, q in zip(ours, stock):
            p.grad = torch.randn(p.shape, generator=g).to(dev)
            q.grad = p.grad.clone()
        a.step()
        torch.nn.utils.clip_grad_norm_(stock, 1.0)
        b.step()
    for p, q in zip(ours, stock):
        assert (p - q).abs().max() <= 24 * 32 * U * (1e-2 + q.abs().max())


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_resumes_bit_by_bit(dev, bits):
    from raft_amd import AdamW
    import io
    ps = tensors(dev, [513, 64, 7, 2000])
    opt = AdamW(ps, state_bits=bits, max_norm=1.0, seed=3)
    opt.step()
    opt.step()
    buffer = io.BytesIO()
    torch.save(opt.state_dict(), buffer)
    buffer.seek(0)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = AdamW(twins, lr=0.5, state_bits=bits, max_norm=1.0)
    other.load_state_dict(torch.load(buffer, weights_only=True))
    third, pair = copy.deepcopy((opt, ps))
    for p, q, r in zip(ps, twins, pair):
        q.grad, r.grad = p.grad.clone(), p.grad.clone()
    for o in (opt, other, third):
        o.step()
    for p, q, r in zip(ps, twins, pair):
        assert torch.equal(p, q) and torch.equal(p, r)
    for x, y, z in zip(opt.packed_moments(), other.packed_moments(), third.packed_moments()):
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) and torch.equal(x[0], z[0])
    opt.state.clear()                                                # starts anew
    check_step(opt, bits=bits)
    assert float(opt.state[ps[0]]["step"]) == 1


def test_state_goes_to_and_from_the_stock_optimizer(dev):
    from raft_amd import AdamW
    ps = tensors(dev, [100, 700])
    stock = torch.optim.AdamW(ps, lr=1e-2)
    stock.step()
    opt = AdamW(ps, lr=1.0)
    opt.load_state_dict(stock.state_dict())
    assert opt.param_groups[0]["lr"] == 1e-2 and float(opt.state[ps[0]]["step"]) == 1
    assert torch.equal(opt.state[ps[1]]["exp_avg"], stock.state[ps[1]]["exp_avg"])
    check_step(opt)
    back = torch.optim.AdamW(ps)
    back.load_state_dict(opt.state_dict())
    back.step()
    with pytest.raises(RuntimeError, match="shape"):
        AdamW(tensors(dev, [100, 701])).load_state_dict(stock.state_dict())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_replays(dev, bits):
    """A captured step, replayed with new gradients and learning rates and eager work between, against an eager twin."""
    from raft_amd import AdamW
    ps = tensors(dev, [1000, 65, 130])
    twins = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in zip(ps, twins):
        q.grad = p.grad.clone()
    lr = torch.tensor(1e-2, device=dev)
    a, b = (AdamW(x, lr=lr, state_bits=bits, max_norm=1.0) for x in (ps, twins))
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            a.step()
    a.step()
    b.step()
    with torch.cuda.graph(graph):
        a.step()
    norm = a.grad_norm
    for k in range(4):
        for p, q in zip(ps, twins):
            p.grad.normal_().mul_(k + 1)
            q.grad.copy_(p.grad)
        lr.fill_(1e-2 / (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        assert torch.equal(norm, b.grad_norm)
        for p, q in zip(ps, twins):
            assert torch.equal(p, q), k
        assert all(torch.equal(x, y) for x, y in zip(a.packed_moments()[0], b.packed_moments()[0]))


@pytest.mark.parametrize("bits", [32, 8])
def test_buffers_stay_where_a_captured_step_expects_them(dev, bits):
    """A state that is loaded, a group that is added, an entry that someone looks up: the captured step goes on with the state's
    buffers, on the loaded values."""
    from raft_amd import AdamW
    ps = tensors(dev, [1000, 65])
    opt = AdamW(ps, state_bits=bits, max_norm=1.0)
    opt.step()
    saved, then = copy.deepcopy(opt.state_dict()), [p.detach().clone() for p in ps]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    want = [p.detach().clone() for p in ps]
    moments = [t.clone() for t in opt.packed_moments()[0]]
    at = opt.state[ps[0]]["exp_avg"].data_ptr()
    other = torch.zeros(3)
    assert not opt.state[other]                                       # (a defaultdict: this makes an entry)
    opt.add_param_group({"params": tensors(dev, [7], seed=3)})
    opt.step()
    del opt.state[other]
    for p, old in zip(ps, then):
        p.data.copy_(old)
    rest = {k: v for k, v in opt.state_dict()["state"].items() if k > 1}
    groups = opt.state_dict()["param_groups"]
    opt.load_state_dict({"state": {**saved["state"], **rest}, "param_groups": groups})
    assert opt.state[ps[0]]["exp_avg"].data_ptr() == at
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(ps, want))
    assert all(torch.equal(x, y) for x, y in zip(opt.packed_moments()[0], moments))
    assert float(opt.state[ps[1]]["step"]) == 2


def test_values_that_are_not_finite(dev):
    """A NaN gradient spoils its value, with 8 bits its block's moments, and nothing else; an infinite norm clips the rest to zero."""
    from raft_amd import AdamW
    for bits in (32, 8):
        ps = tensors(dev, [256, 256])
        opt = AdamW(ps, state_bits=bits)
        ps[0].grad[70] = float("nan")
        ps[0].grad[130] = float("inf")
        opt.step()
        bad = ps[0].isnan().nonzero().view(-1).tolist()
        assert bad == [70, 130]
        m, v = opt.packed_moments()[0]
        spoiled = (~m[:256].isfinite()).nonzero().view(-1).tolist()
        assert spoiled == ([70, 130] if bits == 32 else list(range(64, 192))) and m[512:768].isfinite().all()
        ps = tensors(dev, [256, 256])
        ps[0].grad[70] = float("inf")
        opt = AdamW(ps, state_bits=bits, max_norm=1.0, weight_decay=0.0)
        keep = ps[1].detach().clone()
        opt.step()
        assert torch.equal(ps[1], keep) and ps[0].isnan().sum() == 1 and math.isinf(float(opt.grad_norm))
        ps = tensors(dev, [70, 256])                                # a coefficient of NaN spoils all values, and no gap between them
        ps[0].grad[5] = float("nan")
        opt = AdamW(ps, state_bits=bits, max_norm=1.0)
        opt.step()
        m, v = opt.packed_moments()[0]
        assert m[:70].isnan().all() and m[512:768].isnan().all() and v[512:768].isnan().all()
        gap = slice(128, 512) if bits == 8 else slice(70, 512)      # (blocks of 64 are spoiled as a whole)
        assert (m[gap] == 0).all() and (v[gap] == 0).all() and (m[768:] == 0).all()


@pytest.mark.parametrize("scale", [1e-30, 1e-22, 1e-10, 1e12])
def test_extreme_gradients(dev, scale):
    from raft_amd import AdamW
    opt = AdamW(tensors(dev, [64, 200, 513], scale=scale), state_bits=8, eps=1e-30)
    for _ in range(2):
        check_step(opt, bits=8)


def test_8_bit_moments_follow_their_averages(dev):
    """400 steps of falling gradients, b2 = 0.99: rounding up or down at random keeps the mean over 4096 values on the exact
    average.  A step's error has mean 0 and a deviation of at most half a code, 1/16 of v; sqrt(1 / (1 - b2^2)) = 7.1 of them stay, and
    the mean over 4096 values of them deviates by at most 7.1 / 16 / 64 = 0.7 %.  2 % are three of those."""
    from raft_amd import AdamW
    n = 4096
    p = torch.nn.Parameter(torch.zeros(n, device=dev))
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.99), state_bits=8)
    m = v = 0.0
    for k in range(400):
        e = 0.99 ** k
        p.grad = torch.full((n,), e, device=dev)
        opt.step()
        m, v = 0.9 * m + 0.1 * p.grad[0].item(), 0.99 * v + 0.01 * p.grad[0].item() ** 2
    got = opt.packed_moments()[0]
    assert abs(got[0].mean().item() / m - 1) < 0.02 and abs(got[1].mean().item() / v - 1) < 0.02


def test_decoded_moments_are_the_codes_values(dev):
    from raft_amd import AdamW
    ps = tensors(dev, [1000, 70])
    opt = AdamW(ps, state_bits=8)
    opt.step()
    for dtype in (torch.float32, torch.bfloat16):
        m, v = opt.packed_moments(dtype)[0]
        for (p, at), (_, s) in zip(opt.packed_layout()[0], read(opt)):
            assert np.array_equal(m[at:at + p.numel()].double().cpu().numpy(), s["m"])
            assert np.array_equal(v[at:at + p.numel()].double().cpu().numpy(), s["v"])
        assert m.dtype == dtype and (m[1000:1024] == 0).all() and (v[1000:1024] == 0).all()


def test_refusals(dev):
    from raft_amd import AdamW
    p = torch.nn.Parameter(torch.zeros(8, device=dev))
    opt = AdamW([p])
    p.grad = torch.zeros(8, device=dev).to_sparse()
    with pytest.raises(RuntimeError, match="dense"):
        opt.step()
    p.grad = None
    assert opt.step(lambda: torch.tensor(3.0)) == 3.0
    with pytest.raises(ValueError, match="lr"):
        AdamW([p], lr=torch.zeros(2))
    whole = torch.zeros(40, device=dev)
    for pair in ((whole[:30], whole[20:]), (whole[3:8], whole)):
        with pytest.raises(RuntimeError, match="share memory"):
            AdamW([torch.nn.Parameter(t) for t in pair])._ready()
    with pytest.warns(UserWarning, match="duplicate"):
        twice = AdamW([p, p])
    with pytest.raises(RuntimeError, match="share memory"):
        twice._ready()
    AdamW([torch.nn.Parameter(whole[:30]), torch.nn.Parameter(whole[30:])])._ready()
    with pytest.raises(RuntimeError, match="decoded"):
        AdamW([p], state_bits=8).packed_moments(torch.float64)


@pytest.mark.parametrize("groups", [1, 2])
@pytest.mark.parametrize("option", [{"lr": -1.0}, {"lr": "empty"}, {"lr": "half"}, {"betas": (0.9, 1.0)}, {"eps": -1.0}, {"weight_decay": float("nan")}], ids=str)
def test_options_are_refused_before_anything_changes(dev, option, groups):
    """An option that went bad after the construction, in the last group: the tensors of the others stay as they are too."""
    from raft_amd import AdamW
    ps = [torch.nn.Parameter(torch.ones(700, device=dev)) for _ in range(groups)]
    opt = AdamW([{"params": [p]} for p in ps], max_norm=1.0)
    for p in ps:
        p.grad = torch.ones_like(p)
    opt.step()
    before = [p.detach().clone() for p in ps] + [opt.state[p][k].clone() for p in ps for k in ("step", "exp_avg", "exp_avg_sq")]
    made = {"empty": torch.empty(0, device=dev), "half": torch.ones((), dtype=torch.float16, device=dev)}
    opt.param_groups[-1].update({k: made.get(v, v) if isinstance(v, str) else v for k, v in option.items()})
    with pytest.raises((ValueError, RuntimeError)):
        opt.step()
    after = [p.detach() for p in ps] + [opt.state[p][k] for p in ps for k in ("step", "exp_avg", "exp_avg_sq")]
    assert all(torch.equal(a, b) for a, b in zip(after, before))


def test_large_tensor(dev):
    """33 million values, the last of them a part of a tile."""
    from raft_amd import AdamW
    n = (1 << 25) + 77
    p = torch.nn.Parameter(torch.ones(n, device=dev))
    p.grad = torch.linspace(-1, 1, n, device=dev)
    opt = AdamW([p], lr=1e-3, weight_decay=0.0, state_bits=8)
    opt.step()
    want = 1 - 1e-3 * p.grad.double() / (p.grad.double().abs() + 1e-8)
    assert (p.double() - want).abs().max() <= 1e-6
