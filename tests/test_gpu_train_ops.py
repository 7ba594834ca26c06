"""raft_amd.GroupNorm and raft_amd.AdamW where they are used: in the harness's encoders and in a training step."""
import pytest
import torch

from harness.raft_model import RAFT, BasicEncoder, Bottleneck, InputPadder, ResidualBlock, SmallEncoder, sequence_loss, synthetic_pair

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.mark.parametrize("small", [False, True])
def test_flow_with_fused_norms_matches_stock_norms(dev, small):
    """The same weights with the stock instance norms and with GroupNorm: the flow after 12 iterations within the 0.01 px that the
    correlation blocks are held to."""
    from raft_amd import CorrBlock
    i1, i2, _ = synthetic_pair(1, 200, 320, seed=0, device=dev)
    flows = []
    for fused in (False, True):
        torch.manual_seed(0)
        model = RAFT(lambda a, b: CorrBlock(a, b, num_levels=4, radius=3 if small else 4), small=small, fused_norm=fused).to(dev).eval()
        pad = InputPadder(i1.shape)
        with torch.no_grad():
            flows.append(pad.unpad(model(*pad.pad(i1, i2), iters=12)[-1]))
    assert flows[0].abs().max() > 0.1
    assert float((flows[0] - flows[1]).square().sum(1).sqrt().mean()) <= 0.01


def test_encoders_keep_their_parameter_names():
    for make in (BasicEncoder, SmallEncoder):
        for kind in ("instance", "group"):
            stock, fused = make(32, kind), make(32, kind, True)
            assert [k for k, _ in stock.named_parameters()] == [k for k, _ in fused.named_parameters()]
            fused.load_state_dict(stock.state_dict())


@pytest.mark.parametrize("kind", ["instance", "group"])
@pytest.mark.parametrize("block,cin,cout,stride", [(ResidualBlock, 16, 32, 2), (ResidualBlock, 32, 32, 1), (Bottleneck, 32, 64, 2)],
                         ids=["residual_s2", "residual", "bottleneck_s2"])
def test_block_gradients(dev, kind, block, cin, cout, stride):
    """A residual block with fused norms against the stock block in 64 bits on the CPU.  At most 4 convolutions of 32 * 9 terms and 4
    norms of 64 u lie one behind the other, forward and backward: 8 * (288 + 64) u = 1.7e-4 of the largest value, taken as 5e-4 (a norm
    divides by the deviation: what comes in is of order 1)."""
    torch.manual_seed(3)
    stock = block(cin, cout, kind, stride).double()
    fused = block(cin, cout, kind, stride, True)
    fused.load_state_dict(stock.float().state_dict())
    stock.double()
    fused.to(dev).to(memory_format=torch.channels_last)
    x = torch.randn(2, cin, 18, 22)
    a = x.double().requires_grad_(True)
    b = x.to(dev).contiguous(memory_format=torch.channels_last).requires_grad_(True)
    ya, yb = stock(a), fused(b)
    dy = torch.randn(ya.shape)
    ya.backward(dy.double())
    yb.backward(dy.to(dev))
    pairs = [("y", ya, yb), ("dx", a.grad, b.grad)] + [(k, p.grad, q.grad) for (k, p), (_, q) in zip(stock.named_parameters(), fused.named_parameters())]
    largest = max(p.grad.abs().max().item() for p in stock.parameters())
    for name, want, got in pairs:
        scale = want.abs().max().item() if name in ("y", "dx") else largest       # a bias before a norm has a gradient of zero
        assert (got.detach().cpu().double() - want.detach()).abs().max().item() <= 5e-4 * scale, name


@pytest.mark.parametrize("bits", [32, 8])
def test_training_steps(dev, bits):
    """Correlation block, fused norms, loss, backward pass, clipped step: three of them.  With 32-bit moments the parameters are those
    that clip_grad_norm_ and torch.optim.AdamW make of the same gradients: 3 steps of 32 u of the update (at most 4 lr) and of the
    parameter."""
    from raft_amd import AdamW, CorrBlock
    torch.manual_seed(0)
    model = RAFT(lambda a, b: CorrBlock(a, b, num_levels=4, radius=4), fused_norm=True).to(dev).train()
    for m in model.modules():
        if isinstance(m, torch.nn.BatchNorm2d):
            m.eval()
    i1, i2, gt = synthetic_pair(2, 128, 160, seed=1, device=dev)
    ours = AdamW(model.parameters(), lr=2e-4, weight_decay=5e-5, state_bits=bits, max_norm=1.0)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in model.parameters()]
    stock = torch.optim.AdamW(twins, lr=2e-4, weight_decay=5e-5)
    for _ in range(3):
        ours.zero_grad(set_to_none=True)
        loss, _ = sequence_loss(model(i1, i2, iters=3), gt, torch.ones_like(gt[:, 0]))
        loss.backward()
        for p, q in zip(model.parameters(), twins):
            q.grad = None if p.grad is None else p.grad.clone()
        norm = torch.nn.utils.clip_grad_norm_(twins, 1.0)
        stock.step()
        ours.step()
        assert abs(float(ours.grad_norm) / float(norm) - 1) <= 1e-5
    assert all(bool(p.isfinite().all()) for p in model.parameters())
    if bits == 32:
        for p, q in zip(model.parameters(), twins):
            assert (p - q).abs().max() <= 3 * 32 * U * (4 * 2e-4 + q.abs().max())


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_training_step(dev, bits):
    """Norm, loss, backward pass and step in one graph, replayed on new inputs with eager work between, against the same steps taken
    eagerly: the same bits."""
    from raft_amd import AdamW, GroupNorm

    def make():
        torch.manual_seed(2)
        layers = [GroupNorm(4, 32, activation="relu", device=dev), GroupNorm(32, 32, activation="silu", device=dev)]
        return layers, AdamW([p for m in layers for p in m.parameters()], lr=torch.tensor(1e-2, device=dev), state_bits=bits, max_norm=0.5)

    def step(layers, opt, x):
        for p in opt.param_groups[0]["params"]:
            if p.grad is None:
                p.grad = torch.zeros_like(p)
            else:
                p.grad.zero_()
        y = layers[1](layers[0](x))
        (y * y).mean(dim=(0, 2, 3)).mul(0.01).backward(torch.ones(32, device=dev))
        opt.step()

    g = torch.Generator(dev).manual_seed(5)
    inputs = [torch.randn(3, 32, 21, 23, device=dev, generator=g).contiguous(memory_format=torch.channels_last) for _ in range(6)]
    x = inputs[0].clone(memory_format=torch.channels_last)
    a, b = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*a, x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*a, x)
    step(*b, inputs[0])
    for k in range(1, 6):
        x.copy_(inputs[k])
        graph.replay()
        torch.cuda.synchronize()
        step(*b, inputs[k])
        for p, q in zip(a[1].param_groups[0]["params"], b[1].param_groups[0]["params"]):
            assert torch.equal(p, q), k


def test_two_streams_at_once(dev):
    """Two norms and two optimizers on two streams, their calls interleaved: the results of either alone."""
    from raft_amd import AdamW, group_norm
    g = torch.Generator().manual_seed(6)
    xs = [torch.randn(2, 64, 60, 61, generator=g).to(dev).contiguous(memory_format=torch.channels_last) for _ in range(2)]
    sets = [[torch.nn.Parameter(torch.randn(n, generator=g).to(dev)) for n in (3000, 77)] for _ in range(2)]
    for ps in sets:
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(dev)
    alone = [[torch.nn.Parameter(p.detach().clone()) for p in ps] for ps in sets]
    for ps, qs in zip(sets, alone):
        for p, q in zip(ps, qs):
            q.grad = p.grad.clone()
    want = [group_norm(x, 8, activation="silu") for x in xs]
    for qs in alone:
        opt = AdamW(qs, max_norm=1.0, state_bits=8)
        for _ in range(4):
            opt.step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    opts = [AdamW(ps, max_norm=1.0, state_bits=8) for ps in sets]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(group_norm(xs[i], 8, activation="silu"))
                opts[i].step()
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
        assert all(torch.equal(p, q) for p, q in zip(sets[i], alone[i]))
