"""trainer.FlatMuonEMA on the CPU (its host arithmetic, which the tests of the data-parallel machinery use): which parameters are
matrices, where they lie, the step against the formulas in 64 bits, two gloo ranks against one process, refusals.

Tolerance of the 64-bit comparison: u = 2^-24.  Gradients are compared as they enter the step, so only the step itself counts.
Five fp32 products of inner length n <= 16 a step lose about 16 u each, magnified by the iteration's slope, at most 3.4445 a
step and 3.4445^5 = 485 in all: 5 * 3 * 16 u * 485 = 0.007 relative to the 2-norm 1 of X, in an O of 2-norm >= 1, at the very
worst; the update moves the matrix by lr s |O|.  0.007 of that is the bound (a missing momentum or scale is off by 0.05 or more)."""
import copy
import math
import os
import sys

import pytest
import torch
import torch.multiprocessing as mp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NS = (3.4445, -4.7750, 2.0315)


class _Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.emb = torch.nn.Embedding(5, 6)
        self.conv = torch.nn.Conv1d(6, 8, 3, padding=1)
        self.norm = torch.nn.LayerNorm(8)
        self.up = torch.nn.ConvTranspose1d(8, 4, 2, stride=2)
        self.head = torch.nn.Linear(4, 1)
        self.gain = torch.nn.Parameter(torch.ones(1, 4, 1))
        self.unused = torch.nn.Linear(4, 4)

    def forward(self, i):
        x = self.conv(self.emb(i).transpose(1, 2))
        x = self.up(self.norm(x.transpose(1, 2)).transpose(1, 2)) * self.gain
        return self.head(x.transpose(1, 2))


def _net():
    torch.manual_seed(0)
    return _Net()


def _data(steps=3, n=8):
    g = torch.Generator().manual_seed(1)
    return torch.randint(0, 5, (steps, n, 7), generator=g), torch.randn(steps, n, 14, 1, generator=g)


def _reference(net, idx, y, lr, mu, wd, beta, names):
    """A plain loop in 64 bits over a float64 copy of the net."""
    net = copy.deepcopy(net).double()
    p = {k: v for k, v in net.named_parameters()}
    m = {k: torch.zeros_like(v) for k, v in p.items()}
    v2 = {k: torch.zeros_like(v) for k, v in p.items()}
    ema = {k: v.detach().clone() for k, v in p.items()}
    for step in range(len(idx)):
        net.zero_grad(set_to_none=True)
        ((net(idx[step]) - y[step].double()) ** 2).mean().backward()
        with torch.no_grad():
            for k, w in p.items():
                if w.grad is None:
                    continue
                g = w.grad
                if k in names:
                    m[k] = mu * m[k] + (1 - mu) * g
                    u = (1 - mu) * g + mu * m[k]
                    u = u.transpose(0, 1) if k == "up.weight" else u
                    x = u.reshape(u.shape[0], -1)
                    x = x / (x.norm() + 1e-7)
                    for _ in range(5):
                        a = x @ x.T
                        x = NS[0] * x + (NS[1] * a + NS[2] * a @ a) @ x
                    o = x.reshape(u.shape)
                    o = o.transpose(0, 1) if k == "up.weight" else o
                    w.mul_(1 - lr * wd).sub_(lr * 0.2 * math.sqrt(max(x.shape)) * o)
                else:
                    m[k] = 0.9 * m[k] + 0.1 * g
                    v2[k] = 0.999 * v2[k] + 0.001 * g * g
                    w.sub_(lr * (m[k] / (1 - 0.9 ** (step + 1))) / ((v2[k] / (1 - 0.999 ** (step + 1))).sqrt() + 1e-8))
                ema[k] = beta * ema[k] + (1 - beta) * w
    return p, ema


def test_layout_and_formula():
    from madiff_amd.trainer import FlatMuonEMA
    net, (idx, y) = _net(), _data()
    ema = copy.deepcopy(net)
    lr, mu, wd, beta = 1e-2, 0.9, 0.1, 0.8
    want, want_ema = _reference(net, idx, y, lr, mu, wd, beta, ("conv.weight", "up.weight"))
    opt = FlatMuonEMA(net, ema, lr=lr, momentum=mu, weight_decay=wd, ema_decay=beta, use_hip_kernel=False)
    for step in range(len(idx)):
        opt.set_sync(True)
        ((net(idx[step]) - y[step]) ** 2).mean().backward()
        opt.step(do_ema=1)
        opt.zero_grad()
    assert opt.matrices == ["conv.weight", "up.weight"]                  # not the embedding, the gain, the head of one row
    assert opt.split == opt.offsets[opt.names.index("conv.weight")] and opt.flat_v.numel() == opt.split
    assert opt._mats == [(opt.split, 8, 18), (opt.split + 144, 4, 16)] and opt.total == opt.split + 144 + 64
    assert net.unused.weight.grad is None
    for got, ref in ((net, want), (ema, want_ema)):
        for k, v in got.named_parameters():
            o = ref[k].detach()
            size = lr * 0.2 * math.sqrt(18) * 3 if k in opt.matrices else lr   # (elements of Adam's: rounding of g / |g|)
            assert float((v.detach().double() - o).norm()) <= 0.007 * size * math.sqrt(min(o.shape) if o.dim() > 1 else 1), k


def test_selection():
    from madiff_amd.trainer import FlatMuonEMA
    net, (idx, y) = _net(), _data(1)
    seen = []
    opt = FlatMuonEMA(net, None, use_hip_kernel=False, select=lambda n, p: seen.append((n, p.dim())) or n == "up.weight")
    ((net(idx[0]) - y[0]) ** 2).mean().backward()
    opt.step()
    assert sorted(seen) == [("conv.weight", 3), ("up.weight", 3)] and opt.matrices == ["up.weight"]
    net = _net()                                          # nothing selected: Adam alone
    twin = copy.deepcopy(net)
    opt = FlatMuonEMA(net, None, lr=1e-2, use_hip_kernel=False, select=lambda n, p: False)
    ref = torch.optim.Adam(twin.parameters(), lr=1e-2)
    for m, step in ((net, opt.step), (twin, ref.step)):
        ((m(idx[0]) - y[0]) ** 2).mean().backward()
        step()
    assert opt.matrices == [] and opt.split == opt.total
    for a, b in zip(net.parameters(), twin.parameters()):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def _run(rank, world, port, out):
    sys.path.insert(0, ROOT)
    import torch.distributed as dist
    from madiff_amd.trainer import FlatMuonEMA
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    net, (idx, y) = _net(), _data()
    if rank == 1:
        with torch.no_grad():
            net.conv.weight.add_(1.0)                     # broadcast_parameters has to mend this
    ema = copy.deepcopy(net)
    opt = FlatMuonEMA(net, ema, lr=1e-2, bucket_mb=0.0002, use_hip_kernel=False)
    opt.broadcast_parameters(0)
    half = slice(0, 4) if rank == 0 else slice(4, 8)
    for step in range(3):
        for micro in range(2):
            opt.set_sync(micro == 1)
            part = slice(half.start + 2 * micro, half.start + 2 * micro + 2)
            (((net(idx[step, part]) - y[step, part]) ** 2).mean() / 2).backward()
        opt.begin_step(1)
        opt.step(do_ema=1)
        opt.zero_grad()
    assert len(opt.buckets) > 2
    out[rank] = {k: v.detach().clone() for k, v in list(net.state_dict().items()) + [("ema." + k, v) for k, v in ema.state_dict().items()]}
    dist.destroy_process_group()


def test_two_gloo_ranks_match_one_process():
    from madiff_amd.trainer import FlatMuonEMA
    out = mp.get_context("spawn").Manager().dict()
    mp.spawn(_run, args=(2, 28400 + os.getpid() % 400, out), nprocs=2, join=True)
    a, b = out[0], out[1]
    for k in a:
        assert torch.equal(a[k], b[k]), k
    net, (idx, y) = _net(), _data()
    ema = copy.deepcopy(net)
    opt = FlatMuonEMA(net, ema, lr=1e-2, use_hip_kernel=False)
    for step in range(3):
        opt.set_sync(True)
        ((net(idx[step]) - y[step]) ** 2).mean().backward()
        opt.step(do_ema=1)
        opt.zero_grad()
    for k, v in list(net.state_dict().items()) + [("ema." + k, v) for k, v in ema.state_dict().items()]:
        # the order of the gradient's sum: a few u, magnified at most 485 times, of a step of lr * 0.2 sqrt(18)
        assert float((a[k] - v).abs().max()) <= 3 * 485 * 16 * 2.0 ** -24 * 1e-2, k


def test_refusals(monkeypatch):
    from diffuser.utils import Trainer
    from madiff_amd.trainer import FlatMuonEMA
    for bad in (dict(momentum=1.0), dict(momentum=-0.1), dict(momentum=float("nan")), dict(weight_decay=-1.0),
                dict(weight_decay=float("inf")), dict(ns_steps=0), dict(ns_steps=65)):
        with pytest.raises(ValueError):
            FlatMuonEMA(_net(), None, **bad)
    with pytest.raises(ValueError, match="optimizer"):
        Trainer(_net(), None, None, train_device="cpu", optimizer="sgd")
    with pytest.raises(TypeError):
        Trainer(_net(), None, None, train_device="cpu", optimizer="adam", optimizer_kwargs=dict(ns_steps=3))
    tr = Trainer(_net(), None, None, train_device="cpu", optimizer="muon", optimizer_kwargs=dict(ns_steps=3, weight_decay=0.1))
    assert isinstance(tr.optimizer, FlatMuonEMA) and tr.optimizer.ns_steps == 3 and tr.optimizer.weight_decay == 0.1
    monkeypatch.setattr(FlatMuonEMA, "broadcast_parameters", lambda self, src: None)
    monkeypatch.setenv("MADIFF_FORCE_DP", "1")            # a data-parallel step is not captured
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{28900 + os.getpid() % 400}", rank=0, world_size=1)
    try:
        with pytest.raises(NotImplementedError):
            Trainer(_net(), None, None, train_device="cpu", optimizer="muon", use_graph=True)
        assert not Trainer(_net(), None, None, train_device="cpu", optimizer="muon").use_graph
        assert Trainer(_net(), None, None, train_device="cpu", use_graph=True).use_graph
    finally:
        dist.destroy_process_group()
    net, (idx, y) = _net(), _data(1)
    opt = FlatMuonEMA(net, None)                          # the HIP step needs the module on a GPU
    ((net(idx[0]) - y[0]) ** 2).mean().backward()
    with pytest.raises(RuntimeError):
        opt.step()


def test_gradients_below_eps():
    """|U| around and far below eps = 1e-7: X starts as U / max(|U|, eps), so the update of a matrix shrinks with its gradient and is
    that of a unit matrix from eps on.  The bound is that of the header, relative to the update."""
    from madiff_amd.trainer import FlatMuonEMA
    a, b, c = NS
    lr = 1e-2
    for size in (1e-5, 3e-7, 0.9e-7, 1e-9, 1e-13):
        net, (idx, y) = _net(), _data(1)
        opt = FlatMuonEMA(net, None, lr=lr, momentum=0.0, nesterov=False, use_hip_kernel=False)
        ((net(idx[0]) - y[0]) ** 2).mean().backward()
        opt.step()
        opt.zero_grad()
        g = torch.randn(8, 18, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
        g = (g * (size / g.norm())).float()
        opt.flat_m.zero_()
        net.conv.weight.grad.copy_(g.view(8, 6, 3))
        opt.flat_p.zero_()                                # (so that the update does not drown in the weights)
        opt.step()
        x = g.double() / max(float(g.double().norm()), 1e-7)
        for _ in range(5):
            r = x @ x.T
            x = a * x + (b * r + c * r @ r) @ x
        want = -lr * 0.2 * math.sqrt(18) * x
        got = net.conv.weight.detach().double().reshape(8, 18)
        assert float((got - want).norm()) <= 0.007 * float(want.norm()), size


def test_no_capture_next_to_a_process_group(monkeypatch):
    """The end of a capture next to a live process group is what once ended the process: a Muon step is not captured there, be the
    group of one rank and its gradients not reduced, and be it there from the start or since.  Adam's, older and tested, is."""
    import torch.distributed as dist
    from diffuser.utils import Trainer
    from madiff_amd.trainer import FlatAdamEMA, FlatMuonEMA
    monkeypatch.delenv("MADIFF_FORCE_DP", raising=False)
    before = FlatMuonEMA(_net(), None)
    assert before.graphable and FlatAdamEMA(_net(), None).graphable
    dist.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{29300 + os.getpid() % 400}", rank=0, world_size=1)
    try:
        opt = FlatMuonEMA(_net(), None)
        assert not opt.dp and not opt.graphable and not before.graphable
        assert FlatAdamEMA(_net(), None).graphable
        with pytest.raises(NotImplementedError):
            Trainer(_net(), None, None, train_device="cpu", optimizer="muon", use_graph=True)
        assert not Trainer(_net(), None, None, train_device="cpu", optimizer="muon").use_graph
    finally:
        dist.destroy_process_group()
    assert before.graphable
