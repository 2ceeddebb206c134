"""Training with trainer.FlatMuonEMA on the GPU: each step against the formulas in 64 bits (the bounds of test_gpu_ortho), a
replayed step against eager ones, and the layer norm, the attention in front of which it stands, the Trainer and Muon together."""
import copy
import math
import os

import pytest
import torch

from conftest import record_measured, rel_err
from oracle import madiff_oracle as O
from test_gpu_ortho import NS, U, _expect                                                            # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
A, T, FD, ACT, K, B = 3, 12, 10, 5, 20, 4


@pytest.fixture(autouse=True)
def _clean(monkeypatch):
    from madiff_amd import ops
    monkeypatch.setattr(ops, "_AUTOTUNE", False)         # no variant timed here is left to later tests of the same layer shapes
    ops.set_precision("fp32")
    try:
        yield
    finally:
        ops.SINK = None
        ops.set_precision("bf16")


def _build(**kw):
    import diffuser.models as DM
    torch.manual_seed(0)
    net = DM.SharedConvAttentionDeconv(horizon=T, transition_dim=FD, dim=16, dim_mults=(1, 4, 8), n_agents=A,
                                       returns_condition=True, condition_dropout=0.25, **kw)
    dif = DM.GaussianDiffusion(net, n_agents=A, horizon=T, history_horizon=0, observation_dim=FD, action_dim=ACT,
                               n_timesteps=K, returns_condition=True, hidden_dim=32).to(DEV)
    for a in net.self_attn:
        a.gamma.data.fill_(0.3)
    return dif


def _batch(seed):
    from madiff_amd.host import batch_to_device
    b = O.synthetic_batch(B, T, A, FD, ACT, 0, seed=seed)
    g = torch.Generator().manual_seed(seed + 100)
    b.update(t=torch.randint(0, K, (B,), generator=g), noise=torch.randn(B, T, A, FD, generator=g),
             dropout_mask=(torch.rand(B, A, 1, generator=g) < 0.75).float())
    return batch_to_device(b, torch.device(DEV))


@pytest.mark.parametrize("wd,nesterov", [(0.0, True), (0.05, False)])
def test_steps_against_the_formulas(wd, nesterov):
    from madiff_amd import ops
    from madiff_amd.trainer import FlatMuonEMA
    dif = _build()
    ema = copy.deepcopy(dif)
    lr, mu = 1e-3, 0.9
    opt = FlatMuonEMA(dif, ema, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, ema_decay=0.9)
    for step in range(3):
        opt.set_sync(True)
        opt.begin_step(1)
        loss, _ = dif.loss(**_batch(step))
        loss.backward()
        torch.cuda.synchronize()
        if step:
            p, g, m, v, e = (f.clone() for f in (opt.flat_p, opt.flat_g, opt.flat_m, opt.flat_v, opt.flat_ema))
        opt.step(1)
        opt.zero_grad()
        torch.cuda.synchronize()
        if not step:
            assert not ops.SINK is None and opt.plan is not None and 0 < opt.split < opt.total and opt.split == opt.flat_v.numel()
            names = dict(dif.named_parameters())
            assert all(names[n].dim() > 1 for n in opt.matrices) and len(opt.matrices) == len(opt._mats)
            assert {id(names[n]) for n in opt.matrices} >= set(ops.known_gemm_weights()) & {
                id(q) for q in opt.params if min(q.shape[0], q.numel() // q.shape[0]) > 1 and q.dim() > 1}
            continue
        want, want_m, bounds = _expect(opt._mats, p, g, m, lr, mu, wd, nesterov, opt._scales)
        for (at, r, c), b, n in zip(opt._mats, bounds, opt.matrices):
            s = slice(at, at + r * c)
            off = float((opt.flat_p[s].double() - want[s]).norm())
            assert off <= b, (step, n, r, c, off, b)
            record_measured(off / b, "of_bound")
        s, q = slice(0, opt.split), slice(opt.split, opt.total)
        # Adam as madiff_adam_ema defines it: the betas are fp32 numbers and the rests 1 - beta those of these numbers (at 0.999 off
        # by 2^-26 / 0.001 = 1.5e-5 from 0.001, and the second moment with it); the bias corrections come from the host in 64 bits
        G, k, b1, b2 = g[s].double(), step + 1, *torch.tensor([0.9, 0.999]).double().tolist()
        c1, c2 = 1 - 0.9 ** k, 1 - 0.999 ** k
        M, V = b1 * m[s].double() + (1 - b1) * G, b2 * v.double() + (1 - b2) * G * G
        upd = lr * (M / c1) / ((V / c2).sqrt() + 1e-8)
        # some twenty fp32 roundings in the update, where m's two terms may cancel; two in p
        room = lr * 32 * U * ((b1 * m[s].double().abs() + (1 - b1) * G.abs()) / c1) / ((V / c2).sqrt() + 1e-8)
        assert bool(((opt.flat_p[s].double() - (p[s].double() - upd)).abs() <= room + 2 * U * p[s].double().abs() + 1e-12).all())
        lerp = 0.9 * e.double() + (1 - 0.9) * opt.flat_p.double()
        assert bool(((opt.flat_ema.double() - lerp).abs() <= 4 * U * (e.abs() + opt.flat_p.abs()).double()).all())
        assert torch.equal(opt.flat_p16, opt.flat_p.bfloat16()) and not bool(opt.flat_g.any())
        mom = 3 * U * (mu * m[q].double().abs() + (1 - mu) * g[q].double().abs())
        assert bool(((opt.flat_m[q].double() - want_m[q]).abs() <= mom).all())


def _close(got, ref, opt, steps, what):
    """Two runs that issue the same launches.  Gradient sums by atomics come in another order each run: some 2^-19 of the
    gradient's norm, magnified by at most the iteration's slope at zero, 485: 1e-3 of a matrix's step (lr scale in the 2-norm) at
    the most, more through the parameters that differ from then on: 0.02 times the number of steps.  Adam's elements: the part
    of lr that test_gpu_trainer allows.  A missed step or a wrong EMA mode moves a matrix by its whole step."""
    for (at, r, c), sc, n in zip(opt._mats, opt._scales, opt.matrices):
        s = slice(at, at + r * c)
        off = float((got[s].double() - ref[s].double()).norm())
        assert off <= 0.02 * steps * opt.lr * sc, (what, n, off / (opt.lr * sc))
        record_measured(off / (steps * opt.lr * sc), "of_step")
    d = (got[:opt.split] - ref[:opt.split]).abs()
    assert float(d.max()) <= 0.3 * opt.lr * steps and float(d.mean()) <= 0.02 * opt.lr, what


@pytest.mark.parametrize("dp", [False, pytest.param(True, marks=pytest.mark.skip(
    reason="aborted once at the end of the capture, by a thread that is not Python's; cause unknown: GraphedTrainStep refuses "
           "this optimizer under data parallelism"))], ids=["single", "dp_1rank_rccl"])
def test_replayed_steps_match_eager_ones(dp):
    import torch.distributed as dist
    from madiff_amd import ops
    from madiff_amd.trainer import FlatMuonEMA, GraphedTrainStep, train_step
    if dp:
        os.environ["MADIFF_FORCE_DP"] = "1"
        if not dist.is_initialized():
            dist.init_process_group("nccl", init_method="tcp://127.0.0.1:29519", rank=0, world_size=1, device_id=torch.device(DEV))
    try:
        dif, results = _build(), []
        batches = [_batch(s) for s in range(3)]
        for mode in ("eager", "graph"):
            m = copy.deepcopy(dif)
            opt = FlatMuonEMA(m, copy.deepcopy(m), lr=1e-3, ema_decay=0.9, bucket_mb=0.25)
            train_step(m, opt, [batches[0]], do_ema=2)
            if mode == "eager":
                for i in range(5):
                    loss, _ = train_step(m, opt, [batches[i % 3]], do_ema=(0, 1, 2, 1, 1)[i])
            else:
                gs = GraphedTrainStep(m, opt, batches[0])
                for i in range(1, 5):
                    loss, _ = gs.step(batches[i % 3], do_ema=(0, 1, 2, 1, 1)[i])
                    torch.zeros(1000, device=DEV).add_(1.0)                 # the program's own eager work in between
                    torch.cuda.synchronize()
            torch.cuda.synchronize()
            assert opt.dp == dp and opt.step_count == 6 and (not dp or len(opt.buckets) >= 2)
            results.append((opt.flat_p.clone(), opt.flat_ema.clone()))
            ops.SINK = None
        for a, b, what in zip(results[1], results[0], ("weights", "ema")):
            _close(a, b, opt, 6, what)
    finally:
        os.environ.pop("MADIFF_FORCE_DP", None)
        if dp and dist.is_initialized():
            dist.destroy_process_group()


def test_data_parallel_steps_match_single_ones():
    """Eager steps with the gradient's buckets reduced in a 1-rank RCCL group, against steps without one; no capture there."""
    import torch.distributed as dist
    from madiff_amd import ops
    from madiff_amd.trainer import FlatMuonEMA, GraphedTrainStep, train_step
    dif, results = _build(), []
    batches = [_batch(s) for s in range(3)]
    for dp in (False, True):
        if dp:
            os.environ["MADIFF_FORCE_DP"] = "1"
            dist.init_process_group("nccl", init_method="tcp://127.0.0.1:29523", rank=0, world_size=1, device_id=torch.device(DEV))
        try:
            m = copy.deepcopy(dif)
            opt = FlatMuonEMA(m, copy.deepcopy(m), lr=1e-3, ema_decay=0.9, bucket_mb=0.25)
            for i in range(4):
                train_step(m, opt, [batches[i % 3], batches[(i + 1) % 3]], do_ema=(2, 0, 1, 1)[i], fold=False)
            torch.cuda.synchronize()
            assert opt.dp == dp and opt.graphable != dp and opt.step_count == 4 and (not dp or len(opt.buckets) >= 2)
            if dp:
                with pytest.raises(NotImplementedError):
                    GraphedTrainStep(m, opt, batches[0])
            results.append((opt.flat_p.clone(), opt.flat_ema.clone()))
        finally:
            os.environ.pop("MADIFF_FORCE_DP", None)
            if dp:
                dist.destroy_process_group()
            ops.SINK = None
    for a, b, what in zip(results[1], results[0], ("weights", "ema")):
        _close(a, b, opt, 4, what)


class _Items(torch.utils.data.Dataset):
    def __init__(self, n):
        b = O.synthetic_batch(n, T, A, FD, ACT, 0, seed=11)
        g = torch.Generator().manual_seed(12)
        b.update(t=torch.randint(0, K, (n,), generator=g), noise=torch.randn(n, T, A, FD, generator=g),
                 dropout_mask=(torch.rand(n, A, 1, generator=g) < 0.75).float(), env_ts=torch.randint(0, 100, (n, T), generator=g))
        self.b, self.n = b, n

    def __len__(self):
        return self.n

    def __getitem__(self, i):
        return {k: ({kk: vv[i] for kk, vv in v.items()} if isinstance(v, dict) else v[i]) for k, v in self.b.items()}


@pytest.mark.parametrize("prec,env_ts", [("fp32", True), ("fp32", False), ("bf16", True)])
def test_layer_norm_and_muon_in_the_trainer(prec, env_ts, tmp_path):
    """The operators as a user has them: a denoiser with layer norms, trained by Trainer(optimizer="muon"), eagerly and replayed,
    then sampled from."""
    from diffuser.utils import Trainer
    from madiff_amd import ops
    ops.set_precision(prec)
    runs = []
    for use_graph in (False, True):
        dif = _build(use_layer_norm=True, env_ts_condition=env_ts)
        start = {k: v.detach().clone() for k, v in dif.state_dict().items()}
        tr = Trainer(dif, _Items(B * 2 * 4), None, ema_decay=0.9, train_batch_size=B, train_lr=1e-3, gradient_accumulate_every=2,
                     step_start_ema=3, update_ema_every=2, log_freq=100, sample_freq=0, save_freq=100, eval_freq=0,
                     bucket=str(tmp_path), train_device=DEV, use_graph=use_graph, shuffle=False, bucket_mb=0.25, optimizer="muon",
                     optimizer_kwargs=dict(weight_decay=0.01))
        tr.train(6)
        torch.cuda.synchronize()
        opt = tr.optimizer
        assert opt.step_count == 6 and (tr._graphed is not None) == use_graph
        norms = [n for n in opt.names if ".attn_norm." in n]
        assert norms and not set(norms) & set(opt.matrices) and bool(torch.isfinite(opt.flat_p).all())
        for n in norms + opt.matrices:
            assert not torch.equal(dict(dif.named_parameters())[n], start[n]), n
        b = _Items(2).b                                    # sampling with the trained weights, in the graph and step by step
        draw = torch.Generator().manual_seed(3)
        x0, z = 0.5 * torch.randn(2, T, A, FD, generator=draw).to(DEV), torch.randn(K, 2, T, A, FD, generator=draw).to(DEV)
        cond = {k: (v.to(DEV) if torch.is_tensor(v) else {kk: vv.to(DEV) for kk, vv in v.items()}) for k, v in b["cond"].items()}
        plans = [tr.ema_model.conditional_sample(cond, returns=b["returns"].to(DEV), verbose=False,
                                                 env_ts=b["env_ts"].to(DEV) if env_ts else None, x_init=x0, step_noise=z, use_graph=g) for g in (True, False)]
        assert bool(torch.isfinite(plans[0]).all()) and plans[0].shape == (2, T, A, FD)
        assert rel_err(plans[0].cpu(), plans[1].cpu()) < 1e-5       # the same launches, without atomics
        runs.append((opt.flat_p.clone(), opt.flat_ema.clone(), opt))
        ops.SINK = None
    if prec == "fp32":                     # (in bf16 the activations' roundings turn atomics' order into 2^-8)
        for a, b, what in zip(runs[1], runs[0], ("weights", "ema")):
            _close(a, b, opt, 6, what)
