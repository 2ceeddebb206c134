"""Tensors with a forward-mode tangent are refused by the operators that have no forward-mode derivative: their result would come
back with a derivative of zero, without an error.  (Refused before anything else is looked at, so no GPU is needed.)"""
import pytest
import torch
from torch.autograd import forward_ad


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_tangents_are_refused(device):
    from madiff_amd import ops
    x, w = torch.randn(4, 8, device=device), torch.ones(8, device=device)
    with forward_ad.dual_level():
        dual, dual_w = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, w)
        calls = {"x": lambda: ops.layer_norm(dual), "weight": lambda: ops.layer_norm(x, dual_w), "bias": lambda: ops.layer_norm(x, w, dual_w),
                 "a leaf beside it": lambda: ops.layer_norm(dual, w.clone().requires_grad_(True)),
                 "a view": lambda: ops.layer_norm(dual.t()), "orthogonalize": lambda: ops.orthogonalize(dual),
                 "no grad": lambda: torch.no_grad()(ops.layer_norm)(dual)}
        for name, call in calls.items():
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
                pytest.fail(name)


@pytest.mark.gpu
def test_tangents_in_the_denoiser_form_and_the_optimizer_step():
    from madiff_amd import ops
    from madiff_amd.muon import MuonPlan
    x = torch.randn(4, ops.pad32(20), device="cuda:0", dtype=ops.act_dtype())
    w = torch.ones(20, device="cuda:0")
    plan = MuonPlan([(0, 4, 5)], "cuda:0")
    p, g, m = (torch.ones(20, device="cuda:0") for _ in range(3))
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            ops.layer_norm_cl(forward_ad.make_dual(x, x), w, w, 20)
        with pytest.raises(RuntimeError, match="forward-mode"):
            plan.step(p, forward_ad.make_dual(g, g), m, lr=0.1)
        # a tensor without a tangent passes inside a dual level, and a dual's primal does
        assert torch.equal(ops.layer_norm(x), ops.layer_norm(forward_ad.unpack_dual(forward_ad.make_dual(x, x)).primal))
    assert bool((p == 1).all()) and bool((m == 1).all())
