"""Layer norm (ops.layer_norm, modules.LayerNorm, SharedConvAttentionDeconv(use_layer_norm=True)) against the formula in 64
bits, and its gradients against the formula's and against differences.

Tolerances.  u = 2^-24 is half a step of fp32, e = half a step of the storage type (bf16 2^-8, fp32 2^-24).  A row sum is at
most 32 additions a lane, 6 in a wave and 16 across waves, so a sum of n terms is off by at most 54 u sum|term| =: D u n
mean|term|, D = 54.  With r = rstd, h the normalised row:
  mean off by D u mean|x|;  x - mean by that and one rounding;  variance by (D + 4) u v, so r by (D + 4)/2 + 3 < 33 u r;
  h by u (D r mean|x| + 36 |h|);  y = h w + b by that |w|, two roundings, and e |y| for its storage.
  dx = r (g - mean g - h mean(g h)): each mean by D u mean|.| and by what h is off, the rest by 33 + 4 roundings.
  dw = sum over rows of dy h: n roundings of a sum of depth rows / groups + 96, and what h is off."""
import math

import pytest
import torch

from conftest import record_measured, rel_err
from oracle import madiff_oracle as O

pytestmark = pytest.mark.gpu
U, D = 2.0 ** -24, 54
DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _e(t):
    return torch.finfo(t).eps / 2


def _formula(x, w, b, eps, dy=None):
    """-> y, dx, dw, db in float64, and the bounds of each element."""
    t = x.dtype
    x = x.double()
    C = x.shape[-1]
    w = torch.ones(C, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(C, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    r = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    h = (x - mean) * r
    y = h * w + b
    dh = U * (D * r * x.abs().mean(-1, keepdim=True) + 36 * h.abs())
    out = {"y": (y, dh * w.abs() + 3 * U * (y.abs() + (h * w).abs()) + _e(t) * y.abs())}
    if dy is not None:
        dy = dy.double()
        g = dy * w
        m1, m2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
        a1, a2 = g.abs().mean(-1, keepdim=True), (g * h).abs().mean(-1, keepdim=True)
        dx = r * (g - m1 - h * m2)
        off = U * (D * a1 + 2 * g.abs() + h.abs() * D * a2) + dh * m2.abs() + h.abs() * (g.abs() * dh).mean(-1, keepdim=True)
        bound = r * off + 40 * U * r * (g.abs() + m1.abs() + (h * m2).abs()) + _e(t) * dx.abs()
        out["dx"] = (dx, bound)
        rows = x.reshape(-1, C).shape[0]
        depth = rows + 96
        s = lambda v: v.reshape(-1, C).sum(0)                                                        # noqa: E731
        out["dw"] = (s(dy * h), U * depth * s((dy * h).abs()) + s(dy.abs() * dh))
        out["db"] = (s(dy), U * depth * s(dy.abs()))
    return out


def _close(got, want, what):
    ref, bound = want
    got = got.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    bad = (got - ref).abs() - bound
    assert float(bad.max() if bad.numel() else -1.0) <= 0, (what, float((got - ref).abs().max()), float(bad.max()))
    if ref.numel():
        record_measured(float(((got - ref).abs() / bound.clamp_min(1e-300)).max()), "of_bound")


def _data(rows, C, t, seed=0, affine=True):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(rows, C, device=DEV, generator=g) * 1.5 + torch.randn(rows, 1, device=DEV, generator=g)).to(t)
    dy = torch.randn(rows, C, device=DEV, generator=g).to(t)
    w = 1 + 0.3 * torch.randn(C, device=DEV, generator=g) if affine else None
    b = 0.2 * torch.randn(C, device=DEV, generator=g) if affine else None
    return x, dy, w, b


SIZES = [(1, 1), (1, 7), (5, 8), (3, 64), (129, 65), (5, 100), (18, 1024), (7, 333), (2000, 96), (64, 512), (33, 777), (1025, 520),
         (9, 1536), (9, 2048), (5, 2049), (3, 4097), (7, 8192), (3, 16384), (600, 10001), (2, 16385), (3, 32768)]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,C", SIZES)
def test_forward_and_gradients(rows, C, t):
    from madiff_amd import ops
    x, dy, w, b = _data(rows, C, TYPES[t])
    want = _formula(x, w, b, 1e-5, dy)
    _close(ops.layer_norm(x, w, b), want["y"], "no grad")
    for v in (x, w, b):
        v.requires_grad_(True)
    y = ops.layer_norm(x, w, b)
    assert y.dtype == x.dtype
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert dx.dtype == x.dtype and dw.dtype == torch.float32
    for k, v in (("y", y.detach()), ("dx", dx), ("dw", dw), ("db", db)):
        _close(v, want[k], k)


@pytest.mark.parametrize("t", list(TYPES))
def test_without_gain_or_shift_and_partial_gradients(t):
    from madiff_amd import ops
    x, dy, w, b = _data(37, 200, TYPES[t])
    for ww, bb in ((None, None), (w, None), (None, b)):
        want = _formula(x, ww, bb, 1e-5, dy)
        for mask in ("xwb", "x", "wb", "w", "b"):
            args = [v.clone().requires_grad_(k in mask) if v is not None else None for k, v in (("x", x), ("w", ww), ("b", bb))]
            ins = [(k, v) for k, v in zip(("dx", "dw", "db"), args) if v is not None and v.requires_grad]
            if not ins:
                continue
            y = ops.layer_norm(*args)
            _close(y.detach(), want["y"], "y")
            for (k, _), got in zip(ins, torch.autograd.grad(y, [v for _, v in ins], dy)):
                _close(got, want[k], (k, mask))


@pytest.mark.parametrize("t", list(TYPES))
def test_strides_offsets_and_shapes(t):
    from madiff_amd import ops
    base, dyb, _, _ = _data(60, 130, TYPES[t])
    g = torch.Generator(device=DEV).manual_seed(3)
    views = {"columns": base[:, 3:104], "rows": base[::3, :101], "transposed": base[:, :60].t(), "one row": base[7],
             "three axes": base.view(4, 15, 130)[:, 2:, 1:], "expanded": base[:1].expand(50, 130), "columns of one": base[:, 5:6],
             "odd start": base.view(-1)[1:1 + 40 * 33].view(40, 33)}
    for name, x in views.items():
        C = x.shape[-1]
        w, b = 1 + 0.1 * torch.randn(C, device=DEV, generator=g), torch.randn(C, device=DEV, generator=g)
        dy = torch.randn(x.shape, device=DEV, generator=g).to(x.dtype)
        want = _formula(x, w, b, 1e-5, dy)
        xx = x.detach().requires_grad_(True)
        ww, bb = w.requires_grad_(True), b.requires_grad_(True)
        for grad in (dy, dy.mT.contiguous().mT if dy.dim() > 1 else dy):
            y = ops.layer_norm(xx, ww, bb)
            got = torch.autograd.grad(y, (xx, ww, bb), grad)
            for k, v in zip(("y", "dx", "dw", "db"), (y.detach(), *got)):
                _close(v, want[k], (name, k))
        y = ops.layer_norm(xx, ww, bb)                       # sum().backward(): the gradient is one expanded number
        got = torch.autograd.grad(y.float().sum(), (xx, ww, bb))
        one = _formula(x, w, b, 1e-5, torch.ones_like(dy))
        for k, v in zip(("dx", "dw", "db"), got):
            _close(v, one[k], (name, "sum", k))


def test_rows_behind_and_columns_beside_are_left_alone():
    """The C entry writes rows x Cpad of a wider, longer matrix and nothing else; pad columns become zeros."""
    from madiff_amd import lib
    for dt, t in ((lib.BF16, torch.bfloat16), (lib.F32, torch.float32)):
        x, dy, w, b = _data(20, 300, t)
        out = torch.full((24, 360), 7.0, device=DEV, dtype=t)
        dx = torch.full((24, 360), 7.0, device=DEV, dtype=t)
        stats = torch.full((2, 24), 7.0, device=DEV)
        st = torch.cuda.current_stream().cuda_stream
        lib.call("madiff_layer_norm_fwd", dt, x.data_ptr(), 300, out.data_ptr(), 360, w.data_ptr(), b.data_ptr(),
                 stats[0].data_ptr(), stats[1].data_ptr(), 20, 290, 320, 1e-5, st)
        n = 2 * 290 * lib._lib.madiff_layer_norm_groups(dt, 20, 290)
        ws = torch.empty(n, device=DEV)
        dw, db = torch.full((290,), 2.0, device=DEV), torch.full((290,), 2.0, device=DEV)
        lib.call("madiff_layer_norm_bwd", dt, x.data_ptr(), 300, dy.data_ptr(), 300, w.data_ptr(), stats[0].data_ptr(),
                 stats[1].data_ptr(), dx.data_ptr(), 360, dw.data_ptr(), db.data_ptr(), 1, ws.data_ptr(), n, 20, 290, 320, st)
        want = _formula(x[:, :290], w[:290], b[:290], 1e-5, dy[:, :290])
        for m, k in ((out, "y"), (dx, "dx")):
            _close(m[:20, :290], want[k], k)
            assert bool((m[:20, 290:320] == 0).all()) and bool((m[20:] == 7).all()) and bool((m[:, 320:] == 7).all())
        assert bool((stats[:, 20:] == 7).all())
        for v, k in ((dw - 2, "dw"), (db - 2, "db")):        # accumulated onto what was there: one more rounding of it
            ref, bound = want[k]
            _close(v, (ref, bound + 4 * U * (2 + ref.abs())), k)


def test_nan_and_infinity_stay_in_their_rows():
    from madiff_amd import ops
    x, dy, w, b = _data(40, 700, torch.float32)
    x[3, 5], x[9, 0], x[21, 699] = float("nan"), float("inf"), float("-inf")
    x[30] = 4.25                                             # a constant row: variance zero, y = b, dx = 0 up to eps
    keep = [i for i in range(40) if i not in (3, 9, 21)]
    x.requires_grad_(True)
    y = ops.layer_norm(x, w, b)
    dx, = torch.autograd.grad(y, x, dy)
    want = _formula(x.detach()[keep], w, b, 1e-5, dy[keep])
    _close(y.detach()[keep], want["y"], "y")
    _close(dx[keep], want["dx"], "dx")
    for i in (3, 9, 21):
        assert bool(torch.isnan(y[i]).all()) and bool(torch.isnan(dx[i]).all())
    assert torch.equal(y[30], b)


def test_far_mean_and_tiny_and_large_values():
    from madiff_amd import ops
    for shift, scale in ((1e4, 1.0), (0.0, 1e-12), (0.0, 1e15), (-300.0, 1e-2)):
        x, dy, w, b = _data(16, 999, torch.float32)
        x = x * scale + shift
        want = _formula(x, w, b, 1e-5, dy)
        _close(ops.layer_norm(x, w, b), want["y"], (shift, scale))


def test_gradients_straight_into_a_flat_buffer():
    """As the flat optimizers install it (ops.GradSink): two backward passes add up; one tensor as gain and shift gets both sums."""
    from madiff_amd import ops
    rows, C = 77, 96
    x, dy, w, b = _data(rows, C, torch.float32, seed=8)
    want = _formula(x, w, b, 1e-5, dy)
    flat, sink = torch.zeros(3 * C, device=DEV), ops.GradSink()
    w, b, both = (v.clone().requires_grad_(True) for v in (w, b, w))
    for k, v in enumerate((w, b, both)):
        v.grad = flat[k * C:(k + 1) * C]
        sink.register(v, v.grad)
    ops.SINK = sink
    try:
        for k in (1, 2):
            ops.layer_norm(x, w, b).backward(dy)
            for n, v in (("dw", w), ("db", b)):
                _close(v.grad, (k * want[n][0], k * want[n][1] + 2 * U * want[n][0].abs()), (n, k))
        same = _formula(x, both, both, 1e-5, dy)
        ops.layer_norm(x, both, both).backward(dy)
        _close(flat[2 * C:], (same["dw"][0] + same["db"][0],
                              same["dw"][1] + same["db"][1] + 2 * U * (same["dw"][0].abs() + same["db"][0].abs())), "both")
        assert w.grad.data_ptr() == flat.data_ptr()
    finally:
        ops.SINK = None


def test_launches_are_timed_by_name():
    """Under the per-launch timer the calls go another way in Python: the same results, and a record each."""
    from madiff_amd import ops
    x, dy, w, b = _data(33, 200, torch.bfloat16, seed=4)
    x, w, b = (v.requires_grad_(True) for v in (x, w, b))
    run = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, (x, w, b), dy)))(ops.layer_norm(x, w, b))              # noqa: E731
    plain = run()
    ops.TIMER = ops.KernelTimer()
    try:
        timed = run()
        torch.cuda.synchronize()
        names = [r[0] for r in ops.TIMER.records]
    finally:
        ops.TIMER = None
    assert names == ["layer_norm_fwd_kernel", "layer_norm_bwd_kernel"]
    assert all(torch.equal(p, q) for p, q in zip(plain, timed))


def test_empty():
    from madiff_amd import ops
    w, b = torch.ones(9, device=DEV, requires_grad=True), torch.zeros(9, device=DEV, requires_grad=True)
    for shape in ((0, 9), (3, 0, 9)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        y = ops.layer_norm(x, w, b)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.empty(shape, device=DEV))
        assert y.shape == dx.shape == torch.Size(shape) and not dw.any() and not db.any()


def test_differences():
    """Directional derivatives of a scalar of y by central differences of the 64-bit formula, at step s: the truncation is
    s^2 |f'''| / 6 and far below the fp32 gradient's own error, which the bounds of the gradients sum to."""
    from madiff_amd import ops
    x, dy, w, b = _data(11, 77, torch.float32)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    got = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
    want = _formula(x.detach(), w.detach(), b.detach(), 1e-5, dy)
    g = torch.Generator(device=DEV).manual_seed(5)
    for i, k in enumerate(("dx", "dw", "db")):
        v = torch.randn(leaves[i].shape, device=DEV, generator=g, dtype=torch.float64)
        f = lambda s: float((_formula(*[l.detach().double() + (s * v if j == i else 0) for j, l in enumerate(leaves)],  # noqa: E731,E741
                                      1e-5)["y"][0] * dy.double()).sum())
        s = 1e-4
        num = (f(s) - f(-s)) / (2 * s)
        # truncation: f is a product of a smooth function of x at scale >= 1; 1e-8 times the sum of the terms covers s^2/6
        slack = float((want[k][1] * v.abs()).sum()) + 1e-7 * float((want[k][0] * v).abs().sum()) + 1e-7 * float(dy.abs().sum())
        assert abs(num - float((got[i].double() * v).sum())) <= slack, (k, num, float((got[i].double() * v).sum()), slack)


def test_same_bits_on_other_stream_and_in_a_graph():
    from madiff_amd import ops
    x, dy, w, b = _data(3000, 640, torch.bfloat16)
    leaves = [v.requires_grad_(True) for v in (x, w, b)]
    one = lambda: (lambda y: (y.detach(), *torch.autograd.grad(y, leaves, dy)))(ops.layer_norm(*leaves))      # noqa: E731
    first = one()
    assert all(torch.equal(p, q) for p, q in zip(first, one()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = one()
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(first, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        one()
    side.synchronize()
    with torch.cuda.graph(graph):
        held = one()
    old = x.detach().clone()
    for k in range(3):
        with torch.no_grad():
            x.copy_(old if k != 1 else old.flip(0))
        eager = one()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(eager, held)), k


def test_offsets_past_32_bits():
    from madiff_amd import ops
    rows, C = 70001, 32768                                    # 2.29e9 elements
    x = torch.zeros(rows, C, device=DEV, dtype=torch.bfloat16)
    some = torch.tensor([0, 1, 32767, 65535, 65536, 65537, rows - 1], device=DEV)
    part, dpart, w, b = _data(len(some), C, torch.bfloat16)
    x[some] = part
    dy = torch.zeros_like(x)
    dy[some] = dpart
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = ops.layer_norm(x, w, b)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = _formula(part, w.detach(), b, 1e-5, dpart)
    _close(y.detach()[some], want["y"], "y")
    _close(dx[some], want["dx"], "dx")
    _close(dw, want["dw"], "dw")


def test_second_derivative_is_refused():
    from madiff_amd import ops
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(ops.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ---------------------------------------------------------------------------------------------------- in the denoiser
def _normed_attention(p, key, x, temb, nheads=4, residual=True, plain=O.agent_attention):
    """x + gamma attention(norm(x)), the norm over the channels of every (agent, time)."""
    name = key.replace("self_attn", "attn_norm")
    m = x.mean(2, keepdim=True)
    v = (x - m).square().mean(2, keepdim=True)
    n = (x - m) / (v + 1e-5).sqrt() * p[name + ".weight"].to(x.dtype)[:, None] + p[name + ".bias"].to(x.dtype)[:, None]
    return plain(p, key, n, temb, nheads, residual) - n + x


@pytest.mark.parametrize("prec", ["fp32", "bf16"])
def test_denoiser_with_layer_norm(prec, monkeypatch):
    """The whole denoiser, output and every gradient, against the oracle with the norm in front of its attention.
    Tolerances: those of the denoiser without norm (fp32 1e-5 on the output, bf16 2e-2; gradients as in the parity tests)."""
    import diffuser.models as DM
    from madiff_amd import ops
    monkeypatch.setattr(O, "agent_attention", _normed_attention)
    monkeypatch.setattr(ops, "_AUTOTUNE", False)         # no variant timed here is left to later tests of the same layer shapes
    kw = dict(dim=16, dim_mults=(1, 4, 8), returns_condition=True, condition_dropout=0.25, env_ts_condition=True)
    ops.set_precision(prec)
    try:
        net = DM.SharedConvAttentionDeconv(horizon=24, transition_dim=10, n_agents=3, use_layer_norm=True, **kw).to(DEV)
        sd = {k: O.closed_form_param(k, tuple(v.shape)) for k, v in net.state_dict().items()}
        net.load_state_dict(sd)
        cfg = O.DenoiserCfg(horizon=24, transition_dim=10, n_agents=3, **kw)
        p = {k: v.double().requires_grad_(True) for k, v in sd.items()}
        g = torch.Generator().manual_seed(2)
        x = torch.randn(4, 24, 3, 10, generator=g)
        t, r, ets = torch.tensor([0, 3, 7, 100]), torch.rand(4, 1, 3, generator=g), torch.randint(0, 100, (4, 24), generator=g)
        mask = torch.ones(4, 3, 1)
        xr = x.double().requires_grad_(True)
        ref = O.denoiser_forward(p, cfg, xr, t, r.double(), mask.double(), env_timestep=ets)
        dy = torch.randn(ref.shape, generator=g)
        ref.backward(dy.double())
        y = net(x.to(DEV), t.to(DEV), returns=r.to(DEV), env_timestep=ets.to(DEV), dropout_mask=mask.to(DEV))
        y.backward(dy.to(DEV))
        assert rel_err(y.detach().cpu(), ref.detach()) < (1e-5 if prec == "fp32" else 2e-2)
        with torch.no_grad():                                # the sampler's form, no gradients: the same values
            again = net(x.to(DEV), t.to(DEV), returns=r.to(DEV), env_timestep=ets.to(DEV), dropout_mask=mask.to(DEV))
        assert rel_err(again.cpu(), ref.detach()) < (1e-5 if prec == "fp32" else 2e-2)
        seen = 0
        for k, v in net.named_parameters():
            if p[k].grad is None:
                assert v.grad is None, k
                continue
            want = p[k].grad
            if float(want.abs().max()) < 1e-4:               # softmax is shift invariant: key biases
                continue
            l2 = float((v.grad.cpu().double() - want).norm() / want.norm())
            assert l2 < (2e-4 if prec == "fp32" else 0.1), (k, l2)
            seen += k.startswith("attn_norm")
        assert seen == 6                                     # three live norms, weight and bias
    finally:
        ops.set_precision("bf16")
