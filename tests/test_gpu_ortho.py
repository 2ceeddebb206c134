"""Newton-Schulz orthogonalisation (ops.orthogonalize) and the Muon step (muon.MuonPlan) against their formulas in 64 bits.

Tolerance of the orthogonalised matrix.  The iteration magnifies rounding errors in a way that depends on the spectrum, so the
measure is what the same iteration in fp32 is off by on the same input, E32 (2-norm of the difference over 2-norm of the result).
An operand kept as two fp16 numbers is within 2^-23 of its value where fp32 rounds by 2^-24, the product leaves out a term below
2^-22 of the product's and sums in fp32 as the fp32 product does: each product is within (2 x 2^-23 + 2^-22) / (2 x 2^-24) = 4
times its fp32 counterpart's operand rounding plus its sum's rounding, at most 5 times the fp32 product's error altogether, and
so is the result to first order: E <= 5 E32 + 2^-23 (the final rounding to fp32; 2^-8 instead where the output is bf16).
E32 is one sample, though, and for a matrix of one or few elements its roundings can cancel (to 2^-27 for the 1 x 1 below), so
what ONE step may lose is added.  With u = 2^-24 and singular values near 1, from an exact X: a split product is within 8 u of
its terms and storing one within 2 u, so A is off by 10 u A, A A by (2 x 10 + 8) u = 28 u, R = b A + c A A by 4.775 x 10 u +
2.0315 x 28 u + 2 u |R| <= 110 u (|R| <= 2.75), R X by 110 u + 8 u |R| = 132 u, and X' = a X + R X by 2 u (a + |R|) more: 145 u,
which over |X'| >= 0.69 is 210 u = LAST.  Leaving out one of the three products costs 2^-12 = 4096 u before any magnification."""
import math

import pytest
import torch

from conftest import record_measured

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NS = (3.4445, -4.7750, 2.0315)
U = 2.0 ** -24
LAST = 210 * U
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def newton_schulz(x, steps=5, coef=NS, eps=1e-7):
    a, b, c = coef
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT.contiguous() if tall else x
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp_min(eps)
    for _ in range(steps):
        g = x @ x.mT.contiguous()
        x = a * x + (b * g + c * (g @ g)) @ x
    return x.mT.contiguous() if tall else x


def _check(got, x, steps=5, coef=NS, eps=1e-7, what=""):
    """got [.., r, c] against the 64-bit iteration on x, matrix by matrix."""
    want = newton_schulz(x.double(), steps, coef, eps)
    f32 = newton_schulz(x.float(), steps, coef, eps).double()
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    last = 2.0 ** -8 if x.dtype == torch.bfloat16 else 2.0 ** -23
    norm = lambda v: v.double().square().sum((-2, -1)).sqrt()                                        # noqa: E731
    size = norm(want)
    bound = 5 * norm(f32 - want) + (last + LAST) * size
    off = norm(got.double() - want)
    assert bool((off <= bound).all()), (what, (off / size).max().item(), (bound / size).min().item())
    if size.numel():
        record_measured(float((off / bound.clamp_min(1e-300)).max()), "of_bound")


def _grad(shape, seed, rank=None, scale=1e-3, noise=0.1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    *b, r, c = shape
    k = rank or max(1, min(r, c) // 8)
    fall = torch.arange(1, k + 1, device=DEV).float().pow(-0.7)
    return ((torch.randn(*b, r, k, device=DEV, generator=g) * fall) @ torch.randn(*b, k, c, device=DEV, generator=g)
            + noise * torch.randn(*b, r, c, device=DEV, generator=g)) * scale


SHAPES = [(1, 1), (1, 5), (7, 1), (2, 3), (16, 128), (31, 33), (127, 129), (128, 128), (129, 128), (128, 640), (130, 1000), (700, 100),
          (333, 1001), (1024, 256), (257, 511), (512, 2560), (5, 20011), (1100, 1100),
          (32, 1216), (1248, 30), (64, 512), (64, 513), (128, 192), (190, 127), (97, 224), (96, 290), (128, 256)]


@pytest.mark.parametrize("t", list(TYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_shapes(rows, cols, t):
    from madiff_amd import ops
    x = _grad((rows, cols), rows * 7 + cols).to(TYPES[t])
    _check(ops.orthogonalize(x), x)
    xb = _grad((3, rows, cols), rows + cols).to(TYPES[t])
    _check(ops.orthogonalize(xb), xb)


@pytest.mark.parametrize("kind", ["gauss", "low rank", "orthogonal", "one row large", "tiny", "huge", "diagonal"])
def test_spectra(kind):
    from madiff_amd import ops
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(200, 600, device=DEV, generator=g)
    if kind == "low rank":
        x = torch.randn(200, 10, device=DEV, generator=g) @ torch.randn(10, 600, device=DEV, generator=g) + 1e-4 * x
    elif kind == "orthogonal":
        x = torch.linalg.qr(x.t().cpu())[0].t().contiguous().to(DEV)
    elif kind == "one row large":
        x[3] *= 1e6
    elif kind == "tiny":
        x *= 1e-30                        # the squares leave fp32; |x| is far below eps, so X0 = x / eps
    elif kind == "huge":
        x *= 1e25
    elif kind == "diagonal":
        x = torch.zeros(200, 600, device=DEV)
        x[torch.arange(200), torch.arange(200) * 3] = torch.logspace(-6, 0, 200, device=DEV)
    if kind == "huge":                    # (the fp32 yardstick needs squares in range: the same matrix, 2^-80 of it)
        _check(ops.orthogonalize(x), x * 2.0 ** -80)
    elif kind == "tiny":
        want = newton_schulz(x.double())
        got = ops.orthogonalize(x).double()
        # X0 = x 1e7 is far below fp16's smallest stored step 2^-24 / 2^11: the result is its scale, rounded to that step
        assert float((got - want).abs().max()) <= 3.5 ** 5 * 2.0 ** -35 and float(want.abs().max()) < 1e-19
    else:
        _check(ops.orthogonalize(x), x, what=kind)


def test_other_steps_and_coefficients():
    from madiff_amd import ops
    x = _grad((3, 96, 200), 4)
    for steps, coef in ((1, NS), (2, NS), (10, NS), (6, (2.0, -1.5, 0.5)), (12, (1.875, -1.25, 0.375)), (3, (1.5, -0.5, 0.0))):
        _check(ops.orthogonalize(x, steps=steps, coefficients=coef), x, steps, coef, what=(steps, coef))
    x = torch.randn(64, 64, device=DEV)
    _check(ops.orthogonalize(x, eps=1e3), x, eps=1e3)                   # eps above the norm


def test_singular_values_near_one():
    from madiff_amd import ops
    s = torch.linalg.svdvals(ops.orthogonalize(torch.randn(300, 900, device=DEV)).double().cpu())
    assert float(s.min()) > 0.6 and float(s.max()) < 1.3


def test_zero_nan_and_infinity_stay_in_their_matrix():
    from madiff_amd import ops
    x = _grad((6, 150, 300), 3)
    x[1] = 0
    x[2, 140, 7] = float("nan")
    x[4, 0, 0] = float("inf")
    y = ops.orthogonalize(x)
    keep = [0, 3, 5]
    _check(y[keep], x[keep])
    assert bool((y[1] == 0).all())
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[4]).all())


@pytest.mark.parametrize("shape", [(16, 40), (130, 300)])
def test_tiny_matrices(shape):
    """A power of two cancels exactly against the norm, which is summed in 64 bits; zeros stay zeros at the smallest eps."""
    from madiff_amd import ops
    x = _grad(shape, 21)
    want = ops.orthogonalize(x)
    assert torch.equal(ops.orthogonalize(x * 2.0 ** -70, eps=1e-30), want)
    assert torch.equal(ops.orthogonalize(x * 2.0 ** 70), want)
    assert not bool(ops.orthogonalize(torch.zeros_like(x), eps=1e-30).any())


@pytest.mark.parametrize("shape", [(8, 20, 30), (7, 130, 300)])
def test_batches_in_several_calls(shape, monkeypatch):
    """A batch too large for one call goes in several: the matrices' results do not depend on where it is cut."""
    from madiff_amd import ops
    x = _grad(shape, 31)
    _check(ops.orthogonalize(x), x)
    monkeypatch.setattr(ops, "ORTHO_MAX_BATCH", 3)
    _check(ops.orthogonalize(x), x)
    monkeypatch.setattr(ops, "ORTHO_WS_BYTES", 1)
    _check(ops.orthogonalize(x), x)


def test_offsets_past_32_bits(monkeypatch):
    """8400 matrices of 64 x 4096 in one call: 2.2e9 elements, 17.6 GB of workspace."""
    from madiff_amd import ops
    monkeypatch.setattr(ops, "ORTHO_WS_BYTES", 1 << 36)
    x = torch.randn(8400, 64, 4096, device=DEV, dtype=torch.bfloat16, generator=torch.Generator(device=DEV).manual_seed(3))
    y = ops.orthogonalize(x)
    pick = [0, 1, 8190, 8191, 8192, 8193, 8399]                # (matrix 8192 begins at element 2^31)
    _check(y[pick], x[pick])
    del x, y
    torch.cuda.empty_cache()


def test_strides_empty_streams_and_bits():
    from madiff_amd import ops
    base = _grad((4, 200, 330), 8)
    for x in (base[:, ::2, 5:300], base.mT, base[0].t(), base.permute(1, 0, 2)[:50], base[1:2].expand(3, 200, 330)):
        _check(ops.orthogonalize(x), x)
    for shape in ((0, 4, 5), (3, 0, 5), (3, 5, 0)):
        assert ops.orthogonalize(torch.empty(shape, device=DEV)).shape == torch.Size(shape)
    one = ops.orthogonalize(base)
    assert torch.equal(one, ops.orthogonalize(base))
    assert torch.equal(one[2], ops.orthogonalize(base[2]))              # a matrix does not depend on its neighbours
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.orthogonalize(base)
    here = ops.orthogonalize(base * 1.0)                                # two calls at once
    side.synchronize()
    assert torch.equal(one, other) and torch.equal(one, here)


def test_in_a_graph():
    from madiff_amd import ops
    x = _grad((2, 140, 270), 1)
    keep = x.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.orthogonalize(x)
    side.synchronize()
    graphs, outs = [], []
    for _ in range(2):                                                  # two graphs, each with its own workspace
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.orthogonalize(x))
        graphs.append(gr)
    for k in range(3):
        x.copy_(keep * (k + 1) if k != 1 else keep.flip(1))
        eager = ops.orthogonalize(x)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(eager, o) for o in outs), k


# ---------------------------------------------------------------------------------------------------- Muon
MATS = [(20, 64), (128, 80), (1, 9), (300, 40), (16, 16), (128, 640), (257, 129), (33, 1), (200, 200)]


def _flat(mats, gap=5, seed=0):
    at, layout = 3, []
    for r, c in mats:
        layout.append((at, r, c))
        at += r * c + gap
    g = torch.Generator(device=DEV).manual_seed(seed)
    return layout, [torch.randn(at, device=DEV, generator=g) * s for s in (0.05, 1e-3, 1e-3, 0.05)]


def _expect(layout, p, g, m, lr, mu, wd, nesterov, scales, gs=1.0):
    """-> float64 p, m, and the bound of |p - got| per matrix in 2-norm."""
    p, g, m = p.double().clone(), g.double() * gs, m.double().clone()
    bounds = []
    for (at, r, c), sc in zip(layout, scales):
        s = slice(at, at + r * c)
        m[s] = mu * m[s] + (1 - mu) * g[s]
        u = ((1 - mu) * g[s] + mu * m[s] if nesterov else m[s]).view(r, c)
        want, f32 = newton_schulz(u), newton_schulz(u.float()).double()
        p[s] = (1 - lr * wd) * p[s] - lr * sc * want.reshape(-1)
        # O as in the header, the rounding of U's two terms (2 u, magnified as E32 is), three roundings of the update
        bounds.append(lr * sc * (5 * float((f32 - want).norm()) * 2 + (2.0 ** -22 + LAST) * float(want.norm())) + 4 * U * float(p[s].norm()))
    return p, m, bounds


@pytest.mark.parametrize("nesterov,wd,ema,shadow,zero,gs", [(True, 0.0, 1, True, False, 1.0), (False, 0.1, 0, False, True, 0.25),
                                                            (True, 0.01, 2, True, True, 1.0)])
def test_muon_step(nesterov, wd, ema, shadow, zero, gs):
    from madiff_amd.muon import MuonPlan
    layout, (p, g, m, e) = _flat(MATS)
    scales = [0.2 * math.sqrt(max(r, c)) for _, r, c in layout]
    inside = torch.zeros(p.numel(), dtype=torch.bool, device=DEV)
    for at, r, c in layout:
        inside[at:at + r * c] = True
    sh = torch.full((p.numel(),), 7.0, device=DEV, dtype=torch.bfloat16)
    plan = MuonPlan(layout, DEV, scales)
    lr, mu = 0.02, 0.9
    for k in range(3):
        old = [v.clone() for v in (p, g, m, e)]
        want_p, want_m, bounds = _expect(layout, p, g, m, lr, mu, wd, nesterov, scales, gs)
        plan.step(p, g, m, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, ema=e if ema else None, ema_beta=0.9,
                  do_ema=ema, shadow=sh if shadow else None, grad_scale=gs, zero_grad=zero)
        for (at, r, c), b in zip(layout, bounds):
            s = slice(at, at + r * c)
            off = float((p[s].double() - want_p[s]).norm())
            assert off <= b, (k, r, c, off, b)
            record_measured(off / b, "of_bound")
        bound_m = 3 * U * (mu * old[2].double().abs() + (1 - mu) * abs(gs) * old[1].double().abs())
        assert bool(((m.double() - want_m).abs() <= bound_m)[inside].all())
        if shadow:
            assert torch.equal(sh[inside], p[inside].bfloat16()) and bool((sh[~inside] == 7).all())
        if ema == 2:
            assert torch.equal(e[inside], p[inside])
        elif ema == 1:
            w = 0.9 * old[3].double() + (1 - 0.9) * p.double()
            assert bool(((e.double() - w).abs() <= 4 * U * (old[3].abs() + p.abs()).double())[inside].all())
        assert bool((g[inside] == 0).all()) if zero else torch.equal(g, old[1])
        for now, was in zip((p, g, m, e), old):
            assert torch.equal(now[~inside], was[~inside])
        if zero:
            g.copy_(old[1])


def test_muon_single_and_many_small():
    from madiff_amd.muon import MuonPlan
    for mats in ([(64, 200)], [(3, 4)] * 200, [(1024, 130), (130, 1024), (2, 2)]):
        layout, (p, g, m, _) = _flat(mats, gap=0)
        want_p, want_m, bounds = _expect(layout, p, g, m, 0.1, 0.95, 0.0, True, [1.0] * len(mats))
        MuonPlan(layout[::-1], DEV).step(p, g, m, lr=0.1)
        for (at, r, c), b in zip(layout, bounds):
            assert float((p[at:at + r * c].double() - want_p[at:at + r * c]).norm()) <= b, (r, c)


def test_muon_in_graphs_with_device_side_ema_mode():
    from madiff_amd.muon import MuonPlan
    layout, start = _flat(MATS, seed=4)
    plan = MuonPlan(layout, DEV)
    state = torch.zeros(2, dtype=torch.int32, device=DEV)
    a, b = [v.clone() for v in start], [v.clone() for v in start]
    run = lambda v: plan.step(v[0], v[1], v[2], lr=0.05, ema=v[3], ema_beta=0.9, state=state)         # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run([v.clone() for v in start])
    side.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        run(a)
    for mode in (0, 1, 2, 1):
        state[1] = mode
        gr.replay()
        b[1].add_(0.0)
        plan.step(b[0], b[1], b[2], lr=0.05, ema=b[3], ema_beta=0.9, do_ema=mode)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, b)), mode


def test_refusals_on_the_gpu():
    from madiff_amd import ops
    from madiff_amd.muon import MuonPlan
    x = torch.randn(4, 5, device=DEV)
    for bad in (dict(steps=0), dict(steps=65), dict(eps=0.0), dict(coefficients=(4.0, -4.0, 2.5)), dict(eps=float("nan"))):
        with pytest.raises(ValueError):
            ops.orthogonalize(x, **bad)
    with pytest.raises(TypeError):
        ops.orthogonalize(x.half())
    with pytest.raises(ValueError):
        ops.orthogonalize(x[0])
    with pytest.raises(RuntimeError):
        ops.orthogonalize(x.clone().requires_grad_(True))
    plan = MuonPlan([(0, 4, 5)], DEV)
    p, g, m = (torch.zeros(20, device=DEV) for _ in range(3))
    both = torch.zeros(40, device=DEV)
    for args, kw in (((p[:19], g, m), {}), ((p, g.double(), m), {}), ((p, g, p), {}), ((p, g, m), dict(do_ema=1)),
                     ((p, g, m), dict(momentum=1.0)), ((p, g, m), dict(steps=0)), ((p.cpu(), g, m), {}),
                     ((p, g, m), dict(shadow=torch.zeros(20, device=DEV))), ((p, g, m), dict(ema=p)),
                     ((p, torch.zeros(40, device=DEV)[::2], m), {}), ((both[:20], both[10:], m), {}), ((both, both[20:], m), {}),
                     ((p, g, m), dict(do_ema=1, state=torch.zeros(2, device=DEV, dtype=torch.int32))), ((p, g, m), dict(ema=g.clone(), state=torch.zeros(1, device=DEV))),
                     ((p, g, m), dict(ema=g.clone(), state=torch.zeros(4, device=DEV, dtype=torch.int32)[::2]))):
        with pytest.raises(ValueError):
            plan.step(*args, lr=0.1, **kw)
    with pytest.raises(ValueError):
        MuonPlan([(0, 4, 5), (19, 2, 2)], DEV)
