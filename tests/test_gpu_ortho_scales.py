"""Newton-Schulz orthogonalisation of matrices whose rows differ by orders of magnitude, row by row against 64 bits.

Tolerance of one row of X (the shorter side's rows): 5 E32 + (LAST + 2^-23) |row|, E32 the row's error of the same iteration in fp32,
as test_gpu_ortho derives it for the whole matrix, plus what the stored form leaves out whatever a value's size.  An operand is hi + lo,
two fp16 numbers at 2^11 and 2^23 times the value, so a value below 2^-25 is held to a step of 2^-47, off by 2^-48 at most.  With s rows
of length l >= s and |X| <= 1.3: X itself contributes sqrt(l) 2^-48 a row, A the same a row of s numbers, A A twice |A| <= 1.7 times that,
R = b A + c A A so 4.8 + 2.1 x 3.4 + 1 = 13 times, R X as much times 1.3, and the left-out lo lo of a small value (2^-25 of its own unit
times 2^-11 of the other's) adds no more than the step once more: below (2 + 2 x 13 x 1.3) sqrt(l) 2^-48 < 36 sqrt(l) 2^-48 a step, which the
steps that follow magnify at most a = 3.4445 times each: 36 (1 + 3.4 + .. + 3.4^4) = 36 x 198 = 7130 and in all
FLOOR = 7200 sqrt(l) 2^-48."""
import math

import pytest
import torch

from conftest import record_measured
from test_gpu_ortho import LAST, newton_schulz

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rows(x):
    return x.double().square().sum(-1).sqrt()


def _check(got, x, what, times=1):
    """got against the orthogonalised x, row by row of the shorter side; `times` the bound."""
    want = newton_schulz(x.double())
    f32 = newton_schulz(x.float()).double()
    if x.shape[-2] > x.shape[-1]:
        want, f32, got = want.mT, f32.mT, got.mT
    floor = 7200 * math.sqrt(want.shape[-1]) * 2.0 ** -48
    size = _rows(want)
    bound = 5 * _rows(f32 - want) + (LAST + 2.0 ** -23) * size + floor
    off = _rows(got.double() - want)
    assert bool((off <= times * bound).all()), (what, float((off / size).max()), float((off / bound).max()))
    record_measured(float((off / bound).max()), "of_bound")


SHAPES = [(16, 128), (64, 512), (128, 160), (200, 600), (600, 200), (333, 1001), (1024, 1500), (2048, 256)]


def _graded(rows, cols, kind, seed=3):
    x = torch.randn(rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed))
    s = min(rows, cols)
    f = torch.ones(s, device=DEV)
    if kind == "one row large":
        f[s // 3] = 1e6
    elif kind == "graded":
        f = torch.logspace(-6, 0, s, device=DEV)
    else:
        f[s // 2:] = kind
    return x * f[:, None] if rows <= cols else x * f


@pytest.mark.parametrize("kind", [1e-4, 1e-5, 1e-6, "one row large", "graded"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_small_rows(rows, cols, kind):
    from madiff_amd import ops
    x = _graded(rows, cols, kind)
    _check(ops.orthogonalize(x), x, (rows, cols, kind))


@pytest.mark.parametrize("kind", [1e-5, "one row large"])
def test_small_rows_of_a_muon_update(kind):
    """p = 0 and no momentum: one step leaves p = -lr scale O(g), its rows as accurate as the orthogonalised matrix's.  Two steps that
    share one A are 1.3 to 1.8 times as far off, so twice the bound of one; the update rounds twice more (2 x 2^-24 < 2^-23)."""
    from madiff_amd.muon import MuonPlan
    mats, at = [], 0
    for r, c in SHAPES:
        mats.append((at, r, c))
        at += r * c
    g = torch.cat([_graded(r, c, kind).reshape(-1) for _, r, c in mats])
    p, m = torch.zeros_like(g), torch.zeros_like(g)
    MuonPlan(mats, DEV).step(p, g, m, lr=0.5, momentum=0.0, nesterov=False)
    for o, r, c in mats:
        x = g[o:o + r * c].view(r, c)
        _check(p[o:o + r * c].view(r, c) / -0.5, x, (r, c, kind), times=2)


# Matrices below eps start as G / eps, as small as that may be.  The bound is that of one at eps or above, relative to the result's
# 2-norm: a power of two that keeps the stored values in range changes nothing else, and the growth from there is a per step as ever.
STARTS = [(steps, coef, eps, part) for steps, coef, eps, parts in (
    (5, (3.4445, -4.7750, 2.0315), 1e-7, (0.7, 1e-2, 1e-4, 1e-6, 1e-9, 1e-13, 1e-20)), (1, (3.4445, -4.7750, 2.0315), 1e-7, (1e-8,)),
    (24, (3.4445, -4.7750, 2.0315), 1e-7, (1e-6, 1e-10)), (6, (3.4445, -4.7750, 2.0315), 1e3, (1e-12,)), (4, (1.5, -0.5, 0.0), 1e-12, (1e-5,)),
    (40, (0.5, 0.25, 0.0), 1e-7, (1e4, 1e-3))) for part in parts]


def _start(rows, cols, norm, seed=5):
    x = torch.randn(rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed), dtype=torch.float64)
    return (x * (norm / float(x.norm()))).float()


@pytest.mark.parametrize("steps,coef,eps,part", STARTS)
def test_matrices_below_eps(steps, coef, eps, part):
    from madiff_amd import ops
    for rows, cols in ((16, 128), (130, 40), (300, 500), (128, 160)):
        x = _start(rows, cols, part * eps)
        want, f32 = newton_schulz(x.double(), steps, coef, eps), newton_schulz(x, steps, coef, eps).double()
        got = ops.orthogonalize(x, steps=steps, coefficients=coef, eps=eps).double()
        bound = 5 * float((f32 - want).norm()) + (LAST + 2.0 ** -23) * float(want.norm())
        off = float((got - want).norm())
        assert off <= bound, (rows, cols, off / float(want.norm()), bound / float(want.norm()))
        record_measured(off / bound, "of_bound")
        b16 = ops.orthogonalize(x.bfloat16(), steps=steps, coefficients=coef, eps=eps).double()       # two steps in one where they pay
        want = newton_schulz(x.bfloat16().double(), steps, coef, eps)
        assert float((b16 - want).norm()) <= 2 * bound + 2.0 ** -8 * float(want.norm()), (rows, cols)


def test_matrices_of_all_sizes_together():
    """One call, one plan: what a matrix's own norm needs is not another's."""
    from madiff_amd import ops
    from madiff_amd.muon import MuonPlan
    parts = [1e6, 1e-3, 1.5, 1e-9, 0.0, 1e-16]
    for rows, cols in ((200, 300), (24, 50)):
        x = torch.stack([_start(rows, cols, q * 1e-7, seed=k) if q else torch.zeros(rows, cols, device=DEV) for k, q in enumerate(parts)])
        got = ops.orthogonalize(x).double()
        mats = [(k * rows * cols, rows, cols) for k in range(len(parts))]
        p, m, g = torch.zeros(x.numel(), device=DEV), torch.zeros(x.numel(), device=DEV), x.reshape(-1).clone()
        MuonPlan(mats, DEV).step(p, g, m, lr=0.5, momentum=0.0, nesterov=False)
        p = p.view_as(x).double() / -0.5
        for k, q in enumerate(parts):
            want, f32 = newton_schulz(x[k].double()), newton_schulz(x[k]).double()
            bound = 5 * float((f32 - want).norm()) + (LAST + 2.0 ** -23) * float(want.norm())
            assert float((got[k] - want).norm()) <= bound, (rows, q, float((got[k] - want).norm() / want.norm()))
            assert float((p[k] - want).norm()) <= 2 * bound, (rows, q, float((p[k] - want).norm() / want.norm()))


@pytest.mark.parametrize("rows,cols", [(64, 512), (200, 600), (600, 200)])
def test_small_columns(rows, cols):
    """Columns of X (the longer side) keep their bits as rows do: sqrt(s) numbers of a column instead of sqrt(l) of a row."""
    from madiff_amd import ops
    x = torch.randn(rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(8))
    l = max(rows, cols)
    f = torch.ones(l, device=DEV)
    f[l // 2:] = 1e-6
    x = x * f if rows < cols else x * f[:, None]
    want, f32, got = newton_schulz(x.double()), newton_schulz(x).double(), ops.orthogonalize(x).double()
    if rows < cols:
        want, f32, got = want.mT, f32.mT, got.mT
    bound = 5 * _rows(f32 - want) + (LAST + 2.0 ** -23) * _rows(want) + 7200 * math.sqrt(min(rows, cols)) * 2.0 ** -48
    off = _rows(got - want)
    assert bool((off <= bound).all()), float((off / bound).max())


@pytest.mark.parametrize("batch,rows,cols", [(64, 128, 640), (64, 200, 600), (70, 600, 200)])
def test_the_form_does_not_depend_on_the_batch(batch, rows, cols, monkeypatch):
    """bf16 results may take two steps in one; whether they do goes by a matrix's own sides.  No reduction is cut at these sizes, so a
    matrix has the same bits alone, in a batch, and in the shorter call at a batch's end."""
    from madiff_amd import ops
    x = torch.randn(batch, rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)).bfloat16()
    whole = ops.orthogonalize(x)
    assert torch.equal(whole[5], ops.orthogonalize(x[5]))
    monkeypatch.setattr(ops, "ORTHO_MAX_BATCH", batch - 1)
    assert torch.equal(whole, ops.orthogonalize(x))


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_cut_reductions_in_batches(t):
    """333 x 1001 is cut into 5, 4, 3 and 1 parts in batches of 1, 2, 4 and 12: other bits, the same bound (twice for two steps in one)."""
    from madiff_amd import ops
    x = torch.randn(12, 333, 1001, device=DEV, generator=torch.Generator(device=DEV).manual_seed(6)).to(t)
    want, f32 = newton_schulz(x.double()), newton_schulz(x.float()).double()
    n = lambda v: v.square().sum((-2, -1)).sqrt()                                                    # noqa: E731
    last, times = (2.0 ** -23, 1) if t == torch.float32 else (2.0 ** -8, 2)
    bound = times * (5 * n(f32 - want) + LAST * n(want)) + last * n(want)
    for batch in (1, 2, 4, 12):
        got = torch.cat([ops.orthogonalize(p) for p in x.split(batch)]).double()
        assert bool((n(got - want) <= bound).all()), (batch, float((n(got - want) / bound).max()))


# up to 32 rows: another kernel for every range of columns, fp32 throughout
FEW = [(1, 1), (2, 2), (16, 16), (3, 31), (16, 32), (16, 33), (32, 16), (9, 127), (16, 128), (16, 129), (200, 13), (15, 512), (16, 513), (777, 16),
       (2, 2047), (16, 2048), (16, 2049), (17, 17), (32, 32), (20, 64), (32, 65), (64, 31), (25, 128), (32, 129), (17, 256), (32, 257), (300, 20),
       (31, 512), (32, 513), (513, 32), (1000, 18), (32, 1024), (32, 1025)]


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols", FEW)
def test_few_rows(rows, cols, t):
    """Three matrices in a batch and each alone, against 64 bits (the bound of test_gpu_ortho), and the same bits in both."""
    from madiff_amd import ops
    x = torch.randn(3, rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(rows + 40 * cols)).to(t)
    got = ops.orthogonalize(x)
    want, f32 = newton_schulz(x.double()), newton_schulz(x.float()).double()
    n = lambda v: v.double().square().sum((-2, -1)).sqrt()                                           # noqa: E731
    bound = 5 * n(f32 - want) + (LAST + (2.0 ** -23 if t == torch.float32 else 2.0 ** -8)) * n(want)
    off = n(got.double() - want)
    assert bool((off <= bound).all()), float((off / bound).max())
    if min(rows, cols) <= 16 and max(rows, cols) <= 2048 or min(rows, cols) <= 32 and max(rows, cols) <= 512:
        assert all(torch.equal(got[k], ops.orthogonalize(x[k])) for k in range(3))


@pytest.mark.parametrize("rows,cols", [(2, 64), (5, 300), (8, 128), (128, 8), (8, 512), (12, 2000), (20, 1000), (28, 64), (32, 128)])
def test_few_rows_are_as_near_as_in_fp32(rows, cols):
    """The error of 64 matrices on average against that of the same iteration in fp32 products.  Both round operands to 24 bits and sum in
    fp32, ours in more and shorter sums and with fewer roundings between the products, so ours is no larger but for the spread of
    an average of 64, some tenth: 1.25 times at most.  Operands of 22 bits make it 1.3 to 1.7."""
    from madiff_amd import ops
    x = torch.randn(64, rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(11))
    want = newton_schulz(x.double())
    n = lambda v: float((v.double() - want).square().sum((-2, -1)).sqrt().mean())                    # noqa: E731
    ours, plain = n(ops.orthogonalize(x)), n(newton_schulz(x))
    assert ours <= 1.25 * plain, (ours, plain, ours / plain)
    record_measured(ours / plain, "of_fp32")


@pytest.mark.parametrize("rows,cols", [(16, 128), (10, 2000), (32, 500), (700, 24)])
def test_few_rows_of_any_size(rows, cols):
    """fp32 keeps its bits at every size: rows 1e-12 of the others, without the stored form's step in the bound."""
    from madiff_amd import ops
    x = _graded(rows, cols, 1e-12)
    want, f32, got = newton_schulz(x.double()), newton_schulz(x).double(), ops.orthogonalize(x).double()
    if rows > cols:
        want, f32, got = want.mT, f32.mT, got.mT
    bound = 5 * _rows(f32 - want) + (LAST + 2.0 ** -23) * _rows(want)
    assert bool((_rows(got - want) <= bound).all()), float((_rows(got - want) / bound).max())


@pytest.mark.parametrize("rows,cols", [(2, 30), (16, 40), (12, 1500), (30, 100), (600, 32), (20, 900)])
def test_few_rows_zero_nan_and_infinity(rows, cols):
    from madiff_amd import ops
    x = torch.randn(6, rows, cols, device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
    whole = ops.orthogonalize(x)
    y = x.clone()
    y[1] = 0
    y[2, rows - 1, 7] = float("nan")
    y[4, 0, cols - 1] = float("-inf")
    y[5] *= 2.0 ** 90                                         # squares beyond fp32: the same bits, a power of two cancels
    got = ops.orthogonalize(y)
    assert torch.equal(got[[0, 3, 5]], whole[[0, 3, 5]]) and bool((got[1] == 0).all())
    assert bool(torch.isnan(got[2]).all()) and bool(torch.isnan(got[4]).all())
    assert not bool(ops.orthogonalize(torch.zeros_like(x), eps=1e-30).any())
    inner = x.clone()                                         # in place through the C entry, as its comment allows
    import ctypes
    from madiff_amd import lib
    need = ctypes.c_long()
    lib.call("madiff_ortho_ws", 6, rows, cols, ctypes.byref(need))
    assert need.value == 0
    lib.call("madiff_orthogonalize", lib.F32, inner.data_ptr(), inner.data_ptr(), 6, rows, cols, 5, *ops.NEWTON_SCHULZ, 1e-7, None, 0,
             torch.cuda.current_stream().cuda_stream)
    assert torch.equal(inner, whole)
