"""What ops.orthogonalize, muon.MuonPlan and their C entry points refuse before anything is launched, and the layout of a plan
(no GPU needed)."""
import ctypes as C

import pytest
import torch


def test_python_refusals():
    from madiff_amd import ops
    from madiff_amd.muon import MuonPlan
    with pytest.raises(ValueError):
        ops.orthogonalize(torch.zeros(3, 4))
    for mats, kw in (([], {}), ([(0, 0, 4)], {}), ([(-1, 2, 2)], {}), ([(0, 3, 3), (8, 2, 2)], {}), ([(0, 2, 2)], dict(scales=[1, 2])),
                     ([(0, 2, 2)], dict(device="cpu"))):
        with pytest.raises(ValueError):
            MuonPlan(mats, **kw)


def test_c_refusals():
    from madiff_amd import lib
    L = lib._lib
    ns = (3.4445, -4.7750, 2.0315)
    assert L.madiff_ortho_check(5, *ns, 1e-7) == 0
    for bad in ((0, *ns, 1e-7), (65, *ns, 1e-7), (5, *ns, 0.0), (5, *ns, float("nan")), (5, float("nan"), 0.0, 0.0, 1e-7),
                (5, 16.0, 0.0, 0.0, 1e-7), (5, 4.0, -4.0, 2.5, 1e-7)):
        assert L.madiff_ortho_check(*bad) == -1, bad
    need = C.c_long()
    assert L.madiff_ortho_ws(3, 100, 800, C.byref(need)) == 0 and need.value > 0 and need.value % 256 == 0
    assert L.madiff_ortho_ws(3, 50, 200, C.byref(need)) == 0 and need.value == 0      # whole in LDS: no workspace
    for bad in ((-1, 4, 4), (1, 0, 4), (1, 4, 0), (1, 16385, 16385), (1, 2, (1 << 22) + 1), (1 << 30, 128, 128)):
        assert L.madiff_ortho_ws(*bad, C.byref(need)) == -1, bad
    L.madiff_ortho_ws(3, 100, 800, C.byref(need))
    p = 1 << 20
    ok = [1, p, p, 3, 100, 800, 5, *ns, 1e-7, p, need.value, None]
    for at, bad in ((0, 2), (1, None), (2, None), (3, -1), (4, 0), (5, 0), (6, 0), (10, 0.0), (11, None), (11, p + 16), (12, need.value - 1)):
        args = list(ok)
        args[at] = bad
        assert L.madiff_orthogonalize(*args) == -1, (at, bad)


def _plan(mats):
    from madiff_amd import lib
    n = len(mats)
    at, rows, cols = (C.c_long * n)(*[m[0] for m in mats]), (C.c_int * n)(*[m[1] for m in mats]), (C.c_int * n)(*[m[2] for m in mats])
    need = C.c_long()
    rc = lib._lib.madiff_muon_plan(n, at, rows, cols, None, None, 0, C.byref(need))
    if rc:
        return rc, None
    blob = torch.full((need.value + 64,), 7, dtype=torch.uint8)
    assert lib._lib.madiff_muon_plan(n, at, rows, cols, None, blob.data_ptr(), need.value - 1, C.byref(need)) == -1
    rc = lib._lib.madiff_muon_plan(n, at, rows, cols, None, blob.data_ptr(), need.value, C.byref(need))
    assert bool((blob[need.value:] == 7).all())                         # not a byte behind what it asked for
    return rc, blob


def test_plan_layout_and_refusals():
    from madiff_amd import lib
    L = lib._lib
    assert _plan([(0, 16385, 16385)])[0] == -1 and _plan([(-4, 2, 2)])[0] == -1 and _plan([(0, 0, 2)])[0] == -1
    mats = [(0, 20, 300), (6000, 1, 1), (6004, 700, 129)]
    rc, blob = _plan(mats)
    assert rc == 0
    ws, el = C.c_long(), C.c_long()
    assert L.madiff_muon_plan_ws(blob.data_ptr(), C.byref(ws), C.byref(el)) == 0
    assert el.value == 6004 + 700 * 129 and ws.value % 256 == 0
    # every chunk, and every tile on and above the diagonal / of the long side, exactly once
    w = blob[:256].view(torch.int64).tolist()
    i32 = lambda lo, n: blob[lo:lo + 4 * n].view(torch.int32).tolist()                                # noqa: E731
    n_mats, chunks, areas, *rest = i32(40, 12)
    shapes, works, counters = rest[:3], rest[3:6], rest[6]
    at_mats, at_chunks, at_areas = w[11:14]
    at_works = w[14:17]
    up = lambda v, d: -(-v // d)                                                                      # noqa: E731
    sides = [(32 * up(min(r, c), 32), 32 * up(max(r, c), 32)) for _, r, c in mats]
    ck = i32(at_chunks, 2 * chunks)
    assert n_mats == 3 and list(zip(ck[::2], ck[1::2])) == [(i, k) for i, (_, r, c) in enumerate(mats) for k in range(up(r * c, 16384))]
    ar = i32(at_areas, 4 * areas)
    assert list(zip(ar[::4], ar[1::4], ar[2::4])) == [(i, a, b) for i, (s, l) in enumerate(sides) for a in range(up(s, 64))
                                                      for b in range(up(l, 64))]
    for kind in range(3):
        b = (64, 128)[shapes[kind]]
        want = {(i, x, y) for i, (s, l) in enumerate(sides) for x in range(up(s, b)) for y in (range(up(l, b)) if kind == 2 else range(x, up(s, b)))}
        t = i32(at_works[kind], 8 * works[kind])
        got = [t[8 * k:8 * k + 6] for k in range(works[kind]) if t[8 * k] != -1]          # (-1: filler)
        parts, slots = {}, set()
        for m, x, y, part, n, slot in got:
            assert (part, n) not in parts.setdefault((m, x, y), []) and 0 <= part < n
            parts[(m, x, y)].append((part, n))
            if n > 1:
                assert slot + part not in slots                          # no two parts share a slot
                slots.add(slot + part)
        assert set(parts) == want and all(len(v) == v[0][1] for v in parts.values())
        # partial sums, then a counter for every slot
        assert (max(slots, default=-1) + 1) * b * b * 4 + w[4] + 4 * counters <= ws.value and max(slots, default=-1) < counters + (not slots)
    bad = blob.clone()
    bad[0] ^= 1
    assert L.madiff_muon_plan_ws(bad.data_ptr(), C.byref(ws), C.byref(el)) == -1
    p, f = 1 << 20, blob.data_ptr()
    ok = [f, p, p, p, p, p, None, el.value, 0.1, 0.9, 0.1, 1, 1.0, 1.0, 0, 1, 0.9, 0.1, None, 5, 3.4445, -4.7750, 2.0315, 1e-7, p, ws.value, None]
    for at, v in ((0, None), (0, bad.data_ptr()), (1, None), (2, None), (3, None), (4, None), (5, None), (7, el.value - 1), (9, 1.0), (9, -0.1),
                  (9, float("nan")), (15, 3), (15, -1), (19, 0), (23, 0.0), (24, None), (24, p + 8), (25, ws.value - 1)):
        args = list(ok)
        args[at] = v
        assert L.madiff_muon_step(*args) == -1, (at, v)
    args = list(ok)                                  # an EMA mode without a buffer, with and without a mode on the device
    args[5] = None
    assert L.madiff_muon_step(*args) == -1
    args[18] = p
    assert L.madiff_muon_step(*args) == -1


def test_smallest_eps_and_largest_offset():
    """2^11 / eps has to stay an fp32 number (a zero matrix would be NaN), an offset plus its matrix a 64-bit one."""
    from madiff_amd import lib
    L = lib._lib
    assert L.madiff_ortho_check(5, 3.4445, -4.7750, 2.0315, 1e-30) == 0
    for eps in (9e-31, 1e-38, 1e-45, 1e30):
        assert L.madiff_ortho_check(5, 3.4445, -4.7750, 2.0315, eps) == -1, eps
    need = C.c_long()
    one = lambda at: L.madiff_muon_plan(1, (C.c_long * 1)(at), (C.c_int * 1)(4), (C.c_int * 1)(5), None, None, 0, C.byref(need))  # noqa: E731
    assert one(2 ** 63 - 21) == 0 and one(2 ** 63 - 20) == -1 and one(2 ** 63 - 1) == -1
