"""What ops.layer_norm and its C entry points refuse, before anything is launched (no GPU needed)."""
import pytest
import torch


def test_python_refusals():
    from madiff_amd import ops
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros(3, 4))                    # not on the GPU
    with pytest.raises(ValueError):
        ops.layer_norm([1.0, 2.0])


def test_c_refusals():
    from madiff_amd import lib
    f, b, n = lib._lib.madiff_layer_norm_fwd, lib._lib.madiff_layer_norm_bwd, lib._lib.madiff_layer_norm_groups
    p = 1 << 20                                              # never read: every call below is refused
    ok = [1, p, 64, p, 64, p, p, p, p, 5, 64, 64, 1e-5, None]
    for at, bad in ((0, 2), (0, -1), (2, 63), (4, 63), (9, -1), (10, 0), (10, 32769), (11, 63), (12, -1e-5), (12, float("nan")),
                    (7, None), (8, None), (1, None), (3, None)):
        args = list(ok)
        args[at] = bad
        assert f(*args) == -1, (at, bad)
    groups = n(1, 5, 64)
    assert groups >= 1 and n(1, -1, 64) == -1 and n(1, 5, 0) == -1 and n(3, 5, 64) == -1 and n(0, 5, 32769) == -1
    ok = [1, p, 64, p, 64, p, p, p, p, 64, p, p, 0, p, 2 * 64 * groups, 5, 64, 64, None]
    for at, bad in ((0, 7), (2, 63), (4, 10), (9, 63), (13, None), (14, 2 * 64 * groups - 1), (15, -1), (16, 0), (16, 32769),
                    (17, 63), (1, None), (3, None), (6, None), (7, None)):
        args = list(ok)
        args[at] = bad
        assert b(*args) == -1, (at, bad)
