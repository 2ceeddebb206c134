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


def test_workgroups_cover_the_rows_as_the_kernel_takes_them():
    """Backward's workgroups take four rows a group of lanes, up to 1024 x 256 lanes in all: 8 .. 64 lanes a row while 16 elements a lane
    hold it (a multiple of 16 bytes each), then workgroups of 128 .. 1024 lanes.  A grid for fewer lanes a row than the kernel uses leaves
    half of it to a second pass over the rows."""
    from madiff_amd import lib
    n = lib._lib.madiff_layer_norm_groups
    for dt, per in ((1, 8), (0, 4)):
        for C in list(range(1, 1100)) + [2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 32768]:
            v = -(-C // per)
            lanes = next((k for k in (8, 16, 32, 64) if v <= k), None) or next(k for k in (64, 128, 256, 512, 1024, 2048) if v <= k * 16 // per)
            lanes = min(lanes, 1024)
            block, rows_a_group = max(lanes, 256) if lanes <= 64 else lanes, 256 // lanes if lanes <= 64 else 1
            for rows in (1, 64, 1000, 10 ** 7):
                want = max(1, min(-(-rows // (4 * rows_a_group)), 1024 * 256 // block))
                assert n(dt, rows, C) == want, (dt, rows, C, n(dt, rows, C), want)
