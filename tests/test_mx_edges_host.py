"""Microscaled rows without a GPU: calls that have to be refused before anything is launched."""
import ctypes as C

import numpy as np
import pytest

from lidar_ai_solution_amd import capi


@pytest.mark.parametrize("shape, at, where", [((4, 3, 3, 3, 64), (1, 2, 0, 1, 40), "channel 1, kernel offset 19, input channels 32 to 63"),
                                              ((40, 1, 1, 1, 5), (39, 0, 0, 0, 4), "channel 39, kernel offset 0, input channels 0 to 4"),
                                              ((16, 1, 3, 1, 160), (0, 0, 1, 0, 159), "channel 0, kernel offset 1, input channels 128 to 159")])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_convolution_refuses_weights_that_are_not_finite(shape, at, where, bad):
    """A block that is not finite would make a NaN of rows without a neighbour at its offset, too."""
    w = np.ones(shape, np.float16)
    w[at] = bad
    assert not capi.lib().scn_conv_create(w.ctypes.data_as(C.c_void_p), capi.i5(*shape), None, None, capi.PRECISION_MXFP4)
    text = capi.lib().scn_last_error().decode()
    assert "finite" in text and where in text


GOOD = 1 << 20   # an aligned address that no refused call reads


def _product_io(**over):
    """40 x 320 rows times 24 weight rows, every array far from the others: rows at 1 MB, weights at 2, and so on."""
    io = capi.MxProductIO()
    base = dict(a_dev=GOOD, a_dtype=capi.DTYPE_MXFP4, a_ld=176, a_scales_dev=GOOD + 160, a_scales_ld=176, b_codes_dev=2 * GOOD, b_codes_ld=176,
                b_scales_dev=2 * GOOD + 160, b_scales_ld=176, m=40, n=24, k=320, bias_dev=3 * GOOD, bias_dtype=capi.DTYPE_FP32,
                res_dev=4 * GOOD, res_dtype=capi.DTYPE_FP16, res_ld=30, out_dev=5 * GOOD, out_dtype=capi.DTYPE_FP16, out_ld=30,
                m_dev=6 * GOOD, workspace_dev=7 * GOOD, workspace_bytes=7040)
    base.update(over)
    for key, v in base.items():
        setattr(io, key, v)
    return io


FP16_ROWS = dict(a_dtype=capi.DTYPE_FP16, a_ld=320)
OVER = [dict(out_dev=GOOD + 39 * 176 + 158),                              # the last row's last codes
        dict(out_dev=GOOD - 39 * 60 - 46),                                # the last output row, the first codes
        dict(out_dev=GOOD + 160 + 10), dict(out_dev=2 * GOOD + 23 * 176), dict(out_dev=2 * GOOD + 23 * 176 + 166),
        dict(out_dev=3 * GOOD + 94), dict(out_dev=4 * GOOD + 2), dict(out_dev=4 * GOOD + 60), dict(out_dev=4 * GOOD - 60),
        dict(out_dev=4 * GOOD + 36),                                      # columns that run into the next row's
        dict(out_dev=6 * GOOD), dict(out_dev=GOOD + 100, out_ld=88),      # (stride of the rows, columns of them)
        dict(FP16_ROWS, out_dev=GOOD + 2), dict(FP16_ROWS, out_dev=GOOD + 39 * 640 + 638), dict(FP16_ROWS, out_dev=GOOD, m=3),
        dict(FP16_ROWS, workspace_dev=GOOD), dict(FP16_ROWS, workspace_dev=GOOD + 16), dict(FP16_ROWS, workspace_dev=2 * GOOD - 16), dict(FP16_ROWS, workspace_dev=3 * GOOD + 80),
        dict(FP16_ROWS, workspace_dev=4 * GOOD + 48), dict(FP16_ROWS, workspace_dev=5 * GOOD - 7024), dict(FP16_ROWS, workspace_dev=6 * GOOD - 16)]


@pytest.mark.parametrize("over", OVER)
def test_product_refuses_overlaps(over):
    assert capi.lib().scn_mx_product(C.byref(_product_io(**over)), None) == 1
    assert b"overlap" in capi.lib().scn_last_error()


@pytest.mark.parametrize("codes, scales, codes_ld, scales_ld", [(GOOD, 3 * GOOD, 32, 4), (GOOD + 4 * 128 + 112, 3 * GOOD, 32, 4),
                                                                (3 * GOOD, GOOD + 124, 32, 4), (3 * GOOD, GOOD - 4, 32, 4), (3 * GOOD, 3 * GOOD + 28, 48, 48),
                                                                (3 * GOOD, 3 * GOOD + 4 * 32, 32, 4), (GOOD + 128, 3 * GOOD, 144, 4)])
def test_quantize_and_dequantize_refuse_overlaps(codes, scales, codes_ld, scales_ld):
    """Rows of 64 fp16 channels, 5 of them at 1 MB (in the last case every 144 bytes), over their codes or scales."""
    ld = 72 if codes_ld == 144 else 64
    L = capi.lib()
    if codes_ld == 144:
        codes -= 16                                                       # beside the channels it would be allowed
    assert L.scn_mx_quantize_rows(GOOD, capi.DTYPE_FP16, 64, ld, 0.0, 0, codes, codes_ld, scales, scales_ld, 5, None, None) == 1
    assert b"overlap" in L.scn_last_error()
    if codes < 3 * GOOD or scales < 3 * GOOD:
        assert L.scn_mx_dequantize_rows(codes, codes_ld, scales, scales_ld, 64, GOOD, capi.DTYPE_FP16, ld, 5, None, None) == 1
        assert b"overlap" in L.scn_last_error()


def test_overlap_of_runs_of_rows():
    """Against sets of bytes; the answer for two different strides may only err towards yes."""
    from lidar_ai_solution_amd.mx import _overlap
    rng = np.random.default_rng(1)

    def bytes_of(s):
        return {s[0] + r * s[3] + i for r in range(s[1]) for i in range(s[2])}

    seen = [0, 0]
    for _ in range(20000):
        la = int(rng.integers(1, 12))
        lb = la if rng.random() < 0.7 else int(rng.integers(1, 12))
        a = (100, int(rng.integers(0, 5)), int(rng.integers(1, la + 1)), la)
        b = (int(rng.integers(60, 140)), int(rng.integers(0, 5)), int(rng.integers(1, lb + 1)), lb)
        got, want = _overlap(a, b), bool(bytes_of(a) & bytes_of(b))
        assert got == want or (got and la != lb and a[1] > 1 and b[1] > 1), (a, b)
        assert _overlap(b, a) == got, (a, b)
        seen[want] += 1
    assert min(seen) > 2000


def test_rows_live_on_a_gpu():
    from lidar_ai_solution_amd import mx
    with pytest.raises(ValueError, match="GPU"):
        mx.MxRows.empty(4, 64, "cpu")


def test_rulebook_refuses_a_stream_of_another_device():
    """(The device is checked before anything else, so that a stand-in for a stream does.)"""
    from types import SimpleNamespace

    from lidar_ai_solution_amd import mx
    rb = mx.Rulebook.__new__(mx.Rulebook)
    rb.index = 0
    there = SimpleNamespace(device_index=1, cuda_stream=0)
    with pytest.raises(ValueError, match="stream of cuda:1"):
        rb.build_subm(None, (9, 9, 9), (3, 3, 3), stream=there)
    with pytest.raises(ValueError, match="stream of cuda:1"):
        rb.build_sparse(None, (9, 9, 9), (3, 3, 3), (2, 2, 2), (1, 1, 1), stream=there)


def test_assembly_that_writes_m0_says_so():
    """The compiler keeps values of its own in m0 (loads to LDS, indexed registers); a statement that writes it names it."""
    import glob
    import os
    import re
    src = os.path.join(os.path.dirname(os.path.abspath(capi.__file__)), "csrc")
    found = 0
    for path in glob.glob(os.path.join(src, "*.h*")):
        with open(path) as f:
            text = f.read()
        for statement in re.findall(r"\basm\b[^;]*?\((?:[^;\"]|\"[^\"]*\")*\);", text):
            if re.search(r"\bs_\w+\s+m0\b", statement):
                found += 1
                assert re.search(r":[^:]*\"m0\"[^:]*\);$", statement), (path, statement)
    assert found >= 4


def test_rows_quantised_in_the_products_launch_fit_it():
    """64 rows of more than 128 channels are 512 threads: the last row counts below 2^29 would make 2^32."""
    L = capi.lib()
    assert L.scn_mx_product_workspace((1 << 29) - 65, 64, 256) == 0
    for m in ((1 << 29) - 64, (1 << 29) - 1, 1 << 29):
        assert L.scn_mx_product_workspace(m, 64, 256) == m * L.scn_mx_row_bytes(256)
