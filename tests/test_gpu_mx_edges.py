"""Microscaled rows on the GPU: values, layouts and calls at the edges of what the operators take."""
import numpy as np
import pytest
import torch

from lidar_ai_solution_amd import capi, graphs
from tests import mx_reference as R
from tests.test_gpu_mx import DEV, _mx, conv_case, rows

pytestmark = pytest.mark.gpu


def test_engine_refuses_weights_that_are_not_finite():
    from lidar_ai_solution_amd.scn import Engine
    g, _ = graphs.unet_scn(seed=3, weight_std=0.08)
    node = next(n for n in g.nodes if n.op_type == "SparseConvolution")
    node.attrs["precision"] = "mxfp4"
    w = g.initializers[node.inputs[1]]
    w[w.shape[0] - 1, 0, 0, 0, 0] = np.inf
    with pytest.raises(RuntimeError, match="finite"):
        Engine.from_graph(g, "mxfp4")
    Engine.from_graph(g, "fp16")                                          # where the mark is ignored


@pytest.mark.parametrize("cin", [16, 64, 160])
def test_convolution_with_the_largest_weights(cin):
    """Finite weights of every fp16 magnitude: rows without a neighbour stay finite."""
    mx = _mx()
    rng = np.random.default_rng(cin)
    rb, table, n_out, _, _, _ = conv_case(rng, 300, (9, 24, 21), cin, 32, (3, 3, 3), (1, 1, 1), (1, 1, 1), True)
    w = np.ldexp(rng.uniform(0.5, 1, (32, 3, 3, 3, cin)) * rng.choice([-1, 1], (32, 3, 3, 3, cin)), rng.integers(-24, 17, (32, 27, 1)).reshape(32, 3, 3, 3, 1))
    w = np.clip(w, -65504, 65504).astype(np.float16)
    x = (rows(rng, 300, cin) * np.float16(2.0 ** -8)).astype(np.float16)
    y, mag = R.convolution(R.fake(x), R.fake(w.reshape(32 * 27, cin)).reshape(32, 27, cin), None, table)
    got = mx.Conv(w).forward(mx.quantize_rows(torch.from_numpy(x).to(DEV)), rb, n_out).double().cpu().numpy()
    R.within(got, y, R.tolerance(y, mag, 27 * cin, 2.0 ** -11))
    assert np.isfinite(y).all() and not np.isnan(got).any()


# one row, the few-row kernel, the product's own quantisation, tiles of every size, k in parts
@pytest.mark.parametrize("m, n, k", [(1, 40, 100), (4, 40, 100), (40, 70, 100), (200, 130, 300), (300, 64, 64), (2050, 2061, 600), (4111, 2300, 300),
                                     (70, 70, 4000)])
@pytest.mark.parametrize("x", ["mx", "fp16"])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
def test_product_relu_keeps_nan(m, n, k, x, out_dtype):
    mx = _mx()
    rng = np.random.default_rng(m + n)
    wh, ah = rng.standard_normal((n, k)).astype(np.float16), rng.standard_normal((m, k)).astype(np.float16)
    wh[5, k - 1], wh[n - 1, 0] = np.inf, np.nan
    if m > 1:
        ah[1, k // 2] = -np.inf
    w, a = mx.quantize_rows(torch.from_numpy(wh).to(DEV)), torch.from_numpy(ah).to(DEV)
    a = mx.quantize_rows(a) if x == "mx" else a
    res = torch.full((m, n), -1.0, dtype=torch.float16, device=DEV)
    want = np.zeros((m, n), bool)
    want[:, [5, n - 1]] = True
    want[1:2] = True
    for kw in (dict(relu=True), dict(relu_after_add=True), dict(relu=True, residual=res, relu_after_add=True), dict(relu=True, residual=res)):
        got = mx.product(a, w, out_dtype=out_dtype, **kw).double().cpu().numpy()
        assert np.array_equal(np.isnan(got), want), kw
        floor = -1.0 if "residual" in kw and "relu_after_add" not in kw else 0.0
        assert (got[~want] >= floor).all() and (got[~want] == floor).any(), kw
