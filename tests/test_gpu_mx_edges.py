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
