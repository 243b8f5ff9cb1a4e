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


def test_arrays_side_by_side_in_one_buffer():
    """Columns of one buffer: rows, their codes and scales, the output; nothing overlaps, so nothing is refused."""
    mx = _mx()
    rng = np.random.default_rng(1)
    n = 70
    buf = torch.zeros((n, 512), dtype=torch.uint8, device=DEV)
    x = buf[:, :192].view(torch.float16)                                  # 96 channels
    x.copy_(torch.from_numpy(rows(rng, n, 96)))
    q = mx.quantize_rows(x, out=mx.MxRows(buf[:, 192:240], buf[:, 240:244], 96))
    xv = R.fake(x.cpu().numpy())
    wh = rows(rng, 33, 96)
    w, wv = mx.quantize_rows(torch.from_numpy(wh).to(DEV)), R.fake(wh)
    y, mag = R.product(xv, wv)
    for a in (q, x):
        out = mx.product(a, w, out=buf[:, 256:322].view(torch.float16))
        R.within(out.double().cpu().numpy(), y, R.tolerance(y, mag, 96, 2.0 ** -11))
    back = mx.dequantize_rows(q, out=buf[:, 320:512].view(torch.float16))
    assert np.array_equal(back.cpu().numpy(), xv.astype(np.float16))


def test_convolution_refuses_overlaps():
    mx = _mx()
    rng = np.random.default_rng(2)
    rb, table, n_out, conv, wv, b = conv_case(rng, 200, (9, 24, 21), 64, 64, (3, 3, 3), (1, 1, 1), (1, 1, 1), True)
    x = rows(rng, 200, 64)
    buf = torch.zeros((400, 384), dtype=torch.uint8, device=DEV)
    q = mx.quantize_rows(torch.from_numpy(x).to(DEV), out=mx.MxRows(buf[:200, :32], buf[:200, 32:36], 64))

    def half(first_row, column):
        return buf[first_row:first_row + 200, column:column + 128].view(torch.float16)

    def mx_out(first_row, column):
        return mx.MxRows(buf[first_row:first_row + 200, column:column + 32], buf[first_row:first_row + 200, column + 32:column + 36], 64)

    for out in (half(0, 16), half(199, 0), mx_out(0, 16), mx_out(199, 0), buf.flatten()[:200 * 128].view(200, 128).view(torch.float16)):
        with pytest.raises(RuntimeError, match="overlap"):
            conv.forward(q, rb, n_out, out=out)
    for res in (half(0, 80), half(1, 64), half(199, 64)):
        with pytest.raises(RuntimeError, match="overlap"):
            conv.forward(q, rb, n_out, out=half(0, 64), residual=res)
    with pytest.raises(RuntimeError, match="overlap"):
        conv.forward(q, rb, n_out, out=mx_out(0, 64), residual=half(0, 64))
    assert not buf[:, 48:].any() and not buf[200:].any()
    # beside each other, behind each other, and over the residual
    y, mag = R.convolution(R.fake(x), wv, b, table)
    tol = R.tolerance(y, mag, 27 * 64, 2.0 ** -11)
    for out in (half(0, 48), half(200, 0), half(200, 256)):
        R.within(conv.forward(q, rb, n_out, out=out).double().cpu().numpy(), y, tol)
    res = rng.standard_normal((200, 64)).astype(np.float16)
    half(0, 256).copy_(torch.from_numpy(res))
    want = y + res
    tol = tol + R.tolerance(want, 0 * mag, 0, 2.0 ** -11)
    for out in (half(0, 128), half(0, 256)):
        R.within(conv.forward(q, rb, n_out, out=out, residual=half(0, 256)).double().cpu().numpy(), want, tol)


@pytest.mark.parametrize("m", [3, 60, 300])
def test_product_refuses_overlaps_from_python(m):
    mx = _mx()
    w = mx.quantize_rows(torch.randn(24, 320, device=DEV))
    buf = torch.zeros((m + 2, 320), dtype=torch.float16, device=DEV)
    a, res = buf[1:m + 1], torch.zeros((m + 1, 24), dtype=torch.float16, device=DEV)
    q = mx.MxRows.empty(m, 320, DEV)
    q._buffer.zero_()
    for x, out in ((a, buf[:m, :24]), (a, buf[2:, 296:]), (q, q._buffer[:48 * m].view(m, 48).view(torch.float16))):
        with pytest.raises(RuntimeError, match="overlap"):
            mx.product(x, w, out=out)
    with pytest.raises(RuntimeError, match="overlap"):
        mx.product(a, w, out=res[1:], residual=res[:m])
    if m > 16:
        with pytest.raises(RuntimeError, match="overlap"):
            mx.product(a, w, workspace=buf.view(-1).view(torch.uint8))
    with pytest.raises(RuntimeError, match="overlap"):
        mx.quantize_rows(a, out=mx.MxRows(buf[:m].view(torch.uint8)[:, :160], buf[:m].view(torch.uint8)[:, 160:172], 320))
    narrow = mx.MxRows(q.codes[:, :16], q.scales[:, :4], 32)
    with pytest.raises(RuntimeError, match="overlap"):
        mx.dequantize_rows(narrow, out=q._buffer[8:8 + 64 * m].view(m, 64).view(torch.float16))
    assert not buf.any() and not res.any() and not q._buffer.any()


@pytest.mark.parametrize("m, n, k", [(4, 5000, 3900), (16, 8200, 3900), (1, 12300, 3900), (3, 40, 100)])
@pytest.mark.parametrize("far", ["codes", "scales"])
def test_product_of_a_few_rows_far_apart(m, n, k, far):
    """Up to 16 rows may lie 16 MB apart and more, whichever kernel takes that many of them."""
    mx = _mx()
    rng = np.random.default_rng(m)
    w = mx.quantize_rows(torch.from_numpy(rng.standard_normal((n, k)).astype(np.float16)).to(DEV))
    a = mx.quantize_rows(torch.from_numpy(rng.standard_normal((m, k)).astype(np.float16)).to(DEV))
    apart = torch.empty((m, (1 << 24) + 16), dtype=torch.uint8, device=DEV)
    part = getattr(a, far)
    apart[:, :part.shape[1]] = part
    parts = dict(codes=a.codes, scales=a.scales)
    parts[far] = apart[:, :part.shape[1]]
    got = mx.product(mx.MxRows(parts["codes"], parts["scales"], k), w, out_dtype=torch.float32)
    av, wv = (R.values(r.codes.cpu().numpy(), r.scales.cpu().numpy(), k) for r in (a, w))
    y, mag = R.product(av, wv)
    R.within(got.double().cpu().numpy(), y, R.tolerance(y, mag, k, 2.0 ** -24))


@pytest.mark.parametrize("m, n, k", [(1, 16448, 4096), (4, 17000, 3900), (4, 8192, 8192), (8, 10240, 4000), (2, 20000, 3900)])
def test_few_rows_stay_with_the_kernel_of_few_rows(m, n, k):
    """... beside as many weight rows as it is the faster one for: its sums, bit for bit, which the tiled kernels add in
    another order.  (Blocks of very different strength: the sums have to be rounded.)"""
    mx = _mx()
    torch.manual_seed(m)
    strength = torch.exp2(torch.randint(-10, 11, (-(-k // 32),), device=DEV).float()).repeat_interleave(32)[:k]
    w = mx.quantize_rows(torch.randn(n, k, device=DEV) * strength)
    a = mx.quantize_rows(torch.randn(m, k, device=DEV) * strength)
    got = mx.product(a, w, out_dtype=torch.float32)
    for first in (0, n // 2, n - 640):
        part = mx.product(a, mx.MxRows(w.codes[first:first + 640], w.scales[first:first + 640], k), out_dtype=torch.float32)
        assert torch.equal(got[:, first:first + 640], part)


# either side of 72, 160 (one row: 192) and 256 tiles of 64 weight rows, of 8 rows, and of the sum of both beyond 256; many weight rows
@pytest.mark.parametrize("m, n, k", [(1, 4544, 3900), (9, 4545, 3872), (8, 10240, 3900), (8, 10241, 3900), (2, 12300, 4100), (16, 16384, 3880),
                                     (4, 16385, 3900), (8, 16385, 3900), (16, 17000, 4097), (1, 24900, 3900), (1, 25000, 3900), (1, 37000, 3872),
                                     (13, 37000, 3872), (1, 12288, 3900), (1, 12289, 3900)])
def test_few_rows_beside_many_weight_rows(m, n, k):
    mx = _mx()
    torch.manual_seed(m + n)
    wh, ah = torch.randn(n, k, device=DEV).half(), torch.randn(m, k, device=DEV).half()
    w, a = mx.quantize_rows(wh), mx.quantize_rows(ah)
    wv, av = (mx.dequantize_rows(r, torch.float32).double() for r in (w, a))     # (exact in fp32)
    bias = torch.randn(n, device=DEV)
    y, mag = (av @ wv.T + bias).cpu().numpy(), (av.abs() @ wv.abs().T + bias.abs()).cpu().numpy()
    for x in (a, ah):
        got = mx.product(x, w, bias=bias, out_dtype=torch.float32).double().cpu().numpy()
        R.within(got, y, R.tolerance(y, mag, k, 2.0 ** -24))


def test_rulebook_whose_build_failed_is_not_read():
    """Neither the old table nor half of a new one."""
    mx = _mx()
    rng = np.random.default_rng(6)
    rb, _, n_out, conv, _, _ = conv_case(rng, 50, (9, 24, 21), 64, 32, (3, 3, 3), (1, 1, 1), (1, 1, 1), True)
    q = mx.quantize_rows(torch.zeros((50, 64), dtype=torch.float16, device=DEV))
    conv.forward(q, rb, n_out)
    idx = torch.zeros((5, 4), dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError):
        rb.build_sparse(idx, (9, 24, 21), (3, 3, 3), (1, 1, 1), (-1, 0, 0))
    with pytest.raises(ValueError, match="built"):
        conv.forward(q, rb, n_out)
    rb.build_subm(idx, (9, 24, 21), (3, 3, 3))
    conv.forward(q, rb, n_out)


# ------------------------------------------------------------------------------------------------- one row, one column
def signed_rows(rng, n, c, dtype=np.float16):
    """Rows without a zero channel."""
    x = (rng.uniform(0.5, 2, (n, c)) * rng.choice([-1, 1], (n, c)) * np.exp(rng.standard_normal((n, 1)))).astype(dtype)
    assert x.all()
    return x


@pytest.mark.parametrize("m, n, k", [(1, 1, 1), (1, 1, 33), (1, 16, 32), (1, 33, 100), (1, 70, 1000), (1, 500, 8192), (1, 40, 33000), (1, 16400, 3900),
                                     (1, 12300, 4100), (2, 1, 5000), (16, 1, 70), (17, 1, 3), (300, 1, 64), (300, 1, 300), (40, 1, 1500), (1000, 1, 4097)])
@pytest.mark.parametrize("x", ["mx", "fp16", "fp32"])
def test_product_of_one_row_or_one_column(m, n, k, x):
    mx = _mx()
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    wh, h = signed_rows(rng, n, k), signed_rows(rng, m, k, np.float32 if x == "fp32" else np.float16)
    w, a = mx.quantize_rows(torch.from_numpy(wh).to(DEV)), torch.from_numpy(h).to(DEV)
    bias, res = rng.standard_normal(n).astype(np.float32), rng.standard_normal((m, n)).astype(np.float16)
    kw = dict(bias=torch.from_numpy(bias).to(DEV), residual=torch.from_numpy(res).to(DEV))
    y, mag = R.product(R.fake(h), R.values(w.codes.cpu().numpy(), w.scales.cpu().numpy(), k), bias, False, res, False)
    a = mx.quantize_rows(a) if x == "mx" else a
    for out_dtype, half in ((torch.float16, 2.0 ** -11), (torch.float32, 2.0 ** -24)):
        got = mx.product(a, w, out_dtype=out_dtype, **kw)
        R.within(got.double().cpu().numpy(), y, R.tolerance(y, mag, k, half))
        assert torch.equal(mx.product(a, w, out_dtype=out_dtype, **kw), got)


def test_convolution_of_one_row():
    mx = _mx()
    rng = np.random.default_rng(5)
    for cin, cout in ((5, 16), (64, 64), (128, 40), (160, 32)):
        rb, table, n_out, conv, wv, b = conv_case(rng, 1, (9, 24, 21), cin, cout, (3, 3, 3), (1, 1, 1), (1, 1, 1), True)
        x = signed_rows(rng, 1, cin)
        y, mag = R.convolution(R.fake(x), wv, b, table)
        assert np.abs(y - b).max() > 0.01
        got = conv.forward(mx.quantize_rows(torch.from_numpy(x).to(DEV)), rb, n_out).double().cpu().numpy()
        R.within(got, y, R.tolerance(y, mag, 27 * cin, 2.0 ** -11))


# ------------------------------------------------------------------------------------------------- sums without a rounding
def whole(rng, n, k, only_from=0):
    """Rows of codes under a scale of 1, the channels before `only_from` zero, at least one other that is not: (MxRows, values).
    Products are quarters up to 36, so that fp32 holds every sum of fewer than 2^24 / 144 = 116,508 of them exactly."""
    mx = _mx()
    blocks = -(-k // 32)
    code = rng.integers(0, 16, (n, 32 * blocks)).astype(np.uint8)
    code[:, :only_from] = 0
    code[:, k:] = 0
    code[:, k - 1] |= 1
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    scales = np.zeros((n, -(-blocks // 4) * 4), np.uint8)
    scales[:, :blocks] = 127
    r = mx.MxRows.empty(n, k, DEV)
    r.codes.copy_(torch.from_numpy(codes))
    r.scales.copy_(torch.from_numpy(scales))
    return r, R.values(codes, scales, k)


# every kernel and tile, stages and scale spans of every length, k in parts of unequal length
WHOLE = [(1, 70, 100), (3, 40, 4096), (16, 33, 8190), (20, 100, 1500), (40, 70, 33), (65, 61, 3873), (64, 1000, 4100), (130, 300, 8192), (33, 70, 12289),
         (1000, 1, 4097), (16, 8200, 4128), (1, 12300, 3900), (16, 17000, 3900), (100, 130, 257), (100, 130, 513), (100, 130, 769), (300, 200, 1111),
         (2100, 2200, 1500), (2177, 2049, 515), (4100, 4111, 290), (4111, 4099, 2080)]


@pytest.mark.parametrize("m, n, k", WHOLE)
def test_products_add_every_block_once(m, n, k):
    """Equal to the sums, over all channels and with only the last block, the last few blocks or the last stage not zero."""
    mx = _mx()
    rng = np.random.default_rng(m + n + k)
    last = (k - 1) // 32 * 32
    for first in sorted({0, last, max(0, last - 96), max(0, last // 256 * 256)}):
        w, wv = whole(rng, n, k, first)
        a, av = whole(rng, m, k)
        got = mx.product(a, w, out_dtype=torch.float32)
        want = torch.from_numpy(av.astype(np.float32)).to(DEV).double() @ torch.from_numpy(wv.astype(np.float32)).to(DEV).double().T
        assert want.any() and torch.equal(got.double(), want), first


@pytest.mark.parametrize("m, n, k", [(5, 70, 200), (100, 64, 31), (70, 300, 96), (200, 1000, 128), (130, 200, 250), (64, 64, 256), (40, 300, 1111)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_products_that_quantise_add_every_block_once(m, n, k, dtype):
    """Rows whose channels are values of the format: a 6 in every block makes its scale 1, so quantisation keeps them."""
    mx = _mx()
    rng = np.random.default_rng(m + n + k)
    w, wv = whole(rng, n, k)
    _, av = whole(rng, m, k)
    av[:, ::32] = 6
    got = mx.product(torch.from_numpy(av).to(dtype).to(DEV), w, out_dtype=torch.float32).double().cpu().numpy()
    assert np.array_equal(got, av @ wv.T)


@pytest.mark.parametrize("cin, cout, n, bound", [(16, 16, 500, 500), (32, 64, 500, 40000), (64, 64, 500, 500), (64, 128, 500, 70000), (96, 48, 300, 300),
                                                 (128, 32, 400, 200000), (160, 96, 200, 200), (256, 128, 90, 90)])
@pytest.mark.parametrize("ks", [(3, 3, 3), (5, 3, 3), (1, 1, 1)])
def test_convolutions_add_every_neighbour_once(cin, cout, n, bound, ks):
    """The sums that the kernel dumps, equal to whole numbers (quarters)."""
    import ctypes as C
    mx = _mx()
    rng = np.random.default_rng(cin + cout)
    coords = np.stack(np.unravel_index(np.sort(rng.choice(9 * 24 * 21, n, replace=False)), (9, 24, 21)), 1)
    idx = torch.zeros((bound, 4), dtype=torch.int32, device=DEV)
    idx[:n, 1:] = torch.from_numpy(coords.astype(np.int32)).to(DEV)
    kv = int(np.prod(ks))
    rb = mx.Rulebook(bound, bound, kv)
    rb.build_subm(idx, (9, 24, 21), ks, num=torch.tensor([n], dtype=torch.int32, device=DEV))
    _, table = R.neighbours(coords, (9, 24, 21), ks, (1, 1, 1), (1, 1, 1), (1, 1, 1), True)
    q, xv = whole(rng, n, cin)
    w = rng.choice(R.LEVELS, (cout, kv, cin)) * rng.choice([-1, 1], (cout, kv, cin))
    w[:, :, ::32] = 6
    conv = mx.Conv(w.reshape(cout, *ks, cin).astype(np.float16))
    acc = torch.full((n, cout), 7.0, device=DEV)
    out = torch.empty((n, cout), dtype=torch.float16, device=DEV)
    io = capi.ConvIO()
    io.x_dev, io.x_ld, io.out_dtype = q.codes_ptr, q.codes_ld, capi.DTYPE_FP16
    io.out_dev, io.out_ld, io.acc_dev = out.data_ptr(), cout, acc.data_ptr()
    capi.check(capi.lib().scn_conv_forward(conv._h, rb._h, C.byref(io), torch.cuda.current_stream().cuda_stream))
    y, _ = R.convolution(xv, w, None, table)
    assert np.array_equal(acc.double().cpu().numpy(), y)


# tiles of 64, 128 and 256, k in parts, rows quantised in the same launch (narrow, wide, long, beyond the caches)
@pytest.mark.parametrize("m, n, k, x", [(200, 128, 300, "mx"), (2100, 2304, 600, "mx"), (4200, 4352, 300, "mx"), (70, 128, 4000, "mx"), (200, 64, 64, "fp16"),
                                        (300, 1024, 128, "fp16"), (100, 256, 256, "fp32"), (33000, 256, 100, "fp16")])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.float32])
def test_product_results_in_rows_of_whole_lines_and_others(m, n, k, x, out_dtype):
    """How results are stored depends on whether their rows are whole 128-byte lines; what is stored does not, nor does
    anything else get written."""
    mx = _mx()
    torch.manual_seed(m)
    w, a = mx.quantize_rows(torch.randn(n, k, device=DEV)), torch.randn(m, k, device=DEV)
    a = mx.quantize_rows(a) if x == "mx" else a.to(torch.float16 if x == "fp16" else torch.float32)
    res = torch.randn(m, n, device=DEV).half()
    want = mx.product(a, w, out_dtype=out_dtype, relu=True, residual=res)
    av = mx.dequantize_rows(a if x == "mx" else mx.quantize_rows(a), torch.float32)[:64].double()
    y, mag = R.product(av.cpu().numpy(), mx.dequantize_rows(w, torch.float32).double().cpu().numpy(), None, True, res[:64].double().cpu().numpy())
    R.within(want[:64].double().cpu().numpy(), y, R.tolerance(y, mag, k, 2.0 ** -11 if out_dtype == torch.float16 else 2.0 ** -24))
    for lead, extra in ((0, 32 // want.element_size() * 4), (0, 8), (64 // want.element_size(), 0), (1, 0), (3, 5)):
        flat = torch.full((lead + m * (n + extra) + 64,), 9.0, dtype=out_dtype, device=DEV)
        out = flat[lead:lead + m * (n + extra)].view(m, n + extra)[:, :n]
        mx.product(a, w, relu=True, residual=res, out=out)
        assert torch.equal(out, want), (lead, extra)
        out.fill_(9)
        assert (flat == 9).all(), (lead, extra)


@pytest.mark.parametrize("cin, cout", [(16, 16), (64, 64), (96, 48)])
def test_convolutions_of_medium_and_large_bounds_share_a_tile_between_two_waves(cin, cout):
    """The bound of the row count chooses how many waves share a tile, and so the order of the sums: these bounds have the
    same one.  (Blocks of very different strength: the sums have to be rounded.)"""
    import ctypes as C
    mx = _mx()
    rng = np.random.default_rng(cin)
    n, kv = 900, 27
    coords = np.stack(np.unravel_index(np.sort(rng.choice(9 * 12 * 12, n, replace=False)), (9, 12, 12)), 1)
    x = (rng.standard_normal((n, cin)) * np.exp2(rng.integers(-8, 9, (n, 1)))).astype(np.float16)
    conv = mx.Conv((rng.standard_normal((cout, 3, 3, 3, cin)) * np.exp2(rng.integers(-8, 9, (1, 3, 3, 3, 1)))).astype(np.float16))
    q = mx.quantize_rows(torch.from_numpy(x).to(DEV))
    sums = []
    for bound in (40000, 66000, 98304, 163841, 190000, 200000):
        idx = torch.zeros((bound, 4), dtype=torch.int32, device=DEV)
        idx[:n, 1:] = torch.from_numpy(coords.astype(np.int32)).to(DEV)
        rb = mx.Rulebook(bound, bound, kv)
        rb.build_subm(idx, (9, 12, 12), (3, 3, 3), num=torch.tensor([n], dtype=torch.int32, device=DEV))
        acc = torch.full((n, cout), 7.0, device=DEV)
        out = torch.empty((n, cout), dtype=torch.float16, device=DEV)
        io = capi.ConvIO()
        io.x_dev, io.x_ld, io.out_dtype = q.codes_ptr, q.codes_ld, capi.DTYPE_FP16
        io.out_dev, io.out_ld, io.acc_dev = out.data_ptr(), cout, acc.data_ptr()
        capi.check(capi.lib().scn_conv_forward(conv._h, rb._h, C.byref(io), torch.cuda.current_stream().cuda_stream))
        sums.append(acc)
        assert torch.equal(acc, sums[0]), bound
