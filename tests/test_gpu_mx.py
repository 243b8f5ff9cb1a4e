"""Microscaled 4-bit rows on the GPU against their float64 oracle (tests/mx_reference.py)."""
import ctypes as C

import numpy as np
import pytest
import torch

from lidar_ai_solution_amd import capi
from tests import mx_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HALF = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}   # half a step, relative
NP = {torch.float16: np.float16, torch.float32: np.float32}


def _mx():
    from lidar_ai_solution_amd import mx
    return mx


def rows(rng, n, c, dtype=np.float16, outliers=True):
    x = rng.standard_normal((n, c)) * np.exp(rng.standard_normal((n, 1)))
    if outliers and n and c:
        x[rng.integers(0, n, max(1, n // 8))] = 0
        x[:, rng.integers(0, c, max(1, c // 16))] *= 37
    return x.astype(dtype)


def strided(a, ld, lead=0):
    """A device tensor whose rows are ld elements apart and start `lead` elements into an allocation."""
    a = np.asarray(a)
    t = {np.dtype(np.float16): torch.float16, np.dtype(np.float32): torch.float32, np.dtype(np.int8): torch.int8}[a.dtype]
    flat = torch.full((lead + a.shape[0] * ld + 1,), 3, dtype=t, device=DEV)
    v = flat[lead:lead + a.shape[0] * ld].view(a.shape[0], ld)[:, :a.shape[1]]
    v.copy_(torch.from_numpy(np.ascontiguousarray(a)))
    return v


def assert_same_rows(got, want, c):
    codes, scales = want
    nb = -(-c // 32)
    assert np.array_equal(got.scales[:, :-(-nb // 4) * 4].cpu().numpy(), scales)
    assert np.array_equal(got.codes[:, :16 * nb].cpu().numpy(), codes)


def mx_rows(rng, n, c):
    """Quantised rows made on the host: (MxRows, their values)."""
    mx = _mx()
    x = rows(rng, n, c)
    codes, scales = R.quantize(x)
    r = mx.MxRows.empty(n, c, DEV)
    r.codes.copy_(torch.from_numpy(codes))
    r.scales.copy_(torch.from_numpy(scales))
    return r, R.values(codes, scales, c)


# ------------------------------------------------------------------------------------------------- quantise
@pytest.mark.parametrize("top", [6.0, 7.99, 1.0, 3.5, 65504.0, 2.0 ** -14, 2.0 ** -24, 2.0 ** -20, 0.0999755859375])
def test_every_fp16_value_below_a_block_maximum(top):
    top = np.float16(top)
    v = np.arange(1 << 16, dtype=np.uint16).view(np.float16)
    v = v[np.abs(v) <= top]
    v = np.concatenate([v, np.zeros(-v.size % 31, np.float16)]).reshape(-1, 31)
    x = np.concatenate([np.full((v.shape[0], 1), top), v], 1)
    assert_same_rows(_mx().quantize_rows(torch.from_numpy(x).to(DEV)), R.quantize(x), 32)


def test_fp32_from_subnormal_to_huge_and_not_finite():
    rng = np.random.default_rng(1)
    e = rng.integers(-149, 128, (4096, 1))
    x = np.ldexp(rng.uniform(-1, 1, (4096, 64)), e + rng.integers(-6, 1, (4096, 64))).astype(np.float32)
    x[7] = -0.0
    x[8, 3], x[9, 40], x[10, 63], x[11, :] = np.nan, np.inf, -np.inf, np.finfo(np.float32).max
    x[12, 0], x[12, 1] = np.finfo(np.float32).min, 2.0 ** -149
    assert_same_rows(_mx().quantize_rows(torch.from_numpy(x).to(DEV)), R.quantize(x), 64)


@pytest.mark.parametrize("dtype", [np.float16, np.float32, np.int8])
@pytest.mark.parametrize("n, c, extra, lead", [(1, 1, 0, 0), (0, 5, 0, 0), (3, 2, 1, 1), (65, 31, 2, 1), (64, 32, 0, 0), (7, 33, 0, 3), (5, 63, 1, 0),
                                               (129, 64, 8, 0), (33, 96, 0, 8), (11, 129, 3, 5), (6, 1000, 0, 1), (2, 4100, 4, 2)])
def test_quantize_shapes_strides_and_alignment(dtype, n, c, extra, lead):
    rng = np.random.default_rng(n * 1000 + c)
    if dtype == np.int8:
        x = rng.integers(-127, 128, (n, c)).astype(np.int8)
        want = x.astype(np.float32) * (np.float32(3.7) / np.float32(127))
    else:
        x = want = rows(rng, n, c, dtype)
    for relu in (False, True):
        got = _mx().quantize_rows(strided(x, c + extra, lead), relu=relu, dynamic_range=3.7)
        assert_same_rows(got, R.quantize(np.where(want > 0, want, 0) if relu else want), c)


def test_quantize_relu_clears_nan_like_the_other_row_operators():
    x = np.array([[np.nan, 2.0, -3.0, 1.0]], np.float16)
    assert_same_rows(_mx().quantize_rows(torch.from_numpy(x).to(DEV), relu=True), R.quantize(np.array([[0, 2.0, 0, 1.0]])), 4)


def test_separate_arrays_device_count_and_rows_behind_it():
    mx = _mx()
    rng = np.random.default_rng(5)
    n, c, live = 50, 200, 17
    x = rows(rng, n, c)
    codes = torch.full((n, 128), 0xAB, dtype=torch.uint8, device=DEV)
    scales = torch.full((n, 12), 0xCD, dtype=torch.uint8, device=DEV)
    out = mx.MxRows(codes, scales, c)
    mx.quantize_rows(torch.from_numpy(x).to(DEV), num=torch.tensor([live], dtype=torch.int32, device=DEV), out=out)
    wc, ws = R.quantize(x[:live])
    assert np.array_equal(codes[:live, :112].cpu().numpy(), wc) and np.array_equal(scales[:live, :8].cpu().numpy(), ws)
    assert (codes[live:] == 0xAB).all() and (scales[live:] == 0xCD).all() and (codes[:, 112:] == 0xAB).all() and (scales[:, 8:] == 0xCD).all()
    back = torch.full((n, c + 3), 7.0, dtype=torch.float32, device=DEV)
    mx.dequantize_rows(out, out=back[:, :c], num=torch.tensor([live], dtype=torch.int32, device=DEV))
    assert np.array_equal(back[:live, :c].cpu().numpy(), R.values(wc, ws, c)) and (back[live:] == 7).all() and (back[:, c:] == 7).all()
    mx.quantize_rows(torch.from_numpy(x).to(DEV), num=torch.tensor([0], dtype=torch.int32, device=DEV), out=out)
    assert (codes[live:] == 0xAB).all()


def test_rows_past_four_gigabytes():
    """The last rows of a buffer of more than 2^32 bytes."""
    mx = _mx()
    rng = np.random.default_rng(6)
    n, c = 70000, 32800
    x = torch.zeros((n, c), dtype=torch.float16, device=DEV)
    tail = rows(rng, 3, c)
    x[-3:] = torch.from_numpy(tail).to(DEV)
    q = mx.quantize_rows(x)
    wc, ws = R.quantize(tail)
    assert np.array_equal(q.codes[-3:].cpu().numpy(), wc) and np.array_equal(q.scales[-3:].cpu().numpy(), ws)
    assert not q.codes[:-3].any() and not q.scales[:-3].any()
    back = mx.dequantize_rows(q, out=x)
    assert np.array_equal(back[-3:].cpu().numpy(), R.values(wc, ws, c).astype(np.float16)) and not back[:-3].any()


def test_quantize_wrapper_refusals():
    mx = _mx()
    x = torch.zeros((4, 64), dtype=torch.float16, device=DEV)
    for bad in (x.cpu(), x.t(), x.double(), x[0], x[:, ::2], x[:1].expand(4, 64)):
        with pytest.raises(ValueError):
            mx.quantize_rows(bad)
    with pytest.raises(RuntimeError):
        mx.quantize_rows(x.to(torch.int8))                       # no dynamic range
    with pytest.raises(ValueError):
        mx.quantize_rows(x, out=mx.MxRows.empty(3, 64))
    with pytest.raises(ValueError):
        mx.quantize_rows(x, num=torch.tensor([3], dtype=torch.int64, device=DEV))
    q = mx.quantize_rows(x)
    with pytest.raises(ValueError):
        mx.MxRows(q.codes[:, :16], q.scales, 64)
    with pytest.raises(ValueError):
        mx.product(q, mx.quantize_rows(x[:, :32].contiguous()))
    with pytest.raises(ValueError):
        mx.product(q, q, bias=torch.zeros(3, device=DEV))
    with pytest.raises(ValueError):
        mx.quantize_rows(torch.empty_strided((1, 4), (1 << 32, 1), dtype=torch.float16, device=DEV))   # stride beyond 32 bits
    with pytest.raises(RuntimeError):
        mx.product(x, mx.quantize_rows(torch.zeros((64, 64), dtype=torch.float16, device=DEV)), out=x)
    with pytest.raises(ValueError):
        mx.MxRows.empty(-1, 4)


# ------------------------------------------------------------------------------------------------- dequantise
@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_every_code_with_every_scale(dtype):
    mx = _mx()
    pairs = np.arange(256, dtype=np.uint8).reshape(16, 16)                # every byte = every pair of codes
    codes = np.tile(pairs, (256, 1))
    scales = np.zeros((4096, 4), np.uint8)
    scales[:, 0] = np.repeat(np.arange(256), 16)
    r = mx.MxRows(torch.from_numpy(codes).to(DEV), torch.from_numpy(scales).to(DEV), 32)
    with np.errstate(over="ignore"):
        want = R.values(codes, scales, 32).astype(NP[dtype])
    got = mx.dequantize_rows(r, dtype).cpu().numpy()
    assert np.array_equal(got, want, equal_nan=True) and np.array_equal(np.signbit(got)[:4080], np.signbit(want)[:4080])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("n, c, extra, lead", [(1, 1, 0, 0), (0, 9, 0, 0), (5, 31, 0, 1), (64, 32, 0, 0), (9, 45, 3, 0), (17, 130, 0, 1), (3, 2051, 1, 3)])
def test_dequantize_shapes(dtype, n, c, extra, lead):
    rng = np.random.default_rng(c)
    q, want = mx_rows(rng, n, c)
    out = strided(np.full((n, c), 5, NP[dtype]), c + extra, lead)
    _mx().dequantize_rows(q, out=out)
    assert np.array_equal(out.cpu().numpy(), want.astype(NP[dtype]))


# ------------------------------------------------------------------------------------------------- product
SHAPES = [(1, 1, 1), (1, 16, 32), (1, 33, 100), (2, 70, 4096), (15, 17, 2080), (16, 64, 129), (17, 5, 31), (31, 129, 96), (33, 16, 33), (64, 64, 512),
          (65, 257, 64), (100, 100, 1000), (127, 130, 257), (128, 128, 256), (200, 300, 520), (257, 513, 300), (300, 1, 64), (513, 260, 1111),
          (1000, 48, 16), (40, 1000, 2500)]


@pytest.mark.parametrize("m, n, k", SHAPES)
@pytest.mark.parametrize("x", ["mx", "fp16", "fp32"])
def test_product(m, n, k, x):
    mx = _mx()
    rng = np.random.default_rng(m * 7 + n * 3 + k)
    w, wv = mx_rows(rng, n, k)
    if x == "mx":
        a, av = mx_rows(rng, m, k)
    else:
        h = rows(rng, m, k, np.float16 if x == "fp16" else np.float32)
        a, av = strided(h, k + (m % 3), m % 2), R.fake(h)
    for i, out_dtype in enumerate((torch.float16, torch.float32)):
        bias = res = None
        relu, relu2 = bool((m + i) % 2), bool((n + i) % 2)
        if (m + n + i) % 2:
            bias = rng.standard_normal(n).astype(np.float32 if k % 2 else np.float16)
        if (k + i) % 2:
            res = rng.standard_normal((m, n)).astype(np.float16 if n % 2 else np.float32)
        out = strided(np.full((m, n), 9, NP[out_dtype]), n + (k % 5), i)
        got = mx.product(a, w, bias=None if bias is None else torch.from_numpy(bias).to(DEV), relu=relu,
                         residual=None if res is None else strided(res, n + (m % 4), i), relu_after_add=relu2, out=out)
        y, mag = R.product(av, wv, bias, relu, res, relu2)
        R.within(got.double().cpu().numpy(), y, R.tolerance(y, mag, k, HALF[out_dtype]))


# enough tiles of 128 x 128 or 256 x 256 for the GPU, and tiles of 64 x 64; k of one stage, of a short last stage, of a short scale span
@pytest.mark.parametrize("m, n, k", [(2050, 2061, 96), (2177, 2049, 515), (5000, 1030, 256), (4100, 4111, 290), (4097, 4300, 777), (16400, 1290, 1024),
                                     (4111, 4099, 2080), (16500, 1030, 70)])
def test_large_products(m, n, k):
    mx = _mx()
    rng = np.random.default_rng(m + n + k)
    w, wv = mx_rows(rng, n, k)
    a, av = mx_rows(rng, m, k)
    res = rng.standard_normal((m, n)).astype(np.float16)
    bias = rng.standard_normal(n).astype(np.float32)
    y, mag = R.product(av, wv, bias, False, res, True)
    for out_dtype in (torch.float16, torch.float32):
        out = strided(np.full((m, n), 9, NP[out_dtype]), n + 3, 1)
        num = torch.tensor([m - 130], dtype=torch.int32, device=DEV)
        mx.product(a, w, bias=torch.from_numpy(bias).to(DEV), residual=torch.from_numpy(res).to(DEV), relu_after_add=True, out=out, num=num)
        got = out.double().cpu().numpy()
        R.within(got[:m - 130], y[:m - 130], R.tolerance(y, mag, k, HALF[out_dtype])[:m - 130])
        assert (got[m - 130:] == 9).all()


# tiles of 128 x 128 with many stages; few tiles down a long k, whose stages are divided: a short last part, an empty one
# (17 stages), equal ones, a last stage of one block
@pytest.mark.parametrize("m, n, k", [(2100, 2200, 1500), (65, 61, 3873), (64, 1000, 4100), (130, 300, 8192), (33, 70, 12289), (1000, 1, 4097),
                                     (3, 5000, 4000), (1, 16400, 3900), (16, 8200, 4128), (30, 600, 1500)])
@pytest.mark.parametrize("res_dtype", [np.float16, np.float32])
def test_products_down_a_long_k(m, n, k, res_dtype):
    mx = _mx()
    rng = np.random.default_rng(m + n + k)
    w, wv = mx_rows(rng, n, k)
    a, av = mx_rows(rng, m, k)
    res = rng.standard_normal((m, n)).astype(res_dtype)
    bias = rng.standard_normal(n).astype(np.float32)
    y, mag = R.product(av, wv, bias, True, res, False)
    for out_dtype, kept in ((torch.float16, m), (torch.float32, m // 2), (torch.float16, 0)):
        out = strided(np.full((m, n), 9, NP[out_dtype]), n + 3, 1)
        num = torch.tensor([kept], dtype=torch.int32, device=DEV)
        mx.product(a, w, bias=torch.from_numpy(bias).to(DEV), relu=True, residual=torch.from_numpy(res).to(DEV), out=out, num=num)
        got = out.double().cpu().numpy()
        R.within(got[:kept], y[:kept], R.tolerance(y, mag, k, HALF[out_dtype])[:kept])
        assert (got[kept:] == 9).all()
        again = torch.full_like(out, 9)
        mx.product(a, w, bias=torch.from_numpy(bias).to(DEV), relu=True, residual=torch.from_numpy(res).to(DEV), out=again, num=num)
        assert torch.equal(again, out)


# quantised in the product's launch (k up to 128 with n up to 1024, up to 256 with n up to 256), and just beyond
@pytest.mark.parametrize("m, n, k", [(70, 300, 1), (129, 65, 7), (200, 129, 33), (65, 1024, 127), (100, 1025, 128), (64, 256, 256), (63, 257, 256),
                                     (1000, 255, 250), (90, 20, 200), (300, 64, 64), (260, 128, 9), (17, 70, 3), (5000, 100, 129), (33, 200, 257)])
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("res_dtype", [None, np.float16, np.float32])
def test_product_of_short_rows(m, n, k, dtype, res_dtype):
    mx = _mx()
    rng = np.random.default_rng(m + n + k)
    w, wv = mx_rows(rng, n, k)
    w.scales[:, -(-k // 32):] = 255                                        # (padding: not read)
    h = rows(rng, m, k, dtype)
    a = strided(h, k + 3, 1)
    bias = rng.standard_normal(n).astype(np.float32)
    res = None if res_dtype is None else rng.standard_normal((m, n)).astype(res_dtype)
    y, mag = R.product(R.fake(h), wv, bias, True, res, False)
    for out_dtype, kept in ((torch.float16, m), (torch.float32, m - 5), (torch.float32, 0)):
        out = strided(np.full((m, n), 9, NP[out_dtype]), n + 2, 1)
        num = torch.tensor([kept], dtype=torch.int32, device=DEV)
        mx.product(a, w, bias=torch.from_numpy(bias).to(DEV), relu=True, residual=None if res is None else strided(res, n + 1, 1), out=out, num=num)
        got = out.double().cpu().numpy()
        R.within(got[:kept], y[:kept], R.tolerance(y, mag, k, HALF[out_dtype])[:kept])
        assert (got[kept:] == 9).all()
    if res_dtype == np.float16:                                            # over its residual
        t = torch.from_numpy(res).to(DEV)
        mx.product(a, w, bias=torch.from_numpy(bias).to(DEV), relu=True, residual=t, out=t)
        R.within(t.double().cpu().numpy(), y, R.tolerance(y, mag, k, 2.0 ** -11))


@pytest.mark.parametrize("m", [5, 60, 400])
def test_product_device_count_strides_and_untouched_memory(m):
    mx = _mx()
    rng = np.random.default_rng(m)
    n, k, live = 75, 320, m - 3
    w, wv = mx_rows(rng, n, k)
    a, av = mx_rows(rng, m, k)
    buf = torch.full((m, n + 6), 11.0, dtype=torch.float16, device=DEV)
    num = torch.tensor([live], dtype=torch.int32, device=DEV)
    mx.product(a, w, num=num, out=buf[:, 2:n + 2])
    y, mag = R.product(av, wv)
    R.within(buf[:live, 2:n + 2].double().cpu().numpy(), y[:live], R.tolerance(y, mag, k, 2.0 ** -11)[:live])
    assert (buf[live:] == 11).all() and (buf[:, :2] == 11).all() and (buf[:, n + 2:] == 11).all()
    num.zero_()
    buf.fill_(11)
    mx.product(a, w, num=num, out=buf[:, 2:n + 2])
    assert (buf == 11).all()


@pytest.mark.parametrize("m", [3, 40, 300])
def test_product_into_its_own_residual(m):
    mx = _mx()
    rng = np.random.default_rng(m)
    w, wv = mx_rows(rng, 130, 200)
    a, av = mx_rows(rng, m, 200)
    res = rng.standard_normal((m, 130)).astype(np.float16)
    t = torch.from_numpy(res).to(DEV)
    mx.product(a, w, residual=t, out=t)
    y, mag = R.product(av, wv, res=res)
    R.within(t.double().cpu().numpy(), y, R.tolerance(y, mag, 200, 2.0 ** -11))


@pytest.mark.parametrize("m", [2, 50, 260])
def test_product_scale_padding_and_missing_channels_are_not_read(m):
    """Rows with 3 blocks and 80 channels whose scale padding holds 255 (a NaN if it were used)."""
    mx = _mx()
    rng = np.random.default_rng(m)
    w, wv = mx_rows(rng, 70, 80)
    a, av = mx_rows(rng, m, 80)
    w.scales[:, 3] = 255
    a.scales[:, 3] = 255
    y, mag = R.product(av, wv)
    got = mx.product(a, w, out_dtype=torch.float32).double().cpu().numpy()
    R.within(got, y, R.tolerance(y, mag, 80, 2.0 ** -24))


@pytest.mark.parametrize("m", [4, 40, 200])
@pytest.mark.parametrize("x", ["mx", "fp16"])
def test_product_spreads_nan_to_its_rows_and_columns_only(m, x):
    mx = _mx()
    rng = np.random.default_rng(m)
    wh, ah = rows(rng, 40, 100), rows(rng, m, 100)
    wh[5, 50], ah[1, 99] = np.inf, np.nan
    w = mx.quantize_rows(torch.from_numpy(wh).to(DEV))
    a = torch.from_numpy(ah).to(DEV)
    got = mx.product(mx.quantize_rows(a) if x == "mx" else a, w).isnan().cpu().numpy()
    want = np.zeros((m, 40), bool)
    want[1] = want[:, 5] = True
    assert np.array_equal(got, want)


def test_product_of_extreme_scales():
    """Scales at both ends: products that underflow to 0 and overflow to infinity in fp32."""
    mx = _mx()
    one = torch.full((20, 16), 0x22, dtype=torch.uint8, device=DEV)    # every code 2: value 1
    def with_scale(s):
        return mx.MxRows(one, torch.tensor([[s, 0, 0, 0]], dtype=torch.uint8, device=DEV).repeat(20, 1), 32)
    for sa, sb, want in [(0, 0, 0.0), (0, 254, 32.0), (254, 254, np.inf), (127, 127, 32.0), (1, 127, 32 * 2.0 ** -126), (250, 127, 32 * 2.0 ** 123 if 123 + 5 < 128 else np.inf)]:
        got = mx.product(with_scale(sa), with_scale(sb), out_dtype=torch.float32)
        assert (got == want).all(), (sa, sb, got[0, 0].item())


def test_product_is_the_same_every_time_and_on_another_stream():
    mx = _mx()
    rng = np.random.default_rng(9)
    w, _ = mx_rows(rng, 500, 1500)
    for m in (1, 16, 90, 700):
        x = torch.from_numpy(rows(rng, m, 1500)).to(DEV)
        first = mx.product(x, w)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        second = mx.product(x, w, stream=s, workspace=torch.empty(1 << 21, dtype=torch.uint8, device=DEV))
        torch.cuda.synchronize()
        assert torch.equal(first, second)


def test_calls_on_a_stream_of_their_own_own_their_memory():
    """Buffers that a call allocates belong to the stream it was given: work on the current stream does not get them while the
    other stream still uses them."""
    mx = _mx()
    rng = np.random.default_rng(12)
    w, wv = mx_rows(rng, 256, 512)
    h = rows(rng, 3000, 512)
    x = torch.from_numpy(h).to(DEV)
    y, mag = R.product(R.fake(h), wv)
    side = torch.cuda.Stream()
    for stream in (side, side.cuda_stream):
        torch.cuda.synchronize()
        got = []
        for _ in range(4):
            got.append(mx.dequantize_rows(mx.quantize_rows(mx.product(x, w, stream=stream), stream=stream), torch.float32, stream=stream))
            junk = [torch.full((3000, 256), 7.0, dtype=torch.float16, device=DEV) for _ in range(3)]   # wants freed memory
        torch.cuda.synchronize()
        first = mx.product(x, w)
        R.within(first.double().cpu().numpy(), y, R.tolerance(y, mag, 512, 2.0 ** -11))
        want = mx.dequantize_rows(mx.quantize_rows(first), torch.float32)
        assert all(torch.equal(g.view(torch.int32), want.view(torch.int32)) for g in got) and len(junk) == 3   # (bits: infinite products quantise to NaN)


# ------------------------------------------------------------------------------------------------- convolution
def scene(rng, n, grid):
    cells = np.sort(rng.choice(grid[0] * grid[1] * grid[2], n, replace=False))
    return np.stack([cells // (grid[1] * grid[2]), cells // grid[2] % grid[1], cells % grid[2]], 1)


def conv_case(rng, n, grid, cin, cout, ks, stride, pad, subm, shuffle=False):
    mx = _mx()
    coords = scene(rng, n, grid)
    if shuffle:
        coords = coords[rng.permutation(n)]
    out, table = R.neighbours(coords, grid, ks, stride, pad, (1, 1, 1), subm)
    idx = torch.from_numpy(np.concatenate([np.zeros((n, 1)), coords], 1).astype(np.int32)).to(DEV)
    kv = int(np.prod(ks))
    n_out = table.shape[1]
    rb = mx.Rulebook(n, max(n, n_out), kv) if subm else mx.Rulebook(n, n_out, kv)
    rb.build_subm(idx, grid, ks) if subm else rb.build_sparse(idx, grid, ks, stride, pad)
    w = (rng.standard_normal((cout, *ks, cin)) / np.sqrt(4 * cin)).astype(np.float16)
    b = rng.standard_normal(cout).astype(np.float16)
    wv = R.fake(w.reshape(cout * kv, cin)).reshape(cout, kv, cin)
    return rb, table, n_out, mx.Conv(w, b), wv, b.astype(np.float64)


CONVS = [(5, 16, 900, (3, 3, 3), (1, 1, 1), (1, 1, 1), True), (16, 16, 400, (3, 3, 3), (1, 1, 1), (1, 1, 1), True),
         (16, 32, 700, (3, 3, 3), (2, 2, 2), (1, 1, 1), False), (32, 32, 1000, (3, 3, 3), (1, 1, 1), (1, 1, 1), True),
         (32, 64, 500, (3, 3, 3), (2, 2, 2), (0, 1, 1), False), (64, 64, 1, (3, 3, 3), (1, 1, 1), (1, 1, 1), True),
         (64, 64, 1500, (3, 3, 3), (1, 1, 1), (1, 1, 1), True), (64, 128, 600, (3, 3, 3), (2, 2, 2), (1, 1, 1), False),
         (128, 128, 333, (3, 3, 3), (1, 1, 1), (1, 1, 1), True), (128, 128, 500, (3, 1, 1), (2, 1, 1), (0, 0, 0), False),
         (96, 48, 400, (3, 3, 3), (1, 1, 1), (1, 1, 1), True), (24, 20, 300, (1, 1, 3), (1, 1, 2), (0, 0, 0), False),
         (64, 96, 200, (1, 1, 1), (1, 1, 1), (0, 0, 0), True), (160, 256, 150, (3, 3, 3), (1, 1, 1), (1, 1, 1), True),
         (256, 130, 100, (3, 3, 1), (1, 1, 1), (1, 1, 0), True), (33, 40, 260, (5, 3, 3), (1, 1, 1), (2, 1, 1), True)]


@pytest.mark.parametrize("cin, cout, n, ks, stride, pad, subm", CONVS)
def test_convolution(cin, cout, n, ks, stride, pad, subm):
    mx = _mx()
    rng = np.random.default_rng(cin * 31 + cout + n)
    rb, table, n_out, conv, wv, b = conv_case(rng, n, (9, 24, 21), cin, cout, ks, stride, pad, subm, shuffle=bool(cin % 3))
    x = rows(rng, n, cin)
    xv = R.fake(x)
    y, mag = R.convolution(xv, wv, b, table)
    terms = cin * table.shape[0]
    q = mx.quantize_rows(torch.from_numpy(x).to(DEV))
    for relu in (False, True):
        got = conv.forward(q, rb, n_out, relu=relu).double().cpu().numpy()
        want = np.where(y > 0, y, 0) if relu else y
        R.within(got, want, R.tolerance(want, mag, terms, 2.0 ** -11))
    # residual: the convolution is rounded to fp16 first, as the separate Add would read it
    wide = -(-cout // 16) * 16
    res = rng.standard_normal((n_out, wide)).astype(np.float16)
    got = conv.forward(q, rb, n_out, residual=torch.from_numpy(res).to(DEV), relu_after_add=True).double().cpu().numpy()
    want = np.maximum(y + res[:, :cout], 0)
    tol = R.tolerance(y, mag, terms, 2.0 ** -11) + R.tolerance(want, 0 * mag, terms, 2.0 ** -11)
    R.within(got, want, tol)


@pytest.mark.parametrize("bound", [40000, 70000, 200000])
@pytest.mark.parametrize("cin, cout, n, ks, stride, pad, subm", [CONVS[i] for i in (0, 2, 3, 4, 6, 7, 8, 10, 15)])
def test_convolution_with_a_large_bound(cin, cout, n, ks, stride, pad, subm, bound):
    """The bound of the row count chooses how many waves share a tile of rows; the count stays on the device."""
    mx = _mx()
    rng = np.random.default_rng(cin * 7 + cout + n)
    grid = (9, 24, 21)
    coords = scene(rng, n, grid)
    out_coords, table = R.neighbours(coords, grid, ks, stride, pad, (1, 1, 1), subm)
    idx = torch.zeros((bound, 4), dtype=torch.int32, device=DEV)
    idx[:n, 1:] = torch.from_numpy(coords.astype(np.int32)).to(DEV)
    num = torch.tensor([n], dtype=torch.int32, device=DEV)
    kv, n_out = int(np.prod(ks)), table.shape[1]
    rb = mx.Rulebook(bound, bound, kv)
    rb.build_subm(idx, grid, ks, num=num) if subm else rb.build_sparse(idx, grid, ks, stride, pad, num=num)
    w = (rng.standard_normal((cout, *ks, cin)) / np.sqrt(4 * cin)).astype(np.float16)
    b = rng.standard_normal(cout).astype(np.float16)
    x = rows(rng, n, cin)
    q = mx.MxRows.empty(bound, cin, DEV)
    mx.quantize_rows(torch.cat([torch.from_numpy(x), torch.full((bound - n, cin), float("nan"), dtype=torch.float16)]).to(DEV), num=num, out=q)
    y, mag = R.convolution(R.fake(x), R.fake(w.reshape(cout * kv, cin)).reshape(cout, kv, cin), b.astype(np.float64), table)
    out = torch.full((bound, -(-cout // 16) * 16), 3.0, dtype=torch.float16, device=DEV)
    mx.Conv(w, b).forward(q, rb, bound, out=out)
    R.within(out[:n_out, :cout].double().cpu().numpy(), y, R.tolerance(y, mag, kv * cin, 2.0 ** -11))
    assert (out[n_out:] == 3).all()


@pytest.mark.parametrize("cin, cout, n, ks, stride, pad, subm", [c for c in CONVS if c[0] <= 128])
def test_convolution_stores_microscaled_rows(cin, cout, n, ks, stride, pad, subm):
    """out = MxRows gets, bit for bit, what quantize_rows makes of the fp16 result (also of results that are not finite)."""
    mx = _mx()
    rng = np.random.default_rng(cin + cout * 5 + n)
    rb, table, n_out, conv, _, _ = conv_case(rng, n, (9, 24, 21), cin, cout, ks, stride, pad, subm)
    x = rows(rng, n, cin)
    x[n // 2] = np.nan
    q = mx.quantize_rows(torch.from_numpy(x).to(DEV))
    res = torch.from_numpy(rng.standard_normal((n_out, -(-cout // 16) * 16)).astype(np.float16)).to(DEV)
    for kw in (dict(relu=True), dict(residual=res, relu_after_add=True)):
        want = mx.quantize_rows(conv.forward(q, rb, n_out, **kw))
        got = mx.MxRows.empty(n_out + 3, cout, DEV)
        got.codes.fill_(0xAA), got.scales.fill_(0xBB)
        assert conv.forward(q, rb, n_out, out=got, **kw) is got
        assert torch.equal(got.codes[:n_out], want.codes) and torch.equal(got.scales[:n_out], want.scales)
        assert (got.codes[n_out:] == 0xAA).all() and (got.scales[n_out:] == 0xBB).all()


@pytest.mark.parametrize("cin, cout, bound", [(16, 16, 500), (64, 64, 500), (64, 64, 40000), (96, 128, 500), (32, 48, 120000), (160, 32, 500)])
@pytest.mark.parametrize("res", [None, "fp16", "int8", "requantised"])
def test_convolution_int8_output_and_every_residual(cin, cout, bound, res):
    """The epilogue's arithmetic on the sums that the kernel dumps, in fp32 step by step: bit for bit."""
    mx = _mx()
    f32 = np.float32
    rng = np.random.default_rng(cin + cout)
    coords = scene(rng, 500, (9, 24, 21))
    idx = torch.zeros((bound, 4), dtype=torch.int32, device=DEV)
    idx[:500, 1:] = torch.from_numpy(coords.astype(np.int32)).to(DEV)
    rb = mx.Rulebook(bound, bound, 27)
    rb.build_subm(idx, (9, 24, 21), (3, 3, 3), num=torch.tensor([500], dtype=torch.int32, device=DEV))
    w = (rng.standard_normal((cout, 3, 3, 3, cin)) / np.sqrt(4 * cin)).astype(np.float16)
    b = rng.standard_normal(cout).astype(np.float16)
    conv = mx.Conv(w, b)
    q = mx.quantize_rows(torch.from_numpy(rows(rng, 500, cin)).to(DEV))
    r16, r8 = rng.standard_normal((500, cout)).astype(np.float16), rng.integers(-127, 128, (500, cout)).astype(np.int8)

    def quant(y, amax):
        return np.clip(np.rint(y * (f32(127) / f32(amax))), -127, 127).astype(f32)

    def step(amax):
        return f32(amax) / f32(127)

    for relu in (0, 1):
        acc = torch.full((500, cout), 7.0, device=DEV)
        out = torch.full((503, cout), 9, dtype=torch.int8, device=DEV)
        io = capi.ConvIO()
        io.x_dev, io.x_ld, io.relu, io.out_dtype, io.out_dynamic_range = q.codes_ptr, q.codes_ld, relu, capi.DTYPE_INT8, 5.0
        io.out_dev, io.out_ld, io.acc_dev = out.data_ptr(), cout, acc.data_ptr()
        keep = None
        if res is not None:
            keep = torch.from_numpy(r8 if res == "int8" else r16).to(DEV)
            io.res_dev, io.res_ld, io.relu_after_add = keep.data_ptr(), cout, 1 - relu
            io.res_dtype = capi.DTYPE_INT8 if res == "int8" else capi.DTYPE_FP16
            io.mid_dtype = io.res_dtype
            if res == "int8":
                io.res_dynamic_range, io.mid_dynamic_range = 3.0, 4.0
            if res == "requantised":
                io.a_requant_range, io.b_requant_range = 2.5, 3.5
        capi.check(capi.lib().scn_conv_forward(conv._h, rb._h, C.byref(io), torch.cuda.current_stream().cuda_stream))
        y = acc.cpu().numpy() + b.astype(f32)
        if relu:
            y = np.maximum(y, f32(0))
        if res == "int8":
            y = quant(y, 4.0) * step(4.0) + r8.astype(f32) * step(3.0)
        elif res is not None:
            y, r = y.astype(np.float16).astype(f32), r16.astype(f32)
            if res == "requantised":
                y, r = quant(y, 2.5) * step(2.5), quant(r, 3.5) * step(3.5)
            y = y + r
        if res is not None and not relu:
            y = np.maximum(y, f32(0))
        got = out.cpu().numpy()
        assert np.array_equal(got[:500], quant(y, 5.0).astype(np.int8)) and (got[500:] == 9).all()


@pytest.mark.parametrize("cin, ld", [(16, 256), (64, 272), (96, 4096), (128, 256), (160, 65536), (64, 1 << 22)])
def test_convolution_of_rows_far_apart(cin, ld):
    """The last one spans 4.8 GB."""
    mx = _mx()
    rng = np.random.default_rng(cin + ld)
    rb, _, n_out, conv, _, _ = conv_case(rng, 1200, (9, 24, 21), cin, 48, (3, 3, 3), (1, 1, 1), (1, 1, 1), True)
    q = mx.quantize_rows(torch.from_numpy(rows(rng, 1200, cin)).to(DEV))
    b = 16 * ((cin + 31) // 32)
    big = torch.empty((1200, ld), dtype=torch.uint8, device=DEV)
    big[:, :b], big[:, b:b + q.scales.shape[1]] = q.codes, q.scales
    if ld < 1 << 20:
        big[:, b + q.scales.shape[1]:] = 0xFF
    far = mx.MxRows(big[:, :b], big[:, b:b + q.scales.shape[1]], cin)
    assert torch.equal(conv.forward(far, rb, n_out), conv.forward(q, rb, n_out))


def test_convolution_nan_rows_reach_their_neighbours_only():
    mx = _mx()
    rng = np.random.default_rng(3)
    rb, table, n_out, conv, _, _ = conv_case(rng, 500, (9, 24, 21), 64, 64, (3, 3, 3), (1, 1, 1), (1, 1, 1), True)
    x = rows(rng, 500, 64)
    x[100, 40] = np.inf
    got = conv.forward(mx.quantize_rows(torch.from_numpy(x).to(DEV)), rb, n_out)
    assert np.array_equal(got.isnan().any(1).cpu().numpy(), (table == 100).any(0))
    assert got.isnan().any(1).equal(got.isnan().all(1))


def test_convolution_device_count_leaves_later_rows():
    mx = _mx()
    rng = np.random.default_rng(4)
    n, grid = 400, (9, 24, 21)
    coords = scene(rng, n, grid)
    idx = torch.from_numpy(np.concatenate([np.zeros((n, 1)), coords], 1).astype(np.int32)).to(DEV)
    rb = mx.Rulebook(n, n, 27)
    num = torch.tensor([150], dtype=torch.int32, device=DEV)
    rb.build_subm(idx, grid, (3, 3, 3), num=num)
    w = rng.standard_normal((32, 3, 3, 3, 64)).astype(np.float16)
    x = rows(rng, n, 64)
    q = mx.quantize_rows(torch.from_numpy(x).to(DEV), num=num)
    out = torch.full((n, 32), 3.0, dtype=torch.float16, device=DEV)
    mx.Conv(w).forward(q, rb, n, out=out)
    _, table = R.neighbours(coords[:150], grid, (3, 3, 3), (1, 1, 1), (1, 1, 1), (1, 1, 1), True)
    y, mag = R.convolution(R.fake(x[:150]), R.fake(w.reshape(32 * 27, 64)).reshape(32, 27, 64), None, table)
    R.within(out[:150].double().cpu().numpy(), y, R.tolerance(y, mag, 27 * 64, 2.0 ** -11))
    assert (out[150:] == 3).all()


def test_convolution_refusals():
    mx = _mx()
    rng = np.random.default_rng(2)
    rb, _, n_out, conv, _, _ = conv_case(rng, 50, (9, 24, 21), 64, 32, (3, 3, 3), (1, 1, 1), (1, 1, 1), True)
    q = mx.quantize_rows(torch.zeros((50, 64), dtype=torch.float16, device=DEV))
    apart = mx.MxRows(q.codes.contiguous(), q.scales.contiguous(), 64)
    with pytest.raises(ValueError):
        conv.forward(apart, rb, n_out)
    with pytest.raises(ValueError):
        conv.forward(q, rb, n_out - 1)
    with pytest.raises(ValueError):
        conv.forward(mx.quantize_rows(torch.zeros((49, 64), dtype=torch.float16, device=DEV)), rb, n_out)
    with pytest.raises(ValueError):
        conv.forward(q, mx.Rulebook(50, 50, 27), n_out)
    wide = mx.Conv(np.zeros((32, 3, 3, 3, 160), np.float16))
    with pytest.raises(RuntimeError):                                     # microscaled output of a wide layer
        wide.forward(mx.quantize_rows(torch.zeros((50, 160), dtype=torch.float16, device=DEV)), rb, n_out, out=mx.MxRows.empty(n_out, 32, DEV))
    with pytest.raises(ValueError):
        conv.forward(q, rb, n_out, out=mx.MxRows.empty(n_out, 64, DEV))
    same = mx.Conv(np.zeros((64, 3, 3, 3, 64), np.float16))
    with pytest.raises(RuntimeError):                                     # in place
        same.forward(q, rb, n_out, out=q)
    rb.index, there = rb.index + 1, rb.index                              # (a rulebook of another device)
    with pytest.raises(ValueError):
        conv.forward(q, rb, n_out)
    with pytest.raises(ValueError):
        rb.build_subm(torch.zeros((5, 4), dtype=torch.int32, device=DEV), (9, 24, 21), (3, 3, 3))
    rb.index = there
    with pytest.raises(RuntimeError):                                     # kernel volume
        mx.Conv(np.zeros((32, 1, 1, 1, 64), np.float16)).forward(q, rb, n_out)


# ------------------------------------------------------------------------------------------------- together
def test_layers_in_a_row_captured_and_replayed():
    """quantise -> convolution -> linear with residual -> dequantised copy, captured once and replayed on other rows."""
    mx = _mx()
    rng = np.random.default_rng(8)
    rb, _, n_out, conv, _, _ = conv_case(rng, 800, (9, 24, 21), 64, 64, (3, 3, 3), (1, 1, 1), (1, 1, 1), True)
    w, _ = mx_rows(rng, 200, 64)
    bias = torch.randn(200, device=DEV)
    x = torch.zeros((800, 64), dtype=torch.float16, device=DEV)
    q = mx.MxRows.empty(800, 64, DEV)
    y = torch.empty((800, 64), dtype=torch.float16, device=DEV)
    z = torch.empty((800, 200), dtype=torch.float16, device=DEV)
    one = torch.empty((1, 200), dtype=torch.float32, device=DEV)
    ws = torch.empty(800 * mx.row_bytes(64), dtype=torch.uint8, device=DEV)

    def step():
        conv.forward(mx.quantize_rows(x, out=q), rb, n_out, relu=True, out=y)
        mx.product(y, w, bias=bias, relu=True, out=z, workspace=ws)
        mx.product(y[:1], w, bias=bias, out=one)

    x.copy_(torch.from_numpy(rows(rng, 800, 64)).to(DEV))
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for i in range(4):
        x.copy_(torch.from_numpy(rows(rng, 800, 64)).to(DEV))
        g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, z, one)]
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (y, z, one)):
            assert torch.equal(a, b), i
