"""Microscaled 4-bit rows in float64, from the definition: the oracle of the MXFP4 tests."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """[n, c] -> (codes uint8 [n, 16 * blocks], scales uint8 [n, round_up(blocks, 4)])."""
    x = np.asarray(x, np.float64)
    n, c = x.shape
    blocks = -(-c // 32)
    v = np.zeros((n, 32 * blocks))
    v[:, :c] = x
    v = v.reshape(n, blocks, 32)
    top = np.abs(v).max(2)
    bad = ~np.isfinite(v).all(2)
    e = np.maximum(np.frexp(np.where(bad, 1.0, top))[1] - 3, -127)      # floor(log2 top) - 2
    e = np.where(top == 0, -127, e)
    with np.errstate(over="ignore", invalid="ignore"):
        a = np.abs(v) / np.ldexp(1.0, e)[:, :, None]
    dist = np.abs(np.where(bad[:, :, None], 0.0, a)[..., None] - LEVELS)
    best = dist.min(-1, keepdims=True)
    near = dist == best                                             # two of them on a tie: take the even code
    code = np.where(near.sum(-1) == 2, np.where(near.argmax(-1) % 2 == 0, near.argmax(-1), near.argmax(-1) + 1), near.argmax(-1))
    code = np.where(bad[:, :, None], 0, code | np.where(np.signbit(v), 8, 0)).reshape(n, 32 * blocks).astype(np.uint8)
    scales = np.zeros((n, -(-blocks // 4) * 4), np.uint8)
    scales[:, :blocks] = np.where(bad, 255, e + 127)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def values(codes, scales, c):
    """The numbers microscaled rows stand for, [n, c] float64."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    n = codes.shape[0]
    blocks = -(-c // 32)
    code = np.stack([codes[:, :16 * blocks] & 15, codes[:, :16 * blocks] >> 4], 2).reshape(n, blocks, 32)
    s = scales[:, :blocks].astype(np.int64)
    x = np.where(s == 255, np.nan, np.ldexp(1.0, np.where(s == 255, 0, s - 127)))
    level = np.where(code & 8, -1.0, 1.0) * LEVELS[code & 7]
    return (level * x[:, :, None]).reshape(n, 32 * blocks)[:, :c]


def fake(x):
    return values(*quantize(x), np.asarray(x).shape[1])


def product(a, b, bias=None, relu=False, res=None, relu2=False):
    """(y, sum of |a| |b| + |bias| + |res|: what rounding errors scale with)."""
    y, mag = a @ b.T, np.abs(a) @ np.abs(b).T
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    if relu:
        y = np.where(y > 0, y, 0.0)
    if res is not None:
        y, mag = y + res, mag + np.abs(res)
    return (np.where(y > 0, y, 0.0) if relu2 else y), mag


def tolerance(y, mag, terms, out_eps):
    """Sums of `terms` products held in fp32: each addition is off by at most 2^-23 of a partial sum (<= mag) whichever way
    the matrix core rounds; the products themselves are exact (4 significant bits).  Then half a step of the output type,
    or half its smallest subnormal."""
    tiny = {2.0 ** -11: 2.0 ** -25, 2.0 ** -24: 2.0 ** -150}[out_eps]
    return (terms + 4) * 2.0 ** -23 * mag * 1.001 + out_eps * np.abs(y) * 1.001 + tiny


def within(got, y, tol):
    """got is y up to tol; a value that rounds past the largest fp16 number (65504, half a step above it: 65520) is an
    infinity of its sign."""
    over = np.isinf(got) & (np.sign(got) == np.sign(y)) & (np.abs(y) + tol >= 65520.0)
    with np.errstate(invalid="ignore"):
        good = over | (np.abs(got - y) <= tol)
    worst = np.unravel_index(np.argmin(good), good.shape) if good.size else ()
    assert good.all(), (f"{(~good).sum()} of {good.size} values off, first at {worst}: {got[worst]} for {y[worst]}, tolerance {tol[worst]}")


def neighbours(coords, grid, ksize, stride, padding, dilation, subm):
    """(output coordinates, table [kvol][n_out]) of a sparse convolution by dictionary look-ups; coords [n, 3]."""
    where = {}
    for i, c in enumerate(map(tuple, coords.tolist())):
        where.setdefault(c, i)
    out_grid = [(grid[a] + 2 * padding[a] - dilation[a] * (ksize[a] - 1) - 1) // stride[a] + 1 for a in range(3)]
    offsets = [(a, b, c) for a in range(ksize[0]) for b in range(ksize[1]) for c in range(ksize[2])]
    if subm:
        stride, padding = (1, 1, 1), [dilation[a] * (ksize[a] // 2) for a in range(3)]
        outs = [tuple(c) for c in coords.tolist()]
    else:
        outs = set()
        for c in coords.tolist():
            for k in offsets:
                t = [c[a] + padding[a] - k[a] * dilation[a] for a in range(3)]
                if all(t[a] % stride[a] == 0 and 0 <= t[a] // stride[a] < out_grid[a] for a in range(3)):
                    outs.add(tuple(t[a] // stride[a] for a in range(3)))
        outs = sorted(outs)
    table = np.full((len(offsets), len(outs)), -1, np.int64)
    for j, o in enumerate(outs):
        for k, off in enumerate(offsets):
            table[k, j] = where.get(tuple(o[a] * stride[a] - padding[a] + off[a] * dilation[a] for a in range(3)), -1)
    return np.array(outs, np.int64).reshape(-1, 3), table


def convolution(x, w, bias, table):
    """x: values [n_in, cin]; w: values [cout, kvol, cin]; -> (y, magnitude) [n_out, cout]."""
    pad = np.concatenate([x, np.zeros((1, x.shape[1]))])
    y = np.zeros((table.shape[1], w.shape[0]))
    mag = np.zeros_like(y)
    for k in range(table.shape[0]):
        y += pad[table[k]] @ w[:, k].T
        mag += np.abs(pad[table[k]]) @ np.abs(w[:, k]).T
    if bias is not None:
        y, mag = y + bias, mag + np.abs(bias)
    return y, mag
