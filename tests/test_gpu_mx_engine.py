"""The engine at precision mxfp4: every layer from the engine's own input of that layer, against the float64 oracle."""
import numpy as np
import pytest
import torch

from lidar_ai_solution_amd import capi, graphs, onnx_dialect
from tests import mx_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
GRID = (17, 40, 36)


def frame(seed, n=1200, channels=5, grid=GRID):
    rng = np.random.default_rng(seed)
    cells = np.sort(rng.choice(grid[0] * grid[1] * grid[2] // 3, n, replace=False))    # the lower third: dense enough for neighbours
    idx = np.stack([0 * cells, cells // (grid[1] * grid[2]), cells // grid[2] % grid[1], cells % grid[2]], 1).astype(np.int32)
    feats = (rng.standard_normal((n, channels)) * [20, 20, 2, 0.5, 0.1][:channels]).astype(np.float16)
    return torch.from_numpy(feats).to(DEV), torch.from_numpy(idx).to(DEV)


def run(eng, f, i, grid=GRID):
    eng.set_input(f, i, grid)
    eng.forward()
    torch.cuda.synchronize()
    return eng


def bits(view):
    t = view.torch()
    t = t if view.dense else t[0]
    return t.cpu().numpy().view(np.uint16)


def tensor(eng, name, f, i):
    """(values float64 [n, c], coordinates [n, 3], dtype) of a kept tensor or of the input."""
    if name == "0":
        return f.double().cpu().numpy(), i.cpu().numpy()[:, 1:], capi.DTYPE_FP16
    view, _ = eng.tensor(name)
    t, idx = view.torch()
    v = t.double().cpu().numpy()
    return (v * np.float32(view.scale) if view.dtype == capi.DTYPE_INT8 else v), idx.cpu().numpy()[:, 1:], view.dtype


def table_of(attrs, cin_xyz, cout_xyz):
    ks, st, pd = attrs["kernel_size"], attrs["stride"], attrs["padding"]
    if attrs["subm"]:
        st, pd = [1, 1, 1], [k // 2 for k in ks]
    where = {tuple(c): r for r, c in enumerate(cin_xyz.tolist())}
    offs = [(a, b, c) for a in range(ks[0]) for b in range(ks[1]) for c in range(ks[2])]
    table = np.full((len(offs), len(cout_xyz)), -1, np.int64)
    for k, off in enumerate(offs):
        for r, o in enumerate(cout_xyz.tolist()):
            if attrs.get("inverse"):    # the strided convolution's pairs with the two sides swapped
                t = [o[a] + pd[a] - off[a] for a in range(3)]
                if all(t[a] % st[a] == 0 for a in range(3)):
                    table[k, r] = where.get(tuple(t[a] // st[a] for a in range(3)), -1)
            else:
                table[k, r] = where.get(tuple(o[a] * st[a] - pd[a] + off[a] for a in range(3)), -1)
    return table


def check_layers(graph, eng, f, i, mx_nodes):
    seen = 0
    for n in graph.nodes:
        if n.op_type == "SparseConvolution":
            x, xi, dtype = tensor(eng, n.inputs[0], f, i)
            got, oi, _ = tensor(eng, n.outputs[0], f, i)
            w = graph.initializers[n.inputs[1]]
            b = graph.initializers[n.inputs[2]].astype(np.float64)
            cout, cin, kv = w.shape[0], w.shape[4], int(np.prod(w.shape[1:4]))
            if n.name not in mx_nodes:
                continue
            xv = R.fake(x[:, :cin].astype(np.float32))
            y, mag = R.convolution(xv, R.fake(w.reshape(cout * kv, cin)).reshape(cout, kv, cin), b, table_of(n.attrs, xi, oi))
            y = np.where(y > 0, y, 0) if n.attrs["activation"] == "ReLU" else y
            R.within(got[:, :cout], y, R.tolerance(y, mag, kv * cin, 2.0 ** -11))
            seen += 1
        elif n.op_type in ("Add", "Relu"):
            a, _, da = tensor(eng, n.inputs[0], f, i)
            got, _, dt = tensor(eng, n.outputs[0], f, i)
            if dt != capi.DTYPE_FP16 or da != capi.DTYPE_FP16:
                continue
            if n.op_type == "Add":
                a = (a.astype(np.float32) + tensor(eng, n.inputs[1], f, i)[0].astype(np.float32)).astype(np.float16)
            else:
                a = np.maximum(a, 0)
            assert np.array_equal(got, a.astype(np.float64)), n.name
    return seen


def mark(graph, precision):
    names = []
    for n in graph.nodes:
        if n.op_type == "SparseConvolution":
            n.attrs["precision"] = precision
            names.append(n.name)
    return names


@pytest.mark.parametrize("maker", [graphs.centerpoint_scn, graphs.unet_scn])
@pytest.mark.parametrize("marked", ["mxfp4", "int8"])
def test_every_layer(maker, marked):
    from lidar_ai_solution_amd.scn import Engine
    g, _ = maker(seed=3, weight_std=0.08)
    if maker is graphs.centerpoint_scn:
        g.nodes = [n for n in g.nodes if n.op_type not in ("ScatterDense", "Reshape")]
        g.outputs = [g.nodes[-1].outputs[0]]
    names = mark(g, marked)
    f, i = frame(1)
    kept = run(Engine.from_graph(g, "mxfp4", keep_all=True), f, i)
    assert check_layers(g, kept, f, i, names) == len(names) > 8
    want = bits(kept.output(0))
    fused = Engine.from_graph(g, "mxfp4")
    assert np.array_equal(bits(run(fused, f, i).output(0)), want)
    aux = Engine.from_graph(g, "mxfp4", with_auxiliary_stream=True)
    for seed in (2, 1):                                                  # another frame in between
        run(aux, *frame(seed, 900 if seed == 2 else 1200))
    assert np.array_equal(bits(aux.output(0)), want)


def test_plan_keeps_the_unmarked_layers_in_fp16(tmp_path):
    """The CenterPoint int8 plan at precision mxfp4: the layers it leaves in fp16 give the fp16 engine's bits."""
    from lidar_ai_solution_amd.scn import Engine
    g, tags = graphs.centerpoint_scn(seed=5, weight_std=0.08)
    amax = {t: 1.0 for t in ["0"] + [n.outputs[0] for n in g.nodes]}
    graphs.apply_int8_plan(g, tags, amax, "centerpoint")
    f, i = frame(3, grid=(41, 40, 40))
    mx = run(Engine.from_graph(g, "mxfp4", keep_all=True), f, i, (41, 40, 40))
    half = run(Engine.from_graph(g, "fp16", keep_all=True), f, i, (41, 40, 40))
    same = {tags.get(n.name): np.array_equal(bits(mx.tensor(n.outputs[0])[0]), bits(half.tensor(n.outputs[0])[0]))
            for n in g.nodes if n.op_type == "SparseConvolution"}
    assert same["conv_input"] and same["conv1.0.conv1"] and same["conv1.0.conv2"] and not same["conv1.1.conv1"]
    path = str(tmp_path / "m.scn.onnx")
    onnx_dialect.save(g, path)
    loaded = run(Engine.from_onnx(path, "mxfp4"), f, i, (41, 40, 40))
    assert np.array_equal(bits(loaded.output(0)), bits(mx.output(0)))


def test_marks_and_overrides(tmp_path):
    """A layer marked mxfp4 in an int8 engine, in an fp16 engine (ignored), and by override."""
    from lidar_ai_solution_amd.scn import Engine
    g, tags = graphs.unet_scn(seed=7, weight_std=0.08)
    plain = run(Engine.from_graph(g, "fp16"), *frame(4))
    path = str(tmp_path / "plain.scn.onnx")
    onnx_dialect.save(g, path)
    over = run(Engine.from_onnx(path, "mxfp4", precision_overrides=[("SparseConvolution", True, "mxfp4", None)]), *frame(4))
    assert np.array_equal(bits(run(Engine.from_onnx(path, "mxfp4"), *frame(4)).output(0)), bits(plain.output(0)))
    names = mark(g, "mxfp4")
    assert np.array_equal(bits(run(Engine.from_graph(g, "fp16"), *frame(4)).output(0)), bits(plain.output(0)))
    assert np.array_equal(bits(run(Engine.from_graph(g, "mxfp4"), *frame(4)).output(0)), bits(over.output(0)))
    onnx_dialect.save(g, path)
    assert np.array_equal(bits(run(Engine.from_onnx(path, "mxfp4"), *frame(4)).output(0)), bits(over.output(0)))
    # int8 everywhere but two layers
    f, i = frame(4)
    kept = run(Engine.from_graph(g, "fp16", keep_all=True), f, i)
    amax = {"0": 60.0, **{n.outputs[0]: float(np.abs(tensor(kept, n.outputs[0], f, i)[0]).max()) for n in g.nodes}}
    graphs.apply_int8_plan(g, tags, amax, "all-int8")
    chosen = [names[2], names[6]]
    for n in g.nodes:
        if n.name in chosen:
            n.attrs["precision"] = "mxfp4"
    mixed = run(Engine.from_graph(g, "int8", keep_all=True), f, i)
    got = {}
    for n in g.nodes:
        if n.name in chosen:
            x, xi, dt = tensor(mixed, n.inputs[0], f, i)
            y8, oi, _ = tensor(mixed, n.outputs[0], f, i)
            w, b = graph_weights(g, n)
            cout, cin, kv = w.shape[0], w.shape[4], int(np.prod(w.shape[1:4]))
            y, mag = R.convolution(R.fake(x[:, :cin].astype(np.float32)), R.fake(w.reshape(cout * kv, cin)).reshape(cout, kv, cin), b,
                                   table_of(n.attrs, xi, oi))
            y = np.where(y > 0, y, 0) if n.attrs["activation"] == "ReLU" else y
            view, _ = mixed.tensor(n.outputs[0])
            got[n.name] = (dt, view.dtype)
            if view.dtype == capi.DTYPE_INT8:                            # clamped to the range, then half a step of its grid
                r = float(view.dynamic_range)
                y = np.clip(y, -r, r)
                R.within(y8[:, :cout], y, R.tolerance(y, mag, kv * cin, 2.0 ** -24) + r / 127 * (0.5 + 127 * 2.0 ** -22))
            else:
                R.within(y8[:, :cout], y, R.tolerance(y, mag, kv * cin, 2.0 ** -11))
    assert len(got) == 2


def graph_weights(g, n):
    return g.initializers[n.inputs[1]], g.initializers[n.inputs[2]].astype(np.float64)


def test_captured_engine_replays_on_other_frames():
    from lidar_ai_solution_amd.scn import Engine
    g, _ = graphs.unet_scn(seed=11, weight_std=0.08)
    mark(g, "mxfp4")
    eng, fresh = Engine.from_graph(g, "mxfp4"), Engine.from_graph(g, "mxfp4")
    f = torch.zeros((1500, 5), dtype=torch.float16, device=DEV)
    i = torch.zeros((1500, 4), dtype=torch.int32, device=DEV)
    num = torch.zeros(1, dtype=torch.int32, device=DEV)

    def put(seed, n):
        a, b = frame(seed, n)
        f[:n], i[:n], num[0] = a, b, n
        return a, b

    put(0, 1000)
    eng.set_input(f, i, GRID)
    eng.set_dds_num_of_points_pointer(num)
    capi.check(capi.lib().scn_engine_prepare(eng._h, capi.i3(*GRID)))
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        eng.forward()
    for seed, n in ((1, 700), (2, 1500), (3, 1), (4, 1100)):
        a, b = put(seed, n)
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(bits(eng.output(0)), bits(run(fresh, a, b).output(0))), n
