"""The GCN driver on 8-bit rows and with group norm (run with -m gpu).

--features int8 against the exact layers in 64 bits, within the bound that the held
steps allow, carried through the layers element by element: a value held in 8 bits is
off by at most half a step of its row, s / 2 (plus what it was off before), where
s <= (max|v| + its error) / 127; an aggregation carries errors with its weights; a
product adds |x| * sw / 2 for the weights; ReLU carries errors as they are. fp32
roundings are 2^-24 against 2^-8 and are covered by 0.1 % on top.

With a norm in between, the driver's result is compared bit for bit with the same calls
made one by one.
"""
import numpy as np
import pytest
import torch

from gnn_cuda_b200 import synth
from gnn_cuda_b200.GNN_cuda_common import agg_ops, gcn_inference, gcn_ops, int8_ops, norm_ops, npz_utils

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.fixture(scope="module")
def graph_dir(tmp_path_factory):
    d = tmp_path_factory.mktemp("graphs8")
    u, v = synth.rmat_undirected(3000, 24000, seed=41)
    s, t = synth.symmetrize(u, v)
    npz_utils.save_graph_npz(str(d / "rmat3k.npz"), s.numpy(), t.numpy(), 3000)
    return d


def _run(graph_dir, *extra):
    cap = {}
    rc = gcn_inference.run_gcn_inference(
        framework_label="pyg", select_device=npz_utils.select_device,
        load_graph_features=npz_utils.load_pyg_graph_features_from_npz, load_kind="pyg",
        argv=["--dataset", "rmat3k", "--data_root", str(graph_dir), "--dim", "72", "--num_layers", "3", "--warmup",
              "1", "--iters", "2", "--seed", "5", "--memory_mode", "device", *extra], capture=cap)
    assert rc == 0
    return cap


def _np(t):
    return t.detach().cpu().numpy()


def _held(v, err):
    """(v, err) of rows held in 8 bits."""
    return v, err + ((np.abs(v) + err).max(1, keepdims=True) / 127) / 2


@pytest.mark.parametrize("impl", ["legacy_fused", "pyg_baseline"])
def test_int8_features_within_the_held_steps(graph_dir, impl, capsys):
    import scipy.sparse as sp
    cap = _run(graph_dir, "--features", "int8", "--gcn_kernel_impl", impl)
    assert "Feature Rows:\tint8" in capsys.readouterr().out
    rp, ci = _np(cap["row_ptr"]), _np(cap["col_ind"])
    n = len(rp) - 1
    if impl == "legacy_fused":
        dis = _np(cap["deg_inv_sqrt"]).astype(np.float64)
        val = dis[np.repeat(np.arange(n), np.diff(rp))] * dis[ci]
    else:
        val = _np(cap["edge_weight"]).astype(np.float64)
    a = sp.csr_matrix((val, ci, rp), shape=(n, n), copy=True)
    x = _np(cap["features"]).astype(np.float64)
    x, err = _held(x, np.zeros_like(x))
    for i, layer in enumerate(cap["layers"]):
        w, b = _np(layer.weight).astype(np.float64), _np(layer.bias).astype(np.float64)
        sw = np.abs(w).max(0) / 127
        g, ge = _held(a @ x, abs(a) @ err)
        x = g @ w + b
        err = ge @ np.abs(w) + (np.abs(g) + ge).sum(1, keepdims=True) * sw / 2
        if i < len(cap["layers"]) - 1:
            x, err = _held(np.maximum(x, 0), err)
    got = _np(cap["output"]).astype(np.float64)
    assert np.all(np.abs(got - x) <= 1.001 * err)
    assert np.linalg.norm(got - x) <= 0.05 * np.linalg.norm(x)  # and far inside it: half steps do not add up


@pytest.mark.parametrize("norm", ["node", "graph"])
@pytest.mark.parametrize("features", ["fp32", "int8"])
def test_norm_equals_the_calls_one_by_one(graph_dir, norm, features, capsys):
    cap = _run(graph_dir, "--features", features, "--norm", norm, "--norm_groups", "6", "--no-tf32")
    assert f"Norm:\t{norm} (6 groups)" in capsys.readouterr().out
    rp, ci, dis = (cap[k].to(DEV) for k in ("row_ptr", "col_ind", "deg_inv_sqrt"))
    x = cap["features"].to(DEV)
    n = x.size(0)
    ptr = torch.tensor([0, n], device=DEV) if norm == "graph" else None
    for i, layer in enumerate(cap["layers"]):
        agg, out = torch.empty(n, x.size(1), device=DEV), torch.empty(n, layer.weight.size(1), device=DEV)
        if features == "int8":
            q, s = int8_ops.empty_rows(n, x.size(1), DEV), torch.empty(n, device=DEV)
            int8_ops.quantize_rows_(x, q, s)
            wq, ws = int8_ops.empty_rows(out.size(1), x.size(1), DEV), torch.empty(out.size(1), device=DEV)
            int8_ops.quantize_weight_(layer.weight, wq, ws)
            int8_ops.spmm_int8_forward_(rp, ci, q, s, agg, "gcn", deg_inv_sqrt=dis)
            int8_ops.linear_int8_forward_(agg, None, wq, ws, layer.bias, out)
        else:
            gcn_ops.spmm_gcn_forward_(rp, ci, dis, x, agg, spmm_mode="plain")
            agg_ops.linear_forward_(agg, layer.weight, layer.bias, out, False)
        if i < len(cap["layers"]) - 1:
            norm_ops.group_norm_forward_(out, 6, None, None, out, graph_ptr=ptr, activation="relu")
        x = out
    assert torch.equal(x.cpu(), cap["output"])


def test_layer_run_captured_and_replayed():
    """Quantise, aggregate, transform to 8 bits, transform to fp32, normalise: one captured graph."""
    n, f = 2000, 64
    g = torch.Generator(device=DEV).manual_seed(3)
    deg = torch.randint(0, 20, (n,), device=DEV, generator=g)
    rp = torch.cat([deg.new_zeros(1), deg.cumsum(0)]).to(torch.int32)
    ci = torch.randint(0, n, (int(rp[-1]),), device=DEV, generator=g).to(torch.int32)
    x = torch.randn(n, f, device=DEV, generator=g)
    q, s = int8_ops.empty_rows(n, f, DEV), torch.empty(n, device=DEV)
    h, hs = int8_ops.empty_rows(n, f, DEV), torch.empty(n, device=DEV)
    wq, ws = int8_ops.empty_rows(f, f, DEV), torch.empty(f, device=DEV)
    int8_ops.quantize_weight_(torch.randn(f, f, device=DEV, generator=g), wq, ws)
    agg, out = torch.empty(n, f, device=DEV), torch.empty(n, f, device=DEV)
    ptr = torch.tensor([0, 500, 2000], device=DEV)

    def layer():
        int8_ops.quantize_rows_(x, q, s)
        int8_ops.spmm_int8_forward_(rp, ci, q, s, agg, "mean")
        int8_ops.linear_int8_forward_(agg, None, wq, ws, None, h, True, out_scale=hs)
        int8_ops.linear_int8_forward_(h, hs, wq, ws, None, out)
        norm_ops.group_norm_forward_(out, 4, None, None, out, graph_ptr=ptr, activation="silu")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # on another stream than the default one
        layer()
    torch.cuda.current_stream().wait_stream(side)
    want = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for _ in range(3):
        out.fill_(float("nan"))
        graph.replay()
        assert torch.equal(out, want)
    x.mul_(-0.5)  # new inputs in the same place
    graph.replay()
    got = out.clone()
    layer()
    assert torch.equal(got, out) and not torch.equal(got, want)
