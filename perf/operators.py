"""Workloads of the 8-bit inference path and of group normalisation.

Three operators, each in its plain form (elementary torch operations) and as the
calls a program makes of the framework:

  linear   y = relu?(x·W + b) with x and W in signed 8-bit integers, one scale per
           row of x and one per output channel. x is either held in 8 bits, or
           fp32 and quantised row by row on the way; `form` "mlp" is two of them
           with the hidden layer held in 8 bits.
  norm     group normalisation with an activation over [nodes, channels]: each node
           on its own, or the nodes of each graph of a batch together.
  spmm     neighbour aggregation over a CSR whose feature rows are held in 8 bits
           with one scale per row.

Quantisation of a row v: s = max|v| / 127 in 32 bits, q = v / s rounded to the
nearest integer, ties to even (decided on the exact quotient); a row of zeros has
s = 0 and q = 0, a row that holds a NaN or an infinity has s = NaN and q = 0.
The transform's result is a 32-bit value after each of its steps,
((float(sum of products)) * row scale) * channel scale + bias: what is quantised
again afterwards is that value.
"""
import math

import torch

own = False

DEV = "cuda"


# --- cases -------------------------------------------------------------------

def listed():
    return [
        # one new node's features through one layer: latency
        {"name": "linear_one_node", "op": "linear", "form": "dynamic", "m": 1, "k": 512, "n": 512, "relu": True},
        # citation graph: sparse word features of odd width, one column per class
        {"name": "linear_classes_odd", "op": "linear", "form": "static", "m": 19717, "k": 501, "n": 47,
         "relu": False},
        # first layer over the stored 8-bit features of a product graph
        {"name": "linear_products", "op": "linear", "form": "static", "m": 2449029, "k": 128, "n": 128,
         "relu": True},
        # a layer's two-transform MLP over fp32 aggregates, hidden layer in 8 bits
        {"name": "mlp_hidden_int8", "op": "linear", "form": "mlp", "m": 232965, "k": 256, "n": 256, "relu": True},
        # wide features: bound by the matrix units
        {"name": "linear_wide", "op": "linear", "form": "static", "m": 16384, "k": 4096, "n": 4096, "relu": False},
        # one small molecule-sized graph: latency
        {"name": "norm_one_graph", "op": "norm", "mode": "batch", "rows": 30, "graphs": 1, "c": 128, "groups": 1,
         "act": "relu"},
        # every node of a social graph on its own
        {"name": "norm_nodes", "op": "norm", "mode": "node", "rows": 232965, "graphs": 0, "c": 256, "groups": 16,
         "act": "silu"},
        # a training-set batch of small graphs, ragged, some empty, rows of padding behind the last
        {"name": "norm_batch", "op": "norm", "mode": "batch", "rows": 200003, "graphs": 8192, "c": 100, "groups": 4,
         "act": "gelu"},
        # one whole product graph as a single sample
        {"name": "norm_whole_graph", "op": "norm", "mode": "batch", "rows": 2449029, "graphs": 1, "c": 128,
         "groups": 8, "act": "relu"},
        # citation graph, one layer's normalised aggregation
        {"name": "spmm_citation", "op": "spmm", "agg": "gcn", "nodes": 19717, "entries": 108365, "f": 128},
        # mean over the neighbours of a dense graph, feature width odd
        {"name": "spmm_mean_odd", "op": "spmm", "agg": "mean", "nodes": 23297, "entries": 5730794, "f": 201},
        # a quarter of a product graph
        {"name": "spmm_products_quarter", "op": "spmm", "agg": "gcn", "nodes": 612257, "entries": 16077042,
         "f": 128},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "norm", "spmm"])
    if op == "linear":
        form = rng.choice(["static", "dynamic", "mlp"])
        k, n = _log(rng, 16, 4096), _log(rng, 7, 4096)
        if form == "mlp":
            k, n = min(k, 640), min(n, 256)
        m = _log(rng, 1, max(2, min(1500000, (1 << 37) // (k * n), (1 << 28) // (k + n))))
        return {"op": op, "form": form, "m": m, "k": k, "n": n, "relu": rng.random() < 0.5}
    if op == "norm":
        mode = rng.choice(["node", "batch"])
        groups = rng.choice([1, 2, 3, 4, 8, 16, 32])
        c = groups * _log(rng, max(1, 8 // groups), 512 // groups)
        rows = _log(rng, 1, min(2000000, (1 << 28) // c))
        graphs = 0 if mode == "node" else _log(rng, 1, max(1, min(rows, 20000)))
        return {"op": op, "mode": mode, "rows": rows, "graphs": graphs, "c": c, "groups": groups,
                "act": rng.choice(["none", "relu", "silu", "gelu"])}
    f = _log(rng, 8, 512)
    nodes = _log(rng, 500, 600000)
    entries = min(int(nodes * math.exp(rng.uniform(0.0, math.log(50)))), 16000000 * 128 // f, 16000000)
    return {"op": op, "agg": rng.choice(["gcn", "weighted", "sum", "mean"]), "nodes": nodes, "entries": entries,
            "f": f}


def work(case):
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        x = m * (k + 4) if case["form"] == "static" else 4 * m * k
        weights = n * k + 8 * n
        flops = 2 * m * k * n
        if case["form"] == "mlp":
            weights += n * n + 8 * n
            flops += 2 * m * n * n
        return {"bytes": x + weights + 4 * m * n, "flops": flops}
    if case["op"] == "norm":
        return {"bytes": 8 * case["rows"] * case["c"] + 8 * case["c"], "flops": 8 * case["rows"] * case["c"]}
    n, e, f = case["nodes"], case["entries"], case["f"]
    extra = {"gcn": 4 * n, "weighted": 4 * e, "sum": 0, "mean": 0}[case["agg"]]
    return {"bytes": 4 * (n + 1) + 4 * e + extra + n * (f + 4) + 4 * n * f, "flops": 2 * e * f}


# --- inputs --------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _features(rows, cols, g):
    """Rows of different magnitude, as aggregates of different degree have, some of them zero."""
    x = torch.randn(rows, cols, device=DEV, generator=g)
    x *= torch.exp(torch.randn(rows, 1, device=DEV, generator=g))
    x *= torch.rand(rows, 1, device=DEV, generator=g) > 0.01
    return x


def _rows8(rows, cols):
    """Storage for 8-bit rows: each starts on a 16-byte boundary."""
    return torch.empty(rows, (cols + 15) // 16 * 16, dtype=torch.int8, device=DEV)[:, :cols]


def _stored8(v):
    q, s = _quantize(v)
    held = _rows8(v.shape[0], v.shape[1])
    held.copy_(q)
    return held, s


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": dict(case)}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        x = _features(m, k, g)
        if case["form"] == "static":
            st["x"], st["sx"] = _stored8(x)
        else:
            st["x"], st["sx"] = x, None
        # 8-bit weights, one row and one scale per output channel, laid out once when a model is loaded
        st["w"], st["sw"] = _stored8(torch.randn(n, k, device=DEV, generator=g) / math.sqrt(k))
        st["b"] = torch.randn(n, device=DEV, generator=g) * 0.1
        if case["form"] == "mlp":
            st["w2"], st["sw2"] = _stored8(torch.randn(n, n, device=DEV, generator=g) / math.sqrt(n))
            st["b2"] = torch.randn(n, device=DEV, generator=g) * 0.1
            st["h"], st["sh"] = _rows8(m, n), torch.empty(m, device=DEV)
        st["out"] = torch.empty(m, n, device=DEV)
        return st
    if case["op"] == "norm":
        rows, c = case["rows"], case["c"]
        x = torch.randn(rows, c, device=DEV, generator=g)
        x = x * (0.5 + torch.rand(c, device=DEV, generator=g)) + torch.randn(c, device=DEV, generator=g)
        st["x"] = x.contiguous()
        st["w"] = 1.0 + 0.2 * torch.randn(c, device=DEV, generator=g)
        st["b"] = 0.2 * torch.randn(c, device=DEV, generator=g)
        st["ptr"] = None
        if case["mode"] == "batch":
            # ragged graphs; with more than one, the last rows belong to none (padding)
            graphs = case["graphs"]
            end = rows if graphs == 1 else rows - rows // 50
            cuts = torch.randint(0, end + 1, (graphs - 1,), device=DEV, generator=g).sort().values
            zero = torch.zeros(1, dtype=torch.int64, device=DEV)
            st["ptr"] = torch.cat([zero, cuts, zero + end]).to(torch.int32)
        st["out"] = torch.randn(rows, c, device=DEV, generator=g)
        return st
    n, e, f = case["nodes"], case["entries"], case["f"]
    # skewed degrees on both sides: a few hubs, some nodes without neighbours
    perm = torch.randperm(n, device=DEV, generator=g)
    dst = perm[(torch.rand(e, device=DEV, generator=g, dtype=torch.float64).square() * n).long().clamp_(max=n - 1)]
    src = perm[(torch.rand(e, device=DEV, generator=g, dtype=torch.float64).square() * n).long().clamp_(max=n - 1)]
    key = (dst * n + src).sort().values
    deg = torch.bincount(key // n, minlength=n)
    st["row_ptr"] = torch.cat([deg.new_zeros(1), deg.cumsum(0)]).to(torch.int32)
    st["col"] = (key % n).to(torch.int32)
    st["dis"] = deg.clamp(min=1).double().rsqrt().float() if case["agg"] == "gcn" else None
    st["ew"] = torch.rand(e, device=DEV, generator=g) if case["agg"] == "weighted" else None
    st["x"], st["sx"] = _stored8(_features(n, f, g))
    st["out"] = torch.empty(n, f, device=DEV)
    return st


# --- plain forms ----------------------------------------------------------------

def _quantize(v):
    """Values in -127..127 (64 bits, so that no quotient next to a border is misjudged) and the 32-bit scales."""
    s = (v.abs().amax(dim=1).double() / 127.0).float()
    bad = ~torch.isfinite(s)
    s = torch.where(bad, torch.full_like(s, float("nan")), s)
    none = (bad | (s == 0)).unsqueeze(1)
    q = torch.round(v.double() / s.double().unsqueeze(1)).clamp(-127.0, 127.0)
    return torch.where(none, torch.zeros_like(q), q), s


def _linear(q, sx, w, sw, b, relu):
    acc = (q.double() @ w.double().t()).float()  # sums of products of whole numbers: 32 bits would round long ones
    y = (acc * sx.unsqueeze(1)) * sw.unsqueeze(0) + b.unsqueeze(0)
    return torch.where(y < 0, torch.zeros_like(y), y) if relu else y


def _activate(y, act):
    if act == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y


def _norm(st):
    case, x = st["case"], st["x"]
    rows, c, groups = case["rows"], case["c"], case["groups"]
    xg = x.double().view(rows, groups, c // groups)  # sums over millions of values: 64 bits
    if st["ptr"] is None:
        d = xg - xg.sum(2, keepdim=True) / (c // groups)
        var = (d * d).sum(2, keepdim=True) / (c // groups)
        y = (d / torch.sqrt(var + 1e-5)).view(rows, c).float() * st["w"] + st["b"]
        return _activate(y, case["act"])
    ptr = st["ptr"].long()
    at = torch.arange(rows, device=x.device)
    seg = torch.searchsorted(ptr, at, right=True) - 1
    inside = (at >= ptr[0]) & (at < ptr[-1])
    seg = seg.clamp(0, case["graphs"] - 1)
    count = ((ptr[1:] - ptr[:-1]).clamp(min=1) * (c // groups)).double().unsqueeze(1)
    part = torch.where(inside.unsqueeze(1), xg.sum(2), torch.zeros((), dtype=torch.float64, device=x.device))
    mean = torch.zeros(case["graphs"], groups, dtype=torch.float64, device=x.device).index_add_(0, seg, part) / count
    d = xg - mean[seg].unsqueeze(2)
    part = torch.where(inside.unsqueeze(1), (d * d).sum(2), torch.zeros((), dtype=torch.float64, device=x.device))
    var = torch.zeros(case["graphs"], groups, dtype=torch.float64, device=x.device).index_add_(0, seg, part) / count
    y = (d / torch.sqrt(var + 1e-5)[seg].unsqueeze(2)).view(rows, c).float() * st["w"] + st["b"]
    return torch.where(inside.unsqueeze(1), _activate(y, case["act"]), st["out"])


def _spmm(st):
    case = st["case"]
    n, col = case["nodes"], st["col"].long()
    deg = (st["row_ptr"][1:] - st["row_ptr"][:-1]).long()
    row = torch.repeat_interleave(torch.arange(n, device=col.device), deg, output_size=case["entries"])
    w = st["sx"].double()[col]
    if case["agg"] == "gcn":
        w = w * st["dis"].double()[row] * st["dis"].double()[col]
    elif case["agg"] == "weighted":
        w = w * st["ew"].double()
    elif case["agg"] == "mean":
        w = w / deg.double()[row]
    # hubs sum tens of thousands of rows: 64 bits
    out = torch.zeros(n, case["f"], dtype=torch.float64, device=col.device)
    return out.index_add_(0, row, st["x"][col].double() * w.unsqueeze(1)).float()


def run(state):
    case = state["case"]
    if own:
        from gnn_cuda_b200.GNN_cuda_common import int8_ops, norm_ops
        out = state["out"]
        if case["op"] == "linear":
            if case["form"] == "mlp":
                int8_ops.linear_int8_forward_(state["x"], None, state["w"], state["sw"], state["b"], state["h"], True,
                                              out_scale=state["sh"])
                int8_ops.linear_int8_forward_(state["h"], state["sh"], state["w2"], state["sw2"], state["b2"], out,
                                              case["relu"])
            else:
                int8_ops.linear_int8_forward_(state["x"], state["sx"], state["w"], state["sw"], state["b"], out,
                                              case["relu"])
        elif case["op"] == "norm":
            norm_ops.group_norm_forward_(state["x"], case["groups"], state["w"], state["b"], out,
                                         graph_ptr=state["ptr"], eps=1e-5, activation=case["act"])
        else:
            int8_ops.spmm_int8_forward_(state["row_ptr"], state["col"], state["x"], state["sx"], out,
                                        aggregation=case["agg"], deg_inv_sqrt=state["dis"], edge_weight=state["ew"])
        return out
    if case["op"] == "linear":
        q, s = (state["x"], state["sx"]) if case["form"] == "static" else _quantize(state["x"])
        if case["form"] == "mlp":
            q, s = _quantize(_linear(q, s, state["w"], state["sw"], state["b"], True))
            return _linear(q, s, state["w2"], state["sw2"], state["b2"], case["relu"])
        return _linear(q, s, state["w"], state["sw"], state["b"], case["relu"])
    return _norm(state) if case["op"] == "norm" else _spmm(state)


# --- 64 bits ---------------------------------------------------------------------

def _exact_held(v):
    """A 32-bit matrix as its 8-bit rows stand for it: whole multiples of the rows' 32-bit scales."""
    s = torch.linalg.vector_norm(v.double(), float("inf"), dim=1).div(127.0).float().double()
    r = v.double() / s.where(s > 0, torch.ones_like(s))[:, None]
    low = torch.floor(r)
    up = (r - low > 0.5) | ((r - low == 0.5) & (low % 2 != 0))
    return (low + up.double()) * s[:, None]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        x = _exact_held(st["x"]) if st["sx"] is None else st["x"].double() * st["sx"].double()[:, None]
        if case["form"] == "mlp":
            # the hidden value is a 32-bit value by definition, and its rounding decides what is held of it:
            # its steps are rounded as they are defined
            s = torch.linalg.vector_norm(st["x"].double(), float("inf"), dim=1).div(127.0).float()
            q = torch.round(x / s.double().where(s > 0, torch.ones_like(s, dtype=torch.float64))[:, None])
            h = torch.nn.functional.linear(q, st["w"].double()).float().mul_(s[:, None]).mul_(st["sw"]).add_(st["b"])
            x = _exact_held(h.clamp_(min=0))
            w, sw, b = st["w2"], st["sw2"], st["b2"]
        else:
            w, sw, b = st["w"], st["sw"], st["b"]
        y = torch.addmm(b.double(), x, (w.double() * sw.double()[:, None]).t())
        return y.clamp(min=0) if case["relu"] else y
    if case["op"] == "norm":
        rows, c, groups = case["rows"], case["c"], case["groups"]
        x = st["x"].double()
        if st["ptr"] is None:
            var, mean = torch.var_mean(x.view(rows, groups, -1), dim=2, unbiased=False)
            begin, end = 0, rows
        else:
            ptr = st["ptr"].long()
            begin, end = int(ptr[0]), int(ptr[-1])
            lengths = ptr[1:] - ptr[:-1]
            inner = x[begin:end]
            m1 = torch.segment_reduce(inner, "mean", lengths=lengths).view(len(lengths), groups, -1).mean(2)
            m1 = m1.repeat_interleave(lengths, 0)
            off = (inner.view(-1, groups, c // groups) - m1[:, :, None]).square().mean(2)
            mean, var = m1, torch.segment_reduce(off, "mean", lengths=lengths).repeat_interleave(lengths, 0)
        y = (x[begin:end].view(-1, groups, c // groups) - mean[:, :, None]) * (var + 1e-5).pow(-0.5)[:, :, None]
        y = y.reshape(-1, c) * st["w"].double() + st["b"].double()
        if case["act"] == "relu":
            y = y.clamp(min=0)
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "gelu":
            y = torch.nn.functional.gelu(y)
        full = st["out"].double()
        full[begin:end] = y
        return full
    n = case["nodes"]
    deg = st["row_ptr"].diff().double()
    val = torch.ones(case["entries"], dtype=torch.float64, device=DEV) if st["ew"] is None else st["ew"].double()
    a = torch.sparse_csr_tensor(st["row_ptr"].long(), st["col"].long(), val, size=(n, n))
    h = st["x"].double() * st["sx"].double()[:, None]
    if case["agg"] == "gcn":
        return (a @ (h * st["dis"].double()[:, None])) * st["dis"].double()[:, None]
    y = a @ h
    return y / deg.clamp(min=1)[:, None] if case["agg"] == "mean" else y
