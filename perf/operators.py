"""Measured cases of the row operators that stand around the sparse ones in a routed or relational layer: the
root-mean-square norm with a residual (and its 8-bit output), the choice of k experts a row with the lists it
gives, the products grouped by expert, and the weighted sum back.

A case is a dict of plain values; ``run`` computes it in plain torch (``own`` false) or through
``featgraph_b200.module`` (``own`` true).  Plain forms compute in 32 bits and round once at the end.
"""
import math

import torch

own = False

EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


def listed():
    return [
        # one decoding step of a few requests: the norm in front of an 8-bit product, latency alone
        dict(name="norm-serve-e4m3", op="norm", rows=16, d=2048, dtype="bf16", residual=True, e4m3=True, train=False),
        # a training step's pre-norm on a residual stream, forward and backward
        dict(name="norm-train-bf16", op="norm", rows=32768, d=4096, dtype="bf16", residual=True, e4m3=False, train=True),
        # node features of an odd width, the framework's own type
        dict(name="norm-nodes-f32", op="norm", rows=100003, d=331, dtype="f32", residual=False, e4m3=False, train=True),
        # a router at decode: a handful of rows
        dict(name="route-serve", op="route", rows=24, experts=64, k=4, scoring="softmax", normalize=True, closed=0.0, train=False),
        # a router over a training batch, some experts closed to some rows, with the logits' gradient
        dict(name="route-train", op="route", rows=65536, experts=128, k=8, scoring="softmax", normalize=True, closed=0.05, train=True),
        # decode through the experts' first product: weights are read once, for a row or two each
        dict(name="product-serve-bf16", op="product", rows=4, k=2, groups=16, inner=2048, outer=4096, dtype="bf16", skew=0.0, gather=True, train=False),
        # a prefill chunk through the experts, rows gathered
        dict(name="product-prefill-bf16", op="product", rows=4096, k=2, groups=32, inner=1024, outer=2816, dtype="bf16", skew=0.5, gather=True, train=False),
        # the largest: a training step's expert product with both gradients
        dict(name="product-train-bf16", op="product", rows=16384, k=4, groups=64, inner=2048, outer=4096, dtype="bf16", skew=0.5, gather=True, train=True),
        # node types of a graph, one weight a type, skewed counts, the framework's own type, both gradients
        dict(name="product-types-f32", op="product", rows=100003, k=1, groups=7, inner=256, outer=128, dtype="f32", skew=1.0, gather=False, train=True),
        # prefill with 8-bit rows and weights
        dict(name="product-prefill-e4m3", op="product", rows=8192, k=2, groups=16, inner=4096, outer=2048, dtype="e4m3", skew=0.5, gather=True, train=False),
        # decode: the experts' outputs summed back
        dict(name="combine-serve-f32", op="combine", rows=16, k=8, d=1024, dtype="f32", train=False),
        # a training step's sum over the experts, with the gradients of rows and weights
        dict(name="combine-train-bf16", op="combine", rows=32768, k=4, d=2048, dtype="bf16", train=True),
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]; odd ones as they come."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    v = _between(rng, lo, hi)
    return v if rng.random() < 0.4 else max(lo, v // 16 * 16)


def draw(rng):
    op = rng.choice(["norm", "route", "product", "product", "combine"])
    if op == "norm":
        d = _width(rng, 32, 8192)
        e4m3 = rng.random() < 0.4
        dtype = rng.choice(["f32", "f16", "bf16"])
        return dict(op=op, rows=_between(rng, 1, max(64, (1 << 26) // d)), d=d, dtype=dtype, residual=rng.random() < 0.6, e4m3=e4m3,
                    train=not e4m3 and rng.random() < 0.6)
    if op == "route":
        experts = _between(rng, 2, 512)
        return dict(op=op, rows=_between(rng, 1, 65536), experts=experts, k=_between(rng, 1, min(experts, 12)), scoring=rng.choice(["softmax", "sigmoid"]),
                    normalize=rng.random() < 0.6, closed=rng.choice([0.0, 0.1, 0.6]), train=rng.random() < 0.5)
    if op == "combine":
        k, d = _between(rng, 1, 10), _width(rng, 16, 4096)
        return dict(op=op, rows=_between(rng, 1, max(16, (1 << 26) // (k * d))), k=k, d=d, dtype=rng.choice(["f32", "f16", "bf16"]), train=rng.random() < 0.5)
    inner, outer, k = _width(rng, 32, 4096), _width(rng, 32, 4096), _between(rng, 1, 8)
    dtype = rng.choice(["f32", "f16", "bf16", "e4m3"])
    if dtype == "e4m3":
        inner = max(32, inner // 16 * 16)
    most = (1 << 38) // (inner * outer * k) if dtype != "f32" else (1 << 36) // (inner * outer * k)
    groups = _between(rng, 2, min(128, max(2, (1 << 28) // (inner * outer))))
    return dict(op=op, rows=_between(rng, 1, max(2, min(131072 // k, most))), k=min(k, groups), groups=groups, inner=inner, outer=outer, dtype=dtype,
                skew=rng.choice([0.0, 0.5, 1.0]), gather=rng.random() < 0.6, train=dtype != "e4m3" and rng.random() < 0.5)


# ---- inputs ----

def _lists(keys, groups):
    """(offsets, order, position) of the entries' keys [n, k], stable; entries with key -1 are in no group."""
    flat = torch.where(keys.reshape(-1) < 0, groups, keys.reshape(-1).long())
    counts = torch.bincount(flat, minlength=groups + 1)
    ends = torch.cumsum(counts, 0)
    offsets = torch.cat([ends.new_zeros(1), ends[:groups]]).int()
    order = torch.argsort(flat, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    dropped = flat == groups
    position = torch.where(dropped, -1, position).int().view(keys.shape)
    order = torch.where(dropped[order], -1, order).int()
    return offsets, order, position


def _choices(n, k, groups, skew, gen, dev):
    """k different groups for each row; with skew, low groups are chosen more often."""
    score = torch.rand((n, groups), device=dev, generator=gen) - skew * torch.log1p(torch.arange(groups, device=dev, dtype=torch.float32)) / math.log(groups + 1)
    return torch.topk(score, k, dim=1).indices.int()


def _e4m3_rows(v):
    scale = v.abs().amax(-1) / 448.0
    scale = torch.where(scale == 0, 1.0, scale)
    return (v / scale.unsqueeze(-1)).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, device=dev, generator=gen) * scale).to(dtype)

    s = dict(case=case)
    op, train = case["op"], case["train"]
    if op == "norm":
        n, d, t = case["rows"], case["d"], TYPES[case["dtype"]]
        s["x"] = normal(n, d, dtype=t)
        s["residual"] = normal(n, d, scale=2.0, dtype=t) if case["residual"] else None
        s["weight"] = (1 + normal(d, scale=0.1)).to(t)
        if train:
            s["dy"] = normal(n, d, dtype=t)
            s["dh"] = normal(n, d, dtype=t) if case["residual"] else None
    elif op == "route":
        n, e = case["rows"], case["experts"]
        s["logits"] = normal(n, e, scale=1.5)
        if case["closed"]:
            shut = torch.rand((n, e), device=dev, generator=gen) < case["closed"]
            s["logits"].masked_fill_(shut, float("-inf"))
        s["dw"] = normal(n, case["k"]) if train else None
    elif op == "product":
        n, k, g, i, o = (case[c] for c in ("rows", "k", "groups", "inner", "outer"))
        keys = _choices(n, k, g, case["skew"], gen, dev)
        s["offsets"], s["order"], s["position"] = _lists(keys, g)
        s["host_offsets"] = s["offsets"].tolist()
        rows = n if case["gather"] else n * k
        if case["dtype"] == "e4m3":
            s["x"], s["x_scale"] = _e4m3_rows(normal(rows, i))
            s["weight"], s["weight_scale"] = _e4m3_rows(normal(g, o, i, scale=i ** -0.5))
        else:
            t = TYPES[case["dtype"]]
            s["x"] = normal(rows, i, dtype=t)
            s["weight"] = normal(g, o, i, scale=i ** -0.5, dtype=t)
            s["dy"] = normal(n * k, o, dtype=t) if train else None
    else:
        n, k, d, t = case["rows"], case["k"], case["d"], TYPES[case["dtype"]]
        s["offsets"], s["order"], s["position"] = _lists(_choices(n, k, max(16, k), 0.0, gen, dev), max(16, k))
        s["y"] = normal(n * k, d, dtype=t)
        s["weights"] = torch.softmax(normal(n, k), 1)
        s["dout"] = normal(n, d, dtype=t) if train else None
    for name in ("x", "residual", "weight", "logits", "y", "weights"):
        if train and s.get(name) is not None:
            s[name].requires_grad_(True)
    return s


# ---- one pass ----

def run(s):
    case = s["case"]
    if own:
        return _OWN[case["op"]](s, case)
    with torch.no_grad():
        return _PLAIN[case["op"]](s, case)


def _norm_plain(s, case):
    x, w, t = s["x"], s["weight"].float(), s["x"].dtype
    h = (x.float() + s["residual"].float()).to(t) if case["residual"] else x
    hf = h.float()
    r = torch.rsqrt((hf * hf).mean(1, keepdim=True) + EPS)
    v = hf * r * w
    out = {}
    if case["residual"]:
        out["h"] = h
    if case["e4m3"]:
        out["y"], out["scales"] = _e4m3_rows(v)
        return out
    out["y"] = v.to(t)
    if case["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = r * g - hf * (r * r * r) * ((g * hf).sum(1, keepdim=True) / case["d"])
        if case["residual"]:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(t)
        out["dweight"] = (dy * hf * r).sum(0).to(t)
    return out


def _norm_own(s, case):
    from featgraph_b200.module import rms_norm
    got = rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS, quantize=case["e4m3"])
    y, h = got if case["residual"] else (got, None)
    out = {}
    if case["residual"]:
        out["h"] = h
    if case["e4m3"]:
        out["y"], out["scales"] = y.values, y.scales
        return out
    out["y"] = y
    if case["train"]:
        outs, grads = ((y, h), (s["dy"], s["dh"])) if case["residual"] else ((y,), (s["dy"],))
        out["dx"], out["dweight"] = torch.autograd.grad(outs, (s["x"], s["weight"]), grads)
    return out


def _route_plain(s, case):
    x, k = s["logits"], case["k"]
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    value, index = value[:, :k], index[:, :k]
    taken = value > float("-inf")
    if case["scoring"] == "softmax":
        top = value[:, :1].clamp(min=torch.finfo(x.dtype).min)
        chosen = torch.exp(value - top)
        score = torch.exp(x - top)
        total = (chosen if case["normalize"] else score).sum(1, keepdim=True)
    else:
        chosen = torch.where(value >= 0, 1 / (1 + torch.exp(-value)), torch.exp(value) / (1 + torch.exp(value)))
        total = chosen.sum(1, keepdim=True) if case["normalize"] else torch.ones_like(value[:, :1])
    weights = torch.where(taken, chosen / torch.where(total > 0, total, 1.0), 0.0)
    experts = torch.where(taken, index, -1).int()
    offsets, order, position = _lists(experts, case["experts"])
    out = dict(weights=weights, experts=experts, offsets=offsets, order=order, position=position)
    if case["train"]:
        g = torch.where(taken, s["dw"], 0.0)
        dot = (g * weights).sum(1, keepdim=True)
        if case["scoring"] == "softmax":
            if case["normalize"]:
                out["dlogits"] = torch.zeros_like(x).scatter_(1, index, weights * (g - dot))
            else:
                p = score / torch.where(total > 0, total, 1.0)
                out["dlogits"] = torch.zeros_like(x).scatter_(1, index, weights * g) - p * dot
        else:
            slope = torch.where(taken, torch.exp(-value.abs()) / (1 + torch.exp(-value.abs())) ** 2, 0.0)
            inner = (g - dot) / torch.where(total > 0, total, 1.0) if case["normalize"] else g
            out["dlogits"] = torch.zeros_like(x).scatter_(1, index, slope * inner)
    return out


def _route_own(s, case):
    from featgraph_b200.module import route
    r = route(s["logits"], case["k"], scoring=case["scoring"], normalize=case["normalize"])
    out = dict(weights=r.weights, experts=r.experts, offsets=r.groups.offsets, order=r.groups.order, position=r.groups.position)
    if case["train"]:
        out["dlogits"], = torch.autograd.grad((r.weights,), (s["logits"],), (s["dw"],))
    return out


def _product_plain(s, case):
    """One library product a group, on the rows that are its own: the counts differ too much for a padded batch."""
    x, w, at, k = s["x"], s["weight"], s["host_offsets"], case["k"]
    n, i, o, m = case["rows"], case["inner"], case["outer"], case["rows"] * case["k"]
    if case["dtype"] == "e4m3":
        xf = x.float() * s["x_scale"].unsqueeze(1)
        t = torch.bfloat16
    else:
        xf, t = x.float(), x.dtype
    xf = xf[(s["order"] // k).long()] if case["gather"] else xf
    y = torch.zeros((m, o), device=x.device, dtype=t)
    train = case["train"]
    if train:
        dyf = s["dy"].float()
        dxg = torch.zeros((m, i), device=x.device)
        dw = torch.zeros_like(w)
    for g in range(case["groups"]):
        a, b = at[g], at[g + 1]
        if a == b:
            continue
        wg = w[g].float()
        if case["dtype"] == "e4m3":
            wg = wg * s["weight_scale"][g].unsqueeze(1)
        y[a:b] = (xf[a:b] @ wg.t()).to(t)
        if train:
            dxg[a:b] = dyf[a:b] @ wg
            dw[g] = (dyf[a:b].t() @ xf[a:b]).to(t)
    if not train:
        return dict(y=y)
    dx = dxg[s["position"].long().reshape(-1)].view(n, k, i).sum(1) if case["gather"] else dxg
    return dict(y=y, dx=dx.to(t), dweight=dw)


def _product_own(s, case):
    from featgraph_b200.module import QuantizedRows, RowGroups, grouped_matmul
    groups = RowGroups(s["offsets"], s["order"], s["position"])
    x, w = s["x"], s["weight"]
    if case["dtype"] == "e4m3":
        x, w = QuantizedRows(x, s["x_scale"]), QuantizedRows(w, s["weight_scale"])
    y = grouped_matmul(x, w, groups, gather=case["gather"])
    if not case["train"]:
        return dict(y=y)
    dx, dw = torch.autograd.grad((y,), (x, w), (s["dy"],))
    return dict(y=y, dx=dx, dweight=dw)


def _combine_plain(s, case):
    at = s["position"].long()
    rows = s["y"].float()[at]
    w = s["weights"].unsqueeze(2)
    out = dict(out=(rows * w).sum(1).to(s["y"].dtype))
    if case["train"]:
        dout = s["dout"].float().unsqueeze(1)
        dy = torch.empty((case["rows"] * case["k"], case["d"]), device=at.device, dtype=s["y"].dtype)
        dy[at.reshape(-1)] = (dout * w).to(s["y"].dtype).view(-1, case["d"])
        out["dy"], out["dweights"] = dy, (rows * dout).sum(2)
    return out


def _combine_own(s, case):
    from featgraph_b200.module import RowGroups, combine_rows
    out = combine_rows(s["y"], RowGroups(s["offsets"], s["order"], s["position"]), weights=s["weights"])
    if not case["train"]:
        return dict(out=out)
    dy, dw = torch.autograd.grad((out,), (s["y"], s["weights"]), (s["dout"],))
    return dict(out=out, dy=dy, dweights=dw)


_PLAIN = dict(norm=_norm_plain, route=_route_plain, product=_product_plain, combine=_combine_plain)
_OWN = dict(norm=_norm_own, route=_route_own, product=_product_own, combine=_combine_own)


# ---- compulsory work ----

def work(case):
    op, train = case["op"], case["train"]
    if op == "norm":
        n, d, b = case["rows"], case["d"], SIZE[case["dtype"]]
        passes = 1 + 2 * case["residual"]  # x, and with a residual that and the sum
        size = n * d * (passes * b + (1 if case["e4m3"] else b)) + d * b + (4 * n if case["e4m3"] else 0)
        if train:
            size += n * d * b * (2 + case["residual"]) + d * b  # dy, dx, and the sum's own gradient; dweight
        return dict(bytes=size, flops=n * d * (5 + 10 * train))
    if op == "route":
        n, e, k = case["rows"], case["experts"], case["k"]
        return dict(bytes=n * e * 4 + n * k * 16 + (e + 1) * 4 + train * (n * k * 4 + n * e * 4), flops=n * e * (4 + 4 * train))
    if op == "combine":
        n, k, d, b = case["rows"], case["k"], case["d"], SIZE[case["dtype"]]
        # with gradients: dout read, dy and the weights' gradient written; y is an input that is read once
        return dict(bytes=n * k * d * b + n * d * b + n * k * 8 + train * (n * d * b + n * k * d * b + n * k * 4), flops=2 * n * k * d * (1 + 2 * train))
    n, k, g, i, o = (case[c] for c in ("rows", "k", "groups", "inner", "outer"))
    m, b = n * k, SIZE[case["dtype"]]
    out = 2 if case["dtype"] == "e4m3" else b
    rows = n if case["gather"] else m
    size = rows * i * b + min(g, m) * i * o * b + m * o * out + 8 * m
    if train:
        size += m * o * b + rows * i * b + g * i * o * b  # dy read, dx and dweight written
    return dict(bytes=size, flops=2 * m * i * o * (1 + 2 * train))


# ---- the definitions in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return _EXACT[case["op"]](s, case)


def _norm_exact(s, case):
    h = s["x"].double()
    if case["residual"]:
        h = (h + s["residual"].double()).to(s["x"].dtype).double()
    w = s["weight"].double()
    inverse = 1 / torch.sqrt(h.pow(2).sum(1) / case["d"] + EPS)
    unit = torch.einsum("nd,n->nd", h, inverse)
    y = unit * w
    out = dict(h=h) if case["residual"] else {}
    if case["e4m3"]:
        # which 8-bit value a number next to a border gets depends on its last bits: the scales alone have a value
        return dict(out, y=None, scales=torch.where(y.abs().amax(1) == 0, 1.0, y.abs().amax(1) / 448))
    out["y"] = y
    if case["train"]:
        dy = s["dy"].double()
        along = torch.einsum("nd,nd->n", dy * w, unit) / case["d"]
        out["dx"] = inverse.unsqueeze(1) * (dy * w - unit * along.unsqueeze(1)) + (s["dh"].double() if case["residual"] else 0)
        out["dweight"] = torch.einsum("nd,nd->d", dy, unit)
    return out


def _route_exact(s, case):
    x, k = s["logits"].double(), case["k"]
    leaf = x.clone().requires_grad_(True)
    with torch.enable_grad():
        open_ = leaf > float("-inf")
        empty = ~open_.any(1, keepdim=True)
        if case["scoring"] == "softmax":
            score = torch.softmax(torch.where(empty, torch.zeros_like(leaf), leaf), 1)
        else:
            score = torch.sigmoid(leaf)
        rank = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
        keep = open_.gather(1, rank)
        picked = torch.where(keep, score.gather(1, rank), torch.zeros((), dtype=torch.float64, device=x.device))
        if case["normalize"]:
            total = picked.sum(1, keepdim=True)
            picked = picked / torch.where(total > 0, total, torch.ones_like(total))
        out = dict(weights=picked.detach(), experts=None, offsets=None, order=None, position=None)
        if case["train"]:
            out["dlogits"], = torch.autograd.grad((picked,), (leaf,), (s["dw"].double(),))
            out["dlogits"] = torch.where(open_, out["dlogits"], 0.0)
    return out


def _product_exact(s, case):
    if case["rows"] * case["k"] * case["inner"] * case["outer"] * (1 + 2 * case["train"]) > 4e12:
        return None
    k, m = case["k"], case["rows"] * case["k"]
    x, w = s["x"].double(), s["weight"]
    if case["dtype"] == "e4m3":
        x = x * s["x_scale"].double().unsqueeze(1)
    source = torch.div(s["order"], k, rounding_mode="floor").long() if case["gather"] else torch.arange(m, device=x.device)
    owner = torch.bucketize(torch.arange(m, device=x.device), s["offsets"][1:].long(), right=True)
    y = torch.zeros((m, case["outer"]), dtype=torch.float64, device=x.device)
    out = dict(y=y)
    if case["train"]:
        dy = s["dy"].double()
        out["dx"], out["dweight"] = torch.zeros_like(x), torch.zeros(w.shape, dtype=torch.float64, device=x.device)
    for g in range(case["groups"]):
        p = torch.nonzero(owner == g).flatten()
        wg = w[g].double()
        if case["dtype"] == "e4m3":
            wg = wg * s["weight_scale"][g].double().unsqueeze(1)
        y[p] = torch.einsum("ri,oi->ro", x[source[p]], wg)
        if case["train"]:
            out["dx"].index_add_(0, source[p], torch.einsum("ro,oi->ri", dy[p], wg))
            out["dweight"][g] = torch.einsum("ro,ri->oi", dy[p], x[source[p]])
    return out


def _combine_exact(s, case):
    n, k, d = case["rows"], case["k"], case["d"]
    entry = s["order"].long()
    row, w = entry // k, s["weights"].double().reshape(-1)[entry]
    y = s["y"].double()
    out = dict(out=torch.zeros((n, d), dtype=torch.float64, device=y.device).index_add_(0, row, y * w.unsqueeze(1)))
    if case["train"]:
        dout = s["dout"].double()[row]
        out["dy"] = dout * w.unsqueeze(1)
        dw = torch.zeros(n * k, dtype=torch.float64, device=y.device)
        dw[entry] = (dout * y).sum(1)
        out["dweights"] = dw.view(n, k)
    return out


_EXACT = dict(norm=_norm_exact, route=_route_exact, product=_product_exact, combine=_combine_exact)
