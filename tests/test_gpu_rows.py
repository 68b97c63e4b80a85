"""Row operators (``featgraph_b200.module.rows``) against plain formulations in 64 bits.

Tolerances count roundings.  A value rounded to type t is off by at most half a step, ``finfo(t).eps / 2`` of itself;
32-bit arithmetic adds u = 2^-24 of each intermediate.  A sum of terms s_i taken in any order with at most c additions on
each term's way is off by at most c u sum|s_i|; the tensor cores' sums may truncate, which doubles the step."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    """Half the spacing of t's subnormal numbers."""
    return torch.finfo(t).tiny * torch.finfo(t).eps / 2


def close(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    finite = torch.isfinite(want)
    assert torch.equal(finite, torch.isfinite(got)), "%s: finite in different places" % what
    off = torch.where(finite, (got - want).abs() - tol, torch.zeros_like(want))
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0.0, "%s: over its tolerance by %.3g (largest value %.3g)" % (what, worst, float(want[finite].abs().max()))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(shape, seed, t=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=gen(seed)) * scale).to(t)


# ---- norm ----

# row statistics: at most 16 additions a thread, 5 in its warp, 32 across warps, twice that for the squares' own
# rounding, halved by the root: 60 u of the value cover them with the products
STAT = 60 * U


def norm_reference(h, w, eps=1e-6):
    r = 1 / torch.sqrt(h.double().pow(2).mean(-1, keepdim=True) + eps)
    return h.double() * r * (1.0 if w is None else w.double()), r


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,d", [(1, 1), (3, 7), (5, 32), (60001, 32), (333, 64), (1000, 128), (77, 129), (9001, 99), (1, 255), (9, 256), (17, 300), (6, 512), (4, 513), (5, 1024), (3, 1500), (2, 2048),
                                 (3, 2050), (2, 4096), (3, 5001), (2, 8192), (2, 16384), (1, 16383)])
def test_norm_forward(t, n, d):
    from featgraph.module import rms_norm
    dt = TYPES[t]
    x, res, w = normal((n, d), 1, dt), normal((n, d), 2, dt, 2.0), normal((d,), 3, dt)
    for weight in (None, w, w.float()):
        want, _ = norm_reference(x, weight)
        close(rms_norm(x, weight), want, want.abs() * (half_step(dt) + STAT) + tiny(dt), "y")
    y, h = rms_norm(x, w, residual=res)
    assert torch.equal(h, (x.float() + res.float()).to(dt))
    want, _ = norm_reference(h, w)
    close(y, want, want.abs() * (half_step(dt) + STAT) + tiny(dt), "y with a residual")


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,d", [(1, 1), (7, 40), (5001, 32), (70003, 64), (2600, 100), (9, 128), (40001, 31), (300, 331), (33, 512), (5, 1024), (1000, 96), (70, 2048), (9, 4096), (3, 8192), (2, 16384), (700, 130)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm_gradients(t, n, d, with_residual):
    from featgraph.module import rms_norm
    dt = TYPES[t]
    x, w, dy = normal((n, d), 1, dt), normal((d,), 3, dt) + 1, normal((n, d), 4, dt)
    res, dh = (normal((n, d), 2, dt), normal((n, d), 5, dt)) if with_residual else (None, None)
    leaves = [v.requires_grad_(True) for v in (x, w, res) if v is not None]
    out = rms_norm(x, w, residual=res)
    y, h = out if with_residual else (out, x)
    grads = torch.autograd.grad([y, h] if with_residual else [y], leaves, [dy, dh] if with_residual else [dy])
    hd, _w, g = h.detach().double(), w.detach().double(), dy.double() * w.detach().double()
    _, r = norm_reference(h.detach(), None)
    first, second = r * g, hd * r ** 3 * (g * hd).sum(1, keepdim=True) / d
    want = first - second + (dh.double() if with_residual else 0)
    parts = first.abs() + hd.abs() * r ** 3 * (g * hd).abs().sum(1, keepdim=True) / d
    close(grads[0], want, want.abs() * half_step(dt) + 4 * STAT * parts + (U * want.abs() if with_residual else 0) + tiny(dt), "dx")
    if with_residual:
        assert torch.equal(grads[0], grads[2])
    terms = dy.double() * hd * r
    # a term passes its block's rows (n / blocks + 8), the partial rows (blocks / 8 + 8) and the statistics of its row
    blocks = min(n, 148 * 4)
    adds = n / blocks + 16 + blocks / 8 + 8
    want = terms.sum(0)
    close(grads[1], want, want.abs() * half_step(dt) + (adds * U + STAT) * terms.abs().sum(0) + tiny(dt), "dweight")


def test_norm_gradient_against_differences():
    """The formula itself: central differences of the 64-bit forward, at step 1e-5 off by about 1e-10, the 32-bit
    gradient by 1e-5 of its terms."""
    from featgraph.module import rms_norm
    x, w, dy = normal((4, 24), 1), normal((24,), 2), normal((4, 24), 3)
    leaf = x.clone().requires_grad_(True)
    got, = torch.autograd.grad((rms_norm(leaf, w),), (leaf,), (dy,))
    want = torch.zeros_like(x, dtype=torch.float64)
    for i in range(x.numel()):
        e = torch.zeros(x.numel(), dtype=torch.float64, device="cuda")
        e[i] = 1e-5
        e = e.view_as(x)
        hi, lo = (norm_reference(x.double() + s * e, w)[0] for s in (1, -1))
        want.view(-1)[i] = ((hi - lo) * dy.double()).sum() / 2e-5
    close(got, want, 1e-5 * (1 + want.abs()), "dx")


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,d", [(1, 1), (16, 2048), (5, 77), (4001, 32), (63, 128), (40, 512), (3, 8192), (2, 16384), (9, 1000)])
def test_norm_in_8_bits(t, n, d):
    from featgraph.module import quantize_rows, rms_norm
    dt = TYPES[t]
    x, w, res = normal((n, d), 1, dt), normal((d,), 2, dt), normal((n, d), 3, dt)
    x[0] = 0
    res[0] = 0
    q, h = rms_norm(x, w, residual=res, quantize=True)
    assert q.values.dtype == torch.float8_e4m3fn and q.scales.shape == (n,)
    want, _ = norm_reference(h, w)
    for got, v in ((q, want), (quantize_rows(h), h.double())):
        most = v.abs().amax(1)
        scale = torch.where(most == 0, torch.ones_like(most), most / 448)
        close(got.scales, scale, scale * (STAT + 2 * U), "scales")
        back = got.values.double() * got.scales.double().unsqueeze(1)
        # half a step of 2^-3 of the value, half of e4m3's smallest step (2^-9) near zero, and the value's own error
        close(back, v, v.abs() * (2.0 ** -4 + 2 * STAT) + scale.unsqueeze(1) * 2.0 ** -10 * 1.001, "values")
    assert float(q.scales[0]) == 1.0 and not bool(q.values[0].float().any())


def test_norm_strided_rows_and_leading_dimensions():
    from featgraph.module import rms_norm
    big = normal((6, 5, 96), 1, torch.bfloat16)
    w = normal((64,), 2, torch.bfloat16)
    for x in (big[:, 2, :64], big[:, 2, 3:67], big[..., :64], big[:, :, ::2][:, :, :40], big[0, :1, :64].expand(4, 64)):
        weight = w[:x.shape[-1]]
        for v in (x, x.detach().clone()):
            assert torch.equal(rms_norm(v, weight), rms_norm(x.contiguous(), weight))
    y, h = rms_norm(big[..., :64], w, residual=big[..., 32:])
    assert y.shape == h.shape == (6, 5, 64)
    assert rms_norm(big[:0, 0], None).shape == (0, 96)
    x = big[:0, 0].clone().requires_grad_(True)
    w = normal((96,), 2, torch.bfloat16).requires_grad_(True)
    dx, dw = torch.autograd.grad(rms_norm(x, w).sum(), (x, w))
    assert dx.shape == (0, 96) and not bool(dw.any())


def test_norm_weight_gradient_over_many_rows_has_the_same_bits_again():
    from featgraph.module import rms_norm
    x, w, dy = normal((20001, 200), 1), normal((200,), 2).requires_grad_(True), normal((20001, 200), 3)
    got = [torch.autograd.grad(rms_norm(x, w), w, dy)[0] for _ in range(3)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


# ---- routing ----

def lists_reference(keys, groups):
    flat = keys.cpu().numpy().reshape(-1)
    flat = np.where((flat < 0) | (flat >= groups), groups, flat)
    order = np.argsort(flat, kind="stable")
    position = np.empty_like(order)
    position[order] = np.arange(order.size)
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat, minlength=groups + 1))[:groups]])
    return offsets, np.where(flat[order] == groups, -1, order), np.where(flat == groups, -1, position).reshape(keys.shape)


def check_lists(groups, keys, count):
    offsets, order, position = lists_reference(keys, count)
    assert np.array_equal(groups.offsets.cpu().numpy(), offsets)
    assert np.array_equal(groups.order.cpu().numpy(), order)
    assert np.array_equal(groups.position.cpu().numpy(), position)


@pytest.mark.parametrize("n,k,groups", [(0, 1, 3), (1, 1, 1), (5, 2, 3), (31, 3, 7), (64, 4, 64), (100, 8, 1024), (2047, 1, 5), (1024, 8, 100),
                                        (1025, 8, 100), (8193, 1, 2), (70001, 3, 33), (50000, 1, 1024), (300000, 8, 17)])
def test_lists(n, k, groups):
    from featgraph.module import group_rows
    for seed, lo in ((1, 0), (2, -2)):
        keys = torch.randint(lo, groups + (lo < 0), (n, k), device="cuda", generator=gen(seed), dtype=torch.int32)
        check_lists(group_rows(keys, groups), keys, groups)
    keys = torch.full((n, k), groups - 1, dtype=torch.int64, device="cuda")
    if n > 3:
        keys[1] = 2 ** 40  # no wrap-around into a valid group
        keys[2] = -2 ** 40
    check_lists(group_rows(keys if k > 1 else keys[:, 0], groups), keys, groups)


def route_reference(logits, k, scoring, normalize):
    x = logits.double().cpu()
    open_ = x > float("-inf")
    ranked = torch.where(open_, x, torch.full_like(x, float("-inf")))
    value, index = torch.sort(ranked, dim=1, descending=True, stable=True)
    value, index, keep = value[:, :k], index[:, :k], torch.isfinite(value[:, :k])
    if scoring == "softmax":
        p = torch.softmax(torch.where(open_.any(1, keepdim=True), ranked, torch.zeros_like(ranked)), 1)
    else:
        p = torch.sigmoid(ranked)
    w = torch.where(keep, p.gather(1, index), torch.zeros_like(value))
    if normalize:
        s = w.sum(1, keepdim=True)
        w = w / torch.where(s > 0, s, torch.ones_like(s))
    return w.cuda(), torch.where(keep, index, torch.full_like(index, -1)).int().cuda()


# exp takes the difference of two logits, rounded (here below 64 in size: 32 u of the result's exponent each way), its
# own 2 steps, sums of at most 32 + 5 terms, a quotient
WEIGHT = 160 * U


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,experts,k", [(1, 1, 1), (3, 2, 2), (17, 8, 2), (9, 33, 5), (40, 64, 32), (5, 100, 7), (13, 256, 8), (4, 511, 1), (3, 1024, 32)])
def test_route(scoring, normalize, t, n, experts, k):
    from featgraph.module import route
    dt = TYPES[t]
    x = normal((n, experts), 1, dt, 2.0)
    x[:, experts // 2:] = x[:, :experts - experts // 2]  # ties
    shut = torch.rand((n, experts), device="cuda", generator=gen(2)) < 0.3
    x[shut] = float("-inf")
    x[0] = float("-inf")  # a row with nothing open
    if n > 2:
        x[1] = 0.0
        x[1, ::2] = -0.0  # equal to +0
        x[2, 0] = float("nan")
    want, chosen = route_reference(x, k, scoring, normalize)
    x = x.requires_grad_(True)
    r = route(x, k, scoring=scoring, normalize=normalize)
    assert torch.equal(r.experts, chosen)
    close(r.weights.detach(), want, want * WEIGHT + 1e-37, "weights")
    check_lists(r.groups, chosen, experts)
    dw = normal((n, k), 3)
    got, = torch.autograd.grad(r.weights, x, dw)
    leaf = torch.where(x.detach() > float("-inf"), x.detach().double(), torch.full_like(x, -1e4, dtype=torch.float64)).requires_grad_(True)
    p = torch.softmax(leaf, 1) if scoring == "softmax" else torch.sigmoid(leaf)
    keep = chosen >= 0
    w = torch.where(keep, p.gather(1, chosen.clamp(min=0).long()), torch.zeros((), dtype=torch.float64, device="cuda"))
    if normalize:
        s = w.sum(1, keepdim=True)
        w = w / torch.where(s > 0, s, torch.ones_like(s))
    grad, = torch.autograd.grad(w, leaf, dw.double())
    grad = torch.where((x.detach() > float("-inf")) & keep.any(1, keepdim=True), grad, torch.zeros_like(grad))
    size = dw.double().abs().sum(1, keepdim=True)  # every weight and slope is at most 1
    close(got, grad, grad.abs() * half_step(dt) + 4 * WEIGHT * size + tiny(dt), "dlogits")


def test_route_extreme_logits():
    from featgraph.module import route
    big = torch.finfo(torch.float32).max
    x = torch.tensor([[big, -big, 0.0, float("-inf")], [-big, -big, float("-inf"), float("-inf")], [300.0, 299.0, -300.0, 0.0]], device="cuda")
    r = route(x, 3)
    assert r.experts.tolist() == [[0, 2, 1], [0, 1, -1], [0, 1, 3]]
    assert torch.allclose(r.weights[:2].cpu(), torch.tensor([[1.0, 0, 0], [0.5, 0.5, 0]]))
    assert torch.isfinite(route(x, 3, scoring="sigmoid").weights).all()


# ---- products ----

def make_groups(n, k, count, seed, sizes=None, dropped=0.0):
    from featgraph.module import group_rows
    if sizes is not None:
        keys = torch.cat([torch.full((s,), g, dtype=torch.int32) for g, s in enumerate(sizes)] + [torch.full((n * k - sum(sizes),), -1, dtype=torch.int32)])
        keys = keys[torch.randperm(n * k, generator=torch.Generator().manual_seed(seed))].view(n, k).cuda()
    else:
        keys = torch.randint(0, count, (n, k), device="cuda", generator=gen(seed), dtype=torch.int32)
    if dropped:
        keys[torch.rand((n, k), device="cuda", generator=gen(seed + 1)) < dropped] = -1
    return group_rows(keys, count)


def product_reference(x, w, groups, gather, dy=None):
    x, w = x.detach().double(), w.detach().double()
    at = groups.offsets.tolist()
    m, k = groups.num_entries, groups.choices
    source = (groups.order.long() // k) if gather else torch.arange(m, device="cuda")
    y = torch.zeros((m, w.shape[1]), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(y)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    dxs, dws = torch.zeros_like(x), torch.zeros_like(w)
    for g in range(groups.num_groups):
        rows = slice(at[g], at[g + 1])
        xg = x[source[rows]]
        y[rows] = xg @ w[g].t()
        size[rows] = xg.abs() @ w[g].abs().t()
        if dy is not None:
            d = dy.double()[rows]
            dx.index_add_(0, source[rows], d @ w[g])
            dxs.index_add_(0, source[rows], d.abs() @ w[g].abs())
            dw[g] = d.t() @ xg
            dws[g] = d.abs().t() @ xg.abs()
    return y, size, dx, dxs, dw, dws


def steps(terms):
    """Roundings on a term's way through a sum of that many: each may truncate (2 u); the 32-bit inputs' parts and the
    scaling add a few."""
    return (2 * (terms / 8 + 24)) * U


def check_product(x, w, groups, gather, dy, what=""):
    from featgraph.module import grouped_matmul
    dt = x.dtype
    xl, wl = x.detach().clone(memory_format=torch.preserve_format), w
    xl = x.detach().requires_grad_(True)
    wl = w.detach().requires_grad_(True)
    y = grouped_matmul(xl, wl, groups, gather=gather)
    dx, dw = torch.autograd.grad(y, (xl, wl), dy)
    want, size, wdx, sdx, wdw, sdw = product_reference(x, w, groups, gather, dy)
    inner, outer = w.shape[2], w.shape[1]
    most = int((groups.offsets[1:] - groups.offsets[:-1]).max()) if groups.num_entries else 0
    close(y.detach(), want, want.abs() * half_step(dt) + steps(inner) * size + tiny(dt), what + " y")
    # with several slots a row each slot's part is rounded to the type before the sum
    parts = 2 * half_step(dt) * sdx.clamp(min=0) if gather else 0
    if gather and dt != torch.float32:
        parts = half_step(dt) * per_slot_size(groups, w, dy)
    close(dx, wdx, wdx.abs() * half_step(dt) + parts + steps(outer) * sdx + 8 * tiny(dt), what + " dx")
    close(dw, wdw, wdw.abs() * half_step(dt) + steps(most) * sdw + tiny(dt), what + " dw")
    return y


def per_slot_size(groups, w, dy):
    at, k = groups.offsets.tolist(), groups.choices
    total = torch.zeros((groups.num_rows, w.shape[2]), dtype=torch.float64, device="cuda")
    for g in range(groups.num_groups):
        rows = slice(at[g], at[g + 1])
        total.index_add_(0, groups.order[rows].long() // k, (dy.double()[rows] @ w[g].detach().double()).abs())
    return total


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("n,k,count,inner,outer", [
    (1, 1, 1, 1, 1), (3, 2, 4, 16, 8), (5, 1, 3, 17, 33), (130, 1, 2, 64, 64), (257, 2, 5, 128, 96), (64, 4, 40, 200, 264), (1000, 3, 7, 72, 520),
    (300, 1, 1, 96, 24), (2000, 2, 3, 331, 127), (40, 8, 300, 64, 40), (129, 2, 2, 512, 1024), (777, 1, 4, 1000, 160),
    (10000, 1, 4, 1304, 1000), (5001, 2, 2, 520, 1301), (30, 1, 9, 520, 264), (8, 4, 5, 72, 1000), (33, 1, 3, 264, 520),
    (4100, 2, 5, 520, 96), (9001, 1, 3, 72, 250)])
def test_product_and_gradients(t, gather, n, k, count, inner, outer):
    dt = TYPES[t]
    groups = make_groups(n, k, count, 5)
    x = normal((n if gather else n * k, inner), 1, dt)
    w = normal((count, outer, inner), 2, dt, inner ** -0.5)
    check_product(x, w, groups, gather, normal((n * k, outer), 3, dt))


@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("sizes", [[0, 0, 0], [0, 500, 0, 12, 0], [128, 128, 256], [127, 1, 129, 255], [1, 1, 1, 1], [0, 0, 640], [64, 65, 63, 0, 192]])
def test_product_group_sizes(t, sizes):
    """Empty groups, groups that end on and beside tile borders, rows in no group (their output and gradient are 0)."""
    dt = TYPES[t]
    n = sum(sizes) + 37
    groups = make_groups(n, 1, len(sizes), 5, sizes=sizes)
    x, w = normal((n, 80), 1, dt), normal((len(sizes), 144, 80), 2, dt, 0.1)
    for gather in (False, True):
        y = check_product(x, w, groups, gather, normal((n, 144), 3, dt), str(sizes))
        assert not bool(y.detach()[sum(sizes):].any())


@pytest.mark.parametrize("t", sorted(TYPES))
def test_product_keeps_groups_apart(t):
    """NaN and infinities in one group's rows, in rows in no group, and in one group's weight stay there."""
    from featgraph.module import grouped_matmul
    dt = TYPES[t]
    sizes = [70, 61, 40, 200]
    n = sum(sizes) + 50
    groups = make_groups(n, 1, 4, 5, sizes=sizes)
    x, w, dy = normal((n, 96), 1, dt), normal((4, 104, 96), 2, dt, 0.1), normal((n, 104), 3, dt)
    at = groups.offsets.tolist()
    x[at[1]:at[2]] = float("nan")
    x[at[4]:] = float("inf")
    dy[at[4]:] = float("nan")
    w[3] = float("nan")
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_matmul(xl, wl, groups)
    dx, dw = torch.autograd.grad(y, (xl, wl), dy)
    fine = torch.isfinite(y).all(1)
    assert fine[:at[1]].all() and fine[at[2]:at[3]].all() and not fine[at[1]:at[2]].any() and not fine[at[3]:at[4]].any()
    assert not bool(y.detach()[at[4]:].any()) and not bool(dx[at[4]:].any())
    fine = torch.isfinite(dx).all(1)
    assert fine[:at[3]].all() and not fine[at[3]:at[4]].any()
    assert torch.isfinite(dw[0]).all() and torch.isfinite(dw[2]).all() and torch.isfinite(dw[3]).all() and not torch.isfinite(dw[1]).any()


@pytest.mark.parametrize("t", sorted(TYPES))
def test_product_strides(t):
    """Weights stored [groups, in, out], with padding, as one broadcast weight; rows with a stride or an odd start."""
    dt = TYPES[t]
    n, inner, outer = 150, 64, 48
    groups = make_groups(n, 2, 3, 5)
    dy = normal((2 * n, outer + 8), 3, dt)[:, 3:outer + 3]
    big = normal((2 * n, inner + 16), 1, dt)
    store = normal((3, inner, outer), 2, dt, 0.1)
    padded = normal((3, outer + 2, inner + 5), 4, dt, 0.1)
    for x in (big[:, :inner], big[:, 1:inner + 1], big[:, 8:inner + 8], big[:, :inner].t().contiguous().t()):
        for w in (store.transpose(1, 2), padded[:, 1:outer + 1, 2:inner + 2], padded[:1, :outer, :inner].expand(3, outer, inner), padded[:, :outer, ::2][:, :, :32]):
            check_product(x[:, :w.shape[2]], w, groups, False, dy)
    shared = padded[0, :outer, :inner].clone().requires_grad_(True)
    from featgraph.module import grouped_matmul
    y = grouped_matmul(big[:, :inner], shared.expand(3, outer, inner), groups)
    got, = torch.autograd.grad(y, shared, dy)
    want = dy.double().t() @ big[:, :inner].double()
    size = dy.double().abs().t() @ big[:, :inner].double().abs()
    # each group's gradient is rounded to the type, then their sum
    close(got, want, 4 * half_step(dt) * size + steps(2 * n) * size, "broadcast weight")


@pytest.mark.parametrize("n,k,count,inner,outer", [(1, 1, 1, 16, 8), (5, 2, 3, 32, 24), (300, 2, 4, 128, 136), (129, 1, 2, 1040, 520), (64, 4, 33, 77, 45), (2000, 1, 5, 256, 128), (10000, 1, 4, 272, 1000), (16, 2, 9, 272, 264), (3000, 3, 7, 400, 130)])
@pytest.mark.parametrize("out", sorted(TYPES))
def test_product_of_8_bit_rows(n, k, count, inner, outer, out):
    from featgraph.module import QuantizedRows, grouped_matmul, quantize_rows
    dt = TYPES[out]
    groups = make_groups(n, k, count, 5, dropped=0.1)
    for gather in (False, True):
        x = quantize_rows(normal((n if gather else n * k, inner), 1))
        w = quantize_rows(normal((count, outer, inner), 2, scale=inner ** -0.5))
        y = grouped_matmul(x, w, groups, gather=gather, out_dtype=dt)
        assert y.dtype == dt
        xd, wd = (q.values.double() * q.scales.double().unsqueeze(-1) for q in (x, w))
        want, size, *_ = product_reference(xd, wd, groups, gather)
        close(y, want, want.abs() * half_step(dt) + steps(inner) * size + tiny(dt), "y")
    odd = quantize_rows(normal((count, outer, inner), 2))
    w = QuantizedRows(odd.values.transpose(1, 2).contiguous().transpose(1, 2), odd.scales)
    assert torch.equal(grouped_matmul(x, w, groups, gather=True).double(), grouped_matmul(x, odd, groups, gather=True).double())


def test_gradients_are_not_differentiable_again():
    from featgraph.module import combine_rows, grouped_matmul, rms_norm, route
    x = normal((6, 8), 1).requires_grad_(True)
    groups = make_groups(6, 1, 2, 5)
    w = normal((2, 8, 8), 2).requires_grad_(True)
    for out in (rms_norm(x), route(x, 2).weights, grouped_matmul(x, w, groups), combine_rows(x, groups)):
        grad, = torch.autograd.grad(out.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            grad.sum().backward()


def test_expanded_gradients_and_repeated_choices():
    """A sum's gradient arrives as an expanded tensor; a row may name the same group twice."""
    from featgraph.module import combine_rows, group_rows, grouped_matmul, rms_norm
    keys = torch.tensor([[0, 0], [1, 0], [2, 2], [-1, 1]], dtype=torch.int32, device="cuda")
    groups = group_rows(keys, 3)
    for t in sorted(TYPES):
        dt = TYPES[t]
        x, w = normal((4, 16), 1, dt).requires_grad_(True), normal((3, 8, 16), 2, dt).requires_grad_(True)
        weights = normal((4, 2), 3).requires_grad_(True)
        out = combine_rows(grouped_matmul(x, w, groups, gather=True), groups, weights)
        got = torch.autograd.grad(out.sum(), (x, w, weights))
        xd, wd, sd = (v.detach().double().requires_grad_(True) for v in (x, w, weights))
        want = sum(torch.where(keys[:, j:j + 1] >= 0, sd[:, j:j + 1] * torch.einsum("ni,noi->no", xd, wd[keys[:, j].clamp(min=0).long()]), torch.zeros((), dtype=torch.float64, device="cuda"))
                   for j in range(2))
        # three roundings to the type on each way (slot, sum, gradient) of values below 8
        close(out.detach(), want.detach(), 24 * half_step(dt) * (1 + want.detach().abs()), "out")
        for a, b in zip(got, torch.autograd.grad(want.sum(), (xd, wd, sd))):
            close(a, b, 24 * half_step(dt) * (1 + b.abs().max()), "gradients")
        y = normal((5, 24), 4, dt).requires_grad_(True)
        g = normal((24,), 5).requires_grad_(True)  # a 32-bit weight beside rows of fewer bits
        dy, dg = torch.autograd.grad(rms_norm(y, g).sum(), (y, g))
        assert dg.dtype == torch.float32
        yd, gd = y.detach().double().requires_grad_(True), g.detach().double().requires_grad_(True)
        by, bg = torch.autograd.grad(norm_reference_graph(yd, gd).sum(), (yd, gd))
        close(dy, by, half_step(dt) * by.abs() + 200 * U * (1 + by.abs().max()), "dx")
        close(dg, bg, 200 * U * (1 + bg.abs().max()), "dweight")


def norm_reference_graph(h, w, eps=1e-6):
    return h / torch.sqrt(h.pow(2).mean(-1, keepdim=True) + eps) * w


def test_product_from_a_thread_that_made_no_cuda_call_yet():
    """A host thread has no CUDA context until its first runtime call; the tensor maps need one."""
    import threading

    from featgraph.module import grouped_matmul
    groups = make_groups(200, 1, 2, 5)
    x, w = normal((200, 64), 1, torch.bfloat16), normal((2, 64, 64), 2, torch.bfloat16)
    want, got = grouped_matmul(x, w, groups), []
    torch.cuda.synchronize()
    thread = threading.Thread(target=lambda: got.append(grouped_matmul(x, w, groups)))
    thread.start()
    thread.join()
    assert got and torch.equal(got[0], want)


def test_product_has_the_same_bits_again():
    from featgraph.module import grouped_matmul
    for t in sorted(TYPES):
        groups = make_groups(5000, 2, 6, 5)
        x, w, dy = normal((5000, 136), 1, TYPES[t]), normal((6, 72, 136), 2, TYPES[t]), normal((10000, 72), 3, TYPES[t])
        x, w = x.requires_grad_(True), w.requires_grad_(True)
        runs = []
        for _ in range(3):
            y = grouped_matmul(x, w, groups, gather=True)
            runs.append((y.detach(), *torch.autograd.grad(y, (x, w), dy)))
        for other in runs[1:]:
            assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_lists_out_of_range_are_skipped_not_followed():
    """Lists that name entries beyond the rows give zero rows; nothing is read outside the arrays."""
    from featgraph.module import RowGroups, combine_rows, grouped_matmul
    offsets = torch.tensor([0, 2, 4, 900], dtype=torch.int32, device="cuda")
    order = torch.tensor([0, 77, -5, 3, 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    position = torch.tensor([[0, 99], [-1, 3], [2 ** 31 - 1, -7]], dtype=torch.int32, device="cuda")
    groups = RowGroups(offsets, order, position)
    for t in sorted(TYPES):
        x, w = normal((3, 32), 1, TYPES[t]), normal((3, 16, 32), 2, TYPES[t])
        x.requires_grad_(True), w.requires_grad_(True)
        y = grouped_matmul(x, w, groups, gather=True)
        zero = ~y.detach().any(1)
        assert zero.tolist() == [False, True, True, False, False, True]
        torch.autograd.grad(y, (x, w), torch.ones_like(y))
        assert torch.isfinite(combine_rows(y.detach(), groups)).all()


# ---- weighted sum back ----

@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,k,d", [(1, 1, 1), (3, 2, 7), (50, 4, 64), (16, 8, 1024), (33, 32, 100), (1000, 3, 72), (9, 1, 5000), (257, 2, 331)])
def test_combine(t, n, k, d):
    from featgraph.module import combine_rows
    dt = TYPES[t]
    groups = make_groups(n, k, 9, 5, dropped=0.2)
    y, w, dout = normal((n * k, d), 1, dt), normal((n, k), 2), normal((n, d), 3, dt)
    used = int(groups.offsets[-1])
    y[used:] = float("nan")  # rows in no group are never read
    for weights in (None, w):
        yl = y.clone().requires_grad_(True)
        wl = None if weights is None else weights.clone().requires_grad_(True)
        out = combine_rows(yl, groups, wl)
        at = groups.position.long()
        rows = torch.where((at >= 0).unsqueeze(2), y.double()[at.clamp(min=0)], torch.zeros((), dtype=torch.float64, device="cuda"))
        scale = torch.ones_like(w, dtype=torch.float64) if weights is None else w.double()
        terms = rows * scale.unsqueeze(2)
        want = terms.sum(1)
        close(out.detach(), want, want.abs() * half_step(dt) + (k + 1) * U * terms.abs().sum(1) + tiny(dt), "out")
        grads = torch.autograd.grad(out, [yl] if weights is None else [yl, wl], dout)
        dy = torch.zeros((n * k + 1, d), dtype=torch.float64, device="cuda")
        dy[torch.where(at >= 0, at, n * k).reshape(-1)] = (dout.double().unsqueeze(1) * scale.unsqueeze(2)).reshape(-1, d)
        dy = dy[:n * k]
        dy[used:] = 0
        close(grads[0], dy, dy.abs() * (half_step(dt) + U) + tiny(dt), "dy")
        if weights is not None:
            dot = rows * dout.double().unsqueeze(1)
            # a lane adds at most d / 32 + 8 terms, its warp 5
            close(grads[1], dot.sum(2), (d / 32 + 16) * U * dot.abs().sum(2), "dweights")


def test_combine_strided_rows():
    from featgraph.module import combine_rows
    groups = make_groups(40, 2, 3, 5)
    big = normal((80, 100), 1)
    w = normal((40, 2), 2)
    for y in (big[:, :64], big[:, 1:65], big[:, ::2]):
        assert torch.equal(combine_rows(y, groups, w), combine_rows(y.contiguous(), groups, w))


# ---- together, as they are used ----

def _layer(x, res, p, k, count, rows):
    y, h = rows.rms_norm(x, p["norm"], residual=res)
    r = rows.route(y @ p["router"].to(y.dtype), k)
    a = rows.grouped_matmul(y, p["up"], r.groups, gather=True)
    b = rows.grouped_matmul(torch.nn.functional.silu(a), p["down"], r.groups)
    return h + rows.combine_rows(b, r.groups, r.weights), r


@pytest.mark.parametrize("n", [1, 9, 400])
def test_a_routed_layer_and_an_aggregation_after_it(n):
    """Norm, router, two grouped products, weighted sum, then the framework's SpMM on the result: values and gradients
    against 64 bits.  The chain's 32-bit errors are a few hundred u of its largest intermediate: 1e-4 covers them."""
    import scipy.sparse as sp

    from featgraph_b200.module import rows
    from featgraph_b200.module.autograd import GraphOps
    d, hidden, count, k = 48, 72, 6, 2
    adj = sp.random(n, n, density=min(1.0, 4 / n), format="csr", random_state=1).astype(np.float32)
    adj.data[:] = 1
    x, res, dout = normal((n, d), 1), normal((n, d), 2), normal((n, d), 3)
    p = dict(norm=1 + normal((d,), 4, scale=0.1), router=normal((d, count), 5), up=normal((count, hidden, d), 6, scale=0.15),
             down=normal((count, d, hidden), 7, scale=0.15))
    leaves = [v.requires_grad_(True) for v in (x, res, *p.values())]
    out, r = _layer(x, res, p, k, count, rows)
    out = GraphOps(adj).spmm(out)
    grads = torch.autograd.grad(out, leaves, dout)
    xd, rd, *pd = [v.detach().double().requires_grad_(True) for v in leaves]
    nw, router, up, down = pd
    h = xd + rd
    y = h / torch.sqrt(h.pow(2).mean(1, keepdim=True) + 1e-6) * nw
    logits = y @ router
    index = r.experts.long()
    weights = torch.softmax(logits.gather(1, index), 1)
    moved = 0
    for j in range(k):
        a = torch.einsum("ni,noi->no", y, up[index[:, j]])
        moved = moved + weights[:, j:j + 1] * torch.einsum("ni,noi->no", torch.nn.functional.silu(a), down[index[:, j]])
    want = torch.from_numpy(adj.toarray()).cuda().double() @ (h + moved)
    close(out.detach(), want.detach(), 1e-4 * (1 + want.detach().abs()), "out")
    for name, a, b in zip(("x", "residual", *p), grads, torch.autograd.grad(want, (xd, rd, *pd), dout.double())):
        close(a, b, 1e-4 * (1 + b.abs().max()), name)


def test_a_captured_step_gives_what_an_eager_one_gives():
    """The layer's forward and backward as one graph, replayed on new contents; the groups' sizes change between
    replays.  Gradients go through torch.autograd.grad."""
    from featgraph_b200.module import rows
    from featgraph_b200 import graph_capture
    n, d, hidden, count, k = 200, 64, 96, 5, 2
    for t in sorted(TYPES):
        dt = TYPES[t]
        x, res, dout = (normal((n, d), s, dt) for s in (1, 2, 3))
        p = dict(norm=1 + normal((d,), 4, dt, 0.1), router=normal((d, count), 5, dt), up=normal((count, hidden, d), 6, dt, 0.15),
                 down=normal((count, d, hidden), 7, dt, 0.15))
        leaves = [v.requires_grad_(True) for v in (x, res, *p.values())]

        def step():
            out, r = _layer(x, res, p, k, count, rows)
            grads = torch.autograd.grad(out, leaves, dout)
            return [out.detach(), r.experts, r.groups.offsets, *grads]  # no graph stays alive between steps

        captured = graph_capture.capture(step)
        second = graph_capture.capture(step)  # two captured graphs share no workspace
        for seed in (11, 12):
            with torch.no_grad():
                x.copy_(normal((n, d), seed, dt))
                p["up"].copy_(normal((count, hidden, d), seed + 50, dt, 0.15))
            got = [v.clone() for v in captured.replay()]
            other = [v.clone() for v in second.replay()]
            want = step()
            for a, b, c in zip(got, other, want):
                assert torch.equal(a, c) and torch.equal(b, c)


def test_two_streams_at_once():
    from featgraph_b200.module import rows
    n, d, count, k = 3000, 128, 8, 2
    sets = []
    for s in range(2):
        x, res = normal((n, d), s, torch.bfloat16), normal((n, d), 10 + s, torch.bfloat16)
        p = dict(norm=normal((d,), 20 + s, torch.bfloat16), router=normal((d, count), 30 + s, torch.bfloat16), up=normal((count, 256, d), 40 + s, torch.bfloat16, 0.1),
                 down=normal((count, d, 256), 50 + s, torch.bfloat16, 0.1))
        sets.append((x, res, p))
    want = [_layer(*a, k, count, rows)[0] for a in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_layer(*sets[i], k, count, rows)[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_no_rows_at_all():
    from featgraph.module import combine_rows, group_rows, grouped_matmul, quantize_rows, rms_norm, route
    for t in sorted(TYPES):
        dt = TYPES[t]
        x = torch.empty((0, 24), device="cuda", dtype=dt).requires_grad_(True)
        w = normal((3, 8, 24), 1, dt).requires_grad_(True)
        r = route(torch.empty((0, 3), device="cuda", dtype=dt).requires_grad_(True), 2)
        assert r.weights.shape == (0, 2) and r.groups.offsets.tolist() == [0, 0, 0, 0]
        for groups in (r.groups, group_rows(torch.empty((0, 2), dtype=torch.int64, device="cuda"), 3)):
            y = grouped_matmul(x, w, groups, gather=True)
            out = combine_rows(y, groups, r.weights)
            dx, dw = torch.autograd.grad(out.sum() + rms_norm(x).sum(), (x, w))
            assert y.shape == (0, 8) and out.shape == (0, 8) and dx.shape == (0, 24) and not bool(dw.any())
        assert quantize_rows(x.detach()).scales.shape == (0,)
    # rows, but none of them in a group
    groups = group_rows(torch.full((5, 2), -1, dtype=torch.int32, device="cuda"), 3)
    x, w = normal((5, 24), 1).requires_grad_(True), normal((3, 8, 24), 2).requires_grad_(True)
    weights = normal((5, 2), 3).requires_grad_(True)
    out = combine_rows(grouped_matmul(x, w, groups, gather=True), groups, weights)
    assert not bool(out.any())
    assert not any(bool(g.any()) for g in torch.autograd.grad(out.sum(), (x, w, weights)))


def test_arrays_of_more_than_2_to_the_31_values():
    from featgraph.module import combine_rows, group_rows, grouped_matmul, rms_norm
    n, d, t = 140001, 16384, torch.bfloat16
    x = torch.empty((n, d), device="cuda", dtype=t)
    x[:2], x[-2:] = normal((2, d), 1, t), normal((2, d), 2, t)
    x[2:-2] = 1
    y = rms_norm(x)
    for rows in (slice(0, 2), slice(n - 2, n)):
        want, _ = norm_reference(x[rows], None)
        close(y[rows], want, want.abs() * (half_step(t) + STAT), "norm")
    del x, y
    n, inner, outer = 530001, 64, 4096
    groups = group_rows(torch.arange(n, device="cuda", dtype=torch.int32) % 3, 3)
    x, w = normal((n, inner), 3, t), normal((3, outer, inner), 4, t, inner ** -0.5)
    z = grouped_matmul(x, w, groups, gather=True)
    assert z.numel() > 2 ** 31
    out = combine_rows(z, groups)
    for row in (0, 1, n - 2, n - 1):
        xd, wd = x[row].double(), w[row % 3].double()
        want, size = wd @ xd, wd.abs() @ xd.abs()
        close(out[row], want, want.abs() * half_step(t) + steps(inner) * size, "row %d" % row)
    dx = torch.autograd.grad(combine_rows(z.requires_grad_(True), groups), z, out)[0]
    assert torch.equal(dx[-1], out[groups.order[-1].long()])


def test_refusals_that_need_a_device():
    from featgraph.module import grouped_matmul, quantize_rows, rms_norm
    x = normal((4, 8), 1).requires_grad_(True)
    with pytest.raises(ValueError, match="no gradient"):
        rms_norm(x, quantize=True)
    with pytest.raises(ValueError, match="no gradient"):
        quantize_rows(x)
    with torch.no_grad():
        rms_norm(x, quantize=True)
    with pytest.raises(ValueError, match="lives on cpu"):
        rms_norm(x, torch.ones(8))
    with pytest.raises(ValueError, match="lives on cpu"):
        grouped_matmul(x, torch.zeros(3, 5, 8), make_groups(4, 1, 3, 1))


def test_no_wait_ever_ran_out():
    """Runs last: the products' bounded waits (for their own copies) all ended in time in this process."""
    from featgraph_b200 import _native
    assert _native.lib().fg_wait_status(torch.cuda.current_stream().cuda_stream) == 0
