"""Row operators (``featgraph_b200.module.rows``) at the ends of their range: sums that cancel or leave a 16-bit type's range
on the way, the smallest and largest 32-bit values, infinities, lists that change under a backward pass, limits that two
host threads need at once.  Tolerances count roundings: half a step of the type for a rounding to it, u = 2^-24 for one to 32 bits,
twice that where the tensor cores cut a sum off."""
import threading

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


def within(got, want, tol, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all()), "%s: not finite" % what
    over = float(((got - want).abs() - tol).max())
    assert over <= 0.0, "%s: over its tolerance by %.3g (largest value %.3g)" % (what, over, float(want.abs().max()))


def normal(shape, seed, t=torch.float32, scale=1.0):
    return (torch.randn(shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) * scale).to(t)


def choose(n, k, count, seed):
    """k different groups for each row."""
    from featgraph.module import group_rows
    score = torch.rand((n, count), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return group_rows(torch.topk(score, k, dim=1).indices.int(), count)


# ---- the gradient of gathered rows: a sum over a row's slots ----

@pytest.mark.parametrize("t", sorted(TYPES))
@pytest.mark.parametrize("n,k,count,inner,outer", [(3, 2, 4, 16, 8), (130, 4, 9, 72, 48), (700, 8, 16, 128, 264), (33, 32, 40, 31, 17), (900, 1, 3, 64, 40),
                                                   (5000, 3, 5, 264, 96)])
def test_gradient_of_gathered_rows_is_rounded_once(t, n, k, count, inner, outer):
    """dx[t] = sum over j of W[g(t, j)]^T dy[slot(t, j)]: 32-bit sums throughout, and one rounding to the type."""
    from featgraph.module import grouped_matmul
    dt = TYPES[t]
    groups = choose(n, k, count, 1)
    x, w, dy = normal((n, inner), 2, dt).requires_grad_(True), normal((count, outer, inner), 3, dt), normal((n * k, outer), 4, dt)
    dx, = torch.autograd.grad(grouped_matmul(x, w, groups, gather=True), x, dy)
    want, size = (torch.zeros((n, inner), dtype=torch.float64, device="cuda") for _ in range(2))
    at, source = groups.offsets.tolist(), groups.order.long() // k
    for g in range(count):
        rows = slice(at[g], at[g + 1])
        want.index_add_(0, source[rows], dy[rows].double() @ w[g].double())
        size.index_add_(0, source[rows], dy[rows].double().abs() @ w[g].double().abs())
    # a term passes outer / 16 cut-off additions and the inside of one, in fp32 six parts' sums, then k slots
    within(dx, want, want.abs() * half_step(dt) + (2 * (outer / 16 + 24) + k) * U * size + tiny(dt), "dx")


@pytest.mark.parametrize("parts", [(70000.0, -20000.0), (70000.0, -70000.0), (-60000.0, 30000.0), (65504.0, 0.0)])
def test_gradient_of_gathered_rows_whose_slots_leave_the_range_of_fp16(parts):
    """The parts of two slots may be larger than fp16 holds where their sum is not."""
    from featgraph.module import group_rows, grouped_matmul
    n, inner, outer = 40, 24, 16
    groups = group_rows(torch.tensor([[0, 1]] * n, dtype=torch.int32, device="cuda"), 2)
    x = normal((n, inner), 1, torch.float16).requires_grad_(True)
    w = torch.zeros((2, outer, inner), device="cuda", dtype=torch.float16)
    dy = torch.zeros((2 * n, outer), device="cuda", dtype=torch.float16)
    dy[:, 3] = 1024.0
    w[0, 3], w[1, 3] = parts[0] / 1024, parts[1] / 1024
    dx, = torch.autograd.grad(grouped_matmul(x, w, groups, gather=True), x, dy)
    want = (1024 * (w[0, 3].double() + w[1, 3].double())).expand(n, inner)
    within(dx, want, want.abs() * half_step(torch.float16), "dx")


# ---- 8-bit rows of very small values ----

@pytest.mark.parametrize("d", [2, 31, 128, 129, 1000, 4096])
@pytest.mark.parametrize("most", [1.4e-45, 1e-44, 3.1e-43, 3.2e-43, 6.2e-43, 9e-43, 1e-42, 3e-42, 1e-41, 1e-40, 1e-38])
def test_8_bit_rows_of_the_smallest_values(d, most):
    """A finite row stays finite: no scale of 0, nothing beyond the largest 8-bit value."""
    from featgraph.module import quantize_rows, rms_norm
    x = torch.zeros((3, d), device="cuda")
    x[0, 0] = most
    x[1] = normal((d,), 1).clamp(-1, 1) * most
    x[1, d // 2] = -most
    unit = 2.0 ** -149
    for q in (quantize_rows(x), rms_norm(x * 2 ** 60, eps=1.0, weight=torch.full((d,), 2.0 ** -60, device="cuda"), quantize=True)):
        values, scales = q.values.double(), q.scales.double()
        assert bool(torch.isfinite(values).all()) and bool((scales > 0).all())
        # half a step of 2^-3 of the value (and of the next 8-bit number down, near 0), and the smallest 32-bit steps; a row that
        # is too small for a scale of its own becomes zeros
        back = values * scales.unsqueeze(1)
        want = x.double()
        lost = torch.where(scales == 1.0, 224.5 * unit, 0.0).unsqueeze(1)
        held = torch.where(scales == 1.0, 0.0, scales).unsqueeze(1)
        within(back, want, want.abs() * (2.0 ** -4 + 2.0 ** -10) + held * 2.0 ** -10 * 1.001 + lost + 2 * unit, "values")
        quotient = x[:2].double().abs().amax(1) / 448
        given = scales[:2]
        assert bool(torch.where(given == 1.0, quotient <= 0.51 * unit, (given - quotient).abs() <= 1.01 * unit + quotient * 4 * U).all())
        assert float(scales[2]) == 1.0 and not bool(values[2].any())


# ---- fp32 products: parts of the operands ----

def patterns():
    """Significands whose bits after the eighth are all ones, all zeros but the last, halfway, and random ones; both signs."""
    base = [1 + 2.0 ** -7 - 2.0 ** -23, 2 - 2.0 ** -23, 1 + 2.0 ** -8, 1 + 2.0 ** -8 - 2.0 ** -23, 1 + 2.0 ** -16, 1 + 2.0 ** -16 - 2.0 ** -23,
            1 + 2.0 ** -8 + 2.0 ** -16, 1.5 + 2.0 ** -7 - 2.0 ** -15, 1 + 2.0 ** -23, 1.0]
    some = (1 + torch.rand(54, generator=torch.Generator().manual_seed(3), dtype=torch.float64)).tolist()
    v = torch.tensor(base + some, dtype=torch.float32, device="cuda")
    return torch.cat([v, -v])


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("inner", [1, 4, 40])
@pytest.mark.parametrize("outer", [128, 200])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** 40, 2.0 ** -60])
def test_a_single_fp32_product_is_within_its_bound(gather, inner, outer, scale):
    """One nonzero term a sum: what the parts leave out is below 2^-24 (1 + 2^-9) of it, the last of the six sums is cut
    off at 24 bits (2 u), the five before it are below 2^-6 of the term (2^-6 x 5 x 2 u)."""
    from featgraph.module import group_rows, grouped_matmul
    v = patterns()
    n = v.numel()
    x, w = torch.zeros((n, inner), device="cuda"), torch.zeros((2, outer, inner), device="cuda")
    x[:, 0] = v * scale
    column = v.repeat(outer // n + 1)[:outer]
    w[0, :, 0], w[1, :, 0] = column, -column.flip(0)
    keys = (torch.arange(n, device="cuda", dtype=torch.int32) % 2)
    groups = group_rows(keys, 2)
    order = groups.order.long()
    leaf, weight = (x if gather else x[order].contiguous()).requires_grad_(True), w.clone().requires_grad_(True)
    y = grouped_matmul(leaf, weight, groups, gather=gather)
    want = x.detach().double()[order][:, :1] * w.double()[keys[order].long()][:, :, 0]
    bound = (1 + 2.0 ** -9 + 2 + 10 * 2.0 ** -6) * U
    within(y.detach(), want, bound * want.abs(), "y")
    # the gradient of x reads the weight the other way: one nonzero output a row
    dy = torch.zeros_like(y)
    dy[torch.arange(n, device="cuda"), torch.arange(n, device="cuda") % outer] = v * scale
    dx, = torch.autograd.grad(y, leaf, dy)
    dx = dx[order] if gather else dx
    want = (v.double() * scale) * w.double()[keys[order].long(), torch.arange(n, device="cuda") % outer, 0]
    within(dx[:, 0], want, (bound + U) * want.abs(), "dx")


def test_largest_and_smallest_fp32_values():
    from featgraph.module import group_rows, grouped_matmul
    n = 64
    groups = group_rows(torch.zeros(n, dtype=torch.int32, device="cuda"), 1)
    top = torch.finfo(torch.float32).max
    x = torch.zeros((n, 8), device="cuda")
    x[:, 0] = torch.tensor([top, -top, top * (1 - 2.0 ** -9), top / 2, 2.0 ** 127, 1.0, (1 + 2.0 ** -23) * 2.0 ** -112,
                            (1 + 2.0 ** -7 - 2.0 ** -23) * 2.0 ** -105], device="cuda").repeat(8)
    w = torch.zeros((1, 16, 8), device="cuda")
    w[0, :, 0] = torch.tensor([1.0, -1.0, 0.5, 0.75] * 4, device="cuda")
    y = grouped_matmul(x, w, groups)
    want = x.double()[:, :1] * w[0].double()[:, 0]
    # below 2^-110 a value's bits under 2^-133 are cut off
    within(y, want, (1 + 2.0 ** -9 + 2 + 10 * 2.0 ** -6) * U * want.abs() + 2.0 ** -133, "y")


# ---- infinities ----

@pytest.mark.parametrize("n", [1, 8, 32, 33, 200])
@pytest.mark.parametrize("t", sorted(TYPES))
def test_an_infinity_stays_in_its_row(t, n):
    """16 bits: what the sum gives.  fp32: the sum's infinity for up to 32 slots of a weight with a dense inner axis, NaN for more."""
    from featgraph.module import group_rows, grouped_matmul
    dt = TYPES[t]
    groups = group_rows(torch.zeros(n, dtype=torch.int32, device="cuda"), 1)
    x, w = normal((n, 40), 1, dt), normal((1, 24, 40), 2, dt)
    row = n // 2
    x[row, 5] = float("-inf")
    y = grouped_matmul(x, w, groups)
    others = torch.arange(n, device="cuda") != row
    assert bool(torch.isfinite(y[others]).all())
    if dt == torch.float32 and n > 32:
        assert bool(torch.isnan(y[row]).all())
    else:
        assert torch.equal(y[row], torch.where(w[0, :, 5] > 0, float("-inf"), float("inf")).to(dt))


# ---- lists that change under a backward pass ----

@pytest.mark.parametrize("which", ["offsets", "order", "position"])
def test_lists_refilled_before_the_backward_pass_are_noticed(which):
    from featgraph.module import RowGroups, combine_rows, grouped_matmul
    made = choose(50, 2, 4, 1)
    x, w = normal((50, 16), 2).requires_grad_(True), normal((4, 24, 16), 3).requires_grad_(True)
    rows, weights = normal((100, 24), 4).requires_grad_(True), normal((50, 2), 5).requires_grad_(True)
    for call in (lambda g: grouped_matmul(x, w, g, gather=True), lambda g: combine_rows(rows, g, weights)):
        groups = RowGroups(made.offsets.clone(), made.order.clone(), made.position.clone())
        out = call(groups)
        getattr(groups, which).copy_(getattr(choose(50, 2, 4, 9), which))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
        out = call(made)
        out.sum().backward()  # untouched lists are fine


def test_lists_made_in_inference_mode_serve_a_training_step():
    from featgraph.module import combine_rows, group_rows, grouped_matmul
    keys = torch.arange(100, device="cuda", dtype=torch.int32).view(50, 2) % 4
    with torch.inference_mode():
        fixed = group_rows(keys, 4)
    x, w = normal((50, 16), 2).requires_grad_(True), normal((4, 24, 16), 3).requires_grad_(True)
    weights, dout = normal((50, 2), 5).requires_grad_(True), normal((50, 24), 6)
    got, want = (torch.autograd.grad(combine_rows(grouped_matmul(x, w, groups, gather=True), groups, weights), (x, w, weights), dout)
                 for groups in (fixed, group_rows(keys, 4)))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- waits ----

def test_waits_are_reported():
    from featgraph.module import check_waits
    x = normal((100, 300), 1)
    from featgraph.module import quantize_rows
    quantize_rows(x)
    assert check_waits() is None and check_waits("cuda:0") is None and check_waits(x.device) is None


def test_a_wait_that_ran_out_is_raised(monkeypatch):
    """The answer of the library is a fake here: no wait is made to run out."""
    from featgraph.module import check_waits
    from featgraph_b200 import _native
    from featgraph_b200.module import rows
    monkeypatch.setitem(rows._entries, "fg_wait_status", lambda stream: 2)
    with pytest.raises(_native.FeatGraphError):
        check_waits()


def test_waits_are_not_asked_for_in_a_capture():
    from featgraph.module import check_waits
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="cannot be captured"):
            check_waits()
    graph.replay()
    assert check_waits() is None and float(x[0]) == 1.0


# ---- two host threads ----

def test_gradients_of_different_widths_from_two_threads():
    """The widest fp32 rows with a residual's gradient take more shared memory than others of the same kernel: a limit that one
    thread sets is never below what another one's launch needs."""
    from featgraph_b200 import _native
    call, refused = _native.lib().fg_rms_norm_backward, []

    def work(d, n=2):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            h, dy, dh, dx = (torch.ones((n, d), device="cuda") for _ in range(4))
            args = (h.data_ptr(), d, None, dy.data_ptr(), d, dh.data_ptr(), d, dx.data_ptr(), None, None, n, n, d, 1e-6, 0, 0, stream.cuda_stream)
            for i in range(20000):
                if call(*args):
                    refused.append((d, i))
                if i % 256 == 0:
                    stream.synchronize()
            stream.synchronize()

    threads = [threading.Thread(target=work, args=(d,)) for d in (16384, 9000)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not refused, "%d launches were refused, the first %s" % (len(refused), refused[0])


# ---- norm without eps ----

@pytest.mark.parametrize("d", [24, 128, 300, 2048])
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -50, 2.0 ** 40])
def test_norm_gradient_of_small_and_large_rows_without_eps(d, size):
    """r = 1 / |h| reaches 1e18 and its square leaves the 32-bit range where the gradient, r times g, does not."""
    from featgraph.module import rms_norm
    x, dy = normal((20, d), 1, scale=size).requires_grad_(True), normal((20, d), 2, scale=1e4)
    dx, = torch.autograd.grad(rms_norm(x, eps=0.0), x, dy)
    h, g = x.detach().double(), dy.double()
    r = 1 / torch.sqrt(h.pow(2).mean(1, keepdim=True))
    first, second = r * g, h * r ** 3 * (g * h).sum(1, keepdim=True) / d
    parts = first.abs() + h.abs() * r ** 3 * (g * h).abs().sum(1, keepdim=True) / d
    within(dx, first - second, (first - second).abs() * U + 240 * U * parts, "dx")  # 240 u: the statistics' additions, as for rows near 1


# ---- row numbers near 2^31 ----

def test_weight_gradient_of_almost_2_to_the_31_rows():
    """A group's last part ends with the group, also where row numbers and part sizes add up to more than 32 bits hold."""
    from featgraph.module import RowGroups, grouped_matmul
    m, width = 2 ** 31 - 2048, 8
    x = torch.zeros((m, width), device="cuda", dtype=torch.bfloat16)
    x[-5:] = 1
    x[:3] = 2
    lists = torch.empty(m, device="cuda", dtype=torch.int32)  # not read: the rows are in slot order
    groups = RowGroups(torch.tensor([0, m - 3000, m], dtype=torch.int32, device="cuda"), lists, lists.view(m, 1))
    w = torch.ones((2, width, width), device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    y = grouped_matmul(x, w, groups)
    assert bool((y.detach()[-5:] == 8).all()) and bool((y.detach()[:3] == 16).all()) and not bool(y.detach()[-6].any())
    dw, = torch.autograd.grad(y, w, y.detach())
    assert bool((dw[0] == 3 * 16 * 2).all()) and bool((dw[1] == 5 * 8).all()), dw[:, 0, 0]  # whole numbers below 2^8: exact
    del x, y, lists, groups  # 77 GB: not kept from the tests that follow
    torch.cuda.empty_cache()
