"""Linear layer with bias, activation and residual against the formula in 64 bits.

Tolerances.  u = 2^-24; e half a step of the operands' type; S = sum_k |x w|.
  z    16-bit and 8-bit products are exact in fp32; an MMA step adds 16 (32) of them to the running sum
       and cuts the result, at most 2 u of S a step and as much again for each product inside it:
       2 (K / 16 + 16) u S.  fp32: the split operands drop at most 2^-19 + 2^-20 of a product
       (truncated low parts, low times low), 24 cutting steps of 2 u, then K / 64 + 8 rounding adds.
  act  no activation has a slope beyond 1.13; its own evaluation is off by at most 2^-20 |z| (the gelu of
       16-bit results: 0.75e-7 |z| from its approximation and 8 u |z| from the exponential).
  gz   grad_y * act'(z) at the stored z: no second derivative is beyond 1, so e |z| (z rounded to its type)
       and the error of z itself count once each; relu and leaky_relu have a step where z is within
       its error of zero.  gz is rounded once before its products (e), whose sums are bounded as above."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = [None, "relu", "leaky_relu", "elu", "gelu", "silu"]
SLOPE = 0.1
# rows, inner, outer
SIZES = [(1, 1, 1), (1, 64, 128), (3, 7, 5), (1, 1000, 77), (2, 4096, 96), (8, 512, 40), (9, 520, 264), (16, 136, 1000),
         (17, 256, 64), (31, 90, 33), (32, 1024, 512), (33, 64, 64), (100, 602, 41), (128, 128, 128), (200, 48, 300),
         (300, 1433, 64), (513, 256, 257), (1000, 128, 1000), (64, 9000, 70), (2600, 136, 2100), (5000, 64, 8)]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return torch.finfo(dt).smallest_normal * half_step(dt)


def within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.3g} x tolerance"


def sum_error(dt, k):
    """Error of a product's sum of k terms, in units of the sum of magnitudes."""
    if dt == torch.float32:
        return 2.0 ** -19 + 2.0 ** -20 + 48 * U + (k / 64 + 8) * U
    return 2 * (k / 16 + 16) * U


def act64(z, act):
    f = torch.nn.functional
    return {None: lambda v: v, "relu": f.relu, "leaky_relu": lambda v: f.leaky_relu(v, SLOPE), "elu": f.elu, "gelu": f.gelu,
            "silu": f.silu}[act](z)


def forward_bound(x, w, b, act, r, dt, e_sum, extra=0.0):
    """(z, error of z, y, tolerance of y) in 64 bits."""
    z, s = x @ w.t(), x.abs() @ w.abs().t()
    err = (e_sum + extra) * s
    if b is not None:
        z = z + b
        err = err + U * (s + b.abs())
    y = act64(z, act)
    err_y = 1.13 * err + (2.0 ** -20 * z.abs() if act in ("gelu", "silu", "elu") else 2 * U * z.abs())
    if r is not None:
        y = y + r
        err_y = err_y + U * y.abs() + U * err_y
    return z, err, y, (half_step(dt) * y.abs() + err_y) * (1 + half_step(dt)) + tiny(dt)


def make(cuda, m, k, n, dt, seed=0):
    gen = torch.Generator().manual_seed(m * 7 + k * 3 + n + seed)
    rnd = lambda *s: torch.randn(*s, generator=gen)
    return ((rnd(m, k)).to(dt).to(cuda), (rnd(n, k) / k ** 0.5).to(dt).to(cuda), (0.3 * rnd(n)).to(dt).to(cuda),
            rnd(m, n).to(dt).to(cuda), rnd(m, n).to(dt).to(cuda))


def check(cuda, m, k, n, dt, act, bias, residual):
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    x, w, b, r, g = make(cuda, m, k, n, dt)
    b, r = (b if bias else None), (r if residual else None)
    D = lambda t: None if t is None else t.double()
    z, err_z, want, tol = forward_bound(D(x), D(w), D(b), act, D(r), dt, sum_error(dt, k))
    y0 = linear_act(x, w, b, act, r, SLOPE)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    args = [None if t is None else next(it) for t in (x, w, b, r)]
    y = linear_act(args[0], args[1], args[2], act, args[3], SLOPE)
    dense.check_status()
    assert y.shape == (m, n) and y.dtype == dt and torch.equal(y, y0)
    within(y, want, tol, "y")

    grads = torch.autograd.grad(y, leaves, g)
    dense.check_status()
    gx, gw = grads[0], grads[1]
    assert all(a.dtype == dt and a.shape == t.shape for a, t in zip(grads, leaves))
    if residual:
        assert torch.equal(grads[-1], g)
    zl = z.detach().clone().requires_grad_(True)
    slope = torch.autograd.grad(act64(zl, act).sum(), zl)[0]
    gd = g.double()
    gz = gd * slope
    e = half_step(dt)
    err = torch.zeros_like(gz)
    if act in ("elu", "gelu", "silu"):
        err = gd.abs() * (e * z.abs() + err_z + 2.0 ** -20 * (1 + z.abs())) + U * gz.abs()
    elif act in ("relu", "leaky_relu"):
        err = gd.abs() * (z.abs() <= err_z + tiny(dt)) + U * gz.abs()
    if bias:
        tol = e * gz.sum(0).abs() + err.sum(0) + (m / 8 + 300) * U * gz.abs().sum(0)
        within(grads[2], gz.sum(0), tol * (1 + e) + tiny(dt), "grad_bias")
    if act is not None:
        err = err + e * gz.abs() + e * err + tiny(dt)
    W, X = w.double(), x.double()
    want = gz @ W
    tol = e * want.abs() + err @ W.abs() + sum_error(dt, n) * ((gz.abs() + err) @ W.abs())
    within(gx, want, tol * (1 + e) + tiny(dt), "grad_x")
    want = gz.t() @ X
    tol = e * want.abs() + err.t() @ X.abs() + sum_error(dt, m) * ((gz.abs() + err).t() @ X.abs())
    within(gw, want, tol * (1 + e) + tiny(dt), "grad_w")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,k,n", SIZES)
def test_forward_and_backward(cuda, m, k, n, dtype):
    check(cuda, m, k, n, DT[dtype], "gelu", True, True)
    check(cuda, m, k, n, DT[dtype], None, False, False)


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("bias,residual", [(True, False), (False, True)])
def test_every_activation(cuda, act, bias, residual, dtype):
    for m, k, n in ((5, 200, 72), (150, 96, 100), (260, 128, 136)):
        check(cuda, m, k, n, DT[dtype], act, bias, residual)


def to_8_bits(v):
    scale = v.abs().amax(1, keepdim=True).clamp_min(1e-30) / 448
    return (v / scale).to(torch.float8_e4m3fn), scale


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("m,k,n", SIZES)
def test_8_bit_operands(cuda, m, k, n, dtype):
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act_fp8

    dt = DT[dtype]
    gen = torch.Generator().manual_seed(m + k + n)
    x8, xs = to_8_bits(torch.randn(m, k, generator=gen).to(cuda))
    w8, ws = to_8_bits((torch.randn(n, k, generator=gen) / k ** 0.5).to(cuda))
    b = torch.randn(n, generator=gen).to(dt).to(cuda)
    r = torch.randn(m, n, generator=gen).to(dt).to(cuda)
    x, w = x8.to(torch.float64) * xs.double(), w8.to(torch.float64) * ws.double()
    for act, bias, res in ((None, None, None), ("silu", b, r), ("relu", None, r)):
        y = linear_act_fp8(x8, xs, w8, ws.view(-1), bias, act, res, SLOPE, dt)
        dense.check_status()
        assert y.dtype == dt
        # two more factors: 3 u
        _, _, want, tol = forward_bound(x, w, None if bias is None else b.double(), act, None if res is None else r.double(),
                                        dt, 2 * (k / 16 + 32) * U, 3 * U)
        within(y, want, tol, f"y ({act})")


def test_norm_and_product_in_8_bits(cuda):
    """The two 8-bit operators as a block uses them: norm with the residual -> product, against the same
    steps in 64 bits on the values that the 8 bits stand for."""
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act_fp8
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm_fp8

    gen = torch.Generator().manual_seed(1)
    x, r = (torch.randn(3, 50, 512, generator=gen).to(torch.bfloat16).to(cuda) for _ in range(2))
    g = torch.ones(512, dtype=torch.bfloat16, device=cuda)
    w8, ws = to_8_bits((torch.randn(384, 512, generator=gen) / 512 ** 0.5).to(cuda))
    q, s, h = add_rms_norm_fp8(x, g, r)
    y = linear_act_fp8(q, s, w8, ws, None, "gelu", None)
    dense.check_status()
    assert y.shape == (3, 50, 384)
    xq = (q.to(torch.float64) * s.double()).view(-1, 512)
    _, _, want, tol = forward_bound(xq, w8.to(torch.float64) * ws.double(), None, "gelu", None, torch.bfloat16,
                                    2 * (512 / 16 + 32) * U, 3 * U)
    within(y.view(-1, 384), want, tol, "y")


def test_block_with_experts(cuda):
    """The operators together, forward and backward: norm with residual, rows to their experts, each
    expert's two layers on its rows, back with weights.  In fp32 against the same block in 64 bits."""
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm

    gen = torch.Generator().manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(cuda)
    t, d, hidden, e, k = 90, 64, 96, 4, 2
    x, res, gain = rnd(t, d), rnd(t, d), 1 + 0.1 * rnd(d)
    w1, b1, w2 = rnd(e, hidden, d) / 8, 0.1 * rnd(e, hidden), rnd(e, d, hidden) / 10
    router = rnd(e, d) / 8
    go = rnd(t, d)

    def ours(x, res, gain, w1, b1, w2, router):
        y, h = add_rms_norm(x, gain, res)
        probs, ids = torch.softmax(dense.linear(y, router), -1).topk(k, -1)
        order = expert_sort(ids, e)
        xs = expert_dispatch(y, order)
        at = order.offsets.tolist()
        parts = [linear_act(linear_act(xs[a:b], w1[i], b1[i], "silu"), w2[i]) for i, (a, b) in enumerate(zip(at, at[1:]))]
        return expert_combine(torch.cat(parts), probs, order) + h

    def plain(x, res, gain, w1, b1, w2, router):
        h = x + res
        y = h * (h.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * gain
        probs, ids = torch.softmax(y @ router.t(), -1).topk(k, -1)
        out = h
        for i in range(e):
            f = torch.nn.functional.silu(y @ w1[i].t() + b1[i]) @ w2[i].t()
            out = out + f * (probs * (ids == i)).sum(-1, keepdim=True)
        return out

    a = [v.clone().requires_grad_(True) for v in (x, res, gain, w1, b1, w2, router)]
    b = [v.double().requires_grad_(True) for v in (x, res, gain, w1, b1, w2, router)]
    out, want = ours(*a), plain(*b)
    got = torch.autograd.grad(out, a, go)
    dense.check_status()
    exp = torch.autograd.grad(want, b, go.double())
    # five operators in a row, each within a few 1e-6 of its largest terms
    for u, v in zip((out, *got), (want, *exp)):
        assert float((u.detach().double() - v.detach()).norm() / v.detach().norm()) < 2e-5


def test_leading_dimensions_strides_and_alignment(cuda):
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    for dt in DT.values():
        x, w, b, r, _ = make(cuda, 60, 72, 40, dt)
        y = linear_act(x, w, b, "silu", r)
        y3 = linear_act(x.view(4, 15, 72), w, b, "silu", r.view(4, 15, 40))
        assert y3.shape == (4, 15, 40) and torch.equal(y3.view(60, 40), y)
        assert torch.equal(linear_act(x[0], w, b, "silu", r[0]), linear_act(x[:1], w, b, "silu", r[:1])[0])
        wide = torch.zeros(60, 100, dtype=dt, device=cuda)
        wide[:, 5:77] = x
        assert torch.equal(linear_act(wide[:, 5:77], w, b, "silu", r), y)
        assert torch.equal(linear_act(x, w.t().contiguous().t(), b, "silu", r.t().contiguous().t()), y)
        shift = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view(t.shape).copy_(t)
        s = [shift(t) for t in (x, w, b, r)]
        assert all(t.data_ptr() % 16 for t in s)
        got = linear_act(s[0], s[1], s[2], "silu", s[3])
        assert float((got.double() - y.double()).abs().max()) <= 4 * half_step(dt) * float(y.double().abs().max())
        lx, lw = (t.clone().requires_grad_(True) for t in (s[0], s[1]))
        for a in torch.autograd.grad(linear_act(lx, lw, s[2], "silu", s[3]).sum(), (lx, lw)):
            assert bool(torch.isfinite(a).all())


def test_8_bit_operands_strided_shifted_and_empty(cuda):
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act_fp8

    gen = torch.Generator().manual_seed(14)
    for m, k in ((40, 96), (40, 100), (300, 96)):
        x8, xs = to_8_bits(torch.randn(m, k, generator=gen).to(cuda))
        w8, ws = to_8_bits(torch.randn(72, k, generator=gen).to(cuda))
        y = linear_act_fp8(x8, xs, w8, ws)
        wide = torch.zeros(m, k + 30, device=cuda).to(torch.float8_e4m3fn)
        wide[:, 7:7 + k] = x8
        assert torch.equal(linear_act_fp8(wide[:, 7:7 + k], xs, w8, ws), y)
        flat = torch.zeros(m * k + 3, device=cuda).to(torch.float8_e4m3fn)
        shifted = flat[3:].view(m, k)
        shifted.copy_(x8)
        assert torch.equal(linear_act_fp8(shifted, xs, w8, ws), y)
        assert torch.equal(linear_act_fp8(x8.view(4, m // 4, k), xs, w8, ws).view(m, 72), y)
        assert linear_act_fp8(x8[:0], xs[:0], w8, ws).shape == (0, 72)
        with torch.inference_mode():
            assert torch.equal(linear_act_fp8(x8, xs, w8, ws), y)


def test_empty_and_special_values(cuda):
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    for dt in DT.values():
        x, w, b, r, g = make(cuda, 40, 64, 48, dt)
        lx, lw, lb = (t.clone().requires_grad_(True) for t in (x[:0], w, b))
        y = linear_act(lx, lw, lb, "gelu")
        assert y.shape == (0, 48)
        gx, gw, gb = torch.autograd.grad(y.sum(), (lx, lw, lb))
        assert gx.shape == (0, 64) and not bool(gw.any()) and not bool(gb.any())
        clean = linear_act(x, w, b, "relu")
        x[7, 3], x[20, 5] = float("nan"), float("inf")
        y = linear_act(x, w, b, "relu")
        keep = [i for i in range(40) if i not in (7, 20)]
        assert torch.equal(y[keep], clean[keep]) and bool(y[7].isnan().all())
        # far out on both sides the activations stay finite
        far = torch.full((2, 64), 100.0, dtype=dt, device=cuda)
        far[1] = -100
        for act in ACTS[1:]:
            lf = far.clone().requires_grad_(True)
            y = linear_act(lf, torch.ones(8, 64, dtype=dt, device=cuda), None, act)
            assert bool(torch.isfinite(y).all()) and bool(torch.isfinite(torch.autograd.grad(y.sum(), lf)[0]).all())


def test_slopes_where_z_overflowed(cuda):
    """fp16 pre-activations of +-infinity: the activations' slopes are at their limits, 1 and 0."""
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    w = torch.full((8, 64), 60000.0, dtype=torch.float16, device=cuda)
    g = torch.ones(200, 8, dtype=torch.float16, device=cuda)
    b = torch.zeros(8, dtype=torch.float16, device=cuda, requires_grad=True)
    for sign, slope in ((1.0, 1.0), (-1.0, 0.0)):
        x = torch.full((200, 64), sign, dtype=torch.float16, device=cuda)
        for act in ("gelu", "silu", "relu", "elu"):
            gb, = torch.autograd.grad(linear_act(x, w, b, act), b, g)
            assert torch.equal(gb, torch.full_like(gb, 200 * slope))


def test_beyond_32_bit_offsets(cuda):
    """More than 2^31 elements in the output, its gradient and the saved pre-activation: the last rows
    are those of a small call."""
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    m, k, n = 270000, 64, 8192
    gen = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(m, k, generator=gen, device=cuda).to(torch.bfloat16).requires_grad_(True)
    w = (torch.randn(n, k, generator=gen, device=cuda) / 8).to(torch.bfloat16).requires_grad_(True)
    y = linear_act(x, w, None, "silu")
    g = torch.zeros_like(y)
    g[-300:] = torch.randn(300, n, generator=gen, device=cuda).to(torch.bfloat16)
    gx, gw = torch.autograd.grad(y, (x, w), g)
    dense.check_status()
    xs = x[-300:].detach().clone().requires_grad_(True)
    ys = linear_act(xs, w, None, "silu")
    gxs, gws = torch.autograd.grad(ys, (xs, w), g[-300:].contiguous())
    assert torch.equal(y[-300:], ys)
    for a, b in ((gx[-300:], gxs), (gw, gws)):  # other splits of the sums, one rounding each
        assert float((a.double() - b.double()).norm() / b.double().norm()) < 2 * half_step(torch.bfloat16)
    assert not bool(gx[:-300].any())


def test_parts_of_the_gradient(cuda):
    """Each leaf alone gives what all of them together give."""
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    for dt in (torch.bfloat16, torch.float32):
        t = make(cuda, 70, 40, 50, dt)
        ts, g = list(t[:4]), t[4]
        for act in (None, "gelu"):
            leaves = [v.clone().requires_grad_(True) for v in ts]
            want = torch.autograd.grad(linear_act(leaves[0], leaves[1], leaves[2], act, leaves[3]), leaves, g)
            for i in range(4):
                args = [v.clone() for v in ts]
                args[i].requires_grad_(True)
                got, = torch.autograd.grad(linear_act(args[0], args[1], args[2], act, args[3]), args[i], g)
                assert torch.equal(got, want[i])


def test_gradient_against_differences(cuda):
    """<grad, v> against a central difference of the fp32 forward.  Third derivatives along v are at
    most 3 |v|^3-sized at these sizes, so the quotient is off by t^2 times the loss's magnitude, plus the
    forward's rounding, sum_error, at both points over 2 t."""
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    x, w, b, r, g = make(cuda, 20, 32, 24, torch.float32)
    t = 2.0 ** -6
    for act in ("elu", "gelu", "silu", None):
        f = lambda a: (linear_act(a[0], a[1], a[2], act, a[3]).double() * g.double()).sum()
        leaves = [v.clone().requires_grad_(True) for v in (x, w, b, r)]
        grads = torch.autograd.grad(linear_act(leaves[0], leaves[1], leaves[2], act, leaves[3]), leaves, g)
        size = float((g.double().abs() * (x.double().abs() @ w.double().abs().t() + 1)).sum())
        gen = torch.Generator().manual_seed(4)
        for i in range(4):
            v = torch.randn(leaves[i].shape, generator=gen).to(cuda) / (4 if i == 1 else 1)
            up, down = [x, w, b, r], [x, w, b, r]
            up[i], down[i] = up[i] + t * v, down[i] - t * v
            quotient = float(f(up) - f(down)) / (2 * t)
            want = float((grads[i].double() * v.double()).sum())
            assert abs(quotient - want) <= (t * t + 2 * sum_error(torch.float32, 32) / t) * size


def test_long_reduction_does_not_drift(cuda):
    """Same-sign terms: the tensor core cuts off what does not fit its sum, 2^-26 of it a step on average;
    the sums are split before that shows in a 16-bit result, and sooner in fp32."""
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    gen = torch.Generator().manual_seed(6)
    for dt, k in ((torch.float16, 140000), (torch.float32, 40000)):
        x = (0.01 * (0.5 + torch.rand(40, k, generator=gen))).to(dt).to(cuda)
        w = (0.5 + torch.rand(24, k, generator=gen)).to(dt).to(cuda)
        y = linear_act(x, w)
        dense.check_status()
        want = x.double() @ w.double().t()
        rel = ((y.double() - want) / want).mean().abs()
        # 8192 steps without a break at most in 16 bits, 24 in fp32
        assert float(rel) < (8192 * 2.0 ** -26 if dt == torch.float16 else 2e-6)


def test_streams_graphs_and_scratch(cuda):
    """Captured forward and backward replay on new inputs; two graphs replayed at once on two streams
    share no scratch (the products are split over the reduction here)."""
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act

    gen = torch.Generator().manual_seed(9)
    sets = [[(torch.randn(s, generator=gen) / 8).to(torch.bfloat16).to(cuda) for s in ((200, 2048), (96, 2048), (96,), (200, 96))]
            for _ in range(2)]

    def step(x, w, b, g):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = linear_act(leaves[0], leaves[1], leaves[2], "gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, g))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    graphs, got = [], []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append(step(*s))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    dense.check_status()
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
    sets[0][0].copy_(sets[1][0])
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0][0], step(*sets[0])[0])


def test_two_streams_at_once(cuda):
    """Calls of every kernel on two streams at the same time give what they give alone."""
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act, linear_act_fp8

    gen = torch.Generator().manual_seed(12)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(cuda)
    calls = []
    for m in (3, 30, 60, 200, 1500):
        x, w, r = rnd(m, 1024).bfloat16(), (rnd(1000, 1024) / 32).bfloat16(), rnd(m, 1000).bfloat16()
        x8, xs = to_8_bits(rnd(m, 1024))
        w8, ws = to_8_bits(rnd(1000, 1024) / 32)
        calls.append(lambda x=x, w=w, r=r: linear_act(x, w, None, "gelu", r))
        calls.append(lambda x=x.float(), w=w.float(): linear_act(x, w, None, "silu"))
        calls.append(lambda x8=x8, xs=xs, w8=w8, ws=ws: linear_act_fp8(x8, xs, w8, ws))
    want = [f() for f in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = {s: [] for s in streams}
    for _ in range(6):
        for f in calls:
            for s in streams:
                with torch.cuda.stream(s):
                    got[s].append(f())
    torch.cuda.synchronize()
    dense.check_status()
    for s in streams:
        for i, y in enumerate(got[s]):
            assert torch.equal(y, want[i % len(calls)])


def test_training_step_as_one_graph(cuda):
    """A block of the operators with its optimizer as one captured step: the parameters after replays
    are those of the same steps run eagerly."""
    from ae_mlsys_gnn_b200.graphed import GraphedStep
    from ae_mlsys_gnn_b200.operators import dense
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm

    gen = torch.Generator().manual_seed(21)
    rnd = lambda *s: torch.randn(*s, generator=gen).to(cuda)
    x, res, target = rnd(300, 64), rnd(300, 64), rnd(300, 64)
    ids = torch.stack([torch.randperm(6, generator=gen)[:2] for _ in range(300)]).to(cuda)
    probs = torch.full((300, 2), 0.5, device=cuda)
    start = [torch.ones(64, device=cuda), rnd(96, 64) / 8, torch.zeros(96, device=cuda), rnd(64, 96) / 10]

    def build():
        params = [p.clone().requires_grad_(True) for p in start]
        opt = torch.optim.SGD(params, lr=0.05)

        def step():
            opt.zero_grad(set_to_none=True)
            y, h = add_rms_norm(x, params[0], res)
            order = expert_sort(ids, 6)
            f = linear_act(linear_act(expert_dispatch(y, order), params[1], params[2], "gelu"), params[3])
            loss = (expert_combine(f, probs, order) + h - target).square().mean()
            loss.backward()
            opt.step()
            return loss.detach()

        return params, step

    dense._status_word(cuda)
    eager, step = build()
    losses = [float(step()) for _ in range(7)]
    captured, step = build()
    graphed = GraphedStep(step, warmup=3)  # capturing runs nothing: three steps so far
    for k in range(4):
        graphed.replay()
    torch.cuda.synchronize()
    dense.check_status()
    for a, b in zip(captured, eager):
        assert torch.equal(a, b)
    assert float(graphed.result) == losses[-1]


def test_refusals(cuda):
    from ae_mlsys_gnn_b200.operators.linear_act import linear_act, linear_act_fp8

    x, w, b, r, _ = make(cuda, 8, 16, 24, torch.bfloat16)
    for bad in ((x.double(), w), (x, w.float())):
        with pytest.raises(TypeError):
            linear_act(*bad)
    for bad in ((x, w[:, :8]), (x[:, :0], w[:, :0]), (x, w.view(-1))):
        with pytest.raises(ValueError):
            linear_act(*bad)
    with pytest.raises(ValueError):
        linear_act(x, w, b[:5])
    with pytest.raises(TypeError):
        linear_act(x, w, b.float())
    with pytest.raises(ValueError):
        linear_act(x, w, b, None, r[:4])
    with pytest.raises(ValueError):
        linear_act(x, w, b, None, r[0])
    with pytest.raises(ValueError, match="activation"):
        linear_act(x, w, b, "tanh")
    x8, xs = to_8_bits(x.float())
    w8, ws = to_8_bits(w.float())
    with pytest.raises(TypeError):
        linear_act_fp8(x, xs, w8, ws)
    with pytest.raises(ValueError):
        linear_act_fp8(x8, xs[:3], w8, ws)
    with pytest.raises(TypeError):
        linear_act_fp8(x8, xs.double(), w8, ws)
    with pytest.raises(TypeError):
        linear_act_fp8(x8, xs, w8, ws, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="gradient"):
        linear_act_fp8(x8, xs, w8, ws, b.clone().requires_grad_(True))
