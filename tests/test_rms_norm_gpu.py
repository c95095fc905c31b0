"""Root-mean-square norm with the residual's addition against the formula in 64 bits.

Tolerances.  u = 2^-24 is half a step of fp32, e half a step of the rows' type (2^-8 of bf16's
finfo.eps / 2 and so on).  A sum of squares is formed by at most 32 adds in a thread and 10 in the tree,
so rstd is off by at most 21 u from the sum, 4 u from rsqrtf (2 ulp) and 1 u from the division;
h, h * rstd and the weight's product add one u each: 32 u bounds y, 40 u is used.  Then one rounding, e."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = [(1, 1), (5, 2), (3, 7), (70, 47), (33, 64), (200, 100), (9, 128), (129, 256), (31, 602), (17, 1433),
         (40, 2048), (6, 2050), (5, 4096), (3, 5120), (4, 8192), (3, 8200), (2, 16384), (3, 20001), (2, 32768)]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    """Half a step among the type's subnormal numbers."""
    return torch.finfo(dt).smallest_normal * half_step(dt)


def within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.3g} x tolerance"


def make(cuda, n, d, dt, residual, wdt=None, seed=0):
    gen = torch.Generator().manual_seed(1000 * n + d + seed)
    x = torch.randn(n, d, generator=gen).to(dt).to(cuda)
    w = (1 + 0.2 * torch.randn(d, generator=gen)).to(wdt or dt).to(cuda)
    r = (2 * torch.randn(n, d, generator=gen)).to(dt).to(cuda) if residual else None
    gy = torch.randn(n, d, generator=gen).to(dt).to(cuda)
    gh = torch.randn(n, d, generator=gen).to(dt).to(cuda)
    return x, w, r, gy, gh


def formula(x, w, r, eps):
    h = x.double() + (0 if r is None else r.double())
    rstd = (h.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h, rstd, h * rstd * w.double()


def check_backward(x, w, r, gy, gh, eps, gx, gw):
    dt = x.dtype
    h, rstd, _ = formula(x, w, r, eps)
    u, xhat = gy.double() * w.double(), h * rstd
    want = rstd * (u - xhat * (u * xhat).mean(-1, keepdim=True)) + (0 if gh is None else gh.double())
    # the backward reads h as it was stored: one rounding more with a residual
    rel = (half_step(dt) if r is not None else 0) + 40 * U
    tol = (half_step(dt) * want.abs() + rel * rstd * (u.abs() + 3 * xhat.abs() * (u * xhat).abs().mean(-1, keepdim=True))
           + 4 * U * (0 if gh is None else gh.double().abs()) + tiny(dt))
    within(gx, want, tol * (1 + half_step(dt)), "grad_x")
    want = (gy.double() * xhat).sum(0)
    # a column's sum: n / 592 rows in a thread, at most 64 groups, 19 + 5 parts
    tol = half_step(gw.dtype) * want.abs() + (rel + (x.shape[0] / 592 + 100) * U) * (gy.double() * xhat).abs().sum(0)
    within(gw, want, tol * (1 + half_step(gw.dtype)) + tiny(gw.dtype), "grad_w")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("residual", [True, False])
@pytest.mark.parametrize("n,d", SIZES)
def test_forward_and_backward(cuda, n, d, dtype, residual):
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm

    dt, eps = DT[dtype], 1e-5
    x, w, r, gy, gh = make(cuda, n, d, dt, residual)
    h64, _, y64 = formula(x, w, r, eps)
    with torch.no_grad():
        y0, h0 = add_rms_norm(x, w, r, eps)
    leaves = [t.clone().requires_grad_(True) for t in ([x, w] if r is None else [x, w, r])]
    y, h = add_rms_norm(leaves[0], leaves[1], None if r is None else leaves[2], eps)
    assert torch.equal(y, y0) and torch.equal(h, h0) and y.dtype == h.dtype == dt
    within(y, y64, (half_step(dt) + 40 * U) * (1 + half_step(dt)) * y64.abs() + tiny(dt), "y")
    within(h, h64, half_step(dt) * (1 + U) * h64.abs() + tiny(dt), "h")
    if residual:
        gx, gw, gr = torch.autograd.grad((y, h), leaves, (gy, gh))
        assert torch.equal(gx, gr)
    else:
        gx, gw = torch.autograd.grad(y, leaves, gy)
    check_backward(x, w, r, gy, gh if residual else None, eps, gx, gw)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_weight_in_32_bits(cuda, dtype):
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm, add_rms_norm_fp8

    for n, d in ((37, 1024), (5, 47), (9, 130)):
        x, w, r, gy, gh = make(cuda, n, d, DT[dtype], True, torch.float32)
        lx, lw, lr = (t.clone().requires_grad_(True) for t in (x, w, r))
        y, h = add_rms_norm(lx, lw, lr)
        y64 = formula(x, w, r, 1e-6)[2]
        within(y, y64, (half_step(x.dtype) + 40 * U) * 1.01 * y64.abs() + tiny(x.dtype), "y")
        gx, gw = torch.autograd.grad((y, h), (lx, lw), (gy, gh))
        assert gw.dtype == torch.float32
        check_backward(x, w, r, gy, gh, 1e-6, gx, gw)
        q, s, _ = add_rms_norm_fp8(x, w, r)
        check_8_bits(q, s, y64, 0)


def check_8_bits(q, scale, y64, block):
    d = y64.shape[-1]
    b = block or d
    parts = -(-d // b)
    amax = torch.stack([c.abs().amax(-1) for c in y64.split(b, -1)], -1)
    want = (amax / 448).clamp_min(2.0 ** -126)
    assert scale.shape == (*y64.shape[:-1], parts)
    # amax is a y (40 u), the division adds one u
    within(scale, want, 41 * U * want, "scale")
    s = want.repeat_interleave(b, -1)[..., :d]
    # e4m3: half a step is 2^-4 of the value, 2^-10 among its subnormals; y / scale is off by 82 u
    v = (y64 / s).abs()
    tol = (v * (2.0 ** -4 + 82 * U)).clamp_min(2.0 ** -10) + v * 82 * U
    within(q.float(), y64 / s, tol, "q")


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("block", [0, 128])
@pytest.mark.parametrize("n,d", SIZES)
def test_8_bit_output(cuda, n, d, dtype, block):
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm, add_rms_norm_fp8

    x, w, r, _, _ = make(cuda, n, d, DT[dtype], n % 2 == 0)
    q, scale, h = add_rms_norm_fp8(x, w, r, 1e-5, block)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape
    assert torch.equal(h, add_rms_norm(x, w, r, 1e-5)[1])
    check_8_bits(q, scale, formula(x, w, r, 1e-5)[2], block)


def test_leading_dimensions_and_strides(cuda):
    """Any leading dimensions; rows that are not laid out one after the other, or that start off a
    16-byte boundary, give what their copies give."""
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm, add_rms_norm_fp8

    x, w, r, _, _ = make(cuda, 60, 96, torch.bfloat16, True)
    y, h = add_rms_norm(x, w, r)
    y3, h3 = add_rms_norm(x.view(5, 12, 96), w, r.view(5, 12, 96))
    assert y3.shape == (5, 12, 96) and torch.equal(y3.view(60, 96), y) and torch.equal(h3.view(60, 96), h)
    wide = torch.zeros(60, 200, dtype=x.dtype, device=cuda)
    wide[:, 3:99] = x
    assert torch.equal(add_rms_norm(wide[:, 3:99], w, r)[0], y)
    shifted = torch.zeros(60 * 96 + 1, dtype=x.dtype, device=cuda)[1:].view(60, 96).copy_(x)
    assert shifted.data_ptr() % 16 and shifted.is_contiguous()
    within(add_rms_norm(shifted, w, r)[0], y.double(), 2 * half_step(x.dtype) * y.double().abs(), "y")
    assert torch.equal(add_rms_norm(x[:0], w, r[:0])[0], y[:0])
    q, s, _ = add_rms_norm_fp8(x.view(5, 12, 96), w, r.view(5, 12, 96), 1e-6, 128)
    assert q.shape == (5, 12, 96) and s.shape == (5, 12, 1)
    lw = w.clone().requires_grad_(True)
    y0, _ = add_rms_norm(x[:0], lw, None)
    assert torch.equal(torch.autograd.grad(y0.sum(), lw)[0], torch.zeros_like(w))


def test_special_rows(cuda):
    """A row of zeros, a NaN, an infinity: each stays in its own row (or block of columns)."""
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm, add_rms_norm_fp8

    for d in (96, 512, 4096):
        x, w, _, _, _ = make(cuda, 8, d, torch.float32, False)
        clean = add_rms_norm(x, w)[0]
        x[1] = 0
        x[3, 5] = float("nan")
        x[6, 7] = float("inf")
        y, _ = add_rms_norm(x, w)
        keep = [0, 2, 4, 5, 7]
        assert torch.equal(y[keep], clean[keep]) and bool((y[1] == 0).all())
        assert bool(y[3].isnan().all()) and bool(y[6, 7].isnan())
        q, s, _ = add_rms_norm_fp8(x, w)
        assert bool((q[1].float() == 0).all()) and float(s[1]) == 2.0 ** -126
        assert bool(s[3].isnan()) and bool(q[3].float().isnan().all()) and not bool(q[keep].float().isnan().any())


def test_gradient_against_differences(cuda):
    """<grad, v> against a central difference of the kernel's own forward (fp32, the loss summed in 64
    bits).  With step t the quotient is off by t^2 / 6 times the third derivative along v, and by the
    forward's rounding, at most 40 u * sum |g y| / t at each point; entries and v are of order one in d = 24."""
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm

    x, w, r, gy, gh = make(cuda, 6, 24, torch.float32, True)
    lx, lw, lr = (t.clone().requires_grad_(True) for t in (x, w, r))
    y, h = add_rms_norm(lx, lw, lr)
    grads = torch.autograd.grad((y, h), (lx, lw, lr), (gy, gh))
    gen = torch.Generator().manual_seed(3)
    t = 2.0 ** -6

    def loss(a):
        y, h = add_rms_norm(*a)
        return (y.double() * gy.double()).sum() + (h.double() * gh.double()).sum()

    y, h = y.detach(), h.detach()
    size = float((y.double() * gy.double()).abs().sum() + (h.double() * gh.double()).abs().sum())
    for i, base in enumerate((x, w, r)):
        v = torch.randn(base.shape, generator=gen).to(cuda)
        up, down = [x, w, r], [x, w, r]
        up[i], down[i] = base + t * v, base - t * v
        quotient = (loss(up) - loss(down)) / (2 * t)
        want = (grads[i].double() * v.double()).sum()
        tol = t * t * size + 2 * 40 * U * size / t
        assert abs(float(quotient - want)) <= tol


def test_only_h_or_only_y_used(cuda):
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm

    x, w, r, gy, gh = make(cuda, 12, 64, torch.float32, True)
    lx, lw, lr = (t.clone().requires_grad_(True) for t in (x, w, r))
    _, h = add_rms_norm(lx, lw, lr)
    h.backward(gh)
    assert torch.equal(lx.grad, gh) and torch.equal(lr.grad, gh) and lw.grad is None
    y, _ = add_rms_norm(lx, w, lr)
    gx, = torch.autograd.grad(y, lx, gy)
    check_backward(x, w, r, gy, None, 1e-6, gx, torch.autograd.grad(add_rms_norm(x, lw, r)[0], lw, gy)[0])
    lx.grad = lr.grad = None
    y, h = add_rms_norm(lx, lw, lr)
    torch.autograd.backward((y, h), (gy, gh))
    lx.grad.zero_()  # the two gradients are equal but not one buffer
    assert float(lr.grad.abs().sum()) > 0


def test_many_rows_and_repeatability(cuda):
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm

    x, w, r, gy, gh = make(cuda, 30011, 72, torch.bfloat16, True)
    got = []
    for _ in range(2):
        lx, lw, lr = (t.clone().requires_grad_(True) for t in (x, w, r))
        y, h = add_rms_norm(lx, lw, lr)
        got.append(torch.autograd.grad((y, h), (lx, lw), (gy, gh)))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    check_backward(x, w, r, gy, gh, 1e-6, *got[0])


def test_streams_and_graph(cuda):
    """The current stream is used, and a captured call replays on new inputs."""
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm, add_rms_norm_fp8

    x, w, r, _, _ = make(cuda, 50, 256, torch.bfloat16, True)
    y, h = add_rms_norm(x, w, r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys, _ = add_rms_norm(x, w, r)
    side.synchronize()
    assert torch.equal(ys, y)
    sx = torch.zeros_like(x)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        gy, gh = add_rms_norm(sx, w, r)
        q, s, _ = add_rms_norm_fp8(sx, w, r)
    sx.copy_(x)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(gy, y) and torch.equal(gh, h)
    q0, s0, _ = add_rms_norm_fp8(x, w, r)
    assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s, s0)


def test_beyond_32_bit_offsets(cuda):
    """More than 2^31 elements: the last rows are those of a small call."""
    from ae_mlsys_gnn_b200.operators.rms_norm import add_rms_norm, add_rms_norm_fp8

    n, d = 530000, 4096
    gen = torch.Generator(device=cuda).manual_seed(2)
    x = torch.zeros(n, d, dtype=torch.bfloat16, device=cuda)
    x[-9:] = torch.randn(9, d, generator=gen, device=cuda).to(torch.bfloat16)
    w = torch.randn(d, generator=gen, device=cuda).to(torch.bfloat16)
    lx, lw = x.requires_grad_(True), w.requires_grad_(True)
    y, _ = add_rms_norm(lx, lw)
    sx = x[-9:].detach().clone().requires_grad_(True)
    ys, _ = add_rms_norm(sx, lw)
    assert torch.equal(y[-9:], ys)
    gy = torch.zeros_like(y)
    gy[-9:] = torch.randn(9, d, generator=gen, device=cuda).to(torch.bfloat16)
    gx, gw = torch.autograd.grad(y, (lx, lw), gy)
    gxs, gws = torch.autograd.grad(ys, (sx, lw), gy[-9:].contiguous())
    assert torch.equal(gx[-9:], gxs)
    assert float((gw.double() - gws.double()).norm() / gws.double().norm()) < 2 * half_step(torch.bfloat16)
    with torch.no_grad():
        q, s, _ = add_rms_norm_fp8(x, w)
        qs, ss, _ = add_rms_norm_fp8(sx, w)
    assert torch.equal(q[-9:].view(torch.uint8), qs.view(torch.uint8)) and torch.equal(s[-9:], ss)
