"""Rows between token order and expert order against plain indexing in 64 bits.

Tolerances: u = 2^-24, e half a step of the rows' type.  A sum over k choices takes at most k fused
multiply-adds, (k + 1) u of the sum of magnitudes, then one rounding e.  A weight's gradient is a dot
product of D terms: a lane adds at most D / 32 + 8 of them in a row (8 per access), then 5 + 8 adds."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# tokens, k, experts, width
SIZES = [(1, 1, 1, 1), (1, 4, 8, 64), (3, 2, 5, 7), (16, 4, 64, 128), (100, 8, 16, 130), (257, 3, 7, 602),
         (33, 9, 40, 96), (700, 8, 256, 264), (5, 32, 1024, 40), (9, 2, 4, 8192), (5000, 6, 100, 48)]


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return torch.finfo(dt).smallest_normal * half_step(dt)


def within(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off"


def make_ids(t, k, e, dropped, seed=0):
    gen = torch.Generator().manual_seed(t * 31 + k + e + seed)
    ids = torch.multinomial(torch.rand(t, e, generator=gen) + 1e-3, min(k, e), generator=gen) if e >= k else \
        torch.randint(e, (t, k), generator=gen)
    if dropped:
        ids[torch.rand(t, k, generator=gen) < 0.3] = -1
    return ids


def places(ids, e):
    """(offsets, slots) by a stable sort on the host."""
    flat = ids.reshape(-1)
    ok = (flat >= 0) & (flat < e)
    key = torch.where(ok, flat, torch.full_like(flat, e))
    order = torch.argsort(key, stable=True)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(flat.numel())
    counts = torch.bincount(key, minlength=e + 1)[:e]
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])
    return offsets.int(), torch.where(ok, slots, -1).int().view(ids.shape)


@pytest.mark.parametrize("dropped", [False, True])
@pytest.mark.parametrize("t,k,e,d", SIZES)
def test_sort_is_exact(cuda, t, k, e, d, dropped):
    from ae_mlsys_gnn_b200.operators.experts import expert_sort

    ids = make_ids(t, k, e, dropped)
    for kind in (torch.int32, torch.int64):
        order = expert_sort(ids.to(kind).to(cuda), e)
        offsets, slots = places(ids, e)
        assert torch.equal(order.offsets.cpu(), offsets) and torch.equal(order.slots.cpu(), slots)


@pytest.mark.parametrize("pairs,e", [(1024, 3), (1025, 2), (2048, 3), (2049, 1), (4096, 1024), (65536, 8), (303105, 128), (1000003, 1000),
                                     (2600000, 64)])
def test_sort_of_many_pairs(cuda, pairs, e):
    """Several chunks, ids out of range on both sides, one expert far ahead of the others."""
    from ae_mlsys_gnn_b200.operators.experts import expert_sort

    gen = torch.Generator().manual_seed(pairs)
    ids = torch.randint(-2, e + 2, (pairs, 1), generator=gen)
    ids[torch.rand(pairs, 1, generator=gen) < 0.4] = e // 2
    ids[pairs // 3] = 2 ** 40
    order = expert_sort(ids.to(cuda), e)
    offsets, slots = places(ids, e)
    assert torch.equal(order.offsets.cpu(), offsets) and torch.equal(order.slots.cpu(), slots)


def test_sort_of_nothing(cuda):
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort

    order = expert_sort(torch.empty(0, 4, dtype=torch.int64, device=cuda), 5)
    assert torch.equal(order.offsets.cpu(), torch.zeros(6, dtype=torch.int32))
    x = torch.empty(0, 16, device=cuda)
    xs = expert_dispatch(x, order)
    assert xs.shape == (0, 16)
    assert expert_combine(xs, torch.empty(0, 4, device=cuda), order).shape == (0, 16)
    none = expert_sort(torch.full((6, 3), -1, device=cuda), 5)  # nobody chose anything
    assert int(none.offsets[-1]) == 0 and bool((none.slots == -1).all())
    assert not bool(expert_dispatch(torch.ones(6, 16, device=cuda), none).any())
    out = expert_combine(torch.full((18, 16), float("nan"), device=cuda), torch.ones(6, 3, device=cuda), none)
    assert torch.equal(out, torch.zeros(6, 16, device=cuda))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("dropped", [False, True])
@pytest.mark.parametrize("t,k,e,d", SIZES)
def test_rows_there_and_back(cuda, t, k, e, d, dropped, dtype):
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort

    dt = DT[dtype]
    ids = make_ids(t, k, e, dropped)
    gen = torch.Generator().manual_seed(t + k + e + d)
    rnd = lambda *s: torch.randn(*s, generator=gen)
    order = expert_sort(ids.to(cuda), e)
    slots = places(ids, e)[1].long()
    ok = slots >= 0
    kept = int(ok.sum())
    x = rnd(t, d).to(dt).to(cuda).requires_grad_(True)
    ye = rnd(t * k, d).to(dt)
    ye[kept:] = float("nan")  # rows that no pair fills are not read
    ye = ye.to(cuda).requires_grad_(True)
    for wdt in {dt, torch.float32}:
        w = torch.rand(t, k, generator=gen).to(wdt).to(cuda).requires_grad_(True)
        xs = expert_dispatch(x, order)
        want = torch.zeros(t * k, d, dtype=dt)
        want[slots[ok]] = x.detach().cpu()[torch.nonzero(ok)[:, 0]]
        assert torch.equal(xs.detach().cpu(), want)
        out = expert_combine(ye, w, order)
        at = slots.clamp_min(0).to(cuda)
        picked = torch.where(ok.to(cuda)[:, :, None], ye.detach().double()[at], 0.0)
        terms = picked * w.detach().double()[:, :, None]
        want = terms.sum(1)
        within(out, want, half_step(dt) * (1 + U) * want.abs() + (k + 1) * U * 1.01 * terms.abs().sum(1) + tiny(dt), "out")
        # gradients
        gxs, go = rnd(t * k, d).to(dt).to(cuda), rnd(t, d).to(dt).to(cuda)
        gx, = torch.autograd.grad(xs, x, gxs)
        terms = torch.where(ok.to(cuda)[:, :, None], gxs.double()[at], 0.0)
        want = terms.sum(1)
        within(gx, want, half_step(dt) * (1 + U) * want.abs() + (k + 1) * U * 1.01 * terms.abs().sum(1) + tiny(dt), "grad_x")
        gye, gw = torch.autograd.grad(out, (ye, w), go)
        want = torch.zeros(t * k, d, dtype=torch.float64, device=cuda)
        want[slots[ok].to(cuda)] = (go.double()[:, None] * w.detach().double()[:, :, None])[ok.to(cuda)]
        within(gye, want, half_step(dt) * (1 + U) * want.abs() + U * want.abs() + tiny(dt), "grad_rows")
        assert not bool(gye[kept:].any())
        terms = picked * go.double()[:, None]
        want = terms.sum(2)
        tol = half_step(wdt) * (1 + U) * want.abs() + (d / 32 + 22) * U * terms.abs().sum(2) * 1.01
        within(gw, want, tol + tiny(wdt), "grad_w")
        assert gw.dtype == wdt and not bool(gw[~ok.to(cuda)].any())


def test_gradient_against_differences(cuda):
    """The whole way, tokens to experts to tokens, is bilinear in rows and weights: a central
    difference along v is exact up to rounding, (k + 2) u of the loss's magnitude at both points."""
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort

    gen = torch.Generator().manual_seed(2)
    t, k, e, d = 40, 4, 6, 32
    order = expert_sort(make_ids(t, k, e, True).to(cuda), e)
    x = torch.randn(t, d, generator=gen).to(cuda)
    w = torch.rand(t, k, generator=gen).to(cuda)
    go = torch.randn(t, d, generator=gen).to(cuda)

    def loss(x, w):
        out = expert_combine(expert_dispatch(x, order), w, order)
        return (out.double() * go.double()).sum(), float((out.double() * go.double()).abs().sum().detach())

    lx, lw = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    grads = torch.autograd.grad(loss(lx, lw)[0], (lx, lw))
    step = 0.25
    for i, base in enumerate((x, w)):
        v = torch.randn(base.shape, generator=gen).to(cuda)
        up, down = [x, w], [x, w]
        up[i], down[i] = base + step * v, base - step * v
        (a, sa), (b, sb) = loss(*up), loss(*down)
        got = float((grads[i].double() * v.double()).sum())
        size = float((grads[i].double() * v.double()).abs().sum())
        # the loss's terms can be k times its magnitude after they cancel within a token
        assert abs(got - float(a - b) / (2 * step)) <= (k + 3) * U * (k * (sa + sb) / (2 * step) + size) * 4


def test_same_results_twice_on_streams_and_in_graphs(cuda):
    """Bit-equal from run to run; two graphs captured one after the other and replayed on two streams
    at once do not share scratch."""
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort

    gen = torch.Generator().manual_seed(8)
    t, k, e, d = 3000, 4, 32, 256
    sets = []
    for s in range(2):
        ids = make_ids(t, k, e, True, seed=s).to(cuda)
        sets.append((ids, torch.randn(t, d, generator=gen).to(cuda), torch.rand(t, k, generator=gen).to(cuda)))

    def step(ids, x, w):
        order = expert_sort(ids, e)
        return order.slots, expert_combine(expert_dispatch(x, order), w, order)

    want = [step(*s) for s in sets]
    graphs, got = [], []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(step(*s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (slots, out), (slots0, out0) in zip(got, want):
        assert torch.equal(slots, slots0) and torch.equal(out, out0)


def test_strided_and_shifted_inputs(cuda):
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort

    gen = torch.Generator().manual_seed(4)
    ids = make_ids(50, 3, 9, False).to(cuda)
    order = expert_sort(ids, 9)
    wide = torch.zeros(50, 6, dtype=torch.int64, device=cuda)
    wide[:, ::2] = ids
    assert torch.equal(expert_sort(wide[:, ::2], 9).slots, order.slots)
    x = torch.randn(50, 64, generator=gen).to(torch.bfloat16).to(cuda)
    xs = expert_dispatch(x, order)
    shifted = torch.zeros(50 * 64 + 1, dtype=x.dtype, device=cuda)[1:].view(50, 64).copy_(x)
    assert torch.equal(expert_dispatch(shifted, order), xs)
    assert torch.equal(expert_dispatch(x.t().contiguous().t(), order), xs)
    w = torch.rand(3, 50, generator=gen).to(cuda).t()
    assert torch.equal(expert_combine(xs, w, order), expert_combine(xs, w.contiguous(), order))


def test_refusals(cuda):
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort

    ids = torch.zeros(4, 2, dtype=torch.int32, device=cuda)
    order = expert_sort(ids, 3)
    x, rows, w = torch.zeros(4, 8, device=cuda), torch.zeros(8, 8, device=cuda), torch.zeros(4, 2, device=cuda)
    with pytest.raises(TypeError):
        expert_sort(ids.float(), 3)
    with pytest.raises(ValueError):
        expert_sort(ids.view(-1), 3)
    for e in (0, 1025):
        with pytest.raises(ValueError):
            expert_sort(ids, e)
    with pytest.raises(ValueError):
        expert_sort(torch.zeros(4, 33, dtype=torch.int32, device=cuda), 3)
    with pytest.raises(ValueError):
        expert_dispatch(x[:3], order)
    with pytest.raises(TypeError):
        expert_dispatch(x.double(), order)
    with pytest.raises(TypeError):
        expert_dispatch(x, ids)
    with pytest.raises(ValueError):
        expert_combine(rows[:7], w, order)
    with pytest.raises(ValueError):
        expert_combine(rows, w[:, :1], order)
    with pytest.raises(TypeError):
        expert_combine(rows, w.half(), order)


def test_beyond_32_bit_offsets(cuda):
    """More than 2^31 elements in expert order: rows at the far end go there and back."""
    from ae_mlsys_gnn_b200.operators.experts import expert_combine, expert_dispatch, expert_sort

    t, k, d, e = 66000, 8, 4160, 16
    gen = torch.Generator(device=cuda).manual_seed(3)
    ids = torch.rand(t, e, generator=gen, device=cuda).topk(k, 1).indices
    order = expert_sort(ids, e)
    x = torch.randn(t, d, generator=gen, device=cuda).to(torch.bfloat16).requires_grad_(True)
    xs = expert_dispatch(x, order)
    some = torch.arange(0, t, 997, device=cuda)
    at = order.slots[some].long()
    assert int(at.max()) * d > 2 ** 31
    assert torch.equal(xs[at[:, 5]], x[some]) and torch.equal(xs[at[:, 0]], x[some])
    w = torch.rand(t, k, generator=gen, device=cuda).requires_grad_(True)
    out = expert_combine(xs, w, order)
    want = x[some].double() * w[some].double().sum(1, keepdim=True)
    within(out[some], want, half_step(torch.bfloat16) * 1.01 * want.abs() + 10 * U * x[some].double().abs() * k, "out")
    g = torch.randn(t, d, generator=gen, device=cuda).to(torch.bfloat16)
    gxs, gw = torch.autograd.grad(out, (xs, w), g, retain_graph=True)
    assert torch.equal(gxs[at[:, 3]], (g[some].float() * w[some, 3:4]).to(torch.bfloat16))
    want = (g[some].double() * x[some].double()).sum(1)
    size = (g[some].double() * x[some].double()).abs().sum(1)
    within(gw[some, 2], want, (d / 32 + 22) * U * size * 1.01, "grad_w")
    gx, = torch.autograd.grad(xs, x, gxs)
    want = g[some].double() * 0
    for j in range(k):
        want = want + gxs[at[:, j]].double()
    within(gx[some], want, half_step(torch.bfloat16) * 1.01 * want.abs() + 10 * U * k * gxs[at].double().abs().amax(1), "grad_x")
