"""models.GAT with a normed residual stream against the same layers composed with the formula."""
import pytest
import torch

from tests.util import power_law_graph

pytestmark = pytest.mark.gpu


def test_gat_with_rms_norm(cuda):
    from ae_mlsys_gnn_b200.models import GAT
    from ae_mlsys_gnn_b200.operators.csr2csc import csr2csc

    g = power_law_graph(1500, 20, seed=3)
    rp, ci = g.row_ptr.to(cuda), g.col_ind.to(cuda)
    cp, ri, _ = csr2csc(rp, ci)
    torch.manual_seed(0)
    model = GAT(30, 16, [4, 4, 2], 7, norm="rms").to(cuda)
    with torch.no_grad():
        for w in model.norm_weights:
            w.copy_(1 + 0.2 * torch.randn_like(w))
    x = torch.randn(g.n, 30, device=cuda)
    go = torch.randn(g.n, 7, device=cuda)

    def composed():
        h, stream = x, None
        for layer, w in zip(model.gat_layers[:-1], model.norm_weights):
            h = layer(rp, ci, cp, ri, h).flatten(1)
            stream = h + stream if stream is not None and stream.shape == h.shape else h
            h = stream * (stream.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        return model.gat_layers[-1](rp, ci, cp, ri, h).squeeze(1)

    params = list(model.parameters())
    out = model(rp, ci, cp, ri, x)
    want = composed()
    got, exp = torch.autograd.grad(out, params, go), torch.autograd.grad(want, params, go)
    # the same kernels on both sides but for the norm, whose fp32 forms differ by about 2e-6 of a value
    for a, b in zip((out, *got), (want, *exp)):
        assert a.shape == b.shape and float((a - b).detach().norm() / b.detach().norm()) < 1e-4
    with pytest.raises(ValueError, match="norm"):
        GAT(30, 16, [4], 7, norm="layer")


def test_gat_without_norm_is_unchanged(cuda):
    from ae_mlsys_gnn_b200.models import GAT

    assert set(GAT(30, 16, [4], 7).state_dict()) == {
        f"gat_layers.{i}.{n}" for i in range(2) for n in ("W", "attn_l", "attn_r")}
