"""The layers' block options (hyperconnections_b200.block) and the gated blocks
of e2e_models: what they add to a layer and nothing else, on the CPU; on the
GPU the layer against the same layer with the options' formulas in torch
(float64 for the block, the layer's own mixing weights), with gradients, and a
training step of a small gated model.

The float32 layer sums over a few thousand tokens and through GEMMs of width
n * embed_dim, so outputs are held to 1e-5 of their largest magnitude and
parameter gradients to 5e-5, as the layers' own tests hold them."""

import numpy as np
import pytest
import torch
import torch.nn as nn

import e2e_models as em
from hyperconnections_b200.block import BlockOptions
from hyperconnections_b200.cghc import ContinuousGenHyperConnections as CGHC
from hyperconnections_b200.ghc import GeneralizedHyperConnections as GHC
from hyperconnections_b200.mhc import ManifoldHyperConnections as MHC

FULL = BlockOptions(pre_norm="layer", post_norm="rms", gate=True, residual_scale=0.2, dropout=0.25, eps=1e-5)


def layer(cls, n, m, E, block=None, **kw):
    torch.manual_seed(0)
    return cls(n, m, n * E // m, E, nn.Linear(E, E), block=block, **kw)


@pytest.mark.parametrize("cls", [CGHC, GHC, MHC])
def test_options_add_their_parameters_and_nothing_else(cls):
    plain, full = layer(cls, 4, 2, 16), layer(cls, 4, 2, 16, FULL)
    extra = set(full.state_dict()) - set(plain.state_dict())
    assert set(plain.state_dict()) <= set(full.state_dict())
    assert extra == {"block.pre_norm.weight", "block.pre_norm.bias", "block.post_norm.weight", "block.gate.weight",
                     "block.gate.bias", "block.scale"}
    assert set(layer(cls, 4, 2, 16, BlockOptions()).state_dict()) == set(plain.state_dict())


def test_options_are_checked():
    with pytest.raises(ValueError, match="norm"):
        BlockOptions(pre_norm="batch")
    with pytest.raises(ValueError, match="dropout"):
        BlockOptions(dropout=1.5)


def test_gated_specs():
    spec = em.gated(em.LM)
    assert spec.gated and spec.block is em.GATED and (spec.dim, spec.depth) == (em.LM.dim, em.LM.depth)
    assert em.flops_per_token(spec) > em.flops_per_token(em.LM)
    assert em.describe(spec)["mlp"] == "4x gated" and em.describe(em.LM)["mlp"] == "4x"
    with torch.device("meta"):
        net = em.GatedMLP(8, spec.block)
    assert isinstance(net.norm, nn.Identity) and isinstance(em.own_norm(8, None), nn.LayerNorm)


def reference_forward(lay, x, seed, offset):
    """The layer's forward with the block's part in float64 torch operations; the mixing weights come from a plain
    layer's own forward (its read, write and mix matrices, caught at the operators)."""
    from oracle import block as ob

    caught = {}
    import hyperconnections_b200.block as hb

    saved = hb.hc_read_norm, hb.hc_mix_write_norm
    try:
        hb.hc_read_norm = lambda R, xs, *a, **k: (caught.update(R=R, xs=xs), saved[0](R, xs, *a, **k))[1]
        hb.hc_mix_write_norm = lambda H, xs, W, f, v, **k: (caught.update(H=H, W=W, v=v), saved[1](H, xs, W, f, v, **k))[1]
        lay(x)
    finally:
        hb.hc_read_norm, hb.hc_mix_write_norm = saved
    o, b = lay.block.options, lay.block
    R, H, W, v = (None if caught[k] is None else caught[k].double() for k in ("R", "H", "W", "v"))
    xs = caught["xs"].double()
    T, m, _ = R.shape
    E = lay.embed_dim

    def norm(u, part):
        c = u - u.mean(-1, keepdim=True) if part.kind == "layer" else u
        y = c * (c.square().mean(-1, keepdim=True) + o.eps).rsqrt() * part.weight.double()
        return y if part.bias is None else y + part.bias.double()

    u = norm((R @ xs).reshape(T, E), b.pre_norm)
    f = nn.functional.linear(u, lay.module.weight.double(), lay.module.bias.double())
    gate = torch.sigmoid(nn.functional.linear(u, b.gate.weight.double(), b.gate.bias.double()))
    z = norm(f, b.post_norm) * gate * b.scale.double()
    keep = torch.from_numpy(ob.keep_mask(T * E, o.dropout, seed, offset)).view(T, E).cuda()
    z = torch.where(keep, z / (1 - o.dropout), 0.0).view(T, m, -1)
    if v is not None:
        H = H + (v - (H @ v[..., None])[..., 0])[..., None] * v[..., None, :]
    return (H @ xs + W @ z).reshape(x.shape)


def close(got, want, tol, what):
    got, want = got.detach().double().cpu().numpy(), want.detach().double().cpu().numpy()
    assert np.abs(got - want).max() <= tol * max(1.0, np.abs(want).max()), what


@pytest.mark.gpu
@pytest.mark.parametrize("cls,n,m,kw", [(CGHC, 4, 1, {}), (CGHC, 4, 2, {"projection": "v"}), (GHC, 3, 1, {}), (MHC, 4, 4, {})])
def test_layer_against_its_formulas(cls, n, m, kw):
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    E = 96
    lay = layer(cls, n, m, E, FULL, **kw).cuda()
    with torch.no_grad():
        for p in lay.block.parameters():
            p.add_(0.05 * torch.randn_like(p))
    x = torch.randn(3, 40, n * E // m, device="cuda")
    g = torch.randn_like(x)
    lay.block.drop_state.copy_(torch.tensor([77, 5]))
    xo = x.clone().requires_grad_(True)
    out = lay(xo)
    assert lay.block.drop_state.tolist() == [77, 6]
    out.backward(g)
    grads = {k: p.grad.clone() for k, p in lay.named_parameters() if p.grad is not None}
    lay.zero_grad(set_to_none=True)
    lay.block.drop_state.copy_(torch.tensor([77, 5]))
    xr = x.clone().requires_grad_(True)
    want = reference_forward(lay, xr, 77, 5)
    close(out, want, 1e-5, "out")
    want.backward(g.double())
    close(xo.grad, xr.grad, 5e-5, "grad_x")
    refs = {k: p.grad for k, p in lay.named_parameters() if p.grad is not None}
    assert refs.keys() == grads.keys()
    for k in refs:
        close(grads[k], refs[k], 5e-5, k)
    # evaluation drops nothing and leaves the state alone
    lay.eval()
    state = lay.block.drop_state.clone()
    assert torch.equal(lay(x), lay(x)) and torch.equal(state, lay.block.drop_state)


@pytest.mark.gpu
def test_gated_model_steps():
    """A training step of each gated workload at a small size runs and gives every parameter a finite gradient, and two
    steps from the same state draw different dropout."""
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    from dataclasses import replace

    for spec in (replace(em.gated(em.VIT), dim=96, depth=2, heads=2, global_batch=8, micro_batch=4),
                 replace(em.gated(em.LM), dim=128, depth=2, heads=2, global_batch=4, micro_batch=2, seq=32, vocab=100)):
        tr = em.Trainer(spec, torch.device("cuda:0"))
        before = [p.detach().clone() for p in tr.model.parameters()]
        loss = tr.step()
        assert torch.isfinite(loss)
        for (name, p), b in zip(tr.model.named_parameters(), before):
            if p.requires_grad and p.grad is not None:
                assert p.grad.isfinite().all(), name
        assert any(not torch.equal(p, b) for p, b in zip(tr.model.parameters(), before))
        states = [m.drop_state[1].item() for m in tr.model.modules() if hasattr(m, "drop_state")]
        assert states == [2] * (2 * spec.depth)  # two micro-batches


@pytest.mark.gpu
def test_chain_in_a_graph():
    """read + pre-norm -> gated feed-forward -> post-norm + gate + dropout + mix-write -> dropout, forward and backward,
    captured once and replayed on new inputs: bit for bit the eager call."""
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    from hyperconnections_b200.ops import gated_ffn, hc_dropout, hc_mix_write_norm, hc_read_norm
    from tests.test_cuda_graph_gpu import _graph_vs_eager

    for T, n, D, F, dt in ((640, 4, 256, 512, torch.bfloat16), (16, 3, 128, 264, torch.float16), (70, 2, 33, 50, torch.float32)):
        def make(seed):
            g = torch.Generator().manual_seed(seed)
            r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
            ts = [r(T, n, D).to(dt), torch.sigmoid(r(T, 1, n)), 1 + 0.1 * r(D), torch.eye(n) + 0.2 * r(T, n, n),
                  torch.rand(T, n, 1, generator=g), r(F, D).div(D ** 0.5).to(dt), r(F, D).div(D ** 0.5).to(dt),
                  r(D, F).div(F ** 0.5).to(dt), r(T, 1, D).to(dt), 0.1 * r(D), r(T, n, D).to(dt)]
            return [t.cuda() for t in ts]

        def step(x, R, w, H, W, wg, wu, wd, gate, scale, g):
            leaves = [t.detach().requires_grad_(True) for t in (x, R, w, H, W, wg, wu, wd, gate, scale)]
            x, R, w, H, W, wg, wu, wd, gate, scale = leaves
            y = hc_read_norm(R, x, w)
            f = gated_ffn(y, wg, wu, wd)
            z = hc_mix_write_norm(H, x, W, f, weight=w, gate=gate, gate_activation="sigmoid", scale=scale, dropout_p=0.1,
                                  seed=5, offset=1)
            out = hc_dropout(z, 0.2, 5, 2)
            return [out.detach(), *torch.autograd.grad(out, leaves, g)]

        _graph_vs_eager(make, step)
