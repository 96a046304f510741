"""GPU tests of the norm kernels where a group of warps walks many tokens: what
one token gives does not depend on the tokens before and behind it in its
group's walk. A call over many tokens is compared bit for bit with calls over
so few that every group has one (148 tokens: the grid has at least one group an
SM), which nothing can overtake. The kernels' arithmetic for a token is the
same in both, so any difference is a sum or a matrix of another token."""

import pytest
import torch

from tests.test_block_gpu import leaf, ops, write_inputs

pytestmark = pytest.mark.gpu

FEW = 148  # tokens of a call in which no group walks on to another


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


def write_step(t, g, **kw):
    """The output and the per-token gradients of hc_mix_write_norm."""
    leaves = {k: leaf(a) for k, a in t.items()}
    out = ops().hc_mix_write_norm(**leaves, **kw)
    names = [k for k in ("H", "x", "W", "f", "v", "gate") if leaves[k] is not None]
    return [out.detach(), *torch.autograd.grad(out, [leaves[k] for k in names], g)]


def part(t, i):
    return {k: a if a is None or k in ("weight", "bias", "scale") else a[i:i + FEW] for k, a in t.items()}


@pytest.mark.parametrize("T,n,m,D,dt,norm,proj", [
    (FEW * 60, 4, 1, 768, "bf16", "rms", False),   # groups of three warps, the usual training case
    (FEW * 60, 4, 1, 512, "bf16", "rms", False),
    (FEW * 60, 2, 1, 272, "fp16", "none", False),
    (FEW * 40, 4, 2, 768, "fp16", "layer", False),
    (FEW * 40, 4, 1, 769, "bf16", "rms", False),   # ragged rows
    (FEW * 40, 4, 1, 768, "fp32", "layer", False),
    (FEW * 30, 8, 2, 1024, "fp16", "layer", False),
    (FEW * 30, 8, 2, 1024, "fp16", "layer", True),
    (FEW * 12, 4, 1, 4096, "bf16", "rms", False),  # sixteen warps
    (FEW * 120, 4, 1, 96, "bf16", "rms", True),    # one warp a token
])
def test_mix_write_gradients_of_a_token(T, n, m, D, dt, norm, proj):
    t, g = write_inputs(T, n, m, D, dt, "wbs", "sigmoid", proj)
    kw = dict(norm=norm, gate_activation="sigmoid")
    alone = [write_step(part(t, i), g[i:i + FEW], **kw) for i in range(0, T, FEW)]
    alone = [torch.cat(a) for a in zip(*alone)]
    for _ in range(3):
        for a, b in zip(write_step(t, g, **kw), alone):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T,n,m,D,dt,norm", [
    (FEW * 120, 4, 1, 256, "bf16", "rms"),
    (FEW * 120, 4, 1, 768, "bf16", "layer"),  # one warp, three chunks a thread
    (FEW * 60, 8, 2, 200, "fp16", "layer"),
    (FEW * 60, 3, 1, 77, "fp32", "rms"),
])
def test_projected_mix_of_one_warp(T, n, m, D, dt, norm):
    """The projected mix of a token is made by its warp's lanes for one another."""
    t, _ = write_inputs(T, n, m, D, dt, "wbs", "sigmoid", True)
    kw = dict(norm=norm, gate_activation="sigmoid")
    alone = torch.cat([ops().hc_mix_write_norm(**part(t, i), **kw) for i in range(0, T, FEW)])
    for _ in range(3):
        assert torch.equal(ops().hc_mix_write_norm(**t, **kw), alone)
