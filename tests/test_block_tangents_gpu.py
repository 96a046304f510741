"""GPU tests that the block's operators, which are differentiable backward and
once, refuse an input that carries a forward-mode tangent instead of returning
an output without one; and that a second backward raises."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from tests.test_block_gpu import ops, read_inputs, write_inputs
from tests.test_ffn_gpu import inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


def calls():
    """(operator on a dict of tensors, the tensors)"""
    R, x, w, b, _ = read_inputs(5, 4, 2, 64, "fp32", "wb")
    yield lambda t: ops().hc_read_norm(**t, norm="layer"), dict(R=R, x=x, weight=w, bias=b)
    t, _ = write_inputs(5, 4, 2, 64, "fp32", "wbs", "sigmoid", True)
    yield lambda t: ops().hc_mix_write_norm(**t, norm="rms", gate_activation="sigmoid", dropout_p=0.2, seed=1), t
    yield lambda t: ops().hc_dropout(t["x"], 0.3, 5), dict(x=x)
    f, _ = inputs(5, 64, 72, 32, "fp32")
    yield lambda t: ops().gated_ffn(**t), dict(zip(("x", "w_gate", "w_up", "w_down"), f))


@pytest.mark.parametrize("grads", [True, False])
def test_tangents_are_refused(grads):
    for call, t in calls():
        for name in t:
            with torch.set_grad_enabled(grads), fwd.dual_level():
                dual = {**t, name: fwd.make_dual(t[name], torch.ones_like(t[name]))}
                with pytest.raises((RuntimeError, NotImplementedError)):
                    call(dual)
        call(t)  # outside the level


def test_a_tangent_that_a_cast_carries_on_is_refused():
    f, _ = inputs(5, 64, 72, 32, "bf16")
    with fwd.dual_level():
        w = f[1].float()
        with pytest.raises((RuntimeError, NotImplementedError)):
            ops().gated_ffn(f[0], fwd.make_dual(w, torch.ones_like(w)), *f[2:])


def test_a_second_derivative_raises():
    for call, t in calls():
        leaves = {k: a.clone().requires_grad_(True) for k, a in t.items()}
        out = call(leaves)
        for g in torch.autograd.grad(out, list(leaves.values()), torch.ones_like(out), create_graph=True):
            with pytest.raises(RuntimeError, match="once differentiable"):
                g.sum().backward(retain_graph=True)
