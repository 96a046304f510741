"""GPU tests of hc_dropout: the mask bit for bit against the oracle's Philox,
the values, the backward, seeds on the device and in graphs."""

import numpy as np
import pytest
import torch

from oracle import block as ob
from tests.bounds import half_step, np64, tiny

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


def drop(*a, **k):
    from hyperconnections_b200.ops import hc_dropout

    return hc_dropout(*a, **k)


def check(got, x, p, seed, offset):
    ref = ob.dropout(np64(x), p, seed, offset)
    err = np.abs(np64(got) - ref)
    # 1 / (1 - p) in float32, one product in float32, one rounding to the type
    assert (err <= (half_step(got.dtype) + 2 ** -23) * np.abs(ref) + tiny(got.dtype)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 7, 8, 9, 31, 1000, 4097, 300001])
def test_values_and_backward(dtype, N):
    for p, seed, offset in ((0.1, 0, 0), (0.5, (1 << 63) + 12345, (1 << 33) + 1), (0.875, -1, -2)):
        x = torch.randn(N, generator=torch.Generator().manual_seed(N)).to(dtype).cuda().requires_grad_(True)
        y = drop(x, p, seed, offset)
        assert y.dtype == dtype
        check(y, x, p, seed % (1 << 64), offset % (1 << 64))
        g = torch.ones_like(x)
        y.backward(g)
        check(x.grad, g, p, seed % (1 << 64), offset % (1 << 64))


@pytest.mark.parametrize("p", [0.0, 1.0])
def test_keep_all_and_none(p):
    x = torch.randn(1000, device="cuda", dtype=torch.bfloat16)
    y = drop(x, p, 7)
    assert torch.equal(y, x if p == 0 else torch.zeros_like(x))


def test_dropped_places_hold_zero_whatever_they_held():
    x = torch.full((4096,), float("nan"), device="cuda")
    x[::2] = float("inf")
    keep = torch.from_numpy(ob.keep_mask(4096, 0.5, 3, 1)).cuda()
    y = drop(x, 0.5, 3, 1)
    assert (y[~keep] == 0).all() and torch.equal(y[keep].isnan(), x[keep].isnan()) and (~y[keep].isfinite()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unaligned_and_strided(dtype):
    base = torch.randn(3001, device="cuda").to(dtype)
    for x in (base[1:], base[3:2050], base.view(1, -1)[:, 1:], base[:3000].view(50, 60).t(), base[::3]):
        assert torch.equal(drop(x, 0.3, 5), drop(x.contiguous().clone(), 0.3, 5))


def test_empty():
    assert drop(torch.empty(0, 5, device="cuda"), 0.5, 1).shape == (0, 5)


def test_seed_tensor_and_graph_replays():
    """A seed held on the device is read when the kernel runs: each replay of a graph that moves it on drops other
    places, the backward the same as its forward, and the gradient of an earlier forward keeps its own mask."""
    x = torch.randn(5000, device="cuda")
    state = torch.tensor([42, 7], device="cuda")
    assert torch.equal(drop(x, 0.5, state), drop(x, 0.5, 42, 7))
    xg = x.clone().requires_grad_(True)
    y = drop(xg, 0.5, state)
    state[1] += 1  # before the backward
    (gx,) = torch.autograd.grad(y, xg, torch.ones_like(x))
    assert torch.equal(gx != 0, y.detach() != 0)
    del y

    def step():
        leaf = x.detach().requires_grad_(True)
        out = drop(leaf, 0.5, state)
        state[1].add_(1)
        (grad,) = torch.autograd.grad(out, leaf, torch.ones_like(x))
        return out.detach(), grad

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = step()
    state.copy_(torch.tensor([42, 100]))
    seen = []
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        check(out, x, 0.5, 42, 100 + k)
        assert torch.equal(grad != 0, out != 0)
        seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1])


def test_share_of_kept_places():
    """Over 2^20 places the kept share is within five standard deviations of 1 - p."""
    n = 1 << 20
    for p in (0.1, 0.5):
        kept = (drop(torch.ones(n, device="cuda"), p, 2024, 11) != 0).sum().item()
        assert abs(kept - n * (1 - p)) <= 5 * (n * p * (1 - p)) ** 0.5
