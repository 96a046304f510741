"""GPU tests of the block's operators at their edges: offsets past 32 bits,
calls on two streams at once, a replayed training step, the same tensor in two
places, a wait that gives up."""

import ctypes

import numpy as np
import pytest
import torch

from oracle import block as ob
from tests.test_ffn_gpu import DT, check_all, inputs
from tests.test_block_gpu import check_read, leaf, read_inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")
    yield
    torch.cuda.empty_cache()


def ops():
    from hyperconnections_b200 import ops as o

    return o


# ------------------------------------------------------------ a few tokens
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 7, 8, 9, 16, 24, 25, 31, 32, 33, 64, 65])
@pytest.mark.parametrize("dt,act", [("bf16", "silu"), ("fp16", "gelu_tanh"), ("fp32", "silu")])
def test_ffn_around_the_few_token_limit(T, dt, act):
    t, g = inputs(T, 264, 520, 136, dt, seed=T)
    leaves = [k.clone().requires_grad_(True) for k in t]
    y = ops().gated_ffn(*leaves, activation=act)
    y.backward(g)
    check_all(t, g, act, y, [k.grad for k in leaves])
    with torch.no_grad():
        assert torch.equal(ops().gated_ffn(*t, activation=act), y)


# ------------------------------------------------------ offsets past 32 bits
def test_ffn_past_32_bits():
    """h holds more than 2^31 elements; g is 0 but in the last rows, so that the weights' gradients are theirs."""
    T, D, F, O, tail = 270_000, 64, 8192, 72, 500
    t, g = inputs(tail, D, F, O, "bf16")
    x = torch.zeros(T, D, dtype=torch.bfloat16, device="cuda")
    x[-tail:] = t[0]
    gy = torch.zeros(T, O, dtype=torch.bfloat16, device="cuda")
    gy[-tail:] = g
    leaves = [x.requires_grad_(True)] + [k.clone().requires_grad_(True) for k in t[1:]]
    y = ops().gated_ffn(*leaves)
    y.backward(gy)
    assert (y[:-tail] == 0).all() and (leaves[0].grad[:-tail] == 0).all()
    check_all(t, g, "silu", y[-tail:], [leaves[0].grad[-tail:]] + [k.grad for k in leaves[1:]])


def test_norms_past_32_bits():
    """x holds more than 2^31 elements: the last tokens come out as in a call of their own."""
    T, n, D, tail = 530_000, 8, 512, 64
    R, x, w, _, gy = read_inputs(tail, n, 1, D, "bf16", "w")
    big = torch.ones(T, n, D, dtype=torch.bfloat16, device="cuda")
    big[-tail:] = x
    bigR = torch.ones(T, 1, n, device="cuda")
    bigR[-tail:] = R
    gbig = torch.zeros(T, 1, D, dtype=torch.bfloat16, device="cuda")
    gbig[-tail:] = gy
    bigR.requires_grad_(True)
    big.requires_grad_(True)
    w1 = leaf(w)
    y = ops().hc_read_norm(bigR, big, w1)
    y.backward(gbig)
    small = [leaf(R), leaf(x), leaf(w)]
    z = ops().hc_read_norm(*small)
    z.backward(gy)
    assert torch.equal(y[-tail:], z)
    assert torch.equal(big.grad[-tail:], small[1].grad) and torch.equal(bigR.grad[-tail:], small[0].grad)
    assert (big.grad[:-tail] == 0).all()
    check_read(R, x, w, None, gy, "rms", 1e-6, (y[-tail:], None, None, w1.grad, None))
    del y, z, gbig
    big.grad = bigR.grad = None

    # the mix-write of the same streams: its dropout draws by the element's own number, past 2^28 here
    H = torch.eye(n, device="cuda").expand(T, n, n)
    W = torch.ones(T, n, 1, device="cuda")
    f = big.detach()[:, :1]
    out = ops().hc_mix_write_norm(H, big.detach(), W, f, norm="none", dropout_p=0.25, seed=11, offset=5)
    first = (T - tail) * D
    blocks = np.arange(first // 4, (T * D + 3) // 4, dtype=np.uint64)
    keep = torch.from_numpy(keep_from(blocks, 0.25, 11, 5)).cuda().view(tail, 1, D)
    z = torch.where(keep, f[-tail:].float() * (1 / 0.75), torch.zeros((), device="cuda"))
    want = big.detach()[-tail:].float() + z
    # one rounding of the sum, three float32 ones before it
    assert ((out[-tail:].float() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -21 * (want.abs() + z.abs()) + 1e-30).all()


def keep_from(blocks, p, seed, offset):
    """The elements of these generator blocks that dropout keeps."""
    index = (np.uint64(4) * blocks[:, None] + np.arange(4, dtype=np.uint64)).reshape(-1)
    return ob.philox_words(index, seed, offset) >= np.uint64(int(p * 2 ** 32))


def test_dropout_past_32_bits():
    N, p, tail = (1 << 32) + 4099, 0.25, 8195
    x = torch.ones(N, dtype=torch.bfloat16, device="cuda")
    y = ops().hc_dropout(x, p, 3, 9)
    first = (N - tail) // 4 * 4
    keep = keep_from(np.arange(first // 4, (N + 3) // 4, dtype=np.uint64), p, 3, 9)[: N - first]
    assert np.array_equal((y[first:] != 0).cpu().numpy(), keep)


# ------------------------------------------------------------------ sharing
def test_ffn_one_tensor_in_two_places():
    """w_gate and w_up the same tensor: its gradient is the sum of both."""
    t, g = inputs(200, 128, 256, 64, "bf16")
    w = t[1].clone().requires_grad_(True)
    ops().gated_ffn(t[0], w, w, t[3]).backward(g)
    two = [t[1].clone().requires_grad_(True) for _ in range(2)]
    ops().gated_ffn(t[0], *two, t[3]).backward(g)
    assert torch.equal(w.grad, two[0].grad + two[1].grad)


def test_ffn_backward_twice_and_of_an_expanded_gradient():
    t, g = inputs(300, 128, 256, 64, "fp16")
    leaves = [k.clone().requires_grad_(True) for k in t]
    y = ops().gated_ffn(*leaves)
    a = torch.autograd.grad(y, leaves, g, retain_graph=True)
    b = torch.autograd.grad(y, leaves, g, retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    one = torch.ones((), dtype=DT["fp16"], device="cuda")
    c = torch.autograd.grad(y, leaves, one.expand_as(y), retain_graph=True)
    d = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert all(torch.equal(p, q) for p, q in zip(c, d))


@pytest.mark.parametrize("T,dt", [(8, "bf16"), (700, "bf16"), (90, "fp32")])
def test_ffn_two_at_once(T, dt):
    sets = [inputs(T, 256, 512, 256, dt, seed=s) for s in (1, 2)]

    def step(t, g):
        leaves = [k.clone().requires_grad_(True) for k in t]
        y = ops().gated_ffn(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got.clear()
        for s, inp in zip(streams, sets):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(step(*inp))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("T,dt", [(8, "bf16"), (700, "fp16"), (90, "fp32")])
def test_ffn_step_in_two_graphs(T, dt):
    """Two captured training steps, replayed in turn and at once with new inputs, give what eager calls give."""
    steps = []
    for seed in (1, 2):
        t, g = inputs(T, 256, 512, 256, dt, seed=seed)
        leaves = [k.clone().requires_grad_(True) for k in t]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.autograd.grad(ops().gated_ffn(*leaves), leaves, g)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops().gated_ffn(*leaves)
            out = [y.detach(), *torch.autograd.grad(y, leaves, g)]
        steps.append((graph, leaves, g, out))
    for turn in range(2):
        fresh = [inputs(T, 256, 512, 256, dt, seed=10 + 2 * turn + i) for i in range(2)]
        for (graph, leaves, g, _), (t, gy) in zip(steps, fresh):
            with torch.no_grad():
                for p, q in zip(leaves, t):
                    p.copy_(q)
                g.copy_(gy)
        torch.cuda.synchronize()
        for graph, *_ in steps:
            with torch.cuda.stream(torch.cuda.Stream()):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, out), (t, gy) in zip(steps, fresh):
            leaves = [k.clone().requires_grad_(True) for k in t]
            y = ops().gated_ffn(*leaves)
            want = [y.detach(), *torch.autograd.grad(y, leaves, gy)]
            assert all(torch.equal(p, q) for p, q in zip(out, want))


# ------------------------------------------------------------------- values
@pytest.mark.parametrize("act", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("T", [3, 40])
def test_ffn_of_enormous_pre_activations(T, dt, act):
    """act and act' at the ends of float32's range: 0 and 0 below, a and 1 above, no NaN on the way."""
    x = torch.zeros(T, 8, device="cuda", dtype=DT[dt])
    x[0], x[1], x[2] = 1e30, -1e30, -20.0
    eye = torch.eye(8, device="cuda", dtype=DT[dt])
    up = torch.zeros_like(eye)
    up[:, 0] = 1e-30  # b = 1 for the first row, -1 and about 0 for the others
    leaves = [k.clone().requires_grad_(True) for k in (x, eye, up, eye)]
    y = ops().gated_ffn(*leaves, activation=act)
    assert torch.allclose(y[0].float(), torch.full((8,), 1e30, device="cuda"), rtol=2 ** -6)
    assert (y[1] == 0).all() and (y[2].float().abs() < 1e-6).all() and (y[3:] == 0).all()
    y.backward(torch.ones_like(y))
    assert all(leaves[i].grad.isfinite().all() for i in (0, 1, 3))  # w_up's is 1e30 x 1e30


# ------------------------------------------------------------ bounded waits
@pytest.fixture
def lib():
    from hyperconnections_b200 import _lib

    handle = _lib.lib()
    _lib.wait_timeouts(reset=True)
    yield handle
    assert handle.hc_debug_set_wait_limit(0) == 0
    _lib.wait_timeouts(reset=True)


def test_ffn_wait_gives_up(lib):
    """Waits of one poll end the tensor cores' pipeline early: the call returns, the status sticks until it is reset,
    and the same call then gives the same result."""
    from hyperconnections_b200 import _lib

    t, g = inputs(2000, 256, 768, 256, "bf16")
    leaves = [k.clone().requires_grad_(True) for k in t]
    want = ops().gated_ffn(*leaves)
    grads = torch.autograd.grad(want, leaves, g, retain_graph=True)
    torch.cuda.synchronize()
    assert _lib.timeout_status() == 0
    for launch in (lambda: ops().gated_ffn(*t), lambda: torch.autograd.grad(want, leaves, g, retain_graph=True)):
        assert lib.hc_debug_set_wait_limit(1) == 0
        try:
            for _ in range(5):
                try:
                    launch()
                except RuntimeError as e:
                    assert "gave up" in str(e)
                torch.cuda.synchronize()
                if _lib.timeout_status():
                    break
        finally:
            assert lib.hc_debug_set_wait_limit(0) == 0
        assert _lib.timeout_status() > 0, "no wait gave up with a one-poll limit"
        with pytest.raises(RuntimeError, match="gave up"):
            ops().gated_ffn(*t)
        count = ctypes.c_uint(0)
        assert lib.hc_wait_timeouts(ctypes.byref(count), 1) == 0 and count.value > 0
        assert torch.equal(ops().gated_ffn(*t), want)
        again = torch.autograd.grad(want, leaves, g, retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(again, grads))
