"""GPU tests of gated_ffn's tensor-core products where a pair of CTAs makes many
tiles, one behind the other in two accumulators: h, its slopes and da, db of a
call with many tiles a pair equal bit for bit those of calls with at most one
(a tile's sums do not depend on the walk), and calls repeat themselves."""

import pytest
import torch

from tests.test_ffn_gpu import DT, ffn, inputs

pytestmark = pytest.mark.gpu

CODE = {"fp16": 1, "bf16": 2}


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


def inner(t, g, act):
    """h, the slopes, da, db and grad_x by the C calls."""
    from hyperconnections_b200 import _lib

    lib = _lib.lib()
    x, wg, wu, wd = t
    (T, D), (O, F) = x.shape, wd.shape
    dt = x.dtype
    code = CODE[{v: k for k, v in DT.items()}[dt]]
    h, sg, su, da, db = (torch.empty(T, (F + 7) // 8 * 8, dtype=dt, device="cuda") for _ in range(5))
    y, gx = torch.empty(T, O, dtype=dt, device="cuda"), torch.empty_like(x)
    p = lambda a: a.data_ptr()  # noqa: E731
    stream = torch.cuda.current_stream().cuda_stream
    sizes = [lib.hc_gated_ffn_scratch_bytes(b, T, D, F, O, code) for b in (0, 1)]
    scratch = torch.empty(max(sizes) + 256, dtype=torch.uint8, device="cuda")
    assert lib.hc_gated_ffn_fwd(p(x), p(wg), p(wu), p(wd), p(y), p(h), p(sg), p(su), p(scratch), sizes[0], T, D, F, O, act,
                                code, stream) == 0
    assert lib.hc_gated_ffn_bwd(p(g), p(x), p(wg), p(wu), p(wd), p(h), p(sg), p(su), p(da), p(db), p(gx), None, None, None,
                                p(scratch), sizes[1], T, D, F, O, act, code, stream) == 0
    return [a[:, :F] for a in (h, sg, su, da, db)]


@pytest.mark.parametrize("T,D,F,O,dt,act", [
    (256 * 160, 64, 512, 64, "bf16", 2),
    (256 * 100, 192, 1024, 128, "fp16", 3),
    (256 * 90, 128, 1000, 192, "bf16", 3),
])
def test_many_tiles_a_pair(T, D, F, O, dt, act):
    t, g = inputs(T, D, F, O, dt)
    rows = 256 * (148 // 2 // ((F + 127) // 128))  # tiles for half of the pairs at most
    alone = [inner([t[0][i:i + rows], *t[1:]], g[i:i + rows], act) for i in range(0, T, rows)]
    alone = [torch.cat(a) for a in zip(*alone)]
    for _ in range(3):
        for a, b in zip(inner(t, g, act), alone):
            assert torch.equal(a, b)


@pytest.mark.parametrize("T,D,F,O,dt", [(9000, 72, 1112, 64, "bf16"), (20000, 64, 264, 136, "fp16"), (6000, 512, 1536, 512, "bf16")])
def test_steps_repeat_themselves(T, D, F, O, dt):
    t, g = inputs(T, D, F, O, dt)
    leaves = [k.clone().requires_grad_(True) for k in t]

    def step():
        y = ffn(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, g)]

    first = step()
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip(step(), first))
