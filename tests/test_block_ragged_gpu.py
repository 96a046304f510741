"""GPU tests of hc_read_norm and hc_mix_write_norm where rows are not whole
chunks of eight columns or begin off a 16-byte boundary: odd and even lengths,
rows that end inside a word, many tokens a CTA (rows of both parities take
turns in the same shared memory), and what lies around the outputs."""

import pytest
import torch

from tests.test_block_gpu import check_read, check_write, leaf, ops, read_inputs, write_inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _cuda():
    if not torch.cuda.is_available():
        pytest.skip("CUDA not available")


READ = [
    # T, n, m, D, type, norm, affine
    (5, 4, 1, 769, "bf16", "rms", "w"),
    (300, 4, 1, 767, "bf16", "layer", "wb"),
    (64, 4, 1, 770, "fp16", "layer", "wb"),
    (64, 4, 4, 258, "fp16", "rms", "wb"),
    (4000, 3, 2, 61, "bf16", "layer", "wb"),
    (4000, 2, 1, 13, "fp16", "rms", "w"),
    (2500, 1, 1, 9, "fp32", "layer", "wb"),
    (1500, 8, 3, 131, "bf16", "rms", "b"),
    (40, 8, 4, 517, "fp32", "layer", "wb"),
    (7, 5, 1, 1001, "fp32", "rms", "w"),
    (9, 4, 2, 2047, "bf16", "layer", "w"),
    (3, 4, 1, 4095, "fp16", "rms", "wb"),
    (11, 8, 1, 3, "bf16", "layer", "wb"),
    (11, 6, 2, 1, "fp16", "rms", "wb"),
    (6, 4, 1, 257, "bf16", "layer", "w"),
    (6, 4, 1, 255, "fp32", "layer", "w"),
    # tokens that take more threads, and tokens too wide for a CTA
    (300, 8, 4, 4096, "bf16", "layer", "wb"),
    (5, 8, 1, 4095, "fp16", "rms", "w"),
    (5, 4, 4, 4096, "fp16", "layer", "wb"),
    (5, 8, 2, 2600, "fp32", "rms", "w"),
    (3, 8, 4, 6000, "fp32", "layer", "wb"),
    (3, 4, 4, 5001, "bf16", "rms", "w"),
    (600, 8, 1, 4100, "fp32", "layer", "wb"),
    (3, 1, 4, 100, "fp32", "layer", "wb"),
    (3, 2, 3, 77, "bf16", "rms", "wb"),
]


@pytest.mark.parametrize("T,n,m,D,dt,norm,affine", READ)
def test_read_norm(T, n, m, D, dt, norm, affine):
    R, x, w, b, gy = read_inputs(T, n, m, D, dt, affine)
    leaves = [leaf(t) for t in (R, x, w, b)]
    y = ops().hc_read_norm(*leaves, norm=norm, eps=1e-5)
    y.backward(gy)
    check_read(R, x, w, b, gy, norm, 1e-5, [y] + [None if t is None else t.grad for t in leaves])
    with torch.no_grad():
        assert torch.equal(ops().hc_read_norm(R, x, w, b, norm=norm, eps=1e-5), y)


WRITE = [
    # T, n, m, D, type, norm, affine, gate, proj, p
    (5, 4, 1, 769, "bf16", "rms", "ws", "sigmoid", False, 0.1),
    (300, 4, 1, 767, "bf16", "layer", "wbs", "linear", False, 0.0),
    (64, 4, 1, 770, "fp16", "layer", "wbs", "sigmoid", True, 0.3),
    (64, 4, 4, 258, "fp16", "rms", "wb", "", False, 0.2),
    (4000, 3, 2, 61, "bf16", "layer", "wbs", "sigmoid", True, 0.1),
    (4000, 2, 1, 13, "fp16", "none", "w", "linear", False, 0.5),
    (2500, 1, 1, 9, "fp32", "layer", "wb", "", True, 0.1),
    (1500, 8, 3, 131, "bf16", "rms", "bs", "sigmoid", True, 0.3),
    (40, 8, 4, 517, "fp32", "layer", "wbs", "linear", True, 0.1),
    (7, 5, 1, 1001, "fp32", "rms", "w", "sigmoid", False, 0.9),
    (9, 4, 2, 1023, "bf16", "layer", "ws", "", False, 0.1),
    (3, 4, 1, 2049, "fp16", "rms", "wb", "sigmoid", True, 0.1),
    (11, 8, 1, 3, "bf16", "none", "s", "linear", False, 0.1),
    (11, 6, 2, 1, "fp16", "rms", "wb", "", True, 0.0),
    (6, 4, 1, 257, "bf16", "layer", "w", "sigmoid", False, 0.1),
    (6, 4, 1, 255, "fp32", "layer", "w", "sigmoid", False, 0.1),
    (200, 8, 4, 4096, "bf16", "layer", "wbs", "sigmoid", True, 0.1),
    (5, 8, 1, 4095, "fp16", "rms", "ws", "linear", False, 0.3),
    (5, 4, 4, 4096, "fp16", "layer", "wb", "", True, 0.1),
    (5, 8, 2, 2056, "fp32", "rms", "ws", "sigmoid", True, 0.0),
    (3, 8, 4, 6000, "fp32", "layer", "wbs", "sigmoid", True, 0.2),
    (3, 4, 4, 5001, "bf16", "rms", "w", "linear", False, 0.1),
    (600, 8, 1, 4100, "fp32", "layer", "wb", "sigmoid", True, 0.1),
    (3, 1, 4, 100, "fp32", "layer", "wbs", "linear", True, 0.1),
    (3, 2, 3, 77, "bf16", "none", "s", "sigmoid", False, 0.1),
]


@pytest.mark.parametrize("T,n,m,D,dt,norm,affine,gate,proj,p", WRITE)
def test_mix_write_norm(T, n, m, D, dt, norm, affine, gate, proj, p):
    t, g = write_inputs(T, n, m, D, dt, affine, gate, proj)
    seed, offset = 0x1234567890ABCDEF, (1 << 40) + 3
    kw = dict(norm=norm, eps=1e-5, gate_activation=gate or "linear", dropout_p=p, seed=seed, offset=offset)
    call = lambda s: ops().hc_mix_write_norm(s["H"], s["x"], s["W"], s["f"], s["v"], weight=s["weight"],  # noqa: E731
                                             bias=s["bias"], gate=s["gate"], scale=s["scale"], **kw)
    leaves = {k: leaf(a) for k, a in t.items()}
    out = call(leaves)
    out.backward(g)
    check_write(t, g, norm, 1e-5, gate or "linear", p, seed, offset, out,
                {k: a.grad for k, a in leaves.items() if a is not None})
    with torch.no_grad():
        assert torch.equal(call(t), out)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("n,m,D", [(4, 1, 771), (8, 2, 130), (3, 1, 7), (4, 1, 768)])
def test_nothing_around_the_outputs_is_written(dt, n, m, D):
    """Every output of the four C calls lies inside a larger buffer, one element off a 16-byte boundary; what is around
    it keeps its value, and the results are those of the operators."""
    from hyperconnections_b200 import _lib

    lib, T, code = _lib.lib(), 70, {"fp32": 0, "fp16": 1, "bf16": 2}[dt]
    t, g = write_inputs(T, n, m, D, dt, "wbs", "sigmoid", False)
    R, x, w, b, gy = read_inputs(T, n, m, D, dt, "wb")
    stream = torch.cuda.current_stream().cuda_stream
    pad, rooms = 129, []

    def room(like, dtype=None):
        dtype = dtype or like.dtype
        whole = torch.full((like.numel() + 2 * pad,), 7.0, dtype=dtype, device="cuda")
        rooms.append((whole, like.numel()))
        return whole[pad:pad + like.numel()].view(like.shape)

    p = lambda a: a.data_ptr()  # noqa: E731
    f32 = torch.float32
    words = lib.hc_norm_scratch_words(T, n, m, D, code)
    scratch, stats = torch.empty(words, device="cuda"), torch.empty(T, 2, device="cuda")
    y, gx, gR, gw, gb = room(gy), room(x), room(R, f32), room(w, f32), room(b, f32)
    assert lib.hc_read_norm_fwd(p(R), p(x), p(w), p(b), p(y), p(stats), T, n, m, D, 2, 1e-5, code, stream) == 0
    assert lib.hc_read_norm_bwd(p(gy), p(R), p(x), p(w), p(stats), p(gx), p(gR), p(gw), p(gb), p(scratch), words, T, n, m, D,
                                2, code, stream) == 0
    check_read(R, x, w, b, gy, "layer", 1e-5, (y, gR, gx, gw, gb))
    out = room(t["x"])
    grads = {k: room(t[k], f32 if k in ("H", "W", "weight", "bias", "scale") else None)
             for k in ("H", "x", "W", "f", "weight", "bias", "gate", "scale")}
    assert lib.hc_mix_write_norm_fwd(p(t["H"]), p(t["x"]), p(t["W"]), p(t["f"]), None, p(t["weight"]), p(t["bias"]),
                                     p(t["gate"]), p(t["scale"]), p(out), p(stats), T, n, m, D, 2, 1, 1e-5, 0.25, None, 3, 4,
                                     code, stream) == 0
    assert lib.hc_mix_write_norm_bwd(
        p(g), p(t["H"]), p(t["x"]), p(t["W"]), p(t["f"]), None, p(t["weight"]), p(t["bias"]), p(t["gate"]), p(t["scale"]),
        p(stats), p(grads["x"]), p(grads["f"]), p(grads["gate"]), p(grads["H"]), p(grads["W"]), None, p(grads["weight"]),
        p(grads["bias"]), p(grads["scale"]), p(scratch), words, T, n, m, D, 2, 1, 0.25, None, 3, 4, code, stream) == 0
    check_write(t, g, "layer", 1e-5, "sigmoid", 0.25, 3, 4, out, grads)
    for whole, count in rooms:
        assert (whole[:pad] == 7).all() and (whole[pad + count:] == 7).all()
