"""CPU tests of the operators around a layer's block: what the C entry points
and the Python operators refuse, before any launch."""

import ctypes

import pytest
import torch

from hyperconnections_b200 import _lib

OK, NULL, SIZE, N, DTYPE, ALIGN, SCRATCH = range(7)
P = 0x1000  # never dereferenced: every call below ends at a host-side check


def read_fwd(R=P, x=P, w=P, b=P, y=P, st=P, T=4, n=4, m=1, D=64, norm=1, eps=1e-6, dt=2):
    return _lib.lib().hc_read_norm_fwd(R, x, w, b, y, st, T, n, m, D, norm, eps, dt, None)


@pytest.mark.parametrize("kw,want", [
    (dict(n=9), N), (dict(n=0), N), (dict(m=5), N), (dict(m=0), N), (dict(T=-1), SIZE), (dict(D=-1), SIZE),
    (dict(T=1 << 31), SIZE), (dict(D=(1 << 24) + 1), SIZE), (dict(norm=0), SIZE), (dict(norm=3), SIZE),
    (dict(eps=-1.0), SIZE), (dict(eps=float("nan")), SIZE), (dict(dt=3), DTYPE), (dict(R=None), NULL),
    (dict(x=None), NULL), (dict(y=None), NULL), (dict(w=P + 2), ALIGN), (dict(st=P + 1), ALIGN),
    (dict(T=0, x=None), OK), (dict(D=0, x=None), OK),
])
def test_read_norm_fwd(kw, want):
    assert read_fwd(**kw) == want


def test_read_norm_bwd():
    lib = _lib.lib()
    words = lib.hc_norm_scratch_words(100, 4, 2, 64, 2)
    assert words > 0 and words % (2 * 2 * 64) == 0
    call = lambda g=P, st=P, gw=P, sc=P, w=words, n=4, norm=1, dt=2: lib.hc_read_norm_bwd(  # noqa: E731
        g, P, P, P, st, P, P, gw, P, sc, w, 100, n, 2, 64, norm, dt, None)
    assert call(w=words - 1) == SCRATCH and call(sc=None) == SCRATCH
    assert call(g=None) == NULL and call(st=None) == NULL and call(n=9) == N and call(norm=0) == SIZE
    assert call(dt=7) == DTYPE and call(gw=P + 2) == ALIGN
    for bad in ((-1, 4, 1, 64, 2), (10, 9, 1, 64, 2), (10, 4, 1, 64, 9), (0, 4, 1, 64, 2)):
        assert lib.hc_norm_scratch_words(*bad) == 0


def write_fwd(H=P, x=P, W=P, f=P, v=P, out=P, T=4, n=4, m=1, D=64, norm=1, act=1, eps=1e-6, p=0.1, dt=2):
    return _lib.lib().hc_mix_write_norm_fwd(H, x, W, f, v, P, P, P, P, out, P, T, n, m, D, norm, act, eps, p, None, 1, 2, dt,
                                            None)


@pytest.mark.parametrize("kw,want", [
    (dict(n=9), N), (dict(m=5), N), (dict(T=-1), SIZE), (dict(norm=-1), SIZE), (dict(norm=3), SIZE), (dict(act=2), SIZE),
    (dict(p=-0.1), SIZE), (dict(p=1.5), SIZE), (dict(p=float("nan")), SIZE), (dict(eps=-1.0), SIZE), (dict(dt=5), DTYPE),
    (dict(H=None), NULL), (dict(f=None), NULL), (dict(out=None), NULL), (dict(v=P + 2), ALIGN), (dict(T=0), OK),
])
def test_mix_write_norm_fwd(kw, want):
    assert write_fwd(**kw) == want


def test_mix_write_norm_bwd():
    lib = _lib.lib()
    words = lib.hc_norm_scratch_words(100, 4, 1, 64, 2)

    def call(ptrs=(), w=words, norm=1, act=1, p=0.1, dt=2, n=4):
        a = [P] * 21
        for i, q in ptrs:
            a[i] = q
        return lib.hc_mix_write_norm_bwd(*a, w, 100, n, 1, 64, norm, act, p, None, 1, 2, dt, None)

    assert call(w=words - 1) == SCRATCH and call([(20, None)]) == SCRATCH
    assert call([(0, None)]) == NULL and call([(1, None)]) == NULL and call([(10, None)]) == NULL
    assert call([(14, P + 2)]) == ALIGN and call(norm=4) == SIZE and call(act=3) == SIZE and call(p=2.0) == SIZE
    assert call(dt=-1) == DTYPE and call(n=0) == N


def test_dropout():
    lib = _lib.lib()
    call = lambda x=P, y=P, N=8, p=0.5, dt=2: lib.hc_dropout(x, y, N, p, None, 1, 2, dt, None)  # noqa: E731
    assert call(N=-1) == SIZE and call(p=-0.5) == SIZE and call(p=1.01) == SIZE and call(p=float("nan")) == SIZE
    assert call(dt=3) == DTYPE and call(x=None) == NULL and call(y=None) == NULL and call(x=None, N=0) == OK


def test_gated_ffn():
    lib = _lib.lib()
    size = lib.hc_gated_ffn_scratch_bytes
    for bwd in (0, 1):
        assert size(bwd, 8, 64, 128, 64, 2) >= 0
        for bad in ((-1, 64, 128, 64, 2), (8, 0, 128, 64, 2), (8, 64, 0, 64, 2), (8, 64, 128, 0, 2), (8, 64, 128, 64, 3),
                    (8, (1 << 20) + 1, 128, 64, 2), (1 << 40, 64, 128, 64, 2)):
            assert size(bwd, *bad) == -1
    big = 1 << 40

    def fwd(ptrs=(), scratch=P, nbytes=big, T=8, D=64, F=128, O=64, act=2, dt=2):
        a = [P] * 8
        for i, q in ptrs:
            a[i] = q
        return lib.hc_gated_ffn_fwd(*a, scratch, nbytes, T, D, F, O, act, dt, None)

    assert fwd(T=-1) == SIZE and fwd(D=0) == SIZE and fwd(act=1) == SIZE and fwd(act=4) == SIZE and fwd(dt=9) == DTYPE
    assert fwd([(0, None)]) == NULL and fwd([(5, None)]) == NULL and fwd([(6, None)]) == NULL and fwd(T=0) == OK
    assert fwd([(4, P + 2)]) == ALIGN and fwd(D=63, scratch=P + 32) == ALIGN and fwd(D=63, scratch=None) == SCRATCH

    def bwd(ptrs=(), T=8, act=2, dt=2):
        a = [P] * 15
        for i, q in ptrs:
            a[i] = q
        return lib.hc_gated_ffn_bwd(*a, big, T, 64, 128, 64, act, dt, None)

    assert bwd(T=-1) == SIZE and bwd(act=0) == SIZE and bwd(dt=4) == DTYPE
    for i in (0, 1, 4, 5, 6, 8):
        assert bwd([(i, None)]) == NULL


def test_cpu_tensors_raise_without_fallback():
    from hyperconnections_b200 import ops

    x, R = torch.randn(2, 4, 8), torch.randn(2, 1, 4)
    H, W, f = torch.randn(2, 4, 4), torch.randn(2, 4, 1), torch.randn(2, 1, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hc_read_norm(R, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hc_mix_write_norm(H, x, W, f)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.hc_dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.gated_ffn(x, torch.randn(16, 8), torch.randn(16, 8), torch.randn(8, 16))



def test_python_refusals(monkeypatch):
    from hyperconnections_b200 import ops
    from hyperconnections_b200.ops import block, dropout, ffn

    monkeypatch.setattr(block, "_require_cuda", lambda *a: None)
    x, R = torch.randn(2, 4, 8), torch.randn(2, 1, 4)
    H, W, f = torch.randn(2, 4, 4), torch.randn(2, 4, 1), torch.randn(2, 1, 8)
    with pytest.raises(ValueError, match="norm"):
        ops.hc_read_norm(R, x, norm="none")
    with pytest.raises(ValueError, match="eps"):
        ops.hc_read_norm(R, x, eps=-1e-6)
    with pytest.raises(AssertionError, match="R must be"):
        ops.hc_read_norm(R[:1], x)
    with pytest.raises(AssertionError, match="weight"):
        ops.hc_read_norm(R, x, torch.ones(7))
    with pytest.raises(RuntimeError, match="streams"):
        ops.hc_read_norm(torch.randn(2, 1, 9), torch.randn(2, 9, 8))
    with pytest.raises(RuntimeError, match="one device"):
        ops.hc_read_norm(R.to("meta"), x)
    with pytest.raises(ValueError, match="norm"):
        ops.hc_mix_write_norm(H, x, W, f, norm="batch")
    with pytest.raises(ValueError, match="gate_activation"):
        ops.hc_mix_write_norm(H, x, W, f, gate_activation="tanh")
    with pytest.raises(AssertionError, match="f must be"):
        ops.hc_mix_write_norm(H, x, W, f[:, :, :4])
    with pytest.raises(ValueError, match="seed"):
        ops.hc_mix_write_norm(H, x, W, f, dropout_p=0.5)
    with pytest.raises(ValueError, match="dropout_p"):
        ops.hc_mix_write_norm(H, x, W, f, dropout_p=1.5, seed=1)
    with pytest.raises(ValueError, match="seed tensor"):
        ops.hc_mix_write_norm(H, x, W, f, dropout_p=0.5, seed=torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="offset"):
        ops.hc_mix_write_norm(H, x, W, f, dropout_p=0.5, seed=torch.zeros(2, dtype=torch.int64), offset=3)
    assert dropout.drop_words(-1, 1 << 64) == (-1, 0) and dropout.drop_words(1 << 63, 5) == (-(1 << 63), 5)
    assert set(ffn._ACT) == {"silu", "gelu_tanh"}


def test_philox_words_at_the_counters_edges():
    """Counter halves carry: element 2^34 is block 2^32, whose high counter word is 1."""
    import numpy as np

    from oracle.block import philox_words

    lo, hi = philox_words(np.array([0, 1 << 34], np.uint64), 5, 9)
    assert lo != hi
    assert ctypes.c_uint32(int(hi)).value == int(hi)


def test_philox_published_words():
    """The words that the generator's authors publish for counter and key zero."""
    import numpy as np

    from oracle.block import philox_words

    assert [int(w) for w in philox_words(np.arange(4), 0, 0)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
