"""CPU test: the C calls of the block's operators refuse pointers that are not
aligned to their type (the kernels would fault on them), before any launch."""

import pytest

from hyperconnections_b200 import _lib

ALIGN, NULL = 5, 1
P = 0x1000  # never dereferenced: every call below ends at a host-side check


def status(name, pointers, bad, *rest):
    a = [P] * pointers
    for i, by in bad.items():
        a[i] = P + by
    return getattr(_lib.lib(), name)(*a, *rest)


@pytest.mark.parametrize("dt,by", [(0, 1), (0, 2), (1, 1), (2, 1)])
def test_streams(dt, by):
    size = (4, 4, 1, 64)
    for i in (1, 4):  # x, y
        assert status("hc_read_norm_fwd", 6, {i: by}, *size, 1, 1e-6, dt, None) == ALIGN
    words = _lib.lib().hc_norm_scratch_words(*size, dt)
    for i in (0, 2, 5):  # g, x, grad_x
        assert status("hc_read_norm_bwd", 10, {i: by}, words, *size, 1, dt, None) == ALIGN
    for i in (1, 3, 7, 9):  # x, f, gate, out
        assert status("hc_mix_write_norm_fwd", 11, {i: by}, *size, 1, 1, 1e-6, 0.1, None, 1, 2, dt, None) == ALIGN
    for i in (0, 2, 4, 8, 11, 12, 13):  # g, x, f, gate and the gradients of x, f, gate
        assert status("hc_mix_write_norm_bwd", 21, {i: by}, words, *size, 1, 1, 0.1, None, 1, 2, dt, None) == ALIGN
    for i in (0, 1):
        assert status("hc_dropout", 2, {i: by}, 8, 0.5, None, 1, 2, dt, None) == ALIGN


@pytest.mark.parametrize("by", [1, 2, 4])
def test_seed_on_the_device(by):
    size = (4, 4, 1, 64)
    words = _lib.lib().hc_norm_scratch_words(*size, 2)
    assert status("hc_mix_write_norm_fwd", 11, {}, *size, 1, 1, 1e-6, 0.1, P + by, 1, 2, 2, None) == ALIGN
    assert status("hc_mix_write_norm_bwd", 21, {}, words, *size, 1, 1, 0.1, P + by, 1, 2, 2, None) == ALIGN
    assert status("hc_dropout", 2, {}, 8, 0.5, P + by, 1, 2, 2, None) == ALIGN


@pytest.mark.parametrize("dt,by", [(0, 2), (1, 8), (2, 2)])
def test_feed_forward(dt, by):
    for i in range(8):
        assert status("hc_gated_ffn_fwd", 8, {i: by}, P, 1 << 40, 8, 64, 128, 64, 2, dt, None) == ALIGN
    for i in range(14):
        assert status("hc_gated_ffn_bwd", 14, {i: by}, P, 1 << 40, 8, 64, 128, 64, 2, dt, None) == ALIGN
