"""Newton-Schulz orthogonalisation, host side: workspace and refusals of the C entry, without a GPU."""

import ctypes

from torchft_amd import _lib

I64 = ctypes.c_int64


def shapes(*s):
    return (I64 * (2 * len(s)))(*[v for p in s for v in p])


def test_workspace():
    L = _lib.load()
    half = L.tftq_newton_schulz_workspace(1, shapes((4096, 14336)), 0)
    full = L.tftq_newton_schulz_workspace(1, shapes((4096, 14336)), 1)
    x, a = 4096 * 14336 * 2, 4096 * 4096 * 2
    # X and its remainder, X^T twice, A and B; precise: remainders of X^T, A and B too
    assert 4 * x + 2 * a <= half <= 4 * x + 2 * a + (1 << 20)
    assert 6 * x + 4 * a <= full <= 6 * x + 4 * a + (1 << 20)
    assert L.tftq_newton_schulz_workspace(1, shapes((14336, 4096)), 0) >= 4 * x + 2 * a
    assert half % 128 == 0 and L.tftq_newton_schulz_workspace(1, shapes((3, 5)), 1) % 128 == 0
    one = L.tftq_newton_schulz_workspace(1, shapes((100, 200)), 0)
    assert L.tftq_newton_schulz_workspace(24, shapes(*[(100, 200)] * 24), 0) == 24 * one
    assert L.tftq_newton_schulz_workspace(70, shapes(*[(100, 200)] * 70), 0) == 24 * one  # one launch's matrices at a time
    assert L.tftq_newton_schulz_workspace(2, shapes((0, 5), (5, 0)), 0) == 0
    assert L.tftq_newton_schulz_workspace(0, None, 0) == 0
    assert L.tftq_newton_schulz_workspace(1, None, 0) == -1
    assert L.tftq_newton_schulz_workspace(1, shapes((-1, 4)), 0) == -3
    assert L.tftq_newton_schulz_workspace(1, shapes((4, 2 ** 24 + 1)), 0) == -3


def test_refuses_before_it_launches():
    L = _lib.load()
    buf = (ctypes.c_uint8 * 4096)()
    at = (ctypes.addressof(buf) + 127) & ~127

    def call(workspace=at, size=1 << 40, **changes):
        one = (ctypes.c_void_p * 1)(at)
        kept = dict(n=1, shapes=shapes((4, 6)), inputs=one, in_stride=(I64 * 1)(6), in_dtype=0, out=one, out_stride=(I64 * 1)(6),
                    out_dtype=0, iterations=1, coefficients=(ctypes.c_float * 3)(1, 2, 3), eps=1e-7)
        kept.update(changes)
        return L.tftq_newton_schulz(ctypes.byref(_lib.NewtonSchulz(**kept)), workspace, size, -1, None)
    assert L.tftq_newton_schulz(None, at, 0, -1, None) == -1
    assert call(n=-1) == -1 and call(n=0) == 0
    assert call(shapes=None) == -1 and call(inputs=None) == -1 and call(out=None) == -1 and call(coefficients=None) == -1
    assert call(iterations=0) == -1
    assert call(in_dtype=3) == -2 and call(out_dtype=-1) == -2
    assert call(shapes=shapes((4, -6))) == -3
    assert call(in_stride=(I64 * 1)(5)) == -1 and call(out_stride=(I64 * 1)(5)) == -1
    assert call(inputs=(ctypes.c_void_p * 1)(None)) == -1
    assert call(momenta=(ctypes.c_void_p * 1)(at)) == -1
    assert call(momenta=(ctypes.c_void_p * 1)(None), momenta_stride=(I64 * 1)(6)) == -1
    assert call(size=64) == -4
    assert call(workspace=None) == -1 and call(workspace=at + 64) == -1
    assert call(shapes=shapes((0, 6))) == 0


def test_workspace_of_the_largest():
    """Refused before anything is queued; a list of large ones is taken in parts."""
    L = _lib.load()
    assert L.tftq_newton_schulz_workspace(1, shapes((2 ** 24, 2 ** 12)), 0) == -3
    one = L.tftq_newton_schulz_workspace(1, shapes((2 ** 17, 2 ** 17)), 0)
    assert one > 4 * 2 * 2 ** 34
    assert L.tftq_newton_schulz_workspace(2, shapes((2 ** 17, 2 ** 17), (2 ** 17, 2 ** 17)), 0) == 2 * one
    assert L.tftq_newton_schulz_workspace(5, shapes(*[(2 ** 17, 2 ** 17)] * 5), 0) == 2 * one
