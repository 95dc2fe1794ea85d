"""CPU: what the C entry of the attention refuses before any launch, at the ends of its ranges."""
import ctypes

import pytest

pytest.importorskip("torch")
ARG, UNSUPPORTED, ALIGN = -1, -2, -4
I3, I2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2


def _run(**kw):
    """Two sequences of four tokens; the pointers are never followed."""
    from hbq_b200 import _lib
    p = ctypes.c_void_p(1 << 20)
    a = _lib.Attention(p, p, p, p, 2, 4, 4, 2, 9, 64, I3(1024, 256, 64), I3(64 * 18, 64 * 9, 64), I3(64 * 18, 64 * 9, 64), I3(1024, 256, 64),
                       None, None, None, None, 0, I2(0, 0), I2(0, 0), 0, 0, 0.125, 0)
    for n, v in kw.items():
        setattr(a, n, v)
    return _lib.lib().hbq_attention_run(ctypes.byref(a), None, 0, None)


def test_key_counts_next_to_32_bits():
    """Key positions are 32-bit numbers in the kernels, and a tile of 128 keys may end behind the last key."""
    p = ctypes.c_void_p(1 << 20)
    for n in (2 ** 31 - 1, 2 ** 31 - 128, 2 ** 31 - 255):
        assert _run(S=n) == UNSUPPORTED
        assert _run(P=n, prefix_k=p, prefix_v=p, pk_stride=I2(64, 64), pv_stride=I2(64, 64)) == UNSUPPORTED


def test_strides_that_the_kernels_maps_cannot_hold():
    """Caches with negative strides, outputs whose elements are not separate: the copies' maps would take the axis for a dense one."""
    p = ctypes.c_void_p(1 << 20)
    for axis in range(3):
        down = [64 * 18, 64 * 9, 64]
        down[axis] *= -1
        assert _run(k_stride=I3(*down)) == ALIGN and _run(v_stride=I3(*down)) == ALIGN
        for s in (0, -64):
            out = [1024, 256, 64]
            out[axis] = s
            assert _run(out_stride=I3(*out)) == ALIGN
    for axis in range(2):
        down = [64 * 9, 64]
        down[axis] *= -1
        prefix = dict(P=9, prefix_k=p, prefix_v=p)
        assert _run(**prefix, pk_stride=I2(*down), pv_stride=I2(64 * 9, 64)) == ALIGN
        assert _run(**prefix, pk_stride=I2(64 * 9, 64), pv_stride=I2(*down)) == ALIGN


def test_scales_at_the_ends_of_32_bits():
    """The kernels work in powers of two: the scale times log2(e) has to be a number of 32 bits."""
    for scale in (2.5e38, 3.4e38, 1e39, 0.0, 1e-46):
        assert _run(scale=scale) == ARG
