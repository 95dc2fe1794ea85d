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


@pytest.mark.parametrize("window,sinks", [(2 ** 64 + 5, 0), (5, 2 ** 64 + 3), (2 ** 70, 2 ** 70)])
def test_windows_beyond_64_bits_are_all_of_the_cache(window, sinks, monkeypatch):
    """A count beyond any cache means the whole of it and must not wrap around."""
    import torch

    from hbq_b200 import _lib, attention
    seen = []

    class Library:
        @staticmethod
        def hbq_attention_workspace_bytes(a):
            seen.append((a._obj.window, a._obj.sinks))
            return 0

        @staticmethod
        def hbq_attention_run(a, *rest):
            return 0
    monkeypatch.setattr(attention._lib, "lib", lambda: Library)
    monkeypatch.setattr(attention, "_check_devices", lambda *a: None)
    monkeypatch.setattr(attention, "_stream_ptr", lambda d: 0)
    monkeypatch.setattr(_lib, "device_guard", lambda d: __import__("contextlib").nullcontext())
    q, k = torch.zeros((1, 2, 2, 64), dtype=torch.float16), torch.zeros((1, 2, 9, 64), dtype=torch.float16)
    attention.window_attention(q, k, k.clone(), window=window, sinks=sinks, out=torch.empty_like(q))
    assert all(a == b if b < 9 else 9 <= a for a, b in zip(seen[0], (window, sinks)))
