"""CPU: frequencies of the rotary embedding against their formulas, and what the rotary and attention entry points refuse."""
import math

import pytest

torch = pytest.importorskip("torch")


def test_plain_and_linear_frequencies():
    import hbq_b200 as H
    f, m = H.rope_frequencies(128, 500000.0)
    assert f.dtype == torch.float64 and f.shape == (64,) and m == 1.0
    for i in (0, 1, 31, 63):
        assert math.isclose(f[i].item(), 500000.0 ** (-2 * i / 128), rel_tol=1e-14)
    g, m = H.rope_frequencies(128, 500000.0, {"type": "linear", "factor": 4.0})
    assert torch.equal(g, f / 4) and m == 1.0
    h, _ = H.rope_frequencies(128, 500000.0, {"rope_type": "default"})
    assert torch.equal(h, f)


def test_ntk_frequencies_slow_the_last_pair_alone_by_the_factor():
    import hbq_b200 as H
    f, _ = H.rope_frequencies(64, 10000.0)
    g, m = H.rope_frequencies(64, 10000.0, {"type": "ntk", "factor": 8.0})
    # base' = base * s^(r / (r - 2)): pair r / 2 - 1 has exponent (r - 2) / r, so it slows by s exactly; pair 0 keeps its 1
    assert m == 1.0 and g[0] == 1.0 and math.isclose((f[-1] / g[-1]).item(), 8.0, rel_tol=1e-12)
    assert bool((g[1:] < f[1:]).all())


def test_llama3_frequencies_in_bands():
    import hbq_b200 as H
    s = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}
    f, _ = H.rope_frequencies(128, 500000.0)
    g, m = H.rope_frequencies(128, 500000.0, s)
    assert m == 1.0
    for a, b in zip(f.tolist(), g.tolist()):
        wavelength = 2 * math.pi / a
        if wavelength < 8192 / 4.0:
            want = a
        elif wavelength > 8192 / 1.0:
            want = a / 8.0
        else:
            smooth = (8192 / wavelength - 1.0) / (4.0 - 1.0)
            want = (1 - smooth) * a / 8.0 + smooth * a
        assert math.isclose(b, want, rel_tol=1e-12)


def test_yarn_frequencies():
    import hbq_b200 as H
    s = {"type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    f, _ = H.rope_frequencies(64, 10000.0)
    g, m = H.rope_frequencies(64, 10000.0, s)
    assert math.isclose(m, 0.1 * math.log(16.0) + 1.0, rel_tol=1e-15)
    at = lambda turns: 64 * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))  # noqa: E731
    low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), 63)
    for i, (a, b) in enumerate(zip(f.tolist(), g.tolist())):
        ramp = min(max((i - low) / (high - low), 0.0), 1.0)
        assert math.isclose(b, a / 16.0 * ramp + a * (1 - ramp), rel_tol=1e-12)
    assert H.rope_frequencies(64, 10000.0, dict(s, attention_factor=1.5))[1] == 1.5


@pytest.mark.parametrize("call", [
    lambda H: H.rope_frequencies(63, 1e4), lambda H: H.rope_frequencies(0, 1e4), lambda H: H.rope_frequencies(64, 0.0),
    lambda H: H.rope_frequencies(64, 1e4, {"type": "linear", "factor": 0.0}), lambda H: H.rope_frequencies(64, 1e4, {"type": "other", "factor": 2.0}),
    lambda H: H.rope_frequencies(2, 1e4, {"type": "ntk", "factor": 2.0}),
    lambda H: H.rope_frequencies(64, 1e4, {"type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0,
                                           "original_max_position_embeddings": 8192})])
def test_frequencies_refused(call):
    import hbq_b200 as H
    with pytest.raises(ValueError):
        call(H)


def _rope_args(**kw):
    a = dict(x=torch.zeros((2, 5, 3, 64), dtype=torch.float16), inv_freq=torch.ones(32, dtype=torch.float64), positions=torch.arange(5))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error", [
    (dict(x=torch.zeros((5, 64), dtype=torch.float16)), ValueError), (dict(x=torch.zeros((2, 5, 3, 64))), NotImplementedError),
    (dict(inv_freq=torch.ones(32)), ValueError), (dict(inv_freq=torch.ones(33, dtype=torch.float64)), ValueError),
    (dict(inv_freq=torch.ones(0, dtype=torch.float64)), ValueError), (dict(inv_freq=torch.ones((1, 32), dtype=torch.float64)), ValueError),
    (dict(positions=torch.arange(4)), ValueError), (dict(positions=torch.zeros((3, 5), dtype=torch.int64)), ValueError),
    (dict(positions=torch.zeros(5)), ValueError), (dict(out=torch.zeros((2, 5, 3, 32), dtype=torch.float16)), ValueError),
    (dict(out=torch.zeros((2, 5, 3, 64), dtype=torch.bfloat16)), ValueError),
    (dict(out=torch.zeros((1, 5, 3, 64), dtype=torch.float16).expand(2, 5, 3, 64)), ValueError),
    (dict(out=torch.zeros((2, 5, 64, 3), dtype=torch.float16).transpose(2, 3)), ValueError),
    (dict(x=torch.zeros((2, 5, 3, 64), dtype=torch.float16, requires_grad=True)), NotImplementedError)])
def test_rope_refusals(kw, error):
    import hbq_b200 as H
    with pytest.raises(error):
        H.rope_rotate(**_rope_args(**kw))


def _norm_args(**kw):
    a = dict(q=torch.zeros((2, 5, 4, 64), dtype=torch.float16), k=torch.zeros((2, 5, 2, 64), dtype=torch.float16),
             q_weight=torch.ones(64, dtype=torch.float16), k_weight=torch.ones(64, dtype=torch.float16), eps=1e-5,
             inv_freq=torch.ones(32, dtype=torch.float64), positions=torch.arange(5))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error", [
    (dict(k=torch.zeros((2, 5, 2, 32), dtype=torch.float16)), ValueError), (dict(k=torch.zeros((2, 4, 2, 64), dtype=torch.float16)), ValueError),
    (dict(k=torch.zeros((2, 5, 2, 64), dtype=torch.bfloat16)), ValueError), (dict(q_weight=torch.ones(32, dtype=torch.float16)), ValueError),
    (dict(k_weight=torch.ones(64)), ValueError), (dict(q=torch.zeros((5, 64), dtype=torch.float16)), ValueError),
    (dict(q_weight=torch.ones(64, dtype=torch.float16, requires_grad=True)), NotImplementedError)])
def test_norm_refusals(kw, error):
    import hbq_b200 as H
    with pytest.raises(error):
        H.qk_norm_rope(**_norm_args(**kw))


def _attn_args(**kw):
    h = torch.float16
    a = dict(q=torch.zeros((2, 3, 4, 64), dtype=h), k=torch.zeros((2, 2, 9, 64), dtype=h), v=torch.zeros((2, 2, 9, 64), dtype=h))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,error", [
    (dict(q=torch.zeros((3, 4, 64), dtype=torch.float16)), ValueError), (dict(v=torch.zeros((2, 2, 8, 64), dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros((2, 3, 5, 64), dtype=torch.float16)), ValueError), (dict(q=torch.zeros((1, 3, 4, 64), dtype=torch.float16)), ValueError),
    (dict(v=torch.zeros((2, 2, 9, 64), dtype=torch.bfloat16)), NotImplementedError), (dict(q=torch.zeros((2, 3, 4, 64))), NotImplementedError),
    (dict(window=-1), ValueError), (dict(sinks=-1), ValueError), (dict(scale=0.0), ValueError), (dict(scale=-1.0), ValueError),
    (dict(scale=float("inf")), ValueError), (dict(scale=float("nan")), ValueError),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(lengths=torch.zeros(2)), ValueError),
    (dict(starts=torch.zeros((2, 1), dtype=torch.int32)), ValueError), (dict(out=torch.zeros((2, 4, 3, 64), dtype=torch.float16)), ValueError),
    (dict(q=torch.zeros((2, 3, 4, 64), dtype=torch.float16, requires_grad=True)), NotImplementedError)])
def test_window_attention_refusals(kw, error):
    import hbq_b200 as H
    with pytest.raises(error):
        H.window_attention(**_attn_args(**kw))


@pytest.mark.parametrize("D", [4, 12, 136, 256])
def test_head_lengths_refused(D):
    import hbq_b200 as H
    h = torch.float16
    with pytest.raises(NotImplementedError):
        H.window_attention(torch.zeros((1, 1, 2, D), dtype=h), torch.zeros((1, 2, 3, D), dtype=h), torch.zeros((1, 2, 3, D), dtype=h))


def test_out_is_no_input():
    import hbq_b200 as H
    a = _attn_args()
    with pytest.raises(ValueError):
        H.window_attention(**a, out=a["q"])


@pytest.mark.parametrize("pk,pv,error", [
    ((2, 7, 32), (2, 7, 32), ValueError), ((2, 7, 64), (2, 6, 64), ValueError), ((1, 7, 64), (1, 7, 64), ValueError), (None, None, ValueError)])
def test_shared_prefix_refusals(pk, pv, error):
    import hbq_b200 as H
    t = [None if s is None else torch.zeros(s, dtype=torch.float16) for s in (pk, pv)]
    a = _attn_args()
    with pytest.raises(error):
        H.shared_prefix_attention(a["q"], t[0], t[1], a["k"], a["v"])


def test_no_cpu_fallback():
    import hbq_b200 as H
    with pytest.raises(H.HbqError):
        H.rope_rotate(**_rope_args())
    with pytest.raises(H.HbqError):
        H.qk_norm_rope(**_norm_args())
    with pytest.raises(H.HbqError):
        H.window_attention(**_attn_args())
    a, p = _attn_args(), torch.zeros((2, 7, 64), dtype=torch.float16)
    with pytest.raises(H.HbqError):
        H.shared_prefix_attention(a["q"], p, p, a["k"], a["v"])


def test_c_entry_points_check_their_arguments():
    """Return codes before any launch: nothing of the call reaches a GPU."""
    import ctypes

    from hbq_b200 import _lib
    L, i3, i2 = _lib.lib(), ctypes.c_int64 * 3, ctypes.c_int64 * 2
    p = ctypes.c_void_p(1 << 20)

    def attention(**kw):
        a = _lib.Attention(p, p, p, p, 1, 1, 4, 2, 9, 64, i3(64 * 4, 64 * 4, 64), i3(64 * 18, 64 * 9, 64), i3(64 * 18, 64 * 9, 64),
                           i3(64 * 4, 64 * 4, 64), None, None, None, None, 0, i2(0, 0), i2(0, 0), 0, 0, 0.125, 0)
        for n, v in kw.items():
            setattr(a, n, v)
        return L.hbq_attention_run(ctypes.byref(a), None, 0, None)
    assert attention(B=-1) == -1 and attention(H=5) == -1 and attention(Hkv=0) == -1 and attention(scale=-1.0) == -1
    assert attention(scale=float("nan")) == -1 and attention(dtype=2) == -1 and attention(sinks=-1) == -1 and attention(q=None) == -1
    assert attention(k=None) == -1 and attention(P=3) == -1
    assert attention(D=136) == -2 and attention(D=60) == -2 and attention(S=1 << 31) == -2 and attention(B=1 << 17) == -2
    assert attention(q=ctypes.c_void_p((1 << 20) + 2)) == -4 and attention(k_stride=i3(64 * 18, 64 * 9, 68)) == -4
    assert attention(B=0) == 0 and attention(L=0) == 0 and attention(H=0) == 0
    assert L.hbq_attention_run(None, None, 0, None) == -1

    def rope(T=1, D=64, dtype=0, heads=2, **kw):
        h = _lib.Heads(p, p, p, heads, i3(128, 128, 64), i3(128, 128, 64))
        r = _lib.Rotary(p, p, i2(0, 1), 64, 0, 1, 1.0)
        for n, v in kw.items():
            setattr(r if hasattr(r, n) else h, n, v)
        return L.hbq_rope_rotate(ctypes.byref(h), ctypes.byref(r), dtype, 1, T, D, None)
    assert rope(rot=0) == -1 and rope(rot=63) == -1 and rope(rot=66) == -1 and rope(dtype=5) == -1 and rope(T=-1) == -1 and rope(D=0) == -1
    assert rope(inv_freq=None) == -1 and rope(positions=None) == -1 and rope(data=None) == -1 and rope(out=None) == -1
    assert rope(T=0) == 0 and rope(heads=0) == 0 and rope(T=1 << 31) == -2
