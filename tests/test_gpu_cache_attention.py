"""GPU: attention over a cache (window and first tokens, shared prefix) against the formulas in 64 bits.

Tolerance, for a row with weights w (sum 1) over n keys: the output's rounding, half a step of |o|; the weights' rounding to
the tensors' type, half a step of sum w |v|; the scores' 32-bit sums of D products, whose error in an exponent is at most
2^-20 of A = max sum |q k| scale (a relative error of that size in every weight, numerator and denominator: 4 of them), and
the additions of the weighted sum, 16 keys at a time, each to 2^-22 of sum w |v|."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _visible(L, S, lengths, starts, window, sinks):
    n = lengths.clamp(0, S)
    p = ((starts if starts is not None else n - L)[:, None] + torch.arange(L, device=lengths.device))[..., None]
    j = torch.arange(S, device=lengths.device)
    see = (j <= p) & (j < n[:, None, None])
    if window:
        see &= (j > p - window) | (j < sinks)
    inside = p < n[:, None, None]
    return see & inside, inside


def _reference(q, k, v, lengths, starts, window, sinks, scale, prefix=None):
    """``(o, tolerance)`` [B, L, H, D] in fp64."""
    B, L, H, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    see, inside = _visible(L, S, lengths.long(), None if starts is None else starts.long(), window, sinks)
    if prefix is not None:
        k, v = (torch.cat((p[None].expand(B, -1, -1, -1), t), 2) for p, t in zip(prefix, (k, v)))
        see = torch.cat((inside.expand(B, L, prefix[0].shape[1]), see), -1)
    qd = q.double().view(B, L, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4)
    kd, vd = k.double()[:, :, None], v.double()[:, :, None]
    s = (qd @ kd.transpose(-1, -2)) * scale
    size = ((qd.abs() @ kd.abs().transpose(-1, -2)) * scale).masked_fill(~see[:, None, None], 0).amax(-1, keepdim=True) if see.shape[-1] else s.sum(-1, keepdim=True)
    s = s.masked_fill(~see[:, None, None], -math.inf)
    w = torch.softmax(s, -1).nan_to_num(0.0) if see.shape[-1] else s
    o, mass = w @ vd, w @ vd.abs()
    half, n = torch.finfo(q.dtype).eps / 2, see.shape[-1]
    tol = half * o.abs() + mass * (half * 1.01 + 4 * 2.0 ** -20 * size * math.log2(math.e) + (n / 16 + 16) * 2.0 ** -22) + 2.0 ** -25
    back = lambda t: t.permute(0, 3, 1, 2, 4).reshape(B, L, H, D)  # noqa: E731
    return back(o), back(tol)


def _close(got, o, tol):
    bad = ~((got.double() - o).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} values off, by up to {float(((got.double() - o).abs() / tol).nan_to_num(9e9).max()):.2f} of the tolerance"


def _inputs(B, L, H, Hkv, S, D, dtype, seed=0, peak=1.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    return (r(B, L, H, D) * peak).to(dtype), r(B, Hkv, S, D).to(dtype), r(B, Hkv, S, D).to(dtype)


def _lengths(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _all(S, B):
    return torch.full((B,), S, dtype=torch.int32, device="cuda")


TOKEN = [(1, 1, 1, 1, 64), (1, 32, 8, 2048, 128), (3, 8, 8, 77, 64), (2, 16, 1, 300, 128), (2, 40, 2, 129, 64), (4, 5, 5, 1000, 80), (1, 14, 2, 513, 96),
         (2, 7, 1, 4099, 112), (1, 4, 2, 65, 8), (5, 6, 3, 33, 72), (1, 8, 1, 20011, 128), (1, 3, 1, 16, 32)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 0), (64, 4), (1, 0), (17, 70), (5000, 3)])
@pytest.mark.parametrize("B,H,Hkv,S,D", TOKEN)
def test_one_token(B, H, Hkv, S, D, window, sinks, dtype):
    import hbq_b200 as h
    q, k, v = _inputs(B, 1, H, Hkv, S, D, dtype, S + D)
    lengths = _lengths([max(1, S - 37 * b) for b in range(B)])
    for b in range(B):                                           # nothing behind a sequence's end is looked at
        k[b, :, lengths[b]:] = float("nan")
        v[b, :, lengths[b]:] = float("nan")
    got = h.window_attention(q, k, v, window=window, sinks=sinks, lengths=lengths)
    _close(got, *_reference(q, k.nan_to_num(0), v.nan_to_num(0), lengths, None, window, sinks, 1 / math.sqrt(D)))


PROMPT = [(1, 2, 1, 1, 2, 64), (1, 16, 4, 1, 16, 128), (2, 100, 4, 2, 100, 64), (1, 257, 8, 2, 257, 128), (3, 65, 6, 2, 130, 80), (1, 300, 7, 1, 1000, 128),
          (2, 33, 40, 2, 33, 64), (1, 1000, 2, 2, 1000, 96), (1, 513, 5, 1, 2000, 64), (2, 3, 32, 8, 700, 128), (1, 64, 3, 3, 64, 8), (1, 129, 16, 16, 129, 112),
          (1, 8, 20, 1, 5000, 128), (4, 90, 40, 2, 90, 64), (2, 150, 5, 1, 180, 72), (20, 16, 4, 1, 16, 128), (9, 33, 24, 3, 40, 128), (3, 100, 6, 6, 260, 8)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 0), (129, 4), (1, 1), (20, 200), (1, 0)])
@pytest.mark.parametrize("B,L,H,Hkv,S,D", PROMPT)
def test_prompts(B, L, H, Hkv, S, D, window, sinks, dtype):
    import hbq_b200 as h
    q, k, v = _inputs(B, L, H, Hkv, S, D, dtype, S + L)
    got = h.window_attention(q, k, v, window=window, sinks=sinks)
    assert got.shape == (B, L, H, D) and got.is_contiguous()
    _close(got, *_reference(q, k, v, _all(S, B), None, window, sinks, 1 / math.sqrt(D)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 3)])
@pytest.mark.parametrize("L,S", [(150, 150), (1, 150), (40, 300), (9, 150)])
def test_lengths_and_starts(L, S, window, sinks, dtype):
    """Padded prompts, sequences shorter than their rows (rows that see nothing), empty ones, values outside the cache."""
    import hbq_b200 as h
    values = [S, 0, 1, S // 2, -5, S + 1000, 5, 129]
    B = len(values)
    q, k, v = _inputs(B, L, 8, 2, S, 64, dtype, L)
    lengths = _lengths(values)
    kk, vv = k.clone(), v.clone()
    for b, n in enumerate(values):
        kk[b, :, min(max(n, 0), S):] = float("nan")
        vv[b, :, min(max(n, 0), S):] = float("inf")
    for starts in (None, _lengths([0] * B), _lengths([S - L, 0, -3, S // 2 - 4, 7, 2 ** 31 - 1, -2 ** 31, 128])):
        got = h.window_attention(q, kk, vv, window=window, sinks=sinks, lengths=lengths, starts=starts)
        o, tol = _reference(q, k, v, lengths, starts, window, sinks, 1 / 8)
        _close(got, o, tol)
        assert not bool(got[1].any()) and not bool(got[4].any())
        if starts is not None and starts[5] > 0:
            assert not bool(got[5].any()) and not bool(got[6].any())
    big = torch.tensor([n * (1 << 33) if n < 0 else n for n in values], device="cuda")
    assert torch.equal(h.window_attention(q, kk, vv, lengths=big), h.window_attention(q, kk, vv, lengths=lengths))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("L,S,window,sinks", [(40, 200, 0, 0), (300, 300, 0, 0), (300, 700, 90, 2), (1, 300, 30, 2), (2, 5, 0, 0), (149, 260, 0, 0), (149, 400, 60, 2), (200, 200, 5, 130)])
def test_what_a_mask_hides_does_not_reach_a_row(L, S, window, sinks, dtype):
    import hbq_b200 as h
    q, k, v = _inputs(1, L, 4, 2, S, 64, dtype, 5)
    see, _ = _visible(L, S, _all(S, 1), None, window, sinks)
    want, tol = _reference(q, k, v, _all(S, 1), None, window, sinks, 1 / 8)
    for j, value in ((S - 1, float("nan")), (S - L // 2 - 1, float("inf")), (max(0, S - L - 3), float("-inf")), (sinks, float("nan"))):
        kk, vv = k.clone(), v.clone()
        vv[:, :, j] = value
        vv[:, 1, j, 3:] = v[:, 1, j, 3:]
        got = h.window_attention(q, k, vv, window=window, sinks=sinks)[0]
        sees = see[0, :, j]
        _close(got[~sees], want[0][~sees], tol[0][~sees])
        assert not bool(torch.isfinite(got[sees][:, :2]).any()) and not bool(torch.isfinite(got[sees][:, 2:, :3]).any())
        _close(got[:, 2:, 3:], want[0][:, 2:, 3:], tol[0][:, 2:, 3:])
        kk[:, :, j] = float("nan")
        got = h.window_attention(q, kk, v, window=window, sinks=sinks)[0]
        _close(got[~sees], want[0][~sees], tol[0][~sees])
        assert bool(torch.isnan(got[sees]).all())


@pytest.mark.parametrize("peak,scale", [(0.0, None), (30.0, None), (1.0, 3.0), (1.0, 1e-4), (200.0, 1.0)])
@pytest.mark.parametrize("L", [1, 70, 90])
def test_flat_and_peaked_weights(peak, scale, L):
    import hbq_b200 as h
    for dtype in (torch.float16, torch.bfloat16):
        q, k, v = _inputs(2, L, 8, 2, 600, 128, dtype, 9, peak)
        got = h.window_attention(q, k, v, window=300, sinks=2, scale=scale)
        _close(got, *_reference(q, k, v, _all(600, 2), None, 300, 2, scale or 1 / math.sqrt(128)))


@pytest.mark.parametrize("L", [1, 50, 90])
def test_layouts(L):
    import hbq_b200 as h
    q, k, v = _inputs(2, L, 8, 2, 90, 64, torch.float16, 3)
    want = h.window_attention(q, k, v, window=30, sinks=1)
    token = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    assert torch.equal(h.window_attention(token(q), token(k), token(v), window=30, sinks=1), want)
    qkv = torch.cat((q.reshape(2, L, -1), torch.zeros((2, L, 256), device="cuda").half()), -1)
    assert torch.equal(h.window_attention(qkv[..., :512].view(2, L, 8, 64), k, v, window=30, sinks=1), want)
    cache = torch.full((2, 2, 200, 64), float("nan"), device="cuda").half()                        # a longer cache, cut and counted
    cache[:, :, :90] = k
    assert torch.equal(h.window_attention(q, cache[:, :, :90], v, window=30, sinks=1), want)
    vc = torch.full_like(cache, float("nan"))
    vc[:, :, :90] = v
    _close(h.window_attention(q, cache, vc, window=30, sinks=1, lengths=_all(90, 2)), *_reference(q, k, v, _all(90, 2), None, 30, 1, 1 / 8))
    odd = torch.empty(k.numel() + 3, device="cuda", dtype=k.dtype)[3:].view(k.shape).copy_(k)      # not 16-byte aligned: copied
    assert torch.equal(h.window_attention(q, odd, v, window=30, sinks=1), want)
    wide = torch.zeros((2, 2, 90, 67), device="cuda", dtype=k.dtype)
    wide[..., :64] = v
    assert torch.equal(h.window_attention(q, k, wide[..., :64], window=30, sinks=1), want)
    one = k[:, :1].expand(2, 2, 90, 64)                                                            # broadcast heads and sequences
    assert torch.equal(h.window_attention(q, one, v, window=30, sinks=1), h.window_attention(q, one.contiguous(), v, window=30, sinks=1))
    one = k[:1].expand(2, 2, 90, 64)
    assert torch.equal(h.window_attention(q, one, one, window=30, sinks=1), h.window_attention(q, one.contiguous(), one.contiguous(), window=30, sinks=1))
    out = torch.full((2, L + 2, 8, 64), 5.0, device="cuda").half()
    o = h.window_attention(q, k, v, window=30, sinks=1, out=out[:, 1:-1])
    assert o.data_ptr() == out[:, 1:-1].data_ptr() and torch.equal(out[:, 1:-1], want) and bool((out[:, 0] == 5).all()) and bool((out[:, -1] == 5).all())
    byhead = torch.empty((2, 8, L, 64), device="cuda").half()
    h.window_attention(q, k, v, window=30, sinks=1, out=byhead.transpose(1, 2))
    assert torch.equal(byhead.transpose(1, 2), want)


PREFIX = [(2, 1, 4, 2, 100, 7, 64), (8, 1, 32, 8, 1000, 50, 128), (5, 1, 3, 3, 129, 1, 80), (64, 1, 8, 2, 700, 33, 128), (3, 17, 8, 2, 300, 40, 64), (2, 130, 4, 1, 257, 130, 128),
          (1, 1, 1, 1, 1, 1, 8), (1, 300, 4, 4, 64, 300, 96), (33, 1, 20, 1, 4000, 5, 112), (70, 2, 6, 2, 900, 20, 72), (64, 1, 8, 2, 3000, 33, 128),
          (8, 1, 32, 8, 5000, 50, 128), (3, 17, 8, 2, 3000, 40, 64), (5, 1, 3, 3, 20000, 1, 80), (2, 90, 24, 3, 600, 95, 96)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("B,L,H,Hkv,P,S,D", PREFIX)
def test_shared_prefix(B, L, H, Hkv, P, S, D, ragged, dtype):
    import hbq_b200 as h
    q, k, v = _inputs(B, L, H, Hkv, S, D, dtype, P)
    pk, pv = (torch.randn((Hkv, P, D), device="cuda").to(dtype) for _ in range(2))
    lengths = _lengths([S - (b * 5) % (S + 1) for b in range(B)]) if ragged else None     # empty own caches among them
    starts = _lengths([0] * B) if ragged and L > 1 else None
    o, tol = _reference(q, k, v, _all(S, B) if lengths is None else lengths, starts, 0, 0, 1 / math.sqrt(D), (pk, pv))
    if ragged:
        for b in range(B):
            k[b, :, lengths[b]:] = float("inf")
            v[b, :, lengths[b]:] = float("nan")
    _close(h.shared_prefix_attention(q, pk, pv, k, v, lengths=lengths, starts=starts), o, tol)


def test_shared_prefix_edges():
    import hbq_b200 as h
    q, k, v = _inputs(3, 1, 8, 2, 40, 64, torch.float16, 1)
    pk, pv = (torch.randn((2, 90, 64), device="cuda").half() for _ in range(2))
    none = torch.empty((3, 2, 0, 64), device="cuda").half()
    o, tol = _reference(q, none, none, _all(0, 3), None, 0, 0, 1 / 8, (pk, pv))
    _, inside = _visible(1, 0, _all(0, 3).long(), None, 0, 0)
    assert bool(inside.all())                                           # position -1 of an empty cache is not behind its end
    _close(h.shared_prefix_attention(q, pk, pv, none, none), o, tol)     # no own keys at all
    _close(h.shared_prefix_attention(q, pk[:, :0], pv[:, :0], k, v), *_reference(q, k, v, _all(40, 3), None, 0, 0, 1 / 8))
    assert not bool(h.shared_prefix_attention(q, pk[:, :0], pv[:, :0], none, none).any())
    token = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    assert torch.equal(h.shared_prefix_attention(q, token(pk), token(pv), k, v), h.shared_prefix_attention(q, pk, pv, k, v))
    # a prefix given as every sequence's first keys is the same attention
    both = [torch.cat((p[None].expand(3, -1, -1, -1), t), 2) for p, t in ((pk, k), (pv, v))]
    _close(h.window_attention(q, *both), *_reference(q, k, v, _all(40, 3), None, 0, 0, 1 / 8, (pk, pv)))
    q2, k2, v2 = _inputs(3, 50, 8, 2, 50, 64, torch.float16, 1)
    o, tol = _reference(q2, k2, v2, _lengths([50, 20, 0]), _lengths([0, 0, 0]), 0, 0, 1 / 8, (pk, pv))
    got = h.shared_prefix_attention(q2, pk, pv, k2, v2, lengths=_lengths([50, 20, 0]), starts=_lengths([0, 0, 0]))
    _close(got, o, tol)
    assert not bool(got[1, 20:].any()) and not bool(got[2].any())


@pytest.mark.parametrize("B,L,H,Hkv", [(8, 40, 8, 2), (200, 1, 8, 2), (1, 200, 6, 2), (3, 70, 6, 6), (300, 2, 3, 1)])
@pytest.mark.parametrize("P", [100, 1000])
def test_a_prefix_alone(B, L, H, Hkv, P):
    """No keys of the sequences' own: the prefix' kernel writes the output, in any layout."""
    import hbq_b200 as h
    q, none, _ = _inputs(B, L, H, Hkv, 0, 64, torch.float16, P)
    pk, pv = (torch.randn((Hkv, P, 64), device="cuda").half() for _ in range(2))
    lengths, starts = _all(0, B), _lengths([-L if b % 3 else -L // 2 - 1 for b in range(B)])      # rows from position 0 on are padding
    for st in (None, starts):
        o, tol = _reference(q, none, none, lengths, st, 0, 0, 1 / 8, (pk, pv))
        _close(h.shared_prefix_attention(q, pk, pv, none, none, starts=st), o, tol)
        wide = torch.full((B, L + 1, H + 1, 72), 3.0, device="cuda").half()
        h.shared_prefix_attention(q, pk, pv, none, none, starts=st, out=wide[:, 1:, :-1, :64])
        _close(wide[:, 1:, :-1, :64], o, tol)
        assert bool((wide[:, 0] == 3).all()) and bool((wide[:, :, -1] == 3).all()) and bool((wide[..., 64:] == 3).all())
        byhead = torch.empty((H, L, B, 64), device="cuda").half()
        h.shared_prefix_attention(q, pk, pv, none, none, starts=st, out=byhead.permute(2, 1, 0, 3))
        _close(byhead.permute(2, 1, 0, 3), o, tol)


def test_queries_beyond_32_bit_offsets():
    """A prompt whose queries, keys turned in place and outputs pass 2^31 elements, against single rows of it."""
    import hbq_b200 as h
    L, H, Hkv, D = 540001, 32, 8, 128
    if torch.cuda.get_device_properties(0).total_memory < 60e9:
        pytest.skip("needs 20 GB")
    g = torch.Generator(device="cuda").manual_seed(2)
    q = torch.empty((1, L, H, D), device="cuda", dtype=torch.float16)
    for part in q.split(60000, 1):
        part.copy_(torch.randn(part.shape, device="cuda", generator=g, dtype=torch.float16))
    k, v = (torch.randn((1, Hkv, L, D), device="cuda", generator=g, dtype=torch.float16) for _ in range(2))
    got = h.window_attention(q, k, v, window=200, sinks=3)
    f, _ = h.rope_frequencies(D, 500000.0, device="cuda")
    pos = torch.arange(L, device="cuda")
    some = [0, 1, 1023, 199999, 524287, 524288, 530000, L - 1]
    for p in some:
        keys = list(range(min(3, max(0, p - 199)))) + list(range(max(0, p - 199), p + 1))
        o, tol = _reference(q[:, p:p + 1], k[:, :, keys], v[:, :, keys], _all(len(keys), 1), None, 0, 0, 1 / math.sqrt(D))
        _close(got[:, p:p + 1], o, tol)
    rows = q[:, some].clone()
    h.rope_rotate(q, f, pos, out=q)
    assert torch.equal(q[:, some], h.rope_rotate(rows, f, pos[some]))


def test_of_nothing():
    import hbq_b200 as h
    z = lambda *s: torch.empty(s, device="cuda").half()  # noqa: E731
    assert h.window_attention(z(0, 3, 4, 64), z(0, 2, 5, 64), z(0, 2, 5, 64)).shape == (0, 3, 4, 64)
    assert h.window_attention(z(2, 0, 4, 64), z(2, 2, 5, 64), z(2, 2, 5, 64)).shape == (2, 0, 4, 64)
    for L in (1, 60, 200):
        got = h.window_attention(torch.ones((2, L, 4, 64), device="cuda").half(), z(2, 2, 0, 64), z(2, 2, 0, 64))
        assert got.shape == (2, L, 4, 64) and not bool(got.any())


@pytest.mark.parametrize("H,Hkv", [(64, 1), (96, 2), (40, 1)])
def test_many_heads_of_one_key_head(H, Hkv):
    import hbq_b200 as h
    for L, S in ((1, 700), (1, 40), (9, 300), (60, 300), (150, 150)):
        q, k, v = _inputs(2, L, H, Hkv, S, 64, torch.bfloat16, 8)
        lengths = _lengths([S, S - 7])
        got = h.window_attention(q, k, v, window=200, sinks=2, lengths=lengths)
        _close(got, *_reference(q, k, v, lengths, None, 200, 2, 1 / 8))
        pk, pv = (torch.randn((Hkv, 150, 64), device="cuda").bfloat16() for _ in range(2))
        got = h.shared_prefix_attention(q, pk, pv, k, v, lengths=lengths)
        _close(got, *_reference(q, k, v, lengths, None, 0, 0, 1 / 8, (pk, pv)))


@pytest.mark.parametrize("B,L,H,Hkv", [(1, 3, 2, 2), (2, 4, 4, 4), (1, 15, 1, 1), (1, 17, 1, 1)])
def test_few_tokens_behind_a_prefix(B, L, H, Hkv):
    import hbq_b200 as h
    q, k, v = _inputs(B, L, H, Hkv, 30, 64, torch.float16, 8)
    pk, pv = (torch.randn((Hkv, 77, 64), device="cuda").half() for _ in range(2))
    for lengths, starts in ((None, None), (_lengths([25, 2][:B]), None), (_lengths([25, 2][:B]), _lengths([0, 1][:B]))):
        got = h.shared_prefix_attention(q, pk, pv, k, v, lengths=lengths, starts=starts)
        _close(got, *_reference(q, k, v, _all(30, B) if lengths is None else lengths, starts, 0, 0, 1 / 8, (pk, pv)))


@pytest.mark.parametrize("H", [4, 6])
@pytest.mark.parametrize("step", [1, 2, 4, 8])
def test_outputs_of_any_alignment(step, H):
    """Rows of the output that are not 16 bytes apart, and outputs that begin off a 16-byte boundary."""
    import hbq_b200 as h
    for L in (1, 40, 90):
        q, k, v = _inputs(2, L, H, 2, 90, 64, torch.float16, 3)
        want = h.window_attention(q, k, v)
        wide = torch.full((2, L, H, 64 + step), 9.0, device="cuda").half()
        h.window_attention(q, k, v, out=wide[..., :64])
        assert torch.equal(wide[..., :64], want) and bool((wide[..., 64:] == 9).all())
        wide.fill_(9.0)
        h.window_attention(q, k, v, out=wide[..., step:])
        assert torch.equal(wide[..., step:], want) and bool((wide[..., :step] == 9).all())


def test_windows_and_first_tokens_beyond_the_cache():
    """The same keys by another division of the work: each result is off by half a step (2^-12) of itself and of its weighted sum
    of |v|, which is below 3 here -- 2 * 2^-12 * 3 < 2^-9 between them."""
    import hbq_b200 as h
    for L in (1, 50, 90):
        q, k, v = _inputs(2, L, 8, 2, 90, 64, torch.float16, 3)
        want = h.window_attention(q, k, v)
        for window, sinks in ((90, 0), (2 ** 40, 5), (2 ** 62, 2 ** 62), (1, 90), (1, 2 ** 62)):
            _close(h.window_attention(q, k, v, window=window, sinks=sinks), want.double(), 2.0 ** -10 * want.double().abs() + 2.0 ** -9)


@pytest.mark.parametrize("L,S,P", [(1, 5000, 3000), (90, 5000, 3000), (1, 900, 300), (3, 100, 50)])
def test_streams_graphs_and_two_calls_at_once(L, S, P):
    import hbq_b200 as h
    q, k, v = _inputs(2, L, 8, 2, S, 128, torch.bfloat16, 3)
    pk, pv = (torch.randn((2, P, 128), device="cuda").bfloat16() for _ in range(2))
    lengths = _lengths([S, S // 4])
    call = lambda: (h.window_attention(q, k, v, window=S * 4 // 5, sinks=4, lengths=lengths), h.shared_prefix_attention(q, pk, pv, k, v, lengths=lengths))  # noqa: E731
    want = call()
    assert all(torch.equal(a, b) for a, b in zip(call(), want))           # the same bits every time
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams * 3:
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for a, b in zip(pair, want))
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(call())
    k.copy_(torch.randn_like(k)); lengths.copy_(_lengths([S * 6 // 7, S]))
    want = call()
    torch.cuda.synchronize()
    for s, g in zip(streams, graphs):                                      # two graphs in flight at once
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in outs for a, b in zip(pair, want))
    with pytest.raises(NotImplementedError):
        h.window_attention(q.clone().requires_grad_(), k, v)
    with pytest.raises(ValueError):
        h.window_attention(q, k, v, lengths=lengths.cpu())


def test_a_cache_beyond_32_bit_offsets():
    """Keys at element offsets past 2^32 (and byte offsets past 2^33) of one cache."""
    import hbq_b200 as h
    B, Hkv, S, D = 3, 1, 1 << 24, 128
    if torch.cuda.get_device_properties(0).total_memory < 40e9:
        pytest.skip("needs 13 GB for the cache")
    cache = torch.zeros((B, Hkv, S, D), device="cuda", dtype=torch.float16)
    g = torch.Generator(device="cuda").manual_seed(1)
    n = S - 3
    for L in (1, 20, 120):
        q = torch.randn((B, L, 4, D), device="cuda", generator=g).half()
        part = torch.randn((B, Hkv, 433, D), device="cuda", generator=g).half()
        cache[:, :, n - 433:n] = part
        got = h.window_attention(q, cache, cache, window=300, lengths=_all(n, B))
        _close(got, *_reference(q, part, part, _all(433, B), None, 300, 0, 1 / math.sqrt(D)))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_projection_to_output_with_a_growing_cache(dtype):
    """The operators as a decoder uses them: norm and rotation of a packed projection written into the cache, a prompt, then
    token after token with a window and first tokens; and the same tokens behind a shared prefix."""
    import hbq_b200 as h
    B, T, H, Hkv, D, window, sinks = 2, 45, 8, 2, 64, 20, 2
    g = torch.Generator(device="cuda").manual_seed(7)
    qkv = torch.randn((B, T, (H + 2 * Hkv) * D), device="cuda", generator=g).to(dtype)
    wq, wk = (1 + 0.1 * torch.randn(D, device="cuda", generator=g).to(dtype) for _ in range(2))
    f, m = h.rope_frequencies(D // 2, 10000.0, {"type": "linear", "factor": 2.0}, device="cuda")
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split((H * D, Hkv * D, Hkv * D), -1))
    pos = torch.arange(T, device="cuda")
    qr, kr = h.qk_norm_rope(q, k, wq, wk, 1e-5, f, pos, factor=m)
    kc, vc = (torch.full((B, Hkv, 64, D), float("nan"), device="cuda", dtype=dtype) for _ in range(2))
    vc[:, :, :T] = v.transpose(1, 2)
    whole, tol = _reference(qr, kr.transpose(1, 2), v.transpose(1, 2), _all(T, B), None, window, sinks, 1 / 8)
    full, ftol = _reference(qr, kr.transpose(1, 2), v.transpose(1, 2), _all(T, B), None, 0, 0, 1 / 8)
    n = 30
    for t0, t1 in [(0, n)] + [(t, t + 1) for t in range(n, T)]:
        qs = torch.empty((B, t1 - t0, H, D), device="cuda", dtype=dtype)
        h.qk_norm_rope(q[:, t0:t1], k[:, t0:t1], wq, wk, 1e-5, f, pos[t0:t1], factor=m, out=(qs, kc[:, :, t0:t1].transpose(1, 2)))
        assert torch.equal(qs, qr[:, t0:t1]) and torch.equal(kc[:, :, t0:t1].transpose(1, 2), kr[:, t0:t1])
        got = h.window_attention(qs, kc, vc, window=window, sinks=sinks, lengths=_all(t1, B))
        _close(got, whole[:, t0:t1], tol[:, t0:t1])
        if t0 >= n:                                                       # sequence 0's first tokens as the prefix of a batch of one
            got = h.shared_prefix_attention(qs[:1], kc[0, :, :n], vc[0, :, :n], kc[:1, :, n:], vc[:1, :, n:], lengths=_all(t1 - n, 1))
            _close(got, full[:1, t0:t1], ftol[:1, t0:t1])


@pytest.mark.parametrize("L", [1, 40])
def test_a_chain_that_changes_its_inputs_in_place(L):
    """Calls one after the other without a synchronisation, each on inputs that were written just before: kernels that start under
    the one before them see all of it and leave what it still reads."""
    import hbq_b200 as h
    D = 128
    for wait in (True, False):
        g = torch.Generator(device="cuda").manual_seed(4)
        q, k, v = _inputs(8, L, 8, 2, 600, D, torch.float16, 3)
        pk, pv = (torch.randn((2, 500, D), device="cuda", generator=g).half() for _ in range(2))
        f, _ = h.rope_frequencies(D, 10000.0, device="cuda")
        w, lengths, pos = torch.ones(D, device="cuda").half(), _all(600, 8), torch.arange(L, device="cuda")
        steps = []
        for n in range(6):
            o = h.shared_prefix_attention(q, pk, pv, k, v, lengths=lengths)
            q2, k2 = h.qk_norm_rope(o, k[:, :, :L].transpose(1, 2), w, w, 1e-5, f, pos)
            k[:, :, 100:100 + L] = k2.transpose(1, 2)
            v[:, :, 7 + n] = o[:, 0, :2]
            lengths.sub_(17)
            h.rope_rotate(q2, f, pos, out=q)
            pv[:, :L] = o[0].transpose(0, 1)[:2]
            steps += [o, h.window_attention(q, k, v, window=150 + n, sinks=9, lengths=lengths), q.clone()]
            if wait:
                torch.cuda.synchronize()
        if wait:
            want = steps
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(steps, want))


def test_no_wait_ran_out():
    import hbq_b200 as h
    torch.cuda.synchronize()
    assert h.gemm_status() == 0
