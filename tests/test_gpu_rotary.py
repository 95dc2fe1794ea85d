"""GPU: rotary positions and head norms against the formulas in 64 bits.

Tolerance: one rounding to the tensor's type, at most half a step (finfo.eps / 2) of the value, and the 32-bit arithmetic before
it: a pair's two products and sum, the cosine and sine (a few units of 2^-24 each of the pair's magnitudes) and, with the norm,
a sum of up to 256 squares and its root, all below 2^-17 of the magnitudes; 2^-25 is half the smallest fp16 step."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _turned(x, f, pos, interleaved, factor):
    """``(y, |u| + |w| of each value's pair)`` of x [B, T, H, D] in fp64."""
    r = 2 * f.numel()
    a = pos.double().expand(x.shape[0], x.shape[1])[..., None, None] * f
    c, s = a.cos() * factor, a.sin() * factor
    u, w = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    parts, size = (u * c - w * s, w * c + u * s), (u.abs() + w.abs()) * abs(factor)
    if interleaved:
        y, z = torch.stack(parts, -1).flatten(-2), torch.stack((size, size), -1).flatten(-2)
    else:
        y, z = torch.cat(parts, -1), torch.cat((size, size), -1)
    return torch.cat((y, x[..., r:]), -1), torch.cat((z, x[..., r:].abs()), -1)


def _close(got, y, size):
    eps = torch.finfo(got.dtype).eps
    bad = (got.double() - y).abs() > y.abs() * (eps / 2) * (1 + 2.0 ** -10) + size * 2.0 ** -17 + 2.0 ** -25
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} values off"


def _normed(x, w, eps):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


SHAPES = [(1, 1, 1, 64, 64), (2, 37, 3, 64, 32), (1, 5, 32, 128, 128), (3, 19, 5, 80, 80), (2, 9, 7, 80, 20), (1, 33, 2, 96, 48), (2, 3, 4, 112, 28),
          (1, 17, 3, 256, 256), (1, 4, 2, 16, 16), (1, 6, 3, 10, 6), (2, 5, 1, 2, 2), (1, 3, 2, 512, 128), (1, 7, 3, 72, 72), (1, 2500, 5, 128, 64),
          (2, 1301, 9, 64, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,heads,D,rot", SHAPES)
def test_rotation(B, T, heads, D, rot, interleaved, dtype):
    import hbq_b200 as H
    g = torch.Generator(device="cuda").manual_seed(T + D)
    x = torch.randn((B, T, heads, D), device="cuda", generator=g).to(dtype)
    f, _ = H.rope_frequencies(rot, 10000.0, device="cuda")
    pos = torch.randint(-50, 5000, (B, T), device="cuda", generator=g)
    _close(H.rope_rotate(x, f, pos, interleaved=interleaved, factor=1.25), *_turned(x.double(), f, pos, interleaved, 1.25))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,heads,D,rot", SHAPES)
def test_norm_and_rotation(B, T, heads, D, rot, interleaved, dtype):
    import hbq_b200 as H
    g = torch.Generator(device="cuda").manual_seed(T + D + 1)
    kv = max(1, heads // 3)
    x = torch.randn((B, T, (heads + 2 * kv) * D), device="cuda", generator=g).mul_(3).to(dtype)
    x[0, 0, :D] = 0                                                         # a head of zeros stays zeros
    q, k = x[..., :heads * D].view(B, T, heads, D), x[..., heads * D:(heads + kv) * D].view(B, T, kv, D)
    wq, wk = (1 + 0.3 * torch.randn(D, device="cuda", generator=g).to(dtype) for _ in range(2))
    f, m = H.rope_frequencies(rot, 10000.0, {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 512}, device="cuda")
    pos = torch.randint(0, 100000, (B, T), device="cuda", generator=g, dtype=torch.int32)
    got = H.qk_norm_rope(q, k, wq, wk, 1e-5, f, pos, interleaved=interleaved, factor=m)
    for o, t, w in zip(got, (q, k), (wq, wk)):
        assert o.shape == t.shape and o.is_contiguous()
        _close(o, *_turned(_normed(t, w, 1e-5), f, pos, interleaved, m))
    assert not bool(got[0][0, 0, 0].any())


@pytest.mark.parametrize("first", [2 ** 31 - 3, 2 ** 31 + 11, 2 ** 40, -2 ** 33])
def test_far_positions(first):
    import hbq_b200 as H
    x = torch.randn((6, 4, 64), device="cuda").half()
    # whole turns are exact in 64 bits only; one pair turns by 1 radian a token, whose product with 2^40 keeps 2^-12 in fp64's
    # 53 bits: the reference reduces the same product
    f = torch.tensor([1.0 / 1024, 0.5, 3.0], dtype=torch.float64, device="cuda")
    pos = first + torch.arange(6, device="cuda")
    turns = pos.double()[:, None] * (f * 0.15915494309189535)
    a = (turns - turns.round()) * (2 * torch.pi)
    u, w = x[..., :3].double(), x[..., 3:6].double()
    c, s = a.cos()[:, None], a.sin()[:, None]
    got = H.rope_rotate(x, f, pos)
    y = torch.cat((u * c - w * s, w * c + u * s, x[..., 6:].double()), -1)
    _close(got, y, torch.cat((u.abs() + w.abs(),) * 2 + (x[..., 6:].double().abs(),), -1))


def test_positions_and_layouts():
    import hbq_b200 as H
    g = torch.Generator(device="cuda").manual_seed(3)
    B, T, heads, D = 3, 11, 4, 64
    x = torch.randn((B, T, heads, D), device="cuda", generator=g).bfloat16()
    f, _ = H.rope_frequencies(64, 10000.0, device="cuda")
    one = torch.arange(5, 5 + T, device="cuda")
    want = H.rope_rotate(x, f, one.expand(B, T).contiguous())
    for pos in (one, one[None], one.to(torch.int32), one.expand(B, T), torch.stack((one, one), -1)[:, 0], one.expand(2, T).t().contiguous()[:, 1]):
        assert torch.equal(H.rope_rotate(x, f, pos), want)
    assert torch.equal(H.rope_rotate(x[1], f, one), want[1]) and torch.equal(H.rope_rotate(x[1], f, one[None]), want[1])
    assert torch.equal(H.rope_rotate(x.transpose(1, 2).contiguous().transpose(1, 2), f, one), want)
    assert torch.equal(H.rope_rotate(x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2), f, one), want)       # the last axis strided
    assert torch.equal(H.rope_rotate(x[:1].expand(B, T, heads, D), f, one), want[:1].expand(B, T, heads, D))
    shifted = torch.empty(x.numel() + 8, dtype=x.dtype, device="cuda")
    for k in (1, 4):                                                        # pointers that are not 16-byte aligned
        y = shifted[k:k + x.numel()].view(x.shape)
        y.copy_(x)
        assert torch.equal(H.rope_rotate(y, f, one), want)
    wide = torch.zeros((B, T, heads, D + 3), dtype=x.dtype, device="cuda")
    wide[..., :D] = x
    assert torch.equal(H.rope_rotate(wide[..., :D], f, one), want)


@pytest.mark.parametrize("D", [64, 72])
def test_out(D):
    import hbq_b200 as H
    g = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn((2, 9, 3, D), device="cuda", generator=g).half()
    f, _ = H.rope_frequencies(D, 10000.0, device="cuda")
    pos = torch.arange(9, device="cuda")
    want = H.rope_rotate(x, f, pos)
    cache = torch.full((2, 3, 40, D), 7.0, device="cuda", dtype=torch.float16)     # a slice of a cache stored by head
    o = H.rope_rotate(x, f, pos, out=cache[:, :, 20:29].transpose(1, 2))
    assert o.data_ptr() == cache[:, :, 20:29].data_ptr() and torch.equal(cache[:, :, 20:29].transpose(1, 2), want)
    assert bool((cache[:, :, :20] == 7).all()) and bool((cache[:, :, 29:] == 7).all())
    w = torch.rand(D, device="cuda", generator=g).half()
    wq, wk = H.qk_norm_rope(x, x[:, :, :2], w, w, 1e-6, f, pos)
    q = x.clone()
    H.qk_norm_rope(q, x[:, :, :2], w, w, 1e-6, f, pos, out=(q, cache[:, :2, :9].transpose(1, 2)))
    assert torch.equal(q, wq) and torch.equal(cache[:, :2, :9].transpose(1, 2), wk)
    assert H.rope_rotate(x, f, pos, out=x) is x and torch.equal(x, want)           # in place


def test_special_values_stay_in_their_head():
    import hbq_b200 as H
    x = torch.ones((4, 3, 64), device="cuda").half()
    x[1, 1, 5] = float("nan")
    x[2, 0, 40] = float("inf")
    f, _ = H.rope_frequencies(32, 10000.0, device="cuda")
    y = H.rope_rotate(x, f, torch.arange(4, device="cuda"))
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    want[1, 1, 5] = want[1, 1, 21] = want[2, 0, 40] = True
    assert torch.equal(bad, want) and y[2, 0, 40] == float("inf")
    q, k = H.qk_norm_rope(x, x[:, :1], x[0, 0], x[0, 0], 1e-5, f, torch.arange(4, device="cuda"))
    clean = torch.ones((4, 3), dtype=torch.bool, device="cuda")
    clean[1, 1] = clean[2, 0] = False
    assert bool(torch.isfinite(q[clean]).all()) and bool(torch.isnan(q[1, 1]).all()) and bool(torch.isfinite(k[[0, 1, 3]]).all())


def test_very_many_heads():
    """More groups of heads than a grid's second axis holds."""
    import hbq_b200 as H
    x = torch.randn((2, 600001, 16), device="cuda").half()
    f, _ = H.rope_frequencies(16, 10000.0, device="cuda")
    pos = torch.tensor([3, 70], device="cuda")
    _close(H.rope_rotate(x, f, pos)[None], *_turned(x.double()[None], f, pos[None], False, 1.0))


@pytest.mark.parametrize("shape", [(0, 5, 2, 64), (2, 0, 2, 64), (2, 5, 0, 64)])
def test_of_nothing(shape):
    import hbq_b200 as H
    f, _ = H.rope_frequencies(64, 10000.0, device="cuda")
    x, w = torch.empty(shape, device="cuda").half(), torch.ones(64, device="cuda").half()
    pos = torch.arange(shape[1], device="cuda")
    assert H.rope_rotate(x, f, pos).shape == shape
    q, k = H.qk_norm_rope(x, torch.ones((shape[0], shape[1], 1, 64), device="cuda").half(), w, w, 1e-5, f, pos)
    assert q.shape == shape and k.shape == (shape[0], shape[1], 1, 64)


def test_streams_graphs_and_refusals():
    import hbq_b200 as H
    f, _ = H.rope_frequencies(128, 10000.0, device="cuda")
    x = torch.randn((2, 7, 5, 128), device="cuda").half()
    w = torch.rand(128, device="cuda").half()
    pos = torch.arange(7, device="cuda")
    want = H.qk_norm_rope(x, x[:, :, :2], w, w, 1e-5, f, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = H.qk_norm_rope(x, x[:, :, :2], w, w, 1e-5, f, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = H.rope_rotate(H.qk_norm_rope(x, x[:, :, :2], w, w, 1e-5, f, pos)[0], f, pos)
    x.copy_(torch.randn_like(x)); pos.add_(100)
    graph.replay()
    assert torch.equal(y, H.rope_rotate(H.qk_norm_rope(x, x[:, :, :2], w, w, 1e-5, f, pos)[0], f, pos))
    with pytest.raises(NotImplementedError):
        H.rope_rotate(x.clone().requires_grad_(), f, pos)
    with torch.no_grad():
        H.rope_rotate(x.clone().requires_grad_(), f, pos)
    with pytest.raises(ValueError):
        H.rope_rotate(x, f.cpu(), pos)
    with pytest.raises(ValueError):
        H.rope_rotate(x, f, pos.cpu())
