"""GPU: rotary positions and head norms where no result may be a NaN, and calls of more head groups than a grid's second axis holds.

Tolerance as for the other rotary tests: one rounding to the tensor's type (half a step, finfo.eps / 2, of the value), the 32-bit
arithmetic before it (below 2^-17 of the pair's magnitudes) and half of fp16's smallest step.  A NaN meets no tolerance."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def _turned(x, f, pos, interleaved, factor):
    """``(y, |u| + |w| of each value's pair)`` of x [B, T, H, D] in fp64."""
    r = 2 * f.numel()
    z = torch.stack((x[..., 0:r:2], x[..., 1:r:2]), -1) if interleaved else torch.stack((x[..., :r // 2], x[..., r // 2:r]), -1)
    a = pos.double()[..., None, None] * f
    y = torch.view_as_real(torch.view_as_complex(z.contiguous()) * torch.polar(torch.full_like(a, factor), a))
    size = z.abs().sum(-1, keepdim=True).expand(z.shape) * abs(factor)
    flat = lambda t: t.flatten(-2) if interleaved else torch.cat((t[..., 0], t[..., 1]), -1)  # noqa: E731
    return torch.cat((flat(y), x[..., r:]), -1), torch.cat((flat(size), x[..., r:].abs()), -1)


def _close(got, y, size):
    tol = y.abs() * (torch.finfo(got.dtype).eps / 2) * (1 + 2.0 ** -10) + size * 2.0 ** -17 + 2.0 ** -25
    good = (got.double() - y).abs() <= tol
    assert bool(good.all()), f"{int((~good).sum())} of {good.numel()} values off, {int(got.isnan().sum())} of them NaN"


def _normed(x, w, eps):
    x = x.double()
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()


SHAPES = [(1, 1, 1, 64, 64), (2, 37, 3, 64, 32), (1, 5, 32, 128, 128), (3, 19, 5, 80, 80), (2, 9, 7, 80, 20), (1, 33, 2, 96, 48), (2, 3, 4, 112, 28),
          (1, 17, 3, 256, 256), (1, 4, 2, 16, 16), (1, 6, 3, 10, 6), (2, 5, 1, 2, 2), (1, 3, 2, 512, 128), (1, 7, 3, 72, 72), (1, 2500, 5, 128, 64),
          (2, 1301, 9, 64, 64), (1, 700, 40, 48, 16), (2, 3, 5, 240, 224)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("B,T,heads,D,rot", SHAPES)
def test_every_value(B, T, heads, D, rot, interleaved, dtype):
    import hbq_b200 as H
    g = torch.Generator(device="cuda").manual_seed(T + D)
    x, y = (torch.randn((B, T, n, D), device="cuda", generator=g).to(dtype) for n in (heads, 1 + heads // 3))
    x[-1, -1, -1] = 0
    wx, wy = (1 + 0.3 * torch.randn(D, device="cuda", generator=g).to(dtype) for _ in range(2))
    f, _ = H.rope_frequencies(rot, 10000.0, device="cuda")
    pos = torch.randint(-50, 100000, (B, T), device="cuda", generator=g)
    _close(H.rope_rotate(x, f, pos, interleaved=interleaved, factor=1.25), *_turned(x.double(), f, pos, interleaved, 1.25))
    for o, t, w in zip(H.qk_norm_rope(x, y, wx, wy, 1e-5, f, pos, interleaved=interleaved, factor=0.75), (x, y), (wx, wy)):
        _close(o, *_turned(_normed(t, w, 1e-5), f, pos, interleaved, 0.75))


@pytest.mark.parametrize("T,heads,more", [(1, 524289, 3), (2, 3, 524300), (1, 530001, 500001)])
def test_more_groups_than_a_grids_second_axis(T, heads, more):
    """Heads of 256 are two to a warp and eight to a block: above 65535 * 8 heads a block takes several rounds of them."""
    import hbq_b200 as H
    g = torch.Generator(device="cuda").manual_seed(heads)
    q, k = (torch.randn((1, T, n, 256), device="cuda", generator=g, dtype=torch.float16) for n in (heads, more))
    w = 1 + 0.1 * torch.randn(256, device="cuda", generator=g).half()
    f, _ = H.rope_frequencies(256, 10000.0, device="cuda")
    pos = torch.tensor([[3, 70000][:T]], device="cuda")

    def every(got, of):                                              # (in pieces: the reference takes 32 bytes a value)
        for x, y in zip(got.split(60000, 2), of.split(60000, 2)):
            yield x, y
    for t in (q, k):
        for o, x in every(H.rope_rotate(t, f, pos), t):
            _close(o, *_turned(x.double(), f, pos, False, 1.0))
    for out, t in zip(H.qk_norm_rope(q, k, w, w, 1e-5, f, pos), (q, k)):
        for o, x in every(out, t):
            _close(o, *_turned(_normed(x, w, 1e-5), f, pos, False, 1.0))
