"""GPU: infinities and NaNs among the values that a row of the attention sees.

The definition is a sum of positive weights times values: an infinity that a row sees, however small its weight, makes the
result that infinity; infinities of both signs, or a NaN, make it a NaN; every other value of the row is what it is without them."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def _sees(L, S, n, window, sinks, P):
    """[L, P + S]: what row i of a sequence of n keys, its last L tokens, sees."""
    p, j = (n - L + torch.arange(L, device="cuda"))[:, None], torch.arange(S, device="cuda")[None]
    see = (j <= p) & (j < n)
    if window:
        see &= (j > p - window) | (j < sinks)
    return torch.cat((torch.ones((L, P), dtype=torch.bool, device="cuda"), see), 1)


# (B, L, H, Hkv, S, P, window, sinks): every way a row's result comes about.  One block a row group, clusters, equal shares with
# slots, with and without a prefix in the list; row tiles with whole and masked key tiles, in one piece and in several; a prefix'
# kernel with either kernel beside it
CASES = [(1, 1, 8, 2, 40, 0, 0, 0), (1, 1, 8, 2, 1500, 0, 700, 3), (1, 1, 4, 1, 20011, 0, 0, 0), (3, 1, 40, 2, 3000, 0, 0, 0), (300, 1, 8, 2, 600, 0, 0, 0),
         (2, 1, 8, 2, 300, 500, 0, 0), (3, 2, 8, 2, 64, 30, 0, 0), (40, 1, 8, 2, 900, 3000, 0, 0), (2, 90, 8, 2, 90, 700, 0, 0), (8, 40, 8, 2, 0, 1000, 0, 0),
         (1, 300, 8, 2, 1000, 0, 0, 0), (40, 300, 8, 2, 700, 0, 0, 0), (1, 600, 6, 2, 900, 0, 300, 200), (2, 40, 8, 2, 5000, 0, 4000, 2)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("peak", [1.5, 40.0])                       # with 40 most weights are far below the types' smallest
@pytest.mark.parametrize("B,L,H,Hkv,S,P,window,sinks", CASES)
def test_infinities_that_a_row_sees(B, L, H, Hkv, S, P, window, sinks, peak, dtype):
    import hbq_b200 as h
    D = 64
    g = torch.Generator(device="cuda").manual_seed(S + L + P)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    q, k, v = (r(B, L, H, D) * peak).to(dtype), r(B, Hkv, S, D).to(dtype), r(B, Hkv, S, D).to(dtype)
    pk, pv = r(Hkv, P, D).to(dtype), r(Hkv, P, D).to(dtype)
    n = [S - (b * 11) % 30 if S > 60 else S for b in range(B)]
    lengths = torch.tensor(n, dtype=torch.int32, device="cuda")

    def call(v, pv):
        return (h.shared_prefix_attention(q, pk, pv, k, v, lengths=lengths) if P else
                h.window_attention(q, k, v, window=window, sinks=sinks, lengths=lengths))

    plain = call(v, pv)
    N = P + S
    places = sorted({x for x in (0, 1, P // 2, P - 1, P, P + 2, P + S // 3, N - 35, N - 1) if 0 <= x < N})
    for x in places:
        y = (x * 7 + 5) % N                                          # another key
        vv, pp = v.clone(), pv.clone()

        def put(at, d, value):
            if at < P:
                pp[:, at, d] = value
            else:
                vv[:, :, at - P, d] = value
        put(x, 0, INF); put(x, 13, -INF); put(x, 30, INF); put(x, 63, NAN)
        if y != x:
            put(y, 30, -INF); put(y, 0, INF); put(y, 40, -INF)
        got = call(vv, pp)
        for b in range(B):
            see = _sees(L, S, n[b], window, sinks, P)
            at_x, at_y = see[:, x], see[:, y] & (y != x)
            want = plain[b].clone()
            for d, cx, cy in ((0, INF, INF), (13, -INF, 0.0), (30, INF, -INF), (63, NAN, 0.0), (40, 0.0, -INF)):
                total = torch.where(at_x, cx, 0.0) + torch.where(at_y, cy, 0.0)      # [L]: 0, an infinity or a NaN
                odd = total != 0
                want[odd, :, d] = total[odd][:, None].to(dtype)
            assert torch.equal(got[b].isnan(), want.isnan()), (x, b)
            assert torch.equal(got[b].nan_to_num(0, INF, -INF), want.nan_to_num(0, INF, -INF)), (x, b)


def test_a_nan_among_queries_or_keys_stays_a_nan():
    import hbq_b200 as h
    for L, S in ((1, 700), (200, 700)):
        q, k, v = torch.randn((1, L, 8, 64), device="cuda").half(), torch.randn((1, 2, S, 64), device="cuda").half(), torch.randn((1, 2, S, 64), device="cuda").half()
        q[0, L // 2, 3, 9] = NAN
        v[0, :, 3, 5] = INF
        got = h.window_attention(q, k, v)
        assert bool(got[0, L // 2, 3].isnan().all()) and bool((got[0, :, :3, 5] == INF).all()) and int(got.isnan().sum()) == 64


@pytest.mark.parametrize("L,P", [(1, 2000), (90, 700), (40, 3000)])
def test_values_written_just_before(L, P):
    """Infinities that come and go between calls without a synchronisation, behind a prefix: the kernel that starts beside the
    prefix' one sees the values of its own call."""
    import hbq_b200 as h
    g = torch.Generator(device="cuda").manual_seed(L)
    r = lambda *s: torch.randn(s, device="cuda", generator=g).bfloat16()  # noqa: E731
    q, k, v, pk, pv = r(16, L, 8, 64), r(16, 2, 150, 64), r(16, 2, 150, 64), r(2, P, 64), r(2, P, 64)
    plain = h.shared_prefix_attention(q, pk, pv, k, v)
    torch.cuda.synchronize()
    got = []
    for n in range(8):
        kept = v[:, :, 5 + n, n].clone()
        v[:, :, 5 + n, n] = INF if n % 2 else -INF
        got.append(h.shared_prefix_attention(q, pk, pv, k, v))
        v[:, :, 5 + n, n] = kept
    torch.cuda.synchronize()
    for n, o in enumerate(got):
        odd = (150 - L + torch.arange(L, device="cuda")) >= 5 + n
        want = plain.clone()
        want[:, odd, :, n] = INF if n % 2 else -INF
        assert torch.equal(o, want)


@pytest.mark.parametrize("size", [3e38, 1e-33])
@pytest.mark.parametrize("B,L,H,Hkv,S,P,window,sinks", CASES)
def test_values_at_the_ends_of_bf16(B, L, H, Hkv, S, P, window, sinks, size):
    """Values up to bf16's largest, and values near its smallest: a mean of them stays in range, and so has the sum it is made of.
    Tolerance: half a step (2^-8) of the result for its rounding, the same of sum w |v| for the weights' rounding, and 2^-12 of that
    for the scores' 32-bit sums and the additions; half of bf16's smallest normal number where the results are that small."""
    import hbq_b200 as h
    D = 64
    g = torch.Generator(device="cuda").manual_seed(S + L)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    u = lambda *s: ((torch.rand(s, device="cuda", generator=g) * 0.9 + 0.1) * size * r(*s).sign()).bfloat16()  # noqa: E731
    q, k, v = r(B, L, H, D).bfloat16(), r(B, Hkv, S, D).bfloat16(), u(B, Hkv, S, D)
    pk, pv = r(Hkv, P, D).bfloat16(), u(Hkv, P, D)
    lengths = torch.full((B,), S, dtype=torch.int32, device="cuda")
    got = (h.shared_prefix_attention(q, pk, pv, k, v, lengths=lengths) if P else h.window_attention(q, k, v, window=window, sinks=sinks, lengths=lengths))
    see = _sees(L, S, S, window, sinks, P)
    for b in range(min(B, 3)):
        kk, vv = (torch.cat((a, t[b]), 1).double().repeat_interleave(H // Hkv, 0) for a, t in ((pk, k), (pv, v)))
        s = (q[b].double().transpose(0, 1) @ kk.transpose(-1, -2) / math.sqrt(D)).masked_fill(~see, -math.inf)
        w = torch.softmax(s, -1)
        o, mass = (w @ vv).transpose(0, 1), (w @ vv.abs()).transpose(0, 1)
        assert bool(((got[b].double() - o).abs() <= o.abs() * 2.0 ** -8 + mass * (2.0 ** -8 * 1.01 + 2.0 ** -12) + 2.0 ** -127).all())


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("B,L,S", [(1, 1, 131072), (300, 1, 4096), (1, 4096, 4096)])
def test_a_special_value_does_not_stop_the_batch(B, L, S, value):
    """One key's values of each head: the rows that see them take their keys once or twice more, not a lane's time for each key (which was
    some hundred times the call)."""
    import hbq_b200 as h
    g = torch.Generator(device="cuda").manual_seed(5)
    q = (torch.randn((B, L, 32, 128), device="cuda", generator=g) * 20).half()
    k, v = (torch.randn((B, 8, S, 128), device="cuda", generator=g).half() for _ in range(2))

    def time_of(n=5):
        h.window_attention(q, k, v)
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(n):
            h.window_attention(q, k, v)
        b.record()
        torch.cuda.synchronize()
        return a.elapsed_time(b)
    clean = time_of()
    v[:, :, S // 3] = value
    assert time_of() < 40 * clean
