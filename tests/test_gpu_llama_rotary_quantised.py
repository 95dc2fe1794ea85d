"""GPU: decoders with norms of their heads, other rotations than the tables' or a window, whose queries, caches and
probabilities are quantised: against the separate operations, and prefills in runs of queries against whole ones."""
import json
import math
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

KINDS = {
    "norms": dict(qk_norm=True),
    "norms, pairs": dict(qk_norm=True, rotary_dim=64, rope_interleaved=True),
    "scaled": dict(rope_scaling=dict(type="yarn", factor=4.0, original_max_position_embeddings=64)),
    "window": dict(window=150, sinks=3),
    "short window, norms": dict(window=40, qk_norm=True),
    "many first tokens": dict(window=100, sinks=200, rotary_dim=32),
}


def _model(kind, layers=1):
    import hbq_b200 as H
    with open(os.path.join(HERE, "golden", "ptq_configs.json")) as fh:
        cfg = json.load(fh)["hbq_a_kv.yaml"]["config"]
    a = H.LlamaArch(**{**dict(hidden=256, layers=layers, heads=4, kv_heads=2, head_dim=128, ffn=512, vocab=512, eps=1e-5, theta=10000.0), **KINDS[kind]})
    m = H.QLlamaModel(a, device="cuda")
    m.init_weights(5)
    if a.qk_norm:
        for layer in m.layers:
            for t in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                t.data.uniform_(0.5, 1.5, generator=torch.Generator(device="cuda").manual_seed(3))
    m.apply_ptq(H.PTQConfig(cfg))
    return m


def _attention(at, x, B, T, arch):
    """The block by separate operations: rotation in fp64 rounded to fp16, the quantizers as they are, softmax in fp64 of the
    product's fp16 scores."""
    import hbq_b200 as H
    D, G = arch.head_dim, arch.heads // arch.kv_heads
    q, k, v = (p(x).view(B, T, -1, D) for p in (at.q_proj, at.k_proj, at.v_proj))

    def turned(t, g):
        f, factor = H.rope_frequencies(arch.rotary_dim or D, arch.theta, arch.rope_scaling, device="cuda")
        t = t.double()
        if arch.qk_norm:
            t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + arch.eps) * g.double()
        a = torch.arange(T, device="cuda").double()[:, None, None] * f
        c, s, n = a.cos() * factor, a.sin() * factor, 2 * f.numel()
        if arch.tables():
            c, s = c.half().double(), s.half().double()
        u, w = (t[..., 0:n:2], t[..., 1:n:2]) if arch.rope_interleaved else (t[..., :n // 2], t[..., n // 2:n])
        y = (u * c - w * s, w * c + u * s)
        y = torch.stack(y, -1).flatten(-2) if arch.rope_interleaved else torch.cat(y, -1)
        return torch.cat((y, t[..., n:]), -1).half().transpose(1, 2).contiguous()
    Q, K = at.q_proj.aq.q(turned(q, at.q_norm)), at.kv_quantizer.q(turned(k, at.k_norm))
    V = at.kv_quantizer.q(v.transpose(1, 2).transpose(-1, -2).contiguous()).transpose(-1, -2)
    i, j = torch.arange(T, device="cuda")[:, None], torch.arange(T, device="cuda")[None]
    hidden = j > i
    if arch.window:
        hidden = hidden | ((j <= i - arch.window) & (j >= arch.sinks))
    K, V = K.repeat_interleave(G, 1), V.repeat_interleave(G, 1)
    s = torch.matmul(Q, K.transpose(-1, -2)).double() / math.sqrt(D)
    P = at.attn_wgt_quantizer.q(torch.softmax(s.masked_fill(hidden, -math.inf), -1).half())
    O = (P.double() @ V.double()).half().transpose(1, 2).reshape(B * T, -1)
    return at.o_proj(O)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T,chunk", [(2, 256, 512), (1, 384, 128), (2, 512, 256)])
@torch.no_grad()
def test_a_quantised_block_against_the_separate_operations(kind, B, T, chunk):
    """A value that lands on the other side of a quantizer's border moves by one of its steps, 2^-2 of it (two mantissa bits).  Values
    differ in front of a quantizer by at most two fp16 roundings, 2^-10 of them, so 2^-10 / 2^-2 = 2^-8 of them cross: 2^-2 * 2^-4 = 2^-6
    of the norm; block scales cross as often as 2^-10 / 2^-3 and move a block by its rounding noise, no more than that again.  Four
    quantizers (queries, keys, probabilities, the output projection's input): sqrt(4 * 2) * 2^-6 = 2^-4.5, held to 2^-4, and nine rows
    of ten to twice that.  Rows that see other keys would be off by their own size."""
    m = _model(kind)
    at = m.layers[0].self_attn
    at.query_chunk = chunk
    x = torch.randn((B * T, 256), device="cuda", generator=torch.Generator(device="cuda").manual_seed(7)).half()
    from hbq_b200.llama import rope_tables
    cos, sin = rope_tables(T, 128, 10000.0, x.device)
    got, want = at(x, B, T, cos, sin).double(), _attention(at, x, B, T, m.arch).double()
    rel = (got - want).view(B, T, -1).norm(dim=-1) / want.view(B, T, -1).norm(dim=-1)
    assert float((got - want).norm() / want.norm()) <= 2.0 ** -4 and float(rel.flatten().quantile(0.9)) <= 2.0 ** -3, (float((got - want).norm() / want.norm()), rel.max())


@pytest.mark.parametrize("kind", KINDS)
@torch.no_grad()
def test_prefill_in_runs_is_the_same_attention(kind):
    """Keys beyond a run's end are hidden from all of its queries: whole blocks of zero probabilities.  The library's products
    may add in another order: within a rounding of the fp16 output, as for the plain models."""
    m = _model(kind)
    at = m.layers[0].self_attn
    from hbq_b200.llama import rope_tables
    B, T = 2, 512
    x = torch.randn((B * T, 256), device="cuda", generator=torch.Generator(device="cuda").manual_seed(8)).half()
    cos, sin = rope_tables(T, 128, 10000.0, x.device)
    out = []
    for chunk in (1 << 30, 128, 256):
        at.query_chunk = chunk
        out.append(at(x, B, T, cos, sin).double())
    for o in out[1:]:
        assert float((o - out[0]).norm() / out[0].norm()) <= 2.0 ** -9


@pytest.mark.parametrize("kind", KINDS)
@torch.no_grad()
def test_prefill_in_runs_holds_no_square_of_scores(kind):
    """4096 tokens in runs of 256: scores and probabilities of one run at a time (and its mask), not of the whole prompt."""
    m = _model(kind)
    at = m.layers[0].self_attn
    from hbq_b200.llama import rope_tables
    B, T = 1, 4096
    x = torch.randn((B * T, 256), device="cuda").half()
    cos, sin = rope_tables(T, 128, 10000.0, x.device)
    at.query_chunk = 256
    at(x, B, T, cos, sin)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    at(x, B, T, cos, sin)
    # queries, keys, values, outputs and their copies are below 16 of [T, 4, 128]; the square of scores alone is four heads of T * T
    assert torch.cuda.max_memory_allocated() - before < 16 * T * 4 * 128 * 2 + 4 * T * 256 * 2 * 2


@torch.no_grad()
def test_heads_beyond_the_one_pass_kernel_in_runs():
    """Heads of 256 without quantizers take the masked path: runs against the whole prompt, and against the formula in fp64 of fp16
    queries, keys and values.  Scores, probabilities and the output are each rounded to fp16: the scores' half step, 2^-11 of up to 8,
    is at most 2^-8 of a weight; in a mean of many that is independent of the values, well below 2^-7 of its norm."""
    import hbq_b200 as H
    from hbq_b200.llama import QLlamaAttention
    at = QLlamaAttention(H.LlamaArch(hidden=256, layers=1, heads=4, kv_heads=2, head_dim=256, ffn=512, vocab=512, window=100, sinks=5), device="cuda")
    g = torch.Generator(device="cuda").manual_seed(4)
    B, T, D = 2, 512, 256
    Q, K, V = (torch.randn((B, n, T, D), device="cuda", generator=g).half() for n in (4, 2, 2))
    out = []
    for chunk in (1 << 30, 128, 256):
        at.query_chunk = chunk
        out.append(at._windowed(Q, K, V).double())
    i, j = torch.arange(T, device="cuda")[:, None], torch.arange(T, device="cuda")[None]
    hidden = (j > i) | ((j <= i - 100) & (j >= 5))
    s = (Q.double() @ K.double().repeat_interleave(2, 1).transpose(-1, -2) / 16).masked_fill(hidden, -math.inf)
    want = (torch.softmax(s, -1) @ V.double().repeat_interleave(2, 1)).transpose(1, 2).reshape(B * T, -1)
    for o in out:
        assert float((o - out[0]).norm() / want.norm()) <= 2.0 ** -9
        assert float((o - want).norm() / want.norm()) <= 2.0 ** -7
