"""GPU: decoders whose attention has a window and first tokens, norms of its heads, and other rotations than the tables'.

The unquantised model is held to a restatement of the block in fp64 that rounds to fp16 where the fp16 model does (the
projections, the norms, the rotated heads, the attention's output).  A value that lands on the other side of a rounding
border there moves by one step, 2^-10 of it, in a random direction; some twenty roundings a layer and two layers give
relative errors of a few 2^-11 in the logits, and 5e-3 is the bound that the model's other tests use."""
import json
import math
import os

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))

KINDS = {
    "window": dict(window=40, sinks=3),
    "window of all": dict(window=1000),
    "norms": dict(qk_norm=True),
    "norms, part, pairs": dict(qk_norm=True, rotary_dim=32, rope_interleaved=True, window=17),
    "scaled": dict(rope_scaling=dict(type="yarn", factor=4.0, original_max_position_embeddings=64)),
    "part": dict(rotary_dim=16, window=64, sinks=130),
}


def _arch(**kw):
    import hbq_b200 as H
    return H.LlamaArch(**{**dict(hidden=256, layers=2, heads=8, kv_heads=2, head_dim=64, ffn=512, vocab=512, eps=1e-5, theta=10000.0), **kw})


def _logits(m, ids):
    """The unquantised model's logits from its weights."""
    import hbq_b200 as H
    a = m.arch
    w = {k: v.detach().double() for k, v in m.state_dict().items()}
    r = lambda t: t.half().double()  # noqa: E731
    B, T = ids.shape
    D, G = a.head_dim, a.heads // a.kv_heads

    def norm(x, g):
        return r(g * r(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + a.eps)))

    def turned(x, g):                                                        # [B, T, H, D]
        f, factor = H.rope_frequencies(a.rotary_dim or D, a.theta, a.rope_scaling, device="cuda")
        if a.qk_norm:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + a.eps) * g
        ang = torch.arange(T, device="cuda").double()[:, None, None] * f
        c, s = ang.cos() * factor, ang.sin() * factor
        n = 2 * f.numel()
        if a.tables():                                                       # fp16 tables, each op rounded
            c, s = r(c.float().double()), r(s.float().double())
            u, v = x[..., :n // 2], x[..., n // 2:]
            return torch.cat((r(r(u * c) - r(v * s)), r(r(v * c) + r(u * s))), -1)
        u, v = (x[..., 0:n:2], x[..., 1:n:2]) if a.rope_interleaved else (x[..., :n // 2], x[..., n // 2:n])
        y = (u * c - v * s, v * c + u * s)
        return r(torch.cat((torch.stack(y, -1).flatten(-2) if a.rope_interleaved else torch.cat(y, -1), x[..., n:]), -1))

    i, j = torch.arange(T, device="cuda")[:, None], torch.arange(T, device="cuda")[None]
    hidden = j > i
    if a.window:
        hidden = hidden | ((j <= i - a.window) & (j >= a.sinks))
    x = w["embed_tokens.weight"][ids]
    for n in range(a.layers):
        p = f"layers.{n}."
        h = norm(x, w[p + "input_layernorm"])
        q, k, v = (r(h @ w[p + f"self_attn.{t}_proj.weight"].T).view(B, T, -1, D) for t in "qkv")
        q, k = turned(q, w.get(p + "self_attn.q_norm")), turned(k, w.get(p + "self_attn.k_norm"))
        q, k, v = q.transpose(1, 2), k.transpose(1, 2).repeat_interleave(G, 1), v.transpose(1, 2).repeat_interleave(G, 1)
        s = (q @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill(hidden, -math.inf)
        o = r(torch.softmax(s, -1) @ v).transpose(1, 2).reshape(B, T, -1)
        x = r(x + r(o @ w[p + "self_attn.o_proj.weight"].T))
        h = norm(x, w[p + "post_attention_layernorm"])
        g, u = r(h @ w[p + "mlp.gate_proj.weight"].T), r(h @ w[p + "mlp.up_proj.weight"].T)
        x = r(x + r(r(r(torch.nn.functional.silu(g)) * u) @ w[p + "mlp.down_proj.weight"].T))
    return (norm(x, w["norm"]) @ w["lm_head.weight"].T).reshape(B * T, -1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("B,T", [(2, 130), (1, 1), (3, 37)])
def test_logits(kind, B, T):
    import hbq_b200 as H
    m = H.QLlamaModel(_arch(**KINDS[kind]), device="cuda")
    m.init_weights(5)
    if m.arch.qk_norm:
        for layer in m.layers:
            for t in (layer.self_attn.q_norm, layer.self_attn.k_norm):
                t.data.uniform_(0.5, 1.5, generator=torch.Generator(device="cuda").manual_seed(3))
    ids = torch.randint(0, 512, (B, T), generator=torch.Generator().manual_seed(1)).cuda()
    got, want = m(ids).double(), _logits(m, ids)
    rel = float((got - want).norm() / want.norm())
    assert rel <= 5e-3, rel


def test_a_window_changes_nothing_before_it_closes():
    import hbq_b200 as H
    ids = torch.randint(0, 512, (1, 90), generator=torch.Generator().manual_seed(2)).cuda()
    out = []
    for window, sinks in ((30, 0), (30, 5), (90, 0)):
        m = H.QLlamaModel(_arch(layers=1, window=window, sinks=sinks), device="cuda")
        m.init_weights(5)
        out.append(m(ids))
    assert torch.equal(out[0][:30], out[2][:30]) and torch.equal(out[1][:30], out[2][:30])
    assert not torch.equal(out[0][35:], out[2][35:]) and not torch.equal(out[1][36:], out[0][36:])


def test_quantised_probabilities_under_a_window():
    """The path with the mask in memory and quantised weights: with a window over everything it is the causal attention.  What
    stands before the window closes is the same in one layer; a second layer's values are quantised in blocks of 128 tokens,
    whose scales the later tokens change."""
    import hbq_b200 as H
    with open(os.path.join(HERE, "golden", "ptq_configs.json")) as fh:
        cfg = json.load(fh)["hbq_a_kv.yaml"]["config"]
    ids = torch.randint(0, 512, (2, 128), generator=torch.Generator().manual_seed(2)).cuda()
    for layers in (1, 2):
        out = []
        for window in (0, 128, 40):
            m = H.QLlamaModel(_arch(head_dim=128, heads=4, window=window, layers=layers), device="cuda")
            m.init_weights(5)
            m.apply_ptq(H.PTQConfig(cfg))
            out.append(m(ids))
        assert bool(torch.isfinite(out[2]).all()) and torch.equal(out[0], out[1]) and not torch.equal(out[0][45:128], out[2][45:128])
        if layers == 1:
            assert torch.equal(out[0][:40], out[2][:40])
