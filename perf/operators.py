"""Timed cases of the operators between an attention block's projections and its output projection.

Kinds of case (``case["op"]``):

``rotate``       rotary positions of projected heads (``rope_rotate``): half or interleaved pairs, the whole head or its first
                 part, plain frequencies or frequencies scaled for long contexts, positions anywhere.
``norm_rotate``  RMS norm of every query and key head and the rotation in one pass (``qk_norm_rope``), from the packed
                 projection ``[tokens, (heads + 2 kv_heads) * head_dim]``.
``window``       attention over a K / V cache with a sliding window and a few first tokens that stay visible
                 (``window_attention``): one token a sequence (decode) or prompts.
``prefix``       attention of a batch whose sequences share a long prefix (``shared_prefix_attention``).

Sizes are those of the attention blocks of the Llama-3-8B and Mixtral-8x7B shapes that the benchmark and the tests use
(32 query and 8 key heads of 128), prompts of 8 x 2048 tokens, windows of 4096, and smaller blocks with other heads; token
counts from one up, odd ones among them.  Everything is random: queries and keys N(0, 1) with queries scaled so that some
keys stand out, values N(0, 1), norm weights around 1.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # queries of one decode step: eight sequences, each at its own position
        dict(name="rotate 8 tokens", op="rotate", B=1, T=8, H=32, D=128, rot=128, interleaved=False, scaling="none", first=0, type="fp16"),
        # an odd prompt far into a long context: pairs side by side, a quarter of the head, yarn frequencies
        dict(name="rotate far part", op="rotate", B=3, T=1365, H=32, D=80, rot=32, interleaved=True, scaling="yarn", first=1000003, type="bf16"),
        # the queries of a prefill of 8 x 2048 tokens with frequencies in bands
        dict(name="rotate prompts", op="rotate", B=8, T=2048, H=32, D=128, rot=128, interleaved=False, scaling="bands", first=0, type="bf16"),
        # queries and keys of a decode step of four sequences
        dict(name="norm 4 tokens", op="norm_rotate", B=1, T=4, H=32, Hkv=8, D=128, rot=128, interleaved=False, scaling="none", first=777, type="fp16"),
        # queries and keys of a prefill of 8 x 2048 tokens
        dict(name="norm prompts", op="norm_rotate", B=8, T=2048, H=32, Hkv=8, D=128, rot=128, interleaved=False, scaling="linear", first=0, type="bf16"),
        # one token of one sequence: the smallest decode step
        dict(name="window 1 token", op="window", B=1, L=1, H=32, Hkv=8, S=2048, D=128, window=1024, sinks=4, ragged=True, type="fp16"),
        # a decode batch over long caches of different lengths
        dict(name="window 32 tokens", op="window", B=32, L=1, H=32, Hkv=8, S=16384, D=128, window=4096, sinks=4, ragged=True, type="bf16"),
        # short prompts of odd lengths, padded to the longest, small heads
        dict(name="window short prompts", op="window", B=5, L=999, H=16, Hkv=4, S=999, D=64, window=256, sinks=3, ragged=True, type="fp16"),
        # one long prompt
        dict(name="window long prompt", op="window", B=1, L=8192, H=32, Hkv=8, S=8192, D=128, window=4096, sinks=4, ragged=False, type="bf16"),
        # a few samples of one short prompt
        dict(name="prefix 4 samples", op="prefix", B=4, L=1, H=32, Hkv=8, P=1024, S=256, D=128, ragged=True, type="fp16"),
        # a serving batch behind one long system prompt
        dict(name="prefix 64 sequences", op="prefix", B=64, L=1, H=32, Hkv=8, P=16384, S=1024, D=128, ragged=True, type="bf16"),
        # the prompts of eight requests behind a shared document
        dict(name="prefix 8 prompts", op="prefix", B=8, L=131, H=32, Hkv=8, P=8192, S=131, D=128, ragged=True, type="fp16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges; no case has more work than the largest listed one of its kind."""
    op = rng.choice(["rotate", "norm_rotate", "window", "window", "window", "prefix", "prefix"])
    kind = rng.choice(["fp16", "bf16"])
    G, Hkv = rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([1, 2, 4, 8])
    if op in ("rotate", "norm_rotate"):
        D = rng.choice([64, 80, 96, 112, 128, 256])
        rot = rng.choice([D, D, D // 2, D // 4 // 2 * 2])
        c = dict(op=op, B=rng.choice([1, 1, 2, 3, 8]), T=1, H=G * Hkv, D=D, rot=rot, interleaved=rng.random() < 0.5,
                 scaling=rng.choice(["none", "linear", "ntk", "bands", "yarn"]), first=rng.choice([0, 0, _log(rng, 1, 2000000)]), type=kind)
        heads = c["H"]
        if op == "norm_rotate":
            c["Hkv"] = Hkv
            heads += 2 * Hkv
        most = 8 * 2048 * (32 if op == "rotate" else 48) * 128 // (c["B"] * heads * D)
        c["T"] = _log(rng, 1, max(1, min(most, 16384)))
        return c
    D = rng.choice([64, 80, 96, 128, 128])
    if op == "window" and rng.random() < 0.5:       # one token
        B, window, sinks = _log(rng, 1, 64), rng.choice([0, _log(rng, 16, 8192)]), rng.choice([0, 1, 4, 64])
        S = _log(rng, 1, max(1, min(65536, 32 * 8 * 8192 * 128 // (B * Hkv * D))))
        return dict(op=op, B=B, L=1, H=G * Hkv, Hkv=Hkv, S=S, D=D, window=window, sinks=sinks, ragged=rng.random() < 0.7, type=kind)
    if op == "window":                              # prompts, or the next piece of a prompt behind its cached start
        B = rng.choice([1, 1, 2, 3, 8])
        L = _log(rng, 2, max(2, int(math.sqrt(8192 * 8192 * 32 * 128 / (2 * B * G * Hkv * D)))))
        L = min(L, 8192)
        S = L + rng.choice([0, 0, _log(rng, 1, L)])
        return dict(op=op, B=B, L=L, H=G * Hkv, Hkv=Hkv, S=S, D=D, window=rng.choice([0, _log(rng, 1, 4096)]),
                    sinks=rng.choice([0, 1, 4, 130]), ragged=rng.random() < 0.5, type=kind)
    B, L = _log(rng, 2, 64), rng.choice([1, 1, _log(rng, 2, 131)])
    most = 8 * 131 * 32 * 8323 * 128 // (B * L * G * Hkv * D)
    P = _log(rng, 64, max(64, min(16384, most)))
    S = L + rng.choice([0, _log(rng, 1, max(1, min(1024, most // 4)))])
    return dict(op=op, B=B, L=L, H=G * Hkv, Hkv=Hkv, P=P, S=S, D=D, ragged=rng.random() < 0.7, type=kind)


# ---- inputs ------------------------------------------------------------------------------------------------------
def _lengths(c):
    """Keys in each sequence's cache: all of it, or (ragged) from about half of it up, never fewer than one."""
    if not c["ragged"]:
        return [c["S"]] * c["B"]
    return [max(1, c["S"] - (b * 2654435761 + 12345) % (c["S"] // 2 + 1)) for b in range(c["B"])]


def _padded(c):
    """Whole prompts, each at the front of its rows, padded to the longest."""
    return c["L"] == c["S"] and c["L"] > 1


def _frequencies(c):
    """``(f, factor)``: the rotation's angle per position for each pair, in 64 bits, and what cosine and sine are multiplied by."""
    r, theta = c["rot"], 500000.0
    scaling, factor = c["scaling"], 8.0
    if scaling == "ntk":                                    # a larger base, so that the slowest pair turns `factor` times slower
        theta *= factor ** (r / max(r - 2, 1))
    f = theta ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "bands":                                  # long wavelengths slowed, short ones kept, a ramp between them
        low, high, context = 1.0, 4.0, 8192
        turns = context * f / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        return keep * f + (1 - keep) * f / factor, 1.0
    if scaling == "yarn":                                   # a ramp over the pairs' indices, and a factor for the sharper softmax
        context, fast, slow = 8192, 32.0, 1.0
        at = lambda turns: r * math.log(context / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(at(fast)), 0), min(math.ceil(at(slow)), r - 1)
        keep = 1 - ((torch.arange(r // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        return keep * f + (1 - keep) * f / factor, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["type"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, device="cuda", generator=g, dtype=torch.float32).mul_(scale).to(t)

    s = {"case": case}
    if case["op"] in ("rotate", "norm_rotate"):
        B, T, H, D = (case[n] for n in "BTHD")
        f, s["factor"] = _frequencies(case)
        s["inv_freq"] = f.cuda()
        if B == 1:      # a decode step: each token of another sequence, at a position of its own
            s["positions"] = case["first"] + torch.randint(0, 8192, (B, T), device="cuda", generator=g)
        else:           # prompts: each continues at its own place
            s["positions"] = case["first"] + torch.arange(T, device="cuda")[None] + torch.randint(0, 64, (B, 1), device="cuda", generator=g)
        if case["op"] == "rotate":
            s["x"] = normal(B, T, H, D)
        else:
            s["qkv"] = normal(B, T, (H + 2 * case["Hkv"]) * D)
            s["q_weight"], s["k_weight"] = (normal(D, scale=0.1) + 1 for _ in range(2))
        return s
    B, L, H, Hkv, S, D = (case[n] for n in ("B", "L", "H", "Hkv", "S", "D"))
    s["q"] = normal(B, L, H, D, scale=1.5)
    s["k"], s["v"] = normal(B, Hkv, S, D), normal(B, Hkv, S, D)
    s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    # prompts of different lengths stand at the front of their rows; a single token, or a piece that continues, at the end of its keys
    s["starts"] = torch.zeros_like(s["lengths"]) if _padded(case) else None
    if case["op"] == "prefix":
        s["pk"], s["pv"] = normal(Hkv, case["P"], D), normal(Hkv, case["P"], D)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _rotate(x, f, positions, interleaved, factor):
    """x [B, T, H, D] in 32 bits; angles in 64."""
    a = positions.double()[..., None, None] * f
    c, s = (a.cos() * factor).float(), (a.sin() * factor).float()
    r = 2 * f.numel()
    first, second = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    u, w = first * c - second * s, second * c + first * s
    pairs = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((pairs, x[..., r:]), -1)


def _heads_norm(x, weight, eps):
    x = x.float()
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * weight.float()


def _inside(L, lengths, starts):
    """[B, L, 1]: the rows that are not padding behind their sequence's end."""
    return ((starts if starts is not None else lengths - L)[:, None] + torch.arange(L, device=lengths.device) < lengths[:, None])[..., None]


def _visible(L, S, lengths, starts, window, sinks):
    """[B, L, S]: which keys a row sees; a row at or behind its sequence's end sees none."""
    p = (starts if starts is not None else lengths - L)[:, None, None] + torch.arange(L, device=lengths.device)[None, :, None]
    j, n = torch.arange(S, device=lengths.device)[None, None], lengths[:, None, None]
    see = (j <= p) & (j < n) & (p < n)
    return see & ((j > p - window) | (j < sinks)) if window else see


def _softmax_(s):
    """Softmax over the last axis, in place; rows of -inf alone become zeros."""
    m = s.amax(-1, keepdim=True)
    s.sub_(m.masked_fill_(m == -math.inf, 0)).exp_()
    n = s.sum(-1, keepdim=True)
    return s.div_(n.masked_fill_(n == 0, 1))


def _by_kv_head(q, Hkv):
    """[B, L, H, D] -> [B, Hkv, G * L, D] in 32 bits: the rows that share a key head."""
    B, L, H, D = q.shape
    return q.float().view(B, L, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, H // Hkv * L, D)


def _by_token(o, L, H):
    B, Hkv, _, D = o.shape
    return o.view(B, Hkv, H // Hkv, L, D).permute(0, 3, 1, 2, 4).reshape(B, L, H, D)


def _window(q, k, v, lengths, starts, window, sinks):
    B, L, H, D = q.shape
    Hkv, S = k.shape[1], k.shape[2]
    s = torch.matmul(_by_kv_head(q, Hkv), k.float().transpose(-1, -2)).mul_(1 / math.sqrt(D))
    see = _visible(L, S, lengths, starts, window, sinks)
    s.view(B, H, L, S).masked_fill_(~see[:, None], -math.inf)
    return _by_token(torch.matmul(_softmax_(s), v.float()), L, H).to(q.dtype)


def _prefix(q, pk, pv, k, v, lengths, starts):
    B, L, H, D = q.shape
    Hkv, P, S = pk.shape[0], pk.shape[1], k.shape[2]
    rows = _by_kv_head(q, Hkv)
    s = torch.empty((B, Hkv, rows.shape[2], P + S), dtype=torch.float32, device=q.device)
    s[..., :P] = torch.matmul(rows, pk.float().transpose(-1, -2))
    s[..., P:] = torch.matmul(rows, k.float().transpose(-1, -2))
    s.mul_(1 / math.sqrt(D))
    see = torch.cat((_inside(L, lengths, starts).expand(B, L, P), _visible(L, S, lengths, starts, 0, 0)), -1)
    s.view(B, H, L, P + S).masked_fill_(~see[:, None], -math.inf)
    _softmax_(s)
    return _by_token(torch.matmul(s[..., :P], pv.float()) + torch.matmul(s[..., P:], v.float()), L, H).to(q.dtype)


def run(state):
    c = state["case"]
    if c["op"] == "rotate":
        x, f, positions, interleaved, factor = state["x"], state["inv_freq"], state["positions"], c["interleaved"], state["factor"]
        if own:
            from hbq_b200 import rope_rotate
            return rope_rotate(x, f, positions, interleaved=interleaved, factor=factor)
        return _rotate(x.float(), f, positions, interleaved, factor).to(x.dtype)
    if c["op"] == "norm_rotate":
        qkv, H, Hkv, D = state["qkv"], c["H"], c["Hkv"], c["D"]
        B, T = qkv.shape[0], qkv.shape[1]
        q, k = qkv[..., :H * D].view(B, T, H, D), qkv[..., H * D:(H + Hkv) * D].view(B, T, Hkv, D)
        f, positions, interleaved, factor = state["inv_freq"], state["positions"], c["interleaved"], state["factor"]
        if own:
            from hbq_b200 import qk_norm_rope
            return qk_norm_rope(q, k, state["q_weight"], state["k_weight"], 1e-5, f, positions, interleaved=interleaved, factor=factor)
        return tuple(_rotate(_heads_norm(x, w, 1e-5), f, positions, interleaved, factor).to(x.dtype)
                     for x, w in ((q, state["q_weight"]), (k, state["k_weight"])))
    if c["op"] == "window":
        if own:
            from hbq_b200 import window_attention
            return window_attention(state["q"], state["k"], state["v"], window=c["window"], sinks=c["sinks"], lengths=state["lengths"],
                                    starts=state["starts"])
        return _window(state["q"], state["k"], state["v"], state["lengths"], state["starts"], c["window"], c["sinks"])
    if own:
        from hbq_b200 import shared_prefix_attention
        return shared_prefix_attention(state["q"], state["pk"], state["pv"], state["k"], state["v"], lengths=state["lengths"], starts=state["starts"])
    return _prefix(state["q"], state["pk"], state["pv"], state["k"], state["v"], state["lengths"], state["starts"])


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def _pairs(c):
    """(row, key) pairs that a head computes over all sequences, and the keys that some row sees."""
    pairs = keys = 0
    for n in _lengths(c):
        L, window, sinks = c["L"], c.get("window", 0), c.get("sinks", 0)
        first = 0 if _padded(c) else n - L
        low = n
        for p in range(max(first, 0), min(first + L, n)):
            start = max(p + 1 - window, 0) if window else 0
            pairs += p + 1 - start + min(sinks, start)
            low = min(low, start)
        keys += n - low + min(sinks, low) if low < n else 0
    return pairs, keys


def work(case):
    D = case["D"]
    if case["op"] == "rotate":
        n = case["B"] * case["T"] * case["H"]
        return {"bytes": 4.0 * n * D + 8 * case["B"] * case["T"], "flops": 3.0 * n * case["rot"]}
    if case["op"] == "norm_rotate":
        n = case["B"] * case["T"] * (case["H"] + case["Hkv"])
        return {"bytes": 4.0 * n * D + 8 * case["B"] * case["T"], "flops": n * (4.0 * D + 3 * case["rot"])}
    pairs, keys = _pairs(case)
    rows = case["B"] * case["L"] * case["H"]
    shared = case.get("P", 0)
    inside = sum(min(n, case["L"]) for n in _lengths(case)) if _padded(case) else case["B"] * case["L"]
    return {"bytes": 4.0 * rows * D + 4.0 * (keys + shared) * case["Hkv"] * D, "flops": 4.0 * D * case["H"] * (pairs + inside * shared)}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------
def _exact_turned(x, s, c):
    """Each pair as a complex number times factor * e^(i angle)."""
    r = c["rot"]
    a = torch.outer(s["positions"].reshape(-1).to(torch.float64), s["inv_freq"]).view(c["B"], c["T"], 1, r // 2)
    turn = torch.polar(torch.full_like(a, s["factor"]), a)
    y = x.clone()
    if c["interleaved"]:
        y[..., :r] = torch.view_as_real(torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * turn).flatten(-2)
    else:
        z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
        y[..., :r // 2], y[..., r // 2:r] = z.real, z.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotate":
        return _exact_turned(s["x"].double(), s, case)
    if case["op"] == "norm_rotate":
        D, H = case["D"], case["H"]
        heads = s["qkv"].double().unflatten(-1, (-1, D))
        out = []
        for x, w in ((heads[..., :H, :], s["q_weight"]), (heads[..., H:H + case["Hkv"], :], s["k_weight"])):
            size = torch.linalg.vector_norm(x, dim=-1, keepdim=True).pow(2) / D
            out.append(_exact_turned(x / (size + 1e-5).sqrt() * w.double(), s, case))
        return tuple(out)
    # one sequence and head at a time: rows of weights that sum to one, over the keys that the row's position leaves
    B, L, H, D, S = (case[n] for n in ("B", "L", "H", "D", "S"))
    G, dev = H // case["Hkv"], s["q"].device
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    out = torch.zeros((B, L, H, D), dtype=torch.float64, device=dev)
    for b, n in enumerate(_lengths(case)):
        first = 0 if s["starts"] is not None else n - L
        p = first + torch.arange(L, device=dev)[:, None]
        j = torch.arange(n, device=dev)[None]
        hidden = (j > p) | (p >= n)
        if window:
            hidden |= (p - j >= window) & (j >= sinks)
        for h in range(case["Hkv"]):
            k, v = s["k"][b, h, :n].double(), s["v"][b, h, :n].double()
            mask = hidden
            if case["op"] == "prefix":
                k, v = torch.cat((s["pk"][h].double(), k)), torch.cat((s["pv"][h].double(), v))
                mask = torch.cat(((p >= n).expand(L, case["P"]), hidden), 1)
            rows = s["q"][b, :, h * G:(h + 1) * G].double()
            z = torch.einsum("lgd,sd->gls", rows, k) / D ** 0.5
            z.masked_fill_(mask, -torch.inf)
            weights = torch.exp(z - torch.logsumexp(z, -1, keepdim=True)).nan_to_num_(0.0)
            out[b, :, h * G:(h + 1) * G] = torch.einsum("gls,sd->lgd", weights, v)
    return out
