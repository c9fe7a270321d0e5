"""Cases of the decoding operators: the quantised KV cache, attention over a
cache with a prefix shared by the batch, the recurrent gated delta rule, and the
verification of drafted tokens.

``run`` computes one operator either in its plain form (elementary torch
operations in 32 bits, rounded once at the end) or, with ``own`` set, through
the package's public entry points.
"""
import math

import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0


# --------------------------------------------------------------------- cases
def listed():
    return [
        # One user's decode step: a single token of one sequence written and read (latency).
        dict(name="kv_one_token", op="kv", batch=1, tokens=1, kv_heads=4, head_dim=64, capacity=4096),
        # Prompts of a batch written at once, ragged counts, each at its own offset; read back as bf16.
        dict(name="kv_prompts", op="kv", batch=16, tokens=4096, kv_heads=4, head_dim=128, capacity=4500),
        # One user's decode step over its own 4 K context, no shared prefix (latency).
        dict(name="attn_one_user", op="attn", batch=1, tokens=1, q_heads=16, kv_heads=4, head_dim=64,
             prefix=0, capacity=4096, window=0, cache="bf16"),
        # A served batch behind one system prompt, a token each, own contexts of all lengths.
        dict(name="attn_served_batch", op="attn", batch=64, tokens=1, q_heads=16, kv_heads=4, head_dim=64,
             prefix=4096, capacity=1024, window=0, cache="fp8"),
        # Five drafted positions a sequence to verify, odd prefix, head dim 128, quantised cache.
        dict(name="attn_drafted", op="attn", batch=32, tokens=5, q_heads=16, kv_heads=4, head_dim=128,
             prefix=8191, capacity=777, window=0, cache="fp8"),
        # Many short continuations of one long document: the shared prefix is nearly all of the work.
        dict(name="attn_long_document", op="attn", batch=256, tokens=4, q_heads=16, kv_heads=4, head_dim=64,
             prefix=32768, capacity=256, window=0, cache="bf16"),
        # One sequence's decode step through a recurrent layer (latency).
        dict(name="kda_one_token", op="kda", batch=1, tokens=1, heads=16, head_dim=64, dtype="fp32", shared_state=False),
        # A large served batch, a token each: the states' traffic is the work.
        dict(name="kda_served_batch", op="kda", batch=256, tokens=1, heads=16, head_dim=64, dtype="fp32",
             shared_state=False),
        # Prompt remainders behind a shared prefix state, ragged, head dim 128, 16-bit rows.
        dict(name="kda_prompts", op="kda", batch=16, tokens=509, heads=16, head_dim=128, dtype="bf16",
             shared_state=True),
        # One sequence with four drafted tokens (latency), a draft without probabilities (prompt lookup).
        dict(name="verify_one", op="verify", batch=1, drafted=4, vocab=32768, dtype="fp32", draft="tokens"),
        # A served batch, five drafted tokens each from a draft model, odd vocabulary, 16-bit logits.
        dict(name="verify_odd_vocab", op="verify", batch=24, drafted=5, vocab=50257, dtype="bf16", draft="logits"),
        # A large batch with long drafts.
        dict(name="verify_large", op="verify", batch=128, drafted=7, vocab=32768, dtype="fp32", draft="logits"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


#: The work of the largest listed case of each operator: a drawn one costs no more.
_MOST = {}


def draw(rng):
    if not _MOST:
        for c in listed():
            _MOST[c["op"]] = max(_MOST.get(c["op"], 0.0), _cost(c))
    op = rng.choice(["kv", "attn", "attn", "kda", "verify"])
    while True:
        if op == "kv":
            tokens = _log_int(rng, 1, 4096)
            c = dict(op=op, batch=_log_int(rng, 1, 64), tokens=tokens, kv_heads=rng.choice([1, 2, 3, 4, 8]),
                     head_dim=rng.choice([32, 64, 128]), capacity=tokens + _log_int(rng, 1, 2000))
        elif op == "attn":
            tokens = rng.choice([1, 1, 2, 3, 4, 5, 8])
            kv = rng.choice([1, 2, 4])
            prefix = rng.choice([0, 1, 1, 1]) * _log_int(rng, 1, 32768)
            c = dict(op=op, batch=_log_int(rng, 1, 256), tokens=tokens, q_heads=kv * rng.choice([1, 2, 3, 4, 8]),
                     kv_heads=kv, head_dim=rng.choice([32, 64, 128]), prefix=prefix,
                     capacity=tokens + _log_int(rng, 1, 8192), window=rng.choice([0, 0, 0, _log_int(rng, 16, 8192)]),
                     cache=rng.choice(["bf16", "fp8"]))
        elif op == "kda":
            c = dict(op=op, batch=_log_int(rng, 1, 256), tokens=rng.choice([1, 2, 5, _log_int(rng, 1, 700)]),
                     heads=rng.choice([2, 4, 16, 16, 24]), head_dim=rng.choice([32, 64, 64, 128]),
                     dtype=rng.choice(["fp32", "bf16"]), shared_state=rng.random() < 0.3)
        else:
            c = dict(op=op, batch=_log_int(rng, 1, 128), drafted=rng.choice([1, 2, 3, 4, 5, 7]),
                     vocab=_log_int(rng, 256, 66000), dtype=rng.choice(["fp32", "bf16"]),
                     draft=rng.choice(["logits", "logits", "tokens"]))
        if _cost(c) <= _MOST[op]:
            return c


def _cost(c):
    w = work(c)
    return max(w["bytes"], w["flops"] / 50)


def work(case):
    c = case
    if c["op"] == "kv":
        rows = c["batch"] * c["tokens"] * c["kv_heads"] * 2   # keys and values
        H = c["head_dim"]
        # bf16 in, 8-bit code and exponent out; code and exponent in, bf16 out
        return {"bytes": rows * (2 * H + (H + 1) + (H + 1) + 2 * H), "flops": rows * H * 4}
    if c["op"] == "attn":
        H, rows = c["head_dim"], c["batch"] * c["tokens"]
        el = (2 if c["cache"] == "bf16" else 1) * H + (0 if c["cache"] == "bf16" else 1)
        pre, own_keys = c["prefix"], c["batch"] * _mean_length(c)
        if c["window"]:
            pre = min(pre, c["window"])
            own_keys = c["batch"] * min(_mean_length(c), c["window"])
        per_query = pre + own_keys / c["batch"]
        return {"bytes": 2 * el * c["kv_heads"] * (pre + own_keys) + 2 * 2 * rows * c["q_heads"] * H,
                "flops": 4 * H * rows * c["q_heads"] * per_query}
    if c["op"] == "kda":
        K, n = c["head_dim"], c["batch"] * c["heads"]
        el = 4 if c["dtype"] == "fp32" else 2
        toks = n * c["tokens"]
        states = n + (c["heads"] if c["shared_state"] else n)
        # q, k, v in their type; decay, beta and output in 32 bits
        return {"bytes": states * K * K * 4 + toks * (3 * K * el + K * 4 + 4 + K * 4), "flops": toks * 7 * K * K}
    B, K, V = c["batch"], c["drafted"], c["vocab"]
    el = 4 if c["dtype"] == "fp32" else 2
    rows = B * (K + 1) + (B * K if c["draft"] == "logits" else 0)
    return {"bytes": rows * V * el + B * V * 4, "flops": rows * V * 5}


def _mean_length(c):
    return (c["capacity"] + c["tokens"]) / 2


# -------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _pow2(e):
    """2^e as fp32, exactly, for integers -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _quantise(x):
    """Rows of H values as 8-bit floats and one power-of-two exponent a row."""
    x = x.float()
    finite = torch.isfinite(x)
    amax = torch.where(finite, x.abs(), torch.zeros_like(x)).amax(-1)
    # amax = m * 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    m, e = torch.frexp(amax)
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(-120, 119)
    e = torch.where(amax == 0, torch.zeros_like(e), e)
    y = (x * _pow2(-e)[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    return y.to(torch.float8_e4m3fn), e.to(torch.int8)


def _dequantise(code, e):
    return code.float() * _pow2(e)[..., None]


def _filled(g, shape, kind):
    """Cached rows of earlier tokens (bf16, or 8-bit codes with exponents)."""
    x = _randn(g, *shape)
    x[..., 0] *= 3   # a dominant channel, as trained keys and values have
    x = x.bfloat16()
    return (x, None) if kind == "bf16" else _quantise(x)


def prepare(case, seed):
    c, g = case, _gen(seed)
    B = c["batch"]
    if c["op"] == "kv":
        N, H, S, C = c["kv_heads"], c["head_dim"], c["tokens"], c["capacity"]
        # rows of one projection buffer [k | v], as the layer's product leaves them
        kv = _randn(g, B, S, 2 * N * H)
        kv *= torch.exp(0.7 * _randn(g, B, S, 1))   # token norms spread over a factor of a few
        kv = kv.bfloat16()
        starts = (_rand(g, B) * (C - S + 1)).to(torch.int32).clamp_(max=C - S)
        counts = (S - (_rand(g, B) * max(1, S // 2)).to(torch.int32)).clamp_(min=1)
        return dict(case=c, k=kv[..., :N * H].unflatten(-1, (N, H)), v=kv[..., N * H:].unflatten(-1, (N, H)),
                    starts=starts, counts=counts,
                    k_cache=torch.zeros(B, C, N, H, device=DEV).to(torch.float8_e4m3fn),
                    v_cache=torch.zeros(B, C, N, H, device=DEV).to(torch.float8_e4m3fn),
                    k_exp=torch.zeros(B, C, N, dtype=torch.int8, device=DEV),
                    v_exp=torch.zeros(B, C, N, dtype=torch.int8, device=DEV))
    if c["op"] == "attn":
        N, H, S, C, P = c["kv_heads"], c["head_dim"], c["tokens"], c["capacity"], c["prefix"]
        st = dict(case=c)
        st["q"] = (1.5 * _randn(g, B, S, c["q_heads"], H)).bfloat16()
        st["k"], st["k_exp"] = _filled(g, (B, C, N, H), c["cache"])
        st["v"], st["v_exp"] = _filled(g, (B, C, N, H), c["cache"])
        st["lengths"] = (S + (_rand(g, B) * (C - S + 1)).to(torch.int32)).clamp_(max=C)
        st["counts"] = (S - (_rand(g, B) * S).to(torch.int32)).clamp_(min=1)
        if P:
            st["pk"], st["pk_exp"] = _filled(g, (1, P, N, H), c["cache"])
            st["pv"], st["pv_exp"] = _filled(g, (1, P, N, H), c["cache"])
        return st
    if c["op"] == "kda":
        S, N, K = c["tokens"], c["heads"], c["head_dim"]
        dt = torch.float32 if c["dtype"] == "fp32" else torch.bfloat16

        def unit(x):
            return x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)

        q, k = unit(_randn(g, B, S, N, K)).to(dt), unit(_randn(g, B, S, N, K)).to(dt)
        x = _randn(g, B, S, N, K)
        v = (x * torch.sigmoid(x)).to(dt)
        decay = -(1 + 15 * _rand(g, N))[:, None] * torch.exp(_randn(g, B, S, N, K) - 4.0)
        beta = torch.sigmoid(_randn(g, B, S, N))
        state = 0.3 * _randn(g, 1 if c["shared_state"] else B, N, K, K)
        counts = (S - (_rand(g, B) * max(1, S // 2)).to(torch.int32)).clamp_(min=1)
        return dict(case=c, q=q, k=k, v=v, g=decay, beta=beta, state=state, counts=counts, scale=K ** -0.5)
    K, V = c["drafted"], c["vocab"]
    dt = torch.float32 if c["dtype"] == "fp32" else torch.bfloat16
    target = 2.5 * _randn(g, B, K + 1, V)
    # nucleus-like rows: every third sequence keeps its larger logits only
    target[::3] = torch.where(target[::3] > 4.0, target[::3], torch.full_like(target[::3], float("-inf")))
    target[..., 0] = 5.0
    draft = (target[:, :K] + 0.7 * _randn(g, B, K, V)).to(dt)
    target = target.to(dt)
    temperature = 0.6 + 0.6 * _rand(g, B)
    temperature[3::4] = 0.0   # greedy sequences in the same batch
    warm = torch.where(temperature > 0, temperature, torch.ones_like(temperature))
    race = torch.softmax(draft.float() / warm[:, None, None], -1) / _exponential(g, B, K, V)
    tokens = torch.where((temperature > 0)[:, None], race.argmax(-1), draft.float().argmax(-1))
    lens = (K - (_rand(g, B) * 2).to(torch.int32)).clamp_(min=0)
    return dict(case=c, target=target, draft=draft if c["draft"] == "logits" else None, tokens=tokens, lens=lens,
                uniform=_rand(g, B, K), noise=_exponential(g, B, V), temperature=temperature)


def _exponential(g, *shape):
    return -torch.log1p(-_rand(g, *shape)).clamp(max=-1e-30)


# --------------------------------------------------------------- plain forms
def _kv_plain(s):
    S = s["k"].shape[1]
    pos = s["starts"][:, None].long() + torch.arange(S, device=DEV)   # [B, S]
    live = torch.arange(S, device=DEV) < s["counts"][:, None]
    rows = torch.arange(pos.shape[0], device=DEV)[:, None]
    out = []
    for x, code, e in ((s["k"], s["k_cache"].view(torch.uint8), s["k_exp"]),
                       (s["v"], s["v_cache"].view(torch.uint8), s["v_exp"])):
        y, ye = _quantise(x)
        code[rows, pos] = torch.where(live[..., None, None], y.view(torch.uint8), code[rows, pos])
        e[rows, pos] = torch.where(live[..., None], ye, e[rows, pos])
        out.append(_dequantise(code[rows, pos].view(torch.float8_e4m3fn), e[rows, pos]).bfloat16())
    return out


def _values(x, e):
    return x.float() if e is None else _dequantise(x, e)


def _attn_plain(s):
    c, q = s["case"], s["q"].float()
    B, S, Nq, H = q.shape
    N, P, C, W = c["kv_heads"], c["prefix"], c["capacity"], c["window"]
    G = Nq // N
    q = q.view(B, S, N, G, H).permute(2, 0, 1, 3, 4)                       # N B S G H
    step = torch.arange(S, device=DEV)
    pos = P + (s["lengths"] - s["counts"])[:, None].long() + step          # [B, S]
    live = step < s["counts"][:, None]
    key = P + torch.arange(C, device=DEV)
    seen = live[..., None] & (key <= pos[..., None])
    if W:
        seen &= pos[..., None] - key < W
    k, v = _values(s["k"], s["k_exp"]), _values(s["v"], s["v_exp"])        # B C N H
    own_s = torch.einsum("nbsgh,bcnh->nbsgc", q, k) / math.sqrt(H)
    own_s = own_s.masked_fill(~seen[None, :, :, None, :], float("-inf"))
    m = own_s.amax(-1, keepdim=True)
    if P:
        pk, pv = _values(s["pk"], s["pk_exp"])[0], _values(s["pv"], s["pv_exp"])[0]
        pre_s = torch.matmul(q.reshape(N, B * S * G, H), pk.permute(1, 2, 0)).view(N, B, S, G, P) / math.sqrt(H)
        if W:
            pre_seen = pos[..., None] - torch.arange(P, device=DEV) < W
            pre_s = pre_s.masked_fill(~pre_seen[None, :, :, None, :], float("-inf"))
        m = torch.maximum(m, pre_s.amax(-1, keepdim=True))
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    own_p = torch.exp(own_s - m)
    total = own_p.sum(-1, keepdim=True)
    o = torch.einsum("nbsgc,bcnh->nbsgh", own_p, v)
    if P:
        pre_p = torch.exp(pre_s - m)
        total = total + pre_p.sum(-1, keepdim=True)
        o = o + torch.matmul(pre_p.view(N, B * S * G, P), pv.permute(1, 0, 2)).view(N, B, S, G, H)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o * live[None, :, :, None, None]
    return o.permute(1, 2, 0, 3, 4).reshape(B, S, Nq, H).bfloat16()


def _kda_plain(s):
    q, k, v, g, beta = (s[x].float() for x in ("q", "k", "v", "g", "beta"))
    B, S, N, K = q.shape
    state = s["state"].expand(B, N, K, K)
    live = torch.arange(S, device=DEV) < s["counts"][:, None]
    # a token past its sequence's count decays by 1 and writes nothing
    decay = torch.exp(g * live[..., None, None])[..., None]
    beta = (beta * live[..., None])[..., None]
    outs = []
    for t in range(S):   # the recurrence
        state = state * decay[:, t]
        seen = (state * k[:, t, :, :, None]).sum(-2)
        new = beta[:, t] * (v[:, t] - beta[:, t] * seen)
        state = state + k[:, t, :, :, None] * new[..., None, :]
        outs.append((state * q[:, t, :, :, None]).sum(-2))
    o = torch.stack(outs, 1) * s["scale"] * live[..., None, None]
    return o, state


def _verify_plain(s):
    t, tok, lens = s["target"].float(), s["tokens"], s["lens"].long()
    B, K1, V = t.shape
    K = K1 - 1
    T = s["temperature"]
    greedy = T == 0
    inv = (1.0 / torch.where(greedy, torch.ones_like(T), T))[:, None, None]
    top = t.amax(-1, keepdim=True)
    lowest = torch.where(t == top, torch.arange(V, device=DEV), V).amin(-1)   # the lowest index of the maximum
    x = (t - top) * inv
    e = torch.exp(x)
    z = e.sum(-1, keepdim=True)
    p = e / z
    step = torch.arange(K, device=DEV)
    pt = p[:, :K].gather(-1, tok[..., None])[..., 0]
    if s["draft"] is None:
        q = None
        qt = torch.ones_like(pt)
    else:
        d = s["draft"].float()
        f = torch.exp((d - d.amax(-1, keepdim=True)) * inv)
        q = f / f.sum(-1, keepdim=True)
        qt = q.gather(-1, tok[..., None])[..., 0]
    ok = torch.where(greedy[:, None], tok == lowest[:, :K], s["uniform"] * qt < pt)
    ok = ok & (step < lens[:, None])
    n = ok.long().cumprod(-1).sum(-1)                                          # accepted
    rows = torch.arange(B, device=DEV)
    pn = p[rows, n]
    at = n.clamp(max=K - 1)
    if q is None:
        taken = torch.nn.functional.one_hot(tok[rows, at], V).to(pn.dtype)
    else:
        taken = q[rows, at]
    rest = (pn - taken).clamp(min=0)
    if q is None:
        rest = pn * (1 - taken)
    none = (rest.sum(-1) == 0) | (n >= lens)
    rest = torch.where(none[:, None], pn, rest)
    score = rest / s["noise"]
    best = torch.where(score == score.amax(-1, keepdim=True), torch.arange(V, device=DEV), V).amin(-1)
    last = torch.where(greedy, lowest[rows, n], best)
    slot = torch.arange(K1, device=DEV)
    padded = torch.nn.functional.pad(tok, (0, 1))
    out = torch.where(slot < n[:, None], padded, torch.where(slot == n[:, None], last[:, None], -1))
    logp = x.gather(-1, out.clamp(min=0)[..., None])[..., 0] - torch.log(z[..., 0])
    logp = torch.where((out >= 0) & ~greedy[:, None], logp, torch.zeros_like(logp))
    return out, n, logp


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"kv": _kv_plain, "attn": _attn_plain, "kda": _kda_plain, "verify": _verify_plain}[op](s)
    from hanuman_b200 import ops
    if op == "kv":
        cache = ops.KVCache(s["k_cache"], s["v_cache"], s["k_exp"], s["v_exp"])
        ops.kv_cache_write(cache, s["k"], s["v"], s["starts"], s["counts"])
        return list(ops.kv_cache_read(cache, s["starts"], s["k"].shape[1]))
    if op == "attn":
        cache = ops.KVCache(s["k"], s["v"], s["k_exp"], s["v_exp"])
        prefix = ops.KVCache(s["pk"], s["pv"], s["pk_exp"], s["pv_exp"]) if s["case"]["prefix"] else None
        return ops.decode_attention(s["q"], cache, s["lengths"], counts=s["counts"], prefix=prefix,
                                    window=s["case"]["window"])
    if op == "kda":
        return ops.kda_recurrent(s["q"], s["k"], s["v"], s["g"], s["beta"], s["scale"], state=s["state"],
                                 counts=s["counts"])
    return ops.verify_draft(s["target"], s["tokens"], s["uniform"], s["noise"], draft_logits=s["draft"],
                            draft_lens=s["lens"], temperature=s["temperature"])


# --------------------------------------------------------------------- exact
def _wide_pow2(e):
    """2^e as fp64, exactly (a library power may be an ulp off, which moves ties)."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_round(x):
    """The value, in 64 bits, that a row of x has after it was cached."""
    x = x.double()
    out = torch.zeros_like(x)
    amax = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(amax.clamp(min=1e-300) / 448.0))
    e = torch.where(amax > 448.0 * _wide_pow2(e), e + 1, e)
    e = torch.where(amax <= 448.0 * _wide_pow2(e - 1), e - 1, e).clamp(-120, 119)
    y = x / _wide_pow2(e)
    # 3 mantissa bits, the least normal exponent -6: spacing 2^(floor(log2 |y|) - 3)
    _, k = torch.frexp(y)
    step = _wide_pow2((k - 1).clamp(min=-6) - 3)
    out = torch.round(y / step) * step * _wide_pow2(e)
    return torch.where(amax > 0, out, torch.zeros_like(out))


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["op"] == "kv":
        S = c["tokens"]
        live = torch.arange(S, device=DEV)[None, :] < s["counts"][:, None]
        return [torch.where(live[..., None, None], _exact_round(s[x]), torch.zeros((), dtype=torch.float64, device=DEV))
                for x in ("k", "v")]
    if c["op"] == "attn":
        return _exact_attention(s, c)
    if c["op"] == "kda":
        return _exact_recurrence(s, c)
    return _exact_verify(s, c)


def _exact_attention(s, c):
    B, S, Nq, H = s["q"].shape
    N, P = c["kv_heads"], c["prefix"]
    G = Nq // N
    out = torch.zeros(B, S, Nq, H, dtype=torch.float64, device=DEV)
    lengths, counts = s["lengths"].tolist(), s["counts"].tolist()

    def wide(x, e, b, n):
        y = x[b, :, n].double()
        return y if e is None else y * _wide_pow2(e[b, :, n])[:, None]

    for n in range(N):
        pk = wide(s["pk"], s["pk_exp"], 0, n) if P else None
        pv = wide(s["pv"], s["pv_exp"], 0, n) if P else None
        for b in range(B):
            L, cnt = lengths[b], counts[b]
            k, v = wide(s["k"], s["k_exp"], b, n)[:L], wide(s["v"], s["v_exp"], b, n)[:L]
            if P:
                k, v = torch.cat([pk, k]), torch.cat([pv, v])
            q = s["q"][b, :cnt, n * G:(n + 1) * G].double()
            a = (q.reshape(cnt * G, H) @ k.t() / H ** 0.5).view(cnt, G, -1)
            at = P + L - cnt + torch.arange(cnt, device=DEV)[:, None, None]
            kp = torch.arange(P + L, device=DEV)
            hide = kp > at
            if c["window"]:
                hide = hide | (at - kp >= c["window"])
            w = torch.softmax(a.masked_fill(hide, float("-inf")), -1)
            out[b, :cnt, n * G:(n + 1) * G] = (w.view(cnt * G, -1) @ v).view(cnt, G, H)
    return out


def _exact_recurrence(s, c):
    B, S, N, K = s["q"].shape
    d = {x: s[x].double() for x in ("q", "k", "v", "g", "beta")}
    state = s["state"].double().expand(B, N, K, K).clone()
    o = torch.zeros(B, S, N, K, dtype=torch.float64, device=DEV)
    for t in range(S):
        on = (t < s["counts"]).nonzero()[:, 0]
        if not len(on):
            break
        st = state[on] * d["g"][on, t].exp()[..., None]
        k, b = d["k"][on, t], d["beta"][on, t][..., None]
        vn = d["v"][on, t] - b * torch.einsum("bnkv,bnk->bnv", st, k)
        st = st + torch.einsum("bnk,bnv->bnkv", b * k, vn)
        state[on] = st
        o[on, t] = torch.einsum("bnkv,bnk->bnv", st, d["q"][on, t]) * s["scale"]
    return o, state


def _exact_verify(s, c):
    B, K1, V = s["target"].shape
    logp = torch.zeros(B, K1, dtype=torch.float64, device=DEV)
    for b in range(B):
        T = float(s["temperature"][b])
        t = s["target"][b].double()
        n, lens = 0, int(s["lens"][b])
        drawn = s["tokens"][b].tolist()
        if T == 0:
            continue
        lp = torch.log_softmax(t / T, -1)
        lq = None if s["draft"] is None else torch.log_softmax(s["draft"][b].double() / T, -1)
        while n < lens:
            q = 1.0 if lq is None else float(lq[n, drawn[n]].exp())
            if not float(s["uniform"][b, n]) * q < float(lp[n, drawn[n]].exp()):
                break
            logp[b, n] = lp[n, drawn[n]]
            n += 1
        w = lp[n].exp()
        if n < lens:
            r = w.clone()
            if lq is None:
                r[drawn[n]] = 0
            else:
                r = (w - lq[n].exp()).clamp(min=0)
            w = r if float(r.sum()) > 0 else w
        logp[b, n] = lp[n, int((w / s["noise"][b].double()).argmax())]
    return None, None, logp
