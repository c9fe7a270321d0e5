"""Decoding operators: the quantised KV cache, attention over a cache with a
shared prefix, the recurrent gated delta rule with its state, the verification
of drafted tokens.  The plain forms run here in 64 bits; the ``gpu`` tests hold
the kernels against them."""
import math

import pytest
import torch

from hanuman_b200 import ops
from hanuman_b200.ops import reference as ref

gpu = pytest.mark.gpu
DEVS = ["cpu", pytest.param("cuda", marks=gpu)]


def _gen(seed, dev="cpu"):
    return torch.Generator(device=dev).manual_seed(seed)


def _randn(g, *shape, dev="cpu"):
    return torch.randn(*shape, generator=g).to(dev)


def _status_clean():
    from hanuman_b200.ops._ext import ext
    torch.cuda.synchronize()
    s = ext().read_status()
    ext().clear_status()
    return s == 0


# ------------------------------------------------------------------ KV cache
def _round_e4m3(y):
    """Nearest-even e4m3 value of |y| <= 448 from the definition, in 64 bits."""
    y = y.double()
    _, k = torch.frexp(y)
    step = torch.ldexp(torch.ones_like(y), (k - 1).clamp(min=-6) - 3)
    return torch.round(y / step) * step


def _values64(x):
    """What a row of x is worth after quantisation, from the definition."""
    x = x.double()
    a = x.abs().masked_fill(~torch.isfinite(x), 0).amax(-1)
    e = torch.full_like(a, -120)
    for c in range(-120, 119):
        e = torch.where(a > 448.0 * 2.0 ** c, torch.full_like(e, c + 1), e)
    e = e.clamp(max=119).masked_fill(a == 0, 0)
    s = torch.ldexp(torch.ones_like(a), e.int())[..., None]
    return _round_e4m3((x / s).clamp(-448, 448)) * s


def _awkward_rows(H, dev):
    g = _gen(3)
    x = _randn(g, 12, H)
    x[1] = 0
    x[2] = 448.0
    x[3] = 449.0                       # needs the next exponent
    x[4] *= 1e30
    x[5] *= 1e-38                      # exponent at its lower limit
    x[6] *= torch.logspace(-6, 3, H)
    x[7, 3] = float("inf")
    x[7, 4] = -float("inf")
    x[8] = 3.3e38
    x[9] = 2.0 ** -9 * 1.5             # ties
    x[9, 0] = 448.0
    x[10] = -x[10].abs()
    x[11] = float("inf")
    return x.to(dev)


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("H", [32, 64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_kv_cache_rows_are_the_quantised_values(dev, H, dtype):
    """Round trip of awkward rows equals the definition bit for bit (the only
    rounding is e4m3's, whose nearest-even value 64 bits give exactly)."""
    x = _awkward_rows(H, dev).to(dtype)
    k, v = x[None, :, None], (-x)[None, :, None].flip(1)
    cache = ops.new_kv_cache(1, 20, 1, H, dev, torch.float8_e4m3fn)
    ops.kv_cache_write(cache, k, v, 5)
    kb, vb = ops.kv_cache_read(cache, 5, 12)
    assert torch.equal(kb.double(), _values64(k)) and torch.equal(vb.double(), _values64(v))
    rest = ops.kv_cache_read(cache, 0, 5)[0]
    assert torch.equal(rest, torch.zeros_like(rest))   # nothing else was written


@pytest.mark.parametrize("dev", DEVS)
def test_kv_cache_keeps_nan_in_its_place(dev):
    x = _randn(_gen(1), 1, 2, 1, 64)
    x[0, 1, 0, 7] = float("nan")
    x = x.bfloat16().to(dev)
    cache = ops.new_kv_cache(1, 2, 1, 64, dev, torch.float8_e4m3fn)
    ops.kv_cache_write(cache, x, x, 0)
    k, _ = ops.kv_cache_read(cache, 0, 2)
    assert k.isnan().nonzero().tolist() == [[0, 1, 0, 7]]
    clean = x.clone()
    clean[0, 1, 0, 7] = 0
    assert torch.equal(k.nan_to_num(0.0).double(), _values64(clean))


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("B,S,N,H", [(1, 1, 1, 64), (3, 7, 3, 32), (5, 33, 4, 128)])
def test_kv_cache_ragged_strided(dev, quant, B, S, N, H):
    """Column slices of a fused projection, per-sequence starts and counts (0
    among them), into a strided view of a larger cache."""
    g = _gen(B * S)
    buf = _randn(g, B, S, 2 * N * H + 8, dev=dev).bfloat16()
    k = buf[..., 8:8 + N * H].unflatten(-1, (N, H))
    v = buf[..., 8 + N * H:].unflatten(-1, (N, H))
    big = ops.new_kv_cache(B, 2 * (S + 9), N, H, dev, torch.float8_e4m3fn if quant else torch.bfloat16)
    cache = ops.KVCache(*(None if t is None else t[:, ::2] for t in big))
    starts = torch.randint(0, 9, (B,), generator=g).to(dev)
    counts = torch.randint(0, S + 1, (B,), generator=g).to(dev)
    ops.kv_cache_write(cache, k, v, starts, counts)
    kb, vb = ops.kv_cache_read(cache, starts, S)
    live = (torch.arange(S, device=dev) < counts[:, None])[..., None, None]
    for x, y in ((k, kb), (v, vb)):
        want = (_values64(x) if quant else x.double()) * live
        assert torch.equal(y.double(), want)
    if dev == "cuda":
        assert _status_clean()


@gpu
def test_kv_cache_row_outside_the_cache_is_skipped_and_recorded():
    from hanuman_b200.ops._ext import ext
    x = torch.ones(2, 3, 1, 64, device="cuda", dtype=torch.bfloat16)
    cache = ops.new_kv_cache(2, 4, 1, 64, "cuda", torch.float8_e4m3fn)
    ops.kv_cache_write(cache, x, x, torch.tensor([0, 3], device="cuda"))
    torch.cuda.synchronize()
    assert ext().read_status() == 5
    ext().clear_status()
    k, _ = ops.kv_cache_read(cache, 0, 4)
    assert k[0, :3].eq(1).all() and k[0, 3].eq(0).all() and k[1, 3].eq(1).all() and k[1, :3].eq(0).all()
    k, _ = ops.kv_cache_read(cache, 2, 3)    # the last row is outside: zeros, recorded
    torch.cuda.synchronize()
    assert ext().read_status() == 5 and k[:, 2].eq(0).all()
    ext().clear_status()


def test_kv_cache_refusals():
    cache = ops.new_kv_cache(2, 4, 2, 64, "cpu", torch.float8_e4m3fn)
    x = torch.ones(2, 1, 2, 64)
    for bad in (lambda: ops.kv_cache_write(cache, x[:1], x[:1], 0),                  # batch
                lambda: ops.kv_cache_write(cache, x, x.bfloat16(), 0),               # types differ
                lambda: ops.kv_cache_write(cache, x[..., :32], x[..., :32], 0),      # head dim
                lambda: ops.kv_cache_write(cache, x, x, torch.zeros(3)),             # starts
                lambda: ops.kv_cache_write(cache, x, x, torch.zeros(2)),             # not whole numbers
                lambda: ops.kv_cache_write(cache._replace(v_exp=None), x, x, 0),
                lambda: ops.kv_cache_write(ops.KVCache(cache.k, cache.v), x, x, 0),  # codes without exponents
                lambda: ops.kv_cache_write(cache, x.requires_grad_(), x, 0),
                lambda: ops.kv_cache_read(cache, 0, -1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(IndexError):
        ops.kv_cache_write(cache, torch.ones(2, 1, 2, 64), torch.ones(2, 1, 2, 64), 4)


# ----------------------------------------------------------------- attention
def _attn_case(B, S, Nq, N, H, P, C, quant, seed=0, dev="cpu"):
    g = _gen(seed)
    q = (2 * _randn(g, B, S, Nq, H)).bfloat16().to(dev)

    def filled(b, c):
        k, v = (_randn(g, b, c, N, H).bfloat16() for _ in range(2))
        k[:, :, :, 0] *= 4
        cache = ops.new_kv_cache(b, c, N, H, "cpu", torch.float8_e4m3fn if quant else torch.bfloat16)
        if c:
            ops.kv_cache_write(cache, k, v, 0)
        return ops.KVCache(*(None if t is None else t.to(dev) for t in cache))

    return q, filled(B, C), filled(1, P) if P else None, g


def _attn_check(out, q, cache, lengths, counts, prefix, window, scale=None):
    """Against 64 bits: the weights round to bf16 (2^-9 each, at most 2^-9 of
    A = sum_j p_j |v_j|), the output rounds to bf16 (2^-9 of |o| <= A), scores
    and sums are fp32 (far below): |error| <= 2^-8 A, doubled for the exp2 of
    fp32 scores of size up to 2^5, plus an absolute 1e-6."""
    cpu = lambda c: None if c is None else ops.KVCache(*(None if t is None else t.cpu() for t in c))
    cache, prefix = cpu(cache), cpu(prefix)
    args = (lengths.cpu(), None if counts is None else counts.cpu(), prefix, window, scale)
    want = ref.decode_attention(q.cpu().double(), cache, *args)
    k, v = ref.cache_values(cache)
    absv = ops.KVCache(k, v.float().abs())
    if prefix is not None:
        pk, pv = ref.cache_values(prefix)
        args = (args[0], args[1], ops.KVCache(pk, pv.float().abs()), window, scale)
    A = ref.decode_attention(q.cpu().double(), absv, *args)
    err = (out.cpu().double() - want).abs()
    assert torch.isfinite(out).all()
    assert (err <= 2.0 ** -7 * A + 1e-6).all(), (err / (A + 1e-9)).max()
    return want


def test_decode_attention_plain_form_is_causal_attention():
    """The plain form with the prefix copied into every sequence's cache is the
    framework's causal attention at an offset."""
    B, S, Nq, N, H, P, L = 3, 4, 6, 2, 32, 5, 9
    g = _gen(0)
    q = torch.randn(B, S, Nq, H, generator=g, dtype=torch.float64)
    pk, pv = (torch.randn(1, P, N, H, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(B, L, N, H, generator=g, dtype=torch.float64) for _ in range(2))
    for window in (0, 6):
        o = ops.decode_attention(q, ops.KVCache(k, v), L, prefix=ops.KVCache(pk, pv), window=window)
        full_k, full_v = torch.cat([pk.expand(B, -1, -1, -1), k], 1), torch.cat([pv.expand(B, -1, -1, -1), v], 1)
        want = ref.causal_attention(q, full_k, full_v, window, q_offset=P + L - S)
        assert (o - want).abs().max() < 1e-5     # causal_attention computes in fp32


ATTN_SHAPES = [  # B, S, Nq, N, H, P, C
    (1, 1, 1, 1, 64, 0, 1), (1, 1, 16, 4, 64, 0, 300), (2, 1, 8, 8, 32, 33, 40), (3, 2, 12, 4, 128, 7, 65),
    (5, 5, 16, 4, 64, 129, 77), (4, 5, 16, 4, 128, 500, 64), (33, 1, 16, 4, 64, 200, 30), (2, 9, 16, 2, 64, 64, 100),
    (17, 3, 4, 1, 32, 1000, 17), (40, 4, 16, 4, 64, 700, 9), (40, 4, 8, 2, 128, 260, 9), (2, 40, 8, 2, 64, 31, 130),
    (70, 2, 8, 2, 64, 1023, 3)]


@gpu
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("window", [0, 1, 50])
@pytest.mark.parametrize("shape", ATTN_SHAPES)
def test_decode_attention_against_64_bits(shape, quant, window):
    B, S, Nq, N, H, P, C = shape
    q, cache, prefix, g = _attn_case(*shape, quant, dev="cuda")
    lengths = torch.randint(1, C + 1, (B,), generator=g)
    counts = torch.minimum(torch.randint(0, S + 1, (B,), generator=g), lengths)
    lengths[0], counts[0] = C, min(S, C)
    if B > 2:
        lengths[1], counts[1] = 0, 0            # an idle sequence
    lengths, counts = lengths.cuda(), counts.cuda()
    out = ops.decode_attention(q, cache, lengths, counts, prefix, window)
    _attn_check(out, q, cache, lengths, counts, prefix, window)
    idle = torch.arange(S, device="cuda") >= counts[:, None]
    assert out[idle].eq(0).all()
    assert _status_clean()


@gpu
@pytest.mark.parametrize("quant", [False, True])
def test_decode_attention_long_keys_every_split(quant):
    """One sequence of many keys (every CTA a piece) and a batch of one very
    long and many short sequences."""
    q, cache, prefix, g = _attn_case(1, 1, 8, 2, 64, 5000, 20011, quant, dev="cuda")
    L = torch.tensor([20011], device="cuda")
    _attn_check(ops.decode_attention(q, cache, L, prefix=prefix), q, cache, L, None, prefix, 0)
    for H, window in ((64, 0), (64, 700), (128, 0)):   # many rows: every CTA several tiles of two row blocks
        q, cache, prefix, g = _attn_case(64, 4, 8, 2, H, 9001, 12, quant, dev="cuda")
        L = torch.randint(4, 13, (64,), generator=g).cuda()
        _attn_check(ops.decode_attention(q, cache, L, prefix=prefix, window=window), q, cache, L, None, prefix, window)
    q, cache, prefix, g = _attn_case(9, 2, 8, 2, 64, 0, 6000, quant, dev="cuda")
    L = torch.tensor([3, 6000, 2, 31, 32, 33, 64, 2, 5], device="cuda")
    _attn_check(ops.decode_attention(q, cache, L), q, cache, L, None, None, 0)
    assert _status_clean()


@gpu
@pytest.mark.parametrize("quant", [False, True])
def test_decode_attention_never_reads_past_the_lengths(quant):
    """Rows past a sequence's length hold NaN and infinities."""
    q, cache, prefix, g = _attn_case(4, 3, 8, 2, 64, 40, 100, quant, dev="cuda")
    L = torch.tensor([3, 50, 99, 64], device="cuda")
    clean = ops.decode_attention(q, cache, L, prefix=prefix)
    for b in range(4):
        for t in (cache.k, cache.v):
            if quant:
                t.view(torch.uint8)[b, int(L[b]):] = 0x7f       # NaN
            else:
                t[b, int(L[b]):] = float("nan")
        if quant:
            cache.k_exp[b, int(L[b]):] = 127
            cache.v_exp[b, int(L[b]):] = 127
    assert torch.equal(ops.decode_attention(q, cache, L, prefix=prefix), clean)


@gpu
@pytest.mark.parametrize("quant", [False, True])
def test_decode_attention_large_values_and_exponents(quant):
    """Scores far apart, rows scaled by 2^-40 .. 2^20, a query of zeros."""
    g = _gen(8)
    B, N, H, C = 2, 2, 64, 90
    k = _randn(g, B, C, N, H) * 30
    v = _randn(g, B, C, N, H) * torch.exp2(torch.randint(-40, 21, (B, C, N, 1), generator=g).float())
    cache = ops.new_kv_cache(B, C, N, H, "cuda", torch.float8_e4m3fn if quant else torch.bfloat16)
    ops.kv_cache_write(cache, k.bfloat16().cuda(), v.bfloat16().cuda(), 0)
    q = (_randn(g, B, 2, 4, H) * torch.tensor([1e-3, 1.0, 30.0, 0.0])[:, None]).bfloat16().cuda()
    L = torch.tensor([C, 40], device="cuda")
    _attn_check(ops.decode_attention(q, cache, L), q, cache, L, None, None, 0)


@gpu
def test_decode_attention_strided_queries_streams_and_replay():
    """q as a column slice of a fused projection, the cache's head-major order,
    a side stream; the same call twice gives the same bits."""
    g = _gen(4)
    B, S, Nq, N, H, C = 3, 2, 8, 2, 64, 70
    buf = _randn(g, B, S, (Nq + 2 * N) * H, dev="cuda").bfloat16()
    q = buf[..., :Nq * H].unflatten(-1, (Nq, H))
    k, v = (_randn(g, B, N, C, H, dev="cuda").bfloat16().transpose(1, 2) for _ in range(2))
    cache = ops.KVCache(k, v)
    L = torch.tensor([70, 2, 33], device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = ops.decode_attention(q, cache, L)
        again = ops.decode_attention(q, cache, L)
    side.synchronize()
    assert torch.equal(out, again)
    _attn_check(out, q, cache, L, None, None, 0)
    odd = torch.zeros(B * S * Nq * H + 1, device="cuda", dtype=torch.bfloat16)[1:].view(B, S, Nq, H)
    odd.copy_(q)                                     # not 16-byte aligned: copied by the wrapper
    assert torch.equal(ops.decode_attention(odd, cache, L), out)


@gpu
def test_decode_attention_offsets_past_32_bits():
    """Sequences whose rows start more than 2^32 bytes into the cache."""
    N, H, C = 4, 128, 2100000          # 1.07 G elements a sequence
    cache = ops.KVCache(*(torch.zeros(3, C, N, H, dtype=torch.bfloat16, device="cuda") for _ in range(2)))
    g = _gen(5)
    k, v = (_randn(g, 3, 50, N, H).bfloat16().cuda() for _ in range(2))
    ops.kv_cache_write(cache, k, v, C - 50)
    assert torch.equal(ops.kv_cache_read(cache, C - 50, 50)[1], v)
    q = _randn(g, 3, 1, 8, H).bfloat16().cuda()
    # a window of 50 rows: the same as a small cache of those rows
    out = ops.decode_attention(q, cache, C, window=50)
    want = ops.decode_attention(q, ops.KVCache(k, v), 50)
    err = (out.double() - want.double()).abs().max()
    assert err <= 2.0 ** -7 * v.double().abs().max()
    assert _status_clean()


def test_decode_attention_refusals():
    q, cache, prefix, _ = _attn_case(2, 1, 4, 2, 64, 3, 4, True)
    other = ops.new_kv_cache(1, 3, 2, 64, "cpu", torch.bfloat16)
    for bad in (lambda: ops.decode_attention(q[:, :, :3], cache, 1),               # 3 heads over 2
                lambda: ops.decode_attention(q[:1], cache, 1),
                lambda: ops.decode_attention(q, cache, torch.ones(3, dtype=torch.int32)),
                lambda: ops.decode_attention(q, cache, 1, prefix=other),           # another type
                lambda: ops.decode_attention(q, cache, 1, prefix=cache),           # two sequences
                lambda: ops.decode_attention(q, cache, 1, window=-1),
                lambda: ops.decode_attention(q, cache, 1, scale=0.0),
                lambda: ops.decode_attention(q.float().requires_grad_(), cache, 1),
                lambda: ops.decode_attention(q[..., :32], cache, 1)):
        with pytest.raises(ValueError):
            bad()


@gpu
def test_decode_attention_refusals_on_the_gpu():
    q, cache, _, _ = _attn_case(2, 1, 4, 2, 64, 0, 4, False, dev="cuda")
    with pytest.raises(ValueError):
        ops.decode_attention(q.float(), cache, 1)
    with pytest.raises(ValueError):
        ops.decode_attention(q, ops.KVCache(cache.k[..., :48], cache.v[..., :48]), 1)
    with pytest.raises(ValueError):
        ops.decode_attention(q, ops.KVCache(cache.k.cpu(), cache.v.cpu()), 1)


# ------------------------------------------------------- recurrent delta rule
def _kda_case(B, S, H, K, dtype, seed, dev):
    g = _gen(seed)
    unit = lambda x: x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6)
    q, k = (unit(_randn(g, B, S, H, K)).to(dtype) for _ in range(2))
    v = torch.nn.functional.silu(_randn(g, B, S, H, K)).to(dtype)
    decay = -torch.exp(_randn(g, B, S, H, K) - 2)
    beta = torch.sigmoid(_randn(g, B, S, H))
    state = _randn(g, B, H, K, K)
    return [t.to(dev) for t in (q, k, v, decay, beta, state)], g


def _kda_check(o, st, q, k, v, g, beta, scale, state, counts):
    """A token's rounding is sqrt(K + 8) roundings of 2^-24 relative to the state
    and passes on with norm <= 1 (decay <= 1, beta <= 1, |k| <= 1): after S
    tokens sqrt(S (K + 8)) 2^-24 of the largest norm, times 4."""
    B, S, H, K = q.shape
    d = [t.cpu().double() for t in (q, k, v, g, beta)]
    state = None if state is None else state.cpu().double()
    wo = torch.zeros(B, S, H, K, dtype=torch.float64)
    st64 = torch.zeros(B, H, K, K, dtype=torch.float64) if state is None else state.expand(B, H, K, K).clone()
    top = st64.flatten(2).norm(dim=-1).max().clamp(min=1)
    for b in range(B):
        n = S if counts is None else int(counts[b])
        for t in range(n):
            s = st64[b] * d[3][b, t].exp()[..., None]
            vn = d[2][b, t] - d[4][b, t][:, None] * torch.einsum("hkv,hk->hv", s, d[1][b, t])
            s = s + d[4][b, t][:, None, None] * d[1][b, t][..., None] * vn[:, None]
            st64[b] = s
            wo[b, t] = torch.einsum("hkv,hk->hv", s, d[0][b, t]) * scale
            top = max(top, s.flatten(1).norm(dim=-1).max())
    tol = 4 * math.sqrt(max(1, S) * (K + 8)) * 2.0 ** -24 * float(top)
    assert (st.cpu().double() - st64).flatten(2).norm(dim=-1).max() <= tol
    if S:
        assert (o.cpu().double() - wo).norm(dim=-1).max() <= tol


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,S,H,K", [(1, 1, 1, 64), (2, 1, 3, 16), (3, 2, 2, 32), (2, 5, 3, 64), (2, 8, 2, 128),
                                     (2, 9, 2, 64), (3, 37, 2, 128), (2, 70, 3, 64), (1, 33, 2, 16), (1, 17, 1, 32)])
def test_kda_recurrent_against_64_bits(dev, dtype, B, S, H, K):
    (q, k, v, g, beta, state), gen = _kda_case(B, S, H, K, dtype, S * K, dev)
    scale = K ** -0.5
    before = state.clone()
    counts = torch.randint(0, S + 1, (B,), generator=gen).to(dev)
    for st0, cnt in ((state, None), (state, counts), (state[:1], None), (None, counts)):
        o, st = ops.kda_recurrent(q, k, v, g, beta, scale, st0, cnt)
        assert o.dtype == st.dtype == torch.float32
        _kda_check(o, st, q, k, v, g, beta, scale, st0, cnt)
        if cnt is not None:
            idle = torch.arange(S, device=dev) >= cnt[:, None]
            assert o[idle].eq(0).all()
    assert torch.equal(state, before)      # the given state is not written


@pytest.mark.parametrize("dev", DEVS)
def test_kda_recurrent_in_parts_equals_the_whole(dev):
    """Tokens in two calls, the state handed over, give the bits of one call
    within the rounding; no tokens leave the state as it is."""
    (q, k, v, g, beta, state), _ = _kda_case(2, 40, 3, 64, torch.float32, 1, dev)
    o, st = ops.kda_recurrent(q, k, v, g, beta, state=state)
    cut = lambda a, b: [t[:, a:b] for t in (q, k, v, g, beta)]
    o1, s1 = ops.kda_recurrent(*cut(0, 7), state=state)
    o2, s2 = ops.kda_recurrent(*cut(7, 40), state=s1)
    assert (torch.cat([o1, o2], 1) - o).abs().max() < 1e-5 and (s2 - st).abs().max() < 1e-5
    o0, s0 = ops.kda_recurrent(*cut(0, 0), state=state)
    assert o0.shape == (2, 0, 3, 64) and torch.equal(s0, state)
    _, sz = ops.kda_recurrent(*cut(0, 5), state=state, counts=torch.zeros(2, dtype=torch.int64, device=dev))
    assert torch.equal(sz, state)


@gpu
def test_kda_recurrent_strided_rows_and_chunked_form():
    """Head-major and column-sliced inputs; and the training kernels' chunked
    form gives the same outputs from a zero state (their 3xTF32 products: 1e-4)."""
    (q, k, v, g, beta, state), _ = _kda_case(2, 130, 4, 64, torch.float32, 2, "cuda")
    o, st = ops.kda_recurrent(q, k, v, g, beta)
    hm = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)
    o2, st2 = ops.kda_recurrent(hm(q), hm(k), hm(v), hm(g), hm(beta))
    assert torch.equal(o, o2) and torch.equal(st, st2)
    wide = torch.cat([q, k, v], -1)
    o3, _ = ops.kda_recurrent(wide[..., :64], wide[..., 64:128], wide[..., 128:], g, beta)
    assert torch.equal(o, o3)
    oc = ops.kda_core(q, k, v, g, beta, 64 ** -0.5, 64)
    assert (oc - o).norm() / o.norm() < 1e-4


def test_kda_recurrent_refusals():
    (q, k, v, g, beta, state), _ = _kda_case(2, 3, 2, 32, torch.float32, 0, "cpu")
    for bad in (lambda: ops.kda_recurrent(q, k[:, :2], v, g, beta),
                lambda: ops.kda_recurrent(q, k, v, g, beta[..., None]),
                lambda: ops.kda_recurrent(q, k, v, g, beta, state=state[:, :1]),
                lambda: ops.kda_recurrent(q, k, v, g, beta, state=state.double()),
                lambda: ops.kda_recurrent(q.requires_grad_(), k, v, g, beta),
                lambda: ops.kda_recurrent(q.detach(), k, v, g, beta, counts=torch.zeros(3, dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()


# --------------------------------------------------------------- verification
def _verify_case(B, K, V, dtype, seed, with_draft, dev):
    g = _gen(seed)
    t = (2.5 * _randn(g, B, K + 1, V)).to(dtype)
    d = (t[:, :K].float() + 0.7 * _randn(g, B, K, V)).to(dtype)
    temp = 0.5 + torch.rand(B, generator=g)
    temp[::3] = 0.0
    tok = torch.where((temp > 0)[:, None],
                      torch.distributions.Categorical(logits=d.float()).sample() if K else torch.zeros(B, 0).long(),
                      t[:, :K].float().argmax(-1))
    if K:
        tok[B // 2, K - 1] = V - 1
    u = torch.rand(B, K, generator=g)
    e = -torch.log1p(-torch.rand(B, V, generator=g)).clamp(max=-1e-30)
    lens = torch.randint(0, K + 1, (B,), generator=g)
    return [x.to(dev) for x in (t, tok, u, e, d, lens, temp)]


def _verify_same(got, want):
    """Tokens equal; log probabilities: fp32 exponentials of arguments up to 2^5
    (2^-19 absolute) and sums of at most 2^17 values in a tree (2^-20)."""
    assert torch.equal(got[0].cpu(), want[0].cpu()) and torch.equal(got[1].cpu(), want[1].cpu())
    assert (got[2].cpu() - want[2].cpu()).abs().max() <= 2.0 ** -17


@pytest.mark.parametrize("dev", DEVS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 0, 50), (4, 4, 7), (7, 3, 257), (3, 7, 1000), (6, 5, 8191)])
def test_verify_draft_against_64_bits(dev, dtype, B, K, V):
    torch.manual_seed(0)
    for seed in range(3):
        t, tok, u, e, d, lens, temp = _verify_case(B, K, V, dtype, 100 * seed + K, True, dev)
        for draft in (d, None):
            for ln in (lens, None):
                got = ops.verify_draft(t, tok, u, e, draft, ln, temp)
                want = ref.verify_draft(t.cpu().double(), tok.cpu(), u.cpu(), e.cpu(),
                                        None if draft is None else draft.cpu().double(),
                                        None if ln is None else ln.cpu(), temp.cpu())
                _verify_same(got, want)
    if dev == "cuda":
        assert _status_clean()


@pytest.mark.parametrize("dev", DEVS)
def test_verify_draft_masked_rows_ties_and_empty_rows(dev):
    inf = float("inf")
    V = 40
    t = torch.zeros(6, 3, V)
    t[0, 0] = -inf                        # nothing left: no token
    t[1, :, 5:] = torch.finfo(torch.float32).min      # masks of the lowest value
    t[2, 0, :] = torch.finfo(torch.float32).min       # all of them: uniform
    t[3, :, 7] = inf                      # certain
    t[4, :, 3] = float("nan")             # counts as minus infinity
    t[5, :, 11], t[5, :, 29] = 4.0, 4.0   # a tie: the lowest index
    tok = torch.tensor([[1, 1], [2, 30], [0, 0], [7, 8], [3, 1], [11, 29]])
    u = torch.full((6, 2), 0.3)
    e = torch.linspace(1, 2, V).expand(6, V).contiguous()
    for temp in (1.0, 0.0, 0.25):
        args = [x.to(dev) for x in (t, tok, u, e)]
        got = ops.verify_draft(*args, temperature=temp)
        want = ref.verify_draft(t.double(), tok, u, e, None, None, torch.full((6,), temp))
        _verify_same(got, want)
        assert got[0][0].tolist() == [-1, -1, -1] and got[1][0] == 0
    assert got[0][4, 0] != 3


@pytest.mark.parametrize("dev", DEVS)
def test_verify_draft_emits_the_target_distribution(dev):
    """The first emitted token is a draw from the target whatever the draft:
    over 40000 trials every probability within 5 standard deviations."""
    g = _gen(2)
    V, n = 6, 40000
    t, d = _randn(g, 2, V), _randn(g, 1, V)
    q = torch.softmax(d[0] / 0.8, -1)
    tok = torch.multinomial(q, n, replacement=True, generator=g)[:, None]
    u = torch.rand(n, 1, generator=g)
    e = -torch.log1p(-torch.rand(n, V, generator=g)).clamp(max=-1e-30)
    if dev == "cpu":
        n = 4000
        tok, u, e = tok[:n], u[:n], e[:n]
    out, _, _ = ops.verify_draft(t.expand(n, 2, V).to(dev).contiguous(), tok.to(dev), u.to(dev), e.to(dev),
                                 d.expand(n, 1, V).to(dev).contiguous(), temperature=0.8)
    p = torch.softmax(t[0] / 0.8, -1)
    freq = torch.bincount(out[:, 0].cpu(), minlength=V) / n
    assert ((freq - p).abs() <= 5 * torch.sqrt(p * (1 - p) / n)).all()


def test_verify_draft_refusals():
    t, tok, u, e, d, lens, temp = _verify_case(3, 2, 10, torch.float32, 0, True, "cpu")
    for bad in (lambda: ops.verify_draft(t, tok[:, :1], u, e),
                lambda: ops.verify_draft(t, tok.int(), u, e),
                lambda: ops.verify_draft(t, tok, u, e[:, :9]),
                lambda: ops.verify_draft(t, tok, u.double(), e),
                lambda: ops.verify_draft(t, tok, u, e, d[:, :1]),
                lambda: ops.verify_draft(t, tok, u, e, d.bfloat16()),
                lambda: ops.verify_draft(t, tok, u, e, temperature=temp[:2]),
                lambda: ops.verify_draft(t.requires_grad_(), tok, u, e)):
        with pytest.raises(ValueError):
            bad()


@gpu
def test_verify_draft_token_outside_the_vocabulary_is_rejected_and_recorded():
    from hanuman_b200.ops._ext import ext
    t, tok, u, e, d, lens, temp = _verify_case(3, 2, 10, torch.float32, 0, True, "cuda")
    tok[1, 0] = 10
    out, n, _ = ops.verify_draft(t, tok, u, e, d, temperature=1.0)
    torch.cuda.synchronize()
    assert ext().read_status() == 5 and int(n[1]) == 0 and 0 <= int(out[1, 0]) < 10
    ext().clear_status()
