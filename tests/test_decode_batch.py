"""Batched decoding on the decoding operators: shared prompts, 8-bit caches and
drafted tokens against decoding one sequence at a time."""
import pytest
import torch

from hanuman_b200.config import get_config
from hanuman_b200.data import get_tokenizer
from hanuman_b200.decode import BatchCache, generate_batch, generate_cached, lookup_draft
from hanuman_b200.models.transformer import Transformer

PROMPTS = ["hello world", "abcabcabcab", "z", "the quick brown fox jumps"]


def _model(name, seed=0, **kw):
    c = get_config(name).replace(dtype="fp32", **kw)
    return Transformer(c, seed=seed), get_tokenizer(c)


@pytest.mark.parametrize("name", ["smoke", "smoke_kda"])
@pytest.mark.parametrize("shared", ["", "once upon a time there was a "])
@pytest.mark.parametrize("draft", ["none", "lookup", "model"])
def test_greedy_batches_give_the_tokens_of_single_decoding(name, shared, draft):
    """Ragged prompts in one batch, with a shared prompt run once, and with
    drafts right and wrong: the greedy tokens of each sequence alone."""
    model, tok = _model(name)
    drafter = _model(name, seed=1)[0] if draft == "model" else None
    got = generate_batch(model, tok, PROMPTS, max_tokens=10, temperature=0.0, shared_prompt=shared,
                         n_draft=0 if draft == "none" else 3, draft_model=drafter)
    for p, (_, ids) in zip(PROMPTS, got):
        _, want = generate_cached(model, tok, shared + p, max_tokens=10, temperature=0.0)
        assert ids == want


def test_a_draft_that_is_the_target_is_always_accepted():
    """With the target as its own draft model every greedy draft is right, so
    12 tokens take 1 + ceil(11 / 4) steps of three drafts."""
    model, tok = _model("smoke_kda")
    steps = []
    real = BatchCache.run
    try:
        BatchCache.run = lambda self, m, t, c=None: (steps.append(t.shape[1]), real(self, m, t, c))[1]
        got = generate_batch(model, tok, ["hello"], max_tokens=12, temperature=0.0, n_draft=3, draft_model=model)
    finally:
        BatchCache.run = real
    _, want = generate_cached(model, tok, "hello", max_tokens=12, temperature=0.0)
    assert got[0][1] == want
    assert steps.count(4) == 2 * 3     # target and draft-cache step per round


def test_sampled_batches_are_reproducible_and_8_bit_caches_run():
    model, tok = _model("smoke_kda")
    a = generate_batch(model, tok, PROMPTS, 8, 0.9, seed=3, n_draft=2)
    assert a == generate_batch(model, tok, PROMPTS, 8, 0.9, seed=3, n_draft=2)
    assert a != generate_batch(model, tok, PROMPTS, 8, 0.9, seed=4, n_draft=2)
    b = generate_batch(model, tok, PROMPTS, 8, 0.0, shared_prompt="again and ", kv_dtype=torch.float8_e4m3fn)
    assert all(len(ids) > len(p) for p, (_, ids) in zip(PROMPTS, b))


def test_lookup_draft():
    assert lookup_draft([1, 2, 3, 4, 1, 2], 3) == [3, 4, 1]
    assert lookup_draft([1, 2, 9, 1, 2, 7, 1, 2], 1) == [7]
    assert lookup_draft([1, 2, 3], 2) == [] and lookup_draft([1], 2) == []


def test_cache_refusals():
    model, _ = _model("smoke_kda")
    cache = BatchCache(model, 2, 3)
    with pytest.raises(ValueError):
        cache.run(model, torch.zeros(2, 4, dtype=torch.int64))
    with pytest.raises(ValueError):
        cache.fork(model, 2, 4)


def test_cli_generates_a_prompt_file(tmp_path, monkeypatch, capsys):
    from hanuman_b200.main import main
    monkeypatch.chdir(tmp_path)
    from hanuman_b200.train import train
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    train(get_config("smoke_kda").replace(train_steps=2, batch_size=2, seq_len=32), log=lambda *a, **k: None)
    (tmp_path / "p.txt").write_text("hello\n\nworld\n")
    main(["generate", "--config", "smoke_kda", "--prompt_file", "p.txt", "--max_tokens", "4", "--temperature", "0",
          "--shared_prompt", "say ", "--n_draft", "2", "--kv", "fp8"])
    out = capsys.readouterr().out
    assert "=== Generated 0 ===" in out and "=== Generated 1 ===" in out and "=== Generated 2" not in out


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_batch_cache_on_gpu_matches_full_recompute(kv):
    """Teacher-forced logits of ragged steps behind a shared prefix, kept in part,
    against the full forward of each sequence (bf16 projections 5e-2; e4m3 rows
    round to 2^-4 of a value, averaged over the keys: 1e-1)."""
    from hanuman_b200.train import Trainer
    c = get_config("tiny_hybrid").replace(dtype="bf16", router_type="sigmoid_bias", layers=4)
    model = Trainer(c, device="cuda").model
    for m in model.moe_layers():       # pin the routing: a nearly tied expert may swap
        b = torch.zeros_like(m.bias)
        b[1], b[5] = 20.0, 19.0
        m.bias.data.copy_(b)
    g = torch.Generator().manual_seed(3)
    P, B, L = 37, 3, 30
    pre = torch.randint(0, c.vocab_size, (P,), generator=g).cuda()
    own = torch.randint(0, c.vocab_size, (B, L), generator=g).cuda()
    with torch.no_grad():
        seq = torch.cat([pre.expand(B, -1), own], 1)
        full = model.logits(model(seq)[0]).float()[:, P:]
        one = BatchCache(model, 1, P, torch.float8_e4m3fn if kv == "fp8" else None)
        one.run(model, pre[None])
        one.commit()
        cache = one.fork(model, B, 64)
        done = torch.zeros(B, dtype=torch.int64)
        worst = 0.0
        for step in range(12):
            S = [1, 4, 2, 5][step % 4]
            cnt = torch.minimum(torch.randint(0, S + 1, (B,), generator=g), L - done).clamp(min=0)
            keep = torch.minimum(torch.randint(0, S + 1, (B,), generator=g), cnt)
            at = (done[:, None] + torch.arange(S)).clamp(max=L - 1)
            h = cache.run(model, torch.gather(own, 1, at.cuda()), cnt.cuda())
            got = model.logits(h).float()
            for b in range(B):
                n = int(cnt[b])
                want = full[b, int(done[b]):int(done[b]) + n]
                if n:
                    worst = max(worst, ((got[b, :n] - want).norm(dim=-1) / want.norm(dim=-1)).max().item())
            cache.commit(keep.cuda())
            done += keep
            cache.at_most(int(done.max()))
    assert worst < (5e-2 if kv == "bf16" else 1e-1), worst
    from hanuman_b200.ops._ext import ext
    torch.cuda.synchronize()
    assert ext().read_status() == 0


@pytest.mark.gpu
def test_generate_batch_on_gpu_runs_with_drafts():
    """Greedy tokens do not depend on the drafts (same kernels, other step
    sizes: the logits differ by bf16 rounding, so the first tokens are compared)."""
    from hanuman_b200.train import Trainer
    c = get_config("tiny_hybrid").replace(dtype="bf16")
    tr = Trainer(c, device="cuda")
    tok = get_tokenizer(c)
    a = generate_batch(tr.model, tok, PROMPTS, 6, 0.0, shared_prompt="once upon a time ")
    b = generate_batch(tr.model, tok, PROMPTS, 6, 0.0, shared_prompt="once upon a time ", n_draft=3, draft_model=tr.model)
    assert [len(x[1]) for x in a] == [len(x[1]) for x in b]
    n = len(tok.encode("once upon a time "))
    for p, x, y in zip(PROMPTS, a, b):
        k = n + len(tok.encode(p))
        assert x[1][:k + 1] == y[1][:k + 1]
