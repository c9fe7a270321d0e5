"""Verification of drafted tokens (csrc/serve/verify.cu); the public entry point
is :func:`hanuman_b200.ops.verify_draft`."""
from __future__ import annotations

import torch

from . import reference as ref
from ._ext import ext
from .kv_cache import _int32, _need, _no_grad

MAX_DRAFTED = 32


def verify_draft(target_logits, draft_tokens, uniform, noise, draft_logits=None, draft_lens=None, temperature=1.0):
    t = target_logits
    _need(t.dim() == 3 and t.shape[1] >= 1 and t.shape[2] >= 1, "verify_draft: target logits [B, K + 1, V]")
    B, K, V = t.shape[0], t.shape[1] - 1, t.shape[2]
    device = t.device
    _need(draft_tokens.shape == (B, K) and draft_tokens.dtype == torch.int64 and draft_tokens.device == device,
          f"verify_draft: drafted tokens [{B}, {K}] int64")
    _need(uniform.shape == (B, K) and uniform.dtype == torch.float32 and uniform.device == device,
          f"verify_draft: uniform [{B}, {K}] fp32")
    _need(noise.shape == (B, V) and noise.dtype == torch.float32 and noise.device == device,
          f"verify_draft: noise [{B}, {V}] fp32")
    if draft_logits is not None:
        _need(draft_logits.shape == (B, K, V) and draft_logits.dtype == t.dtype and draft_logits.device == device,
              f"verify_draft: draft logits [{B}, {K}, {V}] of the target's type")
    _no_grad("verify_draft", t, draft_logits)
    lens = None if draft_lens is None else _int32(draft_lens, "verify_draft: draft_lens", B, device)
    temps, temp = None, 1.0
    if isinstance(temperature, torch.Tensor):
        _need(temperature.shape == (B,) and temperature.dtype == torch.float32 and temperature.device == device,
              f"verify_draft: temperature [{B}] fp32, or a number")
        temps = temperature.contiguous()
    else:
        temp = float(temperature)
    if not t.is_cuda:
        temps = torch.full((B,), temp) if temps is None else temps
        return ref.verify_draft(t, draft_tokens, uniform, noise, draft_logits, lens, temps)
    _need(t.dtype in (torch.float32, torch.bfloat16), "verify_draft: fp32 or bf16 logits")
    _need(K <= MAX_DRAFTED, f"verify_draft: at most {MAX_DRAFTED} drafted tokens")
    out = torch.empty(B, K + 1, dtype=torch.int64, device=device)
    accepted = torch.empty(B, dtype=torch.int64, device=device)
    logp = torch.empty(B, K + 1, dtype=torch.float32, device=device)
    ext().verify_draft(t.contiguous(), None if draft_logits is None else draft_logits.contiguous(),
                       draft_tokens.contiguous(), uniform.contiguous(), noise.contiguous(), lens, temps, temp, out,
                       accepted, logp)
    return out, accepted, logp
