"""Greedy and sampled generation with chunked prefill (greedy: yoco/criterions/needle_haystack.py:135-160).

The prompt except its last token is prefilled in chunks of ``chunk_length`` tokens with ``skip_cross_decoder=True``
(YOCO fills the self-decoder states and the single shared K/V cache only; the cross-decoder layers do not run over
the prompt), then each step feeds the previous token, masks BOS and PAD out of the logits, takes the argmax, and
stops once every row produced EOS. Works for any model with the ``model(ids, start_pos=, incremental_state=,
is_prefilling=, skip_cross_decoder=)`` signature (YOCO, and LLaMA which ignores the YOCO-only flags).

With ``temperature`` > 0 the next token is drawn (``ops.sample``) instead of the argmax. With ``num_samples`` > 1 every
prompt is prefilled once and continued ``num_samples`` times: YOCO's shared K/V of the prompt stays stored once and the
continuations decode against it together (``YOCO.fork_state``, ``ops.shared_prefix_attention``); other models repeat
the prompt. The reference generates greedily only.
"""
from __future__ import annotations

import math

from typing import Optional

import torch

from .. import ops
from ..parallel import tp as TP


@torch.no_grad()
def generate(model, prompt: torch.Tensor, tokenizer, generate_tokens: int = 20, chunk_length: int = 32768,
             yoco: bool = True, num_samples: int = 1, temperature: float = 0.0, top_k: int = 0, top_p: float = 1.0,
             min_p: float = 0.0, generator: Optional[torch.Generator] = None) -> torch.Tensor:
    """prompt: [B, P] ids on the model's device -> [B * num_samples, P + generate_tokens] (pad where nothing was
    produced); rows b * num_samples .. (b + 1) * num_samples - 1 continue prompt b. temperature 0 is greedy; top_k,
    top_p and min_p as in ``ops.sample``; generator: source of its uniform numbers (on the model's device; of
    tensor-parallel ranks the first one's decide). A sampled row whose logits leave nothing to draw (all NaN or -inf)
    raises RuntimeError."""
    if num_samples < 1 or not temperature >= 0:
        raise ValueError(f"generate: num_samples = {num_samples}, temperature = {temperature}")
    fork = num_samples > 1 and yoco and hasattr(model, "fork_state")
    if num_samples > 1 and not fork:
        prompt = prompt.repeat_interleave(num_samples, 0)
    B, P = prompt.shape
    dev = prompt.device
    out = torch.cat([prompt, torch.full((B, generate_tokens), tokenizer.pad_id, dtype=torch.long, device=dev)], 1)
    begin = P
    state = {}
    eos = torch.zeros(B, dtype=torch.bool, device=dev)
    extra = {"skip_cross_decoder": True} if yoco else {}
    for s in range(0, begin - 1, chunk_length):
        e = min(s + chunk_length, begin - 1)
        model(out[:, s:e], incremental_state=state, start_pos=s, is_prefilling=True, **extra)
    if fork:
        state = model.fork_state(state, B, num_samples)
        out = out.repeat_interleave(num_samples, 0)
        eos = eos.repeat_interleave(num_samples, 0)
    extra = {"skip_cross_decoder": False} if yoco else {}
    for idx in range(begin, out.shape[1]):
        logits, _ = model(out[:, idx - 1:idx], incremental_state=state, start_pos=idx - 1, is_prefilling=False,
                          **extra)
        logits = logits[:, -1, :].float()
        logits[:, tokenizer.bos_id] = -math.inf
        logits[:, tokenizer.pad_id] = -math.inf
        if temperature > 0:
            u = torch.rand(logits.shape[0], generator=generator, device=dev)
            nxt = TP.from_first_rank(ops.sample(logits, u, temperature, top_k, top_p, min_p))
        else:
            nxt = logits.argmax(-1)
        cur = out[:, idx]
        live = (cur == tokenizer.pad_id) & ~eos
        stuck = live & (nxt < 0)           # ops.sample's -1: a row without candidates, no token to go on with
        nxt = torch.where(live, nxt, cur)
        out[:, idx] = nxt
        eos |= nxt == tokenizer.eos_id
        ended, failed = torch.stack([eos.all(), stuck.any()]).tolist()
        if failed:
            raise RuntimeError(f"generate: no token can be drawn at position {idx} for rows "
                               f"{stuck.nonzero().flatten().tolist()}: all their logits are NaN or -inf")
        if ended:
            break
    return out
