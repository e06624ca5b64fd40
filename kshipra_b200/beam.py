"""Beam search over the block pool.

The beams of a request share the pages of what they have in common: each step's
survivors go through ``fork_pages``, which shares whole pages, copies the page
being filled for all but one of a beam's continuations and frees what no beam
holds any more, all on the GPU.  A step has no host synchronisation (with
``eos_token_id``, one: whether every beam has ended).
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from .kv_cache import fork_pages


class BeamDecoder:
    """Beam search with ``beams`` beams a request through a ``KshipraModel``.

    ``generate(prompts, max_new_tokens)`` returns each request's beams, best first,
    as (tokens, score): the sum of the tokens' log probabilities over
    ``len(tokens) ** length_penalty``.  A beam that emits ``eos_token_id`` (kept)
    stays as it is and competes with the others.  One beam is greedy decoding.
    The cache has the model's ``kv_dtype``.
    """

    def __init__(self, model, beams: int = 4, block_size: int = 16, length_penalty: float = 0.0):
        if model.tp_world > 1:
            raise ValueError("beam search needs the whole vocabulary on one GPU")
        if beams < 1 or block_size < 1:
            raise ValueError("beams and block_size must be positive")
        if beams > model.vocab_size:
            raise ValueError(f"{beams} beams, the vocabulary has {model.vocab_size} tokens")
        self.m = model
        self.beams = beams
        self.block_size = block_size
        self.length_penalty = float(length_penalty)

    @torch.inference_mode()
    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int = 20,
                 eos_token_id: Optional[int] = None,
                 prefill_chunk: Optional[int] = None) -> List[List[Tuple[List[int], float]]]:
        m, bs, K, R = self.m, self.block_size, self.beams, len(prompts)
        if R == 0:
            return []
        if max_new_tokens < 1 or any(len(p) < 1 for p in prompts):
            raise ValueError("prompts need a token and max_new_tokens must be positive")
        longest = max(len(p) for p in prompts) + max_new_tokens - 1
        if longest > m.max_positions:
            raise ValueError(f"{longest} positions, the model has {m.max_positions}")
        if eos_token_id is not None and not 0 <= eos_token_id < m.vocab_size:
            eos_token_id = None                              # never emitted
        with torch.cuda.device(m.device):
            return self._generate(prompts, max_new_tokens, eos_token_id, prefill_chunk)

    def _generate(self, prompts, steps: int, eos: Optional[int], chunk: Optional[int]):
        from .model import _check_flags
        m, bs, K, R, dev = self.m, self.block_size, self.beams, len(prompts), self.m.device
        # pages: the prompt's (all but its last token is cached first), and for each beam
        # those from the one that the prompt ends in on
        own = [-(-(len(p) - 1) // bs) for p in prompts]
        grow = [(len(p) + steps) // bs - (len(p) - 1) // bs + 1 for p in prompts]
        width = max((len(p) + steps) // bs + 1 for p in prompts)
        pool = m.new_pool(sum(own) + K * sum(grow), bs).pool
        tables = torch.zeros((R, width), dtype=torch.int32)
        refs = torch.zeros(pool.shape[0], dtype=torch.int32)
        at = 0
        for i, (p, n) in enumerate(zip(prompts, own)):
            tables[i, :n] = torch.arange(at, at + n, dtype=torch.int32)
            if len(p) > 1:
                m.prefill(list(p[:-1]), pool, list(range(at, at + n)), chunk)
            at += n
        refs[:at] = 1
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        parents = torch.arange(R, dtype=torch.int32, device=dev)
        tables, lens, slots, refs = fork_pages(pool, tables.to(dev), i32([len(p) - 1 for p in prompts]), parents,
                                               refs.to(dev), flags=m.flags)
        tokens = torch.tensor([p[-1] for p in prompts], dtype=torch.int64, device=dev)
        scores = torch.zeros((R, 1), dtype=torch.float32, device=dev)
        ended = torch.zeros((R, 1), dtype=torch.bool, device=dev)
        history = torch.empty((R, 0), dtype=torch.int64, device=dev)
        length = torch.zeros((R, 1), dtype=torch.int64, device=dev)
        base = torch.arange(R, device=dev)[:, None]
        total = max(len(p) for p in prompts)
        for step in range(steps):
            width_now = scores.shape[1]                       # beams a request: 1, then K
            logp = torch.log_softmax(self._logits(tokens, lens, slots, tables, pool, total + step), 1)
            V = logp.shape[1]
            cand = scores[:, :, None] + logp.view(R, width_now, V)
            if eos is not None:                               # an ended beam goes on with itself alone
                cand = cand.masked_fill(ended[:, :, None], -torch.inf)
                cand[:, :, eos] = torch.where(ended, scores, cand[:, :, eos])
            top, idx = cand.view(R, -1).topk(K, 1)
            beam, tok = idx // V, idx % V
            row = (base * width_now + beam).view(-1)          # of the old beams
            done = ended.gather(1, beam)
            history = torch.cat([history[row], tok.view(-1, 1)], 1)
            length = length.gather(1, beam) + (~done).long()
            scores = top
            if eos is not None:
                ended = done | (tok == eos)
            else:
                ended = done
            if step + 1 == steps or (eos is not None and bool(ended.all())):
                break
            tables, lens, slots, refs = fork_pages(pool, tables, lens + 1, row.int(), refs, flags=m.flags)
            tokens = tok.reshape(-1)
        _check_flags(m.flags)
        final = scores / length.to(torch.float32) ** self.length_penalty
        order = final.argsort(dim=1, descending=True, stable=True)
        out = []
        for r, (best, vals, hist, lng) in enumerate(zip(order.tolist(), final.tolist(),
                                                        history.view(R, K, -1).tolist(), length.tolist())):
            out.append([(hist[b][:lng[b]], vals[b]) for b in best])
        return out

    def _logits(self, tokens, lens, slots, tables, pool, longest: int) -> torch.Tensor:
        """Logits [N, vocab] after one token a sequence, at the positions ``lens``."""
        m, N, dev = self.m, tokens.shape[0], self.m.device
        q_start = torch.arange(N + 1, dtype=torch.int32, device=dev)
        hid = m._run_layers(m._alloc_acts(N), tokens, lens.long(), slots, tables, q_start, lens, N, 1, longest, pool,
                            m._lin_ws, m._attn_ws)
        logits = torch.empty((N, m.vocab_size), dtype=torch.float32, device=dev)
        best = torch.empty(N, dtype=torch.int64, device=dev)
        m._lm_head_argmax(hid, best, logits=logits)
        return logits
